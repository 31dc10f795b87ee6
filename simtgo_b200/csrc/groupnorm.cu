// groupnorm.cu -- group norm with an activation over channels-last batches,
// forward and backward, with the input kept as an 8-bit checkpoint on request.
//
// Mathematics. A thread sums x - K and (x - K)^2, K being the first value it
// meets: the shift keeps the variance exact to a few ulps however far the mean
// is from zero, since K is one of the values that are summed. Threads, blocks
// and chunks of a sample are then joined by counts, means and sums of squared
// deviations (Chan, Golub and LeVeque's pairwise formula), never by raw
// squares; a mean stays K plus a small offset until the last join, so
// differences of means do not cancel. The backward pass needs, for each channel
// of a sample, A = sum dz and B = sum dz*xh: weighted and summed over a group's
// channels they give the group's two means in dx, and summed over the samples
// they are dbias and dweight, so one pass over x and dy serves both. All joins
// run in a fixed order.
//
// Two ways through the data, both reading it once from HBM:
//
// - k_norm, k_norm_back: a cluster of up to eight blocks takes a slab of whole
//   groups of one sample. Each block sums its share of the rows, keeping them in
//   shared memory (what does not fit is read again, last rows first, from L2);
//   the blocks exchange their sums over distributed shared memory, and each
//   finishes its own rows. One launch, nothing in HBM between.
// - k_stats, k_join, k_apply (and their backward forms): where too few such
//   clusters exist to fill the GPU -- a few samples of very many positions --
//   every SM takes a chunk of a sample's rows, the chunks' sums are joined by a
//   small kernel, and a third pass walks the chunks from their ends, whose rows
//   L2 still holds.
#include <algorithm>
#include <atomic>
#include <cmath>
#include <numeric>
#include <type_traits>

#include "channels.cuh"

using namespace chan;

namespace {

constexpr int kThreads = 256;
constexpr int64_t kMaxElems = int64_t(1) << 46;

struct Batch {
    const void *x, *dy, *w, *b;
    void* out;  // y, or dx
    const float *mean, *rstd;
    float *mean_out, *rstd_out;
    const int32_t* lengths;
    Kept kept;  // written forward, read backward
    int64_t xs, xr, ys, yr, os, orow;
    int n, s, c, g, d;
    int units, tile, tiles, phases;  // of a row, or of a slab's row
    int slab, slabs;                 // channels of a cluster's slab, slabs of a sample
    int chunks;                      // blocks that share a sample's rows
    int keep;                        // iterations whose rows stay in shared memory
    int ptype, act;
    float param, eps;
};

// Rows a thread loads before it uses any: while summing, and while finishing.
template <class T>
constexpr int kSumRows = sizeof(T) == 2 ? 8 : 4;
template <class T>
constexpr int kOutRows = sizeof(T) == 2 ? 4 : 2;

__device__ __forceinline__ int valid_rows(const Batch& B, int n) {
    return B.lengths ? min(max(__ldg(B.lengths + n), 0), B.s) : B.s;
}
// Rows [r0, r1) of chunk k of a sample of len rows.
__device__ __forceinline__ void chunk_rows(int len, int chunks, int k, int& r0, int& r1) {
    const int per = (len + chunks - 1) / chunks;
    r0 = (int)min((int64_t)k * per, (int64_t)len);
    r1 = min(r0 + per, len);
}

// ---- between blocks and grids --------------------------------------------------

__device__ __forceinline__ void cluster_arrive() {
    asm volatile("barrier.cluster.arrive.release;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() {
    asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
}
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
// The word at p's place in the shared memory of the cluster's block `rank`.
__device__ __forceinline__ float ld_cluster(const float* p, uint32_t rank) {
    uint32_t a = (uint32_t)__cvta_generic_to_shared(p), r;
    float v;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(rank));
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(r) : "memory");
    return v;
}
// Programmatic dependent launch: the kernel before has finished; the kernel
// after may take the SMs that are free.
__device__ __forceinline__ void grid_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void grid_release() {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

// ---- sums ---------------------------------------------------------------------
// A cell is what a thread sums together: a channel, or -- where groups are whole
// units (kSame) -- a unit.

struct Moments {  // the mean is k + off; m2: the sum of squared deviations from it
    float k, off, m2;
};

// Joins (na, a) and (nb, b).
__device__ __forceinline__ Moments join(float na, Moments a, float nb, Moments b) {
    if (na == 0.0f) return b;
    const float f = nb / (na + nb), d = nb > 0.0f ? (b.k - a.k) + (b.off - a.off) : 0.0f;
    return {a.k, __fmaf_rn(d, f, a.off), __fmaf_rn(d * d, na * f, a.m2 + b.m2)};
}

// Joins the phases of a block's threads: red holds phase p's moments of
// cell i at [p*width + i], cnt[p] its count. Phase 0 ends with them all. Every
// thread calls it, after a barrier.
template <int E>
__device__ void join_phases(Moments* red, float* cnt, int phases, int width, int phase, int cell) {
    float* in = cnt;
    float* out = cnt + kThreads;
    for (int m = phases; m > 1;) {
        const int h = (m + 1) / 2;
        if (phase < h) {
            const bool two = phase + h < m;
            const float na = in[phase], nb = two ? in[phase + h] : 0.0f;
            if (two) {
#pragma unroll
                for (int i = 0; i < E; i++) {
                    Moments* a = red + phase * width + cell + i;
                    *a = join(na, *a, nb, a[h * width]);
                }
            }
            if (cell == 0) out[phase] = na + nb;
        }
        float* t = in;
        in = out;
        out = t;
        m = h;
        __syncthreads();
    }
}

// Moments of this thread's cells over rows r0 + phase, + phases, ... < r1;
// keep(it, raw) is handed every row's unit. Returns the number of rows.
template <class T, int AW, bool kSame, class F>
__device__ __forceinline__ int unit_moments(const T* x, int64_t pitch, int r, int r1, int step,
                                            int cnt, Moments (&out)[kSame ? 1 : 8], F&& keep) {
    constexpr int U = kSumRows<T>, P = kSame ? 1 : 4;
    if (r >= r1) {
#pragma unroll
        for (int i = 0; i < (kSame ? 1 : 8); i++) out[i] = {0.0f, 0.0f, 0.0f};
        return 0;
    }
    float2 k[P], s1[P] = {}, s2[P] = {};
    const int n = (r1 - r + step - 1) / step;
    const T* at = x + (int64_t)r * pitch;
    const int64_t next = step * pitch;
    bool first = true;
    for (int it = 0; it < n; it += U) {
        Raw<T> raw[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (it + u < n) raw[u] = ld_unit<T, AW>(at, cnt);
            at += next;
        }
        if (first) {
            const V8 v = unpack(raw[0]);
#pragma unroll
            for (int i = 0; i < P; i++) k[i] = kSame ? both(v.p[0].x) : v.p[i];
            first = false;
        }
#pragma unroll
        for (int u = 0; u < U; u++)
            if (it + u < n) {
                keep(it + u, raw[u]);
                const V8 v = unpack(raw[u]);
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float2 dv = sub2(v.p[i], k[kSame ? 0 : i]);
                    s1[kSame ? 0 : i] = add2(s1[kSame ? 0 : i], dv);
                    s2[kSame ? 0 : i] = fma2(dv, dv, s2[kSame ? 0 : i]);
                }
            }
    }
    if (kSame) {
        const float a = s1[0].x + s1[0].y, q = s2[0].x + s2[0].y, m = a / (float)(8 * n);
        const float m2 = __fmaf_rn(-m, a, q);
        out[0] = {k[0].x, m, m2 < 0.0f ? 0.0f : m2};
    } else {
        const float inv = 1.0f / (float)n;
#pragma unroll
        for (int i = 0; i < (kSame ? 1 : 8); i++) {
            const float2 a = s1[i / 2 % P], q = s2[i / 2 % P], kk = k[i / 2 % P];
            const float m = (i & 1 ? a.y : a.x) * inv;
            const float m2 = __fmaf_rn(-m, i & 1 ? a.y : a.x, i & 1 ? q.y : q.x);
            out[i] = {i & 1 ? kk.y : kk.x, m, m2 < 0.0f ? 0.0f : m2};
        }
    }
    return n;
}

// Group moments from the moments of `d` cells each of `count` values: sub-warps
// take a group each; f(group, moments) on the sub-warp's first lane.
template <class F>
__device__ __forceinline__ void group_moments(const Moments* cells, int groups, int d, float count,
                                              F&& f) {
    int lanes = 1;
    while (lanes < d && lanes < 32) lanes *= 2;
    const int per = kThreads / lanes, lane = threadIdx.x % lanes;
    for (int g0 = 0; g0 < groups; g0 += per) {
        const int g = g0 + threadIdx.x / lanes;
        const Moments* c = cells + (int64_t)g * d;
        const float k = g < groups ? c[0].k : 0.0f;
        float off = 0.0f, m2 = 0.0f;
        if (g < groups)
            for (int i = lane; i < d; i += lanes) off += (c[i].k - k) + c[i].off;
        for (int o = lanes / 2; o; o /= 2) off += __shfl_xor_sync(~0u, off, o);
        off /= (float)d;
        if (g < groups)
            for (int i = lane; i < d; i += lanes) {
                const float dv = (c[i].k - k) + (c[i].off - off);
                m2 += __fmaf_rn(count * dv, dv, c[i].m2);
            }
        for (int o = lanes / 2; o; o /= 2) m2 += __shfl_xor_sync(~0u, m2, o);
        if (g < groups && lane == 0) f(g, Moments{k, off, m2});
    }
}

// ---- a unit's parameters ---------------------------------------------------------

__device__ __forceinline__ V8 ld_params(const void* p, int type, int c0, int cnt, float fallback) {
    V8 v;
    float f[8];
    if (!p) {
#pragma unroll
        for (int i = 0; i < 4; i++) v.p[i] = both(fallback);
        return v;
    }
    const char* at = (const char*)p + (int64_t)c0 * (type == SIMTGO_F32 ? 4 : 2);
    if (cnt == kUnit && ((uintptr_t)at & 15) == 0) {
        if (type == SIMTGO_F32) return unpack(ld_unit<float, 16>((const float*)at, 8));
        if (type == SIMTGO_BF16)
            return unpack(ld_unit<__nv_bfloat16, 16>((const __nv_bfloat16*)at, 8));
        return unpack(ld_unit<__half, 16>((const __half*)at, 8));
    }
#pragma unroll
    for (int i = 0; i < 8; i++) f[i] = i < cnt ? ld_param(p, type, c0 + i) : 0.0f;
#pragma unroll
    for (int i = 0; i < 4; i++) v.p[i] = make_float2(f[2 * i], f[2 * i + 1]);
    return v;
}

// One value per group, spread over a unit's channels.
template <bool kSame>
struct PerGroup {
    float2 v[kSame ? 1 : 4];
    __device__ __forceinline__ float2 operator[](int i) const { return v[kSame ? 0 : i]; }
};
// f(group) for each of the unit's channels, at most `last`: the unit's first
// group by a division, the next ones by counting.
template <bool kSame, class F>
__device__ __forceinline__ PerGroup<kSame> per_group(int c0, int last, int d, F&& f) {
    PerGroup<kSame> r;
    int g = c0 / d;
    if (kSame) {
        r.v[0] = both(f(g));
        return r;
    }
    int in = c0 - g * d;
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; i++) {
        v[i] = f(g);
        if (c0 + i < last && ++in == d) {
            in = 0;
            g++;
        }
    }
#pragma unroll
    for (int i = 0; i < (kSame ? 1 : 4); i++) r.v[i] = make_float2(v[2 * i], v[2 * i + 1]);
    return r;
}

// ---- finishing rows, forward -----------------------------------------------------------

// y (and the checkpoint) of rows [r0, r1) of this thread's unit, last rows
// first; rows of iterations below B.keep come from `kept_rows`.
template <class T, int AW, bool kSame, bool kKeep>
__device__ __forceinline__ void apply_rows(const Batch& B, int n, int r0, int r1, int phase,
                                           int unit, int cnt, bool on, const PerGroup<kSame>& mean,
                                           const V8& scale, const V8& bias,
                                           const Raw<T>* kept_rows) {
    constexpr int U = kOutRows<T>;
    const int most = (r1 - r0 + B.phases - 1) / B.phases;
    if (most <= 0) return;
    const int rows = phase < B.phases ? (r1 - r0 - phase + B.phases - 1) / B.phases : 0;
    int it = (most - 1) / U * U;
    const int64_t row = r0 + phase + (int64_t)it * B.phases;
    const T* x = (const T*)B.x + n * B.xs + row * B.xr + unit * kUnit;
    T* y = (T*)B.out + n * B.os + row * B.orow + unit * kUnit;
    const int64_t xstep = B.phases * B.xr, ystep = B.phases * B.orow;
    KeptAt kept;
    if (kKeep) kept = kept_at(B.kept, (int64_t)n * B.s + row, B.phases, unit);
    for (; it >= 0; it -= U) {
        bool live[U];
        Raw<T> raw[U] = {};
#pragma unroll
        for (int u = 0; u < U; u++) live[u] = it + u < rows;
        if (it + U <= B.keep) {
#pragma unroll
            for (int u = 0; u < U; u++)
                if (on && live[u]) raw[u] = kept_rows[(it + u) * kThreads + threadIdx.x];
        } else {
            const T* at = x;
#pragma unroll
            for (int u = 0; u < U; u++) {
                if (on && live[u]) raw[u] = ld_unit<T, AW>(at, cnt);
                at += xstep;
            }
        }
        T* to = y;
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (on && live[u]) {
                V8 v = unpack(raw[u]);
#pragma unroll
                for (int i = 0; i < 4; i++)
                    v.p[i] = fma2(sub2(v.p[i], mean[i]), scale.p[i], bias.p[i]);
                activate<sizeof(T) == 2>(v, B.act, B.param);
                Raw<T> o;
                pack(v, o);
                st_unit<T, AW>(to, o, cnt);
            }
            to += ystep;
        }
        if (kKeep) {
            keep_units<T, AW, U>(raw, B.kept, kept, live, unit, cnt, on);
            kept.codes -= U * kept.codes_step;
            kept.scale -= U * kept.scale_step;
        }
        x -= U * xstep;
        y -= U * ystep;
    }
}

// ---- forward in one launch: a cluster per slab of a sample -------------------------------

template <class T, int AW, bool kSame, bool kKeep>
__global__ void __launch_bounds__(kThreads, 2) k_norm(Batch B) {
    constexpr int E = kSame ? 1 : 8;
    extern __shared__ uint4 dyn[];
    __shared__ float cnt_sm[2 * kThreads];
    const int phase = threadIdx.x / B.tile, u = threadIdx.x % B.tile, width = B.tile * E;
    Raw<T>* rows_sm = reinterpret_cast<Raw<T>*>(dyn);
    float2* stat = reinterpret_cast<float2*>(rows_sm + B.keep * kThreads);  // mean, rstd
    Moments* red = reinterpret_cast<Moments*>(stat + B.slab / B.d);
    Moments* own = red + B.phases * width;                                  // this block's groups

    const int rank = (int)cluster_rank();
    const int id = blockIdx.x / B.chunks, n = id / B.slabs, c0 = id % B.slabs * B.slab;
    const int cw = min(B.slab, B.c - c0), groups = cw / B.d, g0 = c0 / B.d;
    const int len = valid_rows(B, n);
    int r0, r1;
    chunk_rows(len, B.chunks, rank, r0, r1);
    const int unit = c0 / kUnit + u, cnt = min(kUnit, c0 + cw - unit * kUnit);
    const bool on = phase < B.phases && u * kUnit < cw;

    Moments m[E] = {};
    int rows = 0;
    if (on)
        rows = unit_moments<T, AW, kSame>(
            (const T*)B.x + (int64_t)n * B.xs + unit * kUnit, B.xr, r0 + phase, r1, B.phases, cnt,
            m, [&](int it, const Raw<T>& raw) {
                if (it < B.keep) rows_sm[it * kThreads + threadIdx.x] = raw;
            });
    V8 scale = ld_params(on ? B.w : nullptr, B.ptype, unit * kUnit, cnt, 1.0f);
    const V8 bias = ld_params(on ? B.b : nullptr, B.ptype, unit * kUnit, cnt, 0.0f);
    if (phase < B.phases) {
#pragma unroll
        for (int i = 0; i < E; i++) red[phase * width + u * E + i] = m[i];
        if (u == 0) cnt_sm[phase] = (float)(rows * (kSame ? kUnit : 1));
    }
    __syncthreads();
    join_phases<E>(red, cnt_sm, B.phases, width, phase, u * E);
    const int cells = kSame ? B.d / kUnit : B.d, per = kSame ? kUnit : 1;
    group_moments(red, groups, cells, (float)(r1 - r0) * per,
                  [&](int g, Moments q) { own[g] = q; });
    cluster_arrive();
    cluster_wait();
    for (int g = threadIdx.x; g < groups; g += kThreads) {
        Moments q = {0.0f, 0.0f, 0.0f};
        float have = 0.0f;
        for (int k = 0; k < B.chunks; k++) {
            int a, b;
            chunk_rows(len, B.chunks, k, a, b);
            const float c = (float)(b - a) * (float)B.d;
            const Moments o = {ld_cluster(&own[g].k, k), ld_cluster(&own[g].off, k),
                               ld_cluster(&own[g].m2, k)};
            if (c > 0.0f) q = join(have, q, c, o);
            have += c;
        }
        const float mu = q.k + q.off, var = have > 0.0f ? q.m2 / have : 0.0f;
        const float rs = __fdiv_rn(1.0f, __fsqrt_rn(var + B.eps));
        stat[g] = make_float2(mu, rs);
        if (rank == 0) {
            const int64_t at = (int64_t)n * B.g + g0 + g;
            if (B.mean_out) B.mean_out[at] = mu;
            if (B.rstd_out) B.rstd_out[at] = rs;
        }
    }
    cluster_arrive();  // the others' shared memory has been read
    __syncthreads();
    const int last = c0 + cw - 1, first = min(unit * kUnit, last);
    const auto mean = per_group<kSame>(first, last, B.d, [&](int g) { return stat[g - g0].x; });
    const auto rstd = per_group<kSame>(first, last, B.d, [&](int g) { return stat[g - g0].y; });
#pragma unroll
    for (int i = 0; i < 4; i++) scale.p[i] = mul2(scale.p[i], rstd[i]);
    apply_rows<T, AW, kSame, kKeep>(B, n, r0, r1, phase, unit, cnt, on, mean, scale, bias, rows_sm);
    cluster_wait();
}

// ---- forward over chunks: moments, joined, then applied ---------------------------

template <class T, int AW, bool kSame>
__global__ void __launch_bounds__(kThreads, 2) k_stats(Batch B, Moments* __restrict__ part) {
    constexpr int E = kSame ? 1 : 8;
    extern __shared__ Moments sm[];
    __shared__ float cnt_sm[2 * kThreads];
    Moments* cell_m = sm;                         // every cell of the row
    Moments* red = sm + (int64_t)B.units * E;     // phases * tile * E
    const int n = blockIdx.x / B.chunks, k = blockIdx.x % B.chunks;
    int r0, r1;
    chunk_rows(valid_rows(B, n), B.chunks, k, r0, r1);
    const T* x = (const T*)B.x + (int64_t)n * B.xs;
    const int phase = threadIdx.x / B.tile, u = threadIdx.x % B.tile, width = B.tile * E;
    for (int t = 0; t < B.tiles; t++) {
        const int unit = t * B.tile + u;
        if (phase < B.phases) {
            Moments m[E] = {};
            int rows = 0;
            if (unit < B.units)
                rows = unit_moments<T, AW, kSame>(x + unit * kUnit, B.xr, r0 + phase, r1, B.phases,
                                                  min(kUnit, B.c - unit * kUnit), m,
                                                  [](int, const Raw<T>&) {});
#pragma unroll
            for (int i = 0; i < E; i++) red[phase * width + u * E + i] = m[i];
            if (u == 0) cnt_sm[phase] = (float)(rows * (kSame ? kUnit : 1));
        }
        __syncthreads();
        join_phases<E>(red, cnt_sm, B.phases, width, phase, u * E);
        if (phase == 0 && unit < B.units) {
#pragma unroll
            for (int i = 0; i < E; i++) cell_m[unit * E + i] = red[u * E + i];
        }
        __syncthreads();
    }
    grid_release();
    Moments* o = part + ((int64_t)n * B.chunks + k) * B.g;
    group_moments(cell_m, B.g, kSame ? B.d / kUnit : B.d, (float)(r1 - r0) * (kSame ? kUnit : 1),
                  [&](int g, Moments m) { o[g] = m; });
}

// A block joins the chunks of up to `wide` groups of a sample: its threads take
// wide groups by kJoin/wide chunks at a time. In double, about the first
// chunk's mean, so one pass over the parts serves both moments.
constexpr int kJoin = 512;
__global__ void __launch_bounds__(kJoin)
    k_join(Batch B, const Moments* __restrict__ part, int wide, int blocks) {
    __shared__ double s1[kJoin], s2[kJoin];
    grid_wait();
    const int n = blockIdx.x / blocks, g = blockIdx.x % blocks * wide + threadIdx.x % wide;
    const int lane = threadIdx.x / wide, lanes = kJoin / wide;
    const int len = valid_rows(B, n);
    double a = 0.0, q = 0.0, ref = 0.0;
    if (g < B.g) {
        const Moments* p = part + (int64_t)n * B.chunks * B.g + g;
        ref = (double)p[0].k + p[0].off;
#pragma unroll 4
        for (int k = lane; k < B.chunks; k += lanes) {
            int r0, r1;
            chunk_rows(len, B.chunks, k, r0, r1);
            const Moments m = p[(int64_t)k * B.g];
            const double c = (double)(r1 - r0) * B.d, dv = ((double)m.k + m.off) - ref;
            if (r1 > r0) {
                a += c * dv;
                q += m.m2 + c * dv * dv;
            }
        }
    }
    s1[threadIdx.x] = a;
    s2[threadIdx.x] = q;
    __syncthreads();
    for (int h = lanes / 2; h; h /= 2) {
        if (lane < h) {
            s1[threadIdx.x] += s1[threadIdx.x + h * wide];
            s2[threadIdx.x] += s2[threadIdx.x + h * wide];
        }
        __syncthreads();
    }
    grid_release();
    if (lane == 0 && g < B.g) {
        const double count = (double)len * B.d;
        const double off = len ? s1[threadIdx.x] / count : 0.0;
        const double var = len ? s2[threadIdx.x] / count - off * off : 0.0;
        const int64_t at = (int64_t)n * B.g + g;
        B.mean_out[at] = len ? (float)(ref + off) : 0.0f;
        B.rstd_out[at] = (float)(1.0 / sqrt((var < 0.0 ? 0.0 : var) + (double)B.eps));
    }
}

template <class T, int AW, bool kSame, bool kKeep>
__global__ void __launch_bounds__(kThreads, 2) k_apply(Batch B) {
    grid_wait();
    const int id = gridDim.x - 1 - blockIdx.x, n = id / B.chunks;
    int r0, r1;
    chunk_rows(valid_rows(B, n), B.chunks, id % B.chunks, r0, r1);
    if (r0 >= r1) return;
    const int phase = threadIdx.x / B.tile, u = threadIdx.x % B.tile;
    const float *mu = B.mean_out + (int64_t)n * B.g, *rs = B.rstd_out + (int64_t)n * B.g;
    for (int t = 0; t < B.tiles; t++) {
        const int unit = t * B.tile + u, cnt = min(kUnit, B.c - unit * kUnit);
        const bool on = phase < B.phases && unit < B.units;
        const int first = min(unit * kUnit, B.c - 1);
        const auto mean = per_group<kSame>(first, B.c - 1, B.d, [&](int g) { return mu[g]; });
        const auto rstd = per_group<kSame>(first, B.c - 1, B.d, [&](int g) { return rs[g]; });
        V8 scale = ld_params(on ? B.w : nullptr, B.ptype, unit * kUnit, cnt, 1.0f);
        const V8 bias = ld_params(on ? B.b : nullptr, B.ptype, unit * kUnit, cnt, 0.0f);
#pragma unroll
        for (int i = 0; i < 4; i++) scale.p[i] = mul2(scale.p[i], rstd[i]);
        apply_rows<T, AW, kSame, kKeep>(B, n, r0, r1, phase, unit, cnt, on, mean, scale, bias,
                                        nullptr);
    }
}

// ---- backward ---------------------------------------------------------------------

// A unit of x and of dy, x from the tensor or from its checkpoint.
template <class T, int AW, bool kFrom>
struct Pair {
    Raw<T> dy, x;
    Codes codes;
    float scale;
    __device__ __forceinline__ V8 input() const { return kFrom ? decode(codes, scale) : unpack(x); }
};
// A thread's walk along its rows of both.
template <class T, int AW, bool kFrom>
struct PairWalk {
    const T *dy, *x;
    KeptAt kept;
    int64_t dy_step, x_step;
    __device__ __forceinline__ PairWalk(const Batch& B, int n, int64_t row, int unit) {
        dy = (const T*)B.dy + n * B.ys + row * B.yr + unit * kUnit;
        dy_step = B.phases * B.yr;
        if (kFrom) {
            kept = kept_at(B.kept, (int64_t)n * B.s + row, B.phases, unit);
        } else {
            x = (const T*)B.x + n * B.xs + row * B.xr + unit * kUnit;
            x_step = B.phases * B.xr;
        }
    }
    __device__ __forceinline__ void load(Pair<T, AW, kFrom>& v, int cnt) const {
        v.dy = ld_unit<T, AW>(dy, cnt);
        if (kFrom) {
            v.codes = ld_codes<AW == 16>(kept.codes, cnt);
            v.scale = __ldg(kept.scale);
        } else {
            v.x = ld_unit<T, AW>(x, cnt);
        }
    }
    __device__ __forceinline__ void move(int rows) {
        dy += rows * dy_step;
        if (kFrom) {
            kept.codes += rows * kept.codes_step;
            kept.scale += rows * kept.scale_step;
        } else {
            x += rows * x_step;
        }
    }
};
// The same in shared memory: arrays of iterations by threads.
template <class T, bool kFrom>
struct PairStore {
    Raw<T>* dy;
    Raw<T>* x;
    uint2* codes;
    float* scale;
    static constexpr int kBytes = (int)sizeof(Raw<T>) + (kFrom ? 12 : (int)sizeof(Raw<T>));
    __device__ __forceinline__ PairStore(void* base, int iters) {
        char* p = (char*)base;
        const int64_t cells = (int64_t)iters * kThreads;
        dy = (Raw<T>*)p;
        x = (Raw<T>*)(p + cells * sizeof(Raw<T>));
        codes = (uint2*)x;
        scale = (float*)(codes + cells);
    }
    template <int AW>
    __device__ __forceinline__ void put(int it, const Pair<T, AW, kFrom>& v) {
        const int at = it * kThreads + threadIdx.x;
        dy[at] = v.dy;
        if (kFrom) {
            codes[at] = v.codes.q;
            scale[at] = v.scale;
        } else {
            x[at] = v.x;
        }
    }
    template <int AW>
    __device__ __forceinline__ void get(int it, Pair<T, AW, kFrom>& v) const {
        const int at = it * kThreads + threadIdx.x;
        v.dy = dy[at];
        if (kFrom) {
            v.codes.q = codes[at];
            v.scale = scale[at];
        } else {
            v.x = x[at];
        }
    }
};

template <bool kSame>
struct BackParams {
    PerGroup<kSame> mean, rstd;
    V8 w, b;
};
template <bool kSame>
__device__ __forceinline__ BackParams<kSame> back_params(const Batch& B, int n, int unit, int cnt,
                                                         bool on) {
    BackParams<kSame> q;
    const int first = min(unit * kUnit, B.c - 1);
    const float *mu = B.mean + (int64_t)n * B.g, *rs = B.rstd + (int64_t)n * B.g;
    q.mean = per_group<kSame>(first, B.c - 1, B.d, [&](int g) { return __ldg(mu + g); });
    q.rstd = per_group<kSame>(first, B.c - 1, B.d, [&](int g) { return __ldg(rs + g); });
    q.w = ld_params(on ? B.w : nullptr, B.ptype, unit * kUnit, cnt, 1.0f);
    q.b = ld_params(on ? B.b : nullptr, B.ptype, unit * kUnit, cnt, 0.0f);
    return q;
}

// xh and dz = dy * act'(z) of one unit.
template <class T, int AW, bool kFrom, bool kSame>
__device__ __forceinline__ void slopes(const Batch& B, const BackParams<kSame>& q,
                                       const Pair<T, AW, kFrom>& in, V8& xh, V8& dz) {
    V8 z, f;
    xh = in.input();
#pragma unroll
    for (int i = 0; i < 4; i++) {
        xh.p[i] = mul2(sub2(xh.p[i], q.mean[i]), q.rstd[i]);
        z.p[i] = fma2(xh.p[i], q.w.p[i], q.b.p[i]);
    }
    const V8 g = unpack(in.dy);
    if (B.act == SIMTGO_ACT_NONE) {
        dz = g;
        return;
    }
    activate_slope<sizeof(T) == 2>(z, f, dz, B.act, B.param);
#pragma unroll
    for (int i = 0; i < 4; i++) dz.p[i] = mul2(dz.p[i], g.p[i]);
}

// Sums A = dz and C = dz*xh of the unit's channels over the thread's rows.
template <class T, int AW, bool kFrom, bool kSame, class F>
__device__ __forceinline__ void back_sums(const Batch& B, const BackParams<kSame>& q, int n, int r,
                                          int r1, int unit, int cnt, float2 (&a)[4], float2 (&c)[4],
                                          F&& keep) {
    constexpr int U = kOutRows<T>;
    const int rows = (r1 - r + B.phases - 1) / B.phases;
    PairWalk<T, AW, kFrom> walk(B, n, r, unit);
    for (int it = 0; it < rows; it += U) {
        Pair<T, AW, kFrom> in[U];
#pragma unroll
        for (int j = 0; j < U; j++) {
            if (it + j < rows) walk.load(in[j], cnt);
            walk.move(1);
        }
#pragma unroll
        for (int j = 0; j < U; j++)
            if (it + j < rows) {
                keep(it + j, in[j]);
                V8 xh, dz;
                slopes(B, q, in[j], xh, dz);
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    a[i] = add2(a[i], dz.p[i]);
                    c[i] = fma2(dz.p[i], xh.p[i], c[i]);
                }
            }
    }
}

// Adds the phases' (A, B) of every channel; phase 0 ends with the sums. Every
// thread calls it; it begins with a barrier.
__device__ __forceinline__ void add_phases(float2* red, int phases, int width, int phase, int u,
                                           const float2 (&a)[4], const float2 (&b)[4]) {
    // (A, A, B, B) of two channels at a time: 16 bytes a thread.
    float4* mine = reinterpret_cast<float4*>(red + phase * width) + u * 4;
    if (phase < phases) {
#pragma unroll
        for (int i = 0; i < 4; i++) mine[i] = make_float4(a[i].x, a[i].y, b[i].x, b[i].y);
    }
    __syncthreads();
    for (int m = phases; m > 1;) {
        const int h = (m + 1) / 2;
        if (phase + h < m) {
            const float4* o = reinterpret_cast<const float4*>(red + (phase + h) * width) + u * 4;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float4 v = o[i], w = mine[i];
                mine[i] = make_float4(w.x + v.x, w.y + v.y, w.z + v.z, w.w + v.w);
            }
        }
        m = h;
        __syncthreads();
    }
}
// Channel i's (A, B) after add_phases.
__device__ __forceinline__ float2 channel_sum(const float2* red, int i) {
    const float4 v = reinterpret_cast<const float4*>(red)[i / 2];
    return i & 1 ? make_float2(v.y, v.w) : make_float2(v.x, v.z);
}

// sum of w*A and w*B over each group's d channels, at(i) giving channel i's
// (A, B): f(group, sums) on the first lane of a sub-warp.
template <class At, class F>
__device__ __forceinline__ void group_sums(const Batch& B, int c0, int groups, At&& at, F&& f) {
    int lanes = 1;
    while (lanes < B.d && lanes < 32) lanes *= 2;
    const int per = kThreads / lanes, lane = threadIdx.x % lanes;
    for (int g0 = 0; g0 < groups; g0 += per) {
        const int g = g0 + threadIdx.x / lanes;
        float x = 0.0f, y = 0.0f;
        if (g < groups)
            for (int i = lane; i < B.d; i += lanes) {
                const float2 v = at(g * B.d + i);
                const float w = B.w ? ld_param(B.w, B.ptype, c0 + g * B.d + i) : 1.0f;
                x = __fmaf_rn(w, v.x, x);
                y = __fmaf_rn(w, v.y, y);
            }
        for (int o = lanes / 2; o; o /= 2) {
            x += __shfl_xor_sync(~0u, x, o);
            y += __shfl_xor_sync(~0u, y, o);
        }
        if (g < groups && lane == 0) f(g, make_float2(x, y));
    }
}

// dx of rows [r0, r1) of this thread's unit, last rows first. s1 and s2 are the
// negated means, added.
template <class T, int AW, bool kFrom, bool kSame>
__device__ __forceinline__ void back_rows(const Batch& B, const BackParams<kSame>& q,
                                          const PerGroup<kSame>& s1, const PerGroup<kSame>& s2,
                                          int n, int r0, int r1, int phase, int unit, int cnt,
                                          const PairStore<T, kFrom>& store) {
    constexpr int U = kOutRows<T>;
    const int rows = (r1 - r0 - phase + B.phases - 1) / B.phases;
    if (rows <= 0) return;
    int it = (rows - 1) / U * U;
    const int64_t row = r0 + phase + (int64_t)it * B.phases;
    PairWalk<T, AW, kFrom> walk(B, n, row, unit);
    T* dx = (T*)B.out + n * B.os + row * B.orow + unit * kUnit;
    const int64_t step = B.phases * B.orow;
    for (; it >= 0; it -= U) {
        Pair<T, AW, kFrom> in[U];
        if (it + U <= B.keep) {
#pragma unroll
            for (int j = 0; j < U; j++)
                if (it + j < rows) store.get(it + j, in[j]);
            walk.move(-U);
        } else {
#pragma unroll
            for (int j = 0; j < U; j++) {
                if (it + j < rows) walk.load(in[j], cnt);
                walk.move(1);
            }
            walk.move(-2 * U);
        }
        T* to = dx;
#pragma unroll
        for (int j = 0; j < U; j++) {
            if (it + j < rows) {
                V8 xh, dz;
                slopes(B, q, in[j], xh, dz);
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float2 v = fma2(dz.p[i], q.w.p[i], s1[i]);
                    dz.p[i] = mul2(q.rstd[i], fma2(xh.p[i], s2[i], v));
                }
                Raw<T> o;
                pack(dz, o);
                st_unit<T, AW>(to, o, cnt);
            }
            to += step;
        }
        dx -= U * step;
    }
}

// One launch for dx: a cluster per slab of a sample. part, where wanted,
// receives every block's (A, B) of its channels, for k_back_join.
template <class T, int AW, bool kFrom, bool kSame>
__global__ void __launch_bounds__(kThreads, 2) k_norm_back(Batch B, float2* __restrict__ part) {
    extern __shared__ uint4 dyn[];
    const int phase = threadIdx.x / B.tile, u = threadIdx.x % B.tile, width = B.tile * kUnit;
    PairStore<T, kFrom> store(dyn, B.keep);
    float2* red = reinterpret_cast<float2*>(
        (char*)dyn + (int64_t)B.keep * kThreads * PairStore<T, kFrom>::kBytes);
    float2* own = red + B.phases * width;     // this block's group sums
    float2* means = own + B.slab / B.d;       // the cluster's, over the count

    const int rank = (int)cluster_rank();
    const int id = blockIdx.x / B.chunks, n = id / B.slabs, c0 = id % B.slabs * B.slab;
    const int cw = min(B.slab, B.c - c0), groups = cw / B.d, g0 = c0 / B.d;
    const int len = valid_rows(B, n);
    int r0, r1;
    chunk_rows(len, B.chunks, rank, r0, r1);
    const int unit = c0 / kUnit + u, cnt = min(kUnit, c0 + cw - unit * kUnit);
    const bool on = phase < B.phases && u * kUnit < cw;

    const BackParams<kSame> q = back_params<kSame>(B, n, unit, cnt, on);
    float2 a[4] = {}, b[4] = {};
    if (on)
        back_sums<T, AW, kFrom>(B, q, n, r0 + phase, r1, unit, cnt, a, b,
                                [&](int it, const Pair<T, AW, kFrom>& v) {
                                    if (it < B.keep) store.put(it, v);
                                });
    add_phases(red, B.phases, width, phase, u, a, b);
    if (part)
        for (int i = threadIdx.x; i < cw; i += kThreads)
            part[((int64_t)n * B.chunks + rank) * B.c + c0 + i] = channel_sum(red, i);
    grid_release();
    if (!B.out) return;  // the same for every block of the grid
    group_sums(B, c0, groups, [&](int i) { return channel_sum(red, i); },
               [&](int g, float2 v) { own[g] = v; });
    cluster_arrive();
    cluster_wait();
    for (int g = threadIdx.x; g < groups; g += kThreads) {
        float x = 0.0f, y = 0.0f;
        for (int k = 0; k < B.chunks; k++) {
            x += ld_cluster(&own[g].x, k);
            y += ld_cluster(&own[g].y, k);
        }
        const float inv = len ? -1.0f / ((float)len * (float)B.d) : 0.0f;
        means[g] = make_float2(x * inv, y * inv);
    }
    cluster_arrive();
    __syncthreads();
    if (on) {
        const int last = c0 + cw - 1, first = min(unit * kUnit, last);
        const auto s1 = per_group<kSame>(first, last, B.d, [&](int g) { return means[g - g0].x; });
        const auto s2 = per_group<kSame>(first, last, B.d, [&](int g) { return means[g - g0].y; });
        back_rows<T, AW, kFrom, kSame>(B, q, s1, s2, n, r0, r1, phase, unit, cnt, store);
    }
    cluster_wait();
}

// Over chunks: (A, B) of every channel of a chunk.
template <class T, int AW, bool kFrom, bool kSame>
__global__ void __launch_bounds__(kThreads, 2) k_back_stats(Batch B, float2* __restrict__ part) {
    extern __shared__ float4 red4[];
    float2* red = reinterpret_cast<float2*>(red4);
    const int n = blockIdx.x / B.chunks, k = blockIdx.x % B.chunks;
    int r0, r1;
    chunk_rows(valid_rows(B, n), B.chunks, k, r0, r1);
    float2* o = part + ((int64_t)n * B.chunks + k) * B.c;
    const int phase = threadIdx.x / B.tile, u = threadIdx.x % B.tile, width = B.tile * kUnit;
    for (int t = 0; t < B.tiles; t++) {
        const int unit = t * B.tile + u, cnt = min(kUnit, B.c - unit * kUnit);
        const bool on = phase < B.phases && unit < B.units;
        float2 a[4] = {}, b[4] = {};
        if (on && r0 < r1) {
            const BackParams<kSame> q = back_params<kSame>(B, n, unit, cnt, on);
            back_sums<T, AW, kFrom>(B, q, n, r0 + phase, r1, unit, cnt, a, b,
                                    [](int, const Pair<T, AW, kFrom>&) {});
        }
        add_phases(red, B.phases, width, phase, u, a, b);
        const int c0 = t * width;
        for (int i = threadIdx.x; i < min(width, B.c - c0); i += kThreads)
            o[c0 + i] = channel_sum(red, i);
        __syncthreads();
    }
    grid_release();
}

// Adds `rows` rows of part for each of a number of spans, in double: to
// tot[span][c], and to dbias and dweight where there is one span. A block takes
// 32 channels of a span, its warps the rows in turn.
constexpr int kAdd = 1024;
__global__ void __launch_bounds__(kAdd)
    k_back_join(const float2* __restrict__ part, int64_t rows, int c, int blocks,
                float2* __restrict__ tot, float* __restrict__ dw, float* __restrict__ db) {
    __shared__ double2 sm[kAdd / 32][33];
    grid_wait();
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    const int64_t span = blockIdx.x / blocks;
    const int ch = blockIdx.x % blocks * 32 + lane;
    const float2* p = part + span * rows * c + ch;
    double2 s = make_double2(0.0, 0.0);
    if (ch < c) {
#pragma unroll 4
        for (int64_t r = warp; r < rows; r += kAdd / 32) {
            const float2 v = p[r * c];
            s.x += v.x;
            s.y += v.y;
        }
    }
    sm[warp][lane] = s;
    __syncthreads();
    for (int h = kAdd / 64; h; h /= 2) {
        if (warp < h) {
            sm[warp][lane].x += sm[warp + h][lane].x;
            sm[warp][lane].y += sm[warp + h][lane].y;
        }
        __syncthreads();
    }
    grid_release();
    if (warp == 0 && ch < c) {
        s = sm[0][lane];
        if (tot) tot[span * c + ch] = make_float2((float)s.x, (float)s.y);
        if (db) db[ch] = (float)s.x;
        if (dw) dw[ch] = (float)s.y;
    }
}

template <class T, int AW, bool kFrom, bool kSame>
__global__ void __launch_bounds__(kThreads, 2)
    k_back_apply(Batch B, const float2* __restrict__ tot) {
    extern __shared__ float2 means[];  // of every group
    grid_wait();
    const int id = gridDim.x - 1 - blockIdx.x, n = id / B.chunks;
    const int len = valid_rows(B, n);
    int r0, r1;
    chunk_rows(len, B.chunks, id % B.chunks, r0, r1);
    if (r0 >= r1) return;
    const float inv = -1.0f / ((float)len * (float)B.d);
    group_sums(B, 0, B.g, [&](int i) { return __ldg(tot + (int64_t)n * B.c + i); },
               [&](int g, float2 v) { means[g] = make_float2(v.x * inv, v.y * inv); });
    __syncthreads();
    const int phase = threadIdx.x / B.tile, u = threadIdx.x % B.tile;
    if (phase >= B.phases) return;
    const PairStore<T, kFrom> none(nullptr, 0);
    for (int t = 0; t < B.tiles; t++) {
        const int unit = t * B.tile + u, cnt = min(kUnit, B.c - unit * kUnit);
        if (unit >= B.units) break;
        const BackParams<kSame> q = back_params<kSame>(B, n, unit, cnt, true);
        const int first = unit * kUnit;
        const auto s1 = per_group<kSame>(first, B.c - 1, B.d, [&](int g) { return means[g].x; });
        const auto s2 = per_group<kSame>(first, B.c - 1, B.d, [&](int g) { return means[g].y; });
        back_rows<T, AW, kFrom, kSame>(B, q, s1, s2, n, r0, r1, phase, unit, cnt, none);
    }
}

// ---- host -------------------------------------------------------------------

struct Scratch {
    void* p = nullptr;
    cudaStream_t s = 0;
    ~Scratch() {
        if (p) cudaFreeAsync(p, s);
    }
    int alloc(size_t bytes, cudaStream_t st) {
        s = st;
        return sg::scratch_alloc(&p, bytes, st);
    }
};

// Shape and option checks the two directions share.
int check_cfg(const char* K, const simtgo_group_norm& c, bool kept) {
    int rc;
    if (c.samples < 0 || c.positions < 0 || c.channels < 0)
        return sg::fail(SIMTGO_EARG, "channels: %s: a negative extent", K);
    if ((rc = check_type(K, "type", c.type)) || (rc = check_type(K, "param_type", c.param_type)) ||
        (rc = check_act(K, c.act, c.act_param)))
        return rc;
    if (c.groups <= 0 || c.channels % c.groups)
        return sg::fail(SIMTGO_EARG, "channels: %s: %d channels are not a whole number of %d "
                        "groups", K, c.channels, c.groups);
    if (!(c.eps > 0.0f) || !std::isfinite(c.eps))
        return sg::fail(SIMTGO_EARG, "channels: %s: eps must be positive, got %g", K, c.eps);
    if (c.channels > SIMTGO_GROUP_NORM_MAX_CHANNELS)
        return sg::fail(SIMTGO_ESIZE, "channels: %s: %d channels, at most %d", K, c.channels,
                        SIMTGO_GROUP_NORM_MAX_CHANNELS);
    if (c.positions > SIMTGO_GROUP_NORM_MAX_POSITIONS)
        return sg::fail(SIMTGO_ESIZE, "channels: %s: %d positions, at most %d", K, c.positions,
                        SIMTGO_GROUP_NORM_MAX_POSITIONS);
    if ((__int128)c.samples * c.positions * c.channels > kMaxElems)
        return sg::fail(SIMTGO_ESIZE, "channels: %s: more than 2^46 elements", K);
    return kept ? check_block(K, c.block) : 0;
}

// One batch-shaped buffer of the call, as a region; rc is set where it cannot
// be used.
Region batch(const char* K, const char* name, const void* p, const simtgo_group_norm& c,
             int64_t sample, int64_t row, bool written, int* rc) {
    const int64_t e = elem_size(c.type);
    const int64_t ns = c.samples > 1 ? sample : 0, nr = c.positions > 1 ? row : 0;
    Region r = {name, p, c.channels * e, nr * e, ns * e, 0, written};
    if (*rc || !p) return r;
    if (ns < 0 || nr < 0 || ns > kMaxElems || nr > kMaxElems ||
        (__int128)(c.samples - 1) * ns + (__int128)(c.positions - 1) * nr > kMaxElems) {
        *rc = sg::fail(SIMTGO_EARG, "channels: %s: %s has pitches of %lld and %lld elements", K,
                       name, (long long)sample, (long long)row);
        return r;
    }
    const int64_t span_s = (c.samples - 1) * ns, span_r = (c.positions - 1) * nr;
    r.bytes = (span_s + span_r + c.channels) * e;
    // Rows of their own: samples of rows, or rows of samples.
    const bool rows_in = (c.positions < 2 || nr >= c.channels) &&
                         (c.samples < 2 || ns >= span_r + c.channels);
    const bool samples_in = (c.samples < 2 || ns >= c.channels) &&
                            (c.positions < 2 || nr >= span_s + c.channels);
    if (written && !rows_in && !samples_in)
        *rc = sg::fail(SIMTGO_EALIAS, "channels: %s: the rows of %s overlap (pitches %lld and %lld, "
                       "%d channels) and the kernel writes through it", K, name, (long long)sample,
                       (long long)row, c.channels);
    else
        *rc = check_aligned(K, name, p, (int)e);
    return r;
}

// Lets a kernel have as much shared memory as a block may, once per device.
template <auto Kernel>
int allow_smem(const sg::DevInfo& d, size_t bytes) {
    static std::atomic<bool> done[64];
    if (bytes <= 48 * 1024 || done[d.device & 63].load(std::memory_order_relaxed)) return 0;
    cudaFuncAttributes at;
    int rc = sg::cuda_status(cudaFuncGetAttributes(&at, Kernel), "cudaFuncGetAttributes(GroupNorm)");
    if (!rc)
        rc = sg::cuda_status(cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                  d.max_smem_optin - (int)at.sharedSizeBytes),
                             "cudaFuncSetAttribute(GroupNorm)");
    if (!rc) done[d.device & 63].store(true, std::memory_order_relaxed);
    return rc;
}

// Launches Kernel, as clusters of `cluster` blocks, and with `after` as soon as
// the kernel before it releases it (it then waits for that one's end itself).
template <auto Kernel, class... A>
int launch(const sg::DevInfo& d, unsigned grid, int threads, size_t smem, cudaStream_t s,
           int cluster, bool after, A... args) {
    if (int rc = allow_smem<Kernel>(d, smem)) return rc;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute at[2];
    cfg.attrs = at;
    if (cluster > 1) {
        at[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
        at[cfg.numAttrs].val.clusterDim.x = cluster;
        at[cfg.numAttrs].val.clusterDim.y = 1;
        at[cfg.numAttrs].val.clusterDim.z = 1;
        cfg.numAttrs++;
    }
    if (after) {
        at[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        at[cfg.numAttrs].val.programmaticStreamSerializationAllowed = 1;
        cfg.numAttrs++;
    }
    sg::before_launch();
    return sg::cuda_status(cudaLaunchKernelEx(&cfg, Kernel, args...), "GroupNorm");
}

// Tiles of at most 256 units for rows of `units`, whole blocks of `lanes`.
void tile_units(Batch& B, int units, int lanes) {
    const int upad = (units + lanes - 1) / lanes * lanes;
    B.units = units;
    B.tiles = (upad + kThreads - 1) / kThreads;
    B.tile = ((upad + B.tiles - 1) / B.tiles + lanes - 1) / lanes * lanes;
    B.tiles = (upad + B.tile - 1) / B.tile;
    B.phases = kThreads / B.tile;
}

// How a call goes through its data. `elem` is the bytes of all inputs per
// element; `sum_rows`, the rows a thread takes at a time; `iter_bytes`, what an
// iteration of a block's threads keeps; `cell_bytes`, a thread's sums.
struct Plan {
    bool cluster;
    unsigned grid;
    size_t smem;
};
Plan make_plan(Batch& B, const simtgo_group_norm& c, const sg::DevInfo& d, bool keep_codes,
               double elem, int sum_rows, int iter_bytes, int cell_bytes, int group_bytes) {
    B.n = c.samples;
    B.s = c.positions;
    B.c = c.channels;
    B.g = c.groups;
    B.d = c.channels / c.groups;
    B.ptype = c.param_type;
    B.act = c.act;
    B.param = c.act_param;
    B.eps = c.eps;
    const int units = (c.channels + kUnit - 1) / kUnit;

    // A slab: whole groups, units and checkpoint blocks; 128 bytes of every row
    // where the channels allow it, more while a slab would be a small load.
    int64_t q = std::lcm((int64_t)B.d, (int64_t)kUnit);
    if (keep_codes) q = std::lcm(q, (int64_t)c.block);
    const int64_t most = kThreads * kUnit;
    int64_t slab = c.channels;
    if (q < c.channels) {
        const int64_t least = 128 / elem_size(c.type);
        slab = (least + q - 1) / q * q;
        while (2 * slab <= std::min<int64_t>(c.channels, most) && slab * c.positions * elem < 65536)
            slab *= 2;
        slab = std::min<int64_t>(slab, c.channels);
        const int64_t parts = (c.channels + slab - 1) / slab;
        slab = std::min<int64_t>(((c.channels + parts - 1) / parts + q - 1) / q * q, c.channels);
    }
    Plan p = {};
    if (slab <= most) {
        const int slabs = (int)((c.channels + slab - 1) / slab);
        const int su = (int)((slab + kUnit - 1) / kUnit);
        const int lanes =
            keep_codes ? std::min(c.block / kUnit, ceil_pow2(std::min(su, 32))) : 1;
        Batch t = B;
        tile_units(t, su, lanes);
        t.slab = (int)slab;
        t.slabs = slabs;
        const int64_t clusters = (int64_t)c.samples * slabs;
        const double bytes = (double)slab * c.positions * elem;
        int k = 1;
        while (k < 8 && c.positions / (2 * k) >= t.phases &&
               (clusters * k < 2 * d.sms || bytes / k > 96 * 1024))
            k *= 2;
        t.chunks = k;
        // A block moves about 36 GB/s; a chunked pass fills the GPU but costs
        // two more launches, about 6 us.
        const double us = bytes * clusters / (std::min<double>(clusters * k, 2 * d.sms) * 36e3);
        const double chunked = bytes * clusters / 6.4e6 + 6.0;
        if (us <= chunked && clusters * k <= 0x7fffffff) {
            const size_t fixed = (size_t)t.phases * t.tile * cell_bytes +
                                 (size_t)(slab / B.d + 1) * group_bytes + 32;
            const size_t room = (clusters * k > d.sms ? (size_t)d.smem_per_sm / 2 : (size_t)d.max_smem_optin) - 4096;
            const int64_t need = (c.positions / k + t.phases) / t.phases + 1;
            int64_t keep = fixed < room ? (int64_t)(room - fixed) / iter_bytes : 0;
            keep = std::min(keep, (need + sum_rows - 1) / sum_rows * sum_rows);
            t.keep = (int)(keep / sum_rows * sum_rows);
            p.smem = fixed + (size_t)t.keep * iter_bytes;
            p.cluster = p.smem + 4096 <= (size_t)d.max_smem_optin;
            p.grid = (unsigned)(clusters * k);
            if (p.cluster) {
                t.kept.lanes = lanes;
                B = t;
                return p;
            }
        }
    }
    const int lanes = keep_codes ? std::min(c.block / kUnit, ceil_pow2(std::min(units, 32))) : 1;
    tile_units(B, units, lanes);
    B.kept.lanes = lanes;
    B.slab = c.channels;
    B.slabs = 1;
    B.keep = 0;
    // One wave of blocks, eight rows a thread at least.
    const int64_t rows = std::max<int64_t>(1, sg::ceil_div(B.s, 8 * B.phases));
    B.chunks = (int)std::max<int64_t>(1, std::min(rows, (int64_t)3 * d.sms / std::max(1, B.n)));
    p.grid = (unsigned)B.n * (unsigned)B.chunks;
    return p;
}

// The checkpoint that is written, or -- backward -- read.
void set_kept(Batch& B, const simtgo_group_norm& c, bool kept, const int8_t* codes,
              const float* scales) {
    B.kept = {const_cast<int8_t*>(codes), const_cast<float*>(scales), c.channels, 0, 0, 1};
    if (!kept) return;
    while ((kUnit << B.kept.shift) < c.block) B.kept.shift++;
    B.kept.nblk = (c.channels + c.block - 1) / c.block;
}

}  // namespace

extern "C" {

int simtgo_GroupNorm(void* y, float* mean, float* rstd, const void* x, const void* weight,
                     const void* bias, const int32_t* lengths, int8_t* codes, float* scales,
                     const simtgo_group_norm* cfg, void* stream) {
    const char* K = "GroupNorm";
    sg::clear_error();
    int rc;
    if (!cfg) return sg::fail(SIMTGO_ENULL, "channels: %s: no configuration", K);
    const simtgo_group_norm c = *cfg;
    const bool kept = codes || scales;
    if ((rc = check_cfg(K, c, kept))) return rc;
    if (c.samples == 0 || c.channels == 0) return 0;
    const int64_t rows = (int64_t)c.samples * c.positions, stats = (int64_t)c.samples * c.groups;
    const int64_t elems = rows * c.channels;
    if ((rc = sg::check_ptr(K, "y", y, elems)) || (rc = sg::check_ptr(K, "x", x, elems))) return rc;
    if (kept && elems && (!codes || !scales))
        return sg::fail(SIMTGO_ENULL, "channels: %s: the checkpoint needs both codes and scales", K);
    const Region ry = batch(K, "y", y, c, c.y_sample, c.y_row, true, &rc);
    const Region rx = batch(K, "x", x, c, c.x_sample, c.x_row, false, &rc);
    if (rc || (rc = check_aligned(K, "mean", mean, 4)) || (rc = check_aligned(K, "rstd", rstd, 4)) ||
        (rc = check_aligned(K, "weight", weight, elem_size(c.param_type))) ||
        (rc = check_aligned(K, "bias", bias, elem_size(c.param_type))) ||
        (rc = check_aligned(K, "lengths", lengths, 4)) ||
        (rc = check_aligned(K, "scales", scales, 4)))
        return rc;
    const int64_t pbytes = (int64_t)c.channels * elem_size(c.param_type);
    const int nblk = kept ? (c.channels + c.block - 1) / c.block : 0;
    if ((rc = check_regions(K, {ry, rx, solid("mean", mean, 4 * stats, true),
                                solid("rstd", rstd, 4 * stats, true),
                                solid("weight", weight, pbytes, false),
                                solid("bias", bias, pbytes, false),
                                solid("lengths", lengths, 4LL * c.samples, false),
                                solid("codes", codes, elems, true),
                                solid("scales", scales, 4 * rows * nblk, true)})))
        return rc;
    const sg::DevInfo* d;
    if ((rc = sg::current_device(&d))) return rc;

    Batch B = {};
    B.x = x;
    B.out = y;
    B.w = weight;
    B.b = bias;
    B.lengths = lengths;
    B.mean_out = mean;
    B.rstd_out = rstd;
    B.xs = c.x_sample;
    B.xr = c.x_row;
    B.os = c.y_sample;
    B.orow = c.y_row;
    set_kept(B, c, kept, codes, scales);
    const int e = elem_size(c.type);
    int width = access_width(
        c.type, {{x, rx.pitch0 / e, rx.pitch1 / e}, {y, ry.pitch0 / e, ry.pitch1 / e}});
    if (kept && width == 16 && (c.channels % kUnit || ((uintptr_t)codes & 7))) width = 4;
    const bool same = (c.channels / c.groups) % kUnit == 0;
    const Plan p = make_plan(B, c, *d, kept, e, e == 2 ? 8 : 4, kThreads * kUnit * e,
                             (int)sizeof(Moments) * (same ? 1 : kUnit),
                             (int)(sizeof(Moments) + sizeof(float2)));
    cudaStream_t s = (cudaStream_t)stream;
    return by_type(c.type, width, [&](auto* t, auto w) {
        using T = std::remove_pointer_t<decltype(t)>;
        constexpr int AW = decltype(w)::value;
        const auto run = [&](auto same_, auto kept_) -> int {
            constexpr bool S = decltype(same_)::value, Q = decltype(kept_)::value;
            if (p.cluster)
                return launch<k_norm<T, AW, S, Q>>(*d, p.grid, kThreads, p.smem, s, B.chunks, false,
                                                   B);
            const int64_t parts = stats * B.chunks;
            Scratch scratch;
            if (int rc2 = scratch.alloc(sizeof(Moments) * parts + 8 * stats, s)) return rc2;
            Moments* part = (Moments*)scratch.p;
            float* own = (float*)(part + parts);
            if (!mean) B.mean_out = own;
            if (!rstd) B.rstd_out = own + stats;
            const size_t smem =
                sizeof(Moments) * (S ? 1 : kUnit) * ((size_t)B.units + (size_t)B.phases * B.tile);
            if (int rc2 = launch<k_stats<T, AW, S>>(*d, p.grid, kThreads, smem, s, 1, false, B,
                                                    part))
                return rc2;
            const int wide = std::min(32, ceil_pow2(c.groups));
            const int blocks = (c.groups + wide - 1) / wide;
            if (int rc2 = launch<k_join>(*d, (unsigned)c.samples * blocks, kJoin, 0, s, 1, true, B,
                                         (const Moments*)part, wide, blocks))
                return rc2;
            if (!elems) return 0;
            return launch<k_apply<T, AW, S, Q>>(*d, p.grid, kThreads, 0, s, 1, true, B);
        };
        if (same) return kept ? run(std::true_type(), std::true_type())
                              : run(std::true_type(), std::false_type());
        return kept ? run(std::false_type(), std::true_type())
                    : run(std::false_type(), std::false_type());
    });
}

int simtgo_GroupNorm_backward(void* dx, float* dweight, float* dbias, const void* dy,
                              const void* x, const int8_t* codes, const float* scales,
                              const float* mean, const float* rstd, const void* weight,
                              const void* bias, const int32_t* lengths,
                              const simtgo_group_norm* cfg, void* stream) {
    const char* K = "GroupNorm_backward";
    sg::clear_error();
    int rc;
    if (!cfg) return sg::fail(SIMTGO_ENULL, "channels: %s: no configuration", K);
    const simtgo_group_norm c = *cfg;
    const bool from = codes || scales;
    if ((rc = check_cfg(K, c, from))) return rc;
    if (c.channels == 0 || (!dx && !dweight && !dbias)) return 0;
    const int64_t rows = (int64_t)c.samples * c.positions, stats = (int64_t)c.samples * c.groups;
    const int64_t elems = rows * c.channels;
    if (elems) {
        if (from == (x != nullptr))
            return sg::fail(SIMTGO_EARG, "channels: %s: exactly one of x and its checkpoint is "
                            "given", K);
        if (from && (!codes || !scales))
            return sg::fail(SIMTGO_ENULL, "channels: %s: the checkpoint needs both codes and "
                            "scales", K);
        if ((rc = sg::check_ptr(K, "dy", dy, elems)) || (rc = sg::check_ptr(K, "mean", mean, stats)) ||
            (rc = sg::check_ptr(K, "rstd", rstd, stats)))
            return rc;
    }
    const Region rd = batch(K, "dx", dx, c, c.d_sample, c.d_row, true, &rc);
    const Region ry = batch(K, "dy", dy, c, c.y_sample, c.y_row, false, &rc);
    const Region rx = batch(K, "x", x, c, c.x_sample, c.x_row, false, &rc);
    if (rc || (rc = check_aligned(K, "dweight", dweight, 4)) ||
        (rc = check_aligned(K, "dbias", dbias, 4)) || (rc = check_aligned(K, "mean", mean, 4)) ||
        (rc = check_aligned(K, "rstd", rstd, 4)) ||
        (rc = check_aligned(K, "weight", weight, elem_size(c.param_type))) ||
        (rc = check_aligned(K, "bias", bias, elem_size(c.param_type))) ||
        (rc = check_aligned(K, "lengths", lengths, 4)) ||
        (rc = check_aligned(K, "scales", scales, 4)))
        return rc;
    const int64_t pbytes = (int64_t)c.channels * elem_size(c.param_type);
    const int nblk = from ? (c.channels + c.block - 1) / c.block : 0;
    if ((rc = check_regions(K, {rd, ry, rx, solid("dweight", dweight, 4LL * c.channels, true),
                                solid("dbias", dbias, 4LL * c.channels, true),
                                solid("mean", mean, 4 * stats, false),
                                solid("rstd", rstd, 4 * stats, false),
                                solid("weight", weight, pbytes, false),
                                solid("bias", bias, pbytes, false),
                                solid("lengths", lengths, 4LL * c.samples, false),
                                solid("codes", codes, elems, false),
                                solid("scales", scales, 4 * rows * nblk, false)})))
        return rc;
    const sg::DevInfo* d;
    if ((rc = sg::current_device(&d))) return rc;
    cudaStream_t s = (cudaStream_t)stream;
    if (!elems) {  // sums over nothing
        if (dweight && (rc = sg::cuda_status(cudaMemsetAsync(dweight, 0, 4LL * c.channels, s), K)))
            return rc;
        return dbias ? sg::cuda_status(cudaMemsetAsync(dbias, 0, 4LL * c.channels, s), K) : 0;
    }

    Batch B = {};
    B.x = x;
    B.dy = dy;
    B.out = dx;
    B.mean = mean;
    B.rstd = rstd;
    B.w = weight;
    B.b = bias;
    B.lengths = lengths;
    B.xs = c.x_sample;
    B.xr = c.x_row;
    B.ys = c.y_sample;
    B.yr = c.y_row;
    B.os = c.d_sample;
    B.orow = c.d_row;
    set_kept(B, c, from, codes, scales);
    const int e = elem_size(c.type);
    int width = access_width(c.type, {{x, rx.pitch0 / e, rx.pitch1 / e},
                                      {dy, ry.pitch0 / e, ry.pitch1 / e},
                                      {dx, rd.pitch0 / e, rd.pitch1 / e}});
    if (from && width == 16 && (c.channels % kUnit || ((uintptr_t)codes & 7))) width = 4;
    const bool same = (c.channels / c.groups) % kUnit == 0;
    const int unit_bytes = kUnit * e + (from ? 12 : kUnit * e);
    const Plan p = make_plan(B, c, *d, false, from ? e + 1.1 : 2.0 * e, e == 2 ? 4 : 2,
                             kThreads * unit_bytes, (int)sizeof(float2) * kUnit,
                             2 * (int)sizeof(float2));
    const bool params = dweight || dbias;
    const int64_t parts = params || !p.cluster ? (int64_t)c.samples * B.chunks * c.channels : 0;
    // A sample's own sums: the parts themselves where it is one chunk.
    const bool spans = !p.cluster && dx && B.chunks > 1;
    const int64_t tots = spans ? (int64_t)c.samples * c.channels : 0;
    Scratch scratch;
    if (parts && (rc = scratch.alloc(sizeof(float2) * (parts + tots), s))) return rc;
    float2* part = (float2*)scratch.p;
    float2* tot = spans ? part + parts : part;
    const unsigned add = (unsigned)sg::ceil_div(c.channels, 32);
    if (spans && (int64_t)add * c.samples > 0x7fffffff)
        return sg::fail(SIMTGO_ESIZE, "channels: %s: too many samples of so many channels", K);
    return by_type(c.type, width, [&](auto* t, auto w) {
        using T = std::remove_pointer_t<decltype(t)>;
        constexpr int AW = decltype(w)::value;
        const auto run = [&](auto from_, auto same_) -> int {
            constexpr bool F = decltype(from_)::value, S = decltype(same_)::value;
            if (p.cluster) {
                if (int r = launch<k_norm_back<T, AW, F, S>>(*d, p.grid, kThreads, p.smem, s,
                                                             B.chunks, false, B, part))
                    return r;
            } else {
                const size_t smem = sizeof(float2) * kUnit * (size_t)B.phases * B.tile;
                if (int r = launch<k_back_stats<T, AW, F, S>>(*d, p.grid, kThreads, smem, s, 1,
                                                              false, B, part))
                    return r;
            }
            const int64_t all = (int64_t)c.samples * B.chunks;
            if (spans) {
                const bool one = c.samples == 1;
                if (int r = launch<k_back_join>(*d, add * c.samples, kAdd, 0, s, 1, true,
                                                (const float2*)part, (int64_t)B.chunks, c.channels,
                                                (int)add, tot, one ? dweight : nullptr,
                                                one ? dbias : nullptr))
                    return r;
            }
            if (params && !(spans && c.samples == 1))
                if (int r = launch<k_back_join>(*d, add, kAdd, 0, s, 1, true,
                                                (const float2*)(spans ? tot : part),
                                                spans ? (int64_t)c.samples : all, c.channels,
                                                (int)add, (float2*)nullptr, dweight, dbias))
                    return r;
            if (p.cluster || !dx) return 0;
            return launch<k_back_apply<T, AW, F, S>>(*d, p.grid, kThreads,
                                                     sizeof(float2) * (size_t)c.groups, s, 1, true,
                                                     B, (const float2*)tot);
        };
        if (from) return same ? run(std::true_type(), std::true_type())
                              : run(std::true_type(), std::false_type());
        return same ? run(std::false_type(), std::true_type())
                    : run(std::false_type(), std::false_type());
    });
}

}  // extern "C"
