// groupnorm.cu -- group norm with an activation over channels-last batches,
// forward and backward, with the input kept as an 8-bit checkpoint on request.
//
// Mathematics. A thread sums x - K and (x - K)^2 for the eight channels of its
// unit, K being the first value it meets: the shift keeps the variance exact
// to a few ulps however far the mean is from zero, since K is one of the
// values that are summed. Threads, blocks and chunks of a sample are then
// joined by counts, means and sums of squared deviations (Chan, Golub and
// LeVeque's pairwise formula), never by raw squares; a mean stays K plus a
// small offset until the last join, so differences of means do not cancel. The backward pass needs,
// for each channel of a sample, A = sum dz and B = sum dz*xh: weighted and summed
// over a group's channels they give the group's two means in dx, and summed
// over the samples they are dbias and dweight, so one pass over x and dy serves
// both. All joins run in a fixed order.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "channels.cuh"

using namespace chan;

namespace {

constexpr int kThreads = 256;
constexpr int64_t kMaxElems = int64_t(1) << 46;

struct Batch {
    const void *x, *dy, *w, *b;
    void* out;  // y, or dx
    const int8_t* codes_in;
    const float* scales_in;
    int8_t* codes;
    float* scales;
    const float *mean, *rstd;
    const int32_t* lengths;
    int64_t xs, xr, ys, yr, os, orow;
    int n, s, c, g, d;
    int units, lanes, tile, tiles, phases;  // lanes: that share a checkpoint block
    int shift, nblk;
    int chunks;  // parts a sample's rows are cut into
    int ptype, act;
    float param, eps;
};

__device__ __forceinline__ int valid_rows(const Batch& B, int n) {
    return B.lengths ? min(max(__ldg(B.lengths + n), 0), B.s) : B.s;
}
// Rows [r0, r1) of chunk k of a sample of len rows.
__device__ __forceinline__ void chunk_rows(int len, int chunks, int k, int& r0, int& r1) {
    const int per = (len + chunks - 1) / chunks;
    r0 = (int)min((int64_t)k * per, (int64_t)len);
    r1 = min(r0 + per, len);
}

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
// channel i at [p*width + i], cnt[p] its rows. Phase 0 ends with them all.
__device__ void join_phases(Moments* red, float* cnt, int phases, int width, int phase, int unit8,
                            int lead) {
    float* in = cnt;
    float* out = cnt + kThreads;
    for (int m = phases; m > 1;) {
        const int h = (m + 1) / 2;
        if (phase < h && unit8 < width) {
            const bool two = phase + h < m;
            const float na = in[phase], nb = two ? in[phase + h] : 0.0f;
            if (two) {
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    Moments* a = red + phase * width + unit8 + i;
                    *a = join(na, *a, nb, a[h * width]);
                }
            }
            if (lead) out[phase] = na + nb;
        }
        float* t = in;
        in = out;
        out = t;
        m = h;
        __syncthreads();
    }
}

// Sums of x - K and (x - K)^2 down rows r, r + step, ... < r1 of one unit.
template <class T, int AW>
__device__ __forceinline__ int unit_moments(const T* x, int64_t pitch, int r, int r1, int step,
                                            int cnt, Moments (&out)[8]) {
    constexpr int U = sizeof(T) == 2 ? 8 : 4;
    if (r >= r1) {
#pragma unroll
        for (int i = 0; i < 8; i++) out[i] = {0.0f, 0.0f, 0.0f};
        return 0;
    }
    float k[8], s1[8] = {}, s2[8] = {};
    unpack(ld_unit<T, AW>(x + (int64_t)r * pitch, cnt), k);
    int n = 0;
    for (; r < r1; r += U * step) {
        Raw<T> raw[U];
#pragma unroll
        for (int u = 0; u < U; u++)
            if (r + u * step < r1) raw[u] = ld_unit<T, AW>(x + (int64_t)(r + u * step) * pitch, cnt);
#pragma unroll
        for (int u = 0; u < U; u++)
            if (r + u * step < r1) {
                float v[8];
                unpack(raw[u], v);
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const float dv = v[i] - k[i];
                    s1[i] += dv;
                    s2[i] = __fmaf_rn(dv, dv, s2[i]);
                }
                n++;
            }
    }
    const float inv = 1.0f / (float)n;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const float m = s1[i] * inv;
        out[i] = {k[i], m, fmaxf(__fmaf_rn(-m, s1[i], s2[i]), 0.0f)};
    }
    return n;
}

// Group moments from channel moments of equal counts: sub-warps of `lanes`
// lanes take a group each; f(group, moments) on the sub-warp's first lane.
template <class F>
__device__ __forceinline__ void group_moments(const Moments* chan_m, int groups, int d, float rows,
                                              F&& f) {
    int lanes = 1;
    while (lanes < d && lanes < 32) lanes *= 2;
    const int per = kThreads / lanes, lane = threadIdx.x % lanes;
    for (int g0 = 0; g0 < groups; g0 += per) {
        const int g = g0 + threadIdx.x / lanes;
        const Moments* c = chan_m + (int64_t)g * d;
        const float k = g < groups ? c[0].k : 0.0f;
        float off = 0.0f, m2 = 0.0f;
        if (g < groups)
            for (int i = lane; i < d; i += lanes) off += (c[i].k - k) + c[i].off;
        for (int o = lanes / 2; o; o /= 2) off += __shfl_xor_sync(~0u, off, o);
        off /= (float)d;
        if (g < groups)
            for (int i = lane; i < d; i += lanes) {
                const float dv = (c[i].k - k) + (c[i].off - off);
                m2 += __fmaf_rn(rows * dv, dv, c[i].m2);
            }
        for (int o = lanes / 2; o; o /= 2) m2 += __shfl_xor_sync(~0u, m2, o);
        if (g < groups && lane == 0) f(g, Moments{k, off, m2});
    }
}

// ---- forward: moments of each (chunk, sample), joined, then applied ----------

template <class T, int AW>
__global__ void __launch_bounds__(kThreads) k_stats(Batch B, Moments* __restrict__ part) {
    extern __shared__ Moments sm[];
    __shared__ float cnt[2 * kThreads];
    Moments* chan_m = sm;                              // B.c, rounded up to units
    Moments* red = sm + (int64_t)B.units * kUnit;      // phases * tile * 8
    const int n = blockIdx.x / B.chunks, k = blockIdx.x % B.chunks;
    int r0, r1;
    chunk_rows(valid_rows(B, n), B.chunks, k, r0, r1);
    const T* x = (const T*)B.x + (int64_t)n * B.xs;
    const int phase = threadIdx.x / B.tile, u = threadIdx.x % B.tile;
    for (int t = 0; t < B.tiles; t++) {
        const int unit = t * B.tile + u, width = B.tile * kUnit;
        if (phase < B.phases) {
            Moments m[8] = {};
            int rows = 0;
            if (unit < B.units)
                rows = unit_moments<T, AW>(x + unit * kUnit, B.xr, r0 + phase, r1, B.phases,
                                           min(kUnit, B.c - unit * kUnit), m);
#pragma unroll
            for (int i = 0; i < 8; i++) red[phase * width + u * 8 + i] = m[i];
            if (u == 0) cnt[phase] = (float)rows;
        }
        __syncthreads();
        join_phases(red, cnt, B.phases, width, phase, u * 8, u == 0);
        if (phase == 0 && unit < B.units) {
#pragma unroll
            for (int i = 0; i < 8; i++) chan_m[unit * kUnit + i] = red[u * 8 + i];
        }
        __syncthreads();
    }
    Moments* o = part + ((int64_t)n * B.chunks + k) * B.g;
    group_moments(chan_m, B.g, B.d, (float)(r1 - r0), [&](int g, Moments m) { o[g] = m; });
}

// One warp per (sample, group) joins the chunks, in double.
__global__ void __launch_bounds__(kThreads)
    k_join(Batch B, const Moments* __restrict__ part, float* __restrict__ mean,
           float* __restrict__ rstd) {
    const int64_t id = ((int64_t)blockIdx.x * kThreads + threadIdx.x) / 32;
    const int lane = threadIdx.x % 32;
    if (id >= (int64_t)B.n * B.g) return;
    const int n = (int)(id / B.g), g = (int)(id % B.g);
    const int len = valid_rows(B, n);
    const Moments* p = part + (int64_t)n * B.chunks * B.g + g;
    const double count = (double)len * B.d;
    double mu = 0.0, m2 = 0.0;
    for (int k = lane; k < B.chunks; k += 32) {
        int r0, r1;
        chunk_rows(len, B.chunks, k, r0, r1);
        const Moments q = p[(int64_t)k * B.g];
        mu += (double)(r1 - r0) * B.d * ((double)q.k + q.off);
    }
    for (int o = 16; o; o /= 2) mu += __shfl_xor_sync(~0u, mu, o);
    mu = len ? mu / count : 0.0;
    for (int k = lane; k < B.chunks; k += 32) {
        int r0, r1;
        chunk_rows(len, B.chunks, k, r0, r1);
        const Moments q = p[(int64_t)k * B.g];
        const double dv = (double)q.k + q.off - mu;
        m2 += q.m2 + (double)(r1 - r0) * B.d * dv * dv;
    }
    for (int o = 16; o; o /= 2) m2 += __shfl_xor_sync(~0u, m2, o);
    if (lane == 0) {
        mean[id] = (float)mu;
        rstd[id] = (float)(1.0 / sqrt((len ? m2 / count : 0.0) + (double)B.eps));
    }
}

// The eight channels' parameters of a unit.
struct Params {
    float mean[8], rstd[8], w[8], b[8];
};
__device__ __forceinline__ void load_params(const Batch& B, int n, int unit, Params& q) {
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const int c = min(unit * kUnit + i, B.c - 1);
        const int64_t g = (int64_t)n * B.g + c / B.d;
        q.mean[i] = __ldg(B.mean + g);
        q.rstd[i] = __ldg(B.rstd + g);
        q.w[i] = B.w ? ld_param(B.w, B.ptype, c) : 1.0f;
        q.b[i] = B.b ? ld_param(B.b, B.ptype, c) : 0.0f;
    }
}

template <class T, int AW>
__device__ __forceinline__ void keep_row(const Batch& B, const Raw<T>& raw, int64_t row, int unit,
                                         int cnt, bool on) {
    float v[8];
    unpack(raw, v);
    const uint32_t m = block_max(on ? largest(v) : 0u, B.lanes);
    float scale, inverse;
    block_scale(m, scale, inverse);
    if (!on) return;
    st_codes<AW == 16>(B.codes + row * B.c + unit * kUnit, encode(v, inverse), cnt);
    if (unit % B.lanes == 0) B.scales[row * B.nblk + (unit >> B.shift)] = scale;
}

template <class T, int AW>
__global__ void __launch_bounds__(kThreads) k_apply(Batch B) {
    constexpr int U = sizeof(T) == 2 ? 4 : 2;
    const int n = blockIdx.x / B.chunks;
    int r0, r1;
    chunk_rows(valid_rows(B, n), B.chunks, blockIdx.x % B.chunks, r0, r1);
    if (r0 >= r1) return;
    const T* x = (const T*)B.x + (int64_t)n * B.xs;
    T* y = (T*)B.out + (int64_t)n * B.os;
    const int phase = threadIdx.x / B.tile, u = threadIdx.x % B.tile;
    for (int t = 0; t < B.tiles; t++) {
        const int unit = t * B.tile + u, cnt = min(kUnit, B.c - unit * kUnit);
        const bool on = phase < B.phases && unit < B.units;
        Params q;
        if (on) load_params(B, n, unit, q);
#pragma unroll
        for (int i = 0; i < 8; i++) q.w[i] *= q.rstd[i];
        for (int base = r0; base < r1; base += U * B.phases) {
            Raw<T> raw[U] = {};
#pragma unroll
            for (int j = 0; j < U; j++) {
                const int r = base + phase + j * B.phases;
                if (on && r < r1)
                    raw[j] = ld_unit<T, AW>(x + (int64_t)r * B.xr + unit * kUnit, cnt);
            }
#pragma unroll
            for (int j = 0; j < U; j++) {
                const int r = base + phase + j * B.phases;
                if (on && r < r1) {
                    float v[8];
                    unpack(raw[j], v);
#pragma unroll
                    for (int i = 0; i < 8; i++) v[i] = __fmaf_rn(v[i] - q.mean[i], q.w[i], q.b[i]);
                    activate<sizeof(T) == 2>(v, B.act, B.param);
                    Raw<T> o;
                    pack(v, o);
                    st_unit<T, AW>(y + (int64_t)r * B.orow + unit * kUnit, o, cnt);
                }
                if (B.codes)
                    keep_row<T, AW>(B, raw[j], (int64_t)n * B.s + r, unit, cnt, on && r < r1);
            }
        }
    }
}

// ---- backward ---------------------------------------------------------------------

// A unit of x: from the tensor, or from its checkpoint.
template <class T, int AW, bool kFrom>
struct Input {
    Raw<T> raw;
    Codes codes;
    float scale;
    __device__ __forceinline__ void load(const Batch& B, int n, int r, int unit, int cnt) {
        if (kFrom) {
            const int64_t row = (int64_t)n * B.s + r;
            codes = ld_codes<AW == 16>(B.codes_in + row * B.c + unit * kUnit, cnt);
            scale = __ldg(B.scales_in + row * B.nblk + (unit >> B.shift));
        } else {
            raw = ld_unit<T, AW>((const T*)B.x + (int64_t)n * B.xs + (int64_t)r * B.xr + unit * kUnit,
                                 cnt);
        }
    }
    __device__ __forceinline__ void get(float (&v)[8]) const {
        if (kFrom)
            decode(codes, scale, v);
        else
            unpack(raw, v);
    }
};

// xh and dz = dy * act'(z) of one unit.
template <class T>
__device__ __forceinline__ void slopes(const Batch& B, const Params& q, const Raw<T>& dy,
                                       float (&xh)[8], float (&dz)[8]) {
    float z[8], f[8], s[8];
#pragma unroll
    for (int i = 0; i < 8; i++) {
        xh[i] = (xh[i] - q.mean[i]) * q.rstd[i];
        z[i] = __fmaf_rn(xh[i], q.w[i], q.b[i]);
    }
    activate_slope<sizeof(T) == 2>(z, f, s, B.act, B.param);
    unpack(dy, dz);
#pragma unroll
    for (int i = 0; i < 8; i++) dz[i] *= s[i];
}

// A = sum dz and B = sum dz*xh of every channel of a chunk.
template <class T, int AW, bool kFrom>
__global__ void __launch_bounds__(kThreads) k_back_stats(Batch B, float2* __restrict__ part) {
    extern __shared__ float2 red2[];
    constexpr int U = sizeof(T) == 2 ? 4 : 2;
    const int n = blockIdx.x / B.chunks, k = blockIdx.x % B.chunks;
    int r0, r1;
    chunk_rows(valid_rows(B, n), B.chunks, k, r0, r1);
    const T* dy = (const T*)B.dy + (int64_t)n * B.ys;
    float2* o = part + ((int64_t)n * B.chunks + k) * B.c;
    const int phase = threadIdx.x / B.tile, u = threadIdx.x % B.tile, width = B.tile * kUnit;
    for (int t = 0; t < B.tiles; t++) {
        const int unit = t * B.tile + u, cnt = min(kUnit, B.c - unit * kUnit);
        const bool on = phase < B.phases && unit < B.units;
        float a[8] = {}, b[8] = {};
        if (on && r0 < r1) {
            Params q;
            load_params(B, n, unit, q);
            for (int r = r0 + phase; r < r1; r += U * B.phases) {
                Raw<T> g[U];
                Input<T, AW, kFrom> x[U];
#pragma unroll
                for (int j = 0; j < U; j++) {
                    const int rr = r + j * B.phases;
                    if (rr < r1) {
                        g[j] = ld_unit<T, AW>(dy + (int64_t)rr * B.yr + unit * kUnit, cnt);
                        x[j].load(B, n, rr, unit, cnt);
                    }
                }
#pragma unroll
                for (int j = 0; j < U; j++)
                    if (r + j * B.phases < r1) {
                        float xh[8], dz[8];
                        x[j].get(xh);
                        slopes(B, q, g[j], xh, dz);
#pragma unroll
                        for (int i = 0; i < 8; i++) {
                            a[i] += dz[i];
                            b[i] = __fmaf_rn(dz[i], xh[i], b[i]);
                        }
                    }
            }
        }
        if (phase < B.phases) {
#pragma unroll
            for (int i = 0; i < 8; i++) red2[phase * width + u * 8 + i] = make_float2(a[i], b[i]);
        }
        __syncthreads();
        for (int m = B.phases; m > 1;) {
            const int h = (m + 1) / 2;
            if (phase + h < m) {
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    float2* p = red2 + phase * width + u * 8 + i;
                    const float2 w = p[h * width];
                    p->x += w.x;
                    p->y += w.y;
                }
            }
            m = h;
            __syncthreads();
        }
        if (phase == 0 && unit < B.units) {
            for (int i = 0; i < cnt; i++) o[unit * kUnit + i] = red2[u * 8 + i];
        }
        __syncthreads();
    }
}

// One warp per (sample, group): its means of dz*w and dz*w*xh.
__global__ void __launch_bounds__(kThreads)
    k_back_groups(Batch B, const float2* __restrict__ part, float2* __restrict__ means) {
    const int64_t id = ((int64_t)blockIdx.x * kThreads + threadIdx.x) / 32;
    const int lane = threadIdx.x % 32;
    if (id >= (int64_t)B.n * B.g) return;
    const int n = (int)(id / B.g), g = (int)(id % B.g);
    const int len = valid_rows(B, n);
    double s1 = 0.0, s2 = 0.0;
    const int64_t items = (int64_t)B.chunks * B.d;
    for (int64_t i = lane; i < items; i += 32) {
        const int k = (int)(i / B.d), c = g * B.d + (int)(i % B.d);
        const float2 v = part[((int64_t)n * B.chunks + k) * B.c + c];
        const double w = B.w ? ld_param(B.w, B.ptype, c) : 1.0f;
        s1 += w * v.x;
        s2 += w * v.y;
    }
    for (int o = 16; o; o /= 2) {
        s1 += __shfl_xor_sync(~0u, s1, o);
        s2 += __shfl_xor_sync(~0u, s2, o);
    }
    const double count = len ? (double)len * B.d : 1.0;
    if (lane == 0) means[id] = make_float2((float)(s1 / count), (float)(s2 / count));
}

// dbias and dweight: 32 channels per block, its warps taking the rows of part
// in turn.
__global__ void __launch_bounds__(kThreads)
    k_back_params(const float2* __restrict__ part, int64_t rows, int c, float* __restrict__ dw,
                  float* __restrict__ db) {
    __shared__ double2 sm[kThreads / 32][32];
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    const int ch = blockIdx.x * 32 + lane;
    double2 s = make_double2(0.0, 0.0);
    if (ch < c)
        for (int64_t r = warp; r < rows; r += kThreads / 32) {
            const float2 v = part[r * c + ch];
            s.x += v.x;
            s.y += v.y;
        }
    sm[warp][lane] = s;
    __syncthreads();
    if (warp == 0 && ch < c) {
        for (int w = 1; w < kThreads / 32; w++) {
            s.x += sm[w][lane].x;
            s.y += sm[w][lane].y;
        }
        if (db) db[ch] = (float)s.x;
        if (dw) dw[ch] = (float)s.y;
    }
}

template <class T, int AW, bool kFrom>
__global__ void __launch_bounds__(kThreads)
    k_back_apply(Batch B, const float2* __restrict__ means) {
    constexpr int U = 2;
    const int n = blockIdx.x / B.chunks;
    int r0, r1;
    chunk_rows(valid_rows(B, n), B.chunks, blockIdx.x % B.chunks, r0, r1);
    if (r0 >= r1) return;
    const T* dy = (const T*)B.dy + (int64_t)n * B.ys;
    T* dx = (T*)B.out + (int64_t)n * B.os;
    const int phase = threadIdx.x / B.tile, u = threadIdx.x % B.tile;
    if (phase >= B.phases) return;
    for (int t = 0; t < B.tiles; t++) {
        const int unit = t * B.tile + u, cnt = min(kUnit, B.c - unit * kUnit);
        if (unit >= B.units) break;
        Params q;
        load_params(B, n, unit, q);
        float s1[8], s2[8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int c = min(unit * kUnit + i, B.c - 1);
            const float2 v = __ldg(means + (int64_t)n * B.g + c / B.d);
            s1[i] = v.x;
            s2[i] = v.y;
        }
        for (int r = r0 + phase; r < r1; r += U * B.phases) {
            Raw<T> g[U];
            Input<T, AW, kFrom> x[U];
#pragma unroll
            for (int j = 0; j < U; j++) {
                const int rr = r + j * B.phases;
                if (rr < r1) {
                    g[j] = ld_unit<T, AW>(dy + (int64_t)rr * B.yr + unit * kUnit, cnt);
                    x[j].load(B, n, rr, unit, cnt);
                }
            }
#pragma unroll
            for (int j = 0; j < U; j++) {
                const int rr = r + j * B.phases;
                if (rr < r1) {
                    float xh[8], dz[8];
                    x[j].get(xh);
                    slopes(B, q, g[j], xh, dz);
#pragma unroll
                    for (int i = 0; i < 8; i++)
                        dz[i] = q.rstd[i] * (__fmaf_rn(dz[i], q.w[i], -s1[i]) - xh[i] * s2[i]);
                    Raw<T> o;
                    pack(dz, o);
                    st_unit<T, AW>(dx + (int64_t)rr * B.orow + unit * kUnit, o, cnt);
                }
            }
        }
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

void fill(Batch& B, const simtgo_group_norm& c, const sg::DevInfo& d, bool kept) {
    B.n = c.samples;
    B.s = c.positions;
    B.c = c.channels;
    B.g = c.groups;
    B.d = c.channels / c.groups;
    B.units = (c.channels + kUnit - 1) / kUnit;
    B.lanes = kept ? std::min(c.block / kUnit, ceil_pow2(std::min(B.units, 32))) : 1;
    B.shift = 0;
    while (kept && (kUnit << B.shift) < c.block) B.shift++;
    B.nblk = kept ? (c.channels + c.block - 1) / c.block : 0;
    const int upad = (B.units + B.lanes - 1) / B.lanes * B.lanes;
    B.tiles = (upad + kThreads - 1) / kThreads;
    B.tile = ((upad + B.tiles - 1) / B.tiles + B.lanes - 1) / B.lanes * B.lanes;
    B.tiles = (upad + B.tile - 1) / B.tile;
    B.phases = kThreads / B.tile;
    // Six blocks for each SM over the whole batch, but eight rows a thread.
    const int64_t most = std::max<int64_t>(1, sg::ceil_div(B.s, 8 * B.phases));
    B.chunks = (int)std::max<int64_t>(1, std::min(most, sg::ceil_div(6 * d.sms, B.n)));
    B.ptype = c.param_type;
    B.act = c.act;
    B.param = c.act_param;
    B.eps = c.eps;
}

template <class K>
int allow_smem(K kernel, size_t bytes, const char* name) {
    if (bytes <= 48 * 1024) return 0;
    return sg::cuda_status(
        cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes), name);
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
    B.codes = codes;
    B.scales = scales;
    B.xs = c.x_sample;
    B.xr = c.x_row;
    B.os = c.y_sample;
    B.orow = c.y_row;
    fill(B, c, *d, kept);
    int width = access_width(c.type, {{x, rx.pitch0 / elem_size(c.type), rx.pitch1 / elem_size(c.type)},
                                      {y, ry.pitch0 / elem_size(c.type), ry.pitch1 / elem_size(c.type)}});
    if (kept && width == 16 && (c.channels % kUnit || ((uintptr_t)codes & 7))) width = 4;
    cudaStream_t s = (cudaStream_t)stream;
    const int64_t parts = stats * B.chunks;
    Scratch scratch;
    if ((rc = scratch.alloc(sizeof(Moments) * parts + 8 * stats, s))) return rc;
    Moments* part = (Moments*)scratch.p;
    float* own = (float*)(part + parts);
    float* mu = mean ? mean : own;
    float* rs = rstd ? rstd : own + stats;
    B.mean = mu;
    B.rstd = rs;
    const unsigned grid = (unsigned)B.chunks * (unsigned)B.n;
    const size_t smem = sizeof(Moments) * kUnit * ((size_t)B.units + (size_t)B.phases * B.tile);
    return by_type(c.type, width, [&](auto* t, auto w) {
        using T = std::remove_pointer_t<decltype(t)>;
        constexpr int AW = decltype(w)::value;
        if (int e = allow_smem(k_stats<T, AW>, smem, K)) return e;
        sg::before_launch();
        k_stats<T, AW><<<grid, kThreads, smem, s>>>(B, part);
        if (int e = sg::launch_status(K)) return e;
        k_join<<<(unsigned)sg::ceil_div(stats, kThreads / 32), kThreads, 0, s>>>(B, part, mu, rs);
        if (int e = sg::launch_status(K)) return e;
        if (!elems) return 0;
        k_apply<T, AW><<<grid, kThreads, 0, s>>>(B);
        return sg::launch_status(K);
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
    B.codes_in = codes;
    B.scales_in = scales;
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
    fill(B, c, *d, from);
    const int e = elem_size(c.type);
    int width = access_width(c.type, {{x, rx.pitch0 / e, rx.pitch1 / e},
                                      {dy, ry.pitch0 / e, ry.pitch1 / e},
                                      {dx, rd.pitch0 / e, rd.pitch1 / e}});
    if (from && width == 16 && (c.channels % kUnit || ((uintptr_t)codes & 7))) width = 4;
    const int64_t parts = (int64_t)c.samples * B.chunks * c.channels;
    Scratch scratch;
    if ((rc = scratch.alloc(sizeof(float2) * (parts + stats), s))) return rc;
    float2* part = (float2*)scratch.p;
    float2* means = part + parts;
    const unsigned grid = (unsigned)B.chunks * (unsigned)B.n;
    const size_t smem = sizeof(float2) * kUnit * (size_t)B.phases * B.tile;
    return by_type(c.type, width, [&](auto* t, auto w) {
        using T = std::remove_pointer_t<decltype(t)>;
        constexpr int AW = decltype(w)::value;
        sg::before_launch();
        if (from)
            k_back_stats<T, AW, true><<<grid, kThreads, smem, s>>>(B, part);
        else
            k_back_stats<T, AW, false><<<grid, kThreads, smem, s>>>(B, part);
        if (int r = sg::launch_status(K)) return r;
        if (dweight || dbias) {
            k_back_params<<<(unsigned)sg::ceil_div(c.channels, 32), kThreads, 0, s>>>(
                part, (int64_t)c.samples * B.chunks, c.channels, dweight, dbias);
            if (int r = sg::launch_status(K)) return r;
        }
        if (!dx) return 0;
        k_back_groups<<<(unsigned)sg::ceil_div(stats, kThreads / 32), kThreads, 0, s>>>(B, part,
                                                                                      means);
        if (int r = sg::launch_status(K)) return r;
        if (from)
            k_back_apply<T, AW, true><<<grid, kThreads, 0, s>>>(B, means);
        else
            k_back_apply<T, AW, false><<<grid, kThreads, 0, s>>>(B, means);
        return sg::launch_status(K);
    });
}

}  // extern "C"
