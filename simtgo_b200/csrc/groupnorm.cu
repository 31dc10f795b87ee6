// groupnorm.cu -- group norm with an activation over channels-last batches,
// forward and backward, with the input kept as an 8-bit checkpoint on request.
//
// Mathematics. A thread sums x - K and (x - K)^2 over short runs of rows, K being
// the mean of the runs before (at first a value that it meets), and joins the
// runs: the variance stays exact to a few ulps however far the mean is from zero
// and whatever the first values are. Threads, blocks and chunks of a sample are
// then joined by counts, means and sums of squared deviations (Chan, Golub and
// LeVeque's pairwise formula), never by raw squares; a mean stays K plus a small
// offset until the last join, so differences of means do not cancel. The backward
// pass needs, for each channel of a sample, A = sum dz and B = sum dz*xh: weighted
// and summed over a group's channels they give the group's two means in dx, and
// summed over the samples they are dbias and dweight, so one pass over x and dy
// serves both. All joins run in a fixed order.
//
// Two ways through the data, both reading it once from HBM:
//
// - k_norm, k_norm_back: a cluster of up to eight blocks takes a slab of whole
//   groups of one sample. Each block sums its share of the rows, keeping them in
//   shared memory (what does not fit is read again, last rows first, from L2);
//   the blocks exchange their sums over distributed shared memory, and each
//   finishes its own rows. One launch, nothing in HBM between. 8x4096x320 bf16
//   (82 KB a block, 256 blocks): 21 us with SiLU, of which 7 sum, 7 finish and 4
//   join and exchange; the HBM floor is 6.5. Backward 31 us, floor 9.7.
// - k_stats, k_join, k_apply (and their backward forms): where too few such
//   clusters exist to fill the GPU -- a few samples of very many positions --
//   every SM takes a chunk of a sample's rows, the chunks' sums are joined by a
//   small kernel, and a third pass walks the chunks from their ends, whose rows
//   L2 still holds. One 518400x128 bf16 sample: 29 us for the sums (4.6 TB/s,
//   profiled), 92 us with the join and the GELU pass; the floor is 41. The last
//   pass is bound by its arithmetic: exponential and reciprocal for every value, 55 % of
//   the special-function unit and 61 % of the issue slots at 16 warps an SM. A
//   4x16384x512 step, forward with its checkpoint and backward from it: 129 us.
#include <algorithm>
#include <atomic>
#include <cmath>
#include <numeric>
#include <type_traits>

#include "channels.cuh"

using namespace chan;

namespace {

constexpr int kThreads = 256;
// Blocks that an SM's registers hold, at least, and chunks that an SM takes: three
// and four of both measured slower (the 518400x128 sample 93 and 104 us, 90 with
// two). Fewer registers and shorter chunks were not measured apart.
constexpr int kBlocks = 2;
constexpr int kAhead = 2;  // batches of a ring where rows do not stay; four measured the same
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
    int keep, ahead;                 // batches of rows that stay in shared memory; in flight
    int keep_all;                    // every batch stays: there is no ring
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

// Rows of [r0, r1) that fall to a phase.
__device__ __forceinline__ int phase_rows(const Batch& B, int r0, int r1, int phase) {
    return phase < B.phases ? (r1 - r0 - phase + B.phases - 1) / B.phases : 0;
}

// ---- between blocks and grids --------------------------------------------------

// Blocks of a cluster, at most: 16 left SMs idle (backward above 48 us, not 31).
constexpr int kCluster = 8;

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

// ---- rows through shared memory --------------------------------------------------
// A thread copies its own rows' units to its own places in shared memory,
// asynchronously and several batches ahead, and reads them back itself: the
// loads in flight cost no registers, no barrier is needed, and a batch that
// stays there is read again without leaving the SM. The first `keep` batches of
// a thread's rows have places of their own; the others share a ring of `ahead`.

__device__ __forceinline__ uint32_t shared_addr(const void* p) {
    return (uint32_t)__cvta_generic_to_shared(p);
}
template <int kBytes>
__device__ __forceinline__ void copy_async(uint32_t dst, const void* src) {
    if (kBytes == 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
    else
        asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(src), "n"(kBytes)
                     : "memory");
}
__device__ __forceinline__ void copy_commit() {
    asm volatile("cp.async.commit_group;" ::: "memory");
}
// All but the newest `ahead` - 1 groups of this thread have arrived.
__device__ __forceinline__ void copy_wait(int ahead) {
    if (ahead == 8)
        asm volatile("cp.async.wait_group 7;" ::: "memory");
    else if (ahead == 4)
        asm volatile("cp.async.wait_group 3;" ::: "memory");
    else if (ahead == 2)
        asm volatile("cp.async.wait_group 1;" ::: "memory");
    else
        asm volatile("cp.async.wait_group 0;" ::: "memory");
}
__device__ __forceinline__ void st_shared(uint32_t a, uint32_t v) {
    asm volatile("st.shared.u32 [%0], %1;" ::"r"(a), "r"(v) : "memory");
}

constexpr int kPlane = 16 * kThreads;  // 16 bytes of every thread

// Unit of cnt channels at p to this thread's 16 bytes (two planes for float32)
// at dst; channels it lacks become zeros.
template <class T, int AW>
__device__ __forceinline__ void copy_unit(uint32_t dst, const T* p, int cnt) {
    if (AW == 16 && cnt == kUnit) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; i++)
            copy_async<16>(dst + i * kPlane, reinterpret_cast<const char*>(p) + 16 * i);
    } else if (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const uint32_t to = dst + i / 4 * kPlane + i % 4 * 4;
            if (i < cnt)
                copy_async<4>(to, p + i);
            else
                st_shared(to, 0);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if (2 * i + 1 < cnt)
                copy_async<4>(dst + 4 * i, p + 2 * i);
            else
                st_shared(dst + 4 * i, 2 * i < cnt ? (uint32_t)*reinterpret_cast<const uint16_t*>(
                                                         p + 2 * i)
                                                   : 0u);
        }
    }
}
template <class T>
__device__ __forceinline__ void store_unit(uint32_t dst, const Raw<T>& r) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; i++)
        asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(dst + i * kPlane),
                     "r"(r.q[i].x), "r"(r.q[i].y), "r"(r.q[i].z), "r"(r.q[i].w)
                     : "memory");
}
template <class T>
__device__ __forceinline__ Raw<T> shared_unit(uint32_t src) {
    Raw<T> r;
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; i++)
        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(r.q[i].x), "=r"(r.q[i].y), "=r"(r.q[i].z), "=r"(r.q[i].w)
                     : "r"(src + i * kPlane));
    return r;
}

// f(j) for the first `live` of a batch's U rows. A whole batch has no conditions
// in it, so that its rows' instructions interleave.
template <int U, class F>
__device__ __forceinline__ void each_row(int live, F&& f) {
    if (live >= U) {
#pragma unroll
        for (int j = 0; j < U; j++) f(j);
    } else {
#pragma unroll
        for (int j = 0; j < U; j++)
            if (j < live) f(j);
    }
}

// What a row gives a thread: forward a unit of x; backward one of dy and one of
// x, or of its checkpoint.
template <class T>
struct FwdRow {
    static constexpr int kBytes = (int)sizeof(Raw<T>);
    static constexpr int kRows = sizeof(T) == 2 ? 4 : 2;  // of a batch
    const T* x;
    int64_t step;
    __device__ __forceinline__ FwdRow(const Batch& B, int n, int64_t row, int unit)
        : x((const T*)B.x + n * B.xs + row * B.xr + unit * kUnit), step(B.phases * B.xr) {}
    __device__ __forceinline__ void move(int rows) { x += rows * step; }
    // The next U rows (where live) to consecutive slots; at ends past them.
    template <int AW>
    __device__ __forceinline__ void copy(uint32_t slot, int live, int cnt) {
        constexpr int U = kRows;
        if constexpr (AW == 2) {
            Raw<T> r[U];
#pragma unroll
            for (int u = 0; u < U; u++) {
                if (u < live) r[u] = ld_unit<T, AW>(x, cnt);
                x += step;
            }
#pragma unroll
            for (int u = 0; u < U; u++)
                if (u < live) store_unit<T>(slot + u * kBytes * kThreads, r[u]);
        } else {
            each_row<U>(live, [&](int u) {
                copy_unit<T, AW>(slot + u * kBytes * kThreads, x + u * step, cnt);
            });
            x += U * step;
        }
    }
};
template <class T, bool kFrom>
struct BackRow {
    static constexpr int kX = (int)sizeof(Raw<T>) * kThreads;  // dy first
    static constexpr int kBytes = (int)sizeof(Raw<T>) + (kFrom ? 12 : (int)sizeof(Raw<T>));
    static constexpr int kRows = sizeof(T) == 2 ? 2 : 1;
    const T *dy, *x;
    const int8_t* codes;
    const float* scale;
    int64_t dy_step, x_step, scale_step;
    __device__ __forceinline__ BackRow(const Batch& B, int n, int64_t row, int unit) {
        dy = (const T*)B.dy + n * B.ys + row * B.yr + unit * kUnit;
        dy_step = B.phases * B.yr;
        if (kFrom) {
            const KeptAt at = kept_at(B.kept, (int64_t)n * B.s + row, B.phases, unit);
            codes = at.codes;
            scale = at.scale;
            x_step = at.codes_step;
            scale_step = at.scale_step;
        } else {
            x = (const T*)B.x + n * B.xs + row * B.xr + unit * kUnit;
            x_step = B.phases * B.xr;
        }
    }
    __device__ __forceinline__ void move(int rows) {
        dy += rows * dy_step;
        if (kFrom) {
            codes += rows * x_step;
            scale += rows * scale_step;
        } else {
            x += rows * x_step;
        }
    }
    template <int AW>
    __device__ __forceinline__ void copy(uint32_t slot, int live, int cnt) {
        constexpr int U = kRows;
        const uint32_t cs = kX + threadIdx.x * 8 - threadIdx.x * 16;        // codes' place
        const uint32_t ss = kX + 8 * kThreads + threadIdx.x * 4 - threadIdx.x * 16;
        // Asynchronously where a unit is few copies: 4x16384x130 f16 43 us, 59 us
        // through registers; 4x16384x129 float32 (16 copies a row) 76 and 69.
        if constexpr (AW == 16 || (AW == 4 && sizeof(T) == 2 && !kFrom)) {
#pragma unroll
            for (int u = 0; u < U; u++) {
                const uint32_t to = slot + u * kBytes * kThreads;
                if (u < live) {
                    copy_unit<T, AW>(to, dy, cnt);
                    if (kFrom) {
                        copy_async<8>(to + cs, codes);
                        copy_async<4>(to + ss, scale);
                    } else {
                        copy_unit<T, AW>(to + kX, x, cnt);
                    }
                }
                move(1);
            }
        } else {
            Raw<T> a[U], b[U];
            Codes c[U];
            float f[U];
#pragma unroll
            for (int u = 0; u < U; u++) {
                if (u < live) {
                    a[u] = ld_unit<T, AW>(dy, cnt);
                    if (kFrom) {
                        c[u] = ld_codes<false>(codes, cnt);
                        f[u] = __ldg(scale);
                    } else {
                        b[u] = ld_unit<T, AW>(x, cnt);
                    }
                }
                move(1);
            }
#pragma unroll
            for (int u = 0; u < U; u++) {
                const uint32_t to = slot + u * kBytes * kThreads;
                if (u < live) {
                    store_unit<T>(to, a[u]);
                    if (kFrom) {
                        st_shared(to + cs, c[u].q.x);
                        st_shared(to + cs + 4, c[u].q.y);
                        st_shared(to + ss, __float_as_uint(f[u]));
                    } else {
                        store_unit<T>(to + kX, b[u]);
                    }
                }
            }
        }
    }
    static __device__ __forceinline__ V8 input(uint32_t slot) {
        if (!kFrom) return unpack(shared_unit<T>(slot + kX));
        Codes c;
        float f;
        asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];"
                     : "=r"(c.q.x), "=r"(c.q.y)
                     : "r"(slot + kX + threadIdx.x * 8 - threadIdx.x * 16));
        asm volatile("ld.shared.f32 %0, [%1];"
                     : "=f"(f)
                     : "r"(slot + kX + 8 * kThreads + threadIdx.x * 4 - threadIdx.x * 16));
        return decode(c, f);
    }
};

// A thread's rows in batches: `most` rows for the block's busiest thread, `mine`
// for this one. start() asks for the first batches, so that whatever comes
// between it and down() (or up()) hides their latency.
template <class Row, int AW>
struct Feed {
    Row row;
    uint32_t base;
    int keep, ahead, batches, mine, next, cnt;
    __device__ __forceinline__ Feed(const Batch& B, const Row& first, void* smem, int most,
                                    int rows, int channels)
        : row(first),
          base(shared_addr(smem) + threadIdx.x * 16),
          keep(B.keep),
          ahead(B.ahead),
          batches((most + Row::kRows - 1) / Row::kRows),
          mine(rows),
          cnt(channels) {}
    __device__ __forceinline__ uint32_t slot(int b) const {
        const int at = b < keep ? b : keep + (b & (ahead - 1));
        return base + at * (Row::kRows * Row::kBytes * kThreads);
    }
    __device__ __forceinline__ void ask_down() {
        if (next < batches) row.template copy<AW>(slot(next), mine - next * Row::kRows, cnt);
        copy_commit();
        next++;
    }
    __device__ __forceinline__ void start_down() {
        next = 0;
        for (int j = 0; j < ahead; j++) ask_down();
    }
    // Batch by batch, first to last: f(slot, first row of the batch).
    template <class F>
    __device__ __forceinline__ void down(F&& f) {
        for (int b = 0; b < batches; b++) {
            copy_wait(ahead);
            f(slot(b), b * Row::kRows);
            ask_down();
        }
    }
    // Last to first; the kept batches are not copied again.
    __device__ __forceinline__ void ask_up() {
        if (next >= keep) {
            row.template copy<AW>(slot(next), mine - next * Row::kRows, cnt);
            row.move(-2 * Row::kRows);
            next--;
        }
        copy_commit();
    }
    __device__ __forceinline__ void start_up(const Row& first) {
        row = first;
        next = batches - 1;
        row.move(next * Row::kRows);
        for (int j = 0; j < ahead; j++) ask_up();
    }
    template <class F>
    __device__ __forceinline__ void up(F&& f) {
        for (int b = batches - 1; b >= 0; b--) {
            if (b >= keep) copy_wait(ahead);
            f(slot(b), b * Row::kRows);
            if (b >= keep) ask_up();
        }
    }
};

// ---- moments ------------------------------------------------------------------
// A cell is what a thread sums together: a channel, or -- where groups are whole
// units (kSame) -- a unit.

struct Moments {  // the mean is k + off; m2: the sum of squared deviations from it
    float k, off, m2;
};

// Joins (na, a) and (nb, b).
__device__ __forceinline__ Moments join(float na, Moments a, float nb, Moments b) {
    if (na == 0.0f) return b;
    const float f = __fdividef(nb, na + nb), d = nb > 0.0f ? (b.k - a.k) + (b.off - a.off) : 0.0f;
    return {a.k, __fmaf_rn(d, f, a.off), __fmaf_rn(d * d, na * f, nb > 0.0f ? a.m2 + b.m2 : a.m2)};
}

// The cells' moments of every phase in shared memory, arrays apart.
struct CellSums {
    float *k, *off, *m2;
    int width;  // cells of a phase, padded so that phases start in other banks
    __device__ __forceinline__ CellSums(float* base, int phases, int cells, bool units)
        : width(units ? cells | 1 : cells + 4) {
        k = base;
        off = k + phases * width;
        m2 = off + phases * width;
    }
};
__host__ __device__ constexpr int cell_floats(int phases, int cells, bool units) {
    return 3 * phases * (units ? cells | 1 : cells + 4);
}

// A thread sums its rows in runs of at most kRun, which its own places in shared
// memory collect: however many rows it has, no float32 sum is of more than a run
// of rows or of runs, and the errors grow with the square root of either.
constexpr int kRun = 64;
__device__ __forceinline__ void add4(float* to, float2 a, float2 b) {
    float4* p = reinterpret_cast<float4*>(to);
    const float4 v = *p;
    *p = make_float4(v.x + a.x, v.y + a.y, v.z + b.x, v.w + b.y);
}

// Sums this thread's cells down its rows and stores their moments: run by run,
// the first about the first row's value (kSame: the mean of its eight) and each
// further one about the mean so far. About a value K that lies D from a run's
// mean, n values' squares hold n D^2 that the run's own moment has not; an
// outlier for K, kept for all rows, would cancel nearly all of the sum (rstd of
// 64 channels by 65536 positions 3e-5 off for one first value of 4096). A run is
// at most three times as long as all rows before it, so that of n D^2 the join
// keeps a quarter at least.
template <class T, int AW, bool kSame>
__device__ __forceinline__ void sum_rows(Feed<FwdRow<T>, AW>& feed, const CellSums& out, int phase,
                                         int u) {
    constexpr int U = FwdRow<T>::kRows, P = kSame ? 1 : 4;
    constexpr float kPer = kSame ? kUnit : 1;  // values of a row in a cell
    float2 k[P] = {}, s1[P] = {}, s2[P] = {};
    const int at = phase * out.width + u * (kSame ? 1 : 8);
    int before = 0;  // rows of the runs that ended
    // Ends the run of rows [before, rows): its offset from k and its moment, joined
    // to those before it. Unless it is the last one, k moves to the mean so far,
    // and the offset becomes what that rounding left.
    const auto end_run = [&](int rows, bool last) {
        const float n = (float)(rows - before);
        const float inv = rows > before ? 1.0f / (n * kPer) : 0.0f;
        const float f = before ? n / (float)rows : 1.0f, w = (float)before * kPer * f;
        if constexpr (kSame) {
            const float a = s1[0].x + s1[0].y, q = s2[0].x + s2[0].y;
            float off = a * inv, m2 = __fmaf_rn(-off, a, q);
            m2 = m2 < 0.0f ? 0.0f : m2;
            if (before) {
                const float o = out.off[at], d = off - o;
                off = __fmaf_rn(d, f, o);
                m2 = __fmaf_rn(d * d, w, m2 + out.m2[at]);
            }
            if (!last) {
                const float to = k[0].x + off, moved = to - k[0].x;
                off = (k[0].x - (to - moved)) + (off - moved);
                k[0] = both(to);
            } else {
                out.k[at] = k[0].x;
            }
            out.off[at] = off;
            out.m2[at] = m2;
        } else {
#pragma unroll
            for (int i = 0; i < 2; i++) {
                float4* o4 = reinterpret_cast<float4*>(out.off + at + 4 * i);
                float4* m4 = reinterpret_cast<float4*>(out.m2 + at + 4 * i);
                const float4 ob = *o4, mb = *m4;
                float2 off[2], m2[2];
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    float2& kj = k[2 * i + j];
                    const float2 a = s1[2 * i + j];
                    off[j] = mul2(a, both(inv));
                    m2[j] = fma2(neg2(off[j]), a, s2[2 * i + j]);
                    m2[j].x = m2[j].x < 0.0f ? 0.0f : m2[j].x;
                    m2[j].y = m2[j].y < 0.0f ? 0.0f : m2[j].y;
                    if (before) {
                        const float2 o = j ? make_float2(ob.z, ob.w) : make_float2(ob.x, ob.y);
                        const float2 m = j ? make_float2(mb.z, mb.w) : make_float2(mb.x, mb.y);
                        const float2 d = sub2(off[j], o);
                        off[j] = fma2(d, both(f), o);
                        m2[j] = fma2(mul2(d, d), both(w), add2(m2[j], m));
                    }
                    if (!last) {
                        const float2 to = add2(kj, off[j]), moved = sub2(to, kj);
                        off[j] = add2(sub2(kj, sub2(to, moved)), sub2(off[j], moved));
                        kj = to;
                    }
                }
                if (last)
                    *reinterpret_cast<float4*>(out.k + at + 4 * i) = make_float4(
                        k[2 * i].x, k[2 * i].y, k[2 * i + 1].x, k[2 * i + 1].y);
                *o4 = make_float4(off[0].x, off[0].y, off[1].x, off[1].y);
                *m4 = make_float4(m2[0].x, m2[0].y, m2[1].x, m2[1].y);
            }
        }
#pragma unroll
        for (int i = 0; i < P; i++) s1[i] = s2[i] = both(0.0f);
        before = rows;
    };
    feed.down([&](uint32_t slot, int first) {
        if (first == 0 && feed.mine > 0) {
            const V8 v = unpack(shared_unit<T>(slot));
            if constexpr (kSame) {
                float2 m = both(0.0f);
#pragma unroll
                for (int i = 0; i < 4; i++) m = fma2(v.p[i], both(0.125f), m);
                k[0] = both(m.x + m.y);
            } else {
#pragma unroll
                for (int i = 0; i < P; i++) k[i] = v.p[i];
            }
        }
        // A thread that has rows has them all here: at most its last is missing.
        if (first && feed.mine > 0 &&
            (first % kRun == 0 || first == U || first == 4 * U || first == 16 * U))
            end_run(first, false);
        each_row<U>(feed.mine - first, [&](int j) {
            const V8 v = unpack(shared_unit<T>(slot + j * FwdRow<T>::kBytes * kThreads));
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float2 dv = sub2(v.p[i], k[kSame ? 0 : i]);
                s1[kSame ? 0 : i] = add2(s1[kSame ? 0 : i], dv);
                s2[kSame ? 0 : i] = fma2(dv, dv, s2[kSame ? 0 : i]);
            }
        });
    });
    end_run(feed.mine, true);
}

// Joins the cells [t0, t1) that lie in `sums` over all phases into the moments
// of the groups of d cells they belong to, a cell's row holding `per` values:
// f(group, count, moments) on one lane, for the part of the group inside. Rows
// are dealt to the phases in turn. A sub-warp takes a group: two passes, the
// mean of the cells' means about the first one, then the squares about it.
template <class F>
__device__ __forceinline__ void join_groups(const CellSums& sums, int phases, int rows, int t0,
                                            int t1, int d, int per, F&& f) {
    const int g_lo = t0 / d, groups = (t1 - 1) / d - g_lo + 1;
    int along = 1;  // lanes along a group's cells; the others share out the phases
    while (along < d && along < 32) along *= 2;
    int lanes = 32;
    while (lanes > along && groups * lanes > kThreads) lanes /= 2;
    const int lane = threadIdx.x % lanes, lc = lane % along, lp = lane / along;
    const int skip = lanes / along;
    // Phase p has `each` rows, and one more below `extra`. A phase without rows
    // has zeros in every cell and counts nothing.
    const int extra = rows % phases;
    const float each = (float)(rows / phases);
    for (int base = 0; base < groups; base += kThreads / lanes) {
        const int i = base + threadIdx.x / lanes, g = g_lo + i;
        const bool on = i < groups;
        const int c0 = on ? max(g * d, t0) - t0 : 0, c1 = on ? min(g * d + d, t1) - t0 : 0;
        const float k0 = on ? sums.k[c0] : 0.0f, total = (float)rows * (float)(c1 - c0);
        float a = 0.0f, q = 0.0f;
        for (int c = c0 + lc; c < c1; c += along) {
            const float *k = sums.k + c, *off = sums.off + c;
#pragma unroll 4
            for (int p = lp; p < phases; p += skip) {
                const float n = p < extra ? each + 1.0f : each;
                a = __fmaf_rn(n, (k[p * sums.width] - k0) + off[p * sums.width], a);
            }
        }
        for (int o = lanes / 2; o; o /= 2) a += __shfl_xor_sync(~0u, a, o);
        const float off0 = total > 0.0f ? a / total : 0.0f;
        for (int c = c0 + lc; c < c1; c += along) {
            const float *k = sums.k + c, *off = sums.off + c, *m2 = sums.m2 + c;
#pragma unroll 4
            for (int p = lp; p < phases; p += skip) {
                const float n = (float)per * (p < extra ? each + 1.0f : each);
                const float dv = (k[p * sums.width] - k0) + (off[p * sums.width] - off0);
                q += __fmaf_rn(n * dv, dv, m2[p * sums.width]);
            }
        }
        for (int o = lanes / 2; o; o /= 2) q += __shfl_xor_sync(~0u, q, o);
        if (on && lane == 0) f(g, total * (float)per, Moments{k0, off0, q});
    }
}

// Joins a group's moments over the cluster's blocks, which hold the chunks of a
// sample of len rows, all at the same place `own`: on the first of kCluster
// neighbouring lanes. Returns the count. Every lane calls it.
__device__ __forceinline__ float join_cluster(const Batch& B, const Moments* own, bool on, int len,
                                              Moments& q) {
    const int k = threadIdx.x % kCluster;
    float have = 0.0f;
    if (on && k < B.chunks) {
        int a, e;
        chunk_rows(len, B.chunks, k, a, e);
        have = (float)(e - a) * (float)B.d;
        q = {ld_cluster(&own->k, k), ld_cluster(&own->off, k), ld_cluster(&own->m2, k)};
    }
#pragma unroll
    for (int o = kCluster / 2; o; o /= 2) {
        const float more = __shfl_down_sync(~0u, have, o, kCluster);
        const Moments m = {__shfl_down_sync(~0u, q.k, o, kCluster),
                           __shfl_down_sync(~0u, q.off, o, kCluster),
                           __shfl_down_sync(~0u, q.m2, o, kCluster)};
        q = join(have, q, more, m);
        have += more;
    }
    return have;
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
    if constexpr (kSame) {
        r.v[0] = both(f(g));
    } else {
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
        for (int i = 0; i < 4; i++) r.v[i] = make_float2(v[2 * i], v[2 * i + 1]);
    }
    return r;
}

// ---- finishing rows, forward -----------------------------------------------------------

struct Stat {
    float mean, rstd;
};
// z = (x - mean)*scale + bias: the deviation first, so that it is exact where
// the group hardly varies. The mean is held negated.
template <bool kSame>
struct Affine {
    PerGroup<kSame> minus;
    V8 scale, bias;
};
template <bool kSame, class F>
__device__ __forceinline__ Affine<kSame> affine(const Batch& B, const V8& w, const V8& b, int first,
                                                int last, F&& stat) {
    Affine<kSame> a;
    a.minus = per_group<kSame>(first, last, B.d, [&](int g) { return -stat(g).mean; });
    const auto rstd = per_group<kSame>(first, last, B.d, [&](int g) { return stat(g).rstd; });
    a.bias = b;
#pragma unroll
    for (int i = 0; i < 4; i++) a.scale.p[i] = mul2(w.p[i], rstd[i]);
    return a;
}

// y (and the checkpoint) of the feed's rows of this thread's unit, last batch
// first; row0 is the first of the `phase_has` rows of its phase (a thread without
// a unit has rows too: its lane may write a block's scale).
template <class T, int AW, bool kSame, bool kKeep>
__device__ __forceinline__ void apply_rows(const Batch& B, Feed<FwdRow<T>, AW>& feed, int n,
                                           int row0, int phase_has, int unit, int cnt, bool on,
                                           const Affine<kSame>& q) {
    constexpr int U = FwdRow<T>::kRows, S = FwdRow<T>::kBytes * kThreads;
    const int64_t last = row0 + (int64_t)(feed.batches - 1) * U * B.phases;
    T* y = (T*)B.out + n * B.os + last * B.orow + unit * kUnit;
    const int64_t ystep = B.phases * B.orow;
    KeptAt kept;
    if (kKeep) kept = kept_at(B.kept, (int64_t)n * B.s + last, B.phases, unit);
    feed.up([&](uint32_t slot, int first) {
        Raw<T> raw[U] = {};
        bool live[U];
#pragma unroll
        for (int j = 0; j < U; j++) {
            live[j] = first + j < phase_has;
            if (kKeep && on && live[j]) raw[j] = shared_unit<T>(slot + j * S);
        }
        each_row<U>(feed.mine - first, [&](int j) {
            V8 v = unpack(kKeep ? raw[j] : shared_unit<T>(slot + j * S));
#pragma unroll
            for (int i = 0; i < 4; i++)
                v.p[i] = fma2(add2(v.p[i], q.minus[i]), q.scale.p[i], q.bias.p[i]);
            activate<sizeof(T) == 2>(v, B.act, B.param);
            Raw<T> o;
            pack(v, o);
            st_unit<T, AW>(y + j * ystep, o, cnt);
        });
        if (kKeep) {
            keep_units<T, AW, U>(raw, B.kept, kept, live, unit, cnt, on);
            kept.codes -= U * kept.codes_step;
            kept.scale -= U * kept.scale_step;
        }
        y -= U * ystep;
    });
}

// ---- forward in one launch: a cluster per slab of a sample -------------------------------

template <class T, int AW, bool kSame, bool kKeep>
__global__ void __launch_bounds__(kThreads, kBlocks) k_norm(Batch B) {
    constexpr int E = kSame ? 1 : 8;
    extern __shared__ uint4 dyn[];
    const int phase = threadIdx.x / B.tile, u = threadIdx.x % B.tile;
    const int rank = (int)cluster_rank();
    const int id = blockIdx.x / B.chunks, n = id / B.slabs, c0 = id % B.slabs * B.slab;
    const int cw = min(B.slab, B.c - c0), groups = cw / B.d, g0 = c0 / B.d;
    const int len = valid_rows(B, n);
    int r0, r1;
    chunk_rows(len, B.chunks, rank, r0, r1);
    const int unit = c0 / kUnit + u, cnt = min(kUnit, c0 + cw - unit * kUnit);
    const bool on = phase < B.phases && u * kUnit < cw;

    using Row = FwdRow<T>;
    const int most = (r1 - r0 + B.phases - 1) / B.phases;
    const Row rows(B, n, r0 + phase, unit);
    Feed<Row, AW> feed(B, rows, dyn, most, on ? phase_rows(B, r0, r1, phase) : 0, cnt);
    feed.start_down();
    const int places = B.keep + (B.keep_all ? 0 : B.ahead);
    float* sums_at = reinterpret_cast<float*>((char*)dyn + (int64_t)places * Row::kRows *
                                                              Row::kBytes * kThreads);
    const CellSums sums(sums_at, B.phases, B.tile * E, kSame);
    Moments* own = reinterpret_cast<Moments*>(sums_at + cell_floats(B.phases, B.tile * E, kSame));
    Stat* stat = reinterpret_cast<Stat*>(own + B.slab / B.d);

    if (phase < B.phases) sum_rows<T, AW, kSame>(feed, sums, phase, u);
    feed.start_up(rows);
    const V8 w = ld_params(on ? B.w : nullptr, B.ptype, unit * kUnit, cnt, 1.0f);
    const V8 b = ld_params(on ? B.b : nullptr, B.ptype, unit * kUnit, cnt, 0.0f);
    __syncthreads();
    join_groups(sums, B.phases, r1 - r0, 0, kSame ? cw / kUnit : cw, kSame ? B.d / kUnit : B.d,
                kSame ? kUnit : 1, [&](int g, float, Moments m) { own[g] = m; });
    if (B.chunks > 1) {
        cluster_arrive();
        cluster_wait();
    } else {
        __syncthreads();
    }
    // A group's blocks on neighbouring lanes, joined pairwise.
    for (int base = 0; base < groups; base += kThreads / kCluster) {
        const int g = base + threadIdx.x / kCluster, k = threadIdx.x % kCluster;
        Moments q = {0.0f, 0.0f, 0.0f};
        const float have = join_cluster(B, own + min(g, groups - 1), g < groups, len, q);
        if (g < groups && k == 0) {
            const float mu = len ? q.k + q.off : 0.0f, var = have > 0.0f ? q.m2 / have : 0.0f;
            const float rs = __fdiv_rn(1.0f, __fsqrt_rn(var + B.eps));
            stat[g] = {mu, rs};
            if (rank == 0) {
                const int64_t at = (int64_t)n * B.g + g0 + g;
                if (B.mean_out) B.mean_out[at] = mu;
                if (B.rstd_out) B.rstd_out[at] = rs;
            }
        }
    }
    cluster_arrive();  // the others' shared memory has been read
    __syncthreads();
    const int last = c0 + cw - 1;
    const auto q = affine<kSame>(B, w, b, min(unit * kUnit, last), last,
                                 [&](int g) { return stat[g - g0]; });
    apply_rows<T, AW, kSame, kKeep>(B, feed, n, r0 + phase, phase_rows(B, r0, r1, phase), unit, cnt,
                                    on, q);
    cluster_wait();
}

// ---- forward over chunks: moments, joined, then applied ---------------------------

template <class T, int AW, bool kSame>
__global__ void __launch_bounds__(kThreads, kBlocks) k_stats(Batch B, Moments* part) {
    constexpr int E = kSame ? 1 : 8;
    extern __shared__ uint4 dyn[];
    // A group that a tile's end cuts is carried to the next tile.
    __shared__ Moments carry[2];
    __shared__ float carried[2];
    using Row = FwdRow<T>;
    float* sums_at = reinterpret_cast<float*>((char*)dyn + (int64_t)B.ahead * Row::kRows *
                                                              Row::kBytes * kThreads);
    const CellSums sums(sums_at, B.phases, B.tile * E, kSame);
    const int n = blockIdx.x / B.chunks, k = blockIdx.x % B.chunks;
    int r0, r1;
    chunk_rows(valid_rows(B, n), B.chunks, k, r0, r1);
    Moments* o = part + ((int64_t)n * B.chunks + k) * B.g;
    const int phase = threadIdx.x / B.tile, u = threadIdx.x % B.tile;
    const int most = (r1 - r0 + B.phases - 1) / B.phases;
    const int cells = kSame ? B.c / kUnit : B.c, d = kSame ? B.d / kUnit : B.d;
    for (int t = 0; t < B.tiles; t++) {
        const int unit = t * B.tile + u, cnt = min(kUnit, B.c - unit * kUnit);
        const bool on = phase < B.phases && unit < B.units;
        Feed<Row, AW> feed(B, Row(B, n, r0 + phase, unit), dyn, most,
                           on ? phase_rows(B, r0, r1, phase) : 0, cnt);
        feed.start_down();
        if (phase < B.phases) sum_rows<T, AW, kSame>(feed, sums, phase, u);
        __syncthreads();
        if (t == B.tiles - 1) grid_release();
        const int t0 = t * B.tile * E, t1 = min(t0 + B.tile * E, cells), odd = t & 1;
        join_groups(sums, B.phases, r1 - r0, t0, t1, d, kSame ? kUnit : 1,
                    [&](int g, float count, Moments m) {
                        if (g * d < t0) {
                            m = join(carried[odd ^ 1], carry[odd ^ 1], count, m);
                            count += carried[odd ^ 1];
                        }
                        if (g * d + d > t1) {
                            carry[odd] = m;
                            carried[odd] = count;
                        } else {
                            o[g] = m;
                        }
                    });
        __syncthreads();
    }
}

// A block joins the chunks of up to `wide` groups of a sample: its threads take
// wide groups by kJoin/wide chunks at a time. In double, about the first
// chunk's mean, so one pass over the parts serves both moments.
constexpr int kJoin = 512;
__global__ void __launch_bounds__(kJoin)
    k_join(Batch B, const Moments* part, int wide, int blocks) {
    __shared__ double s1[kJoin], s2[kJoin];
    grid_wait();
    const int n = blockIdx.x / blocks, g = blockIdx.x % blocks * wide + threadIdx.x % wide;
    const int lane = threadIdx.x / wide, lanes = kJoin / wide;
    const int len = valid_rows(B, n), parts = B.chunks;
    const int64_t per = (len + parts - 1) / parts;
    double a = 0.0, q = 0.0, ref = 0.0;
    if (g < B.g) {
        const Moments* p = part + (int64_t)n * parts * B.g + g;
        ref = (double)p[0].k + p[0].off;
        for (int k = lane; k < parts; k += 4 * lanes) {
            Moments m[4];
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (k + j * lanes < parts) m[j] = p[(int64_t)(k + j * lanes) * B.g];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int64_t have = min(per, len - (k + j * lanes) * per);
                if (k + j * lanes < parts && have > 0) {
                    const double c = (double)have * B.d, dv = ((double)m[j].k - ref) + m[j].off;
                    a += c * dv;
                    q += m[j].m2 + c * dv * dv;
                }
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
__global__ void __launch_bounds__(kThreads, kBlocks) k_apply(Batch B) {
    extern __shared__ uint4 dyn[];
    const int id = gridDim.x - 1 - blockIdx.x, n = id / B.chunks;
    int r0, r1;
    chunk_rows(valid_rows(B, n), B.chunks, id % B.chunks, r0, r1);
    if (r0 >= r1) {
        grid_wait();
        return;
    }
    using Row = FwdRow<T>;
    const int phase = threadIdx.x / B.tile, u = threadIdx.x % B.tile;
    const int most = (r1 - r0 + B.phases - 1) / B.phases;
    const float *mu = B.mean_out + (int64_t)n * B.g, *rs = B.rstd_out + (int64_t)n * B.g;
    for (int t = 0; t < B.tiles; t++) {
        const int unit = t * B.tile + u, cnt = min(kUnit, B.c - unit * kUnit);
        const bool on = phase < B.phases && unit < B.units;
        const Row rows(B, n, r0 + phase, unit);
        Feed<Row, AW> feed(B, rows, dyn, most, on ? phase_rows(B, r0, r1, phase) : 0, cnt);
        feed.start_up(rows);
        const V8 w = ld_params(on ? B.w : nullptr, B.ptype, unit * kUnit, cnt, 1.0f);
        const V8 b = ld_params(on ? B.b : nullptr, B.ptype, unit * kUnit, cnt, 0.0f);
        // x and the parameters are the caller's; the statistics are the kernel
        // before's.
        if (t == 0) grid_wait();
        const auto q = affine<kSame>(B, w, b, min(unit * kUnit, B.c - 1), B.c - 1, [&](int g) {
            return Stat{mu[g], rs[g]};
        });
        apply_rows<T, AW, kSame, kKeep>(B, feed, n, r0 + phase, phase_rows(B, r0, r1, phase), unit,
                                        cnt, on, q);
    }
}

// ---- backward ---------------------------------------------------------------------

template <bool kSame>
struct BackParams {
    PerGroup<kSame> minus, rstd;  // the mean negated
    V8 w, b;
};
template <bool kSame>
__device__ __forceinline__ BackParams<kSame> back_params(const Batch& B, int n, int unit, int cnt,
                                                         bool on) {
    BackParams<kSame> q;
    const int first = min(unit * kUnit, B.c - 1);
    const float *mu = B.mean + (int64_t)n * B.g, *rs = B.rstd + (int64_t)n * B.g;
    q.minus = per_group<kSame>(first, B.c - 1, B.d, [&](int g) { return -__ldg(mu + g); });
    q.rstd = per_group<kSame>(first, B.c - 1, B.d, [&](int g) { return __ldg(rs + g); });
    q.w = ld_params(on ? B.w : nullptr, B.ptype, unit * kUnit, cnt, 1.0f);
    q.b = ld_params(on ? B.b : nullptr, B.ptype, unit * kUnit, cnt, 0.0f);
    return q;
}

// xh and dz = dy * act'(z) of the unit in a slot.
template <class T, bool kFrom, bool kSame>
__device__ __forceinline__ void slopes(const Batch& B, const BackParams<kSame>& q, uint32_t slot,
                                       V8& xh, V8& dz) {
    xh = BackRow<T, kFrom>::input(slot);
#pragma unroll
    for (int i = 0; i < 4; i++) xh.p[i] = mul2(add2(xh.p[i], q.minus[i]), q.rstd[i]);
    const V8 g = unpack(shared_unit<T>(slot));
    if (B.act == SIMTGO_ACT_NONE) {
        dz = g;
        return;
    }
    V8 z, f;
#pragma unroll
    for (int i = 0; i < 4; i++) z.p[i] = fma2(xh.p[i], q.w.p[i], q.b.p[i]);
    activate_slope<sizeof(T) == 2>(z, f, dz, B.act, B.param);
#pragma unroll
    for (int i = 0; i < 4; i++) dz.p[i] = mul2(dz.p[i], g.p[i]);
}

// A = sum dz and B = sum dz*xh of every channel over the phases, in shared memory.
struct ChannelSums {
    float *a, *b;      // of a phase
    float2 *half, *all;  // of some of the phases; of all
    int width;
    __device__ __forceinline__ ChannelSums(void* base, int phases, int channels)
        : width(channels + 4) {
        a = (float*)base;
        b = a + phases * width;
        half = reinterpret_cast<float2*>(b + phases * width);
        all = half + kThreads;
    }
};
__host__ __device__ constexpr int channel_bytes(int phases, int channels) {
    return 8 * phases * (channels + 4) + 8 * kThreads + 8 * channels;
}

// Sums the thread's rows and then the block's phases into sums.all. Every
// thread calls it; ends with a barrier.
template <class T, int AW, bool kFrom, bool kSame>
__device__ __forceinline__ void back_sums(const Batch& B, Feed<BackRow<T, kFrom>, AW>& feed,
                                          const BackParams<kSame>& q, const ChannelSums& sums,
                                          int phase, int u) {
    using Row = BackRow<T, kFrom>;
    const int channels = B.tile * kUnit;
    if (phase < B.phases) {
        float2 a[4] = {}, b[4] = {};
        const int at = phase * sums.width + u * kUnit;
        const auto flush = [&](bool first) {
#pragma unroll
            for (int i = 0; i < 2; i++) {
                if (first) {
                    *reinterpret_cast<float4*>(sums.a + at + 4 * i) =
                        make_float4(a[2 * i].x, a[2 * i].y, a[2 * i + 1].x, a[2 * i + 1].y);
                    *reinterpret_cast<float4*>(sums.b + at + 4 * i) =
                        make_float4(b[2 * i].x, b[2 * i].y, b[2 * i + 1].x, b[2 * i + 1].y);
                } else {
                    add4(sums.a + at + 4 * i, a[2 * i], a[2 * i + 1]);
                    add4(sums.b + at + 4 * i, b[2 * i], b[2 * i + 1]);
                }
            }
#pragma unroll
            for (int i = 0; i < 4; i++) a[i] = b[i] = both(0.0f);
        };
        bool flushed = false;
        feed.down([&](uint32_t slot, int first) {
            if (first && first % kRun == 0) {
                flush(!flushed);
                flushed = true;
            }
            each_row<Row::kRows>(feed.mine - first, [&](int j) {
                V8 xh, dz;
                slopes<T, kFrom>(B, q, slot + j * Row::kBytes * kThreads, xh, dz);
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    a[i] = add2(a[i], dz.p[i]);
                    b[i] = fma2(dz.p[i], xh.p[i], b[i]);
                }
            });
        });
        flush(!flushed);
    }
    __syncthreads();
    // Several threads to a channel where there are fewer channels than threads.
    const int split = max(1, min(kThreads / channels, B.phases));
    for (int i = threadIdx.x; i < split * channels; i += kThreads) {
        const int c = i % channels;
        float x = 0.0f, y = 0.0f;
#pragma unroll 4
        for (int p = i / channels; p < B.phases; p += split) {
            x += sums.a[p * sums.width + c];
            y += sums.b[p * sums.width + c];
        }
        (split > 1 ? sums.half : sums.all)[i] = make_float2(x, y);
    }
    __syncthreads();
    if (split > 1) {
        for (int c = threadIdx.x; c < channels; c += kThreads) {
            float2 v = sums.half[c];
            for (int k = 1; k < split; k++) {
                v.x += sums.half[k * channels + c].x;
                v.y += sums.half[k * channels + c].y;
            }
            sums.all[c] = v;
        }
        __syncthreads();
    }
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

// dx of the feed's rows of this thread's unit, last batch first, from the
// negated means s1 of dz*w and s2 of dz*w*xh.
template <class T, int AW, bool kFrom, bool kSame>
__device__ __forceinline__ void back_rows(const Batch& B, Feed<BackRow<T, kFrom>, AW>& feed,
                                          const BackParams<kSame>& q, const PerGroup<kSame>& s1,
                                          const PerGroup<kSame>& s2, int n, int row0, int unit,
                                          int cnt) {
    using Row = BackRow<T, kFrom>;
    const int64_t last = row0 + (int64_t)(feed.batches - 1) * Row::kRows * B.phases;
    T* dx = (T*)B.out + n * B.os + last * B.orow + unit * kUnit;
    const int64_t step = B.phases * B.orow;
    feed.up([&](uint32_t slot, int first) {
        each_row<Row::kRows>(feed.mine - first, [&](int j) {
            V8 xh, dz;
            slopes<T, kFrom>(B, q, slot + j * Row::kBytes * kThreads, xh, dz);
#pragma unroll
            for (int i = 0; i < 4; i++)
                dz.p[i] = mul2(q.rstd[i], fma2(xh.p[i], s2[i], fma2(dz.p[i], q.w.p[i], s1[i])));
            Raw<T> o;
            pack(dz, o);
            st_unit<T, AW>(dx + j * step, o, cnt);
        });
        dx -= Row::kRows * step;
    });
}

// One launch for dx: a cluster per slab of a sample. part, where wanted,
// receives every block's (A, B) of its channels, for k_back_join.
template <class T, int AW, bool kFrom, bool kSame>
__global__ void __launch_bounds__(kThreads, kBlocks) k_norm_back(Batch B, float2* part) {
    extern __shared__ uint4 dyn[];
    using Row = BackRow<T, kFrom>;
    const int phase = threadIdx.x / B.tile, u = threadIdx.x % B.tile;
    const int places = B.keep + (B.keep_all ? 0 : B.ahead);
    const ChannelSums sums((char*)dyn + (int64_t)places * Row::kRows * Row::kBytes * kThreads,
                           B.phases, B.tile * kUnit);
    float2* own = sums.all + B.tile * kUnit;  // this block's group sums
    float2* means = own + B.slab / B.d;       // the cluster's, over the count, negated

    const int rank = (int)cluster_rank();
    const int id = blockIdx.x / B.chunks, n = id / B.slabs, c0 = id % B.slabs * B.slab;
    const int cw = min(B.slab, B.c - c0), groups = cw / B.d, g0 = c0 / B.d;
    const int len = valid_rows(B, n);
    int r0, r1;
    chunk_rows(len, B.chunks, rank, r0, r1);
    const int unit = c0 / kUnit + u, cnt = min(kUnit, c0 + cw - unit * kUnit);
    const bool on = phase < B.phases && u * kUnit < cw;

    const int most = (r1 - r0 + B.phases - 1) / B.phases;
    const Row rows(B, n, r0 + phase, unit);
    Feed<Row, AW> feed(B, rows, dyn, most, on ? phase_rows(B, r0, r1, phase) : 0, cnt);
    feed.start_down();
    const BackParams<kSame> q = back_params<kSame>(B, n, unit, cnt, on);
    back_sums<T, AW, kFrom, kSame>(B, feed, q, sums, phase, u);
    if (B.out) feed.start_up(rows);
    if (part)
        for (int i = threadIdx.x; i < cw; i += kThreads)
            part[((int64_t)n * B.chunks + rank) * B.c + c0 + i] = sums.all[i];
    grid_release();
    if (!B.out) return;  // the same for every block of the grid
    group_sums(B, c0, groups, [&](int i) { return sums.all[i]; },
               [&](int g, float2 v) { own[g] = v; });
    cluster_arrive();
    cluster_wait();
    for (int base = 0; base < groups; base += kThreads / kCluster) {
        const int g = base + threadIdx.x / kCluster, k = threadIdx.x % kCluster;
        float x = 0.0f, y = 0.0f;
        if (g < groups && k < B.chunks) {
            x = ld_cluster(&own[g].x, k);
            y = ld_cluster(&own[g].y, k);
        }
#pragma unroll
        for (int o = kCluster / 2; o; o /= 2) {
            x += __shfl_down_sync(~0u, x, o, kCluster);
            y += __shfl_down_sync(~0u, y, o, kCluster);
        }
        const float inv = len ? -1.0f / ((float)len * (float)B.d) : 0.0f;
        if (g < groups && k == 0) means[g] = make_float2(x * inv, y * inv);
    }
    cluster_arrive();  // the others' shared memory has been read
    __syncthreads();
    if (on) {
        const int last = c0 + cw - 1, first = min(unit * kUnit, last);
        const auto s1 = per_group<kSame>(first, last, B.d, [&](int g) { return means[g - g0].x; });
        const auto s2 = per_group<kSame>(first, last, B.d, [&](int g) { return means[g - g0].y; });
        back_rows<T, AW, kFrom, kSame>(B, feed, q, s1, s2, n, r0 + phase, unit, cnt);
    }
    cluster_wait();
}

// Over chunks: (A, B) of every channel of a chunk.
template <class T, int AW, bool kFrom, bool kSame>
__global__ void __launch_bounds__(kThreads, kBlocks) k_back_stats(Batch B, float2* part) {
    extern __shared__ uint4 dyn[];
    using Row = BackRow<T, kFrom>;
    const ChannelSums sums((char*)dyn + (int64_t)B.ahead * Row::kRows * Row::kBytes * kThreads,
                           B.phases, B.tile * kUnit);
    const int n = blockIdx.x / B.chunks, k = blockIdx.x % B.chunks;
    int r0, r1;
    chunk_rows(valid_rows(B, n), B.chunks, k, r0, r1);
    float2* o = part + ((int64_t)n * B.chunks + k) * B.c;
    const int phase = threadIdx.x / B.tile, u = threadIdx.x % B.tile;
    const int most = (r1 - r0 + B.phases - 1) / B.phases;
    for (int t = 0; t < B.tiles; t++) {
        const int unit = t * B.tile + u, cnt = min(kUnit, B.c - unit * kUnit);
        const bool on = phase < B.phases && unit < B.units;
        Feed<Row, AW> feed(B, Row(B, n, r0 + phase, unit), dyn, most,
                           on ? phase_rows(B, r0, r1, phase) : 0, cnt);
        feed.start_down();
        const BackParams<kSame> q = back_params<kSame>(B, n, unit, cnt, on);
        back_sums<T, AW, kFrom, kSame>(B, feed, q, sums, phase, u);
        const int c0 = t * B.tile * kUnit;
        if (t == B.tiles - 1) grid_release();
        for (int i = threadIdx.x; i < min(B.tile * kUnit, B.c - c0); i += kThreads)
            o[c0 + i] = sums.all[i];
    }
}

// Adds `rows` rows of part, in double: channels 32*block and on, a block's warps
// taking the rows in turn. The first warp ends with the sums.
template <int kWarps>
__device__ __forceinline__ double2 add_rows(const float2* part, int64_t rows, int c, int block,
                                            double2 (*sm)[33]) {
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, ch = block * 32 + lane;
    double2 s = make_double2(0.0, 0.0);
    if (ch < c) {
#pragma unroll 4
        for (int64_t r = warp; r < rows; r += kWarps) {
            const float2 v = part[r * c + ch];
            s.x += v.x;
            s.y += v.y;
        }
    }
    sm[warp][lane] = s;
    __syncthreads();
    for (int h = kWarps / 2; h; h /= 2) {
        if (warp < h) {
            sm[warp][lane].x += sm[warp + h][lane].x;
            sm[warp][lane].y += sm[warp + h][lane].y;
        }
        __syncthreads();
    }
    return sm[warp][lane];
}

// For each of a number of spans of `rows` rows of part: their sum to
// tot[span][c], and to dbias and dweight where there is one span.
constexpr int kAdd = 512;
__global__ void __launch_bounds__(kAdd)
    k_back_join(const float2* part, int64_t rows, int c, int blocks, float2* tot, float* dw,
                float* db) {
    __shared__ double2 sm[kAdd / 32][33];
    grid_wait();
    const int64_t span = blockIdx.x / blocks;
    const int block = blockIdx.x % blocks, ch = block * 32 + threadIdx.x % 32;
    const double2 s = add_rows<kAdd / 32>(part + span * rows * c, rows, c, block, sm);
    grid_release();
    if (threadIdx.x < 32 && ch < c) {
        if (tot) tot[span * c + ch] = make_float2((float)s.x, (float)s.y);
        if (db) db[ch] = (float)s.x;
        if (dw) dw[ch] = (float)s.y;
    }
}

template <class T, int AW, bool kFrom, bool kSame>
__global__ void __launch_bounds__(kThreads, kBlocks)
    k_back_apply(Batch B, const float2* tot, float* dw, float* db) {
    extern __shared__ uint4 dyn[];
    // Blocks past the chunks add the samples' sums for dbias and dweight.
    const int chunks = B.n * B.chunks;
    if ((int)blockIdx.x >= chunks) {
        const int block = blockIdx.x - chunks, ch = block * 32 + threadIdx.x % 32;
        grid_wait();
        const double2 s = add_rows<kThreads / 32>(tot, B.n, B.c, block,
                                                  reinterpret_cast<double2(*)[33]>(dyn));
        if (threadIdx.x < 32 && ch < B.c) {
            if (db) db[ch] = (float)s.x;
            if (dw) dw[ch] = (float)s.y;
        }
        return;
    }
    using Row = BackRow<T, kFrom>;
    float2* means = reinterpret_cast<float2*>(  // of every group, negated
        (char*)dyn + (int64_t)B.ahead * Row::kRows * Row::kBytes * kThreads);
    const int phase = threadIdx.x / B.tile, u = threadIdx.x % B.tile;
    const int id = chunks - 1 - blockIdx.x, n = id / B.chunks;
    const int len = valid_rows(B, n);
    int r0, r1;
    chunk_rows(len, B.chunks, id % B.chunks, r0, r1);
    if (r0 >= r1) {
        grid_wait();
        return;
    }
    const int most = (r1 - r0 + B.phases - 1) / B.phases;
    for (int t = 0; t < B.tiles; t++) {
        const int unit = t * B.tile + u, cnt = min(kUnit, B.c - unit * kUnit);
        const bool on = phase < B.phases && unit < B.units;
        const Row rows(B, n, r0 + phase, unit);
        Feed<Row, AW> feed(B, rows, dyn, most, on ? phase_rows(B, r0, r1, phase) : 0, cnt);
        feed.start_up(rows);
        const BackParams<kSame> q = back_params<kSame>(B, n, unit, cnt, on);
        if (t == 0) {  // the rest is the caller's; the sums are the kernel before's
            grid_wait();
            const float inv = -1.0f / ((float)len * (float)B.d);
            group_sums(B, 0, B.g, [&](int i) { return tot[(int64_t)n * B.c + i]; },
                       [&](int g, float2 v) { means[g] = make_float2(v.x * inv, v.y * inv); });
            __syncthreads();
        }
        if (!on) continue;
        const int first = unit * kUnit;
        const auto s1 = per_group<kSame>(first, B.c - 1, B.d, [&](int g) { return means[g].x; });
        const auto s2 = per_group<kSame>(first, B.c - 1, B.d, [&](int g) { return means[g].y; });
        back_rows<T, AW, kFrom, kSame>(B, feed, q, s1, s2, n, r0 + phase, unit, cnt);
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
    Region r = {name, p, c.channels * e, nr * e, ns * e, 0, written, c.positions, c.samples};
    if (*rc || !p || !c.samples || !c.positions) return r;
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

// Lets a kernel have as much shared memory as a block may, once per device: the
// 48 KB that need no leave hold its static shared memory too, so that any
// dynamic size may be past them.
template <auto Kernel>
int allow_smem(const sg::DevInfo& d, size_t bytes) {
    static std::atomic<bool> done[64];
    if (!bytes || done[d.device & 63].load(std::memory_order_relaxed)) return 0;
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

// How a call goes through its data.
struct Plan {
    bool cluster;
    unsigned grid;
    size_t smem;
};
// What a kernel of the call needs: bytes of all inputs per element, rows of a
// batch and shared bytes of one, and the shared bytes beside the rows for a tile
// of so many units, phases and groups.
struct Needs {
    double elem;
    int rows;
    int64_t batch_bytes;
    size_t (*beside)(int tile, int phases, int groups, bool same);
    int per_sm;  // blocks an SM's registers hold
};
Plan make_plan(Batch& B, const simtgo_group_norm& c, const sg::DevInfo& d, bool keep_codes,
               const Needs& need) {
    B.n = c.samples;
    B.s = c.positions;
    B.c = c.channels;
    B.g = c.groups;
    B.d = c.channels / c.groups;
    B.ptype = c.param_type;
    B.act = c.act;
    B.param = c.act_param;
    B.eps = c.eps;
    const bool same = B.d % kUnit == 0;
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
        while (2 * slab <= std::min<int64_t>(c.channels, most) &&
               slab * c.positions * need.elem < 65536)
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
        const double bytes = (double)slab * c.positions * need.elem;
        int k = 1;
        while (k < kCluster && c.positions / (2 * k) >= t.phases &&
               (2 * k * clusters <= need.per_sm * d.sms || bytes / k > 96 * 1024))
            k *= 2;
        t.chunks = k;
        // A block gets through about 5.4 GB/s of its input; chunks, which fill
        // the GPU, through 1600 GB/s, after about 5 us more of launches and joins.
        // Clusters that fill it reach the same rate, and keep a call up to 8 GB.
        // Measured both ways (us, clusters and chunks): 8x4096x320 bf16 forward
        // 21 and 26, backward 31 and 34; 4x16384x512 bf16 forward with its
        // checkpoint 150 and 57, backward 81 and 75; 600x1000x96 bf16 forward 86
        // and 104, backward 180 and 151; 64x4096x1024 float32 forward 989 and 851;
        // above the limit 256x16384x1024 bf16 forward 4791 and 4364, backward 8295
        // and 8033, 130x16384x1024 float32 without an activation 6031 and 6892.
        const double us = bytes * clusters / (std::min<double>(clusters * k, need.per_sm * d.sms) * 5.4e3);
        const double chunked = bytes * clusters / 1.6e6 + 5.0;
        if (us <= chunked && clusters * k <= 0x7fffffff) {
            const size_t fixed = need.beside(t.tile, t.phases, (int)(slab / B.d), same);
            // The blocks that will share an SM, and their room in it.
            const int share = (int)std::max<int64_t>(
                1, std::min<int64_t>(need.per_sm, sg::ceil_div(clusters * k, d.sms)));
            const size_t room = std::min<size_t>(d.smem_per_sm / share - 1024,
                                                 d.max_smem_optin) - 64;
            const int per_block = (c.positions + k - 1) / k;
            const int64_t rows = (per_block + t.phases - 1) / t.phases;
            const int64_t batches = std::max<int64_t>(1, (rows + need.rows - 1) / need.rows);
            const int64_t fit = fixed < room ? (int64_t)((room - fixed) / need.batch_bytes) : 0;
            if (batches <= fit) {  // every row stays; all are asked for at once
                t.keep = (int)batches;
                t.ahead = batches > 4 ? 8 : batches > 2 ? 4 : batches > 1 ? 2 : 1;
                // No ring: its batches are never reached.
                p.smem = fixed + (size_t)batches * need.batch_bytes;
                t.keep_all = 1;
                p.cluster = true;
            } else if (fit >= 4) {
                t.ahead = fit >= 12 ? 4 : 2;
                t.keep = (int)(fit - t.ahead);
                t.keep_all = 0;
                p.smem = fixed + (size_t)fit * need.batch_bytes;
                p.cluster = true;
            }
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
    B.keep_all = 0;
    B.ahead = kAhead;
    // One wave of blocks, eight rows a thread at least.
    const int64_t rows = std::max<int64_t>(1, sg::ceil_div(B.s, 8 * B.phases));
    const int64_t wave = (int64_t)need.per_sm * d.sms / std::max(1, B.n);
    B.chunks = (int)std::max<int64_t>(1, std::min(rows, wave));
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
    const bool half = c.type != SIMTGO_F32;
    const int64_t batch_bytes = half ? FwdRow<__half>::kRows * FwdRow<__half>::kBytes * kThreads
                                     : FwdRow<float>::kRows * FwdRow<float>::kBytes * kThreads;
    const Needs need = {(double)e, half ? FwdRow<__half>::kRows : FwdRow<float>::kRows, batch_bytes,
                        [](int tile, int phases, int groups, bool same) {
                            return 4 * (size_t)cell_floats(phases, tile * (same ? 1 : kUnit), same) +
                                   groups * (sizeof(Moments) + sizeof(Stat));
                        },
                        kBlocks};
    const Plan p = make_plan(B, c, *d, kept, need);
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
            const size_t ring = (size_t)B.ahead * batch_bytes;
            const size_t smem =
                ring + 4 * (size_t)cell_floats(B.phases, B.tile * (S ? 1 : kUnit), S);
            if (int rc2 = launch<k_stats<T, AW, S>>(*d, p.grid, kThreads, smem, s, 1, false, B,
                                                    part))
                return rc2;
            // Few enough groups to a block that its threads take every chunk in
            // one round of four loads.
            int wide = std::min(32, ceil_pow2(c.groups));
            while (wide > 1 && 4 * (kJoin / wide) < B.chunks) wide /= 2;
            const int blocks = (c.groups + wide - 1) / wide;
            if (int rc2 = launch<k_join>(*d, (unsigned)c.samples * blocks, kJoin, 0, s, 1, true, B,
                                         (const Moments*)part, wide, blocks))
                return rc2;
            if (!elems) return 0;
            return launch<k_apply<T, AW, S, Q>>(*d, p.grid, kThreads, ring, s, 1, true, B);
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
    const bool half = c.type != SIMTGO_F32;
    const int back_rows_ = half ? BackRow<__half, true>::kRows : BackRow<float, true>::kRows;
    const int64_t batch_bytes =
        (int64_t)back_rows_ * kThreads *
        (half ? (from ? BackRow<__half, true>::kBytes : BackRow<__half, false>::kBytes)
              : (from ? BackRow<float, true>::kBytes : BackRow<float, false>::kBytes));
    const Needs need = {from ? e + 1.1 : 2.0 * e, back_rows_, batch_bytes,
                        [](int tile, int phases, int groups, bool) {
                            return (size_t)channel_bytes(phases, tile * kUnit) +
                                   groups * 2 * sizeof(float2);
                        },
                        kBlocks};
    const Plan p = make_plan(B, c, *d, false, need);
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
                const size_t smem = (size_t)B.ahead * batch_bytes +
                                    channel_bytes(B.phases, B.tile * kUnit);
                if (int r = launch<k_back_stats<T, AW, F, S>>(*d, p.grid, kThreads, smem, s, 1,
                                                              false, B, part))
                    return r;
            }
            const bool one = c.samples == 1;
            if (spans)
                if (int r = launch<k_back_join>(*d, add * c.samples, kAdd, 0, s, 1, true,
                                                (const float2*)part, (int64_t)B.chunks, c.channels,
                                                (int)add, tot, one ? dweight : nullptr,
                                                one ? dbias : nullptr))
                    return r;
            if (p.cluster || !dx) {
                if (!params) return 0;
                return launch<k_back_join>(*d, add, kAdd, 0, s, 1, true, (const float2*)part,
                                           (int64_t)c.samples * B.chunks, c.channels, (int)add,
                                           (float2*)nullptr, dweight, dbias);
            }
            // dbias and dweight that the sums of one sample did not give: added by
            // blocks of the last launch.
            const unsigned more = params && !(spans && one) ? add : 0;
            const size_t smem =
                std::max((size_t)B.ahead * batch_bytes + sizeof(float2) * (size_t)c.groups,
                         sizeof(double2) * 33 * (kThreads / 32));
            return launch<k_back_apply<T, AW, F, S>>(*d, p.grid + more, kThreads, smem, s, 1, true,
                                                     B, (const float2*)tot, dweight, dbias);
        };
        if (from) return same ? run(std::true_type(), std::true_type())
                              : run(std::true_type(), std::false_type());
        return same ? run(std::false_type(), std::true_type())
                    : run(std::false_type(), std::false_type());
    });
}

}  // extern "C"
