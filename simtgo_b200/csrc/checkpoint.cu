// checkpoint.cu -- the row-wise channels-last operators: the 8-bit checkpoint
// (Pack8, Unpack8) and the gated unit y = act(a)*b with its gradient, which
// writes and reads checkpoints on the way.
//
// Every element is read once and written once, so HBM binds all four. A
// thread owns one unit of eight channels and steps down the rows; the lanes
// that share a checkpoint block are neighbours (4 to 32 of them), so a block's
// largest magnitude is a few shuffles and the codes are written from the
// registers that held the values. Blocks take a tile of at most 256 units
// times a run of rows, many more than are resident, as in elementwise.cu.
//
// Measured on one B200 (6462 GB/s copied): 16384x4096 bf16 in blocks of 128
// packed in 31 us and restored in 30 us (6.5 TB/s both); an 8192x8192 bf16 gated
// unit with both inputs kept 84 us forward and 80 us backward from the kept
// codes (6.5 and 6.7 TB/s). Rows that cannot be walked flat cost more, for two reasons.
// A tile is a whole number of rows' units, so that from 129 to 255 units the rest
// of 256 threads idle (8192x1112 bf16, 139 units, packed in 11 us; 8192x2048 in
// 10). And rows off 16-byte boundaries are moved by words or single elements,
// codes by bytes (8192x1111 packed in 15 us and restored in 26, 1112 in 11 and 7,
// all from L2).
#include <algorithm>
#include <cmath>
#include <numeric>
#include <type_traits>

#include "channels.cuh"

namespace chan {

int check_type(const char* K, const char* name, int32_t type) {
    if (type < SIMTGO_F32 || type > SIMTGO_F16)
        return sg::fail(SIMTGO_EARG, "channels: %s: %s %d is none of SIMTGO_F32, _BF16, _F16", K,
                        name, type);
    return 0;
}
int check_act(const char* K, int32_t act, float param) {
    if (act < SIMTGO_ACT_NONE || act > SIMTGO_ACT_SOFTCLIP)
        return sg::fail(SIMTGO_EARG, "channels: %s: %d is no activation", K, act);
    if (act == SIMTGO_ACT_SOFTCLIP && !(param >= 0.0f && std::isfinite(param)))
        return sg::fail(SIMTGO_EARG, "channels: %s: a softclip threshold is finite and not "
                        "negative, got %g", K, param);
    return 0;
}
int check_block(const char* K, int32_t block) {
    if (block != 32 && block != 64 && block != 128 && block != 256)
        return sg::fail(SIMTGO_EARG, "channels: %s: a checkpoint block is 32, 64, 128 or 256 "
                        "channels, got %d", K, block);
    return 0;
}
int check_aligned(const char* K, const char* name, const void* p, int bytes) {
    if ((uintptr_t)p & (uintptr_t)(bytes - 1))
        return sg::fail(SIMTGO_EARG, "channels: %s: %s is not aligned to its %d-byte elements", K,
                        name, bytes);
    return 0;
}

// Largest whole number not above a/b, for b > 0.
static int64_t floor_div(int64_t a, int64_t b) { return a / b - (a % b < 0); }

// Whether a row of b, `off` bytes on, meets one of a, for regions of the same
// pitches and counts: rows i, j and i', j' meet where off + (i'-i) in + (j'-j) out
// lies in (-width, width), and `out` steps over a stretch of all `in` steps, so few
// differences come near zero.
static bool rows_meet(const Region& a, const Region& b, int64_t off) {
    const bool swap = a.pitch0 > a.pitch1;
    const int64_t in = swap ? a.pitch1 : a.pitch0, n_in = swap ? a.times1 : a.times0;
    const int64_t out = swap ? a.pitch0 : a.pitch1, n_out = swap ? a.times0 : a.times1;
    const int64_t j0 = out ? floor_div(-off, out) : 0;
    for (int64_t j = j0 - 1; j <= j0 + 2; j++) {
        if (j <= -n_out || j >= n_out) continue;
        const int64_t at = off + j * out, i0 = in ? floor_div(-at, in) : 0;
        for (int64_t i = i0; i <= i0 + 1; i++) {
            const int64_t k = std::max(1 - n_in, std::min(i, n_in - 1)), d = at + k * in;
            if (d > -b.width && d < a.width) return true;
        }
    }
    return false;
}

static bool may_meet(const Region& a, const Region& b) {
    const int64_t off = (int64_t)((uintptr_t)b.p - (uintptr_t)a.p);
    const int64_t in = std::min(a.pitch0, a.pitch1), out = std::max(a.pitch0, a.pitch1);
    const int64_t n_in = a.pitch0 > a.pitch1 ? a.times1 : a.times0;
    if (a.pitch0 == b.pitch0 && a.pitch1 == b.pitch1 && a.times0 == b.times0 &&
        a.times1 == b.times1 && (out == 0 || out >= (n_in - 1) * in + std::max(a.width, b.width)))
        return rows_meet(a, b, off);
    const int64_t period =
        std::gcd(std::gcd(a.pitch0, a.pitch1), std::gcd(b.pitch0, b.pitch1));
    if (period <= 0) return true;
    int64_t r = off % period;
    if (r < 0) r += period;
    return r < a.width || r + b.width > period;
}

int check_regions(const char* K, std::initializer_list<Region> regions) {
    for (const Region* a = regions.begin(); a != regions.end(); a++) {
        if (!a->p || a->bytes <= 0) continue;
        for (const Region* b = a + 1; b != regions.end(); b++) {
            if (!b->p || b->bytes <= 0 || (!a->written && !b->written)) continue;
            const uintptr_t pa = (uintptr_t)a->p, pb = (uintptr_t)b->p;
            if (pa >= pb + (uintptr_t)b->bytes || pb >= pa + (uintptr_t)a->bytes) continue;
            if (!may_meet(*a, *b)) continue;
            const Region &w = a->written ? *a : *b, &o = a->written ? *b : *a;
            return sg::fail(SIMTGO_EALIAS, "channels: %s: %s and %s were given overlapping device "
                            "memory, and the kernel writes through %s", K, w.name, o.name, w.name);
        }
    }
    return 0;
}

}  // namespace chan

using namespace chan;

namespace {

constexpr int kThreads = 256;
constexpr int kIters = 8;  // units a thread takes at most: 16 and 32 measured the same
// Rows of a backward step: as many as the registers hold beside the walk.
template <class T, bool kFlat>
constexpr int kRows = (sizeof(T) == 2 ? 4 : 2) / (kFlat ? 1 : 2);
constexpr int64_t kMaxElems = int64_t(1) << 46;  // keeps every byte offset far inside 64 bits

// How units fall on blocks. Rows of units: a tile of `tile` units by `phases`
// rows at a time, `iters` times down the rows. Where every matrix is contiguous
// and there is no checkpoint, or rows are whole blocks of it (flat), rows mean
// nothing: a block takes kThreads consecutive units, `iters` times, and no index
// needs a division or a product. The elements past the last whole unit, fewer
// than eight, are one more unit of the last block.
struct RowGrid {
    int64_t rows, units_total;
    int channels, units, lanes, tiles, tile, phases, iters;
    int shift;  // log2(units per checkpoint block)
    int nblk;   // checkpoint blocks per row
    int tail;
    bool flat;
};

RowGrid row_grid(int64_t rows, int channels, int block, bool contiguous, int sms) {
    RowGrid g;
    g.rows = rows;
    g.channels = channels;
    g.units = (int)sg::ceil_div(channels, kUnit);  // in 64 bits: any channels may come
    // Lanes that reduce one block together; a row shorter than a block takes
    // only as many as hold it.
    g.lanes = block ? std::min(block / kUnit, ceil_pow2(std::min(g.units, 32))) : 1;
    g.shift = 0;
    while (block && (kUnit << g.shift) < block) g.shift++;
    g.nblk = block ? (int)sg::ceil_div(channels, block) : 0;
    g.flat = contiguous && (!block || channels % block == 0);
    g.units_total = g.flat ? rows * channels / kUnit : 0;
    g.tail = g.flat ? (int)(rows * channels % kUnit) : 0;
    const int upad = (g.units + g.lanes - 1) / g.lanes * g.lanes;
    g.tiles = (upad + kThreads - 1) / kThreads;
    g.tile = ((upad + g.tiles - 1) / g.tiles + g.lanes - 1) / g.lanes * g.lanes;
    g.tiles = (upad + g.tile - 1) / g.tile;
    g.phases = kThreads / g.tile;
    // Eight units a thread where there is work for many blocks, fewer when
    // that would leave SMs idle.
    const int64_t groups =
        g.flat ? sg::ceil_div(g.units_total, kThreads) : sg::ceil_div(rows, g.phases) * g.tiles;
    g.iters = (int)std::max<int64_t>(1, std::min<int64_t>(kIters, groups / (sms * 8)));
    while (groups / g.iters > 0x7f000000) g.iters *= 2;  // a grid of blocks
    return g;
}
Kept kept(const RowGrid& g, int8_t* codes, float* scales) {
    return {codes, scales, g.channels, g.nblk, g.shift, g.lanes};
}
int64_t row_blocks(const RowGrid& g) {
    if (g.flat)
        return std::max<int64_t>(1, sg::ceil_div(g.units_total, (int64_t)kThreads * g.iters));
    return sg::ceil_div(g.rows, (int64_t)g.phases * g.iters) * g.tiles;
}

// This thread's unit, its first row and the number of its rows (phases apart);
// `most` is the block's largest such number, over which every thread loops so
// that shuffles find whole warps. `on` is false for threads beyond the tile's or
// the row's units. Flat: `row` is the thread's first unit, and the next ones lie
// kThreads units apart.
template <bool kFlat>
struct Place {
    int64_t row;
    int rows, most, unit, cnt, phases;
    bool on;
    __device__ __forceinline__ Place(const RowGrid& g) {
        if (kFlat) {
            const int64_t first = (int64_t)blockIdx.x * kThreads * g.iters;
            const int64_t left = g.units_total - first;
            most = (int)min((int64_t)g.iters, (left + kThreads - 1) / kThreads);
            const int64_t mine = left - threadIdx.x;
            rows = (int)min((int64_t)most, mine > 0 ? (mine + kThreads - 1) / kThreads : 0);
            row = first + threadIdx.x;
            unit = threadIdx.x & 31;  // a block's lanes are told by it
            cnt = kUnit;
            on = true;
            return;
        }
        const int tile = blockIdx.x % g.tiles, phase = threadIdx.x / g.tile;
        const int64_t row0 = (int64_t)(blockIdx.x / g.tiles) * g.phases * g.iters;
        const int left = (int)min((int64_t)g.phases * g.iters, g.rows - row0);
        row = row0 + phase;
        most = (left + g.phases - 1) / g.phases;
        rows = phase < g.phases ? (left - phase + g.phases - 1) / g.phases : 0;
        unit = tile * g.tile + threadIdx.x % g.tile;
        on = unit < g.units;
        cnt = min(kUnit, g.channels - unit * kUnit);
        phases = g.phases;
    }
};
// A thread's walk down one matrix: its unit in the first of its rows, and the
// elements to the next.
template <class T, bool kFlat>
struct Walk {
    T* at;
    int64_t apart;
    __device__ __forceinline__ Walk(T* base, int64_t pitch, const Place<kFlat>& p) {
        at = base + (kFlat ? p.row * kUnit : p.row * pitch + p.unit * kUnit);
        apart = kFlat ? 0 : p.phases * pitch;
    }
    __device__ __forceinline__ int64_t step() const { return kFlat ? kThreads * kUnit : apart; }
    __device__ __forceinline__ T* ahead(int u) const { return at + u * step(); }
    __device__ __forceinline__ void move(int u) { at += u * step(); }
};
// The same down a checkpoint.
template <bool kFlat>
struct KeptWalk {
    KeptAt at;
    __device__ __forceinline__ KeptWalk(const Kept& k, const Place<kFlat>& p) {
        if (kFlat)
            at = {k.codes + p.row * kUnit, k.scales + (p.row >> k.shift), kThreads * kUnit,
                  kThreads >> k.shift};
        else
            at = kept_at(k, p.row, p.phases, p.unit);
    }
    __device__ __forceinline__ void move(int u) {
        at.codes += u * (kFlat ? kThreads * kUnit : at.codes_step);
        at.scale += u * at.scale_step;
    }
};

// Largest magnitude by shuffles, codes from the same registers: one read of x,
// one write. Instructions (71 % of the issue slots) come close to HBM.
template <class T, int AW, bool kFlat>
__global__ void __launch_bounds__(kThreads)
    k_pack8(Kept kept, const T* __restrict__ x, int64_t pitch, RowGrid g) {
    constexpr int U = 4;
    const Place<kFlat> p(g);
    Walk<const T, kFlat> in(x, pitch, p);
    KeptWalk<kFlat> out(kept, p);
    for (int it = 0; it < p.most; it += U) {
        bool live[U];
        Raw<T> raw[U] = {};
#pragma unroll
        for (int u = 0; u < U; u++) {
            live[u] = it + u < p.rows;
            if (p.on && live[u]) raw[u] = ld_unit<T, AW>(in.ahead(u), p.cnt);
        }
        keep_units<T, AW, U, kFlat>(raw, kept, out.at, live, p.unit, p.cnt, p.on);
        in.move(U);
        out.move(U);
    }
}

// code * scale: HBM.
template <class T, int AW, bool kFlat>
__global__ void __launch_bounds__(kThreads)
    k_unpack8(T* __restrict__ x, Kept kept, int64_t pitch, RowGrid g) {
    constexpr int U = 4;
    const Place<kFlat> p(g);
    if (!p.on) return;
    Walk<T, kFlat> out(x, pitch, p);
    KeptWalk<kFlat> in(kept, p);
    for (int it = 0; it < p.rows; it += U) {
        Codes c[U];
        float s[U];
#pragma unroll
        for (int u = 0; u < U; u++)
            if (it + u < p.rows) {
                c[u] = ld_codes<AW == 16>(in.at.codes + u * in.at.codes_step, p.cnt);
                s[u] = __ldg(in.at.scale + u * in.at.scale_step);
            }
#pragma unroll
        for (int u = 0; u < U; u++)
            if (it + u < p.rows) {
                Raw<T> r;
                pack(decode(c[u], s[u]), r);
                st_unit<T, AW>(out.ahead(u), r, p.cnt);
            }
        in.move(U);
        out.move(U);
    }
}

// ---- the gated unit --------------------------------------------------------------

struct GatedArgs {
    void* y;
    const void *a, *b;
    Kept ka, kb;  // codes null: not kept
    int64_t a_pitch, b_pitch, y_pitch;
    int act;
    float param;
};

template <class T, bool kGate>
__device__ __forceinline__ Raw<T> gated_unit(const GatedArgs& k, const Raw<T>& a, const Raw<T>& b) {
    V8 v = unpack(a);
    activate<sizeof(T) == 2>(v, k.act, k.param);
    if (kGate) {
        const V8 w = unpack(b);
#pragma unroll
        for (int i = 0; i < 4; i++) v.p[i] = mul2(v.p[i], w.p[i]);
    }
    Raw<T> r;
    pack(v, r);
    return r;
}

// Four blocks an SM: the walk's eight registers a matrix fit beside 64 in all, and
// the warps hide the loads (8192x8192 bf16 with checkpoints: 84 us, 90 us at three
// blocks; packed float32 instructions, or issue would bound it).
template <class T, int AW, bool kFlat, bool kGate, bool kKeep>
__global__ void __launch_bounds__(kThreads, 4) k_gated(GatedArgs k, RowGrid g) {
    constexpr int U = sizeof(T) == 2 ? 4 : 2;
    if (kFlat && !kKeep && g.tail && blockIdx.x == gridDim.x - 1 && threadIdx.x == 0) {
        const int64_t at = g.units_total * kUnit;
        const Raw<T> a = ld_unit<T, AW>((const T*)k.a + at, g.tail);
        Raw<T> b = {};
        if (kGate) b = ld_unit<T, AW>((const T*)k.b + at, g.tail);
        st_unit<T, AW>((T*)k.y + at, gated_unit<T, kGate>(k, a, b), g.tail);
    }
    const Place<kFlat> p(g);
    Walk<const T, kFlat> a((const T*)k.a, k.a_pitch, p), b((const T*)k.b, k.b_pitch, p);
    Walk<T, kFlat> y((T*)k.y, k.y_pitch, p);
    KeptWalk<kFlat> ka(k.ka, p), kb(k.kb, p);
    for (int it = 0; it < p.most; it += U) {
        bool live[U];
        Raw<T> ra[U] = {}, rb[U] = {};
#pragma unroll
        for (int u = 0; u < U; u++) {
            live[u] = it + u < p.rows;
            if (p.on && live[u]) {
                ra[u] = ld_unit<T, AW>(a.ahead(u), p.cnt);
                if (kGate) rb[u] = ld_unit<T, AW>(b.ahead(u), p.cnt);
            }
        }
#pragma unroll
        for (int u = 0; u < U; u++)
            if (p.on && live[u])
                st_unit<T, AW>(y.ahead(u), gated_unit<T, kGate>(k, ra[u], rb[u]), p.cnt);
        if (kKeep) {
            if (k.ka.codes)
                keep_units<T, AW, U, kFlat>(ra, k.ka, ka.at, live, p.unit, p.cnt, p.on);
            if (kGate && k.kb.codes)
                keep_units<T, AW, U, kFlat>(rb, k.kb, kb.at, live, p.unit, p.cnt, p.on);
            ka.move(U);
            kb.move(U);
        }
        a.move(U);
        b.move(U);
        y.move(U);
    }
}

struct GatedBackArgs {
    void *da, *db;
    const void *dy, *a, *b;
    Kept ka, kb;
    int64_t a_pitch, b_pitch, y_pitch, da_pitch, db_pitch;
    int act;
    float param;
};

// A thread's walk down one input: the tensor, or its checkpoint.
template <class T, int AW, bool kFlat, bool kFrom>
struct Source {
    Walk<const T, kFlat> x;
    KeptWalk<kFlat> kept;
    __device__ __forceinline__ Source(const void* base, const Kept& k, int64_t pitch,
                                      const Place<kFlat>& p)
        : x((const T*)base, pitch, p), kept(k, p) {}
    struct Unit {
        Raw<T> raw;
        Codes codes;
        float scale;
        __device__ __forceinline__ V8 get() const {
            return kFrom ? decode(codes, scale) : unpack(raw);
        }
    };
    __device__ __forceinline__ void load(Unit& v, int u, int cnt) const {
        if (kFrom) {
            v.codes = ld_codes<AW == 16>(kept.at.codes + u * kept.at.codes_step, cnt);
            v.scale = __ldg(kept.at.scale + u * kept.at.scale_step);
        } else {
            v.raw = ld_unit<T, AW>(x.ahead(u), cnt);
        }
    }
    __device__ __forceinline__ void move(int u) {
        if (kFrom)
            kept.move(u);
        else
            x.move(u);
    }
};

template <class T, int AW, bool kGate>
__device__ __forceinline__ void gated_back_unit(const GatedBackArgs& k, const V8& a, const V8& b,
                                                const Raw<T>& dy, T* da, T* db, int cnt) {
    V8 f, s;
    activate_slope<sizeof(T) == 2>(a, f, s, k.act, k.param);
    const V8 d = unpack(dy);
    Raw<T> r;
    if (kGate && k.db) {
#pragma unroll
        for (int i = 0; i < 4; i++) f.p[i] = mul2(f.p[i], d.p[i]);
        pack(f, r);
        st_unit<T, AW>(db, r, cnt);
    }
    if (k.da) {
#pragma unroll
        for (int i = 0; i < 4; i++)
            s.p[i] = mul2(s.p[i], kGate ? mul2(d.p[i], b.p[i]) : d.p[i]);
        pack(s, r);
        st_unit<T, AW>(da, r, cnt);
    }
}

// Three blocks an SM with four rows in flight, or four with two where rows have
// pitches (8192x1112 bf16 halves of one buffer, forward and back: 51 us, 59 us the
// other way); 8192x8192 bf16 from checkpoints 80 us, 92 us at two blocks.
template <class T, int AW, bool kFlat, bool kFrom, bool kGate>
__global__ void __launch_bounds__(kThreads, kFlat ? 3 : 4)
    k_gated_back(GatedBackArgs k, RowGrid g) {
    constexpr int U = kRows<T, kFlat>;
    if (kFlat && !kFrom && g.tail && blockIdx.x == gridDim.x - 1 && threadIdx.x == 0) {
        const int64_t at = g.units_total * kUnit;
        const Raw<T> a = ld_unit<T, AW>((const T*)k.a + at, g.tail);
        Raw<T> b = {};
        if (kGate) b = ld_unit<T, AW>((const T*)k.b + at, g.tail);
        gated_back_unit<T, AW, kGate>(k, unpack(a), unpack(b),
                                      ld_unit<T, AW>((const T*)k.dy + at, g.tail), (T*)k.da + at,
                                      (T*)k.db + at, g.tail);
    }
    const Place<kFlat> p(g);
    if (!p.on) return;
    using In = Source<T, AW, kFlat, kFrom>;
    In sa(k.a, k.ka, k.a_pitch, p), sb(k.b, k.kb, k.b_pitch, p);
    Walk<const T, kFlat> y((const T*)k.dy, k.y_pitch, p);
    Walk<T, kFlat> oa((T*)k.da, k.da_pitch, p), ob((T*)k.db, k.db_pitch, p);
    for (int it = 0; it < p.rows; it += U) {
        typename In::Unit a[U], b[U];
        Raw<T> dy[U];
#pragma unroll
        for (int u = 0; u < U; u++)
            if (it + u < p.rows) {
                dy[u] = ld_unit<T, AW>(y.ahead(u), p.cnt);
                sa.load(a[u], u, p.cnt);
                if (kGate) sb.load(b[u], u, p.cnt);
            }
#pragma unroll
        for (int u = 0; u < U; u++)
            if (it + u < p.rows)
                gated_back_unit<T, AW, kGate>(k, a[u].get(), kGate ? b[u].get() : V8{}, dy[u],
                                              oa.ahead(u), ob.ahead(u), p.cnt);
        y.move(U);
        sa.move(U);
        sb.move(U);
        oa.move(U);
        ob.move(U);
    }
}

// ---- host ---------------------------------------------------------------------

int check_rows(const char* K, int64_t rows, int32_t channels, int32_t type) {
    if (rows < 0 || channels < 0)
        return sg::fail(SIMTGO_EARG, "channels: %s: negative rows or channels", K);
    if (int rc = check_type(K, "type", type)) return rc;
    if ((__int128)rows * channels > kMaxElems)
        return sg::fail(SIMTGO_ESIZE, "channels: %s: more than 2^46 elements", K);
    return 0;
}

// One matrix of the call: null and alignment, and a pitch that reads no
// element twice where it is written.
int check_matrix(const char* K, const char* name, const void* p, int64_t rows, int32_t channels,
                 int64_t pitch, int32_t type, bool written) {
    if (int rc = sg::check_ptr(K, name, p, rows * channels)) return rc;
    if (int rc = check_aligned(K, name, p, elem_size(type))) return rc;
    if (rows > 1 && (pitch < 0 || pitch > kMaxElems / rows))
        return sg::fail(SIMTGO_EARG, "channels: %s: %s has a row pitch of %lld elements", K, name,
                        (long long)pitch);
    if (written && rows > 1 && pitch < channels)
        return sg::fail(SIMTGO_EALIAS, "channels: %s: the rows of %s overlap (pitch %lld, %d "
                        "channels) and the kernel writes through it", K, name, (long long)pitch,
                        channels);
    return 0;
}
int check_codes(const char* K, const char* name, const void* codes, const void* scales,
                int32_t block) {
    if (!codes || !scales)
        return sg::fail(SIMTGO_ENULL, "channels: %s: the checkpoint %s needs both codes and scales",
                        K, name);
    if (int rc = check_block(K, block)) return rc;
    return check_aligned(K, name, scales, 4);
}

Region matrix(const char* name, const void* p, int64_t rows, int64_t pitch, int32_t channels,
              int32_t type, bool written) {
    const int64_t e = elem_size(type), apart = rows > 1 ? pitch * e : 0;
    return {name, p, channels * e, apart, 0, (rows - 1) * apart + channels * e, written, rows, 1};
}
int64_t n_scales(int64_t rows, int32_t channels, int32_t block) {
    return rows * ((channels + (int64_t)block - 1) / block);
}

// A unit's codes are moved eight bytes at a time only where they, and every
// row of them, start on such a boundary.
int with_codes(int width, int32_t channels, std::initializer_list<const void*> codes) {
    uintptr_t bits = 0;
    for (const void* c : codes) bits |= (uintptr_t)c;
    return width == 16 && (channels % kUnit || (bits & 7)) ? 4 : width;
}

}  // namespace

extern "C" {

int simtgo_Pack8(int8_t* codes, float* scales, const void* x, int32_t type, int64_t rows,
                 int32_t channels, int64_t row_pitch, int32_t block, void* stream) {
    const char* K = "Pack8";
    sg::clear_error();
    int rc;
    if ((rc = check_rows(K, rows, channels, type)) || (rc = check_block(K, block))) return rc;
    if (rows == 0 || channels == 0) return 0;
    if ((rc = check_codes(K, "of x", codes, scales, block)) ||
        (rc = check_matrix(K, "x", x, rows, channels, row_pitch, type, false)))
        return rc;
    if ((rc = check_regions(K, {solid("codes", codes, rows * channels, true),
                                solid("scales", scales, 4 * n_scales(rows, channels, block), true),
                                matrix("x", x, rows, row_pitch, channels, type, false)})))
        return rc;
    const sg::DevInfo* d;
    if ((rc = sg::current_device(&d))) return rc;
    const RowGrid g = row_grid(rows, channels, block, rows == 1 || row_pitch == channels, d->sms);
    const int64_t apart = g.flat || rows == 1 ? 0 : row_pitch;
    const int width = with_codes(access_width(type, {{x, apart, 0}}), channels, {codes});
    return by_type(type, width, [&](auto* t, auto w) {
        using T = std::remove_pointer_t<decltype(t)>;
        const auto kernel = g.flat ? k_pack8<T, decltype(w)::value, true>
                                   : k_pack8<T, decltype(w)::value, false>;
        sg::before_launch();
        kernel<<<(unsigned)row_blocks(g), kThreads, 0, (cudaStream_t)stream>>>(
                kept(g, codes, scales), (const T*)x, row_pitch, g);
        return sg::launch_status(K);
    });
}

int simtgo_Unpack8(void* x, const int8_t* codes, const float* scales, int32_t type, int64_t rows,
                   int32_t channels, int64_t row_pitch, int32_t block, void* stream) {
    const char* K = "Unpack8";
    sg::clear_error();
    int rc;
    if ((rc = check_rows(K, rows, channels, type)) || (rc = check_block(K, block))) return rc;
    if (rows == 0 || channels == 0) return 0;
    if ((rc = check_codes(K, "of x", codes, scales, block)) ||
        (rc = check_matrix(K, "x", x, rows, channels, row_pitch, type, true)))
        return rc;
    if ((rc = check_regions(K, {matrix("x", x, rows, row_pitch, channels, type, true),
                                solid("codes", codes, rows * channels, false),
                                solid("scales", scales, 4 * n_scales(rows, channels, block),
                                      false)})))
        return rc;
    const sg::DevInfo* d;
    if ((rc = sg::current_device(&d))) return rc;
    const RowGrid g = row_grid(rows, channels, block, rows == 1 || row_pitch == channels, d->sms);
    const int64_t apart = g.flat || rows == 1 ? 0 : row_pitch;
    const int width = with_codes(access_width(type, {{x, apart, 0}}), channels, {codes});
    return by_type(type, width, [&](auto* t, auto w) {
        using T = std::remove_pointer_t<decltype(t)>;
        const auto kernel = g.flat ? k_unpack8<T, decltype(w)::value, true>
                                   : k_unpack8<T, decltype(w)::value, false>;
        sg::before_launch();
        kernel<<<(unsigned)row_blocks(g), kThreads, 0, (cudaStream_t)stream>>>(
                (T*)x, kept(g, const_cast<int8_t*>(codes), const_cast<float*>(scales)), row_pitch,
                g);
        return sg::launch_status(K);
    });
}

int simtgo_Gated(void* y, const void* a, const void* b, int8_t* a_codes, float* a_scales,
                 int8_t* b_codes, float* b_scales, const simtgo_gated_unit* cfg, void* stream) {
    const char* K = "Gated";
    sg::clear_error();
    int rc;
    if (!cfg) return sg::fail(SIMTGO_ENULL, "channels: %s: no configuration", K);
    const simtgo_gated_unit c = *cfg;
    if ((rc = check_rows(K, c.rows, c.channels, c.type)) ||
        (rc = check_act(K, c.act, c.act_param)))
        return rc;
    const bool ka = a_codes || a_scales, kb = b_codes || b_scales;
    if ((ka || kb) && (rc = check_block(K, c.block))) return rc;
    if (kb && !b)
        return sg::fail(SIMTGO_EARG, "channels: %s: a checkpoint of b, but no b", K);
    if (c.rows == 0 || c.channels == 0) return 0;
    if ((ka && (rc = check_codes(K, "of a", a_codes, a_scales, c.block))) ||
        (kb && (rc = check_codes(K, "of b", b_codes, b_scales, c.block))) ||
        (rc = check_matrix(K, "y", y, c.rows, c.channels, c.y_pitch, c.type, true)) ||
        (rc = check_matrix(K, "a", a, c.rows, c.channels, c.a_pitch, c.type, false)) ||
        (b && (rc = check_matrix(K, "b", b, c.rows, c.channels, c.b_pitch, c.type, false))))
        return rc;
    const int64_t ns = ka || kb ? 4 * n_scales(c.rows, c.channels, c.block) : 0;
    if ((rc = check_regions(K, {matrix("y", y, c.rows, c.y_pitch, c.channels, c.type, true),
                                matrix("a", a, c.rows, c.a_pitch, c.channels, c.type, false),
                                matrix("b", b, c.rows, c.b_pitch, c.channels, c.type, false),
                                solid("a_codes", a_codes, c.rows * c.channels, true),
                                solid("a_scales", a_scales, ns, true),
                                solid("b_codes", b_codes, c.rows * c.channels, true),
                                solid("b_scales", b_scales, ns, true)})))
        return rc;
    const sg::DevInfo* d;
    if ((rc = sg::current_device(&d))) return rc;
    const bool solid_rows = c.rows == 1 || (c.a_pitch == c.channels && c.y_pitch == c.channels &&
                                            (!b || c.b_pitch == c.channels));
    const RowGrid g = row_grid(c.rows, c.channels, ka || kb ? c.block : 0, solid_rows, d->sms);
    const int m = c.rows > 1 && !g.flat;
    int width = access_width(c.type, {{y, m * c.y_pitch, 0}, {a, m * c.a_pitch, 0},
                                      {b, m * c.b_pitch, 0}});
    if (ka || kb) width = with_codes(width, c.channels, {a_codes, b_codes});
    const GatedArgs k = {y, a, b, kept(g, a_codes, a_scales), kept(g, b_codes, b_scales),
                         c.a_pitch, c.b_pitch, c.y_pitch, c.act, c.act_param};
    return by_type(c.type, width, [&](auto* t, auto w) {
        using T = std::remove_pointer_t<decltype(t)>;
        constexpr int AW = decltype(w)::value;
        const auto pick = [&](auto flat) {
            constexpr bool F = decltype(flat)::value;
            return b ? (ka || kb ? k_gated<T, AW, F, true, true> : k_gated<T, AW, F, true, false>)
                     : (ka ? k_gated<T, AW, F, false, true> : k_gated<T, AW, F, false, false>);
        };
        const auto kernel = g.flat ? pick(std::true_type()) : pick(std::false_type());
        sg::before_launch();
        kernel<<<(unsigned)row_blocks(g), kThreads, 0, (cudaStream_t)stream>>>(k, g);
        return sg::launch_status(K);
    });
}

int simtgo_Gated_backward(void* da, void* db, const void* dy, const void* a, const void* b,
                          const int8_t* a_codes, const float* a_scales, const int8_t* b_codes,
                          const float* b_scales, const simtgo_gated_unit* cfg, void* stream) {
    const char* K = "Gated_backward";
    sg::clear_error();
    int rc;
    if (!cfg) return sg::fail(SIMTGO_ENULL, "channels: %s: no configuration", K);
    const simtgo_gated_unit c = *cfg;
    if ((rc = check_rows(K, c.rows, c.channels, c.type)) ||
        (rc = check_act(K, c.act, c.act_param)))
        return rc;
    if (c.rows == 0 || c.channels == 0 || (!da && !db)) return 0;
    const bool from = a_codes || a_scales, gate = b || b_codes || b_scales;
    if (from == (a != nullptr))
        return sg::fail(SIMTGO_EARG, "channels: %s: a comes from exactly one of the tensor and its "
                        "checkpoint", K);
    if (gate && (from == (b != nullptr) || from != (b_codes || b_scales)))
        return sg::fail(SIMTGO_EARG, "channels: %s: b comes from the same kind of source as a", K);
    if (db && !gate) return sg::fail(SIMTGO_EARG, "channels: %s: db, but no b", K);
    if ((from && (rc = check_codes(K, "of a", a_codes, a_scales, c.block))) ||
        (from && gate && (rc = check_codes(K, "of b", b_codes, b_scales, c.block))) ||
        (rc = check_matrix(K, "dy", dy, c.rows, c.channels, c.y_pitch, c.type, false)) ||
        (a && (rc = check_matrix(K, "a", a, c.rows, c.channels, c.a_pitch, c.type, false))) ||
        (b && (rc = check_matrix(K, "b", b, c.rows, c.channels, c.b_pitch, c.type, false))) ||
        (da && (rc = check_matrix(K, "da", da, c.rows, c.channels, c.da_pitch, c.type, true))) ||
        (db && (rc = check_matrix(K, "db", db, c.rows, c.channels, c.db_pitch, c.type, true))))
        return rc;
    const int64_t ns = from ? 4 * n_scales(c.rows, c.channels, c.block) : 0;
    if ((rc = check_regions(K, {matrix("dy", dy, c.rows, c.y_pitch, c.channels, c.type, false),
                                matrix("a", a, c.rows, c.a_pitch, c.channels, c.type, false),
                                matrix("b", b, c.rows, c.b_pitch, c.channels, c.type, false),
                                solid("a_codes", a_codes, c.rows * c.channels, false),
                                solid("a_scales", a_scales, ns, false),
                                solid("b_codes", b_codes, c.rows * c.channels, false),
                                solid("b_scales", b_scales, ns, false),
                                matrix("da", da, c.rows, c.da_pitch, c.channels, c.type, true),
                                matrix("db", db, c.rows, c.db_pitch, c.channels, c.type, true)})))
        return rc;
    const sg::DevInfo* d;
    if ((rc = sg::current_device(&d))) return rc;
    const bool solid_rows =
        c.rows == 1 || (c.y_pitch == c.channels && (!a || c.a_pitch == c.channels) &&
                        (!b || c.b_pitch == c.channels) && (!da || c.da_pitch == c.channels) &&
                        (!db || c.db_pitch == c.channels));
    const RowGrid g = row_grid(c.rows, c.channels, from ? c.block : 0, solid_rows, d->sms);
    const int m = c.rows > 1 && !g.flat;
    int width = access_width(c.type, {{dy, m * c.y_pitch, 0}, {a, m * c.a_pitch, 0},
                                      {b, m * c.b_pitch, 0}, {da, m * c.da_pitch, 0},
                                      {db, m * c.db_pitch, 0}});
    if (from) width = with_codes(width, c.channels, {a_codes, b_codes});
    const GatedBackArgs k = {da, db, dy, a, b,
                             kept(g, const_cast<int8_t*>(a_codes), const_cast<float*>(a_scales)),
                             kept(g, const_cast<int8_t*>(b_codes), const_cast<float*>(b_scales)),
                             c.a_pitch, c.b_pitch, c.y_pitch, c.da_pitch, c.db_pitch,
                             c.act, c.act_param};
    return by_type(c.type, width, [&](auto* t, auto w) {
        using T = std::remove_pointer_t<decltype(t)>;
        constexpr int AW = decltype(w)::value;
        const auto pick = [&](auto flat) {
            constexpr bool F = decltype(flat)::value;
            return from ? (gate ? k_gated_back<T, AW, F, true, true>
                                : k_gated_back<T, AW, F, true, false>)
                        : (gate ? k_gated_back<T, AW, F, false, true>
                                : k_gated_back<T, AW, F, false, false>);
        };
        const auto kernel = g.flat ? pick(std::true_type()) : pick(std::false_type());
        sg::before_launch();
        kernel<<<(unsigned)row_blocks(g), kThreads, 0, (cudaStream_t)stream>>>(k, g);
        return sg::launch_status(K);
    });
}

}  // extern "C"
