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

int check_regions(const char* K, std::initializer_list<Region> regions) {
    for (const Region* a = regions.begin(); a != regions.end(); a++) {
        if (!a->p || a->bytes <= 0) continue;
        for (const Region* b = a + 1; b != regions.end(); b++) {
            if (!b->p || b->bytes <= 0 || (!a->written && !b->written)) continue;
            const uintptr_t pa = (uintptr_t)a->p, pb = (uintptr_t)b->p;
            if (pa >= pb + (uintptr_t)b->bytes || pb >= pa + (uintptr_t)a->bytes) continue;
            const int64_t period = std::gcd(std::gcd(a->pitch0, a->pitch1),
                                            std::gcd(b->pitch0, b->pitch1));
            if (period > 0) {
                int64_t off = (int64_t)(pb - pa) % period;
                if (off < 0) off += period;
                if (off >= a->width && off + b->width <= period) continue;
            }
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
constexpr int64_t kMaxElems = int64_t(1) << 46;  // keeps every byte offset far inside 64 bits

// How rows of units fall on blocks: a tile of `tile` units by `phases` rows
// at a time, `iters` times down the rows.
struct RowGrid {
    int64_t rows;
    int channels, units, lanes, tiles, tile, phases, iters;
    int shift;  // log2(units per checkpoint block)
    int nblk;   // checkpoint blocks per row
};

RowGrid row_grid(int64_t rows, int channels, int block, int sms) {
    RowGrid g;
    g.rows = rows;
    g.channels = channels;
    g.units = (channels + kUnit - 1) / kUnit;
    // Lanes that reduce one block together; a row shorter than a block takes
    // only as many as hold it.
    g.lanes = block ? std::min(block / kUnit, ceil_pow2(std::min(g.units, 32))) : 1;
    g.shift = 0;
    while (block && (kUnit << g.shift) < block) g.shift++;
    g.nblk = block ? (channels + block - 1) / block : 0;
    const int upad = (g.units + g.lanes - 1) / g.lanes * g.lanes;
    g.tiles = (upad + kThreads - 1) / kThreads;
    g.tile = ((upad + g.tiles - 1) / g.tiles + g.lanes - 1) / g.lanes * g.lanes;
    g.tiles = (upad + g.tile - 1) / g.tile;
    g.phases = kThreads / g.tile;
    // Eight rows a thread where there is work for many blocks, fewer when
    // that would leave SMs idle.
    const int64_t groups = sg::ceil_div(rows, g.phases) * g.tiles;
    g.iters = (int)std::max<int64_t>(1, std::min<int64_t>(8, groups / (sms * 8)));
    while (sg::ceil_div(rows, (int64_t)g.phases * g.iters) * g.tiles > 0x7fffffff) g.iters *= 2;
    return g;
}
Kept kept(const RowGrid& g, int8_t* codes, float* scales) {
    return {codes, scales, g.channels, g.nblk, g.shift, g.lanes};
}
int64_t row_blocks(const RowGrid& g) {
    return sg::ceil_div(g.rows, (int64_t)g.phases * g.iters) * g.tiles;
}

// This thread's unit and first row. `on` is false for threads beyond the
// tile's or the row's units; they still take part in shuffles.
struct Place {
    int64_t row0, end;  // block's first row and one past its last
    int phase, unit, cnt;
    bool on;
};
__device__ __forceinline__ Place place(const RowGrid& g) {
    Place p;
    const int tile = blockIdx.x % g.tiles;
    p.row0 = (int64_t)(blockIdx.x / g.tiles) * g.phases * g.iters;
    p.end = min(p.row0 + (int64_t)g.phases * g.iters, g.rows);
    p.phase = threadIdx.x / g.tile;
    p.unit = tile * g.tile + threadIdx.x % g.tile;
    p.on = p.phase < g.phases && p.unit < g.units;
    p.cnt = min(kUnit, g.channels - p.unit * kUnit);
    return p;
}

// The rows of one step of a thread's loop: row0 + u*phases for u < U.
template <int U>
__device__ __forceinline__ void live_rows(const RowGrid& g, const Place& p, int64_t row,
                                          bool (&live)[U]) {
#pragma unroll
    for (int u = 0; u < U; u++)
        live[u] = p.phase < g.phases && row + (int64_t)u * g.phases < p.end;
}

template <class T, int AW>
__global__ void __launch_bounds__(kThreads)
    k_pack8(Kept kept, const T* __restrict__ x, int64_t pitch, RowGrid g) {
    constexpr int U = 4;
    const Place p = place(g);
    const T* at = x + p.unit * kUnit;
    for (int64_t row = p.row0 + p.phase; row - p.phase < p.end; row += (int64_t)U * g.phases) {
        bool live[U];
        live_rows<U>(g, p, row, live);
        Raw<T> raw[U] = {};
#pragma unroll
        for (int u = 0; u < U; u++)
            if (p.on && live[u])
                raw[u] = ld_unit<T, AW>(at + (row + (int64_t)u * g.phases) * pitch, p.cnt);
        keep_units<T, AW, U>(raw, kept, row, g.phases, live, p.unit, p.cnt, p.on);
    }
}

template <class T, int AW>
__global__ void __launch_bounds__(kThreads)
    k_unpack8(T* __restrict__ x, const int8_t* __restrict__ codes,
              const float* __restrict__ scales, int64_t pitch, RowGrid g) {
    constexpr int U = 4;
    const Place p = place(g);
    if (!p.on) return;
    for (int64_t base = p.row0 + p.phase; base < p.end; base += (int64_t)U * g.phases) {
        Codes c[U];
        float s[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int64_t row = base + (int64_t)u * g.phases;
            if (row < p.end) {
                c[u] = ld_codes<AW == 16>(codes + row * g.channels + p.unit * kUnit, p.cnt);
                s[u] = __ldg(scales + row * g.nblk + (p.unit >> g.shift));
            }
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int64_t row = base + (int64_t)u * g.phases;
            if (row < p.end) {
                Raw<T> r;
                pack(decode(c[u], s[u]), r);
                st_unit<T, AW>(x + row * pitch + p.unit * kUnit, r, p.cnt);
            }
        }
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

template <class T, int AW, bool kGate, bool kKeep>
__global__ void __launch_bounds__(kThreads) k_gated(GatedArgs k, RowGrid g) {
    constexpr int U = sizeof(T) == 2 ? 4 : 2;
    const Place p = place(g);
    const T* a = (const T*)k.a + p.unit * kUnit;
    const T* b = (const T*)k.b + p.unit * kUnit;
    T* y = (T*)k.y + p.unit * kUnit;
    for (int64_t row = p.row0 + p.phase; row - p.phase < p.end; row += (int64_t)U * g.phases) {
        bool live[U];
        live_rows<U>(g, p, row, live);
        Raw<T> ra[U] = {}, rb[U] = {};
#pragma unroll
        for (int u = 0; u < U; u++)
            if (p.on && live[u]) {
                const int64_t at = row + (int64_t)u * g.phases;
                ra[u] = ld_unit<T, AW>(a + at * k.a_pitch, p.cnt);
                if (kGate) rb[u] = ld_unit<T, AW>(b + at * k.b_pitch, p.cnt);
            }
#pragma unroll
        for (int u = 0; u < U; u++)
            if (p.on && live[u]) {
                V8 v = unpack(ra[u]);
                activate<sizeof(T) == 2>(v, k.act, k.param);
                if (kGate) {
                    const V8 w = unpack(rb[u]);
#pragma unroll
                    for (int i = 0; i < 4; i++) v.p[i] = mul2(v.p[i], w.p[i]);
                }
                Raw<T> r;
                pack(v, r);
                st_unit<T, AW>(y + (row + (int64_t)u * g.phases) * k.y_pitch, r, p.cnt);
            }
        if (kKeep) {
            if (k.ka.codes)
                keep_units<T, AW, U>(ra, k.ka, row, g.phases, live, p.unit, p.cnt, p.on);
            if (kGate && k.kb.codes)
                keep_units<T, AW, U>(rb, k.kb, row, g.phases, live, p.unit, p.cnt, p.on);
        }
    }
}

struct GatedBackArgs {
    void *da, *db;
    const void *dy, *a, *b;
    const int8_t *a_codes, *b_codes;
    const float *a_scales, *b_scales;
    int64_t a_pitch, b_pitch, y_pitch, da_pitch, db_pitch;
    int act;
    float param;
};

// A unit of an input, from the tensor or from its checkpoint.
template <class T, int AW, bool kFrom>
struct Source {
    Raw<T> raw;
    Codes codes;
    float scale;
    __device__ __forceinline__ void load(const T* x, const int8_t* c, const float* s, int64_t pitch,
                                         const RowGrid& g, const Place& p, int64_t row) {
        if (kFrom) {
            codes = ld_codes<AW == 16>(c + row * g.channels + p.unit * kUnit, p.cnt);
            scale = __ldg(s + row * g.nblk + (p.unit >> g.shift));
        } else {
            raw = ld_unit<T, AW>(x + row * pitch + p.unit * kUnit, p.cnt);
        }
    }
    __device__ __forceinline__ V8 get() const { return kFrom ? decode(codes, scale) : unpack(raw); }
};

template <class T, int AW, bool kFrom, bool kGate>
__global__ void __launch_bounds__(kThreads) k_gated_back(GatedBackArgs k, RowGrid g) {
    constexpr int U = sizeof(T) == 2 ? 4 : 2;
    const Place p = place(g);
    if (!p.on) return;
    for (int64_t base = p.row0 + p.phase; base < p.end; base += (int64_t)U * g.phases) {
        Source<T, AW, kFrom> a[U], b[U];
        Raw<T> dy[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int64_t row = base + (int64_t)u * g.phases;
            if (row < p.end) {
                dy[u] = ld_unit<T, AW>((const T*)k.dy + row * k.y_pitch + p.unit * kUnit, p.cnt);
                a[u].load((const T*)k.a, k.a_codes, k.a_scales, k.a_pitch, g, p, row);
                if (kGate) b[u].load((const T*)k.b, k.b_codes, k.b_scales, k.b_pitch, g, p, row);
            }
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int64_t row = base + (int64_t)u * g.phases;
            if (row < p.end) {
                V8 f, s;
                activate_slope<sizeof(T) == 2>(a[u].get(), f, s, k.act, k.param);
                const V8 d = unpack(dy[u]);
                Raw<T> r;
                if (kGate && k.db) {
#pragma unroll
                    for (int i = 0; i < 4; i++) f.p[i] = mul2(f.p[i], d.p[i]);
                    pack(f, r);
                    st_unit<T, AW>((T*)k.db + row * k.db_pitch + p.unit * kUnit, r, p.cnt);
                }
                if (k.da) {
                    V8 w = d;
                    if (kGate) {
                        const V8 gate = b[u].get();
#pragma unroll
                        for (int i = 0; i < 4; i++) w.p[i] = mul2(w.p[i], gate.p[i]);
                    }
#pragma unroll
                    for (int i = 0; i < 4; i++) s.p[i] = mul2(s.p[i], w.p[i]);
                    pack(s, r);
                    st_unit<T, AW>((T*)k.da + row * k.da_pitch + p.unit * kUnit, r, p.cnt);
                }
            }
        }
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
    return {name, p, channels * e, apart, 0, (rows - 1) * apart + channels * e, written};
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
    const RowGrid g = row_grid(rows, channels, block, d->sms);
    const int width =
        with_codes(access_width(type, {{x, rows > 1 ? row_pitch : 0, 0}}), channels, {codes});
    return by_type(type, width, [&](auto* t, auto w) {
        using T = std::remove_pointer_t<decltype(t)>;
        sg::before_launch();
        k_pack8<T, decltype(w)::value>
            <<<(unsigned)row_blocks(g), kThreads, 0, (cudaStream_t)stream>>>(
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
    RowGrid g = row_grid(rows, channels, block, d->sms);
    const int width =
        with_codes(access_width(type, {{x, rows > 1 ? row_pitch : 0, 0}}), channels, {codes});
    return by_type(type, width, [&](auto* t, auto w) {
        using T = std::remove_pointer_t<decltype(t)>;
        sg::before_launch();
        k_unpack8<T, decltype(w)::value><<<(unsigned)row_blocks(g), kThreads, 0,
                                           (cudaStream_t)stream>>>((T*)x, codes, scales, row_pitch,
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
    const RowGrid g = row_grid(c.rows, c.channels, ka || kb ? c.block : 0, d->sms);
    const int m = c.rows > 1;
    int width = access_width(c.type, {{y, m * c.y_pitch, 0}, {a, m * c.a_pitch, 0},
                                      {b, m * c.b_pitch, 0}});
    if (ka || kb) width = with_codes(width, c.channels, {a_codes, b_codes});
    const GatedArgs k = {y, a, b, kept(g, a_codes, a_scales), kept(g, b_codes, b_scales),
                         c.a_pitch, c.b_pitch, c.y_pitch, c.act, c.act_param};
    return by_type(c.type, width, [&](auto* t, auto w) {
        using T = std::remove_pointer_t<decltype(t)>;
        constexpr int AW = decltype(w)::value;
        const auto kernel = b ? (ka || kb ? k_gated<T, AW, true, true> : k_gated<T, AW, true, false>)
                              : (ka ? k_gated<T, AW, false, true> : k_gated<T, AW, false, false>);
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
    const RowGrid g = row_grid(c.rows, c.channels, from ? c.block : 0, d->sms);
    const int m = c.rows > 1;
    int width = access_width(c.type, {{dy, m * c.y_pitch, 0}, {a, m * c.a_pitch, 0},
                                      {b, m * c.b_pitch, 0}, {da, m * c.da_pitch, 0},
                                      {db, m * c.db_pitch, 0}});
    if (from) width = with_codes(width, c.channels, {a_codes, b_codes});
    const GatedBackArgs k = {da, db, dy, a, b, a_codes, b_codes, a_scales, b_scales,
                             c.a_pitch, c.b_pitch, c.y_pitch, c.da_pitch, c.db_pitch,
                             c.act, c.act_param};
    return by_type(c.type, width, [&](auto* t, auto w) {
        using T = std::remove_pointer_t<decltype(t)>;
        constexpr int AW = decltype(w)::value;
        const auto kernel =
            from ? (gate ? k_gated_back<T, AW, true, true> : k_gated_back<T, AW, true, false>)
                 : (gate ? k_gated_back<T, AW, false, true> : k_gated_back<T, AW, false, false>);
        sg::before_launch();
        kernel<<<(unsigned)row_blocks(g), kThreads, 0, (cudaStream_t)stream>>>(k, g);
        return sg::launch_status(K);
    });
}

}  // extern "C"
