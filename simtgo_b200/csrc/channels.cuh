// channels.cuh -- what the channels-last operators share (groupnorm.cu,
// checkpoint.cu): eight consecutive channels of a row as one unit, loaded and
// stored at the width the caller's alignment allows, the activations with
// their slopes, and the 8-bit checkpoint's codes.
//
// A unit is the same eight channels whatever the element type and the
// alignment, so that a group's or a block's arithmetic never depends on
// either; only the access instructions do (AW, bytes per access: 16 when every
// row starts on a 16-byte boundary, 4 for two-byte types on a 4-byte
// boundary, else the element).
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace chan {

constexpr int kUnit = 8;  // channels per unit

// ---- units of eight channels ------------------------------------------------

template <class T>
struct Raw {  // eight elements as they lie in memory
    uint4 q[sizeof(T) / 2];
};

__device__ __forceinline__ uint4 ldg16(const void* p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "l"(p));
    return v;
}
__device__ __forceinline__ uint2 ldg8(const void* p) {
    uint2 v;
    asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0,%1}, [%2];"
                 : "=r"(v.x), "=r"(v.y)
                 : "l"(p));
    return v;
}
__device__ __forceinline__ void stg16(void* p, uint4 v) {
    asm volatile("st.global.cs.v4.u32 [%0], {%1,%2,%3,%4};" ::"l"(p), "r"(v.x), "r"(v.y),
                 "r"(v.z), "r"(v.w)
                 : "memory");
}
__device__ __forceinline__ void stg8(void* p, uint2 v) {
    asm volatile("st.global.cs.v2.u32 [%0], {%1,%2};" ::"l"(p), "r"(v.x), "r"(v.y) : "memory");
}

// The first cnt (1..8) elements at p; the others are zero.
template <class T, int AW>
__device__ __forceinline__ Raw<T> ld_unit(const T* p, int cnt) {
    Raw<T> r;
    if (AW == 16 && cnt == kUnit) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; i++)
            r.q[i] = ldg16(reinterpret_cast<const char*>(p) + 16 * i);
        return r;
    }
    uint32_t w[2 * sizeof(T)];
    if constexpr (sizeof(T) == 4) {
        const uint32_t* u = reinterpret_cast<const uint32_t*>(p);
#pragma unroll
        for (int i = 0; i < 8; i++) w[i] = i < cnt ? __ldg(u + i) : 0u;
    } else {
        if (AW >= 4 && cnt == kUnit) {
            const uint32_t* u = reinterpret_cast<const uint32_t*>(p);
#pragma unroll
            for (int i = 0; i < 4; i++) w[i] = __ldg(u + i);
        } else {
            const uint16_t* u = reinterpret_cast<const uint16_t*>(p);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const uint32_t lo = 2 * i < cnt ? __ldg(u + 2 * i) : 0;
                const uint32_t hi = 2 * i + 1 < cnt ? __ldg(u + 2 * i + 1) : 0;
                w[i] = lo | hi << 16;
            }
        }
    }
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; i++)
        r.q[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
    return r;
}

template <class T, int AW>
__device__ __forceinline__ void st_unit(T* p, const Raw<T>& r, int cnt) {
    if (AW == 16 && cnt == kUnit) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; i++)
            stg16(reinterpret_cast<char*>(p) + 16 * i, r.q[i]);
        return;
    }
    uint32_t w[2 * sizeof(T)];
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; i++) {
        w[4 * i] = r.q[i].x;
        w[4 * i + 1] = r.q[i].y;
        w[4 * i + 2] = r.q[i].z;
        w[4 * i + 3] = r.q[i].w;
    }
    if constexpr (sizeof(T) == 4) {
        uint32_t* u = reinterpret_cast<uint32_t*>(p);
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (i < cnt) u[i] = w[i];
    } else {
        if (AW >= 4 && cnt == kUnit) {
            uint32_t* u = reinterpret_cast<uint32_t*>(p);
#pragma unroll
            for (int i = 0; i < 4; i++) u[i] = w[i];
        } else {
            uint16_t* u = reinterpret_cast<uint16_t*>(p);
#pragma unroll
            for (int i = 0; i < 8; i++)
                if (i < cnt) u[i] = (uint16_t)(w[i / 2] >> (16 * (i & 1)));
        }
    }
}

// Eight values as four pairs: Blackwell's packed float32 instructions take two
// at once, each rounded as the scalar ones are, which halves the instructions
// of kernels that issue slots would otherwise bound before HBM does.
struct V8 {
    float2 p[4];
};

// The assembler may contract a packed product with the addition after it: where
// the product's own rounding counts (the checkpoint's codes) it is scalar.
__device__ __forceinline__ float2 mul2(float2 a, float2 b) { return __fmul2_rn(a, b); }
__device__ __forceinline__ float2 add2(float2 a, float2 b) { return __fadd2_rn(a, b); }
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) { return __ffma2_rn(a, b, c); }

__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }
__device__ __forceinline__ float2 neg2(float2 v) { return make_float2(-v.x, -v.y); }
// a - b, rounded once.
__device__ __forceinline__ float2 sub2(float2 a, float2 b) { return fma2(b, both(-1.0f), a); }

__device__ __forceinline__ V8 unpack(const Raw<float>& r) {
    V8 v;
#pragma unroll
    for (int i = 0; i < 2; i++) {
        v.p[2 * i] = make_float2(__uint_as_float(r.q[i].x), __uint_as_float(r.q[i].y));
        v.p[2 * i + 1] = make_float2(__uint_as_float(r.q[i].z), __uint_as_float(r.q[i].w));
    }
    return v;
}
__device__ __forceinline__ V8 unpack(const Raw<__nv_bfloat16>& r) {
    const uint32_t w[4] = {r.q[0].x, r.q[0].y, r.q[0].z, r.q[0].w};
    V8 v;
#pragma unroll
    for (int i = 0; i < 4; i++)
        v.p[i] = make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
    return v;
}
__device__ __forceinline__ V8 unpack(const Raw<__half>& r) {
    const uint32_t w[4] = {r.q[0].x, r.q[0].y, r.q[0].z, r.q[0].w};
    V8 v;
#pragma unroll
    for (int i = 0; i < 4; i++) v.p[i] = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    return v;
}

// Rounded to nearest even, once.
__device__ __forceinline__ void pack(const V8& v, Raw<float>& r) {
#pragma unroll
    for (int i = 0; i < 2; i++)
        r.q[i] = make_uint4(__float_as_uint(v.p[2 * i].x), __float_as_uint(v.p[2 * i].y),
                            __float_as_uint(v.p[2 * i + 1].x), __float_as_uint(v.p[2 * i + 1].y));
}
__device__ __forceinline__ void pack(const V8& v, Raw<__nv_bfloat16>& r) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const __nv_bfloat162 h = __float22bfloat162_rn(v.p[i]);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    r.q[0] = make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ void pack(const V8& v, Raw<__half>& r) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const __half2 h = __float22half2_rn(v.p[i]);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    r.q[0] = make_uint4(w[0], w[1], w[2], w[3]);
}

// One element of a parameter array of any of the three types.
__device__ __forceinline__ float ld_param(const void* p, int type, int64_t i) {
    if (type == SIMTGO_F32) return __ldg(static_cast<const float*>(p) + i);
    const uint16_t u = __ldg(static_cast<const uint16_t*>(p) + i);
    if (type == SIMTGO_BF16) return __uint_as_float((uint32_t)u << 16);
    return __half2float(__ushort_as_half(u));
}

// ---- activations --------------------------------------------------------------
// Two-byte types take the special-function unit's exp2 and reciprocal: the exact
// functions would bind the kernels before HBM does. The unit is within a few
// 2^-22; exp2's argument z*log2(e) carries a rounding of its own size, so
// sigmoid is within |z| 2^-23 relative in its tail, and Phi within 2^-15 down to
// z = -13, where float32's normal numbers end (half steps: 2^-9 and 2^-12).
// float32 keeps expf, erfcf and IEEE division; there the tail of Phi carries
// the rounding of erfc's argument, 2^-23 (z^2 + 1).

__device__ __forceinline__ float ex2_fast(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
// For 1 <= x, where a flushed result is one that no sum notices.
__device__ __forceinline__ float rcp_ftz(float x) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float rcp_fast(float x) {
    float r;
    asm("rcp.approx.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
// min and max that keep a NaN.
__device__ __forceinline__ float min_nan(float a, float b) {
    float r;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

template <bool kFast>
__device__ __forceinline__ float2 sigmoid2(float2 z) {
    if (!kFast)
        return make_float2(__fdiv_rn(1.0f, 1.0f + expf(-z.x)), __fdiv_rn(1.0f, 1.0f + expf(-z.y)));
    const float2 e = mul2(z, both(-1.44269504f));
    const float2 d = add2(make_float2(ex2_fast(e.x), ex2_fast(e.y)), both(1.0f));
    return make_float2(rcp_ftz(d.x), rcp_ftz(d.y));
}

// Fast GELU: with q = Phi(-|z|) and e = exp(-z^2/2), z*Phi(z) is
// max(z, 0) - |z|*q. q/e, half the scaled complement of erf, falls from 1/2 as
// 1/|z|: t times a polynomial in t = 1/(1 + p |z|), fitted for the least
// relative error over |z| <= 20 (6e-6; six terms by linear programming, p by
// search; a seventh term, 1.1e-6, made the GELU passes 2 % slower), so that the
// tail, which is q alone, is right to its own size. Past |z| = 20 e is zero in
// float32, so |z| stops there and no infinity meets a zero.
struct Normal2 {
    float2 az, q, e;
};
__device__ __forceinline__ Normal2 normal2(float2 z) {
    Normal2 r;
    r.az = make_float2(min_nan(fabsf(z.x), 20.0f), min_nan(fabsf(z.y), 20.0f));
    const float2 d = fma2(r.az, both(0.3125f), both(1.0f));
    const float2 t = make_float2(rcp_ftz(d.x), rcp_ftz(d.y));
    const float2 h = mul2(mul2(r.az, r.az), both(-0.5f * 1.44269504f));
    r.e = make_float2(ex2_fast(h.x), ex2_fast(h.y));
    float2 q = fma2(both(-0.071931385f), t, both(0.16906056f));
    q = fma2(q, t, both(0.025909422f));
    q = fma2(q, t, both(0.12987943f));
    q = fma2(q, t, both(0.122284167f));
    q = fma2(q, t, both(0.12479526f));
    r.q = mul2(mul2(q, t), r.e);
    return r;
}
__device__ __forceinline__ float2 gelu2(float2 z, const Normal2& n) {
    return sub2(make_float2(max_nan(z.x, 0.0f), max_nan(z.y, 0.0f)), mul2(n.az, n.q));
}

// softclip of kernels/softclip.go:11-23 and its slope, 1 or 1/(1+over)^2.
template <bool kFast>
__device__ __forceinline__ float softclip(float z, float t, float& slope) {
    const float a = fabsf(z), over = a - t;
    const float r = kFast ? rcp_fast(1.0f + over) : __fdiv_rn(1.0f, 1.0f + over);
    const float shaped = t + (kFast ? over * r : __fdiv_rn(over, 1.0f + over));
    slope = a <= t ? 1.0f : r * r;
    return a <= t ? z : copysignf(shaped, z);
}

// v <- act(v), eight at a time (one uniform branch per unit).
template <bool kFast>
__device__ __forceinline__ void activate(V8& v, int act, float param) {
    if (act == SIMTGO_ACT_SILU) {
#pragma unroll
        for (int i = 0; i < 4; i++) v.p[i] = mul2(v.p[i], sigmoid2<kFast>(v.p[i]));
    } else if (act == SIMTGO_ACT_GELU) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if (kFast) {
                v.p[i] = gelu2(v.p[i], normal2(v.p[i]));
            } else {
                v.p[i].x *= 0.5f * erfcf(-0.70710678f * v.p[i].x);
                v.p[i].y *= 0.5f * erfcf(-0.70710678f * v.p[i].y);
            }
        }
    } else if (act == SIMTGO_ACT_SOFTCLIP) {
        float s;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            v.p[i].x = softclip<kFast>(v.p[i].x, param, s);
            v.p[i].y = softclip<kFast>(v.p[i].y, param, s);
        }
    }
}

// f <- act(z), d <- act'(z).
template <bool kFast>
__device__ __forceinline__ void activate_slope(const V8& z, V8& f, V8& d, int act, float param) {
    if (act == SIMTGO_ACT_SILU) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float2 s = sigmoid2<kFast>(z.p[i]);
            f.p[i] = mul2(z.p[i], s);
            d.p[i] = fma2(f.p[i], sub2(both(1.0f), s), s);
        }
    } else if (act == SIMTGO_ACT_GELU) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if (kFast) {
                const Normal2 n = normal2(z.p[i]);
                f.p[i] = gelu2(z.p[i], n);
                // Phi is q itself below zero; z*phi with |z| stopped as above.
                const float2 h = sub2(both(1.0f), n.q);
                const float2 c = make_float2(z.p[i].x < 0.0f ? n.q.x : h.x,
                                             z.p[i].y < 0.0f ? n.q.y : h.y);
                const float2 zc =
                    make_float2(copysignf(n.az.x, z.p[i].x), copysignf(n.az.y, z.p[i].y));
                d.p[i] = fma2(mul2(zc, both(0.39894228f)), n.e, c);
            } else {
                const float px = 0.5f * erfcf(-0.70710678f * z.p[i].x);
                const float py = 0.5f * erfcf(-0.70710678f * z.p[i].y);
                f.p[i] = make_float2(z.p[i].x * px, z.p[i].y * py);
                d.p[i].x = __fmaf_rn(z.p[i].x * 0.39894228f, expf(-0.5f * z.p[i].x * z.p[i].x), px);
                d.p[i].y = __fmaf_rn(z.p[i].y * 0.39894228f, expf(-0.5f * z.p[i].y * z.p[i].y), py);
            }
        }
    } else if (act == SIMTGO_ACT_SOFTCLIP) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            f.p[i].x = softclip<kFast>(z.p[i].x, param, d.p[i].x);
            f.p[i].y = softclip<kFast>(z.p[i].y, param, d.p[i].y);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            f.p[i] = z.p[i];
            d.p[i] = both(1.0f);
        }
    }
}

// ---- the 8-bit checkpoint ---------------------------------------------------------
// A block of `block` consecutive channels of a row shares a float32 scale:
// a = max(largest magnitude, 2^-100), scale = a/127, code = rint(x * (127/a)),
// each step rounded to float32 (the largest float's scale down, so that 127 of it
// are finite). The floor keeps 127/a finite and makes an all-zero block need no
// case of its own. Magnitudes are compared as bit
// patterns, where NaN is above infinity: a block that holds either gets
// scale NaN, so it restores to NaN throughout and nothing is hidden.

struct Codes {
    uint2 q;  // eight signed bytes
};

// Bit patterns of the largest magnitudes of the blocks that U rows' units lie
// in, over the `lanes` (a power of two) neighbouring lanes that hold a block.
// Every lane of the warp calls it. Two-byte types carry two rows in a
// register's halves.
template <int U>
__device__ __forceinline__ void block_max(const Raw<float> (&raw)[U], int lanes,
                                          uint32_t (&m)[U]) {
#pragma unroll
    for (int u = 0; u < U; u++) {
        m[u] = 0;
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const uint4 q = raw[u].q[i];
            m[u] = max(max(m[u], max(q.x & 0x7fffffffu, q.y & 0x7fffffffu)),
                       max(q.z & 0x7fffffffu, q.w & 0x7fffffffu));
        }
    }
    for (int off = lanes / 2; off; off /= 2)
#pragma unroll
        for (int u = 0; u < U; u++) m[u] = max(m[u], __shfl_xor_sync(~0u, m[u], off));
}
template <int U>
__device__ __forceinline__ void block_max16(const uint4 (&raw)[U], int lanes, uint32_t (&m)[U]) {
    static_assert(U % 2 == 0, "rows go in pairs");
    uint32_t pair[U / 2];
#pragma unroll
    for (int u = 0; u < U; u += 2) {
        uint32_t h[2];
#pragma unroll
        for (int j = 0; j < 2; j++) {
            const uint4 q = raw[u + j];
            h[j] = __vmaxu2(__vmaxu2(q.x & 0x7fff7fffu, q.y & 0x7fff7fffu),
                            __vmaxu2(q.z & 0x7fff7fffu, q.w & 0x7fff7fffu));
        }
        pair[u / 2] = __vmaxu2(__byte_perm(h[0], h[1], 0x5410), __byte_perm(h[0], h[1], 0x7632));
    }
    for (int off = lanes / 2; off; off /= 2)
#pragma unroll
        for (int u = 0; u < U / 2; u++)
            pair[u] = __vmaxu2(pair[u], __shfl_xor_sync(~0u, pair[u], off));
#pragma unroll
    for (int u = 0; u < U; u++) m[u] = u & 1 ? pair[u / 2] >> 16 : pair[u / 2] & 0xffffu;
}
template <int U>
__device__ __forceinline__ void block_max(const Raw<__nv_bfloat16> (&raw)[U], int lanes,
                                          uint32_t (&m)[U]) {
    uint4 q[U];
#pragma unroll
    for (int u = 0; u < U; u++) q[u] = raw[u].q[0];
    block_max16<U>(q, lanes, m);
#pragma unroll
    for (int u = 0; u < U; u++) m[u] <<= 16;
}
template <int U>
__device__ __forceinline__ void block_max(const Raw<__half> (&raw)[U], int lanes,
                                          uint32_t (&m)[U]) {
    uint4 q[U];
#pragma unroll
    for (int u = 0; u < U; u++) q[u] = raw[u].q[0];
    block_max16<U>(q, lanes, m);
#pragma unroll
    for (int u = 0; u < U; u++)
        m[u] = __float_as_uint(__half2float(__ushort_as_half((unsigned short)m[u])));
}

// A block's scale and its inverse from the bit pattern of its largest
// magnitude.
__device__ __forceinline__ void block_scale(uint32_t m, float& scale, float& inverse) {
    if (m >= 0x7f800000u) {
        scale = __uint_as_float(0x7fffffffu);
        inverse = 0.0f;
        return;
    }
    const float a = fmaxf(__uint_as_float(m), 0x1p-100f);
    scale = fminf(__fdiv_rn(a, 127.0f), 0x1.02040600p+121f);  // FLT_MAX/127, rounded down
    inverse = __fdiv_rn(127.0f, a);
}

// rint(v * inverse) as signed bytes: adding 1.5 * 2^23 leaves the rounded
// whole number (nearest even) in the low mantissa bits, whose low byte is its
// two's complement.
__device__ __forceinline__ Codes encode(const V8& v, float inverse) {
    uint32_t b[8];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float2 q =
            make_float2(__fmul_rn(v.p[i].x, inverse), __fmul_rn(v.p[i].y, inverse));
        const float2 r = add2(q, both(12582912.0f));
        b[2 * i] = __float_as_uint(r.x);
        b[2 * i + 1] = __float_as_uint(r.y);
    }
    Codes c;
    c.q.x = __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
    c.q.y = __byte_perm(__byte_perm(b[4], b[5], 0x0040), __byte_perm(b[6], b[7], 0x0040), 0x5410);
    return c;
}

// What the codes stand for, in float32: fl(code * scale). A byte k with its
// sign bit flipped is k + 128; placed under the exponent of 2^23 it reads as
// 2^23 + 128 + k, exactly.
__device__ __forceinline__ V8 decode(const Codes& c, float scale) {
    const uint32_t w[2] = {c.q.x ^ 0x80808080u, c.q.y ^ 0x80808080u};
    V8 v;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t a = __byte_perm(w[i / 2], 0x4b000000u, 0x7440 | (2 * i & 3));
        const uint32_t b = __byte_perm(w[i / 2], 0x4b000000u, 0x7440 | ((2 * i + 1) & 3));
        v.p[i] = mul2(
            add2(make_float2(__uint_as_float(a), __uint_as_float(b)), both(-8388736.0f)),
            both(scale));
    }
    return v;
}

template <bool kVec>
__device__ __forceinline__ Codes ld_codes(const int8_t* p, int cnt) {
    Codes c;
    if (kVec) {
        c.q = ldg8(p);
        return c;
    }
    uint32_t w[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 8; i++)
        if (i < cnt)
            w[i / 4] |= (uint32_t)__ldg(reinterpret_cast<const uint8_t*>(p) + i) << (8 * (i & 3));
    c.q = make_uint2(w[0], w[1]);
    return c;
}

template <bool kVec>
__device__ __forceinline__ void st_codes(int8_t* p, const Codes& c, int cnt) {
    if (kVec) {
        stg8(p, c.q);
        return;
    }
    const uint32_t w[2] = {c.q.x, c.q.y};
#pragma unroll
    for (int i = 0; i < 8; i++)
        if (i < cnt) p[i] = (int8_t)(w[i / 4] >> (8 * (i & 3)));
}

// Where a tensor's checkpoint lies, and how a row's units map to its blocks.
struct Kept {
    int8_t* codes;
    float* scales;
    int channels, nblk;  // bytes of codes and scales per row
    int shift, lanes;    // log2(units per block); lanes that hold one block
};

// A thread's place in a checkpoint: its unit's codes and its block's scale in
// the first of its rows, and how far on the next of its rows are.
struct KeptAt {
    int8_t* codes;
    float* scale;
    int64_t codes_step, scale_step;
};
__device__ __forceinline__ KeptAt kept_at(const Kept& k, int64_t row, int64_t step, int unit) {
    return {k.codes + row * k.channels + unit * kUnit, k.scales + row * k.nblk + (unit >> k.shift),
            step * k.channels, step * k.nblk};
}

// Writes the checkpoint of the units that a warp's lanes hold of U rows: unit
// `unit` (cnt channels; only where unit_on) of the thread's rows from `at` on,
// where live[u]. Every lane of the warp calls it, with zeros where it has no
// unit; live is the same for the lanes of a block. The two divisions of a
// block's scale are shared out: lane u of each block's lanes makes row u's,
// where there are that many.
template <class T, int AW, int U, bool kFlat = false>
__device__ __forceinline__ void keep_units(const Raw<T> (&raw)[U], const Kept& k, const KeptAt& at,
                                           const bool (&live)[U], int unit, int cnt,
                                           bool unit_on) {
    uint32_t m[U];
    block_max<U>(raw, k.lanes, m);
    float inverse[U];
    const bool block_on = kFlat || (unit >> k.shift) < k.nblk;
    if (k.lanes >= U) {
        const int mine = threadIdx.x & (U - 1);
        uint32_t sel = m[0];
        bool sel_on = live[0];
        float* to = at.scale;
#pragma unroll
        for (int u = 1; u < U; u++) {
            sel = mine == u ? m[u] : sel;
            sel_on = mine == u ? live[u] : sel_on;
        }
        float scale, inv;
        block_scale(sel, scale, inv);
#pragma unroll
        for (int u = 0; u < U; u++)
            inverse[u] = __shfl_sync(~0u, inv, (threadIdx.x & 31 & ~(U - 1)) + u);
        if (sel_on && (unit & (k.lanes - 1)) == mine && block_on) to[mine * at.scale_step] = scale;
    } else {
#pragma unroll
        for (int u = 0; u < U; u++) {
            float scale;
            block_scale(m[u], scale, inverse[u]);
            if (live[u] && (unit & (k.lanes - 1)) == 0 && block_on)
                at.scale[u * at.scale_step] = scale;
        }
    }
#pragma unroll
    for (int u = 0; u < U; u++)
        if (unit_on && live[u])
            st_codes<AW == 16>(at.codes + u * at.codes_step, encode(unpack(raw[u]), inverse[u]),
                               cnt);
}

// ---- host helpers -------------------------------------------------------------------

inline int elem_size(int32_t type) { return type == SIMTGO_F32 ? 4 : 2; }

// A matrix or batch as the access width sees it.
struct Access {
    const void* p;
    int64_t pitch0, pitch1;  // elements; a pitch never taken is passed as 0
};
// Bytes per access that every row of the given arrays allows: 16, 4 or the
// element size.
inline int access_width(int32_t type, std::initializer_list<Access> arrays) {
    const int e = elem_size(type);
    int64_t bits = 0;
    for (const Access& a : arrays)
        if (a.p) bits |= (int64_t)(uintptr_t)a.p | a.pitch0 * e | a.pitch1 * e;
    return (bits & 15) == 0 ? 16 : (bits & 3) == 0 ? 4 : e;
}

inline int ceil_pow2(int v) {
    int p = 1;
    while (p < v) p *= 2;
    return p;
}

// Calls f with a null pointer of the element type and the access width as an
// integral constant.
template <class F>
int by_type(int32_t type, int width, F&& f) {
    if (type == SIMTGO_F32)
        return width == 16 ? f((float*)nullptr, std::integral_constant<int, 16>())
                           : f((float*)nullptr, std::integral_constant<int, 4>());
    if (type == SIMTGO_BF16) {
        if (width == 16) return f((__nv_bfloat16*)nullptr, std::integral_constant<int, 16>());
        if (width == 4) return f((__nv_bfloat16*)nullptr, std::integral_constant<int, 4>());
        return f((__nv_bfloat16*)nullptr, std::integral_constant<int, 2>());
    }
    if (width == 16) return f((__half*)nullptr, std::integral_constant<int, 16>());
    if (width == 4) return f((__half*)nullptr, std::integral_constant<int, 4>());
    return f((__half*)nullptr, std::integral_constant<int, 2>());
}

// A buffer of rows: `width` bytes at each combination of up to two pitches
// (bytes; 0 where it is taken once only), each taken so many times; `bytes` from
// its first to its last.
struct Region {
    const char* name;
    const void* p;
    int64_t width, pitch0, pitch1, bytes;
    bool written;
    int64_t times0, times1;
};
inline Region solid(const char* name, const void* p, int64_t bytes, bool written) {
    return {name, p, bytes, 0, 0, bytes, written, 1, 1};
}
// SIMTGO_EALIAS for two regions that may overlap, one of them written. Parts of
// one buffer (channel slices, crops of positions, every second sample of the same
// batch) do not where none of their rows meet: exactly, where both have the same
// pitches and counts and one pitch steps over all of the other's rows. Else, with
// all pitches multiples of P, a region lies in one stretch of the residues mod
// P, and two such stretches are compared.
int check_regions(const char* K, std::initializer_list<Region> regions);

// Argument checks the operators share. Each returns 0 or a status code.
int check_type(const char* K, const char* name, int32_t type);
int check_act(const char* K, int32_t act, float param);
int check_block(const char* K, int32_t block);
int check_aligned(const char* K, const char* name, const void* p, int bytes);

}  // namespace chan
