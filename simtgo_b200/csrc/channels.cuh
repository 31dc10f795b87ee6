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

__device__ __forceinline__ void unpack(const Raw<float>& r, float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 2; i++) {
        v[4 * i] = __uint_as_float(r.q[i].x);
        v[4 * i + 1] = __uint_as_float(r.q[i].y);
        v[4 * i + 2] = __uint_as_float(r.q[i].z);
        v[4 * i + 3] = __uint_as_float(r.q[i].w);
    }
}
__device__ __forceinline__ void unpack(const Raw<__nv_bfloat16>& r, float (&v)[8]) {
    const uint32_t w[4] = {r.q[0].x, r.q[0].y, r.q[0].z, r.q[0].w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
}
__device__ __forceinline__ void unpack(const Raw<__half>& r, float (&v)[8]) {
    const uint32_t w[4] = {r.q[0].x, r.q[0].y, r.q[0].z, r.q[0].w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
    }
}

// Rounded to nearest even, once.
__device__ __forceinline__ void pack(const float (&v)[8], Raw<float>& r) {
#pragma unroll
    for (int i = 0; i < 2; i++)
        r.q[i] = make_uint4(__float_as_uint(v[4 * i]), __float_as_uint(v[4 * i + 1]),
                            __float_as_uint(v[4 * i + 2]), __float_as_uint(v[4 * i + 3]));
}
__device__ __forceinline__ void pack(const float (&v)[8], Raw<__nv_bfloat16>& r) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    r.q[0] = make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ void pack(const float (&v)[8], Raw<__half>& r) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
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
// Two-byte types take the special-function unit's exponential and reciprocal
// (a few 2^-22, far below their 2^-9 and 2^-12 half steps): the exact ones
// would bind the kernels before HBM does. float32 keeps expf, erff and IEEE
// division.

__device__ __forceinline__ float rcp_fast(float x) {
    float r;
    asm("rcp.approx.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

template <bool kFast>
__device__ __forceinline__ float sigmoid(float z) {
    return kFast ? __fdividef(1.0f, 1.0f + __expf(-z)) : __fdiv_rn(1.0f, 1.0f + expf(-z));
}

// Phi(z), the normal distribution function, and e = exp(-z^2/2). The fast
// form is Abramowitz and Stegun's 7.1.26 for erf (Hastings), within 1.5e-7,
// in the variable t = 1/(1 + p |z|/sqrt 2); the negative side is taken from
// the complement itself, so it does not cancel.
template <bool kFast>
__device__ __forceinline__ float normal_cdf(float z, float& e) {
    if (!kFast) {
        e = expf(-0.5f * z * z);
        return 0.5f * erfcf(-0.70710678f * z);
    }
    const float x = fabsf(z) * 0.70710678f;
    const float t = __fdividef(1.0f, __fmaf_rn(0.3275911f, x, 1.0f));
    e = __expf(-x * x);
    float q = __fmaf_rn(1.061405429f, t, -1.453152027f);
    q = __fmaf_rn(q, t, 1.421413741f);
    q = __fmaf_rn(q, t, -0.284496736f);
    q = __fmaf_rn(q, t, 0.254829592f);
    q = 0.5f * q * t * e;  // Phi(-|z|)
    return z < 0.0f ? q : 1.0f - q;
}

// softclip of kernels/softclip.go:11-23 and its slope factor 1/(1+over).
template <bool kFast>
__device__ __forceinline__ float softclip(float z, float t, float& slope) {
    const float a = fabsf(z), over = a - t;
    const float r = kFast ? rcp_fast(1.0f + over) : __fdiv_rn(1.0f, 1.0f + over);
    const float shaped = t + (kFast ? over * r : __fdiv_rn(over, 1.0f + over));
    slope = a <= t ? 1.0f : r * r;
    return a <= t ? z : z < 0.0f ? -shaped : shaped;
}

// v <- act(v), eight at a time (one uniform branch per unit).
template <bool kFast>
__device__ __forceinline__ void activate(float (&v)[8], int act, float param) {
    float s;
    if (act == SIMTGO_ACT_SILU) {
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] *= sigmoid<kFast>(v[i]);
    } else if (act == SIMTGO_ACT_GELU) {
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] *= normal_cdf<kFast>(v[i], s);
    } else if (act == SIMTGO_ACT_SOFTCLIP) {
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = softclip<kFast>(v[i], param, s);
    }
}

// f <- act(z), d <- act'(z).
template <bool kFast>
__device__ __forceinline__ void activate_slope(const float (&z)[8], float (&f)[8], float (&d)[8],
                                               int act, float param) {
    if (act == SIMTGO_ACT_SILU) {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const float s = sigmoid<kFast>(z[i]);
            f[i] = z[i] * s;
            d[i] = __fmaf_rn(f[i], 1.0f - s, s);
        }
    } else if (act == SIMTGO_ACT_GELU) {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            float e;
            const float p = normal_cdf<kFast>(z[i], e);
            f[i] = z[i] * p;
            d[i] = __fmaf_rn(z[i] * 0.39894228f, e, p);
        }
    } else if (act == SIMTGO_ACT_SOFTCLIP) {
#pragma unroll
        for (int i = 0; i < 8; i++) f[i] = softclip<kFast>(z[i], param, d[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            f[i] = z[i];
            d[i] = 1.0f;
        }
    }
}

// ---- the 8-bit checkpoint ---------------------------------------------------------
// A block of `block` consecutive channels of a row shares a float32 scale:
// a = max(largest magnitude, 2^-100), scale = a/127, code = rint(x * (127/a)),
// each step rounded to float32. The floor keeps 127/a finite and makes an
// all-zero block need no case of its own. Magnitudes are compared as bit
// patterns, where NaN is above infinity: a block that holds either gets
// scale NaN, so it restores to NaN throughout and nothing is hidden.

struct Codes {
    uint2 q;  // eight signed bytes
};

__device__ __forceinline__ uint32_t largest(const float (&v)[8]) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
    return m;
}

// The block's scale and its inverse from the bit pattern of its largest
// magnitude.
__device__ __forceinline__ void block_scale(uint32_t m, float& scale, float& inverse) {
    if (m >= 0x7f800000u) {
        scale = __uint_as_float(0x7fffffffu);
        inverse = 0.0f;
        return;
    }
    const float a = fmaxf(__uint_as_float(m), 0x1p-100f);
    scale = __fdiv_rn(a, 127.0f);
    inverse = __fdiv_rn(127.0f, a);
}

// rint(v * inverse) as signed bytes: adding 1.5 * 2^23 leaves the rounded
// whole number (nearest even) in the low mantissa bits, whose low byte is its
// two's complement.
__device__ __forceinline__ Codes encode(const float (&v)[8], float inverse) {
    uint32_t b[8];
#pragma unroll
    for (int i = 0; i < 8; i++)
        b[i] = __float_as_uint(__fadd_rn(__fmul_rn(v[i], inverse), 12582912.0f));
    Codes c;
    c.q.x = __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
    c.q.y = __byte_perm(__byte_perm(b[4], b[5], 0x0040), __byte_perm(b[6], b[7], 0x0040), 0x5410);
    return c;
}

// What the codes stand for, in float32: fl(code * scale). A byte k with its
// sign bit flipped is k + 128; placed under the exponent of 2^23 it reads as
// 2^23 + 128 + k, exactly.
__device__ __forceinline__ void decode(const Codes& c, float scale, float (&v)[8]) {
    const uint32_t w[2] = {c.q.x ^ 0x80808080u, c.q.y ^ 0x80808080u};
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const uint32_t u = __byte_perm(w[i / 4], 0x4b000000u, 0x7440 | (i & 3));
        v[i] = __fmul_rn(__uint_as_float(u) - 8388736.0f, scale);
    }
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

// Largest bit pattern over the `lanes` (a power of two) neighbouring lanes
// that hold one block. Every lane of the warp calls it.
__device__ __forceinline__ uint32_t block_max(uint32_t m, int lanes) {
    for (int off = lanes / 2; off; off /= 2) m = max(m, __shfl_xor_sync(~0u, m, off));
    return m;
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
// (bytes; 0 where it is taken once only), `bytes` from its first to its last.
struct Region {
    const char* name;
    const void* p;
    int64_t width, pitch0, pitch1, bytes;
    bool written;
};
inline Region solid(const char* name, const void* p, int64_t bytes, bool written) {
    return {name, p, bytes, 0, 0, bytes, written};
}
// SIMTGO_EALIAS for two regions that may overlap, one of them written. Rows of
// one buffer that interleave (channel slices of the same batch) do not: with
// all pitches multiples of P, a region lies in one stretch of the residues mod
// P, and two such stretches are compared.
int check_regions(const char* K, std::initializer_list<Region> regions);

// Argument checks the operators share. Each returns 0 or a status code.
int check_type(const char* K, const char* name, int32_t type);
int check_act(const char* K, int32_t act, float param);
int check_block(const char* K, int32_t block);
int check_aligned(const char* K, const char* name, const void* p, int bytes);

}  // namespace chan
