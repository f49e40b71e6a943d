// Device code shared by the quantisers (quant.cu) and the norm (norm.cu): 16-element vector loads, one thread's 16 elements, and
// the conversions to E4M3 and e2m1 with IEEE fp32 arithmetic throughout (see quant.cu for the rules).
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "ptx.cuh"

namespace dsl {

// ---- 16-element vector loads ------------------------------------------------------------
template <typename T> struct dsl_is_half { static constexpr bool value = false; };
template <> struct dsl_is_half<__half> { static constexpr bool value = true; };
template <typename T>
__device__ __forceinline__ void load16(const T* p, float (&v)[16]);

template <>
__device__ __forceinline__ void load16<float>(const float* p, float (&v)[16]) {
    const float4* q = reinterpret_cast<const float4*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float4 t = __ldg(q + i);
        v[4 * i] = t.x; v[4 * i + 1] = t.y; v[4 * i + 2] = t.z; v[4 * i + 3] = t.w;
    }
}
template <>
__device__ __forceinline__ void load16<__nv_bfloat16>(const __nv_bfloat16* p, float (&v)[16]) {
    const uint4* q = reinterpret_cast<const uint4*>(p);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        uint4 t = __ldg(q + i);
        uint32_t w[4] = {t.x, t.y, t.z, t.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            v[8 * i + 2 * j] = __uint_as_float(w[j] << 16);
            v[8 * i + 2 * j + 1] = __uint_as_float(w[j] & 0xFFFF0000u);
        }
    }
}
template <>
__device__ __forceinline__ void load16<__half>(const __half* p, float (&v)[16]) {
    const uint4* q = reinterpret_cast<const uint4*>(p);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        uint4 t = __ldg(q + i);
        uint32_t w[4] = {t.x, t.y, t.z, t.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float2 f = __half22float2(*reinterpret_cast<__half2*>(&w[j]));
            v[8 * i + 2 * j] = f.x;
            v[8 * i + 2 * j + 1] = f.y;
        }
    }
}
// The same 16 elements with 256-bit loads (one for 16-bit types, two for fp32): a warp's request then covers whole
// 128-byte lines instead of every other 16 bytes of them, which halves the requests the L1 has to replay for these
// streaming kernels.  The address must be 32-byte aligned (`wide` is decided on the host from the base pointer and the
// row pitch); the data is read once, so it bypasses L1 allocation.
__device__ __forceinline__ void ldg256(const void* p, uint32_t (&r)[8]) {
    asm volatile("ld.global.nc.L1::no_allocate.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "l"(p));
}
template <typename T>
__device__ __forceinline__ void load16w(const T* p, float (&v)[16], bool wide) {
    if (!wide) { load16<T>(p, v); return; }
    if (sizeof(T) == 4) {
        uint32_t a[8], b[8];
        ldg256(p, a);
        ldg256(reinterpret_cast<const uint8_t*>(p) + 32, b);
#pragma unroll
        for (int i = 0; i < 8; ++i) { v[i] = __uint_as_float(a[i]); v[8 + i] = __uint_as_float(b[i]); }
    } else {
        uint32_t w[8];
        ldg256(p, w);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            if (sizeof(T) == 2 && !dsl_is_half<T>::value) {
                v[2 * j] = __uint_as_float(w[j] << 16);
                v[2 * j + 1] = __uint_as_float(w[j] & 0xFFFF0000u);
            } else {
                float2 f = __half22float2(*reinterpret_cast<__half2*>(&w[j]));
                v[2 * j] = f.x;
                v[2 * j + 1] = f.y;
            }
        }
    }
}
// ---- one thread's 16 elements --------------------------------------------------------------
// Generic form: 16 floats.  bf16 (the activations' usual type) has a form that keeps the raw 8 words: the block
// maximum comes from packed |x| / max on bf16 pairs (exact: they are comparisons), and the e2m1 conversion widens,
// scales two values per instruction (mul.rn.f32x2, the same bits as two __fmul_rn) and merges the nibble pairs with
// byte permutes.  These kernels run at 0.76 instructions per scheduler and cycle (ncu), so instructions are time.
__device__ __forceinline__ void mul2(float a0, float a1, unsigned long long s2, float& r0, float& r1) {
    unsigned long long a, r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(a) : "f"(a0), "f"(a1));
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(s2));
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r0), "=f"(r1) : "l"(r));
}
__device__ __forceinline__ uint32_t pack4(uint32_t b0, uint32_t b1, uint32_t b2, uint32_t b3) {
    return __byte_perm(__byte_perm(b0, b1, 0x0040), __byte_perm(b2, b3, 0x0040), 0x5410);
}
template <typename T>
struct Chunk16 {
    float v[16];
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = 0.f;
    }
    __device__ __forceinline__ void load(const T* p, bool wide) { load16w<T>(p, v, wide); }
    __device__ __forceinline__ float amax() const {
        float m = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) m = fmaxf(m, fabsf(v[i]));
        return m;
    }
    __device__ __forceinline__ uint2 quant_e2m1(float inv) const {
        uint32_t w[2] = {0u, 0u};
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            uint32_t b = cvt_e2m1x2(__fmul_rn(v[2 * i], inv), __fmul_rn(v[2 * i + 1], inv));
            w[i >> 2] |= b << (8 * (i & 3));
        }
        return make_uint2(w[0], w[1]);
    }
    __device__ __forceinline__ void to_float(float (&o)[16]) const {
#pragma unroll
        for (int i = 0; i < 16; ++i) o[i] = v[i];
    }
};
template <>
struct Chunk16<__nv_bfloat16> {
    uint32_t w[8];
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = 0u;
    }
    __device__ __forceinline__ void load(const __nv_bfloat16* p, bool wide) {
        if (wide) {
            ldg256(p, w);
        } else {
            const uint4 a = __ldg(reinterpret_cast<const uint4*>(p)), b = __ldg(reinterpret_cast<const uint4*>(p) + 1);
            w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w; w[4] = b.x; w[5] = b.y; w[6] = b.z; w[7] = b.w;
        }
    }
    // max(|a|, |b|) per half with the signs xor-ed into the result: the magnitude is what the next step looks at, so
    // the eight words chain without masking the signs first (a NaN half yields the other operand, as fmaxf does)
    static __device__ __forceinline__ uint32_t absmax2(uint32_t a, uint32_t b) {
        uint32_t d;
        asm("max.xorsign.abs.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
        return d;
    }
    __device__ __forceinline__ float amax() const {
        const uint32_t m = absmax2(absmax2(absmax2(w[0], w[1]), absmax2(w[2], w[3])),
                                   absmax2(absmax2(w[4], w[5]), absmax2(w[6], w[7]))) & 0x7FFF7FFFu;
        return fmaxf(__uint_as_float(m << 16), __uint_as_float(m & 0xFFFF0000u));
    }
    __device__ __forceinline__ uint2 quant_e2m1(float inv) const {
        unsigned long long s2;
        asm("mov.b64 %0, {%1, %1};" : "=l"(s2) : "f"(inv));
        uint32_t b[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            float lo, hi;
            mul2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xFFFF0000u), s2, lo, hi);
            b[i] = cvt_e2m1x2(lo, hi);
        }
        return make_uint2(pack4(b[0], b[1], b[2], b[3]), pack4(b[4], b[5], b[6], b[7]));
    }
    __device__ __forceinline__ void to_float(float (&o)[16]) const {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            o[2 * i] = __uint_as_float(w[i] << 16);
            o[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
        }
    }
};

template <typename T>
__device__ __forceinline__ float to_f32(T x);
template <> __device__ __forceinline__ float to_f32<float>(float x) { return x; }
template <> __device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }
template <> __device__ __forceinline__ float to_f32<__half>(__half x) { return __half2float(x); }

__device__ __forceinline__ float amax16(const float (&v)[16]) {
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) m = fmaxf(m, fabsf(v[i]));
    return m;
}
// max(amax / 448, 1e-12).  The division is RN(amax * RN(1/448)) plus one residual correction, which equals the IEEE
// quotient for every amax from 2^-100 up (checked exhaustively on the CPU: oracle/quotient_check.c, mode 4); below that
// both are far under 1e-12, and an infinite amax (its residual would be NaN) keeps the infinite first product.
__device__ __forceinline__ float fp8_scale_from_amax(float amax) {
    constexpr float r448 = 0x1.24924ap-9f;                                   // RN(1/448)
    const float q0 = __fmul_rn(amax, r448);
    float s = __fmaf_rn(__fmaf_rn(-q0, 448.0f, amax), r448, q0);
    s = q0 > 3.0e38f ? q0 : s;
    return s < 1e-12f ? 1e-12f : s;
}
// x / s for the E4M3 conversion without a division per element.  With y = RN(1/s) shared by the
// 16 elements, q0 = RN(x*y) is within 2 ulp of the quotient; one residual correction
// (r = x - q*s exactly, by FMA; q' = RN(q + r*y)) brings it within half an ulp plus a sliver, and a
// second one gives the correctly rounded quotient (Markstein's theorem: a faithful q and a correctly
// rounded reciprocal suffice), i.e. the very value __fdiv_rn returns.  The residual is exact unless
// it underflows, which needs |x| < 2^-125; with a scale of at least 1e-12 such a quotient is below
// 2^-85, far under the smallest E4M3 rounding boundary (2^-10), and converts to zero either way.
// Scales the library derives are never smaller; a caller-given scale can be (its reciprocal may even
// overflow), so quant16_e4m3 takes this path only for scales inside [1e-12, 3e38] and divides for
// real otherwise.
// Two values of q0 need care: a zero (the zero residual is +0 and would turn -0 into +0) and an infinity (Inf - Inf
// poisons the residual).  With a scale DERIVED from the maximum of the very elements being divided, |x / s| <= 448 and
// x is never infinite next to a finite scale, so only the zero remains, and since s > 0 the quotient simply takes the
// sign of x (one logic instruction per element; GIVEN = false).  With a scale the caller GIVES, x * y can overflow,
// and both are caught as the fixed points of q -> 2q (GIVEN = true).  A NaN stays a NaN through the corrections.
// Written for two elements at a time with the packed fp32 instructions (mul / fma / add .f32x2: each half is the
// IEEE operation of the scalar form q0 = x*y, q1 = fma(fma(-q0, s, x), y, q0), q2 likewise from q1, and
// fma(-q, s, x) == fma(q, -s, x) bit for bit), which halves the instruction count of the E4M3 quantisers - they run
// close to the issue limit.
template <bool GIVEN>
__device__ __forceinline__ void div2_for_e4m3(float x0, float x1, unsigned long long neg_s2, unsigned long long inv2, float& r0,
                                              float& r1) {
    unsigned long long x, q0, q1, q2, r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(x) : "f"(x0), "f"(x1));
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(q0) : "l"(x), "l"(inv2));
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(q0), "l"(neg_s2), "l"(x));
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(q1) : "l"(r), "l"(inv2), "l"(q0));
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(q1), "l"(neg_s2), "l"(x));
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(q2) : "l"(r), "l"(inv2), "l"(q1));
    float b0, b1;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(b0), "=f"(b1) : "l"(q2));
    if (GIVEN) {
        unsigned long long d;
        asm("add.rn.f32x2 %0, %1, %1;" : "=l"(d) : "l"(q0));
        float a0, a1, d0, d1;
        asm("mov.b64 {%0, %1}, %2;" : "=f"(a0), "=f"(a1) : "l"(q0));
        asm("mov.b64 {%0, %1}, %2;" : "=f"(d0), "=f"(d1) : "l"(d));
        r0 = d0 == a0 ? a0 : b0;
        r1 = d1 == a1 ? a1 : b1;
    } else {
        r0 = __uint_as_float((__float_as_uint(b0) & 0x7FFFFFFFu) | (__float_as_uint(x0) & 0x80000000u));
        r1 = __uint_as_float((__float_as_uint(b1) & 0x7FFFFFFFu) | (__float_as_uint(x1) & 0x80000000u));
    }
}
template <bool GIVEN>
__device__ __forceinline__ uint4 quant16_e4m3(const float (&v)[16], float s) {
    uint32_t w[4];
    if (s >= 1e-12f && s <= 3.0e38f) {
        const float inv = __frcp_rn(s);
        const float ns = -s;
        unsigned long long inv2, neg_s2;
        asm("mov.b64 %0, {%1, %1};" : "=l"(inv2) : "f"(inv));
        asm("mov.b64 %0, {%1, %1};" : "=l"(neg_s2) : "f"(ns));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float a, b, c, d;
            div2_for_e4m3<GIVEN>(v[4 * i], v[4 * i + 1], neg_s2, inv2, a, b);
            div2_for_e4m3<GIVEN>(v[4 * i + 2], v[4 * i + 3], neg_s2, inv2, c, d);
            w[i] = __byte_perm(cvt_e4m3x2(a, b), cvt_e4m3x2(c, d), 0x5410);
        }
    } else {   // an infinite scale (an Inf among the inputs: 0 * Inf would poison the residual), or a given
               // scale too small for the residual argument above (also zero, negative, NaN): divide for real
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t lo = cvt_e4m3x2(__fdiv_rn(v[4 * i], s), __fdiv_rn(v[4 * i + 1], s));
            uint32_t hi = cvt_e4m3x2(__fdiv_rn(v[4 * i + 2], s), __fdiv_rn(v[4 * i + 3], s));
            w[i] = lo | (hi << 16);
        }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ uint2 quant16_e2m1(const float (&v)[16], float inv) {
    uint32_t w[2] = {0u, 0u};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        uint32_t b = cvt_e2m1x2(__fmul_rn(v[2 * i], inv), __fmul_rn(v[2 * i + 1], inv));
        w[i >> 2] |= b << (8 * (i & 3));
    }
    return make_uint2(w[0], w[1]);
}

}  // namespace dsl
