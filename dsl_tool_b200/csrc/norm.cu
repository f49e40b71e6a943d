// Row-wise kernels that end in 8 bits: the root-mean-square norm with the residual's addition, and the int8 quantiser (the same
// kernel without the norm).
//
//   t = round(x + r) to the type of x          (r optional; t is written, and is what the norm reads)
//   y = (t * rsqrt(mean(t^2) + eps)) * w       in fp32, sum of squares in fp32
//   int8:        s = max(amax_row |y| / 127, 1e-12),  q = rne(y / s)
//   FP8 1x128:   s = max(amax_128 |y| / 448, 1e-12),  q = e4m3(y / s)
//   FP8 given:   q = e4m3(y / s) with the caller's s
//   none:        y in the type of x
// q and s are those of the stand-alone quantisers on the fp32 y, bit for bit (quotients are correctly rounded).
//
// Bound by memory: x, r and w are read once, t, q and s written once (8192 x 8192 bf16 with residual: 470 MB, 72 us at the rate of
// a copy, 77 measured in a row of launches on the same few buffers, 83-90 a call on new ones).  One CTA takes a row and keeps it in registers, 16 consecutive elements a thread, so the three looks at it
// (sum of squares, maximum, conversion) cost one trip to memory; a CTA has as many threads as the row has 16-element pieces (a row
// of 4096: 256 threads), and rows beyond 1024 pieces give every thread two.  The reductions over a row are a shuffle tree and one
// meeting in shared memory each.
//
// A NaN anywhere in a row makes an int8 row's scale NaN (an integer cannot carry it): the maximum propagates it, and over the
// block it is taken of bit patterns, where a NaN is above infinity.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <float.h>

#include <atomic>

#include "dslgemm.h"
#include "gemm.cuh"
#include "norm.cuh"
#include "ptx.cuh"
#include "quant_math.cuh"

namespace dsl {

enum { ROW_NONE = 0, ROW_INT8 = 1, ROW_FP8_GROUP = 2, ROW_FP8_GIVEN = 3 };

struct RowArgs {
    const void* x;
    const void* residual;      // type of x, or nullptr
    const void* gain;          // [cols]
    int gain_dtype;
    void* sum_out;             // x + residual, type of x (only with a residual)
    void* out;                 // int8 / E4M3 bytes, or the type of x
    float* scale_out;          // int8 [rows]; FP8 1x128 [rows, ceil(cols / 128)]
    const float* scale_in;     // FP8 given: one float
    float eps;
    long long rows;
    int cols;
    bool wide;                 // rows of x and residual start on 32-byte boundaries
    bool wide_out;             // so do those of sum_out and of a 16-bit out
};

// 16 elements to global memory in the type of x.
template <typename T>
__device__ __forceinline__ void store16(T* p, const float (&v)[16], bool wide) {
    if (sizeof(T) == 4) {
        float4* d = reinterpret_cast<float4*>(p);
#pragma unroll
        for (int i = 0; i < 4; ++i) d[i] = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
    } else {
        uint32_t w[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (dsl_is_half<T>::value) {
                const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
                w[i] = *reinterpret_cast<const uint32_t*>(&h);
            } else {
                const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
                w[i] = *reinterpret_cast<const uint32_t*>(&h);
            }
        }
        if (wide) {      // whole lines a warp: 8192 x 8192 with residual 79.9 -> 76.2 us
            asm volatile("st.global.L1::no_allocate.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};"
                         ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7]) : "memory");
        } else {
            uint4* d = reinterpret_cast<uint4*>(p);
            d[0] = make_uint4(w[0], w[1], w[2], w[3]);
            d[1] = make_uint4(w[4], w[5], w[6], w[7]);
        }
    }
}
template <typename T> __device__ __forceinline__ float round_to(float v);
template <> __device__ __forceinline__ float round_to<float>(float v) { return v; }
template <> __device__ __forceinline__ float round_to<__nv_bfloat16>(float v) { return __bfloat162float(__float2bfloat16_rn(v)); }
template <> __device__ __forceinline__ float round_to<__half>(float v) { return __half2float(__float2half_rn(v)); }

__device__ __forceinline__ void load_gain(const void* gain, int dtype, int at, float (&w)[16]) {
    if (dtype == DSL_F32) load16<float>(static_cast<const float*>(gain) + at, w);
    else if (dtype == DSL_BF16) load16<__nv_bfloat16>(static_cast<const __nv_bfloat16*>(gain) + at, w);
    else load16<__half>(static_cast<const __half*>(gain) + at, w);
}

// 16 quotients y / s to the nearest whole numbers (ties to even), packed.  |y / s| <= 127 by the scale's definition; a row whose
// scale is infinite or NaN gets zeros.  The quotient is the IEEE one: RN(y * RN(1/s)) corrected twice by its residual, as
// div2_for_e4m3 does it and for the reasons given there.  Adding 1.5 * 2^23 rounds it to a whole number whose low byte is the
// result (a conversion instruction runs at a quarter of that rate: norm of 8192 x 8192 bf16 68 -> 63 us).
__device__ __forceinline__ uint4 quant16_int8(const float (&v)[16], float s) {
    if (!(s <= FLT_MAX)) return make_uint4(0u, 0u, 0u, 0u);
    const float inv = __frcp_rn(s), ns = -s, magic = 12582912.0f;
    unsigned long long inv2, neg_s2, magic2;
    asm("mov.b64 %0, {%1, %1};" : "=l"(inv2) : "f"(inv));
    asm("mov.b64 %0, {%1, %1};" : "=l"(neg_s2) : "f"(ns));
    asm("mov.b64 %0, {%1, %1};" : "=l"(magic2) : "f"(magic));
    uint32_t b[16];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        unsigned long long x, q, r;
        asm("mov.b64 %0, {%1, %2};" : "=l"(x) : "f"(v[2 * i]), "f"(v[2 * i + 1]));
        asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(q) : "l"(x), "l"(inv2));
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(q), "l"(neg_s2), "l"(x));
            asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(q) : "l"(r), "l"(inv2));
        }
        asm("add.rn.f32x2 %0, %0, %1;" : "+l"(q) : "l"(magic2));
        asm("mov.b64 {%0, %1}, %2;" : "=r"(b[2 * i]), "=r"(b[2 * i + 1]) : "l"(q));
    }
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = __byte_perm(__byte_perm(b[4 * i], b[4 * i + 1], 0x0040), __byte_perm(b[4 * i + 2], b[4 * i + 3], 0x0040), 0x5410);
    return make_uint4(w[0], w[1], w[2], w[3]);
}
// max(|a|, |b|), a NaN if either is one.
__device__ __forceinline__ float abs_max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(fabsf(a)), "f"(fabsf(b)));
    return r;
}

// max(amax / 127, 1e-12), one IEEE division; a NaN stays one.
__device__ __forceinline__ float int8_scale_from_amax(float amax) {
    const float s = __fdiv_rn(amax, 127.0f);
    return s < 1e-12f ? 1e-12f : s;
}

// All threads of the block: the sum / the largest bit pattern over the block.  `slots`: 32 words of its own for each call, so that
// one barrier a call is enough.
__device__ __forceinline__ float block_sum(float v, float* slots) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
    const int warps = blockDim.x >> 5, lane = threadIdx.x & 31;
    if (warps == 1) return v;
    if (lane == 0) slots[threadIdx.x >> 5] = v;
    __syncthreads();
    v = lane < warps ? slots[lane] : 0.f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
    return v;
}
__device__ __forceinline__ uint32_t block_max(uint32_t v, uint32_t* slots) {
    v = __reduce_max_sync(0xFFFFFFFFu, v);
    const int warps = blockDim.x >> 5, lane = threadIdx.x & 31;
    if (warps == 1) return v;
    if (lane == 0) slots[threadIdx.x >> 5] = v;
    __syncthreads();
    return __reduce_max_sync(0xFFFFFFFFu, lane < warps ? slots[lane] : 0u);
}

// 16 elements as they lie in memory: 8 words of a 16-bit type, 16 of fp32.
template <typename T>
struct Raw16 {
    static constexpr int WORDS = static_cast<int>(sizeof(T)) * 4;
    uint32_t w[WORDS];
    // Ordinary loads, past the L1: sum_out may be x or residual itself, and the non-coherent path is for memory that a kernel does
    // not write.
    __device__ __forceinline__ void load(const T* p, bool wide) {
        if (wide) {
#pragma unroll
            for (int i = 0; i < WORDS; i += 8)
                asm volatile("ld.global.L1::no_allocate.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                             : "=r"(w[i]), "=r"(w[i + 1]), "=r"(w[i + 2]), "=r"(w[i + 3]), "=r"(w[i + 4]), "=r"(w[i + 5]), "=r"(w[i + 6]),
                               "=r"(w[i + 7])
                             : "l"(reinterpret_cast<const uint32_t*>(p) + i));
        } else {
#pragma unroll
            for (int i = 0; i < WORDS; i += 4) {
                const uint4 t = __ldcg(reinterpret_cast<const uint4*>(reinterpret_cast<const uint32_t*>(p) + i));
                w[i] = t.x; w[i + 1] = t.y; w[i + 2] = t.z; w[i + 3] = t.w;
            }
        }
    }
    __device__ __forceinline__ float at(int i) const {
        if (sizeof(T) == 4) return __uint_as_float(w[i]);
        if (dsl_is_half<T>::value) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i / 2]));
            return i & 1 ? f.y : f.x;
        }
        return __uint_as_float(i & 1 ? w[i / 2] & 0xFFFF0000u : w[i / 2] << 16);
    }
};

// PIECES: 16-element pieces a thread holds; piece p of thread i starts at (p * blockDim.x + i) * 16.  A CTA walks rows blockIdx.x,
// + gridDim.x, ...; the next row's loads are issued before this row's meetings (where registers allow it: one piece a thread), so
// that memory is busy while the CTA waits for itself (8192 x 8192 bf16, residual, FP8 groups: 102 us without, 76 with).  A result in
// the type of x waits for one sum only and is faster without (86 / 93 us).
template <typename T, int OUT, bool NORM, int PIECES, int MAX_THREADS>
__global__ void __launch_bounds__(MAX_THREADS, sizeof(T) == 2 ? 1024 / MAX_THREADS : 1) row_kernel(const RowArgs a) {
    constexpr bool AHEAD = OUT != ROW_NONE && PIECES == 1 && (sizeof(T) == 2 || MAX_THREADS <= 512);
    __shared__ float s_sum[2][32];
    __shared__ uint32_t s_max[2][32];
    // Launched as a dependent: placed while the kernel before it drains.  What follows may do the same once that one is complete.
    griddep_wait();
    griddep_launch_dependents();
    const bool with_residual = NORM && a.residual != nullptr;
    Raw16<T> rx[PIECES], rr[PIECES];
    auto fetch = [&](long long row, int p) {
        const int at = (p * blockDim.x + threadIdx.x) * 16;
        if (at < a.cols) {
            rx[p].load(static_cast<const T*>(a.x) + row * a.cols + at, a.wide);
            if (with_residual) rr[p].load(static_cast<const T*>(a.residual) + row * a.cols + at, a.wide);
        }
    };
    if (AHEAD) fetch(blockIdx.x, 0);
    int parity = 0;
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x, parity ^= 1) {
        float v[PIECES][16];
#pragma unroll
        for (int p = 0; p < PIECES; ++p) {
            if (!AHEAD) fetch(row, p);
            const int at = (p * blockDim.x + threadIdx.x) * 16;
            if (at < a.cols) {
#pragma unroll
                for (int i = 0; i < 16; ++i) v[p][i] = rx[p].at(i);
                if (with_residual) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) v[p][i] = round_to<T>(__fadd_rn(v[p][i], rr[p].at(i)));
                    store16<T>(static_cast<T*>(a.sum_out) + row * a.cols + at, v[p], a.wide_out);
                }
            } else {
#pragma unroll
                for (int i = 0; i < 16; ++i) v[p][i] = 0.f;
            }
        }
        if (AHEAD && row + gridDim.x < a.rows) fetch(row + gridDim.x, 0);
        if (NORM) {
            float squares = 0.f;
#pragma unroll
            for (int p = 0; p < PIECES; ++p)
#pragma unroll
                for (int i = 0; i < 16; ++i) squares = fmaf(v[p][i], v[p][i], squares);
            squares = block_sum(squares, s_sum[parity]);
            const float inv = __frsqrt_rn(__fadd_rn(__fdiv_rn(squares, static_cast<float>(a.cols)), a.eps));
#pragma unroll
            for (int p = 0; p < PIECES; ++p) {
                const int at = (p * blockDim.x + threadIdx.x) * 16;
                if (at < a.cols) {
                    float w[16];
                    load_gain(a.gain, a.gain_dtype, at, w);
#pragma unroll
                    for (int i = 0; i < 16; ++i) v[p][i] = __fmul_rn(__fmul_rn(v[p][i], inv), w[i]);
                }
            }
        }
        uint8_t* q = static_cast<uint8_t*>(a.out) + row * a.cols;
        float s = 0.f;
        if (OUT == ROW_INT8) {
            float m = 0.f;
#pragma unroll
            for (int p = 0; p < PIECES; ++p)
#pragma unroll
                for (int i = 0; i < 16; ++i) m = abs_max_nan(m, v[p][i]);
            s = int8_scale_from_amax(__uint_as_float(block_max(__float_as_uint(m), s_max[parity])));
            if (threadIdx.x == 0) a.scale_out[row] = s;
        }
        if (OUT == ROW_FP8_GIVEN) s = *a.scale_in;
#pragma unroll
        for (int p = 0; p < PIECES; ++p) {
            const int at = (p * blockDim.x + threadIdx.x) * 16;
            if (OUT == ROW_FP8_GROUP) {      // eight neighbouring threads hold a group; threads past the row's end hold zeros
                float m = 0.f;
#pragma unroll
                for (int i = 0; i < 16; ++i) m = fmaxf(m, fabsf(v[p][i]));
#pragma unroll
                for (int o = 4; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
                s = fp8_scale_from_amax(m);
                if (at < a.cols && (threadIdx.x & 7) == 0) a.scale_out[row * ((a.cols + 127) / 128) + at / 128] = s;
            }
            if (at < a.cols) {
                if (OUT == ROW_NONE) store16<T>(static_cast<T*>(a.out) + row * a.cols + at, v[p], a.wide_out);
                else if (OUT == ROW_INT8) *reinterpret_cast<uint4*>(q + at) = quant16_int8(v[p], s);
                else *reinterpret_cast<uint4*>(q + at) = quant16_e4m3<OUT == ROW_FP8_GIVEN>(v[p], s);
            }
        }
    }
}

template <typename T, int OUT, bool NORM, int PIECES, int MAX_THREADS>
static cudaError_t launch_threads(const RowArgs& a, int threads, cudaStream_t st) {
    // CTAs an SM holds, by warps a CTA, asked once per device
    static std::atomic<int> resident_of[DSL_MAX_DEVICES][33];
    const int dev = current_device_slot();
    if (dev < 0) return cudaErrorInvalidDevice;
    int resident = resident_of[dev][threads / 32].load(std::memory_order_relaxed);
    if (resident == 0) {
        const cudaError_t e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&resident, row_kernel<T, OUT, NORM, PIECES, MAX_THREADS>, threads, 0);
        if (e != cudaSuccess) return e;
        if (resident < 1) resident = 1;
        resident_of[dev][threads / 32].store(resident, std::memory_order_relaxed);
    }
    const long long ctas = static_cast<long long>(sm_count()) * resident;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(a.rows < ctas ? a.rows : ctas));
    cfg.blockDim = dim3(threads);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, row_kernel<T, OUT, NORM, PIECES, MAX_THREADS>, a);
}

template <typename T, int OUT, bool NORM>
static cudaError_t launch_row(const RowArgs& a, cudaStream_t st) {
    const int pieces = a.cols / 16;
    const int threads = (pieces + 31) / 32 * 32;
    if (threads <= 512) return launch_threads<T, OUT, NORM, 1, 512>(a, threads, st);
    if (threads <= 1024) return launch_threads<T, OUT, NORM, 1, 1024>(a, threads, st);
    return launch_threads<T, OUT, NORM, 2, 1024>(a, ((pieces + 1) / 2 + 31) / 32 * 32, st);
}

template <typename T>
static cudaError_t launch_type(const RowArgs& a, int format, bool norm, cudaStream_t st) {
    if (!norm) return launch_row<T, ROW_INT8, false>(a, st);
    switch (format) {
        case ROW_INT8: return launch_row<T, ROW_INT8, true>(a, st);
        case ROW_FP8_GROUP: return launch_row<T, ROW_FP8_GROUP, true>(a, st);
        case ROW_FP8_GIVEN: return launch_row<T, ROW_FP8_GIVEN, true>(a, st);
        default: return launch_row<T, ROW_NONE, true>(a, st);
    }
}

static cudaError_t launch_dtype(RowArgs& a, int dtype, int format, bool norm, long long rows, cudaStream_t st) {
    a.rows = rows;
    const uintptr_t all = reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.residual);
    a.wide = (all & 31u) == 0;           // a row is a multiple of 16 elements, i.e. of 32 bytes
    a.wide_out = ((reinterpret_cast<uintptr_t>(a.sum_out) | (format == ROW_NONE ? reinterpret_cast<uintptr_t>(a.out) : 0)) & 31u) == 0;
    if (dtype == DSL_F32) return launch_type<float>(a, format, norm, st);
    if (dtype == DSL_BF16) return launch_type<__nv_bfloat16>(a, format, norm, st);
    return launch_type<__half>(a, format, norm, st);
}

cudaError_t launch_quant_int8(const void* x, int dtype, long long rows, int cols, float* scale_out, int8_t* q, cudaStream_t st) {
    RowArgs a{};
    a.x = x;
    a.out = q;
    a.scale_out = scale_out;
    a.cols = cols;
    return launch_dtype(a, dtype, ROW_INT8, false, rows, st);
}

cudaError_t launch_rms_norm(const void* x, int dtype, long long rows, int cols, const void* residual, const void* gain, int gain_dtype,
                            float eps, int out_format, void* sum_out, void* out, float* scale_out, const float* scale_in,
                            cudaStream_t st) {
    RowArgs a{};
    a.x = x;
    a.residual = residual;
    a.gain = gain;
    a.gain_dtype = gain_dtype;
    a.sum_out = sum_out;
    a.out = out;
    a.scale_out = scale_out;
    a.scale_in = scale_in;
    a.eps = eps;
    a.cols = cols;
    static_assert(ROW_NONE == DSL_NORM_NONE && ROW_INT8 == DSL_NORM_INT8 && ROW_FP8_GROUP == DSL_NORM_FP8_GROUP_1X128 &&
                  ROW_FP8_GIVEN == DSL_NORM_FP8_GIVEN, "the header's codes");
    return launch_dtype(a, dtype, out_format, true, rows, st);
}

}  // namespace dsl
