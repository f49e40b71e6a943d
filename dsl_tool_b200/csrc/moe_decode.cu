// A whole mixture-of-experts feed-forward layer for a few tokens, in two kernels:
//
//   up     p, e = softmax top-k of the logits;   h[t, s] = silu(g) * u,  (g, u) = pairs of rows of  Wgu[e(t, s)] x[t]
//   down   y[t, s] = Wdn[e(t, s)] h[t, s];       out[t] = sum over s, in slot order, of p[t, s] * y[t, s]
//
// With one or two rows for each chosen expert the layer is the reading of those experts' weights, so everything is arranged round
// that stream and the activations stay unquantised (nothing would be gained from fewer bits of them).
//
//   * Work is the list of (expert, tile of 16 weight rows) pairs, expert by expert; CTA b of the grid (one an SM) takes the b-th
//     equal share.  The list follows from the logits; every CTA makes it for itself in shared memory (a few hundred
//     nanoseconds), so nothing has to be launched, sorted or copied before.
//   * A CTA keeps the rows of x (or h) that its current expert multiplies in shared memory, as 16-bit values in the order in which
//     the tensor core's B fragments want them.  Weights go from global memory straight into registers (16 warps x 8 loads of 16
//     bytes a lane in flight: 64 KB an SM), are widened there to f16 or bf16, exactly, and meet the rows in mma.sync m16n8k16 with
//     fp32 sums.  The order of K inside a 16-row x 64-byte chunk is free as long as both sides agree: lane (g, t) of a warp holds
//     16 consecutive bytes of weight rows g and g + 8, every load of a warp covers whole 64-byte pieces, and no weight passes
//     through shared memory.  (tcgen05 would want the widened weight written to shared memory first, for tiles of which at most
//     one column in eight is used; the warp-wide instruction runs far below its rate here.)
//   * K of a tile is cut over `split` warps when there are few tiles; their sums meet in shared memory, in order.
//   * Down's results go to scratch by (token, slot); the CTA that delivers a tile's last one adds the slots and writes the output.
//     Which CTA that is changes nothing: it adds in slot order.
//
// Rounding.  Weights are exact in the 16-bit type: E4M3, e2m1 x UE4M3 and int8 in f16, bf16 in bf16; MXFP4's power-of-two scales
// are taken relative to the largest of a chunk's row and applied to its fp32 sum.  x in bf16 or f16 is exact too: for f16 products
// a row is scaled by a power of two that brings its largest value just under 2^15, which leaves every value within 2^-39 of that
// largest one.  An fp32 x and the hidden activation round to 11 bits (f16), or to 16 (two bf16 terms) with bf16 weights - more than
// the 8 bits of the bf16 hidden activation that the layer of quantised GEMMs passes on.  All sums are fp32.
//
// Layer of 64 experts, top 8, K = D = 4096, H = 1536:
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <float.h>

#include <atomic>

#include "dslgemm.h"
#include "gemm.cuh"
#include "ptx.cuh"

namespace dsl {
namespace md {

constexpr int THREADS = 512;
constexpr int WARPS = THREADS / 32;
constexpr int STEP = 256;                // bytes of a weight row that a warp takes at once: 4 chunks of 64
constexpr int MAX_ENTRIES = DSL_MOE_DECODE_MAX_TOKENS * 32;
constexpr int RED_PITCH = 20;            // floats between two columns of a warp's 16-row sums: no bank conflicts on either side

enum { F8 = 0, F8G = 1, I8 = 2, NV = 3, MX = 4, BF = 5 };

template <int FMT>
struct Fmt {
    static constexpr int ELEMS = FMT == NV || FMT == MX ? 32 : (FMT == BF ? 8 : 16);     // in 16 bytes
    static constexpr bool BF16 = FMT == BF;                                              // type of the products
    static constexpr int PARTS = FMT == BF ? 2 : 1;                                      // 16-bit terms of an activation, at most
};

struct Args {
    const void* logits;
    int logits_dtype, tokens, experts, k, renorm;
    const void* x;               // up: [tokens, kdim] of x_dtype; down: h, fp32 [entries, kdim]
    int x_dtype;
    const uint8_t* w;            // [experts, n, row_bytes]
    const uint8_t* scale;        // as the packed weight has it
    const float* global_scale;
    int n, kdim, row_bytes, katoms, tiles, steps, split;
    int block_rows;              // rows of one expert that a CTA holds at a time
    int parts;                   // 16-bit terms an activation (2 only with bf16 products)
    float* h;                    // up: [entries, n / 2]
    float* y;                    // down: [entries, n]
    int* arrived;                // down: one counter a tile, zeroed by up
    int arrived_count;
    void* out;                   // down: [tokens, n]
    int out_dtype;
};

// ---- routing -------------------------------------------------------------------------------------------------------------------
// Shared-memory tables of the list of work: entry = token * k + slot.
struct Plan {
    int* ids;          // [entries] expert, or -1
    float* weights;    // [entries]
    int* order;        // entries sorted by expert, stable
    int* seg_expert;   // [segments]: an expert with at most block_rows of its rows
    int* seg_first;    //             first place in `order`
    int* seg_rows;
    int* count;        // [experts]
    int segments;
};

// Softmax over the experts and the k largest, ties to the lower index; the arithmetic of moe_route_kernel (moe.cu).  A logit of
// minus infinity or NaN is never chosen: an entry without an expert gets -1.  One warp a token, the row in shared memory.
template <typename T>
__device__ __forceinline__ void route_token(const Args& a, int t, float* v, const Plan& p, int lane) {
    const T* row = static_cast<const T*>(a.logits) + static_cast<size_t>(t) * a.experts;
    float mx = -FLT_MAX;
    for (int e = lane; e < a.experts; e += 32) {
        const float f = static_cast<float>(row[e]);
        v[e] = f;
        mx = fmaxf(mx, f);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, o));
    float sum = 0.f;
    for (int e = lane; e < a.experts; e += 32) sum += expf(v[e] - mx);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
    __syncwarp();
    float chosen_p = 0.f, psum = 0.f;
    int chosen_e = -1;
    for (int j = 0; j < a.k; ++j) {
        // order-preserving keys: 0 stands for "not to be chosen"
        uint32_t best = 0u;
        int bi = 0x7FFFFFFF;
        for (int e = lane; e < a.experts; e += 32) {
            const float f = v[e];
            const uint32_t b = __float_as_uint(f + 0.0f);              // one zero
            const uint32_t key = f >= -FLT_MAX ? (b & 0x80000000u ? ~b : b | 0x80000000u) : 0u;
            if (key > best) { best = key; bi = e; }
        }
        const uint32_t top = __reduce_max_sync(0xFFFFFFFFu, best);
        if (top == 0u) break;                                          // uniform: nobody has one left
        const int e = static_cast<int>(__reduce_min_sync(0xFFFFFFFFu, best == top ? static_cast<unsigned>(bi) : 0x7FFFFFFFu));
        const float pr = __fdiv_rn(expf(v[e] - mx), sum);
        psum += pr;
        if (lane == j) { chosen_p = pr; chosen_e = e; }
        __syncwarp();
        if (lane == (e & 31)) v[e] = __uint_as_float(0xFF800000u);     // taken
        __syncwarp();
    }
    if (lane < a.k) {
        p.ids[t * a.k + lane] = chosen_e;
        p.weights[t * a.k + lane] = a.renorm ? __fdiv_rn(chosen_p, psum) : chosen_p;
    }
}

// All threads.  `work`: WARPS * experts floats that nothing else uses yet.
__device__ __forceinline__ void make_plan(const Args& a, Plan& p, float* work, int* s_segments) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int e = threadIdx.x; e < a.experts; e += THREADS) p.count[e] = 0;
    for (int t = warp; t < a.tokens; t += WARPS) {
        if (a.logits_dtype == DSL_F32) route_token<float>(a, t, work + warp * a.experts, p, lane);
        else route_token<__nv_bfloat16>(a, t, work + warp * a.experts, p, lane);
    }
    __syncthreads();
    const int entries = a.tokens * a.k;
    for (int i = threadIdx.x; i < entries; i += THREADS)
        if (p.ids[i] >= 0) atomicAdd(&p.count[p.ids[i]], 1);           // counts: the order of the additions is nobody's business
    __syncthreads();
    if (warp == 0) {
        // experts 32 at a time: where an expert's rows begin, and its segments
        int rows = 0, segments = 0;
        for (int e0 = 0; e0 < a.experts; e0 += 32) {
            const int e = e0 + lane;
            const int c = e < a.experts ? p.count[e] : 0;
            const int b = (c + a.block_rows - 1) / a.block_rows;
            int rc = c, rb = b;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int vc = __shfl_up_sync(0xFFFFFFFFu, rc, o), vb = __shfl_up_sync(0xFFFFFFFFu, rb, o);
                if (lane >= o) { rc += vc; rb += vb; }
            }
            if (e < a.experts) {
                const int first = rows + rc - c;
                p.count[e] = first;                                    // from here on: next free place of the expert
                for (int i = 0; i < b; ++i) {
                    const int s = segments + rb - b + i;
                    p.seg_expert[s] = e;
                    p.seg_first[s] = first + i * a.block_rows;
                    p.seg_rows[s] = min(a.block_rows, c - i * a.block_rows);
                }
            }
            rows += __shfl_sync(0xFFFFFFFFu, rc, 31);
            segments += __shfl_sync(0xFFFFFFFFu, rb, 31);
        }
        __syncwarp();
        for (int i0 = 0; i0 < entries; i0 += 32) {                     // stable: every CTA makes the same list
            const int i = i0 + lane;
            const int e = i < entries ? p.ids[i] : -1;
            const unsigned peers = __match_any_sync(0xFFFFFFFFu, e);
            const int leader = __ffs(peers) - 1;
            int base = 0;
            if (e >= 0 && lane == leader) {
                base = p.count[e];
                p.count[e] = base + __popc(peers);
            }
            base = __shfl_sync(0xFFFFFFFFu, base, leader);
            if (e >= 0) p.order[base + __popc(peers & ((1u << lane) - 1u))] = i;
            __syncwarp();
        }
        if (lane == 0) *s_segments = segments;
    }
    __syncthreads();
    p.segments = *s_segments;
}

// ---- 16-bit products ---------------------------------------------------------------------------------------------------------------
template <bool BF16>
__device__ __forceinline__ void mma16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if (BF16)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t hmul2(uint32_t a, uint32_t b) {
    const __half2 r = __hmul2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
}
// two E4M3 bytes (low 16 bits of w) -> two f16
__device__ __forceinline__ uint32_t widen_e4m3(uint32_t w) {
    uint32_t r;
    asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\t}" : "=r"(r) : "r"(w));
    return r;
}
// byte I of w: two e2m1 nibbles -> two f16 (low nibble in the low half)
template <int I>
__device__ __forceinline__ uint32_t widen_e2m1(uint32_t w) {
    uint32_t r;
    if (I == 0) asm("{\n\t.reg .b8 a, b, c, d;\n\tmov.b32 {a, b, c, d}, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, a;\n\t}" : "=r"(r) : "r"(w));
    else if (I == 1) asm("{\n\t.reg .b8 a, b, c, d;\n\tmov.b32 {a, b, c, d}, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, b;\n\t}" : "=r"(r) : "r"(w));
    else if (I == 2) asm("{\n\t.reg .b8 a, b, c, d;\n\tmov.b32 {a, b, c, d}, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, c;\n\t}" : "=r"(r) : "r"(w));
    else asm("{\n\t.reg .b8 a, b, c, d;\n\tmov.b32 {a, b, c, d}, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, d;\n\t}" : "=r"(r) : "r"(w));
    return r;
}
// two int8 (bytes 0, 1 of w ^ 0x80808080, i.e. value + 128) -> two f16: 0x6400 | u is 1024 + u
__device__ __forceinline__ uint32_t widen_int8(uint32_t biased, uint32_t selector) {
    const uint32_t m = __byte_perm(biased, 0x64646464u, selector);
    const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&m), __half2half2(__ushort_as_half(0x6480)));      // 1024 + 128
    return *reinterpret_cast<const uint32_t*>(&r);
}

__device__ __forceinline__ uint4 load_stream(const uint8_t* p) {
    uint4 r;
    asm volatile("ld.global.nc.L1::no_allocate.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(p));
    return r;
}

// What a lane holds of one step: rows g and g + 8, four chunks, with the scales of its pieces.
template <int FMT>
struct Piece {
    uint4 w[2][4];
    uint32_t s[FMT == NV || FMT == MX ? 2 : 1][FMT == F8G ? 2 : 4];      // NV: two UE4M3 bytes; MX: one E8M0 byte; F8G: fp32 of a 128-group

    __device__ __forceinline__ void load(const Args& a, const uint8_t* row0, const uint8_t* row1, const uint8_t* sc0, const uint8_t* sc1,
                                         int step, int t) {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const int at = step * STEP + c * 64 + t * 16;
            const bool in = at < a.row_bytes;
            w[0][c] = in ? load_stream(row0 + at) : make_uint4(0u, 0u, 0u, 0u);
            w[1][c] = in ? load_stream(row1 + at) : make_uint4(0u, 0u, 0u, 0u);
            if (FMT == NV) {             // blocks 2 * (16-byte piece), + 1: atom piece / 2, bytes (piece % 2) * 2
                const int piece = at >> 4;
                const size_t o = static_cast<size_t>(piece >> 1) * 512 + (piece & 1) * 2;
                s[0][c] = in ? __ldg(reinterpret_cast<const unsigned short*>(sc0 + o)) : 0u;
                s[1][c] = in ? __ldg(reinterpret_cast<const unsigned short*>(sc1 + o)) : 0u;
            }
            if (FMT == MX) {             // block = 16-byte piece
                const int piece = at >> 4;
                const size_t o = static_cast<size_t>(piece >> 2) * 512 + (piece & 3);
                s[0][c] = in ? __ldg(sc0 + o) : 0u;
                s[1][c] = in ? __ldg(sc1 + o) : 0u;
            }
            if (FMT == F8G && c % 2 == 0)      // sc0: this tile's row of block scales
                s[0][c / 2] = in ? __float_as_uint(__ldg(reinterpret_cast<const float*>(sc0) + (step * STEP + c * 64) / 128)) : 0u;
        }
    }
};

// Sums of one step: acc[nt] += weights (16 rows) x the rows in shared memory (columns nt * 8 ...).  `b`: this lane's place in them.
template <int FMT, int NT>
__device__ __forceinline__ void step_products(const Piece<FMT>& p, const uint8_t* const (&b)[NT], int step, int nt_used, int parts, int part_bytes,
                                              float (&acc)[NT][4]) {
    using F = Fmt<FMT>;
    constexpr int VECS = F::ELEMS / 8;                  // 16-byte vectors of activations against one 16-byte piece of weights
    constexpr bool APART = FMT == F8G || FMT == MX;     // chunk sums are scaled before they are added
    float sum[NT][4];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        if (APART && (FMT == MX || c % 2 == 0)) {
#pragma unroll
            for (int i = 0; i < NT; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) sum[i][j] = 0.f;
        }
        uint32_t hs[2][2];           // f16 scales of this lane's blocks (NV: two a piece, MX: one)
        float top[2];                // MX: the chunk's largest scale of either row
        if (FMT == NV) {
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const uint32_t two = widen_e4m3(p.s[r][c]);
                hs[r][0] = __byte_perm(two, two, 0x1010);
                hs[r][1] = __byte_perm(two, two, 0x3232);
            }
        }
        if (FMT == MX) {
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const uint32_t e = p.s[r][c];
                uint32_t m = max(e, __shfl_xor_sync(0xFFFFFFFFu, e, 1));
                m = max(m, __shfl_xor_sync(0xFFFFFFFFu, m, 2));
                // 2^(e - m) in f16: normal down to 2^-14, then 2^-24 at the least, 0 below (under a 2^-24th of the chunk's largest)
                const int d = static_cast<int>(m - e);
                const uint32_t one = d < 15 ? static_cast<uint32_t>(15 - d) << 10 : (d < 25 ? 1u << (24 - d) : 0u);
                hs[r][0] = one | (one << 16);
                // byte 255 is NaN; 2^(m - 127) for m = 0 is subnormal
                top[r] = m == 255u ? __uint_as_float(0x7FC00000u) : __uint_as_float(m == 0u ? 0x00400000u : m << 23);
            }
        }
#pragma unroll
        for (int v = 0; v < VECS; ++v) {
            uint4 x[NT];
#pragma unroll
            for (int i = 0; i < NT; ++i)
                if (i < nt_used) x[i] = *reinterpret_cast<const uint4*>(b[i] + ((step * 4 + c) * VECS + v) * 64);
            uint32_t a[2][2][2];     // [k16 step][row half][k half]
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const uint4 q = p.w[r][c];
                if (FMT == BF) {
                    a[0][r][0] = q.x; a[0][r][1] = q.y; a[1][r][0] = q.z; a[1][r][1] = q.w;
                } else if (FMT == F8 || FMT == F8G) {
                    const uint32_t w0 = v == 0 ? q.x : q.z, w1 = v == 0 ? q.y : q.w;
                    a[0][r][0] = widen_e4m3(w0);
                    a[0][r][1] = widen_e4m3(w0 >> 16);
                    a[1][r][0] = widen_e4m3(w1);
                    a[1][r][1] = widen_e4m3(w1 >> 16);
                } else if (FMT == I8) {
                    const uint32_t w0 = (v == 0 ? q.x : q.z) ^ 0x80808080u, w1 = (v == 0 ? q.y : q.w) ^ 0x80808080u;
                    a[0][r][0] = widen_int8(w0, 0x4140);
                    a[0][r][1] = widen_int8(w0, 0x4342);
                    a[1][r][0] = widen_int8(w1, 0x4140);
                    a[1][r][1] = widen_int8(w1, 0x4342);
                } else {
                    const uint32_t w0 = v == 0 ? q.x : (v == 1 ? q.y : (v == 2 ? q.z : q.w));
                    const uint32_t f = FMT == NV ? hs[r][v / 2] : hs[r][0];
                    a[0][r][0] = hmul2(widen_e2m1<0>(w0), f);
                    a[0][r][1] = hmul2(widen_e2m1<1>(w0), f);
                    a[1][r][0] = hmul2(widen_e2m1<2>(w0), f);
                    a[1][r][1] = hmul2(widen_e2m1<3>(w0), f);
                }
            }
            const uint32_t a0[4] = {a[0][0][0], a[0][1][0], a[0][0][1], a[0][1][1]};
            const uint32_t a1[4] = {a[1][0][0], a[1][1][0], a[1][0][1], a[1][1][1]};
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                if (i < nt_used) {
                    float(&d)[4] = APART ? sum[i] : acc[i];
                    mma16<F::BF16>(d, a0, x[i].x, x[i].y);
                    mma16<F::BF16>(d, a1, x[i].z, x[i].w);
                    if (F::PARTS == 2 && parts == 2) {
                        const uint4 lo = *reinterpret_cast<const uint4*>(b[i] + part_bytes + ((step * 4 + c) * VECS + v) * 64);
                        mma16<F::BF16>(d, a0, lo.x, lo.y);
                        mma16<F::BF16>(d, a1, lo.z, lo.w);
                    }
                }
            }
        }
        if (APART && (FMT == MX || c % 2 == 1)) {
            const float t0 = FMT == MX ? top[0] : __uint_as_float(p.s[0][c / 2]), t1 = FMT == MX ? top[1] : t0;
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                acc[i][0] = fmaf(sum[i][0], t0, acc[i][0]);
                acc[i][1] = fmaf(sum[i][1], t0, acc[i][1]);
                acc[i][2] = fmaf(sum[i][2], t1, acc[i][2]);
                acc[i][3] = fmaf(sum[i][3], t1, acc[i][3]);
            }
        }
    }
}

// ---- a segment's rows into shared memory ----------------------------------------------------------------------------------------------
__device__ __forceinline__ void load8(const void* x, int dtype, size_t at, float (&f)[8]) {
    if (dtype == DSL_F32) {
        const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(x) + at);
        const float4 u = __ldcg(p), v = __ldcg(p + 1);      // the hidden activation is the kernel before's: past the L1
        f[0] = u.x; f[1] = u.y; f[2] = u.z; f[3] = u.w; f[4] = v.x; f[5] = v.y; f[6] = v.z; f[7] = v.w;
        return;
    }
    const uint4 u = __ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(x) + at));
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (dtype == DSL_BF16) {
            f[2 * i] = __uint_as_float(w[i] << 16);
            f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
        } else {
            const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
            f[2 * i] = h.x;
            f[2 * i + 1] = h.y;
        }
    }
}

// Power of two that brings a row whose largest magnitude has the bits `amax` just under 2^15, and its inverse.  Rows of zeros,
// infinities and NaN (which stay what they are) come out finite too.
__device__ __forceinline__ float row_factor(uint32_t amax, float* inverse) {
    const int e = static_cast<int>(amax >> 23) - 127;                 // -127 for zero and subnormals
    const int s = max(-126, min(126, 14 - e));
    *inverse = __uint_as_float(static_cast<uint32_t>(127 - s) << 23);
    return __uint_as_float(static_cast<uint32_t>(127 + s) << 23);
}

// Rows seg_first .. + rows of the list; element j of a row lies in chunk j / (4 E), lane t = j / E % 4, vector j % E / 8, i.e. at
// ((chunk * E / 8 + vector) * 4 + t) * 16 bytes.  Elements past the row's end up to whole steps are zeros.
template <int FMT, bool DOWN>
__device__ __forceinline__ void stage_rows(const Args& a, const Plan& p, int first, int rows, uint8_t* dst, int pitch, int part_bytes,
                                           uint32_t* s_amax, float* s_inverse) {
    using F = Fmt<FMT>;
    constexpr int VECS = F::ELEMS / 8;
    const int vectors = a.steps * (STEP / 16) * VECS;                 // 8-element vectors of a padded row
    const int dtype = DOWN ? DSL_F32 : a.x_dtype;
    auto source = [&](int r) {
        const int entry = p.order[first + r];
        return static_cast<size_t>(DOWN ? entry : entry / a.k) * a.kdim;
    };
    // f16 rows are what they are, bf16 ones as bf16 too; the second bf16 term of an fp32 value wants room below the first
    const bool scaled = dtype == DSL_F32 || (dtype == DSL_BF16 && !F::BF16);
    if (threadIdx.x < rows) {
        s_amax[threadIdx.x] = 0u;
        s_inverse[threadIdx.x] = 1.0f;
    }
    __syncthreads();
    if (scaled) {
        for (int r = 0; r < rows; ++r) {
            const size_t src = source(r);
            uint32_t m = 0u;
            for (int v = threadIdx.x; v * 8 < a.kdim; v += THREADS) {
                float f[8];
                load8(a.x, dtype, src + v * 8, f);
#pragma unroll
                for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(f[i]) & 0x7FFFFFFFu);
            }
            m = __reduce_max_sync(0xFFFFFFFFu, m);
            if ((threadIdx.x & 31) == 0 && m != 0u) atomicMax(&s_amax[r], m);
        }
        __syncthreads();
    }
    for (int r = 0; r < rows; ++r) {
        const size_t src = source(r);
        float inverse = 1.0f;
        const float factor = scaled ? row_factor(s_amax[r], &inverse) : 1.0f;
        if (scaled && threadIdx.x == 0) s_inverse[r] = inverse;
        for (int v = threadIdx.x; v < vectors; v += THREADS) {
            float f[8];
            if (v * 8 < a.kdim) {
                load8(a.x, dtype, src + v * 8, f);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) f[i] = 0.f;
            }
            const int piece = v / VECS;
            uint8_t* d = dst + static_cast<size_t>(r) * pitch + (((piece >> 2) * VECS + v % VECS) * 4 + (piece & 3)) * 16;
            uint32_t w[4], lo[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (F::BF16) {
                    const float f0 = f[2 * i] * factor, f1 = f[2 * i + 1] * factor;
                    const __nv_bfloat162 hi = __floats2bfloat162_rn(f0, f1);
                    const float h0 = __low2float(hi), h1 = __high2float(hi);       // an infinity leaves no rest
                    const __nv_bfloat162 rest = __floats2bfloat162_rn(isinf(h0) ? 0.f : f0 - h0, isinf(h1) ? 0.f : f1 - h1);
                    w[i] = *reinterpret_cast<const uint32_t*>(&hi);
                    lo[i] = *reinterpret_cast<const uint32_t*>(&rest);
                } else {
                    const __half2 h = __floats2half2_rn(f[2 * i] * factor, f[2 * i + 1] * factor);
                    w[i] = *reinterpret_cast<const uint32_t*>(&h);
                }
            }
            *reinterpret_cast<uint4*>(d) = make_uint4(w[0], w[1], w[2], w[3]);
            if (F::PARTS == 2 && a.parts == 2) *reinterpret_cast<uint4*>(d + part_bytes) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
        }
    }
    __syncthreads();
}

// ---- shared memory ----------------------------------------------------------------------------------------------------------------
struct Layout {
    int ids, weights, order, seg_expert, seg_first, seg_rows, count, misc, red, rows, total;
    int pitch, part_bytes;
};
// `elems`: elements of a weight in 16 bytes; the rows' region doubles as the router's room.
__host__ __device__ inline Layout layout_of(const Args& a, int elems, int nt) {
    Layout l;
    const int entries = a.tokens * a.k;
    int at = 0;
    auto take = [&](int bytes) { const int here = at; at += (bytes + 15) / 16 * 16; return here; };
    l.ids = take(entries * 4);
    l.weights = take(entries * 4);
    l.order = take(entries * 4);
    l.seg_expert = take(entries * 4);
    l.seg_first = take(entries * 4);
    l.seg_rows = take(entries * 4);
    l.count = take(a.experts * 4);
    l.misc = take(32 + 32 * 8);                                        // segments, flags; amax and inverse factor of 16 rows
    l.red = take(2 * WARPS * nt * 8 * RED_PITCH * 4);
    l.part_bytes = a.steps * (STEP / 16) * elems * 2;                  // a multiple of 256
    l.pitch = l.part_bytes * a.parts + 64;                             // two rows start half a bank round apart
    l.rows = take(0);
    const int rows = a.block_rows * l.pitch, room = WARPS * a.experts * 4;
    l.total = l.rows + (rows > room ? rows : room);
    return l;
}

__device__ __forceinline__ void group_sync(int group, int split) {
    if (split == 1) __syncwarp();
    else asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "r"(split * 32) : "memory");
}

}  // namespace md

template <int FMT, int NT, bool DOWN>
__global__ void __launch_bounds__(md::THREADS, 1) moe_decode_kernel(const md::Args a) {
    using F = md::Fmt<FMT>;
    using md::THREADS;
    using md::WARPS;
    extern __shared__ __align__(16) uint8_t smem[];
    const md::Layout l = md::layout_of(a, F::ELEMS, NT);
    md::Plan plan;
    plan.ids = reinterpret_cast<int*>(smem + l.ids);
    plan.weights = reinterpret_cast<float*>(smem + l.weights);
    plan.order = reinterpret_cast<int*>(smem + l.order);
    plan.seg_expert = reinterpret_cast<int*>(smem + l.seg_expert);
    plan.seg_first = reinterpret_cast<int*>(smem + l.seg_first);
    plan.seg_rows = reinterpret_cast<int*>(smem + l.seg_rows);
    plan.count = reinterpret_cast<int*>(smem + l.count);
    int* s_misc = reinterpret_cast<int*>(smem + l.misc);
    uint32_t* s_amax = reinterpret_cast<uint32_t*>(smem + l.misc + 32);
    float* s_inverse = reinterpret_cast<float*>(smem + l.misc + 32 + 64);
    float* s_red = reinterpret_cast<float*>(smem + l.red);
    uint8_t* s_rows = smem + l.rows;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2, t4 = lane & 3;
    if (!DOWN) {
        // Launched as a dependent, and lets its own successor be placed once everything before it is complete.
        griddep_wait();
        griddep_launch_dependents();
        if (blockIdx.x == 0)
            for (int i = threadIdx.x; i < a.arrived_count; i += THREADS) a.arrived[i] = 0;
    }
    // Down may get this far while up still runs: logits and weights were complete before up started.
    md::make_plan(a, plan, reinterpret_cast<float*>(s_rows), s_misc);
    const long long items = static_cast<long long>(plan.segments) * a.tiles;
    const long long begin = items * blockIdx.x / gridDim.x, end = items * (blockIdx.x + 1) / gridDim.x;

    const int groups = WARPS / a.split, group = warp / a.split, slice = warp - group * a.split;
    const int my_steps = (a.steps - slice + a.split - 1) / a.split;
    float* red = s_red + warp * (NT * 8 * md::RED_PITCH);
    const float* red_group = s_red + group * a.split * (NT * 8 * md::RED_PITCH);
    constexpr int RED_ALL = WARPS * NT * 8 * md::RED_PITCH;
    int parity = 0;
    bool waited = !DOWN;

    for (long long item = begin; item < end;) {
        const int seg = static_cast<int>(item / a.tiles);
        const int tile0 = static_cast<int>(item - static_cast<long long>(seg) * a.tiles);
        const int tile1 = static_cast<int>(min(static_cast<long long>(a.tiles), tile0 + (end - item)));
        const int expert = plan.seg_expert[seg], first = plan.seg_first[seg], rows = plan.seg_rows[seg];
        item += tile1 - tile0;

        // this warp's tiles: tile0 + group, + groups, ...; a tile's steps: slice, + split, ...
        int tile = tile0 + group, step = slice;
        const uint8_t *row0, *row1, *sc0 = nullptr, *sc1 = nullptr;
        auto locate = [&]() {
            const int r0 = min(tile * 16 + g, a.n - 1), r1 = min(tile * 16 + g + 8, a.n - 1);       // rows past the end: any that exist
            row0 = a.w + (static_cast<size_t>(expert) * a.n + r0) * a.row_bytes;
            row1 = a.w + (static_cast<size_t>(expert) * a.n + r1) * a.row_bytes;
            if (FMT == md::NV || FMT == md::MX) {
                const size_t t128 = static_cast<size_t>(expert) * ((a.n + 127) / 128);
                sc0 = a.scale + (t128 + r0 / 128) * a.katoms * 512 + (r0 % 32) * 16 + (r0 % 128) / 32 * 4;
                sc1 = a.scale + (t128 + r1 / 128) * a.katoms * 512 + (r1 % 32) * 16 + (r1 % 128) / 32 * 4;
            }
            if (FMT == md::F8G)
                sc0 = a.scale + (static_cast<size_t>(expert) * ((a.n + 127) / 128) + tile / 8) * (a.kdim / 128) * 4;
        };
        // moves on to this warp's next step; false past the last one
        auto advance = [&](int& tl, int& st) {
            st += a.split;
            if (st >= a.steps) { st = slice; tl += groups; }
            return tl < tile1;
        };
        md::Piece<FMT> even, odd;
        bool more = tile < tile1 && my_steps > 0;
        if (more) {
            locate();
            even.load(a, row0, row1, sc0, sc1, step, t4);
        }
        if (!waited) {           // the hidden activation is up's
            griddep_wait();
            griddep_launch_dependents();
            waited = true;
        }
        __syncthreads();         // the rows of the segment before are read, the router's room is free
        md::stage_rows<FMT, DOWN>(a, plan, first, rows, s_rows, l.pitch, l.part_bytes, s_amax, s_inverse);
        const int nt_used = NT == 1 ? 1 : (rows + 7) / 8;
        const uint8_t* b[NT];
#pragma unroll
        for (int i = 0; i < NT; ++i) b[i] = s_rows + static_cast<size_t>(min(i * 8 + g, rows - 1)) * l.pitch + t4 * 16;
        float acc[NT][4];
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[i][j] = 0.f;

        // the sums of a finished tile: over the group's warps, in order, then scales and the activation
        auto finish = [&](int done) {
            float* mine = red + parity * RED_ALL;
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                if (i < nt_used) {
                    float* c = mine + (i * 8 + 2 * t4) * md::RED_PITCH + g;
                    c[0] = acc[i][0];
                    c[md::RED_PITCH] = acc[i][1];
                    c[8] = acc[i][2];
                    c[md::RED_PITCH + 8] = acc[i][3];
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = 0.f;
            }
            md::group_sync(group, a.split);
            const float* theirs = red_group + parity * RED_ALL;
            parity ^= 1;
            auto total = [&](int col, int row) {
                float s = 0.f;
                for (int w = 0; w < a.split; ++w) s += theirs[w * (NT * 8 * md::RED_PITCH) + col * md::RED_PITCH + row];
                s *= s_inverse[col];
                if (FMT == md::F8) s *= *reinterpret_cast<const float*>(a.scale);
                if (FMT == md::NV) s *= *a.global_scale;
                if (FMT == md::I8) s *= reinterpret_cast<const float*>(a.scale)[static_cast<size_t>(expert) * a.n + min(done * 16 + row, a.n - 1)];
                return s;
            };
            const int me = slice * 32 + lane, all = a.split * 32;
            if (DOWN) {
                for (int i = me; i < rows * 16; i += all) {
                    const int col = i >> 4, row = i & 15;
                    if (done * 16 + row < a.n) a.y[static_cast<size_t>(plan.order[first + col]) * a.n + done * 16 + row] = total(col, row);
                }
            } else {
                for (int i = me; i < rows * 8; i += all) {
                    const int col = i >> 3, j = i & 7;
                    if (done * 16 + 2 * j + 1 < a.n) {
                        const float gate = total(col, 2 * j), up = total(col, 2 * j + 1);
                        a.h[static_cast<size_t>(plan.order[first + col]) * (a.n / 2) + done * 8 + j] =
                            __fmul_rn(__fdiv_rn(gate, 1.0f + expf(-gate)), up);
                    }
                }
            }
        };
        // two steps at a time, so that the two sets of registers keep their names
        while (more) {
            int tl = tile, st = step;
            bool next = advance(tl, st);
            if (next) {
                const int was = tile;
                tile = tl;
                if (tl != was) locate();
                odd.load(a, row0, row1, sc0, sc1, st, t4);
                tile = was;
            }
            md::step_products<FMT, NT>(even, b, step, nt_used, a.parts, l.part_bytes, acc);
            if (!next || tl != tile) finish(tile);
            tile = tl;
            step = st;
            if (!next) break;
            more = advance(tl, st);
            if (more) {
                const int was = tile;
                tile = tl;
                if (tl != was) locate();
                even.load(a, row0, row1, sc0, sc1, st, t4);
                tile = was;
            }
            md::step_products<FMT, NT>(odd, b, step, nt_used, a.parts, l.part_bytes, acc);
            if (!more || tl != tile) finish(tile);
            tile = tl;
            step = st;
        }
    }

    if (DOWN) {
        if (!waited) {           // a CTA without work: the counters and the output are still up's
            griddep_wait();
            griddep_launch_dependents();
        }
        // Every result of this CTA is in memory before it counts itself in.
        __threadfence();
        __syncthreads();
        int* s_last = reinterpret_cast<int*>(s_rows);               // flags of the tiles that this CTA completes
        const long long mine = end - begin;
        for (long long i = threadIdx.x; i < a.tiles; i += THREADS) s_last[i] = 0;
        __syncthreads();
        for (long long i = threadIdx.x; i < mine; i += THREADS) {
            const int tile = static_cast<int>((begin + i) % a.tiles);
            if (atomicAdd(&a.arrived[tile], 1) == plan.segments - 1) s_last[tile] = 1;
        }
        __syncthreads();
        __threadfence();
        // with no entry at all (every logit masked) nobody counts: the CTAs share the zeros
        const bool none = plan.segments == 0;
        for (int tile = none ? blockIdx.x : 0; tile < a.tiles; tile += none ? gridDim.x : 1) {
            if (!none && s_last[tile] == 0) continue;
            for (int i = threadIdx.x; i < a.tokens * 16; i += THREADS) {
                const int t = i >> 4, col = tile * 16 + (i & 15);
                if (col >= a.n) continue;
                float s = 0.f;
                for (int j = 0; j < a.k; ++j) {
                    const int entry = t * a.k + j;
                    if (plan.ids[entry] >= 0) s = fmaf(plan.weights[entry], __ldcg(a.y + static_cast<size_t>(entry) * a.n + col), s);
                }
                const size_t at = static_cast<size_t>(t) * a.n + col;
                if (a.out_dtype == DSL_BF16) static_cast<__nv_bfloat16*>(a.out)[at] = __float2bfloat16_rn(s);
                else static_cast<float*>(a.out)[at] = s;
            }
        }
    }
}

// ---- host side -------------------------------------------------------------------------------------------------------------------
namespace md {

constexpr int SMEM_LIMIT = 227 * 1024;

// Rows an expert's CTA may hold, K cut and shared memory; false when not even one row fits.
static bool plan_launch(Args& a, int elems, int nt, int sms, int* smem_bytes) {
    a.tiles = (a.n + 15) / 16;
    a.steps = (a.row_bytes + STEP - 1) / STEP;
    a.block_rows = 1;
    const int most = a.tokens < nt * 8 ? a.tokens : nt * 8;
    for (int r = 1; r <= most; ++r) {
        Args t = a;
        t.block_rows = r;
        const Layout l = layout_of(t, elems, nt);
        if (l.total > SMEM_LIMIT) {
            if (r == 1) return false;
            break;
        }
        a.block_rows = r;
        *smem_bytes = l.total;
    }
    // flags of the finished tiles share the rows' region
    const int flags = layout_of(a, elems, nt).rows + a.tiles * 4;
    if (flags > SMEM_LIMIT) return false;
    if (flags > *smem_bytes) *smem_bytes = flags;
    // Warps on one tile: enough of them that each of a CTA's groups has about four tiles to run through, never more than steps.
    // Tiles a CTA: of the experts that `tokens` random choices reach on average.
    double miss = 1.0;
    for (int i = 0; i < a.tokens; ++i) miss *= 1.0 - static_cast<double>(a.k) / a.experts;
    const double per_cta = a.experts * (1.0 - miss) * a.tiles / sms;
    int split = 1;
    while (split < WARPS && split * 2 <= a.steps && per_cta * split < 4.0 * WARPS) split *= 2;
    a.split = split;
    return true;
}

template <int FMT, int NT, bool DOWN>
static int launch_one(const Args& a, int smem_bytes, int sms, cudaStream_t st) {
    static PerDeviceInt attr_set;   // per device; idempotent, a race here only repeats the same call
    const int dev = current_device_slot();
    if (dev < 0) return static_cast<int>(cudaErrorInvalidDevice);
    if (attr_set.v[dev].load(std::memory_order_acquire) == 0) {
        const cudaError_t e = cudaFuncSetAttribute(moe_decode_kernel<FMT, NT, DOWN>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_LIMIT);
        if (e != cudaSuccess) return static_cast<int>(e);
        attr_set.v[dev].store(1, std::memory_order_release);
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(sms));
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = smem_bytes;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return static_cast<int>(cudaLaunchKernelEx(&cfg, moe_decode_kernel<FMT, NT, DOWN>, a));
}

static Args side(const dsl_weight* w, int tokens, int k, int x_dtype) {
    Args a{};
    a.tokens = tokens;
    a.experts = w->groups;
    a.k = k;
    a.x_dtype = x_dtype;
    a.w = static_cast<const uint8_t*>(w->q);
    a.scale = static_cast<const uint8_t*>(w->scale);
    a.global_scale = w->global_scale;
    a.n = w->n;
    a.kdim = w->k;
    const bool fp4 = w->format == DSL_W_NVFP4 || w->format == DSL_W_MXFP4;
    a.row_bytes = fp4 ? w->k / 2 : (w->format == DSL_W_BF16 ? 2 * w->k : w->k);
    a.katoms = fp4 ? (w->k / (w->format == DSL_W_NVFP4 ? 16 : 32) + 3) / 4 : 0;
    a.parts = w->format == DSL_W_BF16 && x_dtype != DSL_BF16 ? 2 : 1;
    return a;
}

template <int FMT>
static int launch_fmt(Args& up, Args& down, int sms, cudaStream_t st) {
    const int nt = up.tokens > 8 ? 2 : 1;
    int bytes_up = 0, bytes_down = 0;
    if (!plan_launch(up, Fmt<FMT>::ELEMS, nt, sms, &bytes_up) || !plan_launch(down, Fmt<FMT>::ELEMS, nt, sms, &bytes_down))
        return DSL_ERR_TOO_LARGE;
    up.arrived_count = down.tiles;
    int rc = nt == 1 ? launch_one<FMT, 1, false>(up, bytes_up, sms, st) : launch_one<FMT, 2, false>(up, bytes_up, sms, st);
    if (rc != 0) return rc;
    return nt == 1 ? launch_one<FMT, 1, true>(down, bytes_down, sms, st) : launch_one<FMT, 2, true>(down, bytes_down, sms, st);
}

static int elems_of(int format) { return format == DSL_W_NVFP4 || format == DSL_W_MXFP4 ? 32 : (format == DSL_W_BF16 ? 8 : 16); }

// What the entry point takes; 0 or DSL_ERR_*.
static int check(const dsl_weight* gu, const dsl_weight* dn, int tokens, int k, int x_dtype) {
    if (gu == nullptr || dn == nullptr) return DSL_ERR_NULL;
    if (gu->format != dn->format || gu->format < DSL_W_FP8 || gu->format > DSL_W_INT8) return DSL_ERR_ENUM;
    if (x_dtype < DSL_F32 || x_dtype > DSL_F16) return DSL_ERR_ENUM;
    if (gu->groups < 1 || gu->groups > DSL_MAX_GROUPS || gu->groups != dn->groups || gu->n <= 0 || gu->n % 2 != 0 || dn->k != gu->n / 2 ||
        gu->k <= 0 || dn->n <= 0)
        return DSL_ERR_SHAPE;
    const bool fp4 = gu->format == DSL_W_NVFP4 || gu->format == DSL_W_MXFP4;
    const int multiple = fp4 ? 32 : (gu->format == DSL_W_FP8_BLOCK128 ? 128 : (gu->format == DSL_W_BF16 ? 8 : 16));
    if (gu->k % multiple != 0 || dn->k % multiple != 0) return DSL_ERR_SHAPE;
    if (tokens < 0 || k < 1 || k > 32 || k > gu->groups) return DSL_ERR_SHAPE;
    if (tokens > DSL_MOE_DECODE_MAX_TOKENS) return DSL_ERR_TOO_LARGE;
    // rows that a CTA cannot hold, or sizes that 32-bit offsets inside a row or a tile table could not take
    if (gu->k > (1 << 20) || dn->k > (1 << 20) || dn->n > (1 << 20)) return DSL_ERR_TOO_LARGE;
    if (tokens > 0) {
        int bytes;
        for (int i = 0; i < 2; ++i) {
            Args a = side(i == 0 ? gu : dn, tokens, k, i == 0 ? x_dtype : DSL_F32);
            if (!plan_launch(a, elems_of(gu->format), tokens > 8 ? 2 : 1, 148, &bytes)) return DSL_ERR_TOO_LARGE;
        }
    }
    return 0;
}

static size_t up256(size_t v) { return (v + 255) / 256 * 256; }

}  // namespace md
}  // namespace dsl

using namespace dsl;

extern "C" size_t dsl_moe_decode_scratch_bytes(const dsl_weight* gate_up, const dsl_weight* down, int tokens, int k, int x_dtype) {
    if (md::check(gate_up, down, tokens, k, x_dtype) != 0 || tokens == 0) return 0;
    const size_t entries = static_cast<size_t>(tokens) * k;
    return md::up256(entries * down->k * 4) + md::up256(entries * down->n * 4) + md::up256((down->n + 15) / 16 * 4ull);
}

extern "C" int dsl_moe_decode(const void* x, int x_dtype, const void* logits, int logits_dtype, int tokens, int k, int renorm,
                              const dsl_weight* gate_up, const dsl_weight* down, void* scratch, size_t scratch_bytes, void* out,
                              int out_dtype, void* stream) {
    int rc = md::check(gate_up, down, tokens, k, x_dtype);
    if (rc != 0) return rc;
    if (logits_dtype != DSL_F32 && logits_dtype != DSL_BF16) return DSL_ERR_ENUM;
    if (out_dtype != DSL_F32 && out_dtype != DSL_BF16) return DSL_ERR_ENUM;
    if (tokens == 0) return 0;
    const int format = gate_up->format;
    if (x == nullptr || logits == nullptr || out == nullptr || scratch == nullptr || gate_up->q == nullptr || down->q == nullptr)
        return DSL_ERR_NULL;
    if (format != DSL_W_BF16 && (gate_up->scale == nullptr || down->scale == nullptr)) return DSL_ERR_NULL;
    if (format == DSL_W_NVFP4 && (gate_up->global_scale == nullptr || down->global_scale == nullptr)) return DSL_ERR_NULL;
    const uintptr_t vectors = reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(gate_up->q) | reinterpret_cast<uintptr_t>(down->q);
    const uintptr_t words = reinterpret_cast<uintptr_t>(gate_up->scale) | reinterpret_cast<uintptr_t>(down->scale);
    if ((vectors & 15u) != 0 || (words & 3u) != 0 || (reinterpret_cast<uintptr_t>(scratch) & 255u) != 0) return DSL_ERR_ALIGN;
    if (scratch_bytes < dsl_moe_decode_scratch_bytes(gate_up, down, tokens, k, x_dtype)) return DSL_ERR_TOO_LARGE;
    md::Args up = md::side(gate_up, tokens, k, x_dtype), dn = md::side(down, tokens, k, DSL_F32);
    const size_t entries = static_cast<size_t>(tokens) * k;
    uint8_t* base = static_cast<uint8_t*>(scratch);
    float* h = reinterpret_cast<float*>(base);
    float* y = reinterpret_cast<float*>(base + md::up256(entries * down->k * 4));
    int* arrived = reinterpret_cast<int*>(base + md::up256(entries * down->k * 4) + md::up256(entries * down->n * 4));
    for (md::Args* a : {&up, &dn}) {
        a->logits = logits;
        a->logits_dtype = logits_dtype;
        a->renorm = renorm;
        a->arrived = arrived;
    }
    up.x = x;
    up.h = h;
    dn.x = h;
    dn.y = y;
    dn.out = out;
    dn.out_dtype = out_dtype;
    const int sms = sm_count();
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    switch (format) {
        case DSL_W_FP8: return md::launch_fmt<md::F8>(up, dn, sms, st);
        case DSL_W_FP8_BLOCK128: return md::launch_fmt<md::F8G>(up, dn, sms, st);
        case DSL_W_INT8: return md::launch_fmt<md::I8>(up, dn, sms, st);
        case DSL_W_NVFP4: return md::launch_fmt<md::NV>(up, dn, sms, st);
        case DSL_W_MXFP4: return md::launch_fmt<md::MX>(up, dn, sms, st);
        default: return md::launch_fmt<md::BF>(up, dn, sms, st);
    }
}
