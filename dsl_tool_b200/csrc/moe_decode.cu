// A whole mixture-of-experts feed-forward layer for a few tokens, in three kernels:
//
//   up       p, e = softmax top-k of the logits;   h[t, s] = silu(g) * u,  (g, u) = pairs of rows of  Wgu[e(t, s)] x[t]
//   down     y[t, s] = Wdn[e(t, s)] h[t, s]
//   combine  out[t] = sum over s, in slot order, of p[t, s] * y[t, s]
//
// With one or two rows for each chosen expert the layer is the reading of those experts' weights, so everything is arranged round
// that stream and the activations stay unquantised (nothing would be gained from fewer bits of them).
//
//   * Work is the list of (expert, unit of 16 weight rows) pairs, expert by expert; CTA b of the grid (one an SM) takes the b-th
//     equal share.  The list follows from the logits; every CTA makes it for itself in shared memory, so nothing has to be launched,
//     sorted or copied before.
//   * Two units make a tile of 32 rows, {q * 8 + g + 32 j : g < 8, j < 4} of a block of 128: the rows whose FP4 scale bytes lie
//     side by side, so that one 16-byte load brings a lane the scales of all its rows.  A step is 64 bytes of a tile's rows.
//   * A CTA's steps, tile after tile, are dealt to its 16 warps in equal runs.  A tile that lies inside a run is finished by its
//     warp; the pieces of the others meet in shared memory after the last step and are added in order.
//   * The rows of x (or h) that the current expert multiplies are kept in shared memory, as 16-bit values in the order in which the
//     tensor core's B fragments want them.  Weights go from global memory straight into registers (two steps of four 16-byte loads
//     a lane in flight while a third is multiplied: 64 KB an SM; three, or a ring in shared memory, gained nothing), are widened
//     there to f16 or bf16, exactly, and meet the rows in mma.sync m16n8k16 with fp32 sums.  The order of K inside a step is free as
//     long as both sides agree: lane (g, t) of a warp holds 16 consecutive bytes of its four rows, every load covers whole 64-byte
//     pieces, and no weight passes through shared memory.  (tcgen05 would want the widened weight written to shared memory first,
//     for tiles of which at most one column in eight is used.  The products and the widening are not what bounds: without either,
//     8 tokens NVFP4 took 102 us a layer instead of 111.)
//   * Code that runs once a launch is kept small (loops not unrolled): its instructions come from memory, behind the weights, and
//     unrolled by the compiler they were two thirds of a kernel (8 tokens NVFP4 102 -> 97 us a layer, FP8 145 -> 141).
//   * The loads in flight live in the L1, so the kernels ask for as little shared memory as they can do with: with the largest
//     share of it 8 tokens FP8 took 184 us a layer instead of 142, and kernels that want different shares slow each other
//     (3 tokens BF16 400 -> 278).
//
// Rounding.  Weights are exact in the 16-bit type: E4M3, e2m1 (x UE4M3) and int8 in f16, bf16 in bf16; FP4 scales that meet the sum
// of a block instead do so in fp32.  For f16 products a row whose largest magnitude lies in [1, 2^15) is taken as it is: 16-bit
// values are exact down to 2^-17, off by 2^-25 at most below.  Other rows are scaled by a power of two that brings the largest just
// under 2^15, which leaves every 16-bit value within 2^-39 of that one.  What has more bits than one 16-bit value holds:
//   * x in fp32: x and the hidden activation are two f16 terms each, 22 bits (values below 2^-3 to 2^-25, as above); the caller asks
//     for fp32 by giving it, and pays for the second products: 8 tokens FP8 128x128 141 -> 146 us, INT8 143 -> 146, NVFP4 95 -> 120,
//     one token NVFP4 33 -> 38, MXFP4 33 -> 36, 16 tokens MXFP4 129 -> 187.
//   * x in 16 bits: the hidden activation rounds to f16's 11 bits - three more than bf16, the type that such a model's layers and the
//     layer of quantised GEMMs pass it on in.
//   * bf16 weights: the hidden activation, and an x that is not bf16, are two bf16 terms, 16 bits.
// All sums are fp32.
//
// Layer of 64 experts, top 8, K = D = 4096, H = 1536, weights cold, us a call (share of the rate at which the chosen experts' bytes
// can be copied): one token NVFP4 34 (38 %), FP8 40 (58 %); 8 tokens NVFP4 98 (72 %), FP8 128x128 132-146 (83-90 %, by the experts
// chosen and the GPU); 16 tokens NVFP4 129 (73 %).  8 experts, top 2, H = 14336, 3 tokens BF16 294 (85 %).  What is left: about 18 us
// of a layer in which nothing streams (a kernel's start, routing and list 4 us and the first rows 2 us, of up and of down; the last
// sums), and CTAs that wait for the slowest.
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
constexpr int COMBINE_THREADS = 128;
constexpr int SUM_PLACE = 36;            // the sums of a tile's 32 rows with one row of the activations
constexpr int SUM_COLUMN = 3 * WARPS * SUM_PLACE + 4;      // three places a warp; the next activation row's (no bank conflicts: 4 mod 16)
constexpr int STEP = 64;                 // bytes of a weight row that a warp takes at once
constexpr int MIN_STEPS = 4;             // of a tile (short rows: steps without bytes)

enum { F8 = 0, F8G = 1, I8 = 2, NV = 3, MX = 4, BF = 5 };

template <int FMT>
struct Fmt {
    static constexpr int ELEMS = FMT == NV || FMT == MX ? 32 : (FMT == BF ? 8 : 16);     // in 16 bytes
    static constexpr bool BF16 = FMT == BF;                                              // type of the products
    static constexpr bool FP4 = FMT == NV || FMT == MX;
    static constexpr int ROWS = FMT == MX ? 4 : 8;       // activation rows that a CTA multiplies at a time, at most
};

// Steps that a lane has registers for: all but one in flight.  MXFP4 with two terms has two sets of sums beside them and spills with
// three (one token 36 us a layer with two, 40 with three; 16 tokens 187 / 183).
template <int FMT, int PARTS>
struct Ahead { static constexpr int STEPS = FMT == MX && PARTS == 2 ? 2 : 3; };

struct Router {
    const void* logits;          // [tokens, experts]
    int dtype, tokens, experts, k, renorm;
    __device__ __forceinline__ float at(size_t i) const {
        return dtype == DSL_F32 ? static_cast<const float*>(logits)[i] : __bfloat162float(static_cast<const __nv_bfloat16*>(logits)[i]);
    }
};

struct Args {
    Router route;
    int tokens, experts, k;
    const void* x;               // up: [tokens, kdim] of x_dtype; down: h, fp32 [entries, kdim]
    int x_dtype;
    const uint8_t* w;            // [experts, n, row_bytes]
    const uint8_t* scale;        // as the packed weight has it
    const float* global_scale;
    int n, kdim, row_bytes, katoms;
    int units;                   // of 16 rows: 8 for every 128, the last ones possibly without rows
    int entry_cost;              // what starting on an expert costs a CTA, in eighths of a unit against one row
    int steps;                   // of a tile
    unsigned div_steps, div_grid, div_k, div_block;      // 2^32 / steps, / CTAs, / k, / block_rows: see quotient()
    int block_rows;              // rows of one expert that a CTA holds at a time
    int parts;                   // 16-bit terms an activation
    float* h;                    // up: [entries, n / 2]
    float* y;                    // down: [entries, n]
};

// n / d for n < 2^31, with m = floor((2^32 - 1) / d): the estimate is at most one too small.
__device__ __forceinline__ int quotient(int n, int d, unsigned m) {
    const int q = static_cast<int>(__umulhi(static_cast<unsigned>(n), m));
    return n - q * d >= d ? q + 1 : q;
}

// ---- routing -------------------------------------------------------------------------------------------------------------------
// Shared-memory tables of the list of work: entry = token * k + slot.
struct Plan {
    int* ids;          // [entries] expert, or -1
    int* order;        // entries sorted by expert, an expert's by token
    int* seg_expert;   // [segments]: an expert with at most block_rows of its rows
    int* seg_first;    //             first place in `order`
    int* seg_rows;
    int* seg_start;    //             first place in the list of work; [segments] its end
    uint32_t* tokens;  // [experts] who chose it, a bit each
    int* base;         // [experts] its first place in `order`
    int segments;
};

// Order-preserving key of a logit; 0 stands for "not to be chosen" (minus infinity, NaN, taken).
__device__ __forceinline__ uint32_t logit_key(float f) {
    const uint32_t b = __float_as_uint(f + 0.0f);              // one zero
    return f >= -FLT_MAX ? (b & 0x80000000u ? ~b : b | 0x80000000u) : 0u;
}

// The k largest logits of token t, ties to the lower index, as in dsl_moe_route: lane j's expert (-1: none left).  One warp; `v`:
// room for a row of keys.
__device__ __forceinline__ int choose(const Router& r, int t, uint32_t* v, int lane) {
    const size_t row = static_cast<size_t>(t) * r.experts;
    uint32_t keep[4];                                          // up to 128 experts stay in registers
    const bool small = r.experts <= 128;
    if (small) {
#pragma unroll
        for (int i = 0; i < 4; ++i) keep[i] = lane + 32 * i < r.experts ? logit_key(r.at(row + lane + 32 * i)) : 0u;
    } else {
#pragma unroll 1
        for (int e = lane; e < r.experts; e += 32) v[e] = logit_key(r.at(row + e));
    }
    int mine = -1;
#pragma unroll 1
    for (int j = 0; j < r.k; ++j) {
        uint32_t best = 0u;
        unsigned bi = 0x7FFFFFFFu;
        if (small) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (keep[i] > best) { best = keep[i]; bi = lane + 32 * i; }
        } else {
#pragma unroll 1
            for (int e = lane; e < r.experts; e += 32) {
                const uint32_t key = v[e];
                if (key > best) { best = key; bi = e; }
            }
        }
        const uint32_t top = __reduce_max_sync(0xFFFFFFFFu, best);
        if (top == 0u) break;                                  // uniform: nobody has one left
        const int e = static_cast<int>(__reduce_min_sync(0xFFFFFFFFu, best == top ? bi : 0x7FFFFFFFu));
        if (lane == j) mine = e;
        if (small) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (e == lane + 32 * i) keep[i] = 0u;
        } else if (lane == (e & 31)) {
            v[e] = 0u;                                         // its own lane's alone to read
        }
    }
    return mine;
}

// Weight of lane j's choice `e`: softmax over all experts, with the arithmetic of moe_route_kernel (moe.cu), so that it is
// dsl_moe_route's.  `sum`: the softmax's denominator, NaN where a logit of the token is.  One warp.
__device__ __forceinline__ float weigh(const Router& r, int t, int e, int lane, float& sum) {
    const size_t row = static_cast<size_t>(t) * r.experts;
    const float own = e >= 0 ? r.at(row + e) + 0.0f : 0.f, mx = __shfl_sync(0xFFFFFFFFu, own, 0);      // the first is the largest
    sum = 0.f;
#pragma unroll 1
    for (int i = lane; i < r.experts; i += 32) sum += expf(r.at(row + i) - mx);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
    const float pr = e >= 0 ? __fdiv_rn(expf(own - mx), sum) : 0.f;
    if (!r.renorm) return pr;
    float psum = 0.f;
#pragma unroll 1
    for (int j = 0; j < r.k; ++j) psum += __shfl_sync(0xFFFFFFFFu, pr, j);
    return __fdiv_rn(pr, psum);
}

// Cost of a unit, in eighths, against so many rows.  Measured a unit, us: NVFP4 1 / 2 / 3 rows 0.89 / 1.06 / 1.06 (K = 4096), MXFP4
// 1 / 2 / 3 / 4 rows 0.67 / 0.67 / 0.87 / 0.86 (K = 2912), FP8 128x128 1.31 whatever the rows.  In the shares: 8 tokens NVFP4 142 ->
// 123 us a layer, 16 tokens MXFP4 196 -> 172.
template <int FMT>
__device__ __forceinline__ bool heavy(int rows) { return FMT == NV ? rows > 1 : FMT == MX && rows > 2; }
template <int FMT>
__device__ __forceinline__ int unit_cost(int rows) { return heavy<FMT>(rows) ? (FMT == NV ? 9 : 10) : 8; }
// Units that `cost` pays for.
template <int FMT>
__device__ __forceinline__ int units_for(int cost, int rows) {
    const int each = unit_cost<FMT>(rows);
    return cost <= 0 ? 0 : (each == 8 ? cost >> 3 : (each == 9 ? cost / 9 : cost / 10));
}

// All threads.  `work`: WARPS * experts words that nothing else uses yet.  [begin, end): this CTA's share of the list of work, which
// starts in segment `seg`.
template <int FMT>
__device__ __forceinline__ void make_plan(const Args& a, Plan& p, uint32_t* work, int* s_misc, int& begin, int& end, int& seg) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll 1
    for (int e = threadIdx.x; e < a.experts; e += THREADS) p.tokens[e] = 0u;
    __syncthreads();
#pragma unroll 1
    for (int t = warp; t < a.tokens; t += WARPS) {
        const int e = choose(a.route, t, work + warp * a.experts, lane);
        if (lane < a.k) {
            p.ids[t * a.k + lane] = e;
            if (e >= 0) atomicOr(&p.tokens[e], 1u << t);
        }
    }
    __syncthreads();
    if (warp == 0) {
        // experts 32 at a time: their places and segments.  Three sums in a word: rows (at most 1024), segments (1024), segments
        // that cost more (two rows at least, so 512).
        const int plain = a.entry_cost + a.units * 8, extra = a.units * (FMT == NV ? 1 : 2), full_heavy = heavy<FMT>(a.block_rows) ? 1 : 0;
        uint32_t before = 0u;
#pragma unroll 1
        for (int e = lane; e - lane < a.experts; e += 32) {
            const int c = e < a.experts ? __popc(p.tokens[e]) : 0, b = quotient(c + a.block_rows - 1, a.block_rows, a.div_block);
            const int more = b > 0 ? (b - 1) * full_heavy + (heavy<FMT>(c - (b - 1) * a.block_rows) ? 1 : 0) : 0;
            const uint32_t what = static_cast<uint32_t>(c | (b << 11) | (more << 22));
            uint32_t run = before + what;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t v = __shfl_up_sync(0xFFFFFFFFu, run, o);
                if (lane >= o) run += v - before;
            }
            const uint32_t at = run - what;
            int first = at & 0x7FF, place = at >> 11 & 0x7FF, start = place * plain + static_cast<int>(at >> 22) * extra;
            if (c > 0) p.base[e] = first;
#pragma unroll 1
            for (int left = c; left > 0; left -= a.block_rows) {
                p.seg_expert[place] = e;
                p.seg_first[place] = first;
                p.seg_rows[place] = min(a.block_rows, left);
                p.seg_start[place] = start;
                first += a.block_rows;
                ++place;
                start += plain + full_heavy * extra;
            }
            before = __shfl_sync(0xFFFFFFFFu, run, 31);
        }
        const int segments = before >> 11 & 0x7FF, start = segments * plain + static_cast<int>(before >> 22) * extra;
        if (lane == 0) {
            s_misc[0] = segments;
            p.seg_start[segments] = start;
        }
    }
    __syncthreads();
#pragma unroll 1
    for (int t = warp; t < a.tokens; t += WARPS) {
        const int e = lane < a.k ? p.ids[t * a.k + lane] : -1;
        if (e >= 0) p.order[p.base[e] + __popc(p.tokens[e] & ((1u << t) - 1u))] = t * a.k + lane;
    }
    p.segments = s_misc[0];
    const int places = p.seg_start[p.segments], ctas = static_cast<int>(gridDim.x), bid = static_cast<int>(blockIdx.x);
    const int share = quotient(places, ctas, a.div_grid), more_than = places - share * ctas;
    begin = bid * share + min(bid, more_than);
    end = begin + share + (bid < more_than ? 1 : 0);
#pragma unroll 1
    for (int i = threadIdx.x; i < p.segments; i += THREADS)
        if (p.seg_start[i] <= begin && begin < p.seg_start[i + 1]) s_misc[1] = i;
    __syncthreads();
    seg = s_misc[1];
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
// two UE8M0 bytes (low 16 bits of w) -> two bf16: 2^(byte - 127), a subnormal for 0, and NaN for 255
__device__ __forceinline__ uint32_t widen_ue8m0(uint32_t w) {
    uint32_t r;
    asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.bf16x2.ue8m0x2 %0, lo;\n\t}" : "=r"(r) : "r"(w));
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

// 16 bytes that are read once.  The L2 is asked for 256 bytes of the row, which the warp comes to in its next steps: the memory reads
// longer pieces (8 tokens FP8 171 -> 157 us a layer, NVFP4 111 -> 107, 3 tokens BF16 390 -> 331).
__device__ __forceinline__ uint4 load_stream(const uint8_t* p) {
    uint4 r;
    asm volatile("ld.global.nc.L1::no_allocate.L2::256B.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(p));
    return r;
}
// Scale bytes: past the L1 too, which the lines of a whole atom would run through (8 tokens NVFP4 124 -> 114 us a layer).
__device__ __forceinline__ uint4 load_table(const uint8_t* p) {
    uint4 r;
    asm volatile("ld.global.nc.L1::no_allocate.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(p));
    return r;
}
__device__ __forceinline__ uint32_t word(const uint4& v, int j) { return j == 0 ? v.x : (j == 1 ? v.y : (j == 2 ? v.z : v.w)); }

// What a lane holds of one step: 16 bytes of each of its four rows (g + 32 j of the tile), with the scales.
template <int FMT>
struct Piece {
    static constexpr bool TABLE = FMT == NV || FMT == MX;
    uint4 w[4];
    uint4 s;                             // NV, MX: word j = the scale bytes of row j's atom
    float group;                         // F8G: scale of the step's 128-element group

    // `row`: row j = 0 of this lane, `rows`: from there to its rows.  Behind a row's end its last piece comes again, against zeros:
    // a NaN that it holds is in the row's sum already (bf16, whose infinities would make one, gets zeros).
    __device__ __forceinline__ void load(const Args& a, const uint8_t* row, const unsigned (&rows)[4], const uint8_t* scale, int step, int t) {
        const int there = step * STEP + t * 16, at = min(there, a.row_bytes - 16);
        const uint8_t* p = row + at;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            w[j] = load_stream(p + rows[j]);
            if (FMT == BF && there != at) w[j] = make_uint4(0u, 0u, 0u, 0u);
        }
        // NV: two blocks a piece, so atom piece / 2; MX: one, atom piece / 4 (the step)
        if (FMT == NV) s = load_table(scale + static_cast<size_t>(at >> 5) * 512);
        if (FMT == MX) s = load_table(scale + static_cast<size_t>(min(step, (a.row_bytes - 1) / STEP)) * 512);
        if (FMT == F8G) group = step * STEP < a.row_bytes ? __ldg(reinterpret_cast<const float*>(scale) + (step >> 1)) : 0.f;
    }
};

// A fragments of two k16 steps (a0, a1) from vector v, eight values each, of a lane's pieces of two rows: the widened weights
// without FP4 scales.
template <int FMT>
__device__ __forceinline__ void widen_rows(const uint4& q0, const uint4& q1, int v, uint32_t (&a0)[4], uint32_t (&a1)[4]) {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        const uint4& q = r == 0 ? q0 : q1;
        if (FMT == BF) {
            a0[r] = q.x; a0[r + 2] = q.y; a1[r] = q.z; a1[r + 2] = q.w;
        } else if (FMT == F8 || FMT == F8G) {
            const uint32_t w0 = word(q, 2 * v), w1 = word(q, 2 * v + 1);
            a0[r] = widen_e4m3(w0);
            a0[r + 2] = widen_e4m3(w0 >> 16);
            a1[r] = widen_e4m3(w1);
            a1[r + 2] = widen_e4m3(w1 >> 16);
        } else if (FMT == I8) {
            const uint32_t w0 = word(q, 2 * v) ^ 0x80808080u, w1 = word(q, 2 * v + 1) ^ 0x80808080u;
            a0[r] = widen_int8(w0, 0x4140);
            a0[r + 2] = widen_int8(w0, 0x4342);
            a1[r] = widen_int8(w1, 0x4140);
            a1[r + 2] = widen_int8(w1, 0x4342);
        } else {
            const uint32_t w = word(q, v);
            a0[r] = widen_e2m1<0>(w);
            a0[r + 2] = widen_e2m1<1>(w);
            a1[r] = widen_e2m1<2>(w);
            a1[r + 2] = widen_e2m1<3>(w);
        }
    }
}

// Sums of one step, columns = rows of the activations: acc[m * 4 ..] += weights (rows g + 64 m and g + 64 m + 32) x the rows in
// shared memory (eight columns).  `b`: this lane's place in them; a second term lies part_bytes behind the first.  NVFP4's scales are
// multiplied into the weights (exactly).
template <int FMT, int PARTS>
__device__ __forceinline__ void step_products(const Piece<FMT>& p, const uint8_t* b, int step, int t, int part_bytes, float (&acc)[8]) {
    using F = Fmt<FMT>;
    constexpr int VECS = F::ELEMS / 8;                  // 16-byte vectors of activations against one 16-byte piece of weights
    float sum[2][4];                                    // F8G: scaled before they are added
    uint32_t hs[4][2];                                  // NV: f16 scales of this lane's two blocks, by row
    if (FMT == NV) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t pair = widen_e4m3(word(p.s, j) >> ((t & 1) * 16));
            hs[j][0] = __byte_perm(pair, pair, 0x1010);
            hs[j][1] = __byte_perm(pair, pair, 0x3232);
        }
    }
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int j = 0; j < 4; ++j) sum[m][j] = FMT == F8G ? 0.f : acc[m * 4 + j];
#pragma unroll
    for (int v = 0; v < VECS; ++v) {
        const uint8_t* at = b + (step * VECS + v) * 64;
        const uint4 x = *reinterpret_cast<const uint4*>(at);
        uint4 lo;
        if (PARTS == 2) lo = *reinterpret_cast<const uint4*>(at + part_bytes);
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            uint32_t a0[4], a1[4];
            widen_rows<FMT>(p.w[2 * m], p.w[2 * m + 1], v, a0, a1);
            if (FMT == NV) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    a0[i] = hmul2(a0[i], hs[2 * m + (i & 1)][v / 2]);
                    a1[i] = hmul2(a1[i], hs[2 * m + (i & 1)][v / 2]);
                }
            }
            mma16<F::BF16>(sum[m], a0, x.x, x.y);
            mma16<F::BF16>(sum[m], a1, x.z, x.w);
            if (PARTS == 2) {
                mma16<F::BF16>(sum[m], a0, lo.x, lo.y);
                mma16<F::BF16>(sum[m], a1, lo.z, lo.w);
            }
        }
    }
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[m * 4 + j] = FMT == F8G ? fmaf(sum[m][j], p.group, acc[m * 4 + j]) : sum[m][j];
}

// Sums of one step, columns = scale blocks, for FP4 weights against few rows: a step has eight (NVFP4) or four (MXFP4) blocks along
// K, and B holds a row's values in the column of their block alone (zeros elsewhere), so that column n of the product is block n's
// sum and its scale meets one fp32 number instead of sixteen weights - half of the instructions that the widening above takes.
// Lane t holds blocks 2 t and 2 t + 1, as values and as columns (NVFP4), or block t, and columns t % 2 * 2 and + 1 (MXFP4).
// acc[set * 4 + j]: row j of the weights, of the lane's columns; a set is a row (NVFP4) or two rows (MXFP4) of the activations.
// `b`: per set and half of a piece, this lane's place in its row or among the zeros of one step; `own`: all ones or zero, whether it
// moves on with the steps and has a second term.
template <int FMT, int SETS, int PARTS>
__device__ __forceinline__ void step_blocks(const Piece<FMT>& p, const uint8_t* const (&b)[SETS][2], const unsigned (&own)[SETS][2], int step,
                                            int t, int part_bytes, float (&acc)[8]) {
    float sum[SETS][2][4];
#pragma unroll
    for (int k = 0; k < SETS; ++k)
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int j = 0; j < 4; ++j) sum[k][m][j] = 0.f;
#pragma unroll
    for (int v = 0; v < 4; ++v) {
        uint4 x[SETS], lo[SETS];
#pragma unroll
        for (int k = 0; k < SETS; ++k) {
            const int i = FMT == NV ? v / 2 : 0;
            const uint8_t* at = b[k][i] + (PARTS == 2 ? static_cast<unsigned>(step * 256) & own[k][i] : step * 256) + v * 64;
            x[k] = *reinterpret_cast<const uint4*>(at);
            if (PARTS == 2) lo[k] = *reinterpret_cast<const uint4*>(at + (static_cast<unsigned>(part_bytes) & own[k][i]));
        }
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            uint32_t a0[4], a1[4];
            widen_rows<FMT>(p.w[2 * m], p.w[2 * m + 1], v, a0, a1);
#pragma unroll
            for (int k = 0; k < SETS; ++k) {
                mma16<false>(sum[k][m], a0, x[k].x, x[k].y);
                mma16<false>(sum[k][m], a1, x[k].z, x[k].w);
                if (PARTS == 2) {
                    mma16<false>(sum[k][m], a0, lo[k].x, lo[k].y);
                    mma16<false>(sum[k][m], a1, lo[k].z, lo[k].w);
                }
            }
        }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const uint32_t pair = word(p.s, j) >> ((t & 1) * 16);
        float s0, s1;
        if (FMT == NV) {
            const uint32_t h = widen_e4m3(pair);
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
            s0 = f.x;
            s1 = f.y;
        } else {
            const uint32_t h = widen_ue8m0(pair);
            s0 = __uint_as_float(h << 16);
            s1 = __uint_as_float(h & 0xFFFF0000u);
        }
#pragma unroll
        for (int k = 0; k < SETS; ++k) {
            acc[k * 4 + j] = fmaf(sum[k][j >> 1][(j & 1) * 2], s0, acc[k * 4 + j]);
            acc[k * 4 + j] = fmaf(sum[k][j >> 1][(j & 1) * 2 + 1], s1, acc[k * 4 + j]);
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
// Rows whose largest magnitude lies here are taken as they are: f16 holds 16-bit values down to 2^-17 exactly and is off by
// 2^-25 at most below, 2^-25 of the largest.  Normed activations do.
__device__ __forceinline__ bool fits_f16(uint32_t amax) { return amax >= __float_as_uint(1.0f) && amax < __float_as_uint(32768.0f); }

// Zeros behind the rows, which FP4's columns without a value multiply: a row of them, or one step's (256 bytes) where rows of two
// terms leave less room; there the lane's place in them does not move on with the steps.
__host__ __device__ inline int zero_bytes(int parts, int part_bytes) { return parts == 2 ? 256 : part_bytes; }

// Rows first .. first + rows of the list; element j of a row lies in step j / (4 E), lane t = j / E % 4, vector j % E / 8, i.e. at
// ((step * E / 8 + vector) * 4 + t) * 16 bytes.  Elements past the row's end up to whole steps are zeros; with FP4 weights
// zeros follow the last one.  One look at the rows, a second one where some have to be scaled (`scaled`: they may have to be).
template <int FMT, bool DOWN, int PARTS>
__device__ __forceinline__ void stage_rows(const Args& a, const Plan& p, int first, int rows, uint8_t* dst, int pitch, int part_bytes,
                                           bool scaled, uint32_t* s_amax, float* s_inverse) {
    using F = Fmt<FMT>;
    constexpr int VECS = F::ELEMS / 8;
    const int vectors = a.steps * (STEP / 16) * VECS;                 // 8-element vectors of a padded row
    const int dtype = DOWN ? DSL_F32 : a.x_dtype;
    if (threadIdx.x < rows) s_amax[threadIdx.x] = 0u;
    __syncthreads();
#pragma unroll 1
    for (bool again = false;; again = true) {
        bool more = false;
#pragma unroll 1
        for (int r = 0; r < rows; ++r) {
            const int entry = p.order[first + r];
            const size_t src = static_cast<size_t>(DOWN ? entry : quotient(entry, a.k, a.div_k)) * a.kdim;
            float factor = 1.0f, inverse = 1.0f;
            if (again) {
                if (fits_f16(s_amax[r])) continue;
                factor = row_factor(s_amax[r], &inverse);
            }
            if (threadIdx.x == 0) s_inverse[r] = inverse;
            uint32_t m = 0u;
#pragma unroll 1
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
                    const float f0 = f[2 * i] * factor, f1 = f[2 * i + 1] * factor;
                    m = max(m, max(__float_as_uint(f[2 * i]) & 0x7FFFFFFFu, __float_as_uint(f[2 * i + 1]) & 0x7FFFFFFFu));
                    // the second term is the exact rest of the first, rounded; an infinity leaves none
                    if (F::BF16) {
                        const __nv_bfloat162 hi = __floats2bfloat162_rn(f0, f1);
                        const float h0 = __low2float(hi), h1 = __high2float(hi);
                        const __nv_bfloat162 rest = __floats2bfloat162_rn(isinf(h0) ? 0.f : f0 - h0, isinf(h1) ? 0.f : f1 - h1);
                        w[i] = *reinterpret_cast<const uint32_t*>(&hi);
                        lo[i] = *reinterpret_cast<const uint32_t*>(&rest);
                    } else {
                        const __half2 hi = __floats2half2_rn(f0, f1);
                        const float h0 = __low2float(hi), h1 = __high2float(hi);
                        const __half2 rest = __floats2half2_rn(isinf(h0) ? 0.f : f0 - h0, isinf(h1) ? 0.f : f1 - h1);
                        w[i] = *reinterpret_cast<const uint32_t*>(&hi);
                        lo[i] = *reinterpret_cast<const uint32_t*>(&rest);
                    }
                }
                *reinterpret_cast<uint4*>(d) = make_uint4(w[0], w[1], w[2], w[3]);
                if (PARTS == 2) *reinterpret_cast<uint4*>(d + part_bytes) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
            }
            if (scaled && !again) {
                m = __reduce_max_sync(0xFFFFFFFFu, m);
                if ((threadIdx.x & 31) == 0 && m != 0u) atomicMax(&s_amax[r], m);
            }
        }
        if (F::FP4 && !again)
#pragma unroll 1
            for (int v = threadIdx.x; v < zero_bytes(PARTS, part_bytes) / 16; v += THREADS)
                *reinterpret_cast<uint4*>(dst + static_cast<size_t>(rows) * pitch + v * 16) = make_uint4(0u, 0u, 0u, 0u);
        __syncthreads();
        if (!scaled || again) return;
#pragma unroll 1
        for (int r = 0; r < rows; ++r) more |= !fits_f16(s_amax[r]);
        if (!more) return;
    }
}

// ---- shared memory ----------------------------------------------------------------------------------------------------------------
struct Layout {
    int ids, order, seg_expert, seg_first, seg_rows, seg_start, chosen, base, misc, sums, rows, total;
    int pitch, part_bytes;
};
// `elems`: elements of a weight in 16 bytes; the rows' region doubles as the router's room.
__host__ __device__ inline Layout layout_of(const Args& a, int elems, bool fp4) {
    Layout l;
    const int entries = a.tokens * a.k;
    int at = 0;
    auto take = [&](int bytes) { const int here = at; at += (bytes + 15) / 16 * 16; return here; };
    l.ids = take(entries * 4);
    l.order = take(entries * 4);
    l.seg_expert = take(entries * 4);
    l.seg_first = take(entries * 4);
    l.seg_rows = take(entries * 4);
    l.seg_start = take((entries + 1) * 4);
    l.chosen = take(a.experts * 4);
    l.base = take(a.experts * 4);
    l.misc = take(16 + 2 * 8 * 4);                                     // two numbers; amax of the rows, their inverse factors
    l.sums = take(a.block_rows * SUM_COLUMN * 4);                     // a run's first piece of a tile, its last one, a whole one
    l.part_bytes = a.steps * (STEP / 16) * elems * 2;                  // a multiple of 128
    l.pitch = l.part_bytes * a.parts + 64;                             // two rows start half a bank round apart
    l.rows = take(0);
    int room = a.block_rows * l.pitch + (fp4 ? zero_bytes(a.parts, l.part_bytes) : 0);
    if (room < WARPS * a.experts * 4) room = WARPS * a.experts * 4;
    l.total = l.rows + room;
    return l;
}

template <int N> struct Way { static constexpr int value = N; };

// Row j (of four) of unit pair `tile` that belongs to lane group g.
__device__ __forceinline__ int row_of(int tile, int g, int j) { return (tile >> 2) * 128 + (tile & 3) * 8 + g + 32 * j; }

}  // namespace md

template <int FMT, bool DOWN, int PARTS>
__global__ void __launch_bounds__(md::THREADS, 1) moe_decode_kernel(const md::Args a) {
    using F = md::Fmt<FMT>;
    constexpr int AHEAD = md::Ahead<FMT, PARTS>::STEPS;
    using md::THREADS;
    using md::WARPS;
    extern __shared__ __align__(16) uint8_t smem[];
    const md::Layout l = md::layout_of(a, F::ELEMS, F::FP4);
    md::Plan plan;
    plan.ids = reinterpret_cast<int*>(smem + l.ids);
    plan.order = reinterpret_cast<int*>(smem + l.order);
    plan.seg_expert = reinterpret_cast<int*>(smem + l.seg_expert);
    plan.seg_first = reinterpret_cast<int*>(smem + l.seg_first);
    plan.seg_rows = reinterpret_cast<int*>(smem + l.seg_rows);
    plan.seg_start = reinterpret_cast<int*>(smem + l.seg_start);
    plan.tokens = reinterpret_cast<uint32_t*>(smem + l.chosen);
    plan.base = reinterpret_cast<int*>(smem + l.base);
    int* s_misc = reinterpret_cast<int*>(smem + l.misc);               // [0] segments, [1] this CTA's first one
    uint32_t* s_amax = reinterpret_cast<uint32_t*>(smem + l.misc + 16);
    float* s_inverse = reinterpret_cast<float*>(smem + l.misc + 16 + 32);
    float* s_sums = reinterpret_cast<float*>(smem + l.sums);
    uint8_t* s_rows = smem + l.rows;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2, t4 = lane & 3;
    if (!DOWN) {
        // Launched as a dependent, and lets its own successor be placed once everything before it is complete.
        griddep_wait();
        griddep_launch_dependents();
    }
    // f16 rows are what they are, bf16 ones as bf16 too; the second bf16 term of an fp32 value wants room below the first
    const bool scaled = DOWN || a.x_dtype == DSL_F32 || (a.x_dtype == DSL_BF16 && !F::BF16);
    // Down may get this far while up still runs - on an SM that up's CTA has left, since either fills the registers: logits and weights
    // were complete before up started.
    // The list of work: every expert's units behind entry_cost places without work, so that a CTA which passes from one expert to
    // the next, and has to fetch that one's rows, is dealt less.
    int begin, end, seg0;
    md::make_plan<FMT>(a, plan, reinterpret_cast<uint32_t*>(s_rows), s_misc, begin, end, seg0);
    bool waited = !DOWN;
    auto units_of = [&](int seg, int& unit0, int& unit1) {
        const int start = plan.seg_start[seg], rows = plan.seg_rows[seg];
        unit0 = md::units_for<FMT>(max(begin, start) - start - a.entry_cost, rows);
        unit1 = md::units_for<FMT>(min(end, plan.seg_start[seg + 1]) - start - a.entry_cost, rows);
    };

#pragma unroll 1
    for (int seg = seg0; begin < end && seg < plan.segments && plan.seg_start[seg] < end; ++seg) {
        int unit0, unit1;
        units_of(seg, unit0, unit1);
        if (unit0 == unit1) continue;
        const int expert = plan.seg_expert[seg], first = plan.seg_first[seg], rows = plan.seg_rows[seg];
        // this CTA's tiles of the expert, and this warp's run of their steps
        const int tile0 = unit0 >> 1, tiles = ((unit1 + 1) >> 1) - tile0;
        const int all = tiles * a.steps;
        const int run0 = all * warp / WARPS, run1 = all * (warp + 1) / WARPS;
        int at = run0, tile = md::quotient(run0, a.steps, a.div_steps), step = run0 - tile * a.steps;      // tile counts from tile0

        // Where the loads are: up to AHEAD - 1 steps before the products.
        static_assert(AHEAD <= md::MIN_STEPS, "two tiles could end in one round of the loop below");
        int l_at = run0, l_step = step, l_tile = tile0 + tile;
        const uint8_t *l_row = nullptr, *l_scale = nullptr;
        unsigned l_rows[4] = {0u, 0u, 0u, 0u};      // from l_row to the lane's rows: where one is not there or not this CTA's, to another
        auto locate = [&]() {
            const int r0 = min(md::row_of(l_tile, g, 0), a.n - 1), last = (a.n - 1 - r0) / 32;
            l_row = a.w + (static_cast<size_t>(expert) * a.n + r0) * a.row_bytes;
#pragma unroll
            for (int j = 0; j < 4; ++j)
                l_rows[j] = static_cast<unsigned>(min(last, min(max(j, 2 * l_tile < unit0 ? 2 : 0), 2 * l_tile + 1 >= unit1 ? 1 : 3))) * 32u * a.row_bytes;
            const size_t block = static_cast<size_t>(expert) * ((a.n + 127) / 128) + (l_tile >> 2);
            if (FMT == md::NV || FMT == md::MX) l_scale = a.scale + block * a.katoms * 512 + ((l_tile & 3) * 8 + g) * 16;
            if (FMT == md::F8G) l_scale = a.scale + block * (a.kdim / 128) * 4;
        };
        md::Piece<FMT> buf[AHEAD];
        auto fetch = [&](md::Piece<FMT>& p) {
            if (l_at < run1) {
                p.load(a, l_row, l_rows, l_scale, l_step, t4);
                ++l_at;
                if (++l_step == a.steps) {
                    l_step = 0;
                    ++l_tile;
                    locate();
                }
            }
        };
        if (run0 < run1) locate();
#pragma unroll
        for (int i = 0; i + 1 < AHEAD; ++i) fetch(buf[i]);
        if (!waited) {           // the hidden activation is up's
            griddep_wait();
            griddep_launch_dependents();
            waited = true;
        }
        __syncthreads();         // the segment before is finished, the router's room is free
        md::stage_rows<FMT, DOWN, PARTS>(a, plan, first, rows, s_rows, l.pitch, l.part_bytes, scaled, s_amax, s_inverse);
        float acc[8];
        auto clear = [&]() {
#pragma unroll
            for (int j = 0; j < 8; ++j) acc[j] = 0.f;
        };
        clear();
        // The sums of a tile that ends, or of the piece of it that the run has, go to one of the warp's three places in shared
        // memory: 0 a tile that begins before the run, 1 one that ends behind it, 2 a whole one, which is finished at once.
        float* mine = s_sums + warp * (3 * md::SUM_PLACE);
        // Everything from here to the segment's end, for one way of forming the products (sets: 0 rows as columns, else blocks).
        auto stream = [&](auto way) {
            constexpr int SETS = decltype(way)::value;
            constexpr int HELD = SETS > 0 ? SETS : 1;
            const uint8_t* b[HELD][2];
            unsigned own[HELD][2];
            if (SETS == 0) {
                b[0][0] = b[0][1] = s_rows + static_cast<size_t>(min(g, rows - 1)) * l.pitch + t4 * 16;      // columns past the rows: any
            } else {
#pragma unroll
                for (int k = 0; k < HELD; ++k)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        // column g: block g of row k (NVFP4), block g % 4 of row 2 k + g / 4 (MXFP4)
                        const int r = FMT == md::NV ? k : 2 * k + (g >> 2);
                        const bool mine_too = (FMT == md::NV ? g == 2 * t4 + i : (g & 3) == t4) && r < rows;
                        b[k][i] = s_rows + static_cast<size_t>(mine_too ? r : rows) * l.pitch + t4 * 16;
                        own[k][i] = mine_too ? ~0u : 0u;
                    }
            }
            auto multiply = [&](const md::Piece<FMT>& p) {
                if constexpr (SETS == 0) md::step_products<FMT, PARTS>(p, b[0][0], step, t4, l.part_bytes, acc);
                else md::step_blocks<FMT, HELD, PARTS>(p, b, own, step, t4, l.part_bytes, acc);
            };
            int whole = -1;
            auto close = [&](int tl) {
                const int from = tl * a.steps, to = from + a.steps;
                const int place = from < run0 ? 0 : (to > run1 ? 1 : 2);
                if (place == 2) whole = tl;
                float* d = mine + place * md::SUM_PLACE + g;
                if constexpr (SETS == 0) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        if (2 * t4 < rows) d[(2 * t4) * md::SUM_COLUMN + 8 * j] = acc[(j >> 1) * 4 + (j & 1) * 2];
                        if (2 * t4 + 1 < rows) d[(2 * t4 + 1) * md::SUM_COLUMN + 8 * j] = acc[(j >> 1) * 4 + (j & 1) * 2 + 1];
                    }
                } else {
#pragma unroll
                    for (int k = 0; k < HELD; ++k) {
                        float v[4];
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            v[j] = acc[k * 4 + j];
                            v[j] += __shfl_xor_sync(0xFFFFFFFFu, v[j], 1);
                            if (FMT == md::NV) v[j] += __shfl_xor_sync(0xFFFFFFFFu, v[j], 2);
                        }
                        if (FMT == md::NV) {             // lane t has row j = t to write, of column k
                            d[k * md::SUM_COLUMN + 8 * t4] = t4 == 0 ? v[0] : (t4 == 1 ? v[1] : (t4 == 2 ? v[2] : v[3]));
                        } else {                         // rows t % 2 * 2 and + 1, of column 2 k + t / 2
                            float* e = d + (2 * k + (t4 >> 1)) * md::SUM_COLUMN + 16 * (t4 & 1);
                            if (2 * k + (t4 >> 1) < rows) {
                                e[0] = t4 & 1 ? v[2] : v[0];
                                e[8] = t4 & 1 ? v[3] : v[1];
                            }
                        }
                    }
                }
                clear();
            };
#pragma unroll 1
            for (bool met = false;;) {
                int place = 2, others = warp + 1;          // whose pieces make up the tile that is finished below
                if (at < run1) {
#pragma unroll
                    for (int i = 0; i < AHEAD; ++i) {  // a tile has at least MIN_STEPS steps: at most one ends here
                        if (at < run1) {
                            fetch(buf[(i + AHEAD - 1) % AHEAD]);
                            multiply(buf[i]);
                            ++at;
                            const bool ends = ++step == a.steps;
                            if (ends || at == run1) close(tile);
                            if (ends) {
                                step = 0;
                                ++tile;
                            }
                        }
                    }
                } else if (!met) {
                    // every piece is there: the warp whose run has a tile's first step adds them
                    __syncthreads();
                    met = true;
                    const int last = tile - (step == 0 ? 1 : 0), from = last * a.steps, to = from + a.steps;
                    if (run0 < run1 && from >= run0 && to > run1) {
                        whole = last;
                        place = 1;
                        while (others < WARPS && all * others / WARPS < to) ++others;
                    }
                } else {
                    break;
                }
                if (whole < 0) continue;
                __syncwarp();        // the lanes' sums are there
                // Scales and the activation of a tile's sums, and the results to memory: a lane is a row.
                const int tt = tile0 + whole;
                whole = -1;
                const int r = md::row_of(tt, lane & 7, lane >> 3);
                const bool ours = r < a.n && 2 * tt + (lane >> 4) >= unit0 && 2 * tt + (lane >> 4) < unit1;
                float common = 1.0f;
                if (FMT == md::F8) common = *reinterpret_cast<const float*>(a.scale);
                if (FMT == md::NV) common = *a.global_scale;
                if (FMT == md::I8) common = ours ? __ldg(reinterpret_cast<const float*>(a.scale) + static_cast<size_t>(expert) * a.n + r) : 0.f;
#pragma unroll 1
                for (int c = 0; c < rows; ++c) {
                    float v = mine[place * md::SUM_PLACE + c * md::SUM_COLUMN + lane];
#pragma unroll 1
                    for (int w = warp + 1; w < others; ++w)
                        if (all * w / WARPS < all * (w + 1) / WARPS) v += s_sums[w * (3 * md::SUM_PLACE) + c * md::SUM_COLUMN + lane];      // (not of an empty run)
                    v = v * common * s_inverse[c];      // in this order: the last, a power of two, leads out of the range of the sums
                    const int entry = plan.order[first + c];
                    if (DOWN) {
                        if (ours) a.y[static_cast<size_t>(entry) * a.n + r] = v;
                    } else {
                        // rows 2i (gate) and 2i + 1 (up) are neighbouring lanes
                        const float up = __shfl_down_sync(0xFFFFFFFFu, v, 1);
                        if (ours && (lane & 1) == 0)
                            a.h[static_cast<size_t>(entry) * (a.n / 2) + (r >> 1)] = __fmul_rn(__fdiv_rn(v, 1.0f + expf(-v)), up);
                    }
                }
                __syncwarp();        // read, before the warp's next sums
            }
        };
        if constexpr (FMT == md::NV) {
            if (rows == 1) stream(md::Way<1>());
            else stream(md::Way<0>());
        } else if constexpr (FMT == md::MX) {
            if (rows <= 2) stream(md::Way<1>());
            else stream(md::Way<2>());
        } else {
            stream(md::Way<0>());
        }
    }

    if (DOWN && !waited) {       // a CTA without work: the last kernel relies on up's being complete
        griddep_wait();
        griddep_launch_dependents();
    }
}

// out[t] = sum over s of p[t, s] * y[t, s], in slot order, in fp32.  A CTA has 512 columns of a token, a thread four of them, eight
// slots' loads in flight.  Choices and weights it makes for itself while down still runs.  A kernel of its own, since a unit is
// complete only when its last expert is: added by the CTA that delivers a unit's last result (counters), the sums fell to the CTAs
// that finished last, 16 tokens MXFP4 up to 115 units, 25 us.
__global__ void __launch_bounds__(md::COMBINE_THREADS) moe_decode_combine_kernel(const md::Router r, const float* __restrict__ y, int n,
                                                                                 void* out, int out_dtype) {
    __shared__ uint32_t s_keys[DSL_MAX_GROUPS];
    __shared__ int s_ids[32];
    __shared__ float s_weights[32];
    __shared__ float s_start;
    const int t = blockIdx.y, k = r.k, col = (blockIdx.x * md::COMBINE_THREADS + threadIdx.x) * 4;
    if (threadIdx.x < 32) {
        const int e = md::choose(r, t, s_keys, threadIdx.x);
        s_ids[threadIdx.x] = e;                      // slots past k: none
        float total;
        s_weights[threadIdx.x] = md::weigh(r, t, e, threadIdx.x, total);
        if (threadIdx.x == 0) s_start = 0.f * total;      // a NaN among the logits is the token's result, chosen experts or not
    }
    __syncthreads();
    griddep_wait();
    griddep_launch_dependents();
    if (col >= n) return;
    const bool vec = n % 4 == 0;
    const float* row = y + static_cast<size_t>(t) * k * n + col;
    float s[4] = {s_start, s_start, s_start, s_start};
#pragma unroll 1
    for (int j0 = 0; j0 < k; j0 += 8) {
        float4 u[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int slot = min(j0 + j, k - 1);
            const float* q = row + static_cast<size_t>(slot) * n;
            if (vec) {
                u[j] = __ldcg(reinterpret_cast<const float4*>(q));
            } else {
                u[j] = make_float4(__ldcg(q), 0.f, 0.f, 0.f);
                if (col + 1 < n) u[j].y = __ldcg(q + 1);
                if (col + 2 < n) u[j].z = __ldcg(q + 2);
                if (col + 3 < n) u[j].w = __ldcg(q + 3);
            }
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            if (s_ids[j0 + j] < 0) continue;         // not written
            const float p = s_weights[j0 + j];
            s[0] = fmaf(p, u[j].x, s[0]);
            s[1] = fmaf(p, u[j].y, s[1]);
            s[2] = fmaf(p, u[j].z, s[2]);
            s[3] = fmaf(p, u[j].w, s[3]);
        }
    }
    const size_t to = static_cast<size_t>(t) * n + col;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        if (col + c >= n) break;
        if (out_dtype == DSL_BF16) static_cast<__nv_bfloat16*>(out)[to + c] = __float2bfloat16_rn(s[c]);
        else static_cast<float*>(out)[to + c] = s[c];
    }
}

// ---- host side -------------------------------------------------------------------------------------------------------------------
namespace md {

constexpr int SMEM_LIMIT = 227 * 1024;

// Rows of an expert that a CTA may hold, and its shared memory; false when not even one row fits.
static bool plan_launch(Args& a, int format, int* smem_bytes) {
    a.units = (a.n + 127) / 128 * 8;
    a.steps = (a.row_bytes + STEP - 1) / STEP;
    if (a.steps < MIN_STEPS) a.steps = MIN_STEPS;
    // Starting on an expert (its rows fetched, the pipeline filled and drained) costs a CTA about what 110 KB of weight take it;
    // one token NVFP4 / FP8 47 / 47 us without that in the shares, 43 / 45 with, 42 / 43 with twice as much, but 16 tokens MXFP4
    // 253 / 264 with once / twice.
    a.entry_cost = 8 * 7000 / a.row_bytes;
    const auto inverse = [](int d) { return static_cast<unsigned>(0xFFFFFFFFull / static_cast<unsigned>(d)); };
    a.div_steps = inverse(a.steps);
    a.div_k = inverse(a.k);
    const bool fp4 = format == DSL_W_NVFP4 || format == DSL_W_MXFP4;
    const int elems = fp4 ? 32 : (format == DSL_W_BF16 ? 8 : 16);
    const int cap = format == DSL_W_MXFP4 ? Fmt<MX>::ROWS : Fmt<NV>::ROWS, most = a.tokens < cap ? a.tokens : cap;
    int fits = 0;
    for (int r = 1; r <= most; ++r) {
        a.block_rows = r;
        const Layout l = layout_of(a, elems, fp4);
        if (l.total > SMEM_LIMIT) break;
        *smem_bytes = l.total;
        fits = r;
    }
    a.block_rows = fits;
    if (fits > 0) a.div_block = inverse(fits);
    return fits > 0;
}

// As little shared memory as a launch needs.
template <typename K>
static cudaError_t prefer_l1(K kernel) {
    return cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxL1);
}

template <int FMT, bool DOWN, int PARTS>
static int launch_one(Args& a, int smem_bytes, int sms, cudaStream_t st) {
    static PerDeviceInt attr_set;   // per device; idempotent, a race here only repeats the same call
    const int dev = current_device_slot();
    if (dev < 0) return static_cast<int>(cudaErrorInvalidDevice);
    if (attr_set.v[dev].load(std::memory_order_acquire) == 0) {
        const cudaError_t e = cudaFuncSetAttribute(moe_decode_kernel<FMT, DOWN, PARTS>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_LIMIT);
        if (e != cudaSuccess) return static_cast<int>(e);
        const cudaError_t c = prefer_l1(moe_decode_kernel<FMT, DOWN, PARTS>);
        if (c != cudaSuccess) return static_cast<int>(c);
        attr_set.v[dev].store(1, std::memory_order_release);
    }
    a.div_grid = 0xFFFFFFFFu / static_cast<unsigned>(sms);
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
    return static_cast<int>(cudaLaunchKernelEx(&cfg, moe_decode_kernel<FMT, DOWN, PARTS>, a));
}

// One of the two products.  `x_dtype`: of the layer; the hidden activation is fp32.
static Args side(const dsl_weight* w, bool is_down, int tokens, int k, int x_dtype) {
    Args a{};
    a.tokens = tokens;
    a.experts = w->groups;
    a.k = k;
    a.x_dtype = is_down ? DSL_F32 : x_dtype;
    a.w = static_cast<const uint8_t*>(w->q);
    a.scale = static_cast<const uint8_t*>(w->scale);
    a.global_scale = w->global_scale;
    a.n = w->n;
    a.kdim = w->k;
    const bool fp4 = w->format == DSL_W_NVFP4 || w->format == DSL_W_MXFP4;
    a.row_bytes = fp4 ? w->k / 2 : (w->format == DSL_W_BF16 ? 2 * w->k : w->k);
    a.katoms = fp4 ? (w->k / (w->format == DSL_W_NVFP4 ? 16 : 32) + 3) / 4 : 0;
    // a layer with an fp32 x keeps its activations in two terms; bf16 products need a second one for whatever is not bf16
    a.parts = x_dtype == DSL_F32 || (w->format == DSL_W_BF16 && a.x_dtype != DSL_BF16) ? 2 : 1;
    return a;
}

template <int FMT>
static int launch_fmt(int format, Args& up, Args& down, int sms, cudaStream_t st) {
    int bytes_up = 0, bytes_down = 0;
    if (!plan_launch(up, format, &bytes_up) || !plan_launch(down, format, &bytes_down))
        return DSL_ERR_TOO_LARGE;
    const int rc = up.parts == 2 ? launch_one<FMT, false, 2>(up, bytes_up, sms, st) : launch_one<FMT, false, 1>(up, bytes_up, sms, st);
    if (rc != 0) return rc;
    if (down.parts == 2) return launch_one<FMT, true, 2>(down, bytes_down, sms, st);
    if constexpr (FMT == BF) return DSL_ERR_ENUM;             // always two there
    else return launch_one<FMT, true, 1>(down, bytes_down, sms, st);
}

static int launch_combine(const Router& r, const float* y, int n, void* out, int out_dtype, cudaStream_t st) {
    static PerDeviceInt attr_set;
    const int dev = current_device_slot();
    if (dev < 0) return static_cast<int>(cudaErrorInvalidDevice);
    if (attr_set.v[dev].load(std::memory_order_acquire) == 0) {
        const cudaError_t e = prefer_l1(moe_decode_combine_kernel);
        if (e != cudaSuccess) return static_cast<int>(e);
        attr_set.v[dev].store(1, std::memory_order_release);
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(((n + 3) / 4 + COMBINE_THREADS - 1) / COMBINE_THREADS), static_cast<unsigned>(r.tokens));
    cfg.blockDim = dim3(COMBINE_THREADS);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return static_cast<int>(cudaLaunchKernelEx(&cfg, moe_decode_combine_kernel, r, y, n, out, out_dtype));
}

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
    // sizes whose products the kernels form in 32 bits: 96 rows of a weight, units and steps of all segments
    if (gu->k > (1 << 20) || dn->k > (1 << 20) || dn->n > (1 << 18)) return DSL_ERR_TOO_LARGE;
    if (tokens > 0) {
        int bytes;
        for (int i = 0; i < 2; ++i) {
            Args a = side(i == 0 ? gu : dn, i == 1, tokens, k, x_dtype);
            if (!plan_launch(a, gu->format, &bytes)) return DSL_ERR_TOO_LARGE;
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
    return md::up256(entries * down->k * 4) + md::up256(entries * down->n * 4);
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
    const unsigned table = format == DSL_W_NVFP4 || format == DSL_W_MXFP4 ? 15u : 3u;      // FP4: 16 scale bytes at a time
    if ((vectors & 15u) != 0 || (words & table) != 0 || (reinterpret_cast<uintptr_t>(scratch) & 255u) != 0) return DSL_ERR_ALIGN;
    if (scratch_bytes < dsl_moe_decode_scratch_bytes(gate_up, down, tokens, k, x_dtype)) return DSL_ERR_TOO_LARGE;
    md::Args up = md::side(gate_up, false, tokens, k, x_dtype), dn = md::side(down, true, tokens, k, x_dtype);
    const size_t entries = static_cast<size_t>(tokens) * k;
    uint8_t* base = static_cast<uint8_t*>(scratch);
    float* h = reinterpret_cast<float*>(base);
    float* y = reinterpret_cast<float*>(base + md::up256(entries * down->k * 4));
    const md::Router route = {logits, logits_dtype, tokens, gate_up->groups, k, renorm};
    up.route = route;
    dn.route = route;
    up.x = x;
    up.h = h;
    dn.x = h;
    dn.y = y;
    const int sms = sm_count();
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    switch (format) {
        case DSL_W_FP8: rc = md::launch_fmt<md::F8>(format, up, dn, sms, st); break;
        case DSL_W_FP8_BLOCK128: rc = md::launch_fmt<md::F8G>(format, up, dn, sms, st); break;
        case DSL_W_INT8: rc = md::launch_fmt<md::I8>(format, up, dn, sms, st); break;
        case DSL_W_NVFP4: rc = md::launch_fmt<md::NV>(format, up, dn, sms, st); break;
        case DSL_W_MXFP4: rc = md::launch_fmt<md::MX>(format, up, dn, sms, st); break;
        default: rc = md::launch_fmt<md::BF>(format, up, dn, sms, st); break;
    }
    return rc != 0 ? rc : md::launch_combine(route, y, down->n, out, out_dtype, st);
}
