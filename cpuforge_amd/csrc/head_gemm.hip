// The LM head's products for the targets' log-probabilities of many rows
// (cfops_lm_head_logprobs, cfops_lm_head_logprobs_backward), on the f16 matrix
// cores, with what follows a product in its epilogue: the logits never reach
// memory.
//
// f32 operands as two f16 pieces: x 2^-e = h + l with h = f16(x 2^-e), l = f16 of
// what is left, the power of two such that the largest value of its group is in
// [2^14, 2^15).  A signed 11-bit piece beside an 11-bit one hold 22 to 23 bits of x;
// below 2^-17 of the group's largest value l is subnormal, and what is lost is at
// most 2^-40 of that largest value.  a b is the three products hl, lh and hh
// (each exact, 11 x 11 bits), summed in f32 by the MFMA; ll, at most 2^-24 of |a b|,
// is left out.  Half the MFMAs of three bf16 pieces (gemm_f32.hip), at the price
// of a group's exponent: rows of hidden states have one each, 32 rows of the
// head share one.  A logit's error is so bounded by 2^-22 sum |h_k w_k| and 2^-39 of
// the largest |h| times the largest |w| of the 32 rows, which is no more than f32
// sums leave.
//
// The hidden states' gradient, dlogp (head[target] - sum_v P_v head[v]), takes P
// from the forward: beside its statistics that keeps, for each token and 128
// rows of the head, exp(x - m) with m their largest logit, in f32 and in the order
// of the gradient's product (4 bytes a logit).  The product adds 128 rows at a time
// and scales their sum by exp(m - lse), a factor of the result's own column, and by the
// power of two of those rows of the head; where that changes by more than kRun from 32
// rows to the next, a sum ends there.  No exponential or product is formed twice.  (The
// logits formed again in the backward instead, 3686 x 576 x 49152: 0.81 ms, where keeping
// them takes 0.2.)
// The exponentials are kept in f32 and split by the waves of that product (2 to 4% of the
// time of both).  As pieces, whose last bit is 2^-34 of the largest of 128, they
// would be exact enough for the hidden states' gradient, where that largest one stands in
// the same sum, but not for the head's: there a rare token's row is a sum of its own over
// tokens (e^-20 below the others it lost 4e-3 of itself, at e^-25 all).
//
// Packed operands: both are first written as MFMA operands (1 KiB: a lane's eight
// f16, 64 lanes) of 32 rows and 16 k, the two pieces side by side, so a
// stage goes to LDS by direct loads of whole KiB and is read without bank
// conflicts, and no wave spends instructions on splitting.
#include <hip/hip_runtime.h>
#include <limits.h>

#include <algorithm>
#include <type_traits>

#include "cfattn_common.hpp"
#include "cfattn_kernels.hpp"
#include "cfops_kernels.hpp"

namespace cfattn {
namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr int kFrag = 1024;        // bytes of an operand of one MFMA
constexpr int kBN = 128;           // tokens of a tile
constexpr int kWgs = 512;          // two workgroups to a CU
constexpr int kStages = 3;           // two workgroups' stages fill 147 of 160 KiB
constexpr int kGroup = 8;          // token tiles
constexpr float kTop = 4096.0f;    // of a kept exponential in a product
constexpr int kRun = 3;            // powers of two between the rows of the head of a run

__device__ __forceinline__ float exp2i(int e) { return __builtin_bit_cast(float, (uint32_t)(e + 127) << 23); }
// 2^e within f32's normal range.
__device__ __forceinline__ float pow2_clamped(int e) { return exp2i(min(max(e, -126), 127)); }

// The exponent e of a group whose largest finite magnitude is `top`: 2^-e and 2^e
// are normal.
__device__ __forceinline__ int group_exponent(float top) {
    const int e = (int)(__builtin_bit_cast(uint32_t, top) >> 23) - 127 - 14;
    return max(e, -112);
}
__device__ __forceinline__ float finite_abs(float x) {
    const float a = fabsf(x);
    return a < INFINITY ? a : 0.0f;
}

// Memory that the whole launch only reads.
typedef const __attribute__((address_space(4))) int* ScalarInts;

__device__ __forceinline__ f32x16 mfma_f16(const f16x8& a, const f16x8& b, const f32x16& c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

struct Pieces {
    f16x8 h, l;
};
typedef float f32x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ Pieces split8(const float (&x)[8], float scale) {
#pragma clang fp contract(off)
    Pieces p;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const float y = x[i] * scale;
        p.h[i] = (_Float16)y;
        p.l[i] = (_Float16)(y - (float)p.h[i]);
    }
    return p;
}
// The same by one fused operation a piece.
__device__ __forceinline__ Pieces split8(const f32x4& a, const f32x4& b, float scale) {
    Pieces p;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const float x = i < 4 ? a[i] : b[i - 4];
        p.h[i] = (_Float16)fmaf(x, scale, 0.0f);
        p.l[i] = (_Float16)fmaf(x, scale, -(float)p.h[i]);
    }
    return p;
}
__device__ __forceinline__ void store_pieces(char* frag, int lane, const Pieces& p) {
    *reinterpret_cast<f16x8*>(frag + lane * 16) = p.h;
    *reinterpret_cast<f16x8*>(frag + kFrag + lane * 16) = p.l;
}

// Eight values of a row from k on, zeros past d.
__device__ __forceinline__ void load8(float (&x)[8], const float* row, int k, int d, bool vec) {
    if (vec && k + 8 <= d) {
        const float4 a = *reinterpret_cast<const float4*>(row + k), b = *reinterpret_cast<const float4*>(row + k + 4);
        x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = row && k + i < d ? row[k + i] : 0.0f;
    }
}

// Scored rows of [j0, j0 + chunk); none where `count` is another plan's.
__device__ __forceinline__ int scored_rows(const int* __restrict__ count, int tag, int j0, int chunk) {
    return count[1] == tag ? max(min(count[0] - j0, chunk), 0) : 0;
}

struct PackArgs {
    const float *hn, *head;
    const int *idx, *count;
    char *rows, *packed, *back, *rows_back;  // rows and rows_back may be null
    float* scale;
    int* exponents;
    int row_blocks, vocab, d, k16, v16, t16, vec_rows, vec_head, tag;
};

// 32 rows to a workgroup, as operands [32 rows][16 k][piece]: first the scored rows
// of hn, each with its own 2^e, zeros from row n on; then the head's, with one e,
// and, for the gradients, whose k are these rows, as [32 columns][16 rows][piece]
// too.  There lane l holds column l % 32 and of 16 rows those that it holds of a
// product's 32 x 32 result: 4 (l / 32) + 0..3 and the same eight on.
// A wave takes the pairs of operands (32 columns) w, w + NW, ..; with U > 0 at most U
// of them, which stay in registers between the largest value and the pieces.
// Bound by HBM: 128256 x 2048 411 us, 5.1 TB/s of one read and one write.  (Read
// twice, the second time came from HBM again, since the 32 rows of all workgroups in
// flight are 0.5 GB: 640 us.)
template <bool BACK, int NW, int U>
__global__ __launch_bounds__(64 * NW) void pack_kernel(const PackArgs g) {
    __shared__ float red[NW][32];
    __shared__ uint32_t tile[BACK ? NW : 1][32][33];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l32 = lane & 31;
    const bool is_head = (int)blockIdx.x >= g.row_blocks;
    const int blk = is_head ? blockIdx.x - g.row_blocks : blockIdx.x, r = blk * 32 + l32, k16 = g.k16, d = g.d;
    const float* row = nullptr;
    if (is_head) {
        if (r < g.vocab) row = g.head + (long)r * d;
    } else {
        const int n = scored_rows(g.count, g.tag, 0, INT_MAX);
        if (blk * 32 >= (n + kBN - 1) / kBN * kBN) return;
        if (r < n) row = g.hn + (long)g.idx[r] * d;
    }
    const bool v = (is_head ? g.vec_head : g.vec_rows) && row;
    const int c = 8 * (lane >> 5), pairs = (k16 + 1) / 2;
    float top = 0.0f, x[U ? U : 1][2][8];
    auto load = [&](float (&y)[2][8], int s) {
#pragma unroll
        for (int q = 0; q < 2; q++) {
            const bool in = 2 * s + q < k16;
            load8(y[q], in ? row : nullptr, 16 * (2 * s + q) + c, d, v && in);
        }
    };
    auto widen = [&](const float (&y)[2][8]) {
#pragma unroll
        for (int q = 0; q < 2; q++)
#pragma unroll
            for (int i = 0; i < 8; i++) top = fmaxf(top, finite_abs(y[q][i]));
    };
    if constexpr (U > 0) {
#pragma unroll
        for (int u = 0; u < U; u++)
            if (wave + u * NW < pairs) load(x[u], wave + u * NW);
#pragma unroll
        for (int u = 0; u < U; u++)
            if (wave + u * NW < pairs) widen(x[u]);
    } else {
        for (int s = wave; s < pairs; s += NW) {
            load(x[0], s);
            widen(x[0]);
        }
    }
    top = max_halves(top);
    if (lane < 32) red[wave][lane] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < NW; w++) top = fmaxf(top, red[w][l32]);
    if (is_head)
#pragma unroll
        for (int o = 16; o >= 1; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
    const int e = group_exponent(top);
    if (is_head && threadIdx.x == 0) g.exponents[blk] = e;
    if (!is_head && threadIdx.x < 32) g.scale[r] = exp2i(e);
    const float sc = exp2i(-e);
    char* out = is_head ? g.packed : g.rows;
    auto store = [&](const float (&y)[2][8], int s) {
#pragma unroll
        for (int q = 0; q < 2; q++) {
            const Pieces p = split8(y[q], sc);
            if (out && 2 * s + q < k16) store_pieces(out + ((long)blk * k16 + 2 * s + q) * 2 * kFrag, lane, p);
            if constexpr (BACK)
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    // (Copies: a bit cast of a vector's element itself takes element 0.)
                    const _Float16 h = p.h[i], l = p.l[i];
                    tile[wave][l32][16 * q + c + i] = (uint32_t)__builtin_bit_cast(uint16_t, h) |
                                                      (uint32_t)__builtin_bit_cast(uint16_t, l) << 16;
                }
        }
        if constexpr (BACK) {
            char* to = is_head ? g.back : g.rows_back;
            if (!to) return;
            const int steps = is_head ? g.v16 : g.t16;
            // (A wave's own part of LDS: its own order of accesses is enough.)
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int q = 0; q < 2; q++) {
                Pieces p;
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const uint32_t u = tile[wave][16 * q + 8 * (i >> 2) + 4 * (lane >> 5) + (i & 3)][l32];
                    p.h[i] = __builtin_bit_cast(_Float16, (uint16_t)u);
                    p.l[i] = __builtin_bit_cast(_Float16, (uint16_t)(u >> 16));
                }
                store_pieces(to + ((long)s * steps + blk * 2 + q) * 2 * kFrag, lane, p);
            }
            __builtin_amdgcn_wave_barrier();
        }
    };
    if constexpr (U > 0) {
#pragma unroll
        for (int u = 0; u < U; u++)
            if (wave + u * NW < pairs) store(x[u], wave + u * NW);
    } else {
        for (int s = wave; s < pairs; s += NW) {
            load(x[0], s);
            store(x[0], s);
        }
    }
}

enum class Product { kStats, kRows, kHead };

struct HeadArgs {
    // Operands: rows of the result along a (64 MB to a tile), columns (kBN) along b: the
    // scored rows, or (head) the columns of the head.
    const char *a, *b;
    int ka, kb;         // 16-k steps from one 32 rows of a (of b) to the next
    int mt, nt;         // tiles along a, and (head) along b
    const int* count;   // scored rows
    int tag;
    int j0, chunk;      // this launch's: [j0, min(j0 + chunk, count)); b, stats, keep and part start at j0
    long ld;            // of stats, xt and factor
    // statistics: a is the head
    const int *exponents, *targets;  // targets: of scored rows
    const float* scale;
    int vocab, v16;
    float2* stats;      // [128 rows of the head][ld]: max and sum of exp2, in log2 units
    float* xt;          // the targets' logits
    char* keep;         // [32 tokens][v16][half of a lane's eight values], or null
    // the rows' gradient: a is the head by columns, b what statistics kept
    const float* factor;  // [128 rows of the head][ld]; exponents as above
    float* part;          // [split][chunk][64 MB mt], chunk a pass's rows
    int splits_max;
    // the head's gradient: a is the dlogits by columns, b the rows by columns
    const unsigned* col_top;  // [vocab]: a bound of the dlogits of a column, as f32 bits
    float* dhead;
    int d, acc;         // acc: added to dhead, else written
};

// Splits of the gradient's k (the vocabulary) over workgroups: a multiple of the
// XCDs, so that one XCD's L2 holds what its workgroups share.  The one with the
// least rounds of an XCD's share over its 64 workgroups times its length; a split's
// partial sums cost their way through memory.
struct Splits {
    int count;
    float cost;  // in steps of a tile
};
__host__ __device__ __forceinline__ Splits splits_of(int tiles, int k16, int splits_max) {
    Splits best{8, INFINITY};
    for (int s = 8; s <= splits_max; s += 8) {
        const int rounds = (tiles * (s / 8) + kWgs / 8 - 1) / (kWgs / 8);
        const float cost = rounds * ((k16 + s - 1) / s + 24.0f) + 0.35f * tiles * s / 64.0f;
        if (cost < best.cost) best = {s, cost};
    }
    return best;
}

// A tile of 64 MB rows and kBN columns to a workgroup of four waves, each 32 MB x 64, or, in
// the rows' gradient, 64 MB x 32, so that no two split the same exponentials (32 MB x 64
// there: 668 us where this takes 650, 182 where 171); two workgroups to a CU: one's epilogue
// runs beside the other's products.
// Bound by the power of the products: statistics of 2048 rows x 576 x 49152 297 us (three
// times 116 GFLOP on f16, 1.17 PFLOP/s, where a library's f16 product of 8192^3 has 1.16),
// MFMAs busy in 62% of the cycles at 1.76 GHz, no bank conflicts; 3686 rows with what the
// gradients need kept 583, their gradient's product 650 (603 of operands that need no
// splitting).  Not faster: 256 x 256 tiles of
// eight waves, waves of 128 x 128 with a SIMD each (593 us where this took 403), a branch
// for each 32 columns of a last tile (its registers spill).
template <int MB, Product P>
__global__ __launch_bounds__(256, 2) void head_gemm_kernel(const HeadArgs g) {
    constexpr bool ROWS = P == Product::kRows;
    // Blocks of 32 rows and columns of a wave's part of the tile.
    constexpr int RB = ROWS ? 2 * MB : MB, CB = ROWS ? 1 : 2;
    constexpr int BM = 64 * MB, CH = 4 * MB + 8, PER = CH / 4 + ROWS, STAGE = CH * kFrag + ROWS * 1024;
    static_assert(CH % 4 == 0, "whole loads a wave");
    __shared__ __attribute__((aligned(1024))) char lds[kStages * STAGE];
    const int lane = threadIdx.x & 63, wave = wave_uniform(threadIdx.x >> 6);
    const int wm = ROWS ? 0 : wave >> 1, wn = ROWS ? wave : wave & 1, l32 = lane & 31, hh = lane >> 5;
    const int n = wave_uniform(scored_rows(g.count, g.tag, g.j0, g.chunk));
    const bool other = P == Product::kHead && wave_uniform(g.count[1]) != g.tag;
    if (n == 0 && !(P == Product::kHead && (!g.acc || other))) return;
    const int nt = P == Product::kHead ? g.nt : (n + kBN - 1) / kBN;
    // Items of an XCD: a contiguous run of the tiles along a (of the splits), every
    // tile along b with each.
    const int xcd = blockIdx.x % 8, local = blockIdx.x / 8;
    int outer = g.mt, inner = nt;
    if constexpr (ROWS) {
        outer = wave_uniform(splits_of(g.mt * nt, g.ka, g.splits_max).count);
        inner = g.mt * nt;
    }
    const int o0 = (int)((long)outer * xcd / 8), o1 = (int)((long)outer * (xcd + 1) / 8);
    const uint32_t lds0 = lds_offset(lds), voff = lane * 16;
    for (int item = local; item < (o1 - o0) * inner; item += kWgs / 8) {
        // Without splits: kGroup tiles along b with every tile along a of the XCD, then
        // the next ones: what 64 workgroups read at a time is near a square.
        int o, tm, tt, k0 = 0, k1 = P == Product::kHead ? (n + 15) / 16 : g.ka;
        if constexpr (ROWS) {
            o = wave_uniform(o0 + item / inner);
            tm = wave_uniform(item % inner % g.mt);
            tt = wave_uniform(item % inner / g.mt);
            // (Whole runs of 128 rows of the head.)
            k0 = wave_uniform((int)((long)(g.ka / 8) * o / outer) * 8);
            k1 = wave_uniform((int)((long)(g.ka / 8) * (o + 1) / outer) * 8);
        } else {
            const int grp = item / ((o1 - o0) * kGroup), left = item - grp * (o1 - o0) * kGroup;
            const int w = min(kGroup, nt - grp * kGroup);
            o = tm = wave_uniform(o0 + left / w);
            tt = wave_uniform(grp * kGroup + left % w);
        }
        const char* src[CH / 4];
#pragma unroll
        for (int i = 0; i < CH / 4; i++) {
            const int c = CH / 4 * wave + i;  // the stage's KiB: operand c / 2, piece c % 2
            const int blk = c / 2;
            const char* base = blk < 2 * MB ? g.a + ((long)(tm * 2 * MB + blk) * g.ka + k0) * 2 * kFrag
                                            : g.b + ((long)(tt * 4 + blk - 2 * MB) * g.kb + k0) * 2 * kFrag;
            src[i] = base + (c % 2) * kFrag;
        }
        const int col0 = tt * kBN + wn * 32 * CB;  // this wave's first column
        int kl = k0;                               // the next stage's k
        auto load = [&](uint32_t stage) {
#pragma unroll
            for (int i = 0; i < CH / 4; i++) {
                lds_load16_so(src[i], voff, lds0 + stage + (CH / 4 * wave + i) * kFrag);
                src[i] += 2 * kFrag;
            }
            if constexpr (ROWS) {
                // The factors of the stage's 128 rows for the wave's tokens.
                lds_load4_so(g.factor + (long)(kl / 8) * g.ld + col0, l32 * 4, lds0 + stage + CH * kFrag + wave * 256);
                kl++;
            }
        };
        // (A wave of a last tile whose columns all lie behind the last one forms nothing.)
        const bool live_cols = P == Product::kHead || col0 < n;
        f32x16 acc[RB][CB], tot[ROWS ? RB : 1][CB];
#pragma unroll
        for (int i = 0; i < RB; i++)
#pragma unroll
            for (int j = 0; j < CB; j++) {
                acc[i][j] = zero16();
                if constexpr (ROWS) tot[i][j] = zero16();
            }
        // Every wave is done with the LDS of the item before, and with its stores
        // (they would count among the loads waited for below).
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        // (Through the scalar cache: a vector load's wait would be one for the stages' too.)
        const ScalarInts exponents = ROWS ? (ScalarInts)(uintptr_t)g.exponents : nullptr;
        int exponent = ROWS && k0 < k1 ? exponents[k0 / 2] : 0, run = exponent;
        float kept = 1.0f;
        uint32_t cur = 0, nxt = 2 * STAGE;
        if (k0 < k1) load(0);  // (more splits than runs: some have none)
        if (k0 + 1 < k1) load(STAGE);
        for (int k = k0; k < k1; k++) {
            if (k + 1 < k1)
                asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"i"(PER) : "memory");
            else
                asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
            if (k + 2 < k1) load(nxt);
            nxt = nxt == (kStages - 1) * STAGE ? 0 : nxt + STAGE;
            if constexpr (ROWS) {
                // The exponentials meet 32 rows of the head, whose power of two is within
                // kRun of that of the sums.
                if (k % 2 == 0) {
                    kept = kTop * exp2i(exponent - run);
                    exponent = exponents[min(k + 2, k1 - 1) / 2];
                }
            }
            const char* s = lds + cur;
            cur = cur == (kStages - 1) * STAGE ? 0 : cur + STAGE;
            f16x8 a[RB][2], b[CB][2];
            f32x4 kept_b[2];
            if constexpr (ROWS) {
                kept_b[0] = *reinterpret_cast<const f32x4*>(s + (2 * MB + wn) * 2 * kFrag + voff);
                kept_b[1] = *reinterpret_cast<const f32x4*>(s + ((2 * MB + wn) * 2 + 1) * kFrag + voff);
            } else {
#pragma unroll
                for (int p = 0; p < 2; p++)
#pragma unroll
                    for (int j = 0; j < CB; j++)
                        b[j][p] = *reinterpret_cast<const f16x8*>(s + ((2 * MB + wn * CB + j) * 2 + p) * kFrag + voff);
            }
#pragma unroll
            for (int p = 1; p >= 0; p--) {
#pragma unroll
                for (int i = 0; i < RB; i++)
                    a[i][p] = *reinterpret_cast<const f16x8*>(s + ((wm * RB + i) * 2 + p) * kFrag + voff);
                // (The first products' operands are read together.)
                if (ROWS && (p == 1 || MB == 2)) __builtin_amdgcn_sched_barrier(0);
            }
            if constexpr (ROWS) {
                const Pieces x = split8(kept_b[0], kept_b[1], kept);
                b[0][0] = x.h, b[0][1] = x.l;
            }
            // (The order that shares an operand from one to the next: 1% less time.)
            constexpr int pa[3] = {1, 0, 0}, pb[3] = {0, 0, 1};
            if (live_cols)
#pragma unroll
                for (int q = 0; q < 3; q++)
#pragma unroll
                    for (int i = 0; i < RB; i++)
#pragma unroll
                        for (int jj = 0; jj < CB; jj++) {
                            const int j = (i + q) & 1 ? CB - 1 - jj : jj;
                            acc[i][j] = mfma_f16(a[i][pa[q]], b[j][pb[q]], acc[i][j]);
                        }
            if constexpr (ROWS) {
                if (k % 8 != 7 && (k % 2 == 0 || abs(exponent - run) <= kRun)) continue;
                const float unit = exp2i(run) * (1.0f / kTop);
                run = exponent;
                const float* f = reinterpret_cast<const float*>(s + CH * kFrag + wave * 256);
#pragma unroll
                for (int j = 0; j < CB; j++) {
                    const float fj = f[32 * j + l32] * unit;
#pragma unroll
                    for (int i = 0; i < RB; i++) {
#pragma unroll
                        for (int q = 0; q < 16; q++) tot[i][j][q] = fmaf(acc[i][j][q], fj, tot[i][j][q]);
                        acc[i][j] = zero16();
                    }
                }
            }
        }

        const int m0 = tm * BM + wm * 32 * RB;  // this wave's first row
        if constexpr (P == Product::kHead) {
#pragma unroll
            for (int i = 0; i < MB; i++) {
                const int v0 = m0 + 32 * i + 4 * hh;
                float u[16];
#pragma unroll
                for (int q = 0; q < 16; q++) {
                    const int v = min(v0 + 8 * (q >> 2) + (q & 3), g.vocab - 1);
                    u[q] = other ? __builtin_nanf("")
                                 : exp2i(group_exponent(__builtin_bit_cast(float, g.col_top[v]))) * (1.0f / 16384.0f);
                }
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    const int col = col0 + 32 * j + l32;
                    float* out = g.dhead + (long)v0 * g.d + col;
                    float old[16];
                    // (All reads before the first write: they are in flight together.)
#pragma unroll
                    for (int q = 0; q < 16; q++) {
                        const int r = 8 * (q >> 2) + (q & 3);
                        old[q] = g.acc && col < g.d && v0 + r < g.vocab ? out[(long)r * g.d] : 0.0f;
                    }
#pragma unroll
                    for (int q = 0; q < 16; q++) {
                        const int r = 8 * (q >> 2) + (q & 3);
                        if (col < g.d && v0 + r < g.vocab) out[(long)r * g.d] = fmaf(acc[i][j][q], u[q], old[q]);
                    }
                }
            }
        } else if constexpr (ROWS) {
            const int rows = g.mt * BM;
#pragma unroll
            for (int j = 0; j < CB; j++) {
                const int col = col0 + 32 * j + l32;
                float* out = g.part + ((long)o * g.chunk + col) * rows + m0 + 4 * hh;
                if (col < n)
#pragma unroll
                    for (int i = 0; i < RB; i++)
#pragma unroll
                        for (int q = 0; q < 4; q++)
                            *reinterpret_cast<float4*>(out + 32 * i + 8 * q) =
                                make_float4(tot[i][j][4 * q], tot[i][j][4 * q + 1], tot[i][j][4 * q + 2],
                                            tot[i][j][4 * q + 3]);
            }
        } else {
            if (!live_cols) continue;
            const int live = g.vocab - m0;  // rows of the head in this wave's part
            int e[MB];
#pragma unroll
            for (int i = 0; i < MB; i++) e[i] = wave_uniform(g.exponents[m0 / 32 + i]);
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const int col = col0 + 32 * j + l32;
                const bool scored = col < n;
                const int et = (int)(__builtin_bit_cast(uint32_t, g.scale[g.j0 + col]) >> 23) - 127;
                // The target's row within this wave's part; the rows of q lie at 4 hh.
                const int target = (scored ? g.targets[g.j0 + col] : -1) - m0;
                const int at = (target >= 0 && target < 32 * MB ? target : -1000) - 4 * hh;
                if (live < 32 * MB) {
                    const int end = live - 4 * hh;
#pragma unroll
                    for (int i = 0; i < MB; i++)
#pragma unroll
                        for (int q = 0; q < 16; q++)
                            if (32 * i + 8 * (q >> 2) + (q & 3) >= end) acc[i][j][q] = -INFINITY;
                }
                if (__any(at > -500)) {
                    float x = 0.0f;
                    bool hit = false;
                    int et_i = 0;
#pragma unroll
                    for (int i = 0; i < MB; i++)
#pragma unroll
                        for (int q = 0; q < 16; q++) {
                            const bool here = 32 * i + 8 * (q >> 2) + (q & 3) == at;
                            x = here ? acc[i][j][q] : x;
                            hit |= here;
                            if (q == 15) et_i = at >= 32 * i ? e[i] : et_i;
                        }
                    if (hit) g.xt[col] = x * pow2_clamped(et_i + et);
                }
                float c[MB], m = -INFINITY;
#pragma unroll
                for (int i = 0; i < MB; i++) {
                    c[i] = pow2_clamped(e[i] + et) * kLog2e;
                    float t = acc[i][j][0];
#pragma unroll
                    for (int q = 1; q < 16; q++) t = fmaxf(t, acc[i][j][q]);
                    m = fmaxf(m, t * c[i]);
                }
                m = max_halves(m);
                if (live <= 0) m = 0.0f;  // (its exponentials are zeros)
                float sum = 0.0f;
#pragma unroll
                for (int i = 0; i < MB; i++) {
                    float y[16];
#pragma unroll
                    for (int q = 0; q < 16; q += 4) {
#pragma unroll
                        for (int z = 0; z < 4; z++)
                            y[q + z] = __builtin_amdgcn_exp2f(fmaf(acc[i][j][q + z], c[i], -m));
                        sum += (y[q] + y[q + 1]) + (y[q + 2] + y[q + 3]);
                        __builtin_amdgcn_sched_barrier(0);  // (all at once take more registers than there are)
                    }
                    if (!g.keep) continue;
                    char* to = g.keep + ((long)(col0 / 32 + j) * g.v16 + m0 / 16 + 2 * i) * 2 * kFrag + lane * 16;
#pragma unroll
                    for (int q = 0; q < 16; q += 4) {
                        const f32x4 x = {y[q], y[q + 1], y[q + 2], y[q + 3]};
                        *reinterpret_cast<f32x4*>(to + q / 4 * kFrag) = scored ? x : f32x4{};
                    }
                }
                sum = sum_halves(sum);
                if (scored && hh == 0 && live > 0) g.stats[(long)(m0 / (32 * MB)) * g.ld + col] = make_float2(m, sum);
            }
        }
    }
}

// Sums of exp2 with their maxima.
__device__ __forceinline__ float2 join(const float2& a, const float2& b) {
    const float t = fmaxf(a.x, b.x);
    // (A sum of 0 is an empty part's, beside -inf; a NaN sum passes through.)
    return make_float2(t, (a.y == 0.0f ? 0.0f : a.y * exp2f(a.x - t)) + (b.y == 0.0f ? 0.0f : b.y * exp2f(b.x - t)));
}

struct MidArgs {
    const float* head;
    const char* rows;     // packed
    const int *count, *targets;  // targets: of scored rows
    const float* scale;
    float2* stats;        // [128 rows of the head][ld]
    float* xt;
    long ld;
    int vocab, d, k16, tag, groups, tiles, vec;
};
// Statistics of a thousand rows at most, the head split into pieces on its way from
// memory: where it is used by few tiles of tokens, packing it first costs more than
// splitting it for each (2048 x 128256 408 us).  128 rows of the head and 32 NB tokens to a workgroup, 32
// rows to a wave, whose pieces stay in registers; the tokens' operands go through LDS for
// all four waves.  The power of two of a wave's rows is that of the largest value so far:
// where a chunk has one that f16 does not hold, the sums are scaled down (rarely: after the
// first chunk one bit of room is left).  So it ends no higher than the packed head's.
// Bound by reading the head up to 64 rows (2048 x 128256 in all 250 us, 1.05 GB at 4.8 TB/s
// 220), then by the matrix cores beside the splitting (1024 rows, 538 GFLOP in three
// products, 1.6 ms, 1.0 PFLOP/s; MFMAs busy in half of the cycles).  The head's values two
// chunks ahead are not faster: 3% at 1024 rows, but 5% slower at 128 of 576 columns.
template <int NB, int K>
__global__ __launch_bounds__(256, 2) void head_mid_kernel(const MidArgs g) {
    constexpr int CHUNK = NB * K * 2 * kFrag;  // bytes of a chunk's operands of the tokens
    __shared__ __attribute__((aligned(1024))) char lds[2 * CHUNK];
    __shared__ float2 red[4][32 * NB];
    const int lane = threadIdx.x & 63, wave = wave_uniform(threadIdx.x >> 6), l32 = lane & 31, hh = lane >> 5;
    const int n = wave_uniform(scored_rows(g.count, g.tag, 0, INT_MAX));
    // The tiles of tokens of 128 rows of the head follow one another on one XCD.
    const int xcd = blockIdx.x % 8, local = blockIdx.x / 8;
    const int group = local / g.tiles * 8 + xcd, col0 = local % g.tiles * 32 * NB;
    if (group >= g.groups || col0 >= n) return;
    const bool upper = col0 + 16 * NB < n;  // tokens in the second half of the tile
    const int m0 = group * 128 + wave * 32;
    const float* row = g.head + (long)min(m0 + l32, g.vocab - 1) * g.d;
    const uint32_t lds0 = lds_offset(lds), voff = lane * 16;
    const int chunks = (g.k16 + K - 1) / K;
    auto load_head = [&](float (&x)[K][8], int c) {
        const int k = c * 16 * K + 8 * hh;
        if (g.vec && (c + 1) * 16 * K <= g.d) {
#pragma unroll
            for (int s = 0; s < K; s++) load8(x[s], row, k + 16 * s, INT_MAX, true);
        } else {
#pragma unroll
            for (int s = 0; s < K; s++) load8(x[s], row, k + 16 * s, g.d, g.vec);
        }
    };
    auto load_rows = [&](int c) {
        const int steps = min(K, g.k16 - c * K);
#pragma unroll
        for (int i = 0; i < NB * K / 2; i++) {
            const int at = NB * K / 2 * wave + i, j = at / (2 * K), s = at % (2 * K);  // block, KiB of it
            if (s / 2 < steps && (upper || j < NB / 2))
                lds_load16_so(g.rows + (((long)(col0 / 32 + j) * g.k16 + c * K) * 2 + s) * kFrag, voff,
                              lds0 + (c & 1) * CHUNK + at * kFrag);
        }
    };
    f32x16 acc[NB];
#pragma unroll
    for (int j = 0; j < NB; j++) acc[j] = zero16();
    float x[K][8], next[K][8];
    int e = -112;
    load_rows(0);
    load_head(x, 0);
    for (int c = 0; c < chunks; c++) {
        // The chunk's operands are there, and no wave reads the other buffer any more.
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        if (c + 1 < chunks) {
            load_rows(c + 1);
            load_head(next, c + 1);
        }
        float top = 0.0f;
#pragma unroll
        for (int s = 0; s < K; s++)
#pragma unroll
            for (int i = 0; i < 8; i++) top = fmaxf(top, fabsf(x[s][i]));
        if (__any(top * exp2i(-e) > 65504.0f)) {
            top = 0.0f;
#pragma unroll
            for (int s = 0; s < K; s++)
#pragma unroll
                for (int i = 0; i < 8; i++) top = fmaxf(top, finite_abs(x[s][i]));
#pragma unroll
            for (int o = 32; o >= 1; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
            const int more = wave_uniform(max(e, group_exponent(top)));
            const float down = pow2_clamped(e - more);
            e = more;
#pragma unroll
            for (int j = 0; j < NB; j++)
#pragma unroll
                for (int q = 0; q < 16; q++) acc[j][q] *= down;
        }
        const float sc = exp2i(-e);
        const char* b = lds + (c & 1) * CHUNK + voff;
#pragma unroll
        for (int s = 0; s < K; s++) {
            if (c * K + s >= g.k16) break;
            const Pieces a = split8(x[s], sc);
#pragma unroll
            for (int half = 0; half < 2; half++) {
                if (half && !upper) break;
                f16x8 h[NB / 2], l[NB / 2];
                const int j0 = half * NB / 2;
#pragma unroll
                for (int j = 0; j < NB / 2; j++) {
                    h[j] = *reinterpret_cast<const f16x8*>(b + (((j0 + j) * K + s) * 2) * kFrag);
                    l[j] = *reinterpret_cast<const f16x8*>(b + (((j0 + j) * K + s) * 2 + 1) * kFrag);
                }
#pragma unroll
                for (int j = 0; j < NB / 2; j++) acc[j0 + j] = mfma_f16(a.l, h[j], acc[j0 + j]);
#pragma unroll
                for (int j = 0; j < NB / 2; j++) acc[j0 + j] = mfma_f16(a.h, l[j], acc[j0 + j]);
#pragma unroll
                for (int j = 0; j < NB / 2; j++) acc[j0 + j] = mfma_f16(a.h, h[j], acc[j0 + j]);
            }
        }
#pragma unroll
        for (int s = 0; s < K; s++)
#pragma unroll
            for (int i = 0; i < 8; i++) x[s][i] = next[s][i];
    }
    const int live = g.vocab - m0;  // rows of the head of this wave
#pragma unroll
    for (int j = 0; j < NB; j++) {
        if (j >= NB / 2 && !upper) break;
        const int col = col0 + 32 * j + l32;
        const int et = (int)(__builtin_bit_cast(uint32_t, g.scale[col]) >> 23) - 127;
        const int target = (col < n ? g.targets[col] : -1) - m0;
        const int at = (target >= 0 && target < 32 ? target : -1000) - 4 * hh;
        float t = 0.0f;
        bool hit = false;
#pragma unroll
        for (int q = 0; q < 16; q++) {
            const int r = 8 * (q >> 2) + (q & 3);
            hit |= r == at;
            t = r == at ? acc[j][q] : t;
            if (r + 4 * hh >= live) acc[j][q] = -INFINITY;
        }
        if (hit) g.xt[col] = t * pow2_clamped(e + et);
        const float c = pow2_clamped(e + et) * kLog2e;
        float m = acc[j][0];
#pragma unroll
        for (int q = 1; q < 16; q++) m = fmaxf(m, acc[j][q]);
        m = max_halves(m * c);
        float sum = 0.0f;
#pragma unroll
        for (int q = 0; q < 16; q++) sum += __builtin_amdgcn_exp2f(fmaf(acc[j][q], c, -m));
        sum = sum_halves(sum);
        if (hh == 0) red[wave][32 * j + l32] = live > 0 ? make_float2(m, sum) : make_float2(-INFINITY, 0.0f);
    }
    __syncthreads();
    if (threadIdx.x < 32 * NB && col0 + (int)threadIdx.x < n) {
        float2 a = red[0][threadIdx.x];
#pragma unroll
        for (int w = 1; w < 4; w++) a = join(a, red[w][threadIdx.x]);
        g.stats[(long)group * g.ld + col0 + threadIdx.x] = a;
    }
}

// lse and logp (or null) of scored rows [j0, ..) from their parts' maxima and sums,
// and what the gradient scales a part by (or null).  16 rows to a workgroup, lane l
// has row l % 16, so that a part's are read side by side.  Bound by the latency of a
// thread's parts: 7 us for 384 of them, 14 for 1002.
__global__ __launch_bounds__(1024) void head_finish_kernel(const float2* __restrict__ stats, long ld, int parts,
                                                           int all_parts, const float* __restrict__ xt,
                                                           const int* __restrict__ idx, const int* __restrict__ count,
                                                           int tag, int j0, int chunk, float* __restrict__ logp,
                                                           float* __restrict__ lse, float* __restrict__ factor) {
    __shared__ float2 red[16][16];
    __shared__ float2 all[16];
    const int c = threadIdx.x & 15, p0 = threadIdx.x >> 4, j = blockIdx.x * 16 + c;
    const int n = scored_rows(count, tag, j0, chunk);
    if ((int)blockIdx.x * 16 >= (n + kBN - 1) / kBN * kBN) return;
    float2 a = make_float2(-INFINITY, 0.0f);
    if (j < n)
        for (int p = p0; p < parts; p += 64) a = join(a, stats[p * ld + j]);
    a = join(a, make_float2(__shfl_xor(a.x, 16), __shfl_xor(a.y, 16)));
    a = join(a, make_float2(__shfl_xor(a.x, 32), __shfl_xor(a.y, 32)));
    if ((threadIdx.x & 63) < 16) red[threadIdx.x >> 6][c] = a;
    __syncthreads();
    if (p0 == 0) {
        for (int w = 1; w < 16; w++) a = join(a, red[w][c]);
        all[c] = make_float2(a.x, 1.0f / a.y);
        if (j < n && logp) {
            // Units of kLog2e as rounded: the quotient has the largest logit's own bits.
            const double l = (double)a.x / (double)kLog2e + log((double)a.y);
            const int r = idx[j0 + j];
            lse[r] = (float)l;
            logp[r] = (float)((double)xt[j] - l);
        }
    }
    if (!factor) return;
    __syncthreads();
    // (By the largest logit and the sum: an lse in f32 is off by 2^-24 of itself, and so would
    // be every probability; 1 - P of a likely token is much less.)
    for (int p = p0; p < all_parts; p += 64)
        factor[p * ld + j] = j < n && p < parts ? exp2f(stats[p * ld + j].x - all[c].x) * all[c].y : 0.0f;
}

// dhn of scored rows [j0, ..): dlogp (head[target] - the splits' sums in order).
// Four columns to a thread, eight splits' sums in flight: bound by memory, 3686 x 576 with
// 16 splits (136 MB) 29 us.
__global__ __launch_bounds__(256) void head_grad_reduce_kernel(const float* __restrict__ part, int chunk, int rows,
                                                               int mt, int k16, int splits_max,
                                                               const int* __restrict__ idx,
                                                               const int* __restrict__ targets,
                                                               const int* __restrict__ count, int tag, int j0,
                                                               const float* __restrict__ head,
                                                               const float* __restrict__ dlogp,
                                                               float* __restrict__ dhn, int d) {
    const int n = scored_rows(count, tag, j0, chunk);
    const int quads = (d + 3) / 4;
    const long at = (long)blockIdx.x * 256 + threadIdx.x;
    const int col = (int)(at / quads), i0 = (int)(at % quads) * 4;
    if (col >= n) return;
    const int splits = splits_of(mt * ((n + kBN - 1) / kBN), k16, splits_max).count;  // (a multiple of 8)
    const float* p = part + (long)col * rows + i0;
    const long step = (long)chunk * rows;
    float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int q = 0; q < splits; q += 8) {
        float4 x[8];
#pragma unroll
        for (int z = 0; z < 8; z++) x[z] = *reinterpret_cast<const float4*>(p + (q + z) * step);
#pragma unroll
        for (int z = 0; z < 8; z++) s.x += x[z].x, s.y += x[z].y, s.z += x[z].z, s.w += x[z].w;
    }
    const long r = idx[j0 + col];
    const float* w = head + (long)targets[j0 + col] * d + i0;
    float* out = dhn + r * d + i0;
    const float f = dlogp[r], t[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (i0 + i < d) out[i] = f * (w[i] - t[i]);
}

// What the head's gradient takes of what statistics kept, for scored rows [j0, ..).
struct DlogitsArgs {
    const char* keep;     // from row j0 on
    const float* factor;
    const int *idx, *targets, *count;
    const float *dlogp, *scale;
    unsigned* col_top;
    char* out;            // [32 columns][t16][piece]
    long ld;
    int v16, t16, tag, j0, chunk, vocab;
};

// 2^14 and the power of two of a row of hn: a power of two near its largest value, so
// that a dlogit times it is as large as what the row adds to the head's gradient.
__device__ __forceinline__ float row_top(float scale) { return scale * 16384.0f; }

// The largest of every column's dlogits times their rows' row_top: a column's power of
// two is its own, since a token that is rarely likely has gradients far below the
// others', which an optimizer that divides by their size scales up.  128 columns and
// every 8th 32 rows to a workgroup: 819 rows x 50001 (180 MB) 31 us.  (At a target 1 - P
// counts as 1.)
__global__ __launch_bounds__(256) void head_col_top_kernel(const DlogitsArgs g) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l32 = lane & 31, hh = lane >> 5;
    const int n = scored_rows(g.count, g.tag, g.j0, g.chunk);
    float top[2][8] = {};
    for (int t0 = 32 * blockIdx.y; t0 < n; t0 += 32 * gridDim.y) {
        const int j = t0 + l32;
        if (j >= n) continue;
        const float row = fabsf(g.dlogp[g.idx[g.j0 + j]] * row_top(g.scale[g.j0 + j]));
        const float f = g.factor[blockIdx.x * g.ld + j];
#pragma unroll
        for (int q = 0; q < 2; q++) {
            const f32x4* y = reinterpret_cast<const f32x4*>(
                g.keep + ((long)(t0 / 32) * g.v16 + blockIdx.x * 8 + 2 * wave + q) * 2 * kFrag + lane * 16);
            const f32x4 a = y[0], b = y[kFrag / 16];
#pragma unroll
            for (int i = 0; i < 8; i++)
                top[q][i] = fmaxf(top[q][i], finite_abs((i < 4 ? a[i] : b[i - 4]) * f * row));
        }
        // (One workgroup of the columns sees to a row's target.)
        if (blockIdx.x == 0 && wave == 0 && hh == 0)
            atomicMax(g.col_top + g.targets[g.j0 + j], __builtin_bit_cast(unsigned, finite_abs(row)));
    }
#pragma unroll
    for (int q = 0; q < 2; q++)
#pragma unroll
        for (int i = 0; i < 8; i++) {
            float x = top[q][i];
#pragma unroll
            for (int o = 16; o >= 1; o >>= 1) x = fmaxf(x, __shfl_xor(x, o));
            const int v = blockIdx.x * 128 + 16 * (2 * wave + q) + 8 * (i >> 2) + 4 * hh + (i & 3);
            if (l32 == 0 && v < g.vocab) atomicMax(g.col_top + v, __builtin_bit_cast(unsigned, x));
        }
}

// The dlogits times their rows' row_top as operands by columns: 32 rows and 128 columns
// to a workgroup, turned round in LDS.  Bound by memory: 819 x 50001, read and written,
// (328 MB) 54 us.
__global__ __launch_bounds__(256) void head_pack_dlogits_kernel(const DlogitsArgs g) {
    __shared__ float tile[32][129];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l32 = lane & 31, hh = lane >> 5;
    const int n = scored_rows(g.count, g.tag, g.j0, g.chunk), t0 = blockIdx.y * 32, j = t0 + l32;
    if (t0 >= n) return;
    const bool scored = j < n;
    const long r = scored ? g.idx[g.j0 + j] : 0;
    const float row = scored ? g.dlogp[r] * row_top(g.scale[g.j0 + j]) : 0.0f;
    const float f = scored ? g.factor[blockIdx.x * g.ld + j] : 0.0f;
    const int target = scored ? g.targets[g.j0 + j] - (int)blockIdx.x * 128 : -1;
#pragma unroll
    for (int q = 0; q < 2; q++) {
        const int s = 2 * wave + q;  // 16 columns
        const f32x4* y = reinterpret_cast<const f32x4*>(
            g.keep + ((long)blockIdx.y * g.v16 + blockIdx.x * 8 + s) * 2 * kFrag + lane * 16);
        const f32x4 a = y[0], b = y[kFrag / 16];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int c = 16 * s + 8 * (i >> 2) + 4 * hh + (i & 3);
            // (Rows from n on are zeros, whatever their factor.)
            tile[l32][c] = scored ? row * ((c == target ? 1.0f : 0.0f) - (i < 4 ? a[i] : b[i - 4]) * f) : 0.0f;
        }
    }
    __syncthreads();
    const int v = blockIdx.x * 128 + 32 * wave + l32;
    const float sc = exp2i(-group_exponent(v < g.vocab ? __builtin_bit_cast(float, g.col_top[v]) : 0.0f));
#pragma unroll
    for (int q = 0; q < 2; q++) {
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = tile[16 * q + 8 * (i >> 2) + 4 * hh + (i & 3)][32 * wave + l32];
        store_pieces(g.out + ((long)(blockIdx.x * 4 + wave) * g.t16 + blockIdx.y * 2 + q) * 2 * kFrag, lane,
                     split8(x, sc));
    }
}

// Zeros in the rows that are not among the ascending idx.
__global__ __launch_bounds__(256) void head_zero_rows_kernel(const int* __restrict__ idx,
                                                             const int* __restrict__ count, int tag,
                                                             float* __restrict__ dhn, int d) {
    const int r = blockIdx.x, n = scored_rows(count, tag, 0, INT_MAX);
    int lo = 0, hi = n;
    while (lo < hi) {
        const int mid = (lo + hi) / 2;
        if (idx[mid] < r)
            lo = mid + 1;
        else
            hi = mid;
    }
    if (lo < n && idx[lo] == r) return;
    const float x = count[1] == tag ? 0.0f : __builtin_nanf("");
    for (int i = threadIdx.x; i < d; i += 256) dhn[(long)r * d + i] = x;
}

inline bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }
size_t up(size_t x, size_t to) { return (x + to - 1) / to * to; }

constexpr int kSplitsMax = 32;
constexpr size_t kPartBytes = (size_t)512 << 20;

// Rows of a pass of their gradient: those whose sums, by eight splits (of which there are
// no fewer), fit kPartBytes, and of them those that fill whole rounds of an XCD's workgroups
// with their tiles (mt to 128 rows).  (Us of the gradient in such passes, in ones of half
// the bytes and in one: 20000 x 1024 x 32000 4930, 4810 and 4940, 32768 x 2048 x 16000 7240,
// 7250 and 7480, 65536 x 576 x 8000 2390, 2400 and 2360, 16384 x 4096 x 32000 14830, 17240 and
// 15660; the third in passes of half the bytes that fill no whole rounds 3010.)
size_t pass_rows(size_t d_pad, size_t mt, size_t chunk) {
    const size_t fit = std::max<size_t>(kPartBytes / (8 * d_pad * sizeof(float) * kBN), 1);
    if (fit * kBN >= chunk) return chunk;
    const size_t round = kWgs / 8, tiles = mt * fit / round * round;
    return kBN * (tiles ? tiles / mt : fit);
}

}  // namespace

HeadPlan head_plan(size_t t, size_t d, size_t vocab, size_t chunk_bytes) {
    HeadPlan p{};
    p.tag = (int)((uint32_t)t * 0x9E3779B1u ^ (uint32_t)d * 0x85EBCA77u ^ (uint32_t)vocab * 0xC2B2AE3Du ^ 0x6C6F6770u);
    p.k16 = (int)((d + 15) / 16);
    p.v_pad = up(vocab, 256);
    p.t_pad = up(t, kBN);
    p.chunk = std::min(std::max<size_t>(chunk_bytes / (p.v_pad * 4) / kBN * kBN, kBN), p.t_pad);
    // Half the blocks of 32 columns of the head of a wave in the rows' gradient (whose sums take
    // twice the registers): two or three, by which the tiles fill the card better, were
    // all rows of a pass scored.  (Us of the gradient by three and by two: 500 x 2048 x 49152
    // 417 and 394, 300 x 576 x 49152 107 and 98, 1000 x 768 x 32000 174 and 206, 2000 x 129 x
    // 49152 145 and 191.)
    float least = INFINITY;
    for (int mb = 3; mb >= 2; mb--) {
        const size_t d_pad = up(d, 64 * mb);
        const size_t pass = pass_rows(d_pad, d_pad / (64 * mb), p.chunk);
        const size_t most = std::min(kPartBytes / 2 / (pass * d_pad * sizeof(float)), p.v_pad / 256) / 8 * 8;
        const int splits_max = (int)std::min<size_t>(std::max<size_t>(most, 8), kSplitsMax);
        const Splits s = splits_of((int)(d_pad / (64 * mb) * (pass / kBN)), (int)(p.v_pad / 16), splits_max);
        const float cost = (mb == 3 ? 2.9f : 2.0f) * s.cost / pass;
        if (cost >= least) continue;
        least = cost;
        p.back_mb = mb, p.d_pad = d_pad, p.splits_max = splits_max, p.pass = pass;
    }
    p.rows_bytes = p.t_pad * p.k16 * 64;
    p.head_bytes = p.v_pad * p.k16 * 64;
    p.back_bytes = p.d_pad * p.v_pad * 4;
    p.stats_bytes = (p.v_pad / 128) * p.chunk * sizeof(float2);
    p.keep_bytes = p.chunk * p.v_pad * 4;
    p.factor_bytes = (p.v_pad / 128) * p.chunk * sizeof(float);
    p.rows_back_bytes = up(d, kBN) * p.t_pad * 4;
    p.part_bytes = (size_t)p.splits_max * p.pass * p.d_pad * sizeof(float);
    return p;
}

hipError_t launch_head_pack(const HeadPlan& p, const HeadBuffers& b, const float* hn, const float* head, size_t d,
                            size_t vocab, hipStream_t st) {
    PackArgs g{};
    g.hn = hn, g.head = head, g.idx = b.idx, g.count = b.count, g.rows = b.rows, g.packed = b.packed, g.back = b.back;
    g.rows_back = b.rows_back, g.t16 = (int)(p.t_pad / 16);
    g.scale = b.scale, g.exponents = b.exponents, g.row_blocks = (int)(p.t_pad / 32);
    g.vocab = (int)vocab, g.d = (int)d, g.k16 = p.k16, g.v16 = (int)(p.v_pad / 16);
    g.vec_rows = d % 4 == 0 && aligned16(hn), g.vec_head = d % 4 == 0 && aligned16(head);
    g.tag = p.tag;
    const size_t blocks = (p.t_pad + (head ? p.v_pad : 0)) / 32;
    const int pairs = (p.k16 + 1) / 2;
    auto pack = [&](auto back, auto nw, auto u) {
        constexpr int kNw = decltype(nw)::value;
        hipLaunchKernelGGL((pack_kernel<decltype(back)::value, kNw, decltype(u)::value>),
                           dim3((unsigned)blocks), dim3(64 * kNw), 0, st, g);
    };
    using std::integral_constant;
    auto sized = [&](auto back) {
        // The fewest registers that hold the rows.
        if (pairs <= 8)
            pack(back, integral_constant<int, 8>{}, integral_constant<int, 1>{});
        else if (pairs <= 24)
            pack(back, integral_constant<int, 8>{}, integral_constant<int, 3>{});
        else if (pairs <= 64)
            pack(back, integral_constant<int, 16>{}, integral_constant<int, 4>{});
        else
            pack(back, integral_constant<int, 8>{}, integral_constant<int, 0>{});
    };
    if (b.back || b.rows_back)
        sized(std::true_type{});
    else
        sized(std::false_type{});
    return hipGetLastError();
}

hipError_t launch_head_stats(const HeadPlan& p, const HeadBuffers& b, size_t t, size_t j0, size_t vocab,
                             float* logp, float* lse, hipStream_t st) {
    HeadArgs g{};
    g.a = b.packed, g.b = b.rows + j0 / 32 * p.k16 * 2 * kFrag, g.ka = g.kb = p.k16, g.mt = (int)(p.v_pad / 256);
    g.count = b.count, g.j0 = (int)j0, g.chunk = (int)p.chunk, g.ld = (long)p.chunk, g.exponents = b.exponents;
    g.targets = b.idx + t, g.scale = b.scale, g.tag = p.tag, g.vocab = (int)vocab;
    g.v16 = (int)(p.v_pad / 16), g.stats = static_cast<float2*>(b.stats), g.xt = b.xt, g.keep = b.keep;
    hipLaunchKernelGGL((head_gemm_kernel<4, Product::kStats>), dim3(kWgs), dim3(256), 0, st, g);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(head_finish_kernel, dim3((unsigned)(p.chunk / 16)), dim3(1024), 0, st, g.stats, g.ld,
                       (int)((vocab + 127) / 128), (int)(p.v_pad / 128), b.xt, b.idx, b.count, p.tag, (int)j0,
                       (int)p.chunk, logp, lse, b.keep ? b.factor : nullptr);
    return hipGetLastError();
}

hipError_t launch_head_mid(const HeadPlan& p, const HeadBuffers& b, const float* head, size_t t, size_t d, size_t vocab,
                           float* logp, float* lse, hipStream_t st) {
    MidArgs g{};
    g.head = head, g.rows = b.rows, g.count = b.count, g.targets = b.idx + t, g.scale = b.scale;
    g.stats = static_cast<float2*>(b.stats), g.xt = b.xt, g.ld = (long)p.chunk, g.vocab = (int)vocab, g.d = (int)d;
    g.k16 = p.k16, g.tag = p.tag, g.groups = (int)((vocab + 127) / 128), g.vec = d % 4 == 0 && aligned16(head);
    // Tiles of 256 tokens, which split the head half as often, take 1.75 times as long as
    // ones of 128: the ones with less time in rounds of two workgroups to a CU.  (Us by 128
    // and by 256: 200 rows 2048 x 32000 139 and 184, 2048 x 49152 238 and 218, 400 rows 252
    // and 234, 371 and 392.)
    auto rounds = [&](size_t tile) { return (g.groups * ((t + tile - 1) / tile) + kWgs - 1) / kWgs; };
    const int nb = t <= 64 ? 2 : 4 * rounds(128) <= 7 * rounds(256) ? 4 : 8;
    g.tiles = (int)((t + 32 * nb - 1) / (32 * nb));
    hipLaunchKernelGGL((nb == 2 ? head_mid_kernel<2, 4> : nb == 4 ? head_mid_kernel<4, 4> : head_mid_kernel<8, 2>),
                       dim3((unsigned)((g.groups + 7) / 8 * 8 * g.tiles)), dim3(256), 0, st, g);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(head_finish_kernel, dim3((unsigned)(p.chunk / 16)), dim3(1024), 0, st, g.stats, g.ld, g.groups,
                       g.groups, b.xt, b.idx, b.count, p.tag, 0, (int)p.chunk, logp, lse, nullptr);
    return hipGetLastError();
}

hipError_t launch_head_dhn(const HeadPlan& p, const HeadBuffers& b, size_t t, const float* head,
                           const float* dlogp, size_t j0, size_t local, size_t rows, size_t d, float* dhn,
                           hipStream_t st) {
    const int mb = p.back_mb;
    HeadArgs g{};
    g.a = b.back, g.b = b.keep + local * p.v_pad * 4, g.ka = g.kb = (int)(p.v_pad / 16);
    g.mt = (int)(p.d_pad / (64 * mb)), g.count = b.count, g.j0 = (int)(j0 + local), g.chunk = (int)rows;
    g.ld = (long)p.chunk, g.factor = b.factor + local, g.part = b.part;
    g.splits_max = p.splits_max, g.tag = p.tag, g.exponents = b.exponents;
    if (mb == 3)
        hipLaunchKernelGGL((head_gemm_kernel<3, Product::kRows>), dim3(kWgs), dim3(256), 0, st, g);
    else
        hipLaunchKernelGGL((head_gemm_kernel<2, Product::kRows>), dim3(kWgs), dim3(256), 0, st, g);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    const size_t quads = rows * ((d + 3) / 4);
    hipLaunchKernelGGL(head_grad_reduce_kernel, dim3((unsigned)((quads + 255) / 256)), dim3(256), 0, st, b.part, g.chunk,
                       (int)p.d_pad, g.mt, g.ka, g.splits_max, b.idx, b.idx + t, b.count, p.tag, g.j0, head,
                       dlogp, dhn, (int)d);
    return hipGetLastError();
}

hipError_t launch_head_dhead(const HeadPlan& p, const HeadBuffers& b, size_t t, const float* dlogp,
                             size_t j0, size_t local, size_t rows, size_t d, size_t vocab, char* packed_dlogits,
                             unsigned* col_top, float* dhead, int acc, hipStream_t st) {
    DlogitsArgs g{};
    g.keep = b.keep + local * p.v_pad * 4, g.factor = b.factor + local;
    g.idx = b.idx, g.count = b.count, g.targets = b.idx + t, g.dlogp = dlogp, g.tag = p.tag;
    g.scale = b.scale, g.col_top = col_top, g.out = packed_dlogits, g.ld = (long)p.chunk, g.v16 = (int)(p.v_pad / 16);
    g.t16 = (int)(up(rows, 32) / 16), g.j0 = (int)(j0 + local), g.chunk = (int)rows, g.vocab = (int)vocab;
    hipError_t e = launch_fill_zero(reinterpret_cast<float*>(col_top), vocab, st);
    if (e != hipSuccess) return e;
    const unsigned t32 = (unsigned)((rows + 31) / 32), v128 = (unsigned)(p.v_pad / 128);
    hipLaunchKernelGGL(head_col_top_kernel, dim3(v128, std::min(t32, 8u)), dim3(256), 0, st, g);
    if ((e = hipGetLastError()) != hipSuccess) return e;
    hipLaunchKernelGGL(head_pack_dlogits_kernel, dim3(v128, t32), dim3(256), 0, st, g);
    if ((e = hipGetLastError()) != hipSuccess) return e;
    HeadArgs h{};
    h.a = packed_dlogits, h.b = b.rows_back + (j0 + local) / 16 * 2 * kFrag, h.ka = g.t16, h.kb = (int)(p.t_pad / 16);
    h.mt = (int)(p.v_pad / 256), h.nt = (int)((d + kBN - 1) / kBN), h.count = b.count, h.j0 = g.j0, h.chunk = g.chunk;
    h.tag = p.tag, h.vocab = (int)vocab, h.col_top = col_top, h.dhead = dhead, h.d = (int)d, h.acc = acc;
    hipLaunchKernelGGL((head_gemm_kernel<4, Product::kHead>), dim3(kWgs), dim3(256), 0, st, h);
    return hipGetLastError();
}

hipError_t launch_head_zero_rows(const HeadPlan& p, const HeadBuffers& b, size_t t, float* dhn, size_t d,
                                 hipStream_t st) {
    hipLaunchKernelGGL(head_zero_rows_kernel, dim3((unsigned)t), dim3(256), 0, st, b.idx, b.count, p.tag, dhn, (int)d);
    return hipGetLastError();
}

}  // namespace cfattn
