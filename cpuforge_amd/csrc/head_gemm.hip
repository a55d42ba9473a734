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
// sums leave.  The gradients of logits lie in [-1, 1] times their row's dlogp: they
// are formed without it, times 2^15 at most, and it multiplies the row at the end.
//
// Packed operands: both are first written as MFMA operands (1 KiB: a lane's eight
// f16, 64 lanes) of 32 rows and 16 k, the two pieces side by side, so a
// stage goes to LDS by direct loads of whole KiB and is read without bank
// conflicts, and no wave spends instructions on splitting.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "cfattn_common.hpp"
#include "cfops_kernels.hpp"

namespace cfattn {
namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr int kFrag = 1024;        // bytes of an operand of one MFMA
constexpr int kBN = 128;           // tokens of a tile
constexpr int kWgs = 512;          // two workgroups to a CU
constexpr int kStages = 3;
constexpr int kGroup = 8;          // token tiles
constexpr float kTop = 32768.0f;   // of a dlogit over dlogp

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

struct Pieces {
    f16x8 h, l;
};
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

// The scored rows of hn, 32 to a workgroup, as operands [32 rows][16 k][piece], and
// each row's 2^e; rows from n on are zeros.
__global__ __launch_bounds__(256) void pack_rows_kernel(const float* __restrict__ hn, const int* __restrict__ idx,
                                                        const int* __restrict__ count, char* __restrict__ out,
                                                        float* __restrict__ scale, int d, int k16, int vec) {
    __shared__ float red[4][32];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, j = blockIdx.x * 32 + (lane & 31);
    const int n = *count;
    if ((int)blockIdx.x * 32 >= (n + kBN - 1) / kBN * kBN) return;
    const float* row = j < n ? hn + (long)idx[j] * d : nullptr;
    const bool v = vec && row;
    float top = 0.0f, x[8];
    for (int s = wave; s < k16; s += 4) {
        load8(x, row, 16 * s + 8 * (lane >> 5), d, v);
#pragma unroll
        for (int i = 0; i < 8; i++) top = fmaxf(top, finite_abs(x[i]));
    }
    top = max_halves(top);
    if (lane < 32) red[wave][lane] = top;
    __syncthreads();
    top = fmaxf(fmaxf(red[0][lane & 31], red[1][lane & 31]), fmaxf(red[2][lane & 31], red[3][lane & 31]));
    const int e = group_exponent(top);
    if (wave == 0 && lane < 32) scale[j] = exp2i(e);
    for (int s = wave; s < k16; s += 4) {
        load8(x, row, 16 * s + 8 * (lane >> 5), d, v);
        store_pieces(out + ((long)blockIdx.x * k16 + s) * 2 * kFrag, lane, split8(x, exp2i(-e)));
    }
}

// 32 rows of the head to a workgroup, as operands [32 rows][16 k][piece] with
// their e, and, for the hidden states' gradient, whose k are these rows, as
// [32 columns][16 rows][piece].  There lane l holds column l % 32 and of 16 rows
// those that it holds of a product's 32 x 32 result: 4 (l / 32) + 0..3 and the
// same eight on.
// A wave takes the pairs of operands (32 columns) w, w + NW, ..; with U > 0 at most U
// of them, which stay in registers between the largest value and the pieces.  (The 32
// rows of 2048 columns that each workgroup has read are 0.5 GB on all CUs together:
// read again, they came from HBM again, 640 us for 128256 x 2048 at 3.3 TB/s of one
// read and one write.)
template <bool BACK, int NW, int U>
__global__ __launch_bounds__(64 * NW) void pack_head_kernel(const float* __restrict__ head, char* __restrict__ out,
                                                            char* __restrict__ back, int* __restrict__ exponents,
                                                            int* __restrict__ largest, int vocab, int d, int k16,
                                                            int v16, int vec) {
    __shared__ float red[NW];
    __shared__ uint32_t tile[BACK ? NW : 1][32][33];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r0 = blockIdx.x * 32, r = r0 + (lane & 31);
    const float* row = r < vocab ? head + (long)r * d : nullptr;
    const bool v = vec && row;
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
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
    if (lane == 0) red[wave] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < NW; w++) top = fmaxf(top, red[w]);
    const int e = group_exponent(top);
    if (threadIdx.x == 0) {
        exponents[blockIdx.x] = e;
        if (BACK) atomicMax(largest, e);
    }
    const float sc = exp2i(-e);
    auto store = [&](const float (&y)[2][8], int s) {
#pragma unroll
        for (int q = 0; q < 2; q++) {
            const Pieces p = split8(y[q], sc);
            if (2 * s + q < k16)
                store_pieces(out + ((long)blockIdx.x * k16 + 2 * s + q) * 2 * kFrag, lane, p);
            if constexpr (BACK)
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    // (Copies: a bit cast of a vector's element itself takes element 0.)
                    const _Float16 h = p.h[i], l = p.l[i];
                    tile[wave][lane & 31][16 * q + c + i] = (uint32_t)__builtin_bit_cast(uint16_t, h) |
                                                            (uint32_t)__builtin_bit_cast(uint16_t, l) << 16;
                }
        }
        if constexpr (BACK) {
            // (A wave's own part of LDS: its own order of accesses is enough.)
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int q = 0; q < 2; q++) {
                Pieces p;
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const uint32_t u = tile[wave][16 * q + 8 * (i >> 2) + 4 * (lane >> 5) + (i & 3)][lane & 31];
                    p.h[i] = __builtin_bit_cast(_Float16, (uint16_t)u);
                    p.l[i] = __builtin_bit_cast(_Float16, (uint16_t)(u >> 16));
                }
                store_pieces(back + ((long)s * v16 + blockIdx.x * 2 + q) * 2 * kFrag, lane, p);
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

enum class Epi { kStats, kGrad, kPartial };

struct HeadArgs {
    const char *a, *b;   // operands: rows of the result along a (BM to a tile), tokens along b
    int k16;             // 16-k steps of an operand
    int mt;              // tiles along a
    const int* count;    // scored rows
    int j0, chunk;       // this launch's: [j0, min(j0 + chunk, count))
    // stats and grad: a is the head
    const int* exponents;
    const float* scale;
    const int64_t* targets;
    const int* idx;
    int vocab;
    float2* stats;       // [128 rows of the head][ld]: max and sum of exp2, in log2 units
    long ld;
    float* xt;           // the targets' logits
    // grad
    const float* lse;
    const float* dlogp;
    const int* largest;
    char* grad;          // [32 tokens][v16][piece]
    int v16;
    float* dlogits;      // or null: [chunk][vocab]
    // partial: a is the head by columns, b the gradients
    float* part;         // [split][chunk][BM * mt]
    int splits_max;
};

// Splits of the hidden states' gradient's k (the vocabulary) over workgroups: a
// multiple of the XCDs, so that one XCD's L2 holds what its workgroups share.  The
// one with the least rounds of its share of the 64 workgroups of an XCD times its
// length; a split's partial sums cost their way through memory.
__device__ __forceinline__ int splits_of(int tiles, int k16, int splits_max) {
    int best = 8;
    float least = INFINITY;
    for (int s = 8; s <= splits_max; s += 8) {
        const int rounds = (tiles * (s / 8) + kWgs / 8 - 1) / (kWgs / 8);
        const float cost = rounds * ((k16 + s - 1) / s + 24.0f) + 0.35f * tiles * s / 64.0f;
        if (cost < least) least = cost, best = s;
    }
    return best;
}

// A tile of BM = 64 MB rows and kBN tokens to a workgroup of four waves, each 32 MB x 64;
// two workgroups to a CU: one's epilogue runs beside the other's products.
template <int MB, Epi E>
__global__ __launch_bounds__(256, 2) void head_gemm_kernel(const HeadArgs g) {
    constexpr int BM = 64 * MB, CH = 4 * MB + 8, STAGE = CH * kFrag, PER = CH / 4;
    static_assert(CH % 4 == 0, "whole loads a wave");
    __shared__ __attribute__((aligned(1024))) char lds[kStages * STAGE];
    const int lane = threadIdx.x & 63, wave = wave_uniform(threadIdx.x >> 6);
    const int wm = wave >> 1, wn = wave & 1, l32 = lane & 31, hh = lane >> 5;
    const int n = min(wave_uniform(*g.count) - g.j0, g.chunk);
    if (n <= 0) return;
    const int nt = (n + kBN - 1) / kBN;
    // Items of an XCD: a contiguous run of the tiles along a (of the splits), every
    // token tile with each.
    const int xcd = blockIdx.x % 8, local = blockIdx.x / 8;
    int outer = g.mt, inner = nt, splits = 1;
    if constexpr (E == Epi::kPartial) {
        splits = wave_uniform(splits_of(g.mt * nt, g.k16, g.splits_max));
        outer = splits;
        inner = g.mt * nt;
    }
    const int o0 = (int)((long)outer * xcd / 8), o1 = (int)((long)outer * (xcd + 1) / 8);
    const uint32_t lds0 = lds_offset(lds), voff = lane * 16;
    for (int item = local; item < (o1 - o0) * inner; item += kWgs / 8) {
        // Stats and grad: kGroup token tiles with every tile along a of the XCD, then the
        // next ones: what 64 workgroups read at a time is near a square, and the tokens'
        // operands stay in the XCD's L2.
        int o, tm, tt;
        if constexpr (E == Epi::kPartial) {
            o = wave_uniform(o0 + item / inner);
            tm = wave_uniform(item % inner % g.mt);
            tt = wave_uniform(item % inner / g.mt);
        } else {
            const int grp = item / ((o1 - o0) * kGroup), left = item - grp * (o1 - o0) * kGroup;
            const int w = min(kGroup, nt - grp * kGroup);
            o = tm = wave_uniform(o0 + left / w);
            tt = wave_uniform(grp * kGroup + left % w);
        }
        int k0 = 0, k1 = g.k16;
        if constexpr (E == Epi::kPartial) {
            k0 = wave_uniform((int)((long)g.k16 * o / splits));
            k1 = wave_uniform((int)((long)g.k16 * (o + 1) / splits));
        }
        const char* src[PER];
#pragma unroll
        for (int i = 0; i < PER; i++) {
            const int c = PER * wave + i;  // the stage's KiB: operand c / 2, piece c % 2
            const int blk = c / 2;
            const char* base = blk < 2 * MB ? g.a + ((long)(tm * 2 * MB + blk) * g.k16 + k0) * 2 * kFrag
                                            : g.b + ((long)(tt * 4 + blk - 2 * MB) * g.k16 + k0) * 2 * kFrag;
            src[i] = base + (c % 2) * kFrag;
        }
        auto load = [&](uint32_t stage) {
#pragma unroll
            for (int i = 0; i < PER; i++) {
                lds_load16_so(src[i], voff, lds0 + stage + (PER * wave + i) * kFrag);
                src[i] += 2 * kFrag;
            }
        };
        f32x16 acc[MB][2];
#pragma unroll
        for (int i = 0; i < MB; i++) acc[i][0] = acc[i][1] = zero16();
        // Every wave is done with the LDS of the item before, and with its stores
        // (they would count among the loads waited for below).
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        uint32_t cur = 0, nxt = 2 * STAGE;
        load(0);
        if (k0 + 1 < k1) load(STAGE);
        for (int k = k0; k < k1; k++) {
            if (k + 1 < k1) {
                if constexpr (PER == 6)
                    asm volatile("s_waitcnt vmcnt(6) lgkmcnt(0)" ::: "memory");
                else
                    asm volatile("s_waitcnt vmcnt(5) lgkmcnt(0)" ::: "memory");
            } else {
                asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
            }
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
            if (k + 2 < k1) load(nxt);
            nxt = nxt == (kStages - 1) * STAGE ? 0 : nxt + STAGE;
            const char* s = lds + cur;
            cur = cur == (kStages - 1) * STAGE ? 0 : cur + STAGE;
            f16x8 a[MB][2], b[2][2];
#pragma unroll
            for (int p = 0; p < 2; p++) {
#pragma unroll
                for (int j = 0; j < 2; j++)
                    b[j][p] = *reinterpret_cast<const f16x8*>(s + ((2 * MB + wn * 2 + j) * 2 + p) * kFrag + voff);
#pragma unroll
                for (int i = 0; i < MB; i++)
                    a[i][p] = *reinterpret_cast<const f16x8*>(s + ((wm * MB + i) * 2 + p) * kFrag + voff);
            }
            constexpr int pa[3] = {1, 0, 0}, pb[3] = {0, 1, 0};
#pragma unroll
            for (int q = 0; q < 3; q++)
#pragma unroll
                for (int i = 0; i < MB; i++)
#pragma unroll
                    for (int j = 0; j < 2; j++)
                        acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[i][pa[q]], b[j][pb[q]], acc[i][j], 0, 0, 0);
        }

        const int m0 = tm * BM + wm * 32 * MB;  // this wave's first row
        if constexpr (E == Epi::kPartial) {
            const int rows = g.mt * BM;
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const int col = tt * kBN + wn * 64 + 32 * j + l32;
                float* out = g.part + ((long)o * g.chunk + col) * rows + m0 + 4 * hh;
                if (col < n)
#pragma unroll
                    for (int i = 0; i < MB; i++)
#pragma unroll
                        for (int q = 0; q < 4; q++)
                            *reinterpret_cast<float4*>(out + 32 * i + 8 * q) =
                                make_float4(acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2],
                                            acc[i][j][4 * q + 3]);
            }
            continue;
        } else {
            const int live = g.vocab - m0;  // rows of the head in this wave's part
            if (live <= 0 && E == Epi::kStats) continue;
            int e[MB];
#pragma unroll
            for (int i = 0; i < MB; i++) e[i] = wave_uniform(g.exponents[m0 / 32 + i]);
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const int col = tt * kBN + wn * 64 + 32 * j + l32;
                const bool scored = col < n;
                const long r = scored ? g.idx[g.j0 + col] : 0;
                const int et = (int)(__builtin_bit_cast(uint32_t, g.scale[g.j0 + col]) >> 23) - 127;
                // The target's row within this wave's part.
                const long target = (scored ? g.targets[r] : -1) - m0;
                const bool here = __any(target >= 0 && target < 32 * MB);
                if constexpr (E == Epi::kStats) {
                    if (live < 32 * MB)
#pragma unroll
                        for (int i = 0; i < MB; i++)
#pragma unroll
                            for (int q = 0; q < 16; q++)
                                if (32 * i + 8 * (q >> 2) + 4 * hh + (q & 3) >= live) acc[i][j][q] = -INFINITY;
                    if (here)
#pragma unroll
                        for (int i = 0; i < MB; i++)
#pragma unroll
                            for (int q = 0; q < 16; q++)
                                if (32 * i + 8 * (q >> 2) + 4 * hh + (q & 3) == target)
                                    g.xt[g.j0 + col] = acc[i][j][q] * pow2_clamped(e[i] + et);
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
                    float sum = 0.0f;
#pragma unroll
                    for (int i = 0; i < MB; i++)
#pragma unroll
                        for (int q = 0; q < 16; q += 4) {
                            float x[4];
#pragma unroll
                            for (int z = 0; z < 4; z++) x[z] = __builtin_amdgcn_exp2f(fmaf(acc[i][j][q + z], c[i], -m));
                            sum += (x[0] + x[1]) + (x[2] + x[3]);
                            __builtin_amdgcn_sched_barrier(0);  // (all at once take more registers than there are)
                        }
                    sum = sum_halves(sum);
                    if (scored && hh == 0) g.stats[(long)(m0 / (32 * MB)) * g.ld + g.j0 + col] = make_float2(m, sum);
                } else {
                    const float lse2 = (scored ? g.lse[r] : 0.0f) * kLog2e;
                    const float dl = g.dlogits && scored ? g.dlogp[r] : 0.0f;
                    const int big = wave_uniform(*g.largest);
#pragma unroll
                    for (int i = 0; i < MB; i++) {
                        const float c = pow2_clamped(e[i] + et) * kLog2e;
                        const float f = kTop * pow2_clamped(e[i] - big);
                        float y[16];
#pragma unroll
                        for (int q = 0; q < 16; q++) {
                            const int row = 32 * i + 8 * (q >> 2) + 4 * hh + (q & 3);
                            float p = __builtin_amdgcn_exp2f(fmaf(acc[i][j][q], c, -lse2));
                            if (here && row == target) p -= 1.0f;
                            y[q] = scored && row < live ? p : 0.0f;
                        }
                        if (g.dlogits && col < g.chunk) {
                            float* out = g.dlogits + (long)col * g.vocab + m0 + 32 * i + 4 * hh;
#pragma unroll
                            for (int q = 0; q < 16; q++)
                                if (32 * i + 8 * (q >> 2) + 4 * hh + (q & 3) < live)
                                    out[8 * (q >> 2) + (q & 3)] = -dl * y[q];
                        }
                        if (!g.grad) continue;
#pragma unroll
                        for (int q = 0; q < 2; q++) {
                            float x[8];
#pragma unroll
                            for (int z = 0; z < 8; z++) x[z] = y[8 * q + z];
                            store_pieces(g.grad + ((long)(tt * 4 + wn * 2 + j) * g.v16 + m0 / 16 + 2 * i + q) * 2 * kFrag,
                                         lane, split8(x, f));
                        }
                    }
                }
            }
        }
    }
}

// lse and logp of scored row j from its parts' maxima and sums, a wave to a row.
__global__ __launch_bounds__(256) void head_finish_kernel(const float2* __restrict__ stats, long ld, int parts,
                                                          const float* __restrict__ xt, const int* __restrict__ idx,
                                                          const int* __restrict__ count, float* __restrict__ logp,
                                                          float* __restrict__ lse) {
    // 16 rows to a workgroup: lane l has row l % 16, so that a part's are read side by side.
    __shared__ float2 red[16][17];
    const int c = threadIdx.x & 15, p0 = threadIdx.x >> 4, j = blockIdx.x * 16 + c, n = *count;
    float m = -INFINITY, s = 0.0f;
    if (j < n)
        for (int p = p0; p < parts; p += 16) {
            const float2 x = stats[p * ld + j];
            const float t = fmaxf(m, x.x);
            // (NaN sums pass through; an empty m is -inf beside a sum of 0.)
            s = (s == 0.0f ? 0.0f : s * exp2f(m - t)) + x.y * exp2f(x.x - t);
            m = t;
        }
    red[p0][c] = make_float2(m, s);
    __syncthreads();
    if (p0 || j >= n) return;
    for (int p = 1; p < 16; p++) {
        const float2 x = red[p][c];
        const float t = fmaxf(m, x.x);
        s = (s == 0.0f ? 0.0f : s * exp2f(m - t)) + (x.y == 0.0f ? 0.0f : x.y * exp2f(x.x - t));
        m = t;
    }
    // Units of kLog2e as rounded: the quotient has the largest logit's own bits.
    const double l = (double)m / (double)kLog2e + log((double)s);
    const int r = idx[j];
    lse[r] = (float)l;
    logp[r] = (float)((double)xt[j] - l);
}

// dhn of the chunk's scored rows: the splits' sums in order, times dlogp.
__global__ __launch_bounds__(256) void head_grad_reduce_kernel(const float* __restrict__ part, int chunk, int rows,
                                                               int mt, int k16, int splits_max,
                                                               const int* __restrict__ idx,
                                                               const int* __restrict__ count, int j0,
                                                               const float* __restrict__ dlogp,
                                                               const int* __restrict__ largest,
                                                               float* __restrict__ dhn, int d) {
    const int n = min(*count - j0, chunk);
    const int col = blockIdx.x;
    if (col >= n) return;
    const int splits = splits_of(mt * ((n + kBN - 1) / kBN), k16, splits_max);
    const long r = idx[j0 + col];
    const float f = -dlogp[r];
    const int big = *largest;
    const float u = pow2_clamped(big - 15);
    for (int i = threadIdx.x; i < d; i += 256) {
        float s = 0.0f;
        for (int p = 0; p < splits; p++) s += part[((long)p * chunk + col) * rows + i];
        dhn[r * d + i] = f * (s * u);
    }
}

// Zeros in the rows of dlogits behind the last tile.
__global__ __launch_bounds__(256) void head_zero_tail_kernel(const int* __restrict__ count, int j0, int chunk,
                                                             float* __restrict__ dlogits, long vocab) {
    const int n = max(min(*count - j0, chunk), 0);
    const long r = blockIdx.x;
    if (r < (n + kBN - 1) / kBN * kBN) return;
    for (long i = threadIdx.x; i < vocab; i += 256) dlogits[r * vocab + i] = 0.0f;
}

// Zeros in the rows that are not scored.
__global__ __launch_bounds__(256) void head_zero_rows_kernel(const int64_t* __restrict__ targets, long vocab,
                                                             float* __restrict__ dhn, int d) {
    const long r = blockIdx.x;
    if (targets[r] >= 0 && targets[r] < vocab) return;
    for (int i = threadIdx.x; i < d; i += 256) dhn[r * d + i] = 0.0f;
}

inline bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }
size_t up(size_t x, size_t to) { return (x + to - 1) / to * to; }

// Blocks of 32 along the columns of the head, to a tile: three (192) to a wave's 96
// or four (256), whichever pads less.
int back_mb(size_t d) { return up(d, 192) < up(d, 256) ? 3 : 4; }
constexpr int kSplitsMax = 32;

}  // namespace

HeadPlan head_plan(size_t t, size_t d, size_t vocab, size_t chunk_bytes) {
    HeadPlan p{};
    p.k16 = (int)((d + 15) / 16);
    p.v_pad = up(vocab, 256);
    p.t_pad = up(t, kBN);
    p.d_pad = up(d, 64 * back_mb(d));
    p.chunk = std::min(std::max<size_t>(chunk_bytes / (p.v_pad * 4) / kBN * kBN, kBN), p.t_pad);
    p.rows_bytes = p.t_pad * p.k16 * 64;
    p.head_bytes = p.v_pad * p.k16 * 64;
    p.back_bytes = p.d_pad * p.v_pad * 4;
    p.stats_bytes = (p.v_pad / 128) * p.t_pad * sizeof(float2);
    p.grad_bytes = p.chunk * p.v_pad * 4;
    p.part_bytes = (size_t)kSplitsMax * p.chunk * p.d_pad * sizeof(float);
    return p;
}

hipError_t launch_head_pack(const HeadPlan& p, const float* hn, const int* idx, const int* count, const float* head,
                            size_t d, size_t vocab, char* rows, float* scale, char* packed, char* back, int* exponents,
                            int* largest, hipStream_t st) {
    hipLaunchKernelGGL(pack_rows_kernel, dim3((unsigned)(p.t_pad / 32)), dim3(256), 0, st, hn, idx, count, rows, scale,
                       (int)d, p.k16, d % 4 == 0 && aligned16(hn));
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    const int vec = d % 4 == 0 && aligned16(head), pairs = (p.k16 + 1) / 2;
    auto pack = [&](auto b, auto nw, auto u) {
        constexpr int kNw = decltype(nw)::value;
        hipLaunchKernelGGL((pack_head_kernel<decltype(b)::value, kNw, decltype(u)::value>),
                           dim3((unsigned)(p.v_pad / 32)), dim3(64 * kNw), 0, st, head, packed, back, exponents,
                           largest, (int)vocab, (int)d, p.k16, (int)(p.v_pad / 16), vec);
    };
    using std::integral_constant;
    auto sized = [&](auto b) {
        // The fewest registers that hold the rows.
        if (pairs <= 8)
            pack(b, integral_constant<int, 8>{}, integral_constant<int, 1>{});
        else if (pairs <= 24)
            pack(b, integral_constant<int, 8>{}, integral_constant<int, 3>{});
        else if (pairs <= 64)
            pack(b, integral_constant<int, 16>{}, integral_constant<int, 4>{});
        else if (pairs <= 128)
            pack(b, integral_constant<int, 16>{}, integral_constant<int, 8>{});
        else
            pack(b, integral_constant<int, 8>{}, integral_constant<int, 0>{});
    };
    if (back)
        sized(std::true_type{});
    else
        sized(std::false_type{});
    return hipGetLastError();
}

hipError_t launch_head_stats(const HeadPlan& p, const char* rows, const float* scale, const char* packed,
                             const int* exponents, const int64_t* targets, const int* idx, const int* count,
                             size_t vocab, void* stats, float* xt, float* logp, float* lse, hipStream_t st) {
    HeadArgs g{};
    g.a = packed, g.b = rows, g.k16 = p.k16, g.mt = (int)(p.v_pad / 256), g.count = count, g.j0 = 0;
    g.chunk = (int)p.t_pad, g.exponents = exponents, g.scale = scale, g.targets = targets, g.idx = idx;
    g.vocab = (int)vocab, g.stats = static_cast<float2*>(stats), g.ld = (long)p.t_pad, g.xt = xt;
    hipLaunchKernelGGL((head_gemm_kernel<4, Epi::kStats>), dim3(kWgs), dim3(256), 0, st, g);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(head_finish_kernel, dim3((unsigned)(p.t_pad / 16)), dim3(256), 0, st, g.stats, g.ld,
                       (int)((vocab + 127) / 128), xt, idx, count, logp, lse);
    return hipGetLastError();
}

hipError_t launch_head_grad(const HeadPlan& p, const char* rows, const float* scale, const char* packed,
                            const char* back, const int* exponents, const int* largest, const int64_t* targets,
                            const int* idx, const int* count, const float* lse, const float* dlogp, size_t j0,
                            size_t d, size_t vocab, char* grad, float* dlogits, float* part, float* dhn,
                            hipStream_t st) {
    HeadArgs g{};
    g.a = packed, g.b = rows + j0 / 32 * p.k16 * 2 * kFrag, g.k16 = p.k16, g.mt = (int)(p.v_pad / 256);
    g.count = count, g.j0 = (int)j0, g.chunk = (int)p.chunk, g.exponents = exponents, g.scale = scale;
    g.targets = targets, g.idx = idx, g.vocab = (int)vocab, g.lse = lse, g.dlogp = dlogp, g.largest = largest;
    g.grad = dhn ? grad : nullptr, g.v16 = (int)(p.v_pad / 16), g.dlogits = dlogits;
    hipLaunchKernelGGL((head_gemm_kernel<4, Epi::kGrad>), dim3(kWgs), dim3(256), 0, st, g);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || !dhn) return e;
    const int mb = back_mb(d);
    HeadArgs h{};
    h.a = back, h.b = grad, h.k16 = g.v16, h.mt = (int)(p.d_pad / (64 * mb)), h.count = count, h.j0 = (int)j0;
    h.chunk = (int)p.chunk, h.part = part, h.splits_max = std::min(kSplitsMax, std::max(8, h.k16 / 4 / 8 * 8));
    if (mb == 3)
        hipLaunchKernelGGL((head_gemm_kernel<3, Epi::kPartial>), dim3(kWgs), dim3(256), 0, st, h);
    else
        hipLaunchKernelGGL((head_gemm_kernel<4, Epi::kPartial>), dim3(kWgs), dim3(256), 0, st, h);
    e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(head_grad_reduce_kernel, dim3((unsigned)p.chunk), dim3(256), 0, st, part, (int)p.chunk,
                       (int)p.d_pad, h.mt, h.k16, h.splits_max, idx, count, (int)j0, dlogp, largest, dhn, (int)d);
    return hipGetLastError();
}

hipError_t launch_head_zero_tail(const HeadPlan& p, const int* count, size_t j0, size_t rows, size_t vocab,
                                 float* dlogits, hipStream_t st) {
    hipLaunchKernelGGL(head_zero_tail_kernel, dim3((unsigned)rows), dim3(256), 0, st, count, (int)j0, (int)p.chunk,
                       dlogits, (long)vocab);
    return hipGetLastError();
}

hipError_t launch_head_zero_rows(const int64_t* targets, size_t t, size_t vocab, float* dhn, size_t d,
                                 hipStream_t st) {
    hipLaunchKernelGGL(head_zero_rows_kernel, dim3((unsigned)t), dim3(256), 0, st, targets, (long)vocab, dhn, (int)d);
    return hipGetLastError();
}

}  // namespace cfattn
