// Rotary positions of up to kRotaryTensors tensors of heads in one launch (cfops_rotary
// of include/cfops.h): pair i of a head's first `rot` values, at position p,
//   (a, b) -> (a c - b s, b c + a s),  c = cos[p][i], s = sin[p][i] (inverse: s negated),
// the pairs (i, i + rot / 2) or, interleaved, (2 i, 2 i + 1); the values behind them are
// copied, or left where they are when a tensor is turned in place.
//
// Loads and stores are as wide at any alignment and stride; the table's values of a token are
// shared by its heads through the L1 cache.  Bound by HBM.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "cfattn_common.hpp"
#include "cfops_kernels.hpp"

namespace cfattn {
namespace {

// N consecutive values at their own alignment.
template <typename T, int N>
struct Vec {
    typedef T type __attribute__((ext_vector_type(N), aligned(sizeof(T))));
};
template <typename T, int N>
__device__ __forceinline__ typename Vec<T, N>::type load_n(const T* p) {
    return *reinterpret_cast<const typename Vec<T, N>::type*>(p);
}
template <typename T, int N>
__device__ __forceinline__ float value(const typename Vec<T, N>::type& v, int i) {
    const T e = v[i];
    return to_f32<T>(e);
}
template <typename T>
__device__ __forceinline__ T rounded(float x) {
    if constexpr (sizeof(T) == 2)
        return __builtin_bit_cast(T, (__bf16)x);
    else
        return x;
}

// a / d for a d < 2^32, m = ceil(2^32 / d) (0 for d = 1).
__device__ __forceinline__ unsigned divide(unsigned a, unsigned m) { return m ? __umulhi(a, m) : a; }
unsigned reciprocal(unsigned d) { return d == 1 ? 0 : (unsigned)(((1ull << 32) + d - 1) / d); }

// A thread takes a piece of a head: the values of kPairs pairs, or 2 kPairs to copy; a workgroup
// `tokens_wg` whole tokens of one tensor, or, where a token has more than 256 pieces, one of
// `parts` of it.  (All of a workgroup in one tensor: its pointers and strides come
// through the scalar cache.  With the tensors' heads side by side each lane had to load them,
// 16384 tokens of 32 + 8 heads of 128 bf16 values 89 us where this takes 64, 5.3 TB/s.)
constexpr int kPairs = 8;
template <typename X, typename Y, bool INTER>
__global__ __launch_bounds__(256) void rotary_kernel(const RotaryArgs g) {
    int tensor = 0;
#pragma unroll
    for (int i = 1; i < kRotaryTensors; i++) tensor = blockIdx.x >= g.t[i].block0 ? i : tensor;
    const RotaryTensor& t = g.t[tensor];
    unsigned block = blockIdx.x - t.block0, dt = 0, in = threadIdx.x;
    if (t.parts == 1) {
        dt = divide(threadIdx.x, t.per_token_rcp);
        in -= dt * t.per_token;
    } else {
        if (threadIdx.x >= t.part) return;
        const unsigned token = block / t.parts;
        in += (block - token * t.parts) * t.part;
        block = token;
    }
    const unsigned token = g.token0 + block * t.tokens_wg + dt;
    if (dt >= t.tokens_wg || token >= g.tokens || in >= t.per_token) return;
    const unsigned head = divide(in, t.pieces_rcp);
    const int piece = in - head * t.pieces;
    const unsigned batch = token / g.seq, place = token - batch * g.seq;
    const X* x = static_cast<const X*>(t.x) + batch * t.xs[0] + place * t.xs[1] + head * t.xs[2];
    Y* y = static_cast<Y*>(t.y) + batch * t.ys[0] + place * t.ys[1] + head * t.ys[2];
    const bool turn = piece < g.turned;
    // The piece's first pair, and its two runs of values, from a and from b on.
    const int i0 = piece * kPairs, n = g.half - i0;
    const int behind = 2 * g.half + 2 * (piece - g.turned) * kPairs;
    const int a = turn ? (INTER ? 2 * i0 : i0) : behind;
    const int b = !turn || INTER ? a + kPairs : g.half + i0;
    if (turn ? n >= kPairs : behind + 2 * kPairs <= g.head_dim) {
        // (The values are on their way before the position is waited for.)
        const auto xa = load_n<X, kPairs>(x + a), xb = load_n<X, kPairs>(x + b);
        const long p = !turn ? -1 : g.positions ? g.positions[token] : g.pos0 + place;
        typename Vec<float, kPairs>::type c, s = {};
#pragma unroll
        for (int i = 0; i < kPairs; i++) c[i] = __builtin_nanf("");
        if (p >= 0 && p < g.max_pos) {
            c = load_n<float, kPairs>(g.cos + p * g.half + i0);
            s = load_n<float, kPairs>(g.sin + p * g.half + i0);
        }
        float u[2 * kPairs];
#pragma unroll
        for (int i = 0; i < kPairs; i++) u[i] = value<X, kPairs>(xa, i), u[kPairs + i] = value<X, kPairs>(xb, i);
        if (turn) {
#pragma unroll
            for (int i = 0; i < kPairs; i++) {
                float &lo = u[INTER ? 2 * i : i], &hi = u[INTER ? 2 * i + 1 : kPairs + i];
                const float cn = c[i], sn = g.inverse ? -s[i] : s[i], t = lo;
                lo = lo * cn - hi * sn;
                hi = hi * cn + t * sn;
            }
        }
        typename Vec<Y, kPairs>::type ya, yb;
#pragma unroll
        for (int i = 0; i < kPairs; i++) ya[i] = rounded<Y>(u[i]), yb[i] = rounded<Y>(u[kPairs + i]);
        *reinterpret_cast<typename Vec<Y, kPairs>::type*>(y + a) = ya;
        *reinterpret_cast<typename Vec<Y, kPairs>::type*>(y + b) = yb;
    } else if (turn) {
        const long p = g.positions ? g.positions[token] : g.pos0 + place;
        const bool held = p >= 0 && p < g.max_pos;
        const float *cos = g.cos + p * g.half + i0, *sin = g.sin + p * g.half + i0;
        for (int i = 0; i < n; i++) {
            const int l = INTER ? a + 2 * i : a + i, r = INTER ? l + 1 : b + i;
            const float lo = to_f32<X>(x[l]), hi = to_f32<X>(x[r]);
            const float cn = held ? cos[i] : __builtin_nanf(""), si = held ? sin[i] : 0.0f, sn = g.inverse ? -si : si;
            y[l] = rounded<Y>(lo * cn - hi * sn);
            y[r] = rounded<Y>(hi * cn + lo * sn);
        }
    } else {
        for (int i = behind; i < g.head_dim; i++) y[i] = rounded<Y>(to_f32<X>(x[i]));
    }
}

template <typename X, typename Y>
hipError_t go(RotaryArgs g, hipStream_t st) {
    g.turned = (g.half + kPairs - 1) / kPairs;
    unsigned parts = 0;
    for (int i = 0; i < g.count; i++) {
        RotaryTensor& t = g.t[i];
        t.pieces = g.turned + (t.copy ? (g.head_dim - 2 * g.half + 2 * kPairs - 1) / (2 * kPairs) : 0);
        t.per_token = (unsigned)(t.heads * t.pieces);
        t.per_token_rcp = reciprocal(t.per_token), t.pieces_rcp = reciprocal(t.pieces);
        t.parts = (t.per_token + 255) / 256;
        t.part = (t.per_token + t.parts - 1) / t.parts;
        t.tokens_wg = t.parts > 1 ? 1 : 256 / t.per_token;
        parts += t.parts;
    }
    // (A launch has fewer than 2^32 threads.)
    const unsigned all = g.tokens, most = (1u << 23) / parts;
    for (g.token0 = 0; g.token0 < all; g.token0 += most) {
        const unsigned n = std::min(all - g.token0, most);
        // (The last workgroup of a launch may have room for tokens of the next one, which turns them.)
        g.tokens = g.token0 + n;
        unsigned blocks = 0;
        for (int i = 0; i < kRotaryTensors; i++) {
            g.t[i].block0 = blocks;
            if (i < g.count) blocks += (n + g.t[i].tokens_wg - 1) / g.t[i].tokens_wg * g.t[i].parts;
        }
        // (Those that are not there begin behind the last block.)
        hipLaunchKernelGGL((g.interleaved ? rotary_kernel<X, Y, true> : rotary_kernel<X, Y, false>), dim3(blocks),
                           dim3(256), 0, st, g);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace

bool rotary_fits(size_t tokens, size_t heads, size_t head_dim) {  // heads of a tensor
    // (The products of the kernel's divisions, a launch's grid and the tokens' numbers hold 32
    // bits.)
    const size_t pieces = head_dim / (2 * kPairs) + 2, per_token = heads * pieces;
    return head_dim <= 65536 && heads <= 65536 && per_token * std::max<size_t>(pieces, 256) < (size_t)1 << 32 &&
           tokens < (size_t)1 << 31;
}

hipError_t launch_rotary(const RotaryArgs& g, bool x_bf16, bool y_bf16, hipStream_t st) {
    if (g.tokens == 0 || g.count == 0) return hipSuccess;
    return x_bf16 ? y_bf16 ? go<bf16_bits, bf16_bits>(g, st) : go<bf16_bits, float>(g, st)
                  : y_bf16 ? go<float, bf16_bits>(g, st) : go<float, float>(g, st);
}

}  // namespace cfattn
