// Rotary positions of up to kRotaryTensors tensors of heads in one launch (cfops_rotary
// of include/cfops.h): pair i of a head's first `rot` values, at position p,
//   (a, b) -> (a c - b s, b c + a s),  c = cos[p][i], s = sin[p][i] (inverse: s negated),
// the pairs (i, i + rot / 2) or, interleaved, (2 i, 2 i + 1); the values behind them are
// copied, or left where they are when a tensor is turned in place.
//
// A thread takes 16 bytes of a head's values that are turned together, or 16 copied ones, at
// any alignment and stride; the table's values of a token are shared by its heads through
// the L1 cache.  Bound by HBM.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "cfattn_common.hpp"
#include "cfops_kernels.hpp"

namespace cfattn {
namespace {

// N consecutive values, of which n are there, at their own alignment.
template <typename T, int N>
struct Vec {
    typedef T type __attribute__((ext_vector_type(N), aligned(sizeof(T))));
};
template <typename T, int N>
__device__ __forceinline__ void load_n(float (&x)[N], const T* p, int n) {
    if (n >= N) {
        const typename Vec<T, N>::type v = *reinterpret_cast<const typename Vec<T, N>::type*>(p);
#pragma unroll
        for (int i = 0; i < N; i++) {
            const T e = v[i];
            x[i] = to_f32<T>(e);
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; i++) x[i] = i < n ? to_f32<T>(p[i]) : 0.0f;
    }
}
template <typename T, int N>
__device__ __forceinline__ void store_n(T* p, const float (&x)[N], int n) {
    if (n >= N) {
        typename Vec<T, N>::type v;
#pragma unroll
        for (int i = 0; i < N; i++) {
            if constexpr (sizeof(T) == 2)
                v[i] = __builtin_bit_cast(T, (__bf16)x[i]);
            else
                v[i] = x[i];
        }
        *reinterpret_cast<typename Vec<T, N>::type*>(p) = v;
    } else {
#pragma unroll
        for (int i = 0; i < N; i++)
            if (i < n) p[i] = from_f32<T>(x[i]);
    }
}

// a / d for a d < 2^32, m = ceil(2^32 / d) (0 for d = 1).
__device__ __forceinline__ unsigned divide(unsigned a, unsigned m) { return m ? __umulhi(a, m) : a; }
unsigned reciprocal(unsigned d) { return d == 1 ? 0 : (unsigned)(((1ull << 32) + d - 1) / d); }

// A piece of a head: the values to turn, or (in lo, then hi) to copy.
constexpr int kPairs = 8;
struct Item {
    float lo[kPairs], hi[kPairs], c[kPairs], s[kPairs];
};

// `tokens` whole tokens to a workgroup, or, where a token has more pieces than 256 U, part
// blockIdx.y of one.  The loads of a thread's U items are in flight together.
template <typename X, typename Y, int U, bool INTER>
__global__ __launch_bounds__(256) void rotary_kernel(const RotaryArgs g) {
    Item it[U];
    Y* to[U];
    int first[U];  // of the head's values; negative: nothing to write
    bool turn[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
        const unsigned at = threadIdx.x + 256 * u;
        unsigned dt = 0, in = blockIdx.y * g.part + at;
        if (g.parts == 1) {
            dt = divide(at, g.per_token_rcp);
            in = at - dt * g.per_token;
        }
        const unsigned token = g.token0 + blockIdx.x * g.tokens_wg + dt;
        const unsigned head = divide(in, g.pieces_rcp);
        const int piece = in - head * g.pieces;
        first[u] = -1;
        if (dt >= g.tokens_wg || token >= g.tokens || in >= g.per_token || (g.parts > 1 && at >= g.part)) continue;
        const unsigned batch = token / g.seq, place = token - batch * g.seq;
        // (Few tensors: the last one whose first head is not beyond this one.)
        const RotaryTensor* a = &g.t[0];
        const char* xp = static_cast<const char*>(a->x);
        char* yp = static_cast<char*>(a->y);
        long x0 = a->xs[0], x1 = a->xs[1], x2 = a->xs[2], y0 = a->ys[0], y1 = a->ys[1], y2 = a->ys[2];
        int head0 = 0, copy = a->copy;
#pragma unroll
        for (int i = 1; i < kRotaryTensors; i++) {
            const RotaryTensor& b = g.t[i];
            if ((int)head < b.head0) continue;
            xp = static_cast<const char*>(b.x), yp = static_cast<char*>(b.y);
            x0 = b.xs[0], x1 = b.xs[1], x2 = b.xs[2], y0 = b.ys[0], y1 = b.ys[1], y2 = b.ys[2];
            head0 = b.head0, copy = b.copy;
        }
        const long h = (int)head - head0;
        const X* x = reinterpret_cast<const X*>(xp) + batch * x0 + place * x1 + h * x2;
        to[u] = reinterpret_cast<Y*>(yp) + batch * y0 + place * y1 + h * y2;
        turn[u] = piece < g.turned;
        if (turn[u]) {
            const int i0 = piece * kPairs, n = g.half - i0;
            first[u] = i0;
            const long p = g.positions ? g.positions[token] : g.pos0 + place;
            if constexpr (INTER) {
                float v[2 * kPairs];
                load_n<X, 2 * kPairs>(v, x + 2 * i0, 2 * n);
#pragma unroll
                for (int i = 0; i < kPairs; i++) it[u].lo[i] = v[2 * i], it[u].hi[i] = v[2 * i + 1];
            } else {
                load_n<X, kPairs>(it[u].lo, x + i0, n);
                load_n<X, kPairs>(it[u].hi, x + g.half + i0, n);
            }
            if (p >= 0 && p < g.max_pos) {
                load_n<float, kPairs>(it[u].c, g.cos + p * g.half + i0, n);
                load_n<float, kPairs>(it[u].s, g.sin + p * g.half + i0, n);
            } else {
#pragma unroll
                for (int i = 0; i < kPairs; i++) it[u].c[i] = it[u].s[i] = __builtin_nanf("");
            }
        } else if (copy) {
            const int i0 = 2 * g.half + (piece - g.turned) * 2 * kPairs, n = g.head_dim - i0;
            first[u] = i0;
            load_n<X, kPairs>(it[u].lo, x + i0, n);
            load_n<X, kPairs>(it[u].hi, x + i0 + kPairs, n - kPairs);
        }
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int i0 = first[u];
        if (i0 < 0) continue;
        Y* y = to[u];
        if (!turn[u]) {
            store_n<Y, kPairs>(y + i0, it[u].lo, g.head_dim - i0);
            store_n<Y, kPairs>(y + i0 + kPairs, it[u].hi, g.head_dim - i0 - kPairs);
            continue;
        }
        float a[kPairs], b[kPairs];
#pragma unroll
        for (int i = 0; i < kPairs; i++) {
            const float c = it[u].c[i], s = g.inverse ? -it[u].s[i] : it[u].s[i];
            a[i] = it[u].lo[i] * c - it[u].hi[i] * s;
            b[i] = it[u].hi[i] * c + it[u].lo[i] * s;
        }
        const int n = g.half - i0;
        if constexpr (INTER) {
            float v[2 * kPairs];
#pragma unroll
            for (int i = 0; i < kPairs; i++) v[2 * i] = a[i], v[2 * i + 1] = b[i];
            store_n<Y, 2 * kPairs>(y + 2 * i0, v, 2 * n);
        } else {
            store_n<Y, kPairs>(y + i0, a, n);
            store_n<Y, kPairs>(y + g.half + i0, b, n);
        }
    }
}

template <typename X, typename Y, int U>
hipError_t go(RotaryArgs g, hipStream_t st) {
    constexpr unsigned kItems = 256 * U;
    g.parts = (g.per_token + kItems - 1) / kItems;
    g.part = (g.per_token + g.parts - 1) / g.parts;
    g.tokens_wg = g.parts > 1 ? 1 : kItems / g.per_token;
    // (A launch has fewer than 2^32 threads.)
    const unsigned most = ((1u << 23) / g.parts) * g.tokens_wg;
    for (g.token0 = 0; g.token0 < g.tokens; g.token0 += most) {
        const dim3 grid((std::min(g.tokens - g.token0, most) + g.tokens_wg - 1) / g.tokens_wg, g.parts);
        if (g.interleaved)
            hipLaunchKernelGGL((rotary_kernel<X, Y, U, true>), grid, dim3(256), 0, st, g);
        else
            hipLaunchKernelGGL((rotary_kernel<X, Y, U, false>), grid, dim3(256), 0, st, g);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace

bool rotary_fits(size_t tokens, size_t heads, size_t head_dim) {
    // (The products of the kernel's divisions, the last one's grid and the tokens' numbers hold
    // 32 bits.)
    const size_t pieces = head_dim / 16 + 2, per_token = heads * pieces;
    return head_dim <= 65536 && heads <= 65536 && per_token * std::max<size_t>(pieces, 512) < (size_t)1 << 32 &&
           tokens < (size_t)1 << 31;
}

hipError_t launch_rotary(RotaryArgs g, bool x_bf16, bool y_bf16, hipStream_t st) {
    bool copy = false;
    for (int i = 0; i < g.count; i++) copy |= g.t[i].copy;
    g.turned = (g.half + kPairs - 1) / kPairs;
    g.pieces = g.turned + (copy ? (g.head_dim - 2 * g.half + 2 * kPairs - 1) / (2 * kPairs) : 0);
    g.per_token = (unsigned)(g.heads * g.pieces);
    if (g.tokens == 0 || g.per_token == 0) return hipSuccess;
    g.per_token_rcp = reciprocal(g.per_token), g.pieces_rcp = reciprocal(g.pieces);
    for (int i = g.count; i < kRotaryTensors; i++) g.t[i].head0 = g.heads;
    auto typed = [&](auto u) {
        constexpr int U = decltype(u)::value;
        return x_bf16 ? y_bf16 ? go<bf16_bits, bf16_bits, U>(g, st) : go<bf16_bits, float, U>(g, st)
                      : y_bf16 ? go<float, bf16_bits, U>(g, st) : go<float, float, U>(g, st);
    };
    // Two items a thread where that leaves every CU four workgroups.
    if ((size_t)g.tokens * g.per_token >= 1024 * 512) return typed(std::integral_constant<int, 2>{});
    return typed(std::integral_constant<int, 1>{});
}

}  // namespace cfattn
