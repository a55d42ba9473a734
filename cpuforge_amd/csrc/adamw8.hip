// AdamW over many tensors whose moments are held in 8 bits or in 32
// (cfops_adamw8_update_multi of include/cfops.h).
//
// An 8-bit state holds blocks of 256 consecutive values of a tensor.  With E
// the block's power of two, its largest magnitude in (2^E, 2^(E+1)]:
//   m: sign, 4 exponent, 3 mantissa bits; the binade [2^E, 2^(E+1)) is exponent
//      field 14, fields 1 and up are normal, field 0 subnormal; 0x7f is NaN;
//   v: 5 exponent, 3 mantissa bits; [2^E, 2^(E+1)) is field 30; 0xff is infinity.
// E is held as a byte, E + 127.  A power of two costs a float code none of its
// bits (an absmax scale would round the block's values once more), and a state
// that is read, given as f32 and packed again is the same state.
//
// Rounding: up or down by the value's fraction of a step against 17 bits that
// are a function of its index and the step count.  beta2 = 0.999 moves v by a
// thousandth of itself a step and beta1 = 0.95 m by a twentieth, less than half a
// step of three mantissa bits (1/16 to 1/8): rounded to nearest such a moment would
// never move; so the mean of its roundings is the value.  A positive v is
// never held as zero: the update divides by its root.
// m' = b1 m + (1-b1) g and v' are formed in f64 (products of a held value, at most
// four significant bits, and of f32s: one rounding in 53 bits), since a rounding
// to 8 bits goes by what lies below f32; the update itself is f32 on (float)m'
// and (float)v', not on the held values.
//
// What bounds it: HBM, 16 bytes a value a step (p read and written, g read, two
// bytes read and written) against 28 with f32 states.  134.5 M values: an update
// 380 to 430 us (5.0 to 5.7 TB/s; a copy of 4 GiB runs at 4.8), a state read as f32
// 256 us.  448 tensors of 4.9 M values: 16.2 us, 11 of them its bytes.
#include <limits.h>

#include <algorithm>

#include "adamw_math.hpp"
#include "cfattn_common.hpp"
#include "cfops_kernels.hpp"

namespace cfattn {
namespace {

constexpr int kBlock = 4096;  // values of a workgroup: 16 blocks, one to 16 lanes

template <int N>
struct Args : Adamw8Step {
    int first[N];  // each tensor's first workgroup; past the last one INT_MAX
    Adamw8Tensor t[N];
};

inline bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

// The layout of a state of n values: codes of m and of v, a byte for every value
// of whole blocks, then a byte for every block's exponent of m and of v.
struct State8 {
    uint8_t *m, *v, *em, *ev;
};
__device__ __forceinline__ State8 state8(uint8_t* s, long n) {
    const long nb = (n + 255) / 256;
    return {s, s + nb * 256, s + nb * 512, s + nb * 513};
}

__device__ __forceinline__ double pow2(int e) { return __builtin_bit_cast(double, (uint64_t)(uint32_t)(e + 1023) << 52); }
__device__ __forceinline__ uint32_t hi_word(double a) { return (uint32_t)(__builtin_bit_cast(uint64_t, a) >> 32); }

// A code's magnitude in units of 2^(E + 113) (m) or 2^(E + 97) (v): its fields are
// an f32's, subnormals with them.
__device__ __forceinline__ float code_unit(uint32_t c) { return __builtin_bit_cast(float, c << 20); }
constexpr int kUnitM = -14, kUnitV = -30;  // of 2^byte

__device__ __forceinline__ double decode_m(uint32_t c, double unit) {
    const float y = code_unit(c & 0x7f);
    const double x = (double)((c & 0x80) ? -y : y) * unit;
    return (c & 0x7f) == 0x7f ? __builtin_nan("") : x;
}
__device__ __forceinline__ double decode_v(uint32_t c, double unit) {
    return c == 0xff ? __builtin_inf() : (double)code_unit(c) * unit;
}

// The code of the magnitude whose high word is `hi`; `least` is the biased exponent
// of the first normal binade.  r: 17 bits, the rounding threshold.  In the high word
// of a double lie its exponent, the three mantissa bits of a code and the 17 below
// them; what lies below those can carry nothing into the code.  Below the first
// normal binade the steps are that binade's: the sum with its power of two has them.
__device__ __forceinline__ uint32_t encode(uint32_t hi, uint32_t least, uint32_t r) {
    const bool normal = hi >> 20 >= least;
    const double a = __builtin_bit_cast(double, (uint64_t)hi << 32);
    const double low = __builtin_bit_cast(double, (uint64_t)(least << 20) << 32);
    const uint32_t u = ((normal ? hi : hi_word(a + low)) + r) >> 17;
    return u - (least << 3) + (normal ? 8 : 0);
}

// What f32 does not hold.
__device__ __forceinline__ bool odd(uint32_t hi) { return (hi & 0x7fffffff) >= (1023u + 128) << 20; }

// Byte of a block's exponent, from the largest high word of its magnitudes (up to
// 2^-20 above a power of two counts as that power).
__device__ __forceinline__ int exponent_byte(uint32_t hi) {
    return max(0, (int)(hi >> 20) - 1023 + 127 - ((hi & 0xfffff) == 0));
}

// Largest of 16 lanes.
__device__ __forceinline__ uint32_t max16(uint32_t x) {
#pragma unroll
    for (int o = 8; o >= 1; o >>= 1) x = max(x, (uint32_t)__shfl_xor((int)x, o));
    return x;
}

// Two rounds of a 32-bit multiplicative mix.  (Its odd multipliers have no meaning of
// their own; that the bits are uniform, and those of neighbours, of steps and of m and v
// uncorrelated, is tested.)
__device__ __forceinline__ uint32_t mix(uint32_t x) {
    x = (x ^ (x >> 16)) * 0xA511E9B3u;
    x = (x ^ (x >> 15)) * 0x63D83595u;
    return x ^ (x >> 16);
}

// The tensor that workgroup b falls in.  Every lane reads its share of the first
// workgroups: two reads one after the other where a search of halves takes ten, each
// waiting for the last (448 tensors of 4.9 M values: an update 16.2 us, by halves
// 17.9; a state read 7.4 and 9.4).
template <int N>
__device__ __forceinline__ const Adamw8Tensor& find(const Args<N>& a, int b) {
    const int lane = threadIdx.x & 63;
    int n = 0;
#pragma unroll
    for (int i = 0; i < N; i += 64) n += __popcll(__ballot(i + lane < N && a.first[min(i + lane, N - 1)] <= b));
    return a.t[wave_uniform(n - 1)];
}

// Four consecutive values p[i..i+3] of n, those at or past n as zeros.
__device__ __forceinline__ float4 load4(const float* p, long i, long n, bool vec) {
    if (vec && i + 3 < n) return *reinterpret_cast<const float4*>(p + i);
    float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (i < n) x.x = p[i];
    if (i + 1 < n) x.y = p[i + 1];
    if (i + 2 < n) x.z = p[i + 2];
    if (i + 3 < n) x.w = p[i + 3];
    return x;
}
__device__ __forceinline__ void store4(float* p, long i, long n, bool vec, const float4& x) {
    if (vec && i + 3 < n) {
        *reinterpret_cast<float4*>(p + i) = x;
        return;
    }
    if (i < n) p[i] = x.x;
    if (i + 1 < n) p[i + 1] = x.y;
    if (i + 2 < n) p[i + 2] = x.z;
    if (i + 3 < n) p[i + 3] = x.w;
}

// Rounding thresholds of a value's m and v, 17 bits each.
struct Thresholds {
    uint32_t m, v;
};
constexpr Thresholds kNearest{1u << 16, 1u << 16};  // (the middle goes up)
// From 32 bits: the two share two of them.
__device__ __forceinline__ Thresholds thresholds(uint32_t r) { return {r & 0x1ffff, r >> 15}; }

// Codes of a block's 16 values of this lane, four to a word, from their high words
// (m with its sign); threshold(e) are the Thresholds of value e.
template <typename F>
__device__ __forceinline__ void encode_block(const uint32_t (&m)[16], const uint32_t (&v)[16], F threshold,
                                             uint32_t (&cm)[4], uint32_t (&cv)[4], int& em, int& ev) {
    uint32_t tm = 0, tv = 0;
#pragma unroll
    for (int e = 0; e < 16; e++) {
        const uint32_t hm = m[e] & 0x7fffffff;
        tm = max(tm, odd(hm) ? 0u : hm);
        tv = max(tv, odd(v[e]) ? 0u : v[e]);
    }
    em = exponent_byte(max16(tm));
    ev = exponent_byte(max16(tv));
    // Biased exponents of the first normal binades: E - 13 and E - 29.
    const uint32_t lm = (uint32_t)(em - 127 - 13 + 1023), lv = (uint32_t)(ev - 127 - 29 + 1023);
#pragma unroll
    for (int j = 0; j < 4; j++) {
        cm[j] = cv[j] = 0;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const int e = 4 * j + k;
            const Thresholds r = threshold(e);
            const uint32_t hm = m[e] & 0x7fffffff;
            uint32_t c = odd(hm) ? 0x7fu : encode(hm, lm, r.m);
            c |= (m[e] >> 31) << 7;
            cm[j] |= c << (8 * k);
            c = odd(v[e]) ? 0xffu : encode(v[e], lv, r.v);
            cv[j] |= max(c, v[e] ? 1u : 0u) << (8 * k);
        }
    }
}

template <int N>
__global__ __launch_bounds__(256) void adamw8_kernel(const Args<N> a) {
    const Adamw8Tensor& t = find(a, blockIdx.x);
    const long e0 = ((long)blockIdx.x - t.block0) * kBlock;
    const float ob1 = 1.0f - a.beta1, ob2 = 1.0f - a.beta2;
    if (!t.state8) {  // 32-bit states
        const long e1 = min(e0 + kBlock, t.n);
        for (long i = e0 + 4 * threadIdx.x; i < e1; i += 1024) {
            float4 p = load4(t.p, i, t.n, t.vec), m = load4(t.m, i, t.n, t.vec), v = load4(t.v, i, t.n, t.vec);
            const float4 g = load4(t.g, i, t.n, t.vec);
            adamw_one(p.x, g.x, m.x, v.x, a.lr, a.beta1, a.beta2, ob1, ob2, a.eps, t.weight_decay, a.bc1, a.bc2);
            adamw_one(p.y, g.y, m.y, v.y, a.lr, a.beta1, a.beta2, ob1, ob2, a.eps, t.weight_decay, a.bc1, a.bc2);
            adamw_one(p.z, g.z, m.z, v.z, a.lr, a.beta1, a.beta2, ob1, ob2, a.eps, t.weight_decay, a.bc1, a.bc2);
            adamw_one(p.w, g.w, m.w, v.w, a.lr, a.beta1, a.beta2, ob1, ob2, a.eps, t.weight_decay, a.bc1, a.bc2);
            store4(t.p, i, t.n, t.vec, p);
            store4(t.m, i, t.n, t.vec, m);
            store4(t.v, i, t.n, t.vec, v);
        }
        return;
    }
    // 16 lanes to a block; of each run of 64 values a lane has four.
    const long b = e0 / 256 + threadIdx.x / 16;
    if (b * 256 >= t.n) return;  // (whole groups of 16 lanes)
    const State8 s = state8(t.state8, t.n);
    const long i0 = b * 256 + 4 * (threadIdx.x % 16);
    uint32_t cm[4], cv[4];
    float p[16], g[16];
#pragma unroll
    for (int j = 0; j < 4; j++) {
        cm[j] = *reinterpret_cast<const uint32_t*>(s.m + i0 + 64 * j);
        cv[j] = *reinterpret_cast<const uint32_t*>(s.v + i0 + 64 * j);
        const float4 x = load4(t.p, i0 + 64 * j, t.n, t.vec), y = load4(t.g, i0 + 64 * j, t.n, t.vec);
        p[4 * j] = x.x, p[4 * j + 1] = x.y, p[4 * j + 2] = x.z, p[4 * j + 3] = x.w;
        g[4 * j] = y.x, g[4 * j + 1] = y.y, g[4 * j + 2] = y.z, g[4 * j + 3] = y.w;
    }
    const double um = pow2(s.em[b] + kUnitM), uv = pow2(s.ev[b] + kUnitV);
    const double b1 = a.beta1, b2 = a.beta2, d1 = ob1, d2 = ob2;
    uint32_t m[16], v[16];
#pragma unroll
    for (int j = 0; j < 4; j++) {
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const int e = 4 * j + k;
            const double gd = g[e];
            const double md = fma(d1, gd, b1 * decode_m(cm[j] >> (8 * k) & 0xff, um));
            const double vd = fma(d2 * gd, gd, b2 * decode_v(cv[j] >> (8 * k) & 0xff, uv));
            const float mf = (float)md, vf = (float)vd;
            // (The instructions' square root and reciprocal, to a step of f32 each: 2^-22 of the
            // update.  2-norm of the error of p against 64 bits, so and correctly rounded, both in
            // f32: 2.54e-8 and 2.54e-8 where the update is a thousandth of p, 2.72e-8 and 2.63e-8
            // where it is a twentieth, 7.3e-8 and 6.7e-8 where p starts from zeros.)
            const float den = fmaf(__builtin_amdgcn_sqrtf(vf), a.c2, a.eps);
            const float upd = fmaf(mf * a.c1, __builtin_amdgcn_rcpf(den), t.weight_decay * p[e]);
            p[e] = fmaf(-a.lr, upd, p[e]);
            m[e] = hi_word(md);
            v[e] = hi_word(vd) & 0x7fffffff;
        }
        store4(t.p, i0 + 64 * j, t.n, t.vec, make_float4(p[4 * j], p[4 * j + 1], p[4 * j + 2], p[4 * j + 3]));
    }
    int em, ev;
    encode_block(
        m, v, [&](int e) { return thresholds(mix((uint32_t)(i0 + 64 * (e / 4) + e % 4) + a.key)); }, cm, cv, em, ev);
#pragma unroll
    for (int j = 0; j < 4; j++) {
        *reinterpret_cast<uint32_t*>(s.m + i0 + 64 * j) = cm[j];
        *reinterpret_cast<uint32_t*>(s.v + i0 + 64 * j) = cv[j];
    }
    if (threadIdx.x % 16 == 0) {
        s.em[b] = (uint8_t)em;
        s.ev[b] = (uint8_t)ev;
    }
}

// f32 moments into an 8-bit state, each to the nearest of its steps, and back.
template <int N, bool PACK>
__global__ __launch_bounds__(256) void adamw8_convert_kernel(const Args<N> a) {
    const Adamw8Tensor& t = find(a, blockIdx.x);
    const long b = ((long)blockIdx.x - t.block0) * (kBlock / 256) + threadIdx.x / 16;
    if (b * 256 >= t.n) return;
    const State8 s = state8(t.state8, t.n);
    const long i0 = b * 256 + 4 * (threadIdx.x % 16);
    uint32_t cm[4], cv[4];
    if constexpr (PACK) {
        uint32_t m[16], v[16];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const float4 x = load4(t.m, i0 + 64 * j, t.n, t.vec), y = load4(t.v, i0 + 64 * j, t.n, t.vec);
            const float xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
            for (int k = 0; k < 4; k++) {
                m[4 * j + k] = hi_word((double)xs[k]);
                v[4 * j + k] = hi_word((double)ys[k]) & 0x7fffffff;
            }
        }
        int em, ev;
        encode_block(
            m, v, [](int) { return kNearest; }, cm, cv, em, ev);
#pragma unroll
        for (int j = 0; j < 4; j++) {
            *reinterpret_cast<uint32_t*>(s.m + i0 + 64 * j) = cm[j];
            *reinterpret_cast<uint32_t*>(s.v + i0 + 64 * j) = cv[j];
        }
        if (threadIdx.x % 16 == 0) {
            s.em[b] = (uint8_t)em;
            s.ev[b] = (uint8_t)ev;
        }
    } else {
        const double um = pow2(s.em[b] + kUnitM), uv = pow2(s.ev[b] + kUnitV);
#pragma unroll
        for (int j = 0; j < 4; j++) {
            cm[j] = *reinterpret_cast<const uint32_t*>(s.m + i0 + 64 * j);
            cv[j] = *reinterpret_cast<const uint32_t*>(s.v + i0 + 64 * j);
            float m[4], v[4];
#pragma unroll
            for (int k = 0; k < 4; k++) {
                m[k] = (float)decode_m(cm[j] >> (8 * k) & 0xff, um);
                v[k] = (float)decode_v(cv[j] >> (8 * k) & 0xff, uv);
            }
            store4(t.m, i0 + 64 * j, t.n, t.vec, make_float4(m[0], m[1], m[2], m[3]));
            store4(t.v, i0 + 64 * j, t.n, t.vec, make_float4(v[0], v[1], v[2], v[3]));
        }
    }
}

}  // namespace

size_t adamw8_state_bytes(size_t n) { return (n + 255) / 256 * 514; }

uint32_t adamw8_key(uint64_t t) {
    auto mix32 = [](uint32_t x) {
        x = (x ^ (x >> 16)) * 0xA511E9B3u;
        x = (x ^ (x >> 15)) * 0x63D83595u;
        return x ^ (x >> 16);
    };
    return mix32((uint32_t)t * 0x9E3779B1u + 0x7F4A7C15u);
}

template <int N>
static hipError_t launch(const Adamw8Tensor* t, const Adamw8Step& step, Adamw8Op op, unsigned blocks, hipStream_t st) {
    Args<N> a;
    static_cast<Adamw8Step&>(a) = step;
    std::copy(t, t + step.count, a.t);
    for (int i = 0; i < N; i++) a.first[i] = i < step.count ? (int)t[i].block0 : INT_MAX;
    const auto kernel = op == Adamw8Op::kUpdate ? adamw8_kernel<N>
                        : op == Adamw8Op::kPack ? adamw8_convert_kernel<N, true>
                                                : adamw8_convert_kernel<N, false>;
    hipLaunchKernelGGL(kernel, dim3(blocks), dim3(256), 0, st, a);
    return hipGetLastError();
}

hipError_t launch_adamw8(Adamw8Tensor* tensors, const Adamw8Step& step, Adamw8Op op, hipStream_t st) {
    long blocks = 0;
    for (int i = 0; i < step.count; i++) {
        Adamw8Tensor& t = tensors[i];
        const bool pg = op != Adamw8Op::kUpdate || (aligned16(t.p) && aligned16(t.g));
        const bool mv = (op == Adamw8Op::kUpdate && t.state8) || (aligned16(t.m) && aligned16(t.v));
        t.vec = pg && mv;
        t.block0 = blocks;
        blocks += (t.n + kBlock - 1) / kBlock;
    }
    if (blocks == 0) return hipSuccess;
    if (blocks > 0xffffffL) return hipErrorInvalidConfiguration;  // fewer than 2^32 threads
    return step.count <= kAdamw8Few ? launch<kAdamw8Few>(tensors, step, op, (unsigned)blocks, st)
                                    : launch<kAdamw8Batch>(tensors, step, op, (unsigned)blocks, st);
}

}  // namespace cfattn
