// The loss of distillation from a teacher's top logits (cfops_lm_head_distill of
// include/cfops.h) by rows, given the student's logits x (of the hidden states over the
// temperature):
//   q = softmax(x),  p_k = exp(z_k / T - L) for the teacher's entries k,
//   loss = sum_k p_k (log p_k - log q_k) + p_rest (log p_rest - log q_rest),
// the rest being every token that is no entry (p_rest = 1 - sum p_k; without the teacher's
// log-sum-exp L is the entries' own, and there is none), and
//   d loss / d x_v = q_v - p_v for an entry,  a q_v else,  a = 1 - p_rest / q_rest.
// q_rest is a sum over the others, not 1 less the entries': a confident student's is far
// below what is lost there.  What is of a row alone is f64.
#include <hip/hip_runtime.h>
#include <limits.h>

#include "cfattn_common.hpp"
#include "cfops_kernels.hpp"

namespace cfattn {
namespace {

constexpr long kIgnoreIndex = -100;  // crates/core/src/ops/loss.rs:4

__device__ __forceinline__ double sum_wave(double x) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) x += __shfl_xor(x, o);
    return x;
}
__device__ __forceinline__ float max_wave(float x) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) x = fmaxf(x, __shfl_xor(x, o));
    return x;
}
__device__ __forceinline__ bool finite(float x) { return fabsf(x) < INFINITY; }

// A row's entries by rising token, a wave to a row: ids, z and e [t][k] (count of them), their
// exponentials below the largest's; the row's L, p_rest (negative: no rest) and p / e; target is a token of the row, kIgnoreIndex without entries, -1 where
// the row is bad: a token out of the vocabulary or named twice, or a value of the teacher's that
// is not finite.  (An entry whose id is kIgnoreIndex or whose logit is -inf is not there.)
// Places are counts of smaller tokens: 4096 x 64 entries TODO us.
__global__ __launch_bounds__(256) void distill_entries_kernel(const DistillEntries g) {
    extern __shared__ int tokens[];  // [4][k]
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const long r = (long)blockIdx.x * 4 + wave;
    if (r >= g.t) return;  // (no barrier follows: each wave has its own part of LDS)
    int* mine = tokens + wave * g.k;
    const int64_t* ids = g.raw_ids + r * g.k;
    const float* z = g.teacher + r * g.k;
    bool bad = false;
    int n = 0;
    float top = -INFINITY;
    for (int k0 = 0; k0 < g.k; k0 += 64) {
        const int k = k0 + lane;
        int v = INT_MAX;
        if (k < g.k) {
            const long id = ids[k];
            const float x = z[k];
            const bool there = id != kIgnoreIndex && !(x == -INFINITY);
            if (there) {
                bad |= id < 0 || id >= g.vocab || !finite(x);
                v = id < 0 || id >= g.vocab ? INT_MAX : (int)id;
                top = fmaxf(top, x);
            }
            mine[k] = v;
        }
        n += __popcll(__ballot(v != INT_MAX));
    }
    __builtin_amdgcn_wave_barrier();
    top = max_wave(top);
    double sum = 0.0;
    int least = INT_MAX;
    for (int k0 = 0; k0 < g.k; k0 += 64) {
        const int k = k0 + lane;
        const int v = k < g.k ? mine[k] : INT_MAX;
        int place = 0;
        for (int i = 0; i < g.k; i++) {
            const int o = mine[i];
            place += o < v;
            bad |= o == v && i != k && v != INT_MAX;
        }
        if (v == INT_MAX) continue;
        // (Twice the same token: two entries in one place, of which nothing is read.)
        g.ids[r * g.k + place] = v;
        const double e = exp(((double)z[k] - (double)top) * g.inv_t);
        g.z[r * g.k + place] = z[k];
        g.e[r * g.k + place] = (float)e;
        least = min(least, v);
        sum += e;
    }
    sum = sum_wave(sum);
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) least = min(least, __shfl_xor(least, o));
    const double own = (double)top * g.inv_t + log(sum);
    double whole = own, p_rest = -1.0;
    if (g.teacher_lse && n > 0 && n < g.vocab) {
        const float l = g.teacher_lse[r];
        bad |= !finite(l);
        whole = fmax(own, (double)l);
        p_rest = -expm1(own - whole);
    }
    const bool any_bad = __any(bad);
    if (lane) return;
    g.count[r] = any_bad ? 0 : n;
    g.row[r] = {whole, p_rest, exp(own - whole) / sum};
    g.target[r] = any_bad ? -1 : n == 0 ? kIgnoreIndex : least;
}

// The first of n rising tokens that is not below v.
__device__ __forceinline__ int lower_bound(const int* tokens, int n, int v) {
    int lo = 0, hi = n;
    while (lo < hi) {
        const int mid = (lo + hi) / 2;
        if (tokens[mid] < v)
            lo = mid + 1;
        else
            hi = mid;
    }
    return lo;
}

// What the rest makes of a row's loss, given the logarithm of its probability.
struct Rest {
    double loss = 0.0, ratio = 0.0;  // ratio: p_rest / q_rest
    __device__ __forceinline__ Rest(double p_rest, double log_q_rest) {
        if (!(p_rest > 0.0)) return;
        const double log_p = log(p_rest);
        loss = p_rest * (log_p - log_q_rest);
        ratio = exp(log_p - log_q_rest);
    }
};
// An entry's part of the loss, and in dl the gradient of its logit.
__device__ __forceinline__ double entry_loss(const TeacherRow& row, float z, float e, double inv_t, double q,
                                             double log_q, double& dl) {
    const double p = (double)e * row.scale;
    dl = q - p;
    return p * ((double)z * inv_t - row.l - log_q);
}

// 2^x; the f32 instruction where f32 holds it.
__device__ __forceinline__ double pow2(double x) { return x > -120.0 ? (double)__builtin_amdgcn_exp2f((float)x) : exp2(x); }

// Rows whose product kept exp2(y - m) of 128 logits each (y in units of log2, m the largest):
// a wave to a row, 8 rows to a workgroup.  An entry whose exponential is too small, and
// a rest of 128 that is, are formed again from hidden state and head.  Where the entries hold
// all but little of such 128, the rest of them is summed, not left over.
//
// For the gradients an entry's exponential becomes what the product has to find there for its
// own gradient, dl / (a factor), so that the product adds it up with the others'; where that is
// much larger than its 128's largest (a near 0, a student that holds the token for unlikely), or
// the rest is far below the entry, it becomes 0 and the entry stays in ids and dl (count of them).
// (A sure student's a q would cancel in the entries: a is -p_rest / q_rest then.)
// 3686 rows of 64 entries, 49152 tokens: TODO us, latency.
__global__ __launch_bounds__(512) void distill_kept_kernel(const DistillKept g) {
    extern __shared__ int tokens[];  // [8][k]
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int j = blockIdx.x * 8 + wave;
    const int scored = g.scored[1] == g.tag ? min(g.scored[0] - g.j0, g.chunk) : 0;
    if (j >= scored) return;  // (no barrier follows)
    const long r = g.idx[g.j0 + j];
    const int n = g.count[r];
    int* mine = tokens + wave * g.k;
    for (int k = lane; k < n; k += 64) mine[k] = g.ids[r * g.k + k];
    __builtin_amdgcn_wave_barrier();
    const TeacherRow row = g.row[r];
    const bool with_rest = row.p_rest > 0.0;
    auto kept = [&](int v) -> float& {
        char* p = g.keep + ((long)(j / 32) * g.v16 + v / 32 * 2) * 2048 + v % 32 / 8 * 1024 +
                  ((v % 8 / 4) * 32 + j % 32) * 16;
        return reinterpret_cast<float*>(p)[v % 4];
    };
    auto stat = [&](int part) { return g.stats[(long)part * g.ld + j]; };
    auto has_entry = [&](int part) {
        const int at = lower_bound(mine, n, part * 128);
        return at < n && mine[at] < part * 128 + 128;
    };
    // A logit in units of log2, by the whole wave.
    auto logit = [&](int v) {
        const float *h = g.hn + r * g.d, *w = g.head + (long)v * g.d;
        double s = 0.0;
        for (int i = lane; i < g.d; i += 64) s += (double)(h[i] * g.mul) * (double)w[i];
        return sum_wave(s) * (double)kLog2e;
    };
    float m = -INFINITY, m_rest = -INFINITY;
    for (int p = lane; p < g.parts; p += 64) {
        const float x = stat(p).x;
        m = fmaxf(m, x);
        if (with_rest && !has_entry(p)) m_rest = fmaxf(m_rest, x);
    }
    m = max_wave(m);
    m_rest = max_wave(m_rest);
    const double top = (double)m;
    double total = 0.0, rest = 0.0;  // in units of 2^top
    for (int p = lane; p < g.parts; p += 64) {
        const float2 s = stat(p);
        total += (double)(s.y * __builtin_amdgcn_exp2f(s.x - m));
        if (with_rest && !has_entry(p)) rest += (double)(s.y * __builtin_amdgcn_exp2f(s.x - m_rest));
    }
    total = sum_wave(total);
    constexpr float kLost = 0x1p-100f;  // of a kept exponential
    // The kept values of the 128 that entry `at` is the first of, four to each of 32 lanes, without
    // those of entries; the first entry behind them.
    const int v4 = lane % 32 * 4;
    auto others = [&](int at, float (&x4)[4]) {
        const int part = mine[at] / 128, v0 = part * 128 + v4;
#pragma unroll
        for (int i = 0; i < 4; i++) x4[i] = lane < 32 && v0 + i < g.vocab ? kept(v0 + i) : 0.0f;
        int last = at;
        for (; last < n && mine[last] / 128 == part; last++) {
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (mine[last] == v0 + i) x4[i] = 0.0f;
        }
        return last;
    };
    auto is_first = [&](int k) { return k < n && (k == 0 || mine[k - 1] / 128 != mine[k] / 128); };
    if (with_rest) {
        rest = sum_wave(rest);
        if (rest > 0.0) rest *= exp2((double)m_rest - top);
        // The 128s that have entries, by their first: what is left of their sums, then, where that
        // is not exact enough, the sum of the others.
        double left = 0.0;
        auto left_of = [&](int k, double& size) {
            const int part = mine[k] / 128;
            const float2 s = stat(part);
            double x = (double)s.y;
            for (int i = k; i < n && mine[i] / 128 == part; i++) x -= (double)kept(mine[i]);
            const double scale = pow2((double)s.x - top);
            size = (double)s.y * scale;
            return fmax(x, 0.0) * scale;
        };
        for (int k = lane; k < n; k += 64) {
            double size;
            if (is_first(k)) left += left_of(k, size);
        }
        const double about = rest + sum_wave(left);
        left = 0.0;
        for (int k0 = 0; k0 < n; k0 += 64) {
            const int k = k0 + lane;
            const bool first = is_first(k);
            double size = 0.0, x = 0.0;
            if (first) x = left_of(k, size);
            // (Kept values and their sum are off by some 2^-23 of it.)
            const bool again = first && !(size * 0x1p-22 <= about * 0x1p-18);
            if (!again) left += x;
            for (unsigned long long todo = __ballot(again); todo; todo &= todo - 1) {
                const int at = k0 + __ffsll(todo) - 1, part = mine[at] / 128;
                float x4[4];
                const int last = others(at, x4);
                const double sum = sum_wave((double)x4[0] + (double)x4[1] + (double)x4[2] + (double)x4[3]);
                const double scale = exp2((double)stat(part).x - top);
                double exact = sum * scale;
                if (!(128.0 * kLost * scale <= about * 0x1p-18) && !(sum > 128.0 * kLost * 0x1p18)) {
                    exact = 0.0;
                    const int end = min(part * 128 + 128, g.vocab);
                    for (int v = part * 128, i = at; v < end; v++) {
                        if (i < last && mine[i] == v)
                            i++;
                        else
                            exact += exp2(logit(v) - top);
                    }
                }
                if (lane == 0) left += exact;
            }
        }
        rest += sum_wave(left);
    }
    const double log_total = log(total), unit = 1.0 / (double)kLog2e;
    const Rest r_(row.p_rest, log(rest) - log_total);
    // (A rest so small has no exponentials in f32 either.)
    const float a = (float)(1.0 - fmin(r_.ratio, 1e30));
    double terms = 0.0;
    int stay = 0;
    for (int k0 = 0; k0 < n; k0 += 64) {
        const int k = k0 + lane;
        const bool live = k < n;
        const int v = live ? mine[k] : 0;
        const float e = live ? kept(v) : 1.0f;
        const double up = live ? (double)stat(v / 128).x - top : 0.0;
        double y = log2((double)e) + up, q = (double)e * pow2(up) / total;
        for (unsigned long long todo = __ballot(live && e < kLost); todo; todo &= todo - 1) {
            const int at = __ffsll(todo) - 1;
            const double x = logit(mine[k0 + at]) - top;
            if (lane == at) y = x, q = exp2(x) / total;
        }
        double dl = 0.0;
        if (live)
            terms += entry_loss(row, g.z[r * g.k + k], g.e[r * g.k + k], g.inv_t, q, y * unit - log_total, dl);
        if (!g.dl) continue;
        const bool far = with_rest && pow2(up) * 0x1p-10 > rest;
        const float in = live ? (float)dl / (a * g.factor[(long)(v / 128) * g.ld + j]) : 0.0f;
        // (Up to 2 the product's f16 pieces hold it.)
        const bool stays = live && (far || !(fabsf(in) <= 1.5f));
        const unsigned long long staying = __ballot(stays);
        if (stays) {
            const int to = stay + __popcll(staying & ((1ull << lane) - 1));
            g.ids[r * g.k + to] = v;
            g.dl[r * g.k + to] = (float)dl;
        }
        if (live) kept(v) = stays ? 0.0f : in;
        stay += __popcll(staying);
    }
    terms = sum_wave(terms);
    // The gradient's product takes a kept value to 2^-36: where an entry lies so far above the rest
    // that this shows in a q, the others of its 128 are scaled up.
    for (int k0 = 0; g.dl && with_rest && k0 < n; k0 += 64) {
        const int k = k0 + lane;
        const bool far = is_first(k) && pow2((double)stat(mine[k] / 128).x - top) * 0x1p-10 > rest;
        for (unsigned long long todo = __ballot(far); todo; todo &= todo - 1) {
            const int at = k0 + __ffsll(todo) - 1, part = mine[at] / 128;
            float x4[4];
            others(at, x4);
            const float most = max_wave(fmaxf(fmaxf(x4[0], x4[1]), fmaxf(x4[2], x4[3])));
            const int up = min(max(127 - (int)(__builtin_bit_cast(uint32_t, most) >> 23), 0), 126);
            if (!(most > 0.0f) || up == 0) continue;
            const float times = __builtin_bit_cast(float, (uint32_t)(127 + up) << 23);
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (lane < 32 && part * 128 + v4 + i < g.vocab) kept(part * 128 + v4 + i) = x4[i] * times;
            if (lane == 0) g.factor[(long)part * g.ld + j] *= __builtin_bit_cast(float, (uint32_t)(127 - up) << 23);
        }
    }
    if (lane) return;
    if (g.loss) g.loss[r] = (float)(r_.loss + terms);
    if (!g.dl) return;
    g.a[r] = a;
    g.count[r] = stay;
}

// Rows of logits in memory, a workgroup to one: the loss, where it is wanted, and with GRAD the
// logits become their gradients (zeros from the last scored row on).  The entries are taken out
// of the row before its sum, so the rest is one of its own.
template <bool GRAD>
__global__ __launch_bounds__(512) void distill_logits_kernel(float* __restrict__ logits, const DistillRows g) {
    extern __shared__ char lds[];
    int* tokens = reinterpret_cast<int*>(lds);            // [k]
    float* xs = reinterpret_cast<float*>(tokens + g.k);   // [k]
    __shared__ double red[2][8];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    float* x = logits + (long)blockIdx.x * g.vocab;
    if (g.j0 + (int)blockIdx.x >= *g.scored) {
        if (GRAD)
            for (long i = threadIdx.x; i < g.vocab; i += 512) x[i] = 0.0f;
        return;
    }
    const long r = g.idx[g.j0 + blockIdx.x];
    const int n = g.count[r];
    for (int k = threadIdx.x; k < n; k += 512) {
        const int v = g.ids[r * g.k + k];
        tokens[k] = v;
        xs[k] = x[v];
        x[v] = -INFINITY;
    }
    __syncthreads();
    float m = -INFINITY;
#pragma unroll 4
    for (long i = threadIdx.x; i < g.vocab; i += 512) m = fmaxf(m, x[i]);
    m = max_wave(m);
    if (lane == 0) red[0][wave] = (double)m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 8; w++) m = fmaxf(m, (float)red[0][w]);
    float s = 0.0f;
    if (m > -INFINITY)
#pragma unroll 4
        for (long i = threadIdx.x; i < g.vocab; i += 512) s += expf(x[i] - m);
    const double part = sum_wave((double)s);
    if (lane == 0) red[1][wave] = part;
    __syncthreads();
    double rest = 0.0;
#pragma unroll
    for (int w = 0; w < 8; w++) rest += red[1][w];
    // (Every wave for itself: a few entries a lane.)
    float top = m;
    for (int k = lane; k < n; k += 64) top = fmaxf(top, xs[k]);
    top = max_wave(top);
    double named = 0.0;
    for (int k = lane; k < n; k += 64) named += exp((double)xs[k] - (double)top);
    const double shift = rest > 0.0 ? (double)m - (double)top : 0.0;
    const double total = sum_wave(named) + rest * exp(shift), log_total = log(total);
    const TeacherRow row = g.row[r];
    const Rest r_(row.p_rest, log(rest) + shift - log_total);
    // An entry's part of the loss, and in dl the gradient of its logit.
    auto entry = [&](int k, double& dl) {
        const double log_q = (double)xs[k] - (double)top - log_total;
        return entry_loss(row, g.z[r * g.k + k], g.e[r * g.k + k], g.inv_t, exp(log_q), log_q, dl);
    };
    if (g.loss && wave == 0) {
        double terms = 0.0, dl;
        for (int k = lane; k < n; k += 64) terms += entry(k, dl);
        terms = sum_wave(terms);
        if (lane == 0) g.loss[r] = (float)(r_.loss + terms);
    }
    if (!GRAD) return;
    // (By the rest's own largest: a q of a confident student's is not small where q is.)
    const float f = (float)((1.0 - r_.ratio) * exp(shift) / total), base = m > -INFINITY ? m : 0.0f;
#pragma unroll 4
    for (long i = threadIdx.x; i < g.vocab; i += 512) x[i] = f * expf(x[i] - base);
    __syncthreads();
    for (int k = threadIdx.x; k < n; k += 512) {
        double dl;
        entry(k, dl);
        x[tokens[k]] = (float)dl;
    }
}

}  // namespace

hipError_t launch_distill_entries(const DistillEntries& g, hipStream_t st) {
    hipLaunchKernelGGL(distill_entries_kernel, dim3((unsigned)((g.t + 3) / 4)), dim3(256), 4 * g.k * sizeof(int), st, g);
    return hipGetLastError();
}
hipError_t launch_distill_kept(const DistillKept& g, hipStream_t st) {
    hipLaunchKernelGGL(distill_kept_kernel, dim3((unsigned)((g.chunk + 7) / 8)), dim3(512), 8 * g.k * sizeof(int), st,
                       g);
    return hipGetLastError();
}
hipError_t launch_distill_logits(float* logits, size_t nrows, bool grad, const DistillRows& g, hipStream_t st) {
    const size_t lds = g.k * (sizeof(int) + sizeof(float));
    hipLaunchKernelGGL((grad ? distill_logits_kernel<true> : distill_logits_kernel<false>), dim3((unsigned)nrows),
                       dim3(512), lds, st, logits, g);
    return hipGetLastError();
}

}  // namespace cfattn
