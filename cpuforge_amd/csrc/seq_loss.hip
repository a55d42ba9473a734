// Losses over the log-probabilities of packed sequences, with their gradients:
// a preference loss over pairs and a clipped policy loss with a KL term
// (cfops_preference_loss, cfops_policy_loss of include/cfops.h).
//
// Sequence i is rows [offsets[i], offsets[i+1]); a row whose target is
// kIgnoreIndex is not scored (its log-probabilities are not read, its gradient
// is 0).  Sums run over f64 values in a fixed order: a difference of two f32
// log-probabilities is exact there, and so is the side of the clipping border
// that a ratio falls on (a difference against the border's logarithm, to f64).
// Offsets that do not rise within [0, rows] are not followed: their sequence is
// empty, the loss is NaN and the result names it.
#include <limits.h>

#include <algorithm>

#include "cfattn_common.hpp"
#include "cfops_kernels.hpp"

namespace cfattn {
namespace {

constexpr long kIgnoreIndex = -100;  // crates/core/src/ops/loss.rs:4

struct Span {
    long lo, hi;
    bool bad;
};
__device__ __forceinline__ Span span(const int64_t* __restrict__ offsets, long i, long rows) {
    const long lo = offsets[i], hi = offsets[i + 1];
    const bool bad = lo < 0 || hi < lo || hi > rows;
    return {bad ? 0 : lo, bad ? 0 : hi, bad};
}

// Sum over a group of NW waves, every lane getting it, in a fixed order.
template <int NW>
__device__ __forceinline__ double group_sum(double x, double* red) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) x += __shfl_xor(x, o);
    if constexpr (NW > 1) {
        __syncthreads();
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = x;
        __syncthreads();
        x = 0.0;
#pragma unroll
        for (int i = 0; i < NW; i++) x += red[i];
    }
    return x;
}

struct PairTerms {
    double loss, margin;
    int accurate;
};

// log(1 + exp(x)).
__device__ __forceinline__ double softplus(double x) { return fmax(x, 0.0) + log1p(exp(-fabs(x))); }

// l(z) and its derivative.
__device__ __forceinline__ void preference_term(const PreferenceArgs& a, double z, double& l, double& dz) {
    if (a.form == 0) {
        const double s = 1.0 / (1.0 + exp(-fabs(z))), sig = z >= 0.0 ? s : exp(-fabs(z)) * s;
        l = (1.0 - a.label_smoothing) * softplus(-z) + a.label_smoothing * softplus(z);
        dz = (1.0 - a.label_smoothing) * (sig - 1.0) + a.label_smoothing * sig;
    } else if (a.form == 1) {
        l = fmax(1.0 - z, 0.0);
        dz = z < 1.0 ? -1.0 : 0.0;
        if (z != z) l = dz = z;
    } else {
        l = (z - 0.5) * (z - 0.5);
        dz = 2.0 * (z - 0.5);
    }
}

// One pair, by NW waves (of a workgroup of as many, or each on its own with NW == 1).
template <int NW>
__device__ __forceinline__ void one_pair(const PreferenceArgs& a, long pair, double* red) {
    const int tid = NW == 1 ? threadIdx.x & 63 : threadIdx.x;
    const Span s[2] = {span(a.offsets, 2 * pair, a.rows), span(a.offsets, 2 * pair + 1, a.rows)};
    double reward[2], share[2];
#pragma unroll
    for (int k = 0; k < 2; k++) {
        double sum = 0.0, cnt = 0.0;
        for (long r = s[k].lo + tid; r < s[k].hi; r += 64 * NW)
            if (!a.targets || a.targets[r] != kIgnoreIndex) {
                sum += (double)a.logp[r] - (a.ref_logp ? (double)a.ref_logp[r] : 0.0);
                cnt += 1.0;
            }
        sum = group_sum<NW>(sum, red);
        cnt = group_sum<NW>(cnt, red);
        share[k] = a.length_mean ? a.beta / fmax(cnt, 1.0) : a.beta;
        reward[k] = sum * share[k];
    }
    double l, dz;
    preference_term(a, reward[0] - reward[1] - a.margin, l, dz);
    dz /= (double)a.pairs;
#pragma unroll
    for (int k = 0; k < 2; k++) {
        const float d = (float)(k ? -dz * share[k] : dz * share[k]);
        for (long r = s[k].lo + tid; r < s[k].hi; r += 64 * NW)
            a.dlogp[r] = !a.targets || a.targets[r] != kIgnoreIndex ? d : 0.0f;
    }
    if (tid == 0) {
        a.rewards[2 * pair] = (float)reward[0];
        a.rewards[2 * pair + 1] = (float)reward[1];
        a.terms[2 * pair] = s[0].bad || s[1].bad ? __builtin_nan("") : l;
        a.terms[2 * pair + 1] = reward[0] - reward[1];
    }
}

// The result from the pairs' terms, by one workgroup of NW waves.
template <int NW>
__device__ __forceinline__ void preference_result(const PreferenceArgs& a, double* red) {
    double loss = 0.0, margin = 0.0, accurate = 0.0;
    int bad = INT_MAX;
    for (long i = threadIdx.x; i < a.pairs; i += 64 * NW) {
        loss += a.terms[2 * i];
        margin += a.terms[2 * i + 1];
        accurate += a.terms[2 * i + 1] > 0.0;
        for (int k = 1; k >= 0; k--)
            if (span(a.offsets, 2 * i + k, a.rows).bad) bad = min(bad, (int)(2 * i + k));
    }
    loss = group_sum<NW>(loss, red);
    margin = group_sum<NW>(margin, red);
    accurate = group_sum<NW>(accurate, red);
    __shared__ int first;
    if (threadIdx.x == 0) first = INT_MAX;
    __syncthreads();
    if (bad != INT_MAX) atomicMin(&first, bad);
    __syncthreads();
    if (threadIdx.x == 0) {
        const double n = fmax((double)a.pairs, 1.0);
        *a.result = {first, (float)(loss / n), (float)(accurate / n), (float)(margin / n)};
    }
}

__global__ __launch_bounds__(1024) void preference_small_kernel(const PreferenceArgs a) {
    __shared__ double red[16];
    for (long pair = threadIdx.x >> 6; pair < a.pairs; pair += 16) one_pair<1>(a, pair, red);
    __threadfence_block();
    __syncthreads();
    preference_result<16>(a, red);
}
__global__ __launch_bounds__(512) void preference_pair_kernel(const PreferenceArgs a) {
    __shared__ double red[8];
    one_pair<8>(a, blockIdx.x, red);
}
__global__ __launch_bounds__(1024) void preference_finish_kernel(const PreferenceArgs a) {
    __shared__ double red[16];
    preference_result<16>(a, red);
}

// ------------------------------------------------------------------- policy

// Scored rows of a sequence, by one workgroup of four waves.
__global__ __launch_bounds__(256) void policy_count_kernel(const PolicyArgs a) {
    __shared__ double red[4];
    const Span s = span(a.offsets, blockIdx.x, a.rows);
    double n = 0.0;
    for (long r = s.lo + threadIdx.x; r < s.hi; r += 256) n += !a.targets || a.targets[r] != kIgnoreIndex;
    n = group_sum<4>(n, red);
    if (threadIdx.x == 0) a.counts[blockIdx.x] = (int)n;
}

// N, the scored rows, and M, the sequences with any, by a workgroup of NW waves.
template <int NW>
__device__ __forceinline__ void totals(const PolicyArgs& a, double& n, double& m, double* red) {
    n = m = 0.0;
    for (long i = threadIdx.x; i < a.seqs; i += 64 * NW) {
        const int c = a.counts[i];
        n += c;
        m += c > 0;
    }
    n = group_sum<NW>(n, red);
    m = group_sum<NW>(m, red);
}

// Rows [r0, r1) of sequence `seq` whose scored rows weigh w: their gradients, and
// their terms added to the lane's sums.
__device__ __forceinline__ void policy_rows(const PolicyArgs& a, long seq, double w, long r, long r1, int step,
                                            double& loss, double& kl, double& cuts) {
    for (; r < r1; r += step) {
        float d = 0.0f;
        if (!a.targets || a.targets[r] != kIgnoreIndex) {
            const double lp = a.logp[r];
            const double adv = a.advantages[a.per_token ? r : seq];
            const double diff = a.old_logp ? lp - (double)a.old_logp[r] : 0.0;
            const double ratio = exp(diff);
            // min(r A, clip(r) A) is the clipped one past the border on the side A
            // pushes to.
            const bool up = adv > 0.0 && diff > a.log_high, down = adv < 0.0 && diff < a.log_low;
            double l = -ratio * adv, dl = l;
            if (up || down) {
                l = -(up ? a.high : a.low) * adv;
                dl = 0.0;
                cuts += 1.0;
            }
            if (a.ref_logp) {
                const double x = (double)a.ref_logp[r] - lp, e = expm1(x);
                kl += w * (e - x);
                l += a.kl_coef * (e - x);
                dl -= a.kl_coef * e;
            }
            loss += w * l;
            d = (float)(dl * w);
        }
        a.dlogp[r] = d;
    }
}

__device__ __forceinline__ double row_weight(const PolicyArgs& a, long seq, double n, double m) {
    const double c = fmax((double)a.counts[seq], 1.0);
    return a.sequence_mean ? 1.0 / (c * fmax(m, 1.0)) : 1.0 / fmax(n, 1.0);
}

template <int NW>
__device__ __forceinline__ void policy_result(const PolicyArgs& a, double loss, double kl, double cuts, double n,
                                              double* red) {
    loss = group_sum<NW>(loss, red);
    kl = group_sum<NW>(kl, red);
    cuts = group_sum<NW>(cuts, red);
    __shared__ int first;
    if (threadIdx.x == 0) first = INT_MAX;
    __syncthreads();
    for (long i = threadIdx.x; i < a.seqs; i += 64 * NW)
        if (span(a.offsets, i, a.rows).bad) atomicMin(&first, (int)i);
    __syncthreads();
    if (threadIdx.x == 0)
        *a.result = {(int)n, first, first == INT_MAX ? (float)loss : __builtin_nanf(""), (float)kl,
                     (float)(cuts / fmax(n, 1.0))};
}

// A wave to a sequence, one workgroup for all.
__global__ __launch_bounds__(1024) void policy_small_kernel(const PolicyArgs a) {
    __shared__ double red[16];
    const int lane = threadIdx.x & 63;
    for (long i = threadIdx.x >> 6; i < a.seqs; i += 16) {
        const Span s = span(a.offsets, i, a.rows);
        double n = 0.0;
        for (long r = s.lo + lane; r < s.hi; r += 64) n += !a.targets || a.targets[r] != kIgnoreIndex;
        n = group_sum<1>(n, red);
        if (lane == 0) a.counts[i] = (int)n;
    }
    __threadfence_block();
    __syncthreads();
    double n, m, loss = 0.0, kl = 0.0, cuts = 0.0;
    totals<16>(a, n, m, red);
    for (long i = threadIdx.x >> 6; i < a.seqs; i += 16) {
        const Span s = span(a.offsets, i, a.rows);
        policy_rows(a, i, row_weight(a, i, n, m), s.lo + lane, s.hi, 64, loss, kl, cuts);
    }
    policy_result<16>(a, loss, kl, cuts, n, red);
}

// A workgroup to a sequence: its terms go to `terms`.
__global__ __launch_bounds__(256) void policy_seq_kernel(const PolicyArgs a) {
    __shared__ double red[4];
    double n, m, loss = 0.0, kl = 0.0, cuts = 0.0;
    totals<4>(a, n, m, red);
    const long i = blockIdx.x;
    const Span s = span(a.offsets, i, a.rows);
    policy_rows(a, i, row_weight(a, i, n, m), s.lo + threadIdx.x, s.hi, 256, loss, kl, cuts);
    loss = group_sum<4>(loss, red);
    kl = group_sum<4>(kl, red);
    cuts = group_sum<4>(cuts, red);
    if (threadIdx.x == 0) {
        a.terms[3 * i] = loss;
        a.terms[3 * i + 1] = kl;
        a.terms[3 * i + 2] = cuts;
    }
}
__global__ __launch_bounds__(1024) void policy_finish_kernel(const PolicyArgs a) {
    __shared__ double red[16];
    double n, m, loss = 0.0, kl = 0.0, cuts = 0.0;
    totals<16>(a, n, m, red);
    for (long i = threadIdx.x; i < a.seqs; i += 1024) {
        loss += a.terms[3 * i];
        kl += a.terms[3 * i + 1];
        cuts += a.terms[3 * i + 2];
    }
    policy_result<16>(a, loss, kl, cuts, n, red);
}

}  // namespace

size_t preference_scratch_bytes(size_t pairs) { return 2 * std::max<size_t>(pairs, 1) * sizeof(double); }
size_t policy_scratch_bytes(size_t seqs) {
    return std::max<size_t>(seqs, 1) * (3 * sizeof(double) + sizeof(int));
}

hipError_t launch_preference(PreferenceArgs a, void* scratch, hipStream_t st) {
    a.terms = static_cast<double*>(scratch);
    if (a.rows <= 16384 && a.pairs <= 64) {
        hipLaunchKernelGGL(preference_small_kernel, dim3(1), dim3(1024), 0, st, a);
        return hipGetLastError();
    }
    hipLaunchKernelGGL(preference_pair_kernel, dim3((unsigned)a.pairs), dim3(512), 0, st, a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(preference_finish_kernel, dim3(1), dim3(1024), 0, st, a);
    return hipGetLastError();
}

hipError_t launch_policy(PolicyArgs a, void* scratch, hipStream_t st) {
    a.terms = static_cast<double*>(scratch);
    a.counts = reinterpret_cast<int*>(a.terms + 3 * std::max<size_t>(a.seqs, 1));
    if (a.rows <= 16384 && a.seqs <= 64) {
        hipLaunchKernelGGL(policy_small_kernel, dim3(1), dim3(1024), 0, st, a);
        return hipGetLastError();
    }
    hipLaunchKernelGGL(policy_count_kernel, dim3((unsigned)a.seqs), dim3(256), 0, st, a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(policy_seq_kernel, dim3((unsigned)a.seqs), dim3(256), 0, st, a);
    e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(policy_finish_kernel, dim3(1), dim3(1024), 0, st, a);
    return hipGetLastError();
}

}  // namespace cfattn
