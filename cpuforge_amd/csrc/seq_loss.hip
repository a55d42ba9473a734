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

// Sums of K values over a group of NW waves, every lane getting them, in a fixed
// order.  red: K * NW values, free again after the caller's next barrier.
template <int NW, int K>
__device__ __forceinline__ void group_sums(double (&x)[K], double* red) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1)
#pragma unroll
        for (int k = 0; k < K; k++) x[k] += __shfl_xor(x[k], o);
    if constexpr (NW > 1) {
        __syncthreads();
        if ((threadIdx.x & 63) == 0)
#pragma unroll
            for (int k = 0; k < K; k++) red[k * NW + (threadIdx.x >> 6)] = x[k];
        __syncthreads();
#pragma unroll
        for (int k = 0; k < K; k++) {
            x[k] = 0.0;
#pragma unroll
            for (int i = 0; i < NW; i++) x[k] += red[k * NW + i];
        }
    }
}

__device__ __forceinline__ bool is_scored(const int64_t* __restrict__ targets, long r) {
    return !targets || targets[r] != kIgnoreIndex;
}

constexpr int kRows = 2;  // rows of a lane whose loads are in flight together

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
    double sums[4] = {};  // of either sequence, and its scored rows
#pragma unroll
    for (int k = 0; k < 2; k++)
        for (long r0 = s[k].lo + tid; r0 < s[k].hi; r0 += kRows * 64 * NW) {
            float x[kRows], y[kRows];
            bool use[kRows];
#pragma unroll
            for (int i = 0; i < kRows; i++) {
                const long r = r0 + i * 64 * NW, at = min(r, s[k].hi - 1);
                use[i] = is_scored(a.targets, at) && r < s[k].hi;
                x[i] = a.logp[at];
                y[i] = a.ref_logp ? a.ref_logp[at] : 0.0f;
            }
#pragma unroll
            for (int i = 0; i < kRows; i++)
                if (use[i]) {
                    sums[k] += (double)x[i] - (double)y[i];
                    sums[2 + k] += 1.0;
                }
        }
    group_sums<NW>(sums, red);
    double reward[2], share[2];
#pragma unroll
    for (int k = 0; k < 2; k++) {
        share[k] = a.length_mean ? a.beta / fmax(sums[2 + k], 1.0) : a.beta;
        reward[k] = sums[k] * share[k];
    }
    double l, dz;
    preference_term(a, reward[0] - reward[1] - a.margin, l, dz);
    dz /= (double)a.pairs;
#pragma unroll
    for (int k = 0; k < 2; k++) {
        const float d = (float)(k ? -dz * share[k] : dz * share[k]);
#pragma unroll 4
        for (long r = s[k].lo + tid; r < s[k].hi; r += 64 * NW) a.dlogp[r] = is_scored(a.targets, r) ? d : 0.0f;
    }
    if (tid == 0) {
        a.rewards[2 * pair] = (float)reward[0];
        a.rewards[2 * pair + 1] = (float)reward[1];
        a.terms[2 * pair] = s[0].bad || s[1].bad ? __builtin_nan("") : l;
        a.terms[2 * pair + 1] = reward[0] - reward[1];
    }
}

// The first sequence whose offsets do not rise within the rows, by a workgroup of NW
// waves (its barriers: two).
template <int NW>
__device__ __forceinline__ int first_bad(const int64_t* __restrict__ offsets, long seqs, long rows) {
    __shared__ int first;
    if (threadIdx.x == 0) first = INT_MAX;
    __syncthreads();
    for (long i = threadIdx.x; i < seqs; i += 64 * NW)
        if (span(offsets, i, rows).bad) atomicMin(&first, (int)i);
    __syncthreads();
    return first;
}

// The result from the pairs' terms, by one workgroup of NW waves.
template <int NW>
__device__ __forceinline__ void preference_result(const PreferenceArgs& a, double* red) {
    double sums[3] = {};
    for (long i = threadIdx.x; i < a.pairs; i += 64 * NW) {
        sums[0] += a.terms[2 * i];
        sums[1] += a.terms[2 * i + 1] > 0.0;
        sums[2] += a.terms[2 * i + 1];
    }
    const int bad = first_bad<NW>(a.offsets, 2 * a.pairs, a.rows);
    group_sums<NW>(sums, red);
    if (threadIdx.x == 0) {
        const double n = (double)a.pairs;
        *a.result = {bad, (float)(sums[0] / n), (float)(sums[1] / n), (float)(sums[2] / n)};
    }
}

__global__ __launch_bounds__(1024) void preference_small_kernel(const PreferenceArgs a) {
    __shared__ double red[3 * 16];
    for (long pair = threadIdx.x >> 6; pair < a.pairs; pair += 16) one_pair<1>(a, pair, red);
    __threadfence_block();
    __syncthreads();
    preference_result<16>(a, red);
}
__global__ __launch_bounds__(512) void preference_pair_kernel(const PreferenceArgs a) {
    __shared__ double red[4 * 8];
    one_pair<8>(a, blockIdx.x, red);
}
__global__ __launch_bounds__(1024) void preference_finish_kernel(const PreferenceArgs a) {
    __shared__ double red[3 * 16];
    preference_result<16>(a, red);
}

// ------------------------------------------------------------------- policy

// Scored rows of [lo, hi), by NW waves from lane `tid` on.
template <int NW>
__device__ __forceinline__ double count_rows(const PolicyArgs& a, const Span& s, int tid, double* red) {
    double n[1] = {};
    for (long r0 = s.lo + tid; r0 < s.hi; r0 += 8 * 64 * NW) {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const long r = r0 + i * 64 * NW;
            n[0] += is_scored(a.targets, min(r, s.hi - 1)) && r < s.hi;
        }
    }
    group_sums<NW>(n, red);
    return n[0];
}
__global__ __launch_bounds__(256) void policy_count_kernel(const PolicyArgs a) {
    __shared__ double red[4];
    const double n = count_rows<4>(a, span(a.offsets, blockIdx.x, a.rows), threadIdx.x, red);
    if (threadIdx.x == 0) a.counts[blockIdx.x] = (int)n;
}

// N, the scored rows, and M, the sequences with any, by a workgroup of NW waves.
template <int NW>
__device__ __forceinline__ void totals(const PolicyArgs& a, double& n, double& m, double* red) {
    double x[2] = {};
    for (long i = threadIdx.x; i < a.seqs; i += 64 * NW) {
        const int c = a.counts[i];
        x[0] += c;
        x[1] += c > 0;
    }
    group_sums<NW>(x, red);
    n = x[0], m = x[1];
}

// One row's gradient, its terms added to the lane's sums (loss, KL, cut rows).
__device__ __forceinline__ float policy_row(const PolicyArgs& a, double w, double lp, double old, double ref, double adv,
                                            double (&sums)[3]) {
    const double diff = a.old_logp ? lp - old : 0.0;
    const double ratio = exp(diff);
    // min(r A, clip(r) A) is the clipped one past the border on the side A pushes to.
    const bool up = adv > 0.0 && diff > a.log_high, down = adv < 0.0 && diff < a.log_low;
    double l = -ratio * adv, dl = l;
    if (up || down) {
        l = -(up ? a.high : a.low) * adv;
        dl = 0.0;
        sums[2] += 1.0;
    }
    if (a.ref_logp) {
        const double x = ref - lp, e = expm1(x);
        sums[1] += w * (e - x);
        l += a.kl_coef * (e - x);
        dl -= a.kl_coef * e;
    }
    sums[0] += w * l;
    return (float)(dl * w);
}

// The rows of sequence `seq`, whose scored ones weigh w, from lane `tid` of NW waves on.
template <int NW>
__device__ __forceinline__ void policy_rows(const PolicyArgs& a, long seq, const Span& s, double w, int tid,
                                            double (&sums)[3]) {
    for (long r0 = s.lo + tid; r0 < s.hi; r0 += kRows * 64 * NW) {
        float lp[kRows], old[kRows], ref[kRows], adv[kRows];
        bool use[kRows];
#pragma unroll
        for (int i = 0; i < kRows; i++) {
            const long r = min(r0 + i * 64 * NW, s.hi - 1);
            use[i] = is_scored(a.targets, r);
            lp[i] = a.logp[r];
            old[i] = a.old_logp ? a.old_logp[r] : 0.0f;
            ref[i] = a.ref_logp ? a.ref_logp[r] : 0.0f;
            adv[i] = a.advantages[a.per_token ? r : seq];
        }
#pragma unroll
        for (int i = 0; i < kRows; i++) {
            const long r = r0 + i * 64 * NW;
            if (r >= s.hi) break;
            a.dlogp[r] = use[i] ? policy_row(a, w, lp[i], old[i], ref[i], adv[i], sums) : 0.0f;
        }
    }
}

__device__ __forceinline__ double row_weight(const PolicyArgs& a, long seq, double n, double m) {
    const double c = fmax((double)a.counts[seq], 1.0);
    return a.sequence_mean ? 1.0 / (c * fmax(m, 1.0)) : 1.0 / fmax(n, 1.0);
}

template <int NW>
__device__ __forceinline__ void policy_result(const PolicyArgs& a, double (&sums)[3], double n, double* red) {
    const int bad = first_bad<NW>(a.offsets, a.seqs, a.rows);
    group_sums<NW>(sums, red);
    if (threadIdx.x == 0)
        *a.result = {(int)n, bad, bad == INT_MAX ? (float)sums[0] : __builtin_nanf(""), (float)sums[1],
                     (float)(sums[2] / fmax(n, 1.0))};
}

// A wave to a sequence, one workgroup for all.
__global__ __launch_bounds__(1024) void policy_small_kernel(const PolicyArgs a) {
    __shared__ double red[3 * 16];
    const int lane = threadIdx.x & 63;
    for (long i = threadIdx.x >> 6; i < a.seqs; i += 16) {
        const double n = count_rows<1>(a, span(a.offsets, i, a.rows), lane, red);
        if (lane == 0) a.counts[i] = (int)n;
    }
    __threadfence_block();
    __syncthreads();
    double n, m, sums[3] = {};
    totals<16>(a, n, m, red);
    for (long i = threadIdx.x >> 6; i < a.seqs; i += 16)
        policy_rows<1>(a, i, span(a.offsets, i, a.rows), row_weight(a, i, n, m), lane, sums);
    policy_result<16>(a, sums, n, red);
}

// A workgroup to a sequence: its terms go to `terms`.
__global__ __launch_bounds__(256) void policy_seq_kernel(const PolicyArgs a) {
    __shared__ double red[3 * 4];
    double n, m, sums[3] = {};
    totals<4>(a, n, m, red);
    const long i = blockIdx.x;
    policy_rows<4>(a, i, span(a.offsets, i, a.rows), row_weight(a, i, n, m), threadIdx.x, sums);
    group_sums<4>(sums, red);
    if (threadIdx.x < 3) a.terms[3 * i + threadIdx.x] = threadIdx.x == 0 ? sums[0] : threadIdx.x == 1 ? sums[1] : sums[2];
}
__global__ __launch_bounds__(1024) void policy_finish_kernel(const PolicyArgs a) {
    __shared__ double red[3 * 16];
    double n, m, sums[3] = {};
    totals<16>(a, n, m, red);
    for (long i = threadIdx.x; i < a.seqs; i += 1024)
#pragma unroll
        for (int k = 0; k < 3; k++) sums[k] += a.terms[3 * i + k];
    policy_result<16>(a, sums, n, red);
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
