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
//
// A pass over a sequence needs what another pass summed over it (a pair's rewards;
// the rows or sequences that a mean is over), so there are two to four launches, most
// with `parts` workgroups to a sequence: long ones are split, and a part's sums are
// added in order by whoever needs them.  Bound by those launches: 400 pairs of 2 x 1024
// rows (13 MB) 9.3 us, 1024 rollouts of 1100 (32 MB) 21 us.
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
constexpr int kWaves = 4;  // of a part's workgroup
constexpr size_t kWgs = 1024;
// Workgroups of the policy loss up to which each adds all counts for itself, which saves a
// launch: beyond, their reads grow with the square of the sequences.  (Us of a captured
// call, each for itself and once for all: 1024 sequences of 1100 rows 20.8 and 20.4, 2048 of
// 100 21.7 and 19.2, 4096 of 400 38.3 and 30.3, 16384 of 50 162 and 66, 131072 of 4 5900 and
// 499.)
constexpr unsigned kTotalsWgs = 1024;

// Part p of a sequence's rows.
__device__ __forceinline__ Span part_of(const Span& s, long p, int parts) {
    const unsigned n = (unsigned)(s.hi - s.lo);
    const long size = (n + (unsigned)parts - 1) / (unsigned)parts;
    return {s.lo + min(size * p, (long)n), s.lo + min(size * (p + 1), (long)n), s.bad};
}

// log(1 + exp(x)).
__device__ __forceinline__ double softplus(double x) { return fmax(x, 0.0) + log1p(exp(-fabs(x))); }

// l(z) and its derivative.
__device__ __forceinline__ void preference_term(const PreferenceArgs& a, double z, double& l, double& dz) {
    if (a.form == 0) {
        const double s = 1.0 / (1.0 + exp(-fabs(z))), sig = z >= 0.0 ? s : exp(-fabs(z)) * s;
        l = (1.0 - a.label_smoothing) * softplus(-z);
        if (a.label_smoothing != 0.0) l += a.label_smoothing * softplus(z);  // (0 times infinity is no term)
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

// The sum over rows [s.lo, s.hi) of logp - ref_logp and the scored rows, by NW waves from
// lane `tid` on.
template <int NW>
__device__ __forceinline__ void preference_rows(const PreferenceArgs& a, const Span& s, int tid, double (&sums)[2],
                                                double* red) {
    sums[0] = sums[1] = 0.0;
    for (long r0 = s.lo + tid; r0 < s.hi; r0 += kRows * 64 * NW) {
        float x[kRows], y[kRows];
        bool use[kRows];
#pragma unroll
        for (int i = 0; i < kRows; i++) {
            const long r = r0 + i * 64 * NW, at = min(r, s.hi - 1);
            use[i] = is_scored(a.targets, at) && r < s.hi;
            x[i] = a.logp[at];
            y[i] = a.ref_logp ? a.ref_logp[at] : 0.0f;
        }
#pragma unroll
        for (int i = 0; i < kRows; i++)
            if (use[i]) {
                sums[0] += (double)x[i] - (double)y[i];
                sums[1] += 1.0;
            }
    }
    group_sums<NW>(sums, red);
}

// A sequence's reward and what a row's log-probability moves it by, from its parts'
// sums: lane `lane` of `lanes` (a power of two).
struct Reward {
    double value, share;
};
__device__ __forceinline__ Reward reward_of(const PreferenceArgs& a, long seq, int lane, int lanes) {
    double x = 0.0, n = 0.0;
    for (int i = lane; i < a.parts; i += lanes) {
        const double2 t = a.terms[seq * a.parts + i];
        x += t.x, n += t.y;
    }
    for (int o = lanes >> 1; o >= 1; o >>= 1) x += __shfl_xor(x, o), n += __shfl_xor(n, o);
    const double share = a.length_mean ? a.beta / fmax(n, 1.0) : a.beta;
    return {x * share, share};
}

struct Pair {
    Reward chosen, rejected;
    double loss, dz;
};
__device__ __forceinline__ Pair one_pair(const PreferenceArgs& a, long pair, int lane, int lanes) {
    Pair p;
    p.chosen = reward_of(a, 2 * pair, lane, lanes);
    p.rejected = reward_of(a, 2 * pair + 1, lane, lanes);
    preference_term(a, p.chosen.value - p.rejected.value - a.margin, p.loss, p.dz);
    return p;
}

// The gradient of sequence `seq` of the pair in rows [s.lo, s.hi), and its reward.
template <int NW>
__device__ __forceinline__ void preference_grad(const PreferenceArgs& a, const Pair& p, long seq, const Span& s, int tid,
                                                bool first) {
    const double dz = p.dz / (double)a.pairs, up = dz * p.chosen.share, down = -dz * p.rejected.share;
    const float d = seq & 1 ? (float)down : (float)up;
#pragma unroll 4
    for (long r = s.lo + tid; r < s.hi; r += 64 * NW) a.dlogp[r] = is_scored(a.targets, r) ? d : 0.0f;
    const float chosen = (float)p.chosen.value, rejected = (float)p.rejected.value;
    if (first && tid == 0) a.rewards[seq] = seq & 1 ? rejected : chosen;
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

// The result, by one workgroup of NW waves.
template <int NW>
__device__ __forceinline__ void preference_result(const PreferenceArgs& a, double* red) {
    int lanes = 1;  // to a pair
    while (lanes < min(a.parts, 64)) lanes *= 2;
    const int lane = threadIdx.x & (lanes - 1);
    double sums[3] = {};
    for (long i = threadIdx.x / lanes; i < a.pairs; i += 64 * NW / lanes) {
        const Pair p = one_pair(a, i, lane, lanes);
        if (lane) continue;
        sums[0] += p.loss;
        const double more = p.chosen.value - p.rejected.value;
        sums[1] += more > 0.0;
        sums[2] += more;
    }
    const int bad = first_bad<NW>(a.offsets, 2 * a.pairs, a.rows);
    group_sums<NW>(sums, red);
    if (threadIdx.x == 0) {
        const double n = (double)a.pairs;
        *a.result = {bad, bad == INT_MAX ? (float)(sums[0] / n) : __builtin_nanf(""), (float)(sums[1] / n),
                     (float)(sums[2] / n)};
    }
}

// A wave to a sequence, then to its gradient: one workgroup, parts == 1.
__global__ __launch_bounds__(1024) void preference_small_kernel(const PreferenceArgs a) {
    __shared__ double red[3 * 16];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (long i = wave; i < 2 * a.pairs; i += 16) {
        double sums[2];
        preference_rows<1>(a, span(a.offsets, i, a.rows), lane, sums, red);
        if (lane == 0) a.terms[i] = make_double2(sums[0], sums[1]);
    }
    __threadfence_block();
    __syncthreads();
    for (long i = wave; i < 2 * a.pairs; i += 16)
        preference_grad<1>(a, one_pair(a, i / 2, 0, 1), i, span(a.offsets, i, a.rows), lane, true);
    preference_result<16>(a, red);
}
__global__ __launch_bounds__(64 * kWaves) void preference_sum_kernel(const PreferenceArgs a) {
    __shared__ double red[2 * kWaves];
    const long seq = blockIdx.x / (unsigned)a.parts;
    const int part = (int)(blockIdx.x % (unsigned)a.parts);
    double sums[2];
    preference_rows<kWaves>(a, part_of(span(a.offsets, seq, a.rows), part, a.parts), threadIdx.x, sums, red);
    if (threadIdx.x == 0) a.terms[blockIdx.x] = make_double2(sums[0], sums[1]);
}
// The first workgroup has the result, the others a part's gradient each.
__global__ __launch_bounds__(64 * kWaves) void preference_grad_kernel(const PreferenceArgs a) {
    __shared__ double red[3 * kWaves];
    if (blockIdx.x == 0) return preference_result<kWaves>(a, red);
    const unsigned b = blockIdx.x - 1;
    const long seq = b / (unsigned)a.parts;
    const int part = (int)(b % (unsigned)a.parts);
    const bool one = a.parts == 1;
    const Pair p = one_pair(a, seq / 2, one ? 0 : threadIdx.x & 63, one ? 1 : 64);
    preference_grad<kWaves>(a, p, seq, part_of(span(a.offsets, seq, a.rows), part, a.parts), threadIdx.x, part == 0);
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
__global__ __launch_bounds__(64 * kWaves) void policy_count_kernel(const PolicyArgs a) {
    __shared__ double red[kWaves];
    const Span s = span(a.offsets, blockIdx.x / (unsigned)a.parts, a.rows);
    const double n = count_rows<kWaves>(a, part_of(s, blockIdx.x % (unsigned)a.parts, a.parts), threadIdx.x, red);
    if (threadIdx.x == 0) a.counts[blockIdx.x] = (int)n;
}

// N, the scored rows, and, for means over sequences, M, those with any, by a workgroup
// of NW waves.
template <int NW>
__device__ __forceinline__ void totals(const PolicyArgs& a, double& n, double& m, double* red) {
    double x[2] = {};
    if (a.sequence_mean) {
        int lanes = 1;  // to a sequence
        while (lanes < min(a.parts, 64)) lanes *= 2;
        const int lane = threadIdx.x & (lanes - 1);
        for (long i = threadIdx.x / lanes; i < a.seqs; i += 64 * NW / lanes) {
            int c = 0;
            for (int p = lane; p < a.parts; p += lanes) c += a.counts[i * a.parts + p];
            for (int o = lanes >> 1; o >= 1; o >>= 1) c += __shfl_xor(c, o);
            if (lane) continue;
            x[0] += c;
            x[1] += c > 0;
        }
    } else {
        for (long i = threadIdx.x; i < a.seqs * a.parts; i += 64 * NW) x[0] += a.counts[i];
    }
    group_sums<NW>(x, red);
    n = x[0], m = x[1];
}

// The same once for all workgroups.
__global__ __launch_bounds__(1024) void policy_totals_kernel(const PolicyArgs a) {
    __shared__ double red[2 * 16];
    double n, m;
    totals<16>(a, n, m, red);
    if (threadIdx.x == 0) a.totals[0] = n, a.totals[1] = m;
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
    if (!a.sequence_mean) return 1.0 / fmax(n, 1.0);
    int c = 0;
    for (int p = threadIdx.x & 63; p < a.parts; p += 64) c += a.counts[seq * a.parts + p];
    for (int o = 32; o >= 1; o >>= 1) c += __shfl_xor(c, o);
    return 1.0 / (fmax((double)c, 1.0) * fmax(m, 1.0));
}

template <int NW>
__device__ __forceinline__ void policy_result(const PolicyArgs& a, double (&sums)[3], double n, double* red) {
    const int bad = first_bad<NW>(a.offsets, a.seqs, a.rows);
    group_sums<NW>(sums, red);
    if (threadIdx.x == 0)
        *a.result = {(int)n, bad, bad == INT_MAX ? (float)sums[0] : __builtin_nanf(""), (float)sums[1],
                     (float)(sums[2] / fmax(n, 1.0))};
}

// A wave to a sequence, one workgroup for all, parts == 1.
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

// A part's gradient; its terms go to `terms`.
__global__ __launch_bounds__(64 * kWaves) void policy_part_kernel(const PolicyArgs a) {
    __shared__ double red[3 * kWaves];
    double n, m, sums[3] = {};
    if (a.totals)
        n = a.totals[0], m = a.totals[1];
    else
        totals<kWaves>(a, n, m, red);
    const long seq = blockIdx.x / (unsigned)a.parts;
    const Span s = part_of(span(a.offsets, seq, a.rows), blockIdx.x % (unsigned)a.parts, a.parts);
    policy_rows<kWaves>(a, seq, s, row_weight(a, seq, n, m), threadIdx.x, sums);
    group_sums<kWaves>(sums, red);
    if (threadIdx.x < 3) a.terms[3l * blockIdx.x + threadIdx.x] = threadIdx.x == 0 ? sums[0] : threadIdx.x == 1 ? sums[1] : sums[2];
}
__global__ __launch_bounds__(1024) void policy_finish_kernel(const PolicyArgs a) {
    __shared__ double red[3 * 16];
    double n, m, sums[3] = {};
    if (a.totals)
        n = a.totals[0];
    else
        totals<16>(a, n, m, red);
    for (long i = threadIdx.x; i < a.seqs * a.parts; i += 1024)
#pragma unroll
        for (int k = 0; k < 3; k++) sums[k] += a.terms[3 * i + k];
    policy_result<16>(a, sums, n, red);
}

}  // namespace

// One workgroup, a wave to a sequence, where that is a few reads long: it is bound by
// latency, and so is a second launch.  Us of a captured call (of one from the host, which
// a launch takes longer to issue than to run), against the form for many:
//   preference: 8 sequences, 1024 rows 7.1 (7.4) and 5.9 (10.0); 2 of 1000 9.6 and 6.5;
//   policy:     8 sequences, 1024 rows 8.2 (8.3) and 12 (13.5);  1 of 1000 16.7 and 12.
static bool small(size_t rows, size_t seqs) { return seqs <= 16 && rows <= 1024 && rows <= 256 * seqs; }
// Workgroups to a sequence: with few long sequences as many as fill the card, of no
// fewer than two rows a lane on average.  (One of 65536 rows: preference 61 and policy
// 195 us by one workgroup, 6.8 and 12.6 by 128.  As many to every sequence, 128 of 128
// rows by 8 each: 22 where one takes 6.)  By the mean length: one long sequence beside
// hundreds of short ones has one workgroup.
static int parts_of(size_t rows, size_t seqs) {
    if (small(rows, seqs)) return 1;
    return (int)std::max<size_t>(1, std::min(kWgs / seqs, rows / (seqs * kRows * 64 * kWaves)));
}

size_t preference_scratch_bytes(size_t rows, size_t pairs) {
    return 2 * pairs * parts_of(rows, 2 * pairs) * sizeof(double2);
}
size_t policy_scratch_bytes(size_t rows, size_t seqs) {
    return 2 * sizeof(double) + seqs * parts_of(rows, seqs) * (3 * sizeof(double) + sizeof(int));
}

hipError_t launch_preference(PreferenceArgs a, void* scratch, hipStream_t st) {
    a.terms = static_cast<double2*>(scratch);
    a.parts = parts_of(a.rows, 2 * a.pairs);
    if (small(a.rows, 2 * a.pairs)) {
        hipLaunchKernelGGL(preference_small_kernel, dim3(1), dim3(1024), 0, st, a);
        return hipGetLastError();
    }
    const unsigned wgs = (unsigned)(2 * a.pairs * a.parts);
    hipLaunchKernelGGL(preference_sum_kernel, dim3(wgs), dim3(64 * kWaves), 0, st, a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(preference_grad_kernel, dim3(wgs + 1), dim3(64 * kWaves), 0, st, a);
    return hipGetLastError();
}

hipError_t launch_policy(PolicyArgs a, void* scratch, hipStream_t st) {
    a.parts = parts_of(a.rows, a.seqs);
    a.totals = nullptr;
    a.terms = static_cast<double*>(scratch) + 2;
    a.counts = reinterpret_cast<int*>(a.terms + 3 * a.seqs * a.parts);
    if (small(a.rows, a.seqs)) {
        hipLaunchKernelGGL(policy_small_kernel, dim3(1), dim3(1024), 0, st, a);
        return hipGetLastError();
    }
    const unsigned wgs = (unsigned)(a.seqs * a.parts);
    hipLaunchKernelGGL(policy_count_kernel, dim3(wgs), dim3(64 * kWaves), 0, st, a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    if (wgs > kTotalsWgs) {
        a.totals = static_cast<double*>(scratch);
        hipLaunchKernelGGL(policy_totals_kernel, dim3(1), dim3(1024), 0, st, a);
        if ((e = hipGetLastError()) != hipSuccess) return e;
    }
    hipLaunchKernelGGL(policy_part_kernel, dim3(wgs), dim3(64 * kWaves), 0, st, a);
    e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(policy_finish_kernel, dim3(1), dim3(1024), 0, st, a);
    return hipGetLastError();
}

}  // namespace cfattn
