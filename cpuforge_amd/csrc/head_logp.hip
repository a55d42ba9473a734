// Log-probabilities of the targets under logits = hn . head^T, and their
// gradient (cfops_lm_head_logprobs of include/cfops.h), over rows of logits:
//   lse = log sum_v exp(x_v),  logp = x_target - lse,
//   d x_v = dlogp ((v == target) - exp(x_v - lse)).
#include <limits.h>

#include "cfattn_common.hpp"
#include "cfops_kernels.hpp"

namespace cfattn {
namespace {

constexpr long kIgnoreIndex = -100;  // crates/core/src/ops/loss.rs:4

// A running maximum and the sum of exp(x - maximum).
struct MaxSum {
    float m, s;
};
__device__ __forceinline__ MaxSum merge(const MaxSum& a, const MaxSum& b) {
    const float m = fmaxf(a.m, b.m);
    // (An empty side has m = -inf and s = 0.)
    const float sa = a.s == 0.0f ? 0.0f : a.s * expf(a.m - m), sb = b.s == 0.0f ? 0.0f : b.s * expf(b.m - m);
    return {m, sa + sb};
}

// The scored rows (targets within the vocabulary) and their targets: idx[0..n) and
// idx[rows..rows + n) in row order, n and the caller's tag at count[0] and
// count[1]; the result's counts; logp and lse of the other rows, 0 where the
// target is ignored and NaN where it is out of range.  One workgroup: 1024
// targets a round, their places from a scan (4096 targets 5.6 us, latency).
__global__ __launch_bounds__(1024) void logp_select_kernel(const int64_t* __restrict__ targets, long rows, long vocab,
                                                           int* __restrict__ idx, int* __restrict__ count, int tag,
                                                           float* __restrict__ logp, float* __restrict__ lse,
                                                           CeMisc* __restrict__ misc) {
    __shared__ int wave_n[16], bad_row;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if (threadIdx.x == 0) bad_row = INT_MAX;
    __syncthreads();
    int n = 0, ignored = 0;
    for (long r0 = 0; r0 < rows; r0 += 1024) {
        const long r = r0 + threadIdx.x;
        const int64_t t = r < rows ? targets[r] : kIgnoreIndex;
        const bool scored = t >= 0 && t < vocab;
        if (r < rows && !scored) {
            ignored += t == kIgnoreIndex;
            if (t != kIgnoreIndex) atomicMin(&bad_row, (int)r);
            if (logp) logp[r] = lse[r] = t == kIgnoreIndex ? 0.0f : __builtin_nanf("");
        }
        const unsigned long long m = __ballot(scored);
        if (lane == 0) wave_n[wave] = __popcll(m);
        __syncthreads();
        int at = n;
        for (int w = 0; w < 16; w++) {
            at += w < wave ? wave_n[w] : 0;
            n += wave_n[w];
        }
        if (scored) {
            at += __popcll(m & ((1ull << lane) - 1));
            idx[at] = (int)r;
            idx[rows + at] = (int)t;
        }
        __syncthreads();
    }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) ignored += __shfl_xor(ignored, o);
    if (lane == 0) wave_n[wave] = ignored;
    __syncthreads();
    if (threadIdx.x == 0) {
        count[0] = n;
        count[1] = tag;
        if (misc) {
            int all = 0;
            for (int w = 0; w < 16; w++) all += wave_n[w];
            *misc = {(int)(rows - all), bad_row, 0.0f};
        }
    }
}

// out[j] = hn[idx[j]], zeros from row n on.
__global__ __launch_bounds__(256) void logp_gather_kernel(const float* __restrict__ hn, const int* __restrict__ idx,
                                                          const int* __restrict__ count, float* __restrict__ out,
                                                          long d) {
    const long j = blockIdx.x;
    const float* x = j < *count ? hn + (long)idx[j] * d : nullptr;
    for (long i = threadIdx.x; i < d; i += 256) out[j * d + i] = x ? x[i] : 0.0f;
}

// dhn[idx[j]] = in[j] for j < n, the other rows zeros.
__global__ __launch_bounds__(256) void logp_scatter_kernel(const float* __restrict__ in, const int* __restrict__ idx,
                                                           const int* __restrict__ count, float* __restrict__ dhn,
                                                           long d) {
    // The place of row blockIdx.x among the ascending idx.
    const int r = blockIdx.x, n = *count;
    int lo = 0, hi = n;
    while (lo < hi) {
        const int mid = (lo + hi) / 2;
        if (idx[mid] < r)
            lo = mid + 1;
        else
            hi = mid;
    }
    const float* x = lo < n && idx[lo] == r ? in + (long)lo * d : nullptr;
    for (long i = threadIdx.x; i < d; i += 256) dhn[r * d + i] = x ? x[i] : 0.0f;
}

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));

// Elements [0, 4) of p, those at or past n zero (and not read).
__device__ __forceinline__ f32x4 load4(const float* __restrict__ p, int n) {
    if (n >= 4) return *reinterpret_cast<const f32x4u*>(p);
    f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int i = 0; i < n; i++) v[i] = p[i];
    return v;
}

constexpr int kFewVocab = 64;  // rows of the head of a workgroup

// Few rows: a wave forms the logits of 16 rows of the head and 16 TT tokens on the f32
// MFMA, straight from memory (v_mfma_f32_16x16x4_f32: lane l has A[l % 16][l / 16],
// B[l / 16][l % 16] and C[4 (l / 16) + i][l % 16]; four consecutive k a lane, one
// per MFMA and sum), and a workgroup the maximum and sum of exp of its 64. Bound by
// reading the head once: 1 x 576 x 49152 (113 MB) 21 us, 5.4 TB/s.
template <int TT>
__global__ __launch_bounds__(256) void logp_few_kernel(const float* __restrict__ hn, const float* __restrict__ head,
                                                       const int64_t* __restrict__ targets, int t, int d, int vocab,
                                                       MaxSum* __restrict__ stats, float* __restrict__ xt) {
    __shared__ MaxSum red[4][16 * TT];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l16 = lane & 15, kq = (lane >> 4) * 4;
    const int v0 = blockIdx.x * kFewVocab + wave * 16;
    const float* w = head + (long)min(v0 + l16, vocab - 1) * d + kq;
    const float* h[TT];
    f32x4 acc[TT][4] = {};
#pragma unroll
    for (int i = 0; i < TT; i++) h[i] = hn + (long)min(16 * i + l16, t - 1) * d + kq;
    auto add = [&](const f32x4& a, const f32x4 (&b)[TT]) {
#pragma unroll
        for (int i = 0; i < TT; i++)
#pragma unroll
            for (int q = 0; q < 4; q++)
                acc[i][q] = __builtin_amdgcn_mfma_f32_16x16x4f32(a[q], b[i][q], acc[i][q], 0, 0, 0);
    };
    constexpr int U = 4;  // runs of 16 k whose loads are in flight together
    const int whole = d / 16;
    int c = 0;
    for (; c + U <= whole; c += U) {
        f32x4 a[U], b[U][TT];
#pragma unroll
        for (int u = 0; u < U; u++) a[u] = load4(w + (c + u) * 16, 4);
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
            for (int i = 0; i < TT; i++) b[u][i] = load4(h[i] + (c + u) * 16, 4);
#pragma unroll
        for (int u = 0; u < U; u++) add(a[u], b[u]);
    }
    for (; c * 16 < d; c++) {
        const int n = max(0, min(4, d - c * 16 - kq));
        f32x4 b[TT];
#pragma unroll
        for (int i = 0; i < TT; i++) b[i] = load4(h[i] + c * 16, n);
        add(load4(w + c * 16, n), b);
    }
#pragma unroll
    for (int i = 0; i < TT; i++) {
        const int token = 16 * i + l16;
        const f32x4 x = (acc[i][0] + acc[i][1]) + (acc[i][2] + acc[i][3]);
        const long target = token < t ? targets[token] - v0 - kq : -1;
        MaxSum s{-INFINITY, 0.0f};
#pragma unroll
        for (int q = 0; q < 4; q++) {
            if (v0 + kq + q >= vocab) continue;
            s = merge(s, {x[q], 1.0f});
            if (q == target) xt[token] = x[q];
        }
        s = merge(s, {__shfl_xor(s.m, 16), __shfl_xor(s.s, 16)});
        s = merge(s, {__shfl_xor(s.m, 32), __shfl_xor(s.s, 32)});
        if (lane < 16) red[wave][token] = s;
    }
    __syncthreads();
    if (threadIdx.x < (unsigned)t) {
        MaxSum s = red[0][threadIdx.x];
        for (int k = 1; k < 4; k++) s = merge(s, red[k][threadIdx.x]);
        stats[(long)threadIdx.x * gridDim.x + blockIdx.x] = s;
    }
}

// lse, logp and the result of few rows, a wave to a row, one workgroup: 5.4 us for one
// row of 49152, latency.
__global__ __launch_bounds__(1024) void logp_few_finish_kernel(const MaxSum* __restrict__ stats, int parts,
                                                               const float* __restrict__ xt,
                                                               const int64_t* __restrict__ targets, int t, long vocab,
                                                               float* __restrict__ logp, float* __restrict__ lse,
                                                               CeMisc* __restrict__ misc) {
    __shared__ float row[kLogpFew];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int r = wave; r < t; r += 16) {
        const int64_t target = targets[r];
        float l = target == kIgnoreIndex ? 0.0f : __builtin_nanf(""), lp = l;
        if (target >= 0 && target < vocab) {
            MaxSum s{-INFINITY, 0.0f};
            for (int p = lane; p < parts; p += 64) s = merge(s, stats[(long)r * parts + p]);
#pragma unroll
            for (int o = 32; o >= 1; o >>= 1) s = merge(s, {__shfl_xor(s.m, o), __shfl_xor(s.s, o)});
            // (In f64: logp of a likely target is far below an lse, whose rounding it would have.)
            const double sum = (double)s.m + log((double)s.s);
            l = (float)sum;
            lp = (float)((double)xt[r] - sum);
        }
        if (lane == 0) {
            lse[r] = l;
            logp[r] = row[r] = lp;
        }
    }
    __syncthreads();
    if (threadIdx.x) return;
    int n = 0, bad = INT_MAX;
    double sum = 0.0;
    for (int r = 0; r < t; r++) {
        const int64_t target = targets[r];
        if (target == kIgnoreIndex) continue;
        n++;
        sum -= (double)row[r];
        if (bad == INT_MAX && (target < 0 || target >= vocab)) bad = r;
    }
    *misc = {n, bad, n > 0 ? (float)(sum / n) : 0.0f};
}

// dlogits over the logits of scored rows [j0, ..); zeros from row n on.  lse serves the
// exponentials' range alone: as an f32 it is off by 2^-24 of itself, and so would be every
// probability, where 1 - P of a likely token is much less.  Their sum, formed again, sets
// that right: P = exp(x - lse) / sum, and at the target 1 - P = -expm1(x - lse - log(sum)).
// (The whole backward of 64 rows of 2048 x 128256 665 us, where one pass of loads that
// waited for each other took 685.)
__global__ __launch_bounds__(512) void logp_grad_rows_kernel(float* __restrict__ logits,
                                                             const int64_t* __restrict__ targets,
                                                             const int* __restrict__ idx,
                                                             const int* __restrict__ count,
                                                             const float* __restrict__ lse,
                                                             const float* __restrict__ dlogp, int j0, long vocab) {
    __shared__ float red[8];
    const int j = j0 + blockIdx.x;
    const bool scored = j < *count;
    float* x = logits + (long)blockIdx.x * vocab;
    if (!scored) {
        for (long i = threadIdx.x; i < vocab; i += 512) x[i] = 0.0f;
        return;
    }
    const long r = idx[j], t = targets[r];
    const float g = dlogp[r], l = lse[r];
    float s = 0.0f;
#pragma unroll 4
    for (long i = threadIdx.x; i < vocab; i += 512) s += expf(x[i] - l);
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) s += __shfl_xor(s, o);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    s = 0.0f;
#pragma unroll
    for (int w = 0; w < 8; w++) s += red[w];
    const float f = -g / s, more = logf(s);
#pragma unroll 4
    for (long i = threadIdx.x; i < vocab; i += 512)
        x[i] = i == t ? -g * expm1f((x[i] - l) - more) : f * expf(x[i] - l);
}

// The mean of sign logp over the scored rows, summed in f64 in a fixed order by one
// workgroup: 4096 rows 5.2 us.
__global__ __launch_bounds__(1024) void logp_finish_kernel(const int64_t* __restrict__ targets,
                                                           const float* __restrict__ logp, double sign, long rows,
                                                           CeMisc* __restrict__ m) {
    __shared__ double red[16];
    double s = 0.0;
#pragma unroll 4
    for (long r = threadIdx.x; r < rows; r += 1024) {
        const float x = logp[r];
        s += targets[r] != kIgnoreIndex ? sign * (double)x : 0.0;
    }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) s += __shfl_xor(s, o);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        double tot = 0.0;
        for (int i = 0; i < 16; i++) tot += red[i];
        const int n = m->n_valid;
        m->loss = n > 0 ? (float)(tot / (double)n) : 0.0f;
    }
}

}  // namespace

hipError_t launch_logp_select(const int64_t* targets, size_t rows, size_t vocab, int* idx, int* count, int tag,
                              float* logp, float* lse, void* misc, hipStream_t st) {
    hipLaunchKernelGGL(logp_select_kernel, dim3(1), dim3(1024), 0, st, targets, (long)rows, (long)vocab, idx, count,
                       tag, logp, lse, static_cast<CeMisc*>(misc));
    return hipGetLastError();
}
hipError_t launch_logp_gather(const float* hn, const int* idx, const int* count, float* out, size_t rows, size_t d,
                              hipStream_t st) {
    hipLaunchKernelGGL(logp_gather_kernel, dim3((unsigned)rows), dim3(256), 0, st, hn, idx, count, out, (long)d);
    return hipGetLastError();
}
hipError_t launch_logp_scatter(const float* in, const int* idx, const int* count, float* dhn, size_t rows, size_t d,
                               hipStream_t st) {
    hipLaunchKernelGGL(logp_scatter_kernel, dim3((unsigned)rows), dim3(256), 0, st, in, idx, count, dhn, (long)d);
    return hipGetLastError();
}
size_t logp_few_bytes(size_t t, size_t vocab) {
    return kLogpFew * sizeof(float) + t * ((vocab + kFewVocab - 1) / kFewVocab) * sizeof(MaxSum);
}
hipError_t launch_logp_few(const float* hn, const float* head, const int64_t* targets, size_t t, size_t d, size_t vocab,
                           float* logp, float* lse, void* misc, void* scratch, hipStream_t st) {
    float* xt = static_cast<float*>(scratch);
    MaxSum* stats = reinterpret_cast<MaxSum*>(xt + kLogpFew);
    const unsigned parts = (unsigned)((vocab + kFewVocab - 1) / kFewVocab);
    static_assert(kLogpFew == 32, "the tokens of a wave");
    const auto kernel = t <= 16 ? logp_few_kernel<1> : logp_few_kernel<2>;
    hipLaunchKernelGGL(kernel, dim3(parts), dim3(256), 0, st, hn, head, targets, (int)t, (int)d, (int)vocab, stats, xt);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(logp_few_finish_kernel, dim3(1), dim3(1024), 0, st, stats, (int)parts, xt, targets, (int)t,
                       (long)vocab, logp, lse, static_cast<CeMisc*>(misc));
    return hipGetLastError();
}
hipError_t launch_logp_grad_rows(float* logits, const int64_t* targets, const int* idx, const int* count,
                                 const float* lse, const float* dlogp, size_t j0, size_t nrows, size_t vocab,
                                 hipStream_t st) {
    hipLaunchKernelGGL(logp_grad_rows_kernel, dim3((unsigned)nrows), dim3(512), 0, st, logits, targets, idx, count,
                       lse, dlogp, (int)j0, (long)vocab);
    return hipGetLastError();
}
hipError_t launch_logp_finish(const int64_t* targets, const float* logp, double sign, size_t rows, void* misc,
                              hipStream_t st) {
    hipLaunchKernelGGL(logp_finish_kernel, dim3(1), dim3(1024), 0, st, targets, logp, sign, (long)rows,
                       static_cast<CeMisc*>(misc));
    return hipGetLastError();
}

}  // namespace cfattn
