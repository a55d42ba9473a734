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

#include <algorithm>

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
// What a wave's lanes wrote to its LDS is there for the others.
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}
__device__ __forceinline__ bool finite(float x) { return fabsf(x) < INFINITY; }

// A row's entries by rising token, a wave to a row: ids, z and e [t][k] (count of them), their
// exponentials below the largest's; the row's L, p_rest (negative: no rest) and p / e; target is a
// token of the row, kIgnoreIndex without entries, -1 where the row is bad: a token out of the
// vocabulary or named twice, or a value of the teacher's that is NaN or +inf.  (An entry whose id
// is kIgnoreIndex or whose logit is -inf is not there.)
// Places are counts of smaller tokens: 4096 x 64 entries 10 us.
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
    wave_sync();
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
        bad |= !(l < INFINITY);  // (-inf is below the entries' own.)
        whole = fmax(own, (double)l);
        p_rest = -expm1(own - whole);
    }
    const bool any_bad = __any(bad);
    if (lane) return;
    g.count[r] = any_bad ? 0 : n;
    g.row[r] = {whole, p_rest, exp(own - whole) / sum};
    g.target[r] = any_bad ? -1 : n == 0 ? kIgnoreIndex : least;
    if (r == 0 && g.tag_at) *g.tag_at = g.tag;
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
__device__ __forceinline__ double pow2(double x) {
    return x > -120.0 ? (double)__builtin_amdgcn_exp2f((float)x) : exp2(x);
}

// Rows whose product kept exp2(y - m) of 128 logits each (y in units of log2, m the largest):
// a wave to a row.  An entry whose exponential is too small, and
// a rest of 128 that is, are formed again from hidden state and head.  Where the entries hold
// all but little of such 128, the rest of them is summed, not left over.
//
// For the gradients an entry's exponential becomes what the product has to find there for its
// own gradient, dl / (a factor), so that the product adds it up with the others'; where that is
// much larger than its 128's largest (a near 0, a student that holds the token for unlikely), or
// the rest is far below the entry, it becomes 0 and the entry stays in ids and dl (count of them).
// (A sure student's a q would cancel in the entries: a is -p_rest / q_rest then.)
// 3686 rows of 64 entries, 49152 tokens: 45 us, a chain of a few loads, values of a row far apart: what
// a row needs is loaded at once, the entries' to LDS (one by one where it was used 55).
struct EntryLds {
    int v;
    float kept;
    float2 stat;
};
constexpr int kStats = 16;  // of a lane in registers
// (Two workgroups to a CU: with 129 registers, which leave one, 57 us.)
__global__ __launch_bounds__(512, 4) void distill_kept_kernel(const DistillKept g) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int j = blockIdx.x * (blockDim.x >> 6) + wave;
    const int scored = g.scored[1] == g.tag ? min(g.scored[0] - g.j0, g.chunk) : 0;
    if (j >= scored) return;  // (no barrier follows: each wave has its own part of LDS)
    const long r = g.idx[g.j0 + j];
    const int n = g.count[r];
    EntryLds* mine = reinterpret_cast<EntryLds*>(lds) + wave * g.k;
    auto kept = [&](int v) -> float& {
        char* p = g.keep + ((long)(j / 32) * g.v16 + v / 32 * 2) * 2048 + v % 32 / 8 * 1024 +
                  ((v % 8 / 4) * 32 + j % 32) * 16;
        return reinterpret_cast<float*>(p)[v % 4];
    };
    auto stat = [&](int part) { return g.stats[(long)part * g.ld + j]; };
    float2 st[kStats];
#pragma unroll
    for (int i = 0; i < kStats; i++)
        st[i] = lane + 64 * i < g.parts ? stat(lane + 64 * i) : make_float2(-INFINITY, 0.0f);
    for (int k = lane; k < n; k += 64) {
        const int v = g.ids[r * g.k + k];
        mine[k] = {v, kept(v), stat(v / 128)};
    }
    wave_sync();
    const TeacherRow row = g.row[r];
    bool with_rest = row.p_rest > 0.0;
    auto has_entry = [&](int part) {
        int lo = 0, hi = n;  // the first that is not below the 128
        while (lo < hi) {
            const int mid = (lo + hi) / 2;
            if (mine[mid].v < part * 128)
                lo = mid + 1;
            else
                hi = mid;
        }
        return lo < n && mine[lo].v < part * 128 + 128;
    };
    // A logit in units of log2, by the whole wave.
    auto logit = [&](int v) {
        const float *h = g.hn + r * g.d, *w = g.head + (long)v * g.d;
        double s = 0.0;
        for (int i = lane; i < g.d; i += 64) s += (double)(h[i] * g.mul) * (double)w[i];
        return sum_wave(s) * (double)kLog2e;
    };
    // (Every lane's statistics, those past the registers' from memory again.)
    auto each = [&](auto f) {
#pragma unroll
        for (int i = 0; i < kStats; i++)
            if (lane + 64 * i < g.parts) f(lane + 64 * i, st[i]);
        for (int p = lane + 64 * kStats; p < g.parts; p += 64) f(p, stat(p));
    };
    float m = -INFINITY, m_rest = -INFINITY;
    each([&](int p, const float2& s) {
        m = fmaxf(m, s.x);
        if (with_rest && !has_entry(p)) m_rest = fmaxf(m_rest, s.x);
    });
    m = max_wave(m);
    m_rest = max_wave(m_rest);
    const double top = (double)m;
    double total = 0.0, rest = 0.0;  // in units of 2^top
    each([&](int p, const float2& s) {
        total += (double)(s.y * __builtin_amdgcn_exp2f(s.x - m));
        if (with_rest && !has_entry(p)) rest += (double)(s.y * __builtin_amdgcn_exp2f(s.x - m_rest));
    });
    total = sum_wave(total);
    // (A row that is not finite has a loss of NaN, whatever its rest.)
    with_rest = with_rest && total < INFINITY;
    constexpr float kLost = 0x1p-100f;  // of a kept exponential
    // The kept values of the 128 that entry `at` is the first of, four to each of 32 lanes, without
    // those of entries; the first entry behind them.
    const int v4 = lane % 32 * 4;
    auto others = [&](int at, float (&x4)[4]) {
        const int part = mine[at].v / 128, v0 = part * 128 + v4;
#pragma unroll
        for (int i = 0; i < 4; i++) x4[i] = lane < 32 && v0 + i < g.vocab ? kept(v0 + i) : 0.0f;
        int last = at;
        for (; last < n && mine[last].v / 128 == part; last++) {
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (mine[last].v == v0 + i) x4[i] = 0.0f;
        }
        return last;
    };
    auto is_first = [&](int k) { return k < n && (k == 0 || mine[k - 1].v / 128 != mine[k].v / 128); };
    // The others of the 128 that entry `at` is the first of, as add(y, s): s 2^y of them; from what was
    // kept, or, where too little of it was to be `enough`, each formed again.
    auto add_others = [&](int at, bool enough, auto add) {
        const int part = mine[at].v / 128;
        float x4[4];
        const int last = others(at, x4);
        const double sum = sum_wave((double)x4[0] + (double)x4[1] + (double)x4[2] + (double)x4[3]);
        if (enough || sum > 128.0 * kLost * 0x1p18) return add((double)mine[at].stat.x, sum);
        const int end = min(part * 128 + 128, g.vocab);
        for (int v = part * 128, i = at; v < end; v++) {
            if (i < last && mine[i].v == v)
                i++;
            else
                add(logit(v), 1.0);
        }
    };
    double low = 0.0;  // log2 of the rest's sum in units of 2^top
    if (with_rest) {
        rest = sum_wave(rest);
        if (rest > 0.0) rest *= exp2((double)m_rest - top);
        // The 128s that have entries, by their first: what is left of their sums, then, where that
        // is not exact enough beside what the rest is at least, the sum of the others.  (f32 sums of
        // up to 128 and kept values are off by less than 2^-19 of the sum: so much may be left of
        // entries alone, and counts for nothing in the least.)
        double left = 0.0;
        auto left_of = [&](int k, double& size, bool least) {
            const int part = mine[k].v / 128;
            const float2 s = mine[k].stat;
            double x = (double)s.y;
            for (int i = k; i < n && mine[i].v / 128 == part; i++) x -= (double)mine[i].kept;
            const double scale = pow2((double)s.x - top);
            size = (double)s.y * scale;
            return fmax(least ? x - 0x1p-19 * (double)s.y : x, 0.0) * scale;
        };
        for (int k = lane; k < n; k += 64) {
            double size;
            if (is_first(k)) left += left_of(k, size, true);
        }
        const double least = rest + sum_wave(left);
        left = 0.0;
        for (int k0 = 0; k0 < n; k0 += 64) {
            const int k = k0 + lane;
            const bool first = is_first(k);
            double size = 0.0, x = 0.0;
            if (first) x = left_of(k, size, false);
            const bool again = first && !(size * 0x1p-22 <= least * 0x1p-18);
            if (!again) left += x;
            for (unsigned long long todo = __ballot(again); todo; todo &= todo - 1) {
                const int at = k0 + __ffsll(todo) - 1;
                double exact = 0.0;
                add_others(at, 128.0 * kLost * exp2((double)mine[at].stat.x - top) <= least * 0x1p-18,
                           [&](double y, double s) { exact += s * exp2(y - top); });
                if (lane == 0) left += exact;
            }
        }
        rest += sum_wave(left);
        low = log2(rest);
        // Where f64 holds it no more, all of it again in units of its own largest.
        if (rest < 0x1p-900) {
            double unit = -INFINITY;
            rest = 0.0;
            auto add = [&](double y, double s) {
                if (y > unit) rest *= exp2(unit - y), unit = y;
                rest += s * exp2(y - unit);
            };
            if (m_rest > -INFINITY) {
                double parts = 0.0;
                for (int p = lane; p < g.parts; p += 64) {
                    const float2 s = stat(p);
                    if (!has_entry(p)) parts += (double)(s.y * __builtin_amdgcn_exp2f(s.x - m_rest));
                }
                add((double)m_rest, sum_wave(parts));
            }
            for (int k0 = 0; k0 < n; k0 += 64)
                for (unsigned long long todo = __ballot(is_first(k0 + lane)); todo; todo &= todo - 1)
                    add_others(k0 + __ffsll(todo) - 1, false, add);
            low = unit - top + log2(rest);
        }
    }
    const double log_total = log(total), unit = 1.0 / (double)kLog2e;
    const Rest r_(row.p_rest, low * M_LN2 - log_total);
    // Where the rest is so small that f32 holds neither a nor all of its exponentials, a is 2^-lift
    // of itself and every factor 2^lift (a part's largest is up to 2^10 above the rest, or its entries
    // stay in the list and its factor follows below).
    const double above = with_rest ? log2(total) - low : 0.0, lift = above > 60.0 ? floor(above) : 0.0;
    const float a = lift > 0.0 ? (float)(exp2(-lift) - row.p_rest * exp2(above - lift))
                               : (float)(1.0 - fmin(r_.ratio, 1e30));
    auto lifted = [&](float x) { return (float)(exp2(fmin((double)x - top + lift, 120.0)) / total); };
    if (g.dl && lift > 0.0)
        for (int p = lane; p < g.parts; p += 64) g.factor[(long)p * g.ld + j] = lifted(stat(p).x);
    double terms = 0.0;
    int stay = 0;
    for (int k0 = 0; k0 < n; k0 += 64) {
        const int k = k0 + lane;
        const bool live = k < n;
        const EntryLds en = live ? mine[k] : EntryLds{0, 1.0f, make_float2(0.0f, 0.0f)};
        const int v = en.v;
        const float e = en.kept;
        const double up = live ? (double)en.stat.x - top : 0.0;
        double y = log2((double)e) + up, q = (double)e * pow2(up) / total;
        for (unsigned long long todo = __ballot(live && e < kLost); todo; todo &= todo - 1) {
            const int at = __ffsll(todo) - 1;
            const double x = logit(mine[k0 + at].v) - top;
            if (lane == at) y = x, q = exp2(x) / total;
        }
        double dl = 0.0;
        if (live)
            terms += entry_loss(row, g.z[r * g.k + k], g.e[r * g.k + k], g.inv_t, q, y * unit - log_total, dl);
        if (!g.dl) continue;
        const bool far = with_rest && up - 10.0 > low;
        const float factor = !live ? 1.0f : lift > 0.0 ? lifted(en.stat.x) : g.factor[(long)(v / 128) * g.ld + j];
        const float in = live ? (float)dl / (a * factor) : 0.0f;
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
    // that this shows in a q, the others of its 128 are scaled up, to at most 1.
    for (int k0 = 0; g.dl && with_rest && k0 < n; k0 += 64) {
        const int k = k0 + lane;
        const bool far = is_first(k) && (double)mine[k].stat.x - top - 10.0 > low;
        for (unsigned long long todo = __ballot(far); todo; todo &= todo - 1) {
            const int at = k0 + __ffsll(todo) - 1, part = mine[at].v / 128;
            float x4[4];
            const int last = others(at, x4);
            const float most = max_wave(fmaxf(fmaxf(x4[0], x4[1]), fmaxf(x4[2], x4[3])));
            if (lift > 0.0) {
                // (By a factor of their own, and formed again where f32 holds too little of them.)
                double y4[4], y_most = -INFINITY;
                if (most >= 128.0f * kLost * 0x1p18f) {
#pragma unroll
                    for (int i = 0; i < 4; i++) y4[i] = log2((double)x4[i]) + (double)mine[at].stat.x - top;
                } else {
#pragma unroll
                    for (int i = 0; i < 4; i++) y4[i] = -INFINITY;
                    const int end = min(part * 128 + 128, g.vocab);
                    for (int v = part * 128, e = at; v < end; v++) {
                        if (e < last && mine[e].v == v) {
                            e++;
                            continue;
                        }
                        const double y = logit(v) - top;
#pragma unroll
                        for (int i = 0; i < 4; i++)
                            if (lane < 32 && v4 + i == v % 128) y4[i] = y;
                    }
                }
#pragma unroll
                for (int i = 0; i < 4; i++) y_most = fmax(y_most, y4[i]);
#pragma unroll
                for (int o = 32; o >= 1; o >>= 1) y_most = fmax(y_most, __shfl_xor(y_most, o));
                if (!(y_most > -INFINITY)) continue;
                y_most = floor(y_most) + 1.0;
#pragma unroll
                for (int i = 0; i < 4; i++)
                    if (lane < 32 && part * 128 + v4 + i < g.vocab)
                        kept(part * 128 + v4 + i) = (float)exp2(y4[i] - y_most);
                if (lane == 0) g.factor[(long)part * g.ld + j] = (float)(exp2(y_most + lift) / total);
                continue;
            }
            const int up = min(max(126 - (int)(__builtin_bit_cast(uint32_t, most) >> 23), 0), 126);
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

// Rows of products hn . head in memory (x times mul), kSlice of them to a workgroup, in two
// launches: the largest and the sum of exponentials of each slice's tokens that are no entries (so
// the rest is a sum of its own), and the entries' logits; then the loss, where it is wanted, and
// with GRAD the products become the logits' gradients (zeros in rows that are not scored and from t
// on).  24 rows of 49152, 16 of them scored, with their gradients 12.5 us (a row to a workgroup 27).
constexpr int kSlice = 4096, kSliceThreads = 512, kPer = kSlice / kSliceThreads;

// Whether value i of a slice is an entry's, for the values of this thread.
__device__ __forceinline__ void mark_entries(unsigned (&bits)[kSlice / 32], const int* ids, int n, long v0) {
    if (threadIdx.x < kSlice / 32) bits[threadIdx.x] = 0;
    __syncthreads();
    for (int k = threadIdx.x; k < n; k += kSliceThreads) {
        const long at = ids[k] - v0;
        if (at >= 0 && at < kSlice) atomicOr(&bits[at / 32], 1u << at % 32);
    }
    __syncthreads();
}

__global__ __launch_bounds__(kSliceThreads) void distill_slices_kernel(const float* __restrict__ logits,
                                                                       const DistillRows g) {
    __shared__ unsigned bits[kSlice / 32];
    __shared__ float red[2][8];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, j = blockIdx.y;
    const long r = g.j0 + j, v0 = (long)blockIdx.x * kSlice;
    if (r >= g.t || g.target[r] < 0) return;
    const int n = g.count[r];
    const int* ids = g.ids + r * g.k;
    const float* x = logits + j * g.vocab;
    mark_entries(bits, ids, n, v0);
    float v[kPer], m = -INFINITY;
#pragma unroll
    for (int i = 0; i < kPer; i++) {
        const int at = threadIdx.x + i * kSliceThreads;
        const bool in = v0 + at < g.vocab && !(bits[at / 32] >> at % 32 & 1);
        v[i] = in ? g.mul * x[v0 + at] : -INFINITY;
        m = fmaxf(m, v[i]);
    }
    for (int k = threadIdx.x; k < n; k += kSliceThreads) {
        const long at = ids[k] - v0;
        if (at >= 0 && at < kSlice) g.xs[(long)j * g.k + k] = g.mul * x[ids[k]];
    }
    m = max_wave(m);
    if (lane == 0) red[0][wave] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 8; w++) m = fmaxf(m, red[0][w]);
    float s = 0.0f;
    // (A slice of entries alone, or of nothing but NaN, has no largest.)
    const float base = m > -INFINITY ? m : 0.0f;
#pragma unroll
    for (int i = 0; i < kPer; i++) s += expf(v[i] - base);
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) s += __shfl_xor(s, o);
    if (lane == 0) red[1][wave] = s;
    __syncthreads();
    if (threadIdx.x) return;
    s = 0.0f;
    for (int w = 0; w < 8; w++) s += red[1][w];
    g.slices[(long)j * gridDim.x + blockIdx.x] = make_float2(m, s);
}

template <bool GRAD>
__global__ __launch_bounds__(kSliceThreads) void distill_logits_kernel(float* __restrict__ logits, int slices,
                                                                       const DistillRows g) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, j = blockIdx.y;
    const long v0 = (long)blockIdx.x * kSlice;
    float* x = logits + j * g.vocab;
    const long r = g.j0 + j;
    const bool scored = r < g.t && g.target[r] >= 0;
    if (!scored) {
        if (g.loss && r < g.t && blockIdx.x == 0 && threadIdx.x == 0)
            g.loss[r] = g.target[r] == kIgnoreIndex ? 0.0f : __builtin_nanf("");
        if (GRAD)
            for (long v = v0 + threadIdx.x; v < min(v0 + kSlice, g.vocab); v += kSliceThreads) x[v] = 0.0f;
        return;
    }
    const int n = g.count[r];
    const int* ids = g.ids + r * g.k;
    const float* xs = g.xs + (long)j * g.k;
    // (Every wave for itself: a few slices and entries a lane.)
    float m = -INFINITY;
    for (int p = lane; p < slices; p += 64) m = fmaxf(m, g.slices[(long)j * slices + p].x);
    m = max_wave(m);
    double rest = 0.0;
    for (int p = lane; p < slices; p += 64) {
        const float2 s = g.slices[(long)j * slices + p];
        rest += s.y == 0.0f ? 0.0 : (double)s.y * exp((double)s.x - (double)m);
    }
    rest = sum_wave(rest);
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
    if (g.loss && blockIdx.x == 0 && wave == 0) {
        double terms = 0.0, dl;
        for (int k = lane; k < n; k += 64) terms += entry(k, dl);
        terms = sum_wave(terms);
        if (lane == 0) g.loss[r] = (float)(r_.loss + terms);
    }
    if (!GRAD) return;
    // a q of the others by their own largest: a q of a sure student's is not small where q is (and
    // p_rest / q_rest may be past what f64 holds).
    const float f = (float)(exp(shift) / total - (row.p_rest > 0.0 ? row.p_rest / rest : 0.0));
    const float base = m > -INFINITY ? m : 0.0f;
#pragma unroll
    for (int i = 0; i < kPer; i++) {
        const long v = v0 + threadIdx.x + i * kSliceThreads;
        if (v < g.vocab) x[v] = f * expf(g.mul * x[v] - base);
    }
    __syncthreads();
    for (int k = threadIdx.x; k < n; k += kSliceThreads) {
        const long at = ids[k] - v0;
        if (at < 0 || at >= kSlice) continue;
        double dl;
        entry(k, dl);
        x[ids[k]] = (float)dl;
    }
}

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
// Elements [0, 4) of p, those at or past n zero (and not read).
__device__ __forceinline__ f32x4 load4(const float* __restrict__ p, long n) {
    if (n >= 4) return *reinterpret_cast<const f32x4u*>(p);
    f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int i = 0; i < n; i++) v[i] = p[i];
    return v;
}

// part[split][row][d] = rows' gradients . head over a split of the vocabulary, for up to 16 TT rows on
// the f32 MFMA: a workgroup 64 columns of the head, a wave 16 of its tokens at a time (v_mfma_f32_16x16x4:
// lane l has A[l % 16][l / 16] and B[l / 16][l % 16]; product s of 16 tokens takes 4 (l / 16) + s, product
// q of 64 columns 4 (l % 16) + q, so that every load is of four values side by side).
// Bound by reading the head: 9 rows of 49152 x 576 (113 MB) 23 us, 4.9 TB/s; 24 rows 37, with as many bytes
// of gradients again from the caches (split into bf16 pieces, by launch_gemm_f32, 55).
template <int TT>
__global__ __launch_bounds__(256) void distill_rows_head_kernel(const float* __restrict__ grads, long vocab, int t,
                                                                const float* __restrict__ head, int d, int blocks,
                                                                int splits, float* __restrict__ part) {
    __shared__ f32x4 sum[TT * 16 * 16];  // [row][columns of a lane]
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l16 = lane & 15, kq = lane >> 4;
    // The columns of a split follow one another on one XCD, whose L2 holds its gradients.
    const int local = blockIdx.x / 8, split = local / blocks * 8 + blockIdx.x % 8, c0 = local % blocks * 64;
    if (split >= splits) return;
    const int c = c0 + 4 * l16;
    const long chunks = (vocab + 15) / 16, end = chunks * (split + 1) / splits;
    const float* g[TT];
#pragma unroll
    for (int i = 0; i < TT; i++) g[i] = grads + min(16 * i + l16, t - 1) * vocab;
    f32x4 acc[TT][4] = {};
    for (long k = chunks * split / splits + wave; k < end; k += 4) {
        const long v = k * 16 + 4 * kq, live = vocab - v;
        f32x4 a[TT], b[4];
#pragma unroll
        for (int i = 0; i < TT; i++) a[i] = load4(g[i] + v, live);
#pragma unroll
        for (int s = 0; s < 4; s++) b[s] = load4(head + (v + s) * d + c, s < live ? d - c : 0);
#pragma unroll
        for (int s = 0; s < 4; s++)
#pragma unroll
            for (int i = 0; i < TT; i++)
#pragma unroll
                for (int q = 0; q < 4; q++)
                    acc[i][q] = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i][s], b[s][q], acc[i][q], 0, 0, 0);
    }
    // Row 16 i + 4 kq + e and column 4 l16 + q of the result are in acc[i][q][e]; wave after wave.
    for (int w = 0; w < 4; w++) {
        if (wave == w)
#pragma unroll
            for (int i = 0; i < TT; i++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    f32x4& to = sum[(16 * i + 4 * kq + e) * 16 + l16];
                    const f32x4 x = {acc[i][0][e], acc[i][1][e], acc[i][2][e], acc[i][3][e]};
                    to = w ? to + x : x;
                }
        __syncthreads();
    }
    for (int at = threadIdx.x; at < t * 64; at += 256) {
        const int row = at / 64, col = at % 64;
        if (c0 + col < d) part[((long)split * t + row) * d + c0 + col] = sum[row * 16 + col / 4][col % 4];
    }
}

// Few rows' mean and counts, by one wave.
__global__ __launch_bounds__(64) void distill_finish_kernel(const int64_t* __restrict__ target,
                                                            const float* __restrict__ loss, int t,
                                                            CeMisc* __restrict__ m) {
    double s = 0.0;
    int n = 0, bad = INT_MAX;
    for (int r = threadIdx.x; r < t; r += 64) {
        if (target[r] == kIgnoreIndex) continue;
        n++;
        if (target[r] < 0) bad = min(bad, r);
        s += (double)loss[r];
    }
    s = sum_wave(s);
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) n += __shfl_xor(n, o), bad = min(bad, __shfl_xor(bad, o));
    if (threadIdx.x == 0) *m = {n, bad, n > 0 ? (float)(s / (double)n) : 0.0f};
}

// out[r] = mul dloss[r] hn[r] of scored rows, zeros of others and from t on; NaN where what was kept
// is another forward's.
__global__ __launch_bounds__(256) void distill_scaled_kernel(const float* __restrict__ hn, float mul,
                                                             const float* __restrict__ dloss, const DistillScored g,
                                                             float* __restrict__ out, long d) {
    const int r = blockIdx.x;
    const bool known = !g.tag_at || *g.tag_at == g.tag;
    const bool scored = known && r < g.t && g.target[r] >= 0;
    const float f = scored ? mul * dloss[r] : 0.0f, none = known ? 0.0f : __builtin_nanf("");
    for (long i = threadIdx.x; i < d; i += 256) out[r * d + i] = scored ? f * hn[r * d + i] : none;
}

// dhn of rows r, [j0, j0 + n), = mul dloss (the sum of its parts), 64 columns to a workgroup, every
// fourth split to a wave; zeros of rows that are not scored, NaN where what was kept is another
// forward's.
__global__ __launch_bounds__(256) void distill_rows_sum_kernel(const float* __restrict__ part, int splits, int j0,
                                                               int n, int d, float mul, const float* __restrict__ dloss,
                                                               const DistillScored g, float* __restrict__ dhn) {
    __shared__ float red[4][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, j = blockIdx.y, r = j0 + j;
    const int c = blockIdx.x * 64 + lane;
    const bool known = !g.tag_at || *g.tag_at == g.tag;
    const bool scored = known && g.target[r] >= 0;
    float s = 0.0f;
    if (scored && c < d)
#pragma unroll 8
        for (int p = wave; p < splits; p += 4) s += part[((long)p * n + j) * d + c];
    red[wave][lane] = s;
    __syncthreads();
    if (wave || c >= d) return;
    const float all = (red[0][lane] + red[1][lane]) + (red[2][lane] + red[3][lane]);
    dhn[(long)r * d + c] = !known ? __builtin_nanf("") : scored ? mul * dloss[r] * all : 0.0f;
}

}  // namespace

hipError_t launch_distill_entries(const DistillEntries& g, hipStream_t st) {
    hipLaunchKernelGGL(distill_entries_kernel, dim3((unsigned)((g.t + 3) / 4)), dim3(256), 4 * g.k * sizeof(int), st,
                       g);
    return hipGetLastError();
}
hipError_t launch_distill_kept(const DistillKept& g, hipStream_t st) {
    const int waves = g.k <= 256 ? 8 : 2;  // (32 KiB of LDS)
    hipLaunchKernelGGL(distill_kept_kernel, dim3((unsigned)((g.chunk + waves - 1) / waves)), dim3(64 * waves),
                       waves * g.k * sizeof(EntryLds), st, g);
    return hipGetLastError();
}
size_t distill_slices(size_t vocab) { return (vocab + kSlice - 1) / kSlice; }
hipError_t launch_distill_logits(float* logits, size_t nrows, bool grad, const DistillRows& g, hipStream_t st) {
    const unsigned slices = (unsigned)distill_slices((size_t)g.vocab);
    hipLaunchKernelGGL(distill_slices_kernel, dim3(slices, (unsigned)nrows), dim3(kSliceThreads), 0, st, logits, g);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((grad ? distill_logits_kernel<true> : distill_logits_kernel<false>),
                       dim3(grad ? slices : 1, (unsigned)nrows), dim3(kSliceThreads), 0, st, logits, (int)slices, g);
    return hipGetLastError();
}

// Splits of the product: two workgroups to a CU (us with four, of 9 rows of 49152 x 576 and 24 of them:
// 23 and 35 where two take 23 and 37, but 64 of 49152 x 1024 111 and 79).
static size_t rows_head_splits(size_t d, size_t vocab) {
    const size_t blocks = (d + 63) / 64;
    return std::max<size_t>(std::min((512 + blocks - 1) / blocks, (vocab + 63) / 64), 1);
}
size_t distill_dhn_floats(size_t n, size_t d, size_t vocab) {
    return (n <= kDistillRowsHead ? rows_head_splits(d, vocab) : 1) * n * d;
}
hipError_t launch_distill_rows_head(const float* grads, size_t n, size_t d, size_t vocab, const float* head,
                                    float* part, hipStream_t st) {
    const unsigned blocks = (unsigned)((d + 63) / 64), splits = (unsigned)rows_head_splits(d, vocab);
    static_assert(kDistillRowsHead == 32, "the rows of a wave");
    hipLaunchKernelGGL((n <= 16 ? distill_rows_head_kernel<1> : distill_rows_head_kernel<2>),
                       dim3((splits + 7) / 8 * 8 * blocks), dim3(256), 0, st, grads, (long)vocab, (int)n, head, (int)d,
                       (int)blocks, (int)splits, part);
    return hipGetLastError();
}
hipError_t launch_distill_rows_sum(const float* part, size_t j0, size_t n, size_t d, size_t vocab, float mul,
                                   const float* dloss, const DistillScored& g, float* dhn, hipStream_t st) {
    const size_t splits = distill_dhn_floats(n, d, vocab) / (n * d);
    hipLaunchKernelGGL(distill_rows_sum_kernel, dim3((unsigned)((d + 63) / 64), (unsigned)n), dim3(256), 0, st, part,
                       (int)splits, (int)j0, (int)n, (int)d, mul, dloss, g, dhn);
    return hipGetLastError();
}
hipError_t launch_distill_scaled(const float* hn, float mul, const float* dloss, const DistillScored& g, size_t padded,
                                 size_t d, float* out, hipStream_t st) {
    hipLaunchKernelGGL(distill_scaled_kernel, dim3((unsigned)padded), dim3(256), 0, st, hn, mul, dloss, g, out, (long)d);
    return hipGetLastError();
}
hipError_t launch_distill_finish(const int64_t* target, const float* loss, size_t t, void* misc, hipStream_t st) {
    hipLaunchKernelGGL(distill_finish_kernel, dim3(1), dim3(64), 0, st, target, loss, (int)t,
                       static_cast<CeMisc*>(misc));
    return hipGetLastError();
}

}  // namespace cfattn
