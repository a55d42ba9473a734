// Layer norm, forward and backward (cfops_layernorm_* of include/cfops.h):
//   mean = sum x / dim,  rstd = 1 / sqrt(sum (x - mean)^2 / dim + eps),
//   xh = (x - mean) rstd,  y = xh w + b;
//   g = dy w,  dx = rstd (g - sum g / dim - xh sum(g xh) / dim),
//   dw = sum over rows of dy xh,  db = sum over rows of dy.
// x, y, dy and dx are f32 or bf16; everything between is f32, rounded once at the end.
//
// A row is held in registers by NW waves, V chunks of 16 bytes a lane, so that it is read
// once, and the deviations that the variance sums are taken from the mean itself: a row
// far from zero loses nothing.  Both directions are bound by HBM.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "cfattn_common.hpp"
#include "cfops_kernels.hpp"

namespace cfattn {
namespace {

// 16 bytes of values, at the values' own alignment: rows of odd lengths are read as wide
// as others (the loads are the same instructions).
template <typename T>
struct Pack;
template <>
struct Pack<float> {
    static constexpr int N = 4;
    typedef float vec __attribute__((ext_vector_type(4), aligned(4)));
};
template <>
struct Pack<bf16_bits> {
    static constexpr int N = 8;
    typedef uint16_t vec __attribute__((ext_vector_type(8), aligned(2)));
};

// Values [0, N) of p as they lie in memory, those at or past n zero (and not read).
template <typename T>
__device__ __forceinline__ typename Pack<T>::vec load_raw(const T* p, int n) {
    typedef typename Pack<T>::vec Vec;
    if (n >= Pack<T>::N) return *reinterpret_cast<const Vec*>(p);
    Vec v = {};
#pragma unroll
    for (int i = 0; i < Pack<T>::N; i++)
        if (i < n) v[i] = p[i];
    return v;
}
template <typename T>
__device__ __forceinline__ float value(const typename Pack<T>::vec& v, int i) {
    const T e = v[i];
    return to_f32<T>(e);
}
template <typename T>
__device__ __forceinline__ void load_chunk(float (&x)[Pack<T>::N], const T* p, int n) {
    const typename Pack<T>::vec v = load_raw<T>(p, n);
#pragma unroll
    for (int i = 0; i < Pack<T>::N; i++) x[i] = value<T>(v, i);
}
template <typename T>
__device__ __forceinline__ void store_chunk(T* p, const float (&x)[Pack<T>::N], int n) {
    constexpr int N = Pack<T>::N;
    if (n >= N) {
        typedef typename Pack<T>::vec Vec;
        if constexpr (sizeof(T) == 2)
            *reinterpret_cast<Vec*>(p) = __builtin_bit_cast(Vec, cvt_bf16x8(x));
        else
            *reinterpret_cast<Vec*>(p) = Vec{x[0], x[1], x[2], x[3]};
    } else {
#pragma unroll
        for (int i = 0; i < N; i++)
            if (i < n) p[i] = from_f32<T>(x[i]);
    }
}
// N floats that belong to the same columns.
template <int N>
__device__ __forceinline__ void load_floats(float (&x)[N], const float* p, int n) {
#pragma unroll
    for (int q = 0; q < N; q += 4) {
        float t[4];
        load_chunk<float>(t, p + q, n - q);
#pragma unroll
        for (int i = 0; i < 4; i++) x[q + i] = t[i];
    }
}

template <int CTRL>
__device__ __forceinline__ float dpp(float x) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ float read_lane(float x, int lane) {
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), lane));
}
// The sum over a wave, in every lane: within rows of 16 lanes by lane permutations of the
// adder's own operand (xor 1, xor 2, the halves of 8, the halves of 16).
__device__ __forceinline__ float wave_sum(float x) {
    x += dpp<0xB1>(x);
    x += dpp<0x4E>(x);
    x += dpp<0x141>(x);
    x += dpp<0x140>(x);
    return (read_lane(x, 0) + read_lane(x, 16)) + (read_lane(x, 32) + read_lane(x, 48));
}
// The sums of K values over the NW waves of a row; `red` is theirs alone.
template <int NW, int K>
__device__ __forceinline__ void row_sums(float (&x)[K], float (*red)[K], int wave) {
#pragma unroll
    for (int k = 0; k < K; k++) x[k] = wave_sum(x[k]);
    if constexpr (NW > 1) {
        if ((threadIdx.x & 63) == 0)
#pragma unroll
            for (int k = 0; k < K; k++) red[wave][k] = x[k];
        __syncthreads();
#pragma unroll
        for (int k = 0; k < K; k++) x[k] = 0.0f;
#pragma unroll
        for (int w = 0; w < NW; w++)
#pragma unroll
            for (int k = 0; k < K; k++) x[k] += red[w][k];
    }
}

// R rows to NW waves (4 such to a workgroup with NW == 1, else one), which share the
// weights' loads and the barriers.
template <typename T, int NW, int V, int R>
__global__ __launch_bounds__(NW == 1 ? 256 : 64 * NW) void layernorm_fwd_kernel(
    const T* __restrict__ x, const float* __restrict__ w, const float* __restrict__ b, T* __restrict__ y,
    float* __restrict__ mean, float* __restrict__ rstd, long rows, int dim, float eps) {
    constexpr int N = Pack<T>::N, STEP = 64 * NW * N, ROWS = R * (NW == 1 ? 4 : 1);
    __shared__ float red[2][NW][R];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int c0 = (NW == 1 ? lane : (int)threadIdx.x) * N;
    // (With NW > 1 all waves of a workgroup have the same rows, and pass its barriers together.)
    for (long r0 = (long)blockIdx.x * ROWS + (NW == 1 ? wave * R : 0); r0 < rows; r0 += (long)gridDim.x * ROWS) {
        typename Pack<T>::vec v[R][V];
#pragma unroll
        for (int k = 0; k < R; k++)
#pragma unroll
            for (int i = 0; i < V; i++)
                v[k][i] = load_raw<T>(x + (r0 + k) * dim + c0 + i * STEP, r0 + k < rows ? dim - c0 - i * STEP : 0);
        // One row at a time, and registers for it: the weights are on their way beside it (65536 x 576
        // f32 53 us where this took 62, 999 x 1001 3.9 and 4.5).
        constexpr int AHEAD = R == 1 && V * N <= 16 ? V : 0;
        float wa[AHEAD ? AHEAD : 1][N], ba[AHEAD ? AHEAD : 1][N];
#pragma unroll
        for (int i = 0; i < AHEAD; i++) {
            load_floats<N>(wa[i], w + c0 + i * STEP, dim - c0 - i * STEP);
            if (b)
                load_floats<N>(ba[i], b + c0 + i * STEP, dim - c0 - i * STEP);
            else
#pragma unroll
                for (int e = 0; e < N; e++) ba[i][e] = 0.0f;
        }
        float mu[R], rs[R];
#pragma unroll
        for (int k = 0; k < R; k++) {
            mu[k] = 0.0f;
#pragma unroll
            for (int i = 0; i < V; i++)
#pragma unroll
                for (int e = 0; e < N; e++) mu[k] += value<T>(v[k][i], e);
        }
        row_sums<NW, R>(mu, red[0], wave);
#pragma unroll
        for (int k = 0; k < R; k++) {
            mu[k] /= (float)dim;
            rs[k] = 0.0f;
#pragma unroll
            for (int i = 0; i < V; i++)
#pragma unroll
                for (int e = 0; e < N; e++) {
                    const float d = c0 + i * STEP + e < dim ? value<T>(v[k][i], e) - mu[k] : 0.0f;
                    rs[k] = fmaf(d, d, rs[k]);
                }
        }
        row_sums<NW, R>(rs, red[1], wave);
#pragma unroll
        for (int k = 0; k < R; k++) {
            rs[k] = 1.0f / sqrtf(rs[k] / (float)dim + eps);
            if (c0 == 0 && r0 + k < rows) {
                mean[r0 + k] = mu[k];
                rstd[r0 + k] = rs[k];
            }
        }
#pragma unroll
        for (int i = 0; i < V; i++) {
            const int c = c0 + i * STEP;
            if (c >= dim) break;
            float ww[N], bb[N];
            if constexpr (AHEAD > 0) {
#pragma unroll
                for (int e = 0; e < N; e++) ww[e] = wa[i][e], bb[e] = ba[i][e];
            } else {
                load_floats<N>(ww, w + c, dim - c);
                if (b)
                    load_floats<N>(bb, b + c, dim - c);
                else
#pragma unroll
                    for (int e = 0; e < N; e++) bb[e] = 0.0f;
            }
#pragma unroll
            for (int k = 0; k < R; k++) {
                float o[N];
#pragma unroll
                for (int e = 0; e < N; e++) o[e] = fmaf((value<T>(v[k][i], e) - mu[k]) * rs[k], ww[e], bb[e]);
                if (r0 + k < rows) store_chunk<T>(y + (r0 + k) * dim + c, o, dim - c);
            }
        }
    }
}

// dx of rows g, g + G, .. to the g-th of G groups of NW waves over the grid, whose sums of
// dy xh and dy over their rows stay in registers; the next row's values are on their way
// while one is formed.  A workgroup of 8 waves adds up its groups' sums in LDS (dw's, then
// db's) and writes them to partial[block][2][dim].
constexpr int kBwdThreads = 512;
template <typename T, int NW, int V>
__global__ __launch_bounds__(kBwdThreads, V == 1 ? 4 : 2) void layernorm_bwd_kernel(
    const T* __restrict__ dy, const T* __restrict__ x, const float* __restrict__ w, const float* __restrict__ mean,
    const float* __restrict__ rstd, T* dx, float* __restrict__ partial, int want_b, long rows, int dim, int acc) {
    constexpr int N = Pack<T>::N, GROUPS = 8 / NW, STEP = 64 * NW * N;
    typedef typename Pack<T>::vec Vec;
    __shared__ float red[2][GROUPS][NW][2];
    extern __shared__ float sums[];  // [GROUPS][dim]
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, group = wave / NW;
    const int c0 = (lane + 64 * (wave % NW)) * N;
    float aw[V][N], ab[V][N], ww[V][N];
#pragma unroll
    for (int i = 0; i < V; i++) {
        load_floats<N>(ww[i], w + c0 + i * STEP, dim - c0 - i * STEP);
#pragma unroll
        for (int k = 0; k < N; k++) aw[i][k] = ab[i][k] = 0.0f;
    }
    const float inv_dim = 1.0f / (float)dim;
    const long stride = (long)gridDim.x * GROUPS;
    Vec xn[V], gn[V];
    float mn = 0.0f, rn = 0.0f;
    auto load = [&](long r) {
        const bool live = r < rows;
        const long at = live ? r : 0;
#pragma unroll
        for (int i = 0; i < V; i++) {
            const int n = live ? dim - c0 - i * STEP : 0;
            xn[i] = load_raw<T>(x + at * dim + c0 + i * STEP, n);
            gn[i] = load_raw<T>(dy + at * dim + c0 + i * STEP, n);
        }
        mn = live ? mean[at] : 0.0f, rn = live ? rstd[at] : 0.0f;
    };
    int turn = 0;
    load((long)blockIdx.x * GROUPS + group);
    // (The groups of a workgroup pass the barriers of row_sums together.)
    for (long r0 = (long)blockIdx.x * GROUPS; r0 < rows; r0 += stride, turn ^= 1) {
        const long r = r0 + group;
        Vec xv[V], gv[V];
#pragma unroll
        for (int i = 0; i < V; i++) xv[i] = xn[i], gv[i] = gn[i];
        const float mu = mn, rs = rn;
        if (r0 + stride < rows) load(r + stride);
        float s[2] = {0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < V; i++)
#pragma unroll
            for (int k = 0; k < N; k++) {
                // (Past the row's end dy is 0, and so is what x's deviation meets.)
                const float h = (value<T>(xv[i], k) - mu) * rs, g = value<T>(gv[i], k);
                aw[i][k] = fmaf(g, h, aw[i][k]);
                ab[i][k] += g;
                s[0] = fmaf(g, ww[i][k], s[0]);
                s[1] = fmaf(g * ww[i][k], h, s[1]);
            }
        row_sums<NW, 2>(s, red[turn][group], wave % NW);
        const float m0 = s[0] * inv_dim, m1 = s[1] * inv_dim;
        if (r >= rows) continue;
        T* dr = dx + r * dim;
#pragma unroll
        for (int i = 0; i < V; i++) {
            const int c = c0 + i * STEP;
            if (c >= dim) break;
            float o[N];
            if (acc)
                load_chunk<T>(o, dr + c, dim - c);
            else
#pragma unroll
                for (int k = 0; k < N; k++) o[k] = 0.0f;
#pragma unroll
            for (int k = 0; k < N; k++) {
                const float h = (value<T>(xv[i], k) - mu) * rs;
                o[k] += rs * (fmaf(value<T>(gv[i], k), ww[i][k], -m0) - h * m1);
            }
            store_chunk<T>(dr + c, o, dim - c);
        }
    }
    if (!partial) return;
    float* out = partial + (long)blockIdx.x * 2 * dim;
#pragma unroll
    for (int which = 0; which < 2; which++) {
        if (which && !want_b) return;
        if (GROUPS > 1 && which) __syncthreads();
#pragma unroll
        for (int i = 0; i < V; i++) {
            const int c = c0 + i * STEP;
#pragma unroll
            for (int k = 0; k < N; k++) {
                if (c + k >= dim) break;
                if constexpr (GROUPS > 1)
                    sums[group * dim + c + k] = which ? ab[i][k] : aw[i][k];
                else
                    out[which * dim + c + k] = which ? ab[i][k] : aw[i][k];
            }
        }
        if constexpr (GROUPS > 1) {
            __syncthreads();
            for (int c = threadIdx.x; c < dim; c += kBwdThreads) {
                float t = sums[c];
#pragma unroll
                for (int g = 1; g < GROUPS; g++) t += sums[g * dim + c];
                out[which * dim + c] = t;
            }
        }
    }
}

// dw and db from the workgroups' sums: 16 columns to a workgroup, 16 threads to a column,
// each every 16th of the sums in order, joined by halves.
__global__ __launch_bounds__(256) void layernorm_reduce_kernel(const float* __restrict__ partial,
                                                               float* __restrict__ dw, float* __restrict__ db,
                                                               int parts, long dim, int acc) {
    __shared__ float red[16][17];
    const int cl = threadIdx.x & 15, j = threadIdx.x >> 4;
    float* out = blockIdx.y ? db : dw;
    if (!out) return;
    const long c = (long)blockIdx.x * 16 + cl;
    const float* p = partial + (long)blockIdx.y * dim + c;
    float s = 0.0f;
    if (c < dim)
#pragma unroll 8
        for (int b = j; b < parts; b += 16) s += p[(long)b * 2 * dim];
    red[j][cl] = s;
    __syncthreads();
#pragma unroll
    for (int o = 8; o >= 1; o >>= 1) {
        if (j < o) red[j][cl] += red[j + o][cl];
        __syncthreads();
    }
    if (j == 0 && c < dim) out[c] = red[0][cl] + (acc ? out[c] : 0.0f);
}

// Rows that registers do not hold: a workgroup to a row, which passes over it for the mean,
// the deviations and the result; the weight's gradient in a kernel over columns.
constexpr int kWide = 1024;
__device__ __forceinline__ float block_sum(float x, float* red) {
    x = wave_sum(x);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = x;
    __syncthreads();
    float s = 0.0f;
#pragma unroll
    for (int w = 0; w < kWide / 64; w++) s += red[w];
    return s;
}
template <typename T>
__global__ __launch_bounds__(kWide) void layernorm_fwd_wide_kernel(const T* __restrict__ x, const float* __restrict__ w,
                                                                   const float* __restrict__ b, T* __restrict__ y,
                                                                   float* __restrict__ mean, float* __restrict__ rstd,
                                                                   long rows, int dim, float eps) {
    constexpr int N = Pack<T>::N;
    __shared__ float red[kWide / 64];
    const int c0 = threadIdx.x * N;
    for (long r = blockIdx.x; r < rows; r += gridDim.x) {
        const T* xr = x + r * dim;
        float s = 0.0f;
        for (long c = c0; c < dim; c += kWide * N) {
            float v[N], t = 0.0f;
            load_chunk<T>(v, xr + c, (int)min((long)N, dim - c));
#pragma unroll
            for (int k = 0; k < N; k++) t += v[k];
            s += t;
        }
        const float mu = block_sum(s, red) / (float)dim;
        s = 0.0f;
        for (long c = c0; c < dim; c += kWide * N) {
            float v[N], t = 0.0f;
            load_chunk<T>(v, xr + c, (int)min((long)N, dim - c));
#pragma unroll
            for (int k = 0; k < N; k++) t = c + k < dim ? fmaf(v[k] - mu, v[k] - mu, t) : t;
            s += t;
        }
        const float rs = 1.0f / sqrtf(block_sum(s, red) / (float)dim + eps);
        if (threadIdx.x == 0) mean[r] = mu, rstd[r] = rs;
        for (long c = c0; c < dim; c += kWide * N) {
            float v[N], ww[N], bb[N] = {};
            const int n = (int)min((long)N, dim - c);
            load_chunk<T>(v, xr + c, n);
            load_floats<N>(ww, w + c, n);
            if (b) load_floats<N>(bb, b + c, n);
#pragma unroll
            for (int k = 0; k < N; k++) v[k] = fmaf((v[k] - mu) * rs, ww[k], bb[k]);
            store_chunk<T>(y + r * dim + c, v, n);
        }
    }
}
template <typename T>
__global__ __launch_bounds__(kWide) void layernorm_bwd_wide_kernel(const T* __restrict__ dy, const T* __restrict__ x,
                                                                   const float* __restrict__ w,
                                                                   const float* __restrict__ mean,
                                                                   const float* __restrict__ rstd, T* dx, long rows,
                                                                   int dim, int acc) {
    constexpr int N = Pack<T>::N;
    __shared__ float red[kWide / 64];
    for (long r = blockIdx.x; r < rows; r += gridDim.x) {
        const T *xr = x + r * dim, *gr = dy + r * dim;
        T* dr = dx + r * dim;
        const float mu = mean[r], rs = rstd[r];
        float s0 = 0.0f, s1 = 0.0f;
        for (long c = threadIdx.x * N; c < dim; c += kWide * N) {
            float xv[N], gv[N], ww[N], t0 = 0.0f, t1 = 0.0f;
            const int n = (int)min((long)N, dim - c);
            load_chunk<T>(xv, xr + c, n);
            load_chunk<T>(gv, gr + c, n);
            load_floats<N>(ww, w + c, n);
#pragma unroll
            for (int k = 0; k < N; k++) {
                const float g = gv[k] * ww[k];
                t0 += g;
                t1 = fmaf(g, (xv[k] - mu) * rs, t1);
            }
            s0 += t0, s1 += t1;
        }
        const float m0 = block_sum(s0, red) / (float)dim, m1 = block_sum(s1, red) / (float)dim;
        for (long c = threadIdx.x * N; c < dim; c += kWide * N) {
            float xv[N], gv[N], ww[N], o[N] = {};
            const int n = (int)min((long)N, dim - c);
            load_chunk<T>(xv, xr + c, n);
            load_chunk<T>(gv, gr + c, n);
            load_floats<N>(ww, w + c, n);
            if (acc) load_chunk<T>(o, dr + c, n);
#pragma unroll
            for (int k = 0; k < N; k++) o[k] += rs * (gv[k] * ww[k] - m0 - (xv[k] - mu) * rs * m1);
            store_chunk<T>(dr + c, o, n);
        }
    }
}
// Sums over the rows of slice blockIdx.y, 256 columns to a workgroup.
template <typename T>
__global__ __launch_bounds__(256) void layernorm_columns_kernel(const T* __restrict__ dy, const T* __restrict__ x,
                                                                const float* __restrict__ mean,
                                                                const float* __restrict__ rstd,
                                                                float* __restrict__ partial, long rows, long dim) {
    const long c = (long)blockIdx.x * 256 + threadIdx.x;
    if (c >= dim) return;
    const long r0 = rows * blockIdx.y / gridDim.y, r1 = rows * (blockIdx.y + 1) / gridDim.y;
    float sw = 0.0f, sb = 0.0f;
#pragma unroll 4
    for (long r = r0; r < r1; r++) {
        const float g = to_f32<T>(dy[r * dim + c]);
        sw = fmaf(g, (to_f32<T>(x[r * dim + c]) - mean[r]) * rstd[r], sw);
        sb += g;
    }
    float* out = partial + (long)blockIdx.y * 2 * dim;
    out[c] = sw, out[dim + c] = sb;
}

// How a row lies in registers: waves, and chunks of a lane.  0 waves: it does not fit.
struct Form {
    int nw, v;
};
// The forward: the fewest waves whose lanes hold the row in up to four chunks each, of bf16 three where
// a wave has it alone (8192 x 2048 bf16 14.5 us of four waves, 18 of one; 30000 x 1001 f32 45 and 40).
template <typename T>
Form fwd_form(size_t chunks) {
    for (int nw : {1, 4, 8})
        if (chunks <= (size_t)(nw == 1 && sizeof(T) == 2 ? 192 : 256 * nw))
            return {nw, (int)((chunks + 64 * nw - 1) / (64 * nw))};
    return {0, 0};
}
// The backward, whose lanes hold the weight and two sums of each column too: one wave while it
// holds the row in three chunks, then the most that have one, and up to four in eight waves.
// (Us in one chunk of several waves and in four of one, or two of four: 8192 x 2048 bf16 20 and
// 30, 16384 x 4096 bf16 80 and 98, 999 x 1001 f32 5.1 and 8.6; but 65536 x 576 f32, which three
// chunks of a wave hold and four waves' not whole, 144 and 91.)
Form bwd_form(size_t chunks) {
    if (chunks <= 192) return {1, (int)((chunks + 63) / 64)};
    if (chunks <= 256) return {4, 1};
    if (chunks <= 2048) return {8, (int)((chunks + 511) / 512)};
    return {0, 0};
}
template <typename T>
size_t chunks_of(size_t dim) {
    return (dim + Pack<T>::N - 1) / Pack<T>::N;
}

// A grid of as many workgroups, or of fewer that take several rows each (a launch has fewer
// than 2^32 threads).
unsigned blocks_of(size_t n) { return (unsigned)std::min<size_t>(n, (size_t)1 << 21); }

// The backward's persistent grid by waves of a row (half of the workgroups, and of the
// partial sums, cost nothing where eight waves share a row: 16384 x 4096 bf16 80 us and 85; 65536
// x 576 f32 95 and 91), and slices of rows of the wide one.
size_t bwd_blocks(int nw) { return nw == 1 ? 512 : 256; }
constexpr size_t kSlices = 32;

template <typename T>
hipError_t fwd(const T* x, const float* w, const float* b, T* y, float* mean, float* rstd, size_t rows, size_t dim,
               float eps, hipStream_t st) {
    const Form f = fwd_form<T>(chunks_of<T>(dim));
    if (f.nw == 0) {
        hipLaunchKernelGGL(layernorm_fwd_wide_kernel<T>, dim3(blocks_of(rows)), dim3(kWide), 0, st, x, w, b, y, mean,
                           rstd, (long)rows, (int)dim, eps);
        return hipGetLastError();
    }
    auto go = [&](auto kernel, size_t per) {
        hipLaunchKernelGGL(kernel, dim3(blocks_of((rows + per - 1) / per)), dim3(f.nw == 1 ? 256 : 64 * f.nw), 0, st, x,
                           w, b, y, mean, rstd, (long)rows, (int)dim, eps);
        return hipGetLastError();
    };
    if (f.nw == 1) {
        if (f.v == 1) return go(layernorm_fwd_kernel<T, 1, 1, 1>, 4);
        if (f.v == 2) return go(layernorm_fwd_kernel<T, 1, 2, 1>, 4);
        if (f.v == 3 || sizeof(T) == 2) return go(layernorm_fwd_kernel<T, 1, 3, 1>, 4);
        return go(layernorm_fwd_kernel<T, 1, sizeof(T) == 2 ? 3 : 4, 1>, 4);
    }
    // Two rows at a time where that leaves every CU eight workgroups (16384 x 4096 bf16 54 us and
    // 63; a wave that has a row alone gains nothing).
    const bool two = rows >= 4096;
    if (f.nw == 4) {
        if constexpr (sizeof(T) == 2)
            if (f.v == 1)
                return two ? go(layernorm_fwd_kernel<T, 4, 1, 2>, 2) : go(layernorm_fwd_kernel<T, 4, 1, 1>, 1);
        if (f.v == 2) return two ? go(layernorm_fwd_kernel<T, 4, 2, 2>, 2) : go(layernorm_fwd_kernel<T, 4, 2, 1>, 1);
        if (f.v == 3) return two ? go(layernorm_fwd_kernel<T, 4, 3, 2>, 2) : go(layernorm_fwd_kernel<T, 4, 3, 1>, 1);
        return two ? go(layernorm_fwd_kernel<T, 4, 4, 2>, 2) : go(layernorm_fwd_kernel<T, 4, 4, 1>, 1);
    }
    if (f.v == 3) return two ? go(layernorm_fwd_kernel<T, 8, 3, 2>, 2) : go(layernorm_fwd_kernel<T, 8, 3, 1>, 1);
    return two ? go(layernorm_fwd_kernel<T, 8, 4, 2>, 2) : go(layernorm_fwd_kernel<T, 8, 4, 1>, 1);
}

template <typename T>
hipError_t bwd(const T* dy, const T* x, const float* w, const float* mean, const float* rstd, T* dx, float* dw,
               float* db, float* partial, size_t rows, size_t dim, int acc, hipStream_t st) {
    const Form f = bwd_form(chunks_of<T>(dim));
    const bool sums = dw || db;
    size_t parts;
    hipError_t e;
    if (f.nw == 0) {
        hipLaunchKernelGGL(layernorm_bwd_wide_kernel<T>, dim3(blocks_of(rows)), dim3(kWide), 0, st, dy, x, w, mean,
                           rstd, dx, (long)rows, (int)dim, acc);
        if ((e = hipGetLastError()) != hipSuccess || !sums) return e;
        parts = std::min(kSlices, rows);
        hipLaunchKernelGGL(layernorm_columns_kernel<T>, dim3((unsigned)((dim + 255) / 256), (unsigned)parts),
                           dim3(256), 0, st, dy, x, mean, rstd, partial, (long)rows, (long)dim);
        if ((e = hipGetLastError()) != hipSuccess) return e;
    } else {
        const size_t groups = 8 / f.nw;
        parts = std::min(bwd_blocks(f.nw), (rows + groups - 1) / groups);
        auto go = [&](auto kernel) {
            hipLaunchKernelGGL(kernel, dim3((unsigned)parts), dim3(kBwdThreads),
                               sums && groups > 1 ? groups * dim * sizeof(float) : 0, st, dy, x, w, mean, rstd, dx,
                               sums ? partial : nullptr, db != nullptr, (long)rows, (int)dim, acc);
            return hipGetLastError();
        };
        if (f.nw == 1)
            e = f.v == 1   ? go(layernorm_bwd_kernel<T, 1, 1>)
                : f.v == 2 ? go(layernorm_bwd_kernel<T, 1, 2>)
                           : go(layernorm_bwd_kernel<T, 1, 3>);
        else if (f.nw == 4)
            e = go(layernorm_bwd_kernel<T, 4, 1>);
        else
            e = f.v == 1   ? go(layernorm_bwd_kernel<T, 8, 1>)
                : f.v == 2 ? go(layernorm_bwd_kernel<T, 8, 2>)
                : f.v == 3 ? go(layernorm_bwd_kernel<T, 8, 3>)
                           : go(layernorm_bwd_kernel<T, 8, 4>);
        if (e != hipSuccess || !sums) return e;
    }
    hipLaunchKernelGGL(layernorm_reduce_kernel, dim3((unsigned)((dim + 15) / 16), 2), dim3(256), 0, st, partial, dw, db,
                       (int)parts, (long)dim, acc);
    return hipGetLastError();
}

}  // namespace

size_t layernorm_partial_floats(size_t rows, size_t dim) { return std::min(bwd_blocks(1), rows) * 2 * dim; }

hipError_t launch_layernorm_fwd(bool bf16, const void* x, const float* w, const float* b, void* y, float* mean,
                                float* rstd, size_t rows, size_t dim, float eps, hipStream_t st) {
    if (bf16)
        return fwd(static_cast<const bf16_bits*>(x), w, b, static_cast<bf16_bits*>(y), mean, rstd, rows, dim, eps, st);
    return fwd(static_cast<const float*>(x), w, b, static_cast<float*>(y), mean, rstd, rows, dim, eps, st);
}

hipError_t launch_layernorm_bwd(bool bf16, const void* dy, const void* x, const float* w, const float* mean,
                                const float* rstd, void* dx, float* dw, float* db, float* partial, size_t rows,
                                size_t dim, int acc, hipStream_t st) {
    if (bf16)
        return bwd(static_cast<const bf16_bits*>(dy), static_cast<const bf16_bits*>(x), w, mean, rstd,
                   static_cast<bf16_bits*>(dx), dw, db, partial, rows, dim, acc, st);
    return bwd(static_cast<const float*>(dy), static_cast<const float*>(x), w, mean, rstd, static_cast<float*>(dx), dw,
               db, partial, rows, dim, acc, st);
}

}  // namespace cfattn
