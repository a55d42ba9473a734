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

// Values [0, N) of p, those at or past n zero (and not read).
template <typename T>
__device__ __forceinline__ void load_chunk(float (&x)[Pack<T>::N], const T* p, int n) {
    constexpr int N = Pack<T>::N;
    if (n >= N) {
        const typename Pack<T>::vec v = *reinterpret_cast<const typename Pack<T>::vec*>(p);
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

// 4 rows to a workgroup with NW == 1, else one.
template <typename T, int NW, int V>
__global__ __launch_bounds__(NW == 1 ? 256 : 64 * NW) void layernorm_fwd_kernel(
    const T* __restrict__ x, const float* __restrict__ w, const float* __restrict__ b, T* __restrict__ y,
    float* __restrict__ mean, float* __restrict__ rstd, long rows, int dim, float eps) {
    constexpr int N = Pack<T>::N;
    __shared__ float red[2][NW][1];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int c0 = (NW == 1 ? lane : (int)threadIdx.x) * N;
    // (With NW > 1 all waves of a workgroup have the same rows, and pass its barriers together.)
    constexpr int ROWS = NW == 1 ? 4 : 1;
    for (long r = (long)blockIdx.x * ROWS + (NW == 1 ? wave : 0); r < rows; r += (long)gridDim.x * ROWS) {
        const T* xr = x + r * dim;
        float v[V][N];
#pragma unroll
        for (int i = 0; i < V; i++) load_chunk<T>(v[i], xr + c0 + i * 64 * NW * N, dim - c0 - i * 64 * NW * N);
        float s[1] = {0.0f};
#pragma unroll
        for (int i = 0; i < V; i++)
#pragma unroll
            for (int k = 0; k < N; k++) s[0] += v[i][k];
        row_sums<NW, 1>(s, red[0], wave);
        const float mu = s[0] / (float)dim;
        float q[1] = {0.0f};
#pragma unroll
        for (int i = 0; i < V; i++)
#pragma unroll
            for (int k = 0; k < N; k++) {
                const float d = c0 + i * 64 * NW * N + k < dim ? v[i][k] - mu : 0.0f;
                v[i][k] = d;
                q[0] = fmaf(d, d, q[0]);
            }
        row_sums<NW, 1>(q, red[1], wave);
        const float rs = 1.0f / sqrtf(q[0] / (float)dim + eps);
        if (c0 == 0) {
            mean[r] = mu;
            rstd[r] = rs;
        }
        T* yr = y + r * dim;
#pragma unroll
        for (int i = 0; i < V; i++) {
            const int c = c0 + i * 64 * NW * N;
            if (c >= dim) break;
            float ww[N], bb[N];
            load_floats<N>(ww, w + c, dim - c);
            if (b)
                load_floats<N>(bb, b + c, dim - c);
            else
#pragma unroll
                for (int k = 0; k < N; k++) bb[k] = 0.0f;
#pragma unroll
            for (int k = 0; k < N; k++) v[i][k] = fmaf(v[i][k] * rs, ww[k], bb[k]);
            store_chunk<T>(yr + c, v[i], dim - c);
        }
    }
}

// dx of rows g, g + G, .. to the g-th of G groups of NW waves over the grid, whose sums of
// dy xh and dy over their rows stay in registers; a workgroup of 8 waves adds up its
// groups' in LDS and writes them to partial[block][2][dim].
constexpr int kBwdThreads = 512;
template <typename T, int NW, int V>
__global__ __launch_bounds__(kBwdThreads) void layernorm_bwd_kernel(
    const T* __restrict__ dy, const T* __restrict__ x, const float* __restrict__ w, const float* __restrict__ mean,
    const float* __restrict__ rstd, T* dx, float* __restrict__ partial, int want_b, long rows, int dim, int acc) {
    constexpr int N = Pack<T>::N, GROUPS = 8 / NW;
    __shared__ float red[2][GROUPS][NW][2];
    extern __shared__ float sums[];  // [dim]
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, group = wave / NW;
    const int c0 = (lane + 64 * (wave % NW)) * N;
    float aw[V][N], ab[V][N], ww[V][N];
#pragma unroll
    for (int i = 0; i < V; i++) {
        load_floats<N>(ww[i], w + c0 + i * 64 * NW * N, dim - c0 - i * 64 * NW * N);
#pragma unroll
        for (int k = 0; k < N; k++) aw[i][k] = ab[i][k] = 0.0f;
    }
    const float inv_dim = 1.0f / (float)dim;
    int turn = 0;
    // (The groups of a workgroup pass the barriers of row_sums together.)
    for (long r0 = (long)blockIdx.x * GROUPS; r0 < rows; r0 += (long)gridDim.x * GROUPS, turn ^= 1) {
        const long r = r0 + group;
        const bool live = r < rows;
        const int n = live ? dim : 0;
        const T *xr = x + (live ? r : 0) * dim, *gr = dy + (live ? r : 0) * dim;
        float xv[V][N], gv[V][N];
#pragma unroll
        for (int i = 0; i < V; i++) {
            const int c = c0 + i * 64 * NW * N;
            load_chunk<T>(xv[i], xr + c, n - c);
            load_chunk<T>(gv[i], gr + c, n - c);
        }
        const float mu = live ? mean[r] : 0.0f, rs = live ? rstd[r] : 0.0f;
        float s[2] = {0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < V; i++)
#pragma unroll
            for (int k = 0; k < N; k++) {
                // (Past the row's end dy is 0, and so is what x's deviation meets.)
                const float h = (xv[i][k] - mu) * rs, g = gv[i][k];
                aw[i][k] = fmaf(g, h, aw[i][k]);
                ab[i][k] += g;
                const float gw = g * ww[i][k];
                s[0] += gw;
                s[1] = fmaf(gw, h, s[1]);
                xv[i][k] = h;
                gv[i][k] = gw;
            }
        row_sums<NW, 2>(s, red[turn][group], wave % NW);
        const float m0 = s[0] * inv_dim, m1 = s[1] * inv_dim;
        if (!live) continue;
        T* dr = dx + r * dim;
#pragma unroll
        for (int i = 0; i < V; i++) {
            const int c = c0 + i * 64 * NW * N;
            if (c >= dim) break;
            float o[N];
            if (acc)
                load_chunk<T>(o, dr + c, dim - c);
            else
#pragma unroll
                for (int k = 0; k < N; k++) o[k] = 0.0f;
#pragma unroll
            for (int k = 0; k < N; k++) o[k] += rs * (gv[i][k] - m0 - xv[i][k] * m1);
            store_chunk<T>(dr + c, o, dim - c);
        }
    }
    if (!partial) return;
    float* out = partial + (long)blockIdx.x * 2 * dim;
    for (int which = 0; which < (want_b ? 2 : 1); which++) {
        for (int g = 0; g < GROUPS; g++) {
            if (group == g) {
#pragma unroll
                for (int i = 0; i < V; i++)
#pragma unroll
                    for (int k = 0; k < N; k++) {
                        const int c = c0 + i * 64 * NW * N + k;
                        if (c >= dim) continue;
                        const float a = (which ? ab[i][k] : aw[i][k]) + (g ? sums[c] : 0.0f);
                        if (g + 1 < GROUPS)
                            sums[c] = a;
                        else
                            out[which * dim + c] = a;
                    }
            }
            if (GROUPS > 1) __syncthreads();
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

// How a row lies in registers: the fewest waves whose lanes hold it in up to four chunks
// each (eight of f32 in the widest form).  0 waves: it does not fit.
struct Form {
    int nw, v;
};
template <typename T>
Form form_of(size_t dim) {
    const size_t chunks = (dim + Pack<T>::N - 1) / Pack<T>::N;
    for (int nw : {1, 4, 8})
        for (int v = 1; v <= (nw == 8 && sizeof(T) == 4 ? 8 : 4); v++)
            if (chunks <= (size_t)64 * nw * v) return {nw, nw == 8 && v > 4 ? 8 : nw == 1 ? v : std::max(v, 2)};
    return {0, 0};
}

// A grid of as many workgroups, or of fewer that take several rows each (a launch has fewer
// than 2^32 threads).
unsigned blocks_of(size_t n) { return (unsigned)std::min<size_t>(n, (size_t)1 << 21); }

// The persistent grid of the backward, and slices of rows of the wide one.
constexpr size_t kBwdBlocks = 512, kSlices = 32;

template <typename T>
hipError_t fwd(const T* x, const float* w, const float* b, T* y, float* mean, float* rstd, size_t rows, size_t dim,
               float eps, hipStream_t st) {
    const Form f = form_of<T>(dim);
    if (f.nw == 0) {
        hipLaunchKernelGGL(layernorm_fwd_wide_kernel<T>, dim3(blocks_of(rows)), dim3(kWide), 0, st, x, w, b, y, mean,
                           rstd, (long)rows, (int)dim, eps);
        return hipGetLastError();
    }
    auto go = [&](auto kernel, int nw) {
        hipLaunchKernelGGL(kernel, dim3(blocks_of(nw == 1 ? (rows + 3) / 4 : rows)), dim3(nw == 1 ? 256 : 64 * nw), 0,
                           st, x, w, b, y, mean, rstd, (long)rows, (int)dim, eps);
        return hipGetLastError();
    };
    if (f.nw == 1) {
        if (f.v == 1) return go(layernorm_fwd_kernel<T, 1, 1>, 1);
        if (f.v == 2) return go(layernorm_fwd_kernel<T, 1, 2>, 1);
        if (f.v == 3) return go(layernorm_fwd_kernel<T, 1, 3>, 1);
        return go(layernorm_fwd_kernel<T, 1, 4>, 1);
    }
    if (f.nw == 4) {
        if (f.v == 2) return go(layernorm_fwd_kernel<T, 4, 2>, 4);
        if (f.v == 3) return go(layernorm_fwd_kernel<T, 4, 3>, 4);
        return go(layernorm_fwd_kernel<T, 4, 4>, 4);
    }
    if constexpr (sizeof(T) == 4)
        if (f.v == 8) return go(layernorm_fwd_kernel<T, 8, 8>, 8);
    if (f.v == 3) return go(layernorm_fwd_kernel<T, 8, 3>, 8);
    return go(layernorm_fwd_kernel<T, 8, 4>, 8);
}

template <typename T>
hipError_t bwd(const T* dy, const T* x, const float* w, const float* mean, const float* rstd, T* dx, float* dw,
               float* db, float* partial, size_t rows, size_t dim, int acc, hipStream_t st) {
    const Form f = form_of<T>(dim);
    const bool sums = dw || db;
    size_t parts;
    hipError_t e;
    if (f.nw == 0) {
        hipLaunchKernelGGL(layernorm_bwd_wide_kernel<T>, dim3(blocks_of(rows)), dim3(kWide), 0, st, dy, x, w, mean, rstd,
                           dx, (long)rows, (int)dim, acc);
        if ((e = hipGetLastError()) != hipSuccess || !sums) return e;
        parts = std::min(kSlices, rows);
        hipLaunchKernelGGL(layernorm_columns_kernel<T>, dim3((unsigned)((dim + 255) / 256), (unsigned)parts),
                           dim3(256), 0, st, dy, x, mean, rstd, partial, (long)rows, (long)dim);
        if ((e = hipGetLastError()) != hipSuccess) return e;
    } else {
        const size_t groups = 8 / f.nw;
        parts = std::min(kBwdBlocks, (rows + groups - 1) / groups);
        auto go = [&](auto kernel) {
            hipLaunchKernelGGL(kernel, dim3((unsigned)parts), dim3(kBwdThreads),
                               sums && groups > 1 ? dim * sizeof(float) : 0, st, dy, x, w, mean, rstd, dx,
                               sums ? partial : nullptr, db != nullptr, (long)rows, (int)dim, acc);
            return hipGetLastError();
        };
        e = f.nw == 1   ? f.v == 1   ? go(layernorm_bwd_kernel<T, 1, 1>)
                          : f.v == 2 ? go(layernorm_bwd_kernel<T, 1, 2>)
                          : f.v == 3 ? go(layernorm_bwd_kernel<T, 1, 3>)
                                     : go(layernorm_bwd_kernel<T, 1, 4>)
            : f.nw == 4 ? f.v == 2   ? go(layernorm_bwd_kernel<T, 4, 2>)
                          : f.v == 3 ? go(layernorm_bwd_kernel<T, 4, 3>)
                                     : go(layernorm_bwd_kernel<T, 4, 4>)
            : f.v == 3  ? go(layernorm_bwd_kernel<T, 8, 3>)
            : f.v == 4  ? go(layernorm_bwd_kernel<T, 8, 4>)
                        : go(layernorm_bwd_kernel<T, 8, sizeof(T) == 4 ? 8 : 4>);
        if (e != hipSuccess || !sums) return e;
    }
    hipLaunchKernelGGL(layernorm_reduce_kernel, dim3((unsigned)((dim + 15) / 16), 2), dim3(256), 0, st, partial, dw, db,
                       (int)parts, (long)dim, acc);
    return hipGetLastError();
}

}  // namespace

size_t layernorm_partial_floats(size_t rows, size_t dim) { return std::min(kBwdBlocks, rows) * 2 * dim; }

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
