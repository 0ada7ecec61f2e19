// abh_norm.hip -- layer norm over the last axis, forward and backward.
//
//   y = (x - mean) rstd w + b,   rstd = 1 / sqrt(mean((x - mean)^2) + eps)
//   dx = rstd (g w - mean(g w) - xh mean(g w xh)),   xh = (x - mean) rstd
//   dw = sum over rows of g xh,   db = sum over rows of g
//
// Everything is FP32 between the loads and the one rounding of each result.  The bytes bound it: x in and
// y out forward, x and g in and dx out backward.  So a row is read once and stays in registers, where
// its mean and then the mean of its squared deviations are taken (no difference of large squares), and
// the backward pass takes dx and the row's share of dw and db from one reading.  The weight's gradient is a
// sum over all rows: each workgroup takes every P-th row, keeps its columns' sums in registers, and writes
// them once; a second kernel adds the P partial sums in order, so that no result depends on the schedule.

#include <hip/hip_runtime.h>

#include <stdint.h>

#include <algorithm>

#include "../../include/adambridge_hip.h"
#include "abh_device.hpp"
#include "abh_host.hpp"
#include "abh_rows.hpp"

namespace abh {

struct NormArgs {
    const void* x;
    const void* g;
    const void* w;
    const void* b;
    void* y;        // or dx
    float* stats;   // mean, rstd a row
    float* part;    // P x 2 x cols: sums of g xh, of g
    int64_t rows, cols;
    float eps;
};

// G lanes a row, NV vectors a lane.  A row of up to 64 lanes has a wavefront (four a workgroup), a longer one
// a workgroup.
template <int G>
constexpr int kNormThreads = G < 256 ? 256 : G;

template <int DT, int WT, int G, int NV>
__global__ __launch_bounds__(kNormThreads<G>) void k_norm(NormArgs A)
{
    constexpr int K = kLane<DT>, T = kNormThreads<G>;
    __shared__ float part[2 * T / kWave];
    const int lane = threadIdx.x % G;
    const int64_t row = (int64_t)blockIdx.x * (T / G) + threadIdx.x / G;
    if (G < T && row >= A.rows) return;   // whole wavefronts, and no barrier follows
    const void* x = at<DT>(A.x, row * A.cols);
    float v[NV][K];
    float sum = 0.0f, none = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) load_vec<DT>(x, (int64_t)(i * G + lane) * K, A.cols, v[i]);
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int k = 0; k < K; ++k) sum += v[i][k];
    block_sum2<G>(sum, none, part);
    const float mean = sum / (float)A.cols;
    float sq = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int k = 0; k < K; ++k) {
            v[i][k] -= mean;
            if ((int64_t)(i * G + lane) * K + k < A.cols) sq = __builtin_fmaf(v[i][k], v[i][k], sq);
        }
    block_sum2<G>(sq, none, part);
    const float rstd = 1.0f / sqrtf(sq / (float)A.cols + A.eps);
    if (A.stats && lane == 0) {
        A.stats[2 * row] = mean;
        A.stats[2 * row + 1] = rstd;
    }
    void* y = at<DT>(A.y, row * A.cols);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int64_t c = (int64_t)(i * G + lane) * K;
        if (c >= A.cols) break;
        float w[K], b[K];
        load_like<WT, K>(A.w, c, A.cols, 1.0f, w);
        load_like<WT, K>(A.b, c, A.cols, 0.0f, b);
#pragma unroll
        for (int k = 0; k < K; ++k) w[k] = __builtin_fmaf(v[i][k] * rstd, w[k], b[k]);
        store_vec<DT>(y, c, A.cols, w);
    }
}

// Rows that no register file holds: read three times (the second and third time mostly out of the L2).
template <int DT, int WT>
__global__ __launch_bounds__(1024) void k_norm_long(NormArgs A)
{
    constexpr int K = kLane<DT>, T = 1024;
    __shared__ float part[2 * T / kWave];
    const int64_t row = blockIdx.x;
    const void* x = at<DT>(A.x, row * A.cols);
    float sum = 0.0f, sq = 0.0f, none = 0.0f, v[K];
    for (int64_t c = (int64_t)threadIdx.x * K; c < A.cols; c += T * K) {
        load_vec<DT>(x, c, A.cols, v);
#pragma unroll
        for (int k = 0; k < K; ++k) sum += v[k];
    }
    block_sum2<T>(sum, none, part);
    const float mean = sum / (float)A.cols;
    for (int64_t c = (int64_t)threadIdx.x * K; c < A.cols; c += T * K) {
        load_vec<DT>(x, c, A.cols, v);
#pragma unroll
        for (int k = 0; k < K; ++k)
            if (c + k < A.cols) sq = __builtin_fmaf(v[k] - mean, v[k] - mean, sq);
    }
    block_sum2<T>(sq, none, part);
    const float rstd = 1.0f / sqrtf(sq / (float)A.cols + A.eps);
    if (A.stats && threadIdx.x == 0) {
        A.stats[2 * row] = mean;
        A.stats[2 * row + 1] = rstd;
    }
    void* y = at<DT>(A.y, row * A.cols);
    for (int64_t c = (int64_t)threadIdx.x * K; c < A.cols; c += T * K) {
        float w[K], b[K];
        load_vec<DT>(x, c, A.cols, v);
        load_like<WT, K>(A.w, c, A.cols, 1.0f, w);
        load_like<WT, K>(A.b, c, A.cols, 0.0f, b);
#pragma unroll
        for (int k = 0; k < K; ++k) v[k] = __builtin_fmaf((v[k] - mean) * rstd, w[k], b[k]);
        store_vec<DT>(y, c, A.cols, v);
    }
}

// dx and this workgroup's partial sums of dw and db.
template <int DT, int WT, int G, int NV>
__global__ __launch_bounds__(kNormThreads<G>) void k_norm_back(NormArgs A)
{
    constexpr int K = kLane<DT>, T = kNormThreads<G>, R = T / G;
    __shared__ float part[2 * T / kWave];
    __shared__ float cross[R > 1 ? 2 * R * G * K : 1];
    const int lane = threadIdx.x % G, sub = threadIdx.x / G;
    float w[NV][K], dw[NV][K], db[NV][K];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        load_like<WT, K>(A.w, (int64_t)(i * G + lane) * K, A.cols, 1.0f, w[i]);
#pragma unroll
        for (int k = 0; k < K; ++k) dw[i][k] = db[i][k] = 0.0f;
    }
    const float inv = 1.0f / (float)A.cols;
    for (int64_t row = (int64_t)blockIdx.x * R + sub; row < A.rows; row += (int64_t)gridDim.x * R) {
        const void* xr = at<DT>(A.x, row * A.cols);
        const void* gr = at<DT>(A.g, row * A.cols);
        const float mean = A.stats[2 * row], rstd = A.stats[2 * row + 1];
        float x[NV][K], g[NV][K];
        float c1 = 0.0f, c2 = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            load_vec<DT>(xr, (int64_t)(i * G + lane) * K, A.cols, x[i]);
            load_vec<DT>(gr, (int64_t)(i * G + lane) * K, A.cols, g[i]);
        }
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int k = 0; k < K; ++k) {
                x[i][k] = (x[i][k] - mean) * rstd;
                dw[i][k] = __builtin_fmaf(g[i][k], x[i][k], dw[i][k]);
                db[i][k] += g[i][k];
                g[i][k] *= w[i][k];
                c1 += g[i][k];
                c2 = __builtin_fmaf(g[i][k], x[i][k], c2);
            }
        if (A.y) {
            block_sum2<G>(c1, c2, part);
            c1 *= inv;
            c2 *= inv;
            void* dx = at<DT>(A.y, row * A.cols);
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int64_t c = (int64_t)(i * G + lane) * K;
                if (c >= A.cols) break;
#pragma unroll
                for (int k = 0; k < K; ++k) g[i][k] = rstd * (g[i][k] - c1 - x[i][k] * c2);
                store_vec<DT>(dx, c, A.cols, g[i]);
            }
        }
    }
    if (!A.part) return;
    float* out = A.part + (int64_t)blockIdx.x * 2 * A.cols;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int64_t c = (int64_t)(i * G + lane) * K;
        if constexpr (R > 1) {   // the wavefronts' sums, added in order
            __syncthreads();
#pragma unroll
            for (int k = 0; k < K; ++k) {
                cross[(sub * 2 * K + k) * G + lane] = dw[i][k];
                cross[(sub * 2 * K + K + k) * G + lane] = db[i][k];
            }
            __syncthreads();
            if (sub == 0) {
#pragma unroll
                for (int r = 1; r < R; ++r)
#pragma unroll
                    for (int k = 0; k < K; ++k) {
                        dw[i][k] += cross[(r * 2 * K + k) * G + lane];
                        db[i][k] += cross[(r * 2 * K + K + k) * G + lane];
                    }
            }
        }
        if (sub == 0) {
#pragma unroll
            for (int k = 0; k < K; ++k)
                if (c + k < A.cols) {
                    out[c + k] = dw[i][k];
                    out[A.cols + c + k] = db[i][k];
                }
        }
    }
}

// The same for rows that no register file holds: dx a row a workgroup, reading the row twice ...
template <int DT, int WT>
__global__ __launch_bounds__(1024) void k_norm_back_long(NormArgs A)
{
    constexpr int K = kLane<DT>, T = 1024;
    __shared__ float part[2 * T / kWave];
    const int64_t row = blockIdx.x;
    const void* xr = at<DT>(A.x, row * A.cols);
    const void* gr = at<DT>(A.g, row * A.cols);
    const float mean = A.stats[2 * row], rstd = A.stats[2 * row + 1];
    float c1 = 0.0f, c2 = 0.0f, x[K], g[K], w[K];
    for (int64_t c = (int64_t)threadIdx.x * K; c < A.cols; c += T * K) {
        load_vec<DT>(xr, c, A.cols, x);
        load_vec<DT>(gr, c, A.cols, g);
        load_like<WT, K>(A.w, c, A.cols, 1.0f, w);
#pragma unroll
        for (int k = 0; k < K; ++k) {
            c1 = __builtin_fmaf(g[k], w[k], c1);
            c2 = __builtin_fmaf(g[k] * w[k], (x[k] - mean) * rstd, c2);
        }
    }
    block_sum2<T>(c1, c2, part);
    c1 /= (float)A.cols;
    c2 /= (float)A.cols;
    void* dx = at<DT>(A.y, row * A.cols);
    for (int64_t c = (int64_t)threadIdx.x * K; c < A.cols; c += T * K) {
        load_vec<DT>(xr, c, A.cols, x);
        load_vec<DT>(gr, c, A.cols, g);
        load_like<WT, K>(A.w, c, A.cols, 1.0f, w);
#pragma unroll
        for (int k = 0; k < K; ++k) g[k] = rstd * (g[k] * w[k] - c1 - (x[k] - mean) * rstd * c2);
        store_vec<DT>(dx, c, A.cols, g);
    }
}

// ... and the partial sums of columns 256 K blockIdx.x on over the rows blockIdx.y, + gridDim.y, ...
template <int DT>
__global__ __launch_bounds__(256) void k_norm_columns(NormArgs A)
{
    constexpr int K = kLane<DT>;
    const int64_t c = ((int64_t)blockIdx.x * 256 + threadIdx.x) * K;
    if (c >= A.cols) return;
    float dw[K], db[K], x[K], g[K];
#pragma unroll
    for (int k = 0; k < K; ++k) dw[k] = db[k] = 0.0f;
    for (int64_t row = blockIdx.y; row < A.rows; row += gridDim.y) {
        load_vec<DT>(at<DT>(A.x, row * A.cols), c, A.cols, x);
        load_vec<DT>(at<DT>(A.g, row * A.cols), c, A.cols, g);
        const float mean = A.stats[2 * row], rstd = A.stats[2 * row + 1];
#pragma unroll
        for (int k = 0; k < K; ++k) {
            dw[k] = __builtin_fmaf(g[k], (x[k] - mean) * rstd, dw[k]);
            db[k] += g[k];
        }
    }
    float* out = A.part + (int64_t)blockIdx.y * 2 * A.cols;
#pragma unroll
    for (int k = 0; k < K; ++k)
        if (c + k < A.cols) {
            out[c + k] = dw[k];
            out[A.cols + c + k] = db[k];
        }
}

// The P partial sums of 64 columns a workgroup: 16 lanes a column each take every 16th, then a tree.
constexpr int kSumLanes = 16;

template <int WT>
__global__ __launch_bounds__(64 * kSumLanes) void k_norm_sums(const float* part, int32_t parts, int64_t cols, void* dw, void* db)
{
    __shared__ float tree[kSumLanes][64];
    const int col = threadIdx.x & 63, at_row = threadIdx.x >> 6;
    const int64_t c = (int64_t)blockIdx.x * 64 + col;   // of 2 cols: dw's, then db's
    float s = 0.0f;
    if (c < 2 * cols)
        for (int p = at_row; p < parts; p += kSumLanes) s += part[(int64_t)p * 2 * cols + c];
    tree[at_row][col] = s;
    for (int d = kSumLanes / 2; d; d /= 2) {
        __syncthreads();
        if (at_row < d) tree[at_row][col] += tree[at_row + d][col];
    }
    if (at_row == 0 && c < 2 * cols) {
        void* out = c < cols ? dw : db;
        if (out) put<WT>(out, c < cols ? c : c - cols, tree[0][col]);
    }
}

static bool type_ok(int32_t t) { return t == ADAMBRIDGE_DT_F32 || t == ADAMBRIDGE_DT_BF16; }

// Lanes a row (0: the long form) and vectors a lane.  Backward, whose lanes hold five values a column, the
// registers of 1024 lanes end at two.
struct Shape {
    int lanes, vectors;
};

static Shape norm_shape(int64_t cols, int32_t dtype, bool back)
{
    const int64_t v = (cols + (dtype == ADAMBRIDGE_DT_BF16 ? 7 : 3)) / (dtype == ADAMBRIDGE_DT_BF16 ? 8 : 4);
    if (v <= 64) return {64, 1};
    if (v <= 128) return {64, 2};
    if (v <= 256) return {64, 4};
    if (v <= 512) return {256, 2};
    if (v <= 1024) return {256, 4};
    if (v <= 2048) return {1024, 2};
    if (v <= 4096 && !back) return {1024, 4};
    return {0, 0};
}

// Workgroups of the backward pass, each with its partial sums.
static int norm_parts(int64_t rows, int64_t cols, int32_t dtype)
{
    const Shape s = norm_shape(cols, dtype, true);
    const int64_t a_group = s.lanes == 64 ? 4 : 1;
    return (int)std::max<int64_t>(1, std::min<int64_t>(512, (rows + a_group * 4 - 1) / (a_group * 4)));
}

template <int DT, int WT>
static void launch_norm(const NormArgs& A, bool back, int parts)
{
    const Shape s = norm_shape(A.cols, DT, back);
#define ABH_NORM(G, NV)                                                                                                 \
    if (!back && s.lanes == G && s.vectors == NV) {                                                                     \
        constexpr int R = kNormThreads<G> / G;                                                                          \
        hipLaunchKernelGGL((k_norm<DT, WT, G, NV>), dim3((unsigned)((A.rows + R - 1) / R)), dim3(kNormThreads<G>), 0,    \
                           t_stream, A);                                                                                \
        return;                                                                                                         \
    }
    ABH_NORM(64, 1) ABH_NORM(64, 2) ABH_NORM(64, 4) ABH_NORM(256, 2) ABH_NORM(256, 4) ABH_NORM(1024, 2) ABH_NORM(1024, 4)
#undef ABH_NORM
#define ABH_NORM_BACK(G, NV)                                                                                            \
    if (back && s.lanes == G && s.vectors == NV) {                                                                      \
        hipLaunchKernelGGL((k_norm_back<DT, WT, G, NV>), dim3(parts), dim3(kNormThreads<G>), 0, t_stream, A);            \
        return;                                                                                                         \
    }
    ABH_NORM_BACK(64, 1) ABH_NORM_BACK(64, 2) ABH_NORM_BACK(64, 4) ABH_NORM_BACK(256, 2) ABH_NORM_BACK(256, 4)
    ABH_NORM_BACK(1024, 2)
#undef ABH_NORM_BACK
    if (!back) {
        hipLaunchKernelGGL((k_norm_long<DT, WT>), dim3((unsigned)A.rows), dim3(1024), 0, t_stream, A);
        return;
    }
    if (A.y) hipLaunchKernelGGL((k_norm_back_long<DT, WT>), dim3((unsigned)A.rows), dim3(1024), 0, t_stream, A);
    if (A.part)
        hipLaunchKernelGGL((k_norm_columns<DT>), dim3((unsigned)((A.cols + 256 * kLane<DT> - 1) / (256 * kLane<DT>)), (unsigned)parts),
                           dim3(256), 0, t_stream, A);
}

static void norm_by_type(const NormArgs& A, int32_t dtype, int32_t w_dtype, bool back, int parts)
{
    const bool bf = dtype == ADAMBRIDGE_DT_BF16, wbf = w_dtype == ADAMBRIDGE_DT_BF16;
    if (bf && wbf) launch_norm<DT_BF16, DT_BF16>(A, back, parts);
    else if (bf) launch_norm<DT_BF16, DT_F32>(A, back, parts);
    else if (wbf) launch_norm<DT_F32, DT_BF16>(A, back, parts);
    else launch_norm<DT_F32, DT_F32>(A, back, parts);
}

constexpr int64_t kNormMost = (int64_t)1 << 30;   // rows (a workgroup or a wavefront each) and columns

}  // namespace abh

using namespace abh;

extern "C" {

ADAMBRIDGE_API int adambridge_layer_norm(const void* x, int32_t dtype, const void* weight, const void* bias, int32_t w_dtype,
                                         int64_t rows, int64_t cols, float eps, void* y, float* stats)
{
    if (rows < 1 || cols < 1 || rows > kNormMost || cols > kNormMost) return ADAMBRIDGE_EBADN;
    if (!type_ok(dtype) || !type_ok(w_dtype)) return ADAMBRIDGE_EMVDTYPE;
    if (!x || !y) return ADAMBRIDGE_ENULL;
    const NormArgs A{x, nullptr, weight, bias, y, stats, nullptr, rows, cols, eps};
    norm_by_type(A, dtype, w_dtype, false, 0);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? 0 : hip_fail(e, "hipLaunchKernelGGL (layer norm)");
}

ADAMBRIDGE_API int64_t adambridge_layer_norm_work(int64_t rows, int64_t cols, int32_t dtype)
{
    if (rows < 1 || cols < 1 || rows > kNormMost || cols > kNormMost) return ADAMBRIDGE_EBADN;
    if (!type_ok(dtype)) return ADAMBRIDGE_EMVDTYPE;
    return (int64_t)norm_parts(rows, cols, dtype) * 2 * cols * 4;
}

ADAMBRIDGE_API int adambridge_layer_norm_backward(const void* gout, const void* x, int32_t dtype, const void* weight,
                                                  int32_t w_dtype, const float* stats, int64_t rows, int64_t cols, void* dx,
                                                  void* dweight, void* dbias, void* work)
{
    if (rows < 1 || cols < 1 || rows > kNormMost || cols > kNormMost) return ADAMBRIDGE_EBADN;
    if (!type_ok(dtype) || !type_ok(w_dtype)) return ADAMBRIDGE_EMVDTYPE;
    const bool sums = dweight || dbias;
    if (!gout || !x || !stats || (sums && !work)) return ADAMBRIDGE_ENULL;
    if (!dx && !sums) return 0;
    const int parts = norm_parts(rows, cols, dtype);
    const NormArgs A{x, gout, weight, nullptr, dx, const_cast<float*>(stats), sums ? static_cast<float*>(work) : nullptr,
                     rows, cols, 0.0f};
    norm_by_type(A, dtype, w_dtype, true, parts);
    if (sums) {
        const dim3 grid((unsigned)((2 * cols + 63) / 64)), block(64 * kSumLanes);
        if (w_dtype == ADAMBRIDGE_DT_BF16)
            hipLaunchKernelGGL((k_norm_sums<DT_BF16>), grid, block, 0, t_stream, A.part, parts, cols, dweight, dbias);
        else
            hipLaunchKernelGGL((k_norm_sums<DT_F32>), grid, block, 0, t_stream, A.part, parts, cols, dweight, dbias);
    }
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? 0 : hip_fail(e, "hipLaunchKernelGGL (layer norm's gradient)");
}

}  // extern "C"
