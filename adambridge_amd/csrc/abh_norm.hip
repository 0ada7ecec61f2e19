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
    void* dw;
    void* db;
    float* part;    // P x 2 x cols: sums of g xh, of g
    int64_t rows, cols;
    float eps;
};

// G lanes a row, NV vectors a lane: part of a wavefront, a wavefront, or a workgroup.
template <int G>
constexpr int kNormThreads = G < 256 ? 256 : G;

template <int DT, int WT, int G, int NV>
__global__ __launch_bounds__(kNormThreads<G>) void k_norm(NormArgs A)
{
    constexpr int K = kLane<DT>, T = kNormThreads<G>;
    __shared__ float part[2][2 * T / kWave];
    const int lane = threadIdx.x % G;
    const int64_t row = block_index() * (T / G) + threadIdx.x / G;
    if (row >= A.rows) return;   // whole groups of lanes that sum together, or the workgroup
    const void* x = at<DT>(A.x, row * A.cols);
    raw16 v[NV];
    float sum = 0.0f, none = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) v[i] = load_vec_raw<DT>(x, (int64_t)(i * G + lane) * K, A.cols);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        float f[K];
        to_floats<DT>(v[i], f);
#pragma unroll
        for (int k = 0; k < K; ++k) sum += f[k];
    }
    block_sum2<G>(sum, none, part[0], lane);
    const float mean = sum / (float)A.cols;
    float sq = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        float f[K];
        hold(v[i]);
        to_floats<DT>(v[i], f);
        const int64_t c = (int64_t)(i * G + lane) * K;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const float d = c + k < A.cols ? f[k] - mean : 0.0f;
            sq = __builtin_fmaf(d, d, sq);
        }
    }
    block_sum2<G>(sq, none, part[1], lane);
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
        float f[K], w[K], b[K];
        hold(v[i]);
        to_floats<DT>(v[i], f);
        load_like<WT, K>(A.w, c, A.cols, 1.0f, w);
        load_like<WT, K>(A.b, c, A.cols, 0.0f, b);
#pragma unroll
        for (int k = 0; k < K; ++k) w[k] = __builtin_fmaf((f[k] - mean) * rstd, w[k], b[k]);
        stream_vec<DT>(y, c, A.cols, w);
    }
}

// Rows that no register file holds: read three times (the second and third time mostly out of the L2).
template <int DT, int WT>
__global__ __launch_bounds__(1024) void k_norm_long(NormArgs A)
{
    constexpr int K = kLane<DT>, T = 1024;
    __shared__ float part[2][2 * T / kWave];
    const int64_t row = block_index();
    if (row >= A.rows) return;
    const void* x = at<DT>(A.x, row * A.cols);
    float sum = 0.0f, sq = 0.0f, none = 0.0f, v[K];
    for (int64_t c = (int64_t)threadIdx.x * K; c < A.cols; c += T * K) {
        load_vec<DT>(x, c, A.cols, v);
#pragma unroll
        for (int k = 0; k < K; ++k) sum += v[k];
    }
    block_sum2<T>(sum, none, part[0], threadIdx.x);
    const float mean = sum / (float)A.cols;
    for (int64_t c = (int64_t)threadIdx.x * K; c < A.cols; c += T * K) {
        load_vec<DT>(x, c, A.cols, v);
#pragma unroll
        for (int k = 0; k < K; ++k)
            if (c + k < A.cols) sq = __builtin_fmaf(v[k] - mean, v[k] - mean, sq);
    }
    block_sum2<T>(sq, none, part[1], threadIdx.x);
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
        stream_vec<DT>(y, c, A.cols, v);
    }
}

// dx and this workgroup's partial sums of dw and db: T lanes, T / G rows at a time, every gridDim.x-th of them.  The next
// rows are on their way while these are worked on (but in workgroups of 1024 lanes, which have no registers for
// it, nor for the weights).  ONCE: streamed past the caches, for x and g that are larger than those (65536 x 4096
// BF16 283 -> 269 us, 16384 x 8192 153 -> 146; 4096 x 2048, whose x and g may be in them, 16 -> 18).
template <int DT, int WT, int G, int NV, int T, bool ONCE>
__global__ __launch_bounds__(T) void k_norm_back(NormArgs A)
{
    constexpr int K = kLane<DT>, R = T / G;
    constexpr bool AHEAD = T < 1024;
    __shared__ float part[2][R][G > kWave ? 2 * G / kWave : 1];
    __shared__ float cross[R > 1 ? R * G * K : 1];
    const int lane = threadIdx.x % G, sub = threadIdx.x / G;
    float w[NV][K], dw[NV][K], db[NV][K];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        if (AHEAD) load_like<WT, K>(A.w, (int64_t)(i * G + lane) * K, A.cols, 1.0f, w[i]);
#pragma unroll
        for (int k = 0; k < K; ++k) dw[i][k] = db[i][k] = 0.0f;
    }
    const float inv = 1.0f / (float)A.cols;
    const int64_t step = (int64_t)gridDim.x * R;
    raw16 xr[NV], gr[NV];
    float mean = 0.0f, rstd = 0.0f;
    auto read = [&](int64_t r) {   // past the last row: zeros, which add nothing
        const int64_t n = r < A.rows ? A.cols : 0;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            xr[i] = load_vec_raw<DT, ONCE>(at<DT>(A.x, r * A.cols), (int64_t)(i * G + lane) * K, n);
            gr[i] = load_vec_raw<DT, ONCE>(at<DT>(A.g, r * A.cols), (int64_t)(i * G + lane) * K, n);
        }
        mean = n ? A.stats[2 * r] : 0.0f;
        rstd = n ? A.stats[2 * r + 1] : 0.0f;
    };
    int64_t first = (int64_t)blockIdx.x * R;   // of the rows taken at a time: the same turns for all lanes
    if (AHEAD && first < A.rows) read(first + sub);
    for (int turn = 0; first < A.rows; first += step, turn ^= 1) {
        const int64_t row = first + sub;
        if (!AHEAD) read(row);
        const float scale = rstd;
        float x[NV][K], g[NV][K];
        float c1 = 0.0f, c2 = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            to_floats<DT>(xr[i], x[i]);
            to_floats<DT>(gr[i], g[i]);
            if (!AHEAD) load_like<WT, K>(A.w, (int64_t)(i * G + lane) * K, A.cols, 1.0f, w[i]);
#pragma unroll
            for (int k = 0; k < K; ++k) {
                x[i][k] = (x[i][k] - mean) * scale;
                dw[i][k] = __builtin_fmaf(g[i][k], x[i][k], dw[i][k]);
                db[i][k] += g[i][k];
                g[i][k] *= w[i][k];
                c1 += g[i][k];
                c2 = __builtin_fmaf(g[i][k], x[i][k], c2);
            }
        }
        if (AHEAD && first + step < A.rows) read(row + step);
        if (A.y) {
            block_sum2<G>(c1, c2, part[turn][sub], lane);
            if (row >= A.rows) continue;
            c1 *= inv;
            c2 *= inv;
            void* dx = at<DT>(A.y, row * A.cols);
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int64_t c = (int64_t)(i * G + lane) * K;
                if (c >= A.cols) break;
#pragma unroll
                for (int k = 0; k < K; ++k) g[i][k] = scale * (g[i][k] - c1 - x[i][k] * c2);
                stream_vec<DT>(dx, c, A.cols, g[i]);
            }
        }
    }
    if (!A.dw && !A.db) return;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int64_t c = (int64_t)(i * G + lane) * K;
#pragma unroll
        for (int d = R / 2; d; d /= 2) {   // the rows' sums, a tree
            __syncthreads();
            if (sub >= d && sub < 2 * d)
#pragma unroll
                for (int k = 0; k < K; ++k) {
                    cross[((sub - d) * 2 * K + k) * G + lane] = dw[i][k];
                    cross[((sub - d) * 2 * K + K + k) * G + lane] = db[i][k];
                }
            __syncthreads();
            if (sub < d)
#pragma unroll
                for (int k = 0; k < K; ++k) {
                    dw[i][k] += cross[(sub * 2 * K + k) * G + lane];
                    db[i][k] += cross[(sub * 2 * K + K + k) * G + lane];
                }
        }
        if (sub > 0 || c >= A.cols) continue;
        if (gridDim.x == 1) {   // the only workgroup: its sums are the gradients
            if (A.dw) store_like<WT, K>(A.dw, c, A.cols, dw[i]);
            if (A.db) store_like<WT, K>(A.db, c, A.cols, db[i]);
        } else {
            float* out = A.part + (int64_t)blockIdx.x * 2 * A.cols;
            store_like<DT_F32, K>(out, c, A.cols, dw[i]);
            store_like<DT_F32, K>(out + A.cols, c, A.cols, db[i]);
        }
    }
}

// The same for rows that no register file holds: dx a row a workgroup, reading the row twice ...
template <int DT, int WT>
__global__ __launch_bounds__(1024) void k_norm_back_long(NormArgs A)
{
    constexpr int K = kLane<DT>, T = 1024;
    __shared__ float part[2][2 * T / kWave];
    const int64_t row = block_index();
    if (row >= A.rows) return;
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
    block_sum2<T>(c1, c2, part[0], threadIdx.x);
    c1 /= (float)A.cols;
    c2 /= (float)A.cols;
    void* dx = at<DT>(A.y, row * A.cols);
    for (int64_t c = (int64_t)threadIdx.x * K; c < A.cols; c += T * K) {
        load_vec<DT>(xr, c, A.cols, x);
        load_vec<DT>(gr, c, A.cols, g);
        load_like<WT, K>(A.w, c, A.cols, 1.0f, w);
#pragma unroll
        for (int k = 0; k < K; ++k) g[k] = rstd * (g[k] * w[k] - c1 - (x[k] - mean) * rstd * c2);
        stream_vec<DT>(dx, c, A.cols, g);
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

// The P partial sums of 64 columns a workgroup: 64 lanes of 4 columns each take every 64th, then their sums in order.
template <int WT>
__global__ __launch_bounds__(1024) void k_norm_sums(NormArgs A, int32_t parts)
{
    constexpr int L = 64;
    __shared__ float sums[L][64 + 4];
    const int col = (threadIdx.x & 15) * 4, at_row = threadIdx.x >> 4;
    const int64_t c0 = (int64_t)blockIdx.x * 64;   // of 2 cols: dw's, then db's
    float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (c0 + col < 2 * A.cols) {
#pragma unroll 4
        for (int p = at_row; p < parts; p += L) {
            float x[4];
            load_vec<DT_F32>(A.part + (int64_t)p * 2 * A.cols, c0 + col, 2 * A.cols, x);
#pragma unroll
            for (int k = 0; k < 4; ++k) s[k] += x[k];
        }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) sums[at_row][col + k] = s[k];
    __syncthreads();
    float some = 0.0f;   // sixteen at a time first
    const int g = threadIdx.x >> 6, cc = threadIdx.x & 63;
    if (g < L / 16)
#pragma unroll
        for (int i = 0; i < 16; ++i) some += sums[16 * g + i][cc];
    __syncthreads();
    if (g < L / 16) sums[g][cc] = some;
    __syncthreads();
    const int64_t c = c0 + threadIdx.x;
    if (threadIdx.x < 64 && c < 2 * A.cols) {
        float all = 0.0f;
#pragma unroll
        for (int i = 0; i < L / 16; ++i) all += sums[i][threadIdx.x];
        void* out = c < A.cols ? A.dw : A.db;
        if (out) put<WT>(out, c < A.cols ? c : c - A.cols, all);
    }
}

constexpr int64_t kNormCached = (int64_t)128 << 20;   // x or g of this many bytes: both fill the 256 MB before the memory

static bool type_ok(int32_t t) { return t == ADAMBRIDGE_DT_F32 || t == ADAMBRIDGE_DT_BF16; }

// Lanes a row (0: the long form), values a lane, lanes of a workgroup.
struct Shape {
    int lanes, values, group;
};

// A row of up to 1024 columns is a part of a wavefront's or a wavefront's, a wider one a workgroup's.  Measured on MI355X in BF16,
// us, beside one of fewer lanes with more values: 4096 columns, 256 lanes or 64: 64 rows 3.8 / 6.7, 2048 rows 8.5 / 10.5, 65536
// rows 187 / 187; 2048 columns, 256 or 64: 512 rows 3.7 / 4.7, 1024 rows 4.6 / 5.0, 2048 rows 6.0 / 5.6, 65536 rows 115 / 92; 8192
// columns, 512 or 256: 64 rows 4.2 / 4.9, 2048 rows 14.3 / 14.7, 16384 rows 99 / 96; 16384 columns, 1024 or 512: 64 rows 5.0 /
// 5.6, 1024 rows 15.0 / 14.6, 8192 rows 106 / 100.
static Shape norm_shape(int64_t rows, int64_t cols)
{
    if (cols <= 64) return {8, 8, 256};
    if (cols <= 128) return {16, 8, 256};
    if (cols <= 256) return {32, 8, 256};
    if (cols <= 512) return {64, 8, 256};
    if (cols <= 1024) return {64, 16, 256};
    const bool few = rows < 2048;
    if (cols <= 2048) return few ? Shape{256, 8, 256} : Shape{64, 32, 256};
    if (cols <= 4096) return {256, 16, 256};
    if (cols <= 8192) return few ? Shape{512, 16, 512} : Shape{256, 32, 256};
    if (cols <= 16384) return few ? Shape{1024, 16, 1024} : Shape{512, 32, 512};
    return {0, 0, 0};
}

// Backward a lane holds five values a column and the next row's two: fewer columns a lane (2048 columns, 256 lanes or 64 with
// four times the values: 512 rows 8.0 / 18.6 us, 65536 rows 145 / 217).
static Shape norm_back_shape(int64_t cols)
{
    if (cols <= 64) return {8, 8, 512};
    if (cols <= 128) return {16, 8, 512};
    if (cols <= 256) return {32, 8, 512};
    if (cols <= 512) return {64, 8, 512};
    if (cols <= 1024) return {64, 16, 512};
    if (cols <= 2048) return {256, 8, 512};
    if (cols <= 4096) return {256, 16, 512};
    if (cols <= 8192) return {512, 16, 512};
    if (cols <= 16384) return {1024, 16, 1024};
    return {0, 0, 0};
}

// Workgroups of the backward pass, each with its partial sums: one a CU, of two turns at least (65536 x 4096 BF16: 287 us; 512
// workgroups 294, 768 325 and 1024 350, as the partial sums grow and more rows compete).  Of the long form 1024 in all, each of
// 2048 columns or 1024, for the same reason (2048 x 40000 BF16: 199 us; 512 of them 231, 2048 203, 256 a strip of columns 239).
static int norm_parts(int64_t rows, int64_t cols)
{
    const Shape s = norm_back_shape(cols);
    const int64_t at_a_time = s.lanes ? s.group / s.lanes : 1, most = s.lanes ? 256 : std::min<int64_t>(256, 1024 / ((cols + 2047) / 2048));
    return (int)std::max<int64_t>(1, std::min<int64_t>(most, (rows + at_a_time * 2 - 1) / (at_a_time * 2)));
}

template <int DT, int WT>
static void launch_norm(const NormArgs& A, bool back, int parts)
{
    constexpr int K = kLane<DT>;
    const Shape s = back ? norm_back_shape(A.cols) : norm_shape(A.rows, A.cols);
#define ABH_NORM(G, N)                                                                                                  \
    if (!back && s.lanes == G && s.values == N) {                                                                       \
        constexpr int R = kNormThreads<G> / G;                                                                          \
        hipLaunchKernelGGL((k_norm<DT, WT, G, N / K>), block_grid((A.rows + R - 1) / R), dim3(kNormThreads<G>), 0, t_stream, A); \
        return;                                                                                                         \
    }
    ABH_NORM(8, 8) ABH_NORM(16, 8) ABH_NORM(32, 8) ABH_NORM(64, 8) ABH_NORM(64, 16) ABH_NORM(64, 32) ABH_NORM(256, 8) ABH_NORM(256, 16) ABH_NORM(256, 32)
    ABH_NORM(512, 16) ABH_NORM(512, 32) ABH_NORM(1024, 16)
#undef ABH_NORM
#define ABH_NORM_BACK(G, N, T)                                                                                          \
    if (back && s.lanes == G && s.values == N && s.group == T) {                                                        \
        if (A.rows * A.cols * kSize<DT> > kNormCached)                                                                  \
            hipLaunchKernelGGL((k_norm_back<DT, WT, G, N / K, T, true>), dim3(parts), dim3(T), 0, t_stream, A);          \
        else                                                                                                            \
            hipLaunchKernelGGL((k_norm_back<DT, WT, G, N / K, T, false>), dim3(parts), dim3(T), 0, t_stream, A);         \
        return;                                                                                                         \
    }
    ABH_NORM_BACK(8, 8, 512) ABH_NORM_BACK(16, 8, 512) ABH_NORM_BACK(32, 8, 512) ABH_NORM_BACK(64, 8, 512) ABH_NORM_BACK(64, 16, 512) ABH_NORM_BACK(256, 8, 512) ABH_NORM_BACK(256, 16, 512)
    ABH_NORM_BACK(512, 16, 512) ABH_NORM_BACK(1024, 16, 1024)
#undef ABH_NORM_BACK
    if (!back) {
        hipLaunchKernelGGL((k_norm_long<DT, WT>), block_grid(A.rows), dim3(1024), 0, t_stream, A);
        return;
    }
    if (A.y) hipLaunchKernelGGL((k_norm_back_long<DT, WT>), block_grid(A.rows), dim3(1024), 0, t_stream, A);
    if (A.dw || A.db)
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
    const NormArgs A{x, nullptr, weight, bias, y, stats, nullptr, nullptr, nullptr, rows, cols, eps};
    norm_by_type(A, dtype, w_dtype, false, 0);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? 0 : hip_fail(e, "hipLaunchKernelGGL (layer norm)");
}

ADAMBRIDGE_API int64_t adambridge_layer_norm_work(int64_t rows, int64_t cols, int32_t dtype)
{
    if (rows < 1 || cols < 1 || rows > kNormMost || cols > kNormMost) return ADAMBRIDGE_EBADN;
    if (!type_ok(dtype)) return ADAMBRIDGE_EMVDTYPE;
    return (int64_t)norm_parts(rows, cols) * 2 * cols * 4;
}

ADAMBRIDGE_API int adambridge_layer_norm_backward(const void* gout, const void* x, int32_t dtype, const void* weight,
                                                  int32_t w_dtype, const float* stats, int64_t rows, int64_t cols, void* dx,
                                                  void* dweight, void* dbias, void* work)
{
    if (rows < 1 || cols < 1 || rows > kNormMost || cols > kNormMost) return ADAMBRIDGE_EBADN;
    if (!type_ok(dtype) || !type_ok(w_dtype)) return ADAMBRIDGE_EMVDTYPE;
    const bool sums = dweight || dbias;
    if (!gout || !x || !stats || (sums && !work)) return ADAMBRIDGE_ENULL;
    if (sums && (uintptr_t)work % 4) return ADAMBRIDGE_EALIGN;
    if (!dx && !sums) return 0;
    const int parts = norm_parts(rows, cols);
    const NormArgs A{x, gout, weight, nullptr, dx, const_cast<float*>(stats), dweight, dbias, static_cast<float*>(work),
                     rows, cols, 0.0f};
    norm_by_type(A, dtype, w_dtype, true, parts);
    if (sums && (parts > 1 || !norm_back_shape(cols).lanes)) {
        const dim3 grid((unsigned)((2 * cols + 63) / 64));
        if (w_dtype == ADAMBRIDGE_DT_BF16) hipLaunchKernelGGL((k_norm_sums<DT_BF16>), grid, dim3(1024), 0, t_stream, A, parts);
        else hipLaunchKernelGGL((k_norm_sums<DT_F32>), grid, dim3(1024), 0, t_stream, A, parts);
    }
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? 0 : hip_fail(e, "hipLaunchKernelGGL (layer norm's gradient)");
}

}  // extern "C"
