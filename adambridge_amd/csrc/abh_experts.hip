// abh_experts.hip -- matrix products grouped by expert: rows sorted by expert, each expert's with its own weights.
//
//   y[r] = W[e] x[r]          (W: experts x n x k, as stacked Linear weights)
//   dx[r] = W[e]^T g[r]
//   dW[e] = sum over e's rows of g[r] x[r]^T
//
// for the rows ends[e - 1] <= r < ends[e] of each expert e; rows from the last end on are no expert's and give
// zeros.  The ends are read on the device: the host knows the number of rows only, so a launch has a
// workgroup for every tile there could be (an expert's last tile may be partial) and a workgroup finds its
// expert and tile from the ends; those beyond the last tile leave at once.
//
// All three are C[i, j] = sum over k of A[i, k] B[j, k], with the sum along a row of an operand (the operand is
// "long" in k) or across its rows.

#include <hip/hip_runtime.h>

#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "../../include/adambridge_hip.h"
#include "abh_device.hpp"
#include "abh_host.hpp"
#include "abh_tiles.hpp"

namespace abh {

constexpr int kExpertsMost = 4096;
enum { MODE_Y = 0, MODE_DX = 1, MODE_DW = 2 };

struct ExpertArgs {
    const void* a;      // x, g, g
    const void* b;      // W, W, x
    void* c;            // y, dx, dW
    const int32_t* ends;
    int32_t rows, experts;
    int32_t ni, nj;     // MODE_DW: C's rows (n); columns of C
    int32_t len;        // the sum's length, but for MODE_DW
    int32_t tiles_i, tiles_j;
    int32_t splits;     // parts of a sum (MODE_DW: of an expert's rows), each with a result of its own ...
    float* part;        // ... splits x the result
};

// Rows lo .. hi of expert e0 + the lane's number (expert `experts`: the rows that are no expert's), of 64 experts at a time
// from 0 on; `before` (0 at first) is the last end before them.  An end outside 0 .. rows, or below one before it, is the
// nearest that is not: whatever the ends are, no two experts share a row, and the experts' tiles are no more than
// the launch reckons with.
__device__ __forceinline__ void wave_rows(const ExpertArgs& A, int e0, int& before, int& lo, int& hi)
{
    const int lane = threadIdx.x & 63, e = e0 + lane;
    lo = e > 0 && e <= A.experts ? A.ends[e - 1] : e == 0 ? 0 : A.rows;
    hi = e < A.experts ? A.ends[e] : A.rows;
    lo = lo < 0 ? 0 : lo > A.rows ? A.rows : lo;
    hi = hi < 0 ? 0 : hi > A.rows ? A.rows : hi;
    if (__builtin_amdgcn_ballot_w64(hi < lo || lo < before)) {   // the largest so far
        hi = hi > before ? hi : before;
#pragma unroll
        for (int d = 1; d < kWave; d *= 2) {
            const int y = __shfl_up(hi, d);
            if (lane >= d && y > hi) hi = y;
        }
        lo = __shfl_up(hi, 1);
        if (lane == 0) lo = before;
    }
    before = __builtin_amdgcn_readlane(hi, kWave - 1);
}

struct Tile {
    int e, lo, hi, ti, tj;
    int split, splits;   // which part of its sum, of how many
    int rest;            // which of the split tiles
};

// The tiles of BM rows that all experts' rows make.  Every wavefront counts them for itself.
template <int BM>
__device__ __forceinline__ int count_row_tiles(const ExpertArgs& A)
{
    int total = 0, last = 0;
    for (int e0 = 0; e0 <= A.experts; e0 += kWave) {
        int lo, hi;
        wave_rows(A, e0, last, lo, hi);
        total += group_reduce<kWave>((hi - lo + BM - 1) / BM, [](int a, int b) { return a + b; });
    }
    return scalar(total) * A.tiles_j;
}

// Tile idx of them, expert by expert, kGroupTiles row tiles at a time down the columns.
template <int BM>
__device__ __forceinline__ bool locate_row_tile(const ExpertArgs& A, int idx, Tile& t)
{
    const int lane = threadIdx.x & 63, q = idx / A.tiles_j;
    int before = 0, last = 0;
    for (int e0 = 0; e0 <= A.experts; e0 += kWave) {
        int lo, hi;
        wave_rows(A, e0, last, lo, hi);
        const int n = (hi - lo + BM - 1) / BM;
        int s = n;
#pragma unroll
        for (int d = 1; d < kWave; d *= 2) {
            const int y = __shfl_up(s, d);
            if (lane >= d) s += y;
        }
        const uint64_t past = __builtin_amdgcn_ballot_w64(before + s > q);
        if (past) {
            const int w = __builtin_ctzll(past);
            t.e = e0 + w;
            t.lo = __builtin_amdgcn_readlane(lo, w);
            t.hi = __builtin_amdgcn_readlane(hi, w);
            const int mine = __builtin_amdgcn_readlane(n, w);
            idx -= (before + __builtin_amdgcn_readlane(s, w) - mine) * A.tiles_j;
            const int g = idx / (kGroupTiles * A.tiles_j), first = g * kGroupTiles;
            const int wide = mine - first < kGroupTiles ? mine - first : kGroupTiles;
            const int r = idx - first * A.tiles_j;
            t.ti = scalar(first + r % wide);
            t.tj = scalar(r / wide);
            return true;
        }
        before += __builtin_amdgcn_readlane(s, kWave - 1);
    }
    return false;
}

// This workgroup's row tile: consecutive tiles go to one XCD, whose L2 then holds an expert's weights for the tiles of its
// rows.
template <int BM>
__device__ __forceinline__ bool find_row_tile(const ExpertArgs& A, Tile& t)
{
    const int items = count_row_tiles<BM>(A) * A.splits, per = (items + kXcd - 1) / kXcd;
    const int block = (int)block_index(), slot = block / kXcd, item = block % kXcd * per + slot;
    const int idx = scalar(item / A.splits);
    t.split = scalar(item - idx * A.splits);
    t.splits = A.splits;
    t.rest = 0;
    return slot < per && item < items && locate_row_tile<BM>(A, idx, t);
}

// The same where a CU has one workgroup: whole rounds of kCus tiles, spread over the XCDs, and the rest of them over the XCDs
// again.  A short rest would hold all CUs for a whole tile's time: it is cut along the sum into as many parts as fill
// them (at the price of 512 KB of partial sums a part, written and added up by another kernel, about 30 us, which is 64 steps).
constexpr int kCus = 256, kMostRest = 128, kMostParts = 16;

struct Rounds {
    int full, rest, splits;
};

template <int BM, int BK>
__device__ __forceinline__ Rounds rounds_of(const ExpertArgs& A)
{
    const int tiles = count_row_tiles<BM>(A), steps = (A.len + BK - 1) / BK;
    Rounds r{tiles / kCus * kCus, tiles % kCus, 1};
    if (A.part && r.rest > 0 && r.rest <= kMostRest) {
        const int fit = kCus / r.rest < kMostParts ? kCus / r.rest : kMostParts;
        if (steps / fit * (fit - 1) >= 64) r.splits = fit;
    }
    return r;
}

template <int BM, int BK>
__device__ __forceinline__ bool find_round_tile(const ExpertArgs& A, Tile& t)
{
    const Rounds r = rounds_of<BM, BK>(A);
    const int b = (int)block_index();
    int idx;
    t.split = t.rest = 0;
    t.splits = 1;
    if (b < r.full) {
        idx = b % kXcd * (r.full / kXcd) + b / kXcd;
    } else {
        const int items = r.rest * r.splits, per = (items + kXcd - 1) / kXcd, slot = (b - r.full) / kXcd;
        const int item = (b - r.full) % kXcd * per + slot;
        if (slot >= per || item >= items) return false;
        t.rest = scalar(item / r.splits);
        t.split = scalar(item - t.rest * r.splits);
        t.splits = scalar(r.splits);
        idx = r.full + t.rest;
    }
    return locate_row_tile<BM>(A, idx, t);
}

// A tile of dW (and of one of the parts of its expert's rows).  The XCDs share every expert's tiles evenly, because
// experts differ in rows and so in work.
__device__ __forceinline__ bool find_weight_tile(const ExpertArgs& A, Tile& t)
{
    const int an = A.tiles_i * A.tiles_j, per = (an + kXcd - 1) / kXcd;
    const int block = (int)block_index(), slot = block / kXcd, turn = slot / per;
    if (turn >= A.experts * A.splits) return false;
    const int local = (block % kXcd + turn) % kXcd * per + slot - turn * per;   // the first XCD changes: an may be below 8
    if (local >= an) return false;
    t.e = turn / A.splits;
    t.split = turn - t.e * A.splits;
    // an XCD's tiles near a square: 6 of them as 2 x 3 read 1.56 GB in all, as 6 x 1 1.94 (64 experts 1536 x 2048: 424 us, 437)
    const int high = per < 4 ? 1 : per < 8 ? 2 : per < 32 ? 4 : kGroupTiles;
    const int g = local / (high * A.tiles_j), first = g * high;
    const int wide = A.tiles_i - first < high ? A.tiles_i - first : high;
    const int r = local - first * A.tiles_j;
    t.ti = scalar(first + r % wide);
    t.tj = scalar(r / wide);
    t.e = scalar(t.e);
    t.split = scalar(t.split);
    t.splits = A.splits;
    int lo = 0, hi = A.ends[t.e];   // as wave_rows has them
    for (int e = threadIdx.x & 63; e < t.e; e += kWave) lo = lo > A.ends[e] ? lo : A.ends[e];
    lo = scalar(group_reduce<kWave>(lo, [](int a, int b) { return a > b ? a : b; }));
    lo = lo < A.rows ? lo : A.rows;
    hi = scalar(hi < lo ? lo : hi < A.rows ? hi : A.rows);
    const int chunk = ((hi - lo + A.splits - 1) / A.splits + 31) / 32 * 32;   // whole steps of 32 rows
    t.lo = scalar(chunk * t.split < hi - lo ? lo + chunk * t.split : hi);
    t.hi = scalar(t.lo + chunk < hi ? t.lo + chunk : hi);
    return true;
}

// Where this part's sums go: FP32, rows of nj, those of the tile's expert.
template <int MODE>
__device__ __forceinline__ float* part_of(const ExpertArgs& A, const Tile& t)
{
    const int64_t row = MODE == MODE_DW ? ((int64_t)t.split * A.experts + t.e) * A.ni : (int64_t)t.split * A.rows + t.lo;
    return A.part + row * A.nj;
}

// c = the parts' sums, in order, rounded once.
template <int DT>
__global__ __launch_bounds__(256) void k_experts_sum(const float* part, int64_t size, int32_t splits, void* c)
{
    const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
    if (i >= size) return;
    float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int p = 0; p < splits; ++p) {
        float x[4];
        load_vec<DT_F32>(part + p * size, i, size, x);
#pragma unroll
        for (int k = 0; k < 4; ++k) s[k] += x[k];
    }
#pragma unroll
    for (int k = 0; k < 4; ++k)
        if (i + k < size) put<DT>(c, i + k, s[k]);
}

// ------------------------------------------------------------- any sizes, any alignment
//
// For rows shorter than a piece of 16 bytes and sizes beyond 2^20; right for all of them.
// Tiles of 128 x 128, four wavefronts of 64 x 64, 32 terms a step; the next step's values are loaded to registers while
// the one before is multiplied.  LDS rows of 32 terms are padded by 16 bytes, so that the 16-byte reads of 16
// rows fall on different banks.  A lane's values of k come 16 bytes at a time: the matrix instructions take
// whatever order of k both operands share.  The product is taken transposed (B's rows first), which leaves a
// lane four neighbouring columns of a row of C.

constexpr int kTile = 128, kStep = 32, kMmThreads2 = 256;

template <int DT>
constexpr int kPitch = kStep + 16 / kSize<DT>;
template <int DT>
using Element = typename std::conditional<DT == DT_BF16, uint16_t, float>::type;

// One operand's tile: rows r0 .. limit of the tile's 128 and terms s0 .. s0 + 31 of len, zeros elsewhere.
template <int DT, bool LONG>
struct Stage {
    static constexpr int V = kLane<DT>, N = kTile * kStep / V / kMmThreads2;
    raw16 r[N];
    // lane's chunk c: (row, k) of its first value
    static __device__ __forceinline__ void where(int c, int& row, int& k)
    {
        const int i = c * kMmThreads2 + (int)threadIdx.x;
        if constexpr (LONG) {
            row = i / (kStep / V);
            k = i % (kStep / V) * V;
        } else {   // 8 neighbouring chunks of rows by 8 terms a wavefront: 128 bytes a load, few LDS conflicts
            const int q = i / 64, l = i % 64;
            row = (q % (kTile / V / 8) * 8 + l % 8) * V;
            k = q / (kTile / V / 8) * 8 + l / 8;
        }
    }
    __device__ __forceinline__ void load(const uint8_t* base, int64_t pitch, int limit, int s0, int len)
    {
#pragma unroll
        for (int c = 0; c < N; ++c) {
            int row, k;
            where(c, row, k);
            k += s0;
            float v[V];
            if constexpr (LONG) {
                if (row < limit && k + V <= len) {
                    r[c] = load_raw<DT>(base, (int64_t)row * pitch + k);
                    continue;
                }
#pragma unroll
                for (int j = 0; j < V; ++j) v[j] = row < limit && k + j < len ? get<DT>(base, (int64_t)row * pitch + k + j) : 0.0f;
            } else {
                if (k < len && row + V <= limit) {
                    r[c] = load_raw<DT>(base, (int64_t)k * pitch + row);
                    continue;
                }
#pragma unroll
                for (int j = 0; j < V; ++j) v[j] = k < len && row + j < limit ? get<DT>(base, (int64_t)k * pitch + row + j) : 0.0f;
            }
            r[c] = to_raw<DT>(v);   // exact: the values are of this type
        }
    }
    __device__ __forceinline__ void store(Element<DT>* lds) const
    {
#pragma unroll
        for (int c = 0; c < N; ++c) {
            int row, k;
            where(c, row, k);
            if constexpr (LONG) {
                *reinterpret_cast<raw16*>(lds + row * kPitch<DT> + k) = r[c];
            } else {
                const uint32_t u[4] = {r[c].x, r[c].y, r[c].z, r[c].w};
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    if constexpr (DT == DT_BF16) lds[(row + j) * kPitch<DT> + k] = (uint16_t)(u[j / 2] >> (16 * (j & 1)));
                    else lds[(row + j) * kPitch<DT> + k] = bitsf(u[j]);
                }
            }
        }
    }
};

// CHAINS: sums of more than kF32Chain steps in FP32.  (Two sets of sums leave two workgroups a CU of three: 65000 rows 3 -> 1000
// 186 us with them, 168 without.)
template <int DT, int MODE, bool CHAINS>
__global__ __launch_bounds__(kMmThreads2, 2) void k_experts_any(ExpertArgs A)
{
    constexpr bool ALONG = MODE != MODE_DW, BLONG = MODE == MODE_Y;
    __shared__ __attribute__((aligned(16))) Element<DT> la[kTile * kPitch<DT>], lb[kTile * kPitch<DT>];
    Tile t;
    if constexpr (MODE == MODE_DW) {
        if (!find_weight_tile(A, t)) return;
    } else {
        if (!find_row_tile<kTile>(A, t)) return;
    }
    const int i0 = t.ti * kTile, j0 = t.tj * kTile;
    const int limit_i = MODE == MODE_DW ? A.ni - i0 : t.hi - t.lo - i0, limit_j = A.nj - j0;
    const int len = MODE == MODE_DW ? t.hi - t.lo : t.e < A.experts ? A.len : 0;
    const uint8_t *pa, *pb;
    int64_t pitch_a, pitch_b;
    if constexpr (MODE == MODE_DW) {
        pitch_a = A.ni;
        pitch_b = A.nj;
        pa = at<DT>(A.a, (int64_t)t.lo * pitch_a + i0);
        pb = at<DT>(A.b, (int64_t)t.lo * pitch_b + j0);
    } else {
        pitch_a = A.len;
        pa = at<DT>(A.a, (int64_t)(t.lo + i0) * pitch_a);
        pitch_b = MODE == MODE_Y ? A.len : A.nj;
        const int64_t of_e = (int64_t)(t.e < A.experts ? t.e : 0) * A.len * A.nj;
        pb = at<DT>(A.b, of_e + (MODE == MODE_Y ? (int64_t)j0 * pitch_b : j0));
    }
    const int lane = threadIdx.x & 63, wave = threadIdx.x / kWave, col = lane & 15, quarter = lane >> 4;
    const int wi = (wave & 1) * 64, wj = (wave >> 1) * 64;
    const int live_i = scalar(limit_i - wi + 15) / 16, live_j = scalar(limit_j - wj + 15) / 16;   // FP32: the 16 x 16 that have results
    mm_f32x4 acc[4][4], sum[4][4];   // sum: CHAINS'
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = sum[i][j] = mm_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    Stage<DT, ALONG> sa;
    Stage<DT, BLONG> sb;
    if (len > 0) {
        sa.load(pa, pitch_a, limit_i, 0, len);
        sb.load(pb, pitch_b, limit_j, 0, len);
    }
    for (int s = 0; s < len; s += kStep) {
        sa.store(la);
        sb.store(lb);
        __syncthreads();
        if (s + kStep < len) {
            sa.load(pa, pitch_a, limit_i, s + kStep, len);
            sb.load(pb, pitch_b, limit_j, s + kStep, len);
        }
        if constexpr (DT == DT_BF16) {
            mm_bf16x8 fa[4], fb[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                fa[i] = __builtin_bit_cast(mm_bf16x8, *reinterpret_cast<const raw16*>(la + (wi + 16 * i + col) * kPitch<DT> + 8 * quarter));
                fb[i] = __builtin_bit_cast(mm_bf16x8, *reinterpret_cast<const raw16*>(lb + (wj + 16 * i + col) * kPitch<DT> + 8 * quarter));
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fb[j], fa[i], acc[i][j], 0, 0, 0);
        } else {
#pragma unroll 1
            for (int h = 0; h < kStep; h += 16) {
                mm_f32x4 fa[4], fb[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    fa[i] = *reinterpret_cast<const mm_f32x4*>(la + (wi + 16 * i + col) * kPitch<DT> + h + 4 * quarter);
                    fb[i] = *reinterpret_cast<const mm_f32x4*>(lb + (wj + 16 * i + col) * kPitch<DT> + h + 4 * quarter);
                }
#pragma unroll
                for (int q = 0; q < 4; ++q)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            if (i < live_i && j < live_j)
                                acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(fb[j][q], fa[i][q], acc[i][j], 0, 0, 0);
            }
            if (CHAINS && (s / kStep % kF32Chain == kF32Chain - 1 || s + kStep >= len)) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        sum[i][j] += acc[i][j];
                        acc[i][j] = mm_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
                    }
            }
        }
        __syncthreads();
    }
    uint8_t* out = MODE == MODE_DW ? at<DT>(A.c, ((int64_t)t.e * A.ni + i0) * A.nj + j0)
                                   : at<DT>(A.c, (int64_t)(t.lo + i0) * A.nj + j0);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int row = wi + 16 * i + col;
        if (row >= limit_i) continue;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int c = wj + 16 * j + 4 * quarter;
            const int64_t o = (int64_t)row * A.nj + c;
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (c + r < limit_j) put<DT>(out, o + r, CHAINS ? sum[i][j][r] : acc[i][j][r]);
        }
    }
}

// ---------------------------------------------------------------------------- few rows
//
// y of few rows is its experts' weights read once: no tile to share, so they go to the registers in 16-byte pieces,
// 16 columns of C a workgroup, whose four wavefronts split the sum and add their parts in order.  The rows are the
// matrix instruction's other side, 16 at a time (whatever their number costs nothing beside the weights) and up to
// 64 for one reading.  Any size and alignment; a workgroup finds the expert that is the blockIdx-th with rows.
//
// Measured on MI355X, 64 experts 1536 x 2048 in BF16 that are in no cache: 8 rows 10.8 us (4.65 TB/s of weights), 64 rows 40 us
// (5.19), 256 rows 69 us (5.29); FP32, 256 rows 135 us (5.42).  Bound by the reads on their way: 16 of a wavefront instead of 8
// take 12.1, eight wavefronts a workgroup 15.5 us for 8 rows.

constexpr int kFewColumns = 16, kFewWaves = 4, kFewAhead = 8;
template <int DT, bool EVEN>
__global__ __launch_bounds__(kFewWaves * kWave) void k_experts_few(ExpertArgs A)
{
    constexpr int V = kLane<DT>, STEP = 4 * V, CH = 4, U = kFewAhead, W = kFewWaves;
    __shared__ mm_f32x4 parts[W - 1][CH][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / kWave);
    const int col = lane & 15, quarter = lane >> 4;
    const int block = (int)block_index(), tj = block % A.tiles_j;
    int skip = block / A.tiles_j;
    int e = -1, lo = 0, hi = 0, last = 0;
    for (int e0 = 0; e0 <= A.experts; e0 += kWave) {
        int l, h;
        wave_rows(A, e0, last, l, h);
        const uint64_t with = __builtin_amdgcn_ballot_w64(h > l);
        const int count = __builtin_popcountll(with);
        if (skip < count) {
            const int before = __builtin_popcountll(with & (((uint64_t)1 << lane) - 1));
            const int at_lane = __builtin_ctzll(__builtin_amdgcn_ballot_w64(h > l && before == skip));
            e = e0 + at_lane;
            lo = __builtin_amdgcn_readlane(l, at_lane);
            hi = __builtin_amdgcn_readlane(h, at_lane);
            break;
        }
        skip -= count;
    }
    if (e < 0) return;
    const int steps = e < A.experts ? (A.len + STEP - 1) / STEP : 0;   // rows that are no expert's: zeros
    const int s0 = steps * wave / W, s1 = steps * (wave + 1) / W;
    const int j0 = tj * kFewColumns, columns = A.nj - j0 < kFewColumns ? A.nj - j0 : kFewColumns;
    const Pieces<DT, EVEN> w{at<DT>(A.b, ((int64_t)(e < A.experts ? e : 0) * A.nj + j0) * A.len), (uint32_t)(columns * A.len * kSize<DT>),
                             A.len, columns};
    const Pieces<DT, EVEN> x{at<DT>(A.a, (int64_t)lo * A.len), (uint32_t)((hi - lo) * A.len * kSize<DT>), A.len, hi - lo};
    for (int r0 = 0; r0 < hi - lo; r0 += 16 * CH) {
        mm_f32x4 acc[CH];
#pragma unroll
        for (int c = 0; c < CH; ++c) acc[c] = mm_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        for (int s = s0; s < s1; s += U) {
            raw16 wv[U];
#pragma unroll
            for (int u = 0; u < U; ++u) wv[u] = w.load(col, (s + u) * STEP + quarter * V, s + u < s1);
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                if (r0 + 16 * c >= hi - lo) break;
                raw16 xv[U];
#pragma unroll
                for (int u = 0; u < U; ++u) xv[u] = x.load(r0 + 16 * c + col, (s + u) * STEP + quarter * V, s + u < s1);
                mm_f32x4 some = DT == DT_BF16 ? acc[c] : mm_f32x4{0.0f, 0.0f, 0.0f, 0.0f};   // FP32: short chains of sums
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    if constexpr (DT == DT_BF16) {
                        some = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(mm_bf16x8, wv[u]),
                                                                       __builtin_bit_cast(mm_bf16x8, xv[u]), some, 0, 0, 0);
                    } else {
                        const mm_f32x4 wf = __builtin_bit_cast(mm_f32x4, wv[u]), xf = __builtin_bit_cast(mm_f32x4, xv[u]);
#pragma unroll
                        for (int q = 0; q < 4; ++q) some = __builtin_amdgcn_mfma_f32_16x16x4f32(wf[q], xf[q], some, 0, 0, 0);
                    }
                }
                if constexpr (DT == DT_BF16) acc[c] = some;
                else acc[c] += some;
            }
        }
        if (r0 > 0) __syncthreads();   // the parts before have been read
        if (wave > 0)
#pragma unroll
            for (int c = 0; c < CH; ++c)
                if (r0 + 16 * c < hi - lo) parts[wave - 1][c][lane] = acc[c];
        __syncthreads();
        if (wave > 0) continue;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            if (r0 + 16 * c >= hi - lo) break;
            const int row = r0 + 16 * c + col, j4 = j0 + 4 * quarter;
#pragma unroll
            for (int p = 0; p < W - 1; ++p) acc[c] += parts[p][c][lane];
            if (row >= hi - lo) continue;
            void* y = at<DT>(A.c, (int64_t)(lo + row) * A.nj);
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (j4 + r < A.nj) put<DT>(y, j4 + r, acc[c][r]);
        }
    }
}

// ------------------------------------------------------------- BF16 rows of whole 16-byte pieces
//
// Tiles of 256 x 256, eight wavefronts of 128 x 64 (2 x 4), 32 terms a step, four buffers of 32 KB in the LDS.  A step's
// tiles go from memory to the LDS past the registers, three steps ahead of the one that is multiplied; what lies
// outside an operand is out of its buffer's range and arrives as zeros.  A wavefront reads the fragments of its next
// 8 matrix products of 32 x 32 x 16 while the matrix cores work on these.
//
// Rows that are not whole 16-byte pieces go through the registers (StagedFeed): 8192 rows of 8 experts 2047 x 1999, a training
// pass 439 us, 2048 x 2000 308.
//
// Measured on MI355X, one expert, 8192^3: y 873 us (1259 TFLOP/s), dx 827 (1329), dW 821 (1339); the BLAS library's products
// 1501, 1228, 1152 TFLOP/s.  The matrix cores are busy 73% of the cycles, at 1.6 GHz of 2.4 (y of zeros: 750 us): power is the bound, and
// what takes stalls away alone gives the clock back (workgroups that go on to the next tile while the last one's
// results are stored, those stores beside the next loads: 0-3% slower).  Slower too: 64 terms a step with two buffers 891 (y),
// wavefronts of 128 x 128 (one a SIMD) 890, tiles of 128 x 256 with two workgroups a CU 1010, three buffers 989, a long operand's
// steps loaded two at a time, as whole lines of 128 bytes, 1-6%; five buffers change nothing.
//
// A long operand's tile is its rows by 64 bytes, a row's 16-byte pieces exchanged by the row, so that the reads of
// neighbouring rows meet different banks.  One across its rows is 32 terms by its rows, read transposed
// (ds_read_b64_tr_b16: 16 lanes take 4 terms x 16 values, a lane 4 terms of one value), its pieces exchanged in
// fours by the term mod 4: the 4 terms x 2 pairs of pieces of 32 lanes then cover the 256 bytes of all banks.

static_assert(LargeTile::BM == 256 && LargeTile::BN == 256 && SmallTile::BM == 128 && SmallTile::BN == 128, "plan_experts counts these");

// A tile in numbers: C's rows and columns from i0, j0 and how many there are, the operands' terms from k0 on.
struct Cut {
    Tile t;
    int i0, j0, limit_i, limit_j, k0, len, steps;
};

template <int MODE, class C>
__device__ __forceinline__ Cut cut_of(const ExpertArgs& A, const Tile& t)
{
    Cut u;
    u.t = t;
    u.i0 = t.ti * C::BM;
    u.j0 = t.tj * C::BN;
    u.limit_i = MODE == MODE_DW ? A.ni - u.i0 : t.hi - t.lo - u.i0;
    u.limit_j = A.nj - u.j0;
    u.len = MODE == MODE_DW ? t.hi - t.lo : t.e < A.experts ? A.len : 0;
    u.k0 = 0;
    if (MODE != MODE_DW && t.splits > 1 && u.len > 0) {
        const int all = (u.len + C::BK - 1) / C::BK;
        u.k0 = scalar(all * t.split / t.splits * C::BK);
        const int end = scalar(all * (t.split + 1) / t.splits * C::BK);
        u.len = (end < u.len ? end : u.len) - u.k0;
    }
    u.steps = (u.len + C::BK - 1) / C::BK;
    return u;
}

// Where the results of a wavefront's products go.
template <int MODE, class C, bool EVEN>
__device__ __forceinline__ void store_tile(const ExpertArgs& A, const Cut& u, const mm_f32x16 (&acc)[C::NI][C::NJ], int wi, int wj)
{
    const int lane = threadIdx.x & 63;
    if constexpr (MODE == MODE_DW || !C::ROUNDS) {
        if (A.splits > 1) {   // a part of the sums
            float* to = part_of<MODE>(A, u.t) + u.j0;
#pragma unroll
            for (int i = 0; i < C::NI; ++i) {
                const int row = u.i0 + wi + 32 * i + (lane & 31);
                if (row >= u.i0 + u.limit_i) continue;
#pragma unroll
                for (int j = 0; j < C::NJ; ++j)
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const float four[4] = {acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
                        store_like<DT_F32, 4>(to + (int64_t)row * A.nj, wj + 32 * j + 8 * q + 4 * (lane >> 5), u.limit_j, four);
                    }
            }
            return;
        }
    } else if constexpr (C::ROUNDS) {
        if (u.t.splits > 1) {   // a part of the sums of a tile
            float* to = A.part + ((int64_t)u.t.rest * u.t.splits + u.t.split) * C::BM * C::BN;
#pragma unroll
            for (int i = 0; i < C::NI; ++i)
#pragma unroll
                for (int j = 0; j < C::NJ; ++j)
#pragma unroll
                    for (int q = 0; q < 4; ++q)
                        *reinterpret_cast<mm_f32x4*>(to + (wi + 32 * i + (lane & 31)) * C::BN + wj + 32 * j + 8 * q + 4 * (lane >> 5)) =
                            mm_f32x4{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
            return;
        }
    }
    uint8_t* out = MODE == MODE_DW ? at<DT_BF16>(A.c, ((int64_t)u.t.e * A.ni + u.i0) * A.nj + u.j0)
                                   : at<DT_BF16>(A.c, (int64_t)(u.t.lo + u.i0) * A.nj + u.j0);
    store_bf16<C, EVEN>(out, A.nj, u.limit_i, u.limit_j, acc, wi, wj);
}

template <int MODE, class C, bool EVEN>
__global__ __launch_bounds__(C::T, C::OCC) void k_experts_fast(ExpertArgs A)
{
    constexpr bool ALONG = MODE != MODE_DW, BLONG = MODE == MODE_Y, ROUND = MODE != MODE_DW && C::ROUNDS;
    constexpr int BM = C::BM, BN = C::BN, BK = C::BK;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[C::NB * C::BYTES];
    Tile t;
    if constexpr (MODE == MODE_DW) {
        if (!find_weight_tile(A, t)) return;
    } else if constexpr (ROUND) {
        if (!find_round_tile<BM, BK>(A, t)) return;
    } else {
        if (!find_row_tile<BM>(A, t)) return;
    }
    const int wave = threadIdx.x / kWave;
    const int wi = wave / C::WJ * (BM / C::WI), wj = wave % C::WJ * (BN / C::WJ);   // a SIMD's two wavefronts: other rows each
    TileFeed<ALONG, BM, BK, C::W, EVEN> fa;
    TileFeed<BLONG, BN, BK, C::W, EVEN> fb;
    const Cut u = cut_of<MODE, C>(A, t);
    {
        // the operands' first values: of this expert's rows and weights
        const int64_t first_row = MODE == MODE_DW ? u.t.lo : u.t.lo + u.i0;
        const int pitch_a = MODE == MODE_DW ? A.ni : A.len, pitch_b = MODE == MODE_Y ? A.len : A.nj;
        const uint8_t* pa = at<DT_BF16>(A.a, first_row * pitch_a);
        const uint8_t* pb = MODE == MODE_DW ? at<DT_BF16>(A.b, (int64_t)u.t.lo * A.nj)
                                            : at<DT_BF16>(A.b, (int64_t)(u.t.e < A.experts ? u.t.e : 0) * A.len * A.nj);
        if (MODE == MODE_Y) pb = at<DT_BF16>(pb, (int64_t)u.j0 * A.len);
        if (MODE != MODE_DW) {
            pa = at<DT_BF16>(pa, u.k0);
            pb = at<DT_BF16>(pb, MODE == MODE_Y ? (int64_t)u.k0 : (int64_t)u.k0 * A.nj);
        }
        if constexpr (EVEN) {
            fa.start(MODE == MODE_DW ? pa + (int64_t)u.i0 * 2 : pa, pitch_a * 2, u.limit_i, u.len, (ALONG ? u.k0 : u.i0) * 2);
            fb.start(MODE == MODE_Y ? pb : pb + (int64_t)u.j0 * 2, pitch_b * 2, u.limit_j, u.len, (BLONG ? u.k0 : u.j0) * 2);
        } else {
            fa.start(pa, pitch_a, ALONG ? 0 : u.i0, ALONG ? u.limit_i : A.ni, u.len);
            fb.start(pb, pitch_b, BLONG ? 0 : u.j0, BLONG ? u.limit_j : A.nj, u.len);
        }
    }
    mm_f32x16 acc[C::NI][C::NJ];
    // an expert's last rows: no row of this wavefront
    if (!multiply_tile<C, ALONG, BLONG, EVEN>(lds, fa, fb, u.steps, wi, wj, wi < u.limit_i, acc)) return;
    store_tile<MODE, C, EVEN>(A, u, acc, wi, wj);
}

// C's tiles of the rest (find_round_tile) from their parts, in order: 16 rows of a tile a workgroup, 16 columns a lane.
template <class C>
__global__ __launch_bounds__(256) void k_experts_rest(ExpertArgs A)
{
    const Rounds r = rounds_of<C::BM, C::BK>(A);
    const int rest = (int)blockIdx.x / (C::BM / 16);
    Tile t;
    if (r.splits < 2 || rest >= r.rest || !locate_row_tile<C::BM>(A, r.full + rest, t)) return;
    const int row = (int)blockIdx.x % (C::BM / 16) * 16 + (int)threadIdx.x / 16, col = (int)threadIdx.x % 16 * (C::BN / 16);
    const int i = t.ti * C::BM + row, j = t.tj * C::BN + col;
    if (i >= t.hi - t.lo || j >= A.nj) return;
    const float* part = A.part + (int64_t)rest * r.splits * C::BM * C::BN + row * C::BN + col;
    float s[C::BN / 16];
#pragma unroll
    for (int k = 0; k < C::BN / 16; ++k) s[k] = 0.0f;
    for (int p = 0; p < r.splits; ++p)
#pragma unroll
        for (int k = 0; k < C::BN / 16; k += 4) {
            const mm_f32x4 x = *reinterpret_cast<const mm_f32x4*>(part + (int64_t)p * C::BM * C::BN + k);
#pragma unroll
            for (int q = 0; q < 4; ++q) s[k + q] += x[q];
        }
    void* c = at<DT_BF16>(A.c, (int64_t)(t.lo + i) * A.nj);
#pragma unroll
    for (int k = 0; k < C::BN / 16; k += 8) store_like<DT_BF16, 8>(c, j + k, A.nj, s + k);
}

// (Named here: the host's compilation leaves out their launch functions otherwise.)
#define ABH_EXPERTS_FAST(C)                                                        \
    template __global__ void k_experts_fast<MODE_Y, C, true>(ExpertArgs);          \
    template __global__ void k_experts_fast<MODE_Y, C, false>(ExpertArgs);         \
    template __global__ void k_experts_fast<MODE_DX, C, true>(ExpertArgs);         \
    template __global__ void k_experts_fast<MODE_DX, C, false>(ExpertArgs);        \
    template __global__ void k_experts_fast<MODE_DW, C, true>(ExpertArgs);         \
    template __global__ void k_experts_fast<MODE_DW, C, false>(ExpertArgs);
ABH_EXPERTS_FAST(LargeTile)
ABH_EXPERTS_FAST(SmallTile)
#undef ABH_EXPERTS_FAST

// ------------------------------------------------------------------------------------ FP32
//
// The same with FP32 matrix instructions (32 x 32 x 2, a sixteenth of BF16's rate, which bounds it): tiles of 128 x 128 or,
// where those are few, 64 x 64, four wavefronts of a quarter each, 32 terms a step, two buffers.  A long operand is read
// four terms a lane, and the instructions take the terms in that order from both.  4096 x 4096 of 8192 rows: 128 / 124 / 127
// TFLOP/s (y, dx, dW) of the 157 there are.

template <int MODE, int B>
__global__ __launch_bounds__(256, 2) void k_experts_f32(ExpertArgs A)
{
    constexpr bool ALONG = MODE != MODE_DW, BLONG = MODE == MODE_Y;
    constexpr int BK = 32, NI = B / 64;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[2][2 * B * BK * 4];
    Tile t;
    if constexpr (MODE == MODE_DW) {
        if (!find_weight_tile(A, t)) return;
    } else {
        if (!find_row_tile<B>(A, t)) return;
    }
    const int i0 = t.ti * B, j0 = t.tj * B;
    const int limit_i = MODE == MODE_DW ? A.ni - i0 : t.hi - t.lo - i0, limit_j = A.nj - j0;
    const int len = MODE == MODE_DW ? t.hi - t.lo : t.e < A.experts ? A.len : 0;
    const int steps = (len + BK - 1) / BK;
    StagedFeed<DT_F32, ALONG, B, BK, 4> fa;
    StagedFeed<DT_F32, BLONG, B, BK, 4> fb;
    {
        const int64_t first_row = MODE == MODE_DW ? t.lo : t.lo + i0;
        const int pitch_a = MODE == MODE_DW ? A.ni : A.len, pitch_b = MODE == MODE_Y ? A.len : A.nj;
        const uint8_t* pa = at<DT_F32>(A.a, first_row * pitch_a);
        const uint8_t* pb = MODE == MODE_DW ? at<DT_F32>(A.b, (int64_t)t.lo * A.nj)
                                            : at<DT_F32>(A.b, (int64_t)(t.e < A.experts ? t.e : 0) * A.len * A.nj);
        if (MODE == MODE_Y) pb = at<DT_F32>(pb, (int64_t)j0 * A.len);
        fa.start(pa, pitch_a, ALONG ? 0 : i0, ALONG ? limit_i : A.ni, len);
        fb.start(pb, pitch_b, BLONG ? 0 : j0, BLONG ? limit_j : A.nj, len);
    }
    const int lane = threadIdx.x & 63, wave = threadIdx.x / kWave;
    const int wi = (wave & 1) * (B / 2), wj = (wave >> 1) * (B / 2);
    mm_f32x16 sum[NI][NI];
    multiply_tile_f32<B, ALONG, BLONG>(lds, fa, fb, steps, wi, wj, sum);
    float* out;
    if constexpr (MODE == MODE_DW) {
        out = (A.splits > 1 ? part_of<MODE>(A, t) : static_cast<float*>(A.c) + (int64_t)t.e * A.ni * A.nj) + (int64_t)i0 * A.nj + j0;
    } else {
        out = static_cast<float*>(A.c) + (int64_t)(t.lo + i0) * A.nj + j0;
    }
#pragma unroll
    for (int i = 0; i < NI; ++i) {
        const int row = wi + 32 * i + (lane & 31);
        if (row >= limit_i) continue;
#pragma unroll
        for (int j = 0; j < NI; ++j)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const float four[4] = {sum[i][j][4 * q], sum[i][j][4 * q + 1], sum[i][j][4 * q + 2], sum[i][j][4 * q + 3]};
                store_like<DT_F32, 4>(out + (int64_t)row * A.nj, wj + 32 * j + 8 * q + 4 * (lane >> 5), limit_j, four);
            }
    }
}

// --------------------------------------------------------------------- launches

constexpr int64_t kExpertSize = (int64_t)1 << 22, kExpertRows = (int64_t)1 << 30;

// How a call is cut: which kernel, its tile, and the parts of the rows of a dW.
struct Plan {
    enum { FEW, ANY, LARGE, SMALL, F32_128, F32_64 } kernel;
    int tile, splits;
    bool rest;   // whether the tiles after the last whole round may be cut
    // bytes of scratch, of a result of so many values
    int64_t work(int64_t values) const { return rest ? (int64_t)kCus * LargeTile::BM * LargeTile::BN * 4 : splits > 1 ? splits * values * 4 : 0; }
};

// Measured on MI355X, us, both sides of each line (experts of 1536 x 2048 unless said):
//   few rows: y of 512 rows, 64 experts 85 streamed / 106 on tiles, 1024 rows 111 / 108; 16 rows of one expert 4096 x 4096 14.0 /
//     15.9, 24 rows 17.1 / 16.0, 64 rows 25.9 / 17.3; 64 rows of one expert 1024 x 1024 8.8 / 10.9, 2048 x 8192 43 / 19;
//   cut sums of small tiles: one expert 4096 x 4096, y of 128 rows 35.5 whole / 18.2 cut, 512 rows 35.8 / 30.5; 600 rows of one
//     512 x 1024 11.5 / 12.1; 300 rows of 2 experts 8192 x 2048 y 21.5 / 30 in two (192 tiles, so whole), dx 65 / 33;
//   large or small BF16 tiles: dx of 1024 rows, 8 experts 8192 x 2048 (64 large ones) 155 / 102, 2048 (104) 175 / 168, 4096 (160)
//     188 / 229; dW of 16 experts 512 x 512 (64) 98 / 42; y of 4096 rows, 64 experts 122 / 102, 8192 (128 an expert) 124 / 126, 12288
//     136 / 147;
//   FP32 tiles of 128 or 64: 1237 rows, 5 experts 193 x 333, a training pass 142 / 48; 8192 rows, 8 experts 2048 x 2048 1984 on 128;
//   parts of a dW: 13499 rows of one expert 704 x 65 382 whole / 30 in parts.
static Plan plan_experts(int mode, int32_t dtype, int64_t rows, int64_t experts, int64_t n, int64_t k)
{
    const bool bf = dtype == ADAMBRIDGE_DT_BF16;
    const int64_t used = std::min(rows, experts), ni = n, nj = mode == MODE_Y ? n : k;
    // rows of a piece or more, a tile of 256 of them within 32-bit offsets
    const int64_t piece = bf ? 8 : 4;
    const bool any = n < piece || k < piece || n > kExpertSize / 4 || k > kExpertSize / 4;
    // tiles, if every expert's last one is half empty
    auto tiles = [&](int64_t t) {
        const int64_t j = (nj + t - 1) / t;
        return mode == MODE_DW ? experts * ((ni + t - 1) / t) * j : (rows / t + (used + 1) / 2) * j;
    };
    // few rows an expert: the weights' bytes are all there is; or more, read at once, of too few tiles whose sums are not cut.  By
    // the average, the host knows no other: rows that are all one expert's are slower so than on tiles (512 rows, us, spread
    // evenly / all one expert's / that expert alone, on tiles: 64 experts 87 / 81 / 18, 8 experts 1024 x 1024 14 / 43 / 14)
    if (mode == MODE_Y && (rows <= std::max<int64_t>(bf ? 16 : 64, 8 * experts) || (rows <= 64 * experts && tiles(64) < 256 && (!bf || k <= 1024))))
        return {Plan::FEW, 0, 1, false};
    if (any) return {Plan::ANY, kTile, 1, false};
    Plan p = bf ? Plan{Plan::LARGE, LargeTile::BM, 1, false} : Plan{Plan::F32_128, 128, 1, false};
    // tiles too few for the CUs, or large ones mostly without rows: smaller ones
    if (tiles(p.tile) < (bf ? 128 : 512) || (bf && mode != MODE_DW && rows <= 128 * experts))
        p = bf ? Plan{Plan::SMALL, SmallTile::BM, 1, false} : Plan{Plan::F32_64, 64, 1, false};
    if (mode == MODE_DW) {   // few tiles with many rows: parts of 256 rows or more, two workgroups a CU
        const int64_t t = std::max<int64_t>(1, tiles(p.tile));
        p.splits = (int)std::max<int64_t>(1, std::min<int64_t>(512 / t, rows / experts / 256));
    }
    // few tiles with long sums: parts of 16 steps or more, about a workgroup a CU (by the reckoned tiles: the experts' last ones make
    // up to half a row tile an expert more or fewer)
    if (mode != MODE_DW && p.kernel == Plan::SMALL)
        p.splits = (int)std::max<int64_t>(1, std::min<int64_t>(320 / std::max<int64_t>(1, tiles(p.tile)), (mode == MODE_Y ? k : n) / (16 * SmallTile::BK)));
    // a long sum, and so few rounds that a cut rest may count
    if (mode != MODE_DW && p.kernel == Plan::LARGE) p.rest = (mode == MODE_Y ? k : n) >= 128 * LargeTile::BK && tiles(LargeTile::BM) <= 4 * kCus;
    return p;
}

static int64_t result_values(int mode, int64_t rows, int64_t experts, int64_t n, int64_t k)
{
    return mode == MODE_DW ? experts * n * k : rows * (mode == MODE_Y ? n : k);
}

template <int MODE>
static int experts_mm(const void* a, const void* b, const int32_t* ends, void* c, int32_t dtype, int64_t rows, int64_t experts,
                      int64_t n, int64_t k, void* work)
{
    if (rows < 0 || rows > kExpertRows || experts < 1 || experts > kExpertsMost || n < 1 || n > kExpertSize || k < 1 || k > kExpertSize)
        return ADAMBRIDGE_EBADN;
    if (dtype != ADAMBRIDGE_DT_F32 && dtype != ADAMBRIDGE_DT_BF16) return ADAMBRIDGE_EMVDTYPE;
    if (MODE != MODE_DW && rows == 0) return 0;
    const Plan p = plan_experts(MODE, dtype, rows, experts, n, k);
    const int64_t values = result_values(MODE, rows, experts, n, k);
    if ((!a && rows) || (!b && rows) || !ends || !c || (p.work(1) && !work)) return ADAMBRIDGE_ENULL;
    if (p.work(1) && (uintptr_t)work % 16) return ADAMBRIDGE_EALIGN;
    const bool bf = dtype == ADAMBRIDGE_DT_BF16;
    const int64_t size = bf ? 2 : 4;
    ExpertArgs A;
    A.a = a;
    A.b = b;
    A.c = c;
    A.ends = ends;
    A.rows = (int32_t)rows;
    A.experts = (int32_t)experts;
    A.ni = (int32_t)n;
    A.nj = (int32_t)(MODE == MODE_Y ? n : k);
    A.len = (int32_t)(MODE == MODE_Y ? k : n);
    A.splits = p.splits;
    A.part = p.splits > 1 || p.rest ? static_cast<float*>(work) : nullptr;
    if (p.kernel == Plan::FEW) {
        A.tiles_j = (A.nj + kFewColumns - 1) / kFewColumns;
        const bool even = k * size % 16 == 0 && ((uintptr_t)a | (uintptr_t)b) % 16 == 0 && std::max<int64_t>(rows, kFewColumns) * k * size < (int64_t)1 << 31;
        const dim3 grid = block_grid(std::min(rows, experts + 1) * A.tiles_j), block(kFewWaves * kWave);   // experts that may have rows
        if (bf && even) hipLaunchKernelGGL((k_experts_few<DT_BF16, true>), grid, block, 0, t_stream, A);
        else if (bf) hipLaunchKernelGGL((k_experts_few<DT_BF16, false>), grid, block, 0, t_stream, A);
        else if (even) hipLaunchKernelGGL((k_experts_few<DT_F32, true>), grid, block, 0, t_stream, A);
        else hipLaunchKernelGGL((k_experts_few<DT_F32, false>), grid, block, 0, t_stream, A);
    } else {
        const bool even = n % 8 == 0 && k % 8 == 0 && ((uintptr_t)a | (uintptr_t)b | (uintptr_t)c) % 16 == 0;
        A.tiles_j = (A.nj + p.tile - 1) / p.tile;
        A.tiles_i = (A.ni + p.tile - 1) / p.tile;
        // every expert, and the rows that are no expert's, may have a partial tile
        const int64_t tiles = MODE == MODE_DW ? experts * p.splits * (((int64_t)A.tiles_i * A.tiles_j + kXcd - 1) / kXcd * kXcd)
                                              : std::min(rows, rows / p.tile + experts + 1) * A.tiles_j * p.splits;
        if (tiles > (int64_t)1 << 30) return ADAMBRIDGE_EBADN;   // tiles are counted in 32 bits
        const dim3 grid = block_grid((tiles + kXcd - 1) / kXcd * kXcd + (p.rest ? kCus : 0));
        if (p.kernel == Plan::LARGE && even)
            hipLaunchKernelGGL((k_experts_fast<MODE, LargeTile, true>), grid, dim3(LargeTile::T), 0, t_stream, A);
        else if (p.kernel == Plan::LARGE)
            hipLaunchKernelGGL((k_experts_fast<MODE, LargeTile, false>), grid, dim3(LargeTile::T), 0, t_stream, A);
        else if (p.kernel == Plan::SMALL && even)
            hipLaunchKernelGGL((k_experts_fast<MODE, SmallTile, true>), grid, dim3(SmallTile::T), 0, t_stream, A);
        else if (p.kernel == Plan::SMALL)
            hipLaunchKernelGGL((k_experts_fast<MODE, SmallTile, false>), grid, dim3(SmallTile::T), 0, t_stream, A);
        else if (p.kernel == Plan::F32_128) hipLaunchKernelGGL((k_experts_f32<MODE, 128>), grid, dim3(256), 0, t_stream, A);
        else if (p.kernel == Plan::F32_64) hipLaunchKernelGGL((k_experts_f32<MODE, 64>), grid, dim3(256), 0, t_stream, A);
        else if (bf) hipLaunchKernelGGL((k_experts_any<DT_BF16, MODE, false>), grid, dim3(kMmThreads2), 0, t_stream, A);
        else if (A.len > kF32Chain * kStep) hipLaunchKernelGGL((k_experts_any<DT_F32, MODE, true>), grid, dim3(kMmThreads2), 0, t_stream, A);
        else hipLaunchKernelGGL((k_experts_any<DT_F32, MODE, MODE == MODE_DW>), grid, dim3(kMmThreads2), 0, t_stream, A);   // (dW's: the rows)
    }
    if (p.rest)
        hipLaunchKernelGGL((k_experts_rest<LargeTile>), dim3(kMostRest * LargeTile::BM / 16), dim3(256), 0, t_stream, A);
    if (p.splits > 1) {
        const dim3 grid((unsigned)((values + 1023) / 1024));
        if (bf) hipLaunchKernelGGL((k_experts_sum<DT_BF16>), grid, dim3(256), 0, t_stream, A.part, values, p.splits, c);
        else hipLaunchKernelGGL((k_experts_sum<DT_F32>), grid, dim3(256), 0, t_stream, A.part, values, p.splits, c);
    }
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? 0 : hip_fail(e, "hipLaunchKernelGGL (expert product)");
}

}  // namespace abh

using namespace abh;

extern "C" {

ADAMBRIDGE_API int64_t adambridge_expert_mm_work(int32_t product, int32_t dtype, int64_t rows, int64_t experts, int64_t n, int64_t k)
{
    if (product < MODE_Y || product > MODE_DW || rows < 0 || rows > kExpertRows || experts < 1 || experts > kExpertsMost || n < 1 ||
        n > kExpertSize || k < 1 || k > kExpertSize)
        return ADAMBRIDGE_EBADN;
    if (dtype != ADAMBRIDGE_DT_F32 && dtype != ADAMBRIDGE_DT_BF16) return ADAMBRIDGE_EMVDTYPE;
    return rows ? plan_experts(product, dtype, rows, experts, n, k).work(result_values(product, rows, experts, n, k)) : 0;
}

ADAMBRIDGE_API int adambridge_expert_mm(const void* x, const void* weight, const int32_t* ends, void* y, int32_t dtype,
                                        int64_t rows, int64_t experts, int64_t n, int64_t k, void* work)
{
    return experts_mm<MODE_Y>(x, weight, ends, y, dtype, rows, experts, n, k, work);
}

ADAMBRIDGE_API int adambridge_expert_mm_dx(const void* gout, const void* weight, const int32_t* ends, void* dx, int32_t dtype,
                                           int64_t rows, int64_t experts, int64_t n, int64_t k, void* work)
{
    return experts_mm<MODE_DX>(gout, weight, ends, dx, dtype, rows, experts, n, k, work);
}

ADAMBRIDGE_API int adambridge_expert_mm_dw(const void* gout, const void* x, const int32_t* ends, void* dw, int32_t dtype,
                                           int64_t rows, int64_t experts, int64_t n, int64_t k, void* work)
{
    return experts_mm<MODE_DW>(gout, x, ends, dw, dtype, rows, experts, n, k, work);
}

}  // extern "C"
