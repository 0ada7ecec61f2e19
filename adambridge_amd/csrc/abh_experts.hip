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
#include "abh_rows.hpp"

namespace abh {

constexpr int kExpertsMost = 4096;
constexpr int kXcd = 8;
constexpr int kGroupTiles = 8;   // row tiles that share their columns' weights while those are in the L2

typedef float mm_f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t mm_u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t mm_u32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 mm_bf16x8 __attribute__((ext_vector_type(8)));

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
};

// Rows lo .. hi of expert e (e = experts: the rows that are no expert's).  Ends outside 0 .. rows, or one below the
// one before it, are pulled to the nearest that are not, so that no value of them leads out of the arrays.
__device__ __forceinline__ void expert_rows(const ExpertArgs& A, int e, int& lo, int& hi)
{
    lo = e > 0 && e <= A.experts ? A.ends[e - 1] : e == 0 ? 0 : A.rows;
    hi = e < A.experts ? A.ends[e] : A.rows;
    lo = lo < 0 ? 0 : lo > A.rows ? A.rows : lo;
    hi = hi < lo ? lo : hi > A.rows ? A.rows : hi;
}

struct Tile {
    int e, lo, hi, ti, tj;
};

// This workgroup's row tile of BM rows: consecutive tiles go to one XCD, whose L2 then holds an expert's weights for
// the tiles of its rows.  Every wavefront finds it for itself.
template <int BM>
__device__ __forceinline__ bool find_row_tile(const ExpertArgs& A, Tile& t)
{
    const int lane = threadIdx.x & 63;
    int total = 0;
    for (int e0 = 0; e0 <= A.experts; e0 += kWave) {
        int lo, hi;
        expert_rows(A, e0 + lane, lo, hi);
        int n = (hi - lo + BM - 1) / BM;
#pragma unroll
        for (int d = 1; d < kWave; d *= 2) n += __shfl_xor(n, d);
        total += n;
    }
    total = __builtin_amdgcn_readfirstlane(total);
    const int tiles = total * A.tiles_j;
    const int per = (tiles + kXcd - 1) / kXcd;
    const int slot = (int)(blockIdx.x / kXcd);
    int idx = (int)(blockIdx.x % kXcd) * per + slot;
    if (slot >= per || idx >= tiles) return false;
    const int q = idx / A.tiles_j;
    int before = 0;
    for (int e0 = 0; e0 <= A.experts; e0 += kWave) {
        int lo, hi;
        expert_rows(A, e0 + lane, lo, hi);
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
            t.ti = first + r % wide;
            t.tj = r / wide;
            return true;
        }
        before += __builtin_amdgcn_readlane(s, kWave - 1);
    }
    return false;
}

// A tile of dW: expert by expert, an expert's tiles on one XCD.
__device__ __forceinline__ bool find_weight_tile(const ExpertArgs& A, Tile& t)
{
    const int an = A.tiles_i * A.tiles_j;
    const int tiles = an * A.experts;
    const int per = (tiles + kXcd - 1) / kXcd;
    const int slot = (int)(blockIdx.x / kXcd);
    const int idx = (int)(blockIdx.x % kXcd) * per + slot;
    if (slot >= per || idx >= tiles) return false;
    t.e = idx / an;
    const int local = idx - t.e * an;
    const int g = local / (kGroupTiles * A.tiles_j), first = g * kGroupTiles;
    const int wide = A.tiles_i - first < kGroupTiles ? A.tiles_i - first : kGroupTiles;
    const int r = local - first * A.tiles_j;
    t.ti = first + r % wide;
    t.tj = r / wide;
    expert_rows(A, t.e, t.lo, t.hi);
    t.lo = __builtin_amdgcn_readfirstlane(t.lo);
    t.hi = __builtin_amdgcn_readfirstlane(t.hi);
    return true;
}

// ------------------------------------------------------------- any sizes, any alignment
//
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

template <int DT, int MODE>
__global__ __launch_bounds__(kMmThreads2, 2) void k_experts_any(ExpertArgs A)
{
    constexpr bool ALONG = MODE != MODE_DW, BLONG = MODE == MODE_Y;
    __shared__ __attribute__((aligned(16))) Element<DT> la[kTile * kPitch<DT>], lb[kTile * kPitch<DT>];
    Tile t;
    if (!(MODE == MODE_DW ? find_weight_tile(A, t) : find_row_tile<kTile>(A, t))) return;
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
    mm_f32x4 acc[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = mm_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
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
#pragma unroll
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
                            acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(fb[j][q], fa[i][q], acc[i][j], 0, 0, 0);
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
                if (c + r < limit_j) put<DT>(out, o + r, acc[i][j][r]);
        }
    }
}

// ------------------------------------------------------------- BF16 rows of whole 16-byte pieces
//
// Tiles of 256 x 256, eight wavefronts of 128 x 64 (2 x 4), 64 terms a step, two buffers of 64 KB in the LDS.  A step's
// tiles go from memory to the LDS past the registers while the step before is multiplied; what lies outside an
// operand is out of its buffer's range and arrives as zeros.  A wavefront's 8 matrix products of 32 x 32 x 16
// take 6 KB from the LDS, three quarters of the time the products take.
//
// A long operand's tile is 256 rows of 128 bytes, its 16-byte pieces exchanged by the row (piece c at place c ^ row mod 8), so
// that the reads of 8 rows meet 8 different places.  One across its rows is 64 terms of 512 bytes, read transposed
// (ds_read_b64_tr_b16: 16 lanes take 4 terms x 16 values, a lane 4 terms of one value), its pieces exchanged in
// pairs by the term's bits 0, 1 and 3, in which the terms of one read differ.

constexpr int kFast = 256, kFastStep = 64, kFastThreads = 512;
constexpr int kFastBytes = kFast * kFastStep * 2;   // of an operand's tile
constexpr uint32_t kOutside = 0x80000000u;          // an offset outside every buffer

typedef float mm_f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 mm_bf16x4 __attribute__((ext_vector_type(4)));

template <bool LONG>
struct Feed {
    const uint8_t* base;   // the tile's first value
    uint32_t offset[4];    // of this lane's pieces
    int64_t left;          // !LONG: bytes from base to the operand's end
    int32_t pitch;         // bytes
    bool past;             // LONG: whether this lane's pieces are past the end in the last step

    // rows: LONG: the tile's rows; else the operand's terms.  lead: !LONG: bytes before base in its first row.
    __device__ __forceinline__ void start(const uint8_t* p, int64_t pitch_bytes, int rows, int len, int64_t lead)
    {
        const int lane = threadIdx.x & 63, wave = threadIdx.x / kWave;
        base = p;
        pitch = (int32_t)pitch_bytes;
        const int piece = LONG ? (lane & 7) ^ (lane >> 3) : 0;
        past = LONG && len % kFastStep && piece * 8 >= len % kFastStep;
        left = LONG ? (int64_t)(rows < kFast ? rows : kFast) * pitch_bytes : (int64_t)rows * pitch_bytes - lead;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            if constexpr (LONG) {
                const int row = (q * 8 + wave) * 8 + (lane >> 3);
                offset[q] = (uint32_t)(row * pitch + piece * 16);
            } else {
                const int term = (q * 8 + wave) * 2 + (lane >> 5), swap = (term & 3) | ((term >> 3) & 1) << 2;
                offset[q] = (uint32_t)(term * pitch + ((lane & 31) ^ (swap << 1)) * 16);
            }
        }
    }
    __device__ __forceinline__ void issue(int step, bool last, uint8_t* lds) const
    {
        const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / kWave);
        const int64_t skip = LONG ? 0 : (int64_t)step * kFastStep * pitch;
        const int64_t bytes = left - skip;
        const int32_t range = (int32_t)(bytes < 0x7fffffff ? bytes : 0x7fffffff);
        const __amdgpu_buffer_rsrc_t buffer = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(base + skip), 0, range, 0x00020000);
#pragma unroll
        for (int q = 0; q < 4; ++q)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(
                buffer, (__attribute__((address_space(3))) void*)(lds + (q * 8 + wave) * 1024), 16,
                LONG && last && past ? kOutside : offset[q], LONG ? step * kFastStep * 2 : 0, 0, 0);
    }
};

// Reads of a wavefront's fragments: 32 rows, from row `first` of the tile, by 16 terms.
template <bool LONG, int N>
struct Fragments {
    uint32_t place[LONG ? 4 : N];
    __device__ __forceinline__ void start(int first)
    {
        const int lane = threadIdx.x & 63;
        if constexpr (LONG) {
#pragma unroll
            for (int h = 0; h < 4; ++h) place[h] = (first + (lane & 31)) * 128 + (((2 * h + (lane >> 5)) ^ (lane & 7)) * 16);
        } else {
            const int within = (lane & 15) >> 2, term = 8 * (lane >> 5) + within, swap = within | (lane >> 5) << 2;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int piece = (first + 32 * i) / 8 + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
                place[i] = term * 512 + ((piece ^ (swap << 1)) * 16) + (lane & 1) * 8;
            }
        }
    }
    __device__ __forceinline__ mm_bf16x8 read(const uint8_t* lds, int i, int h) const
    {
        if constexpr (LONG) {
            return __builtin_bit_cast(mm_bf16x8, *reinterpret_cast<const raw16*>(lds + place[h] + i * 4096));
        } else {
            typedef __attribute__((address_space(3))) mm_bf16x4* Local;
            const uint8_t* p = lds + place[i] + h * 8192;
            const mm_bf16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((Local)(p));
            const mm_bf16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((Local)(p + 2048));
            return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        }
    }
};

template <int MODE>
__global__ __launch_bounds__(kFastThreads, 2) void k_experts_fast(ExpertArgs A)
{
    constexpr bool ALONG = MODE != MODE_DW, BLONG = MODE == MODE_Y;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[4 * kFastBytes];
    Tile t;
    if (!(MODE == MODE_DW ? find_weight_tile(A, t) : find_row_tile<kFast>(A, t))) return;
    const int i0 = t.ti * kFast, j0 = t.tj * kFast;
    const int limit_i = MODE == MODE_DW ? A.ni - i0 : t.hi - t.lo - i0, limit_j = A.nj - j0;
    const int len = MODE == MODE_DW ? t.hi - t.lo : t.e < A.experts ? A.len : 0;
    const int steps = (len + kFastStep - 1) / kFastStep;
    Feed<ALONG> fa;
    Feed<BLONG> fb;
    if constexpr (MODE == MODE_DW) {
        fa.start(at<DT_BF16>(A.a, (int64_t)t.lo * A.ni + i0), (int64_t)A.ni * 2, len, len, (int64_t)i0 * 2);
        fb.start(at<DT_BF16>(A.b, (int64_t)t.lo * A.nj + j0), (int64_t)A.nj * 2, len, len, (int64_t)j0 * 2);
    } else {
        const uint8_t* w = at<DT_BF16>(A.b, (int64_t)(t.e < A.experts ? t.e : 0) * A.len * A.nj);
        fa.start(at<DT_BF16>(A.a, (int64_t)(t.lo + i0) * A.len), (int64_t)A.len * 2, limit_i, len, 0);
        if constexpr (MODE == MODE_Y) fb.start(w + (int64_t)j0 * A.len * 2, (int64_t)A.len * 2, limit_j, len, 0);
        else fb.start(w + (int64_t)j0 * 2, (int64_t)A.nj * 2, len, len, (int64_t)j0 * 2);
    }
    const int lane = threadIdx.x & 63, wave = threadIdx.x / kWave;
    const int wi = (wave & 1) * 128, wj = (wave >> 1) * 64;
    Fragments<ALONG, 4> ra;
    Fragments<BLONG, 2> rb;
    ra.start(wi);
    rb.start(wj);
    mm_f32x16 acc[4][2];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.0f;
    if (steps > 0) {
        fa.issue(0, steps == 1, lds);
        fb.issue(0, steps == 1, lds + kFastBytes);
    }
    for (int s = 0; s < steps; ++s) {
        uint8_t* now = lds + (s & 1) * 2 * kFastBytes;
        uint8_t* next = lds + ((s & 1) ^ 1) * 2 * kFastBytes;
        __builtin_amdgcn_s_waitcnt(0x0f70);   // vmcnt(0): this step's pieces have arrived
        __syncthreads();                      // everyone's, and the step before has been read
        if (s + 1 < steps) {
            fa.issue(s + 1, s + 2 == steps, next);
            fb.issue(s + 1, s + 2 == steps, next + kFastBytes);
        }
#pragma unroll
        for (int h = 0; h < 4; ++h) {
            mm_bf16x8 a[4], b[2];
#pragma unroll
            for (int i = 0; i < 4; ++i) a[i] = ra.read(now, i, h);
#pragma unroll
            for (int j = 0; j < 2; ++j) b[j] = rb.read(now + kFastBytes, j, h);
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(b[j], a[i], acc[i][j], 0, 0, 0);
        }
    }
    // a lane has row lane mod 32 and, of each 8 columns, 4: the two halves exchange fours for whole 16 bytes
    uint8_t* out = MODE == MODE_DW ? at<DT_BF16>(A.c, ((int64_t)t.e * A.ni + i0) * A.nj + j0)
                                   : at<DT_BF16>(A.c, (int64_t)(t.lo + i0) * A.nj + j0);
    const int half = lane >> 5;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int row = wi + 32 * i + (lane & 31);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
#pragma unroll
            for (int q = 0; q < 4; q += 2) {
                uint32_t x[2][2];
#pragma unroll
                for (int p = 0; p < 2; ++p) {
                    x[p][0] = bf16x2_rne(acc[i][j][4 * (q + p)], acc[i][j][4 * (q + p) + 1]);
                    x[p][1] = bf16x2_rne(acc[i][j][4 * (q + p) + 2], acc[i][j][4 * (q + p) + 3]);
                }
                // half 0 keeps its four of the first eight and takes half 1's; half 1 those of the second
                const auto s0 = __builtin_amdgcn_permlane32_swap(x[0][0], x[1][0], false, false);
                const auto s1 = __builtin_amdgcn_permlane32_swap(x[0][1], x[1][1], false, false);
                const int c = wj + 32 * j + 8 * (q + half);
                if (row < limit_i && c < limit_j)
                    store_raw<DT_BF16>(out, (int64_t)row * A.nj + c, raw16{s0[0], s1[0], s0[1], s1[1]});
            }
        }
    }
}

// --------------------------------------------------------------------- launches

template <int MODE>
static int experts_mm(const void* a, const void* b, const int32_t* ends, void* c, int32_t dtype, int64_t rows, int64_t experts,
                      int64_t n, int64_t k)
{
    constexpr int64_t most = (int64_t)1 << 22;
    if (rows < 0 || rows > (int64_t)1 << 30 || experts < 1 || experts > kExpertsMost || n < 1 || n > most || k < 1 || k > most)
        return ADAMBRIDGE_EBADN;
    if (dtype != ADAMBRIDGE_DT_F32 && dtype != ADAMBRIDGE_DT_BF16) return ADAMBRIDGE_EMVDTYPE;
    if (MODE != MODE_DW && rows == 0) return 0;
    if ((!a && rows) || (!b && rows) || !ends || !c) return ADAMBRIDGE_ENULL;
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
    // rows of whole 16-byte pieces, 256 of them within a buffer's offsets
    const bool fast = dtype == ADAMBRIDGE_DT_BF16 && n % 8 == 0 && k % 8 == 0 && n <= (int64_t)1 << 21 && k <= (int64_t)1 << 21 &&
                      ((uintptr_t)a | (uintptr_t)b | (uintptr_t)c) % 16 == 0;
    const int tile = fast ? kFast : kTile;
    A.tiles_j = (A.nj + tile - 1) / tile;
    A.tiles_i = (A.ni + tile - 1) / tile;
    // every expert, and the rows that are no expert's, may have a partial tile
    const int64_t tiles = MODE == MODE_DW ? experts * A.tiles_i * A.tiles_j
                                          : std::min(rows, rows / tile + experts + 1) * A.tiles_j;
    if (tiles > ((int64_t)1 << 31) - 64) return ADAMBRIDGE_EBADN;
    const dim3 grid((unsigned)((tiles + kXcd - 1) / kXcd * kXcd));
    if (fast) hipLaunchKernelGGL((k_experts_fast<MODE>), grid, dim3(kFastThreads), 0, t_stream, A);
    else if (dtype == ADAMBRIDGE_DT_BF16) hipLaunchKernelGGL((k_experts_any<DT_BF16, MODE>), grid, dim3(kMmThreads2), 0, t_stream, A);
    else hipLaunchKernelGGL((k_experts_any<DT_F32, MODE>), grid, dim3(kMmThreads2), 0, t_stream, A);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? 0 : hip_fail(e, "hipLaunchKernelGGL (expert product)");
}

}  // namespace abh

using namespace abh;

extern "C" {

ADAMBRIDGE_API int adambridge_expert_mm(const void* x, const void* weight, const int32_t* ends, void* y, int32_t dtype,
                                        int64_t rows, int64_t experts, int64_t n, int64_t k)
{
    return experts_mm<MODE_Y>(x, weight, ends, y, dtype, rows, experts, n, k);
}

ADAMBRIDGE_API int adambridge_expert_mm_dx(const void* gout, const void* weight, const int32_t* ends, void* dx, int32_t dtype,
                                           int64_t rows, int64_t experts, int64_t n, int64_t k)
{
    return experts_mm<MODE_DX>(gout, weight, ends, dx, dtype, rows, experts, n, k);
}

ADAMBRIDGE_API int adambridge_expert_mm_dw(const void* gout, const void* x, const int32_t* ends, void* dw, int32_t dtype,
                                           int64_t rows, int64_t experts, int64_t n, int64_t k)
{
    return experts_mm<MODE_DW>(gout, x, ends, dw, dtype, rows, experts, n, k);
}

}  // extern "C"
