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

// A tile of dW.  The XCDs share every expert's tiles evenly, because experts differ in rows and so in work.
__device__ __forceinline__ bool find_weight_tile(const ExpertArgs& A, Tile& t)
{
    const int an = A.tiles_i * A.tiles_j, per = (an + kXcd - 1) / kXcd;
    const int slot = (int)(blockIdx.x / kXcd);
    t.e = slot / per;
    if (t.e >= A.experts) return false;
    const int local = (int)((blockIdx.x + t.e) % kXcd) * per + slot - t.e * per;   // the first XCD changes: an may be below 8
    if (local >= an) return false;
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
// Tiles of 256 x 256, eight wavefronts of 128 x 64 (2 x 4), 32 terms a step, four buffers of 32 KB in the LDS.  A step's
// tiles go from memory to the LDS past the registers, three steps ahead of the one that is multiplied; what lies
// outside an operand is out of its buffer's range and arrives as zeros.  A wavefront reads the fragments of its next
// 8 matrix products of 32 x 32 x 16 while the matrix cores work on these.
//
// Measured on MI355X, one expert, 8192^3: y 873 us (1259 TFLOP/s), dx 827 (1329), dW 821 (1339); the matrix cores are busy
// 73% of the cycles, at 1.6 GHz of 2.4: power is the bound.  Slower: 64 terms a step with two buffers 891 (y),
// wavefronts of 128 x 128 (one a SIMD) 890, tiles of 128 x 256 with two workgroups a CU 1010, three buffers 989; five
// buffers change nothing.
//
// A long operand's tile is its rows by 64 bytes, a row's 16-byte pieces exchanged by the row, so that the reads of
// neighbouring rows meet different banks.  One across its rows is 32 terms by its rows, read transposed
// (ds_read_b64_tr_b16: 16 lanes take 4 terms x 16 values, a lane 4 terms of one value), its pieces exchanged in
// fours by the term mod 4: the 4 terms x 2 pairs of pieces of 32 lanes then cover the 256 bytes of all banks.

constexpr uint32_t kOutside = 0x80000000u;          // an offset outside every buffer

typedef float mm_f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 mm_bf16x4 __attribute__((ext_vector_type(4)));

// Tile BM x BN by BK terms, NB buffers, WI x WJ wavefronts.
template <int BM_, int BN_, int BK_, int NB_, int WI_, int WJ_, int OCC_>
struct Config {
    static constexpr int BM = BM_, BN = BN_, BK = BK_, NB = NB_, WI = WI_, WJ = WJ_, OCC = OCC_, W = WI * WJ, T = W * kWave;
    static constexpr int NI = BM / WI / 32, NJ = BN / WJ / 32;
    static constexpr int LOADS = (BM + BN) * BK * 2 / 1024 / W;   // of a wavefront and step
    static constexpr int BYTES = (BM + BN) * BK * 2;
};

// vmcnt(n): all but the last n of this wavefront's loads have arrived.
template <int N>
__device__ __forceinline__ void wait_loads()
{
    __builtin_amdgcn_s_waitcnt(0x0f70 | (N & 15) | (N >> 4) << 14);
}

// One operand's tile of R rows by BK terms, on its way to the LDS in W wavefronts' pieces of 1 KB.
template <bool LONG, int R, int BK, int W>
struct Feed {
    static constexpr int N = R * BK * 2 / 1024 / W, CH = BK / 8;
    const uint8_t* base;   // the tile's first value
    uint32_t offset[N];    // of this lane's pieces
    int64_t left;          // !LONG: bytes from base to the operand's end
    int32_t pitch;         // bytes
    bool past;             // LONG: whether this lane's pieces are past the end in the last step

    static __device__ __forceinline__ int swap_of_row(int row) { return BK == 64 ? row & 7 : (row >> 2) & 3; }

    // rows: LONG: the tile's rows; else the operand's terms.  lead: !LONG: bytes before base in its first row.
    __device__ __forceinline__ void start(const uint8_t* p, int64_t pitch_bytes, int rows, int len, int64_t lead)
    {
        const int lane = threadIdx.x & 63, wave = threadIdx.x / kWave;
        base = p;
        pitch = (int32_t)pitch_bytes;
        past = false;
        left = LONG ? (int64_t)(rows < R ? rows : R) * pitch_bytes : (int64_t)rows * pitch_bytes - lead;
#pragma unroll
        for (int q = 0; q < N; ++q) {
            if constexpr (LONG) {
                const int row = (q * W + wave) * (64 / CH) + lane / CH, piece = (lane % CH) ^ swap_of_row(row);
                offset[q] = (uint32_t)(row * pitch + piece * 16);
                if (q == 0) past = len % BK && piece * 8 >= len % BK;   // the same piece in all of them
            } else {
                const int term = (q * W + wave) * (512 / R) + lane / (R / 8);
                offset[q] = (uint32_t)(term * pitch + ((lane % (R / 8)) ^ (term & 3) << 2) * 16);
            }
        }
    }
    __device__ __forceinline__ void issue(int step, int steps, uint8_t* lds) const
    {
        const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / kWave);
        const int64_t skip = LONG ? 0 : (int64_t)step * BK * pitch;
        const int64_t bytes = left - skip;
        const int32_t range = step >= steps ? 0 : (int32_t)(bytes < 0x7fffffff ? bytes : 0x7fffffff);   // past the end: zeros
        const uint64_t first = (uint64_t)(base + skip);
        const raw16 buffer = {(uint32_t)first, (uint32_t)(first >> 32) & 0xffffu, (uint32_t)range, 0x00020000u};
        const uint32_t along = LONG ? (uint32_t)step * BK * 2 : 0u;
#pragma unroll
        for (int q = 0; q < N; ++q) {
            // In assembly, so that the compiler does not wait for it before each transposed read: no register is written, and
            // the arrival is waited for by wait_loads.
            const uint32_t to = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)(lds + (q * W + wave) * 1024);
            const uint32_t from = LONG && step + 1 == steps && past ? kOutside : offset[q];
            asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds"
                         :: "s"(to), "v"(from), "s"(buffer), "s"(along) : "memory");
        }
    }
};

// Reads of a wavefront's fragments: 32 rows, from row `first` of the tile of R rows, by 16 terms.
template <bool LONG, int R, int BK, int N>
struct Fragments {
    uint32_t place[LONG ? BK / 16 : N];
    __device__ __forceinline__ void start(int first)
    {
        const int lane = threadIdx.x & 63;
        if constexpr (LONG) {
            const int row = first + (lane & 31);   // first and the fragments are multiples of 32 apart: the same exchange
#pragma unroll
            for (int h = 0; h < BK / 16; ++h)
                place[h] = row * BK * 2 + (((2 * h + (lane >> 5)) ^ Feed<LONG, R, BK, 1>::swap_of_row(row)) * 16);
        } else {
            const int within = (lane & 15) >> 2, term = 8 * (lane >> 5) + within;   // within: the term mod 4
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int piece = (first + 32 * i) / 8 + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
                place[i] = term * R * 2 + ((piece ^ within << 2) * 16) + (lane & 1) * 8;
            }
        }
    }
    __device__ __forceinline__ mm_bf16x8 read(const uint8_t* lds, int i, int h) const
    {
        if constexpr (LONG) {
            return __builtin_bit_cast(mm_bf16x8, *reinterpret_cast<const raw16*>(lds + place[h] + i * 32 * BK * 2));
        } else {
            typedef __attribute__((address_space(3))) mm_bf16x4* Local;
            const uint8_t* p = lds + place[i] + h * 16 * R * 2;
            const mm_bf16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((Local)(p));
            const mm_bf16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((Local)(p + 4 * R * 2));
            return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        }
    }
};

typedef Config<256, 256, 32, 4, 2, 4, 2> FastConfig;

// Asks the scheduler for READS reads of the LDS spread among the next PRODUCTS matrix products.
template <int READS, int PRODUCTS, int M = 0>
__device__ __forceinline__ void spread_reads()
{
    if constexpr (M < PRODUCTS) {
        constexpr int n = READS * (M + 1) / PRODUCTS - READS * M / PRODUCTS;
        if constexpr (n > 0) __builtin_amdgcn_sched_group_barrier(0x100, n, 0);
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        spread_reads<READS, PRODUCTS, M + 1>();
    }
}

template <int MODE, class C>
__global__ __launch_bounds__(C::T, C::OCC) void k_experts_fast(ExpertArgs A)
{
    constexpr bool ALONG = MODE != MODE_DW, BLONG = MODE == MODE_Y;
    constexpr int BM = C::BM, BN = C::BN, BK = C::BK, NB = C::NB;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[NB * C::BYTES];
    Tile t;
    if (!(MODE == MODE_DW ? find_weight_tile(A, t) : find_row_tile<BM>(A, t))) return;
    const int i0 = t.ti * BM, j0 = t.tj * BN;
    const int limit_i = MODE == MODE_DW ? A.ni - i0 : t.hi - t.lo - i0, limit_j = A.nj - j0;
    const int len = MODE == MODE_DW ? t.hi - t.lo : t.e < A.experts ? A.len : 0;
    const int steps = (len + BK - 1) / BK;
    Feed<ALONG, BM, BK, C::W> fa;
    Feed<BLONG, BN, BK, C::W> fb;
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
    const int wi = wave % C::WI * (BM / C::WI), wj = wave / C::WI * (BN / C::WJ);
    Fragments<ALONG, BM, BK, C::NI> ra;
    Fragments<BLONG, BN, BK, C::NJ> rb;
    ra.start(wi);
    rb.start(wj);
    mm_f32x16 acc[C::NI][C::NJ];
#pragma unroll
    for (int i = 0; i < C::NI; ++i)
#pragma unroll
        for (int j = 0; j < C::NJ; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.0f;
    constexpr int H = BK / 16;
    auto issue = [&](int s, int buffer) {
        fa.issue(s, steps, lds + buffer * C::BYTES);
        fb.issue(s, steps, lds + buffer * C::BYTES + BM * BK * 2);
    };
    // fragments are read one product ahead, so that the LDS works while the matrix cores do
    mm_bf16x8 a[2][C::NI], b[2][C::NJ];
    auto fetch = [&](int set, int buffer, int h) {
        const uint8_t* la = lds + buffer * C::BYTES;
#pragma unroll
        for (int i = 0; i < C::NI; ++i) a[set][i] = ra.read(la, i, h);
#pragma unroll
        for (int j = 0; j < C::NJ; ++j) b[set][j] = rb.read(la + BM * BK * 2, j, h);
    };
    auto multiply = [&](int set) {
#pragma unroll
        for (int i = 0; i < C::NI; ++i)
#pragma unroll
            for (int j = 0; j < C::NJ; ++j)
                acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(b[set][j], a[set][i], acc[i][j], 0, 0, 0);
    };
    constexpr int READS = (ALONG ? 1 : 2) * C::NI + (BLONG ? 1 : 2) * C::NJ, PRODUCTS = C::NI * C::NJ;
    auto interleave = [&]() { spread_reads<READS, PRODUCTS>(); };
    if (steps > 0) {
#pragma unroll
        for (int s = 0; s < NB - 1; ++s) issue(s, s);
        wait_loads<(NB - 2) * C::LOADS>();
        __syncthreads();
        fetch(0, 0, 0);
        int now = 0, next = 1, ahead = NB - 1;
        for (int s = 0; s + 1 < steps; ++s) {
#pragma unroll
            for (int h = 0; h + 1 < H; ++h) {
                fetch((h + 1) & 1, now, h + 1);
                multiply(h & 1);
                interleave();
            }
            // the next step's pieces have arrived, everyone's after the barrier, and the step before has been read
            wait_loads<(NB - 3) * C::LOADS>();
            __syncthreads();
            issue(s + NB - 1, ahead);
            fetch(0, next, 0);
            multiply((H - 1) & 1);
            interleave();
            now = next;
            next = next + 1 == NB ? 0 : next + 1;
            ahead = ahead + 1 == NB ? 0 : ahead + 1;
        }
#pragma unroll
        for (int h = 0; h < H; ++h) {
            if (h + 1 < H) fetch((h + 1) & 1, now, h + 1);
            multiply(h & 1);
        }
        wait_loads<0>();   // nothing is on its way to the LDS when the workgroup ends
    }
    // a lane has row lane mod 32 and, of each 8 columns, 4: the two halves exchange fours for whole 16 bytes
    uint8_t* out = MODE == MODE_DW ? at<DT_BF16>(A.c, ((int64_t)t.e * A.ni + i0) * A.nj + j0)
                                   : at<DT_BF16>(A.c, (int64_t)(t.lo + i0) * A.nj + j0);
    const int half = lane >> 5;
#pragma unroll
    for (int i = 0; i < C::NI; ++i) {
        const int row = wi + 32 * i + (lane & 31);
#pragma unroll
        for (int j = 0; j < C::NJ; ++j) {
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

// (named here: the host's compilation leaves out their launch functions otherwise)
template __global__ void k_experts_fast<MODE_Y, FastConfig>(ExpertArgs);
template __global__ void k_experts_fast<MODE_DX, FastConfig>(ExpertArgs);
template __global__ void k_experts_fast<MODE_DW, FastConfig>(ExpertArgs);

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
    typedef FastConfig C;
    const int tile_i = fast ? C::BM : kTile, tile_j = fast ? C::BN : kTile;
    A.tiles_j = (A.nj + tile_j - 1) / tile_j;
    A.tiles_i = (A.ni + tile_i - 1) / tile_i;
    // every expert, and the rows that are no expert's, may have a partial tile
    const int64_t tiles = MODE == MODE_DW ? experts * (((int64_t)A.tiles_i * A.tiles_j + kXcd - 1) / kXcd * kXcd)
                                          : std::min(rows, rows / tile_i + experts + 1) * A.tiles_j;
    if (tiles > ((int64_t)1 << 31) - 64) return ADAMBRIDGE_EBADN;
    const dim3 grid((unsigned)((tiles + kXcd - 1) / kXcd * kXcd));
    if (fast) hipLaunchKernelGGL((k_experts_fast<MODE, C>), grid, dim3(C::T), 0, t_stream, A);
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
