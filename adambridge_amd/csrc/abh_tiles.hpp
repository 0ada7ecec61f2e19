// abh_tiles.hpp -- what the kernels of matrix products share: operands' tiles on their way to the LDS, the fragments
// read there, a tile's sums, and their stores.
//
// All are C[i, j] = sum over k of A[i, k] B[j, k], with the sum along a row of an operand (the operand is "long" in k) or
// across its rows.  abh_experts.hip says why the tiles are what they are, and what they measured.
#pragma once

#include <hip/hip_runtime.h>

#include <stdint.h>

#include <type_traits>

#include "abh_device.hpp"
#include "abh_rows.hpp"

namespace abh {

constexpr int kXcd = 8;
constexpr int kGroupTiles = 8;   // row tiles that share their columns' weights while those are in the L2

typedef float mm_f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 mm_bf16x8 __attribute__((ext_vector_type(8)));

// The tile's numbers in scalar registers: divisions leave them, the same in all lanes, in vector ones, where the addresses made
// of them cannot describe a buffer.
__device__ __forceinline__ int scalar(int x) { return __builtin_amdgcn_readfirstlane(x); }

// A long FP32 sum's rounding errors grow with the chain it is taken in: every kF32Chain steps (256 terms) the products' sums are
// added to others (norm of the error over the result's, 4096 terms on tiles: 1.1e-6 in one chain, 2.3e-7 in chains of 128; those
// cost 3% of the time, 256 terms half of it; a gradient of 60000 rows of 3 values, below: 4.3e-6 in one chain, 3.9e-7).
constexpr int kF32Chain = 8;

constexpr uint32_t kOutside = 0x80000000u;   // an offset outside every buffer

// 16-byte pieces of rows of a matrix: whole ones through a buffer, whose range ends them, or (EVEN false) rows of any
// length at any address.
template <int DT, bool EVEN>
struct Pieces {
    const uint8_t* base;
    uint32_t bytes;
    int64_t len;
    int rows;
    // Values k .. of row `row`; zeros past the rows' end and past the row's.
    __device__ __forceinline__ raw16 load(int row, int k, bool real) const
    {
        if constexpr (EVEN) {
            const __amdgpu_buffer_rsrc_t buffer = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(base), 0, (int)bytes, 0x00020000);
            const uint32_t offset = real && k < len ? (uint32_t)((row * (int)len + k) * kSize<DT>) : kOutside;
            return __builtin_bit_cast(raw16, __builtin_amdgcn_raw_buffer_load_b128(buffer, offset, 0, 0));
        } else {
            return load_vec_raw<DT>(base + (int64_t)(row < rows ? row : 0) * len * kSize<DT>, k, real && row < rows ? len : 0);
        }
    }
};

typedef float mm_f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 mm_bf16x4 __attribute__((ext_vector_type(4)));

// Tile BM x BN by BK terms, NB buffers, WI x WJ wavefronts.
template <int BM_, int BN_, int BK_, int NB_, int WI_, int WJ_, int OCC_>
struct Config {
    static constexpr int BM = BM_, BN = BN_, BK = BK_, NB = NB_, WI = WI_, WJ = WJ_, OCC = OCC_, W = WI * WJ, T = W * kWave;
    static constexpr int NI = BM / WI / 32, NJ = BN / WJ / 32;
    static constexpr bool ROUNDS = NB * (BM + BN) * BK * 2 > 80 * 1024;   // a CU's LDS holds one workgroup's buffers
    static constexpr int LOADS = (BM + BN) * BK * 2 / 1024 / W;   // of a wavefront and step
    static constexpr int BYTES = (BM + BN) * BK * 2;
};

// vmcnt(n): all but the last n of this wavefront's loads have arrived.
template <int N>
__device__ __forceinline__ void wait_loads()
{
    __builtin_amdgcn_s_waitcnt(0x0f70 | (N & 15) | (N >> 4) << 14);
}

// How the 16-byte pieces of a row of CH of them, or of a term of R rows, change places in the LDS.
template <int CH>
__device__ __forceinline__ int swap_of_row(int row)
{
    return CH == 8 ? (row >> 1) & 7 : (row >> 2) & 3;   // 16 rows' pieces of a number: 16 places of the 256 bytes of all banks
}
template <int DT, int R>
__device__ __forceinline__ int swap_of_term(int term)
{
    if (DT == DT_F32) return (term & 4) << 1;              // read a value a lane: terms 4 apart, 128 bytes of each
    return R >= 128 ? (term & 3) << 2 : (term & 2) << 1;   // read transposed
}

// One operand's tile of R rows by BK terms, on its way to the LDS in W wavefronts' pieces of 1 KB.
template <bool LONG, int R, int BK, int W>
struct Feed {
    static constexpr int N = R * BK * 2 / 1024 / W, CH = BK / 8;
    const uint8_t* base;   // the next step's first value (LONG: the tile's)
    uint32_t offset[N];    // of this lane's pieces
    int32_t pitch;         // bytes
    int32_t left;          // terms from the next step's first one on
    int32_t lead;          // !LONG: bytes before base in its row.  LONG: the range
    int32_t along;         // LONG: bytes from base to the next step
    bool past;             // LONG: whether this lane's pieces are past the end in the last step

    // rows: LONG: those of the tile.  before: bytes before base in its first row.
    __device__ __forceinline__ void start(const uint8_t* p, int pitch_bytes, int rows, int len, int before)
    {
        const int lane = threadIdx.x & 63, wave = threadIdx.x / kWave;
        base = p;
        pitch = pitch_bytes;
        left = len;
        along = 0;
        lead = LONG ? (rows < R ? rows < 0 ? 0 : rows : R) * pitch_bytes - before : before;
        past = false;
#pragma unroll
        for (int q = 0; q < N; ++q) {
            if constexpr (LONG) {
                const int row = (q * W + wave) * (64 / CH) + lane / CH, piece = (lane % CH) ^ swap_of_row<CH>(row);
                offset[q] = (uint32_t)(row * pitch + piece * 16);
                if (q == 0) past = len % BK && piece * 8 >= len % BK;   // the same piece in all of them
            } else {
                const int term = (q * W + wave) * (512 / R) + lane / (R / 8);
                offset[q] = (uint32_t)(term * pitch + ((lane % (R / 8)) ^ swap_of_term<DT_BF16, R>(term)) * 16);
            }
        }
    }
    // The next step's pieces to the LDS; past the last step: zeros.  Piece by piece: where from, a piece, the step after.
    __device__ __forceinline__ raw16 source() const
    {
        // the range ends with the operand: pieces over the end of its last term, and terms past it, are outside
        const int terms = left < BK + 1 ? left : BK + 1;
        const int bytes = LONG ? lead : terms * pitch - lead;
        const int range = left > 0 ? bytes : 0;
        const uint64_t first = (uint64_t)base;
        return raw16{(uint32_t)first, (uint32_t)(first >> 32) & 0xffffu, (uint32_t)range, 0x00020000u};
    }
    __device__ __forceinline__ void issue_piece(int q, const raw16 buffer, uint8_t* lds) const
    {
        const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / kWave);
        // In assembly, so that the compiler does not wait for it before each transposed read: no register is written, and
        // the arrival is waited for by wait_loads.
        const uint32_t to = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)(lds + (q * W + wave) * 1024);
        const uint32_t from = LONG && left <= BK && past ? kOutside : offset[q];
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"   // m0 is never allocated ("reserved"), but the compiler reuses what it put there itself
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds"
                     :: "s"(to), "v"(from), "s"(buffer), "s"(along) : "m0", "memory");
#pragma clang diagnostic pop
    }
    __device__ __forceinline__ void advance()
    {
        left -= BK;
        if constexpr (LONG) along += BK * 2;
        else base += BK * pitch;
    }
    __device__ __forceinline__ void issue(uint8_t* lds)
    {
        const raw16 buffer = source();
#pragma unroll
        for (int q = 0; q < N; ++q) issue_piece(q, buffer, lds);
        advance();
    }
};

// The same tile, of rows of any length (a piece or more) of BF16 or FP32 at any address: through the registers, a step ahead of
// the LDS.  A piece over the end of its row is the row's last whole one, moved down once it has arrived.
template <int DT, bool LONG, int R, int BK, int W>
struct StagedFeed {
    static constexpr int V = kLane<DT>, S = kSize<DT>, N = R * BK * S / 1024 / W, CH = BK / V, RH = R / V;
    const uint8_t* base;   // LONG: the tile's first row; else the operand's first term (whole rows)
    uint32_t offset[N];    // of this lane's pieces from there, bytes
    int32_t moved[N];      // !LONG: values to move down
    int32_t pitch, len;    // values of a row; terms
    bool edge;             // !LONG: whether any piece of the tile is over the end of its row
    raw16 piece[N];

    static __device__ __forceinline__ void where(int q, int& row, int& term)
    {
        const int lane = threadIdx.x & 63, wave = threadIdx.x / kWave;
        if constexpr (LONG) {
            row = (q * W + wave) * (64 / CH) + lane / CH;
            term = ((lane % CH) ^ swap_of_row<CH>(row)) * V;
        } else {
            term = (q * W + wave) * (64 / RH) + lane / RH;
            row = ((lane % RH) ^ swap_of_term<DT, R>(term)) * V;
        }
    }
    // first: the tile's first row; rows: how many there are in all of the operand (from LONG: the tile's) on
    __device__ __forceinline__ void start(const uint8_t* p, int pitch_values, int first, int rows, int terms)
    {
        base = p;
        pitch = pitch_values;
        len = terms;
        edge = !LONG && first + R > rows;
#pragma unroll
        for (int q = 0; q < N; ++q) {
            int row, term;
            where(q, row, term);
            if constexpr (LONG) {
                offset[q] = (uint32_t)((row < rows ? row : 0) * pitch + term) * (uint32_t)S;   // past the end: any, not stored
                moved[q] = 0;
            } else {
                const int from = first + row < rows - V ? first + row : rows - V;
                offset[q] = (uint32_t)(term * pitch + from) * (uint32_t)S;
                moved[q] = first + row - from < V ? first + row - from : V;
            }
        }
    }
    __device__ __forceinline__ void load(int step)
    {
        const uint8_t* p = base + (LONG ? (int64_t)step * BK * S : (int64_t)step * BK * pitch * S);
        const int left = len - step * BK;   // terms from here on
        const bool last = left < BK;
#pragma unroll
        for (int q = 0; q < N; ++q) {
            uint32_t o = offset[q];
            if (last) {
                int row, term;
                where(q, row, term);
                // LONG: back to the row's last piece (which may lie before p); else to a term that there is
                const int back = LONG ? (term > left - V ? term - (left - V) : 0) : term >= left ? term * pitch : 0;
                o -= (uint32_t)back * (uint32_t)S;
            }
            piece[q] = load_raw<DT>(p + (int32_t)o, 0);
        }
    }
    __device__ __forceinline__ void store(int step, uint8_t* lds) const
    {
        const int lane = threadIdx.x & 63, wave = threadIdx.x / kWave;
        const int left = len - step * BK;
        const bool last = left < BK;
#pragma unroll
        for (int q = 0; q < N; ++q) {
            raw16 w = piece[q];
            int row, term;
            where(q, row, term);
            if (LONG && last) {
                const int back = term > left - V ? term - (left - V) : 0;
                w = drop_values<DT>(w, back < V ? back : V);
            }
            if (!LONG && edge) w = drop_values<DT>(w, moved[q]);
            if (!LONG && last && term >= left) w = raw16{0u, 0u, 0u, 0u};
            *reinterpret_cast<raw16*>(lds + (q * W + wave) * 1024 + lane * 16) = w;
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
                place[h] = row * BK * 2 + (((2 * h + (lane >> 5)) ^ swap_of_row<BK / 8>(row)) * 16);
        } else {
            const int within = (lane & 15) >> 2, term = 8 * (lane >> 5) + within;   // within: the term mod 4
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int piece = (first + 32 * i) / 8 + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
                place[i] = term * R * 2 + ((piece ^ swap_of_term<DT_BF16, R>(term)) * 16) + (lane & 1) * 8;
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

typedef Config<256, 256, 32, 4, 2, 4, 2> LargeTile;
typedef Config<128, 128, 32, 4, 2, 2, 2> SmallTile;   // where large ones are too few for the CUs
typedef Config<256, 256, 64, 2, 2, 2, 1> WideTile;    // four wavefronts of 128 x 128: multiply_wide
typedef Config<256, 128, 32, 3, 2, 2, 2> HalfTile;    // two workgroups a CU: one's products beside the other's results

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

template <bool LONG, int R, int BK, int W, bool EVEN>
using TileFeed = typename std::conditional<EVEN, Feed<LONG, R, BK, W>, StagedFeed<DT_BF16, LONG, R, BK, W>>::type;

// A tile's sums, of two operands whose feeds have been started; lds: C::NB buffers of C::BYTES.  False where the wavefront has
// no row (`live`): it feeds the others, and leaves its SIMD to them.
template <class C, bool ALONG, bool BLONG, bool EVEN>
__device__ __forceinline__ bool multiply_tile(uint8_t* lds, TileFeed<ALONG, C::BM, C::BK, C::W, EVEN>& fa, TileFeed<BLONG, C::BN, C::BK, C::W, EVEN>& fb,
                                              int steps, int wi, int wj, bool live, mm_f32x16 (&acc)[C::NI][C::NJ])
{
    constexpr int BM = C::BM, BN = C::BN, BK = C::BK, NB = C::NB, H = BK / 16;
    constexpr int LEAD = EVEN ? NB - 1 : 2;   // steps from the one that is multiplied to the one on its way to the LDS
    Fragments<ALONG, BM, BK, C::NI> ra;
    Fragments<BLONG, BN, BK, C::NJ> rb;
    ra.start(wi);
    rb.start(wj);
    // the pieces of step s on their way to the LDS (EVEN); else step s's from the registers, and those of the next loaded
    auto issue = [&](int s, int buffer) {
        uint8_t* la = lds + buffer * C::BYTES;
        if constexpr (EVEN) {
            fa.issue(la);
            fb.issue(la + BM * BK * 2);
        } else {
            if (s < steps) {
                fa.store(s, la);
                fb.store(s, la + BM * BK * 2);
            }
            if (s + 1 < steps) {
                fa.load(s + 1);
                fb.load(s + 1);
            }
        }
    };
    if (steps > 0) {
        if constexpr (!EVEN) {
            fa.load(0);
            fb.load(0);
        }
#pragma unroll
        for (int s = 0; s < LEAD; ++s) issue(s, s);
    }
#pragma unroll
    for (int i = 0; i < C::NI; ++i)
#pragma unroll
        for (int j = 0; j < C::NJ; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.0f;
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
    if (steps > 0) {
        if constexpr (EVEN) wait_loads<(NB - 2) * C::LOADS>();
        __syncthreads();
        int now = 0, next = 1, ahead = LEAD;
        auto turn = [&]() {
            now = next;
            next = next + 1 == NB ? 0 : next + 1;
            ahead = ahead + 1 == NB ? 0 : ahead + 1;
        };
        fetch(0, 0, 0);
        if (!live) {
            for (int s = 0; s + 1 < steps; ++s) {
                if constexpr (EVEN) wait_loads<(NB - 3) * C::LOADS>();
                __syncthreads();
                issue(s + LEAD, ahead);
                turn();
            }
            if constexpr (EVEN) wait_loads<0>();
            return false;
        }
        for (int s = 0; s + 1 < steps; ++s) {
#pragma unroll
            for (int h = 0; h + 1 < H; ++h) {
                fetch((h + 1) & 1, now, h + 1);
                multiply(h & 1);
                spread_reads<READS, PRODUCTS>();
            }
            // the next step's pieces have arrived, everyone's after the barrier, and the step before has been read
            if constexpr (EVEN) wait_loads<(NB - 3) * C::LOADS>();
            __syncthreads();
            issue(s + LEAD, ahead);
            fetch(0, next, 0);
            multiply((H - 1) & 1);
            spread_reads<READS, PRODUCTS>();
            turn();
        }
#pragma unroll
        for (int h = 0; h < H; ++h) {
            if (h + 1 < H) fetch((h + 1) & 1, now, h + 1);
            multiply(h & 1);
        }
        if constexpr (EVEN) wait_loads<0>();   // nothing is on its way to the LDS when the workgroup ends
    }
    return true;
}

// ------------------------------------------------------------------- 16 x 16 x 32
//
// The same tiles by matrix instructions of 16 x 16 x 32, a step's 32 terms at once: a wavefront's 128 x 64 are 8 x 4 of them.

// Reads of a wavefront's fragments: 16 rows, from row `first` of the tile of R rows, by 32 terms: the h-th of the step's.
template <bool LONG, int R, int BK, int N>
struct Fragments16 {
    uint32_t place[LONG ? BK / 32 : N];
    __device__ __forceinline__ void start(int first)
    {
        const int lane = threadIdx.x & 63, quarter = lane >> 4;
        if constexpr (LONG) {
            const int row = first + (lane & 15);   // the fragments are multiples of 16 apart: the same exchange
#pragma unroll
            for (int h = 0; h < BK / 32; ++h) place[h] = row * BK * 2 + (((4 * h + quarter) ^ swap_of_row<BK / 8>(row)) * 16);
        } else {
            const int within = (lane & 15) >> 2, term = 8 * quarter + within;   // within: the term mod 4
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int piece = (first + 16 * i) / 8 + ((lane & 3) >> 1);
                place[i] = term * R * 2 + ((piece ^ swap_of_term<DT_BF16, R>(term)) * 16) + (lane & 1) * 8;
            }
        }
    }
    __device__ __forceinline__ mm_bf16x8 read(const uint8_t* lds, int i, int h) const
    {
        if constexpr (LONG) {
            return __builtin_bit_cast(mm_bf16x8, *reinterpret_cast<const raw16*>(lds + place[h] + i * 16 * BK * 2));
        } else {
            typedef __attribute__((address_space(3))) mm_bf16x4* Local;
            const uint8_t* p = lds + place[i] + h * 32 * R * 2;
            const mm_bf16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((Local)(p));
            const mm_bf16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((Local)(p + 4 * R * 2));
            return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        }
    }
};

// multiply_tile with them (us, 32 x 32 x 16 / 16 x 16 x 32: dW of 2703 rows and 50688 words of 896 values 244 / 232, 4096 x 32000
// sums of 4096 terms 909 / 900).  A step is two halves of A's fragments: while the matrix cores work on one, the other's are read, or the
// next step's first ones.
template <class C, bool ALONG, bool BLONG, bool EVEN>
__device__ __forceinline__ bool multiply_tile16(uint8_t* lds, TileFeed<ALONG, C::BM, C::BK, C::W, EVEN>& fa, TileFeed<BLONG, C::BN, C::BK, C::W, EVEN>& fb,
                                                int steps, int wi, int wj, bool live, mm_f32x4 (&acc)[C::BM / C::WI / 16][C::BN / C::WJ / 16])
{
    constexpr int BM = C::BM, BN = C::BN, BK = C::BK, NB = C::NB, NI = BM / C::WI / 16, NJ = BN / C::WJ / 16, HI = NI / 2;
    static_assert(BK == 32, "a step is one instruction deep");
    constexpr int LEAD = EVEN ? NB - 1 : 2;
    Fragments16<ALONG, BM, BK, NI> ra;
    Fragments16<BLONG, BN, BK, NJ> rb;
    ra.start(wi);
    rb.start(wj);
    auto issue = [&](int s, int buffer) {
        uint8_t* la = lds + buffer * C::BYTES;
        if constexpr (EVEN) {
            fa.issue(la);
            fb.issue(la + BM * BK * 2);
        } else {
            if (s < steps) {
                fa.store(s, la);
                fb.store(s, la + BM * BK * 2);
            }
            if (s + 1 < steps) {
                fa.load(s + 1);
                fb.load(s + 1);
            }
        }
    };
    if (steps > 0) {
        if constexpr (!EVEN) {
            fa.load(0);
            fb.load(0);
        }
#pragma unroll
        for (int s = 0; s < LEAD; ++s) issue(s, s);
    }
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int j = 0; j < NJ; ++j) acc[i][j] = mm_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    mm_bf16x8 a[2][HI], b[NJ];
    auto fetch_a = [&](int half, int buffer) {
#pragma unroll
        for (int i = 0; i < HI; ++i) a[half][i] = ra.read(lds + buffer * C::BYTES, half * HI + i, 0);
    };
    auto fetch_b = [&](int j, int buffer) { b[j] = rb.read(lds + buffer * C::BYTES + BM * BK * 2, j, 0); };
    auto multiply = [&](int half, int j) {
#pragma unroll
        for (int i = 0; i < HI; ++i)
            acc[half * HI + i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b[j], a[half][i], acc[half * HI + i][j], 0, 0, 0);
    };
    constexpr int RA = ALONG ? 1 : 2, RB = BLONG ? 1 : 2;   // reads of a fragment
    if (steps > 0) {
        if constexpr (EVEN) wait_loads<(NB - 2) * C::LOADS>();
        __syncthreads();
        int now = 0, next = 1, ahead = LEAD;
        auto turn = [&]() {
            now = next;
            next = next + 1 == NB ? 0 : next + 1;
            ahead = ahead + 1 == NB ? 0 : ahead + 1;
        };
        if (!live) {
            for (int s = 0; s + 1 < steps; ++s) {
                if constexpr (EVEN) wait_loads<(NB - 3) * C::LOADS>();
                __syncthreads();
                issue(s + LEAD, ahead);
                turn();
            }
            if constexpr (EVEN) wait_loads<0>();
            return false;
        }
#pragma unroll
        for (int j = 0; j < NJ; ++j) fetch_b(j, 0);
        fetch_a(0, 0);
        for (int s = 0; s + 1 < steps; ++s) {
            fetch_a(1, now);
#pragma unroll
            for (int j = 0; j < NJ; ++j) multiply(0, j);
            spread_reads<RA * HI, HI * NJ / 2>();   // early: the barrier waits for them
            __builtin_amdgcn_sched_group_barrier(0x008, HI * NJ / 2, 0);
            // the next step's pieces have arrived, everyone's after the barrier, and the step before has been read
            if constexpr (EVEN) wait_loads<(NB - 3) * C::LOADS>();
            __syncthreads();
            issue(s + LEAD, ahead);
            fetch_a(0, next);
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                multiply(1, j);
                fetch_b(j, next);   // in place of the one that these were the last products of
            }
            __builtin_amdgcn_sched_group_barrier(0x100, RA * HI / NJ, 0);
            __builtin_amdgcn_sched_group_barrier(0x008, HI, 0);
#pragma unroll
            for (int j = 1; j < NJ; ++j) {
                __builtin_amdgcn_sched_group_barrier(0x100, RA * HI / NJ + RB, 0);
                __builtin_amdgcn_sched_group_barrier(0x008, HI, 0);
            }
            __builtin_amdgcn_sched_group_barrier(0x100, RB, 0);
            turn();
        }
        fetch_a(1, now);
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int j = 0; j < NJ; ++j) multiply(half, j);
        if constexpr (EVEN) wait_loads<0>();   // nothing is on its way to the LDS when the workgroup ends
    }
    return true;
}

// The same by four wavefronts of 128 x 128, one a SIMD (rows of whole pieces).  They read two thirds of the LDS's bytes that eight
// of 128 x 64 do.  A step is 64 terms, two instructions deep: a row's piece is then a whole line of 128 bytes, which steps of 32
// terms ask the L2 for twice (4096 x 32000 sums of 4096 terms and a softmax's statistics: 127 million requests and 889 us by 32
// terms, 843 by 64; eight wavefronts 886).  A half's fragments are in registers before its products begin.  In turns of 8 products
// the other half's, or the next step's, are read beside them, B's early, A's each in the place of the one just used, and the step
// after is sent on its way, two pieces a turn: what a CU takes from the L2.  The barrier stands where no read is pending.
template <class C, bool ALONG, bool BLONG>
__device__ __forceinline__ void multiply_wide(uint8_t* lds, Feed<ALONG, C::BM, C::BK, C::W>& fa, Feed<BLONG, C::BN, C::BK, C::W>& fb, int steps, int wi, int wj,
                                              mm_f32x4 (&acc)[C::BM / C::WI / 16][C::BN / C::WJ / 16])
{
    constexpr int BM = C::BM, BN = C::BN, BK = C::BK, NB = C::NB, NI = BM / C::WI / 16, NJ = BN / C::WJ / 16;
    typedef Feed<ALONG, C::BM, C::BK, C::W> FeedA;
    typedef Feed<BLONG, C::BN, C::BK, C::W> FeedB;
    static_assert(BK == 64 && NB == 2 && NI == 8 && NJ == 8 && FeedA::N == 8 && FeedB::N == 8, "the turns");
    Fragments16<ALONG, BM, BK, NI> ra;
    Fragments16<BLONG, BN, BK, NJ> rb;
    ra.start(wi);
    rb.start(wj);
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            acc[i][j] = mm_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            asm("" : "+a"(acc[i][j]));   // the sums live in the accumulation registers: the others are the fragments'
        }
    if (steps <= 0) return;
    uint8_t *here = lds, *next = lds + C::BYTES;
    auto issue = [&](const raw16 from_a, const raw16 from_b, int q, uint8_t* to) {
        if (q < FeedA::N) fa.issue_piece(q, from_a, to);
        else fb.issue_piece(q - FeedA::N, from_b, to + BM * BK * 2);
    };
    fa.issue(here);
    fb.issue(here + BM * BK * 2);
    fa.issue(next);
    fb.issue(next + BM * BK * 2);
    mm_bf16x8 a[NI], b[2][NJ];
    wait_loads<C::LOADS>();
    __syncthreads();
#pragma unroll
    for (int j = 0; j < NJ; ++j) b[0][j] = rb.read(here + BM * BK * 2, j, 0);
#pragma unroll
    for (int i = 0; i < NI; ++i) a[i] = ra.read(here, i, 0);
    auto products = [&](int set, int i) {
#pragma unroll
        for (int j = 0; j < NJ; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b[set][j], a[i], acc[i][j], 0, 0, 0);
    };
    raw16 from_a = fa.source(), from_b = fb.source();
    for (int s = 0; s < steps; ++s) {
#pragma unroll
        for (int i = 0; i < NI; ++i) {   // the first half of the terms
            if (s && i < 2) {
                issue(from_a, from_b, 12 + 2 * i, next);
                issue(from_a, from_b, 13 + 2 * i, next);
            }
            if (i == 1 && s) {
                fa.advance();
                fb.advance();
            }
            if (i < 4) {
                b[1][2 * i] = rb.read(here + BM * BK * 2, 2 * i, 1);
                b[1][2 * i + 1] = rb.read(here + BM * BK * 2, 2 * i + 1, 1);
            }
            products(0, i);
            a[i] = ra.read(here, i, 1);
            __builtin_amdgcn_sched_barrier(0);
        }
        from_a = fa.source();
        from_b = fb.source();
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            if (i == 2) {
                wait_loads<0>();   // the next step's pieces
                __syncthreads();   // everyone's; and everyone has read this step's
            }
            if (i >= 2) {
                issue(from_a, from_b, 2 * i - 4, here);
                issue(from_a, from_b, 2 * i - 3, here);
            }
            if (i >= 2 && i < 6) {
                b[0][2 * i - 4] = rb.read(next + BM * BK * 2, 2 * i - 4, 0);
                b[0][2 * i - 3] = rb.read(next + BM * BK * 2, 2 * i - 3, 0);
                if (i < 4) a[i - 2] = ra.read(next, i - 2, 0);
            }
            products(1, i);
            if (i >= 2) a[i] = ra.read(next, i, 0);
            __builtin_amdgcn_sched_barrier(0);
        }
        uint8_t* const now = next;
        next = here;
        here = now;
    }
    wait_loads<0>();   // nothing is on its way to the LDS when the workgroup ends
}

// store_bf16 of such sums: a lane has row lane mod 16 and, of each 16 columns, four; neighbouring sixteens exchange fours.
template <class C, bool EVEN, int NI, int NJ>
__device__ __forceinline__ void store_bf16(uint8_t* out, int pitch, int limit_i, int limit_j, const mm_f32x4 (&acc)[NI][NJ], int wi, int wj)
{
    const int lane = threadIdx.x & 63, quarter = lane >> 4;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
        const int row = wi + 16 * i + (lane & 15);
#pragma unroll
        for (int j = 0; j < NJ; j += 2) {
            // sixteens 0 and 2 take the first 16 columns' eights, 1 and 3 the second's
            const auto s0 = __builtin_amdgcn_permlane16_swap(bf16x2_rne(acc[i][j][0], acc[i][j][1]), bf16x2_rne(acc[i][j + 1][0], acc[i][j + 1][1]), false, false);
            const auto s1 = __builtin_amdgcn_permlane16_swap(bf16x2_rne(acc[i][j][2], acc[i][j][3]), bf16x2_rne(acc[i][j + 1][2], acc[i][j + 1][3]), false, false);
            const int c = wj + 16 * (j + (quarter & 1)) + 8 * (quarter >> 1);
            const raw16 eight = {s0[0], s1[0], s0[1], s1[1]};
            const int64_t o = (int64_t)row * pitch + c;
            if (row >= limit_i || c >= limit_j) continue;
            if (EVEN || c + 8 <= limit_j) {
                store_raw<DT_BF16>(out, o, eight);
            } else {
                const uint32_t v[4] = {eight.x, eight.y, eight.z, eight.w};
#pragma unroll
                for (int r = 0; r < 8; ++r)
                    if (c + r < limit_j) reinterpret_cast<uint16_t*>(out)[o + r] = (uint16_t)(v[r / 2] >> (16 * (r & 1)));
            }
        }
    }
}

// A tile's results in BF16: rows of `pitch` values from out on, limit_i of them by limit_j.  EVEN: whole 16-byte pieces.
template <class C, bool EVEN>
__device__ __forceinline__ void store_bf16(uint8_t* out, int pitch, int limit_i, int limit_j, const mm_f32x16 (&acc)[C::NI][C::NJ], int wi, int wj)
{
    const int lane = threadIdx.x & 63;
    // a lane has row lane mod 32 and, of each 8 columns, 4: the two halves exchange fours for whole 16 bytes
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
                const raw16 eight = {s0[0], s1[0], s0[1], s1[1]};
                const int64_t o = (int64_t)row * pitch + c;
                if (row >= limit_i || c >= limit_j) continue;
                if (EVEN || c + 8 <= limit_j) {
                    store_raw<DT_BF16>(out, o, eight);
                } else {
                    const uint32_t v[4] = {eight.x, eight.y, eight.z, eight.w};
#pragma unroll
                    for (int r = 0; r < 8; ++r)
                        if (c + r < limit_j) reinterpret_cast<uint16_t*>(out)[o + r] = (uint16_t)(v[r / 2] >> (16 * (r & 1)));
                }
            }
        }
    }
}

// ------------------------------------------------------------------------------------ FP32

template <bool LONG, int R, int N>
struct FragmentsF32 {
    int row;
    __device__ __forceinline__ void start(int first) { row = first + (threadIdx.x & 31); }
    // 32 rows from row + 32 i, terms 8 h + 4 (lane / 32) ..
    __device__ __forceinline__ mm_f32x4 read(const uint8_t* lds, int i, int h) const
    {
        const int half = (threadIdx.x & 63) >> 5, r = row + 32 * i;
        if constexpr (LONG) {
            return *reinterpret_cast<const mm_f32x4*>(lds + r * 128 + ((2 * h + half) ^ swap_of_row<8>(r)) * 16);
        } else {
            const float* f = reinterpret_cast<const float*>(lds);
            mm_f32x4 x;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int term = 8 * h + 4 * half + q;
                x[q] = f[term * R + ((r >> 2) ^ swap_of_term<DT_F32, R>(term)) * 4 + (r & 3)];
            }
            return x;
        }
    }
};

// multiply_tile's sums in FP32, of tiles of B x B by four wavefronts.
template <int B, bool ALONG, bool BLONG>
__device__ __forceinline__ void multiply_tile_f32(uint8_t (&lds)[2][2 * B * 32 * 4], StagedFeed<DT_F32, ALONG, B, 32, 4>& fa,
                                                  StagedFeed<DT_F32, BLONG, B, 32, 4>& fb, int steps, int wi, int wj, mm_f32x16 (&sum)[B / 64][B / 64])
{
    constexpr int BK = 32, NI = B / 64, BYTES = B * BK * 4;
    FragmentsF32<ALONG, B, NI> ra;
    FragmentsF32<BLONG, B, NI> rb;
    ra.start(wi);
    rb.start(wj);
    mm_f32x16 acc[NI][NI];
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int j = 0; j < NI; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = sum[i][j][r] = 0.0f;
    auto gather = [&]() {
#pragma unroll
        for (int i = 0; i < NI; ++i)
#pragma unroll
            for (int j = 0; j < NI; ++j)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    sum[i][j][r] += acc[i][j][r];
                    acc[i][j][r] = 0.0f;
                }
    };
    if (steps > 0) {
        fa.load(0);
        fb.load(0);
    }
    for (int s = 0; s < steps; ++s) {
        uint8_t* now = lds[s & 1];
        fa.store(s, now);
        fb.store(s, now + BYTES);
        if (s + 1 < steps) {
            fa.load(s + 1);
            fb.load(s + 1);
        }
        __syncthreads();   // written; and whoever is here has read the buffer that the next step writes
#pragma unroll
        for (int h = 0; h < BK / 8; ++h) {
            mm_f32x4 a[NI], b[NI];
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                a[i] = ra.read(now, i, h);
                b[i] = rb.read(now + BYTES, i, h);
            }
#pragma unroll
            for (int q = 0; q < 4; ++q)
#pragma unroll
                for (int i = 0; i < NI; ++i)
#pragma unroll
                    for (int j = 0; j < NI; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x2f32(b[j][q], a[i][q], acc[i][j], 0, 0, 0);
        }
        if (s % kF32Chain == kF32Chain - 1) gather();
    }
    gather();
}

}  // namespace abh
