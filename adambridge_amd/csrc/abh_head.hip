// abh_head.hip -- each row's cross-entropy over a vocabulary, from the rows before the head's product, and its gradients.
//
//   x[t, v]  = <h[t], W[v]>
//   loss[t]  = log(sum over v of exp x[t, v]) - x[t, target[t]]
//   G[t, v]  = gout[t] (exp(x[t, v]) / sum - [v = target[t]]),   dh = G W,   dW = G^T h
//
// No logit is kept.  Forward, a tile of the product ends in its rows' maxima and sums of exponentials, 8 bytes a row and
// tile, which are merged in order; the logits are the products' FP32 sums, never rounded.  Backward, the vocabulary goes by
// in pieces: a piece's logits are computed again and end as G (in the operands' type: its rounding is the only one between
// the sums, and what a matrix product of that type takes), then the piece's rows of dW are G^T h, written once, and
// dh's FP32 sums grow by G W.  So each piece of W is read once for all rows, where slices of rows would read W, and
// add to dW, once a slice.
//
// Rows that are not scored reach nothing, whatever they hold: the scored ones are copied together first, and the
// products end with them (how many they are is known on the device only); 16 rows or fewer are all multiplied, and only the losses
// tell them apart.  The matrix products bound all of it (6 T H V operations forward
// and backward and 2 T H V for the logits again); a few rows are the weights read once, which HBM bounds.  (16384 rows of 32000 x 4096 BF16: logits 3.3-3.4 ms,
// 1255-1285 TFLOP/s; G, dW and dh of a half of the words 1.67-1.72, 1.68-1.72, 1.72-1.78, 1210-1290.  8 rows of 151936 x 896: 46 us, 5.9 TB/s.)

#include <hip/hip_runtime.h>

#include <stdint.h>

#include <algorithm>

#include "../../include/adambridge_hip.h"
#include "abh_device.hpp"
#include "abh_host.hpp"
#include "abh_rows.hpp"
#include "abh_tiles.hpp"

namespace abh {

constexpr float kHeadLog2e = 1.4426950408889634f;
constexpr float kHeadNegInf = -__builtin_inff();
constexpr int kHeadCus = 256;
constexpr int kFewGroups = 2;        // words, by 16, of a wavefront of k_head_few
constexpr int kFinishLanes = 1024;

// A maximum and the sum of exp(x - m) over what was seen.  m = -inf: nothing above -inf yet.
struct Sums {
    float m, s;
};

// x - m and its product with log2 e are rounded to FP32, so that the largest logit's exponential is exact, one of e^-8 off by at most
// 2^-20 of itself; expf, which is exact to a step, takes several instructions of each of a tile's logits to one here.
__device__ __forceinline__ float exp_of(float x, float m) { return __builtin_amdgcn_exp2f((x - m) * kHeadLog2e); }
// The subtrahend that stands for a maximum, so that exp(-inf + inf) is never taken.
__device__ __forceinline__ float shift_for(float m) { return m == kHeadNegInf ? 0.0f : m; }

__device__ __forceinline__ Sums merged(const Sums a, const Sums b)
{
    const float m = __builtin_fmaxf(a.m, b.m), t = shift_for(m);
    return Sums{m, a.s * exp_of(a.m, t) + b.s * exp_of(b.m, t)};
}

// A scored row's target (-1: none of the vocabulary's), and what its gradient takes.
struct HeadRow {
    int32_t word;
    float top, scale, seed;   // the logits' maximum, gout / sum, gout
};

struct HeadArgs {
    const void* h;            // the scored rows, together: count x hidden
    const void* w;            // vocab x hidden
    const int64_t* targets;   // of all rows
    const HeadRow* facts;     // of the scored rows
    const int32_t* count;     // how many are scored
    int32_t rows, hidden;     // rows: all
    int64_t vocab, v0;        // the piece: words v0 .. v0 + width
    int32_t width, pitch;     // pitch: a row of G
    int32_t tiles_j, splits;  // splits: of the logits' or dW's terms
    float* parts;             // of split sums: splits x rows x pitch, or splits x width x hidden
    Sums* part;               // column tiles x rows
    float* picked;            // a scored row's logit of its target
    void* g;                  // count x pitch
    float* dh;                // parts x count x hidden
    void* dw;                 // vocab x hidden
    int32_t fresh;            // dh's first piece
    int32_t places;           // tiles that the CUs hold at a time
};

// ------------------------------------------------------------------------ the scored rows

// index[i] = the i-th scored row, place[t] = its number or -1; losses of the others are 0.  One workgroup.
__global__ __launch_bounds__(1024) void k_head_rows(const int64_t* targets, int64_t ignore, int32_t rows, int32_t* index, int32_t* place,
                                                    int32_t* count, float* losses)
{
    __shared__ int32_t waves[2][16];
    const int lane = threadIdx.x & 63, wave = threadIdx.x / kWave;
    int32_t before = 0;
    for (int32_t t0 = 0, turn = 0; t0 < rows; t0 += 1024, turn ^= 1) {
        const int32_t t = t0 + (int32_t)threadIdx.x;
        const bool scored = t < rows && targets[t] != ignore;
        const uint64_t mask = __builtin_amdgcn_ballot_w64(scored);
        if (lane == 0) waves[turn][wave] = __builtin_popcountll(mask);
        __syncthreads();
        int32_t at = before, all = 0;
#pragma unroll
        for (int w = 0; w < 16; ++w) {
            const int32_t n = waves[turn][w];
            at += w < wave ? n : 0;
            all += n;
        }
        before += all;
        at += __builtin_popcountll(mask & (((uint64_t)1 << lane) - 1));
        if (scored) index[at] = t;
        if (t < rows) {
            if (place) place[t] = scored ? at : -1;
            if (losses && !scored) losses[t] = 0.0f;
        }
    }
    if (threadIdx.x == 0) *count = before;
}

// What the gather kernel takes for the rows' facts.  gout, stats: of all rows (maximum, 1 / sum); NULL in the forward call.
struct HeadFacts {
    HeadRow* out;
    int64_t vocab;
    const float *stats, *gout;
    __device__ __forceinline__ void put(int64_t to, int64_t from, int64_t target) const
    {
        HeadRow row{target < 0 || target >= vocab ? -1 : (int32_t)target, 0.0f, 0.0f, 0.0f};
        if (gout) {
            row.seed = row.word < 0 ? __builtin_nanf("") : gout[from];
            row.top = stats[2 * from];
            row.scale = stats[2 * from + 1] * row.seed;
        }
        out[to] = row;
    }
};

// The scored rows of h, together: a row a workgroup.  FIND: a row counts the scored ones before it for itself, which for a few
// thousand rows is less than another launch (the row's place is one of T; what k_head_rows writes is written here).
template <int DT, bool FIND>
__global__ __launch_bounds__(256) void k_head_gather(const void* h, const int64_t* targets, int64_t ignore, int32_t rows, int32_t* index, int32_t* place,
                                                     int32_t* count, float* losses, HeadFacts facts, int32_t hidden, void* out)
{
    constexpr int L = kLane<DT>;
    int64_t to = block_index(), from;
    if constexpr (FIND) {
        __shared__ int32_t part[4];
        from = to;
        const bool scored = targets[from] != ignore;
        int32_t n = 0;
        for (int64_t t = threadIdx.x; t < from; t += 256) n += targets[t] != ignore;
        n = group_reduce<kWave>(n, [](int32_t a, int32_t b) { return a + b; });
        if (threadIdx.x % kWave == 0) part[threadIdx.x / kWave] = n;
        __syncthreads();
        n = part[0] + part[1] + part[2] + part[3];
        if (threadIdx.x == 0) {
            if (scored) index[n] = (int32_t)from;
            if (place) place[from] = scored ? n : -1;
            if (losses && !scored) losses[from] = 0.0f;
            if (from == rows - 1) *count = n + scored;
        }
        if (!scored) return;
        to = n;
    } else {
        if (to >= *count) return;
        from = index[to];
    }
    if (threadIdx.x == 0) facts.put(to, from, targets[from]);
    const void* row = at<DT>(h, from * hidden);
    void* copy = at<DT>(out, to * hidden);
    for (int32_t c = threadIdx.x * L; c < hidden; c += 256 * L) {
        if (c + L <= hidden) {
            store_raw<DT>(copy, c, load_raw<DT>(row, c));
        } else {
            for (int32_t k = c; k < hidden; ++k) put<DT>(copy, k, get<DT>(row, k));
        }
    }
}

// ------------------------------------------------------------------------------ tiles

struct HeadTile {
    int ti, tj, split;
};

// This workgroup's of tiles_i x tiles_j tiles in `splits` parts: consecutive ones to one XCD, kGroupTiles row tiles at a time
// down the columns.
__device__ __forceinline__ bool head_tile(int tiles_i, int tiles_j, int splits, HeadTile& t)
{
    const int items = tiles_i * tiles_j * splits, per = (items + kXcd - 1) / kXcd;
    const int block = (int)block_index(), slot = block / kXcd, item = block % kXcd * per + slot;
    if (slot >= per || item >= items) return false;
    const int idx = item / splits;
    t.split = scalar(item - idx * splits);
    const int g = idx / (kGroupTiles * tiles_j), first = g * kGroupTiles;
    const int wide = tiles_i - first < kGroupTiles ? tiles_i - first : kGroupTiles;
    const int r = idx - first * tiles_j;
    t.ti = scalar(first + r % wide);
    t.tj = scalar(r / wide);
    return true;
}

// How many parts sums are cut in whose tiles are few: so that they fill the CUs' places, of 512 terms or more.
__device__ __host__ __forceinline__ int splits_of(int64_t tiles, int places, int64_t terms)
{
    const int64_t fit = places / (tiles < 1 ? 1 : tiles), most = terms / 512;
    const int64_t n = fit < most ? fit : most;
    return (int)(n < 1 ? 1 : n);
}

// A part's terms: whole steps.
struct HeadTerms {
    int first, len;
};
template <class H>
__device__ __forceinline__ HeadTerms terms_of(int terms, int split, int splits)
{
    const int steps = (terms + H::BK - 1) / H::BK;
    const int k0 = scalar(steps * split / splits * H::BK), k1 = scalar(steps * (split + 1) / splits * H::BK);
    const int len = (k1 < terms ? k1 : terms) - k0;
    return HeadTerms{k0, len < 0 ? 0 : len};
}

// What a kernel's type and tile are.  BF16: abh_tiles.hpp's; FP32: B x B of four wavefronts.
template <class C_, bool EVEN_>
struct HeadBf16 {
    typedef C_ C;
    static constexpr int DT = DT_BF16, BM = C::BM, BN = C::BN, BK = C::BK, WJ = C::WJ, T = C::T, OCC = C::OCC;
    static constexpr int NI = BM / C::WI / 16, NJ = BN / WJ / 16, R = 4, SIDE = 16;   // sums of 16 x 16, four a lane
    typedef mm_f32x4 Sum;
    static constexpr bool EVEN = EVEN_;
    static constexpr int LDS = C::NB * C::BYTES;
    static __device__ __forceinline__ int wi() { return (int)threadIdx.x / kWave / WJ * (BM / C::WI); }
    static __device__ __forceinline__ int wj() { return (int)threadIdx.x / kWave % WJ * (BN / WJ); }
};
template <int B>
struct HeadF32 {
    static constexpr int DT = DT_F32, BM = B, BN = B, BK = 32, NI = B / 64, NJ = B / 64, WJ = 2, T = 256, OCC = 2, R = 16, SIDE = 32;
    typedef mm_f32x16 Sum;
    static constexpr bool EVEN = false;
    static constexpr int LDS = 2 * 2 * B * 32 * 4;
    static __device__ __forceinline__ int wi() { return (int)(threadIdx.x / kWave & 1) * (B / 2); }
    static __device__ __forceinline__ int wj() { return (int)(threadIdx.x / kWave >> 1) * (B / 2); }
};

// One operand of a tile.  LONG: p is its first row, `rows` of them are left; else p is the operand's first term, its rows have
// `rows` values and the tile begins at `first`.  len: terms.
struct Operand {
    const uint8_t* p;
    int pitch, first, rows, len;
};

// The tile's sums; false where the wavefront has no row.
template <class H, bool ALONG, bool BLONG>
__device__ __forceinline__ bool head_multiply(uint8_t* lds, const Operand& a, const Operand& b, bool live, typename H::Sum (&acc)[H::NI][H::NJ])
{
    const int steps = ((a.len > b.len ? a.len : b.len) + H::BK - 1) / H::BK;
    if constexpr (H::DT == DT_BF16) {
        typedef typename H::C C;
        TileFeed<ALONG, H::BM, H::BK, C::W, H::EVEN> fa;
        TileFeed<BLONG, H::BN, H::BK, C::W, H::EVEN> fb;
        if constexpr (H::EVEN) {   // (rows past the operand's last: zeros)
            fa.start(ALONG ? a.p : a.p + (int64_t)a.first * 2, a.pitch * 2, a.rows, a.len, ALONG ? 0 : a.first * 2);
            fb.start(BLONG ? b.p : b.p + (int64_t)b.first * 2, b.pitch * 2, b.rows, b.len, BLONG ? 0 : b.first * 2);
        } else {
            fa.start(a.p, a.pitch, ALONG ? 0 : a.first, a.rows, a.len);
            fb.start(b.p, b.pitch, BLONG ? 0 : b.first, b.rows, b.len);
        }
        if constexpr (std::is_same<C, WideTile>::value) {
            multiply_wide<C, ALONG, BLONG>(lds, fa, fb, steps, H::wi(), H::wj(), acc);
            return true;
        } else {
            return multiply_tile16<C, ALONG, BLONG, H::EVEN>(lds, fa, fb, steps, H::wi(), H::wj(), live, acc);
        }
    } else {
        StagedFeed<DT_F32, ALONG, H::BM, 32, 4> fa;
        StagedFeed<DT_F32, BLONG, H::BN, 32, 4> fb;
        fa.start(a.p, a.pitch, ALONG ? 0 : a.first, a.rows, a.len);
        fb.start(b.p, b.pitch, BLONG ? 0 : b.first, b.rows, b.len);
        multiply_tile_f32<H::BM, ALONG, BLONG>(*reinterpret_cast<uint8_t(*)[2][2 * H::BM * 32 * 4]>(lds), fa, fb, steps, H::wi(), H::wj(), acc);
        return true;
    }
}

// Column of the tile that is a lane's value r of its columns j, and its row of the rows i.
template <class H>
__device__ __forceinline__ int column_of(int wj, int j, int r)
{
    const int lane = threadIdx.x & 63;
    if constexpr (H::SIDE == 16) return wj + 16 * j + 4 * (lane >> 4) + r;
    else return wj + 32 * j + 8 * (r >> 2) + 4 * (lane >> 5) + (r & 3);
}
template <class H>
__device__ __forceinline__ int row_of(int wi, int i) { return wi + H::SIDE * i + (int)(threadIdx.x & (H::SIDE - 1)); }

// op over the lanes that have a row's values.
template <class H, class Op>
__device__ __forceinline__ float over_row(float x, Op op)
{
    if constexpr (H::SIDE == 16) x = op(x, __shfl_xor(x, 16));
    return op(x, __shfl_xor(x, 32));
}

// A target's column in the tile that begins at word `first`; -1 outside the tile.
__device__ __forceinline__ int hot_column(int word, int64_t first, int limit) { return word >= first && word < first + limit ? (int)(word - first) : -1; }

// What lies behind the vocabulary's last word.
template <class H>
__device__ __forceinline__ void mask_columns(typename H::Sum (&acc)[H::NI][H::NJ], int wj, int limit, float to)
{
#pragma unroll
    for (int i = 0; i < H::NI; ++i)
#pragma unroll
        for (int j = 0; j < H::NJ; ++j)
#pragma unroll
            for (int r = 0; r < H::R; ++r)
                if (column_of<H>(wj, j, r) >= limit) acc[i][j][r] = to;
}

// The tile's sums in FP32.
template <class H>
__device__ __forceinline__ void store_sums(float* out, int64_t pitch, int limit_i, int limit_j, const typename H::Sum (&acc)[H::NI][H::NJ], int wi, int wj)
{
#pragma unroll
    for (int i = 0; i < H::NI; ++i) {
        const int row = row_of<H>(wi, i);
        if (row >= limit_i) continue;
#pragma unroll
        for (int j = 0; j < H::NJ; ++j)
#pragma unroll
            for (int q = 0; q < H::R / 4; ++q) {
                const float four[4] = {acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
                store_like<DT_F32, 4>(out + row * pitch, column_of<H>(wj, j, 4 * q), limit_j, four);
            }
    }
}

// --------------------------------------------------------------- few tiles: logits in parts
//
// Where the logits' tiles are too few for the CUs, their sums are cut along the terms: parts in FP32, which a workgroup a row adds
// in order on its way over the row.

template <class H>
__global__ __launch_bounds__(H::T, H::OCC) void k_head_logits(HeadArgs A)
{
    __shared__ __attribute__((aligned(1024))) uint8_t lds[H::LDS];
    const int count = scalar(*A.count);
    HeadTile t;
    if (!head_tile((count + H::BM - 1) / H::BM, A.tiles_j, A.splits, t)) return;
    const int i0 = t.ti * H::BM, j0 = t.tj * H::BN, limit_i = count - i0, limit_j = A.width - j0;
    const HeadTerms k = terms_of<H>(A.hidden, t.split, A.splits);
    const Operand a{at<H::DT>(A.h, (int64_t)i0 * A.hidden + k.first), A.hidden, 0, limit_i, k.len};
    const Operand b{at<H::DT>(A.w, (A.v0 + j0) * A.hidden + k.first), A.hidden, 0, limit_j, k.len};
    typename H::Sum acc[H::NI][H::NJ];
    const int wi = H::wi(), wj = H::wj();
    if (!head_multiply<H, true, true>(lds, a, b, wi < limit_i, acc)) return;
    store_sums<H>(A.parts + ((int64_t)t.split * A.rows + i0) * A.pitch + j0, A.pitch, limit_i, limit_j, acc, wi, wj);
}

// Four logits of a row, from word v of the piece; to: what stands behind the last word.
__device__ __forceinline__ void joined(const HeadArgs& A, int64_t row, int v, float to, float (&x)[4])
{
#pragma unroll
    for (int k = 0; k < 4; ++k) x[k] = 0.0f;
    for (int s = 0; s < A.splits; ++s) {
        float y[4];
        to_floats<DT_F32>(load_raw<DT_F32>(A.parts + ((int64_t)s * A.rows + row) * A.pitch, v), y);   // a row has whole pieces
#pragma unroll
        for (int k = 0; k < 4; ++k) x[k] += y[k];
    }
#pragma unroll
    for (int k = 0; k < 4; ++k)
        if (v + k >= A.width) x[k] = to;
}

// A row's loss, and what the gradient takes.
__device__ __forceinline__ void finish_row(Sums all, float picked, int64_t t, int64_t target, int64_t vocab, int64_t ignore, float* losses, float* stats)
{
    if (all.m == kHeadNegInf) all.s = __builtin_nanf("");   // every logit -inf: no distribution
    if (stats) {
        stats[2 * t] = all.m;
        stats[2 * t + 1] = 1.0f / all.s;
    }
    losses[t] = target == ignore ? 0.0f : target < 0 || target >= vocab ? __builtin_nanf("") : logf(all.s) - (picked - all.m);
}

// The losses, LANES a row: the whole vocabulary is one piece here.
template <int LANES>
__global__ __launch_bounds__(LANES < 256 ? 256 : LANES) void k_head_join(HeadArgs A, const int32_t* index, const int64_t* targets, int64_t ignore,
                                                                        float* losses, float* stats)
{
    constexpr int ROWS = LANES < 256 ? 256 / LANES : 1, WAVES = LANES / kWave;
    __shared__ Sums waves[ROWS][WAVES];
    __shared__ float picked[ROWS];
    const int slot = threadIdx.x / LANES, lane = threadIdx.x % LANES;
    const int64_t row = block_index() * ROWS + slot;
    const bool real = row < *A.count;
    const int word = real ? A.facts[row].word : -1;
    Sums all{kHeadNegInf, 0.0f};
    if (real)
        for (int v = lane * 4; v < A.width; v += LANES * 4) {
            float x[4];
            joined(A, row, v, kHeadNegInf, x);
            const float m = __builtin_fmaxf(__builtin_fmaxf(all.m, x[0]), __builtin_fmaxf(__builtin_fmaxf(x[1], x[2]), x[3])), shift = shift_for(m);
            float s = all.s * exp_of(all.m, shift);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                s += exp_of(x[k], shift);
                if (v + k == word) picked[slot] = x[k];
            }
            all = Sums{m, s};
        }
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) all = merged(all, Sums{__shfl_xor(all.m, d), __shfl_xor(all.s, d)});
    if (lane % kWave == 0) waves[slot][lane / kWave] = all;
    __syncthreads();
    if (lane || !real) return;
    all = waves[slot][0];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) all = merged(all, waves[slot][w]);
    const int64_t t = index[row];
    finish_row(all, picked[slot], t, targets[t], A.vocab, ignore, losses, stats);
}

// A piece's gradient at the logits: 4 words a lane, zeros behind the last one up to whole pieces.
template <int DT>
__global__ __launch_bounds__(256) void k_head_join_grad(HeadArgs A, int32_t columns)
{
    const int64_t row = block_index() / columns;
    if (row >= *A.count) return;
    const int v = ((int)(block_index() - row * columns) * 256 + (int)threadIdx.x) * 4;
    if (v >= ((A.width + 7) & ~7)) return;
    const HeadRow facts = A.facts[row];
    float x[4];
    joined(A, row, v, 0.0f, x);
#pragma unroll
    for (int k = 0; k < 4; ++k)
        x[k] = v + k < A.width ? exp_of(x[k], facts.top) * facts.scale - (A.v0 + v + k == facts.word ? facts.seed : 0.0f) : 0.0f;
    store_like<DT, 4>(at<DT>(A.g, row * A.pitch), v, A.pitch, x);
}

// ------------------------------------------------------------------------------ forward

// Each row's maximum and sum over the tile's words, and the target's logit.
template <class H>
__global__ __launch_bounds__(H::T, H::OCC) void k_head_sums(HeadArgs A)
{
    __shared__ __attribute__((aligned(1024))) uint8_t lds[H::LDS];
    __shared__ Sums row_sums[H::WJ][H::BM];
    const int count = scalar(*A.count);
    HeadTile t;
    if (!head_tile((count + H::BM - 1) / H::BM, A.tiles_j, 1, t)) return;
    const int i0 = t.ti * H::BM, j0 = t.tj * H::BN, limit_i = count - i0, limit_j = A.width - j0;
    const Operand a{at<H::DT>(A.h, (int64_t)i0 * A.hidden), A.hidden, 0, limit_i, A.hidden};
    const Operand b{at<H::DT>(A.w, (A.v0 + j0) * A.hidden), A.hidden, 0, limit_j, A.hidden};
    typename H::Sum acc[H::NI][H::NJ];
    const int wi = H::wi(), wj = H::wj(), lane = threadIdx.x & 63;
    int word[H::NI];   // the rows' targets, asked for before the product, with no condition: eight loads on their way at once
#pragma unroll
    for (int i = 0; i < H::NI; ++i) {
        const int row = row_of<H>(wi, i);
        word[i] = A.facts[i0 + (row < limit_i ? row : 0)].word;
    }
    const bool live = head_multiply<H, true, true>(lds, a, b, wi < limit_i, acc);
    if (live) {
        if (limit_j < H::BN) mask_columns<H>(acc, wj, limit_j, kHeadNegInf);
#pragma unroll
        for (int i = 0; i < H::NI; ++i) {
            const int row = row_of<H>(wi, i), hot = row < limit_i ? hot_column(word[i], j0, limit_j) : -1;
            if (__builtin_amdgcn_ballot_w64(hot >= wj && hot < wj + H::BN / H::WJ)) {
#pragma unroll
                for (int j = 0; j < H::NJ; ++j)
#pragma unroll
                    for (int r = 0; r < H::R; ++r)
                        if (column_of<H>(wj, j, r) == hot) A.picked[i0 + row] = acc[i][j][r];
            }
            float m = kHeadNegInf;
#pragma unroll
            for (int j = 0; j < H::NJ; ++j)
#pragma unroll
                for (int r = 0; r < H::R; ++r) m = __builtin_fmaxf(m, acc[i][j][r]);
            m = over_row<H>(m, [](float a, float b) { return __builtin_fmaxf(a, b); });
            const float shift = shift_for(m);
            float s = 0.0f;
#pragma unroll
            for (int j = 0; j < H::NJ; ++j)
#pragma unroll
                for (int r = 0; r < H::R; ++r) s += exp_of(acc[i][j][r], shift);
            s = over_row<H>(s, [](float a, float b) { return a + b; });
            if (lane < H::SIDE) row_sums[wj / (H::BN / H::WJ)][row] = Sums{m, s};
        }
    }
    __syncthreads();
    for (int row = threadIdx.x; row < H::BM && row < limit_i; row += H::T) {
        Sums all = row_sums[0][row];
#pragma unroll
        for (int w = 1; w < H::WJ; ++w) all = merged(all, row_sums[w][row]);
        A.part[(int64_t)t.tj * A.rows + i0 + row] = all;
    }
}

// The same of 16 rows or fewer: the weights are read once, NG times 16 words a wavefront, which share the rows' loads.  part:
// workgroups x rows.
template <int DT, bool EVEN>
__global__ __launch_bounds__(256) void k_head_few(HeadArgs A)
{
    constexpr int V = kLane<DT>, STEP = 4 * V, NG = kFewGroups, U = 4;
    __shared__ Sums row_sums[4][16];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / kWave);
    const int col = lane & 15, quarter = lane >> 4;
    const int64_t j0 = (block_index() * 4 + wave) * (16 * NG);
    const int words = j0 >= A.vocab ? 0 : (int)(A.vocab - j0 < 16 * NG ? A.vocab - j0 : 16 * NG);
    const int steps = words ? (A.hidden + STEP - 1) / STEP : 0;
    const Pieces<DT, EVEN> w{at<DT>(A.w, (words ? j0 : 0) * A.hidden), (uint32_t)(words * A.hidden * kSize<DT>), A.hidden, words};
    const Pieces<DT, EVEN> x{static_cast<const uint8_t*>(A.h), (uint32_t)(A.rows * A.hidden * kSize<DT>), A.hidden, A.rows};
    mm_f32x4 acc[NG];
#pragma unroll
    for (int n = 0; n < NG; ++n) acc[n] = mm_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    raw16 even[NG][U], odd[NG][U];   // (BF16's products are exact in FP32, and a row's sum is one chain of its size / 32 steps)
    auto load = [&](int s, raw16 (&to)[NG][U]) {
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int n = 0; n < NG; ++n) to[n][u] = w.load(16 * n + col, (s + u) * STEP + quarter * V, s + u < steps);
    };
    // loads arrive in their order: a step's rows are asked for before the next one's weights, which are then on their way while
    // this one is multiplied
    auto turn = [&](int s, const raw16 (&now)[NG][U], raw16 (&next)[NG][U]) {
        raw16 xv[U];
#pragma unroll
        for (int u = 0; u < U; ++u) xv[u] = x.load(col, (s + u) * STEP + quarter * V, s + u < steps);
        __builtin_amdgcn_sched_barrier(0);
        if (s + U < steps) load(s + U, next);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int n = 0; n < NG; ++n) {
            mm_f32x4 some = DT == DT_BF16 ? acc[n] : mm_f32x4{0.0f, 0.0f, 0.0f, 0.0f};   // FP32: short chains of sums
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if constexpr (DT == DT_BF16) {
                    some = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(mm_bf16x8, now[n][u]), __builtin_bit_cast(mm_bf16x8, xv[u]), some, 0, 0, 0);
                } else {
                    const mm_f32x4 wf = __builtin_bit_cast(mm_f32x4, now[n][u]), xf = __builtin_bit_cast(mm_f32x4, xv[u]);
#pragma unroll
                    for (int q = 0; q < 4; ++q) some = __builtin_amdgcn_mfma_f32_16x16x4f32(wf[q], xf[q], some, 0, 0, 0);
                }
            }
            if constexpr (DT == DT_BF16) acc[n] = some;
            else acc[n] += some;
        }
    };
    if (steps) load(0, even);
    for (int s = 0; s < steps; s += 2 * U) {
        turn(s, even, odd);
        if (s + U < steps) turn(s + U, odd, even);
    }
    const int64_t target = col < A.rows ? A.targets[col] : -1;
    const int hot = target >= j0 && target < j0 + words ? (int)(target - j0) : -1;   // (a target may be any number)
    Sums all{kHeadNegInf, 0.0f};
#pragma unroll
    for (int n = 0; n < NG; ++n)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int word = 16 * n + 4 * quarter + r;
            if (word >= words) acc[n][r] = kHeadNegInf;
            else if (word == hot) A.picked[col] = acc[n][r];
            all.m = __builtin_fmaxf(all.m, acc[n][r]);
        }
    all.m = __builtin_fmaxf(all.m, __shfl_xor(all.m, 16));
    all.m = __builtin_fmaxf(all.m, __shfl_xor(all.m, 32));
    const float shift = shift_for(all.m);
#pragma unroll
    for (int n = 0; n < NG; ++n)
#pragma unroll
        for (int r = 0; r < 4; ++r) all.s += exp_of(acc[n][r], shift);
    all.s += __shfl_xor(all.s, 16);
    all.s += __shfl_xor(all.s, 32);
    if (quarter == 0) row_sums[wave][col] = all;
    __syncthreads();
    if ((int)threadIdx.x < A.rows) {
        Sums sums = row_sums[0][threadIdx.x];
#pragma unroll
        for (int k = 1; k < 4; ++k) sums = merged(sums, row_sums[k][threadIdx.x]);
        A.part[block_index() * A.rows + threadIdx.x] = sums;
    }
}

// The parts of R rows a workgroup, in an order of their own; losses, and what the gradient takes.  index: NULL where the parts'
// rows are all rows.
template <int R>
__global__ __launch_bounds__(kFinishLanes) void k_head_finish(const Sums* part, int32_t parts, int32_t stride, const int32_t* index, const int32_t* count,
                                                              const int64_t* targets, int64_t vocab, int64_t ignore, const float* picked, float* losses,
                                                              float* stats)
{
    constexpr int S = kFinishLanes / R;
    __shared__ Sums tree[S][R];
    const int r = threadIdx.x % R, slice = threadIdx.x / R;
    const int64_t row = block_index() * R + r, rows = index ? *count : stride;
    if (block_index() * R >= rows) return;
    Sums all{kHeadNegInf, 0.0f};
    if (row < rows)
        for (int32_t p = slice; p < parts; p += 4 * S) {   // four reads on their way
            Sums next[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) next[k] = part[(int64_t)(p + k * S < parts ? p + k * S : p) * stride + row];
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (p + k * S < parts) all = merged(all, next[k]);
        }
    tree[slice][r] = all;
    __syncthreads();
#pragma unroll
    for (int d = S / 2; d > 0; d >>= 1) {
        if (slice < d) tree[slice][r] = merged(tree[slice][r], tree[slice + d][r]);
        __syncthreads();
    }
    if (slice || row >= rows) return;
    const int64_t t = index ? index[row] : row;
    finish_row(tree[0][r], picked[row], t, targets[t], vocab, ignore, losses, stats);
}

// ------------------------------------------------------------------------------ backward

// A piece's gradient at the logits.
template <class H>
__global__ __launch_bounds__(H::T, H::OCC) void k_head_grad(HeadArgs A)
{
    __shared__ __attribute__((aligned(1024))) uint8_t lds[H::LDS];
    const int count = scalar(*A.count);
    HeadTile t;
    if (!head_tile((count + H::BM - 1) / H::BM, A.tiles_j, 1, t)) return;
    const int i0 = t.ti * H::BM, j0 = t.tj * H::BN, limit_i = count - i0, limit_j = A.width - j0;
    const Operand a{at<H::DT>(A.h, (int64_t)i0 * A.hidden), A.hidden, 0, limit_i, A.hidden};
    const Operand b{at<H::DT>(A.w, (A.v0 + j0) * A.hidden), A.hidden, 0, limit_j, A.hidden};
    typename H::Sum acc[H::NI][H::NJ];
    const int wi = H::wi(), wj = H::wj();
    // the rows' numbers, asked for before the product, with no condition
    HeadRow facts[H::NI];
#pragma unroll
    for (int i = 0; i < H::NI; ++i) {
        const int row = row_of<H>(wi, i);
        facts[i] = A.facts[i0 + (row < limit_i ? row : 0)];
    }
    if (!head_multiply<H, true, true>(lds, a, b, wi < limit_i, acc)) return;
#pragma unroll
    for (int i = 0; i < H::NI; ++i) {
        const int hot = hot_column(facts[i].word, A.v0 + j0, limit_j);
#pragma unroll
        for (int j = 0; j < H::NJ; ++j)
#pragma unroll
            for (int r = 0; r < H::R; ++r) acc[i][j][r] = exp_of(acc[i][j][r], facts[i].top) * facts[i].scale;
        if (__builtin_amdgcn_ballot_w64(hot >= wj && hot < wj + H::BN / H::WJ)) {
#pragma unroll
            for (int j = 0; j < H::NJ; ++j)
#pragma unroll
                for (int r = 0; r < H::R; ++r) acc[i][j][r] -= column_of<H>(wj, j, r) == hot ? facts[i].seed : 0.0f;
        }
    }
    if (limit_j < H::BN) mask_columns<H>(acc, wj, limit_j, 0.0f);
    const int wide = (limit_j + 7) & ~7;   // whole pieces: zeros behind the vocabulary's last word
    if constexpr (H::DT == DT_BF16) {
        store_bf16<typename H::C, true>(at<DT_BF16>(A.g, (int64_t)i0 * A.pitch + j0), A.pitch, limit_i, wide, acc, wi, wj);
    } else {
#pragma unroll
        for (int i = 0; i < H::NI; ++i) {
            const int row = row_of<H>(wi, i);
            if (row >= limit_i) continue;
            float* out = static_cast<float*>(A.g) + (int64_t)(i0 + row) * A.pitch + j0;
#pragma unroll
            for (int j = 0; j < H::NJ; ++j)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int c = column_of<H>(wj, j, 4 * q);
                    if (c < wide) *reinterpret_cast<mm_f32x4*>(out + c) = mm_f32x4{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
                }
        }
    }
}

// dh (FP32) += G W of a piece.
template <class H>
__global__ __launch_bounds__(H::T, H::OCC) void k_head_dh(HeadArgs A)
{
    __shared__ __attribute__((aligned(1024))) uint8_t lds[H::LDS];
    const int count = scalar(*A.count), tiles_i = (count + H::BM - 1) / H::BM;
    const int splits = splits_of((int64_t)tiles_i * A.tiles_j, A.places, A.pitch);   // by the pitch: the same for every piece
    HeadTile t;
    if (!head_tile(tiles_i, A.tiles_j, splits, t)) return;
    const int i0 = t.ti * H::BM, j0 = t.tj * H::BN, limit_i = count - i0, limit_j = A.hidden - j0;
    const HeadTerms k = terms_of<H>(A.width, t.split, splits);
    if (k.len == 0 && !A.fresh) return;
    // G has zeros up to whole pieces, where W has ended
    const Operand a{at<H::DT>(A.g, (int64_t)i0 * A.pitch + k.first), A.pitch, 0, limit_i, (k.len + 7) & ~7};
    const Operand b{at<H::DT>(A.w, (A.v0 + k.first) * A.hidden), A.hidden, j0, A.hidden, k.len};
    typename H::Sum acc[H::NI][H::NJ];
    const int wi = H::wi(), wj = H::wj();
    if (!head_multiply<H, true, false>(lds, a, b, wi < limit_i, acc)) return;
    float* out = A.dh + ((int64_t)t.split * count + i0) * A.hidden + j0;
#pragma unroll
    for (int i = 0; i < H::NI; ++i) {
        const int row = row_of<H>(wi, i);
        if (row >= limit_i) continue;
#pragma unroll
        for (int j = 0; j < H::NJ; ++j)
#pragma unroll
            for (int q = 0; q < H::R / 4; ++q) {
                const int c = column_of<H>(wj, j, 4 * q);
                float four[4] = {acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
                if (!A.fresh) {
                    float old[4];
                    load_like<DT_F32, 4>(out + (int64_t)row * A.hidden, c, limit_j, 0.0f, old);
#pragma unroll
                    for (int k = 0; k < 4; ++k) four[k] += old[k];
                }
                store_like<DT_F32, 4>(out + (int64_t)row * A.hidden, c, limit_j, four);
            }
    }
}

// A piece's rows of dW.
template <class H>
__global__ __launch_bounds__(H::T, H::OCC) void k_head_dw(HeadArgs A)
{
    __shared__ __attribute__((aligned(1024))) uint8_t lds[H::LDS];
    const int count = scalar(*A.count);
    HeadTile t;
    if (!head_tile((A.width + H::BM - 1) / H::BM, A.tiles_j, A.splits, t)) return;
    const int i0 = t.ti * H::BM, j0 = t.tj * H::BN, limit_i = A.width - i0, limit_j = A.hidden - j0;
    const HeadTerms k = terms_of<H>(count, t.split, A.splits);
    const Operand a{at<H::DT>(A.g, (int64_t)k.first * A.pitch), A.pitch, i0, A.pitch, k.len};
    const Operand b{at<H::DT>(A.h, (int64_t)k.first * A.hidden), A.hidden, j0, A.hidden, k.len};
    typename H::Sum acc[H::NI][H::NJ];
    const int wi = H::wi(), wj = H::wj();
    if (!head_multiply<H, false, false>(lds, a, b, wi < limit_i, acc)) return;
    if (A.splits > 1) {
        store_sums<H>(A.parts + ((int64_t)t.split * A.width + i0) * A.hidden + j0, A.hidden, limit_i, limit_j, acc, wi, wj);
        return;
    }
    uint8_t* out = at<H::DT>(A.dw, (A.v0 + i0) * A.hidden + j0);
    if constexpr (H::DT == DT_BF16) store_bf16<typename H::C, H::EVEN>(out, A.hidden, limit_i, limit_j, acc, wi, wj);
    else store_sums<H>(reinterpret_cast<float*>(out), A.hidden, limit_i, limit_j, acc, wi, wj);
}

// A row of dW a workgroup: its parts, in order.
template <int DT>
__global__ __launch_bounds__(256) void k_head_join_dw(HeadArgs A)
{
    constexpr int L = kLane<DT>;
    const int64_t v = block_index();
    if (v >= A.width) return;
    void* out = at<DT>(A.dw, (A.v0 + v) * A.hidden);
    for (int32_t c = threadIdx.x * L; c < A.hidden; c += 256 * L) {
        float x[L];
#pragma unroll
        for (int k = 0; k < L; ++k) x[k] = 0.0f;
        for (int s = 0; s < A.splits; ++s) {
            float y[L];
            load_like<DT_F32, L>(A.parts + ((int64_t)s * A.width + v) * A.hidden, c, A.hidden, 0.0f, y);
#pragma unroll
            for (int k = 0; k < L; ++k) x[k] += y[k];
        }
        stream_vec<DT>(out, c, A.hidden, x);
    }
}

// dh's rows at their places, the parts summed in order and rounded once; zeros for rows that are not scored.
template <int DT>
__global__ __launch_bounds__(256) void k_head_scatter(const float* sums, const int32_t* place, const int32_t* count, int32_t rows, int32_t hidden,
                                                      int32_t tile_m, int32_t tile_n, int32_t places, int32_t width, void* dh)
{
    constexpr int L = kLane<DT>;
    const int64_t t = block_index();
    if (t >= rows) return;
    const int n = *count, p = place[t];
    const int splits = splits_of((int64_t)((n + tile_m - 1) / tile_m) * ((hidden + tile_n - 1) / tile_n), places, width);
    void* out = at<DT>(dh, t * hidden);
    for (int32_t c = threadIdx.x * L; c < hidden; c += 256 * L) {
        float x[L];
#pragma unroll
        for (int k = 0; k < L; ++k) x[k] = 0.0f;
        if (p >= 0)
            for (int s = 0; s < splits; ++s) {
                float y[L];
                load_like<DT_F32, L>(sums + ((int64_t)s * n + p) * hidden, c, hidden, 0.0f, y);
#pragma unroll
                for (int k = 0; k < L; ++k) x[k] += y[k];
            }
        stream_vec<DT>(out, c, hidden, x);
    }
}

// ------------------------------------------------------------------------------ launches

constexpr int64_t kHeadRows = (int64_t)1 << 23, kHeadVocab = (int64_t)1 << 22, kHeadHidden = (int64_t)1 << 20;
constexpr int64_t kPieceValues = (int64_t)1 << 28, kLeastPiece = 4096;   // of G

static int head_check(int32_t dtype, int64_t rows, int64_t vocab, int64_t hidden)
{
    if (dtype != ADAMBRIDGE_DT_F32 && dtype != ADAMBRIDGE_DT_BF16) return ADAMBRIDGE_EMVDTYPE;
    const int piece = dtype == ADAMBRIDGE_DT_BF16 ? 8 : 4;
    if (rows < 1 || rows > kHeadRows || vocab < 1 || vocab > kHeadVocab || hidden < piece || hidden > kHeadHidden) return ADAMBRIDGE_EBADN;
    return 0;
}

static int64_t up(int64_t n, int64_t to) { return (n + to - 1) / to * to; }

// Scratch, handed out in whole 256 bytes.
struct Scratch {
    uint8_t* base;
    int64_t used = 0;
    template <class T>
    T* take(int64_t n)
    {
        T* p = reinterpret_cast<T*>(base + used);
        used += up(n * (int64_t)sizeof(T), 256);
        return p;
    }
};

// A kernel's tile.  WIDE and LARGE have the same one: rows of whole pieces, and of any length.
enum Kind { WIDE, LARGE, HALF, F32_128, F32_64 };
static int tile_m(Kind k) { return k == F32_64 ? 64 : k == F32_128 ? 128 : 256; }
static int tile_n(Kind k) { return k == WIDE || k == LARGE ? 256 : k == F32_64 ? 64 : 128; }
static int places_of(Kind k) { return (k == WIDE || k == LARGE ? 1 : k == F32_64 ? 4 : 2) * kHeadCus; }
static int64_t tiles_of(Kind k, int64_t m, int64_t n) { return (m + tile_m(k) - 1) / tile_m(k) * ((n + tile_n(k) - 1) / tile_n(k)); }
static_assert(HalfTile::BM == 256 && HalfTile::BN == 128 && WideTile::BM == LargeTile::BM && WideTile::BN == LargeTile::BN, "tile_m, tile_n");

// The tile for m x n sums of so many terms.  FP32: as the expert products' rule, 64 where tiles of 128 are few.  BF16: 256 x 256;
// dW's 256 x 128, two workgroups a CU, where their columns end closer behind the last one (us, 256 / 128 columns: dW of 2703 rows
// and 50688 words of 896 values 286 / 240, of 16384 rows and 16128 words of 4096 1649 / 1732; the other kernels are 8-18% slower on
// half tiles).  Logits whose large tiles are half the CUs or fewer are on half tiles too (us of the forward call, 256 / 128 columns: 2048 rows
// of 3328 x 4096 102 / 90, of 2816 x 1024 39 / 36, 512 of 16000 x 2048 59 / 53, 256 of 32000 x 4096 103 / 96, of 32000 x 1024 34 / 36).
// Four wavefronts a workgroup where the sums are long, else eight, whose epilogues hide one another's waits (us, four
// / eight: 4096 rows of 32768 words of 1024 values 321 / 303, 2048 487 / 486, 4096 853 / 901, 8192 1599 / 1705).
enum Product { SUMS, WEIGHTS, ROWS };   // the logits, dW, dh
static Kind kind_of(int32_t dtype, int64_t m, int64_t n, int64_t terms, Product product)
{
    if (dtype != ADAMBRIDGE_DT_BF16) return tiles_of(F32_128, m, n) < 512 ? F32_64 : F32_128;
    if (product == WEIGHTS && tiles_of(HALF, m, n) * 21 < tiles_of(LARGE, m, n) * 40) return HALF;   // 1.05 times the values
    if (product == SUMS && tiles_of(LARGE, m, n) <= kHeadCus / 2) return HALF;
    if (product != SUMS) terms /= splits_of(tiles_of(LARGE, m, n), places_of(LARGE), terms);
    return terms >= 2048 ? WIDE : LARGE;
}

// The forward call's plan and scratch.
struct HeadForward {
    bool few;
    Kind kind;
    int parts, splits;
    int32_t *index, *count;
    HeadRow* facts;
    float *picked, *logits;
    Sums* part;
    void* h;
    int64_t bytes;
    HeadForward(void* work, int32_t dtype, int64_t rows, int64_t vocab, int64_t hidden)
    {
        // Rows that stream the weights, or go on tiles: a wavefront streams its words' whole rows, which takes as long as they are
        // unless there are words enough for all CUs.  (us, streamed / tiles, 16 rows, BF16 and FP32: 8000 words of 512 values
        // 11 / 18 and 17 / 21, of 2048 27 / 20 and 49 / 35, 16000 of 2048 27 / 27 and 49 / 55, 38000 of 2048 49 / 54 and 100 / 132,
        // 8000 of 8192 89 / 39 and 173 / 96.  32 rows of 151936 x 896 BF16 72 streamed, 69 on tiles.)
        few = rows <= 16 && (hidden <= 1024 || vocab >= 16000);
        kind = kind_of(dtype, rows, vocab, hidden, SUMS);
        parts = (int)(few ? (vocab + 64 * kFewGroups - 1) / (64 * kFewGroups) : (vocab + tile_n(kind) - 1) / tile_n(kind));
        // parts of the terms only where they are three or more (us, whole / two parts: 200 rows of 32000 x 4096 92 / 97; three or more:
        // 121 rows of 10197 x 4608 78 / 49)
        splits = splits_of(tiles_of(kind, rows, vocab), places_of(kind), hidden);
        if (few || tiles_of(kind, rows, vocab) * 3 > places_of(kind)) splits = 1;
        Scratch s{static_cast<uint8_t*>(work)};
        picked = s.take<float>(rows);
        part = s.take<Sums>(splits > 1 ? 0 : parts * rows);
        logits = s.take<float>(splits > 1 ? splits * rows * up(vocab, 4) : 0);
        index = few ? nullptr : s.take<int32_t>(rows);
        facts = few ? nullptr : s.take<HeadRow>(rows);
        count = few ? nullptr : s.take<int32_t>(1);
        h = few ? nullptr : s.take<uint8_t>(rows * hidden * (dtype == ADAMBRIDGE_DT_BF16 ? 2 : 4));
        bytes = s.used;
    }
};

// The backward call's.
struct HeadBackward {
    Kind grad, dw, dh_kind;
    int32_t pitch;   // words of a piece
    int grad_splits, dw_splits;
    int32_t *index, *place, *count;
    HeadRow* facts;
    void *h, *g;
    float *dh, *parts;
    int64_t bytes;
    HeadBackward(void* work, int32_t dtype, int64_t rows, int64_t vocab, int64_t hidden)
    {
        const int64_t size = dtype == ADAMBRIDGE_DT_BF16 ? 2 : 4;
        const int64_t most = std::max(kPieceValues / rows, kLeastPiece), pieces = (vocab + most - 1) / most;
        pitch = (int32_t)up((vocab + pieces - 1) / pieces, 256);
        const int64_t width = std::min<int64_t>(pitch, vocab);
        grad = kind_of(dtype, rows, width, hidden, SUMS);
        dw = kind_of(dtype, width, hidden, rows, WEIGHTS);
        dh_kind = kind_of(dtype, rows, hidden, pitch, ROWS);
        Scratch s{static_cast<uint8_t*>(work)};
        index = s.take<int32_t>(rows);
        facts = s.take<HeadRow>(rows);
        place = s.take<int32_t>(rows);
        count = s.take<int32_t>(1);
        h = s.take<uint8_t>(rows * hidden * size);
        g = s.take<uint8_t>(rows * pitch * size);
        // parts x rows x hidden: as many as fill the CUs with tiles, or one
        dh = s.take<float>(std::max(rows * hidden, (int64_t)places_of(dh_kind) * tile_m(dh_kind) * tile_n(dh_kind)));
        grad_splits = splits_of(tiles_of(grad, rows, width), places_of(grad), hidden);
        // two parts no more than forward (us, whole / two: 2048 rows of 3500 x 2048 BF16 149 / 158, 1000 of 7000 x 1024 94 / 108, of 7000 x
        // 4096 211 / 212; 500 of 3500 x 1024 FP32 142 / 146)
        if (tiles_of(grad, rows, width) * 3 > places_of(grad)) grad_splits = 1;
        dw_splits = splits_of(tiles_of(dw, width, hidden), places_of(dw), rows);
        if (tiles_of(dw, width, hidden) * 3 > places_of(dw)) dw_splits = 1;   // (1237 rows, 5003 x 333 FP32: 55 us whole, 55 + 6 in two parts)
        parts = s.take<float>(std::max(grad_splits > 1 ? grad_splits * rows * pitch : 0, dw_splits > 1 ? dw_splits * width * hidden : 0));
        bytes = s.used;
    }
};

static dim3 tile_grid(int64_t tiles) { return block_grid(up(tiles, kXcd)); }

#define ABH_HEAD_BF16(KERNEL, TILE, EVEN, GRID)                                                                    \
    do {                                                                                                           \
        if (EVEN) hipLaunchKernelGGL((KERNEL<HeadBf16<TILE, true>>), GRID, dim3(TILE::T), 0, t_stream, A);         \
        else hipLaunchKernelGGL((KERNEL<HeadBf16<TILE, false>>), GRID, dim3(TILE::T), 0, t_stream, A);             \
    } while (0)
#define ABH_HEAD_WHOLE(KERNEL, KIND, EVEN, GRID)   /* (dh's tiles are never halves) */                              \
    do {                                                                                                           \
        if ((KIND) == WIDE && (EVEN)) hipLaunchKernelGGL((KERNEL<HeadBf16<WideTile, true>>), GRID, dim3(WideTile::T), 0, t_stream, A); \
        else if ((KIND) == WIDE || (KIND) == LARGE) ABH_HEAD_BF16(KERNEL, LargeTile, EVEN, GRID);                  \
        else if ((KIND) == F32_128) hipLaunchKernelGGL((KERNEL<HeadF32<128>>), GRID, dim3(256), 0, t_stream, A);   \
        else hipLaunchKernelGGL((KERNEL<HeadF32<64>>), GRID, dim3(256), 0, t_stream, A);                           \
    } while (0)
#define ABH_HEAD_LAUNCH(KERNEL, KIND, EVEN, GRID)                                                                  \
    do {                                                                                                           \
        if ((KIND) == HALF) ABH_HEAD_BF16(KERNEL, HalfTile, EVEN, GRID);                                           \
        else ABH_HEAD_WHOLE(KERNEL, KIND, EVEN, GRID);                                                             \
    } while (0)

// Split logits' tiles are the smaller ones: the larger are taken where there are enough.
static void launch_logits(const HeadArgs& A, bool bf, bool even, dim3 grid)
{
    if (bf) ABH_HEAD_BF16(k_head_logits, HalfTile, even, grid);
    else hipLaunchKernelGGL((k_head_logits<HeadF32<64>>), grid, dim3(256), 0, t_stream, A);
}

// The scored rows: their numbers, how many, and copies of them.  One launch for a few thousand rows, whose counts grow with the
// square of them, else two (us, one / two: the forward call of 100 rows of 151936 x 896 71.1 / 73.5; the kernels alone at 4096 rows
// 10.8 / 11.3, at 16384 the first of two 17).
constexpr int64_t kFindRows = 2048;

static void launch_rows(bool bf, const void* h, const int64_t* targets, int64_t ignore, int64_t rows, int32_t* index, int32_t* place, int32_t* count,
                        float* losses, const HeadFacts& facts, int64_t hidden, void* out)
{
    const dim3 grid = block_grid(rows), block(256);
    const int32_t n = (int32_t)rows, size = (int32_t)hidden;
    if (rows <= kFindRows) {
        if (bf) hipLaunchKernelGGL((k_head_gather<DT_BF16, true>), grid, block, 0, t_stream, h, targets, ignore, n, index, place, count, losses, facts, size, out);
        else hipLaunchKernelGGL((k_head_gather<DT_F32, true>), grid, block, 0, t_stream, h, targets, ignore, n, index, place, count, losses, facts, size, out);
        return;
    }
    hipLaunchKernelGGL(k_head_rows, dim3(1), dim3(1024), 0, t_stream, targets, ignore, n, index, place, count, losses);
    if (bf) hipLaunchKernelGGL((k_head_gather<DT_BF16, false>), grid, block, 0, t_stream, h, targets, ignore, n, index, place, count, losses, facts, size, out);
    else hipLaunchKernelGGL((k_head_gather<DT_F32, false>), grid, block, 0, t_stream, h, targets, ignore, n, index, place, count, losses, facts, size, out);
}

}  // namespace abh

using namespace abh;

extern "C" {

ADAMBRIDGE_API int64_t adambridge_token_losses_work(int32_t dtype, int64_t rows, int64_t vocab, int64_t hidden)
{
    const int rc = head_check(dtype, rows, vocab, hidden);
    return rc ? rc : HeadForward(nullptr, dtype, rows, vocab, hidden).bytes;
}

ADAMBRIDGE_API int adambridge_token_losses(const void* hidden, const void* weight, int32_t dtype, const int64_t* targets, int64_t rows,
                                           int64_t vocab, int64_t size, int64_t ignore_index, float* losses, float* stats, void* work)
{
    const int rc = head_check(dtype, rows, vocab, size);
    if (rc) return rc;
    if (!hidden || !weight || !targets || !losses || !work) return ADAMBRIDGE_ENULL;
    if ((uintptr_t)work % 16) return ADAMBRIDGE_EALIGN;
    const bool bf = dtype == ADAMBRIDGE_DT_BF16;
    const HeadForward p(work, dtype, rows, vocab, size);
    HeadArgs A{};
    A.w = weight;
    A.targets = targets;
    A.rows = (int32_t)rows;
    A.hidden = (int32_t)size;
    A.vocab = vocab;
    A.part = p.part;
    A.picked = p.picked;
    if (p.few) {
        A.h = hidden;
        const int64_t bytes = size * (bf ? 2 : 4);
        const bool even = bytes % 16 == 0 && ((uintptr_t)hidden | (uintptr_t)weight) % 16 == 0;
        const dim3 grid = block_grid(p.parts), block(256);
        if (bf && even) hipLaunchKernelGGL((k_head_few<DT_BF16, true>), grid, block, 0, t_stream, A);
        else if (bf) hipLaunchKernelGGL((k_head_few<DT_BF16, false>), grid, block, 0, t_stream, A);
        else if (even) hipLaunchKernelGGL((k_head_few<DT_F32, true>), grid, block, 0, t_stream, A);
        else hipLaunchKernelGGL((k_head_few<DT_F32, false>), grid, block, 0, t_stream, A);
        hipLaunchKernelGGL((k_head_finish<4>), dim3((unsigned)((rows + 3) / 4)), dim3(kFinishLanes), 0, t_stream, p.part, p.parts, A.rows, nullptr,
                           nullptr, targets, vocab, ignore_index, p.picked, losses, stats);
    } else {
        launch_rows(bf, hidden, targets, ignore_index, rows, p.index, nullptr, p.count, losses, HeadFacts{p.facts, vocab, nullptr, nullptr}, size, p.h);
        A.h = p.h;
        A.facts = p.facts;
        A.count = p.count;
        A.width = (int32_t)vocab;
        A.tiles_j = p.parts;
        const bool even = size % 8 == 0 && (uintptr_t)weight % 16 == 0;
        if (p.splits > 1) {
            A.pitch = (int32_t)up(vocab, 4);
            A.splits = p.splits;
            A.parts = p.logits;
            launch_logits(A, bf, even, tile_grid(tiles_of(p.kind, rows, vocab) * p.splits));
            // a wavefront a row, or a workgroup (8270 rows of 59 words: 1024 lanes 80 us)
            if (vocab <= 1024) hipLaunchKernelGGL((k_head_join<64>), block_grid((rows + 3) / 4), dim3(256), 0, t_stream, A, p.index, targets, ignore_index, losses, stats);
            else hipLaunchKernelGGL((k_head_join<1024>), block_grid(rows), dim3(1024), 0, t_stream, A, p.index, targets, ignore_index, losses, stats);
        } else {
            ABH_HEAD_LAUNCH(k_head_sums, p.kind, even, tile_grid(tiles_of(p.kind, rows, vocab)));
            hipLaunchKernelGGL((k_head_finish<16>), block_grid((rows + 15) / 16), dim3(kFinishLanes), 0, t_stream, p.part, p.parts, A.rows, p.index,
                               p.count, targets, vocab, ignore_index, p.picked, losses, stats);
        }
    }
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? 0 : hip_fail(e, "hipLaunchKernelGGL (token losses)");
}

ADAMBRIDGE_API int64_t adambridge_token_losses_backward_work(int32_t dtype, int64_t rows, int64_t vocab, int64_t hidden)
{
    const int rc = head_check(dtype, rows, vocab, hidden);
    return rc ? rc : HeadBackward(nullptr, dtype, rows, vocab, hidden).bytes;
}

ADAMBRIDGE_API int adambridge_token_losses_backward(const float* gout, const void* hidden, const void* weight, int32_t dtype,
                                                    const int64_t* targets, int64_t rows, int64_t vocab, int64_t size, int64_t ignore_index,
                                                    const float* stats, void* dhidden, void* dweight, void* work)
{
    const int rc = head_check(dtype, rows, vocab, size);
    if (rc) return rc;
    if (!dhidden && !dweight) return 0;
    if (!gout || !hidden || !weight || !targets || !stats || !work) return ADAMBRIDGE_ENULL;
    if ((uintptr_t)work % 16) return ADAMBRIDGE_EALIGN;
    const bool bf = dtype == ADAMBRIDGE_DT_BF16;
    const HeadBackward p(work, dtype, rows, vocab, size);
    launch_rows(bf, hidden, targets, ignore_index, rows, p.index, p.place, p.count, nullptr, HeadFacts{p.facts, vocab, stats, gout}, size, p.h);
    HeadArgs A{};
    A.h = p.h;
    A.w = weight;
    A.facts = p.facts;
    A.count = p.count;
    A.rows = (int32_t)rows;
    A.hidden = (int32_t)size;
    A.vocab = vocab;
    A.pitch = p.pitch;
    A.g = p.g;
    A.dh = p.dh;
    A.dw = dweight;
    A.fresh = 1;
    A.parts = p.parts;
    const bool even = size % 8 == 0 && ((uintptr_t)weight | (uintptr_t)dweight) % 16 == 0;
    for (int64_t v0 = 0; v0 < vocab; v0 += p.pitch) {
        A.v0 = v0;
        A.width = (int32_t)std::min<int64_t>(p.pitch, vocab - v0);
        A.tiles_j = (A.width + tile_n(p.grad) - 1) / tile_n(p.grad);
        A.splits = p.grad_splits;
        if (p.grad_splits > 1) {
            launch_logits(A, bf, even, tile_grid(tiles_of(p.grad, rows, A.width) * p.grad_splits));
            const int32_t columns = (A.width + 1023) / 1024;
            if (bf) hipLaunchKernelGGL((k_head_join_grad<DT_BF16>), block_grid(rows * columns), dim3(256), 0, t_stream, A, columns);
            else hipLaunchKernelGGL((k_head_join_grad<DT_F32>), block_grid(rows * columns), dim3(256), 0, t_stream, A, columns);
        } else {
            ABH_HEAD_LAUNCH(k_head_grad, p.grad, even, tile_grid(tiles_of(p.grad, rows, A.width)));
        }
        if (dweight) {
            A.tiles_j = (int32_t)((size + tile_n(p.dw) - 1) / tile_n(p.dw));
            A.splits = p.dw_splits;
            ABH_HEAD_LAUNCH(k_head_dw, p.dw, even, tile_grid(tiles_of(p.dw, A.width, size) * p.dw_splits));
            if (p.dw_splits > 1 && bf) hipLaunchKernelGGL((k_head_join_dw<DT_BF16>), block_grid(A.width), dim3(256), 0, t_stream, A);
            else if (p.dw_splits > 1) hipLaunchKernelGGL((k_head_join_dw<DT_F32>), block_grid(A.width), dim3(256), 0, t_stream, A);
        }
        if (dhidden) {
            A.tiles_j = (int32_t)((size + tile_n(p.dh_kind) - 1) / tile_n(p.dh_kind));
            A.places = places_of(p.dh_kind);
            ABH_HEAD_WHOLE(k_head_dh, p.dh_kind, even, tile_grid(std::max<int64_t>(tiles_of(p.dh_kind, rows, size), A.places)));
        }
        A.fresh = 0;
    }
    if (dhidden) {
        if (bf)
            hipLaunchKernelGGL((k_head_scatter<DT_BF16>), block_grid(rows), dim3(256), 0, t_stream, p.dh, p.place, p.count, A.rows, A.hidden,
                               tile_m(p.dh_kind), tile_n(p.dh_kind), A.places, p.pitch, dhidden);
        else
            hipLaunchKernelGGL((k_head_scatter<DT_F32>), block_grid(rows), dim3(256), 0, t_stream, p.dh, p.place, p.count, A.rows, A.hidden,
                               tile_m(p.dh_kind), tile_n(p.dh_kind), A.places, p.pitch, dhidden);
    }
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? 0 : hip_fail(e, "hipLaunchKernelGGL (token losses backward)");
}

}  // extern "C"
