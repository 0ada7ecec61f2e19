// abh_embed.hip -- rows of an embedding for token ids, and the embedding's gradient.
//
//   y[i] = scale W[ids[i]]                       (an id outside the vocabulary: a row of NaN)
//   dW[v] = scale sum of g[i] over ids[i] = v    (zeros for a word without tokens, and for the padding)
//
// Bytes bound both: T rows read and written; T rows read and V written, most of them zeros.  (65536 tokens of 32000 x 4096 BF16: rows
// 124 us; gradient 47 for the order, 43 for long words' parts, 98 for the words' rows, 5.7 TB/s of the two.  4096 of 151936 x 896:
// 4.9; 5.3, 7.0, 51, 5.5 TB/s.)
//
// The gradient's sums run over the tokens sorted by id, then by position, so that they have an order of their own and
// dW is written once, by the words' rows, without atomics on values or a pass that clears it.  Text has a few words
// very often: the sorted tokens are cut into chunks, and a word that has all tokens of a chunk is summed chunk by chunk by as
// many workgroups, whose parts the word's wavefront adds in order; any other word's rows are its wavefront's.
//
// The sort: runs of 4096 tokens by counting, then up to 32 runs at a time become one, each token's place being its own in its
// run plus how many of every other run are below it.  (Id, position) pairs differ, so the order is a total one.

#include <hip/hip_runtime.h>

#include <stdint.h>

#include <algorithm>

#include "../../include/adambridge_hip.h"
#include "abh_device.hpp"
#include "abh_host.hpp"
#include "abh_rows.hpp"
#include "abh_tiles.hpp"

namespace abh {

constexpr int kRun = 4096, kSortThreads = 1024;
// Words of a wavefront, fewer than its lanes.  (us of a backward pass with 4 / 8 / 16: 65536 tokens of 32000 x 4096 BF16 215 / 224 / 225, of
// 151936 x 896 110 / 113 / 118, of 200000 x 2048 228 / 244 / 244; 4096 of 151936 x 896 62 / 63 / 65; 2021 of 5003 x 897 FP32 17 / 17 / 17.  Without a sort, 4 / 8:
// 8 tokens of 151936 x 896 50 / 53, 256 of 32000 x 4096 48 / 50, of 1000 x 8192 7.5 / 7.4)
constexpr int kMostWords = 4;
constexpr int kFewIds = 256;      // tokens whose ids every wavefront reads for itself
constexpr int kLeastChunk = 32;   // tokens.  (the words' rows and the parts: 146 us with 32, 149 with 64)

__device__ __forceinline__ int64_t id_at(const void* ids, int32_t id_bytes, int64_t i)
{
    return id_bytes == 8 ? static_cast<const int64_t*>(ids)[i] : (int64_t)static_cast<const int32_t*>(ids)[i];
}

// ------------------------------------------------------------------------------- the rows

struct EmbedArgs {
    const void* ids;
    const void* weight;
    void* y;
    int64_t tokens, vocab;
    int32_t id_bytes, hidden, segments;   // segments: a row's pieces of G x U vectors
    float scale;
};

// G lanes a piece of a row, U vectors a lane, all loaded before the first is stored.
template <int DT, int G, int U>
__global__ __launch_bounds__(256) void k_embed(EmbedArgs A)
{
    constexpr int L = kLane<DT>;
    const int64_t item = (block_index() * 256 + threadIdx.x) / G;
    if (item >= A.tokens * A.segments) return;
    const int64_t token = A.segments == 1 ? item : item / A.segments;
    const int32_t first = (int32_t)(item - token * A.segments) * (G * U * L) + (int32_t)(threadIdx.x % G) * L;
    const int64_t id = id_at(A.ids, A.id_bytes, token);
    const bool real = id >= 0 && id < A.vocab;
    const void* row = at<DT>(A.weight, (real ? id : 0) * A.hidden);
    void* out = at<DT>(A.y, token * A.hidden);
    raw16 w[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int32_t i = first + u * G * L;
        if (i < A.hidden) w[u] = load_vec_raw<DT>(row, i, A.hidden);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int32_t i = first + u * G * L;
        if (i >= A.hidden) continue;
        float x[L];
        to_floats<DT>(w[u], x);
#pragma unroll
        for (int k = 0; k < L; ++k) x[k] = real ? x[k] * A.scale : __builtin_nanf("");
        stream_vec<DT>(out, i, A.hidden, x);
    }
}

// ------------------------------------------------------------------------------- the sort

// Runs of kRun (id, position) in one word each; an id outside the vocabulary is the vocabulary's size, behind all words.  A token's place in
// its run is counted: the tokens before it whose id is no larger, and those behind it whose id is smaller.  I tokens a workgroup,
// each compared with the run's 4096 ids in the LDS by 1024 / I lanes.  (4096 tokens 4.5 us, where a sorting network in one
// workgroup's LDS took 20; a run twice as long costs twice the comparisons and saves a step of the merge.)
template <int I>
__global__ __launch_bounds__(kSortThreads) void k_embed_sort(const void* ids, int32_t id_bytes, int64_t tokens, int64_t vocab, uint64_t* out)
{
    constexpr int S = kSortThreads / I, N = kRun / S, PAD = 4;   // S slices of N ids, 16 bytes apart: other banks
    __shared__ __attribute__((aligned(16))) uint32_t key[S * (N + PAD)];
    __shared__ uint32_t rank[I];
    const int64_t i0 = block_index() * I, t0 = i0 / kRun * kRun;
    if (i0 >= tokens) return;
    const int n = (int)(tokens - t0 < kRun ? tokens - t0 : kRun);
    for (int i = threadIdx.x; i < kRun; i += kSortThreads) {
        uint32_t x = ~0u;   // none
        if (i < n) {
            const int64_t id = id_at(ids, id_bytes, t0 + i);
            x = (uint32_t)(id >= 0 && id < vocab ? id : vocab);
        }
        key[i / N * (N + PAD) + i % N] = x;
    }
    if (threadIdx.x < I) rank[threadIdx.x] = 0;
    __syncthreads();
    const int item = (int)(i0 - t0) + (int)threadIdx.x % I, slice = threadIdx.x / I;
    const uint32_t mine = key[item / N * (N + PAD) + item % N];
    const uint32_t* const ids_of = key + slice * (N + PAD);
    uint32_t below = 0;
    if (slice * N < n) {
        if (item / N != slice) {
            const uint32_t limit = mine + (slice * N < item);
#pragma unroll 4
            for (int j = 0; j < N; j += 4) {
                const raw16 k = *reinterpret_cast<const raw16*>(ids_of + j);
                below += (k.x < limit) + (k.y < limit) + (k.z < limit) + (k.w < limit);
            }
        } else {
            for (int j = 0; j < N; ++j) below += ids_of[j] < mine + (slice * N + j < item);
        }
        atomicAdd(&rank[threadIdx.x % I], below);
    }
    __syncthreads();
    if ((int)threadIdx.x < I && item < n) out[t0 + rank[threadIdx.x]] = (uint64_t)mine << 32 | (uint32_t)(t0 + item);
}

// How many of in[0 .. n) are below x.
__device__ __forceinline__ int64_t below(const uint64_t* in, int64_t n, uint64_t x)
{
    int64_t lo = 0, hi = n;
    while (lo < hi) {
        const int64_t mid = (lo + hi) >> 1;
        if (in[mid] < x) lo = mid + 1;
        else hi = mid;
    }
    return lo;
}

// Runs of `run` sorted items, R of them at a time: one item a lane, all runs' searches step by step together, every read taken
// whether it counts or not, so that a step's reads overlap (65536 tokens, 16 runs: 20 us).
template <int R>
__global__ __launch_bounds__(256) void k_embed_merge(const uint64_t* in, int64_t tokens, uint32_t run, uint64_t* out)
{
    const int64_t i = block_index() * 256 + threadIdx.x;
    if (i >= tokens) return;
    const uint64_t x = in[i];
    const uint32_t n = (uint32_t)tokens, mine = (uint32_t)i / run, first = mine / R * R;   // places below 2^31 + run
    uint32_t place = first * run + ((uint32_t)i - mine * run), lo[R];
#pragma unroll
    for (int r = 0; r < R; ++r) lo[r] = 0;
    for (uint32_t step = run; step > 0; step >>= 1) {   // runs are powers of two
        uint64_t y[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const uint32_t at = (first + r) * run + lo[r] + step - 1;   // below it: this and all before it are
            y[r] = in[at < n ? at : n - 1];
        }
#pragma unroll
        for (int r = 0; r < R; ++r) lo[r] += lo[r] + step <= run && (first + r) * run + lo[r] + step <= n && y[r] < x ? step : 0u;
    }
#pragma unroll
    for (int r = 0; r < R; ++r) place += first + r == mine ? 0u : lo[r];
    out[place] = x;
}

// ------------------------------------------------------------------------------- the gradient

struct EmbedBackArgs {
    const void* ids;
    const uint64_t* sorted;
    const void* gout;
    void* dweight;
    float* part;          // chunks x 2 x hidden
    int32_t* starts;      // vocab + 1
    int64_t tokens, vocab, padding, part_blocks;
    int32_t id_bytes, hidden, chunk, part_columns, words, pieces;   // words, pieces: of a wavefront of k_embed_rows, of a row
    float scale;
};

__device__ __forceinline__ uint32_t word_of(uint64_t item) { return (uint32_t)(item >> 32); }

// A lane's vector of a row.  One over the end of the row is the row's last whole one instead (then two lanes have the same
// values, and store them); SHORT: rows of less than a vector.
template <int DT, bool SHORT>
struct Columns {
    static constexpr int L = kLane<DT>;
    int32_t first;
    bool real;
    __device__ __forceinline__ Columns(int32_t column, int32_t hidden) : first(SHORT || column + L <= hidden ? column : hidden - L), real(column < hidden) {}
    __device__ __forceinline__ raw16 load(const void* row, int32_t hidden) const
    {
        if constexpr (SHORT) return real ? load_vec_raw<DT>(row, first, hidden) : raw16{0u, 0u, 0u, 0u};
        else return load_raw<DT>(row, first);
    }
    __device__ __forceinline__ void add(const raw16 w, float (&acc)[L]) const
    {
        float x[L];
        to_floats<DT>(w, x);
#pragma unroll
        for (int k = 0; k < L; ++k) acc[k] += x[k];
    }
    __device__ __forceinline__ void load_part(const float* part, int32_t hidden, float (&x)[L]) const
    {
        if constexpr (SHORT) {
            load_like<DT_F32, L>(part, real ? first : 0, real ? hidden : 0, 0.0f, x);
        } else {
#pragma unroll
            for (int k = 0; k < L; k += 4) to_floats<DT_F32>(load_raw<DT_F32>(part, first + k), x + k);
        }
    }
    __device__ __forceinline__ void store_part(float* part, int32_t hidden, const float (&x)[L]) const
    {
        if (!real) return;
        if constexpr (SHORT) {
            store_like<DT_F32, L>(part, first, hidden, x);
        } else {
#pragma unroll
            for (int k = 0; k < L; k += 4) store_raw<DT_F32>(part, first + k, to_raw<DT_F32>(x + k));
        }
    }
    __device__ __forceinline__ void stream(void* row, int32_t hidden, const float (&x)[L]) const
    {
        if (!real) return;
        if constexpr (SHORT) stream_vec<DT>(row, first, hidden, x);
        else stream_raw<DT>(row, first, to_raw<DT>(x));
    }
};

// A word is long that all tokens of some chunk belong to.
__device__ __forceinline__ bool is_long(const EmbedBackArgs& A, int from, int to)
{
    return (from + A.chunk - 1) / A.chunk * A.chunk + A.chunk <= to;
}

// Two things at once.  The first workgroups: a chunk's parts of long words, of the one its first token belongs to and of the one its
// last does.  The others: where each word's tokens begin, 256 words a workgroup.
template <int DT, bool SHORT>
__global__ __launch_bounds__(256) void k_embed_parts(EmbedBackArgs A)
{
    constexpr int L = kLane<DT>, AHEAD = 16;
    const int64_t block = block_index();
    if (block >= A.part_blocks) {
        const int64_t v = (block - A.part_blocks) * 256 + threadIdx.x;
        if (v <= A.vocab) A.starts[v] = (int32_t)below(A.sorted, A.tokens, (uint64_t)v << 32);
        return;
    }
    const int64_t c = block / A.part_columns, p0 = c * A.chunk;
    const int64_t p1 = p0 + A.chunk < A.tokens ? p0 + A.chunk : A.tokens, p2 = p1 + A.chunk;
    const uint32_t first = word_of(A.sorted[p0]), last = word_of(A.sorted[p1 - 1]);
    const uint32_t before = word_of(A.sorted[p0 >= A.chunk ? p0 - A.chunk : 0]), after = word_of(A.sorted[p2 <= A.tokens ? p2 - 1 : A.tokens - 1]);
    const Columns<DT, SHORT> columns((int32_t)((block - c * A.part_columns) * 256 + threadIdx.x) * L, A.hidden);
    const int lane = threadIdx.x & 63;
#pragma unroll 1
    for (int s = 0; s < 2; ++s) {
        const uint32_t word = s ? last : first;
        // the word has all of this chunk; of the one before, if it does not begin here; or of the next, if it begins here
        const bool whole = first == last && p1 - p0 == A.chunk;
        if (s ? first == last || p2 > A.tokens || after != word : !whole && (p0 < A.chunk || before != word)) continue;
        if (word >= A.vocab || word == A.padding) continue;
        int from = scalar((int)p0), to = scalar((int)p1);
        if (first != last) {
            const int edge = scalar((int)(p0 + below(A.sorted + p0, p1 - p0, (uint64_t)(s ? word : word + 1) << 32)));
            from = s ? edge : from;
            to = s ? to : edge;
        }
        float acc[L];
#pragma unroll
        for (int k = 0; k < L; ++k) acc[k] = 0.0f;
        for (int p = from; p < to; p += kWave) {
            const int n = to - p < kWave ? to - p : kWave;
            const uint32_t position = (uint32_t)A.sorted[p + (lane < n ? lane : n - 1)];   // a lane reads one for its wavefront
            for (int i = 0; i < n; i += AHEAD) {
                raw16 w[AHEAD];
#pragma unroll
                for (int a = 0; a < AHEAD; ++a)
                    w[a] = columns.load(at<DT>(A.gout, (int64_t)(uint32_t)__builtin_amdgcn_readlane((int)position, i + a < n ? i + a : n - 1) * A.hidden), A.hidden);
#pragma unroll
                for (int a = 0; a < AHEAD; ++a)
                    if (i + a < n) columns.add(w[a], acc);
            }
        }
        columns.store_part(A.part + (c * 2 + s) * A.hidden, A.hidden, acc);
    }
}

// dW: a wavefront has a piece of 64 vectors of A.words words' rows.  Their tokens lie together in the sorted order, and their rows are
// loaded one after the other whichever word they belong to; a word is stored when its last one has been added.
template <int DT, bool SHORT>
__global__ __launch_bounds__(256) void k_embed_rows(EmbedBackArgs A)
{
    constexpr int L = kLane<DT>, AHEAD = 8, N = 4;
    const int lane = threadIdx.x & 63;
    const int64_t item = block_index() * 4 + __builtin_amdgcn_readfirstlane((int)threadIdx.x / kWave);
    const int64_t group = item / A.pieces, v0 = group * A.words;
    if (v0 >= A.vocab) return;
    const int words = (int)(A.vocab - v0 < A.words ? A.vocab - v0 : A.words);
    const Columns<DT, SHORT> columns((int32_t)(item - group * A.pieces) * (64 * L) + lane * L, A.hidden);
    const int start = A.starts[v0 + (lane < words ? lane : words)], next = __shfl_down(start, 1);
    // words that are not sums of their rows: the padding, and long ones
    uint64_t apart = __builtin_amdgcn_ballot_w64(lane < words && (v0 + lane == A.padding || is_long(A, start, next)));
    const uint64_t some = __builtin_amdgcn_ballot_w64(lane < words && next > start && v0 + lane != A.padding);
    float acc[L];
    auto clear = [&]() {
#pragma unroll
        for (int k = 0; k < L; ++k) acc[k] = 0.0f;
    };
    auto flush = [&](int w) {
        const float by = some >> w & 1 ? A.scale : 0.0f;   // zeros without tokens, whatever the scale
#pragma unroll
        for (int k = 0; k < L; ++k) acc[k] *= by;
        columns.stream(at<DT>(A.dweight, (v0 + w) * A.hidden), A.hidden, acc);
        clear();
    };
    clear();
    for (int w = 0; w < words;) {
        const int stop = apart ? __builtin_ctzll(apart) : words;   // words w .. stop are sums of their rows
        const int to = __builtin_amdgcn_readlane(start, stop);
        int end = __builtin_amdgcn_readlane(start, w + 1);
        for (int p = __builtin_amdgcn_readlane(start, w); p < to; p += kWave) {
            const int n = to - p < kWave ? to - p : kWave;
            const uint32_t position = (uint32_t)A.sorted[p + (lane < n ? lane : n - 1)];
            for (int i = 0; i < n; i += AHEAD) {
                raw16 row[AHEAD];
#pragma unroll
                for (int a = 0; a < AHEAD; ++a)
                    row[a] = columns.load(at<DT>(A.gout, (int64_t)(uint32_t)__builtin_amdgcn_readlane((int)position, i + a < n ? i + a : n - 1) * A.hidden), A.hidden);
#pragma unroll
                for (int a = 0; a < AHEAD; ++a)
                    if (i + a < n) {
                        while (p + i + a >= end) {
                            flush(w);
                            end = __builtin_amdgcn_readlane(start, ++w + 1);
                        }
                        columns.add(row[a], acc);
                    }
            }
        }
        for (; w < stop; ++w) flush(w);
        if (!apart) continue;
        apart &= apart - 1;
        if (v0 + w != A.padding) {   // its chunks' parts, in order: the other word's in the first chunk, unless it begins with it
            const int from = __builtin_amdgcn_readlane(start, w), q0 = from / A.chunk, q1 = (__builtin_amdgcn_readlane(start, w + 1) - 1) / A.chunk;
            for (int q = q0; q <= q1; q += N) {
                float x[N][L];
#pragma unroll
                for (int a = 0; a < N; ++a) {
                    const int qa = q + a <= q1 ? q + a : q1;
                    columns.load_part(A.part + ((int64_t)qa * 2 + (qa == q0 && from % A.chunk != 0)) * A.hidden, A.hidden, x[a]);
                }
#pragma unroll
                for (int a = 0; a < N; ++a)
                    if (q + a <= q1)
#pragma unroll
                        for (int k = 0; k < L; ++k) acc[k] += x[a][k];
            }
        }
        flush(w++);
    }
}

// The same of a few tokens in one launch: a wavefront has all ids, four a lane, and a word's tokens are the bits of four ballots, in
// order.  (us of a forward and backward pass, 256 tokens so / 257 sorted: 5003 words of 897 BF16 values 26 / 31, 32000 of 4096 52 / 59;
// one word's 256 rows of 897, which are then one wavefront's, 32 / 31, of 4096 59 / 60.)
template <int DT, bool SHORT>
__global__ __launch_bounds__(256) void k_embed_few(EmbedBackArgs A)
{
    constexpr int L = kLane<DT>, AHEAD = 8, B = kFewIds / kWave;
    const int lane = threadIdx.x & 63;
    const int64_t item = block_index() * 4 + __builtin_amdgcn_readfirstlane((int)threadIdx.x / kWave);
    const int64_t group = item / A.pieces, v0 = group * A.words;
    if (v0 >= A.vocab) return;
    const int words = (int)(A.vocab - v0 < A.words ? A.vocab - v0 : A.words), tokens = (int)A.tokens;
    const Columns<DT, SHORT> columns((int32_t)(item - group * A.pieces) * (64 * L) + lane * L, A.hidden);
    int64_t id[B];
#pragma unroll
    for (int b = 0; b < B; ++b) {
        const int i = b * kWave + lane;
        id[b] = id_at(A.ids, A.id_bytes, i < tokens ? i : tokens - 1);
        if (i >= tokens) id[b] = -1;
    }
    for (int w = 0; w < words; ++w) {
        float acc[L];
#pragma unroll
        for (int k = 0; k < L; ++k) acc[k] = 0.0f;
        float by = 0.0f;   // zeros without tokens, whatever the scale
        if (v0 + w != A.padding) {
#pragma unroll
            for (int b = 0; b < B; ++b) {
                uint64_t mine = __builtin_amdgcn_ballot_w64(id[b] == v0 + w);
                by = mine ? A.scale : by;
                while (mine) {
                    raw16 row[AHEAD];
                    int n = 0, from = 0;
#pragma unroll
                    for (int a = 0; a < AHEAD; ++a) {   // past the last one: it again, not added
                        from = mine ? b * kWave + __builtin_ctzll(mine) : from;
                        n += mine != 0;
                        mine &= mine - 1;
                        row[a] = columns.load(at<DT>(A.gout, (int64_t)from * A.hidden), A.hidden);
                    }
#pragma unroll
                    for (int a = 0; a < AHEAD; ++a)
                        if (a < n) columns.add(row[a], acc);
                }
            }
        }
#pragma unroll
        for (int k = 0; k < L; ++k) acc[k] *= by;
        columns.stream(at<DT>(A.dweight, (v0 + w) * A.hidden), A.hidden, acc);
    }
}

// ------------------------------------------------------------------------------- launches

constexpr int64_t kEmbedTokens = (int64_t)1 << 30, kEmbedVocab = (int64_t)1 << 30, kEmbedHidden = (int64_t)1 << 22;

static int embed_check(int32_t id_bytes, int64_t tokens, int32_t dtype, int64_t vocab, int64_t hidden)
{
    if (tokens < 1 || tokens > kEmbedTokens || vocab < 1 || vocab > kEmbedVocab || hidden < 1 || hidden > kEmbedHidden) return ADAMBRIDGE_EBADN;
    if ((id_bytes != 4 && id_bytes != 8) || (dtype != ADAMBRIDGE_DT_F32 && dtype != ADAMBRIDGE_DT_BF16)) return ADAMBRIDGE_EMVDTYPE;
    return 0;
}

// Tokens of a chunk: so many that there are at most 2048 chunks, whose parts are at most 16 KB times the row's values.
static int64_t chunk_of(int64_t tokens)
{
    return std::max<int64_t>(kLeastChunk, ((tokens + 2047) / 2048 + 31) / 32 * 32);
}

static int64_t part_bytes(int64_t tokens, int64_t hidden)
{
    const int64_t chunk = chunk_of(tokens);
    return tokens >= chunk ? (tokens + chunk - 1) / chunk * 2 * hidden * 4 : 0;   // else no word has a whole chunk
}

template <int DT>
static void launch_embed(EmbedArgs& A)
{
    const int vectors = (A.hidden + kLane<DT> - 1) / kLane<DT>;
    const int lanes = vectors <= 8 ? 8 : vectors <= 16 ? 16 : vectors <= 32 ? 32 : 64;
    const int u = vectors <= 64 ? 1 : vectors <= 128 ? 2 : 4;
    A.segments = (vectors + lanes * u - 1) / (lanes * u);
    const dim3 grid = block_grid((A.tokens * A.segments * lanes + 255) / 256), block(256);
    if (lanes == 8) hipLaunchKernelGGL((k_embed<DT, 8, 1>), grid, block, 0, t_stream, A);
    else if (lanes == 16) hipLaunchKernelGGL((k_embed<DT, 16, 1>), grid, block, 0, t_stream, A);
    else if (lanes == 32) hipLaunchKernelGGL((k_embed<DT, 32, 1>), grid, block, 0, t_stream, A);
    else if (u == 1) hipLaunchKernelGGL((k_embed<DT, 64, 1>), grid, block, 0, t_stream, A);
    else if (u == 2) hipLaunchKernelGGL((k_embed<DT, 64, 2>), grid, block, 0, t_stream, A);
    else hipLaunchKernelGGL((k_embed<DT, 64, 4>), grid, block, 0, t_stream, A);
}

template <int DT>
static void launch_embed_back(EmbedBackArgs& A)
{
    const int vectors = (A.hidden + kLane<DT> - 1) / kLane<DT>;
    const bool few = A.tokens <= kFewIds, tiny = A.hidden < kLane<DT>;
    if (!few) {
        A.part_columns = (vectors + 255) / 256;
        A.part_blocks = A.tokens >= A.chunk ? (A.tokens + A.chunk - 1) / A.chunk * A.part_columns : 0;
        const dim3 parts = block_grid(A.part_blocks + (A.vocab + 256) / 256);
        if (tiny) hipLaunchKernelGGL((k_embed_parts<DT, true>), parts, dim3(256), 0, t_stream, A);
        else hipLaunchKernelGGL((k_embed_parts<DT, false>), parts, dim3(256), 0, t_stream, A);
    }
    A.pieces = (vectors + 63) / 64;
    // fewer words a wavefront where there would be too few wavefronts (5003 words of 897 FP32 values: 2 words 7 us, 16 19)
    A.words = kMostWords;
    while (A.words > 2 && (A.vocab + A.words - 1) / A.words * A.pieces < 4096) A.words /= 2;
    const dim3 grid = block_grid(((A.vocab + A.words - 1) / A.words * A.pieces + 3) / 4);
    if (few && tiny) hipLaunchKernelGGL((k_embed_few<DT, true>), grid, dim3(256), 0, t_stream, A);
    else if (few) hipLaunchKernelGGL((k_embed_few<DT, false>), grid, dim3(256), 0, t_stream, A);
    else if (tiny) hipLaunchKernelGGL((k_embed_rows<DT, true>), grid, dim3(256), 0, t_stream, A);
    else hipLaunchKernelGGL((k_embed_rows<DT, false>), grid, dim3(256), 0, t_stream, A);
}

}  // namespace abh

using namespace abh;

extern "C" {

ADAMBRIDGE_API int adambridge_embed(const void* ids, int32_t id_bytes, int64_t tokens, const void* weight, int32_t dtype,
                                    int64_t vocab, int64_t hidden, float scale, void* y)
{
    const int rc = embed_check(id_bytes, tokens, dtype, vocab, hidden);
    if (rc) return rc;
    if (!ids || !weight || !y) return ADAMBRIDGE_ENULL;
    EmbedArgs A{ids, weight, y, tokens, vocab, id_bytes, (int32_t)hidden, 0, scale};
    if (dtype == ADAMBRIDGE_DT_BF16) launch_embed<DT_BF16>(A);
    else launch_embed<DT_F32>(A);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? 0 : hip_fail(e, "hipLaunchKernelGGL (embed)");
}

ADAMBRIDGE_API int64_t adambridge_embed_work(int64_t tokens, int64_t vocab, int64_t hidden)
{
    const int rc = embed_check(8, tokens, ADAMBRIDGE_DT_F32, vocab, hidden);
    return rc ? rc : (tokens > kRun ? 2 : 1) * tokens * 8 + part_bytes(tokens, hidden) + (vocab + 1) * 4;
}

ADAMBRIDGE_API int adambridge_embed_backward(const void* ids, int32_t id_bytes, int64_t tokens, const void* gout, int32_t dtype,
                                             int64_t vocab, int64_t hidden, float scale, int64_t padding, void* dweight, void* work)
{
    const int rc = embed_check(id_bytes, tokens, dtype, vocab, hidden);
    if (rc) return rc;
    if (!ids || !gout || !dweight || !work) return ADAMBRIDGE_ENULL;
    if ((uintptr_t)work % 8) return ADAMBRIDGE_EALIGN;
    uint64_t* sorted = static_cast<uint64_t*>(work);
    uint64_t* other = tokens > kRun ? sorted + tokens : nullptr;
    // no order of a few; a few thousand over many CUs; many read their run's ids a quarter as often
    if (tokens > kFewIds && tokens <= 4 * kRun) hipLaunchKernelGGL((k_embed_sort<16>), block_grid((tokens + 15) / 16), dim3(kSortThreads), 0, t_stream, ids, id_bytes, tokens, vocab, sorted);
    else if (tokens > kFewIds) hipLaunchKernelGGL((k_embed_sort<64>), block_grid((tokens + 63) / 64), dim3(kSortThreads), 0, t_stream, ids, id_bytes, tokens, vocab, sorted);
    float* const part = reinterpret_cast<float*>(sorted + (tokens > kRun ? 2 : 1) * tokens);
    for (int64_t run = kRun; run < tokens;) {
        const dim3 grid = block_grid((tokens + 255) / 256);
        const int64_t runs = (tokens + run - 1) / run;
        if (runs <= 4) hipLaunchKernelGGL((k_embed_merge<4>), grid, dim3(256), 0, t_stream, sorted, tokens, (uint32_t)run, other);
        else if (runs <= 8) hipLaunchKernelGGL((k_embed_merge<8>), grid, dim3(256), 0, t_stream, sorted, tokens, (uint32_t)run, other);
        else if (runs <= 16) hipLaunchKernelGGL((k_embed_merge<16>), grid, dim3(256), 0, t_stream, sorted, tokens, (uint32_t)run, other);
        else hipLaunchKernelGGL((k_embed_merge<32>), grid, dim3(256), 0, t_stream, sorted, tokens, (uint32_t)run, other);
        run *= runs <= 4 ? 4 : runs <= 8 ? 8 : runs <= 16 ? 16 : 32;
        std::swap(sorted, other);
    }
    EmbedBackArgs A{};
    A.ids = ids;
    A.id_bytes = id_bytes;
    A.sorted = sorted;
    A.gout = gout;
    A.dweight = dweight;
    A.part = part;
    A.starts = reinterpret_cast<int32_t*>(reinterpret_cast<uint8_t*>(part) + part_bytes(tokens, hidden));
    A.tokens = tokens;
    A.vocab = vocab;
    A.padding = padding;
    A.hidden = (int32_t)hidden;
    A.chunk = (int32_t)chunk_of(tokens);
    A.scale = scale;
    if (dtype == ADAMBRIDGE_DT_BF16) launch_embed_back<DT_BF16>(A);
    else launch_embed_back<DT_F32>(A);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? 0 : hip_fail(e, "hipLaunchKernelGGL (embed backward)");
}

}  // extern "C"
