// abh_embed.hip -- rows of an embedding for token ids, and the embedding's gradient.
//
//   y[i] = scale W[ids[i]]                       (an id outside the vocabulary: a row of NaN)
//   dW[v] = scale sum of g[i] over ids[i] = v    (zeros for a word without tokens, and for the padding)
//
// Bytes bound both: T rows read and written; T rows read and V written, most of them zeros.
//
// The gradient's sums run over the tokens sorted by id, then by position, so that they have an order of their own and
// dW is written once, by the words' rows, without atomics on values or a pass that clears it.  Text has a few words
// very often: the tokens in their order are cut into chunks, and a word of more tokens than a chunk has is summed chunk
// by chunk by as many workgroups, whose parts another kernel adds in order; any other word is one wavefront's.
//
// The sort: runs of 2048 (id, position) in a workgroup's LDS, then up to 32 runs at a time become one, each pair's
// place being its own in its run plus how many of every other run are below it (a binary search each: all searches of a
// lane are on their way at once).  Pairs differ, so the order is a total one.

#include <hip/hip_runtime.h>

#include <stdint.h>

#include <algorithm>

#include "../../include/adambridge_hip.h"
#include "abh_device.hpp"
#include "abh_host.hpp"
#include "abh_rows.hpp"

namespace abh {

constexpr int kRun = 2048, kSortThreads = 1024, kMergeRuns = 32;
constexpr int kWords = 16;        // of a workgroup of k_embed_rows
constexpr int kLeastChunk = 64;   // tokens

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

// (id, position) in one word; an id outside the vocabulary is the vocabulary's size, behind all words.
__global__ __launch_bounds__(kSortThreads) void k_embed_sort(const void* ids, int32_t id_bytes, int64_t tokens, int64_t vocab, uint64_t* out)
{
    __shared__ uint64_t item[kRun];
    const int64_t t0 = block_index() * kRun;
    if (t0 >= tokens) return;
    const int n = (int)(tokens - t0 < kRun ? tokens - t0 : kRun);
    int size = 2;   // what is sorted: the next power of two
    while (size < n) size *= 2;
    for (int i = threadIdx.x; i < size; i += kSortThreads) {
        uint64_t x = ~(uint64_t)0;
        if (i < n) {
            const int64_t id = id_at(ids, id_bytes, t0 + i);
            x = (uint64_t)(id >= 0 && id < vocab ? id : vocab) << 32 | (uint32_t)(t0 + i);
        }
        item[i] = x;
    }
    __syncthreads();
    for (int k = 2; k <= size; k *= 2)
        for (int j = k / 2; j > 0; j /= 2) {
            const int i = threadIdx.x;
            if (i < size / 2) {
                const int a = (i & ~(j - 1)) << 1 | (i & (j - 1)), b = a | j;
                const uint64_t x = item[a], y = item[b];
                if ((x > y) == ((a & k) == 0)) {
                    item[a] = y;
                    item[b] = x;
                }
            }
            __syncthreads();
        }
    for (int i = threadIdx.x; i < n; i += kSortThreads) out[t0 + i] = item[i];
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

// Runs of `run` sorted items, kMergeRuns of them at a time: one item a lane.
__global__ __launch_bounds__(256) void k_embed_merge(const uint64_t* in, int64_t tokens, int64_t run, uint64_t* out)
{
    const int64_t i = block_index() * 256 + threadIdx.x;
    if (i >= tokens) return;
    const uint64_t x = in[i];
    const int64_t mine = i / run, first = mine / kMergeRuns * kMergeRuns;
    int64_t place = first * run + (i - mine * run);
    // all runs' searches step by step together, so that their reads overlap
    int32_t lo[kMergeRuns];
#pragma unroll
    for (int r = 0; r < kMergeRuns; ++r) lo[r] = 0;
    int64_t step = 1;
    while (step * 2 <= run) step *= 2;
    for (; step > 0; step >>= 1) {
#pragma unroll
        for (int r = 0; r < kMergeRuns; ++r) {
            const int64_t at = (first + r) * run + lo[r] + step - 1;   // below it: this and all before it are
            if (lo[r] + step <= run && at < tokens && in[at] < x) lo[r] += (int32_t)step;
        }
    }
#pragma unroll
    for (int r = 0; r < kMergeRuns; ++r) place += first + r == mine ? 0 : lo[r];
    out[place] = x;
}

// ------------------------------------------------------------------------------- the gradient

struct EmbedBackArgs {
    const uint64_t* sorted;
    const void* gout;
    void* dweight;
    float* part;          // chunks x 2 x hidden
    int64_t tokens, vocab, padding;
    int32_t hidden, chunk;
    float scale;
};

__device__ __forceinline__ uint32_t word_of(uint64_t item) { return (uint32_t)(item >> 32); }

// Where a word's tokens begin and end, in lo .. hi.
__device__ __forceinline__ int64_t first_of(const uint64_t* sorted, int64_t lo, int64_t hi, uint64_t word)
{
    return lo + below(sorted + lo, hi - lo, word << 32);
}

// Whether the word of the token at place p has more tokens than a chunk.
__device__ __forceinline__ bool is_long(const EmbedBackArgs& A, int64_t p, uint32_t word)
{
    const int64_t lo = p > A.chunk ? p - A.chunk : 0, hi = p + A.chunk < A.tokens ? p + A.chunk + 1 : A.tokens;
    return first_of(A.sorted, p, hi, (uint64_t)word + 1) - first_of(A.sorted, lo, p, word) > A.chunk;
}

// acc += the rows of g at the sorted places from .. to.
template <int DT, int U>
__device__ __forceinline__ void add_rows(const EmbedBackArgs& A, int64_t from, int64_t to, int32_t column, int32_t stride, float (&acc)[U][kLane<DT>])
{
    constexpr int L = kLane<DT>, AHEAD = 8 / U;
    for (int64_t p = from; p < to; p += AHEAD) {
        raw16 w[AHEAD][U];
#pragma unroll
        for (int a = 0; a < AHEAD; ++a) {
            const int64_t place = p + a < to ? p + a : to - 1;
            const void* row = at<DT>(A.gout, (int64_t)(uint32_t)A.sorted[place] * A.hidden);
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (column + u * stride < A.hidden) w[a][u] = load_vec_raw<DT>(row, column + u * stride, A.hidden);
        }
#pragma unroll
        for (int a = 0; a < AHEAD; ++a) {
            if (p + a >= to) break;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (column + u * stride >= A.hidden) continue;
                float x[L];
                to_floats<DT>(w[a][u], x);
#pragma unroll
                for (int k = 0; k < L; ++k) acc[u][k] += x[k];
            }
        }
    }
}

// A chunk's parts of the words that have more tokens than it: one that its first token belongs to, one that its last does.
template <int DT>
__global__ __launch_bounds__(256) void k_embed_parts(EmbedBackArgs A)
{
    constexpr int L = kLane<DT>;
    const int64_t c = block_index(), p0 = c * A.chunk;
    if (p0 >= A.tokens) return;
    const int64_t p1 = p0 + A.chunk < A.tokens ? p0 + A.chunk : A.tokens;
    const uint32_t first = word_of(A.sorted[p0]), last = word_of(A.sorted[p1 - 1]);
    const int32_t column = (int32_t)(blockIdx.y * 256 + threadIdx.x) * L;
    if (column >= A.hidden) return;
#pragma unroll 1
    for (int s = 0; s < 2; ++s) {
        const uint32_t word = s ? last : first;
        if ((s && last == first) || word >= A.vocab || word == A.padding || !is_long(A, s ? p1 - 1 : p0, word)) continue;
        const int64_t from = s ? first_of(A.sorted, p0, p1, word) : p0, to = s ? p1 : first_of(A.sorted, p0, p1, (uint64_t)word + 1);
        float acc[1][L];
#pragma unroll
        for (int k = 0; k < L; ++k) acc[0][k] = 0.0f;
        add_rows<DT, 1>(A, from, to, column, 0, acc);
        store_like<DT_F32, L>(A.part + (c * 2 + s) * A.hidden, column, A.hidden, acc[0]);
    }
}

// The rows of the words of more tokens than a chunk, by the chunk they begin in (no two do in one).
template <int DT>
__global__ __launch_bounds__(256) void k_embed_long(EmbedBackArgs A)
{
    constexpr int L = kLane<DT>;
    const int64_t c = block_index(), p0 = c * A.chunk;
    if (p0 + A.chunk >= A.tokens) return;   // fewer tokens than a chunk's from here on
    const int64_t p1 = p0 + A.chunk;
    const uint32_t word = word_of(A.sorted[p1 - 1]);
    if (word >= A.vocab || word == A.padding || (c > 0 && word_of(A.sorted[p0 - 1]) == word) || !is_long(A, p1 - 1, word)) return;
    const int64_t from = first_of(A.sorted, p0, p1, word), to = first_of(A.sorted, p1, A.tokens, (uint64_t)word + 1);
    const int32_t column = (int32_t)(blockIdx.y * 256 + threadIdx.x) * L;
    if (column >= A.hidden) return;
    float acc[L];
#pragma unroll
    for (int k = 0; k < L; ++k) acc[k] = 0.0f;
    const int64_t end = (to - 1) / A.chunk;
    const int s = from > p0;   // the other chunks begin with the word
    for (int64_t q = c; q <= end; ++q) {
        float x[L];
        load_like<DT_F32, L>(A.part + (q * 2 + (q == c ? s : 0)) * A.hidden, column, A.hidden, 0.0f, x);
#pragma unroll
        for (int k = 0; k < L; ++k) acc[k] += x[k];
    }
#pragma unroll
    for (int k = 0; k < L; ++k) acc[k] *= A.scale;
    stream_vec<DT>(at<DT>(A.dweight, (int64_t)word * A.hidden), column, A.hidden, acc);
}

// All other rows, kWords words a workgroup, pieces of 64 x U vectors a wavefront.
template <int DT, int U>
__global__ __launch_bounds__(256) void k_embed_rows(EmbedBackArgs A)
{
    constexpr int L = kLane<DT>;
    __shared__ int64_t bound[kWords + 1];
    const int64_t v0 = block_index() * kWords;
    if (v0 >= A.vocab) return;
    if (threadIdx.x <= kWords) bound[threadIdx.x] = first_of(A.sorted, 0, A.tokens, (uint64_t)v0 + threadIdx.x);
    __syncthreads();
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / 64);
    const int words = (int)(A.vocab - v0 < kWords ? A.vocab - v0 : kWords);
    const int pieces = (A.hidden + 64 * U * L - 1) / (64 * U * L);
    for (int i = wave; i < words * pieces; i += 4) {
        const int w = i / pieces;
        const int64_t from = bound[w], to = v0 + w == A.padding ? from : bound[w + 1];
        if (to - from > A.chunk) continue;   // k_embed_long's
        const int32_t column = (i - w * pieces) * (64 * U * L) + lane * L;
        if (column >= A.hidden) continue;
        float acc[U][L];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int k = 0; k < L; ++k) acc[u][k] = 0.0f;
        add_rows<DT, U>(A, from, to, column, 64 * L, acc);
        void* out = at<DT>(A.dweight, (v0 + w) * A.hidden);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (column + u * 64 * L >= A.hidden) continue;
#pragma unroll
            for (int k = 0; k < L; ++k) acc[u][k] *= A.scale;
            stream_vec<DT>(out, column + u * 64 * L, A.hidden, acc[u]);
        }
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

// Tokens of a chunk: so many that there are at most 1024 chunks, whose parts are at most 8 KB times the row's values.
static int64_t chunk_of(int64_t tokens)
{
    return std::max<int64_t>(kLeastChunk, (tokens + 1023) / 1024);
}

static int64_t part_bytes(int64_t tokens, int64_t hidden)
{
    const int64_t chunk = chunk_of(tokens);
    return tokens > chunk ? (tokens + chunk - 1) / chunk * 2 * hidden * 4 : 0;   // else no word is longer than a chunk
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
static void launch_embed_back(const EmbedBackArgs& A)
{
    const int vectors = (A.hidden + kLane<DT> - 1) / kLane<DT>;
    if (A.tokens > A.chunk) {
        const dim3 grid = block_grid((A.tokens + A.chunk - 1) / A.chunk, (vectors + 255) / 256);
        hipLaunchKernelGGL((k_embed_parts<DT>), grid, dim3(256), 0, t_stream, A);
        hipLaunchKernelGGL((k_embed_long<DT>), grid, dim3(256), 0, t_stream, A);
    }
    const dim3 grid = block_grid((A.vocab + kWords - 1) / kWords);
    if (vectors <= 64) hipLaunchKernelGGL((k_embed_rows<DT, 1>), grid, dim3(256), 0, t_stream, A);
    else hipLaunchKernelGGL((k_embed_rows<DT, 2>), grid, dim3(256), 0, t_stream, A);
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
    return rc ? rc : (tokens > kRun ? 2 : 1) * tokens * 8 + part_bytes(tokens, hidden);
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
    hipLaunchKernelGGL(k_embed_sort, block_grid((tokens + kRun - 1) / kRun), dim3(kSortThreads), 0, t_stream, ids, id_bytes, tokens, vocab, sorted);
    float* const part = reinterpret_cast<float*>(sorted + (tokens > kRun ? 2 : 1) * tokens);
    for (int64_t run = kRun; run < tokens; run *= kMergeRuns) {
        hipLaunchKernelGGL(k_embed_merge, block_grid((tokens + 255) / 256), dim3(256), 0, t_stream, sorted, tokens, run, other);
        std::swap(sorted, other);
    }
    const EmbedBackArgs A{sorted, gout, dweight, part, tokens, vocab, padding, (int32_t)hidden, (int32_t)chunk_of(tokens), scale};
    if (dtype == ADAMBRIDGE_DT_BF16) launch_embed_back<DT_BF16>(A);
    else launch_embed_back<DT_F32>(A);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? 0 : hip_fail(e, "hipLaunchKernelGGL (embed backward)");
}

}  // extern "C"
