// abh_route.hip -- tokens to experts and back: the router's choice, the order of the chosen, and the rows'
// way there (dispatch) and back (combine).
//
// A token's top_k largest logits are chosen (the lower index of equal ones; a NaN counts as the largest), and
// their weights are the softmax over the chosen or over all.  The T k assignments, token by token, are sorted by
// expert, stably, so that an expert's rows lie together in the tokens' order:
//
//   ends[e]      = how many assignments have experts 0 .. e
//   order[r]     = the assignment t k + j that row r is
//   position[t, j] = its row
//
// Bytes bound all of it: the logits once; x once and its k copies; k rows and their sum.  Nothing depends on
// the order of atomics: 64 tokens are a block, an expert's tokens in a block are one 64-bit mask (set by or, whose order
// does not matter), a token's rank among them the bits below its own, and the blocks' counts are summed
// in order.  Up to 64 tokens are one launch; more are three: choice and counts, the counts' prefix
// sums, and the places.

#include <hip/hip_runtime.h>

#include <stdint.h>

#include "../../include/adambridge_hip.h"
#include "abh_choice.hpp"
#include "abh_device.hpp"
#include "abh_host.hpp"
#include "abh_rows.hpp"

namespace abh {

constexpr int kBlockTokens = 64;
constexpr int kRouteThreads = 1024;   // so that a block of tokens is chosen from in few passes: blocks are few
constexpr int kMostExperts = 1024;
constexpr int kMostChosen = 64;

struct RouteArgs {
    const void* logits;
    int64_t tokens;
    int32_t experts, top_k, normalize, blocks;
    float* weights;      // tokens x top_k
    int32_t* chosen;     // tokens x top_k
    int32_t* ends;       // experts
    int32_t* order;      // tokens top_k
    int32_t* position;   // tokens x top_k
    uint8_t* counts;     // experts x blocks
    int32_t* bases;      // experts x blocks
};

// Masks of a block's tokens by expert, and the rows of its assignments: base[e] + the bits below.
__device__ __forceinline__ void place_block(const RouteArgs& A, const uint64_t* mask, const int32_t* base, int64_t base_stride,
                                            int64_t t0, int tokens)
{
    for (int i = threadIdx.x; i < tokens * A.top_k; i += kRouteThreads) {
        const int64_t a = t0 * A.top_k + i;
        const int e = A.chosen[a], t = i / A.top_k;
        const int row = base[(int64_t)e * base_stride] + __builtin_popcountll(mask[e] & (((uint64_t)1 << t) - 1));
        A.position[a] = row;
        A.order[row] = (int32_t)a;
    }
}

// 64 tokens a workgroup, G lanes a token, NV logits a lane (expert lane * NV + v).  Bound by its instructions, not by its
// bytes: few lanes a token, so that a step over the lanes serves several tokens.
template <int DT, int G, int NV>
__global__ __launch_bounds__(kRouteThreads) void k_route(RouteArgs A)
{
    __shared__ uint64_t mask[kMostExperts];
    __shared__ int32_t base[kMostExperts];
    constexpr int kPass = kRouteThreads / G;   // tokens at a time
    const int lane = threadIdx.x % G, sub = threadIdx.x / G;
    const int64_t block = block_index(), t0 = block * kBlockTokens;
    if (block >= A.blocks) return;
    const int tokens = (int)(A.tokens - t0 < kBlockTokens ? A.tokens - t0 : kBlockTokens);
    for (int e = threadIdx.x; e < A.experts; e += kRouteThreads) mask[e] = 0;
    __syncthreads();
    for (int t = sub; t < kBlockTokens; t += kPass) {
        const bool real = t < tokens;
        if (!__builtin_amdgcn_ballot_w64(real)) break;   // a wavefront's groups go on together: they share its sums' lanes
        float x[NV];
        uint32_t key[NV];
        const void* row = at<DT>(A.logits, (t0 + (real ? t : 0)) * A.experts);
        if constexpr (NV % kLane<DT> == 0) {
#pragma unroll
            for (int v = 0; v < NV; v += kLane<DT>) load_vec<DT>(row, lane * NV + v, A.experts, x + v);
        } else {
#pragma unroll
            for (int v = 0; v < NV; ++v) x[v] = lane * NV + v < A.experts ? get<DT>(row, lane * NV + v) : 0.0f;
        }
#pragma unroll
        for (int v = 0; v < NV; ++v) key[v] = lane * NV + v < A.experts ? order_key(x[v]) : 0u;
        float top = 0.0f, sum = 0.0f, mine = 0.0f;
        int my_expert = 0;
        for (int j = 0; j < A.top_k; ++j) {
            uint32_t most = key[0];
#pragma unroll
            for (int v = 1; v < NV; ++v) most = most > key[v] ? most : key[v];
            most = group_max<G>(most);
            uint32_t e = ~0u;   // the lowest index that has it
#pragma unroll
            for (int v = NV - 1; v >= 0; --v) e = key[v] == most ? (uint32_t)v : e;
            e = e == ~0u ? e : lane * NV + e;
            e = group_reduce<G>(e, [](uint32_t a, uint32_t b) { return a < b ? a : b; });
#pragma unroll
            for (int v = 0; v < NV; ++v) key[v] = e == (uint32_t)(lane * NV + v) ? 0u : key[v];
            const float value = key_value(most);
            if (j == 0) {
                top = value;
                if (!A.normalize) {   // the sum over all experts
#pragma unroll
                    for (int v = 0; v < NV; ++v) sum += lane * NV + v < A.experts ? exp_below(x[v], top) : 0.0f;
                    sum = group_sum<G>(sum);
                }
            }
            const float w = exp_below(value, top);
            if (A.normalize) sum += w;
            if (lane == j) {
                mine = w;
                my_expert = (int)e;
            }
        }
        if (real && lane < A.top_k) {
            const int64_t a = (t0 + t) * A.top_k + lane;
            A.weights[a] = top == kRouteNegInf ? 0.0f : mine / sum;
            A.chosen[a] = my_expert;
            atomicOr(reinterpret_cast<unsigned long long*>(&mask[my_expert]), 1ull << t);
        }
    }
    __syncthreads();
    if (A.blocks > 1) {
        for (int e = threadIdx.x; e < A.experts; e += kRouteThreads)
            A.counts[(int64_t)e * A.blocks + block] = (uint8_t)__builtin_popcountll(mask[e]);
        return;
    }
    if (threadIdx.x < kWave) {   // one wavefront sums the experts' counts
        int32_t before = 0;
        for (int e0 = 0; e0 < A.experts; e0 += kWave) {
            const int e = e0 + (int)threadIdx.x;
            const int32_t n = e < A.experts ? (int32_t)__builtin_popcountll(mask[e]) : 0;
            int32_t s = n;
#pragma unroll
            for (int d = 1; d < kWave; d *= 2) {
                const int32_t y = __shfl_up(s, d);
                if ((int)threadIdx.x >= d) s += y;
            }
            if (e < A.experts) {
                base[e] = before + s - n;
                A.ends[e] = before + s;
            }
            before += __shfl(s, kWave - 1);
        }
    }
    __threadfence_block();
    __syncthreads();
    place_block(A, mask, base, 1, t0, tokens);
}

// One expert a workgroup: the rows of the experts before it, then its blocks' prefix sums.
__global__ __launch_bounds__(1024) void k_route_bases(RouteArgs A)
{
    constexpr int T = 1024;
    __shared__ int32_t part[T / kWave];
    const int e = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x / kWave;
    // bytes 0 .. e * blocks, four at a time where they are aligned (the array is)
    const int64_t n = (int64_t)e * A.blocks;
    int32_t s = 0;
    const uint32_t* words = reinterpret_cast<const uint32_t*>(A.counts);
    for (int64_t i = threadIdx.x; i < n / 4; i += T) {
        const uint32_t w = words[i];
        s += (int32_t)((w & 255u) + (w >> 8 & 255u) + (w >> 16 & 255u) + (w >> 24));
    }
    for (int64_t i = n / 4 * 4 + threadIdx.x; i < n; i += T) s += A.counts[i];
    s = group_reduce<kWave>(s, [](int32_t a, int32_t b) { return a + b; });
    if (lane == 0) part[wave] = s;
    __syncthreads();
    int32_t before = 0;
    for (int w = 0; w < T / kWave; ++w) before += part[w];
    for (int b0 = 0; b0 < A.blocks; b0 += T) {
        const int b = b0 + (int)threadIdx.x;
        const int32_t c = b < A.blocks ? A.counts[n + b] : 0;
        int32_t x = c;
#pragma unroll
        for (int d = 1; d < kWave; d *= 2) {
            const int32_t y = __shfl_up(x, d);
            if (lane >= d) x += y;
        }
        __syncthreads();
        if (lane == kWave - 1) part[wave] = x;
        __syncthreads();
        int32_t waves = 0, all = 0;
        for (int w = 0; w < T / kWave; ++w) {
            if (w < wave) waves += part[w];
            all += part[w];
        }
        if (b < A.blocks) A.bases[n + b] = before + waves + x - c;
        before += all;
    }
    if (threadIdx.x == 0) A.ends[e] = before;
}

__global__ __launch_bounds__(kRouteThreads) void k_route_places(RouteArgs A)
{
    __shared__ uint64_t mask[kMostExperts];
    const int64_t block = block_index(), t0 = block * kBlockTokens;
    if (block >= A.blocks) return;
    const int tokens = (int)(A.tokens - t0 < kBlockTokens ? A.tokens - t0 : kBlockTokens);
    for (int e = threadIdx.x; e < A.experts; e += kRouteThreads) mask[e] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < tokens * A.top_k; i += kRouteThreads)
        atomicOr(reinterpret_cast<unsigned long long*>(&mask[A.chosen[t0 * A.top_k + i]]), 1ull << (i / A.top_k));
    __syncthreads();
    place_block(A, mask, A.bases + block, A.blocks, t0, tokens);
}

// dlogits of the chosen's softmax, w_j (g_j - sum w g), or of all's, [e = chosen_j] w_j g_j - p_e sum w g.  A wavefront a
// token, which spreads the chosen's values over the experts in its part of the LDS.
template <int DT>
__global__ __launch_bounds__(256) void k_route_back(const float* weights, const int32_t* chosen, const float* gout,
                                                    const void* logits, int64_t tokens, int32_t experts, int32_t top_k,
                                                    int32_t normalize, void* grad)
{
    __shared__ float spread[4][kMostExperts];
    const int lane = threadIdx.x & 63, wave = threadIdx.x / kWave;
    const int64_t t = block_index() * 4 + wave;
    const bool real = t < tokens, picks = real && lane < top_k;
    const float w = picks ? weights[t * top_k + lane] : 0.0f;
    const float g = picks ? gout[t * top_k + lane] : 0.0f;
    const int at_e = picks ? chosen[t * top_k + lane] : -1;
    for (int e = lane; e < experts; e += kWave) spread[wave][e] = 0.0f;
    const float total = wave_sum(picks ? w * g : 0.0f);
    __syncthreads();   // zeros before values, values before reads
    if (picks && at_e >= 0 && at_e < experts) spread[wave][at_e] = normalize ? w * (g - total) : w * g;
    __syncthreads();
    if (!real) return;
    const int64_t row = t * experts;
    if (normalize) {
        for (int e = lane; e < experts; e += kWave) put<DT>(grad, row + e, spread[wave][e]);
        return;
    }
    float most = kRouteNegInf, sum = 0.0f;
    bool nan = false;
    for (int e = lane; e < experts; e += kWave) {
        const float x = get<DT>(logits, row + e);
        most = __builtin_fmaxf(most, x);
        nan |= x != x;
    }
    most = group_reduce<kWave>(most, [](float a, float b) { return __builtin_fmaxf(a, b); });
    const float top = __builtin_amdgcn_ballot_w64(nan) ? __builtin_nanf("") : most;
    for (int e = lane; e < experts; e += kWave) sum += exp_below(get<DT>(logits, row + e), top);
    sum = wave_sum(sum);
    const float inv = top == kRouteNegInf ? 0.0f : 1.0f / sum;
    for (int e = lane; e < experts; e += kWave)
        put<DT>(grad, row + e, spread[wave][e] - exp_below(get<DT>(logits, row + e), top) * inv * total);
}

// ---------------------------------------------------------------- dispatch and combine

struct ShuffleArgs {
    const void* x;            // tokens x cols, or rows x cols
    const void* g;
    const float* weights;     // tokens x top_k
    const int32_t* position;  // tokens x top_k
    void* out;
    float* dw;
    int64_t tokens, cols;
    int32_t top_k;
};

// The rows of a token's assignments, one a lane; -1 where it is none (a position that no routing gives): nothing is
// read or written there.  One load for all of them, not one before each row.
__device__ __forceinline__ int rows_of(const ShuffleArgs& A, int64_t t)
{
    const int lane = threadIdx.x & 63;
    const int r = lane < A.top_k ? A.position[t * A.top_k + lane] : -1;
    return r >= 0 && r < A.tokens * A.top_k ? r : -1;
}

// Tokens have a wavefront each, which takes `vectors` vectors of a lane of it (blockIdx.y the ones after).
struct Place {
    int64_t t, c0, c1;
};

template <int DT>
__device__ __forceinline__ bool place_of(const ShuffleArgs& A, int vectors, Place& p)
{
    constexpr int64_t a_load = kWave * kLane<DT>;
    p.t = block_index() * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    p.c0 = (int64_t)blockIdx.y * vectors * a_load + (threadIdx.x & 63) * kLane<DT>;
    p.c1 = ((int64_t)blockIdx.y + 1) * vectors * a_load;
    p.c1 = p.c1 < A.cols ? p.c1 : A.cols;
    return p.t < A.tokens;
}

// out[position[t, j]] = x[t]: the token's row read once, written top_k times.
template <int DT>
__global__ __launch_bounds__(256) void k_dispatch(ShuffleArgs A, int vectors)
{
    constexpr int K = kLane<DT>;
    Place p;
    if (!place_of<DT>(A, vectors, p)) return;
    const int rows = rows_of(A, p.t);
    for (int64_t c = p.c0; c < p.c1; c += kWave * K) {
        const raw16 v = load_vec_raw<DT>(at<DT>(A.x, p.t * A.cols), c, A.cols);
        float f[K];
        to_floats<DT>(v, f);
        for (int j = 0; j < A.top_k; ++j) {
            const int r = __builtin_amdgcn_readlane(rows, j);
            if (r < 0) continue;
            void* out = at<DT>(A.out, (int64_t)r * A.cols);
            if (c + K <= A.cols) stream_raw<DT>(out, c, v);
            else stream_vec<DT>(out, c, A.cols, f);
        }
    }
}

// out[t] = sum over j of weights[t, j] x[position[t, j]] (without weights: of the rows), in order, rounded once.  The
// rows of four choices are on their way at a time.
template <int DT>
__global__ __launch_bounds__(256) void k_combine(ShuffleArgs A, int vectors)
{
    constexpr int K = kLane<DT>, U = 4;
    Place p;
    if (!place_of<DT>(A, vectors, p)) return;
    const int rows = rows_of(A, p.t), lane = threadIdx.x & 63;
    const float weight = !A.weights ? 1.0f : lane < A.top_k ? A.weights[p.t * A.top_k + lane] : 0.0f;
    for (int64_t c = p.c0; c < p.c1; c += kWave * K) {
        float s[K];
#pragma unroll
        for (int k = 0; k < K; ++k) s[k] = 0.0f;
        for (int j0 = 0; j0 < A.top_k; j0 += U) {
            raw16 v[U];
            int r[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                r[u] = j0 + u < A.top_k ? __builtin_amdgcn_readlane(rows, j0 + u) : -1;
                if (r[u] >= 0) v[u] = load_vec_raw<DT>(at<DT>(A.x, (int64_t)r[u] * A.cols), c, A.cols);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (r[u] < 0) continue;
                const float w = bitsf(__builtin_amdgcn_readlane(fbits(weight), j0 + u));
                float f[K];
                to_floats<DT>(v[u], f);
#pragma unroll
                for (int k = 0; k < K; ++k) s[k] = __builtin_fmaf(w, f[k], s[k]);
            }
        }
        stream_vec<DT>(at<DT>(A.out, p.t * A.cols), c, A.cols, s);
    }
}

// An assignment a wavefront: out[row] = w g[t], dw = <g[t], x[row]>.  The rows, kept since the forward pass, are in no
// cache and read once (streamed: 113 -> 100 us for 16384 x 4 of 2048; combine's own, just written, are in one).
template <int DT>
__global__ __launch_bounds__(256) void k_combine_back(ShuffleArgs A)
{
    constexpr int K = kLane<DT>, U = 4;
    const int lane = threadIdx.x & 63;
    const int64_t a = block_index() * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    if (a >= A.tokens * A.top_k) return;
    const int64_t t = a / A.top_k, r = A.position[a];
    float dot = 0.0f;
    if (r >= 0 && r < A.tokens * A.top_k) {
        const float w = A.weights[a];
        const void* gt = at<DT>(A.g, t * A.cols);
        const void* xr = at<DT>(A.x, r * A.cols);
        for (int64_t c = (int64_t)lane * K; c < A.cols; c += U * kWave * K) {
            raw16 g[U], v[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int64_t cu = c + u * kWave * K;
                if (cu >= A.cols) continue;
                g[u] = load_vec_raw<DT>(gt, cu, A.cols);
                if (A.dw) v[u] = load_vec_raw<DT, true>(xr, cu, A.cols);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int64_t cu = c + u * kWave * K;
                if (cu >= A.cols) continue;
                float gf[K], vf[K];
                to_floats<DT>(g[u], gf);
                if (A.dw) {
                    to_floats<DT>(v[u], vf);
#pragma unroll
                    for (int k = 0; k < K; ++k) dot = __builtin_fmaf(gf[k], vf[k], dot);
                }
                if (A.out) {
#pragma unroll
                    for (int k = 0; k < K; ++k) gf[k] *= w;
                    stream_vec<DT>(at<DT>(A.out, r * A.cols), cu, A.cols, gf);
                }
            }
        }
    }
    if (A.dw) {
        dot = wave_sum(dot);
        if (lane == 0) A.dw[a] = dot;
    }
}

static bool route_type_ok(int32_t t) { return t == ADAMBRIDGE_DT_F32 || t == ADAMBRIDGE_DT_BF16; }

static int route_sizes(int64_t tokens, int64_t experts, int64_t top_k)
{
    const int64_t most = ((int64_t)1 << 31) - 1;
    return tokens >= 1 && tokens <= most && experts >= 1 && experts <= kMostExperts && top_k >= 1 && top_k <= kMostChosen &&
           top_k <= experts && tokens * top_k <= most ? 0 : ADAMBRIDGE_EBADN;
}

template <int DT>
static void launch_route(const RouteArgs& A)
{
    // 16 lanes a token while its choices fit them and its logits their registers: four tokens share a wavefront (measured on MI355X,
    // us, beside 64 lanes a token: 64 tokens choosing 4 of 64 4.6 / 9.6, 4096 choosing 8 of 128 13.0 / 23.5, 32768 choosing 8 of 256
    // 38 / 51)
#define ABH_ROUTE(G, NV)                                                                                        \
    if (A.experts <= G * NV && A.top_k <= G) {                                                                  \
        hipLaunchKernelGGL((k_route<DT, G, NV>), block_grid(A.blocks), dim3(kRouteThreads), 0, t_stream, A);     \
        return;                                                                                                 \
    }
    ABH_ROUTE(16, 1) ABH_ROUTE(16, 2) ABH_ROUTE(16, 4) ABH_ROUTE(16, 8) ABH_ROUTE(16, 16) ABH_ROUTE(64, 16)
#undef ABH_ROUTE
}

static int done(const char* what)
{
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? 0 : hip_fail(e, what);
}

static int shuffle_check(const void* a, const void* out, const int32_t* position, int32_t dtype, int64_t tokens, int64_t top_k,
                         int64_t cols)
{
    const int rc = route_sizes(tokens, kMostExperts, top_k);
    if (rc || cols < 1 || cols > (int64_t)1 << 22) return ADAMBRIDGE_EBADN;
    if (!route_type_ok(dtype)) return ADAMBRIDGE_EMVDTYPE;
    return a && out && position ? 0 : ADAMBRIDGE_ENULL;
}

// Many tokens: a wavefront takes `many` vectors a lane of a token.  Few: one, so that more wavefronts share them.  Measured on
// MI355X in BF16 that is in no cache, us, one / many.  dispatch: 256 tokens to 4 rows of 2048 3.2 / 4.7, 4096 18.7 / 17.9, 16384
// 76.8 / 62.3; combine: 512 tokens of 8 rows of 4096 8.0 / 25.4, 2048 of 4 of 2048 8.5 / 10.2, 4096 15.5 / 15.6, 8192 of 2 of 8192
// 94.7 / 88.9.
static int shuffle_vectors(const ShuffleArgs& A, int many) { return A.tokens >= 4096 ? many : 1; }
constexpr int kDispatchVectors = 1 << 20, kCombineVectors = 8;

static dim3 shuffle_grid(const ShuffleArgs& A, int32_t dtype, int vectors)
{
    const int64_t a_wave = (int64_t)vectors * kWave * (dtype == ADAMBRIDGE_DT_BF16 ? kLane<DT_BF16> : kLane<DT_F32>);
    return block_grid((A.tokens + 3) / 4, (A.cols + a_wave - 1) / a_wave);
}

}  // namespace abh

using namespace abh;

extern "C" {

ADAMBRIDGE_API int64_t adambridge_route_work(int64_t tokens, int64_t experts, int64_t top_k)
{
    if (route_sizes(tokens, experts, top_k)) return ADAMBRIDGE_EBADN;
    const int64_t blocks = (tokens + kBlockTokens - 1) / kBlockTokens;
    return blocks == 1 ? 0 : (experts * blocks + 3) / 4 * 4 + experts * blocks * 4;
}

ADAMBRIDGE_API int adambridge_route(const void* logits, int32_t dtype, int64_t tokens, int64_t experts, int64_t top_k,
                                    int32_t normalize, float* weights, int32_t* chosen, int32_t* ends, int32_t* order,
                                    int32_t* position, void* work)
{
    if (route_sizes(tokens, experts, top_k)) return ADAMBRIDGE_EBADN;
    if (!route_type_ok(dtype)) return ADAMBRIDGE_EMVDTYPE;
    const int64_t blocks = (tokens + kBlockTokens - 1) / kBlockTokens;
    if (!logits || !weights || !chosen || !ends || !order || !position || (blocks > 1 && !work)) return ADAMBRIDGE_ENULL;
    if ((uintptr_t)work % 4) return ADAMBRIDGE_EALIGN;
    RouteArgs A{logits, tokens, (int32_t)experts, (int32_t)top_k, normalize != 0, (int32_t)blocks, weights, chosen, ends, order,
                position, static_cast<uint8_t*>(work), nullptr};
    if (blocks > 1) A.bases = reinterpret_cast<int32_t*>(A.counts + (experts * blocks + 3) / 4 * 4);
    if (dtype == ADAMBRIDGE_DT_BF16) launch_route<DT_BF16>(A);
    else launch_route<DT_F32>(A);
    if (blocks > 1) {
        hipLaunchKernelGGL(k_route_bases, dim3((unsigned)experts), dim3(1024), 0, t_stream, A);
        hipLaunchKernelGGL(k_route_places, block_grid(blocks), dim3(kRouteThreads), 0, t_stream, A);
    }
    return done("hipLaunchKernelGGL (route)");
}

ADAMBRIDGE_API int adambridge_route_backward(const float* weights, const int32_t* chosen, const float* gout, const void* logits,
                                             int32_t dtype, int64_t tokens, int64_t experts, int64_t top_k, int32_t normalize,
                                             void* grad)
{
    if (route_sizes(tokens, experts, top_k)) return ADAMBRIDGE_EBADN;
    if (!route_type_ok(dtype)) return ADAMBRIDGE_EMVDTYPE;
    if (!weights || !chosen || !gout || !grad || (!normalize && !logits)) return ADAMBRIDGE_ENULL;
    const dim3 grid = block_grid((tokens + 3) / 4);
    if (dtype == ADAMBRIDGE_DT_BF16)
        hipLaunchKernelGGL((k_route_back<DT_BF16>), grid, dim3(256), 0, t_stream, weights, chosen, gout, logits, tokens,
                           (int32_t)experts, (int32_t)top_k, normalize, grad);
    else
        hipLaunchKernelGGL((k_route_back<DT_F32>), grid, dim3(256), 0, t_stream, weights, chosen, gout, logits, tokens,
                           (int32_t)experts, (int32_t)top_k, normalize, grad);
    return done("hipLaunchKernelGGL (route's gradient)");
}

ADAMBRIDGE_API int adambridge_dispatch(const void* x, int32_t dtype, const int32_t* position, int64_t tokens, int64_t top_k,
                                       int64_t cols, void* rows)
{
    if (const int rc = shuffle_check(x, rows, position, dtype, tokens, top_k, cols)) return rc;
    const ShuffleArgs A{x, nullptr, nullptr, position, rows, nullptr, tokens, cols, (int32_t)top_k};
    const int vectors = shuffle_vectors(A, kDispatchVectors);
    if (dtype == ADAMBRIDGE_DT_BF16) hipLaunchKernelGGL((k_dispatch<DT_BF16>), shuffle_grid(A, dtype, vectors), dim3(256), 0, t_stream, A, vectors);
    else hipLaunchKernelGGL((k_dispatch<DT_F32>), shuffle_grid(A, dtype, vectors), dim3(256), 0, t_stream, A, vectors);
    return done("hipLaunchKernelGGL (dispatch)");
}

ADAMBRIDGE_API int adambridge_combine(const void* rows, int32_t dtype, const float* weights, const int32_t* position,
                                      int64_t tokens, int64_t top_k, int64_t cols, void* out)
{
    if (const int rc = shuffle_check(rows, out, position, dtype, tokens, top_k, cols)) return rc;
    const ShuffleArgs A{rows, nullptr, weights, position, out, nullptr, tokens, cols, (int32_t)top_k};
    const int vectors = shuffle_vectors(A, kCombineVectors);
    if (dtype == ADAMBRIDGE_DT_BF16) hipLaunchKernelGGL((k_combine<DT_BF16>), shuffle_grid(A, dtype, vectors), dim3(256), 0, t_stream, A, vectors);
    else hipLaunchKernelGGL((k_combine<DT_F32>), shuffle_grid(A, dtype, vectors), dim3(256), 0, t_stream, A, vectors);
    return done("hipLaunchKernelGGL (combine)");
}

ADAMBRIDGE_API int adambridge_combine_backward(const void* gout, const void* rows, int32_t dtype, const float* weights,
                                               const int32_t* position, int64_t tokens, int64_t top_k, int64_t cols, void* drows,
                                               float* dweights)
{
    if (const int rc = shuffle_check(gout, weights, position, dtype, tokens, top_k, cols)) return rc;
    if (dweights && !rows) return ADAMBRIDGE_ENULL;
    if (!drows && !dweights) return 0;
    const ShuffleArgs A{rows, gout, weights, position, drows, dweights, tokens, cols, (int32_t)top_k};
    const dim3 grid = block_grid((tokens * top_k + 3) / 4);
    if (dtype == ADAMBRIDGE_DT_BF16) hipLaunchKernelGGL((k_combine_back<DT_BF16>), grid, dim3(256), 0, t_stream, A);
    else hipLaunchKernelGGL((k_combine_back<DT_F32>), grid, dim3(256), 0, t_stream, A);
    return done("hipLaunchKernelGGL (combine's gradient)");
}

}  // extern "C"
