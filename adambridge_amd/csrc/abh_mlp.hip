// abh_mlp.hip -- a layer of expert MLPs for a few tokens, from the router's logits to the result, in two kernels.
//
//   out[t] = sum over the top_k experts e of token t, w[t, e] down[e] a(t, e)
//   a(t, e) = act(up[e] x[t]),  or  act(gate[e] x[t]) * up[e] x[t]
//
// A few tokens' layer is the chosen experts' weights, read once from HBM, and what a
// call costs beside: as route, dispatch, two or three products, an activation and combine it is seven launches, each with its
// results through memory.  Here the first kernel chooses (every workgroup for itself: a few tokens' logits are a few KB), takes
// its 16 rows of one chosen expert's up (and gate) times all tokens, and stores the activations; the second takes 16
// rows of down of all chosen experts, weights and adds their products, and stores the result.
//
// The tokens, up to 16, are the other side of the matrix instructions, whatever their number: an expert's weights are read once
// for all tokens that chose it.  (One token, 8 of 64 experts 1536 x 2048 BF16: 12.8 and 11.1 us for 50 MB each; 13 tokens, 2 of 8 gated experts
// 8192 x 2048: 100 us for 537 MB, 57 for 268.)  Activations are rounded to the operands' type, which the instructions take; all other
// sums are FP32, in an order of their own.

#include <hip/hip_runtime.h>

#include <stdint.h>

#include <algorithm>

#include "../../include/adambridge_hip.h"
#include "abh_choice.hpp"
#include "abh_device.hpp"
#include "abh_host.hpp"
#include "abh_rows.hpp"
#include "abh_tiles.hpp"

namespace abh {

constexpr int kMlpTokens = 16, kMlpExperts = 1024, kMlpChosen = 64;
constexpr int kMlpColumns = 16;   // a matrix instruction's
constexpr int kUpWaves = 4, kDownWaves = 16;
constexpr int kMlpCus = 256;

// A chosen expert: which tokens chose it, and their weights.
struct Chosen {
    int32_t expert;
    uint32_t tokens;
    float weight[kMlpTokens];
};

struct MlpArgs {
    const void *x, *logits, *up, *gate, *down;
    void* out;
    Chosen* list;      // the chosen experts, in order of their number
    int32_t* count;    // how many
    void* a;           // chosen experts x 16 x inter
    int32_t tokens, experts, top_k, inter, hidden;
    int32_t used;      // the most experts that can be chosen
    int32_t logits_bf16, normalize, silu;
    int32_t columns;   // workgroups of a chosen expert
};

// x Phi(x), and x / (1 + exp(-x)).
__device__ __forceinline__ float activated(float x, bool silu)
{
    return silu ? x / (1.0f + expf(-x)) : 0.5f * x * (1.0f + erff(x * 0.70710678118654752f));
}

__device__ __forceinline__ float logit(const MlpArgs& A, int64_t i)
{
    return A.logits_bf16 ? get<DT_BF16>(A.logits, i) : get<DT_F32>(A.logits, i);
}

// The choice of all tokens, a wavefront a token, NV logits a lane (expert 64 v + lane).
template <int NV>
__device__ __forceinline__ void choose(const MlpArgs& A, uint32_t* mask, int32_t* expert, float* weight)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x / kWave;
    for (int e = threadIdx.x; e < A.experts; e += kUpWaves * kWave) mask[e] = 0;
    __syncthreads();
    constexpr int TOKENS = kMlpTokens / kUpWaves;   // of a wavefront; their logits are asked for at once
    float logits[TOKENS][NV];
#pragma unroll
    for (int i = 0; i < TOKENS; ++i)
#pragma unroll
        for (int v = 0; v < NV; ++v)
            logits[i][v] = wave + i * kUpWaves < A.tokens && 64 * v + lane < A.experts ? logit(A, (int64_t)(wave + i * kUpWaves) * A.experts + 64 * v + lane) : 0.0f;
#pragma unroll
    for (int i = 0; i < TOKENS; ++i) {
        const int t = wave + i * kUpWaves;
        if (t >= A.tokens) break;
        float(&x)[NV] = logits[i];
        uint32_t key[NV];
#pragma unroll
        for (int v = 0; v < NV; ++v) key[v] = 64 * v + lane < A.experts ? order_key(x[v]) : 0u;
        float top = 0.0f, sum = 0.0f, mine = 0.0f;
        int my_expert = 0;
        for (int j = 0; j < A.top_k; ++j) {
            uint32_t most = key[0];
#pragma unroll
            for (int v = 1; v < NV; ++v) most = most > key[v] ? most : key[v];
            most = group_max<kWave>(most);
            int e = 0;   // the lowest index that has it
#pragma unroll
            for (int v = NV - 1; v >= 0; --v) {
                const uint64_t with = __builtin_amdgcn_ballot_w64(key[v] == most);
                e = with ? 64 * v + __builtin_ctzll(with) : e;
            }
#pragma unroll
            for (int v = 0; v < NV; ++v) key[v] = 64 * v + lane == e ? 0u : key[v];
            const float value = key_value(most);
            if (j == 0) {
                top = value;
                if (!A.normalize) {   // the sum over all experts
#pragma unroll
                    for (int v = 0; v < NV; ++v) sum += 64 * v + lane < A.experts ? exp_below(x[v], top) : 0.0f;
                    sum = wave_sum(sum);
                }
            }
            const float w = exp_below(value, top);
            if (A.normalize) sum += w;
            if (lane == j) {
                mine = w;
                my_expert = e;
            }
        }
        if (lane < A.top_k) {
            weight[t * A.top_k + lane] = top == kRouteNegInf ? 0.0f : mine / sum;
            expert[t * A.top_k + lane] = my_expert;
            atomicOr(&mask[my_expert], 1u << t);
        }
    }
    __syncthreads();
}

// 16 NG columns of up (and gate) of a chosen expert at a time: the wavefronts split the sum, the first adds their parts in order, while
// the next columns' first weights are on their way.
template <int DT, bool EVEN, bool GATE, int NG, int NV>
__global__ __launch_bounds__(kUpWaves * kWave, EVEN ? 4 : 2) void k_mlp_up(MlpArgs A)
{
    constexpr int V = kLane<DT>, STEP = 4 * V, W = kUpWaves, M = (GATE ? 2 : 1) * NG, U = M == 4 ? 2 : 4, COLS = kMlpColumns * NG;   // M: up's columns, then gate's
    __shared__ uint32_t mask[kMlpExperts];
    __shared__ int32_t expert[kMlpTokens * kMlpChosen];
    __shared__ float weight[kMlpTokens * kMlpChosen];
    __shared__ uint16_t list[kMlpExperts];
    __shared__ mm_f32x4 parts[2][W - 1][M][64];
    choose<NV>(A, mask, expert, weight);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / kWave);
    const int col = lane & 15, quarter = lane >> 4;
    int count = 0;   // the chosen experts, in order of their number
    for (int e0 = 0; e0 < A.experts; e0 += kWave) {
        const bool chosen = e0 + lane < A.experts && mask[e0 + lane < A.experts ? e0 + lane : 0] != 0;
        const uint64_t with = __builtin_amdgcn_ballot_w64(chosen);
        if (chosen && wave == 0) list[count + __builtin_popcountll(with & (((uint64_t)1 << lane) - 1))] = (uint16_t)(e0 + lane);
        count += __builtin_popcountll(with);
    }
    __syncthreads();
    if (blockIdx.x == 0 && threadIdx.x == 0) *A.count = count;
    const int steps = (A.hidden + STEP - 1) / STEP, s0 = steps * wave / W, s1 = steps * (wave + 1) / W;
    const int turns = ((steps + W - 1) / W + U - 1) / U;   // of every wavefront; by twos, the odd one out without anything to load
    const Pieces<DT, EVEN> x{static_cast<const uint8_t*>(A.x), (uint32_t)(A.tokens * A.hidden * kSize<DT>), A.hidden, A.tokens};
    raw16 even[M][U], odd[M][U];
    auto load = [&](int item, int s, raw16 (&to)[M][U]) {
        const int rank = item / A.columns, j0 = (item - rank * A.columns) * COLS;
        const int e = scalar(list[rank]);
#pragma unroll
        for (int m = 0; m < M; ++m) {
            const int j = j0 + m % NG * kMlpColumns, columns = A.inter - j < kMlpColumns ? A.inter - j < 0 ? 0 : A.inter - j : kMlpColumns;
            const Pieces<DT, EVEN> w{at<DT>(m < NG ? A.up : A.gate, ((int64_t)e * A.inter + (columns ? j : 0)) * A.hidden),
                                     (uint32_t)(columns * A.hidden * kSize<DT>), A.hidden, columns};
#pragma unroll
            for (int u = 0; u < U; ++u) to[m][u] = w.load(col, (s + u) * STEP + quarter * V, s + u < s1);
        }
    };
    const int items = count * A.columns;
    int item = (int)blockIdx.x, buffer = 0;
    if (item < items) load(item, s0, even);
    for (; item < items; item += (int)gridDim.x, buffer ^= 1) {
        mm_f32x4 acc[M];
#pragma unroll
        for (int m = 0; m < M; ++m) acc[m] = mm_f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        auto turn = [&](int t, const raw16 (&now)[M][U], raw16 (&next)[M][U]) {   // as k_mlp_down's
            const int s = s0 + t * U;
            raw16 xv[U];
#pragma unroll
            for (int u = 0; u < U; ++u) xv[u] = x.load(col, (s + u) * STEP + quarter * V, s + u < s1);
            __builtin_amdgcn_sched_barrier(0);
            const bool last = t + 1 >= turns && (t & 1);   // the next columns' first
            const int ahead = last ? item + (int)gridDim.x : item;
            if (ahead < items) load(ahead, last ? s0 : s + U, next);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int m = 0; m < M; ++m) {
                mm_f32x4 some = DT == DT_BF16 ? acc[m] : mm_f32x4{0.0f, 0.0f, 0.0f, 0.0f};   // FP32: short chains of sums
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    if constexpr (DT == DT_BF16) {
                        some = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(mm_bf16x8, now[m][u]), __builtin_bit_cast(mm_bf16x8, xv[u]),
                                                                       some, 0, 0, 0);
                    } else {
                        const mm_f32x4 wf = __builtin_bit_cast(mm_f32x4, now[m][u]), xf = __builtin_bit_cast(mm_f32x4, xv[u]);
#pragma unroll
                        for (int q = 0; q < 4; ++q) some = __builtin_amdgcn_mfma_f32_16x16x4f32(wf[q], xf[q], some, 0, 0, 0);
                    }
                }
                if constexpr (DT == DT_BF16) acc[m] = some;
                else acc[m] += some;
            }
        };
        for (int t = 0; t < turns; t += 2) {
            turn(t, even, odd);
            turn(t + 1, odd, even);
        }
        if (wave > 0)
#pragma unroll
            for (int m = 0; m < M; ++m) parts[buffer][wave - 1][m][lane] = acc[m];
        __syncthreads();   // and the first wavefront has read the other buffer
        if (wave > 0) continue;
        const int rank = item / A.columns, j0 = (item - rank * A.columns) * COLS, e = list[rank];
        const uint32_t tokens = mask[e];
        if (j0 == 0 && lane < kMlpTokens) {   // for the other kernel
            Chosen* const c = A.list + rank;
            float w = 0.0f;
            if (lane < A.tokens)
                for (int j = 0; j < A.top_k; ++j) w = expert[lane * A.top_k + j] == e ? weight[lane * A.top_k + j] : w;
            c->weight[lane] = w;
            if (lane == 0) {
                c->expert = e;
                c->tokens = tokens;
            }
        }
        if (!(tokens >> col & 1)) continue;
#pragma unroll
        for (int p = 0; p < W - 1; ++p)
#pragma unroll
            for (int m = 0; m < M; ++m) acc[m] += parts[buffer][p][m][lane];
        void* row = at<DT>(A.a, ((int64_t)rank * kMlpTokens + col) * A.inter);
#pragma unroll
        for (int n = 0; n < NG; ++n)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int j = j0 + n * kMlpColumns + 4 * quarter + r;
                const float y = GATE ? activated(acc[M - NG + n][r], A.silu) * acc[n][r] : activated(acc[n][r], A.silu);
                if (j < A.inter) put<DT>(row, j, y);
            }
    }
}

// COLS columns of the result: the wavefronts share the chosen experts' pieces of U loads, whose products are weighted and added in
// the order of the experts, then the wavefronts' parts in theirs.  Fewer than 16 columns leave rows of the matrix instruction for
// other terms of the same columns (G slices of 4 lanes' vectors each, multiplied one slice at a time; a product's other rows are not
// looked at): 2048 columns are 256 workgroups of 8, a CU each, where 128 of 16 reach 3.0 TB/s.
template <int DT, bool EVEN, int COLS>
__global__ __launch_bounds__(kDownWaves * kWave) void k_mlp_down(MlpArgs A)
{
    constexpr int V = kLane<DT>, STEP = 4 * V, W = kDownWaves, G = 16 / COLS, U = COLS == 4 ? 2 : 4, PIECE = U * G * STEP;
    __shared__ mm_f32x4 parts[W][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / kWave);
    const int col = lane & 15, quarter = lane >> 4;
    const int j0 = (int)block_index() * COLS, columns = A.hidden - j0 < COLS ? A.hidden - j0 : COLS;
    const int pieces = (A.inter + PIECE - 1) / PIECE, rank0 = wave / pieces;
    const int first = scalar(A.list[rank0 < A.used ? rank0 : 0].expert);   // asked for beside the count; not looked at behind it
    const int items = scalar(*A.count) * pieces;
    mm_f32x4 sum{0.0f, 0.0f, 0.0f, 0.0f};
    raw16 pieces_of[3][U];   // two ahead of the one that is multiplied
    auto load = [&](int i, int e, raw16 (&to)[U]) {
        const int rank = i / pieces, k0 = (i - rank * pieces) * PIECE + (col / COLS * 4 + quarter) * V;
        const Pieces<DT, EVEN> w{at<DT>(A.down, ((int64_t)e * A.hidden + j0) * A.inter), (uint32_t)(columns * A.inter * kSize<DT>), A.inter, columns};
#pragma unroll
        for (int u = 0; u < U; ++u) to[u] = w.load(col % COLS, k0 + u * G * STEP, true);
    };
    // loads arrive in their order: this piece's activations are asked for before a later piece's weights, which are then on their
    // way while this one is multiplied
    auto turn = [&](int i, const raw16 (&now)[U], raw16 (&ahead)[U]) {
        const int rank = i / pieces, k0 = (i - rank * pieces) * PIECE + quarter * V;
        const Chosen* const c = A.list + rank;
        const bool mine = c->tokens >> col & 1;
        const float by = c->weight[col];
        const Pieces<DT, EVEN> a{at<DT>(A.a, (int64_t)rank * kMlpTokens * A.inter), (uint32_t)(kMlpTokens * A.inter * kSize<DT>), A.inter, kMlpTokens};
        raw16 av[G][U];
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
            for (int u = 0; u < U; ++u) av[g][u] = a.load(col, k0 + (u * G + g) * STEP, mine);   // another token's row: never written
        __builtin_amdgcn_sched_barrier(0);
        if (i + 2 * W < items) load(i + 2 * W, scalar(A.list[(i + 2 * W) / pieces].expert), ahead);
        __builtin_amdgcn_sched_barrier(0);
        mm_f32x4 product{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int g = 0; g < G; ++g) {
            mm_f32x4 acc{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if constexpr (DT == DT_BF16) {
                    acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(mm_bf16x8, now[u]), __builtin_bit_cast(mm_bf16x8, av[g][u]), acc, 0, 0, 0);
                } else {
                    const mm_f32x4 wf = __builtin_bit_cast(mm_f32x4, now[u]), af = __builtin_bit_cast(mm_f32x4, av[g][u]);
#pragma unroll
                    for (int q = 0; q < 4; ++q) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(wf[q], af[q], acc, 0, 0, 0);
                }
            }
            const bool slice = 4 * quarter / COLS == g;   // whose rows this lane holds
#pragma unroll
            for (int r = 0; r < 4; ++r) product[r] = slice ? acc[r] : product[r];
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) sum[r] = mine ? sum[r] + by * product[r] : sum[r];   // what an expert holds stays with its tokens
    };
    if (wave < items) load(wave, first, pieces_of[0]);
    if (wave + W < items) load(wave + W, scalar(A.list[(wave + W) / pieces].expert), pieces_of[1]);
    for (int i = wave; i < items; i += 3 * W) {
        turn(i, pieces_of[0], pieces_of[2]);
        if (i + W < items) turn(i + W, pieces_of[1], pieces_of[0]);
        if (i + 2 * W < items) turn(i + 2 * W, pieces_of[2], pieces_of[1]);
    }
    parts[wave][lane] = sum;
    __syncthreads();
    if (threadIdx.x >= kMlpTokens * COLS) return;
    const int token = threadIdx.x / COLS, j = threadIdx.x % COLS;
    if (token >= A.tokens || j >= columns) return;
    float y = 0.0f;
#pragma unroll
    for (int p = 0; p < W; ++p)
#pragma unroll
        for (int g = 0; g < G; ++g) y += parts[p][(g * COLS + j) / 4 * 16 + token][(g * COLS + j) % 4];
    put<DT>(A.out, (int64_t)token * A.hidden + j0 + j, y);
}

// ------------------------------------------------------------------------------ launches

constexpr int64_t kMlpSize = (int64_t)1 << 22;

static int mlp_check(int32_t dtype, int64_t tokens, int64_t experts, int64_t top_k, int64_t inter, int64_t hidden)
{
    if (dtype != ADAMBRIDGE_DT_F32 && dtype != ADAMBRIDGE_DT_BF16) return ADAMBRIDGE_EMVDTYPE;
    if (tokens < 1 || tokens > kMlpTokens || experts < 1 || experts > kMlpExperts || top_k < 1 || top_k > kMlpChosen || top_k > experts ||
        inter < 1 || inter > kMlpSize || hidden < 1 || hidden > kMlpSize)
        return ADAMBRIDGE_EBADN;
    return 0;
}

// Scratch: how many experts are chosen, which, and their activations, at 256 bytes each.
static int64_t list_bytes(int64_t used) { return (used * (int64_t)sizeof(Chosen) + 255) / 256 * 256; }

template <int DT, bool EVEN, bool GATE, int NG>
static void launch_up(const MlpArgs& A, const dim3 grid)
{
    const dim3 block(kUpWaves * kWave);
    if (A.experts <= 64) hipLaunchKernelGGL((k_mlp_up<DT, EVEN, GATE, NG, 1>), grid, block, 0, t_stream, A);
    else if (A.experts <= 256) hipLaunchKernelGGL((k_mlp_up<DT, EVEN, GATE, NG, 4>), grid, block, 0, t_stream, A);
    else hipLaunchKernelGGL((k_mlp_up<DT, EVEN, GATE, NG, 16>), grid, block, 0, t_stream, A);
}

template <int DT, bool EVEN>
static void launch_up(const MlpArgs& A, const dim3 grid, int groups)
{
    if (A.gate) groups == 2 ? launch_up<DT, EVEN, true, 2>(A, grid) : launch_up<DT, EVEN, true, 1>(A, grid);
    else groups == 2 ? launch_up<DT, EVEN, false, 2>(A, grid) : launch_up<DT, EVEN, false, 1>(A, grid);
}

template <int DT, bool EVEN>
static void launch_down(const MlpArgs& A)
{
    // Columns of a workgroup: the fewest with which a CU has one workgroup of them and not two (us of both kernels, 4 / 8 / 16: 13
    // tokens, 2 of 8 experts of 8192, 1024 columns 64 / 74 / 103, 1536 121 / 100 / 127, 2048 133 / 114 / 138, 2560 184 / 178 / 160, 3500
    // 238 / 204 / 194; of 4096, 4096 columns 134 / 117 / 107, 8192 270 / 225 / 209; one token of 8 experts of 1536, 1536 columns 25.8 / 21.6 / 26.8.
    // FP32, 13 tokens of 4096: 1024 75 / 80 / 107, 1280 134 / 98 / 124, 2048 150 / 116 / 138, 2560 194 / 169 / 147, 4096 296 / 227 / 217, 6144 431 / 329 / 347)
    const dim3 block(kDownWaves * kWave);
    if (A.hidden <= 4 * kMlpCus) hipLaunchKernelGGL((k_mlp_down<DT, EVEN, 4>), block_grid((A.hidden + 3) / 4), block, 0, t_stream, A);
    else if (A.hidden <= 8 * kMlpCus) hipLaunchKernelGGL((k_mlp_down<DT, EVEN, 8>), block_grid((A.hidden + 7) / 8), block, 0, t_stream, A);
    else hipLaunchKernelGGL((k_mlp_down<DT, EVEN, 16>), block_grid((A.hidden + 15) / 16), block, 0, t_stream, A);
}

template <int DT>
static void launch_mlp(MlpArgs& A)
{
    const bool up_even = A.hidden % kLane<DT> == 0 && ((uintptr_t)A.x | (uintptr_t)A.up | (uintptr_t)A.gate) % 16 == 0;
    const bool down_even = A.inter % kLane<DT> == 0 && (uintptr_t)A.down % 16 == 0;
    // two groups of columns share the tokens' rows and the choice, where that leaves a CU four workgroups (us, one / two: 13 tokens of 8
    // gated experts 8192 x 2048 109 / 101; one token of 8 experts 1536 x 2048, which does not, 12.8 / 14.5)
    const int groups = (int64_t)A.used * ((A.inter + 31) / 32) >= 4 * kMlpCus ? 2 : 1;
    A.columns = (A.inter + groups * kMlpColumns - 1) / (groups * kMlpColumns);
    const dim3 grid((unsigned)std::min<int64_t>((int64_t)A.used * A.columns, 4 * kMlpCus));   // as many as the CUs hold
    if (up_even) launch_up<DT, true>(A, grid, groups);
    else launch_up<DT, false>(A, grid, groups);
    if (down_even) launch_down<DT, true>(A);
    else launch_down<DT, false>(A);
}

}  // namespace abh

using namespace abh;

extern "C" {

ADAMBRIDGE_API int64_t adambridge_expert_mlp_work(int32_t dtype, int64_t tokens, int64_t experts, int64_t top_k, int64_t inter, int64_t hidden)
{
    const int rc = mlp_check(dtype, tokens, experts, top_k, inter, hidden);
    if (rc) return rc;
    const int64_t used = std::min(tokens * top_k, experts);
    return 256 + list_bytes(used) + used * kMlpTokens * inter * (dtype == ADAMBRIDGE_DT_BF16 ? 2 : 4);
}

ADAMBRIDGE_API int adambridge_expert_mlp(const void* x, const void* logits, int32_t logits_dtype, const void* up, const void* gate, const void* down,
                                         int32_t dtype, int64_t tokens, int64_t experts, int64_t top_k, int64_t inter, int64_t hidden,
                                         int32_t activation, int32_t normalize, void* out, void* work)
{
    const int rc = mlp_check(dtype, tokens, experts, top_k, inter, hidden);
    if (rc) return rc;
    if (logits_dtype != ADAMBRIDGE_DT_F32 && logits_dtype != ADAMBRIDGE_DT_BF16) return ADAMBRIDGE_EMVDTYPE;
    if (activation != ADAMBRIDGE_GELU && activation != ADAMBRIDGE_SILU) return ADAMBRIDGE_EMVDTYPE;
    if (!x || !logits || !up || !down || !out || !work) return ADAMBRIDGE_ENULL;
    if ((uintptr_t)work % 16) return ADAMBRIDGE_EALIGN;
    const int64_t used = std::min(tokens * top_k, experts);
    MlpArgs A{};
    A.x = x;
    A.logits = logits;
    A.up = up;
    A.gate = gate;
    A.down = down;
    A.out = out;
    A.count = static_cast<int32_t*>(work);
    A.list = reinterpret_cast<Chosen*>(static_cast<uint8_t*>(work) + 256);
    A.a = static_cast<uint8_t*>(work) + 256 + list_bytes(used);
    A.tokens = (int32_t)tokens;
    A.used = (int32_t)used;
    A.experts = (int32_t)experts;
    A.top_k = (int32_t)top_k;
    A.inter = (int32_t)inter;
    A.hidden = (int32_t)hidden;
    A.logits_bf16 = logits_dtype == ADAMBRIDGE_DT_BF16;
    A.normalize = normalize;
    A.silu = activation == ADAMBRIDGE_SILU;
    if (dtype == ADAMBRIDGE_DT_BF16) launch_mlp<DT_BF16>(A);
    else launch_mlp<DT_F32>(A);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? 0 : hip_fail(e, "hipLaunchKernelGGL (expert MLP)");
}

}  // extern "C"
