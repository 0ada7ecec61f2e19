// abh_rows.hpp -- what the kernels over rows of BF16 or FP32 values share: 16-byte accesses at any element's
// address, their FP32 forms, and sums over a wavefront.
#pragma once

#include <hip/hip_runtime.h>

#include <stdint.h>

#include "abh_device.hpp"

namespace abh {

constexpr int kWave = 64;

// Values of a 16-byte access.
template <int DT>
constexpr int kLane = DT == DT_BF16 ? 8 : 4;
template <int DT>
constexpr int kSize = DT == DT_BF16 ? 2 : 4;

// 16 bytes at any element's address: gfx950 takes global accesses of any alignment, at full width (a row of
// odd length starts anywhere; one cache line more now and then is what it costs).
template <int DT>
struct Vec16;
template <>
struct Vec16<DT_BF16> {
    typedef uint32_t type __attribute__((ext_vector_type(4), aligned(2)));
};
template <>
struct Vec16<DT_F32> {
    typedef uint32_t type __attribute__((ext_vector_type(4), aligned(4)));
};
typedef uint32_t raw16 __attribute__((ext_vector_type(4)));

template <int DT>
__device__ __forceinline__ const uint8_t* at(const void* base, int64_t i)
{
    return static_cast<const uint8_t*>(base) + i * kSize<DT>;
}
template <int DT>
__device__ __forceinline__ uint8_t* at(void* base, int64_t i)
{
    return static_cast<uint8_t*>(base) + i * kSize<DT>;
}

template <int DT>
__device__ __forceinline__ float get(const void* base, int64_t i)
{
    if constexpr (DT == DT_BF16) return bitsf((uint32_t)static_cast<const uint16_t*>(base)[i] << 16);
    else return static_cast<const float*>(base)[i];
}

template <int DT>
__device__ __forceinline__ void put(void* base, int64_t i, float x)
{
    if constexpr (DT == DT_BF16) static_cast<uint16_t*>(base)[i] = (uint16_t)bf16_rne(x);
    else static_cast<float*>(base)[i] = x;
}

template <int DT>
__device__ __forceinline__ void to_floats(const raw16 w, float* x)
{
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        if constexpr (DT == DT_BF16) {
            x[2 * k] = bitsf(u[k] << 16);
            x[2 * k + 1] = bitsf(u[k] & 0xffff0000u);
        } else {
            x[k] = bitsf(u[k]);
        }
    }
}

template <int DT>
__device__ __forceinline__ raw16 to_raw(const float* x)
{
    uint32_t u[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        if constexpr (DT == DT_BF16) u[k] = bf16x2_rne(x[2 * k], x[2 * k + 1]);
        else u[k] = fbits(x[k]);
    }
    return raw16{u[0], u[1], u[2], u[3]};
}

template <int DT>
__device__ __forceinline__ raw16 load_raw(const void* base, int64_t i)
{
    return *reinterpret_cast<const typename Vec16<DT>::type*>(at<DT>(base, i));
}
template <int DT>
__device__ __forceinline__ void store_raw(void* base, int64_t i, raw16 w)
{
    *reinterpret_cast<typename Vec16<DT>::type*>(at<DT>(base, i)) = w;
}
// For results that the kernel does not read again: not kept in the caches in place of what it reads (4096 x 2048 layer norm
// 9.8 -> 7.7 us, combine of 16384 x 4 rows of 2048 79 -> 51).
template <int DT>
__device__ __forceinline__ void stream_raw(void* base, int64_t i, raw16 w)
{
    __builtin_nontemporal_store(w, reinterpret_cast<typename Vec16<DT>::type*>(at<DT>(base, i)));
}

// Values i .. i + kLane - 1 of a row of n, zeros past its end.
template <int DT>
__device__ __forceinline__ void load_vec(const void* row, int64_t i, int64_t n, float* x)
{
    if (i + kLane<DT> <= n) {
        to_floats<DT>(load_raw<DT>(row, i), x);
    } else {
#pragma unroll
        for (int k = 0; k < kLane<DT>; ++k) x[k] = i + k < n ? get<DT>(row, i + k) : 0.0f;
    }
}

template <int DT>
__device__ __forceinline__ void stream_vec(void* row, int64_t i, int64_t n, const float* x)
{
    if (i + kLane<DT> <= n) {
        stream_raw<DT>(row, i, to_raw<DT>(x));
    } else {
#pragma unroll
        for (int k = 0; k < kLane<DT>; ++k)
            if (i + k < n) put<DT>(row, i + k, x[k]);
    }
}

// 16 bytes that are read once, of arrays that the caches do not hold anyway: not kept there (combine's gradient 113 -> 100 us, a
// norm's of 65536 x 4096 283 -> 269; arrays that may be in a cache are slower to read so).
template <int DT>
__device__ __forceinline__ raw16 once_raw(const void* base, int64_t i)
{
    return __builtin_nontemporal_load(reinterpret_cast<const typename Vec16<DT>::type*>(at<DT>(base, i)));
}

// The same as they lie in memory.
template <int DT, bool ONCE = false>
__device__ __forceinline__ raw16 load_vec_raw(const void* row, int64_t i, int64_t n)
{
    if (i + kLane<DT> <= n) return ONCE ? once_raw<DT>(row, i) : load_raw<DT>(row, i);
    float x[kLane<DT>];
    load_vec<DT>(row, i, n, x);
    return to_raw<DT>(x);   // exact
}

// 8 BF16 values moved d places down (0 .. 8), zeros after them.
__device__ __forceinline__ raw16 drop_bf16(const raw16 w, int d)
{
    uint64_t lo = (uint64_t)w.y << 32 | w.x, hi = (uint64_t)w.w << 32 | w.z;
    lo = d & 4 ? hi : lo;
    hi = d & 4 ? 0u : hi;
    const int bits = (d & 3) * 16;
    lo = lo >> bits | (hi << 1) << (63 - bits);
    hi >>= bits;
    return d & 8 ? raw16{0u, 0u, 0u, 0u} : raw16{(uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)hi, (uint32_t)(hi >> 32)};
}

// 4 FP32 values moved d places down (0 .. 4).
__device__ __forceinline__ raw16 drop_f32(raw16 w, int d)
{
    if (d & 2) w = raw16{w.z, w.w, 0u, 0u};
    if (d & 1) w = raw16{w.y, w.z, w.w, 0u};
    return d & 4 ? raw16{0u, 0u, 0u, 0u} : w;
}

template <int DT>
__device__ __forceinline__ raw16 drop_values(const raw16 w, int d)
{
    if constexpr (DT == DT_BF16) return drop_bf16(w, d);
    else return drop_f32(w, d);
}

// N values of WT at i .. of a row of n (N a lane's values of another type), `none` without a row.
template <int WT, int N>
__device__ __forceinline__ void load_like(const void* row, int64_t i, int64_t n, float none, float* x)
{
    if (!row) {
#pragma unroll
        for (int k = 0; k < N; ++k) x[k] = none;
    } else if (i + N <= n) {
        if constexpr (N >= kLane<WT>) {
#pragma unroll
            for (int k = 0; k < N; k += kLane<WT>) to_floats<WT>(load_raw<WT>(row, i + k), x + k);
        } else {
#pragma unroll
            for (int k = 0; k < N; ++k) x[k] = get<WT>(row, i + k);
        }
    } else {
#pragma unroll
        for (int k = 0; k < N; ++k) x[k] = i + k < n ? get<WT>(row, i + k) : 0.0f;
    }
}

// A value of another lane, chosen by a pattern of the data-parallel primitives (no LDS): the lanes paired are each
// other's, so that a sum over pairs is the same in both.
template <int PATTERN, class T>
__device__ __forceinline__ T paired(T x)
{
    const uint32_t u = __builtin_bit_cast(uint32_t, x);
    return __builtin_bit_cast(T, (uint32_t)__builtin_amdgcn_update_dpp((int)u, (int)u, PATTERN, 0xf, 0xf, false));
}

// op over groups of G (2 .. 64) neighbouring lanes, the same result in every lane of a group.
template <int G, class T, class Op>
__device__ __forceinline__ T group_reduce(T x, Op op)
{
    if constexpr (G >= 2) x = op(x, paired<0xb1>(x));    // lanes 1 0 3 2
    if constexpr (G >= 4) x = op(x, paired<0x4e>(x));    // 2 3 0 1
    if constexpr (G >= 8) x = op(x, paired<0x141>(x));   // 7 - i of 8
    if constexpr (G >= 16) x = op(x, paired<0x140>(x));  // 15 - i of 16
    if constexpr (G >= 32) {
        const uint32_t u = __builtin_bit_cast(uint32_t, x);
        const auto s = __builtin_amdgcn_permlane16_swap(u, u, false, false);   // even sixteens' and odd sixteens'
        x = op(__builtin_bit_cast(T, (uint32_t)s[0]), __builtin_bit_cast(T, (uint32_t)s[1]));
    }
    if constexpr (G >= 64) {
        const uint32_t u = __builtin_bit_cast(uint32_t, x);
        const auto s = __builtin_amdgcn_permlane32_swap(u, u, false, false);
        x = op(__builtin_bit_cast(T, (uint32_t)s[0]), __builtin_bit_cast(T, (uint32_t)s[1]));
    }
    return x;
}

template <int G>
__device__ __forceinline__ float group_sum(float x)
{
    return group_reduce<G>(x, [](float a, float b) { return a + b; });
}
// The other way: N values to a row of n of another type.
template <int WT, int N>
__device__ __forceinline__ void store_like(void* row, int64_t i, int64_t n, const float* x)
{
    if (i + N <= n && N >= kLane<WT>) {
#pragma unroll
        for (int k = 0; k < N; k += kLane<WT>) store_raw<WT>(row, i + k, to_raw<WT>(x + k));
    } else {
#pragma unroll
        for (int k = 0; k < N; ++k)
            if (i + k < n) put<WT>(row, i + k, x[k]);
    }
}

__device__ __forceinline__ float wave_sum(float x) { return group_sum<kWave>(x); }

// Two sums over T lanes of a workgroup whose lanes all take part (in groups of T, this one's number `lane` in its own), for
// each of them, in an order of its own whatever the schedule.  `part` is the group's 2 T / 64 floats of LDS, not
// those of the call before: two that take turns need one barrier a call.  A wavefront or less (T 8, 16, 32) uses none.
template <int T>
__device__ __forceinline__ void block_sum2(float& a, float& b, float* part, int lane)
{
    constexpr int G = T < kWave ? T : kWave;
    a = group_sum<G>(a);
    b = group_sum<G>(b);
    if constexpr (T > kWave) {
        if (lane % kWave == 0) {
            part[lane / kWave] = a;
            part[T / kWave + lane / kWave] = b;
        }
        __syncthreads();
        a = b = 0.0f;
#pragma unroll
        for (int w = 0; w < T / kWave; ++w) {
            a += part[w];
            b += part[T / kWave + w];
        }
    }
}

// A launch has fewer than 2^32 lanes along x: workgroups from kGridX on (a multiple of the XCDs) go along z, where the last of
// them may be more than there is work for.
constexpr int64_t kGridX = 1 << 21;   // of 1024 lanes at most

__device__ __forceinline__ int64_t block_index() { return (int64_t)blockIdx.z * kGridX + blockIdx.x; }

inline dim3 block_grid(int64_t blocks, int64_t y = 1)
{
    return blocks <= kGridX ? dim3((unsigned)blocks, (unsigned)y) : dim3((unsigned)kGridX, (unsigned)y, (unsigned)((blocks + kGridX - 1) / kGridX));
}

// Keeps a value in its register as it is: what is computed from it again later is computed again, not kept.
__device__ __forceinline__ void hold(raw16& w) { asm volatile("" : "+v"(w)); }

}  // namespace abh
