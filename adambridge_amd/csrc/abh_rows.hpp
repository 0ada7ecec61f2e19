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
__device__ __forceinline__ void store_vec(void* row, int64_t i, int64_t n, const float* x)
{
    if (i + kLane<DT> <= n) {
        store_raw<DT>(row, i, to_raw<DT>(x));
    } else {
#pragma unroll
        for (int k = 0; k < kLane<DT>; ++k)
            if (i + k < n) put<DT>(row, i + k, x[k]);
    }
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

__device__ __forceinline__ float wave_sum(float x)
{
#pragma unroll
    for (int d = 1; d < kWave; d *= 2) x += __shfl_xor(x, d);
    return x;
}

// Two sums over a workgroup of T lanes, for every lane, in an order of their own whatever the schedule.  `part` is
// 2 T / 64 floats of LDS; a workgroup of one wavefront uses none.
template <int T>
__device__ __forceinline__ void block_sum2(float& a, float& b, float* part)
{
    a = wave_sum(a);
    b = wave_sum(b);
    if constexpr (T > kWave) {
        __syncthreads();   // the sums before these have been read
        if ((threadIdx.x & (kWave - 1)) == 0) {
            part[threadIdx.x / kWave] = a;
            part[T / kWave + threadIdx.x / kWave] = b;
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

}  // namespace abh
