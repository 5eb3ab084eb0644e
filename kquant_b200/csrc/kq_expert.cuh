// Pieces shared by the expert-layer kernels: the groups of rows behind the
// offsets, activations, 16-bit vector access, operand layout.
#pragma once
#include <cuda_bf16.h>
#include "kq_umma.cuh"

namespace kq {

constexpr int kMaxExperts = 1024;

// Word of the current device that a kernel sets when a bounded wait ran out.  It lies in host memory that the kernels can
// write, so that the next call sees it without waiting for the GPU: wait_error_flag gives it, wait_error_word does unless it is
// set (KQ_ERR_TIMEOUT; kq_wait_errors clears it).
int wait_error_flag(int** out);
int wait_error_word(int** out, const char* what);
__device__ __forceinline__ void report_wait_error(int* word) {
    *reinterpret_cast<volatile int*>(word) = 1;
    __threadfence_system();
}

// Rows offsets[e] .. offsets[e+1] belong to expert e.  The offsets live on the
// device, so every value is clamped into 0 .. rows before it is used as an
// index.  Without offsets all rows are expert 0's.
__device__ __forceinline__ void group_of(const int64_t* offsets, int e, int rows, int& lo, int& count) {
    if (!offsets) { lo = 0; count = rows; return; }
    const int64_t a = offsets[e], b = offsets[e + 1];
    const int64_t ca = a < 0 ? 0 : (a > rows ? rows : a);
    const int64_t cb = b < ca ? ca : (b > rows ? rows : b);
    lo = (int)ca;
    count = (int)(cb - ca);
}

// Whole block: lo[e], count[e], and cum[e] = row tiles of `tile` rows before expert e (cum[experts] = all).
__device__ __forceinline__ void scan_groups(const int64_t* offsets, int experts, int rows, int tile, int* lo, int* count,
                                            int* cum) {
    for (int e = threadIdx.x; e < experts; e += blockDim.x) group_of(offsets, e, rows, lo[e], count[e]);
    __syncthreads();
    if (threadIdx.x < 32) {
        int carry = 0;
        for (int base = 0; base < experts; base += 32) {
            const int e = base + threadIdx.x;
            int v = e < experts ? (count[e] + tile - 1) / tile : 0;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const int o = __shfl_up_sync(0xFFFFFFFFu, v, d);
                if ((int)threadIdx.x >= d) v += o;
            }
            if (e < experts) cum[e + 1] = carry + v;
            carry += __shfl_sync(0xFFFFFFFFu, v, 31);
        }
        if (threadIdx.x == 0) cum[0] = 0;
    }
    __syncthreads();
}

// Expert of row tile t (cum[e] <= t < cum[e+1]).
__device__ __forceinline__ int expert_of(const int* cum, int experts, int t) {
    int a = 0, b = experts - 1;
    while (a < b) {
        const int m = (a + b) >> 1;
        if (cum[m + 1] > t) b = m;
        else a = m + 1;
    }
    return a;
}

template <int ACT>
__device__ __forceinline__ float activate(float z) {
    if constexpr (ACT == KQ_ACT_RELU) return z < 0.f ? 0.f : z;      // NaN stays NaN
    else if constexpr (ACT == KQ_ACT_SILU) return __fdividef(z, 1.f + __expf(-z));
    else if constexpr (ACT == KQ_ACT_GELU) return 0.5f * z * (1.f + erff(z * 0.70710678118654752f));
    else return z;
}

template <int ACT>
__device__ __forceinline__ float slope(float z) {
    if constexpr (ACT == KQ_ACT_RELU) return z > 0.f ? 1.f : 0.f;
    else if constexpr (ACT == KQ_ACT_SILU) {
        const float p = __fdividef(1.f, 1.f + __expf(-z));
        return p * (1.f + z * (1.f - p));
    } else if constexpr (ACT == KQ_ACT_GELU) {
        return 0.5f * (1.f + erff(z * 0.70710678118654752f)) + z * __expf(-0.5f * z * z) * 0.39894228040143268f;
    } else return 1.f;
}

template <typename T> __device__ __forceinline__ float to_f(T v);
template <> __device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_f<__half>(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }

// What rounding v to T leaves out, itself rounded (nothing of what is not finite).
template <typename T>
__device__ __forceinline__ float left_out(float v) {
    const float r = v - to_f<T>(from_f<T>(v));
    return fabsf(r) <= 3.4e38f ? r : 0.f;
}

// 8 consecutive elements: one 16-byte access when `vec`, else the first `nv` one by one.
template <typename T>
__device__ __forceinline__ void load8(const T* p, bool vec, int nv, float (&f)[8]) {
    if (vec) {
        const uint4 q = *reinterpret_cast<const uint4*>(p);
        const T* h = reinterpret_cast<const T*>(&q);
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = to_f<T>(h[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = i < nv ? to_f<T>(p[i]) : 0.f;
    }
}

template <typename T>
__device__ __forceinline__ void store8(T* p, bool vec, int nv, const float (&f)[8]) {
    if (vec) {
        uint4 q;
        T* h = reinterpret_cast<T*>(&q);
#pragma unroll
        for (int i = 0; i < 8; ++i) h[i] = from_f<T>(f[i]);
        *reinterpret_cast<uint4*>(p) = q;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < nv) p[i] = from_f<T>(f[i]);
    }
}

}  // namespace kq
