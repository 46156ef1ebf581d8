// Element types of the token and training-memory kernels (embedding, 8-bit checkpoints,
// beam selection): 32-bit arithmetic on fp32, bf16 or fp16 storage.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math_constants.h>

#include "common.cuh"

namespace slg {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }

template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

// E = 16 / sizeof(T) elements that move in one 16-byte access
template <typename T>
union Vec16 {
    static constexpr int E = 16 / sizeof(T);
    uint4 u;
    T e[E];
    __device__ __forceinline__ Vec16() {}
};

inline bool aligned_to(const void* p, int64_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// Calls F.template operator()<T>() for an SLG_DT_* code; false when the code is unknown.
template <typename F>
inline bool for_dtype(int dtype, F&& f) {
    switch (dtype) {
        case SLG_DT_F32: f(float()); return true;
        case SLG_DT_BF16: f(__nv_bfloat16()); return true;
        case SLG_DT_F16: f(__half()); return true;
        default: return false;
    }
}

}  // namespace slg
