// Element types of the token and training-memory kernels (embedding, 8-bit checkpoints,
// beam selection): 32-bit arithmetic on fp32, bf16 or fp16 storage.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math_constants.h>

#include <type_traits>

#include "common.cuh"

namespace slg {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }

template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

// the E = 16 / sizeof(T) elements of one 16-byte access as fp32, in registers
template <typename T> struct Pack16 { static constexpr int E = 16 / sizeof(T); };

template <typename T>
__device__ __forceinline__ void unpack2(uint32_t w, float* x) {
    if constexpr (sizeof(T) == 4) x[0] = __uint_as_float(w);
    else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        x[0] = __uint_as_float(w << 16);
        x[1] = __uint_as_float(w & 0xffff0000u);
    } else {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
        x[0] = f.x;
        x[1] = f.y;
    }
}

template <typename T>
__device__ __forceinline__ void unpack16(const uint4& u, float* x) {
    constexpr int S = 4 / sizeof(T);
    unpack2<T>(u.x, x);
    unpack2<T>(u.y, x + S);
    unpack2<T>(u.z, x + 2 * S);
    unpack2<T>(u.w, x + 3 * S);
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(const float* x) {
    if constexpr (sizeof(T) == 4) return __float_as_uint(x[0]);
    else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(x[0], x[1]);
        return *reinterpret_cast<const uint32_t*>(&h);
    } else {
        const __half2 h = __floats2half2_rn(x[0], x[1]);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
}

template <typename T>
__device__ __forceinline__ uint4 pack16(const float* x) {
    constexpr int S = 4 / sizeof(T);
    return make_uint4(pack2<T>(x), pack2<T>(x + S), pack2<T>(x + 2 * S), pack2<T>(x + 3 * S));
}

inline bool aligned_to(const void* p, int64_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// Calls f with a value of the element type of an SLG_DT_* code; false when the code is unknown.
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
