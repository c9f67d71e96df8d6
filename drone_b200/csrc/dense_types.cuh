// What the dense operators share: element types, activations, reads of several values at once.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

#include <type_traits>

namespace drone {

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
template <typename T> __device__ __forceinline__ T from_float(float x);
template <> __device__ __forceinline__ float from_float<float>(float x) { return x; }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <> __device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }

// N values side by side in memory (all or nothing: 1, 2, 4 ... of them) to floats and back, 16-bit ones in pairs: an instruction for two.
template <typename T, int N>
struct alignas(N * sizeof(T)) Values {
    T v[N];
    __device__ __forceinline__ void get(float *to) const {
#pragma unroll
        for (int i = 0; i < N; ++i) to[i] = to_float(v[i]);
    }
    __device__ __forceinline__ void set(const float *from) {
        if constexpr (sizeof(T) == 4 || N == 1) {
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = from_float<T>(from[i]);
        } else {
#pragma unroll
            for (int i = 0; i < N; i += 2) {
                unsigned pair;
                if constexpr (std::is_same_v<T, __half>) {
                    const __half2 p = __floats2half2_rn(from[i], from[i + 1]);
                    pair = reinterpret_cast<const unsigned &>(p);
                } else {
                    const __nv_bfloat162 p = __floats2bfloat162_rn(from[i], from[i + 1]);
                    pair = reinterpret_cast<const unsigned &>(p);
                }
                reinterpret_cast<unsigned *>(v)[i / 2] = pair;
            }
        }
    }
};

template <typename T> constexpr int kVector = 16 / sizeof(T);      // values in 16 bytes

// f(std::integral_constant) of an activation
template <typename F>
__host__ __device__ __forceinline__ void with_activation(int activation, const F &f) {
    switch (activation) {
        case DRONE_ACT_RELU: f(std::integral_constant<int, DRONE_ACT_RELU>()); break;
        case DRONE_ACT_GELU: f(std::integral_constant<int, DRONE_ACT_GELU>()); break;
        case DRONE_ACT_SILU: f(std::integral_constant<int, DRONE_ACT_SILU>()); break;
        default: f(std::integral_constant<int, DRONE_ACT_NONE>());
    }
}

__device__ __forceinline__ float exp2_fast(float x) {      // off by 2^-22 of the value
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float reciprocal_fast(float x) {      // one unit in the last place
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// 1 - Phi(|z|), of the normal distribution, and exp(-z^2 / 2), for results of 16 bits: their quotient as a polynomial in t = 1 / (1 + 0.2925 |z|), fitted by
// reweighted least squares to the smallest largest error, of 1.5e-7 absolutely where the tail is large and of 1e-4 relatively where it is small: it is off by 6.6e-8
// of 1 and by 4.4e-5 of the value at most, as far out as there is anything, where a bfloat16 result keeps 2^-8 of the value.  A dozen instructions
// where erff and expf take fifty.
__device__ __forceinline__ float normal_tail(float z, float *bell) {
    const float t = reciprocal_fast(fmaf(0.2925f, fabsf(z), 1.f));
    *bell = exp2_fast(z * -0.72134752f * z);
    return t * fmaf(t, fmaf(t, fmaf(t, fmaf(t, fmaf(t, -0.08615099f, 0.26702819f), -0.07182564f), 0.16864968f), 0.10471195f), 0.11758675f) * *bell;
}

// Phi(z) of the tail that normal_tail gives: the tail below 0, what it leaves of 1 above.
__device__ __forceinline__ float normal_part(float z, float tail) {
    float above;
    asm("set.ge.f32.f32 %0, %1, 0f00000000;" : "=f"(above) : "f"(z));      // 1 or 0
    return fabsf(above - tail);
}

// z -> activation(z) + added, and the activation's derivative, for values of type T.  A NaN stays one, also in the ReLU (max(NaN, 0) would be 0).  The
// last product and the addition are one instruction, in words: left to the compiler, they would be one on some ways out of a product and two on others.
template <typename T, int ACTIVATION>
__device__ __forceinline__ float activate(float z, float added) {
    if constexpr (ACTIVATION == DRONE_ACT_RELU) {
        return (z < 0.f ? 0.f : z) + added;
    } else if constexpr (ACTIVATION == DRONE_ACT_GELU) {
        if (sizeof(T) == 4) return fmaf(0.5f * z, 1.f + erff(z * 0.70710678f), added);
        float bell;
        const float tail = normal_tail(z, &bell);
        return fmaf(z, normal_part(z, tail), added);
    } else if constexpr (ACTIVATION == DRONE_ACT_SILU) {
        return sizeof(T) == 4 ? __fadd_rn(z / (1.f + expf(-z)), added) : fmaf(z, reciprocal_fast(1.f + exp2_fast(z * -1.44269504f)), added);
    } else {
        return z + added;
    }
}
template <typename T, int ACTIVATION>
__device__ __forceinline__ float activation_slope(float z) {
    if constexpr (ACTIVATION == DRONE_ACT_RELU) {
        return z > 0.f ? 1.f : 0.f;
    } else if constexpr (ACTIVATION == DRONE_ACT_GELU) {
        if (sizeof(T) == 4) return 0.5f * (1.f + erff(z * 0.70710678f)) + z * 0.39894228f * expf(-0.5f * z * z);
        float bell;
        const float tail = normal_tail(z, &bell);
        return fmaf(z * 0.39894228f, bell, normal_part(z, tail));
    } else if constexpr (ACTIVATION == DRONE_ACT_SILU) {
        const float p = sizeof(T) == 4 ? 1.f / (1.f + expf(-z)) : reciprocal_fast(1.f + exp2_fast(z * -1.44269504f));
        return p * (1.f + z * (1.f - p));
    } else {
        return 1.f;
    }
}

// Whether every row of such a matrix can be read 16 bytes at a time.
inline bool rows_on_16_bytes(const void *p, long long ld, int size) {
    return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && ld * size % 16 == 0;
}

inline int type_size(int type) { return type == DRONE_F32 ? 4 : 2; }

inline int device_sms(int *sms) {
    int dev = 0;
    DRONE_CUDA(cudaGetDevice(&dev));
    DRONE_CUDA(cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, dev));
    return DRONE_OK;
}

// f(tag) with the element type that `type` stands for as decltype(tag)::T
template <typename E> struct TypeTag { using T = E; };
template <typename F>
int with_type(int type, const F &f) {
    return type == DRONE_F32 ? f(TypeTag<float>()) : type == DRONE_BF16 ? f(TypeTag<__nv_bfloat16>()) : f(TypeTag<__half>());
}

}  // namespace drone

#define DRONE_TYPE_OK(type) ((type) == DRONE_F32 || (type) == DRONE_BF16 || (type) == DRONE_F16)
#define DRONE_ALIGNED(p, type) ((reinterpret_cast<uintptr_t>(p) & (drone::type_size(type) - 1)) == 0)
