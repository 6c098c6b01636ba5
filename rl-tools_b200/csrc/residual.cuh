// What the operators of residual networks share: their element types, accesses to rows at any alignment, and the activations that they take.
#pragma once
#include "common.cuh"
#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace b200rl {

inline bool valid_type(int t){ return t >= B200RL_TYPE_FLOAT32 && t <= B200RL_TYPE_FLOAT16; }
inline bool valid_16_bit_type(int t){ return t == B200RL_TYPE_BFLOAT16 || t == B200RL_TYPE_FLOAT16; }
inline bool valid_residual_activation(int a){ return a >= B200RL_ACT_IDENTITY && a <= B200RL_ACT_SILU; }
inline size_t type_bytes(int t){ return t == B200RL_TYPE_FLOAT32 ? 4 : 2; }

// the pitch of a matrix with one row is never used: whatever the caller passed, its rows count as following one another
inline long long row_pitch(int ld, int rows, int cols){ return rows > 1 ? ld : cols; }
inline bool valid_matrix(const void* p, int ld, int rows, int cols, size_t element){ return p && (rows <= 1 || ld >= cols) && reinterpret_cast<uintptr_t>(p) % element == 0; }
// every row of the matrix starts on a 16-byte boundary
inline bool rows_aligned(const void* p, long long pitch, size_t element){ return reinterpret_cast<uintptr_t>(p) % 16 == 0 && pitch * element % 16 == 0; }

__device__ __forceinline__ float to_float(float v){ return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v){ return __bfloat162float(v); }
__device__ __forceinline__ float to_float(__half v){ return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v){ return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v){ return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_float<__half>(float v){ return __float2half_rn(v); }

// N consecutive elements as fp32 (N * sizeof(T) == 16: one 16-byte access; N == 1: one element)
template <typename T, int N> __device__ __forceinline__ void load_elements(const T* p, float (&v)[N]){
    if constexpr(N == 1) v[0] = to_float(*p);
    else{
        static_assert(N * sizeof(T) == 16);
        union { uint4 raw; T e[N]; } u;
        u.raw = *reinterpret_cast<const uint4*>(p);
#pragma unroll
        for(int i = 0; i < N; i++) v[i] = to_float(u.e[i]);
    }
}
template <typename T, int N> __device__ __forceinline__ void store_elements(T* p, const float (&v)[N]){
    if constexpr(N == 1) *p = from_float<T>(v[0]);
    else{
        static_assert(N * sizeof(T) == 16);
        union { uint4 raw; T e[N]; } u;
#pragma unroll
        for(int i = 0; i < N; i++) u.e[i] = from_float<T>(v[i]);
        *reinterpret_cast<uint4*>(p) = u.raw;
    }
}

// Activations and their slopes: the framework's definitions and two more, with few instructions, since they run on every element that a product leaves (a tile of 128 x 256 over
// 1024 k takes the tensor core 8,200 cycles; 256 threads that spend 45 instructions an element on erff take 11,500). Errors stay below 1e-6, a thousandth of the rounding to 16 bits.
//   Phi(x): erfc by Abramowitz and Stegun, "Handbook of Mathematical Functions", 7.1.26: erfc(z) = t (a1 + t (a2 + ...)) exp(-z^2) within 1.5e-7, t = 1 / (1 + p z), z >= 0
struct NormalTail { float phi, density; };                               // Phi(x) and exp(-x^2 / 2)
__device__ __forceinline__ NormalTail normal_tail(float x){
    const float z = fabsf(x) * 0.70710678118654752f, t = __fdividef(1.0f, fmaf(0.3275911f, z, 1.0f)), density = __expf(-0.5f * x * x);
    const float tail = 0.5f * t * fmaf(t, fmaf(t, fmaf(t, fmaf(t, 1.061405429f, -1.453152027f), 1.421413741f), -0.284496736f), 0.254829592f) * density;
    return {x < 0.0f ? tail : 1.0f - tail, density};
}
__device__ __forceinline__ float fast_sigmoid(float x){ return __fdividef(1.0f, 1.0f + __expf(-x)); }      // exp(-x) = inf: 1 / inf = 0
template <int ACT> __device__ __forceinline__ float residual_activation(float x){
    if constexpr(ACT == B200RL_ACT_GELU) return x * normal_tail(x).phi;
    else if constexpr(ACT == B200RL_ACT_SILU) return x * fast_sigmoid(x);
    else if constexpr(ACT == B200RL_ACT_SIGMOID) return fast_sigmoid(x);
    else return activation<ACT>(x);
}
template <int ACT> __device__ __forceinline__ float residual_d_activation(float x){
    if constexpr(ACT == B200RL_ACT_GELU){ const NormalTail n = normal_tail(x); return fmaf(x * 0.39894228040143268f, n.density, n.phi); }
    else if constexpr(ACT == B200RL_ACT_SILU){ const float s = fast_sigmoid(x); return s * fmaf(x, 1.0f - s, 1.0f); }
    else if constexpr(ACT == B200RL_ACT_SIGMOID){ const float s = fast_sigmoid(x); return s * (1.0f - s); }
    else return d_activation<ACT>(x);
}
#define B200RL_DISPATCH_RESIDUAL_ACT(act, ...) \
    switch(act){ \
        case B200RL_ACT_GELU: { constexpr int ACT = B200RL_ACT_GELU; __VA_ARGS__; break; } \
        case B200RL_ACT_SILU: { constexpr int ACT = B200RL_ACT_SILU; __VA_ARGS__; break; } \
        default: B200RL_DISPATCH_ACT(act, __VA_ARGS__) \
    }
#define B200RL_DISPATCH_16_BIT_TYPE(type, ...) \
    if((type) == B200RL_TYPE_BFLOAT16){ using T = __nv_bfloat16; __VA_ARGS__; } else { using T = __half; __VA_ARGS__; }
#define B200RL_DISPATCH_TYPE(type, ...) \
    if((type) == B200RL_TYPE_FLOAT32){ using T = float; __VA_ARGS__; } else { B200RL_DISPATCH_16_BIT_TYPE(type, __VA_ARGS__) }

}  // namespace b200rl
