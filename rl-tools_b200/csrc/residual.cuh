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

// Pairs of fp32 values: one instruction for both.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c){
    float2 d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(reinterpret_cast<unsigned long long&>(d))
        : "l"(reinterpret_cast<const unsigned long long&>(a)), "l"(reinterpret_cast<const unsigned long long&>(b)), "l"(reinterpret_cast<const unsigned long long&>(c)));
    return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b){
    float2 d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(reinterpret_cast<unsigned long long&>(d)) : "l"(reinterpret_cast<const unsigned long long&>(a)), "l"(reinterpret_cast<const unsigned long long&>(b)));
    return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b){
    float2 d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(reinterpret_cast<unsigned long long&>(d)) : "l"(reinterpret_cast<const unsigned long long&>(a)), "l"(reinterpret_cast<const unsigned long long&>(b)));
    return d;
}
__device__ __forceinline__ float2 both(float v){ return make_float2(v, v); }
__device__ __forceinline__ float across(float2 v){ return v.x + v.y; }

// Activations and their slopes: the framework's definitions and two more, with few instructions, since they run on every element that a product leaves (a tile of 128 x 256 over
// 1024 k takes the tensor core 8,200 cycles; with erff the activation alone took 9,000 of the multiprocessor's, this way about 3,000).
// The normal distribution: Phi(-|x|) = exp(-x^2 / 2) P(t), t = 1 / (1 + c z), z = |x| / sqrt 2, with P(t) = t (b1 + t (b2 + ... t b6)) in place of exp(z^2) erfc(z) / 2. P and c are the
// minimax fit of this form over 0 <= z <= 9.4, by linear programming on the relative error weighted by max(erfc(z), 1/30): off by 4e-7 of the value at 0, by at most 1.2e-5 of it
// in the tail, where the values themselves vanish, a three-hundredth of half a step of bfloat16 and a fortieth of float16's, whatever x is. (Nothing is subtracted from 1 for
// x < 0: it would leave nothing of the tail.) Two at a time (|x| is cut at 20, where the density has long been 0), each
// with a reciprocal of its own: one for both, of the product, takes 0.7% off 4096 x 1024 x 4096 and makes the last bit of a result depend on its neighbour, which behind the last of an
// odd number of rows is whatever a register holds.
struct NormalPair { float2 size, tail, density; };                       // |x| up to 20, -Phi(-|x|), exp(-x^2 / 2)
__device__ __forceinline__ NormalPair normal_pair(float2 x){
    NormalPair n;
    n.size = make_float2(fminf(fabsf(x.x), 20.0f), fminf(fabsf(x.y), 20.0f));
    const float2 d = fma2(n.size, both(0.42263395f * 0.70710678118654752f), both(1.0f));
    const float2 t = make_float2(__fdividef(1.0f, d.x), __fdividef(1.0f, d.y));
    const float2 e = mul2(mul2(x, x), both(-0.5f));
    n.density = make_float2(__expf(e.x), __expf(e.y));
    float2 p = fma2(t, both(0.0805534029f), both(-0.229271916f));
    p = fma2(t, p, both(0.0306924702f));
    p = fma2(t, p, both(-0.15041971f));
    p = fma2(t, p, both(-0.111817672f));
    n.tail = mul2(mul2(t, fma2(t, p, both(-0.119736333f))), n.density);
    return n;
}
__device__ __forceinline__ float2 gelu_pair(float2 x){                   // x Phi(x) = max(x, 0) - |x| Phi(-|x|)
    const NormalPair n = normal_pair(x);
    return fma2(n.size, n.tail, make_float2(fmaxf(x.x, 0.0f), fmaxf(x.y, 0.0f)));
}
__device__ __forceinline__ float2 gelu_slope_pair(float2 x){             // Phi(x) + x phi(x)
    const NormalPair n = normal_pair(x);
    const float2 rest = add2(n.tail, both(1.0f));
    return fma2(mul2(x, both(0.39894228040143268f)), n.density, make_float2(x.x < 0.0f ? -n.tail.x : rest.x, x.y < 0.0f ? -n.tail.y : rest.y));
}
__device__ __forceinline__ float fast_sigmoid(float x){ return __fdividef(1.0f, 1.0f + __expf(-x)); }      // exp(-x) = inf: 1 / inf = 0
template <int ACT> __device__ __forceinline__ float residual_activation(float x){
    if constexpr(ACT == B200RL_ACT_GELU) return gelu_pair(both(x)).x;
    else if constexpr(ACT == B200RL_ACT_SILU) return x * fast_sigmoid(x);
    else if constexpr(ACT == B200RL_ACT_SIGMOID) return fast_sigmoid(x);
    else return activation<ACT>(x);
}
template <int ACT> __device__ __forceinline__ float residual_d_activation(float x){
    if constexpr(ACT == B200RL_ACT_GELU)return gelu_slope_pair(both(x)).x;
    else if constexpr(ACT == B200RL_ACT_SILU){ const float s = fast_sigmoid(x); return s * fmaf(x, 1.0f - s, 1.0f); }
    else if constexpr(ACT == B200RL_ACT_SIGMOID){ const float s = fast_sigmoid(x); return s * (1.0f - s); }
    else return d_activation<ACT>(x);
}
// eight values in place; eight values times the slopes at eight places
template <int ACT> __device__ __forceinline__ void activate_pairs(float2 (&v)[4]){
#pragma unroll
    for(int c = 0; c < 4; c++){
        if constexpr(ACT == B200RL_ACT_GELU) v[c] = gelu_pair(v[c]);
        else v[c] = make_float2(residual_activation<ACT>(v[c].x), residual_activation<ACT>(v[c].y));
    }
}
template <int ACT> __device__ __forceinline__ void times_slope_pairs(float2 (&v)[4], const float (&at)[8]){
#pragma unroll
    for(int c = 0; c < 4; c++){
        const float2 x = make_float2(at[2 * c], at[2 * c + 1]);
        if constexpr(ACT == B200RL_ACT_GELU) v[c] = mul2(v[c], gelu_slope_pair(x));
        else v[c] = mul2(v[c], make_float2(residual_d_activation<ACT>(x.x), residual_d_activation<ACT>(x.y)));
    }
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
