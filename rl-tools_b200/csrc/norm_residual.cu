// The norms around a block of a residual network, fused with the block's gate and residual scale:
//   u = post(branch), out = residual + scale gate u, normed = pre(out)
// and its gradients. Memory-bound: forward reads branch and residual and writes out and normed, backward reads out, d_normed, d_out and branch and writes
// d_residual and d_branch, each once. A row is held in the registers of 32 to 1,024 threads as fp32, so the two passes of a variance (mean, then squared deviations)
// cost no second read. The statistics are not stored for the backward pass: it holds the rows in registers anyway and computes them again.
// Measured, 16384 x 4096 bfloat16, calls in a graph: root-mean-square norms on both sides, forward 89 us without a gate, 90 with one per channel (5.9 TB/s), 102 with one per element;
// gradients 143, 161 and 200 us (5.6, 5.0 and 5.3 TB/s; 537 and 805 MB cannot be avoided, a gate per element is 134 and 268 more). Layer norms with biases and a gate per channel 122 and 347.
// The forward pass is bound by memory; the gradients by issue (half of all cycles, eight or sixteen warps resident that meet three times a row), with biases and a gate by the shared
// memory that holds seven values a column too. One row of 4096: 2.6 and 6.6 us, the launches and a chain of barriers. Before rows were fetched ahead and parameters kept in
// shared memory: 154 and 404 us.
#include "residual.cuh"
#include <atomic>
#include <type_traits>

namespace b200rl {

namespace {
constexpr int ROW_THREADS_MAX = 512, ELEMENTS_MAX = 16;      // 512 x 16 = B200RL_NORM_MAX_DIM
static_assert(ROW_THREADS_MAX * ELEMENTS_MAX == B200RL_NORM_MAX_DIM);
constexpr int SUMS = 4;                                      // parameter gradients: post weight, post bias, pre weight, pre bias
}

// Threads and elements per thread that hold a row of T: up to 16 elements a thread, 8 of fp32, so that the raw row that is under way takes the same registers either way.
template <int TPR, int E> struct Shape { static constexpr int tpr = TPR, e = E; };
template <typename T, typename F>
static int dispatch_row(int dim, F f){
    if(dim <= 256) return f(Shape<32, 8>{});
    if constexpr(sizeof(T) == 2){
        if(dim <= 512) return f(Shape<32, 16>{});
        if(dim <= 1024) return f(Shape<128, 8>{});
        if(dim <= 2048) return f(Shape<128, 16>{});
        return dim <= 4096 ? f(Shape<256, 16>{}) : f(Shape<512, 16>{});
    }
    else{
        if(dim <= 1024) return f(Shape<128, 8>{});
        if(dim <= 2048) return f(Shape<256, 8>{});
        return dim <= 4096 ? f(Shape<512, 8>{}) : f(Shape<1024, 8>{});
    }
}
// CTAs of the backward pass on a multiprocessor that leave a thread 64 to 168 registers
template <typename T> constexpr int backward_ctas(int tpr, int e){
    const bool narrow = sizeof(T) == 2;
    return tpr == 32 ? (narrow && e == 8 ? 5 : 3) : tpr == 128 ? (narrow && e == 8 ? 5 : 4) : tpr == 256 ? 2 : 1;
}

struct NormForward {
    const void* branch; long long ldb;
    const void* gate; long long ldg; int gate_rows;
    const void* residual; long long ldr;
    void* out; long long ldo;
    void* normed; long long ldn;
    const float *post_weight, *post_bias, *pre_weight, *pre_bias;
    int post, pre, rows, dim;
    float scale, epsilon;
};

struct NormBackward {
    const void* branch; long long ldb;
    const void* gate; long long ldg; int gate_rows;
    const void* out; long long ldo;
    const void* d_out; long long lddo;
    const void* d_normed; long long lddn;
    void* d_branch; long long lddb;
    void* d_residual; long long lddr;
    void* d_gate; long long lddg;
    const float *post_weight, *post_bias, *pre_weight;
    float* d_params[SUMS];                                   // post weight, post bias, pre weight, pre bias (NULL: not asked for)
    float* partials;                                         // [SUMS][workers][dim]
    float* pieces;                                           // [workers][2][dim]: gate rows whose rows lie with more than one worker
    int sums[SUMS], n_sums;                                  // those of d_params that are there
    int post, pre, rows, dim, workers, rows_per_worker, accumulate;
    float scale, epsilon;
};

// Sums of N values over the threads of a row (one warp, or the whole CTA); every thread gets them. Within a warp the lanes share the values out first: each exchange halves what a
// lane carries, so four values take six exchanges instead of twenty. `buffer` is used in turns, so one barrier per call is enough.
template <int TPR, int N>
__device__ __forceinline__ void row_sums(float (&v)[N], float (*buffer)[4][TPR / 32], int& turn){
    static_assert(N == 1 || N == 2 || N == 4);
    const int lane = threadIdx.x & 31;
    float mine = v[0];                                       // of value lane / (32 / N)
    if constexpr(N == 4){
        const bool upper = lane & 16, odd = lane & 8;
        float a = upper ? v[2] : v[0], b = upper ? v[3] : v[1];
        a += __shfl_xor_sync(0xffffffffu, upper ? v[0] : v[2], 16);
        b += __shfl_xor_sync(0xffffffffu, upper ? v[1] : v[3], 16);
        mine = odd ? b : a;
        mine += __shfl_xor_sync(0xffffffffu, odd ? a : b, 8);
    }
    if constexpr(N == 2){
        const bool upper = lane & 16;
        mine = upper ? v[1] : v[0];
        mine += __shfl_xor_sync(0xffffffffu, upper ? v[0] : v[1], 16);
    }
#pragma unroll
    for(int o = 16 / N; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
    if constexpr(TPR == 32){
#pragma unroll
        for(int i = 0; i < N; i++) v[i] = __shfl_sync(0xffffffffu, mine, i * (32 / N));
    }
    else{
        float (&shared)[4][TPR / 32] = buffer[turn];
        turn ^= 1;
        const int warp = threadIdx.x >> 5;
        if((lane & (32 / N - 1)) == 0) shared[lane / (32 / N)][warp] = mine;
        __syncthreads();
#pragma unroll
        for(int i = 0; i < N; i++){
            float4 part[TPR / 128];
#pragma unroll
            for(int w = 0; w < TPR / 128; w++) part[w] = *reinterpret_cast<const float4*>(&shared[i][4 * w]);
            v[i] = 0.0f;
#pragma unroll
            for(int w = 0; w < TPR / 128; w++) v[i] += (part[w].x + part[w].y) + (part[w].z + part[w].w);
        }
    }
}
// The row's first element, which lies in v[0] of its first thread (N rows at once). A call of row_sums has to follow before the next one.
template <int TPR, int N>
__device__ __forceinline__ void row_first(float (&v)[N]){
    if constexpr(TPR == 32){
#pragma unroll
        for(int i = 0; i < N; i++) v[i] = __shfl_sync(0xffffffffu, v[i], 0);
    }
    else{
        __shared__ float first[N];
        if(threadIdx.x == 0)
#pragma unroll
            for(int i = 0; i < N; i++) first[i] = v[i];
        __syncthreads();
#pragma unroll
        for(int i = 0; i < N; i++) v[i] = first[i];
    }
}

// The row's elements of one thread: vectors of VEC, TPR VEC apart. What lies behind the row's end reads as 0 (parameters: `fill`).
template <typename T, int VEC, int TPR, int E>
struct Row {
    struct Raw { T e[E]; };
    int lane, dim;
    __device__ __forceinline__ int column(int i) const { return (i * TPR + lane) * VEC; }
    __device__ __forceinline__ bool inside(int e) const { return column(e / VEC) < dim; }
    __device__ __forceinline__ void fetch(const void* base, long long at, Raw& raw) const {
        const T* row = static_cast<const T*>(base) + at;
#pragma unroll
        for(int i = 0; i < E / VEC; i++){
            if constexpr(VEC > 1){
                uint4 v = make_uint4(0, 0, 0, 0);
                if(column(i) < dim) v = *reinterpret_cast<const uint4*>(row + column(i));
                *reinterpret_cast<uint4*>(&raw.e[i * VEC]) = v;
            }
            else raw.e[i] = column(i) < dim ? row[column(i)] : from_float<T>(0.0f);
        }
    }
    __device__ __forceinline__ void pairs(const Raw& raw, float2 (&v)[E / 2]) const {
#pragma unroll
        for(int i = 0; i < E / 2; i++) v[i] = make_float2(to_float(raw.e[2 * i]), to_float(raw.e[2 * i + 1]));
    }
    __device__ __forceinline__ void clear_outside(float2 (&v)[E / 2]) const {
#pragma unroll
        for(int i = 0; i < E / 2; i++){ if(!inside(2 * i)) v[i].x = 0.0f; if(!inside(2 * i + 1)) v[i].y = 0.0f; }
    }
    __device__ __forceinline__ void store_sums(float* p, const float (&v)[E]) const {
#pragma unroll
        for(int e = 0; e < E; e += VEC > 1 ? 4 : 1)
            if(inside(e)){
                float* at = p + column(e / VEC) + e % VEC;
                if constexpr(VEC > 1) *reinterpret_cast<float4*>(at) = make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]);
                else *at = v[e];
            }
    }
    __device__ __forceinline__ void store(void* base, long long at, const float2 (&v)[E / 2]) const {
        float f[E];
#pragma unroll
        for(int i = 0; i < E / 2; i++){ f[2 * i] = v[i].x; f[2 * i + 1] = v[i].y; }
        store(base, at, f);
    }
    __device__ __forceinline__ void store(void* base, long long at, const float (&v)[E]) const {
        T* row = static_cast<T*>(base) + at;
#pragma unroll
        for(int i = 0; i < E / VEC; i++){
            float e[VEC];
#pragma unroll
            for(int j = 0; j < VEC; j++) e[j] = v[i * VEC + j];
            if(column(i) < dim) store_elements(row + column(i), e);
        }
    }
    // ordinary loads: read-only ones could be moved in front of the wait for the kernel before, which may be the optimizer step that writes these parameters
    __device__ __forceinline__ void parameters(const float* p, float fill, float (&v)[E]) const {
        if(VEC > 1 && reinterpret_cast<uintptr_t>(p) % 16 == 0){
#pragma unroll
            for(int e = 0; e < E; e += 4){
                float4 q = make_float4(fill, fill, fill, fill);
                if(p && inside(e)) q = *reinterpret_cast<const float4*>(p + column(e / VEC) + e % VEC);
                v[e] = q.x; v[e + 1] = q.y; v[e + 2] = q.z; v[e + 3] = q.w;
            }
        }
        else
#pragma unroll
            for(int e = 0; e < E; e++) v[e] = p && inside(e) ? p[column(e / VEC) + e % VEC] : fill;
    }
};

// v <- (v - mean) rstd in place (0 behind the row's end); returns rstd. The mean is summed about the row's first element: a constant row has variance 0 whatever its value,
// and the error of the mean goes by the row's spread.
template <int TPR, typename R, int P>
__device__ __forceinline__ void normalise(const R& row, int kind, float2 (&v)[P], float epsilon, float (*buffer)[4][TPR / 32], int& turn){
    const float inv = 1.0f / (float)row.dim;
    if(kind == B200RL_NORM_LAYER){
        float first[1] = {v[0].x}, s[1] = {0.0f};
        row_first<TPR>(first);
#pragma unroll
        for(int i = 0; i < P; i++) v[i] = add2(v[i], both(-first[0]));
        row.clear_outside(v);
#pragma unroll
        for(int i = 0; i < P; i++) s[0] += across(v[i]);
        row_sums<TPR>(s, buffer, turn);
        const float mean = s[0] * inv;
#pragma unroll
        for(int i = 0; i < P; i++) v[i] = add2(v[i], both(-mean));
        row.clear_outside(v);
    }
    float2 squares = both(0.0f);
#pragma unroll
    for(int i = 0; i < P; i++) squares = fma2(v[i], v[i], squares);
    float s[1] = {across(squares)};
    row_sums<TPR>(s, buffer, turn);
    const float rstd = rsqrtf(s[0] * inv + epsilon);
#pragma unroll
    for(int i = 0; i < P; i++) v[i] = mul2(v[i], both(rstd));
}

// A CTA (or a warp, for short rows) takes every so many-th row. What a thread keeps over its rows, its columns' parameters, lies in shared memory at places of its own; the next
// row's loads are under way while a row is summed.
template <typename T, int VEC, int TPR, int E>
__global__ void __launch_bounds__(TPR < 128 ? 128 : TPR) norm_forward_kernel(NormForward a){
    constexpr int ROWS = TPR < 128 ? 128 / TPR : 1, P = E / 2;
    using R = Row<T, VEC, TPR, E>;
    extern __shared__ __align__(16) float4 kept_memory[];                // [parameters that are there][ROWS][E / 4][TPR]
    __shared__ __align__(16) float buffer[2][4][TPR / 32];
    after_predecessor();
    int turn = 0;
    const R row{(int)(threadIdx.x % TPR), a.dim};
    const float* const parameters[4] = {a.post_weight, a.post_bias, a.pre_weight, a.pre_bias};
    int place[4], n = 0;
#pragma unroll
    for(int k = 0; k < 4; k++) if(parameters[k]) place[k] = n++; else place[k] = -1;
    auto kept = [&](int k, int i) -> float4& { return kept_memory[((place[k] * ROWS + threadIdx.x / TPR) * (E / 4) + i) * TPR + threadIdx.x % TPR]; };
    {
        float p[4][E];                                                   // all loads under way before the first is put away
#pragma unroll
        for(int k = 0; k < 4; k++) if(parameters[k]) row.parameters(parameters[k], 0.0f, p[k]);
#pragma unroll
        for(int k = 0; k < 4; k++)
            if(parameters[k])
#pragma unroll
                for(int i = 0; i < E / 4; i++) kept(k, i) = make_float4(p[k][4 * i], p[k][4 * i + 1], p[k][4 * i + 2], p[k][4 * i + 3]);
    }
    auto affine = [&](float2 (&v)[P], int weight, int bias){
        if(parameters[weight])
#pragma unroll
            for(int i = 0; i < E / 4; i++){
                const float4 w = kept(weight, i);
                v[2 * i] = mul2(v[2 * i], make_float2(w.x, w.y)); v[2 * i + 1] = mul2(v[2 * i + 1], make_float2(w.z, w.w));
            }
        if(parameters[bias])
#pragma unroll
            for(int i = 0; i < E / 4; i++){
                const float4 w = kept(bias, i);
                v[2 * i] = add2(v[2 * i], make_float2(w.x, w.y)); v[2 * i + 1] = add2(v[2 * i + 1], make_float2(w.z, w.w));
            }
    };
    typename R::Raw raw_r{}, raw_u{}, raw_gate{};                        // 0 where there is no such operand
    long long gate_row = -1;
    auto fetch = [&](long long r){
        if(a.branch) row.fetch(a.branch, r * a.ldb, raw_u);
        if(a.residual) row.fetch(a.residual, r * a.ldr, raw_r);
        if(a.gate){
            const long long g = a.gate_rows >= a.rows ? 0 : a.gate_rows == 1 ? r : (long long)((uint32_t)r / (uint32_t)a.gate_rows);
            if(g != gate_row) row.fetch(a.gate, g * a.ldg, raw_gate);
            gate_row = g;
        }
    };
    constexpr bool AHEAD = VEC > 1;
    const long long step = (long long)gridDim.x * ROWS;
    long long r = (long long)blockIdx.x * ROWS + threadIdx.x / TPR;
    if(AHEAD && r < a.rows) fetch(r);
    for(; r < a.rows; r += step){
        if(!AHEAD) fetch(r);
        float2 o[P];
        row.pairs(raw_r, o);
        if(a.branch){
            float2 u[P], gate[P];
            row.pairs(raw_u, u);
            if(a.gate) row.pairs(raw_gate, gate);
            if(AHEAD && r + step < a.rows) fetch(r + step);
            if(a.post != B200RL_NORM_NONE){
                normalise<TPR>(row, a.post, u, a.epsilon, buffer, turn);
                affine(u, 0, 1);
            }
            if(a.gate)
#pragma unroll
                for(int i = 0; i < P; i++) u[i] = mul2(u[i], gate[i]);
#pragma unroll
            for(int i = 0; i < P; i++) o[i] = fma2(both(a.scale), u[i], o[i]);
        }
        else if(AHEAD && r + step < a.rows) fetch(r + step);
        if(a.out) row.store(a.out, r * a.ldo, o);
        if(a.pre != B200RL_NORM_NONE){
            normalise<TPR>(row, a.pre, o, a.epsilon, buffer, turn);
            affine(o, 2, 3);
            row.store(a.normed, r * a.ldn, o);
        }
    }
}

// ---- backward -----------------------------------------------------------------------------------------------------------------------------------------
// A worker (the threads of a row) takes rows_per_worker consecutive rows. What a thread keeps over its rows -- its columns' parameters and the sums of their gradients -- lies
// in shared memory at places of its own (registers for it would leave one CTA per multiprocessor); the next row's loads are under way while a row is summed. BIAS: sums for the
// biases too, and the post norm's bias, which the gate's gradient sees.
template <int TPR, int E, bool BIAS, bool GATE> struct Kept {
    enum { PRE_WEIGHT, POST_WEIGHT, SUM_POST_WEIGHT, SUM_PRE_WEIGHT, SUM_POST_BIAS, SUM_PRE_BIAS = SUM_POST_BIAS + (BIAS ? 1 : 0), SUM_GATE = SUM_PRE_BIAS + (BIAS ? 1 : 0),
           COUNT = SUM_GATE + (GATE ? 1 : 0) };
    static constexpr int worker_bytes = COUNT * E * TPR * 4;
    static_assert(worker_bytes + 1024 <= 232448, "rows of B200RL_NORM_MAX_DIM elements fit");
    float4* mine;                                            // [COUNT][E / 4][TPR]
    __device__ __forceinline__ float4& at(int array, int quad){ return mine[(array * (E / 4) + quad) * TPR]; }
};
// CTAs that are resident at once, their shared memory counted too: what they keep, the exchanges' buffers, 1 KB that each costs besides. Only 16-bit rows of 1025 to 2048 elements with
// biases and a gate are held to fewer by it (three instead of four: 16384 x 2048 with a gate per channel 129 us, planned and compiled for four 209).
template <typename T, int TPR, int E, bool BIAS, bool GATE> constexpr int backward_resident(){
    constexpr int bytes = (TPR < 128 ? 128 / TPR : 1) * Kept<TPR, E, BIAS, GATE>::worker_bytes + 2 * 4 * (TPR / 32) * 4 + 16 + 1024, fit = 228 * 1024 / bytes;
    static_assert(fit >= 1);
    return fit < backward_ctas<T>(TPR, E) ? fit : backward_ctas<T>(TPR, E);
}
template <typename T, int VEC, int TPR, int E, bool BIAS, bool GATE>
__global__ void __launch_bounds__(TPR < 128 ? 128 : TPR, backward_resident<T, TPR, E, BIAS, GATE>()) norm_backward_kernel(NormBackward a){
    constexpr int WORKERS = TPR < 128 ? 128 / TPR : 1, P = E / 2;
    using R = Row<T, VEC, TPR, E>;
    using K = Kept<TPR, E, BIAS, GATE>;
    extern __shared__ __align__(16) float4 kept_memory[];
    __shared__ __align__(16) float buffer[2][4][TPR / 32];
    after_predecessor();
    int turn = 0;
    const int worker = blockIdx.x * WORKERS + threadIdx.x / TPR;
    const long long first = (long long)worker * a.rows_per_worker, last = min((long long)a.rows, first + a.rows_per_worker);
    if(first >= last) return;                                // a whole row's threads leave together
    const R row{(int)(threadIdx.x % TPR), a.dim};
    K kept{kept_memory + (threadIdx.x / TPR) * (K::worker_bytes / 16) + threadIdx.x % TPR};
    const bool gated = GATE && a.gate;                       // the form for rows at odd addresses is built once, with everything in it
    const bool pre = a.pre != B200RL_NORM_NONE, post = a.post != B200RL_NORM_NONE, layer = a.pre == B200RL_NORM_LAYER || a.post == B200RL_NORM_LAYER;
    const float inv = 1.0f / (float)a.dim;
    {
        float p[E];
        auto keep = [&](int array){
#pragma unroll
            for(int i = 0; i < E / 4; i++) kept.at(array, i) = make_float4(p[4 * i], p[4 * i + 1], p[4 * i + 2], p[4 * i + 3]);
        };
        row.parameters(a.pre_weight, 1.0f, p);
        keep(K::PRE_WEIGHT);
        row.parameters(a.post_weight, 1.0f, p);
        keep(K::POST_WEIGHT);
#pragma unroll
        for(int e = 0; e < E; e++) p[e] = 0.0f;
        keep(K::SUM_POST_WEIGHT);
        keep(K::SUM_PRE_WEIGHT);
        if constexpr(BIAS){ keep(K::SUM_POST_BIAS); keep(K::SUM_PRE_BIAS); }
        if constexpr(GATE) keep(K::SUM_GATE);
    }
    // array += a b for the pairs 2 i, 2 i + 1
    auto add_to = [&](int array, int i, float2 a0, float2 b0, float2 a1, float2 b1){
        float4 v = kept.at(array, i);
        const float2 lo = fma2(a0, b0, make_float2(v.x, v.y)), hi = fma2(a1, b1, make_float2(v.z, v.w));
        kept.at(array, i) = make_float4(lo.x, lo.y, hi.x, hi.y);
    };
    auto hand_out = [&](int array, float (&v)[E]){
#pragma unroll
        for(int i = 0; i < E / 4; i++){ const float4 q = kept.at(array, i); v[4 * i] = q.x; v[4 * i + 1] = q.y; v[4 * i + 2] = q.z; v[4 * i + 3] = q.w; }
    };
    long long group = 0, group_begin = 0, group_end = 0;     // rows that share a gate row
    if(gated){
        group = first / a.gate_rows;
        group_begin = group * a.gate_rows;
        group_end = min((long long)a.rows, group_begin + a.gate_rows);
    }
    typename R::Raw raw_d{}, raw_u{}, raw_q{}, raw_x{}, raw_gate{};      // 0 where there is no such operand
    auto fetch = [&](long long r){
        if(a.d_out) row.fetch(a.d_out, r * a.lddo, raw_d);
        if(a.branch) row.fetch(a.branch, r * a.ldb, raw_u);
        if(pre){ row.fetch(a.d_normed, r * a.lddn, raw_q); row.fetch(a.out, r * a.ldo, raw_x); }
    };
    constexpr bool AHEAD = VEC > 1 || sizeof(T) == 4;        // single 16-bit elements would take a register each
    if(gated) row.fetch(a.gate, group * a.ldg, raw_gate);
    if(AHEAD) fetch(first);
    for(long long r = first; r < last; r++){
        float2 d[P], u[P], x[P], q[P];
        if(!AHEAD) fetch(r);
        row.pairs(raw_d, d); row.pairs(raw_u, u); row.pairs(raw_x, x); row.pairs(raw_q, q);
        if(AHEAD && r + 1 < last) fetch(r + 1);
        // the statistics of both norms with the same barriers: means about the first elements, then squares
        if(layer){
            float start[2] = {x[0].x, u[0].x}, s[2] = {0.0f, 0.0f};
            row_first<TPR>(start);
            if(a.pre != B200RL_NORM_LAYER) start[0] = 0.0f;
            if(a.post != B200RL_NORM_LAYER) start[1] = 0.0f;
#pragma unroll
            for(int i = 0; i < P; i++){ x[i] = add2(x[i], both(-start[0])); u[i] = add2(u[i], both(-start[1])); }
            row.clear_outside(x); row.clear_outside(u);
#pragma unroll
            for(int i = 0; i < P; i++){ s[0] += across(x[i]); s[1] += across(u[i]); }
            row_sums<TPR>(s, buffer, turn);
            const float mean_x = a.pre == B200RL_NORM_LAYER ? s[0] * inv : 0.0f, mean_u = a.post == B200RL_NORM_LAYER ? s[1] * inv : 0.0f;
#pragma unroll
            for(int i = 0; i < P; i++){ x[i] = add2(x[i], both(-mean_x)); u[i] = add2(u[i], both(-mean_u)); }
            row.clear_outside(x); row.clear_outside(u);
        }
        float rstd_u = 1.0f;
        {
            // squares of both rows; the sums of the pre norm's gradient g = q weight go with them: sum g hat = rstd sum g x
            float2 xx = both(0.0f), uu = xx, gg = xx, gx = xx;
#pragma unroll
            for(int i = 0; i < E / 4; i++){
                const float4 w = kept.at(K::PRE_WEIGHT, i);
                const float2 g0 = mul2(q[2 * i], make_float2(w.x, w.y)), g1 = mul2(q[2 * i + 1], make_float2(w.z, w.w));
                xx = fma2(x[2 * i], x[2 * i], xx); xx = fma2(x[2 * i + 1], x[2 * i + 1], xx);
                uu = fma2(u[2 * i], u[2 * i], uu); uu = fma2(u[2 * i + 1], u[2 * i + 1], uu);
                gg = add2(gg, add2(g0, g1));
                gx = fma2(g0, x[2 * i], gx); gx = fma2(g1, x[2 * i + 1], gx);
            }
            float s[4] = {across(xx), across(uu), across(gg), across(gx)};
            row_sums<TPR>(s, buffer, turn);
            if(pre){
                const float rstd = rsqrtf(s[0] * inv + a.epsilon), mean = a.pre == B200RL_NORM_LAYER ? s[2] * inv : 0.0f, along = s[3] * rstd * inv;
#pragma unroll
                for(int i = 0; i < E / 4; i++){
                    const float4 w = kept.at(K::PRE_WEIGHT, i);
                    const float2 h0 = mul2(x[2 * i], both(rstd)), h1 = mul2(x[2 * i + 1], both(rstd)), q0 = q[2 * i], q1 = q[2 * i + 1];
                    add_to(K::SUM_PRE_WEIGHT, i, q0, h0, q1, h1);
                    if constexpr(BIAS) add_to(K::SUM_PRE_BIAS, i, q0, both(1.0f), q1, both(1.0f));
                    d[2 * i] = fma2(fma2(h0, both(-along), fma2(q0, make_float2(w.x, w.y), both(-mean))), both(rstd), d[2 * i]);
                    d[2 * i + 1] = fma2(fma2(h1, both(-along), fma2(q1, make_float2(w.z, w.w), both(-mean))), both(rstd), d[2 * i + 1]);
                }
                if(a.pre == B200RL_NORM_LAYER) row.clear_outside(d);     // the post norm sums what lies behind the row's end too
            }
            if(post) rstd_u = rsqrtf(s[1] * inv + a.epsilon);
        }
        if(a.d_residual) row.store(a.d_residual, r * a.lddr, d);
        if(!a.branch) continue;
        // d: from here on the gradient of gate u; u: the normalised row
#pragma unroll
        for(int i = 0; i < P; i++){ d[i] = mul2(d[i], both(a.scale)); u[i] = mul2(u[i], both(rstd_u)); }
        if constexpr(GATE) if(gated){
            const bool group_ends = r + 1 == group_end, flush = group_ends || r + 1 == last;
            if constexpr(BIAS){
                if(a.d_gate){
                    float b[E];
                    if(post) row.parameters(opaque(a.post_bias), 0.0f, b);      // asked for with every row: kept over the rows it takes registers that lead to spills
#pragma unroll
                    for(int i = 0; i < E / 4; i++){
                        float2 v0 = u[2 * i], v1 = u[2 * i + 1];
                        if(post){
                            const float4 w = kept.at(K::POST_WEIGHT, i);
                            v0 = fma2(v0, make_float2(w.x, w.y), make_float2(b[4 * i], b[4 * i + 1]));
                            v1 = fma2(v1, make_float2(w.z, w.w), make_float2(b[4 * i + 2], b[4 * i + 3]));
                        }
                        add_to(K::SUM_GATE, i, d[2 * i], v0, d[2 * i + 1], v1);
                    }
                }
            }
            else
#pragma unroll
                for(int i = 0; i < E / 4; i++) add_to(K::SUM_GATE, i, d[2 * i], u[2 * i], d[2 * i + 1], u[2 * i + 1]);
            if(flush){
                float sum[E];
                hand_out(K::SUM_GATE, sum);
                if constexpr(!BIAS) if(post)
                    // without biases one sum of d u over the group gives both gradients: weight times it the gate's, gate times it the weight's
#pragma unroll
                    for(int i = 0; i < E / 4; i++){
                        const float4 w = kept.at(K::POST_WEIGHT, i);
                        float4 t = kept.at(K::SUM_POST_WEIGHT, i);
                        t.x = fmaf(to_float(raw_gate.e[4 * i]), sum[4 * i], t.x); t.y = fmaf(to_float(raw_gate.e[4 * i + 1]), sum[4 * i + 1], t.y);
                        t.z = fmaf(to_float(raw_gate.e[4 * i + 2]), sum[4 * i + 2], t.z); t.w = fmaf(to_float(raw_gate.e[4 * i + 3]), sum[4 * i + 3], t.w);
                        kept.at(K::SUM_POST_WEIGHT, i) = t;
                        sum[4 * i] *= w.x; sum[4 * i + 1] *= w.y; sum[4 * i + 2] *= w.z; sum[4 * i + 3] *= w.w;
                    }
                if(a.d_gate){
                    // the gate row's sum is complete here, or a piece of it: the group's rows go on with the next worker, or began with one before
                    if(group_ends && group_begin >= first) row.store(a.d_gate, group * a.lddg, sum);
                    else row.store_sums(a.pieces + ((long long)worker * 2 + (group_begin >= first ? 1 : 0)) * a.dim, sum);
                }
#pragma unroll
                for(int i = 0; i < E / 4; i++) kept.at(K::SUM_GATE, i) = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            }
#pragma unroll
            for(int i = 0; i < P; i++) d[i] = mul2(d[i], make_float2(to_float(raw_gate.e[2 * i]), to_float(raw_gate.e[2 * i + 1])));
            if(r + 1 == group_end && r + 1 < last){
                group++;
                group_begin = group_end;
                group_end = min((long long)a.rows, group_end + a.gate_rows);
                row.fetch(a.gate, group * a.ldg, raw_gate);
            }
        }
        if(post){
            float2 gg = both(0.0f), gh = gg;
#pragma unroll
            for(int i = 0; i < E / 4; i++){
                const float4 w = kept.at(K::POST_WEIGHT, i);
                if(BIAS || !GATE) add_to(K::SUM_POST_WEIGHT, i, d[2 * i], u[2 * i], d[2 * i + 1], u[2 * i + 1]);
                if constexpr(BIAS) add_to(K::SUM_POST_BIAS, i, d[2 * i], both(1.0f), d[2 * i + 1], both(1.0f));
                d[2 * i] = mul2(d[2 * i], make_float2(w.x, w.y));
                d[2 * i + 1] = mul2(d[2 * i + 1], make_float2(w.z, w.w));
                gg = add2(gg, add2(d[2 * i], d[2 * i + 1]));
                gh = fma2(d[2 * i], u[2 * i], gh); gh = fma2(d[2 * i + 1], u[2 * i + 1], gh);
            }
            float s[2] = {across(gg), across(gh)};
            row_sums<TPR>(s, buffer, turn);
            const float mean = a.post == B200RL_NORM_LAYER ? s[0] * inv : 0.0f, along = s[1] * inv;
#pragma unroll
            for(int i = 0; i < P; i++) d[i] = mul2(fma2(u[i], both(-along), add2(d[i], both(-mean))), both(rstd_u));
        }
        if(a.d_branch) row.store(a.d_branch, r * a.lddb, d);
    }
    constexpr int sums[SUMS] = {K::SUM_POST_WEIGHT, K::SUM_POST_BIAS, K::SUM_PRE_WEIGHT, K::SUM_PRE_BIAS};
#pragma unroll
    for(int i = 0; i < SUMS; i++)
        if(a.d_params[i] && (BIAS || i % 2 == 0)){
            float sum[E];
            hand_out(sums[i], sum);
            row.store_sums(a.partials + ((long long)i * a.workers + worker) * a.dim, sum);
        }
}

// A gate row whose rows lie with more than one worker: its pieces are those of workers first .. first + n - 1 (slot 1 of the first, which it goes beyond, slot 0 of the others).
struct GatePieces { long long group; int first, n; };
__device__ __forceinline__ GatePieces gate_pieces(const NormBackward& a, long long group){
    const long long begin = group * a.gate_rows, end = min((long long)a.rows, begin + a.gate_rows);
    const int w = (int)(begin / a.rows_per_worker);
    return {group, w, (int)((end - 1) / a.rows_per_worker) - w + 1};
}

// The sums over the workers, in their order, one launch for all. The first CTAs take the parameter gradients that are asked for and, if gate rows that several workers share are few
// (and have many pieces), those: 32 columns a CTA, 16 threads a column. Behind them, for many gate rows of few pieces, a CTA takes 512 columns of the gate row that lies across
// the boundary between one worker and the next, a thread a column.
template <typename T>
__global__ void __launch_bounds__(512) norm_backward_sums_kernel(NormBackward a, int few_gates){
    __shared__ float shared[16][33];
    after_predecessor();
    const int columns = (a.dim - 1) / 32 + 1, sum_ctas = (a.n_sums + few_gates) * columns;
    if((int)blockIdx.x >= sum_ctas){
        const int parts = (a.dim - 1) / 512 + 1, at = blockIdx.x - sum_ctas, worker = at / parts, c = (at - worker * parts) * 512 + threadIdx.x;
        const long long row = (worker + 1ll) * a.rows_per_worker;                       // the next worker's first row
        const GatePieces g = gate_pieces(a, row / a.gate_rows);
        if(c >= a.dim || g.first != worker) return;                                     // a gate row begins at the boundary, or its first boundary is an earlier one
        float v = a.pieces[(2ll * g.first + 1) * a.dim + c];
        for(int i = 1; i < g.n; i++) v += a.pieces[2ll * (g.first + i) * a.dim + c];
        static_cast<T*>(a.d_gate)[g.group * a.lddg + c] = from_float<T>(v);
        return;
    }
    const int lane = threadIdx.x & 31, slice = threadIdx.x >> 5, what = blockIdx.x / columns, c = (blockIdx.x - what * columns) * 32 + lane;
    const bool parameter = what < a.n_sums;
    const int index = parameter ? a.sums[what] : 0;
    const float* part; long long stride; int n, skip = 0;
    GatePieces g{};
    if(parameter){ part = a.partials + (long long)index * a.workers * a.dim; stride = a.dim; n = a.workers; }
    else{
        g = gate_pieces(a, what - a.n_sums);
        if(g.n == 1) return;
        part = a.pieces + 2ll * g.first * a.dim; stride = 2ll * a.dim; n = g.n; skip = a.dim;
    }
    float v = 0.0f;
    if(c < a.dim)
        for(int i = slice; i < n; i += 128){                 // eight loads under way
            float e[8];
#pragma unroll
            for(int j = 0; j < 8; j++) e[j] = i + 16 * j < n ? part[(i + 16 * j) * stride + (i + 16 * j == 0 ? skip : 0) + c] : 0.0f;
#pragma unroll
            for(int j = 0; j < 8; j++) v += e[j];
        }
    shared[slice][lane] = v;
    __syncthreads();
    if(slice || c >= a.dim) return;
#pragma unroll
    for(int i = 1; i < 16; i++) v += shared[i][lane];
    if(parameter){ float* out = a.d_params[index] + c; *out = a.accumulate ? *out + v : v; }
    else static_cast<T*>(a.d_gate)[g.group * a.lddg + c] = from_float<T>(v);
}

// Workers of the backward pass, and the consecutive rows that each takes: as many as are resident at once, a row each where there are fewer rows than that. `whole`: the form with biases
// and gate, of which fewer may be.
template <typename T>
static void plan_workers(int rows, int dim, bool whole, int* workers, int* rows_per_worker){
    const int most = dispatch_row<T>(dim, [&](auto shape){
        constexpr int TPR = decltype(shape)::tpr, E = decltype(shape)::e, all = backward_resident<T, TPR, E, true, true>(), less = backward_resident<T, TPR, E, false, false>();
        static_assert(backward_resident<T, TPR, E, true, false>() == less && backward_resident<T, TPR, E, false, true>() == less);
        return NUM_SMS * (whole ? all : less) * (TPR == 32 ? 4 : 1);
    });
    *rows_per_worker = (rows - 1) / most + 1;
    *workers = (rows - 1) / *rows_per_worker + 1;
}

template <typename T, int VEC, int TPR, int E>
static int launch_forward(const NormForward& a, cudaStream_t s){
    auto* kernel = norm_forward_kernel<T, VEC, TPR, E>;
    constexpr int ROWS = TPR < 128 ? 128 / TPR : 1, THREADS = TPR < 128 ? 128 : TPR, each = ROWS * E * TPR * 4;
    static_assert(4 * each + 1024 <= 232448, "four parameters of B200RL_NORM_MAX_DIM elements fit");
    const int bytes = each * ((a.post_weight != nullptr) + (a.post_bias != nullptr) + (a.pre_weight != nullptr) + (a.pre_bias != nullptr));
    static std::atomic<int> resident[MAX_DEVICES][5];        // CTAs a multiprocessor, by the number of parameters: 0 until looked up
    int dev = 0;
    const int rc = current_device(&dev);
    if(rc) return rc;
    int n = resident[dev][bytes / each].load(std::memory_order_acquire);
    if(n == 0){
        B200RL_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 4 * each));
        B200RL_CUDA_TRY(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, THREADS, bytes));
        if(n < 1) return B200RL_ERR_UNSUPPORTED;
        resident[dev][bytes / each].store(n, std::memory_order_release);
    }
    const int most = NUM_SMS * n, ctas = (a.rows - 1) / ROWS + 1;
    B200RL_CUDA_TRY(launch_after(kernel, dim3(ctas < most ? ctas : most), dim3(THREADS), bytes, s, a));
    return B200RL_OK;
}

template <typename T, int VEC, int TPR, int E, bool BIAS, bool GATE>
static int launch_backward(const NormBackward& a, cudaStream_t s){
    auto* kernel = norm_backward_kernel<T, VEC, TPR, E, BIAS, GATE>;
    constexpr int WORKERS = TPR < 128 ? 128 / TPR : 1, bytes = WORKERS * Kept<TPR, E, BIAS, GATE>::worker_bytes;
    static std::atomic<bool> configured[MAX_DEVICES];
    int dev = 0;
    const int rc = current_device(&dev);
    if(rc) return rc;
    if(!configured[dev].load(std::memory_order_acquire)){
        B200RL_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
        configured[dev].store(true, std::memory_order_release);
    }
    B200RL_CUDA_TRY(launch_after(kernel, dim3((a.workers + WORKERS - 1) / WORKERS), dim3(TPR < 128 ? 128 : TPR), bytes, s, a));
    return B200RL_OK;
}

}  // namespace b200rl
using namespace b200rl;

extern "C" {

int b200rl_norm_residual_forward(int type, int post, const float* post_weight, const float* post_bias, const void* branch, int ldb, const void* gate, int ldg,
                                 int gate_rows, float scale, const void* residual, int ldr, void* out, int ldo, int pre, const float* pre_weight,
                                 const float* pre_bias, void* normed, int ldn, int rows, int dim, float epsilon, b200rl_stream_t stream){
    if(!valid_type(type) || post < B200RL_NORM_NONE || post > B200RL_NORM_RMS || pre < B200RL_NORM_NONE || pre > B200RL_NORM_RMS) return B200RL_ERR_UNSUPPORTED;
    if(rows < 0 || dim < 1 || !(epsilon >= 0.0f)) return B200RL_ERR_INVALID_ARGUMENT;
    if(dim > B200RL_NORM_MAX_DIM) return B200RL_ERR_UNSUPPORTED;
    if(rows == 0) return B200RL_OK;
    if((!branch && !residual) || (gate && (!branch || gate_rows < 1)) || (!branch && post != B200RL_NORM_NONE) || (!out && !normed) || (pre != B200RL_NORM_NONE) != (normed != nullptr)) return B200RL_ERR_INVALID_ARGUMENT;
    const size_t e = type_bytes(type);
    const int gates = gate && rows > 0 ? (rows - 1) / gate_rows + 1 : 0;
    if((branch && !valid_matrix(branch, ldb, rows, dim, e)) || (residual && !valid_matrix(residual, ldr, rows, dim, e)) || (out && !valid_matrix(out, ldo, rows, dim, e)) ||
       (normed && !valid_matrix(normed, ldn, rows, dim, e)) || (gate && !valid_matrix(gate, ldg, gates, dim, e))) return B200RL_ERR_INVALID_ARGUMENT;
    NormForward a{branch, row_pitch(ldb, rows, dim), gate, row_pitch(ldg, gates, dim), gate_rows, residual, row_pitch(ldr, rows, dim), out, row_pitch(ldo, rows, dim),
                  normed, row_pitch(ldn, rows, dim), post_weight, post_bias, pre_weight, pre_bias, post, pre, rows, dim, scale, epsilon};
    const int n = 16 / (int)e;
    const bool vector = dim % n == 0 && (!branch || rows_aligned(branch, a.ldb, e)) && (!gate || rows_aligned(gate, a.ldg, e)) &&
                        (!residual || rows_aligned(residual, a.ldr, e)) && (!out || rows_aligned(out, a.ldo, e)) && (!normed || rows_aligned(normed, a.ldn, e));
    int rc = B200RL_ERR_UNSUPPORTED;
    B200RL_DISPATCH_TYPE(type, rc = dispatch_row<T>(dim, [&](auto shape){
        constexpr int TPR = decltype(shape)::tpr, E = decltype(shape)::e;
        return vector ? launch_forward<T, 16 / sizeof(T), TPR, E>(a, (cudaStream_t)stream) : launch_forward<T, 1, TPR, E>(a, (cudaStream_t)stream);
    }))
    return rc;
}

size_t b200rl_norm_residual_backward_scratch_bytes(int rows, int dim){
    if(rows < 1 || dim < 1 || dim > B200RL_NORM_MAX_DIM) return 0;
    int workers, workers32, per;
    plan_workers<__half>(rows, dim, false, &workers, &per);          // enough for the other form too, which has no more workers
    plan_workers<float>(rows, dim, false, &workers32, &per);
    return (size_t)(workers > workers32 ? workers : workers32) * (SUMS + 2) * dim * sizeof(float);
}

int b200rl_norm_residual_backward(int type, int post, const float* post_weight, const float* post_bias, const void* branch, int ldb, const void* gate, int ldg,
                                  int gate_rows, float scale, const void* out, int ldo, int pre, const float* pre_weight, const void* d_out, int lddo,
                                  const void* d_normed, int lddn, void* d_branch, int lddb, void* d_residual, int lddr, void* d_gate, int lddg,
                                  float* d_post_weight, float* d_post_bias, float* d_pre_weight, float* d_pre_bias, int accumulate, int rows, int dim,
                                  float epsilon, void* scratch, size_t scratch_bytes, b200rl_stream_t stream){
    if(!valid_type(type) || post < B200RL_NORM_NONE || post > B200RL_NORM_RMS || pre < B200RL_NORM_NONE || pre > B200RL_NORM_RMS) return B200RL_ERR_UNSUPPORTED;
    if(rows < 0 || dim < 1 || !(epsilon >= 0.0f) || (rows > 0 && (pre != B200RL_NORM_NONE) != (d_normed != nullptr))) return B200RL_ERR_INVALID_ARGUMENT;
    if(dim > B200RL_NORM_MAX_DIM) return B200RL_ERR_UNSUPPORTED;
    if((rows > 0 && ((gate && (!branch || gate_rows < 1)) || (!branch && (post != B200RL_NORM_NONE || d_branch)) || (d_gate && !gate))) ||
       ((d_post_weight || d_post_bias) && post == B200RL_NORM_NONE) || ((d_pre_weight || d_pre_bias) && pre == B200RL_NORM_NONE)) return B200RL_ERR_INVALID_ARGUMENT;
    const size_t e = type_bytes(type);
    const int gates = gate && rows > 0 ? (rows - 1) / gate_rows + 1 : 0;
    if(rows > 0 && ((branch && !valid_matrix(branch, ldb, rows, dim, e)) || (pre != B200RL_NORM_NONE && !valid_matrix(out, ldo, rows, dim, e)) ||
                    (d_out && !valid_matrix(d_out, lddo, rows, dim, e)) || (d_normed && !valid_matrix(d_normed, lddn, rows, dim, e)) ||
                    (d_branch && !valid_matrix(d_branch, lddb, rows, dim, e)) || (d_residual && !valid_matrix(d_residual, lddr, rows, dim, e)) ||
                    (gate && !valid_matrix(gate, ldg, gates, dim, e)) || (d_gate && !valid_matrix(d_gate, lddg, gates, dim, e)))) return B200RL_ERR_INVALID_ARGUMENT;
    float* const d_params[SUMS] = {d_post_weight, d_post_bias, d_pre_weight, d_pre_bias};
    if(rows == 0){
        if(!accumulate)
            for(float* p : d_params)
                if(p) B200RL_CUDA_TRY(cudaMemsetAsync(p, 0, dim * sizeof(float), (cudaStream_t)stream));
        return B200RL_OK;
    }
    if(!scratch || reinterpret_cast<uintptr_t>(scratch) % 16 || scratch_bytes < b200rl_norm_residual_backward_scratch_bytes(rows, dim)) return B200RL_ERR_INVALID_ARGUMENT;
    NormBackward a{branch, row_pitch(ldb, rows, dim), gate, row_pitch(ldg, gates, dim), gate_rows, out, row_pitch(ldo, rows, dim), d_out, row_pitch(lddo, rows, dim),
                   d_normed, row_pitch(lddn, rows, dim), d_branch, row_pitch(lddb, rows, dim), d_residual, row_pitch(lddr, rows, dim), d_gate, row_pitch(lddg, gates, dim),
                   post_weight, post_bias, pre_weight, {d_post_weight, d_post_bias, d_pre_weight, d_pre_bias}};
    a.post = post; a.pre = pre; a.rows = rows; a.dim = dim; a.accumulate = accumulate; a.scale = scale; a.epsilon = epsilon;
    const int n = 16 / (int)e;
    const bool vector = dim % n == 0 && (!branch || rows_aligned(branch, a.ldb, e)) && (!gate || rows_aligned(gate, a.ldg, e)) && (pre == B200RL_NORM_NONE || rows_aligned(out, a.ldo, e)) &&
                        (!d_out || rows_aligned(d_out, a.lddo, e)) && (!d_normed || rows_aligned(d_normed, a.lddn, e)) && (!d_branch || rows_aligned(d_branch, a.lddb, e)) &&
                        (!d_residual || rows_aligned(d_residual, a.lddr, e)) && (!d_gate || rows_aligned(d_gate, a.lddg, e));
    for(int i = 0; i < SUMS; i++) if(a.d_params[i]) a.sums[a.n_sums++] = i;
    const bool bias = d_post_bias || d_pre_bias || (post_bias && gate);
    const bool whole = !vector || (bias && gate);
    if(type == B200RL_TYPE_FLOAT32) plan_workers<float>(rows, dim, whole, &a.workers, &a.rows_per_worker); else plan_workers<__half>(rows, dim, whole, &a.workers, &a.rows_per_worker);
    a.partials = static_cast<float*>(scratch);
    a.pieces = a.partials + (size_t)SUMS * a.workers * dim;
    int rc = B200RL_ERR_UNSUPPORTED;
    B200RL_DISPATCH_TYPE(type, rc = dispatch_row<T>(dim, [&](auto shape){
        constexpr int TPR = decltype(shape)::tpr, E = decltype(shape)::e, V = 16 / sizeof(T);
        const cudaStream_t st = (cudaStream_t)stream;
        if(!vector) return launch_backward<T, 1, TPR, E, true, true>(a, st);
        if(bias) return gate ? launch_backward<T, V, TPR, E, true, true>(a, st) : launch_backward<T, V, TPR, E, true, false>(a, st);
        return gate ? launch_backward<T, V, TPR, E, false, true>(a, st) : launch_backward<T, V, TPR, E, false, false>(a, st);
    }))
    if(rc) return rc;
    const bool shared_gates = d_gate && a.workers > 1 && gate_rows > 1;
    const int few_gates = shared_gates && gates <= 32 ? gates : 0;
    const int ctas = (a.n_sums + few_gates) * ((dim - 1) / 32 + 1) + (shared_gates && !few_gates ? (a.workers - 1) * ((dim - 1) / 512 + 1) : 0);
    if(ctas) B200RL_DISPATCH_TYPE(type, B200RL_CUDA_TRY(launch_after(norm_backward_sums_kernel<T>, dim3(ctas), dim3(512), 0, (cudaStream_t)stream, a, few_gates)))
    return B200RL_OK;
}

}
