// The norms around a block of a residual network, fused with the block's gate and residual scale:
//   u = post(branch), out = residual + scale gate u, normed = pre(out)
// and its gradients. Memory-bound: forward reads branch and residual and writes out and normed, backward reads out, d_normed, d_out and branch and writes
// d_residual and d_branch, each once. A row is held in the registers of 32, 128 or 512 threads as fp32, so the two passes of a variance (mean, then squared deviations)
// cost no second read. The statistics are not stored for the backward pass: it holds the rows in registers anyway and computes them again.
#include "residual.cuh"
#include <type_traits>

namespace b200rl {

namespace {
constexpr int ROW_THREADS_MAX = 512, ELEMENTS_MAX = 16;      // 512 x 16 = B200RL_NORM_MAX_DIM
static_assert(ROW_THREADS_MAX * ELEMENTS_MAX == B200RL_NORM_MAX_DIM);
constexpr int SUMS = 4;                                      // parameter gradients: post weight, post bias, pre weight, pre bias
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
    int post, pre, rows, dim, workers, rows_per_worker, accumulate;
    float scale, epsilon;
};

// Sums of N values over the threads of a row (one warp, or the whole CTA); every thread gets them. `buffer` is used in turns, so one barrier per call is enough.
template <int TPR, int N>
__device__ __forceinline__ void row_sums(float (&v)[N], float (*buffer)[N][TPR / 32], int& turn){
#pragma unroll
    for(int i = 0; i < N; i++)
#pragma unroll
        for(int o = 16; o > 0; o >>= 1) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
    if constexpr(TPR > 32){
        float (&shared)[N][TPR / 32] = buffer[turn];
        turn ^= 1;
        const int warp = threadIdx.x >> 5;
        if((threadIdx.x & 31) == 0)
#pragma unroll
            for(int i = 0; i < N; i++) shared[i][warp] = v[i];
        __syncthreads();
#pragma unroll
        for(int i = 0; i < N; i++){
            v[i] = 0.0f;
#pragma unroll
            for(int w = 0; w < TPR / 32; w++) v[i] += shared[i][w];
        }
    }
}

// The row's elements of one thread: vectors of VEC, TPR VEC apart. What lies behind the row's end reads as `fill`.
template <typename T, int VEC, int TPR, int E>
struct Row {
    int lane, dim;
    __device__ __forceinline__ int column(int i) const { return (i * TPR + lane) * VEC; }
    __device__ __forceinline__ void load(const T* row, float (&v)[E]) const {
#pragma unroll
        for(int i = 0; i < E / VEC; i++){
            float e[VEC];
#pragma unroll
            for(int j = 0; j < VEC; j++) e[j] = 0.0f;
            if(column(i) < dim) load_elements(row + column(i), e);
#pragma unroll
            for(int j = 0; j < VEC; j++) v[i * VEC + j] = e[j];
        }
    }
    __device__ __forceinline__ void store(T* row, const float (&v)[E]) const {
#pragma unroll
        for(int i = 0; i < E / VEC; i++){
            float e[VEC];
#pragma unroll
            for(int j = 0; j < VEC; j++) e[j] = v[i * VEC + j];
            if(column(i) < dim) store_elements(row + column(i), e);
        }
    }
    // fp32 parameters (NULL: `fill`)
    __device__ __forceinline__ void parameters(const float* p, float fill, float (&v)[E]) const {
#pragma unroll
        for(int i = 0; i < E / VEC; i++)
#pragma unroll
            for(int j = 0; j < VEC; j++) v[i * VEC + j] = p && column(i) < dim ? __ldg(p + column(i) + j) : fill;
    }
    __device__ __forceinline__ bool inside(int e) const { return column(e / VEC) < dim; }
};

// The row's first element, which lies in v[0] of its first thread. A call of row_sums has to follow before the next one.
template <int TPR>
__device__ __forceinline__ float row_first(float v){
    if constexpr(TPR == 32) return __shfl_sync(0xffffffffu, v, 0);
    else{
        __shared__ float first;
        if(threadIdx.x == 0) first = v;
        __syncthreads();
        return first;
    }
}

// v <- (v - mean) rstd in place (0 behind the row's end); returns rstd. The mean is summed about the row's first element: a constant row has variance 0 whatever its value,
// and the error of the mean goes by the row's spread.
template <typename R, int TPR, int E>
__device__ __forceinline__ float normalise(const R& row, int kind, float (&v)[E], float epsilon, float (*buffer)[1][TPR / 32], int& turn){
    const float inv = 1.0f / (float)row.dim;
    if(kind == B200RL_NORM_LAYER){
        const float first = row_first<TPR>(v[0]);
        float s[1] = {0.0f};
#pragma unroll
        for(int e = 0; e < E; e++){ v[e] = row.inside(e) ? v[e] - first : 0.0f; s[0] += v[e]; }
        row_sums<TPR>(s, buffer, turn);
        const float mean = s[0] * inv;
#pragma unroll
        for(int e = 0; e < E; e++) v[e] = row.inside(e) ? v[e] - mean : 0.0f;
    }
    float s[1] = {0.0f};
#pragma unroll
    for(int e = 0; e < E; e++) s[0] = fmaf(v[e], v[e], s[0]);
    row_sums<TPR>(s, buffer, turn);
    const float rstd = 1.0f / sqrtf(s[0] * inv + epsilon);
#pragma unroll
    for(int e = 0; e < E; e++) v[e] *= rstd;
    return rstd;
}

template <typename T, int VEC, int TPR, int E>
__global__ void __launch_bounds__(TPR < 128 ? 128 : TPR) norm_forward_kernel(NormForward a){
    constexpr int ROWS = TPR < 128 ? 128 / TPR : 1;
    __shared__ float buffer[2][1][TPR / 32];
    int turn = 0;
    const Row<T, VEC, TPR, E> R{(int)(threadIdx.x % TPR), a.dim};
    for(long long r = (long long)blockIdx.x * ROWS + threadIdx.x / TPR; r < a.rows; r += (long long)gridDim.x * ROWS){
        float o[E];
        if(a.residual) R.load(static_cast<const T*>(a.residual) + r * a.ldr, o);
        else
#pragma unroll
            for(int e = 0; e < E; e++) o[e] = 0.0f;
        if(a.branch){
            float u[E], p[E];
            R.load(static_cast<const T*>(a.branch) + r * a.ldb, u);
            if(a.post != B200RL_NORM_NONE){
                normalise<Row<T, VEC, TPR, E>, TPR>(R, a.post, u, a.epsilon, buffer, turn);
                if(a.post_weight){
                    R.parameters(a.post_weight, 1.0f, p);
#pragma unroll
                    for(int e = 0; e < E; e++) u[e] *= p[e];
                }
                if(a.post_bias){
                    R.parameters(a.post_bias, 0.0f, p);
#pragma unroll
                    for(int e = 0; e < E; e++) u[e] += p[e];
                }
            }
            if(a.gate){
                R.load(static_cast<const T*>(a.gate) + r / a.gate_rows * a.ldg, p);
#pragma unroll
                for(int e = 0; e < E; e++) u[e] *= p[e];
            }
#pragma unroll
            for(int e = 0; e < E; e++) o[e] = fmaf(a.scale, u[e], o[e]);
        }
        if(a.out) R.store(static_cast<T*>(a.out) + r * a.ldo, o);
        if(a.pre != B200RL_NORM_NONE){
            float p[E];
            normalise<Row<T, VEC, TPR, E>, TPR>(R, a.pre, o, a.epsilon, buffer, turn);
            if(a.pre_weight){
                R.parameters(a.pre_weight, 1.0f, p);
#pragma unroll
                for(int e = 0; e < E; e++) o[e] *= p[e];
            }
            if(a.pre_bias){
                R.parameters(a.pre_bias, 0.0f, p);
#pragma unroll
                for(int e = 0; e < E; e++) o[e] += p[e];
            }
            R.store(static_cast<T*>(a.normed) + r * a.ldn, o);
        }
    }
}

// q <- the gradient in front of a norm, from the gradient q of the normalised row: rstd (q - [mean q] - hat mean(q hat)); hat is the normalised row
template <typename R, int TPR, int E>
__device__ __forceinline__ void through_norm(const R& row, int kind, float (&q)[E], const float (&hat)[E], float rstd, float (*buffer)[2][TPR / 32], int& turn){
    const float inv = 1.0f / (float)row.dim;
    float s[2] = {0.0f, 0.0f};
#pragma unroll
    for(int e = 0; e < E; e++){ s[0] += q[e]; s[1] = fmaf(q[e], hat[e], s[1]); }
    row_sums<TPR>(s, buffer, turn);
    const float mean = kind == B200RL_NORM_LAYER ? s[0] * inv : 0.0f, along = s[1] * inv;
#pragma unroll
    for(int e = 0; e < E; e++) q[e] = row.inside(e) ? rstd * (q[e] - mean - hat[e] * along) : 0.0f;     // the next norm sums what lies behind the row's end too
}

// A worker (the threads of a row) takes rows_per_worker consecutive rows; the column sums of the parameter gradients stay in its registers.
template <typename T, int VEC, int TPR, int E>
__global__ void __launch_bounds__(TPR < 128 ? 128 : TPR) norm_backward_kernel(NormBackward a){
    constexpr int WORKERS = TPR < 128 ? 128 / TPR : 1;
    __shared__ float buffer1[2][1][TPR / 32], buffer2[2][2][TPR / 32];
    int turn1 = 0, turn2 = 0;
    const int worker = blockIdx.x * WORKERS + threadIdx.x / TPR;
    const long long first = (long long)worker * a.rows_per_worker, last = min((long long)a.rows, first + a.rows_per_worker);
    if(first >= last) return;                                // a whole row's threads leave together
    const Row<T, VEC, TPR, E> R{(int)(threadIdx.x % TPR), a.dim};
    float sum[SUMS][E], d_gate[E];
#pragma unroll
    for(int e = 0; e < E; e++){
        d_gate[e] = 0.0f;
#pragma unroll
        for(int i = 0; i < SUMS; i++) sum[i][e] = 0.0f;
    }
    for(long long r = first; r < last; r++){
        float d[E], u[E];
        if(a.d_out) R.load(static_cast<const T*>(a.d_out) + r * a.lddo, d);
        else
#pragma unroll
            for(int e = 0; e < E; e++) d[e] = 0.0f;
        if(a.branch) R.load(static_cast<const T*>(a.branch) + r * a.ldb, u);
        if(a.pre != B200RL_NORM_NONE){
            float x[E], q[E], p[E];
            R.load(static_cast<const T*>(a.d_normed) + r * a.lddn, q);
            R.load(static_cast<const T*>(a.out) + r * a.ldo, x);
            const float rstd = normalise<Row<T, VEC, TPR, E>, TPR>(R, a.pre, x, a.epsilon, buffer1, turn1);
            R.parameters(a.pre_weight, 1.0f, p);
#pragma unroll
            for(int e = 0; e < E; e++){
                sum[2][e] = fmaf(q[e], x[e], sum[2][e]);
                sum[3][e] += q[e];
                q[e] *= p[e];
            }
            through_norm<Row<T, VEC, TPR, E>, TPR>(R, a.pre, q, x, rstd, buffer2, turn2);
#pragma unroll
            for(int e = 0; e < E; e++) d[e] += q[e];
        }
        if(a.d_residual) R.store(static_cast<T*>(a.d_residual) + r * a.lddr, d);
        if(!a.branch) continue;
#pragma unroll
        for(int e = 0; e < E; e++) d[e] *= a.scale;          // from here on the gradient of gate u
        float rstd = 0.0f, hat[E];
        if(a.post != B200RL_NORM_NONE) rstd = normalise<Row<T, VEC, TPR, E>, TPR>(R, a.post, u, a.epsilon, buffer1, turn1);
#pragma unroll
        for(int e = 0; e < E; e++) hat[e] = u[e];
        float w[E];
        if(a.post != B200RL_NORM_NONE) R.parameters(a.post_weight, 1.0f, w);
        if(a.gate){
            float p[E];
            if(a.d_gate){
                if(a.post != B200RL_NORM_NONE){
                    R.parameters(a.post_bias, 0.0f, p);
#pragma unroll
                    for(int e = 0; e < E; e++) u[e] = fmaf(hat[e], w[e], p[e]);
                }
#pragma unroll
                for(int e = 0; e < E; e++) d_gate[e] = fmaf(d[e], u[e], d_gate[e]);
                const long long g = r / a.gate_rows, begin = g * a.gate_rows;
                const bool ends = r + 1 == a.rows || (r + 1) % a.gate_rows == 0;
                if(ends || r + 1 == last){
                    // the gate row's sum is complete here, or a piece of it: the group's rows go on with the next worker, or began with one before
                    if(ends && begin >= first) R.store(static_cast<T*>(a.d_gate) + g * a.lddg, d_gate);
                    else{
                        float* piece = a.pieces + ((long long)worker * 2 + (begin >= first ? 1 : 0)) * a.dim;
#pragma unroll
                        for(int e = 0; e < E; e++) if(R.inside(e)) piece[R.column(e / VEC) + e % VEC] = d_gate[e];
                    }
#pragma unroll
                    for(int e = 0; e < E; e++) d_gate[e] = 0.0f;
                }
            }
            R.load(static_cast<const T*>(a.gate) + r / a.gate_rows * a.ldg, p);
#pragma unroll
            for(int e = 0; e < E; e++) d[e] *= p[e];
        }
        if(a.post != B200RL_NORM_NONE){
#pragma unroll
            for(int e = 0; e < E; e++){
                sum[0][e] = fmaf(d[e], hat[e], sum[0][e]);
                sum[1][e] += d[e];
                d[e] *= w[e];
            }
            through_norm<Row<T, VEC, TPR, E>, TPR>(R, a.post, d, hat, rstd, buffer2, turn2);
        }
        if(a.d_branch) R.store(static_cast<T*>(a.d_branch) + r * a.lddb, d);
    }
#pragma unroll
    for(int i = 0; i < SUMS; i++)
        if(a.d_params[i]){
            float* partial = a.partials + ((long long)i * a.workers + worker) * a.dim;
#pragma unroll
            for(int e = 0; e < E; e++) if(R.inside(e)) partial[R.column(e / VEC) + e % VEC] = sum[i][e];
        }
}

// The sums over the workers, in their order: blockIdx.y < SUMS the parameter gradients, behind them the gate rows that begin with worker blockIdx.y - SUMS and go on
// with the next. 32 columns a CTA, eight threads a column.
template <typename T>
__global__ void __launch_bounds__(256) norm_backward_sums_kernel(NormBackward a){
    __shared__ float shared[8][33];
    const int c = blockIdx.x * 32 + (threadIdx.x & 31), slice = threadIdx.x >> 5;
    const float* part; long long stride; int n;
    long long g = 0;
    if(blockIdx.y < SUMS){
        if(!a.d_params[blockIdx.y]) return;
        part = a.partials + (long long)blockIdx.y * a.workers * a.dim; stride = a.dim; n = a.workers;
    }
    else{
        const long long w = blockIdx.y - SUMS, next = (w + 1) * a.rows_per_worker;      // the next worker's first row
        g = next / a.gate_rows;
        const long long begin = g * a.gate_rows;
        if(begin == next || begin < w * a.rows_per_worker) return;                       // a gate row begins there, or began with an earlier worker
        const long long end = min((long long)a.rows, begin + a.gate_rows);
        n = (int)((end - 1) / a.rows_per_worker - w) + 1;
        part = a.pieces + w * 2 * a.dim; stride = 2ll * a.dim;
    }
    float v = 0.0f;
    if(c < a.dim)
        for(int i = slice; i < n; i += 8) v += part[i * stride + (blockIdx.y >= SUMS && i == 0 ? a.dim : 0) + c];
    shared[slice][threadIdx.x & 31] = v;
    __syncthreads();
    if(slice || c >= a.dim) return;
#pragma unroll
    for(int i = 1; i < 8; i++) v += shared[i][threadIdx.x];
    if(blockIdx.y < SUMS) a.d_params[blockIdx.y][c] = a.accumulate ? a.d_params[blockIdx.y][c] + v : v;
    else static_cast<T*>(a.d_gate)[g * a.lddg + c] = from_float<T>(v);
}

// threads and elements per thread that hold a row
template <typename F>
static int dispatch_row(int dim, F f){
    if(dim <= 32 * 8) return f(std::integral_constant<int, 32>{}, std::integral_constant<int, 8>{});
    if(dim <= 32 * 16) return f(std::integral_constant<int, 32>{}, std::integral_constant<int, 16>{});
    if(dim <= 128 * 8) return f(std::integral_constant<int, 128>{}, std::integral_constant<int, 8>{});
    if(dim <= 128 * 16) return f(std::integral_constant<int, 128>{}, std::integral_constant<int, 16>{});
    if(dim <= 512 * 8) return f(std::integral_constant<int, 512>{}, std::integral_constant<int, 8>{});
    return f(std::integral_constant<int, 512>{}, std::integral_constant<int, 16>{});
}

// workers of the backward pass and the consecutive rows that each takes
static void plan_workers(int rows, int dim, int* workers, int* rows_per_worker){
    const int most = NUM_SMS * (dim <= 512 ? 16 : dim <= 2048 ? 4 : 1);
    const int per = rows <= 4 * most ? (rows <= most ? 1 : 4) : (rows + most - 1) / most;
    *rows_per_worker = per;
    *workers = (rows + per - 1) / per;
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
    return dispatch_row(dim, [&](auto tpr, auto el){
        constexpr int TPR = decltype(tpr)::value, E = decltype(el)::value, ROWS = TPR < 128 ? 128 / TPR : 1, THREADS = TPR < 128 ? 128 : TPR;
        const int grid = (rows - 1) / ROWS + 1;
        B200RL_DISPATCH_TYPE(type, if(vector) norm_forward_kernel<T, 16 / sizeof(T), TPR, E><<<grid, THREADS, 0, (cudaStream_t)stream>>>(a);
                                   else norm_forward_kernel<T, 1, TPR, E><<<grid, THREADS, 0, (cudaStream_t)stream>>>(a))
        B200RL_LAUNCH_CHECK("norm_residual_forward");
        return B200RL_OK;
    });
}

size_t b200rl_norm_residual_backward_scratch_bytes(int rows, int dim){
    if(rows < 1 || dim < 1 || dim > B200RL_NORM_MAX_DIM) return 0;
    int workers, per;
    plan_workers(rows, dim, &workers, &per);
    return (size_t)workers * (SUMS + 2) * dim * sizeof(float);
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
    plan_workers(rows, dim, &a.workers, &a.rows_per_worker);
    a.partials = static_cast<float*>(scratch);
    a.pieces = a.partials + (size_t)SUMS * a.workers * dim;
    a.post = post; a.pre = pre; a.rows = rows; a.dim = dim; a.accumulate = accumulate; a.scale = scale; a.epsilon = epsilon;
    const int n = 16 / (int)e;
    const bool vector = dim % n == 0 && (!branch || rows_aligned(branch, a.ldb, e)) && (!gate || rows_aligned(gate, a.ldg, e)) && (pre == B200RL_NORM_NONE || rows_aligned(out, a.ldo, e)) &&
                        (!d_out || rows_aligned(d_out, a.lddo, e)) && (!d_normed || rows_aligned(d_normed, a.lddn, e)) && (!d_branch || rows_aligned(d_branch, a.lddb, e)) &&
                        (!d_residual || rows_aligned(d_residual, a.lddr, e)) && (!d_gate || rows_aligned(d_gate, a.lddg, e));
    const int rc = dispatch_row(dim, [&](auto tpr, auto el){
        constexpr int TPR = decltype(tpr)::value, E = decltype(el)::value, WORKERS = TPR < 128 ? 128 / TPR : 1, THREADS = TPR < 128 ? 128 : TPR;
        const int grid = (a.workers + WORKERS - 1) / WORKERS;
        B200RL_DISPATCH_TYPE(type, if(vector) norm_backward_kernel<T, 16 / sizeof(T), TPR, E><<<grid, THREADS, 0, (cudaStream_t)stream>>>(a);
                                   else norm_backward_kernel<T, 1, TPR, E><<<grid, THREADS, 0, (cudaStream_t)stream>>>(a))
        B200RL_LAUNCH_CHECK("norm_residual_backward");
        return B200RL_OK;
    });
    if(rc) return rc;
    const bool shared_gates = d_gate && a.workers > 1;
    if(shared_gates || d_post_weight || d_post_bias || d_pre_weight || d_pre_bias){
        const dim3 grid((dim + 31) / 32, SUMS + (shared_gates ? a.workers - 1 : 0));
        B200RL_DISPATCH_TYPE(type, norm_backward_sums_kernel<T><<<grid, 256, 0, (cudaStream_t)stream>>>(a))
        B200RL_LAUNCH_CHECK("norm_residual_backward sums");
    }
    return B200RL_OK;
}

}
