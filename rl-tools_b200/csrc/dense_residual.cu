// Dense layers of residual networks in 16-bit types: products whose epilogue carries bias, activation and residual, and their gradients.
#include "residual.cuh"

namespace b200rl {

enum { EPI_FORWARD, EPI_INPUT, EPI_WEIGHTS };

// C(m, n) = sum_k A(m, k) B(n, k) with element (r, k) of an operand at p[r * row + k * col]
struct Product {
    const void* a; long long a_row, a_col;
    const void* b; long long b_row, b_col;
    int m, n, k;
    const float* bias;                          // EPI_FORWARD: out = add + scale act(sum + bias), pre = sum + bias
    const void* add; long long ld_add;          // EPI_INPUT: out = act'(pre) (sum + add)
    void* pre; long long ld_pre;
    void* out; long long ld_out;                // EPI_WEIGHTS: fp32, out (+)= sum
    float scale;
    int accumulate;
};

template <typename T, int EPI, int ACT>
__device__ __forceinline__ void finish_element(const Product& g, int m, int n, float v){
    if constexpr(EPI == EPI_FORWARD){
        if(g.bias) v += __ldg(g.bias + n);
        if(g.pre) static_cast<T*>(g.pre)[m * g.ld_pre + n] = from_float<T>(v);
        v = g.scale * residual_activation<ACT>(v);
        if(g.add) v += to_float(static_cast<const T*>(g.add)[m * g.ld_add + n]);
        static_cast<T*>(g.out)[m * g.ld_out + n] = from_float<T>(v);
    }
    else if constexpr(EPI == EPI_INPUT){
        if(g.add) v += to_float(static_cast<const T*>(g.add)[m * g.ld_add + n]);
        if constexpr(ACT != B200RL_ACT_IDENTITY) v *= residual_d_activation<ACT>(to_float(static_cast<const T*>(g.pre)[m * g.ld_pre + n]));
        static_cast<T*>(g.out)[m * g.ld_out + n] = from_float<T>(v);
    }
    else{
        float* out = static_cast<float*>(g.out) + m * g.ld_out + n;
        *out = g.accumulate ? *out + v : v;
    }
}

// 64 x 64 tile, 4 x 4 elements a thread, operands staged as fp32
template <typename T, int EPI, int ACT>
__global__ void __launch_bounds__(256) product_kernel(Product g){
    __shared__ float a[16][65], b[16][65];
    const int tid = threadIdx.x, m0 = blockIdx.y * 64, n0 = blockIdx.x * 64, tm = tid >> 4, tn = tid & 15;
    float acc[4][4] = {}, total[4][4] = {};
    for(int k0 = 0; k0 < g.k; k0 += 16){
        if(k0 % 512 == 0)                                    // long sums in pieces
            for(int i = 0; i < 4; i++)
                for(int j = 0; j < 4; j++){ total[i][j] += acc[i][j]; acc[i][j] = 0.0f; }
        for(int i = tid; i < 64 * 16; i += 256){
            const int r = i >> 4, k = i & 15;
            a[k][r] = m0 + r < g.m && k0 + k < g.k ? to_float(static_cast<const T*>(g.a)[(m0 + r) * g.a_row + (k0 + k) * g.a_col]) : 0.0f;
            b[k][r] = n0 + r < g.n && k0 + k < g.k ? to_float(static_cast<const T*>(g.b)[(n0 + r) * g.b_row + (k0 + k) * g.b_col]) : 0.0f;
        }
        __syncthreads();
        for(int k = 0; k < 16; k++)
            for(int i = 0; i < 4; i++)
                for(int j = 0; j < 4; j++) acc[i][j] += a[k][tm * 4 + i] * b[k][tn * 4 + j];
        __syncthreads();
    }
    for(int i = 0; i < 4; i++)
        for(int j = 0; j < 4; j++)
            if(m0 + tm * 4 + i < g.m && n0 + tn * 4 + j < g.n) finish_element<T, EPI, ACT>(g, m0 + tm * 4 + i, n0 + tn * 4 + j, total[i][j] + acc[i][j]);
}

template <typename T, int EPI, int ACT>
int launch_product(const Product& g, cudaStream_t s){
    product_kernel<T, EPI, ACT><<<dim3((g.n + 63) / 64, (g.m + 63) / 64), 256, 0, s>>>(g);
    B200RL_LAUNCH_CHECK("dense_residual product");
    return B200RL_OK;
}

template <typename T>
__global__ void __launch_bounds__(256) column_sums_kernel(const T* d, long long ld, int rows, int cols, float* out, int accumulate){
    const int c = blockIdx.x * 256 + threadIdx.x;
    if(c >= cols) return;
    float v = 0.0f;
    for(int r0 = 0; r0 < rows; r0 += 512){
        float piece = 0.0f;
        for(int r = r0; r < min(rows, r0 + 512); r++) piece += to_float(d[r * ld + c]);
        v += piece;
    }
    out[c] = accumulate ? out[c] + v : v;
}

template <typename T, int ACT>
__global__ void __launch_bounds__(256) backward_activation_kernel(const T* pre, long long ldp, const T* d_y, long long ldd, float scale, T* d_pre, long long ldo, int rows, int cols){
    const size_t n = (size_t)rows * cols;
    for(size_t i = blockIdx.x * (size_t)256 + threadIdx.x; i < n; i += (size_t)gridDim.x * 256){
        const long long r = i / cols; const int c = (int)(i - r * cols);
        float v = scale * to_float(d_y[r * ldd + c]);
        if constexpr(ACT != B200RL_ACT_IDENTITY) v *= residual_d_activation<ACT>(to_float(pre[r * ldp + c]));
        d_pre[r * ldo + c] = from_float<T>(v);
    }
}

}  // namespace b200rl
using namespace b200rl;

extern "C" {

size_t b200rl_dense_residual_forward_workspace_bytes(const void*, int, const void*, int, int, int, int){ return 0; }
size_t b200rl_dense_residual_backward_input_workspace_bytes(const void*, int, const void*, int, int, int, int){ return 0; }
size_t b200rl_dense_residual_backward_weights_workspace_bytes(const void*, int, const void*, int, int, int, int){ return 0; }

int b200rl_dense_residual_forward(int type, const void* W, int ldw, const float* bias, const void* x, int ldx, const void* residual, int ldr, float scale,
                                  void* pre, int ldpre, void* y, int ldy, int batch, int input_dim, int output_dim, int activation,
                                  void* workspace, size_t workspace_bytes, b200rl_stream_t stream){
    if(!valid_16_bit_type(type) || !valid_residual_activation(activation)) return B200RL_ERR_UNSUPPORTED;
    if(batch < 0 || input_dim < 1 || output_dim < 1) return B200RL_ERR_INVALID_ARGUMENT;
    if(batch == 0) return B200RL_OK;
    if(!valid_matrix(W, ldw, output_dim, input_dim, 2) || !valid_matrix(x, ldx, batch, input_dim, 2) || !valid_matrix(y, ldy, batch, output_dim, 2) ||
       (residual && !valid_matrix(residual, ldr, batch, output_dim, 2)) || (pre && !valid_matrix(pre, ldpre, batch, output_dim, 2)) ||
       reinterpret_cast<uintptr_t>(bias) % 4) return B200RL_ERR_INVALID_ARGUMENT;
    Product g{};
    g.a = x; g.a_row = row_pitch(ldx, batch, input_dim); g.a_col = 1;
    g.b = W; g.b_row = row_pitch(ldw, output_dim, input_dim); g.b_col = 1;
    g.m = batch; g.n = output_dim; g.k = input_dim;
    g.bias = bias; g.scale = scale;
    g.add = residual; g.ld_add = row_pitch(ldr, batch, output_dim);
    g.pre = pre; g.ld_pre = row_pitch(ldpre, batch, output_dim);
    g.out = y; g.ld_out = row_pitch(ldy, batch, output_dim);
    B200RL_DISPATCH_16_BIT_TYPE(type, B200RL_DISPATCH_RESIDUAL_ACT(activation, return (launch_product<T, EPI_FORWARD, ACT>(g, (cudaStream_t)stream))))
    return B200RL_ERR_UNSUPPORTED;
}

int b200rl_dense_residual_backward_activation(int type, const void* pre, int ldpre, const void* d_y, int ldd, float scale, void* d_pre, int lddp, int rows,
                                              int cols, int activation, b200rl_stream_t stream){
    if(!valid_16_bit_type(type) || !valid_residual_activation(activation)) return B200RL_ERR_UNSUPPORTED;
    if(rows < 0 || cols < 1) return B200RL_ERR_INVALID_ARGUMENT;
    if(rows == 0) return B200RL_OK;
    if(!valid_matrix(d_y, ldd, rows, cols, 2) || !valid_matrix(d_pre, lddp, rows, cols, 2) ||
       (activation != B200RL_ACT_IDENTITY && !valid_matrix(pre, ldpre, rows, cols, 2))) return B200RL_ERR_INVALID_ARGUMENT;
    const size_t blocks = ((size_t)rows * cols + 255) / 256;
    const int grid = (int)(blocks < NUM_SMS * 8 ? blocks : NUM_SMS * 8);
    B200RL_DISPATCH_16_BIT_TYPE(type, B200RL_DISPATCH_RESIDUAL_ACT(activation, (backward_activation_kernel<T, ACT><<<grid, 256, 0, (cudaStream_t)stream>>>(
        static_cast<const T*>(pre), row_pitch(ldpre, rows, cols), static_cast<const T*>(d_y), row_pitch(ldd, rows, cols), scale, static_cast<T*>(d_pre),
        row_pitch(lddp, rows, cols), rows, cols))))
    B200RL_LAUNCH_CHECK("dense_residual_backward_activation");
    return B200RL_OK;
}

int b200rl_dense_residual_backward_input(int type, const void* W, int ldw, const void* d_pre, int ldd, const void* add, int lda, const void* pre_in, int ldp,
                                         int activation_in, void* d_in, int ldi, int batch, int input_dim, int output_dim, void* workspace,
                                         size_t workspace_bytes, b200rl_stream_t stream){
    if(!valid_16_bit_type(type) || !valid_residual_activation(activation_in)) return B200RL_ERR_UNSUPPORTED;
    if(batch < 0 || input_dim < 1 || output_dim < 1) return B200RL_ERR_INVALID_ARGUMENT;
    if(batch == 0) return B200RL_OK;
    if(!valid_matrix(W, ldw, output_dim, input_dim, 2) || !valid_matrix(d_pre, ldd, batch, output_dim, 2) || !valid_matrix(d_in, ldi, batch, input_dim, 2) ||
       (add && !valid_matrix(add, lda, batch, input_dim, 2)) ||
       (activation_in != B200RL_ACT_IDENTITY && !valid_matrix(pre_in, ldp, batch, input_dim, 2))) return B200RL_ERR_INVALID_ARGUMENT;
    Product g{};
    g.a = d_pre; g.a_row = row_pitch(ldd, batch, output_dim); g.a_col = 1;
    g.b = W; g.b_row = 1; g.b_col = row_pitch(ldw, output_dim, input_dim);
    g.m = batch; g.n = input_dim; g.k = output_dim;
    g.add = add; g.ld_add = row_pitch(lda, batch, input_dim);
    g.pre = const_cast<void*>(pre_in); g.ld_pre = row_pitch(ldp, batch, input_dim);
    g.out = d_in; g.ld_out = row_pitch(ldi, batch, input_dim);
    B200RL_DISPATCH_16_BIT_TYPE(type, B200RL_DISPATCH_RESIDUAL_ACT(activation_in, return (launch_product<T, EPI_INPUT, ACT>(g, (cudaStream_t)stream))))
    return B200RL_ERR_UNSUPPORTED;
}

int b200rl_dense_residual_backward_weights(int type, const void* x, int ldx, const void* d_pre, int ldd, float* d_W, float* d_bias, int accumulate, int batch,
                                           int input_dim, int output_dim, void* workspace, size_t workspace_bytes, b200rl_stream_t stream){
    if(!valid_16_bit_type(type)) return B200RL_ERR_UNSUPPORTED;
    if(batch < 0 || input_dim < 1 || output_dim < 1) return B200RL_ERR_INVALID_ARGUMENT;
    if(!d_W && !d_bias) return B200RL_OK;
    if(reinterpret_cast<uintptr_t>(d_W) % 4 || reinterpret_cast<uintptr_t>(d_bias) % 4) return B200RL_ERR_INVALID_ARGUMENT;
    if(batch > 0 && (!valid_matrix(d_pre, ldd, batch, output_dim, 2) || (d_W && !valid_matrix(x, ldx, batch, input_dim, 2)))) return B200RL_ERR_INVALID_ARGUMENT;
    if(d_W){
        Product g{};
        g.a = d_pre; g.a_row = 1; g.a_col = row_pitch(ldd, batch, output_dim);
        g.b = x; g.b_row = 1; g.b_col = row_pitch(ldx, batch, input_dim);
        g.m = output_dim; g.n = input_dim; g.k = batch;
        g.out = d_W; g.ld_out = input_dim; g.accumulate = accumulate;
        int rc = 0;
        B200RL_DISPATCH_16_BIT_TYPE(type, rc = (launch_product<T, EPI_WEIGHTS, B200RL_ACT_IDENTITY>(g, (cudaStream_t)stream)))
        if(rc) return rc;
    }
    if(d_bias){
        B200RL_DISPATCH_16_BIT_TYPE(type, column_sums_kernel<T><<<(output_dim + 255) / 256, 256, 0, (cudaStream_t)stream>>>(static_cast<const T*>(d_pre),
            row_pitch(ldd, batch, output_dim), batch, output_dim, d_bias, accumulate))
        B200RL_LAUNCH_CHECK("dense_residual bias gradient");
    }
    return B200RL_OK;
}

}
