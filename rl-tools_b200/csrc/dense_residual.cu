// Dense layers of residual networks in 16-bit types: products whose epilogue carries bias, activation and residual, and their gradients.
#include "product.cuh"

namespace b200rl {

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

// the three products of a layer
static Product forward_product(const void* W, int ldw, const void* x, int ldx, int batch, int input_dim, int output_dim){
    Product g{};
    g.a = {x, row_pitch(ldx, batch, input_dim), false};
    g.b = {W, row_pitch(ldw, output_dim, input_dim), false};
    g.m = batch; g.n = output_dim; g.k = input_dim;
    return g;
}
static Product input_product(const void* W, int ldw, const void* d_pre, int ldd, int batch, int input_dim, int output_dim){
    Product g{};
    g.a = {d_pre, row_pitch(ldd, batch, output_dim), false};
    g.b = {W, row_pitch(ldw, output_dim, input_dim), true};
    g.m = batch; g.n = input_dim; g.k = output_dim;
    return g;
}
static Product weights_product(const void* x, int ldx, const void* d_pre, int ldd, const float* d_W, int batch, int input_dim, int output_dim){
    Product g{};
    g.a = {d_pre, row_pitch(ldd, batch, output_dim), true};
    g.b = {x, row_pitch(ldx, batch, input_dim), true};
    g.m = output_dim; g.n = input_dim; g.k = batch;
    g.out = const_cast<float*>(d_W); g.ld_out = input_dim;
    return g;
}
static bool valid_workspace(const void* workspace, size_t bytes, size_t needed){
    return needed == 0 || (workspace && reinterpret_cast<uintptr_t>(workspace) % 16 == 0 && bytes >= needed);
}

}  // namespace b200rl
using namespace b200rl;

extern "C" {

size_t b200rl_dense_residual_forward_workspace_bytes(const void* W, int ldw, const void* x, int ldx, int batch, int input_dim, int output_dim){
    if(batch < 1 || input_dim < 1 || output_dim < 1) return 0;
    const Product g = forward_product(W, ldw, x, ldx, batch, input_dim, output_dim);
    return product_rows_takes(g) ? 0 : product_tc_workspace_bytes(g, EPI_FORWARD);
}
size_t b200rl_dense_residual_backward_input_workspace_bytes(const void* W, int ldw, const void* d_pre, int ldd, int batch, int input_dim, int output_dim){
    return batch < 1 || input_dim < 1 || output_dim < 1 ? 0 : product_tc_workspace_bytes(input_product(W, ldw, d_pre, ldd, batch, input_dim, output_dim), EPI_INPUT);
}
size_t b200rl_dense_residual_backward_weights_workspace_bytes(const void* x, int ldx, const void* d_pre, int ldd, const float* d_W, int batch, int input_dim, int output_dim){
    return !d_W || batch < 1 || input_dim < 1 || output_dim < 1 ? 0 : product_tc_workspace_bytes(weights_product(x, ldx, d_pre, ldd, d_W, batch, input_dim, output_dim), EPI_SUM);
}

int b200rl_dense_residual_forward(int type, const void* W, int ldw, const float* bias, const void* x, int ldx, const void* residual, int ldr, float scale,
                                  void* pre, int ldpre, void* y, int ldy, int batch, int input_dim, int output_dim, int activation,
                                  void* workspace, size_t workspace_bytes, b200rl_stream_t stream){
    if(!valid_16_bit_type(type) || !valid_residual_activation(activation)) return B200RL_ERR_UNSUPPORTED;
    if(batch < 0 || input_dim < 1 || output_dim < 1) return B200RL_ERR_INVALID_ARGUMENT;
    if(batch == 0) return B200RL_OK;
    if(!valid_matrix(W, ldw, output_dim, input_dim, 2) || !valid_matrix(x, ldx, batch, input_dim, 2) || !valid_matrix(y, ldy, batch, output_dim, 2) ||
       (residual && !valid_matrix(residual, ldr, batch, output_dim, 2)) || (pre && !valid_matrix(pre, ldpre, batch, output_dim, 2)) ||
       reinterpret_cast<uintptr_t>(bias) % 4) return B200RL_ERR_INVALID_ARGUMENT;
    Product g = forward_product(W, ldw, x, ldx, batch, input_dim, output_dim);
    const bool few = product_rows_takes(g);
    if(!few && !valid_workspace(workspace, workspace_bytes, product_tc_workspace_bytes(g, EPI_FORWARD))) return B200RL_ERR_INVALID_ARGUMENT;
    g.bias = bias; g.scale = scale;
    g.add = residual; g.ld_add = row_pitch(ldr, batch, output_dim);
    g.pre = pre; g.ld_pre = row_pitch(ldpre, batch, output_dim);
    g.out = y; g.ld_out = row_pitch(ldy, batch, output_dim);
    g.act = activation;
    return few ? product_rows(g, type, (cudaStream_t)stream) : product_tc(g, type, EPI_FORWARD, workspace, (cudaStream_t)stream);
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
    Product g = input_product(W, ldw, d_pre, ldd, batch, input_dim, output_dim);
    if(!valid_workspace(workspace, workspace_bytes, product_tc_workspace_bytes(g, EPI_INPUT))) return B200RL_ERR_INVALID_ARGUMENT;
    g.add = add; g.ld_add = row_pitch(lda, batch, input_dim);
    g.act = activation_in;
    if(activation_in != B200RL_ACT_IDENTITY) g.pre = const_cast<void*>(pre_in); g.ld_pre = row_pitch(ldp, batch, input_dim);
    g.out = d_in; g.ld_out = row_pitch(ldi, batch, input_dim);
    return product_tc(g, type, EPI_INPUT, workspace, (cudaStream_t)stream);
}

int b200rl_dense_residual_backward_weights(int type, const void* x, int ldx, const void* d_pre, int ldd, float* d_W, float* d_bias, int accumulate, int batch,
                                           int input_dim, int output_dim, void* workspace, size_t workspace_bytes, b200rl_stream_t stream){
    if(!valid_16_bit_type(type)) return B200RL_ERR_UNSUPPORTED;
    if(batch < 0 || input_dim < 1 || output_dim < 1) return B200RL_ERR_INVALID_ARGUMENT;
    if(!d_W && !d_bias) return B200RL_OK;
    if(reinterpret_cast<uintptr_t>(d_W) % 4 || reinterpret_cast<uintptr_t>(d_bias) % 4) return B200RL_ERR_INVALID_ARGUMENT;
    if(batch > 0 && (!valid_matrix(d_pre, ldd, batch, output_dim, 2) || (d_W && !valid_matrix(x, ldx, batch, input_dim, 2)))) return B200RL_ERR_INVALID_ARGUMENT;
    if(batch == 0){
        if(accumulate) return B200RL_OK;
        if(d_W) B200RL_CUDA_TRY(cudaMemsetAsync(d_W, 0, sizeof(float) * (size_t)output_dim * input_dim, (cudaStream_t)stream));
        if(d_bias) B200RL_CUDA_TRY(cudaMemsetAsync(d_bias, 0, sizeof(float) * (size_t)output_dim, (cudaStream_t)stream));
        return B200RL_OK;
    }
    if(d_W){
        Product g = weights_product(x, ldx, d_pre, ldd, d_W, batch, input_dim, output_dim);
        if(!valid_workspace(workspace, workspace_bytes, product_tc_workspace_bytes(g, EPI_SUM))) return B200RL_ERR_INVALID_ARGUMENT;
        g.accumulate = accumulate; g.row_sums = d_bias;
        return product_tc(g, type, EPI_SUM, workspace, (cudaStream_t)stream);
    }
    if(d_bias){
        B200RL_DISPATCH_16_BIT_TYPE(type, column_sums_kernel<T><<<(output_dim + 255) / 256, 256, 0, (cudaStream_t)stream>>>(static_cast<const T*>(d_pre),
            row_pitch(ldd, batch, output_dim), batch, output_dim, d_bias, accumulate))
        B200RL_LAUNCH_CHECK("dense_residual bias gradient");
    }
    return B200RL_OK;
}

}
