// Dense layers of residual networks in 16-bit types: products whose epilogue carries bias, activation and residual, and their gradients.
#include "product.cuh"

namespace b200rl {

// Column sums (the bias gradient where the weights' is not asked for): 32 columns a CTA, 32 threads a column, each every 32nd row, then one after another in their order
template <typename T>
__global__ void __launch_bounds__(1024) column_sums_kernel(const T* d, long long ld, int rows, int cols, float* out, int accumulate){
    __shared__ float shared[32][32];
    after_predecessor();
    const int lane = threadIdx.x & 31, slice = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
    float v = 0.0f;
    if(c < cols)
#pragma unroll 8
        for(long long r = slice; r < rows; r += 32) v += to_float(d[r * ld + c]);            // rows may be 2^31 - 1
    shared[slice][lane] = v;
    __syncthreads();
    if(slice || c >= cols) return;
#pragma unroll
    for(int i = 1; i < 32; i++) v += shared[i][lane];
    out[c] = accumulate ? out[c] + v : v;
}

// Bound by memory: two or three 16-bit elements each. N elements a thread, of one row; rows on 16-byte boundaries are taken eight elements at a time.
template <typename T, int ACT, int N>
__global__ void __launch_bounds__(256) backward_activation_kernel(const T* pre, long long ldp, const T* d_y, long long ldd, float scale, T* d_pre, long long ldo, int rows, int cols){
    after_predecessor();
    const int chunks = (cols - 1) / N + 1;
    const long long total = (long long)rows * chunks;
    for(long long i = blockIdx.x * 256ll + threadIdx.x; i < total; i += gridDim.x * 256ll){
        const long long r = i / chunks; const int c = (int)(i - r * chunks) * N;
        float v[N], p[N];
        load_elements(d_y + r * ldd + c, v);
        if constexpr(ACT != B200RL_ACT_IDENTITY) load_elements(pre + r * ldp + c, p);
#pragma unroll
        for(int j = 0; j < N; j++){ v[j] *= scale; if constexpr(ACT != B200RL_ACT_IDENTITY) v[j] *= residual_d_activation<ACT>(p[j]); }
        store_elements(d_pre + r * ldo + c, v);
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
    g.bias = bias; g.scale = scale;
    g.add = residual; g.ld_add = row_pitch(ldr, batch, output_dim);
    g.pre = pre; g.ld_pre = row_pitch(ldpre, batch, output_dim);
    g.out = y; g.ld_out = row_pitch(ldy, batch, output_dim);
    g.act = activation;
    return product_rows_takes(g) ? product_rows(g, type, (cudaStream_t)stream) : product_tc(g, type, EPI_FORWARD, workspace, workspace_bytes, (cudaStream_t)stream);
}

int b200rl_dense_residual_backward_activation(int type, const void* pre, int ldpre, const void* d_y, int ldd, float scale, void* d_pre, int lddp, int rows,
                                              int cols, int activation, b200rl_stream_t stream){
    if(!valid_16_bit_type(type) || !valid_residual_activation(activation)) return B200RL_ERR_UNSUPPORTED;
    if(rows < 0 || cols < 1) return B200RL_ERR_INVALID_ARGUMENT;
    if(rows == 0) return B200RL_OK;
    if(!valid_matrix(d_y, ldd, rows, cols, 2) || !valid_matrix(d_pre, lddp, rows, cols, 2) ||
       (activation != B200RL_ACT_IDENTITY && !valid_matrix(pre, ldpre, rows, cols, 2))) return B200RL_ERR_INVALID_ARGUMENT;
    const long long ldp = row_pitch(ldpre, rows, cols), lds = row_pitch(ldd, rows, cols), ldo = row_pitch(lddp, rows, cols);
    const bool vector = cols % 8 == 0 && rows_aligned(d_y, lds, 2) && rows_aligned(d_pre, ldo, 2) && (activation == B200RL_ACT_IDENTITY || rows_aligned(pre, ldp, 2));
    const long long blocks = ((long long)rows * (vector ? cols / 8 : cols) + 255) / 256;
    const dim3 grid((unsigned)(blocks < NUM_SMS * 8 ? blocks : NUM_SMS * 8));
    B200RL_DISPATCH_16_BIT_TYPE(type, B200RL_DISPATCH_RESIDUAL_ACT(activation,
        B200RL_CUDA_TRY(launch_after(vector ? backward_activation_kernel<T, ACT, 8> : backward_activation_kernel<T, ACT, 1>, grid, dim3(256), 0, (cudaStream_t)stream,
                                     static_cast<const T*>(pre), ldp, static_cast<const T*>(d_y), lds, scale, static_cast<T*>(d_pre), ldo, rows, cols))))
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
    g.add = add; g.ld_add = row_pitch(lda, batch, input_dim);
    g.act = activation_in;
    if(activation_in != B200RL_ACT_IDENTITY) g.pre = const_cast<void*>(pre_in); g.ld_pre = row_pitch(ldp, batch, input_dim);
    g.out = d_in; g.ld_out = row_pitch(ldi, batch, input_dim);
    return product_tc(g, type, EPI_INPUT, workspace, workspace_bytes, (cudaStream_t)stream);
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
        g.accumulate = accumulate; g.row_sums = d_bias;
        return product_tc(g, type, EPI_SUM, workspace, workspace_bytes, (cudaStream_t)stream);
    }
    if(d_bias){
        B200RL_DISPATCH_16_BIT_TYPE(type, B200RL_CUDA_TRY(launch_after(column_sums_kernel<T>, dim3((output_dim - 1) / 32 + 1), dim3(1024), 0, (cudaStream_t)stream,
                                                                        static_cast<const T*>(d_pre), row_pitch(ldd, batch, output_dim), batch, output_dim, d_bias, accumulate)))
    }
    return B200RL_OK;
}

}
