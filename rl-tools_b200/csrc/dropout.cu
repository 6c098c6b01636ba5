// Dropout whose mask is never stored: element e is kept or dropped by 16 bits of the Philox block e / 8, so the backward pass draws the same mask again.
#include "residual.cuh"
#include "rollout.cuh"

namespace b200rl {

struct Dropout {
    const void* x; long long ldx;
    const void* residual; long long ldr;
    void* y; long long ldy;
    int rows, cols;
    uint32_t threshold;             // an element is dropped when its 16 bits are below
    float scale;
    unsigned long long seed, call;
    const unsigned long long* call_counter;
    uint32_t stream_id;
};

// A thread takes the eight elements of a block. VECTOR: they lie in one row, 16-byte accesses.
template <typename T, bool VECTOR>
__global__ void __launch_bounds__(256) dropout_kernel(Dropout d){
    const unsigned long long n = (unsigned long long)d.rows * d.cols, blocks = (n + 7) / 8, call = d.call + (d.call_counter ? *d.call_counter : 0ull);
    for(unsigned long long b = blockIdx.x * 256ull + threadIdx.x; b < blocks; b += gridDim.x * 256ull){
        uint32_t c[4] = {(uint32_t)b, (uint32_t)call, (uint32_t)(call >> 32), 0x80000000u + ((uint32_t)(b >> 32) << 16) + d.stream_id};
        Philox::block(c, (uint32_t)d.seed, (uint32_t)(d.seed >> 32));
        long long row = (long long)(b * 8 / d.cols); int col = (int)(b * 8 - (unsigned long long)row * d.cols);
        if constexpr(VECTOR){
            constexpr int N = 16 / sizeof(T);
#pragma unroll
            for(int part = 0; part < 8 / N; part++){
                float v[N], r[N];
                load_elements(static_cast<const T*>(d.x) + row * d.ldx + col + part * N, v);
                if(d.residual) load_elements(static_cast<const T*>(d.residual) + row * d.ldr + col + part * N, r);
#pragma unroll
                for(int i = 0; i < N; i++){
                    const int e = part * N + i;
                    const uint32_t draw = (c[e >> 1] >> (16 * (e & 1))) & 0xFFFFu;
                    v[i] = (draw >= d.threshold ? v[i] * d.scale : 0.0f) + (d.residual ? r[i] : 0.0f);
                }
                store_elements(static_cast<T*>(d.y) + row * d.ldy + col + part * N, v);
            }
        }
        else{
#pragma unroll
            for(int e = 0; e < 8; e++){
                if(b * 8 + e < n){
                    const uint32_t draw = (c[e >> 1] >> (16 * (e & 1))) & 0xFFFFu;
                    float v = draw >= d.threshold ? to_float(static_cast<const T*>(d.x)[row * d.ldx + col]) * d.scale : 0.0f;
                    if(d.residual) v += to_float(static_cast<const T*>(d.residual)[row * d.ldr + col]);
                    static_cast<T*>(d.y)[row * d.ldy + col] = from_float<T>(v);
                    if(++col == d.cols){ col = 0; row++; }
                }
            }
        }
    }
}

}  // namespace b200rl
using namespace b200rl;

extern "C" int b200rl_dropout(int type, const void* x, int ldx, const void* residual, int ldr, void* y, int ldy, int rows, int cols, float p, unsigned long long seed,
                              unsigned int stream_id, unsigned long long call_index, const unsigned long long* call_counter, b200rl_stream_t stream){
    if(!valid_type(type)) return B200RL_ERR_UNSUPPORTED;
    if(rows < 0 || cols < 1 || !(p >= 0.0f && p <= 1.0f) || stream_id >= 65536u || (unsigned long long)rows * cols > 1ull << 50) return B200RL_ERR_INVALID_ARGUMENT;
    if(rows == 0) return B200RL_OK;
    const size_t e = type_bytes(type);
    if(!valid_matrix(x, ldx, rows, cols, e) || !valid_matrix(y, ldy, rows, cols, e) || (residual && !valid_matrix(residual, ldr, rows, cols, e)) ||
       reinterpret_cast<uintptr_t>(call_counter) % 8) return B200RL_ERR_INVALID_ARGUMENT;
    Dropout d{x, row_pitch(ldx, rows, cols), residual, row_pitch(ldr, rows, cols), y, row_pitch(ldy, rows, cols), rows, cols};
    d.threshold = (uint32_t)((double)p * 65536.0 + 0.5);
    d.scale = d.threshold < 65536u ? 65536.0f / (float)(65536u - d.threshold) : 0.0f;
    d.seed = seed; d.call = call_index; d.call_counter = call_counter; d.stream_id = stream_id;
    const bool vector = cols % 8 == 0 && rows_aligned(x, d.ldx, e) && rows_aligned(y, d.ldy, e) && (!residual || rows_aligned(residual, d.ldr, e));
    const unsigned long long blocks = ((unsigned long long)rows * cols + 7) / 8, ctas = (blocks + 255) / 256;
    const unsigned grid = (unsigned)(ctas < NUM_SMS * 8 ? ctas : NUM_SMS * 8);
    B200RL_DISPATCH_TYPE(type, if(vector) dropout_kernel<T, true><<<grid, 256, 0, (cudaStream_t)stream>>>(d); else dropout_kernel<T, false><<<grid, 256, 0, (cudaStream_t)stream>>>(d))
    B200RL_LAUNCH_CHECK("dropout");
    return B200RL_OK;
}
