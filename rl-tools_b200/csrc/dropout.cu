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

// How the elements lie: FLAT: one after another from the first row to the last in every operand, ROWS: the eight elements of a block lie in one row, both by 16-byte
// accesses; ANY: one by one.
enum { FLAT, ROWS, ANY };

// the four words of block b: a draw of 16 bits for each of its elements
__device__ __forceinline__ void draw_block(const Dropout& d, unsigned long long call, unsigned long long b, uint32_t (&c)[4]){
    c[0] = (uint32_t)b; c[1] = (uint32_t)call; c[2] = (uint32_t)(call >> 32); c[3] = 0x80000000u + ((uint32_t)(b >> 32) << 16) + d.stream_id;
    Philox::block(c, (uint32_t)d.seed, (uint32_t)(d.seed >> 32));
}
__device__ __forceinline__ float drop(const Dropout& d, const uint32_t (&c)[4], int e, float v){
    return ((c[e >> 1] >> (16 * (e & 1))) & 0xFFFFu) >= d.threshold ? v * d.scale : 0.0f;
}

// A thread takes the eight elements of a block. Bound by memory: 16384 x 4096 bfloat16 with a residual 64.5 us = 6.2 TB/s, 1003 x 777 float32 2.4 us. The ten rounds of a block cost
// each of its eight elements about ten instructions, half of what the loads leave room for -- 32 bits an element, four elements a block, would take all of it.
template <typename T, int LAYOUT>
__global__ void __launch_bounds__(256) dropout_kernel(Dropout d){
    after_predecessor();
    const unsigned long long n = (unsigned long long)d.rows * d.cols, blocks = (n + 7) / 8, call = d.call + (d.call_counter ? *opaque(d.call_counter) : 0ull);
    const T *x = static_cast<const T*>(d.x), *residual = static_cast<const T*>(d.residual);
    T* y = static_cast<T*>(d.y);
    for(unsigned long long b = blockIdx.x * 256ull + threadIdx.x; b < blocks; b += gridDim.x * 256ull){
        uint32_t c[4];
        long long row = 0, col = (long long)(b * 8);
        if constexpr(LAYOUT != FLAT){ row = (long long)(b * 8 / d.cols); col = (long long)(b * 8) - row * d.cols; }
        if(LAYOUT != ANY && b * 8 + 8 <= n){
            constexpr int N = 16 / sizeof(T), PARTS = 8 / N;
            float v[PARTS][N], r[PARTS][N];
#pragma unroll
            for(int part = 0; part < PARTS; part++){
                load_elements(x + row * d.ldx + col + part * N, v[part]);
                if(residual) load_elements(residual + row * d.ldr + col + part * N, r[part]);
            }
            draw_block(d, call, b, c);
#pragma unroll
            for(int part = 0; part < PARTS; part++){
#pragma unroll
                for(int i = 0; i < N; i++) v[part][i] = drop(d, c, part * N + i, v[part][i]) + (residual ? r[part][i] : 0.0f);
                store_elements(y + row * d.ldy + col + part * N, v[part]);
            }
        }
        else{
            draw_block(d, call, b, c);
#pragma unroll
            for(int e = 0; e < 8; e++){
                if(b * 8 + e < n){
                    float v = drop(d, c, e, to_float(x[row * d.ldx + col]));
                    if(residual) v += to_float(residual[row * d.ldr + col]);
                    y[row * d.ldy + col] = from_float<T>(v);
                    col++;
                    if constexpr(LAYOUT != FLAT) if(col == d.cols){ col = 0; row++; }
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
    const bool flat = d.ldx == cols && d.ldy == cols && (!residual || d.ldr == cols) && rows_aligned(x, 16, e) && rows_aligned(y, 16, e) && (!residual || rows_aligned(residual, 16, e));
    const bool vector = cols % 8 == 0 && rows_aligned(x, d.ldx, e) && rows_aligned(y, d.ldy, e) && (!residual || rows_aligned(residual, d.ldr, e));
    const unsigned long long blocks = ((unsigned long long)rows * cols + 7) / 8, ctas = (blocks + 255) / 256;
    const dim3 grid((unsigned)(ctas < NUM_SMS * 8 ? ctas : NUM_SMS * 8));
    B200RL_DISPATCH_TYPE(type, B200RL_CUDA_TRY(launch_after(flat ? dropout_kernel<T, FLAT> : vector ? dropout_kernel<T, ROWS> : dropout_kernel<T, ANY>, grid, dim3(256), 0,
                                                            (cudaStream_t)stream, d)))
    return B200RL_OK;
}
