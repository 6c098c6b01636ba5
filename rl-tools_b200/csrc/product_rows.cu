// The forward product of a few rows (single tokens of a serving loop): C(m, n) = sum_k x(m, k) W(n, k) for m <= 32. Bound by reading W once; nothing is set up before the first
// load (no tensor maps, barriers or tensor memory, which cost the tensor-memory kernel of product_tc.cu 1.5 us before its first sum). A warp takes 16 rows of W and every
// eighth block of 32 k; W is the left operand of mma.sync (16 of its rows x 16 k), the rows of x the right one (8 at a time). Which k an instruction's slots stand for does not
// matter as long as both operands agree, so a lane loads eight consecutive k of its rows by one 16-byte access and feeds two instructions with them. The eight warps' sums meet in
// shared memory, in their order, and the layer's epilogue follows.
// Measured (bfloat16, 1024 -> 4096, calls in a graph): 1 row 3.2 us, 16 rows 3.5 us, 32 rows 4.9 us (64 would be 7.5; the library's product takes 5, 3.7 and 3.8), where W's 8.4 MB take 1.3 us at the rate of memory and a launch about 2; the
// tensor-memory kernel takes 8.5 us.
#include "product.cuh"
#include <limits.h>

namespace b200rl {

struct RowsArgs {
    const void* x; long long ldx;
    const void* w; long long ldw;
    int m, n, k;
    const float* bias;
    const void* add; long long ld_add;
    void* pre; long long ld_pre;
    void* out; long long ld_out;
    float scale;
    int act;
};

template <typename T> __device__ __forceinline__ void mma_16_8_16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1);
template <> __device__ __forceinline__ void mma_16_8_16<__nv_bfloat16>(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1){
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <> __device__ __forceinline__ void mma_16_8_16<__half>(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1){
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// elements k .. k + 7 of a row, 0 behind its end
template <typename T, bool ALIGNED> __device__ __forceinline__ uint4 load_eight(const T* row, int k, int end){
    if(ALIGNED && k + 8 <= end) return *reinterpret_cast<const uint4*>(row + k);
    union { uint4 v; T e[8]; } u;
    u.v = make_uint4(0, 0, 0, 0);
#pragma unroll
    for(int j = 0; j < 8; j++) if(k + j < end) u.e[j] = row[k + j];
    return u.v;
}

// NT: groups of 8 rows of x; AHEAD: blocks of 32 k whose loads are under way together
template <typename T, int NT, int AHEAD, bool ALIGNED>
__global__ void __launch_bounds__(256) product_rows_kernel(RowsArgs a){
    __shared__ float shared[8][16][NT * 8 + 1];
    after_predecessor();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3, n0 = blockIdx.x * 16;
    const T *w[2], *x[NT];
#pragma unroll
    for(int h = 0; h < 2; h++) w[h] = static_cast<const T*>(a.w) + min(n0 + h * 8 + g, a.n - 1) * a.ldw;     // rows behind the last are computed and not stored
#pragma unroll
    for(int j = 0; j < NT; j++) x[j] = static_cast<const T*>(a.x) + min(j * 8 + g, a.m - 1) * a.ldx;
    float acc[NT][4] = {};
    const int blocks = (a.k - 1) / 32 + 1;
    for(int kb = warp; kb < blocks; kb += 8 * AHEAD){
        uint4 wv[AHEAD][2], xv[AHEAD][NT];
#pragma unroll
        for(int s = 0; s < AHEAD; s++){
            const int k = (kb + 8 * s) * 32 + 8 * t;
#pragma unroll
            for(int h = 0; h < 2; h++) wv[s][h] = kb + 8 * s < blocks ? load_eight<T, ALIGNED>(w[h], k, a.k) : make_uint4(0, 0, 0, 0);
#pragma unroll
            for(int j = 0; j < NT; j++) xv[s][j] = kb + 8 * s < blocks ? load_eight<T, ALIGNED>(x[j], k, a.k) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for(int s = 0; s < AHEAD; s++)
#pragma unroll
            for(int j = 0; j < NT; j++){
                mma_16_8_16<T>(acc[j], wv[s][0].x, wv[s][1].x, wv[s][0].y, wv[s][1].y, xv[s][j].x, xv[s][j].y);
                mma_16_8_16<T>(acc[j], wv[s][0].z, wv[s][1].z, wv[s][0].w, wv[s][1].w, xv[s][j].z, xv[s][j].w);
            }
    }
#pragma unroll
    for(int j = 0; j < NT; j++)
#pragma unroll
        for(int c = 0; c < 4; c++) shared[warp][(c >> 1) * 8 + g][j * 8 + 2 * t + (c & 1)] = acc[j][c];
    __syncthreads();
    for(int i = tid; i < 16 * NT * 8; i += 256){
        const int o = i % 16, row = i / 16, col = n0 + o;
        if(row >= a.m || col >= a.n) continue;
        float v = 0.0f;
#pragma unroll
        for(int s = 0; s < 8; s++) v += shared[s][o][row];
        if(a.bias) v += a.bias[col];
        if(a.pre) static_cast<T*>(a.pre)[row * a.ld_pre + col] = from_float<T>(v);
        B200RL_DISPATCH_RESIDUAL_ACT(a.act, v = residual_activation<ACT>(v))
        v = fmaf(a.scale, v, a.add ? to_float(static_cast<const T*>(a.add)[row * a.ld_add + col]) : 0.0f);
        static_cast<T*>(a.out)[row * a.ld_out + col] = from_float<T>(v);
    }
}

template <typename T, bool ALIGNED>
static int launch_rows(const RowsArgs& a, cudaStream_t s){
    const dim3 grid16((a.n - 1) / 16 + 1), block(256);
    if(a.m <= 8) B200RL_CUDA_TRY(launch_after(product_rows_kernel<T, 1, 4, ALIGNED>, grid16, block, 0, s, a));
    else if(a.m <= 16) B200RL_CUDA_TRY(launch_after(product_rows_kernel<T, 2, 4, ALIGNED>, grid16, block, 0, s, a));
    else B200RL_CUDA_TRY(launch_after(product_rows_kernel<T, 4, 2, ALIGNED>, grid16, block, 0, s, a));
    return B200RL_OK;
}

bool product_rows_takes(const Product& g){ return g.m <= 32 && !g.a.k_rows && !g.b.k_rows && g.n <= INT_MAX - 1024 && g.k <= INT_MAX - 1024; }
int product_rows(const Product& g, int type, cudaStream_t s){
    const RowsArgs a{g.a.p, g.a.ld, g.b.p, g.b.ld, g.m, g.n, g.k, g.bias, g.add, g.ld_add, g.pre, g.ld_pre, g.out, g.ld_out, g.scale, g.act};
    const bool aligned = (g.m == 1 ? reinterpret_cast<uintptr_t>(g.a.p) % 16 == 0 : rows_aligned(g.a.p, g.a.ld, 2)) &&
                         (g.n == 1 ? reinterpret_cast<uintptr_t>(g.b.p) % 16 == 0 : rows_aligned(g.b.p, g.b.ld, 2));
    B200RL_DISPATCH_16_BIT_TYPE(type, return aligned ? (launch_rows<T, true>(a, s)) : (launch_rows<T, false>(a, s)))
}

}  // namespace b200rl
