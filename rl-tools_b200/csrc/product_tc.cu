// Products of 16-bit matrices on the tensor cores: operands by TMA into 128-byte-swizzled shared memory, tcgen05.mma with fp32 sums in tensor memory, the layer's epilogue on
// the way out. C(m, n) = sum_k A(m, k) B(n, k); either operand may have k as the contiguous index of its matrix (the forward pass) or its row index (weights in the
// input gradient, both operands in the weight gradient): TMA brings either form in, the operand descriptors say which it is, nothing is transposed.
//
// A CTA (or a pair of CTAs: CG = 2, one MMA over both SMs, each holding half of A and half of B) is persistent over output tiles of 128 CG x BN. Its warps:
//   0  loads: stages of 64 k through a ring          1  issues the MMAs          2, 3  row sums of A (the bias gradient), straight from its matrix, beside the products
//   4-19  epilogue: 32 rows x BN / 4 columns each, from one of two accumulators while the tensor core fills the other. Sixteen warps, because a warp's way from tensor memory to the
//         outputs is a chain of waits: with eight, the epilogue of a tile (10,000 cycles) was longer than its products over 1024 k (8,200)
// Weight gradients (EPI_SUM) are summed in pieces of PIECE k: the tensor core's accumulator truncates with every addition, which over a long batch adds up (4,096 additions lose
// 1e-4); pieces of 32 additions are added in registers with rounding, while the next piece runs. Error of a weight gradient over 4,096 rows: 4.8e-7 (2-norm), an fp32 loop's 6.1e-7.
// Products of few tiles share each tile's k among the CTAs of a cluster, which add up through one another's shared memory.
//
// Bound by the tensor cores where the products are long: the tensor pipe is busy 91% of the cycles at 8192 x 4096 x 4096. A stage's operands would have to come from L2 at 64 bytes a
// cycle and multiprocessor to keep it busy all the time; so they come at 58. Tiles of 256 x 256 over a pair are what the tensor memory holds twice (128 x 128 by one CTA: 740 us for
// 16384 x 4096 x 4096). Small products are bound by the way through the kernel (256 x 256 x 256: 0.9 us until the first operands are there, 1 for the products, 0.8 for the epilogue, the
// rest launch). us of one bfloat16 product, calls in a graph with inputs that stay, and in brackets the library's product on the same box:
//   16384 x 4096 x 4096  forward 331 (334), gradient of the input 328 (333), of the weights 391 (374)
//   4096 x 1024 x 4096   26 (29), 27 (25), 34 (26); forward with bias, gelu, residual and pre-activations 39, gradient of the input with gelu's slope and an addend 31
//   2048 x 2048 x 2048   17 (14), 16 (14), 18 (14)
//   1024 x 1024 x 1024   7.8 (4.9), 7.5 (4.8), 7.9 (4.7)
//   256 x 256 x 256      4.4 (2.7), 4.1 (2.7), 4.4 (2.7)
#include "product.cuh"
#include "tcgen05.cuh"
#include <cuda.h>
#include <atomic>
#include <limits.h>

namespace b200rl {

namespace {
constexpr int KB = 64;                                   // k of a stage: 128 bytes
constexpr int PIECE = 512;                               // k in one accumulator of EPI_SUM
constexpr int EPI_WARPS = 16, EPI_THREADS = EPI_WARPS * 32, THREADS = 128 + EPI_THREADS;
constexpr uint32_t A_BYTES = 128 * 128;
constexpr uint32_t STAGING = 4096;                       // per epilogue warp: a slab of 32 x 32 fp32
constexpr uint32_t SMEM_LIMIT = 232448;
constexpr long long WAIT_LIMIT = 2000000000LL;           // cycles: about a second
constexpr int SUM_COLUMNS = 16, SUM_THREADS = 64;        // columns of a work item of the row sums: 32 bytes, a sector

__host__ __device__ constexpr uint32_t stage_bytes(int CG, int BN){ return A_BYTES + (uint32_t)(BN / CG) * 128; }
__host__ __device__ constexpr int stage_count(int CG, int BN){ return (int)((SMEM_LIMIT - 1024 - EPI_WARPS * STAGING - 512) / stage_bytes(CG, BN)) > 8 ? 8 : (int)((SMEM_LIMIT - 1024 - EPI_WARPS * STAGING - 512) / stage_bytes(CG, BN)); }
__host__ __device__ constexpr uint32_t smem_bytes(int CG, int BN){ return 1024 + stage_count(CG, BN) * stage_bytes(CG, BN) + EPI_WARPS * STAGING + 512; }
}

__device__ int g_product_tc_error = 0;                   // set when a bounded wait ran out

struct TcArgs {
    int m, n, k;
    int m_tiles, n_tiles, splits, split_blocks;          // split_blocks: k blocks of 64 in a split
    int whole_tiles;                                     // tiles from here on are taken in two halves of BN / 2 columns (CG == 2)
    int cluster_splits;                                  // > 1: so many CTAs of a cluster share a tile, each with split_blocks of its k, and add up through one another's shared memory
    uint32_t idesc, idesc_half;
    const float* bias;
    const void* add; long long ld_add;
    void* pre; long long ld_pre;
    void* out; long long ld_out, split_stride;           // of EPI_SUM: elements from one split's sums to the next
    float scale;
    int act, accumulate;
    int fast;                                            // rows of the outputs, add and pre start on 16-byte boundaries
    const void* sum_source; long long ld_sum; float* sums; // row sums of A: [splits][m] (or the gradient itself: one split)
    int sums_accumulate;
};

// ---- a tile's cooperating CTAs ------------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t cluster_rank(){ uint32_t r; asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ uint32_t leader_address(const void* p){ uint32_t r; asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(tc::smem_u32(p))); return r; }
__device__ __forceinline__ void cluster_sync(){ asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ float4 peer_load(uint32_t address){      // of a CTA of the cluster
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(address) : "memory");
    return v;
}
__device__ __forceinline__ uint32_t peer_address(const void* p, uint32_t rank){ uint32_t r; asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(tc::smem_u32(p)), "r"(rank)); return r; }
__device__ __forceinline__ void arrive_expect(uint64_t* bar, uint32_t bytes){ asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" :: "r"(tc::smem_u32(bar)), "r"(bytes) : "memory"); }
template <int CG> __device__ __forceinline__ void arrive_at_leader(uint64_t* bar){
    if constexpr(CG == 1) tc::mbar_arrive(bar);
    // what it hands over is tensor memory that has been read (ordered by the fence in front of it), so no store of this warp has to be waited for, as a release to the cluster would
    else asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" :: "r"(leader_address(bar)) : "memory");
}
// a box of a matrix into this CTA's shared memory; its bytes count at the leader's barrier
template <int CG> __device__ __forceinline__ void load_box(void* smem, const CUtensorMap* map, int x, int y, uint64_t* bar){
    if constexpr(CG == 1)
        asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
                     :: "r"(tc::smem_u32(smem)), "l"(map), "r"(tc::smem_u32(bar)), "r"(x), "r"(y) : "memory");
    else
        asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
                     :: "r"(tc::smem_u32(smem)), "l"(map), "r"(leader_address(bar)), "r"(x), "r"(y) : "memory");
}
// One lane of a converged warp. The loops that issue loads and MMAs are run by whole warps and only the instructions themselves by this lane: their operands then stay in uniform
// registers. Run by a single thread, the same loop takes 650 cycles for a stage whatever the tile, more than the MMAs of the largest (512).
__device__ __forceinline__ bool elected(){
    uint32_t one;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
    return one != 0;
}
// a bounded wait of a whole warp, which goes on or gives up together
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity){ return __all_sync(0xffffffffu, tc::mbar_wait_bounded(bar, parity, WAIT_LIMIT)); }
__device__ __forceinline__ void prefetch_map(const CUtensorMap* map){ asm volatile("prefetch.tensormap [%0];" :: "l"(map) : "memory"); }
template <int CG> __device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate){
    if constexpr(CG == 1) tc::mma_f16_ss(d, a, b, idesc, accumulate);
    else asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, {%5, %5, %5, %5, %5, %5, %5, %5}, p;\n\t}"
                      :: "r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(0u) : "memory");
}
// arrives at the barrier (of both CTAs) when all MMAs issued so far have completed
template <int CG> __device__ __forceinline__ void commit(uint64_t* bar){
    if constexpr(CG == 1) tc::commit(bar);
    else asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" :: "r"(tc::smem_u32(bar)), "h"((uint16_t)3) : "memory");
}
template <int CG> __device__ __forceinline__ void tensor_memory_alloc(uint32_t* slot, uint32_t columns){
    if constexpr(CG == 1){ tc::tmem_alloc(slot, columns); tc::tmem_relinquish(); }
    else{
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" :: "r"(tc::smem_u32(slot)), "r"(columns) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
}
template <int CG> __device__ __forceinline__ void tensor_memory_free(uint32_t address, uint32_t columns){
    if constexpr(CG == 1) tc::tmem_dealloc(address, columns);
    else asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" :: "r"(address), "r"(columns) : "memory");
}
// Descriptor of an operand whose rows are contiguous (k_rows), 128-byte swizzle: boxes of 64 rows of the operand x 64 k, [k][128 bytes], 8 k 1024 bytes apart (stride byte
// offset), the next 64 rows of the operand 8192 bytes on (leading byte offset). 16 k further is 2048 bytes.
__device__ __forceinline__ uint64_t make_desc_rows_sw128(uint32_t smem_addr){
    return (uint64_t)((smem_addr >> 4) & 0x3FFF) | (uint64_t)(8192 >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}

struct TileIndex { int m, n, z, half; };                 // half: -1 a whole tile, 0 or 1 a half of it
// Tiles in groups of GROUP rows of tiles, along the rows first: what runs at the same time shares operands in L2 (two rows for the layer's products, whose B are the weights, eight for
// their gradient: 1.5% for 16384 x 4096 x 4096 either way). Behind the whole tiles come those of the last round, in halves where that lets twice as many pairs of CTAs work on them.
template <int GROUP> __device__ __forceinline__ TileIndex tile_index(const TcArgs& a, int t){
    TileIndex i;
    i.half = -1;
    if(t >= a.whole_tiles){ i.half = (t - a.whole_tiles) & 1; t = a.whole_tiles + ((t - a.whole_tiles) >> 1); }
    const int per_split = a.m_tiles * a.n_tiles;
    i.z = t / per_split; t -= i.z * per_split;
    const int group = t / (GROUP * a.n_tiles), first = group * GROUP, rows = min(GROUP, a.m_tiles - first);
    t -= group * GROUP * a.n_tiles;
    i.m = first + t % rows; i.n = t / rows;
    return i;
}

template <typename T> __device__ __forceinline__ uint32_t pack(float lo, float hi);
template <> __device__ __forceinline__ uint32_t pack<__nv_bfloat16>(float lo, float hi){ __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi); return *reinterpret_cast<uint32_t*>(&v); }
template <> __device__ __forceinline__ uint32_t pack<__half>(float lo, float hi){ __half2 v = __floats2half2_rn(lo, hi); return *reinterpret_cast<uint32_t*>(&v); }
template <typename T> __device__ __forceinline__ float2 unpack(uint32_t v);
template <> __device__ __forceinline__ float2 unpack<__nv_bfloat16>(uint32_t v){ return __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&v)); }
template <> __device__ __forceinline__ float2 unpack<__half>(uint32_t v){ return __half22float2(*reinterpret_cast<__half2*>(&v)); }

template <typename T> __device__ __forceinline__ void unpack_chunk(float (&f)[8], const uint4& raw){
    const uint32_t u[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for(int e = 0; e < 4; e++){ const float2 p = unpack<T>(u[e]); f[2 * e] = p.x; f[2 * e + 1] = p.y; }
}
template <typename T> __device__ __forceinline__ uint4 pack_pairs(const float2 (&v)[4]){ return make_uint4(pack<T>(v[0].x, v[0].y), pack<T>(v[1].x, v[1].y), pack<T>(v[2].x, v[2].y), pack<T>(v[3].x, v[3].y)); }
// eight consecutive elements at p (16-byte aligned), of which `count` exist
template <typename T> __device__ __forceinline__ uint4 load_chunk(const T* p, int count){
    if(count >= 8) return *reinterpret_cast<const uint4*>(p);
    union { uint4 v; T e[8]; } u;
    u.v = make_uint4(0, 0, 0, 0);
#pragma unroll
    for(int j = 0; j < 8; j++) if(j < count) u.e[j] = p[j];
    return u.v;
}
template <typename T> __device__ __forceinline__ void store_chunk(T* p, const uint4& v, int count){
    if(count >= 8) *reinterpret_cast<uint4*>(p) = v;
    else{
        union { uint4 v; T e[8]; } u;
        u.v = v;
#pragma unroll
        for(int j = 0; j < 8; j++) if(j < count) p[j] = u.e[j];
    }
}

// A slab: 32 x 32 sums, transposed through shared memory from a lane a row (as tensor memory is read) to accesses along rows of the matrices, so that every global access of the warp
// covers whole sectors. 16-byte piece c of row r lies at piece c ^ (r % 8). A lane a row in global memory too touches 32 lines with every access (4096 x 1024 x 4096 with a residual 44 us,
// this way 39, both with eight warps).
__device__ __forceinline__ void slab_in(uint8_t* slab, const uint32_t (&r)[32], int lane){
    const uint32_t row = tc::smem_u32(slab) + lane * 128 + ((lane & 7) << 4);        // piece 0; the others differ from it in bits 4 to 6
#pragma unroll
    for(int c = 0; c < 8; c++)
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" :: "r"(row ^ (c << 4)), "r"(r[4 * c]), "r"(r[4 * c + 1]), "r"(r[4 * c + 2]), "r"(r[4 * c + 3]) : "memory");
}
__device__ __forceinline__ float4 slab_load(uint32_t address){
    float4 v;
    asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(address) : "memory");
    return v;
}
__device__ __forceinline__ float4 slab_out(const uint8_t* slab, int row, int piece){ return *reinterpret_cast<const float4*>(slab + row * 128 + ((piece ^ (row & 7)) << 4)); }
__device__ __forceinline__ float slab_element(const uint8_t* slab, int row, int column){ return *reinterpret_cast<const float*>(slab + row * 128 + (((column >> 2) ^ (row & 7)) << 4) + (column & 3) * 4); }

// The operands of a slab's epilogue that lie in memory, 16-bit rows on 16-byte boundaries: a lane has eight columns (8 (lane % 4) on) of every eighth row, so that neighbours share a row's
// sectors. WHOLE: all of the slab is inside the matrix.
struct SlabOperands { uint4 add[4], pre[4]; };
template <typename T> __device__ __forceinline__ void fetch_chunks(uint4 (&raw)[4], const T* p, long long ld, int rows, int count){
    if(rows >= 32 && count >= 8)
#pragma unroll
        for(int i = 0; i < 4; i++, p += 8 * ld) raw[i] = *reinterpret_cast<const uint4*>(p);
    else
#pragma unroll
        for(int i = 0; i < 4; i++, p += 8 * ld) if(8 * i < rows && count > 0) raw[i] = load_chunk(p, count);
}
template <typename T, int EPI> __device__ __forceinline__ void fetch_slab(SlabOperands& o, const TcArgs& a, int row0, int col0, int lane){
    const int col = col0 + 8 * (lane & 3), row = row0 + (lane >> 2), count = a.n - col, rows = row0 + 32 <= a.m ? 32 : a.m - row;
    if(a.add) fetch_chunks(o.add, static_cast<const T*>(a.add) + (long long)row * a.ld_add + col, a.ld_add, rows, count);
    if constexpr(EPI == EPI_INPUT) if(a.act != B200RL_ACT_IDENTITY) fetch_chunks(o.pre, static_cast<const T*>(a.pre) + (long long)row * a.ld_pre + col, a.ld_pre, rows, count);
}
template <typename T, int EPI, int ACT, bool WHOLE>
__device__ __forceinline__ void finish_slab(const TcArgs& a, const uint8_t* slab, const SlabOperands& o, const float (&bias)[8], int row0, int col0, int lane){
    const int col = col0 + 8 * (lane & 3), row = row0 + (lane >> 2), count = a.n - col, rows = a.m - row;
    const uint32_t from = tc::smem_u32(slab) + (lane >> 2) * 128 + (((2 * (lane & 3)) ^ (lane >> 2)) << 4);
    T* out = static_cast<T*>(a.out) + (long long)row * a.ld_out + col;
    T* pre = EPI == EPI_FORWARD && a.pre ? static_cast<T*>(a.pre) + (long long)row * a.ld_pre + col : nullptr;
    const float2 scale = both(a.scale);
#pragma unroll
    for(int i = 0; i < 4; i++, out += 8 * a.ld_out){
        const float4 lo = slab_load(from + i * 1024), hi = slab_load((from ^ 16) + i * 1024);
        float2 v[4] = {make_float2(lo.x, lo.y), make_float2(lo.z, lo.w), make_float2(hi.x, hi.y), make_float2(hi.z, hi.w)};
        float add[8];
        const bool there = WHOLE || (8 * i < rows && count > 0);
        const int elements = WHOLE ? 8 : count;
        if constexpr(EPI == EPI_FORWARD){
            if(a.bias)
#pragma unroll
                for(int c = 0; c < 4; c++) v[c] = add2(v[c], make_float2(bias[2 * c], bias[2 * c + 1]));
            if(pre){
                if(there) store_chunk(pre, pack_pairs<T>(v), elements);
                pre += 8 * a.ld_pre;
            }
            activate_pairs<ACT>(v);
            if(a.add){
                unpack_chunk<T>(add, o.add[i]);
#pragma unroll
                for(int c = 0; c < 4; c++) v[c] = fma2(v[c], scale, make_float2(add[2 * c], add[2 * c + 1]));
            }
            else
#pragma unroll
                for(int c = 0; c < 4; c++) v[c] = mul2(v[c], scale);
        }
        else{
            if(a.add){
                unpack_chunk<T>(add, o.add[i]);
#pragma unroll
                for(int c = 0; c < 4; c++) v[c] = add2(v[c], make_float2(add[2 * c], add[2 * c + 1]));
            }
            if constexpr(ACT != B200RL_ACT_IDENTITY){
                unpack_chunk<T>(add, o.pre[i]);
                times_slope_pairs<ACT>(v, add);
            }
        }
        if(there) store_chunk(out, pack_pairs<T>(v), elements);
    }
}
template <typename T, int EPI> __device__ __forceinline__ void finish_whole_or_part(const TcArgs& a, const uint8_t* slab, const SlabOperands& o, int row0, int col, int lane){
    float bias[8];
    if constexpr(EPI == EPI_FORWARD) if(a.bias)
#pragma unroll
        for(int c = 0; c < 8; c++) bias[c] = a.bias[min(col + 8 * (lane & 3) + c, a.n - 1)];
    if(row0 + 32 <= a.m && col + 32 <= a.n){ B200RL_DISPATCH_RESIDUAL_ACT(a.act, (finish_slab<T, EPI, ACT, true>(a, slab, o, bias, row0, col, lane))) }
    else { B200RL_DISPATCH_RESIDUAL_ACT(a.act, (finish_slab<T, EPI, ACT, false>(a, slab, o, bias, row0, col, lane))) }
}
// The same where rows start at odd addresses: a lane has a column. Eight rows at a time, so that their operands are under way together and the places in the slab differ in
// constants; WHOLE: all of the slab's rows are there.
template <typename T, int EPI, int ACT, bool WHOLE>
__device__ __forceinline__ void finish_rows(const TcArgs& a, const uint8_t* slab, int row0, int col, int lane){
    const float bias = EPI == EPI_FORWARD && a.bias ? a.bias[col] : 0.0f;
    const int rows = WHOLE ? 32 : min(32, a.m - row0);
    const T* add_at = a.add ? static_cast<const T*>(a.add) + (long long)row0 * a.ld_add + col : nullptr;
    T* pre_at = a.pre ? static_cast<T*>(a.pre) + (long long)row0 * a.ld_pre + col : nullptr;
    T* out_at = static_cast<T*>(a.out) + (long long)row0 * a.ld_out + col;
    const uint32_t from = tc::smem_u32(slab) + ((lane >> 2) << 4) + (lane & 3) * 4;
    const long long ld_add = a.ld_add, ld_pre = a.ld_pre, ld_out = a.ld_out;
#pragma unroll 1
    for(int r0 = 0; r0 < rows; r0 += 8){
        T add_raw[8], pre_raw[8];
        if(add_at)
#pragma unroll
            for(int r = 0; r < 8; r++, add_at += ld_add) if(WHOLE || r0 + r < rows) add_raw[r] = *add_at;
        if constexpr(EPI == EPI_INPUT && ACT != B200RL_ACT_IDENTITY)
#pragma unroll
            for(int r = 0; r < 8; r++, pre_at += ld_pre) if(WHOLE || r0 + r < rows) pre_raw[r] = *pre_at;
        float x[8];
#pragma unroll
        for(int r = 0; r < 8; r++) asm volatile("ld.shared.f32 %0, [%1];" : "=f"(x[r]) : "r"((from ^ (r << 4)) + (r0 + r) * 128) : "memory");
        float2 v[4] = {make_float2(x[0], x[1]), make_float2(x[2], x[3]), make_float2(x[4], x[5]), make_float2(x[6], x[7])};
        if constexpr(EPI == EPI_FORWARD){
            if(a.bias)
#pragma unroll
                for(int r = 0; r < 4; r++) v[r] = add2(v[r], both(bias));
            if(pre_at)
#pragma unroll
                for(int r = 0; r < 8; r++, pre_at += ld_pre) if(WHOLE || r0 + r < rows) *pre_at = from_float<T>(r & 1 ? v[r / 2].y : v[r / 2].x);
            activate_pairs<ACT>(v);
#pragma unroll
            for(int r = 0; r < 4; r++) v[r] = mul2(v[r], both(a.scale));
        }
        if(add_at)
#pragma unroll
            for(int r = 0; r < 4; r++) v[r] = add2(v[r], make_float2(to_float(add_raw[2 * r]), to_float(add_raw[2 * r + 1])));
        if constexpr(EPI == EPI_INPUT && ACT != B200RL_ACT_IDENTITY){
            float p[8];
#pragma unroll
            for(int r = 0; r < 8; r++) p[r] = to_float(pre_raw[r]);
            times_slope_pairs<ACT>(v, p);
        }
#pragma unroll
        for(int r = 0; r < 8; r++, out_at += ld_out) if(WHOLE || r0 + r < rows) *out_at = from_float<T>(r & 1 ? v[r / 2].y : v[r / 2].x);
    }
}
template <typename T, int EPI>
__device__ __forceinline__ void finish_slab_by_rows(const TcArgs& a, const uint8_t* slab, int row0, int col0, int lane){
    const int col = col0 + lane;
    if(col >= a.n) return;
    if(row0 + 32 <= a.m){ B200RL_DISPATCH_RESIDUAL_ACT(a.act, (finish_rows<T, EPI, ACT, true>(a, slab, row0, col, lane))) }
    else { B200RL_DISPATCH_RESIDUAL_ACT(a.act, (finish_rows<T, EPI, ACT, false>(a, slab, row0, col, lane))) }
}
// A slab of an fp32 result
__device__ __forceinline__ void store_sums(const TcArgs& a, const uint8_t* slab, int z, int row0, int col0, int lane){
    float* out = static_cast<float*>(a.out) + z * a.split_stride;
    if(a.fast && col0 + 32 <= a.n){
#pragma unroll
        for(int i = 0; i < 8; i++){
            const int r = 4 * i + (lane >> 3);
            if(row0 + r >= a.m) continue;
            float4 v = slab_out(slab, r, lane & 7);
            float4* p = reinterpret_cast<float4*>(out + (long long)(row0 + r) * a.ld_out + col0 + 4 * (lane & 7));
            if(a.accumulate){ const float4 q = *p; v.x += q.x; v.y += q.y; v.z += q.z; v.w += q.w; }
            *p = v;
        }
    }
    else if(col0 + lane < a.n){
        const int rows = min(32, a.m - row0);
#pragma unroll 4
        for(int r = 0; r < rows; r++){
            float* p = out + (long long)(row0 + r) * a.ld_out + col0 + lane;
            const float v = slab_element(slab, r, lane);
            *p = a.accumulate ? *p + v : v;
        }
    }
}

template <typename T>
__device__ __forceinline__ void sum_rows(const TcArgs& a, float* shared, int tid, int warp, int lane);

// FAST: 16-bit outputs, add and pre by 16-byte accesses (both epilogues in one kernel take registers from one another: 4096 x 1024 x 4096 with everything 41 us instead of 39)
template <int CG, int BN, bool A_ROWS, bool B_ROWS, typename T, int EPI, bool FAST>
__global__ void __launch_bounds__(THREADS, 1) product_tc_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                                                                const __grid_constant__ TcArgs a){
    constexpr int STAGES = stage_count(CG, BN);
    constexpr uint32_t STAGE = stage_bytes(CG, BN);
    constexpr int GROUPS = BN < 128 ? BN / 32 : 4, CW = BN / GROUPS, SLABS = CW / 32;       // groups of four epilogue warps at work; columns of a warp, slabs of them
    static_assert(CW % 32 == 0);
    extern __shared__ uint8_t smem_raw[];
    uint8_t* base = smem_raw + ((1024u - (tc::smem_u32(smem_raw) & 1023u)) & 1023u);
    uint8_t* staging = base + STAGES * STAGE;
    uint64_t* full = reinterpret_cast<uint64_t*>(staging + EPI_WARPS * STAGING);
    uint64_t *empty = full + STAGES, *acc_full = empty + STAGES, *acc_empty = acc_full + 2;
    uint32_t* slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
    float* sum_buffer = reinterpret_cast<float*>(slot + 4);                  // [2][SUM_COLUMNS]
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t rank = CG == 2 ? cluster_rank() : 0;                 // in a pair
    const int sharers = CG == 1 && EPI != EPI_SUM ? a.cluster_splits : 1, share = sharers > 1 ? (int)cluster_rank() : 0;
    if(tid == 0){
        prefetch_map(&map_a); prefetch_map(&map_b);
        for(int s = 0; s < STAGES; s++){ tc::mbar_init(full + s, 1); tc::mbar_init(empty + s, 1); }
        for(int b = 0; b < 2; b++){ tc::mbar_init(acc_full + b, 1); tc::mbar_init(acc_empty + b, CG * 4 * GROUPS); }
        tc::fence_mbar_init();
    }
    if(warp == 2) tensor_memory_alloc<CG>(slot, 2 * BN);
    tc::fence_before_thread_sync();
    __syncthreads();
    if constexpr(CG == 2) cluster_sync();
    tc::fence_after_thread_sync();
    const uint32_t tmem = *slot;
    after_predecessor();
    const int all = a.m_tiles * a.n_tiles * a.splits, tiles = CG == 2 ? a.whole_tiles + 2 * (all - a.whole_tiles) : all, first_tile = blockIdx.x / (CG * sharers), tile_step = gridDim.x / (CG * sharers);
    const int k_blocks = (a.k - 1) / KB + 1;

    if(warp < 4){
        tc::setmaxnreg_dec<64>();
        if(warp == 0){
            uint32_t it = 0;
            bool ok = true;
            for(int t = first_tile; t < tiles && ok; t += tile_step){
                const TileIndex i = tile_index<EPI == EPI_SUM ? 8 : 2>(a, t);
                const bool half = CG == 2 && i.half >= 0;
                const int m0 = i.m * 128 * CG + (int)rank * 128, n0 = i.n * BN + (half ? i.half * (BN / 2) + (int)rank * (BN / CG / 2) : (int)rank * (BN / CG));
                const uint32_t bytes = half ? STAGE - (STAGE - A_BYTES) / 2 : STAGE;
                const int part = i.z + share, kb_end = min(k_blocks, (part + 1) * a.split_blocks);
                for(int kb = part * a.split_blocks; kb < kb_end; kb++, it++){
                    const uint32_t s = it % STAGES, phase = (it / STAGES) & 1;
                    if(!warp_wait(empty + s, phase ^ 1)){ ok = false; break; }
                    uint8_t* stage = base + s * STAGE;
                    if(elected()){
                        if(rank == 0) arrive_expect(full + s, CG * bytes);
                        if constexpr(A_ROWS){
                            load_box<CG>(stage, &map_a, m0, kb * KB, full + s);
                            load_box<CG>(stage + 8192, &map_a, m0 + 64, kb * KB, full + s);
                        }
                        else load_box<CG>(stage, &map_a, kb * KB, m0, full + s);
#pragma unroll
                        for(int j = 0; j < BN / CG / 64; j++){                // boxes of 64 rows of B either way
                            if(j >= BN / CG / 128 && half) break;
                            if constexpr(B_ROWS) load_box<CG>(stage + A_BYTES + j * 8192, &map_b, n0 + 64 * j, kb * KB, full + s);
                            else load_box<CG>(stage + A_BYTES + j * 8192, &map_b, kb * KB, n0 + 64 * j, full + s);
                        }
                    }
                    __syncwarp();
                }
            }
            // no CTA leaves while its copies or its peer's signals are under way: the last use of every stage has been released
            for(uint32_t s = 0; s < STAGES && s < it; s++){
                const uint32_t last = (it - 1 - s) / STAGES * STAGES + s;         // the last step of this stage
                if(!warp_wait(empty + s, (last / STAGES) & 1)) ok = false;
            }
            if(!ok) g_product_tc_error = 1;
        }
        else if(warp == 1 && rank == 0){
            uint32_t it = 0, acc = 0;
            bool ok = true;
            for(int t = first_tile; t < tiles && ok; t += tile_step){
                const TileIndex i = tile_index<EPI == EPI_SUM ? 8 : 2>(a, t);
                const int part = i.z + share;
                const uint32_t idesc = CG == 2 && i.half >= 0 ? a.idesc_half : a.idesc;
                const int kb_end = min(k_blocks, (part + 1) * a.split_blocks);
                for(int kb0 = part * a.split_blocks; kb0 < kb_end && ok; acc++){
                    const int piece_end = EPI == EPI_SUM ? min(kb_end, kb0 + PIECE / KB) : kb_end;
                    const uint32_t b = acc & 1, d = tmem + b * BN;
                    if(!warp_wait(acc_empty + b, ((acc >> 1) & 1) ^ 1)){ ok = false; break; }
                    tc::fence_after_thread_sync();
                    for(int kb = kb0; kb < piece_end; kb++, it++){
                        const uint32_t s = it % STAGES;
                        if(!warp_wait(full + s, (it / STAGES) & 1)){ ok = false; break; }
                        tc::fence_after_thread_sync();
                        const uint32_t stage = tc::smem_u32(base + s * STAGE);
                        const uint64_t da = A_ROWS ? make_desc_rows_sw128(stage) : tc::make_desc_kmajor_sw128(stage);
                        const uint64_t db = B_ROWS ? make_desc_rows_sw128(stage + A_BYTES) : tc::make_desc_kmajor_sw128(stage + A_BYTES);
                        if(elected()){
#pragma unroll
                            for(int ks = 0; ks < KB / 16; ks++)
                                mma<CG>(d, da + (uint64_t)(ks * (A_ROWS ? 128 : 2)), db + (uint64_t)(ks * (B_ROWS ? 128 : 2)), idesc, (kb > kb0 || ks) ? 1u : 0u);
                            commit<CG>(empty + s);
                            if(kb + 1 == piece_end) commit<CG>(acc_full + b);
                        }
                        __syncwarp();
                    }
                    if(!ok) break;
                    kb0 = piece_end;
                }
            }
            if(!ok) g_product_tc_error = 1;
        }
        else if(EPI == EPI_SUM && warp >= 2 && a.sums) sum_rows<T>(a, sum_buffer, tid - 64, warp - 2, lane);
        __syncwarp();
        if constexpr(CG == 1 && EPI != EPI_SUM) if(sharers > 1){ cluster_sync(); cluster_sync(); }       // as the epilogue warps do
    }
    else{
        tc::setmaxnreg_inc<104>();
        const int w = warp - 4, q = w & 3, group = w >> 2;               // tensor memory lanes 32 q .. +31, columns group CW .. +CW - 1
        const uint32_t lanes = (uint32_t)(q * 32) << 16;
        uint8_t* slab = staging + w * STAGING;
        uint32_t acc = 0;
        bool ok = true;
        for(int t = first_tile; t < tiles && ok && group < GROUPS; t += tile_step){
            const TileIndex i = tile_index<EPI == EPI_SUM ? 8 : 2>(a, t);
            const bool half = CG == 2 && i.half >= 0;                    // a half tile's columns go round all groups too: half the slabs for each
            const int slabs = half ? SLABS / 2 : SLABS, tile_col = group * slabs * 32;
            const int row0 = i.m * 128 * CG + (int)rank * 128 + q * 32, col0 = i.n * BN + (half ? i.half * (BN / 2) : 0) + tile_col;
            if constexpr(EPI == EPI_SUM){
                const int kb_begin = i.z * a.split_blocks, kb_end = min(k_blocks, kb_begin + a.split_blocks);
                const int pieces = (kb_end - kb_begin + PIECE / KB - 1) / (PIECE / KB);
                float sum[SLABS][32];
#pragma unroll
                for(int j = 0; j < SLABS; j++)
#pragma unroll
                    for(int c = 0; c < 32; c++) sum[j][c] = 0.0f;
                for(int p = 0; p < pieces; p++, acc++){
                    const uint32_t b = acc & 1;
                    if(!warp_wait(acc_full + b, (acc >> 1) & 1)){ ok = false; break; }
                    tc::fence_after_thread_sync();
#pragma unroll
                    for(int j = 0; j < SLABS; j++){
                        if(j >= slabs) break;
                        uint32_t r[32];
                        tc::tmem_load_32x32(tmem + lanes + b * BN + tile_col + j * 32, r);
#pragma unroll
                        for(int c = 0; c < 32; c++) sum[j][c] += __uint_as_float(r[c]);
                    }
                    tc::fence_before_thread_sync();
                    __syncwarp();
                    if(lane == 0) arrive_at_leader<CG>(acc_empty + b);
                }
                if(!ok) break;
#pragma unroll
                for(int j = 0; j < SLABS; j++){
                    if(j >= slabs) break;
                    uint32_t r[32];
#pragma unroll
                    for(int c = 0; c < 32; c++) r[c] = __float_as_uint(sum[j][c]);
                    __syncwarp();
                    slab_in(slab, r, lane);
                    __syncwarp();
                    if(row0 < a.m && col0 + 32 * j < a.n) store_sums(a, slab, i.z, row0, col0 + 32 * j, lane);
                }
            }
            else{
                const uint32_t b = acc & 1, phase = (acc >> 1) & 1;
                acc++;
                SlabOperands o;
                if(FAST && sharers == 1) fetch_slab<T, EPI>(o, a, row0, col0, lane);
                if(!warp_wait(acc_full + b, phase)){ ok = false; break; }
                tc::fence_after_thread_sync();
                uint32_t r[32];
                if(sharers > 1){                                         // one tile a cluster: its sums go where the operands were
#pragma unroll
                    for(int j = 0; j < SLABS; j++){
                        tc::tmem_load_32x32(tmem + lanes + b * BN + group * CW + j * 32, r);
                        slab_in(base + (w * SLABS + j) * 4096, r, lane);
                    }
                    break;
                }
#pragma unroll 1
                for(int j = 0; j < slabs; j++){
                    const int col = col0 + j * 32;
                    tc::tmem_load_32x32(tmem + lanes + b * BN + tile_col + j * 32, r);
                    __syncwarp();                                        // the slab before has been read
                    slab_in(slab, r, lane);
                    if(j + 1 == slabs) tc::fence_before_thread_sync();
                    __syncwarp();
                    if(j + 1 == slabs && lane == 0) arrive_at_leader<CG>(acc_empty + b);
                    if constexpr(!FAST){ if(row0 < a.m && col < a.n) finish_slab_by_rows<T, EPI>(a, slab, row0, col, lane); }
                    else{
                        if(row0 >= a.m || col >= a.n) continue;
                        finish_whole_or_part<T, EPI>(a, slab, o, row0, col, lane);
                        if(j + 1 < slabs) fetch_slab<T, EPI>(o, a, row0, col + 32, lane);
                    }
                }
            }
        }
        if(!ok) g_product_tc_error = 1;
        __syncwarp();
        if constexpr(CG == 1 && EPI != EPI_SUM) if(sharers > 1){
            // every CTA's sums are in place; each takes every so many-th slab, adds up the shares in their order and finishes it
            const TileIndex i = tile_index<2>(a, first_tile);
            const int row0 = i.m * 128 + q * 32;
            const bool works = group < GROUPS && row0 < a.m;
            cluster_sync();
            if(works)
#pragma unroll 1
                for(int j = 0; j < SLABS; j++){
                    const int col = i.n * BN + group * CW + j * 32;
                    if((w * SLABS + j) % sharers != share || col >= a.n) continue;
                    SlabOperands o;
                    if constexpr(FAST) fetch_slab<T, EPI>(o, a, row0, col, lane);
                    uint8_t* slab = staging + w * STAGING;
                    __syncwarp();
#pragma unroll 1
                    for(int half = 0; half < 2; half++){
                        float4 sum[4];
                        for(int s = 0; s < sharers; s++){
                            const uint32_t from = peer_address(base + (w * SLABS + j) * 4096 + half * 2048, s);
#pragma unroll
                            for(int c = 0; c < 4; c++){
                                const float4 v = peer_load(from + (c * 32 + lane) * 16);
                                if(s == 0) sum[c] = v;
                                else { sum[c].x += v.x; sum[c].y += v.y; sum[c].z += v.z; sum[c].w += v.w; }
                            }
                        }
#pragma unroll
                        for(int c = 0; c < 4; c++) *reinterpret_cast<float4*>(slab + half * 2048 + (c * 32 + lane) * 16) = sum[c];
                    }
                    __syncwarp();
                    if constexpr(FAST) finish_whole_or_part<T, EPI>(a, slab, o, row0, col, lane);
                    else finish_slab_by_rows<T, EPI>(a, slab, row0, col, lane);
                }
            __syncwarp();
            cluster_sync();                                                  // no CTA leaves while its sums are read
        }
    }
    tc::fence_before_thread_sync();
    __syncthreads();
    if constexpr(CG == 2) cluster_sync();
    tc::fence_after_thread_sync();
    if(warp == 2) tensor_memory_free<CG>(tmem, 2 * BN);
}

// Row sums of A (the bias gradient) by two warps that run beside the products: item = 16 columns of A's matrix over one split of k, a thread a row in 64, four rows of
// loads under way at a time.
template <typename T>
__device__ __forceinline__ void sum_rows(const TcArgs& a, float* shared, int tid, int warp, int lane){
    const int groups = (a.m + SUM_COLUMNS - 1) / SUM_COLUMNS, items = groups * a.splits;
    for(int item = blockIdx.x; item < items; item += gridDim.x){
        const int z = item / groups, c0 = (item - z * groups) * SUM_COLUMNS;
        const long long begin = (long long)z * a.split_blocks * KB, end = min((long long)a.k, begin + (long long)a.split_blocks * KB);
        const T* column = static_cast<const T*>(a.sum_source) + c0;                         // rows 16-byte aligned
        float v[SUM_COLUMNS];
#pragma unroll
        for(int c = 0; c < SUM_COLUMNS; c++) v[c] = 0.0f;
        if(c0 + SUM_COLUMNS <= a.m){
            long long k = begin + tid;
            for(; k + 3 * SUM_THREADS < end; k += 4 * SUM_THREADS){
                uint4 raw[4][2];
#pragma unroll
                for(int i = 0; i < 4; i++)
#pragma unroll
                    for(int h = 0; h < 2; h++) raw[i][h] = *reinterpret_cast<const uint4*>(column + (k + i * SUM_THREADS) * a.ld_sum + 8 * h);
#pragma unroll
                for(int i = 0; i < 4; i++)
#pragma unroll
                    for(int h = 0; h < 2; h++){
                        float e[8];
                        unpack_chunk<T>(e, raw[i][h]);
#pragma unroll
                        for(int c = 0; c < 8; c++) v[8 * h + c] += e[c];
                    }
            }
            for(; k < end; k += SUM_THREADS)
#pragma unroll
                for(int h = 0; h < 2; h++){
                    float e[8];
                    load_elements(column + k * a.ld_sum + 8 * h, e);
#pragma unroll
                    for(int c = 0; c < 8; c++) v[8 * h + c] += e[c];
                }
        }
        else
            for(long long k = begin + tid; k < end; k += SUM_THREADS)
#pragma unroll
                for(int c = 0; c < SUM_COLUMNS; c++) if(c0 + c < a.m) v[c] += to_float(column[k * a.ld_sum + c]);
#pragma unroll
        for(int c = 0; c < SUM_COLUMNS; c++)
#pragma unroll
            for(int o = 16; o > 0; o >>= 1) v[c] += __shfl_xor_sync(0xffffffffu, v[c], o);
        if(lane == 0)
#pragma unroll
            for(int c = 0; c < SUM_COLUMNS; c++) shared[warp * SUM_COLUMNS + c] = v[c];
        tc::named_barrier_sync(1, SUM_THREADS);
        if(tid < SUM_COLUMNS && c0 + tid < a.m){
            const float total = shared[tid] + shared[SUM_COLUMNS + tid];
            float* out = a.sums + (long long)z * a.m + c0 + tid;
            *out = a.sums_accumulate ? *out + total : total;
        }
        tc::named_barrier_sync(1, SUM_THREADS);
    }
}

// ---- finishing partial sums -----------------------------------------------------------------------------------------------------------------------
struct FinishArgs {
    const float* partial; long long ld_partial, split_stride; int splits;
    const float* row_sums;                               // [splits][m]
    TcArgs a;
    float* sums;
};
// out (+)= sum over the splits, in their order, a thread an element
__global__ void __launch_bounds__(256) finish_kernel(FinishArgs f){
    after_predecessor();
    const TcArgs& a = f.a;
    const long long total = (long long)a.m * a.n;
    for(long long i = blockIdx.x * 256ll + threadIdx.x; i < total; i += gridDim.x * 256ll){
        const long long row = i / a.n; const int col = (int)(i - row * a.n);
        const float* p = f.partial + row * f.ld_partial + col;
        float x = 0.0f;
#pragma unroll 4
        for(int z = 0; z < f.splits; z++) x += p[z * f.split_stride];
        float* out = static_cast<float*>(a.out) + row * a.ld_out + col;
        *out = a.accumulate ? *out + x : x;
    }
    if(f.row_sums)
        for(int r = blockIdx.x * 256 + threadIdx.x; r < a.m; r += gridDim.x * 256){
            float x = 0.0f;
            for(int z = 0; z < f.splits; z++) x += f.row_sums[(long long)z * a.m + r];
            f.sums[r] = a.sums_accumulate ? f.sums[r] + x : x;
        }
}

// `count` elements (1 to 8) at any address, 0 behind them: the one or two 16-byte pieces of memory that they lie in (no piece without one of them is touched), shifted into place
__device__ __forceinline__ uint4 unaligned_eight(const uint16_t* p, int count){
    const uint32_t shift = (uint32_t)(reinterpret_cast<uintptr_t>(p) & 15);
    const uint4* piece = reinterpret_cast<const uint4*>(reinterpret_cast<uintptr_t>(p) - shift);
    const uint4 lo = piece[0];
    uint4 hi = make_uint4(0, 0, 0, 0);
    if(shift + 2 * count > 16) hi = piece[1];
    uint32_t w[7] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z};
    uint32_t last = hi.w;
    if(shift & 8){
#pragma unroll
        for(int i = 0; i < 5; i++) w[i] = w[i + 2];
        w[5] = last; w[6] = 0; last = 0;
    }
    if(shift & 4){
#pragma unroll
        for(int i = 0; i < 6; i++) w[i] = w[i + 1];
        w[6] = last;
    }
    uint32_t out[4];
#pragma unroll
    for(int i = 0; i < 4; i++){
        const uint32_t v = shift & 2 ? w[i] >> 16 | w[i + 1] << 16 : w[i];
        out[i] = 2 * i + 1 < count ? v : 2 * i < count ? v & 0xFFFFu : 0u;
    }
    return make_uint4(out[0], out[1], out[2], out[3]);
}

// Rows of 16-bit elements at any address -> rows that start on 16-byte boundaries, eight elements a thread; one operand or both
struct AlignRows { const uint16_t* src; long long ld; uint16_t* dst; long long ld_dst, rows; int cols; };
__global__ void __launch_bounds__(256) align_rows_kernel(AlignRows first, AlignRows second){
    after_predecessor();
    const long long chunks_1 = first.rows * (first.ld_dst / 8), total = chunks_1 + second.rows * (second.ld_dst / 8);
    for(long long i = blockIdx.x * 256ll + threadIdx.x; i < total; i += gridDim.x * 256ll){
        const bool one = i < chunks_1;
        const AlignRows& o = one ? first : second;
        const long long at = one ? i : i - chunks_1;
        const int chunks = (int)(o.ld_dst / 8);
        const long long r = at / chunks; const int c = (int)(at - r * chunks) * 8;
        *reinterpret_cast<uint4*>(o.dst + r * o.ld_dst + c) = unaligned_eight(o.src + r * o.ld + c, min(8, o.cols - c));
    }
}

// ---- host -----------------------------------------------------------------------------------------------------------------------------------------
typedef CUresult (*EncodeTiled)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
static int encode_tiled(EncodeTiled* out){
    static std::atomic<EncodeTiled> cached{nullptr};
    EncodeTiled f = cached.load(std::memory_order_relaxed);
    if(!f){
        void* p = nullptr;
        cudaDriverEntryPointQueryResult found;
        B200RL_CUDA_TRY(cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &found));
        if(found != cudaDriverEntryPointSuccess || !p) return B200RL_ERR_UNSUPPORTED;
        f = reinterpret_cast<EncodeTiled>(p);
        cached.store(f, std::memory_order_relaxed);
    }
    *out = f;
    return B200RL_OK;
}
// an operand: rows x cols 16-bit elements with rows ld elements apart, boxes of box_rows x 64
static int make_map(CUtensorMap* map, CUtensorMapDataType type, const void* p, long long rows, long long cols, long long ld, int box_rows){
    EncodeTiled encode;
    int rc = encode_tiled(&encode);
    if(rc) return rc;
    // the pitch of a single row is not used, but has to be a multiple of 16 bytes
    const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows}, strides[1] = {rows > 1 ? (cuuint64_t)ld * 2 : ((cuuint64_t)cols * 2 + 15) / 16 * 16};
    const cuuint32_t box[2] = {64, (cuuint32_t)box_rows}, steps[2] = {1, 1};
    if(encode(map, type, 2, const_cast<void*>(p), dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS) return B200RL_ERR_UNSUPPORTED;
    return B200RL_OK;
}

struct TcPlan {
    int cg, bn, m_tiles, n_tiles, splits, split_blocks, cluster_splits, whole_tiles;
    bool copy_a, copy_b, partial;
    long long ld_copy_a, ld_copy_b, ld_partial;
    size_t off_b, off_partial, off_sums, bytes;
};
static long long matrix_rows(const Operand& o, int r, int k){ return o.k_rows ? k : r; }
static long long matrix_cols(const Operand& o, int r, int k){ return o.k_rows ? r : k; }
static TcPlan plan_product(const Product& g, int epilogue){
    TcPlan p{};
    const int k_blocks = (g.k - 1) / KB + 1;
    // Shape of the tiles and shares of k, by the cycles that a CTA needs: for a block of 64 k the bytes of its stage at 48 a cycle, what L2 gives a multiprocessor in short
    // products, which the rule is for (long ones of pairs get 58; the MMAs take 128 to 512), for a tile 1,500 until its sums are out, for a shared tile 1,500 and 1,000 a share more. Sharing a tile needs a CTA for each share at the
    // same time. us by tiles of 64 / 128 / 256 columns (* the rule's choice): 1024 x 1024 x 1024 7.8* / 8.9 / 7.7, 128 x 4096 x 4096 13.8 / 12.0* / 16.6, 2048 x 2048 x 2048
    // 37.5 / 23.2 / 16.4*, 4096 x 512 x 512 8.2 / 6.8* / 6.9, 512 x 1024 x 1024 7.6* / 8.7 / 7.6.
    if(g.m > INT_MAX - 1024 || g.n > INT_MAX - 1024 || g.k > INT_MAX - 1024) return p;
    double best = 0.0;
    for(int option = 0; option < 3; option++){
        const int cg = option == 2 ? 2 : 1, bn = option == 0 ? 64 : option == 1 ? 128 : 256, groups = NUM_SMS / cg;
        const long long m_tiles = (g.m - 1) / (128 * cg) + 1, n_tiles = (g.n - 1) / bn + 1, tiles = m_tiles * n_tiles;
        if(tiles > INT_MAX / 64) continue;
        const double block = stage_bytes(cg, bn) / 48.0;
        for(int shares = 1; shares <= (cg == 1 ? 8 : 1); shares *= 2){
            const bool by_cluster = epilogue != EPI_SUM;
            const int most = by_cluster ? (shares == 8 ? 15 : shares == 4 ? 33 : 74) : NUM_SMS / shares;     // clusters that are resident together
            if(shares > 1 && (tiles > most || k_blocks < 2 * shares)) break;
            const int blocks = (k_blocks - 1) / shares + 1;
            const long long whole = tiles * shares / groups, rest = tiles * shares % groups;
            const double rounds = whole + (rest == 0 ? 0.0 : cg == 2 && whole > 0 && 2 * rest <= groups ? 0.75 : 1.0);     // a half tile loads all of A
            const double cycles = rounds * (blocks * block + 1500.0) + (shares == 1 ? 0.0 : by_cluster ? 1500.0 + 1000.0 * shares : 6000.0);      // the last: a launch and a pass over the partial sums
            if(best == 0.0 || cycles < best){
                best = cycles;
                p.cg = cg; p.bn = bn; p.m_tiles = (int)m_tiles; p.n_tiles = (int)n_tiles; p.split_blocks = blocks;
                p.splits = by_cluster ? 1 : (k_blocks - 1) / blocks + 1;
                p.cluster_splits = by_cluster ? (k_blocks - 1) / blocks + 1 : 1;
            }
        }
    }
    if(epilogue == EPI_SUM && p.cg == 1){
        // long sums of few tiles: as many splits as fill the device, a piece each at the least
        const long long tiles = (long long)p.m_tiles * p.n_tiles;
        const long long most = (k_blocks - 1) / (PIECE / KB) + 1, fill = NUM_SMS / tiles;
        const long long splits = fill < most ? fill : most;
        if(splits > p.splits){
            p.split_blocks = (int)((k_blocks - 1) / splits + 1);
            p.splits = (k_blocks - 1) / p.split_blocks + 1;
        }
    }
    if(p.cg == 0) return p;                                              // more tiles than any memory holds
    const long long all = (long long)p.m_tiles * p.n_tiles * p.splits, last = all % (NUM_SMS / 2);
    p.whole_tiles = (int)(p.cg == 2 && 2 * last <= NUM_SMS / 2 ? all - last : all);
    // operands that TMA cannot address are copied
    p.copy_a = !rows_aligned(g.a.p, g.a.ld, 2) && !(matrix_rows(g.a, g.m, g.k) <= 1 && reinterpret_cast<uintptr_t>(g.a.p) % 16 == 0);
    p.copy_b = !rows_aligned(g.b.p, g.b.ld, 2) && !(matrix_rows(g.b, g.n, g.k) <= 1 && reinterpret_cast<uintptr_t>(g.b.p) % 16 == 0);
    p.partial = p.splits > 1;
    p.ld_copy_a = (matrix_cols(g.a, g.m, g.k) + 7) / 8 * 8;
    p.ld_copy_b = (matrix_cols(g.b, g.n, g.k) + 7) / 8 * 8;
    p.ld_partial = (g.n + 31) / 32 * 32;
    size_t at = 0;
    auto take = [&](bool wanted, size_t bytes){ const size_t here = at; if(wanted) at += (bytes + 255) / 256 * 256; return here; };
    take(p.copy_a, 2 * (size_t)p.ld_copy_a * matrix_rows(g.a, g.m, g.k));
    p.off_b = take(p.copy_b, 2 * (size_t)p.ld_copy_b * matrix_rows(g.b, g.n, g.k));
    p.off_partial = take(p.partial, sizeof(float) * (size_t)p.ld_partial * g.m * p.splits);
    p.off_sums = take(p.splits > 1 && epilogue == EPI_SUM, sizeof(float) * (size_t)g.m * p.splits);
    p.bytes = at;
    return p;
}
size_t product_tc_workspace_bytes(const Product& g, int epilogue){ return plan_product(g, epilogue).bytes; }

template <int CG, int BN, bool A_ROWS, bool B_ROWS, typename T, int EPI, bool FAST>
static int launch_tc(const CUtensorMap (&maps)[2], const TcArgs& a, cudaStream_t s){
    auto* kernel = product_tc_kernel<CG, BN, A_ROWS, B_ROWS, T, EPI, FAST>;
    static std::atomic<int> groups[MAX_DEVICES];           // tiles that run at the same time: 0 until the kernel is set up on the device
    int dev = 0, sms = 0;
    int rc = current_device(&dev);
    if(rc || (rc = sm_count(&sms))) return rc;
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute attr[2];
    const int cluster = CG * a.cluster_splits;
    attr[0].id = cudaLaunchAttributeClusterDimension; attr[0].val.clusterDim.x = cluster; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization; attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.blockDim = THREADS; cfg.dynamicSmemBytes = smem_bytes(CG, BN); cfg.stream = s; cfg.attrs = attr; cfg.numAttrs = 1;
    int most = groups[dev].load(std::memory_order_acquire);
    if(most == 0){
        B200RL_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem_bytes(CG, BN)));
        most = sms;
        if(CG > 1){
            cfg.gridDim = sms / CG * CG;
            B200RL_CUDA_TRY(cudaOccupancyMaxActiveClusters(&most, kernel, &cfg));
            if(most < 1) return B200RL_ERR_UNSUPPORTED;
        }
        groups[dev].store(most, std::memory_order_release);
    }
    // a tile that is shared has a cluster of its own; else as many CTAs (or pairs) as run at the same time take the tiles in turn
    const long long all = (long long)a.m_tiles * a.n_tiles * a.splits, tiles = 2 * all - a.whole_tiles;
    cfg.gridDim = (unsigned)(a.cluster_splits > 1 ? tiles * cluster : CG * (tiles < most ? tiles : most));
    cfg.numAttrs = 2;
    B200RL_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, maps[0], maps[1], a));
    return B200RL_OK;
}
template <bool A_ROWS, bool B_ROWS, typename T, int EPI, bool FAST>
static int launch_tile(const TcPlan& p, const CUtensorMap (&maps)[2], const TcArgs& a, cudaStream_t s){
    if(p.cg == 2) return launch_tc<2, 256, A_ROWS, B_ROWS, T, EPI, FAST>(maps, a, s);
    if(p.bn == 128) return launch_tc<1, 128, A_ROWS, B_ROWS, T, EPI, FAST>(maps, a, s);
    return launch_tc<1, 64, A_ROWS, B_ROWS, T, EPI, FAST>(maps, a, s);
}
static int launch_finish(const FinishArgs& f, cudaStream_t s){
    const long long blocks = ((long long)f.a.m * f.a.n + 255) / 256;
    B200RL_CUDA_TRY(launch_after(finish_kernel, dim3((unsigned)(blocks < NUM_SMS * 8 ? blocks : NUM_SMS * 8)), dim3(256), 0, s, f));
    return B200RL_OK;
}

template <typename T>
static int product_tc_typed(const Product& g, int type, int epilogue, void* workspace, size_t workspace_bytes, cudaStream_t s){
    const TcPlan p = plan_product(g, epilogue);
    if(p.cg == 0) return B200RL_ERR_UNSUPPORTED;
    if(p.bytes && (!workspace || reinterpret_cast<uintptr_t>(workspace) % 16 || workspace_bytes < p.bytes)) return B200RL_ERR_INVALID_ARGUMENT;
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    Operand A = g.a, B = g.b;
    int rc;
    if(p.copy_a || p.copy_b){
        AlignRows copies[2] = {};
        int n = 0;
        auto copy = [&](Operand& o, int r, void* dst, long long ld_dst){
            copies[n++] = {static_cast<const uint16_t*>(o.p), o.ld, static_cast<uint16_t*>(dst), ld_dst, matrix_rows(o, r, g.k), (int)matrix_cols(o, r, g.k)};
            o.p = dst; o.ld = ld_dst;
        };
        if(p.copy_a) copy(A, g.m, ws, p.ld_copy_a);
        if(p.copy_b) copy(B, g.n, ws + p.off_b, p.ld_copy_b);
        if(n == 1) copies[1] = {nullptr, 0, nullptr, 8, 0, 0};
        const long long blocks = (copies[0].rows * (copies[0].ld_dst / 8) + copies[1].rows * (copies[1].ld_dst / 8) + 255) / 256;
        B200RL_CUDA_TRY(launch_after(align_rows_kernel, dim3((unsigned)(blocks < NUM_SMS * 16 ? blocks : NUM_SMS * 16)), dim3(256), 0, s, copies[0], copies[1]));
    }
    float* partial = reinterpret_cast<float*>(ws + p.off_partial);
    TcArgs a{};
    a.m = g.m; a.n = g.n; a.k = g.k;
    a.m_tiles = p.m_tiles; a.n_tiles = p.n_tiles; a.splits = p.splits; a.split_blocks = p.split_blocks; a.cluster_splits = p.cluster_splits;
    const uint32_t format = type == B200RL_TYPE_BFLOAT16 ? 1u : 0u;
    // fp32 sums, both operands of one type, their k_rows forms, N / 8, M / 16
    a.idesc = 1u << 4 | format << 7 | format << 10 | (A.k_rows ? 1u << 15 : 0u) | (B.k_rows ? 1u << 16 : 0u) | (uint32_t)(p.bn / 8) << 17 | (uint32_t)(128 * p.cg / 16) << 24;
    a.idesc_half = (a.idesc & ~(0x3Fu << 17)) | (uint32_t)(p.bn / 16) << 17;
    a.whole_tiles = p.whole_tiles;
    a.bias = g.bias; a.add = g.add; a.ld_add = g.ld_add; a.pre = g.pre; a.ld_pre = g.ld_pre; a.out = g.out; a.ld_out = g.ld_out;
    a.scale = g.scale; a.act = g.act; a.accumulate = g.accumulate;
    CUtensorMap maps[2] = {};
    const CUtensorMapDataType dt = type == B200RL_TYPE_BFLOAT16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    if((rc = make_map(&maps[0], dt, A.p, matrix_rows(A, g.m, g.k), matrix_cols(A, g.m, g.k), A.ld, A.k_rows ? 64 : 128))) return rc;
    if((rc = make_map(&maps[1], dt, B.p, matrix_rows(B, g.n, g.k), matrix_cols(B, g.n, g.k), B.ld, 64))) return rc;
    FinishArgs f{partial, p.ld_partial, p.ld_partial * (long long)g.m, p.splits, nullptr, a, g.row_sums};
    if(epilogue == EPI_SUM){
        TcArgs b = a;
        if(p.partial){ b.out = partial; b.ld_out = p.ld_partial; b.split_stride = f.split_stride; b.accumulate = 0; }
        b.fast = rows_aligned(b.out, b.ld_out, 4);
        if(g.row_sums){
            b.sum_source = A.p; b.ld_sum = A.ld;
            b.sums = p.splits > 1 ? reinterpret_cast<float*>(ws + p.off_sums) : g.row_sums;
            b.sums_accumulate = p.splits > 1 ? 0 : g.accumulate;
            f.row_sums = p.splits > 1 ? b.sums : nullptr;
            f.a.sums_accumulate = g.accumulate;
        }
        if((rc = launch_tile<true, true, T, EPI_SUM, true>(p, maps, b, s)) || !p.partial) return rc;
        return launch_finish(f, s);
    }
    a.fast = rows_aligned(g.out, g.ld_out, 2) && (!g.add || rows_aligned(g.add, g.ld_add, 2)) && (!g.pre || rows_aligned(g.pre, g.ld_pre, 2));
    if(epilogue == EPI_INPUT) return a.fast ? launch_tile<false, true, T, EPI_INPUT, true>(p, maps, a, s) : launch_tile<false, true, T, EPI_INPUT, false>(p, maps, a, s);
    return a.fast ? launch_tile<false, false, T, EPI_FORWARD, true>(p, maps, a, s) : launch_tile<false, false, T, EPI_FORWARD, false>(p, maps, a, s);
}
int product_tc(const Product& g, int type, int epilogue, void* workspace, size_t workspace_bytes, cudaStream_t s){
    B200RL_DISPATCH_16_BIT_TYPE(type, return (product_tc_typed<T>(g, type, epilogue, workspace, workspace_bytes, s)))
}
int product_tc_error_get(int* word){ B200RL_CUDA_TRY(cudaMemcpyFromSymbol(word, g_product_tc_error, sizeof(int))); return B200RL_OK; }
int product_tc_error_clear(){ const int zero = 0; B200RL_CUDA_TRY(cudaMemcpyToSymbol(g_product_tc_error, &zero, sizeof(int))); return B200RL_OK; }

}  // namespace b200rl
