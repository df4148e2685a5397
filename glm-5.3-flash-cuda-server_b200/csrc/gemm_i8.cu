// gemm_i8.cu -- y[M,N] = sx[m] * sw[n] * (xq[M,K] . W[N,K]^T) on tcgen05.mma kind::i8 (8-bit integers, sums in 32 bits).
//
// The sum of K <= 65536 products of two 8-bit numbers stays below 2^31, so it is exact and its order does not matter; what is
// rounded is the conversion of the sum to f32 and the two multiplications by the scales.
//
// Persistent: one CTA per SM walks items (128 weight rows) x (NT tokens), K in steps of 128.  The accumulators
// D[128 weight rows (lanes), NT tokens (columns)] lie in TMEM, two sets, so that the epilogue of an item overlaps the MMAs of
// the next.  Weights are the operand of 128 rows because a batch may have one token only, and because the lanes of a warp then
// hold consecutive n: stores of a token's outputs are coalesced straight from registers.
//   warp 0      TMA: per step a 128B-swizzled box of weights [128 B x 128 rows] and one of activations [128 B x NT]
//   warp 1      MMA issuer: four tcgen05.mma (K = 32 each) per step; tcgen05.commit frees the stage
//   warp 2      allocates / frees TMEM
//   warps 4-11  epilogue: two groups of four warps (one per TMEM lane quadrant) take alternate 16-token chunks
// Where the items would leave SMs idle, a cluster of CTAs shares one item (SPLIT): each takes a part of K, leaves its sums in its own
// shared memory, and adds and writes its share of the tokens over distributed shared memory; two CTAs per SM.
// Behind the quantiser of its own call (`early`) a kernel starts when every CTA of the quantiser has returned from its dependency wait.
// What ran before has ended then, so TMEM is taken while the quantiser still runs.  No input is read before the kernel's own
// dependency wait, the weights neither: only that wait makes an earlier kernel's writes visible.
// Rows past N or M and columns past K come as zero from the tensor maps.  Every wait is bounded (tma_pipe.cuh).
//
// Bound by what an SM takes in: between the first and the last step of an item 50 to 70 bytes a clock (time stamps; 301 rows x [8192 x 4096], whose
// weights come out of L2 for the second tile of tokens, 70; 150 x [12288 x 4096] 60), where pairs with 256 tokens a tile need 64 to keep the matrix
// instructions busy.  Few tokens are bound by the weights' stream from HBM (24 rows x [4096 x 12288] on finished rows 12.5 us: 7.0 from the first
// step to the last, 2.5 for the two cluster barriers and the sums), 2048 rows by the matrix instructions and the power that they draw ([12288 x 4096]
// on finished rows 71 us, 2.91 POP/s, in a short run; with the quantiser 75, and 89 in a long run).
#include "b200_internal.h"
#include "umma_mxf4.cuh"
#include <cuda.h>
#include <cuda_bf16.h>
#include <cooperative_groups.h>

namespace b200 {
namespace cg = cooperative_groups;

constexpr int GI_THREADS = 384;
constexpr int GI_MAX_STAGES = 12;
constexpr int GI_PREFETCH = 2;                     // K steps asked into L2 behind a quantiser
constexpr int GI_MAX_NT = 256, GI_MAX_SPLIT = 8;
constexpr uint32_t GI_A_BYTES = 16384;
constexpr size_t GI_STATIC = 4096;                 // static shared memory, at most
constexpr size_t GI_SMEM = 227 * 1024 - GI_STATIC, GI_SMEM_SPLIT = 113 * 1024 - GI_STATIC;

struct GiParams {
    void* y; const float* sw; const float* sx; unsigned int* status;
    int M, N, nst, NT, n_jobs, total, stages, split, tmem_cols, early;
};

__device__ __forceinline__ void gi_prefetch(const void* map, int x, int y) {
    asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global [%0, {%1, %2}];" :: "l"(map), "r"(x), "r"(y) : "memory");
}

__device__ __forceinline__ void gi_store(void* y, size_t o, int acc, float sx, float sw, bool bf16) {
    const float v = __fmul_rn(__fmul_rn(__int2float_rn(acc), sx), sw);
    if (bf16) static_cast<__nv_bfloat16*>(y)[o] = __float2bfloat16_rn(v);
    else static_cast<float*>(y)[o] = v;
}

// Sixteen tokens' outputs of this lane's weight row: y + j * N, j < left.  All sixteen at once where they exist: with a test for
// each, one waits for the other (the epilogue of 160 tokens: 5800 clocks, 3700 so).
template <bool BF16>
__device__ __forceinline__ void gi_store16(void* y, size_t o, int N, const float (&d)[16], const float* sx, float sw, int left) {
    float v[16];
    #pragma unroll
    for (int j = 0; j < 16; j += 4) {
        const float4 f = *reinterpret_cast<const float4*>(sx + j);
        v[j] = __fmul_rn(__fmul_rn(__int2float_rn(__float_as_int(d[j])), f.x), sw);
        v[j + 1] = __fmul_rn(__fmul_rn(__int2float_rn(__float_as_int(d[j + 1])), f.y), sw);
        v[j + 2] = __fmul_rn(__fmul_rn(__int2float_rn(__float_as_int(d[j + 2])), f.z), sw);
        v[j + 3] = __fmul_rn(__fmul_rn(__int2float_rn(__float_as_int(d[j + 3])), f.w), sw);
    }
    if (BF16) {
        __nv_bfloat16* q = static_cast<__nv_bfloat16*>(y) + o;
        if (left >= 16) {
            #pragma unroll
            for (int j = 0; j < 16; ++j, q += N) *q = __float2bfloat16_rn(v[j]);
        } else {
            #pragma unroll
            for (int j = 0; j < 16; ++j, q += N) if (j < left) *q = __float2bfloat16_rn(v[j]);
        }
    } else {
        float* q = static_cast<float*>(y) + o;
        if (left >= 16) {
            #pragma unroll
            for (int j = 0; j < 16; ++j, q += N) *q = v[j];
        } else {
            #pragma unroll
            for (int j = 0; j < 16; ++j, q += N) if (j < left) *q = v[j];
        }
    }
}

template <bool BF16, bool SPLIT>
__global__ void __launch_bounds__(GI_THREADS, SPLIT ? 2 : 1)
k_gemm_i8(const __grid_constant__ GiParams p, const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x) {
    extern __shared__ __align__(1024) unsigned char smem[];
    __shared__ uint64_t full_bar[GI_MAX_STAGES], empty_bar[GI_MAX_STAGES], acc_full[2], acc_empty[2];
    __shared__ uint32_t tmem_base_s;
    __shared__ __align__(16) float sxs[2][GI_MAX_NT];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int S = p.stages, NT = p.NT;
    const uint32_t slot = GI_A_BYTES + (uint32_t)NT * 128u;
    // SPLIT: one item per cluster, this CTA's part of its K steps; otherwise every gridDim-th item, all of its steps
    const int rank = SPLIT ? (int)cg::this_cluster().block_rank() : 0;
    const int first = SPLIT ? (int)blockIdx.x / p.split : (int)blockIdx.x, stride = SPLIT ? p.total : (int)gridDim.x;
    const int k_first = SPLIT ? p.nst * rank / p.split : 0, nst = SPLIT ? p.nst * (rank + 1) / p.split - k_first : p.nst;
    if (warp == 1) {
        if (lane < S) { mbar_init(smem_u32(&full_bar[lane]), 1); mbar_init(smem_u32(&empty_bar[lane]), 1); }
        if (lane < 2) { mbar_init(smem_u32(&acc_full[lane]), 1); mbar_init(smem_u32(&acc_empty[lane]), 8); }
        mbar_fence_init();
    }
    if (tid == 0) asm volatile("prefetch.tensormap [%0];\n prefetch.tensormap [%1];" :: "l"(&map_w), "l"(&map_x) : "memory");
    __syncthreads();
    if (!p.early) pdl_wait();
    const int n_items = (p.total - first + stride - 1) / stride;      // the grid is no larger than the number of items
    const uint32_t pad = (1024u - (smem_u32(smem) & 1023u)) & 1023u, ring0 = smem_u32(smem) + pad;
    const uint32_t full0 = smem_u32(&full_bar[0]), empty0 = smem_u32(&empty_bar[0]);

    if (warp == 0) {
        // While the quantiser runs the first weights are asked into L2.  Nothing is read: L2 is where an earlier kernel's writes go, too.
        // (us with 0, 2, 4 and 12 steps: 24 rows x [4096 x 12288] 15.2, 14.8, 14.9, 14.8; 4 rows x [4096 x 12288] 14.0, 13.7, 13.6, 14.0;
        // 777 x [5003 x 2051] in pairs 18.2, 18.3, 18.3, 18.9; 64 x [4096 x 4096] - , 10.4, 10.5, 10.2.)
        if (p.early) {
            if (elect_one())
                for (int it = 0; it < min(GI_PREFETCH, nst); ++it) gi_prefetch(&map_w, (k_first + it) * 128, first / p.n_jobs * 128);
            __syncwarp();
            pdl_wait();
        }
        int s = 0; uint32_t ph = 1;
        for (int i = 0; i < n_items; ++i) {
            const int q = first + i * stride, tile = q / p.n_jobs, job = q - tile * p.n_jobs;
            for (int it = 0; it < nst; ++it) {
                mbar_wait_spin(empty0 + s * 8, ph, p.status, 16);
                if (elect_one()) {
                    const uint32_t bar = full0 + s * 8, dst = ring0 + (uint32_t)s * slot;
                    mbar_expect_tx(bar, slot);
                    gx_tma_2d(dst, &map_w, (k_first + it) * 128, tile * 128, bar);
                    gx_tma_2d(dst + GI_A_BYTES, &map_x, (k_first + it) * 128, job * NT, bar);
                }
                __syncwarp();
                if (++s == S) { s = 0; ph ^= 1; }
            }
        }
        // The commits that free the stages arrive asynchronously: wait for the last one of every stage, or it could
        // land in the shared memory of the next CTA on this SM.
        for (int k = 0; k < S; ++k) {
            mbar_wait_spin(empty0 + s * 8, ph, p.status, 17);
            if (++s == S) { s = 0; ph ^= 1; }
        }
    } else if (warp == 2) {
        // TMEM is taken after the kernel before has ended (`early`: one that takes none is left) and before the kernel after may start:
        // a kernel that held the columns while it waits for another that wants them on the same SM would wait for good.
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" :: "r"(smem_u32(&tmem_base_s)), "r"(p.tmem_cols));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
        gx_fence_before();
        pdl_launch_dependents();
        asm volatile("bar.arrive 2, 320;" ::: "memory");
    } else if (warp == 1) {
        named_sync(2, 320);                            // TMEM is there: this warp and the epilogue's
        gx_fence_after();
        const uint32_t tmem = tmem_base_s;
        // D s32 (2), A and B s8 (1), both K-major
        const uint32_t idesc = (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(NT >> 3) << 17) | ((128u >> 4) << 24);
        const uint64_t d0 = gx_desc(ring0);
        int s = 0; uint32_t ph = 0;
        for (int i = 0; i < n_items; ++i) {
            const int buf = i & 1, use = i >> 1;
            if (use > 0) mbar_wait_spin(smem_u32(&acc_empty[buf]), (use - 1) & 1, p.status, 18);
            const uint32_t tD = tmem + (uint32_t)(buf * NT);
            for (int it = 0; it < nst; ++it) {
                mbar_wait_spin(full0 + s * 8, ph, p.status, 19);
                gx_fence_after();
                if (elect_one()) {
                    const uint64_t dA = d0 + (uint64_t)(((uint32_t)s * slot) >> 4), dB = dA + (GI_A_BYTES >> 4);
                    #pragma unroll
                    for (int kb = 0; kb < 4; ++kb)
                        asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
                                     " tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n}"
                                     :: "r"(tD), "l"(dA + kb * 2), "l"(dB + kb * 2), "r"(idesc), "r"((uint32_t)(it | kb)) : "memory");
                    gx_commit(empty0 + s * 8);
                    if (it == nst - 1) gx_commit(smem_u32(&acc_full[buf]));
                }
                __syncwarp();
                if (++s == S) { s = 0; ph ^= 1; }
            }
        }
    } else if (warp >= 4) {
        const int te = tid - 128, grp = te >> 7, q4 = warp & 3;
        named_sync(2, 320);
        gx_fence_after();
        const uint32_t tmem = tmem_base_s;
        const uint32_t tq = tmem + ((uint32_t)(q4 * 32) << 16);
        if (p.early) pdl_wait();                       // the tokens' scales
        for (int i = 0; i < n_items; ++i) {
            const int q = first + i * stride, tile = q / p.n_jobs, m0 = (q - tile * p.n_jobs) * NT, rows = min(NT, p.M - m0);
            const int buf = i & 1, row = tile * 128 + q4 * 32 + lane;
            if (te < rows) sxs[buf][te] = p.sx[m0 + te];
            const float sw = row < p.N ? p.sw[row] : 0.f;
            named_sync(1, 256);
            mbar_wait_spin(smem_u32(&acc_full[buf]), (i >> 1) & 1, p.status, 20);
            gx_fence_after();
            for (int c0 = grp * 16; c0 < rows; c0 += 32) {
                float d[16];
                gx_ld16(tq + (uint32_t)(buf * NT + c0), d);
                asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                if (SPLIT) {                           // sums [token][128 rows], where the operands were
                    int* o = reinterpret_cast<int*>(smem + pad) + c0 * 128 + q4 * 32 + lane;
                    #pragma unroll
                    for (int j = 0; j < 16; ++j) o[j * 128] = __float_as_int(d[j]);
                } else if (row < p.N) gi_store16<BF16>(p.y, (size_t)(m0 + c0) * p.N + row, p.N, d, &sxs[buf][c0], sw, rows - c0);
            }
            gx_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&acc_empty[buf]));
        }
    }
    gx_fence_before();
    __syncwarp();
    if (SPLIT) {
        cg::cluster_group cluster = cg::this_cluster();
        cluster.sync();
        const int tile = first / p.n_jobs, m0 = (first - tile * p.n_jobs) * NT, rows = min(NT, p.M - m0);
        const int c1 = rows * (rank + 1) / p.split;
        const int n = tile * 128 + (tid & 127);
        const float sw = n < p.N ? p.sw[n] : 0.f;
        const int* part = reinterpret_cast<const int*>(smem + pad) + (tid & 127);
        for (int c = rows * rank / p.split + (tid >> 7); c < c1; c += GI_THREADS / 128) {
            int v[GI_MAX_SPLIT];
            #pragma unroll
            for (int r = 0; r < GI_MAX_SPLIT; ++r) v[r] = r < p.split ? cluster.map_shared_rank(part, r)[c * 128] : 0;
            int acc = 0;
            #pragma unroll
            for (int r = 0; r < GI_MAX_SPLIT; ++r) acc += v[r];
            if (n < p.N) gi_store(p.y, (size_t)(m0 + c) * p.N + n, acc, sxs[0][c], sw, BF16);
        }
        cluster.sync();
    } else __syncthreads();
    if (warp == 2) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" :: "r"(tmem_base_s), "r"(p.tmem_cols));
}

// ---- many tokens: two CTAs of a cluster share a tile of 256 weight rows x NT <= 256 tokens (cta_group::2) -------------------
// One CTA's tile of 128 x 256 takes in 48 KB per step of 512 clocks of MMA, 94 bytes per clock: more than an SM's share of L2.  The pair's
// CTAs bring 128 weight rows and half of the tokens each, 32 KB.  The first CTA issues the MMAs for both; both load into their own
// shared memory and signal the first one's barrier; a commit frees the stage in both.  Plain loads, no multicast.
__device__ __forceinline__ uint32_t gi_mapa(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ void gi_tma_pair(uint32_t dst, const void* map, int x, int y, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                 :: "r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar) : "memory");
}
__device__ __forceinline__ void gi_commit_pair(uint32_t bar) {         // arrives on the barrier at this offset in both CTAs
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                 :: "r"(bar), "h"((uint16_t)3) : "memory");
}
__device__ __forceinline__ void gi_arrive_remote(uint32_t bar) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" :: "r"(bar) : "memory");
}

template <bool BF16>
__global__ void __launch_bounds__(GI_THREADS, 1) __cluster_dims__(2, 1, 1)
k_gemm_i8_pair(const __grid_constant__ GiParams p, const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x) {
    extern __shared__ __align__(1024) unsigned char smem[];
    __shared__ uint64_t full_bar[GI_MAX_STAGES], empty_bar[GI_MAX_STAGES], acc_full[2], acc_empty[2], peer_tmem;
    __shared__ uint32_t tmem_base_s;
    __shared__ __align__(16) float sxs[2][GI_MAX_NT];
    cg::cluster_group cluster = cg::this_cluster();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int S = p.stages, NT = p.NT, nst = p.nst, rank = (int)cluster.block_rank();
    const uint32_t slot = GI_A_BYTES + (uint32_t)NT * 64u;
    if (warp == 1) {
        if (lane < S) { mbar_init(smem_u32(&full_bar[lane]), 1); mbar_init(smem_u32(&empty_bar[lane]), 1); }
        if (lane < 2) { mbar_init(smem_u32(&acc_full[lane]), 1); mbar_init(smem_u32(&acc_empty[lane]), 16); }
        if (lane == 0) mbar_init(smem_u32(&peer_tmem), 1);
        mbar_fence_init();
    }
    if (tid == 0) asm volatile("prefetch.tensormap [%0];\n prefetch.tensormap [%1];" :: "l"(&map_w), "l"(&map_x) : "memory");
    __syncwarp();
    cluster.sync();                                    // both CTAs' barriers stand
    if (!p.early) pdl_wait();
    const int first = blockIdx.x >> 1, stride = gridDim.x >> 1;
    const int n_items = (p.total - first + stride - 1) / stride;
    const uint32_t ring0 = smem_u32(smem) + ((1024u - (smem_u32(smem) & 1023u)) & 1023u);
    const uint32_t full0 = smem_u32(&full_bar[0]), empty0 = smem_u32(&empty_bar[0]);

    if (warp == 0) {
        const uint32_t lead0 = gi_mapa(full0, 0);
        if (p.early) {                                 // as above
            if (elect_one())
                for (int it = 0; it < min(GI_PREFETCH, nst); ++it) gi_prefetch(&map_w, it * 128, first / p.n_jobs * 256 + rank * 128);
            __syncwarp();
            pdl_wait();
        }
        int s = 0; uint32_t ph = 1;
        for (int i = 0; i < n_items; ++i) {
            const int q = first + i * stride, tile = q / p.n_jobs, job = q - tile * p.n_jobs;
            for (int it = 0; it < nst; ++it) {
                mbar_wait_spin(empty0 + s * 8, ph, p.status, 16);
                if (elect_one()) {
                    const uint32_t bar = lead0 + s * 8, dst = ring0 + (uint32_t)s * slot;
                    if (rank == 0) mbar_expect_tx(full0 + s * 8, 2 * slot);          // of both CTAs
                    gi_tma_pair(dst, &map_w, it * 128, tile * 256 + rank * 128, bar);
                    gi_tma_pair(dst + GI_A_BYTES, &map_x, it * 128, job * NT + rank * (NT / 2), bar);
                }
                __syncwarp();
                if (++s == S) { s = 0; ph ^= 1; }
            }
        }
        for (int k = 0; k < S; ++k) {                  // the last commits have arrived
            mbar_wait_spin(empty0 + s * 8, ph, p.status, 17);
            if (++s == S) { s = 0; ph ^= 1; }
        }
    } else if (warp == 2) {                            // as above
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" :: "r"(smem_u32(&tmem_base_s)), "r"(p.tmem_cols));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::);
        gx_fence_before();
        pdl_launch_dependents();
        if (rank && lane == 0) gi_arrive_remote(gi_mapa(smem_u32(&peer_tmem), 0));
        __syncwarp();
        asm volatile("bar.arrive 2, 320;" ::: "memory");
    } else if (warp == 1) {
        named_sync(2, 320);
        gx_fence_after();
        const uint32_t tmem = tmem_base_s;
        if (rank == 0) {
            mbar_wait_spin(smem_u32(&peer_tmem), 0, p.status, 31);      // the other CTA has its columns
            const uint32_t idesc = (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(NT >> 3) << 17) | ((256u >> 4) << 24);
            const uint64_t d0 = gx_desc(ring0);
            int s = 0; uint32_t ph = 0;
            for (int i = 0; i < n_items; ++i) {
                const int buf = i & 1, use = i >> 1;
                if (use > 0) mbar_wait_spin(smem_u32(&acc_empty[buf]), (use - 1) & 1, p.status, 18);
                const uint32_t tD = tmem + (uint32_t)(buf * NT);
                for (int it = 0; it < nst; ++it) {
                    mbar_wait_spin(full0 + s * 8, ph, p.status, 19);
                    gx_fence_after();
                    if (elect_one()) {
                        const uint64_t dA = d0 + (uint64_t)(((uint32_t)s * slot) >> 4), dB = dA + (GI_A_BYTES >> 4);
                        #pragma unroll
                        for (int kb = 0; kb < 4; ++kb)
                            asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
                                         " tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n}"
                                         :: "r"(tD), "l"(dA + kb * 2), "l"(dB + kb * 2), "r"(idesc), "r"((uint32_t)(it | kb)) : "memory");
                        gi_commit_pair(empty0 + s * 8);
                        if (it == nst - 1) gi_commit_pair(smem_u32(&acc_full[buf]));
                    }
                    __syncwarp();
                    if (++s == S) { s = 0; ph ^= 1; }
                }
            }
        }
    } else if (warp >= 4) {
        const int te = tid - 128, grp = te >> 7, q4 = warp & 3;
        named_sync(2, 320);
        gx_fence_after();
        const uint32_t tmem = tmem_base_s;
        const uint32_t tq = tmem + ((uint32_t)(q4 * 32) << 16);
        const uint32_t done = gi_mapa(smem_u32(&acc_empty[0]), 0);
        if (p.early) pdl_wait();                       // the tokens' scales
        for (int i = 0; i < n_items; ++i) {
            const int q = first + i * stride, tile = q / p.n_jobs, m0 = (q - tile * p.n_jobs) * NT, rows = min(NT, p.M - m0);
            const int buf = i & 1, row = tile * 256 + rank * 128 + q4 * 32 + lane;
            if (te < rows) sxs[buf][te] = p.sx[m0 + te];
            const float sw = row < p.N ? p.sw[row] : 0.f;
            named_sync(1, 256);
            mbar_wait_spin(smem_u32(&acc_full[buf]), (i >> 1) & 1, p.status, 20);
            gx_fence_after();
            for (int c0 = grp * 16; c0 < rows; c0 += 32) {
                float d[16];
                gx_ld16(tq + (uint32_t)(buf * NT + c0), d);
                asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                if (row < p.N) gi_store16<BF16>(p.y, (size_t)(m0 + c0) * p.N + row, p.N, d, &sxs[buf][c0], sw, rows - c0);
            }
            gx_fence_before();
            __syncwarp();
            if (lane == 0) gi_arrive_remote(done + buf * 8);
        }
    }
    gx_fence_before();
    __syncwarp();
    cluster.sync();                                    // nothing of the other CTA's is under way to this one any more
    if (warp == 2) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" :: "r"(tmem_base_s), "r"(p.tmem_cols));
}

template <bool BF16>
static int gi_launch_pair(GiParams& p, const b200_i8_rows* W, const b200_i8_rows* x, int K, cudaStream_t s) {
    CUtensorMap mw, mx;
    const size_t pitch = i8_pitch(K);
    if (!tmap_u8_pitched(&mw, W->q, (size_t)p.N, (size_t)K, pitch, 128, 128, true, true) ||
        !tmap_u8_pitched(&mx, x->q, (size_t)p.M, (size_t)K, pitch, 128, p.NT / 2, true, true)) return B200_ENOTIMPL;
    auto kern = k_gemm_i8_pair<BF16>;
    const size_t slot = GI_A_BYTES + (size_t)p.NT * 64;
    static bool ready[64] = {};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return launch_failed("gemm_i8: cudaGetDevice");
    if (dev < 0 || dev >= 64 || !ready[dev]) {
        if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)GI_SMEM) != cudaSuccess)
            return launch_failed("gemm_i8: cudaFuncSetAttribute");
        if (dev >= 0 && dev < 64) ready[dev] = true;
    }
    p.stages = (int)std::min<size_t>(GI_MAX_STAGES, (GI_SMEM - 1024) / slot);
    p.tmem_cols = 32;
    while (p.tmem_cols < 2 * p.NT) p.tmem_cols *= 2;
    if (launch_pdl(kern, dim3(2 * std::min(p.total, sm_count() / 2)), dim3(GI_THREADS), 1024 + p.stages * slot, s, p, mw, mx) != cudaSuccess)
        return launch_failed("k_gemm_i8_pair");
    return check_launch("k_gemm_i8_pair");
}

template <bool BF16, bool SPLIT>
static int gi_launch(GiParams& p, const b200_i8_rows* W, const b200_i8_rows* x, int K, cudaStream_t s) {
    CUtensorMap mw, mx;
    const size_t pitch = i8_pitch(K);
    if (!tmap_u8_pitched(&mw, W->q, (size_t)p.N, (size_t)K, pitch, 128, 128, true, true) ||
        !tmap_u8_pitched(&mx, x->q, (size_t)p.M, (size_t)K, pitch, 128, p.NT, true, true)) return B200_ENOTIMPL;
    auto kern = k_gemm_i8<BF16, SPLIT>;
    const size_t most = SPLIT ? GI_SMEM_SPLIT : GI_SMEM, slot = GI_A_BYTES + (size_t)p.NT * 128;
    static bool ready[64] = {};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return launch_failed("gemm_i8: cudaGetDevice");
    if (dev < 0 || dev >= 64 || !ready[dev]) {
        if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most) != cudaSuccess)
            return launch_failed("gemm_i8: cudaFuncSetAttribute");
        if (dev >= 0 && dev < 64) ready[dev] = true;
    }
    p.stages = (int)std::min<size_t>(GI_MAX_STAGES, (most - 1024) / slot);
    p.tmem_cols = 32;
    while (p.tmem_cols < (SPLIT ? 1 : 2) * p.NT) p.tmem_cols *= 2;
    // SPLIT: the sums of a tile lie where the operands were
    const size_t smem = 1024 + std::max((size_t)p.stages * slot, SPLIT ? (size_t)p.NT * 512 : 0);
    cudaLaunchConfig_t lc{};
    lc.gridDim = dim3(SPLIT ? p.total * p.split : std::min(p.total, sm_count()));
    lc.blockDim = dim3(GI_THREADS); lc.dynamicSmemBytes = smem; lc.stream = s;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = p.split; at[1].val.clusterDim.y = 1; at[1].val.clusterDim.z = 1;
    lc.attrs = at; lc.numAttrs = SPLIT ? 2 : 1;
    if (cudaLaunchKernelEx(&lc, kern, p, mw, mx) != cudaSuccess) return launch_failed("k_gemm_i8");
    return check_launch("k_gemm_i8");
}

// Which kernel, and how many tokens per tile: what takes the fewest clocks by this estimate.  A step of 128 k is 2 NT clocks of MMA, or
// as long as an SM takes to bring its part of the tile at 60 B per clock; what an item has besides is about 1000 clocks, 2500 for a
// pair, and where CTAs share it also the sums that they pass on (these three fitted to the shapes below and some twenty more; 44 B per clock
// chose worse on 200 x [4096 x 4096], 600 x [1000 x 2000] and 300 x [6000 x 1500]).  us on finished rows:
//   shared   as many CTAs share an item as one per SM leaves room for: 24 rows x [4096 x 12288], 32 items, 22.9 with one, 16.4, 13.7
//            and 12.5 with 2, 3 and 4; but on the SMs' second places they lose (16 rows x [12288 x 4096], 96 items, 11.5 with one, 13.1 with 2)
//   tiles    777 rows x [5003 x 2048], in pairs: four tiles of 224 tokens are 80 items for 74 pairs, 16.8, seven of 128 are 140, 13.2
//   pairs    2048 rows x [12288 x 4096] 82 with single CTAs, 71 in pairs; 301 x [8192 x 4096] 15.6 and 12.6; but 48 x [12288 x 4096]
//            11.9 and 11.9; 250 x [2000 x 4096] 9.6 shared, 10.0 in pairs; 600 x [1000 x 2000] 6.7 with single CTAs, 7.0 in pairs, 9.2 shared
struct GiPlan { int M, N, K, pair, NT, n_jobs, total, split; };
static GiPlan gi_plan(int M, int N, int K) {
    GiPlan g{M, N, K, 0, 0, 0, 0, 1};
    const int sms = sm_count(), least = (M + GI_MAX_NT - 1) / GI_MAX_NT, nst = (K + 127) / 128;
    long best = 0;
    for (int jobs = least; jobs < least + 8 && (jobs == least || (M + jobs - 1) / jobs > 16); ++jobs) {
        for (int two = 0; two < 2; ++two) {
            const int per = (M + jobs - 1) / jobs, nt = two ? (per + 31) & ~31 : (per + 15) & ~15, n_jobs = (M + nt - 1) / nt;
            const long items = (long)((N + 127) / 128 + two) / (1 + two) * n_jobs, places = sms / (1 + two);
            // (the sums of an item that is shared lie where its operands were: up to 128 tokens)
            const int split = two || nt > 128 ? 1 : (int)std::max(1l, std::min({places / items, (long)GI_MAX_SPLIT, (long)nst / 4}));
            const long step = std::max(2 * nt, (int)(GI_A_BYTES + (two ? 64 : 128) * nt) / 60);
            const long cost = (items * split + places - 1) / places * ((nst + split - 1) / split * step + (split > 1 ? 2500 + 25 * nt : two ? 2500 : 1000));
            if (!best || cost < best) { best = cost; g.pair = two; g.NT = nt; g.n_jobs = n_jobs; g.total = (int)items; g.split = split; }
        }
    }
    return g;
}

// early: the launch before on the stream is the quantiser of x, which releases its dependents after its own dependency wait.
int gemm_i8_wide(void* y, int y_bf16, const b200_i8_rows* W, const b200_i8_rows* x, int M, int N, int K, int early, cudaStream_t s) {
    GiParams p{};
    p.early = early;
    p.y = y; p.sw = W->scale; p.sx = x->scale; p.status = device_status_ptr();
    if (!p.status || !tmap_available()) return B200_ENOTIMPL;
    p.M = M; p.N = N; p.nst = (K + 127) / 128;
    // The plan depends on the sizes alone; a model has few of them, and the divisions above take a microsecond.
    static thread_local GiPlan plans[64];
    GiPlan& g = plans[((unsigned)M * 2654435761u ^ (unsigned)N * 40503u ^ (unsigned)K * 9973u) >> 7 & 63u];
    if (g.M != M || g.N != N || g.K != K) g = gi_plan(M, N, K);
    p.NT = g.NT; p.n_jobs = g.n_jobs; p.total = g.total; p.split = g.split;
    credit(B200_CREDIT_GEMM, (double)N * K);
    if (g.pair) return y_bf16 ? gi_launch_pair<true>(p, W, x, K, s) : gi_launch_pair<false>(p, W, x, K, s);
    if (p.split > 1) return y_bf16 ? gi_launch<true, true>(p, W, x, K, s) : gi_launch<false, true>(p, W, x, K, s);
    return y_bf16 ? gi_launch<true, false>(p, W, x, K, s) : gi_launch<false, false>(p, W, x, K, s);
}

}  // namespace b200
