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
// Rows past N or M and columns past K come as zero from the tensor maps.  Every wait is bounded (tma_pipe.cuh).
#include "b200_internal.h"
#include "umma_mxf4.cuh"
#include <cuda.h>
#include <cuda_bf16.h>

namespace b200 {

constexpr int GI_THREADS = 384;
constexpr int GI_MAX_STAGES = 12;
constexpr int GI_TMEM_COLS = 512;

struct GiParams {
    void* y; const float* sw; const float* sx; unsigned int* status;
    int M, N, nst, n_jobs, total, stages;
};

template <int NT, bool BF16>
__global__ void __launch_bounds__(GI_THREADS, 1)
k_gemm_i8(const __grid_constant__ GiParams p, const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x) {
    constexpr uint32_t A_BYTES = 16384, B_BYTES = NT * 128u, SLOT = A_BYTES + B_BYTES;
    static_assert(SLOT % 1024 == 0, "swizzled operands start on 1024-byte boundaries");
    extern __shared__ __align__(1024) unsigned char smem[];
    __shared__ uint64_t full_bar[GI_MAX_STAGES], empty_bar[GI_MAX_STAGES], acc_full[2], acc_empty[2];
    __shared__ uint32_t tmem_base_s;
    __shared__ float sxs[2][NT];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int nst = p.nst, S = p.stages;
    // TMEM is taken after the kernel before has ended and before the kernel after may start: a kernel that held the columns
    // while it waits for another that wants them on the same SM would wait for good.
    pdl_wait();
    if (warp == 2) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" :: "r"(smem_u32(&tmem_base_s)), "r"(GI_TMEM_COLS));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
    } else if (warp == 1) {
        if (lane < S) { mbar_init(smem_u32(&full_bar[lane]), 1); mbar_init(smem_u32(&empty_bar[lane]), 1); }
        if (lane < 2) { mbar_init(smem_u32(&acc_full[lane]), 1); mbar_init(smem_u32(&acc_empty[lane]), 8); }
        mbar_fence_init();
    }
    gx_fence_before();
    __syncthreads();
    gx_fence_after();
    pdl_launch_dependents();
    const uint32_t tmem = tmem_base_s;
    const int first = blockIdx.x, stride = gridDim.x;
    const int n_items = (p.total - first + stride - 1) / stride;      // the grid is no larger than the number of items
    const uint32_t ring0 = smem_u32(smem) + ((1024u - (smem_u32(smem) & 1023u)) & 1023u);
    const uint32_t full0 = smem_u32(&full_bar[0]), empty0 = smem_u32(&empty_bar[0]);

    if (warp == 0) {
        int s = 0; uint32_t ph = 1;
        for (int i = 0; i < n_items; ++i) {
            const int q = first + i * stride, tile = q / p.n_jobs, job = q - tile * p.n_jobs;
            for (int it = 0; it < nst; ++it) {
                mbar_wait_spin(empty0 + s * 8, ph, p.status, 16);
                if (elect_one()) {
                    const uint32_t bar = full0 + s * 8, dst = ring0 + (uint32_t)s * SLOT;
                    mbar_expect_tx(bar, SLOT);
                    gx_tma_2d(dst, &map_w, it * 128, tile * 128, bar);
                    gx_tma_2d(dst + A_BYTES, &map_x, it * 128, job * NT, bar);
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
    } else if (warp == 1) {
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
                    const uint64_t dA = d0 + (uint64_t)(((uint32_t)s * SLOT) >> 4), dB = dA + (A_BYTES >> 4);
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
        const uint32_t tq = tmem + ((uint32_t)(q4 * 32) << 16);
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
                if (row < p.N) {
                    const size_t o = (size_t)(m0 + c0) * p.N + row;
                    #pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        if (c0 + j >= rows) break;
                        const float v = __fmul_rn(__fmul_rn(__int2float_rn(__float_as_int(d[j])), sxs[buf][c0 + j]), sw);
                        if (BF16) static_cast<__nv_bfloat16*>(p.y)[o + (size_t)j * p.N] = __float2bfloat16_rn(v);
                        else static_cast<float*>(p.y)[o + (size_t)j * p.N] = v;
                    }
                }
            }
            gx_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&acc_empty[buf]));
        }
    }
    gx_fence_before();
    __syncthreads();
    if (warp == 2) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" :: "r"(tmem), "r"(GI_TMEM_COLS));
}

template <int NT, bool BF16>
static int gi_launch(GiParams p, const b200_i8_rows* W, const b200_i8_rows* x, int K, cudaStream_t s) {
    CUtensorMap mw, mx;
    const size_t pitch = i8_pitch(K);
    if (!tmap_u8_pitched(&mw, W->q, (size_t)p.N, (size_t)K, pitch, 128, 128, true, true) ||
        !tmap_u8_pitched(&mx, x->q, (size_t)p.M, (size_t)K, pitch, 128, NT, true, true)) return B200_ENOTIMPL;
    auto kern = k_gemm_i8<NT, BF16>;
    constexpr size_t slot = 16384 + NT * 128;
    constexpr int most = (int)std::min<size_t>(GI_MAX_STAGES, (227 * 1024 - 1024 - 4096) / slot);      // 4 KB: static shared memory
    constexpr size_t smem = most * slot + 1024;
    static bool ready[64] = {};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return launch_failed("gemm_i8: cudaGetDevice");
    if (dev < 0 || dev >= 64 || !ready[dev]) {
        if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess)
            return launch_failed("gemm_i8: cudaFuncSetAttribute");
        if (dev >= 0 && dev < 64) ready[dev] = true;
    }
    p.stages = most;
    p.n_jobs = (p.M + NT - 1) / NT;
    p.total = (p.N + 127) / 128 * p.n_jobs;
    if (launch_pdl(kern, dim3(std::min(p.total, sm_count())), dim3(GI_THREADS), smem, s, p, mw, mx) != cudaSuccess) return launch_failed("k_gemm_i8");
    return check_launch("k_gemm_i8");
}

int gemm_i8_wide(void* y, int y_bf16, const b200_i8_rows* W, const b200_i8_rows* x, int M, int N, int K, cudaStream_t s) {
    GiParams p{};
    p.y = y; p.sw = W->scale; p.sx = x->scale; p.status = device_status_ptr();
    if (!p.status || !tmap_available()) return B200_ENOTIMPL;
    p.M = M; p.N = N; p.nst = (K + 127) / 128;
    credit(B200_CREDIT_GEMM, (double)N * K);
    auto go = [&](auto bf) {
        constexpr bool B = decltype(bf)::value;
        return M <= 16 ? gi_launch<16, B>(p, W, x, K, s) : M <= 32 ? gi_launch<32, B>(p, W, x, K, s) : M <= 64 ? gi_launch<64, B>(p, W, x, K, s)
             : M <= 128 ? gi_launch<128, B>(p, W, x, K, s) : gi_launch<256, B>(p, W, x, K, s);
    };
    return y_bf16 ? go(std::true_type{}) : go(std::false_type{});
}

}  // namespace b200
