// gemv_i8.cu -- 8-bit integer products of 1 to 8 activation rows, quantised inside the kernel or before it.
//
// Bound by the weight stream.  The weights go from global memory straight into the registers that mma.sync takes them from: a
// lane's 16 bytes are two operands of k = 32, because the order of k is free as long as both operands have the same one.  The
// tokens are the operand of 16 rows (8 of them zero), 8 weight rows the other one.  Through shared memory and tcgen05 (gemm_i8.cu)
// the same stream waits for barriers, TMEM and a whole tile of 128 rows; here 8 warps share 8 rows, each a slice of K.
//
//   units of 8 weight rows; a CTA of 8 warps takes every gridDim-th unit, warp w the w-th slice of K of each; partial sums go to
//   shared memory, whole numbers, so that their order does not matter; after a batch of units the CTA adds and writes them.
//   A warp has the next 8 loads (4 KB) in flight while it multiplies the present ones.
// One row, quantised in the kernel, in replays: x [154880 x 4096] 92 us (6.9 TB/s: reads alone exceed the rate of a copy), [12288 x 4096] 10.5 us,
// [4096 x 4096] 5.9 us (5.2 with the weights in L2), about 3.5 of them the start, the row's codes and the last sums, which no byte costs.  What
// mattered is the number of instructions: with a test and a copy for every load 52 per 512 bytes of weights instead of 23, and 112 us.
#include "b200_internal.h"
#include "tma_pipe.cuh"
#include <cuda_bf16.h>

namespace b200 {

constexpr int GV_WARPS = 8, GV_THREADS = GV_WARPS * 32, GV_ROWS = 8;
constexpr int GV_LOADS = 8;                        // 64-k blocks a warp loads at once
constexpr int GV_KEEP = 2;                         // vectors of 8 activations a thread keeps between maximum and codes
constexpr int GV_PART = 4096;                      // partial sums of a batch of units
// Activations of a CTA, in bytes of shared memory, at most: every CTA brings all of them.  us here and in gemm_i8.cu, on finished rows: 8 rows
// (33 KB) x [4096 x 4096] 7.0 and 6.8, x [2000 x 4096] 4.7 and 6.0, 4 rows (33 KB) x [1000 x 6500] 5.4 and 5.7, but 8 rows (42 KB) x [4096 x 5120] 8.8 and
// 7.5, 4 rows (60 KB) x [4096 x 12288] 13.3 and 12.0; 2 rows (37 KB) x [4096 x 12288] 10.7 and 11.9, (43 KB) x [4096 x 14336] 13.7 and 13.3.  Behind
// the quantiser, whose end they have to wait for: 4 rows (21 KB) x [4096 x 4096] 8.0 and 8.4, x [12288 x 4096] 12.4 and 12.7, but 5 rows (25 KB) 8.5 and
// 8.4, 13.0 and 12.7, 8 rows (33 KB) 9.4 and 8.4, 14.1 and 12.8; 2 rows (37 KB) x [4096 x 12288] 12.9 and 13.8, 1 row (47 KB) x [4096 x 24000] 23.4 and 25.8.
constexpr size_t GV_SMEM = 34 * 1024, GV_SMEM_QUANTISED = 24 * 1024, GV_SMEM_2 = 38 * 1024, GV_SMEM_2_QUANTISED = 48 * 1024, GV_SMEM_MAX = 48 * 1024;

struct GvParams {
    void* y; const int8_t* w; const float* sw; const void* x; const float* sx;
    size_t ldx, pitch;
    int M, N, K, blocks, xpitch, units, batch;             // 64-k blocks of a row; bytes between activation rows in shared memory
};

enum { GV_X_F32 = B200_F32, GV_X_BF16 = B200_BF16, GV_X_I8 = B200_I8 };

// Activation rows -> codes in shared memory (zero past K), scales in sxs.  By the rule of i8_rows.cu, the same f32 operations.
template <int XT>
__device__ __forceinline__ void gv_stage_x(const GvParams& p, int8_t* xs, float* sxs, uint32_t* red, int warp, int lane) {
    const int kp = p.blocks * 64;
    if (p.M < 8)                                       // the row of zeros
        for (int i = warp * 32 + lane; i < kp / 16; i += GV_THREADS) *reinterpret_cast<uint4*>(xs + (size_t)p.M * p.xpitch + i * 16) = make_uint4(0u, 0u, 0u, 0u);
    if (XT == GV_X_I8) {
        const int8_t* q = static_cast<const int8_t*>(p.x);
        const int nv = kp / 16;
        for (int i = warp * 32 + lane; i < p.M * nv; i += GV_THREADS) {
            const int m = i / nv, k = (i - m * nv) * 16;
            uint4 v = make_uint4(0u, 0u, 0u, 0u);
            if (k < p.K) {
                v = *reinterpret_cast<const uint4*>(q + (size_t)m * p.pitch + k);
                if (k + 16 > p.K) {                    // the bytes past K are not used
                    uint32_t* u = &v.x;
                    #pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int left = p.K - k - 4 * j;
                        u[j] &= left >= 4 ? 0xffffffffu : left <= 0 ? 0u : (1u << (8 * left)) - 1u;
                    }
                }
            }
            *reinterpret_cast<uint4*>(xs + (size_t)m * p.xpitch + k) = v;
        }
        if (warp == 0 && lane < p.M) sxs[lane] = p.sx[lane];
        return;
    }
    // a row belongs to 8, 4, 2 or 1 warps
    constexpr bool F32 = XT == GV_X_F32;
    const int wpr = p.M == 1 ? 8 : p.M == 2 ? 4 : p.M <= 4 ? 2 : 1;
    const int m = warp / wpr, sub = warp - m * wpr, step = wpr * 32;
    const char* xr = static_cast<const char*>(p.x) + (size_t)m * p.ldx * (F32 ? 4 : 2);
    const bool vec = !((uintptr_t)xr & 15);
    auto ld = [&](int c, float (&v)[8]) {              // elements 8c .. 8c + 7, zero past K
        if (vec && 8 * c + 8 <= p.K) {
            if (F32) {
                const float4 a = reinterpret_cast<const float4*>(xr)[2 * c], b = reinterpret_cast<const float4*>(xr)[2 * c + 1];
                v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
            } else {
                const uint4 a = reinterpret_cast<const uint4*>(xr)[c];
                const uint32_t w[4] = {a.x, a.y, a.z, a.w};
                #pragma unroll
                for (int j = 0; j < 4; ++j) { v[2 * j] = __uint_as_float(w[j] << 16); v[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u); }
            }
        } else {
            #pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int k = 8 * c + j;
                v[j] = k >= p.K ? 0.f : F32 ? reinterpret_cast<const float*>(xr)[k] : __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(xr)[k]);
            }
        }
    };
    const int nc = m < p.M ? kp >> 3 : 0, c0 = sub * 32 + lane;
    uint32_t ai = 0u;
    auto take = [&](const float (&v)[8]) {
        #pragma unroll
        for (int j = 0; j < 8; ++j) ai = max(ai, __float_as_uint(v[j]) & 0x7fffffffu);
    };
    float keep[GV_KEEP][8];
    #pragma unroll
    for (int i = 0; i < GV_KEEP; ++i) if (c0 + i * step < nc) ld(c0 + i * step, keep[i]);
    #pragma unroll
    for (int i = 0; i < GV_KEEP; ++i) if (c0 + i * step < nc) take(keep[i]);
    for (int c = c0 + GV_KEEP * step; c < nc; c += step) { float v[8]; ld(c, v); take(v); }
    ai = __reduce_max_sync(0xffffffffu, ai);
    if (lane == 0) red[warp] = ai;
    __syncthreads();
    if (m >= p.M) return;
    for (int w = 0; w < wpr; ++w) ai = max(ai, red[m * wpr + w]);
    const bool bad = ai >= 0x7f800000u;
    const float a = fmaxf(__uint_as_float(ai), 0x1p-119f);
    const float inv = bad ? 0.f : __fdiv_rn(127.f, a);
    if (c0 == 0) sxs[m] = bad ? __uint_as_float(0x7fc00000u) : __fdiv_rn(a, 127.f);
    auto put = [&](int c, const float (&v)[8]) {
        uint32_t w[2] = {0u, 0u};
        #pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int code = bad ? 0 : __float2int_rn(__fmul_rn(v[j], inv));
            w[j >> 2] |= (uint32_t)(code & 0xff) << (8 * (j & 3));
        }
        *reinterpret_cast<uint2*>(xs + (size_t)m * p.xpitch + (size_t)c * 8) = make_uint2(w[0], w[1]);
    };
    #pragma unroll
    for (int i = 0; i < GV_KEEP; ++i) if (c0 + i * step < nc) put(c0 + i * step, keep[i]);
    for (int c = c0 + GV_KEEP * step; c < nc; c += step) { float v[8]; ld(c, v); put(c, v); }      // a second read, out of L1
}

__device__ __forceinline__ uint4 gv_ldw(const int8_t* p) {
    uint4 v;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}
__device__ __forceinline__ void gv_mma(int (&d)[4], uint32_t a0, uint32_t a2, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%5}, {%7,%8}, {%0,%1,%2,%3};"
                 : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3]) : "r"(a0), "r"(0u), "r"(a2), "r"(b0), "r"(b1));
}

template <int XT, bool BF16>
__global__ void __launch_bounds__(GV_THREADS, 2)
k_gemv_i8(const __grid_constant__ GvParams p) {
    extern __shared__ __align__(16) int8_t xs[];       // [M][xpitch]
    __shared__ __align__(16) int part[GV_PART];        // [unit of the batch][warp][token][8 rows]
    static_assert(__alignof__(part) >= alignof(int2), "partial sums are stored in pairs");
    __shared__ float sxs[8];
    __shared__ uint32_t red[GV_WARPS];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int r = lane >> 2, kq = (lane & 3) * 16;
    const int b0 = (int)((long long)p.blocks * warp / GV_WARPS), b1 = (int)((long long)p.blocks * (warp + 1) / GV_WARPS);
    const int chunks = max(1, (b1 - b0 + GV_LOADS - 1) / GV_LOADS);
    const int full = min(b1, (int)(p.pitch >> 6));      // blocks of the slice that lie within the row
    const int n_units = (p.units - (int)blockIdx.x + (int)gridDim.x - 1) / (int)gridDim.x;
    const int steps = n_units * chunks;
    pdl_launch_dependents();
    // Steps: the chunks of GV_LOADS blocks of this warp's slice, unit by unit.  A slice of no blocks has one chunk of zeros.
    int lu = 0, lc = 0;                                // unit and chunk of the next load
    const int8_t* row = p.w;
    auto load = [&](uint4 (&w)[GV_LOADS]) {
        if (lc == 0) row = p.w + (size_t)min(((int)blockIdx.x + lu * (int)gridDim.x) * GV_ROWS + r, p.N - 1) * p.pitch;      // rows past N: their sums are not written
        const int bl = b0 + lc * GV_LOADS;
        const int8_t* q = row + (size_t)bl * 64 + kq;
        if (bl + GV_LOADS <= full) {
            #pragma unroll
            for (int i = 0; i < GV_LOADS; ++i) w[i] = gv_ldw(q + i * 64);
        } else {
            #pragma unroll
            for (int i = 0; i < GV_LOADS; ++i)
                w[i] = bl + i < b1 && (size_t)(bl + i) * 64 + kq < p.pitch ? gv_ldw(q + i * 64) : make_uint4(0u, 0u, 0u, 0u);
        }
        if (++lc == chunks) { lc = 0; ++lu; }
    };
    uint4 wa[GV_LOADS], wb[GV_LOADS];
    // The first weights are asked into L2 while the kernel before still runs.  Nothing is read: L2 is where its writes go, too.
    // 7.1 -> 6.4 us for one row x [4096 x 4096] in a row of calls; two units instead of one: 6.7.
    const int ahead = (int)blockIdx.x * GV_ROWS + (lane & 7), bytes = min((b1 - b0) * 64, (int)p.pitch - b0 * 64);
    if (lane < 8 && ahead < p.N && bytes > 0)
        asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" :: "l"(p.w + (size_t)ahead * p.pitch + b0 * 64), "r"(bytes) : "memory");
    // The scales of the units too, which are wanted last (one row x [4096 x 12288] 10.2 -> 9.95 us, [4096 x 4096] 5.1 -> 5.0).
    for (int i = tid; i < n_units; i += GV_THREADS)
        asm volatile("prefetch.global.L2 [%0];" :: "l"(p.sw + ((size_t)blockIdx.x + (size_t)i * gridDim.x) * GV_ROWS));
    pdl_wait();
    load(wa);
    gv_stage_x<XT>(p, xs, sxs, red, warp, lane);
    __syncthreads();

    // rows past M read a row of zeros
    const int8_t* xrow = xs + (size_t)min(r, p.M) * p.xpitch + b0 * 64 + kq;
    const int per = p.M * GV_ROWS;                     // outputs of a unit
    int d[4] = {0, 0, 0, 0}, c = 0, u = 0, u0 = 0;     // chunk; unit of the batch; the batch's first unit
    auto consume = [&](const uint4 (&w)[GV_LOADS]) {
        const int8_t* xc = xrow + c * (GV_LOADS * 64);
        #pragma unroll
        for (int i = 0; i < GV_LOADS; ++i) {
            const uint4 x = *reinterpret_cast<const uint4*>(xc + i * 64);
            gv_mma(d, x.x, x.y, w[i].x, w[i].y);
            gv_mma(d, x.z, x.w, w[i].z, w[i].w);
        }
        if (++c < chunks) return;
        // token r, weight rows 2 * (lane & 3) and the next
        if (r < p.M) *reinterpret_cast<int2*>(&part[(u * GV_WARPS + warp) * per + r * GV_ROWS + 2 * (lane & 3)]) = make_int2(d[0], d[1]);
        d[0] = d[1] = c = 0;
        if (++u < p.batch && u0 + u < n_units) return;
        __syncthreads();
        for (int i = tid; i < u * per; i += GV_THREADS) {
            const int v = i / per, j = i - v * per, m = j / GV_ROWS;
            const int n = ((int)blockIdx.x + (u0 + v) * (int)gridDim.x) * GV_ROWS + (j - m * GV_ROWS);
            if (n < p.N) {
                int acc = 0;
                #pragma unroll
                for (int q = 0; q < GV_WARPS; ++q) acc += part[(v * GV_WARPS + q) * per + j];
                const float f = __fmul_rn(__fmul_rn(__int2float_rn(acc), sxs[m]), p.sw[n]);
                if (BF16) static_cast<__nv_bfloat16*>(p.y)[(size_t)m * p.N + n] = __float2bfloat16_rn(f);
                else static_cast<float*>(p.y)[(size_t)m * p.N + n] = f;
            }
        }
        __syncthreads();
        u0 += u; u = 0;
    };
    for (int s = 0; s < steps; s += 2) {
        if (s + 1 < steps) load(wb);
        consume(wa);
        if (s + 1 == steps) break;
        if (s + 2 < steps) load(wa);
        consume(wb);
    }
}

template <int XT, bool BF16>
static int gv_launch(const GvParams& p, size_t smem, cudaStream_t s) {
    auto kern = k_gemv_i8<XT, BF16>;
    static bool ready[64] = {};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return launch_failed("gemv_i8: cudaGetDevice");
    if (dev < 0 || dev >= 64 || !ready[dev]) {
        if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)GV_SMEM_MAX) != cudaSuccess)
            return launch_failed("gemv_i8: cudaFuncSetAttribute");
        if (dev >= 0 && dev < 64) ready[dev] = true;
    }
    if (launch_pdl(kern, dim3(std::min(p.units, 2 * sm_count())), dim3(GV_THREADS), smem, s, p) != cudaSuccess) return launch_failed("k_gemv_i8");
    return check_launch("k_gemv_i8");
}

static int gv_xpitch(int K) {
    const int blocks = (K + 63) / 64;
    return blocks * 64 + (blocks % 2 ? 0 : 64);        // an odd multiple of 64: the rows of a load lie in different banks
}
// The rows, one of zeros, and what the last chunk of a slice may read past the end (and multiplies by zero).
static size_t gv_x_bytes(int M, int K) { return (size_t)std::min(M + 1, 8) * gv_xpitch(K) + GV_LOADS * 64; }

// Five and more rows of a matrix that fills the GPU many times over are the tensor-core kernel's: 8 rows x [154880 x 2048] 77.3 us here and 53.3 there,
// x [154880 x 4096] 100.0 and 100.5 (5 rows 96.3 and 99.3); 4 rows 93.6 and 99.8, 8 rows x [40000 x 4096] 28.0 and 32.4.
bool gemv_i8_takes(int M, int N, int K, bool quantised) {
    const size_t most = M <= 2 ? (quantised ? GV_SMEM_2_QUANTISED : GV_SMEM_2) : quantised ? GV_SMEM_QUANTISED : GV_SMEM;
    return M <= 8 && gv_x_bytes(M, K) <= most && (M <= 4 || (size_t)N * K <= ((size_t)1 << 28));
}

// x: M rows of x_dtype (B200_F32, B200_BF16 with ldx; B200_I8 with their scales sx).
int gemv_i8(void* y, int y_bf16, const b200_i8_rows* W, const void* x, int x_dtype, size_t ldx, const float* sx, int M, int N, int K, cudaStream_t s) {
    GvParams p{};
    p.y = y; p.w = W->q; p.sw = W->scale; p.x = x; p.sx = sx; p.ldx = ldx; p.pitch = i8_pitch(K);
    p.M = M; p.N = N; p.K = K;
    p.blocks = (K + 63) / 64;
    p.xpitch = gv_xpitch(K);
    p.units = (N + GV_ROWS - 1) / GV_ROWS;
    p.batch = GV_PART / (GV_WARPS * M * GV_ROWS);
    credit(B200_CREDIT_GEMM, (double)N * K);
    const size_t smem = gv_x_bytes(M, K);
    if (x_dtype == B200_I8) return y_bf16 ? gv_launch<GV_X_I8, true>(p, smem, s) : gv_launch<GV_X_I8, false>(p, smem, s);
    if (x_dtype == B200_F32) return y_bf16 ? gv_launch<GV_X_F32, true>(p, smem, s) : gv_launch<GV_X_F32, false>(p, smem, s);
    return y_bf16 ? gv_launch<GV_X_BF16, true>(p, smem, s) : gv_launch<GV_X_BF16, false>(p, smem, s);
}

}  // namespace b200
