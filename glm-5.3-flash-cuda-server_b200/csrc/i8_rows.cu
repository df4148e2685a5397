// i8_rows.cu -- rows of 8-bit integers with one scale per row: the quantiser, and the entry point of the products on them.
//
//   a = max(max |x[r, :]|, 2^-119)    scale[r] = a / 127    q[r, k] = rint(x[r, k] * (127 / a))
//
// |x| * fl(127 / a) is at most 127 (1 + 2^-23), so no code leaves -127 .. 127.  The floor of 2^-119 keeps both quotients
// normal numbers (2^-119 / 127 > 2^-126): a row of zeros has codes of zero and needs no case of its own.  The maximum runs
// over the bit patterns of |x|, which order like the values with infinities and NaN on top.
#include "b200_internal.h"
#include "tma_pipe.cuh"
#include <cuda_bf16.h>

namespace b200 {

constexpr int I8Q_THREADS = 256;
constexpr int I8Q_KEEP = 4;                        // vectors of 8 elements a thread keeps: rows of up to 8192 are read once

// One CTA per row.  VEC: rows start on 16-byte boundaries.  HBM-bound for weights and prefill chunks (es + 1 bytes per element).
template <bool F32, bool VEC>
__global__ void __launch_bounds__(I8Q_THREADS)
k_i8_quantize(const void* __restrict__ xin, size_t ldx, int K, int8_t* __restrict__ q, float* __restrict__ scale) {
    __shared__ uint32_t red[I8Q_THREADS / 32];
    const int tid = threadIdx.x;
    const size_t row = blockIdx.x, pitch = i8_pitch(K);
    pdl_launch_dependents();
    pdl_wait();
    const char* xr = static_cast<const char*>(xin) + row * ldx * (F32 ? 4 : 2);
    auto one = [&](int k) -> float {
        return F32 ? reinterpret_cast<const float*>(xr)[k] : __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(xr)[k]);
    };
    auto ld = [&](int c, float (&v)[8]) {              // elements 8c .. 8c + 7, zero past K
        if (VEC && 8 * c + 8 <= K) {
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
            for (int j = 0; j < 8; ++j) v[j] = 8 * c + j < K ? one(8 * c + j) : 0.f;
        }
    };
    const int nc = (int)(pitch >> 3);                  // the row's vectors, the zero bytes past K among them
    uint32_t ai = 0u;
    auto most = [&](const float (&v)[8]) {
        #pragma unroll
        for (int j = 0; j < 8; ++j) ai = max(ai, __float_as_uint(v[j]) & 0x7fffffffu);
    };
    float keep[I8Q_KEEP][8];
    #pragma unroll
    for (int i = 0; i < I8Q_KEEP; ++i) if (tid + i * I8Q_THREADS < nc) ld(tid + i * I8Q_THREADS, keep[i]);
    #pragma unroll
    for (int i = 0; i < I8Q_KEEP; ++i) if (tid + i * I8Q_THREADS < nc) most(keep[i]);
    for (int c = tid + I8Q_KEEP * I8Q_THREADS; c < nc; c += I8Q_THREADS) { float v[8]; ld(c, v); most(v); }
    #pragma unroll
    for (int o = 16; o; o >>= 1) ai = max(ai, __shfl_xor_sync(0xffffffffu, ai, o));
    if ((tid & 31) == 0) red[tid >> 5] = ai;
    __syncthreads();
    ai = red[0];
    #pragma unroll
    for (int w = 1; w < I8Q_THREADS / 32; ++w) ai = max(ai, red[w]);
    const bool bad = ai >= 0x7f800000u;
    const float a = fmaxf(__uint_as_float(ai), 0x1p-119f);
    const float inv = bad ? 0.f : __fdiv_rn(127.f, a);
    if (tid == 0) scale[row] = bad ? __uint_as_float(0x7fc00000u) : __fdiv_rn(a, 127.f);
    auto put = [&](int c, const float (&v)[8]) {
        uint32_t w[2] = {0u, 0u};
        #pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int code = bad ? 0 : __float2int_rn(__fmul_rn(v[j], inv));
            w[j >> 2] |= (uint32_t)(code & 0xff) << (8 * (j & 3));
        }
        *reinterpret_cast<uint2*>(q + row * pitch + (size_t)c * 8) = make_uint2(w[0], w[1]);
    };
    #pragma unroll
    for (int i = 0; i < I8Q_KEEP; ++i) if (tid + i * I8Q_THREADS < nc) put(tid + i * I8Q_THREADS, keep[i]);
    for (int c = tid + I8Q_KEEP * I8Q_THREADS; c < nc; c += I8Q_THREADS) { float v[8]; ld(c, v); put(c, v); }
}

int i8_quantize_launch(const void* x, int x_is_f32, size_t ldx, int rows, int K, int8_t* q, float* scale, cudaStream_t s) {
    const size_t es = x_is_f32 ? 4 : 2;
    const bool vec = !((uintptr_t)x & 15) && !((ldx * es) & 15);
    auto kern = x_is_f32 ? (vec ? k_i8_quantize<true, true> : k_i8_quantize<true, false>)
                         : (vec ? k_i8_quantize<false, true> : k_i8_quantize<false, false>);
    if (launch_pdl(kern, dim3(rows), dim3(I8Q_THREADS), 0, s, x, ldx, K, q, scale) != cudaSuccess) return launch_failed("k_i8_quantize");
    return check_launch("k_i8_quantize");
}

// Up to so many bytes of activations the few-row kernel quantises them itself, in every CTA; beyond, in a launch of its own:
// [4096 x 4096] 1 row 7.1 us and 7.9, 2 rows f32 (32 KB) 9.1 and 9.2, [12288 x 4096] 5 rows bf16 (40 KB) 18.9 and 15.0.
constexpr size_t I8_GEMV_QUANT_BYTES = 32768;

static size_t up256(size_t v) { return (v + 255) / 256 * 256; }

}  // namespace b200

using namespace b200;

extern "C" size_t b200_i8_pitch(int K) { return K < 1 ? 0 : i8_pitch(K); }

// x and its row stride, for both entry points: type, alignment of the type, rows that do not overlap.
static int check_x(const void* x, int dtype, size_t ldx, int rows, int K) {
    if (!x || rows < 1 || K < 1 || (dtype != B200_F32 && dtype != B200_BF16) || ldx < (size_t)K) return B200_EINVAL;
    if (K > I8_MAX_K || rows > I8_MAX_ROWS) return B200_ELIMIT;
    if ((uintptr_t)x & (dtype == B200_F32 ? 3 : 1)) return B200_EALIGN;
    return B200_OK;
}

extern "C" int b200_i8_quantize(const void* x, int dtype, size_t ldx, int rows, int K, int8_t* q, float* scale, b200_stream stream) {
    if (!q || !scale) return B200_EINVAL;
    if (int rc = check_x(x, dtype, ldx, rows, K)) return rc;
    if (((uintptr_t)q & 15) || ((uintptr_t)scale & 3)) return B200_EALIGN;
    return i8_quantize_launch(x, dtype == B200_F32, ldx, rows, K, q, scale, stream);
}

extern "C" size_t b200_i8_gemm_workspace_bytes(int M, int K) {
    if (M < 1 || K < 1) return 256;
    return up256((size_t)M * i8_pitch(K)) + up256((size_t)M * 4);
}

extern "C" int b200_i8_gemm(void* y, int y_dtype, const b200_i8_rows* W, const void* x, int x_dtype, size_t ldx, int M, int N, int K,
                            void* ws, b200_stream stream) {
    if (!y || !W || !W->q || !W->scale || !x || M < 1 || N < 1 || K < 1 || (y_dtype != B200_F32 && y_dtype != B200_BF16)) return B200_EINVAL;
    if (M > I8_MAX_ROWS || N > I8_MAX_ROWS || K > I8_MAX_K) return B200_ELIMIT;
    if (((uintptr_t)y & (y_dtype == B200_F32 ? 3 : 1)) || ((uintptr_t)W->q & 15) || ((uintptr_t)W->scale & 3)) return B200_EALIGN;
    b200_i8_rows xq;
    if (x_dtype == B200_I8) {
        xq = *static_cast<const b200_i8_rows*>(x);
        if (!xq.q || !xq.scale) return B200_EINVAL;
        if (((uintptr_t)xq.q & 15) || ((uintptr_t)xq.scale & 3)) return B200_EALIGN;
    } else {
        if (int rc = check_x(x, x_dtype, ldx, M, K)) return rc;
        if (!ws) return B200_EINVAL;
        if ((uintptr_t)ws & 255) return B200_EALIGN;
        if (gemv_i8_takes(M, K) && (size_t)M * K * (x_dtype == B200_F32 ? 4 : 2) <= I8_GEMV_QUANT_BYTES)
            return gemv_i8(y, y_dtype == B200_BF16, W, x, x_dtype, ldx, nullptr, M, N, K, stream);
        int8_t* q = static_cast<int8_t*>(ws);
        float* scale = reinterpret_cast<float*>(q + up256((size_t)M * i8_pitch(K)));
        if (int rc = i8_quantize_launch(x, x_dtype == B200_F32, ldx, M, K, q, scale, stream)) return rc;
        xq = b200_i8_rows{q, scale};
    }
    if (gemv_i8_takes(M, K)) return gemv_i8(y, y_dtype == B200_BF16, W, xq.q, B200_I8, 0, xq.scale, M, N, K, stream);
    return gemm_i8_wide(y, y_dtype == B200_BF16, W, &xq, M, N, K, stream);
}
