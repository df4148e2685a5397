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

// Codes of four values: fl(v * inv) + 1.5 * 2^23 is rounded to a whole number, half to even, whose low byte is the code.  The
// conversion instruction runs at a quarter of the rate.
__device__ __forceinline__ uint32_t i8_codes(float a, float b, float c, float d, float inv) {
    const uint32_t x = __float_as_uint(__fadd_rn(__fmul_rn(a, inv), 12582912.f)), y = __float_as_uint(__fadd_rn(__fmul_rn(b, inv), 12582912.f));
    const uint32_t z = __float_as_uint(__fadd_rn(__fmul_rn(c, inv), 12582912.f)), w = __float_as_uint(__fadd_rn(__fmul_rn(d, inv), 12582912.f));
    return __byte_perm(__byte_perm(x, y, 0x0040), __byte_perm(z, w, 0x0040), 0x5410);
}

// One CTA per row, or one warp (I8Q_THREADS 32, four rows per CTA).  VEC: rows start on 16-byte boundaries; otherwise the aligned
// vectors around a row's are shifted into place ([777 x 2051] f32 4.5 -> 3.4 us against loads of single elements).  A thread keeps KEEP
// loads of 8 elements (as they came) between the maximum and the codes, which covers rows of 64 (bf16) or 32 (f32) times the threads; what is
// longer is read twice.  HBM-bound for weights and prefill chunks (es + 1 bytes per element; [2048 x 4096] bf16 6.3 us, 4 TB/s, with the
// rows in L2 and HBM by turns).
template <bool F32, bool VEC, int I8Q_THREADS>
__global__ void __launch_bounds__(I8Q_THREADS == 32 ? 128 : I8Q_THREADS)
k_i8_quantize(const void* xin, size_t ldx, int rows, int K, int8_t* q, float* scale) {
    constexpr int KEEP = F32 ? 4 : 8, W = F32 ? 8 : 4;        // words of 8 elements
    constexpr bool WARP = I8Q_THREADS == 32;
    __shared__ uint32_t red[I8Q_THREADS / 32];
    const int tid = WARP ? threadIdx.x & 31 : threadIdx.x;
    const size_t row = WARP ? (size_t)blockIdx.x * 4 + (threadIdx.x >> 5) : blockIdx.x, pitch = i8_pitch(K);
    // In this order: what starts now starts after all that came before this launch has ended (gemm_i8.cu takes its TMEM on that).
    pdl_wait();
    pdl_launch_dependents();
    if (WARP && row >= (size_t)rows) return;
    const char* xr = static_cast<const char*>(xin) + row * ldx * (F32 ? 4 : 2);
    struct Vec { uint32_t u[W]; };
    // !VEC: `off` elements lie between a 16-byte boundary and the row; a vector is cut out of the aligned ones that hold it.
    constexpr int PER = F32 ? 4 : 8, HOLD = W / 4 + !VEC;
    const int off = VEC ? 0 : (int)((uintptr_t)xr & 15) / (F32 ? 4 : 2);
    const uint4* xa = reinterpret_cast<const uint4*>(xr - off * (F32 ? 4 : 2));
    // The row's vectors of 8 codes, the zero bytes past K among them; those of lo .. hi - 1 lie in aligned ones within the row.
    const int nc = (int)(pitch >> 3), lo = off ? 1 : 0;
    const int hi = off ? max(lo, (K + off - HOLD * PER + 8) >> 3) : K >> 3;
    auto ld = [&](int c, Vec& v) {                     // elements 8c .. 8c + 7
        uint32_t w[4 * HOLD];
        #pragma unroll
        for (int j = 0; j < HOLD; ++j) {
            if (j == W / 4 && !off) { w[4 * j] = w[4 * j + 1] = w[4 * j + 2] = w[4 * j + 3] = 0u; continue; }
            const uint4 a = VEC ? __ldcs(xa + (W / 4) * c + j) : xa[(W / 4) * c + j];
            w[4 * j] = a.x; w[4 * j + 1] = a.y; w[4 * j + 2] = a.z; w[4 * j + 3] = a.w;
        }
        if constexpr (!VEC) {                          // by words, then by a half
            const int by = F32 ? off : off >> 1;
            #pragma unroll
            for (int j = 0; j < W + 2; ++j) w[j] = by & 2 ? w[(j + 2) % (4 * HOLD)] : w[j];
            #pragma unroll
            for (int j = 0; j < W + 1; ++j) w[j] = by & 1 ? w[j + 1] : w[j];
            #pragma unroll
            for (int j = 0; j < W; ++j) if (!F32) w[j] = __funnelshift_r(w[j], w[j + 1], (off & 1) * 16);
        }
        #pragma unroll
        for (int j = 0; j < W; ++j) v.u[j] = w[j];
    };
    auto ld_end = [&](int c, Vec& v) {                 // one at a row's end, zero past K
        #pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int k = 8 * c + j;
            if (F32) v.u[j % W] = k < K ? reinterpret_cast<const uint32_t*>(xr)[k] : 0u;
            else {
                const uint32_t h = k < K ? reinterpret_cast<const uint16_t*>(xr)[k] : 0u;
                v.u[(j >> 1) % W] = (j & 1) ? v.u[(j >> 1) % W] | (h << 16) : h;
            }
        }
    };
    const int end = tid < lo ? tid : hi + tid - lo;    // the first threads take one of those each, six at most
    uint32_t ai = 0u;
    auto most = [&](const Vec& v) {                    // over the bits of |x|; bf16 in pairs
        #pragma unroll
        for (int j = 0; j < W; ++j) ai = F32 ? max(ai, v.u[j] & 0x7fffffffu) : __vmaxu2(ai, v.u[j] & 0x7fff7fffu);
    };
    Vec keep[KEEP], last;
    const int c0 = lo + tid;
    #pragma unroll
    for (int i = 0; i < KEEP; ++i) if (c0 + i * I8Q_THREADS < hi) ld(c0 + i * I8Q_THREADS, keep[i]);
    if (end < nc) { ld_end(end, last); most(last); }
    #pragma unroll
    for (int i = 0; i < KEEP; ++i) if (c0 + i * I8Q_THREADS < hi) most(keep[i]);
    for (int c = c0 + KEEP * I8Q_THREADS; c < hi; c += I8Q_THREADS) { Vec v; ld(c, v); most(v); }
    if (!F32) ai = max(ai & 0xffff0000u, ai << 16);
    ai = __reduce_max_sync(0xffffffffu, ai);
    if (!WARP) {
        if ((tid & 31) == 0) red[tid >> 5] = ai;
        __syncthreads();
        ai = red[0];
        #pragma unroll
        for (int w = 1; w < I8Q_THREADS / 32; ++w) ai = max(ai, red[w]);
    }
    const bool bad = ai >= 0x7f800000u;
    const float a = fmaxf(__uint_as_float(ai), 0x1p-119f);
    const float inv = __fdiv_rn(127.f, a);
    if (tid == 0) scale[row] = bad ? __uint_as_float(0x7fc00000u) : __fdiv_rn(a, 127.f);
    auto put = [&](int c, const Vec& v) {
        float f[8];
        #pragma unroll
        for (int j = 0; j < 8; ++j) {
            const uint32_t u = v.u[(F32 ? j : j >> 1) % W];
            f[j] = __uint_as_float(F32 ? u : (j & 1) ? u & 0xffff0000u : u << 16);
        }
        uint2 o = make_uint2(i8_codes(f[0], f[1], f[2], f[3], inv), i8_codes(f[4], f[5], f[6], f[7], inv));
        if (bad) o = make_uint2(0u, 0u);
        *reinterpret_cast<uint2*>(q + row * pitch + (size_t)c * 8) = o;
    };
    #pragma unroll
    for (int i = 0; i < KEEP; ++i) if (c0 + i * I8Q_THREADS < hi) put(c0 + i * I8Q_THREADS, keep[i]);
    if (end < nc) put(end, last);
    for (int c = c0 + KEEP * I8Q_THREADS; c < hi; c += I8Q_THREADS) { Vec v; ld(c, v); put(c, v); }
}

int i8_quantize_launch(const void* x, int x_is_f32, size_t ldx, int rows, int K, int8_t* q, float* scale, cudaStream_t s) {
    const size_t es = x_is_f32 ? 4 : 2;
    const bool vec = !((uintptr_t)x & 15) && !((ldx * es) & 15);
    // [2048 x 12288] bf16: 19.3 us with 128 threads, whose second read comes out of L2, and 15.0 with 256.
    const bool wide = K > (x_is_f32 ? 4096 : 8192);
    // A warp per row where rows are short and many, us with a CTA of 128 and with a warp per row: bf16 [154880 x 1024] 195 and 77,
    // [2048 x 512] 3.1 and 1.8, [800 x 1024] 2.2 and 1.7, but [300 x 2048] 1.61 and 1.64, [24 x 2048] 1.46 and 1.55; unaligned f32
    // [1500 x 501] 2.9 and 2.2, [1100 x 501] 2.0 and 2.1, [1500 x 1001] 3.7 and 4.3.
    const bool warp = K <= (!x_is_f32 ? 2048 : vec ? 1024 : 512) && rows > (vec ? 2 : 8) * sm_count();
    auto go = [&](auto t) {
        constexpr int T = decltype(t)::value;
        auto kern = x_is_f32 ? (vec ? k_i8_quantize<true, true, T> : k_i8_quantize<true, false, T>)
                             : (vec ? k_i8_quantize<false, true, T> : k_i8_quantize<false, false, T>);
        return launch_pdl(kern, dim3(T == 32 ? (rows + 3) / 4 : rows), dim3(T == 32 ? 128 : T), 0, s, x, ldx, rows, K, q, scale);
    };
    if ((warp ? go(std::integral_constant<int, 32>{}) : wide ? go(std::integral_constant<int, 256>{}) : go(std::integral_constant<int, 128>{})) != cudaSuccess)
        return launch_failed("k_i8_quantize");
    return check_launch("k_i8_quantize");
}

// Up to so many activations the few-row kernel quantises them itself, in every CTA; beyond, in a launch of its own.  us with either in
// replays (and for calls from the host, where a launch costs more), bf16: 1 row x [4096 x 4096] 5.9 and 6.8 (6.1 and 8.0), x [4096 x 12288]
// 11.9 and 12.2, x [4096 x 16384] 16.6 and 14.7; 2 rows x [4096 x 4096] 6.9 and 7.0, x [4096 x 8192] 10.4 and 10.0; 3 rows x [4096 x 4096] 8.5 and
// 7.6 (8.7 and 8.3); 4 rows x [4096 x 2048] 5.9 and 6.3; 5 rows x [4096 x 1600] 6.8 and 6.3 (7.1 and 7.9).
static bool i8_gemv_quantises(int M, int K) { return (size_t)M * K <= (M == 1 ? 12288 : 8192); }

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
    const bool quantised = x_dtype != B200_I8;
    if (x_dtype == B200_I8) {
        xq = *static_cast<const b200_i8_rows*>(x);
        if (!xq.q || !xq.scale) return B200_EINVAL;
        if (((uintptr_t)xq.q & 15) || ((uintptr_t)xq.scale & 3)) return B200_EALIGN;
    } else {
        if (int rc = check_x(x, x_dtype, ldx, M, K)) return rc;
        if (!ws) return B200_EINVAL;
        if ((uintptr_t)ws & 255) return B200_EALIGN;
        if (gemv_i8_takes(M, N, K, false) && i8_gemv_quantises(M, K))
            return gemv_i8(y, y_dtype == B200_BF16, W, x, x_dtype, ldx, nullptr, M, N, K, stream);
        int8_t* q = static_cast<int8_t*>(ws);
        float* scale = reinterpret_cast<float*>(q + up256((size_t)M * i8_pitch(K)));
        if (int rc = i8_quantize_launch(x, x_dtype == B200_F32, ldx, M, K, q, scale, stream)) return rc;
        xq = b200_i8_rows{q, scale};
    }
    if (gemv_i8_takes(M, N, K, quantised)) return gemv_i8(y, y_dtype == B200_BF16, W, xq.q, B200_I8, 0, xq.scale, M, N, K, stream);
    return gemm_i8_wide(y, y_dtype == B200_BF16, W, &xq, M, N, K, quantised, stream);
}
