// logprobs.cu -- log probabilities of given tokens, the entropy, and the likeliest tokens, from one pass over the logits.
//
//   m = max x      S = sum exp(x - m)      log p(t) = (x_t - m) - ln S      H = ln S - (1 / S) sum (x - m) exp(x - m)
//
// A cluster of CTAs takes a row, each CTA a contiguous part of it; parts are joined over distributed shared memory.
//
// Statistics.  Every thread keeps (m, n, S, T): n elements equal to m (they count as exactly 1 and are not added), S and T in base 2
// over the others:
//   S = sum 2^d,  T = sum d 2^d,  d = (x - m) log2 e.
// So S is what is left beside the likeliest token, and ln(1 + S) of a token that is nearly certain keeps its relative precision
// (1 + S in f32 would not).  The threads start from the maximum of the CTA's first tile; a vector that holds nothing above it
// (nearly all) takes the short path: one multiply-add, one exponential, two sums per element.  d is the multiply-add
// fma(x, log2 e, -fl(m log2 e)): its distance from (x - m) log2 e is the same for every element and corrected when parts are joined.
//
// The likeliest tokens.  Order: logit descending, then index ascending, as one 64-bit key.  Every thread has the largest key of its
// part of the first tile; the top-th largest of these is a bound that at least `top` elements reach, and later elements count only
// above its value (an equal one has a larger index).  Those go to a list in shared memory, a few hundred for a vocabulary of 154880
// in no particular order, from which warps sort 32 at a time and merge.  A list that overflows (logits in ascending order; a first
// tile of masked tokens before many others) is dropped, and the CTA finds its bound by radix selection over its part instead.
#include "b200_internal.h"
#include "tma_pipe.cuh"
#include <cuda_bf16.h>
#include <cooperative_groups.h>
#include <math_constants.h>

namespace b200 {
namespace cg = cooperative_groups;

constexpr int LP_THREADS = 512, LP_WARPS = LP_THREADS / 32;
constexpr int LP_LIST = 2048;                      // candidates of a CTA
constexpr int LP_VECS = 4;                         // 16-byte loads a thread has in a tile
constexpr float LP_LOG2E = 1.44269504088896341f, LP_LN2 = 0.693147180559945309f;

struct LpParams {
    const void* x; const int32_t* tokens; float* lp; float* entropy; int32_t* top_ids; float* top_lp;
    size_t ld; int V, G, top;
};

struct LpStat { float m, n, s, t; };               // see above; n as a float (n <= 2^24 exact; beyond it its last bit does not matter)

// 64-bit key of logit x at index i: orders by x descending, then i ascending; never 0.  -0 and +0 are the same logit.
__device__ __forceinline__ unsigned long long lp_key(float x, int i) {
    const uint32_t b = __float_as_uint(x + 0.f);
    return ((unsigned long long)(b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u)) << 32) | (uint32_t)~i;
}
__device__ __forceinline__ int lp_index(unsigned long long key) { return (int)~(uint32_t)key; }
__device__ __forceinline__ float lp_value(unsigned long long key) {
    const uint32_t o = (uint32_t)(key >> 32);
    return __uint_as_float((o & 0x80000000u) ? o ^ 0x80000000u : ~o);
}
__device__ __forceinline__ float lp_exp2(float d) { float e; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(d)); return e; }
__device__ __forceinline__ float lp_max(float a, float b) { float r; asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b)); return r; }

// d = (x - m) log2 e in two steps, for any finite x and m.  -216 and below: 2^d is zero, d finite.
__device__ __forceinline__ float lp_d(float x, float m) { return fmaxf((x - m) * LP_LOG2E, -216.f); }

// Joins b into a.  Parts without elements have m = -inf, n = s = t = 0.  s = t = NaN marks a row that holds +inf or NaN.
__device__ __forceinline__ LpStat lp_join(LpStat a, LpStat b) {
    if (a.m < b.m) { const LpStat c = a; a = b; b = c; }
    if (a.m == b.m) return LpStat{a.m, a.n + b.n, a.s + b.s, a.t + b.t};
    const float d = lp_d(b.m, a.m), f = exp2f(d), all = b.n + b.s;         // b.m == -inf: f = 0
    return LpStat{a.m, a.n, fmaf(f, all, a.s), a.t + f * (b.t + all * d)};
}
__device__ __forceinline__ LpStat lp_shfl(LpStat a, int o) {
    return LpStat{__shfl_xor_sync(0xffffffffu, a.m, o), __shfl_xor_sync(0xffffffffu, a.n, o), __shfl_xor_sync(0xffffffffu, a.s, o),
                  __shfl_xor_sync(0xffffffffu, a.t, o)};
}

// A warp's 32 keys (one per lane), descending.
__device__ __forceinline__ unsigned long long lp_stage(unsigned long long k, int j, bool keep_max) {
    const unsigned long long o = __shfl_xor_sync(0xffffffffu, k, j);
    return (o > k) == keep_max ? o : k;
}
__device__ __forceinline__ unsigned long long lp_sort(unsigned long long k, int lane) {
    #pragma unroll
    for (int n = 2; n <= 32; n <<= 1)
        #pragma unroll
        for (int j = n >> 1; j; j >>= 1) k = lp_stage(k, j, ((lane & j) == 0) == ((lane & n) == 0));
    return k;
}
// The 32 largest of two descending lists, descending.
__device__ __forceinline__ unsigned long long lp_merge(unsigned long long a, unsigned long long b, int lane) {
    const unsigned long long r = __shfl_sync(0xffffffffu, b, 31 - lane);
    a = a > r ? a : r;
    #pragma unroll
    for (int j = 16; j; j >>= 1) a = lp_stage(a, j, (lane & j) == 0);
    return a;
}
// lists[0] <- the 32 largest of lists[0 .. n - 1] (n a power of two); every thread calls it.
__device__ __forceinline__ void lp_tree(unsigned long long (*lists)[32], int n, int warp, int lane) {
    for (int h = n >> 1; h; h >>= 1) {
        __syncthreads();
        if (warp < h) lists[warp][lane] = lp_merge(lists[warp][lane], lists[warp + h][lane], lane);
    }
    __syncthreads();
}

template <bool F32> struct LpVec { static constexpr int N = F32 ? 4 : 8; };
template <bool F32>
__device__ __forceinline__ void lp_unpack(const uint4& a, float (&v)[LpVec<F32>::N]) {
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
    #pragma unroll
    for (int j = 0; j < 4; ++j) {
        if (F32) v[j] = __uint_as_float(w[j]);
        else { v[2 * j] = __uint_as_float(w[j] << 16); v[(2 * j + 1) % LpVec<F32>::N] = __uint_as_float(w[j] & 0xffff0000u); }
    }
}

template <bool F32>
__global__ void __launch_bounds__(LP_THREADS, 2)
k_token_logprobs(const __grid_constant__ LpParams p) {
    constexpr int NV = LpVec<F32>::N;
    __shared__ unsigned long long list[LP_LIST];
    __shared__ unsigned long long lists[LP_WARPS][32];
    __shared__ LpStat stats[LP_WARPS];
    __shared__ LpStat part;                            // this CTA's, read by the cluster's first CTA
    __shared__ int count;
    __shared__ unsigned int hist[256];
    __shared__ unsigned int pick[2];
    cg::cluster_group cluster = cg::this_cluster();
    const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const size_t row = blockIdx.x / C;
    const int V = p.V, top = p.top;
    pdl_launch_dependents();
    pdl_wait();

    // The row: `head` single elements up to a 16-byte boundary, nb vectors, the rest single elements.
    using T = typename std::conditional<F32, float, __nv_bfloat16>::type;
    const T* x = static_cast<const T*>(p.x) + row * p.ld;
    auto one = [&](int i) -> float { return F32 ? reinterpret_cast<const float*>(x)[i] : __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(x)[i]); };
    const int head = min(V, (int)(((16u - ((uint32_t)(uintptr_t)x & 15u)) & 15u) / sizeof(T)));
    const int nb = (V - head) / NV;
    const uint4* xv = reinterpret_cast<const uint4*>(x + head);
    const int v0 = (int)((long long)nb * rank / C), v1 = (int)((long long)nb * (rank + 1) / C);
    // single elements: the head belongs to the first CTA, the tail to the last; thread i has one of them or none
    int si = -1;
    if (rank == 0 && tid < head) si = tid;
    if (rank == C - 1 && tid >= 32 && tid - 32 < V - head - nb * NV) si = head + nb * NV + tid - 32;

    uint4 a[LP_VECS];
    auto load = [&](int v) {
        #pragma unroll
        for (int u = 0; u < LP_VECS; ++u) {
            const int i = v + u * LP_THREADS + tid;
            if (i < v1) a[u] = __ldcs(xv + i);
        }
    };
    if (tid == 0) count = 0;
    load(v0);
    const float sv = si >= 0 ? one(si) : -CUDART_INF_F;

    // ---- first tile: the maximum, and the bound that `top` elements reach ----
    float m = sv;
    // (a tail element is no witness of the bound: elements between the tile and the tail come before it at the same value)
    unsigned long long best = si >= 0 && si < head ? lp_key(sv, si) : 0ull;
    #pragma unroll
    for (int u = 0; u < LP_VECS; ++u) {
        const int i = v0 + u * LP_THREADS + tid;
        if (i < v1) {
            float v[NV];
            lp_unpack<F32>(a[u], v);
            #pragma unroll
            for (int j = 0; j < NV; ++j) {
                m = fmaxf(m, v[j]);
                if (top) { const unsigned long long k = lp_key(v[j], head + i * NV + j); best = best > k ? best : k; }
            }
        }
    }
    unsigned long long bound = ~0ull;
    if (top) {
        lists[warp][lane] = lp_sort(best, lane);
        lp_tree(lists, LP_WARPS, warp, lane);
        bound = lists[0][top - 1];
    }
    #pragma unroll
    for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (lane == 0) stats[warp].m = m;
    __syncthreads();
    #pragma unroll
    for (int w = 0; w < LP_WARPS; ++w) m = fmaxf(m, stats[w].m);

    // ---- the pass ----
    LpStat st{m, 0.f, 0.f, 0.f};
    // what the short path needs of st.m: the product that it subtracts, and the bound below which it may run
    float m2, quick;
    auto raise = [&](float to) {
        const float d = lp_d(st.m, to), f = exp2f(d), all = st.n + st.s;      // st.m == -inf: all = 0, or NaN, which stays
        st.t = f * (st.t + all * d); st.s = f * all;
        st.n = 0.f; st.m = to;
    };
    float drift;                                       // m2 - m log2 e: every d of the short path is too small by it
    auto settle = [&] {
        const bool fine = fabsf(st.m) < 1e6f;          // |drift| < 1/8
        m2 = fine ? st.m * LP_LOG2E : 0.f;
        drift = fine ? fmaf(-st.m, LP_LOG2E, m2) : 0.f;
        quick = fine ? st.m : -CUDART_INF_F;
    };
    float qs = 0.f, qt = 0.f;                          // the short path's sums since the last change of st.m
    auto flush = [&] {
        const float f = exp2f(drift);
        st.s = fmaf(f, qs, st.s);
        st.t += f * fmaf(drift, qs, qt);
        qs = qt = 0.f;
    };
    settle();
    auto slow = [&](float v) {
        if (!(v < CUDART_INF_F)) { st.s = st.t = CUDART_NAN_F; return; }
        if (v == -CUDART_INF_F) return;
        if (v > st.m) { flush(); raise(v); settle(); }
        if (v == st.m) st.n += 1.f;
        else { const float d = lp_d(v, st.m), e = exp2f(d); st.s += e; st.t = fmaf(e, d, st.t); }
    };
    auto push = [&](float v, int i) {
        const int c = atomicAdd(&count, 1);
        if (c < LP_LIST) list[c] = lp_key(v, i);
    };
    if (si >= 0) { slow(sv); if (top) push(sv, si); }
    const float bv = top ? lp_value(bound) : CUDART_INF_F;                // bound 0 (fewer elements than `top`): a NaN, and everything of the tile is pushed
    for (int v = v0; v < v1; v += LP_VECS * LP_THREADS) {
        uint4 b[LP_VECS];
        #pragma unroll
        for (int u = 0; u < LP_VECS; ++u) b[u] = a[u];
        if (v + LP_VECS * LP_THREADS < v1) load(v + LP_VECS * LP_THREADS);
        #pragma unroll
        for (int u = 0; u < LP_VECS; ++u) {
            const int i = v + u * LP_THREADS + tid;
            if (i >= v1) continue;
            float e[NV];
            lp_unpack<F32>(b[u], e);
            float c = e[0];
            #pragma unroll
            for (int j = 1; j < NV; ++j) c = lp_max(c, e[j]);
            if (c < quick) {
                #pragma unroll
                for (int j = 0; j < NV; ++j) {
                    const float d = fmaxf(fmaf(e[j], LP_LOG2E, -m2), -216.f), f = lp_exp2(d);
                    qs += f; qt = fmaf(f, d, qt);
                }
            } else {
                #pragma unroll
                for (int j = 0; j < NV; ++j) slow(e[j]);
            }
            if (top) {
                if (v == v0) {
                    #pragma unroll
                    for (int j = 0; j < NV; ++j) if (lp_key(e[j], head + i * NV + j) >= bound) push(e[j], head + i * NV + j);
                } else if (c > bv) {
                    #pragma unroll
                    for (int j = 0; j < NV; ++j) if (e[j] > bv) push(e[j], head + i * NV + j);
                }
            }
        }
    }
    flush();

    // ---- join the CTA's parts ----
    #pragma unroll
    for (int o = 16; o; o >>= 1) st = lp_join(st, lp_shfl(st, o));
    __syncthreads();
    if (lane == 0) stats[warp] = st;
    __syncthreads();
    if (warp == 0) {
        st = lane < LP_WARPS ? stats[lane] : LpStat{-CUDART_INF_F, 0.f, 0.f, 0.f};
        #pragma unroll
        for (int o = LP_WARPS / 2; o; o >>= 1) st = lp_join(st, lp_shfl(st, o));
        if (lane == 0) part = st;
    }
    if (top) {
        int n = count;
        if (n > LP_LIST) {
            // ---- radix selection: the digits of the bound from the top, until what reaches it fits the list ----
            unsigned long long prefix = 0ull;
            int want = top, shift = 56;
            auto each = [&](auto f) {                   // f(key), 0 for none; whole warps
                f(si >= 0 ? lp_key(sv, si) : 0ull);
                for (int v = v0; v < v1; v += LP_THREADS) {
                    const int i = v + tid;
                    float e[NV];
                    lp_unpack<F32>(i < v1 ? xv[i] : make_uint4(0u, 0u, 0u, 0u), e);
                    #pragma unroll
                    for (int j = 0; j < NV; ++j) f(i < v1 ? lp_key(e[j], head + i * NV + j) : 0ull);
                }
            };
            for (;; shift -= 8) {
                __syncthreads();
                if (tid < 256) hist[tid] = 0u;
                __syncthreads();
                each([&](unsigned long long k) {
                    const bool in = k && (shift == 56 || (k >> (shift + 8)) == (prefix >> (shift + 8)));
                    const unsigned int digit = in ? (unsigned int)(k >> shift) & 255u : 256u;
                    const unsigned int peers = __match_any_sync(0xffffffffu, digit);      // equal logits are what brings a row here
                    if (in && lane == __ffs(peers) - 1) atomicAdd(&hist[digit], (unsigned int)__popc(peers));
                });
                __syncthreads();
                if (tid == 0) {
                    unsigned int above = 0u;
                    int d = 255;
                    while (d > 0 && above + hist[d] < (unsigned int)want) above += hist[d--];
                    pick[0] = (unsigned int)d; pick[1] = above;
                }
                __syncthreads();
                prefix |= (unsigned long long)pick[0] << shift;
                want -= (int)pick[1];
                // top - want elements are above the prefix, hist[digit] share it
                if (shift == 0 || (unsigned int)(top - want) + hist[pick[0]] <= (unsigned int)LP_LIST) break;
            }
            __syncthreads();
            if (tid == 0) count = 0;
            __syncthreads();
            each([&](unsigned long long k) { if (k && k >= prefix) { const int c = atomicAdd(&count, 1); if (c < LP_LIST) list[c] = k; } });
            __syncthreads();
            n = min(count, LP_LIST);
        }
        unsigned long long k = 0ull;
        for (int c = warp * 32; c < n; c += LP_THREADS) {
            const unsigned long long q = lp_sort(c + lane < n ? list[c + lane] : 0ull, lane);
            k = lp_merge(k, q, lane);
        }
        lists[warp][lane] = k;
        lp_tree(lists, LP_WARPS, warp, lane);
    }

    // ---- join the cluster's parts in its first CTA ----
    LpStat all;
    if (C > 1) {
        cluster.sync();
        if (rank == 0) {
            all = part;
            for (int r = 1; r < C; ++r) all = lp_join(all, *cluster.map_shared_rank(&part, r));
            if (top) {
                if (warp > 0 && warp < C) lists[warp][lane] = (*cluster.map_shared_rank(&lists, warp))[0][lane];
                lp_tree(lists, C, warp, lane);
            }
        }
        cluster.sync();
        if (rank) return;
    } else {
        __syncthreads();
        all = part;
    }

    // ---- results ----
    const bool bad = !(all.s <= CUDART_INF_F), none = !bad && all.n == 0.f;        // +inf or NaN in the row; every logit -inf
    const float ln_s = all.n == 1.f ? log1pf(all.s) : logf(all.n + all.s);
    auto logp = [&](float v) { return bad ? CUDART_NAN_F : none ? -CUDART_INF_F : (v - all.m) - ln_s; };
    if (tid == 0) p.entropy[row] = bad ? CUDART_NAN_F : none ? 0.f : fmaxf(ln_s - all.t * LP_LN2 / (all.n + all.s), 0.f);
    for (int g = tid; g < p.G; g += LP_THREADS) {
        const int t = p.tokens[row * p.G + g];
        p.lp[row * p.G + g] = t < 0 ? 0.f : t >= V ? CUDART_NAN_F : logp(one(t));
    }
    if (tid < top) {
        const unsigned long long k = lists[0][tid];
        p.top_ids[row * top + tid] = bad ? -1 : lp_index(k);
        p.top_lp[row * top + tid] = logp(lp_value(k));
    }
}

template <bool F32>
static int lp_launch(const LpParams& p, int M, cudaStream_t s) {
    // CTAs per row: as many as leave the whole batch on the GPU at once (two CTAs per SM), and a tile's worth of work to each.
    int C = 8;
    while (C > 1 && ((long long)M * C > 2 * sm_count() || p.V / C < LP_THREADS * LpVec<F32>::N)) C >>= 1;
    cudaLaunchConfig_t lc{};
    lc.gridDim = dim3((unsigned)M * C); lc.blockDim = dim3(LP_THREADS); lc.stream = s;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = C; at[1].val.clusterDim.y = 1; at[1].val.clusterDim.z = 1;
    lc.attrs = at; lc.numAttrs = 2;
    if (cudaLaunchKernelEx(&lc, k_token_logprobs<F32>, p) != cudaSuccess) return launch_failed("k_token_logprobs");
    return check_launch("k_token_logprobs");
}

}  // namespace b200

using namespace b200;

extern "C" int b200_token_logprobs(const void* logits, int dtype, size_t ld, int M, int V, const int32_t* tokens, int G, float* logprobs,
                                   float* entropy, int top, int32_t* top_ids, float* top_logprobs, b200_stream stream) {
    if (!logits || !entropy || M < 1 || V < 1 || G < 0 || top < 0 || top > V || ld < (size_t)V || (dtype != B200_F32 && dtype != B200_BF16)) return B200_EINVAL;
    if ((G && (!tokens || !logprobs)) || (top && (!top_ids || !top_logprobs))) return B200_EINVAL;
    if (top > B200_LOGPROBS_TOP_MAX || M > I8_MAX_ROWS || V > (1 << 30)) return B200_ELIMIT;
    if (((uintptr_t)logits & (dtype == B200_F32 ? 3 : 1)) || ((uintptr_t)tokens & 3) || ((uintptr_t)logprobs & 3) || ((uintptr_t)entropy & 3) ||
        ((uintptr_t)top_ids & 3) || ((uintptr_t)top_logprobs & 3)) return B200_EALIGN;
    const LpParams p{logits, tokens, logprobs, entropy, top_ids, top_logprobs, ld, V, G, top};
    return dtype == B200_F32 ? lp_launch<true>(p, M, stream) : lp_launch<false>(p, M, stream);
}
