// logprobs.cu -- log probabilities of given tokens, the entropy, and the likeliest tokens, from one pass over the logits.
//
//   m = max x      S = sum exp(x - m)      log p(t) = (x_t - m) - ln S      H = ln S - (1 / S) sum (x - m) exp(x - m)
//
// A cluster of CTAs takes a row, each CTA a contiguous part of it, which bulk copies bring through a ring in shared memory; parts
// are joined over distributed shared memory.
//
// Statistics.  Every thread keeps (m, n, S, T): n elements equal to m (they count as exactly 1 and are not added), S and T in base 2
// over the others:
//   S = sum 2^d,  T = sum d 2^d,  d = (x - m) log2 e.
// So S is what is left beside the likeliest token, and ln(1 + S) of a token that is nearly certain keeps its relative precision
// (1 + S in f32 would not).  The threads start from the maximum of the CTA's first tile; a thread whose part of a tile holds nothing
// above it (nearly all) takes the short path: one multiply-add, one exponential, two sums per element.  d is the multiply-add
// fma(x, log2 e, -fl(m log2 e)): its distance from (x - m) log2 e is the same for every element and corrected when m changes.
//
// The likeliest tokens.  Order: logit descending, then index ascending, as one 64-bit key.  A bound is a value that at least `top`
// elements reach: the top-th of the largest maxima of every warp, 32 in all.  The first tile gives one, and later elements count only
// above it (an equal one has a larger index).  Vectors whose maximum counts go to a list in shared memory, and after 1, 4, 16, ...
// tiles the list gives a higher bound: some 200 vectors of a vocabulary of 154880 in no particular order.  In the end the elements
// of these vectors that reach the last bound, little more than `top`, are put in order by counting who is larger.  A list that
// overflows (logits in ascending order; a first tile of masked tokens before thousands of others) is dropped, and the CTA
// finds the top-th key by radix selection over its part instead.
//
// In replays: [2048 x 154880] f32 186 us (6.8 TB/s: reads alone exceed the rate of a copy), with 20 alternatives 214; bf16 126 and 169, where the
// exponential bounds the sums (16 a clock and SM are 75 us; the instructions of an element, about 10 in all, take not much less) and the top costs
// bounds and lists for which the stream waits at a row's two ends.  A long run of calls on f32 rows with 20
// alternatives takes 234 us a call.
// [512 x 154880] bf16 42 us: 512 rows on 148 SMs are 4 rows on some and 3 on others.  One row of 154880, top 5, 9.0 us, none of them a unit's limit: a
// chain of loads, barriers and exchanges.
#include "b200_internal.h"
#include "tma_pipe.cuh"
#include <cuda_bf16.h>
#include <cooperative_groups.h>
#include <math_constants.h>

namespace b200 {
namespace cg = cooperative_groups;

constexpr int LP_LIST = 512;                       // candidates of a CTA
constexpr int LP_VECS = 4;                         // 16-byte vectors of a tile that a thread has
constexpr int LP_STAGES = 3;
constexpr int LP_CLUSTER = 8;                      // CTAs of a row, at most
constexpr float LP_LOG2E = 1.44269504088896341f, LP_LN2 = 0.693147180559945309f;
static_assert(B200_LOGPROBS_TOP_MAX <= 32, "a bound is one of 32 maxima");

struct LpParams {
    const void* x; const int32_t* tokens; float* lp; float* entropy; int32_t* top_ids; float* top_lp;
    unsigned int* status; size_t ld; int V, G, top;
};

struct LpStat { float m, n, s, t; };               // see above; n as a float (n <= 2^24 exact; beyond it its last bit does not matter)

// Bits of logit x that order like it, never 0 but for a NaN.  -0 and +0 are the same logit.
__device__ __forceinline__ uint32_t lp_ordered(float x) {
    const uint32_t b = __float_as_uint(x + 0.f);
    return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float lp_unordered(uint32_t o) { return __uint_as_float((o & 0x80000000u) ? o ^ 0x80000000u : ~o); }
// 64-bit key of logit x at index i: orders by x descending, then i ascending.
__device__ __forceinline__ unsigned long long lp_key(float x, int i) { return ((unsigned long long)lp_ordered(x) << 32) | (0x7fffffffu - (uint32_t)i); }
__device__ __forceinline__ int lp_index(unsigned long long key) { return (int)(0x7fffffffu - (uint32_t)key); }
__device__ __forceinline__ float lp_value(unsigned long long key) { return lp_unordered((uint32_t)(key >> 32)); }
__device__ __forceinline__ float lp_exp2(float d) { float e; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(d)); return e; }
__device__ __forceinline__ float lp_max(float a, float b) { float r; asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b)); return r; }

// d = (x - m) log2 e in two steps, for any finite x and m.  -216 and below: 2^d is zero, d finite.
__device__ __forceinline__ float lp_d(float x, float m) { return fmaxf((x - m) * LP_LOG2E, -216.f); }

// The two halves of a cluster's barrier.  Shared memory of another CTA may be touched only when that CTA is known to have started: every
// thread arrives where it starts, and waits, long after all have, before the first store into the first CTA's memory.
__device__ __forceinline__ void lp_cluster_arrive() { asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory"); }
__device__ __forceinline__ void lp_cluster_wait() { asm volatile("barrier.cluster.wait;" ::: "memory"); }

// The warp's parts as one, in every lane.  Parts without elements have m = -inf, n = s = t = 0; s = NaN marks a row that holds +inf or NaN.
__device__ __forceinline__ LpStat lp_join(LpStat a) {
    const float m = lp_unordered(__reduce_max_sync(0xffffffffu, lp_ordered(a.m)));
    if (a.m != m) {
        const float d = lp_d(a.m, m), f = exp2f(d), all = a.n + a.s;
        a.t = f * (a.t + all * d); a.s = f * all; a.n = 0.f;
    }
    #pragma unroll
    for (int o = 16; o; o >>= 1) {
        a.n += __shfl_xor_sync(0xffffffffu, a.n, o);
        a.s += __shfl_xor_sync(0xffffffffu, a.s, o);
        a.t += __shfl_xor_sync(0xffffffffu, a.t, o);
    }
    return LpStat{m, a.n, a.s, a.t};
}

// A bound: the top-th of the largest two (four, eight) k of every one of 16 (8, 4) warps, 0 if there are not so many.  Every thread calls it and
// gets it.
template <int LP_THREADS>
__device__ __noinline__ uint32_t lp_bound(uint32_t k, int top) {
    __shared__ uint32_t w[32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    constexpr int EACH = 32 / (LP_THREADS / 32);
    uint32_t most[EACH];
    #pragma unroll
    for (int i = 0; i < EACH; ++i) {
        most[i] = __reduce_max_sync(0xffffffffu, k);
        if (lane == __ffs(__ballot_sync(0xffffffffu, k == most[i])) - 1) k = 0u;
    }
    __syncthreads();
    if (lane == 0) {
        #pragma unroll
        for (int i = 0; i < EACH; ++i) w[EACH * warp + i] = most[i];
    }
    __syncthreads();
    if (warp == 0) {
        const uint32_t v = w[lane];
        int r = 0;
        #pragma unroll
        for (int i = 0; i < 32; ++i) {
            const uint32_t o = __shfl_sync(0xffffffffu, v, i);
            r += o > v || (o == v && i < lane);
        }
        __syncwarp();
        if (r == top - 1) w[0] = v;
    }
    __syncthreads();
    return w[0];
}

// best[0 .. top - 1] <- the largest of list[0 .. n - 1], descending; all keys differ.
template <int LP_THREADS>
__device__ __forceinline__ void lp_rank(const unsigned long long (&list)[LP_LIST], int n, int top, unsigned long long (&best)[B200_LOGPROBS_TOP_MAX]) {
    for (int c = threadIdx.x; c < n; c += LP_THREADS) {
        const unsigned long long k = list[c];
        int r = 0;
        #pragma unroll 4
        for (int i = 0; i < n; ++i) r += list[i] > k;
        if (r < top) best[r] = k;
    }
}

__device__ __forceinline__ unsigned long long lp_pack(float a, float b) {
    unsigned long long r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 lp_unpack2(unsigned long long v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ unsigned long long lp_fma2(unsigned long long a, unsigned long long b, unsigned long long c) {
    unsigned long long r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ unsigned long long lp_add2(unsigned long long a, unsigned long long b) {
    unsigned long long r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
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

// The larger of two words: an f32 each, or two bf16 each.  A NaN wins.
template <bool F32>
__device__ __forceinline__ uint32_t lp_maxw(uint32_t a, uint32_t b) {
    uint32_t r;
    if (F32) r = __float_as_uint(lp_max(__uint_as_float(a), __uint_as_float(b)));
    else asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
// bf16: no element below -1e38, whose exponential is 0 and whose multiple by log2 e is finite (0 * inf would be a NaN).
template <bool F32>
__device__ __forceinline__ uint4 lp_finite(uint4 a) {
    if (!F32) {
        uint32_t* w = &a.x;
        #pragma unroll
        for (int j = 0; j < 4; ++j) asm("max.bf16x2 %0, %0, %1;" : "+r"(w[j]) : "r"(0xfe96fe96u));
    }
    return a;
}
template <bool F32>
__device__ __forceinline__ float lp_maxof(uint32_t w) {
    return F32 ? __uint_as_float(w) : lp_max(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}

template <bool F32, int LP_THREADS>
__global__ void __launch_bounds__(LP_THREADS, 1024 / LP_THREADS)
k_token_logprobs(const __grid_constant__ LpParams p) {
    constexpr int NV = LpVec<F32>::N, LP_WARPS = LP_THREADS / 32;
    constexpr int LP_TILE = LP_VECS * LP_THREADS;      // vectors
    constexpr uint32_t LP_TILE_BYTES = LP_TILE * 16;
    extern __shared__ __align__(128) unsigned char ring[];
    __shared__ uint64_t full_bar[LP_STAGES], empty_bar[LP_STAGES];
    __shared__ unsigned long long vecs[LP_LIST];       // candidates: (ordered maximum, vector)
    __shared__ unsigned long long list[LP_LIST];       // keys
    __shared__ unsigned long long best[B200_LOGPROBS_TOP_MAX];
    __shared__ LpStat stats[LP_WARPS];
    __shared__ LpStat part;
    __shared__ unsigned long long all_best[LP_CLUSTER][B200_LOGPROBS_TOP_MAX];      // in the cluster's first CTA: every CTA's
    __shared__ LpStat all_part[LP_CLUSTER];
    __shared__ int n_vecs, n_list;
    __shared__ unsigned int hist[256];
    __shared__ unsigned int pick[2];
    cg::cluster_group cluster = cg::this_cluster();
    const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const size_t row = blockIdx.x / C;
    const int V = p.V, top = p.top;
    if (C > 1) lp_cluster_arrive();
    if (tid == 0) {
        n_vecs = n_list = 0;
        #pragma unroll
        for (int i = 0; i < LP_STAGES; ++i) { mbar_init(smem_u32(&full_bar[i]), 1); mbar_init(smem_u32(&empty_bar[i]), LP_WARPS); }
        mbar_fence_init();
    }
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

    const int nt = (v1 - v0 + LP_TILE - 1) / LP_TILE;
    auto request = [&](int t) {                        // one thread: tile t into its stage
        const uint32_t bytes = (uint32_t)min(LP_TILE, v1 - v0 - t * LP_TILE) * 16u, s = (uint32_t)t % LP_STAGES;
        mbar_expect_tx(smem_u32(&full_bar[s]), bytes);
        bulk_g2s(smem_u32(ring) + s * LP_TILE_BYTES, xv + v0 + t * LP_TILE, bytes, smem_u32(&full_bar[s]));
    };
    // The first tile alone, the next ones when it has come: three at once from every CTA of a full GPU keep each of them waiting for 28 MB
    // ([296 x 154880] bf16 25.8 -> 23.8 us).
    if (tid == 0 && nt) request(0);
    const float sv = si >= 0 ? one(si) : -CUDART_INF_F;
    // this thread's given token, long before its log probability is known
    int token = -1;
    float token_x = 0.f;
    if (rank == 0 && tid < p.G) {
        token = p.tokens[row * p.G + tid];
        if ((unsigned)token < (unsigned)V) token_x = one(token);
    }
    __syncthreads();

    constexpr uint32_t MASKED = F32 ? 0xff800000u : 0xff80ff80u;
    uint4 a[LP_VECS];
    auto load = [&](int t) {                           // vectors u * LP_THREADS + tid of tile t; -inf past the part
        const int s = t % LP_STAGES;
        if (warp == 0 && t > 0 && t + LP_STAGES - 1 < nt) {        // the stage of the tile before, once every warp has read it
            mbar_wait(smem_u32(&empty_bar[(t - 1) % LP_STAGES]), (uint32_t)((t - 1) / LP_STAGES) & 1u, p.status, 26);
            if (elect_one()) request(t + LP_STAGES - 1);
            __syncwarp();
        }
        mbar_wait(smem_u32(&full_bar[s]), (uint32_t)(t / LP_STAGES) & 1u, p.status, 30);
        if (t == 0 && tid == 0)
            for (int i = 1; i < min(nt, LP_STAGES); ++i) request(i);
        const uint4* q = reinterpret_cast<const uint4*>(ring + (size_t)s * LP_TILE_BYTES) + tid;
        const int left = v1 - v0 - t * LP_TILE;
        if (left >= LP_TILE) {
            #pragma unroll
            for (int u = 0; u < LP_VECS; ++u) a[u] = q[u * LP_THREADS];
        } else {
            #pragma unroll
            for (int u = 0; u < LP_VECS; ++u) a[u] = u * LP_THREADS + tid < left ? q[u * LP_THREADS] : make_uint4(MASKED, MASKED, MASKED, MASKED);
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&empty_bar[s]));
    };

    // ---- first tile: the maximum, and a bound ----
    if (nt) load(0);
    else {
        #pragma unroll
        for (int u = 0; u < LP_VECS; ++u) a[u] = make_uint4(MASKED, MASKED, MASKED, MASKED);
    }
    float m = -CUDART_INF_F;
    #pragma unroll
    for (int u = 0; u < LP_VECS; ++u) {
        float v[NV];
        lp_unpack<F32>(a[u], v);
        #pragma unroll
        for (int j = 0; j < NV; ++j) m = fmaxf(m, v[j]);
    }
    uint32_t lo = top ? lp_bound<LP_THREADS>(v0 + tid < v1 ? lp_ordered(m) : 0u, top) : 0u;
    // A bound at the value of a mask would make candidates of all masked elements: if it is the maximum of many threads, what is above
    // it counts, and if that is too little in the end, the first elements of its value are added.  `held`: `top` elements of earlier
    // tiles reach the bound.
    const float low = lp_unordered(lo);
    bool held = true;
    {
        const uint32_t most = __reduce_max_sync(0xffffffffu, lp_ordered(fmaxf(m, sv)));
        if (lane == 0) hist[warp] = most;
        if (__syncthreads_count(lo && v0 + tid < v1 && lp_ordered(m) == lo) > LP_THREADS / 8) { ++lo; held = false; }
        m = lp_unordered(__reduce_max_sync(0xffffffffu, hist[lane & (LP_WARPS - 1)]));
    }
    // nothing to look for: +inf; no bound (fewer than 512 vectors): everything counts
    float bv = !top ? CUDART_INF_F : lo ? lp_unordered(lo) : -CUDART_INF_F;

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
    unsigned long long qs = 0ull, qt = 0ull;           // the short path's sums since the last change of st.m, two halves
    auto flush = [&] {
        const float2 s2 = lp_unpack2(qs), t2 = lp_unpack2(qt);
        const float s1 = s2.x + s2.y, t1 = t2.x + t2.y, f = exp2f(drift);
        st.s = fmaf(f, s1, st.s);
        st.t += f * fmaf(drift, s1, t1);
        qs = qt = 0ull;
    };
    settle();
    auto add = [&](float (&e)[NV]) {                   // elements below st.m, which is `fine`
        const unsigned long long l2 = lp_pack(LP_LOG2E, LP_LOG2E), n2 = lp_pack(-m2, -m2);
        #pragma unroll
        for (int j = 0; j < NV; j += 2) {
            float2 d = lp_unpack2(lp_fma2(lp_pack(e[j], e[j + 1]), l2, n2));
            if (F32) { d.x = fmaxf(d.x, -216.f); d.y = fmaxf(d.y, -216.f); }
            const unsigned long long f = lp_pack(lp_exp2(d.x), lp_exp2(d.y));
            qs = lp_add2(qs, f); qt = lp_fma2(f, lp_pack(d.x, d.y), qt);
        }
    };
    auto slow = [&](float v) {                         // an element that is no larger than st.m
        const float d = lp_d(v, st.m), e = v == st.m ? 0.f : lp_exp2(d);
        st.n += v == st.m ? 1.f : 0.f;
        st.s += e; st.t = fmaf(e, d, st.t);
    };
    auto push = [&](float v, int i) {
        const int c = atomicAdd(&n_list, 1);
        if (c < LP_LIST) list[c] = lp_key(v, i);
    };
    // the candidates' maxima, a thread's largest; entry e belongs to warp e % LP_WARPS, so that every warp has some
    auto entry = [&](int n) {
        uint32_t k = 0u;
        for (int e = lane * LP_WARPS + warp; e < n; e += LP_THREADS) k = max(k, (uint32_t)(vecs[e] >> 32));
        return k;
    };
    #pragma unroll 1
    for (int t = 0; t < nt; ++t) {
        uint32_t c[LP_VECS];                           // the vectors' maxima, a NaN if they hold one (bf16: of even and of odd elements)
        #pragma unroll
        for (int u = 0; u < LP_VECS; ++u) c[u] = lp_maxw<F32>(lp_maxw<F32>(a[u].x, a[u].y), lp_maxw<F32>(a[u].z, a[u].w));
        const float most = lp_maxof<F32>(lp_maxw<F32>(lp_maxw<F32>(c[0], c[1]), lp_maxw<F32>(c[2], c[3])));
        if (most < quick) {
            #pragma unroll
            for (int u = 0; u < LP_VECS; ++u) {
                float e[NV];
                lp_unpack<F32>(lp_finite<F32>(a[u]), e);
                add(e);
            }
        } else if (!(most < CUDART_INF_F)) st.s = st.t = CUDART_NAN_F;
        else if (most > -CUDART_INF_F) {               // a new maximum, or an equal one: those that equal it are counted, not added
            if (most > st.m) { flush(); raise(most); settle(); }
            #pragma unroll 1
            for (int u = 0; u < LP_VECS; ++u) {
                uint4 w = a[0];
                #pragma unroll
                for (int i = 1; i < LP_VECS; ++i) if (u == i) w = a[i];
                float e[NV];
                lp_unpack<F32>(w, e);
                #pragma unroll
                for (int j = 0; j < NV; ++j)
                    if (e[j] == st.m) { st.n += 1.f; e[j] = -CUDART_INF_F; }
                if (quick == st.m) {                   // `fine`
                    #pragma unroll
                    for (int j = 0; j < NV; ++j) e[j] = fmaxf(e[j], -1e38f);
                    add(e);
                }
                else {
                    #pragma unroll
                    for (int j = 0; j < NV; ++j) slow(e[j]);
                }
            }
        }
        if (top && most >= bv) {
            const int left = v1 - v0 - t * LP_TILE;
            #pragma unroll
            for (int u = 0; u < LP_VECS; ++u) {
                const int i = u * LP_THREADS + tid;
                const float cu = lp_maxof<F32>(c[u]);
                if ((t == 0 || !held ? cu >= bv : cu > bv) && i < left) {
                    const int e = atomicAdd(&n_vecs, 1);
                    if (e < LP_LIST) vecs[e] = ((unsigned long long)lp_ordered(cu) << 32) | (uint32_t)(v0 + t * LP_TILE + i);
                }
            }
        }
        if (t + 1 < nt) load(t + 1);
        if (!(t & (t + 1)) && ((t + 1) & 0x55555555) && t + 4 < nt) {      // 1, 4, 16, ... tiles are done and more than three are left
            // the CTA's maximum so far for all, at places that do not change from run to run
            const uint32_t most_o = __reduce_max_sync(0xffffffffu, lp_ordered(st.m));
            __syncthreads();
            if (lane == 0) hist[warp] = most_o;
            const int n = n_vecs;
            __syncthreads();
            const float mm = lp_unordered(__reduce_max_sync(0xffffffffu, hist[lane & (LP_WARPS - 1)]));
            if (mm > st.m) { flush(); raise(mm); settle(); }
            if (top && n <= LP_LIST) {
                const uint32_t b = lp_bound<LP_THREADS>(entry(n), top);
                if (b >= lo && b) { lo = b; bv = lp_unordered(b); held = true; }
            }
        }
    }
    // single elements; those of the tail come after all others
    flush();
    if (si >= 0) {
        if (!(sv < CUDART_INF_F)) st.s = st.t = CUDART_NAN_F;
        else if (sv > -CUDART_INF_F) slow(sv);         // st.m started no lower
        if (top && lp_ordered(sv) >= lo) push(sv, si);
    }

    // ---- join the CTA's parts ----
    st = lp_join(st);
    if (lane == 0) stats[warp] = st;
    __syncthreads();
    if (warp == 0) {
        st = lp_join(lane < LP_WARPS ? stats[lane] : LpStat{-CUDART_INF_F, 0.f, 0.f, 0.f});
        if (lane == 0) part = st;
    }
    if (top) {
        const int n = n_vecs;
        if (n <= LP_LIST) {
            lo = max(lo, lp_bound<LP_THREADS>(entry(n), top));
            for (int i = tid; i < n; i += LP_THREADS) {
                if ((uint32_t)(vecs[i] >> 32) < lo) continue;
                const int q = (int)(uint32_t)vecs[i];
                float f[NV];
                const int o = q - v0, t = o / LP_TILE;             // the last tiles still lie in the ring
                lp_unpack<F32>(t + LP_STAGES >= nt ? reinterpret_cast<const uint4*>(ring + (size_t)(t % LP_STAGES) * LP_TILE_BYTES)[o - t * LP_TILE] : xv[q], f);
                #pragma unroll
                for (int j = 0; j < NV; ++j) if (lp_ordered(f[j]) >= lo) push(f[j], head + q * NV + j);
            }
        }
        __syncthreads();
        if (n <= LP_LIST && n_list < top) {            // no more than top - 1 are above `low`; if no other element lies below it, the first 64 are enough
            __syncthreads();
            const int i = (rank == 0 ? 0 : head + v0 * NV) + tid;
            if (tid < 2 * B200_LOGPROBS_TOP_MAX && i < (rank == C - 1 ? V : head + v1 * NV)) {
                const float f = one(i);
                if (f == low) push(f, i);
            }
            __syncthreads();
        }
        if ((n > LP_LIST || n_list > LP_LIST || n_list < top) && !(part.s != part.s)) {
            // ---- radix selection: the digits of the top-th key from the top, until few enough reach it ----
            constexpr unsigned int FEW = 128;
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
                for (int i = tid; i < 256; i += LP_THREADS) hist[i] = 0u;
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
                if (shift == 0 || (unsigned int)(top - want) + hist[pick[0]] <= FEW) break;
            }
            __syncthreads();
            if (tid == 0) n_list = 0;
            __syncthreads();
            each([&](unsigned long long k) { if (k && k >= prefix) { const int c = atomicAdd(&n_list, 1); if (c < LP_LIST) list[c] = k; } });
            __syncthreads();
        }
        lp_rank<LP_THREADS>(list, min(n_list, LP_LIST), top, best);
    }

    // ---- join the cluster's parts in its first CTA ----
    if (C > 1) {
        lp_cluster_wait();                             // the first CTA has started
        __syncthreads();                               // best and part
        if (tid < top) cluster.map_shared_rank(&all_best[0][0], 0)[rank * B200_LOGPROBS_TOP_MAX + tid] = best[tid];
        if (tid == 0) { cluster.map_shared_rank(all_part, 0)[rank] = part; n_list = 0; }
        __syncwarp();
        cluster.sync();
        if (rank) return;
        if (top) {
            // no CTA's last one is above the row's top-th
            unsigned long long least = all_best[0][top - 1];
            for (int r = 1; r < C; ++r) least = max(least, all_best[r][top - 1]);
            for (int r = warp; r < C; r += LP_WARPS) {
                const unsigned long long k = lane < top ? all_best[r][lane] : 0ull;
                if (k && k >= least) list[atomicAdd(&n_list, 1)] = k;
            }
            __syncthreads();
            lp_rank<LP_THREADS>(list, n_list, top, best);
        }
        if (warp == 0) {
            const LpStat all = lp_join(lane < C ? all_part[lane] : LpStat{-CUDART_INF_F, 0.f, 0.f, 0.f});
            if (lane == 0) stats[0] = all;
        }
    } else if (tid == 0) stats[0] = part;
    __syncthreads();
    const LpStat all = stats[0];

    // ---- results ----
    const bool bad = !(all.s <= CUDART_INF_F), none = !bad && all.n == 0.f;        // +inf or NaN in the row; every logit -inf
    const float ln_s = all.n == 1.f ? log1pf(all.s) : logf(all.n + all.s);
    auto logp = [&](float v) { return bad ? CUDART_NAN_F : none ? -CUDART_INF_F : (v - all.m) - ln_s; };
    if (tid == 0) p.entropy[row] = bad ? CUDART_NAN_F : none ? 0.f : fmaxf(ln_s - all.t * LP_LN2 / (all.n + all.s), 0.f);
    for (int g = tid; g < p.G; g += LP_THREADS) {
        if (g >= LP_THREADS) {
            token = p.tokens[row * p.G + g];
            if ((unsigned)token < (unsigned)V) token_x = one(token);
        }
        p.lp[row * p.G + g] = token < 0 ? 0.f : token >= V ? CUDART_NAN_F : logp(token_x);
    }
    if (tid < top) {
        const unsigned long long k = best[tid];
        p.top_ids[row * top + tid] = bad ? -1 : lp_index(k);
        p.top_lp[row * top + tid] = logp(lp_value(k));
    }
}

template <bool F32, int THREADS>
static int lp_launch(const LpParams& p, int M, int C, cudaStream_t s) {
    auto kern = k_token_logprobs<F32, THREADS>;
    constexpr size_t smem = (size_t)LP_STAGES * LP_VECS * THREADS * 16;
    static bool ready[64] = {};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return launch_failed("token_logprobs: cudaGetDevice");
    if (dev < 0 || dev >= 64 || !ready[dev]) {
        if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess)
            return launch_failed("token_logprobs: cudaFuncSetAttribute");
        if (dev >= 0 && dev < 64) ready[dev] = true;
    }
    cudaLaunchConfig_t lc{};
    lc.gridDim = dim3((unsigned)M * C); lc.blockDim = dim3(THREADS); lc.dynamicSmemBytes = smem; lc.stream = s;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = C; at[1].val.clusterDim.y = 1; at[1].val.clusterDim.z = 1;
    lc.attrs = at; lc.numAttrs = C > 1 ? 2 : 1;
    if (cudaLaunchKernelEx(&lc, kern, p) != cudaSuccess) return launch_failed("k_token_logprobs");
    return check_launch("k_token_logprobs");
}

template <bool F32>
static int lp_choose(const LpParams& p, int M, cudaStream_t s) {
    // CTAs per row: as many as leave the whole batch on the GPU at once (two CTAs per SM), and a tile's worth of work to each.
    int C = LP_CLUSTER;
    while (C > 1 && ((long long)M * C > 2 * sm_count() || p.V / C < 512 * LP_VECS * LpVec<F32>::N)) C >>= 1;
    // Threads per CTA: few large CTAs where a row's time counts, small ones, whose barriers cost the others nothing, where there are rows enough.
    // 12 KB of an SM's shared memory go to each CTA besides its ring (and 1 KB to the system), so two of 512 threads have room on it, three of 256
    // or six of 128; the launch bounds hold each form to 64 registers, which only the first needs.  us with 512 / 256 / 128: [1 x 154880] f32,
    // top 5 9.2 / 11.7 / 16.1; [200 x 20000] f32, top 20 11.7 / 15.0 / 21.9; [300 x 1000] f32, top 5 11.7 / 6.8 / 7.2; [2048 x 154880] f32, top 20
    // 223 / 214 / 236, bf16 181 / 170 / 167; [2000 x 20000] bf16, top 20 69.7 / 54.4 / 54.3; [2000 x 600] bf16, top 5 53.3 / 33.6 / 21.3.
    const size_t vecs = (size_t)p.V / LpVec<F32>::N;
    if (M > 4 * sm_count()) return vecs <= 8192 ? lp_launch<F32, 128>(p, M, C, s) : lp_launch<F32, 256>(p, M, C, s);
    return C == 1 && vecs <= 1024 ? lp_launch<F32, 256>(p, M, C, s) : lp_launch<F32, 512>(p, M, C, s);
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
    LpParams p{logits, tokens, logprobs, entropy, top_ids, top_logprobs, device_status_ptr(), ld, V, G, top};
    if (!p.status) return B200_ENOTIMPL;
    return dtype == B200_F32 ? lp_choose<true>(p, M, stream) : lp_choose<false>(p, M, stream);
}
