// What given tokens weigh in whole rows of logits (sz_logprob_rows): their log probabilities and ranks, the rows' entropies and best alternatives.
//
// With x_i = (v_i - max) / T and s = the sum of e^x over all but one largest, log p = x - log1p(s) and the entropy is log1p(s) - sum(e^x x) / (1 + s):
// no difference of like numbers, whatever the distribution.  One pass over the row: a warp keeps the largest so far (the same for its lanes, so that a
// new one is rare) and both sums beside it.  A thread's elements come in groups of LP_G vectors; what a group's largest is stays in shared memory, and the
// best `top` are looked for afterwards in the few groups that can hold them: a bound that `top` threads reach, by halving, then what is not below it.
// A row is a cluster of 1 to 8 blocks, each with its part of it.  Rows of 151,936: one of f32, top 5, 8.3 us (the chain load, bound, gather, order and two barriers of the
// cluster); 64 of f32, top 20, 17.4 (39 MB: 5.9); 1,021 of bf16, top 1, 69 where they score their best, 87 with a fifth of them scoring any token (310 MB: 47; the exponentials' pipe alone takes 35, and an element some 8 instructions).
// A token that is masked itself has all that is not before it, and its row's elements are looked at one by one again: 64 such rows of f32 take 76 us instead of 21, 250 of bf16 150 instead of 23.
#include "sz_common.cuh"

#include <cuda_bf16.h>

#include <math.h>

namespace {

constexpr int LP_G = 4, LP_MAX_VOCAB = 1 << 18, LP_ID = 18, LP_TOP = 64, LP_LIST = 2048, LP_SM = 148;

struct LpArgs {
    const u8* logits;
    long long stride;                // bytes
    int rows, vocab, per, C, top;    // per: elements of a block's part
    int groups;                      // of a thread
    const int32_t* tokens;
    const float* temperature;
    float *logprob, *entropy;
    int32_t *rank, *top_ids;
    float* top_logprobs;
};

template <int LP_NTH> struct LpSmem {
    static constexpr int LP_NW = LP_NTH / 32;
    u64 list[LP_LIST];               // keys of the candidates
    u64 best[8 * LP_TOP];            // block 0: what the blocks found, in order
    u32 hit[8 * LP_TOP];             // groups that can hold any of the best
    u32 tmax[LP_NTH];
    float wm[LP_NW], ws[LP_NW], wx[LP_NW];
    u32 wc[LP_NW];
    float4 part[8];                  // block 0: the parts' sums, and how many are larger than the token's
    float m, thr;                    // of the block's part
    u32 n, hits;
};

template <int TYPE> struct LpVec { static constexpr int ESZ = TYPE == SZ_TYPE_F32 ? 4 : 2, N = 16 / ESZ; };
template <int TYPE>
__device__ __forceinline__ float lp_at(const u32* w, int i) {       // element i of vectors side by side
    if constexpr (TYPE == SZ_TYPE_F32) return __uint_as_float(w[i]);
    else if constexpr (TYPE == SZ_TYPE_F16) return __half2float(__ushort_as_half((u16)(w[i / 2] >> (16 * (i & 1)))));
    else return __uint_as_float(i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
}
template <int TYPE>
__device__ __forceinline__ float lp_one(const u8* p) {
    if constexpr (TYPE == SZ_TYPE_F32) return __ldcg((const float*)p);
    else if constexpr (TYPE == SZ_TYPE_F16) return __half2float(__ushort_as_half(__ldcg((const u16*)p)));
    else return __uint_as_float((u32)__ldcg((const u16*)p) << 16);
}
// NaN counts as -inf
__device__ __forceinline__ float lp_clean(float v) { return fmaxf(v, -INFINITY); }
// larger logits first, equal ones (0 and -0 too) by id
__device__ __forceinline__ u32 lp_up(float v) { const u32 x = __float_as_uint(v), b = x == 0x80000000u ? 0u : x; return b & 0x80000000u ? ~b : b | 0x80000000u; }
__device__ __forceinline__ float lp_down(u32 up) { return __uint_as_float(up & 0x80000000u ? up & 0x7fffffffu : ~up); }
__device__ __forceinline__ u64 lp_key(float v, u32 id) { return ((u64)(~lp_up(v)) << LP_ID) | id; }
__device__ __forceinline__ u32 lp_remote(const void* p, int rank) {
    u32 a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(sz_smem_addr(p)), "r"(rank));
    return a;
}
__device__ __forceinline__ void lp_st64(void* p, int rank, u64 v) { asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(lp_remote(p, rank)), "l"(v) : "memory"); }
__device__ __forceinline__ void lp_st128(void* p, int rank, float4 v) {
    asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(lp_remote(p, rank)), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w) : "memory");
}
__device__ __forceinline__ float lp_exp2(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
__device__ __forceinline__ void lp_sync(int C) { if (C > 1) sz_cluster_sync(); else __syncthreads(); }

// f32x2 arithmetic
__device__ __forceinline__ u64 lp_pack(float a, float b) { u64 d; asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(a), "f"(b)); return d; }
__device__ __forceinline__ u64 lp_add2(u64 a, u64 b) { u64 d; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b)); return d; }
__device__ __forceinline__ u64 lp_mul2(u64 a, u64 b) { u64 d; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b)); return d; }
__device__ __forceinline__ void lp_fma2(u64& a, u64 f, u64 x) { asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(a) : "l"(f), "l"(x)); }
// (largest, sum of the others' weights beside it, sum of weights times exponents) of two parts; exponents to the base 2
struct LpSum { float m, s, x; };
__device__ __forceinline__ LpSum lp_join(const LpSum a, const LpSum b, float c) {
    const LpSum hi = a.m >= b.m ? a : b, lo = a.m >= b.m ? b : a;
    if (lo.m == -INFINITY) return hi;
    const float d = fmaxf((lo.m - hi.m) * c, -200.f), w = lp_exp2(d);      // (of equal infinities: whatever, such a row is its first largest alone)
    return {hi.m, fmaf(w, 1.f + lo.s, hi.s), fmaf(w, fmaf(1.f + lo.s, d, lo.x), hi.x)};
}

template <int TYPE, int LP_NTH>
__global__ void __launch_bounds__(LP_NTH, 1024 / LP_NTH)
sz_logprob_kernel(const LpArgs a) {
    using V = LpVec<TYPE>;
    using Sm = LpSmem<LP_NTH>;
    constexpr int LP_NW = LP_NTH / 32;
    constexpr int N = V::N, GE = LP_G * N;               // elements of a vector and of a group
    extern __shared__ __align__(16) u8 lp_smem[];
    Sm* const S = (Sm*)lp_smem;
    float* const gmax = (float*)(lp_smem + sizeof(Sm));        // [group][thread]
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, row = blockIdx.x / a.C, rank = blockIdx.x % a.C;
    if (tid == 0) S->n = 0;
    if (a.C > 1) sz_cluster_arrive();                    // (block 0's shared memory is written to once all have begun)
    sz_pdl_wait();
    sz_pdl_trigger();
    const u8* const base = a.logits + (size_t)row * a.stride;
    const int e0 = min(rank * a.per, a.vocab), e1 = min(e0 + a.per, a.vocab);      // the block's part
    // whole 16-byte vectors of memory from element `id0` on, and up to N - 1 elements before and behind them
    const int lead = min(e1 - e0, (int)((16 - (((size_t)base + (size_t)e0 * V::ESZ) & 15)) & 15) / V::ESZ);
    const int id0 = e0 + lead, nvec = (e1 - id0) / N;
    const u8* const vbase = base + (size_t)id0 * V::ESZ;
    constexpr u32 NONE = TYPE == SZ_TYPE_F32 ? 0xff800000u : TYPE == SZ_TYPE_F16 ? 0xfc00fc00u : 0xff80ff80u;      // -inf
    auto load = [&](int v, u32* w) {
        const uint4 q = __ldcg((const uint4*)(vbase + (size_t)v * 16));
        w[0] = q.x; w[1] = q.y; w[2] = q.z; w[3] = q.w;
    };
    const int whole = nvec / (LP_G * LP_NTH), last = a.groups - 1;       // (the last group: what lies beside the vectors)
    auto ask = [&](int g, u32* w) {                      // the vectors of a group
        const int v0 = g * LP_G * LP_NTH + tid;
        if (g < whole) {
#pragma unroll
            for (int j = 0; j < LP_G; j++) load(v0 + j * LP_NTH, w + 4 * j);
        } else {
#pragma unroll
            for (int j = 0; j < LP_G; j++) {
                w[4 * j] = w[4 * j + 1] = w[4 * j + 2] = w[4 * j + 3] = NONE;
                if (v0 + j * LP_NTH < nvec) load(v0 + j * LP_NTH, w + 4 * j);
            }
        }
    };
    // few rows: a group ahead (with many, other blocks' warps are under way meanwhile, and registers are few)
    constexpr bool AHEAD = LP_NTH == 512;
    u32 ahead[AHEAD ? 4 * LP_G : 1];
    if constexpr (AHEAD) ask(0, ahead);
    int token = a.tokens ? a.tokens[row] : -1;
    if ((u32)token >= (u32)a.vocab) token = -1;
    const float tv = token >= 0 ? lp_clean(lp_one<TYPE>(base + (size_t)token * V::ESZ)) : INFINITY;
    const float tv_next = lp_down(lp_up(tv) + 1);        // (of a finite one; of the largest: infinity)
    const float T = a.temperature ? a.temperature[row] : 1.f, inv_t = 1.f / T;
    const bool alone = !(T > 0.f) || !(inv_t <= 3.4e38f);            // the best token has it all
    const float c = alone ? 0.f : fminf(inv_t * 1.4426950408889634f, 3.4e38f);      // (finite, so that equal largest ones, 0 times it, weigh 1)
    auto edge = [&](int v, u32* w) {                     // vector -1: the elements before the first, nvec: those behind the last
#pragma unroll
        for (int i = 0; i < 4; i++) {
            constexpr int P = 4 / V::ESZ;                // elements a word
            w[i] = 0;
#pragma unroll
            for (int k = 0; k < P; k++) {
                const int id = id0 + v * N + i * P + k;
                u32 e = NONE >> (32 - 8 * V::ESZ);
                if (id >= e0 && id < e1) { if constexpr (TYPE == SZ_TYPE_F32) e = __ldcg((const u32*)(base + (size_t)id * 4)); else e = __ldcg((const u16*)(base + (size_t)id * 2)); }
                w[i] |= e << (8 * V::ESZ * k) % 32;
            }
        }
    };
    float m = -INFINITY, s = 0.f, x = 0.f, tmax = -INFINITY;         // of the warp (m), of the thread (the others)
    u32 cnt = 0;
    // one group: vectors v0, v0 + LP_NTH, .. (elements that are nobody's are -inf)
    auto take = [&](int g, int v0, const u32* w) {
        float gm = -INFINITY;
        if constexpr (TYPE == SZ_TYPE_F32) {
#pragma unroll
            for (int i = 0; i < GE; i++) gm = fmaxf(gm, lp_at<TYPE>(w, i));
        } else {                                         // two at a time
            u32 p = NONE;
#pragma unroll
            for (int i = 0; i < 4 * LP_G; i++) {
                if constexpr (TYPE == SZ_TYPE_F16) { const __half2 h = __hmax2(*(const __half2*)&p, *(const __half2*)(w + i)); p = *(const u32*)&h; }
                else { const __nv_bfloat162 h = __hmax2(*(const __nv_bfloat162*)&p, *(const __nv_bfloat162*)(w + i)); p = *(const u32*)&h; }
            }
            gm = fmaxf(lp_at<TYPE>(&p, 0), lp_at<TYPE>(&p, 1));
        }
        if (a.top) gmax[g * LP_NTH + tid] = gm;
        tmax = fmaxf(tmax, gm);
        // larger than the token's logit, or equal with a lower id: not below it before the token, not below the next number behind it
        if (gm >= tv && token >= 0) {
            if (tv == -INFINITY || g == last) {
#pragma unroll 1
                for (int i = 0; i < GE; i++) {
                    const int at = v0 + (i / N) * LP_NTH, id = id0 + at * N + i % N;
                    const bool there = g == last ? tid < 2 && i < N : at < nvec;
                    if (!there || id < e0 || id >= e1) continue;
                    const float v = lp_clean(lp_one<TYPE>(base + (size_t)id * V::ESZ));
                    cnt += v > tv || (v == tv && id < token) ? 1u : 0u;
                }
            } else {
#pragma unroll
                for (int j = 0; j < LP_G; j++) {
                    const int id = id0 + (v0 + j * LP_NTH) * N;
                    if (id <= token && token < id + N) {             // the token's own vector
#pragma unroll
                        for (int i = 0; i < N; i++) { const float v = lp_at<TYPE>(w + 4 * j, i); cnt += v > tv || (v == tv && id + i < token) ? 1u : 0u; }
                    } else {
                        const float from = id < token ? tv : tv_next;
#pragma unroll
                        for (int i = 0; i < N; i++) cnt += lp_at<TYPE>(w + 4 * j, i) >= from ? 1u : 0u;
                    }
                }
            }
        }
        const float wm = lp_down(__reduce_max_sync(0xffffffffu, lp_up(gm)));
        const bool wm_new = wm > m;
        bool skip = false;
        if (wm_new) {                                    // (the same for the whole warp)
            if (m > -INFINITY) {                             // the old largest is one of the others now: lane 0 has it
                const float d = fmaxf((m - wm) * c, -200.f), f = lp_exp2(d);
                const float t = s + (lane == 0 ? 1.f : 0.f);
                x = f * fmaf(t, d, x);
                s = f * t;
            }
            m = wm;
            skip = lane == __ffs(__ballot_sync(0xffffffffu, gm == wm)) - 1;
        }
        const u64 m2 = lp_pack(-m, -m), c2 = lp_pack(c, c);
        u64 gs = 0, gx = 0;
        if (wm_new) {                                    // .. where there is a new largest, it (and what equals it in its lane) weighs nothing here
            int n = skip ? -1 : 0;                           // .. the others of these are put back: they weigh 1
#pragma unroll
            for (int i = 0; i < GE; i += 2) {
                const u64 e2 = lp_mul2(lp_add2(lp_pack(lp_at<TYPE>(w, i), lp_at<TYPE>(w, i + 1)), m2), c2);
                float e = fmaxf(__uint_as_float((u32)e2), -200.f), f = fmaxf(__uint_as_float((u32)(e2 >> 32)), -200.f);
                if (skip && lp_at<TYPE>(w, i) == m) { n++; e = -200.f; }
                if (skip && lp_at<TYPE>(w, i + 1) == m) { n++; f = -200.f; }
                const u64 p = lp_pack(lp_exp2(e), lp_exp2(f));
                gs = lp_add2(gs, p);
                lp_fma2(gx, p, lp_pack(e, f));
            }
            s += (float)n;
        } else {
#pragma unroll
            for (int i = 0; i < GE; i += 2) {
                const u64 e2 = lp_mul2(lp_add2(lp_pack(lp_at<TYPE>(w, i), lp_at<TYPE>(w, i + 1)), m2), c2);
                const float e = fmaxf(__uint_as_float((u32)e2), -200.f), f = fmaxf(__uint_as_float((u32)(e2 >> 32)), -200.f);
                const u64 p = lp_pack(lp_exp2(e), lp_exp2(f));
                gs = lp_add2(gs, p);
                lp_fma2(gx, p, lp_pack(e, f));
            }
        }
        s += __uint_as_float((u32)gs) + __uint_as_float((u32)(gs >> 32));
        x += __uint_as_float((u32)gx) + __uint_as_float((u32)(gx >> 32));
    };
#pragma unroll 1
    for (int g = 0; g < last; g++) {
        u32 w[4 * LP_G];
        const int v0 = g * LP_G * LP_NTH + tid;
        if constexpr (AHEAD) {
#pragma unroll
            for (int i = 0; i < 4 * LP_G; i++) w[i] = ahead[i];
            ask(g + 1, ahead);
        } else ask(g, w);
        take(g, v0, w);
    }
    if (a.top) gmax[last * LP_NTH + tid] = -INFINITY;
    if (warp == 0 && (lead || (e1 - id0) % N)) {         // threads 0 and 1: before and behind
        u32 w[4 * LP_G];
#pragma unroll
        for (int i = 0; i < 4 * LP_G; i++) w[i] = NONE;
        const int v = tid == 0 ? -1 : tid == 1 ? nvec : 0x3fffff;        // (a vector that no element is in)
        if (tid < 2) edge(v, w);
        take(last, v, w);
    }
    // ---- the block's part, then the row's
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) { s += __shfl_xor_sync(0xffffffffu, s, o); x += __shfl_xor_sync(0xffffffffu, x, o); }
    cnt = __reduce_add_sync(0xffffffffu, cnt);
    if (lane == 0) { S->wm[warp] = m; S->ws[warp] = s; S->wx[warp] = x; S->wc[warp] = cnt; }
    __syncthreads();
    float4 mine = make_float4(0.f, 0.f, 0.f, 0.f);       // (warp 0's)
    if (warp == 0) {
        LpSum t = lane < LP_NW ? LpSum{S->wm[lane], S->ws[lane], S->wx[lane]} : LpSum{-INFINITY, 0.f, 0.f};
        u32 n = lane < LP_NW ? S->wc[lane] : 0;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) t = lp_join(t, {__shfl_xor_sync(0xffffffffu, t.m, o), __shfl_xor_sync(0xffffffffu, t.s, o), __shfl_xor_sync(0xffffffffu, t.x, o)}, c);
        n = __reduce_add_sync(0xffffffffu, n);
        mine = {t.m, t.s, t.x, __uint_as_float(n)};
        if (lane == 0) S->m = t.m;
    }
    __syncthreads();
    const int top = a.top, have = e1 - e0, want = min(top, have);
    if (a.C > 1) sz_cluster_wait();
    if (tid == 0) { if (a.C > 1) lp_st128(&S->part[rank], 0, mine); else S->part[0] = mine; }
    if (want > 0) {
        // ---- the part's best: a bound that `want` threads' largest reach
        float thr = S->m;
        if (want > 1) {                                  // (one warp looks at all threads' largest: no barrier a step)
            S->tmax[tid] = lp_up(tmax);
            __syncthreads();
            if (warp == 0) {
                u32 k[LP_NW];
#pragma unroll
                for (int i = 0; i < LP_NW; i++) k[i] = S->tmax[32 * i + lane];
                u32 hi = lp_up(thr), lo = k[0];
#pragma unroll
                for (int i = 1; i < LP_NW; i++) lo = min(lo, k[i]);
                lo = __reduce_min_sync(0xffffffffu, lo);
                // (lo: reached by all; hi: by one at least)
                for (int step = 0; step < 32 && hi - lo > 1; step++) {
                    const u32 mid = lo + (hi - lo) / 2;
                    u32 n = 0;
#pragma unroll
                    for (int i = 0; i < LP_NW; i++) n += k[i] >= mid;
                    n = __reduce_add_sync(0xffffffffu, n);
                    if (n >= (u32)want) lo = mid; else hi = mid;
                    if (n >= (u32)want && n <= (u32)want + 16) break;
                }
                if (lane == 0) S->thr = lp_down(lo);
            }
            __syncthreads();
            thr = S->thr;
        }
        // the elements not below a bound (or above it): the groups that hold any are listed, then each element is one thread's
        auto gather = [&](float from, bool equal) {
            u32* const hits = S->hit;
            constexpr u32 HITS = 8 * LP_TOP;
            if (tid == 0) S->hits = 0;
            __syncthreads();
            for (int g = 0; g < a.groups; g++) {
                const float gm = gmax[g * LP_NTH + tid];
                if (equal ? gm >= from : gm > from) { const u32 at = atomicAdd(&S->hits, 1u); if (at < HITS) hits[at] = (u32)(g * LP_NTH + tid); }
            }
            __syncthreads();
            const u32 n = S->hits;
            if (n > HITS) { if (tid == 0) S->n = LP_LIST + 1; return; }
            for (u32 i = tid; i < n * GE; i += LP_NTH) {
                const u32 hit = hits[i / GE], e = i % GE;
                const int g = hit / LP_NTH, who = hit % LP_NTH, v = g == last ? (who == 0 ? -1 : nvec) : (g * LP_G + (int)(e / N)) * LP_NTH + who;
                const int id = id0 + v * N + (int)(e % N);
                if (id < e0 || id >= e1 || (g == last ? e >= N || who > 1 : v >= nvec)) continue;
                const float f = lp_clean(lp_one<TYPE>(base + (size_t)id * V::ESZ));
                if (!(equal ? f >= from : f > from)) continue;
                const u32 place = atomicAdd(&S->n, 1u);
                if (place < LP_LIST) S->list[place] = lp_key(f, id);
            }
        };
        gather(thr, true);
        __syncthreads();
        u32 n = S->n;
        if (n > (u32)LP_LIST) {                          // thousands that reach it (equal ones, masked rows): the bound is made exact
            u32 lo = lp_up(-INFINITY), hi = lp_up(S->m);
            __syncthreads();
            if (tid == 0) S->n = 0;
            while (lo < hi) {                            // the want-th largest of the groups' largest: `lo` is reached by `want` of them at least
                const u32 mid = lo + (hi - lo + 1) / 2;
                u32 k = 0;
                for (int g = 0; g < a.groups; g++) k += lp_up(gmax[g * LP_NTH + tid]) >= mid;
                k = __reduce_add_sync(0xffffffffu, k);
                if (lane == 0) S->wc[warp] = k;
                __syncthreads();
                u32 sum = 0;
                for (int i = 0; i < LP_NW; i++) sum += S->wc[i];
                __syncthreads();
                if (sum >= (u32)want) lo = mid; else hi = mid - 1;
            }
            thr = lp_down(lo);
            gather(thr, false);                          // (of fewer than `want` groups: they fit)
            __syncthreads();
            n = S->n;
            // .. and equal ones from the lowest id on
            for (int v0 = -1; n < (u32)want && v0 <= nvec; v0 += LP_NTH) {
                u32 w[4], k = 0, before = 0;
                const int at_v = v0 + tid;
                w[0] = w[1] = w[2] = w[3] = NONE;
                if (at_v == -1 || at_v == nvec) edge(at_v, w); else if (at_v < nvec) load(at_v, w);
#pragma unroll
                for (int i = 0; i < N; i++) {
                    const int id = id0 + (v0 + tid) * N + i;
                    k += id >= e0 && id < e1 && lp_clean(lp_at<TYPE>(w, i)) == thr;
                }
                u32 upto = k;
#pragma unroll
                for (int o = 1; o < 32; o *= 2) { const u32 y = __shfl_up_sync(0xffffffffu, upto, o); if (lane >= o) upto += y; }
                if (lane == 31) S->wc[warp] = upto;
                __syncthreads();
                u32 all = 0;
                for (int i = 0; i < LP_NW; i++) { if (i < warp) before += S->wc[i]; all += S->wc[i]; }
                u32 at = n + before + upto - k;
#pragma unroll
                for (int i = 0; i < N; i++) {
                    const int id = id0 + (v0 + tid) * N + i;
                    if (id >= e0 && id < e1 && lp_clean(lp_at<TYPE>(w, i)) == thr) { if (at < (u32)want) S->list[at] = lp_key(thr, id); at++; }
                }
                __syncthreads();
                n = min(n + all, (u32)want);
            }
            __syncthreads();
        }
        // each one's place among them; the first go to block 0
        for (u32 i = tid; i < n; i += LP_NTH) {
            const u64 key = S->list[i];
            u32 at = 0;
#pragma unroll 4
            for (u32 j = 0; j < n; j++) at += S->list[j] < key;
            if (at < (u32)want) { if (a.C > 1) lp_st64(&S->best[rank * LP_TOP + at], 0, key); else S->best[at] = key; }
        }
    }
    if (top)                                             // (a part with fewer elements than are asked for)
        for (int i = want + tid; i < top; i += LP_NTH) { if (a.C > 1) lp_st64(&S->best[rank * LP_TOP + i], 0, ~0ull); else S->best[i] = ~0ull; }
    lp_sync(a.C);
    if (rank == 0) {
        LpSum t = {S->part[0].x, S->part[0].y, S->part[0].z};
        u32 n = __float_as_uint(S->part[0].w);
        for (int r = 1; r < a.C; r++) {
            const float4 o = S->part[r];
            t = lp_join(t, {o.x, o.y, o.z}, c);
            n += __float_as_uint(o.w);
        }
        const bool one = alone || !(fabsf(t.m) < INFINITY);
        const float lz = log1pf(t.s);
        auto score = [&](float v) { return v == -INFINITY ? v : (v - t.m) * inv_t - lz; };      // (what is masked stays so at an infinite temperature)
        if (tid == 0) {
            if (a.logprob) a.logprob[row] = token < 0 ? -INFINITY : one ? (n == 0 ? 0.f : -INFINITY) : score(tv);
            if (a.rank) a.rank[row] = token < 0 ? -1 : (int32_t)n;
            if (a.entropy) a.entropy[row] = one ? 0.f : lz - t.x * 0.6931471805599453f / (1.f + t.s);
        }
        if (top) {
            auto give = [&](int at, u64 key) {
                const float v = lp_down(~(u32)(key >> LP_ID));
                a.top_ids[(size_t)row * top + at] = key == ~0ull ? -1 : (int32_t)(key & ((1u << LP_ID) - 1));
                a.top_logprobs[(size_t)row * top + at] = key == ~0ull ? -INFINITY : one ? (at == 0 ? 0.f : -INFINITY) : score(v);
            };
            if (a.C == 1) { if (tid < top) give(tid, S->best[tid]); }
            else {
                // a list's last key has `top` before it or at its place: what is behind any list's last is not among the best, which leaves about as many as
                // are asked for; each one's place among them is counted
                u64 bound = ~0ull;
                for (int r = 0; r < a.C; r++) bound = min(bound, S->best[r * LP_TOP + top - 1]);
                if (tid == 0) S->n = 0;
                __syncthreads();
                for (int i = tid; i < a.C * LP_TOP; i += LP_NTH) {
                    if (i % LP_TOP >= top) continue;
                    const u64 key = S->best[i];
                    if (key <= bound && key != ~0ull) S->list[atomicAdd(&S->n, 1u)] = key;
                }
                __syncthreads();
                const u32 k = S->n;
                for (u32 i = tid; i < k; i += LP_NTH) {
                    const u64 key = S->list[i];
                    u32 at = 0;
#pragma unroll 4
                    for (u32 j = 0; j < k; j++) at += S->list[j] < key;
                    if (at < (u32)top) give((int)at, key);
                }
                for (u32 i = k + tid; i < (u32)top; i += LP_NTH) give((int)i, ~0ull);      // (a vocabulary of fewer)
            }
        }
    }
    lp_sync(a.C);                                        // (shared memory is read by block 0 until here)
}

template <int TYPE, int LP_NTH>
int lp_launch(LpArgs a, cudaStream_t st) {
    constexpr int VEC = LpVec<TYPE>::N;
    a.groups = (a.per / VEC + LP_G * LP_NTH - 1) / (LP_G * LP_NTH) + 1;      // (a part may begin and end inside vectors)
    const size_t smem = sizeof(LpSmem<LP_NTH>) + (a.top ? (size_t)a.groups * LP_NTH * 4 : 0);
    const int rc = sz_allow_smem((const void*)sz_logprob_kernel<TYPE, LP_NTH>, 112 * 1024);
    if (rc) return rc;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)a.rows * a.C);
    cfg.blockDim = dim3(LP_NTH);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)a.C;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = a.C > 1 ? 2 : 1;
    SZ_CUDA(cudaLaunchKernelEx(&cfg, sz_logprob_kernel<TYPE, LP_NTH>, a));
    sz_trace_mark("logprob_rows", st);
    return SZ_OK;
}

}  // namespace

extern "C" int sz_logprob_rows(int logits_type, uint64_t logits, int64_t logits_stride, int rows, int vocab, uint64_t tokens, uint64_t temperature, int top, uint64_t logprob, uint64_t rank,
                               uint64_t entropy, uint64_t top_ids, uint64_t top_logprobs, uint64_t stream) {
    const char* who = "sz_logprob_rows";
    if (logits_type != SZ_TYPE_F32 && logits_type != SZ_TYPE_F16 && logits_type != SZ_TYPE_BF16) return sz_fail(SZ_E_TYPE, "%s: logits of type %d", who, logits_type);
    const int esz = logits_type == SZ_TYPE_F32 ? 4 : 2;
    if (rows < 1 || rows > (1 << 20) || vocab < 1 || vocab > LP_MAX_VOCAB || (rows > 1 && logits_stride < vocab) || logits_stride > (1ll << 40))
        return sz_fail(SZ_E_ARG, "%s: %d rows (1 .. 1048576) of %d logits (1 .. %d), %lld apart", who, rows, vocab, LP_MAX_VOCAB, (long long)logits_stride);
    if (top < 0 || top > LP_TOP || (top && (!top_ids || !top_logprobs))) return sz_fail(SZ_E_ARG, "%s: %d best (0 .. %d), with places for their ids and log probabilities", who, top, LP_TOP);
    if (!tokens && (logprob || rank)) return sz_fail(SZ_E_ARG, "%s: log probabilities and ranks of no tokens", who);
    if (!logprob && !rank && !entropy && !top) return sz_fail(SZ_E_ARG, "%s: nothing is asked for", who);
    if (!logits || (logits & (esz - 1)) || ((tokens | temperature | logprob | rank | entropy | top_ids | top_logprobs) & 3)) return sz_fail(SZ_E_ARG, "%s: null or misaligned argument", who);
    LpArgs a = {};
    a.logits = (const u8*)logits; a.stride = logits_stride * esz; a.rows = rows; a.vocab = vocab; a.top = top;
    a.tokens = (const int32_t*)tokens; a.temperature = (const float*)temperature;
    a.logprob = (float*)logprob; a.entropy = (float*)entropy; a.rank = (int32_t*)rank; a.top_ids = (int32_t*)top_ids; a.top_logprobs = (float*)top_logprobs;
    // Up to one row a multiprocessor: blocks of 512 threads, as many a row (up to 8) as all have a multiprocessor each; more rows: a block a row, of 256 threads, four blocks a
    // multiprocessor, where a row is up to 352 KB, else of 512 (longer rows leave too few threads with loads under way, and the groups' largest of four such blocks have no place).
    // Device us of rows of 151,936 with 512 threads and 1, 2, 4, 8 blocks a row, with 256 threads and one: 1 row of f32 16.2, 12.4, 9.5, 8.3, 25; 16 rows 17.5, 13.9,
    // 11.6, 12.6, 26; 37 rows 17.6, 14.1, 14.9, 21.9, 26; 64 rows 17.8, 14.3, 15.3, 26, 26; 128 rows 17.4, 19, 26.5, 44, 27; 250 of bf16 25.3, 34, 50, 91, 24.8; 1,021
    // 75, 101, 166, 315, 69.  One block a row, 512 / 256 threads, called one by one, top 20: 250 rows of f32, 32,000 14.2 / 13.3, 64,000 20.9 / 20.7, 96,000 28.6 / 36.2, 151,936
    // 40.5 / 58.6; 1,021 rows 44.0 / 38.6, 65.3 / 64.9, 87.1 / 92.2, 131 / 170; 250 of bf16, 128,000 29.0 / 28.8, 180,000 36.9 / 37.9, 220,000 45.4 / 51.4, 262,144 50.2 / 71.9; 1,021
    // 91 / 85, 116 / 110, 141 / 131, 158 / 177.
    const int most = vocab > 16384 ? 8 : vocab > 4096 ? 4 : vocab > 1024 ? 2 : 1;
    const bool few = rows <= LP_SM, wide = few || (long long)vocab * esz > (352 << 10);
    a.C = 1;
    while (few && 2 * a.C <= most && (long long)rows * 2 * a.C <= LP_SM) a.C *= 2;
    a.per = ((vocab + a.C - 1) / a.C + 7) & ~7;
    cudaStream_t st = (cudaStream_t)stream;
#define SZ_LP(N_) (logits_type == SZ_TYPE_F32 ? lp_launch<SZ_TYPE_F32, N_>(a, st) : logits_type == SZ_TYPE_F16 ? lp_launch<SZ_TYPE_F16, N_>(a, st) : lp_launch<SZ_TYPE_BF16, N_>(a, st))
    return wide ? SZ_LP(512) : SZ_LP(256);
#undef SZ_LP
}
