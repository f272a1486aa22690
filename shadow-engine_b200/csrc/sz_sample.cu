// Draws over whole rows of logits (sz_sample_rows): Sampler::sample (crates/shadowzero-serve/src/sampler.rs:112-210) for many rows at once.
//
// In order of logit (equal ones by id) the candidates have weights w_i = e^(x_i), x_i = (v_i - max) / T in [-18, 0].  Every rule of the sampler
// is a prefix of that order - the first top_k; those with w >= min_p; up to the one where the running sum reaches top_p Z - and so is the draw:
// the first whose running sum exceeds u M.  No rule needs the order itself, only "which element has rank k" and "in which element does the running
// sum pass t".  So nothing is sorted but a few hundred candidates: x is cut into SA_BINS bins of width 18 / SA_BINS, one pass sums the bins'
// counts and weights, a scan over the bins says which one holds the element asked for, and that bin's members (or, where they are few, all from the
// top down to it) are gathered and ranked.  A bin with more members than the list holds (thousands of equal logits) is cut again by
// (logit, id) as an integer until they fit.
//
// Sums are integers: exact whatever the order of the atomics, so the token depends on nothing but the inputs.  f32 would not do: between two of
// 150,000 candidates lie 10^-5 of the sum or less, and an error of 10^-8 at every border moves a draw in a thousand.  A candidate in bin b weighs
// e^(-b width) (1 + r), r = e^d - 1, d = x + b width: x and b width are f32 numbers close to each other, so d is exact; r is d itself
// plus d^2 / 2 + .. <= 5 10^-5, which f32 holds to 10^-11 (a unit's half is 10^-10 of a weight, and those of a bin's members cancel).  A bin's sum of r in units of 2^-32 and its count then give its weight in f64, in units of
// 2^-45 (2^18 candidates stay below 2^63); the listed candidates' weights are f64 exponentials.
//
// A row is a cluster of 1 to 8 blocks, each with its part of the row, in shared memory where two blocks fit so.  What bounds it: with few rows
// the chain of steps (load, maximum, sums, scan, gather, order; a cluster barrier between), with many the sums' instructions - 29 and two
// atomics in shared memory an element - and the passes of the rows that ask for several elements.  Rows of 151,936, chat settings: 1 row 13.9 us;
// 64 rows of mixed settings, f32, 51 us (39 MB: 6 us of them); 250 rows of bf16 drawn from whole, 98 us (76 MB: 12 us of them).
#include "sz_common.cuh"

#include <cuda_bf16.h>

#include <math.h>

namespace {

constexpr int SA_BINS = 1024, SA_LIST = 1024, SA_NTH = 512, SA_MAX_VOCAB = 1 << 18, SA_ID = 18, SA_FEW = 512;
constexpr int SA_ROUNDS = 64;
constexpr int SA_RANK = 256;                                   // keys that are put in order by counting (at most SA_NTH)
constexpr int SA_PLACES = 2 * 148;                             // blocks that run at once
constexpr double SA_FIXED = 40000;                             // a block's time beside its part of the row, in elements of it
constexpr size_t SA_KEEP = 113 * 1024;                         // shared memory of a block, two a multiprocessor
constexpr float SA_CUT = 18.0f, SA_W = 37.0f / 2048;           // a bin's width: its multiples are exact, and SA_CUT is 997 of them
constexpr double SA_ONE = 35184372088832.0;                    // 2^45: the weight 1
static_assert(SA_BINS == 2 * SA_NTH, "a thread scans two bins");

struct SaArgs {
    const u8* logits;
    long long stride;                // bytes
    int rows, vocab, per, C;         // per: elements of a block's part; C: blocks a row
    int keep;                        // the part stays in shared memory (0: it is read again, from L2)
    const float *temperature, *top_p, *min_p;
    const int32_t* top_k;
    const double* uniform;
    int32_t* token;
    float* prob;
};

// What the blocks of a row do next; block 0 decides.
enum { SA_DONE = 0, SA_GATHER = 1, SA_SUM = 2, SA_LARGEST = 3 };
struct SaCtrl {
    int cmd, bin0, bin1;             // SA_GATHER: the members of bins bin0 .. bin1 into the list.  SA_SUM: their bins' sums
    int shift;                       // .. only those whose key >> shift is `prefix` (63: all)
    int cut;                         // SA_SUM, >= 0: in bins by the ten bits of their keys from bit `cut` on
    int count;                       // SA_SUM: and how many weigh min_p and more
    u64 prefix;
};
struct SaSmem {
    struct { u32 lo[SA_BINS + 32], hi[SA_BINS + 32]; } h;      // a bin's sums of this block (sa_term); behind them those of no candidates, a lane each
    u64 list[SA_LIST];               // block 0: keys of the gathered, then in order
    u64 cum[SA_LIST + 1];            // weight of the sorted list before i
    u64 gmass[SA_BINS + 1];          // block 0: weights before bin b, of the whole row
    u32 gcnt[SA_BINS + 1];
    float top[8 * SA_NTH / 32];      // the largest of every warp of every block
    u32 redi[SA_NTH / 32];
    u64 redm[SA_NTH / 32];
    uint4 edge[2];                   // the part's first and last 16 bytes, where they are not all its own
    u32 top_id, above;               // this block's lowest id of the largest; block 0: candidates with a weight of min_p and more
    SaCtrl c;
    u32 n;                           // the list's length
    int at;                          // found by a search
};

constexpr size_t SA_SMEM = (sizeof(SaSmem) + 15) & ~(size_t)15;

__device__ __forceinline__ u32 sa_at(const void* p, int rank) {
    u32 a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(sz_smem_addr(p)), "r"(rank));
    return a;
}
__device__ __forceinline__ u32 sa_ld32(const void* p, int rank) { u32 v; asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(sa_at(p, rank)) : "memory"); return v; }
__device__ __forceinline__ u64 sa_ld64(const void* p, int rank) { u64 v; asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(sa_at(p, rank)) : "memory"); return v; }
__device__ __forceinline__ void sa_st32(void* p, int rank, u32 v) { asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(sa_at(p, rank)), "r"(v) : "memory"); }
__device__ __forceinline__ void sa_st64(void* p, int rank, u64 v) { asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(sa_at(p, rank)), "l"(v) : "memory"); }
__device__ __forceinline__ u32 sa_add32(void* p, int rank, u32 v) { u32 o; asm volatile("atom.shared::cluster.add.u32 %0, [%1], %2;" : "=r"(o) : "r"(sa_at(p, rank)), "r"(v) : "memory"); return o; }

// larger logits first: a key that ascends as the logit descends, the id below it (-0 is 0: equal logits go by id)
__device__ __forceinline__ u64 sa_key(float v, u32 id) {
    const u32 x = __float_as_uint(v), b = x == 0x80000000u ? 0u : x, up = b & 0x80000000u ? ~b : b | 0x80000000u;
    return ((u64)(~up) << SA_ID) | id;
}
__device__ __forceinline__ float sa_value(u64 key) {
    const u32 up = ~(u32)(key >> SA_ID);
    return __uint_as_float(up & 0x80000000u ? up & 0x7fffffffu : ~up);
}
struct SaRow { float max, inv_t, cut, floor_x; };                    // floor_x: the least x whose weight is min_p and more
__device__ __forceinline__ float sa_x(const SaRow& R, float v) { return (v - R.max) * R.inv_t; }
// The bin nearest to x, and d = x + bin * width (exact), at most half a width in size (x from -18.25 on).
__device__ __forceinline__ int sa_bin(float x, float& d) {
    const float t = fmaf(x, -1.0f / SA_W, 12582912.0f);          // + 1.5 * 2^23: the integer nearest, in the low bits
    d = fmaf(t - 12582912.0f, SA_W, x);
    return (int)(__float_as_uint(t) - 0x4b400000u);
}
// A bin's sums: members, and e^d - 1 of each in units of 2^-32, 2^26 added so that it is positive: below 2^27, and 2^45 for the 2^18 members a
// block can have; count and the sum's upper 13 bits share a word.  (One 64-bit atomic in shared memory costs five times these two.)
__device__ __forceinline__ u32 sa_term(float d) {
    constexpr float U = 4294967296.0f;
    // (d^2 / 2 + .. is below 2^18 units: the integer nearest is in the low bits of the sum with 1.5 * 2^23; d^5 / 120 is below 2^-40)
    const float q = fmaf(d * d, fmaf(fmaf(d, U / 24, U / 6), d, U / 2), 12582912.0f);
    return (u32)__float2int_rn(d * U) + __float_as_uint(q) + ((1u << 26) - 0x4b400000u);
}
constexpr u32 SA_MEMBER = 1u << 13;
__device__ __forceinline__ u64 sa_weight(const SaRow& R, float v) { return (u64)__double2ull_rn(exp((double)sa_x(R, v)) * SA_ONE); }

// The first n keys of the list in order, by all threads.  Up to SA_RANK each one's place is counted (through `other`): 128 keys 0.7 us, 1,024 would be 17.
// More are compared and exchanged in pairs (a bitonic network; pairs up to 32 apart lie in one warp's 64 keys): 128 keys 2.5 us, 1,024 4.
__device__ void sa_sort(u64* list, u64* other, u32 n, int tid) {
    if (n <= (u32)SA_RANK) {
        if (tid < (int)n) {
            const u64 key = list[tid];
            int at = 0;
#pragma unroll 8
            for (u32 j = 0; j < n; j++) at += list[j] < key;
            other[at] = key;
        }
        __syncthreads();
        if (tid < (int)n) list[tid] = other[tid];
        __syncthreads();
        return;
    }
    u32 m = 2;
    while (m < n) m *= 2;
    for (u32 i = n + tid; i < m; i += SA_NTH) list[i] = ~0ull;
    __syncthreads();
#pragma unroll 1
    for (u32 k = 2; k <= m; k *= 2)
#pragma unroll 1
        for (u32 j = k / 2; j; j /= 2) {
            const u32 i = 2 * tid - (tid & (j - 1));
            if (i + j < m) {
                const u64 a = list[i], b = list[i + j];
                if ((a > b) == !(i & k)) { list[i] = b; list[i + j] = a; }
            }
            if (j > 32 || (j == 1 && k >= 64)) __syncthreads(); else __syncwarp();
        }
    __syncthreads();
}

// 16 bytes as their 4 or 8 values (NaN is below every one: no comparison holds)
template <int TYPE> struct SaVec { static constexpr int E = TYPE == SZ_TYPE_F32 ? 4 : 8, ESZ = 16 / E; };
template <int TYPE>
__device__ __forceinline__ void sa_spread(uint4 w, float* v) {
    const u32 x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if (TYPE == SZ_TYPE_F32) v[i] = __uint_as_float(x[i]);
        else if (TYPE == SZ_TYPE_F16) { const float2 f = __half22float2(*(const __half2*)&x[i]); v[2 * i] = f.x; v[2 * i + 1] = f.y; }
        else { v[2 * i] = __uint_as_float(x[i] << 16); v[2 * i + 1] = __uint_as_float(x[i] & 0xffff0000u); }
    }
}
// The larger of two in every place, a number before NaN; the largest of a word's or a pair's
template <int TYPE>
__device__ __forceinline__ u32 sa_max2(u32 a, u32 b) {
    if (TYPE == SZ_TYPE_F32) return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
    if (TYPE == SZ_TYPE_F16) { const __half2 m = __hmax2(*(const __half2*)&a, *(const __half2*)&b); return *(const u32*)&m; }
    const __nv_bfloat162 m = __hmax2(*(const __nv_bfloat162*)&a, *(const __nv_bfloat162*)&b);
    return *(const u32*)&m;
}
template <int TYPE> __device__ __forceinline__ u32 sa_none() { return TYPE == SZ_TYPE_F32 ? 0xff800000u : TYPE == SZ_TYPE_F16 ? 0xfc00u : 0xff80u; }      // -inf

__device__ __forceinline__ void sa_sync(int C) { if (C > 1) sz_cluster_sync(); else __syncthreads(); }

template <int TYPE>
__global__ void __launch_bounds__(SA_NTH, 2) sz_sample_kernel(const __grid_constant__ SaArgs a) {
    constexpr int E = SaVec<TYPE>::E, ESZ = SaVec<TYPE>::ESZ;
    extern __shared__ __align__(16) u8 smem[];
    SaSmem* const S = (SaSmem*)smem;
    uint4* const val = (uint4*)(smem + SA_SMEM);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int row = blockIdx.x / a.C, rank = blockIdx.x % a.C;
    const int i0 = rank * a.per, n = max(0, min(a.per, a.vocab - i0));
    // the part in units of 16 aligned bytes: w0 .. w1 - 1 are all its own; element 0 is element `skew` of unit 0
    const u8* const p0 = a.logits + (long long)row * a.stride + (long long)i0 * ESZ;
    const int skew = (int)((u64)p0 & 15) / ESZ, units = n ? (n + skew + E - 1) / E : 0, w0 = skew ? 1 : 0, w1 = max(w0, (n + skew) / E);
    const uint4* const p = (const uint4*)(p0 - skew * ESZ);
    if (a.C > 1) sz_cluster_arrive();
    sz_pdl_wait();
    sz_pdl_trigger();
    // ---- the part of the row, its largest (thread t has units t, t + 512 .. throughout)
    u32 big = TYPE == SZ_TYPE_F32 ? 0xff800000u : sa_none<TYPE>() * 65537u;        // the type's values side by side
    {
        const int first = w0 + (tid - w0 % SA_NTH + SA_NTH) % SA_NTH;
#pragma unroll 8
        for (int u = first; u < w1; u += SA_NTH) {
            const uint4 w = __ldg(p + u);
            if (a.keep) val[u] = w;
            big = sa_max2<TYPE>(sa_max2<TYPE>(big, sa_max2<TYPE>(w.x, w.y)), sa_max2<TYPE>(w.z, w.w));
        }
#pragma unroll 1
        for (int side = 0; side < 2; side++) {                       // the first and the last
            const int u = side ? w1 : 0;
            if (tid != u % SA_NTH || u >= units || (!side && !w0)) continue;
            u32 w[4] = {};
#pragma unroll
            for (int k = 0; k < E; k++) {
                const int i = u * E + k - skew;
                const u32 x = i < 0 || i >= n ? sa_none<TYPE>() : TYPE == SZ_TYPE_F32 ? __ldg((const u32*)p0 + i) : (u32)__ldg((const u16*)p0 + i);
                w[k * ESZ / 4] |= TYPE == SZ_TYPE_F32 ? x : x << (16 * (k & 1));
            }
            const uint4 q = make_uint4(w[0], w[1], w[2], w[3]);
            if (a.keep) val[u] = q;
            else S->edge[side] = q;
            big = sa_max2<TYPE>(sa_max2<TYPE>(big, sa_max2<TYPE>(w[0], w[1])), sa_max2<TYPE>(w[2], w[3]));
        }
    }
    float mine;
    {
        float v[8];
        sa_spread<TYPE>(make_uint4(big, big, big, big), v);
        mine = fmaxf(v[0], v[1]);
    }
    const float T = a.temperature ? __ldg(a.temperature + row) : 1.f, min_p = a.min_p ? __ldg(a.min_p + row) : 0.f, top_p = a.top_p ? __ldg(a.top_p + row) : 1.f;
    const int top_k = a.top_k ? max(__ldg(a.top_k + row), 1) : 0x7fffffff;
    const double u01 = __ldg(a.uniform + row);
    // .. of the whole row: every warp writes its largest to every block
    {
        float m = mine;
#pragma unroll
        for (int s = 16; s > 0; s >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, s));
        if (a.C > 1) sz_cluster_wait();                              // (the others have begun)
        if (lane < a.C) sa_st32(&S->top[rank * (SA_NTH / 32) + warp], lane, __float_as_uint(m));
    }
    if (tid == 0) { S->top_id = 0xffffffffu; S->above = 0; }
    sa_sync(a.C);
    SaRow R;
    {
        float m = -INFINITY;
        for (int i = lane; i < a.C * (SA_NTH / 32); i += 32) m = fmaxf(m, S->top[i]);
#pragma unroll
        for (int s = 16; s > 0; s >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, s));
        R.max = m;
    }
    R.inv_t = 1.0f / T;
    // The least candidate: v >= max - 18 T in f32, a difference that does not overflow, and - where the logits' own steps are wider than T - no
    // float behind it that the rounding let in
    R.cut = fmaxf(R.max - SA_CUT * T, R.max - 3.402823466e38f);
    if (!(sa_x(R, R.cut) >= -18.25f)) R.cut = nextafterf(R.cut, INFINITY);
    auto each = [&](auto f) {                                        // f(E values, the first's id) of the thread's units
        const uint4* const at = a.keep ? val : p;
        const int v0 = a.keep ? 0 : w0, v1 = a.keep ? units : w1;
        auto unit = [&](int u) { return *(u >= v0 && u < v1 ? at + u : &S->edge[u >= v1]); };
        uint4 next = tid < units ? unit(tid) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll 1
        for (int u = tid; u < units; u += SA_NTH) {
            const uint4 w = next;
            if (u + SA_NTH < units) next = unit(u + SA_NTH);
            float v[E];
            sa_spread<TYPE>(w, v);
            f(v, (u32)(i0 + u * E - skew));
        }
    };
    if (!(T > 0.f) || isinf(R.inv_t) || isinf(R.max)) {             // the best token (no finite largest: the lowest id that has it)
        u32 id = 0xffffffffu;
        each([&](const float* v, u32 i) {
#pragma unroll
            for (int k = 0; k < E; k++) if ((v[k] == R.max || R.max == -INFINITY) && i + k < (u32)a.vocab) id = min(id, i + k);
        });
        id = __reduce_min_sync(0xffffffffu, id);
        if (lane == 0) atomicMin(&S->top_id, id);
        sa_sync(a.C);
        if (rank == 0 && tid == 0) {
            for (int c = 0; c < a.C; c++) id = min(id, sa_ld32(&S->top_id, c));
            a.token[row] = (int32_t)min(id, (u32)a.vocab - 1);       // (none: somebody writes meanwhile)
            if (a.prob) a.prob[row] = 1.f;
        }
        sa_sync(a.C);                                                // (the others' shared memory is read until here)
        return;
    }
    // e^x >= min_p where x >= log min_p: the least float that is
    R.floor_x = min_p > 0.f ? __double2float_ru(log((double)min_p)) : min_p <= 0.f ? -INFINITY : INFINITY;
    // With a small top_k the bins of the threads' largest elements say as much as all elements': k of them above a line are k elements above it.
    bool few = top_k <= SA_FEW;
    SaCtrl c;
    c.cmd = few ? SA_LARGEST : SA_SUM; c.bin0 = 0; c.bin1 = SA_BINS - 1; c.shift = 63; c.cut = -1; c.count = 1; c.prefix = 0;
    // block 0: what the list holds - `len` elements in order from rank rank0 on, running sums from mass0 on, up to the weights of mass1 -, the search under way
    u32 len = 0, rank0 = 0, N = 0, n_above = 0, K = 0, kept = 0;
    u64 mass0 = 0, mass1 = 0, Z = 0, M = 0;
    bool bins_valid = true, descending = false, whole = false, known = false;
    u32 s_from = 0, s_count = 0;
    u64 s_m0 = 0, s_m1 = 0;
    int stage = 0;
#pragma unroll 1
    for (int round = 0;; round++) {                                  // (a row needs some thirty at most)
        // ---- all blocks
        if (c.cmd == SA_GATHER) {
            // those near the bins by |v - mid| <= half, a little wider than they are, then by their bins
            const float lo = fmaxf(R.max - ((float)c.bin1 + 0.75f) * SA_W * T, R.cut), hi = fminf(R.max - ((float)c.bin0 - 0.75f) * SA_W * T, R.max);
            const float mid = 0.5f * lo + 0.5f * hi, half = (0.5f * hi - 0.5f * lo) * 1.00001f + fmaxf(fabsf(lo), fabsf(hi)) * 1e-6f;
            each([&](const float* v, u32 i) {
                u32 hits = 0;
#pragma unroll
                for (int k = 0; k < E; k++) hits |= fabsf(v[k] - mid) <= half ? 1u << k : 0u;
                while (hits) {
                    const int k = __ffs(hits) - 1;
                    hits &= hits - 1;
                    float vk = v[0];
#pragma unroll
                    for (int j = 1; j < E; j++) vk = k == j ? v[j] : vk;
                    if (!(vk >= R.cut)) continue;
                    float d;
                    const int b = sa_bin(sa_x(R, vk), d);
                    const u64 key = sa_key(vk, i + k);
                    if (b >= c.bin0 && b <= c.bin1 && (c.shift >= 63 || (key >> c.shift) == c.prefix)) {
                        const u32 at = sa_add32(&S->n, 0, 1u);
                        if (at < (u32)SA_LIST) sa_st64(&S->list[at], 0, key);
                    }
                }
            });
        } else {
            for (int b = tid; b < SA_BINS; b += SA_NTH) { S->h.lo[b] = 0; S->h.hi[b] = 0; }
            __syncthreads();
            if (c.cmd == SA_LARGEST) {
                const float x = sa_x(R, mine);
                float d;
                if (mine >= R.cut) atomicAdd(&S->h.hi[sa_bin(x, d)], SA_MEMBER);
            } else {
                u32 above = 0;
                const u32 lo0 = sz_smem_addr(S->h.lo), none = lo0 + 4u * (SA_BINS + lane);
                each([&](const float* v, u32 i) {
#pragma unroll
                    for (int h = 0; h < E; h += 4) {
                        u32 at[4], r[4], old[4];
#pragma unroll
                        for (int k = 0; k < 4; k++) {
                            const float x = sa_x(R, v[h + k]);
                            float d;
                            const u32 b = lo0 + 4u * min((u32)sa_bin(x, d), (u32)SA_BINS - 1);      // (a logit that grew since its largest was taken has no bin)
                            const bool in = v[h + k] >= R.cut;
                            at[k] = in ? b : none;
                            r[k] = sa_term(d);
                            above += in && x >= R.floor_x;
                        }
                        if (c.cut >= 0) {
#pragma unroll
                            for (int k = 0; k < 4; k++) {
                                const u64 key = sa_key(v[h + k], i + h + k);
                                const bool in = at[k] == lo0 + 4u * (u32)c.bin0 && (c.shift >= 63 || (key >> c.shift) == c.prefix);
                                at[k] = in ? lo0 + 4u * ((u32)(key >> c.cut) & (SA_BINS - 1)) : none;
                            }
                        }
#pragma unroll
                        for (int k = 0; k < 4; k++) asm volatile("atom.shared.add.u32 %0, [%1], %2;" : "=r"(old[k]) : "r"(at[k]), "r"(r[k]) : "memory");
#pragma unroll
                        for (int k = 0; k < 4; k++) {
                            u32 more;
                            asm("{\n\t.reg .u32 t;\n\tadd.cc.u32 t, %1, %2;\n\taddc.u32 %0, %3, 0;\n\t}" : "=r"(more) : "r"(old[k]), "r"(r[k]), "r"(SA_MEMBER));
                            asm volatile("red.shared.add.u32 [%0], %1;" ::"r"(at[k] + (u32)sizeof(S->h.lo)), "r"(more) : "memory");
                        }
                    }
                });
                if (c.count) {
                    above = __reduce_add_sync(0xffffffffu, above);
                    if (lane == 0 && above) sa_add32(&S->above, 0, above);
                }
            }
            // every block adds up its share of the bins over the row's blocks, for block 0
            sa_sync(a.C);
            const int share = SA_BINS / a.C;
            for (int b = rank * share + tid; b < (rank + 1) * share; b += SA_NTH) {
                u64 sum = 0;
                u32 n_b = 0, h[8], l[8];
#pragma unroll
                for (int k = 0; k < 8; k++) { h[k] = k < a.C ? sa_ld32(&S->h.hi[b], k) : 0; l[k] = k < a.C ? sa_ld32(&S->h.lo[b], k) : 0; }
#pragma unroll
                for (int k = 0; k < 8; k++) { n_b += h[k] / SA_MEMBER; sum += ((u64)(h[k] % SA_MEMBER) << 32) + l[k]; }
                const double more = (double)((long long)sum - ((long long)n_b << 26)) * (1.0 / 4294967296.0);
                sa_st32(&S->gcnt[b], 0, n_b);
                sa_st64(&S->gmass[b], 0, n_b ? __double2ull_rn(exp(-(double)SA_W * (c.cut >= 0 ? c.bin0 : b)) * SA_ONE * ((double)n_b + more)) : 0ull);
            }
        }
        sa_sync(a.C);
        // ---- block 0: sums before the bins, or the list in order; then on with the row until something is missing
        if (rank == 0) {
            u32 count;
            if (c.cmd != SA_GATHER) count = SA_BINS;
            else {
                count = S->n;
                if (few && !whole) {
                    whole = count <= (u32)SA_LIST;
                    s_count = count; s_from = 0; s_m0 = 0;
                    few = whole;
                }
                if (whole || !few) count = min(count, (u32)SA_LIST);
                sa_sort(S->list, S->cum, count, tid);
            }
            // two elements a thread: sums before them
            u32 n0 = 0, n1 = 0;
            u64 w0 = 0, w1 = 0;
            if (c.cmd != SA_GATHER) { n0 = S->gcnt[2 * tid]; n1 = S->gcnt[2 * tid + 1]; w0 = S->gmass[2 * tid]; w1 = S->gmass[2 * tid + 1]; }
            else {
                n0 = (u32)(2 * tid) < count; n1 = (u32)(2 * tid + 1) < count;
                if (n0) w0 = sa_weight(R, sa_value(S->list[2 * tid]));
                if (n1) w1 = sa_weight(R, sa_value(S->list[2 * tid + 1]));
                if (whole && c.cmd == SA_GATHER) {
                    u32 above = (n0 && sa_x(R, sa_value(S->list[2 * tid])) >= R.floor_x) + (n1 && sa_x(R, sa_value(S->list[2 * tid + 1])) >= R.floor_x);
                    above = __reduce_add_sync(0xffffffffu, above);
                    if (lane == 0 && above) atomicAdd(&S->above, above);
                }
            }
            u32 n_s = n0 + n1;
            u64 m = w0 + w1;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const u32 x = __shfl_up_sync(0xffffffffu, n_s, o);
                const u64 y = __shfl_up_sync(0xffffffffu, m, o);
                if (lane >= o) { n_s += x; m += y; }
            }
            if (lane == 31) { S->redi[warp] = n_s; S->redm[warp] = m; }
            __syncthreads();
            u32 nb = lane < warp ? S->redi[lane] : 0;
            u64 mb = lane < warp ? S->redm[lane] : 0;
#pragma unroll
            for (int o = SA_NTH / 64; o > 0; o >>= 1) { nb += __shfl_xor_sync(0xffffffffu, nb, o); mb += __shfl_xor_sync(0xffffffffu, mb, o); }
            nb = __shfl_sync(0xffffffffu, nb, 0); mb = __shfl_sync(0xffffffffu, mb, 0);
            u64* const mass = c.cmd != SA_GATHER ? S->gmass : S->cum;
            mass[2 * tid] = mb + m - w0 - w1; mass[2 * tid + 1] = mb + m - w1;
            if (tid == SA_NTH - 1) mass[SA_BINS] = mb + m;
            if (c.cmd != SA_GATHER) {
                S->gcnt[2 * tid] = nb + n_s - n0 - n1; S->gcnt[2 * tid + 1] = nb + n_s - n1;
                if (tid == SA_NTH - 1) S->gcnt[SA_BINS] = nb + n_s;
                len = 0;                                             // (the sorted list lies where the bins are summed)
            }
            __syncthreads();
            if (c.cmd == SA_GATHER) { len = count; rank0 = s_from; mass0 = s_m0; mass1 = whole ? S->cum[len] : s_m1; }
            auto search = [&](auto at, int n_at) {                   // the one place of n_at for which at() is true
                for (int i = tid; i < n_at; i += SA_NTH) if (at(i)) S->at = i;
                __syncthreads();
                const int i = min(max(S->at, 0), n_at - 1);          // (logits that somebody writes meanwhile may have none)
                __syncthreads();
                return i;
            };
            SaCtrl t = {};
            t.shift = 63; t.cut = -1;
#pragma unroll 1
            for (;;) {
                bool by_rank = false;
                u32 k = 0;
                u64 goal = 0;
                if (stage == 0) {                                    // the candidates, or as many of them as may be kept
                    if (c.cmd == SA_LARGEST) {
                        int line = SA_BINS - 1;
                        if (S->gcnt[SA_BINS] >= (u32)top_k) line = search([&](int b) { return S->gcnt[b] < (u32)top_k && (u32)top_k <= S->gcnt[b + 1]; }, SA_BINS);
                        t.cmd = SA_GATHER; t.bin1 = line;
                        break;
                    }
                    if (c.cmd == SA_GATHER && !whole) { t.cmd = SA_SUM; t.bin1 = SA_BINS - 1; t.count = 1; break; }      // more equal ones than the list holds
                    N = whole ? len : S->gcnt[SA_BINS];
                    n_above = S->above;
                    K = min((u32)top_k, N);
                    Z = whole ? S->cum[K] : S->gmass[SA_BINS];
                    kept = min(K, max(n_above, 1u));
                    known = kept == K;
                    stage = !whole && K < N ? 1 : 2;
                    M = Z;
                }
                if (stage == 1) { by_rank = true; k = K - 1; }       // Z: the sum up to the last of top_k
                if (stage == 2) {                                    // the first whose running sum is top_p Z and more
                    if (!(top_p < 1.f)) stage = 3;
                    else {
                        const double need = ceil((double)top_p * (double)Z);
                        goal = need >= 1.0 ? (need > (double)(Z - 1) ? Z - 1 : (u64)need - 1) : 0;
                    }
                }
                if (stage == 3) { if (known) stage = 4; else { by_rank = true; k = kept - 1; } }      // M: the sum of what is kept
                if (stage == 4) {                                    // the draw
                    const double g = floor(u01 * (double)M);
                    goal = g > 0.0 ? (g >= (double)(M - 1) ? M - 1 : (u64)g) : 0;
                }
                if (stage == 5) { by_rank = true; k = kept - 1; }    // .. which a rounding of the bins' sums put behind the last kept
                if (len && (by_rank ? k >= rank0 && k < rank0 + len : goal >= mass0 && goal < mass1)) {
                    // (the last of the list, where a rounding of the bins' sums leaves none)
                    const u32 i = by_rank ? k - rank0 : (u32)search([&](int j) { return (j == 0 || mass0 + S->cum[j] <= goal) && (j == (int)len - 1 || goal < mass0 + S->cum[j + 1]); }, (int)len);
                    const u64 upto = mass0 + S->cum[i + 1];
                    if (stage == 1) { Z = upto; if (known) M = Z; stage = 2; }
                    else if (stage == 2) { if (rank0 + i + 1 <= kept) { kept = rank0 + i + 1; M = upto; known = true; } stage = 3; }
                    else if (stage == 3) { M = upto; stage = 4; }
                    else if (stage == 4 && rank0 + i >= kept) stage = 5;
                    else {
                        if (tid == 0) {
                            a.token[row] = (int32_t)(S->list[i] & ((1u << SA_ID) - 1));
                            if (a.prob) a.prob[row] = (float)((double)(S->cum[i + 1] - S->cum[i]) / (double)M);
                        }
                        t.cmd = SA_DONE;
                        break;
                    }
                    continue;
                }
                if (!bins_valid && !descending) {                    // (a full bin was cut finer where they lay)
                    bins_valid = true;
                    t.cmd = SA_SUM; t.bin1 = SA_BINS - 1;
                    break;
                }
                const u32 r_at = descending ? s_from : 0;
                const u64 m_at = descending ? s_m0 : 0;
                const int b = search([&](int j) {
                    if (S->gcnt[j] == S->gcnt[j + 1]) return false;
                    if (by_rank) return r_at + S->gcnt[j] <= k && k < r_at + S->gcnt[j + 1];
                    return (S->gcnt[j] == 0 || m_at + S->gmass[j] <= goal) && (S->gcnt[j + 1] == S->gcnt[SA_BINS] || goal < m_at + S->gmass[j + 1]);
                }, SA_BINS);
                s_count = S->gcnt[b + 1] - S->gcnt[b];
                s_from = r_at + S->gcnt[b];
                s_m0 = m_at + S->gmass[b];
                s_m1 = m_at + S->gmass[b + 1];
                if (descending) { t.bin0 = t.bin1 = c.bin0; t.prefix = (c.shift >= 63 ? 0 : c.prefix << 10) | (u64)b; t.shift = c.cut; }
                else {
                    t.bin0 = t.bin1 = b;
                    if (S->gcnt[b + 1] <= (u32)SA_LIST / 4) { t.bin0 = 0; s_from = 0; s_m0 = 0; s_count = S->gcnt[b + 1]; }      // all from the top on
                }
                descending = s_count > (u32)SA_LIST;
                t.cmd = descending ? SA_SUM : SA_GATHER;
                if (descending) { bins_valid = false; t.cut = (t.shift >= 63 ? SA_ID + 32 : t.shift) - 10; }      // (ten bits are left at least: fewer would fit the list)
                break;
            }
            if (round == SA_ROUNDS && t.cmd != SA_DONE) {            // logits that somebody writes meanwhile: no two passes agree
                t.cmd = SA_DONE;
                if (tid == 0) {
                    a.token[row] = 0;
                    if (a.prob) a.prob[row] = 0.f;
                }
            }
            if (tid == 0) { S->c = t; S->n = 0; }
            c = t;
        }
        sa_sync(a.C);
        if (rank != 0) {
            c.cmd = (int)sa_ld32(&S->c.cmd, 0); c.bin0 = (int)sa_ld32(&S->c.bin0, 0); c.bin1 = (int)sa_ld32(&S->c.bin1, 0);
            c.shift = (int)sa_ld32(&S->c.shift, 0); c.cut = (int)sa_ld32(&S->c.cut, 0); c.count = (int)sa_ld32(&S->c.count, 0);
            c.prefix = sa_ld64(&S->c.prefix, 0);
        }
        if (c.cmd == SA_DONE) break;
    }
    sa_sync(a.C);                                                    // (block 0's shared memory is read until here)
}

template <int TYPE>
int sa_launch(const SaArgs& a, cudaStream_t st) {
    const size_t smem = SA_SMEM + (a.keep ? (size_t)a.per * SaVec<TYPE>::ESZ + 16 : 0);
    const int rc = sz_allow_smem((const void*)sz_sample_kernel<TYPE>, 227 * 1024);
    if (rc) return rc;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)a.rows * a.C);
    cfg.blockDim = dim3(SA_NTH);
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
    SZ_CUDA(cudaLaunchKernelEx(&cfg, sz_sample_kernel<TYPE>, a));
    sz_trace_mark("sample_rows", st);
    return SZ_OK;
}

}  // namespace

extern "C" int sz_sample_rows(int logits_type, uint64_t logits, int64_t logits_stride, int rows, int vocab, uint64_t temperature, uint64_t top_k, uint64_t top_p, uint64_t min_p,
                              uint64_t uniform, uint64_t token, uint64_t prob, uint64_t stream) {
    const char* who = "sz_sample_rows";
    if (logits_type != SZ_TYPE_F32 && logits_type != SZ_TYPE_F16 && logits_type != SZ_TYPE_BF16) return sz_fail(SZ_E_TYPE, "%s: logits of type %d", who, logits_type);
    const int esz = logits_type == SZ_TYPE_F32 ? 4 : 2;
    if (rows < 1 || rows > (1 << 20) || vocab < 1 || vocab > SA_MAX_VOCAB || (rows > 1 && logits_stride < vocab))
        return sz_fail(SZ_E_ARG, "%s: %d rows (1 .. 1048576) of %d logits (1 .. %d), %lld apart", who, rows, vocab, SA_MAX_VOCAB, (long long)logits_stride);
    if (!logits || (logits & (esz - 1)) || !uniform || (uniform & 7) || !token || ((token | prob | temperature | top_k | top_p | min_p) & 3))
        return sz_fail(SZ_E_ARG, "%s: null or misaligned argument", who);
    SaArgs a = {};
    a.logits = (const u8*)logits; a.stride = logits_stride * esz; a.rows = rows; a.vocab = vocab;
    a.temperature = (const float*)temperature; a.top_k = (const int32_t*)top_k; a.top_p = (const float*)top_p; a.min_p = (const float*)min_p;
    a.uniform = (const double*)uniform; a.token = (int32_t*)token; a.prob = (float*)prob;
    // Blocks a row: the fewer, the more rows are under way at once and the less their steps wait for one another; the more, the sooner a row is
    // through.  Waves of blocks times what a block takes (rows of 151,936, us, 1 / 2 / 4 / 8 blocks: 1 row 30 / 22 / 16 / 13.4, 64 rows
    // 105 / 62 / 51 / 55, 250 rows of bf16 93 / 97 / 115 / 175).
    const int most = vocab > 16384 ? 8 : vocab > 4096 ? 4 : vocab > 1024 ? 2 : 1;
    double least = 0;
    for (int C = 1; C <= most; C *= 2) {
        const double cost = (double)(((long long)rows * C + SA_PLACES - 1) / SA_PLACES) * (SA_FIXED + (double)vocab / C);
        if (C == 1 || cost < least) { least = cost; a.C = C; }
    }
    a.per = ((vocab + a.C - 1) / a.C + 7) & ~7;
    // read again from L2 where shared memory would hold fewer blocks with their parts than without
    a.keep = SA_SMEM + (size_t)a.per * esz + 16 <= SA_KEEP;
    cudaStream_t st = (cudaStream_t)stream;
    return logits_type == SZ_TYPE_F32 ? sa_launch<SZ_TYPE_F32>(a, st) : logits_type == SZ_TYPE_F16 ? sa_launch<SZ_TYPE_F16>(a, st) : sa_launch<SZ_TYPE_BF16>(a, st);
}
