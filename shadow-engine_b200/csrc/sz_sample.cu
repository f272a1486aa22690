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
// Sums are integers, weights times 2^45 (2^18 of them stay below 2^63): exact whatever the order of the atomics, so the token depends on
// nothing but the inputs.  f32 would not do: between two of 150,000 candidates lie 10^-5 of the sum or less, and an error of 10^-8 at every
// border moves a draw in a thousand.  A weight is e^(-b width), from a table, times e^d with d = x + b width exact in f32 and below the bin's
// width in size: five terms of the exponential series in f64 leave 10^-15.
//
// A row is a cluster of blocks, each with its part of the row in shared memory: logits are read from memory once.  What bounds it: with few rows
// the chain of steps (load, maximum, sums, scan, gather, rank; a cluster barrier between), with many the sums' pass over all candidates.
#include "sz_common.cuh"

#include <math.h>

namespace {

constexpr int SA_BINS = 1024, SA_LIST = 1024, SA_NTH = 512, SA_MAX_VOCAB = 1 << 18, SA_ID = 18;
constexpr float SA_CUT = 18.0f, SA_W = SA_CUT / SA_BINS;       // (a bin's width, 9 / 512: exact, as are its multiples)
static_assert(SA_BINS == 2 * SA_NTH, "a thread scans two bins");

struct SaArgs {
    const u8* logits;
    long long stride;                // bytes
    int rows, vocab, per, C;         // per: elements of a block's part; C: blocks a row
    const float *temperature, *top_p, *min_p;
    const int32_t* top_k;
    const double* uniform;
    int32_t* token;
    float* prob;
};

enum { SA_DONE = 0, SA_GATHER = 1, SA_FINER = 2, SA_AGAIN = 3 };
struct SaCtrl {                      // block 0 of the cluster tells the others what to do
    int cmd, bin0, bin1;             // members of bins bin0 .. bin1
    int shift;                       // .. whose (key, id) >> shift is `prefix` (shift 63: all)
    u64 prefix;
    int n;                           // the list's length
    // found by a search
    int at;
    u32 rank0;
    u64 mass0;
};
struct SaSmem {
    double table[SA_BINS];           // e^(-b width) 2^45
    u64 mass[SA_BINS];
    u64 gmass[SA_BINS + 1];          // block 0: weights before bin b, of the whole row
    u64 list[SA_LIST];               // (key, id) of the gathered
    u64 sorted[SA_LIST + 1];
    u64 cum[SA_LIST + 1];            // weight of the sorted list before i
    u32 cnt[SA_BINS];
    u32 gcnt[SA_BINS + 1];
    float red[SA_NTH / 32];
    u32 redi[SA_NTH / 32];
    u64 redm[SA_NTH / 32];
    float top;                       // this block's largest
    u32 top_id, above;               // .. its lowest id; members with a weight of min_p and more
    SaCtrl c;
};

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

// larger logits first: a key that ascends as the logit descends, the id below it
__device__ __forceinline__ u64 sa_key(float v, u32 id) {
    const u32 b = __float_as_uint(v), up = b & 0x80000000u ? ~b : b | 0x80000000u;
    return ((u64)(~up) << SA_ID) | id;
}
__device__ __forceinline__ float sa_value(u64 key) {
    const u32 up = ~(u32)(key >> SA_ID);
    return __uint_as_float(up & 0x80000000u ? up & 0x7fffffffu : ~up);
}
struct SaRow { float max, inv_t, cut; };
__device__ __forceinline__ int sa_bin(float x, float& d) {           // d = x + bin * width, in (-width, 0] but for the last bin
    x = fmaxf(x, -1.5f * SA_CUT);                                    // (a difference that overflowed)
    int b = min((int)(-x * (SA_BINS / SA_CUT)), SA_BINS - 1);
    d = fmaf((float)b, SA_W, x);
    if (d > 0.f) { b--; d = fmaf((float)b, SA_W, x); }              // (the product above was rounded up)
    return b;
}
__device__ __forceinline__ u64 sa_weight(const double* table, int b, float d) {
    const double y = (double)d;
    const double e = fma(fma(fma(fma(fma(y, 1.0 / 120, 1.0 / 24), y, 1.0 / 6), y, 0.5), y, 1.0), y, 1.0);
    return (u64)(__double_as_longlong(fma(table[b], e, 4503599627370496.0)) & 0xfffffffffffffll);      // + 2^52: the integer nearest, in the low bits
}
__device__ __forceinline__ u64 sa_weight_of(const SaSmem* S, const SaRow& R, float v) {
    float d;
    const int b = sa_bin((v - R.max) * R.inv_t, d);
    return sa_weight(S->table, b, d);
}

template <int TYPE>
__device__ __forceinline__ float sa_one(const u8* p, long long i) {
    float v;
    if (TYPE == SZ_TYPE_F32) v = __ldg((const float*)p + i);
    else if (TYPE == SZ_TYPE_F16) v = sz_f16_to_f32(__ldg((const u16*)p + i));
    else v = sz_bf16_to_f32(__ldg((const u16*)p + i));
    return v != v ? -INFINITY : v;
}
// 16 bytes as their 4 or 8 values
template <int TYPE>
__device__ __forceinline__ void sa_spread(uint4 w, float* v) {
    const u32 x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if (TYPE == SZ_TYPE_F32) v[i] = __uint_as_float(x[i]);
        else if (TYPE == SZ_TYPE_F16) { const float2 f = __half22float2(*(const __half2*)&x[i]); v[2 * i] = f.x; v[2 * i + 1] = f.y; }
        else { v[2 * i] = __uint_as_float(x[i] << 16); v[2 * i + 1] = __uint_as_float(x[i] & 0xffff0000u); }
    }
#pragma unroll
    for (int i = 0; i < (TYPE == SZ_TYPE_F32 ? 4 : 8); i++) v[i] = v[i] != v[i] ? -INFINITY : v[i];
}

__device__ __forceinline__ void sa_sync(int C) { if (C > 1) sz_cluster_sync(); else __syncthreads(); }

template <int TYPE>
__global__ void __launch_bounds__(SA_NTH) sz_sample_kernel(const __grid_constant__ SaArgs a) {
    extern __shared__ __align__(16) u8 smem[];
    SaSmem* const S = (SaSmem*)smem;
    float* const val = (float*)(smem + sizeof(SaSmem));
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int row = blockIdx.x / a.C, rank = blockIdx.x % a.C;
    const int i0 = rank * a.per, n = max(0, min(a.per, a.vocab - i0));
    sz_pdl_wait();
    sz_pdl_trigger();
    // ---- the part of the row, its largest
    float big = -INFINITY;
    {
        const u8* p = a.logits + (long long)row * a.stride + (long long)i0 * (TYPE == SZ_TYPE_F32 ? 4 : 2);
        constexpr int E = TYPE == SZ_TYPE_F32 ? 4 : 8;
        const int whole = ((u64)p & 15) == 0 ? n / E : 0;
#pragma unroll 4
        for (int i = tid; i < whole; i += SA_NTH) {
            float v[E];
            sa_spread<TYPE>(__ldg((const uint4*)p + i), v);
#pragma unroll
            for (int k = 0; k < E; k += 4) *(float4*)(val + i * E + k) = make_float4(v[k], v[k + 1], v[k + 2], v[k + 3]);
#pragma unroll
            for (int k = 0; k < E; k++) big = fmaxf(big, v[k]);
        }
#pragma unroll 4
        for (int i = whole * E + tid; i < n; i += SA_NTH) { const float v = sa_one<TYPE>(p, i); val[i] = v; big = fmaxf(big, v); }
    }
    const float T = a.temperature ? __ldg(a.temperature + row) : 1.f, inv_t = 1.0f / T;
    for (int b = tid; b < SA_BINS; b += SA_NTH) { S->table[b] = exp(-(double)SA_W * b) * 35184372088832.0; S->cnt[b] = 0; S->mass[b] = 0; }
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, s));
    if (lane == 0) S->red[warp] = big;
    __syncthreads();
    if (tid == 0) {
        for (int w = 0; w < SA_NTH / 32; w++) big = fmaxf(big, S->red[w]);
        S->top = big;
        S->top_id = 0xffffffffu;
        S->above = 0;
        S->c.n = 0;
    }
    sa_sync(a.C);
    SaRow R;
    R.max = -INFINITY;
    for (int c = 0; c < a.C; c++) R.max = fmaxf(R.max, __uint_as_float(sa_ld32(&S->top, c)));
    R.inv_t = inv_t;
    R.cut = R.max - SA_CUT * T;
    if (!(T > 0.f) || isinf(inv_t) || isinf(R.max)) {               // the best token (no finite largest: the lowest id that has it)
        u32 id = 0xffffffffu;
        for (int i = tid; i < n; i += SA_NTH)
            if (val[i] == R.max) { id = min(id, (u32)(i0 + i)); break; }
        id = __reduce_min_sync(0xffffffffu, id);
        if (lane == 0) atomicMin(&S->top_id, id);
        sa_sync(a.C);
        if (rank == 0 && tid == 0) {
            for (int c = 0; c < a.C; c++) id = min(id, sa_ld32(&S->top_id, c));
            a.token[row] = (int32_t)id;
            if (a.prob) a.prob[row] = 1.f;
        }
        sa_sync(a.C);                                                // (the others' shared memory is read until here)
        return;
    }
    const float min_p = a.min_p ? __ldg(a.min_p + row) : 0.f;
    const double floor_m = (double)min_p * 35184372088832.0;
    // ---- counts and weights of the bins; returns how many of this thread's weigh min_p and more
    auto sum_bins = [&]() {
        u32 above = 0;
#pragma unroll 2
        for (int i = tid; i < n; i += SA_NTH) {
            const float v = val[i];
            if (v >= R.cut && v > -INFINITY) {
                float d;
                const int b = sa_bin((v - R.max) * R.inv_t, d);
                const u64 w = sa_weight(S->table, b, d);
                atomicAdd(&S->cnt[b], 1u);
                atomicAdd((unsigned long long*)&S->mass[b], (unsigned long long)w);
                above += (double)w >= floor_m;
            }
        }
        return above;
    };
    {
        const u32 above = __reduce_add_sync(0xffffffffu, sum_bins());
        if (lane == 0) atomicAdd(&S->above, above);
    }
    // every block adds up its share of the bins over the row's blocks, in block 0 (which scans them)
    auto add_bins = [&]() {
        sa_sync(a.C);
        const int share = SA_BINS / a.C;
        for (int b = rank * share + tid; b < (rank + 1) * share; b += SA_NTH) {
            u32 c = 0;
            u64 m = 0;
            for (int k = 0; k < a.C; k++) { c += sa_ld32(&S->cnt[b], k); m += sa_ld64(&S->mass[b], k); }
            sa_st32(&S->gcnt[b], 0, c);
            sa_st64(&S->gmass[b], 0, m);
        }
        sa_sync(a.C);
    };
    add_bins();

    // members of bins bin0 .. bin1 with (key >> shift) == prefix
    auto member = [&](const SaCtrl& c, float v, int i, u64& key) {
        if (!(v >= R.cut && v > -INFINITY)) return false;
        float d;
        const int b = sa_bin((v - R.max) * R.inv_t, d);
        if (b < c.bin0 || b > c.bin1) return false;
        key = sa_key(v, (u32)(i0 + i));
        return c.shift >= 63 || (key >> c.shift) == c.prefix;
    };
    auto gather = [&](const SaCtrl& c) {
        for (int i = tid; i < n; i += SA_NTH) {
            u64 key;
            if (member(c, val[i], i, key)) {
                const u32 at = sa_add32(&S->c.n, 0, 1u);
                if (at < (u32)SA_LIST) sa_st64(&S->list[at], 0, key);
            }
        }
    };
    // the same members into SA_BINS finer bins by the next ten bits of their keys
    auto finer = [&](const SaCtrl& c) {
        for (int b = tid; b < SA_BINS; b += SA_NTH) { S->cnt[b] = 0; S->mass[b] = 0; }
        __syncthreads();
        const int sh = (c.shift >= 63 ? SA_ID + 32 : c.shift) - 10;
        for (int i = tid; i < n; i += SA_NTH) {
            u64 key;
            const float v = val[i];
            if (member(c, v, i, key)) {
                const int b = (int)(key >> sh) & (SA_BINS - 1);          // (ten bits of keys are left at least: fewer would fit the list)
                atomicAdd(&S->cnt[b], 1u);
                atomicAdd((unsigned long long*)&S->mass[b], (unsigned long long)sa_weight_of(S, R, v));
            }
        }
        add_bins();
    };
    auto again = [&]() {
        for (int b = tid; b < SA_BINS; b += SA_NTH) { S->cnt[b] = 0; S->mass[b] = 0; }
        __syncthreads();
        sum_bins();
        add_bins();
    };
    if (rank != 0) {                                                 // ---- the other blocks do as they are told
        for (;;) {
            sz_cluster_sync();
            SaCtrl c;
            c.cmd = (int)sa_ld32(&S->c.cmd, 0);
            c.bin0 = (int)sa_ld32(&S->c.bin0, 0);
            c.bin1 = (int)sa_ld32(&S->c.bin1, 0);
            c.shift = (int)sa_ld32(&S->c.shift, 0);
            c.prefix = sa_ld64(&S->c.prefix, 0);
            if (c.cmd == SA_GATHER) { gather(c); sz_cluster_sync(); }
            else if (c.cmd == SA_FINER) finer(c);
            else if (c.cmd == SA_AGAIN) again();
            else break;
        }
        sz_cluster_sync();
        return;
    }
    // ---- block 0: exclusive sums over the bins, in place
    auto scan_bins = [&]() {
        const u32 c0 = S->gcnt[2 * tid], c1 = S->gcnt[2 * tid + 1];
        const u64 m0 = S->gmass[2 * tid], m1 = S->gmass[2 * tid + 1];
        u32 c = c0 + c1;
        u64 m = m0 + m1;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const u32 x = __shfl_up_sync(0xffffffffu, c, o);
            const u64 y = __shfl_up_sync(0xffffffffu, m, o);
            if (lane >= o) { c += x; m += y; }
        }
        if (lane == 31) { S->redi[warp] = c; S->redm[warp] = m; }
        __syncthreads();
        u32 cb = 0;
        u64 mb = 0;
        for (int w = 0; w < warp; w++) { cb += S->redi[w]; mb += S->redm[w]; }
        S->gcnt[2 * tid] = cb + c - c0 - c1; S->gcnt[2 * tid + 1] = cb + c - c1;
        S->gmass[2 * tid] = mb + m - m0 - m1; S->gmass[2 * tid + 1] = mb + m - m1;
        if (tid == SA_NTH - 1) { S->gcnt[SA_BINS] = cb + c; S->gmass[SA_BINS] = mb + m; }
        __syncthreads();
    };
    scan_bins();
    const u32 N = S->gcnt[SA_BINS];
    const u64 total = S->gmass[SA_BINS];
    u32 n_above = 0;
    for (int c = 0; c < a.C; c++) n_above += sa_ld32(&S->above, c);
    // what the list holds: `len` elements from rank `rank0` on, their running sums from mass0 on
    u32 len = 0, rank0 = 0;
    u64 mass0 = 0;
    bool bins_valid = true;
    auto tell = [&](int cmd, int bin0, int bin1, int shift, u64 prefix) {
        if (tid == 0) { S->c.cmd = cmd; S->c.bin0 = bin0; S->c.bin1 = bin1; S->c.shift = shift; S->c.prefix = prefix; S->c.n = 0; }
        sa_sync(a.C);
        const SaCtrl c = S->c;
        if (cmd == SA_GATHER) { gather(c); sa_sync(a.C); }
        else { if (cmd == SA_FINER) finer(c); else again(); scan_bins(); }
    };
    auto rank_list = [&](u32 count) {                                // the gathered keys in order, their running sums
        u64 key[SA_LIST / SA_NTH];
        int at[SA_LIST / SA_NTH];
#pragma unroll
        for (int k = 0; k < SA_LIST / SA_NTH; k++) { key[k] = (u32)(tid + k * SA_NTH) < count ? S->list[tid + k * SA_NTH] : ~0ull; at[k] = 0; }
        for (u32 j = 0; j < count; j++) {
            const u64 x = S->list[j];
#pragma unroll
            for (int k = 0; k < SA_LIST / SA_NTH; k++) at[k] += x < key[k];
        }
#pragma unroll
        for (int k = 0; k < SA_LIST / SA_NTH; k++) if ((u32)(tid + k * SA_NTH) < count) S->sorted[at[k]] = key[k];
        __syncthreads();
        const u64 w0 = (u32)(2 * tid) < count ? sa_weight_of(S, R, sa_value(S->sorted[2 * tid])) : 0, w1 = (u32)(2 * tid + 1) < count ? sa_weight_of(S, R, sa_value(S->sorted[2 * tid + 1])) : 0;
        u64 m = w0 + w1;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) { const u64 y = __shfl_up_sync(0xffffffffu, m, o); if (lane >= o) m += y; }
        if (lane == 31) S->redm[warp] = m;
        __syncthreads();
        u64 mb = 0;
        for (int w = 0; w < warp; w++) mb += S->redm[w];
        S->cum[2 * tid] = mb + m - w0 - w1; S->cum[2 * tid + 1] = mb + m - w1;
        if (tid == SA_NTH - 1) S->cum[SA_LIST] = mb + m;
        __syncthreads();
    };
    // The element of rank k (by_rank), or the first whose running sum exceeds t: its place in the list, which is made to hold it.
    auto find = [&](bool by_rank, u32 k, u64 t) -> u32 {
        for (;;) {
            const bool here = len && (by_rank ? k >= rank0 && k < rank0 + len : t >= mass0 && t < mass0 + S->cum[len]);
            if (here) {
                __syncthreads();
                if (by_rank) return k - rank0;
                for (u32 i = tid; i < len; i += SA_NTH)
                    if (mass0 + S->cum[i] <= t && t < mass0 + S->cum[i + 1]) S->c.at = (int)i;
                __syncthreads();
                return (u32)S->c.at;
            }
            if (!bins_valid) {                                       // (an overfull bin was cut finer: the row's bins again)
                tell(SA_AGAIN, 0, 0, 0, 0);
                bins_valid = true;
            }
            __syncthreads();
            for (int b = tid; b < SA_BINS; b += SA_NTH)
                if (by_rank ? S->gcnt[b] <= k && k < S->gcnt[b + 1] : S->gmass[b] <= t && t < S->gmass[b + 1]) { S->c.at = b; S->c.rank0 = S->gcnt[b]; S->c.mass0 = S->gmass[b]; }
            __syncthreads();
            int b = S->c.at, shift = 63;
            u64 prefix = 0;
            rank0 = S->c.rank0; mass0 = S->c.mass0;
            u32 count = S->gcnt[b + 1] - rank0;
            const int bin = b;
            int first = bin;
            if (S->gcnt[b + 1] <= (u32)SA_LIST) { first = 0; rank0 = 0; mass0 = 0; count = S->gcnt[b + 1]; }      // all from the top on
            while (count > (u32)SA_LIST) {
                bins_valid = false;
                tell(SA_FINER, bin, bin, shift, prefix);
                for (int x = tid; x < SA_BINS; x += SA_NTH)
                    if (by_rank ? rank0 + S->gcnt[x] <= k && k < rank0 + S->gcnt[x + 1] : mass0 + S->gmass[x] <= t && t < mass0 + S->gmass[x + 1]) {
                        S->c.at = x; S->c.rank0 = rank0 + S->gcnt[x]; S->c.mass0 = mass0 + S->gmass[x];
                    }
                __syncthreads();
                b = S->c.at;
                count = S->gcnt[b + 1] - S->gcnt[b];
                rank0 = S->c.rank0; mass0 = S->c.mass0;
                prefix = (shift >= 63 ? 0 : prefix << 10) | (u64)b;
                shift = (shift >= 63 ? SA_ID + 32 : shift) - 10;
                __syncthreads();
            }
            tell(SA_GATHER, first, bin, shift, prefix);
            len = count;
            rank_list(count);
        }
    };
    const u32 K = min((u32)max(a.top_k ? __ldg(a.top_k + row) : 0x7fffffff, 1), N);
    const double top_p = a.top_p ? (double)__ldg(a.top_p + row) : 1.0, u01 = __ldg(a.uniform + row);
    u64 Z = total;
    if (K < N) { const u32 i = find(true, K - 1, 0); Z = mass0 + S->cum[i + 1]; }
    u32 kept = min(K, max(n_above, 1u));
    u64 M = Z;
    bool known = kept == K;
    if (top_p < 1.0) {
        const double need = ceil(top_p * (double)Z);                 // the first whose running sum is `need` and more (at least the first of all)
        const u64 t = need >= 1.0 ? (need > (double)(Z - 1) ? Z - 1 : (u64)need - 1) : 0;
        const u32 i = find(false, 0, t);
        if (rank0 + i + 1 <= kept) { kept = rank0 + i + 1; M = mass0 + S->cum[i + 1]; known = true; }
    }
    if (!known) { const u32 i = find(true, kept - 1, 0); M = mass0 + S->cum[i + 1]; }
    const double goal = floor(u01 * (double)M);
    const u64 t = goal > 0.0 ? (goal >= (double)(M - 1) ? M - 1 : (u64)goal) : 0;
    const u32 i = find(false, 0, t);
    if (tid == 0) {
        a.token[row] = (int32_t)(S->sorted[i] & ((1u << SA_ID) - 1));
        if (a.prob) a.prob[row] = (float)((double)(S->cum[i + 1] - S->cum[i]) / (double)M);
        S->c.cmd = SA_DONE;
    }
    if (a.C > 1) { sz_cluster_sync(); sz_cluster_sync(); }
}

template <int TYPE>
int sa_launch(const SaArgs& a, cudaStream_t st) {
    const size_t smem = sizeof(SaSmem) + (size_t)a.per * 4;
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
    a.C = vocab > 16384 ? 8 : vocab > 4096 ? 4 : vocab > 1024 ? 2 : 1;
    a.per = ((vocab + a.C - 1) / a.C + 7) & ~7;
    cudaStream_t st = (cudaStream_t)stream;
    return logits_type == SZ_TYPE_F32 ? sa_launch<SZ_TYPE_F32>(a, st) : logits_type == SZ_TYPE_F16 ? sa_launch<SZ_TYPE_F16>(a, st) : sa_launch<SZ_TYPE_BF16>(a, st);
}
