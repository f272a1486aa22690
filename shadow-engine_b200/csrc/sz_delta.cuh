// The DeltaNet layer of a served step (sz_delta_*): what its kernels share.
#pragma once
#include "sz_common.cuh"

#include <cuda_bf16.h>

// bits of the status word
constexpr u32 DL_E_SLOT = 1, DL_E_ROWS = 2, DL_E_CLASH = 4, DL_E_WAIT = 8;

struct DlBatch {
    int n_seq, rows, n_slots;
    const int32_t *row_start, *lens, *from, *to, *take;      // take may be null
    u32* err;
};

// What a call does of one sequence: rows r0 .. r0 + n of the inputs, counted ones; the state comes from slot `from` (-1: from nothing) and goes to `to`.
struct DlSeq {
    int r0, n, from, to;
    bool on;                         // (off: without rows, or left out)
};

#ifdef __CUDACC__
// f32x2 arithmetic
__device__ __forceinline__ void dl_fma2(u64& a, u64 f, u64 x) { asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(a) : "l"(f), "l"(x)); }
__device__ __forceinline__ u64 dl_mul2(u64 a, u64 b) { u64 d; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b)); return d; }
__device__ __forceinline__ u64 dl_pack2(float a, float b) { u64 d; asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(a), "f"(b)); return d; }
__device__ __forceinline__ float dl_lo(u64 a) { return __uint_as_float((u32)a); }
__device__ __forceinline__ float dl_hi(u64 a) { return __uint_as_float((u32)(a >> 32)); }

template <int TYPE> struct DlIo {
    static constexpr int ESZ = TYPE == SZ_TYPE_F32 ? 4 : 2;
};
// N neighbouring elements (N * ESZ a multiple of 4 bytes, aligned to it or to 16)
template <int TYPE, int N>
__device__ __forceinline__ void dl_unpack(const u32* w, float* f) {
    if constexpr (TYPE == SZ_TYPE_F32) {
#pragma unroll
        for (int i = 0; i < N; i++) f[i] = __uint_as_float(w[i]);
    } else {
#pragma unroll
        for (int i = 0; i < N / 2; i++) {
            if constexpr (TYPE == SZ_TYPE_F16) {
                const float2 x = __half22float2(*(const __half2*)&w[i]);
                f[2 * i] = x.x; f[2 * i + 1] = x.y;
            } else {
                f[2 * i] = __uint_as_float(w[i] << 16); f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
            }
        }
    }
}
template <int TYPE, int N>
__device__ __forceinline__ void dl_load(const u8* p, float* f) {
    constexpr int W = N * DlIo<TYPE>::ESZ / 4;
    u32 w[W];
    if constexpr (W % 4 == 0) {
#pragma unroll
        for (int i = 0; i < W / 4; i++) *(uint4*)(w + 4 * i) = *((const uint4*)p + i);
    } else if constexpr (W == 2) *(uint2*)w = *(const uint2*)p;
    else w[0] = *(const u32*)p;
    dl_unpack<TYPE, N>(w, f);
}
template <int TYPE, int N>
__device__ __forceinline__ void dl_store(u8* p, const float* f) {
    constexpr int W = N * DlIo<TYPE>::ESZ / 4;
    u32 w[W];
#pragma unroll
    for (int i = 0; i < W; i++) {
        if constexpr (TYPE == SZ_TYPE_F32) w[i] = __float_as_uint(f[i]);
        else if constexpr (TYPE == SZ_TYPE_F16) { const __half2 h = __floats2half2_rn(f[2 * i], f[2 * i + 1]); w[i] = *(const u32*)&h; }
        else { const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]); w[i] = *(const u32*)&h; }
    }
    if constexpr (W % 4 == 0) {
#pragma unroll
        for (int i = 0; i < W / 4; i++) *((uint4*)p + i) = *(const uint4*)(w + 4 * i);
    } else if constexpr (W == 2) *(uint2*)p = *(const uint2*)w;
    else *(u32*)p = w[0];
}
template <int TYPE>
__device__ __forceinline__ float dl_load1(const u8* p) {
    if constexpr (TYPE == SZ_TYPE_F32) return *(const float*)p;
    else if constexpr (TYPE == SZ_TYPE_F16) return __half2float(*(const __half*)p);
    else return __uint_as_float((u32) * (const u16*)p << 16);
}

// sigmoid: where 16 bits are kept of what it is multiplied with, by the fast exponential and quotient (2^-21 relative); for f32 e^y = 2^e (1 + rest log 2) with y log2(e) as a sum of two
// f32 numbers, e and the rest that rounding it leaves (log2(e) itself in two numbers, products by fused multiply-adds), and the fast reciprocal with a step of Newton's method, r (2 - den r): 2^-22, a third
// of the time of sz_sigmoid.  Beyond 87 it is 1, or 0 (2^-125 and less); of NaN it is NaN.
template <int TYPE> __device__ __forceinline__ float dl_sigmoid(float x) {
    if (TYPE != SZ_TYPE_F32) return __fdividef(1.f, 1.f + __expf(-x));
    constexpr float L = 1.4426950408889634f, L_LOW = 1.925963033500e-8f;      // log2(e), and what f32 leaves of it
    const float y = x < -87.f ? 87.f : x > 87.f ? -87.f : -x, e = y * L, rest = fmaf(y, L_LOW, fmaf(y, L, -e));
    float w, r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(w) : "f"(e));
    const float den = 1.f + fmaf(w, rest * 0.6931471805599453f, w);
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(den));
    r *= fmaf(-den, r, 2.f);
    return x < -87.f ? 0.f : r;
}
// The logarithm of a row's decay, a softplus(alpha + dt).  A decay above 1 (a positive `a`) counts as 1; one below e^-1000 is 0 in f32 as it is, and sums of these
// keep the others' digits (in f64).
__device__ __forceinline__ float dl_log_decay(float alpha, float a, float dt) {
    const float x = alpha + dt, g = a * (x > 20.f ? x : log1pf(expf(x)));
    return g > 0.f ? 0.f : g < -1000.f ? -1000.f : g;
}

// Sequence b as one warp sees it (all lanes with the same b).  An earlier sequence with rows that writes a slot which b reads or writes, or reads one
// that b writes, keeps b out: whatever the order of the blocks, the results are the same.  One whose own entries do not fit touches no slot and keeps nobody out.
__device__ __forceinline__ DlSeq dl_seq(const DlBatch& d, int b, int lane, bool report) {
    DlSeq s;
    // (a lane's first sequence before b is asked for together with b itself: one wait, not three)
    int p0 = 0, p1 = 0, pt = 0, pf = 0, pl = 0;
    auto ask = [&](int i) { p0 = d.row_start[i]; p1 = d.row_start[i + 1]; pt = d.to[i]; pf = d.from[i]; pl = d.lens[i]; };
    if (lane < b) ask(lane);
    const int r0 = d.row_start[b], r1 = d.row_start[b + 1], len = d.lens[b];
    const int from = d.from[b], to = d.to[b], take = d.take ? d.take[b] : 0x7fffffff;
    u32 bad = 0;
    if (r0 < 0 || r1 < r0 || r1 > d.rows) bad |= DL_E_ROWS;
    const int count = bad ? 0 : r1 - r0;
    s.r0 = r0;
    s.n = min(count, max(take, 0));
    s.from = len > count ? from : -1;
    s.to = to;
    if (count > 0 && ((u32)to >= (u32)d.n_slots || (len > count && (u32)from >= (u32)d.n_slots))) bad |= DL_E_SLOT;
    if (count > 0 && !bad) {
        bool clash = false;
        for (int i = lane; i < b; i += 32) {
            if (i >= 32) ask(i);
            const bool reads = pl > p1 - p0;
            if (p0 < 0 || p1 <= p0 || p1 > d.rows || (u32)pt >= (u32)d.n_slots || (reads && (u32)pf >= (u32)d.n_slots)) continue;      // (without rows, or left out itself)
            clash |= pt == to || pt == s.from || (reads && pf == to);
        }
        if (__any_sync(0xffffffffu, clash)) bad |= DL_E_CLASH;
    }
    s.on = count > 0 && !bad;
    if (bad && report && lane == 0) atomicOr(d.err, bad);
    return s;
}
#endif

// ---- the rule over the sequences of many rows, in chunks (sz_delta_chunk.cu)
struct DlRule {
    const u8 *q, *k, *v, *alpha, *beta, *z;                      // q null: no outputs (a replay)
    u8* out;
    long long q_stride, k_stride, v_stride, alpha_stride, beta_stride, z_stride, out_stride;      // bytes
    const float *a, *dt, *norm;
    float eps, q_scale;
    int kh, vh, grouped;
    u8* state;
    long long state_stride;
    int least;                       // sequences of at least so many rows go in chunks, the others row by row (0: none in chunks)
};
int64_t dl_chunk_bytes(int d, int kh, int vh, int io_type, int n_seq, int rows, int least);
int dl_chunk_launch(int d, int io_type, const DlBatch& b, const DlRule& r, uint64_t scratch, cudaStream_t st);
