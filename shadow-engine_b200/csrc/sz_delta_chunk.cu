// The gated delta rule over many rows of a sequence, in chunks of CK = 64 (sz_delta.cuh has the row-by-row form's neighbours).
//
// With S the state before a chunk, G_i the sum of the decays' logarithms up to its row i, and k, q the normed rows, the rows' changes d_i solve a triangular system:
//   (I + A) D = diag(beta) (V - diag(e^G) K S),   A_ij = beta_i e^(G_i - G_j) k_i.k_j for j < i
//   O = diag(e^G) Q S + P D,   P_ij = e^(G_i - G_j) q_i.k_j for j <= i
//   S' = e^G_C S + sum_j e^(G_C - G_j) k_j d_j^T
// so that a chunk is a few matrix products instead of 64 steps.  Two kernels:
//  sz_delta_prep_kernel, a block a chunk and key head: what does not need S - the products of its rows, T = (I + A)^-1 diag(beta) and P of every value head of the
//   key head - side by side, over all chunks at once;
//  sz_delta_chunk_kernel, a block of warps for 16 NG value dimensions of a sequence's value head: the chain over its chunks, on mma.sync.  Everything is
//   transposed, so that a warp's 16 value dimensions are a product's rows: S^T (f32) stays in its registers, and what one product gives is in the layout in which
//   the next one takes it.  At 128 key dimensions two warps have 64 of them each and add up K S and Q S through shared memory.
// tcgen05 would have the products' time, but every one of the chain's links would go through tensor memory and back (300 - 400 cycles a wait, three
// a chunk) and S through a conversion by four warps: no sooner.
//
// Numbers.  A row k = rho 2^e (k 2^-e) enters the products as k 2^-e with its largest element in [1, 2): a bf16 or f16 row is exact in f16, an f32 row is two f16
// numbers (22 bits); the rows' lengths and powers are factors in f32.  S, R = V - e^G K S and D enter as two f16 numbers each, in units of a power of two that
// the warp takes from the largest there is: 22 bits, and what is less than 2^-35 of that largest is lost.  Sums are f32.  T and the decays' sums: f32 and f64.  The
// last products of a bf16 output take one f16 number a factor (11 bits, where the output keeps 8).
#include "sz_delta.cuh"

namespace {

constexpr int CK = 64, DL_TILES = 20;                    // rows of a chunk; 8 x 16 tiles of a lower triangle
constexpr int DL_FRAG = DL_TILES * 32 * 8;               // bytes of a triangle in f16, in the order in which the matrix instruction takes it
constexpr float DL_P = 1024.f;                           // P's elements are at most 1 / sqrt(d): times this they keep their 22 bits
constexpr int64_t DL_SLAB = 96ll << 20;                  // scratch that a pass over chunks may take (what the first kernel leaves is in L2 for the second)

struct DlScalars { float gr[CK], gq[CK], wj[CK], gc, pad[15]; };      // e^G rho_k, e^G rho_q, e^(G_C - G_j) rho_k; e^G_C

template <int D, int TYPE> struct DlChunk {
    static constexpr int NK = TYPE == SZ_TYPE_F32 ? 2 : 1;                // f16 numbers of an element of k and q
    static constexpr bool FULL = TYPE != SZ_TYPE_BF16;                    // outputs' products with both numbers of a factor
    static constexpr int TILE = CK * D * 2, ROWS = 2 * NK * TILE;         // a key head's rows: k (high, low), q (high, low)
    static constexpr int HEAD = (FULL ? 4 : 3) * DL_FRAG + (int)sizeof(DlScalars);      // a value head's T (high, low), P (high, low), scalars
};
int64_t dl_chunk_one(int d, int kh, int vh, int io_type) {
    const int nk = io_type == SZ_TYPE_F32 ? 2 : 1;
    return (int64_t)kh * 2 * nk * CK * d * 2 + (int64_t)vh * ((io_type == SZ_TYPE_BF16 ? 3 : 4) * DL_FRAG + (int)sizeof(DlScalars));
}

// The sequences of many rows, in order: the y-th of them (y >= 0), or the one whose chunks have index idx.  Chunk c of a sequence has index
// row_start / CK + its place among them + c: no two have the same.  A warp looks for itself.
struct DlLong { int b, base; };
__device__ __forceinline__ DlLong dl_find(const DlBatch& d, int least, int y, int idx, int lane) {
    int seen = 0;
    for (int b0 = 0; b0 < d.n_seq; b0 += 32) {
        const int b = b0 + lane;
        int r0 = 0, n = 0;
        if (b < d.n_seq) { r0 = d.row_start[b]; n = d.row_start[b + 1] - r0; }
        const bool lg = n >= least && r0 >= 0 && r0 < d.rows && n <= d.rows;
        const u32 m = __ballot_sync(0xffffffffu, lg);
        const int rank = seen + __popc(m & ((1u << lane) - 1)), base = r0 / CK + rank;
        const bool hit = lg && (y >= 0 ? rank == y : idx >= base && idx < base + (n + CK - 1) / CK);
        const u32 f = __ballot_sync(0xffffffffu, hit);
        if (f) {
            const int src = __ffs(f) - 1;
            return {b0 + src, __shfl_sync(0xffffffffu, base, src)};
        }
        seen += __popc(m);
    }
    return {-1, 0};
}

__device__ __forceinline__ u32 dl_h2(float a, float b) { const __half2 h = __floats2half2_rn(a, b); return *(const u32*)&h; }
// two f16 numbers of a pair: high, and what is left
__device__ __forceinline__ void dl_split(float a, float b, u32& hi, u32& lo) {
    const __half2 h = __floats2half2_rn(a, b);
    const float2 f = __half22float2(h);
    hi = *(const u32*)&h;
    lo = dl_h2(a - f.x, b - f.y);
}
__device__ __forceinline__ void dl_mma(float* c, const u32* a, u32 b0, u32 b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void dl_ldsm(u32* r, u32 addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void dl_ldsm_t(u32* r, u32 addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
// byte of the 16-byte piece c of row r of a tile [rows][D] of f16: pieces exchanged so that ldmatrix meets no bank twice
template <int D> __device__ __forceinline__ u32 dl_at(int r, int c) { return (u32)(r * D * 2 + ((c ^ (r & 7)) << 4)); }
// the first of the tiles of 8 rows n of a lower triangle (its 16-column tiles are side by side)
__host__ __device__ constexpr int dl_tile(int n) { return (n / 2) * (n / 2 + 1) + (n & 1) * (n / 2 + 1); }
__device__ __forceinline__ float dl_pow2(int e) { return e < -126 ? 0.f : __uint_as_float((u32)(min(e, 127) + 127) << 23); }

// ---- what does not need the state -----------------------------------------------------------------------------------------------------------
constexpr int DL_AS = 68, DL_TS = 72;                    // strides of a value head's A (by columns) and T (by rows), which share their place
template <int D, int TYPE> struct DlPrep {
    static constexpr int ROWS = DlChunk<D, TYPE>::ROWS, A = CK * DL_TS * 4;
    static constexpr size_t SMEM = ROWS + 2 * A;
};

template <int D, int TYPE, bool OUT>
__global__ void __launch_bounds__(128)
sz_delta_prep_kernel(const DlBatch d, const DlRule a, int idx0, u8* __restrict__ scratch, long long one) {
    using C = DlChunk<D, TYPE>;
    constexpr int ESZ = DlIo<TYPE>::ESZ, NK = C::NK, E = D / 8;
    extern __shared__ __align__(16) u8 sm[];
    __shared__ double sG[2][CK];
    __shared__ float sRk[CK], sRq[CK], sBeta[2][CK];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, kx = blockIdx.y, g = lane >> 2, t = lane & 3;
    sz_pdl_wait();
    sz_pdl_trigger();
    const int idx = idx0 + blockIdx.x;
    const DlLong lg = dl_find(d, a.least, -1, idx, lane);
    if (lg.b < 0) return;
    const DlSeq s = dl_seq(d, lg.b, lane, false);
    const int c = idx - lg.base, n = min(CK, s.n - c * CK);
    if (!s.on || n <= 0) return;
    const size_t row0 = (size_t)s.r0 + (size_t)c * CK;
    u8* const mine = scratch + (size_t)blockIdx.x * one;
    u8* const rows = mine + (size_t)kx * C::ROWS;
    // the rows, scaled by powers of two: eight lanes a row
    const int sub = lane & 7;
#pragma unroll 1
    for (int i = 0; i < (OUT ? 8 : 4); i++) {
        const bool isq = i >= 4;
        const int r = warp * 16 + (i & 3) * 4 + (lane >> 3);
        float f[E];
#pragma unroll
        for (int e = 0; e < E; e++) f[e] = 0.f;
        if (r < n) dl_load<TYPE, E>((isq ? a.q + (row0 + r) * a.q_stride : a.k + (row0 + r) * a.k_stride) + (size_t)(kx * D + sub * E) * ESZ, f);
        float ss = 0.f, mx = 0.f;
#pragma unroll
        for (int e = 0; e < E; e++) { ss = fmaf(f[e], f[e], ss); mx = fmaxf(mx, fabsf(f[e])); }
#pragma unroll
        for (int o = 1; o < 8; o *= 2) { ss += __shfl_xor_sync(0xffffffffu, ss, o); mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o)); }
        int ex = (int)(__float_as_uint(mx) >> 23) - 127;      // the largest is in [2^ex, 2^(ex + 1))
        ex = mx == 0.f ? 0 : max(-120, min(120, ex));
        // (a row of zeros has no length to be divided by; any other's factor is at most 1, which keeps what is multiplied by it in f16's range)
        const float down = dl_pow2(-ex), unit = mx == 0.f ? 0.f : (float)sz_rsqrt64((double)ss + 1e-6);
        if (sub == 0) { if (isq) sRq[r] = unit * dl_pow2(ex) * a.q_scale; else sRk[r] = unit * dl_pow2(ex); }
        u32 hi[E / 2], lo[E / 2];
#pragma unroll
        for (int e = 0; e < E / 2; e++) dl_split(f[2 * e] * down, f[2 * e + 1] * down, hi[e], lo[e]);
#pragma unroll
        for (int p = 0; p < E / 8; p++) {
            const u32 at = (isq ? NK * C::TILE : 0) + dl_at<D>(r, sub * (E / 8) + p);
            *(uint4*)(sm + at) = *(uint4*)(hi + 4 * p);
            *(uint4*)(rows + at) = *(uint4*)(hi + 4 * p);
            if (NK == 2) { *(uint4*)(sm + C::TILE + at) = *(uint4*)(lo + 4 * p); *(uint4*)(rows + C::TILE + at) = *(uint4*)(lo + 4 * p); }
        }
    }
    __syncthreads();
    // k.k and q.k of the warp's 16 rows with those up to them: row g (+ 8), columns 8 m + 2 t (+ 1)
    float kk[8][4], qk[8][4];
#pragma unroll
    for (int m = 0; m < 8; m++)
#pragma unroll
        for (int i = 0; i < 4; i++) kk[m][i] = qk[m][i] = 0.f;
    const u32 sk = sz_smem_addr(sm);
#pragma unroll
    for (int ks = 0; ks < D / 16; ks++) {
        u32 ka[NK][4], qa[NK][4];
#pragma unroll
        for (int p = 0; p < NK; p++) {
            const u32 at = dl_at<D>(16 * warp + (lane & 15), 2 * ks + (lane >> 4)) + p * C::TILE;
            dl_ldsm(ka[p], sk + at);
            if (OUT) dl_ldsm(qa[p], sk + NK * C::TILE + at);
        }
#pragma unroll
        for (int m = 0; m < 8; m += 2)
            if (m <= 2 * warp + 1) {
                u32 b[NK][4];
#pragma unroll
                for (int p = 0; p < NK; p++) dl_ldsm(b[p], sk + p * C::TILE + dl_at<D>(8 * m + ((lane >> 4) << 3) + (lane & 7), 2 * ks + ((lane >> 3) & 1)));
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    dl_mma(kk[m + h], ka[0], b[0][2 * h], b[0][2 * h + 1]);
                    if (OUT) dl_mma(qk[m + h], qa[0], b[0][2 * h], b[0][2 * h + 1]);
                    if (NK == 2) {
                        dl_mma(kk[m + h], ka[0], b[1][2 * h], b[1][2 * h + 1]);
                        dl_mma(kk[m + h], ka[1], b[0][2 * h], b[0][2 * h + 1]);
                        if (OUT) { dl_mma(qk[m + h], qa[0], b[1][2 * h], b[1][2 * h + 1]); dl_mma(qk[m + h], qa[1], b[0][2 * h], b[0][2 * h + 1]); }
                    }
                }
            }
    }
    const int ratio = a.vh / a.kh;
    const int half = warp >> 1, part = warp & 1;             // the pair's value head of the warp's inverse, and its 32 columns
#pragma unroll 1
    for (int v0 = 0; v0 < ratio; v0 += 2) {
        auto head = [&](int i) { return a.grouped ? kx * ratio + v0 + i : (v0 + i) * a.kh + kx; };
        if (part == 0 && v0 + half < ratio) {                // gates of two rows a lane, and the sums of their logarithms
            const int h = head(half);
            double G[2];
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const int r = 2 * lane + i;
                float lgd = 0.f, be = 0.f;
                if (r < n) {
                    lgd = dl_log_decay(dl_load1<TYPE>(a.alpha + (row0 + r) * a.alpha_stride + (size_t)h * ESZ), a.a[h], a.dt[h]);
                    be = sz_sigmoid(dl_load1<TYPE>(a.beta + (row0 + r) * a.beta_stride + (size_t)h * ESZ));
                }
                G[i] = (double)lgd;
                sBeta[half][r] = be;
            }
            double sum = G[0] + G[1];
#pragma unroll
            for (int o = 1; o < 32; o *= 2) { const double y = __shfl_up_sync(0xffffffffu, sum, o); if (lane >= o) sum += y; }
            sG[half][2 * lane] = sum - G[1];
            sG[half][2 * lane + 1] = sum;
        }
        __syncthreads();
        // A by columns into shared memory, P as it is taken
#pragma unroll 1
        for (int i = 0; i < 2 && v0 + i < ratio; i++) {
            float* const At = (float*)(sm + C::ROWS) + i * (CK * DL_TS);
            u8* const hp = mine + (size_t)a.kh * C::ROWS + (size_t)head(i) * C::HEAD;
#pragma unroll
            for (int m = 0; m < 8; m++)
                if (m <= 2 * warp + 1) {
                    float p[4];
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const int r = 16 * warp + g + 8 * (e >> 1), j = 8 * m + 2 * t + (e & 1);
                        const float f = j <= r ? expf((float)(sG[i][r] - sG[i][j])) * sRk[j] : 0.f;
                        if (j < r) At[j * DL_AS + r] = sBeta[i][r] * f * sRk[r] * kk[m][e];
                        p[e] = j <= r ? f * sRq[r] * qk[m][e] * DL_P : 0.f;
                    }
                    if (OUT) {
#pragma unroll
                        for (int u = 0; u < 2; u++) {        // rows 8 (2 warp + u) + g: number m & 1 of the tile m / 2
                            u32 hi, lo;
                            dl_split(p[2 * u], p[2 * u + 1], hi, lo);
                            u32* const at = (u32*)(hp + 2 * DL_FRAG) + ((dl_tile(2 * warp + u) + m / 2) * 32 + lane) * 2 + (m & 1);
                            *at = hi;
                            if (C::FULL) *(at + DL_FRAG / 4) = lo;
                        }
                    }
                }
        }
        __syncthreads();
        // column j of (I + A)^-1 a thread: its elements from the top down, each one taken from those below it as soon as it is known
        const bool live = v0 + half < ratio;
        float x[CK];
        float* const At = (float*)(sm + C::ROWS) + half * (CK * DL_TS);
        const int col = part * 32 + lane;
        if (live) {
#pragma unroll
            for (int i = 0; i < CK; i++) x[i] = i == col ? 1.f : 0.f;
#pragma unroll
            for (int m = 0; m < CK - 1; m++)
                if (m >= 32 || part == 0) {                  // (columns from 32 on are nothing above their own row)
#pragma unroll
                    for (int i4 = (m + 1) & ~3; i4 < CK; i4 += 4) {
                        const float4 w = *(const float4*)(At + m * DL_AS + i4);
                        const float wa[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                        for (int e = 0; e < 4; e++) if (i4 + e > m) x[i4 + e] = fmaf(-wa[e], x[m], x[i4 + e]);
                    }
                }
        }
        __syncthreads();                                     // (T takes A's place)
        if (live) {
            const float be = sBeta[half][col];
#pragma unroll
            for (int i = 0; i < CK; i++) At[i * DL_TS + col] = x[i] * be;
        }
        __syncthreads();
        if (live) {
            const int h = head(half);
            u8* const hp = mine + (size_t)a.kh * C::ROWS + (size_t)h * C::HEAD;
#pragma unroll
            for (int m = 0; m < 8; m++)
#pragma unroll
                for (int k2 = 0; k2 <= m / 2; k2++)
                    if (((dl_tile(m) + k2) & 1) == part) {
                        const float* w = At + (8 * m + g) * DL_TS + 16 * k2 + 2 * t;
                        const float2 w0 = *(const float2*)w, w1 = *(const float2*)(w + 8);
                        uint2 hi, lo;
                        dl_split(w0.x, w0.y, hi.x, lo.x);
                        dl_split(w1.x, w1.y, hi.y, lo.y);
                        const int at = (dl_tile(m) + k2) * 32 + lane;
                        ((uint2*)hp)[at] = hi;
                        ((uint2*)(hp + DL_FRAG))[at] = lo;
                    }
            DlScalars* const sc = (DlScalars*)(hp + (C::FULL ? 4 : 3) * DL_FRAG);
            const int r = col;
            const double G = sG[half][r], GC = sG[half][CK - 1];
            const float eg = expf((float)G);
            sc->gr[r] = eg * sRk[r];
            if (OUT) sc->gq[r] = eg * sRq[r];
            sc->wj[r] = expf((float)(GC - G)) * sRk[r];
            if (r == 0) sc->gc = expf((float)GC);
        }
        __syncthreads();                                     // (the next pair's gates)
    }
}

// ---- the chain over a sequence's chunks --------------------------------------------------------------------------------------------------------
template <int D, int TYPE, int NG> struct DlMain {
    using C = DlChunk<D, TYPE>;
    static constexpr int ESZ = DlIo<TYPE>::ESZ, NQ = D / 64, NW = NG * NQ, NTH = 32 * NW, CS = D / 16 / NG;      // warps on one 16 dimensions; warps; blocks of a head
    static constexpr int VS = 16 * NG * ESZ + 16;                                          // bytes between rows of v and z in shared memory
    static constexpr int STAGE = C::ROWS + C::HEAD + 2 * CK * VS, STAGES = D == 128 && TYPE == SZ_TYPE_F32 ? 1 : 2;
    static constexpr int XB = NQ == 2 ? 12 * 32 * 16 : 0;                                  // what a warp gives its partner
    static constexpr int OS = 16 * ESZ + 16, OB = CK / NQ * OS;                            // a warp's outputs on their way
    static constexpr int SSQ = 2 * CS * NG * CK * 4;
    static constexpr size_t SMEM = (size_t)STAGES * STAGE + NW * (XB + OB) + SSQ + 64;
};

template <int D, int TYPE, int NG, bool OUT>
__global__ void __launch_bounds__(DlMain<D, TYPE, NG>::NTH, 1)
sz_delta_chunk_kernel(const DlBatch d, const DlRule a, int idx0, int idx1, const u8* __restrict__ scratch, long long one) {
    using M = DlMain<D, TYPE, NG>;
    using C = DlChunk<D, TYPE>;
    constexpr int ESZ = M::ESZ, NQ = M::NQ, NK = C::NK, CS = M::CS, ST = M::STAGES, OT = 8 / NQ;      // OT: 8-row tiles whose outputs a warp finishes
    extern __shared__ __align__(16) u8 sm[];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, p = warp / NQ, q = warp % NQ, g = lane >> 2, t = lane & 3;
    const int h = blockIdx.x / CS, rank = blockIdx.x % CS, kx = a.grouped ? h / (a.vh / a.kh) : h % a.kh;
    u8* const xb = sm + ST * M::STAGE;
    u8* const ob = xb + M::NW * M::XB + warp * M::OB;
    float* const ssq = (float*)(xb + M::NW * (M::XB + M::OB));            // [parity][block][group][row]
    u64* const bar = (u64*)(ssq + M::SSQ / 4);
    const bool norm = OUT && a.norm != nullptr, joined = norm && CS > 1;
    if (tid == 0) {
        for (int i = 0; i < ST; i++) sz_mbar_init(&bar[i], 1);
        sz_mbar_fence_init();
    }
    sz_pdl_wait();
    sz_pdl_trigger();
    const DlLong lg = dl_find(d, a.least, blockIdx.y, 0, lane);
    if (lg.b < 0) return;                                                 // (the blocks of a head are all of one sequence: they leave together)
    const DlSeq s = dl_seq(d, lg.b, lane, false);
    const int chunks = (s.n + CK - 1) / CK;
    const int c0 = max(0, idx0 - lg.base), c1 = min(chunks, idx1 - lg.base);
    // (a sequence none of whose rows count still moves its state, in the pass that has its first place)
    const bool only = s.on && chunks == 0 && lg.base >= idx0 && lg.base < idx1;
    if (!s.on || (c0 >= c1 && !only)) return;
    const int dv = (rank * NG + p) * 16;                                  // the warp's value dimensions
    __syncthreads();
    // S^T: dimensions g, g + 8; key dimensions 64 q + 8 m + 2 t, + 1
    float S[8][4];
    int es = 0;                                                           // .. in units of 2^es
    {
        const int from = c0 > 0 ? s.to : s.from;
        const float* src = (const float*)(a.state + (size_t)max(from, 0) * a.state_stride) + ((size_t)h * D + 64 * q + 2 * t) * D + dv + g;
#pragma unroll
        for (int m = 0; m < 8; m++)
#pragma unroll
            for (int e = 0; e < 4; e++) S[m][e] = from >= 0 ? src[(size_t)(8 * m + (e & 1)) * D + 8 * (e >> 1)] : 0.f;
    }
    auto issue = [&](int c) {
        u8* const st = sm + ((c - c0) % ST) * M::STAGE;
        const int n = min(CK, s.n - c * CK);
        if (tid == 0) {
            const u8* src = scratch + (size_t)(lg.base + c - idx0) * one;
            u64* const full = &bar[(c - c0) % ST];
            asm volatile("fence.proxy.async;" ::: "memory");
            sz_mbar_expect_tx(full, (OUT ? C::ROWS : C::ROWS / 2) + C::HEAD);
            sz_bulk_g2s(st, src + (size_t)kx * C::ROWS, OUT ? C::ROWS : C::ROWS / 2, full);
            sz_bulk_g2s(st + C::ROWS, src + (size_t)a.kh * C::ROWS + (size_t)h * C::HEAD, C::HEAD, full);
        }
        constexpr int PIECES = 16 * NG * ESZ / 16;
        const size_t row0 = (size_t)s.r0 + (size_t)c * CK;
        for (int i = tid; i < CK * PIECES; i += M::NTH) {
            const int r = i / PIECES, x = i % PIECES;
            const u32 to = sz_smem_addr(st + C::ROWS + C::HEAD + r * M::VS + 16 * x);
            const int take = r < n ? 16 : 0;                              // (rows behind the last are zeros, and not read)
            const size_t row = row0 + (r < n ? r : 0), col = (size_t)(h * D + rank * NG * 16) * ESZ + 16 * x;
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(a.v + row * a.v_stride + col), "r"(take) : "memory");
            if (norm) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to + CK * M::VS), "l"(a.z + row * a.z_stride + col), "r"(take) : "memory");
        }
        sz_cp_async_commit();
    };
    // 16 value dimensions of a tile's rows, transposed: dimensions g, g + 8 of rows 8 m + 2 t, + 1
    auto turned = [&](const u8* tile, int m, float* f) {                  // (two tiles of 8 rows: m, m + 1)
        if constexpr (TYPE == SZ_TYPE_F32) {
#pragma unroll
            for (int i = 0; i < 2; i++)
#pragma unroll
                for (int e = 0; e < 4; e++) f[4 * i + e] = *(const float*)(tile + (8 * (m + i) + 2 * t + (e & 1)) * M::VS + (16 * p + g + 8 * (e >> 1)) * 4);
        } else {
            u32 w[4];
            dl_ldsm_t(w, sz_smem_addr(tile + (8 * m + ((lane >> 4) << 3) + (lane & 7)) * M::VS + (16 * p + ((lane >> 3) & 1) * 8) * 2));
            dl_unpack<TYPE, 8>(w, f);
        }
    };
    float O[4 * OT];                                                      // outputs of the chunk before, on their way to their norm
    float nw[2] = {0.f, 0.f};
    if (norm) { nw[0] = a.norm[dv + g]; nw[1] = a.norm[dv + g + 8]; }
    // the tiles whose outputs the warp finishes: pairs of like work
    auto mine = [&](int i) { return NQ == 1 ? i : q == 0 ? (i < 2 ? i : i + 4) : i + 2; };
    auto finish = [&](int c) {                                            // outputs of chunk c: their norm's factor, into shared memory by rows, out
        const int n = min(CK, s.n - c * CK);
#pragma unroll
        for (int i = 0; i < OT; i++) {
            float r0 = 1.f, r1 = 1.f;
            const int row = 8 * mine(i) + 2 * t;
            if (norm) {
                float2 sum = make_float2(0.f, 0.f);
                const float* w = ssq + (size_t)((c - c0) & 1) * CS * NG * CK + row;
#pragma unroll
                for (int j = 0; j < CS * NG; j++) { const float2 y = *(const float2*)(w + j * CK); sum.x += y.x; sum.y += y.y; }
                r0 = rsqrtf(sum.x * (1.f / D) + a.eps); r1 = rsqrtf(sum.y * (1.f / D) + a.eps);
            }
            O[4 * i] *= r0; O[4 * i + 1] *= r1; O[4 * i + 2] *= r0; O[4 * i + 3] *= r1;
            // row 8 i + 2 t (+ 1) of the warp's, dimension g (+ 8)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                u8* const at = ob + (8 * i + 2 * t + (e & 1)) * M::OS + (g + 8 * (e >> 1)) * ESZ;
                if constexpr (TYPE == SZ_TYPE_F32) *(float*)at = O[4 * i + e];
                else if constexpr (TYPE == SZ_TYPE_F16) *(__half*)at = __float2half_rn(O[4 * i + e]);
                else *(__nv_bfloat16*)at = __float2bfloat16_rn(O[4 * i + e]);
            }
        }
        __syncwarp();
        constexpr int PIECES = ESZ;                                       // of 16 bytes, a row's 16 dimensions
        for (int i = lane; i < 8 * OT * PIECES; i += 32) {
            const int r = i / PIECES, x = i % PIECES, row = 8 * mine(r / 8) + r % 8;
            if (row < n) *(uint4*)(a.out + ((size_t)s.r0 + (size_t)c * CK + row) * a.out_stride + (size_t)(h * D + dv) * ESZ + 16 * x) = *(const uint4*)(ob + r * M::OS + 16 * x);
        }
        __syncwarp();
    };
    if (joined) sz_cluster_sync();                                        // (all blocks of the head have begun)
    bool dead = false;
    if (c0 < c1) issue(c0);
#pragma unroll 1
    for (int c = c0; c < c1; c++) {
        const int slot = (c - c0) % ST;
        const bool more = c + 1 < c1;
        if (ST == 2 && more) { issue(c + 1); sz_cp_async_wait<1>(); }
        else sz_cp_async_wait<0>();
        if (!dead && !sz_mbar_wait_warp(&bar[slot], ((c - c0) / ST) & 1)) { dead = true; if (lane == 0) atomicOr(d.err, DL_E_WAIT); }
        __syncthreads();
        const u8* const st = sm + slot * M::STAGE;
        const u32 sk = sz_smem_addr(st), sq = sk + NK * C::TILE;
        const u8* const hp = st + C::ROWS;
        const DlScalars* const sc = (const DlScalars*)(hp + (C::FULL ? 4 : 3) * DL_FRAG);
        const u8* const vt = st + C::ROWS + C::HEAD;
        // ---- the state into f16's range
        {
            float mx = 0.f;
#pragma unroll
            for (int m = 0; m < 8; m++)
#pragma unroll
                for (int e = 0; e < 4; e++) mx = fmaxf(mx, fabsf(S[m][e]));
            const u32 top = __reduce_max_sync(0xffffffffu, __float_as_uint(mx)) >> 23;
            const int ex = (int)top - 127;
            if (top != 0 && top != 255 && (ex > 13 || ex < 4)) {
                const int up = max(-120, min(120, 10 - ex));
                const float f = dl_pow2(up);
#pragma unroll
                for (int m = 0; m < 8; m++)
#pragma unroll
                    for (int e = 0; e < 4; e++) S[m][e] *= f;
                es -= up;
            }
        }
        // ---- (K S)^T and (Q S)^T: dimensions x rows
        float X[8][4], Y[8][4];
#pragma unroll
        for (int m = 0; m < 8; m++)
#pragma unroll
            for (int e = 0; e < 4; e++) X[m][e] = Y[m][e] = 0.f;
#pragma unroll
        for (int ks = 0; ks < 4; ks++) {
            u32 hi[4], lo[4];
#pragma unroll
            for (int e = 0; e < 4; e++) dl_split(S[2 * ks + (e >> 1)][2 * (e & 1)], S[2 * ks + (e >> 1)][2 * (e & 1) + 1], hi[e], lo[e]);
#pragma unroll
            for (int m = 0; m < 8; m += 2) {
                const u32 at = dl_at<D>(8 * m + ((lane >> 4) << 3) + (lane & 7), 8 * q + 2 * ks + ((lane >> 3) & 1));
                u32 b[4], b2[4];
                dl_ldsm(b, sk + at);
                if (NK == 2) dl_ldsm(b2, sk + C::TILE + at);
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    dl_mma(X[m + i], hi, b[2 * i], b[2 * i + 1]);
                    dl_mma(X[m + i], lo, b[2 * i], b[2 * i + 1]);
                    if (NK == 2) dl_mma(X[m + i], hi, b2[2 * i], b2[2 * i + 1]);
                }
                if (OUT) {
                    dl_ldsm(b, sq + at);
                    if (NK == 2) dl_ldsm(b2, sq + C::TILE + at);
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        dl_mma(Y[m + i], hi, b[2 * i], b[2 * i + 1]);
                        if (C::FULL) dl_mma(Y[m + i], lo, b[2 * i], b[2 * i + 1]);
                        if (NK == 2) dl_mma(Y[m + i], hi, b2[2 * i], b2[2 * i + 1]);
                    }
                }
            }
        }
        const float true_s = dl_pow2(es);
#pragma unroll
        for (int m = 0; m < 8; m++)
#pragma unroll
            for (int e = 0; e < 4; e++) { X[m][e] *= true_s; if (OUT) Y[m][e] *= true_s; }
        if constexpr (NQ == 2) {                                          // with the other key dimensions'
            float4* const to = (float4*)(xb + warp * M::XB);
            const float4* const from = (const float4*)(xb + (warp ^ 1) * M::XB);
#pragma unroll
            for (int m = 0; m < 8; m++) to[m * 32 + lane] = make_float4(X[m][0], X[m][1], X[m][2], X[m][3]);
            if (OUT)
#pragma unroll
                for (int i = 0; i < 4; i++) {                             // the tiles that the partner finishes
                    const int mq0 = i + 2, mq1 = i < 2 ? i : i + 4;       // .. of q = 1, of q = 0
                    to[(8 + i) * 32 + lane] = q == 0 ? make_float4(Y[mq0][0], Y[mq0][1], Y[mq0][2], Y[mq0][3]) : make_float4(Y[mq1][0], Y[mq1][1], Y[mq1][2], Y[mq1][3]);
                }
            asm volatile("bar.sync %0, 64;" ::"r"(1 + p) : "memory");
#pragma unroll
            for (int m = 0; m < 8; m++) {
                const float4 y = from[m * 32 + lane];
                X[m][0] += y.x; X[m][1] += y.y; X[m][2] += y.z; X[m][3] += y.w;
            }
            if (OUT)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float4 y = from[(8 + i) * 32 + lane];
                    const int m0 = i < 2 ? i : i + 4, m1 = i + 2;
                    // (own tiles side by side in Y's first four)
                    const float o0 = q == 0 ? Y[m0][0] : Y[m1][0], o1 = q == 0 ? Y[m0][1] : Y[m1][1], o2 = q == 0 ? Y[m0][2] : Y[m1][2], o3 = q == 0 ? Y[m0][3] : Y[m1][3];
                    Y[i][0] = o0 + y.x; Y[i][1] = o1 + y.y; Y[i][2] = o2 + y.z; Y[i][3] = o3 + y.w;
                }
        }
        // ---- R = V - e^G K S, in units of 2^ew
        float mx = 0.f;
#pragma unroll
        for (int m = 0; m < 8; m += 2) {
            float v[8];
            turned(vt, m, v);
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const float2 gr = *(const float2*)(sc->gr + 8 * (m + i) + 2 * t);
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    X[m + i][e] = fmaf(-(e & 1 ? gr.y : gr.x), X[m + i][e], v[4 * i + e]);
                    mx = fmaxf(mx, fabsf(X[m + i][e]));
                }
            }
        }
        int ew = es;
        {
            const u32 top = __reduce_max_sync(0xffffffffu, __float_as_uint(mx)) >> 23;
            if (top != 0 && top != 255) ew = max(max((int)top - 127 - 8, -120), es - 100);      // (changes are at most 64 times the largest of R: below 2^15)
        }
        u32 rh[4][4], rl[4][4];
        {
            const float f = dl_pow2(-ew);
#pragma unroll
            for (int ks = 0; ks < 4; ks++)
#pragma unroll
                for (int e = 0; e < 4; e++) dl_split(X[2 * ks + (e >> 1)][2 * (e & 1)] * f, X[2 * ks + (e >> 1)][2 * (e & 1) + 1] * f, rh[ks][e], rl[ks][e]);
        }
        // ---- the rows' changes D^T = R^T T^T
#pragma unroll
        for (int m = 0; m < 8; m++) {
#pragma unroll
            for (int e = 0; e < 4; e++) X[m][e] = 0.f;
#pragma unroll
            for (int ks = 0; ks <= m / 2; ks++) {
                const uint2 th = ((const uint2*)hp)[(dl_tile(m) + ks) * 32 + lane], tl = ((const uint2*)(hp + DL_FRAG))[(dl_tile(m) + ks) * 32 + lane];
                dl_mma(X[m], rh[ks], th.x, th.y);
                dl_mma(X[m], rl[ks], th.x, th.y);
                dl_mma(X[m], rh[ks], tl.x, tl.y);
            }
        }
        // ---- outputs: e^G Q S + P D
        if (OUT) {
            if (norm && c > c0) {                                         // the chunk before: its sums are here
                if (joined) sz_cluster_wait();
                finish(c - 1);
            }
            u32 dh[4][4], dlo[4][4];
#pragma unroll
            for (int ks = 0; ks < 4; ks++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    if (C::FULL) dl_split(X[2 * ks + (e >> 1)][2 * (e & 1)], X[2 * ks + (e >> 1)][2 * (e & 1) + 1], dh[ks][e], dlo[ks][e]);
                    else dh[ks][e] = dl_h2(X[2 * ks + (e >> 1)][2 * (e & 1)], X[2 * ks + (e >> 1)][2 * (e & 1) + 1]);
                }
            const float tw = dl_pow2(ew) * (1.f / DL_P);
            const u8* const zt = vt + CK * M::VS;
#pragma unroll
            for (int i = 0; i < OT; i += 2) {
                const int m0 = mine(i);                                   // (tiles m0, m0 + 1: their 16-row columns end with theirs)
                float acc[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
                for (int u = 0; u < 2; u++)
#pragma unroll
                    for (int ks = 0; ks < 4; ks++)
                        if (ks <= m0 / 2) {
                            const int at = (dl_tile(m0 + u) + ks) * 32 + lane;
                            const uint2 ph = ((const uint2*)(hp + 2 * DL_FRAG))[at];
                            dl_mma(acc[u], dh[ks], ph.x, ph.y);
                            if (C::FULL) {
                                const uint2 pl = ((const uint2*)(hp + 3 * DL_FRAG))[at];
                                dl_mma(acc[u], dlo[ks], ph.x, ph.y);
                                dl_mma(acc[u], dh[ks], pl.x, pl.y);
                            }
                        }
                float z[8];
                if (norm) turned(zt, m0, z);
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    const float2 gq = *(const float2*)(sc->gq + 8 * (m0 + u) + 2 * t);
#pragma unroll
                    for (int e = 0; e < 4; e++) O[4 * (i + u) + e] = fmaf(e & 1 ? gq.y : gq.x, Y[i + u][e], acc[u][e] * tw);
                    if (norm) {
                        float s0 = fmaf(O[4 * (i + u)], O[4 * (i + u)], O[4 * (i + u) + 2] * O[4 * (i + u) + 2]);
                        float s1 = fmaf(O[4 * (i + u) + 1], O[4 * (i + u) + 1], O[4 * (i + u) + 3] * O[4 * (i + u) + 3]);
#pragma unroll
                        for (int o = 4; o < 32; o *= 2) { s0 += __shfl_xor_sync(0xffffffffu, s0, o); s1 += __shfl_xor_sync(0xffffffffu, s1, o); }
                        float* const at = ssq + ((size_t)((c - c0) & 1) * CS * NG + rank * NG + p) * CK + 8 * (m0 + u) + 2 * t;
                        if (CS == 1) { if (g == 0) *(float2*)at = make_float2(s0, s1); }
                        else if (g < CS) {                                // lanes of g: to block g of the head
                            u32 there;
                            asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(sz_smem_addr(at)), "r"(g));
                            asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(there), "f"(s0), "f"(s1) : "memory");
                        }
#pragma unroll
                        for (int e = 0; e < 4; e++) O[4 * (i + u) + e] *= nw[e >> 1] * sz_sigmoid(z[4 * u + e]);
                    }
                }
            }
            if (joined) sz_cluster_arrive();
            if (!norm) finish(c);
        }
        // ---- the state: e^G_C S + K^T (e^(G_C - G_j) D)
        {
#pragma unroll
            for (int m = 0; m < 8; m++) {
                const float2 w = *(const float2*)(sc->wj + 8 * m + 2 * t);
                X[m][0] *= w.x; X[m][1] *= w.y; X[m][2] *= w.x; X[m][3] *= w.y;
            }
            const float f = sc->gc * dl_pow2(max(es - ew, -126));
#pragma unroll
            for (int m = 0; m < 8; m++)
#pragma unroll
                for (int e = 0; e < 4; e++) S[m][e] *= f;
            es = ew;
#pragma unroll
            for (int ks = 0; ks < 4; ks++) {
                u32 hi[4], lo[4];
#pragma unroll
                for (int e = 0; e < 4; e++) dl_split(X[2 * ks + (e >> 1)][2 * (e & 1)], X[2 * ks + (e >> 1)][2 * (e & 1) + 1], hi[e], lo[e]);
#pragma unroll
                for (int m = 0; m < 8; m += 2) {
                    const u32 at = dl_at<D>(16 * ks + (((lane >> 3) & 1) << 3) + (lane & 7), 8 * q + m + (lane >> 4));
                    u32 b[4], b2[4];
                    dl_ldsm_t(b, sk + at);
                    if (NK == 2) dl_ldsm_t(b2, sk + C::TILE + at);
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        dl_mma(S[m + i], hi, b[2 * i], b[2 * i + 1]);
                        dl_mma(S[m + i], lo, b[2 * i], b[2 * i + 1]);
                        if (NK == 2) dl_mma(S[m + i], hi, b2[2 * i], b2[2 * i + 1]);
                    }
                }
            }
        }
        __syncthreads();                                                  // (the stage is free, and the sums of squares of this block are there)
        if (ST == 1 && more) issue(c + 1);
    }
    if (norm && c0 < c1) {
        if (joined) sz_cluster_wait();
        finish(c1 - 1);
    }
    float* to = (float*)(a.state + (size_t)s.to * a.state_stride) + ((size_t)h * D + 64 * q + 2 * t) * D + dv + g;
    const float f0 = dl_pow2(es / 2), f1 = dl_pow2(es - es / 2);          // (in two steps: 2^es alone may be out of range)
#pragma unroll
    for (int m = 0; m < 8; m++)
#pragma unroll
        for (int e = 0; e < 4; e++) to[(size_t)(8 * m + (e & 1)) * D + 8 * (e >> 1)] = S[m][e] * f0 * f1;
}

template <int D, int TYPE, int NG, bool OUT>
int dl_chunk_go(const DlBatch& b, const DlRule& r, int longest, int64_t total, int64_t per, uint64_t scratch, cudaStream_t st) {
    using P = DlPrep<D, TYPE>;
    using M = DlMain<D, TYPE, NG>;
    static_assert(M::SMEM <= 227 * 1024 && P::SMEM <= 113 * 1024, "");
    const auto prep = sz_delta_prep_kernel<D, TYPE, OUT>;
    const auto chain = sz_delta_chunk_kernel<D, TYPE, NG, OUT>;
    int rc = sz_allow_smem((const void*)prep, (int)P::SMEM);
    if (rc || (rc = sz_allow_smem((const void*)chain, (int)M::SMEM))) return rc;
    const long long one = (long long)dl_chunk_one(D, r.kh, r.vh, TYPE);
    for (int64_t i0 = 0; i0 < total; i0 += per) {
        const int64_t i1 = i0 + per < total ? i0 + per : total;
        SZ_CUDA(sz_launch("delta_prep", prep, dim3((unsigned)(i1 - i0), r.kh), dim3(128), P::SMEM, st, true, b, r, (int)i0, (u8*)scratch, one));
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(r.vh * M::CS, longest);
        cfg.blockDim = dim3(M::NTH);
        cfg.dynamicSmemBytes = M::SMEM;
        cfg.stream = st;
        cudaLaunchAttribute attr[2];
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        attr[1].id = cudaLaunchAttributeClusterDimension;
        attr[1].val.clusterDim.x = M::CS;
        attr[1].val.clusterDim.y = 1;
        attr[1].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = M::CS > 1 ? 2 : 1;
        SZ_CUDA(cudaLaunchKernelEx(&cfg, chain, b, r, (int)i0, (int)i1, (const u8*)scratch, one));
        sz_trace_mark("delta_chunk", st);
    }
    return SZ_OK;
}

int64_t dl_total(int n_seq, int rows, int least) { return rows / CK + (n_seq < rows / least ? n_seq : rows / least) + 1; }

}  // namespace

int64_t dl_chunk_bytes(int d, int kh, int vh, int io_type, int n_seq, int rows, int least) {
    const int64_t one = dl_chunk_one(d, kh, vh, io_type), total = dl_total(n_seq, rows, least), per = DL_SLAB / one < 8 ? 8 : DL_SLAB / one;
    return one * (total < per ? total : per);
}

int dl_chunk_launch(int d, int io_type, const DlBatch& b, const DlRule& r, uint64_t scratch, cudaStream_t st) {
    const int64_t one = dl_chunk_one(d, r.kh, r.vh, io_type), total = dl_total(b.n_seq, b.rows, r.least), per = DL_SLAB / one < 8 ? 8 : DL_SLAB / one;
    const int longest = b.n_seq < b.rows / r.least ? b.n_seq : b.rows / r.least;
    const bool out = r.q != nullptr;
#define SZ_DL_GO(D_, T_, N_) (out ? dl_chunk_go<D_, T_, N_, true>(b, r, longest, total, per, scratch, st) : dl_chunk_go<D_, T_, N_, false>(b, r, longest, total, per, scratch, st))
#define SZ_DL_IO(D_, N_) (io_type == SZ_TYPE_F32 ? SZ_DL_GO(D_, SZ_TYPE_F32, N_) : io_type == SZ_TYPE_F16 ? SZ_DL_GO(D_, SZ_TYPE_F16, N_) : SZ_DL_GO(D_, SZ_TYPE_BF16, N_))
    return d == 128 ? SZ_DL_IO(128, 2) : SZ_DL_IO(64, 4);
#undef SZ_DL_IO
#undef SZ_DL_GO
}
