// The gated delta rule over many rows of a sequence, in chunks of CK = 64 (sz_delta.cuh has the row-by-row form's neighbours).
//
// With S the state before a chunk, G_i the sum of the decays' logarithms up to its row i, and k, q the normed rows, the rows' changes d_i solve a triangular system:
//   (I + A) D = R = diag(beta) (V - diag(e^G) K S),   A_ij = beta_i e^(G_i - G_j) k_i.k_j for j < i
//   O = diag(e^G) Q S + P D,   P_ij = e^(G_i - G_j) q_i.k_j for j <= i (held without q_i's length)
//   S' = e^G_C S + sum_j e^(G_C - G_j) k_j d_j^T
// so that a chunk is a few matrix products instead of 64 steps.  Two kernels:
//  sz_delta_prep_kernel, a block a chunk and key head: what does not need S - the products of its rows, T = (I + A)^-1 and P of every value head of the
//   key head - side by side, over all chunks at once;
//  sz_delta_chunk_kernel, a block of warps for 16 NG value dimensions of a sequence's value head: the chain over its chunks, on mma.sync.  Everything is
//   transposed, so that a warp's 16 value dimensions are a product's rows: S^T (f32) stays in its registers, and what one product gives is in the layout in which
//   the next one takes it.  At 128 key dimensions two warps have 64 of them each and add up K S and Q S through shared memory.
// 4,093 rows of 32 heads of 128 on 16, bf16: 48 us and 185 (137 MB: 21 of them); a chunk of the chain is some 5,400 cycles, 42 % of them with the matrix pipe at work, the rest what lies between one
// product and the next: the largest of the state, the partner's part, R, two numbers of a factor, waits.
// tcgen05 would have the products' time, but every one of the chain's links would go through tensor memory and back (300 - 400 cycles a wait, three
// a chunk) and S through a conversion by four warps: no sooner.
//
// Numbers.  A row k = rho 2^e (k 2^-e) enters the products as k 2^-e with its largest element in [1, 2): a bf16 or f16 row is exact in f16, an f32 row is two f16
// numbers (22 bits); the rows' lengths and powers are factors in f32, and so is beta: a chunk whose gates are all but closed keeps the digits of its small changes, where T diag(beta) in f16
// has none below 2^-25.  (T's elements are at most 1, its diagonal is 1.)  S, R and D enter as two f16 numbers each, in units of a power of two that
// the warp takes from the largest there is: 22 bits, and what is less than 2^-35 of that largest is lost.  Sums are f32.  T and the decays' sums: f32 and f64.
// (One f16 number a factor in the last products of bf16 outputs, 11 bits where they keep 8: their difference from rounded f32 outputs is 1.1 10^-3 of their size instead of 3 10^-5; 4,093 rows took 202 us so, and 221 with two.)
#include "sz_delta.cuh"

namespace {

constexpr int CK = 64, DL_TILES = 20;                    // rows of a chunk; 8 x 16 tiles of a lower triangle
constexpr int DL_FRAG = DL_TILES * 32 * 8;               // bytes of a triangle in f16, in the order in which the matrix instruction takes it
constexpr int64_t DL_SLAB = 96ll << 20;                  // scratch that a pass over chunks may take (what the first kernel leaves is in L2 for the second)

struct DlScalars { float gr[CK], beta[CK], wj[CK], gc; int ex; float pad[14]; };      // - beta e^G rho_k, beta, 2^-ex e^(G_C - G_j) rho_k; e^G_C, and what makes the largest wj 0.5 to 1

template <int D, int TYPE> struct DlChunk {
    static constexpr int NK = TYPE == SZ_TYPE_F32 ? 2 : 1;                // f16 numbers of an element of k and q
    static constexpr int TILE = CK * D * 2, ROWS = 2 * NK * TILE;         // a key head's rows: k (high, low), q (high, low)
    // a value head's T (high, low) and scalars, for the chain; P (high, low), e^G rho_q and rho_q, for the outputs
    static constexpr int HA = 2 * DL_FRAG + (int)sizeof(DlScalars), HB = 2 * DL_FRAG + 2 * CK * 4, HEAD = HA + HB;
};
int64_t dl_chunk_one(int d, int kh, int vh, int io_type) {
    const int nk = io_type == SZ_TYPE_F32 ? 2 : 1;
    return (int64_t)kh * 2 * nk * CK * d * 2 + (int64_t)vh * (4 * DL_FRAG + 2 * CK * 4 + (int)sizeof(DlScalars));
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
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void dl_ldsm(u32* r, u32 addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void dl_ldsm_t(u32* r, u32 addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void dl_stsm_t(u32 addr, const u32* r) {
    asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]) : "memory");
}
__device__ __forceinline__ void dl_scale4(float* x, float f) {
    const u64 f2 = dl_pack2(f, f), a = dl_mul2(dl_pack2(x[0], x[1]), f2), b = dl_mul2(dl_pack2(x[2], x[3]), f2);
    x[0] = dl_lo(a); x[1] = dl_hi(a); x[2] = dl_lo(b); x[3] = dl_hi(b);
}
// byte of the 16-byte piece c of row r of a tile [rows][D] of f16: pieces exchanged so that ldmatrix meets no bank twice
template <int D> __device__ __forceinline__ u32 dl_at(int r, int c) { return (u32)(r * D * 2 + ((c ^ (r & 7)) << 4)); }
// the first of the tiles of 8 rows n of a lower triangle (its 16-column tiles are side by side)
__host__ __device__ constexpr int dl_tile(int n) { return (n / 2) * (n / 2 + 1) + (n & 1) * (n / 2 + 1); }
__device__ __forceinline__ float dl_pow2(int e) { return e < -126 ? 0.f : __uint_as_float((u32)(min(e, 127) + 127) << 23); }

// ---- what does not need the state -----------------------------------------------------------------------------------------------------------
// The inverse goes by blocks of 16 rows: those on the diagonal in f32, a column a lane, top down; the others column of blocks by column of blocks,
//   X_ab = - X_aa sum_{b <= c < a} A_ac X_cb,
// on mma.sync with two f16 numbers a factor, transposed, so that a product's result is the next one's factor.  e^(G_i - G_j) of different blocks is the product of two
// exponentials that meet at the first row of i's block (both at most 1), of one block an exponential of its own.
constexpr int DL_OFF = 12, DL_DS = 20;                   // 8 x 16 tiles below the diagonal's blocks; stride of a block on it
template <int D, int TYPE> struct DlPrep {
    static constexpr int ROWS = DlChunk<D, TYPE>::ROWS;
    static constexpr int AF = DL_OFF * 32 * 8 * 2, DG = 4 * 16 * DL_DS * 4, HEAD = AF + DG;      // a value head's A (high, low), and its blocks on the diagonal, then their inverses
    static constexpr size_t SMEM = ROWS > 2 * HEAD ? ROWS : 2 * HEAD;                            // (where the rows were)
};
__device__ __forceinline__ u32 dl_turn(u32 a) { u32 d; asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a)); return d; }

template <int D, int TYPE, bool OUT>
__global__ void __launch_bounds__(128, TYPE == SZ_TYPE_F32 ? 2 : 4)
sz_delta_prep_kernel(const DlBatch d, const DlRule a, int idx0, u8* __restrict__ scratch, long long one) {
    using C = DlChunk<D, TYPE>;
    using P = DlPrep<D, TYPE>;
    constexpr int ESZ = DlIo<TYPE>::ESZ, NK = C::NK, E = D / 8, W = E * ESZ / 16;
    extern __shared__ __align__(16) u8 sm[];
    __shared__ double sG[2][CK];
    __shared__ float sRk[CK], sRq[CK], sBeta[2][CK], sE[2][CK], sB[2][4][CK];      // e^(G_i - G_first of its block); e^(G_first of a block - G_j) rho_k
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
    const int ratio = a.vh / a.kh;
    auto head = [&](int i) { return a.grouped ? kx * ratio + i : i * a.kh + kx; };      // the key head's i-th value head
    // a pair's gates: two rows a lane of warps 0 and 1, and the sums of the decays' logarithms
    float al[2] = {0.f, 0.f}, be[2] = {0.f, 0.f};
    auto ask_gates = [&](int v0) {
        if (warp < 2 && v0 + warp < ratio)
#pragma unroll
            for (int i = 0; i < 2; i++)
                if (2 * lane + i < n) {
                    const size_t row = row0 + 2 * lane + i;
                    al[i] = dl_load1<TYPE>(a.alpha + row * a.alpha_stride + (size_t)head(v0 + warp) * ESZ);
                    be[i] = dl_load1<TYPE>(a.beta + row * a.beta_stride + (size_t)head(v0 + warp) * ESZ);
                }
    };
    auto sum_gates = [&](int v0) {
        if (warp < 2 && v0 + warp < ratio) {
            const int h = head(v0 + warp);
            double G[2];
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const bool in = 2 * lane + i < n;
                G[i] = in ? (double)dl_log_decay(al[i], a.a[h], a.dt[h]) : 0.0;
                sBeta[warp][2 * lane + i] = in ? sz_sigmoid(be[i]) : 0.f;
            }
            double sum = G[0] + G[1];
#pragma unroll
            for (int o = 1; o < 32; o *= 2) { const double y = __shfl_up_sync(0xffffffffu, sum, o); if (lane >= o) sum += y; }
            sG[warp][2 * lane] = sum - G[1];
            sG[warp][2 * lane + 1] = sum;
        }
    };
    ask_gates(0);
    // the rows, scaled by powers of two: eight lanes a row
    const int sub = lane & 7;
    uint4 raw[ESZ == 2 && OUT ? 8 : 4][W];
    auto ask = [&](int i, bool isq) {                        // .. of the warp's 16, every fourth
        const int r = warp * 16 + i * 4 + (lane >> 3);
        const u8* p = (isq ? a.q + (row0 + r) * a.q_stride : a.k + (row0 + r) * a.k_stride) + (size_t)(kx * D + sub * E) * ESZ;
        uint4* to = raw[(ESZ == 2 && isq ? 4 : 0) + i];
#pragma unroll
        for (int x = 0; x < W; x++) to[x] = r < n ? __ldcg((const uint4*)p + x) : make_uint4(0, 0, 0, 0);
    };
    auto keep = [&](int i, bool isq) {
        const int r = warp * 16 + i * 4 + (lane >> 3);
        float f[E];
        dl_unpack<TYPE, E>((const u32*)raw[(ESZ == 2 && isq ? 4 : 0) + i], f);
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
    };
#pragma unroll
    for (int i = 0; i < 4; i++) ask(i, false);
    if (OUT && ESZ == 2)
#pragma unroll
        for (int i = 0; i < 4; i++) ask(i, true);
    sum_gates(0);
#pragma unroll
    for (int i = 0; i < 4; i++) keep(i, false);
    if (OUT) {
        if (ESZ == 4)
#pragma unroll
            for (int i = 0; i < 4; i++) ask(i, true);
#pragma unroll
        for (int i = 0; i < 4; i++) keep(i, true);
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
    const int half = warp >> 1, part = warp & 1;             // the pair's value head whose inverse the warp works on, with one more warp
#pragma unroll 1
    for (int v0 = 0; v0 < ratio; v0 += 2) {
        const int heads = min(2, ratio - v0);
        // the exponentials that rows of different blocks share
        {
            const int i = tid >> 6, r = tid & 63;
            if (i < heads) {
                sE[i][r] = expf((float)(sG[i][r] - sG[i][r & ~15]));
#pragma unroll
                for (int b = 1; b < 4; b++) if (r < 16 * b) sB[i][b][r] = expf((float)(sG[i][16 * b] - sG[i][r])) * sRk[r];
            }
        }
        if (v0 + 2 < ratio) ask_gates(v0 + 2);
        __syncthreads();                                     // (and nobody needs the rows in shared memory any more)
        // A into shared memory - below the diagonal's blocks as the products take it, those by columns -, P as it is taken
#pragma unroll 1
        for (int i = 0; i < heads; i++) {
            u8* const af = sm + i * P::HEAD;
            float* const dg = (float*)(af + P::AF) + warp * 16 * DL_DS;
            u8* const hp = mine + (size_t)a.kh * C::ROWS + (size_t)head(v0 + i) * C::HEAD;
            float ra[2];
#pragma unroll
            for (int u = 0; u < 2; u++) {
                const int r = 16 * warp + g + 8 * u;
                ra[u] = sBeta[i][r] * sRk[r];
            }
#pragma unroll
            for (int m = 0; m < 8; m++)
                if (m <= 2 * warp + 1) {
                    const bool own = m >= 2 * warp;          // on the diagonal
                    float x[4], p[4];
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const int u = e >> 1, r = 16 * warp + g + 8 * u, j = 8 * m + 2 * t + (e & 1);
                        float f;
                        if (own) f = j <= r ? expf((float)(sG[i][r] - sG[i][j])) * sRk[j] : 0.f;
                        else f = sE[i][r] * sB[i][warp][j];
                        x[e] = ra[u] * f * kk[m][e];
                        p[e] = f * qk[m][e];
                        if (own && j > r) p[e] = 0.f;        // (whatever the product there is)
                        if (own) dg[(j & 15) * DL_DS + (r & 15)] = x[e];
                    }
#pragma unroll
                    for (int u = 0; u < 2; u++) {            // rows 8 (2 warp + u) + g: number m & 1 of the tile m / 2
                        u32 hi, lo;
                        if (!own) {
                            dl_split(x[2 * u], x[2 * u + 1], hi, lo);
                            u32* const at = (u32*)af + ((warp * (warp - 1) + u * warp + m / 2) * 32 + lane) * 2 + (m & 1);
                            *at = hi;
                            *(at + P::AF / 8) = lo;
                        }
                        if (OUT) {
                            dl_split(p[2 * u], p[2 * u + 1], hi, lo);
                            u32* const at = (u32*)(hp + C::HA) + ((dl_tile(2 * warp + u) + m / 2) * 32 + lane) * 2 + (m & 1);
                            *at = hi;
                            *(at + DL_FRAG / 4) = lo;
                        }
                    }
                }
        }
        __syncthreads();
        // the blocks on the diagonal: column `col` of (I + A)^-1 a lane, its elements from the top down, each one taken from those below it as soon as it is known
        {
            const int i = tid >> 6, b = (tid >> 4) & 3, col = tid & 15;
            float* const dg = (float*)(sm + i * P::HEAD + P::AF) + b * 16 * DL_DS;
            float x[16];
            if (i < heads) {
#pragma unroll
                for (int r = 0; r < 16; r++) x[r] = r == col ? 1.f : 0.f;
#pragma unroll
                for (int m = 0; m < 15; m++)
#pragma unroll
                    for (int r4 = (m + 1) & ~3; r4 < 16; r4 += 4) {
                        const float4 w = *(const float4*)(dg + m * DL_DS + r4);
                        const float wa[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                        for (int e = 0; e < 4; e++) if (r4 + e > m) x[r4 + e] = fmaf(-wa[e], x[m], x[r4 + e]);
                    }
            }
            __syncwarp();                                    // (a block is 16 lanes' of one warp)
            if (i < heads)
#pragma unroll
                for (int r = 0; r < 16; r++) dg[r * DL_DS + col] = x[r];      // by rows now
        }
        __syncthreads();
        if (half < heads) {
            const u8* const af = sm + half * P::HEAD;
            const float* const dg = (const float*)(af + P::AF);
            u8* const hp = mine + (size_t)a.kh * C::ROWS + (size_t)head(v0 + half) * C::HEAD;
            uint2* const th = (uint2*)hp;
            uint2* const tl = (uint2*)(hp + DL_FRAG);
            // T of the blocks on the diagonal: two blocks a warp
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const int b = 2 * part + (k >> 1), m = 2 * b + (k & 1);
                const float* w = dg + b * 16 * DL_DS + (8 * (k & 1) + g) * DL_DS + 2 * t;
                uint2 hi, lo;
                dl_split(w[0], w[1], hi.x, lo.x);
                dl_split(w[8], w[9], hi.y, lo.y);
                th[(dl_tile(m) + b) * 32 + lane] = hi;
                tl[(dl_tile(m) + b) * 32 + lane] = lo;
            }
            // the columns of blocks below them: the first, or the second and third
#pragma unroll
            for (int b = 0; b < 3; b++)
                if ((b > 0) == (part == 1)) {
                    u32 xh[3][4], xl[3][4];                  // X_cb^T, c = b ..
                    {
                        const float* w = dg + b * 16 * DL_DS + 2 * t * DL_DS + g;
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            const float* y = w + (e >> 1) * 8 * DL_DS + (e & 1) * 8;
                            dl_split(y[0], y[DL_DS], xh[0][e], xl[0][e]);
                        }
                    }
#pragma unroll
                    for (int ab = b + 1; ab < 4; ab++) {
                        float y[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}}, z[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
                        for (int cb = b; cb < ab; cb++)
#pragma unroll
                            for (int u = 0; u < 2; u++) {
                                const uint2* at = (const uint2*)af + (ab * (ab - 1) + u * ab + cb) * 32 + lane;
                                const uint2 wh = at[0], wl = at[P::AF / 16];
                                dl_mma(y[u], xh[cb - b], wh.x, wh.y);
                                dl_mma(y[u], xl[cb - b], wh.x, wh.y);
                                dl_mma(y[u], xh[cb - b], wl.x, wl.y);
                            }
                        u32 yh[4], yl[4];
#pragma unroll
                        for (int e = 0; e < 4; e++) dl_split(y[e >> 1][2 * (e & 1)], y[e >> 1][2 * (e & 1) + 1], yh[e], yl[e]);
#pragma unroll
                        for (int u = 0; u < 2; u++) {
                            const float* w = dg + ab * 16 * DL_DS + (8 * u + g) * DL_DS + 2 * t;
                            u32 wh[2], wl[2];
                            dl_split(w[0], w[1], wh[0], wl[0]);
                            dl_split(w[8], w[9], wh[1], wl[1]);
                            dl_mma(z[u], yh, wh[0], wh[1]);
                            dl_mma(z[u], yl, wh[0], wh[1]);
                            dl_mma(z[u], yh, wl[0], wl[1]);
                        }
                        if (ab < 3)
#pragma unroll
                            for (int e = 0; e < 4; e++) dl_split(-z[e >> 1][2 * (e & 1)], -z[e >> 1][2 * (e & 1) + 1], xh[ab - b][e], xl[ab - b][e]);
#pragma unroll
                        for (int u = 0; u < 2; u++) {        // rows 8 (2 ab + u) .., columns 16 b ..: turned around
                            u32 h0, l0, h1, l1;
                            dl_split(-z[u][0], -z[u][1], h0, l0);
                            dl_split(-z[u][2], -z[u][3], h1, l1);
                            const int at = (dl_tile(2 * ab + u) + b) * 32 + lane;
                            th[at] = make_uint2(dl_turn(h0), dl_turn(h1));
                            tl[at] = make_uint2(dl_turn(l0), dl_turn(l1));
                        }
                    }
                }
            DlScalars* const sc = (DlScalars*)(hp + 2 * DL_FRAG);
            const int r = 32 * part + lane;
            const double G = sG[half][r], GC = sG[half][CK - 1];
            const float eg = expf((float)G);
            sc->gr[r] = -sBeta[half][r] * (eg * sRk[r]);
            sc->beta[r] = sBeta[half][r];
            if (OUT) { ((float*)(hp + C::HEAD))[r - 2 * CK] = eg * sRq[r]; ((float*)(hp + C::HEAD))[r - CK] = sRq[r]; }
            const float wj = expf((float)(GC - G)) * sRk[r], wo = expf((float)(GC - sG[half][r ^ 32])) * sRk[r ^ 32];
            const int top = (int)(__reduce_max_sync(0xffffffffu, __float_as_uint(fmaxf(wj, wo))) >> 23);
            const int ex = top == 0 || top == 255 ? 0 : max(-100, min(0, top - 126));      // (below 1: a change times it is below 2^15)
            sc->wj[r] = wj * dl_pow2(-ex);
            if (r == 0) sc->ex = ex;
            if (r == 0) sc->gc = expf((float)GC);
        }
        if (v0 + 2 < ratio) {
            __syncthreads();                                 // (the next pair's gates take these' place)
            sum_gates(v0 + 2);
            __syncthreads();
        }
    }
}

// ---- the chain over a sequence's chunks --------------------------------------------------------------------------------------------------------
// A block has four kinds of warps, which meet at mbarriers only: NC of the chain (16 value dimensions and 64 key dimensions each); two or four for the outputs of every 16
// dimensions, which take S and D as the chain's products had them (f16, from shared memory); one that copies the chunks' operands into two rings; and one for the
// outputs' norms.  The blocks of a head form a cluster: a row's sums of squares go to all of them, and a chunk's outputs leave while the next one's are made.
// (The releases that this takes wait for every store of their thread, 1,300 cycles a chunk where the outputs' warps made them.)
template <int D, int TYPE, int NG, bool OUT> struct DlMain {
    using C = DlChunk<D, TYPE>;
    static constexpr int ESZ = DlIo<TYPE>::ESZ, NQ = D / 64, NC = NG * NQ, CS = D / 16 / NG;      // warps on one 16 dimensions; of the chain; blocks of a head
    // warps on the outputs of 16 dimensions, which share the rows: with two of them a chunk's outputs take longer than the chain's part at 128 dimensions (4,093 rows of bf16 259 us, with four
    // 221; of f32, whose rings have room for one chunk only, 387 and 397); and of copies, of norms
    static constexpr int NO = !OUT ? 0 : D == 128 && TYPE != SZ_TYPE_F32 ? 4 : 2, NS = OUT ? NO : 1, NTH = 32 * (NC + NG * NO + (OUT ? 2 : 1));
    static constexpr bool STAGED = TYPE != SZ_TYPE_F32;                                    // gates and outputs through shared memory (f32: whole sectors a warp without)
    static constexpr int VS = 16 * NG * ESZ + 16;                                          // bytes between rows of v and z in shared memory
    // a chunk's operands in two rings, of the chain (k, T, scalars, v) and of the outputs (q, P, e^G, z), each as deep as there is room
    static constexpr int A = C::ROWS / 2 + C::HA + CK * VS, B = OUT ? C::ROWS / 2 + C::HB + (STAGED ? CK * VS : 0) : 0;
    static constexpr int SA = D == 128 ? (TYPE == SZ_TYPE_F32 ? 1 : 2) : (TYPE == SZ_TYPE_F32 ? 2 : 3), SB = D == 128 && TYPE == SZ_TYPE_F32 ? 1 : 2;
    static constexpr int XB = NQ == 2 ? (8 + 4) * 32 * 16 : 0;                             // what a chain's warp gives its partner: its part of K S, half of D
    static constexpr int FB = OUT ? 2 * 4 * 32 * 16 : 0;                                   // a product's factor of 16 x 64 in two f16 numbers: S of a warp, D of a group; two turns of each
    static constexpr int OS = 16 * ESZ + 16, OB = OUT && STAGED ? CK / NS * OS : 0;        // a warp's outputs on their way
    static constexpr int SSQ = OUT ? 2 * (NG + CS + 1) * CK * 4 : 0;                       // a row's sums of squares and its norm's factor, two turns: [group], [block], the factor
    static constexpr int BARS = 2 * SA + 2 * SB + 6 * NG + 6;
    static constexpr size_t SMEM = (size_t)SA * A + (size_t)SB * B + NC * (XB + 2 * FB) + NG * (2 * FB + NO * OB) + SSQ + BARS * 8 + 2 * (NC + NG) * 4;
};

template <int D, int TYPE, int NG, bool OUT>
__global__ void __launch_bounds__(DlMain<D, TYPE, NG, OUT>::NTH, 1)
sz_delta_chunk_kernel(const DlBatch d, const DlRule a, int idx0, int idx1, const u8* __restrict__ scratch, long long one) {
    using M = DlMain<D, TYPE, NG, OUT>;
    using C = DlChunk<D, TYPE>;
    constexpr int ESZ = M::ESZ, NQ = M::NQ, NK = C::NK, NC = M::NC, CS = M::CS, SA = M::SA, SB = M::SB, NO = M::NO, NS = M::NS, OT = 8 / NS;      // OT: 8-row tiles whose outputs a warp finishes
    extern __shared__ __align__(16) u8 sm[];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const int w = warp < NC ? warp : warp - NC, p = warp < NC ? w / NQ : w / NS, q = warp < NC ? w % NQ : w % NS;      // (an output's warp: q is its share of the rows)
    const int h = blockIdx.x / CS, rank = blockIdx.x % CS, kx = a.grouped ? h / (a.vh / a.kh) : h % a.kh;
    u8* const rb = sm + SA * M::A;
    u8* const xb = rb + SB * M::B;
    uint4* const sf = (uint4*)(xb + NC * M::XB);                          // [turn][chain's warp][number][16 key dimensions][lane]
    uint4* const df = (uint4*)((u8*)sf + NC * 2 * M::FB);                 // [turn][group][number][16 rows][lane]
    u8* const ob = (u8*)df + NG * 2 * M::FB + w * M::OB;
    float* const ssq = (float*)((u8*)df + NG * (2 * M::FB + NO * M::OB));
    u64* const bars = (u64*)((u8*)ssq + M::SSQ);
    u64 *const fulla = bars, *const emptya = fulla + SA, *const fullb = emptya + SA, *const emptyb = fullb + SB, *const s_there = emptyb + SB, *const d_there = s_there + 2 * NG,
        *const s_free = d_there + 2 * NG, *const sums_there = s_free + 2 * NG, *const all_there = sums_there + 2, *const factor_there = all_there + 2;
    float *const all = ssq + 2 * NG * CK, *const factor = all + 2 * CS * CK;
    float* const s_unit = (float*)(bars + M::BARS);                       // [turn][chain's warp], then [turn][group]: what a unit of S, of D is
    float* const d_unit = s_unit + 2 * NC;
    const bool norm = OUT && a.norm != nullptr, joined = norm && CS > 1;
    if (tid == 0) {
        for (int i = 0; i < SA; i++) { sz_mbar_init(&fulla[i], 1 + 32); sz_mbar_init(&emptya[i], NC); }
        if (OUT) {
            for (int i = 0; i < SB; i++) { sz_mbar_init(&fullb[i], 1 + 32); sz_mbar_init(&emptyb[i], NG * NO); }
            for (int i = 0; i < 2 * NG; i++) { sz_mbar_init(&s_there[i], NQ); sz_mbar_init(&d_there[i], NQ); sz_mbar_init(&s_free[i], NO); }
            for (int i = 0; i < 2; i++) { sz_mbar_init(&sums_there[i], NG * NO); sz_mbar_init(&all_there[i], CS); sz_mbar_init(&factor_there[i], 1); }
        }
        sz_mbar_fence_init();
    }
    sz_pdl_wait();
    sz_pdl_trigger();
    const DlLong lg = dl_find(d, a.least, blockIdx.y, 0, lane);
    if (lg.b < 0) return;                                                 // (the blocks of a head are all of one sequence: they leave together)
    const DlSeq s = dl_seq(d, lg.b, lane, false);
    const int chunks = (s.n + CK - 1) / CK;
    const int c0 = max(0, idx0 - lg.base), c1 = min(chunks, idx1 - lg.base), nc = max(0, c1 - c0);
    // (a sequence none of whose rows count still moves its state, in the pass that has its first place)
    const bool only = s.on && chunks == 0 && lg.base >= idx0 && lg.base < idx1;
    if (!s.on || (nc == 0 && !only)) return;
    const int dv = (rank * NG + p) * 16;                                  // the warp's value dimensions
    if (joined) sz_cluster_sync(); else __syncthreads();                  // (mbarriers are ready, in all blocks of the head)
    bool dead = false;
    auto wait = [&](u64* bar, int turn) {                                 // (a look first: what is there already costs less than the wait that may sleep)
        u32 ok;
        asm volatile("{ .reg .pred p; mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2; selp.u32 %0, 1, 0, p; }" : "=r"(ok) : "r"(sz_smem_addr(bar)), "r"((u32)turn & 1) : "memory");
        if (__all_sync(0xffffffffu, ok)) return;
        if (!dead && !sz_mbar_wait_warp(bar, turn & 1)) { dead = true; if (lane == 0) atomicOr(d.err, DL_E_WAIT); }
    };
    auto arrive = [&](u64* bar) { __syncwarp(); if (lane == 0) sz_mbar_arrive(bar); };
    // 16 value dimensions of two 8-row tiles m, m + 1 of a tile of rows, transposed: dimensions g, g + 8 of rows 8 m + 2 t, + 1
    auto turned = [&](const u8* tile, int m, float* f) {
        if constexpr (TYPE == SZ_TYPE_F32) {
#pragma unroll
            for (int i = 0; i < 2; i++)
#pragma unroll
                for (int e = 0; e < 4; e++) f[4 * i + e] = *(const float*)(tile + (8 * (m + i) + 2 * t + (e & 1)) * M::VS + (16 * p + g + 8 * (e >> 1)) * 4);
        } else {
            u32 r[4];
            dl_ldsm_t(r, sz_smem_addr(tile + (8 * m + ((lane >> 4) << 3) + (lane & 7)) * M::VS + (16 * p + ((lane >> 3) & 1) * 8) * 2));
            dl_unpack<TYPE, 8>(r, f);
        }
    };
    if (warp == NC + NG * NO) {
        // ---- copies
        if (lane == 0) asm volatile("fence.proxy.async;" ::: "memory");   // (they read what the kernel before has written)
        // (a chunk's operands in two pieces; v and z row by row in 16 bytes a lane: a copy of a row at a time by the TMA engine takes 58 cycles, 7,500 a chunk)
        constexpr int PIECES = NG * ESZ, STEP = 32 / PIECES;              // of 16 bytes, a row's; rows the warp takes at once
        const u32 col = (u32)(h * D + rank * NG * 16) * ESZ + 16 * (lane % PIECES);
        auto tile = [&](u8* at, const u8* src, long long stride, int c) { // 16 NG dimensions of a chunk's rows (those behind the last are zeros, and not read)
            const int n = min(CK, s.n - c * CK);
            const u32 to = sz_smem_addr(at + (lane / PIECES) * M::VS + 16 * (lane % PIECES));
            const size_t row0 = (size_t)s.r0 + (size_t)c * CK;
#pragma unroll 4
            for (int k = 0; k < CK / STEP; k++) {
                const int r = k * STEP + lane / PIECES;
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to + k * STEP * M::VS), "l"(src + (row0 + (r < n ? r : 0)) * stride + col), "r"(r < n ? 16 : 0) : "memory");
            }
        };
        auto both = [&](u8* st, const u8* x, int nx, const u8* y, int ny, u64* full) {
            if (lane == 0) {
                sz_mbar_expect_tx(full, nx + ny);
                sz_bulk_g2s(st, x, nx, full);
                sz_bulk_g2s(st + nx, y, ny, full);
            }
            __syncwarp();
        };
        int na = 0, nb = 0;                                               // chunks asked for (none any more after a wait that ran out)
        auto copy_a = [&](int i) {
            const int slot = i % SA;
            u8* const st = sm + slot * M::A;
            const u8* const src = scratch + (size_t)(lg.base + c0 + i - idx0) * one;
            if (i >= SA) wait(&emptya[slot], i / SA - 1);
            if (dead) return;
            na = i + 1;
            both(st, src + (size_t)kx * C::ROWS, C::ROWS / 2, src + (size_t)a.kh * C::ROWS + (size_t)h * C::HEAD, C::HA, &fulla[slot]);
            tile(st + C::ROWS / 2 + C::HA, a.v, a.v_stride, c0 + i);
            asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(sz_smem_addr(&fulla[slot])) : "memory");
        };
        auto copy_b = [&](int i) {
            const int slot = i % SB;
            u8* const st = rb + slot * M::B;
            const u8* const src = scratch + (size_t)(lg.base + c0 + i - idx0) * one;
            if (i >= SB) wait(&emptyb[slot], i / SB - 1);
            if (dead) return;
            nb = i + 1;
            both(st, src + (size_t)kx * C::ROWS + C::ROWS / 2, C::ROWS / 2, src + (size_t)a.kh * C::ROWS + (size_t)h * C::HEAD + C::HA, C::HB, &fullb[slot]);
            if (M::STAGED && norm) tile(st + C::ROWS / 2 + C::HB, a.z, a.z_stride, c0 + i);
            asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(sz_smem_addr(&fullb[slot])) : "memory");
        };
        // (the chain's a chunk ahead where its ring is the deeper one)
        constexpr int LEAD = SA > SB ? 1 : 0;
        if (LEAD && nc > 0) copy_a(0);
        for (int i = 0; i < nc; i++) {
            if (!LEAD) copy_a(i);
            if (OUT) copy_b(i);
            if (LEAD && i + 1 < nc) copy_a(i + 1);
        }
        // (nothing is under way when the block ends, whoever gave up)
        bool all = true;
        for (int i = max(0, na - SA); i < na; i++) all &= sz_mbar_wait_warp(&fulla[i % SA], (i / SA) & 1);
        for (int i = max(0, nb - SB); i < nb; i++) all &= sz_mbar_wait_warp(&fullb[i % SB], (i / SB) & 1);
        if (!all && lane == 0) atomicOr(d.err, DL_E_WAIT);
        return;
    }
    if (OUT && warp == NC + NG * NO + 1) {
        // ---- the outputs' norms: a row's sums of squares over this block's groups go to all blocks of the head, theirs come here, and what divides the row is
        // ready for the warps that finish it.  Two turns are enough: a warp sends its k-th sums after it has used the k - 2nd factor, and a block its k-th after it has
        // all of the k - 1st, whose senders had read the k - 2nd.
        if (!norm) return;
        for (int k = 0; k < nc; k++) {
            const int turn = k & 1;
            wait(&sums_there[turn], k / 2);
            float2 sum = make_float2(0.f, 0.f);
#pragma unroll
            for (int j = 0; j < NG; j++) { const float2 y = *(const float2*)(ssq + (turn * NG + j) * CK + 2 * lane); sum.x += y.x; sum.y += y.y; }
            if constexpr (CS > 1) {
#pragma unroll
                for (int r = 0; r < CS; r++) {
                    u32 there;
                    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(sz_smem_addr(all + (turn * CS + rank) * CK + 2 * lane)), "r"(r));
                    asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(there), "f"(sum.x), "f"(sum.y) : "memory");
                }
                __syncwarp();
                if (lane < CS) {
                    u32 bar;
                    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(bar) : "r"(sz_smem_addr(&all_there[turn])), "r"(lane));
                    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
                }
                bool there = dead;                                        // (from other blocks' stores: acquired at the cluster's scope)
                for (u32 i = 0; !there && i < 20000000u; i++) {
                    u32 ok;
                    asm volatile("{ .reg .pred p; mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2; selp.u32 %0, 1, 0, p; }" : "=r"(ok) : "r"(sz_smem_addr(&all_there[turn])), "r"((u32)(k / 2) & 1) : "memory");
                    there = ok != 0;
                }
                if (!__all_sync(0xffffffffu, there)) { dead = true; if (lane == 0) atomicOr(d.err, DL_E_WAIT); }
                sum = make_float2(0.f, 0.f);
#pragma unroll
                for (int r = 0; r < CS; r++) { const float2 y = *(const float2*)(all + (turn * CS + r) * CK + 2 * lane); sum.x += y.x; sum.y += y.y; }
            }
            *(float2*)(factor + turn * CK + 2 * lane) = make_float2(rsqrtf(sum.x * (1.f / D) + a.eps), rsqrtf(sum.y * (1.f / D) + a.eps));
            arrive(&factor_there[turn]);
        }
        if (CS > 1) sz_cluster_sync();                                    // (.. with the other blocks' warps of this task: none leaves while another may still write to it, had a wait run out)
        return;
    }
    if (warp < NC) {
        // ---- the chain.  S^T: dimensions g, g + 8; key dimensions 64 q + 8 m + 2 t, + 1
        float S[8][4];
        int es = 0;                                                       // .. in units of 2^es
        {
            const int from = c0 > 0 ? s.to : s.from;
            const float* src = (const float*)(a.state + (size_t)max(from, 0) * a.state_stride) + ((size_t)h * D + 64 * q + 2 * t) * D + dv + g;
#pragma unroll
            for (int m = 0; m < 8; m++)
#pragma unroll
                for (int e = 0; e < 4; e++) S[m][e] = from >= 0 ? src[(size_t)(8 * m + (e & 1)) * D + 8 * (e >> 1)] : 0.f;
        }
        auto exponent = [&](float (*x)[4]) {                              // of the largest of the warp's numbers, and 127
            float mx[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int m = 0; m < 8; m++)
#pragma unroll
                for (int e = 0; e < 4; e++) mx[e] = fmaxf(mx[e], fabsf(x[m][e]));
            return (int)(__reduce_max_sync(0xffffffffu, __float_as_uint(fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])))) >> 23);
        };
#pragma unroll 1
        for (int i = 0; i < nc; i++) {
            const int slot = i % SA, turn = i & 1;
            const u8* const st = sm + slot * M::A;
            const u32 sk = sz_smem_addr(st);
            const u8* const hp = st + C::ROWS / 2;
            const DlScalars* const sc = (const DlScalars*)(hp + 2 * DL_FRAG);
            {                                                             // the state into f16's range
                const int top = exponent(S), ex = top - 127;
                if (top != 0 && top != 255 && (ex > 13 || ex < 4)) {
                    const int up = max(-120, min(120, 10 - ex));
#pragma unroll
                    for (int m = 0; m < 8; m++) dl_scale4(S[m], dl_pow2(up));
                    es -= up;
                }
            }
            if (OUT && i >= 2) wait(&s_free[turn * NG + p], i / 2 - 1);   // (the outputs have taken what lies there)
            wait(&fulla[slot], i / SA);
            // ---- (K S)^T: dimensions x rows.  (Terms one after the other over all rows, so that no product waits for the one before it.)
            float X[8][4];
#pragma unroll
            for (int m = 0; m < 8; m++)
#pragma unroll
                for (int e = 0; e < 4; e++) X[m][e] = 0.f;
#pragma unroll
            for (int ks = 0; ks < 4; ks++) {
                u32 hi[4], lo[4], b[4][4];
                auto load = [&](u32 tile) {
#pragma unroll
                    for (int m = 0; m < 4; m++) dl_ldsm(b[m], tile + dl_at<D>(16 * m + ((lane >> 4) << 3) + (lane & 7), 8 * q + 2 * ks + ((lane >> 3) & 1)));
                };
                auto times = [&](const u32* f) {
#pragma unroll
                    for (int m = 0; m < 8; m++) dl_mma(X[m], f, b[m / 2][2 * (m & 1)], b[m / 2][2 * (m & 1) + 1]);
                };
                load(sk);
#pragma unroll
                for (int e = 0; e < 4; e++) dl_split(S[2 * ks + (e >> 1)][2 * (e & 1)], S[2 * ks + (e >> 1)][2 * (e & 1) + 1], hi[e], lo[e]);
                if (OUT) {
                    sf[(((turn * NC + w) * 2) * 4 + ks) * 32 + lane] = *(uint4*)hi;
                    sf[(((turn * NC + w) * 2 + 1) * 4 + ks) * 32 + lane] = *(uint4*)lo;
                }
                times(hi);
                times(lo);
                if (NK == 2) { load(sk + C::TILE); times(hi); }
            }
            const float true_s = dl_pow2(es);
            if (OUT) { if (lane == 0) s_unit[turn * NC + w] = true_s; arrive(&s_there[turn * NG + p]); }
#pragma unroll
            for (int m = 0; m < 8; m++) dl_scale4(X[m], true_s);
            if constexpr (NQ == 2) {                                      // with the other key dimensions'
                float4* const to = (float4*)(xb + w * M::XB) + lane;
                const float4* const from = (const float4*)(xb + (w ^ 1) * M::XB) + lane;
#pragma unroll
                for (int m = 0; m < 8; m++) to[m * 32] = make_float4(X[m][0], X[m][1], X[m][2], X[m][3]);
                asm volatile("bar.sync %0, 64;" ::"r"(1 + p) : "memory");
#pragma unroll
                for (int m = 0; m < 8; m++) {
                    const float4 y = from[m * 32];
                    X[m][0] += y.x; X[m][1] += y.y; X[m][2] += y.z; X[m][3] += y.w;
                }
            }
            // ---- R = beta (V - e^G K S), in units of 2^ew
#pragma unroll
            for (int m = 0; m < 8; m += 2) {
                float v[8];
                turned(hp + C::HA, m, v);
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    const u64 gr = *(const u64*)(sc->gr + 8 * (m + u) + 2 * t), be = *(const u64*)(sc->beta + 8 * (m + u) + 2 * t);
#pragma unroll
                    for (int e = 0; e < 4; e += 2) {
                        u64 y = dl_mul2(dl_pack2(v[4 * u + e], v[4 * u + e + 1]), be);
                        dl_fma2(y, gr, dl_pack2(X[m + u][e], X[m + u][e + 1]));
                        X[m + u][e] = dl_lo(y); X[m + u][e + 1] = dl_hi(y);
                    }
                }
            }
            int ew = 0, next_es = es;
            {
                const int top = exponent(X);
                if (top != 0 && top != 255) {
                    ew = max(top - 127 - 8, -120);                        // (changes are at most 64 times the largest of R: below 2^15)
                    next_es = max(ew + sc->ex, es - 100);                 // .. and the state's next ones (short keys: the changes times their factors keep their digits)
                }
            }
            u32 rh[4][4], rl[4][4];
            {
                const float f = dl_pow2(-ew);
#pragma unroll
                for (int m = 0; m < 8; m++) dl_scale4(X[m], f);
#pragma unroll
                for (int ks = 0; ks < 4; ks++)
#pragma unroll
                    for (int e = 0; e < 4; e++) dl_split(X[2 * ks + (e >> 1)][2 * (e & 1)], X[2 * ks + (e >> 1)][2 * (e & 1) + 1], rh[ks][e], rl[ks][e]);
            }
            // ---- the rows' changes D^T = R^T T^T: a pair of warps halves the rows
            auto change = [&](float (*x)[4], int tiles, auto tile_of) {
#pragma unroll
                for (int j = 0; j < tiles; j++)
#pragma unroll
                    for (int e = 0; e < 4; e++) x[j][e] = 0.f;
#pragma unroll
                for (int ks = 0; ks < 4; ks++) {
                    uint2 f[8];
#pragma unroll
                    for (int j = 0; j < tiles; j++) if (ks <= tile_of(j) / 2) f[j] = ((const uint2*)hp)[(dl_tile(tile_of(j)) + ks) * 32 + lane];
#pragma unroll
                    for (int j = 0; j < tiles; j++) if (ks <= tile_of(j) / 2) dl_mma(x[j], rh[ks], f[j].x, f[j].y);
#pragma unroll
                    for (int j = 0; j < tiles; j++) if (ks <= tile_of(j) / 2) dl_mma(x[j], rl[ks], f[j].x, f[j].y);
#pragma unroll
                    for (int j = 0; j < tiles; j++) if (ks <= tile_of(j) / 2) f[j] = ((const uint2*)(hp + DL_FRAG))[(dl_tile(tile_of(j)) + ks) * 32 + lane];
#pragma unroll
                    for (int j = 0; j < tiles; j++) if (ks <= tile_of(j) / 2) dl_mma(x[j], rh[ks], f[j].x, f[j].y);
                }
            };
            if constexpr (NQ == 2) {
                float Z[4][4];
                if (q == 0) change(Z, 4, [](int j) { return j < 2 ? j : j + 4; });
                else change(Z, 4, [](int j) { return j + 2; });
                float4* const to = (float4*)(xb + w * M::XB) + 8 * 32 + lane;
                const float4* const from = (const float4*)(xb + (w & ~1) * M::XB) + 8 * 32 + lane;
#pragma unroll
                for (int j = 0; j < 4; j++) to[j * 32] = make_float4(Z[j][0], Z[j][1], Z[j][2], Z[j][3]);
                asm volatile("bar.sync %0, 64;" ::"r"(1 + p) : "memory");
#pragma unroll
                for (int m = 0; m < 8; m++) {
                    const float4 y = from[(m >= 2 && m < 6 ? M::XB / 16 : 0) + (m < 2 ? m : m < 6 ? m - 2 : m - 4) * 32];
                    X[m][0] = y.x; X[m][1] = y.y; X[m][2] = y.z; X[m][3] = y.w;
                }
            } else change(X, 8, [](int j) { return j; });
            if (OUT) {                                                    // for the outputs: half of it a warp
#pragma unroll
                for (int k = 0; k < 4 / NQ; k++) {
                    u32 hi[4], lo[4];
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const int m0 = 2 * k + (e >> 1), m1 = (4 / NQ) * 2 % 8 + m0;      // (of q = 0, of q = 1)
                        const float x0 = NQ == 2 && q ? X[m1][2 * (e & 1)] : X[m0][2 * (e & 1)], x1 = NQ == 2 && q ? X[m1][2 * (e & 1) + 1] : X[m0][2 * (e & 1) + 1];
                        dl_split(x0, x1, hi[e], lo[e]);
                    }
                    df[(((turn * NG + p) * 2) * 4 + q * (4 / NQ) + k) * 32 + lane] = *(uint4*)hi;
                    df[(((turn * NG + p) * 2 + 1) * 4 + q * (4 / NQ) + k) * 32 + lane] = *(uint4*)lo;
                }
                if (lane == 0 && q == 0) d_unit[turn * NG + p] = dl_pow2(ew);
                arrive(&d_there[turn * NG + p]);
            }
            // ---- the state: e^G_C S + K^T (e^(G_C - G_j) D), in units of 2^next_es
            const float unit = dl_pow2(ew + sc->ex - next_es);            // (1 but for a state that is 2^92 times the changes)
#pragma unroll
            for (int m = 0; m < 8; m++) {
                const u64 wj = dl_mul2(*(const u64*)(sc->wj + 8 * m + 2 * t), dl_pack2(unit, unit)), lo = dl_mul2(dl_pack2(X[m][0], X[m][1]), wj), hi = dl_mul2(dl_pack2(X[m][2], X[m][3]), wj);
                X[m][0] = dl_lo(lo); X[m][1] = dl_hi(lo); X[m][2] = dl_lo(hi); X[m][3] = dl_hi(hi);
            }
            const float f = sc->gc * dl_pow2(max(es - next_es, -126));
#pragma unroll
            for (int m = 0; m < 8; m++) dl_scale4(S[m], f);
            es = next_es;
#pragma unroll
            for (int ks = 0; ks < 4; ks++) {
                u32 hi[4], lo[4], b[4][4];
                auto load = [&](u32 tile) {
#pragma unroll
                    for (int m = 0; m < 4; m++) dl_ldsm_t(b[m], tile + dl_at<D>(16 * ks + (((lane >> 3) & 1) << 3) + (lane & 7), 8 * q + 2 * m + (lane >> 4)));
                };
                auto times = [&](const u32* x) {
#pragma unroll
                    for (int m = 0; m < 8; m++) dl_mma(S[m], x, b[m / 2][2 * (m & 1)], b[m / 2][2 * (m & 1) + 1]);
                };
                load(sk);
#pragma unroll
                for (int e = 0; e < 4; e++) dl_split(X[2 * ks + (e >> 1)][2 * (e & 1)], X[2 * ks + (e >> 1)][2 * (e & 1) + 1], hi[e], lo[e]);
                times(hi);
                times(lo);
                if (NK == 2) { load(sk + C::TILE); times(hi); }
            }
            arrive(&emptya[slot]);
        }
        float* to = (float*)(a.state + (size_t)s.to * a.state_stride) + ((size_t)h * D + 64 * q + 2 * t) * D + dv + g;
        const float f0 = dl_pow2(es / 2), f1 = dl_pow2(es - es / 2);      // (in two steps: 2^es alone may be out of range)
#pragma unroll
        for (int m = 0; m < 8; m++)
#pragma unroll
            for (int e = 0; e < 4; e++) to[(size_t)(8 * m + (e & 1)) * D + 8 * (e >> 1)] = S[m][e] * f0 * f1;
        return;
    }
    if constexpr (OUT) {
        // ---- the outputs: e^G Q S + P D, of OT 8-row tiles a warp (of pairs of like work)
        auto mine = [&](int i) { return OT == 2 ? 2 * q + i : q == 0 ? (i < 2 ? i : i + 4) : i + 2; };
        float O[4 * OT];
        float nw[2] = {0.f, 0.f};
        if (norm) { nw[0] = a.norm[dv + g]; nw[1] = a.norm[dv + g + 8]; }
        auto finish = [&](int k) {                                        // of the k-th chunk: their norm's factor, into shared memory by rows, out
            const int c = c0 + k, n = min(CK, s.n - c * CK);
#pragma unroll
            for (int i = 0; i < OT; i++) {
                const int row = 8 * mine(i) + 2 * t;
                if (norm) {
                    const float2 f = *(const float2*)(factor + (k & 1) * CK + row);
                    const float r0 = f.x, r1 = f.y;
                    O[4 * i] *= r0; O[4 * i + 1] *= r1; O[4 * i + 2] *= r0; O[4 * i + 3] *= r1;
                }
                // row 8 i + 2 t (+ 1) of the warp's, dimension g (+ 8)
                if constexpr (!M::STAGED) {
                    u8* const at = a.out + ((size_t)s.r0 + (size_t)c * CK + row) * a.out_stride + (size_t)(h * D + dv + g) * 4;
#pragma unroll
                    for (int e = 0; e < 4; e++) if (row + (e & 1) < n) *(float*)(at + (e & 1) * a.out_stride + 32 * (e >> 1)) = O[4 * i + e];
                } else if (i & 1) {
                    u32 r[4];
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const float* o = O + 4 * (i - 1) + 2 * e;
                        if constexpr (TYPE == SZ_TYPE_F16) r[e] = dl_h2(o[0], o[1]);
                        else { const __nv_bfloat162 b = __floats2bfloat162_rn(o[0], o[1]); r[e] = *(const u32*)&b; }
                    }
                    dl_stsm_t(sz_smem_addr(ob + (8 * (i - 1) + ((lane >> 4) << 3) + (lane & 7)) * M::OS + ((lane >> 3) & 1) * 16), r);
                }
            }
            if (!M::STAGED) return;
            __syncwarp();
            constexpr int PIECES = ESZ;                                   // of 16 bytes, a row's 16 dimensions
#pragma unroll
            for (int i = 0; i < OT * PIECES / 4; i++) {
                const int r = (32 * i + lane) / PIECES, x = (32 * i + lane) % PIECES, row = 8 * mine(r / 8) + r % 8;
                if (row < n) *(uint4*)(a.out + ((size_t)s.r0 + (size_t)c * CK + row) * a.out_stride + (size_t)(h * D + dv) * ESZ + 16 * x) = *(const uint4*)(ob + r * M::OS + 16 * x);
            }
            __syncwarp();
        };
#pragma unroll 1
        for (int k = 0; k < nc; k++) {
            const int slot = k % SB, turn = k & 1;
            const u8* const st = rb + slot * M::B;
            const u32 sq = sz_smem_addr(st);
            const u8* const hp = st + C::ROWS / 2;
            const float* const sc = (const float*)(hp + 2 * DL_FRAG);
            const u8* const zt = hp + C::HB;
            float zd[M::STAGED ? 1 : 4 * OT];                             // (f32: the gates, asked for early)
            if (!M::STAGED && norm) {
                const int n = min(CK, s.n - (c0 + k) * CK);
#pragma unroll
                for (int i = 0; i < OT; i++)
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const int row = 8 * mine(i) + 2 * t + (e & 1);
                        zd[M::STAGED ? 0 : 4 * i + e] = row < n ? *(const float*)(a.z + ((size_t)s.r0 + (size_t)(c0 + k) * CK + row) * a.z_stride + (size_t)(h * D + dv + g + 8 * (e >> 1)) * 4) : 0.f;
                    }
            }
            wait(&fullb[slot], k / SB);
            wait(&s_there[turn * NG + p], k / 2);
            float Y[NQ][OT][4];
#pragma unroll
            for (int j = 0; j < NQ; j++)
#pragma unroll
                for (int i = 0; i < OT; i++)
#pragma unroll
                    for (int e = 0; e < 4; e++) Y[j][i][e] = 0.f;
#pragma unroll
            for (int ks = 0; ks < 4; ks++)
#pragma unroll
                for (int j = 0; j < NQ; j++) {
                    u32 hi[4], lo[4];
                    *(uint4*)hi = sf[(((turn * NC + p * NQ + j) * 2) * 4 + ks) * 32 + lane];
                    *(uint4*)lo = sf[(((turn * NC + p * NQ + j) * 2 + 1) * 4 + ks) * 32 + lane];
#pragma unroll
                    for (int i = 0; i < OT; i += 2) {
                        const u32 at = dl_at<D>(8 * mine(i) + ((lane >> 4) << 3) + (lane & 7), 8 * j + 2 * ks + ((lane >> 3) & 1));
                        u32 b[4];
                        dl_ldsm(b, sq + at);
                        dl_mma(Y[j][i], hi, b[0], b[1]);
                        dl_mma(Y[j][i + 1], hi, b[2], b[3]);
                        dl_mma(Y[j][i], lo, b[0], b[1]);
                        dl_mma(Y[j][i + 1], lo, b[2], b[3]);
                        if (NK == 2) {
                            dl_ldsm(b, sq + C::TILE + at);
                            dl_mma(Y[j][i], hi, b[0], b[1]);
                            dl_mma(Y[j][i + 1], hi, b[2], b[3]);
                        }
                    }
                }
#pragma unroll
            for (int j = 0; j < NQ; j++) {
                const float f = s_unit[turn * NC + p * NQ + j];
#pragma unroll
                for (int i = 0; i < OT; i++)
#pragma unroll
                    for (int e = 0; e < 4; e++) Y[0][i][e] = j == 0 ? Y[0][i][e] * f : fmaf(Y[j][i][e], f, Y[0][i][e]);
            }
            wait(&d_there[turn * NG + p], k / 2);
            float acc[OT][4];
#pragma unroll
            for (int i = 0; i < OT; i++)
#pragma unroll
                for (int e = 0; e < 4; e++) acc[i][e] = 0.f;
#pragma unroll
            for (int ks = 0; ks < 4; ks++) {
                u32 hi[4], lo[4];
                *(uint4*)hi = df[(((turn * NG + p) * 2) * 4 + ks) * 32 + lane];
                *(uint4*)lo = df[(((turn * NG + p) * 2 + 1) * 4 + ks) * 32 + lane];
#pragma unroll
                for (int part = 0; part < 3; part++)                      // high high, low high, high low
#pragma unroll
                    for (int i = 0; i < OT; i++)
                        if (ks <= mine(i) / 2) {
                            const uint2 f = ((const uint2*)(hp + (part == 2 ? 1 : 0) * DL_FRAG))[(dl_tile(mine(i)) + ks) * 32 + lane];
                            dl_mma(acc[i], part == 1 ? lo : hi, f.x, f.y);
                        }
            }
            const float tw = d_unit[turn * NG + p];
            arrive(&s_free[turn * NG + p]);
            float N[4 * OT];
#pragma unroll
            for (int i = 0; i < OT; i++) {
                const float2 gq = *(const float2*)(sc + 8 * mine(i) + 2 * t), rq = *(const float2*)(sc + CK + 8 * mine(i) + 2 * t);
#pragma unroll
                for (int e = 0; e < 4; e++) N[4 * i + e] = fmaf(e & 1 ? gq.y : gq.x, Y[0][i][e], acc[i][e] * ((e & 1 ? rq.y : rq.x) * tw));
            }
            if (norm) {
#pragma unroll
                for (int i = 0; i < OT; i++) {
                    const float* o = N + 4 * i;
                    float s0 = fmaf(o[0], o[0], o[2] * o[2]), s1 = fmaf(o[1], o[1], o[3] * o[3]);
#pragma unroll
                    for (int x = 4; x < 32; x *= 2) { s0 += __shfl_xor_sync(0xffffffffu, s0, x); s1 += __shfl_xor_sync(0xffffffffu, s1, x); }
                    if (g == 0) *(float2*)(ssq + (turn * NG + p) * CK + 8 * mine(i) + 2 * t) = make_float2(s0, s1);
                }
                arrive(&sums_there[turn]);
#pragma unroll
                for (int i = 0; i < OT; i += 2) {
                    float z[8];
                    if constexpr (M::STAGED) turned(zt, mine(i), z);
                    else
#pragma unroll
                        for (int e = 0; e < 8; e++) z[e] = zd[4 * i + e];
#pragma unroll
                    for (int e = 0; e < 8; e++) N[4 * i + e] *= nw[(e >> 1) & 1] * dl_sigmoid<TYPE>(z[e]);
                }
            }
            arrive(&emptyb[slot]);
            if (norm && k > 0) { wait(&factor_there[turn ^ 1], (k - 1) / 2); finish(k - 1); }       // the chunk before
#pragma unroll
            for (int e = 0; e < 4 * OT; e++) O[e] = N[e];
            if (!norm) finish(k);
        }
        if (norm && nc > 0) {
            wait(&factor_there[(nc - 1) & 1], (nc - 1) / 2);
            finish(nc - 1);
        }
    }
}

template <int D, int TYPE, int NG, bool OUT>
int dl_chunk_go(const DlBatch& b, const DlRule& r, int longest, int64_t total, int64_t per, uint64_t scratch, cudaStream_t st) {
    using P = DlPrep<D, TYPE>;
    using M = DlMain<D, TYPE, NG, OUT>;
    static_assert(M::SMEM <= 227 * 1024 && P::SMEM <= 72 * 1024 && sizeof(DlScalars) % 16 == 0, "");
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
    // (where not all chunks fit: the whole slab, whatever a chunk takes, so that no type of rows needs more than f32, whose chunks are the largest)
    return total <= per ? one * total : one * per > DL_SLAB ? one * per : DL_SLAB;
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
