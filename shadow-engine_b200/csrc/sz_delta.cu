// The DeltaNet layer of a served step: sequences whose states and carried rows lie in slots of a pool (sz_delta_conv, sz_delta_rows).  This file has the
// causal convolution, the gated delta rule row by row, and the C ABI; sz_delta_chunk.cu has the rule for many rows.
#include "sz_delta.cuh"

#include <math.h>

namespace {

constexpr int DL_SM = 148;           // multiprocessors (a GPU with another number: other sizes of tiles, the same results)

// ---- the causal convolution --------------------------------------------------------------------------------------------------------------
// y[r][c] = silu(bias[c] + sum_t w[c][t] x[r - (K - 1) + t][c]); rows before a sequence's first are those its slot carries (K - 1, the oldest first).  The taps are
// added in f32 from the oldest on.  A thread has DL_V neighbouring channels and `tile` rows, one after the other, with the window in registers and the next
// DL_AHEAD rows asked for.  The block that has a sequence's first row is the only one that looks at its slot: it does the rows up to the K - 1st, those of the next tile
// among them, and then leaves the new carried rows, which are rows of the call or of the old slot (the place is the same where a sequence goes on in place).  8,192 channels over 4 rows, bf16: 4,093 rows 38 us (134 MB, 20.5 us of them; a row of 4 channels is some 45 instructions, two
// exponentials' pipe a channel among them; with 8 rows ahead 42, in tiles of 16 rows 41), 163 rows of 64 sequences 9.2, one row 3.7, four of one sequence 4.6 (a launch and the chain table,
// slot, carried rows, store).  What a tile reads twice are its first K - 1 rows, from L2.
constexpr int DL_AHEAD = 4, DL_V = 4;
template <int ESZ> struct DlRaw { typedef uint2 T; };
template <> struct DlRaw<4> { typedef uint4 T; };
__device__ __forceinline__ void dl_none(uint2& x) { x = make_uint2(0, 0); }
__device__ __forceinline__ void dl_none(uint4& x) { x = make_uint4(0, 0, 0, 0); }
struct DlConv {
    const u8* x;
    u8* y;
    long long x_stride, y_stride;    // bytes
    const float *w, *bias;
    u8* conv;
    long long conv_stride;
    int conv_type, ch, tile;         // tile 0: a block a sequence
};

// The sequence of row r: the last that begins at or before it (-1: none), found by a warp in steps of 32 entries.
__device__ __forceinline__ int dl_seq_of(const DlBatch& d, int r, int lane) {
    int at = 0, n = d.n_seq + 1;                        // entries at .. at + n of row_start
    while (n > 1) {
        const int step = (n + 31) / 32, i = at + lane * step;
        const bool in = lane * step < n && d.row_start[i] <= r;
        const int c = __popc(__ballot_sync(0xffffffffu, in));
        if (c == 0) return at - 1;
        at += (c - 1) * step;
        n = min(step, d.n_seq + 1 - at);
        if (step == 1) break;
        // (entry `at` itself is at or before r; those behind it up to the next step's are looked at again)
    }
    return at;
}

template <int TYPE, int K>
__global__ void __launch_bounds__(128)
sz_delta_conv_kernel(const DlBatch d, const DlConv a) {
    constexpr int ESZ = DlIo<TYPE>::ESZ, V = DL_V;
    using Raw = typename DlRaw<ESZ>::T;
    const int lane = threadIdx.x & 31, c0 = (blockIdx.x * 128 + threadIdx.x) * V;
    const bool mine = c0 < a.ch;                        // (a warp stays together: its lanes look sequences up together)
    sz_pdl_wait();                                      // (weights and bias, too, may come from the kernel before)
    sz_pdl_trigger();
    const int own = a.tile ? -1 : blockIdx.y;
    const int first = a.tile ? blockIdx.y * a.tile : max(d.row_start[own], 0);
    int end = min(a.tile ? first + a.tile : d.row_start[own + 1], d.rows);
    const u8* const xc = a.x + (size_t)c0 * ESZ;
    auto ask = [&](int r) {                             // row r (x is not written meanwhile: y lies elsewhere)
        Raw q;
        dl_none(q);
        if (mine && r < end) q = __ldcg((const Raw*)(xc + (size_t)r * a.x_stride));
        return q;
    };
    auto pairs = [&](const Raw& q, u64* f) {
        float x[V];
        dl_unpack<TYPE, V>((const u32*)&q, x);
#pragma unroll
        for (int i = 0; i < V / 2; i++) f[i] = dl_pack2(x[2 * i], x[2 * i + 1]);
    };
    auto carried = [&](int slot, int i, u64* f) {       // row i of a slot
        const u8* p = a.conv + (size_t)slot * a.conv_stride;
        float x[V];
        if (a.conv_type == SZ_TYPE_F32) dl_load<SZ_TYPE_F32, V>(p + ((size_t)i * a.ch + c0) * 4, x);
        else if (a.conv_type == SZ_TYPE_F16) dl_load<SZ_TYPE_F16, V>(p + ((size_t)i * a.ch + c0) * 2, x);
        else dl_load<SZ_TYPE_BF16, V>(p + ((size_t)i * a.ch + c0) * 2, x);
#pragma unroll
        for (int e = 0; e < V / 2; e++) f[e] = dl_pack2(x[2 * e], x[2 * e + 1]);
    };
    Raw ahead[DL_AHEAD];
#pragma unroll
    for (int j = 0; j < DL_AHEAD; j++) ahead[j] = ask(first + j);
    u64 w[K][V / 2], bias[V / 2];
#pragma unroll
    for (int i = 0; i < V / 2; i++) bias[i] = 0;
    if (mine) {
        float wt[K * V];
        const float4* src = (const float4*)(a.w + (size_t)c0 * K);
#pragma unroll
        for (int i = 0; i < K * V / 4; i++) *(float4*)(wt + 4 * i) = src[i];
#pragma unroll
        for (int i = 0; i < V / 2; i++)
#pragma unroll
            for (int t = 0; t < K; t++) w[t][i] = dl_pack2(wt[2 * i * K + t], wt[(2 * i + 1) * K + t]);
        if (a.bias)
#pragma unroll
            for (int i = 0; i < V / 2; i++) { const float2 x = *(const float2*)(a.bias + c0 + 2 * i); bias[i] = dl_pack2(x.x, x.y); }
    }
    u64 win[K][V / 2];                                  // the rows before the next one, and it
    int b = own, from = first, upto = first;            // the current sequence's rows here: from .. upto
    int next = first;                                   // where the one behind it begins
    auto give = [&](int r, const u64 (*x)[V / 2]) {     // row r, of K rows
        float y[V];
#pragma unroll
        for (int i = 0; i < V / 2; i++) {
            u64 acc = bias[i];
#pragma unroll
            for (int t = 0; t < K; t++) dl_fma2(acc, w[t][i], x[t][i]);
            y[2 * i] = dl_lo(acc) * dl_sigmoid<TYPE>(dl_lo(acc));
            y[2 * i + 1] = dl_hi(acc) * dl_sigmoid<TYPE>(dl_hi(acc));
        }
        dl_store<TYPE, V>(a.y + (size_t)r * a.y_stride + (size_t)c0 * ESZ, y);
    };
    int r = first;
#pragma unroll 1
    while (r < end) {
        if (r >= from && r < next && r + DL_AHEAD <= min(upto, end)) {      // DL_AHEAD rows of the current sequence
            if (mine) {
                u64 x[K - 1 + DL_AHEAD][V / 2];
#pragma unroll
                for (int t = 0; t < K - 1; t++)
#pragma unroll
                    for (int i = 0; i < V / 2; i++) x[t][i] = win[t][i];
#pragma unroll
                for (int j = 0; j < DL_AHEAD; j++) pairs(ahead[j], x[K - 1 + j]);
#pragma unroll
                for (int j = 0; j < DL_AHEAD; j++) ahead[j] = ask(r + DL_AHEAD + j);
#pragma unroll
                for (int j = 0; j < DL_AHEAD; j++) give(r + j, x + j);
#pragma unroll
                for (int t = 0; t < K - 1; t++)
#pragma unroll
                    for (int i = 0; i < V / 2; i++) win[t][i] = x[t + DL_AHEAD][i];
            }
            r += DL_AHEAD;
            continue;
        }
        const Raw now = ahead[0];
#pragma unroll
        for (int j = 0; j + 1 < DL_AHEAD; j++) ahead[j] = ahead[j + 1];
        ahead[DL_AHEAD - 1] = ask(r + DL_AHEAD);
        if (r >= next) {                            // another sequence
            b = b < 0 && d.n_seq > 1 ? dl_seq_of(d, r, lane) : max(b, 0);
            while (b >= 0 && b < d.n_seq && d.row_start[b + 1] <= r && d.row_start[b + 1] >= d.row_start[b]) b++;
            from = upto = 0;
            if (b >= d.n_seq) next = end;           // (rows behind the last sequence)
            else if (b < 0) { b = -1; next = max(r + 1, d.row_start[0]); }
            else if (d.row_start[b] > r) next = d.row_start[b];      // (rows before the first sequence)
            else {
                const int nb = d.row_start[b + 1];
                next = nb > r ? nb : end;           // (a descending table: reported, and nobody's rows)
                const DlSeq s = dl_seq(d, b, lane, blockIdx.x == 0);
                if (s.on) {
                    // (a tile that begins inside a sequence: from its K - 1st row on, the others are the block's that has its first)
                    from = r == s.r0 ? r : max(r, s.r0 + K - 1);
                    upto = s.r0 + s.n;
                    if (r == s.r0 && min(upto, r + K - 1) > end) {
                        const int was = end;
                        end = min(upto, r + K - 1);
#pragma unroll
                        for (int j = 0; j < DL_AHEAD; j++) if (r + 1 + j >= was) ahead[j] = ask(r + 1 + j);
                    }
                    if (mine && (from < upto || r == s.r0)) {
                        // the rows before `from`: of the sequence, of its slot, or zeros
#pragma unroll
                        for (int t = 0; t < K - 1; t++) {
                            const int p = from - (K - 1) + t - s.r0; // row p of the sequence
                            if (p >= 0) { const Raw q = __ldcg((const Raw*)(xc + (size_t)(s.r0 + p) * a.x_stride)); pairs(q, win[t]); }
                            else if (s.from >= 0) carried(s.from, K - 1 + p, win[t]);      // (r is the first row)
                            else
#pragma unroll
                                for (int i = 0; i < V / 2; i++) win[t][i] = 0;
                        }
                        if (r == s.r0) {            // what is carried on: rows n - (K - 1) .. n of [the slot's rows; the sequence's]
                            u8* p = a.conv + (size_t)s.to * a.conv_stride;
#pragma unroll
                            for (int t = 0; t < K - 1; t++) {
                                const int at = s.n - (K - 1) + t;       // (below 0: row n + t of the slot)
                                u64 nw[V / 2];
                                if (at >= 0) { const Raw q = __ldcg((const Raw*)(xc + (size_t)(s.r0 + at) * a.x_stride)); pairs(q, nw); }
                                else if (s.from >= 0) carried(s.from, s.n + t, nw);      // (rows below t alone are overwritten by now)
                                else
#pragma unroll
                                    for (int i = 0; i < V / 2; i++) nw[i] = 0;
                                float f[V];
#pragma unroll
                                for (int i = 0; i < V / 2; i++) { f[2 * i] = dl_lo(nw[i]); f[2 * i + 1] = dl_hi(nw[i]); }
                                if (a.conv_type == SZ_TYPE_F32) dl_store<SZ_TYPE_F32, V>(p + ((size_t)t * a.ch + c0) * 4, f);
                                else if (a.conv_type == SZ_TYPE_F16) dl_store<SZ_TYPE_F16, V>(p + ((size_t)t * a.ch + c0) * 2, f);
                                else dl_store<SZ_TYPE_BF16, V>(p + ((size_t)t * a.ch + c0) * 2, f);
                            }
                        }
                    }
                }
            }
        }
        if (r >= from && r < upto && mine) {
            pairs(now, win[K - 1]);
            give(r, win);
#pragma unroll
            for (int t = 0; t < K - 1; t++)
#pragma unroll
                for (int i = 0; i < V / 2; i++) win[t][i] = win[t + 1][i];
        }
        r++;
    }
    if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x < 32) {       // (tables that no row leads to)
        bool bad = false;
        for (int i = lane; i < d.n_seq; i += 32) bad |= d.row_start[i] < 0 || d.row_start[i + 1] < d.row_start[i] || d.row_start[i + 1] > d.rows;
        if (__any_sync(0xffffffffu, bad) && lane == 0) atomicOr(d.err, DL_E_ROWS);
    }
}

// ---- the gated delta rule, row by row ------------------------------------------------------------------------------------------------------
// S (f32 [key dimension][value dimension]) of a sequence and value head stays in the registers of a block while its rows go by: a warp has 16 value
// dimensions and all key dimensions, a lane 4 and D / 8 of them.  With the row's k and q normed, g its decay and S the state before it:
//   x = g S^T k,  d = beta (v - x),  S = g S + k d^T,  o = S^T q = g S^T q + (k.q) d
// so that both sums over the key dimensions (x and S^T q) go through the lanes' exchange together.  Products are packed pairs of neighbouring key dimensions.
// Rows come in sets of DL_SET: a warp norms one of them for the block (shared memory), and norms and gates its outputs.  With many
// sequences the states' bytes bound it (64 sequences of 32 heads of 128, 163 rows of bf16: 274 MB, 41.9 us of 59; 32 of f32 without outputs 20.9 of 31.7), with few the
// chain load - exchange - store (one row 4.8 us).  The operands are asked for before the state (after it: 74 us).
constexpr int DL_SET = 8;
template <int D> struct DlSet {
    float k[DL_SET][D], q[DL_SET][D], v[DL_SET][D], o[DL_SET][D];
    float g[DL_SET], beta[DL_SET], kq[DL_SET];
};

template <int D, int TYPE, bool OUT>
__global__ void __launch_bounds__(D * 2, D == 128 ? 2 : 4)
sz_delta_rows_kernel(const DlBatch d, const DlRule a) {
    constexpr int ESZ = DlIo<TYPE>::ESZ, NW = D / 16, M = D / 8, E = D / 32;      // warps; key dimensions a lane; elements of a row a lane
    __shared__ __align__(16) DlSet<D> sh;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, h = blockIdx.x, b = blockIdx.y;
    sz_pdl_wait();
    sz_pdl_trigger();
    const DlSeq s = dl_seq(d, b, lane, h == 0 && warp == 0);
    if (!s.on || (a.least && d.row_start[b + 1] - d.row_start[b] >= a.least)) return;
    const int kx = a.grouped ? h / (a.vh / a.kh) : h % a.kh;
    const int j0 = 16 * warp + 4 * (lane & 3), i0 = M * (lane >> 2);              // the lane's value and key dimensions
    // a set's rows, R a warp: asked for (the first ones before the state), then normed into shared memory
    constexpr int R = DL_SET / NW, W = E * ESZ / 4;
    u32 kw[R][W], qw[R][W], vw[R][W], zw[R][W];
    float al[R], be[R];
    const float ah = a.a[h], dth = a.dt[h];
    auto raw = [&](const u8* p, u32* w) {
        if constexpr (W == 4) *(uint4*)w = __ldcg((const uint4*)p);
        else if constexpr (W == 2) *(uint2*)w = __ldcg((const uint2*)p);
        else w[0] = __ldcg((const u32*)p);
    };
    auto ask = [&](int r0) {
#pragma unroll
        for (int i = 0; i < R; i++) {
            const int j = warp + i * NW;
            if (r0 + j >= s.n) continue;
            const size_t r = s.r0 + r0 + j;
            raw(a.k + r * a.k_stride + (size_t)(kx * D + lane * E) * ESZ, kw[i]);
            if (OUT) raw(a.q + r * a.q_stride + (size_t)(kx * D + lane * E) * ESZ, qw[i]);
            raw(a.v + r * a.v_stride + (size_t)(h * D + lane * E) * ESZ, vw[i]);
            if (OUT && a.norm) raw(a.z + r * a.z_stride + (size_t)(h * D + lane * E) * ESZ, zw[i]);
            al[i] = dl_load1<TYPE>(a.alpha + r * a.alpha_stride + (size_t)h * ESZ);
            be[i] = dl_load1<TYPE>(a.beta + r * a.beta_stride + (size_t)h * ESZ);
        }
    };
    ask(0);
    u64 S[M / 2][4];
    if (s.from >= 0) {
        const float* p = (const float*)(a.state + (size_t)s.from * a.state_stride) + ((size_t)h * D + i0) * D + j0;
#pragma unroll
        for (int m = 0; m < M / 2; m++) {
            const float4 e = __ldcg((const float4*)(p + (size_t)(2 * m) * D)), o = __ldcg((const float4*)(p + (size_t)(2 * m + 1) * D));
            S[m][0] = dl_pack2(e.x, o.x); S[m][1] = dl_pack2(e.y, o.y); S[m][2] = dl_pack2(e.z, o.z); S[m][3] = dl_pack2(e.w, o.w);
        }
    } else {
#pragma unroll
        for (int m = 0; m < M / 2; m++)
#pragma unroll
            for (int c = 0; c < 4; c++) S[m][c] = 0;
    }
    for (int r0 = 0; r0 < s.n; r0 += DL_SET) {
        const int nr = min(DL_SET, s.n - r0);
#pragma unroll
        for (int i = 0; i < R; i++) {
            const int j = warp + i * NW;
            if (j >= nr) continue;
            float kv[E], qv[E], vv[E], kk = 0.f, qq = 0.f, kq = 0.f;
            dl_unpack<TYPE, E>(kw[i], kv);
            if (OUT) dl_unpack<TYPE, E>(qw[i], qv);
            dl_unpack<TYPE, E>(vw[i], vv);
#pragma unroll
            for (int e = 0; e < E; e++) {
                kk = fmaf(kv[e], kv[e], kk);
                if (OUT) { qq = fmaf(qv[e], qv[e], qq); kq = fmaf(kv[e], qv[e], kq); }
                sh.v[j][lane * E + e] = vv[e];
            }
            kk = sz_warp_sum(kk);
            const float nk = (float)sz_rsqrt64((double)kk + 1e-6);
#pragma unroll
            for (int e = 0; e < E; e++) sh.k[j][lane * E + e] = kv[e] * nk;
            if (OUT) {
                qq = sz_warp_sum(qq);
                kq = sz_warp_sum(kq);
                const float nq = (float)sz_rsqrt64((double)qq + 1e-6) * a.q_scale;
#pragma unroll
                for (int e = 0; e < E; e++) sh.q[j][lane * E + e] = qv[e] * nq;
                if (lane == 0) sh.kq[j] = kq * nk * nq;
            }
            if (lane == 0) { sh.g[j] = expf(dl_log_decay(al[i], ah, dth)); sh.beta[j] = sz_sigmoid(be[i]); }
        }
        __syncthreads();
        for (int j = 0; j < nr; j++) {
            const float4 v4 = *(const float4*)(sh.v[j] + j0);
            const float v[4] = {v4.x, v4.y, v4.z, v4.w};
            const float g = sh.g[j], beta = sh.beta[j];
            const u64 g2 = dl_pack2(g, g);
            u64 x[4] = {0, 0, 0, 0}, y[4] = {0, 0, 0, 0}, kr[M / 2];
#pragma unroll
            for (int m = 0; m < M / 4; m++) {
                const ulonglong2 kp = *(const ulonglong2*)(sh.k[j] + i0 + 4 * m);
                kr[2 * m] = kp.x; kr[2 * m + 1] = kp.y;
                ulonglong2 qp = {0, 0};
                if (OUT) qp = *(const ulonglong2*)(sh.q[j] + i0 + 4 * m);
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    S[2 * m][c] = dl_mul2(S[2 * m][c], g2); S[2 * m + 1][c] = dl_mul2(S[2 * m + 1][c], g2);
                    dl_fma2(x[c], S[2 * m][c], kp.x); dl_fma2(x[c], S[2 * m + 1][c], kp.y);
                    if (OUT) { dl_fma2(y[c], S[2 * m][c], qp.x); dl_fma2(y[c], S[2 * m + 1][c], qp.y); }
                }
            }
            float xs[4], ys[4];
#pragma unroll
            for (int c = 0; c < 4; c++) { xs[c] = dl_lo(x[c]) + dl_hi(x[c]); ys[c] = dl_lo(y[c]) + dl_hi(y[c]); }
#pragma unroll
            for (int o = 4; o < 32; o *= 2)
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    xs[c] += __shfl_xor_sync(0xffffffffu, xs[c], o);
                    if (OUT) ys[c] += __shfl_xor_sync(0xffffffffu, ys[c], o);
                }
            float dl[4];
#pragma unroll
            for (int c = 0; c < 4; c++) {
                dl[c] = (v[c] - xs[c]) * beta;
                const u64 d2 = dl_pack2(dl[c], dl[c]);
#pragma unroll
                for (int m = 0; m < M / 2; m++) dl_fma2(S[m][c], kr[m], d2);
            }
            if (OUT && lane < 4) {
                const float kq = sh.kq[j];
                *(float4*)(sh.o[j] + j0) = make_float4(fmaf(kq, dl[0], ys[0]), fmaf(kq, dl[1], ys[1]), fmaf(kq, dl[2], ys[2]), fmaf(kq, dl[3], ys[3]));
            }
        }
        __syncthreads();
        if (OUT)
#pragma unroll
            for (int i = 0; i < R; i++) {
                const int j = warp + i * NW;
                if (j >= nr) continue;
                float o[E];
#pragma unroll
                for (int e = 0; e < E; e++) o[e] = sh.o[j][lane * E + e];
                if (a.norm) {
                    float ss = 0.f, z[E];
#pragma unroll
                    for (int e = 0; e < E; e++) ss = fmaf(o[e], o[e], ss);
                    const float rr = (float)sz_rsqrt64((double)sz_warp_sum(ss) * (1.0 / D) + (double)a.eps);
                    dl_unpack<TYPE, E>(zw[i], z);
#pragma unroll
                    for (int e = 0; e < E; e++) o[e] = o[e] * rr * a.norm[lane * E + e] * dl_sigmoid<TYPE>(z[e]);
                }
                dl_store<TYPE, E>(a.out + (size_t)(s.r0 + r0 + j) * a.out_stride + (size_t)(h * D + lane * E) * ESZ, o);
            }
        if (r0 + DL_SET < s.n) ask(r0 + DL_SET);
    }
    float* p = (float*)(a.state + (size_t)s.to * a.state_stride) + ((size_t)h * D + i0) * D + j0;
#pragma unroll
    for (int m = 0; m < M / 2; m++) {
        *(float4*)(p + (size_t)(2 * m) * D) = make_float4(dl_lo(S[m][0]), dl_lo(S[m][1]), dl_lo(S[m][2]), dl_lo(S[m][3]));
        *(float4*)(p + (size_t)(2 * m + 1) * D) = make_float4(dl_hi(S[m][0]), dl_hi(S[m][1]), dl_hi(S[m][2]), dl_hi(S[m][3]));
    }
}

// ---- argument checks -----------------------------------------------------------------------------------------------------------------------
bool dl_io(int type) { return type == SZ_TYPE_F32 || type == SZ_TYPE_F16 || type == SZ_TYPE_BF16; }
int dl_esz(int type) { return type == SZ_TYPE_F32 ? 4 : 2; }

int dl_check(const sz_delta_pool* p, const sz_delta_batch* b, const char* who) {
    if (!p || !b) return sz_fail(SZ_E_ARG, "%s: null pool or batch", who);
    if (p->head_dim != 64 && p->head_dim != 128) return sz_fail(SZ_E_ARG, "%s: heads of %d (64 or 128)", who, p->head_dim);
    if (p->k_heads < 1 || p->v_heads < p->k_heads || p->v_heads > 1024 || p->v_heads % p->k_heads || p->n_slots < 1)
        return sz_fail(SZ_E_ARG, "%s: %d value heads on %d key heads, %d slots", who, p->v_heads, p->k_heads, p->n_slots);
    if (p->grouped != 0 && p->grouped != 1) return sz_fail(SZ_E_ARG, "%s: grouped is 0 or 1", who);
    if (b->n_seq < 1 || b->n_seq > 4096 || b->rows < 1 || b->rows > (1 << 20) || b->max_rows < 0)
        return sz_fail(SZ_E_ARG, "%s: %d sequences (1 .. 4096), %d rows (1 .. 1048576), at most %d of one", who, b->n_seq, b->rows, b->max_rows);
    return SZ_OK;
}
int dl_check_tables(const sz_delta_batch* b, const char* who) {
    if (!b->row_start || !b->lens || !b->from || ((b->row_start | b->lens | b->from | b->to | b->take) & 3)) return sz_fail(SZ_E_ARG, "%s: null or misaligned table", who);
    return SZ_OK;
}
// rows of n elements of esz bytes, `stride` elements apart, 16-byte aligned (align 16) or to an element
int dl_check_rows(uint64_t p, int64_t stride, int64_t n, int rows, int esz, int align, const char* name, const char* who) {
    if (!p || (p & (align - 1)) || (rows > 1 && (stride < n || (stride * esz) & (align - 1))) || stride > (1ll << 40))
        return sz_fail(SZ_E_ARG, "%s: %s: rows of %lld elements, %lld apart, %d-byte aligned", who, name, (long long)n, (long long)stride, align);
    return SZ_OK;
}
// Whether rows of n and m elements, with the same number of rows, lie apart: not in one range, or side by side in rows of one stride
bool dl_apart(uint64_t p, int64_t ps, int64_t n, uint64_t q, int64_t qs, int64_t m, int rows, int esz) {
    const uint64_t pe = p + ((uint64_t)(rows - 1) * ps + n) * esz, qe = q + ((uint64_t)(rows - 1) * qs + m) * esz;
    if (p >= qe || q >= pe) return true;
    if (ps != qs || rows < 2) return false;
    const uint64_t row = (uint64_t)ps * esz, at = p > q ? (row - (p - q) % row) % row : (q - p) % row;      // where a row of q begins in one of p's
    return at >= (uint64_t)n * esz && at + (uint64_t)m * esz <= row;
}
DlBatch dl_batch(const sz_delta_pool* p, const sz_delta_batch* b, uint64_t scratch) {
    DlBatch d = {};
    d.n_seq = b->n_seq; d.rows = b->rows; d.n_slots = p->n_slots;
    d.row_start = (const int32_t*)b->row_start; d.lens = (const int32_t*)b->lens; d.from = (const int32_t*)b->from;
    d.to = (const int32_t*)(b->to ? b->to : b->from); d.take = (const int32_t*)b->take;
    d.err = (u32*)scratch;
    return d;
}
// The most rows that a sequence of the call is said to have.
int dl_most(const sz_delta_batch* b) { return b->max_rows && b->max_rows < b->rows ? b->max_rows : b->rows; }
// From how many rows on a sequence goes in chunks (0: none of the call does).  Row by row costs by the row, a chunk what it costs, and its blocks are one a multiprocessor: the more
// of them have to wait for each other, the later they are worth it.  us, row by row / in chunks, bf16: sequences of 32 heads of 128 (128 blocks each), one of 36 rows 26.1 / 27.7, of 40
// 28.2 / 27.6; two of 44 rows 31.1 / 32.7, of 48 33.2 / 32.7; three of 56 rows 38.1 / 39.8, of 64 43.0 / 40.4; four of 64 rows 43.1 / 48.4, of 80 52.7 / 59.4, of 96 62.5 / 60.1; eight of 72 rows 81 / 105, of 96
// 106 / 107, of 112 123 / 108; 16 of 72 rows 160 / 198, of 96 209 / 198; 32 of 112 rows 423 / 435, of 128 481 / 440; 64 of 112 rows 828 / 948, of 128 941 / 962, of 160 1,166 / 1,153.  Heads of 64, of 4 and of 16
// heads, one of 40 rows 20.2 / 21.7, 20.3 / 24.6, of 48 23.6 / 21.9, 23.9 / 24.6; 64 of 4 heads, 48 rows 28.7 / 30.4, 52 31.1 / 30.0.
int dl_least(const sz_delta_pool* p, const sz_delta_batch* b) {
    const int64_t blocks = (int64_t)p->v_heads * 4 * min(b->n_seq, b->rows / 32 + 1);
    const int least = p->head_dim == 64 ? 48 : blocks <= DL_SM ? 40 : blocks <= 2 * DL_SM ? 48 : blocks <= 3 * DL_SM ? 60 : blocks <= 16 * DL_SM ? 96 : 128;
    return dl_most(b) >= least ? least : 0;
}

template <int TYPE>
using DlConvFn = void (*)(const DlBatch, const DlConv);
template <int TYPE>
DlConvFn<TYPE> dl_conv_fn(int k) {
    switch (k) {
        case 2: return sz_delta_conv_kernel<TYPE, 2>;
        case 3: return sz_delta_conv_kernel<TYPE, 3>;
        case 4: return sz_delta_conv_kernel<TYPE, 4>;
        case 5: return sz_delta_conv_kernel<TYPE, 5>;
        case 6: return sz_delta_conv_kernel<TYPE, 6>;
        case 7: return sz_delta_conv_kernel<TYPE, 7>;
        default: return sz_delta_conv_kernel<TYPE, 8>;
    }
}

}  // namespace

extern "C" int sz_delta_scratch_bytes(const sz_delta_pool* pool, const sz_delta_batch* batch, int io_type, int64_t* bytes) {
    const char* who = "sz_delta_scratch_bytes";
    const int rc = dl_check(pool, batch, who);
    if (rc) return rc;
    if (!dl_io(io_type)) return sz_fail(SZ_E_TYPE, "%s: inputs of type %d", who, io_type);
    if (!bytes) return sz_fail(SZ_E_ARG, "%s: null result", who);
    const int least = dl_least(pool, batch);
    *bytes = 256 + (least ? dl_chunk_bytes(pool->head_dim, pool->k_heads, pool->v_heads, io_type, batch->n_seq, batch->rows, least) : 0);
    return SZ_OK;
}

extern "C" int sz_delta_status(uint64_t scratch, int init, int* code, uint64_t stream) {
    if (!scratch || (scratch & 255)) return sz_fail(SZ_E_ARG, "sz_delta_status: null or misaligned scratch");
    cudaStream_t st = (cudaStream_t)stream;
    if (init) { SZ_CUDA(cudaMemsetAsync((void*)scratch, 0, 256, st)); return SZ_OK; }
    if (!code) return sz_fail(SZ_E_ARG, "sz_delta_status: null code");
    u32 v = 0;
    SZ_CUDA(cudaMemcpyAsync(&v, (const void*)scratch, 4, cudaMemcpyDeviceToHost, st));
    SZ_CUDA(cudaStreamSynchronize(st));
    *code = (int)v;
    return v ? sz_fail(SZ_E_DEVICE, "sz_delta: the tables of a call did not fit (%s%s%s%s)", v & DL_E_SLOT ? " slot out of range;" : "", v & DL_E_ROWS ? " row_start past the rows or descending;" : "",
                       v & DL_E_CLASH ? " a slot that another sequence uses;" : "", v & DL_E_WAIT ? " a bounded wait ran out;" : "")
             : SZ_OK;
}

extern "C" int sz_delta_conv(const sz_delta_pool* pool, const sz_delta_batch* batch, int io_type, uint64_t x, int64_t x_stride, uint64_t w, uint64_t bias, uint64_t y, int64_t y_stride,
                             uint64_t scratch, int64_t scratch_bytes, uint64_t stream) {
    const char* who = "sz_delta_conv";
    int rc = dl_check(pool, batch, who);
    if (rc || (rc = dl_check_tables(batch, who))) return rc;
    if (!dl_io(io_type)) return sz_fail(SZ_E_TYPE, "%s: inputs of type %d", who, io_type);
    if (!dl_io(pool->conv_type)) return sz_fail(SZ_E_TYPE, "%s: carried rows of type %d", who, pool->conv_type);
    const int esz = dl_esz(io_type), ch = (2 * pool->k_heads + pool->v_heads) * pool->head_dim;
    const int64_t slot = (int64_t)(pool->conv_k - 1) * ch * dl_esz(pool->conv_type);
    if (pool->conv_k < 2 || pool->conv_k > 8) return sz_fail(SZ_E_ARG, "%s: a convolution over %d rows (2 .. 8)", who, pool->conv_k);
    if (!pool->conv || (pool->conv & 15) || (pool->n_slots > 1 && (pool->conv_stride < slot || (pool->conv_stride & 15))))
        return sz_fail(SZ_E_ARG, "%s: carried rows: slots of %lld bytes, %lld apart, 16-byte aligned", who, (long long)slot, (long long)pool->conv_stride);
    if ((rc = dl_check_rows(x, x_stride, ch, batch->rows, esz, 16, "x", who)) || (rc = dl_check_rows(y, y_stride, ch, batch->rows, esz, 16, "y", who))) return rc;
    if (!w || ((w | bias) & 15)) return sz_fail(SZ_E_ARG, "%s: weights and bias 16-byte aligned", who);
    if (!dl_apart(x, x_stride, ch, y, y_stride, ch, batch->rows, esz)) return sz_fail(SZ_E_ARG, "%s: y lies over x", who);
    if (!scratch || (scratch & 255) || scratch_bytes < 256) return sz_fail(SZ_E_SCRATCH, "%s: the scratch is 256-byte aligned and holds the status word at least", who);
    const DlBatch d = dl_batch(pool, batch, scratch);
    DlConv a = {};
    a.x = (const u8*)x; a.y = (u8*)y; a.x_stride = x_stride * esz; a.y_stride = y_stride * esz;
    a.w = (const float*)w; a.bias = (const float*)bias;
    a.conv = (u8*)pool->conv; a.conv_stride = pool->conv_stride; a.conv_type = pool->conv_type; a.ch = ch;
    // rows a thread has: as many as leave every multiprocessor 16 warps, up to 32 (a tile's first rows are read twice)
    const int vecs = (ch / DL_V + 127) / 128;
    // a block a sequence where they have a few rows each: one look-up instead of one for every sequence that a tile meets (64 sequences, 163 rows: 10.8 us by tiles, 10.1 so; 9.2 since a sequence is looked up with one wait)
    const bool by_seq = batch->n_seq > 1 && dl_most(batch) <= 8;
    a.tile = 1;
    while (a.tile < 32 && (int64_t)vecs * ((batch->rows + 2 * a.tile - 1) / (2 * a.tile)) >= 4 * DL_SM) a.tile *= 2;
    if (by_seq) a.tile = 0;
    const dim3 grid(vecs, by_seq ? batch->n_seq : (batch->rows + a.tile - 1) / a.tile);
    if (grid.y > 65535) return sz_fail(SZ_E_ARG, "%s: %d rows of %d channels are more than a call takes", who, batch->rows, ch);
    const DlConvFn<SZ_TYPE_F32> fn = io_type == SZ_TYPE_F32 ? dl_conv_fn<SZ_TYPE_F32>(pool->conv_k) : io_type == SZ_TYPE_F16 ? dl_conv_fn<SZ_TYPE_F16>(pool->conv_k) : dl_conv_fn<SZ_TYPE_BF16>(pool->conv_k);
    SZ_CUDA(sz_launch("delta_conv", fn, grid, dim3(128), 0, (cudaStream_t)stream, true, d, a));
    return SZ_OK;
}

extern "C" int sz_delta_rows(const sz_delta_pool* pool, const sz_delta_batch* batch, const sz_delta_gates* gates, int io_type, uint64_t q, int64_t q_stride, uint64_t k, int64_t k_stride,
                             uint64_t v, int64_t v_stride, uint64_t alpha, int64_t alpha_stride, uint64_t beta, int64_t beta_stride, uint64_t z, int64_t z_stride, uint64_t out,
                             int64_t out_stride, uint64_t scratch, int64_t scratch_bytes, uint64_t stream) {
    const char* who = "sz_delta_rows";
    int rc = dl_check(pool, batch, who);
    if (rc || (rc = dl_check_tables(batch, who))) return rc;
    if (!dl_io(io_type)) return sz_fail(SZ_E_TYPE, "%s: inputs of type %d", who, io_type);
    const int esz = dl_esz(io_type), D = pool->head_dim, kw = pool->k_heads * D, vw = pool->v_heads * D, rows = batch->rows;
    const int64_t slot = (int64_t)vw * D * 4;
    if (!pool->state || (pool->state & 15) || (pool->n_slots > 1 && (pool->state_stride < slot || (pool->state_stride & 15))))
        return sz_fail(SZ_E_ARG, "%s: states: slots of %lld bytes, %lld apart, 16-byte aligned", who, (long long)slot, (long long)pool->state_stride);
    if (!gates || !gates->a || !gates->dt || ((gates->a | gates->dt) & 3) || (gates->norm & 15)) return sz_fail(SZ_E_ARG, "%s: a and dt given, the norm's weights 16-byte aligned", who);
    if ((gates->norm != 0) != (z != 0)) return sz_fail(SZ_E_ARG, "%s: the norm's weights and the gate z come together", who);
    if (gates->norm && !(gates->eps >= 0.f)) return sz_fail(SZ_E_ARG, "%s: eps >= 0", who);
    if ((q != 0) != (out != 0)) return sz_fail(SZ_E_ARG, "%s: q and out come together (neither: the states alone)", who);
    if (!q && z) return sz_fail(SZ_E_ARG, "%s: a gate without outputs", who);
    if ((q && ((rc = dl_check_rows(q, q_stride, kw, rows, esz, 16, "q", who)) || (rc = dl_check_rows(out, out_stride, vw, rows, esz, 16, "out", who)))) ||
        (rc = dl_check_rows(k, k_stride, kw, rows, esz, 16, "k", who)) || (rc = dl_check_rows(v, v_stride, vw, rows, esz, 16, "v", who)) ||
        (rc = dl_check_rows(alpha, alpha_stride, pool->v_heads, rows, esz, esz, "alpha", who)) || (rc = dl_check_rows(beta, beta_stride, pool->v_heads, rows, esz, esz, "beta", who)) ||
        (z && (rc = dl_check_rows(z, z_stride, vw, rows, esz, 16, "z", who))))
        return rc;
    if (out && !(dl_apart(out, out_stride, vw, q, q_stride, kw, rows, esz) && dl_apart(out, out_stride, vw, k, k_stride, kw, rows, esz) && dl_apart(out, out_stride, vw, v, v_stride, vw, rows, esz) &&
                 dl_apart(out, out_stride, vw, alpha, alpha_stride, pool->v_heads, rows, esz) && dl_apart(out, out_stride, vw, beta, beta_stride, pool->v_heads, rows, esz) &&
                 (!z || dl_apart(out, out_stride, vw, z, z_stride, vw, rows, esz))))
        return sz_fail(SZ_E_ARG, "%s: out lies over an input", who);
    int64_t need = 0;
    if ((rc = sz_delta_scratch_bytes(pool, batch, io_type, &need))) return rc;
    if (!scratch || (scratch & 255) || scratch_bytes < need) return sz_fail(SZ_E_SCRATCH, "%s: %lld bytes of scratch given, %lld needed, 256-byte aligned", who, (long long)scratch_bytes, (long long)need);
    const DlBatch d = dl_batch(pool, batch, scratch);
    DlRule a = {};
    a.q = (const u8*)q; a.k = (const u8*)k; a.v = (const u8*)v; a.alpha = (const u8*)alpha; a.beta = (const u8*)beta; a.z = (const u8*)z; a.out = (u8*)out;
    a.q_stride = q_stride * esz; a.k_stride = k_stride * esz; a.v_stride = v_stride * esz; a.alpha_stride = alpha_stride * esz; a.beta_stride = beta_stride * esz;
    a.z_stride = z_stride * esz; a.out_stride = out_stride * esz;
    a.a = (const float*)gates->a; a.dt = (const float*)gates->dt; a.norm = (const float*)gates->norm; a.eps = gates->eps; a.q_scale = 1.f / sqrtf((float)D);
    a.kh = pool->k_heads; a.vh = pool->v_heads; a.grouped = pool->grouped;
    a.state = (u8*)pool->state; a.state_stride = pool->state_stride;
    a.least = dl_least(pool, batch);
    cudaStream_t st = (cudaStream_t)stream;
    using Fn = void (*)(const DlBatch, const DlRule);
#define SZ_DL_T(D_, O) (io_type == SZ_TYPE_F32 ? (Fn)sz_delta_rows_kernel<D_, SZ_TYPE_F32, O> : io_type == SZ_TYPE_F16 ? (Fn)sz_delta_rows_kernel<D_, SZ_TYPE_F16, O> : (Fn)sz_delta_rows_kernel<D_, SZ_TYPE_BF16, O>)
    const Fn fn = D == 128 ? (q ? SZ_DL_T(128, true) : SZ_DL_T(128, false)) : (q ? SZ_DL_T(64, true) : SZ_DL_T(64, false));
#undef SZ_DL_T
    SZ_CUDA(sz_launch("delta_rows", fn, dim3(pool->v_heads, batch->n_seq), dim3(2 * D), 0, st, true, d, a));
    return a.least ? dl_chunk_launch(D, io_type, d, a, scratch + 256, st) : SZ_OK;
}
