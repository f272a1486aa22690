// A cache in pages (sz_paged_*): the append kernel, the kernel that joins the attention's parts, and the C ABI.  sz_paged.cuh has the
// attention itself.
#include "sz_paged.cuh"

#include <math.h>

namespace {

constexpr int PG_BLOCKS = 148;       // multiprocessors (a GPU with another number: more or fewer blocks than places, the same results)

// ---- append ------------------------------------------------------------------------------------------------------------------------------------
struct PgAppend {
    const u8 *k, *v, *q;
    u8* qo;
    long long k_stride, v_stride, q_stride, q_head_stride, qo_stride;   // bytes
    const float *q_norm, *k_norm;
    int nh, half, heads;             // heads: nh (0 without q) + 2 nkv
    float eps;
    double freq[128];                // 1 / theta^(2 i / dims)
};

// The sequence of row r (its last one that begins at or before r), by the whole block; -1: none.
template <int NTH>
__device__ int pg_seq_of(const PgBatch& d, int r) {
    int n = 0;
    for (int b0 = 0; b0 <= d.n_seq; b0 += NTH) n += __syncthreads_count(b0 + (int)threadIdx.x <= d.n_seq && pg_row(d, b0 + threadIdx.x) <= r);
    return n > d.n_seq ? -1 : n - 1;
}

// f = head / sqrt(mean(head^2) + eps) * w, then (f_i, f_(i + half)) turned by pos theta^(-2 i / dims).  A lane has hd / 32 neighbouring dimensions, and
// a rotation's partner is hd / 32 dimensions of another lane.  Sums of squares and rotations in f32, one rounding to the stored type.
// R = 1 row a block, a warp a head, for few rows: latency bounds those - sequence, length, page, head, one after the other -, so the head is read
// while its row is looked up.  R = PG_APP where that still gives every multiprocessor a block: a warp a row, its heads two at a time (their loads
// and their norms' shuffles side by side).  16 + 2 + 2 heads of 256, bf16: 1 row 3.9 us, 4,093 rows 22.3 against 51 with R = 1 (83 MB: 12.8 us of
// them; the chains of norm, rotation and store of one wave of warps are the rest); 163 rows of 32 + 8 + 8 heads of 128 5.2.
// A row's angles are taken once a block, in f64 (a far position's angle has no digits left in f32), reduced to [-pi, pi] there, and the sine and
// cosine of the reduced angle in f32 with its rounding put back by their derivatives.
constexpr int PG_APP = 8;
template <int K> struct PgKind { __device__ constexpr operator int() const { return K; } };
template <int E, int type>
__device__ __forceinline__ void pg_load_n(const u8* p, float* f) {      // E neighbouring elements
    if (type == SZ_TYPE_F32) {
#pragma unroll
        for (int e = 0; e < E; e += E == 2 ? 2 : 4) {
            if (E == 2) { const float2 x = *(const float2*)p; f[0] = x.x; f[1] = x.y; }
            else { const float4 x = *(const float4*)(p + 4 * e); f[e] = x.x; f[e + 1] = x.y; f[(e + 2) % E] = x.z; f[(e + 3) % E] = x.w; }
        }
        return;
    }
    u32 w[E / 2];
    if (E == 8) *(uint4*)w = *(const uint4*)p;
    else if (E == 4) *(uint2*)w = *(const uint2*)p;
    else w[0] = *(const u32*)p;
#pragma unroll
    for (int e = 0; e < E; e += 2) {
        const float2 x = type == SZ_TYPE_F16 ? __half22float2(*(const __half2*)&w[e / 2]) : make_float2(__uint_as_float(w[e / 2] << 16), __uint_as_float(w[e / 2] & 0xffff0000u));
        f[e] = x.x; f[e + 1] = x.y;
    }
}
template <int E, int type>
__device__ __forceinline__ void pg_store_n(u8* p, const float* f) {
    if (type == SZ_TYPE_F32) {
#pragma unroll
        for (int e = 0; e < E; e += E == 2 ? 2 : 4) {
            if (E == 2) *(float2*)p = make_float2(f[0], f[1]);
            else *(float4*)(p + 4 * e) = make_float4(f[e], f[e + 1], f[(e + 2) % E], f[(e + 3) % E]);
        }
    } else {
        u32 w[E / 2];
#pragma unroll
        for (int e = 0; e < E; e += 2) w[e / 2] = type == SZ_TYPE_F16 ? pg_pack_f16(f[e], f[e + 1]) : pg_pack_bf16(f[e], f[e + 1]);
        if (E == 8) *(uint4*)p = *(const uint4*)w;
        else if (E == 4) *(uint2*)p = *(const uint2*)w;
        else *(u32*)p = w[0];
    }
}

template <int CT, int HD, int IO, int R>
__global__ void __launch_bounds__(256, R == 1 ? 0 : 4) sz_pg_append_kernel(const __grid_constant__ PgBatch d, const __grid_constant__ PgAppend a) {
    constexpr int E = HD / 32, ESZ = IO == SZ_TYPE_F32 ? 4 : 2, CTY = CT == PG_F16 ? SZ_TYPE_F16 : SZ_TYPE_BF16;
    __shared__ float2 turn[R][HD / 2];
    __shared__ float tmp[8][HD];
    __shared__ int s_pos[R];               // the row's position; -1: the row is left out
    __shared__ long long s_off[R];         // where it lies in the pools; -1: it is not stored
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r0 = blockIdx.x * R, half = a.half, d0 = lane * E, nq = a.q ? a.nh : 0;
    float one[E];                               // R = 1: the warp's head, its kind (0 queries, 1 keys, 2 values) and its number there
    const int x = blockIdx.y * 8 + warp, kind1 = x < nq ? 0 : x < nq + d.nkv ? 1 : 2, h1 = x - (kind1 == 0 ? 0 : kind1 == 1 ? nq : nq + d.nkv);
    if ((int)threadIdx.x < R) { s_pos[threadIdx.x] = -1; s_off[threadIdx.x] = -1; }
    __syncthreads();
    sz_pdl_wait();
    sz_pdl_trigger();
    if (R == 1 && x < a.heads)                  // its elements are under way while the row is looked up
        pg_load_n<E, IO>((kind1 == 0 ? a.q + (long long)r0 * a.q_stride + h1 * a.q_head_stride : (kind1 == 1 ? a.k + (long long)r0 * a.k_stride : a.v + (long long)r0 * a.v_stride) + h1 * (HD * ESZ)) + d0 * ESZ, one);
    int falls = 0;                              // a row_start that descends: a row would be two sequences'
    for (int i = threadIdx.x; i < d.n_seq; i += 256) {
        const int b0 = pg_row(d, i), b1 = pg_row(d, i + 1), end = __ldg(d.row_start + i + 1), len = __ldg(d.lens + i);
        falls |= b1 < b0;
        for (int row = max(b0, r0); row < min(b1, r0 + R); row++) {      // (the block's rows of this sequence)
            const long long at = (long long)len - ((long long)end - row);
            if (at < 0) continue;
            const int pos = (int)at, o = pos - d.shared_len;
            long long off = -1;
            u32 bad = 0;
            if (o < 0) bad = PG_E_SHARED;
            else if ((long long)o >= (long long)d.max_pages << d.ps_log2) bad = PG_E_END;
            else {
                const int page = __ldg(d.pages + (size_t)i * d.max_pages + (o >> d.ps_log2));
                if ((u32)page >= (u32)d.n_pages) bad = PG_E_PAGE;
                else off = (long long)page * d.page_stride + (long long)(o & ((1 << d.ps_log2) - 1)) * d.pos_stride;
            }
            if (bad) atomicOr(d.err, bad);
            s_pos[row - r0] = pos; s_off[row - r0] = off;
        }
    }
    falls = __syncthreads_or(falls);
    if (r0 == 0 && threadIdx.x == 0 && blockIdx.y == 0 && (falls || __ldg(d.row_start + d.n_seq) > d.rows)) atomicOr(d.err, PG_E_ROWS);
    if (falls) return;                          // nothing is stored then
    for (int i = threadIdx.x; i < half * R; i += 256) {
        const int j = i / half, k = i - j * half, pos = s_pos[j];
        if (pos < 0) continue;
        const double f = (double)pos * a.freq[k];
        const double kq = rint(f * 0.15915494309189535);
        double rd = fma(-kq, 6.283185307179586, f);
        rd = fma(-kq, 2.4492935982947064e-16, rd);
        const float hi = (float)rd, lo = (float)(rd - (double)hi);
        float sn, cs;
        sincosf(hi, &sn, &cs);
        turn[j][k] = make_float2(fmaf(-sn, lo, cs), fmaf(cs, lo, sn));
    }
    __syncthreads();
    const int j = R == 1 ? 0 : warp;
    const long long r = r0 + j, off = s_off[j];
    if (s_pos[j] < 0) return;
    // partners of a lane's dimensions: another lane's, where the halves are whole lanes; f' = c f + s partner
    const bool lower = d0 < half, turned = d0 < 2 * half, by_lane = half % E == 0;
    const int partner = half ? (lower ? lane + half / E : lane - half / E) & 31 : lane;
    float c[E], s[E];
#pragma unroll
    for (int e = 0; e < E; e++) {
        const float2 t = by_lane && turned ? turn[j][lower ? d0 + e : d0 + e - half] : make_float2(1.f, 0.f);
        c[e] = t.x;
        s[e] = lower ? -t.y : t.y;
    }
    auto store_cache = [&](u8* dst, const float* f) {
        if (CT != PG_Q8) { pg_store_n<E, CTY>(dst + 2 * d0, f); return; }
        float big = 0.f;                        // packed: a group of 32 dimensions is 32 / E lanes
#pragma unroll
        for (int e = 0; e < E; e++) big = fmaxf(big, fabsf(f[e]));
#pragma unroll
        for (int o = 16 / E; o > 0; o >>= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, o));
        const __half sh = __float2half_rn(big > 0.0f ? big * (1.0f / 127.0f) : 0.0f);
        const float sr = __half2float(sh), inv = sr > 0.0f ? 1.0f / sr : 0.0f;
        u32 code[E];
#pragma unroll
        for (int e = 0; e < E; e++) { int q = __float2int_rn(f[e] * inv); q = q < -127 ? -127 : (q > 127 ? 127 : q); code[e] = (u32)q & 255u; }
        if (E == 8) *(uint2*)(dst + 8 * lane) = make_uint2(code[0] | code[1] << 8 | code[2 % E] << 16 | code[3 % E] << 24, code[4 % E] | code[5 % E] << 8 | code[6 % E] << 16 | code[7 % E] << 24);
        else if (E == 4) *(u32*)(dst + 4 * lane) = code[0] | code[1] << 8 | code[2 % E] << 16 | code[3 % E] << 24;
        else *(u16*)(dst + 2 * lane) = (u16)(code[0] | code[1] << 8);
        if (lane % (32 / E) == 0) *(u16*)(dst + HD + 2 * (lane * E / 32)) = __half_as_ushort(sh);
        if (lane >= HD / 32 && lane < 8) *(u16*)(dst + HD + 2 * lane) = 0;      // the 16 bytes behind the codes: those behind the scales are zero
    };
    auto norm = [&](const float* f) {           // 1 / the root of the mean square
        float ss = 0.f;
#pragma unroll
        for (int e = 0; e < E; e++) ss = fmaf(f[e], f[e], ss);
        return (float)sz_rsqrt64((double)sz_warp_sum(ss) / HD + (double)a.eps);
    };
    auto head = [&](auto kind_, float* f, float rr, const float* w, const float* ww, u8* to) {        // scale, rotation, store of a head
        const int kind = kind_;
        if (kind < 2 && w) {
#pragma unroll
            for (int e = 0; e < E; e++) f[e] = f[e] * rr * ww[e];
        }
        if (kind < 2 && half) {
            if (by_lane) {
#pragma unroll
                for (int e = 0; e < E; e++) {
                    const float p = __shfl_sync(0xffffffffu, f[e], partner), t = fmaf(f[e], c[e], p * s[e]);
                    f[e] = turned ? t : f[e];              // (not by 1 and 0: 0 times another dimension's infinity)
                }
            } else {                            // through shared memory
#pragma unroll
                for (int e = 0; e < E; e++) tmp[warp][d0 + e] = f[e];
                __syncwarp();
                for (int i = lane; i < half; i += 32) {
                    const float2 t2 = turn[j][i];
                    const float u = tmp[warp][i], v = tmp[warp][i + half];
                    tmp[warp][i] = u * t2.x - v * t2.y;
                    tmp[warp][i + half] = v * t2.x + u * t2.y;
                }
                __syncwarp();
#pragma unroll
                for (int e = 0; e < E; e++) f[e] = tmp[warp][d0 + e];
                __syncwarp();
            }
        }
        if (kind == 0) pg_store_n<E, IO>(to + d0 * ESZ, f);
        else store_cache(to, f);
    };
    auto load_w = [&](const float* w, float* ww) {
        if (!w) return;
#pragma unroll
        for (int e = 0; e < E; e += 2) { const float2 u = __ldg((const float2*)(w + d0 + e)); ww[e] = u.x; ww[e + 1] = u.y; }
    };
    if (R == 1) {
        if (x >= a.heads || (kind1 && off < 0)) return;
        const float* w = kind1 == 0 ? a.q_norm : kind1 == 1 ? a.k_norm : nullptr;
        float ww[E];
        load_w(w, ww);
        head(kind1, one, w ? norm(one) : 1.f, w, ww, kind1 == 0 ? a.qo + r * a.qo_stride + h1 * (HD * ESZ) : (u8*)(kind1 == 1 ? d.k : d.v) + off + h1 * d.head_stride);
        return;
    }
    // A warp has a row and takes its heads two at a time: their loads are under way together.  (Four: 80 registers, 24 warps a multiprocessor
    // instead of 32, 29 us at 4,093 rows where this takes 22.)
    auto heads = [&](auto kind, int n, const u8* src, long long step, u8* dst, long long dst_step, const float* w) {
        constexpr int B = 2;
        src += d0 * ESZ;
        float ww[E];
        load_w(w, ww);
        for (int x0 = 0; x0 < n; x0 += B, src += B * step, dst += B * dst_step) {
            float all[B][E], rr[B];
#pragma unroll
            for (int t = 0; t < B; t++) pg_load_n<E, IO>(src + (x0 + t < n ? t * step : 0), all[t]);        // (behind the last: the first once more)
            if (kind < 2 && w) {
#pragma unroll
                for (int t = 0; t < B; t++) rr[t] = norm(all[t]);
            }
#pragma unroll
            for (int t = 0; t < B; t++)
                if (x0 + t < n) head(kind, all[t], rr[t], w, ww, dst + t * dst_step);
        }
    };
    if (nq) heads(PgKind<0>(), nq, a.q + r * a.q_stride, a.q_head_stride, a.qo + r * a.qo_stride, HD * ESZ, a.q_norm);
    if (off < 0) return;
    heads(PgKind<1>(), d.nkv, a.k + r * a.k_stride, HD * ESZ, (u8*)d.k + off, d.head_stride, a.k_norm);
    heads(PgKind<2>(), d.nkv, a.v + r * a.v_stride, HD * ESZ, (u8*)d.v + off, d.head_stride, nullptr);
}

// ---- the plan of a call with more sequences or tiles than a block plans for itself ---------------------------------------------------------
struct PgParts { PgPart p[2]; };      // in the order of the positions
enum { PG_SHARED = 0, PG_OWN = 1 };
__global__ void __launch_bounds__(1024) sz_pg_plan_kernel(const __grid_constant__ PgBatch d, const __grid_constant__ PgParts a) {
    __shared__ u32 scan[32];
    const PgPart& p = a.p[blockIdx.x];
    sz_pdl_wait();
    sz_pdl_trigger();
    if (p.on && p.planned) pg_plan<1024>(d, p.shared, p.unit, p.tq, p.tiles, p.units, scan, nullptr, nullptr);
}

// ---- joining the parts -----------------------------------------------------------------------------------------------------------------------------
// W warps have one row and head: the parts of its items, in the order of the positions.  A lane has hd / 32 columns; the warps take the
// parts in turn and their sums are added in order.  The fewer rows and heads, the more parts each has (units are shared out evenly): 1, 2 or 8
// warps (64 rows of 16 heads, 74 parts: 75 / 69 / 58 us for the whole call; 2,048 rows and heads 129 / 126 / 134; 5,216: 404 / 410 / 425).
// What it waits for is the way to the parts - row, sequence, plan, list, maxima, sums, one after the other: 15 us of 55 with four rows.
struct PgList { int n, first, alone, lane; };     // parts of an item: their number, the block of the first; by row and head; the vector's place in its tile
__device__ PgList pg_list(const PgBatch& d, const PgPart& p, int r, int r0, int b, int h) {
    PgList l = {};
    if (!p.on) return l;
    const int start = p.shared ? pg_row(d, 0) : r0;
    const int vec = (r - start) * d.G + h % d.G, t = vec / p.tq, e = p.shared ? t : (int)p.tiles[b] + t;
    const int E = p.shared ? ((pg_row(d, d.n_seq) - start) * d.G + p.tq - 1) / p.tq : (int)p.tiles[d.n_seq];
    if (vec < 0 || e >= E) return l;      // (a row_start that descends: there are no tiles)
    const u32 us = p.units[e], n = p.units[e + 1] - us;
    if (!n) return l;
    const u32 U = p.units[E] * (u32)d.nkv, at = us * (u32)d.nkv + (u32)(h / d.G) * n;
    const PgShare share = pg_share(U, (int)min((u32)p.blocks, U));
    l.first = pg_block_of(share, at);
    l.n = pg_block_of(share, at + n - 1) - l.first + 1;
    l.alone = l.n == 1;
    l.lane = vec % p.tq;
    return l;
}
template <int HD, int W>
__global__ void __launch_bounds__(256) sz_pg_merge_kernel(const __grid_constant__ PgBatch d, const __grid_constant__ PgIo io, const __grid_constant__ PgParts a) {
    constexpr int E = HD / 32;                                       // columns a lane, in pairs: 2 lane + 64 x
    __shared__ float2 sums[8][W > 1 ? HD / 2 : 1], of_warp[8];
    const int r = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = warp % W, h = blockIdx.y * (8 / W) + warp / W, nh = d.nkv * d.G;
    sz_pdl_wait();
    sz_pdl_trigger();
    const int b = pg_seq_of<256>(d, r);
    if (b < 0 || h >= nh) return;                                    // (h: W = 8 has one head a block)
    const int r0 = pg_row(d, b), m = pg_row(d, b + 1) - r0;
    const bool sees = pg_end(d, b) - (m - 1 - (r - r0)) > 0;     // a position of its own
    PgList l[2] = {};
    if (sees) {
        l[PG_OWN] = pg_list(d, a.p[PG_OWN], r, r0, b, h);
        if (a.p[PG_OWN].direct && l[PG_OWN].alone) return;           // (written by the block that did it)
        l[PG_SHARED] = pg_list(d, a.p[PG_SHARED], r, r0, b, h);
    }
    const int s0 = a.p[0].ways == 4 ? 2 : a.p[0].ways - 1, s1 = a.p[1].ways == 4 ? 2 : a.p[1].ways - 1;      // (ways: 1, 2 or 4)
    const int n0 = l[0].n << s0, n = n0 + (l[1].n << s1);
    auto place = [&](int i, const float2*& ml) -> const float* {     // part i
        const bool own = i >= n0;
        const PgPart& p = a.p[own];
        const PgList& x = own ? l[1] : l[0];
        const int sh = own ? s1 : s0, j = own ? i - n0 : i, k = j >> sh;
        const size_t at = ((x.alone ? (size_t)r * nh + h : (size_t)(k == 0 ? 2 * x.first + 1 : 2 * (x.first + k)) * p.tq + x.lane) << sh) + (j & ((1 << sh) - 1));
        ml = (x.alone ? p.row_ml : p.ml) + at;
        return (x.alone ? p.row_o : p.o) + at * HD;
    };
    // the warp's parts are sub, sub + W ..: their largest maximum, then 32 at a time their weights, one a lane, and their sums
    float M = -INFINITY, L = 0.f;
#pragma unroll 2
    for (int i = sub + W * lane; i < n; i += 32 * W) { const float2* ml; place(i, ml); M = fmaxf(M, ml->x); }
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, s));
    float2 acc[E / 2];
#pragma unroll
    for (int x = 0; x < E / 2; x++) acc[x] = make_float2(0.f, 0.f);
    for (int i0 = sub; i0 < n; i0 += 32 * W) {
        const int i = i0 + W * lane;
        float c = 0.f;
        const float* from = nullptr;
        if (i < n) {
            const float2* ml;
            from = place(i, ml);
            const float2 x = *ml;
            c = x.x == -INFINITY ? 0.f : pg_ex2(x.x - M);
            if (x.x != -INFINITY) L += c * x.y; else from = nullptr;
        }
        u32 left = __ballot_sync(0xffffffffu, from != nullptr);      // (empty parts have no sums)
        while (left) {
            constexpr int B = W == 1 ? 4 : 8;                        // parts in flight (one warp: few parts, and the registers of eight leave half the warps; 2,045 rows 365 -> 350 us)
            float2 f[B][E / 2];
            float cw[B];
#pragma unroll
            for (int k = 0; k < B; k++) {
                const int src = left ? __ffs(left) - 1 : 0;
                const float* pk = (const float*)__shfl_sync(0xffffffffu, (unsigned long long)from, src);
                cw[k] = __shfl_sync(0xffffffffu, c, src);
                const bool ok = left != 0;
                left &= left - 1;
#pragma unroll
                for (int x = 0; x < E / 2; x++) f[k][x] = ok ? *(const float2*)(pk + 2 * lane + 64 * x) : make_float2(0.f, 0.f);
                if (!ok) cw[k] = 0.f;
            }
#pragma unroll
            for (int k = 0; k < B; k++)
#pragma unroll
                for (int x = 0; x < E / 2; x++) { acc[x].x = fmaf(cw[k], f[k][x].x, acc[x].x); acc[x].y = fmaf(cw[k], f[k][x].y, acc[x].y); }
        }
    }
    L = sz_warp_sum(L);
    if (W > 1) {
#pragma unroll
        for (int x = 0; x < E / 2; x++) sums[warp][lane + 32 * x] = acc[x];
        if (lane == 0) of_warp[warp] = make_float2(M, L);
        asm volatile("bar.sync %0, %1;" ::"r"(1 + warp / W), "n"(32 * W) : "memory");      // (the head's warps: others may have left)
        if (sub) return;
        float Mw[W], top = M;
#pragma unroll
        for (int k = 0; k < W; k++) { Mw[k] = of_warp[warp + k].x; top = fmaxf(top, Mw[k]); }
        L = 0.f;
#pragma unroll
        for (int x = 0; x < E / 2; x++) acc[x] = make_float2(0.f, 0.f);
#pragma unroll
        for (int k = 0; k < W; k++) {
            const float c = Mw[k] == -INFINITY ? 0.f : pg_ex2(Mw[k] - top);
            L = fmaf(of_warp[warp + k].y, c, L);
#pragma unroll
            for (int x = 0; x < E / 2; x++) { const float2 f = sums[warp + k][lane + 32 * x]; acc[x].x = fmaf(f.x, c, acc[x].x); acc[x].y = fmaf(f.y, c, acc[x].y); }
        }
        M = top;
    }
    const bool none = n == 0 || L == 0.f;                            // nothing the row may see
    const float inv = none ? 0.f : 1.f / L;
    u8* const op = io.out + (long long)r * io.out_stride + (long long)h * HD * io.esz;
    const u8* const gp = io.gate ? io.gate + (long long)r * io.gate_stride + (long long)h * io.gate_head_stride : nullptr;
#pragma unroll
    for (int x = 0; x < E / 2; x++) {
        const int at = (2 * lane + 64 * x) * io.esz;
        float u = none ? 0.f : acc[x].x * inv, v = none ? 0.f : acc[x].y * inv;
        if (gp) { const float2 g = pg_load2(gp + at, io.type); u *= sz_sigmoid(g.x); v *= sz_sigmoid(g.y); }
        pg_store2(op + at, io.type, u, v);
    }
    if (io.lse && lane == 0) io.lse[(size_t)r * nh + h] = none ? -INFINITY : (M + log2f(L)) * 0.6931471805599453f;
}

// ---- the host side -------------------------------------------------------------------------------------------------------------------------------
int pg_head_bytes(int type, int hd) { return type == SZ_TYPE_Q8_KV ? hd + ((hd / 32 * 2 + 15) & ~15) : 2 * hd; }
int pg_esz(int type) { return type == SZ_TYPE_F32 ? 4 : 2; }

int pg_check(const sz_paged_cache* c, const sz_paged_batch* b, int n_head, const char* who) {
    if (!c || !b) return sz_fail(SZ_E_ARG, "%s: null cache or batch", who);
    if (c->type != SZ_TYPE_F16 && c->type != SZ_TYPE_BF16 && c->type != SZ_TYPE_Q8_KV) return sz_fail(SZ_E_TYPE, "%s: cache type %d (F16, BF16 and Q8_KV have kernels)", who, c->type);
    if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256) return sz_fail(SZ_E_ARG, "%s: heads of %d (64, 128 and 256 have kernels)", who, c->head_dim);
    if (c->n_kv_head < 1 || c->n_kv_head > 1024 || n_head < c->n_kv_head || n_head % c->n_kv_head || n_head > 4096)
        return sz_fail(SZ_E_ARG, "%s: %d heads on %d key heads", who, n_head, c->n_kv_head);
    if (c->page_size < 8 || c->page_size > 1024 || (c->page_size & (c->page_size - 1))) return sz_fail(SZ_E_ARG, "%s: pages of %d positions (a power of two from 8 to 1024)", who, c->page_size);
    if (c->n_pages < 1) return sz_fail(SZ_E_ARG, "%s: %d pages", who, c->n_pages);
    const int64_t hb = pg_head_bytes(c->type, c->head_dim);
    if ((c->page_stride | c->head_stride | c->pos_stride) & 15 || c->page_stride < hb || c->pos_stride < hb || (c->n_kv_head > 1 && c->head_stride < hb) || c->head_stride < 0)
        return sz_fail(SZ_E_ARG, "%s: strides of pages, heads and positions are multiples of 16 and at least a head's %lld bytes", who, (long long)hb);
    if (b->n_seq < 1 || b->n_seq > PG_MAX_SEQ || b->rows < 1 || b->rows > (1 << 20) || b->max_pages < 1 || b->shared_len < 0)
        return sz_fail(SZ_E_ARG, "%s: %d sequences (1 .. %d), %d rows (1 .. 1048576), %d pages a sequence, %d shared positions", who, b->n_seq, PG_MAX_SEQ, b->rows, b->max_pages, b->shared_len);
    return SZ_OK;
}
int pg_check_tables(const sz_paged_cache* c, const sz_paged_batch* b, const char* who) {
    if (!c->k || !c->v || ((c->k | c->v) & 15)) return sz_fail(SZ_E_ARG, "%s: null or misaligned pools (16 bytes)", who);
    if (!b->pages || !b->row_start || !b->lens || (b->shared_len > 0 && !b->shared_pages) || ((b->pages | b->row_start | b->lens | b->shared_pages) & 3))
        return sz_fail(SZ_E_ARG, "%s: null or misaligned tables", who);
    return SZ_OK;
}
int pg_check_rows(uint64_t p, int64_t stride, int64_t head_stride, int n_head, int hd, int rows, int esz, const char* name, const char* who) {
    if (!p || (p & 15) || (stride * esz & 15) || (head_stride * esz & 15)) return sz_fail(SZ_E_ARG, "%s: %s null, or its rows or heads not 16-byte aligned", who, name);
    if (head_stride < hd || (rows > 1 && stride < (n_head - 1) * head_stride + hd)) return sz_fail(SZ_E_ARG, "%s: rows or heads of %s overlap", who, name);
    return SZ_OK;
}
PgBatch pg_batch(const sz_paged_cache* c, const sz_paged_batch* b, int n_head, uint64_t scratch) {
    PgBatch d = {};
    d.k = (const u8*)c->k; d.v = (const u8*)c->v;
    d.page_stride = c->page_stride; d.head_stride = c->head_stride; d.pos_stride = c->pos_stride;
    d.pages = (const int32_t*)b->pages; d.row_start = (const int32_t*)b->row_start; d.lens = (const int32_t*)b->lens; d.shared_pages = (const int32_t*)b->shared_pages;
    d.n_seq = b->n_seq; d.rows = b->rows; d.max_pages = b->max_pages; d.shared_len = b->shared_len; d.n_pages = c->n_pages;
    while ((1 << d.ps_log2) < c->page_size) d.ps_log2++;
    d.nkv = c->n_kv_head; d.G = n_head / c->n_kv_head;
    d.err = (u32*)scratch;
    return d;
}
// Tiles of 16 query vectors a block: as many as a sequence's rows fill on average, up to 4 (more vectors share a key read from memory; a
// sequence with more makes more items).
int pg_tiles_of(long long vectors) { return vectors <= 16 ? 1 : vectors <= 32 ? 2 : 4; }

// Vectors from which the tcgen05 kernel takes whole units: of a sequence on average (own positions), of the batch (shared ones).
constexpr int PG_TC_MIN = 96;
bool pg_tc_type(int cache_type) { return cache_type == SZ_TYPE_F16 || cache_type == SZ_TYPE_BF16; }

// The scratch: the status word, then for every kind of part the plan's tables, the blocks' parts, the whole items by row.
struct PgScratch { PgParts a; int64_t bytes; };
PgScratch pg_scratch(const sz_paged_cache* c, const sz_paged_batch* b, int nh, uint64_t base) {
    PgScratch s = {};
    int64_t off = 256;
    const int hd = c->head_dim, G = nh / c->n_kv_head;
    auto take = [&](int64_t n) { const int64_t at = off; off += (n + 255) & ~(int64_t)255; return base + at; };
    for (PgPart* p = s.a.p; p < s.a.p + 2; p++) {
        const int64_t slots = 2ll * PG_BLOCKS * 256;      // parts of the blocks, by vector: blocks a multiprocessor x vectors a tile x ways is 256 at most, of the tcgen05 kernel too
        p->tiles = (u32*)take(4ll * (b->n_seq + 1));
        p->units = (u32*)take(4ll * ((int64_t)b->rows * G / 16 + b->n_seq + 2));
        p->o = (float*)take(slots * hd * 4);
        p->ml = (float2*)take(slots * 8);
        p->row_o = (float*)take((int64_t)b->rows * nh * 4 * hd * 4);      // (4 ways at most)
        p->row_ml = (float2*)take((int64_t)b->rows * nh * 4 * 8);
    }
    s.bytes = off;
    return s;
}

typedef CUresult (*PgEncodeTiled)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                                  CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
PgEncodeTiled pg_encoder() {
    static const PgEncodeTiled fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q = cudaDriverEntryPointSymbolNotFound;
        return cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess ? (PgEncodeTiled)p : (PgEncodeTiled)nullptr;
    }();
    return fn;
}
// A pool as [page][key head][position][dimension] 16-bit words; a box is `rows` positions of a page and 64 dimensions (128 bytes, swizzled), or
// of whole packed heads.  Its x starts at a multiple of 128 bytes; its outer coordinates may lie outside (a page that is not there: zeros).
int pg_map(const sz_paged_cache* c, int values, int rows, CUtensorMap* map) {
    PgEncodeTiled enc = pg_encoder();
    if (!enc) return sz_fail(SZ_E_CUDA, "sz_paged_attend: the driver has no cuTensorMapEncodeTiled");
    const bool q8 = c->type == SZ_TYPE_Q8_KV;
    const cuuint64_t words = (cuuint64_t)pg_head_bytes(c->type, c->head_dim) / 2;
    const cuuint64_t dim[4] = {words, (cuuint64_t)c->page_size, (cuuint64_t)c->n_kv_head, (cuuint64_t)c->n_pages};
    const cuuint64_t stride[3] = {(cuuint64_t)c->pos_stride, (cuuint64_t)c->head_stride, (cuuint64_t)c->page_stride};
    const cuuint32_t box[4] = {q8 ? (cuuint32_t)words : 64u, (cuuint32_t)rows, 1, 1}, es[4] = {1, 1, 1, 1};
    const CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 4, (void*)(values ? c->v : c->k), dim, stride, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                           q8 ? CU_TENSOR_MAP_SWIZZLE_NONE : CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? SZ_OK : sz_fail(SZ_E_CUDA, "sz_paged_attend: cuTensorMapEncodeTiled failed (%d)", (int)r);
}

int pg_launch_attend(const PgKernels& k, const CUtensorMap* maps, int rows_box, const PgBatch& d, const PgIo& io, const PgPart& p, const char* name, cudaStream_t st) {
    const int rc = sz_allow_smem(k.fn, k.smem);
    if (rc) return rc;
    SZ_CUDA(sz_launch(name, (void (*)(CUtensorMap, CUtensorMap, PgBatch, PgIo, PgPart, int))k.fn, dim3(p.blocks), dim3(k.threads), k.smem, st, true, maps[0], maps[1], d, io, p, rows_box));
    return SZ_OK;
}

}  // namespace

extern "C" int sz_paged_scratch_bytes(const sz_paged_cache* cache, const sz_paged_batch* batch, int n_head, int64_t* bytes) {
    int rc = pg_check(cache, batch, n_head, "sz_paged_scratch_bytes");
    if (rc) return rc;
    if (!bytes) return sz_fail(SZ_E_ARG, "sz_paged_scratch_bytes: null result");
    *bytes = pg_scratch(cache, batch, n_head, 0).bytes;
    return SZ_OK;
}

extern "C" int sz_paged_status(uint64_t scratch, int init, int* code, uint64_t stream) {
    if (!scratch || (scratch & 255)) return sz_fail(SZ_E_ARG, "sz_paged_status: null or misaligned scratch");
    cudaStream_t st = (cudaStream_t)stream;
    if (init) { SZ_CUDA(cudaMemsetAsync((void*)scratch, 0, 256, st)); return SZ_OK; }
    if (!code) return sz_fail(SZ_E_ARG, "sz_paged_status: null code");
    u32 v = 0;
    SZ_CUDA(cudaMemcpyAsync(&v, (const void*)scratch, 4, cudaMemcpyDeviceToHost, st));
    SZ_CUDA(cudaStreamSynchronize(st));
    *code = (int)v;
    return v ? sz_fail(SZ_E_DEVICE, "sz_paged: the tables of a call did not fit (%s%s%s%s%s)", v & PG_E_PAGE ? " page id out of range;" : "", v & PG_E_END ? " position behind the table;" : "",
                       v & PG_E_SHARED ? " row at a shared position;" : "", v & PG_E_ROWS ? " row_start past the rows;" : "", v & PG_E_WAIT ? " a bounded wait ran out;" : "")
             : SZ_OK;
}

extern "C" int sz_paged_append(const sz_paged_cache* cache, const sz_paged_batch* batch, const sz_paged_rope* rope, int io_type, int n_head, uint64_t k, int64_t k_stride, uint64_t v,
                               int64_t v_stride, uint64_t q, int64_t q_stride, int64_t q_head_stride, uint64_t q_out, int64_t q_out_stride, uint64_t scratch, int64_t scratch_bytes,
                               uint64_t stream) {
    const char* who = "sz_paged_append";
    int rc = pg_check(cache, batch, n_head, who);
    if (rc || (rc = pg_check_tables(cache, batch, who))) return rc;
    if (io_type != SZ_TYPE_F32 && io_type != SZ_TYPE_F16 && io_type != SZ_TYPE_BF16) return sz_fail(SZ_E_TYPE, "%s: inputs of type %d", who, io_type);
    const int esz = pg_esz(io_type), hd = cache->head_dim, nkv = cache->n_kv_head;
    if (!rope || rope->dims < 0 || rope->dims > hd || rope->dims % 2 || (rope->dims && !(rope->theta > 0.0 && isfinite(rope->theta))) || !(rope->eps >= 0.f))
        return sz_fail(SZ_E_ARG, "%s: rope: an even number of dimensions up to %d, theta > 0, eps >= 0", who, hd);
    if ((rope->q_norm | rope->k_norm) & 15) return sz_fail(SZ_E_ARG, "%s: norm weights 16-byte aligned", who);
    if ((rc = pg_check_rows(k, k_stride, hd, nkv, hd, batch->rows, esz, "k", who)) || (rc = pg_check_rows(v, v_stride, hd, nkv, hd, batch->rows, esz, "v", who))) return rc;
    if (q && ((rc = pg_check_rows(q, q_stride, q_head_stride, n_head, hd, batch->rows, esz, "q", who)) ||
              (rc = pg_check_rows(q_out, q_out_stride, hd, n_head, hd, batch->rows, esz, "q_out", who))))
        return rc;
    if (q && q == q_out && (q_stride != q_out_stride || q_head_stride != hd)) return sz_fail(SZ_E_ARG, "%s: q_out may be q with the same strides only", who);
    if (!scratch || (scratch & 255) || scratch_bytes < 256) return sz_fail(SZ_E_SCRATCH, "%s: the scratch is 256-byte aligned and holds the status word at least", who);
    const PgBatch d = pg_batch(cache, batch, n_head, scratch);
    PgAppend a = {};
    a.k = (const u8*)k; a.v = (const u8*)v; a.q = (const u8*)q; a.qo = (u8*)q_out;
    a.k_stride = k_stride * esz; a.v_stride = v_stride * esz; a.q_stride = q_stride * esz; a.q_head_stride = q_head_stride * esz; a.qo_stride = q_out_stride * esz;
    a.q_norm = (const float*)rope->q_norm; a.k_norm = (const float*)rope->k_norm;
    a.nh = n_head; a.half = rope->dims / 2; a.heads = (q ? n_head : 0) + 2 * nkv; a.eps = rope->eps;
    for (int i = 0; i < a.half; i++) a.freq[i] = 1.0 / pow(rope->theta, 2.0 * i / rope->dims);
    // eight rows a block where that still gives every multiprocessor one
    const bool many = batch->rows >= 8 * PG_BLOCKS;
    const int per = many ? PG_APP : 1;
    const dim3 grid((batch->rows + per - 1) / per, many ? 1 : (a.heads + 7) / 8);
    using Kernel = void (*)(PgBatch, PgAppend);
#define SZ_PG_APP_R(CT, HD, IO) (many ? (Kernel)sz_pg_append_kernel<CT, HD, IO, PG_APP> : (Kernel)sz_pg_append_kernel<CT, HD, IO, 1>)
#define SZ_PG_APP_IO(CT, HD) (io_type == SZ_TYPE_F32 ? SZ_PG_APP_R(CT, HD, SZ_TYPE_F32) : io_type == SZ_TYPE_F16 ? SZ_PG_APP_R(CT, HD, SZ_TYPE_F16) : SZ_PG_APP_R(CT, HD, SZ_TYPE_BF16))
#define SZ_PG_APP(CT) (hd == 64 ? SZ_PG_APP_IO(CT, 64) : hd == 128 ? SZ_PG_APP_IO(CT, 128) : SZ_PG_APP_IO(CT, 256))
    const Kernel fn = cache->type == SZ_TYPE_F16 ? SZ_PG_APP(PG_F16) : cache->type == SZ_TYPE_BF16 ? SZ_PG_APP(PG_BF16) : SZ_PG_APP(PG_Q8);
#undef SZ_PG_APP_IO
#undef SZ_PG_APP_R
#undef SZ_PG_APP
    SZ_CUDA(sz_launch("paged_append", fn, grid, dim3(256), 0, (cudaStream_t)stream, true, d, a));
    return SZ_OK;
}

extern "C" int sz_paged_attend(const sz_paged_cache* cache, const sz_paged_batch* batch, int io_type, int n_head, float scale, uint64_t q, int64_t q_stride, uint64_t gate,
                               int64_t gate_stride, int64_t gate_head_stride, uint64_t out, int64_t out_stride, uint64_t lse, uint64_t scratch, int64_t scratch_bytes, uint64_t stream) {
    const char* who = "sz_paged_attend";
    int rc = pg_check(cache, batch, n_head, who);
    if (rc || (rc = pg_check_tables(cache, batch, who))) return rc;
    if (io_type != SZ_TYPE_F32 && io_type != SZ_TYPE_F16 && io_type != SZ_TYPE_BF16) return sz_fail(SZ_E_TYPE, "%s: queries of type %d", who, io_type);
    const int esz = pg_esz(io_type), hd = cache->head_dim, nkv = cache->n_kv_head, G = n_head / nkv;
    if (!isfinite(scale)) return sz_fail(SZ_E_ARG, "%s: scale is not finite", who);
    if ((rc = pg_check_rows(q, q_stride, hd, n_head, hd, batch->rows, esz, "q", who)) || (rc = pg_check_rows(out, out_stride, hd, n_head, hd, batch->rows, esz, "out", who))) return rc;
    if (gate && (rc = pg_check_rows(gate, gate_stride, gate_head_stride, n_head, hd, batch->rows, esz, "gate", who))) return rc;
    if (lse & 3) return sz_fail(SZ_E_ARG, "%s: lse misaligned", who);
    PgScratch s = pg_scratch(cache, batch, n_head, scratch);
    if (!scratch || (scratch & 255) || scratch_bytes < s.bytes) return sz_fail(SZ_E_SCRATCH, "%s: %lld bytes of scratch given, %lld needed, 256-byte aligned", who, (long long)scratch_bytes, (long long)s.bytes);
    cudaStream_t st = (cudaStream_t)stream;
    const PgBatch d = pg_batch(cache, batch, n_head, scratch);
    PgIo io = {};
    io.q = (const u8*)q; io.q_stride = q_stride * esz; io.gate = (const u8*)gate; io.gate_stride = gate_stride * esz; io.gate_head_stride = gate_head_stride * esz;
    io.out = (u8*)out; io.out_stride = out_stride * esz; io.lse = (float*)lse; io.type = io_type; io.esz = esz; io.scale_log2 = scale * 1.4426950408889634f;
    const int ct = cache->type == SZ_TYPE_F16 ? PG_F16 : cache->type == SZ_TYPE_BF16 ? PG_BF16 : PG_Q8;
    const bool wide = io_type == SZ_TYPE_F32 || (io_type == SZ_TYPE_F16 && ct != PG_F16);
    auto kernels = [&](int nqt) { return ct == PG_F16 ? pg_kernels_f16(wide, hd, nqt) : ct == PG_BF16 ? pg_kernels_bf16(wide, hd, nqt) : pg_kernels_q8(wide, hd, nqt); };
    const int64_t per_seq = (int64_t)G * ((batch->rows + batch->n_seq - 1) / batch->n_seq), all = (int64_t)G * batch->rows;
    const bool tc = pg_tc_type(cache->type) && io_type == cache->type && scale > 0.f;
    const bool tc_of[2] = {tc && all >= PG_TC_MIN, tc && per_seq >= PG_TC_MIN};
    PgKernels kern[2];
    CUtensorMap maps[2][2];              // [of 16 positions, of a tcgen05 unit][keys, values]
    const int box[2] = {cache->page_size < 16 ? cache->page_size : 16, cache->page_size < pg_tc_unit(hd) ? cache->page_size : pg_tc_unit(hd)};
    bool planned = false;
    for (int i = 0; i < 2; i++) {
        PgPart& p = s.a.p[i];
        p.on = i == PG_OWN || batch->shared_len > 0;
        p.shared = i == PG_SHARED;
        p.ways = 1;                                                        // (the merge counts parts by it, of a launch that is not there too)
        if (!p.on) continue;
        kern[i] = kernels(pg_tiles_of(i == PG_SHARED ? all : per_seq));
        p.unit = tc_of[i] ? pg_tc_unit(hd) : PG_T;
        p.ways = tc_of[i] ? 1 : kern[i].ways;
        p.tq = tc_of[i] ? pg_tc_tile(hd) : kern[i].tq;
        p.blocks = tc_of[i] ? PG_BLOCKS : PG_BLOCKS * kern[i].occ;
        p.planned = batch->n_seq + (all + p.tq - 1) / p.tq > PG_PLAN;      // (a block's copies of the tables have PG_PLAN places, over shared positions too)
        planned |= p.planned;
        const int64_t positions = p.shared ? batch->shared_len : (int64_t)batch->max_pages * cache->page_size;
        const double units = (double)((all + p.tq - 1) / p.tq + (p.shared ? 0 : batch->n_seq)) * (double)((positions + p.unit - 1) / p.unit) * nkv;
        if (units > 4294967295.0) return sz_fail(SZ_E_ARG, "%s: %d rows over %lld positions are more work than a call takes", who, batch->rows, (long long)positions);
        for (int x = 0; x < 2; x++) if ((rc = pg_map(cache, x, box[tc_of[i]], &maps[tc_of[i]][x]))) return rc;
    }
    s.a.p[PG_OWN].direct = tc_of[PG_OWN] && batch->shared_len == 0;
    if (planned) SZ_CUDA(sz_launch("paged_plan", sz_pg_plan_kernel, dim3(2), dim3(1024), 0, st, true, d, s.a));
    for (int i = 0; i < 2; i++) {
        const PgPart& p = s.a.p[i];
        if (!p.on) continue;
        const char* name = p.shared ? "paged_attend_shared" : "paged_attend";
        rc = tc_of[i] ? pg_tc_launch(cache->type == SZ_TYPE_BF16, hd, maps[1], box[1], d, io, p, name, st) : pg_launch_attend(kern[i], maps[0], box[0], d, io, p, name, st);
        if (rc) return rc;
    }
    const int64_t heads = (int64_t)batch->rows * n_head;
    const int W = heads <= 8 * PG_BLOCKS ? 8 : heads <= 16 * PG_BLOCKS ? 2 : 1;
#define SZ_PG_MERGE(HD) (W == 1 ? sz_pg_merge_kernel<HD, 1> : W == 2 ? sz_pg_merge_kernel<HD, 2> : sz_pg_merge_kernel<HD, 8>)
    auto* merge = hd == 64 ? SZ_PG_MERGE(64) : hd == 128 ? SZ_PG_MERGE(128) : SZ_PG_MERGE(256);
#undef SZ_PG_MERGE
    SZ_CUDA(sz_launch("paged_merge", merge, dim3(batch->rows, (n_head * W + 7) / 8), dim3(256), 0, st, true, d, io, s.a));
    return SZ_OK;
}
