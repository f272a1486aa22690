// A cache in pages: what the append, attention and merge kernels share, and the attention kernel for any number of queries a sequence.
//
// Attention of a query vector (row, head) over the positions it may see: s_t = scale q . k_t, o = sum_t e^(s_t) v_t / sum_t e^(s_t).  A
// sum over positions splits into parts that are joined exactly: a part is (m, l, O) = (largest score, sum of 2^(s - m), sum of 2^(s - m) v),
// scores in units of log 2; two parts join with the factors 2^(m_i - M), M the larger m.
//
// Work.  The query vectors of a sequence that share a key head (its rows times the G heads of the group) are cut into tiles of TQ; an ITEM
// is a tile, a key head and the positions that the tile's last row sees; a UNIT is 64 positions of an item.  The units of all items in a row
// are shared out evenly to as many blocks as the GPU holds at once, so that ragged contexts leave no block idle and one long conversation
// fills the GPU; an item cut by a block's boundary leaves parts, which sz_pg_merge_kernel joins in the order of the positions.  The plan (units
// before every item) is made by every block from the lengths in device memory: nothing about a step is fixed when a graph is captured.
// The positions that all sequences share are items of their own, whose tiles run over the rows of the whole batch (SHARED).
#pragma once
#include <cuda.h>   // CUtensorMap
#include "sz_common.cuh"
#include "sz_dense.cuh"

constexpr int PG_T = 64;             // positions a unit
constexpr int PG_PLAN = 256;         // sequences and tiles that a block plans for itself; above, sz_pg_plan_kernel does once
constexpr int PG_MAX_SEQ = 4096;
enum { PG_F16 = 0, PG_BF16 = 1, PG_Q8 = 2 };
enum { PG_E_PAGE = 1, PG_E_END = 2, PG_E_SHARED = 4, PG_E_ROWS = 8, PG_E_WAIT = 16 };

struct PgBatch {                     // the tables of a call, as the kernels read them
    const u8 *k, *v;
    long long page_stride, head_stride, pos_stride;
    const int32_t *pages, *row_start, *lens, *shared_pages;
    int n_seq, rows, max_pages, shared_len, n_pages, ps_log2, nkv, G;
    u32* err;
};
struct PgIo {                        // rows of queries and outputs; strides in bytes
    const u8* q;
    long long q_stride;
    const u8* gate;
    long long gate_stride, gate_head_stride;
    u8* out;
    long long out_stride;
    float* lse;
    int type, esz;                   // SZ_TYPE_F32 / F16 / BF16, bytes an element
    float scale_log2;                // scale / log 2
};
// One attention launch's plan and parts.  Block i of `blocks` takes units [i U / blocks, (i + 1) U / blocks) of U.  Parts: slot 2 i is what
// block i adds to an item that an earlier block began, slot 2 i + 1 what it begins and a later one goes on with; an item that one block
// does alone lies by row and head.
struct PgPart {
    u32 *tiles, *units;              // [n_seq + 1] tiles before a sequence, [tiles + 1] units (of one key head) before a tile
    float* o;                        // [slot][tq][ways][hd]
    float2* ml;                      // [slot][tq][ways]
    float* row_o;                    // [row][head][ways][hd]: an item that one block did alone
    float2* row_ml;                  // [row][head][ways]
    int ways;                        // parts that a block leaves of an item
    int blocks, tq, shared, planned; // planned: the plan was made by sz_pg_plan_kernel
    int unit;                        // positions a unit: PG_T, or the tcgen05 kernel's
    int direct;                      // (tcgen05 kernel) an item that one block does alone goes straight to the output
    int on;
};

__device__ __forceinline__ int pg_row(const PgBatch& d, int i) { return min(max(__ldg(d.row_start + i), 0), d.rows); }
// Where the own positions of sequence i's last row that is there end: before lens[i] where row_start goes on behind the rows of the call.
__device__ __forceinline__ int pg_end(const PgBatch& d, int i) {
    const long long over = max(__ldg(d.row_start + i + 1), d.rows) - d.rows;
    return (int)max(0ll, (long long)__ldg(d.lens + i) - d.shared_len - over);
}
// Of a sequence with m rows whose own positions end at `end` (exclusive), tile t of tq vectors: where what its last row sees ends ..
__device__ __forceinline__ int pg_room(const PgBatch& d) { return (int)min((long long)d.max_pages << d.ps_log2, 0x7fffffc0ll); }
__device__ __forceinline__ int pg_tile_end(const PgBatch& d, int m, long long end, int t, int tq) {
    const int last = (min((t + 1) * tq, m * d.G) - 1) / d.G;
    return (int)max(0ll, min(end - (m - 1 - last), (long long)pg_room(d)));
}
// U units over blocks: the first U % blocks have one more than the others.  First unit of block i, and which block has unit u.
struct PgShare { u32 each, more; };
__device__ __forceinline__ PgShare pg_share(u32 U, int blocks) { PgShare s; s.each = U / (u32)blocks; s.more = U - s.each * (u32)blocks; return s; }
__device__ __forceinline__ u32 pg_first(const PgShare& s, int i) { return (u32)i * s.each + min((u32)i, s.more); }
__device__ __forceinline__ int pg_block_of(const PgShare& s, u32 u) {
    const u32 line = s.more * (s.each + 1);
    return (int)(u < line ? u / (s.each + 1) : s.more + (u - line) / s.each);
}

__device__ __forceinline__ float pg_ex2(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
// two neighbouring elements at p
__device__ __forceinline__ float2 pg_load2(const u8* p, int type) {
    if (type == SZ_TYPE_F32) return *(const float2*)p;
    const u32 w = *(const u32*)p;
    if (type == SZ_TYPE_F16) return __half22float2(*(const __half2*)&w);
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
__device__ __forceinline__ u32 pg_pack_bf16(float a, float b) {      // round to nearest even, as the type's own conversion does
    u32 r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    return r;
}
__device__ __forceinline__ u32 pg_pack_f16(float a, float b) { const __half2 h = __floats2half2_rn(a, b); return *(const u32*)&h; }
__device__ __forceinline__ void pg_store2(u8* p, int type, float a, float b) {
    if (type == SZ_TYPE_F32) *(float2*)p = make_float2(a, b);
    else *(u32*)p = type == SZ_TYPE_F16 ? pg_pack_f16(a, b) : pg_pack_bf16(a, b);
}

// ---- the plan: by all NTH threads of a block, into shared or global memory -----------------------------------------------------------------
template <int NTH>
__device__ u32 pg_scan(u32 v, u32& total, u32* sm) {                // exclusive prefix over the block's threads
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    u32 x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const u32 y = __shfl_up_sync(0xffffffffu, x, o); if (lane >= o) x += y; }
    __syncthreads();
    if (lane == 31) sm[warp] = x;
    __syncthreads();
    u32 before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < NTH / 32; w++) { const u32 s = sm[w]; if (w < warp) before += s; total += s; }
    return before + x - v;
}
// tiles[0 .. n_seq], units[0 .. tiles[n_seq]]; returns the number of tiles.  (SHARED: one tile list over the rows of all sequences.)  rows, ends: copies of the
// tables for the block, row_start and the own positions' ends (null: none).
template <int NTH>
__device__ int pg_plan(const PgBatch& d, int shared, int unit, int tq, u32* tiles, u32* units, u32* sm, int* rows, int* ends) {
    if (rows)
        for (int b = threadIdx.x; b <= d.n_seq; b += NTH) { rows[b] = pg_row(d, b); ends[b] = b < d.n_seq ? pg_end(d, b) : 0; }
    if (shared) {
        const int vec = (pg_row(d, d.n_seq) - pg_row(d, 0)) * d.G, E = max(0, (vec + tq - 1) / tq);
        const u32 un = (u32)((d.shared_len + unit - 1) / unit);
        for (int e = threadIdx.x; e <= E; e += NTH) units[e] = (u32)e * un;
        if (threadIdx.x == 0) tiles[0] = 0;
        __syncthreads();
        return E;
    }
    u32 carry = 0, total;
    int falls = 0;                      // a row_start that descends: more tiles than the tables have room for
    for (int b0 = 0; b0 < d.n_seq; b0 += NTH) {
        const int b = b0 + threadIdx.x;
        falls |= b < d.n_seq && pg_row(d, b + 1) < pg_row(d, b);
        const u32 n = b < d.n_seq ? (u32)((max(pg_row(d, b + 1) - pg_row(d, b), 0) * d.G + tq - 1) / tq) : 0u;
        const u32 at = pg_scan<NTH>(n, total, sm);
        if (b < d.n_seq) tiles[b] = carry + at;
        carry += total;
    }
    if (__syncthreads_or(falls)) {      // nothing is done then
        for (int b = threadIdx.x; b <= d.n_seq; b += NTH) tiles[b] = 0;
        if (threadIdx.x == 0) { units[0] = 0; atomicOr(d.err, PG_E_ROWS); }
        __syncthreads();
        return 0;
    }
    const int E = (int)carry;
    if (threadIdx.x == 0) tiles[d.n_seq] = carry;
    __syncthreads();
    carry = 0;
    for (int e0 = 0; e0 < E; e0 += NTH) {
        const int e = e0 + threadIdx.x;
        u32 n = 0;
        if (e < E) {
            int lo = 0, hi = d.n_seq - 1;                           // the last sequence whose tiles begin at or before e
            while (lo < hi) { const int mid = (lo + hi + 1) >> 1; if (tiles[mid] <= (u32)e) lo = mid; else hi = mid - 1; }
            const int m = pg_row(d, lo + 1) - pg_row(d, lo);
            n = (u32)((pg_tile_end(d, m, pg_end(d, lo), e - (int)tiles[lo], tq) + unit - 1) / unit);
        }
        const u32 at = pg_scan<NTH>(n, total, sm);
        if (e < E) units[e] = carry + at;
        carry += total;
    }
    if (threadIdx.x == 0) units[E] = carry;
    __syncthreads();
    return E;
}

// ---- the attention kernel ---------------------------------------------------------------------------------------------------------------------
// A block has NQT tiles of 16 query vectors (TQ = 16 NQT) and takes its units one after the other.  Warps: NQT tiles x WAYS shares of a unit's
// positions; a warp keeps its tile's (m, l, O) for its positions in registers from unit to unit, so nothing but keys, values and queries
// goes through shared memory, and with one tile (decoding) warps load their own positions and meet only where an item begins or ends.
// Keys and values come by tiled TMA, a box a page, through a ring of half units (64 keys, then their 64 values), 16-bit types with the 128-byte swizzle
// (chunk c of row r at c ^ (r & 7)), so that ldmatrix meets no bank twice; packed rows of 272 / 144 / 80 bytes spread by themselves.
// (Copies of 16 bytes a lane, cp.async, took a third of the issue slots and most of the registers.)
// Both products run on mma.sync m16n8k16 with f32 sums.  (tcgen05 wants 64 rows and more: decoding has G queries a key head, and the
// kernel waits for memory, not for the tensor pipe.)  Rounding: queries and weights enter as sums of QN and PN pieces of the cache's type -
//   WIDE (f32 queries, or f16 ones over a packed or bf16 cache): f16 2 pieces (22 bits), bf16 3 (24), so that f32 results keep f32's accuracy;
//   else the queries are exact in one piece, weights take two (f16 22 bits, bf16 16), one over a packed cache for bf16 results (11 bits, a
//   quarter of the step that the result itself is rounded to).
// f16 pieces are kept in range: queries are divided by a power of two near their largest element, weights are 2^15 times themselves (so
// that small ones do not run into f16's subnormals), and both are taken back in f32.  A packed value's scale goes into the weight (times a
// power of two that follows the scales a row sees, csc), a packed key's into the 32-dimension partial scores in f32: codes themselves are exact in f16.
// Measured: 64 sequences, 163 rows of 32 heads of 128 on 8, bf16, contexts of 3,000 to 15,000: 406 us (360 are the bytes at the measured copy rate: memory
// bounds it).  Few rows wait for one thing after the other instead: plan, pages, keys, products, values, products.  Four rows of 16 heads of 256 on 2
// over 24,576 packed positions 56 us, 101 such rows behind 9,599 shared ones 277: 12 instructions (codes to f16, scales, pieces of weights) for
// every matrix instruction, on the 8 warps that 128 registers of sums each leave room for (issue slots 41 %).
template <int CT, bool WIDE, int HD, int NQT>
struct PgCfg {
    static constexpr int NW = NQT == 1 ? 4 : 8, NTH = 32 * NW, WAYS = NW / NQT, SG = PG_T / 16 / WAYS, TQ = 16 * NQT;
    static constexpr int HB = CT == PG_Q8 ? HD + ((HD / 32 * 2 + 15) & ~15) : 2 * HD, HALF = PG_T * HB;
    static constexpr int BOXES = CT == PG_Q8 ? 1 : HD / 64;      // TMA boxes a row: 64 dimensions of 16 bits, or a packed head
    static constexpr int QN = CT == PG_BF16 ? (WIDE ? 3 : 1) : (WIDE ? 2 : 1);
    static constexpr int PN = CT == PG_BF16 ? (WIDE ? 3 : 2) : CT == PG_F16 ? 2 : (WIDE ? 2 : 1);
    static constexpr int KS = HD / 16, NT = HD / 8;
    static constexpr int QB = QN * NQT * KS * 512;
    static constexpr int MISC = 4 * (PG_PLAN + 1) * 4 + 8 * 4 + TQ * 8 + 8 * 8 + 8 * 4 * 8 + 64;
    static constexpr int OCC = NQT > 1 ? 1 : HD == 256 ? (CT == PG_Q8 || QN == 1 ? 2 : 1) : HD == 128 ? 3 : 4;
    static constexpr int ROOM = (227 * 1024 / OCC - 1024 - 1024 - QB - MISC) / HALF;      // (a block's own kilobyte, and one to align)
    static constexpr int NR = ROOM > 6 ? 6 : ROOM;      // halves in the ring
    static_assert(NR >= 3, "the ring needs three halves");
    static constexpr int SMEM = 1024 + NR * HALF + QB + MISC;      // (1,024 to align)
    static constexpr float PSCALE = CT == PG_BF16 ? 0.f : 15.f;
};

template <int CT>
__device__ __forceinline__ void pg_mma(float* c, const u32* a, u32 b0, u32 b1) {
    if (CT == PG_BF16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else sz_mma16816_z(c, a, b0, b1);
}
template <int CT>
__device__ __forceinline__ void pg_mma_first(float* c, const u32* a, u32 b0, u32 b1) {      // sums that begin at 0 (f16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ float pg_half(u32 w, int i) { const __half2 h = *(const __half2*)&w; return i ? __high2float(h) : __low2float(h); }
template <int CT>
__device__ __forceinline__ u32 pg_pack(float a, float b) { return CT == PG_BF16 ? pg_pack_bf16(a, b) : pg_pack_f16(a, b); }
template <int CT>
__device__ __forceinline__ float2 pg_unpack(u32 w) {
    if (CT == PG_BF16) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
    return __half22float2(*(const __half2*)&w);
}
// a pair as N pieces: the first the pair rounded, each further one what is left, rounded
template <int CT, int N>
__device__ __forceinline__ void pg_pieces(float a, float b, u32* w) {
#pragma unroll
    for (int i = 0; i < N; i++) {
        w[i] = pg_pack<CT>(a, b);
        if (i + 1 < N) { const float2 f = pg_unpack<CT>(w[i]); a -= f.x; b -= f.y; }
    }
}
__device__ __forceinline__ void pg_ldsm4(u32* r, u32 addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void pg_ldsm4t(u32* r, u32 addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}

struct PgItem { int e, h, i, n, b, t, end; };       // tile, key head, unit and units of the item; its sequence, tile of it, end of its positions

template <int CT, bool WIDE, int HD, int NQT>
__global__ void __launch_bounds__(PgCfg<CT, WIDE, HD, NQT>::NTH, PgCfg<CT, WIDE, HD, NQT>::OCC)
sz_pg_attend_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap, const __grid_constant__ PgBatch d, const __grid_constant__ PgIo io,
                    const __grid_constant__ PgPart pt, int rows_box) {
    using C = PgCfg<CT, WIDE, HD, NQT>;
    extern __shared__ __align__(16) u8 raw[];
    u8* const ring = raw + (1024 - (sz_smem_addr(raw) & 1023)) % 1024;      // [half][64-dimension block][64 positions][128 bytes], or [half][64 positions][packed head]
    u8* const qm = ring + C::NR * C::HALF;                // query pieces as A fragments
    u32* const s_tiles = (u32*)(qm + C::QB);
    u32* const s_units = s_tiles + PG_PLAN + 1;
    int* const s_rows = (int*)(s_units + PG_PLAN + 1);    // row_start and own positions' ends, where the block planned for itself
    int* const s_ends = s_rows + PG_PLAN + 1;
    u32* const s_scan = (u32*)(s_ends + PG_PLAN + 1);
    float* const s_fac = (float*)(s_scan + 8);            // [TQ] what a vector's raw scores are multiplied by
    int* const s_lim = (int*)(s_fac + C::TQ);             // [TQ] positions a vector sees
    u64* const s_full = (u64*)(((uintptr_t)(s_lim + C::TQ) + 7) & ~(uintptr_t)7);      // [ring half] (one tile: [ring half][warp]) the copies have arrived
    u16* const s_ok = (u16*)(s_full + 8 * 4);             // [ring half][16 positions] which of the positions are there
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g8 = lane >> 2, q4 = lane & 3;
    const int qt = warp % NQT, way = warp / NQT;
    if (tid < C::NR * 4) sz_mbar_init(&s_full[tid], NQT == 1 ? 1 : 4);
    if (tid < C::NR * 4) sz_mbar_fence_init();
    __syncthreads();
    sz_pdl_wait();
    const u32 *tiles = s_tiles, *units = s_units;
    int E;
    if (pt.planned) {
        tiles = pt.tiles; units = pt.units;
        E = pt.shared ? max(0, ((pg_row(d, d.n_seq) - pg_row(d, 0)) * d.G + C::TQ - 1) / C::TQ) : (int)tiles[d.n_seq];
    } else {
        E = pg_plan<C::NTH>(d, pt.shared, PG_T, C::TQ, s_tiles, s_units, s_scan, s_rows, s_ends);
        if (blockIdx.x == 0) {                            // for the merge
            if (!pt.shared) for (int i = tid; i <= d.n_seq; i += C::NTH) pt.tiles[i] = s_tiles[i];
            for (int i = tid; i <= E; i += C::NTH) pt.units[i] = s_units[i];
        }
    }
    if (blockIdx.x == 0 && !pt.shared) {                  // what the lengths ask for that is not there
        for (int b = tid; b < d.n_seq; b += C::NTH)
            if (pg_row(d, b + 1) > pg_row(d, b) && (long long)__ldg(d.lens + b) - d.shared_len > ((long long)d.max_pages << d.ps_log2)) atomicOr(d.err, PG_E_END);
        if (tid == 0 && __ldg(d.row_start + d.n_seq) > d.rows) atomicOr(d.err, PG_E_ROWS);
    }
    const u32 U = units[E] * (u32)d.nkv;
    const int blocks = (int)min((u32)pt.blocks, U);
    if ((int)blockIdx.x >= blocks) return;                // (blocks that leave count as having triggered)
    const PgShare share = pg_share(U, blocks);
    const u32 u0 = pg_first(share, blockIdx.x), u1 = pg_first(share, blockIdx.x + 1);
    const int room = pg_room(d);
    auto row_of = [&](int b) { return pt.planned ? pg_row(d, b) : s_rows[b]; };
    auto end_of = [&](int b) { return (long long)(pt.planned ? pg_end(d, b) : s_ends[b]); };

    auto locate = [&](u32 u) {
        PgItem it;
        const u32 un = u / (u32)d.nkv;                    // (an entry's units times nkv: the entry of u is that of u / nkv)
        int lo = 0, hi = E - 1;
        while (lo < hi) { const int mid = (lo + hi + 1) >> 1; if (units[mid] <= un) lo = mid; else hi = mid - 1; }
        it.e = lo;
        it.n = (int)(units[lo + 1] - units[lo]);
        const u32 rem = u - units[lo] * (u32)d.nkv;
        it.h = (int)(rem / (u32)it.n);
        it.i = (int)(rem - (u32)it.h * (u32)it.n);
        if (pt.shared) { it.b = 0; it.t = lo; it.end = d.shared_len; return it; }
        int bl = 0, bh = d.n_seq - 1;
        while (bl < bh) { const int mid = (bl + bh + 1) >> 1; if (tiles[mid] <= (u32)lo) bl = mid; else bh = mid - 1; }
        it.b = bl;
        it.t = lo - (int)tiles[bl];
        it.end = pg_tile_end(d, row_of(bl + 1) - row_of(bl), end_of(bl), it.t, C::TQ);
        return it;
    };
    // ---- loads: step s of the block is the keys (even) or values (odd) of unit u0 + s / 2.  Warp w < 4 asks for positions 16 w .. of a half, a
    // box a page and 64 dimensions; a lane has a box.  With one tile a warp's own positions are all it reads.
    PgItem ld = locate(u0);
    u32 lu = u0;
    const int piece = lane / C::BOXES, boxes = 16 / rows_box * C::BOXES;
    int page = -1;                                        // the lane's page of the unit to load next
    auto peek = [&]() {
        const int c = ld.i * PG_T + warp * 16 + piece * rows_box;
        page = -1;
        if (warp < 4 && lane < boxes && c < ld.end) page = __ldg((pt.shared ? d.shared_pages : d.pages + (size_t)ld.b * d.max_pages) + (c >> d.ps_log2));
    };
    int lslot = 0, steps_left = (int)(2 * (u1 - u0)), at_page = 0;
    auto issue = [&](int which) {
        if (steps_left <= 0) return;
        steps_left--;
        if (warp < 4) {
            u64* const bar = &s_full[NQT == 1 ? lslot * 4 + warp : lslot];
            const int c = ld.i * PG_T + warp * 16 + piece * rows_box;
            if (which == 0) {
                const bool there = lane < boxes && c < ld.end, ok = there && (u32)page < (u32)d.n_pages;
                if (there && !ok) atomicOr(d.err, PG_E_PAGE);
                const u32 bits = __ballot_sync(0xffffffffu, ok);
                at_page = ok ? page : d.n_pages;          // (outside the map: zeros)
                if (lane == 0) {
                    u32 m = (bits & 1u) ? (1u << rows_box) - 1u : 0u;
                    if (rows_box < 16 && ((bits >> C::BOXES) & 1u)) m |= 0xff00u;
                    s_ok[lslot * 4 + warp] = (u16)m;
                }
            }
            if (lane == 0) sz_mbar_expect_tx(bar, (u32)(16 * C::HB));
            __syncwarp();
            // (under a predicate, not a branch: what comes next, ldmatrix and mma.sync, is for the whole warp)
            u8* const dst = CT == PG_Q8 ? ring + (size_t)lslot * C::HALF + (size_t)(warp * 16 + piece * rows_box) * C::HB
                                        : ring + (size_t)lslot * C::HALF + (size_t)(lane % C::BOXES) * PG_T * 128 + (size_t)(warp * 16 + piece * rows_box) * 128;
            asm volatile("{ .reg .pred q; setp.ne.b32 q, %7, 0;\n"
                         "  @q cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6]; }" ::"r"(sz_smem_addr(dst)),
                         "l"(which ? &vmap : &kmap), "r"(lane % C::BOXES * 64), "r"(c & ((1 << d.ps_log2) - 1)), "r"(ld.h), "r"(at_page), "r"(sz_smem_addr(bar)), "r"((u32)(lane < boxes))
                         : "memory");
        }
        if (which && ++lu < u1) {                         // on to the next unit
            if (++ld.i == ld.n) ld = locate(lu);
            peek();
        }
        lslot = lslot + 1 == C::NR ? 0 : lslot + 1;
    };
    peek();
#pragma unroll 1
    for (int s = 0; s < C::NR - 1; s++) issue(s & 1);
    int ipar = (C::NR - 1) & 1;                           // which of the two the next issue loads
    bool dead = false;                                    // a wait ran out: no further ones
    u32 cphase = 0;
    auto arrived = [&](int slot) {                        // .. at the consumers, before the half that was used last is filled again
        if (!dead && !sz_mbar_wait_warp(&s_full[NQT == 1 ? slot * 4 + warp : slot], cphase)) {
            dead = true;
            if (lane == 0) atomicOr(d.err, PG_E_WAIT);
            steps_left = -1 - steps_left;                 // nothing more is asked for
        }
        if (NQT > 1) __syncthreads();
    };

    float o[C::NT][4], p[C::SG][8], m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f, csc0 = 1.f, csc1 = 1.f;
    bool fresh = true;                                    // the maxima moved since the values' scales were chosen
    int lim0 = 0, lim1 = 0;
    float f0 = 0.f, f1 = 0.f;
    int cslot = 0;
    const int pw = way * 16 * C::SG;                      // the warp's first position of a unit
    const u32 rbase = sz_smem_addr(ring);

    PgItem it = locate(u0);
#pragma unroll 1
    for (u32 u = u0; u < u1; u++) {
        if (u != u0 && ++it.i == it.n) it = locate(u);
        if (u == u0 || it.i == 0) {                       // ---- an item begins: its queries
            __syncthreads();
            const int r0 = row_of(it.b), m = (pt.shared ? row_of(d.n_seq) : row_of(it.b + 1)) - r0;
            const long long oend = end_of(it.b);
#pragma unroll 4
            for (int v = warp; v < C::TQ; v += C::NW) {
                const int vec = it.t * C::TQ + v, row = vec / d.G, head = it.h * d.G + vec % d.G;
                float2 x[HD / 64];
                float big = 0.f;
#pragma unroll
                for (int i = 0; i < HD / 64; i++) {
                    x[i] = row < m ? pg_load2(io.q + (long long)(r0 + row) * io.q_stride + (long long)(head * HD + 2 * (lane + 32 * i)) * io.esz, io.type) : make_float2(0.f, 0.f);
                    big = fmaxf(big, fmaxf(fabsf(x[i].x), fabsf(x[i].y)));
                }
                float down = 1.f, fac = io.scale_log2;
                if (CT != PG_BF16) {                      // by a power of two to below 1
#pragma unroll
                    for (int s = 16; s > 0; s >>= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, s));
                    const int ex = min(max((int)((__float_as_uint(big) >> 23) & 255u) - 126, -100), 126);
                    down = __uint_as_float((u32)(127 - ex) << 23);
                    fac = io.scale_log2 * __uint_as_float((u32)(127 + ex) << 23);
                }
#pragma unroll
                for (int i = 0; i < HD / 64; i++) {
                    const int dm = 2 * (lane + 32 * i), ks = dm / 16, dd = dm % 16;
                    // the pair's lane and register in the A fragment of k-step ks.  16-bit keys: k slots are the dimensions in order; packed
                    // ones: a lane's four slots are four neighbouring dimensions, a word of codes
                    const int ql = CT == PG_Q8 ? dd / 4 : (dd % 8) / 2, rg = (CT == PG_Q8 ? (dd % 4) / 2 : dd / 8) * 2 + ((v & 15) >> 3);
                    u32 w[C::QN];
                    pg_pieces<CT, C::QN>(x[i].x * down, x[i].y * down, w);
#pragma unroll
                    for (int k = 0; k < C::QN; k++)
                        *(u32*)(qm + (((size_t)(k * NQT + (v >> 4)) * C::KS + ks) * 32 + (v & 7) * 4 + ql) * 16 + rg * 4) = w[k];
                }
                if (lane == 0) {
                    s_fac[v] = fac;
                    // (a vector that is not there sees everything: what becomes of it matters to nobody, and hiding costs, below)
                    s_lim[v] = row >= m ? 0x7fffffff : pt.shared ? d.shared_len : (int)max(0ll, min(oend - (m - 1 - row), (long long)room));
                }
            }
            __syncthreads();
            lim0 = s_lim[qt * 16 + g8]; lim1 = s_lim[qt * 16 + g8 + 8];
            f0 = s_fac[qt * 16 + g8]; f1 = s_fac[qt * 16 + g8 + 8];
#pragma unroll
            for (int b = 0; b < C::NT; b++) { o[b][0] = 0.f; o[b][1] = 0.f; o[b][2] = 0.f; o[b][3] = 0.f; }
            m0 = m1 = -INFINITY; l0 = l1 = 0.f; csc0 = csc1 = 1.f; fresh = true;
        }
        // ---- the unit's keys: scores, maxima, weights
        arrived(cslot);
        issue(ipar); ipar ^= 1;
        const int c0 = it.i * PG_T + pw;
        const u32 kb = rbase + (u32)(cslot * C::HALF);
        u32 okb;                                          // 16 SG bits from the warp's first position on
        if (C::SG == 1) okb = s_ok[cslot * 4 + way]; else okb = *(const u32*)(s_ok + cslot * 4 + 2 * way);
        float s[C::SG][2][4];
#pragma unroll
        for (int g = 0; g < C::SG; g++)
#pragma unroll
            for (int n = 0; n < 2; n++) { s[g][n][0] = 0.f; s[g][n][1] = 0.f; s[g][n][2] = 0.f; s[g][n][3] = 0.f; }
        if constexpr (CT != PG_Q8) {
            const int r = pw + ((lane >> 4) << 3) + (lane & 7);
            const u32 ra = kb + (u32)(r * 128);
            const int cx = (lane >> 3) & 1, sw = r & 7;
#pragma unroll
            for (int ks = 0; ks < C::KS; ks++) {
                u32 b[C::SG][4];
#pragma unroll
                for (int g = 0; g < C::SG; g++) pg_ldsm4(b[g], ra + (u32)((ks >> 2) * PG_T * 128 + g * 16 * 128 + (((2 * (ks & 3) + cx) ^ sw) << 4)));
#pragma unroll
                for (int k = 0; k < C::QN; k++) {
                    const uint4 q = *(const uint4*)(qm + (((size_t)(k * NQT + qt) * C::KS + ks) * 32 + lane) * 16);
                    const u32 a[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
                    for (int g = 0; g < C::SG; g++) { pg_mma<CT>(s[g][0], a, b[g][0], b[g][1]); pg_mma<CT>(s[g][1], a, b[g][2], b[g][3]); }
                }
            }
        } else {
            const u8* kr = ring + (size_t)cslot * C::HALF + (size_t)pw * C::HB;
#pragma unroll 1
            for (int g2 = 0; g2 < HD / 64; g2++) {        // two groups of 32 dimensions: their scales are read together
                u32 sc[C::SG][2][2];
#pragma unroll
                for (int g = 0; g < C::SG; g++)
#pragma unroll
                    for (int n = 0; n < 2; n++) {
                        const u8* sp = kr + (size_t)(16 * g + 8 * n + 2 * q4) * C::HB + HD + 4 * g2;
                        sc[g][n][0] = *(const u32*)sp; sc[g][n][1] = *(const u32*)(sp + C::HB);
                    }
#pragma unroll
                for (int hf = 0; hf < 2; hf++) {
                    const int gr = 2 * g2 + hf;
                    float tt[C::SG][2][4];
                    u32 b0[2][C::SG][2], b1[2][C::SG][2];
#pragma unroll
                    for (int kk = 0; kk < 2; kk++)
#pragma unroll
                        for (int g = 0; g < C::SG; g++)
#pragma unroll
                            for (int n = 0; n < 2; n++) sz_q8_quad(*(const u32*)(kr + (size_t)(16 * g + 8 * n + g8) * C::HB + (2 * gr + kk) * 16 + 4 * q4), b0[kk][g][n], b1[kk][g][n]);
#pragma unroll
                    for (int kk = 0; kk < 2; kk++)
#pragma unroll
                        for (int k = 0; k < C::QN; k++) {
                            const uint4 q = *(const uint4*)(qm + (((size_t)(k * NQT + qt) * C::KS + 2 * gr + kk) * 32 + lane) * 16);
                            const u32 a[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
                            for (int g = 0; g < C::SG; g++)
#pragma unroll
                                for (int n = 0; n < 2; n++) {
                                    if (kk == 0 && k == 0) pg_mma_first<CT>(tt[g][n], a, b0[kk][g][n], b1[kk][g][n]);
                                    else pg_mma<CT>(tt[g][n], a, b0[kk][g][n], b1[kk][g][n]);
                                }
                        }
#pragma unroll
                    for (int g = 0; g < C::SG; g++)
#pragma unroll
                        for (int n = 0; n < 2; n++)
#pragma unroll
                            for (int c = 0; c < 4; c++) s[g][n][c] = fmaf(pg_half(sc[g][n][c & 1], hf), tt[g][n][c], s[g][n][c]);
                }
            }
        }
        bool hidden = false;                              // a position that is there, but not for this lane's rows
        bool part = false;                                // one that is not there, or not for them
        float x0 = -INFINITY, x1 = -INFINITY;
#pragma unroll
        for (int g = 0; g < C::SG; g++)
#pragma unroll
            for (int n = 0; n < 2; n++)
#pragma unroll
                for (int c = 0; c < 2; c++) {
                    const int pi = 16 * g + 8 * n + 2 * q4 + c;
                    const bool ok = (okb >> pi) & 1u, a = ok && c0 + pi < lim0, b = ok && c0 + pi < lim1;
                    s[g][n][c] = a ? s[g][n][c] * f0 : -INFINITY;
                    s[g][n][2 + c] = b ? s[g][n][2 + c] * f1 : -INFINITY;
                    hidden |= ok && c0 + pi < it.end && !(a && b);
                    part |= !(a && b);
                    x0 = fmaxf(x0, s[g][n][c]); x1 = fmaxf(x1, s[g][n][2 + c]);
                }
#pragma unroll
        for (int k = 1; k < 4; k <<= 1) { x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, k)); x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, k)); }
        if (__any_sync(0xffffffffu, x0 > m0 || x1 > m1)) {
            const float n0 = fmaxf(m0, x0), n1 = fmaxf(m1, x1);
            const float a0 = m0 == -INFINITY ? 0.f : pg_ex2(m0 - n0), a1 = m1 == -INFINITY ? 0.f : pg_ex2(m1 - n1);   // (nothing summed yet: 0 times 0)
#pragma unroll
            for (int b = 0; b < C::NT; b++) { o[b][0] *= a0; o[b][1] *= a0; o[b][2] *= a1; o[b][3] *= a1; }
            l0 *= a0; l1 *= a1; m0 = n0; m1 = n1;
            fresh = true;
        }
        {
            const float e0 = (m0 == -INFINITY ? 0.f : m0) - C::PSCALE, e1 = (m1 == -INFINITY ? 0.f : m1) - C::PSCALE;
#pragma unroll
            for (int g = 0; g < C::SG; g++)
#pragma unroll
                for (int n = 0; n < 2; n++)
#pragma unroll
                    for (int c = 0; c < 2; c++) {
                        p[g][4 * n + c] = pg_ex2(s[g][n][c] - e0); p[g][4 * n + 2 + c] = pg_ex2(s[g][n][2 + c] - e1);
                        l0 += p[g][4 * n + c]; l1 += p[g][4 * n + 2 + c];
                    }
        }
        if (++cslot == C::NR) { cslot = 0; cphase ^= 1; }
        // ---- its values: O += P V
        arrived(cslot);
        issue(ipar); ipar ^= 1;
        const u32 vb = rbase + (u32)(cslot * C::HALF);
        if constexpr (CT != PG_Q8) {
            if ((it.i + 1) * PG_T > it.end) {             // behind the sequence's end its last page may hold anything: 0 times NaN would be NaN
                u8* const half = ring + (size_t)cslot * C::HALF;
                const int f = max(it.end - it.i * PG_T, NQT == 1 ? 16 * warp : 0), n = (NQT == 1 ? 16 * (warp + 1) : PG_T) - f;
                for (int x = NQT == 1 ? lane : tid; x < n * HD / 8; x += NQT == 1 ? 32 : C::NTH)      // (the order of a row's 16 bytes does not matter)
                    *(uint4*)(half + (size_t)(x / 8 % (HD / 64)) * PG_T * 128 + (size_t)(f + x / (HD / 8)) * 128 + x % 8 * 16) = make_uint4(0, 0, 0, 0);
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");                           // (the next copy into this half comes after it)
                if (NQT == 1) __syncwarp(); else __syncthreads();
            }
            const int r = pw + (lane & 15), sw = r & 7, cx = lane >> 4;
            const u32 ra = vb + (u32)(r * 128);
            bool plain = true;
            if (__any_sync(0xffffffffu, hidden)) {
                // 0 times an infinity or NaN in a row's hidden positions would reach its sums: looked for where some row hides some
                u32 bad = 0;
#pragma unroll 4
                for (int b2 = 0; b2 < HD / 16; b2++)
#pragma unroll
                    for (int g = 0; g < C::SG; g++) {
                        u32 w[4];
                        pg_ldsm4t(w, ra + (u32)((b2 >> 2) * PG_T * 128 + g * 16 * 128 + (((2 * (b2 & 3) + cx) ^ sw) << 4)));
                        constexpr u32 X = CT == PG_BF16 ? 0x7f80u : 0x7c00u;
#pragma unroll
                        for (int k = 0; k < 4; k++) bad |= (u32)((w[k] & X) == X) | (u32)((w[k] & (X << 16)) == (X << 16));
                    }
                plain = !__any_sync(0xffffffffu, bad != 0);
            }
            if (plain) {
#pragma unroll
                for (int g = 0; g < C::SG; g++) {
                    u32 af[C::PN][4];
#pragma unroll
                    for (int r4 = 0; r4 < 4; r4++) {
                        u32 w[C::PN];
                        pg_pieces<CT, C::PN>(p[g][2 * r4], p[g][2 * r4 + 1], w);
#pragma unroll
                        for (int k = 0; k < C::PN; k++) af[k][r4] = w[k];
                    }
#pragma unroll
                    for (int b2 = 0; b2 < HD / 16; b2++) {
                        u32 w[4];
                        pg_ldsm4t(w, ra + (u32)((b2 >> 2) * PG_T * 128 + g * 16 * 128 + (((2 * (b2 & 3) + cx) ^ sw) << 4)));
#pragma unroll
                        for (int k = 0; k < C::PN; k++) { pg_mma<CT>(o[2 * b2], af[k], w[0], w[1]); pg_mma<CT>(o[2 * b2 + 1], af[k], w[2], w[3]); }
                    }
                }
            } else {                                      // position by position, only for the rows that see it
                const u8* vr = ring + (size_t)cslot * C::HALF;
#pragma unroll
                for (int g = 0; g < C::SG; g++)
#pragma unroll
                    for (int k = 0; k < 16; k++) {
                        const int src = (lane & ~3) | ((k & 7) >> 1), pos = pw + 16 * g + k;
                        const float w0 = __shfl_sync(0xffffffffu, p[g][4 * (k >> 3) + (k & 1)], src), w1 = __shfl_sync(0xffffffffu, p[g][4 * (k >> 3) + 2 + (k & 1)], src);
                        const bool ok = (okb >> (16 * g + k)) & 1u, a = ok && it.i * PG_T + pos < lim0, b = ok && it.i * PG_T + pos < lim1;
#pragma unroll
                        for (int nt = 0; nt < C::NT; nt++) {
                            const float2 f = pg_unpack<CT>(*(const u32*)(vr + (size_t)(nt >> 3) * PG_T * 128 + (size_t)pos * 128 + (((nt & 7) ^ (pos & 7)) << 4) + 4 * q4));
                            if (a) { o[nt][0] = fmaf(w0, f.x, o[nt][0]); o[nt][1] = fmaf(w0, f.y, o[nt][1]); }
                            if (b) { o[nt][2] = fmaf(w1, f.x, o[nt][2]); o[nt][3] = fmaf(w1, f.y, o[nt][3]); }
                        }
                    }
            }
        } else {
            const u8* vr = ring + (size_t)cslot * C::HALF + (size_t)pw * C::HB;
            bool odd;                                     // a scale that is infinite or NaN, or not a row's: it must not reach a hidden position's weight of 0
            {   // the powers of two that bring the largest value scale each of the lane's rows sees to [2^-1, 1) (weights: 2^15 at most).  What a row does
                // not see - later rows' positions, slots that nothing was written to - has no say: one scale of 65,504 there would leave its weights
                // f16's subnormals.  Where all rows see all positions, which is the rule, one maximum does for all.
                u32 t0 = 0, t1 = 0;
                const bool clear = !__any_sync(0xffffffffu, part);
                if (clear) {
#pragma unroll
                    for (int i = 0; i < (16 * C::SG * HD / 64 + 31) / 32; i++) {
                        const int x = lane + 32 * i, r = x / (HD / 64), w2 = x % (HD / 64);
                        if (16 * C::SG * HD / 64 % 32 == 0 || r < 16 * C::SG) {
                            const u32 w = *(const u32*)(vr + (size_t)r * C::HB + HD + 4 * w2);
                            t0 = max(t0, max(w & 0x7fffu, (w >> 16) & 0x7fffu));
                        }
                    }
                    t0 = t1 = __reduce_max_sync(0xffffffffu, t0);
                } else {
#pragma unroll 1
                    for (int r = q4; r < 16 * C::SG; r += 4) {      // the four lanes of a row share its positions
                        u32 big = 0;
#pragma unroll
                        for (int i = 0; i < HD / 64; i++) {
                            const u32 w = *(const u32*)(vr + (size_t)r * C::HB + HD + 4 * i);
                            big = max(big, max(w & 0x7fffu, (w >> 16) & 0x7fffu));
                        }
                        const bool ok = (okb >> r) & 1u;
                        if (ok && c0 + r < lim0) t0 = max(t0, big);
                        if (ok && c0 + r < lim1) t1 = max(t1, big);
                    }
                    __syncwarp();
#pragma unroll
                    for (int k = 1; k < 4; k <<= 1) { t0 = max(t0, __shfl_xor_sync(0xffffffffu, t0, k)); t1 = max(t1, __shfl_xor_sync(0xffffffffu, t1, k)); }
                }
                auto moved = [&](u32 top, float csc) {    // what the row's sums are multiplied by (powers of two: exact)
                    const int ex = top >> 10 ? (int)(top >> 10) - 14 : -14;         // scale < 2^ex
                    const float want = __uint_as_float((u32)(127 - ex) << 23);
                    return top && (want < csc || (fresh && want != csc)) ? __uint_as_float(__float_as_uint(want) - __float_as_uint(csc) + 0x3f800000u) : 1.f;      // (their quotient, by the exponents)
                };
                const float by0 = moved(t0, csc0), by1 = moved(t1, csc1);
                if (__any_sync(0xffffffffu, by0 != 1.f || by1 != 1.f)) {
#pragma unroll
                    for (int b = 0; b < C::NT; b++) { o[b][0] *= by0; o[b][1] *= by0; o[b][2] *= by1; o[b][3] *= by1; }
                    csc0 *= by0; csc1 *= by1;
                }
                fresh = false;
                odd = !clear || t0 >= 0x7c00u;
            }
#pragma unroll
            for (int g = 0; g < C::SG; g++)
#pragma unroll
                for (int e = 0; e < 8; e++) p[g][e] *= e & 2 ? csc1 : csc0;      // (a power of two: exact, but for weights of 2^-100 and less)
#pragma unroll
            for (int g = 0; g < C::SG; g++) {
                u32 vs[4];
#pragma unroll
                for (int gr = 0; gr < HD / 32; gr++) {
                    u32 v4[4];
#pragma unroll
                    for (int r4 = 0; r4 < 4; r4++) {      // positions 2 q4, + 1, + 8, + 9: the lane's k slots; a word: dimensions 32 gr + 4 g8 ..
                        const u8* row = vr + (size_t)(16 * g + 2 * q4 + (r4 & 1) + 8 * (r4 >> 1)) * C::HB;
                        v4[r4] = *(const u32*)(row + 32 * gr + 4 * g8) ^ 0x80808080u;
                        if (gr % 2 == 0) vs[r4] = *(const u32*)(row + HD + 2 * gr);      // (this group's scale and the next one's)
                    }
                    float pv[8];
#pragma unroll
                    for (int e = 0; e < 8; e++) pv[e] = p[g][e] * pg_half(vs[2 * (e >> 2) + (e & 1)], gr & 1);
                    if (odd) {
#pragma unroll
                        for (int e = 0; e < 8; e++) pv[e] = p[g][e] > 0.f ? pv[e] : 0.f;
                    }
                    u32 af[C::PN][4];
#pragma unroll
                    for (int r4 = 0; r4 < 4; r4++) {
                        u32 w[C::PN];
                        pg_pieces<CT, C::PN>(pv[2 * r4], pv[2 * r4 + 1], w);
#pragma unroll
                        for (int k = 0; k < C::PN; k++) af[k][r4] = w[k];
                    }
                    // a position's four bytes beside the next position's, then a pair of each under f16's exponent 0x64 (code + 128 + 1024), less 1,152
                    const u32 x0 = __byte_perm(v4[0], v4[1], 0x5140), x1 = __byte_perm(v4[0], v4[1], 0x7362), y0 = __byte_perm(v4[2], v4[3], 0x5140), y1 = __byte_perm(v4[2], v4[3], 0x7362);
                    const __half2 bias = __halves2half2(__ushort_as_half((u16)0x6480), __ushort_as_half((u16)0x6480));
#pragma unroll
                    for (int b = 0; b < 4; b++) {         // tile b's column n is dimension 32 gr + 4 n + b
                        const u32 u0 = __byte_perm(b < 2 ? x0 : x1, 0x64646464u, b & 1 ? 0x4342 : 0x4140), u1 = __byte_perm(b < 2 ? y0 : y1, 0x64646464u, b & 1 ? 0x4342 : 0x4140);
                        const __half2 h0 = __hsub2(*(const __half2*)&u0, bias), h1 = __hsub2(*(const __half2*)&u1, bias);
#pragma unroll
                        for (int k = 0; k < C::PN; k++) pg_mma<CT>(o[4 * gr + b], af[k], *(const u32*)&h0, *(const u32*)&h1);
                    }
                }
            }
        }
        if (++cslot == C::NR) { cslot = 0; cphase ^= 1; }
        if (u + 1 < u1 && it.i + 1 < it.n) continue;
        // ---- the block's last unit of the item: its parts go out, every way's by itself - but at the block's end, where the ring lies idle, the ways
        // are added up there first, and one part goes out for all (the others' maxima say that they are empty).  One long conversation is split
        // over all blocks: its parts, 16 KB a warp, took longer to write and to join than to make.
        const float back = CT == PG_BF16 ? 1.f : 1.f / 32768.f, un0 = back / csc0, un1 = back / csc1;
#pragma unroll
        for (int k = 1; k < 4; k <<= 1) { l0 += __shfl_xor_sync(0xffffffffu, l0, k); l1 += __shfl_xor_sync(0xffffffffu, l1, k); }
        l0 *= back; l1 *= back;
        if (l0 != l0 && m0 == -INFINITY) m0 = 0.f;        // (scores that are all NaN have no maximum, and are not an empty part)
        if (l1 != l1 && m1 == -INFINITY) m1 = 0.f;
#pragma unroll
        for (int b = 0; b < C::NT; b++) { o[b][0] *= un0; o[b][1] *= un0; o[b][2] *= un1; o[b][3] *= un1; }
        if (C::WAYS > 1 && u + 1 == u1) {
            constexpr int ST = HD + 8;                    // floats a row: rows begin at different banks
            static_assert((C::WAYS - 1) * NQT * 16 * ST * 4 <= C::NR * C::HALF && (C::WAYS - 1) * NQT * 16 * 8 <= C::QB, "the parts fit the ring");
            float* const buf = (float*)ring;
            float2* const ml = (float2*)qm;
            __syncthreads();
            if (way > 0) {
                float* w = buf + ((size_t)((way - 1) * NQT + qt) * 16 + g8) * ST + 2 * q4;
#pragma unroll
                for (int b = 0; b < C::NT; b++) { *(float2*)(w + 8 * b) = make_float2(o[b][0], o[b][1]); *(float2*)(w + 8 * ST + 8 * b) = make_float2(o[b][2], o[b][3]); }
                if (q4 == 0) { ml[((way - 1) * NQT + qt) * 16 + g8] = make_float2(m0, l0); ml[((way - 1) * NQT + qt) * 16 + g8 + 8] = make_float2(m1, l1); }
                m0 = m1 = -INFINITY;
            }
            __syncthreads();
            if (way == 0) {
                float x0 = m0, x1 = m1;
#pragma unroll
                for (int x = 0; x < C::WAYS - 1; x++) { x0 = fmaxf(x0, ml[(x * NQT + qt) * 16 + g8].x); x1 = fmaxf(x1, ml[(x * NQT + qt) * 16 + g8 + 8].x); }
                const float c0 = m0 == -INFINITY ? 0.f : pg_ex2(m0 - x0), c1 = m1 == -INFINITY ? 0.f : pg_ex2(m1 - x1);
                l0 *= c0; l1 *= c1;
#pragma unroll
                for (int b = 0; b < C::NT; b++) { o[b][0] *= c0; o[b][1] *= c0; o[b][2] *= c1; o[b][3] *= c1; }
#pragma unroll 1
                for (int x = 0; x < C::WAYS - 1; x++) {
                    const float2 a = ml[(x * NQT + qt) * 16 + g8], b2 = ml[(x * NQT + qt) * 16 + g8 + 8];
                    const float ca = a.x == -INFINITY ? 0.f : pg_ex2(a.x - x0), cb = b2.x == -INFINITY ? 0.f : pg_ex2(b2.x - x1);
                    l0 = fmaf(a.y, ca, l0); l1 = fmaf(b2.y, cb, l1);
                    const float* w = buf + ((size_t)(x * NQT + qt) * 16 + g8) * ST + 2 * q4;
#pragma unroll
                    for (int b = 0; b < C::NT; b++) {
                        const float2 f = *(const float2*)(w + 8 * b), g = *(const float2*)(w + 8 * ST + 8 * b);
                        o[b][0] = fmaf(f.x, ca, o[b][0]); o[b][1] = fmaf(f.y, ca, o[b][1]); o[b][2] = fmaf(g.x, cb, o[b][2]); o[b][3] = fmaf(g.y, cb, o[b][3]);
                    }
                }
                m0 = x0; m1 = x1;
            }
        }
        const u32 us = units[it.e] * (u32)d.nkv + (u32)it.h * (u32)it.n;                         // the item's first unit
        const int b0 = pg_block_of(share, us), b1 = pg_block_of(share, us + it.n - 1);
        const int r0 = row_of(it.b), mrows = (pt.shared ? row_of(d.n_seq) : row_of(it.b + 1)) - r0;
#pragma unroll
        for (int hf = 0; hf < 2; hf++) {
            const int v = qt * 16 + g8 + 8 * hf, vec = it.t * C::TQ + v, row = vec / d.G;
            if (row >= mrows) continue;
            const size_t at = (b0 == b1 ? (size_t)(r0 + row) * (d.nkv * d.G) + it.h * d.G + (vec - row * d.G)
                                        : (size_t)(2 * blockIdx.x + ((int)blockIdx.x == b0 ? 1 : 0)) * C::TQ + v) * C::WAYS + way;
            float* w = (b0 == b1 ? pt.row_o : pt.o) + at * HD;
            if (q4 == 0) (b0 == b1 ? pt.row_ml : pt.ml)[at] = make_float2(hf ? m1 : m0, hf ? l1 : l0);
            if ((hf ? m1 : m0) == -INFINITY) continue;    // (nobody reads an empty part's sums)
            if (CT == PG_Q8) {                            // the lane's columns of the four tiles of a 32-dimension group are eight neighbouring dimensions
#pragma unroll
                for (int gr = 0; gr < HD / 32; gr++)
#pragma unroll
                    for (int c = 0; c < 2; c++)
                        *(float4*)(w + 32 * gr + 8 * q4 + 4 * c) = make_float4(o[4 * gr][2 * hf + c], o[4 * gr + 1][2 * hf + c], o[4 * gr + 2][2 * hf + c], o[4 * gr + 3][2 * hf + c]);
            } else {
#pragma unroll
                for (int b = 0; b < C::NT; b++) *(float2*)(w + 8 * b + 2 * q4) = make_float2(o[b][2 * hf], o[b][2 * hf + 1]);
            }
        }
    }
    if (dead) {                                           // what is under way is waited for, once more with a limit: the block's memory is another's soon
        const int n = (int)(2 * (u1 - u0)) + 1 + steps_left;      // halves asked for
        for (int i = max(0, n - C::NR); i < n; i++) sz_mbar_wait_warp(&s_full[NQT == 1 ? i % C::NR * 4 + warp : i % C::NR], (u32)(i / C::NR) & 1u);
    }
    // (only now: blocks of the merge that wait on a multiprocessor early took places of this kernel's - 64 sequences 414 -> 530 us)
    sz_pdl_trigger();
}

// What a set of kernels offers the host.
struct PgKernels {
    const void* fn;
    int threads, smem, occ, tq, ways;
};
PgKernels pg_kernels_f16(bool wide, int hd, int nqt);
PgKernels pg_kernels_bf16(bool wide, int hd, int nqt);
PgKernels pg_kernels_q8(bool wide, int hd, int nqt);
// The tcgen05 kernel (sz_paged_tc.cu): vectors a tile; the launch over own or shared positions.
int pg_tc_tile(int hd);
int pg_tc_unit(int hd);
int pg_tc_launch(bool bf16, int hd, const CUtensorMap* maps, int rows_box, const PgBatch& d, const PgIo& io, const PgPart& p, const char* name, cudaStream_t st);

template <int CT, bool WIDE, int HD, int NQT>
PgKernels pg_one() {
    using C = PgCfg<CT, WIDE, HD, NQT>;
    return {(const void*)sz_pg_attend_kernel<CT, WIDE, HD, NQT>, C::NTH, C::SMEM, C::OCC, C::TQ, C::WAYS};
}
template <int CT, bool WIDE, int HD>
PgKernels pg_of_tiles(int nqt) { return nqt == 1 ? pg_one<CT, WIDE, HD, 1>() : nqt == 2 ? pg_one<CT, WIDE, HD, 2>() : pg_one<CT, WIDE, HD, 4>(); }
template <int CT, bool WIDE>
PgKernels pg_of_hd(int hd, int nqt) { return hd == 64 ? pg_of_tiles<CT, WIDE, 64>(nqt) : hd == 128 ? pg_of_tiles<CT, WIDE, 128>(nqt) : pg_of_tiles<CT, WIDE, 256>(nqt); }
template <int CT>
PgKernels pg_of(bool wide, int hd, int nqt) { return wide ? pg_of_hd<CT, true>(hd, nqt) : pg_of_hd<CT, false>(hd, nqt); }
