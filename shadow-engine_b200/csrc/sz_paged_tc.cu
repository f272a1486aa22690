// Attention of many query vectors over the same positions on the 5th-generation tensor cores: a long prefix that a whole batch shares, or what
// was fed before a prompt's chunk.  (Few vectors a key head leave the kernel of sz_paged.cuh waiting for memory, not for its mma.sync; with
// hundreds the products are the work: 4 head_dim operations a vector and position on 4 head_dim bytes.)
//
// Types: 16-bit queries over a cache of the same type.
//
// A block has NQ x 128 query vectors of one key head (two tiles of 128 up to head_dim 128, one above) and the columns of tensor memory:
//     0 .. 255    scores, two buffers a tile of 64 positions (head_dim 256: 128) in f32; the weights lie over the buffer they come from, as pairs of 16 bits
//     256 .. 511  the tiles' sums, NQ x head_dim
// One warp issues the scores' products of unit after unit, another the sums', each when its operands are there and the buffer is free: what they do between
// two units - waits, a commit, descriptors: 500 cycles - is hidden behind the other's instructions, and a tile's softmax goes from unit to
// unit without waiting for its products.  (One warp for both: 2,860 cycles for two tiles and 64 positions, whose instructions need 1,280.  Units of 128
// positions with one buffer a tile, where softmax, products and scores take turns: 5,900 for 128.)
//   warps 0 .. 3 (and 4 .. 7 for the second tile)   a thread has a query vector, lane = row of tensor memory: it reads its 64 scores
//               (tcgen05.ld), moves what it divides by - only when the largest weight would be beyond 2^8 (f16: 2^15), for then the sums have to be
//               read, scaled and written back -, writes the weights (tcgen05.st) and keeps their sum.
// (tcgen05.ld, st, their waits and alloc are for whole warps: wherever lanes went different ways before one, __syncwarp brings them together.)
//   last four   keys, and values, by tiled TMA, a box a page (8 .. 64 positions x 64 dimensions, 128-byte swizzle), each through a ring of 64 positions x
//               128 dimensions; the two issuing warps.
// Operands: queries and keys K-major, values MN-major (their rows are the positions, which the product sums over), weights from tensor memory.
// Measured: 2,045 rows of 16 heads of 256 on 2 behind 7,555 positions, bf16: 317 us, 0.91 PFLOP/s, 336 and 0.86 in a loop of a second (the products alone at the measured rate 175); 64 rows of 32 heads
// of 128 over 24,576 shared positions some 47 us (16 of bytes or products).  What bounds it is the chain of a tile - scores, softmax, weights, product -: at head_dim 256 tensor memory
// holds one tile's sums and two buffers of its scores, so that the softmax of a unit has the products of its neighbours only to run beside; up to 128
// the exponentials (16,384 for 128 vectors and 128 positions) take the multiprocessor as long as both products take the tensor core.
// Rounding: a weight is one number of the rows' type, 8 (bf16) or 11 bits as the result; its sum is of the unrounded ones.  Errors of independent
// weights average out to those of one rounding: the result is 1.4 times as far off as its last rounding alone (f32 rows 1.66e-3 of the results' norm, bf16
// weights 2.33e-3).  A second piece, as the few-vector kernel has it, would double the product with the values.  bf16 has f32's range; in f16 the
// largest weight lies between 2^11 and 2^15, so that those down to 2^-25 of it keep all their bits and those below 2^-36 are lost.  (With the largest
// at 1 .. 2^8, as for bf16, a weight of e^-13 was 0.2 % off and one of e^-17 44 %: four half steps of the result, and nothing left of it, where the rest has no value.)
// A page out of range arrives as zeros (its box lies outside the pool's map) and its positions are masked.  Every wait is bounded.
//
// What a row does not see must not reach it, whatever it is: scores of such positions are replaced, but a weight of 0 times a value that is infinite
// or NaN would be NaN.  So in a unit that not all rows of a tile see whole, the first tile's threads clear the values behind the sequence's end and
// those that are not finite, before the product; should there be any of the latter, the rows that see them add them at the end.
#include "sz_paged.cuh"

namespace {

constexpr u32 PT_WAIT = 4000000u;

__device__ __forceinline__ u64 pt_desc(u32 addr, u32 lbo, u32 sbo) {      // 128-byte swizzle (layout type 2), version 1
    return (u64)((addr & 0x3ffffu) >> 4) | ((u64)(lbo >> 4) << 16) | ((u64)(sbo >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
// kind::f16: D = f32, A and B f16 (0) or bf16 (1), M = 128, N; B K-major or (values) MN-major
__host__ __device__ constexpr u32 pt_idesc(bool bf16, int n, bool b_mn) {
    return (1u << 4) | ((bf16 ? 1u : 0u) << 7) | ((bf16 ? 1u : 0u) << 10) | ((b_mn ? 1u : 0u) << 16) | ((u32)(n >> 3) << 17) | ((128u >> 4) << 24);
}
// Issued by one lane (`one`) of a warp that runs as a whole: in code that a single lane has branched into, every operand of every
// instruction is moved to the uniform registers anew - 110 cycles an instruction, of which the tensor core needs 64.
__device__ __forceinline__ void pt_mma_ss(u32 d, u64 a, u64 b, u32 idesc, u32 acc, u32 one) {
    asm volatile("{ .reg .pred p, q; setp.ne.b32 p, %4, 0; setp.ne.b32 q, %5, 0; @q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p; }" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc),
                 "r"(one) : "memory");
}
__device__ __forceinline__ void pt_mma_ts(u32 d, u32 a, u64 b, u32 idesc, u32 acc, u32 one) {      // A from tensor memory
    asm volatile("{ .reg .pred p, q; setp.ne.b32 p, %4, 0; setp.ne.b32 q, %5, 0; @q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p; }" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(acc),
                 "r"(one) : "memory");
}
__device__ __forceinline__ void pt_commit(u64* bar, u32 one) {
    asm volatile("{ .reg .pred q; setp.ne.b32 q, %1, 0; @q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0]; }" ::"r"(sz_smem_addr(bar)), "r"(one) : "memory");
}
__device__ __forceinline__ u32 pt_elect() {
    u32 x;
    asm volatile("{ .reg .pred p; elect.sync _|p, 0xffffffff; selp.u32 %0, 1, 0, p; }" : "=r"(x));
    return x;
}
__device__ __forceinline__ void pt_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void pt_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void pt_ld32(u32 at, float* v) {              // 32 columns of the thread's row
    u32* r = (u32*)v;
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]),
                   "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
                   "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
                 : "r"(at));
}
__device__ __forceinline__ void pt_loaded(float* v) {                    // the registers go through the wait, so that nothing uses them before it
    u32* r = (u32*)v;
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]),
                   "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]),
                   "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])::"memory");
}
__device__ __forceinline__ void pt_st16(u32 at, const u32* r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]),
                 "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(at) : "memory");
}
__device__ __forceinline__ void pt_stored() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ bool pt_wait(u64* bar, u32 phase) { return sz_mbar_wait(bar, phase & 1, PT_WAIT); }
__device__ __forceinline__ bool pt_wait_warp(u64* bar, u32 phase) { return __all_sync(0xffffffffu, pt_wait(bar, phase)); }
__device__ __forceinline__ void pt_arrive_warp(u64* bar) { __syncwarp(); if ((threadIdx.x & 31) == 0) sz_mbar_arrive(bar); }

// What a row divides by when it moves: the largest score less PT_UP (so the largest weight is 2^PT_UP); it moves where the largest would pass 2^PT_TOP.
template <bool BF> constexpr float PT_UP = BF ? 0.f : 11.f;
template <bool BF> constexpr float PT_TOP = BF ? 8.f : 15.f;
__device__ __forceinline__ float pt_max3(float a, float b, float c) { float r; asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c)); return r; }
template <int HD>
struct PtCfg {
    static constexpr int NQ = HD <= 128 ? 2 : 1, DB = HD < 128 ? HD : 128, NB = HD / DB;     // tiles; dimensions a ring slot, slots a unit's keys
    static constexpr int UT = HD == 256 ? 128 : 64;          // positions a unit
    static constexpr int SOFT = 128 * NQ, NTH = SOFT + 128, TQ = 128 * NQ;
    static constexpr int SLOT = UT * DB * 2, QT = 128 * HD * 2, BLK = UT * 128, QBLK = 128 * 128;      // bytes; BLK, QBLK: 64 dimensions of the positions, of a tile
    static constexpr int SLOTS = 256 / UT;                 // of a ring, one of keys and one of values
    static constexpr int SMEM = 1024 + NQ * QT + 2 * SLOTS * SLOT;                                 // (1,024 to align)
};
struct PtBars {
    u64 full[2][4], empty[2][4], s_full[4], p_full[4], pv_done[4], q_full[2], o_free[2], last[2];      // (per tile two where units have turns: one at most is ahead of a waiter)
    u32 tmem, failed;
    u32 odd[2];                      // of every other piece: its number + 1, once a value that is not finite was cleared
    __align__(16) u32 ok[8][4];                    // which positions of a unit are there, of eight units: the eighth next one's keys are asked for after this one's weights were used
    u32 tiles[PG_PLAN + 1], units[PG_PLAN + 1], scan[16];
    int rows[PG_PLAN + 1], ends[PG_PLAN + 1];
};

template <bool BF, int HD>
__global__ void __launch_bounds__(PtCfg<HD>::NTH, 1)
sz_pg_tc_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap, const __grid_constant__ PgBatch d, const __grid_constant__ PgIo io,
                const __grid_constant__ PgPart pt, int rows_box) {
    using C = PtCfg<HD>;
    constexpr int CT = BF ? PG_BF16 : PG_F16;
    __shared__ PtBars S;
    extern __shared__ __align__(16) u8 raw[];
    u8* const base = raw + (1024 - (sz_smem_addr(raw) & 1023)) % 1024;
    u8* const sq = base;                                   // [tile][HD / 64][128 rows][128 bytes]
    u8* const ring = sq + C::NQ * C::QT;                   // [keys, values][slot][DB / 64][64 positions][128 bytes]
    u8* const vring = ring + C::SLOTS * C::SLOT;
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    constexpr int TMA_WARP = C::SOFT / 32, S_WARP = TMA_WARP + 2, PV_WARP = TMA_WARP + 3;
    if (tid == 0) {
        for (int i = 0; i < 8; i++) { sz_mbar_init(&S.full[0][i], 1); sz_mbar_init(&S.empty[0][i], 1); }
        for (int i = 0; i < 4; i++) { sz_mbar_init(&S.s_full[i], 1); sz_mbar_init(&S.p_full[i], 4); sz_mbar_init(&S.pv_done[i], 1); }
        for (int i = 0; i < 2; i++) { sz_mbar_init(&S.q_full[i], 4); sz_mbar_init(&S.o_free[i], 4); sz_mbar_init(&S.last[i], 1); }
        S.failed = 0;
        S.odd[0] = S.odd[1] = 0;
        sz_mbar_fence_init();
    }
    if (warp == 0) {
        __syncwarp();
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(sz_smem_addr(&S.tmem)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    pt_before();
    __syncthreads();
    pt_after();
    const u32 tmem = __shfl_sync(0xffffffffu, S.tmem, 0);
    sz_pdl_wait();
    const u32 *tiles = S.tiles, *units = S.units;
    int E;
    if (pt.planned) {
        tiles = pt.tiles; units = pt.units;
        E = pt.shared ? max(0, ((pg_row(d, d.n_seq) - pg_row(d, 0)) * d.G + C::TQ - 1) / C::TQ) : (int)tiles[d.n_seq];
    } else {
        E = pg_plan<C::NTH>(d, pt.shared, C::UT, C::TQ, S.tiles, S.units, S.scan, S.rows, S.ends);
        if (blockIdx.x == 0) {
            if (!pt.shared) for (int i = tid; i <= d.n_seq; i += C::NTH) pt.tiles[i] = S.tiles[i];
            for (int i = tid; i <= E; i += C::NTH) pt.units[i] = S.units[i];
        }
    }
    if (blockIdx.x == 0 && !pt.shared) {                   // what the lengths ask for that is not there
        for (int b = tid; b < d.n_seq; b += C::NTH)
            if (pg_row(d, b + 1) > pg_row(d, b) && (long long)__ldg(d.lens + b) - d.shared_len > ((long long)d.max_pages << d.ps_log2)) atomicOr(d.err, PG_E_END);
        if (tid == 0 && __ldg(d.row_start + d.n_seq) > d.rows) atomicOr(d.err, PG_E_ROWS);
    }
    const u32 U = units[E] * (u32)d.nkv;
    const int blocks = (int)min((u32)pt.blocks, U);
    const bool work = (int)blockIdx.x < blocks;
    const PgShare share = work ? pg_share(U, blocks) : PgShare{1u, 0u};
    const u32 u0 = work ? pg_first(share, blockIdx.x) : 0, u1 = work ? pg_first(share, blockIdx.x + 1) : 0;
    auto row_of = [&](int b) { return pt.planned ? pg_row(d, b) : S.rows[b]; };
    auto end_of = [&](int b) { return (long long)(pt.planned ? pg_end(d, b) : S.ends[b]); };
    // the next piece of the block's share: an item, units i .. i + T of it
    auto locate = [&](u32 u) {
        PgItem it;
        const u32 un = u / (u32)d.nkv;
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
    const PgItem first = work ? locate(u0) : PgItem();      // (by all warps at once: the roles' own copies of this code would be fetched one beside the other)
    int failed = 0;
    if (warp == TMA_WARP || warp == TMA_WARP + 1) {
        // ---- loads, of keys and of values: units in order.  Pages are looked up a window of units ahead (32 entries of the table, one a lane): one after the
        // other, each look-up took as long as a unit.  The copies, too, are issued by one lane of the whole warp (above): lanes that issued their own
        // took 300 cycles each.
        const int kind = warp - TMA_WARP, pieces = C::UT / rows_box, ahead = 32 / pieces;      // boxes a unit (1 .. 16) and 64 dimensions, units a window
        const u32 one = pt_elect();
        const CUtensorMap* const map = kind ? &vmap : &kmap;
        u8* const to = kind ? vring : ring;
        u32 g = 0, fills = 0;                              // units so far; slots filled
        for (u32 u = u0; u < u1 && !failed;) {
            const PgItem it = u == u0 ? first : locate(u);
            const int T = (int)min((u32)(it.n - it.i), u1 - u);
            const int32_t* table = pt.shared ? d.shared_pages : d.pages + (size_t)it.b * d.max_pages;
            auto window = [&](int w) {
                const int c = (it.i + w * ahead) * C::UT + lane * rows_box;
                return c < it.end ? __ldg(table + (c >> d.ps_log2)) : -1;
            };
            int now = window(0), next = window(1);
            for (int j = 0; j < T && !failed; j++, g++) {
                const int k0 = j % ahead * pieces;
                if (j && k0 == 0) { now = next; next = window(j / ahead + 1); }
                const u32 there = __ballot_sync(0xffffffffu, (u32)now < (u32)d.n_pages) >> k0;
                if (kind == 0 && lane >= k0 && lane < k0 + pieces && (u32)now >= (u32)d.n_pages && (it.i + j) * C::UT + (lane - k0) * rows_box < it.end)
                    atomicOr(d.err, PG_E_PAGE);            // (behind the end: not there, and no error)
#pragma unroll
                for (int nb = 0; nb < C::NB; nb++) {
                    const u32 n = g * C::NB + nb;
                    const int sl = (int)(n % C::SLOTS);
                    if (n >= C::SLOTS && !pt_wait_warp(&S.empty[kind][sl], n / C::SLOTS - 1)) { failed = 1; break; }
                    if (kind == 0 && nb == 0) {            // (read by the softmax threads after the scores are there, which the copies' arrival comes before)
                        if (lane < C::UT / 32) {
                            u32 w = 0;
                            for (int k = 0; k < 32; k += 8) if ((there >> ((lane * 32 + k) / rows_box)) & 1u) w |= 0xffu << k;
                            S.ok[g & 7][lane] = w;
                        }
                        __syncwarp();
                    }
                    fills = n + 1;
                    u64* const bar = &S.full[kind][sl];
                    const u32 dst = sz_smem_addr(to) + (u32)(sl * C::SLOT);
                    asm volatile("{ .reg .pred q; setp.ne.b32 q, %2, 0; @q mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1; }" ::"r"(sz_smem_addr(bar)), "r"((u32)C::SLOT), "r"(one) : "memory");
                    for (int p = 0; p < pieces; p++) {
                        const int page = __shfl_sync(0xffffffffu, now, k0 + p), y = ((it.i + j) * C::UT + p * rows_box) & ((1 << d.ps_log2) - 1);
                        const int z = (u32)page < (u32)d.n_pages ? page : d.n_pages;
#pragma unroll
                        for (int q = 0; q < C::DB / 64; q++)
                            asm volatile("{ .reg .pred q; setp.ne.b32 q, %7, 0;\n"
                                         "  @q cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6]; }" ::"r"(
                                             dst + (u32)(q * C::BLK + p * rows_box * 128)),
                                         "l"(map), "r"(nb * C::DB + q * 64), "r"(y), "r"(it.h), "r"(z), "r"(sz_smem_addr(bar)), "r"(one)
                                         : "memory");
                    }
                }
            }
            u += T;
        }
        // (a role that gave up a wait leaves copies and products to nobody: each role sees its own to their end, bounded)
        for (u32 n = fills > C::SLOTS ? fills - C::SLOTS : 0; n < fills; n++) if (!pt_wait_warp(&S.full[kind][n % C::SLOTS], n / C::SLOTS)) failed = 11;
        __syncwarp();
    } else if (warp == S_WARP) {
        // ---- the scores' products: a unit's, once its buffer's last weights have been used
        constexpr u32 id_s = pt_idesc(BF, C::UT, false);
        const u32 one = pt_elect();
        const u64 qd = pt_desc(sz_smem_addr(sq), 16, 1024), kd = pt_desc(sz_smem_addr(ring), 16, 1024);
        u32 piece = 0, done = 0;                           // pieces; units before this one
        for (u32 u = u0; u < u1 && !failed; piece++) {
            const PgItem it = u == u0 ? first : locate(u);
            const int T = (int)min((u32)(it.n - it.i), u1 - u);
            for (int q = 0; q < C::NQ && !failed; q++) if (!pt_wait_warp(&S.q_full[q], piece)) failed = 2;
            for (int j = 0; j < T && !failed; j++) {
                const u32 g = done + j;
#pragma unroll
                for (int q = 0; q < C::NQ; q++) {
                    const int buf = q * 2 + (int)(g & 1);
                    if (g >= 2 && !pt_wait_warp(&S.pv_done[buf], (g >> 1) - 1)) { failed = 4; break; }
#pragma unroll
                    for (int nb = 0; nb < C::NB; nb++) {
                        const int sl = (int)((g * C::NB + nb) % C::SLOTS);
                        if (q == 0 && !pt_wait_warp(&S.full[0][sl], (g * C::NB + nb) / C::SLOTS)) { failed = 3; break; }
                        pt_after();
                        const u64 qa = qd + (u32)((q * C::QT + nb * (C::DB / 64) * C::QBLK) / 16), ka = kd + (u32)(sl * (C::SLOT / 16));
#pragma unroll
                        for (int k = 0; k < C::DB / 16; k++)       // (addresses in 16-byte units: 16 dimensions are 32 bytes of a row)
                            pt_mma_ss(tmem + buf * C::UT, qa + (u32)(k / 4 * (C::QBLK / 16) + (k % 4) * 2), ka + (u32)(k / 4 * (C::BLK / 16) + (k % 4) * 2), id_s, nb | k, one);
                        if (q == C::NQ - 1) pt_commit(&S.empty[0][sl], one);
                    }
                    if (failed) break;
                    pt_commit(&S.s_full[buf], one);
                }
            }
            done += T;
            u += T;
        }
        pt_commit(&S.last[0], one);
        if (!pt_wait_warp(&S.last[0], 0)) failed = 12;
        __syncwarp();
    } else if (warp == PV_WARP) {
        // ---- the sums' products: a unit's, once its weights are there
        constexpr u32 id_v = pt_idesc(BF, C::DB, true);
        const u32 one = pt_elect();
        const u64 vd = pt_desc(sz_smem_addr(vring), C::BLK, 1024);
        u32 piece = 0, done = 0;
        for (u32 u = u0; u < u1 && !failed; piece++) {
            const PgItem it = u == u0 ? first : locate(u);
            const int T = (int)min((u32)(it.n - it.i), u1 - u);
            for (int j = 0; j < T && !failed; j++) {
                const u32 g = done + j;
#pragma unroll
                for (int q = 0; q < C::NQ; q++) {
                    const int buf = q * 2 + (int)(g & 1);
                    if (j == 0 && piece > 0 && !pt_wait_warp(&S.o_free[q], piece - 1)) { failed = 5; break; }
                    if (!pt_wait_warp(&S.p_full[buf], g >> 1)) { failed = 4; break; }
#pragma unroll
                    for (int nb = 0; nb < C::NB; nb++) {
                        const int sl = (int)((g * C::NB + nb) % C::SLOTS);
                        if (q == 0 && !pt_wait_warp(&S.full[1][sl], (g * C::NB + nb) / C::SLOTS)) { failed = 6; break; }
                        pt_after();
                        const u64 va = vd + (u32)(sl * (C::SLOT / 16));
                        const u32 od = tmem + 256 + q * HD + nb * C::DB, pa = tmem + buf * C::UT;
#pragma unroll
                        for (int k = 0; k < C::UT / 16; k++)       // 16 positions: 8 columns of weight pairs, 16 rows of 128 bytes
                            pt_mma_ts(od, pa + k * 8, va + (u32)(k * 128), id_v, (u32)(j | k), one);
                        if (q == C::NQ - 1) pt_commit(&S.empty[1][sl], one);
                    }
                    if (failed) break;
                    pt_commit(&S.pv_done[buf], one);
                }
            }
            done += T;
            u += T;
        }
        pt_commit(&S.last[1], one);
        if (!pt_wait_warp(&S.last[1], 0)) failed = 12;
        __syncwarp();
    } else {
        // ---- softmax: thread = query vector
        const int q = warp / 4, row = tid & 127;
        const u32 lanes = (u32)((warp & 3) * 32) << 16;
        u32 piece = 0, done = 0;                           // done: units so far
        for (u32 u = u0; u < u1 && !failed; piece++) {
            const PgItem it = u == u0 ? first : locate(u);
            const int T = (int)min((u32)(it.n - it.i), u1 - u);
            const int r0 = row_of(it.b), m = (pt.shared ? row_of(d.n_seq) : row_of(it.b + 1)) - r0;
            const int v = q * 128 + row, vec = it.t * C::TQ + v, qr = vec / d.G, head = it.h * d.G + vec % d.G;
            // positions this vector sees, and those that all of the tile's do
            const long long oend = end_of(it.b);
            const int room = pg_room(d);
            const int lim = qr >= m ? 0 : pt.shared ? d.shared_len : (int)max(0ll, min(oend - (m - 1 - qr), (long long)room));
            const int all = pt.shared ? d.shared_len : (int)max(0ll, min(oend - (m - 1 - it.t * C::TQ / d.G), (long long)room));
            {   // the warp's query vectors into the K-major order: chunk c of 8 dimensions of row r at chunk c ^ (r & 7) of its 128 bytes; four rows' 128 bytes at a time
                const u8* const src = qr < m ? io.q + (long long)(r0 + qr) * io.q_stride + (long long)head * HD * 2 : nullptr;
                u8* const dst = sq + q * C::QT + (warp & 3) * 4096;
#pragma unroll 4
                for (int i = 0; i < 8; i++) {
                    const int r = 4 * i + (lane >> 3), c = lane & 7;
                    const uint4* const from = (const uint4*)__shfl_sync(0xffffffffu, (unsigned long long)src, r);
#pragma unroll
                    for (int k = 0; k < HD / 64; k++) *(uint4*)(dst + k * C::QBLK + r * 128 + ((c ^ (r & 7)) << 4)) = from ? __ldg(from + 8 * k + c) : make_uint4(0, 0, 0, 0);
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                pt_arrive_warp(&S.q_full[q]);
            }
            float mx = -INFINITY, l = 0.f;                 // what the row's weights are divided by (its logarithm, base 2), their sum
            for (int j = 0; j < T; j++) {
                const int buf = q * 2 + (int)(done & 1);
                if (!pt_wait_warp(&S.s_full[buf], done >> 1)) { failed = 7; break; }
                pt_after();
                float s[C::UT];
                const u32 at = tmem + lanes + buf * C::UT;
#pragma unroll
                for (int k = 0; k < C::UT; k += 32) pt_ld32(at + k, s + k);
                const uint4 ok4 = *(const uint4*)S.ok[done & 7];
                const u32 ok[4] = {ok4.x, ok4.y, ok4.z, ok4.w};
                const int at_pos = (it.i + j) * C::UT, seen = lim - at_pos;
                const bool whole = __all_sync(0xffffffffu, seen >= C::UT && (ok[0] & ok[1] & (C::UT > 64 ? ok[2] & ok[3] : 0xffffffffu)) == 0xffffffffu);
#pragma unroll
                for (int k = 0; k < C::UT; k += 32) pt_loaded(s + k);
                if (!whole) {
#pragma unroll
                    for (int k = 0; k < C::UT; k++) s[k] = k < seen && (ok[k / 32] >> (k & 31)) & 1u ? s[k] : -INFINITY;
                }
                float big[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
                for (int k = 4; k < C::UT - 4; k += 8) {
#pragma unroll
                    for (int e = 0; e < 4; e++) big[e] = pt_max3(big[e], s[k + 2 * e], s[k + 2 * e + 1]);
                }
                const float top = pt_max3(pt_max3(big[0], big[1], s[C::UT - 4]), pt_max3(big[2], big[3], s[C::UT - 3]), pt_max3(s[C::UT - 2], s[C::UT - 1], s[C::UT - 1])) * io.scale_log2;
                if (!(top < INFINITY)) l = NAN;            // (a score that is NaN or infinite: so is the row)
                const bool up = top > mx + PT_TOP<BF> || (mx == -INFINITY && top > -INFINITY);
                if (__any_sync(0xffffffffu, up)) {
                    const float by = !up ? 1.f : mx == -INFINITY ? 0.f : pg_ex2(mx - (top - PT_UP<BF>));
                    if (up) { mx = top - PT_UP<BF>; l *= by; }
                    if (j > 0) {                           // the sums so far, once the last product is in them
                        if (!pt_wait_warp(&S.pv_done[q * 2 + ((done - 1) & 1)], (done - 1) >> 1)) { failed = 8; break; }
                        pt_after();
                        __syncwarp();
#pragma unroll 1
                        for (int k = 0; k < HD; k += 32) {
                            float o[32];
                            pt_ld32(tmem + lanes + 256 + q * HD + k, o);
                            pt_loaded(o);
#pragma unroll
                            for (int e = 0; e < 32; e++) o[e] *= by;
                            pt_st16(tmem + lanes + 256 + q * HD + k, (const u32*)o);
                            pt_st16(tmem + lanes + 256 + q * HD + k + 16, (const u32*)o + 16);
                        }
                    }
                    __syncwarp();
                }
                const float sub = mx == -INFINITY ? 0.f : mx;
                float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int k = 0; k < C::UT; k += 32) {
                    u32 w[16];
#pragma unroll
                    for (int e = 0; e < 32; e += 2) {
                        const float a = pg_ex2(fmaf(s[k + e], io.scale_log2, -sub)), b = pg_ex2(fmaf(s[k + e + 1], io.scale_log2, -sub));
                        sum[(e >> 1) & 3] += a + b;
                        w[e / 2] = pg_pack<CT>(a, b);
                    }
                    pt_st16(at + k / 2, w);
                }
                l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
                if (q == 0 && all < at_pos + C::UT) {      // the values that some row does not see
                    for (int nb = 0; nb < C::NB && !failed; nb++) {
                        const int sl = (int)((done * C::NB + nb) % C::SLOTS);
                        if (!pt_wait_warp(&S.full[1][sl], (done * C::NB + nb) / C::SLOTS)) { failed = 10; break; }
#pragma unroll 4
                        for (int x = tid; x < C::SLOT / 16; x += 128) {      // (a slot is blocks of 64 rows of 128 bytes)
                            uint4* const at16 = (uint4*)(vring + (size_t)sl * C::SLOT) + x;
                            const uint4 w = *at16;
                            const u32 in[4] = {w.x, w.y, w.z, w.w};
                            u32 out[4];
                            const bool behind = at_pos + (x >> 3) % C::UT >= it.end;
                            bool odd = false;
#pragma unroll
                            for (int k = 0; k < 4; k++) {
                                constexpr u32 X = BF ? 0x7f80u : 0x7c00u;
                                const u32 lo = (in[k] & X) == X ? 0u : 0xffffu, hi = (in[k] & (X << 16)) == (X << 16) ? 0u : 0xffff0000u;
                                odd |= (lo & hi >> 16) != 0xffffu;
                                out[k] = behind ? 0u : in[k] & (lo | hi);
                            }
                            if (behind || odd) *at16 = make_uint4(out[0], out[1], out[2], out[3]);
                            if (odd && !behind) S.odd[piece & 1] = piece + 1;
                        }
                    }
                    if (failed) break;
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                }
                pt_stored();
                pt_before();
                pt_arrive_warp(&S.p_full[buf]);
                done++;
            }
            // ---- the piece's part: (maximum, sum of weights, sums)
            if (!failed && !pt_wait_warp(&S.pv_done[q * 2 + ((done - 1) & 1)], (done - 1) >> 1)) failed = 9;
            if (failed) break;
            pt_after();
            const u32 us = units[it.e] * (u32)d.nkv + (u32)it.h * (u32)it.n;
            const int b0 = pg_block_of(share, us), b1 = pg_block_of(share, us + it.n - 1);
            const bool alone = b0 == b1, direct = alone && pt.direct, odd = S.odd[piece & 1] == piece + 1;
            const size_t to = alone ? (size_t)(r0 + qr) * (d.nkv * d.G) + head : (size_t)(2 * blockIdx.x + ((int)blockIdx.x == b0 ? 1 : 0)) * C::TQ + v;
            float* const w = qr < m ? (alone ? pt.row_o : pt.o) + to * HD : nullptr;
            // parts go out through the warp's own 4 KB of the queries' first block (whose products are done): a lane's own row, 16 bytes at a time,
            // would be 32 lines a store, 11,000 cycles for two tiles of 128 columns (the chunk of 2,045 rows 349 -> 314 us)
            u8* const turn = sq + q * C::QT + (warp & 3) * 4096;
            u8* const op = io.out + (long long)(r0 + qr) * io.out_stride + (long long)head * HD * 2;
            const u8* const gp = io.gate ? io.gate + (long long)(r0 + qr) * io.gate_stride + (long long)head * io.gate_head_stride : nullptr;
            const bool none = lim <= 0 || l == 0.f;
            const float inv = none ? 0.f : 1.f / l;
#pragma unroll 1
            for (int k = 0; k < HD; k += 32) {
                float o[32];
                __syncwarp();                                        // (loads from tensor memory want the whole warp, and not all lanes have a row to write)
                pt_ld32(tmem + lanes + 256 + q * HD + k, o);
                pt_loaded(o);
                if (odd && qr < m) {                                 // the values that were cleared, where this row sees them
                    const int32_t* table = pt.shared ? d.shared_pages : d.pages + (size_t)it.b * d.max_pages;
                    for (int t = max(it.i * C::UT, all & ~(C::UT - 1)); t < min(lim, (it.i + T) * C::UT); t++) {
                        const int page = __ldg(table + (t >> d.ps_log2));
                        if ((u32)page >= (u32)d.n_pages) continue;
                        const u8* src = d.v + (long long)page * d.page_stride + (long long)(t & ((1 << d.ps_log2) - 1)) * d.pos_stride + (long long)it.h * d.head_stride + 2 * k;
#pragma unroll
                        for (int e = 0; e < 32; e += 2) {
                            const float2 f = pg_unpack<CT>(*(const u32*)(src + 2 * e));
                            if (!isfinite(f.x)) o[e] += f.x;
                            if (!isfinite(f.y)) o[e + 1] += f.y;
                        }
                    }
                }
                if (!direct) {
#pragma unroll
                    for (int c = 0; c < 8; c++) *(float4*)(turn + lane * 128 + ((c ^ (lane & 7)) << 4)) = make_float4(o[4 * c], o[4 * c + 1], o[4 * c + 2], o[4 * c + 3]);
                    __syncwarp();
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        const int r = 4 * i + (lane >> 3), c = lane & 7;
                        float* const at = (float*)__shfl_sync(0xffffffffu, (unsigned long long)w, r);
                        const float4 f = *(const float4*)(turn + r * 128 + ((c ^ (r & 7)) << 4));
                        if (at) *(float4*)(at + k + 4 * c) = f;
                    }
                    __syncwarp();
                    continue;
                }
                if (qr < m) {
#pragma unroll
                    for (int e = 0; e < 32; e += 8) {
                        u32 y[4], z[4] = {};
                        if (gp) { const uint4 g = __ldg((const uint4*)(gp + 2 * (k + e))); z[0] = g.x; z[1] = g.y; z[2] = g.z; z[3] = g.w; }
#pragma unroll
                        for (int x = 0; x < 4; x++) {
                            float a = none ? 0.f : o[e + 2 * x] * inv, b = none ? 0.f : o[e + 2 * x + 1] * inv;
                            if (gp) { const float2 g = pg_unpack<CT>(z[x]); a *= sz_sigmoid(g.x); b *= sz_sigmoid(g.y); }
                            y[x] = pg_pack<CT>(a, b);
                        }
                        *(uint4*)(op + 2 * (k + e)) = make_uint4(y[0], y[1], y[2], y[3]);
                    }
                }
            }
            __syncwarp();
            if (l != l && mx == -INFINITY) mx = 0.f;       // (scores that are all NaN have no maximum, and are not an empty part)
            if (qr < m && !direct) (alone ? pt.row_ml : pt.ml)[to] = make_float2(mx, l);
            if (qr < m && direct && io.lse) io.lse[to] = none ? -INFINITY : (mx + log2f(l)) * 0.6931471805599453f;
            pt_before();
            pt_arrive_warp(&S.o_free[q]);
            u += T;
        }
        pt_stored();
    }
    sz_pdl_trigger();
    if (failed) atomicMax(&S.failed, (u32)failed);
    pt_before();
    __syncthreads();
    if (warp == 0) {
        pt_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
    if (tid == 0 && S.failed) atomicOr(d.err, PG_E_WAIT);
}

template <bool BF, int HD>
int pt_launch(const CUtensorMap* maps, int rows_box, const PgBatch& d, const PgIo& io, const PgPart& p, const char* name, cudaStream_t st) {
    using C = PtCfg<HD>;
    const int rc = sz_allow_smem((const void*)sz_pg_tc_kernel<BF, HD>, C::SMEM);
    if (rc) return rc;
    SZ_CUDA(sz_launch(name, sz_pg_tc_kernel<BF, HD>, dim3(p.blocks), dim3(C::NTH), C::SMEM, st, true, maps[0], maps[1], d, io, p, rows_box));
    return SZ_OK;
}

}  // namespace

int pg_tc_tile(int hd) { return hd <= 128 ? 256 : 128; }
int pg_tc_unit(int hd) { return hd == 64 ? PtCfg<64>::UT : hd == 128 ? PtCfg<128>::UT : PtCfg<256>::UT; }

int pg_tc_launch(bool bf16, int hd, const CUtensorMap* maps, int rows_box, const PgBatch& d, const PgIo& io, const PgPart& p, const char* name, cudaStream_t st) {
    if (bf16) return hd == 64 ? pt_launch<true, 64>(maps, rows_box, d, io, p, name, st) : hd == 128 ? pt_launch<true, 128>(maps, rows_box, d, io, p, name, st) : pt_launch<true, 256>(maps, rows_box, d, io, p, name, st);
    return hd == 64 ? pt_launch<false, 64>(maps, rows_box, d, io, p, name, st) : hd == 128 ? pt_launch<false, 128>(maps, rows_box, d, io, p, name, st) : pt_launch<false, 256>(maps, rows_box, d, io, p, name, st);
}
