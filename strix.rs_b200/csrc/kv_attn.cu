// Attention over a paged KV cache, ragged batches, grouped-query heads. Contract: include/strix_serve.h.
//
// out = softmax(scale q k^T) v, one pass over the cache with the running maximum and sum of a softmax. Decoding is a read of the
// cache: 4 * rows flops for each element of k and v, so HBM bounds it as long as the arithmetic of a cached element
// takes less than its share of the time (an SM gets about 23 bytes a clock).
//
// Arithmetic. The query heads that share a KV head are the rows of one f16 tensor-core product (mma m16n8k16, f32 sums). e4m3 and
// f16 cache values are exact in f16; q and the probabilities are not, and the results are held to f32 accuracy, so
// both go in as two f16 halves (value, and what rounding it left). Up to eight rows, the two halves ARE the sixteen
// rows of one product: rows 0..7 the values, rows 8..15 the remainders, and the two accumulators of a row meet in one thread.
// Beyond eight rows a warp has sixteen rows and issues two products. q is scaled by a power of two to use f16's range (a row's
// largest value in [2^14, 2^15)). Probabilities go in relative to the tile's largest, which becomes 2^15; where a tile holds pages of
// different scales, the largest product of weight and scale that the row has there goes to [2^14, 2^15) instead. So a weight is off by
// 2^-22 of itself or 2^-39 of the largest of its tile, and no page that a row does not see has a part in that. The sums over a tile
// start from zero and are added to the f32 running sums outside the tensor cores, which round to nearest: chained
// accumulation in the tensor cores truncates, a drift of its own over thousands of tokens.
// The order of the head's dimensions inside a product is free as long as q and k agree, and so is the order of the
// output columns: each thread takes the dimensions that lie next to each other in a cached row, so that shared memory is read in
// 16-byte words.
//
// Work split. A tile is TT tokens of one KV head (about 4 KB of k, as much of v). All tiles of all (sequence, row block, KV
// head) items stand in one line; block c of the grid takes an equal stretch of it, and each of the block's workers an equal part
// of that. A worker is a warp (or several, over the row blocks of a prompt) with a ring of half tiles (k, v, k, v, ...) of its
// own, which its first warp refills by bulk copies as soon as a half is done with: k is on its way again while v is multiplied.
// Page ids and scales are fetched 32 at a time, one to a lane. An item that one worker has whole is written out by it; the
// parts of the others meet in shared memory at the block's end, and where an item goes on in another block, in the workspace:
// the last block to arrive joins the parts, in the order of the line. Cuts that would fall into an item of at most PA_SNAP
// tiles move to its nearer end.
//
// Measured (32 heads, 8 KV heads of 128, e4m3): one row behind 131071 tokens 74 us (3.6 TB/s), 61 rows behind 500-16384 each
// 138 us (4.2 TB/s), one row behind 300 tokens 13.5 us. About 8 us of a call are its two ends (the place in the line, page ids and
// scales, q; the joins where items are shared); in between, instruction issue bounds: some 1000 instructions a tile, of which the
// fragments of k and v, their conversion and the two halves' products are two thirds. With four query heads to a KV head half of the
// sixteen rows of every product are empty, and a tile is 32 tokens (head size 128, e4m3), so what a tile costs besides is paid often.
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>
#include <atomic>

#include "kv_line.cuh"

namespace strix {

// Sizes that follow from the head size, the cache type and the row form (WIDE: 16 rows a warp, else 8).
template <int HD, int TYPE, bool WIDE>
struct PaShape {
    static constexpr int EL = TYPE == STRIX_KV_F16 ? 2 : 1;
    // warps: three to a scheduler where 168 registers do, else two (a wide row block of a large head has 16 rows of O: one)
    static constexpr int NW = HD >= 192 ? (WIDE ? 4 : 8) : (WIDE ? 8 : 12);
    static constexpr int ROWS = WIDE ? 16 : 8;                         // rows of a warp
    static constexpr int TT = HD * EL <= 64 ? 64 : HD * EL <= 128 ? 32 : 16;
    static constexpr int HALF = TT * HD * EL;                          // bytes of the k or the v of a tile
    // In shared memory a half tile is BOXES blocks of TT rows by BOXB bytes. Rows of a multiple of 128 bytes all start in the same
    // bank, so they come as blocks of 128-byte rows whose 16-byte words are swizzled (word c of row r at c ^ (r & 7)); rows of
    // 64, 96 and 192 bytes lie as they are.
    static constexpr bool SWZ = HD * EL % 128 == 0;
    static constexpr int BOXB = SWZ ? 128 : HD * EL, BOXES = HD * EL / BOXB;
    static constexpr int PSTRIDE = HD + 2;                             // floats of a partial row: sums, maximum, sum of weights
    static constexpr bool QSMEM = WIDE && HD >= 192;                   // q fragments in shared memory instead of registers
    static constexpr int QBYTES = QSMEM ? NW * 16 * HD * 4 : 0;
    static constexpr int SLOTS = NW * ROWS * PSTRIDE * 4;              // one partial for each worker
    static constexpr int DESCS = 8;                                    // tiles described at a time; above half the ring
    static constexpr int WORKER = 64 + DESCS * 64;
    __host__ __device__ static constexpr size_t fixed(int workers, int halves) { return SLOTS + QBYTES + workers * (WORKER + halves * 16); }
    // the rings, and the parts that take their place at the end
    __host__ __device__ static constexpr size_t rings(int workers, int halves) {
        return (size_t)workers * halves * HALF > SLOTS ? (size_t)workers * halves * HALF : SLOTS;
    }
    static int halves_for(int wm, size_t smem) {  // half tiles of a ring
        const int workers = NW / wm;
        int n = 2 * DESCS - 4;
#pragma unroll 1
        while (n > 1 && fixed(workers, n) + rings(workers, n) > smem) n--;
        return n;
    }
};

// What the joins need to know about a worker's open parts.
struct __align__(16) PaWorker {
    struct Part {
        uint32_t seq_first, seq_rows, row0, head, item0, item_tiles;
    };
    Part head, tail;
    uint32_t has_head, head_ended, has_tail, pad;
};

__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16_from0(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                 : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
template <int BYTES>
__device__ __forceinline__ void lds_words(uint32_t *w, const uint8_t *p) {
    if constexpr (BYTES == 16) {
        const uint4 u = *reinterpret_cast<const uint4 *>(p);
        w[0] = u.x; w[1] = u.y; w[2] = u.z; w[3] = u.w;
    } else if constexpr (BYTES == 8) {
        const uint2 u = *reinterpret_cast<const uint2 *>(p);
        w[0] = u.x; w[1] = u.y;
    } else {
        w[0] = *reinterpret_cast<const uint32_t *>(p);
    }
}

template <int HD, int TYPE, bool WIDE>
__global__ void __launch_bounds__(PaShape<HD, TYPE, WIDE>::NW * 32, 1) paged_attn_kernel(const __grid_constant__ PagedAttnArgs A) {
    using S = PaShape<HD, TYPE, WIDE>;
    constexpr int EL = S::EL, NW = S::NW, TT = S::TT, NT = TT / 8, KS = HD / 16;
    constexpr int PS = S::PSTRIDE, NO = HD / 8;           // NO: output tiles of eight columns
    constexpr int KW = (HD / 4 * EL) % 16 == 0 ? 16 : 8;  // bytes of a thread's k loads
    constexpr int KL = HD / 4 * EL / KW;                  // ... and how many a token
    constexpr int VB = HD / 8 * EL;                       // bytes of a cached value row that a thread turns into output columns
    constexpr int VW = S::SWZ ? 16 : VB % 16 == 0 ? 16 : VB % 8 == 0 ? 8 : 4, VL = VB / VW;
    // output column n of output tile i is dimension col_dim(n) + tile_dim(i): with swizzled rows a thread's columns are one
    // 16-byte word of each block of 128 bytes, else they are neighbours
    constexpr int WD = S::SWZ ? 16 / EL : NO;
    auto tile_dim = [](int i) { return i / WD * (S::BOXB / EL) + i % WD; };
    constexpr int RW = WIDE ? 2 : 1;                      // rows of a thread
    constexpr uint32_t DESCS = S::DESCS;
    extern __shared__ __align__(128) uint8_t smem_raw[];
    uint8_t *smem = smem_raw + (-smem_u32(smem_raw) & 1023u);  // (the swizzle goes by address)
    const PagedView &V = A.V;
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
    const uint32_t wm = WIDE ? A.wm : 1u, workers = NW / wm, rb = S::ROWS * wm, halves = A.halves;
    uint8_t *rings = smem;
    float *slots = reinterpret_cast<float *>(smem + S::rings(workers, halves));
    uint8_t *qsm = reinterpret_cast<uint8_t *>(slots) + S::SLOTS;
    PaTile *descs = reinterpret_cast<PaTile *>(qsm + S::QBYTES);
    PaWorker *info = reinterpret_cast<PaWorker *>(descs + workers * DESCS);
    uint64_t *full = reinterpret_cast<uint64_t *>(info + workers), *empty = full + workers * halves;
    __shared__ uint32_t last_here[2], scan[NW];
    __shared__ volatile uint32_t gave_up;

    // ---- running tile counts of the sequences (where the rings will be)
    uint32_t *upto = reinterpret_cast<uint32_t *>(rings);
    bool over;
    const uint32_t total = count_tiles<TT, NW * 32>(A, rb, upto, scan, over);
#pragma unroll 1
    for (uint32_t i = threadIdx.x; i < workers * halves; i += NW * 32) {
        mbar_init(&full[i], 1);
        mbar_init(&empty[i], wm);
        mbar_fence_init();
    }
#pragma unroll 1
    for (uint32_t i = threadIdx.x; i < workers * DESCS * 4u; i += NW * 32) descs[i / 4u].ks[i & 3u] = descs[i / 4u].vs[i & 3u] = 0.f;
    if (threadIdx.x == 0) gave_up = 0u;
    if (threadIdx.x < workers) info[threadIdx.x].has_head = info[threadIdx.x].head_ended = info[threadIdx.x].has_tail = 0u;

    // ---- this block's stretch of the line and this worker's part of it
    const uint32_t worker = warp / wm, wi = warp - worker * wm;  // warp of the worker
    const uint32_t line_blocks = min(gridDim.x, (total + workers - 1u) / workers);  // blocks with work
    uint32_t n_block = 0, n_mine = 0;
    PaPlace place{};
    if (blockIdx.x < line_blocks) {
        const PaCuts line(total, line_blocks);
        uint32_t x = line.cut(blockIdx.x + (lane & 1u));
        if (x < total) {
            find_place<TT>(A, rb, upto, x, place);
            x = snapped(place, x, PA_SNAP);
        }
        const uint32_t lo = __shfl_sync(0xffffffffu, x, 0), hi = __shfl_sync(0xffffffffu, x, 1);
        n_block = hi - lo;
        if (n_block) {
            const PaCuts mine(n_block, workers);
            const uint32_t w0 = mine.cut(worker);
            n_mine = mine.cut(worker + 1u) - w0;
            if (n_mine) find_place<TT>(A, rb, upto, lo + w0, place);
        }
    }
    fence_proxy_async_smem();  // copies land where the counts were: all accesses to them come first
    __syncthreads();
    uint8_t *ring = rings + (size_t)worker * halves * S::HALF;
    PaTile *desc = descs + worker * DESCS;
    full += worker * halves;
    empty += worker * halves;

    // ---- the worker's first warp: copies of the next half tile. All of this is the same in every lane but the batch.
    uint32_t is_half = 0, is_tile = 0, is_left = 2u * n_mine;  // ring place, tile and number of the halves still to be issued
    uint32_t ds_half = 0, ds_tile = 0, ds_from = 0, ds_left = is_left;  // the same of those still to be described
    uint32_t b_from = 0, b_stop = 0, seg_stop = 0;             // batch: its next lane, its end and the segment's in tiles of the item
    uint32_t new_flag = 0, end_flag = 0;
    bool started = false;
    int b_page = -1, c_page = -1;                              // this lane's page of the batch; of the tile whose k went last
    float b_ks = 0.f, b_vs = 0.f;
    uint32_t c_y = 0;
    bool bad = false;
    b_stop = seg_stop = place.at;
    const uint32_t sub = TT > 16 ? min((uint32_t)TT, V.page_tokens) : 16u;  // tokens of a copy
    const uint32_t sub_shift = TT / sub == 4u ? 2u : TT / sub == 2u ? 1u : 0u, n_sub = 1u << sub_shift, sub_at = lane & (n_sub - 1u);
    const bool leader = elect_lane();
    // Completes the description of the next issued half: the scales came last from memory, the copies did not wait for them.
    auto describe = [&] {
        if ((ds_left & 1u) == 0u) {
            if (lane - ds_from < n_sub) {
                desc[ds_tile].ks[lane - ds_from] = b_ks;
                desc[ds_tile].vs[lane - ds_from] = b_vs;
            }
            ds_from += n_sub;
            ds_tile = (ds_tile + 1u) & (DESCS - 1u);
            __syncwarp();
        }
        if (leader) mbar_arrive(&full[ds_half]);
        if (++ds_half == halves) ds_half = 0;
        ds_left--;
    };
    // The next segment, if one has ended, and the page ids and scales of its next 32 pages.
    auto next_batch = [&] {
#pragma unroll 1
        while (ds_left > is_left) describe();
        if (place.at == seg_stop) {
            if (started) next_item<TT>(A, rb, place);
            started = true;
            const uint32_t left = is_left / 2u, seg = min(left, place.tiles - place.at);
            const bool ends = place.at + seg == place.tiles;
            seg_stop = place.at + seg;
            new_flag = PA_NEW;
            end_flag = PA_END | (place.at ? PA_HEAD : ends ? PA_WHOLE : 0u);
            if (lane == 0) {  // how the segment relates to its item
                const PaWorker::Part part{place.first, place.rows, place.mb * rb, place.head, place.item0, place.tiles};
                PaWorker *me = info + worker;
                if (place.at) {
                    me->head = part;
                    me->has_head = 1u;
                    me->head_ended = ends;
                } else if (!ends) {
                    me->tail = part;
                    me->has_tail = 1u;
                }
            }
        }
        ds_from = b_from = 0;
        const uint32_t n = min(32u >> sub_shift, seg_stop - place.at);
        b_stop = place.at + n;
        const uint32_t tok = (place.lo_tile + place.at) * TT + lane * sub, nth = tok >> V.page_shift;
        b_page = -1;
        b_ks = b_vs = 0.f;
        if (lane < n << sub_shift && tok <= place.ctx + (place.rows - 1u) && nth < V.pages_ld &&
            still_seen(A, rb, place.ctx, place.mb, tok + sub - 1u)) {
            b_page = V.pages[(size_t)place.s * V.pages_ld + nth];
            if (b_page < 0 || (uint32_t)b_page >= V.n_pages) {
                b_page = -1;
                bad = true;
            } else if (TYPE == STRIX_KV_E4M3) {
                b_ks = V.k_scale[(size_t)b_page * V.n_kv + place.head];
                b_vs = V.v_scale[(size_t)b_page * V.n_kv + place.head];
            } else {
                b_ks = b_vs = 1.f;
            }
        }
    };
    auto issue = [&] {
        const bool is_v = is_left & 1u;
        if (!is_v) {  // k: a new tile
            if (place.at == b_stop) next_batch();
            const uint32_t tile = place.lo_tile + place.at;
            c_page = __shfl_sync(0xffffffffu, b_page, b_from + sub_at);
            c_y = place.head * V.page_tokens + ((tile * TT + sub_at * sub) & (V.page_tokens - 1u));
            const uint32_t valid = __ballot_sync(0xffffffffu, c_page >= 0) & ((1u << n_sub) - 1u);
            if (lane == 0) {
                PaTile &d = desc[is_tile];
                *reinterpret_cast<uint4 *>(&d.tile) = make_uint4(tile, new_flag | (place.at + 1u == seg_stop ? end_flag : 0u), valid, place.mb * rb);
                if (new_flag) *reinterpret_cast<uint4 *>(&d.seq_first) = make_uint4(place.first, place.rows, place.ctx, place.head);
            }
            __syncwarp();
            new_flag = 0u;
            b_from += n_sub;
            place.at++;
            is_tile = (is_tile + 1u) & (DESCS - 1u);
        }
        uint64_t *bar = &full[is_half];
        uint8_t *dst = ring + is_half * S::HALF;
        const CUtensorMap *map = is_v ? &A.v_map : &A.k_map;
#pragma unroll 1
        for (uint32_t i = 0; i < n_sub; i++) {
            const int page = TT > 16 ? __shfl_sync(0xffffffffu, c_page, i) : c_page;
            const uint32_t y = TT > 16 ? __shfl_sync(0xffffffffu, c_y, i) : c_y;
            if (page >= 0 && leader) {
                mbar_expect_tx(bar, sub * HD * EL);
#pragma unroll
                for (int box = 0; box < S::BOXES; box++)
                    tma_load_3d(dst + box * (TT * S::BOXB) + i * sub * S::BOXB, map, box * (S::BOXB / EL), y, (uint32_t)page, bar);
            }
        }
        if (++is_half == halves) is_half = 0;
        is_left--;
    };

    bad |= over || empty_rows<HD, TT>(A, rb, warp, NW);

    // ---- the loop over half tiles: k to weights, v to sums. The worker's first warp runs ahead by a ring.
    float o[NO][2 * RW], m[RW], l[RW];
    bool open_tail = false;
    const uint32_t g = lane >> 2, t = lane & 3u;   // row and column of the fragments
    // Column n of eight tokens is token n ^ 4 for odd n: with the swizzle, that spreads the words that eight neighbouring
    // threads read over all banks, in k (rows g, g + 1) and in v (rows of columns 2 t, or 2 t + 1, and words g, g + 1).
    const uint32_t kr = g ^ ((g & 1u) << 2), vr[2] = {2u * t, (2u * t + 1u) ^ 4u};
    const uint32_t k_off[2] = {S::SWZ ? kr * 128u + ((t ^ kr) << 4) : kr * (HD * EL) + t * KW, S::SWZ ? kr * 128u + (((t + 4u) ^ kr) << 4) : 0u};
    const uint32_t v_off[2] = {S::SWZ ? vr[0] * 128u + ((g ^ vr[0]) << 4) : vr[0] * (HD * EL) + g * VB,
                               S::SWZ ? vr[1] * 128u + ((g ^ vr[1]) << 4) : vr[1] * (HD * EL) + g * VB};
    uint32_t half = 0, phase = 0, e_half = 0, e_phase = 0;  // next half to use; next to refill
    uint32_t qf[S::QSMEM ? 1 : KS][WIDE ? 8 : 4];  // fragments of q: values (and remainders, in the same rows or apart)
    uint4 *qs = reinterpret_cast<uint4 *>(qsm) + warp * (KS * 2 * 32) + lane;
    float qc[RW], wv[RW];                          // factor from the products to exponents of two; of the tile's sums: weight and scale
    uint32_t pos[RW], pos_lo = 0, pos_hi = 0;      // positions of this thread's rows, of the warp's first and last row
    uint32_t pf[TT / 16][WIDE ? 8 : 4];            // fragments of the weights
    bool tail_tok = false;
    uint32_t it_first = 0, it_rows = 0, it_row0 = 0, it_head = 0;  // the item: first row of its sequence, new rows, first row of its own, KV head
    const int steps = (int)(2u * n_mine);
    // by whole warps, whose lanes come to the same answer; a wait that has run out ends all others of the block
    auto wait = [&](uint64_t *bar, uint32_t parity) {
#pragma unroll 1
        for (uint32_t it = 0; !__all_sync(0xffffffffu, mbar_try_wait(bar, parity)); it++)
            if (__any_sync(0xffffffffu, gave_up || it >= 1u << 22)) {
                gave_up = 1u;
                return false;
            }
        return true;
    };
#pragma unroll 1
    for (int step = wi == 0 ? -(int)min(halves, 2u * n_mine) : 0; step < steps; step++) {
        if (step >= 0) {
        const PaTile &d = desc[(uint32_t)step / 2u & (DESCS - 1u)];
        if ((step & 1) == 0) {
            if (wm > 1u) {  // (the other warps get the description with the copy)
                if (wi == 0)
#pragma unroll 1
                    while (ds_left > is_left) describe();
                if (!wait(&full[half], phase)) break;
            }
            if (d.flags & PA_NEW) {
                it_first = d.seq_first;
                it_rows = d.seq_rows;
                it_row0 = d.row0;
                it_head = d.head;
                const uint32_t R = d.seq_rows * A.group, rw = d.row0 + wi * S::ROWS;
                const float *qrow[RW];
                bool on[RW];
#pragma unroll
                for (int i = 0; i < RW; i++) {
                    const uint32_t r = rw + g + 8u * i;
                    on[i] = r < R;
                    const uint32_t rr = min(r, R - 1u), tk = by_group(A, rr);
                    pos[i] = d.ctx + tk;
                    qrow[i] = A.q + (size_t)(d.seq_first + tk) * A.ld_q + (size_t)(d.head * A.group + rr - tk * A.group) * HD;
                }
                pos_lo = d.ctx + by_group(A, min(rw, R - 1u));
                pos_hi = d.ctx + by_group(A, min(rw + S::ROWS - 1u, R - 1u));
                float x[RW][KS][4];
#pragma unroll
                for (int i = 0; i < RW; i++) {
                    float top = 0.f;
#pragma unroll
                    for (int s = 0; s < KS; s++) {
                        // the four dimensions of k-step s in this thread: neighbours in the cached row
                        const uint32_t dim = EL == 1 ? (s / (KW / 4)) * 4 * KW + t * KW + (s % (KW / 4)) * 4 : (s / 2) * 32 + t * 8 + (s % 2) * 4;
                        if (on[i]) {
                            if (A.vec) {
                                const float4 f = *reinterpret_cast<const float4 *>(qrow[i] + dim);
                                x[i][s][0] = f.x; x[i][s][1] = f.y; x[i][s][2] = f.z; x[i][s][3] = f.w;
                            } else {
#pragma unroll
                                for (int e = 0; e < 4; e++) x[i][s][e] = qrow[i][dim + e];
                            }
                        } else {
#pragma unroll
                            for (int e = 0; e < 4; e++) x[i][s][e] = 0.f;
                        }
#pragma unroll
                        for (int e = 0; e < 4; e++) top = fmaxf(top, fabsf(x[i][s][e]));
                    }
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                    // 2^e with top 2^e in [2^14, 2^15); rows of zeros or with infinities as they are
                    const int ex = (int)(__float_as_uint(top) >> 23);
                    const int e2 = top > 0.f && ex < 255 ? min(126, max(-126, 14 + 127 - max(ex, 1))) : 0;
                    const float up = __uint_as_float((uint32_t)(e2 + 127) << 23);
                    qc[i] = A.scale * (1.4426950408889634f * __uint_as_float((uint32_t)(127 - e2) << 23));
#pragma unroll
                    for (int s = 0; s < KS; s++)
#pragma unroll
                        for (int e = 0; e < 4; e++) x[i][s][e] *= up;
                    m[i] = -INFINITY;
                    l[i] = 0.f;
                }
#pragma unroll
                for (int s = 0; s < KS; s++) {
                    uint32_t f[WIDE ? 8 : 4];
                    if constexpr (WIDE) {  // a fragment: row g, row g + 8, row g, row g + 8; the remainders behind
                        split2(x[0][s][0], x[0][s][1], f[0], f[4]);
                        split2(x[RW - 1][s][0], x[RW - 1][s][1], f[1], f[5]);
                        split2(x[0][s][2], x[0][s][3], f[2], f[6]);
                        split2(x[RW - 1][s][2], x[RW - 1][s][3], f[3], f[7]);
                    } else {
                        split2(x[0][s][0], x[0][s][1], f[0], f[1]);
                        split2(x[0][s][2], x[0][s][3], f[2], f[3]);
                    }
                    if constexpr (S::QSMEM) {
                        qs[(2 * s) * 32] = make_uint4(f[0], f[1], f[2], f[3]);
                        qs[(2 * s + 1) * 32] = make_uint4(f[4], f[5], f[6], f[7]);
                    } else {
#pragma unroll
                        for (int e = 0; e < (WIDE ? 8 : 4); e++) qf[s][e] = f[e];
                    }
                }
#pragma unroll
                for (int i = 0; i < NO; i++)
#pragma unroll
                    for (int e = 0; e < 2 * RW; e++) o[i][e] = 0.f;
            }

            // scores: products of q with eight tokens at a time
            if (wm == 1u) {
#pragma unroll 1
                while (ds_left > is_left) describe();
                if (!wait(&full[half], phase)) break;
            }
            const uint8_t *ks = ring + half * S::HALF;
            const uint32_t tok = d.tile * TT, valid = d.valid;
            float sc[NT][4];
            // (the token groups go side by side: a product waits for the one before it on the same sums)
#pragma unroll
            for (int i = 0; i < KL; i++) {
                uint32_t w[NT][KW / 4];
#pragma unroll
                for (int j = 0; j < NT; j++)
                    lds_words<KW>(w[j], S::SWZ ? ks + k_off[i & 1] + (i >> 1) * (TT * 128) + j * 1024 : ks + k_off[0] + j * (8 * HD * EL) + i * 4 * KW);
#pragma unroll
                for (int x = 0; x < KW * 4 / (16 * EL); x++) {
                    const int s = i * (KW * 4 / (16 * EL)) + x;
                    uint32_t b0[NT], b1[NT];
#pragma unroll
                    for (int j = 0; j < NT; j++) {
                        if constexpr (EL == 1) {
                            e4m3x4_to_f16x2(w[j][x], b0[j], b1[j]);
                        } else {
                            b0[j] = w[j][2 * x];
                            b1[j] = w[j][2 * x + 1];
                        }
                    }
                    if constexpr (!WIDE) {
                        const uint32_t(&q)[4] = reinterpret_cast<const uint32_t(&)[4]>(qf[s]);
#pragma unroll
                        for (int j = 0; j < NT; j++) {
                            if (s == 0) mma_f16_from0(sc[j], q, b0[j], b1[j]);
                            else mma_f16(sc[j], q, b0[j], b1[j]);
                        }
                    } else {
                        uint4 h4, l4;
                        if constexpr (S::QSMEM) {
                            h4 = qs[(2 * s) * 32];
                            l4 = qs[(2 * s + 1) * 32];
                        } else {
                            h4 = make_uint4(qf[s][0], qf[s][1], qf[s][2], qf[s][3]);
                            l4 = make_uint4(qf[s][4], qf[s][5], qf[s][6], qf[s][7]);
                        }
                        const uint32_t hi[4] = {h4.x, h4.y, h4.z, h4.w}, lo[4] = {l4.x, l4.y, l4.z, l4.w};
#pragma unroll
                        for (int j = 0; j < NT; j++) {
                            if (s == 0) mma_f16_from0(sc[j], lo, b0[j], b1[j]);
                            else mma_f16(sc[j], lo, b0[j], b1[j]);
                        }
#pragma unroll
                        for (int j = 0; j < NT; j++) mma_f16(sc[j], hi, b0[j], b1[j]);
                    }
                }
            }
            // to exponents of two; scale of the page; masks
            const uint32_t pshift = V.page_shift;
            const bool mixed = TT > 16 && V.page_tokens < TT;  // several pages in a tile
            const bool all = valid == (mixed ? (1u << (TT >> pshift)) - 1u : 1u);
            tail_tok = __any_sync(0xffffffffu, tok + TT - 1u > pos_hi || !all);  // tokens that no row of the warp sees, maybe never written
            float k0 = d.ks[0];  // the largest scale of the tile's pages
            const bool several = TT > 16 && __any_sync(0xffffffffu, mixed);
            if (several) k0 = fmaxf(fmaxf(k0, d.ks[1]), fmaxf(d.ks[2], d.ks[3]));
#pragma unroll
            for (int j = 0; j < NT; j++) {
                if constexpr (!WIDE) {
                    sc[j][0] = (sc[j][0] + sc[j][2]) * (k0 * qc[0]);
                    sc[j][1] = (sc[j][1] + sc[j][3]) * (k0 * qc[0]);
                } else {
                    sc[j][0] *= k0 * qc[0];
                    sc[j][1] *= k0 * qc[0];
                    sc[j][2] *= k0 * qc[RW - 1];
                    sc[j][3] *= k0 * qc[RW - 1];
                }
            }
            if (several) {  // scores take what another page's scale differs by
                const float rk0 = k0 > 0.f ? 1.0f / k0 : 0.f;
#pragma unroll
                for (int j = 0; j < NT; j++) {
                    const float f = d.ks[(8u * j) >> pshift] * rk0;
#pragma unroll
                    for (int e = 0; e < 2 * RW; e++) sc[j][e] *= f;
                }
            }
            if (__any_sync(0xffffffffu, tail_tok || tok + TT - 1u > pos_lo || (A.window && pos_hi >= A.window && tok <= pos_hi - A.window))) {
#pragma unroll
                for (int j = 0; j < NT; j++) {
                    const bool there = (valid >> (mixed ? (8u * j) >> pshift : 0u)) & 1u;
#pragma unroll
                    for (int e = 0; e < 2 * RW; e++) {
                        const uint32_t tk = tok + 8u * j + vr[e & 1], p = pos[e >> 1];
                        const bool see = tk <= p && (!A.window || p < A.window || tk > p - A.window) && there;
                        sc[j][e] = see ? sc[j][e] : -INFINITY;
                    }
                }
            }
            // weights are relative to the tile's own maximum, so that what two halves lose of them goes by the tile and not by the largest
            // score so far: a tile of small weights may hold the large values
            float mx[RW];
#pragma unroll
            for (int i = 0; i < RW; i++) mx[i] = -INFINITY;
#pragma unroll
            for (int j = 0; j < NT; j++)
#pragma unroll
                for (int e = 0; e < 2 * RW; e++) mx[e >> 1] = fmaxf(mx[e >> 1], sc[j][e]);
            bool moved = false;
#pragma unroll
            for (int i = 0; i < RW; i++) {
                mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 1));
                mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 2));
                moved |= mx[i] > m[i];
            }
            if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
                for (int i = 0; i < RW; i++) {
                    const float a = mx[i] > m[i] ? ex2(m[i] - mx[i]) : 1.f;
                    m[i] = fmaxf(m[i], mx[i]);
                    l[i] *= a;
#pragma unroll
                    for (int k = 0; k < NO; k++) {
                        o[k][2 * i] *= a;
                        o[k][2 * i + 1] *= a;
                    }
                }
            }
            float base[RW], lt[RW];
#pragma unroll
            for (int i = 0; i < RW; i++) {
                // weights carry 2^15, as their sum does (rounded up: scores of 2^24 and more would else give 2^16, which f16 does not have)
                base[i] = mx[i] == -INFINITY ? 0.f : __fsub_ru(mx[i], 15.f);
                lt[i] = 0.f;
                wv[i] = mx[i] == m[i] ? 1.f : ex2(mx[i] - m[i]);
            }
#pragma unroll
            for (int j = 0; j < NT; j++)
#pragma unroll
                for (int e = 0; e < 2 * RW; e++) {
                    sc[j][e] = ex2(sc[j][e] - base[e >> 1]);
                    lt[e >> 1] += sc[j][e];
                }
#pragma unroll
            for (int i = 0; i < RW; i++) l[i] = fmaf(lt[i], wv[i], l[i]);
            if (EL == 1 && several) {
                float top[RW], up[RW];
#pragma unroll
                for (int i = 0; i < RW; i++) top[i] = 0.f;
#pragma unroll
                for (int j = 0; j < NT; j++)
#pragma unroll
                    for (int e = 0; e < 2 * RW; e++) top[e >> 1] = fmaxf(top[e >> 1], sc[j][e] * (d.vs[(8u * j) >> pshift] * 0x1p-15f));
#pragma unroll
                for (int i = 0; i < RW; i++) {
                    float back;
                    top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 1));
                    top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 2));
                    row_scale(top[i], up[i], back);
                    wv[i] *= back;
                }
#pragma unroll
                for (int j = 0; j < NT; j++)
#pragma unroll
                    for (int e = 0; e < 2 * RW; e++) sc[j][e] *= page_factor(d.vs[(8u * j) >> pshift] * 0x1p-15f, up[e >> 1]);
            } else if (EL == 1) {
#pragma unroll
                for (int i = 0; i < RW; i++) wv[i] *= d.vs[0];
            }
#pragma unroll
            for (int j = 0; j < NT; j++) {
                const float(&p)[4] = sc[j];
                const int u = j / 2, hf = (j & 1) * 2;
                if constexpr (!WIDE) {
                    split2(p[0], p[1], pf[u][hf], pf[u][hf + 1]);
                } else {
                    split2(p[0], p[1], pf[u][hf], pf[u][4 + hf]);
                    split2(p[2], p[3], pf[u][hf + 1], pf[u][4 + hf + 1]);
                }
            }
        } else {
            if (wi == 0)
#pragma unroll 1
                while (ds_left > is_left) describe();
            if (!wait(&full[half], phase)) break;
            const uint8_t *vs = ring + half * S::HALF;
            const uint32_t tok = d.tile * TT, valid = d.valid, pshift = V.page_shift;
            const bool mixed = TT > 16 && V.page_tokens < TT;
            // weighted values: thread (g, t) reads its output columns of the four tokens its weights are for
#pragma unroll
            for (int c = 0; c < VL; c++) {
                uint32_t r[TT / 16][4][VW / 4];
#pragma unroll
                for (int u = 0; u < TT / 16; u++)
#pragma unroll
                    for (int k = 0; k < 4; k++)
                        lds_words<VW>(r[u][k], vs + v_off[k & 1] + (S::SWZ ? c * (TT * 128) + (16 * u + 8 * (k >> 1)) * 128
                                                                            : c * VW + (16 * u + 8 * (k >> 1)) * (HD * EL)));
                if (__any_sync(0xffffffffu, tail_tok)) {  // what no row sees may hold anything: zeros
#pragma unroll
                    for (int u = 0; u < TT / 16; u++)
#pragma unroll
                        for (int k = 0; k < 4; k++) {
                            const uint32_t row = 16u * u + vr[k & 1] + 8u * (k >> 1);
                            const uint32_t keep = tok + row <= pos_hi && ((valid >> (mixed ? row >> pshift : 0u)) & 1u) ? 0xffffffffu : 0u;
#pragma unroll
                            for (int w = 0; w < VW / 4; w++) r[u][k][w] &= keep;
                        }
                }
#pragma unroll
                for (int w = 0; w < VW / 4; w++) {
                    constexpr int PER = 4 / EL;  // dimensions of a word
                    float acc[PER][4];
#pragma unroll
                    for (int u = 0; u < TT / 16; u++) {
                        uint32_t b0[PER], b1[PER];
                        if constexpr (EL == 1) {
                            const uint32_t a = __byte_perm(r[u][0][w], r[u][1][w], 0x5140), b = __byte_perm(r[u][0][w], r[u][1][w], 0x7362);
                            const uint32_t cc = __byte_perm(r[u][2][w], r[u][3][w], 0x5140), dd = __byte_perm(r[u][2][w], r[u][3][w], 0x7362);
                            e4m3x4_to_f16x2(a, b0[0], b0[1]);
                            e4m3x4_to_f16x2(b, b0[2 % PER], b0[3 % PER]);
                            e4m3x4_to_f16x2(cc, b1[0], b1[1]);
                            e4m3x4_to_f16x2(dd, b1[2 % PER], b1[3 % PER]);
                        } else {
                            b0[0] = __byte_perm(r[u][0][w], r[u][1][w], 0x5410);
                            b0[1] = __byte_perm(r[u][0][w], r[u][1][w], 0x7632);
                            b1[0] = __byte_perm(r[u][2][w], r[u][3][w], 0x5410);
                            b1[1] = __byte_perm(r[u][2][w], r[u][3][w], 0x7632);
                        }
                        if constexpr (!WIDE) {
                            const uint32_t(&p)[4] = reinterpret_cast<const uint32_t(&)[4]>(pf[u]);
#pragma unroll
                            for (int e = 0; e < PER; e++) {
                                if (u == 0) mma_f16_from0(acc[e], p, b0[e], b1[e]);
                                else mma_f16(acc[e], p, b0[e], b1[e]);
                            }
                        } else {
                            const uint32_t hi[4] = {pf[u][0], pf[u][1], pf[u][2], pf[u][3]}, lo[4] = {pf[u][4], pf[u][5], pf[u][6], pf[u][7]};
#pragma unroll
                            for (int e = 0; e < PER; e++) {
                                if (u == 0) mma_f16_from0(acc[e], lo, b0[e], b1[e]);
                                else mma_f16(acc[e], lo, b0[e], b1[e]);
                            }
#pragma unroll
                            for (int e = 0; e < PER; e++) mma_f16(acc[e], hi, b0[e], b1[e]);
                        }
                    }
#pragma unroll
                    for (int e = 0; e < PER; e++) {
                        float(&oo)[2 * RW] = o[(c * (VW / 4) + w) * PER + e];
                        if constexpr (!WIDE) {
                            oo[0] = fmaf(acc[e][0] + acc[e][2], wv[0], oo[0]);
                            oo[1] = fmaf(acc[e][1] + acc[e][3], wv[0], oo[1]);
                        } else {
#pragma unroll
                            for (int k = 0; k < 2 * RW; k++) oo[k] = fmaf(acc[e][k], wv[k >> 1], oo[k]);
                        }
                    }
                }
            }
            const uint32_t flags = d.flags;
            if (flags & PA_END) {
            // the segment's end: the row sums of four threads meet
#pragma unroll
            for (int i = 0; i < RW; i++) {
                l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
                l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
            }
            if (flags & PA_WHOLE) {
#pragma unroll
                for (int i = 0; i < RW; i++) {
                    const uint32_t r = it_row0 + wi * S::ROWS + g + 8u * i, tk = by_group(A, r);
                    if (r >= it_rows * A.group) continue;
                    const float inv = l[i] == 0.f ? 0.f : 1.0f / l[i];
                    float *dst = A.out + (size_t)(it_first + tk) * A.ld_out + (size_t)(it_head * A.group + r - tk * A.group) * HD;
#pragma unroll
                    for (int e = 0; e < 2; e++) {  // columns 2 t and 2 t + 1 of the products
                        float *q = dst + (2u * t + e) * WD;
                        if (A.vec) {
#pragma unroll
                            for (int k = 0; k < NO; k += 4)
                                *reinterpret_cast<float4 *>(q + tile_dim(k)) = make_float4(o[k][2 * i + e] * inv, o[k + 1][2 * i + e] * inv,
                                                                                 o[k + 2][2 * i + e] * inv, o[k + 3][2 * i + e] * inv);
                        } else {
#pragma unroll
                            for (int k = 0; k < NO; k++) q[tile_dim(k)] = o[k][2 * i + e] * inv;
                        }
                    }
                }
            } else if (flags & PA_HEAD) {
#pragma unroll
                for (int i = 0; i < RW; i++) {
                    float *dst = slots + (size_t)(warp * S::ROWS + g + 8u * i) * PS;
#pragma unroll
                    for (int k = 0; k < NO; k += 2) {
                        *reinterpret_cast<float2 *>(dst + 2u * t * WD + tile_dim(k)) = make_float2(o[k][2 * i], o[k + 1][2 * i]);
                        *reinterpret_cast<float2 *>(dst + (2u * t + 1u) * WD + tile_dim(k)) = make_float2(o[k][2 * i + 1], o[k + 1][2 * i + 1]);
                    }
                    if (t == 0) {
                        dst[HD] = m[i];
                        dst[HD + 1] = l[i];
                    }
                }
            } else {
                open_tail = true;
            }
            }
        }
        __syncwarp();  // the half is done with
        if (wm > 1u && lane == 0) mbar_arrive(&empty[half]);
        if (++half == halves) {
            half = 0;
            phase ^= 1u;
        }
        }
        // refill: alone, a warp refills the half it has just used; with others, the one before, which they have mostly left as well
        if (wi == 0 && is_left && (step < 0 || wm == 1u || step > 0)) {
            if (step > 0 && wm > 1u) {
                if (!wait(&empty[e_half], e_phase)) break;  // (nothing is copied over what others may still read)
                if (++e_half == halves) {
                    e_half = 0;
                    e_phase ^= 1u;
                }
            }
            issue();
        }
    }
    report_bad(V, bad);

    // ---- parts of items that more than one worker has: tails go where the rings were
    __syncthreads();
    if (gave_up) {  // copies may still be under way: nothing takes their place, and they end before the block does
        if (threadIdx.x == 0 && V.status) atomicOr(V.status, STATUS_WAIT_TIMEOUT);
#pragma unroll 1
        for (int i = 0; i < 64; i++) __nanosleep(100000u);
        return;
    }
    float *tails = reinterpret_cast<float *>(rings);
    if (open_tail) {
#pragma unroll
        for (int i = 0; i < RW; i++) {
            float *dst = tails + (size_t)(warp * S::ROWS + g + 8u * i) * PS;
#pragma unroll
            for (int k = 0; k < NO; k += 2) {
                *reinterpret_cast<float2 *>(dst + 2u * t * WD + tile_dim(k)) = make_float2(o[k][2 * i], o[k + 1][2 * i]);
                *reinterpret_cast<float2 *>(dst + (2u * t + 1u) * WD + tile_dim(k)) = make_float2(o[k][2 * i + 1], o[k + 1][2 * i + 1]);
            }
            if (t == 0) {
                dst[HD] = m[i];
                dst[HD + 1] = l[i];
            }
        }
    }
    __syncthreads();
    if (n_block == 0u) return;
    // Chains of parts: [the tail of worker a and] heads of the workers behind it up to the one where the item ends. One without a
    // tail comes from the block in front, one without an end goes on in the next. A warp joins a row at a time.
    uint32_t heads, ends, tail_set;
    {
        const bool on = lane < workers;
        heads = __ballot_sync(0xffffffffu, on && info[min(lane, workers - 1u)].has_head);
        ends = __ballot_sync(0xffffffffu, on && info[min(lane, workers - 1u)].head_ended);
        tail_set = __ballot_sync(0xffffffffu, on && info[min(lane, workers - 1u)].has_tail);
    }
    const bool front = heads && (tail_set == 0u || __ffs(heads) <= __ffs(tail_set));
    const uint32_t chains = __popc(tail_set) + front;
    constexpr int DL = (HD / 2 + 31) / 32;  // pairs of a row in a lane
    const PaWorker::Part *cross[2] = {nullptr, nullptr};  // the item that goes on in front, and behind
#pragma unroll 1
    for (uint32_t c = 0, left = tail_set; c < chains; c++) {
        int a = -1;
        if (c > 0u || !front) {
            a = __ffs(left) - 1;
            left &= left - 1u;
        }
        const uint32_t behind = a < 0 ? 0xffffffffu : a == 31 ? 0u : ~0u << (a + 1);
        const uint32_t stop = ends & behind;
        const uint32_t members = heads & behind & (stop ? (stop & -stop) | ((stop & -stop) - 1u) : 0xffffffffu);
        const PaWorker::Part &it = a < 0 ? info[__ffs(members) - 1].head : info[a].tail;
        const bool out = a < 0 || stop == 0u;
        if (out) cross[a < 0 ? 0 : 1] = &it;
        const uint32_t R = min(rb, it.seq_rows * A.group - it.row0);
#pragma unroll 1
        for (uint32_t row = (warp + NW - c % NW) % NW; row < R; row += NW) {
            const bool tl = (int)lane == a, mine = tl || ((members >> lane) & 1u);
            const float *p = (tl ? tails : slots) + (size_t)((mine ? lane : 0u) * rb + row) * PS;
            const float pm = mine ? p[HD] : -INFINITY;
            float M = pm;
#pragma unroll
            for (int d = 16; d > 0; d >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, d));
            const float f = pm == -INFINITY ? 0.f : ex2(pm - M);
            const float L = warp_sum(mine ? f * p[HD + 1] : 0.f);
            float2 acc[DL];
#pragma unroll
            for (int k = 0; k < DL; k++) acc[k] = make_float2(0.f, 0.f);
#pragma unroll 1
            for (uint32_t set = members | (a >= 0 ? 1u << a : 0u); set; set &= set - 1u) {
                const uint32_t w = __ffs(set) - 1u;
                const float fw = __shfl_sync(0xffffffffu, f, w);
                const float2 *src = reinterpret_cast<const float2 *>(((int)w == a ? tails : slots) + (size_t)(w * rb + row) * PS);
#pragma unroll
                for (int k = 0; k < DL; k++)
                    if (k * 32 + lane < HD / 2) {
                        const float2 v = src[k * 32 + lane];
                        acc[k].x = fmaf(fw, v.x, acc[k].x);
                        acc[k].y = fmaf(fw, v.y, acc[k].y);
                    }
            }
            if (out) {
                float *dst = A.part + (((size_t)blockIdx.x * 2u + (a < 0 ? 0u : 1u)) * rb + row) * PS;
#pragma unroll
                for (int k = 0; k < DL; k++)
                    if (k * 32 + lane < HD / 2) __stcg(reinterpret_cast<float2 *>(dst) + k * 32 + lane, acc[k]);
                if (lane == 0) __stcg(reinterpret_cast<float2 *>(dst + HD), make_float2(M, L));
            } else {
                const float inv = L == 0.f ? 0.f : 1.0f / L;
                float *dst = item_row(A, HD, it.seq_first, it.row0, it.head, row);
#pragma unroll
                for (int k = 0; k < DL; k++)
                    if (k * 32 + lane < HD / 2) {
                        dst[2 * (k * 32 + lane)] = acc[k].x * inv;
                        dst[2 * (k * 32 + lane) + 1] = acc[k].y * inv;
                    }
            }
        }
    }
    if (!cross[0] && !cross[1]) return;
    // ---- items that several blocks have: the last of them to come here joins their parts
    const PaCuts line(total, line_blocks);
    __threadfence();
    __syncthreads();
    if (warp < 2u && lane == 0) {
        last_here[warp] = 0u;
        if (const PaWorker::Part *it = cross[warp]) {
            const uint32_t lo = line.part_of(it->item0), hi = line.part_of(it->item0 + it->item_tiles - 1u);
            if (atomicAdd(&A.ticket[lo], 1u) == hi - lo) {
                A.ticket[lo] = 0u;
                last_here[warp] = 1u;
            }
        }
    }
    __syncthreads();
#pragma unroll 1
    for (int e = 0; e < 2; e++) {
        if (!last_here[e]) continue;
        __threadfence();
        const PaWorker::Part &it = *cross[e];
        const uint32_t lo = line.part_of(it.item0), n = line.part_of(it.item0 + it.item_tiles - 1u) - lo + 1u;
        const uint32_t R = min(rb, it.seq_rows * A.group - it.row0);
#pragma unroll 1
        for (uint32_t row = warp; row < R; row += NW) join_row<HD>(A, rb, lo, n, row, item_row(A, HD, it.seq_first, it.row0, it.head, row));
    }
}

// Above this many rows a head on average, blocks of 128 rows on tcgen05 (kv_attn_rows.cu). Both forms measured, 8 KV heads of 128,
// 64-token pages, us with such blocks and without, f16 and e4m3:
//   12 rows, 64 sequences of 4000 tokens: 283 and 259, 336 and 214
//   16 rows,  8 of 3000:  49 and  45,  54 and  42;  32 of 8000: 275 and  258, 331 and 212;  1 of 30000: 61 and 56, 65 and 51
//   20 rows,  8 of 3000:  52 and  71,  57 and  61;  32 of 8000: 280 and  532, 321 and 411;  1 of 30000: 66 and 92, 71 and 76
//   64 rows,  8 of 3000:  70 and 130,  67 and 107;  32 of 8000: 307 and 1050, 368 and 805
// One form serves a call, so a batch of very uneven sequences gets the wrong one for some of them: 512 rows beside 60 single tokens
// behind 4000 each take 1139 us, in two calls 189 (150 rows: 403 and 186).
constexpr uint64_t ROWS_FROM = 16;

// Blocks that the launch may have: one on each SM.
static uint32_t attn_blocks(const strix_cuda *h) { return (uint32_t)std::min<int>(std::max(h->num_sms, 1), (int)PA_MAX_BLOCKS); }

// Rows of a KV head that a sequence brings on average decide the form: up to 8, one product for values and remainders; beyond, on
// tcgen05 with blocks of 128 rows (head sizes 64 and 128), else 16 rows a warp and as many warps to a worker as cover them (at
// most all of a block).
enum : int { FORM_NARROW, FORM_WIDE, FORM_ROWS };
static int attn_form(const PagedView &V, uint32_t group, uint32_t &wm) {
    const uint64_t rows = ((uint64_t)V.n_rows * group + V.n_seq - 1) / std::max(V.n_seq, 1u);
    wm = 1;
    if (rows <= 8) return FORM_NARROW;
    if (rows > ROWS_FROM && (V.head_dim == 64 || V.head_dim == 128)) return FORM_ROWS;
    const uint32_t most = V.head_dim >= 192 ? 4u : 8u;
    while (wm < most && 16ull * wm < rows) wm *= 2;
    return FORM_WIDE;
}

static uint32_t form_rows(int form, uint32_t wm) { return form == FORM_ROWS ? 128u : form == FORM_WIDE ? 16u * wm : 8u; }  // of a block

// What a call of these sizes needs.
static size_t attn_work_bytes(const strix_cuda *h, const PagedView &V, uint32_t group) {
    uint32_t wm;
    const int form = attn_form(V, group, wm);
    const size_t part = (size_t)attn_blocks(h) * 2 * form_rows(form, wm) * (V.head_dim + 2) * 4;
    return (PA_MAX_BLOCKS * 4 + part + 255) & ~(size_t)255;
}

typedef CUresult (*AttnEncodeFn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *,
                                const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                                CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
static AttnEncodeFn attn_encode_fn() {
    static AttnEncodeFn fn = [] {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess)
            p = nullptr;
        return reinterpret_cast<AttnEncodeFn>(p);
    }();
    return fn;
}
bool attn_map(CUtensorMap *map, const PagedView &V, void *base, uint32_t box, uint32_t rows, bool swizzled) {
    AttnEncodeFn fn = attn_encode_fn();
    if (!fn) return false;
    const bool f16 = V.type == STRIX_KV_F16;
    const cuuint64_t dims[3] = {V.head_dim, (cuuint64_t)V.n_kv * V.page_tokens, V.n_pages};
    const cuuint64_t strides[2] = {(cuuint64_t)V.head_dim * (f16 ? 2 : 1), V.page_bytes};
    const cuuint32_t boxes[3] = {box, rows, 1}, one[3] = {1, 1, 1};
    return fn(map, f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, base, dims, strides, boxes, one,
              CU_TENSOR_MAP_INTERLEAVE_NONE, swizzled ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_NONE,
              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int HD, int TYPE, bool WIDE>
static cudaError_t attn_launch(const strix_cuda *h, PagedAttnArgs &A, cudaStream_t stream) {
    using S = PaShape<HD, TYPE, WIDE>;
    const int workers = S::NW / (int)A.wm;
    const int halves = S::halves_for((int)A.wm, h->smem_optin - PA_STATIC);
    const size_t smem = S::rings(workers, halves) + S::fixed(workers, halves) + 1024;
    if (halves < 2 || smem + PA_STATIC - 1024 > h->smem_optin) return cudaErrorInvalidConfiguration;
    const uint32_t sub = std::min<uint32_t>(S::TT, A.V.page_tokens);
    if (!attn_map(&A.k_map, A.V, A.V.k, S::BOXB / S::EL, sub, S::SWZ) || !attn_map(&A.v_map, A.V, A.V.v, S::BOXB / S::EL, sub, S::SWZ))
        return cudaErrorInvalidValue;
    static std::atomic<uint64_t> ready{0};  // devices whose limit of dynamic shared memory is raised for this kernel
    const uint64_t bit = 1ull << (h->device & 63);
    if (!(ready.load(std::memory_order_relaxed) & bit)) {
        cudaError_t e = cudaFuncSetAttribute(paged_attn_kernel<HD, TYPE, WIDE>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             (int)(h->smem_optin - 512));
        if (e != cudaSuccess) return e;
        ready.fetch_or(bit, std::memory_order_relaxed);
    }
    A.halves = (uint32_t)halves;
    paged_attn_kernel<HD, TYPE, WIDE><<<attn_blocks(h), S::NW * 32, smem, stream>>>(A);
    return cudaGetLastError();
}

}  // namespace strix

using namespace strix;

static int attn_check(strix_cuda *h, const char *who, const strix_kv_pages *cache, const strix_kv_batch *batch, uint32_t n_heads, PagedView &V) {
    const int rc = serve_check(h, who, cache, batch, &V);
    if (rc != 1) return rc;
    if (n_heads == 0 || n_heads > 65535u || n_heads % V.n_kv) return 0;
    if (V.n_seq > PA_MAX_SEQ) return serve_fail(h, who, "at most 8192 sequences in one call");
    // the line of tiles is counted in 31 bits
    const uint64_t group = n_heads / V.n_kv;
    uint32_t wm;
    const int form = attn_form(V, (uint32_t)group, wm);
    const uint64_t rb = form_rows(form, wm);
    const uint64_t blocks = ((uint64_t)V.n_rows * group + rb - 1) / rb + V.n_seq, tiles = (uint64_t)V.pages_ld * V.page_tokens / 16 + 1;
    if ((uint64_t)V.n_rows * group > 0x7fffffffull || blocks * V.n_kv > 0x7fffffffull || blocks * V.n_kv * tiles > 0x7fffffffull)
        return serve_fail(h, who, "batch too large for one call");
    return 1;
}

extern "C" size_t strix_cuda_attn_pages_workspace(strix_cuda *h, const strix_kv_pages *cache, const strix_kv_batch *batch,
                                                  uint32_t n_heads) {
    if (!h) return 0;
    h->err.clear();
    PagedView V;
    if (attn_check(h, "attn_pages_workspace", cache, batch, n_heads, V) != 1) return 0;
    V.n_seq = 1;  // all rows in one sequence: the form with the most rows to a block that so many rows can take
    return attn_work_bytes(h, V, n_heads / V.n_kv);
}

extern "C" int strix_cuda_attn_pages_dev(strix_cuda *h, const strix_kv_pages *cache, const strix_kv_batch *batch, uint32_t n_heads,
                                         const float *d_q, size_t ld_q, float scale, uint32_t window, float *d_out, size_t ld_out,
                                         void *d_work, size_t work_bytes, void *stream) {
    if (!h) return -1;
    h->err.clear();
    const char *who = "attn_pages";
    PagedAttnArgs A{};
    const int rc = attn_check(h, who, cache, batch, n_heads, A.V);
    if (rc != 1) return rc;
    const uint32_t hd = A.V.head_dim;
    const size_t qd = (size_t)n_heads * hd;
    A.ld_q = ld_q ? ld_q : qd;
    A.ld_out = ld_out ? ld_out : qd;
    if (A.ld_q < qd || A.ld_out < qd) return serve_fail(h, who, "a row stride is smaller than a row");
    if (!isfinite(scale)) return serve_fail(h, who, "scale must be finite");
    if (A.V.n_seq == 0 || A.V.n_rows == 0) return 1;
    if (!d_q || !d_out) return serve_fail(h, who, "d_q or d_out missing");
    if (d_q == d_out) return serve_fail(h, who, "d_out must not be d_q: rows are read by several blocks");
    if (!d_work || (reinterpret_cast<uintptr_t>(d_work) & 255u)) return serve_fail(h, who, "d_work must be 256-byte aligned");
    A.group = n_heads / A.V.n_kv;
    while ((1u << A.g_shift) < A.group) A.g_shift++;
    A.g_mul = (uint32_t)((((uint64_t)1 << 32) * (((uint64_t)1 << A.g_shift) - A.group)) / A.group + 1u);
    if (work_bytes < attn_work_bytes(h, A.V, A.group)) return serve_fail(h, who, "work_bytes too small");
    A.q = d_q;
    A.out = d_out;
    A.window = window;
    A.cap = A.V.pages_ld * A.V.page_tokens;
    A.scale = scale;
    A.scale_m = (float)frexp((double)scale * 1.4426950408889634, &A.scale_e);
    A.vec = ((reinterpret_cast<uintptr_t>(d_q) | reinterpret_cast<uintptr_t>(d_out)) & 15u) == 0 && ((A.ld_q | A.ld_out) & 3u) == 0;
    A.ticket = static_cast<uint32_t *>(d_work);
    A.part = reinterpret_cast<float *>(static_cast<uint8_t *>(d_work) + PA_MAX_BLOCKS * 4);
    const int form = attn_form(A.V, A.group, A.wm);
    const bool wide = form == FORM_WIDE;
    DeviceGuard dev(h->device);
    if (dev.err != cudaSuccess) return serve_fail(h, who, cudaGetErrorString(dev.err));
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    cudaError_t e = cudaErrorInvalidValue;
    {
        ProfScope prof(h, s, "attn_pages");
        const bool f16 = A.V.type == STRIX_KV_F16;
#define STRIX_ATTN(HD)                                                                                                            \
    case HD:                                                                                                                      \
        e = f16 ? (wide ? attn_launch<HD, STRIX_KV_F16, true>(h, A, s) : attn_launch<HD, STRIX_KV_F16, false>(h, A, s))             \
                : (wide ? attn_launch<HD, STRIX_KV_E4M3, true>(h, A, s) : attn_launch<HD, STRIX_KV_E4M3, false>(h, A, s));          \
        break;
        if (form == FORM_ROWS) e = launch_attn_rows(h, A, attn_blocks(h), s);
        else switch (hd) {
            STRIX_ATTN(64)
            STRIX_ATTN(96)
            STRIX_ATTN(128)
            STRIX_ATTN(192)
            STRIX_ATTN(256)
        }
#undef STRIX_ATTN
    }
    if (e != cudaSuccess) return serve_fail(h, who, cudaGetErrorString(e));
    return 1;
}
