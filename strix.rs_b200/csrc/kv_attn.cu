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
// largest value in [2^14, 2^15)), probabilities by 2^15: what is lost lies below 2^-33 of the row's largest. The sums over a tile
// start from zero and are added to the f32 running sums outside the tensor cores, which round to nearest: chained
// accumulation in the tensor cores truncates, a drift of its own over thousands of tokens.
// The order of the head's dimensions inside a product is free as long as q and k agree, and so is the order of the
// output columns: each thread takes the dimensions that lie next to each other in a cached row, so that shared memory is read in
// 16-byte words.
//
// Work split. A tile is TT tokens of one KV head (about 8 KB of k and v). All tiles of all (sequence, row block, KV head)
// items stand in one line; block c of the grid takes an equal stretch of it, and each of the block's workers an equal part
// of that. A worker is a warp (or several, over the row blocks of a prompt) with a ring of stages of its own, filled by bulk
// copies that the block's producer warp issues, one lane for each worker. An item that one worker has whole is written
// out by it; the parts of the others meet in shared memory at the block's end, and where an item goes on in another block, in the
// workspace: the last block to arrive joins the parts, in the order of the line. Cuts that would fall into an item of at most
// PA_SNAP tiles move to its nearer end.
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "kv_pages.cuh"

namespace strix {

constexpr uint32_t PA_MAX_BLOCKS = 1024;  // tickets at the start of the workspace
constexpr uint32_t PA_SNAP = 16;
constexpr size_t PA_STATIC = 1024;  // static shared memory and what the system keeps

struct PagedAttnArgs {
    PagedView V;
    const float *q;
    float *out;
    size_t ld_q, ld_out;
    uint32_t n_heads, group, window, cap;  // cap: tokens a row of the page table can hold
    float scale;
    uint32_t wm, stages, vec;  // warps of a worker; stages of a ring; q and out rows start on 16 bytes
    uint32_t *ticket;          // [PA_MAX_BLOCKS]
    float *part;               // [blocks][2][rows of a worker][HD + 2]
};

// Sizes that follow from the head size, the cache type and the row form (WIDE: 16 rows a warp, else 8).
template <int HD, int TYPE, bool WIDE>
struct PaShape {
    static constexpr int EL = TYPE == STRIX_KV_F16 ? 2 : 1;
    static constexpr int NW = HD >= 192 && (WIDE || EL == 2) ? 4 : 8;  // consumer warps
    static constexpr int ROWS = WIDE ? 16 : 8;                         // rows of a warp
    static constexpr int TT = HD * EL <= 64 ? 64 : HD * EL <= 128 ? 32 : 16;
    static constexpr int KBYTES = TT * HD * EL, STAGE = 2 * KBYTES;
    static constexpr int PSTRIDE = HD + 2;                             // floats of a partial row: sums, maximum, sum of weights
    static constexpr bool QSMEM = WIDE && HD >= 192;                   // q fragments in shared memory instead of registers
    static constexpr int QBYTES = QSMEM ? NW * 16 * HD * 4 : 0;
    static constexpr int SLOTS = NW * ROWS * PSTRIDE * 4;              // one partial for each worker
    static constexpr int DESC = 64, WORKER = 64;
    static constexpr int fixed(int workers, int stages) { return SLOTS + QBYTES + workers * (WORKER + stages * (DESC + 16)); }
    static int stages_for(int wm, size_t smem) {
        const int workers = NW / wm;
        int s = 16;
        while (s > 1 && (size_t)fixed(workers, s) + (size_t)workers * s * STAGE > smem) s--;
        return s;
    }
};

// What the producer tells a worker about a stage.
struct __align__(16) PaTile {
    uint32_t seq_first, seq_rows, ctx, tile;  // first row of the sequence, its new rows, tokens before them; tile of the item
    uint32_t row0, head, flags, valid;        // first row of the block (in rows of the KV head), KV head; one bit for each page of the tile
    float ks[4], vs[4];                       // the scales of the tile's pages
};
enum : uint32_t { PA_NEW = 1, PA_END = 2, PA_WHOLE = 4, PA_HEAD = 8 };  // first / last tile of the segment here; item complete here; begun elsewhere

// What the joins need to know about a worker's open parts.
struct __align__(16) PaWorker {
    struct Part {
        uint32_t seq_first, seq_rows, row0, head, item0, item_tiles;
    };
    Part head, tail;
    uint32_t has_head, head_ended, has_tail, pad;
};

__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// x0, x1 as f16 (packed) and what that rounding left of them
__device__ __forceinline__ void split2(float x0, float x1, uint32_t &hi, uint32_t &lo) {
    hi = f32_to_f16x2(x0, x1);
    const float2 h = __half22float2(*reinterpret_cast<const __half2 *>(&hi));
    lo = f32_to_f16x2(x0 - h.x, x1 - h.y);
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

// Tiles of row block mb of a sequence: [lo_tile, lo_tile + n).
template <int TT>
__device__ __forceinline__ uint32_t block_tiles(const PagedAttnArgs &A, uint32_t rb, uint32_t rows, uint32_t ctx, uint32_t mb,
                                                uint32_t &lo_tile) {
    const uint32_t R = rows * A.group, r0 = mb * rb, r1 = min(R, r0 + rb) - 1u;
    const uint32_t p0 = ctx + r0 / A.group, p1 = ctx + r1 / A.group;  // positions of the first and last row (below 2^32)
    const uint32_t hi = min(A.cap, p1 + 1u);
    const uint32_t lo = A.window && p0 >= A.window ? p0 + 1u - A.window : 0u;
    lo_tile = lo / TT;
    return hi > lo ? (hi + TT - 1u) / TT - lo_tile : 0u;
}
// All tiles of a sequence; rows and ctx are 0 and < 0 where there is nothing to do.
template <int TT>
__device__ __forceinline__ uint32_t seq_tiles(const PagedAttnArgs &A, uint32_t rb, uint32_t s, uint32_t &first, uint32_t &rows, int &ctx) {
    uint32_t end;
    bool bad = false;
    seq_rows(A.V, s, first, end, bad);
    rows = end - first;
    ctx = A.V.ctx[s];
    if (ctx < 0 || rows == 0u) return 0u;
    uint32_t n = 0, lo;
    const uint32_t blocks = (rows * A.group + rb - 1u) / rb;
    for (uint32_t mb = 0; mb < blocks; mb++) n += block_tiles<TT>(A, rb, rows, (uint32_t)ctx, mb, lo);
    return n * A.V.n_kv;
}

// A place in the line of tiles.
struct PaPlace {
    uint32_t s, first, rows, ctx, mb, head, lo_tile, tiles, at;  // item: tiles of it, `at` the place within
    uint32_t item0;                                              // the line's index of the item's first tile
};

// A lane's place from the sequence that holds line index x (whose own tiles start at base).
template <int TT>
__device__ __forceinline__ void place_in_seq(const PagedAttnArgs &A, uint32_t rb, uint32_t s, uint32_t base, uint32_t x, PaPlace &P) {
    uint32_t first, rows;
    int ctx;
    (void)seq_tiles<TT>(A, rb, s, first, rows, ctx);
    P.s = s;
    P.first = first;
    P.rows = rows;
    P.ctx = (uint32_t)ctx;
    uint32_t off = x - base, mb = 0, lo, n;
    const uint32_t blocks = (rows * A.group + rb - 1u) / rb;
    for (;; mb++) {
        n = block_tiles<TT>(A, rb, rows, P.ctx, mb, lo);
        if (off < n * A.V.n_kv || mb + 1u >= blocks) break;
        off -= n * A.V.n_kv;
    }
    P.mb = mb;
    P.lo_tile = lo;
    P.tiles = n;
    P.head = n ? off / n : 0u;
    P.at = n ? off - P.head * n : 0u;
    P.item0 = x - P.at;
}
// The next item with tiles; the caller knows that there is one.
template <int TT>
__device__ __forceinline__ void next_item(const PagedAttnArgs &A, uint32_t rb, PaPlace &P) {
    P.item0 += P.tiles;
    P.at = 0;
    if (++P.head < A.V.n_kv) return;
    P.head = 0;
    for (;;) {
        const uint32_t blocks = (P.rows * A.group + rb - 1u) / rb;
        if ((int)P.ctx >= 0 && ++P.mb < blocks) {
            P.tiles = block_tiles<TT>(A, rb, P.rows, P.ctx, P.mb, P.lo_tile);
            if (P.tiles) return;
            continue;
        }
        if (++P.s >= A.V.n_seq) {
            P.tiles = 0;
            return;
        }
        uint32_t end;
        bool bad = false;
        seq_rows(A.V, P.s, P.first, end, bad);
        P.rows = end - P.first;
        P.ctx = (uint32_t)A.V.ctx[P.s];
        P.mb = 0xffffffffu;
        if (P.rows == 0u) P.ctx = 0xffffffffu;
    }
}

// Finds the places of up to 8 line indices (x[i] < total, ascending not needed) by one pass over the sequences; lane i gets place i.
template <int TT>
__device__ __forceinline__ void find_places(const PagedAttnArgs &A, uint32_t rb, uint32_t x, uint32_t count, PaPlace &P) {
    const uint32_t lane = threadIdx.x & 31u;
    uint32_t base = 0, mine_s = 0, mine_base = 0;
    uint32_t left = count == 32u ? 0xffffffffu : (1u << count) - 1u;
    for (uint32_t c = 0; c < A.V.n_seq && left; c += 32u) {
        uint32_t first, rows;
        int ctx;
        const uint32_t n = c + lane < A.V.n_seq ? seq_tiles<TT>(A, rb, c + lane, first, rows, ctx) : 0u;
        uint32_t incl = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t v = __shfl_up_sync(0xffffffffu, incl, o);
            if ((int)lane >= o) incl += v;
        }
        for (uint32_t i = 0; i < count; i++) {
            if (!((left >> i) & 1u)) continue;
            const uint32_t xi = __shfl_sync(0xffffffffu, x, i) - base;
            const uint32_t m = __ballot_sync(0xffffffffu, incl > xi);
            if (m == 0u) continue;
            const uint32_t j = __ffs(m) - 1u, before = __shfl_sync(0xffffffffu, incl - n, j);
            if (lane == i) {
                mine_s = c + j;
                mine_base = base + before;
            }
            left &= ~(1u << i);
        }
        base += __shfl_sync(0xffffffffu, incl, 31);
    }
    if (lane < count) place_in_seq<TT>(A, rb, mine_s, mine_base, x, P);
}

// Where cut x of the line falls: cuts inside a short item move to its nearer end.
__device__ __forceinline__ uint32_t snapped(const PaPlace &P, uint32_t x) {
    if (P.at == 0u || P.tiles > PA_SNAP) return x;
    return 2u * P.at < P.tiles ? P.item0 : P.item0 + P.tiles;
}

template <int HD, int TYPE, bool WIDE>
__global__ void __launch_bounds__((PaShape<HD, TYPE, WIDE>::NW + 1) * 32, 1) paged_attn_kernel(const __grid_constant__ PagedAttnArgs A) {
    using S = PaShape<HD, TYPE, WIDE>;
    constexpr int EL = S::EL, NW = S::NW, TT = S::TT, NT = TT / 8, KS = HD / 16;
    constexpr int PS = S::PSTRIDE, NO = HD / 8;          // NO: output tiles of eight columns
    constexpr int KW = (HD / 4 * EL) % 16 == 0 ? 16 : 8;  // bytes of a thread's k loads
    constexpr int KL = HD / 4 * EL / KW;                  // ... and how many a token
    constexpr int VB = HD / 8 * EL;                       // bytes of a cached value row that a thread turns into output columns
    constexpr int VW = VB % 16 == 0 ? 16 : VB % 8 == 0 ? 8 : 4, VL = VB / VW;
    constexpr int RW = WIDE ? 2 : 1;                      // rows of a thread
    extern __shared__ __align__(128) uint8_t smem[];
    const PagedView &V = A.V;
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
    const uint32_t wm = WIDE ? A.wm : 1u, workers = NW / wm, rb = S::ROWS * wm, stages = A.stages;
    uint8_t *rings = smem;
    float *slots = reinterpret_cast<float *>(smem + (size_t)workers * stages * S::STAGE);
    uint8_t *qsm = reinterpret_cast<uint8_t *>(slots) + S::SLOTS;
    PaTile *desc = reinterpret_cast<PaTile *>(qsm + S::QBYTES);
    PaWorker *info = reinterpret_cast<PaWorker *>(desc + workers * stages);
    uint64_t *full = reinterpret_cast<uint64_t *>(info + workers), *empty = full + workers * stages;
    __shared__ uint32_t range[2], last_here;

    if (threadIdx.x < workers * stages) {
        mbar_init(&full[threadIdx.x], 1);
        mbar_init(&empty[threadIdx.x], wm);
        mbar_fence_init();
    }
    if (threadIdx.x < workers) {
        info[threadIdx.x].has_head = info[threadIdx.x].head_ended = info[threadIdx.x].has_tail = 0u;
    }

    // ---- this block's stretch of the line, by the producer warp
    uint32_t total = 0, blocks = 0;
    PaPlace place{};
    uint32_t w_begin = 0, w_end = 0;  // producer lanes: the worker's stretch
    if (warp == NW) {
        for (uint32_t c = lane; c < V.n_seq; c += 32u) {
            uint32_t first, rows;
            int ctx;
            total += seq_tiles<TT>(A, rb, c, first, rows, ctx);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
        blocks = min(gridDim.x, (total + workers - 1u) / workers);  // blocks with work
        uint32_t lo = 0, hi = 0;
        if (blockIdx.x < blocks) {
            uint32_t x = (uint32_t)((uint64_t)(blockIdx.x + (lane == 1u)) * total / blocks);
            const bool at_end = x >= total;
            PaPlace P{};
            find_places<TT>(A, rb, at_end ? total - 1u : x, 2u, P);
            if (!at_end) x = snapped(P, x);
            lo = __shfl_sync(0xffffffffu, x, 0);
            hi = __shfl_sync(0xffffffffu, x, 1);
        }
        if (lane == 0) {
            range[0] = lo;
            range[1] = hi;
        }
        if (hi > lo) {
            const uint32_t n = hi - lo;
            w_begin = lo + (uint32_t)((uint64_t)min(lane, workers) * n / workers);
            w_end = lo + (uint32_t)((uint64_t)min(lane + 1u, workers) * n / workers);
            if (lane >= workers) w_begin = w_end = 0;
            find_places<TT>(A, rb, min(w_begin, total - 1u), workers, place);
        }
    }
    __syncthreads();

    const uint32_t n_block = range[1] - range[0];
    const uint32_t worker = warp == NW ? 0u : warp / wm;
    // consumer state that outlives the loop (a part that goes on in the next worker)
    float o[NO][2 * RW], m[RW], l[RW];
    bool open_tail = false;

    if (warp == NW) {
        // ---- producer: lane w fills the ring of worker w
        uint32_t left = w_end - w_begin, stage = 0, phase = 1;  // (the first pass over a ring finds it empty)
        uint32_t idle = 0;
        bool fresh = true, bad = false;
        PaWorker *me = info + min(lane, workers - 1u);
        const uint32_t sub = TT > 16 ? min((uint32_t)TT, V.page_tokens) : 16u;  // tokens of one copy
        while (__any_sync(0xffffffffu, left > 0u)) {
            if (left > 0u && mbar_test_wait(&empty[lane * stages + stage], phase)) {
                idle = 0;
                const uint32_t tile = place.lo_tile + place.at, tok = tile * TT;
                PaTile d;
                d.seq_first = place.first;
                d.seq_rows = place.rows;
                d.ctx = place.ctx;
                d.tile = tile;
                d.row0 = place.mb * rb;
                d.head = place.head;
                d.flags = fresh ? PA_NEW : 0u;
                const bool item_end = place.at + 1u == place.tiles, seg_end = item_end || left == 1u;
                if (fresh) {  // how the segment relates to its item
                    const uint32_t seg = min(left, place.tiles - place.at);
                    PaWorker::Part part{place.first, place.rows, d.row0, place.head, place.item0, place.tiles};
                    if (place.at > 0u) {
                        me->head = part;
                        me->has_head = 1u;
                        me->head_ended = place.at + seg == place.tiles;
                    } else if (seg < place.tiles) {
                        me->tail = part;
                        me->has_tail = 1u;
                    }
                }
                if (seg_end) {
                    d.flags |= PA_END;
                    if (me->has_head && me->head.item0 == place.item0) d.flags |= PA_HEAD;
                    else if (item_end) d.flags |= PA_WHOLE;
                }
                d.valid = 0u;
                uint32_t bytes = 0;
                int page[4];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    page[i] = -1;
                    if (i * sub < TT) {
                        const uint32_t nth = (tok + i * sub) >> V.page_shift;
                        page[i] = nth < V.pages_ld ? V.pages[(size_t)place.s * V.pages_ld + nth] : -2;  // (-2: past the table's end)
                    }
                }
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    d.ks[i] = d.vs[i] = 0.f;
                    if (i * sub >= TT || tok + i * sub > place.ctx + (place.rows - 1u)) continue;  // behind the sequence: no page to look at
                    if (page[i] < 0 || (uint32_t)page[i] >= V.n_pages) {
                        bad |= page[i] != -2;
                        continue;
                    }
                    d.valid |= 1u << i;
                    bytes += 2u * sub * HD * EL;
                    if (TYPE == STRIX_KV_E4M3) {
                        const size_t at = (size_t)page[i] * V.n_kv + place.head;
                        d.ks[i] = V.k_scale[at];
                        d.vs[i] = V.v_scale[at];
                    } else {
                        d.ks[i] = d.vs[i] = 1.f;
                    }
                }
                desc[lane * stages + stage] = d;
                uint64_t *bar = &full[lane * stages + stage];
                uint8_t *dst = rings + (size_t)(lane * stages + stage) * S::STAGE;
                mbar_arrive_expect_tx(bar, bytes);
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    if (!((d.valid >> i) & 1u)) continue;
                    const size_t src = (size_t)page[i] * V.page_bytes + (size_t)place.head * V.head_bytes +
                                       (size_t)((tok + i * sub) & (V.page_tokens - 1u)) * HD * EL;
                    bulk_g2s(dst + i * sub * HD * EL, V.k + src, sub * HD * EL, bar);
                    bulk_g2s(dst + S::KBYTES + i * sub * HD * EL, V.v + src, sub * HD * EL, bar);
                }
                if (++stage == stages) {
                    stage = 0;
                    phase ^= 1u;
                }
                left--;
                place.at++;
                fresh = seg_end;
                if (item_end && left > 0u) next_item<TT>(A, rb, place);
            } else if (left > 0u && ++idle > (1u << 24)) {  // a worker that takes nothing for seconds: report and stop feeding it
                atomicOr(V.status, STATUS_WAIT_TIMEOUT);
                left = 0;
            }
        }
        report_bad(V, bad);
    } else {
        // ---- rows that see nothing, and lengths beyond the table: each sequence is looked at by one warp of the grid
        for (uint32_t s = blockIdx.x * NW + warp; s < V.n_seq; s += gridDim.x * NW) {
            uint32_t first, end;
            bool bad = false;
            seq_rows(V, s, first, end, bad);
            const int ctx = V.ctx[s];
            const uint32_t rows = end - first;
            if (ctx >= 0 && (uint64_t)(uint32_t)ctx + rows > A.cap && rows) bad = true;
            if (ctx < 0 || (uint64_t)(uint32_t)ctx + rows > A.cap) {
                const uint32_t R = rows * A.group, nb = (R + rb - 1u) / rb;
                for (uint32_t mb = 0; mb < nb; mb++) {
                    uint32_t lo;
                    if (ctx >= 0 && block_tiles<TT>(A, rb, rows, (uint32_t)ctx, mb, lo)) continue;
                    for (uint32_t r = mb * rb; r < min(R, (mb + 1u) * rb); r++)
                        for (uint32_t h = 0; h < V.n_kv; h++) {
                            float *dst = A.out + (size_t)(first + r / A.group) * A.ld_out + (size_t)(h * A.group + r % A.group) * HD;
                            for (uint32_t i = lane; i < HD; i += 32u) dst[i] = 0.f;
                        }
                }
            }
            report_bad(V, bad && lane == 0);
        }

        // ---- consumer
        const uint32_t g = lane >> 2, t = lane & 3u, wi = warp - worker * wm;  // row and column of the fragments; warp of the worker
        const uint32_t n_mine = (uint32_t)((uint64_t)(worker + 1u) * n_block / workers) - (uint32_t)((uint64_t)worker * n_block / workers);
        uint32_t stage = 0, phase = 0;
        uint32_t qf[S::QSMEM ? 1 : KS][WIDE ? 8 : 4];  // fragments of q: values (and remainders, in the same rows or apart)
        uint4 *qs = reinterpret_cast<uint4 *>(qsm) + warp * (KS * 2 * 32) + lane;
        float qc[RW];                                  // factor from the products to exponents of two
        uint32_t pos[RW], pos_lo = 0, pos_hi = 0;      // positions of this thread's rows, of the warp's first and last row
        for (uint32_t n = 0; n < n_mine; n++) {
            if (!mbar_wait_bounded(&full[worker * stages + stage], phase, V.status)) break;  // (the producer gives up as well)
            const PaTile &d = desc[worker * stages + stage];
            const uint8_t *ks = rings + (size_t)(worker * stages + stage) * S::STAGE, *vs = ks + S::KBYTES;
            const uint32_t flags = d.flags;
            if (flags & PA_NEW) {
                const uint32_t R = d.seq_rows * A.group, rw = d.row0 + wi * S::ROWS;
                const float *qrow[RW];
                bool on[RW];
#pragma unroll
                for (int i = 0; i < RW; i++) {
                    const uint32_t r = rw + g + 8u * i;
                    on[i] = r < R;
                    const uint32_t rr = min(r, R - 1u), tk = rr / A.group;
                    pos[i] = d.ctx + tk;
                    qrow[i] = A.q + (size_t)(d.seq_first + tk) * A.ld_q + (size_t)(d.head * A.group + rr - tk * A.group) * HD;
                }
                pos_lo = d.ctx + min(rw, R - 1u) / A.group;
                pos_hi = d.ctx + min(rw + S::ROWS - 1u, R - 1u) / A.group;
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
                    qc[i] = A.scale * 1.4426950408889634f * __uint_as_float((uint32_t)(127 - e2) << 23);
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
            const uint32_t tok = d.tile * TT, valid = d.valid;
            float sc[NT][4];
#pragma unroll
            for (int j = 0; j < NT; j++) {
                const uint8_t *kr = ks + (8 * j + g) * (HD * EL) + t * KW;
                uint32_t w[KL * KW / 4];
#pragma unroll
                for (int i = 0; i < KL; i++) lds_words<KW>(w + i * (KW / 4), kr + i * 4 * KW);
#pragma unroll
                for (int e = 0; e < 4; e++) sc[j][e] = 0.f;
#pragma unroll
                for (int s = 0; s < KS; s++) {
                    uint32_t b0, b1;
                    if constexpr (EL == 1) {
                        b0 = e4m3x2_to_f16x2(w[s] & 0xffffu);
                        b1 = e4m3x2_to_f16x2(w[s] >> 16);
                    } else {
                        b0 = w[2 * s];
                        b1 = w[2 * s + 1];
                    }
                    if constexpr (!WIDE) {
                        mma_f16(sc[j], reinterpret_cast<const uint32_t(&)[4]>(qf[s]), b0, b1);
                    } else if constexpr (!S::QSMEM) {
                        const uint32_t hi[4] = {qf[s][0], qf[s][1], qf[s][2], qf[s][3]}, lo[4] = {qf[s][4], qf[s][5], qf[s][6], qf[s][7]};
                        mma_f16(sc[j], lo, b0, b1);
                        mma_f16(sc[j], hi, b0, b1);
                    } else {
                        const uint4 h4 = qs[(2 * s) * 32], l4 = qs[(2 * s + 1) * 32];
                        const uint32_t hi[4] = {h4.x, h4.y, h4.z, h4.w}, lo[4] = {l4.x, l4.y, l4.z, l4.w};
                        mma_f16(sc[j], lo, b0, b1);
                        mma_f16(sc[j], hi, b0, b1);
                    }
                }
            }
            // to exponents of two; scale of the page; masks
            const uint32_t pshift = V.page_shift;
            const bool all = valid == (TT > 16 && V.page_tokens < TT ? (1u << (TT >> pshift)) - 1u : 1u);
            const bool tail_tok = tok + TT - 1u > pos_hi || !all;  // tokens that no row of the warp sees, maybe never written
            const bool masked = tail_tok || tok + TT - 1u > pos_lo || (A.window && pos_hi >= A.window && tok <= pos_hi - A.window);
            float mx[RW];
#pragma unroll
            for (int i = 0; i < RW; i++) mx[i] = m[i];
#pragma unroll
            for (int j = 0; j < NT; j++) {
                const uint32_t pg = TT > 16 ? (8u * j) >> pshift : 0u;  // (0 where a page is as long as the tile)
                const float kscale = d.ks[pg];
                if constexpr (!WIDE) {
                    sc[j][0] = (sc[j][0] + sc[j][2]) * (kscale * qc[0]);
                    sc[j][1] = (sc[j][1] + sc[j][3]) * (kscale * qc[0]);
                } else {
                    sc[j][0] *= kscale * qc[0];
                    sc[j][1] *= kscale * qc[0];
                    sc[j][2] *= kscale * qc[RW - 1];
                    sc[j][3] *= kscale * qc[RW - 1];
                }
                if (masked) {
#pragma unroll
                    for (int e = 0; e < 2 * RW; e++) {
                        const uint32_t tk = tok + 8u * j + 2u * t + (e & 1), p = pos[e >> 1];
                        const bool see = tk <= p && (!A.window || p < A.window || tk > p - A.window) && ((valid >> pg) & 1u);
                        if (!see) sc[j][e] = -INFINITY;
                    }
                }
#pragma unroll
                for (int e = 0; e < 2 * RW; e++) mx[e >> 1] = fmaxf(mx[e >> 1], sc[j][e]);
            }
            bool moved = false;
#pragma unroll
            for (int i = 0; i < RW; i++) {
                mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 1));
                mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 2));
                moved |= mx[i] != m[i];
            }
            if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
                for (int i = 0; i < RW; i++) {
                    const float a = mx[i] == m[i] ? 1.f : ex2(m[i] - mx[i]);
                    m[i] = mx[i];
                    l[i] *= a;
#pragma unroll
                    for (int k = 0; k < NO; k++) {
                        o[k][2 * i] *= a;
                        o[k][2 * i + 1] *= a;
                    }
                }
            }
            float base[RW];
#pragma unroll
            for (int i = 0; i < RW; i++) base[i] = m[i] == -INFINITY ? 0.f : m[i] - 15.f;  // weights carry 2^15, as their sum does
            // the largest scale among the tile's value pages; the weights take what another page's scale differs by
            float vref = d.vs[0];
            const bool mixed = TT > 16 && V.page_tokens < TT;
            if (mixed) vref = fmaxf(fmaxf(d.vs[0], d.vs[1]), fmaxf(d.vs[2], d.vs[3]));
            const float rvref = mixed && vref > 0.f ? 1.0f / vref : 1.f;
            uint32_t pf[TT / 16][WIDE ? 8 : 4];
#pragma unroll
            for (int j = 0; j < NT; j++) {
                float p[2 * RW];
#pragma unroll
                for (int e = 0; e < 2 * RW; e++) {
                    p[e] = ex2(sc[j][e] - base[e >> 1]);
                    l[e >> 1] += p[e];
                }
                if (mixed) {
                    const float f = d.vs[(8u * j) >> pshift] * rvref;
#pragma unroll
                    for (int e = 0; e < 2 * RW; e++) p[e] *= f;
                }
                const int u = j / 2, hf = (j & 1) * 2;
                if constexpr (!WIDE) {
                    split2(p[0], p[1], pf[u][hf], pf[u][hf + 1]);
                } else {
                    split2(p[0], p[1], pf[u][hf], pf[u][4 + hf]);
                    split2(p[2], p[2 * RW - 1], pf[u][hf + 1], pf[u][4 + hf + 1]);
                }
            }
            // weighted values: thread (g, t) reads the dimensions g VB.. of the four tokens its weights are for
#pragma unroll
            for (int c = 0; c < VL; c++) {
                uint32_t r[TT / 16][4][VW / 4];
#pragma unroll
                for (int u = 0; u < TT / 16; u++)
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        const uint32_t row = 16u * u + 2u * t + (k & 1) + 8u * (k >> 1);
                        lds_words<VW>(r[u][k], vs + row * (HD * EL) + g * VB + c * VW);
                        if (tail_tok && !(tok + row <= pos_hi && ((valid >> (TT > 16 ? row >> pshift : 0u)) & 1u))) {
#pragma unroll
                            for (int w = 0; w < VW / 4; w++) r[u][k][w] = 0u;
                        }
                    }
#pragma unroll
                for (int w = 0; w < VW / 4; w++) {
                    constexpr int PER = 4 / EL;  // dimensions of a word
                    float acc[PER][4];
#pragma unroll
                    for (int e = 0; e < PER; e++)
#pragma unroll
                        for (int k = 0; k < 4; k++) acc[e][k] = 0.f;
#pragma unroll
                    for (int u = 0; u < TT / 16; u++) {
                        uint32_t b0[PER], b1[PER];
                        if constexpr (EL == 1) {
                            const uint32_t a = __byte_perm(r[u][0][w], r[u][1][w], 0x5140), b = __byte_perm(r[u][0][w], r[u][1][w], 0x7362);
                            const uint32_t cc = __byte_perm(r[u][2][w], r[u][3][w], 0x5140), dd = __byte_perm(r[u][2][w], r[u][3][w], 0x7362);
                            b0[0] = e4m3x2_to_f16x2(a & 0xffffu);
                            b0[1] = e4m3x2_to_f16x2(a >> 16);
                            b0[2 % PER] = e4m3x2_to_f16x2(b & 0xffffu);
                            b0[3 % PER] = e4m3x2_to_f16x2(b >> 16);
                            b1[0] = e4m3x2_to_f16x2(cc & 0xffffu);
                            b1[1] = e4m3x2_to_f16x2(cc >> 16);
                            b1[2 % PER] = e4m3x2_to_f16x2(dd & 0xffffu);
                            b1[3 % PER] = e4m3x2_to_f16x2(dd >> 16);
                        } else {
                            b0[0] = __byte_perm(r[u][0][w], r[u][1][w], 0x5410);
                            b0[1] = __byte_perm(r[u][0][w], r[u][1][w], 0x7632);
                            b1[0] = __byte_perm(r[u][2][w], r[u][3][w], 0x5410);
                            b1[1] = __byte_perm(r[u][2][w], r[u][3][w], 0x7632);
                        }
#pragma unroll
                        for (int e = 0; e < PER; e++) {
                            if constexpr (!WIDE) {
                                mma_f16(acc[e], reinterpret_cast<const uint32_t(&)[4]>(pf[u]), b0[e], b1[e]);
                            } else {
                                const uint32_t hi[4] = {pf[u][0], pf[u][1], pf[u][2], pf[u][3]}, lo[4] = {pf[u][4], pf[u][5], pf[u][6], pf[u][7]};
                                mma_f16(acc[e], lo, b0[e], b1[e]);
                                mma_f16(acc[e], hi, b0[e], b1[e]);
                            }
                        }
                    }
#pragma unroll
                    for (int e = 0; e < PER; e++) {
                        float(&oo)[2 * RW] = o[(c * (VW / 4) + w) * PER + e];
                        if constexpr (!WIDE) {
                            oo[0] = fmaf(acc[e][0] + acc[e][2], vref, oo[0]);
                            oo[1] = fmaf(acc[e][1] + acc[e][3], vref, oo[1]);
                        } else {
#pragma unroll
                            for (int k = 0; k < 2 * RW; k++) oo[k] = fmaf(acc[e][k], vref, oo[k]);
                        }
                    }
                }
            }
            const uint32_t sf = d.seq_first, sr = d.seq_rows, r0 = d.row0, hd_ = d.head;
            __syncwarp();
            if (lane == 0) mbar_arrive(&empty[worker * stages + stage]);
            if (++stage == stages) {
                stage = 0;
                phase ^= 1u;
            }
            if (!(flags & PA_END)) continue;
            // the segment's end: the row sums of four threads meet
#pragma unroll
            for (int i = 0; i < RW; i++) {
                l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
                l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
            }
            if (flags & PA_WHOLE) {
#pragma unroll
                for (int i = 0; i < RW; i++) {
                    const uint32_t r = r0 + wi * S::ROWS + g + 8u * i, tk = r / A.group;
                    if (r >= sr * A.group) continue;
                    const float inv = l[i] == 0.f ? 0.f : 1.0f / l[i];
                    float *dst = A.out + (size_t)(sf + tk) * A.ld_out + (size_t)(hd_ * A.group + r - tk * A.group) * HD;
#pragma unroll
                    for (int e = 0; e < 2; e++) {  // columns 2 t and 2 t + 1 of the products: dimensions (2 t + e) NO..
                        float *q = dst + (2u * t + e) * NO;
                        if (A.vec) {
#pragma unroll
                            for (int k = 0; k < NO; k += 4)
                                *reinterpret_cast<float4 *>(q + k) = make_float4(o[k][2 * i + e] * inv, o[k + 1][2 * i + e] * inv,
                                                                                 o[k + 2][2 * i + e] * inv, o[k + 3][2 * i + e] * inv);
                        } else {
#pragma unroll
                            for (int k = 0; k < NO; k++) q[k] = o[k][2 * i + e] * inv;
                        }
                    }
                }
            } else if (flags & PA_HEAD) {
#pragma unroll
                for (int i = 0; i < RW; i++) {
                    float *dst = slots + (size_t)(warp * S::ROWS + g + 8u * i) * PS;
#pragma unroll
                    for (int k = 0; k < NO; k++) {
                        dst[2u * t * NO + k] = o[k][2 * i];
                        dst[(2u * t + 1u) * NO + k] = o[k][2 * i + 1];
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

    // ---- parts of items that more than one worker has: tails go where the rings were
    __syncthreads();
    float *tails = reinterpret_cast<float *>(rings);
    if (open_tail) {
        const uint32_t g = lane >> 2, t = lane & 3u;
#pragma unroll
        for (int i = 0; i < RW; i++) {
            float *dst = tails + (size_t)(warp * S::ROWS + g + 8u * i) * PS;
#pragma unroll
            for (int k = 0; k < NO; k++) {
                dst[2u * t * NO + k] = o[k][2 * i];
                dst[(2u * t + 1u) * NO + k] = o[k][2 * i + 1];
            }
            if (t == 0) {
                dst[HD] = m[i];
                dst[HD + 1] = l[i];
            }
        }
    }
    __syncthreads();
    if (n_block == 0u) return;
    if (warp == NW && lane == 0) range[0] = total, range[1] = blocks;
    __syncthreads();
    const uint32_t line = range[0], line_blocks = range[1];
    constexpr uint32_t THREADS = (NW + 1) * 32;

    // one chain of parts: [tail of worker a,] heads of the workers behind it; `front` / `back`: it goes on in other blocks
    auto emit = [&](int a_tail, uint32_t h0, uint32_t h1, const PaWorker::Part &it, bool front, bool back) {
        const uint32_t R = it.seq_rows * A.group;
        // weight of each part, row by row: 2^(its maximum - the largest)
        float *slot = A.part + ((size_t)blockIdx.x * 2u + (front ? 0u : 1u)) * rb * PS;
        for (uint32_t i = threadIdx.x; i < rb * PS; i += THREADS) {
            const uint32_t row = i / PS, col = i - row * PS;
            if (it.row0 + row >= R) continue;
            const float *tp = a_tail >= 0 ? tails + ((size_t)a_tail * rb + row) * PS : nullptr;
            float M = tp ? tp[HD] : -INFINITY;
            for (uint32_t w = h0; w < h1; w++) M = info[w].has_head ? fmaxf(M, slots[((size_t)w * rb + row) * PS + HD]) : M;
            const float b = M == -INFINITY ? 0.f : M;
            float sum = 0.f, wsum = 0.f;
            auto add = [&](const float *p) {
                const float f = ex2(p[HD] - b);
                sum = fmaf(f, p[col == HD ? 0 : col], sum);
                wsum = fmaf(f, p[HD + 1], wsum);
            };
            if (tp) add(tp);
            for (uint32_t w = h0; w < h1; w++)
                if (info[w].has_head) add(slots + ((size_t)w * rb + row) * PS);
            if (front || back) {
                __stcg(slot + i, col == HD ? M : col == HD + 1 ? wsum : sum);
            } else if (col < HD) {
                const uint32_t r = it.row0 + row, tk = r / A.group;
                A.out[(size_t)(it.seq_first + tk) * A.ld_out + (size_t)(it.head * A.group + r - tk * A.group) * HD + col] =
                    wsum == 0.f ? 0.f : sum * (1.0f / wsum);
            }
        }
        if (!front && !back) return;
        // blocks that have a part: those whose cut lies inside the item, and the one in front of the first such cut
        const uint32_t i0 = it.item0, i1 = it.item0 + it.item_tiles;
        const uint32_t c_lo = (uint32_t)(((uint64_t)(i0 + 1u) * line_blocks - 1u) / line);   // block that holds the item's first tile
        const uint32_t c_hi = (uint32_t)(((uint64_t)i1 * line_blocks - 1u) / line);          // ... and its last
        __threadfence();
        __syncthreads();
        if (threadIdx.x == 0) {
            const uint32_t n = atomicAdd(&A.ticket[c_lo], 1u);
            last_here = n == c_hi - c_lo;
            if (last_here) A.ticket[c_lo] = 0u;
        }
        __syncthreads();
        if (!last_here) return;
        __threadfence();
        for (uint32_t i = threadIdx.x; i < rb * HD; i += THREADS) {
            const uint32_t row = i / HD, col = i - row * HD;
            if (it.row0 + row >= R) continue;
            auto part = [&](uint32_t c) { return A.part + (((size_t)c * 2u + (c == c_lo ? 1u : 0u)) * rb + row) * PS; };
            float M = -INFINITY;
            for (uint32_t c = c_lo; c <= c_hi; c++) M = fmaxf(M, __ldcg(part(c) + HD));
            const float b = M == -INFINITY ? 0.f : M;
            float sum = 0.f, wsum = 0.f;
            for (uint32_t c = c_lo; c <= c_hi; c++) {
                const float *p = part(c);
                const float f = ex2(__ldcg(p + HD) - b);
                sum = fmaf(f, __ldcg(p + col), sum);
                wsum = fmaf(f, __ldcg(p + HD + 1), wsum);
            }
            const uint32_t r = it.row0 + row, tk = r / A.group;
            A.out[(size_t)(it.seq_first + tk) * A.ld_out + (size_t)(it.head * A.group + r - tk * A.group) * HD + col] =
                wsum == 0.f ? 0.f : sum * (1.0f / wsum);
        }
    };
    int a_tail = -1;
    uint32_t h0 = 0;
    bool open = false, front = false;
    PaWorker::Part it{};
    for (uint32_t w = 0; w < workers; w++) {
        const PaWorker &I = info[w];
        if (I.has_head) {
            if (!open) {
                open = front = true;
                a_tail = -1;
                h0 = w;
                it = I.head;
            }
            if (I.head_ended) {
                emit(a_tail, h0, w + 1u, it, front, false);
                open = front = false;
            }
        }
        if (I.has_tail) {
            open = true;
            front = false;
            a_tail = (int)w;
            h0 = w + 1u;
            it = I.tail;
        }
    }
    if (open) emit(a_tail, h0, workers, it, front, true);
}

// Blocks that the launch may have: one on each SM.
static uint32_t attn_blocks(const strix_cuda *h) { return (uint32_t)std::min<int>(std::max(h->num_sms, 1), (int)PA_MAX_BLOCKS); }

// Rows of a KV head that a sequence brings on average decide the form: up to 8, one product for values and remainders; beyond,
// 16 rows a warp and as many warps to a worker as cover them (at most all of a block).
static void attn_form(const PagedView &V, uint32_t group, bool &wide, uint32_t &wm) {
    const uint64_t rows = ((uint64_t)V.n_rows * group + V.n_seq - 1) / std::max(V.n_seq, 1u);
    const bool f16 = V.type == STRIX_KV_F16;
    wide = rows > 8;
    const uint32_t most = V.head_dim >= 192 ? 4u : 8u;
    wm = 1;
    while (wide && wm < most && 16ull * wm < rows) wm *= 2;
    if (wide && V.head_dim >= 192 && f16 && wm < 2) wm = 2;  // (the rings of four workers do not fit)
}

static size_t attn_work_bytes(const strix_cuda *h, const PagedView &V, uint32_t group) {
    bool wide;
    uint32_t wm;
    attn_form(V, group, wide, wm);
    const size_t rb = wide ? 16u * wm : 8u;
    const size_t part = (size_t)attn_blocks(h) * 2 * rb * (V.head_dim + 2) * 4;
    return (PA_MAX_BLOCKS * 4 + part + 255) & ~(size_t)255;
}

template <int HD, int TYPE, bool WIDE>
static cudaError_t attn_launch(const strix_cuda *h, PagedAttnArgs &A, cudaStream_t stream) {
    using S = PaShape<HD, TYPE, WIDE>;
    const int workers = S::NW / (int)A.wm;
    const int stages = S::stages_for((int)A.wm, h->smem_optin - PA_STATIC);
    const size_t smem = (size_t)workers * stages * S::STAGE + S::fixed(workers, stages);
    if (smem + PA_STATIC > h->smem_optin || (size_t)stages * S::STAGE < (size_t)S::ROWS * A.wm * S::PSTRIDE * 4) return cudaErrorInvalidConfiguration;
    cudaError_t e = cudaFuncSetAttribute(paged_attn_kernel<HD, TYPE, WIDE>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return e;
    A.stages = (uint32_t)stages;
    paged_attn_kernel<HD, TYPE, WIDE><<<attn_blocks(h), (S::NW + 1) * 32, smem, stream>>>(A);
    return cudaGetLastError();
}

}  // namespace strix

using namespace strix;

static int attn_check(strix_cuda *h, const char *who, const strix_kv_pages *cache, const strix_kv_batch *batch, uint32_t n_heads, PagedView &V) {
    const int rc = serve_check(h, who, cache, batch, &V);
    if (rc != 1) return rc;
    if (n_heads == 0 || n_heads > 65535u || n_heads % V.n_kv) return 0;
    // the line of tiles is counted in 31 bits
    const uint64_t rb = 8, group = n_heads / V.n_kv;
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
    if (A.V.n_seq == 0 || A.V.n_rows == 0) return 1;
    if (!d_q || !d_out) return serve_fail(h, who, "d_q or d_out missing");
    if (!d_work || (reinterpret_cast<uintptr_t>(d_work) & 255u)) return serve_fail(h, who, "d_work must be 256-byte aligned");
    A.group = n_heads / A.V.n_kv;
    if (work_bytes < attn_work_bytes(h, A.V, A.group)) return serve_fail(h, who, "work_bytes too small");
    A.q = d_q;
    A.out = d_out;
    A.n_heads = n_heads;
    A.window = window;
    A.cap = A.V.pages_ld * A.V.page_tokens;
    A.scale = scale;
    A.vec = ((reinterpret_cast<uintptr_t>(d_q) | reinterpret_cast<uintptr_t>(d_out)) & 15u) == 0 && ((A.ld_q | A.ld_out) & 3u) == 0;
    A.ticket = static_cast<uint32_t *>(d_work);
    A.part = reinterpret_cast<float *>(static_cast<uint8_t *>(d_work) + PA_MAX_BLOCKS * 4);
    bool wide;
    attn_form(A.V, A.group, wide, A.wm);
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
        switch (hd) {
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
