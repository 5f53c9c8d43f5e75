// What the kernels of attention over a paged cache share: their arguments, the line of tiles that is dealt out to blocks, the
// join of parts that several blocks have, and small device helpers.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "kv_pages.cuh"

namespace strix {

constexpr uint32_t PA_MAX_BLOCKS = 1024;  // tickets at the start of the workspace
constexpr uint32_t PA_MAX_SEQ = 8192;     // their running tile counts lie in shared memory while a block finds its place
constexpr uint32_t PA_SNAP = 16;
constexpr size_t PA_STATIC = 2048;  // 1024 to align the rings, the rest static shared memory and what the system keeps

struct PagedAttnArgs {
    CUtensorMap k_map, v_map;  // [page][KV head and slot][element]
    PagedView V;
    const float *q;
    float *out;
    size_t ld_q, ld_out;
    uint32_t group, window, cap;  // cap: tokens a row of the page table can hold
    uint32_t g_mul, g_shift;               // division by group
    float scale, scale_m;
    int scale_e;               // row blocks: scale log2(e) = scale_m (of magnitude [1/2, 1), or 0) times 2^scale_e
    uint32_t wm, halves, vec;  // warps of a worker; half tiles of a ring; q and out rows start on 16 bytes
    uint32_t *ticket;          // [PA_MAX_BLOCKS]
    float *part;               // [blocks][2][rows of a worker][HD + 2]
};

// What the first warp tells a worker about a tile.
struct __align__(16) PaTile {
    uint32_t tile, flags, valid, row0;        // tile of the item; PA_*; one bit for each page of the tile; first row of the block
    uint32_t seq_first, seq_rows, ctx, head;  // first row of the sequence, its new rows, tokens before them, KV head (kv_attn.cu: with PA_NEW)
    float ks[4], vs[4];                       // the scales of the tile's pages
};
enum : uint32_t { PA_NEW = 1, PA_END = 2, PA_WHOLE = 4, PA_HEAD = 8 };  // first / last tile of the segment here; item complete here; begun elsewhere
constexpr uint32_t PA_ITEM = 4;  // with row blocks: flags >> PA_ITEM counts the items of the block

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
// A tile whose pages have scales of their own: its weights meet their pages' scales before the product, and a power of two 2^u
// brings the largest weight times scale of a row (`most`, the scales times 2^-15) to [2^14, 2^15). What multiplies the product is 2^(15 - u).
// (u stops at 127: below scales of 2^-112 the weights are a few bits further down.)
__device__ __forceinline__ void row_scale(float most, float &up, float &back) {
    const int e = max((int)(__float_as_uint(most) >> 23) - 127, -113);
    up = __uint_as_float((uint32_t)(14 - e + 127) << 23);
    back = __uint_as_float((uint32_t)(e + 1 + 127) << 23);
}
// the factor of a page's weights; bounded where its weights are below 2^-126 of the row's largest
__device__ __forceinline__ float page_factor(float vs15, float up) { return fminf(vs15 * up, 8.5e37f); }
__device__ __forceinline__ void tma_load_3d(void *dst, const CUtensorMap *map, uint32_t x, uint32_t y, uint32_t z, uint64_t *bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
                     smem_u32(dst)),
                 "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
                 : "memory");
}
__device__ __forceinline__ void mbar_expect_tx(uint64_t *bar, uint32_t bytes) {
    asm volatile("mbarrier.expect_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}
// true in one lane of the warp, in a form that lets the compiler know it is one
__device__ __forceinline__ bool elect_lane() {
    uint32_t one;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(one));
    return one != 0u;
}
// n / group for n < 2^31
__device__ __forceinline__ uint32_t by_group(const PagedAttnArgs &A, uint32_t n) { return (__umulhi(n, A.g_mul) + n) >> A.g_shift; }

// Tiles of row block mb of a sequence: [lo_tile, lo_tile + n). rb: rows of a block, a power of two.
template <int TT>
__device__ __forceinline__ uint32_t block_tiles(const PagedAttnArgs &A, uint32_t rb, uint32_t rows, uint32_t ctx, uint32_t mb,
                                                uint32_t &lo_tile) {
    const uint32_t R = rows * A.group, r0 = mb * rb, r1 = min(R, r0 + rb) - 1u;
    const uint32_t p0 = ctx + by_group(A, r0), p1 = ctx + by_group(A, r1);  // positions of the first and last row (below 2^32)
    const uint32_t hi = min(A.cap, p1 + 1u);
    const uint32_t lo = A.window && p0 >= A.window ? p0 + 1u - A.window : 0u;
    lo_tile = lo / TT;
    return hi > lo ? (hi + TT - 1u) / TT - lo_tile : 0u;
}

// Does any row of the block see position `last` or a later one? Pages that end before that may be anybody's by now.
__device__ __forceinline__ bool still_seen(const PagedAttnArgs &A, uint32_t rb, uint32_t ctx, uint32_t mb, uint32_t last) {
    if (!A.window) return true;
    const uint32_t p0 = ctx + by_group(A, mb * rb);
    return p0 < A.window || last > p0 - A.window;
}

// A place in the line of tiles.
struct __align__(16) PaPlace {
    uint32_t s, first, rows, ctx, mb, head, lo_tile, tiles, at;  // item: tiles of it, `at` the place within
    uint32_t item0;                                              // the line's index of the item's first tile
};

__device__ __forceinline__ void load_seq(const PagedAttnArgs &A, uint32_t s, PaPlace &P) {
    uint32_t end;
    bool bad = false;
    P.s = s;
    seq_rows(A.V, s, P.first, end, bad);
    P.rows = end - P.first;
    P.ctx = (uint32_t)A.V.ctx[s];
}
// All tiles of a sequence.
template <int TT>
__device__ __forceinline__ uint32_t seq_tiles(const PagedAttnArgs &A, uint32_t rb, uint32_t s) {
    PaPlace P;
    load_seq(A, s, P);
    if ((int)P.ctx < 0 || P.rows == 0u) return 0u;
    uint32_t n = 0, lo;
    const uint32_t blocks = (P.rows * A.group + rb - 1u) / rb;
#pragma unroll 1
    for (uint32_t mb = 0; mb < blocks; mb++) n += block_tiles<TT>(A, rb, P.rows, P.ctx, mb, lo);
    return n * A.V.n_kv;
}
// The place of line index x; upto[s]: tiles of the sequences up to and including s.
template <int TT>
__device__ __forceinline__ void find_place(const PagedAttnArgs &A, uint32_t rb, const uint32_t *upto, uint32_t x, PaPlace &P) {
    uint32_t lo = 0, hi = A.V.n_seq - 1u;  // the first sequence with upto > x
#pragma unroll 1
    while (lo < hi) {
        const uint32_t mid = (lo + hi) / 2u;
        if (upto[mid] > x) hi = mid; else lo = mid + 1u;
    }
    load_seq(A, lo, P);
    uint32_t off = x - (lo ? upto[lo - 1u] : 0u), n = 0, first_tile = 0;
    const uint32_t blocks = (P.rows * A.group + rb - 1u) / rb;
#pragma unroll 1
    for (P.mb = 0;; P.mb++) {
        n = block_tiles<TT>(A, rb, P.rows, P.ctx, P.mb, first_tile);
        if (off < n * A.V.n_kv || P.mb + 1u >= blocks) break;
        off -= n * A.V.n_kv;
    }
    P.lo_tile = first_tile;
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
#pragma unroll 1
    for (;;) {
        const uint32_t blocks = (P.rows * A.group + rb - 1u) / rb;
        if ((int)P.ctx >= 0 && ++P.mb < blocks) {
            P.tiles = block_tiles<TT>(A, rb, P.rows, P.ctx, P.mb, P.lo_tile);
            if (P.tiles) return;
            continue;
        }
        if (P.s + 1u >= A.V.n_seq) {
            P.tiles = 0;
            return;
        }
        load_seq(A, P.s + 1u, P);
        P.mb = 0xffffffffu;
        if (P.rows == 0u) P.ctx = 0xffffffffu;
    }
}

// The line's division among blocks: equal to within a tile.
struct PaCuts {
    uint32_t per, rem;
    __device__ PaCuts(uint32_t total, uint32_t parts) : per(total / parts), rem(total - per * parts) {}
    __device__ uint32_t cut(uint32_t c) const { return c * per + min(c, rem); }
    __device__ uint32_t part_of(uint32_t x) const {  // the part that holds index x
        const uint32_t big = rem * (per + 1u);
        return x < big ? x / (per + 1u) : rem + (x - big) / per;
    }
};

// Where cut x of the line falls: cuts inside an item of at most `most` tiles move to its nearer end.
__device__ __forceinline__ uint32_t snapped(const PaPlace &P, uint32_t x, uint32_t most) {
    if (P.at == 0u || P.tiles > most) return x;
    return 2u * P.at < P.tiles ? P.item0 : P.item0 + P.tiles;
}

// An item that a block has only in part: what the joins need to know of it.
struct PaPart {
    uint32_t seq_first, seq_rows, row0, head, item0, item_tiles;
};
struct PaWorkerParts {  // of a block that is one worker: begun in the block in front, going on in the next
    PaPart front, back;
    uint32_t has_front, has_back;
};

// out row of row `row` of an item
__device__ __forceinline__ float *item_row(const PagedAttnArgs &A, uint32_t hd, uint32_t seq_first, uint32_t row0, uint32_t head, uint32_t row) {
    const uint32_t r = row0 + row, tk = by_group(A, r);
    return A.out + (size_t)(seq_first + tk) * A.ld_out + (size_t)(head * A.group + r - tk * A.group) * hd;
}

// Joins one row of an item from the parts of `n` blocks from block lo on (the first has its part in slot 1, the others in slot
// 0), by a warp: parts are weighted sums, maximum, sum of weights, taken in the order of the blocks.
template <int HD>
__device__ __forceinline__ void join_row(const PagedAttnArgs &A, uint32_t rb, uint32_t lo, uint32_t n, uint32_t row, float *dst) {
    constexpr int PS = HD + 2, DL = (HD / 2 + 31) / 32;  // DL: pairs of a row in a lane
    const uint32_t lane = threadIdx.x & 31u;
    auto part = [&](uint32_t i) { return A.part + (((size_t)(lo + i) * 2u + (i == 0u ? 1u : 0u)) * rb + row) * PS; };
    constexpr int AHEAD = 4;  // parts on their way at once, from before their weights are known: a join is a chain of loads
    float2 v[AHEAD][DL];
    auto fetch = [&](uint32_t i0) {
#pragma unroll
        for (int j = 0; j < AHEAD; j++) {
            const float2 *src = reinterpret_cast<const float2 *>(part(i0 + j));
#pragma unroll
            for (int k = 0; k < DL; k++) v[j][k] = i0 + j < n && k * 32 + lane < HD / 2 ? __ldcg(src + k * 32 + lane) : make_float2(0.f, 0.f);
        }
    };
    float2 ml = lane < n ? __ldcg(reinterpret_cast<const float2 *>(part(lane) + HD)) : make_float2(-INFINITY, 0.f);
    fetch(0u);
    float M = ml.x, L = 0.f;
#pragma unroll 1
    for (uint32_t i = lane + 32u; i < n; i += 32u) M = fmaxf(M, __ldcg(part(i) + HD));
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, d));
    float2 acc[DL];
#pragma unroll
    for (int k = 0; k < DL; k++) acc[k] = make_float2(0.f, 0.f);
    float f = 0.f;
#pragma unroll 1
    for (uint32_t i = 0; i < n; i += AHEAD) {
        if ((i & 31u) == 0u) {  // the weights of the next 32 parts, one to a lane
            if (i) ml = lane + i < n ? __ldcg(reinterpret_cast<const float2 *>(part(lane + i) + HD)) : make_float2(-INFINITY, 0.f);
            f = ml.x == -INFINITY ? 0.f : ex2(ml.x - M);
            L += f * ml.y;
        }
#pragma unroll
        for (int j = 0; j < AHEAD; j++) {
            const float fw = __shfl_sync(0xffffffffu, f, (i + j) & 31u);
            if (i + j >= n) continue;  // (nothing of a part that is none, whatever the weight in its lane)
#pragma unroll
            for (int k = 0; k < DL; k++) {
                acc[k].x = fmaf(fw, v[j][k].x, acc[k].x);
                acc[k].y = fmaf(fw, v[j][k].y, acc[k].y);
            }
        }
        if (i + AHEAD < n) fetch(i + AHEAD);
    }
    L = warp_sum(L);
    const float inv = L == 0.f ? 0.f : 1.0f / L;
#pragma unroll
    for (int k = 0; k < DL; k++)
        if (k * 32 + lane < HD / 2) {
            dst[2 * (k * 32 + lane)] = acc[k].x * inv;
            dst[2 * (k * 32 + lane) + 1] = acc[k].y * inv;
        }
}

// Zeros for rows that see nothing, and the status of lengths beyond the table: each sequence is looked at by one warp of the grid
// (n_warps of a block take part). Returns whether something was wrong.
template <int HD, int TT>
__device__ __forceinline__ bool empty_rows(const PagedAttnArgs &A, uint32_t rb, uint32_t warp, uint32_t n_warps) {
    const PagedView &V = A.V;
    const uint32_t lane = threadIdx.x & 31u;
    bool bad = false;
#pragma unroll 1
    for (uint32_t s = blockIdx.x * n_warps + warp; s < V.n_seq; s += gridDim.x * n_warps) {
        uint32_t first, end;
        seq_rows(V, s, first, end, bad);
        const int ctx = V.ctx[s];
        const uint32_t rows = end - first;
        const bool over = ctx >= 0 && rows && (uint64_t)(uint32_t)ctx + rows > A.cap;
        bad |= over;
        if (ctx < 0 || over) {
            const uint32_t R = rows * A.group, nb = (R + rb - 1u) / rb;
#pragma unroll 1
            for (uint32_t mb = 0; mb < nb; mb++) {
                uint32_t lo;
                if (ctx >= 0 && block_tiles<TT>(A, rb, rows, (uint32_t)ctx, mb, lo)) continue;
#pragma unroll 1
                for (uint32_t r = mb * rb; r < min(R, (mb + 1u) * rb); r++)
#pragma unroll 1
                    for (uint32_t h = 0; h < V.n_kv; h++) {
                        float *dst = item_row(A, HD, first, r, h, 0u);
#pragma unroll 1
                        for (uint32_t i = lane; i < HD; i += 32u) dst[i] = 0.f;
                    }
            }
        }
    }
    return bad;
}

// Running tile counts of the sequences, by all THREADS of a block; returns the total. Offsets that go down may give the same rows to
// many sequences: where they give away more rows than there are, nothing is counted and `over` is set (the sizes that the
// host has checked hold only up to there).
template <int TT, int THREADS>
__device__ __forceinline__ uint32_t count_tiles(const PagedAttnArgs &A, uint32_t rb, uint32_t *upto, uint32_t *scan, bool &over) {
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
    bool down = false;
#pragma unroll 1
    for (uint32_t s = threadIdx.x; s < A.V.n_seq; s += THREADS) down |= A.V.row0[s + 1u] < A.V.row0[s];
    over = false;
    if (__syncthreads_or(down)) {
        uint64_t rows = 0;
#pragma unroll 1
        for (uint32_t s = 0; s < A.V.n_seq; s++) {
            uint32_t first, end;
            bool bad = false;
            seq_rows(A.V, s, first, end, bad);
            rows += end - first;
        }
        over = rows > A.V.n_rows;
        if (over) return 0u;
    }
    uint32_t total = 0;
#pragma unroll 1
    for (uint32_t c = 0; c < A.V.n_seq; c += THREADS) {
        uint32_t n = c + threadIdx.x < A.V.n_seq ? seq_tiles<TT>(A, rb, c + threadIdx.x) : 0u;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const uint32_t v = __shfl_up_sync(0xffffffffu, n, d);
            if ((int)lane >= d) n += v;
        }
        if (lane == 31u) scan[warp] = n;
        __syncthreads();
        uint32_t before = total;
#pragma unroll 1
        for (uint32_t w = 0; w < THREADS / 32; w++) {
            if (w < warp) before += scan[w];
            total += scan[w];
        }
        if (c + threadIdx.x < A.V.n_seq) upto[c + threadIdx.x] = before + n;
        __syncthreads();
    }
    return total;
}

// A cache as [page][KV head and slot][element], copied in boxes of `rows` slots by `box` elements (kv_attn.cu).
bool attn_map(CUtensorMap *map, const PagedView &V, void *base, uint32_t box, uint32_t rows, bool swizzled);
// Attention of row blocks of 128 rows on tcgen05 (kv_attn_rows.cu): head sizes 64 and 128.
cudaError_t launch_attn_rows(const strix_cuda *h, PagedAttnArgs &A, uint32_t blocks, cudaStream_t stream);

}  // namespace strix
