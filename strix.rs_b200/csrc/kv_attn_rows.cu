// Attention over a paged KV cache for many rows of a KV head at once (prompt chunks, verify batches): row blocks of 128 rows on the
// tcgen05 tensor cores. Contract: include/strix_serve.h; the form for few rows, the line of tiles and the joins: kv_attn.cu.
//
// Arithmetic as there: f16 products with f32 sums, q and the weights in two f16 halves (the value, and what rounding it left), so
// every product runs twice; q scaled to a largest value in [2^13, 2^15), weights relative to the tile's largest (as
// there, with their pages' scales where those differ); e4m3 cache values widened to f16, exactly. A tile is 64 tokens of one KV head.
//   S = Qhi K^T + Qlo K^T     128 x 64 sums in TMEM, operands in shared memory (K-major, 128-byte swizzle)
//   P = 2^(S c - max), split  by the thread that has the row, written to TMEM as the A operand of
//   O = Phi V + Plo V         128 x head size, from zero for every tile; V as it lies, [token][dimension] (MN-major)
// The running O is kept in registers, a row to a thread: sums over tiles then round to nearest (chained accumulation in the tensor
// cores truncates), and a new maximum costs no pass over TMEM.
//
// Roles of the 20 warps (96 registers each at launch, shared out anew: the sums get 176, the last eight warps 56):
//   0-3, 4-7  softmax of the even and of the odd tiles. A tile's weights are relative to its own largest score, so these warps
//             carry nothing from tile to tile: they leave the tile's maximum and sum of weights in shared memory, and
//   8-11      the sums bring the tiles' products O to the running maximum as they add them, and write the finished rows
//   12-15     make operands: q split, e4m3 to f16, rows of v that nobody sees to zero
//   16        copies by TMA;   17, 18  issue the products S and O
// S, P and O are double-buffered in TMEM. At the end warps 0-15 join the parts of items that other blocks share.
//
// What bounds it: the products are 1024 clocks of a tile at head size 128 (S reads both operands from shared memory, 96 bytes of
// them for each of 64 columns). Measured are about 3000: exponentials, splits and the passes over TMEM take the softmax warps most
// of that, at half of the issue slots. Loops over tiles stay rolled, because instruction fetch bounded the unrolled form (135 KB,
// all roles at once: 460 us, 320 once rolled, in earlier forms). S held in registers, so that its columns are free sooner, was
// no faster (201 against 197 us). 512 rows behind 8000 tokens (32 heads, 8 KV heads of 128, e4m3): 197 us, 352 TFLOP/s
// of useful products, as many again for the second halves (220 us with 16-token pages, whose scales meet the weights row by
// row); 8 x 5 rows behind 1000-5000 tokens, f16: 55 us.
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

#include "kv_line.cuh"

namespace strix {

constexpr uint32_t RA_ROWS = 128, RA_TT = 64, RA_THREADS = 640, RA_DESCS = 16, RA_QBUF = 4, RA_STATS = 8;
constexpr uint32_t RA_SNAP = 4;   // cuts inside an item of at most this many tiles move to its end (256 tokens, as PA_SNAP tiles are)
constexpr uint32_t RA_LEAST = 4;  // tiles a block takes at least

template <int HD, int TYPE>
struct RowsShape {
    static constexpr int EL = TYPE == STRIX_KV_F16 ? 2 : 1;
    static constexpr int BLOCKS = HD / 64;            // blocks of 64 elements, 128 bytes a row
    static constexpr int QB = 128 * HD * 2;           // bytes of one half of q
    static constexpr int OPB = 64 * HD * 2;           // bytes of the k or v of a tile as an operand
    static constexpr int NS = 3;                      // operand tiles of k, and of v
    static constexpr int RAWB = EL == 1 ? 64 * HD : 0;
    static constexpr int NR = EL == 1 ? 2 : 0;        // tiles of codes of k, and of v
    static constexpr int NL = EL == 1 ? NR : NS;      // tiles that copies land in
    static constexpr bool RAWSWZ = HD == 128;         // rows of 128 codes are swizzled on their way, rows of 64 lie as they are
    static constexpr int BARS = 4 * NL + 4 * NS + 2 + 5 * 2 + (int)RA_STATS;
    static constexpr size_t SMEM = 2 * QB + 2 * NS * OPB + 2 * NR * RAWB + RA_DESCS * sizeof(PaTile) + RA_QBUF * 128 * 4 + (EL == 1 ? 3 : 2) * RA_STATS * 128 * 4 + BARS * 8 + 1024;
    // TMEM columns: S 2 x 64, P 2 x (32 + 32), O 2 x HD
    static constexpr uint32_t COL_P = 128, COL_O = 256;
};

__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_commit(uint64_t *bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void tc_mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t add) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, {%5, %5, %5, %5}, p;\n\t}" ::"r"(d),
                 "l"(a), "l"(b), "r"(idesc), "r"(add), "r"(0u)
                 : "memory");
}
__device__ __forceinline__ void tc_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t add) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%5, %5, %5, %5}, p;\n\t}" ::"r"(d),
                 "r"(a), "l"(b), "r"(idesc), "r"(add), "r"(0u)
                 : "memory");
}
#define STRIX_R8(r, i) "=r"(r[i]), "=r"(r[i + 1]), "=r"(r[i + 2]), "=r"(r[i + 3]), "=r"(r[i + 4]), "=r"(r[i + 5]), "=r"(r[i + 6]), "=r"(r[i + 7])
#define STRIX_W8(r, i) "r"(r[i]), "r"(r[i + 1]), "r"(r[i + 2]), "r"(r[i + 3]), "r"(r[i + 4]), "r"(r[i + 5]), "r"(r[i + 6]), "r"(r[i + 7])
__device__ __forceinline__ void tc_ld32(uint32_t taddr, uint32_t *r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : STRIX_R8(r, 0), STRIX_R8(r, 8), STRIX_R8(r, 16), STRIX_R8(r, 24)
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tc_ld16(uint32_t taddr, uint32_t *r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : STRIX_R8(r, 0), STRIX_R8(r, 8)
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tc_st8(uint32_t taddr, const uint32_t *r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x8.b32 [%8], {%0, %1, %2, %3, %4, %5, %6, %7};" ::STRIX_W8(r, 0), "r"(taddr)
        : "memory");
}
#undef STRIX_R8
#undef STRIX_W8
// two f32 multiply-adds, or additions, in one instruction
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 r;
    asm("{\n\t.reg .b64 a, b, c, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
        "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "=f"(r.x), "=f"(r.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return r;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 r;
    asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tadd.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "=f"(r.x), "=f"(r.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}
__device__ __forceinline__ void tc_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Shared-memory matrix descriptor with the 128-byte swizzle (layout type 2, version 1): 8 rows of 128 bytes every 1024 bytes. K-major
// operands need no leading offset; for v, whose rows are tokens and whose contiguous dimension is N, it is the distance
// between blocks of 64 dimensions.
__device__ __forceinline__ uint64_t desc_sw128(uint32_t saddr, uint32_t leading) {
    return (uint64_t)((saddr >> 4) & 0x3fffu) | (uint64_t)(leading >> 4) << 16 | (uint64_t)64u << 32 | (uint64_t)1u << 46 | (uint64_t)2u << 61;
}
// Instruction descriptor (kind::f16): D f32 (bit 4), A and B f16, B MN-major (bit 16), N >> 3 in bits 17-22, M >> 4 in bits 24-28.
constexpr uint32_t rows_idesc(uint32_t n, bool mn) { return 1u << 4 | (mn ? 1u << 16 : 0u) | (n >> 3) << 17 | (RA_ROWS >> 4) << 24; }

template <int HD, int TYPE>
__global__ void __launch_bounds__(RA_THREADS, 1) attn_rows_kernel(const __grid_constant__ PagedAttnArgs A) {
    using S = RowsShape<HD, TYPE>;
    constexpr int EL = S::EL, NS = S::NS, NL = S::NL;
    extern __shared__ __align__(128) uint8_t smem_raw[];
    uint8_t *smem = smem_raw + (-smem_u32(smem_raw) & 1023u);
    uint8_t *q_smem = smem, *op = smem + 2 * S::QB, *raw = op + 2 * NS * S::OPB;  // op, raw: the tiles of k, then those of v
    PaTile *desc = reinterpret_cast<PaTile *>(raw + 2 * S::NR * S::RAWB);
    float *q_factor = reinterpret_cast<float *>(desc + RA_DESCS);  // [RA_QBUF][128]
    float *tile_m = q_factor + RA_QBUF * 128, *tile_l = tile_m + RA_STATS * 128;  // [RA_STATS][128]
    float *tile_v = tile_l + RA_STATS * 128;  // the same, with e4m3: what scales the tile's product
    uint64_t *bars = reinterpret_cast<uint64_t *>(tile_v + (EL == 1 ? RA_STATS * 128 : 0));
    uint64_t *land_full = bars, *land_empty = land_full + 2 * NL;  // [k, v][NL]
    uint64_t *op_full = land_empty + 2 * NL, *op_empty = op_full + 2 * NS;
    uint64_t *q_full = op_empty + 2 * NS, *q_empty = q_full + 1;
    uint64_t *s_full = q_empty + 1, *s_empty = s_full + 2, *p_full = s_empty + 2, *o_full = p_full + 2, *o_empty = o_full + 2, *m_full = o_empty + 2;
    __shared__ uint32_t scan[RA_THREADS / 32], tmem_slot, last_here[2];
    __shared__ volatile uint32_t gave_up;
    __shared__ PaWorkerParts parts;
    const PagedView &V = A.V;
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;

    uint32_t *upto = reinterpret_cast<uint32_t *>(op);
    bool over;
    const uint32_t total = count_tiles<RA_TT, RA_THREADS>(A, RA_ROWS, upto, scan, over);
    if (threadIdx.x == 0) {
        for (int i = 0; i < 2 * NL; i++) {
            mbar_init(&land_full[i], 1);
            mbar_init(&land_empty[i], EL == 1 ? 4 : 1);
        }
        for (int i = 0; i < 2 * NS; i++) {
            mbar_init(&op_full[i], 4);
            mbar_init(&op_empty[i], 1);
        }
        mbar_init(q_full, 4);
        mbar_init(q_empty, 1);
        for (int i = 0; i < 2; i++) {
            mbar_init(&s_full[i], 1);
            mbar_init(&s_empty[i], 4);
            mbar_init(&p_full[i], 4);
            mbar_init(&o_full[i], 1);
            mbar_init(&o_empty[i], 4);
        }
        for (uint32_t i = 0; i < RA_STATS; i++) mbar_init(&m_full[i], 4);
        mbar_fence_init();
        gave_up = 0u;
        parts.has_front = parts.has_back = last_here[0] = last_here[1] = 0u;
    }
    for (uint32_t i = threadIdx.x; i < RA_DESCS * 4u; i += RA_THREADS) desc[i / 4u].ks[i & 3u] = desc[i / 4u].vs[i & 3u] = 0.f;
    if (warp == 17) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    // ---- this block's stretch of the line
    const uint32_t line_blocks = min(gridDim.x, (total + RA_LEAST - 1u) / RA_LEAST);
    uint32_t n_tiles = 0;
    PaPlace place{};
    if (blockIdx.x < line_blocks) {
        const PaCuts line(total, line_blocks);
        uint32_t x = line.cut(blockIdx.x + (lane & 1u));
        if (x < total) {
            find_place<RA_TT>(A, RA_ROWS, upto, x, place);
            x = snapped(place, x, RA_SNAP);
        }
        const uint32_t lo = __shfl_sync(0xffffffffu, x, 0);
        n_tiles = __shfl_sync(0xffffffffu, x, 1) - lo;
        if (n_tiles) find_place<RA_TT>(A, RA_ROWS, upto, lo, place);
    }
    fence_proxy_async_smem();  // f16 copies land where the counts were: all accesses to them come first
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    // A wait that has run out is the last one of the block: every role leaves its loop at its next wait and touches nothing of the tile,
    // whose description may not be there. By whole warps, whose lanes come to the same answer; wait_lane: by one lane.
    auto wait = [&](uint64_t *bar, uint32_t parity) {
#pragma unroll 1
        for (uint32_t it = 0; !__all_sync(0xffffffffu, mbar_try_wait(bar, parity)); it++)
            if (__any_sync(0xffffffffu, gave_up || it >= 1u << 22)) {
                gave_up = 1u;
                return false;
            }
        return true;
    };
    auto wait_lane = [&](uint64_t *bar, uint32_t parity) {
#pragma unroll 1
        for (uint32_t it = 0; !mbar_try_wait(bar, parity); it++)
            if (gave_up || it >= 1u << 22) {
                gave_up = 1u;
                return false;
            }
        return true;
    };
    // ... joins their parts, with warps 0 to 15
    auto join = [&] {
        asm volatile("bar.sync 1, 512;" ::: "memory");
#pragma unroll 1
        for (int e = 0; e < 2; e++) {
            if (!last_here[e]) continue;
            __threadfence();
            const PaCuts line(total, line_blocks);
            const PaPart &it = e == 0 ? parts.front : parts.back;
            const uint32_t lo = line.part_of(it.item0), cnt = line.part_of(it.item0 + it.item_tiles - 1u) - lo + 1u;
            const uint32_t R = min(RA_ROWS, it.seq_rows * A.group - it.row0);
#pragma unroll 1
            for (uint32_t r = warp; r < R; r += 16u) join_row<HD>(A, RA_ROWS, lo, cnt, r, item_row(A, HD, it.seq_first, it.row0, it.head, r));
        }
    };
    const uint32_t pshift = V.page_shift;
    const bool mixed = V.page_tokens < RA_TT;
    const uint32_t sub = min(RA_TT, V.page_tokens), n_sub = RA_TT / sub;

    if (warp < 8) {
        // ---- softmax: warps 0-3 take the even tiles, 4-7 the odd ones; the thread has row 32 (warp & 3) + lane of the block
        const uint32_t b = warp >> 2, row = threadIdx.x & 127u;
        const uint32_t t_row = tmem + (((warp & 3u) * 32u) << 16);
        float f_q = 0.f;
        uint32_t pos = 0, pos_lo = 0, pos_hi = 0, item = ~0u;
#pragma unroll 1
        for (uint32_t n = b; n < n_tiles; n += 2u) {
            if (!wait(&s_full[b], (n >> 1) & 1u)) break;
            tc_fence_after();
            const PaTile &d = desc[n % RA_DESCS];
            const uint32_t valid = d.valid, tok = d.tile * RA_TT;
            if (d.flags >> PA_ITEM != item) {
                item = d.flags >> PA_ITEM;
                const uint32_t R = d.seq_rows * A.group, ctx = d.ctx, row0 = d.row0;
                pos = ctx + by_group(A, min(row0 + row, R - 1u));
                pos_lo = ctx + by_group(A, min(row0 + (row & 96u), R - 1u));
                pos_hi = ctx + by_group(A, min(row0 + (row | 31u), R - 1u));
                f_q = q_factor[(item % RA_QBUF) * 128u + row];
            }
            uint64_t sees = ~0ull;  // one bit for each token that the row sees
            if (tok + RA_TT - 1u > pos_lo || valid != (1u << n_sub) - 1u || (A.window && pos_hi >= A.window && tok <= pos_hi - A.window)) {
                const uint32_t last = pos - tok, from = A.window && pos >= A.window && pos - A.window >= tok ? pos - A.window - tok + 1u : 0u;
                sees = pos < tok || from > 63u ? 0ull : ~0ull >> (63u - min(last, 63u)) & ~0ull << from;
#pragma unroll 1
                for (uint32_t j = 0; j < n_sub; j++)
                    if (!((valid >> j) & 1u)) sees &= ~((~0ull >> (64u - sub)) << (j * sub));
            }
            auto sums32 = [&](uint32_t *s, uint32_t c) {  // the sums of 32 tokens: sixteen are of one page
                tc_ld16(t_row + b * 64u + c, s);
                tc_ld16(t_row + b * 64u + c + 16u, s + 16);
                const uint32_t bits = (uint32_t)(sees >> c);
                tc_wait_ld();
                if (__any_sync(0xffffffffu, bits != ~0u)) {
#pragma unroll
                    for (int i = 0; i < 32; i++) s[i] = (bits >> i) & 1u ? s[i] : 0xff800000u;
                }
            };
            // The factor to exponents of two is positive, so the largest product is the largest score. It is a power of two (the rest of the
            // caller's scale went into q, and the pages' scales are powers of two), so that it can multiply inside the exponent's
            // subtraction: what is taken off there is the maximum without any rounding, however large the scores are.
            auto factor = [&](uint32_t c) { return fmaxf(d.ks[mixed ? c >> pshift : 0u] * f_q, 0x1p-100f); };
            float top = -INFINITY, most = 0.f;  // most: largest weight times scale, with several scales in the tile
#pragma unroll 1
            for (uint32_t c = 0; c < RA_TT; c += 32u) {
                uint32_t s[32];
                sums32(s, c);
#pragma unroll
                for (int h = 0; h < 32; h += 16) {
                    float t0 = __uint_as_float(s[h]), t1 = __uint_as_float(s[h + 1]);
#pragma unroll
                    for (int i = h + 2; i < h + 16; i += 2) {
                        t0 = fmaxf(t0, __uint_as_float(s[i]));
                        t1 = fmaxf(t1, __uint_as_float(s[i + 1]));
                    }
                    const float t = fmaxf(t0, t1) * factor(c + h);
                    if (EL == 1 && mixed) {
                        const float now = fmaxf(top, t);
                        if (now > -INFINITY) most = fmaxf(most * ex2(top - now), ex2(t - now) * d.vs[(c + h) >> pshift]);
                        top = now;
                    } else {
                        top = fmaxf(top, t);
                    }
                }
            }
            const float base = top == -INFINITY ? 0.f : -__fsub_ru(top, 15.f);  // (upwards: no weight above 2^15)
            if (n >= 2u && !wait(&o_full[b], ((n >> 1) & 1u) ^ 1u)) break;  // the product of tile n - 2, which read this buffer of P
            tc_fence_after();
            float2 l2 = make_float2(0.f, 0.f);
            float up = 1.f;
            if constexpr (EL == 1) {
                float back = d.vs[0];
                if (mixed) row_scale(most, up, back);
                tile_v[(n % RA_STATS) * 128u + row] = back;
            }
#pragma unroll 1
            for (uint32_t c = 0; c < RA_TT; c += 32u) {
                uint32_t s[32];
                sums32(s, c);
#pragma unroll
                for (int h = 0; h < 32; h += 16) {
                    uint32_t hi[8], lo[8];
                    const float f = factor(c + h);
                    float2 p[8];
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        const float2 y = fma2(make_float2(__uint_as_float(s[h + 2 * i]), __uint_as_float(s[h + 2 * i + 1])), make_float2(f, f), make_float2(base, base));
                        p[i] = make_float2(ex2(y.x), ex2(y.y));
                        l2 = add2(l2, p[i]);
                    }
                    if (EL == 1 && mixed) {
                        const float w = page_factor(d.vs[(c + h) >> pshift] * 0x1p-15f, up);
#pragma unroll
                        for (int i = 0; i < 8; i++) p[i] = make_float2(p[i].x * w, p[i].y * w);
                    }
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        hi[i] = f32_to_f16x2(p[i].x, p[i].y);
                        const float2 left = fma2(__half22float2(*reinterpret_cast<const __half2 *>(&hi[i])), make_float2(-1.f, -1.f), p[i]);
                        lo[i] = f32_to_f16x2(left.x, left.y);
                    }
                    tc_st8(t_row + S::COL_P + b * 64u + (c + h) / 2u, hi);
                    tc_st8(t_row + S::COL_P + b * 64u + 32u + (c + h) / 2u, lo);
                }
            }
            tile_m[(n % RA_STATS) * 128u + row] = top;
            tile_l[(n % RA_STATS) * 128u + row] = l2.x + l2.y;
            tc_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(&s_empty[b]);
                mbar_arrive(&m_full[n % RA_STATS]);
                mbar_arrive(&p_full[b]);
            }
        }
        join();
    } else if (warp < 12) {
        // ---- sums: warps 8-11 add the tiles' products to O, whose row is kept by a thread, and write the finished items
        asm volatile("setmaxnreg.inc.sync.aligned.u32 176;");
        const uint32_t row = threadIdx.x & 127u, t_row = tmem + (((warp & 3u) * 32u) << 16);
        float o[HD], m = -INFINITY, l = 0.f;
        uint32_t it_first = 0, it_rows = 0, it_row0 = 0, it_head = 0;
        bool wrote = false;
#pragma unroll 1
        for (uint32_t n = 0; n < n_tiles; n++) {
            const uint32_t b = n & 1u;
            const PaTile &d = desc[n % RA_DESCS];
            if (!wait(&m_full[n % RA_STATS], (n / RA_STATS) & 1u)) break;
            const uint32_t flags = d.flags;
            if (flags & PA_NEW) {
                it_first = d.seq_first;
                it_rows = d.seq_rows;
                it_row0 = d.row0;
                it_head = d.head;
                m = -INFINITY;
                l = 0.f;
#pragma unroll
                for (int i = 0; i < HD; i++) o[i] = 0.f;
            }
            const float m_tile = tile_m[(n % RA_STATS) * 128u + row], m_new = fmaxf(m, m_tile);
            const float alpha = m_new == m ? 1.f : ex2(m - m_new), beta = m_new == m_tile ? 1.f : ex2(m_tile - m_new);
            const float w = EL == 1 ? beta * tile_v[(n % RA_STATS) * 128u + row] : beta;
            l = fmaf(tile_l[(n % RA_STATS) * 128u + row], beta, l * alpha);
            m = m_new;
            if (__any_sync(0xffffffffu, alpha != 1.f)) {
#pragma unroll
                for (int i = 0; i < HD; i++) o[i] *= alpha;
            }
            if (!wait(&o_full[b], (n >> 1) & 1u)) break;
            tc_fence_after();
#pragma unroll
            for (int c = 0; c < HD / 32; c++) {
                uint32_t r[32];
                tc_ld32(t_row + S::COL_O + b * HD + c * 32, r);
                tc_wait_ld();
#pragma unroll
                for (int i = 0; i < 32; i += 2) {
                    const float2 x = fma2(make_float2(__uint_as_float(r[i]), __uint_as_float(r[i + 1])), make_float2(w, w), make_float2(o[c * 32 + i], o[c * 32 + i + 1]));
                    o[c * 32 + i] = x.x;
                    o[c * 32 + i + 1] = x.y;
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&o_empty[b]);
            if (!(flags & PA_END)) continue;
            if (it_row0 + row < it_rows * A.group) {
                if (flags & PA_WHOLE) {
                    const float inv = l == 0.f ? 0.f : 1.0f / l;
                    float *dst = item_row(A, HD, it_first, it_row0, it_head, row);
                    if (A.vec) {
#pragma unroll
                        for (int i = 0; i < HD; i += 4)
                            *reinterpret_cast<float4 *>(dst + i) = make_float4(o[i] * inv, o[i + 1] * inv, o[i + 2] * inv, o[i + 3] * inv);
                    } else {
#pragma unroll
                        for (int i = 0; i < HD; i++) dst[i] = o[i] * inv;
                    }
                } else {
                    float *dst = A.part + (((size_t)blockIdx.x * 2u + (flags & PA_HEAD ? 0u : 1u)) * RA_ROWS + row) * (HD + 2);
#pragma unroll
                    for (int i = 0; i < HD; i += 2) __stcg(reinterpret_cast<float2 *>(dst + i), make_float2(o[i], o[i + 1]));
                    __stcg(reinterpret_cast<float2 *>(dst + HD), make_float2(m, l));
                }
            }
            wrote |= !(flags & PA_WHOLE);
        }
        if (wrote) __threadfence();
        asm volatile("bar.sync 2, 128;" ::: "memory");
        if (wrote && !gave_up) {  // items that several blocks have: is this the last of them to come here?
            const PaCuts line(total, line_blocks);
            if (warp < 10u && lane == 0) {
                const uint32_t e = warp - 8u;
                if (e == 0 ? parts.has_front : parts.has_back) {
                    const PaPart &it = e == 0 ? parts.front : parts.back;
                    const uint32_t lo = line.part_of(it.item0), hi = line.part_of(it.item0 + it.item_tiles - 1u);
                    if (atomicAdd(&A.ticket[lo], 1u) == hi - lo) {
                        A.ticket[lo] = 0u;
                        last_here[e] = 1u;
                    }
                }
            }
        }
        join();
    } else if (warp < 16) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
        // ---- operands: q of a new item; every tile's k and v
        const uint32_t tid = threadIdx.x & 127u, tr = tid & 63u, th = tid >> 6;  // token of the tile, half of its dimensions
        const bool bad = over || empty_rows<HD, RA_TT>(A, RA_ROWS, warp - 12u, 4u);
        report_bad(V, bad && lane == 0);
        uint32_t items = 0, pos_hi = 0, land = 0, land_phase = 0, st = 0, st_phase = 0;
        auto arrive = [&](uint64_t *bar) {
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar);
        };
#pragma unroll 1
        for (uint32_t n = 0; n < n_tiles; n++) {
            if (!wait(&land_full[land], land_phase)) break;
            const PaTile &d = desc[n % RA_DESCS];
            if (d.flags & PA_NEW) {
                if (!wait(q_empty, (items & 1u) ^ 1u)) break;
                const uint32_t R = d.seq_rows * A.group, r = d.row0 + tid, rr = min(r, R - 1u), tk = by_group(A, rr);
                pos_hi = d.ctx + by_group(A, min(d.row0 + RA_ROWS - 1u, R - 1u));
                const float *src = A.q + (size_t)(d.seq_first + tk) * A.ld_q + (size_t)(d.head * A.group + rr - tk * A.group) * HD;
                float top = 0.f;
                auto load4 = [&](int i) {
                    if (r >= R) return make_float4(0.f, 0.f, 0.f, 0.f);
                    return A.vec ? *reinterpret_cast<const float4 *>(src + i) : make_float4(src[i], src[i + 1], src[i + 2], src[i + 3]);
                };
#pragma unroll 8
                for (int i = 0; i < HD; i += 4) {
                    const float4 x = load4(i);
                    top = fmaxf(fmaxf(top, fmaxf(fabsf(x.x), fabsf(x.y))), fmaxf(fabsf(x.z), fabsf(x.w)));
                }
                const int ex = (int)(__float_as_uint(top) >> 23);
                const int e2 = top > 0.f && ex < 255 ? min(126, max(-126, 14 + 127 - max(ex, 1))) : 0;
                const float up = A.scale_m * __uint_as_float((uint32_t)(e2 + 127) << 23);
                q_factor[(items % RA_QBUF) * 128u + tid] = __uint_as_float((uint32_t)(min(127, max(-126, A.scale_e - e2)) + 127) << 23);
#pragma unroll 4
                for (int i = 0; i < HD; i += 8) {
                    const float4 x = load4(i), y = load4(i + 4);
                    uint4 hi, lo;
                    split2(x.x * up, x.y * up, hi.x, lo.x);
                    split2(x.z * up, x.w * up, hi.y, lo.y);
                    split2(y.x * up, y.y * up, hi.z, lo.z);
                    split2(y.z * up, y.w * up, hi.w, lo.w);
                    const uint32_t at = (uint32_t)(i / 64) * (128u * 128u) + tid * 128u + ((((uint32_t)i / 8u) & 7u) ^ (tid & 7u)) * 16u;
                    *reinterpret_cast<uint4 *>(q_smem + at) = hi;
                    *reinterpret_cast<uint4 *>(q_smem + S::QB + at) = lo;
                }
                items++;
                arrive(q_full);
            }
            const uint32_t tok = d.tile * RA_TT;
            const bool keep = tok + tr <= pos_hi && ((d.valid >> (mixed ? tr >> pshift : 0u)) & 1u);
            bool ok = true;
#pragma unroll 1
            for (int kv = 0; kv < 2; kv++) {
                if (kv && !(ok = wait(&land_full[NL + land], land_phase))) break;
                uint8_t *dst = op + (size_t)(kv * NS + st) * S::OPB;
                if constexpr (EL == 1) {
                    if (!(ok = wait(&op_empty[kv * NS + st], st_phase ^ 1u))) break;
                    const uint8_t *src = raw + (size_t)(kv * NL + land) * S::RAWB + tr * HD;
                    uint4 x[HD / 32];
#pragma unroll
                    for (int j = 0; j < HD / 32; j++) {
                        const uint32_t c = th * (HD / 32) + j;  // sixteen codes
                        x[j] = *reinterpret_cast<const uint4 *>(src + ((S::RAWSWZ ? c ^ (tr & 7u) : c) << 4));
                    }
                    if (kv && !keep) {
#pragma unroll
                        for (int j = 0; j < HD / 32; j++) x[j] = make_uint4(0u, 0u, 0u, 0u);
                    }
#pragma unroll
                    for (int j = 0; j < HD / 32; j++) {
                        const uint32_t c = th * (HD / 32) + j;
                        uint4 y, z;
                        e4m3x4_to_f16x2(x[j].x, y.x, y.y);
                        e4m3x4_to_f16x2(x[j].y, y.z, y.w);
                        e4m3x4_to_f16x2(x[j].z, z.x, z.y);
                        e4m3x4_to_f16x2(x[j].w, z.z, z.w);
                        uint8_t *row = dst + (c / 4u) * 8192u + tr * 128u;
                        const uint32_t w = (2u * c) & 7u;
                        *reinterpret_cast<uint4 *>(row + ((w ^ (tr & 7u)) << 4)) = y;
                        *reinterpret_cast<uint4 *>(row + (((w + 1u) ^ (tr & 7u)) << 4)) = z;
                    }
                    arrive(&op_full[kv * NS + st]);
                    if (lane == 0) mbar_arrive(&land_empty[kv * NL + land]);
                } else {
                    if (kv && !keep) {  // rows that nobody sees may hold anything
#pragma unroll
                        for (int j = 0; j < HD / 16; j++) {
                            const uint32_t c = th * (HD / 16) + j;
                            *reinterpret_cast<uint4 *>(dst + (c / 8u) * 8192u + tr * 128u + ((c & 7u) << 4)) = make_uint4(0u, 0u, 0u, 0u);
                        }
                    }
                    arrive(&op_full[kv * NS + st]);
                }
            }
            if (!ok) break;
            if (++land == NL) {
                land = 0;
                land_phase ^= 1u;
            }
            if (++st == NS) {
                st = 0;
                st_phase ^= 1u;
            }
        }
        join();
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
        if (warp == 16) {
            // ---- copies: the pages of the next 32 slots of the item to a lane each, one tile after the other
            uint32_t b_from = 0, b_stop = place.at, seg_stop = place.at, new_flag = 0, end_flag = 0, item = ~0u;
            int b_page = -1;
            float b_ks = 0.f, b_vs = 0.f;
            bool bad = false, started = false;
            const bool leader = elect_lane();
            const uint32_t sub_at = lane & (n_sub - 1u);
#pragma unroll 1
            for (uint32_t n = 0; n < n_tiles; n++) {
                const uint32_t land = n % NL, land_phase = (n / NL) & 1u;
                if (place.at == b_stop) {
                    if (place.at == seg_stop) {
                        if (started) next_item<RA_TT>(A, RA_ROWS, place);
                        started = true;
                        const uint32_t seg = min(n_tiles - n, place.tiles - place.at);
                        const bool ends = place.at + seg == place.tiles;
                        seg_stop = place.at + seg;
                        new_flag = PA_NEW;
                        item++;
                        end_flag = PA_END | (place.at ? PA_HEAD : ends ? PA_WHOLE : 0u);
                        if (lane == 0) {
                            const PaPart part{place.first, place.rows, place.mb * RA_ROWS, place.head, place.item0, place.tiles};
                            if (place.at) {
                                parts.front = part;
                                parts.has_front = 1u;
                            } else if (!ends) {
                                parts.back = part;
                                parts.has_back = 1u;
                            }
                        }
                    }
                    b_from = 0;
                    const uint32_t cnt = min(32u / n_sub, seg_stop - place.at);
                    b_stop = place.at + cnt;
                    const uint32_t tok = (place.lo_tile + place.at) * RA_TT + lane * sub, nth = tok >> pshift;
                    b_page = -1;
                    b_ks = b_vs = 0.f;
                    if (lane < cnt * n_sub && tok <= place.ctx + (place.rows - 1u) && nth < V.pages_ld &&
                        still_seen(A, RA_ROWS, place.ctx, place.mb, tok + sub - 1u)) {
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
                }
                const uint32_t tile = place.lo_tile + place.at;
                const int page = __shfl_sync(0xffffffffu, b_page, b_from + sub_at);
                const uint32_t valid = __ballot_sync(0xffffffffu, page >= 0) & ((1u << n_sub) - 1u);
                PaTile &d = desc[n % RA_DESCS];
                if (lane == 0) {
                    *reinterpret_cast<uint4 *>(&d.tile) = make_uint4(tile, item << PA_ITEM | new_flag | (place.at + 1u == seg_stop ? end_flag : 0u), valid, place.mb * RA_ROWS);
                    *reinterpret_cast<uint4 *>(&d.seq_first) = make_uint4(place.first, place.rows, place.ctx, place.head);
                }
                if (lane - b_from < n_sub) {
                    d.ks[lane - b_from] = b_ks;
                    d.vs[lane - b_from] = b_vs;
                }
                __syncwarp();
                bool ok = true;
#pragma unroll 1
                for (int kv = 0; kv < 2; kv++) {
                    uint64_t *bar = &land_full[kv * NL + land];
                    if (!(ok = wait(&land_empty[kv * NL + land], land_phase ^ 1u))) break;
                    if (leader) mbar_arrive_expect_tx(bar, __popc(valid) * sub * HD * EL);
                    __syncwarp();
                    uint8_t *dst = EL == 1 ? raw + (size_t)(kv * NL + land) * S::RAWB : op + (size_t)(kv * NS + land) * S::OPB;
#pragma unroll 1
                    for (uint32_t i = 0; i < n_sub; i++) {
                        const int pg = __shfl_sync(0xffffffffu, page, i);
                        const uint32_t y = place.head * V.page_tokens + ((tile * RA_TT + i * sub) & (V.page_tokens - 1u));
                        if (pg < 0 || !leader) continue;
                        if constexpr (EL == 1) {
                            tma_load_3d(dst + i * sub * HD, kv ? &A.v_map : &A.k_map, 0u, y, (uint32_t)pg, bar);
                        } else {
#pragma unroll
                            for (int x = 0; x < S::BLOCKS; x++) tma_load_3d(dst + x * 8192 + i * sub * 128, kv ? &A.v_map : &A.k_map, x * 64u, y, (uint32_t)pg, bar);
                        }
                    }
                }
                if (!ok) break;
                new_flag = 0u;
                b_from += n_sub;
                place.at++;
            }
            report_bad(V, bad);
        } else if (warp == 17) {
            // ---- products S, by one lane
            if (elect_lane()) {
                const uint32_t q_at = smem_u32(q_smem), op_at = smem_u32(op);
                constexpr uint32_t I_S = rows_idesc(RA_TT, false);
                uint64_t *k_free = EL == 1 ? op_empty : land_empty;
                const uint64_t q = desc_sw128(q_at, 16u);
                uint32_t items = 0, st = 0, phase = 0;
#pragma unroll 1
                for (uint32_t n = 0; n < n_tiles; n++) {
                    const uint32_t b = n & 1u;
                    if (!wait_lane(&op_full[st], phase)) break;
                    const uint32_t flags = desc[n % RA_DESCS].flags;
                    if (flags & PA_NEW && !wait_lane(q_full, items++ & 1u)) break;
                    if (!wait_lane(&s_empty[b], ((n >> 1) & 1u) ^ 1u)) break;
                    tc_fence_after();
                    const uint32_t d = tmem + b * 64u;
                    const uint64_t kk = desc_sw128(op_at + st * S::OPB, 16u);
#pragma unroll
                    for (uint32_t i = 0; i < 2u * S::BLOCKS; i++)  // the remainders first; 64 dimensions at a time
#pragma unroll
                        for (uint32_t k = 0; k < 4u; k++)
                            tc_mma_ss(d, q + (i < S::BLOCKS ? S::QB / 16u : 0u) + (i % S::BLOCKS) * (128u * 128u / 16u) + 2u * k,
                                      kk + (i % S::BLOCKS) * (8192u / 16u) + 2u * k, I_S, i + k);
                    tc_commit(&s_full[b]);
                    tc_commit(&k_free[st]);
                    if (flags & PA_END) tc_commit(q_empty);
                    if (++st == NS) {
                        st = 0;
                        phase ^= 1u;
                    }
                }
            }
        } else if (warp == 18) {
            // ---- products O, by one lane
            if (elect_lane()) {
                const uint32_t op_at = smem_u32(op);
                constexpr uint32_t I_O = rows_idesc(HD, true);
                uint64_t *v_free = EL == 1 ? op_empty + NS : land_empty + NL;
                uint32_t st = 0, phase = 0;
#pragma unroll 1
                for (uint32_t n = 0; n < n_tiles; n++) {
                    const uint32_t b = n & 1u;
                    if (!wait_lane(&op_full[NS + st], phase) || !wait_lane(&o_empty[b], ((n >> 1) & 1u) ^ 1u) || !wait_lane(&p_full[b], (n >> 1) & 1u)) break;
                    tc_fence_after();
                    const uint64_t v = desc_sw128(op_at + (NS + st) * S::OPB, 8192u);
                    const uint32_t d = tmem + S::COL_O + b * HD, p = tmem + S::COL_P + b * 64u;
#pragma unroll
                    for (int h = 0; h < 2; h++)  // the remainders first
#pragma unroll
                        for (int k = 0; k < 4; k++) tc_mma_ts(d, p + (h ? 0u : 32u) + 8u * k, v + (uint64_t)(k * 2048 / 16), I_O, h || k);
                    tc_commit(&o_full[b]);
                    tc_commit(&v_free[st]);
                    if (++st == NS) {
                        st = 0;
                        phase ^= 1u;
                    }
                }
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (gave_up) {  // copies may still be under way: they end before the block does
        if (threadIdx.x == 0 && V.status) atomicOr(V.status, STATUS_WAIT_TIMEOUT);
        for (int i = 0; i < 64; i++) __nanosleep(100000u);
    }
    if (warp == 17) {
        __syncwarp();
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
}

template <int HD, int TYPE>
static cudaError_t rows_launch(const strix_cuda *h, PagedAttnArgs &A, uint32_t blocks, cudaStream_t stream) {
    using S = RowsShape<HD, TYPE>;
    if (S::SMEM + 1024 > h->smem_optin) return cudaErrorInvalidConfiguration;
    const uint32_t sub = A.V.page_tokens < RA_TT ? A.V.page_tokens : RA_TT;
    const uint32_t box = S::EL == 1 ? (uint32_t)HD : 64u;
    const bool swz = S::EL == 2 || S::RAWSWZ;
    if (!attn_map(&A.k_map, A.V, A.V.k, box, sub, swz) || !attn_map(&A.v_map, A.V, A.V.v, box, sub, swz)) return cudaErrorInvalidValue;
    static std::atomic<uint64_t> ready{0};  // devices whose limit of dynamic shared memory is raised for this kernel
    const uint64_t bit = 1ull << (h->device & 63);
    if (!(ready.load(std::memory_order_relaxed) & bit)) {
        cudaFuncAttributes fa;
        const cudaError_t f = cudaFuncGetAttributes(&fa, attn_rows_kernel<HD, TYPE>);
        if (f != cudaSuccess) return f;
        if (fa.numRegs < 96) return cudaErrorInvalidConfiguration;  // the warps' shares (2 x 96, 176, 2 x 56) add up to five times that
        const cudaError_t e = cudaFuncSetAttribute(attn_rows_kernel<HD, TYPE>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)S::SMEM);
        if (e != cudaSuccess) return e;
        ready.fetch_or(bit, std::memory_order_relaxed);
    }
    attn_rows_kernel<HD, TYPE><<<blocks, RA_THREADS, S::SMEM, stream>>>(A);
    return cudaGetLastError();
}

cudaError_t launch_attn_rows(const strix_cuda *h, PagedAttnArgs &A, uint32_t blocks, cudaStream_t stream) {
    const bool f16 = A.V.type == STRIX_KV_F16;
    if (A.V.head_dim == 64) return f16 ? rows_launch<64, STRIX_KV_F16>(h, A, blocks, stream) : rows_launch<64, STRIX_KV_E4M3>(h, A, blocks, stream);
    return f16 ? rows_launch<128, STRIX_KV_F16>(h, A, blocks, stream) : rows_launch<128, STRIX_KV_E4M3>(h, A, blocks, stream);
}

}  // namespace strix
