// Appending to a paged KV cache: per-head RMS norm, position rotation, rounding to the cache's type, in one launch that also
// prepares q. Contract: include/strix_serve.h. The arithmetic follows qk_post_kernel (attention.cu), whose models it serves.
//
// What bounds it: a prompt is HBM traffic (4 bytes read for every element of q, k, v, 4 written for q, 1 or 2 for k and v);
// a decode step is one launch and a chain of four dependent loads (row0, ctx, page id, old scale).
// Measured (32 + 2 x 8 heads of 128): prompts of 8064 rows in all 85 us into e4m3 (4.1 TB/s), 78 into f16; 64 rows into f16 (16 + 2 x 8
// heads of 256) 5.9 us, one row 3.6 us.
//
// Work split. The cache side goes by pages, because a page and head share one scale: a block takes one (page, head) of k
// or v (four heads of it in turn, where sequences bring many rows), holds its new rows in registers, reduces their largest
// magnitude and stores codes. Which page a block has follows
// from a row: a unit is RU consecutive rows and owns the pages whose first new row lies among them. RU = page_tokens when
// sequences bring many rows (a block for each page), 1 when they bring few (a block for each row, most of them one-row pages).
// The q side has no scale to share: a warp takes one row and a few heads, so that the angles of a row are computed once
// for those heads.
//
// Angles: position * theta^(-2j/hd) / f_j in turns, in f64, reduced to [-1/2, 1/2] before it is rounded to f32 (an f32
// product is off by 6e-8 * position radians: 0.008 at position 131072). The rounding error of the f32 angle goes into
// sin and cos as a first-order correction.
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>
#include <string>

#include "kv_pages.cuh"

namespace strix {

struct AppendArgs {
    PagedView V;
    const float *src_k, *src_v, *src_q;
    float *dst_q;
    size_t ld_k, ld_v, ld_q, ld_qo;
    const float *k_norm, *q_norm, *freq;
    double turn[8];  // (theta^(-2/hd))^(2^b), b = 0..7; angles in turns start from 1 / (2 pi)
    float eps;
    int rope, norm_v;
    uint32_t n_heads, kv_blocks, unit_rows, kv_group, heads_per_warp, q_chunks, vec;  // vec: every f32 row starts on 16 bytes
};

// The lanes that share a row: HD / 2 pairs, four to a lane, in a power-of-two group of lanes.
template <int HD>
struct RowLanes {
    static constexpr int USED = HD / 8;                                // lanes with values
    static constexpr int GROUP = USED <= 8 ? 8 : USED <= 16 ? 16 : 32;
    static constexpr int ROWS = 32 / GROUP;                            // rows a warp treats at once
};

// Eight values of a head row in a lane: first[0..3] = elements at o0.., second[0..3] = elements at o1.. .
struct Eight {
    float a[4], b[4];
};

__device__ __forceinline__ void load_eight(Eight &x, const float *row, uint32_t o0, uint32_t o1, bool vec) {
    if (vec) {
        const float4 p = *reinterpret_cast<const float4 *>(row + o0), q = *reinterpret_cast<const float4 *>(row + o1);
        x.a[0] = p.x; x.a[1] = p.y; x.a[2] = p.z; x.a[3] = p.w;
        x.b[0] = q.x; x.b[1] = q.y; x.b[2] = q.z; x.b[3] = q.w;
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            x.a[i] = row[o0 + i];
            x.b[i] = row[o1 + i];
        }
    }
}

// 1 / rms over the row's lanes (all lanes of the warp call this; a lane without values passes zeros)
template <int HD>
__device__ __forceinline__ float inv_rms(const Eight &x, float eps) {
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < 4; i++) ss = fmaf(x.a[i], x.a[i], fmaf(x.b[i], x.b[i], ss));
#pragma unroll
    for (int o = RowLanes<HD>::GROUP / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    // (the approximate root and one step of Newton's: within 2^-23)
    const float s = ss * (1.0f / (float)HD) + eps, r = rsqrtf(s);
    return s > 0.f && s < 3.0e38f ? r * fmaf(-0.5f * s * r, r, 1.5f) : r;
}

struct Turn {
    float c[4], s[4];
};
__device__ __forceinline__ void turn_of(Turn &t, const double inv[4], uint32_t pos) {
#pragma unroll
    for (int p = 0; p < 4; p++) {
        double a = (double)pos * inv[p];
        a -= rint(a);
        const float f = (float)a, d = (float)(a - (double)f) * 6.283185307179586f;
        float s, c;
        sincospif(2.0f * f, &s, &c);
        t.s[p] = fmaf(c, d, s);
        t.c[p] = fmaf(-s, d, c);
    }
}
// pairs: (a[i], b[i]), or the neighbours (a0 a1) (a2 a3) (b0 b1) (b2 b3)
__device__ __forceinline__ void rotate(Eight &x, const Turn &t, int rope) {
    if (rope == STRIX_ROPE_HALVES) {
#pragma unroll
        for (int p = 0; p < 4; p++) {
            const float u = x.a[p], w = x.b[p];
            x.a[p] = u * t.c[p] - w * t.s[p];
            x.b[p] = u * t.s[p] + w * t.c[p];
        }
    } else if (rope == STRIX_ROPE_ADJACENT) {
#pragma unroll
        for (int p = 0; p < 2; p++) {
            float u = x.a[2 * p], w = x.a[2 * p + 1];
            x.a[2 * p] = u * t.c[p] - w * t.s[p];
            x.a[2 * p + 1] = u * t.s[p] + w * t.c[p];
            u = x.b[2 * p], w = x.b[2 * p + 1];
            x.b[2 * p] = u * t.c[p + 2] - w * t.s[p + 2];
            x.b[2 * p + 1] = u * t.s[p + 2] + w * t.c[p + 2];
        }
    }
}

__device__ __forceinline__ float storable(float x, float most) { return x != x ? 0.f : fminf(fmaxf(x, -most), most); }

// the least power of two s >= 2^-120 with amax <= 448 s (448 = 1.75 * 2^8)
__device__ __forceinline__ float scale_for(float amax) {
    const uint32_t u = __float_as_uint(amax);
    const int e = (int)(u >> 23) - 127 - ((u & 0x7fffffu) <= 0x600000u ? 8 : 7);
    return __uint_as_float((uint32_t)(max(e, -120) + 127) << 23);
}

template <int HD, int TYPE, int WARPS>
__global__ void __launch_bounds__(WARPS * 32) kv_append_kernel(const AppendArgs A) {
    using R = RowLanes<HD>;
    constexpr int MAXIT = WARPS >= 16 ? 128 / (16 * R::ROWS) : 2;  // row slots of a lane group held in registers
    constexpr uint32_t CHUNK = MAXIT * WARPS * R::ROWS;            // rows a block holds at once
    __shared__ float red[WARPS];
    const PagedView &V = A.V;
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
    const uint32_t l = lane % R::GROUP, sub = lane / R::GROUP;
    const bool on = l < R::USED;
    // element offsets of the lane's two quads; pair p of the lane is pair 4 l + p of the head
    const uint32_t o0 = A.rope == STRIX_ROPE_ADJACENT ? 8u * l : 4u * l;
    const uint32_t o1 = A.rope == STRIX_ROPE_ADJACENT ? 8u * l + 4u : HD / 2 + 4u * l;
    bool bad = false;
    double inv[4] = {0., 0., 0., 0.};
    auto frequencies = [&] {
        if (A.rope == STRIX_ROPE_NONE || !on) return;
        double f = 0.15915494309189535;  // 1 / (2 pi)
#pragma unroll
        for (int b = 0; b < 5; b++)
            if ((l >> b) & 1u) f *= A.turn[b + 2];
#pragma unroll
        for (int p = 0; p < 4; p++) {
            inv[p] = A.freq ? f / (double)A.freq[4u * l + p] : f;
            f *= A.turn[0];
        }
    };

    if (blockIdx.x >= A.kv_blocks) {  // ---- q: one row and heads_per_warp heads for each warp
        const uint32_t w = (blockIdx.x - A.kv_blocks) * WARPS + warp, row = w / A.q_chunks, chunk = w - row * A.q_chunks;
        if (row >= V.n_rows) return;
        constexpr int NB = WARPS >= 16 ? 4 : 1;  // heads of a lane group on their way at once: what is in flight bounds a prompt
        const uint32_t h1 = min(A.n_heads, (chunk + 1u) * A.heads_per_warp);
        const float *src = A.src_q + (size_t)row * A.ld_q;
        float *dst = A.dst_q + (size_t)row * A.ld_qo;
        Eight x[NB];
        auto fetch = [&](uint32_t h0) {
#pragma unroll
            for (int i = 0; i < NB; i++) {
                const uint32_t hh = h0 + i * R::ROWS + sub;
                x[i] = {};
                if (on && hh < h1) load_eight(x[i], src + hh * HD, o0, o1, A.vec);
            }
        };
        uint32_t h0 = chunk * A.heads_per_warp;
        fetch(h0);
        uint32_t first, end;
        const uint32_t s = seq_of_row(V, row, first, end, bad);
        report_bad(V, bad && lane == 0);
        if (s >= V.n_seq) return;
        const int ctx = V.ctx[s];
        if (ctx < 0) return;
        frequencies();
        Turn t;
        if (A.rope != STRIX_ROPE_NONE) turn_of(t, inv, (uint32_t)ctx + (row - first));
        Eight n = {};
        if (A.q_norm && on) load_eight(n, A.q_norm, o0, o1, false);
#pragma unroll 1
        for (;;) {
#pragma unroll
            for (int i = 0; i < NB; i++) {
                const uint32_t hh = h0 + i * R::ROWS + sub;
                Eight y = x[i];
                if (A.q_norm) {
                    const float r = inv_rms<HD>(y, A.eps);
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        y.a[e] = y.a[e] * r * n.a[e];
                        y.b[e] = y.b[e] * r * n.b[e];
                    }
                }
                rotate(y, t, A.rope);
                if (!(on && hh < h1)) continue;
                float *o = dst + hh * HD;
                if (A.vec) {
                    *reinterpret_cast<float4 *>(o + o0) = make_float4(y.a[0], y.a[1], y.a[2], y.a[3]);
                    *reinterpret_cast<float4 *>(o + o1) = make_float4(y.b[0], y.b[1], y.b[2], y.b[3]);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        o[o0 + e] = y.a[e];
                        o[o1 + e] = y.b[e];
                    }
                }
            }
            h0 += NB * R::ROWS;
            if (h0 >= h1) return;
            fetch(h0);
        }
    }

    // ---- k or v: the pages whose first new row lies in this unit, kv_group heads one after the other
    const uint32_t groups = (V.n_kv + A.kv_group - 1u) / A.kv_group;
    const uint32_t per = 2u * groups, unit = blockIdx.x / per, which = blockIdx.x - unit * per;
    const bool is_v = which >= groups;
    const uint32_t g0 = (is_v ? which - groups : which) * A.kv_group, g1 = min(V.n_kv, g0 + A.kv_group);
    constexpr bool KEEP = MAXIT <= 4;  // the rows' sines and cosines stay in registers from head to head
    const size_t ld = is_v ? A.ld_v : A.ld_k;
    uint8_t *cache = is_v ? V.v : V.k;
    float *scales = is_v ? V.v_scale : V.k_scale;
    const float *nw = is_v ? nullptr : A.k_norm;
    const bool norm = is_v ? A.norm_v != 0 : nw != nullptr;
    const int rope = is_v ? STRIX_ROPE_NONE : A.rope;
    const float most = TYPE == STRIX_KV_F16 ? 65504.f : 3.0e38f;
    if (!is_v) frequencies();
    float w8[8] = {1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f};
    if (nw && on) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            w8[i] = nw[o0 + i];
            w8[4 + i] = nw[o1 + i];
        }
    }
    uint32_t row = unit * A.unit_rows;
    const uint32_t unit_end = min(V.n_rows, row + A.unit_rows);
#pragma unroll 1
    while (row < unit_end) {
        uint32_t first, end;
        const uint32_t s = seq_of_row(V, row, first, end, bad);
        if (s >= V.n_seq) {  // rows of nobody: with ascending offsets only those behind the last sequence
            row++;
            continue;
        }
        const int ctx = V.ctx[s];
        if (ctx < 0) {
            row = end;
            continue;
        }
        const uint64_t pos = (uint64_t)(uint32_t)ctx + (row - first);
        const uint32_t slot = (uint32_t)pos & (V.page_tokens - 1u);
        const uint32_t cnt = min(V.page_tokens - slot, end - row);  // rows from here to the end of the page
        if (row != first && slot != 0u) {                           // the page began in an earlier unit, which has it
            row += cnt;
            continue;
        }
        const uint64_t nth = pos >> V.page_shift;
        const int page = nth < V.pages_ld ? V.pages[(size_t)s * V.pages_ld + nth] : -1;
        if (page < 0 || (uint32_t)page >= V.n_pages) {
            bad = true;
            row += cnt;
            continue;
        }
        Turn turns[KEEP ? MAXIT : 1];
#pragma unroll 1
        for (uint32_t hh = g0; hh < g1; hh++) {
        const float *src = (is_v ? A.src_v : A.src_k) + (size_t)hh * HD;
        uint8_t *dst = cache + (size_t)page * V.page_bytes + (size_t)hh * V.head_bytes;
        float *scale = TYPE == STRIX_KV_E4M3 ? scales + (size_t)page * V.n_kv + hh : nullptr;
        const float s_old = TYPE == STRIX_KV_E4M3 && slot ? *scale : 0.f;

        Eight x[MAXIT];
        auto fetch = [&](uint32_t base) {  // rows base .. base + CHUNK - 1 of the page's new rows into registers
            float m = 0.f;
#pragma unroll
            for (int it = 0; it < MAXIT; it++) {  // all on their way before the first is used
                const uint32_t i = base + it * (WARPS * R::ROWS) + warp * R::ROWS + sub;
                x[it] = {};
                if (on && i < cnt) load_eight(x[it], src + (size_t)(row + i) * ld, o0, o1, A.vec);
            }
#pragma unroll
            for (int it = 0; it < MAXIT; it++) {
                const uint32_t i = base + it * (WARPS * R::ROWS) + warp * R::ROWS + sub;
                if (base + it * (WARPS * R::ROWS) + warp * R::ROWS >= cnt) break;  // (the same for the whole warp)
                if (norm) {
                    const float r = inv_rms<HD>(x[it], A.eps);
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        x[it].a[e] = x[it].a[e] * r * w8[e];
                        x[it].b[e] = x[it].b[e] * r * w8[4 + e];
                    }
                }
                if (rope != STRIX_ROPE_NONE) {
                    Turn &t = turns[KEEP ? it : 0];
                    if (!KEEP || hh == g0 || cnt > CHUNK) turn_of(t, inv, (uint32_t)pos + i);
                    rotate(x[it], t, rope);
                }
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    x[it].a[e] = storable(x[it].a[e], most);
                    x[it].b[e] = storable(x[it].b[e], most);
                    m = fmaxf(m, fmaxf(fabsf(x[it].a[e]), fabsf(x[it].b[e])));
                }
            }
            return m;
        };
        auto store = [&](uint32_t base, float inv_s) {
#pragma unroll
            for (int it = 0; it < MAXIT; it++) {
                const uint32_t i = base + it * (WARPS * R::ROWS) + warp * R::ROWS + sub;
                if (!on || i >= cnt) continue;
                const Eight &y = x[it];
                if (TYPE == STRIX_KV_E4M3) {
                    uint8_t *o = dst + (size_t)(slot + i) * HD;
                    *reinterpret_cast<uint32_t *>(o + o0) =
                        f32_to_e4m3x2(y.a[0] * inv_s, y.a[1] * inv_s) | f32_to_e4m3x2(y.a[2] * inv_s, y.a[3] * inv_s) << 16;
                    *reinterpret_cast<uint32_t *>(o + o1) =
                        f32_to_e4m3x2(y.b[0] * inv_s, y.b[1] * inv_s) | f32_to_e4m3x2(y.b[2] * inv_s, y.b[3] * inv_s) << 16;
                } else {
                    __half *o = reinterpret_cast<__half *>(dst) + (size_t)(slot + i) * HD;
                    *reinterpret_cast<uint2 *>(o + o0) = make_uint2(f32_to_f16x2(y.a[0], y.a[1]), f32_to_f16x2(y.a[2], y.a[3]));
                    *reinterpret_cast<uint2 *>(o + o1) = make_uint2(f32_to_f16x2(y.b[0], y.b[1]), f32_to_f16x2(y.b[2], y.b[3]));
                }
            }
        };
        if (TYPE == STRIX_KV_F16) {
#pragma unroll 1
            for (uint32_t base = 0; base < cnt; base += CHUNK) {
                fetch(base);
                store(base, 1.f);
            }
        } else {
            float m = 0.f;
            uint32_t base = 0;
#pragma unroll 1
            for (;; base += CHUNK) {  // the last chunk stays in registers
                m = fmaxf(m, fetch(base));
                if (base + CHUNK >= cnt) break;
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
            if (lane == 0) red[warp] = m;
            __syncthreads();  // (every thread has read the old scale by now, too)
            m = red[0];
#pragma unroll
            for (int w = 1; w < WARPS; w++) m = fmaxf(m, red[w]);
            const float need = scale_for(m), s_new = s_old > need ? s_old : need, inv_s = 1.0f / s_new;
            if (threadIdx.x == 0) *scale = s_new;
            if (slot && s_new != s_old) {  // the page's other codes move to the new scale
                const float f = s_old * inv_s;
                uint4 *old = reinterpret_cast<uint4 *>(dst);
#pragma unroll 1
                for (uint32_t i = threadIdx.x; i < V.page_tokens * (HD / 16); i += WARPS * 32) {
                    if (i / (HD / 16) - slot < cnt) continue;  // (unsigned: slots from `slot` on, cnt of them, are the new rows')
                    uint4 u = old[i];
                    uint32_t *p = &u.x;
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const float2 lo = e4m3x2_to_f32(p[e] & 0xffffu), hi = e4m3x2_to_f32(p[e] >> 16);
                        p[e] = f32_to_e4m3x2(lo.x * f, lo.y * f) | f32_to_e4m3x2(hi.x * f, hi.y * f) << 16;
                    }
                    old[i] = u;
                }
            }
            store(base, inv_s);
#pragma unroll 1
            while (base > 0u) {  // earlier chunks are prepared once more
                base -= CHUNK;
                fetch(base);
                store(base, inv_s);
            }
            __syncthreads();  // `red` is free for the next head or page
        }
        }
        row += cnt;
    }
    // offsets out of range or going down, whether or not a row leads to them: each sequence is looked at by one thread of the grid
#pragma unroll 1
    for (uint64_t s = (uint64_t)blockIdx.x * (WARPS * 32u) + threadIdx.x; s < V.n_seq; s += (uint64_t)A.kv_blocks * (WARPS * 32u)) {  // (may pass 32 bits)
        uint32_t first, end;
        seq_rows(V, (uint32_t)s, first, end, bad);
    }
    report_bad(V, bad);
}

template <int HD, int TYPE>
static cudaError_t append_launch(const AppendArgs &A, bool by_page, uint32_t q_blocks, cudaStream_t stream) {
    const uint32_t grid = A.kv_blocks + q_blocks;
    if (grid == 0) return cudaSuccess;
    if (by_page)
        kv_append_kernel<HD, TYPE, 16><<<grid, 512, 0, stream>>>(A);
    else
        kv_append_kernel<HD, TYPE, 4><<<grid, 128, 0, stream>>>(A);
    return cudaGetLastError();
}

int serve_fail(strix_cuda *h, const char *what, const char *why) noexcept {
    try {
        h->err = std::string(what) + ": " + why;
    } catch (...) {
    }
    return -1;
}

// 1 and a filled view, 0 = declined, -1 = an argument error and its text in *why
static int kv_view(const strix_kv_pages *c, const strix_kv_batch *b, PagedView &r, const char **why) noexcept {
    auto no = [&](const char *text) {
        *why = text;
        return -1;
    };
    if (!c) return no("cache missing");
    if (c->type != STRIX_KV_F16 && c->type != STRIX_KV_E4M3) return no("unknown cache type");
    const uint32_t P = c->page_tokens, hd = c->head_dim;
    if (P != 16 && P != 32 && P != 64 && P != 128) return 0;
    if (hd != 64 && hd != 96 && hd != 128 && hd != 192 && hd != 256) return 0;
    if (c->n_kv == 0 || c->n_kv > 65535u) return 0;
    if (c->n_pages == 0 || c->n_pages > 0x7fffffffu) return no("n_pages out of range");
    const size_t el = c->type == STRIX_KV_F16 ? 2 : 1, head = (size_t)P * hd, packed = head * c->n_kv;
    const size_t stride = c->page_stride ? c->page_stride : packed;
    if (stride < packed) return no("page_stride smaller than a page");
    if (stride > ((size_t)1 << 32)) return no("page_stride out of range");
    if (!c->k || !c->v || (c->type == STRIX_KV_E4M3 && (!c->d_k_scale || !c->d_v_scale))) return no("a cache buffer is missing");
    if ((reinterpret_cast<uintptr_t>(c->k) | reinterpret_cast<uintptr_t>(c->v) | (stride * el)) & 15u)
        return no("k, v and page_stride must be 16-byte aligned");
    r = PagedView{};
    r.k = static_cast<uint8_t *>(c->k);
    r.v = static_cast<uint8_t *>(c->v);
    r.k_scale = c->d_k_scale;
    r.v_scale = c->d_v_scale;
    r.page_bytes = stride * el;
    r.head_bytes = head * el;
    r.n_pages = c->n_pages;
    r.n_kv = c->n_kv;
    r.page_tokens = P;
    r.page_shift = P == 16 ? 4u : P == 32 ? 5u : P == 64 ? 6u : 7u;
    r.head_dim = hd;
    r.type = c->type;
    if (!b) return 1;
    if (b->n_seq > 0x7fffffu || b->n_rows > 0x7fffffffu || b->pages_ld > 0x7fffffu) return no("batch sizes out of range");
    if (b->n_seq && (!b->d_row0 || !b->d_ctx || (b->pages_ld && !b->d_pages))) return no("a batch array is missing");
    r.row0 = b->d_row0;
    r.ctx = b->d_ctx;
    r.pages = b->d_pages;
    r.n_seq = b->n_seq;
    r.n_rows = b->n_rows;
    r.pages_ld = b->pages_ld;
    return 1;
}

int serve_check(strix_cuda *h, const char *what, const strix_kv_pages *c, const strix_kv_batch *b, PagedView *v) noexcept {
    if (!b) return serve_fail(h, what, "batch missing");
    const char *why = "";
    const int rc = kv_view(c, b, *v, &why);
    v->status = h->d_status + 1;
    return rc < 0 ? serve_fail(h, what, why) : rc;
}

}  // namespace strix

using namespace strix;

extern "C" int strix_cuda_kv_check(const strix_kv_pages *cache, const strix_kv_batch *batch, uint32_t n_heads) {
    PagedView v;
    const char *why;
    const int rc = kv_view(cache, batch, v, &why);
    if (rc != 1 || n_heads == 0) return rc;
    return n_heads <= 65535u && n_heads % v.n_kv == 0 ? 1 : 0;
}

extern "C" int strix_cuda_kv_append_dev(strix_cuda *h, const strix_kv_pages *cache, const strix_kv_batch *batch, const strix_kv_prep *prep,
                                        uint32_t n_heads, const float *d_k, size_t ld_k, const float *d_v, size_t ld_v,
                                        const float *d_q, size_t ld_q, float *d_q_out, size_t ld_q_out, void *stream) {
    if (!h) return -1;
    h->err.clear();
    AppendArgs A{};
    const char *who = "kv_append";
    const int rc = serve_check(h, who, cache, batch, &A.V);
    if (rc != 1) return rc;
    if (!prep) return serve_fail(h, who, "prep missing");
    if (prep->rope != STRIX_ROPE_NONE && prep->rope != STRIX_ROPE_HALVES && prep->rope != STRIX_ROPE_ADJACENT)
        return serve_fail(h, who, "unknown rope");
    if (prep->rope != STRIX_ROPE_NONE && !(prep->theta > 0.f && prep->theta <= 3.4028235e38f)) return serve_fail(h, who, "theta must be positive and finite");
    if (!(prep->eps >= 0.f)) return serve_fail(h, who, "eps must not be negative");
    if (!d_q != !d_q_out) return serve_fail(h, who, "d_q and d_q_out go together");
    if (d_q && (n_heads == 0 || n_heads > 65535u)) return serve_fail(h, who, "n_heads out of range");
    const size_t kvd = (size_t)A.V.n_kv * A.V.head_dim, qd = (size_t)n_heads * A.V.head_dim;
    A.ld_k = ld_k ? ld_k : kvd;
    A.ld_v = ld_v ? ld_v : kvd;
    A.ld_q = ld_q ? ld_q : qd;
    A.ld_qo = ld_q_out ? ld_q_out : qd;
    if (A.ld_k < kvd || A.ld_v < kvd || (d_q && (A.ld_q < qd || A.ld_qo < qd))) return serve_fail(h, who, "a row stride is smaller than a row");
    if (d_q && d_q == d_q_out && A.ld_q != A.ld_qo) return serve_fail(h, who, "in place, ld_q and ld_q_out must be equal");
    if (A.V.n_seq == 0 || A.V.n_rows == 0) return 1;
    if (!d_k || !d_v) return serve_fail(h, who, "d_k or d_v missing");
    A.src_k = d_k;
    A.src_v = d_v;
    A.src_q = d_q;
    A.dst_q = d_q_out;
    A.k_norm = prep->d_k_norm;
    A.q_norm = prep->d_q_norm;
    A.freq = prep->d_freq;
    A.eps = prep->eps;
    A.rope = prep->rope;
    A.norm_v = prep->norm_v;
    A.n_heads = d_q ? n_heads : 0u;
    if (prep->rope != STRIX_ROPE_NONE) {
        A.turn[0] = pow((double)prep->theta, -2.0 / (double)A.V.head_dim);
#pragma unroll 1
        for (int b = 1; b < 8; b++) A.turn[b] = A.turn[b - 1] * A.turn[b - 1];
    }
    A.vec = ((reinterpret_cast<uintptr_t>(d_k) | reinterpret_cast<uintptr_t>(d_v) | reinterpret_cast<uintptr_t>(d_q) |
              reinterpret_cast<uintptr_t>(d_q_out)) & 15u) == 0 &&
            ((A.ld_k | A.ld_v | (d_q ? A.ld_q | A.ld_qo : 0)) & 3u) == 0;
    const uint64_t n_rows = A.V.n_rows;
    // A unit of a page's rows, or of one row, by the rows that a sequence brings on average. Both measured (us, a page's and a row's, f16 and
    // e4m3, 64-token pages, 32 + 2 x 8 heads of 128):
    //   64 sequences of 1 row 269 and 5.7, 375 and 7.0; of 4: 74 and 13, 102 and 14; of 8: 41 and 22, 55 and 23; of 12: 33 and 32, 45 and 32;
    //   of 16: 28 and 41, 39 and 41; of 64: 50 and 157, 58 and 161.  8 sequences of 8: 35 and 4.9, 48 and 5.3; of 32: 20 and 11, 27 and 13;
    //   of 64: 14 and 20, 18 and 23.  1 of 16: 6.9 and 3.7, 8.5 and 4.3; of 256: 14 and 11, 18 and 15; of 2048: 22 and 63, 23 and 66.
    // So with few sequences a row's unit would still be the better one for some hundred rows. One form serves a call: 512 rows of a prompt
    // beside 60 single rows, whose pages then fall to one unit, take 361 us, in two calls 18.5.
    const bool by_page = n_rows > 8ull * A.V.n_seq;
    A.unit_rows = by_page ? A.V.page_tokens : 1u;
    A.kv_group = by_page ? 4u : 1u;
    const uint64_t kvb = (n_rows + A.unit_rows - 1) / A.unit_rows * 2ull * ((A.V.n_kv + A.kv_group - 1) / A.kv_group);
    const uint32_t hd = A.V.head_dim, rows_at_once = hd == 64 ? 4u : hd <= 128 ? 2u : 1u, warps = by_page ? 16u : 4u;
    uint64_t qb = 0;
    if (d_q) {
        A.heads_per_warp = rows_at_once * (by_page ? 8u : 1u);
        A.q_chunks = (n_heads + A.heads_per_warp - 1) / A.heads_per_warp;
        qb = (n_rows * A.q_chunks + warps - 1) / warps;
    }
    if (kvb + qb > 0x7fffffffull) return serve_fail(h, who, "batch too large for one launch");
    A.kv_blocks = (uint32_t)kvb;
    DeviceGuard dev(h->device);
    if (dev.err != cudaSuccess) return serve_fail(h, who, cudaGetErrorString(dev.err));
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    cudaError_t e = cudaErrorInvalidValue;
    {
        ProfScope prof(h, s, "kv_append");
        const bool f16 = A.V.type == STRIX_KV_F16;
#define STRIX_APPEND(HD) \
    case HD: e = f16 ? append_launch<HD, STRIX_KV_F16>(A, by_page, (uint32_t)qb, s) : append_launch<HD, STRIX_KV_E4M3>(A, by_page, (uint32_t)qb, s); break;
        switch (hd) {
            STRIX_APPEND(64)
            STRIX_APPEND(96)
            STRIX_APPEND(128)
            STRIX_APPEND(192)
            STRIX_APPEND(256)
        }
#undef STRIX_APPEND
    }
    if (e != cudaSuccess) return serve_fail(h, who, cudaGetErrorString(e));
    return 1;
}
