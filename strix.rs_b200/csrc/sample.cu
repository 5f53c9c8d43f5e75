// Drawing a token from logits: temperature, top-k, top-p, min-p and the inverse of the distribution function at a given
// number. Contract: include/strix_serve.h. Stands beside the greedy argmax (argmax.cu).
//
// A row lives in the shared memory of a cluster of blocks, so the logits are read from HBM once and every question about them
// is a pass over on-chip data: what bounds a draw is the number of passes and cluster barriers (half a microsecond to a microsecond
// each), not the 4 bytes a logit. (Reading the logits from L2 in every pass, so that more rows run at once, was slower: 58 against
// 52 us at 64 rows of 151936, 60 against 45 at 16 of 262147.)
//
// Nothing as long as the row is sorted. What top-k and top-p keep is, in the order (logit, lower index first), everything down to
// one cut (key, index). The cut is found from a histogram of log2 weight (y = (x - max) log2(e) / T; 2048 bins over the 16
// binary orders below the maximum, which few tokens reach and where most cuts lie; over all 41 that a weight in steps of 2^-40
// can have if the cut is not among those; logits below have no weight and no part in anything):
//   top-k: the bin in which the count passes k;
//   top-p: a bin's mass is its count times its middle weight to within half a bin, so the counts bound where the mass passes
//          top_p of the sum over all, which the same pass takes: mostly a few bins.
// If all that the cut may leave is at most SAMPLE_CAP tokens, they are gathered in one block, sorted and the draw ends there.
// Otherwise the uncertain bins alone are resolved: exact masses on 2048 finer bins, then the tokens of one of those are
// sorted, or, where they are too many (logits that came from 16 bits have thousands of equal values), the cut is bisected
// over their keys. The draw itself is a sum over the row in index order.
// Weights are summed as 64-bit integers in steps of 2^-40 (the sum over all as f32 within a thread's stretch, whose order is
// fixed), so no sum depends on the order of atomics, and neither does the draw.
//
// Measured: one row of 151936 12.8-18 us, 64 of them with mixed parameters 44-62 us, 16 rows of 262147 with top-p over most of their mass
// 30-60 us, depending on where the cuts fall (three inputs each). 33 clusters of eight such blocks run at a time, so 64 rows go in two waves.
//
// A weight is ex2 of an f32 exponent, so it is off by about 2^-22 (1 + |x - max| / T) of itself.
#include <cooperative_groups.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <atomic>

#include "kv_pages.cuh"

namespace cg = cooperative_groups;

namespace strix {

typedef unsigned long long u64;

constexpr int SAMPLE_THREADS = 512, SAMPLE_WARPS = SAMPLE_THREADS / 32;
constexpr uint32_t SAMPLE_BINS = 2048, SAMPLE_CAP = 2048;
constexpr int SAMPLE_BPT = SAMPLE_BINS / SAMPLE_THREADS;  // bins, or list entries, of a thread
constexpr float SAMPLE_ORDERS = 41.f;       // weights below 2^-41 round to no step of 2^-40
constexpr float SAMPLE_NEAR = 16.f;         // binary orders of the first histogram

struct SampleArgs {
    const float *x;
    size_t stride;
    uint32_t n, per;  // logits of a row, of a block (a multiple of 4)
    strix_sample_params p;
    const float *u;
    uint32_t *ids;
    float *probs;
};

// Unsigned keys in the order of the logits (no NaN here: they become -inf on their way into shared memory); -0 equals +0.
__device__ __forceinline__ uint32_t logit_key(float x) {
    const uint32_t b = __float_as_uint(x + 0.f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float ex2(float y) {
    float w;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(w) : "f"(y));
    return w;
}
__device__ __forceinline__ float key_logit(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

struct SampleShared {
    uint32_t hist[SAMPLE_BINS / 2];  // two counts to a word: a block has fewer than 2^16 logits
    union {
        struct {
            u64 mass[SAMPLE_BINS];
            uint32_t count[SAMPLE_BINS];
        } fine;
        struct {
            u64 e[SAMPLE_CAP];      // entries to sort, the smallest first
            u64 sorted[SAMPLE_CAP / 2];
        } list;
    };
    u64 ws[2][2][SAMPLE_WARPS];     // sums of the warps, in turns
    float wf[SAMPLE_WARPS];
    u64 xch[2][2];                  // what the cluster's blocks tell each other, in turns
    uint32_t n_list, first, second, fmax, rank[256];
    u64 found[2];
};
static_assert(sizeof(SampleShared) % 16 == 0, "the logits behind it are read in 16-byte words");

struct OpAdd {
    __device__ u64 operator()(u64 p, u64 q) const { return p + q; }
};
struct OpMin {
    __device__ u64 operator()(u64 p, u64 q) const { return p < q ? p : q; }
};
struct OpMax {
    __device__ u64 operator()(u64 p, u64 q) const { return p > q ? p : q; }
};

// A block's logits in shared memory, padded with -inf to a multiple of four; no NaN among them.
struct Logits {
    const float *p;
    uint32_t cnt;
    __device__ float operator[](uint32_t i) const { return p[i]; }
    // f(logit, its place) for those in [i0, i1) (i0 a multiple of four) that fall to this one of `takers`, in words of four
    template <typename F>
    __device__ __forceinline__ void each(uint32_t i0, uint32_t i1, uint32_t taker, uint32_t takers, F f) const {
#pragma unroll 4
        for (uint32_t i = i0 + 4u * taker; i < i1; i += 4u * takers) {
            const float4 v = *reinterpret_cast<const float4 *>(p + i);
            f(v.x, i);
            f(v.y, i + 1u);
            f(v.z, i + 2u);
            f(v.w, i + 3u);
        }
    }
    template <typename F>
    __device__ __forceinline__ void each(F f) const { each(0u, cnt, threadIdx.x, SAMPLE_THREADS, f); }
};

// One block's view of its row, which C blocks share. Two rules keep the cluster together: what a block shows to the others
// (hist, fine, list, xch, found, fmax) is not written again before a cluster barrier behind their reads, and every branch
// that a barrier depends on is taken on values that all blocks compute from the same data in the same order.
template <int C>
struct SampleRow {
    SampleShared &S;
    const Logits xs;                // this block's
    uint32_t base;                  // index of the first
    float m, c, cb;                 // maximum; log2(e) / T; bins to a unit of logit
    uint32_t turn, wturn;

    __device__ static uint32_t me() { return C > 1 ? cg::this_cluster().block_rank() : 0u; }
    __device__ static void csync() {
        if constexpr (C > 1) cg::this_cluster().sync();
        else __syncthreads();
    }
    template <typename T>
    __device__ static T far(const T *p, uint32_t r) {
        if constexpr (C > 1) return *cg::this_cluster().map_shared_rank(p, r);
        else return *p;
    }
    // log2 of a weight, below -SAMPLE_ORDERS where there is none (NaN for -inf at an infinite temperature: no weight either)
    __device__ float order(float x) const { return (x - m) * c; }
    __device__ void bins_over(float orders) { cb = c * (SAMPLE_BINS / orders); }
    __device__ static bool weighs(float y) { return y >= -SAMPLE_ORDERS; }
    // the weight in steps of 2^-40 (rounded to nearest), as units of 2^20 and the rest
    __device__ static void split(float y, uint32_t &hi, uint32_t &lo) {
        const float w = ex2(y) * 1048576.f, h = __fadd_rd(w, 8388608.f);
        hi = __float_as_uint(h) & 0x7fffffu;
        lo = __float_as_uint(fmaf(w - (h - 8388608.f), 1048576.f, 8388608.f)) & 0x7fffffu;
    }
    __device__ static u64 steps(float y) {
        if (!weighs(y)) return 0ull;
        uint32_t hi, lo;
        split(y, hi, lo);
        return ((u64)hi << 20) + lo;
    }
    // place in the histogram, a number below SAMPLE_BINS where there is weight (the product is rounded by itself: whoever asks for a
    // token's bin, or subtracts from this, gets the same number)
    __device__ float bin_of(float x) const { return __fmul_rn(m - x, cb); }
    __device__ static uint32_t bin(float b) { return __float_as_uint(__fadd_rd(b, 8388608.f)) & 0x7fffffu; }

    // folds up to two values over the cluster
    template <int N, typename F>
    __device__ void fold(u64 (&v)[N], F op) {
        u64(&ws)[2][SAMPLE_WARPS] = S.ws[wturn];
        wturn ^= 1u;
        const uint32_t lane = threadIdx.x & 31u;
#pragma unroll
        for (int k = 0; k < N; k++) {
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) v[k] = op(v[k], __shfl_xor_sync(0xffffffffu, v[k], o));
            if (lane == 0) ws[k][threadIdx.x >> 5] = v[k];
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < N; k++) {
            v[k] = ws[k][lane & (SAMPLE_WARPS - 1)];
#pragma unroll
            for (int o = SAMPLE_WARPS / 2; o > 0; o >>= 1) v[k] = op(v[k], __shfl_xor_sync(0xffffffffu, v[k], o));
            if (C > 1 && threadIdx.x == 0) S.xch[turn][k] = v[k];
        }
        if constexpr (C > 1) {
            csync();
#pragma unroll
            for (int k = 0; k < N; k++) {
                v[k] = far(&S.xch[turn][k], lane & (C - 1));
#pragma unroll
                for (int o = C / 2; o > 0; o >>= 1) v[k] = op(v[k], __shfl_xor_sync(0xffffffffu, v[k], o));
            }
            turn ^= 1u;
        }
    }
    __device__ u64 sum(u64 v) {
        u64 a[1] = {v};
        fold(a, OpAdd());
        return a[0];
    }
    // the sum over the block's threads before this one, and over all
    __device__ u64 before(u64 v, u64 &all) {
        u64 *ws = S.ws[wturn][0];
        wturn ^= 1u;
        const uint32_t lane = threadIdx.x & 31u, w = threadIdx.x >> 5;
        u64 incl = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const u64 p = __shfl_up_sync(0xffffffffu, incl, o);
            if ((int)lane >= o) incl += p;
        }
        if (lane == 31u) ws[w] = incl;
        __syncthreads();
        const u64 mine = ws[lane & (SAMPLE_WARPS - 1)];
        u64 wi = mine;
#pragma unroll
        for (int o = 1; o < SAMPLE_WARPS; o <<= 1) {
            const u64 p = __shfl_up_sync(0xffffffffu, wi, o);
            if ((int)(lane & (SAMPLE_WARPS - 1)) >= o) wi += p;
        }
        all = __shfl_sync(0xffffffffu, wi, SAMPLE_WARPS - 1);
        return __shfl_sync(0xffffffffu, wi - mine, w) + incl - v;
    }
    // the same over the cluster, blocks in rank order
    __device__ u64 before_all(u64 v, u64 &all) {
        u64 mine;
        u64 b = before(v, mine);
        if constexpr (C > 1) {
            if (threadIdx.x == 0) S.xch[turn][0] = mine;
            csync();
            const uint32_t lane = threadIdx.x & 31u, r = me();
            const u64 w = lane < C ? far(&S.xch[turn][0], lane & (C - 1)) : 0ull;
            u64 a = w, l = lane < r ? w : 0ull;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) {
                a += __shfl_xor_sync(0xffffffffu, a, o);
                l += __shfl_xor_sync(0xffffffffu, l, o);
            }
            all = a;
            b += l;
            turn ^= 1u;
        } else {
            all = mine;
        }
        return b;
    }

    // S.list.e[0 .. n) in ascending order (n <= SAMPLE_CAP), by this block
    __device__ void sort_list(uint32_t n) {
        const uint32_t t = threadIdx.x;
        if (n <= 256u) {  // by rank: every entry counts the smaller ones, SAMPLE_THREADS / np threads to an entry
            uint32_t np = 32;
#pragma unroll 1
            while (np < n) np *= 2;
            if (t < 256u) S.rank[t] = 0u;
            __syncthreads();
            const uint32_t e = t & (np - 1u), part = t / np, parts = SAMPLE_THREADS / np;
            if (e < n) {
                const u64 mine = S.list.e[e];
                uint32_t less = 0;
#pragma unroll 1
                for (uint32_t j = part; j < n; j += parts) less += S.list.e[j] < mine || (S.list.e[j] == mine && j < e);
                if (less) atomicAdd(&S.rank[e], less);
            }
            __syncthreads();
            if (t < n) S.list.sorted[S.rank[t]] = S.list.e[t];
            __syncthreads();
            if (t < n) S.list.e[t] = S.list.sorted[t];
            __syncthreads();
            return;
        }
        uint32_t np = 512;  // bitonic
#pragma unroll 1
        while (np < n) np *= 2;
#pragma unroll 1
        for (uint32_t i = n + t; i < np; i += SAMPLE_THREADS) S.list.e[i] = ~0ull;
        __syncthreads();
#pragma unroll 1
        for (uint32_t k = 2; k <= np; k *= 2)
#pragma unroll 1
            for (uint32_t j = k / 2; j > 0; j /= 2) {
#pragma unroll 1
                for (uint32_t h = t; h < np / 2; h += SAMPLE_THREADS) {
                    const uint32_t a = 2 * h - (h & (j - 1u)), b = a + j;
                    const u64 p = S.list.e[a], q = S.list.e[b];
                    if ((p > q) == ((a & k) == 0u)) {
                        S.list.e[a] = q;
                        S.list.e[b] = p;
                    }
                }
                __syncthreads();
            }
    }
    // Puts the tokens that `want` names into this block's list (descending key, index), ends behind a cluster barrier, and
    // brings the other blocks' lists into rank 0's. Returns how many there are (to rank 0 only).
    template <typename F>
    __device__ uint32_t gather(F want) {
        xs.each([&](float x, uint32_t i) {
            if (!want(x, base + i)) return;
            const uint32_t at = atomicAdd(&S.n_list, 1u);
            if (at < SAMPLE_CAP) S.list.e[at] = (u64)(~logit_key(x)) << 32 | (base + i);
        });
        csync();
        uint32_t n = min(S.n_list, SAMPLE_CAP);
        if constexpr (C > 1) {
            if (me() == 0) {
                const uint32_t lane = threadIdx.x & 31u, w = threadIdx.x >> 5, r = w & (C - 1), part = w / C;
                const uint32_t k = far(&S.n_list, lane & (C - 1));
                uint32_t upto = k;
#pragma unroll
                for (int o = 1; o < C; o <<= 1) {
                    const uint32_t p = __shfl_up_sync(0xffffffffu, upto, o);
                    if ((int)(lane & (C - 1)) >= o) upto += p;
                }
                n = __shfl_sync(0xffffffffu, upto, C - 1);
                const uint32_t kr = __shfl_sync(0xffffffffu, k, r), at = __shfl_sync(0xffffffffu, upto, r) - kr;
                if (r > 0u) {
                    const u64 *src = cg::this_cluster().map_shared_rank(&S.list.e[0], r);
#pragma unroll 1
                    for (uint32_t i = part * 32u + lane; i < kr && at + i < SAMPLE_CAP; i += (SAMPLE_WARPS / C) * 32u) S.list.e[at + i] = src[i];
                }
                n = min(n, SAMPLE_CAP);
                __syncthreads();
            }
        }
        return n;
    }
};

// The cut: kept are the tokens with a larger logit, and those with this one up to this index.
struct Cut {
    float x;
    uint32_t last;
    __device__ bool keeps(float v, uint32_t i) const { return v > x || (v == x && i <= last); }
};

template <int C>
__global__ void __launch_bounds__(SAMPLE_THREADS, 2) sample_kernel(const SampleArgs A) {
    using Row = SampleRow<C>;
    extern __shared__ __align__(16) uint8_t raw[];
    SampleShared &S = *reinterpret_cast<SampleShared *>(raw);
    float *own = reinterpret_cast<float *>(raw + sizeof(SampleShared));  // the block's logits
    const uint32_t rank = Row::me(), t = threadIdx.x, lane = t & 31u, row = blockIdx.x / C;
    const uint32_t base = min(A.n, rank * A.per), cnt = min(A.n, base + A.per) - base;
    const float *x = A.x + (size_t)row * A.stride + base;
    const float temp = A.p.d_temperature ? A.p.d_temperature[row] : 1.f;
    const int top_k = A.p.d_top_k ? A.p.d_top_k[row] : 0;
    const float top_p = A.p.d_top_p ? A.p.d_top_p[row] : 1.f, min_p = A.p.d_min_p ? A.p.d_min_p[row] : 0.f;
    const float u = A.u[row];
    const bool greedy = !(temp > 0.f);

    // the row into shared memory (NaN as -inf), its maximum
    float m = -INFINITY;
    const uint32_t quads = (reinterpret_cast<uintptr_t>(x) & 15u) == 0 ? cnt / 4u : 0u;
#pragma unroll 8
    for (uint32_t i = t; i < quads; i += SAMPLE_THREADS) {
        float4 v = __ldcs(reinterpret_cast<const float4 *>(x) + i);
        v = make_float4(fmaxf(v.x, -INFINITY), fmaxf(v.y, -INFINITY), fmaxf(v.z, -INFINITY), fmaxf(v.w, -INFINITY));
        reinterpret_cast<float4 *>(own)[i] = v;
        m = fmaxf(fmaxf(m, fmaxf(v.x, v.y)), fmaxf(v.z, v.w));
    }
#pragma unroll 8
    for (uint32_t i = 4u * quads + t; i < cnt; i += SAMPLE_THREADS) {
        const float v = fmaxf(__ldcs(x + i), -INFINITY);
        own[i] = v;
        m = fmaxf(m, v);
    }
    if (t < (-cnt & 3u)) own[cnt + t] = -INFINITY;
#pragma unroll 1
    for (uint32_t i = t; i < SAMPLE_BINS / 2; i += SAMPLE_THREADS) S.hist[i] = 0u;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (lane == 0) S.wf[t >> 5] = m;
    if (t == 0) {
        S.n_list = 0u;
        S.first = S.second = SAMPLE_BINS - 1u;
    }
    __syncthreads();
    m = S.wf[lane & (SAMPLE_WARPS - 1)];
#pragma unroll
    for (int o = SAMPLE_WARPS / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if constexpr (C > 1) {
        if (t == 0) S.fmax = __float_as_uint(m);
        Row::csync();
        m = __uint_as_float(Row::far(&S.fmax, lane & (C - 1)));
#pragma unroll
        for (int o = C / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    }
    // this thread's stretch where index order matters (of an odd length: no bank conflicts)
    const uint32_t seg = ((cnt + SAMPLE_THREADS - 1) / SAMPLE_THREADS) | 1u, i0 = min(cnt, t * seg), i1 = min(cnt, i0 + seg);
    if (m == INFINITY) {  // only the infinite ones have weight: as if they were the only ones
#pragma unroll 1
        for (uint32_t i = t; i < cnt; i += SAMPLE_THREADS) own[i] = own[i] == INFINITY ? 0.f : -INFINITY;
        m = 0.f;
        __syncthreads();
    }
    const Logits xs{own, cnt};
    const float c = fminf(1.4426950408889634f / temp, 1.0e36f);
    Row R{S, xs, base, m, c, 0.f, 0u, 0u};

    if (m == -INFINITY || greedy) {  // no token, or the first of the largest
        u64 best[1] = {0xffffffffull};
        if (m > -INFINITY)
#pragma unroll 1
            for (uint32_t i = i1; i-- > i0;)
                if (xs[i] == m) best[0] = base + i;
        R.fold(best, OpMin());
        if (rank == 0 && t == 0) {
            A.ids[row] = m > -INFINITY ? (uint32_t)best[0] : 0u;
            if (A.probs) A.probs[row] = m > -INFINITY ? 1.f : 0.f;
        }
        Row::csync();  // (nobody leaves while others read its shared memory)
        return;
    }
    auto write = [&](uint32_t id, u64 w, u64 total) {
        A.ids[row] = id;
        if (A.probs) A.probs[row] = (float)((double)w / (double)total);
    };
    auto target_of = [&](u64 total) {
        const double f = (double)(u >= 0.f ? u : 0.f) * (double)total;
        const u64 g = f < 1.0e19 ? (u64)f : total;
        return g < total ? g : total - 1;
    };
    Cut cut{-INFINITY, 0xffffffffu};
    const bool nucleus = top_p < 1.f;
    if ((top_k > 0 && (uint32_t)top_k < A.n) || nucleus) {
        // ---- histogram of log2 weight, near the maximum, or over all orders
        const uint32_t hist_at = smem_u32(&S.hist[0]);
        const bool want_k = top_k > 0 && (uint32_t)top_k < A.n;
        uint32_t h[SAMPLE_BPT], cc[SAMPLE_BPT], n_weight = 0;
        float sm[SAMPLE_BPT], a_total = 0.f, delta = 0.f, mid = 0.f;
        u64 all = 0;  // the weights of the whole row
        bool by_k = false;
#pragma unroll 1
        for (float orders = SAMPLE_NEAR;; orders = SAMPLE_ORDERS) {
            R.bins_over(orders);
            mid = orders / SAMPLE_BINS;
            delta = orders * (0.69314718f / (2 * SAMPLE_BINS)) * 1.1f + 1.0e-4f;  // half a bin, and f32 sums over the bins
            float sum = 0.f;
            auto count = [&](float v) {  // (in assembly for the predicated add: no branch around it)
                const float b = R.bin_of(v);
                const uint32_t k = Row::bin(b);
                asm volatile("{\n\t.reg .pred p;\n\tsetp.lt.f32 p, %0, %1;\n\t@p red.shared.add.u32 [%2], %3;\n\t}" ::"f"(b), "f"((float)SAMPLE_BINS),
                             "r"(hist_at + (k / 2u) * 4u), "r"((k & 1u) ? 0x10000u : 1u)
                             : "memory");
            };
            if (nucleus && orders == SAMPLE_NEAR)
                xs.each([&](float v, uint32_t) {
                    count(v);
                    sum += ex2(fmaxf(R.order(v), -200.f));
                });
            else
                xs.each([&](float v, uint32_t) { count(v); });
            if (nucleus && orders == SAMPLE_NEAR) {
                all = __float2ull_rn(sum * 1099511627776.f);  // (at most 128 weights)
                all = R.sum(all);                             // (its cluster barrier ends the histogram as well)
                if (C == 1) __syncthreads();
            } else {
                Row::csync();
            }
            // a thread's bins: counts and middle masses up to each (f32 sums in a fixed order: they only bound)
#pragma unroll
            for (int j = 0; j < SAMPLE_BPT; j++) h[j] = 0u;
#pragma unroll
            for (int r = 0; r < C; r++) {
                const uint2 q = Row::far(reinterpret_cast<const uint2 *>(&S.hist[0]) + t, r);
                h[0] += q.x & 0xffffu;
                h[1] += q.x >> 16;
                h[2] += q.y & 0xffffu;
                h[3] += q.y >> 16;
            }
            uint32_t c_all = 0;
            float s_all = 0.f;
#pragma unroll
            for (int j = 0; j < SAMPLE_BPT; j++) {
                c_all += h[j];
                s_all = fmaf((float)h[j], ex2(-((float)(SAMPLE_BPT * t + j) + 0.5f) * mid), s_all);
                cc[j] = c_all;
                sm[j] = s_all;
            }
        {
            uint32_t ci = c_all;
            float si = s_all;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t p = __shfl_up_sync(0xffffffffu, ci, o);
                const float q = __shfl_up_sync(0xffffffffu, si, o);
                if ((int)lane >= o) {
                    ci += p;
                    si += q;
                }
            }
            u64 *ws = S.ws[R.wturn][0];
            R.wturn ^= 1u;
            if (lane == 31u) {
                ws[t >> 5] = ci;
                S.wf[t >> 5] = si;
            }
            __syncthreads();
            const uint32_t cw = (uint32_t)ws[lane & (SAMPLE_WARPS - 1)];
            const float sw = S.wf[lane & (SAMPLE_WARPS - 1)];
            uint32_t cu = cw;
            float su = sw;
#pragma unroll
            for (int o = 1; o < SAMPLE_WARPS; o <<= 1) {
                const uint32_t p = __shfl_up_sync(0xffffffffu, cu, o);
                const float q = __shfl_up_sync(0xffffffffu, su, o);
                if ((int)(lane & (SAMPLE_WARPS - 1)) >= o) {
                    cu += p;
                    su += q;
                }
            }
            n_weight = __shfl_sync(0xffffffffu, cu, SAMPLE_WARPS - 1);
            a_total = __shfl_sync(0xffffffffu, su, SAMPLE_WARPS - 1);
            const float s_up = __shfl_up_sync(0xffffffffu, su, 1), s_in = __shfl_up_sync(0xffffffffu, si, 1);
            const uint32_t cb4 = __shfl_sync(0xffffffffu, cu - cw, t >> 5) + ci - c_all;
            const float sb = ((t >> 5) ? __shfl_sync(0xffffffffu, s_up, t >> 5) : 0.f) + (lane ? s_in : 0.f);
#pragma unroll
            for (int j = 0; j < SAMPLE_BPT; j++) {
                cc[j] += cb4;
                sm[j] += sb;
            }
        }
            // is the cut within these bins?
            by_k = want_k && (uint32_t)top_k < n_weight;
            if (orders == SAMPLE_ORDERS || by_k || (!want_k && (double)a_total * (1.0 - delta) * 1099511627776.0 >= (double)top_p * (double)all)) break;
            Row::csync();  // (all have read the counts)
#pragma unroll 1
            for (uint32_t i = t; i < SAMPLE_BINS / 2; i += SAMPLE_THREADS) S.hist[i] = 0u;
            __syncthreads();
        }
        const uint32_t k = by_k ? (uint32_t)top_k : n_weight;
        // S.first: the bin of the k-th token; S.second: the first bin up to which the masses surely reach top_p of all
        // (without top-k); and the tokens up to either
        const float sure = (float)((double)top_p * (double)all * (1.0 / 1099511627776.0)) / (1.f - delta);
        if (t == 0) S.found[0] = n_weight;
        __syncthreads();
#pragma unroll
        for (int j = 0; j < SAMPLE_BPT; j++) {
            const uint32_t c_prev = cc[j] - h[j];
            if (by_k) {
                if (c_prev < k && k <= cc[j]) {
                    S.first = SAMPLE_BPT * t + j;
                    S.found[0] = cc[j];
                    S.found[1] = c_prev;
                }
            } else if (nucleus && h[j] && sm[j] >= sure) {
                atomicMin(&S.second, SAMPLE_BPT * t + j);
            }
        }
        __syncthreads();
        const uint32_t bk = S.first, b_last = by_k ? bk : S.second;
        if (!by_k) {
            if (b_last / SAMPLE_BPT == t) S.found[0] = cc[b_last % SAMPLE_BPT];
            __syncthreads();
        }
        const uint32_t n_last = (uint32_t)S.found[0], above_k = (uint32_t)S.found[1];

        if (n_last <= SAMPLE_CAP) {
            // ---- few candidates: the whole draw in one block
            const float stop = (float)(b_last + 1u);
            const uint32_t n = R.gather([&](float v, uint32_t) { return R.bin_of(v) < stop; });
            if (rank == 0) {
                const uint32_t kk = by_k ? min(n, k) : n;
                if (n <= 64u) {
                    // ---- eight threads to a token; ranks, and sums in either order, by counting over all
                    const uint32_t i = t / 8u, part = t % 8u;
                    u64 *weight = S.list.sorted;
                    const u64 e = i < n ? S.list.e[i] : ~0ull;
                    const float v = key_logit(~(uint32_t)(e >> 32));
                    const auto eight = [](u64 x) {
                        x += __shfl_xor_sync(0xffffffffu, x, 1);
                        x += __shfl_xor_sync(0xffffffffu, x, 2);
                        return x + __shfl_xor_sync(0xffffffffu, x, 4);
                    };
                    u64 rk = 0;
#pragma unroll 1
                    for (uint32_t j = part; j < n; j += 8u) rk += S.list.e[j] < e;
                    rk = eight(rk);
                    u64 w = i < n && rk < kk ? Row::steps(R.order(v)) : 0ull;
                    if (part == 0u) weight[i] = w;
                    __syncthreads();
                    if (nucleus) {
                        u64 bef = 0, of_k = 0;
#pragma unroll 1
                        for (uint32_t j = part; j < n; j += 8u) {
                            of_k += weight[j];
                            bef += S.list.e[j] < e ? weight[j] : 0ull;
                        }
                        bef = eight(bef);
                        of_k = eight(of_k);
                        if (by_k) all = of_k;
                        if (rk && !((double)bef < (double)top_p * (double)all)) w = 0ull;
                    }
                    if (v != m && !(ex2(R.order(v)) >= min_p)) w = 0ull;
                    __syncthreads();
                    if (part == 0u) weight[i] = w;
                    __syncthreads();
                    u64 upto = 0, total = 0;
#pragma unroll 1
                    for (uint32_t j = part; j < n; j += 8u) {
                        total += weight[j];
                        upto += (uint32_t)S.list.e[j] <= (uint32_t)e ? weight[j] : 0ull;
                    }
                    upto = eight(upto);
                    total = eight(total);
                    const u64 target = target_of(total);
                    if (part == 0u && w && upto > target && upto - w <= target) write((uint32_t)e, w, total);
                } else {
                    R.sort_list(n);
                    u64 e[SAMPLE_BPT], w[SAMPLE_BPT], mine = 0;  // neighbours
#pragma unroll
                    for (int j = 0; j < SAMPLE_BPT; j++) {
                        const uint32_t i = SAMPLE_BPT * t + j;
                        e[j] = i < kk ? S.list.e[i] : ~0ull;
                        w[j] = i < kk ? Row::steps(R.order(key_logit(~(uint32_t)(e[j] >> 32)))) : 0ull;
                        mine += w[j];
                    }
                    u64 of_k;
                    u64 b = R.before(mine, of_k);
                    if (by_k) all = of_k;
                    const double need = (double)top_p * (double)all;
                    u64 kept = 0;
#pragma unroll
                    for (int j = 0; j < SAMPLE_BPT; j++) {
                        const uint32_t i = SAMPLE_BPT * t + j;
                        bool on = i < kk && (!nucleus || i == 0u || (double)b < need);
                        if (on) {
                            const float v = key_logit(~(uint32_t)(e[j] >> 32));
                            on = v == m || ex2(R.order(v)) >= min_p;
                        }
                        // kept tokens by index for the draw; the others go to the end
                        if (i < kk) S.list.e[i] = on ? (e[j] & 0xffffffffull) << 32 | (uint32_t)(e[j] >> 32) : ~0ull;
                        kept += on;
                        b += w[j];
                    }
                    u64 n_kept;
                    (void)R.before(kept, n_kept);
                    R.sort_list(kk);
                    mine = 0;
#pragma unroll
                    for (int j = 0; j < SAMPLE_BPT; j++) {
                        const uint32_t i = SAMPLE_BPT * t + j;
                        e[j] = i < (uint32_t)n_kept ? S.list.e[i] : ~0ull;
                        w[j] = i < (uint32_t)n_kept ? Row::steps(R.order(key_logit(~(uint32_t)e[j]))) : 0ull;
                        mine += w[j];
                    }
                    u64 total;
                    b = R.before(mine, total);
                    const u64 target = target_of(total);
#pragma unroll
                    for (int j = 0; j < SAMPLE_BPT; j++) {
                        if (b <= target && b + w[j] > target) write((uint32_t)(e[j] >> 32), w[j], total);
                        b += w[j];
                    }
                }
            }
            Row::csync();
            return;
        }

        // ---- many: cuts by the uncertain bins. A cut is told to all blocks through rank 0's S.found.
        auto told = [&](bool mine, uint32_t key, uint32_t last) {
            if (mine) S.found[1] = (u64)key << 32 | last;
            Row::csync();
            const u64 f = Row::far(&S.found[1], 0);
            Row::csync();
            return Cut{key_logit((uint32_t)(f >> 32)), (uint32_t)f};
        };
        // the index of the quota-th kept token with this key
        auto tie_index = [&](uint32_t key, const Cut &old, u64 quota) {
            u64 mine = 0, all;
#pragma unroll 1
            for (uint32_t i = i0; i < i1; i++) mine += logit_key(xs[i]) == key && old.keeps(xs[i], base + i);
            const u64 bef = R.before_all(mine, all);
            u64 at[1] = {0};
            if (bef < quota && quota <= bef + mine) {
                u64 q = bef;
#pragma unroll 1
                for (uint32_t i = i0; i < i1; i++)
                    if (logit_key(xs[i]) == key && old.keeps(xs[i], base + i) && ++q == quota) {
                        at[0] = base + i;
                        break;
                    }
            }
            R.fold(at, OpAdd());
            return (uint32_t)at[0];
        };
        // smallest and largest key among the tokens `in` names
        auto key_range = [&](auto in, uint32_t &lo, uint32_t &hi) {
            u64 r[2] = {0ull, 0ull};
#pragma unroll 1
            for (uint32_t i = i0; i < i1; i++)
                if (in(xs[i], base + i)) {
                    const uint32_t key = logit_key(xs[i]);
                    r[0] = max(r[0], (u64)~key);
                    r[1] = max(r[1], (u64)key);
                }
            R.fold(r, OpMax());
            lo = ~(uint32_t)r[0];
            hi = (uint32_t)r[1];
        };
        if (by_k) {
            const uint32_t quota = k - above_k;  // tokens of the bin that stay
            auto in = [&](float v, uint32_t) {
                const float b = R.bin_of(v);
                return b < (float)SAMPLE_BINS && Row::bin(b) == bk;
            };
            if (n_last - above_k <= SAMPLE_CAP) {
                const uint32_t n = R.gather(in);
                if (rank == 0) R.sort_list(n);
                const u64 e = rank == 0 ? S.list.e[quota - 1] : 0ull;
                cut = told(rank == 0 && t == 0, ~(uint32_t)(e >> 32), (uint32_t)e);
                if (t == 0) S.n_list = 0u;
            } else {  // the largest key that `quota` tokens of the bin reach
                uint32_t lo, hi;
                key_range(in, lo, hi);
#pragma unroll 1
                while (lo < hi) {
                    const uint32_t mid_key = lo + (hi - lo + 1u) / 2u;
                    u64 n = 0;
#pragma unroll 1
                    for (uint32_t i = i0; i < i1; i++) n += in(xs[i], 0u) && logit_key(xs[i]) >= mid_key;
                    if (R.sum(n) >= quota) lo = mid_key; else hi = mid_key - 1u;
                }
                u64 n = 0;
#pragma unroll 1
                for (uint32_t i = i0; i < i1; i++) n += in(xs[i], 0u) && logit_key(xs[i]) > lo;
                n = R.sum(n);
                cut = Cut{key_logit(lo), tie_index(lo, cut, quota - n)};
            }
        }
        if (nucleus) {
            if (by_k) {
                float sum = 0.f;
                xs.each([&](float v, uint32_t i) {
                    if (cut.keeps(v, base + i)) sum += ex2(fmaxf(R.order(v), -200.f));
                });
                all = R.sum(__float2ull_rn(sum * 1099511627776.f));
            }
            const double need = (double)top_p * (double)all;
            // bins that are surely kept, and from where on surely nothing is
            if (t == 0) {
                S.first = 0u;
                S.second = bk;
            }
            __syncthreads();
            const float n1 = (float)(need * (1.0 / 1099511627776.0)), lo_d = n1 / (1.f + delta), hi_d = n1 / (1.f - delta);
#pragma unroll
            for (int j = 0; j < SAMPLE_BPT; j++) {
                if (h[j] && sm[j] < lo_d) atomicMax(&S.first, SAMPLE_BPT * t + j + 1u);  // (the bin stays)
                if (h[j] && sm[j] >= hi_d) atomicMin(&S.second, SAMPLE_BPT * t + j);
            }
            __syncthreads();
            const uint32_t b_hi = S.second, b_lo = min(S.first, b_hi);  // the uncertain bins
            // exact masses: of what lies above them, and of 2048 finer bins
            __syncthreads();
#pragma unroll 1
            for (uint32_t i = t; i < SAMPLE_BINS; i += SAMPLE_THREADS) {
                S.fine.mass[i] = 0ull;
                S.fine.count[i] = 0u;
            }
            if (t == 0) S.first = 0u;
            __syncthreads();
            const float f_lo = (float)b_lo, f_hi = (float)(b_hi + 1u), f_scale = (float)SAMPLE_BINS / (f_hi - f_lo);
            auto fine = [&](float b) { return Row::bin(fminf((b - f_lo) * f_scale, (float)(SAMPLE_BINS - 1u))); };
            float above_f = 0.f;
            xs.each([&](float v, uint32_t i) {
                const float b = R.bin_of(v);
                if (b < f_lo) {
                    above_f += ex2(R.order(v));
                } else if (b < f_hi && (!by_k || cut.keeps(v, base + i))) {
                    const u64 w = Row::steps(R.order(v));
                    const uint32_t f = fine(b);
                    atomicAdd(&S.fine.count[f], 1u);
                    uint32_t *half = reinterpret_cast<uint32_t *>(&S.fine.mass[f]);
                    const uint32_t low = (uint32_t)w, was = atomicAdd(half, low);
                    const uint32_t high = (uint32_t)(w >> 32) + (was + low < was);  // (two adds that carry: exact in any order)
                    if (high) atomicAdd(half + 1, high);
                }
            });
            const u64 above = R.sum(__float2ull_rn(above_f * 1099511627776.f));
            if constexpr (C == 1) __syncthreads();  // (in a cluster, the sum's barrier ends the histogram)
            u64 g[SAMPLE_BPT] = {}, bef[SAMPLE_BPT];
            uint32_t q[SAMPLE_BPT] = {};
#pragma unroll
            for (int r = 0; r < C; r++) {
                const ulonglong2 ga = Row::far(reinterpret_cast<const ulonglong2 *>(&S.fine.mass[0]) + 2 * t, r);
                const ulonglong2 gb = Row::far(reinterpret_cast<const ulonglong2 *>(&S.fine.mass[0]) + 2 * t + 1, r);
                const uint4 qa = Row::far(reinterpret_cast<const uint4 *>(&S.fine.count[0]) + t, r);
                g[0] += ga.x;
                g[1] += ga.y;
                g[2] += gb.x;
                g[3] += gb.y;
                q[0] += qa.x;
                q[1] += qa.y;
                q[2] += qa.z;
                q[3] += qa.w;
            }
            u64 g_all;
            bef[0] = above + R.before(g[0] + g[1] + g[2] + g[3], g_all);
            // the last finer bin with tokens before which the mass is below `need`
#pragma unroll
            for (int j = 0; j < SAMPLE_BPT; j++) {
                if (j) bef[j] = bef[j - 1] + g[j - 1];
                if (q[j] && ((double)bef[j] < need || bef[j] == 0ull)) atomicMax(&S.first, SAMPLE_BPT * t + j + 1u);
            }
            __syncthreads();
            const uint32_t fb1 = S.first;
            if (fb1 > 0u) {  // (0: no token in the uncertain bins, nothing to cut)
                const uint32_t fb = fb1 - 1u;
#pragma unroll
                for (int j = 0; j < SAMPLE_BPT; j++)
                    if (fb == SAMPLE_BPT * t + j) {
                        S.found[0] = bef[j];
                        S.second = q[j];
                    }
                Row::csync();  // every block has read the others' masses: the lists may take their place
                const u64 mass_above = S.found[0];
                const uint32_t n_fine = S.second;
                const Cut old = cut;
                auto in = [&](float v, uint32_t i) {
                    const float b = R.bin_of(v);
                    return b >= f_lo && b < f_hi && fine(b) == fb && (!by_k || old.keeps(v, i));
                };
                if (n_fine <= SAMPLE_CAP) {
                    const uint32_t n = R.gather(in);
                    if (rank == 0) {
                        R.sort_list(n);
                        u64 w[SAMPLE_BPT], mine = 0, dummy;
#pragma unroll
                        for (int j = 0; j < SAMPLE_BPT; j++) {
                            const uint32_t i = SAMPLE_BPT * t + j;
                            w[j] = i < n ? Row::steps(R.order(key_logit(~(uint32_t)(S.list.e[i] >> 32)))) : 0ull;
                            mine += w[j];
                        }
                        if (t == 0) S.first = 0u;
                        u64 b = mass_above + R.before(mine, dummy);
                        // the last token before which the mass is below `need`
#pragma unroll
                        for (int j = 0; j < SAMPLE_BPT; j++) {
                            const uint32_t i = SAMPLE_BPT * t + j;
                            if (i < n && ((double)b < need || b == 0ull)) atomicMax(&S.first, i);
                            b += w[j];
                        }
                        __syncthreads();
                    }
                    const u64 e = rank == 0 ? S.list.e[S.first] : 0ull;
                    cut = told(rank == 0 && t == 0, ~(uint32_t)(e >> 32), (uint32_t)e);
                } else {  // the least key above which the mass is below `need`, then how many of its equals
                    uint32_t lo, hi;
                    key_range(in, lo, hi);
#pragma unroll 1
                    while (lo < hi) {
                        const uint32_t mid_key = lo + (hi - lo) / 2u;
                        u64 w = 0;
#pragma unroll 1
                        for (uint32_t i = i0; i < i1; i++)
                            if (logit_key(xs[i]) > mid_key && in(xs[i], base + i)) w += Row::steps(R.order(xs[i]));
                        if ((double)(mass_above + R.sum(w)) < need) hi = mid_key; else lo = mid_key + 1u;
                    }
                    u64 v[2] = {0ull, 0ull};
#pragma unroll 1
                    for (uint32_t i = i0; i < i1; i++)
                        if (in(xs[i], base + i)) {
                            const uint32_t key = logit_key(xs[i]);
                            if (key > lo) v[0] += Row::steps(R.order(xs[i]));
                            v[1] += key == lo;
                        }
                    R.fold(v, OpAdd());
                    const u64 w1 = Row::steps(R.order(key_logit(lo))), s = mass_above + v[0];
                    // the j-th equal (from 0) stays if s + j w1 < need
                    double j = w1 ? ceil((need - (double)s) / (double)w1) : (double)v[1];
                    j = fmin(fmax(j, 1.0), (double)v[1]);
                    cut = Cut{key_logit(lo), tie_index(lo, old, (u64)j)};
                }
            }
        }
    }

    // ---- the draw, in index order
    const float low = min_p > 0.f ? min_p : 0.f;
    auto value = [&](float v, uint32_t i) -> float {
        const float w = ex2(fmaxf(R.order(v), -200.f));
        return cut.keeps(v, base + i) && (w >= low || v == m) ? w : 0.f;
    };
    // a warp sums a stretch of neighbours (f32 within a lane, integers beyond); the block that has the target goes over the stretch
    // that has it once more, a few neighbours to a thread. What f32 rounds differently there moves the end of the stretch by
    // 2^-24 of it: a target beyond that end is the stretch's last kept token.
    const uint32_t w = t >> 5, len = ((cnt + SAMPLE_WARPS - 1) / SAMPLE_WARPS + 3u) & ~3u, w0 = min(cnt, w * len), w1 = min(cnt, w0 + len);
    float lane_sum = 0.f;
    xs.each(w0, w1, lane, 32u, [&](float v, uint32_t i) { lane_sum += value(v, i); });
    u64 mine = __float2ull_rn(lane_sum * 1099511627776.f), total;
    u64 b = R.before_all(mine, total);  // (threads are in warp order, so this is where the warp's stretch begins, at its first lane)
    const u64 target = target_of(total);
    u64 sum = mine;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    b = __shfl_sync(0xffffffffu, b, 0);
    if (t == 0) S.first = SAMPLE_WARPS;
    __syncthreads();
    if (lane == 0 && b <= target && b + sum > target) {
        S.first = w;
        S.found[0] = b;
    }
    __syncthreads();
    if (S.first < SAMPLE_WARPS) {  // (in one block of the cluster)
        const uint32_t s0 = min(cnt, S.first * len), s1 = min(cnt, s0 + len), part = (len + SAMPLE_THREADS - 1) / SAMPLE_THREADS;
        const uint32_t j0 = min(s1, s0 + t * part), j1 = min(s1, j0 + part);
        auto steps = [](float w) { return w > 0.f ? max(1ull, __float2ull_rn(w * 1099511627776.f)) : 0ull; };  // (something is kept here)
        mine = 0;
#pragma unroll 1
        for (uint32_t i = j0; i < j1; i++) mine += steps(value(xs[i], i));
        u64 of_part;
        u64 at = S.found[0] + R.before(mine, of_part);
        const u64 end = S.found[0] + of_part, goal = target < end ? target : end - 1u;
        if (at <= goal && at + mine > goal) {
#pragma unroll 1
            for (uint32_t i = j0; i < j1; i++) {
                const u64 v = steps(value(xs[i], i));
                at += v;
                if (at > goal) {
                    write(base + i, v, total);
                    break;
                }
            }
        }
    }
    Row::csync();
}

template <int C>
static cudaError_t sample_launch(strix_cuda *h, const SampleArgs &A, uint32_t rows, cudaStream_t stream) {
    const size_t smem = sizeof(SampleShared) + (size_t)A.per * 4;
    static std::atomic<uint64_t> ready{0};  // devices whose limit of dynamic shared memory is raised for this kernel
    const uint64_t bit = 1ull << (h->device & 63);
    if (!(ready.load(std::memory_order_relaxed) & bit)) {
        const cudaError_t e = cudaFuncSetAttribute(sample_kernel<C>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(h->smem_optin - 512));
        if (e != cudaSuccess) return e;
        ready.fetch_or(bit, std::memory_order_relaxed);
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(rows * C);
    cfg.blockDim = dim3(SAMPLE_THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = C;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, sample_kernel<C>, A);
}

// A row takes as many blocks as make it 4096 logits or fewer to a block, at most 8: more blocks shorten every pass, a barrier among
// them costs the same, but fewer rows run at once. Measured, us with up to 8 and up to 4 blocks for 151936 logits: one row 12.5 and 15.4,
// 16 nucleus rows 47 and 52, 64 mixed rows 57 and 54. With 4096 and with 8192 to a block: 64 mixed rows of 20000 logits 25 and 13, one
// row 9.2 and 9.0; of 5000 logits 9.9 and 8.3, 8.0 and 6.8. (2048 to a block: 25, 9.2, 11.6, 8.1.)
cudaError_t launch_sample(strix_cuda *h, const float *d_x, uint32_t n, size_t stride, uint32_t rows, const strix_sample_params &p,
                          const float *d_u, uint32_t *d_ids, float *d_probs, cudaStream_t stream) {
    uint32_t c = 1;
    while (c < 8 && (n + c - 1) / c > 4096) c *= 2;
    const SampleArgs A{d_x, stride, n, ((n + c - 1) / c + 3u) & ~3u, p, d_u, d_ids, d_probs};
    static_assert(sizeof(SampleShared) + (STRIX_SAMPLE_MAX_N / 8 + 4) * 4 <= 231000, "the longest row fits eight blocks");
    ProfScope prof(h, stream, "sample");
    switch (c) {
        case 1: return sample_launch<1>(h, A, rows, stream);
        case 2: return sample_launch<2>(h, A, rows, stream);
        case 4: return sample_launch<4>(h, A, rows, stream);
        default: return sample_launch<8>(h, A, rows, stream);
    }
}

}  // namespace strix

using namespace strix;

extern "C" int strix_cuda_sample_dev(strix_cuda *h, const float *d_x, size_t n, size_t stride, size_t rows,
                                     const strix_sample_params *params, const float *d_u, uint32_t *d_ids, float *d_probs,
                                     void *stream) {
    if (!h) return -1;
    h->err.clear();
    const char *who = "sample";
    if (n == 0 || n > STRIX_SAMPLE_MAX_N) return serve_fail(h, who, "1 to STRIX_SAMPLE_MAX_N logits to a row");
    if (rows > 0x7fffffffu / 16u) return serve_fail(h, who, "too many rows");
    if (rows > 1 && stride < n) return serve_fail(h, who, "the row stride is smaller than a row");
    if (rows == 0) return 1;
    if (!d_x || !d_u || !d_ids) return serve_fail(h, who, "d_x, d_u or d_ids missing");
    DeviceGuard dev(h->device);
    if (dev.err != cudaSuccess) return serve_fail(h, who, cudaGetErrorString(dev.err));
    const cudaError_t e = launch_sample(h, d_x, (uint32_t)n, stride, (uint32_t)rows, params ? *params : strix_sample_params{}, d_u, d_ids, d_probs,
                                        static_cast<cudaStream_t>(stream));
    if (e != cudaSuccess) return serve_fail(h, who, cudaGetErrorString(e));
    return 1;
}
