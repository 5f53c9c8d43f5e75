// Drawing a token from logits: temperature, top-k, top-p, min-p and the inverse of the distribution function at a given
// number. Contract: include/strix_serve.h. Stands beside the greedy argmax (argmax.cu).
//
// A row lives in the shared memory of a cluster of blocks, so the logits are read from HBM once and every question about them
// is a pass over on-chip data: what bounds a draw is the number of passes and cluster barriers (about a microsecond each), not the
// 4 bytes a logit.
//
// Nothing as long as the row is sorted. What top-k and top-p keep is, in the order (logit, lower index first), everything down to
// one cut (key, index). The cut is found from a histogram of log2 weight (y = (x - max) log2(e) / T; 2048 bins over the 41
// binary orders that a weight in steps of 2^-40 can have; logits below that have no weight and no part in anything):
//   top-k: the bin in which the count passes k;
//   top-p: a bin's mass is its count times its middle weight to within SAMPLE_DELTA, so the counts bound where the mass
//          passes top_p: mostly a few bins.
// If all that the cut may leave is at most SAMPLE_CAP tokens, they are gathered in one block, sorted and the draw ends there.
// Otherwise the uncertain bins alone are resolved: exact masses on 2048 finer bins, then the tokens of one of those are
// sorted, or, where they are too many (logits that came from 16 bits have thousands of equal values), the cut is bisected
// over their keys. The draw itself is a sum over the row in index order.
// Weights are summed as 64-bit integers in steps of 2^-40, so no sum depends on its order, and neither does the draw.
#include <cooperative_groups.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>

#include "kv_pages.cuh"

namespace cg = cooperative_groups;

namespace strix {

typedef unsigned long long u64;

constexpr int SAMPLE_THREADS = 1024;
constexpr uint32_t SAMPLE_BINS = 2048, SAMPLE_CAP = 2048;
constexpr float SAMPLE_ORDERS = 41.f;       // weights below 2^-41 round to no step of 2^-40
constexpr float SAMPLE_DELTA = 0.008f;      // half a bin: 41 ln 2 / 2047 / 2 = 0.0069, and f32 sums over 2048 bins
constexpr uint32_t SAMPLE_MAX_CLUSTER = 16;

struct SampleArgs {
    const float *x;
    size_t stride;
    uint32_t n, per;  // logits of a row, of a block (a multiple of 4)
    strix_sample_params p;
    const float *u;
    uint32_t *ids;
    float *probs;
};

// Unsigned keys in the order of the logits; NaN ranks as -inf, -0 equals +0.
__device__ __forceinline__ uint32_t logit_key(float x) {
    if (x != x) x = -INFINITY;
    const uint32_t b = __float_as_uint(x + 0.f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_logit(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

struct SampleShared {
    uint32_t hist[SAMPLE_BINS];
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
    u64 warp_sum[SAMPLE_THREADS / 32];
    u64 xch[2][4];                  // what the cluster's blocks tell each other, in turns
    uint32_t n_list, first, second, rank[256];
    u64 found[2];
    float fred[SAMPLE_THREADS / 32];
};

static_assert(sizeof(SampleShared) % 16 == 0, "the logits behind it are read in 16-byte words");

// One block's view of its row.
struct SampleRow {
    SampleShared &S;
    const float *xs;               // this block's logits
    uint32_t cnt, base, seg, i0, i1;  // how many, index of the first; this thread's stretch (an odd length: no bank conflicts)
    float m, c, min_p;
    uint32_t turn;
    cg::cluster_group cl;

    __device__ float order(float x) const {  // log2 of the weight
        return x == m ? 0.f : m == INFINITY || !(x > -INFINITY) ? -INFINITY : (x - m) * c;
    }
    __device__ static u64 steps(float y) { return y < -SAMPLE_ORDERS ? 0ull : __float2ull_rn(exp2f(y) * 1099511627776.f); }
    __device__ static uint32_t bin(float y) {  // SAMPLE_BINS = no weight
        return y < -SAMPLE_ORDERS ? SAMPLE_BINS : (uint32_t)(y * -((float)(SAMPLE_BINS - 1u) / SAMPLE_ORDERS));
    }

    // Sums (or with op a maximum / minimum) of up to four values over the block, then over the cluster; all threads get them.
    template <int N, typename F>
    __device__ void block_fold(u64 (&v)[N], F op) {
#pragma unroll
        for (int k = 0; k < N; k++) {
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) v[k] = op(v[k], __shfl_xor_sync(0xffffffffu, v[k], o));
            __syncthreads();
            if ((threadIdx.x & 31u) == 0) S.warp_sum[threadIdx.x >> 5] = v[k];
            __syncthreads();
            v[k] = S.warp_sum[threadIdx.x & 31u];
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) v[k] = op(v[k], __shfl_xor_sync(0xffffffffu, v[k], o));
        }
    }
    template <int N, typename F>
    __device__ void fold(u64 (&v)[N], F op) {
        block_fold(v, op);
        if (threadIdx.x == 0)
            for (int k = 0; k < N; k++) S.xch[turn][k] = v[k];
        cl.sync();
        for (int k = 0; k < N; k++)
            for (uint32_t r = 0; r < cl.num_blocks(); r++) {
                const u64 w = *cl.map_shared_rank(&S.xch[turn][k], r);
                v[k] = r ? op(v[k], w) : w;
            }
        turn ^= 1u;
    }
    __device__ u64 sum(u64 v) {
        u64 a[1] = {v};
        fold(a, [](u64 p, u64 q) { return p + q; });
        return a[0];
    }
    // this thread's place in the block: the sum over the threads before it, and over all
    __device__ u64 before(u64 v, u64 &all) {
        const uint32_t lane = threadIdx.x & 31u, w = threadIdx.x >> 5;
        u64 incl = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const u64 p = __shfl_up_sync(0xffffffffu, incl, o);
            if ((int)lane >= o) incl += p;
        }
        __syncthreads();
        if (lane == 31u) S.warp_sum[w] = incl;
        __syncthreads();
        u64 ws = S.warp_sum[lane];
        u64 wi = ws;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const u64 p = __shfl_up_sync(0xffffffffu, wi, o);
            if ((int)lane >= o) wi += p;
        }
        all = __shfl_sync(0xffffffffu, wi, 31);
        return __shfl_sync(0xffffffffu, wi - ws, w) + incl - v;
    }
    // the same over the cluster's blocks, in rank order
    __device__ u64 before_all(u64 v, u64 &all) {
        u64 mine;
        u64 b = before(v, mine);
        if (threadIdx.x == 0) S.xch[turn][0] = mine;
        cl.sync();
        all = 0;
        for (uint32_t r = 0; r < cl.num_blocks(); r++) {
            const u64 w = *cl.map_shared_rank(&S.xch[turn][0], r);
            if (r < cl.block_rank()) b += w;
            all += w;
        }
        turn ^= 1u;
        return b;
    }

    // S.list.e[0 .. n) in ascending order (n <= SAMPLE_CAP), by this block
    __device__ void sort_list(uint32_t n) {
        const uint32_t t = threadIdx.x;
        if (n <= 256u) {  // by rank: every entry counts the smaller ones, SAMPLE_THREADS / np threads to an entry
            uint32_t np = 32;
            while (np < n) np *= 2;
            if (t < 256u) S.rank[t] = 0u;
            __syncthreads();
            const uint32_t e = t & (np - 1u), part = t / np, parts = SAMPLE_THREADS / np;
            if (e < n) {
                const u64 mine = S.list.e[e];
                uint32_t less = 0;
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
        while (np < n) np *= 2;
        for (uint32_t i = n + t; i < np; i += SAMPLE_THREADS) S.list.e[i] = ~0ull;
        __syncthreads();
        for (uint32_t k = 2; k <= np; k *= 2)
            for (uint32_t j = k / 2; j > 0; j /= 2) {
                if (t < np / 2) {
                    const uint32_t a = 2 * t - (t & (j - 1u)), b = a + j;
                    const u64 p = S.list.e[a], q = S.list.e[b];
                    if ((p > q) == ((a & k) == 0u)) {
                        S.list.e[a] = q;
                        S.list.e[b] = p;
                    }
                }
                __syncthreads();
            }
    }
    // Gathers the tokens that `want` names, from all blocks, into rank 0's list: (descending key, index). Ends behind a cluster
    // barrier after which only rank 0 has the list; the others' lists stay until the next barrier.
    template <typename F>
    __device__ uint32_t gather(F want) {
        __syncthreads();
        if (threadIdx.x == 0) S.n_list = 0u;
        __syncthreads();
        for (uint32_t i = i0; i < i1; i++) {
            const float x = xs[i];
            if (!want(x)) continue;
            const uint32_t at = atomicAdd(&S.n_list, 1u);
            if (at < SAMPLE_CAP) S.list.e[at] = (u64)(~logit_key(x)) << 32 | (base + i);
        }
        cl.sync();
        uint32_t n = S.n_list;
        if (cl.block_rank() == 0) {
            for (uint32_t r = 1; r < cl.num_blocks(); r++) {
                const uint32_t k = *cl.map_shared_rank(&S.n_list, r);
                const u64 *src = cl.map_shared_rank(&S.list.e[0], r);
                for (uint32_t i = threadIdx.x; i < k && n + i < SAMPLE_CAP; i += SAMPLE_THREADS) S.list.e[n + i] = src[i];
                n += k;
            }
            n = min(n, SAMPLE_CAP);
            __syncthreads();
        }
        return n;
    }
};

// The cut: kept are the tokens with a larger key, and those with this key up to this index.
struct Cut {
    uint32_t key, last;
    __device__ bool keeps(uint32_t k, uint32_t i) const { return k > key || (k == key && i <= last); }
};

__global__ void __launch_bounds__(SAMPLE_THREADS) sample_kernel(const SampleArgs A) {
    extern __shared__ __align__(16) uint8_t raw[];
    SampleShared &S = *reinterpret_cast<SampleShared *>(raw);
    float *xs = reinterpret_cast<float *>(raw + sizeof(SampleShared));
    cg::cluster_group cl = cg::this_cluster();
    const uint32_t C = cl.num_blocks(), rank = cl.block_rank(), t = threadIdx.x, row = blockIdx.x / C;
    const uint32_t base = min(A.n, rank * A.per), cnt = min(A.n, base + A.per) - base;
    const float *x = A.x + (size_t)row * A.stride + base;
    const float temp = A.p.d_temperature ? A.p.d_temperature[row] : 1.f;
    const int top_k = A.p.d_top_k ? A.p.d_top_k[row] : 0;
    const float top_p = A.p.d_top_p ? A.p.d_top_p[row] : 1.f;
    float u = A.u[row];
    const bool greedy = !(temp > 0.f);

    // the row into shared memory, its maximum
    float m = -INFINITY;
    if ((reinterpret_cast<uintptr_t>(x) & 15u) == 0) {
        const uint32_t n4 = cnt / 4;
        const float4 *x4 = reinterpret_cast<const float4 *>(x);
        float4 *s4 = reinterpret_cast<float4 *>(xs);
#pragma unroll 4
        for (uint32_t i = t; i < n4; i += SAMPLE_THREADS) {
            const float4 v = __ldcs(x4 + i);
            s4[i] = v;
            m = fmaxf(fmaxf(m, fmaxf(v.x, v.y)), fmaxf(v.z, v.w));
        }
        for (uint32_t i = n4 * 4 + t; i < cnt; i += SAMPLE_THREADS) {
            const float v = x[i];
            xs[i] = v;
            m = fmaxf(m, v);
        }
    } else {
#pragma unroll 8
        for (uint32_t i = t; i < cnt; i += SAMPLE_THREADS) {
            const float v = __ldcs(x + i);
            xs[i] = v;
            m = fmaxf(m, v);
        }
    }
    for (uint32_t i = t; i < SAMPLE_BINS; i += SAMPLE_THREADS) S.hist[i] = 0u;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if ((t & 31u) == 0) S.fred[t >> 5] = m;
    __syncthreads();
    m = S.fred[t & 31u];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (t == 0) S.xch[1][0] = __float_as_uint(m);
    cl.sync();
    for (uint32_t r = 0; r < C; r++) m = fmaxf(m, __uint_as_float((uint32_t)*cl.map_shared_rank(&S.xch[1][0], r)));
    const uint32_t seg = ((cnt + SAMPLE_THREADS - 1) / SAMPLE_THREADS) | 1u, i0 = min(cnt, t * seg);
    SampleRow R{S, xs, cnt, base, seg, i0, min(cnt, i0 + seg), m, 1.4426950408889634f / temp, A.p.d_min_p ? A.p.d_min_p[row] : 0.f, 0u, cl};
    const uint32_t i1 = R.i1;
    if (greedy) R.c = INFINITY;  // nothing but the maximum has weight

    if (m == -INFINITY || greedy) {  // no token, or the first of the largest
        u64 best[1] = {0xffffffffull};
        if (m > -INFINITY)
            for (uint32_t i = i1; i-- > i0;)
                if (xs[i] == m) best[0] = base + i;
        R.fold(best, [](u64 p, u64 q) { return p < q ? p : q; });
        if (rank == 0 && t == 0) {
            A.ids[row] = m > -INFINITY ? (uint32_t)best[0] : 0u;
            if (A.probs) A.probs[row] = m > -INFINITY ? 1.f : 0.f;
        }
        cl.sync();  // (nobody leaves while others read its shared memory)
        return;
    }
    auto add = [](u64 p, u64 q) { return p + q; };
    auto write = [&](uint32_t id, u64 w, u64 total) {
        A.ids[row] = id;
        if (A.probs) A.probs[row] = (float)((double)w / (double)total);
    };
    auto target_of = [&](u64 total) {
        const double f = (double)(u >= 0.f ? u : 0.f) * (double)total;
        const u64 g = f < 1.0e19 ? (u64)f : total;
        return g < total ? g : total - 1;
    };
    Cut cut{0u, 0xffffffffu};
    const bool nucleus = top_p < 1.f;
    if ((top_k > 0 && (uint32_t)top_k < A.n) || nucleus) {
        // ---- histogram of log2 weight
        for (uint32_t i = i0; i < i1; i++) {
            const uint32_t b = R.bin(R.order(xs[i]));
            if (b < SAMPLE_BINS) atomicAdd(&S.hist[b], 1u);
        }
        cl.sync();
        // thread t: bins 2 t and 2 t + 1 over the cluster; counts and middle masses up to each
        uint32_t h0 = 0, h1 = 0;
        for (uint32_t r = 0; r < C; r++) {
            const uint2 h = reinterpret_cast<const uint2 *>(cl.map_shared_rank(&S.hist[0], r))[t];
            h0 += h.x;
            h1 += h.y;
        }
        u64 n_weight;
        const u64 c_before = R.before(h0 + h1, n_weight), c0 = c_before + h0, c1 = c0 + h1;
        const float mid = SAMPLE_ORDERS / (SAMPLE_BINS - 1u);
        const float a0 = (float)h0 * exp2f(-(2.f * t + 0.5f) * mid), a1 = (float)h1 * exp2f(-(2.f * t + 1.5f) * mid);
        // (in steps of 2^-32: at least 2^18 tokens of weight 1 fit, and smaller ones do not count here)
        u64 a_total;
        const u64 a_before = R.before((u64)__float2ull_rn(a0 * 4294967296.f) + (u64)__float2ull_rn(a1 * 4294967296.f), a_total);
        const double s0 = (double)(a_before + (u64)__float2ull_rn(a0 * 4294967296.f)),
                     s1 = s0 + (double)(u64)__float2ull_rn(a1 * 4294967296.f);
        const bool by_k = top_k > 0 && (u64)top_k < n_weight;
        const u64 k = by_k ? (u64)top_k : n_weight;
        // S.first: bin of the k-th token; S.second: the last bin that may matter
        if (t == 0) S.first = S.second = SAMPLE_BINS - 1u;
        __syncthreads();
        if (by_k) {
            if (c_before < k && k <= c0) S.first = 2u * t;
            if (c0 < k && k <= c1) S.first = 2u * t + 1u;
        }
        // the first bin up to which the masses surely reach top_p of all of them (only without top-k, where all is all)
        const double sure = (double)top_p * (double)a_total * (1.0 + SAMPLE_DELTA) / (1.0 - SAMPLE_DELTA) + SAMPLE_BINS;
        if (!by_k && nucleus) {
            if ((double)a_before < sure && sure <= s0) S.second = 2u * t;
            if (s0 < sure && sure <= s1) S.second = 2u * t + 1u;
        }
        __syncthreads();
        const uint32_t bk = S.first, b_last = by_k ? bk : S.second;
        // tokens up to b_last
        __syncthreads();
        if (b_last / 2u == t) S.found[0] = b_last & 1u ? c1 : c0;
        __syncthreads();
        const u64 n_last = S.found[0];

        if (n_last <= SAMPLE_CAP) {
            // ---- few candidates: the whole draw in one block
            u64 all = 0;
            if (!by_k) {  // top-p of the whole row
                for (uint32_t i = i0; i < i1; i++) all += R.steps(R.order(xs[i]));
                all = R.sum(all);
            }
            const uint32_t n = R.gather([&](float v) { return R.bin(R.order(v)) <= b_last; });
            if (rank == 0) {
                R.sort_list(n);
                const uint32_t keep = by_k ? min(n, (uint32_t)k) : n;
                // two neighbours to a thread
                u64 e[2], w[2];
                for (int j = 0; j < 2; j++) {
                    const uint32_t i = 2u * t + j;
                    e[j] = i < keep ? S.list.e[i] : ~0ull;
                    w[j] = i < keep ? R.steps(R.order(key_logit(~(uint32_t)(e[j] >> 32)))) : 0ull;
                }
                u64 sum_k;
                const u64 b0 = R.before(w[0] + w[1], sum_k);
                if (by_k) all = sum_k;
                const double need = (double)top_p * (double)all;
                u64 kept = 0;
                for (int j = 0; j < 2; j++) {
                    const uint32_t i = 2u * t + j;
                    const u64 bef = j ? b0 + w[0] : b0;
                    bool on = i < keep && (!nucleus || i == 0u || (double)bef < need);
                    if (on) {
                        const float v = key_logit(~(uint32_t)(e[j] >> 32));
                        on = v == m || exp2f(R.order(v)) >= R.min_p;
                    }
                    // kept tokens by index for the draw; the others go to the end
                    if (i < keep) S.list.e[i] = on ? (e[j] & 0xffffffffull) << 32 | (uint32_t)(e[j] >> 32) : ~0ull;
                    kept += on;
                }
                u64 n_kept;
                (void)R.before(kept, n_kept);
                __syncthreads();
                R.sort_list(keep);
                for (int j = 0; j < 2; j++) {
                    const uint32_t i = 2u * t + j;
                    e[j] = i < (uint32_t)n_kept ? S.list.e[i] : ~0ull;
                    w[j] = i < (uint32_t)n_kept ? R.steps(R.order(key_logit(~(uint32_t)e[j]))) : 0ull;
                }
                u64 total;
                const u64 bef = R.before(w[0] + w[1], total), target = target_of(total);
                if (bef <= target && bef + w[0] > target) write((uint32_t)(e[0] >> 32), w[0], total);
                else if (bef + w[0] <= target && bef + w[0] + w[1] > target) write((uint32_t)(e[1] >> 32), w[1], total);
            }
            cl.sync();
            return;
        }

        // ---- many: cuts by the uncertain bins. A cut is told to all blocks through rank 0's S.found.
        auto told = [&](bool mine, uint32_t key, uint32_t last) {
            if (mine) S.found[1] = (u64)key << 32 | last;
            cl.sync();
            const u64 f = *cl.map_shared_rank(&S.found[1], 0);
            cl.sync();
            return Cut{(uint32_t)(f >> 32), (uint32_t)f};
        };
        // the index of the quota-th kept token with this key
        auto tie_index = [&](uint32_t key, const Cut &old, u64 quota) {
            u64 mine = 0, all;
            for (uint32_t i = i0; i < i1; i++) mine += logit_key(xs[i]) == key && old.keeps(key, base + i);
            const u64 bef = R.before_all(mine, all);
            u64 at[1] = {0};
            if (bef < quota && quota <= bef + mine) {
                u64 q = bef;
                for (uint32_t i = i0; i < i1; i++)
                    if (logit_key(xs[i]) == key && old.keeps(key, base + i) && ++q == quota) {
                        at[0] = base + i;
                        break;
                    }
            }
            R.fold(at, add);
            return (uint32_t)at[0];
        };
        // smallest and largest key among the tokens `in` names
        auto key_range = [&](auto in, uint32_t &lo, uint32_t &hi) {
            u64 r[2] = {0ull, 0ull};
            for (uint32_t i = i0; i < i1; i++)
                if (in(xs[i], base + i)) {
                    const uint32_t key = logit_key(xs[i]);
                    r[0] = max(r[0], (u64)~key);
                    r[1] = max(r[1], (u64)key);
                }
            R.fold(r, [](u64 p, u64 q) { return p > q ? p : q; });
            lo = ~(uint32_t)r[0];
            hi = (uint32_t)r[1];
        };
        if (by_k) {
            if (bk / 2u == t) S.found[0] = bk & 1u ? c0 : c_before;  // tokens above the bin
            __syncthreads();
            const u64 above = S.found[0], quota = k - above;
            auto in = [&](float v, uint32_t) { return R.bin(R.order(v)) == bk; };
            if (n_last - above <= SAMPLE_CAP) {
                const uint32_t n = R.gather([&](float v) { return in(v, 0u); });
                if (rank == 0) R.sort_list(n);
                const u64 e = rank == 0 ? S.list.e[quota - 1] : 0ull;
                cut = told(rank == 0 && t == 0, ~(uint32_t)(e >> 32), (uint32_t)e);
            } else {  // the largest key that `quota` tokens of the bin reach
                uint32_t lo, hi;
                key_range(in, lo, hi);
                while (lo < hi) {
                    const uint32_t mid_key = lo + (hi - lo + 1u) / 2u;
                    u64 n = 0;
                    for (uint32_t i = i0; i < i1; i++) n += in(xs[i], 0u) && logit_key(xs[i]) >= mid_key;
                    if (R.sum(n) >= quota) lo = mid_key; else hi = mid_key - 1u;
                }
                u64 n = 0;
                for (uint32_t i = i0; i < i1; i++) n += in(xs[i], 0u) && logit_key(xs[i]) > lo;
                n = R.sum(n);
                cut = Cut{lo, tie_index(lo, cut, quota - n)};
            }
        }
        if (nucleus) {
            u64 all = 0;
            for (uint32_t i = i0; i < i1; i++)
                if (cut.keeps(logit_key(xs[i]), base + i)) all += R.steps(R.order(xs[i]));
            all = R.sum(all);
            const double need = (double)top_p * (double)all;
            // bins that are surely kept, and from where on surely nothing is: masses in steps of 2^-32 against `need` in 2^-40
            const double n32 = need * 0.00390625;
            if (t == 0) {
                S.first = 0u;
                S.second = bk;
            }
            __syncthreads();
            const double lo_d = n32 / (1.0 + SAMPLE_DELTA) - SAMPLE_BINS, hi_d = n32 / (1.0 - SAMPLE_DELTA) + SAMPLE_BINS;
            if (s0 < lo_d) atomicMax(&S.first, 2u * t + 1u);  // (bins up to 2 t stay)
            if (s1 < lo_d) atomicMax(&S.first, 2u * t + 2u);
            if (s0 >= hi_d) atomicMin(&S.second, 2u * t);
            if (s1 >= hi_d) atomicMin(&S.second, 2u * t + 1u);
            __syncthreads();
            const uint32_t b_lo = min(S.first, S.second), b_hi = S.second;  // the uncertain bins
            // exact masses: of what lies above them, and of 2048 finer bins
            __syncthreads();
            for (uint32_t i = t; i < SAMPLE_BINS; i += SAMPLE_THREADS) {
                S.fine.mass[i] = 0ull;
                S.fine.count[i] = 0u;
            }
            __syncthreads();
            const float f_lo = (float)b_lo * mid, f_scale = (SAMPLE_BINS - 1u) / ((float)(b_hi + 1u - b_lo) * mid);
            auto fine = [&](float y) { return (uint32_t)fminf(fmaxf((-y - f_lo) * f_scale, 0.f), (float)(SAMPLE_BINS - 1u)); };
            u64 above = 0;
            for (uint32_t i = i0; i < i1; i++) {
                const float y = R.order(xs[i]);
                const uint32_t b = R.bin(y);
                if (b > b_hi || !cut.keeps(logit_key(xs[i]), base + i)) continue;
                const u64 w = R.steps(y);
                if (b < b_lo) {
                    above += w;
                } else {
                    const uint32_t f = fine(y);
                    atomicAdd(&S.fine.count[f], 1u);
                    uint32_t *half = reinterpret_cast<uint32_t *>(&S.fine.mass[f]);
                    const uint32_t low = (uint32_t)w, was = atomicAdd(half, low);
                    const uint32_t high = (uint32_t)(w >> 32) + (was + low < was);  // (two adds that carry: exact in any order)
                    if (high) atomicAdd(half + 1, high);
                }
            }
            above = R.sum(above);  // (its barrier also ends the histogram)
            u64 g0 = 0, g1 = 0;
            uint32_t q0 = 0, q1 = 0;
            for (uint32_t r = 0; r < C; r++) {
                const ulonglong2 g = reinterpret_cast<const ulonglong2 *>(cl.map_shared_rank(&S.fine.mass[0], r))[t];
                const uint2 q = reinterpret_cast<const uint2 *>(cl.map_shared_rank(&S.fine.count[0], r))[t];
                g0 += g.x;
                g1 += g.y;
                q0 += q.x;
                q1 += q.y;
            }
            u64 g_all;
            const u64 m0 = above + R.before(g0 + g1, g_all), m1 = m0 + g0;
            // the last finer bin with tokens before which the mass is below `need`
            if (t == 0) S.first = 0u;
            __syncthreads();
            if (q0 && ((double)m0 < need || m0 == 0ull)) atomicMax(&S.first, 2u * t + 1u);
            if (q1 && ((double)m1 < need || m1 == 0ull)) atomicMax(&S.first, 2u * t + 2u);
            __syncthreads();
            if (S.first > 0u) {  // (0: no token in the uncertain bins, nothing to cut)
                const uint32_t fb = S.first - 1u;
                __syncthreads();
                if (fb / 2u == t) {
                    S.found[0] = fb & 1u ? m1 : m0;
                    S.second = fb & 1u ? q1 : q0;
                }
                cl.sync();  // every block has read the others' masses: the lists may take their place
                const u64 mass_above = S.found[0];
                const uint32_t n_fine = S.second;
                const Cut old = cut;
                auto in = [&](float v, uint32_t i) {
                    const float y = R.order(v);
                    const uint32_t b = R.bin(y);
                    return b >= b_lo && b <= b_hi && fine(y) == fb && old.keeps(logit_key(v), i);
                };
                if (n_fine <= SAMPLE_CAP) {
                    __syncthreads();
                    if (t == 0) S.n_list = 0u;
                    __syncthreads();
                    for (uint32_t i = i0; i < i1; i++)
                        if (in(xs[i], base + i)) S.list.e[atomicAdd(&S.n_list, 1u)] = (u64)(~logit_key(xs[i])) << 32 | (base + i);
                    cl.sync();
                    if (rank == 0) {
                        uint32_t n = S.n_list;
                        for (uint32_t r = 1; r < C; r++) {
                            const uint32_t kk = *cl.map_shared_rank(&S.n_list, r);
                            const u64 *src = cl.map_shared_rank(&S.list.e[0], r);
                            for (uint32_t i = t; i < kk && n + i < SAMPLE_CAP; i += SAMPLE_THREADS) S.list.e[n + i] = src[i];
                            n += kk;
                        }
                        n = min(n, SAMPLE_CAP);
                        __syncthreads();
                        R.sort_list(n);
                        u64 e[2], w[2], dummy;
                        for (int j = 0; j < 2; j++) {
                            const uint32_t i = 2u * t + j;
                            e[j] = i < n ? S.list.e[i] : 0ull;
                            w[j] = i < n ? R.steps(R.order(key_logit(~(uint32_t)(e[j] >> 32)))) : 0ull;
                        }
                        const u64 p0 = mass_above + R.before(w[0] + w[1], dummy), p1 = p0 + w[0];
                        // the last token before which the mass is below `need`
                        if (t == 0) S.first = 0u;
                        __syncthreads();
                        if (2u * t < n && ((double)p0 < need || p0 == 0ull)) atomicMax(&S.first, 2u * t);
                        if (2u * t + 1u < n && (double)p1 < need) atomicMax(&S.first, 2u * t + 1u);
                        __syncthreads();
                    }
                    const u64 e = rank == 0 ? S.list.e[S.first] : 0ull;
                    cut = told(rank == 0 && t == 0, ~(uint32_t)(e >> 32), (uint32_t)e);
                } else {  // the least key above which the mass is below `need`, then how many of its equals
                    uint32_t lo, hi;
                    key_range(in, lo, hi);
                    while (lo < hi) {
                        const uint32_t mid_key = lo + (hi - lo) / 2u;
                        u64 w = 0;
                        for (uint32_t i = i0; i < i1; i++)
                            if (logit_key(xs[i]) > mid_key && in(xs[i], base + i)) w += R.steps(R.order(xs[i]));
                        if ((double)(mass_above + R.sum(w)) < need) hi = mid_key; else lo = mid_key + 1u;
                    }
                    u64 v[2] = {0ull, 0ull};
                    for (uint32_t i = i0; i < i1; i++)
                        if (in(xs[i], base + i)) {
                            const uint32_t key = logit_key(xs[i]);
                            if (key > lo) v[0] += R.steps(R.order(xs[i]));
                            v[1] += key == lo;
                        }
                    R.fold(v, add);
                    const u64 w1 = R.steps(R.order(key_logit(lo))), s = mass_above + v[0];
                    // the j-th equal (from 0) stays if s + j w1 < need
                    double j = w1 ? ceil((need - (double)s) / (double)w1) : (double)v[1];
                    j = fmin(fmax(j, 1.0), (double)v[1]);
                    cut = Cut{lo, tie_index(lo, old, (u64)j)};
                }
            }
        }
    }

    // ---- the draw, in index order
    auto value = [&](uint32_t i) -> u64 {
        const float v = xs[i], y = R.order(v);
        if (y < -SAMPLE_ORDERS || !cut.keeps(logit_key(v), base + i)) return 0ull;
        if (R.min_p > 0.f && v != m && exp2f(y) < R.min_p) return 0ull;
        return R.steps(y);
    };
    u64 mine = 0, total;
    for (uint32_t i = i0; i < i1; i++) mine += value(i);
    const u64 bef = R.before_all(mine, total), target = target_of(total);
    if (bef <= target && bef + mine > target) {
        u64 s = bef;
        for (uint32_t i = i0; i < i1; i++) {
            const u64 w = value(i);
            s += w;
            if (s > target) {
                write(base + i, w, total);
                break;
            }
        }
    }
    cl.sync();
}

// Blocks to a row. More blocks shorten every pass, a cluster barrier costs the same; the row has to fit their shared memory.
static uint32_t sample_cluster(uint32_t n, uint32_t rows, size_t smem_optin) {
    const size_t room = (smem_optin - sizeof(SampleShared) - 1024) / 4;
    uint32_t c = 1;
    while (c < 8 && (size_t)(n + c - 1) / c > (rows * c >= 296 ? room : 4096)) c *= 2;
    while (c < SAMPLE_MAX_CLUSTER && (size_t)((n + c - 1) / c + 3) > room) c *= 2;
    return c;
}

cudaError_t launch_sample(strix_cuda *h, const float *d_x, uint32_t n, size_t stride, uint32_t rows, const strix_sample_params &p,
                          const float *d_u, uint32_t *d_ids, float *d_probs, cudaStream_t stream) {
    const uint32_t c = sample_cluster(n, rows, h->smem_optin);
    const uint32_t per = ((n + c - 1) / c + 3u) & ~3u;
    const SampleArgs A{d_x, stride, n, per, p, d_u, d_ids, d_probs};
    const size_t smem = sizeof(SampleShared) + (size_t)per * 4;
    cudaError_t e = cudaFuncSetAttribute(sample_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e == cudaSuccess && c > 8) e = cudaFuncSetAttribute(sample_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(rows * c);
    cfg.blockDim = dim3(SAMPLE_THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = c;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    ProfScope prof(h, stream, "sample");
    return cudaLaunchKernelEx(&cfg, sample_kernel, A);
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
