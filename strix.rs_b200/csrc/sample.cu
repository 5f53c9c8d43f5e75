// Drawing a token from logits: temperature, top-k, top-p, min-p and the inverse of the distribution function at a given
// number. Contract: include/strix_serve.h. Stands beside the greedy argmax (argmax.cu).
//
// Everything is a question about the order (logit, then lower index first) and about sums of weights, so nothing is sorted:
// the sets that top-k and top-p keep are each {key > t} and the first `quota` of {key == t} for some key t, found by
// counting and summing over thresholds. Weights are summed as 64-bit integers in steps of 2^-40: the sums do
// not depend on their order, hence neither does the draw.
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "kv_pages.cuh"

namespace strix {

typedef unsigned long long u64;

struct SampleArgs {
    const float *x;
    size_t stride;
    uint32_t n;
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
constexpr uint32_t KEY_MINUS_INF = 0x007fffffu;

constexpr int SAMPLE_THREADS = 1024;

template <typename T>
__device__ T block_sum(T v, T *red) {
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if ((threadIdx.x & 31u) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    T s = 0;
    for (int w = 0; w < SAMPLE_THREADS / 32; w++) s += red[w];
    return s;
}

// One block for each row; thresholds by bisection over the 32 bits of a key.
__global__ void __launch_bounds__(SAMPLE_THREADS) sample_kernel(const SampleArgs A) {
    __shared__ u64 red[SAMPLE_THREADS / 32], part[SAMPLE_THREADS];
    __shared__ float redf[SAMPLE_THREADS / 32];
    __shared__ uint32_t found;
    const uint32_t row = blockIdx.x, t = threadIdx.x, n = A.n;
    const float *x = A.x + (size_t)row * A.stride;
    const float temp = A.p.d_temperature ? A.p.d_temperature[row] : 1.f;
    const int top_k = A.p.d_top_k ? A.p.d_top_k[row] : 0;
    const float top_p = A.p.d_top_p ? A.p.d_top_p[row] : 1.f, min_p = A.p.d_min_p ? A.p.d_min_p[row] : 0.f;
    const bool greedy = !(temp > 0.f);
    uint32_t k = greedy ? 1u : top_k > 0 && (uint32_t)top_k < n ? (uint32_t)top_k : n;
    float m = -INFINITY;
    for (uint32_t i = t; i < n; i += SAMPLE_THREADS) m = fmaxf(m, x[i]);
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if ((t & 31u) == 0) redf[t >> 5] = m;
    __syncthreads();
    for (int w = 0; w < SAMPLE_THREADS / 32; w++) m = fmaxf(m, redf[w]);
    if (m == -INFINITY) {
        if (t == 0) {
            A.ids[row] = 0u;
            if (A.probs) A.probs[row] = 0.f;
        }
        return;
    }
    const float c = greedy ? 1.f : 1.f / temp;
    auto weight = [&](float v) -> float { return v != v ? 0.f : v == m ? 1.f : m == INFINITY ? 0.f : expf((v - m) * c); };
    auto fixed = [&](float w) -> u64 { return __float2ull_rn(w * 1099511627776.f); };
    uint32_t tk = 0, quota = 0xffffffffu;  // kept: key > tk, and the first `quota` with key == tk
    if (k < n) {
        uint32_t lo = 0;  // the largest key that at least k logits reach
        for (int b = 31; b >= 0; b--) {
            const uint32_t c2 = lo | 1u << b;
            u64 cnt = 0;
            for (uint32_t i = t; i < n; i += SAMPLE_THREADS) cnt += logit_key(x[i]) >= c2;
            if (block_sum(cnt, red) >= k) lo = c2;
        }
        u64 above = 0;
        for (uint32_t i = t; i < n; i += SAMPLE_THREADS) above += logit_key(x[i]) > lo;
        above = block_sum(above, red);
        tk = lo;
        quota = k - (uint32_t)above;
    }
    const uint32_t per = (n + SAMPLE_THREADS - 1) / SAMPLE_THREADS, i0 = min(n, t * per), i1 = min(n, i0 + per);
    // the index of the quota-th logit equal to the threshold
    uint32_t last = n;
    auto limit = [&] {
        if (quota == 0xffffffffu) return;
        u64 cnt = 0;
        for (uint32_t i = i0; i < i1; i++) cnt += logit_key(x[i]) == tk;
        __syncthreads();
        part[t] = cnt;
        if (t == 0) found = n;
        __syncthreads();
        u64 before = 0;
        for (uint32_t j = 0; j < t; j++) before += part[j];
        if (before < quota && before + cnt >= quota) {
            u64 q = before;
            for (uint32_t i = i0; i < i1; i++)
                if (logit_key(x[i]) == tk && ++q == quota) {
                    found = i;
                    break;
                }
        }
        __syncthreads();
        last = found;
    };
    limit();
    auto kept = [&](uint32_t i, uint32_t key) { return key > tk || (key == tk && i <= last); };
    if (!greedy && top_p < 1.f) {
        u64 total = 0;
        for (uint32_t i = t; i < n; i += SAMPLE_THREADS) {
            const float v = x[i];
            if (kept(i, logit_key(v))) total += fixed(weight(v));
        }
        total = block_sum(total, red);
        const double need = (double)top_p * (double)total;
        // the largest key such that the kept weights strictly above it sum to less than `need`; its own go by quota
        uint32_t lo = tk;
        if (top_p > 0.f) {
            uint32_t a = tk, b = logit_key(m);  // answer in [a, b]: the least key whose "above" sum is below need
            while (a < b) {
                const uint32_t mid = a + (b - a) / 2;
                u64 s = 0;
                for (uint32_t i = t; i < n; i += SAMPLE_THREADS) {
                    const float v = x[i];
                    const uint32_t key = logit_key(v);
                    if (key > mid && kept(i, key)) s += fixed(weight(v));
                }
                s = block_sum(s, red);
                if ((double)s < need) b = mid; else a = mid + 1;
            }
            lo = a;
        } else {
            lo = logit_key(m);
        }
        u64 s = 0, eq = 0, w1 = 0;
        for (uint32_t i = t; i < n; i += SAMPLE_THREADS) {
            const float v = x[i];
            const uint32_t key = logit_key(v);
            if (key > lo && kept(i, key)) s += fixed(weight(v));
            if (key == lo && kept(i, key)) {
                eq++;
                w1 += fixed(weight(v));
            }
        }
        s = block_sum(s, red);
        eq = block_sum(eq, red);
        w1 = block_sum(w1, red);
        uint32_t q = 0;
        if (eq) {
            const u64 one = w1 / eq;
            // ties kept: the j-th (from 0) stays if s + j * one < need
            double j = one ? ceil((need - (double)s) / (double)one) : (double)eq;
            if (s == 0 && j < 1.) j = 1.;
            q = (uint32_t)fmin(fmax(j, 0.), (double)eq);
        }
        const uint32_t old_t = tk, old_q = quota;
        tk = lo;
        quota = lo == old_t ? min(q, old_q) : q;
        last = n;
        limit();
        if (quota == 0u) {  // no tie stays
            last = 0;
            tk = lo + 1u;
            quota = 0xffffffffu;
            last = n;
        }
    }
    u64 mine = 0;
    auto value = [&](uint32_t i) -> u64 {
        const float v = x[i];
        if (!kept(i, logit_key(v))) return 0;
        const float w = weight(v);
        return w >= min_p || v == m ? fixed(w) : 0;
    };
    for (uint32_t i = i0; i < i1; i++) mine += value(i);
    __syncthreads();
    part[t] = mine;
    if (t == 0) found = 0;
    __syncthreads();
    u64 before = 0, total = 0;
    for (uint32_t j = 0; j < SAMPLE_THREADS; j++) {
        if (j < t) before += part[j];
        total += part[j];
    }
    float u = A.u[row];
    u = u >= 0.f ? u : 0.f;
    u64 target = (u64)((double)u * (double)total);
    if (target >= total) target = total - 1;
    if (before <= target && before + mine > target) {
        u64 s = before;
        for (uint32_t i = i0; i < i1; i++) {
            s += value(i);
            if (s > target) {
                A.ids[row] = i;
                if (A.probs) A.probs[row] = (float)((double)value(i) / (double)total);
                break;
            }
        }
    }
}

cudaError_t launch_sample(strix_cuda *h, const float *d_x, uint32_t n, size_t stride, uint32_t rows, const strix_sample_params &p,
                          const float *d_u, uint32_t *d_ids, float *d_probs, cudaStream_t stream) {
    ProfScope prof(h, stream, "sample");
    const SampleArgs A{d_x, stride, n, p, d_u, d_ids, d_probs};
    sample_kernel<<<rows, SAMPLE_THREADS, 0, stream>>>(A);
    return cudaGetLastError();
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
