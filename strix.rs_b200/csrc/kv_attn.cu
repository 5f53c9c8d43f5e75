// Attention over a paged KV cache, ragged batches, grouped-query heads. Contract: include/strix_serve.h.
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "kv_pages.cuh"

namespace strix {

struct PagedAttnArgs {
    PagedView V;
    const float *q;
    float *out;
    size_t ld_q, ld_out;
    uint32_t n_heads, group, window;
    float scale;
};

constexpr uint32_t PA_TILE = 128;

__device__ __forceinline__ float cached(const uint8_t *head, float s, int type, size_t i) {
    if (type == STRIX_KV_F16) return __half2float(reinterpret_cast<const __half *>(head)[i]);
    return e4m3x2_to_f32(head[i]).x * s;
}

// One block for each (row, head): scores of PA_TILE tokens, one to a thread, then the weighted sum, two dimensions to a thread.
__global__ void __launch_bounds__(PA_TILE) paged_attn_kernel(const PagedAttnArgs A) {
    __shared__ float q[256], p[PA_TILE], red[PA_TILE / 32];
    __shared__ int pg[PA_TILE];
    const PagedView &V = A.V;
    const uint32_t row = blockIdx.x, hh = blockIdx.y, t = threadIdx.x, hd = V.head_dim, kvh = hh / A.group;
    bool bad = false;
    uint32_t first, end;
    const uint32_t s = seq_of_row(V, row, first, end, bad);
    if (s >= V.n_seq) {
        report_bad(V, bad && t == 0);
        return;
    }
    const int ctx = V.ctx[s];
    const uint64_t cap = (uint64_t)V.pages_ld * V.page_tokens;
    uint64_t len = ctx < 0 ? 0 : (uint64_t)ctx + (row - first) + 1u;
    uint64_t tok0 = A.window && len > A.window ? len - A.window : 0u;
    if (len > cap) {
        len = cap;
        bad = true;
    }
    for (uint32_t i = t; i < hd; i += PA_TILE) q[i] = A.q[(size_t)row * A.ld_q + (size_t)hh * hd + i] * A.scale;
    float m = -INFINITY, sum = 0.f, o0 = 0.f, o1 = 0.f;
    for (uint64_t base = tok0; base < len; base += PA_TILE) {
        const uint64_t tok = base + t;
        __syncthreads();
        float x = -INFINITY;
        pg[t] = -1;
        if (tok < len) {
            const int page = V.pages[(size_t)s * V.pages_ld + (tok >> V.page_shift)];
            if (page < 0 || (uint32_t)page >= V.n_pages) {
                bad = true;
            } else {
                pg[t] = page;
                const uint8_t *head = V.k + (size_t)page * V.page_bytes + (size_t)kvh * V.head_bytes;
                const float ks = V.type == STRIX_KV_F16 ? 1.f : V.k_scale[(size_t)page * V.n_kv + kvh];
                const size_t at = (size_t)((uint32_t)tok & (V.page_tokens - 1u)) * hd;
                x = 0.f;
                for (uint32_t i = 0; i < hd; i++) x = fmaf(q[i], cached(head, ks, V.type, at + i), x);
            }
        }
        float mt = x;
        for (int o = 16; o > 0; o >>= 1) mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, o));
        if ((t & 31u) == 0) red[t >> 5] = mt;
        __syncthreads();
        for (uint32_t w = 0; w < PA_TILE / 32; w++) mt = fmaxf(mt, red[w]);
        const float mn = fmaxf(m, mt), f = mn == -INFINITY ? 1.f : expf(m - mn);
        p[t] = pg[t] < 0 ? 0.f : expf(x - mn);
        m = mn;
        __syncthreads();
        sum *= f;
        o0 *= f;
        o1 *= f;
        for (uint32_t j = 0; j < PA_TILE; j++) {
            if (pg[j] < 0) continue;
            const uint8_t *head = V.v + (size_t)pg[j] * V.page_bytes + (size_t)kvh * V.head_bytes;
            const float vs = V.type == STRIX_KV_F16 ? 1.f : V.v_scale[(size_t)pg[j] * V.n_kv + kvh];
            const size_t at = (size_t)((uint32_t)(base + j) & (V.page_tokens - 1u)) * hd;
            sum += p[j];
            if (t < hd) o0 = fmaf(p[j], cached(head, vs, V.type, at + t), o0);
            if (t + PA_TILE < hd) o1 = fmaf(p[j], cached(head, vs, V.type, at + t + PA_TILE), o1);
        }
    }
    float *o = A.out + (size_t)row * A.ld_out + (size_t)hh * hd;
    const float inv = sum == 0.f ? 0.f : 1.0f / sum;
    if (t < hd) o[t] = o0 * inv;
    if (t + PA_TILE < hd) o[t + PA_TILE] = o1 * inv;
    report_bad(V, bad);
}

}  // namespace strix

using namespace strix;

extern "C" size_t strix_cuda_attn_pages_workspace(strix_cuda *h, const strix_kv_pages *cache, const strix_kv_batch *batch,
                                                  uint32_t n_heads) {
    if (!h) return 0;
    h->err.clear();
    PagedView V;
    if (serve_check(h, "attn_pages_workspace", cache, batch, &V) != 1) return 0;
    if (n_heads == 0 || n_heads > 65535u || n_heads % V.n_kv) return 0;
    return 256;
}

extern "C" int strix_cuda_attn_pages_dev(strix_cuda *h, const strix_kv_pages *cache, const strix_kv_batch *batch, uint32_t n_heads,
                                         const float *d_q, size_t ld_q, float scale, uint32_t window, float *d_out, size_t ld_out,
                                         void *d_work, size_t work_bytes, void *stream) {
    if (!h) return -1;
    h->err.clear();
    const char *who = "attn_pages";
    PagedAttnArgs A{};
    const int rc = serve_check(h, who, cache, batch, &A.V);
    if (rc != 1) return rc;
    if (n_heads == 0 || n_heads > 65535u || n_heads % A.V.n_kv) return 0;
    const size_t qd = (size_t)n_heads * A.V.head_dim;
    A.ld_q = ld_q ? ld_q : qd;
    A.ld_out = ld_out ? ld_out : qd;
    if (A.ld_q < qd || A.ld_out < qd) return serve_fail(h, who, "a row stride is smaller than a row");
    if (A.V.n_seq == 0 || A.V.n_rows == 0) return 1;
    if (!d_q || !d_out) return serve_fail(h, who, "d_q or d_out missing");
    if (!d_work || (reinterpret_cast<uintptr_t>(d_work) & 255u)) return serve_fail(h, who, "d_work must be 256-byte aligned");
    if (work_bytes < strix_cuda_attn_pages_workspace(h, cache, batch, n_heads)) return serve_fail(h, who, "work_bytes too small");
    A.q = d_q;
    A.out = d_out;
    A.n_heads = n_heads;
    A.group = n_heads / A.V.n_kv;
    A.window = window;
    A.scale = scale;
    DeviceGuard dev(h->device);
    if (dev.err != cudaSuccess) return serve_fail(h, who, cudaGetErrorString(dev.err));
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    ProfScope prof(h, s, "attn_pages");
    paged_attn_kernel<<<dim3(A.V.n_rows, n_heads), PA_TILE, 0, s>>>(A);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return serve_fail(h, who, cudaGetErrorString(e));
    return 1;
}
