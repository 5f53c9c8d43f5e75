// Internal interface of the serving operators (include/strix_serve.h): kernel arguments and what the host sides share.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include "accel.h"
#include "strix_serve.h"

namespace strix {

// A cache and a batch as the kernels see them; sizes checked and strides resolved on the host (serve_check).
struct PagedView {
    uint8_t *k, *v;
    float *k_scale, *v_scale;
    size_t page_bytes, head_bytes;  // bytes from one page, one KV head of a page, to the next
    uint32_t n_pages, n_kv, page_tokens, page_shift, head_dim;
    int type;
    const int32_t *row0, *ctx, *pages;
    uint32_t n_seq, n_rows, pages_ld;
    uint32_t *status;
};

// Makes the handle's device current for the calling thread while it lives, and puts back what was current before.
struct DeviceGuard {
    int prev = -1;
    bool changed = false;
    cudaError_t err = cudaSuccess;
    explicit DeviceGuard(int device) {
        err = cudaGetDevice(&prev);
        if (err == cudaSuccess && prev != device) {
            err = cudaSetDevice(device);
            changed = err == cudaSuccess;
        }
    }
    ~DeviceGuard() {
        if (changed) cudaSetDevice(prev);
    }
};

int serve_fail(strix_cuda *h, const char *what, const char *why) noexcept;  // sets the error text, returns -1
// 1 and a filled view, 0 = declined, -1 = an argument error (text set)
int serve_check(strix_cuda *h, const char *what, const strix_kv_pages *c, const strix_kv_batch *b, PagedView *v) noexcept;
// One draw per row of d_x (sample.cu); arguments checked by the caller
cudaError_t launch_sample(strix_cuda *h, const float *d_x, uint32_t n, size_t stride, uint32_t rows, const strix_sample_params &p,
                          const float *d_u, uint32_t *d_ids, float *d_probs, cudaStream_t stream);

}  // namespace strix
