// Device helpers shared by the kernels over a paged KV cache: which rows a sequence owns, where its tokens live.
#pragma once
#include <cuda_fp16.h>
#include <stdint.h>

#include "common.cuh"
#include "serve.h"

namespace strix {

// Rows [first, end) of sequence s with the offsets clamped into the batch; bad offsets set `bad`.
__device__ __forceinline__ void seq_rows(const PagedView &V, uint32_t s, uint32_t &first, uint32_t &end, bool &bad) {
    const int a = V.row0[s], b = V.row0[s + 1u];
    const int n = (int)V.n_rows;
    const int ca = min(max(a, 0), n), cb = min(max(b, 0), n);
    bad |= ca != a || cb != b || b < a;
    first = (uint32_t)ca;
    end = (uint32_t)max(ca, cb);
}

// The sequence that owns `row`, or n_seq if none does. Called by a whole warp with one row; a 32-way search over row0.
__device__ __forceinline__ uint32_t seq_of_row(const PagedView &V, uint32_t row, uint32_t &first, uint32_t &end, bool &bad) {
    const uint32_t lane = threadIdx.x & 31u;
    uint32_t lo = 0, n = V.n_seq;
    while (n > 1u) {
        const uint32_t step = (n + 31u) / 32u, at = lane * step;
        const bool below = at < n && V.row0[lo + at] <= (int)row;
        const uint32_t mask = __ballot_sync(0xffffffffu, below);
        if (mask == 0u) return V.n_seq;
        const uint32_t k = 31u - __clz(mask);
        lo += k * step;
        n = min(step, n - k * step);
    }
    seq_rows(V, lo, first, end, bad);
    return row >= first && row < end ? lo : V.n_seq;
}

__device__ __forceinline__ void report_bad(const PagedView &V, bool bad) {
    if (bad && V.status) atomicOr(V.status, STATUS_BAD_ARGS);
}

// two e4m3 codes (low byte first) as two f16; exact
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint32_t two) {
    uint32_t h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)two));
    return h;
}
// four e4m3 codes as two pairs of f16, the lower bytes first (the halves of the word are taken apart inside: no shift)
__device__ __forceinline__ void e4m3x4_to_f16x2(uint32_t four, uint32_t &lo, uint32_t &hi) {
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
        : "=r"(lo), "=r"(hi)
        : "r"(four));
}
__device__ __forceinline__ float2 e4m3x2_to_f32(uint32_t two) {
    const uint32_t h = e4m3x2_to_f16x2(two);
    return __half22float2(*reinterpret_cast<const __half2 *>(&h));
}
// round to nearest even, to +-448 beyond that
__device__ __forceinline__ uint32_t f32_to_e4m3x2(float lo, float hi) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ uint32_t f32_to_f16x2(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

}  // namespace strix
