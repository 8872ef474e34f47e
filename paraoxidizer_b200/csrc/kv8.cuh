// kv8.cuh -- what the kernels of the 8-bit paged KV cache share: the page layout, views of rows, the
// ragged batch and the rotation, as include/pox_cuda.h describes them.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "common.cuh"
#include "gemv.cuh"
#include "model.h"

namespace pox {

// Byte of (token t, dim d) within the page of one kv head. K rows of 128 dims swap their 64-byte halves
// at odd tokens: a warp's 16-byte reads of two neighbouring tokens then cover all 32 banks.
template <int HD>
__host__ __device__ __forceinline__ constexpr int kv8_k_off(int t, int d) {
    return t * HD + (HD == 128 ? d ^ ((t & 1) << 6) : d);
}
template <int HD>
__host__ __device__ __forceinline__ constexpr int kv8_v_off(int t, int d) {
    return kPage * HD + d * kPage + t;
}

struct Kv8Cache {
    int8_t* pages;
    float* scales;
    uint32_t num_blocks;
    int kvh;
};

struct Kv8Batch {
    const uint32_t* row_starts;  // NULL: one row each
    const uint32_t* ctx_lens;
    const int32_t* btab;
    uint32_t seqs, rows, max_rows, max_ctx, mbps;
    const uint32_t* ones;  // row_starts as given where they have to be 0, 1, 2, .. (row_starts is then NULL)
};

template <typename T>
struct RowsView {
    T* data;
    size_t row, head;  // strides in elements
    __device__ __forceinline__ T* at(size_t r, size_t h) const { return data + r * row + h * head; }
};

struct RopeView {
    const float2* table;  // [positions][rot / 2]
    uint32_t positions;
    int rot;   // 0: none
    int half;  // pairs (i, i + rot / 2), else (2 i, 2 i + 1)
};

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) {
    return x;
}
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) {
    return __float2half_rn(x);
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) {
    return __float2bfloat16_rn(x);
}

// One pair turned by (cos, sin): separate products and sums, so that the result does not depend on
// which kernel contracts them (the quantised bytes are then the same everywhere).
__device__ __forceinline__ float2 rope_turn(float a, float b, float2 cs) {
    return make_float2(__fsub_rn(__fmul_rn(a, cs.x), __fmul_rn(b, cs.y)),
                       __fadd_rn(__fmul_rn(a, cs.y), __fmul_rn(b, cs.x)));
}

// Rows, context and first row of sequence s; false (reported) if it breaks the batch's bounds or its row starts do not
// fit: they begin at 0, end at the batch's rows and, in a batch of one row each, count up.
struct SeqSpan {
    uint32_t r0;
    int n, ctx;
};
__device__ __forceinline__ bool seq_span(const Kv8Batch& b, uint32_t s, SeqSpan& o, int* err) {
    const uint32_t* starts = b.row_starts ? b.row_starts : b.ones;
    const uint32_t r0 = starts ? starts[s] : s, r1 = starts ? starts[s + 1] : s + 1, ctx = b.ctx_lens[s];
    o.r0 = r0, o.n = (int)(r1 - r0), o.ctx = (int)ctx;
    const bool fits = b.row_starts ? (s || !r0) && (s + 1 < b.seqs || r1 == b.rows) && r1 >= r0 && r1 <= b.rows &&
                                         r1 - r0 <= b.max_rows
                                   : r0 == s && r1 == s + 1;
    if (!fits || ctx > b.max_ctx) {
        atomicOr(err, kErrBatch);
        return false;
    }
    return true;
}

// (a long division is a hundred instructions)
__device__ __forceinline__ unsigned long long div_u64(unsigned long long a, uint32_t b) {
    return a >> 32 ? a / b : (uint32_t)a / b;
}

// A page of the batch: sequence s owns page items (row_starts[s] + 30 s) / 16 .. (a bound of the pages that
// its n rows touch: n rows reach at most (n + 30) / 16 pages, in closed form, so no scan over the sequences).
__device__ __forceinline__ uint32_t page_base(const Kv8Batch& b, uint32_t s) {
    return !b.row_starts ? s : (uint32_t)(((unsigned long long)b.row_starts[s] + 30ull * s) / 16);
}

// Items of a ragged batch are found through row_starts, where a sequence of fewer than no rows has none: the last CTA
// looks at every sequence instead (true), so that each one at fault is reported.
__device__ __forceinline__ bool check_batch(const Kv8Batch& b, int* err) {
    if (!b.row_starts || blockIdx.x != gridDim.x - 1) return false;
    SeqSpan q;
    for (uint32_t s = threadIdx.x; s < b.seqs; s += blockDim.x) seq_span(b, s, q, err);
    return true;
}

// The sequence of item i, the same for the warp: the largest s with base(s) <= i. 32 candidates a round, so two
// dependent loads serve 1024 sequences.
template <typename F>
__device__ __forceinline__ uint32_t find_seq(const Kv8Batch& b, uint32_t i, F&& base) {
    const uint32_t lane = threadIdx.x & 31;
    uint32_t lo = 0, n = b.seqs;  // the answer is in [lo, lo + n)
    while (n > 1) {
        const uint32_t step = (n + 31) / 32, at = lane * step;
        const uint32_t m = __ballot_sync(0xffffffffu, at < n && base(lo + at) <= i), k = m ? 31 - __clz(m) : 0;
        lo += k * step;
        n = min(step, n - k * step);
    }
    return lo;
}

}  // namespace pox
