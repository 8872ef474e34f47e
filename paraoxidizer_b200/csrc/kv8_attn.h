// kv8_attn.h -- the attention over the 8-bit paged cache, as the entry point of kv8.cu plans and
// launches it.
#pragma once

#include <algorithm>
#include <atomic>

#include "kv8.cuh"

namespace pox {

constexpr int kStepWarps = 4;        // warps of a CTA of the step kernel
constexpr int kStepMostPages = 128;  // pages of a split: one lane of a warp holds the entry of each of its pages

template <typename T>
struct Kv8Attn {
    Kv8Cache c;
    Kv8Batch b;
    RowsView<const T> q;
    RowsView<T> out;
    int G;        // query heads per kv head
    float scale;  // of the scores, times log2 e
    int vec;      // q and out take 4-element loads and stores
    int* err;
};

// How the step kernel splits its work: row tiles of a (sequence, kv head) pair and splits of the context.
struct Kv8StepPlan {
    int row_tiles = 1, splits = 1, pages_per_split = kStepMostPages;
    float* part = nullptr;        // [items][splits][rows of a tile][hd + 2] when splits > 1
    uint32_t* tickets = nullptr;  // [items], zero between launches
    size_t items = 0;
    int device = 0;
    int most_rows = 0x7fffffff;  // sequences of more rows are left to the prompt kernel
    int tiles = 1;  // of 8 rows each in a CTA
};

inline Kv8StepPlan kv8_step_plan(const Kv8Batch& b, int kvh, int G, int sms, int most_rows) {
    Kv8StepPlan p;
    p.most_rows = most_rows;
    const long long rows = std::min((long long)b.max_rows * G, (long long)most_rows);
    p.tiles = rows <= 8 ? 1 : 2;
    const int rt = 8 * p.tiles;
    p.row_tiles = (int)((rows + rt - 1) / rt);
    p.items = (size_t)b.seqs * kvh * p.row_tiles;
    const long long pages = (b.max_ctx + kPage - 1) / kPage;
    // about four CTAs for each of the three places that an SM has, but two pages at least for each warp
    long long pps = (long long)(p.items * (double)pages / (12.0 * sms));
    pps = std::min<long long>(kStepMostPages, std::max<long long>(pps, 2 * kStepWarps));
    p.splits = (int)std::max<long long>(1, (pages + pps - 1) / pps);
    pps = (pages + p.splits - 1) / p.splits;
    p.pages_per_split = (int)std::max<long long>(kStepWarps, (pps + kStepWarps - 1) / kStepWarps * kStepWarps);
    return p;
}

// Allows the kernel `bytes` of dynamic shared memory, once per device (`done`: a bit for each).
template <typename F>
inline cudaError_t kv8_smem_once(F* kernel, int bytes, int device, std::atomic<uint32_t>& done) {
    const uint32_t bit = device < 32 ? 1u << device : 0u;
    if (done.load(std::memory_order_relaxed) & bit) return cudaSuccess;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_relaxed);
    return e;
}

// Sequences of at most p.most_rows rows (tokens times query heads of the group), any head dim.
template <int HD, typename T>
cudaError_t launch_kv8_step(const Kv8Attn<T>& a, const Kv8StepPlan& p, cudaStream_t st);
// Sequences of at least min_rows rows, head dims 64 and 128, f16 and bf16.
template <int HD, typename T>
cudaError_t launch_kv8_prompt(const Kv8Attn<T>& a, int min_rows, int device, cudaStream_t st);

}  // namespace pox
