// kv8_attn.h -- the attention over the 8-bit paged cache, as the entry point of kv8.cu plans and
// launches it.
#pragma once

#include <algorithm>
#include <atomic>

#include "kv8.cuh"

namespace pox {

constexpr int kStepWarps = 4;  // warps of a CTA of the step kernel
// What an item of it costs besides its pages, in pages (8, 16, 32: 20.9, 21.0, 22.2 us for 128 sequences of 50 to 3000
// tokens; long contexts do not mind).
constexpr int kItemUnits = 8;

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

// How the step kernel divides its work (see there).
struct Kv8StepPlan {
    int tiles = 1;      // of 8 rows each in an item
    int grid = 1;       // CTAs, each with an equal run of units (pages of an item)
    int min_units = 1;  // of a run
    int most_rows = 0x7fffffff;  // sequences of more rows are left to the prompt kernel
    int device = 0;
    float* part = nullptr;        // [grid][2][8 tiles][hd + 2]
    uint32_t* tickets = nullptr;  // [grid], zero between launches
    // Bounds over all plans: CTAs of an SM, and the two places of each times its rows times their floats.
    static constexpr int kNarrow = 4, kWide = 3, kTwoTiles = 2;
    static int most_ctas(int sms) { return kNarrow * sms; }
    static size_t most_part_bytes(int sms) {
        return (size_t)sms * 2 * sizeof(float) *
               std::max({kNarrow * 8 * (64 + 2), kWide * 8 * (128 + 2), kTwoTiles * 16 * (128 + 2)});
    }
};

inline Kv8StepPlan kv8_step_plan(const Kv8Batch& b, int kvh, int hd, int G, int sms, int most_rows) {
    Kv8StepPlan p;
    p.most_rows = most_rows;
    const long long rows = std::min((long long)b.max_rows * G, (long long)most_rows);
    p.tiles = rows <= 8 ? 1 : 2;
    p.min_units = 2 * kStepWarps;  // two pages for each warp: fewer, and the joining costs more than it gives
    // as many CTAs as are resident at once, or as there is work for
    const long long items = (long long)b.seqs * kvh * ((rows + 8 * p.tiles - 1) / (8 * p.tiles));
    const long long pages = std::max<long long>((b.max_ctx + kPage - 1) / kPage, 1);
    const long long most = (long long)std::min((double)items * (pages + kItemUnits) / p.min_units + 1, 1e9);
    p.grid = (int)std::min<long long>((p.tiles > 1 ? p.kTwoTiles : hd == 128 ? p.kWide : p.kNarrow) * sms, most);
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
// CTAs of the prompt kernel: one for each tile item and kv head, and the one that checks the batch.
inline unsigned long long kv8_prompt_grid(const Kv8Batch& b, int kvh, int G) {
    return b.row_starts ? ((unsigned long long)b.rows * G + 255ull * b.seqs) / 256 * kvh + 1
                        : (unsigned long long)b.seqs * kvh;
}
// Sequences of at least min_rows rows, head dims 64 and 128, f16 and bf16.
template <int HD, typename T>
cudaError_t launch_kv8_prompt(const Kv8Attn<T>& a, int min_rows, int device, cudaStream_t st);

}  // namespace pox
