// kv8_attn.h -- the attention over the 8-bit paged cache, as the entry point of kv8.cu launches it.
#pragma once

#include "kv8.cuh"

namespace pox {

template <typename T>
struct Kv8Attn {
    Kv8Cache c;
    Kv8Batch b;
    RowsView<const T> q;
    RowsView<T> out;
    int G;        // query heads per kv head
    float scale;  // of the scores
    int* err;
};

template <int HD, typename T>
cudaError_t launch_kv8_attention(const Kv8Attn<T>& a, cudaStream_t st);

}  // namespace pox
