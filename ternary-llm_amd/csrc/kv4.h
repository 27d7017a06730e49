// The 4-bit paged key/value cache as the kernels see it (layout: include/tllm_ternary.h, tllm_kv4_cache).
#pragma once
#include <type_traits>

#include "common.h"

namespace tllm {

constexpr int kKvGroup = TLLM_KV4_GROUP;  // dims that share a step and a minimum

// Offsets inside one (page, kv head) block, in 32-bit words. A page's blocks of all heads lie next to each other.
__host__ __device__ __forceinline__ size_t kv4_code_words(int page_size, int head_dim) { return (size_t)page_size * (head_dim / 8); }
__host__ __device__ __forceinline__ size_t kv4_scale_words(int page_size, int head_dim) {
    return (size_t)page_size * (head_dim / kKvGroup);
}

// Sequence of a row of the batch: the number of sequences that end at or before it (`batch`: behind the last one). All
// lanes of the wave pass the same row. The starts are the caller's data: whatever they hold, the result is in 0..batch.
__device__ __forceinline__ int kv4_find_sequence(const int *__restrict__ starts, int batch, int row) {
    int n = 0;
    for (int base = 0; base < batch; base += kWave) {
        const int i = base + (int)(threadIdx.x & (kWave - 1));
        const unsigned long long before = __ballot(i < batch && starts[i + 1] <= row);
        n += __popcll(before);
        if (before != ~0ull) break;
    }
    return n;
}

// Position of row `row` of sequence `seq` (< batch), or -1 where it has none: the rows of a sequence are its last cached
// tokens. -1 also for rows that do not belong to the sequence (starts that do not begin at 0) and behind the page table.
__device__ __forceinline__ int kv4_position(const Kv4Batch &b, int seq, int row, int capacity) {
    if (b.starts[seq] > row) return -1;
    const long long pos = (long long)b.lengths[seq] - b.starts[seq + 1] + row;
    return pos >= 0 && pos < capacity ? (int)pos : -1;
}

}  // namespace tllm
