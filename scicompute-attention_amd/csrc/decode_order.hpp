// The longest-first schedule of large ragged decode batches (decode.hip, decode8.hip).
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace sca_hip {
namespace {

// Longest-first schedule of ragged batches larger than kRankBatch: entry r of `order` is
// (b, len_b) for the sequence of rank r (descending length, ties by index). The MFMA kernels
// take the sequence of grid row z from entry z, so the longest sequences are dispatched first.
constexpr int kMaxOrderedBatch = 8192;

__global__ __launch_bounds__(256) void decode_order_kernel(const int32_t* seq_lens, int batch,
                                                           int32_t* order) {
    const int b = blockIdx.x * 256 + threadIdx.x;
    if (b >= batch) return;
    const int mine = seq_lens[b];
    int rank = 0;
    for (int j = 0; j < batch; ++j) {
        const int other = seq_lens[j];
        rank += (other > mine) | ((other == mine) & (j < b));
    }
    order[2 * rank] = b;
    order[2 * rank + 1] = mine;
}

}  // namespace
}  // namespace sca_hip
