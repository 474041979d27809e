// What the kernels over a cache in blocks share: how a launch finds its sequence, and where a token lies.
//
// The cache of a layer. A block holds `block` (16, 32, 64 or 128) consecutive tokens of one sequence, for every head
//   k_codes [blocks, kv_heads, block, D]            int8
//   v_codes [blocks, kv_heads, block / 16, D, 16]   int8, 16 tokens innermost
//   k_scale, v_scale [blocks, kv_heads]             fp32: one scale for a block and head
// block_table [sequences, width] names the blocks of a sequence in order; an entry outside [0, blocks) is no block.
// A call's own tokens are the rows query_start[b] .. query_start[b + 1] - 1 of sequence b (row b where there is no
// query_start), at positions cached[b] on; cached[b] < 0: the sequence takes no part.
#pragma once

#include "llmq_device.h"

namespace llmq {

constexpr int kStrip = 16;   // tokens innermost in the value codes

struct BlockTable {
  const int32_t* entries;
  int64_t row_stride;
  int width, blocks;
  // the block that holds tokens `logical` * block on of sequence b, -1 where there is none
  __device__ __forceinline__ int at(int b, int logical) const {
    if (logical < 0 || logical >= width) return -1;
    const int id = entries[b * row_stride + logical];
    return id >= 0 && id < blocks ? id : -1;
  }
};

// The rows of a batch. Everything read from `start` is clamped, so that no content of it leads out of the tensors.
struct Ragged {
  const int32_t* start;   // [sequences + 1], or null: one row each
  int sequences, rows;
  __device__ __forceinline__ int first(int b) const {
    return start == nullptr ? b : min(max(start[b], 0), rows);
  }
  __device__ __forceinline__ int count(int b) const {
    return start == nullptr ? 1 : max(min(max(start[b + 1], 0), rows) - first(b), 0);
  }
  // A launch cannot know on the host how many pieces of `tile` units each sequence's rows make (the starts lie on the
  // device), but it can bound their sum: sequence b's pieces are numbered from floor(first(b) * units / tile) + spare * b,
  // and between two sequences' numbers there is room for floor(rows * units / tile) + spare pieces. Finds the sequence
  // of piece `slot`, 64 starts at a time (they grow with b, so the last one at or below the slot is counted), and leaves in
  // `slot` the piece's index within the sequence. Called by whole waves. sequences > 0.
  __device__ __forceinline__ int find(int64_t units, int tile, int spare, int64_t& slot) const {
    const int lane = threadIdx.x & (kWave - 1);
    int found = 0;
    for (int b0 = 0; b0 < sequences; b0 += kWave) {
      const int b = b0 + lane;
      const bool below = b < sequences && first(b) * units / tile + static_cast<int64_t>(spare) * b <= slot;
      const int n = __popcll(__ballot(below));
      found += n;
      if (n < kWave) break;
    }
    const int b = max(found - 1, 0);
    slot -= first(b) * units / tile + static_cast<int64_t>(spare) * b;
    return b;
  }
};

}  // namespace llmq
