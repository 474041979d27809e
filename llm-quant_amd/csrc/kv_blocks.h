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
};

// The rows of a sequence.
struct Span {
  int first, n;
};
// The rows of a batch. Everything read from `start` is clamped, so that no content of it leads out of the tensors.
struct Ragged {
  const int32_t* start;   // [sequences + 1], or null: one row each
  int sequences, rows;
  __device__ __forceinline__ int first(int b) const {
    return start == nullptr ? b : min(max(start[b], 0), rows);
  }
  // A launch cannot know on the host how many blocks each sequence's rows touch (the starts lie on the device), but it can bound
  // their sum: sequence b's pieces are numbered from floor(first(b) / block) + 2 b on, and up to the next sequence's number
  // there is room for floor(n / block) + 2, which is as many as n rows can touch. Finds the sequence of piece `slot`, 64
  // at a time (the numbers grow with b, so the last one at or below the slot is counted); leaves in `slot` the piece's index
  // within the sequence, its rows in `span` and its entry of `more` (may be null: 0) in `other`, all read in one trip to
  // memory. Called by whole waves. sequences > 0.
  __device__ __forceinline__ int find(int block_shift, const int32_t* more, int& slot, Span& span, int& other) const {
    const int lane = threadIdx.x & (kWave - 1);
    int b = 0, number = 0;
    span = Span{0, 0};   // (a piece in front of the first sequence's rows is nobody's)
    other = 0;
    for (int b0 = 0; b0 < sequences; b0 += kWave) {
      const int at = min(b0 + lane, sequences - 1);
      int from = at, to = at + 1;
      if (start != nullptr) {
        from = start[at];
        to = start[at + 1];
      }
      const int value = more != nullptr ? more[at] : 0;
      from = min(max(from, 0), rows);
      const int n = max(min(max(to, 0), rows) - from, 0), mine = (from >> block_shift) + 2 * (b0 + lane);
      const int below = __popcll(__ballot(b0 + lane < sequences && mine <= slot));
      if (below == 0) break;
      b = b0 + below - 1;
      number = __builtin_amdgcn_readlane(mine, below - 1);
      span = Span{__builtin_amdgcn_readlane(from, below - 1), __builtin_amdgcn_readlane(n, below - 1)};
      other = __builtin_amdgcn_readlane(value, below - 1);
      if (below < kWave) break;
    }
    slot -= number;
    if (slot < 0) span.n = 0;   // (starts that decrease, against the contract: no piece in front of the sequence's first)
    return b;
  }
};

}  // namespace llmq
