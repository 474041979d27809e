// A tile of a product of two dense 16-bit matrices on the matrix core, both with the reduction axis innermost:
//
//   D[m, n] = sum_k A[m, k] B[n, k]        A [rows, K], B [rows, K], fp32 accumulation
//
// the core that the vocabulary loss and the gradient of a quantized Linear build on. fp32 matrices take part as three
// bfloat16 planes each (planes_of: x = x0 + x1 + x2, 8 bits and 8 and 8: exact), of whose nine products the six largest are
// added: what is left out is at most 2^-23 of a term (x1 y2 and x2 y1, 2^-8 times 2^-16 each).
//
// Shape. TM x TN outputs a workgroup, 64 of K a step; both operands reach LDS as they lie in memory (buffer loads into LDS, 16
// bytes a lane, nothing in registers), the chunks of 16 bytes swizzled by the row so that the reads of operands spread over
// the banks; two stages, one barrier a step: behind it the next step's transfers are asked for and run under this step's
// multiplications. A lane's results are 4 MG consecutive m of one column n (kRows below names the rows to the matrix
// core in that order), so that a store is 16 bytes and more of a row of D^T.
#pragma once

#include "llmq_device.h"

namespace llmq {

typedef float tile_v4f __attribute__((ext_vector_type(4)));
typedef __bf16 tile_v8bf __attribute__((ext_vector_type(8)));
typedef _Float16 tile_v8h __attribute__((ext_vector_type(8)));

template <typename T> __device__ __forceinline__ tile_v4f mfma_16x16x32(u32x4 a, u32x4 b, tile_v4f c);
template <> __device__ __forceinline__ tile_v4f mfma_16x16x32<bf16_t>(u32x4 a, u32x4 b, tile_v4f c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(tile_v8bf, a), __builtin_bit_cast(tile_v8bf, b), c, 0, 0, 0);
}
template <> __device__ __forceinline__ tile_v4f mfma_16x16x32<f16_t>(u32x4 a, u32x4 b, tile_v4f c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(tile_v8h, a), __builtin_bit_cast(tile_v8h, b), c, 0, 0, 0);
}

// x as a sum of three bfloat16, each the rounding of what the ones before left (exact subtractions)
__device__ __forceinline__ void planes_of(float x, uint16_t* p) {
  const uint16_t a = bf16_bits_rne(x);
  const float r = x - __builtin_bit_cast(float, static_cast<uint32_t>(a) << 16);
  const uint16_t b = bf16_bits_rne(r);
  p[0] = a;
  p[1] = b;
  p[2] = bf16_bits_rne(r - __builtin_bit_cast(float, static_cast<uint32_t>(b) << 16));
}
// What a value of T is in the operands: itself, or three planes of bfloat16.
template <typename T> struct TileType { using type = T; static constexpr int kPlanes = 1; };
template <> struct TileType<float> { using type = bf16_t; static constexpr int kPlanes = 3; };

// A matrix of 16-bit values, rows of K (a multiple of 64, which all rows have in memory).
struct TileOperand {
  const void* base;
  int64_t plane_bytes;   // between the planes of an fp32 matrix
  uint32_t row_bytes;
  int rows;
};

// tile of a launch for a workgroup: workgroups go to the eight XCDs in turn, and an XCD takes a contiguous run of tiles, so
// that tiles that share an operand share its L2
__device__ __forceinline__ int tile_of_workgroup(int id, int total) {
  constexpr int kXcds = 8;
  const int xcd = id % kXcds, at = id / kXcds, each = total / kXcds, left = total % kXcds;
  return xcd * each + min(xcd, left) + at;
}

template <typename T, int TM, int TN, int WM, int WN> struct DenseTile {
  static constexpr int kWaves = WM * WN, kThreads = kWaves * kWave;
  static constexpr int kStep = 64, kRowBytes = 2 * kStep;                     // of K, and of a row of it in LDS
  static constexpr int MI = TM / WM / 16, NI = TN / WN / 16, MG = MI < 4 ? MI : 4;
  static constexpr int kALoads = TM / 8 / kWaves, kBLoads = TN / 8 / kWaves;   // transfers of a wave a step, eight rows each
  static constexpr int kStageBytes = (TM + TN) * kRowBytes, kLdsBytes = 2 * kStageBytes;
  static_assert(kALoads * 8 * kWaves == TM && kBLoads * 8 * kWaves == TN, "even shares");
  static_assert(MI % MG == 0, "whole groups of row tiles");

  tile_v4f acc[MI][NI];

  // the m and n of acc[mi][ni][i], within the tile
  static __device__ __forceinline__ int row_of(int mi, int i) {
    const int lane = threadIdx.x & (kWave - 1), wm = static_cast<int>(threadIdx.x) / kWave / WN;
    return wm * (TM / WM) + (mi / MG) * 16 * MG + (lane >> 4) * 4 * MG + (mi % MG) * 4 + i;
  }
  static __device__ __forceinline__ int col_of(int ni) {
    const int lane = threadIdx.x & (kWave - 1), wn = static_cast<int>(threadIdx.x) / kWave % WN;
    return wn * (TN / WN) + ni * 16 + (lane & 15);
  }
  // chunks of row r of a stage's A and B lie at slot chunk ^ swizzle: eight neighbouring lanes of a read meet eight slots
  static __device__ __forceinline__ int swizzle_a(int r) { return (r & 3) | ((r / (4 * MG) & 1) << 2); }
  static __device__ __forceinline__ int swizzle_b(int r) { return r & 7; }

  // PAIRS: products of planes (1, or 6 of fp32). k0, k1: the part of K, multiples of 64, k0 < k1.
  template <int PAIRS>
  __device__ __forceinline__ void multiply(uint8_t* lds, const TileOperand& a, int m0, const TileOperand& b, int n0, int k0, int k1) {
    const int lane = threadIdx.x & (kWave - 1);
    const int wv = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / kWave), wm = wv / WN, wn = wv % WN;
#pragma unroll
    for (int mi = 0; mi < MI; ++mi)
#pragma unroll
      for (int ni = 0; ni < NI; ++ni) acc[mi][ni] = tile_v4f{0.0f, 0.0f, 0.0f, 0.0f};

    // (rows past the end repeat the last one: what they make is not stored)
    uint32_t a_off[kALoads], b_off[kBLoads];
#pragma unroll
    for (int i = 0; i < kALoads; ++i) {
      const int r = (wv * kALoads + i) * 8 + (lane >> 3);
      a_off[i] = static_cast<uint32_t>(min(m0 + r, a.rows - 1) - m0) * a.row_bytes + (((lane & 7) ^ swizzle_a(r)) << 4);
    }
#pragma unroll
    for (int i = 0; i < kBLoads; ++i) {
      const int r = (wv * kBLoads + i) * 8 + (lane >> 3);
      b_off[i] = static_cast<uint32_t>(min(n0 + r, b.rows - 1) - n0) * b.row_bytes + (((lane & 7) ^ swizzle_b(r)) << 4);
    }
    const uint8_t* a_tile = static_cast<const uint8_t*>(a.base) + static_cast<int64_t>(m0) * a.row_bytes;
    const uint8_t* b_tile = static_cast<const uint8_t*>(b.base) + static_cast<int64_t>(n0) * b.row_bytes;
    const int steps = (k1 - k0) / kStep, all = steps * PAIRS;
    // the planes of pair p, the smallest products first: (2, 0) (0, 2) (1, 1) (1, 0) (0, 1) (0, 0)
    auto request = [&](int step, int buf) {
      int pair = 0, at = step;
      if constexpr (PAIRS > 1) {
        pair = step / steps;
        at = step - pair * steps;
      }
      const int pa = PAIRS > 1 ? (0x001102 >> (4 * pair)) & 0xf : 0;
      const int pb = PAIRS > 1 ? (0x010120 >> (4 * pair)) & 0xf : 0;
      const BufferBase ab = buffer_base(a_tile + (PAIRS > 1 ? pa * a.plane_bytes : 0)),
                       bb = buffer_base(b_tile + (PAIRS > 1 ? pb * b.plane_bytes : 0));
      const uint32_t offset = static_cast<uint32_t>(k0 + at * kStep) * 2;
      uint8_t* stage = lds + buf * kStageBytes;
#pragma unroll
      for (int i = 0; i < kALoads; ++i) buffer_to_lds<16>(ab, stage + (wv * kALoads + i) * 1024, a_off[i], offset);
#pragma unroll
      for (int i = 0; i < kBLoads; ++i) buffer_to_lds<16>(bb, stage + TM * kRowBytes + (wv * kBLoads + i) * 1024, b_off[i], offset);
    };
    // operands: row of this lane in row tile 0 / column tile 0, chunk lane / 16 of the first half of a step
    const int lr = lane & 15, lg = lane >> 4;
    const int a_row = wm * (TM / WM) + (lr >> 2) * 4 * MG + (lr & 3), b_row = wn * (TN / WN) + lr;
    const uint32_t a_at = a_row * kRowBytes + ((lg ^ swizzle_a(a_row)) << 4);
    const uint32_t b_at = TM * kRowBytes + b_row * kRowBytes + ((lg ^ swizzle_b(b_row)) << 4);
    request(0, 0);
    for (int step = 0; step < all; ++step) {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");   // (no access moves across the barrier)
      if (step + 1 < all) request(step + 1, (step + 1) & 1);
      const uint8_t* stage = lds + (step & 1) * kStageBytes;
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
        u32x4 af[MI], bf[NI];
#pragma unroll
        for (int ni = 0; ni < NI; ++ni) bf[ni] = load16(stage + (b_at ^ (kk << 6)) + ni * 16 * kRowBytes);
#pragma unroll
        for (int mi = 0; mi < MI; ++mi)
          af[mi] = load16(stage + (a_at ^ (kk << 6)) + ((mi / MG) * 16 * MG + (mi % MG) * 4) * kRowBytes);
#pragma unroll
        for (int mi = 0; mi < MI; ++mi)
#pragma unroll
          for (int ni = 0; ni < NI; ++ni) acc[mi][ni] = mfma_16x16x32<T>(af[mi], bf[ni], acc[mi][ni]);
      }
    }
    // (a caller that reuses the stages meets first: other waves may still read operands)
  }
};

}  // namespace llmq
