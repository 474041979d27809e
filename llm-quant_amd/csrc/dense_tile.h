// A tile of a product of two dense 16-bit matrices on the matrix core:
//
//   D[m, n] = sum_k A[m, k] B[n, k]        fp32 accumulation
//
// the core that the vocabulary loss and the gradient of a quantized Linear build on. Each operand lies with the reduction axis innermost
// ([rows, K]) or outermost ([K, rows]: no matrix is turned over on the way). fp32 matrices take part as three bfloat16 planes
// each (planes_of: x = x0 + x1 + x2, 8 bits and 8 and 8: exact), of whose nine products the six largest are added: what is left out is
// at most 2^-23 of a term (x1 y2 and x2 y1, 2^-8 times 2^-16 each). An infinity has no such planes: what it takes part in is NaN.
//
// Shape. TM x TN outputs a workgroup of eight waves, 64 of K a step; both operands reach LDS as they lie in memory (buffer loads into
// LDS, 16 bytes a lane, nothing in registers), their chunks of 16 bytes swizzled by the row so that the reads of operands spread over
// the banks. Rows of K are read 16 bytes a lane; columns of K by the transposing read (ds_read_b64_tr_b16: among 16 lanes, lane l gets as its
// element j element l % 4 of what lane 4 j + l / 4 points at). Two stages; a step is two halves of 32 of K, each half's operands are read under the
// other's multiplications, and the workgroup meets between the halves, when the step's last operands are in registers: behind it the stage
// takes the transfers of the step after next, which have a whole step to arrive.
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

// A matrix of 16-bit values. Rows of K (a multiple of 64, which all rows have in memory), or K rows of `rows` neighbouring values (in
// memory a multiple of 8), of which `k_rows` exist: rows from there on repeat the last one, so that the other operand has zeros there.
struct TileOperand {
  const void* base;
  int64_t plane_bytes;   // between the planes of an fp32 matrix
  int64_t row_bytes;     // a lane's offset into a tile has 32 bits: tile_spans
  int rows;
  int k_rows;
};

// Whether the rows of a tile lie close enough for that: the first to the last of `tile` rows, each `row_bytes` behind the one before, and a step of a row.
inline bool tile_spans(int rows, int tile, int64_t row_bytes, int64_t step_bytes) {
  return ((rows < tile ? rows : tile) - 1) * row_bytes + step_bytes <= int64_t{0xffffffff};
}

// tile of a launch for a workgroup: workgroups go to the eight XCDs in turn, and an XCD takes a contiguous run of tiles, so
// that tiles that share an operand share its L2
__device__ __forceinline__ int tile_of_workgroup(int id, int total) {
  constexpr int kXcds = 8;
  const int xcd = id % kXcds, at = id / kXcds, each = total / kXcds, left = total % kXcds;
  return xcd * each + min(xcd, left) + at;
}

// A_K, B_K: K outermost. MG: how the rows of A are named to the matrix core: lane 16 g + r has rows 4 MG (4 (mi / MG) + g) + 4 (mi % MG) .. + 3 of the wave's,
// so that with 2 two tiles' results are eight neighbours (a 16-byte packet of 16-bit values; A_K: 1).
template <typename T, int TM, int TN, int WM, int WN, bool A_K = false, bool B_K = false, int MG = 1> struct DenseTile {
  static constexpr int kWaves = WM * WN, kThreads = kWaves * kWave;
  static constexpr int kStep = 64;                                             // of K
  static constexpr int MI = TM / WM / 16, NI = TN / WN / 16;
  static constexpr int kALoads = TM / 8 / kWaves, kBLoads = TN / 8 / kWaves;   // transfers of a wave a step, 1024 bytes each
  static constexpr int kStageBytes = (TM + TN) * 2 * kStep, kLdsBytes = 2 * kStageBytes;
  static_assert(kALoads * 8 * kWaves == TM && kBLoads * 8 * kWaves == TN, "even shares");
  static_assert(MI % MG == 0 && (!A_K || MG == 1), "whole groups of row tiles");
  static_assert((MI & (MI - 1)) == 0 && (NI & (NI - 1)) == 0, "the swizzle's arithmetic");

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

 private:
  // One operand's side. EXTENT: its rows of a tile; TILES of 16 of them a wave; GROUP: MG.
  template <int EXTENT, int TILES, int LOADS, bool K_OUT, int GROUP> struct Side {
    static constexpr int kRowBytes = K_OUT ? EXTENT * 2 : 2 * kStep, kSlots = kRowBytes / 16, kRowsPerLoad = 1024 / kRowBytes;
    // K_OUT: pairs of chunks of row r lie at pair ^ fold(r); rows 8 g + j, which a read takes together, meet every bank twice, the least there is
    static __device__ __forceinline__ int fold(int r) { return kSlots >= 16 ? (r & 3) | ((r >> 3 & 1) << 2) : (r >> 1 & 1) | ((r >> 3 & 1) << 1); }
    // else: chunks of row r lie at chunk ^ swizzle(r); eight neighbouring lanes of a read meet eight slots
    static __device__ __forceinline__ int swizzle(int r) { return (r & 3) | ((r / (4 * GROUP) & 1) << 2); }
    const TileOperand& m;
    const uint8_t* tile;   // of plane 0: the tile's first row, or K's first
    int wv, at0;           // at0: the tile's first row
    uint32_t off[LOADS];
    uint32_t read;         // of operands, tile 0, first half

    __device__ __forceinline__ Side(const TileOperand& operand, int first, int wave, int wave_at, uint32_t lds_base) : m(operand), wv(wave), at0(first) {
      const int lane = threadIdx.x & (kWave - 1), lr = lane & 15, lg = lane >> 4;
      tile = static_cast<const uint8_t*>(m.base) + (K_OUT ? 0 : first * m.row_bytes);
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        const int r = (wv * LOADS + i) * kRowsPerLoad + lane / kSlots, slot = lane % kSlots;
        if constexpr (K_OUT) off[i] = static_cast<uint32_t>(r * m.row_bytes) + column(r, slot);
        else off[i] = static_cast<uint32_t>((min(first + r, m.rows - 1) - first) * m.row_bytes) + ((slot ^ swizzle(r)) << 4);
      }
      if constexpr (K_OUT) {
        const int r = 8 * lg + (lr >> 2), i = lr & 3;
        read = lds_base + r * kRowBytes + (((wave_at * TILES) ^ fold(r)) << 5) + (i >> 1) * 16 + (i & 1) * 8;
      } else {
        const int r = wave_at * TILES * 16 + (lr >> 2) * 4 * GROUP + (lr & 3);
        read = lds_base + r * kRowBytes + ((lg ^ swizzle(r)) << 4);
      }
    }
    __device__ __forceinline__ uint32_t column(int r, int slot) const {   // K_OUT: byte of a row of K (columns past the end: the last ones again)
      const int chunk = ((slot >> 1 ^ fold(r)) << 1) | (slot & 1);
      return static_cast<uint32_t>(min(at0 + chunk * 8, (m.rows - 1) / 8 * 8)) * 2;
    }
    // the transfers of a step into the stage
    __device__ __forceinline__ void request(int plane, int k, uint8_t* to) const {
      const uint8_t* from = tile + plane * m.plane_bytes + (K_OUT ? k * m.row_bytes : int64_t{2} * k);
      const BufferBase base = buffer_base(from);
      to += wv * LOADS * 1024;
      if (K_OUT && k + kStep > m.k_rows) {   // (the last step: rows past the end)
        const int lane = threadIdx.x & (kWave - 1);
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
          const int r = (wv * LOADS + i) * kRowsPerLoad + lane / kSlots;
          buffer_to_lds<16>(base, to + i * 1024, static_cast<uint32_t>(min(r, m.k_rows - 1 - k) * m.row_bytes) + column(r, lane % kSlots), 0);
        }
        return;
      }
#pragma unroll
      for (int i = 0; i < LOADS; ++i) buffer_to_lds<16>(base, to + i * 1024, off[i], 0);
    }
    __device__ __forceinline__ u32x4 operand(const uint8_t* stage, int t, int half) const {
      if constexpr (K_OUT) {
        const uint8_t* at = stage + (read ^ (t << 5)) + half * 32 * kRowBytes;
        const u32x2 lo = transposed(at), hi = transposed(at + 4 * kRowBytes);
        return u32x4{lo.x, lo.y, hi.x, hi.y};
      } else {
        return load16(stage + (read ^ (half << 6)) + ((t / GROUP) * 16 * GROUP + (t % GROUP) * 4) * kRowBytes);
      }
    }
    static __device__ __forceinline__ u32x2 transposed(const uint8_t* at) {
#if defined(__HIP_DEVICE_COMPILE__)
      typedef short v4s __attribute__((ext_vector_type(4)));
      return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4s*)(at)));
#else
      return {};
#endif
    }
  };

  __device__ __forceinline__ void products(const u32x4 (&a)[MI], const u32x4 (&b)[NI]) {
#pragma unroll
    for (int mi = 0; mi < MI; ++mi)
#pragma unroll
      for (int ni = 0; ni < NI; ++ni) acc[mi][ni] = mfma_16x16x32<T>(a[mi], b[ni], acc[mi][ni]);
  }

 public:
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int mi = 0; mi < MI; ++mi)
#pragma unroll
      for (int ni = 0; ni < NI; ++ni) acc[mi][ni] = tile_v4f{0.0f, 0.0f, 0.0f, 0.0f};
  }
  // PAIRS: products of planes (1, or 6 of fp32). k0, k1: the part of K, multiples of 64, k0 < k1.
  template <int PAIRS>
  __device__ __forceinline__ void multiply(uint8_t* lds, const TileOperand& a, int m0, const TileOperand& b, int n0, int k0, int k1) {
    const int wv = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / kWave), wm = wv / WN, wn = wv % WN;
    clear();
    const Side<TM, MI, kALoads, A_K, MG> as(a, m0, wv, wm, 0);
    const Side<TN, NI, kBLoads, B_K, 1> bs(b, n0, wv, wn, 2 * kStep * TM);
    const int steps = (k1 - k0) / kStep, all = steps * PAIRS;
    // the planes of pair p, the smallest products first: (2, 0) (0, 2) (1, 1) (1, 0) (0, 1) (0, 0)
    auto request = [&](int step) {
      int pair = 0, at = step;
      if constexpr (PAIRS > 1) {
        pair = step / steps;
        at = step - pair * steps;
      }
      const int pa = PAIRS > 1 ? (0x001102 >> (4 * pair)) & 0xf : 0, pb = PAIRS > 1 ? (0x010120 >> (4 * pair)) & 0xf : 0;
      uint8_t* stage = lds + (step & 1) * kStageBytes;
      as.request(pa, k0 + at * kStep, stage);
      bs.request(pb, k0 + at * kStep, stage + 2 * kStep * TM);
    };
    u32x4 af[2][MI], bf[2][NI];
    auto fetch = [&](int step, int half) {
      const uint8_t* stage = lds + (step & 1) * kStageBytes;
#pragma unroll
      for (int ni = 0; ni < NI; ++ni) bf[half][ni] = bs.operand(stage, ni, half);
#pragma unroll
      for (int mi = 0; mi < MI; ++mi) af[half][mi] = as.operand(stage, mi, half);
    };
    request(0);
    if (all > 1) request(1);
    if (all > 1) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kALoads + kBLoads) : "memory");
    else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");   // (no access moves across the barrier)
    fetch(0, 0);
    for (int step = 0; step < all; ++step) {
      fetch(step, 1);
      products(af[0], bf[0]);
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");   // the next step's transfers, this one's last operands
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      if (step + 2 < all) request(step + 2);
      if (step + 1 < all) fetch(step + 1, 0);
      products(af[1], bf[1]);
    }
    // (a caller that reuses the stages meets first: other waves may still read operands)
  }
};

}  // namespace llmq
