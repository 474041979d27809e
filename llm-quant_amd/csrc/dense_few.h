// Products of a large weight with few rows, for the vocabulary loss and the gradient of a quantized Linear: the weight, dense or codes, is read
// as it lies, once for each 64 rows (bound: HBM, and for fp32 from about 32 rows on the matrix core's fp32). Codes become the values (dtype)(code * scale) in
// registers, the same ones that dequant_weight writes. fp32 is multiplied in fp32.
//
//   FewRows           D[v, t] = sum_k W[v, k] x[t, k]     the reduction runs along the weight's rows
//   columns_kernel    D[t, k] = sum_v g[t, v] W[v, k]     the reduction runs over the weight's rows
//   few_outer_kernel  D[v, k] = sum_t P[t, v] x[t, k]     the reduction runs over the few rows (bound: the result's way to memory)
#pragma once

#include "dense_tile.h"

namespace llmq {

struct FewWeight {
  const uint8_t* base;   // rows of `row_bytes`
  const float* scale;    // of codes: [scale rows, groups]
  int64_t row_bytes;
  int rows, width;       // width: columns, `keep` of each group
  int groups, group_size, keep, out_group;
  __device__ __forceinline__ int64_t scale_row(int row) const { return static_cast<int64_t>(out_group > 0 ? row / out_group : row) * groups; }
};

// eight codes with their scale, as two halves of words: word i of the result holds values 2 i and 2 i + 1
template <typename T> __device__ __forceinline__ uint32_t pair_of(float lo, float hi);
template <> __device__ __forceinline__ uint32_t pair_of<bf16_t>(float lo, float hi) { return bf16_pair_rne(lo, hi); }
template <> __device__ __forceinline__ uint32_t pair_of<f16_t>(float lo, float hi) {
  return static_cast<uint32_t>(__builtin_bit_cast(uint16_t, f16_rne(lo))) | static_cast<uint32_t>(__builtin_bit_cast(uint16_t, f16_rne(hi))) << 16;
}
// values of an operand packet (16 bytes); the products of a lane's packet: K is V (4 k + g) + e for value e of lane 16 g + r
template <typename T> constexpr int kFewPack = 16 / sizeof(T);
template <typename T> __device__ __forceinline__ tile_v4f few_mfma(u32x4 a, u32x4 b, tile_v4f c) { return mfma_16x16x32<T>(a, b, c); }
__device__ __forceinline__ tile_v4f few_mfma_f32(uint32_t a, uint32_t b, tile_v4f c) {
  return __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(float, a), __builtin_bit_cast(float, b), c, 0, 0, 0);
}
template <> __device__ __forceinline__ tile_v4f few_mfma<float>(u32x4 a, u32x4 b, tile_v4f c) {
  return few_mfma_f32(a.w, b.w, few_mfma_f32(a.z, b.z, few_mfma_f32(a.y, b.y, few_mfma_f32(a.x, b.x, c))));
}
// four neighbouring values
template <typename T> __device__ __forceinline__ void store_four(T* to, const float* f) {
  if constexpr (sizeof(T) == 4) *reinterpret_cast<tile_v4f*>(to) = tile_v4f{f[0], f[1], f[2], f[3]};
  else *reinterpret_cast<u32x2*>(to) = u32x2{pair_of<T>(f[0], f[1]), pair_of<T>(f[2], f[3])};
}
// Eight codes, times the scale as 32 bits, as pairs. BITS 8: two words; 4: one word of code + 8, each brought to the upper half of a byte as
// 16 code, against a sixteenth of the scale (exact down to 2^-122). float(int8) of a byte is one instruction.
template <int BITS> struct Codes {
  uint32_t w[2];
  __device__ __forceinline__ explicit Codes(const uint32_t* v) {
    if constexpr (BITS == 8) {
      w[0] = v[0];
      w[1] = v[1];
    } else {
      const uint32_t c = v[0] ^ 0x88888888u;
      w[0] = c << 4 & 0xf0f0f0f0u;
      w[1] = c & 0xf0f0f0f0u;
    }
  }
  static __device__ __forceinline__ float scale_of(float scale) { return BITS == 8 ? scale : scale * 0.0625f; }
  static __device__ __forceinline__ float at(const uint32_t* w, int i) {
    return static_cast<float>(static_cast<int8_t>(BITS == 8 ? w[i / 4] >> (8 * (i % 4)) : w[i % 2] >> (8 * (i / 2))));
  }
};

// Four values of a row of the weight from column c on (a multiple of four), as the products have them.
template <typename T> __device__ __forceinline__ void weight_four(const FewWeight& w, const int bits, const int row, const int c, float* f) {
  const uint8_t* from = w.base + row * w.row_bytes;
  if (bits == 0) {
    const T* at = reinterpret_cast<const T*>(from) + c;
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = to_float(at[i]);
    return;
  }
  const float scale = w.scale[w.scale_row(row) + c / w.group_size];
  if (bits == 8) {
    const uint32_t codes = *reinterpret_cast<const uint32_t*>(from + c);
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = to_float(from_float<T>(static_cast<float>(static_cast<int8_t>(codes >> (8 * i))) * scale));
  } else {
    const int codes = *reinterpret_cast<const uint16_t*>(from + c / 2);
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = to_float(from_float<T>(static_cast<float>((codes >> (4 * i) & 15) - 8) * scale));
  }
}
// What rounding took from the entry of a row's own target, by far the largest of its row of P as a rule: added to the results in fp32.
struct TargetTerm {
  const float* rest;        // [rows], or null: nothing
  const int64_t* target;    // [rows], in the vocabulary where `rest` is not zero
  FewWeight weight;
  int bits;
  template <typename T> __device__ __forceinline__ void add(const int row, const int c, float* f) const {
    const float by = rest[row];
    if (by == 0.0f) return;
    float v[4];
    weight_four<T>(weight, bits, static_cast<int>(target[row]), c, v);
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = __builtin_fmaf(by, v[i], f[i]);
  }
};

// ---- x in operand order -------------------------------------------------------------------------------------------------------
// [block of 16 `tiles` rows][k / 4 V][tile of 16 rows][lane][V values]: lane 16 g + r holds values 4 V k + V g .. of row 16 tile + r; zeros past the rows and
// where `gather` has none. V: a packet's.
template <typename T>
__global__ __launch_bounds__(256) void few_operand_kernel(const T* __restrict__ x, const int64_t stride, const int32_t* __restrict__ gather,
                                                          const int rows, const int k, const int tiles, T* __restrict__ out) {
  constexpr int V = kFewPack<T>;
  const int64_t items = static_cast<int64_t>(k / (4 * V)) * tiles * kWave, item = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (item >= items) return;
  const int lane = item % kWave, tile = static_cast<int>(item / kWave % tiles), at = static_cast<int>(item / kWave / tiles);
  const int t = (blockIdx.y * tiles + tile) * 16 + (lane & 15);
  const int row = t >= rows ? -1 : gather != nullptr ? gather[t] : t;
  u32x4 v{0, 0, 0, 0};
  if (row >= 0) v = load16(x + row * stride + (at * 4 + (lane >> 4)) * V);
  store16(out + (blockIdx.y * items + item) * V, v);
}
// the same for a reduction over the rows: [16 columns][step of 4 V rows][lane][V values], lane 16 g + r: rows 4 V step + V g .. of column few_column(r)
template <typename T> __device__ __forceinline__ int few_column(int tile, int r) {   // (16 bits: two tiles' results are eight neighbours)
  if constexpr (sizeof(T) == 4) return tile * 16 + r;
  else return (tile >> 1) * 32 + (r >> 2) * 8 + (tile & 1) * 4 + (r & 3);
}
template <typename T>
__global__ __launch_bounds__(256) void few_turned_kernel(const T* __restrict__ x, const int64_t stride, const int32_t* __restrict__ gather, const int rows,
                                                         const int k, const int steps, T* __restrict__ out) {
  constexpr int V = kFewPack<T>;
  const int64_t items = static_cast<int64_t>(k / 16) * steps * kWave, item = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (item >= items) return;
  const int lane = item % kWave, step = static_cast<int>(item / kWave % steps), tile = static_cast<int>(item / kWave / steps);
  const int c = few_column<T>(tile, lane & 15);
  T v[V];
#pragma unroll
  for (int e = 0; e < V; ++e) {
    const int t = (step * 4 + (lane >> 4)) * V + e, row = t >= rows ? -1 : gather[t];
    v[e] = row >= 0 ? x[row * stride + c] : from_float<T>(0.0f);
  }
  store16(out + item * V, *reinterpret_cast<const u32x4*>(v));
}

// ---- the reduction along the weight's rows ----------------------------------------------------------------------------------------
constexpr int kFewTokens = 64, kFewWaves = 4;   // rows of the weight a workgroup; waves

// The waves of a workgroup take steps of its 64 rows by turns: 128 bytes of each row (int4, and codes for fp32: less) through LDS of the wave's own, in whole
// lines, two steps in flight, no barrier until the sums meet. RowsStep::operand: a packet of a row's values, from LDS.
template <typename T, int BITS> struct RowsStep {
  static constexpr int V = kFewPack<T>, kK = BITS == 0 ? 128 / sizeof(T) : sizeof(T) == 4 ? 64 : 128;
  static constexpr int kRowBytes = BITS == 0 ? 128 : kK * BITS / 8, kSlots = kRowBytes / 16, kRowsPerLoad = 64 / kSlots;
  static constexpr int kBytes = kFewTokens * kRowBytes, kLoads = kBytes / 1024, kPackets = kK / (4 * V);
  // the chunk of 16 bytes that slot p of row r holds (its own inverse): reads of 16 rows meet every bank as often
  static __device__ __forceinline__ int chunk(int r, int p) {
    if constexpr (BITS == 0) return p ^ (r & 7);
    else if constexpr (kSlots == 8) return p ^ ((r >> 1 & 3) << 1);
    else if constexpr (kSlots == 4) return p ^ (r >> 2 & 3);
    else return p ^ (r >> 3 & 1);
  }
  // values V (4 c + g) .. of row r
  static __device__ __forceinline__ u32x4 operand(const uint8_t* stage, int r, int c, int g, float scale) {
    if constexpr (BITS == 0) {
      return load16(stage + r * kRowBytes + (chunk(r, 4 * c + g) << 4));
    } else {
      constexpr int kBytesEach = V * BITS / 8;   // of a packet's codes: 8, 4 or 2
      const int byte = (4 * c + g) * kBytesEach;
      const uint8_t* from = stage + r * kRowBytes + (chunk(r, byte >> 4) << 4) + (byte & 15);
      uint32_t w[2];
      if constexpr (kBytesEach == 8) {
        const u32x2 v = *reinterpret_cast<const u32x2*>(from);
        w[0] = v.x;
        w[1] = v.y;
      } else if constexpr (kBytesEach == 4) {
        w[0] = *reinterpret_cast<const uint32_t*>(from);
      } else {
        w[0] = *reinterpret_cast<const uint16_t*>(from);
      }
      const Codes<BITS> codes(w);
      const float by = Codes<BITS>::scale_of(scale);
      float f[V];
#pragma unroll
      for (int i = 0; i < V; ++i) f[i] = Codes<BITS>::at(codes.w, i) * by;
      if constexpr (sizeof(T) == 4) return __builtin_bit_cast(u32x4, tile_v4f{f[0], f[1], f[2], f[3]});
      else return u32x4{pair_of<T>(f[0], f[1]), pair_of<T>(f[2], f[3]), pair_of<T>(f[4], f[5]), pair_of<T>(f[6], f[7])};
    }
  }
};

// acc[i]: rows 16 i + 4 g .. + 3 of the workgroup's, of row 16 j + r of x, where the wave is j's (j = wave, while there are so many)
template <typename T, int BITS, int NT> struct FewRows {
  using Step = RowsStep<T, BITS>;
  static constexpr int kTiles = kFewTokens / 16, kSums = kFewWaves * kTiles * NT * 1024, kStages = kFewWaves * 2 * Step::kBytes;
  static constexpr int kLdsBytes = kSums > kStages ? kSums : kStages;
  tile_v4f acc[kTiles];

  struct Asked {
    u32x4 x[Step::kPackets][NT];
    float scale[BITS ? kTiles : 1];
  };
  // live: tiles of x that have rows (fp32, where the multiplications bind: the others are left out)
  __device__ __forceinline__ void multiply(uint8_t* lds, const FewWeight& w, int m0, const T* x, int live) {
    const int lane = threadIdx.x & (kWave - 1), wv = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / kWave), lr = lane & 15, g = lane >> 4;
    const int steps = w.width / Step::kK;
    uint8_t* const mine = lds + wv * 2 * Step::kBytes;
    const BufferBase base = buffer_base(w.base + m0 * w.row_bytes);
    uint32_t off[Step::kLoads];
#pragma unroll
    for (int i = 0; i < Step::kLoads; ++i) {
      const int r = i * Step::kRowsPerLoad + lane / Step::kSlots;
      off[i] = static_cast<uint32_t>((min(m0 + r, w.rows - 1) - m0) * w.row_bytes) + (Step::chunk(r, lane % Step::kSlots) << 4);
    }
    const float* scale[kTiles];
    if constexpr (BITS != 0) {
#pragma unroll
      for (int i = 0; i < kTiles; ++i) scale[i] = w.scale + w.scale_row(min(m0 + i * 16 + lr, w.rows - 1));
    }
    tile_v4f sum[kTiles][NT] = {};
    const auto ask = [&](int at, int buf, Asked& a) {   // (the transfers last: what is waited for below leaves them in flight)
#pragma unroll
      for (int c = 0; c < Step::kPackets; ++c)
#pragma unroll
        for (int j = 0; j < NT; ++j) a.x[c][j] = load16(x + (((static_cast<int64_t>(at) * Step::kPackets + c) * NT + j) * kWave + lane) * Step::V);
      if constexpr (BITS != 0) {
#pragma unroll
        for (int i = 0; i < kTiles; ++i) a.scale[i] = scale[i][at * Step::kK / w.group_size];
      }
#pragma unroll
      for (int i = 0; i < Step::kLoads; ++i) buffer_to_lds<16>(base, mine + buf * Step::kBytes + i * 1024, off[i], at * Step::kRowBytes);
    };
    // the transfers of all steps but the newest have arrived
    const auto arrived = [&](bool newer) {
      if (newer) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(Step::kLoads) : "memory");
      else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    };
    const auto use = [&](int buf, const Asked& a) {
      const uint8_t* stage = mine + buf * Step::kBytes;
#pragma unroll
      for (int c = 0; c < Step::kPackets; ++c)
#pragma unroll
        for (int i = 0; i < kTiles; ++i) {
          const u32x4 v = Step::operand(stage, i * 16 + lr, c, g, a.scale[BITS ? i : 0]);
#pragma unroll
          for (int j = 0; j < NT; ++j)
            if (sizeof(T) == 2 || j < live) sum[i][j] = few_mfma<T>(v, a.x[c][j], sum[i][j]);
        }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // (the stage is asked for again)
    };
    Asked a, b;
    a.scale[0] = b.scale[0] = 1.0f;
    if (wv < steps) {
      ask(wv, 0, a);
      for (int s = wv; s < steps; s += 2 * kFewWaves) {
        const bool second = s + kFewWaves < steps, third = s + 2 * kFewWaves < steps;
        if (second) ask(s + kFewWaves, 1, b);
        arrived(second);
        use(0, a);
        if (!second) break;
        if (third) ask(s + 2 * kFewWaves, 0, a);
        arrived(third);
        use(1, b);
      }
    }
    __syncthreads();
    tile_v4f* const s_sum = reinterpret_cast<tile_v4f*>(lds);   // [wave][tile][row tile][lane]
#pragma unroll
    for (int i = 0; i < kTiles; ++i)
#pragma unroll
      for (int j = 0; j < NT; ++j) s_sum[((wv * kTiles + i) * NT + j) * kWave + lane] = sum[i][j];
    __syncthreads();
    const int j = min(wv, NT - 1);
#pragma unroll
    for (int i = 0; i < kTiles; ++i) {
      acc[i] = s_sum[(i * NT + j) * kWave + lane];
#pragma unroll
      for (int v = 1; v < kFewWaves; ++v) acc[i] += s_sum[((v * kTiles + i) * NT + j) * kWave + lane];
    }
  }
};

// ---- the reduction over the weight's rows -----------------------------------------------------------------------------------------
constexpr int kFewColumns = 128;   // of a wave

struct FewColumns {
  const void* g;         // [rows, stride] of T: values of the weight's rows, in whole packets
  int64_t stride;
  const int32_t* count;  // or null: how many of the rows there are
  int rows;
  float* planes;         // [splits][rows][width]
  int splits;
};

// A workgroup: 128 columns, 16 NT rows of g (blockIdx.y), a part of the weight's rows, which its waves take 32 (fp32: 16) at a time; each lane
// eight columns of eight (four) rows, turned over in registers, a step ahead. The waves' sums meet in LDS.
template <typename T, int BITS, int NT>
__global__ __launch_bounds__(kFewWaves * kWave, 2) void columns_kernel(const FewWeight w, const FewColumns c) {
  constexpr int V = kFewPack<T>, kWords = BITS == 0 ? 2 * sizeof(T) : BITS / 4, kRows = 4 * V;   // words of eight values; rows of a step
  constexpr bool kHalves = sizeof(T) == 4 && BITS == 0;   // a lane's columns: 4 lr .. and 64 + 4 lr .., whole lines of 16 lanes
  __shared__ tile_v4f s_sum[2][NT * 8][kWave];
  const int t0 = blockIdx.y * 16 * NT, rows = c.count != nullptr ? min(*c.count, c.rows) : c.rows;
  if (t0 >= rows) return;
  const int lane = threadIdx.x & (kWave - 1), wv = threadIdx.x / kWave, lr = lane & 15, g = lane >> 4;
  const int steps = (w.rows + kRows - 1) / kRows, per = (steps + c.splits - 1) / c.splits;
  const int parts = (w.width + kFewColumns - 1) / kFewColumns, item = tile_of_workgroup(blockIdx.x, gridDim.x), split = item / parts;
  const int v0 = min(split * per, steps) * kRows, v1 = min((split + 1) * per, steps) * kRows;
  const int c0 = item % parts * kFewColumns, col = c0 + (kHalves ? 4 : 8) * lr, at = min(col, w.width - (kHalves ? 4 : 8));
  const int group = BITS ? at / w.keep : 0;
  const int64_t byte = BITS == 0 ? at * static_cast<int>(sizeof(T)) : (static_cast<int64_t>(group) * w.group_size + (at - group * w.keep)) * BITS / 8;
  const int64_t half = kHalves ? (min(col + 64, w.width - 4) - at) * 4 : 0;
  const T* gr[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j) gr[j] = static_cast<const T*>(c.g) + min(t0 + j * 16 + lr, rows - 1) * c.stride;
  struct Asked {
    uint32_t w[V][kWords];
    float scale[BITS ? V : 1];
    u32x4 g[NT];
  };
  const auto ask = [&](int v, Asked& a) {
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const int row = min(v + V * g + e, w.rows - 1);
      const uint8_t* from = w.base + row * w.row_bytes + byte;
      if constexpr (BITS == 0) {
#pragma unroll
        for (int h = 0; h < kWords / 4; ++h) {
          const u32x4 q = load16(from + h * half);
          a.w[e][4 * h] = q.x; a.w[e][4 * h + 1] = q.y; a.w[e][4 * h + 2] = q.z; a.w[e][4 * h + 3] = q.w;
        }
      } else if constexpr (BITS == 8) {
        const u32x2 q = *reinterpret_cast<const u32x2*>(from);
        a.w[e][0] = q.x; a.w[e][1] = q.y;
      } else {
        a.w[e][0] = *reinterpret_cast<const uint32_t*>(from);
      }
      if constexpr (BITS != 0) a.scale[e] = w.scale[w.scale_row(row) + group];
    }
#pragma unroll
    for (int j = 0; j < NT; ++j) a.g[j] = load16(gr[j] + min(v + V * g, (w.rows - 1) / V * V));
  };
  tile_v4f acc[NT][8] = {};
  const int begin = v0 + wv * kRows, step = kRows * kFewWaves;
  const auto use = [&](int v, Asked& now) {
    if (v + V * g >= w.rows) {   // the weight's last row again, against zeros
#pragma unroll
      for (int j = 0; j < NT; ++j) now.g[j] = u32x4{0, 0, 0, 0};
    }
    float by[BITS ? V : 1];
    uint32_t bytes[V][BITS ? 2 : kWords];
#pragma unroll
    for (int e = 0; e < V; ++e) {
      if constexpr (BITS != 0) {
        const Codes<BITS> codes(now.w[e]);
        bytes[e][0] = codes.w[0];
        bytes[e][1] = codes.w[1];
        by[e] = Codes<BITS>::scale_of(now.scale[e]);
      } else {
#pragma unroll
        for (int i = 0; i < kWords; ++i) bytes[e][i] = now.w[e][i];
      }
    }
#pragma unroll
    for (int q = 0; q < 8; ++q) {   // column q of the lane's eight
      uint32_t word[4];
      if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int e = 0; e < 4; ++e) word[e] = BITS == 0 ? bytes[e][q] : __builtin_bit_cast(uint32_t, Codes<BITS ? BITS : 8>::at(bytes[e], q) * by[e]);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t *lo = bytes[2 * e], *hi = bytes[2 * e + 1];
          if constexpr (BITS == 0) word[e] = __builtin_amdgcn_perm(hi[q / 2], lo[q / 2], q % 2 ? 0x07060302u : 0x05040100u);
          else word[e] = pair_of<T>(Codes<BITS>::at(lo, q) * by[2 * e], Codes<BITS>::at(hi, q) * by[2 * e + 1]);
        }
      }
      const u32x4 operand{word[0], word[1], word[2], word[3]};
#pragma unroll
      for (int j = 0; j < NT; ++j)
        if (sizeof(T) == 2 || t0 + j * 16 < rows) acc[j][q] = few_mfma<T>(now.g[j], operand, acc[j][q]);
    }
  };
  if (begin < v1) {   // (behind the last step: the part's last again)
    Asked a, b;
    ask(begin, a);
    for (int v = begin; v < v1; v += 2 * step) {
      ask(min(v + step, v1 - kRows), b);
      use(v, a);
      if (v + step >= v1) break;
      ask(min(v + 2 * step, v1 - kRows), a);
      use(v + step, b);
    }
  }
  if (wv >= 2) {
#pragma unroll
    for (int i = 0; i < NT * 8; ++i) s_sum[wv - 2][i][lane] = acc[i / 8][i % 8];
  }
  __syncthreads();
  if (wv < 2) {
#pragma unroll
    for (int i = 0; i < NT * 8; ++i) acc[i / 8][i % 8] += s_sum[wv][i][lane];
  }
  __syncthreads();
  if (wv == 1) {
#pragma unroll
    for (int i = 0; i < NT * 8; ++i) s_sum[0][i][lane] = acc[i / 8][i % 8];
  }
  __syncthreads();
  if (wv != 0) return;
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) {   // row 4 g + i, the lane's eight columns
      const int t = t0 + j * 16 + 4 * g + i;
      if (t >= rows) continue;
      float* to = c.planes + (static_cast<int64_t>(split) * c.rows + t) * w.width;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        tile_v4f v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = acc[j][h * 4 + e][i] + s_sum[0][j * 8 + h * 4 + e][lane][i];
        const int k = col + (kHalves ? 64 : 4) * h;
        if (k < w.width) *reinterpret_cast<tile_v4f*>(to + k) = v;
      }
    }
}
// Splits of the weight's rows, 64 at the most. For 256 workgroups: more are only more planes (4096 x 4096 int8, 64 rows: 17 us with 256, 26 with 512, 39
// with 1024; 128256 x 2048, 16 rows: bf16 87, 92 and 95, int8 56, 55 and 59, fp32, 8 rows, 166, 169 and 179), but for 512 where int4's conversion binds and a wave
// still has 16 steps (57, 46 and 43 with more planes to add; 64 rows 71, 61 and 66).
inline int few_splits(int weight_rows, int width, int rows, int bits) {
  const int64_t groups = static_cast<int64_t>((width + kFewColumns - 1) / kFewColumns) * ((rows + 63) / 64), step = 32 * kFewWaves;
  const int64_t most = (weight_rows + step - 1) / step, places = bits == 4 && most >= 512 / groups * 16 ? 512 : 256;
  const int64_t near = (places + groups / 2) / groups, splits = near < most ? near : most;
  return static_cast<int>(splits < 1 ? 1 : splits > 64 ? 64 : splits);
}
template <typename T, int BITS> inline void columns_launch_bits(const FewWeight& w, const FewColumns& c, hipStream_t stream) {
  const unsigned x = (w.width + kFewColumns - 1) / kFewColumns * c.splits;
  if (c.rows <= 16) hipLaunchKernelGGL((columns_kernel<T, BITS, 1>), dim3(x), dim3(kFewWaves * kWave), 0, stream, w, c);
  else if (c.rows <= 32) hipLaunchKernelGGL((columns_kernel<T, BITS, 2>), dim3(x), dim3(kFewWaves * kWave), 0, stream, w, c);
  else hipLaunchKernelGGL((columns_kernel<T, BITS, 4>), dim3(x, (c.rows + 63) / 64), dim3(kFewWaves * kWave), 0, stream, w, c);
}
template <typename T, bool DENSE> inline void columns_launch(const FewWeight& w, const FewColumns& c, int bits, hipStream_t stream) {
  if constexpr (DENSE) {
    if (bits == 0) return columns_launch_bits<T, 0>(w, c, stream);
  }
  if (bits == 8) columns_launch_bits<T, 8>(w, c, stream);
  else columns_launch_bits<T, 4>(w, c, stream);
}

// out[row] = (dtype)(scale[from] * the sum of the planes' row from = `from[row]`); no such row (negative): zeros
template <typename T>
__global__ __launch_bounds__(256) void add_few_kernel(const float* __restrict__ planes, const int splits, const int rows, const int width,
                                                      const float* __restrict__ scale_or_null, const int32_t* __restrict__ from_or_null, const TargetTerm term,
                                                      T* __restrict__ out) {
  constexpr int kAhead = 8;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x, items = static_cast<int64_t>(rows) * (width / 4);
  if (item >= items) return;
  const int row = static_cast<int>(item / (width / 4)), c = static_cast<int>(item % (width / 4)) * 4;
  const int from = from_or_null != nullptr ? from_or_null[row] : row;
  tile_v4f sum{0.0f, 0.0f, 0.0f, 0.0f};
  if (from >= 0) {
    const float* at = planes + static_cast<int64_t>(from) * width + c;
    const int64_t plane = static_cast<int64_t>(rows) * width;
    for (int z0 = 0; z0 < splits; z0 += kAhead) {
      tile_v4f v[kAhead];
#pragma unroll
      for (int z = 0; z < kAhead; ++z) v[z] = *reinterpret_cast<const tile_v4f*>(at + min(z0 + z, splits - 1) * plane);
#pragma unroll
      for (int z = 0; z < kAhead; ++z)
        if (z0 + z < splits) sum += v[z];
    }
  }
  const float scale = scale_or_null != nullptr && from >= 0 ? scale_or_null[from] : 1.0f;
  float f[4] = {sum[0], sum[1], sum[2], sum[3]};
  if (from >= 0 && term.rest != nullptr) term.add<T>(from, c, f);
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] *= scale;
  store_four(out + static_cast<int64_t>(row) * width + c, f);
}
template <typename T>
inline void add_few_launch(const float* planes, int splits, int rows, int width, const float* scale, const int32_t* from, const TargetTerm& term, void* out,
                           hipStream_t stream) {
  const int64_t items = static_cast<int64_t>(rows) * (width / 4);
  hipLaunchKernelGGL((add_few_kernel<T>), dim3(static_cast<unsigned>((items + 255) / 256)), dim3(256), 0, stream, planes, splits, rows, width, scale, from, term,
                     static_cast<T*>(out));
}

// ---- the reduction over the few rows ----------------------------------------------------------------------------------------------
// out[v, k] = scale * sum_t P[v, t] x[t, k] for 64 rows of the result a workgroup, 64 columns a wave at a time. p: [rows in 64, ld], zeros for rows of x that are
// none; turned: few_turned_kernel's. ONE: all of P's packets stay in registers (up to 64 rows of x). 16 bits: up to 64 rows, whose targets' rests are added.
struct FewRests {
  const float* rest;
  const int64_t* target;
  const int32_t *row, *count;   // of x
  const void* x;
  int64_t stride;
};
template <typename T, bool ONE>
__global__ __launch_bounds__(kFewWaves * kWave) void few_outer_kernel(const T* __restrict__ p, const int64_t ld, const T* __restrict__ turned, const int steps,
                                                                      const float* __restrict__ scale, const int rows, const int width, const FewRests rests,
                                                                      T* __restrict__ out) {
  constexpr int V = kFewPack<T>, kSteps = 64 / (4 * V);
  const int lane = threadIdx.x & (kWave - 1), wv = threadIdx.x / kWave, lr = lane & 15, g = lane >> 4;
  const int v0 = blockIdx.x * kFewTokens;
  const float by = *scale;
  const T* from = p + (v0 + lr) * ld + V * g;
  u32x4 held[kSteps][4];
  if constexpr (ONE) {
#pragma unroll
    for (int k = 0; k < kSteps; ++k)
#pragma unroll
      for (int n = 0; n < 4; ++n) held[k][n] = load16(from + n * 16 * ld + min(k, steps - 1) * 4 * V);
  }
  uint64_t here = 0;   // rows whose target is among the workgroup's
  int target = 0;
  if constexpr (sizeof(T) == 2) {
    if (lane < *rests.count) {
      const int64_t at = rests.target[lane] - v0;
      target = at >= 0 && at < kFewTokens && rests.rest[lane] != 0.0f ? static_cast<int>(at) : -1;
    } else {
      target = -1;
    }
    here = __ballot(target >= 0);
  }
  for (int c0 = wv * 64; c0 < width; c0 += kFewWaves * 64) {
    tile_v4f acc[4][4] = {};
    const T* x = turned + (static_cast<int64_t>(c0 / 16) * steps * kWave + lane) * V;
    const auto multiply = [&](int step, const u32x4 (&b)[4]) {
      u32x4 a[4];
#pragma unroll
      for (int m = 0; m < 4; ++m) a[m] = load16(x + (static_cast<int64_t>(m) * steps + step) * kWave * V);
#pragma unroll
      for (int m = 0; m < 4; ++m)
#pragma unroll
        for (int n = 0; n < 4; ++n) acc[m][n] = few_mfma<T>(a[m], b[n], acc[m][n]);
    };
    if constexpr (ONE) {
#pragma unroll
      for (int k = 0; k < kSteps; ++k)
        if (k < steps) multiply(k, held[k]);
    } else {
      for (int k = 0; k < steps; ++k) {
        u32x4 b[4];
#pragma unroll
        for (int n = 0; n < 4; ++n) b[n] = load16(from + n * 16 * ld + k * 4 * V);
        multiply(k, b);
      }
    }
    for (uint64_t left = here; left != 0; left &= left - 1) {
      const int t = __builtin_ctzll(left), at = __builtin_amdgcn_readlane(target, t);
      const T* from = static_cast<const T*>(rests.x) + rests.row[t] * rests.stride + c0;
      const float by = lr == (at & 15) ? rests.rest[t] : 0.0f;
#pragma unroll
      for (int m = 0; m < 4; ++m)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float add = by * to_float(from[(m >> 1) * 32 + 8 * g + 4 * (m & 1) + i]);
#pragma unroll
          for (int n = 0; n < 4; ++n)
            if (n == at >> 4) acc[m][n][i] += lr == (at & 15) ? add : 0.0f;
        }
    }
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      const int v = v0 + n * 16 + lr;
      if (v >= rows) continue;
      T* to = out + static_cast<int64_t>(v) * width + c0;
#pragma unroll
      for (int m = 0; m < 4; ++m)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[m][n][i] *= by;
      if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int m = 0; m < 4; ++m) *reinterpret_cast<tile_v4f*>(to + m * 16 + 4 * g) = acc[m][n];
      } else {
#pragma unroll
        for (int m = 0; m < 4; m += 2)
          store16(to + m * 16 + 8 * g, u32x4{pair_of<T>(acc[m][n][0], acc[m][n][1]), pair_of<T>(acc[m][n][2], acc[m][n][3]),
                                             pair_of<T>(acc[m + 1][n][0], acc[m + 1][n][1]), pair_of<T>(acc[m + 1][n][2], acc[m + 1][n][3])});
      }
    }
  }
}

}  // namespace llmq
