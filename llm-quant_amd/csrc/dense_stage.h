// Matrices brought into the form that the tiles of dense_tile.h take where they are not in it (rows of a multiple of 64, one plane of
// 16-bit values or three of an fp32 matrix): activations, dense weights, and quantized weights as the values (dtype)(code * scale) they
// stand for, which is the matrix that the reference multiplies by when many rows come (`_dequantized_weight`,
// llmquant/quantizers/kernel.py:68-79). And products whose result is a tensor.
#pragma once

#include "dense_few.h"

namespace llmq {

struct StageSource {
  const void* base;        // values [rows, stride], or codes [rows, groups, group_size] (BITS 4: two a byte)
  const float* scale;      // [scale rows, groups] of codes
  const int32_t* gather;   // or null: the row behind each row of the piece; negative: zeros
  int64_t stride;          // elements between rows (values)
  int rows, cols;          // cols: a multiple of 8
  int first_row, piece_rows;   // of the piece; rows at or past `rows` are zeros
  int groups, group_size, keep, out_group;   // codes: `keep` values of a group are columns
};
// [piece_rows, ld] a plane, zeros behind `cols`
struct StageTarget {
  void* rows;
  int64_t plane;   // elements
  int ld;          // a multiple of 8
};

constexpr int kStageAhead = 4;   // packets of a lane in flight
// BITS: 0 values of T, 8 or 4 codes that stand for values of T. Eight values a lane and packet.
template <typename T, int BITS>
__global__ __launch_bounds__(256) void stage_kernel(const StageSource src, const StageTarget to, const int64_t packets) {
  using O = typename TileType<T>::type;
  constexpr int P = TileType<T>::kPlanes;
  const int per_row = to.ld / 8;
  const int64_t threads = static_cast<int64_t>(gridDim.x) * 256;
  for (int64_t p0 = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; p0 < packets; p0 += kStageAhead * threads) {
    u32x4 raw[kStageAhead][sizeof(T) == 4 && BITS == 0 ? 2 : 1];
    float scale[kStageAhead];
    bool real[kStageAhead];
#pragma unroll
    for (int u = 0; u < kStageAhead; ++u) {
      const int64_t p = p0 + u * threads < packets ? p0 + u * threads : packets - 1;
      const int64_t r = p / per_row, row = src.gather != nullptr ? src.gather[r] : src.first_row + r;
      const int c = static_cast<int>(p - r * per_row) * 8;
      real[u] = row >= 0 && row < src.rows && c < src.cols;
      const int64_t from = row < 0 ? 0 : row < src.rows ? row : src.rows - 1;
      const int col = c < src.cols ? c : src.cols - 8;
      scale[u] = 1.0f;
      if constexpr (BITS == 0) {
        const T* x = static_cast<const T*>(src.base) + from * src.stride + col;
        raw[u][0] = load16(x);
        if constexpr (sizeof(T) == 4) raw[u][1] = load16(x + 4);
      } else {
        const int g = col / src.keep, k = col - g * src.keep;
        const int64_t group = from * src.groups + g;
        scale[u] = src.scale[(src.out_group > 0 ? from / src.out_group : from) * src.groups + g];
        const uint8_t* q = static_cast<const uint8_t*>(src.base) + (group * src.group_size + k) * BITS / 8;
        if constexpr (BITS == 8) {
          const u32x2 w = *reinterpret_cast<const u32x2*>(q);
          raw[u][0] = u32x4{w.x, w.y, 0, 0};
        } else {
          raw[u][0] = u32x4{*reinterpret_cast<const uint32_t*>(q), 0, 0, 0};
        }
      }
    }
#pragma unroll
    for (int u = 0; u < kStageAhead; ++u) {
      const int64_t p = p0 + u * threads;
      if (p >= packets) break;
      float f[8];
      if constexpr (BITS == 0) {
        if constexpr (sizeof(T) == 4) {
          Pack<float>::unpack(raw[u][0], f);
          Pack<float>::unpack(raw[u][1], f + 4);
        } else {
          Pack<T>::unpack(raw[u][0], f);
        }
      } else if constexpr (BITS == 8) {
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = static_cast<float>(static_cast<int8_t>((i < 4 ? raw[u][0].x : raw[u][0].y) >> (8 * (i % 4)))) * scale[u];
      } else {
        const uint32_t signs = raw[u][0].x ^ 0x88888888u;   // (code + 8 with its top bit flipped: the code)
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = static_cast<float>(static_cast<int32_t>(signs << (28 - 4 * i)) >> 28) * scale[u];
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = real[u] ? f[i] : 0.0f;
      if constexpr (P == 1) {
        store16(static_cast<uint16_t*>(to.rows) + p * 8, Pack<O>::pack(f));   // (values of T come back as they were)
      } else {
        uint16_t v[3][8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          uint16_t s[3];
          planes_of(f[i], s);
#pragma unroll
          for (int j = 0; j < 3; ++j) v[j][i] = s[j];
        }
#pragma unroll
        for (int j = 0; j < 3; ++j) {
          u32x4 w;
          w.x = v[j][0] | static_cast<uint32_t>(v[j][1]) << 16;
          w.y = v[j][2] | static_cast<uint32_t>(v[j][3]) << 16;
          w.z = v[j][4] | static_cast<uint32_t>(v[j][5]) << 16;
          w.w = v[j][6] | static_cast<uint32_t>(v[j][7]) << 16;
          store16(static_cast<uint16_t*>(to.rows) + j * to.plane + p * 8, w);
        }
      }
    }
  }
}

template <typename T>
inline void stage_launch(const StageSource& src, const StageTarget& to, int bits, hipStream_t stream) {
  const int64_t packets = static_cast<int64_t>(src.piece_rows) * (to.ld / 8), blocks = (packets + 256 * kStageAhead - 1) / (256 * kStageAhead);
  const dim3 grid(static_cast<unsigned>(blocks < 256 * 32 ? blocks : 256 * 32));
  if (bits == 0) hipLaunchKernelGGL((stage_kernel<T, 0>), grid, dim3(256), 0, stream, src, to, packets);
  else if (bits == 8) hipLaunchKernelGGL((stage_kernel<T, 8>), grid, dim3(256), 0, stream, src, to, packets);
  else hipLaunchKernelGGL((stage_kernel<T, 4>), grid, dim3(256), 0, stream, src, to, packets);
}

// ---- products whose result is a tensor ------------------------------------------------------------------------------------
// Rows of B a tile takes: 64 where there are no more, else 256 (a tile of few rows is bound by A's bytes, not by the
// multiplications that its empty rows waste).
constexpr int kFewRows = 64;
constexpr int tile_rows(int rows) { return rows <= kFewRows ? kFewRows : 256; }

// How a sum over K is dealt out: the tiles of the rows there are, and as many splits of K as the chip has places for, `most` at the most.
struct Splits {
  int n_tiles, splits;
  int64_t plane;   // elements of a split's fp32 sums: whole tiles of rows
};
__host__ __device__ inline Splits splits_of_rows(int rows, int tn, int m_tiles, int64_t ld, int most) {
  Splits s;
  s.n_tiles = (rows + tn - 1) / tn;
  const int places = tn == kFewRows ? 512 : 256, tiles = s.n_tiles * m_tiles;
  s.splits = tiles > 0 && places / tiles > 1 ? places / tiles : 1;
  if (s.splits > most) s.splits = most;
  s.plane = static_cast<int64_t>(s.n_tiles) * tn * ld;
  return s;
}
// splits of eight steps at least, sixteen at the most
inline int most_splits(int m_rows, int n_rows, int k) {
  const Splits s = splits_of_rows(n_rows < 256 ? n_rows : 256, tile_rows(n_rows), (m_rows + 255) / 256, m_rows, 16);   // (a tile of rows alone)
  const int most = k / 64 / 8;
  return s.splits < most ? s.splits : most < 1 ? 1 : most;
}
// bytes of the sums, however many of the rows there turn out to be
inline int64_t sums_bytes(int m_rows, int n_rows, int most) {
  const int tn = tile_rows(n_rows), m_tiles = (m_rows + 255) / 256;
  int64_t largest = 0;
  for (int n = tn; n < n_rows + tn; n += tn) {
    const Splits s = splits_of_rows(n, tn, m_tiles, m_rows, most);
    if (s.plane * s.splits > largest) largest = s.plane * s.splits;
  }
  return largest * 4;
}

// out[n, m] = sum_k A[m, k] B[n, k], n < B's rows, m < A's rows, A with K outermost, B (B_K) too or not. SUMS: fp32 planes, one a split of K, added
// to what is there unless `first`; else the type of the call, times *scale (null: 1).
struct ProductOut {
  void* base;
  int64_t ld;          // elements
  const float* scale;
  int first, most;     // most: splits
  const int32_t* count = nullptr;   // or null: how many rows (of B, or with B_K of K) there are; tiles and steps past them are left out
  // B_K, 16 bits: what is added for row t of K to the result's row target[t] - first_token, rest[t] times row `row[t]` of x; null: nothing
  const float* rest = nullptr;
  const int64_t* target = nullptr;
  const int32_t* row = nullptr;
  const void* x = nullptr;
  int64_t x_stride = 0, first_token = 0;
};

template <typename T, int TM, int TN, int WM, int WN, bool SUMS, bool B_K>
__global__ __launch_bounds__(WM * WN * kWave) void product_kernel(const TileOperand a, const TileOperand b, const int k,
                                                                       const int m_tiles, const ProductOut out) {
  using O = typename TileType<T>::type;
  using Tile = DenseTile<O, TM, TN, WM, WN, true, B_K>;
  constexpr int kBlockN = 4;
  __shared__ __attribute__((aligned(16))) uint8_t s_mem[Tile::kLdsBytes];
  const int rows = out.count != nullptr ? *out.count : INT32_MAX;
  const int steps = ((B_K ? min(k, rows) : k) + Tile::kStep - 1) / Tile::kStep;
  const Splits s = splits_of_rows(B_K ? b.rows : min(b.rows, rows), TN, m_tiles, out.ld, out.most);
  const int tiles = m_tiles * s.n_tiles, id = blockIdx.x;
  if (id >= tiles * s.splits) return;
  // Workgroups that run together on an XCD are 32 neighbours of this order: a split's tiles in blocks of four of n, by m, by n: eight tiles of A by four
  // of B. (By m alone, the splits side by side, an XCD's step read 36 tiles of operands where these are 12: 2048 x 4096 over 14336 259 us.)
  const int at = tile_of_workgroup(id, tiles * s.splits), z = at / tiles, tile = at - z * tiles;
  const int block = tile / (m_tiles * kBlockN), in_block = tile - block * m_tiles * kBlockN, wide = min(kBlockN, s.n_tiles - block * kBlockN);
  const int m0 = in_block / wide * TM, n0 = (block * kBlockN + in_block % wide) * TN;
  const int per = (steps + s.splits - 1) / s.splits, k0 = min(z * per, steps) * Tile::kStep, k1 = min((z + 1) * per, steps) * Tile::kStep;
  if (SUMS && k0 >= k1 && !out.first) return;   // nothing of K is this split's; where the sums begin they are zeros
  Tile t;
  if (k0 < k1) t.template multiply<(TileType<T>::kPlanes == 3 ? 6 : 1)>(s_mem, a, m0, b, n0, k0, k1);
  else t.clear();
  if constexpr (!SUMS && B_K && sizeof(T) == 2) {
    // the rows of K whose target is one of the tile's, in their order, 2048 rows a time, and of those 32 a product
    constexpr int kEach = 4, kThreads = WM * WN * kWave;
    struct Rest {
      int row, n;
      float by;
    };
    Rest* const list = reinterpret_cast<Rest*>(s_mem);
    int* const found = reinterpret_cast<int*>(list + kEach * kThreads);   // [kEach][waves]
    const int lane = threadIdx.x & (kWave - 1), wv = threadIdx.x / kWave, lr = lane & 15, g = lane >> 4;
    const int last = min(k, rows) - 1;
    for (int i0 = 0; out.rest != nullptr && i0 <= last; i0 += kEach * kThreads) {
      uint64_t hit[kEach];
      Rest mine[kEach];
      __syncthreads();
#pragma unroll
      for (int j = 0; j < kEach; ++j) {
        const int i = i0 + j * kThreads + threadIdx.x, at = min(i, last);
        const int64_t n = out.target[at] - out.first_token - n0;
        mine[j] = Rest{out.row[at], static_cast<int>(n), out.rest[at]};
        hit[j] = __ballot(i == at && n >= 0 && n < TN && mine[j].by != 0.0f);
        if (lane == 0) found[j * WM * WN + wv] = __popcll(hit[j]);
      }
      __syncthreads();
      int all = 0;
#pragma unroll
      for (int j = 0; j < kEach; ++j) {
        int first = all;
        for (int w = 0; w < WM * WN; ++w) {
          if (w < wv) first += found[j * WM * WN + w];
          all += found[j * WM * WN + w];
        }
        if (hit[j] >> lane & 1) list[first + __popcll(hit[j] & ((uint64_t{1} << lane) - 1))] = mine[j];
      }
      __syncthreads();
      for (int e0 = 0; e0 < all; e0 += 32) {   // lane 16 g + r: rows 8 g .. of the 32, of A's and B's r
        Rest of[8];
        uint32_t word[4];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          of[e] = list[min(e0 + 8 * g + e, all - 1)];
          if (e0 + 8 * g + e >= all) of[e].n = -1;
        }
        u32x4 x[Tile::MI];
#pragma unroll
        for (int mi = 0; mi < Tile::MI; ++mi) {
          const T* from = static_cast<const T*>(out.x) + min(m0 + wv / WN * (TM / WM) + mi * 16 + lr, a.rows - 1);
          uint16_t v[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = __builtin_bit_cast(uint16_t, from[of[e].row * out.x_stride]);
          x[mi] = u32x4{v[0] | static_cast<uint32_t>(v[1]) << 16, v[2] | static_cast<uint32_t>(v[3]) << 16, v[4] | static_cast<uint32_t>(v[5]) << 16,
                        v[6] | static_cast<uint32_t>(v[7]) << 16};
        }
#pragma unroll
        for (int ni = 0; ni < Tile::NI; ++ni) {
          const int n = wv % WN * (TN / WN) + ni * 16 + lr;
#pragma unroll
          for (int e = 0; e < 4; ++e) word[e] = pair_of<T>(of[2 * e].n == n ? of[2 * e].by : 0.0f, of[2 * e + 1].n == n ? of[2 * e + 1].by : 0.0f);
          const u32x4 by{word[0], word[1], word[2], word[3]};
#pragma unroll
          for (int mi = 0; mi < Tile::MI; ++mi) t.acc[mi][ni] = mfma_16x16x32<T>(x[mi], by, t.acc[mi][ni]);
        }
      }
    }
  }
  const float scale = SUMS || out.scale == nullptr ? 1.0f : *out.scale;
#pragma unroll
  for (int ni = 0; ni < Tile::NI; ++ni) {
    const int n = n0 + Tile::col_of(ni);
    if (n >= b.rows) continue;
#pragma unroll
    for (int mi = 0; mi < Tile::MI; ++mi) {
      const int m = m0 + Tile::row_of(mi, 0);
      if (m >= a.rows) continue;   // (rows of A are a multiple of 4)
      if constexpr (SUMS) {
        float* to = static_cast<float*>(out.base) + z * s.plane + n * out.ld + m;
        tile_v4f v = t.acc[mi][ni];
        if (!out.first) v += *reinterpret_cast<const tile_v4f*>(to);
        *reinterpret_cast<tile_v4f*>(to) = v;
      } else {
        T* to = static_cast<T*>(out.base) + n * out.ld + m;
        const float f[4] = {t.acc[mi][ni][0] * scale, t.acc[mi][ni][1] * scale, t.acc[mi][ni][2] * scale, t.acc[mi][ni][3] * scale};
        if constexpr (sizeof(T) == 4) {
          *reinterpret_cast<tile_v4f*>(to) = tile_v4f{f[0], f[1], f[2], f[3]};
        } else {
          const T h[4] = {from_float<T>(f[0]), from_float<T>(f[1]), from_float<T>(f[2]), from_float<T>(f[3])};
          *reinterpret_cast<u32x2*>(to) = __builtin_bit_cast(u32x2, h);
        }
      }
    }
  }
}

template <typename T, bool SUMS, bool B_K>
inline void product_launch(const TileOperand& a, const TileOperand& b, int k, const ProductOut& out, hipStream_t stream) {
  const int m_tiles = (a.rows + 255) / 256, tn = tile_rows(b.rows);
  unsigned groups = 0;   // (the most that there can be, however many rows count)
  for (int n = out.count != nullptr && !B_K ? tn : (b.rows + tn - 1) / tn * tn; n < b.rows + tn; n += tn) {
    const Splits s = splits_of_rows(n, tn, m_tiles, out.ld, out.most);
    if (static_cast<unsigned>(m_tiles) * s.n_tiles * s.splits > groups) groups = static_cast<unsigned>(m_tiles) * s.n_tiles * s.splits;
  }
  // (64 x 128 a wave: the transposing reads bring half as much an instruction, so that fewer of A's are better where B has none)
  if (tn == kFewRows) hipLaunchKernelGGL((product_kernel<T, 256, 64, 4, 2, SUMS, B_K>), dim3(groups), dim3(512), 0, stream, a, b, k, m_tiles, out);
  else hipLaunchKernelGGL((product_kernel<T, 256, 256, 4, 2, SUMS, B_K>), dim3(groups), dim3(512), 0, stream, a, b, k, m_tiles, out);
}

// out[n, m] = (dtype)(scale * the sum of the planes), eight values a lane. from: the planes' row behind each row (negative: zeros), and with it scale: a value for
// each of the planes' rows; or null.
template <typename T>
__global__ __launch_bounds__(256) void add_planes_kernel(const float* __restrict__ planes, const int rows, const int tn, const int m_tiles, const int most,
                                                         const int32_t* __restrict__ count_or_null, const float* __restrict__ scale_or_null,
                                                         const int32_t* __restrict__ from_or_null, const TargetTerm term, T* __restrict__ out,
                                                         const int64_t packets, const int per_row) {
  constexpr int kAhead = 4;
  const Splits s = splits_of_rows(count_or_null == nullptr ? rows : min(rows, *count_or_null), tn, m_tiles, per_row * int64_t{8}, most);
  const int64_t plane = s.plane;
  const int splits = s.splits;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < packets; i += static_cast<int64_t>(gridDim.x) * 256) {
    float f[8] = {};
    int64_t at = i;
    int from = -1;
    if (from_or_null != nullptr) {
      const int64_t row = i / per_row;
      from = from_or_null[row];
      at = from < 0 ? -1 : from * static_cast<int64_t>(per_row) + (i - row * per_row);
    }
    if (at >= 0) {
      for (int z0 = 0; z0 < splits; z0 += kAhead) {
        tile_v4f lo[kAhead], hi[kAhead];
#pragma unroll
        for (int z = 0; z < kAhead; ++z) {
          const float* p = planes + min(z0 + z, splits - 1) * plane + at * 8;
          lo[z] = *reinterpret_cast<const tile_v4f*>(p);
          hi[z] = *reinterpret_cast<const tile_v4f*>(p + 4);
        }
#pragma unroll
        for (int z = 0; z < kAhead; ++z)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (z0 + z < splits) {
              f[e] += lo[z][e];
              f[4 + e] += hi[z][e];
            }
      }
    }
    if (term.rest != nullptr && from >= 0) {   // (with `from` alone)
      const int c = static_cast<int>(i % per_row) * 8;
      term.add<T>(from, c, f);
      term.add<T>(from, c + 4, f + 4);
    }
    const float scale = scale_or_null == nullptr || from < 0 ? 1.0f : scale_or_null[from];
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] *= scale;
#pragma unroll
    for (int e = 0; e < 8; e += Pack<T>::N) store16(out + i * 8 + e, Pack<T>::pack(f + e));
  }
}
// (rows and most as the products had them)
template <typename T>
inline void add_planes_launch(const float* planes, int rows, int width, int most, const int32_t* count, const float* scale, const int32_t* from,
                              const TargetTerm& term, void* out, hipStream_t stream) {
  const int64_t packets = static_cast<int64_t>(rows) * (width / 8), blocks = (packets + 255) / 256;
  hipLaunchKernelGGL((add_planes_kernel<T>), dim3(static_cast<unsigned>(blocks < 8192 ? blocks : 8192)), dim3(256), 0, stream,
                     planes, rows, tile_rows(rows), (width + 255) / 256, most, count, scale, from, term, static_cast<T*>(out), packets, width / 8);
}

inline int64_t round_up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }

}  // namespace llmq
