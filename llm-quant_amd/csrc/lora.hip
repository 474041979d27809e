// Low-rank adapters of many requests beside a shared projection, and their gradients, gfx950 (no counterpart among the
// reference's kernels). For row t of request b with adapter a = adapter[b], A[a] [rank, in], B[a] [out, rank], scaling s[a]:
//
//   low[t] = x[t] A[a]^T          out[t] = base[t] + s[a] low[t] B[a]^T
//   du[t] = s[a] g[t] B[a]        gx[t] = gbase[t] + du[t] A[a]     gA[a] = sum_t du[t]^T x[t]     gB[a] = s[a] sum_t g[t]^T low[t]
//
// shrink   rows by a bank's rows: the reduction is long (in, or out), the result 8 to 128 wide. A workgroup takes a piece of one
//          request's rows, its waves parts of the reduction.
// expand   multiplies that by the other factor into the projection's output: a wave has 128 columns.
// step     both at once for single rows beside small banks: every workgroup of a row makes its `low` again.
// outer    gradients of the bank: the reduction is over rows, which are sorted by adapter (plan) in blocks of 32. Both operands lie
//          with the reduction outermost; a lane loads eight columns of its eight rows and turns them over in registers.
// All on the matrix core in fp32 sums (step: fp32 arithmetic). The 8 to 128 numbers in between stay fp32 in memory; as operands they are two bfloat16 (16 bits of
// them), against bfloat16 values as they are. For fp16: two fp16 with one exponent a row in expand (22 bits; 333 rows of 20 requests by 14336 with the bank as two
// bfloat16 instead 21.1 us, so 19.3), two bfloat16 against values as two bfloat16 (exact) in outer, whose rows are the reduction. fp32 on the fp32 matrix
// instructions. Rounded once, at the end. Every sum has a fixed order.
//
// Bound: HBM for prompts and training (x, base and out once each); the chain of a launch for single tokens.
#include "dense_tile.h"
#include "kv_blocks.h"

namespace {

using namespace llmq;

typedef tile_v4f v4f;

struct Bank {
  const void* m;      // [slots, rows of a slot, width]
  int slots, rank;
  int width;
};
struct Requests {
  const int32_t* adapter;
  Ragged rows;
  // The rows of piece `slot` (of 16 NT rows, or one row a request) and their adapter; no rows: nobody's.
  template <int SHIFT> __device__ __forceinline__ int piece(int slot, int slots, int& first, int& n) const {
    int a = -1;
    if (rows.start == nullptr) {
      first = slot;
      n = 1;
      a = adapter[slot];
    } else {
      Span span;
      const int b = rows.find(SHIFT, adapter, slot, span, a);
      (void)b;
      first = span.first + (slot << SHIFT);
      n = min(span.n - (slot << SHIFT), 1 << SHIFT);
    }
    return a >= 0 && a < slots ? a : -1;
  }
};

template <int NT> constexpr int kPieceShift = NT == 2 ? 5 : 4;

__device__ __forceinline__ v4f mfma_f32(float a, float b, v4f c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }
template <typename T> __device__ __forceinline__ v4f mfma_packet(u32x4 a, u32x4 b, v4f c) { return mfma_16x16x32<T>(a, b, c); }
template <> __device__ __forceinline__ v4f mfma_packet<float>(u32x4 a, u32x4 b, v4f c) {
  c = mfma_f32(__builtin_bit_cast(float, a.x), __builtin_bit_cast(float, b.x), c);
  c = mfma_f32(__builtin_bit_cast(float, a.y), __builtin_bit_cast(float, b.y), c);
  c = mfma_f32(__builtin_bit_cast(float, a.z), __builtin_bit_cast(float, b.z), c);
  return mfma_f32(__builtin_bit_cast(float, a.w), __builtin_bit_cast(float, b.w), c);
}

// eight floats as two bfloat16 each: f = hi + lo to 2^-16 of f
struct HiLo {
  u32x4 hi, lo;
};
__device__ __forceinline__ float bf16_low(uint32_t w) { return __builtin_bit_cast(float, w << 16); }
__device__ __forceinline__ float bf16_high(uint32_t w) { return __builtin_bit_cast(float, w & 0xffff0000u); }
__device__ __forceinline__ HiLo hi_lo(const float* f) {
  HiLo r;
  uint32_t h[4], l[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    h[i] = bf16_pair_rne(f[2 * i], f[2 * i + 1]);
    l[i] = bf16_pair_rne(f[2 * i] - bf16_low(h[i]), f[2 * i + 1] - bf16_high(h[i]));
  }
  r.hi = u32x4{h[0], h[1], h[2], h[3]};
  r.lo = u32x4{l[0], l[1], l[2], l[3]};
  return r;
}

template <typename T> __device__ __forceinline__ void store_four(T* to, const float* f) {   // four neighbouring values
  if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<v4f*>(to) = v4f{f[0], f[1], f[2], f[3]};
  } else {
    const T h[4] = {from_float<T>(f[0]), from_float<T>(f[1]), from_float<T>(f[2]), from_float<T>(f[3])};
    *reinterpret_cast<u32x2*>(to) = __builtin_bit_cast(u32x2, h);
  }
}

// ---- shrink -----------------------------------------------------------------------------------------------------------------
// RT: tiles of 16 of the rank, NT: of rows. A step is 128 bytes of a row. A workgroup of eight waves (four for ranks above 32) takes 16 or 32 rows, each wave every
// eighth step of the reduction, through LDS of its own: transfers of eight whole rows' 128 bytes (read as operands, 16 bytes of 16 rows, an instruction meets
// 64 pieces of lines: 4099 rows of 4096 24.7 us where this takes 11.2), chunks swizzled by the row, no barrier but the one meeting at the end. Where
// rows are few the reduction is cut for several workgroups (splits_of).
constexpr int shrink_waves(int rank) { return rank > 32 ? 4 : 8; }   // (two workgroups a CU at least, for their LDS)
template <int RT> constexpr int kShrinkWaves = RT >= 4 ? 4 : 8;
template <int RT, int NT> constexpr int kShrinkAhead = RT + NT <= 2 ? 2 : 1;   // steps of a wave in flight
template <typename T, int RT, int NT>
__global__ __launch_bounds__((kShrinkWaves<RT> * kWave)) void shrink_kernel(const T* __restrict__ x, const int64_t x_stride, const Bank bank,
                                                                            const Requests req, float* __restrict__ planes, const int64_t plane) {
  constexpr int V = Pack<T>::N, kWaves = kShrinkWaves<RT>, U = kShrinkAhead<RT, NT>, kTile = 2048, kStepBytes = (RT + NT) * kTile;
  constexpr int kStages = kWaves * U * kStepBytes, kSums = kWaves / 2 * RT * NT * 1024;
  __shared__ __attribute__((aligned(16))) uint8_t s_mem[kStages > kSums ? kStages : kSums];
  int first, n;
  const int a = req.template piece<kPieceShift<NT>>(blockIdx.x, bank.slots, first, n);
  if (n <= 0 || a < 0) return;
  const int lane = threadIdx.x & (kWave - 1), wv = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / kWave), lr = lane & 15, g = lane >> 4;
  const int packets = bank.width / V, steps = (packets + 7) / 8, splits = gridDim.y;
  const int s0 = static_cast<int>(static_cast<int64_t>(steps) * blockIdx.y / splits), s1 = static_cast<int>(static_cast<int64_t>(steps) * (blockIdx.y + 1) / splits);
  // transfers: eight rows each, lane = (row, slot); slot p of row r holds chunk p ^ (r & 7)
  const BufferBase xb = buffer_base(x + static_cast<int64_t>(first) * x_stride),
                   mb = buffer_base(static_cast<const T*>(bank.m) + static_cast<int64_t>(a) * bank.rank * bank.width);
  const int tr = lane >> 3, chunk = (lane & 7) ^ tr;
  uint32_t xo[2 * NT], mo[2 * RT];
#pragma unroll
  for (int i = 0; i < 2 * NT; ++i) xo[i] = static_cast<uint32_t>(min(i * 8 + tr, n - 1) * x_stride * static_cast<int64_t>(sizeof(T)));
#pragma unroll
  for (int i = 0; i < 2 * RT; ++i) mo[i] = static_cast<uint32_t>(min(i * 8 + tr, bank.rank - 1)) * static_cast<uint32_t>(bank.width * sizeof(T));
  uint8_t* const mine = s_mem + wv * U * kStepBytes;
  const uint32_t at0 = lr * 128 + ((g ^ (lr & 7)) << 4);   // chunk g of row lr; chunk g + 4: ^ 64
  v4f acc[RT][NT] = {};
  for (int s = s0 + wv; s < s1; s += kWaves * U) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int at = s + u * kWaves;
      if (at >= s1) break;   // (the wave's)
      const uint32_t byte = static_cast<uint32_t>(min(at * 8 + chunk, packets - 1)) * 16u;   // (past the row's end: its last packet, zeros below)
      uint8_t* stage = mine + u * kStepBytes;
#pragma unroll
      for (int i = 0; i < 2 * NT; ++i) buffer_to_lds<16>(xb, stage + i * 1024, xo[i] + byte, 0);
#pragma unroll
      for (int i = 0; i < 2 * RT; ++i) buffer_to_lds<16>(mb, stage + NT * kTile + i * 1024, mo[i] + byte, 0);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int at = s + u * kWaves;
      if (at >= s1) break;
      const uint8_t* stage = mine + u * kStepBytes;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        u32x4 xv[NT], mv[RT];
#pragma unroll
        for (int i = 0; i < NT; ++i) xv[i] = load16(stage + i * kTile + (at0 ^ (h << 6)));
#pragma unroll
        for (int i = 0; i < RT; ++i) mv[i] = load16(stage + (NT + i) * kTile + (at0 ^ (h << 6)));
        if (at * 8 + 8 > packets && at * 8 + 4 * h + g >= packets) {   // the row's last step
#pragma unroll
          for (int i = 0; i < NT; ++i) xv[i] = u32x4{0, 0, 0, 0};
#pragma unroll
          for (int i = 0; i < RT; ++i) mv[i] = u32x4{0, 0, 0, 0};
        }
#pragma unroll
        for (int i = 0; i < RT; ++i)
#pragma unroll
          for (int j = 0; j < NT; ++j) acc[i][j] = mfma_packet<T>(mv[i], xv[j], acc[i][j]);
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // (the stages are asked for again)
  }
  __syncthreads();
  v4f* const s_sum = reinterpret_cast<v4f*>(s_mem);
#pragma unroll
  for (int half = kWaves / 2; half > 0; half /= 2) {   // a tree over the waves
    if (wv >= half && wv < 2 * half) {
#pragma unroll
      for (int i = 0; i < RT * NT; ++i) s_sum[((wv - half) * RT * NT + i) * kWave + lane] = acc[i / NT][i % NT];
    }
    __syncthreads();
    if (wv < half) {
#pragma unroll
      for (int i = 0; i < RT * NT; ++i) acc[i / NT][i % NT] += s_sum[(wv * RT * NT + i) * kWave + lane];
    }
    __syncthreads();
  }
  if (wv > 0) return;
#pragma unroll
  for (int i = 0; i < RT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const int r = i * 16 + 4 * g, t = j * 16 + lr;   // four of the rank, a row
      if (t < n && r < bank.rank)
        *reinterpret_cast<v4f*>(planes + blockIdx.y * plane + static_cast<int64_t>(first + t) * bank.rank + r) = acc[i][j];
    }
}

// ---- expand -----------------------------------------------------------------------------------------------------------------
constexpr int kExpandWaves = 4;

struct Expand {
  const float* planes;     // [splits][rows][rank]
  int64_t plane;
  int splits;
  const float* scaling;    // [slots]
  const void* base;        // or null: zeros
  int64_t base_stride;
  void* out;               // [rows, width], contiguous
  float* low;              // or null: [rows, rank], the sum of the planes (where there are several) and zeros without an adapter
  int rows, columns;       // columns of out
  int pieces, rest;        // pieces of requests, for each 512 columns (blockIdx.y); workgroups of the last y, for rows of no request (0: there is none)
};

// Rows in front of the first request and behind the last one: the base as it is, no sums.
template <typename T> __device__ __forceinline__ void rows_of_nobody(const int rank, const Ragged& rows, const Expand& e, const int id) {
  constexpr int V = Pack<T>::N;
  const int begin = rows.first(0), end = max(rows.first(rows.sequences), begin), packets = e.columns / V;
  const int64_t n = begin + e.rows - end, step = int64_t{kExpandWaves} * kWave * e.rest;
  for (int64_t i = static_cast<int64_t>(id) * kExpandWaves * kWave + threadIdx.x; i < n * packets; i += step) {
    const int64_t at = i / packets, row = at < begin ? at : at - begin + end, c = (i - at * packets) * V;
    const u32x4 v = e.base == nullptr ? u32x4{0, 0, 0, 0} : load16(static_cast<const T*>(e.base) + row * e.base_stride + c);
    store16(static_cast<T*>(e.out) + row * e.columns + c, v);
  }
  if (e.low == nullptr) return;
  for (int64_t i = static_cast<int64_t>(id) * kExpandWaves * kWave + threadIdx.x; i < n * rank; i += step) {
    const int64_t at = i / rank, row = at < begin ? at : at - begin + end;
    e.low[row * rank + (i - at * rank)] = 0.0f;
  }
}

// the power of two that brings a row of largest magnitude `most` (its bits) to [2^13, 2^14); 0 for nothing, an infinity or NaN
__device__ __forceinline__ int row_exponent(uint32_t most) {
  const int e = static_cast<int>(most >> 23);
  return e == 0 || e == 255 ? 0 : 127 + 13 - e;
}

// 128 columns a wave: lane 16 g + r has columns 8 r .. 8 r + 7, one of each of eight tiles, of rows 4 g .. 4 g + 3, so that 16 lanes read and
// write 256 neighbouring bytes of a row (with rows over the lanes, 64 bytes of each of 16: 4099 rows of 4096 23 us where this takes 18.8). What does not depend on the
// rows' sums, the weights and the base, is asked for first. The bank here is [slots][columns][rank].
template <typename T, int RT, int NT>
__global__ __launch_bounds__(kExpandWaves * kWave) void expand_kernel(const Bank bank, const Requests req, const Expand e) {
  constexpr int V = Pack<T>::N, KT = (RT * 16 + 4 * V - 1) / (4 * V);   // steps of the rank: 32 (fp32: 16)
  constexpr int kBlocks = KT * NT, kParts = kBlocks == 1 ? 4 : kBlocks == 2 ? 2 : 1;   // operands of `low`; threads for each packet of one
  constexpr bool kStaged = sizeof(T) == 2 && RT <= 4;   // the bank's rows of a wave's columns through LDS
  __shared__ u32x4 s_low[sizeof(T) == 4 ? 1 : 2][kBlocks][kWave];
  constexpr bool kHalf = __is_same(T, f16_t);
  __shared__ uint32_t s_most[kHalf ? 16 * NT : 1];        // fp16: the largest magnitude of each row of `low`, as bits
  __shared__ __attribute__((aligned(16))) uint8_t s_bank[kStaged ? kExpandWaves * 4096 * RT : 16];
  const int lane = threadIdx.x & (kWave - 1), wv = threadIdx.x / kWave, lr = lane & 15, g = lane >> 4;
  const int groups = static_cast<int>(gridDim.y) - (e.rest > 0 ? 1 : 0);
  if (static_cast<int>(blockIdx.y) >= groups) {
    if (static_cast<int>(blockIdx.x) < e.rest) rows_of_nobody<T>(bank.rank, req.rows, e, blockIdx.x);
    return;
  }
  // the pieces of the same columns to one XCD, whose cache has the bank's rows for them
  const int item = tile_of_workgroup(blockIdx.x + blockIdx.y * gridDim.x, groups * gridDim.x), group = item / e.pieces;
  int first, n;
  const int a = req.template piece<kPieceShift<NT>>(item - group * e.pieces, bank.slots, first, n);
  if (n <= 0) return;
  const int c0 = (group * kExpandWaves + wv) * 128;
  if (a < 0 && e.low != nullptr && c0 == 0) {   // (no adapter: zeros)
    for (int i = lane; i < n * bank.rank; i += kWave) e.low[static_cast<int64_t>(first) * bank.rank + i] = 0.0f;
  }
  const int c = c0 + 8 * lr;   // (columns are a multiple of 8)
  const bool here = c < e.columns;
  u32x4 m[kStaged ? 1 : KT][8], base[NT][4][8 / V];
  uint8_t* const mine = s_bank + __builtin_amdgcn_readfirstlane(wv) * (kStaged ? 4096 * RT : 0);
  const int per = bank.rank / V;   // packets of a column
  if constexpr (kStaged) {
    if (a >= 0 && c0 < e.columns) {   // (past the columns: the last packet again)
      const BufferBase mb = buffer_base(static_cast<const T*>(bank.m) + (static_cast<int64_t>(a) * e.columns + c0) * bank.rank);
      const uint32_t eight = 0xffffffffu / static_cast<uint32_t>(8 * per) + 1;   // (a division by the packets of eight columns)
      const int most = min(e.columns - c0, 128) * per - 1;
#pragma unroll
      for (int i = 0; i < 4 * RT; ++i) {
        if (i >= 2 * per) break;
        const int at = i * kWave + lane, packet = at ^ (static_cast<int>(__umulhi(at, eight)) & 7);
        buffer_to_lds<16>(mb, mine + i * 1024, static_cast<uint32_t>(min(packet, most)) * 16u, 0);
      }
    }
  } else if (a >= 0) {
#pragma unroll
    for (int k = 0; k < KT; ++k)
#pragma unroll
      for (int mi = 0; mi < 8; ++mi)   // (past the rank the operand of `low` is zeros, against weights that are looked at a second time)
        m[k][mi] = load16(static_cast<const T*>(bank.m) + (static_cast<int64_t>(a) * e.columns + min(c + mi, e.columns - 1)) * bank.rank +
                          min((k * 4 + g) * V, bank.rank - V));
  }
  if (e.base != nullptr) {
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const T* from = static_cast<const T*>(e.base) + (first + min(j * 16 + 4 * g + i, n - 1)) * e.base_stride + min(c, e.columns - 8);
#pragma unroll
        for (int h = 0; h < 8 / V; ++h) base[j][i][h] = load16(from + h * V);
      }
  }
  v4f acc[NT][8] = {};
  if (a >= 0) {   // (the workgroup's)
    // `low` of the piece as operands, made once: packet (row 16 j + lr, values (4 k + g) V ..) by kParts threads, a part of the planes each
    constexpr int kEach = kWave / kParts, kTurns = (kBlocks * kParts + kExpandWaves - 1) / kExpandWaves;
    const float s = e.scaling[a];
    float sums[kHalf ? kTurns : 1][V];
    if constexpr (kHalf) {
      if (threadIdx.x < 16 * NT) s_most[threadIdx.x] = 0;
      __syncthreads();
    }
#pragma unroll
    for (int i0 = 0; i0 < kBlocks * kParts; i0 += kExpandWaves) {
      const int packet = (i0 + wv) * kEach + lane % kEach, part = lane / kEach, block = packet / kWave, pl = packet % kWave;
      if (block >= kBlocks) break;
      const int j = block % NT, r = (block / NT * 4 + (pl >> 4)) * V, t = j * 16 + (pl & 15);
      const float* at = e.planes + static_cast<int64_t>(first + min(t, n - 1)) * bank.rank + min(r, bank.rank - V);
      v4f sum[V / 4] = {};
      constexpr int kAhead = 4;
      for (int p0 = part; p0 < e.splits; p0 += kAhead * kParts) {
        v4f v[kAhead][V / 4];
#pragma unroll
        for (int p = 0; p < kAhead; ++p)
#pragma unroll
          for (int i = 0; i < V / 4; ++i) v[p][i] = *reinterpret_cast<const v4f*>(at + min(p0 + p * kParts, e.splits - 1) * e.plane + 4 * i);
#pragma unroll
        for (int p = 0; p < kAhead; ++p)
#pragma unroll
          for (int i = 0; i < V / 4; ++i)
            if (p0 + p * kParts < e.splits) sum[i] += v[p][i];
      }
      float f[V];
#pragma unroll
      for (int i = 0; i < V; ++i) {
        float v = sum[i / 4][i % 4];
        if constexpr (kParts > 1) {
#pragma unroll
          for (int d = kEach; d < kWave; d *= 2) v += __shfl_xor(v, d);
        }
        f[i] = v;
      }
      if (part != 0) continue;
      if (e.splits > 1 && e.low != nullptr && group == 0 && t < n && r < bank.rank) {
        float* to = e.low + static_cast<int64_t>(first + t) * bank.rank + r;
#pragma unroll
        for (int i = 0; i < V; i += 4) *reinterpret_cast<v4f*>(to + i) = v4f{f[i], f[i + 1], f[i + 2], f[i + 3]};
      }
#pragma unroll
      for (int i = 0; i < V; ++i) f[i] = r < bank.rank ? f[i] * s : 0.0f;
      if constexpr (sizeof(T) == 4) {
        s_low[0][block][pl] = Pack<float>::pack(f);
      } else if constexpr (kHalf) {
        uint32_t most = 0;
#pragma unroll
        for (int i = 0; i < V; ++i) {
          sums[i0 / kExpandWaves][i] = f[i];
          most = max(most, __builtin_bit_cast(uint32_t, f[i]) & 0x7fffffffu);
        }
        atomicMax(&s_most[t], most);   // (of positive floats the order of their bits, NaN above all)
      } else {
        const HiLo low = hi_lo(f);
        s_low[0][block][pl] = low.hi;
        s_low[1][block][pl] = low.lo;
      }
    }
    if constexpr (kHalf) {   // rows scaled to at most 2^14, as two fp16: 22 bits, and 2^-38 of the row's largest at the least
      __syncthreads();
#pragma unroll
      for (int i0 = 0; i0 < kBlocks * kParts; i0 += kExpandWaves) {
        const int packet = (i0 + wv) * kEach + lane % kEach, block = packet / kWave, pl = packet % kWave;
        if (block >= kBlocks) break;
        if (lane / kEach != 0) continue;
        const int to = row_exponent(s_most[block % NT * 16 + (pl & 15)]);
        float f[V], rest[V];
#pragma unroll
        for (int i = 0; i < V; ++i) f[i] = __builtin_ldexpf(sums[i0 / kExpandWaves][i], to);
        const u32x4 hi = Pack<f16_t>::pack(f);
        Pack<f16_t>::unpack(hi, rest);
#pragma unroll
        for (int i = 0; i < V; ++i) rest[i] = f[i] - rest[i];
        s_low[0][block][pl] = hi;
        s_low[1][block][pl] = Pack<f16_t>::pack(rest);
      }
    }
    if constexpr (kStaged) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (c0 >= e.columns) return;
#pragma unroll
    for (int k = 0; k < KT; ++k) {
      u32x4 low_hi[NT], low_lo[NT];   // (fp32: low_hi alone)
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        low_hi[j] = s_low[0][k * NT + j][lane];
        if constexpr (sizeof(T) == 2) low_lo[j] = s_low[1][k * NT + j][lane];
      }
#pragma unroll
      for (int mi = 0; mi < 8; ++mi) {
        u32x4 v;
        if constexpr (kStaged) {   // (past the rank: zeros of `low` against its last packet)
          const int packet = (8 * lr + mi) * per + min(k * 4 + g, per - 1);
          v = load16(mine + ((packet ^ (lr & 7)) << 4));
        } else {
          v = m[k][mi];
        }
        if constexpr (sizeof(T) == 4) {
#pragma unroll
          for (int j = 0; j < NT; ++j) acc[j][mi] = mfma_packet<float>(low_hi[j], v, acc[j][mi]);
        } else {
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            acc[j][mi] = mfma_16x16x32<T>(low_lo[j], v, acc[j][mi]);
            acc[j][mi] = mfma_16x16x32<T>(low_hi[j], v, acc[j][mi]);
          }
        }
      }
    }
  }
  if (!here) return;
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int t = j * 16 + 4 * g + i;
      const int64_t row = first + t;
      if (t >= n) continue;
      const int back = kHalf && a >= 0 ? -row_exponent(s_most[t]) : 0;
#pragma unroll
      for (int h = 0; h < 8 / V; ++h) {
        float f[V] = {};
        if (e.base != nullptr) Pack<T>::unpack(base[j][i][h], f);
        if (a >= 0) {   // (else the base to the bit: -0 + 0 is +0)
#pragma unroll
          for (int q = 0; q < V; ++q) f[q] += kHalf ? __builtin_ldexpf(acc[j][h * V + q][i], back) : acc[j][h * V + q][i];
        }
        store16(static_cast<T*>(e.out) + row * e.columns + c + h * V, Pack<T>::pack(f));
      }
    }
}

// ---- a row each, both factors at once ---------------------------------------------------------------------------------------------
// The next token of a few chats: a workgroup has 512 columns of a row, a column a thread, and makes the row's `low` itself, as every other of the row
// does: banks this small come out of the XCD's cache sooner than another launch starts. The rank's rows go over the waves, two at a time, their
// packets over the lanes. All in fp32.
constexpr int kStepThreads = 512;
template <typename T>
__global__ __launch_bounds__(kStepThreads) void step_kernel(const T* __restrict__ x, const int64_t x_stride, const Bank bank, const T* __restrict__ lora_b,
                                                            const int32_t* __restrict__ adapter, const Expand e, const int groups) {
  constexpr int V = Pack<T>::N, kWaves = kStepThreads / kWave, kAhead = 4;
  __shared__ float s_low[128];
  const int item = tile_of_workgroup(blockIdx.x, gridDim.x), row = item / groups, group = item - row * groups;
  const int lane = threadIdx.x & (kWave - 1), wv = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / kWave);
  const int id = adapter[row], a = id >= 0 && id < bank.slots ? id : -1;
  const int c = group * kStepThreads + threadIdx.x, at = min(c, e.columns - 1);
  T* const out = static_cast<T*>(e.out) + static_cast<int64_t>(row) * e.columns + c;
  const T base = static_cast<const T*>(e.base)[row * e.base_stride + at];
  float* const low = e.low != nullptr && group == 0 && static_cast<int>(threadIdx.x) < bank.rank ? e.low + static_cast<int64_t>(row) * bank.rank + threadIdx.x : nullptr;
  if (a < 0) {
    if (c < e.columns) *out = base;
    if (low != nullptr) *low = 0.0f;
    return;
  }
  const T* const column = lora_b + (static_cast<int64_t>(a) * e.columns + at) * bank.rank;
  const int per = bank.rank / V, packets = bank.width / V;
  u32x4 b[kAhead];
#pragma unroll
  for (int i = 0; i < kAhead; ++i) b[i] = load16(column + min(i, per - 1) * V);
  const float scaling = e.scaling[a];
  const T* const from = x + row * x_stride;
  const T* const m = static_cast<const T*>(bank.m) + static_cast<int64_t>(a) * bank.rank * bank.width;
  for (int r = 2 * wv; r < bank.rank; r += 2 * kWaves) {   // (the rank is even)
    float sum[2] = {0.0f, 0.0f};
#pragma unroll 2
    for (int p0 = 0; p0 < packets; p0 += kAhead * kWave) {
      u32x4 v[kAhead], w[2][kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int p = min(p0 + i * kWave + lane, packets - 1) * V;
        v[i] = load16(from + p);
#pragma unroll
        for (int q = 0; q < 2; ++q) w[q][i] = load16(m + static_cast<int64_t>(r + q) * bank.width + p);
      }
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        float f[V], h[V];
        Pack<T>::unpack(v[i], f);
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          Pack<T>::unpack(w[q][i], h);
          float part = 0.0f;
#pragma unroll
          for (int k = 0; k < V; ++k) part = __builtin_fmaf(f[k], h[k], part);
          sum[q] += p0 + i * kWave + lane < packets ? part : 0.0f;
        }
      }
    }
#pragma unroll
    for (int q = 0; q < 2; ++q) {
#pragma unroll
      for (int d = 1; d < kWave; d *= 2) sum[q] += __shfl_xor(sum[q], d);
    }
    if (lane == 0) {
      s_low[r] = sum[0];
      s_low[r + 1] = sum[1];
    }
  }
  __syncthreads();
  if (low != nullptr) *low = s_low[threadIdx.x];
  float sum = 0.0f;
  for (int i0 = 0; i0 < per; i0 += kAhead) {
    if (i0 > 0) {
#pragma unroll
      for (int i = 0; i < kAhead; ++i) b[i] = load16(column + min(i0 + i, per - 1) * V);
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      if (i0 + i >= per) break;
      float f[V];
      Pack<T>::unpack(b[i], f);
#pragma unroll
      for (int k = 0; k < V; ++k) sum = __builtin_fmaf(s_low[(i0 + i) * V + k], f[k], sum);
    }
  }
  if (c < e.columns) *out = from_float<T>(__builtin_fmaf(scaling, sum, to_float(base)));
}

// ---- the plan of a gradient: rows sorted by adapter -----------------------------------------------------------------------------
constexpr int kBlock = 32;          // rows of a block: one step of the matrix core
constexpr int kPlanThreads = 1024;  // and the most slots

// start [slots + 1]: the first virtual row of each slot, a multiple of 32 (rows up to there: none, -1); order: the row behind each
// virtual row; used_start [used + 1]: the starts of the slots that have rows alone, and behind them the end; place [slots]: where a slot stands among
// those. Requests of a slot keep their order. One workgroup; seq_start: [sequences] scratch.
struct Plan {
  int slots, capacity;   // virtual rows at the most
  int used;              // slots that can have rows: there are no more of them than requests
  int32_t* start;
  int32_t* used_start;
  int32_t* place;
  int32_t* order;
  int32_t* seq_start;
};
struct PlanLds {
  int a[kPlanThreads], n[kPlanThreads], at[kPlanThreads], seq[kPlanThreads], scan[kPlanThreads], waves[kPlanThreads / kWave];
};
__device__ __forceinline__ void make_plan(PlanLds& s, const Requests& req, const Plan& p) {
  const int t = threadIdx.x, sequences = req.rows.sequences;
  const bool few = sequences <= kPlanThreads;   // all requests in LDS
  int mine = 0;
  for (int v = t * 4; v < p.capacity; v += kPlanThreads * 4) *reinterpret_cast<int4*>(p.order + v) = make_int4(-1, -1, -1, -1);
  for (int pass = 0; pass < 2; ++pass) {
    int at = pass == 0 ? 0 : s.scan[t] - mine;
    for (int b0 = 0; b0 < sequences; b0 += kPlanThreads) {
      if (!few || pass == 0) {
        __syncthreads();
        if (b0 + t < sequences) {
          s.a[t] = req.adapter[b0 + t];
          s.at[t] = req.rows.first(b0 + t);
          s.n[t] = max(req.rows.first(b0 + t + 1) - s.at[t], 0);
        }
        __syncthreads();
      }
      const int many = min(sequences - b0, kPlanThreads);
      if (t < p.slots) {
        for (int i = 0; i < many; ++i) {
          if (s.a[i] != t) continue;
          if (pass == 1) {
            if (few) s.seq[i] = at;
            else p.seq_start[b0 + i] = at;
          }
          at = min(at + s.n[i], p.capacity);   // (more than that only where query_start decreases)
        }
      }
    }
    if (pass == 1) break;
    mine = t < p.slots ? (at + kBlock - 1) / kBlock * kBlock : 0;
    __syncthreads();
    s.scan[t] = mine;
    __syncthreads();
    for (int d = 1; d < p.slots; d *= 2) {
      const int v = t >= d ? s.scan[t - d] : 0;
      __syncthreads();
      s.scan[t] += v;
      __syncthreads();
    }
    const int begin = min(s.scan[t] - mine, p.capacity), end = min(s.scan[p.slots - 1], p.capacity);
    const uint64_t have = __ballot(mine > 0);   // (0 past the slots)
    if (t % kWave == 0) s.waves[t / kWave] = __popcll(have);
    __syncthreads();
    int place = __popcll(have & ((uint64_t{1} << t % kWave) - 1)), all = 0;
    for (int w = 0; w < kPlanThreads / kWave; ++w) {
      if (w < t / kWave) place += s.waves[w];
      all += s.waves[w];
    }
    if (t < p.slots) {
      p.start[t] = begin;
      p.place[t] = place;
      if (mine > 0 && place < p.used) p.used_start[place] = begin;
    }
    for (int i = all + t; i <= p.used; i += kPlanThreads) p.used_start[i] = end;
    if (t == 0) p.start[p.slots] = end;
  }
  __syncthreads();
  for (int row = t; row < req.rows.rows; row += kPlanThreads) {
    int lo = 0, hi = sequences;   // the last request that begins at or in front of the row
    while (lo + 1 < hi) {
      const int mid = (lo + hi) / 2;
      if ((few ? s.at[mid] : req.rows.first(mid)) <= row) lo = mid; else hi = mid;
    }
    const int from = few ? s.at[lo] : req.rows.first(lo), n = few ? s.n[lo] : max(req.rows.first(lo + 1) - from, 0);
    const int a = few ? s.a[lo] : req.adapter[lo];
    if (row < from || row - from >= n || a < 0 || a >= p.slots) continue;
    const int v = (few ? s.seq[lo] : p.seq_start[lo]) + row - from;
    if (v < p.capacity) p.order[v] = row;
  }
}

// The first workgroup makes the plan, the others turn the banks over: lora_a [slots, rank, in] and lora_b [slots, out, rank], 64 x 64 each.
struct Turn {
  const void* from;
  void* to;
  int rows, cols;   // of a slot
};
template <typename E>
__global__ __launch_bounds__(kPlanThreads) void prepare_kernel(const Requests req, const Plan plan, const Turn a, const Turn b) {
  union Lds {
    PlanLds plan;
    E tile[64][68];
  };
  __shared__ __attribute__((aligned(16))) unsigned char s_mem[sizeof(Lds)];
  Lds& s = *reinterpret_cast<Lds*>(s_mem);
  if (blockIdx.x == 0) {
    make_plan(s.plan, req, plan);
    return;
  }
  struct alignas(4 * sizeof(E)) Four { E v[4]; };
  const int a_cols = (a.cols + 63) / 64, a_tiles = a_cols * ((a.rows + 63) / 64), b_cols = (b.cols + 63) / 64, b_tiles = b_cols * ((b.rows + 63) / 64);
  const int id = blockIdx.x - 1, of_a = a_tiles * plan.slots;
  const Turn& turn = id < of_a ? a : b;
  const int at = id < of_a ? id : id - of_a, tiles = id < of_a ? a_tiles : b_tiles, slot = at / tiles, tile = at - slot * tiles, cols = id < of_a ? a_cols : b_cols;
  const int r0 = tile / cols * 64, c0 = tile % cols * 64, y = threadIdx.x / 16, x = threadIdx.x % 16 * 4;
  const int64_t base = static_cast<int64_t>(slot) * turn.rows * turn.cols;
  if (r0 + y < turn.rows && c0 + x < turn.cols)   // (both are multiples of 8)
    *reinterpret_cast<Four*>(&s.tile[y][x]) = *reinterpret_cast<const Four*>(static_cast<const E*>(turn.from) + base + static_cast<int64_t>(r0 + y) * turn.cols + c0 + x);
  __syncthreads();
  if (c0 + y < turn.cols && r0 + x < turn.rows) {
    const Four f{{s.tile[x][y], s.tile[x + 1][y], s.tile[x + 2][y], s.tile[x + 3][y]}};
    *reinterpret_cast<Four*>(static_cast<E*>(turn.to) + base + static_cast<int64_t>(c0 + y) * turn.rows + r0 + x) = f;
  }
}

// ---- outer ------------------------------------------------------------------------------------------------------------------
struct OuterSide {
  const void* x;           // rows of `width` values of T, or int8 codes with x_scale
  int64_t stride;
  const float* x_scale;    // [rows, width / 128], or null
  const float* u;          // the other factor [rows, rank]: g lora_b, or x lora_a^T (the scaling comes at the end)
  float* records;          // [pieces][rank][width]
  int width;
};
struct Outer {
  OuterSide a, b;          // gradients of A (x and du) and of B (g and low)
  const int32_t* start;
  const int32_t* used_start;   // [used + 1] and place [slots]: as the plan has them
  const int32_t* place;
  const int32_t* order;
  const float* scaling;
  int slots, used, rank, capacity, shift;   // 1 << shift rows a piece
  int a_columns;           // workgroups of side a in blockIdx.x
  void *grad_a, *grad_b;   // or null: records. Where a slot's rows are one piece: the results, blockIdx.y is the slot
};
constexpr int kColumns = 128;   // of a wave: one group of the codes

// One side's sums over the rows of a piece for 128 columns and 16 RTW of the rank. A step's rows are asked for a step ahead, their
// numbers two.
template <typename T, bool CODES> struct OuterRows {   // eight columns of eight rows (fp32 values: four of eight, twice)
  static constexpr int kWords = CODES ? 2 : sizeof(T) == 4 ? 8 : 4;
  uint32_t w[8][kWords];
};
template <typename T, bool CODES, int RTW>
__device__ __forceinline__ void outer_rows(const OuterSide& side, const Outer& o, int c0, int v0, int v1, v4f (&acc)[RTW][8]) {
  const int lane = threadIdx.x & (kWave - 1), wv = threadIdx.x / kWave, lr = lane & 15, g = lane >> 4;
  const int tile0 = blockIdx.z * RTW, step = 4 * kBlock;
  const int begin = v0 + wv * kBlock;
  if (begin >= v1) return;
  const int spare = max(o.order[v0], 0);   // (the first row of a block: real)
  const auto rows_at = [&](int v, int (&row)[8]) {
    const int at = min(v, v1 - kBlock) + 8 * g;
    const int4 lo = *reinterpret_cast<const int4*>(o.order + at), hi = *reinterpret_cast<const int4*>(o.order + at + 4);
    const int got[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) row[i] = got[i];
  };
  const auto ask = [&](const int (&row)[8], OuterRows<T, CODES>& x, float (&f)[RTW][8], float (&s)[8], uint32_t& real) {
    real = 0;   // (applied where the values are used: nothing here waits for them)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      real |= row[i] >= 0 ? 1u << i : 0u;
      const int64_t at = row[i] >= 0 ? row[i] : spare;   // (no row: its other factor is zero; a row of this slot, so that nothing foreign gets in)
      if constexpr (CODES) {
        const u32x2 w = *reinterpret_cast<const u32x2*>(static_cast<const int8_t*>(side.x) + at * side.stride + min(c0 + 8 * lr, side.width - 8));
        x.w[i][0] = w.x;
        x.w[i][1] = w.y;
        s[i] = side.x_scale[at * (side.width / kColumns) + c0 / kColumns];
      } else if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const u32x4 w = load16(static_cast<const float*>(side.x) + at * side.stride + min(c0 + 64 * h + 4 * lr, side.width - 4));
          x.w[i][4 * h] = w.x; x.w[i][4 * h + 1] = w.y; x.w[i][4 * h + 2] = w.z; x.w[i][4 * h + 3] = w.w;
        }
      } else {
        const u32x4 w = load16(static_cast<const T*>(side.x) + at * side.stride + min(c0 + 8 * lr, side.width - 8));
        x.w[i][0] = w.x; x.w[i][1] = w.y; x.w[i][2] = w.z; x.w[i][3] = w.w;
      }
      // (entries RTW lr .. of the rank: one of each tile)
      const float* from = side.u + at * o.rank + min((tile0 * 16) + RTW * lr, o.rank - RTW);
      float value[RTW];
      if constexpr (RTW == 4) {
        const v4f v = *reinterpret_cast<const v4f*>(from);
        value[0] = v[0]; value[1] = v[1]; value[2] = v[2]; value[3] = v[3];
      } else if constexpr (RTW == 2) {
        const float2 v = *reinterpret_cast<const float2*>(from);
        value[0] = v.x; value[1] = v.y;
      } else {
        value[0] = *from;
      }
#pragma unroll
      for (int r = 0; r < RTW; ++r) f[r][i] = value[r];
    }
  };
  int row[8];
  OuterRows<T, CODES> x;
  float f[RTW][8], s[8];
  uint32_t real;
  rows_at(begin, row);
  ask(row, x, f, s, real);
  rows_at(begin + step, row);
  for (int v = begin; v < v1; v += step) {
    OuterRows<T, CODES> now = x;
    float u[RTW][8];
#pragma unroll
    for (int i = 0; i < RTW; ++i)
#pragma unroll
      for (int q = 0; q < 8; ++q) u[i][q] = real >> q & 1 ? (CODES ? f[i][q] * s[q] : f[i][q]) : 0.0f;
    ask(row, x, f, s, real);   // (behind the last step: that one again)
    rows_at(v + 2 * step, row);
    if constexpr (sizeof(T) == 4) {   // e-th product: row 8 g + e of each lane
#pragma unroll
      for (int e = 0; e < 8; ++e)
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          float value;
          if constexpr (CODES) value = static_cast<float>(static_cast<int8_t>(now.w[e][q / 4] >> (8 * (q % 4))));
          else value = __builtin_bit_cast(float, now.w[e][q]);
#pragma unroll
          for (int i = 0; i < RTW; ++i) acc[i][q] = mfma_f32(u[i][e], value, acc[i][q]);
        }
    } else {
      HiLo other[RTW];
#pragma unroll
      for (int i = 0; i < RTW; ++i) other[i] = hi_lo(u[i]);
#pragma unroll
      for (int q = 0; q < 8; ++q) {   // column q of the lane's eight
        HiLo w;
        if constexpr (CODES || __is_same(T, f16_t)) {
          float column[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            if constexpr (CODES) column[e] = static_cast<float>(static_cast<int8_t>(now.w[e][q / 4] >> (8 * (q % 4))));
            else column[e] = static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(now.w[e][q / 2] >> (16 * (q % 2)))));
          }
          w = hi_lo(column);   // (codes: the first alone; fp16: exact)
        } else {
          const uint32_t select = q % 2 ? 0x07060302u : 0x05040100u;   // the halves of two rows' words
          w.hi.x = __builtin_amdgcn_perm(now.w[1][q / 2], now.w[0][q / 2], select);
          w.hi.y = __builtin_amdgcn_perm(now.w[3][q / 2], now.w[2][q / 2], select);
          w.hi.z = __builtin_amdgcn_perm(now.w[5][q / 2], now.w[4][q / 2], select);
          w.hi.w = __builtin_amdgcn_perm(now.w[7][q / 2], now.w[6][q / 2], select);
        }
#pragma unroll
        for (int i = 0; i < RTW; ++i) {
          if constexpr (!CODES && __is_same(T, f16_t)) acc[i][q] = mfma_16x16x32<bf16_t>(other[i].hi, w.lo, acc[i][q]);
          acc[i][q] = mfma_16x16x32<bf16_t>(other[i].lo, w.hi, acc[i][q]);
          acc[i][q] = mfma_16x16x32<bf16_t>(other[i].hi, w.hi, acc[i][q]);
        }
      }
    }
  }
}

template <typename T, bool CODES, int RTW>
__global__ __launch_bounds__(4 * kWave) void outer_kernel(const Outer o) {
  __shared__ v4f s_sum[2][RTW * 8][kWave];
  int v0, v1;
  if (o.grad_a != nullptr) {   // a slot's rows at once
    v0 = o.start[blockIdx.y];
    v1 = o.start[blockIdx.y + 1];
  } else {
    const Ragged slots{o.used_start, o.used, o.capacity};
    int piece = blockIdx.y, none;
    Span span;
    slots.find(o.shift, nullptr, piece, span, none);
    v0 = span.first + (piece << o.shift);
    v1 = min(v0 + (1 << o.shift), span.first + span.n);
    if (span.n <= 0 || v0 >= v1) return;
  }
  const bool side_b = static_cast<int>(blockIdx.x) >= o.a_columns;
  const int c0 = (blockIdx.x - (side_b ? o.a_columns : 0)) * kColumns;
  v4f acc[RTW][8] = {};
  if (v0 >= v1) {}   // (a slot without rows: zeros)
  else if (side_b) outer_rows<T, false, RTW>(o.b, o, c0, v0, v1, acc);
  else outer_rows<T, CODES, RTW>(o.a, o, c0, v0, v1, acc);
  const int lane = threadIdx.x & (kWave - 1), wv = threadIdx.x / kWave, lr = lane & 15, g = lane >> 4;
  if (wv >= 2) {
#pragma unroll
    for (int i = 0; i < RTW * 8; ++i) s_sum[wv - 2][i][lane] = acc[i / 8][i % 8];
  }
  __syncthreads();
  if (wv < 2) {
#pragma unroll
    for (int i = 0; i < RTW * 8; ++i) acc[i / 8][i % 8] += s_sum[wv][i][lane];
  }
  __syncthreads();
  if (wv == 1) {
#pragma unroll
    for (int i = 0; i < RTW * 8; ++i) s_sum[0][i][lane] = acc[i / 8][i % 8];
  }
  __syncthreads();
  if (wv != 0) return;
  const OuterSide& side = side_b ? o.b : o.a;
  if (o.grad_a != nullptr) {
    const float scale = o.scaling[blockIdx.y];
    const bool halved = sizeof(T) == 4 && !(CODES && !side_b), none = v0 >= v1;
    const auto value = [&](int i, int q, int c) { return none ? 0.0f : (acc[i][c][q] + s_sum[0][i * 8 + c][lane][q]) * scale; };
    const int64_t slot = static_cast<int64_t>(blockIdx.y) * o.rank * side.width;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int c = c0 + (halved ? 64 * h + 4 * lr : 8 * lr + 4 * h);
      if (c >= side.width) continue;   // (a multiple of 8)
      if (!side_b) {
#pragma unroll
        for (int i = 0; i < RTW; ++i)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const int r = blockIdx.z * RTW * 16 + RTW * (4 * g + q) + i;
            const float f[4] = {value(i, q, 4 * h), value(i, q, 4 * h + 1), value(i, q, 4 * h + 2), value(i, q, 4 * h + 3)};
            if (r < o.rank) store_four(static_cast<T*>(o.grad_a) + slot + static_cast<int64_t>(r) * side.width + c, f);
          }
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int k = 0; k < 4 * RTW; k += 4) {   // four of the rank
            const int r = blockIdx.z * RTW * 16 + RTW * 4 * g + k;
            const float f[4] = {value(k % RTW, k / RTW, 4 * h + e), value((k + 1) % RTW, (k + 1) / RTW, 4 * h + e), value((k + 2) % RTW, (k + 2) / RTW, 4 * h + e),
                                value((k + 3) % RTW, (k + 3) / RTW, 4 * h + e)};
            if (r < o.rank) store_four(static_cast<T*>(o.grad_b) + slot + static_cast<int64_t>(c + e) * o.rank + r, f);
          }
      }
    }
    return;
  }
  float* record = side.records + static_cast<int64_t>(blockIdx.y) * o.rank * side.width;
  // (lane: entries RTW (4 g + q) + i of the rank's 16 RTW, and of the columns 8 lr .. 8 lr + 7, or of fp32 values 64 h + 4 lr .., h = 0, 1)
  const bool halves = sizeof(T) == 4 && !(CODES && !side_b);
#pragma unroll
  for (int i = 0; i < RTW; ++i)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int r = blockIdx.z * RTW * 16 + RTW * (4 * g + q) + i;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        v4f v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = acc[i][h * 4 + e][q] + s_sum[0][i * 8 + h * 4 + e][lane][q];
        const int c = c0 + (halves ? 64 * h + 4 * lr : 8 * lr + 4 * h);
        if (r < o.rank && c < side.width) *reinterpret_cast<v4f*>(record + static_cast<int64_t>(r) * side.width + c) = v;
      }
    }
}

// The pieces' records of each slot added up in order, scaled, rounded: eight of the width a lane for A [slots, rank, width], eight of the rank
// for B [slots, width, rank]. A slot without rows has a gradient of zero.
template <typename T>
__global__ __launch_bounds__(256) void records_kernel(const Outer o, T* __restrict__ grad_a, T* __restrict__ grad_b, const int64_t a_items, const int64_t items) {
  constexpr int kAhead = 4;
  for (int64_t item = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; item < items; item += static_cast<int64_t>(gridDim.x) * 256) {
    const bool of_b = item >= a_items;
    const OuterSide& side = of_b ? o.b : o.a;
    const int64_t at = of_b ? item - a_items : item, each = static_cast<int64_t>(o.rank) * side.width, per_slot = each / 8;
    const int slot = static_cast<int>(at / per_slot), rest = static_cast<int>(at - slot * per_slot);
    int r, c;
    if (of_b) {
      r = rest / side.width * 8;
      c = rest % side.width;
    } else {
      r = rest / (side.width / 8);
      c = rest % (side.width / 8) * 8;
    }
    const int n = o.start[slot + 1] - o.start[slot], first = (o.start[slot] >> o.shift) + 2 * o.place[slot], pieces = (n + (1 << o.shift) - 1) >> o.shift;
    float f[8] = {};
    const float scale = o.scaling[slot];
    const int64_t next = of_b ? side.width : 1;
    for (int p0 = 0; p0 < pieces; p0 += kAhead) {
      float v[kAhead][8];
#pragma unroll
      for (int p = 0; p < kAhead; ++p) {
        const float* from = side.records + (first + min(p0 + p, pieces - 1)) * each + static_cast<int64_t>(r) * side.width + c;
#pragma unroll
        for (int i = 0; i < 8; ++i) v[p][i] = from[i * next];
      }
#pragma unroll
      for (int p = 0; p < kAhead; ++p)
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (p0 + p < pieces) f[i] += v[p][i];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = pieces > 0 ? f[i] * scale : 0.0f;
    T* to = of_b ? grad_b + slot * each + static_cast<int64_t>(c) * o.rank + r : grad_a + slot * each + static_cast<int64_t>(r) * side.width + c;
#pragma unroll
    for (int i = 0; i < 8; i += Pack<T>::N) store16(to + i, Pack<T>::pack(f + i));
  }
}

// ---- what a call takes ------------------------------------------------------------------------------------------------------
// Row tiles of a piece. expand: one for single rows and short requests, two where requests are longer (a bank's rows are read once a piece).
int row_tiles(int rows, int sequences, bool ragged) { return !ragged || rows < 24 * sequences ? 1 : 2; }
// shrink: one (many workgroups), two where the bank's rows weigh more than twice the activation's
int shrink_tiles(int rows, int sequences, bool ragged, int rank) { return rank > 32 && row_tiles(rows, sequences, ragged) > 1 ? 2 : 1; }
int pieces_of(int rows, int sequences, bool ragged, int nt) { return ragged ? rows / (16 * nt) + 2 * sequences : sequences; }
// Parts of the reduction: for 768 workgroups, of a step a wave at least; up to eight for single rows and few pieces of rows, four for more, two for many
// (14336 by 64, 2 to 340 rows: 13.2 to 21.9 us with four, 11.0 to 18.3 with eight, 10.4 to 19.4 with sixteen; 4096 by 128 13.4 to 19.5, 12.7 to 20.0, 13.0 to 24.6)
// (4099 rows of 4096 by 64, one part: shrink 17.0 us, expand 24.4; two: 14.6 and 25.0; four: 13.8 and 26.5).
int splits_of(int rows, int sequences, bool ragged, int width, int rank, int dtype) {
  const int nt = shrink_tiles(rows, sequences, ragged, rank);
  const int64_t real = ragged ? (rows + 16 * nt - 1) / (16 * nt) : sequences;
  const int steps = (width * (dtype == LLMQ_F32 ? 4 : 2) + 127) / 128, most = !ragged ? 8 : real < 24 ? 8 : real < 96 ? 4 : 2;
  int64_t splits = 768 / (real < 1 ? 1 : real);
  if (splits > steps / shrink_waves(rank)) splits = steps / shrink_waves(rank);
  if (splits > most) splits = most;
  return static_cast<int>(splits < 1 ? 1 : splits);
}

template <typename T, int RT>
void shrink_nt(const T* x, int64_t stride, const Bank& bank, const Requests& req, float* planes, int64_t plane, const dim3& grid, int nt, hipStream_t s) {
  if (nt == 1) hipLaunchKernelGGL((shrink_kernel<T, RT, 1>), grid, dim3(kShrinkWaves<RT> * kWave), 0, s, x, stride, bank, req, planes, plane);
  else if constexpr (RT >= 4) hipLaunchKernelGGL((shrink_kernel<T, RT, 2>), grid, dim3(kShrinkWaves<RT> * kWave), 0, s, x, stride, bank, req, planes, plane);
}
template <typename T>
void shrink(const void* x, int64_t stride, const Bank& bank, const Requests& req, float* planes, int64_t plane, int splits, bool ragged, hipStream_t s) {
  const T* p = static_cast<const T*>(x);
  const int nt = shrink_tiles(req.rows.rows, req.rows.sequences, ragged, bank.rank);
  const dim3 grid(pieces_of(req.rows.rows, req.rows.sequences, ragged, nt), splits);
  if (bank.rank <= 16) shrink_nt<T, 1>(p, stride, bank, req, planes, plane, grid, nt, s);
  else if (bank.rank <= 32) shrink_nt<T, 2>(p, stride, bank, req, planes, plane, grid, nt, s);
  else if (bank.rank <= 64) shrink_nt<T, 4>(p, stride, bank, req, planes, plane, grid, nt, s);
  else shrink_nt<T, 8>(p, stride, bank, req, planes, plane, grid, nt, s);
}
template <typename T, int RT> void expand_nt(const Bank& bank, const Requests& req, const Expand& e, int nt, const dim3& grid, hipStream_t s) {
  const dim3 block(kExpandWaves * kWave);
  if (nt == 1) hipLaunchKernelGGL((expand_kernel<T, RT, 1>), grid, block, 0, s, bank, req, e);
  else hipLaunchKernelGGL((expand_kernel<T, RT, 2>), grid, block, 0, s, bank, req, e);
}
// bank: [slots][columns][rank]
template <typename T> void expand(const Bank& bank, const Requests& req, Expand e, hipStream_t s) {
  const bool ragged = req.rows.start != nullptr;
  const int nt = row_tiles(e.rows, req.rows.sequences, ragged);
  e.pieces = pieces_of(e.rows, req.rows.sequences, ragged, nt);
  e.rest = !ragged || (e.out == e.base && e.low == nullptr) ? 0 : e.pieces < 32 ? e.pieces : 32;   // (usually without a row: the requests have them all)
  const dim3 grid(e.pieces, (e.columns + kExpandWaves * 128 - 1) / (kExpandWaves * 128) + (e.rest > 0 ? 1 : 0));
  if (bank.rank <= 16) expand_nt<T, 1>(bank, req, e, nt, grid, s);
  else if (bank.rank <= 32) expand_nt<T, 2>(bank, req, e, nt, grid, s);
  else if (bank.rank <= 64) expand_nt<T, 4>(bank, req, e, nt, grid, s);
  else expand_nt<T, 8>(bank, req, e, nt, grid, s);
}

// Single rows in one launch (step_kernel): workgroups of a row, or 0. For banks of up to 128 KB and up to two workgroups a CU (bf16, calls among others, us,
// one launch for two: rank 16, 2048 x 2048: 1 row 5.0 for 7.5, 128 rows 5.8 for 8.8; 4096 x 4096: 64 rows 7.3 for 8.7, 128 rows 11.6 for 11.1; rank 64, 4096 x 4096: 1 row
// 11.0 for 8.8).
int step_groups(int rows, int slots, bool ragged, int in, int out, int rank, int dtype) {
  const int groups = (out + kStepThreads - 1) / kStepThreads;
  const int64_t bank = static_cast<int64_t>(rank) * in * (dtype == LLMQ_F32 ? 4 : 2);
  return !ragged && slots > 0 && bank <= (128 << 10) && static_cast<int64_t>(rows) * groups <= 512 ? groups : 0;
}

int64_t round_up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }
int64_t take(int64_t& at, int64_t bytes) {
  const int64_t here = at;
  at = round_up(at + bytes, 256);
  return here;
}

struct GradPlan {
  bool direct;   // no records: a workgroup has all of a slot's rows
  int splits, capacity, used, tiles, rtw, shift, records;   // parts of shrink, virtual rows, slots that can have rows, tiles of the rank, pieces of outer
  int64_t o_start, o_used, o_place, o_order, o_seq, o_at, o_bt, o_planes, o_du, o_rec_a, o_rec_b, bytes;
};
GradPlan grad_plan(int rows, int sequences, bool ragged, int in, int out, int rank, int slots, int dtype) {
  GradPlan p{};
  const int64_t size = dtype == LLMQ_F32 ? 4 : 2;
  p.splits = splits_of(rows, sequences, ragged, out, rank, dtype);
  const int64_t used = slots < sequences ? slots : sequences;   // slots that can have rows
  p.used = static_cast<int>(used);
  p.capacity = static_cast<int>(round_up(rows + 31 * used, kBlock));
  p.tiles = (rank + 15) / 16;
  // outer takes one, two or four tiles of the rank a workgroup: fewer read the rows more often, and are smaller programs of fewer registers (bf16, whole calls, us,
  // by four / two / one: 4096 x 14336 by 64, 32 rows 47 / 35 / 32, 1024 rows 62 / 53 / 52, 2048 77 / 70 / 79, 4096 113 / 118 / 151).
  p.rtw = p.tiles >= 4 && rows > 2048 ? 4 : p.tiles >= 2 && rows > 1024 ? 2 : 1;
  // All of a slot's rows in a workgroup, which leaves the records and their launch out, while slots have up to 1536 on average, or 1024 of ranks above 32 (rank 16,
  // 4096 x 4096, four slots: 64 rows 24.7 -> 18.7 us, 4096 rows 49.9 -> 45.4; 2048 x 2048, one slot: 1024 rows 29.2 -> 26.9; rank 32, 1500 rows 38.2 -> 36.1,
  // 2048 37.2 -> 42.5).
  p.direct = rows <= (p.tiles <= 2 ? 1536 : 1024) * used;
  // Otherwise a piece of 128 to 4096 rows, as long as it takes for the workgroups to be on the chip at once or nearly (with 64 entries of the rank
  // one a CU, for their registers: 4099 rows by 8192 columns, pieces of 512 rows 33 us and 11.6 to add them up, 1024 28.4 + 7.4, 2048 34.8 + 7.3)
  const int64_t columns = (in + kColumns - 1) / kColumns + (out + kColumns - 1) / kColumns, places = p.rtw == 4 ? 400 : p.rtw == 2 ? 512 : 1024;
  p.shift = 7;
  while (p.shift < 12 && columns * ((rows >> p.shift) + used) * ((p.tiles + p.rtw - 1) / p.rtw) > places) ++p.shift;
  p.records = p.direct ? 0 : (p.capacity >> p.shift) + 2 * p.used;
  int64_t at = 0;
  p.o_start = take(at, int64_t{4} * (slots + 1));
  p.o_used = take(at, int64_t{4} * (used + 1));
  p.o_place = take(at, int64_t{4} * slots);
  p.o_order = take(at, int64_t{4} * p.capacity);
  p.o_seq = take(at, int64_t{4} * sequences);
  p.o_at = take(at, size * slots * rank * in);
  p.o_bt = take(at, size * slots * rank * out);
  p.o_planes = take(at, int64_t{4} * p.splits * rows * rank);
  p.o_du = p.splits > 1 ? take(at, int64_t{4} * rows * rank) : p.o_planes;
  p.o_rec_a = take(at, int64_t{4} * p.records * rank * in);
  p.o_rec_b = take(at, int64_t{4} * p.records * rank * out);
  p.bytes = at;
  return p;
}

template <typename T>
void gradients(const GradPlan& p, const void* grad, int64_t grad_stride, const void* x, int64_t x_stride, const float* x_scale, const float* low,
               const void* lora_a, const void* lora_b, const float* scaling, const Requests& req, const void* grad_base, int64_t base_stride,
               void* grad_x, void* grad_a, void* grad_b, uint8_t* ws, int in, int out, int rank, int slots, hipStream_t s) {
  const int rows = req.rows.rows;
  float* planes = reinterpret_cast<float*>(ws + p.o_planes);
  float* du = reinterpret_cast<float*>(ws + p.o_du);   // g lora_b
  const int64_t plane = static_cast<int64_t>(rows) * rank;
  const Plan plan{slots, p.capacity, p.used, reinterpret_cast<int32_t*>(ws + p.o_start), reinterpret_cast<int32_t*>(ws + p.o_used),
                  reinterpret_cast<int32_t*>(ws + p.o_place), reinterpret_cast<int32_t*>(ws + p.o_order), reinterpret_cast<int32_t*>(ws + p.o_seq)};
  const Turn turn_a{lora_a, ws + p.o_at, rank, in}, turn_b{lora_b, ws + p.o_bt, out, rank};
  const unsigned tiles = static_cast<unsigned>(slots) * (((in + 63) / 64 + (out + 63) / 64) * ((rank + 63) / 64));
  if constexpr (sizeof(T) == 4) hipLaunchKernelGGL((prepare_kernel<uint32_t>), dim3(1 + tiles), dim3(kPlanThreads), 0, s, req, plan, turn_a, turn_b);
  else hipLaunchKernelGGL((prepare_kernel<uint16_t>), dim3(1 + tiles), dim3(kPlanThreads), 0, s, req, plan, turn_a, turn_b);
  shrink<T>(grad, grad_stride, Bank{ws + p.o_bt, slots, rank, out}, req, planes, plane, p.splits, req.rows.start != nullptr, s);
  expand<T>(Bank{ws + p.o_at, slots, rank, in}, req, Expand{planes, plane, p.splits, scaling, grad_base, base_stride, grad_x, p.splits > 1 ? du : nullptr, rows, in, 0, 0}, s);
  const Outer o{OuterSide{x, x_stride, x_scale, du, reinterpret_cast<float*>(ws + p.o_rec_a), in},
                OuterSide{grad, grad_stride, nullptr, low, reinterpret_cast<float*>(ws + p.o_rec_b), out},
                plan.start, plan.used_start, plan.place, plan.order, scaling, slots, p.used, rank, p.capacity, p.shift, (in + kColumns - 1) / kColumns, p.direct ? grad_a : nullptr,
                p.direct ? grad_b : nullptr};
  const dim3 grid(o.a_columns + (out + kColumns - 1) / kColumns, p.direct ? slots : p.records, (p.tiles + p.rtw - 1) / p.rtw);
#define LLMQ_OUTER(CODES)                                                                                    \
  if (p.rtw == 4) hipLaunchKernelGGL((outer_kernel<T, CODES, 4>), grid, dim3(4 * kWave), 0, s, o);            \
  else if (p.rtw == 2) hipLaunchKernelGGL((outer_kernel<T, CODES, 2>), grid, dim3(4 * kWave), 0, s, o);       \
  else hipLaunchKernelGGL((outer_kernel<T, CODES, 1>), grid, dim3(4 * kWave), 0, s, o)
  if (x_scale != nullptr) { LLMQ_OUTER(true); } else { LLMQ_OUTER(false); }
#undef LLMQ_OUTER
  if (p.direct) return;
  const int64_t a_items = static_cast<int64_t>(slots) * rank * in / 8, items = a_items + static_cast<int64_t>(slots) * rank * out / 8;
  const int64_t groups = (items + 255) / 256;
  hipLaunchKernelGGL((records_kernel<T>), dim3(static_cast<unsigned>(groups < 4096 ? groups : 4096)), dim3(256), 0, s, o, static_cast<T*>(grad_a),
                     static_cast<T*>(grad_b), a_items, items);
}

int check(int rows, int sequences, bool ragged, int in, int out, int rank, int slots, int dtype) {
  if (rows < 0 || sequences < 0 || slots < 0) return llmq_host::fail_invalid("bad dimension rows=%d sequences=%d slots=%d", rows, sequences, slots);
  if (dtype != LLMQ_F32 && dtype != LLMQ_F16 && dtype != LLMQ_BF16)
    return llmq_host::fail_invalid("dtype code %d is not float32, float16 or bfloat16", dtype);
  if (rank < 8 || rank > 128 || rank % 8) return llmq_host::fail_invalid("rank must be a multiple of 8 from 8 to 128, got %d", rank);
  if (in < 8 || out < 8 || in % 8 || out % 8 || in > (1 << 20) || out > (1 << 20))
    return llmq_host::fail_invalid("in_features and out_features must be multiples of 8 up to 2^20, got %d and %d", in, out);
  if (rows > (1 << 20) || sequences > (1 << 20) || slots > (1 << 20))
    return llmq_host::fail_invalid("at most 2^20 rows, sequences and slots, got %d, %d, %d", rows, sequences, slots);
  if ((rows / 16 + int64_t{2} * sequences) * ((in > out ? in : out) / 512 + 1) > (1 << 30))
    return llmq_host::fail_invalid("too many pieces: %d rows of %d sequences by %d x %d", rows, sequences, in, out);
  if (!ragged && rows != sequences) return llmq_host::fail_invalid("without query_start a sequence has one row: %d rows, %d sequences", rows, sequences);
  return 0;
}
bool misaligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) != 0; }
int bad_stride(int64_t stride, int width, int packet, const char* what) {
  if (stride >= width && stride % packet == 0) return 0;
  return llmq_host::fail_invalid("%s's row stride must be a multiple of %d of at least %d, got %lld", what, packet, width, static_cast<long long>(stride));
}
// (a piece's rows are offsets of 32 bits from its first)
int wide_stride(int64_t stride, int width, int rows, int sequences, bool ragged, int rank, int dtype, const char* what) {
  const int size = dtype == LLMQ_F32 ? 4 : 2, piece = ragged ? 16 * shrink_tiles(rows, sequences, ragged, rank) : 1;
  if (tile_spans(rows, piece, stride * size, int64_t{width} * size)) return 0;
  return llmq_host::fail_invalid("%s's row stride is too wide: %d neighbouring rows must lie within 4 GiB, got a stride of %lld elements", what, piece,
                                 static_cast<long long>(stride));
}

}  // namespace

extern "C" size_t llmq_lora_add_workspace_bytes(int rows, int sequences, int ragged, int in_features, int rank, int dtype) {
  if (rows <= 0 || sequences <= 0 || in_features <= 0 || rank <= 0) return 0;
  return static_cast<size_t>(int64_t{4} * splits_of(rows, sequences, ragged != 0, in_features, rank, dtype) * rows * rank);
}

extern "C" int llmq_lora_add(const void* x, int64_t x_stride, const void* base, int64_t base_stride, const void* lora_a, const void* lora_b,
                             const float* scaling, const int32_t* adapter, const int32_t* query_start_or_null, void* out, float* low_or_null,
                             void* workspace, size_t workspace_bytes, int rows, int sequences, int in_features, int out_features, int rank,
                             int slots, int dtype, llmq_stream_t stream) {
  const bool ragged = query_start_or_null != nullptr;
  if (int rc = check(rows, sequences, ragged, in_features, out_features, rank, slots, dtype)) return rc;
  if (rows == 0 || sequences == 0) return 0;   // (no sequence has a row: nothing is written)
  if (!x || !base || !out || !adapter || (slots > 0 && (!lora_a || !lora_b || !scaling))) return llmq_host::fail_invalid("null tensor pointer");
  const int v = dtype == LLMQ_F32 ? 4 : 8;
  if (int rc = bad_stride(x_stride, in_features, v, "x")) return rc;
  if (int rc = bad_stride(base_stride, out_features, v, "base")) return rc;
  if (int rc = wide_stride(x_stride, in_features, rows, sequences, ragged, rank, dtype, "x")) return rc;
  if (out == base && base_stride != out_features) return llmq_host::fail_invalid("out in place of base needs contiguous rows");
  if (misaligned(x) || misaligned(base) || misaligned(out) || misaligned(lora_a) || misaligned(lora_b) || misaligned(low_or_null))
    return llmq_host::fail_invalid("all tensors must be 16-byte aligned");
  const size_t need = llmq_lora_add_workspace_bytes(rows, sequences, ragged, in_features, rank, dtype);
  if (!workspace || misaligned(workspace) || workspace_bytes < need)
    return llmq_host::fail_invalid("the workspace must be 16-byte aligned and hold %zu bytes, got %zu", need, workspace_bytes);
  const Requests req{adapter, Ragged{query_start_or_null, sequences, rows}};
  const int splits = splits_of(rows, sequences, ragged, in_features, rank, dtype);
  float* planes = splits == 1 && low_or_null ? low_or_null : static_cast<float*>(workspace);   // (one plane is the sum)
  const int64_t plane = static_cast<int64_t>(rows) * rank;
  const Expand e{planes, plane, splits, scaling, base, base_stride, out, low_or_null, rows, out_features, 0, 0};
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (int groups = step_groups(rows, slots, ragged, in_features, out_features, rank, dtype)) {
    const Expand step{nullptr, 0, 0, scaling, base, base_stride, out, low_or_null, rows, out_features, 0, 0};
    const Bank bank{lora_a, slots, rank, in_features};
#define LLMQ_STEP(T)                                                                                                                \
  hipLaunchKernelGGL((step_kernel<T>), dim3(rows * groups), dim3(kStepThreads), 0, s, static_cast<const T*>(x), x_stride, bank,     \
                     static_cast<const T*>(lora_b), adapter, step, groups)
    if (dtype == LLMQ_F32) LLMQ_STEP(float);
    else if (dtype == LLMQ_F16) LLMQ_STEP(f16_t);
    else LLMQ_STEP(bf16_t);
#undef LLMQ_STEP
    return llmq_host::check_launch("lora_add");
  }
#define LLMQ_ADD(T)                                                                                                        \
  shrink<T>(x, x_stride, Bank{lora_a, slots, rank, in_features}, req, planes, plane, splits, ragged, s);                   \
  expand<T>(Bank{lora_b, slots, rank, out_features}, req, e, s)
  switch (dtype) {
    case LLMQ_F32: LLMQ_ADD(float); break;
    case LLMQ_F16: LLMQ_ADD(f16_t); break;
    default: LLMQ_ADD(bf16_t); break;
  }
#undef LLMQ_ADD
  return llmq_host::check_launch("lora_add");
}

extern "C" size_t llmq_lora_grad_workspace_bytes(int rows, int sequences, int ragged, int in_features, int out_features, int rank, int slots, int dtype) {
  if (rows <= 0 || sequences <= 0 || in_features <= 0 || out_features <= 0 || rank <= 0 || slots <= 0) return 0;
  return static_cast<size_t>(grad_plan(rows, sequences, ragged != 0, in_features, out_features, rank, slots, dtype).bytes);
}

extern "C" int llmq_lora_grad(const void* grad, int64_t grad_stride, const void* x, int64_t x_stride, const float* x_scale_or_null,
                              const float* low, const void* lora_a, const void* lora_b, const float* scaling, const int32_t* adapter,
                              const int32_t* query_start_or_null, const void* grad_base_or_null, int64_t base_stride, void* grad_x, void* grad_a,
                              void* grad_b, void* workspace, size_t workspace_bytes, int rows, int sequences, int in_features,
                              int out_features, int rank, int slots, int dtype, llmq_stream_t stream) {
  const bool ragged = query_start_or_null != nullptr;
  if (int rc = check(rows, sequences, ragged, in_features, out_features, rank, slots, dtype)) return rc;
  if (slots > kPlanThreads) return llmq_host::fail_invalid("at most %d slots have gradients, got %d", kPlanThreads, slots);
  if (x_scale_or_null && in_features % kColumns) return llmq_host::fail_invalid("codes of x come in groups of 128, in_features is %d", in_features);
  if (rows == 0 || sequences == 0 || slots == 0) return 0;   // (nothing is written)
  if (!grad || !x || !low || !lora_a || !lora_b || !scaling || !adapter || !grad_x || !grad_a || !grad_b) return llmq_host::fail_invalid("null tensor pointer");
  const int v = dtype == LLMQ_F32 ? 4 : 8;
  if (int rc = bad_stride(grad_stride, out_features, v, "grad")) return rc;
  if (int rc = wide_stride(grad_stride, out_features, rows, sequences, ragged, rank, dtype, "grad")) return rc;
  if (int rc = bad_stride(x_stride, in_features, x_scale_or_null ? 16 : v, "x")) return rc;
  if (grad_base_or_null)
    if (int rc = bad_stride(base_stride, in_features, v, "grad_base")) return rc;
  for (const void* t : {grad, x, static_cast<const void*>(low), lora_a, lora_b, grad_base_or_null, static_cast<const void*>(grad_x),
                        static_cast<const void*>(grad_a), static_cast<const void*>(grad_b)})
    if (misaligned(t)) return llmq_host::fail_invalid("all tensors must be 16-byte aligned");
  const GradPlan p = grad_plan(rows, sequences, ragged, in_features, out_features, rank, slots, dtype);
  if (!workspace || misaligned(workspace) || workspace_bytes < static_cast<size_t>(p.bytes))
    return llmq_host::fail_invalid("the workspace must be 16-byte aligned and hold %lld bytes, got %zu", static_cast<long long>(p.bytes), workspace_bytes);
  const Requests req{adapter, Ragged{query_start_or_null, sequences, rows}};
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  hipStream_t s = static_cast<hipStream_t>(stream);
#define LLMQ_GRAD(T)                                                                                                                 \
  gradients<T>(p, grad, grad_stride, x, x_stride, x_scale_or_null, low, lora_a, lora_b, scaling, req, grad_base_or_null, base_stride, \
               grad_x, grad_a, grad_b, ws, in_features, out_features, rank, slots, s)
  switch (dtype) {
    case LLMQ_F32: LLMQ_GRAD(float); break;
    case LLMQ_F16: LLMQ_GRAD(f16_t); break;
    default: LLMQ_GRAD(bf16_t); break;
  }
#undef LLMQ_GRAD
  return llmq_host::check_launch("lora_grad");
}
