// Softmax cross entropy over a vocabulary and its gradient without the logits, gfx950 (no counterpart among the reference's
// kernels):
//
//   l[t, v] = h[t] . W[v]      lse[t] = log sum_v exp l[t, v]      loss[t] = lse[t] - l[t, target[t]]
//   P[t, v] = (exp(l[t, v] - lse[t]) - [v = target[t]]) g[t]       dh[t] = sum_v P[t, v] W[v]       dW[v] = sum_t P[t, v] h[t]
//
// Logits exist as a tile in registers: 256 tokens of the vocabulary by 256 (or 64) rows on the matrix core (dense_tile.h),
// summed in fp32, of which the largest and the sum of exponentials per row, and the target's own, go to memory: 8 bytes for 256
// logits. The loss is the log of the sum plus (largest - target's), so that a token that the model is sure of keeps its digits.
// The gradient goes over pieces of the vocabulary: the tile is multiplied again, and what is written is P of the piece in the type of the
// call (fp32: three planes), as the operand of the two products behind it. P is rounded to that type, relative to each value; what that takes from the
// entry of the row's target, nearly all of a row where the others share what is left, is kept in fp32 and added to the results (with it rounded away
// gradients are 2^-8 off where their own rounding is 2^-9; 2000 rows of 32000 x 2048, the weight's gradient 329 -> 352 us); g is scaled by a power of two
// first, a row's own where the weight does not learn and the largest row's where it does, so that a mean over many rows does not leave the type's range,
// and the results are scaled back. |P| is at most the scaled g: to [1, 2), for fp16 to [2^14, 2^15), so that its small entries keep their bits
// down to 2^-28 of that and a step of 2^-38 below (at [1, 2), a row of a thousandth of the largest g lost most of a softmax over 128256 tokens).
// A quantized head (the model's lm_head) is brought to the values of its dense form piece by piece. Few rows (few_most) go past the weight as it lies
// instead, dense or codes (dense_few.h; 16 rows of 128256 x 2048, bf16: the tiles' kernel 115 us, this one 87, 6.0 TB/s).
#include "dense_stage.h"

namespace {

using namespace llmq;

constexpr float kLog2e = 1.4426950408889634f;

struct LossRows {
  const int64_t* targets;
  int rows, vocab;
};

// ---- the loss ---------------------------------------------------------------------------------------------------------------
template <typename T, int TN, int WM, int WN>
__global__ __launch_bounds__(WM * WN * kWave) void logits_kernel(const TileOperand weight, const TileOperand hidden, const int k,
                                                                      const int n_tiles, const int first_token, const int first_tile,
                                                                      const LossRows rows, float2* __restrict__ stats, float* __restrict__ chosen) {
  using O = typename TileType<T>::type;
  using Tile = DenseTile<O, 256, TN, WM, WN>;
  __shared__ __attribute__((aligned(16))) uint8_t s_mem[Tile::kLdsBytes];
  const int tile = tile_of_workgroup(blockIdx.x, gridDim.x), n0 = tile % n_tiles * TN, m0 = tile / n_tiles * 256;
  Tile t;
  t.template multiply<(TileType<T>::kPlanes == 3 ? 6 : 1)>(s_mem, weight, m0, hidden, n0, 0, k);
  if (m0 + 256 > weight.rows) {   // (the last tile of the vocabulary)
#pragma unroll
    for (int mi = 0; mi < Tile::MI; ++mi)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (m0 + Tile::row_of(mi, i) >= weight.rows) {
#pragma unroll
          for (int ni = 0; ni < Tile::NI; ++ni) t.acc[mi][ni][i] = -INFINITY;
        }
  }
  __syncthreads();   // (the stages are free)
  float2* s_stat = reinterpret_cast<float2*>(s_mem);   // [WM][TN]
  const int lane = threadIdx.x & (kWave - 1), wm = static_cast<int>(threadIdx.x) / kWave / WN;
#pragma unroll
  for (int ni = 0; ni < Tile::NI; ++ni) {
    const int col = Tile::col_of(ni), n = n0 + col;
    float top = -INFINITY;
#pragma unroll
    for (int mi = 0; mi < Tile::MI; ++mi)
#pragma unroll
      for (int i = 0; i < 4; ++i) top = fmaxf(top, t.acc[mi][ni][i]);
    top = fmaxf(top, __shfl_xor(top, 16));
    top = fmaxf(top, __shfl_xor(top, 32));
    const float from = top == -INFINITY ? 0.0f : top;   // (a wave whose tokens all lie past the vocabulary)
    float sum = 0.0f;
#pragma unroll
    for (int mi = 0; mi < Tile::MI; ++mi)
#pragma unroll
      for (int i = 0; i < 4; ++i) sum += __builtin_amdgcn_exp2f((t.acc[mi][ni][i] - from) * kLog2e);
    sum += __shfl_xor(sum, 16);
    sum += __shfl_xor(sum, 32);
    if ((lane >> 4) == 0) s_stat[wm * TN + col] = make_float2(top, sum);
    if (n < rows.rows) {
      const int64_t at = rows.targets[n] - (first_token + m0);
      if (at >= 0 && at < 256 && first_token + m0 + at < rows.vocab) {
#pragma unroll
        for (int mi = 0; mi < Tile::MI; ++mi)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (Tile::row_of(mi, i) == at) chosen[n] = t.acc[mi][ni][i];
      }
    }
  }
  __syncthreads();
  for (int col = threadIdx.x; col < TN && n0 + col < rows.rows; col += Tile::kThreads) {
    float top = s_stat[col].x;
#pragma unroll
    for (int w = 1; w < WM; ++w) top = fmaxf(top, s_stat[w * TN + col].x);
    const float from = top == -INFINITY ? 0.0f : top;
    float sum = 0.0f;
#pragma unroll
    for (int w = 0; w < WM; ++w) {
      const float2 s = s_stat[w * TN + col];
      sum += s.y * __builtin_amdgcn_exp2f(((s.x == -INFINITY ? from : s.x) - from) * kLog2e);
    }
    stats[static_cast<int64_t>(first_tile + m0 / 256) * rows.rows + n0 + col] = make_float2(top, sum);
  }
}

__device__ __forceinline__ float2 merged(float2 a, float2 b) {   // (largest, sum of exponentials over it)
  const float top = fmaxf(a.x, b.x), from = top == -INFINITY ? 0.0f : top;
  return make_float2(top, a.y * __builtin_amdgcn_exp2f(((a.x == -INFINITY ? from : a.x) - from) * kLog2e) +
                              b.y * __builtin_amdgcn_exp2f(((b.x == -INFINITY ? from : b.x) - from) * kLog2e));
}
// R rows a workgroup, the tiles dealt to 1024 / R threads each, eight in flight, merged in a fixed order. R = 4 where 16 would leave a workgroup or
// a few on the way (16 rows, 2004 tiles: 9.4 us with 16).
template <int R>
__global__ __launch_bounds__(1024) void loss_kernel(const float2* __restrict__ stats, const float* __restrict__ chosen, const int tiles,
                                                               const LossRows rows, const int64_t ignore_index, float* __restrict__ losses,
                                                               float* __restrict__ lse) {
  constexpr int kAhead = 8, kLossParts = 1024 / R;
  __shared__ float2 s_part[kLossParts][R + 1];
  const int at = threadIdx.x % R, part = threadIdx.x / R, n = blockIdx.x * R + at;
  const int row = min(n, rows.rows - 1);
  float2 all = make_float2(-INFINITY, 0.0f);
  for (int i0 = part; i0 < tiles; i0 += kAhead * kLossParts) {
    float2 v[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) v[i] = stats[static_cast<int64_t>(min(i0 + i * kLossParts, tiles - 1)) * rows.rows + row];
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
      if (i0 + i * kLossParts < tiles) all = merged(all, v[i]);
  }
  s_part[part][at] = all;
  __syncthreads();
  for (int half = kLossParts / 2; half > 0; half /= 2) {
    if (part < half) s_part[part][at] = merged(s_part[part][at], s_part[part + half][at]);
    __syncthreads();
  }
  if (part != 0 || n >= rows.rows) return;
  all = s_part[0][at];
  const float rest = logf(all.y);
  lse[n] = all.x + rest;
  const int64_t target = rows.targets[n];
  losses[n] = target == ignore_index ? 0.0f
              : target < 0 || target >= rows.vocab ? NAN : rest + (all.x - chosen[n]);
}

// tiles of 16 that have rows, of the block's NT
template <int NT> __device__ __forceinline__ int live_tiles(int rows) { return min((rows - static_cast<int>(blockIdx.y) * 16 * NT + 15) / 16, NT); }

// A few rows: 64 tokens a workgroup, a row tile of the sums a wave.
template <typename T, int BITS, int NT>
__global__ __launch_bounds__(kFewWaves * kWave, BITS != 0 && NT == 4 ? 1 : 2) void few_logits_kernel(const FewWeight weight, const T* __restrict__ x, const LossRows rows,
                                                                       float2* __restrict__ stats, float* __restrict__ chosen) {
  using Few = FewRows<T, BITS, NT>;
  __shared__ __attribute__((aligned(16))) uint8_t s_mem[Few::kLdsBytes];
  const int m0 = blockIdx.x * kFewTokens;
  Few f;
  f.multiply(s_mem, weight, m0, x + static_cast<int64_t>(blockIdx.y) * 16 * NT * weight.width, live_tiles<NT>(rows.rows));
  const int lane = threadIdx.x & (kWave - 1), wv = threadIdx.x / kWave, n = (blockIdx.y * NT + wv) * 16 + (lane & 15), v0 = 4 * (lane >> 4);
  if (wv >= NT) return;
  float top = -INFINITY;
#pragma unroll
  for (int i = 0; i < Few::kTiles; ++i)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      if (m0 + i * 16 + v0 + q >= weight.rows) f.acc[i][q] = -INFINITY;
      top = fmaxf(top, f.acc[i][q]);
    }
  top = fmaxf(top, __shfl_xor(top, 16));
  top = fmaxf(top, __shfl_xor(top, 32));
  const float from = top == -INFINITY ? 0.0f : top;
  float sum = 0.0f;
#pragma unroll
  for (int i = 0; i < Few::kTiles; ++i)
#pragma unroll
    for (int q = 0; q < 4; ++q) sum += __builtin_amdgcn_exp2f((f.acc[i][q] - from) * kLog2e);
  sum += __shfl_xor(sum, 16);
  sum += __shfl_xor(sum, 32);
  if (n >= rows.rows) return;
  if ((lane >> 4) == 0) stats[static_cast<int64_t>(blockIdx.x) * rows.rows + n] = make_float2(top, sum);
  const int64_t at = rows.targets[n] - m0;
  if (at >= 0 && at < kFewTokens && m0 + at < rows.vocab) {
#pragma unroll
    for (int i = 0; i < Few::kTiles; ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        if (i * 16 + v0 + q == at) chosen[n] = f.acc[i][q];
  }
}

// ---- the gradient -----------------------------------------------------------------------------------------------------------
// The rows that have a part in the gradient (their target is not ignore_index and their g not zero), in front and in order; the others, a
// prompt's tokens for instance, cost nothing from here on.
struct Counted {
  int32_t* row;        // [padded]: the row of each; -1 behind the last
  int32_t* place;      // [rows]: where a row went, or -1
  int64_t* target;     // [padded]
  float* lse;          // [padded]
  float* grad;         // [padded]: g 2^(lift - e) with e its own exponent, or (together) that of the largest finite |g|; 0 behind the last
  float* rest;         // [padded], 16 bits: what P's rounding took from the target's entry
  float* back;         // [padded]: 2^(e - lift)
  int32_t* count;
};
// (2^(e - lift) stays a normal number)
__device__ __forceinline__ int exponent_of(float g, int lift) { return g > 0.0f && g < INFINITY ? max(ilogbf(g), lift - 125) : lift; }
// One workgroup.
__global__ __launch_bounds__(1024) void count_rows_kernel(const float* __restrict__ grad, const int64_t* __restrict__ targets, const float* __restrict__ lse,
                                                          const int rows, const int padded, const int vocab, const int64_t ignore_index, const bool together,
                                                          const int lift, const Counted c) {
  __shared__ float s_top[16];
  __shared__ int s_n[2][16];
  const int wv = threadIdx.x / kWave, lane = threadIdx.x % kWave;
  float top = 0.0f;
  for (int i = threadIdx.x; i < rows; i += 1024) {
    const float g = fabsf(grad[i]);
    if (targets[i] != ignore_index && g < INFINITY) top = fmaxf(top, g);
  }
  top = group_max<64>(top);
  if (lane == 0) s_top[wv] = top;
  __syncthreads();
  top = s_top[0];
  for (int w = 1; w < 16; ++w) top = fmaxf(top, s_top[w]);
  const int largest = exponent_of(top, lift);
  int begin = 0;
  for (int i0 = 0, turn = 0; i0 < rows; i0 += 1024, turn ^= 1) {
    const int i = i0 + threadIdx.x;
    int64_t target = ignore_index;
    float g = 0.0f;
    if (i < rows) {
      target = targets[i];
      g = target == ignore_index ? 0.0f : grad[i];
    }
    const bool counts = g != 0.0f;   // (NaN counts)
    const uint64_t mask = __ballot(counts);
    if (lane == 0) s_n[turn][wv] = __popcll(mask);
    __syncthreads();
    int at = begin, all = 0;
    for (int w = 0; w < 16; ++w) {
      if (w < wv) at += s_n[turn][w];
      all += s_n[turn][w];
    }
    at += __popcll(mask & ((uint64_t{1} << lane) - 1));
    if (i < rows) c.place[i] = counts ? at : -1;
    if (counts) {
      c.row[at] = i;
      c.target[at] = target;
      c.lse[at] = lse[i];
      c.rest[at] = 0.0f;
      const int e = together ? largest : exponent_of(fabsf(g), lift);
      c.grad[at] = target < 0 || target >= vocab ? NAN : ldexpf(g, lift - e);
      c.back[at] = ldexpf(1.0f, e - lift);
    }
    begin += all;
  }
  for (int i = begin + threadIdx.x; i < padded; i += 1024) {
    c.row[i] = -1;
    c.target[i] = -1;
    c.lse[i] = 0.0f;
    c.grad[i] = 0.0f;
    c.back[i] = ldexpf(1.0f, largest - lift);
    c.rest[i] = 0.0f;
  }
  if (threadIdx.x == 0) *c.count = begin;
}

struct PieceOut {
  void* p;        // [padded rows, ld] a plane: zeros for rows behind the last of a step of 64, and tokens past the vocabulary
  int64_t plane;
  int ld, padded;
};

template <typename T, int TN, int WM, int WN>
__global__ __launch_bounds__(WM * WN * kWave) void piece_kernel(const TileOperand weight, const TileOperand hidden, const int k,
                                                                     const int n_tiles, const int first_token, const Counted rows, const PieceOut out) {
  using O = typename TileType<T>::type;
  constexpr int P = TileType<T>::kPlanes;
  using Tile = DenseTile<O, 256, TN, WM, WN, false, false, 2>;
  __shared__ __attribute__((aligned(16))) uint8_t s_mem[Tile::kLdsBytes];
  const int counted = (*rows.count + TN - 1) / TN, tiles = static_cast<int>(gridDim.x) / n_tiles * counted;   // tiles of the rows that count
  if (static_cast<int>(blockIdx.x) >= tiles) return;
  const int tile = tile_of_workgroup(blockIdx.x, tiles), n0 = tile % counted * TN, m0 = tile / counted * 256;
  Tile t;
  t.template multiply<(P == 3 ? 6 : 1)>(s_mem, weight, m0, hidden, n0, 0, k);
#pragma unroll
  for (int ni = 0; ni < Tile::NI; ++ni) {
    const int n = n0 + Tile::col_of(ni);
    if (n >= out.padded) continue;
    const float g = rows.grad[n], lse = rows.lse[n];   // (0 behind the last)
    const int64_t target = rows.target[n] - (first_token + m0);   // within the tile
    float at_target = 0.0f;
#pragma unroll
    for (int mi = 0; mi < Tile::MI; mi += 2) {   // eight neighbouring tokens
      uint16_t v[P][8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int m = Tile::row_of(mi, 0) + i;
        const float e = __builtin_amdgcn_exp2f((t.acc[mi + i / 4][ni][i % 4] - lse) * kLog2e) - (target == m ? 1.0f : 0.0f);
        const float f = g == 0.0f || m0 + m >= weight.rows ? 0.0f : e * g;
        if constexpr (P == 1) {
          v[0][i] = __builtin_bit_cast(uint16_t, from_float<O>(f));
          at_target = target == m ? f : at_target;
        } else {
          uint16_t p[3];
          planes_of(f, p);
#pragma unroll
          for (int j = 0; j < P; ++j) v[j][i] = p[j];
        }
      }
#pragma unroll
      for (int j = 0; j < P; ++j) {
        u32x4 w;
        w.x = v[j][0] | static_cast<uint32_t>(v[j][1]) << 16;
        w.y = v[j][2] | static_cast<uint32_t>(v[j][3]) << 16;
        w.z = v[j][4] | static_cast<uint32_t>(v[j][5]) << 16;
        w.w = v[j][6] | static_cast<uint32_t>(v[j][7]) << 16;
        store16(static_cast<uint16_t*>(out.p) + j * out.plane + static_cast<int64_t>(n) * out.ld + m0 + Tile::row_of(mi, 0), w);
      }
    }
    if constexpr (P == 1) {   // (zero where the target is not the lane's)
      const float rest = at_target - to_float(from_float<O>(at_target));
      if (rest != 0.0f) rows.rest[n] = rest;
    }
  }
}

// P of a few rows: [rows in whole blocks, ld], zeros for tokens past the vocabulary up to a multiple of 64; where the weight learns a second time as
// [tokens in 64, rows].
template <typename T> struct FewPiece {
  T* p;
  int64_t ld;
  T* turned;        // or null
  int turned_ld;
};
template <typename T, int BITS, int NT>
__global__ __launch_bounds__(kFewWaves * kWave, BITS != 0 && NT == 4 ? 1 : 2) void few_piece_kernel(const FewWeight weight, const T* __restrict__ x,
                                                                                                    const Counted rows, const FewPiece<T> out) {
  using Few = FewRows<T, BITS, NT>;
  __shared__ __attribute__((aligned(16))) uint8_t s_mem[Few::kLdsBytes];
  const int m0 = blockIdx.x * kFewTokens, t0 = blockIdx.y * 16 * NT;
  const int lane = threadIdx.x & (kWave - 1), wv = threadIdx.x / kWave, n = t0 + wv * 16 + (lane & 15), v0 = 4 * (lane >> 4);
  Few f;
  const bool none = t0 >= *rows.count;   // (a block of rows that do not count: zeros)
  if (!none) f.multiply(s_mem, weight, m0, x + static_cast<int64_t>(blockIdx.y) * 16 * NT * weight.width, live_tiles<NT>(*rows.count));
  if (wv >= NT) return;
  const float g = rows.grad[n], lse = rows.lse[n];
  const int64_t target = rows.target[n] - m0;
#pragma unroll
  for (int i = 0; i < Few::kTiles; ++i) {
    float e[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int m = i * 16 + v0 + q;
      const float value = none ? 0.0f : __builtin_amdgcn_exp2f((f.acc[i][q] - lse) * kLog2e) - (target == m ? 1.0f : 0.0f);
      e[q] = g == 0.0f || m0 + m >= weight.rows ? 0.0f : value * g;
      if (sizeof(T) == 2 && target == m) rows.rest[n] = e[q] - to_float(from_float<T>(e[q]));
      if (out.turned != nullptr) {
        T* to = out.turned + static_cast<int64_t>(m0 + m) * out.turned_ld + n;
        *to = from_float<T>(e[q]);
        if constexpr (NT == 1 && sizeof(T) == 2) to[16] = from_float<T>(0.0f);   // (a step of 32 rows)
      }
    }
    store_four(out.p + n * out.ld + m0 + i * 16 + v0, e);
  }
}

// ---- what a call takes --------------------------------------------------------------------------------------------------------
struct Plan {
  int rows, vocab, hidden, planes, size;   // size: bytes of an element of the call's type
  int k;                                   // hidden, in whole steps
  int padded;                              // rows, in whole tiles
  bool stage_hidden, stage_weight;         // whether they have to be brought into operand form
  int piece;                               // tokens of a piece, a multiple of 256
  int splits;                              // of dh's products
  bool few;                                // rows that go past the weight once, as it lies
  int row_tiles, blocks;                   // of 16, for these: 1, 2 or 4; of 16 row_tiles rows
  // offsets into the workspace
  int64_t o_stats, o_chosen, o_hidden, o_weight, o_row, o_place, o_target, o_lse, o_grad, o_rest, o_back, o_count, o_x, o_p, o_turned, o_p_turned, o_sums, bytes;
};

int64_t take(int64_t& at, int64_t bytes) {
  const int64_t here = at;
  at = round_up(at + bytes, 256);
  return here;
}

// The piece of the vocabulary: a whole number of rounds of 256 workgroups' tiles, in as much workspace. The loss's pieces stay in the caches (whole: 2047
// rows of a 128256 x 2048 int8 head 1022 us for the tiles, in pieces of up to 192 MB 963, of 68 MB 960 and the codes' pass 168 instead of 133; 1024
// rows of x 4096 967 and 812). The gradient's are several rounds: how many rows count is not known when a call is made, and there the tiles of those
// that do not leave room for others (724 of 1024: 1726 us for all products with 768 MB, 1916 with 500, 1932 with 136).
constexpr int64_t kLossPieceBytes = int64_t{192} << 20, kGradPieceBytes = int64_t{768} << 20;
// Few rows: the whole vocabulary at once, up to 2^20 tokens. 64 rows a pass over the weight: one pass where it is as wide as the operands, more where the
// tiles would have to make operands of it first or take six products (128256 x 2048: int8 in bf16, 128 rows 209 us for 337, 192 rows 353 for 350; fp32, 512 rows 2248
// for 2777, 700 rows 3150 for 2713; with gradients 300 rows 6190 for 5847, over int8 4112 for 4616, of 50257 x 768 974 for 1289, 384 rows 7727, 5008 and 1171 for 6377,
// 5018 and 1389).
constexpr int kFewVocab = 1 << 20;
constexpr int few_most(int wformat, int dtype, bool gradient) { return dtype == LLMQ_F32 ? (gradient ? 320 : 512) : wformat != 0 ? 128 : 64; }

Plan plan_for(int rows, int vocab, int hidden, int group_size, int wformat, int dtype, bool gradient, bool learned) {
  Plan p{};
  p.rows = rows;
  p.vocab = vocab;
  p.hidden = hidden;
  p.planes = dtype == LLMQ_F32 ? 3 : 1;
  p.size = dtype == LLMQ_F32 ? 4 : 2;
  p.k = static_cast<int>(round_up(hidden, 64));
  const int tn = tile_rows(rows);
  p.padded = static_cast<int>(round_up(rows, tn));
  const bool whole_steps = p.planes == 1 && hidden % 64 == 0;
  p.stage_hidden = !whole_steps || gradient;   // (gradient: the rows that count)
  p.stage_weight = !whole_steps || wformat != 0;
  const int64_t row16 = int64_t{2} * p.planes;   // bytes of a value in operand form
  const int64_t whole = round_up(vocab, 256), rows64 = round_up(rows, 64);
  int64_t per_token = p.stage_weight ? p.k * row16 : 0;
  if (gradient) per_token += rows64 * row16;
  int64_t piece = whole;
  if (per_token > 0) {
    const int64_t n_tiles = p.padded / tn, round = n_tiles >= 256 ? 256 : 256 / n_tiles * 256;   // tokens of a round of workgroups
    piece = (gradient ? kGradPieceBytes : kLossPieceBytes) / per_token / 256 * 256;
    if (piece > round) piece = piece / round * round;
    if (piece < 256) piece = 256;
    if (piece > whole) piece = whole;
  }
  p.piece = static_cast<int>(piece);
  int64_t at = 0;
  p.few = rows <= few_most(wformat, dtype, gradient) && vocab <= kFewVocab && hidden % (wformat ? 128 : 64) == 0 && (wformat == 0 || group_size % 128 == 0);
  if (p.few) {
    p.row_tiles = rows <= 16 ? 1 : rows <= 32 ? 2 : 4;
    p.blocks = (rows + 63) / 64;
    p.stage_hidden = p.stage_weight = false;
    p.piece = static_cast<int>(round_up(vocab, kFewTokens));
    const int64_t whole_rows = int64_t{16} * p.row_tiles * p.blocks;
    p.padded = static_cast<int>(round_up(whole_rows, 64));
    p.o_x = take(at, int64_t{p.size} * hidden * whole_rows);
    if (!gradient) {
      p.o_stats = take(at, round_up(vocab, kFewTokens) / kFewTokens * rows * 8);
      p.o_chosen = take(at, int64_t{4} * rows);
    } else {
      p.splits = few_splits(vocab, hidden, rows, wformat);
      p.o_p = take(at, p.size * whole_rows * p.piece);
      if (learned) {
        p.o_turned = take(at, int64_t{p.size} * hidden * p.padded);
        p.o_p_turned = take(at, int64_t{p.size} * p.padded * p.piece);
      }
      p.o_sums = take(at, int64_t{4} * p.splits * rows * hidden);
    }
  }
  if (gradient) {
    p.o_row = take(at, int64_t{4} * p.padded);
    p.o_place = take(at, int64_t{4} * rows);
    p.o_target = take(at, int64_t{8} * p.padded);
    p.o_lse = take(at, int64_t{4} * p.padded);
    p.o_grad = take(at, int64_t{4} * p.padded);
    p.o_rest = take(at, int64_t{4} * p.padded);
    p.o_back = take(at, int64_t{4} * p.padded);
    p.o_count = take(at, 4);
  }
  if (p.few) {
    p.bytes = at;
    return p;
  }
  if (p.stage_hidden) p.o_hidden = take(at, rows64 * p.k * row16);
  if (p.stage_weight) p.o_weight = take(at, piece * p.k * row16);
  if (!gradient) {
    p.o_stats = take(at, whole / 256 * rows * 8);
    p.o_chosen = take(at, int64_t{4} * rows);
  } else {
    p.splits = most_splits(hidden, rows, static_cast<int>(piece));
    p.o_p = take(at, rows64 * piece * row16);
    p.o_sums = take(at, sums_bytes(hidden, rows, p.splits));
  }
  p.bytes = at;
  return p;
}

int check(int rows, int vocab, int hidden, int group_size, int out_group, int wformat, int dtype, int64_t hidden_stride) {
  if (rows < 0 || vocab < 0 || hidden <= 0) return llmq_host::fail_invalid("bad dimension rows=%d vocab=%d hidden=%d", rows, vocab, hidden);
  if (dtype != LLMQ_F32 && dtype != LLMQ_F16 && dtype != LLMQ_BF16)
    return llmq_host::fail_invalid("dtype code %d is not float32, float16 or bfloat16", dtype);
  if (wformat != 0 && wformat != LLMQ_W_INT8 && wformat != LLMQ_W_INT4_PACKED)
    return llmq_host::fail_invalid("unsupported weight format %d, expected 0 (dense), 8 or 4", wformat);
  if (hidden % 8) return llmq_host::fail_invalid("hidden must be a multiple of 8, got %d", hidden);
  if (hidden > 65536) return llmq_host::fail_invalid("hidden must be at most 65536, got %d", hidden);
  if (wformat != 0 && (group_size <= 0 || group_size % 8 || hidden % group_size))
    return llmq_host::fail_invalid("group_size must be a positive multiple of 8 that divides hidden=%d, got %d", hidden, group_size);
  if (out_group < 0) return llmq_host::fail_invalid("out_group must be >= 0, got %d", out_group);
  if (hidden_stride < hidden || hidden_stride % 8)
    return llmq_host::fail_invalid("hidden's row stride must be a multiple of 8 of at least hidden=%d, got %lld", hidden, static_cast<long long>(hidden_stride));
  if (rows > (1 << 20) || vocab > (1 << 24)) return llmq_host::fail_invalid("at most 2^20 rows and 2^24 tokens, got %d and %d", rows, vocab);
  return 0;
}

struct Call {
  const void* hidden;
  const void* weight;
  const float* wscale;
  int64_t hidden_stride;
  int group_size, out_group, wformat;
  uint8_t* workspace;
  hipStream_t stream;
};

template <typename T> void stage_hidden(const Plan& p, const Call& c, const int32_t* gather) {
  const int rows64 = static_cast<int>(round_up(p.rows, 64));
  stage_launch<T>(StageSource{c.hidden, nullptr, gather, c.hidden_stride, p.rows, p.hidden, 0, rows64, 0, 0, 0, 0},
                  StageTarget{c.workspace + p.o_hidden, int64_t{rows64} * p.k, p.k}, 0, c.stream);
}
TileOperand hidden_operand(const Plan& p, const Call& c) {
  if (!p.stage_hidden) return TileOperand{c.hidden, 0, c.hidden_stride * 2, p.rows, 0};
  return TileOperand{c.workspace + p.o_hidden, 2 * round_up(p.rows, 64) * p.k, int64_t{2} * p.k, p.rows, 0};
}
// tokens first .. of the weight, brought into operand form where it is not
template <typename T> int weight_piece(const Plan& p, const Call& c, int first, int tokens, int dtype, TileOperand& weight) {
  weight = TileOperand{static_cast<const uint8_t*>(c.weight) + int64_t{2} * first * p.hidden, 0, int64_t{2} * p.hidden, tokens, tokens};
  if (!p.stage_weight) return 0;
  weight = TileOperand{c.workspace + p.o_weight, int64_t{2} * p.piece * p.k, int64_t{2} * p.k, tokens, tokens};
  const int groups = c.wformat ? p.hidden / c.group_size : 0;
  if (c.wformat && p.planes == 1 && p.k == p.hidden && (c.out_group == 0 || first % c.out_group == 0))
    return llmq_dequant_weight(static_cast<const uint8_t*>(c.weight) + static_cast<int64_t>(first) * p.hidden * c.wformat / 8,
                               c.wscale + static_cast<int64_t>(c.out_group > 0 ? first / c.out_group : first) * groups, c.workspace + p.o_weight, tokens,
                               groups, c.group_size, c.group_size, c.out_group, c.wformat, dtype, c.stream);
  stage_launch<T>(StageSource{c.weight, c.wscale, nullptr, p.hidden, p.vocab, p.hidden, first, tokens, groups, c.group_size, c.group_size, c.out_group},
                  StageTarget{c.workspace + p.o_weight, int64_t{p.piece} * p.k, p.k}, c.wformat, c.stream);
  return 0;
}

void loss_launch(const Plan& p, const Call& c, const float2* stats, const float* chosen, int tiles, const LossRows& rows, int64_t ignore_index,
                 float* losses, float* lse) {
  if (p.rows <= kFewRows)
    hipLaunchKernelGGL((loss_kernel<4>), dim3((p.rows + 3) / 4), dim3(1024), 0, c.stream, stats, chosen, tiles, rows, ignore_index, losses, lse);
  else
    hipLaunchKernelGGL((loss_kernel<16>), dim3((p.rows + 15) / 16), dim3(1024), 0, c.stream, stats, chosen, tiles, rows, ignore_index, losses, lse);
}

FewWeight few_weight(const Plan& p, const Call& c) {
  const int64_t row_bytes = int64_t{p.hidden} * (c.wformat ? c.wformat : 8 * p.size) / 8;
  return FewWeight{static_cast<const uint8_t*>(c.weight), c.wscale, row_bytes, p.vocab, p.hidden, c.wformat ? p.hidden / c.group_size : 0,
                   c.group_size, c.group_size, c.out_group};
}
TargetTerm target_term(const Plan& p, const Call& c, const Counted& rows) {   // (fp32: nothing is rounded away)
  return TargetTerm{p.planes == 1 ? rows.rest : nullptr, rows.target, few_weight(p, c), c.wformat};
}
template <typename T> void few_operand(const Plan& p, const Call& c, const int32_t* gather) {
  const int64_t items = int64_t{p.hidden} / (4 * kFewPack<T>) * p.row_tiles * kWave;
  hipLaunchKernelGGL((few_operand_kernel<T>), dim3(static_cast<unsigned>((items + 255) / 256), p.blocks), dim3(256), 0, c.stream, static_cast<const T*>(c.hidden),
                     c.hidden_stride, gather, p.rows, p.hidden, p.row_tiles, reinterpret_cast<T*>(c.workspace + p.o_x));
}
#define LLMQ_FEW_NT(KERNEL, BITS, ...)                                                                                        \
  if (p.row_tiles == 1) hipLaunchKernelGGL((KERNEL<T, BITS, 1>), grid, dim3(kFewWaves * kWave), 0, c.stream, __VA_ARGS__);    \
  else if (p.row_tiles == 2) hipLaunchKernelGGL((KERNEL<T, BITS, 2>), grid, dim3(kFewWaves * kWave), 0, c.stream, __VA_ARGS__); \
  else hipLaunchKernelGGL((KERNEL<T, BITS, 4>), grid, dim3(kFewWaves * kWave), 0, c.stream, __VA_ARGS__)
#define LLMQ_FEW(KERNEL, ...)                                     \
  if (c.wformat == 0) { LLMQ_FEW_NT(KERNEL, 0, __VA_ARGS__); }    \
  else if (c.wformat == 8) { LLMQ_FEW_NT(KERNEL, 8, __VA_ARGS__); } \
  else { LLMQ_FEW_NT(KERNEL, 4, __VA_ARGS__); }

template <typename T> int few_forward(const Plan& p, const Call& c, const int64_t* targets, int64_t ignore_index, float* losses, float* lse) {
  few_operand<T>(p, c, nullptr);
  const LossRows rows{targets, p.rows, p.vocab};
  float2* stats = reinterpret_cast<float2*>(c.workspace + p.o_stats);
  float* chosen = reinterpret_cast<float*>(c.workspace + p.o_chosen);
  const T* x = reinterpret_cast<const T*>(c.workspace + p.o_x);
  const FewWeight weight = few_weight(p, c);
  const dim3 grid((p.vocab + kFewTokens - 1) / kFewTokens, p.blocks);
  LLMQ_FEW(few_logits_kernel, weight, x, rows, stats, chosen)
  loss_launch(p, c, stats, chosen, static_cast<int>(grid.x), rows, ignore_index, losses, lse);
  return llmq_host::check_launch("vocab_loss");
}

// dW of tokens first ..: over the rows, both with them outermost
template <typename T>
void weight_gradient(const Plan& p, const Call& c, const TileOperand& part, int first, int tokens, const Counted& rows, void* grad_weight) {
  const int rows64 = static_cast<int>(round_up(p.rows, 64));
  TileOperand hidden_k = hidden_operand(p, c), part_k = part;
  hidden_k.rows = p.hidden;
  hidden_k.k_rows = rows64;
  part_k.rows = tokens;
  ProductOut out{static_cast<T*>(grad_weight) + static_cast<int64_t>(first) * p.hidden, p.hidden, rows.back, 0, 1, rows.count};
  if (p.planes == 1) {
    out.rest = rows.rest;
    out.target = rows.target;
    out.row = rows.row;
    out.x = c.hidden;
    out.x_stride = c.hidden_stride;
    out.first_token = first;
  }
  product_launch<T, false, true>(hidden_k, part_k, rows64, out, c.stream);
}

template <typename T>
int few_backward(const Plan& p, const Call& c, const Counted& rows, void* grad_hidden, void* grad_weight) {
  few_operand<T>(p, c, rows.row);
  const T* x = reinterpret_cast<const T*>(c.workspace + p.o_x);
  const bool learned = grad_weight != nullptr;
  const FewPiece<T> part{reinterpret_cast<T*>(c.workspace + p.o_p), p.piece, learned ? reinterpret_cast<T*>(c.workspace + p.o_p_turned) : nullptr, p.padded};
  float* sums = reinterpret_cast<float*>(c.workspace + p.o_sums);
  const FewWeight weight = few_weight(p, c);
  const unsigned tokens = (p.vocab + kFewTokens - 1) / kFewTokens;
  const dim3 grid(tokens, p.blocks);
  LLMQ_FEW(few_piece_kernel, weight, x, rows, part)
  columns_launch<T, true>(weight, FewColumns{part.p, part.ld, rows.count, p.rows, sums, p.splits}, c.wformat, c.stream);
  if (learned) {
    T* turned = reinterpret_cast<T*>(c.workspace + p.o_turned);
    const int steps = (p.rows + 4 * kFewPack<T> - 1) / (4 * kFewPack<T>);
    const int64_t items = int64_t{p.hidden} / 16 * steps * kWave;
    hipLaunchKernelGGL((few_turned_kernel<T>), dim3(static_cast<unsigned>((items + 255) / 256)), dim3(256), 0, c.stream, static_cast<const T*>(c.hidden),
                       c.hidden_stride, rows.row, p.rows, p.hidden, steps, turned);
    const FewRests rests{rows.rest, rows.target, rows.row, rows.count, c.hidden, c.hidden_stride};
#define LLMQ_OUTER(ONE)                                                                                                                             \
  hipLaunchKernelGGL((few_outer_kernel<T, ONE>), dim3(tokens), dim3(kFewWaves * kWave), 0, c.stream, part.turned, int64_t{p.padded}, turned, steps, rows.back, \
                     p.vocab, p.hidden, rests, static_cast<T*>(grad_weight))
    if (sizeof(T) == 2 || p.blocks == 1) LLMQ_OUTER(true);
    else if constexpr (sizeof(T) == 4) LLMQ_OUTER(false);
#undef LLMQ_OUTER
  }
  add_few_launch<T>(sums, p.splits, p.rows, p.hidden, rows.back, rows.place, target_term(p, c, rows), grad_hidden, c.stream);
  return llmq_host::check_launch("vocab_loss_grad");
}

template <typename T> int forward(const Plan& p, const Call& c, const int64_t* targets, int64_t ignore_index, float* losses, float* lse, int dtype) {
  if (p.few) return few_forward<T>(p, c, targets, ignore_index, losses, lse);
  if (p.stage_hidden) stage_hidden<T>(p, c, nullptr);
  const TileOperand hidden = hidden_operand(p, c);
  const LossRows rows{targets, p.rows, p.vocab};
  float2* stats = reinterpret_cast<float2*>(c.workspace + p.o_stats);
  float* chosen = reinterpret_cast<float*>(c.workspace + p.o_chosen);
  const int tn = tile_rows(p.rows), n_tiles = p.padded / tn;
  for (int first = 0; first < p.vocab; first += p.piece) {
    const int tokens = p.vocab - first < p.piece ? p.vocab - first : p.piece;
    TileOperand weight;
    if (int rc = weight_piece<T>(p, c, first, tokens, dtype, weight)) return rc;
    const dim3 grid(static_cast<unsigned>((tokens + 255) / 256) * n_tiles);
    if (tn == kFewRows)
      hipLaunchKernelGGL((logits_kernel<T, 64, 4, 2>), grid, dim3(512), 0, c.stream, weight, hidden, p.k, n_tiles, first, first / 256, rows, stats, chosen);
    else
      hipLaunchKernelGGL((logits_kernel<T, 256, 2, 4>), grid, dim3(512), 0, c.stream, weight, hidden, p.k, n_tiles, first, first / 256, rows, stats, chosen);
  }
  loss_launch(p, c, stats, chosen, (p.vocab + 255) / 256, rows, ignore_index, losses, lse);
  return llmq_host::check_launch("vocab_loss");
}

template <typename T>
int backward(const Plan& p, const Call& c, const int64_t* targets, int64_t ignore_index, const float* lse, const float* grad, void* grad_hidden,
             void* grad_weight, int dtype) {
  float* back = reinterpret_cast<float*>(c.workspace + p.o_back);
  const Counted rows{reinterpret_cast<int32_t*>(c.workspace + p.o_row), reinterpret_cast<int32_t*>(c.workspace + p.o_place),
                     reinterpret_cast<int64_t*>(c.workspace + p.o_target), reinterpret_cast<float*>(c.workspace + p.o_lse),
                     reinterpret_cast<float*>(c.workspace + p.o_grad), reinterpret_cast<float*>(c.workspace + p.o_rest), back,
                     reinterpret_cast<int32_t*>(c.workspace + p.o_count)};
  float* sums = reinterpret_cast<float*>(c.workspace + p.o_sums);
  const bool learned = grad_weight != nullptr;
  const int rows64 = static_cast<int>(round_up(p.rows, 64));
  hipLaunchKernelGGL(count_rows_kernel, dim3(1), dim3(1024), 0, c.stream, grad, targets, lse, p.rows, p.padded, p.vocab, ignore_index, learned,
                     dtype == LLMQ_F16 ? 14 : 0, rows);
  if (p.few) return few_backward<T>(p, c, rows, grad_hidden, grad_weight);
  stage_hidden<T>(p, c, rows.row);
  const TileOperand hidden = hidden_operand(p, c);
  const int tn = tile_rows(p.rows), n_tiles = p.padded / tn;
  for (int first = 0; first < p.vocab; first += p.piece) {
    const int tokens = p.vocab - first < p.piece ? p.vocab - first : p.piece;
    TileOperand weight;
    if (int rc = weight_piece<T>(p, c, first, tokens, dtype, weight)) return rc;
    const PieceOut piece{c.workspace + p.o_p, int64_t{rows64} * p.piece, p.piece, rows64};
    const dim3 grid(static_cast<unsigned>((tokens + 255) / 256) * n_tiles);
    if (tn == kFewRows)
      hipLaunchKernelGGL((piece_kernel<T, 64, 4, 2>), grid, dim3(512), 0, c.stream, weight, hidden, p.k, n_tiles, first, rows, piece);
    else
      hipLaunchKernelGGL((piece_kernel<T, 256, 2, 4>), grid, dim3(512), 0, c.stream, weight, hidden, p.k, n_tiles, first, rows, piece);
    // dh: over the piece's tokens, both as they lie (the weight's last row again behind its end, against zeros)
    TileOperand weight_k = weight;
    weight_k.rows = p.hidden;
    const TileOperand part{c.workspace + p.o_p, int64_t{2} * rows64 * p.piece, int64_t{2} * p.piece, p.rows, 0};
    product_launch<T, true, false>(weight_k, part, static_cast<int>(round_up(tokens, 64)),
                                   ProductOut{sums, p.hidden, nullptr, first == 0, p.splits, rows.count}, c.stream);
    if (learned) {
      TileOperand part_k = part;
      part_k.k_rows = rows64;
      weight_gradient<T>(p, c, part_k, first, tokens, rows, grad_weight);
    }
  }
  add_planes_launch<T>(sums, p.rows, p.hidden, p.splits, rows.count, back, rows.place, target_term(p, c, rows), grad_hidden, c.stream);
  return llmq_host::check_launch("vocab_loss_grad");
}

bool misaligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) != 0; }

}  // namespace

extern "C" size_t llmq_vocab_loss_workspace_bytes(int rows, int vocab, int hidden, int group_size, int wformat, int dtype) {
  if (rows <= 0 || vocab <= 0 || hidden <= 0) return 0;
  return static_cast<size_t>(plan_for(rows, vocab, hidden, group_size, wformat, dtype, false, false).bytes);
}
extern "C" size_t llmq_vocab_loss_grad_workspace_bytes(int rows, int vocab, int hidden, int group_size, int wformat, int dtype, int want_weight) {
  if (rows <= 0 || vocab <= 0 || hidden <= 0) return 0;
  return static_cast<size_t>(plan_for(rows, vocab, hidden, group_size, wformat, dtype, true, want_weight != 0).bytes);
}

extern "C" int llmq_vocab_loss(const void* hidden, int64_t hidden_stride, const void* weight, const float* wscale_or_null,
                               const int64_t* targets, int64_t ignore_index, float* losses, float* lse, void* workspace,
                               size_t workspace_bytes, int rows, int vocab, int hidden_size, int group_size, int out_group,
                               int wformat, int dtype, llmq_stream_t stream) {
  if (int rc = check(rows, vocab, hidden_size, group_size, out_group, wformat, dtype, hidden_stride)) return rc;
  if (rows == 0) return 0;
  if (vocab == 0) return llmq_host::fail_invalid("a vocabulary of no tokens");
  if (!hidden || !weight || !targets || !losses || !lse || (wformat != 0 && !wscale_or_null)) return llmq_host::fail_invalid("null tensor pointer");
  if (misaligned(hidden) || misaligned(weight)) return llmq_host::fail_invalid("hidden and weight must be 16-byte aligned");
  const Plan p = plan_for(rows, vocab, hidden_size, group_size, wformat, dtype, false, false);
  if (!p.few && !p.stage_hidden && !tile_spans(rows, tile_rows(rows), 2 * hidden_stride, 128))
    return llmq_host::fail_invalid("hidden's row stride is too wide: %d neighbouring rows must lie within 4 GiB, got a stride of %lld elements", tile_rows(rows),
                                   static_cast<long long>(hidden_stride));
  if (!workspace || misaligned(workspace) || workspace_bytes < static_cast<size_t>(p.bytes))
    return llmq_host::fail_invalid("the workspace must be 16-byte aligned and hold %lld bytes, got %zu", static_cast<long long>(p.bytes), workspace_bytes);
  const Call c{hidden, weight, wscale_or_null, hidden_stride, group_size, out_group, wformat, static_cast<uint8_t*>(workspace), static_cast<hipStream_t>(stream)};
  switch (dtype) {
    case LLMQ_F32: return forward<float>(p, c, targets, ignore_index, losses, lse, dtype);
    case LLMQ_F16: return forward<f16_t>(p, c, targets, ignore_index, losses, lse, dtype);
    default: return forward<bf16_t>(p, c, targets, ignore_index, losses, lse, dtype);
  }
}

extern "C" int llmq_vocab_loss_grad(const void* hidden, int64_t hidden_stride, const void* weight, const float* wscale_or_null,
                                    const int64_t* targets, int64_t ignore_index, const float* lse, const float* grad, void* grad_hidden,
                                    void* grad_weight_or_null, void* workspace, size_t workspace_bytes, int rows, int vocab, int hidden_size,
                                    int group_size, int out_group, int wformat, int dtype, llmq_stream_t stream) {
  if (int rc = check(rows, vocab, hidden_size, group_size, out_group, wformat, dtype, hidden_stride)) return rc;
  if (wformat != 0 && grad_weight_or_null) return llmq_host::fail_invalid("a quantized weight has no gradient");
  if (rows == 0) return 0;   // (nothing is written: a gradient of no rows has no elements but the weight's, which the caller clears)
  if (vocab == 0) return llmq_host::fail_invalid("a vocabulary of no tokens");
  if (!hidden || !weight || !targets || !lse || !grad || !grad_hidden || (wformat != 0 && !wscale_or_null))
    return llmq_host::fail_invalid("null tensor pointer");
  if (misaligned(hidden) || misaligned(weight) || misaligned(grad_hidden) || misaligned(grad_weight_or_null))
    return llmq_host::fail_invalid("hidden, weight and their gradients must be 16-byte aligned");
  const Plan p = plan_for(rows, vocab, hidden_size, group_size, wformat, dtype, true, grad_weight_or_null != nullptr);
  if (!workspace || misaligned(workspace) || workspace_bytes < static_cast<size_t>(p.bytes))
    return llmq_host::fail_invalid("the workspace must be 16-byte aligned and hold %lld bytes, got %zu", static_cast<long long>(p.bytes), workspace_bytes);
  const Call c{hidden, weight, wscale_or_null, hidden_stride, group_size, out_group, wformat, static_cast<uint8_t*>(workspace), static_cast<hipStream_t>(stream)};
  switch (dtype) {
    case LLMQ_F32: return backward<float>(p, c, targets, ignore_index, lse, grad, grad_hidden, grad_weight_or_null, dtype);
    case LLMQ_F16: return backward<f16_t>(p, c, targets, ignore_index, lse, grad, grad_hidden, grad_weight_or_null, dtype);
    default: return backward<bf16_t>(p, c, targets, ignore_index, lse, grad, grad_hidden, grad_weight_or_null, dtype);
  }
}
