// Attention of a batch over a cache in blocks (layout: kv_blocks.h), on the matrix core, gfx950: row i of sequence b sees
// the tokens 0 .. cached[b] + i,
//   t_j = (q . k_j) s_k(j) scale log2 e,   out = sum_j 2^t_j s_v(j) c_j / sum_j 2^t_j      (k, c: the bare codes)
//
// Mathematics. The value scale goes into the exponent: u_j = t_j + log2 s_v(j), w_j = 2^(u_j - max u), so that
//   out = sum w_j c_j / sum (w_j / s_v(j))
// and the second product meets bare codes with weights of at most 1, whatever the blocks' scales; the division in the sum of the
// softmax is one product for 16 scores, all of one block. The sum is short of weights that underflow, below 2^-126 of the largest, which
// a scale of the least, 1e-8, brings to 2^-99 / max s_v of the sum at the most: 2^-44 a token with scales up to 2^55 (values of 4e18). Codes become fp16 by placing them, sign flipped, in
// the mantissa of 1024 (one byte permute for two codes, exact); the 1152 too many are taken from the value codes (one packed
// add for two), and from the scores through sum q, in fp32. A query row is brought to [1, 2) by a power of two and enters as
// fp16: exact for 16-bit types but for elements 2^-14 below the row's largest (off by 2^-25 of that), the weights as fp16 (off by
// 2^-11, below what a 16-bit output is rounded by). For fp32 both enter as two such pieces, the second 2^11 times as high, and the
// keys without the 1152 too many: 22 bits. Running maximum and sum, and everything that is added up, are fp32.
//
// Layout. A wave takes 64 tokens at a time: four strips of 16. Both products are transposed: S^T = K Q^T leaves lane
// (row, g) with the 16 scores of strip g for its row, so scales and the block of a strip are the lane's own, and its
// weights are, as they lie, the second product's operand: O^T = V^T P^T, whose other operand, 16 tokens of one column, is
// one 16-byte load of the value codes. Keys and values go from memory to registers, with no LDS in between and no barrier in
// the walk. A workgroup has four waves and 64 NR rows (rows of a sequence x query heads of one key head): waves
// take row tiles of 16 NR each, or, where there are fewer than three, share a row tile's tokens and meet in LDS at the end. With
// three row tiles or four (NR = 2) all waves walk the same tokens, each converts a quarter of a tile's codes and hands the operands
// on through LDS: by trace 2000 rows on 6000 tokens, 32 / 8 heads of 128, 347 -> 310 us.
//
// Bound. Steps: HBM, in the walk 5.9 TB/s (131000 tokens of eight heads of 128: 45.5 us by trace, and 4.7 for the merge; 48 ragged
// sequences of 150000 tokens 60.0); short ones the chain lengths -> table -> codes, a trip to memory each (600 tokens of heads of 64: 6.6). Chunks:
// the issue of vector instructions, softmax and conversion (56 % of the time, the matrix core 33 %, LDS 39 %, at 2.1 GHz).
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "kv_blocks.h"

namespace {

using namespace llmq;

typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v2f __attribute__((ext_vector_type(2)));

constexpr int kWaves = 4, kThreads = kWaves * kWave, kTile = 64;
constexpr int kHeader = 4;            // floats in front of a partial result: maximum, sum, two of nothing
constexpr int kMaxSplits = 64;        // of a row: what a wave's lanes hold
constexpr int kUnits = 768;           // workgroups that the work is cut for: a round and a half of those resident with heads of 128
constexpr int kLeastTiles = 8;        // of a split: two for each wave
constexpr int kFewSplits = 8;         // .. that a row's wave merges
constexpr int kMostRecords = 1 << 16; // partial results of a launch (more would cost more than they save)
constexpr float kBias = 1152.0f;      // what a code is too high as an operand: 1024, and 128 of the flipped sign
constexpr float kNoScale = 0x1p-100f; // value scales below count as zero
constexpr float kPiece = 2048.0f;     // the second piece of an fp32 number is this much too high

// Division by a number that the host knows: the estimate is the quotient or one more.
struct Divisor {
  uint32_t by, inverse;   // 2^32 / by, rounded up (by > 1)
  __device__ __forceinline__ uint32_t quotient(uint32_t x) const {
    if (by == 1) return x;
    const uint32_t q = __umulhi(x, inverse);
    return q * by > x ? q - 1 : q;
  }
};

struct Problem {
  const void* query;
  int64_t q_stride;
  const int8_t *k_codes, *v_codes;
  const float *k_scale, *v_scale;
  BlockTable table;
  const int32_t* cached;
  Ragged rows;
  void* out;
  int32_t* split_counts;   // [rows, q_heads]: how many partial results there are
  float* partials;         // [rows, q_heads, splits]
  int splits, q_heads, heads, group, block_shift;
  float scale_log2e;
  Divisor by_group;
};

__device__ __forceinline__ int wave_total(int v) {
  v = row16_sum(v);
  return (__builtin_amdgcn_readlane(v, 0) + __builtin_amdgcn_readlane(v, 16)) + (__builtin_amdgcn_readlane(v, 32) + __builtin_amdgcn_readlane(v, 48));
}
// sum over the lanes up to and with this one
__device__ __forceinline__ int wave_prefix(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, true);   // from 1, 2, 4 and 8 lanes below within a row of 16
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, true);
  const int row = (threadIdx.x & (kWave - 1)) >> 4, a = __builtin_amdgcn_readlane(v, 15), b = __builtin_amdgcn_readlane(v, 31),
            c = __builtin_amdgcn_readlane(v, 47);
  return v + (row > 0 ? a : 0) + (row > 1 ? b : 0) + (row > 2 ? c : 0);
}

// A sequence of the batch, and its work: `groups` row groups of at most `tiles` tiles of 64 tokens.
struct Sequence {
  int first, n, cached, groups, tiles;
};
__device__ __forceinline__ Sequence sequence_of(const Problem& a, int b, int group_rows) {
  // (its three numbers are asked for together: one trip to memory)
  const int at = min(b, a.rows.sequences - 1);
  int from = at, to = at + 1;
  if (a.rows.start != nullptr) {
    from = a.rows.start[at];
    to = a.rows.start[at + 1];
  }
  const int cached = a.cached[at];
  const int first = min(max(from, 0), a.rows.rows), n = b < a.rows.sequences ? max(min(max(to, 0), a.rows.rows) - first, 0) : 0;   // (as in Ragged)
  const int64_t held = min(static_cast<int64_t>(a.table.width) << a.block_shift, static_cast<int64_t>(INT32_MAX - 2 * kTile));
  const int seen = cached < 0 ? 0 : static_cast<int>(min(static_cast<int64_t>(cached) + n, held));
  return Sequence{first, n, cached, (n * a.group + group_rows - 1) / group_rows, (seen + kTile - 1) / kTile};
}
// The piece of work of a workgroup, found by each of its waves.
struct Unit {
  int b, first, n, cached;          // its sequence
  int row_group, split, splits;     // splits of this sequence
};
// Lengths lie on the device: how the tokens are cut is decided here, the same way by everyone. All units are of about as many
// tiles, C = max(kLeastTiles, all tiles / (kUnits / heads)), a sequence is cut into ceil(tiles / C) equal splits, at most
// a.splits; so there are at most sum(groups (tiles / C + 1)) <= kUnits / heads + groups of them, the launch's size.
__device__ __forceinline__ bool find_unit(const Problem& a, int group_rows, int index, Unit& u) {
  const int lane = threadIdx.x & (kWave - 1), sequences = a.rows.sequences;
  constexpr int kBatches = 4;   // of 64 sequences, asked for together
  Sequence s = sequence_of(a, lane, group_rows);
  int size = INT32_MAX / 2;
  if (a.splits > 1) {
    int64_t all = 0;
    const auto add = [&](const Sequence& x) {
      const int64_t product = static_cast<int64_t>(x.groups) * x.tiles;
      all += wave_total(static_cast<int>(product & 0xffff)) + (static_cast<int64_t>(wave_total(static_cast<int>(product >> 16))) << 16);
    };
    add(s);
    for (int b0 = kWave; b0 < sequences; b0 += kBatches * kWave) {
      Sequence more[kBatches];
#pragma unroll
      for (int i = 0; i < kBatches; ++i) more[i] = sequence_of(a, b0 + i * kWave + lane, group_rows);
#pragma unroll
      for (int i = 0; i < kBatches; ++i) add(more[i]);
    }
    const int64_t wanted = (kUnits + a.heads - 1) / a.heads;
    size = static_cast<int>(max((all + wanted - 1) / wanted, static_cast<int64_t>(kLeastTiles)));
  }
  for (int b0 = 0; b0 < sequences; b0 += kWave) {
    if (b0 != 0) s = sequence_of(a, b0 + lane, group_rows);
    const int splits = max(min((s.tiles + size - 1) / size, a.splits), 1), units = s.groups * splits, up_to = wave_prefix(units);
    const int total = __builtin_amdgcn_readlane(up_to, kWave - 1);
    if (index < total) {
      const int at = __popcll(__ballot(up_to <= index));   // (the first lane whose units reach beyond the index)
      u.b = b0 + at;
      u.first = __builtin_amdgcn_readlane(s.first, at);
      u.n = __builtin_amdgcn_readlane(s.n, at);
      u.cached = __builtin_amdgcn_readlane(s.cached, at);
      u.splits = __builtin_amdgcn_readlane(splits, at);
      const int within = index - (__builtin_amdgcn_readlane(up_to, at) - __builtin_amdgcn_readlane(units, at));
      u.row_group = within / u.splits;
      u.split = within % u.splits;
      return true;
    }
    index -= total;
  }
  return false;
}

template <typename T> struct Pieces { static constexpr int N = 1; };
template <> struct Pieces<float> { static constexpr int N = 2; };

// The two values that a lane and the one 32 (16) lanes away have, in either of them.
template <int STEP> __device__ __forceinline__ v2f both(float v) {
#if defined(__HIP_DEVICE_COMPILE__)
  const uint32_t x = __builtin_bit_cast(uint32_t, v);
  uint32_t lo, hi;   // (the cast of a vector's element reads its first one: taken out ahead of it)
  if constexpr (STEP == 32) {
    const auto r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    lo = r[0];
    hi = r[1];
  } else {
    const auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    lo = r[0];
    hi = r[1];
  }
  return v2f{__builtin_bit_cast(float, lo), __builtin_bit_cast(float, hi)};
#else
  return v2f{v, v};
#endif
}
// over the four lanes (row, 0 .. 3)
__device__ __forceinline__ float max_of_rows(float v) {
  v2f x = both<32>(v);
  x = both<16>(fmaxf(x[0], x[1]));
  return fmaxf(x[0], x[1]);
}
__device__ __forceinline__ float sum_of_rows(float v) {
  v2f x = both<32>(v);
  x = both<16>(x[0] + x[1]);
  return x[0] + x[1];
}

__device__ __forceinline__ v4f product(u32x4 a, u32x4 b, v4f c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
}
__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(v2f{lo, hi}, v2h));
}
// four codes as fp16, EXACT or 1152 too high
template <bool EXACT> __device__ __forceinline__ u32x2 codes_to_half(uint32_t word) {
  const uint32_t w = word ^ 0x80808080u;
  u32x2 r{__builtin_amdgcn_perm(0x64646464u, w, 0x04010400u), __builtin_amdgcn_perm(0x64646464u, w, 0x04030402u)};
  if constexpr (EXACT) {
    const v2h bias = {static_cast<_Float16>(-kBias), static_cast<_Float16>(-kBias)};
    r.x = __builtin_bit_cast(uint32_t, __builtin_bit_cast(v2h, r.x) + bias);
    r.y = __builtin_bit_cast(uint32_t, __builtin_bit_cast(v2h, r.y) + bias);
  }
  return r;
}
template <bool EXACT> __device__ __forceinline__ u32x4 operand(uint32_t lo, uint32_t hi) {
  const u32x2 a = codes_to_half<EXACT>(lo), b = codes_to_half<EXACT>(hi);
  return u32x4{a.x, a.y, b.x, b.y};
}

template <typename T> __device__ __forceinline__ void load8(const T* p, float* f) {
#pragma unroll
  for (int i = 0; i < 8; i += Pack<T>::N) Pack<T>::unpack(load16(p + i), f + i);
}
template <typename T> __device__ __forceinline__ void store8(T* p, const float* f) {
#pragma unroll
  for (int i = 0; i < 8; i += Pack<T>::N) store16(p + i, Pack<T>::pack(f + i));
}

// Loads of codes in front of the walk and within it. Of two loads whose results meet at the head of a loop the compiler makes one
// behind it, which is where they are needed; being of different kinds, these stay where they are asked for. ONCE: past the caches,
// where a launch may read more than they hold and a wave what no other one does (streams, the rule below).
template <bool ONCE> struct InWalk {
  static __device__ __forceinline__ u32x4 load(const void* p) {
    if constexpr (!ONCE) return load16(p);
    typedef uint32_t v4u __attribute__((ext_vector_type(4)));
    const v4u r = __builtin_nontemporal_load(static_cast<const v4u*>(p));
    return u32x4{r[0], r[1], r[2], r[3]};
  }
};
template <bool ONCE> struct Ahead {
  static __device__ __forceinline__ u32x4 load(const void* p) {
    if constexpr (ONCE) return load16(p);
    typedef uint32_t v4u __attribute__((ext_vector_type(4)));
    const v4u r = *static_cast<const v4u*>(p);
    return u32x4{r[0], r[1], r[2], r[3]};
  }
};

// waves a SIMD: heads of 256, and fp32 with several row tiles, need more than half of its registers
template <typename T, int D, int NR> constexpr int kOccupancy = D == 256 || (Pieces<T>::N > 1 && NR * D >= 256) ? 1 : 2;

template <typename T, int D, int NR, bool ONCE>
__global__ __launch_bounds__(kThreads, (kOccupancy<T, D, NR>)) void attention_kernel(const Problem a) {
  constexpr int kPieces = Pieces<T>::N;
  constexpr bool kExactKeys = kPieces > 1;
  constexpr int kChunks = D / 64, kSteps = D / 32, kColumns = D / 16;   // 64-element pieces, k-steps of S^T, row tiles of O^T
  constexpr int kRows = 16 * NR, kGroupRows = kWaves * kRows, kRow = D + 4;
  constexpr bool kTogether = NR > 1;   // whether waves with a row tile each share the conversion of the codes
  constexpr int kOperands = 4 * kSteps + 2 * kColumns, kParts = kColumns / kWaves;   // of a tile, 1 KB each; value columns that a wave converts
  constexpr int kResults = kWaves * kRows * kRow * 4, kBuffers = kTogether ? 2 * kOperands * 1024 : 0;
  __shared__ __attribute__((aligned(16))) unsigned char s_mem[kResults > kBuffers ? kResults : kBuffers];
  __shared__ float s_max[kGroupRows], s_sum[kGroupRows];

  const int tid = threadIdx.x, lane = tid & (kWave - 1), r16 = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  // Key heads fastest: with eight of them each XCD's cache holds one. Rows that see most first where nothing is split; where it is,
  // all units are alike, and the launch's spare workgroups stand behind them.
  const int h = blockIdx.x % a.heads, index = blockIdx.x / a.heads;
  Unit unit{0, 0, 1, 0, 0, 0, 1};
  if (a.splits == 1 && a.rows.start == nullptr) {
    const int per = (a.group + kGroupRows - 1) / kGroupRows;
    unit.b = unit.first = index / per;
    unit.row_group = index % per;
    unit.cached = a.cached[unit.b];
  } else if (!find_unit(a, kGroupRows, a.splits > 1 ? index : static_cast<int>(gridDim.x / a.heads) - 1 - index, unit)) {
    return;
  }
  const int n_rows = unit.n * a.group, row0 = unit.row_group * kGroupRows, cached = unit.cached;
  const int here = min(n_rows - row0, kGroupRows), tiles_of_rows = (here + kRows - 1) / kRows;
  const int sharing = tiles_of_rows == 1 ? 4 : tiles_of_rows == 2 ? 2 : 1;   // waves that share a row tile
  const int my_tile = wave / sharing, my_share = wave % sharing;
  const int wave_row = row0 + my_tile * kRows;

  // the walk: tiles of 64 tokens, from the split's first one on. `seen`: the last token of a row of the sequence, -1: none
  const int64_t held = static_cast<int64_t>(a.table.width) << a.block_shift;
  const int most_seen = static_cast<int>(min(held - 1, static_cast<int64_t>(INT32_MAX - 2 * kTile)));
  const auto seen = [&](int token) { return cached < 0 ? -1 : static_cast<int>(min(static_cast<int64_t>(cached) + token, static_cast<int64_t>(most_seen))); };
  const int seen_last = wave_row < n_rows ? seen(static_cast<int>(a.by_group.quotient(min(row0 + (my_tile + 1) * kRows, n_rows) - 1))) : -1;
  const bool together = kTogether && sharing == 1;
  const int seen_here = together ? seen(static_cast<int>(a.by_group.quotient(row0 + here - 1))) : seen_last;   // by what walks as one
  const int tiles = (seen_here + kTile) / kTile, per_split = unit.splits == 1 ? tiles : (tiles + unit.splits - 1) / unit.splits;
  const int begin = unit.split * per_split, end = min(begin + per_split, tiles);

  // the blocks of a tile's strips: for its keys a lane reads strip r16 / 4, for its values and scales strip g
  const int k_strip = r16 >> 2;
  const int32_t* table = a.table.entries + unit.b * a.table.row_stride;
  struct Entries {
    int k, v;   // of the table, as they are
  };
  const auto entries_of = [&](int tile) {
    const int at = tile * kTile, most = a.table.width - 1;
    return Entries{table[min((at + kStrip * k_strip) >> a.block_shift, most)], table[min((at + kStrip * g) >> a.block_shift, most)]};
  };
  // the block of a strip, -1: none, or none that is seen
  const auto block_of = [&](int entry, int at) { return ((at > seen_here) | (entry >= a.table.blocks)) ? -1 : entry; };
  const int in_block = (1 << a.block_shift) - 1;
  // this lane's first bytes of a tile: key codes of token 16 k_strip + r16 % 4 from element 16 g on, value codes of strip g and column r16
  const auto key_address = [&](int tile, int id) {
    const int slot = (tile * kTile + kStrip * k_strip) & in_block;
    return a.k_codes + ((static_cast<int64_t>(max(id, 0)) * a.heads + h) * (in_block + 1) + slot + (r16 & 3)) * D + 16 * g;
  };
  const auto value_address = [&](int tile, int id) {
    const int slot = (tile * kTile + kStrip * g) & in_block;
    return a.v_codes + ((static_cast<int64_t>(max(id, 0)) * a.heads + h) * (in_block + 1) + slot) * D + kStrip * r16;
  };
  u32x4 k_raw[4][kChunks], v_raw[kColumns];
  const auto load_keys = [&](int tile, int id, auto when) {
    const int8_t* p = key_address(tile, id);
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int c = 0; c < kChunks; ++c) k_raw[t][c] = when.load(p + 4 * t * D + 64 * c);
  };
  const auto load_values = [&](int tile, int id, auto when) {
    const int8_t* p = value_address(tile, id);
#pragma unroll
    for (int c = 0; c < kColumns; ++c) v_raw[c] = when.load(p + 16 * kStrip * c);
  };
  float k_scale = 0.0f, v_scale = 0.0f;
  const auto load_scales = [&](int id) {
    const int64_t at = static_cast<int64_t>(max(id, 0)) * a.heads + h;
    k_scale = a.k_scale[at];
    v_scale = a.v_scale[at];
  };

  // what the first tile needs is asked for in the order of its use: table, queries, keys, values
  int tile = begin + my_share;
  Entries now{0, 0}, next{0, 0};
  if (tile < end) {
    now = entries_of(tile);
    next = entries_of(min(tile + sharing, end - 1));
  }
  constexpr int kPackets = 8 / Pack<T>::N;
  u32x4 q_raw[NR][kSteps][kPackets];
  int last[NR];   // the last token that the row sees
#pragma unroll
  for (int n = 0; n < NR; ++n) {
    const uint32_t row = min(wave_row + 16 * n + r16, n_rows - 1), token = a.by_group.quotient(row);
    last[n] = seen(static_cast<int>(token));
    const T* x = static_cast<const T*>(a.query) + (unit.first + static_cast<int64_t>(token)) * a.q_stride +
                 static_cast<int64_t>(h * a.group + (row - token * a.group)) * D + 16 * g;
#pragma unroll
    for (int s = 0; s < kSteps; ++s)
#pragma unroll
      for (int e = 0; e < kPackets; ++e) q_raw[n][s][e] = load16(x + 64 * (s / 2) + 8 * (s % 2) + e * Pack<T>::N);
  }
  const int seen_first = __builtin_amdgcn_readfirstlane(last[0]);   // (rows of a wave see more and more)

  // this lane's rows, with the scale's sign: the largest score is the largest sum of products
  const float sign = a.scale_log2e < 0.0f ? -1.0f : 1.0f;
  u32x4 q[NR][kSteps][kPieces];
  float q_scale[NR], q_bias[NR];
  const auto take_queries = [&]() {
#pragma unroll
  for (int n = 0; n < NR; ++n) {
    float f[kSteps][8], largest = 0.0f;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
#pragma unroll
      for (int e = 0; e < kPackets; ++e) Pack<T>::unpack(q_raw[n][s][e], f[s] + e * Pack<T>::N);
#pragma unroll
      for (int e = 0; e < 8; ++e) largest = fmaxf(largest, fabsf(f[s][e]));
    }
    largest = max_of_rows(largest);
    const int exponent = __builtin_amdgcn_frexp_expf(largest) - 1;
    float total = 0.0f;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      uint32_t hi[4], lo[4];
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        const float x0 = ldexpf(f[s][e] * sign, -exponent), x1 = ldexpf(f[s][e + 1] * sign, -exponent);
        hi[e / 2] = pack_half(x0, x1);
        const v2h top = __builtin_bit_cast(v2h, hi[e / 2]);
        if constexpr (kPieces > 1) lo[e / 2] = pack_half((x0 - static_cast<float>(top[0])) * kPiece, (x1 - static_cast<float>(top[1])) * kPiece);
        else total += static_cast<float>(top[0]) + static_cast<float>(top[1]);
      }
      q[n][s][0] = u32x4{hi[0], hi[1], hi[2], hi[3]};
      if constexpr (kPieces > 1) q[n][s][kPieces - 1] = u32x4{lo[0], lo[1], lo[2], lo[3]};
    }
    q_bias[n] = kExactKeys ? 0.0f : -kBias * sum_of_rows(total);
    q_scale[n] = ldexpf(fabsf(a.scale_log2e), exponent);
  }
  };

  v4f o[NR][kColumns], s[NR][4];
  uint32_t p[NR][2][kPieces][4];
  float m_run[NR], l_run[NR], alpha[NR];
#pragma unroll
  for (int n = 0; n < NR; ++n) {
    m_run[n] = -INFINITY;
    l_run[n] = 0.0f;
#pragma unroll
    for (int c = 0; c < kColumns; ++c) o[n][c] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
  }
  // scores of tokens 16 g + 4 t + i, in s[.][t][i] of lane (row, g): the products of sub-tile t
  const auto scores = [&](int t, const u32x4* k) {
#pragma unroll
    for (int n = 0; n < NR; ++n) s[n][t] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    if constexpr (kPieces > 1) {
#pragma unroll
      for (int n = 0; n < NR; ++n) {
#pragma unroll
        for (int x = 0; x < kSteps; ++x) s[n][t] = product(k[x], q[n][x][kPieces - 1], s[n][t]);
#pragma unroll
        for (int i = 0; i < 4; ++i) s[n][t][i] *= 1.0f / kPiece;
      }
    }
#pragma unroll
    for (int x = 0; x < kSteps; ++x)
#pragma unroll
      for (int n = 0; n < NR; ++n) s[n][t] = product(k[x], q[n][x][0], s[n][t]);
  };
  // their weights in operands p, and the running maximum and sum
  const auto weights = [&](int at_tile, float ks, float vs, bool strip) {
    const bool no_values = vs < kNoScale;   // (not a number: stays so)
    const float log_vs = strip ? __builtin_amdgcn_logf(no_values ? kNoScale : vs) : -INFINITY;
    const float inv_vs = 1.0f / (no_values ? kNoScale : vs);
    const int at = at_tile * kTile + kStrip * g;
    const bool whole = at_tile * kTile + kTile - 1 <= seen_first;
#pragma unroll
    for (int n = 0; n < NR; ++n) {
      const float factor = strip ? q_scale[n] * ks : 0.0f, offset = fmaf(q_bias[n], factor, log_vs);
      float top = -INFINITY;
      if (!whole) {   // the scores in full, with those that are not seen left out
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[n][t][i] = 4 * t + i > last[n] - at ? -INFINITY : fmaf(s[n][t][i], factor, offset);
      }
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) top = fmaxf(top, s[n][t][i]);
      const float by = whole ? factor : 1.0f, plus = whole ? offset : 0.0f;   // (factor is not negative)
      const float m_new = fmaxf(m_run[n], max_of_rows(fmaf(top, by, plus))), base = m_new == -INFINITY ? 0.0f : m_new;
      alpha[n] = __builtin_amdgcn_exp2f(m_run[n] - base);
      m_run[n] = m_new;
      float total = 0.0f;
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int i = 0; i < 4; i += 2) {
          const float w0 = __builtin_amdgcn_exp2f(fmaf(s[n][t][i], by, plus - base)), w1 = __builtin_amdgcn_exp2f(fmaf(s[n][t][i + 1], by, plus - base));
          total += w0 + w1;
          const uint32_t hi = pack_half(w0, w1);
          p[n][t / 2][0][2 * (t % 2) + i / 2] = hi;
          if constexpr (kPieces > 1) {
            const v2h h2 = __builtin_bit_cast(v2h, hi);
            p[n][t / 2][kPieces - 1][2 * (t % 2) + i / 2] =
                pack_half((w0 - static_cast<float>(h2[0])) * kPiece, (w1 - static_cast<float>(h2[1])) * kPiece);
          }
        }
      // (a strip that this row does not see adds nothing, whatever its scale holds)
      l_run[n] = fmaf(l_run[n], alpha[n], total == 0.0f ? 0.0f : total * inv_vs);
    }
    if (__any(strip && no_values)) {   // values of nothing: their tokens count in the sum alone
#pragma unroll
      for (int n = 0; n < NR; ++n)
#pragma unroll
        for (int y = 0; y < 2; ++y)
#pragma unroll
          for (int e = 0; e < kPieces; ++e)
#pragma unroll
            for (int w = 0; w < 4; ++w) p[n][y][e][w] = no_values ? 0u : p[n][y][e][w];
    }
    __builtin_amdgcn_sched_barrier(0);
    bool moved = false;
#pragma unroll
    for (int n = 0; n < NR; ++n) moved = moved || alpha[n] != 1.0f;
    if (__any(moved)) {
#pragma unroll
      for (int n = 0; n < NR; ++n)
#pragma unroll
        for (int c = 0; c < kColumns; ++c)
#pragma unroll
          for (int i = 0; i < 4; ++i) o[n][c][i] *= alpha[n];
    }
  };
  // the weighted codes of 16 columns
  const auto add_values = [&](int c, const u32x4& v0, const u32x4& v1) {
    const auto weight = [&](int n, int y, int e) { return u32x4{p[n][y][e][0], p[n][y][e][1], p[n][y][e][2], p[n][y][e][3]}; };
#pragma unroll
    for (int n = 0; n < NR; ++n) {
      if constexpr (kPieces > 1) {
        v4f low = {0.0f, 0.0f, 0.0f, 0.0f};
        low = product(v0, weight(n, 0, kPieces - 1), low);
        low = product(v1, weight(n, 1, kPieces - 1), low);
#pragma unroll
        for (int i = 0; i < 4; ++i) o[n][c][i] = fmaf(low[i], 1.0f / kPiece, o[n][c][i]);
      }
      o[n][c] = product(v0, weight(n, 0, 0), o[n][c]);
      o[n][c] = product(v1, weight(n, 1, 0), o[n][c]);
    }
  };

  if (!together) {
    // Each wave its own tiles: scores, weights, weighted codes. The next tile's keys are asked for as soon as this one's are in
    // operands, its values likewise. A wave's loads come back in order, so what is waited for stands in front of what is
    // not (the table's entries of the tile after next are read between the next tile's keys and its values), and no load
    // depends on a branch, behind which the compiler would have to wait as if it had not been issued: the last tile asks for
    // itself once more.
    int v_id = -1;
    if (tile < end) {
      v_id = block_of(now.v, tile * kTile + kStrip * g);
      load_keys(tile, block_of(now.k, tile * kTile + kStrip * k_strip), Ahead<ONCE>());
      load_scales(v_id);
      load_values(tile, v_id, Ahead<ONCE>());
    }
    take_queries();
    for (; tile < end; tile += sharing) {
      const int next_tile = min(tile + sharing, end - 1);
      const float ks = k_scale, vs = v_scale;
      const bool strip = v_id >= 0;
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        u32x4 k[kSteps];
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
          k[2 * c] = operand<kExactKeys>(k_raw[t][c].x, k_raw[t][c].y);
          k[2 * c + 1] = operand<kExactKeys>(k_raw[t][c].z, k_raw[t][c].w);
        }
        scores(t, k);
      }
      __builtin_amdgcn_sched_barrier(0);   // (the phases as they stand: mixed, they take more registers than there are)
      v_id = block_of(next.v, next_tile * kTile + kStrip * g);
      load_keys(next_tile, block_of(next.k, next_tile * kTile + kStrip * k_strip), InWalk<ONCE>());
      load_scales(v_id);
      next = entries_of(min(tile + 2 * sharing, end - 1));
      __builtin_amdgcn_sched_barrier(0);
      weights(tile, ks, vs, strip);
#pragma unroll
      for (int c = 0; c < kColumns; ++c) add_values(c, operand<true>(v_raw[c].x, v_raw[c].y), operand<true>(v_raw[c].z, v_raw[c].w));
      __builtin_amdgcn_sched_barrier(0);
      load_values(next_tile, v_id, InWalk<ONCE>());
    }
  } else if constexpr (kTogether) {
    // All waves the same tiles, each with rows of its own: a wave converts a quarter of a tile's codes (keys of sub-tile `wave`,
    // some columns of the values) and hands the operands on through LDS, in the order in which they are read, 16 bytes a lane.
    // Two buffers: while one is read the next tile is written into the other, one barrier a tile.
    u32x4* buffer = reinterpret_cast<u32x4*>(s_mem);
    u32x4 k_part[kChunks], v_part[kParts];
    const auto load_part = [&](int at_tile, const Entries& e, auto when, bool& strip) {
      const int k_id = block_of(e.k, at_tile * kTile + kStrip * k_strip), v_id = block_of(e.v, at_tile * kTile + kStrip * g);
      strip = v_id >= 0;
      const int8_t* k = key_address(at_tile, k_id) + 4 * wave * D;
#pragma unroll
      for (int c = 0; c < kChunks; ++c) k_part[c] = when.load(k + 64 * c);
      load_scales(v_id);
      const int8_t* v = value_address(at_tile, v_id) + 16 * kStrip * kParts * wave;
#pragma unroll
      for (int c = 0; c < kParts; ++c) v_part[c] = when.load(v + 16 * kStrip * c);
    };
    const auto hand_on = [&](int which) {
      u32x4* to = buffer + which * kOperands * kWave + lane;
#pragma unroll
      for (int c = 0; c < kChunks; ++c) {
        to[(wave * kSteps + 2 * c) * kWave] = operand<kExactKeys>(k_part[c].x, k_part[c].y);
        to[(wave * kSteps + 2 * c + 1) * kWave] = operand<kExactKeys>(k_part[c].z, k_part[c].w);
      }
#pragma unroll
      for (int c = 0; c < kParts; ++c) {
        to[(4 * kSteps + 2 * (kParts * wave + c)) * kWave] = operand<true>(v_part[c].x, v_part[c].y);
        to[(4 * kSteps + 2 * (kParts * wave + c) + 1) * kWave] = operand<true>(v_part[c].z, v_part[c].w);
      }
    };
    bool strip = false, next_strip = false;
    float ks = 0.0f, vs = 0.0f;
    int which = 0;
    if (tile < end) {
      load_part(tile, now, Ahead<ONCE>(), strip);
      take_queries();
      hand_on(0);
      ks = k_scale;
      vs = v_scale;
      load_part(min(tile + 1, end - 1), next, Ahead<ONCE>(), next_strip);
      next = entries_of(min(tile + 2, end - 1));
      __syncthreads();
    }
    for (; tile < end; ++tile) {
      if (tile * kTile <= seen_last) {   // (of this wave)
        const u32x4* from = buffer + which * kOperands * kWave + lane;
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          u32x4 k[kSteps];
#pragma unroll
          for (int x = 0; x < kSteps; ++x) k[x] = from[(t * kSteps + x) * kWave];
          scores(t, k);
        }
        __builtin_amdgcn_sched_barrier(0);
        weights(tile, ks, vs, strip);
#pragma unroll
        for (int c = 0; c < kColumns; ++c) add_values(c, from[(4 * kSteps + 2 * c) * kWave], from[(4 * kSteps + 2 * c + 1) * kWave]);
        __builtin_amdgcn_sched_barrier(0);
      }
      which ^= 1;
      hand_on(which);
      ks = k_scale;
      vs = v_scale;
      strip = next_strip;
      load_part(min(tile + 2, end - 1), next, InWalk<ONCE>(), next_strip);
      next = entries_of(min(tile + 3, end - 1));
      __syncthreads();
    }
  }

  float* s_part = reinterpret_cast<float*>(s_mem);   // (behind the walk's last barrier, where it has one)
  // the waves that share a row tile: max m_w, sum l_w 2^(m_w - m), sum O_w 2^(m_w - m), in wave order
#pragma unroll
  for (int n = 0; n < NR; ++n) {
    l_run[n] = sum_of_rows(l_run[n]);
    if (g == 0) {
      s_max[wave * kRows + 16 * n + r16] = m_run[n];
      s_sum[wave * kRows + 16 * n + r16] = l_run[n];
    }
    float* part = s_part + (wave * kRows + 16 * n + r16) * kRow + 4 * g;
#pragma unroll
    for (int c = 0; c < kColumns; ++c) *reinterpret_cast<v4f*>(part + 16 * c) = o[n][c];
  }
  __syncthreads();
  constexpr int kPacketsOut = D / 8;
  const auto finish = [&](auto sharing_tag) {
    constexpr int kSharing = decltype(sharing_tag)::value;
    for (int item = tid; item < here * kPacketsOut; item += kThreads) {
      const int row = item / kPacketsOut, d = item % kPacketsOut * 8, at = row / kRows * kSharing * kRows + row % kRows;
      float m[kSharing], l = 0.0f, f[8] = {}, top = -INFINITY;
      v4f lo[kSharing], hi[kSharing];
#pragma unroll
      for (int w = 0; w < kSharing; ++w) {
        m[w] = s_max[at + w * kRows];
        lo[w] = *reinterpret_cast<const v4f*>(s_part + (at + w * kRows) * kRow + d);
        hi[w] = *reinterpret_cast<const v4f*>(s_part + (at + w * kRows) * kRow + d + 4);
        top = fmaxf(top, m[w]);
      }
      const float base = top == -INFINITY ? 0.0f : top;
#pragma unroll
      for (int w = 0; w < kSharing; ++w) {
        const float weight = __builtin_amdgcn_exp2f(m[w] - base);
        l = fmaf(s_sum[at + w * kRows], weight, l);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          f[e] = fmaf(lo[w][e], weight, f[e]);
          f[e + 4] = fmaf(hi[w][e], weight, f[e + 4]);
        }
      }
      const uint32_t token = a.by_group.quotient(row0 + row);
      const int64_t vector = (unit.first + static_cast<int64_t>(token)) * a.q_heads + h * a.group + (row0 + row - token * a.group);
      if (a.splits > 1 && unit.split == 0 && d == 0) a.split_counts[vector] = unit.splits;
      if (unit.splits == 1) {
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] *= inv;
        store8(static_cast<T*>(a.out) + vector * D + d, f);
      } else {
        float* record = a.partials + (vector * a.splits + unit.split) * (D + kHeader);
        if (d == 0) *reinterpret_cast<v2f*>(record) = v2f{top, l};
        if (top != -INFINITY || l != 0.0f) store8(record + kHeader + d, f);   // (else nobody reads it)
      }
    }
  };
  if (sharing == 4) finish(std::integral_constant<int, 4>());
  else if (sharing == 2) finish(std::integral_constant<int, 2>());
  else finish(std::integral_constant<int, 1>());
}

// The partial results of a row and head, by WAVES waves: four columns of every kAtOnce-th of at most SPLITS a thread, all asked for
// at once. One wave a row where there are many rows, which then have few splits (most_splits); else a workgroup.
template <typename T, int D, int WAVES, int SPLITS>
__global__ __launch_bounds__(kThreads) void merge_kernel(const Problem a) {
  constexpr int kQuads = D / 4, kAtOnce = WAVES * kWave / kQuads, kEach = (SPLITS + kAtOnce - 1) / kAtOnce, kRecord = D + kHeader;
  __shared__ __attribute__((aligned(16))) float s_part[WAVES > 1 ? kAtOnce : 1][D];
  const int tid = threadIdx.x % (WAVES * kWave), lane = tid & (kWave - 1), quad = tid % kQuads, at = tid / kQuads;
  const int64_t vector = static_cast<int64_t>(blockIdx.x) * (kWaves / WAVES) + __builtin_amdgcn_readfirstlane(threadIdx.x / (WAVES * kWave));
  if (vector >= static_cast<int64_t>(a.rows.rows) * a.q_heads) return;
  if (a.rows.start != nullptr) {   // rows of no sequence have none
    const int row = static_cast<int>(vector / a.q_heads);
    if (row < a.rows.first(0) || row >= a.rows.first(a.rows.sequences)) return;
  }
  const int splits = min(a.split_counts[vector], a.splits);
  if (splits <= 1) return;   // (written by its only one)
  const float* record = a.partials + vector * a.splits * kRecord;
  v4f part[kEach];
#pragma unroll
  for (int i = 0; i < kEach; ++i)
    part[i] = at + i * kAtOnce < splits ? *reinterpret_cast<const v4f*>(record + (at + i * kAtOnce) * kRecord + kHeader + 4 * quad) : v4f{0.0f, 0.0f, 0.0f, 0.0f};
  const v2f mine = lane < splits ? *reinterpret_cast<const v2f*>(record + lane * kRecord) : v2f{-INFINITY, 0.0f};
  const float m = group_max<64>(mine[0]), base = m == -INFINITY ? 0.0f : m;
  const float weight = __builtin_amdgcn_exp2f(mine[0] - base);
  const float l = wave_sum(mine[1] * weight);
  v4f total = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const float w = __shfl(weight, (at + i * kAtOnce) & (kWave - 1), kWave);
    if (w != 0.0f) total += part[i] * w;   // (a split that saw nothing has written no columns)
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  if constexpr (WAVES == 1) {
#pragma unroll
    for (int step = kQuads; step < kWave; step *= 2)
#pragma unroll
      for (int e = 0; e < 4; ++e) total[e] += __shfl_xor(total[e], step, kWave);
    if (at != 0) return;
    T* out = static_cast<T*>(a.out) + vector * D + 4 * quad;
#pragma unroll
    for (int e = 0; e < 4; ++e) out[e] = from_float<T>(total[e] * inv);
  } else {
    *reinterpret_cast<v4f*>(&s_part[at][4 * quad]) = total;
    __syncthreads();
    if (tid >= D / 8) return;
    float f[8] = {};
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] += s_part[i][8 * tid + e];
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] *= inv;
    store8(static_cast<T*>(a.out) + vector * D + 8 * tid, f);
  }
}

// Row tiles of 16 that a wave takes: one where an average sequence has no more (its waves then share tokens), else two. The host does
// not know how the rows lie: one prompt of 200 rows, groups of 4, takes 13.3 us by itself (two), 11.0 among 96 places that have none (one),
// 700 rows 27.4, among 256 places 30.5.
int row_tiles(int64_t rows, int sequences, int group) {
  const int64_t average = rows * group / sequences;
  return average <= 16 ? 1 : 2;
}

// row groups of the batch (an upper bound)
int64_t row_groups(int64_t rows, int sequences, int group, int tiles) {
  return rows * group / (kWaves * 16 * tiles) + sequences;
}

// Partial results that a row can have, 1: none. By the table's width, the longest that a sequence can be, which the host knows; what
// is cached it does not: a row on 600 tokens of heads of 64 takes 6.1 us under a table of 640 tokens, 8.2 under one of 1024 to 4096 (a merge
// that finds nothing, a wave a row), 9.1 under 8192 and more (a workgroup a row). And by all rows of the call: a row on 131000 tokens takes 51 us by
// itself, but beside 1100 rows of 32 heads on nothing (43 us) 771, since it is not split.
int most_splits(int64_t vectors, int block, int table_width) {
  const int64_t tiles = (static_cast<int64_t>(table_width) * block + kTile - 1) / kTile;
  if (tiles < 2 * kLeastTiles) return 1;   // (a second launch costs more than half of so short a walk)
  return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({(tiles + kLeastTiles - 1) / kLeastTiles, kMostRecords / vectors, kMaxSplits})));
}
size_t counts_bytes(int64_t vectors) { return (static_cast<size_t>(vectors) * sizeof(int32_t) + 15) / 16 * 16; }

// Whether codes are read past the caches, by the bytes of the longest that the sequences can be (their table's width), against the
// 256 MB Infinity Cache; one row tile a wave. Measured under tables as wide as the longest sequence: 131000 tokens of eight heads of 128
// 51.8 -> 49.9 us, 400000 143 -> 133, two of 200000 together 78.5 -> 73.8; one of 65000, at the border, 30.6 -> 30.9. 48 ragged sequences, which
// hold about half of such a table, of 308 MB together 65.8 -> 64.0, 614 MB 115 -> 113, but 205 MB 46.8 -> 50.1, 102 MB 31.5 -> 34.2. Under a wider table
// the rule takes what is cached for more than it is: 48 sequences of 600 tokens (59 MB) 22.1 us under 4096 tokens each, 25.7 under 8192
// and more, eight of 1000 11.1 and 12.7 (under 32768); heads of 64, 48 of 600, 13.2 and 14.8. Heads of 64, whose requests are the
// smallest, gain earlier: 64 sequences of 154 MB 37.1 -> 34.2. Heads of 256 do not: 48 sequences of 307 MB 78.6 -> 85.0, 205 MB 61 -> 67.
// Two row tiles, which other waves may read again: 20.4 -> 22.9.
bool streams(const Problem& a, int D) {
  const double bytes = 2.0 * a.rows.sequences * a.table.width * (1 << a.block_shift) * a.heads * D;
  return D != 256 && bytes > (D == 64 ? 128e6 : std::min(128e6 * a.rows.sequences, 512e6));
}

template <typename T> int launch(const Problem& a, int D, int tiles, int64_t groups, hipStream_t s) {
  const dim3 grid(static_cast<unsigned>(groups * a.heads)), block(kThreads);
#define LLMQ_ATTEND(DIM)                                                                                           \
  do {                                                                                                             \
    if (tiles > 1) hipLaunchKernelGGL((attention_kernel<T, DIM, 2, false>), grid, block, 0, s, a);                  \
    else if (once) hipLaunchKernelGGL((attention_kernel<T, DIM, 1, (DIM < 256)>), grid, block, 0, s, a);            \
    else hipLaunchKernelGGL((attention_kernel<T, DIM, 1, false>), grid, block, 0, s, a);                            \
  } while (0)
  const bool once = streams(a, D);
  if (D == 64) LLMQ_ATTEND(64);
  else if (D == 128) LLMQ_ATTEND(128);
  else LLMQ_ATTEND(256);
#undef LLMQ_ATTEND
  if (int rc = llmq_host::check_launch("attention_kernel")) return rc;
  if (a.splits == 1) return 0;
  const bool few = a.splits <= kFewSplits;
  const int64_t vectors = static_cast<int64_t>(a.rows.rows) * a.q_heads;
  const dim3 merge_grid(static_cast<unsigned>(few ? (vectors + kWaves - 1) / kWaves : vectors));
#define LLMQ_MERGE(DIM)                                                                                          \
  do {                                                                                                           \
    if (few) hipLaunchKernelGGL((merge_kernel<T, DIM, 1, kFewSplits>), merge_grid, block, 0, s, a);              \
    else hipLaunchKernelGGL((merge_kernel<T, DIM, kWaves, kMaxSplits>), merge_grid, block, 0, s, a);             \
  } while (0)
  if (D == 64) LLMQ_MERGE(64);
  else if (D == 128) LLMQ_MERGE(128);
  else LLMQ_MERGE(256);
#undef LLMQ_MERGE
  return llmq_host::check_launch("merge_kernel");
}

}  // namespace

extern "C" size_t llmq_kv_block_attention_workspace_bytes(int tokens, int sequences, int q_heads, int kv_heads, int head_dim,
                                                          int block, int table_width) {
  if (tokens <= 0 || sequences <= 0 || q_heads <= 0 || kv_heads <= 0 || head_dim <= 0 || block <= 0 || table_width <= 0) return 0;
  const int64_t vectors = static_cast<int64_t>(tokens) * q_heads;
  const int splits = most_splits(vectors, block, table_width);
  return splits == 1 ? 0 : counts_bytes(vectors) + sizeof(float) * static_cast<size_t>(vectors) * splits * (head_dim + kHeader);
}

extern "C" int llmq_kv_block_attention(const void* query, int64_t q_row_stride, const void* k_codes, const void* v_codes,
                                       const float* k_scale, const float* v_scale, const int32_t* block_table,
                                       int64_t table_stride, const int32_t* cached, const int32_t* query_start_or_null, void* out,
                                       void* workspace, size_t workspace_bytes, float sm_scale, int tokens, int sequences,
                                       int q_heads, int kv_heads, int head_dim, int block, int n_blocks, int table_width,
                                       int dtype, llmq_stream_t stream) {
  if (int rc = llmq_host::check_block_shape(tokens, sequences, kv_heads, head_dim, block, n_blocks, table_width, table_stride, dtype)) return rc;
  if (q_heads <= 0 || q_heads % kv_heads != 0) return llmq_host::fail_invalid("q_heads %d is not a multiple of kv_heads %d", q_heads, kv_heads);
  const float scale_log2e = sm_scale * 1.4426950408889634f;
  if (!std::isfinite(scale_log2e)) return llmq_host::fail_invalid("sm_scale must be finite, times log2 e too");
  if (!query_start_or_null && tokens != sequences)
    return llmq_host::fail_invalid("without query_start a sequence has one row: %d rows, %d sequences", tokens, sequences);
  const int v = dtype == LLMQ_F32 ? 4 : 8;
  if (q_row_stride % v) return llmq_host::fail_invalid("row strides must be multiples of %d elements", v);
  if (tokens == 0 || sequences == 0) return 0;
  if (n_blocks == 0) table_width = 0;   // no token has a block
  const int group = q_heads / kv_heads, tiles = row_tiles(tokens, sequences, group);
  // (row numbers, and the launch's workgroups, are counted in 32 bits)
  const int64_t vectors = static_cast<int64_t>(tokens) * q_heads;
  const int splits = most_splits(vectors, block, table_width);
  const int64_t groups = splits > 1            ? row_groups(tokens, sequences, group, tiles) + (kUnits + kv_heads - 1) / kv_heads
                         : query_start_or_null ? row_groups(tokens, sequences, group, tiles)
                                               : static_cast<int64_t>(sequences) * ((group + kWaves * 16 * tiles - 1) / (kWaves * 16 * tiles));
  if (vectors > INT32_MAX / 2 || groups * kv_heads > INT32_MAX)
    return llmq_host::fail_invalid("too many rows and heads for one launch: %d, %d", tokens, q_heads);
  if (!query || !cached || !out || (table_width != 0 && (!k_codes || !v_codes || !k_scale || !v_scale || !block_table)))
    return llmq_host::fail_invalid("null tensor pointer");
  const size_t need = llmq_kv_block_attention_workspace_bytes(tokens, sequences, q_heads, kv_heads, head_dim, block, table_width);
  if (workspace_bytes < need || (need && !workspace))
    return llmq_host::fail_invalid("the workspace has %zu bytes, llmq_kv_block_attention_workspace_bytes() asks for %zu", workspace_bytes, need);
  uintptr_t all = 0;
  for (const void* t : {query, k_codes, v_codes, static_cast<const void*>(out), static_cast<const void*>(workspace)})
    all |= reinterpret_cast<uintptr_t>(t);
  if (all & 15u) return llmq_host::fail_invalid("query, codes, out and workspace must be 16-byte aligned");
  int shift = 4;
  while ((1 << shift) < block) ++shift;
  const Problem a{query, q_row_stride, static_cast<const int8_t*>(k_codes), static_cast<const int8_t*>(v_codes), k_scale, v_scale,
                  {block_table, table_stride, table_width, n_blocks}, cached, {query_start_or_null, sequences, tokens}, out,
                  static_cast<int32_t*>(workspace),
                  workspace ? reinterpret_cast<float*>(static_cast<char*>(workspace) + counts_bytes(vectors)) : nullptr, splits, q_heads, kv_heads, group, shift, scale_log2e,
                  {static_cast<uint32_t>(group), static_cast<uint32_t>(((uint64_t{1} << 32) + group - 1) / group)}};
  hipStream_t s = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case LLMQ_F32: return launch<float>(a, head_dim, tiles, groups, s);
    case LLMQ_F16: return launch<f16_t>(a, head_dim, tiles, groups, s);
    default: return launch<bf16_t>(a, head_dim, tiles, groups, s);
  }
}
