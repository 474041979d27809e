// Writing a cache in blocks (layout: kv_blocks.h), quantized, and reading it back, gfx950.
//
//   append   a = max |x| over the call's tokens in a block, for each head
//            s = max(a (1 / 127), 1e-8) where the call writes the block's first token, else max(s_old, that);
//                not a number where an x is not finite, so that c s is not a number for any token of the block
//            codes of the call's tokens: clamp(rint(x / s)); of the block's earlier tokens: clamp(rint((c s_old) / s))
//   dequant  T(c s)
//
// A lane takes eight columns of eight tokens: a packet of 16-bit values for each token, eight bytes of each token's key codes,
// eight bytes of each column's value codes (16 tokens innermost), so that the transposition of the values is a choice of bytes within a
// lane. Bound: HBM, each tensor read once and written once (40000 tokens
// of eight heads of 128 read back, bf16: 46.6 us by trace, 5.3 TB/s); at few tokens the chain starts and lengths -> table -> scales and
// codes, a trip to memory each (600 tokens read 4.6 us, a step of 64 rows written 4.7), and for prompts the length of append's
// program besides, which few waves run (6011 tokens of eight heads of 64: 9.6).
#include "kv_blocks.h"

namespace {

using namespace llmq;

constexpr int kColumns = 8;   // of a lane's strip

template <typename T> __device__ __forceinline__ void load8(const T* p, float* f) {
#pragma unroll
  for (int i = 0; i < kColumns; i += Pack<T>::N) Pack<T>::unpack(load16(p + i), f + i);
}
template <typename T> __device__ __forceinline__ void store8(T* p, const float* f) {
#pragma unroll
  for (int i = 0; i < kColumns; i += Pack<T>::N) store16(p + i, Pack<T>::pack(f + i));
}
__device__ __forceinline__ float code_of(uint32_t word, int byte) { return static_cast<float>(static_cast<int8_t>(word >> (8 * byte))); }
// A divisor with its correctly rounded reciprocal: the quotient to the last bit in five instructions. x inv is within an ulp and a half,
// one correction by its remainder (a multiply-add, exact but for the last rounding) leaves it within an ulp, and a second
// one is then the rounded quotient (Markstein's theorem). The compiler's division is a dozen instructions and more, in a hundred places.
struct Scale {
  float by, inv;
  explicit __device__ __forceinline__ Scale(float s) : by(s), inv(1.0f / s) {}
  __device__ __forceinline__ float quotient(float x) const {
    float r = x * inv;
    r = fmaf(fmaf(-r, by, x), inv, r);
    return fmaf(fmaf(-r, by, x), inv, r);
  }
};
// rint(x / s), clamped, for eight values
__device__ __forceinline__ void codes_of8(float* f, const Scale& s) {
#pragma unroll
  for (int e = 0; e < kColumns; ++e) f[e] = fminf(fmaxf(rintf(s.quotient(f[e])), -128.0f), 127.0f);
}
__device__ __forceinline__ uint32_t byte_of(float code, int byte) { return (static_cast<uint32_t>(static_cast<int>(code)) & 0xffu) << (8 * byte); }

__device__ __forceinline__ u32x2 bytes_of(const float* f) {
  return u32x2{byte_of(f[0], 0) | byte_of(f[1], 1) | byte_of(f[2], 2) | byte_of(f[3], 3),
               byte_of(f[4], 0) | byte_of(f[5], 1) | byte_of(f[6], 2) | byte_of(f[7], 3)};
}
// The largest magnitude of a head, where what is not a number counts as above infinity. Lanes gather it with the instruction that keeps
// what is not a number (fmaxf passes over it). Over each aligned group of WIDTH lanes, 16, 32 or 64: as bits of magnitudes, which have this order.
template <int WIDTH> __device__ __forceinline__ int largest_bits(float magnitude) {
  static_assert(WIDTH == 16 || WIDTH == 32 || WIDTH == kWave, "a head's lanes");
  int v = __builtin_bit_cast(int, magnitude) & 0x7fffffff;
  v = max(v, dpp<kDppXor1>(v));
  v = max(v, dpp<kDppXor2>(v));
  v = max(v, dpp<kDppHalfMirror>(v));
  v = max(v, dpp<kDppMirror>(v));
  if constexpr (WIDTH == 16) return v;
  const int lo = max(__builtin_amdgcn_readlane(v, 0), __builtin_amdgcn_readlane(v, 16)),
            hi = max(__builtin_amdgcn_readlane(v, 32), __builtin_amdgcn_readlane(v, 48));
  if constexpr (WIDTH == 32) return (threadIdx.x & 32) ? hi : lo;
  return max(lo, hi);
}
// eight codes brought to another scale
__device__ __forceinline__ u32x2 moved8(u32x2 w, float before, const Scale& s) {
  float f[kColumns];
#pragma unroll
  for (int e = 0; e < kColumns; ++e) f[e] = code_of(e < 4 ? w.x : w.y, e % 4) * before;
  codes_of8(f, s);
  return bytes_of(f);
}

// The tokens of the call that lie in one block of a sequence.
struct Touched {
  int entry;       // of the block table, as it is; -1 beyond it
  int lo, hi;      // the block's slots lo .. hi - 1
  int64_t row;     // the row of slot lo
};
// `from`: the position of the sequence's first row; piece: which of the blocks from there on. False: no row in that block.
__device__ __forceinline__ bool touched_block(const BlockTable& table, int b, const Span& rows, int64_t from, int piece, int block_shift,
                                              Touched& t) {
  const int64_t logical = (from >> block_shift) + piece, at = logical << block_shift;
  if (rows.n == 0 || at > from + rows.n - 1) return false;
  t.entry = logical < table.width ? table.entries[b * table.row_stride + logical] : -1;
  t.lo = static_cast<int>(max(from - at, static_cast<int64_t>(0)));
  t.hi = static_cast<int>(min(from + rows.n - at, static_cast<int64_t>(1) << block_shift));
  t.row = rows.first + (at + t.lo - from);
  return true;
}

constexpr int kTokens = 8;   // of a lane of append

// A head's lanes: (BLOCK / 8) (D / 8); a workgroup has as many whole heads as 64 lanes hold, or one.
template <int D, int BLOCK> struct AppendShape {
  static constexpr int kLanes = BLOCK / kTokens * (D / kColumns);
  static constexpr int kThreads = kLanes > kWave ? kLanes : kWave, kHeads = kThreads / kLanes;
};

template <typename T, int D, int BLOCK>
__global__ __launch_bounds__((AppendShape<D, BLOCK>::kThreads)) void append_kernel(
    const T* __restrict__ key, const T* __restrict__ value, const int64_t key_stride, const int64_t value_stride,
    int8_t* __restrict__ k_codes, int8_t* __restrict__ v_codes, float* __restrict__ k_scale, float* __restrict__ v_scale,
    const BlockTable table, const int32_t* __restrict__ cached, const Ragged rows, const int heads) {
  using Shape = AppendShape<D, BLOCK>;
  constexpr int kShift = BLOCK == 16 ? 4 : BLOCK == 32 ? 5 : BLOCK == 64 ? 6 : 7;
  __shared__ int s_max[Shape::kThreads / kWave];
  const int sets = (heads + Shape::kHeads - 1) / Shape::kHeads;   // of heads
  const bool is_value = blockIdx.x & 1;
  const int set = static_cast<int>(blockIdx.x / 2) % sets;
  int piece = blockIdx.x / 2 / sets, b = piece, from = 0;
  Span span{b, 1};
  if (rows.start == nullptr) {
    from = cached[b];
    piece = 0;
  } else {
    b = rows.find(kShift, cached, piece, span, from);
  }
  Touched here;
  if (from < 0 || !touched_block(table, b, span, from, piece, kShift, here)) return;
  const int h = set * Shape::kHeads + static_cast<int>(threadIdx.x) / Shape::kLanes, in_head = threadIdx.x % Shape::kLanes;
  const int slot0 = in_head / (D / kColumns) * kTokens, d = in_head % (D / kColumns) * kColumns;
  const bool active = h < heads;   // (the others stay for the barrier)
  // the lane's tokens of the call: lo .. hi - 1 of its eight; the block's earlier ones: below lo
  const int lo = min(max(here.lo - slot0, 0), kTokens), hi = active ? min(max(here.hi - slot0, 0), kTokens) : 0;
  const int64_t stride = is_value ? value_stride : key_stride;
  const T* x = (is_value ? value : key) + here.row * stride + static_cast<int64_t>(min(h, heads - 1)) * D + d;
  constexpr int kPackets = kColumns / Pack<T>::N;
  u32x4 raw[kTokens][kPackets];
#pragma unroll
  for (int i = 0; i < kTokens; ++i) {   // (a slot without a row of the call reads the nearest one that has: no branch around a load)
    const int64_t at = min(max(slot0 + i, here.lo), here.hi - 1) - here.lo;
#pragma unroll
    for (int e = 0; e < kPackets; ++e) raw[i][e] = load16(x + at * stride + e * Pack<T>::N);
  }
  // (the rows are asked for beside the block, whose scale is a trip to memory behind the table's)
  if (here.entry < 0 || here.entry >= table.blocks) return;   // (the workgroup's: one block)
  const int64_t unit = static_cast<int64_t>(here.entry) * heads + min(h, heads - 1);
  float* scale = (is_value ? v_scale : k_scale) + unit;
  const float before = *scale;
  float largest = 0.0f;
#pragma unroll
  for (int i = 0; i < kTokens; ++i) {
    float f[kColumns];
#pragma unroll
    for (int e = 0; e < kPackets; ++e) Pack<T>::unpack(raw[i][e], f + e * Pack<T>::N);
#pragma unroll
    for (int e = 0; e < kColumns; ++e) largest = __builtin_elementwise_maximum(largest, fabsf(f[e]));   // (rows that are read twice change no maximum)
  }
  int bits = largest_bits<(Shape::kLanes < kWave ? Shape::kLanes : kWave)>(largest);
  if constexpr (Shape::kThreads > kWave) {
    if (threadIdx.x % kWave == 0) s_max[threadIdx.x / kWave] = bits;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < Shape::kThreads / kWave; ++w) bits = max(bits, s_max[w]);
  }
  if (!active) return;
  const float amax = __builtin_bit_cast(float, bits);
  float s = fmaxf(amax * (1.0f / 127.0f), kScaleEps);
  if (here.lo > 0) s = fmaxf(s, before);
  if (!(amax < INFINITY) || (here.lo > 0 && before != before)) s = NAN;
  const bool grown = here.lo > 0 && s > before && lo > 0;   // and this lane has earlier tokens
  if (in_head == 0) *scale = s;
  if (hi <= lo && !grown) return;   // nothing of this lane's changes

  const Scale by(s);
  const auto codes_of = [&](int i) {   // the eight codes of token i
    float f[kColumns];
#pragma unroll
    for (int e = 0; e < kPackets; ++e) Pack<T>::unpack(raw[i][e], f + e * Pack<T>::N);
    codes_of8(f, by);
    return bytes_of(f);
  };
  if (!is_value) {
    int8_t* codes = k_codes + (unit * BLOCK + slot0) * D + d;
#pragma unroll
    for (int i = 0; i < kTokens; ++i)
      if (i >= lo && i < hi) *reinterpret_cast<u32x2*>(codes + i * D) = codes_of(i);
    if (grown) {
#pragma unroll 1   // (rare: short code, since a launch reads it from memory before it runs)
      for (int i = 0; i < lo; ++i) {
        u32x2* at = reinterpret_cast<u32x2*>(codes + i * D);
        *at = moved8(*at, before, by);
      }
    }
    return;
  }
  int8_t* codes = v_codes + ((unit * (BLOCK / kStrip) + slot0 / kStrip) * D + d) * kStrip + slot0 % kStrip;
  if (hi - lo == 1 && !grown) {   // a token: its bytes alone (a step's; nothing is read)
#pragma unroll
    for (int i = 0; i < kTokens; ++i)
      if (i == lo) {
        const u32x2 c = codes_of(i);
#pragma unroll
        for (int e = 0; e < kColumns; ++e) codes[e * kStrip + i] = static_cast<int8_t>((e < 4 ? c.x : c.y) >> (8 * (e % 4)));
      }
    return;
  }
  if (grown) {   // the columns' earlier tokens first, the others as they are
    uint32_t old[2] = {};
#pragma unroll
    for (int i = 0; i < kTokens; ++i) old[i / 4] |= i < lo ? 0xffu << (8 * (i % 4)) : 0u;
#pragma unroll 1
    for (int e = 0; e < kColumns; ++e) {
      u32x2* at = reinterpret_cast<u32x2*>(codes + e * kStrip);
      const u32x2 held = *at, m = moved8(held, before, by);
      *at = u32x2{(held.x & ~old[0]) | (m.x & old[0]), (held.y & ~old[1]) | (m.y & old[1])};
    }
    if (hi <= lo) return;
  }
  // columns of eight tokens, out of tokens of eight columns
  u32x2 tokens[kTokens];
#pragma unroll
  for (int i = 0; i < kTokens; ++i) tokens[i] = codes_of(i);
  // bytes of other tokens among them stay
  uint32_t fresh[2] = {};
#pragma unroll
  for (int i = 0; i < kTokens; ++i) fresh[i / 4] |= i >= lo && i < hi ? 0xffu << (8 * (i % 4)) : 0u;
#pragma unroll
  for (int e = 0; e < kColumns; ++e) {
    u32x2 column{0u, 0u};
#pragma unroll
    for (int i = 0; i < kTokens; ++i) {
      const uint32_t code = ((e < 4 ? tokens[i].x : tokens[i].y) >> (8 * (e % 4)) & 0xffu) << (8 * (i % 4));
      (i < 4 ? column.x : column.y) |= code;
    }
    u32x2* at = reinterpret_cast<u32x2*>(codes + e * kStrip);
    if (lo > 0 || hi < kTokens) {
      const u32x2 held = *at;
      column = u32x2{(held.x & ~fresh[0]) | (column.x & fresh[0]), (held.y & ~fresh[1]) | (column.y & fresh[1])};
    }
    *at = column;
  }
}

constexpr int kDequantThreads = 256;

// The lanes of a block: eight tokens each of all its heads, keys and values in workgroups of their own.
template <typename T, int D>
__global__ __launch_bounds__(kDequantThreads) void dequant_kernel(
    const int8_t* __restrict__ k_codes, const int8_t* __restrict__ v_codes, const float* __restrict__ k_scale,
    const float* __restrict__ v_scale, const BlockTable table, const Ragged rows, const int32_t* __restrict__ first_or_null,
    T* __restrict__ k_out, T* __restrict__ v_out, const int heads, const int block_shift) {
  const int strips = 1 << (block_shift - 4), lanes = heads * strips * (kStrip / kTokens) * (D / kColumns), sets = (lanes + kDequantThreads - 1) / kDequantThreads;
  const bool is_value = blockIdx.x & 1;
  const int set = static_cast<int>(blockIdx.x / 2) % sets;
  int piece = blockIdx.x / 2 / sets, from = 0;
  Span span{0, 0};
  const int b = rows.find(block_shift, first_or_null, piece, span, from);
  Touched here;
  if (!touched_block(table, b, span, max(from, 0), piece, block_shift, here)) return;
  const int item = set * kDequantThreads + static_cast<int>(threadIdx.x);
  if (item >= lanes) return;
  const int groups = strips * (kStrip / kTokens);   // of eight tokens
  const int d = item % (D / kColumns) * kColumns, slot0 = item / (D / kColumns) % groups * kTokens, h = item / (D / kColumns) / groups;
  const int lo = max(here.lo - slot0, 0), hi = min(here.hi - slot0, kTokens);
  if (hi <= lo) return;
  const bool held = here.entry >= 0 && here.entry < table.blocks;
  const int64_t unit = static_cast<int64_t>(held ? here.entry : 0) * heads + h;
  T* out = (is_value ? v_out : k_out) + (static_cast<int64_t>(h) * rows.rows + here.row + slot0 - here.lo) * D + d;
  u32x2 words[kTokens] = {};   // keys: a token's eight codes; values: a column's eight
  float s = 0.0f;
  if (held) {
    s = (is_value ? v_scale : k_scale)[unit];
    const int8_t* codes = is_value ? v_codes + ((unit * strips + slot0 / kStrip) * D + d) * kStrip + slot0 % kStrip
                                   : k_codes + ((unit << block_shift) + slot0) * D + d;
    const int step = is_value ? kStrip : D;
#pragma unroll
    for (int i = 0; i < kTokens; ++i) words[i] = *reinterpret_cast<const u32x2*>(codes + i * step);
  }
#pragma unroll
  for (int i = 0; i < kTokens; ++i) {
    if (i < lo || i >= hi) continue;
    float f[kColumns];
#pragma unroll
    for (int e = 0; e < kColumns; ++e) {
      const uint32_t of_key = e < 4 ? words[i].x : words[i].y, of_value = i < 4 ? words[e].x : words[e].y;
      f[e] = (is_value ? code_of(of_value, i % 4) : code_of(of_key, e % 4)) * s;
    }
    T* to = out + static_cast<int64_t>(i) * D;
    store8(to, f);
  }
}

int check_cache(const void* k_codes, const void* v_codes, const void* k_scale, const void* v_scale, const void* block_table) {
  if (!k_codes || !v_codes || !k_scale || !v_scale || !block_table) return llmq_host::fail_invalid("null tensor pointer");
  if ((reinterpret_cast<uintptr_t>(k_codes) | reinterpret_cast<uintptr_t>(v_codes)) & 15u)
    return llmq_host::fail_invalid("the codes must be 16-byte aligned");
  return 0;
}

// pieces of a ragged batch (Ragged::find): an upper bound of the blocks that its rows touch
int64_t pieces(int rows, int sequences, int block) { return rows / block + 2LL * sequences; }

}  // namespace

int llmq_host::check_block_shape(int rows, int sequences, int kv_heads, int head_dim, int block, int blocks, int table_width,
                                 int64_t table_stride, int dtype) {
  if (rows < 0 || sequences < 0 || kv_heads <= 0 || blocks < 0 || table_width < 0)
    return llmq_host::fail_invalid("bad dimension rows=%d sequences=%d kv_heads=%d blocks=%d table_width=%d", rows, sequences, kv_heads, blocks, table_width);
  if (head_dim != 64 && head_dim != 128 && head_dim != 256) return llmq_host::fail_invalid("head_dim must be 64, 128 or 256, got %d", head_dim);
  if (block != 16 && block != 32 && block != 64 && block != 128) return llmq_host::fail_invalid("block must be 16, 32, 64 or 128 tokens, got %d", block);
  if (dtype != LLMQ_F32 && dtype != LLMQ_F16 && dtype != LLMQ_BF16)
    return llmq_host::fail_invalid("dtype code %d is not float32, float16 or bfloat16", dtype);
  if (table_stride < 0) return llmq_host::fail_invalid("negative stride of the block table");
  if ((rows / 16 + 2LL * sequences) * 2 * kv_heads > INT32_MAX)
    return llmq_host::fail_invalid("too many rows, sequences and heads for one launch: %d, %d, %d", rows, sequences, kv_heads);
  return 0;
}

extern "C" int llmq_kv_block_append(const void* key, const void* value, int64_t key_row_stride, int64_t value_row_stride,
                                    void* k_codes, void* v_codes, float* k_scale, float* v_scale, const int32_t* block_table,
                                    int64_t table_stride, const int32_t* cached, const int32_t* query_start_or_null, int tokens,
                                    int sequences, int kv_heads, int head_dim, int block, int n_blocks, int table_width,
                                    int dtype, llmq_stream_t stream) {
  if (int rc = llmq_host::check_block_shape(tokens, sequences, kv_heads, head_dim, block, n_blocks, table_width, table_stride, dtype)) return rc;
  if (!query_start_or_null && tokens != sequences)
    return llmq_host::fail_invalid("without query_start a sequence has one row: %d rows, %d sequences", tokens, sequences);
  const int v = dtype == LLMQ_F32 ? 4 : 8;
  if (key_row_stride % v || value_row_stride % v) return llmq_host::fail_invalid("row strides must be multiples of %d elements", v);
  if (tokens == 0 || sequences == 0 || n_blocks == 0 || table_width == 0) return 0;
  if (!key || !value || !cached) return llmq_host::fail_invalid("null tensor pointer");
  if (int rc = check_cache(k_codes, v_codes, k_scale, v_scale, block_table)) return rc;
  if ((reinterpret_cast<uintptr_t>(key) | reinterpret_cast<uintptr_t>(value)) & 15u)
    return llmq_host::fail_invalid("key and value must be 16-byte aligned");
  const BlockTable table{block_table, table_stride, table_width, n_blocks};
  const Ragged rows{query_start_or_null, sequences, tokens};
  const int64_t n_pieces = query_start_or_null ? pieces(tokens, sequences, block) : sequences;
  hipStream_t s = static_cast<hipStream_t>(stream);
#define LLMQ_APPEND(T, D, BLOCK)                                                                                             \
  hipLaunchKernelGGL((append_kernel<T, D, BLOCK>),                                                                           \
                     dim3(static_cast<unsigned>(n_pieces * 2 * ((kv_heads + AppendShape<D, BLOCK>::kHeads - 1) / AppendShape<D, BLOCK>::kHeads))), \
                     dim3(AppendShape<D, BLOCK>::kThreads), 0, s, static_cast<const T*>(key), static_cast<const T*>(value),  \
                     key_row_stride, value_row_stride, static_cast<int8_t*>(k_codes), static_cast<int8_t*>(v_codes),         \
                     k_scale, v_scale, table, cached, rows, kv_heads)
#define LLMQ_APPEND_D(T, D)                        \
  switch (block) {                                 \
    case 16: LLMQ_APPEND(T, D, 16); break;         \
    case 32: LLMQ_APPEND(T, D, 32); break;         \
    case 64: LLMQ_APPEND(T, D, 64); break;         \
    default: LLMQ_APPEND(T, D, 128); break;        \
  }
#define LLMQ_APPEND_T(T)                           \
  switch (head_dim) {                              \
    case 64: LLMQ_APPEND_D(T, 64); break;          \
    case 128: LLMQ_APPEND_D(T, 128); break;        \
    default: LLMQ_APPEND_D(T, 256); break;         \
  }
  switch (dtype) {
    case LLMQ_F32: LLMQ_APPEND_T(float); break;
    case LLMQ_F16: LLMQ_APPEND_T(f16_t); break;
    default: LLMQ_APPEND_T(bf16_t); break;
  }
#undef LLMQ_APPEND_T
#undef LLMQ_APPEND_D
#undef LLMQ_APPEND
  return llmq_host::check_launch("append_kernel");
}

extern "C" int llmq_kv_block_dequant(const void* k_codes, const void* v_codes, const float* k_scale, const float* v_scale,
                                     const int32_t* block_table, int64_t table_stride, const int32_t* starts,
                                     const int32_t* first_or_null, void* k_out, void* v_out, int n_tokens, int sequences,
                                     int kv_heads, int head_dim, int block, int n_blocks, int table_width, int dtype,
                                     llmq_stream_t stream) {
  if (int rc = llmq_host::check_block_shape(n_tokens, sequences, kv_heads, head_dim, block, n_blocks, table_width, table_stride, dtype)) return rc;
  if (n_tokens == 0 || sequences == 0) return 0;
  if (!starts || !k_out || !v_out) return llmq_host::fail_invalid("null tensor pointer");
  if (n_blocks != 0 && table_width != 0)   // (tensors of no elements have no address)
    if (int rc = check_cache(k_codes, v_codes, k_scale, v_scale, block_table)) return rc;
  if ((reinterpret_cast<uintptr_t>(k_out) | reinterpret_cast<uintptr_t>(v_out)) & 15u)
    return llmq_host::fail_invalid("the outputs must be 16-byte aligned");
  const BlockTable table{block_table, table_stride, table_width, n_blocks};
  const Ragged rows{starts, sequences, n_tokens};
  int shift = 4;
  while ((1 << shift) < block) ++shift;
  const int64_t lanes = static_cast<int64_t>(kv_heads) * (block / kTokens) * (head_dim / kColumns);
  const int64_t workgroups = pieces(n_tokens, sequences, block) * 2 * ((lanes + kDequantThreads - 1) / kDequantThreads);
  if (lanes > INT32_MAX - kDequantThreads || workgroups > INT32_MAX)
    return llmq_host::fail_invalid("too many rows, sequences and heads for one launch: %d, %d, %d", n_tokens, sequences, kv_heads);
  // (the output through the caches: past them 40000 tokens of eight heads of 128 alone take 38 us instead of 56, but with an operator that
  // reads it behind 94 instead of 84, 20000 tokens 53 instead of 48; not measured for outputs above 164 MB)
  const dim3 grid(static_cast<unsigned>(workgroups));
  hipStream_t s = static_cast<hipStream_t>(stream);
#define LLMQ_DEQUANT(T, D)                                                                                               \
  hipLaunchKernelGGL((dequant_kernel<T, D>), grid, dim3(kDequantThreads), 0, s, static_cast<const int8_t*>(k_codes),     \
                     static_cast<const int8_t*>(v_codes), k_scale, v_scale, table, rows, first_or_null,                  \
                     static_cast<T*>(k_out), static_cast<T*>(v_out), kv_heads, shift)
#define LLMQ_DEQUANT_T(T)                       \
  switch (head_dim) {                           \
    case 64: LLMQ_DEQUANT(T, 64); break;        \
    case 128: LLMQ_DEQUANT(T, 128); break;      \
    default: LLMQ_DEQUANT(T, 256); break;       \
  }
  switch (dtype) {
    case LLMQ_F32: LLMQ_DEQUANT_T(float); break;
    case LLMQ_F16: LLMQ_DEQUANT_T(f16_t); break;
    default: LLMQ_DEQUANT_T(bf16_t); break;
  }
#undef LLMQ_DEQUANT_T
#undef LLMQ_DEQUANT
  return llmq_host::check_launch("dequant_kernel");
}
