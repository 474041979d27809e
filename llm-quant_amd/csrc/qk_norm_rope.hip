// The norm of every query and key head and the position rotation behind it, in one pass, gfx950:
//
//   y = x rsqrt(mean(x^2) + eps) w                                  over a head of D elements
//   z_i = y_i cos_i - y_(i + R/2) sin_i,   z_(i + R/2) = y_(i + R/2) cos_(i + R/2) + y_i sin_(i + R/2)   for i < R/2
//   z_i = y_i                                                       for i >= R
//
// in fp32, rounded once, where it is stored. cos and sin are row positions[t] of the tables (row t without positions).
//
// Bound: HBM, each element read and written once; for a few tokens one trip to memory and the launch. By trace, heads of 128: 4100
// tokens of 40 heads, bf16 17.9 us (4.9 TB/s; back to back 17.2), 77 tokens of 32 heads 4.0, one token 2.8.
#include <cmath>

#include "llmq_device.h"

namespace {

using namespace llmq;

constexpr int kThreads = 256;
constexpr int kPasses = 4;   // heads of a lane, where there are many

// Sum over each aligned group of WIDTH lanes (a power of two up to 32), in every lane of it.
template <int WIDTH> __device__ __forceinline__ float group_sum(float v) {
  if constexpr (WIDTH >= 2) v += dpp<kDppXor1>(v);
  if constexpr (WIDTH >= 4) v += dpp<kDppXor2>(v);
  if constexpr (WIDTH >= 8) v += dpp<kDppHalfMirror>(v);
  if constexpr (WIDTH >= 16) v += dpp<kDppMirror>(v);
  if constexpr (WIDTH == 32) {
    const float lo = lane_value(v, 0) + lane_value(v, 16), hi = lane_value(v, 32) + lane_value(v, 48);
    v = (threadIdx.x & 32) ? hi : lo;
  }
  return v;
}

// V values of a table whose elements are T or float
template <typename T, int V> __device__ __forceinline__ void load_table(const T* p, float* f) {
#pragma unroll
  for (int i = 0; i < V; i += Pack<T>::N) Pack<T>::unpack(load16(p + i), f + i);
}

// LANES lanes a head (a power of two), each with two packets: the pair that is rotated with each other, or two of the
// elements behind the rotated ones. A lane takes PASSES heads of a token, `step` apart, with one reading of its cosines, sines
// and weights: in fp32 tables those are eight times a head's own bytes.
template <typename T, typename TABLE, int LANES, int PASSES>
__global__ __launch_bounds__(kThreads) void qk_norm_rope_kernel(
    const T* __restrict__ q, const T* __restrict__ k, const int64_t q_stride, const int64_t k_stride,
    const T* __restrict__ q_weight, const T* __restrict__ k_weight, const TABLE* __restrict__ cos_table,
    const TABLE* __restrict__ sin_table, const void* __restrict__ positions, const bool wide_positions,
    T* __restrict__ q_out, T* __restrict__ k_out, const uint32_t vectors, const uint32_t q_heads, const uint32_t kv_heads,
    const uint32_t step, const int D, const int R, const int table_rows, const float eps) {
  constexpr int V = Pack<T>::N;
  const uint32_t item = blockIdx.x * kThreads + threadIdx.x, vector = item / LANES;   // (below 2^31: the host's rule)
  if (vector >= vectors) return;   // a head's lanes leave together
  const int p = static_cast<int>(item % LANES), pairs = R / 2 / V;
  const uint32_t t = vector / step, h0 = vector % step;
  const bool active = p < D / 2 / V, rotated = p < pairs;
  const int at0 = rotated ? p * V : R + (p - pairs) * 2 * V, at1 = rotated ? at0 + R / 2 : at0 + V;
  const int64_t position = positions == nullptr ? t
                           : wide_positions     ? static_cast<const int64_t*>(positions)[t]
                                                : static_cast<const int32_t*>(positions)[t];
  const bool known = position >= 0 && position < table_rows;

  u32x4 raw[PASSES][2];
#pragma unroll
  for (int i = 0; i < PASSES; ++i) {
    const uint32_t h = h0 + i * step;
    raw[i][0] = raw[i][1] = u32x4{0u, 0u, 0u, 0u};
    if (h < q_heads + kv_heads && active) {
      const T* x = h >= q_heads ? k + t * k_stride + static_cast<int64_t>(h - q_heads) * D : q + t * q_stride + static_cast<int64_t>(h) * D;
      raw[i][0] = load16(x + at0);
      raw[i][1] = load16(x + at1);
    }
  }
  u32x4 weights[2][2] = {};
  float c0[V], c1[V], s0[V] = {}, s1[V] = {};
#pragma unroll
  for (int e = 0; e < V; ++e) c0[e] = c1[e] = 1.0f;
  if (active) {
    if (h0 < q_heads) {
      weights[0][0] = load16(q_weight + at0);
      weights[0][1] = load16(q_weight + at1);
    }
    if (h0 + (PASSES - 1) * step >= q_heads) {
      weights[1][0] = load16(k_weight + at0);
      weights[1][1] = load16(k_weight + at1);
    }
    if (rotated && known) {   // (tables of no rows have nothing to read)
      const int64_t row = position * R;
      load_table<TABLE, V>(cos_table + row + at0, c0);
      load_table<TABLE, V>(cos_table + row + at1, c1);
      load_table<TABLE, V>(sin_table + row + at0, s0);
      load_table<TABLE, V>(sin_table + row + at1, s1);
    }
  }
#pragma unroll
  for (int i = 0; i < PASSES; ++i) {
    const uint32_t h = h0 + i * step;
    float a[V], b[V], squares = 0.0f;
    Pack<T>::unpack(raw[i][0], a);
    Pack<T>::unpack(raw[i][1], b);
#pragma unroll
    for (int e = 0; e < V; ++e) squares = fmaf(a[e], a[e], fmaf(b[e], b[e], squares));
    squares = group_sum<LANES>(squares);
    if (h >= q_heads + kv_heads || !active) continue;
    // a position outside the tables makes a row of NaN
    const float inv = known ? 1.0f / sqrtf(squares / static_cast<float>(D) + eps) : NAN;
    const bool is_k = h >= q_heads;
    float wa[V], wb[V];
    Pack<T>::unpack(weights[is_k][0], wa);
    Pack<T>::unpack(weights[is_k][1], wb);
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const float y0 = a[e] * (inv * wa[e]), y1 = b[e] * (inv * wb[e]);
      a[e] = rotated ? fmaf(y0, c0[e], -(y1 * s0[e])) : y0;
      b[e] = rotated ? fmaf(y1, c1[e], y0 * s1[e]) : y1;
    }
    T* out = is_k ? k_out + (static_cast<int64_t>(t) * kv_heads + (h - q_heads)) * D : q_out + (static_cast<int64_t>(t) * q_heads + h) * D;
    store16(out + at0, Pack<T>::pack(a));
    store16(out + at1, Pack<T>::pack(b));
  }
}

}  // namespace

extern "C" int llmq_qk_norm_rope(const void* q, const void* k, const void* q_weight, const void* k_weight, const void* cos_table,
                                 const void* sin_table, const void* positions_or_null, int position_bytes, void* q_out,
                                 void* k_out, int tokens, int q_heads, int kv_heads, int head_dim, int rotary_dim, int table_rows,
                                 int64_t q_row_stride, int64_t k_row_stride, float eps, int dtype, int table_dtype,
                                 llmq_stream_t stream) {
  if (tokens < 0 || q_heads < 0 || kv_heads < 0 || table_rows < 0)
    return llmq_host::fail_invalid("bad dimension tokens=%d q_heads=%d kv_heads=%d table_rows=%d", tokens, q_heads, kv_heads, table_rows);
  if (dtype != LLMQ_F32 && dtype != LLMQ_F16 && dtype != LLMQ_BF16)
    return llmq_host::fail_invalid("dtype code %d is not float32, float16 or bfloat16", dtype);
  if (table_dtype != dtype && table_dtype != LLMQ_F32) return llmq_host::fail_invalid("the tables hold float32 or the dtype of q and k");
  const int v = dtype == LLMQ_F32 ? 4 : 8;
  if (head_dim <= 0 || head_dim > 256 || head_dim % (2 * v))
    return llmq_host::fail_invalid("head_dim must be a multiple of %d up to 256, got %d", 2 * v, head_dim);
  if (rotary_dim <= 0 || rotary_dim > head_dim || rotary_dim % (2 * v))
    return llmq_host::fail_invalid("the rotated part must be a multiple of %d up to head_dim, got %d", 2 * v, rotary_dim);
  if (q_row_stride % v || k_row_stride % v) return llmq_host::fail_invalid("row strides must be multiples of %d elements", v);
  if (positions_or_null && position_bytes != 4 && position_bytes != 8)
    return llmq_host::fail_invalid("positions are integers of 4 or 8 bytes, got %d", position_bytes);
  if (!positions_or_null && table_rows < tokens)
    return llmq_host::fail_invalid("without positions the tables need a row for each of %d tokens, they have %d", tokens, table_rows);
  if (!(eps >= 0.0f) || std::isinf(eps)) return llmq_host::fail_invalid("eps must be finite and not negative");
  if (tokens == 0 || q_heads + kv_heads == 0) return 0;
  if (!q_weight || !k_weight || (table_rows && (!cos_table || !sin_table)) || (q_heads && (!q || !q_out)) || (kv_heads && (!k || !k_out)))
    return llmq_host::fail_invalid("null tensor pointer");
  uintptr_t all = 0;
  for (const void* t : {q, k, q_weight, k_weight, cos_table, sin_table, static_cast<const void*>(q_out), static_cast<const void*>(k_out)})
    all |= reinterpret_cast<uintptr_t>(t);
  if (all & 15u) return llmq_host::fail_invalid("tensors must be 16-byte aligned");
  int lanes = 1;
  while (lanes < head_dim / 2 / v) lanes *= 2;
  // several heads a lane where one each would be more lanes than the chip holds at once (256 x 2048)
  const int heads = q_heads + kv_heads;
  const bool many = static_cast<int64_t>(tokens) * heads * lanes > 256 * 2048 && heads >= kPasses;
  const int step = many ? (heads + kPasses - 1) / kPasses : heads;
  const int64_t vectors = static_cast<int64_t>(tokens) * step, items = vectors * lanes;
  if (items > INT32_MAX - kThreads) return llmq_host::fail_invalid("too many heads for one launch: %lld", static_cast<long long>(vectors));
  // (the outputs through the caches: past them 16000 tokens of 40 heads alone take 61 us instead of 65, but with an operator that reads the
  // queries behind 111 instead of 105)
  const dim3 grid(static_cast<unsigned>((items + kThreads - 1) / kThreads));
  hipStream_t s = static_cast<hipStream_t>(stream);
#define LLMQ_NORM_P(T, TABLE, L, P)                                                                                          \
  hipLaunchKernelGGL((qk_norm_rope_kernel<T, TABLE, L, P>), grid, dim3(kThreads), 0, s, static_cast<const T*>(q),               \
                     static_cast<const T*>(k), q_row_stride, k_row_stride, static_cast<const T*>(q_weight),                  \
                     static_cast<const T*>(k_weight), static_cast<const TABLE*>(cos_table),                                  \
                     static_cast<const TABLE*>(sin_table), positions_or_null, position_bytes == 8, static_cast<T*>(q_out),   \
                     static_cast<T*>(k_out), static_cast<uint32_t>(vectors), static_cast<uint32_t>(q_heads),                 \
                     static_cast<uint32_t>(kv_heads), static_cast<uint32_t>(step), head_dim, rotary_dim, table_rows, eps)
#define LLMQ_NORM(T, TABLE, L)                     \
  do {                                             \
    if (many) LLMQ_NORM_P(T, TABLE, L, kPasses);   \
    else LLMQ_NORM_P(T, TABLE, L, 1);              \
  } while (0)
#define LLMQ_NORM_L(T, TABLE)                     \
  switch (lanes) {                                \
    case 1: LLMQ_NORM(T, TABLE, 1); break;        \
    case 2: LLMQ_NORM(T, TABLE, 2); break;        \
    case 4: LLMQ_NORM(T, TABLE, 4); break;        \
    case 8: LLMQ_NORM(T, TABLE, 8); break;        \
    case 16: LLMQ_NORM(T, TABLE, 16); break;      \
    default: LLMQ_NORM(T, TABLE, 32); break;      \
  }
  const bool wide = table_dtype == LLMQ_F32;
  switch (dtype) {
    case LLMQ_F32: LLMQ_NORM_L(float, float); break;
    case LLMQ_F16: if (wide) { LLMQ_NORM_L(f16_t, float); } else { LLMQ_NORM_L(f16_t, f16_t); } break;
    default: if (wide) { LLMQ_NORM_L(bf16_t, float); } else { LLMQ_NORM_L(bf16_t, bf16_t); } break;
  }
#undef LLMQ_NORM_L
#undef LLMQ_NORM
#undef LLMQ_NORM_P
  return llmq_host::check_launch("qk_norm_rope_kernel");
}
