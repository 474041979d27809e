// Writing a cache in blocks (layout: kv_blocks.h), quantized, and reading it back, gfx950.
//
//   append   a = max |x| over the call's tokens in a block, for each head
//            s = max(a / 127, 1e-8) where the call writes the block's first token, else max(s_old, that)
//            codes of the call's tokens: clamp(rint(x / s)); of the block's earlier tokens: clamp(rint((c s_old) / s))
//   dequant  T(c s)
#include "kv_blocks.h"

namespace {

using namespace llmq;

constexpr int kThreads = 256;

__device__ __forceinline__ int64_t code_at(bool value, int64_t id, int h, int heads, int block, int D, int slot, int d) {
  const int64_t base = (id * heads + h) * block * D;
  return base + (value ? (static_cast<int64_t>(slot / kStrip) * D + d) * kStrip + slot % kStrip : static_cast<int64_t>(slot) * D + d);
}

template <typename T>
__global__ __launch_bounds__(kThreads) void append_kernel(
    const T* __restrict__ key, const T* __restrict__ value, const int64_t key_stride, const int64_t value_stride,
    int8_t* __restrict__ k_codes, int8_t* __restrict__ v_codes, float* __restrict__ k_scale, float* __restrict__ v_scale,
    const BlockTable table, const int32_t* __restrict__ cached, const Ragged rows, const int heads, const int D, const int block) {
  __shared__ float red[kThreads / kWave];
  const bool is_value = blockIdx.x & 1;
  const int h = static_cast<int>(blockIdx.x / 2) % heads;
  int64_t piece = blockIdx.x / 2 / heads;
  const int b = rows.find(1, block, 2, piece);
  const int64_t from = cached[b];
  const int n = rows.count(b);
  if (from < 0 || n == 0) return;
  const int64_t logical = from / block + piece;
  if (logical > (from + n - 1) / block) return;
  const int id = table.at(b, static_cast<int>(min(logical, static_cast<int64_t>(INT32_MAX))));
  if (id < 0) return;
  const int64_t at = logical * block;   // the block's first position
  const int lo = static_cast<int>(max(from - at, static_cast<int64_t>(0))), hi = static_cast<int>(min(from + n - at, static_cast<int64_t>(block)));
  const int64_t row0 = rows.first(b) + (at + lo - from);   // the row of slot lo
  const T* x = (is_value ? value + row0 * value_stride : key + row0 * key_stride) + static_cast<int64_t>(h) * D;
  const int64_t stride = is_value ? value_stride : key_stride;
  int8_t* codes = is_value ? v_codes : k_codes;
  float* scale = (is_value ? v_scale : k_scale) + static_cast<int64_t>(id) * heads + h;

  float amax = 0.0f;
  for (int i = threadIdx.x; i < (hi - lo) * D; i += kThreads) amax = fmaxf(amax, fabsf(to_float(x[(i / D) * stride + i % D])));
  amax = group_max<64>(amax);
  if ((threadIdx.x & (kWave - 1)) == 0) red[threadIdx.x / kWave] = amax;
  const float before = *scale;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kThreads / kWave; ++w) amax = fmaxf(amax, red[w]);
  float s = scale_from_amax(amax, 127.0f);
  if (lo > 0) s = fmaxf(s, before);
  if (threadIdx.x == 0) *scale = s;
  if (s > before) {
    for (int i = threadIdx.x; i < lo * D; i += kThreads) {
      int8_t* c = codes + code_at(is_value, id, h, heads, block, D, i / D, i % D);
      *c = static_cast<int8_t>(quant_code(static_cast<float>(*c) * before, s, -128.0f, 127.0f));
    }
  }
  for (int i = threadIdx.x; i < (hi - lo) * D; i += kThreads) {
    const float f = to_float(x[(i / D) * stride + i % D]);
    codes[code_at(is_value, id, h, heads, block, D, lo + i / D, i % D)] = static_cast<int8_t>(quant_code(f, s, -128.0f, 127.0f));
  }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void dequant_kernel(
    const int8_t* __restrict__ k_codes, const int8_t* __restrict__ v_codes, const float* __restrict__ k_scale,
    const float* __restrict__ v_scale, const BlockTable table, const Ragged rows, const int32_t* __restrict__ first_or_null,
    T* __restrict__ k_out, T* __restrict__ v_out, const int heads, const int D, const int block) {
  const bool is_value = blockIdx.x & 1;
  const int h = static_cast<int>(blockIdx.x / 2) % heads;
  int64_t piece = blockIdx.x / 2 / heads;
  const int b = rows.find(1, block, 2, piece);
  const int64_t from = first_or_null == nullptr ? 0 : max(first_or_null[b], 0);
  const int n = rows.count(b);
  const int64_t logical = from / block + piece;
  if (n == 0 || logical > (from + n - 1) / block) return;
  const int id = table.at(b, static_cast<int>(min(logical, static_cast<int64_t>(INT32_MAX))));
  const int64_t at = logical * block;
  const int lo = static_cast<int>(max(from - at, static_cast<int64_t>(0))), hi = static_cast<int>(min(from + n - at, static_cast<int64_t>(block)));
  const int64_t row0 = rows.first(b) + (at + lo - from);
  T* out = (is_value ? v_out : k_out) + (static_cast<int64_t>(h) * rows.rows + row0) * D;
  const int8_t* codes = is_value ? v_codes : k_codes;
  const float s = id < 0 ? 0.0f : (is_value ? v_scale : k_scale)[static_cast<int64_t>(id) * heads + h];
  for (int i = threadIdx.x; i < (hi - lo) * D; i += kThreads) {
    const float c = id < 0 ? 0.0f : static_cast<float>(codes[code_at(is_value, id, h, heads, block, D, lo + i / D, i % D)]);
    out[i] = from_float<T>(c * s);
  }
}

int check_cache(const void* k_codes, const void* v_codes, const void* k_scale, const void* v_scale, const void* block_table) {
  if (!k_codes || !v_codes || !k_scale || !v_scale || !block_table) return llmq_host::fail_invalid("null tensor pointer");
  if ((reinterpret_cast<uintptr_t>(k_codes) | reinterpret_cast<uintptr_t>(v_codes)) & 15u)
    return llmq_host::fail_invalid("the codes must be 16-byte aligned");
  return 0;
}

// pieces of a ragged batch (Ragged::find with spare 2): an upper bound of the blocks that its rows touch
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
  const dim3 grid(static_cast<unsigned>(pieces(tokens, sequences, block) * 2 * kv_heads));
  hipStream_t s = static_cast<hipStream_t>(stream);
#define LLMQ_APPEND(T)                                                                                                       \
  hipLaunchKernelGGL(append_kernel<T>, grid, dim3(kThreads), 0, s, static_cast<const T*>(key), static_cast<const T*>(value), \
                     key_row_stride, value_row_stride, static_cast<int8_t*>(k_codes), static_cast<int8_t*>(v_codes),         \
                     k_scale, v_scale, table, cached, rows, kv_heads, head_dim, block)
  switch (dtype) {
    case LLMQ_F32: LLMQ_APPEND(float); break;
    case LLMQ_F16: LLMQ_APPEND(f16_t); break;
    default: LLMQ_APPEND(bf16_t); break;
  }
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
  const dim3 grid(static_cast<unsigned>(pieces(n_tokens, sequences, block) * 2 * kv_heads));
  hipStream_t s = static_cast<hipStream_t>(stream);
#define LLMQ_DEQUANT(T)                                                                                                  \
  hipLaunchKernelGGL(dequant_kernel<T>, grid, dim3(kThreads), 0, s, static_cast<const int8_t*>(k_codes),                 \
                     static_cast<const int8_t*>(v_codes), k_scale, v_scale, table, rows, first_or_null,                  \
                     static_cast<T*>(k_out), static_cast<T*>(v_out), kv_heads, head_dim, block)
  switch (dtype) {
    case LLMQ_F32: LLMQ_DEQUANT(float); break;
    case LLMQ_F16: LLMQ_DEQUANT(f16_t); break;
    default: LLMQ_DEQUANT(bf16_t); break;
  }
#undef LLMQ_DEQUANT
  return llmq_host::check_launch("dequant_kernel");
}
