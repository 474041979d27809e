// Attention of a batch over a cache in blocks (layout: kv_blocks.h), gfx950: row i of sequence b sees the tokens
// 0 .. cached[b] + i,
//   t_j = (q . k_j) s_k scale,   out = sum 2^t_j s_v c_j / sum 2^t_j
#include <cmath>

#include "kv_blocks.h"

namespace {

using namespace llmq;

constexpr int kMaxDim = 256;

// a wave per row and query head
template <typename T>
__global__ __launch_bounds__(kWave) void attention_kernel(
    const T* __restrict__ query, const int64_t q_stride, const int8_t* __restrict__ k_codes, const int8_t* __restrict__ v_codes,
    const float* __restrict__ k_scale, const float* __restrict__ v_scale, const BlockTable table,
    const int32_t* __restrict__ cached, const Ragged rows, T* __restrict__ out, const int q_heads, const int heads, const int D,
    const int block, const float scale_log2e) {
  __shared__ float s_q[kMaxDim], s_w[kWave];
  const int lane = threadIdx.x, qh = blockIdx.x % q_heads, row = blockIdx.x / q_heads, h = qh / (q_heads / heads);
  int found = 0;
  for (int b0 = 0; b0 < rows.sequences; b0 += kWave) {
    const int b = b0 + lane;
    found += __popcll(__ballot(b < rows.sequences && rows.first(b) <= row));
  }
  const int b = found - 1;
  if (b < 0 || row - rows.first(b) >= rows.count(b)) return;
  T* o = out + (static_cast<int64_t>(row) * q_heads + qh) * D;
  const int64_t limit = cached[b] < 0 ? 0 : min(static_cast<int64_t>(cached[b]) + row - rows.first(b) + 1, static_cast<int64_t>(table.width) * block);
  for (int d = lane; d < D; d += kWave) s_q[d] = to_float(query[row * q_stride + static_cast<int64_t>(qh) * D + d]);
  float m = -INFINITY, l = 0.0f, acc[kMaxDim / kWave] = {};
  for (int64_t j0 = 0; j0 < limit; j0 += kWave) {
    __syncthreads();
    const int64_t j = j0 + lane;
    const int id = j < limit ? table.at(b, static_cast<int>(j / block)) : -1;
    const int64_t at = (static_cast<int64_t>(max(id, 0)) * heads + h) * block * D;
    float t = -INFINITY;
    if (id >= 0) {
      float dot = 0.0f;
      for (int d = 0; d < D; ++d) dot = fmaf(s_q[d], static_cast<float>(k_codes[at + (j % block) * D + d]), dot);
      t = dot * k_scale[static_cast<int64_t>(id) * heads + h] * scale_log2e;
    }
    const float m_new = fmaxf(m, group_max<64>(t)), base = m_new == -INFINITY ? 0.0f : m_new;
    const float alpha = exp2f(m - base), p = exp2f(t - base);
    m = m_new;
    l = l * alpha + wave_sum(p);
    s_w[lane] = id >= 0 ? p * v_scale[static_cast<int64_t>(id) * heads + h] : 0.0f;
    __syncthreads();
    for (int e = 0; e < D / kWave; ++e) {
      float sum = 0.0f;
      for (int i = 0; i < kWave; ++i) {
        const int64_t ji = j0 + i;
        const int idi = ji < limit ? table.at(b, static_cast<int>(ji / block)) : -1;
        if (idi < 0) continue;
        const int64_t ati = (static_cast<int64_t>(idi) * heads + h) * block * D;
        const int slot = static_cast<int>(ji % block);
        sum = fmaf(s_w[i], static_cast<float>(v_codes[ati + (static_cast<int64_t>(slot / kStrip) * D + e * kWave + lane) * kStrip + slot % kStrip]), sum);
      }
      acc[e] = acc[e] * alpha + sum;
    }
  }
  for (int e = 0; e < D / kWave; ++e) o[e * kWave + lane] = from_float<T>(l == 0.0f ? 0.0f : acc[e] / l);
}

}  // namespace

extern "C" size_t llmq_kv_block_attention_workspace_bytes(int, int, int, int, int, int, int) { return 0; }

extern "C" int llmq_kv_block_attention(const void* query, int64_t q_row_stride, const void* k_codes, const void* v_codes,
                                       const float* k_scale, const float* v_scale, const int32_t* block_table,
                                       int64_t table_stride, const int32_t* cached, const int32_t* query_start_or_null, void* out,
                                       void* workspace, size_t workspace_bytes, float sm_scale, int tokens, int sequences,
                                       int q_heads, int kv_heads, int head_dim, int block, int n_blocks, int table_width,
                                       int dtype, llmq_stream_t stream) {
  if (int rc = llmq_host::check_block_shape(tokens, sequences, kv_heads, head_dim, block, n_blocks, table_width, table_stride, dtype)) return rc;
  if (q_heads <= 0 || q_heads % kv_heads != 0) return llmq_host::fail_invalid("q_heads %d is not a multiple of kv_heads %d", q_heads, kv_heads);
  if (!std::isfinite(sm_scale)) return llmq_host::fail_invalid("sm_scale must be finite");
  if (!query_start_or_null && tokens != sequences)
    return llmq_host::fail_invalid("without query_start a sequence has one row: %d rows, %d sequences", tokens, sequences);
  const int v = dtype == LLMQ_F32 ? 4 : 8;
  if (q_row_stride % v) return llmq_host::fail_invalid("row strides must be multiples of %d elements", v);
  if (tokens == 0 || sequences == 0) return 0;
  if (static_cast<int64_t>(tokens) * q_heads > INT32_MAX / 2)
    return llmq_host::fail_invalid("too many rows and heads for one launch: %d, %d", tokens, q_heads);
  const bool empty = n_blocks == 0 || table_width == 0;   // (tensors of no elements have no address)
  if (!query || !cached || !out || (!empty && (!k_codes || !v_codes || !k_scale || !v_scale || !block_table)))
    return llmq_host::fail_invalid("null tensor pointer");
  uintptr_t all = 0;
  for (const void* t : {query, k_codes, v_codes, static_cast<const void*>(out)}) all |= reinterpret_cast<uintptr_t>(t);
  if (all & 15u) return llmq_host::fail_invalid("query, codes and out must be 16-byte aligned");
  const BlockTable table{block_table, table_stride, table_width, n_blocks};
  const Ragged rows{query_start_or_null, sequences, tokens};
  const dim3 grid(static_cast<unsigned>(tokens) * q_heads);
  hipStream_t s = static_cast<hipStream_t>(stream);
#define LLMQ_ATTEND(T)                                                                                                      \
  hipLaunchKernelGGL(attention_kernel<T>, grid, dim3(kWave), 0, s, static_cast<const T*>(query), q_row_stride,              \
                     static_cast<const int8_t*>(k_codes), static_cast<const int8_t*>(v_codes), k_scale, v_scale, table,     \
                     cached, rows, static_cast<T*>(out), q_heads, kv_heads, head_dim, block, sm_scale * 1.4426950408889634f)
  switch (dtype) {
    case LLMQ_F32: LLMQ_ATTEND(float); break;
    case LLMQ_F16: LLMQ_ATTEND(f16_t); break;
    default: LLMQ_ATTEND(bf16_t); break;
  }
#undef LLMQ_ATTEND
  return llmq_host::check_launch("attention_kernel");
}
