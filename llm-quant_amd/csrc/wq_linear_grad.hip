// The gradient of a quantized Linear by its input, gfx950:
//
//   gx[t, k] = sum_n g[t, n] W[n, k],     W = (dtype)(code * scale): the matrix of the reference's many-rows branch
//                                         (llmquant/quantizers/kernel.py:68-79), whose autograd this stands for
//
// Few rows: past the weight as it lies (dense_few.h). Otherwise the weight is brought to its values a piece of its rows at a time (dense_stage.h: a piece that the
// caches hold), and multiplied on the matrix core with the reduction outermost, as it lies (dense_tile.h); sums over the pieces and over the splits of one go
// through fp32 planes. Bound: the matrix core for training batches, the weight's way through memory and the conversion of its codes for few rows.
#include "dense_stage.h"

namespace {

using namespace llmq;

struct Plan {
  int64_t n_padded, piece, ld;   // N in whole steps; rows of W a piece; its columns
  int splits;
  bool stage_grad, few;          // few: rows that go past the weight as it lies
  int64_t o_weight, o_grad, o_sums, bytes;
};

constexpr int64_t kPieceBytes = int64_t{128} << 20;
// Up to so many rows the weight is read as it lies, once for each 64 (whole calls, us, this way for the other; bf16: 4096 x 4096 int8, 1 row 12 for 33, 320 rows 43 for
// 46, 512 46 for 50; 14336 x 4096 int4, 320 rows 75 for 91, 384 rows 106 for 93; fp32, 2048 x 2048 int8, 320 rows 41 for 100; 14336 x 4096 int4, 320 rows 339 for 430,
// 512 500 for 475; 4096 x 4096 int8, 320 rows 170 for 127).
constexpr int kFewMost = 320;

Plan plan_for(int rows, int N, int width, int wformat, int dtype) {
  Plan p{};
  const int64_t row16 = dtype == LLMQ_F32 ? 6 : 2;
  p.few = rows <= kFewMost;
  if (p.few) {
    p.splits = few_splits(N, width, rows, wformat);
    p.bytes = int64_t{4} * p.splits * rows * width;
    return p;
  }
  p.n_padded = round_up(N, 64);
  p.ld = width;
  p.stage_grad = dtype == LLMQ_F32 || N % 64 != 0;
  p.piece = kPieceBytes / (width * row16) / 64 * 64;
  if (p.piece < 64) p.piece = 64;
  if (p.piece > p.n_padded) p.piece = p.n_padded;
  p.splits = most_splits(width, rows, static_cast<int>(p.piece));
  int64_t at = round_up(p.piece * width * row16, 256);
  if (p.stage_grad) {
    p.o_grad = at;
    at += round_up(rows * p.n_padded * row16, 256);
  }
  if (splits_of_rows(rows, tile_rows(rows), (width + 255) / 256, width, p.splits).splits > 1 || p.piece < p.n_padded) {
    p.o_sums = at;
    at += round_up(sums_bytes(width, rows, p.splits), 256);
  }
  p.bytes = at;
  return p;
}

template <typename T>
int launch(const Plan& p, const void* grad, int64_t stride, const void* qweight, const float* wscale, void* out, uint8_t* workspace, int rows,
           int N, int G, int gs, int keep, int out_group, int wformat, int dtype, hipStream_t stream) {
  constexpr int P = TileType<T>::kPlanes;
  if (p.few) {
    float* sums = reinterpret_cast<float*>(workspace);
    columns_launch<T, false>(FewWeight{static_cast<const uint8_t*>(qweight), wscale, static_cast<int64_t>(G) * gs * wformat / 8, N, G * keep, G, gs, keep, out_group},
                      FewColumns{grad, stride, nullptr, rows, sums, p.splits}, wformat, stream);
    add_few_launch<T>(sums, p.splits, rows, G * keep, nullptr, nullptr, TargetTerm{}, out, stream);
    return llmq_host::check_launch("wq_linear_grad");
  }
  const int width = G * keep, n64 = static_cast<int>(p.n_padded);
  if (p.stage_grad)   // (zeros up to a whole step, against rows of W that are looked at again)
    stage_launch<T>(StageSource{grad, nullptr, nullptr, stride, rows, N, 0, rows, 0, 0, 0, 0}, StageTarget{workspace + p.o_grad, rows * p.n_padded, n64}, 0, stream);
  const uint8_t* b_base = p.stage_grad ? workspace + p.o_grad : static_cast<const uint8_t*>(grad);
  const int64_t b_plane = p.stage_grad ? 2 * rows * p.n_padded : 0, b_row = p.stage_grad ? int64_t{2} * n64 : stride * 2;
  float* sums = reinterpret_cast<float*>(workspace + p.o_sums);
  const bool summed = p.o_sums != 0;
  for (int first = 0; first < N; first += static_cast<int>(p.piece)) {
    const int n = N - first < p.piece ? N - first : static_cast<int>(p.piece);
    if (P == 1 && (out_group == 0 || first % out_group == 0)) {
      const int64_t scale_row = out_group > 0 ? first / out_group : first;
      if (int rc = llmq_dequant_weight(static_cast<const uint8_t*>(qweight) + static_cast<int64_t>(first) * G * gs * wformat / 8, wscale + scale_row * G,
                                       workspace, n, G, gs, keep, out_group, wformat, dtype, stream)) return rc;
    } else {
      stage_launch<T>(StageSource{qweight, wscale, nullptr, 0, N, width, first, n, G, gs, keep, out_group}, StageTarget{workspace, p.piece * width, width}, wformat, stream);
    }
    const TileOperand a{workspace, 2 * p.piece * width, int64_t{2} * width, width, n};
    const TileOperand b{b_base + int64_t{2} * first, b_plane, b_row, rows, 0};
    const int k = static_cast<int>(round_up(n, 64));
    if (summed) product_launch<T, true, false>(a, b, k, ProductOut{sums, width, nullptr, first == 0, p.splits}, stream);
    else product_launch<T, false, false>(a, b, k, ProductOut{out, width, nullptr, 1, 1}, stream);
  }
  if (summed) add_planes_launch<T>(sums, rows, width, p.splits, nullptr, nullptr, nullptr, TargetTerm{}, out, stream);
  return llmq_host::check_launch("wq_linear_grad");
}

}  // namespace

extern "C" size_t llmq_wq_linear_grad_workspace_bytes(int rows, int N, int G, int keep_per_group, int wformat, int dtype) {
  if (rows <= 0 || N <= 0 || G <= 0 || keep_per_group <= 0) return 0;
  return static_cast<size_t>(plan_for(rows, N, G * keep_per_group, wformat, dtype).bytes);
}

extern "C" int llmq_wq_linear_grad(const void* grad, int64_t grad_stride, const void* qweight, const float* wscale, void* grad_x,
                                   void* workspace, size_t workspace_bytes, int rows, int N, int G, int gs, int keep_per_group,
                                   int out_group, int wformat, int dtype, llmq_stream_t stream) {
  if (rows < 0 || N < 0 || G < 0) return llmq_host::fail_invalid("negative dimension rows=%d N=%d G=%d", rows, N, G);
  if (wformat != LLMQ_W_INT8 && wformat != LLMQ_W_INT4_PACKED) return llmq_host::fail_invalid("unsupported weight format %d, expected 8 or 4", wformat);
  if (gs <= 0 || gs % 8) return llmq_host::fail_invalid("group_size must be a positive multiple of 8, got %d", gs);
  if (keep_per_group <= 0 || keep_per_group > gs || keep_per_group % 8)
    return llmq_host::fail_invalid("keep_per_group must be a multiple of 8 up to %d, got %d", gs, keep_per_group);
  if (out_group < 0) return llmq_host::fail_invalid("out_group must be >= 0, got %d", out_group);
  if (dtype != LLMQ_F32 && dtype != LLMQ_F16 && dtype != LLMQ_BF16)
    return llmq_host::fail_invalid("dtype code %d is not float32, float16 or bfloat16", dtype);
  if (N % 8) return llmq_host::fail_invalid("the weight's rows must be a multiple of 8, got %d", N);
  if (rows == 0 || G == 0) return 0;
  if (N == 0) return llmq_host::fail_invalid("a weight of no rows");
  if (rows > (1 << 20) || N > (1 << 24) || static_cast<int64_t>(G) * keep_per_group > (1 << 24))
    return llmq_host::fail_invalid("at most 2^20 rows of 2^24 elements, got %d rows, %d x %lld", rows, N, static_cast<long long>(G) * keep_per_group);
  if (grad_stride < N || grad_stride % 8 || grad_stride > (1 << 24))
    return llmq_host::fail_invalid("grad's row stride must be a multiple of 8 of at least %d, got %lld", N, static_cast<long long>(grad_stride));
  if (!grad || !qweight || !wscale || !grad_x) return llmq_host::fail_invalid("null tensor pointer");
  if ((reinterpret_cast<uintptr_t>(grad) | reinterpret_cast<uintptr_t>(qweight) | reinterpret_cast<uintptr_t>(grad_x)) & 15u)
    return llmq_host::fail_invalid("grad, qweight and grad_x must be 16-byte aligned");
  const Plan p = plan_for(rows, N, G * keep_per_group, wformat, dtype);
  if (!p.few && !tile_spans(rows, tile_rows(rows), 2 * (p.stage_grad ? p.n_padded : grad_stride), 128))
    return llmq_host::fail_invalid("grad's row stride is too wide: %d neighbouring rows must lie within 4 GiB, got a stride of %lld elements", tile_rows(rows),
                                   static_cast<long long>(grad_stride));
  if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15u) || workspace_bytes < static_cast<size_t>(p.bytes))
    return llmq_host::fail_invalid("the workspace must be 16-byte aligned and hold %lld bytes, got %zu", static_cast<long long>(p.bytes), workspace_bytes);
  hipStream_t s = static_cast<hipStream_t>(stream);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  switch (dtype) {
    case LLMQ_F32: return launch<float>(p, grad, grad_stride, qweight, wscale, grad_x, ws, rows, N, G, gs, keep_per_group, out_group, wformat, dtype, s);
    case LLMQ_F16: return launch<f16_t>(p, grad, grad_stride, qweight, wscale, grad_x, ws, rows, N, G, gs, keep_per_group, out_group, wformat, dtype, s);
    default: return launch<bf16_t>(p, grad, grad_stride, qweight, wscale, grad_x, ws, rows, N, G, gs, keep_per_group, out_group, wformat, dtype, s);
  }
}
