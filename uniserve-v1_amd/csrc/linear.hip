// SPDX-License-Identifier: Apache-2.0
//
// The dense products on gfx950 (include/uniserve_linear.h states the operators): the entries and their
// refusals. The kernels and the choice among them are in linear_kernels.hpp.
#include "linear.hpp"

namespace uniserve {
namespace linear {
namespace {

/// `rows` rows of `bytes` bytes, `stride` bytes apart.
struct Extent {
  const char *first;
  int64_t rows, bytes, stride;
};

/// Whether two arrays share a byte. Rows of equal strides may interleave (two column ranges of one
/// buffer); of different strides, arrays whose ranges meet count as sharing.
bool overlap(const Extent &a, const Extent &b) {
  if (a.first == nullptr || b.first == nullptr || a.rows == 0 || b.rows == 0) return false;
  const uintptr_t a0 = reinterpret_cast<uintptr_t>(a.first), b0 = reinterpret_cast<uintptr_t>(b.first);
  const uintptr_t a1 = a0 + static_cast<uintptr_t>((a.rows - 1) * a.stride + a.bytes);
  const uintptr_t b1 = b0 + static_cast<uintptr_t>((b.rows - 1) * b.stride + b.bytes);
  if (a1 <= b0 || b1 <= a0) return false;
  if (a.stride != b.stride || a.rows == 1 || b.rows == 1) return true;
  const int64_t apart = static_cast<int64_t>(b0 - a0) % a.stride;
  const int64_t offset = apart < 0 ? apart + a.stride : apart;  // where b's rows start in a's
  return !(offset >= a.bytes && offset + b.bytes <= a.stride);
}

bool aligned_to(const void *pointer, uintptr_t bytes) { return reinterpret_cast<uintptr_t>(pointer) % bytes == 0; }

/// Extents whose product of rows and stride stays far below 2^63 bytes.
constexpr int64_t kMostElements = int64_t{1} << 40;
/// 64 x 64 tiles of 256 threads whose threads an axis of a launch holds (shapes that need more are not chosen).
constexpr int64_t kMostTiles = (int64_t{1} << 32) / 256 - 1;

int32_t run(const uniserve_linear_call *call, void *stream, bool gated, const char *name) {
  const int64_t m = call->m, n = call->n, k = call->k;
  if (m < 0 || n <= 0 || k <= 0) return UNISERVE_REFUSE(call, "%s needs non-negative m and positive n and k", name);
  if (call->dtype != UNISERVE_DTYPE_BF16 && call->dtype != UNISERVE_DTYPE_F16)
    return UNISERVE_REFUSE(call, "%s multiplies bf16 or f16 rows", name);
  if (call->out_dtype != call->dtype && (gated || call->out_dtype != UNISERVE_DTYPE_F32))
    return UNISERVE_REFUSE(call, gated ? "%s writes the inputs' type" : "%s writes the inputs' type or f32", name);
  if (call->bias != nullptr && call->bias_dtype != call->dtype && call->bias_dtype != UNISERVE_DTYPE_F32)
    return UNISERVE_REFUSE(call, "%s takes a bias of the inputs' type or f32", name);
  if (call->activation != UNISERVE_ACTIVATION_SILU && call->activation != UNISERVE_ACTIVATION_GELU_TANH &&
      (gated || call->activation != UNISERVE_ACTIVATION_NONE))
    return UNISERVE_REFUSE(call, gated ? "%s gates by silu or gelu_tanh" : "%s serves no activation, silu or gelu_tanh", name);
  if (gated && (call->gate != nullptr || call->residual != nullptr))
    return UNISERVE_REFUSE(call, "%s has no row gate and no residual", name);
  if (m == 0) return 0;
  if (call->out == nullptr || call->input == nullptr || call->weight == nullptr)
    return UNISERVE_REFUSE(call, "%s needs out, input and weight", name);
  const int64_t weight_rows = gated ? 2 * n : n;
  if ((m > 1 && call->input_row_stride < k) || (weight_rows > 1 && call->weight_row_stride < k) ||
      (m > 1 && call->out_row_stride < n) || (call->residual != nullptr && m > 1 && call->residual_row_stride < n))
    return UNISERVE_REFUSE(call, "%s's row strides are shorter than its rows", name);
  if (call->gate != nullptr && m > 1 && call->gate_stride < 0)
    return UNISERVE_REFUSE(call, "%s's gate stride is negative", name);
  if (m > INT32_MAX || n > INT32_MAX / 2 || k > INT32_MAX)
    return UNISERVE_REFUSE(call, "%s's extents do not fit int32", name);
  // A single row has no stride to go by, an absent array neither.
  const int64_t x_stride = m > 1 ? call->input_row_stride : k;
  const int64_t w_stride = weight_rows > 1 ? call->weight_row_stride : k;
  const int64_t out_stride = m > 1 ? call->out_row_stride : n;
  const int64_t residual_stride = m > 1 && call->residual != nullptr ? call->residual_row_stride : n;
  const int64_t gate_stride = m > 1 && call->gate != nullptr ? call->gate_stride : 0;
  for (const int64_t stride : {x_stride, out_stride, residual_stride, gate_stride})
    if (stride > kMostElements / m) return UNISERVE_REFUSE(call, "%s's arrays are too large", name);
  if (w_stride > kMostElements / weight_rows) return UNISERVE_REFUSE(call, "%s's arrays are too large", name);
  const int64_t out_bytes = call->out_dtype == UNISERVE_DTYPE_F32 ? 4 : 2;
  const int64_t bias_bytes = call->bias_dtype == UNISERVE_DTYPE_F32 ? 4 : 2;
  const auto extent = [](const void *first, int64_t rows, int64_t columns, int64_t stride, int64_t bytes) {
    return Extent{static_cast<const char *>(first), rows, columns * bytes, stride * bytes};
  };
  const Extent out = extent(call->out, m, n, out_stride, out_bytes);
  if (overlap(out, extent(call->input, m, k, x_stride, 2)) || overlap(out, extent(call->weight, weight_rows, k, w_stride, 2)) ||
      overlap(out, extent(call->bias, 1, weight_rows, weight_rows, bias_bytes)) ||
      overlap(out, extent(call->gate, m, 1, gate_stride, 2)))
    return UNISERVE_REFUSE(call, "%s's output overlaps one of its inputs", name);
  if (call->residual != nullptr && !(call->residual == call->out && residual_stride == out_stride) &&
      overlap(out, extent(call->residual, m, n, residual_stride, out_bytes)))
    return UNISERVE_REFUSE(call, "%s's output overlaps its residual in part", name);

  LinearParams p{};
  p.x = static_cast<const uint16_t *>(call->input);
  p.w = static_cast<const uint16_t *>(call->weight);
  p.bias = call->bias;
  p.gate = static_cast<const uint16_t *>(call->gate);
  p.residual = call->residual;
  p.out = call->out;
  p.m = m, p.n = n, p.k = k;
  p.x_stride = x_stride, p.w_stride = w_stride, p.out_stride = out_stride;
  p.residual_stride = residual_stride, p.gate_stride = gate_stride;
  p.bias_f32 = call->bias_dtype == UNISERVE_DTYPE_F32;
  p.out_f32 = call->out_dtype == UNISERVE_DTYPE_F32;
  p.activation = static_cast<int32_t>(call->activation);
  // The tile kernels' DMA reads whole 16 bytes at aligned addresses, a tile's rows within 32-bit offsets.
  constexpr int64_t kMostStride = int64_t{1} << 22;
  p.by_dma = k % 8 == 0 && x_stride % 8 == 0 && w_stride % 8 == 0 && aligned_to(p.x, 16) && aligned_to(p.w, 16) &&
             x_stride <= kMostStride && w_stride <= kMostStride;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (ceil_div<int64_t>(m, 64) * ceil_div<int64_t>(n, gated ? 32 : 64) > kMostTiles)
    return UNISERVE_REFUSE(call, "%s's output has too many tiles", name);
  if (call->dtype == UNISERVE_DTYPE_F16) launch_f16(p, gated, s);
  else launch_bf16(p, gated, s);
  return launched(call, name);
}

}  // namespace
}  // namespace linear
}  // namespace uniserve

extern "C" int32_t uniserve_linear(const uniserve_linear_call *call, void *stream) {
  return uniserve::guarded(call, [&]() { return uniserve::linear::run(call, stream, false, "linear"); });
}

extern "C" int32_t uniserve_gated_linear(const uniserve_linear_call *call, void *stream) {
  return uniserve::guarded(call, [&]() { return uniserve::linear::run(call, stream, true, "gated_linear"); });
}
