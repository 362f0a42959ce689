// SPDX-License-Identifier: Apache-2.0
//
// The dense products on gfx950 (include/uniserve_linear.h states the operators): the entries and their
// refusals. The kernels and the choice among them are in linear_kernels.hpp.
#include "extents.hpp"
#include "linear.hpp"
#include "uniserve_adapter_linear.h"

namespace uniserve {
namespace linear {
namespace {

/// 64 x 64 tiles of 256 threads whose threads an axis of a launch holds (shapes that need more are not chosen).
constexpr int64_t kMostTiles = (int64_t{1} << 32) / 256 - 1;

/// The largest row stride of 256 rows within the DMA's 32-bit byte offsets.
constexpr int64_t kMostStride = int64_t{1} << 22;

/// Whether a product can be served: 0, with its parameters in `p`, or a refusal. A call without rows (m = 0) has no
/// parameters.
int32_t check(const uniserve_linear_call *call, bool gated, const char *name, LinearParams &p) {
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
  const Extent out = extent(call->out, m, n, out_stride, out_bytes);
  if (overlap(out, extent(call->input, m, k, x_stride, 2)) || overlap(out, extent(call->weight, weight_rows, k, w_stride, 2)) ||
      overlap(out, extent(call->bias, 1, weight_rows, weight_rows, bias_bytes)) ||
      overlap(out, extent(call->gate, m, 1, gate_stride, 2)))
    return UNISERVE_REFUSE(call, "%s's output overlaps one of its inputs", name);
  if (call->residual != nullptr && !(call->residual == call->out && residual_stride == out_stride) &&
      overlap(out, extent(call->residual, m, n, residual_stride, out_bytes)))
    return UNISERVE_REFUSE(call, "%s's output overlaps its residual in part", name);

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
  p.by_dma = k % 8 == 0 && x_stride % 8 == 0 && w_stride % 8 == 0 && aligned_to(p.x, 16) && aligned_to(p.w, 16) &&
             x_stride <= kMostStride && w_stride <= kMostStride;
  if (ceil_div<int64_t>(m, 64) * ceil_div<int64_t>(n, gated ? 32 : 64) > kMostTiles)
    return UNISERVE_REFUSE(call, "%s's output has too many tiles", name);
  return 0;
}

/// Rows whose tiles of 32 x 32 rank values, at the largest rank, an axis of a launch holds.
constexpr int64_t kMostAdapterRows = int64_t{1} << 23;

int32_t run(const uniserve_linear_call *call, void *stream, bool gated, const char *name) {
  LinearParams p{};
  const int32_t refused = check(call, gated, name, p);
  if (refused != 0 || call->m == 0) return refused;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (call->dtype == UNISERVE_DTYPE_F16) launch_f16(p, gated, s);
  else launch_bf16(p, gated, s);
  return launched(call, name);
}

int64_t workspace_of(int64_t rows, const LowLayout &layout, int halves) { return rows * layout.row_bytes(halves); }

int32_t run_adapters(const uniserve_adapter_linear_call *adapters, void *stream, bool gated, const char *name) {
  const uniserve_linear_call *call = &adapters->product;
  AdapterParams p{};
  const int32_t refused = check(call, gated, name, p);
  if (refused != 0) return refused;
  const int64_t rank = adapters->rank, count = adapters->adapters, halves = gated ? 2 : 1;
  if (rank <= 0 || count <= 0) return UNISERVE_REFUSE(call, "%s needs a positive rank and adapters", name);
  if (rank > UNISERVE_ADAPTER_MAX_RANK) return UNISERVE_REFUSE(call, "%s serves ranks of up to %d", name, UNISERVE_ADAPTER_MAX_RANK);
  if (count > INT32_MAX) return UNISERVE_REFUSE(call, "%s's extents do not fit int32", name);
  if (p.m == 0) return 0;
  if (p.m > kMostAdapterRows) return UNISERVE_REFUSE(call, "%s serves up to %lld rows", name, static_cast<long long>(kMostAdapterRows));
  if (adapters->down == nullptr || adapters->up == nullptr || adapters->adapter == nullptr || adapters->workspace == nullptr)
    return UNISERVE_REFUSE(call, "%s needs down, up, adapter and a workspace", name);
  const int64_t down_rows = halves * rank, up_rows = halves * p.n;
  // A single row or adapter has no stride to go by.
  p.down_row_stride = down_rows > 1 ? adapters->down_row_stride : p.k;
  p.up_row_stride = up_rows > 1 ? adapters->up_row_stride : rank;
  p.down_stride = count > 1 ? adapters->down_stride : 0;
  p.up_stride = count > 1 ? adapters->up_stride : 0;
  if (p.down_row_stride < p.k || p.up_row_stride < rank || p.down_stride < 0 || p.up_stride < 0)
    return UNISERVE_REFUSE(call, "%s's adapter strides are negative or shorter than the rows", name);
  if (p.down_row_stride > kMostElements / down_rows || p.up_row_stride > kMostElements / up_rows ||
      p.down_stride > kMostElements / count || p.up_stride > kMostElements / count)
    return UNISERVE_REFUSE(call, "%s's adapters are too large", name);
  const int64_t need = workspace_of(p.m, LowLayout(rank), static_cast<int>(halves));
  if (adapters->workspace_bytes < need)
    return UNISERVE_REFUSE(call, "%s needs a workspace of %lld bytes", name, static_cast<long long>(need));
  if (!aligned_to(adapters->workspace, 16)) return UNISERVE_REFUSE(call, "%s's workspace is 16-byte aligned", name);
  const Extent out = extent(p.out, p.m, p.n, p.out_stride, p.out_f32 ? 4 : 2);
  const Extent work = extent(adapters->workspace, 1, need, need, 1);
  // (the stacks as whole ranges: nothing else has a reason to lie between their rows)
  const Extent down = extent(adapters->down, 1, (count - 1) * p.down_stride + (down_rows - 1) * p.down_row_stride + p.k, 0, 2);
  const Extent up = extent(adapters->up, 1, (count - 1) * p.up_stride + (up_rows - 1) * p.up_row_stride + rank, 0, 2);
  const Extent index = extent(adapters->adapter, 1, p.m, p.m, 4), scales = extent(adapters->scales, 1, count, count, 4);
  for (const Extent &array : {down, up, index, scales, work})
    if (overlap(out, array)) return UNISERVE_REFUSE(call, "%s's output overlaps its adapters or its workspace", name);
  for (const Extent &array : {down, up, index, scales, extent(p.x, p.m, p.k, p.x_stride, 2), extent(p.w, up_rows, p.k, p.w_stride, 2),
                              extent(p.bias, 1, up_rows, up_rows, p.bias_f32 ? 4 : 2), extent(p.gate, p.m, 1, p.gate_stride, 2),
                              extent(p.residual, p.m, p.n, p.residual_stride, p.out_f32 ? 4 : 2)})
    if (overlap(work, array)) return UNISERVE_REFUSE(call, "%s's workspace overlaps one of its inputs", name);
  p.down = static_cast<const uint16_t *>(adapters->down);
  p.up = static_cast<const uint16_t *>(adapters->up);
  p.adapter = adapters->adapter;
  p.scales = adapters->scales;
  p.low = static_cast<char *>(adapters->workspace);
  p.adapters = static_cast<int32_t>(count), p.rank = static_cast<int32_t>(rank);
  p.down_by_dma = p.k % 8 == 0 && p.x_stride % 8 == 0 && p.down_stride % 8 == 0 && p.down_row_stride % 8 == 0 &&
                  aligned_to(p.x, 16) && aligned_to(adapters->down, 16) && p.x_stride <= kMostStride &&
                  down_rows * p.down_row_stride <= 256 * kMostStride;
  p.up_whole = rank % 8 == 0 && p.up_stride % 8 == 0 && p.up_row_stride % 8 == 0 && aligned_to(adapters->up, 16) &&
               p.up_row_stride <= kMostStride;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (call->dtype == UNISERVE_DTYPE_F16) launch_adapters_f16(p, gated, s);
  else launch_adapters_bf16(p, gated, s);
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

extern "C" int64_t uniserve_adapter_workspace(int64_t rows, int64_t rank_rows) {
  using namespace uniserve::linear;
  if (rows <= 0 || rank_rows <= 0 || rows > INT32_MAX || rank_rows > 2 * UNISERVE_ADAPTER_MAX_RANK) return 0;
  const int64_t plain = workspace_of(rows, LowLayout(rank_rows), 1), gated = workspace_of(rows, LowLayout((rank_rows + 1) / 2), 2);
  return plain > gated ? plain : gated;
}

extern "C" int32_t uniserve_adapter_linear(const uniserve_adapter_linear_call *call, void *stream) {
  return uniserve::guarded(call == nullptr ? nullptr : &call->product,
                           [&]() { return uniserve::linear::run_adapters(call, stream, false, "adapter_linear"); });
}

extern "C" int32_t uniserve_adapter_gated_linear(const uniserve_adapter_linear_call *call, void *stream) {
  return uniserve::guarded(call == nullptr ? nullptr : &call->product,
                           [&]() { return uniserve::linear::run_adapters(call, stream, true, "adapter_gated_linear"); });
}
