// SPDX-License-Identifier: Apache-2.0
//
// The dense products on gfx950 (include/uniserve_linear.h states the operators): the entries, their
// refusals, the choice of the kernel, and the kernel that serves every stride and extent.
#include "linear.hpp"

namespace uniserve {
namespace linear {
namespace {

constexpr int kThreads = 256;
constexpr int kTile = 64;   // tokens and output columns of a workgroup
constexpr int kStep = 32;   // K elements a step
constexpr int kPitch = 40;  // elements between tile rows in LDS (80 bytes: 16 rows on distinct banks)

/// Elements at .. at + 7 of a row that ends before `limit`, zeros past it; whole 16 bytes where the
/// rows are aligned, else one by one.
__device__ __forceinline__ u32x4 load8(const uint16_t *row, int64_t at, int64_t limit, bool aligned) {
  if (aligned && at + 8 <= limit) return *reinterpret_cast<const u32x4 *>(row + at);
  uint32_t e[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) e[i] = at + i < limit ? row[at + i] : 0u;
  return u32x4{e[0] | (e[1] << 16), e[2] | (e[3] << 16), e[4] | (e[5] << 16), e[6] | (e[7] << 16)};
}

/// Any strides, extents and alignments: a 64 x 64 tile a workgroup, wavefront w the tile's tokens
/// 16 w .. 16 w + 15 by all its columns. Weight rows are MFMA operand A and tokens operand B, so each
/// lane holds four consecutive columns of one token.
template <class T, bool kGated>
__global__ void __launch_bounds__(kThreads) any_kernel(LinearParams p) {
  constexpr int kHalves = kGated ? 2 : 1;
  __shared__ __align__(16) uint16_t shared_x[kTile * kPitch];
  __shared__ __align__(16) uint16_t shared_w[kHalves][kTile * kPitch];
  const int t = static_cast<int>(threadIdx.x);
  const int wave = t / kWave;
  const int lane = lane_id();
  const int r16 = lane & 15;
  const int g = lane >> 4;
  const int64_t m_tiles = ceil_div<int64_t>(p.m, kTile);
  const int64_t m0 = static_cast<int64_t>(blockIdx.x) % m_tiles * kTile;
  const int64_t n0 = static_cast<int64_t>(blockIdx.x) / m_tiles * kTile;

  // Thread t stages K elements 8 (t % 4) .. of tile row t / 4; rows past the edge repeat the last one
  // (their sums are never stored).
  const int stage_row = t >> 2;
  const int stage_k = (t & 3) * 8;
  const uint16_t *x_row = p.x + (m0 + stage_row < p.m ? m0 + stage_row : p.m - 1) * p.x_stride;
  const uint16_t *w_row[kHalves];
#pragma unroll
  for (int h = 0; h < kHalves; ++h) w_row[h] = p.w + ((n0 + stage_row < p.n ? n0 + stage_row : p.n - 1) + h * p.n) * p.w_stride;

  floatx4 acc[kHalves][4];
#pragma unroll
  for (int h = 0; h < kHalves; ++h)
#pragma unroll
    for (int b = 0; b < 4; ++b) acc[h][b] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
  for (int64_t k = 0; k < p.k; k += kStep) {
    const u32x4 x = load8(x_row, k + stage_k, p.k, p.rows_of_16);
    u32x4 w[kHalves];
#pragma unroll
    for (int h = 0; h < kHalves; ++h) w[h] = load8(w_row[h], k + stage_k, p.k, p.rows_of_16);
    __syncthreads();
    *reinterpret_cast<u32x4 *>(shared_x + stage_row * kPitch + stage_k) = x;
#pragma unroll
    for (int h = 0; h < kHalves; ++h) *reinterpret_cast<u32x4 *>(shared_w[h] + stage_row * kPitch + stage_k) = w[h];
    __syncthreads();
    const u32x4 xf = *reinterpret_cast<const u32x4 *>(shared_x + (wave * 16 + r16) * kPitch + g * 8);
#pragma unroll
    for (int h = 0; h < kHalves; ++h)
#pragma unroll
      for (int b = 0; b < 4; ++b)
        acc[h][b] = T::mfma(*reinterpret_cast<const u32x4 *>(shared_w[h] + (b * 16 + r16) * kPitch + g * 8), xf, acc[h][b]);
  }
  const int64_t m = m0 + wave * 16 + r16;
  if (m >= p.m) return;
  const float factor = kGated ? 1.0f : row_gate<T>(p, m);
#pragma unroll
  for (int b = 0; b < 4; ++b) finish4<T, kGated>(p, m, n0 + b * 16 + 4 * g, acc[0][b], acc[kHalves - 1][b], factor);
}

template <class T, bool kGated>
void launch(const LinearParams &p, hipStream_t stream) {
  const int64_t tiles = ceil_div<int64_t>(p.m, kTile) * ceil_div<int64_t>(p.n, kTile);
  hipLaunchKernelGGL((any_kernel<T, kGated>), dim3(static_cast<uint32_t>(tiles)), dim3(kThreads), 0, stream, p);
}

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
  const int64_t strides[] = {call->input_row_stride, call->out_row_stride, call->residual_row_stride, call->gate_stride};
  for (const int64_t stride : strides)
    if (stride > kMostElements / m) return UNISERVE_REFUSE(call, "%s's arrays are too large", name);
  if (call->weight_row_stride > kMostElements / weight_rows) return UNISERVE_REFUSE(call, "%s's arrays are too large", name);
  // A call of one row has no stride to go by.
  const int64_t x_stride = m > 1 ? call->input_row_stride : k;
  const int64_t w_stride = weight_rows > 1 ? call->weight_row_stride : k;
  const int64_t out_stride = m > 1 ? call->out_row_stride : n;
  const int64_t residual_stride = m > 1 ? call->residual_row_stride : n;
  const int64_t gate_stride = m > 1 ? call->gate_stride : 0;
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
  p.rows_of_16 = k % 8 == 0 && x_stride % 8 == 0 && w_stride % 8 == 0 && aligned_to(p.x, 16) && aligned_to(p.w, 16);
  p.out_of_4 = out_stride % 4 == 0 && aligned_to(p.out, static_cast<uintptr_t>(4 * out_bytes)) &&
               (p.residual == nullptr || (residual_stride % 4 == 0 && aligned_to(p.residual, static_cast<uintptr_t>(4 * out_bytes))));
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const bool f16 = call->dtype == UNISERVE_DTYPE_F16;
  if (ceil_div<int64_t>(m, kTile) * ceil_div<int64_t>(n, kTile) > INT32_MAX)
    return UNISERVE_REFUSE(call, "%s's output has too many tiles", name);
  if (gated) f16 ? launch<F16, true>(p, s) : launch<Bf16, true>(p, s);
  else f16 ? launch<F16, false>(p, s) : launch<Bf16, false>(p, s);
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
