// SPDX-License-Identifier: Apache-2.0
//
// The dense products on gfx950 (include/uniserve_linear.h states the operators): the entries, their
// refusals, the choice of the kernel, and the kernel that serves every stride and extent.
#include "linear.hpp"
#include "linear_tile.hpp"

namespace uniserve {
namespace linear {
namespace {

constexpr int kThreads = 256;
constexpr int kTile = 64;   // tokens and output columns of a workgroup
constexpr int kStep = 32;   // K elements a step
constexpr int kPitch = 40;  // elements between tile rows in LDS (80 bytes: 16 rows on distinct banks)

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
  u32x4 x, w[kHalves];
  auto load = [&](int64_t k) {
    x = load8(x_row, k + stage_k, p.k);
#pragma unroll
    for (int h = 0; h < kHalves; ++h) w[h] = load8(w_row[h], k + stage_k, p.k);
  };
  load(0);
  for (int64_t k = 0; k < p.k; k += kStep) {
    __syncthreads();
    *reinterpret_cast<u32x4 *>(shared_x + stage_row * kPitch + stage_k) = x;
#pragma unroll
    for (int h = 0; h < kHalves; ++h) *reinterpret_cast<u32x4 *>(shared_w[h] + stage_row * kPitch + stage_k) = w[h];
    __syncthreads();
    if (k + kStep < p.k) load(k + kStep);
    const u32x4 xf = *reinterpret_cast<const u32x4 *>(shared_x + (wave * 16 + r16) * kPitch + g * 8);
#pragma unroll
    for (int h = 0; h < kHalves; ++h)
#pragma unroll
      for (int b = 0; b < 4; ++b)
        acc[h][b] = T::mfma(*reinterpret_cast<const u32x4 *>(shared_w[h] + (b * 16 + r16) * kPitch + g * 8), xf, acc[h][b]);
  }
  // The wavefront's sums through its own part of LDS, 16 tokens by 64 columns, so that a lane holds eight
  // columns of a token.
  constexpr int kBlocks = 4;
  __shared__ __align__(16) float sums[4][16][kBlocks * 16 + 4];
  const int group = lane & 7;
  const int64_t n = n0 + group * 8;
  const Columns8<T, kGated> columns(p, n);
  floatx4 v[kHalves][2][2];
#pragma unroll
  for (int h = 0; h < kHalves; ++h) {
#pragma unroll
    for (int b = 0; b < kBlocks; ++b) *reinterpret_cast<floatx4 *>(&sums[wave][r16][b * 16 + 4 * g]) = acc[h][b];
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) v[h][i][j] = *reinterpret_cast<const floatx4 *>(&sums[wave][i * 8 + lane / 8][group * 8 + j * 4]);
    __builtin_amdgcn_wave_barrier();
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int64_t m = m0 + wave * 16 + i * 8 + lane / 8;
    if (m >= p.m) continue;
    typename Columns8<T, kGated>::template Extras<1> extras;
    columns.load(p, {m}, n, extras);
    columns.finish(p, m, n, v[0][i], v[kHalves - 1][i], extras.residual[0], extras.factor[0]);
  }
}

// ---- few tokens -----------------------------------------------------------------------------------------

/// Up to kTokens tokens at any strides and alignments: a wavefront reads one weight row (gated: its gate row
/// too) in whole kilobytes, eight elements a lane, and its lanes' sums meet at the end.
template <class T, bool kGated, int kTokens>
__global__ void __launch_bounds__(kThreads) few_tokens_kernel(LinearParams p) {
  constexpr int kRows = kGated ? 2 : 1;
  constexpr int kUnroll = 4;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / kWave);
  const int lane = lane_id();
  const int64_t n = static_cast<int64_t>(blockIdx.x) * (kThreads / kWave) + wave;
  if (n >= p.n) return;
  const uint16_t *row[kRows], *token[kTokens];
#pragma unroll
  for (int r = 0; r < kRows; ++r) row[r] = p.w + (n + r * p.n) * p.w_stride;
#pragma unroll
  for (int t = 0; t < kTokens; ++t) token[t] = p.x + (t < p.m ? t : p.m - 1) * p.x_stride;
  float sum[kRows][kTokens];
#pragma unroll
  for (int r = 0; r < kRows; ++r)
#pragma unroll
    for (int t = 0; t < kTokens; ++t) sum[r][t] = 0.0f;
  auto add = [&](const u32x4 &x, const u32x4 &w, float &into) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      into = __builtin_fmaf(T::low(x[i]), T::low(w[i]), into);
      into = __builtin_fmaf(T::high(x[i]), T::high(w[i]), into);
    }
  };
  constexpr int64_t kChunk = kWave * 8;
  int64_t at = lane * 8;
  for (; at - lane * 8 + kUnroll * kChunk <= p.k; at += kUnroll * kChunk) {
    u32x4 x[kUnroll][kTokens], w[kUnroll][kRows];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
#pragma unroll
      for (int r = 0; r < kRows; ++r) __builtin_memcpy(&w[u][r], row[r] + at + u * kChunk, 16);
#pragma unroll
      for (int t = 0; t < kTokens; ++t) __builtin_memcpy(&x[u][t], token[t] + at + u * kChunk, 16);
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
#pragma unroll
      for (int r = 0; r < kRows; ++r)
#pragma unroll
        for (int t = 0; t < kTokens; ++t) add(x[u][t], w[u][r], sum[r][t]);
  }
  for (; at < p.k; at += kChunk) {
    u32x4 w[kRows];
#pragma unroll
    for (int r = 0; r < kRows; ++r) w[r] = load8(row[r], at, p.k);
#pragma unroll
    for (int t = 0; t < kTokens; ++t) {
      const u32x4 x = load8(token[t], at, p.k);
#pragma unroll
      for (int r = 0; r < kRows; ++r) add(x, w[r], sum[r][t]);
    }
  }
#pragma unroll
  for (int offset = kWave / 2; offset > 0; offset /= 2)
#pragma unroll
    for (int r = 0; r < kRows; ++r)
#pragma unroll
      for (int t = 0; t < kTokens; ++t) sum[r][t] += __shfl_xor(sum[r][t], offset);
  // Lane t finishes token t.
  float v = sum[0][0], g = sum[kRows - 1][0];
#pragma unroll
  for (int t = 1; t < kTokens; ++t) {
    v = lane == t ? sum[0][t] : v;
    g = lane == t ? sum[kRows - 1][t] : g;
  }
  if (lane < kTokens && lane < p.m) finish1<T, kGated>(p, lane, n, v, g);
}

// ---- the choice -------------------------------------------------------------------------------------------

using Tile256 = TileShape<256, 256, 2, 4, 2>;
using Tile128 = TileShape<128, 128, 2, 2, 2>;
using Tile128x64 = TileShape<128, 64, 2, 2, 3>;
using Tile64 = TileShape<64, 64, 2, 2, 4>;
// Few tiles: a team is one wavefront with a ring of its own, and the teams share K out.
using Tile64x32 = TileShape<64, 32, 1, 1, 3, 4>;
using Tile32 = TileShape<32, 32, 1, 1, 4, 4>;
using Tile16 = TileShape<16, 16, 1, 1, 4, 8>;

/// A shape's time in microseconds, fitted to 300 measured (m, n, k) from 1 x 64 x 256 to 8192 x 5632 x 4096:
/// `first` for a launch, `stage` for each 64-element stage of K, both once for every 256 tiles (CUs) begun -
/// shapes of two workgroups a CU go by the fraction - and `round` for each further 256. The choice by it is
/// within 0.4% of the best of these shapes on average, 12% at most.
struct Cost {
  double first, round, stage;
  bool paired;
};

template <class S>
double cost_of(const LinearParams &p, bool gated, const Cost &c) {
  const double tiles = static_cast<double>(tiles_of<S>(p, gated));
  if (tiles * S::kThreads >= 4294967296.0) return 1e30;  // more threads than a launch's axis holds
  const double rounds = c.paired ? (tiles > 256.0 ? tiles / 256.0 : 1.0) : static_cast<double>(ceil_div<int64_t>(tiles_of<S>(p, gated), 256));
  return c.first + c.round * (rounds - 1.0) + c.stage * static_cast<double>(ceil_div<int64_t>(p.k, kStageK)) * rounds;
}

template <class T, bool kGated, int kTokens>
void launch_few(const LinearParams &p, hipStream_t stream) {
  constexpr int kWaves = kThreads / kWave;
  hipLaunchKernelGGL((few_tokens_kernel<T, kGated, kTokens>), dim3(static_cast<uint32_t>(ceil_div<int64_t>(p.n, kWaves))),
                     dim3(kThreads), 0, stream, p);
}

template <class T, bool kGated>
void launch(const LinearParams &p, hipStream_t stream) {
  // Up to four tokens: 1 x 2048 x 5632 6.6 us (the best tile shape 7.3), gated 1 x 5632 x 2048 9.0 (10.2), 4 x
  // 2048 x 5632 8.2 (9.1); with eight tokens 13.2 (9.3).
  if (p.m == 1) return launch_few<T, kGated, 1>(p, stream);
  if (p.m == 2) return launch_few<T, kGated, 2>(p, stream);
  if (p.m <= 4) return launch_few<T, kGated, 4>(p, stream);
  if (!p.by_dma) {
    const int64_t tiles = ceil_div<int64_t>(p.m, kTile) * ceil_div<int64_t>(p.n, kTile);
    hipLaunchKernelGGL((any_kernel<T, kGated>), dim3(static_cast<uint32_t>(tiles)), dim3(kThreads), 0, stream, p);
    return;
  }
  const double costs[] = {
      cost_of<Tile256>(p, kGated, {9.0, 8.0, 1.25, false}),    cost_of<Tile128>(p, kGated, {4.6, 2.0, 0.57, true}),
      cost_of<Tile128x64>(p, kGated, {4.2, 1.6, 0.29, true}),  cost_of<Tile64>(p, kGated, {3.8, 1.4, 0.18, true}),
      cost_of<Tile64x32>(p, kGated, {3.8, 3.0, 0.115, false}), cost_of<Tile32>(p, kGated, {3.6, 2.4, 0.083, false}),
      kGated ? 1e30 : cost_of<Tile16>(p, kGated, {4.0, 2.6, 0.045, false}),
  };
  int best = 0;
  for (int i = 1; i < 7; ++i)
    if (costs[i] < costs[best]) best = i;
  switch (best) {
    case 0: return launch_tiles<T, kGated, Tile256>(p, stream);
    case 1: return launch_tiles<T, kGated, Tile128>(p, stream);
    case 2: return launch_tiles<T, kGated, Tile128x64>(p, stream);
    case 3: return launch_tiles<T, kGated, Tile64>(p, stream);
    case 4: return launch_tiles<T, kGated, Tile64x32>(p, stream);
    case 5: return launch_tiles<T, kGated, Tile32>(p, stream);
    default:
      if constexpr (!kGated) return launch_tiles<T, kGated, Tile16>(p, stream);
  }
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
  // The tile kernels' DMA reads whole 16 bytes at aligned addresses, a tile's rows within 32-bit offsets.
  constexpr int64_t kMostStride = int64_t{1} << 22;
  p.by_dma = k % 8 == 0 && x_stride % 8 == 0 && w_stride % 8 == 0 && aligned_to(p.x, 16) && aligned_to(p.w, 16) &&
             x_stride <= kMostStride && w_stride <= kMostStride;
  p.out_of_8 = out_stride * out_bytes % 16 == 0 && aligned_to(p.out, 16) &&
               (p.residual == nullptr || (residual_stride * out_bytes % 16 == 0 && aligned_to(p.residual, 16)));
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const bool f16 = call->dtype == UNISERVE_DTYPE_F16;
  if (ceil_div<int64_t>(m, kTile) * ceil_div<int64_t>(n, kTile) > (int64_t{1} << 32) / kThreads - 1)
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
