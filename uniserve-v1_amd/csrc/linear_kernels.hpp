// SPDX-License-Identifier: Apache-2.0
//
// The dense products' kernels of one element type and the choice among them (linear_bf16.hip and
// linear_f16.hip compile them): tiles by DMA (linear_tile.hpp), a kernel for up to four tokens, and one
// that serves every stride, extent and alignment.
#pragma once

#include "linear.hpp"
#include "linear_tile.hpp"

namespace uniserve {
namespace linear {

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
// Two workgroups a CU, or (Alone) one with a deeper ring, most of eight wavefronts, where the tiles are few.
using Tile128 = TileShape<128, 128, 2, 2, 2>;
using Tile128Alone = TileShape<128, 128, 2, 4, 3>;
using Tile96x128Alone = TileShape<96, 128, 2, 2, 4>;
using Tile128x64 = TileShape<128, 64, 2, 2, 3>;
using Tile128x64Alone = TileShape<128, 64, 4, 2, 4>;
using Tile64 = TileShape<64, 64, 2, 2, 4>;
using Tile48x64Alone = TileShape<48, 64, 1, 2, 4, 2>;
// Fewer tiles yet: a team is one wavefront with a ring of its own, and the teams share K out.
using Tile64x32 = TileShape<64, 32, 1, 1, 3, 4>;
using Tile32 = TileShape<32, 32, 1, 1, 4, 4>;
using Tile16 = TileShape<16, 16, 1, 1, 4, 8>;

/// A shape's time in microseconds, fitted to 460 measured (m, n, k) from 8 x 64 x 256 to 8192 x 2048 x 4096,
/// plain and gated: `first` for a launch and `stage` for each 64-element stage of K in each round of 256 tiles
/// (CUs), `round` for each round after the first. Shapes of two workgroups a CU (`pair` > 0) take any
/// fraction of a round, from `pair` on. The choice by it is within 1% of the best shape on average, 17% at
/// most; without the four Alone shapes 3.5% and 36%.
struct Cost {
  double first, round, stage, pair;
};

template <class S>
double cost_of(const LinearParams &p, bool gated, const Cost &c) {
  const double tiles = static_cast<double>(tiles_of<S>(p, gated));
  if (tiles * S::kThreads >= 4294967296.0) return 1e30;  // more threads than a launch's axis holds
  double rounds = tiles <= 256.0 ? 1.0 : tiles / 256.0;
  if (tiles > 256.0) rounds = c.pair == 0.0 ? static_cast<double>(ceil_div<int64_t>(tiles_of<S>(p, gated), 256)) : (rounds < c.pair ? c.pair : rounds);
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
      cost_of<Tile256>(p, kGated, {10.3, 11.3, 1.165, 0.0}),
      cost_of<Tile128>(p, kGated, {5.25, 2.5, 0.535, 1.39}),
      cost_of<Tile128Alone>(p, kGated, {4.7, 4.65, 0.41, 0.0}),
      cost_of<Tile96x128Alone>(p, kGated, {5.3, 5.0, 0.341, 0.0}),
      cost_of<Tile128x64>(p, kGated, {4.2, 1.95, 0.289, 1.65}),
      cost_of<Tile128x64Alone>(p, kGated, {4.0, 3.3, 0.268, 0.0}),
      cost_of<Tile64>(p, kGated, {3.65, 1.4, 0.186, 1.68}),
      cost_of<Tile48x64Alone>(p, kGated, {4.05, 3.0, 0.154, 0.0}),
      cost_of<Tile64x32>(p, kGated, {3.95, 2.7, 0.113, 0.0}),
      cost_of<Tile32>(p, kGated, {3.6, 2.5, 0.077, 0.0}),
      kGated ? 1e30 : cost_of<Tile16>(p, kGated, {4.0, 3.0, 0.034, 0.0}),
  };
  int best = 0;
  for (int i = 1; i < 11; ++i)
    if (costs[i] < costs[best]) best = i;
  switch (best) {
    case 0: return launch_tiles<T, kGated, Tile256>(p, stream);
    case 1: return launch_tiles<T, kGated, Tile128>(p, stream);
    case 2: return launch_tiles<T, kGated, Tile128Alone>(p, stream);
    case 3: return launch_tiles<T, kGated, Tile96x128Alone>(p, stream);
    case 4: return launch_tiles<T, kGated, Tile128x64>(p, stream);
    case 5: return launch_tiles<T, kGated, Tile128x64Alone>(p, stream);
    case 6: return launch_tiles<T, kGated, Tile64>(p, stream);
    case 7: return launch_tiles<T, kGated, Tile48x64Alone>(p, stream);
    case 8: return launch_tiles<T, kGated, Tile64x32>(p, stream);
    case 9: return launch_tiles<T, kGated, Tile32>(p, stream);
    default:
      if constexpr (!kGated) return launch_tiles<T, kGated, Tile16>(p, stream);
  }
}

}  // namespace linear
}  // namespace uniserve
