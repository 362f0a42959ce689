// SPDX-License-Identifier: Apache-2.0
//
// The dense products' kernels of one element type and the choice among them (linear_bf16.hip and
// linear_f16.hip compile them): tiles (linear_tile.hpp), by DMA or, for rows that it cannot read, through
// registers, and a kernel for up to four tokens.
#pragma once

#include "linear.hpp"
#include "linear_tile.hpp"

namespace uniserve {
namespace linear {

// ---- few tokens -----------------------------------------------------------------------------------------

constexpr int kFewThreads = 256;

/// Up to kTokens tokens at any strides and alignments: a wavefront reads one weight row (gated: its gate row
/// too) in whole kilobytes, eight elements a lane, and its lanes' sums meet at the end. Bound by the weights: 1 x
/// 2048 x 5632 (23 MB) 6.6 us, gated 1 x 5632 x 2048 (46 MB) 9.0 us, 5.1 TB/s, where a copy reaches 4.8.
template <class T, bool kGated, int kTokens>
__global__ void __launch_bounds__(kFewThreads) few_tokens_kernel(LinearParams p) {
  constexpr int kRows = kGated ? 2 : 1;
  constexpr int kUnroll = 4;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / kWave);
  const int lane = lane_id();
  const int64_t n = static_cast<int64_t>(blockIdx.x) * (kFewThreads / kWave) + wave;
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

// Through registers, for rows that the DMA cannot read.
using Any128 = TileShape<128, 128, 2, 4, 2>;
using Any64 = TileShape<64, 64, 2, 2, 2>;
using Any32 = TileShape<32, 32, 1, 1, 2, 4>;

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
  constexpr int kWaves = kFewThreads / kWave;
  hipLaunchKernelGGL((few_tokens_kernel<T, kGated, kTokens>), dim3(static_cast<uint32_t>(ceil_div<int64_t>(p.n, kWaves))),
                     dim3(kFewThreads), 0, stream, p);
}

template <class T, bool kGated>
void launch(const LinearParams &p, hipStream_t stream) {
  // Up to four tokens: 1 x 2048 x 5632 6.6 us (the best tile shape 7.3), gated 1 x 5632 x 2048 9.0 (10.2), 4 x
  // 2048 x 5632 8.2 (9.1); with eight tokens 13.2 (9.3).
  if (p.m <= 4 && p.n <= (int64_t{1} << 26) - 4) {  // a launch's axis holds fewer than 2^32 threads, a column takes 64
    if (p.m == 1) return launch_few<T, kGated, 1>(p, stream);
    if (p.m == 2) return launch_few<T, kGated, 2>(p, stream);
    return launch_few<T, kGated, 4>(p, stream);
  }
  if (!p.by_dma) {
    // Fitted as above to 273 sizes with odd k: within 0.5% of the best on average, 13% at most. 8192 x 2048 x 5631:
    // 350 us, where rows of 5632 take 150; 64 x 2048 x 4095: 17.5, and 8.5.
    const double wide = cost_of<Any128>(p, kGated, {8.7, 10.0, 0.76, 0.0}), mid = cost_of<Any64>(p, kGated, {6.1, 2.2, 0.44, 1.68}),
                 small = cost_of<Any32>(p, kGated, {6.9, 1.8, 0.17, 0.0});
    if (wide <= mid && wide <= small) return launch_tiles<T, kGated, false, Any128>(p, stream);
    if (mid <= small) return launch_tiles<T, kGated, false, Any64>(p, stream);
    return launch_tiles<T, kGated, false, Any32>(p, stream);
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
    case 0: return launch_tiles<T, kGated, true, Tile256>(p, stream);
    case 1: return launch_tiles<T, kGated, true, Tile128>(p, stream);
    case 2: return launch_tiles<T, kGated, true, Tile128Alone>(p, stream);
    case 3: return launch_tiles<T, kGated, true, Tile96x128Alone>(p, stream);
    case 4: return launch_tiles<T, kGated, true, Tile128x64>(p, stream);
    case 5: return launch_tiles<T, kGated, true, Tile128x64Alone>(p, stream);
    case 6: return launch_tiles<T, kGated, true, Tile64>(p, stream);
    case 7: return launch_tiles<T, kGated, true, Tile48x64Alone>(p, stream);
    case 8: return launch_tiles<T, kGated, true, Tile64x32>(p, stream);
    case 9: return launch_tiles<T, kGated, true, Tile32>(p, stream);
    default:
      if constexpr (!kGated) return launch_tiles<T, kGated, true, Tile16>(p, stream);
  }
}

}  // namespace linear
}  // namespace uniserve
