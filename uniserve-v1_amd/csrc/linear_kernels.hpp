// SPDX-License-Identifier: Apache-2.0
//
// The dense products' kernels of one element type and the choice among them (linear_bf16.hip and
// linear_f16.hip compile them): tiles (linear_tile.hpp), by DMA or, for rows that it cannot read, through
// registers, and a kernel for one or two tokens.
#pragma once

#include "linear.hpp"
#include "linear_tile.hpp"

namespace uniserve {
namespace linear {

// ---- few tokens -----------------------------------------------------------------------------------------

constexpr int kFewThreads = 256;

/// kTokens tokens at any strides and alignments: a wavefront reads one weight row (gated: its gate row
/// too) in whole kilobytes, eight elements a lane, and its lanes' sums meet at the end. Bound by the weights: 1 x
/// 2048 x 5632 (23 MB) 6.3 us, gated 1 x 5632 x 2048 (46 MB) 9.0 us, 5.1 TB/s, where a copy reaches 4.8; with weights
/// that come from HBM 7.2 and 10.1 us, 3.2 and 4.6 TB/s. (The last chunks one by one, each after the one before: 7.5 us
/// at K = 5632.)
template <class T, bool kGated, int kTokens>
__global__ void __launch_bounds__(kFewThreads) few_tokens_kernel(LinearParams p) {
  constexpr int kRows = kGated ? 2 : 1;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / kWave);
  const int lane = lane_id();
  const int64_t n = static_cast<int64_t>(blockIdx.x) * (kFewThreads / kWave) + wave;
  if (n >= p.n) return;
  const uint16_t *row[kRows], *token[kTokens];
#pragma unroll
  for (int r = 0; r < kRows; ++r) row[r] = p.w + (n + r * p.n) * p.w_stride;
#pragma unroll
  for (int t = 0; t < kTokens; ++t) token[t] = p.x + t * p.x_stride;
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
  // `count` chunks of a kilobyte a row from `at` on, all their loads first.
  constexpr int64_t kChunk = kWave * 8;
  int64_t at = lane * 8;
  auto chunks = [&](auto count_of, auto load) {
    constexpr int kCount = decltype(count_of)::value;
    u32x4 x[kCount][kTokens], w[kCount][kRows];
#pragma unroll
    for (int u = 0; u < kCount; ++u) {
#pragma unroll
      for (int r = 0; r < kRows; ++r) w[u][r] = load(row[r], at + u * kChunk);
#pragma unroll
      for (int t = 0; t < kTokens; ++t) x[u][t] = load(token[t], at + u * kChunk);
    }
#pragma unroll
    for (int u = 0; u < kCount; ++u)
#pragma unroll
      for (int r = 0; r < kRows; ++r)
#pragma unroll
        for (int t = 0; t < kTokens; ++t) add(x[u][t], w[u][r], sum[r][t]);
    at += kCount * kChunk;
  };
  const auto inside = [](const uint16_t *from, int64_t i) {
    u32x4 v;
    __builtin_memcpy(&v, from + i, 16);
    return v;
  };
  const auto at_end = [&](const uint16_t *from, int64_t i) { return load8(from, i, p.k); };
  int64_t left = p.k;
  for (; left >= 4 * kChunk; left -= 4 * kChunk) chunks(std::integral_constant<int, 4>{}, inside);
  if (left >= 2 * kChunk) {
    chunks(std::integral_constant<int, 2>{}, inside);
    left -= 2 * kChunk;
  }
  if (left > kChunk) chunks(std::integral_constant<int, 2>{}, at_end);
  else if (left > 0) chunks(std::integral_constant<int, 1>{}, at_end);
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
  if (lane < kTokens) finish1<T, kGated>(p, lane, n, v, g);
}

// ---- the choice -------------------------------------------------------------------------------------------

using Tile256 = TileShape<256, 256, 2, 4, 2>;
using Tile192x256 = TileShape<192, 256, 2, 4, 2>;
using Tile128x256 = TileShape<128, 256, 2, 4, 3>;
using Tile192x128 = TileShape<192, 128, 4, 2, 3>;
// Two workgroups a CU, or (Alone) one with a deeper ring, where the tiles are few.
using Tile128 = TileShape<128, 128, 2, 2, 2>;
using Tile128Alone = TileShape<128, 128, 2, 4, 3>;
using Tile96x128Alone = TileShape<96, 128, 2, 2, 4>;
using Tile128x64Alone = TileShape<128, 64, 4, 2, 4>;
using Tile64 = TileShape<64, 64, 2, 2, 4>;
using Tile48x64Alone = TileShape<48, 64, 1, 2, 4, 2>;
// Fewer tiles yet: a team is one wavefront with a ring of its own, and the teams share K out.
using Tile32x64Alone = TileShape<32, 64, 1, 1, 3, 4>;
using Tile32Alone = TileShape<32, 32, 1, 1, 4, 4>;
using Tile16x32Alone = TileShape<16, 32, 1, 1, 4, 4>;
using Tile16 = TileShape<16, 16, 1, 1, 4, 4>;

// Through registers, for rows that the DMA cannot read.
using Any128 = TileShape<128, 128, 2, 4, 2>;
using Any96x128 = TileShape<96, 128, 2, 2, 2>;
using Any64 = TileShape<64, 64, 2, 2, 2>;
using Any32 = TileShape<32, 32, 1, 1, 2, 4>;
using Any16x32 = TileShape<16, 32, 1, 1, 2, 4>;

/// A shape's time in microseconds, fitted to 1056 measured sizes, plain and gated (m from 3 to 8192, n from 64 to
/// 11264, k from 256 to 5632): `first` for a launch, `round` for each round of 256 tiles (CUs) after the first, `stage`
/// for each 64-element stage of K in each round. Of shapes of two workgroups a CU (`shared` > 0) 512 tiles take 2
/// `shared` a stage; of the tiles past whole 512s up to 256 take `stage`, more `least` times `shared`. The choice by it
/// takes 0.5% longer than the best shape on average, 20% at most. Each shape is chosen at 19 (Tile48x64Alone) to 138
/// (Tile16x32Alone) of these sizes; the choice without it takes 2% (Tile128x256) to 20% (Tile64) longer there on
/// average, 14 to 42% at most. Without the 192 x 256, 128 x 256 and 192 x 128 tiles: 2.2% and 35% over all sizes.
struct Cost {
  double first, round, stage, shared, least;
};

template <class S>
double cost_of(const LinearParams &p, bool gated, const Cost &c) {
  const int64_t tiles = tiles_of<S>(p, gated);
  if (static_cast<double>(tiles) * S::kThreads >= 4294967296.0) return 1e30;  // more threads than a launch's axis holds
  const double rounds = static_cast<double>(ceil_div<int64_t>(tiles, 256)), stages = static_cast<double>(ceil_div<int64_t>(p.k, kStageK));
  double per_stage = c.stage * rounds;
  if (c.shared > 0.0) {
    const int64_t rest = tiles % 512;
    per_stage = 2.0 * c.shared * static_cast<double>(tiles / 512) + (rest == 0 ? 0.0 : rest <= 256 ? c.stage : c.least * c.shared);
  }
  return c.first + c.round * (rounds - 1.0) + per_stage * stages;
}

template <int kShapes>
int cheapest(const double (&costs)[kShapes]) {
  int best = 0;
  for (int i = 1; i < kShapes; ++i)
    if (costs[i] < costs[best]) best = i;
  return best;
}

template <class T, bool kGated, int kTokens>
void launch_few(const LinearParams &p, hipStream_t stream) {
  constexpr int kWaves = kFewThreads / kWave;
  hipLaunchKernelGGL((few_tokens_kernel<T, kGated, kTokens>), dim3(static_cast<uint32_t>(ceil_div<int64_t>(p.n, kWaves))),
                     dim3(kFewThreads), 0, stream, p);
}

template <class T, bool kGated>
void launch(const LinearParams &p, hipStream_t stream) {
  // One or two tokens: 1 x 2048 x 5632 6.3 us (the best tile shape 6.8), gated 1 x 5632 x 2048 9.0 (10.1), 2 x 512 x
  // 2048 3.1 (4.2); four by the same kernel 4 x 2048 x 5632 8.1 (6.9), 4 x 4096 x 2048 6.1 (5.9).
  if (p.m <= 2 && p.n <= (int64_t{1} << 26) - 4) {  // a launch's axis holds fewer than 2^32 threads, a column takes 64
    if (p.m == 1) return launch_few<T, kGated, 1>(p, stream);
    return launch_few<T, kGated, 2>(p, stream);
  }
  if (!p.by_dma) {
    // Fitted as above to 415 sizes with odd k: 0.6% longer than the best on average, 17% at most; without Any96x128
    // and Any16x32 8.0% and 34%. Each is chosen at 44 to 160 of them, where the choice without it takes 8 to 24% longer.
    // 8192 x 2048 x 5631: 306 us, where rows of 5632 take 150; 64 x 2048 x 4095: 12.2, and 7.5. How much of that the
    // loads cost, each over two pieces of a line, and how much the smaller tiles is not known.
    const double costs[] = {
        cost_of<Any128>(p, kGated, {6.12, 4.81, 0.727}),
        cost_of<Any96x128>(p, kGated, {6.95, 1.77, 0.667}),
        cost_of<Any64>(p, kGated, {4.33, 0.812, 0.473, 0.294, 2.11}),
        cost_of<Any32>(p, kGated, {4.4, 0.734, 0.173}),
        cost_of<Any16x32>(p, kGated, {4.09, 0.383, 0.124}),
    };
    switch (cheapest(costs)) {
      case 0: return launch_tiles<T, kGated, false, Any128>(p, stream);
      case 1: return launch_tiles<T, kGated, false, Any96x128>(p, stream);
      case 2: return launch_tiles<T, kGated, false, Any64>(p, stream);
      case 3: return launch_tiles<T, kGated, false, Any32>(p, stream);
      default: return launch_tiles<T, kGated, false, Any16x32>(p, stream);
    }
  }
  const double costs[] = {
      cost_of<Tile256>(p, kGated, {10.3, 9.4, 1.311}),
      cost_of<Tile192x256>(p, kGated, {7.87, 7.8, 1.045}),
      cost_of<Tile128x256>(p, kGated, {6.39, 5.74, 0.763}),
      cost_of<Tile192x128>(p, kGated, {5.21, 4.98, 0.599}),
      cost_of<Tile128>(p, kGated, {4.46, 2.07, 0.611, 0.436, 1.75}),
      cost_of<Tile128Alone>(p, kGated, {4.5, 3.91, 0.434}),
      cost_of<Tile96x128Alone>(p, kGated, {4.87, 3.98, 0.356}),
      cost_of<Tile128x64Alone>(p, kGated, {4.06, 2.87, 0.28}),
      cost_of<Tile64>(p, kGated, {3.67, 0.957, 0.184, 0.168, 1.9}),
      cost_of<Tile48x64Alone>(p, kGated, {3.81, 2.54, 0.151}),
      cost_of<Tile32x64Alone>(p, kGated, {3.51, 2.44, 0.118}),
      cost_of<Tile32Alone>(p, kGated, {3.33, 2.17, 0.08}),
      cost_of<Tile16x32Alone>(p, kGated, {3.22, 2.09, 0.06}),
      kGated ? 1e30 : cost_of<Tile16>(p, kGated, {3.22, 0.707, 0.034, 0.038, 1.78}),
  };
  switch (cheapest(costs)) {
    case 0: return launch_tiles<T, kGated, true, Tile256>(p, stream);
    case 1: return launch_tiles<T, kGated, true, Tile192x256>(p, stream);
    case 2: return launch_tiles<T, kGated, true, Tile128x256>(p, stream);
    case 3: return launch_tiles<T, kGated, true, Tile192x128>(p, stream);
    case 4: return launch_tiles<T, kGated, true, Tile128>(p, stream);
    case 5: return launch_tiles<T, kGated, true, Tile128Alone>(p, stream);
    case 6: return launch_tiles<T, kGated, true, Tile96x128Alone>(p, stream);
    case 7: return launch_tiles<T, kGated, true, Tile128x64Alone>(p, stream);
    case 8: return launch_tiles<T, kGated, true, Tile64>(p, stream);
    case 9: return launch_tiles<T, kGated, true, Tile48x64Alone>(p, stream);
    case 10: return launch_tiles<T, kGated, true, Tile32x64Alone>(p, stream);
    case 11: return launch_tiles<T, kGated, true, Tile32Alone>(p, stream);
    case 12: return launch_tiles<T, kGated, true, Tile16x32Alone>(p, stream);
    default:
      if constexpr (!kGated) return launch_tiles<T, kGated, true, Tile16>(p, stream);
  }
}

}  // namespace linear
}  // namespace uniserve
