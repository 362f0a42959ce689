// SPDX-License-Identifier: Apache-2.0
//
// Low-rank adapters beside the dense products: the first factor's kernel, which leaves each row's rank values in the
// workspace, and the second factor's product, which the product kernels add to their sums behind the walk over K.
//
// Rows of one adapter are found where they are used: a wavefront takes the adapters that its rows name in turn, each
// once, multiplies that adapter's factor by all of its rows and keeps the sums of the rows that name it (a matrix
// instruction's columns do not mix, so the others' are only discarded). No sort of the rows, no list of segments.
#pragma once

#include "linear.hpp"

namespace uniserve {
namespace linear {

/// The adapter of row t, or -1.
__device__ __forceinline__ int adapter_of(const AdapterParams &p, int64_t t) {
  const int a = t < p.m ? p.adapter[t] : -1;
  return a >= 0 && a < p.adapters ? a : -1;
}

/// Elements at .. at + 7 of a row of `width`, zeros past its end. kWhole: of whole 16-byte pieces.
template <bool kWhole>
__device__ __forceinline__ u32x4 load8_of(const uint16_t *row, int64_t at, int64_t width) {
  if constexpr (kWhole) return at < width ? *reinterpret_cast<const u32x4 *>(row + at) : u32x4{0, 0, 0, 0};
  else return load8(row, at, width);
}

// ---- the first factor -------------------------------------------------------------------------------------

/// 16 rows by kBlocks blocks of 16 ranks a workgroup, whose kWaves wavefronts take the 64-element stages of K in
/// turn and add their sums in LDS. blockIdx.y: the rank blocks; blockIdx.z: with gridDim.z > 1 the workgroups
/// share out the adapters that the 16 rows name. kWide: groups of 32 ranks (LowLayout), two blocks each.
template <class T, bool kWhole, bool kWide, int kWaves, int kBlocks>
__global__ void __launch_bounds__(kWaves *kWave) low_rank_kernel(AdapterParams p, int halves) {
  constexpr int kPerGroup = kWide ? 2 : 1;
  static_assert(kBlocks % kPerGroup == 0, "whole groups");
  __shared__ float sums[kWaves][kBlocks][16][16];  // of rank block, row, rank
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / kWave);
  const int lane = lane_id();
  const int r16 = lane & 15, g = lane >> 4;
  const int64_t m0 = static_cast<int64_t>(blockIdx.x) * 16;
  const LowLayout layout(p.rank);
  const int first_block = static_cast<int>(blockIdx.y) * kBlocks;
  const int all_blocks = halves * layout.groups * kPerGroup;
  const uint16_t *x = p.x + (m0 + r16 < p.m ? m0 + r16 : p.m - 1) * p.x_stride;
  // The lane's row of each block in an adapter's factor (past the rank: the last one, its value is dropped).
  int64_t row[kBlocks];
#pragma unroll
  for (int q = 0; q < kBlocks; ++q) {
    const int block = first_block + q < all_blocks ? first_block + q : all_blocks - 1;
    const int half = block / (layout.groups * kPerGroup), in_half = block % (layout.groups * kPerGroup) * 16 + r16;
    row[q] = (half * p.rank + (in_half < p.rank ? in_half : p.rank - 1)) * p.down_row_stride;
  }
  const int mine = adapter_of(p, m0 + r16);
  uint32_t remaining = static_cast<uint32_t>(ballot(mine >= 0)) & 0xffffu;
  for (int turn = 0; remaining != 0; turn = turn + 1 == static_cast<int>(gridDim.z) ? 0 : turn + 1) {
    const int current = __builtin_amdgcn_readlane(mine, __ffs(static_cast<int>(remaining)) - 1);
    remaining &= ~static_cast<uint32_t>(ballot(mine == current));
    if (turn != static_cast<int>(blockIdx.z)) continue;
    const uint16_t *down = p.down + current * p.down_stride;
    floatx4 acc[kBlocks];
#pragma unroll
    for (int q = 0; q < kBlocks; ++q) acc[q] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
    // A lane's 16 bytes are chunks g and g + 4 of a stage's eight, in both operands.
    for (int64_t k = wave * 64; k < p.k; k += kWaves * 64) {
      u32x4 xs[2], ws[kBlocks][2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        xs[i] = load8_of<kWhole>(x, k + (g + 4 * i) * 8, p.k);
#pragma unroll
        for (int q = 0; q < kBlocks; ++q) ws[q][i] = load8_of<kWhole>(down + row[q], k + (g + 4 * i) * 8, p.k);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int q = 0; q < kBlocks; ++q) acc[q] = T::mfma(ws[q][i], xs[i], acc[q]);
    }
    __syncthreads();  // (the adapter before: its sums have been read)
#pragma unroll
    for (int q = 0; q < kBlocks; ++q) *reinterpret_cast<floatx4 *>(&sums[wave][q][r16][4 * g]) = acc[q];
    __syncthreads();
    // A group's values of one row on neighbouring lanes.
    constexpr int kLanes = kPerGroup * 16;
    const float scale = p.scales == nullptr ? 1.0f : p.scales[current];
    for (int i = threadIdx.x; i < kBlocks / kPerGroup * 16 * kLanes; i += kWaves * kWave) {
      const int rank = i % kLanes, r = i / kLanes % 16, of = i / kLanes / 16;
      const int group = first_block / kPerGroup + of;
      float v = 0.0f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) v += sums[w][of * kPerGroup + rank / 16][r][rank % 16];
      const int in_half = group % layout.groups * layout.width + rank;
      v = in_half < p.rank ? v * scale : 0.0f;
      float factor = 1.0f;
      if constexpr (std::is_same<T, F16>::value) {
        // The power of two that brings the group's largest value to [1, 2).
        float most = __builtin_fabsf(v);
#pragma unroll
        for (int offset = kLanes / 2; offset > 0; offset /= 2) most = __builtin_fmaxf(most, __shfl_xor(most, offset));
        if (most > 0.0f && most < __builtin_inff()) {
          const int power = __builtin_amdgcn_frexp_expf(most) - 1;
          v = __builtin_ldexpf(v, -power);
          factor = __builtin_ldexpf(1.0f, power < -126 ? -126 : power);
          if (power < -126) v = __builtin_ldexpf(v, power + 126);
        }
      }
      const uint16_t high = T::from_f32(v);
      const float error = v - T::to_f32(high);
      const int owner = __shfl(mine, r);  // (the lanes of every wavefront hold the 16 rows' adapters)
      if (owner != current || rank >= layout.width || first_block + of * kPerGroup >= all_blocks) continue;
      char *at = p.low + (m0 + r) * layout.row_bytes(halves) + static_cast<int64_t>(group) * layout.group_bytes();
      reinterpret_cast<uint16_t *>(at)[rank] = high;
      reinterpret_cast<uint16_t *>(at)[layout.width + rank] = T::from_f32(error == error ? error : 0.0f);
      if (std::is_same<T, F16>::value && rank == 0) *reinterpret_cast<float *>(at + 4 * layout.width) = factor;
    }
  }
}

template <class T, bool kWhole, bool kWide, int kWaves, int kBlocks>
void launch_low_rank_kernel(const AdapterParams &p, int halves, int shares, hipStream_t stream) {
  const LowLayout layout(p.rank);
  const int blocks = halves * layout.groups * (kWide ? 2 : 1);
  const dim3 grid(static_cast<uint32_t>(ceil_div<int64_t>(p.m, 16)), static_cast<uint32_t>(ceil_div(blocks, kBlocks)), static_cast<uint32_t>(shares));
  hipLaunchKernelGGL((low_rank_kernel<T, kWhole, kWide, kWaves, kBlocks>), grid, dim3(kWaves * kWave), 0, stream, p, halves);
}

template <class T>
void launch_low_rank(const AdapterParams &p, bool gated, hipStream_t stream) {
  const int halves = gated ? 2 : 1;
  const bool wide = LowLayout(p.rank).width == 32;
  if (p.m <= 256) {
    const int shares = p.m < 16 ? static_cast<int>(p.m) : 16;
    if (wide) p.down_whole ? launch_low_rank_kernel<T, true, true, 16, 2>(p, halves, shares, stream)
                           : launch_low_rank_kernel<T, false, true, 16, 2>(p, halves, shares, stream);
    else p.down_whole ? launch_low_rank_kernel<T, true, false, 16, 1>(p, halves, shares, stream)
                      : launch_low_rank_kernel<T, false, false, 16, 1>(p, halves, shares, stream);
    return;
  }
  if (wide) p.down_whole ? launch_low_rank_kernel<T, true, true, 4, 4>(p, halves, 1, stream)
                         : launch_low_rank_kernel<T, false, true, 4, 4>(p, halves, 1, stream);
  else p.down_whole ? launch_low_rank_kernel<T, true, false, 4, 2>(p, halves, 1, stream)
                    : launch_low_rank_kernel<T, false, false, 4, 2>(p, halves, 1, stream);
}

// ---- the second factor ------------------------------------------------------------------------------------

/// Adds the adapters' products to a wavefront's sums: token blocks mb from row m_first on, weight blocks nb from
/// column n_first on (gated: half of them the up rows', then the same columns' gate rows), one adapter that its rows
/// name after the other; of `teams` wavefronts with the same sums, which are added up later, each takes its share of
/// the adapters. Two matrix instructions per 32 ranks, over the values and over their errors, or, up to rank 16,
/// one over both.
template <class T, bool kGated, int NB, int MB>
__device__ __forceinline__ void add_low_rank(const AdapterParams &p, floatx4 (&acc)[NB][MB], int64_t m_first, int64_t n_first, int team,
                                             int teams) {
  const int lane = lane_id();
  const int r16 = lane & 15, g = lane >> 4;
  const LowLayout layout(p.rank);
  constexpr int kHalves = kGated ? 2 : 1, kPerHalf = NB / kHalves;
  int mine[MB];
  uint32_t remaining[MB];
#pragma unroll
  for (int b = 0; b < MB; ++b) mine[b] = adapter_of(p, m_first + b * 16 + r16);
#pragma unroll
  for (int b = 0; b < MB; ++b) remaining[b] = static_cast<uint32_t>(ballot(mine[b] >= 0)) & 0xffffu;
  int64_t row[NB];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    const int64_t n = n_first + nb % kPerHalf * 16 + r16;
    row[nb] = ((n < p.n ? n : p.n - 1) + nb / kPerHalf * p.n) * p.up_row_stride;
  }
  const int64_t row_bytes = layout.row_bytes(kHalves);
  // The lane's chunk of eight ranks in the up rows, and its chunks of the values and of the errors (`both`: the
  // chunk that its place holds of either, in one operand).
  const bool both = layout.width <= 16;
  const int up_chunk = layout.width == 32 ? g : layout.width == 16 ? g & 1 : 0;
  const int low_at = 16 * g;  // bytes; the errors follow the values
  const bool held = layout.width >= 16 || g < 2;
  for (;;) {
    int current = -1;
#pragma unroll
    for (int b = MB - 1; b >= 0; --b)
      if (remaining[b] != 0) current = __builtin_amdgcn_readlane(mine[b], __ffs(static_cast<int>(remaining[b])) - 1);
    if (current < 0) break;
#pragma unroll
    for (int b = 0; b < MB; ++b) remaining[b] &= ~static_cast<uint32_t>(ballot(mine[b] == current));
    if (current % teams != team) continue;  // (by its number: a row's sums do not depend on the other rows' adapters)
    const uint16_t *up = p.up + current * p.up_stride;
    for (int group = 0; group < layout.groups; ++group) {
      const int64_t at = group * 32 + up_chunk * 8;
      u32x4 ws[NB];
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        if (p.up_whole) ws[nb] = load8_of<true>(up + row[nb], at, p.rank);
        else ws[nb] = load8_of<false>(up + row[nb], at, p.rank);
        if (!held) ws[nb] = u32x4{0, 0, 0, 0};
      }
#pragma unroll
      for (int b = 0; b < MB; ++b) {
        if (ballot(mine[b] == current) == 0) continue;
        const bool own = mine[b] == current;
#pragma unroll
        for (int h = 0; h < kHalves; ++h) {
          const char *low = p.low + (m_first + b * 16 + r16) * row_bytes + (h * layout.groups + group) * layout.group_bytes();
          u32x4 values{0, 0, 0, 0}, errors{0, 0, 0, 0};
          float factor = 1.0f;
          if (own) {
            if (held) values = *reinterpret_cast<const u32x4 *>(low + low_at);
            if (!both) errors = *reinterpret_cast<const u32x4 *>(low + 64 + low_at);
            if constexpr (std::is_same<T, F16>::value) factor = *reinterpret_cast<const float *>(low + 4 * layout.width);
          }
#pragma unroll
          for (int j = 0; j < kPerHalf; ++j) {
            const int nb = h * kPerHalf + j;
            floatx4 part = T::mfma(ws[nb], values, floatx4{0.0f, 0.0f, 0.0f, 0.0f});
            if (!both) part = T::mfma(ws[nb], errors, part);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              if constexpr (std::is_same<T, F16>::value) acc[nb][b][i] = own ? __builtin_fmaf(part[i], factor, acc[nb][b][i]) : acc[nb][b][i];
              else acc[nb][b][i] = own ? acc[nb][b][i] + part[i] : acc[nb][b][i];
            }
          }
        }
      }
    }
  }
}

/// The same for column n's (gated: and its gate row's) sums of the first rows, whose lanes' sums meet later: a lane
/// adds every 64th rank.
template <class T, int kRows, int kTokens>
__device__ __forceinline__ void start_low_rank(const AdapterParams &p, int64_t n, float (&sum)[kRows][kTokens]) {
  const LowLayout layout(p.rank);
#pragma unroll
  for (int t = 0; t < kTokens; ++t) {
    const int adapter = adapter_of(p, t);
    if (adapter < 0) continue;
    for (int rank = lane_id(); rank < p.rank; rank += kWave) {
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        const char *low = p.low + t * layout.row_bytes(kRows) + (r * layout.groups + rank / layout.width) * layout.group_bytes();
        const uint16_t *values = reinterpret_cast<const uint16_t *>(low) + rank % layout.width;
        float v = T::to_f32(values[0]) + T::to_f32(values[layout.width]);
        if constexpr (std::is_same<T, F16>::value) v *= *reinterpret_cast<const float *>(low + 4 * layout.width);
        const uint16_t w = p.up[adapter * p.up_stride + (n + r * p.n) * p.up_row_stride + rank];
        sum[r][t] = __builtin_fmaf(v, T::to_f32(w), sum[r][t]);
      }
    }
  }
}

}  // namespace linear
}  // namespace uniserve
