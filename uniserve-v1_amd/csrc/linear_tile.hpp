// SPDX-License-Identifier: Apache-2.0
//
// The dense products by tiles: a workgroup owns kBM tokens by kBN weight rows (gated: kBN / 2 columns,
// their up and their gate rows) and walks K in stages of 64 elements.
//
// A stage's rows (128 bytes each) arrive in LDS by DMA (`global_load_lds_dwordx4`, eight lanes a row),
// kStages stages in a ring. The loads are inline assembly, invisible to the compiler, waited for by exact
// counts. Chunk c (16 bytes) of row r lies at chunk c ^ (r / 2) % 8 of the row, so the 16 lanes that
// read one chunk of 16 rows meet no bank twice; the DMA writes LDS in lane order, so its lanes read
// their row's chunks in that permuted order.
//
// A wavefront multiplies its tokens by its weight rows in 16 x 16 x 32 blocks, weights as operand A, two
// half stages of 32 elements a stage. The operands of a half stage are read from LDS while the half
// before it is multiplied. In the middle of stage k every wavefront has read all of it: one barrier
// there frees its buffer for stage k + kStages and publishes stage k + 1.
//
// What bounds it. Large products, by 256 x 256 tiles: the matrix pipes, busy 0.77 of the time in 8192 x 2048 x
// 5632 (150 us, 1.26 PFLOP/s, a single round of tiles whose ends nothing overlaps) and 0.71 in gated 8192 x 5632
// x 4096 (580 us, 1.30 PFLOP/s); random operands draw the clock down, zeros take 111 us where those take 135 to
// 150. Of the 111 the barriers cost 10, the operand reads 5, the loads 6 (each taken out of a copy). Tried there
// without gain: arrival counters in LDS for the barrier, all reads of a half stage at its start, its loads over
// two halves, 32 x 32 x 16 MFMAs, four wavefronts of 128 x 128. The 256 x 256 kernels without adapters use all 256
// registers and spill 8 (gated 2): written before the walk and in its last stages, read back there and in the epilogue;
// the loops over the stages access no scratch. With adapters they spill 19 and 32, some in the adapters' stages. Smaller
// products: what a CU can load, 115 to 135 GB/s from L2 and 60 to 70 from beyond, so the shape with the fewest rows per CU
// that still gives every CU a tile (gated 200 x 1408 x 4096: 220 tiles of 48 x 64, 0.9 MB each, 14.0 us). By registers and
// 128-byte rows the loads are no faster, in operand layout (16 rows of 64 bytes) 38 GB/s.
#pragma once

#include <type_traits>

#include "grouped_prefill.hpp"
#include "linear.hpp"
#include "linear_adapter.hpp"

namespace uniserve {
namespace linear {

constexpr int kStageBytes = 128;  // of a row
constexpr int kStageK = 64;

/// kSplit: teams of kWavesM x kWavesN wavefronts, each with a ring of its own, that take the stages of K in
/// turn and whose sums are added at the end.
template <int kBM_, int kBN_, int kWavesM_, int kWavesN_, int kStages_, int kSplit_ = 1>
struct TileShape {
  static constexpr int kBM = kBM_, kBN = kBN_, kWavesM = kWavesM_, kWavesN = kWavesN_, kStages = kStages_, kSplit = kSplit_;
  static constexpr int kWaves = kWavesM * kWavesN;  // of a team
  static constexpr int kThreads = kSplit * kWaves * kWave;
  static constexpr int kRows = kBM + kBN;
  static constexpr int kLoads = kRows / 8 / kWaves;  // DMA instructions per wavefront and stage
  static constexpr int kLdsBytes = kStages * kRows * kStageBytes;  // of a team
  static constexpr int kMB = kBM / kWavesM / 16;  // 16-token blocks of a wavefront
  static constexpr int kNB = kBN / kWavesN / 16;  // 16-row weight blocks
  static_assert(kRows % (8 * kWaves) == 0 && kBM % (8 * kWaves) == 0, "whole DMA instructions, each over one operand");
  // Token blocks whose sums (FP32) of all wavefronts fit the ring.
  static constexpr int kFit = kLdsBytes / (kWaves * 16 * kNB * 16 * 4);
  static constexpr int kPassMB = kFit < kMB ? kFit : kMB;
  static_assert(kFit >= 1 && kMB % kPassMB == 0 && (kSplit == 1 || kPassMB == kMB), "whole passes; one where teams meet");
};

__device__ __forceinline__ int tile_slot(int row, int chunk) { return row * 8 + (chunk ^ ((row >> 1) & 7)); }

/// Tile `b` of a grid dealt to the XCDs in turn (block b runs on XCD b % 8): each XCD takes a contiguous
/// run of the tiles, ordered so that the some 32 tiles an XCD holds at a time share rows in its L2: equal groups
/// of up to seven token tiles, weight tile by weight tile inside a group. (Groups of four: gated 8192 x 5632 x
/// 4096 605 us, seven 580, six 592, eight 600; 16000 x 2048 x 2048 124 and 116; gated 200 x 1408 x 4096, whose
/// five token tiles then read each weight row into one L2, 15.1 and 14.4.)
__device__ __forceinline__ void tile_of_block(int64_t m_tiles, int64_t n_tiles, int64_t &m_tile, int64_t &n_tile) {
  constexpr int kXcds = 8, kMostInGroup = 7;
  const int64_t tiles = m_tiles * n_tiles;
  const int64_t b = blockIdx.x;
  const int64_t each = tiles / kXcds, more = tiles % kXcds;
  const int64_t xcd = b % kXcds;
  const int64_t at = xcd * each + (xcd < more ? xcd : more) + b / kXcds;
  const int64_t in_group = ceil_div(m_tiles, ceil_div<int64_t>(m_tiles, kMostInGroup));
  const int64_t group = at / (in_group * n_tiles);
  const int64_t within = at % (in_group * n_tiles);
  const int64_t rows = m_tiles - group * in_group < in_group ? m_tiles - group * in_group : in_group;
  m_tile = group * in_group + within % rows;
  n_tile = within / rows;
}

/// Waits until at most `stages` stages of kLoads loads are outstanding (kMost or more: until kMost are).
template <int kMost, int kLoads>
__device__ __forceinline__ void wait_stages_but(int stages) {
  if constexpr (kMost == 0) {
    prefill::wait_loads_but<0>();
  } else {
    if (stages >= kMost) prefill::wait_loads_but<kMost * kLoads>();
    else wait_stages_but<kMost - 1, kLoads>(stages);
  }
}

/// kDma: rows as p.by_dma says, whole 16-byte pieces, a tile's rows within 32-bit byte offsets. Else any rows:
/// the stages come through registers, by 16-byte loads at any alignment, zeros past the rows' ends.
/// P: LinearParams; AdapterParams, whose rows' adapters join the sums in the walk, behind it or before it (kWalked, kStaged,
/// else); or RankParams, the adapters' first product, whose walk is made for each adapter that the tile's rows name.
template <class T, bool kGated, bool kDma, class S, class P>
__global__ void __launch_bounds__(S::kThreads) tile_kernel(P p) {
  using prefill::dma16;
  using prefill::lds_address;
  __shared__ u32x4 rings[S::kSplit][S::kStages][S::kRows * 8];
  constexpr int MB = S::kMB, NB = S::kNB;
  static_assert(!kGated || NB % 2 == 0, "up and gate blocks");
  const int team = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / (S::kWaves * kWave));
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / kWave) - team * S::kWaves;
  auto &ring = rings[team];
  const int lane = lane_id();
  const int r16 = lane & 15;
  const int g = lane >> 4;
  const int wave_m = wave / S::kWavesN, wave_n = wave % S::kWavesN;
  constexpr int kCols = kGated ? S::kBN / 2 : S::kBN;  // output columns of the tile
  constexpr int kWaveCols = kCols / S::kWavesN;
  int64_t m_tile, n_tile;
  tile_of_block(ceil_div<int64_t>(p.m, S::kBM), ceil_div<int64_t>(p.n, kCols), m_tile, n_tile);
  const int64_t m0 = m_tile * S::kBM, n0 = n_tile * kCols;
  const int rows_left = static_cast<int>(p.m - m0 < S::kBM ? p.m - m0 : S::kBM);
  const int cols_left = static_cast<int>(p.n - n0 < kCols ? p.n - n0 : kCols);
  constexpr bool kRanks = std::is_same<P, RankParams>::value;      // the adapters' first factor
  constexpr bool kAdapters = std::is_same<P, AdapterParams>::value;  // a product with the second one's
  // Where the second one's product is added: in the walk, as stages before K's; through LDS behind the walk; or, of small
  // wavefront tiles, straight from memory before it.
  constexpr bool kMany = kAdapters && S::kSplit == 1 && MB * NB >= 8;
  constexpr bool kWalked = kMany && kDma && std::is_same<T, Bf16>::value;
  constexpr bool kStaged = kMany && !kWalked;
  static_assert(!kStaged || S::kThreads >= S::kBM, "a thread for each row's factor");
  [[maybe_unused]] __shared__ RowsAdapters<kMany ? S::kBM : 0, std::is_same<T, F16>::value> rows_adapters;
  [[maybe_unused]] __shared__ uint32_t columns_known[kWalked ? S::kThreads : 1];  // (in LDS: a register would spill a sum)
  if constexpr (kWalked) columns_known[threadIdx.x] = ~0u;
  if constexpr (kMany) rows_adapters.load(p, m0);
  [[maybe_unused]] typename std::conditional<kRanks, NamedAdapters, int>::type named = named_adapters(p, m0, S::kBM);
  do {  // once, or for each adapter that the tile's rows name (kRanks)
  if constexpr (kRanks) {
    if (!named.next()) return;
  }

  // ---- the loads: instruction i of wavefront w fills LDS rows 8 (w + kWaves i) .. + 7, first the tokens,
  // then the weights (rows past the edge repeat the last one; their sums are never stored). The weights'
  // LDS rows are the wavefronts' in turn, gated: each wavefront's up rows and then its gate rows. Row r
  // keeps its chunk c at c ^ (r / 2) % 8: a lane reads the chunk that its place holds. ----
  const char *base[S::kLoads];
  uint32_t offset[S::kLoads];           // kDma
  const uint16_t *row_at[S::kLoads];    // else: the lane's row
  u32x4 held[S::kLoads];                // and its chunk of the next stage
  const char *x_base = reinterpret_cast<const char *>(p.x + m0 * p.x_stride);
  const char *w_base = reinterpret_cast<const char *>(p.w + n0 * p.w_stride);
  auto chunk_of = [&](int i) { return (lane & 7) ^ ((lane >> 4) & 3) ^ (4 * ((wave + S::kWaves * i) & 1)); };
  auto aim_at_k = [&]() {
#pragma unroll
    for (int i = 0; i < S::kLoads; ++i) {
      const int first = 8 * (wave + S::kWaves * i);
      const int r = first + lane / 8;
      const bool token = i < S::kBM / 8 / S::kWaves;
      int64_t at;
      if (token) {
        base[i] = x_base;
        if constexpr (kRanks) at = named.row(r) * p.x_stride;
        else at = (r < rows_left ? r : rows_left - 1) * p.x_stride;
      } else if constexpr (kRanks) {
        base[i] = reinterpret_cast<const char *>(p.down + named.current * p.down_stride);
        at = p.down_row(n0 + r - S::kBM) * p.down_row_stride;
      } else {
        const int j = r - S::kBM;
        const int of = j / (NB * 16), in = j % (NB * 16);
        const int column = of * kWaveCols + (kGated ? in % kWaveCols : in);
        const bool second = kGated && (first - S::kBM) % (NB * 16) >= kWaveCols;
        base[i] = second ? w_base + p.n * p.w_stride * 2 : w_base;
        at = (column < cols_left ? column : cols_left - 1) * p.w_stride;
      }
      row_at[i] = reinterpret_cast<const uint16_t *>(base[i]) + at;
      base[i] += team * kStageBytes;
      offset[i] = static_cast<uint32_t>(at * 2) + chunk_of(i) * 16;
    }
  };
  if constexpr (!kWalked) aim_at_k();
  // The team's walk takes stages team, team + kSplit, .. of the row; the walks are equally long, and the last
  // stage of a walk holds all eight chunks of a row, the row's last few, or none.
  const int all_stages = static_cast<int>(ceil_div<int64_t>(p.k, kStageK));
  int stages = (all_stages + S::kSplit - 1) / S::kSplit;
  const int last_stage = (stages - 1) * S::kSplit + team;
  const int row_chunks = static_cast<int>(p.k / 8);
  const int last_chunks = !kDma ? 8 : last_stage >= all_stages ? 0 : (row_chunks - last_stage * 8 < 8 ? row_chunks - last_stage * 8 : 8);
  const uint32_t ring_lds = __builtin_amdgcn_readfirstlane(lds_address(&ring[0][wave * 64]));
  uint32_t to = ring_lds;   // where the next one goes
  // The next stage's loads: `begin_stage` (before the walk's last stage), each load, `end_stage`.
  auto begin_stage = [&]() {
    if (last_chunks == 8) return;
    // Chunks past the row's end: the row's first chunk of the stage is read instead (multiplied as zeros).
#pragma unroll
    for (int i = 0; i < S::kLoads; ++i) {
      if (chunk_of(i) >= last_chunks) offset[i] -= chunk_of(i) * 16;
      if (last_chunks == 0) base[i] -= static_cast<int64_t>(last_stage) * kStageBytes;
    }
  };
  auto issue = [&](int i) { dma16(base[i], offset[i], to + i * S::kWaves * 1024); };
  auto end_stage = [&]() {
#pragma unroll
    for (int i = 0; i < S::kLoads; ++i) base[i] += S::kSplit * kStageBytes;
    to = to + S::kRows * kStageBytes == ring_lds + S::kLdsBytes ? ring_lds : to + S::kRows * kStageBytes;
  };

  // kWalked: the walk's first stages are 32 ranks of one adapter each (gated: of one half's factors), `values, errors`
  // against twice the same ranks of the up rows. Zeros, a row's padding, stand for the rows of other adapters, for
  // the other half's weight rows and for a stage's chunks past the values; where a piece of an up row ends, its first
  // chunk comes again (against zeros).
  [[maybe_unused]] typename std::conditional<kWalked, NamedAdapters, int>::type adapter_stages = tile_adapters<kWalked>(rows_adapters, S::kBM);
  [[maybe_unused]] int adapted = 0, stage_group = 0, stage_half = 0;
  if constexpr (kWalked) {
    __syncthreads();
    adapter_stages.find(rows_adapters.id);
    const LowLayout layout(p.rank);
    adapted = adapter_stages.count() * layout.groups * (kGated ? 2 : 1);
    stages += adapted;
    stage_group = layout.groups;
  }
  [[maybe_unused]] auto aim = [&](int s) {
    if constexpr (kWalked) {
      if (s > adapted) return;
      if (s == adapted) return aim_at_k();
      const LowLayout layout(p.rank);
      if (stage_group == layout.groups) {
        stage_group = 0;
        if (stage_half == 1 || !kGated || adapter_stages.current < 0) {
          stage_half = 0;
          adapter_stages.next();
        } else {
          stage_half = 1;
        }
      }
      const int row_bytes = static_cast<int>(layout.row_bytes(kGated ? 2 : 1));
      const char *low = p.low + m0 * row_bytes + static_cast<int64_t>(stage_half * layout.groups + stage_group) * layout.group_bytes();
      const uint16_t *up = p.up + adapter_stages.current * p.up_stride + (n0 + stage_half * p.n) * p.up_row_stride + stage_group * 32;
      const uint32_t zeros = static_cast<uint32_t>(adapter_stages.first_row() * row_bytes + 4 * layout.width);
      const int chunks = p.rank - stage_group * 32 < layout.width ? (p.rank - stage_group * 32) / 8 : layout.width / 8;
#pragma unroll
      for (int i = 0; i < S::kLoads; ++i) {
        const int first = 8 * (wave + S::kWaves * i);
        const int r = first + lane / 8, c = chunk_of(i);
        if (i < S::kBM / 8 / S::kWaves) {
          base[i] = low;
          offset[i] = 4 * c < layout.width && rows_adapters.id[r] == adapter_stages.current ? static_cast<uint32_t>(r * row_bytes + 16 * c) : zeros;
        } else {
          const int j = r - S::kBM;
          const int of = j / (NB * 16), in = j % (NB * 16);
          const int column = of * kWaveCols + (kGated ? in % kWaveCols : in);
          const int half = kGated && (first - S::kBM) % (NB * 16) >= kWaveCols ? 1 : 0;
          const int chunk = c % (layout.width / 8);
          const uint32_t at = static_cast<uint32_t>(column < cols_left ? column : cols_left - 1) * static_cast<uint32_t>(p.up_row_stride);
          base[i] = half == stage_half ? reinterpret_cast<const char *>(up) : low;
          offset[i] = half == stage_half ? at * 2 + (chunk < chunks ? chunk : 0) * 16 : zeros;
        }
      }
      ++stage_group;
    }
  };

  floatx4 acc[NB][MB];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
#pragma unroll
    for (int mb = 0; mb < MB; ++mb) acc[nb][mb] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};

  u32x4 wf[2][NB], xf[2][MB];
  const int x_row = wave_m * MB * 16 + r16;
  const int w_row = S::kBM + wave_n * NB * 16 + r16;
  // Block b of a half stage's operands: weights 0 .. NB - 1, then tokens.
  auto read = [&](int buffer, int half, int b) {
    const u32x4 *rows = ring[buffer];
    if (b < NB) wf[half][b] = rows[tile_slot(w_row, half * 4 + g) + b * 128];
    else xf[half][b - NB] = rows[tile_slot(x_row, half * 4 + g) + (b - NB) * 128];
  };
  // Through registers: `fetch` loads the walk's next stage, if there is one, `put` writes the one held to `buffer`.
  int fetched = 0;
  auto fetch = [&]() {
    if (fetched == stages) return;
    const int64_t k = (static_cast<int64_t>(fetched) * S::kSplit + team) * kStageK;
    ++fetched;
    if (k + kStageK <= p.k) {
#pragma unroll
      for (int i = 0; i < S::kLoads; ++i) __builtin_memcpy(&held[i], row_at[i] + k + chunk_of(i) * 8, 16);
    } else {
#pragma unroll
      for (int i = 0; i < S::kLoads; ++i) held[i] = load8(row_at[i], k + chunk_of(i) * 8, p.k);
    }
  };
  auto put = [&](int buffer) {
#pragma unroll
    for (int i = 0; i < S::kLoads; ++i) ring[buffer][(wave + S::kWaves * i) * 64 + lane] = held[i];
  };
  constexpr int kReadsPer = (NB + MB + NB - 1) / NB;
  constexpr int kIssuesPer = (S::kLoads + NB - 1) / NB;
  // The MFMAs of one half stage, row of weight blocks by row, with the other half's reads from `buffer`
  // and the next stage's loads spread between them.
  auto multiply = [&](auto half_of, auto reads, auto issues, int buffer) {
    constexpr int half = decltype(half_of)::value;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      if constexpr (decltype(reads)::value) {
#pragma unroll
        for (int j = 0; j < kReadsPer; ++j)
          if (nb * kReadsPer + j < NB + MB) read(buffer, half ^ 1, nb * kReadsPer + j);
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int mb = 0; mb < MB; ++mb) {
        acc[nb][mb] = T::mfma(wf[half][nb], xf[half][mb], acc[nb][mb]);
        // The row's loads, spread over its MFMAs.
        if constexpr (decltype(issues)::value) {
#pragma unroll
          for (int j = mb * kIssuesPer / MB; j < (mb + 1) * kIssuesPer / MB; ++j) {
            __builtin_amdgcn_sched_barrier(0);
            if (nb * kIssuesPer + j < S::kLoads) issue(nb * kIssuesPer + j);
            __builtin_amdgcn_sched_barrier(0);
          }
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    if constexpr (decltype(issues)::value) end_stage();
  };
  // Past the row's end both operands are zero (what was read in its place may be infinite).
  auto mask = [&](auto half_of) {
    constexpr int half = decltype(half_of)::value;
    const bool out = half * 4 + g >= last_chunks;
#pragma unroll
    for (int b = 0; b < NB; ++b) wf[half][b] = out ? u32x4{0, 0, 0, 0} : wf[half][b];
#pragma unroll
    for (int b = 0; b < MB; ++b) xf[half][b] = out ? u32x4{0, 0, 0, 0} : xf[half][b];
  };
  constexpr std::integral_constant<int, 0> first_half{};
  constexpr std::integral_constant<int, 1> second_half{};
  constexpr std::true_type yes{};
  constexpr std::false_type no{};

  // The other wavefronts' loads and reads (a wavefront alone waits for its own).
  auto meet = [&]() {
    if constexpr (S::kWaves > 1) __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  // Awaiting a stage by DMA, at most the kStages - 2 stages behind it are outstanding.
  constexpr int kBehind = (S::kStages - 2) * S::kLoads;
  static_assert(kBehind + S::kLoads < 64, "vmcnt holds 6 bits");
  constexpr int kWaitLds = 0xc07f;  // lgkmcnt 0, nothing else
  [[maybe_unused]] typename std::conditional<kAdapters && !kMany, RowAdapters<MB>, int>::type adapters =
      row_adapters<MB, kMany>(p, m0 + wave_m * MB * 16);
#pragma unroll
  for (int s = 0; s < S::kStages; ++s) {
    if constexpr (kDma) {
      if (s < stages) {
        aim(s);
        if (s == stages - 1) begin_stage();
#pragma unroll
        for (int i = 0; i < S::kLoads; ++i) issue(i);
        end_stage();
      }
    } else {
      fetch();
      put(s);
    }
  }
  if constexpr (kAdapters && !kMany)
    add_low_rank<T, kGated>(p, acc, adapters, m0 + wave_m * MB * 16, n0 + wave_n * kWaveCols, team, S::kSplit);
  if constexpr (kDma) {
    wait_stages_but<S::kStages - 1, S::kLoads>(stages - 1);
  } else {
    fetch();
    __builtin_amdgcn_s_waitcnt(kWaitLds);
  }
  meet();
#pragma unroll
  for (int b = 0; b < NB + MB; ++b) read(0, 0, b);
  int buffer = 0;
  // A stage's first half; then it is in registers, its reads done (lgkmcnt 0), and the next one in LDS (DMA: vmcnt,
  // `ends` where no loads follow; else written half a stage or more ago).
  auto step = [&](auto ends, int left) {
    __builtin_amdgcn_sched_barrier(0);
    multiply(first_half, yes, no, buffer);
    if constexpr (kDma && decltype(ends)::value) wait_stages_but<S::kStages - 2, S::kLoads>(left);
    __builtin_amdgcn_s_waitcnt(kDma && !decltype(ends)::value ? 0x0070 | (kBehind & 15) | ((kBehind >> 4) << 14) : kWaitLds);
    meet();
    if constexpr (!kDma) {
      put(buffer);
      fetch();
    }
    buffer = buffer + 1 == S::kStages ? 0 : buffer + 1;
  };
  int k = 0;
  if constexpr (kDma) {
    if constexpr (kWalked) {
      for (; k + S::kStages <= adapted; ++k) {  // the next loads are an adapter's, or K's first
        step(no, 0);
        aim(k + S::kStages);
        if (k + S::kStages == stages - 1) begin_stage();
        multiply(second_half, yes, yes, buffer);
      }
    }
    for (; k + S::kStages < stages - 1; ++k) {  // the next loads are not the walk's last
      step(no, 0);
      multiply(second_half, yes, yes, buffer);
    }
    if (k + S::kStages == stages - 1) {
      step(no, 0);
      begin_stage();
      multiply(second_half, yes, yes, buffer);
      ++k;
    }
  }
  for (; k < stages - 1; ++k) {
    step(yes, stages - 2 - k);
    multiply(second_half, yes, no, buffer);
  }
  if (last_chunks < 8) mask(first_half);
  multiply(first_half, yes, no, buffer);
  if (last_chunks < 8) mask(second_half);
  multiply(second_half, no, no, 0);
  if constexpr (kStaged) {
    // Stage by stage, as above, but multiplied apart from the sums and added to them where a row names the adapter: f16
    // rows have a factor each, and stages through registers need no padding.
    const LowLayout layout(p.rank);
    constexpr int kHalves = kGated ? 2 : 1;
    NamedAdapters tile(S::kBM);
    __syncthreads();  // the ring has been read
    tile.find(rows_adapters.id);
    const bool wide = layout.width == 32;
    int buffer_of = 0;
    auto stage = [&](auto half_of, int group) {
      constexpr int h = decltype(half_of)::value;
      const int part = h * layout.groups + group;
      const char *low = p.low + m0 * layout.row_bytes(kHalves) + static_cast<int64_t>(part) * layout.group_bytes();
      const uint16_t *up = p.up + tile.current * p.up_stride + (n0 + h * p.n) * p.up_row_stride + group * 32;
      // (opaque: what the lanes' addresses share from stage to stage is not kept, the sums need the registers)
      int l = lane;
      asm volatile("" : "+v"(l));
      u32x4 pieces[S::kLoads];
      [[maybe_unused]] float factor_of_row = 1.0f;
      if constexpr (std::is_same<T, F16>::value) factor_of_row = rows_adapters.load_factor(p, m0, layout, kHalves, part);
#pragma unroll
      for (int i = 0; i < S::kLoads; ++i) {
        const int r = 8 * (wave + S::kWaves * i) + l / 8, c = (l & 7) ^ ((l >> 4) & 3) ^ (4 * ((wave + S::kWaves * i) & 1));
        const bool filled = 4 * c < layout.width;
        if (i < S::kBM / 8 / S::kWaves) {
          const uint32_t row = static_cast<uint32_t>(r < rows_left ? r : rows_left - 1);
          pieces[i] = *reinterpret_cast<const u32x4 *>(low + (row * static_cast<uint32_t>(layout.row_bytes(kHalves)) + (filled ? 16 * c : 0)));
        } else {
          const int j = r - S::kBM;
          const int of = j / (NB * 16), in = j % (NB * 16);
          int column = of * kWaveCols + (kGated ? in % kWaveCols : in);
          column = column < cols_left ? column : cols_left - 1;
          const int at = (wide ? c & 3 : layout.width == 16 ? c & 1 : 0) * 8;
          if (p.up_whole)
            pieces[i] = *reinterpret_cast<const u32x4 *>(up + (static_cast<uint32_t>(column) * static_cast<uint32_t>(p.up_row_stride) +
                                                               (group * 32 + at < p.rank ? at : 0)));
          else
            pieces[i] = load8(up + column * p.up_row_stride, at, p.rank - group * 32);
        }
      }
#pragma unroll
      for (int i = 0; i < S::kLoads; ++i) {
        const int c = (l & 7) ^ ((l >> 4) & 3) ^ (4 * ((wave + S::kWaves * i) & 1));
        bool filled = 4 * c < layout.width;
        if (i >= S::kBM / 8 / S::kWaves) {
          // Zeros past the rank (where the row's first chunk was read); no infinities and NaN against errors.
          const int at = (wide ? c & 3 : layout.width == 16 ? c & 1 : 0) * 8;
          filled = filled && group * 32 + at < p.rank;
          pieces[i] = finite_only<T>(pieces[i], 8 * c >= layout.width);
        }
        ring[buffer_of][(wave + S::kWaves * i) * 64 + l] = filled ? pieces[i] : u32x4{0, 0, 0, 0};
      }
      if constexpr (std::is_same<T, F16>::value) rows_adapters.put_factor(buffer_of, factor_of_row);
      // Two buffers in turn: one barrier a stage (a wavefront writes the other one only after all have read it).
      __syncthreads();
      // Both halves of the stage, zeros up to rank 16 (two ways through here would cost registers, and spill sums).
      const u32x4 *rows = ring[buffer_of];
      constexpr int kRowsAtOnce = MB % 4 == 0 ? 4 : MB;
#pragma unroll
      for (int mb = 0; mb < MB; mb += kRowsAtOnce) {
        u32x4 x0[kRowsAtOnce], x1[kRowsAtOnce];
        bool own[kRowsAtOnce];
        float factor[kRowsAtOnce];
#pragma unroll
        for (int j = 0; j < kRowsAtOnce; ++j) {
          const int row = (wave_m * MB + mb + j) * 16 + r16;
          x0[j] = rows[tile_slot(x_row, g) + (mb + j) * 128];
          x1[j] = rows[tile_slot(x_row, 4 + g) + (mb + j) * 128];
          own[j] = rows_adapters.id[row] == tile.current;
          factor[j] = 1.0f;
          if constexpr (std::is_same<T, F16>::value) factor[j] = rows_adapters.factor[buffer_of][row];
        }
#pragma unroll
        for (int nb = h * (NB / kHalves); nb < (h + 1) * (NB / kHalves); ++nb) {
          const u32x4 w0 = rows[tile_slot(w_row, g) + nb * 128], w1 = rows[tile_slot(w_row, 4 + g) + nb * 128];
          floatx4 sum[kRowsAtOnce];
#pragma unroll
          for (int j = 0; j < kRowsAtOnce; ++j) sum[j] = T::mfma(w0, x0[j], floatx4{0.0f, 0.0f, 0.0f, 0.0f});
#pragma unroll
          for (int j = 0; j < kRowsAtOnce; ++j) sum[j] = T::mfma(w1, x1[j], sum[j]);
#pragma unroll
          for (int j = 0; j < kRowsAtOnce; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float v = std::is_same<T, F16>::value ? sum[j][e] * factor[j] : sum[j][e];
              acc[nb][mb + j][e] += own[j] ? v : 0.0f;
            }
        }
        asm volatile("" ::: "memory");  // (the weights are read again, not kept)
      }
      buffer_of ^= 1;
    };
    for (int group = layout.groups;; ++group) {  // (one loop, not two: that costs registers, too)
      if (group == layout.groups) {
        if (!tile.next()) break;
        group = 0;
      }
      stage(first_half, group);
      if constexpr (kGated) stage(second_half, group);
    }
    __syncthreads();
  }

  // ---- the epilogue: each wavefront passes its sums through its own part of the ring (no longer read by
  // anyone), kPassMB token blocks at a time, so that a lane then holds eight consecutive columns of a
  // token: whole 16-byte stores, and one copy of the epilogue's code, not one per block. Teams share the
  // rows of a block out and add each other's sums, in the teams' order. ----
  meet();
  constexpr int kRowChunks = NB * 4;  // 16-byte pieces of a token's sums
  constexpr int kPassMB = S::kPassMB;
  constexpr int kGroups = kWaveCols / 8;  // of eight columns
  static_assert(kWave % kGroups == 0, "a lane's columns stay the same");
  u32x4 *sums = &ring[0][0] + wave * kPassMB * 16 * kRowChunks;
  constexpr int kTeamChunks = S::kStages * S::kRows * 8;  // from one team's sums to the next's
  auto at_chunk = [&](int row, int c) { return row * kRowChunks + (c ^ (row & (kRowChunks < 16 ? kRowChunks - 1 : 15))); };
  const int group = lane % kGroups;
  const int64_t n = n0 + wave_n * kWaveCols + group * 8;
  [[maybe_unused]] const typename std::conditional<kRanks, RankColumns<T>, Columns8<T, kGated>>::type columns(p, n);
#pragma unroll
  for (int pass = 0; pass < MB / kPassMB; ++pass) {
    if (pass > 0) wave_fence();  // (the one before has been read)
#pragma unroll
    for (int b = 0; b < kPassMB; ++b)
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
        sums[at_chunk(b * 16 + r16, nb * 4 + g)] = __builtin_bit_cast(u32x4, acc[nb][pass * kPassMB + b]);
    if constexpr (S::kSplit > 1) {
      __syncthreads();
      sums = &rings[0][0][0] + wave * kPassMB * 16 * kRowChunks;
    } else {
      wave_fence();
    }
    constexpr int kStep = S::kSplit * (kWave / kGroups);  // rows the lanes (and teams) finish at a time
    constexpr int kBatch = kPassMB * 16 / kStep >= 4 ? 4 : (kPassMB * 16 / kStep >= 2 ? 2 : 1);
#pragma unroll 1
    for (int first = lane / kGroups + team * (kWave / kGroups); first < kPassMB * 16; first += kBatch * kStep) {
      const int64_t m_first = m0 + (wave_m * MB + pass * kPassMB) * 16;
      int64_t m[kBatch];
#pragma unroll
      for (int j = 0; j < kBatch; ++j) m[j] = m_first + first + j * kStep < p.m ? m_first + first + j * kStep : p.m - 1;
      typename Columns8<T, kGated>::template Extras<kBatch> extras;
      if constexpr (!kRanks) columns.load(p, m, n, extras);
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        const int row = first + j * kStep;
        if (row >= kPassMB * 16 || m_first + row >= p.m) continue;
        floatx4 v[2], gates[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int c = at_chunk(row, group * 2 + i), d = at_chunk(row, kRowChunks / 2 + group * 2 + i);
          v[i] = __builtin_bit_cast(floatx4, sums[c]);
          if constexpr (kGated) gates[i] = __builtin_bit_cast(floatx4, sums[d]);
          else gates[i] = v[i];
#pragma unroll
          for (int other = 1; other < S::kSplit; ++other) {
            v[i] += __builtin_bit_cast(floatx4, sums[other * kTeamChunks + c]);
            if constexpr (kGated) gates[i] += __builtin_bit_cast(floatx4, sums[other * kTeamChunks + d]);
          }
        }
        if constexpr (kWalked) {
          if (adapted > 0) remake<kGated>(p, m[j], n, rows_adapters.id, S::kBM, static_cast<int>(m[j] - m0), columns_known[threadIdx.x], v, gates);
        }
        if constexpr (kRanks) {
          if (named.holds(static_cast<int>(m[j] - m0))) columns.finish(p, m[j], named.current, v);
        } else {
          columns.finish(p, m[j], n, v, gates, extras.residual[j], extras.factor[j]);
        }
      }
    }
  }
  if constexpr (kRanks) __syncthreads();  // the ring is free again
  } while (kRanks);
}

template <class S>
int64_t tiles_of(const LinearParams &p, bool gated) {
  return ceil_div<int64_t>(p.m, S::kBM) * ceil_div<int64_t>(p.n, gated ? S::kBN / 2 : S::kBN);
}

template <class T, bool kGated, bool kDma, class S, class P>
void launch_tiles(const P &p, hipStream_t stream, uint32_t shares = 1) {
  hipLaunchKernelGGL((tile_kernel<T, kGated, kDma, S, P>), dim3(static_cast<uint32_t>(tiles_of<S>(p, kGated)), shares), dim3(S::kThreads), 0,
                     stream, p);
}

}  // namespace linear
}  // namespace uniserve
