// SPDX-License-Identifier: Apache-2.0
//
// Low-rank adapters beside the dense products: the first factor's epilogue, which leaves each row's rank values in the
// workspace, and the second factor's product, which the product kernels add to their sums before, in or behind the walk over K.
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

/// Eight elements with zeros for those that are infinite or NaN, where `drop` says so. (What a value's error meets: the value
/// itself meets the element, and an infinity times the error would be NaN or the other infinity.)
template <class T>
__device__ __forceinline__ u32x4 finite_only(u32x4 w, bool drop) {
  typedef int16_t i16x2 __attribute__((ext_vector_type(2)));
  constexpr bool kF16 = std::is_same<T, F16>::value;
  constexpr uint32_t kExponents = kF16 ? 0x7c007c00u : 0x7f807f80u, kOne = kF16 ? 0x04000400u : 0x00800080u;
  const uint32_t dropped = drop ? ~0u : 0u;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const i16x2 past = __builtin_bit_cast(i16x2, (w[i] & kExponents) + kOne);  // negative where all of the exponent is set
    w[i] &= ~(__builtin_bit_cast(uint32_t, past >> 15) & dropped);
  }
  return w;
}

// ---- which adapters a tile names ---------------------------------------------------------------------------

/// The distinct adapters of a tile's rows, one after the other, found by every wavefront alike.
struct NamedAdapters {
  int id[4];              ///< of rows lane, 64 + lane, ..
  uint64_t remaining[4];  ///< rows whose adapter has not come yet
  uint64_t members[4];    ///< rows of the current one
  int current = -1;
  uint32_t turn = 0, share = 0, shares = 1;
  int blocks;

  /// (find takes the rows' adapters from LDS)
  __device__ __forceinline__ explicit NamedAdapters(int rows) : blocks((rows + 63) / 64) {}
  __device__ __forceinline__ void find(const int32_t *ids) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < blocks) {
        id[i] = ids[i * 64 + lane_id()];
        remaining[i] = ballot(id[i] >= 0);
      }
  }
  /// Of a workgroup that shares a tile's adapters with gridDim.y - 1 others.
  __device__ __forceinline__ NamedAdapters(const RankParams &p, int64_t m0, int rows) : share(blockIdx.y), shares(gridDim.y), blocks(1) {
    id[0] = lane_id() < rows ? adapter_of(p, m0 + lane_id()) : -1;
    remaining[0] = ballot(id[0] >= 0);
  }
  __device__ __forceinline__ bool next() {
    for (;;) {
      current = -1;
#pragma unroll
      for (int i = 3; i >= 0; --i)
        if (i < blocks && remaining[i] != 0) current = __builtin_amdgcn_readlane(id[i], __ffsll(static_cast<long long>(remaining[i])) - 1);
      if (current < 0) return false;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (i < blocks) {
          members[i] = ballot(id[i] == current);
          remaining[i] &= ~members[i];
        }
      const bool mine = turn == share;
      turn = turn + 1 == shares ? 0 : turn + 1;
      if (mine) return true;
    }
  }
  /// How many there are, from a copy.
  __device__ __forceinline__ int count() const {
    NamedAdapters all = *this;
    int found = 0;
    while (all.next()) ++found;
    return found;
  }
  /// The first row of the current adapter.
  __device__ __forceinline__ int first_row() const {
    int row = 0;
#pragma unroll
    for (int i = 3; i >= 0; --i)
      if (i < blocks && members[i] != 0) row = i * 64 + __ffsll(static_cast<long long>(members[i])) - 1;
    return row;
  }
  /// Of up to 64 rows: whether row r names the current adapter, and row r, or, if it does not, one that does.
  __device__ __forceinline__ bool holds(int r) const { return (members[0] >> r) & 1; }
  __device__ __forceinline__ int row(int r) const { return holds(r) ? r : first_row(); }
};

__device__ __forceinline__ NamedAdapters named_adapters(const RankParams &p, int64_t m0, int rows) { return NamedAdapters(p, m0, rows); }
__device__ __forceinline__ int named_adapters(const LinearParams &, int64_t, int) { return 0; }

/// The adapters of a tile's kRows rows and, f16, the factors of their group in either of two buffers.
template <int kRows, bool kFactors>
struct RowsAdapters {
  static constexpr int kIds = (kRows + 63) / 64 * 64;
  int32_t id[kIds];
  float factor[2][kFactors ? kRows : 1];
  __device__ __forceinline__ void load(const AdapterParams &p, int64_t m0) {
    for (int t = threadIdx.x; t < kIds; t += blockDim.x) id[t] = t < kRows ? adapter_of(p, m0 + t) : -1;
  }
  /// A thread's row's factor (a workgroup has as many threads as its tile has rows, or more).
  __device__ __forceinline__ float load_factor(const AdapterParams &p, int64_t m0, const LowLayout &layout, int halves, int part) const {
    const int64_t m = static_cast<int>(threadIdx.x) < kRows && m0 + threadIdx.x < p.m ? m0 + threadIdx.x : p.m - 1;
    return *reinterpret_cast<const float *>(p.low + m * layout.row_bytes(halves) + static_cast<int64_t>(part) * layout.group_bytes() +
                                            4 * layout.width);
  }
  __device__ __forceinline__ void put_factor(int buffer, float f) {
    if (static_cast<int>(threadIdx.x) < kRows) factor[buffer][threadIdx.x] = f;
  }
};
template <bool kFactors>
struct RowsAdapters<0, kFactors> {};

template <bool kWalked, class Rows>
__device__ __forceinline__ auto tile_adapters(const Rows &, int rows) {
  if constexpr (kWalked) return NamedAdapters(rows);
  else return 0;
}

/// Whether some of eight bf16 elements are infinite or NaN.
__device__ __forceinline__ bool any_not_finite(u32x4 w) {
  uint32_t past = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) past |= (w[i] & 0x7f807f80u) + 0x00800080u;
  return (past & 0x80008000u) != 0;
}

/// Which of columns n .. n + 7 (bits 0 .. 7; gated: and of their gate rows, 8 .. 15) have an up weight that is not finite, in
/// an adapter that one of a tile's rows names.
template <bool kGated>
__device__ __forceinline__ uint32_t columns_not_finite(const AdapterParams &p, int64_t n, const int32_t *ids, int rows) {
  constexpr uint32_t kAll = kGated ? 0xffffu : 0xffu;
  uint32_t found = 0;
  int last = -1;
#pragma unroll 1
  for (int r = 0; r < rows && found != kAll; ++r) {
    const int a = ids[r];
    if (a < 0 || a == last) continue;
    last = a;
#pragma unroll 1
    for (int64_t rank = 0; rank < p.rank; rank += 8)
#pragma unroll 1
      for (int i = 0; i < (kGated ? 16 : 8); ++i) {
        const int64_t column = (n + i % 8 < p.n ? n + i % 8 : p.n - 1) + (i < 8 ? 0 : p.n);
        const uint16_t *up = p.up + a * p.up_stride + column * p.up_row_stride;
        if (any_not_finite(load8_of<true>(up, rank, p.rank))) found |= 1u << i;  // (the walk's rows are whole)
      }
  }
  return found;
}

/// Makes those of a row's sums of eight columns again, from the row's own operands alone, that the walk may have made
/// infinite or NaN: it multiplies other adapters' up rows, pieces past a rank and, gated, one half's rank values by zeros,
/// which gives NaN where they are not finite, and a weight by a value and by its error, which gives NaN where the weight
/// is an infinity. What the row itself makes of its operands stays so: without such weights in the column (`known`: found
/// once a lane, when its first sum asks, ~0 before) or such rank values in the other half, nothing is made again, and
/// what has come to NaN is not carried on. (8192 x 4096 x 2048, rank 16, runs of 300 rows: finite 0.144 ms, all rows NaN
/// 0.30, where making every sum again took 18.3; one of eight adapters NaN 16, its tiles' other rows made again, a lane a
/// sum.)
template <bool kGated>
__device__ __forceinline__ void remake(const AdapterParams &p, int64_t m, int64_t n, const int32_t *ids, int rows, int row, uint32_t &known,
                                       floatx4 (&sums)[2], floatx4 (&gates)[2]) {
  using T = Bf16;
  float none = 0.0f;  // NaN if a sum is not finite
#pragma unroll
  for (int c = 0; c < 8; ++c) {
    none = __builtin_fmaf(sums[c / 4][c % 4], 0.0f, none);
    if (kGated) none = __builtin_fmaf(gates[c / 4][c % 4], 0.0f, none);
  }
  if (none == 0.0f) return;
  constexpr uint32_t kUnknown = ~0u;
  uint32_t weights = known;
  if (weights == kUnknown) known = weights = columns_not_finite<kGated>(p, n, ids, rows);
  const LowLayout layout(p.rank);
  const int adapter = ids[row];
  const char *values = p.low + m * layout.row_bytes(kGated ? 2 : 1);
#pragma unroll 1
  for (int h = 0; h < (kGated ? 2 : 1); ++h) {
    bool others = false;  // the other half's rank values
    if (kGated && adapter >= 0) {
#pragma unroll 1
      for (int at = 0; at < layout.groups * layout.width; at += 8)
        others = others || any_not_finite(*reinterpret_cast<const u32x4 *>(
                               values + static_cast<int64_t>((1 - h) * layout.groups + at / layout.width) * layout.group_bytes() + at % layout.width * 2));
    }
#pragma unroll 1
    for (int i = 0; i < 8; ++i) {
      if (n + i >= p.n || !(others || ((weights >> (h * 8 + i)) & 1))) continue;
      float v = 0.0f;
#pragma unroll
      for (int c = 0; c < 8; ++c)
        if (c == i) v = h == 0 ? sums[c / 4][c % 4] : gates[c / 4][c % 4];
      if (__builtin_fabsf(v) < __builtin_inff()) continue;
      const int64_t column = n + i + h * p.n;
      v = 0.0f;
      if (adapter >= 0) {
        const uint16_t *up = p.up + adapter * p.up_stride + column * p.up_row_stride;
#pragma unroll 1
        for (int rank = 0; rank < p.rank && v == v; ++rank) {
          const uint16_t *low = reinterpret_cast<const uint16_t *>(values + static_cast<int64_t>(h * layout.groups + rank / layout.width) * layout.group_bytes()) +
                                rank % layout.width;
          v = __builtin_fmaf(T::to_f32(low[0]) + T::to_f32(low[layout.width]), T::to_f32(up[rank]), v);
        }
      }
      const uint16_t *x = p.x + m * p.x_stride, *w = p.w + column * p.w_stride;
#pragma unroll 2
      for (int64_t k = 0; k < p.k && v == v; k += 8) {
        const u32x4 xs = load8_of<true>(x, k, p.k), ws = load8_of<true>(w, k, p.k);  // (the walk's rows are whole)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          v = __builtin_fmaf(T::high(xs[e]), T::high(ws[e]), __builtin_fmaf(T::low(xs[e]), T::low(ws[e]), v));
      }
#pragma unroll
      for (int c = 0; c < 8; ++c)
        if (c == i) {
          if (h == 0) sums[c / 4][c % 4] = v;
          else gates[c / 4][c % 4] = v;
        }
    }
  }
}

// ---- the first factor -------------------------------------------------------------------------------------

/// The epilogue of the first factor: eight consecutive rank values of a row, scaled, as elements and their errors.
template <class T>
struct RankColumns {
  int64_t at;     ///< of the values in a row's workspace; -1: past the last group
  int errors_at;  ///< from there
  int factor_at;
  int count;      ///< values below the rank
  __device__ __forceinline__ RankColumns(const RankParams &p, int64_t j) {
    const LowLayout layout(p.rank);
    const int group = static_cast<int>(j / p.width), chunk = static_cast<int>(j % p.width) / 8;
    const int in_half = group % p.groups * p.width + chunk * 8;
    at = j < p.n ? static_cast<int64_t>(group) * layout.group_bytes() + chunk * 16 : -1;
    errors_at = 2 * p.width;
    factor_at = chunk == 0 ? 4 * p.width : -1;
    count = p.rank - in_half;
  }
  __device__ __forceinline__ void finish(const RankParams &p, int64_t m, int adapter, const floatx4 (&sums)[2]) const {
    const float scale = p.scales == nullptr ? 1.0f : p.scales[adapter];
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < count ? sums[i / 4][i % 4] * scale : 0.0f;
    float factor = 1.0f;
    if constexpr (std::is_same<T, F16>::value) {
      // The power of two that brings the group's largest finite value to [1, 2); its lanes are neighbours. (An infinity or
      // NaN stays what it is; the values beside it would be infinities, too, if it decided.)
      float most = 0.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i) most = __builtin_fmaxf(most, __builtin_fabsf(v[i]) < __builtin_inff() ? __builtin_fabsf(v[i]) : 0.0f);
      for (int offset = 1; offset < p.width / 8; offset *= 2) most = __builtin_fmaxf(most, __shfl_xor(most, offset));
      if (most > 0.0f) {
        int power = __builtin_amdgcn_frexp_expf(most) - 1;
        power = power < -126 ? -126 : power;
        factor = __builtin_ldexpf(1.0f, power);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = __builtin_ldexpf(v[i], -power);
      }
    }
    if (at < 0) return;
    u32x4 values, errors;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      values[i] = T::pack2(v[2 * i], v[2 * i + 1]);
      const float low = v[2 * i] - T::low(values[i]), high = v[2 * i + 1] - T::high(values[i]);
      // (a value that is not finite, or rounds to an infinity, has no error: the pair's sum is the value)
      errors[i] = T::pack2(__builtin_fabsf(low) < __builtin_inff() ? low : 0.0f, __builtin_fabsf(high) < __builtin_inff() ? high : 0.0f);
    }
    char *to = p.low + m * LowLayout(p.rank).row_bytes(p.halves) + at;
    *reinterpret_cast<u32x4 *>(to) = values;
    *reinterpret_cast<u32x4 *>(to + errors_at) = errors;
    // (bf16 rows need no factor; 16 zeros stand there)
    if (factor_at >= 0) *reinterpret_cast<u32x4 *>(to + factor_at) = u32x4{std::is_same<T, F16>::value ? __float_as_uint(factor) : 0, 0, 0, 0};
  }
};

// ---- the second factor ------------------------------------------------------------------------------------

/// Adapters whose loads a wavefront has in flight together, by the blocks that one takes.
template <int NB, int MB>
constexpr int adapter_batch() { return NB + 2 * MB <= 4 ? 4 : NB + 2 * MB <= 8 ? 2 : 1; }

/// The adapters of a wavefront's rows: of token block b's row lane % 16.
template <int MB>
struct RowAdapters {
  int of[MB];
  __device__ __forceinline__ RowAdapters(const AdapterParams &p, int64_t m_first) {
#pragma unroll
    for (int b = 0; b < MB; ++b) of[b] = adapter_of(p, m_first + b * 16 + lane_id() % 16);
  }
};

/// What add_low_rank needs, for the kernels that call it.
template <int MB, bool kMany>
__device__ __forceinline__ auto row_adapters(const AdapterParams &p, int64_t m_first) {
  if constexpr (kMany) return 0;
  else return RowAdapters<MB>(p, m_first);
}
template <int MB, bool kMany>
__device__ __forceinline__ int row_adapters(const LinearParams &, int64_t) { return 0; }
template <int MB, bool kMany>
__device__ __forceinline__ int row_adapters(const RankParams &, int64_t) { return 0; }

/// Adds the adapters' products to a wavefront's sums: token blocks b from row m_first on, weight blocks nb from
/// column n_first on (gated: half of them the up rows', then the same columns' gate rows), some of the adapters that
/// its rows name after the others; of `teams` wavefronts with the same sums, which are added up later, each takes
/// its share of the adapters. Two matrix instructions per 32 ranks, over the values and over their errors, or, up to
/// rank 16, one over both. (What keeps infinite up rows from the errors, rows by one of 64 adapters: 64 x 4096 x
/// 2048, rank 64, 28.2 us against 25.9; 64 x 2048 x 4096, rank 16, 18.4 and 18.0; 256 x 4096 x 2048, rank 16, 31.8 and 29.8.)
template <class T, bool kGated, int NB, int MB>
__device__ __forceinline__ void add_low_rank(const AdapterParams &p, floatx4 (&acc)[NB][MB], const RowAdapters<MB> &mine, int64_t m_first,
                                             int64_t n_first, int team, int teams) {
  const int lane = lane_id();
  const int r16 = lane & 15, g = lane >> 4;
  const LowLayout layout(p.rank);
  constexpr int kHalves = kGated ? 2 : 1, kPerHalf = NB / kHalves, kBatch = adapter_batch<NB, MB>();
  uint32_t remaining[MB];
#pragma unroll
  for (int b = 0; b < MB; ++b) remaining[b] = static_cast<uint32_t>(ballot(mine.of[b] >= 0)) & 0xffffu;
  // The next adapter of this wavefront's share, or -1. (Shares by number: a row's sums do not depend on the other
  // rows' adapters.)
  auto next = [&]() {
    for (;;) {
      int current = -1;
#pragma unroll
      for (int b = MB - 1; b >= 0; --b)
        if (remaining[b] != 0) current = __builtin_amdgcn_readlane(mine.of[b], __ffs(static_cast<int>(remaining[b])) - 1);
      if (current < 0) return -1;
#pragma unroll
      for (int b = 0; b < MB; ++b) remaining[b] &= ~static_cast<uint32_t>(ballot(mine.of[b] == current));
      if (current % teams == team) return current;
    }
  };
  int current[kBatch];
#pragma unroll
  for (int j = 0; j < kBatch; ++j) current[j] = next();
  if (current[0] < 0) return;
  int64_t row[NB];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    const int64_t n = n_first + nb % kPerHalf * 16 + r16;
    row[nb] = ((n < p.n ? n : p.n - 1) + nb / kPerHalf * p.n) * p.up_row_stride;
  }
  // Where the lane's row of block b has its rank values (rows past the last and rows without an adapter read some
  // row's, and drop what they make of them).
  auto low_of = [&](int b) {
    const int64_t m = m_first + b * 16 + r16;
    return p.low + (m < p.m ? m : p.m - 1) * layout.row_bytes(kHalves);
  };
  // The lane's chunk of eight ranks in the up rows. Up to rank 16 its place in a group is that of a value or of an error
  // (the errors follow the values), else one of each.
  const bool both = layout.width <= 16;
  const int up_at = (layout.width == 32 ? g : layout.width == 16 ? g & 1 : 0) * 8;
  const bool held = layout.has_piece(g);
  auto products = [&](auto errors_too, int group) {
    constexpr bool kErrors = decltype(errors_too)::value;
    const int64_t at = group * 32 + up_at;
    u32x4 ws[kBatch][NB];
    if (p.up_whole) {
      const int64_t whole_at = at < p.rank ? at : 0;
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        const uint16_t *up = p.up + (current[j] < 0 ? current[0] : current[j]) * p.up_stride;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) ws[j][nb] = *reinterpret_cast<const u32x4 *>(up + (row[nb] + whole_at));
      }
    } else {
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        const uint16_t *up = p.up + (current[j] < 0 ? current[0] : current[j]) * p.up_stride;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) ws[j][nb] = load8(up + row[nb], at, p.rank);
      }
    }
    // Zeros past the rank (where the row's first chunk was read) and for lanes without a piece; no infinities and NaN against
    // errors.
    const bool kept = held && at < p.rank, against_errors = layout.errors(g);
#pragma unroll
    for (int j = 0; j < kBatch; ++j)
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        if (!kept) ws[j][nb] = u32x4{0, 0, 0, 0};
        if constexpr (!kErrors) ws[j][nb] = finite_only<T>(ws[j][nb], against_errors);
      }
    // Two token blocks at a time: all at once do not fit the registers of the large shapes.
    constexpr int kPair = MB < 2 ? MB : 2;
    static_assert(MB == 3 || MB % kPair == 0, "whole pairs");
#pragma unroll
    for (int first = 0; first < MB; first += kPair) {
      u32x4 values[kHalves][kPair], errors[kHalves][kPair];
      float factor[kHalves][kPair];
#pragma unroll
      for (int h = 0; h < kHalves; ++h) {
        const int64_t of = static_cast<int64_t>(h * layout.groups + group) * layout.group_bytes();
#pragma unroll
        for (int i = 0; i < kPair; ++i) {
          if (first + i >= MB) continue;
          const char *from = low_of(first + i) + of;
          values[h][i] = *reinterpret_cast<const u32x4 *>(from + layout.piece_at(g));
          if constexpr (kErrors) errors[h][i] = *reinterpret_cast<const u32x4 *>(from + layout.errors_at(g));
          if constexpr (std::is_same<T, F16>::value) factor[h][i] = *reinterpret_cast<const float *>(from + layout.factor_at());
        }
      }
      const u32x4 nothing{0, 0, 0, 0};
#pragma unroll
      for (int h = 0; h < kHalves; ++h)
#pragma unroll
        for (int i = 0; i < kPair; ++i) {
          const int b = first + i;
          if (b >= MB) continue;
          if (!held) values[h][i] = nothing;
#pragma unroll
          for (int j = 0; j < kBatch; ++j) {
            const bool own = current[j] >= 0 && mine.of[b] == current[j];
            if (ballot(own) == 0) continue;
#pragma unroll
            for (int of = 0; of < kPerHalf; ++of) {
              const int nb = h * kPerHalf + of;
              floatx4 part = T::mfma(ws[j][nb], values[h][i], floatx4{0.0f, 0.0f, 0.0f, 0.0f});
              if constexpr (kErrors) {
                // Not finite only where an up weight is not, and the values' sum is not then either: any finite number leaves it
                // as it is.
                const floatx4 rest = T::mfma(ws[j][nb], errors[h][i], floatx4{0.0f, 0.0f, 0.0f, 0.0f});
#pragma unroll
                for (int c = 0; c < 4; ++c) part[c] += __builtin_amdgcn_fmed3f(rest[c], -3.402823466e38f, 3.402823466e38f);
              }
#pragma unroll
              for (int c = 0; c < 4; ++c) {
                const float v = std::is_same<T, F16>::value ? part[c] * factor[h][i] : part[c];
                acc[nb][b][c] += own ? v : 0.0f;
              }
            }
          }
        }
      if constexpr (MB > kPair) __builtin_amdgcn_sched_barrier(0);
    }
  };
  for (;;) {
    for (int group = 0; group < layout.groups; ++group) {
      if (both) products(std::false_type{}, group);
      else products(std::true_type{}, group);
    }
    if (current[kBatch - 1] < 0) break;
#pragma unroll
    for (int j = 0; j < kBatch; ++j) current[j] = next();
    if (current[0] < 0) break;
  }
  // The last loads, which not every wavefront uses (vmcnt 0, nothing else): else the compiler waits for them, and the
  // stages in flight, in every turn of the walk, where a register is used again (256 x 4096 x 2048 39 us, 30 so).
  __builtin_amdgcn_s_waitcnt(0x0f70);
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
