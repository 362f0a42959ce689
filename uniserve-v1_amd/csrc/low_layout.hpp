// SPDX-License-Identifier: Apache-2.0
//
// Where the adapters' rank values lie between the two products. (Plain C++: the addresses are also checked without a GPU.)
#pragma once

#include <cstdint>

namespace uniserve {
namespace linear {

/// A row's rank values, group by group of at most 32 ranks (gated: the up half's groups, then the gate half's): `width`
/// elements that hold the values rounded, as many their errors, and the group's factor (FP32, f16 only: the power of
/// two that both were divided by), padded to 16 bytes.
struct LowLayout {
  int32_t width;   ///< ranks of a group: 8, 16 or 32
  int32_t groups;  ///< of a half
  constexpr explicit LowLayout(int64_t rank)
      : width(rank <= 8 ? 8 : rank <= 16 ? 16 : 32), groups(static_cast<int32_t>((rank + width - 1) / width)) {}
  constexpr int32_t group_bytes() const { return 4 * width + 16; }
  constexpr int64_t row_bytes(int halves) const { return static_cast<int64_t>(halves) * groups * group_bytes(); }

  // The matrix instruction's operand, of which the lanes l / 16 = g hold 16 bytes each. A group of eight ranks has 32
  // bytes of values and errors: the lanes behind them read the first piece, which is dropped (their own would
  // end past the last row of the workspace).
  constexpr bool has_piece(int g) const { return width >= 16 || g < 2; }
  constexpr bool errors(int g) const { return has_piece(g) && 8 * g >= width; }  ///< whether that piece holds errors
  constexpr int32_t piece_at(int g) const { return has_piece(g) ? 16 * g : 0; }
  constexpr int32_t errors_at(int g) const { return piece_at(g) + 2 * width; }  ///< of width 32, an operand of their own
  constexpr int32_t factor_at() const { return 4 * width; }
};

}  // namespace linear
}  // namespace uniserve
