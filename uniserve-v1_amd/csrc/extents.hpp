// SPDX-License-Identifier: Apache-2.0
//
// What the operators' entries check about the arrays of a call.
#pragma once

#include <cstdint>

namespace uniserve {

/// `rows` rows of `bytes` bytes, `stride` bytes apart.
struct Extent {
  const char *first;
  int64_t rows, bytes, stride;
};

/// `rows` rows of `columns` elements of `element` bytes, `stride` elements apart.
inline Extent extent(const void *first, int64_t rows, int64_t columns, int64_t stride, int64_t element) {
  return Extent{static_cast<const char *>(first), rows, columns * element, stride * element};
}

/// Whether two arrays share a byte. Rows of equal strides may interleave (two column ranges of one
/// buffer); of different strides, arrays whose ranges meet count as sharing.
inline bool overlap(const Extent &a, const Extent &b) {
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

inline bool aligned_to(const void *pointer, uintptr_t bytes) { return reinterpret_cast<uintptr_t>(pointer) % bytes == 0; }

/// Extents whose product of rows and stride stays far below 2^63 bytes.
constexpr int64_t kMostElements = int64_t{1} << 40;

}  // namespace uniserve
