// SPDX-License-Identifier: Apache-2.0
//
// What the dense product kernels share: the launch parameters, the two element types' matrix
// instruction, and the epilogue.
#pragma once

#include "common.hpp"
#include "low_layout.hpp"
#include "uniserve_adapter_linear.h"

namespace uniserve {
namespace linear {

struct LinearParams {
  const uint16_t *x;     ///< [m, k]
  const uint16_t *w;     ///< [n, k]; gated: [2 n, k]
  const void *bias;      ///< [n]; gated: [2 n]; or null
  const uint16_t *gate;  ///< [m] row gate logits, or null
  const void *residual;  ///< [m, n], or null
  void *out;             ///< [m, n]
  int64_t m, n, k;
  int64_t x_stride, w_stride, gate_stride, residual_stride, out_stride;
  int32_t bias_f32;
  int32_t out_f32;
  int32_t activation;
  int32_t by_dma;        ///< input and weight rows suit the tile kernels' loads
};

/// A product whose rows have low-rank adapters.
struct AdapterParams : LinearParams {
  const uint16_t *down;    ///< [adapters, rank, k]; gated: [adapters, 2 rank, k]
  const uint16_t *up;      ///< [adapters, n, rank]; gated: [adapters, 2 n, rank]
  const int32_t *adapter;  ///< [m]
  const float *scales;     ///< [adapters], or null
  char *low;               ///< the workspace: each row's rank values
  int64_t down_stride, down_row_stride, up_stride, up_row_stride;
  int32_t adapters, rank;
  int32_t down_by_dma;  ///< input and down rows suit the tile kernels' loads
  int32_t up_whole;     ///< up rows are whole 16-byte pieces, 256 of them within 32-bit byte offsets
};

/// The adapters' first factor as a product: columns are the rank values in their layout's order, n of them.
struct RankParams : AdapterParams {
  int32_t width, groups, halves;  ///< LowLayout
  /// Column j's row of an adapter's first factor (past the rank: the last one; the value is dropped).
  __device__ __forceinline__ int64_t down_row(int64_t j) const {
    const int at = static_cast<int>(j < n ? j : n - 1);
    const int group = at / width, half = group / groups, in_half = (group - half * groups) * width + at % width;
    return half * rank + (in_half < rank ? in_half : rank - 1);
  }
};

/// Launches a call that was found servable.
void launch_bf16(const LinearParams &p, bool gated, hipStream_t stream);
void launch_f16(const LinearParams &p, bool gated, hipStream_t stream);
void launch_adapters_bf16(const AdapterParams &p, bool gated, hipStream_t stream);
void launch_adapters_f16(const AdapterParams &p, bool gated, hipStream_t stream);

struct Bf16 {
  static __device__ __forceinline__ float low(uint32_t pair) { return __uint_as_float(pair << 16); }
  static __device__ __forceinline__ float high(uint32_t pair) { return __uint_as_float(pair & 0xffff0000u); }
  static __device__ __forceinline__ float to_f32(uint16_t bits) { return bf16_to_f32(bits); }
  static __device__ __forceinline__ uint16_t from_f32(float v) { return f32_to_bf16(v); }
  static __device__ __forceinline__ uint32_t pack2(float lo, float hi) { return pack_bf16x2(lo, hi); }
  static __device__ __forceinline__ floatx4 mfma(u32x4 a, u32x4 b, floatx4 c) { return mfma_16x16x32_bf16(a, b, c); }
};

struct F16 {
  typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
  static __device__ __forceinline__ float low(uint32_t pair) { return to_f32(static_cast<uint16_t>(pair)); }
  static __device__ __forceinline__ float high(uint32_t pair) { return to_f32(static_cast<uint16_t>(pair >> 16)); }
  static __device__ __forceinline__ float to_f32(uint16_t bits) { return static_cast<float>(__builtin_bit_cast(_Float16, bits)); }
  static __device__ __forceinline__ uint16_t from_f32(float v) { return __builtin_bit_cast(uint16_t, static_cast<_Float16>(v)); }
  static __device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    return static_cast<uint32_t>(from_f32(lo)) | (static_cast<uint32_t>(from_f32(hi)) << 16);
  }
  /// As mfma_16x16x32_bf16, over f16.
  static __device__ __forceinline__ floatx4 mfma(u32x4 a, u32x4 b, floatx4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
};

template <class T>
__device__ __forceinline__ float bias_at(const LinearParams &p, int64_t n) {
  return p.bias_f32 ? static_cast<const float *>(p.bias)[n] : T::to_f32(static_cast<const uint16_t *>(p.bias)[n]);
}

template <class T>
__device__ __forceinline__ float residual_at(const LinearParams &p, int64_t m, int64_t n) {
  const int64_t at = m * p.residual_stride + n;
  return p.out_f32 ? static_cast<const float *>(p.residual)[at] : T::to_f32(static_cast<const uint16_t *>(p.residual)[at]);
}

/// Elements at .. at + 7 of a row of `width`, zeros past its end, by one 16-byte load at any alignment: where
/// fewer than eight are left, the row's last eight, moved down.
__device__ __forceinline__ u32x4 load8(const uint16_t *row, int64_t at, int64_t width) {
  uint64_t v[2] = {0, 0};
  if (width >= 8) {
    const int64_t from = at + 8 <= width ? at : width - 8;
    __builtin_memcpy(v, row + from, 16);
    const int past = at - from < 8 ? static_cast<int>(at - from) : 8;  // elements before `at`
    v[0] = past >= 4 ? v[1] : v[0];
    v[1] = past >= 4 ? 0 : v[1];
    const int bits = (past & 3) * 16;
    v[0] = bits == 0 ? v[0] : (v[0] >> bits) | (v[1] << (64 - bits));
    v[1] >>= bits;
    v[0] = past == 8 ? 0 : v[0];
  } else {
#pragma unroll 1
    for (int i = 0; i < 8; ++i) {
      const uint64_t element = at + i < width ? row[at + i] : 0;
      v[0] = (v[0] >> 16) | (v[1] << 48);
      v[1] = (v[1] >> 16) | (element << 48);
    }
  }
  return __builtin_bit_cast(u32x4, v);
}

/// The row's factor: sigmoid of its gate logit.
template <class T>
__device__ __forceinline__ float row_gate(const LinearParams &p, int64_t m) {
  const float g = T::to_f32(p.gate[m * p.gate_stride]);
  return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-g * 1.4426950408889634f));
}

/// The epilogue of eight consecutive columns n .. n + 7 (those below p.n) of some rows: the columns'
/// biases, loaded once, and what turns a row's sums into its outputs - bias, activation, row gate,
/// residual, one rounding.
template <class T, bool kGated>
struct Columns8 {
  float bias[kGated ? 16 : 8];
  int count;
  bool vectors;  ///< all eight columns: 16-byte accesses, at any alignment

  __device__ __forceinline__ Columns8(const LinearParams &p, int64_t n) {
    count = p.n - n < 8 ? (p.n > n ? static_cast<int>(p.n - n) : 0) : 8;
    vectors = count == 8;
    constexpr int kBiases = kGated ? 16 : 8;
    // Columns past the last repeat it, so that all loads go out together.
    int64_t at[kBiases];
#pragma unroll
    for (int i = 0; i < kBiases; ++i) at[i] = (n + i % 8 < p.n ? n + i % 8 : p.n - 1) + (i < 8 ? 0 : p.n);
    if (p.bias == nullptr) {
#pragma unroll
      for (int i = 0; i < kBiases; ++i) bias[i] = 0.0f;
    } else if (p.bias_f32) {
#pragma unroll
      for (int i = 0; i < kBiases; ++i) bias[i] = static_cast<const float *>(p.bias)[at[i]];
    } else {
      uint16_t bits[kBiases];
#pragma unroll
      for (int i = 0; i < kBiases; ++i) bits[i] = static_cast<const uint16_t *>(p.bias)[at[i]];
#pragma unroll
      for (int i = 0; i < kBiases; ++i) bias[i] = T::to_f32(bits[i]);
    }
  }

  /// What kRows rows m[i] read besides their sums: the loads go out together, so their latencies do not add up.
  template <int kRows>
  struct Extras {
    u32x4 residual[kRows][2];
    float factor[kRows];
  };
  template <int kRows>
  __device__ __forceinline__ void load(const LinearParams &p, const int64_t (&m)[kRows], int64_t n, Extras<kRows> &e) const {
    if constexpr (kGated) return;
    if (p.residual != nullptr) {
      const int64_t last = p.n - 1;  // repeated past the last column, whose lanes read element by element
      if (p.out_f32) {
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
          const float *from = static_cast<const float *>(p.residual) + m[i] * p.residual_stride;
          if (vectors) {
            __builtin_memcpy(&e.residual[i][0], from + n, 16);
            __builtin_memcpy(&e.residual[i][1], from + n + 4, 16);
          } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) e.residual[i][j / 4][j % 4] = __float_as_uint(from[n + j < last ? n + j : last]);
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
          const uint16_t *from = static_cast<const uint16_t *>(p.residual) + m[i] * p.residual_stride;
          if (vectors) {
            __builtin_memcpy(&e.residual[i][0], from + n, 16);
          } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
              e.residual[i][0][j] = static_cast<uint32_t>(from[n + 2 * j < last ? n + 2 * j : last]) |
                                    static_cast<uint32_t>(from[n + 2 * j + 1 < last ? n + 2 * j + 1 : last]) << 16;
          }
        }
      }
    }
    if (p.gate != nullptr) {
#pragma unroll
      for (int i = 0; i < kRows; ++i) e.factor[i] = row_gate<T>(p, m[i]);
    }
  }

  /// Row m's outputs from its sums (gated: the up halves' and the gate halves').
  __device__ __forceinline__ void finish(const LinearParams &p, int64_t m, int64_t n, const floatx4 (&sums)[2],
                                         const floatx4 (&gates)[2], const u32x4 (&residual)[2], float factor) const {
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = sums[i / 4][i % 4] + bias[i];
    if constexpr (kGated) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] *= gate(gates[i / 4][i % 4] + bias[8 + i], p.activation);
    } else {
      if (p.activation != UNISERVE_ACTIVATION_NONE) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = gate(v[i], p.activation);
      }
      if (p.gate != nullptr) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] *= factor;
      }
      if (p.residual != nullptr) {
        if (p.out_f32) {
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] += __uint_as_float(residual[i / 4][i % 4]);
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) v[2 * i] += T::low(residual[0][i]), v[2 * i + 1] += T::high(residual[0][i]);
        }
      }
    }
    if (p.out_f32) {
      float *out = static_cast<float *>(p.out) + m * p.out_stride + n;
      if (vectors) {
        __builtin_memcpy(out, v, 32);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (i < count) out[i] = v[i];
      }
    } else {
      uint16_t *out = static_cast<uint16_t *>(p.out) + m * p.out_stride + n;
      if (vectors) {
        const u32x4 packed{T::pack2(v[0], v[1]), T::pack2(v[2], v[3]), T::pack2(v[4], v[5]), T::pack2(v[6], v[7])};
        __builtin_memcpy(out, &packed, 16);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (i < count) out[i] = T::from_f32(v[i]);
      }
    }
  }
};

/// One output from its sum (gated: and its gate's), as Columns8 does eight.
template <class T, bool kGated>
__device__ __forceinline__ void finish1(const LinearParams &p, int64_t m, int64_t n, float v, float gate_sum) {
  if (p.bias != nullptr) v += bias_at<T>(p, n);
  if constexpr (kGated) {
    v *= gate(p.bias != nullptr ? gate_sum + bias_at<T>(p, p.n + n) : gate_sum, p.activation);
  } else {
    if (p.activation != UNISERVE_ACTIVATION_NONE) v = gate(v, p.activation);
    if (p.gate != nullptr) v *= row_gate<T>(p, m);
  }
  if (p.residual != nullptr) v += residual_at<T>(p, m, n);
  const int64_t at = m * p.out_stride + n;
  if (p.out_f32) static_cast<float *>(p.out)[at] = v;
  else static_cast<uint16_t *>(p.out)[at] = T::from_f32(v);
}

}  // namespace linear
}  // namespace uniserve
