// SPDX-License-Identifier: Apache-2.0
//
// What the dense product kernels share: the launch parameters, the two element types' matrix
// instruction, and the epilogue.
#pragma once

#include "common.hpp"
#include "uniserve_linear.h"

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
  int32_t rows_of_16;    ///< input and weight rows start at 16-byte aligned addresses and k is whole 8
  int32_t out_of_4;      ///< out (and residual) rows take four columns at an aligned address
};

struct Bf16 {
  static __device__ __forceinline__ float to_f32(uint16_t bits) { return bf16_to_f32(bits); }
  static __device__ __forceinline__ uint16_t from_f32(float v) { return f32_to_bf16(v); }
  static __device__ __forceinline__ uint32_t pack2(float lo, float hi) { return pack_bf16x2(lo, hi); }
  static __device__ __forceinline__ floatx4 mfma(u32x4 a, u32x4 b, floatx4 c) { return mfma_16x16x32_bf16(a, b, c); }
};

struct F16 {
  typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
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

/// The row's factor: sigmoid of its gate logit, or 1.
template <class T>
__device__ __forceinline__ float row_gate(const LinearParams &p, int64_t m) {
  if (p.gate == nullptr) return 1.0f;
  const float g = T::to_f32(p.gate[m * p.gate_stride]);
  return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-g * 1.4426950408889634f));
}

/// Columns n .. n + 3 (those below p.n) of row m from their four sums (gated: the up halves' and the
/// gate halves'): bias, activation, row gate, residual, one rounding.
template <class T, bool kGated>
__device__ __forceinline__ void finish4(const LinearParams &p, int64_t m, int64_t n, const floatx4 &sums,
                                        const floatx4 &gate_sums, float factor) {
  const int count = p.n - n < 4 ? static_cast<int>(p.n - n) : 4;
  if (count <= 0) return;
  float v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[i] = sums[i];
    if (p.bias != nullptr && i < count) v[i] += bias_at<T>(p, n + i);
  }
  if constexpr (kGated) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float g = gate_sums[i];
      if (p.bias != nullptr && i < count) g += bias_at<T>(p, p.n + n + i);
      v[i] *= gate(g, p.activation);
    }
  } else if (p.activation != UNISERVE_ACTIVATION_NONE) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = gate(v[i], p.activation);
  }
  const int64_t at = m * p.out_stride + n;
  const int64_t from = m * p.residual_stride + n;
  if (!kGated) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] *= factor;
  }
  if (p.out_f32) {
    float *out = static_cast<float *>(p.out) + at;
    const float *residual = static_cast<const float *>(p.residual) + from;
    if (p.out_of_4 && count == 4) {
      floatx4 r = {0.0f, 0.0f, 0.0f, 0.0f};
      if (p.residual != nullptr) r = *reinterpret_cast<const floatx4 *>(residual);
      *reinterpret_cast<floatx4 *>(out) = floatx4{v[0] + r[0], v[1] + r[1], v[2] + r[2], v[3] + r[3]};
      return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < count) out[i] = p.residual != nullptr ? v[i] + residual[i] : v[i];
    return;
  }
  uint16_t *out = static_cast<uint16_t *>(p.out) + at;
  const uint16_t *residual = static_cast<const uint16_t *>(p.residual) + from;
  if (p.out_of_4 && count == 4) {
    if (p.residual != nullptr) {
      const uint2 r = *reinterpret_cast<const uint2 *>(residual);
      v[0] += T::to_f32(static_cast<uint16_t>(r.x));
      v[1] += T::to_f32(static_cast<uint16_t>(r.x >> 16));
      v[2] += T::to_f32(static_cast<uint16_t>(r.y));
      v[3] += T::to_f32(static_cast<uint16_t>(r.y >> 16));
    }
    *reinterpret_cast<uint2 *>(out) = uint2{T::pack2(v[0], v[1]), T::pack2(v[2], v[3])};
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (i < count) out[i] = T::from_f32(p.residual != nullptr ? v[i] + T::to_f32(residual[i]) : v[i]);
}

}  // namespace linear
}  // namespace uniserve
