// SPDX-License-Identifier: Apache-2.0
//
// The row kernel of add_norm and its choice of shape.
#pragma once

#include "common.hpp"
#include "uniserve_add_norm.h"

namespace uniserve {
namespace add_norm {

struct AddNormParams {
  const void *x, *residual, *post, *post_bias, *gate, *channels, *weight, *bias;
  void *total, *out;
  int64_t rows;
  int64_t x_stride, residual_stride, total_stride, out_stride, gate_stride;
  int32_t width;
  int32_t vector_f32;  ///< the vectors are FP32, not the rows' type
  int32_t layer;
  float eps, offset, scale, residual_scale, inverse_width;
};

struct Bf16 {
  typedef uint16_t type;
  static __device__ __forceinline__ float widen(uint16_t v) { return bf16_to_f32(v); }
  static __device__ __forceinline__ uint32_t pack2(float lo, float hi) { return pack_bf16x2(lo, hi); }
};
struct F16 {
  typedef uint16_t type;
  static __device__ __forceinline__ float widen(uint16_t v) { return static_cast<float>(__builtin_bit_cast(_Float16, v)); }
  static __device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    return static_cast<uint32_t>(__builtin_bit_cast(uint16_t, static_cast<_Float16>(lo))) |
           static_cast<uint32_t>(__builtin_bit_cast(uint16_t, static_cast<_Float16>(hi))) << 16;
  }
};
struct F32 {
  typedef float type;
};

/// Eight consecutive elements as they lie in memory.
template <class T>
struct Eight {
  static constexpr bool kWide = sizeof(typename T::type) == 4;
  u32x4 bits[kWide ? 2 : 1];

  /// Elements at .. at + 7 of a row, the first `count` of them where fewer are left (else zeros), at any alignment.
  __device__ __forceinline__ void load(const void *row, int64_t at, int count) {
    const typename T::type *from = static_cast<const typename T::type *>(row) + at;
    if (count >= 8) {
      __builtin_memcpy(bits, from, sizeof(bits));
      return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      uint32_t v = 0;
      if (i < count) {
        if constexpr (kWide) v = __float_as_uint(from[i]);
        else v = from[i];
      }
      if constexpr (kWide) bits[i / 4][i % 4] = v;
      else bits[0][i / 2] = i % 2 == 0 ? v : bits[0][i / 2] | v << 16;
    }
  }
  __device__ __forceinline__ float operator[](int i) const {
    if constexpr (kWide) return __uint_as_float(bits[i / 4][i % 4]);
    else return T::widen(static_cast<uint16_t>(bits[0][i / 2] >> (i % 2 * 16)));
  }
  __device__ __forceinline__ void set(const float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < (kWide ? 8 : 4); ++i) {
      if constexpr (kWide) bits[i / 4][i % 4] = __float_as_uint(v[i]);
      else bits[0][i] = T::pack2(v[2 * i], v[2 * i + 1]);
    }
  }
  __device__ __forceinline__ void store(void *row, int64_t at, int count) const {
    typename T::type *to = static_cast<typename T::type *>(row) + at;
    if (count >= 8) {
      __builtin_memcpy(to, bits, sizeof(bits));
      return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < count) {
        if constexpr (kWide) to[i] = __uint_as_float(bits[i / 4][i % 4]);
        else to[i] = static_cast<uint16_t>(bits[0][i / 2] >> (i % 2 * 16));
      }
  }
};

/// The sum of every lane's value, in all lanes: over each row of sixteen lanes by DPP moves (as row16_max), then over
/// pairs of rows and of halves, by gfx950's swaps.
__device__ __forceinline__ float wave_sum(float v) {
  const auto moved = [](auto of, float x) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), decltype(of)::value, 0xf, 0xf, false));
  };
  v += moved(std::integral_constant<int, 0xb1>{}, v);
  v += moved(std::integral_constant<int, 0x4e>{}, v);
  v += moved(std::integral_constant<int, 0x141>{}, v);
  v += moved(std::integral_constant<int, 0x140>{}, v);
  const auto rows = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(rows[0]) + __uint_as_float(rows[1]);
  const auto halves = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(halves[0]) + __uint_as_float(halves[1]);
}

/// kTeam threads to a row, kChunks chunks of eight elements a thread: chunk c of a row is thread c % kTeam's.
/// kWhole: rows of whole chunks.
template <class X, class R, int kTeam, int kChunks, bool kWhole>
__global__ void __launch_bounds__(kTeam < 128 ? 256 : kTeam) add_norm_kernel(AddNormParams p) {
  constexpr int kTeams = kTeam < 128 ? 256 / kTeam : 1;  // of a workgroup: several are a wavefront each, without barriers
  constexpr int kWaves = kTeam / kWave;
  __shared__ float partial[2][kWaves > 1 ? kWaves : 1];
  const int t = static_cast<int>(threadIdx.x) % kTeam;
  int parity = 0;
  // Two buffers in turn: a wavefront writes one again only after the barrier of the sum between, which all
  // pass after they have read it.
  auto team_sum = [&](float v) {
    v = wave_sum(v);
    if constexpr (kWaves > 1) {
      if (lane_id() == 0) partial[parity][t / kWave] = v;
      __syncthreads();
      v = 0.0f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) v += partial[parity][w];
      parity ^= 1;
    }
    return v;
  };
  auto at = [&](int i) { return (t + i * kTeam) * 8; };
  auto left = [&](int i) { return kWhole ? (at(i) < p.width ? 8 : 0) : p.width - at(i); };
  // v[j] of chunk i becomes f(v, vector[j]).
  auto apply = [&](float (&v)[kChunks][8], const void *vector, auto f) {
    if (p.vector_f32) {
#pragma unroll
      for (int i = 0; i < kChunks; ++i) {
        if (left(i) <= 0) continue;
        Eight<F32> w;
        w.load(vector, at(i), left(i));
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] = f(v[i][j], w[j]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < kChunks; ++i) {
        if (left(i) <= 0) continue;
        Eight<X> w;
        w.load(vector, at(i), left(i));
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] = f(v[i][j], w[j]);
      }
    }
  };
  // Elements past the row's end stay out of the sums.
  auto norm = [&](float (&v)[kChunks][8], const void *weight, const void *bias) {
    if (p.layer) {
      float sum = 0.0f;
#pragma unroll
      for (int i = 0; i < kChunks; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (j < left(i)) sum += v[i][j];
      const float mean = team_sum(sum) * p.inverse_width;
#pragma unroll
      for (int i = 0; i < kChunks; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] -= mean;
    }
    float squares = 0.0f;
#pragma unroll
    for (int i = 0; i < kChunks; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j < left(i)) squares = __builtin_fmaf(v[i][j], v[i][j], squares);
    const float factor = 1.0f / __builtin_sqrtf(team_sum(squares) * p.inverse_width + p.eps);
    apply(v, weight, [&](float a, float w) { return a * factor * (p.offset + w); });
    if (bias != nullptr) apply(v, bias, [](float a, float b) { return a + b; });
  };

  for (int64_t row = static_cast<int64_t>(blockIdx.x) * kTeams + threadIdx.x / kTeam; row < p.rows;
       row += static_cast<int64_t>(gridDim.x) * kTeams) {
    const typename X::type *x = static_cast<const typename X::type *>(p.x) + row * p.x_stride;
    Eight<X> xs[kChunks];
    Eight<R> rs[kChunks];
#pragma unroll
    for (int i = 0; i < kChunks; ++i)
      if (left(i) > 0) xs[i].load(x, at(i), left(i));
    if (p.residual != nullptr) {
      const typename R::type *residual = static_cast<const typename R::type *>(p.residual) + row * p.residual_stride;
#pragma unroll
      for (int i = 0; i < kChunks; ++i)
        if (left(i) > 0) rs[i].load(residual, at(i), left(i));
    }
    float factor = p.scale;
    if (p.gate != nullptr) {
      typename X::type g = static_cast<const typename X::type *>(p.gate)[row * p.gate_stride];
      float logit;
      if constexpr (sizeof(g) == 4) logit = g;
      else logit = X::widen(g);
      // The hardware's exponential of a rounded product is off by the logit's size in u, 80 of them at -80: nothing beside the
      // rounding of 16-bit outputs. FP32 ones take expf and a quotient, four u at most (64 x 4096 on an FP32 stream 3.6 us
      // against 3.5).
      if constexpr (sizeof(typename X::type) == 4 || sizeof(typename R::type) == 4) factor *= 1.0f / (1.0f + expf(-logit));
      else factor *= __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-logit * 1.4426950408889634f));
    }
    float v[kChunks][8];
#pragma unroll
    for (int i = 0; i < kChunks; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] = left(i) > 0 ? xs[i][j] : 0.0f;
    if (p.post != nullptr) norm(v, p.post, p.post_bias);
    if (p.channels != nullptr) apply(v, p.channels, [](float a, float c) { return a * c; });
#pragma unroll
    for (int i = 0; i < kChunks; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        v[i][j] *= factor;
        if (p.residual != nullptr && left(i) > 0) v[i][j] = __builtin_fmaf(p.residual_scale, rs[i][j], v[i][j]);
      }
    if (p.total != nullptr) {
      typename R::type *total = static_cast<typename R::type *>(p.total) + row * p.total_stride;
#pragma unroll
      for (int i = 0; i < kChunks; ++i) {
        if (left(i) <= 0) continue;
        Eight<R> e;
        e.set(v[i]);
        e.store(total, at(i), left(i));
      }
    }
    if (p.weight != nullptr) {
      norm(v, p.weight, p.bias);
      typename X::type *out = static_cast<typename X::type *>(p.out) + row * p.out_stride;
#pragma unroll
      for (int i = 0; i < kChunks; ++i) {
        if (left(i) <= 0) continue;
        Eight<X> e;
        e.set(v[i]);
        e.store(out, at(i), left(i));
      }
    }
  }
}

template <class X, class R, int kTeam, int kChunks>
void launch_shape(const AddNormParams &p, hipStream_t stream) {
  constexpr int kTeams = kTeam < 128 ? 256 / kTeam : 1;
  constexpr int64_t kMostBlocks = int64_t{1} << 20;  // rows past them are the same blocks' next
  const int64_t blocks = ceil_div<int64_t>(p.rows, kTeams);
  const dim3 grid(static_cast<uint32_t>(blocks < kMostBlocks ? blocks : kMostBlocks)), threads(kTeam * kTeams);
  if (p.width % 8 == 0) hipLaunchKernelGGL((add_norm_kernel<X, R, kTeam, kChunks, true>), grid, threads, 0, stream, p);
  else hipLaunchKernelGGL((add_norm_kernel<X, R, kTeam, kChunks, false>), grid, threads, 0, stream, p);
}

/// One chunk a thread as far as a workgroup's threads go. 8192 x 4096 bf16 (268 MB), plain and with a norm after the
/// block: 512 threads a row 39.5 and 43.2 us, 256 of two chunks 42.1 and 45.2, 128 of four 56.4 and 74.2, a
/// wavefront a row 60 and 99 (its registers leave room for one wavefront a SIMD); 64 x 4096: 2.9 and 3.5, 3.3
/// and 4.0, 4.1 and 5.2, 6.5 and 8.6. Bound by the bytes from some hundred rows on (8192 x 4096 at 6.8 TB/s
/// on the same tensors again and again, 4.5 over three sets, where a copy of 4 GiB runs at 4.7), below by the launch
/// and the row's chain of loads and sums (one row of 2048 2.4 us, 2.9 with both norms). Rows of more than 16384
/// elements spill 46 to 357 registers, bf16 ones of more than 8192 on an FP32 stream 8, of no whole eights 6 to 16.
template <class X, class R>
void launch(const AddNormParams &p, hipStream_t stream) {
  const int32_t chunks = ceil_div(p.width, 8);
  if (chunks <= 64) return launch_shape<X, R, 64, 1>(p, stream);
  if (chunks <= 128) return launch_shape<X, R, 128, 1>(p, stream);
  if (chunks <= 256) return launch_shape<X, R, 256, 1>(p, stream);
  if (chunks <= 512) return launch_shape<X, R, 512, 1>(p, stream);
  if (chunks <= 1024) return launch_shape<X, R, 1024, 1>(p, stream);
  if (chunks <= 2048) return launch_shape<X, R, 1024, 2>(p, stream);
  return launch_shape<X, R, 1024, 4>(p, stream);
}

}  // namespace add_norm
}  // namespace uniserve
