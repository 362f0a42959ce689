// SPDX-License-Identifier: Apache-2.0
//
// add_norm: a block's output joined to the residual stream and normed for the next block, in one pass.
// Row by row, with N a norm over the row's `width` elements:
//
//   b      = input, or N(input) with post, post_bias    (the norm after the block)
//   total  = residual_scale * residual + scale * sigmoid(gate) * channels * b
//   out    = N(total) with weight, bias                 (the norm before the next block)
//
//   rms    N(v) = v / sqrt(mean(v^2) + eps) * (offset + w)
//   layer  N(v) = (v - mean(v)) / sqrt(mean((v - mean(v))^2) + eps) * (offset + w) + bias
//
// `offset` is 0, or 1 for weights that are stored as their distance from one. Everything is held in
// FP32 from the inputs to the two outputs, each rounded once: the second norm reads the sums before
// they are rounded into `total`. input and out are bf16, f16 or f32; residual and total are of that
// type or f32; the vectors (post, post_bias, channels, weight, bias; [width] each, contiguous) are all
// of that type or all f32; gate is one logit per row, in the input's type, gate_stride elements apart.
//
// Optional are residual, post, gate, channels, the biases (layer norms alone have them, post_bias with
// post only), total, and weight with out (a join without a norm); not both outputs. Any alignment, any
// width up to UNISERVE_ADD_NORM_MAX_WIDTH and any row stride no shorter than the row is served; strides
// of absent arrays and single rows are not read. An output may be the input or the residual itself
// (same address, stride and element size), in place; an output that overlaps an input or the other output
// in any other way is refused. Nothing is allocated, no workspace is used and the call may be captured.

#pragma once

#include "uniserve_abi.h"

#define UNISERVE_ADD_NORM_MAX_WIDTH 32768

enum uniserve_norm
#ifdef __cplusplus
    : int32_t
#endif
{
  UNISERVE_NORM_RMS = 0,
  UNISERVE_NORM_LAYER = 1,
};

struct uniserve_add_norm_call {
  const void *input;      ///< [rows, width] dtype
  const void *residual;   ///< [rows, width] total_dtype, or null
  const void *post;       ///< [width] vector_dtype, or null: no norm after the block
  const void *post_bias;  ///< [width] vector_dtype, or null
  const void *gate;       ///< [rows] dtype, gate_stride apart, or null
  const void *channels;   ///< [width] vector_dtype, or null
  const void *weight;     ///< [width] vector_dtype; null with `out`
  const void *bias;       ///< [width] vector_dtype, or null
  void *total;            ///< [rows, width] total_dtype, or null
  void *out;              ///< [rows, width] dtype, or null: no norm before the next block
  int64_t rows;
  int64_t width;
  int64_t input_row_stride;
  int64_t residual_row_stride;
  int64_t total_row_stride;
  int64_t out_row_stride;
  int64_t gate_stride;
  int32_t dtype;
  int32_t total_dtype;
  int32_t vector_dtype;
  int32_t norm;
  float eps;
  float offset;
  float scale;
  float residual_scale;
  char error[512];
};

UNISERVE_EXTERN_C int32_t uniserve_add_norm(const struct uniserve_add_norm_call *call, void *stream);
