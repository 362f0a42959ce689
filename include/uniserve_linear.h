// SPDX-License-Identifier: Apache-2.0
//
// Dense products with their epilogue: the projections around the routed experts, and a shared
// expert's two.
//
//   uniserve_linear        out = act(input . weight^T + bias) * sigmoid(gate) + residual
//   uniserve_gated_linear  out = (input . up^T + up_bias) * act(input . gate^T + gate_bias), where
//                          `weight` holds the n up rows and then the n gate rows, as an expert's FC1
//                          stack does
//
// input [m, k] and weight [n, k] (gated: [2 n, k]) are bf16 or f16, row-major with unit column stride
// and row strides in elements. Sums, bias, activation, gate and residual are FP32, rounded once into
// the output. Every factor and addend but the product is optional: bias [n] (gated: [2 n]) in the
// inputs' type or FP32; `activation` UNISERVE_ACTIVATION_NONE, _SILU or _GELU_TANH (gated: not none);
// one gate logit per row, in the inputs' type, gate_stride elements apart; residual [m, n] in the
// output's type. The output is the inputs' type, or FP32 (uniserve_linear: a router's logits).
//
// Any alignment and any k is served. Row strides are no shorter than the rows (the gate's may be 0: one
// logit for all rows); those of absent arrays and single rows are not read. Refused are m or k of 2^31
// and more, n of 2^30 and more, an array of more than 2^40 elements from its first row to its last, and
// an output of more than 2^24 - 1 tiles of 64 x 64 (gated: 64 x 32). The fast kernels take rows of whole
// 16 bytes (k, base addresses and row strides of the input and the weight) at row strides of up to 2^22
// elements; other rows go through registers. The output may be the residual itself (same address and
// stride), in place; an output that overlaps an input in any other way is refused. Nothing is allocated,
// no workspace is used and the calls may be captured. Results do not depend on what else runs.

#pragma once

#include "uniserve_abi.h"

#define UNISERVE_ACTIVATION_NONE (-1)

struct uniserve_linear_call {
  const void *input;     ///< [m, k] dtype
  const void *weight;    ///< [n, k] dtype; gated: [2 n, k], up rows then gate rows
  const void *bias;      ///< [n] (gated: [2 n]) bias_dtype, or null
  const void *gate;      ///< [m] dtype, gate_stride apart, or null; gated: null
  const void *residual;  ///< [m, n] out_dtype, or null; gated: null
  void *out;             ///< [m, n] out_dtype
  int64_t m;
  int64_t n;
  int64_t k;
  int64_t input_row_stride;
  int64_t weight_row_stride;
  int64_t gate_stride;
  int64_t residual_row_stride;
  int64_t out_row_stride;
  int64_t dtype;         ///< bf16 or f16
  int64_t bias_dtype;    ///< dtype or f32
  int64_t out_dtype;     ///< dtype or f32; gated: dtype
  int64_t activation;
  char error[512];
};

UNISERVE_EXTERN_C int32_t uniserve_linear(const struct uniserve_linear_call *call, void *stream);
UNISERVE_EXTERN_C int32_t uniserve_gated_linear(const struct uniserve_linear_call *call, void *stream);
