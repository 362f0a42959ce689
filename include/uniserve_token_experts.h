// SPDX-License-Identifier: Apache-2.0
//
// token_experts: the routed experts of an MoE layer for a few tokens, in two kernels and without a sort's maps:
//
//   out[t] = residual[t] + sum over k of weights[t, k] * down[e] . (act(gate[e] . input[t]) * (up[e] . input[t])),
//   e = ids[t, k] - first_expert
//
// input [tokens, hidden] is bf16 or f16, as are the stacks, both contiguous: up_gate [experts, 2 width, hidden]
// (an expert's up rows and then its gate rows) and down [experts, hidden, width]. ids and weights [tokens, top]
// (int32, FP32, contiguous) are any router's: ids outside [first_expert, first_expert + experts) are routes of other
// ranks or none at all (-1) and add nothing, whatever their weight; an id that comes twice in a row counts twice. act
// is UNISERVE_ACTIVATION_SILU or _GELU_TANH. residual (the output's type, or null) may be the output itself,
// in place. Rows without a route are the residual, or zeros.
//
// Sums are FP32. In the second product a gated value is a pair of the type's elements, the value and its rounding error,
// and the output is rounded once. bf16: 16 bits of significand. f16: 64 consecutive values of a route share a power of two,
// so that values of any size are served; 22 bits, or 2^-25 of the largest of the 64 where a value is small beside it.
// A row's result does not depend on the other rows. (From some 32 tokens on, bf16 layers that uniserve_gather_gemm and
// uniserve_route_gemm serve are computed faster by those.) What an expert holds, infinities and NaN too, reaches the rows
// routed to it and no others, and is there what the formula makes of it.
//
// `workspace` is uniserve_token_experts_workspace(tokens, top, width) bytes, 16-byte aligned; its contents before the
// call do not matter and after it are of no use. Calls that may overlap in time need one each. Nothing is allocated and
// the call may be captured. Any hidden and width are served; rows of whole 16 bytes (hidden, width, addresses,
// the input's stride) are read fastest. Refused are more than UNISERVE_TOKEN_EXPERTS_MAX_TOKENS tokens, a top above
// UNISERVE_TOKEN_EXPERTS_MAX_TOP, more than UNISERVE_TOKEN_EXPERTS_MAX_EXPERTS experts, extents of 2^24 and more, an
// output or workspace that overlaps an input (but for the residual) and each other.

#pragma once

#include "uniserve_abi.h"

#define UNISERVE_TOKEN_EXPERTS_MAX_TOKENS 64
#define UNISERVE_TOKEN_EXPERTS_MAX_TOP 32
#define UNISERVE_TOKEN_EXPERTS_MAX_EXPERTS 1024

struct uniserve_token_experts_call {
  const void *input;       ///< [tokens, hidden] dtype
  const int32_t *ids;      ///< [tokens, top]
  const float *weights;    ///< [tokens, top]
  const void *up_gate;     ///< [experts, 2 width, hidden] dtype
  const void *down;        ///< [experts, hidden, width] dtype
  const void *residual;    ///< [tokens, hidden] dtype, or null
  void *out;               ///< [tokens, hidden] dtype
  void *workspace;
  int64_t workspace_bytes;
  int64_t tokens;
  int64_t top;
  int64_t hidden;
  int64_t width;
  int64_t experts;
  int64_t first_expert;
  int64_t input_row_stride;
  int64_t residual_row_stride;
  int64_t out_row_stride;
  int32_t dtype;
  int32_t activation;
  char error[512];
};

UNISERVE_EXTERN_C int64_t uniserve_token_experts_workspace(int64_t tokens, int64_t top, int64_t width);
UNISERVE_EXTERN_C int32_t uniserve_token_experts(const struct uniserve_token_experts_call *call, void *stream);
