// SPDX-License-Identifier: Apache-2.0
//
// The dense products with the low-rank adapters of many requests beside the shared weight: what
// uniserve_linear and uniserve_gated_linear compute (uniserve_linear.h), with each row's own adapter in the
// product. With a = adapter[t] the adapter of row t and A, B its two factors:
//
//   input[t] . weight^T   becomes   input[t] . weight^T + scales[a] * (input[t] . A^T) . B^T
//
// before the bias, the activation and the rest of the epilogue. down holds the factors A, [adapters, rank,
// k]; up the factors B, [adapters, n, rank]. uniserve_adapter_gated_linear's halves have factors of their
// own: down [adapters, 2 rank, k], the up half's rows and then the gate half's; up [adapters, 2 n, rank]
// likewise. Adapters of a smaller rank than the stack's are padded with zeros. An index below 0 or not below
// `adapters` names none: such a row gets the product alone, and no adapter is read for it. What an adapter
// holds, infinities and NaN too, reaches the rows that name it and no others, and is there what the formula makes of it.
//
// down, up and the rows are of one type (bf16 or f16), their last axes contiguous; scales are FP32, or null
// for ones. Sums are FP32; between the factors a row's rank values are held as a pair of the type's elements
// (the value and its rounding error: 16 bits of significand or more; f16 pairs share a power of two per 32
// values, so they neither overflow nor lose their error to subnormals), so that both products use the matrix units. One
// rounding into the output, as without adapters. Row indices in any order are served; a run of rows with one
// adapter is fastest.
//
// `workspace` is uniserve_adapter_workspace(m, rank rows) bytes, 16-byte aligned, rank rows being the rows of
// one adapter in down; its contents before the call do not matter and after it are of no use. Calls that may
// overlap in time need one each. Two launches; nothing is allocated and the call may be captured. Refused
// besides what the products refuse: more than 2^23 rows, a rank above UNISERVE_ADAPTER_MAX_RANK, stacks of more than 2^40
// elements, an output that overlaps a stack, the indices, the scales or the workspace, and a workspace that
// overlaps any input.

#pragma once

#include "uniserve_linear.h"

#define UNISERVE_ADAPTER_MAX_RANK 512

struct uniserve_adapter_linear_call {
  struct uniserve_linear_call product;  ///< the call without adapters, and where a refusal's message goes
  const void *down;        ///< [adapters, rank, k] product.dtype; gated: [adapters, 2 rank, k]
  const void *up;          ///< [adapters, n, rank] product.dtype; gated: [adapters, 2 n, rank]
  const int32_t *adapter;  ///< [m]
  const float *scales;     ///< [adapters], or null
  void *workspace;
  int64_t workspace_bytes;
  int64_t adapters;
  int64_t rank;
  int64_t down_stride;      ///< elements from an adapter's factor to the next's
  int64_t down_row_stride;
  int64_t up_stride;
  int64_t up_row_stride;
};

UNISERVE_EXTERN_C int64_t uniserve_adapter_workspace(int64_t rows, int64_t rank_rows);
UNISERVE_EXTERN_C int32_t uniserve_adapter_linear(const struct uniserve_adapter_linear_call *call, void *stream);
UNISERVE_EXTERN_C int32_t uniserve_adapter_gated_linear(const struct uniserve_adapter_linear_call *call, void *stream);
