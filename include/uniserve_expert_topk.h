// SPDX-License-Identifier: Apache-2.0
//
// expert_topk: the expert choice of routers that topk_softmax does not serve - sigmoid or softmax
// scores, a per-expert bias that balances the choice but not the weights, and a choice limited to the
// best of several groups of experts. Per row, with l the row's logits:
//
//   score   s[e] = 1 / (1 + exp(-l[e])), or exp(l[e] - max l) / sum exp(l - max l)
//   choice  c[e] = s[e] + bias[e]
//   group   g of G holds the experts g E / G .. (g + 1) E / G - 1 and ranks by the sum of its best
//           `group_top` choices; the `top_groups` best groups stay, the others' experts are out
//   ids     the `top` largest choices left, in descending order
//   weight  s[id], divided by the picked scores' sum (`renormalize`; 0 where that sum is 0), times
//           `factor`, in FP32
//
// Scores, choices and group ranks are held in 64 bits, so that rounding neither makes nor breaks a
// tie; equal choices go to the lower expert id and equal groups to the lower group.
//
// An expert is no candidate in a row where its logit is NaN or -inf, and in every row where its bias
// is: it adds nothing to a softmax's sum or to its group's rank and is never picked. Logits above the
// largest finite float count as that float. Where fewer than `top` candidates are left (a row of -inf,
// padding), the remaining ids are -1 with weight 0; moe_sort skips such routes.
//
// `map` (the slot of each expert), `live` and `load` (the 64-bit count of live rows' picks by expert,
// added to what is there) are topk_softmax's; an id of -1 is neither mapped nor counted.

#pragma once

#include "uniserve_abi.h"

#define UNISERVE_EXPERT_TOPK_MAX_EXPERTS 1024
#define UNISERVE_EXPERT_TOPK_MAX_TOP 32
#define UNISERVE_EXPERT_TOPK_MAX_GROUPS 64

enum uniserve_scoring
#ifdef __cplusplus
    : int32_t
#endif
{
  UNISERVE_SCORING_SOFTMAX = 0,
  UNISERVE_SCORING_SIGMOID = 1,
};

struct uniserve_expert_topk_call {
  const void *scores;    ///< [rows, experts] logits of score_dtype, rows row_stride elements apart
  const float *bias;     ///< [experts], or null
  const int32_t *map;    ///< [experts], or null
  const int32_t *live;   ///< [1] rows that count into load, or null: all
  int64_t *load;         ///< [experts], or null
  int32_t *ids;          ///< [rows, top]
  float *weights;        ///< [rows, top]
  int64_t row_stride;
  int64_t rows;          ///< at most 2^26 - 4, rows * top below 2^31
  int64_t experts;
  int64_t top;
  int64_t groups;        ///< 1: no groups
  int64_t top_groups;    ///< 1 .. groups
  int64_t group_top;     ///< 1 or 2
  int64_t score_dtype;   ///< f32, bf16 or f16
  int64_t scoring;       ///< enum uniserve_scoring
  int64_t renormalize;
  float factor;
  char error[512];
};

/// Launches the choice on `stream`. No output shares memory with an input or another output. Nothing is allocated, no workspace is used and the call may be
/// captured. Returns 0, or nonzero with a message in `error`.
UNISERVE_EXTERN_C int32_t uniserve_expert_topk(const struct uniserve_expert_topk_call *call, void *stream);
