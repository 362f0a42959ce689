// SPDX-License-Identifier: Apache-2.0
//
// expert_topk on gfx950: softmax or sigmoid scores, a balance bias, groups, top-k and weights
// (include/uniserve_expert_topk.h states the operator).
//
// One wavefront per row; lane l holds experts l + 64 i. Scores and choices are doubles: two choices
// a few 1e-9 apart are common among 128 to 512 experts over thousands of rows, and an FP32 sigmoid
// plus bias orders such a pair by its rounding.
#include "common.hpp"
#include "uniserve_expert_topk.h"

#include <cfloat>
#include <cmath>

namespace uniserve {
namespace {

constexpr int kChoiceWaves = 4;

struct ChoiceParams {
  const void *scores;
  const float *bias;
  const int32_t *map;
  const int32_t *live;
  unsigned long long *load;
  int32_t *ids;
  float *weights;
  int64_t row_stride;
  int rows;
  int experts;
  int top;
  int groups;
  int top_groups;
  int group_top;
  int kind;  ///< UNISERVE_DTYPE_F32, _BF16 or _F16
  int sigmoid;
  int renormalize;
  float factor;
};

__device__ __forceinline__ float load_logit(const void *data, int kind, int64_t index) {
  if (kind == UNISERVE_DTYPE_F32) return static_cast<const float *>(data)[index];
  if (kind == UNISERVE_DTYPE_F16) return static_cast<float>(static_cast<const _Float16 *>(data)[index]);
  return bf16_to_f32(static_cast<const uint16_t *>(data)[index]);
}

__device__ __forceinline__ double wave_max(double x) {
#pragma unroll
  for (int offset = 32; offset > 0; offset /= 2) {
    const double other = __shfl_xor(x, offset);
    x = x < other ? other : x;
  }
  return x;
}

__device__ __forceinline__ double wave_sum(double x) {
#pragma unroll
  for (int offset = 32; offset > 0; offset /= 2) x += __shfl_xor(x, offset);
  return x;
}

/// kIter: experts per lane.
template <int kIter>
__global__ void __launch_bounds__(kChoiceWaves *kWave) expert_topk_kernel(ChoiceParams p) {
  extern __shared__ double choices[];  // [waves][experts], where the experts are in groups
  const int wave = static_cast<int>(threadIdx.x) / kWave;
  const int lane = lane_id();
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kChoiceWaves + wave;
  if (row >= p.rows) return;
  const double out = -__builtin_inf();

  double score[kIter], choice[kIter];
  double maximum = out;
#pragma unroll
  for (int i = 0; i < kIter; ++i) {
    const int e = lane + kWave * i;
    float logit = -__builtin_inff(), bias = 0.0f;
    if (e < p.experts) {
      logit = load_logit(p.scores, p.kind, row * p.row_stride + e);
      if (p.bias != nullptr) bias = p.bias[e];
    }
    // Comparisons with NaN are false: a NaN logit or bias is no candidate either.
    const bool candidate = logit > -__builtin_inff() && bias > -__builtin_inff();
    logit = logit > FLT_MAX ? FLT_MAX : logit;
    score[i] = candidate ? static_cast<double>(logit) : out;
    choice[i] = candidate ? static_cast<double>(bias) : out;
    maximum = maximum < score[i] ? score[i] : maximum;
  }
  if (p.sigmoid) {
#pragma unroll
    for (int i = 0; i < kIter; ++i) score[i] = 1.0 / (1.0 + exp(-score[i]));
  } else {
    maximum = wave_max(maximum);
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < kIter; ++i) {
      score[i] = score[i] > out ? exp(score[i] - maximum) : 0.0;
      sum += score[i];
    }
    sum = wave_sum(sum);
#pragma unroll
    for (int i = 0; i < kIter; ++i) score[i] = score[i] / sum;
  }
#pragma unroll
  for (int i = 0; i < kIter; ++i) choice[i] = choice[i] > out ? score[i] + choice[i] : out;

  if (p.groups > 1) {
    // Lane g ranks group g; a group's rank is the number of groups before it.
    double *own = choices + wave * p.experts;
#pragma unroll
    for (int i = 0; i < kIter; ++i) {
      const int e = lane + kWave * i;
      if (e < p.experts) own[e] = choice[i];
    }
    __builtin_amdgcn_wave_barrier();
    const int size = p.experts / p.groups;
    double best = out, second = out;
    if (lane < p.groups) {
      for (int e = lane * size; e < (lane + 1) * size; ++e) {
        const double c = own[e];
        second = c > best ? best : (c > second ? c : second);
        best = c > best ? c : best;
      }
    }
    const double rank = p.group_top == 2 && second > out ? best + second : best;
    int ahead = 0;
    for (int g = 0; g < p.groups; ++g) {
      const double other = __shfl(rank, g);
      ahead += other > rank || (other == rank && g < lane);
    }
    const uint64_t kept = ballot(lane < p.groups && ahead < p.top_groups);
#pragma unroll
    for (int i = 0; i < kIter; ++i) {
      const int e = lane + kWave * i;
      if (e < p.experts && !((kept >> (e / size)) & 1u)) choice[i] = out;
    }
  }

  // `top` rounds: the largest choice left, the lowest expert holding it; lane j keeps round j's.
  double picked = 0.0;
  int id = -1;
  for (int j = 0; j < p.top; ++j) {
    double best = choice[0];
#pragma unroll
    for (int i = 1; i < kIter; ++i) best = best < choice[i] ? choice[i] : best;
    best = wave_max(best);
    if (!(best > out)) break;
    bool found = false;
#pragma unroll
    for (int i = 0; i < kIter; ++i) {
      const uint64_t holders = ballot(choice[i] == best);
      if (found || holders == 0) continue;
      found = true;
      const int holder = __builtin_ctzll(holders);
      const double s = __shfl(score[i], holder);
      if (lane == j) {
        picked = s;
        id = holder + kWave * i;
      }
      if (lane == holder) choice[i] = out;
    }
  }
  if (p.renormalize) {
    const double sum = wave_sum(picked);
    picked = sum > 0.0 ? picked / sum : 0.0;
  }
  if (lane >= p.top) return;
  p.ids[row * p.top + lane] = id >= 0 && p.map != nullptr ? p.map[id] : id;
  p.weights[row * p.top + lane] = static_cast<float>(picked * static_cast<double>(p.factor));
  if (p.load != nullptr && id >= 0 && (p.live == nullptr || row < p.live[0])) atomicAdd(p.load + id, 1ull);
}

template <int kIter>
void launch_choice(const ChoiceParams &p, hipStream_t stream) {
  const size_t lds = p.groups > 1 ? sizeof(double) * kChoiceWaves * p.experts : 0;
  const dim3 grid(static_cast<uint32_t>(ceil_div<int64_t>(p.rows, kChoiceWaves)));
  hipLaunchKernelGGL(expert_topk_kernel<kIter>, grid, dim3(kChoiceWaves * kWave), lds, stream, p);
}

}  // namespace
}  // namespace uniserve

extern "C" int32_t uniserve_expert_topk(const uniserve_expert_topk_call *call, void *stream) {
  using namespace uniserve;
  return guarded(call, [&]() -> int32_t {
    if (call->experts < 1 || call->experts > UNISERVE_EXPERT_TOPK_MAX_EXPERTS)
      return UNISERVE_REFUSE(call, "expert_topk serves 1 to %d experts", UNISERVE_EXPERT_TOPK_MAX_EXPERTS);
    if (call->groups < 1 || call->groups > UNISERVE_EXPERT_TOPK_MAX_GROUPS || call->experts % call->groups != 0)
      return UNISERVE_REFUSE(call, "expert_topk needs 1 to %d groups of equal size", UNISERVE_EXPERT_TOPK_MAX_GROUPS);
    if (call->top_groups < 1 || call->top_groups > call->groups)
      return UNISERVE_REFUSE(call, "expert_topk keeps between one and all of its groups");
    if (call->group_top < 1 || call->group_top > 2)
      return UNISERVE_REFUSE(call, "expert_topk ranks a group by its best expert or its best two");
    if (call->top < 1 || call->top > UNISERVE_EXPERT_TOPK_MAX_TOP ||
        call->top > call->top_groups * (call->experts / call->groups))
      return UNISERVE_REFUSE(call, "expert_topk picks between one and %d experts, no more than the kept groups hold",
                             UNISERVE_EXPERT_TOPK_MAX_TOP);
    if (call->score_dtype != UNISERVE_DTYPE_F32 && call->score_dtype != UNISERVE_DTYPE_BF16 &&
        call->score_dtype != UNISERVE_DTYPE_F16)
      return UNISERVE_REFUSE(call, "expert_topk serves f32, bf16 or f16 scores");
    if (call->scoring != UNISERVE_SCORING_SOFTMAX && call->scoring != UNISERVE_SCORING_SIGMOID)
      return UNISERVE_REFUSE(call, "expert_topk scores by softmax or sigmoid");
    if (!std::isfinite(call->factor)) return UNISERVE_REFUSE(call, "expert_topk needs a finite factor");
    if (call->rows < 0 || call->rows > 0x7fffffffLL / call->top)
      return UNISERVE_REFUSE(call, "expert_topk's routes do not fit int32 indexes");
    if (call->rows > 1 && call->row_stride < call->experts)
      return UNISERVE_REFUSE(call, "expert_topk's row stride is shorter than its rows");
    if (call->rows == 0) return 0;
    if (call->scores == nullptr || call->ids == nullptr || call->weights == nullptr)
      return UNISERVE_REFUSE(call, "expert_topk needs scores, ids and weights");
    ChoiceParams p{};
    p.scores = call->scores;
    p.bias = call->bias;
    p.map = call->map;
    p.live = call->live;
    p.load = reinterpret_cast<unsigned long long *>(call->load);
    p.ids = call->ids;
    p.weights = call->weights;
    p.row_stride = call->row_stride;
    p.rows = static_cast<int>(call->rows);
    p.experts = static_cast<int>(call->experts);
    p.top = static_cast<int>(call->top);
    p.groups = static_cast<int>(call->groups);
    p.top_groups = static_cast<int>(call->top_groups);
    p.group_top = static_cast<int>(call->group_top);
    p.kind = static_cast<int>(call->score_dtype);
    p.sigmoid = call->scoring == UNISERVE_SCORING_SIGMOID;
    p.renormalize = call->renormalize != 0;
    p.factor = call->factor;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    const int needed = ceil_div(p.experts, kWave);
    if (needed <= 1) launch_choice<1>(p, s);
    else if (needed <= 2) launch_choice<2>(p, s);
    else if (needed <= 4) launch_choice<4>(p, s);
    else if (needed <= 8) launch_choice<8>(p, s);
    else launch_choice<16>(p, s);
    return launched(call, "expert_topk");
  });
}
