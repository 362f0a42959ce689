// SPDX-License-Identifier: Apache-2.0
//
// expert_topk on gfx950: softmax or sigmoid scores, a balance bias, groups, top-k and weights
// (include/uniserve_expert_topk.h states the operator).
//
// One wavefront per row. With G groups of S experts the 64 lanes are dealt to the groups, P = 64 over G
// rounded up to a power of two each: lane g P + q holds the group's experts q, q + P, q + 2 P, .. (one group:
// lane l holds l, l + 64, ..), so a group's rank meets in P neighbouring lanes and no choice passes LDS.
//
// The choice is defined in 64 bits: two choices a few 1e-9 apart are common among hundreds of experts over
// thousands of rows, and an FP32 sigmoid plus bias orders such a pair by its rounding. Doubles everywhere
// cost 22.9 us at 8192 x 256 (8 groups, top 8), most of it in their lane exchanges. So a row is first chosen
// from in FP32, whose error is bounded, until the next pick is further below pick `top` than twice that error:
// no expert after it can be among the top. The scores of these candidates (mostly `top`) are evaluated in 64
// bits, which the weights want anyway, and where two neighbours are closer than that the candidates are put in
// order by them. The whole choice is made again from doubles only where FP32 cannot tell the groups at the
// edge of the kept ones apart, or more than 64 candidates lie together.
//
// Bound by vector instructions, some 570 a row at 256 experts in 8 groups (180 in the picks' rounds, 150 in the
// doubles); the reads would take 2 us at 8192 rows. 8192 x 256, 8 groups, top 8: f32 logits and a bias 10.4 us,
// bf16 without one (ties in every other row) 14.4; 64 rows 4.7 and 7.0. With the whole choice from doubles in
// every row with a close pair: 13.1, 24.2, 4.8 and 10.9 us. Two rows a wavefront, 32 lanes each: 14.6 us at 8192
// rows (half the wavefronts to hide the rounds' latency), 45 against 56 at 65536.
#include "common.hpp"
#include "uniserve_expert_topk.h"

#include <cfloat>
#include <climits>
#include <cmath>
#include <type_traits>

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
  int size;       ///< experts of a group
  int lane_bits;  ///< a group has 2^lane_bits lanes
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

/// The maximum over the wavefront, as a scalar: DPP shifts carry it to lane 15 of each 16-lane row, broadcasts
/// from row to row to lane 63. (In place and in one piece: written with the DPP builtin, every step costs a copy
/// too. A DPP read of a register comes two wait states after its write.)
__device__ __forceinline__ int wave_max(int x) {
  asm("s_nop 1\n\t"
      "v_max_i32_dpp %0, %0, %0 row_shr:1 row_mask:0xf bank_mask:0xf\n\ts_nop 1\n\t"
      "v_max_i32_dpp %0, %0, %0 row_shr:2 row_mask:0xf bank_mask:0xf\n\ts_nop 1\n\t"
      "v_max_i32_dpp %0, %0, %0 row_shr:4 row_mask:0xf bank_mask:0xf\n\ts_nop 1\n\t"
      "v_max_i32_dpp %0, %0, %0 row_shr:8 row_mask:0xf bank_mask:0xf\n\ts_nop 1\n\t"
      "v_max_i32_dpp %0, %0, %0 row_bcast:15 row_mask:0xf bank_mask:0xf\n\ts_nop 1\n\t"
      "v_max_i32_dpp %0, %0, %0 row_bcast:31 row_mask:0xf bank_mask:0xf"
      : "+v"(x));
  return __builtin_amdgcn_readlane(x, 63);
}

/// Integers that order as the floats do (and -0 below 0).
__device__ __forceinline__ int ordered(float x) {
  const int bits = __float_as_int(x);
  return bits ^ ((bits >> 31) & INT_MAX);
}
__device__ __forceinline__ float unordered(int key) { return __int_as_float(key ^ ((key >> 31) & INT_MAX)); }
__device__ __forceinline__ float wave_max(float x) { return unordered(wave_max(ordered(x))); }

template <class F>
__device__ __forceinline__ F wave_sum(F x) {
#pragma unroll
  for (int offset = 32; offset > 0; offset /= 2) x += __shfl_xor(x, offset);
  return x;
}

/// The lane's logits first, first + lanes, .. of a row (expert 0's in the place of those from `past` on): all
/// loads in flight together.
template <int kIter>
__device__ __forceinline__ void load_row(const ChoiceParams &p, int64_t row, int first, int lanes, int past, float (&logit)[kIter]) {
  int at[kIter];
#pragma unroll
  for (int i = 0; i < kIter; ++i) at[i] = first + i * lanes < past ? first + i * lanes : 0;
  if (p.kind == UNISERVE_DTYPE_F32) {
    const float *scores = static_cast<const float *>(p.scores) + row * p.row_stride;
#pragma unroll
    for (int i = 0; i < kIter; ++i) logit[i] = scores[at[i]];
    return;
  }
  const uint16_t *scores = static_cast<const uint16_t *>(p.scores) + row * p.row_stride;
  uint16_t bits[kIter];
#pragma unroll
  for (int i = 0; i < kIter; ++i) bits[i] = scores[at[i]];
#pragma unroll
  for (int i = 0; i < kIter; ++i)
    logit[i] = p.kind == UNISERVE_DTYPE_F16 ? static_cast<float>(__builtin_bit_cast(_Float16, bits[i])) : bf16_to_f32(bits[i]);
}

/// The best two of two pairs (the larger first).
template <class F>
__device__ __forceinline__ void merge_best(F &best, F &second, F other, F other_second) {
  const F low = best < other ? best : other;
  best = best < other ? other : best;
  second = second < other_second ? other_second : second;
  second = second < low ? low : second;
}

/// Each lane's group's two best choices, from the lanes' own best two. `lanes`: P.
__device__ __forceinline__ void group_best(int &best, int &second, int lanes) {
  // Quads, then the other quad of eight and the other eight of sixteen (all of a half hold the same by then).
  auto step = [&](auto control) {
    constexpr int kControl = decltype(control)::value;
    merge_best(best, second, __builtin_amdgcn_mov_dpp(best, kControl, 0xf, 0xf, false),
               __builtin_amdgcn_mov_dpp(second, kControl, 0xf, 0xf, false));
  };
  if (lanes > 1) step(std::integral_constant<int, 0xb1>{});   // quad_perm [1, 0, 3, 2]
  if (lanes > 2) step(std::integral_constant<int, 0x4e>{});   // quad_perm [2, 3, 0, 1]
  if (lanes > 4) step(std::integral_constant<int, 0x141>{});  // row_half_mirror
  if (lanes > 8) step(std::integral_constant<int, 0x140>{});  // row_mirror
  for (int offset = 16; offset < lanes; offset *= 2) {
    const int other = __shfl_xor(best, offset), other_second = __shfl_xor(second, offset);
    merge_best(best, second, other, other_second);
  }
}
__device__ __forceinline__ void group_best(double &best, double &second, int lanes) {
  for (int offset = 1; offset < lanes; offset *= 2) {
    const double other = __shfl_xor(best, offset), other_second = __shfl_xor(second, offset);
    merge_best(best, second, other, other_second);
  }
}

/// The lane's keys in descending order (Batcher's odd-even merge sort, kIter a power of two).
template <int kIter>
__device__ __forceinline__ void sort_descending(int (&key)[kIter]) {
#pragma unroll
  for (int run = 1; run < kIter; run *= 2)
#pragma unroll
    for (int step = run; step >= 1; step /= 2)
#pragma unroll
      for (int i = step % run; i + step < kIter; ++i) {
        if ((i - step % run) / step % 2 != 0 || i / (2 * run) != (i + step) / (2 * run)) continue;
        const int high = key[i] < key[i + step] ? key[i + step] : key[i];
        key[i + step] = key[i] < key[i + step] ? key[i] : key[i + step];
        key[i] = high;
      }
}

/// The whole choice in 64 bits: lane j < top answers pick j's expert, or -1. A round takes the largest choice
/// rounded to FP32 (which keeps the order or makes a tie) and, where several candidates share it, the largest
/// double and the lowest expert among them.
template <int kIter, class Score>
__device__ __forceinline__ int choose_exactly(const ChoiceParams &p, int lane, int group, int first, int lanes,
                                                        const float (&logit)[kIter], const float (&bias)[kIter],
                                                        const Score &exact_score, double sum) {
  const double out = -__builtin_inf();
  double choice[kIter];
#pragma unroll
  for (int i = 0; i < kIter; ++i)
    choice[i] = logit[i] > -__builtin_inff() ? (p.sigmoid ? exact_score(logit[i]) : exact_score(logit[i]) / sum) + static_cast<double>(bias[i]) : out;
  if (p.groups > 1) {
    double rank = out, second = out;
#pragma unroll
    for (int i = 0; i < kIter; ++i) merge_best(rank, second, choice[i], out);
    group_best(rank, second, lanes);
    if (p.group_top == 2 && second > out) rank += second;
    int ahead = 0;
    for (int g = 0; g < p.groups; ++g) {
      const double other = __shfl(rank, g << p.lane_bits);
      ahead += other > rank || (other == rank && g < group);
    }
    if (ahead >= p.top_groups) {
#pragma unroll
      for (int i = 0; i < kIter; ++i) choice[i] = out;
    }
  }
  int id = -1;
  for (int j = 0; j < p.top; ++j) {
    float own = -__builtin_inff();
#pragma unroll
    for (int i = 0; i < kIter; ++i) own = own < static_cast<float>(choice[i]) ? static_cast<float>(choice[i]) : own;
    const float best = wave_max(own);
    if (!(best > -__builtin_inff())) break;
    // The lane's best candidate among those that round to `best`: the first of equal ones has the lower id.
    double mine = out;
    int expert = INT_MAX;
#pragma unroll
    for (int i = 0; i < kIter; ++i)
      if (static_cast<float>(choice[i]) == best && choice[i] > mine) {
        mine = choice[i];
        expert = first + i * lanes;
      }
    const uint64_t holders = ballot(expert != INT_MAX);
    if (__popcll(holders) > 1) {
#pragma unroll
      for (int offset = 32; offset > 0; offset /= 2) {
        const double other = __shfl_xor(mine, offset);
        const int other_expert = __shfl_xor(expert, offset);
        if (other > mine || (other == mine && other_expert < expert)) {
          mine = other;
          expert = other_expert;
        }
      }
    } else {
      expert = __builtin_amdgcn_readlane(expert, __builtin_ctzll(holders));
    }
    if (lane == j) id = expert;
#pragma unroll
    for (int i = 0; i < kIter; ++i)
      if (first + i * lanes == expert) choice[i] = out;
  }
  return id;
}

/// kIter: experts per lane.
template <int kIter>
__global__ void __launch_bounds__(kChoiceWaves *kWave) expert_topk_kernel(ChoiceParams p) {
  const int wave = static_cast<int>(threadIdx.x) / kWave;
  const int lane = lane_id();
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kChoiceWaves + wave;
  if (row >= p.rows) return;
  constexpr float kOut = -__builtin_inff();
  const int lanes = 1 << p.lane_bits;
  const int group = lane >> p.lane_bits;
  const int first = group * p.size + (lane & (lanes - 1));  // the lane's expert i is first + i lanes
  const int past = group < p.groups ? (group + 1) * p.size : 0;

  // Logits and biases; no candidate (comparisons with NaN are false) has a logit of -inf.
  float logit[kIter], bias[kIter];
  load_row<kIter>(p, row, first, lanes, past, logit);
#pragma unroll
  for (int i = 0; i < kIter; ++i) bias[i] = 0.0f;
  if (p.bias != nullptr) {
#pragma unroll
    for (int i = 0; i < kIter; ++i) bias[i] = p.bias[first + i * lanes < past ? first + i * lanes : 0];
  }
  float maximum = kOut;
#pragma unroll
  for (int i = 0; i < kIter; ++i) {
    const bool candidate = (first + i * lanes < past) & (logit[i] > kOut) & (bias[i] > kOut);
    logit[i] = candidate ? (logit[i] < FLT_MAX ? logit[i] : FLT_MAX) : kOut;
    maximum = maximum < logit[i] ? logit[i] : maximum;
  }

  // ---- the choice in FP32 ----
  // A sigmoid here is off by less than 2^-22: in steps of 2^-24 the exponent's rounding gives 1.5 |l| s (1 - s)
  // < 0.34, the exponential 0.5, 1 + e and the reciprocal 3. Two of them move against each other by twice that.
  // Two softmax probabilities of a row move against each other by less than 2 (kIter + 12) steps of the row's
  // largest. Each by its own errors: x below the maximum the exponent's rounding gives 2.5 x e^-x < 0.92, the
  // exponential 2, the product 1. And all by one factor, which changes a difference once, not twice: the sum's
  // kIter + 5 additions and the quotient's 1, the exponentials' 2, and 2.5 times the mean of x under the softmax,
  // which is largest where all but the maximum lie equally deep: W((N - 1) / e) for N experts (Lambert's W), 2.3 for
  // 64 and 4.5 for 1024. Together 23 steps of the 26 at kIter = 1, 59 of the 88 at 32. The bias's addition rounds by
  // half a step of the choice, and the slot in a key's low bits moves it by 2 kSlots. Two choices further apart than
  // all this are ordered as in 64 bits.
  constexpr int kSlotBits = kIter <= 1 ? 0 : kIter <= 2 ? 1 : kIter <= 4 ? 2 : kIter <= 8 ? 3 : kIter <= 16 ? 4 : 5;
  constexpr int kSlots = (1 << kSlotBits) - 1;
  constexpr float kUnsureOf = (8.0f + 8.0f * kSlots) * 0x1p-24f;  // of a choice's own size
  float score[kIter];
  float unsure;  // how far apart two scores have to be
  if (p.sigmoid) {
#pragma unroll
    for (int i = 0; i < kIter; ++i) score[i] = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.4426950408889634f * logit[i]));
    unsure = 0x1p-20f;
  } else {
    maximum = wave_max(maximum);
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < kIter; ++i) {
      score[i] = logit[i] > kOut ? __builtin_amdgcn_exp2f(1.4426950408889634f * (logit[i] - maximum)) : 0.0f;
      sum += score[i];
    }
    const float scale = 1.0f / wave_sum(sum);
#pragma unroll
    for (int i = 0; i < kIter; ++i) score[i] *= scale;
    unsure = 2.0f * (kIter + 12) * 0x1p-24f * __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(scale)));
  }
  // The lane's choices as ordered integers; no candidate: below kLowest, the lowest finite float, also with a
  // slot in the low bits.
  constexpr int kLowest = INT_MIN + 0x800000;
  int order[kIter];
#pragma unroll
  for (int i = 0; i < kIter; ++i) {
    const float choice = score[i] + bias[i];
    order[i] = ordered(logit[i] > kOut ? choice : kOut);
  }

  bool sure = true;
  if (p.groups > 1) {
    int best = INT_MIN, second = INT_MIN;
#pragma unroll
    for (int i = 0; i < kIter; ++i) merge_best(best, second, order[i], INT_MIN);
    group_best(best, second, lanes);
    // A rank's error goes by its two choices, which may cancel; a sum past the lowest finite float stays above the
    // rank of a group without candidates, and near every other such sum.
    const float first_of = best < kLowest ? kOut : unordered(best);
    const float second_of = p.group_top < 2 || second < kLowest ? 0.0f : unordered(second);
    float rank = first_of + second_of;
    rank = best < kLowest || rank >= -FLT_MAX ? rank : -FLT_MAX;
    const float size = __builtin_fmaxf(__builtin_fabsf(first_of), __builtin_fabsf(second_of));
    const float margin = 2.0f * unsure + 0x1p-20f * wave_max(size < __builtin_inff() ? size : 0.0f);
    // Lane (g, q) compares group g with the groups q, q + P, ..; the ballots hold the P lanes' answers of a group
    // side by side. `near` counts the groups that may lie ahead, its own among them.
    const float above = rank + margin, below = rank - margin;
    const uint64_t mine = (lanes < kWave ? (1ull << lanes) - 1ull : ~0ull) << (group << p.lane_bits);
    int ahead = 0, near = -1;
    for (int g = 0; g < p.groups; g += lanes) {
      const int with = g + (lane & (lanes - 1));
      const float other = __shfl(rank, (with << p.lane_bits) & (kWave - 1));
      ahead += __popcll(ballot((with < p.groups) & (other > above)) & mine);
      near += __popcll(ballot((with < p.groups) & (other >= below)) & mine);
    }
    const bool out = ahead >= p.top_groups;
    sure = ballot((rank > kOut) & !out & (near >= p.top_groups)) == 0;
#pragma unroll
    for (int i = 0; i < kIter; ++i) order[i] = out ? INT_MIN : order[i];
  }

  // Whether two choices of these sizes are ordered in 64 bits as here (an infinite one and its neighbours: no).
  const auto apart = [&](float here, float there) {
    return here - there > unsure + kUnsureOf * __builtin_fmaxf(__builtin_fabsf(here), __builtin_fabsf(there));
  };
  int id = -1;
  int count = p.top;  // candidates, lane by lane
  bool ordered_here = false;
  if (sure) {
    // The slot in the low bits, the lane's in descending order; a round's offer is the lane's first, and only the
    // lane whose offer won moves on. Lane j keeps pick j and its lane. The first pick clearly below pick top - 1
    // ends the rounds: no other can be among the top.
#pragma unroll
    for (int i = 0; i < kIter; ++i) order[i] = (order[i] & ~kSlots) | i;
    sort_descending(order);
    int pick = INT_MIN, holder_of = 0;
    const auto take = [&](int best) {
      const int holder = __builtin_ctzll(ballot(order[0] == best));
      pick = lane == count ? best : pick;
      holder_of = lane == count ? holder : holder_of;
      if (lane == holder) {
#pragma unroll
        for (int i = 0; i + 1 < kIter; ++i) order[i] = order[i + 1];
        order[kIter - 1] = INT_MIN;
      }
    };
    int best = wave_max(order[0]), last = best;
    for (count = 0; count < p.top && best >= kLowest; ++count) {
      take(best);
      last = best;
      best = wave_max(order[0]);
    }
    while (!(sure = best < kLowest || apart(unordered(last), unordered(best))) && count < kWave) {
      take(best);
      ++count;
      best = wave_max(order[0]);
    }
    if (pick >= kLowest) id = (holder_of >> p.lane_bits) * p.size + (holder_of & (lanes - 1)) + (pick & kSlots) * lanes;
    const int next = __shfl_down(pick, 1);
    ordered_here = ballot((lane + 1 < count) & !apart(unordered(pick), unordered(next))) == 0;
  }

  // ---- 64 bits: the candidates' scores and, where FP32 does not tell, their order, or the whole choice ----
  const auto exact_score = [&](float l) {  // (softmax: times the sum)
    return p.sigmoid ? 1.0 / (1.0 + exp(-static_cast<double>(l))) : exp(static_cast<double>(l) - static_cast<double>(maximum));
  };
  double sum = 1.0;  // of the softmax, where it is wanted
  if (!p.sigmoid && (!sure || !ordered_here || !p.renormalize)) {
    sum = 0.0;
#pragma unroll
    for (int i = 0; i < kIter; ++i)
      if (logit[i] > kOut) sum += exact_score(logit[i]);
    sum = wave_sum(sum);
  }
  if (!sure) {
    id = choose_exactly<kIter>(p, lane, group, first, lanes, logit, bias, exact_score, sum);
    count = p.top;
  }
  double picked = 0.0;
  if (lane < count && id >= 0) {
    const float l = load_logit(p.scores, p.kind, row * p.row_stride + id);
    picked = exact_score(l < FLT_MAX ? l : FLT_MAX);
    if (!p.sigmoid) picked /= sum;
  }
  if (sure && !ordered_here) {
    // Lane j's place among the candidates (lanes past them keep theirs), where it sends what it holds.
    const double choice = picked + (p.bias != nullptr && id >= 0 ? static_cast<double>(p.bias[id]) : 0.0);
    const uint64_t bits = __builtin_bit_cast(uint64_t, choice);
    int place = lane < count ? 0 : lane;
    for (int j = 0; j < count; ++j) {
      const uint32_t low = __builtin_amdgcn_readlane(static_cast<int>(bits), j);
      const uint32_t high = __builtin_amdgcn_readlane(static_cast<int>(bits >> 32), j);
      const double other = __builtin_bit_cast(double, static_cast<uint64_t>(high) << 32 | low);
      const int other_id = __builtin_amdgcn_readlane(id, j);
      place += lane < count && (other > choice || (other == choice && other_id < id));
    }
    const uint64_t held = __builtin_bit_cast(uint64_t, picked);
    id = __builtin_amdgcn_ds_permute(place * 4, id);
    const uint32_t low = __builtin_amdgcn_ds_permute(place * 4, static_cast<int>(held));
    const uint32_t high = __builtin_amdgcn_ds_permute(place * 4, static_cast<int>(held >> 32));
    picked = __builtin_bit_cast(double, static_cast<uint64_t>(high) << 32 | low);
  }
  if (lane >= p.top) picked = 0.0;
  if (p.renormalize) {
    double total = picked;
    for (int offset = 1; offset < p.top; offset *= 2) total += __shfl_xor(total, offset);
    picked = total > 0.0 ? picked / total : 0.0;
  }
  if (lane >= p.top) return;
  p.ids[row * p.top + lane] = id >= 0 && p.map != nullptr ? p.map[id] : id;
  p.weights[row * p.top + lane] = static_cast<float>(picked * static_cast<double>(p.factor));
  if (p.load != nullptr && id >= 0 && (p.live == nullptr || row < p.live[0])) atomicAdd(p.load + id, 1ull);
}

template <int kIter>
void launch_choice(const ChoiceParams &p, hipStream_t stream) {
  const dim3 grid(static_cast<uint32_t>(ceil_div<int64_t>(p.rows, kChoiceWaves)));
  hipLaunchKernelGGL(expert_topk_kernel<kIter>, grid, dim3(kChoiceWaves * kWave), 0, stream, p);
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
    constexpr int64_t kMostRows = ((int64_t{1} << 32) / (kChoiceWaves * kWave) - 1) * kChoiceWaves;  // a launch's axis holds
    if (call->rows > kMostRows) return UNISERVE_REFUSE(call, "expert_topk serves %lld rows in a call", static_cast<long long>(kMostRows));
    if (call->rows > 1 && call->row_stride < call->experts)
      return UNISERVE_REFUSE(call, "expert_topk's row stride is shorter than its rows");
    if (call->rows > 1 && call->row_stride > (int64_t{1} << 40) / call->rows)
      return UNISERVE_REFUSE(call, "expert_topk's scores are too large");
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
    // Groups that all stay limit nothing.
    if (p.top_groups == p.groups) p.groups = p.top_groups = 1;
    p.size = p.experts / p.groups;
    p.lane_bits = 6;
    while ((kWave >> p.lane_bits) < p.groups) --p.lane_bits;
    const int needed = ceil_div(p.size, 1 << p.lane_bits);
    if (needed <= 1) launch_choice<1>(p, s);
    else if (needed <= 2) launch_choice<2>(p, s);
    else if (needed <= 4) launch_choice<4>(p, s);
    else if (needed <= 8) launch_choice<8>(p, s);
    else if (needed <= 16) launch_choice<16>(p, s);
    else launch_choice<32>(p, s);
    return launched(call, "expert_topk");
  });
}
