// SPDX-License-Identifier: Apache-2.0
//
// token_experts on gfx950 (include/uniserve_token_experts.h states the operator). Two kernels stream the named experts'
// weights, each line once, whole lines of 128 bytes (eight lanes a row) that a wavefront regroups into
// the matrix instruction's operand through LDS of its own; weight rows are operand A, up to 16 tokens operand B.
//
// A job is an expert with up to 16 of its tokens. The first kernel's workgroups find their job from the ids (a mask of
// tokens for each expert, and its scan), multiply its up and gate rows and leave the gated values; the first workgroup
// also leaves the list of jobs. The second kernel's workgroups own output columns and walk all jobs, adding
// each one's products, times the routes' weights, to their rows' sums, experts in ascending order: no join across
// workgroups, no atomics on sums.
#include "extents.hpp"
#include "linear.hpp"
#include "uniserve_token_experts.h"

namespace uniserve {
namespace token_experts {
namespace {

using linear::Bf16;
using linear::F16;
using linear::load8;

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;
constexpr int kMostTokens = UNISERVE_TOKEN_EXPERTS_MAX_TOKENS;
constexpr int kMostExperts = UNISERVE_TOKEN_EXPERTS_MAX_EXPERTS;
constexpr int kJobTokens = 16;
constexpr int kLine = 64;  // elements

struct Job {
  int32_t expert, first, count, unused;  ///< entries first .. first + count - 1
};
/// A token of a job: its first route to the expert, and the weights of all of them.
struct Entry {
  int32_t route;
  float weight;
};

struct Params {
  const uint16_t *x, *up_gate, *down, *residual;
  const int32_t *ids;
  const float *weights;
  uint16_t *out;
  int32_t *job_count;
  Job *jobs;
  Entry *entries;
  uint16_t *gated;  ///< [routes, 2, padded]: values, then errors
  int64_t x_stride, residual_stride, out_stride;
  int32_t tokens, top, routes, hidden, width, padded, experts, first_expert, activation;
};

/// Values of f16 pairs are held at this part of themselves.
template <class T>
constexpr float kHeld = std::is_same<T, F16>::value ? 0.015625f : 1.0f;

template <bool kWhole>
__device__ __forceinline__ u32x4 piece_of(const uint16_t *row, int64_t at, int64_t width) {
  if constexpr (kWhole) return at < width ? *reinterpret_cast<const u32x4 *>(row + at) : u32x4{0, 0, 0, 0};
  else return load8(row, at, width);
}

/// An id's expert in the stacks, or -1.
__device__ __forceinline__ int expert_of(const Params &p, int id) {
  const int e = id >= p.first_expert ? id - p.first_expert : -1;  // (the first is not negative)
  return e < p.experts ? e : -1;
}

/// Where the routes lead: the tokens that name each expert, and how many tokens and jobs come before it.
struct Routing {
  uint64_t tokens[kMostExperts];
  uint16_t entries_before[kMostExperts], jobs_before[kMostExperts];
  int32_t wave_entries[kWaves], wave_jobs[kWaves];
  int32_t jobs;

  /// Every thread of the workgroup calls it.
  __device__ __forceinline__ void find(const Params &p) {
    for (int e = threadIdx.x; e < p.experts; e += kThreads) tokens[e] = 0;
    __syncthreads();
    for (int q = threadIdx.x; q < p.routes; q += kThreads) {
      const int e = expert_of(p, p.ids[q]);
      if (e >= 0) atomicOr(reinterpret_cast<unsigned long long *>(&tokens[e]), 1ull << (q / p.top));
    }
    __syncthreads();
    // Thread t's experts: kEach in a row.
    const int each = (p.experts + kThreads - 1) / kThreads;
    const int begin = static_cast<int>(threadIdx.x) * each;
    int own_entries = 0, own_jobs = 0;
    for (int e = begin; e < begin + each && e < p.experts; ++e) {
      const int count = __popcll(tokens[e]);
      own_entries += count;
      own_jobs += (count + kJobTokens - 1) / kJobTokens;
    }
    int entries = own_entries, upto = own_jobs;
#pragma unroll
    for (int step = 1; step < kWave; step *= 2) {
      const int e = __shfl_up(entries, step), j = __shfl_up(upto, step);
      if (lane_id() >= step) entries += e, upto += j;
    }
    const int wave = static_cast<int>(threadIdx.x) / kWave;
    if (lane_id() == kWave - 1) wave_entries[wave] = entries, wave_jobs[wave] = upto;
    __syncthreads();
    entries -= own_entries, upto -= own_jobs;
    int all = 0;
    for (int w = 0; w < kWaves; ++w) {
      if (w < wave) entries += wave_entries[w], upto += wave_jobs[w];
      all += wave_jobs[w];
    }
    if (threadIdx.x == 0) jobs = all;
    for (int e = begin; e < begin + each && e < p.experts; ++e) {
      entries_before[e] = static_cast<uint16_t>(entries), jobs_before[e] = static_cast<uint16_t>(upto);
      const int count = __popcll(tokens[e]);
      entries += count;
      upto += (count + kJobTokens - 1) / kJobTokens;
    }
    __syncthreads();
  }
  /// Job n's expert, for n < jobs (by the threads that have it among their experts).
  __device__ __forceinline__ void write_job(const Params &p, int n, Job *job) const {
    for (int e = threadIdx.x; e < p.experts; e += kThreads) {
      const int count = __popcll(tokens[e]), run = n - jobs_before[e];
      if (run < 0 || run * kJobTokens >= count) continue;
      const int left = count - run * kJobTokens;
      *job = Job{e, entries_before[e] + run * kJobTokens, left < kJobTokens ? left : kJobTokens, 0};
    }
  }
  /// Route q's place among the entries and its weight, if it is its token's first to the expert; else place -1.
  __device__ __forceinline__ int place(const Params &p, int q, float &weight) const {
    const int id = p.ids[q], e = expert_of(p, id);
    if (e < 0) return -1;
    const int t = q / p.top;
    weight = p.weights[q];
    for (int k = t * p.top; k < (t + 1) * p.top; ++k) {
      if (k == q || p.ids[k] != id) continue;
      if (k < q) return -1;
      weight += p.weights[k];
    }
    return entries_before[e] + __popcll(tokens[e] & ((1ull << t) - 1));
  }
};

// ---- up and gate ------------------------------------------------------------------------------------------

/// kCols gated columns of one job a workgroup; a wavefront takes a quarter of K's lines.
template <class T, bool kWhole, int kCols>
__global__ void __launch_bounds__(kThreads) gate_up_kernel(Params p) {
  constexpr int kGroups = 2 * kCols / 8;   // of eight weight rows, the up rows' and then the gate rows'
  constexpr int kBlocks = 2 * kCols / 16;  // of sixteen
  __shared__ Routing routing;
  __shared__ Job job;
  __shared__ int32_t job_route[kJobTokens];
  __shared__ u32x4 regroup[kWaves][kGroups * 64];
  routing.find(p);
  const int n = static_cast<int>(blockIdx.y);
  if (n == 0 && blockIdx.x == 0) {
    for (int i = threadIdx.x; i < p.routes; i += kThreads) {
      float weight;
      const int at = routing.place(p, i, weight);
      if (at >= 0) p.entries[at] = Entry{i, weight};
    }
    for (int e = threadIdx.x; e < p.experts; e += kThreads) {
      const int count = __popcll(routing.tokens[e]);
      for (int run = 0; run * kJobTokens < count; ++run) {
        const int left = count - run * kJobTokens;
        p.jobs[routing.jobs_before[e] + run] = Job{e, routing.entries_before[e] + run * kJobTokens, left < kJobTokens ? left : kJobTokens, 0};
      }
    }
    if (threadIdx.x == 0) *p.job_count = routing.jobs;
  }
  if (n >= routing.jobs) return;
  routing.write_job(p, n, &job);
  __syncthreads();
  // The job's tokens, and their routes.
  for (int q = threadIdx.x; q < p.routes; q += kThreads) {
    float weight;
    if (expert_of(p, p.ids[q]) != job.expert) continue;
    const int at = routing.place(p, q, weight) - job.first;
    if (at >= 0 && at < job.count) job_route[at] = q;
  }
  __syncthreads();

  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / kWave);
  const int lane = lane_id(), r16 = lane & 15, g = lane >> 4;
  const int expert = __builtin_amdgcn_readfirstlane(job.expert), count = __builtin_amdgcn_readfirstlane(job.count);
  const int column = static_cast<int>(blockIdx.x) * kCols;
  const uint16_t *weights = p.up_gate + static_cast<int64_t>(expert) * 2 * p.width * p.hidden;
  const uint16_t *row[kGroups];
#pragma unroll
  for (int i = 0; i < kGroups; ++i) {
    const int half = i / (kGroups / 2), c = column + i % (kGroups / 2) * 8 + lane / 8;
    row[i] = weights + static_cast<int64_t>((c < p.width ? c : p.width - 1) + half * p.width) * p.hidden;
  }
  const uint16_t *x = p.x + static_cast<int64_t>(job_route[r16 < count ? r16 : 0] / p.top) * p.x_stride;
  const int lines = (p.hidden + kLine - 1) / kLine;
  const int line_first = wave * lines / kWaves, line_last = (wave + 1) * lines / kWaves;
  floatx4 acc[kBlocks];
#pragma unroll
  for (int b = 0; b < kBlocks; ++b) acc[b] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
  struct Stage {
    u32x4 w[kGroups], x[2];
  };
  auto load = [&](Stage &s, int line) {
#pragma unroll
    for (int i = 0; i < kGroups; ++i) s.w[i] = piece_of<kWhole>(row[i], line * kLine + (lane & 7) * 8, p.hidden);
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) s.x[ks] = piece_of<kWhole>(x, line * kLine + ks * 32 + g * 8, p.hidden);
  };
  auto multiply = [&](const Stage &s) {
    const int r = lane >> 3, piece = lane & 7;
#pragma unroll
    for (int i = 0; i < kGroups; ++i) regroup[wave][i * 64 + r * 8 + (piece ^ r)] = s.w[i];
#pragma unroll
    for (int ks = 0; ks < 2; ++ks)
#pragma unroll
      for (int b = 0; b < kBlocks; ++b) {
        const int rr = r16 & 7;
        acc[b] = T::mfma(regroup[wave][(2 * b + (r16 >> 3)) * 64 + rr * 8 + ((4 * ks + g) ^ rr)], s.x[ks], acc[b]);
      }
  };
  constexpr int kAhead = 4;
  Stage stages[kAhead];
#pragma unroll
  for (int i = 0; i < kAhead; ++i)
    if (line_first + i < line_last) load(stages[i], line_first + i);
  int line = line_first;
  for (; line + 2 * kAhead <= line_last; line += kAhead) {
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      multiply(stages[i]);
      load(stages[i], line + kAhead + i);
    }
  }
  for (; line < line_last; line += kAhead) {
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      if (line + i < line_last) multiply(stages[i]);
      if (line + kAhead + i < line_last) load(stages[i], line + kAhead + i);
    }
  }
  // The wavefronts' sums, each in its own buffer: [block][token][row].
  float *sums = reinterpret_cast<float *>(&regroup[0][0]);
  constexpr int kWaveSums = kGroups * 64 * 4;
  static_assert(kWaveSums >= kBlocks * 256, "a wavefront's sums fit its buffer");
#pragma unroll
  for (int b = 0; b < kBlocks; ++b) *reinterpret_cast<floatx4 *>(sums + wave * kWaveSums + b * 256 + r16 * 16 + 4 * g) = acc[b];
  __syncthreads();
  for (int i = threadIdx.x; i < count * kCols; i += kThreads) {
    const int token = i / kCols, c = i % kCols;
    float up = 0.0f, gated = 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      up += sums[w * kWaveSums + c / 16 * 256 + token * 16 + c % 16];
      gated += sums[w * kWaveSums + (c / 16 + kBlocks / 2) * 256 + token * 16 + c % 16];
    }
    if (column + c >= p.padded) continue;
    // (the padding: zeros)
    const float v = column + c < p.width ? up * gate(gated, p.activation) * kHeld<T> : 0.0f;
    uint16_t *to = p.gated + static_cast<int64_t>(job_route[token]) * 2 * p.padded + column + c;
    const uint16_t value = T::from_f32(v);
    const float error = v - T::to_f32(value);
    to[0] = value;
    to[p.padded] = T::from_f32(error == error ? error : 0.0f);
  }
}

// ---- down -------------------------------------------------------------------------------------------------

/// kCols output columns a workgroup; a wavefront takes a quarter of each job's lines and keeps its own sums of all
/// rows in LDS.
template <class T, bool kWhole, int kCols>
__global__ void __launch_bounds__(kThreads) down_kernel(Params p) {
  constexpr int kGroups = kCols / 8;
  __shared__ Job jobs[kMostTokens * UNISERVE_TOKEN_EXPERTS_MAX_TOP];
  __shared__ float totals[kWaves][kMostTokens][kCols];
  __shared__ u32x4 regroup[kWaves][kGroups * 64];
  const int count = *p.job_count;
  for (int i = threadIdx.x; i < count; i += kThreads) jobs[i] = p.jobs[i];
  for (int i = threadIdx.x; i < kWaves * kMostTokens * kCols; i += kThreads) (&totals[0][0][0])[i] = 0.0f;
  __syncthreads();
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / kWave);
  const int lane = lane_id(), r16 = lane & 15, g = lane >> 4;
  const int column = static_cast<int>(blockIdx.x) * kCols;
  int64_t row[kGroups];
#pragma unroll
  for (int i = 0; i < kGroups; ++i) {
    const int c = column + i * 8 + lane / 8;
    row[i] = static_cast<int64_t>(c < p.hidden ? c : p.hidden - 1) * p.width;
  }
  const int lines = p.padded / kLine;
  const int line_first = wave * lines / kWaves, line_count = (wave + 1) * lines / kWaves - line_first;
  // Units: the wavefront's lines of every job, one job after the other.
  struct Stage {
    u32x4 w[kGroups], values[2], errors[2];
  };
  int load_job = 0, load_line = 0;
  auto load = [&](Stage &s) {
    const Job job = jobs[load_job];
    const uint16_t *weights = p.down + static_cast<int64_t>(__builtin_amdgcn_readfirstlane(job.expert)) * p.hidden * p.width;
    const int route = p.entries[job.first + (r16 < job.count ? r16 : 0)].route;
    const int at = (line_first + load_line) * kLine;
#pragma unroll
    for (int i = 0; i < kGroups; ++i) s.w[i] = piece_of<kWhole>(weights + row[i], at + (lane & 7) * 8, p.width);
    const uint16_t *gated = p.gated + static_cast<int64_t>(route) * 2 * p.padded + at + g * 8;
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      s.values[ks] = *reinterpret_cast<const u32x4 *>(gated + ks * 32);
      s.errors[ks] = *reinterpret_cast<const u32x4 *>(gated + p.padded + ks * 32);
    }
    if (++load_line == line_count) load_line = 0, ++load_job;
  };
  int job_at = 0, line_at = 0;
  floatx4 acc{0.0f, 0.0f, 0.0f, 0.0f};
  auto multiply = [&](const Stage &s) {
    const int r = lane >> 3, piece = lane & 7;
#pragma unroll
    for (int i = 0; i < kGroups; ++i) regroup[wave][i * 64 + r * 8 + (piece ^ r)] = s.w[i];
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      const int rr = r16 & 7;
      const u32x4 w = regroup[wave][(kGroups == 1 ? 0 : r16 >> 3) * 64 + rr * 8 + ((4 * ks + g) ^ rr)];
      acc = T::mfma(w, s.values[ks], acc);
      acc = T::mfma(w, s.errors[ks], acc);
    }
    if (++line_at < line_count) return;
    // The job's rows are complete (of this wavefront's lines): lane r16's token, rows 4 g .. 4 g + 3.
    const Job job = jobs[job_at];
    if (r16 < job.count && (kGroups > 1 || g < 2)) {
      const Entry entry = p.entries[job.first + r16];
      float *total = &totals[wave][entry.route / p.top][4 * g];
      const float weight = entry.weight * (1.0f / kHeld<T>);
#pragma unroll
      for (int i = 0; i < 4; ++i) total[i] = __builtin_fmaf(weight, acc[i], total[i]);
    }
    acc = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
    line_at = 0;
    ++job_at;
  };
  const int units = count * line_count;
  constexpr int kAhead = 8;
  Stage stages[kAhead];
#pragma unroll
  for (int i = 0; i < kAhead; ++i)
    if (i < units) load(stages[i]);
  int unit = 0;
  for (; unit + 2 * kAhead <= units; unit += kAhead) {
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      multiply(stages[i]);
      load(stages[i]);
    }
  }
  for (; unit < units; unit += kAhead) {
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      if (unit + i < units) multiply(stages[i]);
      if (unit + kAhead + i < units) load(stages[i]);
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < p.tokens * kCols; i += kThreads) {
    const int token = i / kCols, c = i % kCols;
    if (column + c >= p.hidden) continue;
    float v = 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) v += totals[w][token][c];
    if (p.residual != nullptr) v += T::to_f32(p.residual[token * p.residual_stride + column + c]);
    p.out[token * p.out_stride + column + c] = T::from_f32(v);
  }
}

template <class T>
void launch(const Params &p, bool whole_x, bool whole_gated, hipStream_t stream) {
  const int64_t most_jobs = p.routes < p.experts + p.routes / kJobTokens ? p.routes : p.experts + p.routes / kJobTokens;
  constexpr int kUpCols = 16, kDownCols = 16;
  const dim3 up_grid(static_cast<uint32_t>(ceil_div(p.padded, kUpCols)), static_cast<uint32_t>(most_jobs));
  if (whole_x) hipLaunchKernelGGL((gate_up_kernel<T, true, kUpCols>), up_grid, dim3(kThreads), 0, stream, p);
  else hipLaunchKernelGGL((gate_up_kernel<T, false, kUpCols>), up_grid, dim3(kThreads), 0, stream, p);
  const dim3 down_grid(static_cast<uint32_t>(ceil_div(p.hidden, kDownCols)));
  if (whole_gated) hipLaunchKernelGGL((down_kernel<T, true, kDownCols>), down_grid, dim3(kThreads), 0, stream, p);
  else hipLaunchKernelGGL((down_kernel<T, false, kDownCols>), down_grid, dim3(kThreads), 0, stream, p);
}

int64_t padded_width(int64_t width) { return ceil_div<int64_t>(width, kLine) * kLine; }
/// The count, the jobs, the entries, the gated pairs.
int64_t workspace_of(int64_t routes, int64_t width) {
  return 16 + routes * (static_cast<int64_t>(sizeof(Job)) + ceil_div<int64_t>(sizeof(Entry), 16) * 16 + 4 * padded_width(width));
}

int32_t run(const uniserve_token_experts_call *call, void *stream) {
  const int64_t tokens = call->tokens, top = call->top, hidden = call->hidden, width = call->width, experts = call->experts;
  if (tokens < 0 || top <= 0 || hidden <= 0 || width <= 0 || experts <= 0)
    return UNISERVE_REFUSE(call, "token_experts needs non-negative tokens and positive top, hidden, width and experts");
  if (tokens > kMostTokens || top > UNISERVE_TOKEN_EXPERTS_MAX_TOP || experts > kMostExperts)
    return UNISERVE_REFUSE(call, "token_experts serves up to %d tokens, %d routes of each and %d experts", kMostTokens,
                           UNISERVE_TOKEN_EXPERTS_MAX_TOP, kMostExperts);
  if (hidden >= (int64_t{1} << 24) || width >= (int64_t{1} << 24))
    return UNISERVE_REFUSE(call, "token_experts serves extents below 2^24");
  if (call->dtype != UNISERVE_DTYPE_BF16 && call->dtype != UNISERVE_DTYPE_F16)
    return UNISERVE_REFUSE(call, "token_experts multiplies bf16 or f16 rows");
  if (call->activation != UNISERVE_ACTIVATION_SILU && call->activation != UNISERVE_ACTIVATION_GELU_TANH)
    return UNISERVE_REFUSE(call, "token_experts gates by silu or gelu_tanh");
  if (call->first_expert < 0 || call->first_expert > INT32_MAX - experts)
    return UNISERVE_REFUSE(call, "token_experts' first expert is negative or does not fit int32");
  if (tokens == 0) return 0;
  if (call->input == nullptr || call->ids == nullptr || call->weights == nullptr || call->up_gate == nullptr ||
      call->down == nullptr || call->out == nullptr || call->workspace == nullptr)
    return UNISERVE_REFUSE(call, "token_experts needs input, ids, weights, up_gate, down, out and a workspace");
  const auto stride_of = [&](const void *array, int64_t stride) { return array != nullptr && tokens > 1 ? stride : hidden; };
  const int64_t x_stride = stride_of(call->input, call->input_row_stride), out_stride = stride_of(call->out, call->out_row_stride);
  const int64_t residual_stride = stride_of(call->residual, call->residual_row_stride);
  for (const int64_t stride : {x_stride, residual_stride, out_stride}) {
    if (stride < hidden) return UNISERVE_REFUSE(call, "token_experts' row strides are shorter than its rows");
    if (stride > kMostElements / tokens) return UNISERVE_REFUSE(call, "token_experts' arrays are too large");
  }
  if (2 * width > kMostElements / hidden / experts) return UNISERVE_REFUSE(call, "token_experts' arrays are too large");
  const int64_t routes = tokens * top, need = workspace_of(routes, width);
  if (call->workspace_bytes < need)
    return UNISERVE_REFUSE(call, "token_experts needs a workspace of %lld bytes", static_cast<long long>(need));
  if (!aligned_to(call->workspace, 16)) return UNISERVE_REFUSE(call, "token_experts' workspace is 16-byte aligned");
  const Extent out = extent(call->out, tokens, hidden, out_stride, 2), work = extent(call->workspace, 1, need, need, 1);
  const Extent residual = extent(call->residual, tokens, hidden, residual_stride, 2);
  const int64_t stack = experts * width * hidden;
  for (const Extent &from : {extent(call->input, tokens, hidden, x_stride, 2), extent(call->ids, 1, routes, routes, 4),
                             extent(call->weights, 1, routes, routes, 4), extent(call->up_gate, 1, 2 * stack, 0, 2),
                             extent(call->down, 1, stack, 0, 2)}) {
    if (overlap(out, from)) return UNISERVE_REFUSE(call, "token_experts' output overlaps one of its inputs");
    if (overlap(work, from)) return UNISERVE_REFUSE(call, "token_experts' workspace overlaps one of its inputs");
  }
  if (overlap(work, residual) || overlap(work, out)) return UNISERVE_REFUSE(call, "token_experts' workspace overlaps its output or its residual");
  if (call->residual != nullptr && !(call->residual == call->out && residual_stride == out_stride) && overlap(out, residual))
    return UNISERVE_REFUSE(call, "token_experts' output overlaps its residual in part");

  Params p{};
  p.x = static_cast<const uint16_t *>(call->input);
  p.up_gate = static_cast<const uint16_t *>(call->up_gate);
  p.down = static_cast<const uint16_t *>(call->down);
  p.residual = static_cast<const uint16_t *>(call->residual);
  p.ids = call->ids;
  p.weights = call->weights;
  p.out = static_cast<uint16_t *>(call->out);
  char *workspace = static_cast<char *>(call->workspace);
  p.job_count = reinterpret_cast<int32_t *>(workspace);
  p.jobs = reinterpret_cast<Job *>(workspace + 16);
  p.entries = reinterpret_cast<Entry *>(workspace + 16 + routes * static_cast<int64_t>(sizeof(Job)));
  p.gated = reinterpret_cast<uint16_t *>(workspace + need - routes * 4 * padded_width(width));
  p.x_stride = x_stride, p.residual_stride = residual_stride, p.out_stride = out_stride;
  p.tokens = static_cast<int32_t>(tokens), p.top = static_cast<int32_t>(top), p.routes = static_cast<int32_t>(routes);
  p.hidden = static_cast<int32_t>(hidden), p.width = static_cast<int32_t>(width), p.padded = static_cast<int32_t>(padded_width(width));
  p.experts = static_cast<int32_t>(experts), p.first_expert = static_cast<int32_t>(call->first_expert);
  p.activation = call->activation;
  const bool whole_x = hidden % 8 == 0 && x_stride % 8 == 0 && aligned_to(call->input, 16) && aligned_to(call->up_gate, 16);
  const bool whole_gated = width % 8 == 0 && aligned_to(call->down, 16);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (call->dtype == UNISERVE_DTYPE_F16) launch<F16>(p, whole_x, whole_gated, s);
  else launch<Bf16>(p, whole_x, whole_gated, s);
  return launched(call, "token_experts");
}

}  // namespace
}  // namespace token_experts
}  // namespace uniserve

extern "C" int64_t uniserve_token_experts_workspace(int64_t tokens, int64_t top, int64_t width) {
  if (tokens <= 0 || top <= 0 || width <= 0 || tokens > UNISERVE_TOKEN_EXPERTS_MAX_TOKENS ||
      top > UNISERVE_TOKEN_EXPERTS_MAX_TOP || width >= (int64_t{1} << 24))
    return 0;
  return uniserve::token_experts::workspace_of(tokens * top, width);
}

extern "C" int32_t uniserve_token_experts(const uniserve_token_experts_call *call, void *stream) {
  return uniserve::guarded(call, [&]() { return uniserve::token_experts::run(call, stream); });
}
