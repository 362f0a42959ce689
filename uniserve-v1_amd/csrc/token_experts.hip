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
//
// Bound by the weights: 128 experts of 2048 x 768, 64 tokens (1.2 GB, one pass among others, traced) 129 us, 6.2 TB/s, and 90 us,
// 4.5 TB/s, where a stream that is only read reaches 6.9; one token (75 MB) 13.2 and 8.8 us, a launch and a chain of ids,
// routing and first weights in each. (The figures further down compare variants in one run each, from graphs over several
// sets of ids, which take some 15 us longer at 64 tokens.) From 32 tokens on the sorted operators, whose second product has
// workgroups by expert and row slice, take less in bf16: 64 tokens 195 us where these two take 218.
// The second kernel's lines of gated values come from L2, at 64 tokens as many bytes as the weights; neither more
// wavefronts, deeper loads nor less LDS traffic (operands without a way through it) made it faster.
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
constexpr int kMostRoutes = kMostTokens * UNISERVE_TOKEN_EXPERTS_MAX_TOP;
constexpr int kLine = 64;  // elements

struct Job {
  uint16_t expert, count;
  int32_t first;  ///< entries first .. first + count - 1
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
  uint16_t *gated;  ///< [routes, lines, 2, 64]: a line's values, then their errors; f16: [routes, lines, 64] of FP32
  int64_t x_stride, residual_stride, out_stride;
  int32_t tokens, top, routes, hidden, width, padded, experts, first_expert, activation;
  int32_t job_tokens;  ///< the most of a job: 4, 8 or 16
};

/// Whether the gated values are FP32 between the kernels: f16's range does not hold them, so the second kernel splits each
/// line into two elements by a power of two of the line's own. bf16's does, and the first kernel splits them once.
/// (The first kernel's workgroups see sixteen columns of a line each, not its largest value. Both kernels of 128 experts of
/// 2048 x 768, f16 with the split and with pairs at one fixed power, which lose small values: T=1 22.6 and 21.6 us, T=16 142 and
/// 135, T=64 243 and 234; 64 experts of 4096 x 1408, T=64 445 and 412.)
template <class T>
constexpr bool kSplitLate = std::is_same<T, F16>::value;

/// Eight elements of a row from `at` on, zeros past its end; kWhole: rows of whole 16-byte pieces.
template <bool kWhole>
__device__ __forceinline__ u32x4 piece_of(const uint16_t *row, int64_t at, int64_t width) {
  if constexpr (kWhole) return at < width ? *reinterpret_cast<const u32x4 *>(row + at) : u32x4{0, 0, 0, 0};
  else return load8(row, at, width);
}
/// Eight elements of a weight row; kOnce: not kept in the caches.
template <bool kWhole, bool kOnce>
__device__ __forceinline__ u32x4 weights_of(const uint16_t *row, int64_t at, int64_t width) {
  if constexpr (kWhole && kOnce) return at < width ? __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(row + at)) : u32x4{0, 0, 0, 0};
  else return piece_of<kWhole>(row, at, width);
}

/// An id's expert in the stacks, or -1.
__device__ __forceinline__ int expert_of(const Params &p, int id) {
  const int e = id >= p.first_expert ? id - p.first_expert : -1;  // (the first is not negative)
  return e < p.experts ? e : -1;
}

/// Where the routes lead: the tokens that name each expert, and how many tokens and jobs come before it.
struct Routing {
  uint64_t tokens[kMostExperts];
  int16_t experts[kMostRoutes];  ///< of each route, or -1
  uint16_t entries_before[kMostExperts], jobs_before[kMostExperts];
  int32_t wave_entries[kWaves], wave_jobs[kWaves];
  int32_t jobs;

  /// Every thread of the workgroup calls it.
  __device__ __forceinline__ void find(const Params &p) {
    for (int q = threadIdx.x; q < p.routes; q += kThreads) experts[q] = static_cast<int16_t>(expert_of(p, p.ids[q]));
    for (int e = threadIdx.x; e < p.experts; e += kThreads) tokens[e] = 0;
    __syncthreads();
    for (int q = threadIdx.x; q < p.routes; q += kThreads) {
      const int e = experts[q];
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
      own_jobs += (count + p.job_tokens - 1) / p.job_tokens;
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
      upto += (count + p.job_tokens - 1) / p.job_tokens;
    }
    __syncthreads();
  }
  /// Job n's expert, for n < jobs (by the threads that have it among their experts).
  __device__ __forceinline__ void write_job(const Params &p, int n, Job *job) const {
    for (int e = threadIdx.x; e < p.experts; e += kThreads) {
      const int count = __popcll(tokens[e]), run = n - jobs_before[e];
      if (run < 0 || run * p.job_tokens >= count) continue;
      const int left = count - run * p.job_tokens;
      *job = Job{static_cast<uint16_t>(e), static_cast<uint16_t>(left < p.job_tokens ? left : p.job_tokens), entries_before[e] + run * p.job_tokens};
    }
  }
  /// Whether route q is its token's first to its expert.
  __device__ __forceinline__ bool first(const Params &p, int q) const {
    const int start = q / p.top * p.top;
    bool before = false;
    for (int k = start; k < q; ++k) before = before || experts[k] == experts[q];
    return experts[q] >= 0 && !before;
  }
  /// Its place among the entries.
  __device__ __forceinline__ int place(const Params &p, int q) const {
    const int e = experts[q];
    return entries_before[e] + __popcll(tokens[e] & ((1ull << (q / p.top)) - 1));
  }
};

// ---- up and gate ------------------------------------------------------------------------------------------

/// kCols gated columns of one job a workgroup; a wavefront takes a quarter of K's lines, two of them in flight (four:
/// 146 us against 137 at 64 tokens, fewer workgroups to a CU).
template <class T, bool kWhole, bool kOnce, int kCols>
__global__ void __launch_bounds__(kThreads) gate_up_kernel(Params p) {
  constexpr int kGroups = 2 * kCols / 8;   // of eight weight rows, the up rows' and then the gate rows'
  constexpr int kBlocks = 2 * kCols / 16;  // of sixteen
  __shared__ Routing routing;
  __shared__ Job job;
  __shared__ int32_t job_route[16];
  __shared__ u32x4 regroup[kWaves][kGroups * 64];
  routing.find(p);
  const int n = static_cast<int>(blockIdx.y);
  if (n == 0 && blockIdx.x == 0) {
    for (int q = threadIdx.x; q < p.routes; q += kThreads) {
      if (!routing.first(p, q)) continue;
      float weight = p.weights[q];
      for (int k = q + 1; k < (q / p.top + 1) * p.top; ++k)
        if (routing.experts[k] == routing.experts[q]) weight += p.weights[k];
      p.entries[routing.place(p, q)] = Entry{q, weight};
    }
    for (int e = threadIdx.x; e < p.experts; e += kThreads) {
      const int count = __popcll(routing.tokens[e]);
      for (int run = 0; run * p.job_tokens < count; ++run) {
        const int left = count - run * p.job_tokens;
        p.jobs[routing.jobs_before[e] + run] =
            Job{static_cast<uint16_t>(e), static_cast<uint16_t>(left < p.job_tokens ? left : p.job_tokens), routing.entries_before[e] + run * p.job_tokens};
      }
    }
    if (threadIdx.x == 0) *p.job_count = routing.jobs;
  }
  if (n >= routing.jobs) return;
  routing.write_job(p, n, &job);
  __syncthreads();
  // The job's tokens, and their routes.
  for (int q = threadIdx.x; q < p.routes; q += kThreads) {
    if (routing.experts[q] != job.expert || !routing.first(p, q)) continue;
    const int at = routing.place(p, q) - job.first;
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
    for (int i = 0; i < kGroups; ++i) s.w[i] = weights_of<kWhole, kOnce>(row[i], line * kLine + (lane & 7) * 8, p.hidden);
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) s.x[ks] = piece_of<kWhole>(x, line * kLine + ks * 32 + g * 8, p.hidden);
  };
  auto multiply = [&](const Stage &s) {
    const int r = lane >> 3, piece = lane & 7;
    wave_fence();  // (the stage before has been read)
#pragma unroll
    for (int i = 0; i < kGroups; ++i) regroup[wave][i * 64 + r * 8 + (piece ^ r)] = s.w[i];
    wave_fence();
#pragma unroll
    for (int ks = 0; ks < 2; ++ks)
#pragma unroll
      for (int b = 0; b < kBlocks; ++b) {
        const int rr = r16 & 7;
        acc[b] = T::mfma(regroup[wave][(2 * b + (r16 >> 3)) * 64 + rr * 8 + ((4 * ks + g) ^ rr)], s.x[ks], acc[b]);
      }
  };
  constexpr int kAhead = 2;
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
  wave_fence();
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
    const float v = column + c < p.width ? up * gate(gated, p.activation) : 0.0f;
    if constexpr (kSplitLate<T>) {
      reinterpret_cast<float *>(p.gated)[static_cast<int64_t>(job_route[token]) * p.padded + column + c] = v;
      continue;
    }
    uint16_t *to = p.gated + static_cast<int64_t>(job_route[token]) * 2 * p.padded + (column + c) / kLine * 2 * kLine + (column + c) % kLine;
    const uint16_t value = T::from_f32(v);
    const float error = v - T::to_f32(value);
    to[0] = value;
    // (a value that is not finite, or rounds to an infinity, has no error: the pair's sum is the value)
    to[kLine] = T::from_f32(__builtin_fabsf(error) < __builtin_inff() ? error : 0.0f);
  }
}

// ---- down -------------------------------------------------------------------------------------------------

/// A lane's four of a line's sixty-four FP32 values (sixteen lanes in a row hold one) as f16 elements and their errors, in
/// parts of the power of two that brings the line's largest to [1, 2). At most 2^126, also where an infinity is the
/// largest; NaN is passed over. What is not finite has NaN for its error, whose sum is then left out.
struct LineSplit {
  uint2 values, errors;
  float factor;
  __device__ __forceinline__ explicit LineSplit(floatx4 v) {
    typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
    const float own = __builtin_fmaxf(__builtin_fmaxf(__builtin_fabsf(v[0]), __builtin_fabsf(v[1])),
                                      __builtin_fmaxf(__builtin_fabsf(v[2]), __builtin_fabsf(v[3])));
    uint32_t power = row16_max(__float_as_uint(own)) & 0x7f800000u;
    power = power < (1u << 23) ? 1u << 23 : power;
    power = power > (253u << 23) ? 253u << 23 : power;
    factor = __uint_as_float(power);
    const float scale = __uint_as_float((254u << 23) - power);
    const auto pair = [](float lo, float hi) {
      uint32_t bits = __builtin_bit_cast(uint32_t, f16x2{static_cast<_Float16>(lo), static_cast<_Float16>(hi)});
      asm("" : "+v"(bits));  // (opaque: the elements are taken from the pair, not rounded a second time each)
      return __builtin_bit_cast(f16x2, bits);
    };
    const f16x2 a = pair(v[0] * scale, v[1] * scale), b = pair(v[2] * scale, v[3] * scale);
    const auto left = [&](float of, _Float16 value) { return static_cast<_Float16>(__builtin_fmaf(of, scale, -static_cast<float>(value))); };
    const f16x2 c{left(v[0], a[0]), left(v[1], a[1])}, d{left(v[2], b[0]), left(v[3], b[1])};
    values = uint2{__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b)};
    errors = uint2{__builtin_bit_cast(uint32_t, c), __builtin_bit_cast(uint32_t, d)};
  }
};

/// kCols output columns a workgroup, kSets sets of four wavefronts. A set takes the jobs of the experts whose number is its
/// own modulo kSets, a wavefront a quarter of each job's lines; it keeps its own sums of all rows in LDS. (By the
/// experts' numbers: a row's sums come in one order, whatever the other rows name.)
/// (Weights loaded as lane l's chunk of row l % 8, in half l % 16 / 8 of the line, so that the matrix instruction takes them
/// without LDS, are slower: T=16 52 us against 50, T=64 106 against 98.)
/// kTokens of a job at most: their gated values come as whole lines, too, and through LDS (in the operand layout
/// they took four loads of sixteen columns for any number of tokens: T=16 72 us, 50 now). With eight columns and
/// sixteen tokens the bf16 kernels spill 4 registers (of rows that are not whole pieces 13).
template <class T, bool kWhole, bool kOnce, int kCols, int kSets, int kTokens>
__global__ void __launch_bounds__(kSets *kThreads) down_kernel(Params p) {
  constexpr int kGroups = kCols / 8, kAllThreads = kSets * kThreads;
  __shared__ Job jobs[kMostRoutes];  // each set's, one set's after the other's
  __shared__ Entry entries[kMostRoutes];
  __shared__ float totals[kSets * kWaves][kMostTokens][kCols];
  __shared__ u32x4 regroup[kSets * kWaves][kGroups * 64];
  __shared__ u32x4 lines_of[kSets * kWaves][kTokens * 16];
  [[maybe_unused]] __shared__ float line_factor[kSets * kWaves][kTokens];
  const int count = *p.job_count;
  const int all_wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / kWave);
  const int wave = all_wave % kWaves, set = all_wave / kWaves;
  const int lane = lane_id(), r16 = lane & 15, g = lane >> 4;
  for (int i = threadIdx.x; i < p.routes; i += kAllThreads) entries[i] = p.entries[i];  // (those past the last are not read)
  for (int i = threadIdx.x; i < kSets * kWaves * kMostTokens * kCols; i += kAllThreads) (&totals[0][0][0])[i] = 0.0f;
  // Every wavefront counts the jobs of the sets before its own and of its own; the set's first one lists them.
  int first_job = 0, own_jobs = 0;
  for (int i = 0; i < count; i += kWave) {
    const int of = i + lane < count ? p.jobs[i + lane].expert % kSets : kSets;
    first_job += __popcll(ballot(of < set));
    own_jobs += __popcll(ballot(of == set));
  }
  if (wave == 0) {
    int at = first_job;
    for (int i = 0; i < count; i += kWave) {
      const Job job = p.jobs[i + lane < count ? i + lane : 0];
      const uint64_t own = ballot(i + lane < count && job.expert % kSets == set);
      if ((own >> lane) & 1) jobs[at + __popcll(own & ((1ull << lane) - 1))] = job;
      at += __popcll(own);
    }
  }
  __syncthreads();
  const int column = static_cast<int>(blockIdx.x) * kCols;
  int64_t row[kGroups];
#pragma unroll
  for (int i = 0; i < kGroups; ++i) {
    const int c = column + i * 8 + lane / 8;
    row[i] = static_cast<int64_t>(c < p.hidden ? c : p.hidden - 1) * p.width;
  }
  const int lines = p.padded / kLine;
  const int line_first = wave * lines / kWaves, line_count = (wave + 1) * lines / kWaves - line_first;
  // Units: the wavefront's lines of every job of its set, one job after the other.
  struct Stage {
    u32x4 w[kGroups], gated[kTokens / 4];
  };
  int load_job = first_job, load_line = 0;
  const uint16_t *weights[kGroups], *gated[kTokens / 4];  // the lane's rows of the job to load
  auto load = [&](Stage &s) {
    if (load_line == 0) {
      const Job job = jobs[load_job++];
      const uint16_t *down = p.down + static_cast<int64_t>(__builtin_amdgcn_readfirstlane(job.expert)) * p.hidden * p.width;
#pragma unroll
      for (int i = 0; i < kGroups; ++i) weights[i] = down + row[i];
#pragma unroll
      for (int i = 0; i < kTokens / 4; ++i) {
        const int token = i * 4 + lane / 16;
        gated[i] = p.gated + static_cast<int64_t>(entries[job.first + (token < job.count ? token : 0)].route) * 2 * p.padded + (lane & 15) * 8;
      }
    }
    const int at = (line_first + load_line) * kLine;
#pragma unroll
    for (int i = 0; i < kGroups; ++i) s.w[i] = weights_of<kWhole, kOnce>(weights[i], at + (lane & 7) * 8, p.width);
#pragma unroll
    for (int i = 0; i < kTokens / 4; ++i) s.gated[i] = *reinterpret_cast<const u32x4 *>(gated[i] + at * 2);
    load_line = load_line + 1 == line_count ? 0 : load_line + 1;
  };
  int job_at = first_job, line_at = 0;
  constexpr int kApart = kTokens == 16 ? 2 : 1;  // the errors' columns have sums of their own
  floatx4 acc[kApart];
  auto clear = [&]() {
#pragma unroll
    for (int i = 0; i < kApart; ++i) acc[i] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
  };
  clear();
  auto multiply = [&](const Stage &s) {
    wave_fence();  // (the stage before has been read)
#pragma unroll
    for (int i = 0; i < kGroups; ++i) regroup[all_wave][i * 64 + lane / 8 * 8 + ((lane & 7) ^ (lane / 8))] = s.w[i];
    // Chunk c (eight values, then eight errors) of a token's line lies at c ^ 4 token: four tokens' chunks in all banks.
#pragma unroll
    for (int i = 0; i < kTokens / 4; ++i) {
      const int token = i * 4 + lane / 16;
      if constexpr (kSplitLate<T>) {
        const LineSplit split(__builtin_bit_cast(floatx4, s.gated[i]));
        uint2 *line = reinterpret_cast<uint2 *>(&lines_of[all_wave][token * 16]);
        const int piece = (lane & 15) >> 1, swap = token * 4 & 15;
        line[(piece ^ swap) * 2 + (lane & 1)] = split.values;
        line[((piece + 8) ^ swap) * 2 + (lane & 1)] = split.errors;
        if ((lane & 15) == 0) line_factor[all_wave][token] = split.factor;
      } else {
        lines_of[all_wave][token * 16 + ((lane & 15) ^ (token * 4 & 15))] = s.gated[i];
      }
    }
    wave_fence();
    // Operand columns: the tokens' values and then their errors, or, of sixteen tokens, one after the other.
    const int token = r16 % kTokens, errors = kTokens < 16 ? r16 / kTokens % 2 * 8 : 0;
    const u32x4 *line = &lines_of[all_wave][token * 16];
    auto chunk = [&](int c) { return line[c ^ (token * 4 & 15)]; };
    floatx4 line_acc[kApart];
#pragma unroll
    for (int i = 0; i < kApart; ++i) line_acc[i] = kSplitLate<T> ? floatx4{0.0f, 0.0f, 0.0f, 0.0f} : acc[i];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const u32x4 w = regroup[all_wave][(kGroups == 1 ? 0 : r16 >> 3) * 64 + (r16 & 7) * 8 + ((4 * half + g) ^ (r16 & 7))];
      line_acc[0] = T::mfma(w, chunk(errors + 4 * half + g), line_acc[0]);
      if constexpr (kApart == 2) line_acc[1] = T::mfma(w, chunk(8 + 4 * half + g), line_acc[1]);
    }
    [[maybe_unused]] float factor = 1.0f;
    if constexpr (kSplitLate<T>) factor = line_factor[all_wave][token];
#pragma unroll
    for (int i = 0; i < kApart; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[i][e] = kSplitLate<T> ? __builtin_fmaf(line_acc[i][e], factor, acc[i][e]) : line_acc[i][e];
    if (++line_at < line_count) return;
    // The job's rows are complete (of this wavefront's lines): lane r16's token, rows 4 g .. 4 g + 3.
    const Job job = jobs[job_at];
    const Entry entry = entries[job.first + (r16 < job.count ? r16 : 0)];
    const float weight = entry.weight;
    float *total = totals[all_wave][entry.route / p.top];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      // (The errors' sum is added to the values' for any kTokens: the order of a row's additions is one. Where it is not
      // finite a weight is not: the values' sum alone is what the weights make of the row - an exact value's error
      // times an infinity would be NaN, another's may be the other infinity.)
      float errors;
      if constexpr (kApart == 1) errors = __shfl_xor(acc[0][e], kTokens);
      else errors = acc[1][e];
      const float v = acc[0][e] + (__builtin_fabsf(errors) < __builtin_inff() ? errors : 0.0f);
      if (r16 < job.count && (kGroups > 1 || g < 2)) total[4 * g + e] = __builtin_fmaf(weight, v, total[4 * g + e]);
    }
    clear();
    line_at = 0;
    ++job_at;
  };
  const int units = own_jobs * line_count;
  constexpr int kAhead = kSplitLate<T> && kTokens == 16 ? 3 : 4;  // (four spill 31 to 82 registers there)
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
  for (int i = threadIdx.x; i < p.tokens * kCols; i += kAllThreads) {
    const int token = i / kCols, c = i % kCols;
    if (column + c >= p.hidden) continue;
    float v = 0.0f;
#pragma unroll
    for (int w = 0; w < kSets * kWaves; ++w) v += totals[w][token][c];
    if (p.residual != nullptr) v += T::to_f32(p.residual[token * p.residual_stride + column + c]);
    p.out[token * p.out_stride + column + c] = T::from_f32(v);
  }
}

template <class T, bool kWhole, bool kOnce, int kCols, int kSets, int kTokens>
void launch_down_kernel(const Params &p, hipStream_t stream) {
  hipLaunchKernelGGL((down_kernel<T, kWhole, kOnce, kCols, kSets, kTokens>), dim3(static_cast<uint32_t>(ceil_div(p.hidden, kCols))),
                     dim3(kSets * kThreads), 0, stream, p);
}

/// Eight columns and sixteen wavefronts a workgroup where each CU gets one at most, else sixteen columns and eight
/// wavefronts (128 experts of 2048 x 768, T=16: 51 us against 78, T=64 98 against 129; 64 of 4096 x 1408, T=64 184
/// against 141).
template <class T, bool kWhole, bool kOnce>
void launch_down(const Params &p, hipStream_t stream) {
  const bool narrow = ceil_div(p.hidden, 8) <= 256;
  switch (p.job_tokens) {
    case 4: return narrow ? launch_down_kernel<T, kWhole, kOnce, 8, 4, 4>(p, stream) : launch_down_kernel<T, kWhole, kOnce, 16, 2, 4>(p, stream);
    case 8: return narrow ? launch_down_kernel<T, kWhole, kOnce, 8, 4, 8>(p, stream) : launch_down_kernel<T, kWhole, kOnce, 16, 2, 8>(p, stream);
    default: return narrow ? launch_down_kernel<T, kWhole, kOnce, 8, 4, 16>(p, stream) : launch_down_kernel<T, kWhole, kOnce, 16, 2, 16>(p, stream);
  }
}

template <class T, bool kOnce>
void launch_both(const Params &p, bool whole_x, bool whole_gated, hipStream_t stream) {
  constexpr int kCols = 16;  // (32: T=64 134 us against 136, T=1 14.2 against 12.3)
  const int64_t bound = p.experts + p.routes / p.job_tokens;  // of the jobs, without a look at the ids
  const dim3 grid(static_cast<uint32_t>(ceil_div(p.padded, kCols)), static_cast<uint32_t>(p.routes < bound ? p.routes : bound));
  if (whole_x) hipLaunchKernelGGL((gate_up_kernel<T, true, kOnce, kCols>), grid, dim3(kThreads), 0, stream, p);
  else hipLaunchKernelGGL((gate_up_kernel<T, false, kOnce, kCols>), grid, dim3(kThreads), 0, stream, p);
  whole_gated ? launch_down<T, true, kOnce>(p, stream) : launch_down<T, false, kOnce>(p, stream);
}

/// Jobs of at most 4, 8 or 16 tokens, by the tokens that an expert expects: the fewer, the less gated data the second kernel
/// loads (128 experts, top 8, gate_up and down: T=16, one token an expert, 86 + 51 us with four, 85 + 59 with eight;
/// T=64, four an expert, 159 + 106, 137 + 100 and with sixteen 133 + 116; 64 experts of 4096 x 1408, eight tokens
/// each, 337 + 230, 281 + 185, 244 + 166). Where an expert seldom has a second job its weights are loaded past the caches
/// (T=64 151 + 101 us without that, eight experts of 16 tokens 15 + 16 without and 19 + 19 with it).
template <class T>
void launch(Params &p, bool whole_x, bool whole_gated, hipStream_t stream) {
  p.job_tokens = p.tokens <= 4 || p.routes <= 2 * p.experts ? 4 : p.tokens <= 8 || p.routes <= 6 * p.experts ? 8 : 16;
  if (p.tokens <= p.job_tokens || 2 * p.routes <= p.experts * p.job_tokens) launch_both<T, true>(p, whole_x, whole_gated, stream);
  else launch_both<T, false>(p, whole_x, whole_gated, stream);
}

int64_t padded_width(int64_t width) { return ceil_div<int64_t>(width, kLine) * kLine; }
/// The count, the jobs, the entries, the gated pairs.
int64_t workspace_of(int64_t routes, int64_t width) {
  return 16 + routes * (static_cast<int64_t>(sizeof(Job) + sizeof(Entry)) + 4 * padded_width(width));
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
