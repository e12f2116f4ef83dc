// beam_select.hip -- the best continuations of the beams of many searches.
//
//   score(b, v) = s_b + x_bv - log sum_u exp x_bu,   rank = score * length^-power
//
// and of the beams x vocab candidates of a search the `beams` of the largest
// rank, ties to the lower beam, the larger x, the lower token; a beam that has
// ended is its only candidate.  Within a row the order is that of x, so a block that takes a run
// of a row's columns keeps the run's `beams` largest x with its maximum and sum
// of exponentials, in one pass over the logits; a block a search then has the
// rows' sums and ranks what the runs kept, in 64 bits.
//
// The largest `beams` of a block's values: the beams-th largest of the threads'
// own maxima is a value that at least `beams` values reach, and few others do;
// those are gathered and each one's place is the number of better ones.  Where
// more reach it than there is room for (a row of equal logits), the block takes
// one maximum after another instead.
#include "device_common.h"

#include <algorithm>
#include <cfloat>

namespace mmr {

namespace {

constexpr int kRunThreads = 256, kRunEach = 16, kRun = kRunThreads * kRunEach;  // columns of a run
constexpr int kRunRoom = 512;   // at most (kMostBeams - 1) * kRunEach if fewer threads than beams have a value
constexpr int kJoinThreads = 256, kJoinRoom = 512;
static_assert((kMostBeams - 1) * kRunEach <= kRunRoom, "values of fewer threads than beams");

struct RunHead {
  float top, sum;  // the largest x of the run, the sum of 2^((x - top) log2 e); sum NaN: not finite
};

// Of a row's run: its head, then `beams` values and columns, the best first
// (column -1: none).
struct RunLayout {
  RunHead* head;
  float* value;
  int* column;
};
__host__ __device__ inline RunLayout run_layout(void* workspace, int64_t runs, int beams) {
  RunLayout l;
  l.head = static_cast<RunHead*>(workspace);
  l.value = reinterpret_cast<float*>(l.head + runs);
  l.column = reinterpret_cast<int*>(l.value + runs * beams);
  return l;
}
inline int runs_of(int vocab) { return (vocab + kRun - 1) / kRun; }

// A candidate of a search; beam INT_MAX: none.
struct Candidate {
  double rank;
  float x;
  int beam, token;
};
__device__ __forceinline__ bool better(const Candidate& a, const Candidate& b) {
  if (a.rank != b.rank) return a.rank > b.rank;
  if (a.beam != b.beam) return a.beam < b.beam;
  return argmax_better(a.x, a.token, b.x, b.token);
}
__device__ __forceinline__ Candidate no_candidate() { return Candidate{-INFINITY, -INFINITY, INT_MAX, INT_MAX}; }

__global__ __launch_bounds__(kRunThreads) void beam_runs_kernel(BeamArgs a, int runs) {
  constexpr int kWaves = kRunThreads / kWave;
  __shared__ float tops[kRunThreads], sh_sum[kWaves], room_value[kRunRoom], best_value[kWaves], sh_limit;
  __shared__ int room_column[kRunRoom], best_column[kWaves], sh_count;
  const int run = blockIdx.x % runs, row = blockIdx.x / runs, tid = threadIdx.x;
  const int wave = tid / kWave, lane = tid % kWave;
  const RunLayout to = run_layout(a.workspace, static_cast<int64_t>(runs) * a.searches * a.beams, a.beams);
  const int64_t at = static_cast<int64_t>(row) * runs + run;
  if (a.eos >= 0 && a.ended[row] != 0) return;  // not read by the join
  const float* x = a.logits + static_cast<int64_t>(row) * a.vocab;
  const int first = run * kRun, last = min(first + kRun, a.vocab);
  float v[kRunEach];
  float top = -INFINITY;
  bool bad = false;
#pragma unroll
  for (int i = 0; i < kRunEach; ++i) {
    const int c = first + tid + kRunThreads * i;
    v[i] = c < last ? x[c] : -INFINITY;
    bad = bad || !(v[i] < INFINITY);
    top = fmaxf(top, v[i]);
  }
  tops[tid] = top;
  if (tid == 0) {
    sh_count = 0;
    sh_limit = -INFINITY;
  }
  __syncthreads();
  float block_top = -INFINITY;
  int better = 0;
  for (int i = 0; i < kRunThreads; ++i) {
    block_top = fmaxf(block_top, tops[i]);
    better += tops[i] > top || (tops[i] == top && i < tid);
  }
  if (better == a.beams - 1) sh_limit = top;
  const float base = fmaxf(block_top, -FLT_MAX);
  float sum = 0.0f;
#pragma unroll
  for (int i = 0; i < kRunEach; ++i) sum += __builtin_amdgcn_exp2f((v[i] - base) * 1.4426950408889634f);
  if (bad) sum = __builtin_nanf("");
  sum = group_sum<kWave>(sum);
  if (lane == 0) sh_sum[wave] = sum;
  __syncthreads();
  const float limit = sh_limit;
  if (tid == 0) {
    float s = sh_sum[0];
    for (int w = 1; w < kWaves; ++w) s += sh_sum[w];
    to.head[at] = RunHead{base, s};
  }
#pragma unroll
  for (int i = 0; i < kRunEach; ++i) {
    if (v[i] >= limit && v[i] > -INFINITY) {
      const int place = atomicAdd(&sh_count, 1);
      if (place < kRunRoom) {
        room_value[place] = v[i];
        room_column[place] = first + tid + kRunThreads * i;
      }
    }
  }
  __syncthreads();
  const int count = sh_count;
  float* value = to.value + at * a.beams;
  int* column = to.column + at * a.beams;
  if (count <= kRunRoom) {
    for (int n = tid; n < max(count, a.beams); n += kRunThreads) {
      if (n >= count) {
        column[n] = -1;
        continue;
      }
      const float mine = room_value[n];
      const int c = room_column[n];
      int place = 0;
      for (int j = 0; j < count; ++j) place += argmax_better(room_value[j], room_column[j], mine, c);
      if (place < a.beams) {
        value[place] = mine;
        column[place] = c;
      }
    }
    return;
  }
  for (int n = 0; n < a.beams; ++n) {
    float bv = -INFINITY;
    int bc = INT_MAX;
#pragma unroll
    for (int i = 0; i < kRunEach; ++i) {
      const int c = first + tid + kRunThreads * i;
      if (v[i] > -INFINITY && argmax_better(v[i], c, bv, bc)) {
        bv = v[i];
        bc = c;
      }
    }
    wave_argmax(bv, bc);
    if (lane == 0) {
      best_value[wave] = bv;
      best_column[wave] = bc;
    }
    __syncthreads();
    bv = best_value[0];
    bc = best_column[0];
    for (int w = 1; w < kWaves; ++w)
      if (argmax_better(best_value[w], best_column[w], bv, bc)) {
        bv = best_value[w];
        bc = best_column[w];
      }
    if (tid == 0) {
      value[n] = bv;
      column[n] = bc;
    }
#pragma unroll
    for (int i = 0; i < kRunEach; ++i)
      if (first + tid + kRunThreads * i == bc) v[i] = -INFINITY;
    __syncthreads();
  }
}

// A block a search.
__global__ __launch_bounds__(kJoinThreads) void beam_join_kernel(BeamArgs a, int runs) {
  constexpr int kWaves = kJoinThreads / kWave;
  __shared__ double sh_lse[kMostBeams], sh_factor[kMostBeams], tops[kJoinThreads], sh_limit;
  __shared__ float sh_score[kMostBeams];
  __shared__ int sh_state[kMostBeams], sh_length[kMostBeams], sh_count;
  __shared__ Candidate room[kJoinRoom], wave_best[kWaves];
  const int search = blockIdx.x, tid = threadIdx.x, wave = tid / kWave, lane = tid % kWave;
  const RunLayout from = run_layout(a.workspace, static_cast<int64_t>(runs) * a.searches * a.beams, a.beams);
  const int first = search * a.beams;
  // States of a beam: 0 no candidates, 1 those of its row, 2 itself.  All that
  // is read of the beams as they were is read before the barrier: the new ones
  // may take their place.
  for (int b = wave; b < a.beams; b += kWaves) {
    const float score = a.scores[first + b];
    const bool done = a.eos >= 0 && a.ended[first + b] != 0;
    int state = fabsf(score) < INFINITY ? done ? 2 : 1 : 0;
    bool bad = !(score < INFINITY);
    double lse = 0.0;
    if (!done) {
      const RunHead* head = from.head + static_cast<int64_t>(first + b) * runs;
      float top = -FLT_MAX;
      for (int r = lane; r < runs; r += kWave) top = fmaxf(top, head[r].top);
      top = group_max<kWave>(top);
      double sum = 0.0;
      for (int r = lane; r < runs; r += kWave)
        sum += static_cast<double>(head[r].sum) * exp(static_cast<double>(head[r].top) - top);
#pragma unroll
      for (int step = 1; step < kWave; step *= 2) sum += __shfl_xor(sum, step);
      bad = bad || !(sum == sum);
      if (!(sum > 0.0)) state = 0;  // not finite, or every token is masked
      lse = top + log(sum);
    }
    if (lane == 0) {
      if (bad) atomicOr(a.error, kKv8NotFinite);
      sh_state[b] = state;
      sh_score[b] = score;
      sh_lse[b] = lse;
      sh_length[b] = a.lengths[first + b] + (done ? 0 : 1);
      sh_factor[b] = a.length_power == 0.0 ? 1.0 : pow(static_cast<double>(max(sh_length[b], 1)), -a.length_power);
    }
  }
  if (tid == 0) {
    sh_count = 0;
    sh_limit = -INFINITY;
  }
  __syncthreads();
  const int each = runs * a.beams, total = a.beams * each;
  auto score_of = [&](int b, float x) -> double {
    return sh_state[b] == 2 ? sh_score[b] : sh_score[b] + (static_cast<double>(x) - sh_lse[b]);
  };
  auto candidate = [&](int number) {  // (beam * runs + run) * beams + place
    Candidate c = no_candidate();
    const int b = number / each, state = sh_state[b];
    if (state == 0 || (state == 2 && number != b * each)) return c;
    const int64_t at = static_cast<int64_t>(first) * each + number;
    const int token = state == 2 ? a.eos : from.column[at];
    if (token < 0) return c;
    const float x = state == 2 ? 0.0f : from.value[at];
    const double score = score_of(b, x);
    if (static_cast<float>(score) > -INFINITY) c = Candidate{score * sh_factor[b], x, b, token};
    return c;
  };
  double top = -INFINITY;
  for (int n = tid; n < total; n += kJoinThreads) top = fmax(top, candidate(n).rank);
  tops[tid] = top;
  __syncthreads();
  int above = 0;
  for (int i = 0; i < kJoinThreads; ++i) above += tops[i] > top || (tops[i] == top && i < tid);
  if (above == a.beams - 1) sh_limit = top;
  __syncthreads();
  const double limit = sh_limit;
  for (int n = tid; n < total; n += kJoinThreads) {
    const Candidate c = candidate(n);
    if (c.beam != INT_MAX && c.rank >= limit) {
      const int place = atomicAdd(&sh_count, 1);
      if (place < kJoinRoom) room[place] = c;
    }
  }
  __syncthreads();
  const int count = sh_count;
  auto store = [&](int place, const Candidate& c) {
    const int o = first + place;
    const bool none = c.beam == INT_MAX;
    const int token = none ? max(a.eos, 0) : c.token;
    a.scores_out[o] = none ? -INFINITY : static_cast<float>(score_of(c.beam, c.x));
    a.parent[o] = none ? -1 : first + c.beam;
    a.token[o] = token;
    a.lengths_out[o] = none ? 0 : sh_length[c.beam];
    a.ended_out[o] = a.eos >= 0 && token == a.eos;
  };
  if (count <= kJoinRoom) {
    for (int n = tid; n < max(count, a.beams); n += kJoinThreads) {
      if (n >= count) {
        store(n, no_candidate());
        continue;
      }
      const Candidate mine = room[n];
      int place = 0;
      for (int j = 0; j < count; ++j) place += better(room[j], mine);
      if (place < a.beams) store(place, mine);
    }
    return;
  }
  // More than there is room for: one after another, each the best that is worse than the last.
  Candidate last{INFINITY, INFINITY, -1, -1};
  for (int n = 0; n < a.beams; ++n) {
    Candidate best = no_candidate();
    for (int i = tid; i < total; i += kJoinThreads) {
      const Candidate c = candidate(i);
      if (c.beam != INT_MAX && better(last, c) && better(c, best)) best = c;
    }
#pragma unroll
    for (int step = 1; step < kWave; step *= 2) {
      const Candidate other{__shfl_xor(best.rank, step), __shfl_xor(best.x, step), __shfl_xor(best.beam, step),
                            __shfl_xor(best.token, step)};
      if (better(other, best)) best = other;
    }
    if (lane == 0) wave_best[wave] = best;
    __syncthreads();
    best = wave_best[0];
    for (int w = 1; w < kWaves; ++w)
      if (better(wave_best[w], best)) best = wave_best[w];
    if (tid == 0) store(n, best);
    last = best;
    __syncthreads();
  }
}

}  // namespace

int64_t beam_select_workspace(int searches, int beams, int vocab) {
  const int64_t runs = static_cast<int64_t>(runs_of(vocab)) * searches * beams;
  return runs * static_cast<int64_t>(sizeof(RunHead) + beams * (sizeof(float) + sizeof(int)));
}

hipError_t launch_beam_select(const BeamArgs& a, hipStream_t stream) {
  const int runs = runs_of(a.vocab);
  beam_runs_kernel<<<dim3(runs * a.searches * a.beams), kRunThreads, 0, stream>>>(a, runs);
  beam_join_kernel<<<dim3(a.searches), kJoinThreads, 0, stream>>>(a, runs);
  return hipGetLastError();
}

}  // namespace mmr
