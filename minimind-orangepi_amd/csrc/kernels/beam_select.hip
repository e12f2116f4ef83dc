// beam_select.hip -- the best continuations of the beams of many searches.
//
//   score(b, v) = s_b + x_bv - log sum_u exp x_bu,   rank = score * length^-power
//
// and of the beams x vocab candidates of a search the `beams` of the largest
// rank, ties to the lower beam, the larger x, the lower token; a beam that has
// ended is its only candidate.  Within a row the order is that of x, so of a run
// of a row's columns only the `beams` largest x can be chosen: one pass over the
// logits finds those with the run's sum of exponentials, and what is ranked, in
// 64 bits, is few.
//
// The k largest of many values: the k-th largest of the lanes' own maxima (of
// groups of lanes, where k is small) is a value that at least k values reach,
// and few others do; those are gathered in LDS, where each one's place is the
// number of better ones.  Where more reach it than there is room for (a row of
// equal logits), the block takes one maximum after another instead.
//
// Two forms, see launch_beam_select: a block a search, or a block a run of a row
// and a second kernel with a block a search.
#include "device_common.h"

#include <algorithm>
#include <cfloat>
#include <climits>

namespace mmr {

namespace {

constexpr int kRunThreads = 256, kRunWaves = kRunThreads / kWave;
constexpr int kRunQuads = 4, kRun = kRunThreads * 4 * kRunQuads;  // columns of a run
constexpr int kJoinThreads = 512, kJoinWaves = kJoinThreads / kWave;
constexpr int kJoinHeld = 4;  // candidates of its first beam that a lane holds
constexpr int kOneThreads = 1024, kOneWaves = kOneThreads / kWave;
constexpr int kOneQuads = 8, kUnit = kWave * 4 * kOneQuads;  // columns of a wave's turn
constexpr int kMostUnits = 64;                               // turns of a search
constexpr int kRoom = 512, kPlaceLanes = 8;
constexpr float kLog2e = 1.4426950408889634f;
constexpr double kLn2 = 0.6931471805599453;

// The largest x of a run, and the sum of exp(x - top); sum NaN: not all finite.
struct RunHead {
  float top, sum;
};
// Of a row's run: its head, then `beams` values and columns, in any order (column -1: none).
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
inline int units_of(int vocab) { return (vocab + kUnit - 1) / kUnit; }

// 16 bytes at any multiple of 4: where in memory a row begins must not decide
// how its sums are rounded, or equal rows would differ.
struct __attribute__((packed, aligned(4))) Quad {
  float x, y, z, w;
};
// Thread t of n holds columns first + 4 (t + n j) + i of a row as v[4 j + i].
template <int kQuads>
__device__ __forceinline__ void load_columns(const float* x, int vocab, int first, int t, int n, float* v) {
#pragma unroll
  for (int j = 0; j < kQuads; ++j) {
    const int c = first + 4 * (t + n * j);
    if (c + 4 <= vocab) {
      const Quad q = *reinterpret_cast<const Quad*>(x + c);
      v[4 * j] = q.x, v[4 * j + 1] = q.y, v[4 * j + 2] = q.z, v[4 * j + 3] = q.w;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) v[4 * j + i] = c + i < vocab ? x[c + i] : -INFINITY;
    }
  }
}

// A value that at least k values of the wave's lanes reach, of which `top` is
// each lane's largest (no number of them being less than k: the least).
__device__ __forceinline__ float wave_limit(float top, int k) {
  int above = 0;
  if (k <= kWave / 8) {  // of 16 groups of four lanes
    top = fmaxf(top, dpp_move<dpp::kQuadXor1>(top));
    top = fmaxf(top, dpp_move<dpp::kQuadXor2>(top));
#pragma unroll
    for (int i = 0; i < kWave; i += 4) above += read_lane(top, i) > top;
  } else if (k <= kWave / 4) {  // of 32 pairs
    top = fmaxf(top, dpp_move<dpp::kQuadXor1>(top));
#pragma unroll
    for (int i = 0; i < kWave; i += 2) above += read_lane(top, i) > top;
  } else {
#pragma unroll
    for (int i = 0; i < kWave; ++i) above += read_lane(top, i) > top;
  }
  return -group_max<kWave>(above < k ? -top : -INFINITY);
}

// The wave's largest value (at least the lowest finite number) and the sum of
// exp(x - that): sums of 16 terms a lane, then over the lanes.  A NaN makes the
// sum NaN, and so does +inf, from which it is subtracted.
template <int kEach>
__device__ __forceinline__ RunHead wave_head(const float* v, float top) {
  RunHead h;
  h.top = fmaxf(group_max<kWave>(top), -FLT_MAX);
  float sum[kEach / 16] = {};
#pragma unroll
  for (int i = 0; i < kEach; ++i) sum[i / 16] += __builtin_amdgcn_exp2f((v[i] - h.top) * kLog2e);
#pragma unroll
  for (int i = 1; i < kEach / 16; ++i) sum[0] += sum[i];
  h.sum = group_sum<kWave>(sum[0]);
  return h;
}

// Calls put(place, i) for the values v[i] of the wave's lanes that reach limit,
// with places of the room that *count counts; most v[i] have none, and are done
// with after one comparison.
template <int kEach, typename Put>
__device__ __forceinline__ void gather(const float* v, float limit, int* count, Put put) {
  uint64_t hits[kEach];
  int total = 0;
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    hits[i] = __ballot(v[i] >= limit);
    total += __popcll(hits[i]);
  }
  if (total == 0) return;
  int base = 0;
  if (threadIdx.x % kWave == 0) base = atomicAdd(count, total);
  base = __builtin_amdgcn_readfirstlane(base);
#pragma unroll
  for (int i = 0; i < kEach; ++i)
    if (hits[i] != 0) {
      const int place = base + __builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(hits[i] >> 32),
                                                         __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(hits[i]), 0));
      if (v[i] >= limit && place < kRoom) put(place, i);
      base += __popcll(hits[i]);
    }
}

// top + log(sum) to some 2^-25 of 1: the logarithm in 32 bits is of a number near 1.
__device__ __forceinline__ double log_sum(float top, double sum) {
  int e;
  const double m = frexp(sum * 1.3333333333333333, &e) * 1.5;  // sum = m 2^(e - 1), m in [0.75, 1.5)
  return top + kLn2 * (static_cast<double>(__builtin_amdgcn_logf(static_cast<float>(m))) + (e - 1));
}

__device__ __forceinline__ double length_factor(const BeamArgs& a, int length) {
  return a.length_power == 0.0 ? 1.0 : exp2(-a.length_power * log2(static_cast<double>(max(length, 1))));
}

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

// Candidates in LDS; what ranks them apart, so that comparing takes one read.
struct Room {
  double rank[kRoom];
  float x[kRoom];
  int beam[kRoom], token[kRoom];
  __device__ __forceinline__ Candidate get(int n) const { return Candidate{rank[n], x[n], beam[n], token[n]}; }
  // The number of better ones than candidate n, by kPlaceLanes lanes together.
  __device__ __forceinline__ int place(int n, int count) const {
    const Candidate mine = get(n);
    int above = 0;
#pragma unroll 4
    for (int j = threadIdx.x % kPlaceLanes; j < count; j += kPlaceLanes) {
      const double r = rank[j];
      above += r > mine.rank;
      if (r == mine.rank && j != n) above += better(get(j), mine);
    }
    above += dpp_move_int<dpp::kQuadXor1>(above);
    above += dpp_move_int<dpp::kQuadXor2>(above);
    return above + dpp_move_int<dpp::kRowHalfMirror>(above);
  }
};

// What the beams of a search were, and what is chosen.
struct Search {
  double lse[kMostBeams], factor[kMostBeams];
  float score[kMostBeams];
  int state[kMostBeams];  // 0 no candidates, 1 those of its row, 2 itself
  int length[kMostBeams];

  __device__ __forceinline__ double score_of(int b, float x) const {
    return state[b] == 2 ? score[b] : score[b] + (static_cast<double>(x) - lse[b]);
  }
  __device__ __forceinline__ Candidate candidate(int b, float x, int token) const {
    const double s = score_of(b, x);
    return static_cast<float>(s) > -INFINITY ? Candidate{s * factor[b], x, b, token} : no_candidate();
  }
  __device__ __forceinline__ void store(const BeamArgs& a, int first, int place, const Candidate& c) const {
    const int o = first + place;
    const bool none = c.beam == INT_MAX;
    const int token = none ? max(a.eos, 0) : c.token;
    a.scores_out[o] = none ? -INFINITY : static_cast<float>(score_of(c.beam, c.x));
    a.parent[o] = none ? -1 : first + c.beam;
    a.token[o] = token;
    a.lengths_out[o] = none ? 0 : length[c.beam];
    a.ended_out[o] = a.eos >= 0 && token == a.eos;
  }
};

// The best of the block's candidates, in every thread.
template <int kWaves>
__device__ __forceinline__ Candidate block_best(Candidate best, Candidate* wave_best) {
#pragma unroll
  for (int step = 1; step < kWave; step *= 2) {
    const Candidate other{__shfl_xor(best.rank, step), __shfl_xor(best.x, step), __shfl_xor(best.beam, step),
                          __shfl_xor(best.token, step)};
    if (better(other, best)) best = other;
  }
  __syncthreads();
  if (threadIdx.x % kWave == 0) wave_best[threadIdx.x / kWave] = best;
  __syncthreads();
  best = wave_best[0];
  for (int w = 1; w < kWaves; ++w)
    if (better(wave_best[w], best)) best = wave_best[w];
  return best;
}

// ------------------------------------------------- a block a search ----

// Waves take (beam, kUnit columns) in turn.
__global__ __launch_bounds__(kOneThreads) void beam_one_kernel(BeamArgs a, int units) {
  constexpr int kEach = 4 * kOneQuads;
  __shared__ Search search;
  __shared__ Room room;
  __shared__ RunHead heads[kMostUnits];
  __shared__ Candidate wave_best[kOneWaves];
  __shared__ int sh_count, sh_fine;
  const int first = blockIdx.x * a.beams, tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave), lane = tid % kWave;
  if (tid == 0) sh_count = sh_fine = 0;
  if (tid < a.beams) {
    const float score = a.scores[first + tid];
    const bool done = a.eos >= 0 && a.ended[first + tid] != 0;
    search.score[tid] = score;
    search.state[tid] = fabsf(score) < INFINITY ? done ? 2 : 1 : 0;
    search.length[tid] = a.lengths[first + tid] + (done ? 0 : 1);
    search.factor[tid] = length_factor(a, search.length[tid]);
    if (!(score < INFINITY)) atomicOr(a.error, kKv8NotFinite);
  }
  __syncthreads();  // the room is empty, and the beams as they were are read
  for (int u = wave; u < a.beams * units; u += kOneWaves) {
    const int b = u / units, begin = u % units * kUnit;
    if (a.eos >= 0 && search.state[b] == 2) {
      if (u % units == 0 && lane == 0) {
        const int place = atomicAdd(&sh_count, 1);
        if (place < kRoom) room.x[place] = 0.0f, room.beam[place] = b, room.token[place] = a.eos;
      }
      continue;
    }
    float v[kEach];
    load_columns<kOneQuads>(a.logits + static_cast<int64_t>(first + b) * a.vocab, a.vocab, begin, lane, kWave, v);
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < kEach; ++i) top = fmaxf(top, v[i]);
    const RunHead head = wave_head<kEach>(v, top);
    if (lane == 0) heads[u] = head;
    gather<kEach>(v, fmaxf(wave_limit(top, a.beams), -FLT_MAX), &sh_count, [&](int place, int i) {
      room.x[place] = v[i];
      room.beam[place] = b;
      room.token[place] = begin + 4 * (lane + kWave * (i / 4)) + i % 4;
    });
  }
  __syncthreads();
  const int count = sh_count;
  if (tid < a.beams && search.state[tid] != 2) {
    const RunHead* head = heads + tid * units;
    float top = -FLT_MAX;
    for (int u = 0; u < units; ++u) top = fmaxf(top, head[u].top);
    double sum = 0.0;
    for (int u = 0; u < units; ++u)
      sum += static_cast<double>(head[u].sum * __builtin_amdgcn_exp2f((head[u].top - top) * kLog2e));
    search.lse[tid] = log_sum(top, sum);
    if (!(sum > 0.0)) search.state[tid] = 0;  // not finite, or every token is masked
    if (!(sum == sum)) atomicOr(a.error, kKv8NotFinite);
  }
  __syncthreads();
  if (count <= kRoom) {
    for (int n = tid; n < count; n += kOneThreads) {
      const int b = room.beam[n];
      const Candidate c = search.state[b] == 0 ? no_candidate() : search.candidate(b, room.x[n], room.token[n]);
      room.rank[n] = c.rank;
      room.beam[n] = c.beam;
      if (c.beam != INT_MAX) atomicAdd(&sh_fine, 1);
    }
    __syncthreads();
    if (tid >= sh_fine && tid < a.beams) search.store(a, first, tid, no_candidate());
    for (int n = tid / kPlaceLanes; n < count; n += kOneThreads / kPlaceLanes) {
      const int place = room.place(n, count);
      if (tid % kPlaceLanes == 0 && place < a.beams && room.beam[n] != INT_MAX)
        search.store(a, first, place, room.get(n));
    }
    return;
  }
  Candidate last{INFINITY, INFINITY, -1, -1};
  for (int n = 0; n < a.beams; ++n) {  // each the best that is worse than the last
    Candidate best = no_candidate();
    for (int b = 0; b < a.beams; ++b) {
      const int state = search.state[b];
      if (state == 0) continue;
      const float* x = a.logits + static_cast<int64_t>(first + b) * a.vocab;
      for (int t = tid; t < (state == 2 ? 1 : a.vocab); t += kOneThreads) {
        const float value = state == 2 ? 0.0f : x[t];
        if (!(value > -INFINITY)) continue;
        const Candidate c = search.candidate(b, value, state == 2 ? a.eos : t);
        if (c.beam != INT_MAX && better(last, c) && better(c, best)) best = c;
      }
    }
    last = block_best<kOneWaves>(best, wave_best);
    if (tid == 0) search.store(a, first, n, last);
  }
}

// ------------------------------------- a block a run, then a block a search ----

__global__ __launch_bounds__(kRunThreads) void beam_runs_kernel(BeamArgs a, int runs) {
  constexpr int kEach = 4 * kRunQuads;
  __shared__ float sh_limit[kRunWaves], best_value[kRunWaves];
  __shared__ RunHead sh_head[kRunWaves];
  __shared__ int sh_count, best_column[kRunWaves];
  __shared__ float2 room[kRoom];  // value, column
  const int run = blockIdx.x % runs, row = blockIdx.x / runs, tid = threadIdx.x;
  const int wave = tid / kWave, lane = tid % kWave;
  if (a.eos >= 0 && a.ended[row] != 0) return;  // what it keeps is not used
  if (tid == 0) sh_count = 0;
  auto column_of = [&](int i) { return run * kRun + 4 * (tid + kRunThreads * (i / 4)) + i % 4; };
  float v[kEach];
  load_columns<kRunQuads>(a.logits + static_cast<int64_t>(row) * a.vocab, a.vocab, run * kRun, tid, kRunThreads, v);
  float top = -INFINITY;
#pragma unroll
  for (int i = 0; i < kEach; ++i) top = fmaxf(top, v[i]);
  const RunHead head = wave_head<kEach>(v, top);
  const float wave_at_least = wave_limit(top, a.beams);
  if (lane == 0) {
    sh_limit[wave] = wave_at_least;
    sh_head[wave] = head;
  }
  __syncthreads();
  float limit = -FLT_MAX;
#pragma unroll
  for (int w = 0; w < kRunWaves; ++w) limit = fmaxf(limit, sh_limit[w]);
  gather<kEach>(v, limit, &sh_count,
                [&](int place, int i) { room[place] = make_float2(v[i], __int_as_float(column_of(i))); });
  __syncthreads();
  const RunLayout to = run_layout(a.workspace, static_cast<int64_t>(runs) * a.searches * a.beams, a.beams);
  const int64_t at = static_cast<int64_t>(row) * runs + run;
  float* value = to.value + at * a.beams;
  int* column = to.column + at * a.beams;
  if (tid == 0) {
    float all = sh_head[0].top, s = 0.0f;
#pragma unroll
    for (int w = 1; w < kRunWaves; ++w) all = fmaxf(all, sh_head[w].top);
#pragma unroll
    for (int w = 0; w < kRunWaves; ++w) s += sh_head[w].sum * __builtin_amdgcn_exp2f((sh_head[w].top - all) * kLog2e);
    to.head[at] = RunHead{all, s};
  }
  const int count = sh_count;
  if (count <= kRoom) {
    for (int n = tid; n < max(count, a.beams); n += kRunThreads) {
      if (n >= count) {
        column[n] = -1;
        continue;
      }
      const float2 mine = room[n];
      int place = 0;
#pragma unroll 4
      for (int j = 0; j < count; ++j)
        place += argmax_better(room[j].x, __float_as_int(room[j].y), mine.x, __float_as_int(mine.y));
      if (place < a.beams) {
        value[place] = mine.x;
        column[place] = __float_as_int(mine.y);
      }
    }
    return;
  }
  for (int n = 0; n < a.beams; ++n) {
    float bv = -INFINITY;
    int bc = INT_MAX;
#pragma unroll
    for (int i = 0; i < kEach; ++i)
      if (v[i] > -INFINITY && argmax_better(v[i], column_of(i), bv, bc)) {
        bv = v[i];
        bc = column_of(i);
      }
    wave_argmax(bv, bc);
    if (lane == 0) {
      best_value[wave] = bv;
      best_column[wave] = bc;
    }
    __syncthreads();
    bv = best_value[0];
    bc = best_column[0];
#pragma unroll
    for (int w = 1; w < kRunWaves; ++w)
      if (argmax_better(best_value[w], best_column[w], bv, bc)) {
        bv = best_value[w];
        bc = best_column[w];
      }
    if (tid == 0) {
      value[n] = bv;
      column[n] = bc;
    }
#pragma unroll
    for (int i = 0; i < kEach; ++i)
      if (column_of(i) == bc) v[i] = -INFINITY;
    __syncthreads();
  }
}

// A wave a beam, in turn: its sum, then its runs' candidates.
__global__ __launch_bounds__(kJoinThreads) void beam_join_kernel(BeamArgs a, int runs) {
  __shared__ Search search;
  __shared__ Room room;
  __shared__ Candidate wave_best[kJoinWaves];
  __shared__ float sh_limit[kJoinWaves];
  __shared__ int sh_count;
  const RunLayout from = run_layout(a.workspace, static_cast<int64_t>(runs) * a.searches * a.beams, a.beams);
  const int first = blockIdx.x * a.beams, tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave), lane = tid % kWave;
  const int each = runs * a.beams;
  if (tid == 0) sh_count = 0;
  // Asked for before the sums are known; of a beam that has ended, anything.
  float held_x[kJoinHeld];
  int held_token[kJoinHeld];
#pragma unroll
  for (int i = 0; i < kJoinHeld; ++i) {
    const int n = lane + kWave * i;
    const bool there = wave < a.beams && n < each;
    const int64_t at = static_cast<int64_t>(first + wave) * each + n;
    held_x[i] = there ? from.value[at] : 0.0f;
    held_token[i] = there ? from.column[at] : -1;
  }
  // All that is read of the beams as they were is read before the barriers: the
  // new ones may take their place.
  for (int b = wave; b < a.beams; b += kJoinWaves) {
    const float score = a.scores[first + b];
    const bool done = a.eos >= 0 && a.ended[first + b] != 0;
    const int length = a.lengths[first + b] + (done ? 0 : 1);
    int state = fabsf(score) < INFINITY ? done ? 2 : 1 : 0;
    bool bad = !(score < INFINITY);
    double lse = 0.0;
    if (!done) {
      const RunHead* head = from.head + static_cast<int64_t>(first + b) * runs;
      const RunHead mine = lane < runs ? head[lane] : RunHead{-FLT_MAX, 0.0f};
      float top = mine.top;
      for (int r = lane + kWave; r < runs; r += kWave) top = fmaxf(top, head[r].top);
      top = group_max<kWave>(top);
      double sum = static_cast<double>(mine.sum * __builtin_amdgcn_exp2f((mine.top - top) * kLog2e));
      for (int r = lane + kWave; r < runs; r += kWave)
        sum += static_cast<double>(head[r].sum * __builtin_amdgcn_exp2f((head[r].top - top) * kLog2e));
#pragma unroll
      for (int step = 1; step < kWave; step *= 2) sum += __shfl_xor(sum, step);
      lse = log_sum(top, sum);
      bad = bad || !(sum == sum);
      if (!(sum > 0.0)) state = 0;  // not finite, or every token is masked
    }
    if (lane == 0) {
      if (bad) atomicOr(a.error, kKv8NotFinite);
      search.state[b] = state;
      search.score[b] = score;
      search.lse[b] = lse;
      search.length[b] = length;
      search.factor[b] = length_factor(a, length);
    }
  }
  __syncthreads();
  auto every = [&](auto use) {  // of this wave's beams
    for (int b = wave; b < a.beams; b += kJoinWaves) {
      const int state = search.state[b];
      if (state == 0) continue;
      if (state == 2) {
        if (lane == 0) use(search.candidate(b, 0.0f, a.eos));
        continue;
      }
      const int64_t at = static_cast<int64_t>(first + b) * each;
#pragma unroll
      for (int i = 0; i < kJoinHeld; ++i)
        if (kWave * i < each) {
          const int n = lane + kWave * i;
          const float x = b == wave ? held_x[i] : n < each ? from.value[at + n] : 0.0f;
          const int token = b == wave ? held_token[i] : n < each ? from.column[at + n] : -1;
          if (token >= 0) use(search.candidate(b, x, token));
        }
      for (int n = lane + kWave * kJoinHeld; n < each; n += kWave) {
        const int token = from.column[at + n];
        if (token >= 0) use(search.candidate(b, from.value[at + n], token));
      }
    }
  };
  // Ranks in 32 bits are in the order of those in 64, or equal: what reaches the
  // limit in 32 bits is all that may be among the best.
  float limit = -INFINITY;
  if (a.beams * each > kWave) {
    float top = -INFINITY;
    every([&](const Candidate& c) { top = fmaxf(top, static_cast<float>(c.rank)); });
    const float at_least = wave_limit(top, a.beams);
    if (lane == 0) sh_limit[wave] = at_least;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kJoinWaves; ++w) limit = fmaxf(limit, sh_limit[w]);
  }
  every([&](const Candidate& c) {
    if (c.beam != INT_MAX && static_cast<float>(c.rank) >= limit) {
      const int place = atomicAdd(&sh_count, 1);
      if (place < kRoom) {
        room.rank[place] = c.rank;
        room.x[place] = c.x;
        room.beam[place] = c.beam;
        room.token[place] = c.token;
      }
    }
  });
  __syncthreads();
  const int count = sh_count;
  if (count <= kRoom) {
    if (tid >= count && tid < a.beams) search.store(a, first, tid, no_candidate());
    for (int n = tid / kPlaceLanes; n < count; n += kJoinThreads / kPlaceLanes) {
      const int place = room.place(n, count);
      if (tid % kPlaceLanes == 0 && place < a.beams) search.store(a, first, place, room.get(n));
    }
    return;
  }
  Candidate last{INFINITY, INFINITY, -1, -1};
  for (int n = 0; n < a.beams; ++n) {  // each the best that is worse than the last
    Candidate best = no_candidate();
    every([&](const Candidate& c) {
      if (c.beam != INT_MAX && better(last, c) && better(c, best)) best = c;
    });
    last = block_best<kJoinWaves>(best, wave_best);
    if (tid == 0) search.store(a, first, n, last);
  }
}

}  // namespace

int64_t beam_select_workspace(int searches, int beams, int vocab) {
  if (beams * units_of(vocab) <= kMostUnits) return 0;
  const int64_t runs = static_cast<int64_t>(runs_of(vocab)) * searches * beams;
  return runs * static_cast<int64_t>(sizeof(RunHead) + beams * (sizeof(float) + sizeof(int)));
}

hipError_t launch_beam_select(const BeamArgs& a, hipStream_t stream) {
  const int runs = runs_of(a.vocab), units = units_of(a.vocab);
  if (beam_select_workspace(a.searches, a.beams, a.vocab) == 0) {
    beam_one_kernel<<<dim3(a.searches), kOneThreads, 0, stream>>>(a, units);
  } else {
    beam_runs_kernel<<<dim3(runs * a.searches * a.beams), kRunThreads, 0, stream>>>(a, runs);
    beam_join_kernel<<<dim3(a.searches), kJoinThreads, 0, stream>>>(a, runs);
  }
  return hipGetLastError();
}

}  // namespace mmr
