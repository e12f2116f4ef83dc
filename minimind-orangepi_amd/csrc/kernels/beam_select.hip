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
// The k largest of many values: of the maxima of at least 2 k groups of them the
// k-th largest is a limit that at least k values reach, and few others do; those
// are gathered in LDS, where each one's place is the number of better ones.
// Where more reach it than there is room for, the block takes one maximum after
// another instead: a row of equal logits, or of a finite lowest value as a mask that
// leaves fewer tokens than beams (one search of 4 beams of 6,400 logits with one left
// 81, masked by -inf 7.6; 16 of 8 beams of 100,003 with 100 left 53 and 18.5).
//
// Two forms, see launch_beam_select: a block a search, or a block a run of a row
// and a second kernel with a block a search.
//
// Times in this file are us a call in replayed graphs (medians of graphs of 30
// calls over three sets of inputs; a kernel that does nothing takes 1.6 there).
#include "device_common.h"

#include <algorithm>
#include <cfloat>
#include <climits>
#include <type_traits>

namespace mmr {

namespace {

constexpr int kRunThreads = 256, kRunWaves = kRunThreads / kWave;
constexpr int kRunQuads = 4, kRun = kRunThreads * 4 * kRunQuads;  // columns of a run
constexpr int kJoinThreads = 512, kJoinWaves = kJoinThreads / kWave;
constexpr int kJoinHeld = 8;  // candidates of its first beam that a lane holds
constexpr int kOneThreads = 1024, kOneWaves = kOneThreads / kWave;
constexpr int kOneQuads = 8, kUnit = kWave * 4 * kOneQuads;  // columns of one of its waves
constexpr int kRoom = 512, kFours = 512, kPlaceLanes = 8;
constexpr int kFewCandidates = 64;  // that are all placed
static_assert(kRoom <= kJoinThreads && kRoom <= kOneThreads, "a candidate a thread");
constexpr float kLog2e = 1.4426950408889634f;
constexpr double kLn2 = 0.6931471805599453;

// The largest x of a run, the sum of exp(x - top) (NaN: not all finite) and what
// its kept values reach.
struct __attribute__((aligned(16))) RunHead {
  float top, sum, limit;
};
// Of a row's run: its head, then values and columns that are, or may be, among
// its `beams` largest, in any order (column -1: none).
struct RunLayout {
  RunHead* head;
  float2* kept;
};
__host__ __device__ inline int kept_of(int beams) { return 2 * beams; }
__host__ __device__ inline RunLayout run_layout(void* workspace, int64_t runs) {
  RunLayout l;
  l.head = static_cast<RunHead*>(workspace);
  l.kept = reinterpret_cast<float2*>(l.head + runs);
  return l;
}
inline int runs_of(int vocab) { return (vocab + kRun - 1) / kRun; }
inline int units_of(int vocab) { return (vocab + kUnit - 1) / kUnit; }

// 16 bytes at any multiple of 4: where in memory a row begins must not decide
// how its sums are rounded, or equal rows would differ.
struct __attribute__((packed, aligned(4))) Quad {
  float x, y, z, w;
};
// Thread t of n holds columns first + 4 (t + n j) + i of a row as v[4 j + i]; a
// branch for all threads, so that no load waits for another.
template <int kQuads>
__device__ __forceinline__ void load_columns(const float* x, int vocab, int first, int t, int n, float* v) {
  if (first + 4 * kQuads * n <= vocab) {
#pragma unroll
    for (int j = 0; j < kQuads; ++j) {
      const Quad q = *reinterpret_cast<const Quad*>(x + first + 4 * (t + n * j));
      v[4 * j] = q.x, v[4 * j + 1] = q.y, v[4 * j + 2] = q.z, v[4 * j + 3] = q.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4 * kQuads; ++i) v[i] = x[min(first + 4 * (t + n * (i / 4)) + i % 4, vocab - 1)];
#pragma unroll
    for (int i = 0; i < 4 * kQuads; ++i)
      if (first + 4 * (t + n * (i / 4)) + i % 4 >= vocab) v[i] = -INFINITY;
  }
}

// How many of these lanes come before this one.
__device__ __forceinline__ int lanes_before(uint64_t lanes) {
  return __builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(lanes >> 32),
                                   __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(lanes), 0));
}

// The k-th largest of the first n lanes' values, k <= n, where the other lanes
// have some of those.
__device__ __forceinline__ float wave_kth(float v, int n, int k) {
  int above = 0;
  if (n == kWave) {
#pragma unroll
    for (int i = 0; i < kWave; ++i) above += read_lane(v, i) > v;
  } else {
    for (int i = 0; i < n; i += 4) {  // n is a multiple of 4
#pragma unroll
      for (int m = 0; m < 4; ++m) above += read_lane(v, i + m) > v;
    }
  }
  return -group_max<kWave>(above < k ? -v : -INFINITY);
}
// As few groups of lanes as k allows: of 16, 2 k groups or more.
__device__ __forceinline__ float wave_kth_of_groups(float v, int k) {
  if (k > kWave / 8) return wave_kth(v, kWave, k);
  v = fmaxf(v, dpp_move<dpp::kQuadXor1>(v));
  v = fmaxf(v, dpp_move<dpp::kQuadXor2>(v));
  int above = 0;
#pragma unroll
  for (int i = 0; i < kWave; i += 4) above += read_lane(v, i) > v;
  return -group_max<kWave>(above < k ? -v : -INFINITY);
}
// The largest of each 64 / n neighbouring lanes, n being 4, 16 or 64.
__device__ __forceinline__ float lane_groups_max(float v, int n) {
  if (n < 64) {
    v = fmaxf(v, dpp_move<dpp::kQuadXor1>(v));
    v = fmaxf(v, dpp_move<dpp::kQuadXor2>(v));
  }
  if (n < 16) {
    v = fmaxf(v, dpp_move<dpp::kRowHalfMirror>(v));
    v = fmaxf(v, dpp_move<dpp::kRowMirror>(v));
  }
  return v;
}

// The wave's sum of exp(x - top), top being no less than any x: sums of 16 terms
// a lane, then over the lanes.  A NaN makes it NaN, and so does +inf, from which
// it is subtracted.
template <int kEach>
__device__ __forceinline__ float wave_sum(const float* v, float top) {
  float sum[kEach / 16] = {};
#pragma unroll
  for (int i = 0; i < kEach; ++i) sum[i / 16] += __builtin_amdgcn_exp2f((v[i] - top) * kLog2e);
#pragma unroll
  for (int i = 1; i < kEach / 16; ++i) sum[0] += sum[i];
  return group_sum<kWave>(sum[0]);
}

// Fours of values in LDS, and what the first of them is the value of.
struct Fours {
  float4 x[kFours];
  int code[kFours], count;
};
// Of the lanes' fours (of which most[j] is the largest), those that reach limit;
// most do not, and are done with after one comparison.
template <int kQuads, typename Code>
__device__ __forceinline__ void gather(const float* v, const float* most, float limit, Fours* to, Code code) {
  uint64_t hits[kQuads];
  int total = 0;
#pragma unroll
  for (int j = 0; j < kQuads; ++j) {
    hits[j] = __ballot(most[j] >= limit);
    total += __popcll(hits[j]);
  }
  if (total == 0) return;
  int base = 0;
  if (threadIdx.x % kWave == 0) base = atomicAdd(&to->count, total);
  base = __builtin_amdgcn_readfirstlane(base);
#pragma unroll
  for (int j = 0; j < kQuads; ++j)
    if (hits[j] != 0) {
      const int place = base + lanes_before(hits[j]);
      if (most[j] >= limit && place < kFours) {
        to->x[place] = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
        to->code[place] = code(j);
      }
      base += __popcll(hits[j]);
    }
}
template <int kQuads>
__device__ __forceinline__ float largest(const float* v, float* most) {
  float top = -INFINITY;
#pragma unroll
  for (int j = 0; j < kQuads; ++j) {
    most[j] = fmaxf(fmaxf(v[4 * j], v[4 * j + 1]), fmaxf(v[4 * j + 2], v[4 * j + 3]));
    top = fmaxf(top, most[j]);
  }
  return top;
}

// top + log(sum) in 64 bits: it moves all of a beam's scores against the others'.
// With sum = m 2^e, m in [1 / sqrt(2), sqrt(2)), and z = (m - 1) / (m + 1), log m is
// 2 (z + z^3 / 3 + z^5 / 5 + ...); |z| < 0.1716, and the terms from z^21 on are below
// 2^-54 of the sum.  (With a 32-bit logarithm, off by some 2^-24, one search takes 7.7,
// not 7.9, and beams closer than that change places.)
__device__ __forceinline__ double log_sum(float top, double sum) {
  int e;
  double m = frexp(sum, &e);
  if (m < 0.70710678118654752) m += m, --e;
  // 1 / (m + 1) from 32 bits, in two steps.
  const double n = m + 1.0;
  double r = static_cast<double>(__builtin_amdgcn_rcpf(static_cast<float>(n)));
  r = fma(fma(-n, r, 1.0), r, r);
  r = fma(fma(-n, r, 1.0), r, r);
  const double z = (m - 1.0) * r, zz = z * z;
  double series = 1.0 / 19.0;
#pragma unroll
  for (int k = 17; k >= 3; k -= 2) series = fma(series, zz, 1.0 / k);
  return top + fma(kLn2, static_cast<double>(e), 2.0 * fma(series * zz, z, z));
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
  // To be ranked:
  float x[kRoom];
  int code[kRoom];  // beam * 2^24 + token
  int count;
  // Ranked:
  double rank[kRoom];
  float ranked_x[kRoom], score[kRoom];
  int ranked_code[kRoom], ranked;
  float limit[kOneWaves];
  __device__ __forceinline__ Candidate get(int n) const {
    return Candidate{rank[n], ranked_x[n], ranked_code[n] >> 24, ranked_code[n] & 0xFFFFFF};
  }
  // Adds of kEach values of each lane those that are wanted, at once: an atomic
  // takes as long for one as for many.
  template <int kEach>
  __device__ __forceinline__ void add(const bool* wanted, const float* value, const int* c) {
    uint64_t lanes[kEach];
    int total = 0;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      lanes[i] = __ballot(wanted[i]);
      total += __popcll(lanes[i]);
    }
    if (total == 0) return;
    int base = 0;
    if (threadIdx.x % kWave == 0) base = atomicAdd(&count, total);
    base = __builtin_amdgcn_readfirstlane(base);
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int place = base + lanes_before(lanes[i]);
      if (wanted[i] && place < kRoom) {
        x[place] = value[i];
        code[place] = c[i];
      }
      base += __popcll(lanes[i]);
    }
  }
  __device__ __forceinline__ void add(bool wanted, float value, int c) { add<1>(&wanted, &value, &c); }
  // Adds the lanes' candidates, where they are some.
  __device__ __forceinline__ void add_ranked(const Candidate& c, float s) {
    const bool wanted = c.beam != INT_MAX;
    const uint64_t lanes = __ballot(wanted);
    if (lanes == 0) return;
    int base = 0;
    if (threadIdx.x % kWave == 0) base = atomicAdd(&ranked, __popcll(lanes));
    const int n = __builtin_amdgcn_readfirstlane(base) + lanes_before(lanes);
    if (wanted && n < kRoom) {
      rank[n] = c.rank;
      score[n] = s;
      ranked_x[n] = c.x;
      ranked_code[n] = c.beam << 24 | c.token;
    }
  }
  // The number of better ones than candidate n, by kPlaceLanes lanes together.
  __device__ __forceinline__ int place(int n, int all) const {
    const double mine = rank[n];
    int above = 0;
#pragma unroll 4
    for (int j = threadIdx.x % kPlaceLanes; j < all; j += kPlaceLanes) {
      const double r = rank[j];
      above += r > mine;
      if (r == mine && j != n) above += better(get(j), get(n));
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
  int state[kMostBeams];  // 0 no candidates, 1 those of its row, 2 itself, 3 ended without a score
  int length[kMostBeams];

  // Of beam n, as it was: read before the new ones take its place.
  struct Before {
    float score;
    int ended, length;
  };
  __device__ __forceinline__ static Before before(const BeamArgs& a, int row) {
    return Before{a.scores[row], a.eos >= 0 ? a.ended[row] : 0, a.lengths[row]};
  }
  __device__ __forceinline__ void set(const BeamArgs& a, int n, const Before& was) {
    const bool done = was.ended != 0;
    score[n] = was.score;
    state[n] = fabsf(was.score) < INFINITY ? done ? 2 : 1 : done ? 3 : 0;
    length[n] = was.length + (done ? 0 : 1);
    if (!(was.score < INFINITY)) atomicOr(a.error, kKv8NotFinite);
  }
  // Of the sum of exp(x - top) over its row.
  __device__ __forceinline__ void set_sum(const BeamArgs& a, int n, float top, double sum) {
    lse[n] = log_sum(top, sum);
    if (!(sum > 0.0)) state[n] = 0;  // not finite, or every token is masked
    if (!(sum == sum)) atomicOr(a.error, kKv8NotFinite);
  }
  __device__ __forceinline__ Candidate candidate(int b, float x, int token, float* score_out) const {
    const double s = state[b] == 2 ? score[b] : score[b] + (static_cast<double>(x) - lse[b]);
    *score_out = static_cast<float>(s);
    return (state[b] == 1 || state[b] == 2) && *score_out > -INFINITY ? Candidate{s * factor[b], x, b, token}
                                                                      : no_candidate();
  }
  __device__ __forceinline__ void store(const BeamArgs& a, int first, int place, const Candidate& c, float s) const {
    const int o = first + place;
    const bool none = c.beam == INT_MAX;
    const int token = none ? max(a.eos, 0) : c.token;
    a.scores_out[o] = none ? -INFINITY : s;
    a.parent[o] = none ? -1 : first + c.beam;
    a.token[o] = token;
    a.lengths_out[o] = none ? 0 : length[c.beam];
    a.ended_out[o] = a.eos >= 0 && token == a.eos;
  }
  __device__ __forceinline__ void store(const BeamArgs& a, int first, int place, const Candidate& c) const {
    float s = 0.0f;
    if (c.beam != INT_MAX) candidate(c.beam, c.x, c.token, &s);
    store(a, first, place, c, s);
  }
  // Stores the best of the room's ranked candidates.
  template <int kThreads>
  __device__ __forceinline__ void place_and_store(const BeamArgs& a, int first, const Room* room) const {
    const int tid = threadIdx.x, count = room->ranked;
    if (tid >= count && tid < a.beams) store(a, first, tid, no_candidate());
    for (int n = tid / kPlaceLanes; n < count; n += kThreads / kPlaceLanes) {
      const int place = room->place(n, count);
      if (tid % kPlaceLanes == 0 && place < a.beams) store(a, first, place, room->get(n), room->score[n]);
    }
  }
};

// Of `count` ranks, a thread each, a limit that the best reach: 32 bits are in
// the order of 64, or equal, so that what reaches it in 32 is all that may be
// among them.  The block finds it together.
__device__ __forceinline__ float rank_limit(float rank, int count, int beams, float* limits) {
  const int wave = threadIdx.x / kWave;
  if (wave * kWave < count) {
    const float at_least = wave_kth_of_groups(rank, beams);
    if (threadIdx.x % kWave == 0) limits[wave] = at_least;
  }
  __syncthreads();
  float limit = -INFINITY;
  for (int w = 0; w * kWave < count; ++w) limit = fmaxf(limit, limits[w]);
  return limit;
}

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

// A wave takes kUnit columns of a beam: the sum first, and the maxima of groups
// of lanes; those of a beam's waves give its limit, with which they gather.
// One search of 4 beams of 6,400 logits 7.9, of which the exponentials of four
// waves a SIMD are 1.1, the memory 1.2, and the chain limit - gather - rank -
// place, with a barrier between each two, most of the rest.
__global__ __launch_bounds__(kOneThreads) void beam_one_kernel(BeamArgs a, int units, int groups) {
  constexpr int kOthers = kOneThreads - kWave;
  __shared__ Search search;
  __shared__ Room room;
  __shared__ Fours fours;
  __shared__ RunHead heads[kOneWaves];
  __shared__ float maxima[kOneWaves * kWave];
  __shared__ Candidate wave_best[kOneWaves];
  const int first = blockIdx.x * a.beams, tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave), lane = tid % kWave;
  const int b = wave / units, unit = wave - b * units;
  const bool works = b < a.beams;
  float v[4 * kOneQuads], most[kOneQuads];
  if (works)  // also of a beam that has ended, whose logits then count for nothing
    load_columns<kOneQuads>(a.logits + static_cast<int64_t>(first + b) * a.vocab, a.vocab, unit * kUnit, lane, kWave,
                            v);
  const bool has_beam = tid >= kOthers && tid - kOthers < a.beams;
  Search::Before was = {};
  if (has_beam) was = Search::before(a, first + tid - kOthers);
  if (tid == 0) fours.count = room.ranked = 0;
  if (works) {
    const float top = largest<kOneQuads>(v, most);
    const float wave_top = fmaxf(group_max<kWave>(top), -FLT_MAX), group_top = lane_groups_max(top, groups);
    const float sum = wave_sum<4 * kOneQuads>(v, wave_top);
    if (lane == 0) heads[wave] = RunHead{wave_top, sum, 0.0f};
    if (lane % (kWave / groups) == 0) maxima[wave * groups + lane / (kWave / groups)] = group_top;
  }
  if (has_beam) search.set(a, tid - kOthers, was);
  __syncthreads();
  // Of a beam's waves, the first has its sum to do, so another has this.
  if (works && unit == min(1, units - 1) && lane == 0) search.factor[b] = length_factor(a, search.length[b]);
  if (works && search.state[b] < 2) {
    const int all = units * groups;  // at most a wave's lanes, see one_groups
    const float limit = fmaxf(wave_kth(maxima[b * all + min(lane, all - 1)], all, a.beams), -FLT_MAX);
    if (search.state[b] == 1)  // or 0 by now, where the row turns out to have no candidates
      gather<kOneQuads>(v, most, limit, &fours,
                        [&](int j) { return b << 24 | (unit * kUnit + 4 * (lane + kWave * j)); });
    if (unit == 0) {
      const RunHead head = lane < units ? heads[wave + lane] : RunHead{-FLT_MAX, 0.0f, 0.0f};
      const float row_top = group_max<kWave>(head.top);
      double sum = static_cast<double>(head.sum * __builtin_amdgcn_exp2f((head.top - row_top) * kLog2e));
#pragma unroll
      for (int step = 1; step < kOneWaves; step *= 2)
        if (step < units) sum += __shfl_xor(sum, step);
      if (lane == 0) {
        heads[wave].limit = limit;
        search.set_sum(a, b, row_top, sum);
      }
    }
  }
  __syncthreads();
  if (fours.count <= kFours) {
    const int values = 4 * fours.count;
    for (int base = wave * kWave; base < values; base += kOneThreads) {  // a value a lane
      const int at = min(base + lane, values - 1), code = fours.code[at / 4];
      const float x = reinterpret_cast<const float*>(fours.x)[at];
      float score = 0.0f;
      Candidate c = no_candidate();
      if (base + lane < values && x >= heads[(code >> 24) * units].limit)
        c = search.candidate(code >> 24, x, (code & 0xFFFFFF) + at % 4, &score);
      room.add_ranked(c, score);
    }
    if (tid >= kOthers) {
      float score = 0.0f;
      Candidate c = no_candidate();
      if (has_beam && search.state[tid - kOthers] == 2) c = search.candidate(tid - kOthers, 0.0f, a.eos, &score);
      room.add_ranked(c, score);
    }
    __syncthreads();
    const int count = room.ranked;
    if (count <= kRoom) {
      if (count > kFewCandidates) {  // only those that reach a limit
        Candidate c = no_candidate();
        float score = 0.0f;
        if (tid < count) c = room.get(tid), score = room.score[tid];
        const float limit = rank_limit(static_cast<float>(c.rank), count, a.beams, room.limit);
        if (static_cast<float>(c.rank) < limit) c = no_candidate();
        if (tid == 0) room.ranked = 0;
        __syncthreads();
        room.add_ranked(c, score);
        __syncthreads();
      }
      search.place_and_store<kOneThreads>(a, first, &room);
      return;
    }
  }
  Candidate last{INFINITY, INFINITY, -1, -1};
  for (int n = 0; n < a.beams; ++n) {  // each the best that is worse than the last
    Candidate best = no_candidate();
    for (int b = 0; b < a.beams; ++b) {
      const int state = search.state[b];
      if (state != 1 && state != 2) continue;
      const float* x = a.logits + static_cast<int64_t>(first + b) * a.vocab;
      for (int t = tid; t < (state == 2 ? 1 : a.vocab); t += kOneThreads) {
        const float value = state == 2 ? 0.0f : x[t];
        if (!(value > -INFINITY)) continue;
        float s;
        const Candidate c = search.candidate(b, value, state == 2 ? a.eos : t, &s);
        if (c.beam != INT_MAX && better(last, c) && better(c, best)) best = c;
      }
    }
    last = block_best<kOneWaves>(best, wave_best);
    if (tid == 0) search.store(a, first, n, last);
  }
}

// ------------------------------------- a block a run, then a block a search ----

// Of 128 rows of 100,003 logits (51 MB) this kernel takes 12.5 of 20.0: 4.1 TB/s.
// Vector instructions bound it, which is why the limit is of 16 groups of a
// block's lanes where that is enough, sums are against the block's maximum, and
// values are kept as they come (they took 38 with a limit of each thread's
// maximum, sums and a place for each value).
__global__ __launch_bounds__(kRunThreads) void beam_runs_kernel(BeamArgs a, int runs) {
  constexpr int kEach = 4 * kRunQuads;
  __shared__ float maxima[kWave], sh_sum[kRunWaves], best_value[kRunWaves];
  __shared__ int best_column[kRunWaves];
  __shared__ float2 room[kRoom];
  __shared__ int sh_count;
  const int run = blockIdx.x % runs, row = blockIdx.x / runs, tid = threadIdx.x;
  const int wave = tid / kWave, lane = tid % kWave;
  if (a.eos >= 0 && a.ended[row] != 0) return;  // what it keeps is not used
  if (tid == 0) sh_count = 0;
  auto column_of = [&](int i) { return run * kRun + 4 * (tid + kRunThreads * (i / 4)) + i % 4; };
  float v[kEach];
  load_columns<kRunQuads>(a.logits + static_cast<int64_t>(row) * a.vocab, a.vocab, run * kRun, tid, kRunThreads, v);
  // 16 groups of a block's lanes, or 64.
  const int groups = a.beams <= 8 ? 4 : 16, all = groups * kRunWaves;
  float top = v[0];
#pragma unroll
  for (int i = 1; i < kEach; ++i) top = fmaxf(top, v[i]);
  const float group_top = lane_groups_max(top, groups);
  if (lane % (kWave / groups) == 0) maxima[wave * groups + lane / (kWave / groups)] = group_top;
  __syncthreads();
  const float group = maxima[lane % all];
  const float limit = fmaxf(wave_kth(group, all, a.beams), -FLT_MAX);
  const float block_top = fmaxf(group_max<kWave>(group), -FLT_MAX);
  const float sum = wave_sum<kEach>(v, block_top);
  if (lane == 0) sh_sum[wave] = sum;
  uint64_t hits[kEach];
  int total = 0;
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    hits[i] = __ballot(v[i] >= limit);
    total += __popcll(hits[i]);
  }
  if (total > 0) {
    int base = 0;
    if (lane == 0) base = atomicAdd(&sh_count, total);
    base = __builtin_amdgcn_readfirstlane(base);
#pragma unroll
    for (int i = 0; i < kEach; ++i)
      if (hits[i] != 0) {
        const int place = base + lanes_before(hits[i]);
        if (v[i] >= limit && place < kRoom) room[place] = make_float2(v[i], __int_as_float(column_of(i)));
        base += __popcll(hits[i]);
      }
  }
  __syncthreads();
  const RunLayout to = run_layout(a.workspace, static_cast<int64_t>(runs) * a.searches * a.beams);
  const int64_t at = static_cast<int64_t>(row) * runs + run;
  const int keep = kept_of(a.beams), count = sh_count;
  float2* kept = to.kept + at * keep;
  if (tid == 0) {
    float s = sh_sum[0];
#pragma unroll
    for (int w = 1; w < kRunWaves; ++w) s += sh_sum[w];
    to.head[at] = RunHead{block_top, s, limit};
  }
  const float2 none = make_float2(0.0f, __int_as_float(-1));
  if (count <= keep) {
    if (tid < keep) kept[tid] = tid < count ? room[tid] : none;
    return;
  }
  if (tid >= a.beams && tid < keep) kept[tid] = none;
  if (count <= kRoom) {
    for (int n = tid; n < count; n += kRunThreads) {
      const float2 mine = room[n];
      int place = 0;
#pragma unroll 4
      for (int j = 0; j < count; ++j)
        place += argmax_better(room[j].x, __float_as_int(room[j].y), mine.x, __float_as_int(mine.y));
      if (place < a.beams) kept[place] = mine;
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
    if (tid == 0) kept[n] = make_float2(bv, __int_as_float(bc));
#pragma unroll
    for (int i = 0; i < kEach; ++i)
      if (column_of(i) == bc) v[i] = -INFINITY;
    __syncthreads();
  }
}

// A wave a beam, in turn: its sum, then its runs' candidates.  Latency: of about 7
// the loads are 2 (heads, kept values and the beams at once), the rest barriers.
__global__ __launch_bounds__(kJoinThreads) void beam_join_kernel(BeamArgs a, int runs) {
  __shared__ Search search;
  __shared__ Room room;
  __shared__ Candidate wave_best[kJoinWaves];
  __shared__ float sh_limit[kJoinWaves], row_limit[kMostBeams];
  const RunLayout from = run_layout(a.workspace, static_cast<int64_t>(runs) * a.searches * a.beams);
  const int first = blockIdx.x * a.beams, tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave), lane = tid % kWave;
  const int each = runs * kept_of(a.beams);
  const bool has_beam = tid < a.beams;
  Search::Before was = {};
  if (has_beam) was = Search::before(a, first + tid);
  // Asked for before the sums are known; of a beam that has ended, anything.
  float2 held[kJoinHeld] = {};
  auto ask = [&](int b) {
    const float2* kept = from.kept + static_cast<int64_t>(first + b) * each;
#pragma unroll
    for (int i = 0; i < kJoinHeld; ++i)
      if (kWave * i < each) held[i] = kept[min(lane + kWave * i, each - 1)];
  };
  if (wave < a.beams) ask(wave);
  auto head_of = [&](int b) {
    return lane < runs ? from.head[static_cast<int64_t>(first + b) * runs + lane] : RunHead{-FLT_MAX, 0.0f, -FLT_MAX};
  };
  RunHead head = wave < a.beams ? head_of(wave) : RunHead{};
  if (tid == 0) room.count = room.ranked = 0;
  if (has_beam) {
    search.set(a, tid, was);
    search.factor[tid] = length_factor(a, search.length[tid]);
  }
  __syncthreads();
  for (int b = wave; b < a.beams; b += kJoinWaves) {
    if (search.state[b] >= 2) continue;
    if (b != wave) head = head_of(b);
    const RunHead* more = from.head + static_cast<int64_t>(first + b) * runs;
    float top = head.top, limit = head.limit;
    for (int r = lane + kWave; r < runs; r += kWave) {
      top = fmaxf(top, more[r].top);
      limit = fmaxf(limit, more[r].limit);
    }
    // What `beams` values of a run reach, or as many runs.
    limit = fmaxf(group_max<kWave>(limit),
                  wave_kth(lane < runs ? top : -INFINITY, min(kWave, (runs + 3) / 4 * 4), a.beams));
    top = group_max<kWave>(top);
    double sum = static_cast<double>(head.sum * __builtin_amdgcn_exp2f((head.top - top) * kLog2e));
    for (int r = lane + kWave; r < runs; r += kWave)
      sum += static_cast<double>(more[r].sum * __builtin_amdgcn_exp2f((more[r].top - top) * kLog2e));
#pragma unroll
    for (int step = 1; step < kWave; step *= 2) sum += __shfl_xor(sum, step);
    if (lane == 0) {
      row_limit[b] = limit;
      search.set_sum(a, b, top, sum);
    }
  }
  __syncthreads();
  // Of this wave's beams, all lanes together: use<n>(whether there is one, x, code), n of each.
  auto every = [&](auto use) {
    for (int b = wave; b < a.beams; b += kJoinWaves) {
      const int state = search.state[b];
      bool is[kJoinHeld];
      float x[kJoinHeld];
      int code[kJoinHeld];
      if (state == 2) {
        is[0] = lane == 0, x[0] = 0.0f, code[0] = b << 24 | a.eos;
        use(std::integral_constant<int, 1>(), is, x, code);
      }
      if (state != 1) continue;
      const float limit = row_limit[b];  // what `beams` values of the row reach
      if (a.beams > kJoinWaves) ask(b);
      auto one = [&](int i, const float2& k, bool there) {
        const int token = __float_as_int(k.y);
        is[i] = there && token >= 0 && k.x >= limit;
        x[i] = k.x;
        code[i] = b << 24 | token;
      };
      one(0, held[0], lane < each);
      if (each <= kWave) {
        use(std::integral_constant<int, 1>(), is, x, code);
        continue;
      }
#pragma unroll
      for (int i = 1; i < kJoinHeld; ++i) one(i, held[i], lane + kWave * i < each);
      use(std::integral_constant<int, kJoinHeld>(), is, x, code);
      const float2* kept = from.kept + static_cast<int64_t>(first + b) * each;
      for (int n = lane + kWave * kJoinHeld; n - lane < each; n += kWave) {
        one(0, kept[min(n, each - 1)], n < each);
        use(std::integral_constant<int, 1>(), is, x, code);
      }
    }
  };
  auto candidate = [&](float x, int code) {
    float score;
    return search.candidate(code >> 24, x, code & 0xFFFFFF, &score);
  };
  every([&](auto n, const bool* is, const float* x, const int* code) { room.add<decltype(n)::value>(is, x, code); });
  __syncthreads();
  if (room.count > kRoom) {
    // Of many beams.  Ranks in 32 bits are in the order of those in 64, or equal:
    // what reaches a limit in 32 bits is all that may be among the best.
    float top = -INFINITY;
    every([&](auto n, const bool* is, const float* x, const int* code) {
      for (int i = 0; i < decltype(n)::value; ++i)
        if (is[i]) top = fmaxf(top, static_cast<float>(candidate(x[i], code[i]).rank));
    });
    const float at_least = wave_kth(top, kWave, a.beams);
    if (lane == 0) sh_limit[wave] = at_least;
    __syncthreads();
    if (tid == 0) room.count = 0;
    float limit = -INFINITY;
#pragma unroll
    for (int w = 0; w < kJoinWaves; ++w) limit = fmaxf(limit, sh_limit[w]);
    __syncthreads();
    every([&](auto n, const bool* is, const float* x, const int* code) {
      for (int i = 0; i < decltype(n)::value; ++i)
        room.add(is[i] && static_cast<float>(candidate(x[i], code[i]).rank) >= limit, x[i], code[i]);
    });
    __syncthreads();
  }
  if (room.count <= kRoom) {
    float score = 0.0f;
    Candidate c = no_candidate();
    if (tid < room.count) {
      const int code = room.code[tid];
      c = search.candidate(code >> 24, room.x[tid], code & 0xFFFFFF, &score);
    }
    if (room.count > kFewCandidates &&
        static_cast<float>(c.rank) < rank_limit(static_cast<float>(c.rank), room.count, a.beams, room.limit))
      c = no_candidate();
    room.add_ranked(c, score);
    __syncthreads();
    search.place_and_store<kJoinThreads>(a, first, &room);
    return;
  }
  Candidate last{INFINITY, INFINITY, -1, -1};
  for (int n = 0; n < a.beams; ++n) {  // each the best that is worse than the last
    Candidate best = no_candidate();
    every([&](auto n, const bool* is, const float* x, const int* code) {
      for (int i = 0; i < decltype(n)::value; ++i) {
        if (!is[i]) continue;
        const Candidate c = candidate(x[i], code[i]);
        if (c.beam != INT_MAX && better(last, c) && better(c, best)) best = c;
      }
    });
    last = block_best<kJoinWaves>(best, wave_best);
    if (tid == 0) search.store(a, first, n, last);
  }
}

}  // namespace

// Of a wave's lanes, so that a beam has at least 2 k groups; and at most 64, as
// beams x units is at most 16: 4 each of up to 16 waves, 16 where units < beams / 2
// (of up to 2), 64 where units < beams / 8 (of one).
static int one_groups(int units, int beams) {
  return units * 4 >= 2 * beams ? 4 : units * 16 >= 2 * beams ? 16 : 64;
}

// A block a run of every row, and fewer than 2^32 threads in a launch.
bool beam_select_in_range(int64_t rows, int64_t vocab) {
  return rows * ((vocab + kRun - 1) / kRun) * kRunThreads < int64_t{1} << 32;
}

int64_t beam_select_workspace(int searches, int beams, int vocab) {
  if (beams * units_of(vocab) <= kOneWaves) return 0;
  const int64_t runs = static_cast<int64_t>(runs_of(vocab)) * searches * beams;
  return runs * static_cast<int64_t>(sizeof(RunHead) + kept_of(beams) * sizeof(float2));
}

// One block a search as long as a wave has one turn: 32 searches of 4 beams of
// 6,400 logits 8.4 and, in two kernels, 9.3, 128 searches 9.3 and 11.8, one search
// 7.9 and 8.4.  With two turns or more two kernels are faster (8 beams 10.1,
// in one block 15.9; 4 beams of 32,000 logits 8.7 and 22.9).
hipError_t launch_beam_select(const BeamArgs& a, hipStream_t stream) {
  const int runs = runs_of(a.vocab), units = units_of(a.vocab);
  if (beam_select_workspace(a.searches, a.beams, a.vocab) == 0) {
    beam_one_kernel<<<dim3(a.searches), kOneThreads, 0, stream>>>(a, units, one_groups(units, a.beams));
  } else {
    beam_runs_kernel<<<dim3(runs * a.searches * a.beams), kRunThreads, 0, stream>>>(a, runs);
    beam_join_kernel<<<dim3(a.searches), kJoinThreads, 0, stream>>>(a, runs);
  }
  return hipGetLastError();
}

}  // namespace mmr
