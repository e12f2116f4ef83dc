// kv8_attention.hip -- causal attention over the 8-bit paged cache.
//
//   o[m] = sum_j p_mj v_j / sum_j p_mj,  p_mj = 2^(s_mj - r_m),
//   s_mj = (q_m . k_j) log2(e) / sqrt(d)     for keys j <= context + token(m)
//
// with one pass over the keys and a running reference r_m in place of the row
// maximum: a score may pass it a little before everything is scaled down to a
// new one.  Two kernels, by the rows (token, head) that a sequence brings to a
// group of heads that share their keys:
//
// Steps, up to 8 rows (a decode step of eight heads), 4 a block: int8 matrix
// cores on the codes as they are stored.  The fp32 operand goes in as fixed-point digits:
// an integer n is the sum of d_k 256^k with d_k in [-128, 127], and the bytes
// of n + 0x808080 are those digits, the lower three with their top bit
// flipped.  Products and sums of digits and codes are exact in int32; rounded
// are q (by up to 2^-29 of its row's largest value), p times its values' power
// of two (by 2^-29 of the reference's at the row's largest exponent) and the
// fp32 sums over pages.  The 16 columns of a product are 4 rows x 4 digits, so K
// and V are each the operand of one product, and a score is the sum over four
// lanes.
//
// More rows: fp16 matrix cores on codes widened to fp16 (exactly) once per
// block, with the fp32 operand as two fp16 planes: q is rounded by up to 2^-23
// of each value, p by 2^-22, but no finer than 2^-39 of the row's largest value
// and 2^-35 of the reference's at the row's largest exponent.  Per 16 rows this
// takes as many matrix cycles as digits would (a digit operand multiplies
// twice the columns, but takes three digits of q and four of p), but none of
// the adding up and taking apart of digits, which was most of that form's
// time, and a quarter of its accumulators.
//
// In both, S^T = K Q^T has keys as rows and query rows as columns, O^T = V^T
// P^T dimensions as rows.  In the result layout (lane l: column l % 16, rows
// 4 (l / 16) + i) and in the operand layout (lane l: row or column l % 16, a
// run of K from part l / 16) a lane keeps its column, and the keys are dealt
// to the rows of S^T so that the scores that a lane gets are those of the keys
// whose weights it has to supply: P never leaves the lane.
//
// Times in this file are us a call in replayed graphs (medians of graphs of 30
// calls over three sets of inputs; 1.6 us are any kernel's there), with the
// join where a call has one.  Sequences of a batch have a quarter to all of the
// tokens named.
#include "device_common.h"
#include "kv8_common.h"

#include <algorithm>
#include <cfloat>

namespace mmr {

namespace {

constexpr int kStepWaves = 8, kStepThreads = kStepWaves * kWave;
constexpr int kJoinThreads = 256;
constexpr float kNoRow = -FLT_MAX / 2;  // reference of a row that has met no key
constexpr float kStepLead = 2.0f, kRowsLead = 5.0f;  // a score may pass the reference by this much (log2)
constexpr int kStepRows = 8, kStepTile = 4;  // rows that the kernel for steps takes, and of a block
constexpr int kRowsThreads = 256;
constexpr int kFewSplits = 8;
constexpr int kRowsTile = 64;          // rows of a block of the kernel for many
constexpr int kRowsPBits = 10;          // its p in units of 2^-10: at most 2^15 with the lead
constexpr int kPBits = 28;              // p of steps in units of 2^-28: at most 2^30 with the lead
// See kv8_attention_plan.
constexpr int kLeastPages = 2, kLeastRowsPages = 4, kWidePages = 16;
constexpr int kStepBlocks = 256, kRowsBlocks = 1280, kFewRows = 256;
constexpr int kMostSplits = 64;         // a lane of a wave each in the join
using f16x8 = _Float16 __attribute__((ext_vector_type(8)));
using f32x4 = float __attribute__((ext_vector_type(4)));
constexpr int kMostPages = 1024;        // int32 sums: 64 keys x 128 x 127 < 2^20 a page

// D columns of an operand, 64 to a product; of 32 left over, each part's 8
// bytes and 8 zeros.  (The 32-column product is not used: chained to a
// 64-column one, its result was read before it was written.)
template <int D>
struct Operand {
  static constexpr int kFull = D / 64, kHalf = D % 64 / 32;
  i32x4 word[kFull + kHalf];
};

template <int D>
__device__ __forceinline__ i32x4 multiply(const Operand<D>& a, const Operand<D>& b) {
  i32x4 acc = {0, 0, 0, 0};
#pragma unroll
  for (int c = 0; c < Operand<D>::kFull + Operand<D>::kHalf; ++c)
    acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(a.word[c], b.word[c], acc, 0, 0, 0);
  return acc;
}

// Row of codes (or of dimensions) `p`, part g of 4.
template <int D>
__device__ __forceinline__ void load_operand(Operand<D>& o, const int8_t* p, int g) {
#pragma unroll
  for (int c = 0; c < Operand<D>::kFull; ++c) o.word[c] = *reinterpret_cast<const i32x4*>(p + 64 * c + 16 * g);
  if constexpr (Operand<D>::kHalf) {
    const int2 half = *reinterpret_cast<const int2*>(p + 64 * Operand<D>::kFull + 8 * g);
    o.word[Operand<D>::kFull] = i32x4{half.x, half.y, 0, 0};
  }
}

__device__ __forceinline__ float quad_add(float v) {
  v += dpp_move<dpp::kQuadXor1>(v);
  return v + dpp_move<dpp::kQuadXor2>(v);
}
// Over the four lanes of a column.
__device__ __forceinline__ float column_max(float v) {
  v = fmaxf(v, __shfl_xor(v, 16));
  return fmaxf(v, __shfl_xor(v, 32));
}
__device__ __forceinline__ float column_sum(float v) {
  v += __shfl_xor(v, 16);
  return v + __shfl_xor(v, 32);
}

// Byte `which` of each of four words (sel picks it of two), flipped.
__device__ __forceinline__ int gather_digits(const int u[4], uint32_t sel, uint32_t flip) {
  const uint32_t lo = __builtin_amdgcn_perm(u[1], u[0], sel), hi = __builtin_amdgcn_perm(u[3], u[2], sel);
  return static_cast<int>(__builtin_amdgcn_perm(hi, lo, 0x05040100u) ^ flip);
}
__device__ __forceinline__ uint32_t digit_select(int k) { return k | (4 + k) << 8; }
__device__ __forceinline__ uint32_t digit_flip(int k) { return k < 3 ? 0x80808080u : 0u; }

// 0, but not to the compiler: the result of a load that it sees to be the same
// in all lanes it moves to a scalar register right behind the load, which waits
// for it and for all that was asked for before.
__device__ __forceinline__ int zero_of_lanes() {
  int zero = 0;
  asm volatile("" : "+v"(zero));
  return zero;
}

// Of q.k / sqrt(d), in log2.  Powers of two of the query and of the keys are
// added before they scale it: either alone may have no fp32 number.
template <int D>
__device__ __forceinline__ float score_unit() {
  return 1.4426950408889634f / sqrtf(static_cast<float>(D));
}

// The largest of a page's first `blocks` exponents.
__device__ __forceinline__ int largest_exponent(uint32_t exps, int blocks) {
  int e = kKv8MinExp - 1;
#pragma unroll
  for (int b = 0; b < kKv8Blocks; ++b)
    if (b < blocks) e = max(e, static_cast<int>(static_cast<int8_t>(exps >> (8 * b))));
  return e;
}
// Of the page whose first key is `first`, those whose keys a row with the last key `limit` attends.
__device__ __forceinline__ int blocks_seen(int limit, int first) {
  return min(kKv8Blocks, max(0, limit - first + kKv8Block) / kKv8Block);
}

// Splits of at most `chunk` pages each that a row's `pages` are dealt to, evenly.
__device__ __forceinline__ int splits_used(int pages, int chunk) { return (pages + chunk - 1) / chunk; }

// Reference and sum of a row's split, after all the splits' outputs.
__device__ __forceinline__ void store_ml(const Kv8AttnArgs& a, int64_t row, int splits, int split, int d, float ref,
                                         float l) {
  float* ml = a.part + static_cast<int64_t>(a.rows) * a.hq * splits * d + (row * splits + split) * 2;
  ml[0] = ref;
  ml[1] = l;
}

// Steps: waves take the pages of a split in turn and join their results at the
// end.  Waves wait on counters 39 % of their time, the vector units are busy 19 %
// of it: what counts is that a wave always has a page under way.  32 sequences
// of up to 8,192 tokens, two KV heads of d 96: 72 MB in 18.8 us, 3.8 TB/s; one
// query over 32,768 11.6, over 8,192 8.8, over 1,024 8.3, over 500 7.0, over 128
// 5.3: two dependent loads, a page's arithmetic (two of them one after another
// from 513 to 1,024 tokens), the join in LDS and, above, the one of the splits.
// The fp16 cache's attention takes 12.4, 6.9, 6.0, 5.9 and 5.8 there.
template <int D>
__global__ __launch_bounds__(kStepThreads, 2) void kv8_step_kernel(Kv8AttnArgs a, int chunk, int splits) {
  constexpr int kRows = kStepTile, kTiles = D / 16;  // tiles of the output's dimensions
  const int s = blockIdx.y, hkv = a.cache.hkv, group = a.hq / hkv;
  const int split = blockIdx.x % splits, h = blockIdx.x / splits, first = blockIdx.z * kRows;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), lane = threadIdx.x % kWave;
  const int g = lane / 16, col = lane % 16;
  // Page numbers of this wave's next 64 steps, one a lane: read along with the
  // offsets, not after them.
  const int32_t* table = a.cache.table + static_cast<int64_t>(s) * a.cache.per_seq;
  const int begin = split * chunk, from = begin + wave;
  int numbers = table[min(from + kStepWaves * lane, a.cache.per_seq - 1)];
  Kv8Span span;
  const bool fine = kv8_span(a.cache, a.offsets, a.context, s, a.rows, a.max_rows, &span);
  if (!fine || (span.n > 0 && static_cast<int64_t>(span.context) + span.n > a.max_tokens)) {
    if (blockIdx.x == 0 && threadIdx.x == 0) atomicOr(a.error, kKv8BadRows);
    return;
  }
  const int total = min(span.n * group - first, kRows);  // rows of this group of heads, from `first` on
  if (total <= 0) return;
  const int last_key = span.context + (first + total - 1) / group, pages = last_key / kKv8Page + 1;
  const int used = splits_used(pages, chunk), end = min(begin + chunk, pages);
  if (split >= used) return;

  // This lane's column: digit `digit` of row m.  Columns past the last row are
  // that row again: another block's row could change while it is read (out in
  // place of query) and decide when this block's sums are scaled.
  const int m = col / 4, digit = col % 4, at_row = first + min(m, total - 1);
  const int token = at_row / group, head = h * group + at_row % group;
  const int limit = span.context + token;  // its last key
  const int64_t row = (static_cast<int64_t>(span.first) + token) * a.hq + head;

  // The operands of the next page, asked for as soon as those of the page at
  // hand are used.  A page number that is out of range reads page 0, hidden.
  Operand<D> kf[4];
  i32x4 vf[kTiles];
  uint32_t next_key_exps, next_value_exps;
  bool next_hidden;
  const int8_t *next_k, *next_v;
  int ask_at = 0;
  const int lane_zero = zero_of_lanes();
  auto ask = [&]() {  // addresses and exponents of step ask_at, at most the last
    const int step = min(ask_at, (end - 1 - from) / kStepWaves);
    if (ask_at == step && step > 0 && step % kWave == 0) {  // not for the last again
      numbers = table[min(from + kStepWaves * (step + lane), a.cache.per_seq - 1)];
      asm volatile("" : "+v"(numbers));  // waited for here, not wherever it is read
    }
    ++ask_at;
    const int number = __builtin_amdgcn_readlane(numbers, step % kWave);
    next_hidden = number < 0 || number >= a.cache.pages;
    const int page = next_hidden ? 0 : number;
    const int64_t at = kv8_offset(page, h, hkv, D), exp_at = kv8_exp_offset(page, h, hkv);
    next_k = a.cache.keys + at;
    next_v = a.cache.values + at;
    next_key_exps = *reinterpret_cast<const uint32_t*>(a.cache.key_exps + exp_at + lane_zero);
    next_value_exps = *reinterpret_cast<const uint32_t*>(a.cache.value_exps + exp_at + lane_zero);
  };
  // Row 4 g + i of the t-th product is key 16 g + 4 t + i: a lane's scores are
  // those of part g's 16 keys of P.
  auto ask_keys = [&]() {
#pragma unroll
    for (int t = 0; t < 4; ++t) load_operand(kf[t], next_k + (16 * (col / 4) + 4 * t + col % 4) * D, g);
  };
  auto ask_values = [&]() {
#pragma unroll
    for (int t = 0; t < kTiles; ++t)
      vf[t] = *reinterpret_cast<const i32x4*>(next_v + (16 * t + col) * kKv8Page + 16 * g);
  };
  if (from < end) {
    ask();
    ask_keys();
    ask_values();
  }

  Operand<D> q;
  int unit_exp;      // a score's integer has units of 2^unit_exp score_unit<D>(), in log2, before the keys' exponent
  bool bad = false;  // a query that is not finite gives a row of NaN
  {
    constexpr int kQBits = 29;
    const float* p = a.query + row * D;
    constexpr int kFull = Operand<D>::kFull, kHalf = Operand<D>::kHalf;
    float v[16 * kFull + 8 * kHalf];
#pragma unroll
    for (int c = 0; c < kFull; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *reinterpret_cast<float4*>(v + 16 * c + 4 * i) = *reinterpret_cast<const float4*>(p + 64 * c + 16 * g + 4 * i);
#pragma unroll
    for (int i = 0; i < 2 * kHalf; ++i)
      *reinterpret_cast<float4*>(v + 16 * kFull + 4 * i) =
          *reinterpret_cast<const float4*>(p + 64 * kFull + 8 * g + 4 * i);
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < 16 * kFull + 8 * kHalf; ++i) {
      bad = bad || !(fabsf(v[i]) < __builtin_inff());
      top = fmaxf(top, fabsf(v[i]));
    }
    top = column_max(top);
    bad = column_max(bad ? 1.0f : 0.0f) > 0.0f;
    int x = 0;
    if (top > 0.0f && !bad) (void)frexpf(top, &x);
    constexpr int kWords = 4 * kFull + 2 * kHalf;
    int w[kWords];
#pragma unroll
    for (int i = 0; i < kWords; ++i) {
      int n[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        n[j] = (bad ? 0 : static_cast<int>(rintf(ldexpf(v[4 * i + j], kQBits - x)))) + 0x808080;
      w[i] = gather_digits(n, digit_select(digit), digit_flip(digit));
    }
#pragma unroll
    for (int c = 0; c < kFull; ++c) q.word[c] = i32x4{w[4 * c], w[4 * c + 1], w[4 * c + 2], w[4 * c + 3]};
    if constexpr (kHalf) q.word[kFull] = i32x4{w[4 * kFull], w[4 * kFull + 1], 0, 0};
    unit_exp = x - kQBits;
  }
  const float weight = ldexpf(1.0f, 8 * digit);

  i32x4 sum[kTiles] = {};        // digits of the output since the last move
  float out[kTiles][4] = {};     // and before it
  float ref = kNoRow, l = 0.0f;  // l: of this lane's keys
  int held_exp = kKv8MinExp - 1; // of V in sum, for this lane's row
  int since = 0;

  auto move = [&](float factor) {  // sum into out, which then scales by factor
    const float w = ldexpf(weight, held_exp - kPBits);
#pragma unroll
    for (int t = 0; t < kTiles; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        out[t][i] = (out[t][i] + static_cast<float>(sum[t][i]) * w) * factor;
        sum[t][i] = 0;
      }
    l *= factor;
    since = 0;
  };

  for (int p = from; p < end; p += kStepWaves) {
    const uint32_t key_exps = next_key_exps, value_exps = __builtin_amdgcn_readfirstlane(next_value_exps);
    const bool hidden = next_hidden;
    const int my_exp = static_cast<int8_t>(value_exps >> (8 * g));

    float score[4][4];
    const float to_log2 = ldexpf(score_unit<D>(), unit_exp + static_cast<int8_t>(key_exps >> (8 * g)));
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const i32x4 acc = multiply<D>(kf[t], q);
#pragma unroll
      for (int i = 0; i < 4; ++i) score[t][i] = quad_add(static_cast<float>(acc[i]) * weight) * to_log2;
    }
    ask();
    ask_keys();
    // A row's sums are relative to the values that it attends: blocks past its
    // last key, which hold anything, or what later rows attend, don't count.
    int page_exp = largest_exponent(value_exps, kKv8Blocks);
    if (hidden) {
      if (lane == 0) atomicOr(a.error, kKv8BadRows);
      page_exp = kKv8MinExp - 1;
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) score[t][i] = -INFINITY;
    } else if (p * kKv8Page + kKv8Page - 1 > span.context) {  // the first token sees keys up to context
      page_exp = largest_exponent(value_exps, blocks_seen(limit, p * kKv8Page));
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (p * kKv8Page + 16 * g + 4 * t + i > limit) score[t][i] = -INFINITY;
    }
    float top = -INFINITY;
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) top = fmaxf(top, score[t][i]);

    if (__any(top > ref + kStepLead || page_exp > held_exp) || since == kMostPages) {
      const float next = fmaxf(ref, column_max(top));
      if (since > 0) move(__builtin_amdgcn_exp2f(ref - next));  // not before the first page
      ref = next;
      held_exp = max(held_exp, page_exp);
    }
    ++since;
    // Keys of hidden blocks have p = 0: any finite factor will do.
    const float to_int = ldexpf(1.0f, min(my_exp - held_exp, 0) + kPBits);
    i32x4 pf;
    float part = 0.0f;  // of the page first: a sum over long contexts is off by its number of terms
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      int u[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float e = __builtin_amdgcn_exp2f(score[t][i] - ref);
        part += e;
        u[i] = static_cast<int>(fmaf(e, to_int, 0.5f)) + 0x808080;
      }
      pf[t] = gather_digits(u, digit_select(digit), digit_flip(digit));
    }
    l += part;
#pragma unroll
    for (int t = 0; t < kTiles; ++t)
      sum[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(vf[t], pf, sum[t], 0, 0, 0);
    ask_values();
  }
  move(1.0f);
  l = column_sum(l);
  if (bad) l = __builtin_nanf("");
#pragma unroll
  for (int t = 0; t < kTiles; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i) out[t][i] = quad_add(out[t][i]);

  __shared__ float sh_ref[kStepWaves][kRows], sh_l[kStepWaves][kRows];
  __shared__ __align__(16) float sh_out[kStepWaves][kRows][D];
  if (digit == 0) {
    if (g == 0) {
      sh_ref[wave][m] = ref;
      sh_l[wave][m] = l;
    }
#pragma unroll
    for (int t = 0; t < kTiles; ++t)
      *reinterpret_cast<float4*>(&sh_out[wave][m][16 * t + 4 * g]) =
          make_float4(out[t][0], out[t][1], out[t][2], out[t][3]);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < total * D; i += kStepThreads) {
    const int mr = i / D, dim = i - mr * D;
    float top = sh_ref[0][mr];
#pragma unroll
    for (int w = 1; w < kStepWaves; ++w) top = fmaxf(top, sh_ref[w][mr]);
    float o = 0.0f, ll = 0.0f;
#pragma unroll
    for (int w = 0; w < kStepWaves; ++w) {
      const float f = __builtin_amdgcn_exp2f(sh_ref[w][mr] - top);
      o += f * sh_out[w][mr][dim];
      ll += f * sh_l[w][mr];
    }
    const int64_t to =
        (static_cast<int64_t>(span.first) + (first + mr) / group) * a.hq + h * group + (first + mr) % group;
    if (used == 1) {
      a.out[to * D + dim] = ll != 0.0f ? o / ll : 0.0f;
    } else {
      a.part[(to * splits + split) * D + dim] = o;
      if (dim == 0) store_ml(a, to, splits, split, D, top, ll);
    }
  }
}

// 16 codes as fp16: a byte with its top bit flipped is code + 128, and below
// the exponent byte 0x64 it is the fp16 number 1024 + 128 + code.
__device__ __forceinline__ void widen(const uint4& codes, uint4* lo, uint4* hi) {
  const uint32_t w[4] = {codes.x, codes.y, codes.z, codes.w};
  uint32_t h[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t t = w[i] ^ 0x80808080u;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const f16x2 v = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, t, j ? 0x04030402u : 0x04010400u));
      h[2 * i + j] = __builtin_bit_cast(uint32_t, v - f16x2{1152.0f, 1152.0f});
    }
  }
  *lo = make_uint4(h[0], h[1], h[2], h[3]);
  *hi = make_uint4(h[4], h[5], h[6], h[7]);
}

// x = hi + lo in fp16 with hi truncated, which packs two in one instruction;
// lo takes up the difference (split2 rounds hi, in three): 21 bits.
__device__ __forceinline__ void split2_truncated(float x0, float x1, uint32_t& hi, uint32_t& lo) {
  hi = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(x0, x1));
  asm("v_fma_mixlo_f16 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(lo) : "v"(hi), "v"(x0));
  asm("v_fma_mixhi_f16 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "+v"(lo) : "v"(hi), "v"(x1));
}

// 16 rows a wave, all waves over the same pages, which the block widens into
// LDS: the operands of every product, 16 bytes a lane in the order of lanes.
//
// Measured: 3,000 rows after 1,111, 8 heads of d 96 over two KV heads, 75 us a
// call (73 to 76 from card to card), 320 TFLOP/s of the formula's products, of
// which the two planes make twice as many (the fp16 cache's attention: 63.6).
// Vector units are busy 50 % of the kernel, matrix cores 27 %, LDS 27 %.  In an
// earlier state, whose kernel took 78, it took 70 to 75 with the lower planes'
// products, the exponentials or the widening of pages left out, one at a time:
// it is none of them but the chain barrier - LDS - products - weights - products
// with three waves a SIMD.  32 rows a wave (half the LDS reads a row, two waves
// a SIMD) took as long there, blocks of eight waves 101.
template <int D>
__global__ __launch_bounds__(kRowsThreads, D <= 96 ? 3 : 2) void kv8_rows_kernel(Kv8AttnArgs a, int chunk, int splits) {
  constexpr int kTiles = D / 16, kRuns = D / 32;  // tiles of the output, products along D
  constexpr int kPieces = D / 32;                 // 16-byte pieces of a page that a thread widens
  constexpr int kOperand = kWave;                 // of uint4
  __shared__ uint4 stage[2][(4 * kRuns + 2 * kTiles) * kOperand];  // K [4 t][runs], then V [2 u][tiles]
  const int s = blockIdx.y, hkv = a.cache.hkv, group = a.hq / hkv;
  const int grid_tiles = gridDim.x / (splits * hkv);
  const int grid_tile = blockIdx.x % grid_tiles, h = blockIdx.x / grid_tiles % hkv;
  const int split = blockIdx.x / grid_tiles / hkv;
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / kWave), lane = tid % kWave;
  const int g = lane / 16, col = lane % 16;
  Kv8Span span;
  const bool fine = kv8_span(a.cache, a.offsets, a.context, s, a.rows, a.max_rows, &span);
  if (!fine || (span.n > 0 && static_cast<int64_t>(span.context) + span.n > a.max_tokens)) {
    if (blockIdx.x == 0 && tid == 0) atomicOr(a.error, kKv8BadRows);
    return;
  }
  const int total = span.n * group;
  const int tiles = (total + kRowsTile - 1) / kRowsTile, tile = tiles - 1 - grid_tile;  // the longest first
  if (tile < 0) return;
  const int first = tile * kRowsTile;
  const int last_token = (min(first + kRowsTile, total) - 1) / group;
  const int pages = (span.context + last_token) / kKv8Page + 1;
  const int used = splits_used(pages, chunk);
  if (split >= used) return;
  const int each = (pages + used - 1) / used, begin = split * each, end = min(begin + each, pages);

  // This lane's row.
  const int wave_first = first + 16 * wave;
  const bool works = wave_first < total;
  const int all_see = span.context + min(wave_first, total - 1) / group;
  const int m = min(wave_first + col, total - 1), token = m / group;  // lanes past the last row are that row again
  const int limit = span.context + token;                             // its last key
  const int64_t row = (static_cast<int64_t>(span.first) + token) * a.hq + h * group + m % group;

  const int32_t* table = a.cache.table + static_cast<int64_t>(s) * a.cache.per_seq;
  int numbers = table[min(begin + lane, a.cache.per_seq - 1)];
  float v[8 * kRuns];  // of the query, which does not wait for a page's number
#pragma unroll
  for (int c = 0; c < kRuns; ++c)
#pragma unroll
    for (int i = 0; i < 2; ++i)
      *reinterpret_cast<float4*>(v + 8 * c + 4 * i) =
          *reinterpret_cast<const float4*>(a.query + row * D + 32 * c + 8 * g + 4 * i);
  uint4 piece[kPieces];
  uint32_t next_key_exps, next_value_exps;
  bool next_hidden;
  const int lane_zero = zero_of_lanes();
  auto ask = [&](int p) {
    const int step = p - begin;
    if (step > 0 && step % kWave == 0) {
      numbers = table[min(p + lane, a.cache.per_seq - 1)];
      asm volatile("" : "+v"(numbers));  // waited for here, not wherever it is read
    }
    const int number = __builtin_amdgcn_readlane(numbers, step % kWave);
    next_hidden = number < 0 || number >= a.cache.pages;
    const int page = next_hidden ? 0 : number;
    const int64_t at = kv8_offset(page, h, hkv, D), exp_at = kv8_exp_offset(page, h, hkv);
#pragma unroll
    for (int j = 0; j < kPieces; ++j) {
      const int x = tid + kRowsThreads * j;  // keys are 4 D pieces, values as many: a wave is in one of them
      piece[j] = *reinterpret_cast<const uint4*>(x < 4 * D ? a.cache.keys + at + 16 * x
                                                           : a.cache.values + at + 16 * (x - 4 * D));
    }
    next_key_exps = *reinterpret_cast<const uint32_t*>(a.cache.key_exps + exp_at + lane_zero);
    next_value_exps = *reinterpret_cast<const uint32_t*>(a.cache.value_exps + exp_at + lane_zero);
  };
  // Key 32 u + 8 g + 4 w + i is row 4 g + i of product t = 2 u + w, so a lane's
  // scores of products 2 u and 2 u + 1 are of the 8 keys that are its run of
  // the u-th product with V.  Places of an operand are exchanged within runs
  // of 8 (128 bytes, all banks): the 16 lanes that write together hold a few
  // keys' runs of dimensions, or a few dimensions' runs of keys.
  auto key_place = [](int operand, int part) { return (2 * operand + part / 2) & 7; };
  auto value_place = [](int u, int part) { return ((part / 2 ^ u) & 1) * 4; };
  auto put = [&](uint4* to) {
#pragma unroll
    for (int j = 0; j < kPieces; ++j) {
      const int x = tid + kRowsThreads * j;
      uint4 lo, hi;
      widen(piece[j], &lo, &hi);
      uint4* at;
      int place;
      if (x < 4 * D) {  // 16 dimensions of a key
        const int key = x / (D / 16), dims = x % (D / 16);
        const int t = key / 32 * 2 + key % 8 / 4, r = key % 32 / 8 * 4 + key % 4;
        at = to + (t * kRuns + dims / 2) * kOperand + dims % 2 * 32;
        place = r ^ key_place(t * kRuns + dims / 2, dims % 2 * 2);
      } else {  // 16 keys of a dimension
        const int dim = (x - 4 * D) / 4, b = x % 4;
        at = to + (4 * kRuns + b / 2 * kTiles + dim / 16) * kOperand + b % 2 * 32;
        place = dim % 16 ^ value_place(b / 2, b % 2 * 2);
      }
      at[place] = lo;
      at[16 + place] = hi;
    }
  };
  ask(begin);

  f16x8 q_hi[kRuns], q_lo[kRuns];
  int unit_exp;      // as for steps
  bool bad = false;  // a query that is not finite gives a row of NaN
  {
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < 8 * kRuns; ++i) {
      bad = bad || !(fabsf(v[i]) < __builtin_inff());
      top = fmaxf(top, fabsf(v[i]));
    }
    top = column_max(top);
    bad = column_max(bad ? 1.0f : 0.0f) > 0.0f;
    int x = 0;
    if (top > 0.0f && !bad) (void)frexpf(top, &x);
    // The largest below 2^15: rounded off is up to 2^-23 of a value or, where its
    // lower plane is subnormal, 2^-39 of the largest.
#pragma unroll
    for (int c = 0; c < kRuns; ++c) {
      uint4 hi, lo;
      uint32_t *ph = &hi.x, *pl = &lo.x;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        split2(bad ? 0.0f : ldexpf(v[8 * c + 2 * i], 15 - x), bad ? 0.0f : ldexpf(v[8 * c + 2 * i + 1], 15 - x), ph[i],
               pl[i]);
      q_hi[c] = __builtin_bit_cast(f16x8, hi);
      q_lo[c] = __builtin_bit_cast(f16x8, lo);
    }
    unit_exp = x - 15;
  }

  f32x4 out[kTiles] = {};
  float ref = kNoRow, l = 0.0f;
  int held_exp = kKv8MinExp - 1;
  put(stage[0]);
  if (!works) {  // rows past the last: this wave only helps with the pages
    for (int p = begin; p < end; ++p) {
      __syncthreads();
      if (p + 1 < end) {
        ask(p + 1);
        put(stage[(p + 1 - begin) % 2]);
      }
    }
    return;
  }
  // No branch around the loop's sums, of which the compiler would keep copies:
  // a page that no row sees, the last of a tile for some waves or one with a
  // bad number, has all its keys masked.
  for (int p = begin; p < end; ++p) {
    const uint4* now = stage[(p - begin) % 2];
    const uint32_t key_exps = next_key_exps, value_exps = __builtin_amdgcn_readfirstlane(next_value_exps);
    const bool hidden = next_hidden;
    if (hidden && tid == 0) atomicOr(a.error, kKv8BadRows);
    __syncthreads();  // this page is in LDS, and every wave is done with the one before
    if (p + 1 < end) ask(p + 1);
    // Two sums at a time: a sum's products wait for each other.
    f32x4 score[4];
#pragma unroll
    for (int t = 0; t < 4; t += 2) {
      f16x8 kf[2][kRuns];
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        score[t + w] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int c = 0; c < kRuns; ++c) {
          const int o = (t + w) * kRuns + c;
          kf[w][c] = __builtin_bit_cast(f16x8, now[o * kOperand + (lane ^ key_place(o, g))]);
        }
      }
#pragma unroll
      for (int c = 0; c < 2 * kRuns; ++c)
#pragma unroll
        for (int w = 0; w < 2; ++w)
          score[t + w] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
              kf[w][c % kRuns], c < kRuns ? q_lo[c % kRuns] : q_hi[c % kRuns], score[t + w], 0, 0, 0);
    }
    const int shift = 8 * (g / 2);  // of this lane's block of each half page
    float to_log2[2] = {ldexpf(score_unit<D>(), unit_exp + static_cast<int8_t>(key_exps >> shift)),
                        ldexpf(score_unit<D>(), unit_exp + static_cast<int8_t>(key_exps >> (16 + shift)))};
    // As for steps: of the blocks that the row attends.
    int page_exp = largest_exponent(value_exps, kKv8Blocks);
    if (hidden || p * kKv8Page + kKv8Page - 1 > all_see) {
      page_exp = largest_exponent(value_exps, hidden ? 0 : blocks_seen(limit, p * kKv8Page));
      // Scaled first: a factor may be 0 or, of a block that holds anything, infinite.
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          score[t][i] = hidden || p * kKv8Page + 32 * (t / 2) + 8 * g + 4 * (t % 2) + i > limit
                            ? -INFINITY
                            : score[t][i] * to_log2[t / 2];
      to_log2[0] = to_log2[1] = 1.0f;
    }
    float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) top[t / 2] = fmaxf(top[t / 2], score[t][i]);
    const float page_top = fmaxf(top[0] * to_log2[0], top[1] * to_log2[1]);
    if (__any(page_top > ref + kRowsLead || page_exp > held_exp)) {
      const float next = fmaxf(ref, column_max(page_top));
      const int next_exp = max(held_exp, page_exp);
      const float f = __builtin_amdgcn_exp2f(ref - next), down = ldexpf(f, held_exp - next_exp);
      l *= f;
#pragma unroll
      for (int t = 0; t < kTiles; ++t) out[t] *= down;
      ref = next;
      held_exp = next_exp;
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      // The value block's factor goes into the exponent.  Below 2^-60 of the
      // largest block it no longer falls: what it weighs is nothing in fp16.
      const int my_exp = static_cast<int8_t>(value_exps >> (16 * u + shift));
      const int bias = min(max(my_exp - held_exp, -60), 0) + kRowsPBits;
      const float from = static_cast<float>(bias) - ref;
      float part = 0.0f;
      uint4 hi, lo;
      uint32_t *ph = &hi.x, *pl = &lo.x;
#pragma unroll
      for (int w = 0; w < 2; ++w)
#pragma unroll
        for (int i = 0; i < 4; i += 2) {
          const float e0 = __builtin_amdgcn_exp2f(fmaf(score[2 * u + w][i], to_log2[u], from));
          const float e1 = __builtin_amdgcn_exp2f(fmaf(score[2 * u + w][i + 1], to_log2[u], from));
          part += e0;
          part += e1;
          split2_truncated(e0, e1, ph[2 * w + i / 2], pl[2 * w + i / 2]);
        }
      l = fmaf(part, ldexpf(1.0f, -bias), l);
      const f16x8 p_hi = __builtin_bit_cast(f16x8, hi), p_lo = __builtin_bit_cast(f16x8, lo);
#pragma unroll
      for (int t = 0; t < kTiles; t += 2) {
        f16x8 vf[2];
#pragma unroll
        for (int w = 0; w < 2; ++w)
          vf[w] = __builtin_bit_cast(
              f16x8, now[(4 * kRuns + u * kTiles + t + w) * kOperand + (lane ^ value_place(u, g))]);
#pragma unroll
        for (int w = 0; w < 2; ++w)
          out[t + w] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf[w], p_lo, out[t + w], 0, 0, 0);
#pragma unroll
        for (int w = 0; w < 2; ++w)
          out[t + w] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf[w], p_hi, out[t + w], 0, 0, 0);
      }
    }
    if (p + 1 < end) put(stage[(p + 1 - begin) % 2]);
  }
  l = column_sum(l);
  if (bad) l = __builtin_nanf("");
  if (wave_first + col >= total) return;
  const float inv = used > 1 ? 1.0f : l != 0.0f ? 1.0f / l : 0.0f;
  float* to = used > 1 ? a.part + (row * splits + split) * D : a.out + row * D;
#pragma unroll
  for (int t = 0; t < kTiles; ++t) {
    float4 o;
    float* po = &o.x;
#pragma unroll
    for (int i = 0; i < 4; ++i) po[i] = ldexpf(out[t][i], held_exp - kRowsPBits) * inv;
    *reinterpret_cast<float4*>(to + 16 * t + 4 * g) = o;
  }
  if (used > 1 && g == 0) store_ml(a, row, splits, split, D, ref, l);
}

// Splits of row `i` of a sequence's (token, head) rows.
__device__ __forceinline__ int splits_of(const Kv8AttnArgs& a, const Kv8Span& span, int i, int chunk, int tile_rows) {
  const int token = i / a.hq, head = i - token * a.hq, group = a.hq / a.cache.hkv;
  const int m = token * group + head % group;
  const int tile_end = min((m / tile_rows + 1) * tile_rows, span.n * group);
  const int pages = (span.context + (tile_end - 1) / group) / kKv8Page + 1;
  return splits_used(pages, chunk);
}

// Joins a few splits of many rows: d / 4 threads a (token, head).
__global__ __launch_bounds__(kJoinThreads) void kv8_combine_few_kernel(Kv8AttnArgs a, int chunk, int splits,
                                                                       int tile_rows) {
  const int s = blockIdx.y, d = a.cache.d, quads = d / 4, each = kJoinThreads / quads;
  Kv8Span span;
  if (!kv8_span(a.cache, a.offsets, a.context, s, a.rows, a.max_rows, &span)) return;
  if (static_cast<int64_t>(span.context) + span.n > a.max_tokens) return;
  const int part = threadIdx.x / quads, quad = threadIdx.x - part * quads, i = blockIdx.x * each + part;
  if (part >= each || i >= span.n * a.hq) return;
  const int used = splits_of(a, span, i, chunk, tile_rows);
  if (used == 1) return;
  const int64_t to = static_cast<int64_t>(span.first) * a.hq + i;
  const float2* ml =
      reinterpret_cast<const float2*>(a.part + static_cast<int64_t>(a.rows) * a.hq * splits * d) + to * splits;
  const float4* o = reinterpret_cast<const float4*>(a.part + to * splits * d) + quad;
  float4 v[kFewSplits];
  float2 of[kFewSplits];
#pragma unroll
  for (int y = 0; y < kFewSplits; ++y) {
    v[y] = y < used ? o[y * quads] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    of[y] = y < used ? ml[y] : make_float2(kNoRow, 0.0f);
  }
  float top = of[0].x, l = 0.0f;
#pragma unroll
  for (int y = 1; y < kFewSplits; ++y) top = fmaxf(top, of[y].x);
  float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
  for (int y = 0; y < kFewSplits; ++y) {
    const float w = __builtin_amdgcn_exp2f(of[y].x - top);
    l += w * of[y].y;
    sum.x += w * v[y].x, sum.y += w * v[y].y, sum.z += w * v[y].z, sum.w += w * v[y].w;
  }
  const float inv = l != 0.0f ? 1.0f / l : 0.0f;
  reinterpret_cast<float4*>(a.out + to * d)[quad] = make_float4(sum.x * inv, sum.y * inv, sum.z * inv, sum.w * inv);
}

// Joins many splits, a block per (token, head): groups of d / 4 threads take
// splits in turn, four dimensions each, with all loads under way before the
// first wave, a split a lane, has the weights.
template <int D>
__global__ __launch_bounds__(kJoinThreads) void kv8_combine_kernel(Kv8AttnArgs a, int chunk, int splits,
                                                                   int tile_rows) {
  constexpr int kQuads = D / 4, kGroups = kJoinThreads / kQuads, kEach = (kMostSplits + kGroups - 1) / kGroups;
  static_assert(kMostSplits == kWave, "a split a lane");
  __shared__ float weight[kMostSplits], shared_l;
  __shared__ float4 shared_out[kGroups][kQuads];
  const int s = blockIdx.y, i = blockIdx.x, x = threadIdx.x, g = x / kQuads, quad = x - g * kQuads;
  Kv8Span span;
  if (!kv8_span(a.cache, a.offsets, a.context, s, a.rows, a.max_rows, &span)) return;
  if (static_cast<int64_t>(span.context) + span.n > a.max_tokens) return;
  if (i >= span.n * a.hq) return;
  const int used = splits_of(a, span, i, chunk, tile_rows);
  if (used == 1) return;
  const int64_t to = static_cast<int64_t>(span.first) * a.hq + i;
  const float2* ml =
      reinterpret_cast<const float2*>(a.part + static_cast<int64_t>(a.rows) * a.hq * splits * D) + to * splits;
  const float4* o = reinterpret_cast<const float4*>(a.part + to * splits * D) + quad;
  float2 of = make_float2(kNoRow, 0.0f);
  if (x < used) of = ml[x];
  float4 v[kEach];
#pragma unroll
  for (int n = 0; n < kEach; ++n) {
    const int y = g + kGroups * n;
    v[n] = g < kGroups && y < used ? o[y * kQuads] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  }
  if (x < kWave) {
    const float w = __builtin_amdgcn_exp2f(of.x - group_max<kWave>(of.x));
    const float l = group_sum<kWave>(w * of.y);
    weight[x] = w;
    if (x == 0) shared_l = l;
  }
  __syncthreads();
  if (g < kGroups) {
    float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int n = 0; n < kEach; ++n) {
      const float w = weight[min(g + kGroups * n, kMostSplits - 1)];  // of splits past the last: times 0
      sum.x += w * v[n].x, sum.y += w * v[n].y, sum.z += w * v[n].z, sum.w += w * v[n].w;
    }
    shared_out[g][quad] = sum;
  }
  __syncthreads();
  if (x < kQuads) {
    float4 sum = shared_out[0][x];
    for (int y = 1; y < min(kGroups, used); ++y) {
      const float4 more = shared_out[y][x];
      sum.x += more.x, sum.y += more.y, sum.z += more.z, sum.w += more.w;
    }
    const float inv = shared_l != 0.0f ? 1.0f / shared_l : 0.0f;
    reinterpret_cast<float4*>(a.out + to * D)[x] = make_float4(sum.x * inv, sum.y * inv, sum.z * inv, sum.w * inv);
  }
}

}  // namespace

// Splits along the context, sized by the longest one a launch may meet (blocks
// past a sequence's end leave at once).  Measured with d 96 and, where nothing
// else is said, 8 heads on two KV heads:
//   up to kStepRows rows of a KV head are steps, though the second block of four
//   reads the pages again (8 heads on one KV head: one query over 32,768 tokens
//   10.8, 16 over up to 8,000 13.3; as many rows 17.7 and 16.9; 16 heads on two,
//   32 queries over up to 4,000, 16.3 and 20.4);
//   steps of at most kWidePages pages take one block and no join, mostly for
//   batches (32 queries over up to 1,000 tokens 9.1, split from 9 pages on 10.0;
//   one query over 778 8.1 and 8.2, over 1,000 8.4 and 8.3, over 320 6.5 and, split
//   from 5 pages on, 8.0; 24 pages of one query without a split 9.7, with it 8.5);
//   more take kStepBlocks blocks in all (32 queries over up to 4,000 14.1; with
//   384 blocks 19.2, with 192 15.0) and at most kMostSplits splits, which is what
//   the join takes (one query over 32,768: 11.5, with 32 splits 12.7);
//   many rows take kRowsBlocks blocks, whose tiles see different numbers of
//   keys (3,000 rows after 1,111: 75; with 768 blocks 82, with 256 96), but
//   at most kFewSplits splits, whose join is cheap, from kFewRows (row, head)
//   pairs on: 4,096 pairs, 512 rows after 2,000, take 21.6 with 8 splits, 27.9 with
//   16, 29.8 with 64.  256 pairs, 4 sequences of 8 rows after 13,000, take 16.4
//   with 64 and 41.8 with 8.  Between, long contexts would gain from more than 8
//   splits up to some 1,000 pairs (128 rows after 9,000: 32.7, with 64 splits 23.7;
//   after 2,000: 15.6 and 14.8; 16 sequences of up to 8 rows over up to 13,000:
//   42.7 and 30.7);
//   a split has kLeastPages pages (one query over 4,000 tokens 8.6, 5 rows there
//   9.9; with four 8.9 and 12.5), of many rows kLeastRowsPages, which are more
//   to join (1,500 rows 24.9; with three 28.2).
// A launch is sized as if every sequence brought max_rows rows: with a prompt
// among them, single rows get no splits and a wave each (512 rows and 31 single
// rows over up to 8,192 tokens 386; apart 13.5 and 18.2).
Kv8AttnPlan kv8_attention_plan(int hq, int hkv, int d, int seqs, int rows, int max_rows, int64_t max_tokens) {
  Kv8AttnPlan p;
  const int64_t most = static_cast<int64_t>(hq / hkv) * max_rows;
  const int64_t pages = (max_tokens + kKv8Page - 1) / kKv8Page;
  const bool step = most <= kStepRows;
  p.tile_rows = step ? kStepTile : kRowsTile;
  const int64_t blocks = (most + p.tile_rows - 1) / p.tile_rows * hkv * seqs;
  const int64_t wanted = step ? kStepBlocks : kRowsBlocks;
  const bool few = step || static_cast<int64_t>(rows) * hq <= kFewRows;
  const int64_t splits = few ? kMostSplits : kFewSplits, least = few ? kLeastPages : kLeastRowsPages;
  // Of a prompt's tiles, the first sees the context and the last all of max_tokens.
  const int64_t mean = step ? pages : std::max<int64_t>(1, (2 * max_tokens - max_rows) / (2 * kKv8Page));
  int64_t chunk = pages;
  if (blocks < wanted && !(step && pages <= kWidePages))
    chunk = std::max<int64_t>({least, (mean * blocks + wanted - 1) / wanted, (pages + splits - 1) / splits});
  p.chunk_pages = static_cast<int>(chunk);
  p.splits = static_cast<int>((pages + chunk - 1) / chunk);
  if (p.splits > 1) p.partial_floats = static_cast<int64_t>(rows) * hq * p.splits * (d + 2);
  return p;
}

namespace {

template <int D>
void launch_attention_for(const Kv8AttnArgs& a, const Kv8AttnPlan& p, hipStream_t stream) {
  const int hkv = a.cache.hkv, most = a.hq / hkv * a.max_rows;
  const int tiles = (most + p.tile_rows - 1) / p.tile_rows;
  if (p.tile_rows != kStepTile)
    kv8_rows_kernel<D><<<dim3(p.splits * tiles * hkv, a.cache.seqs), kRowsThreads, 0, stream>>>(a, p.chunk_pages,
                                                                                               p.splits);
  else
    kv8_step_kernel<D><<<dim3(p.splits * hkv, a.cache.seqs, tiles), kStepThreads, 0, stream>>>(a, p.chunk_pages,
                                                                                              p.splits);
  if (p.splits > 1 && p.splits <= kFewSplits) {
    const int each = kJoinThreads / (D / 4);
    kv8_combine_few_kernel<<<dim3((a.max_rows * a.hq + each - 1) / each, a.cache.seqs), kJoinThreads, 0, stream>>>(
        a, p.chunk_pages, p.splits, p.tile_rows);
  } else if (p.splits > 1)
    kv8_combine_kernel<D><<<dim3(a.max_rows * a.hq, a.cache.seqs), kJoinThreads, 0, stream>>>(
        a, p.chunk_pages, p.splits, p.tile_rows);
}

}  // namespace

hipError_t launch_kv8_attention(const Kv8AttnArgs& a, hipStream_t stream) {
  const Kv8AttnPlan p =
      kv8_attention_plan(a.hq, a.cache.hkv, a.cache.d, a.cache.seqs, a.rows, a.max_rows, a.max_tokens);
  switch (a.cache.d) {
    case 32: launch_attention_for<32>(a, p, stream); break;
    case 64: launch_attention_for<64>(a, p, stream); break;
    case 96: launch_attention_for<96>(a, p, stream); break;
    case 128: launch_attention_for<128>(a, p, stream); break;
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

}  // namespace mmr
