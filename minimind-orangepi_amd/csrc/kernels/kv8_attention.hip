// kv8_attention.hip -- causal attention over the 8-bit paged cache.
//
//   o[m] = sum_j p_mj v_j / sum_j p_mj,  p_mj = 2^(s_mj - r_m),
//   s_mj = (q_m . k_j) log2(e) / sqrt(d)     for keys j <= context + token(m)
//
// with one pass over the keys and a running reference r_m in place of the row
// maximum.  Both products run on the int8 matrix cores with the cache's codes
// as they are stored.  The fp32 operand goes in as fixed-point digits: an
// integer n is the sum of d_k 256^k with d_k in [-128, 127], and the bytes of
// n + 0x808080 are those digits, the lower three with their top bit flipped.
// Products and sums of digits and codes are exact in int32, so the only
// roundings are those of q (2^-30 or 2^-23 of its row's largest value), of p
// (2^-26) and of the fp32 sums over pages; nothing is converted to fp16.
//
// S^T = K Q^T has keys as rows and query rows as columns, O^T = V^T P^T
// dimensions as rows.  In the result layout (lane l: column l % 16, rows
// 4 (l / 16) + i) and in the operand layout (lane l: row or column l % 16, 16
// bytes of K from part l / 16) a lane therefore keeps its column, and if key
// row 4 g + i of the t-th of a page's four products is key 16 g + 4 t + i, the
// 16 scores that a lane gets are those of the 16 keys whose digits it has to
// supply: P goes from one product to the next in registers.
//
// Two forms of a tile:
//   4 rows:  the 16 columns are 4 rows x 4 digits: the K and V operands are
//            read by one product each, and a score is the sum over four lanes.
//            A decode step of a group of four heads is one tile.
//   16 rows: a column is a row, digits are products of their own (3 of q, 4
//            of p) that a lane adds up itself.
#include "device_common.h"
#include "kv8_common.h"

#include <algorithm>
#include <cfloat>

namespace mmr {

namespace {

constexpr int kAttnWaves = 4;
constexpr int kAttnThreads = kAttnWaves * kWave;
constexpr float kNoRow = -FLT_MAX / 2;  // reference of a row that has met no key
constexpr float kLead = 5.0f;           // a score may pass the reference by 2^kLead
constexpr int kPBits = 25;              // p in units of 2^-25: at most 2^30 with the lead
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
__device__ __forceinline__ uint32_t digit_flip(int k, int top) { return k < top ? 0x80808080u : 0u; }

template <int D, int kRows, bool kKeySplit>
__global__ __launch_bounds__(kAttnThreads) void kv8_attention_kernel(Kv8AttnArgs a, int chunk, int splits) {
  constexpr int kTiles = D / 16;                  // of the output's dimensions
  constexpr int kQ = kRows == 4 ? 1 : 3;          // digit operands of q
  constexpr int kP = kRows == 4 ? 1 : 4;          // and of p
  constexpr int kQTop = kRows == 4 ? 3 : 2;       // the signed digit
  constexpr int kQBits = kRows == 4 ? 29 : 22;
  const int s = blockIdx.y, hkv = a.cache.hkv, group = a.hq / hkv;
  const int split = blockIdx.x % splits, unit_of_grid = blockIdx.x / splits;  // (tile, head), a tile's heads together
  const int h = unit_of_grid % hkv;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), lane = threadIdx.x % kWave;
  const int g = lane / 16, col = lane % 16;
  Kv8Span span;
  const bool fine = kv8_span(a.cache, a.offsets, a.context, s, a.rows, a.max_rows, &span);
  if (!fine || (span.n > 0 && static_cast<int64_t>(span.context) + span.n > a.max_tokens)) {
    if (blockIdx.x == 0 && threadIdx.x == 0) atomicOr(a.error, kKv8BadRows);
    return;
  }
  const int total = span.n * group;  // rows of this group of heads
  const int tile = kKeySplit ? unit_of_grid / hkv : unit_of_grid / hkv * kAttnWaves + wave;
  const int first = tile * kRows;
  if (first >= total) return;  // a wave of the form without a key split has no barrier ahead
  const int last_token = (min(first + kRows, total) - 1) / group;
  const int pages = (span.context + last_token) / kKv8Page + 1;
  const int begin = split * chunk, end = min(begin + chunk, pages);
  if (begin >= end) return;
  const int used = (pages + chunk - 1) / chunk;  // splits of this tile

  // This lane's column.
  const int m = first + (kRows == 4 ? col / 4 : col);
  const int digit = kRows == 4 ? col % 4 : 0;
  const bool is_row = m < total;
  const int token = is_row ? m / group : 0, head = h * group + (is_row ? m % group : 0);
  const int limit = is_row ? span.context + token : -1;  // its last key
  const int64_t row = (static_cast<int64_t>(span.first) + token) * a.hq + head;
  const int all_see = span.context + first / group;  // every row sees keys up to here

  Operand<D> q[kQ];
  float unit;       // of a score's integer, in log2
  bool bad = false; // a query that is not finite gives a row of NaN
  {
    const float* p = a.query + row * D;
    constexpr int kFull = Operand<D>::kFull, kHalf = Operand<D>::kHalf;
    float v[16 * kFull + 8 * kHalf];
#pragma unroll
    for (int c = 0; c < kFull; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) *reinterpret_cast<float4*>(v + 16 * c + 4 * i) = *reinterpret_cast<const float4*>(p + 64 * c + 16 * g + 4 * i);
#pragma unroll
    for (int i = 0; i < 2 * kHalf; ++i)
      *reinterpret_cast<float4*>(v + 16 * kFull + 4 * i) = *reinterpret_cast<const float4*>(p + 64 * kFull + 8 * g + 4 * i);
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
    int n[4 * kWords];
#pragma unroll
    for (int i = 0; i < 4 * kWords; ++i)
      n[i] = (bad ? 0 : static_cast<int>(rintf(ldexpf(v[i], kQBits - x)))) + (kRows == 4 ? 0x808080 : 0x8080);
#pragma unroll
    for (int k = 0; k < kQ; ++k) {
      const int which = kRows == 4 ? digit : k;
      int w[kWords];
#pragma unroll
      for (int i = 0; i < kWords; ++i) w[i] = gather_digits(n + 4 * i, digit_select(which), digit_flip(which, kQTop));
#pragma unroll
      for (int c = 0; c < kFull; ++c) q[k].word[c] = i32x4{w[4 * c], w[4 * c + 1], w[4 * c + 2], w[4 * c + 3]};
      if constexpr (kHalf) q[k].word[kFull] = i32x4{w[4 * kFull], w[4 * kFull + 1], 0, 0};
    }
    unit = ldexpf(1.4426950408889634f / sqrtf(static_cast<float>(D)), x - kQBits);
  }
  const float weight = kRows == 4 ? ldexpf(1.0f, 8 * digit) : 1.0f;

  i32x4 sum[kP][kTiles] = {};    // digits of the output since the last move
  float out[kTiles][4] = {};     // and before it
  float ref = kNoRow, l = 0.0f;  // l: of this lane's keys
  int held_exp = kKv8MinExp - 1; // of V in sum
  int since = 0;

  auto move = [&](float factor) {  // sum into out, which then scales by factor
    const float w = ldexpf(weight, held_exp - kPBits);
#pragma unroll
    for (int t = 0; t < kTiles; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float f;
        if constexpr (kRows == 4) {
          f = static_cast<float>(sum[0][t][i]);
          sum[0][t][i] = 0;
        } else {
          f = static_cast<float>(sum[3][t][i]);
          f = f * 256.0f + static_cast<float>(sum[2][t][i]);
          f = f * 256.0f + static_cast<float>(sum[1][t][i]);
          f = f * 256.0f + static_cast<float>(sum[0][t][i]);
          sum[0][t][i] = sum[1][t][i] = sum[2][t][i] = sum[3][t][i] = 0;
        }
        out[t][i] = (out[t][i] + f * w) * factor;
      }
    l *= factor;
    since = 0;
  };

  const int32_t* table = a.cache.table + static_cast<int64_t>(s) * a.cache.per_seq;
  for (int p = begin + (kKeySplit ? wave : 0); p < end; p += kKeySplit ? kAttnWaves : 1) {
    const int page = table[p];
    if (page < 0 || page >= a.cache.pages) {  // its keys count as hidden
      if (lane == 0) atomicOr(a.error, kKv8BadRows);
      continue;
    }
    const int64_t at = kv8_offset(page, h, hkv, D), exp_at = kv8_exp_offset(page, h, hkv);
    const int8_t* k = a.cache.keys + at;
    const int8_t* v = a.cache.values + at;
    const uint32_t key_exps = *reinterpret_cast<const uint32_t*>(a.cache.key_exps + exp_at);
    const uint32_t value_exps = *reinterpret_cast<const uint32_t*>(a.cache.value_exps + exp_at);
    Operand<D> kf[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) load_operand(kf[t], k + (16 * (col / 4) + 4 * t + col % 4) * D, g);
    i32x4 vf[kTiles];
#pragma unroll
    for (int t = 0; t < kTiles; ++t) vf[t] = *reinterpret_cast<const i32x4*>(v + (16 * t + col) * kKv8Page + 16 * g);

    // Blocks past the tile's last key hold anything: their exponents don't count.
    const int blocks = min(kKv8Blocks, (span.context + last_token - p * kKv8Page) / kKv8Block + 1);
    int page_exp = kKv8MinExp - 1;
#pragma unroll
    for (int b = 0; b < kKv8Blocks; ++b)
      if (b < blocks) page_exp = max(page_exp, static_cast<int>(static_cast<int8_t>(value_exps >> (8 * b))));
    const int my_exp = static_cast<int8_t>(value_exps >> (8 * g));

    float score[4][4];
    const float to_log2 = unit * ldexpf(1.0f, static_cast<int8_t>(key_exps >> (8 * g)));
    float top = -INFINITY;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      i32x4 acc[kQ];
#pragma unroll
      for (int n = 0; n < kQ; ++n) acc[n] = multiply<D>(kf[t], q[n]);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float f;
        if constexpr (kRows == 4) {
          f = quad_add(static_cast<float>(acc[0][i]) * weight);
        } else {
          f = fmaf(static_cast<float>(acc[2][i] * 256 + acc[1][i]), 256.0f, static_cast<float>(acc[0][i]));
        }
        score[t][i] = f * to_log2;
      }
    }
    if (p * kKv8Page + kKv8Page - 1 > all_see) {
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (p * kKv8Page + 16 * g + 4 * t + i > limit) score[t][i] = -INFINITY;
    }
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) top = fmaxf(top, score[t][i]);

    if (__any(top > ref + kLead) || page_exp > held_exp || since == kMostPages) {
      const float next = fmaxf(ref, column_max(top));
      move(__builtin_amdgcn_exp2f(ref - next));
      ref = next;
      held_exp = max(held_exp, page_exp);
    }
    ++since;
    // Keys of hidden blocks have p = 0: any finite factor will do.
    const float to_int = ldexpf(1.0f, min(my_exp - held_exp, 0) + kPBits);
    int digits[kP][4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      int u[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float e = __builtin_amdgcn_exp2f(score[t][i] - ref);
        l += e;
        u[i] = static_cast<int>(fmaf(e, to_int, 0.5f)) + 0x808080;
      }
#pragma unroll
      for (int n = 0; n < kP; ++n) {
        const int which = kRows == 4 ? digit : n;
        digits[n][t] = gather_digits(u, digit_select(which), digit_flip(which, 3));
      }
    }
#pragma unroll
    for (int n = 0; n < kP; ++n) {
      const i32x4 pf = {digits[n][0], digits[n][1], digits[n][2], digits[n][3]};
#pragma unroll
      for (int t = 0; t < kTiles; ++t)
        sum[n][t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(vf[t], pf, sum[n][t], 0, 0, 0);
    }
  }
  move(1.0f);
  l = column_sum(l);
  if (bad) l = __builtin_nanf("");
  if constexpr (kRows == 4) {
#pragma unroll
    for (int t = 0; t < kTiles; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) out[t][i] = quad_add(out[t][i]);
  }

  float* const part_ml = a.part + static_cast<int64_t>(a.rows) * a.hq * splits * D;
  if constexpr (!kKeySplit) {
    if (!is_row) return;
    const float inv = l != 0.0f ? 1.0f / l : 0.0f;
#pragma unroll
    for (int t = 0; t < kTiles; ++t)
      *reinterpret_cast<float4*>(a.out + row * D + 16 * t + 4 * g) =
          make_float4(out[t][0] * inv, out[t][1] * inv, out[t][2] * inv, out[t][3] * inv);
  } else {
    __shared__ float sh_ref[kAttnWaves][kRows], sh_l[kAttnWaves][kRows];
    __shared__ __align__(16) float sh_out[kAttnWaves][kRows][D];
    const int r = kRows == 4 ? col / 4 : col;
    if (digit == 0) {
      if (g == 0) {
        sh_ref[wave][r] = ref;
        sh_l[wave][r] = l;
      }
#pragma unroll
      for (int t = 0; t < kTiles; ++t)
        *reinterpret_cast<float4*>(&sh_out[wave][r][16 * t + 4 * g]) =
            make_float4(out[t][0], out[t][1], out[t][2], out[t][3]);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < kRows * D; i += kAttnThreads) {
      const int mr = i / D, dim = i - mr * D, mm = first + mr;
      if (mm >= total) break;
      float top = sh_ref[0][mr];
#pragma unroll
      for (int w = 1; w < kAttnWaves; ++w) top = fmaxf(top, sh_ref[w][mr]);
      float o = 0.0f, ll = 0.0f;
#pragma unroll
      for (int w = 0; w < kAttnWaves; ++w) {
        const float f = __builtin_amdgcn_exp2f(sh_ref[w][mr] - top);
        o += f * sh_out[w][mr][dim];
        ll += f * sh_l[w][mr];
      }
      const int64_t to = (static_cast<int64_t>(span.first) + mm / group) * a.hq + h * group + mm % group;
      if (used == 1) {
        a.out[to * D + dim] = ll != 0.0f ? o / ll : 0.0f;
      } else {
        a.part[(to * splits + split) * D + dim] = o;
        if (dim == 0) {
          part_ml[(to * splits + split) * 2] = top;
          part_ml[(to * splits + split) * 2 + 1] = ll;
        }
      }
    }
  }
}

// Joins the splits of the rows that had more than one: a wave per (token, head).
__global__ __launch_bounds__(kAttnThreads) void kv8_combine_kernel(Kv8AttnArgs a, int chunk, int splits,
                                                                   int tile_rows) {
  const int s = blockIdx.y, lane = threadIdx.x % kWave, d = a.cache.d;
  Kv8Span span;
  if (!kv8_span(a.cache, a.offsets, a.context, s, a.rows, a.max_rows, &span)) return;
  if (static_cast<int64_t>(span.context) + span.n > a.max_tokens) return;
  const int i = blockIdx.x * kAttnWaves + threadIdx.x / kWave;
  if (i >= span.n * a.hq) return;
  const int token = i / a.hq, head = i - token * a.hq, group = a.hq / a.cache.hkv;
  const int m = token * group + head % group;
  const int tile_end = min((m / tile_rows + 1) * tile_rows, span.n * group);
  const int pages = (span.context + (tile_end - 1) / group) / kKv8Page + 1;
  const int used = (pages + chunk - 1) / chunk;
  if (used == 1) return;
  const int64_t to = static_cast<int64_t>(span.first) * a.hq + i;
  const float* ml = a.part + static_cast<int64_t>(a.rows) * a.hq * splits * d + to * splits * 2;
  const float* o = a.part + to * splits * d;
  float top = kNoRow;
  for (int x = 0; x < used; ++x) top = fmaxf(top, ml[2 * x]);
  float l = 0.0f, acc[2] = {0.0f, 0.0f};
  for (int x = 0; x < used; ++x) {
    const float f = __builtin_amdgcn_exp2f(ml[2 * x] - top);
    l += f * ml[2 * x + 1];
#pragma unroll
    for (int c = 0; c < 2; ++c)
      if (lane + 64 * c < d) acc[c] += f * o[static_cast<int64_t>(x) * d + lane + 64 * c];
  }
#pragma unroll
  for (int c = 0; c < 2; ++c)
    if (lane + 64 * c < d) a.out[to * d + lane + 64 * c] = l != 0.0f ? acc[c] / l : 0.0f;
}

}  // namespace

Kv8AttnPlan kv8_attention_plan(int hq, int hkv, int d, int seqs, int rows, int max_rows, int64_t max_tokens) {
  Kv8AttnPlan p;
  const int group = hq / hkv;
  const int64_t most = static_cast<int64_t>(group) * max_rows;
  const int64_t pages = (max_tokens + kKv8Page - 1) / kKv8Page;
  p.tile_rows = most <= 4 ? 4 : 16;
  const int64_t tiles = (most + p.tile_rows - 1) / p.tile_rows;
  const int64_t blocks = tiles * hkv * seqs;
  if (blocks >= 1024) {
    p.chunk_pages = static_cast<int>(std::max<int64_t>(pages, 1));
    p.splits = 1;
    return p;
  }
  p.chunk_pages = static_cast<int>(std::max<int64_t>(kAttnWaves, pages * blocks / 768));
  p.splits = static_cast<int>(std::max<int64_t>(1, (pages + p.chunk_pages - 1) / p.chunk_pages));
  if (p.splits > 1) p.partial_floats = static_cast<int64_t>(rows) * hq * p.splits * (d + 2);
  return p;
}

namespace {

template <int D>
void launch_attention_for(const Kv8AttnArgs& a, const Kv8AttnPlan& p, hipStream_t stream) {
  const int hkv = a.cache.hkv, most = a.hq / hkv * a.max_rows;
  const int tiles = (most + p.tile_rows - 1) / p.tile_rows;
  const dim3 grid(p.splits * tiles * hkv, a.cache.seqs);
  if (p.tile_rows == 4)
    kv8_attention_kernel<D, 4, true><<<grid, kAttnThreads, 0, stream>>>(a, p.chunk_pages, p.splits);
  else if (p.splits > 1 || tiles < kAttnWaves)
    kv8_attention_kernel<D, 16, true><<<grid, kAttnThreads, 0, stream>>>(a, p.chunk_pages, p.splits);
  else
    kv8_attention_kernel<D, 16, false>
        <<<dim3((tiles + kAttnWaves - 1) / kAttnWaves * hkv, a.cache.seqs), kAttnThreads, 0, stream>>>(
            a, p.chunk_pages, p.splits);
  if (p.splits > 1)
    kv8_combine_kernel<<<dim3((a.max_rows * a.hq + kAttnWaves - 1) / kAttnWaves, a.cache.seqs), kAttnThreads, 0,
                         stream>>>(a, p.chunk_pages, p.splits, p.tile_rows);
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
