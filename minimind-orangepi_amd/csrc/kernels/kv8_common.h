// kv8_common.h -- the 8-bit paged cache as its kernels see it.
//
// A page holds 64 tokens of every KV head in four blocks of 16.  A cached
// value is code * 2^e: an int8 code and the exponent of its (block, head), so
// moving a block to a larger exponent is a rounded shift of its codes and
// decoding is exact in fp32.  Keys are stored [page][head][64][d], values
// transposed, [page][head][d][64]: with the tokens of one dimension
// contiguous, 16 of them are one operand register of the matrix instructions
// that multiply by the probabilities.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "kernels.h"

namespace mmr {

constexpr int kKv8Blocks = kKv8Page / kKv8Block;  // blocks of a page

using i32x4 = int __attribute__((ext_vector_type(4)));

// Codes of one (page, head); the same offset for keys and values.
__device__ __forceinline__ int64_t kv8_offset(int page, int head, int hkv, int d) {
  return (static_cast<int64_t>(page) * hkv + head) * (kKv8Page * d);
}
// Exponents of one (page, head): one byte a block.
__device__ __forceinline__ int64_t kv8_exp_offset(int page, int head, int hkv) {
  return (static_cast<int64_t>(page) * hkv + head) * kKv8Blocks;
}

// The rows that sequence s brings, checked against what the launch was sized
// for: false (nothing of the sequence may be touched) if the offsets fall,
// leave [0, rows], bring more than max_rows rows, or reach past the table.
struct Kv8Span {
  int first, n, context;
};
__device__ __forceinline__ bool kv8_span(const Kv8Pages& c, const int32_t* offsets, const int32_t* context, int s,
                                         int rows, int max_rows, Kv8Span* out) {
  const int lo = offsets[s], hi = offsets[s + 1], at = context[s];
  out->first = lo;
  out->n = hi - lo;
  out->context = at;
  return lo >= 0 && hi >= lo && hi <= rows && hi - lo <= max_rows && at >= 0 &&
         (hi == lo || static_cast<int64_t>(at) + (hi - lo) <= static_cast<int64_t>(c.per_seq) * kKv8Page);
}

}  // namespace mmr
