// matvec_q4.hip -- products with 4-bit weights under group scales.
//
//   y[b][r] = sum_c s[r][c / group] q[r][c] x[b][c],  q in [-8, 7], s fp16
//
// on the int8 matrix cores.  A nibble moved to the upper half of its byte is
// 16 q in two's complement, so eight weights become two operand words by one
// shift and two masks.  x goes in as fixed point: under one power of two for
// each 128 columns, an integer of 31 bits, written as four digits base 256 in
// [-128, 127] (the bytes of n + 0x808080, the lower three with their top bit
// flipped).  The 16 rows of the x operand are 4 rows of the batch x 4 digits,
// its product with 16 rows of W leaves the four digits of one (batch row,
// weight row) in the four registers of one lane, and the sums within a group
// are exact in int32: the roundings are those of x (2^-31 of the largest of
// its 128 columns) and of the fp32 sum over groups.
//
// Codes are packed by 128 columns in 64 bytes: word 4 p + j holds columns
// 32 j + 8 p + 0 .. 7, column 2 i in the low nibble of byte i and 2 i + 1 in
// the high one.  Part p of a product's K is lanes 16 p .. 16 p + 15, so a lane
// loads 16 bytes and has a share of every group, whatever the group's size.
#include "device_common.h"

#include <algorithm>

namespace mmr {

namespace {

constexpr int kQ4Waves = 4;
constexpr int kQ4Threads = kQ4Waves * kWave;
constexpr int kQ4Tile = 16;     // weight rows of a block
constexpr int kQ4Batch = 4;     // batch rows of an x operand
constexpr int kQ4Half = 1024;   // bytes of an x operand for 64 columns
constexpr int kFusedCols = 8192;  // batch x cols that a block itself turns into digits
constexpr int kManyTiles = 4;   // x operands of a block whose digits come from the workspace

using i32x4 = int __attribute__((ext_vector_type(4)));

// 1 / sqrt(mean(x^2) + eps) of a row by the whole block.
__device__ __forceinline__ float rms_scale(const float* x, int cols, float eps, float* partial) {
  float ss = 0.0f;
  for (int i = threadIdx.x; i < cols; i += kQ4Threads) ss += x[i] * x[i];
  ss = group_sum<kWave>(ss);
  __syncthreads();
  if (threadIdx.x % kWave == 0) partial[threadIdx.x / kWave] = ss;
  __syncthreads();
  float total = 0.0f;
#pragma unroll
  for (int i = 0; i < kQ4Waves; ++i) total += partial[i];
  return 1.0f / sqrtf(total / static_cast<float>(cols) + eps);
}

template <GemvPrologue kPro>
__device__ __forceinline__ float x_value(const float* x, const float* w, float scale, int c) {
  if constexpr (kPro == kProRmsNorm) return x[c] * (scale * w[c]);
  if constexpr (kPro == kProRmsNormFinal) return (x[c] * scale) * w[c];
  return x[c];
}

// Digits of one 128-column run of row b of an x operand, by one wave: two
// columns a lane.  to: [2 halves][rows][4 parts][16 bytes].  Returns the
// power of two that the products come in, NaN if a value is not finite.
template <GemvPrologue kPro>
__device__ __forceinline__ float write_digits(const float* x, const float* w, float scale, int cols, int run, int b,
                                              int rows, int8_t* to) {
  const int lane = threadIdx.x % kWave, c = run * kQ4Cols + 2 * lane;
  float v[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) v[i] = c + i < cols ? x_value<kPro>(x, w, scale, c + i) : 0.0f;
  const bool bad = __any(!(fabsf(v[0]) < __builtin_inff()) || !(fabsf(v[1]) < __builtin_inff()));
  const float top = group_max<kWave>(fmaxf(fabsf(v[0]), fabsf(v[1])));
  int e = 0;
  (void)frexpf(bad ? 0.0f : top, &e);
  e = max(e, -90);
  const int j = lane / 16, p = lane % 16 / 4, i = lane % 4;  // columns 32 j + 8 p + 2 i and + 1
  int8_t* at = to + (((j / 2) * rows + kQ4Batch * b) * 4 + p) * 16 + (j % 2) * 8 + i;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const uint32_t n = static_cast<uint32_t>(bad ? 0 : static_cast<int>(rintf(ldexpf(v[k], 30 - e)))) + 0x808080u;
#pragma unroll
    for (int d = 0; d < 4; ++d)
      at[d * 64 + 4 * k] = static_cast<int8_t>((n >> (8 * d)) ^ (d < 3 ? 0x80u : 0u));
  }
  return bad ? __builtin_nanf("") : ldexpf(1.0f, e - 34);  // the weights come as 16 q
}

// The lane's share of a run: 4 groups of 32, 2 of 64 or 1 of 128 columns.
// scales: of the lane's weight row from the run on, `left` of them there.
template <int kGroup>
__device__ __forceinline__ float run_product(const uint4& codes, const i32x4 x[2], const __half* scales, int left) {
  const uint32_t w[4] = {codes.x, codes.y, codes.z, codes.w};
  uint32_t lo[4], hi[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) lo[j] = (w[j] << 4) & 0xF0F0F0F0u, hi[j] = w[j] & 0xF0F0F0F0u;
  float y = 0.0f;
  auto join = [&](const i32x4& a, int n) {
    const float top = static_cast<float>(a[3] * 256 + a[2]), low = static_cast<float>(a[1] * 256 + a[0]);
    const float s = n < left ? __half2float(scales[n]) : 0.0f;
    y = fmaf(fmaf(top, 65536.0f, low), s, y);
  };
  const i32x4 zero = {0, 0, 0, 0};
  if constexpr (kGroup == 32) {
    // Half of a product's columns each, the other weights 0.
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int l = static_cast<int>(lo[j]), h = static_cast<int>(hi[j]);
      const i32x4 b = j % 2 ? i32x4{0, 0, l, h} : i32x4{l, h, 0, 0};
      join(__builtin_amdgcn_mfma_i32_16x16x64_i8(x[j / 2], b, zero, 0, 0, 0), j);
    }
  } else {
    i32x4 acc = zero;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const i32x4 b = {static_cast<int>(lo[2 * k]), static_cast<int>(hi[2 * k]), static_cast<int>(lo[2 * k + 1]),
                       static_cast<int>(hi[2 * k + 1])};
      acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(x[k], b, kGroup == 64 ? zero : acc, 0, 0, 0);
      if (kGroup == 64 || k == 1) join(acc, kGroup == 64 ? k : 0);
    }
  }
  return y;
}

// Weight (r, c) as the formula has it.
__device__ __forceinline__ float weight_at(const MatvecQ4Args& a, int64_t r, int c) {
  const int64_t stride = static_cast<int64_t>((a.cols + kQ4Cols - 1) / kQ4Cols) * 64;
  const int u = c % kQ4Cols;
  const uint32_t byte = a.codes[r * stride + c / kQ4Cols * 64 + (u % 32 / 8 * 4 + u / 32) * 4 + u % 8 / 2];
  const int q = static_cast<int>((u & 1 ? byte >> 4 : byte & 15) ^ 8) - 8;
  return static_cast<float>(q) * __half2float(a.scales[r * ((a.cols + a.group - 1) / a.group) + c / a.group]);
}

// A result whose row of x holds an infinity or a NaN, which fixed point has no
// digits for: the formula column by column.
template <GemvPrologue kPro>
__device__ __noinline__ float plain_product(const MatvecQ4Args& a, int b, int64_t r, float scale) {
  const float* x = a.x + static_cast<int64_t>(b) * a.cols;
  float y = 0.0f;
  for (int c = 0; c < a.cols; ++c) y = fmaf(weight_at(a, r, c), x_value<kPro>(x, a.norm_w, scale, c), y);
  return y;
}

// sums: [batch rows of the block][kQ4Tile] of products, from row0 and batch row b0.
template <GemvEpilogue kEpi>
__device__ __forceinline__ void store_results(const MatvecQ4Args& a, const float* sums, int row0, int b0, int batch) {
  constexpr int kOut = kEpi == kEpiSwiGlu ? kQ4Tile / 2 : kQ4Tile;
  for (int i = threadIdx.x; i < batch * kOut; i += kQ4Threads) {
    const int b = i / kOut, r = i % kOut;
    const int64_t bg = b0 + b;
    if constexpr (kEpi == kEpiSwiGlu) {
      if (row0 + 2 * r < a.rows)
        a.y[bg * (a.rows / 2) + row0 / 2 + r] = silu_fast(sums[b * kQ4Tile + 2 * r]) * sums[b * kQ4Tile + 2 * r + 1];
    } else if (row0 + r < a.rows) {
      const int64_t at = bg * a.rows + row0 + r;
      a.y[at] = sums[b * kQ4Tile + r] + (kEpi == kEpiResidual ? a.residual[at] : 0.0f);
    }
  }
}

// Up to four batch rows: every block writes the digits of x for itself.
template <int kGroup, GemvPrologue kPro, GemvEpilogue kEpi>
__global__ __launch_bounds__(kQ4Threads) void matvec_q4_kernel(MatvecQ4Args a) {
  extern __shared__ __align__(16) int8_t digits[];  // [runs][2][4 batch][4 parts][16]
  __shared__ float sums[kQ4Waves][kQ4Batch][kQ4Tile], partial[kQ4Waves], row_scale[kQ4Batch];
  __shared__ int broken;
  const int runs = (a.cols + kQ4Cols - 1) / kQ4Cols, groups = (a.cols + kGroup - 1) / kGroup;
  float* const units = reinterpret_cast<float*>(digits + static_cast<int64_t>(runs) * a.batch * 512);  // [batch][runs]
  const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave, g = lane / 16, col = lane % 16;
  const int rows = kQ4Batch * a.batch;  // of the x operand
  if (threadIdx.x == 0) broken = 0;
  if constexpr (kPro != kProPlain) {
    for (int b = 0; b < a.batch; ++b) {
      const float scale = rms_scale(a.x + static_cast<int64_t>(b) * a.cols, a.cols, a.eps, partial);
      if (threadIdx.x == 0) row_scale[b] = scale;
    }
  }
  __syncthreads();
  for (int u = wave; u < runs * a.batch; u += kQ4Waves) {
    const int b = u / runs, run = u - b * runs;
    const float unit = write_digits<kPro>(a.x + static_cast<int64_t>(b) * a.cols, a.norm_w,
                                          kPro == kProPlain ? 1.0f : row_scale[b], a.cols, run, b, rows,
                                          digits + static_cast<int64_t>(run) * rows * 128);
    if (lane == 0) units[b * runs + run] = unit;
    if (lane == 0 && unit != unit) broken = 1;
  }
  __syncthreads();

  const int row0 = blockIdx.x * kQ4Tile;
  const int64_t r = min(row0 + col, a.rows - 1);
  const uint8_t* codes = a.codes + r * runs * 64 + 16 * g;
  const __half* scales = a.scales + r * groups;
  const int m = min(col, rows - 1), b = min(g, a.batch - 1);
  float y = 0.0f;
  for (int run = wave; run < runs; run += kQ4Waves) {
    const uint4 w = *reinterpret_cast<const uint4*>(codes + run * 64);
    const int8_t* d = digits + static_cast<int64_t>(run) * rows * 128;
    const i32x4 x[2] = {*reinterpret_cast<const i32x4*>(d + (m * 4 + g) * 16),
                        *reinterpret_cast<const i32x4*>(d + ((rows + m) * 4 + g) * 16)};
    const int first = run * (kQ4Cols / kGroup);
    y = fmaf(run_product<kGroup>(w, x, scales + first, groups - first), units[b * runs + run], y);
  }
  sums[wave][g][col] = y;
  __syncthreads();
  if (threadIdx.x < kQ4Batch * kQ4Tile) {
    const int bb = threadIdx.x / kQ4Tile, rr = threadIdx.x % kQ4Tile;
    float total = 0.0f;
#pragma unroll
    for (int w = 0; w < kQ4Waves; ++w) total += sums[w][bb][rr];
    if (broken && bb < a.batch) {
      bool bad = false;
      for (int i = 0; i < runs; ++i) bad = bad || units[bb * runs + i] != units[bb * runs + i];
      if (bad) total = plain_product<kPro>(a, bb, min(row0 + rr, a.rows - 1), kPro == kProPlain ? 1.0f : row_scale[bb]);
    }
    sums[0][bb][rr] = total;
  }
  __syncthreads();
  store_results<kEpi>(a, &sums[0][0][0], row0, 0, a.batch);
}

// Workspace of the two-launch form: digits [ceil(batch / 4)][runs][2 KB], then
// fp32 units [batch][runs], then scales [batch].
__host__ __device__ inline int64_t q4_units_offset(int runs, int batch) {
  return static_cast<int64_t>((batch + kQ4Batch - 1) / kQ4Batch) * runs * (2 * kQ4Half);
}

template <GemvPrologue kPro>
__global__ __launch_bounds__(kQ4Threads) void q4_digits_kernel(MatvecQ4Args a) {
  __shared__ float partial[kQ4Waves];
  const int b = blockIdx.x, runs = (a.cols + kQ4Cols - 1) / kQ4Cols;
  const float* x = a.x + static_cast<int64_t>(b) * a.cols;
  int8_t* base = static_cast<int8_t*>(a.workspace);
  float* units = reinterpret_cast<float*>(base + q4_units_offset(runs, a.batch));
  const float scale = kPro == kProPlain ? 1.0f : rms_scale(x, a.cols, a.eps, partial);
  if (threadIdx.x == 0) units[static_cast<int64_t>(a.batch) * runs + b] = scale;
  int8_t* to = base + static_cast<int64_t>(b / kQ4Batch) * runs * (2 * kQ4Half);
  for (int run = threadIdx.x / kWave; run < runs; run += kQ4Waves) {
    const float unit = write_digits<kPro>(x, a.norm_w, scale, a.cols, run, b % kQ4Batch, 4 * kQ4Batch,
                                          to + static_cast<int64_t>(run) * (2 * kQ4Half));
    if (threadIdx.x % kWave == 0) units[static_cast<int64_t>(b) * runs + run] = unit;
  }
}

// More rows: 16 weight rows x 16 batch rows a block, x digits from the workspace.
template <int kGroup, GemvPrologue kPro, GemvEpilogue kEpi>
__global__ __launch_bounds__(kQ4Threads) void matvec_q4_rows_kernel(MatvecQ4Args a) {
  __shared__ float sums[kQ4Waves][kManyTiles * kQ4Batch][kQ4Tile];
  const int runs = (a.cols + kQ4Cols - 1) / kQ4Cols, groups = (a.cols + kGroup - 1) / kGroup;
  const int8_t* base = static_cast<const int8_t*>(a.workspace);
  const float* units = reinterpret_cast<const float*>(base + q4_units_offset(runs, a.batch));
  const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave, g = lane / 16, col = lane % 16;
  const int row0 = blockIdx.x * kQ4Tile, b0 = blockIdx.y * kManyTiles * kQ4Batch;
  const int batch = min(kManyTiles * kQ4Batch, a.batch - b0), tiles = (batch + kQ4Batch - 1) / kQ4Batch;
  const int64_t r = min(row0 + col, a.rows - 1);
  const uint8_t* codes = a.codes + r * runs * 64 + 16 * g;
  const __half* scales = a.scales + r * groups;
  float y[kManyTiles] = {};
  for (int run = wave; run < runs; run += kQ4Waves) {
    const uint4 w = *reinterpret_cast<const uint4*>(codes + static_cast<int64_t>(run) * 64);
    const int first = run * (kQ4Cols / kGroup);
#pragma unroll
    for (int t = 0; t < kManyTiles; ++t) {
      if (t < tiles) {
        const int8_t* d = base + (static_cast<int64_t>(b0 / kQ4Batch + t) * runs + run) * (2 * kQ4Half);
        const i32x4 x[2] = {*reinterpret_cast<const i32x4*>(d + (col * 4 + g) * 16),
                            *reinterpret_cast<const i32x4*>(d + kQ4Half + (col * 4 + g) * 16)};
        const int b = min(b0 + t * kQ4Batch + g, a.batch - 1);
        y[t] = fmaf(run_product<kGroup>(w, x, scales + first, groups - first),
                    units[static_cast<int64_t>(b) * runs + run], y[t]);
      }
    }
  }
#pragma unroll
  for (int t = 0; t < kManyTiles; ++t) sums[wave][t * kQ4Batch + g][col] = y[t];
  __syncthreads();
  for (int i = threadIdx.x; i < batch * kQ4Tile; i += kQ4Threads) {
    const int bb = i / kQ4Tile, rr = i % kQ4Tile;
    float total = 0.0f;
#pragma unroll
    for (int w = 0; w < kQ4Waves; ++w) total += sums[w][bb][rr];
    if (total != total) {  // a unit of the row is NaN, or the sum overflowed
      bool bad = false;
      for (int u = 0; u < runs; ++u) {
        const float unit = units[static_cast<int64_t>(b0 + bb) * runs + u];
        bad = bad || unit != unit;
      }
      if (bad)
        total = plain_product<kPro>(a, b0 + bb, min(row0 + rr, a.rows - 1),
                                    units[static_cast<int64_t>(a.batch) * runs + b0 + bb]);
    }
    sums[0][bb][rr] = total;
  }
  __syncthreads();
  store_results<kEpi>(a, &sums[0][0][0], row0, b0, batch);
}

bool fused_digits(int cols, int batch) {
  return batch <= kQ4Batch && static_cast<int64_t>(batch) * cols <= kFusedCols;
}

template <int kGroup, GemvPrologue kPro, GemvEpilogue kEpi>
void launch_q4(const MatvecQ4Args& a, hipStream_t stream) {
  const int tiles = (a.rows + kQ4Tile - 1) / kQ4Tile, runs = (a.cols + kQ4Cols - 1) / kQ4Cols;
  if (fused_digits(a.cols, a.batch)) {
    const size_t lds = static_cast<size_t>(runs) * a.batch * 516;
    matvec_q4_kernel<kGroup, kPro, kEpi><<<tiles, kQ4Threads, lds, stream>>>(a);
    return;
  }
  const int many = kManyTiles * kQ4Batch;
  q4_digits_kernel<kPro><<<a.batch, kQ4Threads, 0, stream>>>(a);
  matvec_q4_rows_kernel<kGroup, kPro, kEpi>
      <<<dim3(tiles, (a.batch + many - 1) / many), kQ4Threads, 0, stream>>>(a);
}

template <int kGroup, GemvPrologue kPro>
void launch_q4_epi(const MatvecQ4Args& a, GemvEpilogue epi, hipStream_t stream) {
  if (epi == kEpiResidual)
    launch_q4<kGroup, kPro, kEpiResidual>(a, stream);
  else if (epi == kEpiSwiGlu)
    launch_q4<kGroup, kPro, kEpiSwiGlu>(a, stream);
  else
    launch_q4<kGroup, kPro, kEpiStore>(a, stream);
}

template <int kGroup>
void launch_q4_pro(const MatvecQ4Args& a, GemvPrologue pro, GemvEpilogue epi, hipStream_t stream) {
  if (pro == kProRmsNorm)
    launch_q4_epi<kGroup, kProRmsNorm>(a, epi, stream);
  else if (pro == kProRmsNormFinal)
    launch_q4_epi<kGroup, kProRmsNormFinal>(a, epi, stream);
  else
    launch_q4_epi<kGroup, kProPlain>(a, epi, stream);
}

}  // namespace

int64_t matvec_q4_workspace(int cols, int batch) {
  if (fused_digits(cols, batch)) return 0;
  const int runs = (cols + kQ4Cols - 1) / kQ4Cols;
  return q4_units_offset(runs, batch) + 4 * (static_cast<int64_t>(batch) * runs + batch);
}

hipError_t launch_matvec_q4(const MatvecQ4Args& a, GemvPrologue pro, GemvEpilogue epi, hipStream_t stream) {
  switch (a.group) {
    case 32: launch_q4_pro<32>(a, pro, epi, stream); break;
    case 64: launch_q4_pro<64>(a, pro, epi, stream); break;
    case 128: launch_q4_pro<128>(a, pro, epi, stream); break;
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

}  // namespace mmr
