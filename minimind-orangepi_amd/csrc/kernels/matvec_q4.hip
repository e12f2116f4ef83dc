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
// are exact in int32: the roundings are those of x (up to 2^-30 of the largest
// of its 128 columns) and of the fp32 sum over groups.
//
// Codes are packed by 128 columns in 64 bytes: word 4 p + j holds columns
// 32 j + 8 p + 0 .. 7, column 2 i in the low nibble of byte i and 2 i + 1 in
// the high one.  Part p of a product's K is lanes 16 p .. 16 p + 15, so a lane
// loads 16 bytes and has a share of every group, whatever the group's size.
//
// Times in this file are us a call in replayed graphs (medians of graphs of 30
// calls over three sets of weights and inputs; 1.6 us are any kernel's there).
// One row, groups of 32: 1152 x 768 under a norm 4.4, 4096 x 768 with norm and
// SwiGLU 4.6, of which the kernels of fp16 weights take 2.5 and 2.8: x becomes
// digits in a chain of load, sum of squares, barrier, maximum, LDS, barrier
// before the first product.  Where weights count it pays: 32768 x 4096 in groups
// of 128 16.0, 69.4 MB at 4.3 TB/s (fp16 weights 46.4).  4096 x 768 for 32 rows of
// x 6.4 (two launches), for 3,000 94, 200 TFLOP/s; 16384 x 4096 for 32 28.4: every
// two tiles of weight rows read all digits of 16 rows of x, 256 KB there, from
// the L2.
#include "device_common.h"

#include <algorithm>

namespace mmr {

namespace {

constexpr int kQ4Waves = 8;
constexpr int kQ4Threads = kQ4Waves * kWave;
constexpr int kQ4Tile = 16;        // weight rows of a product
constexpr int kQ4Batch = 4;        // batch rows of an x operand
constexpr int kQ4Operands = 2048;  // bytes of the two x operands of a run
// Runs of all rows of x, up to kQ4Batch rows, that a block itself turns into
// digits: more of them cost a second launch less (768 x 2048 for 4 rows 9.1
// here and 8.6 in two launches, 4096 x 2048 9.4 and 10.6).
constexpr int kFusedRuns = 64;
// Tiles of rows from which blocks take several in turn, so that x is turned
// into digits once a compute unit (8192 x 4096 in groups of 32: 11.8 with a tile a
// block, 9.6; 4096 x 768 with 256 tiles 4.2 and 4.9).
constexpr int kManyRowTiles = 512;
constexpr int kWideBlocks = 256;    // then: one a compute unit
constexpr int kManyWaves = 2048;    // and its waves
constexpr int kAhead = 4;           // runs of a chunk of them
constexpr int kRing = 3;            // chunks of a wave under way
constexpr int kCodeBytes = 4096;    // of a chunk of 16 rows
constexpr int kChunkBytes = kCodeBytes + 512;  // with their scales
constexpr int kManyTiles = 4;       // x operands of a block whose digits come from the workspace
// Tiles from which such a block takes two and reads the operands for both
// (4096 x 768 for 32 rows: 6.6 with one, 6.4; 768 x 2048 8.8 and 10.3).
constexpr int kTwoTiles = 256;

// Blocks of the form whose codes go through LDS, with kTilesOfWave tiles a wave,
// from which it is taken for many rows of x: one a compute unit (groups of 64,
// 32 rows: 8192 x 2048, 256 blocks, 12.0 and 14.6 without; 4096 x 2048, 128
// blocks, 11.0 and 10.5; 16384 x 4096, 1024 blocks, 28.4 and 39.5).
constexpr int kWideRowsBlocks = 256;
constexpr int kTilesOfWave = 2;

// Under 2^e >= the largest of 128 columns, the integers are x 2^(30 - e) and 16 q:
// a product is theirs times 2^(e - 34), of which 2^-32 goes into the sums of a
// run and the rest, 2^(e - 2), is a normal number for any largest value.  Below
// 2^-124 e stays: x 2^154 is whole for the least subnormal.
constexpr int kUnitPower = 2, kLeastPower = -124;

using i32x4 = int __attribute__((ext_vector_type(4)));

// What the launch decides, beside the shape.
struct Q4Form {
  GemvPrologue pro;
  GemvEpilogue epi;
  int runs, groups;
  bool whole;  // the scales of a run are one load: every run is whole, and they are aligned
  bool even;   // then: a row has an even number of groups
  int share;   // waves of the form for many tiles that share a tile's columns
};

__device__ __forceinline__ float normalised(const Q4Form& f, float x, float w, float scale) {
  return f.pro == kProRmsNorm ? x * (scale * w) : f.pro == kProRmsNormFinal ? (x * scale) * w : x;
}

// Columns c + lane and c + 64 + lane of a run, and the weights of the norm.
struct Columns {
  float x[2], w[2];
};
__device__ __forceinline__ Columns load_columns(const MatvecQ4Args& a, const Q4Form& f, int b, int run) {
  Columns v;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int c = run * kQ4Cols + 64 * k + threadIdx.x % kWave;
    v.x[k] = c < a.cols ? a.x[static_cast<int64_t>(b) * a.cols + c] : 0.0f;
    v.w[k] = c < a.cols && f.pro != kProPlain ? a.norm_w[c] : 0.0f;
  }
  return v;
}

// Digits of a run of row b of an x operand, by one wave.  to: [2 halves][4 parts]
// [rows][16 bytes] (16 rows: in the order of the lanes that read them), half
// j / 2, part p and bytes 8 (j % 2) + i / 2 (even columns) or + 4 (odd ones)
// for column 32 j + 8 p + i.  Returns the power of
// two that run_product's sums come in, NaN if a value is not finite.
__device__ __forceinline__ float write_digits(const float v[2], int b, int rows, int8_t* to) {
  const int lane = threadIdx.x % kWave;
  const bool bad = __any(!(fabsf(v[0]) < __builtin_inff()) || !(fabsf(v[1]) < __builtin_inff()));
  const float top = group_max<kWave>(fmaxf(fabsf(v[0]), fabsf(v[1])));
  int e = 0;
  (void)frexpf(bad ? 0.0f : top, &e);
  e = max(e, kLeastPower);
  const int j = lane / 32, p = lane % 32 / 8, i = lane % 8;
  int8_t* at = to + (p * rows + kQ4Batch * b) * 16 + j * 8 + i % 2 * 4 + i / 2;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const uint32_t n = static_cast<uint32_t>(bad ? 0 : static_cast<int>(rintf(ldexpf(v[k], 30 - e)))) + 0x808080u;
#pragma unroll
    for (int d = 0; d < 4; ++d)
      at[(k * 4 * rows + d) * 16] = static_cast<int8_t>((n >> (8 * d)) ^ (d < 3 ? 0x80u : 0u));
  }
  return bad ? __builtin_nanf("") : ldexpf(1.0f, e - kUnitPower);
}

// A lane's share of a run of its weight row: 16 bytes of codes, and the scales
// of the run's groups.
template <int kGroup>
struct Run {
  static constexpr int kGroups = kQ4Cols / kGroup;
  uint4 codes;
  __half scales[kGroups];
};
template <int kGroup>
__device__ __forceinline__ void load_scales(const MatvecQ4Args& a, const Q4Form& f, int64_t row, int run, __half* to) {
  constexpr int kGroups = Run<kGroup>::kGroups;
  const __half* s = a.scales + row * f.groups + run * kGroups;
  if (f.whole && kGroups == 4) {
    *reinterpret_cast<uint2*>(to) = *reinterpret_cast<const uint2*>(s);
  } else if (f.whole && kGroups == 2) {
    *reinterpret_cast<uint32_t*>(to) = *reinterpret_cast<const uint32_t*>(s);
  } else {
#pragma unroll
    for (int n = 0; n < kGroups; ++n) to[n] = run * kGroups + n < f.groups ? s[n] : __half(0.0f);
  }
}
template <int kGroup>
__device__ __forceinline__ Run<kGroup> load_run(const MatvecQ4Args& a, const Q4Form& f, int64_t row, int run) {
  Run<kGroup> r;
  r.codes = *reinterpret_cast<const uint4*>(a.codes + (row * f.runs + run) * 64 + threadIdx.x % kWave / 16 * 16);
  load_scales<kGroup>(a, f, row, run, r.scales);
  return r;
}

// The run's products with the x operand's row of this lane's part, times
// 2^(kUnitPower - 34): batch row lane / 16, weight row lane % 16.
template <int kGroup>
__device__ __forceinline__ float run_product(const Run<kGroup>& r, const i32x4& x0, const i32x4& x1) {
  const uint32_t w[4] = {r.codes.x, r.codes.y, r.codes.z, r.codes.w};
  int lo[4], hi[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) lo[j] = (w[j] << 4) & 0xF0F0F0F0u, hi[j] = w[j] & 0xF0F0F0F0u;
  float y = 0.0f;
  auto join = [&](const i32x4& d, __half scale) {
    const float top = static_cast<float>(d[3] * 256 + d[2]), low = static_cast<float>(d[1] * 256 + d[0]);
    y = fmaf(fmaf(top, 65536.0f, low), __half2float(scale), y);
  };
  const i32x4 zero = {0, 0, 0, 0};
  if constexpr (kGroup == 32) {
    // Half of a product's columns each, the other weights 0.
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const i32x4 b = j % 2 ? i32x4{0, 0, lo[j], hi[j]} : i32x4{lo[j], hi[j], 0, 0};
      join(__builtin_amdgcn_mfma_i32_16x16x64_i8(j < 2 ? x0 : x1, b, zero, 0, 0, 0), r.scales[j]);
    }
  } else {
    const i32x4 b0 = {lo[0], hi[0], lo[1], hi[1]}, b1 = {lo[2], hi[2], lo[3], hi[3]};
    const i32x4 d0 = __builtin_amdgcn_mfma_i32_16x16x64_i8(x0, b0, zero, 0, 0, 0);
    if constexpr (kGroup == 64) {
      join(d0, r.scales[0]);
      join(__builtin_amdgcn_mfma_i32_16x16x64_i8(x1, b1, zero, 0, 0, 0), r.scales[1]);
    } else {
      join(__builtin_amdgcn_mfma_i32_16x16x64_i8(x1, b1, d0, 0, 0, 0), r.scales[0]);
    }
  }
  return y * 0x1p-32f;
}

// Weight (r, c) as the formula has it.
__device__ __forceinline__ float weight_at(const MatvecQ4Args& a, const Q4Form& f, int64_t r, int c) {
  const int u = c % kQ4Cols;
  const uint32_t byte = a.codes[(r * f.runs + c / kQ4Cols) * 64 + (u % 32 / 8 * 4 + u / 32) * 4 + u % 8 / 2];
  const int q = static_cast<int>((u & 1 ? byte >> 4 : byte & 15) ^ 8) - 8;
  return static_cast<float>(q) * __half2float(a.scales[r * f.groups + c / a.group]);
}

// A result whose row of x holds an infinity or a NaN, which fixed point has no
// digits for: the formula column by column.
__device__ __forceinline__ float plain_product(const MatvecQ4Args& a, const Q4Form& f, int b, int64_t r, float scale) {
  const float* x = a.x + static_cast<int64_t>(b) * a.cols;
  float y = 0.0f;
  for (int c = 0; c < a.cols; ++c)
    y = fmaf(weight_at(a, f, r, c), normalised(f, x[c], f.pro == kProPlain ? 0.0f : a.norm_w[c], scale), y);
  return y;
}

// A wave's results: of batch row b and weight row `row` in each lane.
__device__ __forceinline__ void finish(const MatvecQ4Args& a, const Q4Form& f, float y, int b, int row) {
  const float pair = dpp_move<dpp::kQuadXor1>(y);
  if (b >= a.batch || row >= a.rows) return;
  const int64_t at = static_cast<int64_t>(b) * a.rows + row;
  if (f.epi == kEpiSwiGlu) {
    if (row % 2 == 0) a.y[at / 2] = silu_fast(y) * pair;
  } else {
    a.y[at] = f.epi == kEpiResidual ? y + a.residual[at] : y;
  }
}

// Up to four batch rows: every block writes the digits of x for itself, kUnits
// runs of a row a wave.
template <int kUnits, int kWaves>
struct Digits {
  static constexpr int kMost = kUnits * kWaves;  // runs of all rows
  static_assert(kMost <= kFusedRuns, "and kFusedRuns in the larger form");
  float units[kMost + kAhead][kQ4Batch];         // [runs], then zeros
  float squares[kMost], row_scale[kQ4Batch];
};

// Before: the loads of x; the caller's own loads go between.
template <int kUnits, int kWaves>
__device__ __forceinline__ void load_x(const MatvecQ4Args& a, const Q4Form& f, int wave, Columns v[kUnits]) {
#pragma unroll
  for (int i = 0; i < kUnits; ++i) {
    const int u = wave + kWaves * i;
    if (u < f.runs * a.batch) v[i] = load_columns(a, f, u / f.runs, u % f.runs);
  }
}
// Returns whether a value is not finite.  to: [runs][2][4 parts][4 batch][16].
template <int kUnits, int kWaves>
__device__ __forceinline__ bool make_digits(const MatvecQ4Args& a, const Q4Form& f, int wave, const Columns v[kUnits],
                                            Digits<kUnits, kWaves>& d, int8_t* to) {
  const int lane = threadIdx.x % kWave, rows = kQ4Batch * a.batch;
  if (f.pro != kProPlain) {
#pragma unroll
    for (int i = 0; i < kUnits; ++i) {
      const int u = wave + kWaves * i;
      if (u < f.runs * a.batch) {
        const float ss = group_sum<kWave>(v[i].x[0] * v[i].x[0] + v[i].x[1] * v[i].x[1]);
        if (lane == 0) d.squares[u] = ss;
      }
    }
    __syncthreads();
  }
  bool broken = false;
#pragma unroll
  for (int i = 0; i < kUnits; ++i) {
    const int u = wave + kWaves * i;
    if (u < f.runs * a.batch) {
      const int b = u / f.runs, run = u - b * f.runs;
      float scale = 1.0f;
      if (f.pro != kProPlain) {
        const float total = group_sum<kWave>(lane < f.runs ? d.squares[b * f.runs + lane] : 0.0f);  // runs <= 64
        scale = 1.0f / sqrtf(total / static_cast<float>(a.cols) + a.eps);
        if (run == 0 && lane == 0) d.row_scale[b] = scale;
      }
      float x[2];
#pragma unroll
      for (int k = 0; k < 2; ++k) x[k] = normalised(f, v[i].x[k], v[i].w[k], scale);
      const float unit = write_digits(x, b, rows, to + run * rows * 128);
      if (lane == 0) d.units[run][b] = unit;
      broken = broken || unit != unit;
    }
  }
  if (threadIdx.x < kAhead * kQ4Batch) d.units[f.runs + threadIdx.x / kQ4Batch][threadIdx.x % kQ4Batch] = 0.0f;
  return __syncthreads_or(broken);
}

// A run's products with the digits in LDS; runs past the last have unit 0.
template <int kGroup, typename D>
__device__ __forceinline__ float use_run(const Run<kGroup>& w, const D& d, const int8_t* operand, int rows, int run,
                                         int b, float y) {
  const i32x4 x0 = *reinterpret_cast<const i32x4*>(operand + run * rows * 128);
  const i32x4 x1 = *reinterpret_cast<const i32x4*>(operand + run * rows * 128 + rows * 64);
  return fmaf(run_product<kGroup>(w, x0, x1), d.units[run][b], y);
}

template <typename D>
__device__ __forceinline__ void finish_checked(const MatvecQ4Args& a, const Q4Form& f, const D& d, bool broken, float y,
                                               int row) {
  const int g = threadIdx.x % kWave / 16;
  if (broken && g < a.batch) {
    bool bad = false;
    for (int i = 0; i < f.runs; ++i) bad = bad || d.units[i][g] != d.units[i][g];
    if (bad) y = plain_product(a, f, g, min(row, a.rows - 1), f.pro == kProPlain ? 1.0f : d.row_scale[g]);
  }
  finish(a, f, y, g, row);
}

// Few tiles of rows: one a block, whose waves share its columns.
template <int kGroup, int kUnits>
__global__ __launch_bounds__(kQ4Threads) void matvec_q4_kernel(MatvecQ4Args a, Q4Form f) {
  extern __shared__ __align__(16) int8_t digits[];
  __shared__ Digits<kUnits, kQ4Waves> d;
  __shared__ float sums[kQ4Waves][kWave];
  const int lane = threadIdx.x % kWave, g = lane / 16, col = lane % 16;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int row = blockIdx.x * kQ4Tile + col;
  constexpr int kTogether = 2;
  // Weights do not wait for x.  Runs past the last are read as the last.
  Run<kGroup> w[kTogether];
  auto ask = [&](int first) {
#pragma unroll
    for (int j = 0; j < kTogether; ++j)
      w[j] = load_run<kGroup>(a, f, min(row, a.rows - 1), min(first + j * kQ4Waves, f.runs - 1));
  };
  ask(wave);
  Columns v[kUnits];
  load_x<kUnits, kQ4Waves>(a, f, wave, v);
  const bool broken = make_digits<kUnits, kQ4Waves>(a, f, wave, v, d, digits);
  const int rows = kQ4Batch * a.batch, b = min(g, a.batch - 1);
  const int8_t* const operand = digits + (g * rows + min(col, rows - 1)) * 16;
  float y = 0.0f;
  for (int first = wave; first < f.runs; first += kTogether * kQ4Waves) {
#pragma unroll
    for (int j = 0; j < kTogether; ++j)
      y = use_run(w[j], d, operand, rows, min(first + j * kQ4Waves, f.runs), b, y);
    if (first + kTogether * kQ4Waves < f.runs) ask(first + kTogether * kQ4Waves);
  }
  sums[wave][lane] = y;
  __syncthreads();
  if (wave > 0) return;
  y = sums[0][lane];
#pragma unroll
  for (int i = 1; i < kQ4Waves; ++i) y += sums[i][lane];
  finish_checked(a, f, d, broken, y, row);
}

// Many tiles.  A lane of a product needs 16 bytes of its own weight row, and a
// load that goes by that asks for 64 places a row apart, one a cycle.  So the
// codes of a chunk, kAhead runs of 16 rows, go to LDS with direct loads, 256
// bytes of four rows each, and its scales four bytes a lane; pieces of 16 bytes
// change places within a row by its number, so that lanes that read the same
// piece of 16 rows use all banks.  For whole runs with an even number of groups
// in a row.
template <int kGroup>
struct Chunk {
  static constexpr int kGroups = Run<kGroup>::kGroups;
  static constexpr int kWords = kAhead * kGroups / 2;  // of a row's scales
  static constexpr int kScaleLoads = (16 * kWords + kWave - 1) / kWave;
  static constexpr int kLoads = kAhead + kScaleLoads;

  // Into LDS at `to`.  What is past the last row, run or group is read as the last.
  static __device__ __forceinline__ void ask(const MatvecQ4Args& a, const Q4Form& f, int tile, int first, uint32_t to) {
    const int lane = threadIdx.x % kWave, g = lane / 16, col = lane % 16, row_bytes = f.runs * 64;
    const int last_row = a.rows - 1 - tile * kQ4Tile;
    const uint8_t* codes = a.codes + static_cast<int64_t>(tile) * kQ4Tile * row_bytes;
    const __half* scales = a.scales + static_cast<int64_t>(tile) * kQ4Tile * f.groups;
#pragma unroll
    for (int q = 0; q < kAhead; ++q) {
      const int row = 4 * q + g, piece = col ^ row;
      dma_load<16>(codes, min(row, last_row) * row_bytes + min(first + piece / 4, f.runs - 1) * 64 + piece % 4 * 16,
                   to + q * 1024);
    }
#pragma unroll
    for (int q = 0; q < kScaleLoads; ++q) {
      const int i = q * kWave + lane, row = min(i / kWords, min(last_row, kQ4Tile - 1));
      const int word = min(first * kGroups / 2 + i % kWords, f.groups / 2 - 1);
      dma_load<4>(scales, (row * f.groups + 2 * word) * 2, to + kCodeBytes + q * 256);
    }
  }
  static __device__ __forceinline__ Run<kGroup> run(const int8_t* chunk, int j) {
    const int lane = threadIdx.x % kWave, g = lane / 16, col = lane % 16;
    Run<kGroup> w;
    w.codes = *reinterpret_cast<const uint4*>(chunk + col * 256 + ((4 * j + g) ^ col) * 16);
    const __half* s = reinterpret_cast<const __half*>(chunk + kCodeBytes) + col * 2 * kWords + j * kGroups;
#pragma unroll
    for (int n = 0; n < kGroups; ++n) w.scales[n] = s[n];
    return w;
  }
};

// While `later` chunks after it are under way.
template <int kLoads>
__device__ __forceinline__ void wait_for_chunk(int later) {
  static_assert(kRing == 3, "one wait for each number of later chunks");
  if (later >= 2)
    asm volatile("s_waitcnt vmcnt(%0)" : : "n"(2 * kLoads) : "memory");
  else if (later == 1)
    asm volatile("s_waitcnt vmcnt(%0)" : : "n"(kLoads) : "memory");
  else
    asm volatile("s_waitcnt vmcnt(0)" : : : "memory");
}

// Up to four batch rows: a block takes kQ4Waves / f.share tiles at a time, and
// then further ones; f.share waves share a tile's columns, a chunk each in turn,
// with kRing chunks of a wave under way.  The waits are counted by hand: all that
// a wave has under way are its chunks, kLoads loads each, which return in order.
template <int kGroup, int kUnits>
__global__ __launch_bounds__(kQ4Threads) void matvec_q4_wide_kernel(MatvecQ4Args a, Q4Form f) {
  extern __shared__ __align__(16) int8_t shared[];  // chunks [waves][kRing][codes, scales], then digits
  __shared__ Digits<kUnits, kQ4Waves> d;
  __shared__ float sums[2][kQ4Waves][kWave];
  int8_t* const digits = shared + kQ4Waves * kRing * kChunkBytes;
  const int lane = threadIdx.x % kWave, g = lane / 16, col = lane % 16;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int at_once = kQ4Waves / f.share, part = wave % f.share, slot = wave / f.share;
  const int tiles = (a.rows + kQ4Tile - 1) / kQ4Tile, stride = gridDim.x * at_once;
  const int turns = (tiles - static_cast<int>(blockIdx.x) * at_once + stride - 1) / stride;  // of this block
  const int chunks = (f.runs + kAhead - 1) / kAhead, steps = (chunks + f.share - 1) / f.share;
  int8_t* const ring = shared + wave * kRing * kChunkBytes;
  const uint32_t ring_at = __builtin_amdgcn_readfirstlane(lds_address(ring));

  // What is past the last tile is read as the last, and not used.
  int ask_tile = blockIdx.x * at_once + slot, ask_step = 0, ask_place = 0;
  auto ask = [&]() {
    Chunk<kGroup>::ask(a, f, min(ask_tile, tiles - 1), (ask_step * f.share + part) * kAhead,
                       ring_at + ask_place * kChunkBytes);
    ask_place = ask_place + 1 < kRing ? ask_place + 1 : 0;
    if (++ask_step == steps) ask_step = 0, ask_tile += stride;
  };
  const int total = turns * steps;
  Columns v[kUnits];
  load_x<kUnits, kQ4Waves>(a, f, wave, v);
  // After x has come: the compiler, which counts only the loads it makes, would
  // else wait for the chunks with it.
#pragma unroll
  for (int i = 0; i < kUnits; ++i)
#pragma unroll
    for (int k = 0; k < 2; ++k) asm volatile("" : "+v"(v[i].x[k]), "+v"(v[i].w[k]) : : "memory");
  for (int i = 0; i < min(kRing, total); ++i) ask();
  const bool broken = make_digits<kUnits, kQ4Waves>(a, f, wave, v, d, digits);

  const int rows = kQ4Batch * a.batch, b = min(g, a.batch - 1);
  const int8_t* const operand = digits + (g * rows + min(col, rows - 1)) * 16;
  int tile = blockIdx.x * at_once + slot, step = 0, turn = 0, place = 0;
  float y = 0.0f;
  for (int at = 0; at < total; ++at) {
    wait_for_chunk<Chunk<kGroup>::kLoads>(total - 1 - at);
    const int8_t* chunk = ring + place * kChunkBytes;
    place = place + 1 < kRing ? place + 1 : 0;
    const int first = (step * f.share + part) * kAhead;
    Run<kGroup> w[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) w[j] = Chunk<kGroup>::run(chunk, j);
#pragma unroll
    for (int j = 0; j < kAhead; ++j) y = use_run(w[j], d, operand, rows, min(first + j, f.runs), b, y);
    asm volatile("" : "+v"(y) : : "memory");  // the chunk is read
    if (at + kRing < total) ask();
    if (++step == steps) {
      if (f.share > 1) {
        sums[turn % 2][wave][lane] = y;
        __syncthreads();
        if (part == 0)
          for (int n = 1; n < f.share; ++n) y += sums[turn % 2][wave + n][lane];
      }
      if (part == 0) finish_checked(a, f, d, broken, y, tile * kQ4Tile + col);
      y = 0.0f;
      step = 0;
      ++turn;
      tile += stride;
    }
  }
}

// Workspace of the two-launch form: digits [ceil(batch / 4)][runs][2 KB], then
// fp32 units [batch][runs], then scales [batch].
__host__ __device__ inline int64_t q4_units_offset(int runs, int batch) {
  return static_cast<int64_t>((batch + kQ4Batch - 1) / kQ4Batch) * runs * kQ4Operands;
}

// A block a batch row.
__global__ __launch_bounds__(kQ4Threads) void q4_digits_kernel(MatvecQ4Args a, Q4Form f) {
  __shared__ float partial[kQ4Waves];
  const int b = blockIdx.x, wave = threadIdx.x / kWave;
  int8_t* base = static_cast<int8_t*>(a.workspace);
  float* units = reinterpret_cast<float*>(base + q4_units_offset(f.runs, a.batch));
  Columns v = {};
  if (wave < f.runs) v = load_columns(a, f, b, wave);
  float scale = 1.0f;
  if (f.pro != kProPlain) {
    float ss = v.x[0] * v.x[0] + v.x[1] * v.x[1];
    for (int run = wave + kQ4Waves; run < f.runs; run += kQ4Waves) {
      const Columns u = load_columns(a, f, b, run);
      ss += u.x[0] * u.x[0] + u.x[1] * u.x[1];
    }
    ss = group_sum<kWave>(ss);
    if (threadIdx.x % kWave == 0) partial[wave] = ss;
    __syncthreads();
    float total = 0.0f;
#pragma unroll
    for (int i = 0; i < kQ4Waves; ++i) total += partial[i];
    scale = 1.0f / sqrtf(total / static_cast<float>(a.cols) + a.eps);
  }
  if (threadIdx.x == 0) units[static_cast<int64_t>(a.batch) * f.runs + b] = scale;
  int8_t* to = base + static_cast<int64_t>(b / kQ4Batch) * f.runs * kQ4Operands;
  for (int run = wave; run < f.runs; run += kQ4Waves) {
    if (run != wave) v = load_columns(a, f, b, run);
    float x[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) x[k] = normalised(f, v.x[k], v.w[k], scale);
    const float unit =
        write_digits(x, b % kQ4Batch, 4 * kQ4Batch, to + static_cast<int64_t>(run) * kQ4Operands);
    if (threadIdx.x % kWave == 0) units[static_cast<int64_t>(b) * f.runs + run] = unit;
  }
}

__device__ __forceinline__ void finish_rows(const MatvecQ4Args& a, const Q4Form& f, const float* units, float y, int b,
                                            int row) {
  if (y != y && b < a.batch && row < a.rows) {  // a unit of the row is NaN, or the sum overflowed
    bool bad = false;
    for (int u = 0; u < f.runs; ++u) {
      const float unit = units[static_cast<int64_t>(b) * f.runs + u];
      bad = bad || unit != unit;
    }
    if (bad) y = plain_product(a, f, b, row, units[static_cast<int64_t>(a.batch) * f.runs + b]);
  }
  finish(a, f, y, b, row);
}

// More rows of x: kTiles x 16 weight rows and 16 batch rows a block, whose
// waves share the columns; x digits from the workspace.
template <int kGroup, int kTiles>
__global__ __launch_bounds__(kQ4Threads) void matvec_q4_rows_kernel(MatvecQ4Args a, Q4Form f) {
  __shared__ float sums[kQ4Waves][kManyTiles][kTiles][kWave];
  const int8_t* base = static_cast<const int8_t*>(a.workspace);
  const float* units = reinterpret_cast<const float*>(base + q4_units_offset(f.runs, a.batch));
  const int lane = threadIdx.x % kWave, g = lane / 16, col = lane % 16;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int row0 = blockIdx.x * kTiles * kQ4Tile, b0 = blockIdx.y * kManyTiles * kQ4Batch;
  const int operands = (a.batch + kQ4Batch - 1) / kQ4Batch;
  float y[kManyTiles][kTiles] = {};
  for (int run = wave; run < f.runs; run += kQ4Waves) {
    Run<kGroup> w[kTiles];
#pragma unroll
    for (int k = 0; k < kTiles; ++k)
      w[k] = load_run<kGroup>(a, f, min(row0 + k * kQ4Tile + col, a.rows - 1), run);
    // Operands past the last are read as the last and not stored.
    i32x4 x[kManyTiles][2];
    float unit[kManyTiles];
#pragma unroll
    for (int t = 0; t < kManyTiles; ++t) {
      const int o = min(b0 / kQ4Batch + t, operands - 1);
      const int8_t* d = base + (static_cast<int64_t>(o) * f.runs + run) * kQ4Operands + lane * 16;
      x[t][0] = *reinterpret_cast<const i32x4*>(d);
      x[t][1] = *reinterpret_cast<const i32x4*>(d + kQ4Operands / 2);
      unit[t] = units[static_cast<int64_t>(min(o * kQ4Batch + g, a.batch - 1)) * f.runs + run];
    }
#pragma unroll
    for (int t = 0; t < kManyTiles; ++t)
#pragma unroll
      for (int k = 0; k < kTiles; ++k) y[t][k] = fmaf(run_product<kGroup>(w[k], x[t][0], x[t][1]), unit[t], y[t][k]);
  }
#pragma unroll
  for (int t = 0; t < kManyTiles; ++t)
#pragma unroll
    for (int k = 0; k < kTiles; ++k) sums[wave][t][k][lane] = y[t][k];
  __syncthreads();
  for (int i = wave; i < kManyTiles * kTiles; i += kQ4Waves) {
    const int t = i / kTiles, k = i % kTiles, b = b0 + t * kQ4Batch + g, row = row0 + k * kQ4Tile + col;
    float total = sums[0][t][k][lane];
#pragma unroll
    for (int w = 1; w < kQ4Waves; ++w) total += sums[w][t][k][lane];
    finish_rows(a, f, units, total, b, row);
  }
}

// The same where there are tiles or batch rows enough: two tiles and 16 batch
// rows a group of f.share waves, which share the columns a chunk each in turn,
// codes through LDS (Chunk).  One chunk of a wave at a time: 16 waves a compute
// unit hide each other's waits.
template <int kGroup>
__global__ __launch_bounds__(kQ4Threads, 4) void matvec_q4_wide_rows_kernel(MatvecQ4Args a, Q4Form f) {
  constexpr int kTiles = kTilesOfWave;
  __shared__ __align__(16) int8_t shared[kQ4Waves * kTiles * kChunkBytes];  // chunks, then sums
  const int8_t* base = static_cast<const int8_t*>(a.workspace);
  const float* units = reinterpret_cast<const float*>(base + q4_units_offset(f.runs, a.batch));
  const int lane = threadIdx.x % kWave, g = lane / 16, col = lane % 16;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int part = wave % f.share, slot = wave / f.share, tiles = (a.rows + kQ4Tile - 1) / kQ4Tile;
  const int tile0 = (blockIdx.x * (kQ4Waves / f.share) + slot) * kTiles, b0 = blockIdx.y * kManyTiles * kQ4Batch;
  const int operands = (a.batch + kQ4Batch - 1) / kQ4Batch, chunks = (f.runs + kAhead - 1) / kAhead;
  const int8_t* const own = shared + wave * kTiles * kChunkBytes;
  const uint32_t own_at = __builtin_amdgcn_readfirstlane(lds_address(own));
  float y[kManyTiles][kTiles] = {};
  for (int chunk = part; chunk < chunks; chunk += f.share) {
    // Tiles past the last are read as the last and not stored.
#pragma unroll
    for (int k = 0; k < kTiles; ++k)
      Chunk<kGroup>::ask(a, f, min(tile0 + k, tiles - 1), chunk * kAhead, own_at + k * kChunkBytes);
    asm volatile("s_waitcnt vmcnt(0)" : : : "memory");
#pragma unroll 1
    for (int j = 0; j < min(kAhead, f.runs - chunk * kAhead); ++j) {
      const int run = chunk * kAhead + j;
      Run<kGroup> w[kTiles];
#pragma unroll
      for (int k = 0; k < kTiles; ++k) w[k] = Chunk<kGroup>::run(own + k * kChunkBytes, j);
      // Operands past the last are read as the last and not stored.
      i32x4 x[kManyTiles][2];
      float unit[kManyTiles];
#pragma unroll
      for (int t = 0; t < kManyTiles; ++t) {
        const int o = min(b0 / kQ4Batch + t, operands - 1);
        const int8_t* d = base + (static_cast<int64_t>(o) * f.runs + run) * kQ4Operands + lane * 16;
        x[t][0] = *reinterpret_cast<const i32x4*>(d);
        x[t][1] = *reinterpret_cast<const i32x4*>(d + kQ4Operands / 2);
        unit[t] = units[static_cast<int64_t>(min(o * kQ4Batch + g, a.batch - 1)) * f.runs + run];
      }
#pragma unroll
      for (int t = 0; t < kManyTiles; ++t)
#pragma unroll
        for (int k = 0; k < kTiles; ++k) y[t][k] = fmaf(run_product<kGroup>(w[k], x[t][0], x[t][1]), unit[t], y[t][k]);
    }
#pragma unroll
    for (int t = 0; t < kManyTiles; ++t)
#pragma unroll
      for (int k = 0; k < kTiles; ++k) asm volatile("" : "+v"(y[t][k]) : : "memory");  // the chunk is read
  }
  __syncthreads();
  float* const sums = reinterpret_cast<float*>(shared);  // [waves][batch tiles][tiles][lanes]
#pragma unroll
  for (int t = 0; t < kManyTiles; ++t)
#pragma unroll
    for (int k = 0; k < kTiles; ++k) sums[((wave * kManyTiles + t) * kTiles + k) * kWave + lane] = y[t][k];
  __syncthreads();
  for (int i = part; i < kManyTiles * kTiles; i += f.share) {
    const int t = i / kTiles, k = i % kTiles, b = b0 + t * kQ4Batch + g, row = (tile0 + k) * kQ4Tile + col;
    float total = 0.0f;
    for (int n = 0; n < f.share; ++n)
      total += sums[((slot * f.share + n) * kManyTiles * kTiles + i) * kWave + lane];
    finish_rows(a, f, units, total, b, row);
  }
}

bool fused_digits(int cols, int batch) {
  return batch <= kQ4Batch && batch * ((cols + kQ4Cols - 1) / kQ4Cols) <= kFusedRuns;
}

template <int kGroup>
void launch_q4(const MatvecQ4Args& a, const Q4Form& f, hipStream_t stream) {
  const int tiles = (a.rows + kQ4Tile - 1) / kQ4Tile;
  if (fused_digits(a.cols, a.batch)) {
    const size_t lds = static_cast<size_t>(f.runs + kAhead) * a.batch * 512;
    const bool few = f.runs * a.batch <= 2 * kQ4Waves;
    if (tiles < kManyRowTiles || !f.even) {
      if (few)
        matvec_q4_kernel<kGroup, 2><<<tiles, kQ4Threads, lds, stream>>>(a, f);
      else
        matvec_q4_kernel<kGroup, 8><<<tiles, kQ4Threads, lds, stream>>>(a, f);
    } else {
      const int at_once = kQ4Waves / f.share, blocks = std::min((tiles + at_once - 1) / at_once, kWideBlocks);
      const size_t more = lds + kQ4Waves * kRing * kChunkBytes;
      if (few)
        matvec_q4_wide_kernel<kGroup, 2><<<blocks, kQ4Threads, more, stream>>>(a, f);
      else
        matvec_q4_wide_kernel<kGroup, 8><<<blocks, kQ4Threads, more, stream>>>(a, f);
    }
    return;
  }
  const int many = (a.batch + kManyTiles * kQ4Batch - 1) / (kManyTiles * kQ4Batch);
  q4_digits_kernel<<<a.batch, kQ4Threads, 0, stream>>>(a, f);
  Q4Form wide = f;
  wide.share = 1;
  while (wide.share < kQ4Waves && wide.share * kAhead < f.runs) wide.share *= 2;
  const int at_once = kTilesOfWave * (kQ4Waves / wide.share), blocks = (tiles + at_once - 1) / at_once;
  if (f.even && static_cast<int64_t>(blocks) * many >= kWideRowsBlocks) {
    matvec_q4_wide_rows_kernel<kGroup><<<dim3(blocks, many), kQ4Threads, 0, stream>>>(a, wide);
  } else if (tiles >= kTwoTiles)
    matvec_q4_rows_kernel<kGroup, 2><<<dim3((tiles + 1) / 2, many), kQ4Threads, 0, stream>>>(a, f);
  else
    matvec_q4_rows_kernel<kGroup, 1><<<dim3(tiles, many), kQ4Threads, 0, stream>>>(a, f);
}

}  // namespace

int64_t matvec_q4_workspace(int cols, int batch) {
  if (fused_digits(cols, batch)) return 0;
  const int runs = (cols + kQ4Cols - 1) / kQ4Cols;
  return q4_units_offset(runs, batch) + 4 * (static_cast<int64_t>(batch) * runs + batch);
}

hipError_t launch_matvec_q4(const MatvecQ4Args& a, GemvPrologue pro, GemvEpilogue epi, hipStream_t stream) {
  Q4Form f;
  f.pro = pro;
  f.epi = epi;
  f.runs = (a.cols + kQ4Cols - 1) / kQ4Cols;
  f.groups = (a.cols + a.group - 1) / a.group;
  f.whole = a.cols % kQ4Cols == 0 && reinterpret_cast<uintptr_t>(a.scales) % 8 == 0;
  // As many as give every wave a tile, while each has a chunk.
  f.share = 1;
  while (f.share < kQ4Waves && f.share * kAhead < f.runs && (a.rows + kQ4Tile - 1) / kQ4Tile * f.share < kManyWaves)
    f.share *= 2;
  f.even = f.whole && f.groups % 2 == 0;
  switch (a.group) {
    case 32: launch_q4<32>(a, f, stream); break;
    case 64: launch_q4<64>(a, f, stream); break;
    case 128: launch_q4<128>(a, f, stream); break;
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

}  // namespace mmr
