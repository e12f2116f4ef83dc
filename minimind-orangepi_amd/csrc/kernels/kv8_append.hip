// kv8_append.hip -- QKV rows into the 8-bit paged cache.
//
// For row i of sequence s at position t = context[s] + i:
//   q, k heads:  x <- x * w / sqrt(mean(x^2) + eps)          (where norms are given)
//                (x_j, x_{j + d/2}) <- rotation by t * theta^(-2j/d)
//   block of 16: e = least exponent with max |x| <= 127 * 2^e over its new rows,
//                and at least the exponent that its earlier rows have;
//                earlier codes <- rint(code * 2^(e_old - e)), code <- rint(x * 2^-e)
//
// The codes are fixed by these formulas to the last bit, whatever the launch
// looks like: everything up to the code is computed in fp64 (its error, some
// 2^-50, moves a value across a rounding border once in 10^13), and scaling by
// a power of two is exact.  fp64 costs nothing here: the vector units run its
// FMAs at the fp32 rate without packed math, and the kernel waits on memory.
// The angle is an integer product: turns[j] is theta^(-2j/d) / 2 pi turns a
// position in units of 2^-64, and t * turns[j] modulo 2^64 is the fraction of
// a turn, exact to t * 2^-65 at any position, with no range reduction.
//
// One workgroup owns one 16-token block of one sequence, all heads: it is the
// only one that touches the block's codes and exponents, so a partly filled
// block is read, moved to a larger exponent and written back without atomics.
// Four lanes share a row of a head (a quarter of each half each), so a wave
// holds 16 rows: a block of one head, whose maximum is a wave reduction.  The
// block's queries are other workgroups', which need nothing but the angles.
//
// Measured in replayed graphs (8 + 2 + 2 heads; medians of graphs of 30 calls
// over three sets of inputs): one row of d 96 4.9 us, 1.6 of them any kernel's
// there, the rest a chain of three loads, the sine and two reductions; 2,690
// rows of d 128 in five sequences 11.5 us, 27.4 MB at 2.4 TB/s: its waves wait
// on counters 59 % of their time, in one pass each.  Angles of rows 1 to 15 of a
// block from a table of fixed turns instead of sines of their own changed
// nothing (12.0 and 12.4 us a launch in a kernel trace).
#include "device_common.h"
#include "kv8_common.h"

#include <algorithm>

namespace mmr {

namespace {

constexpr int kAppendThreads = 256;

template <int kCtrl>
__device__ __forceinline__ double dpp_move_double(double v) {
  return __hiloint2double(dpp_move_int<kCtrl>(__double2hiint(v)), dpp_move_int<kCtrl>(__double2loint(v)));
}
__device__ __forceinline__ double quad_sum(double v) {
  v += dpp_move_double<dpp::kQuadXor1>(v);
  return v + dpp_move_double<dpp::kQuadXor2>(v);
}

// Of small whole numbers.
__device__ __forceinline__ int wave_max(int v) { return static_cast<int>(group_max<kWave>(static_cast<float>(v))); }

// 2^n for |n| <= 1000.
__device__ __forceinline__ double pow2(int n) { return __longlong_as_double(static_cast<long long>(1023 + n) << 52); }

// The least e with top <= 127 * 2^e, in [kKv8MinExp, kKv8MaxExp].
__device__ __forceinline__ int exponent_for(double top) {
  if (!(top > 0.0)) return kKv8MinExp;
  int x;
  const double m = frexp(top, &x);
  const int e = x - 7 + (m > 127.0 / 128.0 ? 1 : 0);
  return min(max(e, kKv8MinExp), kKv8MaxExp);
}

// A quarter of a head's row: dimensions 16 c + 4 j + i and d/2 + 16 c + 4 j + i.
template <int D>
struct Quarter {
  static constexpr int kChunks = D / 32;
  double a[kChunks][4], b[kChunks][4];

  struct Raw {
    float4 lo[kChunks], hi[kChunks];
    __device__ __forceinline__ void load(const float* p, int j, bool there) {
#pragma unroll
      for (int c = 0; c < kChunks; ++c) {
        lo[c] = hi[c] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (there) {
          lo[c] = *reinterpret_cast<const float4*>(p + 16 * c + 4 * j);
          hi[c] = *reinterpret_cast<const float4*>(p + D / 2 + 16 * c + 4 * j);
        }
      }
    }
  };
  __device__ __forceinline__ explicit Quarter(const Raw& r) {
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      a[c][0] = r.lo[c].x, a[c][1] = r.lo[c].y, a[c][2] = r.lo[c].z, a[c][3] = r.lo[c].w;
      b[c][0] = r.hi[c].x, b[c][1] = r.hi[c].y, b[c][2] = r.hi[c].z, b[c][3] = r.hi[c].w;
    }
  }
  // All four lanes of the row take part.
  __device__ __forceinline__ void normalise(const float* w, double eps, int j) {
    double sum = 0.0;
#pragma unroll
    for (int c = 0; c < kChunks; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) sum += a[c][i] * a[c][i] + b[c][i] * b[c][i];
    const double scale = 1.0 / sqrt(quad_sum(sum) / D + eps);
#pragma unroll
    for (int c = 0; c < kChunks; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        a[c][i] *= scale * w[16 * c + 4 * j + i];
        b[c][i] *= scale * w[D / 2 + 16 * c + 4 * j + i];
      }
  }
  // cs: (cos, sin) of the row's position, one pair a dimension of the first half.
  __device__ __forceinline__ void rotate(const double2* cs, int j) {
#pragma unroll
    for (int c = 0; c < kChunks; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const double2 r = cs[16 * c + 4 * j + i];
        const double x = a[c][i], y = b[c][i];
        a[c][i] = x * r.x - y * r.y;
        b[c][i] = y * r.x + x * r.y;
      }
  }
  // Largest finite magnitude; *bad where a value is not finite.
  __device__ __forceinline__ double top(bool* bad) const {
    double t = 0.0;
#pragma unroll
    for (int c = 0; c < kChunks; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const double x = fabs(a[c][i]), y = fabs(b[c][i]);
        const bool fx = x < __builtin_inf(), fy = y < __builtin_inf();
        *bad = *bad || !fx || !fy;
        if (fx) t = fmax(t, x);
        if (fy) t = fmax(t, y);
      }
    return t;
  }
};

// rint(x * 2^-e) in [-127, 127]: only infinities need the limit; NaN is 0.
__device__ __forceinline__ int code_of(double x, double scale) {
  const double v = rint(x * scale);
  return v == v ? static_cast<int>(fmin(fmax(v, -127.0), 127.0)) : 0;
}

// Four codes moved to an exponent larger by `shift`.
__device__ __forceinline__ uint32_t moved(uint32_t codes, float scale) {
  uint32_t out = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int c = static_cast<int>(codes << (24 - 8 * i)) >> 24;
    out |= (static_cast<uint32_t>(static_cast<int>(rintf(static_cast<float>(c) * scale))) & 0xFF) << (8 * i);
  }
  return out;
}

// blockIdx.z 0 appends the block's keys and values, the others rotate a share
// of its queries.  Everything that does not wait for the angles is asked for
// before they are computed.
template <int D>
__global__ __launch_bounds__(kAppendThreads) void kv8_append_kernel(Kv8AppendArgs a) {
  constexpr int kHalf = D / 2, kChunks = D / 32, kWaves = kAppendThreads / kWave, kGroups = kAppendThreads / 4;
  __shared__ double2 turn[kKv8Block][kHalf];
  __shared__ __align__(16) int8_t tile[kWaves][D][kKv8Block];
  const int s = blockIdx.y, tid = threadIdx.x;
  Kv8Span span;
  const bool fine = kv8_span(a.cache, a.offsets, a.context, s, a.rows, a.max_rows, &span);
  const bool known = fine && (span.n == 0 || static_cast<int64_t>(span.context) + span.n <= a.max_positions);
  if (!known) {
    if (blockIdx.x == 0 && blockIdx.z == 0 && tid == 0) atomicOr(a.error, kKv8BadRows);
    return;
  }
  const int block = span.context / kKv8Block + blockIdx.x;
  const int lo = max(span.context, block * kKv8Block), hi = min(span.context + span.n, (block + 1) * kKv8Block);
  if (lo >= hi) return;
  const int page = a.cache.table[static_cast<int64_t>(s) * a.cache.per_seq + block / kKv8Blocks];
  const int fresh = lo - block * kKv8Block, end = hi - block * kKv8Block;  // slots [fresh, end) are new
  const int first_row = span.first + (lo - span.context);                  // of slot `fresh`
  const int hq = a.hq, hkv = a.cache.hkv, j = tid & 3;
  const int64_t stride = static_cast<int64_t>(hq + 2 * hkv) * D;

  // What this thread's four lanes work on first.  Queries: (row, head) items.
  // Keys and values: a wave each (K or V, head), lanes 4 i .. 4 i + 3 slot i.
  const int wave = tid / kWave, lane = tid % kWave, slot = lane / 4;
  const bool mine = slot >= fresh && slot < end;
  const int items = (end - fresh) * hq;
  int it = blockIdx.z == 0 ? wave : (blockIdx.z - 1) * kGroups + tid / 4;
  typename Quarter<D>::Raw raw;
  auto load_query = [&]() {
    const int r = it / hq, h = it - r * hq;
    raw.load(a.qkv + (first_row + r) * stride + h * D, j, it < items);
  };
  auto load_cached = [&]() {
    raw.load(a.qkv + (first_row + slot - fresh) * stride + static_cast<int64_t>(hq + it) * D, j,
             mine && it < 2 * hkv);
  };
  if (blockIdx.z == 0)
    load_cached();
  else if (it < items)
    load_query();
  for (int i = tid; i < (end - fresh) * kHalf; i += kAppendThreads) {
    const int r = i / kHalf, d = i - r * kHalf;
    const uint64_t t = static_cast<uint64_t>(lo + r) * a.turns[d];
    double sn, cs;
    sincospi(static_cast<double>(static_cast<int64_t>(t)) * 0x1p-63, &sn, &cs);
    turn[fresh + r][d] = make_double2(cs, sn);
  }
  if (page < 0 || page >= a.cache.pages) {
    if (tid == 0) atomicOr(a.error, kKv8BadRows);
    return;
  }
  __syncthreads();

  if (blockIdx.z > 0) {
    for (; it < items; it += kGroups * (gridDim.z - 1)) {
      const int r = it / hq, h = it - r * hq;
      Quarter<D> x(raw);
      if (a.q_norm) x.normalise(a.q_norm, a.eps, j);
      x.rotate(turn[fresh + r], j);
      float* out = a.query + (static_cast<int64_t>(first_row + r) * hq + h) * D;
#pragma unroll
      for (int c = 0; c < kChunks; ++c) {
        *reinterpret_cast<float4*>(out + 16 * c + 4 * j) = make_float4(x.a[c][0], x.a[c][1], x.a[c][2], x.a[c][3]);
        *reinterpret_cast<float4*>(out + kHalf + 16 * c + 4 * j) =
            make_float4(x.b[c][0], x.b[c][1], x.b[c][2], x.b[c][3]);
      }
      it += kGroups * (gridDim.z - 1);
      if (it < items) load_query();
      it -= kGroups * (gridDim.z - 1);
    }
    return;
  }
  for (; it < 2 * hkv; it += kWaves) {
    const bool is_key = it < hkv;
    const int h = is_key ? it : it - hkv;
    int8_t* exps = (is_key ? a.cache.key_exps : a.cache.value_exps) + kv8_exp_offset(page, h, hkv) + block % kKv8Blocks;
    int8_t* codes = (is_key ? a.cache.keys : a.cache.values) + kv8_offset(page, h, hkv, D);
    const int held = fresh > 0 ? *exps : kKv8MinExp;
    Quarter<D> x(raw);
    if (is_key) {
      if (a.k_norm) x.normalise(a.k_norm, a.eps, j);
      if (mine) x.rotate(turn[slot], j);
    }
    bool bad = false;
    int e = exponent_for(x.top(&bad));
    if (!mine) e = kKv8MinExp, bad = false;
    e = wave_max(e);
    if (bad) atomicOr(a.error, kKv8NotFinite);
    const int grown = fresh > 0 ? max(0, e - held) : 0;  // earlier rows shift by this
    if (fresh > 0) e = max(e, held);
    const float shrink = ldexpf(1.0f, -grown);
    const double scale = pow2(-e);
    if (lane == 0) *exps = static_cast<int8_t>(e);
    if (is_key) {
      int8_t* row = codes + (block % kKv8Blocks * kKv8Block + slot) * D;
      if (mine) {
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
          uint32_t p = 0, q = 0;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            p |= (code_of(x.a[c][i], scale) & 0xFF) << (8 * i);
            q |= (code_of(x.b[c][i], scale) & 0xFF) << (8 * i);
          }
          *reinterpret_cast<uint32_t*>(row + 16 * c + 4 * j) = p;
          *reinterpret_cast<uint32_t*>(row + kHalf + 16 * c + 4 * j) = q;
        }
      } else if (slot < fresh && grown > 0) {
#pragma unroll
        for (int c = 0; c < 2 * kChunks; ++c) {
          uint32_t* w = reinterpret_cast<uint32_t*>(row + 16 * c + 4 * j);
          *w = moved(*w, shrink);
        }
      }
    } else {
      if (mine) {
#pragma unroll
        for (int c = 0; c < kChunks; ++c)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            tile[wave][16 * c + 4 * j + i][slot] = static_cast<int8_t>(code_of(x.a[c][i], scale));
            tile[wave][kHalf + 16 * c + 4 * j + i][slot] = static_cast<int8_t>(code_of(x.b[c][i], scale));
          }
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
      for (int dim = lane; dim < D; dim += kWave) {
        uint4* at = reinterpret_cast<uint4*>(codes + dim * kKv8Page + block % kKv8Blocks * kKv8Block);
        const uint4 fill = *reinterpret_cast<const uint4*>(tile[wave][dim]);
        uint32_t v[4] = {fill.x, fill.y, fill.z, fill.w};
        if (end - fresh < kKv8Block) {  // slots outside [fresh, end) keep what they hold
          const uint4 was = *at;
          const uint32_t w[4] = {was.x, was.y, was.z, was.w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t older = grown > 0 ? moved(w[i], shrink) : w[i];
            uint32_t o = 0;
#pragma unroll
            for (int b = 0; b < 4; ++b) {
              const int t = 4 * i + b;
              o |= (t < fresh ? older : t < end ? v[i] : w[i]) & (0xFFu << (8 * b));
            }
            v[i] = o;
          }
        }
        *at = make_uint4(v[0], v[1], v[2], v[3]);
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
    }
    it += kWaves;
    load_cached();
    it -= kWaves;
  }
}

}  // namespace

hipError_t launch_kv8_append(const Kv8AppendArgs& a, hipStream_t stream) {
  // Rows that start anywhere in a block reach into this many blocks; of a full
  // one, a thread group takes one query row of one head.
  const int shares = (std::min(a.max_rows, kKv8Block) * a.hq + kAppendThreads / 4 - 1) / (kAppendThreads / 4);
  const dim3 grid((a.max_rows + 2 * (kKv8Block - 1)) / kKv8Block, a.cache.seqs, 1 + shares);
  switch (a.cache.d) {
    case 32: kv8_append_kernel<32><<<grid, kAppendThreads, 0, stream>>>(a); break;
    case 64: kv8_append_kernel<64><<<grid, kAppendThreads, 0, stream>>>(a); break;
    case 96: kv8_append_kernel<96><<<grid, kAppendThreads, 0, stream>>>(a); break;
    case 128: kv8_append_kernel<128><<<grid, kAppendThreads, 0, stream>>>(a); break;
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

}  // namespace mmr
