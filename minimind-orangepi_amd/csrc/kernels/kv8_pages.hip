// kv8_pages.hip -- who has which page of the 8-bit paged cache.
//
// Forking: sequence i becomes the first keep[i] tokens of sequence parent[i],
// with room for room[i] more in pages that are its alone.  Compacting: the
// pages in use move to the lowest numbers.  All layers of a model have one
// table, so page numbers are found once and pages copied in every layer.
//
// users[p] counts the table entries (and what else the caller counts) that name
// page p; a page without any is free.  Counting up and down commutes, and new
// pages are the lowest free ones in the order of the sequences and their pages,
// so tables depend on no order of atomics.
#include "device_common.h"
#include "kv8_common.h"

#include <algorithm>
#include <climits>

namespace mmr {

namespace {

constexpr int kThreads = 256;
constexpr int kOneThreads = 1024;  // of a block that is alone
constexpr int kCopyThreads = 256;
constexpr int kCopyBlocks = 2048;

// ---------------------------------------------------------------- fork ----

// What a sequence is to be, checked; an invalid one becomes empty.
struct ForkPlan {
  int parent, keep, room;
  bool bad;
  __device__ __forceinline__ ForkPlan(const Kv8ForkArgs& a, int s) {
    parent = a.parent[s];
    keep = a.keep[s];
    room = a.room[s];
    bad = parent < -1 || parent >= a.seqs || keep < 0 || room < 0 ||
          static_cast<int64_t>(keep) + room > static_cast<int64_t>(a.per_seq) * kKv8Page;
    if (bad) room = 0;
    if (bad || parent < 0) {
      parent = -1;
      keep = 0;
    }
  }
  __device__ __forceinline__ int full() const { return keep / kKv8Page; }       // pages that are full of kept tokens
  __device__ __forceinline__ bool partly() const { return keep % kKv8Page != 0; }
  __device__ __forceinline__ int pages() const { return (keep + room + kKv8Page - 1) / kKv8Page; }
};

struct ForkSpace {
  int* taken;         // [seqs][per_seq] pages that a sequence takes over, or -1
  int* claim;         // [pages] one of the sequences that will write to this partly filled page
  int* first_writer;  // [seqs] of the page that this sequence claims
  int* writers;       // [seqs]
  int* copies;        // [seqs] page that the sequence copies its partly filled one from, or -1
  int* start;         // [seqs + 1] number of the sequence's first new page
  int* got;           // [min(pages, seqs * per_seq)] the new pages
  int* copy;          // [seqs][3] source, target, blocks
  int* counts;        // [2] new pages there were, copies
};
__host__ __device__ inline int64_t fork_layout(ForkSpace* f, int* p, int64_t seqs, int64_t per_seq, int64_t pages) {
  int64_t at = 0;
  auto take = [&](int64_t n) {
    int* mine = p ? p + at : nullptr;
    at += n;
    return mine;
  };
  f->taken = take(seqs * per_seq);
  f->claim = take(pages);
  f->first_writer = take(seqs);
  f->writers = take(seqs);
  f->copies = take(seqs);
  f->start = take(seqs + 1);
  f->got = take(pages < seqs * per_seq ? pages : seqs * per_seq);
  f->copy = take(3 * seqs);
  f->counts = take(2);
  return at;
}

// Counts: what each sequence takes over, against what it had.
__global__ __launch_bounds__(kThreads) void kv8_fork_count_kernel(Kv8ForkArgs a) {
  ForkSpace f;
  fork_layout(&f, a.workspace, a.seqs, a.per_seq, a.pages);
  const int tiles = (a.per_seq + kThreads - 1) / kThreads;
  const int s = blockIdx.x / tiles, place = blockIdx.x % tiles * kThreads + threadIdx.x;
  const ForkPlan plan(a, s);
  if (place >= a.per_seq) return;
  if (place == 0) {
    f.first_writer[s] = INT_MAX;
    f.writers[s] = 0;
    if (plan.bad) atomicOr(a.error, kKv8BadRows);
  }
  auto entry = [&](int seq) {
    const int p = a.table[static_cast<int64_t>(seq) * a.per_seq + place];
    return p >= 0 && p < a.pages ? p : -1;
  };
  const int had = entry(s);
  int takes = -1;
  const int64_t key = static_cast<int64_t>(place) * kKv8Page;
  if (plan.parent >= 0 && key < plan.keep) {
    // Behind the window of the row at position keep, and so of all later ones.
    const bool behind = a.window > 0 && key >= a.sinks && key + kKv8Page - 1 < plan.keep - a.window + 1;
    if (!behind) takes = entry(plan.parent);
    if (place == plan.full() && plan.partly() && takes < 0) atomicOr(a.error, kKv8BadRows);
  }
  f.taken[static_cast<int64_t>(s) * a.per_seq + place] = takes;
  if (had != takes) {
    if (had >= 0) atomicSub(a.users + had, 1);
    if (takes >= 0) atomicAdd(a.users + takes, 1);
  }
  if (takes >= 0 && place == plan.full() && plan.partly() && plan.room > 0) f.claim[takes] = s;  // any of them
}

// Exclusive sum over the block; *total has the sum.  Every thread calls it.
__device__ __forceinline__ int block_scan(int v, int* sh, int* total) {
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  int sum = v;
#pragma unroll
  for (int step = 1; step < kWave; step *= 2) {
    const int other = __shfl_up(sum, step);
    if (lane >= step) sum += other;
  }
  if (lane == kWave - 1) sh[wave] = sum;
  __syncthreads();
  int before = 0, all = 0;
  for (int w = 0; w < kOneThreads / kWave; ++w) {
    const int n = sh[w];
    if (w < wave) before += n;
    all += n;
  }
  __syncthreads();
  *total = all;
  return before + sum - v;
}

// Decides who copies, and finds the new pages.  One block.
__global__ __launch_bounds__(kOneThreads) void kv8_fork_decide_kernel(Kv8ForkArgs a) {
  __shared__ int sh[kOneThreads / kWave], sh_copies;
  ForkSpace f;
  fork_layout(&f, a.workspace, a.seqs, a.per_seq, a.pages);
  const int tid = threadIdx.x;
  if (tid == 0) sh_copies = 0;
  auto partly_filled = [&](const ForkPlan& plan, int s) {
    return plan.partly() ? f.taken[static_cast<int64_t>(s) * a.per_seq + plan.full()] : -1;
  };
  // Those who will write to a page agree on one of them, who counts them.
  for (int s = tid; s < a.seqs; s += kOneThreads) {
    const ForkPlan plan(a, s);
    const int p = partly_filled(plan, s);
    if (p >= 0 && plan.room > 0) {
      const int one = f.claim[p];
      atomicMin(f.first_writer + one, s);
      atomicAdd(f.writers + one, 1);
    }
  }
  __syncthreads();
  // The first of them keeps the page if nobody else has it.
  for (int s = tid; s < a.seqs; s += kOneThreads) {
    const ForkPlan plan(a, s);
    const int p = partly_filled(plan, s);
    int from = -1;
    if (p >= 0 && plan.room > 0) {
      const int one = f.claim[p];
      const bool keeps = a.users[p] == f.writers[one] && f.first_writer[one] == s;
      if (!keeps) from = p;
    }
    f.copies[s] = from;
  }
  __syncthreads();
  int wanted = 0;
  for (int base = 0; base < a.seqs; base += kOneThreads) {
    const int s = base + tid;
    int mine = 0;
    if (s < a.seqs) {
      const ForkPlan plan(a, s);
      const int from = f.copies[s];
      if (from >= 0) atomicSub(a.users + from, 1);
      const int kept = plan.full() + (plan.partly() && partly_filled(plan, s) >= 0 && from < 0 ? 1 : 0);
      mine = max(0, plan.pages() - kept);
    }
    int all;
    const int before = block_scan(mine, sh, &all);
    if (s < a.seqs) f.start[s] = wanted + before;
    wanted += all;
  }
  if (tid == 0) f.start[a.seqs] = wanted;
  // The lowest free pages.
  int got = 0;
  for (int base = 0; base < a.pages && got < wanted; base += 4 * kOneThreads) {
    const int p = base + 4 * tid;
    int n[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) n[i] = p + i < a.pages ? a.users[p + i] : 1;
    int mine = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) mine += n[i] <= 0;
    int all;
    int at = got + block_scan(mine, sh, &all);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (n[i] <= 0) {
        if (at < wanted) {
          f.got[at] = p + i;
          a.users[p + i] = 1;
        }
        ++at;
      }
    got = min(got + all, wanted);
  }
  __syncthreads();
  for (int s = tid; s < a.seqs; s += kOneThreads) {
    const int from = f.copies[s], number = f.start[s];
    if (from < 0 || number >= got) continue;
    const ForkPlan plan(a, s);
    int* c = f.copy + 3 * atomicAdd(&sh_copies, 1);
    c[0] = from;
    c[1] = f.got[number];
    c[2] = (plan.keep % kKv8Page + kKv8Block - 1) / kKv8Block;
  }
  __syncthreads();
  if (tid == 0) {
    f.counts[0] = got;
    f.counts[1] = sh_copies;
    if (got < wanted) atomicOr(a.error, kKv8NoPages);
  }
}

__global__ __launch_bounds__(kThreads) void kv8_fork_table_kernel(Kv8ForkArgs a) {
  ForkSpace f;
  fork_layout(&f, a.workspace, a.seqs, a.per_seq, a.pages);
  const int tiles = (a.per_seq + kThreads - 1) / kThreads;
  const int s = blockIdx.x / tiles, place = blockIdx.x % tiles * kThreads + threadIdx.x;
  if (place >= a.per_seq) return;
  const ForkPlan plan(a, s);
  const int64_t at = static_cast<int64_t>(s) * a.per_seq + place;
  const int start = f.start[s], end = f.start[s + 1], first_new = plan.pages() - (end - start);
  int p = f.taken[at];
  if (place >= first_new && place < plan.pages()) {
    const int number = start + place - first_new;
    p = number < f.counts[0] ? f.got[number] : -1;
  }
  a.table[at] = p;
}

// The first `blocks` blocks of a page of one layer, 16 bytes a thread.
__device__ __forceinline__ void copy_page(const Kv8Layers& l, int layer, int from, int to, int blocks) {
  const int64_t source = kv8_offset(from, 0, l.hkv, l.d), target = kv8_offset(to, 0, l.hkv, l.d);
  const int pieces = l.hkv * l.d * blocks;  // of keys, and of values
  for (int n = threadIdx.x; n < 2 * pieces; n += kCopyThreads) {
    const bool keys = n < pieces;
    const int m = keys ? n : n - pieces;
    int at;
    if (keys) {
      const int each = l.d * blocks;  // of a head
      at = m / each * (kKv8Page * l.d / 16) + m % each;
    } else {
      at = m / blocks * (kKv8Page / 16) + m % blocks;
    }
    int8_t* base = keys ? l.keys[layer] : l.values[layer];
    reinterpret_cast<uint4*>(base + target)[at] = reinterpret_cast<const uint4*>(base + source)[at];
  }
  for (int n = threadIdx.x; n < 2 * l.hkv * blocks; n += kCopyThreads) {
    const int head = n / (2 * blocks), m = n % (2 * blocks);
    int8_t* base = m < blocks ? l.key_exps[layer] : l.value_exps[layer];
    base[kv8_exp_offset(to, head, l.hkv) + m % blocks] = base[kv8_exp_offset(from, head, l.hkv) + m % blocks];
  }
}

__global__ __launch_bounds__(kCopyThreads) void kv8_copy_kernel(Kv8Layers l, const int* list, const int* count) {
  const int units = *count * l.count;
  for (int u = blockIdx.x; u < units; u += gridDim.x) {
    const int* c = list + 3 * (u / l.count);
    copy_page(l, u % l.count, c[0], c[1], c[2]);
  }
}

// ------------------------------------------------------------- compact ----

struct CompactSpace {
  int* copy;    // [pages / 2][3] source, target, blocks
  int* counts;  // [1] of them
};
__host__ __device__ inline int64_t compact_layout(CompactSpace* c, int* p, int64_t pages) {
  c->copy = p;
  c->counts = p ? p + 3 * (pages / 2) : nullptr;
  return 3 * (pages / 2) + 1;
}

// Pairs the k-th page in use from `live` on with the k-th hole below it.  One block.
__global__ __launch_bounds__(kOneThreads) void kv8_compact_decide_kernel(Kv8CompactArgs a) {
  __shared__ int sh[kOneThreads / kWave];
  CompactSpace c;
  compact_layout(&c, a.workspace, a.pages);
  const int tid = threadIdx.x;
  int mine = 0, live, unused;
  for (int p = tid; p < a.pages; p += kOneThreads) mine += a.users[p] > 0;
  block_scan(mine, sh, &live);
  int holes = 0, movers = 0;
  for (int base = 0; base < a.pages; base += kOneThreads) {
    const int p = base + tid;
    const int n = p < a.pages ? a.users[p] : 0;
    const bool hole = p < a.pages && p < live && n <= 0, mover = p >= live && n > 0;
    const int hole_at = holes + block_scan(hole, sh, &unused);
    holes += unused;
    const int mover_at = movers + block_scan(mover, sh, &unused);
    movers += unused;
    if (hole) c.copy[3 * hole_at + 1] = p;
    if (mover) {
      c.copy[3 * mover_at] = p;
      c.copy[3 * mover_at + 2] = kKv8Blocks;
    }
    if (p < a.pages) {
      a.moved[p] = n > 0 ? p : -1;
      if (p < live) a.users_out[p] = max(n, 0);
    }
  }
  __syncthreads();
  for (int k = tid; k < movers; k += kOneThreads) {
    const int from = c.copy[3 * k], to = c.copy[3 * k + 1];
    a.moved[from] = to;
    a.users_out[to] = a.users[from];
  }
  __syncthreads();
  for (int p = live + tid; p < a.pages; p += kOneThreads) a.users_out[p] = 0;
  if (tid == 0) {
    *c.counts = movers;
    *a.live = live;
  }
}

__global__ __launch_bounds__(kThreads) void kv8_compact_table_kernel(Kv8CompactArgs a) {
  const int64_t at = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (at >= static_cast<int64_t>(a.seqs) * a.per_seq) return;
  const int p = a.table[at];
  a.table_out[at] = p >= 0 && p < a.pages ? a.moved[p] : -1;
}

hipError_t launch_copies(const Kv8Layers* layers, int groups, const int* list, const int* count, int64_t most,
                         hipStream_t stream) {
  for (int g = 0; g < groups; ++g) {
    const int64_t blocks = std::min<int64_t>(kCopyBlocks, most * layers[g].count);
    if (blocks > 0) kv8_copy_kernel<<<dim3(blocks), kCopyThreads, 0, stream>>>(layers[g], list, count);
  }
  return hipGetLastError();
}

}  // namespace

int64_t kv8_fork_workspace(int64_t seqs, int64_t per_seq, int64_t pages) {
  ForkSpace f;
  return fork_layout(&f, nullptr, seqs, per_seq, pages) * static_cast<int64_t>(sizeof(int));
}

hipError_t launch_kv8_fork(const Kv8ForkArgs& a, const Kv8Layers* layers, int groups, hipStream_t stream) {
  ForkSpace f;
  fork_layout(&f, a.workspace, a.seqs, a.per_seq, a.pages);
  const int blocks = a.seqs * ((a.per_seq + kThreads - 1) / kThreads);
  kv8_fork_count_kernel<<<dim3(blocks), kThreads, 0, stream>>>(a);
  kv8_fork_decide_kernel<<<dim3(1), kOneThreads, 0, stream>>>(a);
  kv8_fork_table_kernel<<<dim3(blocks), kThreads, 0, stream>>>(a);
  return launch_copies(layers, groups, f.copy, f.counts + 1, a.seqs, stream);
}

int64_t kv8_compact_workspace(int64_t pages) {
  CompactSpace c;
  return compact_layout(&c, nullptr, pages) * static_cast<int64_t>(sizeof(int));
}

hipError_t launch_kv8_compact(const Kv8CompactArgs& a, const Kv8Layers* layers, int groups, hipStream_t stream) {
  CompactSpace c;
  compact_layout(&c, a.workspace, a.pages);
  kv8_compact_decide_kernel<<<dim3(1), kOneThreads, 0, stream>>>(a);
  const int64_t entries = static_cast<int64_t>(a.seqs) * a.per_seq;
  kv8_compact_table_kernel<<<dim3((entries + kThreads - 1) / kThreads), kThreads, 0, stream>>>(a);
  return launch_copies(layers, groups, c.copy, c.counts, a.pages / 2, stream);
}

}  // namespace mmr
