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
//
// Times in this file are us a call in replayed graphs (medians of graphs of 30
// calls over three sets of inputs; a kernel that does nothing takes 1.6 there).
#include "device_common.h"
#include "kv8_common.h"

#include <algorithm>
#include <climits>
#include <type_traits>

namespace mmr {

namespace {

constexpr int kThreads = 256, kWaves = kThreads / kWave;
constexpr int kOneThreads = 1024;    // of a block that is alone
constexpr int kHeldSeqs = 2048;      // sequences whose plans a deciding block holds in LDS
constexpr int kHeldPages = 16;       // pages of a pool that one block decides over, a thread
constexpr int kOnePages = kOneThreads * kHeldPages;
constexpr int kChunk = 1024;         // pages that a wave counts, in larger pools
constexpr int kCountEntries = 1280;  // table entries that a deciding block counts itself
constexpr int kCopyBlocks = 16384;

__host__ __device__ inline int chunks_of(int64_t pages) { return static_cast<int>((pages + kChunk - 1) / kChunk); }

// Users of pages p .. p + 3; of those past the pool, `past`.
__device__ __forceinline__ int4 users_at(const int32_t* users, int p, int pages, int past) {
  if (p + 4 <= pages) return *reinterpret_cast<const int4*>(users + p);
  int4 n = make_int4(past, past, past, past);
  if (p < pages) n.x = users[p];
  if (p + 1 < pages) n.y = users[p + 1];
  if (p + 2 < pages) n.z = users[p + 2];
  return n;
}
__device__ __forceinline__ int used_of(const int4& n) { return (n.x > 0) + (n.y > 0) + (n.z > 0) + (n.w > 0); }

// v and the sum of those lanes before it: shifts within rows of 16 lanes, then
// the last lane of a row (and of two) handed to those after it.
template <int kCtrl, int kRows>
__device__ __forceinline__ int lane_before(int v) {
  return __builtin_amdgcn_update_dpp(0, v, kCtrl, kRows, 0xF, false);
}
__device__ __forceinline__ int wave_scan(int v) {
  v += lane_before<0x111, 0xF>(v);  // row_shr 1, 2, 4, 8
  v += lane_before<0x112, 0xF>(v);
  v += lane_before<0x114, 0xF>(v);
  v += lane_before<0x118, 0xF>(v);
  v += lane_before<0x142, 0xA>(v);  // row_bcast 15 to the second and fourth row
  return v + lane_before<0x143, 0xC>(v);  // row_bcast 31 to the third and fourth
}

// Exclusive sum over a block of kOneThreads; *total has the sum.  Every thread calls it.
__device__ __forceinline__ int block_scan(int v, int* sh, int* total) {
  constexpr int kOneWaves = kOneThreads / kWave;
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const int sum = wave_scan(v);
  if (lane == kWave - 1) sh[wave] = sum;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kOneWaves; ++w) {
    const int n = sh[w];
    if (w < wave) before += n;
    all += n;
  }
  __syncthreads();
  *total = all;
  return before + sum - v;
}

// Pages in use of each chunk of a large pool, a wave a chunk.
__global__ __launch_bounds__(kThreads) void kv8_count_used_kernel(const int32_t* users, int pages, int* used) {
  const int chunk = blockIdx.x * kWaves + threadIdx.x / kWave, lane = threadIdx.x % kWave;
  if (chunk >= chunks_of(pages)) return;
  int mine = 0;
#pragma unroll
  for (int j = 0; j < kChunk / kWave / 4; ++j)
    mine += used_of(users_at(users, chunk * kChunk + 4 * (lane + kWave * j), pages, 0));
  const int sum = wave_scan(mine);
  if (lane == kWave - 1) used[chunk] = sum;
}

// ---------------------------------------------------------------- fork ----

// What a sequence is to be, checked; an invalid one becomes empty.
struct ForkPlan {
  int parent, keep, room;
  bool bad;
  __device__ __forceinline__ ForkPlan(const Kv8ForkArgs& a, int s) {
    parent = a.parent[s];
    keep = a.keep[s];
    room = a.room[s];
    if (parent == -1) keep = 0;  // of nobody, whatever it says
    // No branches: the three loads are under way together.
    bad = (parent < -1) | (parent >= a.seqs) | (keep < 0) | (room < 0) |
          (static_cast<int64_t>(keep) + room > static_cast<int64_t>(a.per_seq) * kKv8Page);
    if (bad) {
      parent = -1;
      keep = room = 0;
    }
  }
  __device__ __forceinline__ int full() const { return keep / kKv8Page; }       // pages that are full of kept tokens
  __device__ __forceinline__ bool partly() const { return keep % kKv8Page != 0; }
  __device__ __forceinline__ int pages() const { return (keep + room + kKv8Page - 1) / kKv8Page; }
};

// Of a sequence, while the block decides; in LDS, or in the workspace where there are many.
struct ForkSeq {
  int page, users;   // that it will write to, and its users
  int one;           // of the sequences that will write to it, all name the same
  int first_writer;  // of those that name this sequence, the first, and how many
  int writers;
};

// What becomes of a sequence's table row: places from `fresh` to `pages` get new
// pages, from number `start` of those on (before that is known: the blocks that a
// copy would have).  `page` is a partly filled one that it will write to, or -1.
struct __attribute__((aligned(16))) ForkRow {
  int fresh, pages, start, page;
};
struct ForkSpace {
  ForkRow* row;   // [seqs]
  int* taken;     // [seqs][per_seq] pages that a sequence takes over, or -1
  int* claim;     // [pages] one of the sequences that will write to this partly filled page
  int* got;       // [min(pages, seqs * per_seq)] the new pages
  int* copy;      // [seqs][3] source, target, blocks
  int* counts;    // [2] new pages that there were, copies
  int* used;      // [chunks] of a large pool: pages in use of each
  ForkSeq* seq;   // [seqs] or nothing
};
__host__ __device__ inline int64_t fork_layout(ForkSpace* f, int* p, int64_t seqs, int64_t per_seq, int64_t pages) {
  int64_t at = 0;
  auto take = [&](int64_t n) {
    int* mine = p ? p + at : nullptr;
    at += n;
    return mine;
  };
  f->row = reinterpret_cast<ForkRow*>(take(4 * seqs));
  f->taken = take(seqs * per_seq);
  f->claim = take(pages);
  f->got = take(pages < seqs * per_seq ? pages : seqs * per_seq);
  f->copy = take(3 * seqs);
  f->counts = take(2);
  f->used = take(pages > kOnePages ? chunks_of(pages) : 0);
  f->seq = reinterpret_cast<ForkSeq*>(take(seqs > kHeldSeqs ? 5 * seqs : 0));
  return at;
}

// What sequence s takes over at a place of its row, against what it had there.
__device__ __forceinline__ void count_entry(const Kv8ForkArgs& a, const ForkSpace& f, int s, int place) {
  const ForkPlan plan(a, s);
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
  if (place == 0 && plan.bad) atomicOr(a.error, kKv8BadRows);
  if (place == (plan.partly() ? plan.full() : 0)) {
    const bool partly = plan.partly() && takes >= 0, writes = partly && plan.room > 0;
    f.row[s] = ForkRow{plan.full() + partly, plan.pages(), (plan.keep % kKv8Page + kKv8Block - 1) / kKv8Block,
                       writes ? takes : -1};
    if (writes) f.claim[takes] = s;  // any of them
  }
}
__global__ __launch_bounds__(kThreads) void kv8_fork_count_kernel(Kv8ForkArgs a) {
  ForkSpace f;
  fork_layout(&f, a.workspace, a.seqs, a.per_seq, a.pages);
  const int tiles = (a.per_seq + kThreads - 1) / kThreads;
  const int s = blockIdx.x / tiles, place = blockIdx.x % tiles * kThreads + threadIdx.x;
  if (place < a.per_seq) count_entry(a, f, s, place);
}

// Decides who copies, and finds the new pages: one block, a sequence a thread.
// What it takes (4.1 of 7.7 for four beams of 777 tokens) is a chain of dependent
// loads (rows, who claims their pages and those pages' users) and two sums over
// the block, so all else is held, or asked for ahead.
template <bool kCount>
__global__ __launch_bounds__(kOneThreads) void kv8_fork_decide_kernel(Kv8ForkArgs a) {
  __shared__ int sh[kOneThreads / kWave], sh_copies, sh_list;
  __shared__ ForkSeq held[kHeldSeqs];
  __shared__ int2 list[kOneThreads];  // chunks with free pages, and the number of their first
  ForkSpace f;
  fork_layout(&f, a.workspace, a.seqs, a.per_seq, a.pages);
  ForkSeq* const seq = a.seqs <= kHeldSeqs ? held : f.seq;
  const int tid = threadIdx.x;
  if (tid == 0) sh_copies = 0;
  for (int s = tid; s < a.seqs; s += kOneThreads) seq[s].first_writer = INT_MAX, seq[s].writers = 0;
  if constexpr (kCount) {
    for (int n = tid; n < a.seqs * a.per_seq; n += kOneThreads) {
      const int s = n / a.per_seq;
      count_entry(a, f, s, n - s * a.per_seq);
    }
  }
  __syncthreads();
  // Which pages are free no longer changes: a page that is copied from stays in use.
  int4 users = users_at(a.users, 4 * tid, a.pages, 1);
  // Those who will write to a page agree on one of them, who counts them.
  ForkRow first_row = {};  // of sequence tid
  for (int s = tid; s < a.seqs; s += kOneThreads) {
    const ForkRow row = f.row[s];
    if (s == tid) first_row = row;
    seq[s].page = row.page;
    if (row.page >= 0) {
      const int one = f.claim[row.page];
      seq[s].users = a.users[row.page];
      seq[s].one = one;
      atomicMin(&seq[one].first_writer, s);
      atomicAdd(&seq[one].writers, 1);
    }
  }
  __syncthreads();
  // The first of them keeps the page if nobody else has it.  Copies are noted with
  // the number of their new page, which is found after.
  int wanted = 0;
  for (int base = 0; base < a.seqs; base += kOneThreads) {
    const int s = base + tid;
    int mine = 0;
    ForkRow row = {};
    bool copies = false;
    if (s < a.seqs) {
      row = base == 0 ? first_row : f.row[s];
      if (seq[s].page >= 0) {
        const int one = seq[s].one;
        copies = seq[s].users != seq[one].writers || seq[one].first_writer != s;
        if (copies) {
          atomicSub(a.users + seq[s].page, 1);
          --row.fresh;
        }
      }
      mine = max(0, row.pages - row.fresh);
    }
    int all;
    const int before = block_scan(mine, sh, &all);
    if (s < a.seqs) {
      if (copies) {
        int* c = f.copy + 3 * atomicAdd(&sh_copies, 1);
        c[0] = seq[s].page;
        c[1] = wanted + before;
        c[2] = row.start;
      }
      row.start = wanted + before;
      f.row[s] = row;
    }
    wanted += all;
  }
  // The lowest free pages: of pages p .. p + 3 with these users, numbers from `at`
  // on (no more than there are pages, whatever the users say).
  const int most = min(wanted, a.pages);
  auto give = [&](int p, const int4& n, int at) {
    const int of[4] = {n.x, n.y, n.z, n.w};
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (of[i] <= 0) {
        if (at < most) {
          f.got[at] = p + i;
          a.users[p + i] = 1;
        }
        ++at;
      }
  };
  int got = 0;
  if (a.pages <= kOnePages) {
    for (int p = 4 * tid; p - 4 * tid < a.pages && got < wanted; p += 4 * kOneThreads) {
      if (p >= 4 * kOneThreads) users = users_at(a.users, p, a.pages, 1);
      int all;
      const int before = block_scan(4 - used_of(users), sh, &all);
      give(p, users, got + before);
      got = min(got + all, wanted);
    }
  } else {  // the chunks that have some are known
    const int chunks = chunks_of(a.pages), wave = tid / kWave, lane = tid % kWave;
    for (int base = 0; base < chunks && got < wanted; base += kOneThreads) {
      const int c = base + tid;
      const int mine = c < chunks ? min(kChunk, a.pages - c * kChunk) - f.used[c] : 0;
      if (tid == 0) sh_list = 0;
      int all;
      const int before = block_scan(mine, sh, &all);
      if (mine > 0 && got + before < most) {
        const int n = atomicAdd(&sh_list, 1);
        list[n] = make_int2(c, got + before);
      }
      __syncthreads();
      for (int n = wave; n < sh_list; n += kOneThreads / kWave) {
        int at = list[n].y;
#pragma unroll
        for (int j = 0; j < kChunk / kWave / 4; ++j) {
          const int p = list[n].x * kChunk + 4 * (lane + kWave * j);
          const int4 of = users_at(a.users, p, a.pages, 1);
          const int sum = wave_scan(4 - used_of(of));
          give(p, of, at + sum - (4 - used_of(of)));
          at += __builtin_amdgcn_readlane(sum, kWave - 1);
        }
      }
      got = min(got + all, wanted);
      __syncthreads();
    }
  }
  if (tid == 0) {
    f.counts[0] = got;
    f.counts[1] = sh_copies;
    if (got < wanted) atomicOr(a.error, kKv8NoPages);
  }
}

// The keys or values of the blocks [0, kBlocks) of every head of a page; all
// blocks lie together.  Memory bounds it where there is much to copy: 5,000 pages
// of which 2,500 are in use, 8 layers, 326 MB in 68.5, 4.8 TB/s (a large copy on
// this card: 4.8).  Stores go past the caches (72 to 76 without, in a state of
// its own); one piece a thread at a time is as fast as several under way.
template <int D, int kBlocks>
__device__ __forceinline__ void copy_codes(int8_t* base, bool keys, int64_t source, int64_t target, int hkv) {
  const int pieces = hkv * D * kBlocks;
  const i32x4* from = reinterpret_cast<const i32x4*>(base + source);
  i32x4* to = reinterpret_cast<i32x4*>(base + target);
  for (int n = threadIdx.x; n < pieces; n += kThreads) {
    // Keys: [head][block][D] pieces of a token; values: [head][D][block].
    const int at = kBlocks == kKv8Blocks ? n
                   : keys                ? n / (D * kBlocks) * (kKv8Blocks * D) + n % (D * kBlocks)
                                         : n / kBlocks * kKv8Blocks + n % kBlocks;
    __builtin_nontemporal_store(from[at], to + at);
  }
}
template <int D>
__device__ __forceinline__ void copy_page(const Kv8Layers& l, int layer, bool keys, int from, int to, int blocks) {
  const int64_t source = kv8_offset(from, 0, l.hkv, D), target = kv8_offset(to, 0, l.hkv, D);
  int8_t* codes = keys ? l.keys[layer] : l.values[layer];
  int8_t* exps = keys ? l.key_exps[layer] : l.value_exps[layer];
  switch (blocks) {
    case 1: copy_codes<D, 1>(codes, keys, source, target, l.hkv); break;
    case 2: copy_codes<D, 2>(codes, keys, source, target, l.hkv); break;
    case 3: copy_codes<D, 3>(codes, keys, source, target, l.hkv); break;
    default: copy_codes<D, 4>(codes, keys, source, target, l.hkv); break;
  }
  static_assert(kKv8Blocks == 4, "a switch over them");
  const int64_t old = kv8_exp_offset(from, 0, l.hkv), now = kv8_exp_offset(to, 0, l.hkv);
  for (int n = threadIdx.x; n < l.hkv * kKv8Blocks; n += kThreads)
    if (n % kKv8Blocks < blocks) exps[now + n] = exps[old + n];
}

// Table rows of a fork, and the copies of a group of layers: the first `tables`
// blocks have the rows.
template <int D>
__global__ __launch_bounds__(kThreads) void kv8_fork_apply_kernel(Kv8ForkArgs a, Kv8Layers l, int tables) {
  ForkSpace f;
  fork_layout(&f, a.workspace, a.seqs, a.per_seq, a.pages);
  if (static_cast<int>(blockIdx.x) < tables) {
    const int tiles = (a.per_seq + kThreads - 1) / kThreads;
    const int s = blockIdx.x / tiles, place = blockIdx.x % tiles * kThreads + threadIdx.x;
    if (place >= a.per_seq) return;
    const int64_t at = static_cast<int64_t>(s) * a.per_seq + place;
    const ForkRow row = f.row[s];
    int p = f.taken[at];
    if (place >= row.fresh && place < row.pages) {
      const int number = row.start + place - row.fresh;
      p = number < f.counts[0] ? f.got[number] : -1;
    }
    a.table[at] = p;
    return;
  }
  const int units = f.counts[1] * l.count * 2, got = f.counts[0];
  for (int u = blockIdx.x - tables; u < units; u += gridDim.x - tables) {
    const int* c = f.copy + 3 * (u / 2 / l.count);
    if (c[1] < got) copy_page<D>(l, u / 2 % l.count, u % 2 == 0, c[0], f.got[c[1]], c[2]);
  }
}

// ------------------------------------------------------------- compact ----

struct CompactSpace {
  int* source;  // [pages / 2] of the k-th move
  int* target;
  int* info;    // [3] moves, pages in use, of those the ones below that number
  int* used;    // [chunks] of a large pool: pages in use of each, then before each
};
__host__ __device__ inline int64_t compact_layout(CompactSpace* c, int* p, int64_t pages) {
  int64_t at = 0;
  auto take = [&](int64_t n) {
    int* mine = p ? p + at : nullptr;
    at += n;
    return mine;
  };
  c->source = take(pages / 2);
  c->target = take(pages / 2);
  c->info = take(3);
  c->used = take(pages > kOnePages ? chunks_of(pages) : 0);
  return at;
}

// Pairs the k-th page in use from `live` on with the k-th hole below it.  With
// the number of pages in use before each page, p is the hole number p - that, or
// the move number that - (those below live): one sum over the pages.  One block,
// whose threads hold the users of their pages, and LDS the holes.
__global__ __launch_bounds__(kOneThreads) void kv8_compact_decide_kernel(Kv8CompactArgs a) {
  __shared__ int sh[kOneThreads / kWave], sh_below, holes[kOnePages / 2], movers[kOnePages / 2];
  CompactSpace c;
  compact_layout(&c, a.workspace, a.pages);
  const int tid = threadIdx.x;
  const int each = ((a.pages + kOneThreads - 1) / kOneThreads + 3) / 4 * 4;  // neighbouring pages of a thread
  const int first = min(tid * each, a.pages), last = min(first + each, a.pages);
  int held[kHeldPages];
  int mine = 0;
#pragma unroll
  for (int i = 0; i < kHeldPages; i += 4) {
    int4 n = make_int4(0, 0, 0, 0);
    if (i < each) n = users_at(a.users, first + i, last, 0);
    held[i] = n.x, held[i + 1] = n.y, held[i + 2] = n.z, held[i + 3] = n.w;
    mine += used_of(n);
  }
  int live;
  const int before = block_scan(mine, sh, &live);
  auto pages_of = [&](auto use) {  // of the thread: use(page, users, pages in use before it)
    int used = before;
#pragma unroll
    for (int i = 0; i < kHeldPages; i += 4) {
      if (i >= each) continue;  // of all threads
#pragma unroll
      for (int m = i; m < i + 4; ++m)
        if (first + m < last) {
          use(first + m, held[m], used);
          used += held[m] > 0;
        }
    }
  };
  if (tid == 0 && live == a.pages) sh_below = live;
  if (first <= live && live < last) pages_of([&](int p, int, int used) {
    if (p == live) sh_below = used;
  });
  __syncthreads();
  const int below = sh_below;
  pages_of([&](int p, int n, int used) {
    if (p < live && n <= 0) holes[p - used] = p;
    if (p >= live && n > 0) movers[used - below] = n;
  });
  __syncthreads();  // and nothing of users is read after: users_out may be users
  // Four pages a store: one at a time, stores take most of the time.
  int used = before;
#pragma unroll
  for (int i = 0; i < kHeldPages; i += 4) {
    if (i >= each) continue;
    int to[4], n[4];
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      const int p = first + i + m;
      n[m] = held[i + m];
      to[m] = n[m] > 0 ? p : -1;
      if (p < last && p < live && n[m] <= 0) n[m] = movers[p - used];
      else if (p < last && p >= live && n[m] > 0) {
        const int k = used - below;
        to[m] = holes[k];
        c.source[k] = p;
        c.target[k] = to[m];
      }
      if (p >= live) n[m] = 0;
      used += held[i + m] > 0;
    }
    if (first + i + 4 <= last) {
      *reinterpret_cast<int4*>(a.moved + first + i) = make_int4(to[0], to[1], to[2], to[3]);
      *reinterpret_cast<int4*>(a.users_out + first + i) = make_int4(n[0], n[1], n[2], n[3]);
    } else {
#pragma unroll
      for (int m = 0; m < 3; ++m)
        if (first + i + m < last) {
          a.moved[first + i + m] = to[m];
          a.users_out[first + i + m] = n[m];
        }
    }
  }
  if (tid == 0) {
    c.info[0] = live - below;
    *a.live = live;
  }
}

// The same of large pools, whose chunks are counted first: sums over the chunks
// (one block), lists (a wave a chunk), pairs (a thread a move).
__global__ __launch_bounds__(kOneThreads) void kv8_compact_sums_kernel(Kv8CompactArgs a) {
  __shared__ int sh[kOneThreads / kWave], sh_below;
  CompactSpace c;
  compact_layout(&c, a.workspace, a.pages);
  const int tid = threadIdx.x, chunks = chunks_of(a.pages);
  int live = 0;
  for (int base = 0; base < chunks; base += kOneThreads) {
    const int n = base + tid < chunks ? c.used[base + tid] : 0;
    int all;
    const int before = block_scan(n, sh, &all);
    if (base + tid < chunks) c.used[base + tid] = live + before;
    live += all;
  }
  if (tid == 0) sh_below = live;  // of a pool that is full
  __syncthreads();
  if (live < a.pages) {
    const int chunk = live / kChunk, p = chunk * kChunk + tid;
    static_assert(kChunk == kOneThreads, "a page a thread");
    int all;
    const int before = block_scan(p < a.pages && a.users[p] > 0, sh, &all);
    if (p == live) sh_below = c.used[chunk] + before;
    __syncthreads();
  }
  if (tid == 0) {
    c.info[0] = live - sh_below;
    c.info[1] = live;
    c.info[2] = sh_below;
    *a.live = live;
  }
}
__global__ __launch_bounds__(kThreads) void kv8_compact_lists_kernel(Kv8CompactArgs a) {
  CompactSpace c;
  compact_layout(&c, a.workspace, a.pages);
  const int chunk = blockIdx.x * kWaves + threadIdx.x / kWave, lane = threadIdx.x % kWave;
  if (chunk >= chunks_of(a.pages)) return;
  const int live = c.info[1], below = c.info[2];
  int before = c.used[chunk];
#pragma unroll
  for (int j = 0; j < kChunk / kWave / 4; ++j) {
    const int first = chunk * kChunk + 4 * (lane + kWave * j);
    const int4 n = users_at(a.users, first, a.pages, 0);
    const int sum = wave_scan(used_of(n)), of[4] = {n.x, n.y, n.z, n.w};
    int used = before + sum - used_of(n);
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      const int p = first + m;
      if (p >= a.pages) continue;
      const bool is = of[m] > 0;
      a.moved[p] = is ? p : -1;
      if (p < live && !is) c.target[p - used] = p;
      if (p >= live && is) c.source[used - below] = p;  // its users are read after
      else a.users_out[p] = max(of[m], 0);
      used += is;
    }
    before += __builtin_amdgcn_readlane(sum, kWave - 1);
  }
}
__global__ __launch_bounds__(kThreads) void kv8_compact_pairs_kernel(Kv8CompactArgs a) {
  CompactSpace c;
  compact_layout(&c, a.workspace, a.pages);
  const int k = blockIdx.x * kThreads + threadIdx.x;
  if (k >= c.info[0]) return;
  const int from = c.source[k], to = c.target[k], n = a.users[from];
  a.moved[from] = to;
  a.users_out[from] = 0;
  a.users_out[to] = n;
}

// The table, and the moves of a group of layers.
template <int D>
__global__ __launch_bounds__(kThreads) void kv8_compact_apply_kernel(Kv8CompactArgs a, Kv8Layers l, int tables) {
  if (static_cast<int>(blockIdx.x) < tables) {
    const int64_t at = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
    if (at >= static_cast<int64_t>(a.seqs) * a.per_seq) return;
    const int p = a.table[at];
    a.table_out[at] = p >= 0 && p < a.pages ? a.moved[p] : -1;
    return;
  }
  CompactSpace c;
  compact_layout(&c, a.workspace, a.pages);
  const int units = c.info[0] * l.count * 2;
  for (int u = blockIdx.x - tables; u < units; u += gridDim.x - tables) {
    const int k = u / 2 / l.count;
    copy_page<D>(l, u / 2 % l.count, u % 2 == 0, c.source[k], c.target[k], kKv8Blocks);
  }
}

// Calls launch(D, layers, table blocks, all blocks) for each group of layers; the
// first has the table's blocks.
template <typename Launch>
hipError_t launch_groups(const Kv8Layers* layers, int groups, int64_t table_blocks, int64_t most_copies,
                         Launch launch) {
  for (int g = 0; g < groups; ++g) {
    const int tables = static_cast<int>(g == 0 ? table_blocks : 0);
    const int blocks = tables + static_cast<int>(std::min<int64_t>(kCopyBlocks, most_copies * layers[g].count * 2));
    if (blocks == 0) continue;
    switch (layers[g].d) {
      case 32: launch(std::integral_constant<int, 32>(), layers[g], tables, blocks); break;
      case 64: launch(std::integral_constant<int, 64>(), layers[g], tables, blocks); break;
      case 96: launch(std::integral_constant<int, 96>(), layers[g], tables, blocks); break;
      case 128: launch(std::integral_constant<int, 128>(), layers[g], tables, blocks); break;
      default: return hipErrorInvalidValue;
    }
  }
  return hipGetLastError();
}

}  // namespace

int64_t kv8_fork_workspace(int64_t seqs, int64_t per_seq, int64_t pages) {
  ForkSpace f;
  return fork_layout(&f, nullptr, seqs, per_seq, pages) * static_cast<int64_t>(sizeof(int));
}

// The deciding block counts the entries of small tables itself: 1,120 entries 9.6
// and, by a kernel of many blocks, 10.4; 2,240 both 12.4; 4,480 13.5 and 11.0.
// Up to kOnePages it looks for free pages from the first on; in larger pools a
// kernel counts those in use by chunks first, so that the time no longer grows with
// the number of the first free page.  64 sequences that take a page each, the last
// free ones: 16,384 pages 9.7 by one block; 20,000 pages 11.8 and, by one block,
// 10.6; 65,536 11.5 and 18.2; 262,144 11.4 and 50.5.  Where the first pages are free
// the two kernels more cost 3 (11.0 and 7.8).
hipError_t launch_kv8_fork(const Kv8ForkArgs& a, const Kv8Layers* layers, int groups, hipStream_t stream) {
  const int blocks = a.seqs * ((a.per_seq + kThreads - 1) / kThreads);
  if (static_cast<int64_t>(a.seqs) * a.per_seq <= kCountEntries && a.pages <= kOnePages) {
    kv8_fork_decide_kernel<true><<<dim3(1), kOneThreads, 0, stream>>>(a);
  } else {
    kv8_fork_count_kernel<<<dim3(blocks), kThreads, 0, stream>>>(a);
    if (a.pages > kOnePages) {
      ForkSpace f;
      fork_layout(&f, a.workspace, a.seqs, a.per_seq, a.pages);
      kv8_count_used_kernel<<<dim3((chunks_of(a.pages) + kWaves - 1) / kWaves), kThreads, 0, stream>>>(a.users, a.pages,
                                                                                                      f.used);
    }
    kv8_fork_decide_kernel<false><<<dim3(1), kOneThreads, 0, stream>>>(a);
  }
  return launch_groups(layers, groups, blocks, a.seqs, [&](auto d, const Kv8Layers& l, int tables, int all) {
    kv8_fork_apply_kernel<decltype(d)::value><<<dim3(all), kThreads, 0, stream>>>(a, l, tables);
  });
}

int64_t kv8_compact_workspace(int64_t pages) {
  CompactSpace c;
  return compact_layout(&c, nullptr, pages) * static_cast<int64_t>(sizeof(int));
}

hipError_t launch_kv8_compact(const Kv8CompactArgs& a, const Kv8Layers* layers, int groups, hipStream_t stream) {
  if (a.pages <= kOnePages) {
    kv8_compact_decide_kernel<<<dim3(1), kOneThreads, 0, stream>>>(a);
  } else {
    CompactSpace c;
    compact_layout(&c, a.workspace, a.pages);
    const dim3 chunk_blocks((chunks_of(a.pages) + kWaves - 1) / kWaves);
    kv8_count_used_kernel<<<chunk_blocks, kThreads, 0, stream>>>(a.users, a.pages, c.used);
    kv8_compact_sums_kernel<<<dim3(1), kOneThreads, 0, stream>>>(a);
    kv8_compact_lists_kernel<<<chunk_blocks, kThreads, 0, stream>>>(a);
    kv8_compact_pairs_kernel<<<dim3((a.pages / 2 + kThreads - 1) / kThreads), kThreads, 0, stream>>>(a);
  }
  const int64_t entries = static_cast<int64_t>(a.seqs) * a.per_seq;
  return launch_groups(layers, groups, (entries + kThreads - 1) / kThreads, a.pages / 2,
                       [&](auto d, const Kv8Layers& l, int tables, int all) {
                         kv8_compact_apply_kernel<decltype(d)::value><<<dim3(all), kThreads, 0, stream>>>(a, l, tables);
                       });
}

}  // namespace mmr
