// Pages of the cache as sequences come, branch and go: giving pages back,
// forking sequences, moving the live pages together.
//
// The state is what the reference's BlockAllocator keeps on the host
// (src/engine/memory/allocator.py: a reference count per page, block tables
// per sequence), here as device tensors, so a step that branches or drops
// sequences needs no host loop and no synchronisation:
//   ref_counts[p]      how many tables (or other holders, such as a prefix
//                      cache) reference page p; 0: the page is free
//   block_tables[r, j] page of tokens [16 j, 16 j + 16) of sequence r; -1: the
//                      page was given back (behind a sliding window)
//   seq_lens[r]        tokens in the cache: entries j < ceil(len / 16) hold
// There is no free list to keep in step: free pages are those with count 0,
// and pages are handed out lowest number first, which keeps the pool dense.
#pragma once

#include "pa_common.cuh"

namespace pa {

// ------------------------------------------------------------ bulk page copy
// Copies (pair, layer) blocks of page_bytes: pages src[i] -> dst[i] for
// i < *count, every layer. Bound by HBM (each byte read and written once): a
// warp per CTA runs a ring of kCopyStages slices of kCopySlice bytes through
// shared memory with bulk copies in both directions, so no byte passes
// through registers. One thread issues them; the addresses of 32 units at a
// time are worked out lane by lane.
constexpr int kCopySlice = 16 * 1024;
constexpr int kCopyStages = 6;
constexpr int kCopyCtas = 2;  // per SM
constexpr int kCopySmem = kCopySlice * kCopyStages + 128;
static_assert(kCopyStages < 32, "a load is at most one batch of units ahead of its store");

struct CopyParams {
  uint8_t* pool;
  int64_t layer_stride, page_stride, page_bytes;  // bytes
  int32_t num_layers;
  const int32_t* src;
  const int32_t* dst;
  const int32_t* count;  // device word
};

__global__ void __launch_bounds__(32, kCopyCtas) copy_pages_kernel(const CopyParams p) {
  extern __shared__ uint8_t copy_smem[];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(copy_smem) + 127) &
                                             ~uintptr_t(127));
  __shared__ uint64_t full[kCopyStages];
  const int lane = threadIdx.x;
  if (lane == 0) {
    for (int s = 0; s < kCopyStages; ++s) mbar_init(&full[s], 1);
    fence_mbar_init();
  }
  __syncwarp();
  griddep_wait();
  const int64_t slices = (p.page_bytes + kCopySlice - 1) / kCopySlice;
  const int64_t per_pair = slices * p.num_layers;
  const int64_t total = per_pair * __ldcg(p.count);
  // this CTA's units: blockIdx.x + i * gridDim.x, i < mine
  const int64_t mine =
      total > blockIdx.x ? (total - blockIdx.x + gridDim.x - 1) / gridDim.x : 0;
  struct Unit {
    uint64_t from, to;
    uint32_t bytes;
  };
  auto batch = [&](int64_t first) {  // lane l: unit first + l of this CTA
    Unit n{0, 0, 0};
    if (first + lane < mine) {
      const int64_t u = blockIdx.x + (first + lane) * gridDim.x;
      const int64_t pair = u / per_pair, rem = u - pair * per_pair;
      const int64_t layer = rem / slices, sl = rem - layer * slices;
      const uint64_t at =
          reinterpret_cast<uint64_t>(p.pool) + layer * p.layer_stride + sl * kCopySlice;
      const int64_t left = p.page_bytes - sl * kCopySlice;
      n.bytes = static_cast<uint32_t>(left < kCopySlice ? left : kCopySlice);
      n.from = at + __ldcg(p.src + pair) * p.page_stride;
      n.to = at + __ldcg(p.dst + pair) * p.page_stride;
    }
    return n;
  };
  Unit a = batch(0), b = batch(32);  // the current 32 units and the next
  int64_t a0 = 0;
  auto load = [&](int64_t i, int stage) {  // every lane calls it
    const int l = static_cast<int>(i - a0);
    const uint64_t from = __shfl_sync(0xffffffffu, l < 32 ? a.from : b.from, l & 31);
    const uint32_t bytes = __shfl_sync(0xffffffffu, l < 32 ? a.bytes : b.bytes, l & 31);
    if (lane == 0) {
      mbar_arrive_expect_tx(&full[stage], bytes);
      bulk_load(ring + stage * kCopySlice, reinterpret_cast<const void*>(from), bytes,
                &full[stage]);
    }
  };
  int64_t loaded = 0;
  for (; loaded < mine && loaded < kCopyStages; ++loaded) load(loaded, static_cast<int>(loaded));
  int stage = 0;
  uint32_t phase = 0;
  bool failed = false;
  for (int64_t i = 0; i < mine; ++i) {
    if (i - a0 == 32) {
      a0 += 32;
      a = b;
      b = batch(a0 + 32);
    }
    const int l = static_cast<int>(i - a0);
    const uint64_t to = __shfl_sync(0xffffffffu, a.to, l);
    const uint32_t bytes = __shfl_sync(0xffffffffu, a.bytes, l);
    if (!mbar_wait_warp(&full[stage], phase)) {
      failed = true;
      break;
    }
    if (lane == 0) {
      bulk_store(reinterpret_cast<void*>(to), ring + stage * kCopySlice, bytes);
      bulk_commit();
    }
    // refill the stage of unit i - 1, whose store has had a unit's time to
    // read it
    if (i >= 1 && loaded < mine) {
      if (lane == 0) bulk_wait_read_but<1>();
      __syncwarp();
      load(loaded, stage == 0 ? kCopyStages - 1 : stage - 1);
      ++loaded;
    }
    if (++stage == kCopyStages) {
      stage = 0;
      phase ^= 1;
    }
  }
  if (failed) {
    if (lane == 0) set_status(PA_ERR_TIMEOUT);
    // the other loads in flight land (or time out too) before this CTA ends
    for (int s = 1; s < kCopyStages; ++s) {
      if (++stage == kCopyStages) {
        stage = 0;
        phase ^= 1;
      }
      mbar_wait_warp(&full[stage], phase);
    }
  }
  if (lane == 0) bulk_wait_all();
}

// ------------------------------------------------------------ giving pages back
struct ReleaseParams {
  int32_t* tables;
  int64_t stride;
  int32_t width, batch, page_size;
  int32_t* lens;          // window < 0: set to 0
  int32_t window, sinks;  // window < 0: every page of the sequence
  int32_t* refs;
  int64_t num_pages;
  int32_t* counts;  // entries given back, pages that became free, errors (zeroed before)
};

// One CTA row per sequence (blockIdx.x), kReleaseThreads entries per step;
// bound by one atomic per entry given back, at random counts in L2: 512 rows,
// 0.51 M entries in 12.1 us of a CUDA graph, 7.9 with nothing left to give back
// (the call with its memset; the kernel takes 11.7 cold under ncu). Counting is
// commutative, so the results do not depend on the order of the atomics.
constexpr int kReleaseThreads = 512;
constexpr int kReleaseUnroll = 4;  // entries per thread whose loads are in flight together

__global__ void __launch_bounds__(kReleaseThreads) release_pages_kernel(const ReleaseParams p) {
  griddep_wait();
  griddep_launch_dependents();
  const int b = blockIdx.x;
  const int len = p.lens[b];
  int32_t* row = p.tables + b * p.stride;
  bool bad = len < 0 || len > static_cast<int64_t>(p.width) * p.page_size;
  int64_t lo = 0, hi = bad ? 0 : (static_cast<int64_t>(len) + p.page_size - 1) / p.page_size;
  if (p.window >= 0) {
    // pages wholly behind the window of the last token's query
    lo = (static_cast<int64_t>(p.sinks) + p.page_size - 1) / p.page_size;
    const int64_t start = static_cast<int64_t>(len) - 1 - p.window;
    hi = bad || start <= 0 ? 0 : start / p.page_size;
  }
  __shared__ int s_counts[3];
  if (threadIdx.x < 3) s_counts[threadIdx.x] = 0;
  __syncthreads();
  int gone = 0, freed = 0, errors = bad && threadIdx.x == 0 ? 1 : 0;
  for (int64_t j0 = lo + threadIdx.x; j0 < hi; j0 += kReleaseThreads * kReleaseUnroll) {
    int page[kReleaseUnroll], old[kReleaseUnroll];
#pragma unroll
    for (int i = 0; i < kReleaseUnroll; ++i) {
      const int64_t j = j0 + i * kReleaseThreads;
      page[i] = j < hi ? row[j] : -1;
    }
#pragma unroll
    for (int i = 0; i < kReleaseUnroll; ++i)
      old[i] = page[i] >= 0 && page[i] < p.num_pages ? atomicSub(p.refs + page[i], 1) : 0;
#pragma unroll
    for (int i = 0; i < kReleaseUnroll; ++i) {
      if (page[i] < 0) continue;
      if (old[i] <= 0) {  // not a page, or nobody held it: its count and the entry stay
        if (page[i] < p.num_pages) atomicAdd(p.refs + page[i], 1);
        ++errors;
        continue;
      }
      row[j0 + i * kReleaseThreads] = -1;
      ++gone;
      freed += old[i] == 1;
    }
  }
  gone = __reduce_add_sync(0xffffffffu, gone);
  freed = __reduce_add_sync(0xffffffffu, freed);
  errors = __reduce_add_sync(0xffffffffu, errors);
  if ((threadIdx.x & 31) == 0) {
    if (gone) atomicAdd(&s_counts[0], gone);
    if (freed) atomicAdd(&s_counts[1], freed);
    if (errors) atomicAdd(&s_counts[2], errors);
  }
  __syncthreads();  // (every thread has read the length, too)
  // One addition per CTA: one per warp, all to the same two words, took as
  // long as the rest (the 512 rows with 4 us of the caller's copies: 22.7 us, so
  // 16.1).
  if (threadIdx.x < 3 && s_counts[threadIdx.x] != 0) {
    atomicAdd(p.counts + threadIdx.x, s_counts[threadIdx.x]);
    if (threadIdx.x == 2) set_status(PA_ERR_DEVICE_CHECK);
  }
  if (p.window < 0 && threadIdx.x == 0 && !bad) p.lens[b] = 0;
}

// ------------------------------------------------------------------ scans
constexpr int kScanThreads = 1024;

// Exclusive prefix of `v` over the CTA's threads; *total its sum. Every
// thread calls it; s_warp is 32 ints of shared memory.
__device__ __forceinline__ int block_exclusive(int v, int* s_warp, int* total) {
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  int incl = v;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, incl, off);
    if (lane >= off) incl += u;
  }
  if (lane == 31) s_warp[wid] = incl;
  __syncthreads();
  const int w = s_warp[lane];
  int winc = w;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, winc, off);
    if (lane >= off) winc += u;
  }
  *total = __shfl_sync(0xffffffffu, winc, 31);
  const int before = wid > 0 ? __shfl_sync(0xffffffffu, winc, wid - 1) : 0;
  __syncthreads();  // s_warp may be written again
  return before + incl - v;
}

// kPerThread consecutive counts per thread, read past L1 (atomics and other
// CTAs write them); entries at or past n read as `fill`.
constexpr int kPerThread = 16;

__device__ __forceinline__ void load_counts(const int32_t* refs, int64_t at, int64_t n, int fill,
                                            int (&v)[kPerThread]) {
  if ((reinterpret_cast<uintptr_t>(refs) & 15) == 0 && at + kPerThread <= n) {
#pragma unroll
    for (int i = 0; i < kPerThread; i += 4) {
      const int4 x = __ldcg(reinterpret_cast<const int4*>(refs + at + i));
      v[i] = x.x;
      v[i + 1] = x.y;
      v[i + 2] = x.z;
      v[i + 3] = x.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) v[i] = at + i < n ? __ldcg(refs + at + i) : fill;
  }
}

// ------------------------------------------------------------------ fork
// Row r of the new tables continues row parents[r] of the old ones. With
// c(s) = rows that continue s:
//   full pages j < len / P of s:  ref += c(s) - 1 (shared by its children)
//   the page the next token goes to (entry len / P of the child) is private:
//     - len % P == 0: a free page;
//     - else the parent's unfinished page: its holders among the old rows let
//       go of it; if nobody else holds it the first row that continues it
//       keeps it, every other one gets a free page and a copy.
// A row with parent -1 ends: it holds nothing. (A row of length 0 that goes on
// takes a page like any other, which it would hold until its next token; a row
// that stays in the batch without going on has to say so.)
// An unfinished page that the table does not name (-1): with all_held it is
// lost (an earlier fork found no free page for the row), and so are its tokens.
// The row is reported, takes no page (a free one holds some other sequence's
// tokens) and comes back with the length of its full pages, as does a row that
// this fork leaves without the copy. Without all_held it counts as given back
// behind a window, and the row goes on in a free page.
// Three launches: per row (counts of the full pages, the gathered table),
// one CTA (who keeps, who gets which page), the copies.
struct ForkSeqParams {
  const int32_t* tables;
  int64_t stride;
  int32_t width, rows, page_size;
  const int32_t* lens;
  const int32_t* parents;
  int32_t* refs;
  int64_t num_pages;
  int32_t* out_tables;  // [rows, out_stride]
  int64_t out_stride;
  int32_t* out_lens;
  int32_t* counts;  // copies, pages taken, rows left without a page
  bool all_held;    // no unfinished page was given back
  // scratch, [rows] each
  int32_t* avail;  // free pages, lowest number first
  int32_t* dst;    // copies: to
  int32_t* state;  // per row between the passes; at the end copies: from
};

struct ForkRow {
  int parent, len, full, last;  // last: the unfinished page, -1: none (or given back)
  bool ok;                      // parent and length are sound
  bool ended;                   // continues nothing, and is not meant to
  bool lost;                    // its unfinished page is not there
};

__device__ __forceinline__ ForkRow fork_row(const ForkSeqParams& p, int r) {
  ForkRow f;
  f.parent = __ldg(p.parents + r);
  f.ended = f.parent == -1;
  f.ok = f.parent >= 0 && f.parent < p.rows;
  f.len = f.ok ? __ldg(p.lens + f.parent) : 0;
  if (f.len < 0 || f.len > static_cast<int64_t>(p.width) * p.page_size) f.ok = false;
  if (!f.ok) f.len = 0;
  f.full = f.len / p.page_size;
  f.last = -1;
  f.lost = false;
  if (f.len % p.page_size) {
    f.last = __ldg(p.tables + f.parent * p.stride + f.full);
    if (f.last >= p.num_pages) f.ok = false;
    if (f.last < 0) {  // nothing to keep or copy
      f.last = -1;
      f.lost = p.all_held;
      if (f.lost) f.len = f.full * p.page_size;
    }
  }
  return f;
}

constexpr int kForkThreads = 256;

__global__ void __launch_bounds__(kForkThreads) fork_rows_kernel(const ForkSeqParams p) {
  griddep_wait();
  griddep_launch_dependents();
  const int r = blockIdx.x, tid = threadIdx.x;
  __shared__ int s_children;
  if (tid == 0) s_children = 0;
  __syncthreads();
  int mine = 0;
  for (int i = tid; i < p.rows; i += kForkThreads) mine += __ldg(p.parents + i) == r;
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, off);
  if ((tid & 31) == 0 && mine) atomicAdd(&s_children, mine);
  __syncthreads();
  // row r as a parent: its full pages, and its hold on its unfinished one
  const int len = __ldg(p.lens + r);
  const bool sound = len >= 0 && len <= static_cast<int64_t>(p.width) * p.page_size;
  if (sound) {
    const int32_t* row = p.tables + r * p.stride;
    const int full = len / p.page_size;
    const int last = len % p.page_size ? __ldg(row + full) : 0;
    const bool usable = last < p.num_pages;  // else its children have no state
    const int delta = (usable ? s_children : 0) - 1;
    if (delta != 0)
      for (int j = tid; j < full; j += kForkThreads) {
        const int page = __ldg(row + j);
        if (page < 0) continue;
        // (sound counts stay >= 0 in any order: each holder leaves only once)
        if (page >= p.num_pages || atomicAdd(p.refs + page, delta) + delta < 0)
          set_status(PA_ERR_DEVICE_CHECK);
      }
    if (tid == 0 && len % p.page_size && usable && last >= 0 && atomicSub(p.refs + last, 1) <= 0)
      set_status(PA_ERR_DEVICE_CHECK);
  }
  // row r as a child: the parent's full pages
  const ForkRow f = fork_row(p, r);
  int32_t* out = p.out_tables + r * p.out_stride;
  const int32_t* from = p.tables + (f.ok ? f.parent : 0) * p.stride;
  for (int j = tid; j < p.width; j += kForkThreads)
    if (j != f.full) out[j] = f.ok && j < f.full ? __ldg(from + j) : -1;
  if (tid == 0) p.out_lens[r] = f.ok ? f.len : 0;
}

// One CTA; bound by its chain of dependent L2 reads, so the first 1024 rows
// and the first kScanThreads * kPerThread counts stay in registers, and the
// free pages' numbers in shared memory.
__global__ void __launch_bounds__(kScanThreads) fork_assign_kernel(const ForkSeqParams p) {
  griddep_wait();
  griddep_launch_dependents();
  __shared__ int s_warp[32];
  __shared__ int s_avail[kScanThreads];
  const int tid = threadIdx.x;
  const int rounds = (p.rows + kScanThreads - 1) / kScanThreads;
  const ForkRow none{0, 0, 0, -1, false, true, false};
  const ForkRow first = tid < p.rows ? fork_row(p, tid) : none;
  int state0 = 0;  // state of row `tid`; later rows' in p.state
  auto row = [&](int k) {
    const int r = k * kScanThreads + tid;
    return k == 0 ? first : r < p.rows ? fork_row(p, r) : none;
  };
  auto get = [&](int k) {
    const int r = k * kScanThreads + tid;
    return k == 0 ? state0 : r < p.rows ? p.state[r] : 0;
  };
  auto set = [&](int k, int v) {
    const int r = k * kScanThreads + tid;
    if (k == 0)
      state0 = v;
    else if (r < p.rows)
      p.state[r] = v;
  };
  // Claims on unfinished pages that nobody else holds: the count (0 now)
  // serves as the ballot, rows - r being larger for earlier rows. Every row
  // looks before any row claims, and claims are settled before any is
  // answered.
  for (int k = 0; k < rounds; ++k) {
    const ForkRow f = row(k);
    set(k, f.last >= 0 && f.ok && __ldcg(p.refs + f.last) == 0);
  }
  __syncthreads();
  for (int k = 0; k < rounds; ++k)
    if (get(k)) atomicMax(p.refs + row(k).last, p.rows - (k * kScanThreads + tid));
  __syncthreads();
  for (int k = 0; k < rounds; ++k)
    if (get(k) && __ldcg(p.refs + row(k).last) != p.rows - (k * kScanThreads + tid)) set(k, 0);
  __syncthreads();
  int total = 0;
  for (int k = 0; k < rounds; ++k) {
    const int r = k * kScanThreads + tid;
    const ForkRow f = row(k);
    const bool keep = get(k) != 0;
    if (keep) {
      p.refs[f.last] = 1;
      p.out_tables[r * p.out_stride + f.full] = f.last;
    }
    // state: rank among the rows that want a page, -1: wants none (keeps its
    // page, has lost it, has ended, or is not sound)
    const bool wants = r < p.rows && f.ok && !f.lost && !keep && f.full < p.width;
    int n;
    const int at = total + block_exclusive(wants ? 1 : 0, s_warp, &n);
    total += n;
    set(k, wants ? at : -1);
  }
  // the first `total` free pages in ascending order
  __syncthreads();
  int found = 0;
  for (int64_t base = 0; base < p.num_pages && found < total;
       base += static_cast<int64_t>(kScanThreads) * kPerThread) {
    const int64_t at = base + static_cast<int64_t>(tid) * kPerThread;
    int v[kPerThread];
    load_counts(p.refs, at, p.num_pages, 1, v);
    int zeros = 0;
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) zeros += v[i] == 0;
    int n;
    int rank = found + block_exclusive(zeros, s_warp, &n);
#pragma unroll
    for (int i = 0; i < kPerThread; ++i)
      if (v[i] == 0) {
        if (rank < total) {
          if (rank < kScanThreads)
            s_avail[rank] = static_cast<int>(at + i);
          else
            p.avail[rank] = static_cast<int>(at + i);
        }
        ++rank;
      }
    found += n;
  }
  found = min(found, total);
  __syncthreads();
  int missing = 0, copies = 0;
  for (int k = 0; k < rounds; ++k) {
    const int r = k * kScanThreads + tid;
    const ForkRow f = row(k);
    const int at = get(k);
    int page = -1, from = -1;
    if (r < p.rows) {
      if (at >= 0) {
        if (at < found) {
          page = at < kScanThreads ? s_avail[at] : __ldcg(p.avail + at);
          p.refs[page] = 1;
          from = f.last;
        }
        p.out_tables[r * p.out_stride + f.full] = page;
        missing += page < 0;
        if (page < 0 && p.all_held) p.out_lens[r] = f.full * p.page_size;
      } else if (!f.ok || f.lost || f.full >= p.width) {
        if (f.full < p.width) p.out_tables[r * p.out_stride + f.full] = -1;
        missing += !f.ended;
      }
    }
    int n;
    const int c = copies + block_exclusive(from >= 0 ? 1 : 0, s_warp, &n);
    copies += n;
    if (from >= 0) {
      // pairs are packed into dst and state: entry c is at most the row's own,
      // which every thread of this round has read
      p.dst[c] = page;
      p.state[c] = from;
    }
    __syncthreads();
  }
  int n;
  block_exclusive(missing, s_warp, &n);
  if (tid == 0) {
    p.counts[0] = copies;
    p.counts[1] = found;
    p.counts[2] = n;
    if (n) set_status(PA_ERR_DEVICE_CHECK);
  }
}

// --------------------------------------------------------------- compaction
// With n live pages, the k-th live page at or past n moves into the k-th free
// page before n. Sources and targets are disjoint, so the copies need no
// order.
struct CompactParams {
  int32_t* refs;
  int64_t num_pages;
  int32_t* remap;   // [num_pages]: new number of a live page, -1: free
  int32_t* src;     // scratch, [num_pages / 2 + 1]
  int32_t* dst;     // scratch, [num_pages / 2 + 1]
  int32_t* counts;  // live pages, pages moved, errors
};

__global__ void __launch_bounds__(kScanThreads) compact_plan_kernel(const CompactParams p) {
  griddep_wait();
  griddep_launch_dependents();
  __shared__ int s_warp[32];
  const int tid = threadIdx.x;
  constexpr int64_t kStep = static_cast<int64_t>(kScanThreads) * kPerThread;
  const int64_t mine = static_cast<int64_t>(tid) * kPerThread;
  int v[kPerThread];
  int live = 0;
  // last step first, so that the first one's counts are at hand for the ranks
  for (int64_t base = (p.num_pages - 1) / kStep * kStep; base >= 0; base -= kStep) {
    load_counts(p.refs, base + mine, p.num_pages, 0, v);
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) live += v[i] > 0;
  }
  int n_live;
  block_exclusive(live, s_warp, &n_live);
  int moved = 0, holes = 0;
  for (int64_t base = 0; base < p.num_pages; base += kStep) {
    const int64_t at = base + mine;
    if (base > 0) load_counts(p.refs, at, p.num_pages, 0, v);
    int out = 0, in = 0;
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) {
      out += v[i] > 0 && at + i >= n_live;
      in += v[i] <= 0 && at + i < n_live;
    }
    // both ranks in one scan: at most 16384 of each per step
    int n_both;
    const int both = block_exclusive(out << 16 | in, s_warp, &n_both);
    int o = moved + (both >> 16), h = holes + (both & 0xffff);
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) {
      const int64_t page = at + i;
      if (page >= p.num_pages) continue;
      if (page >= n_live) {
        if (v[i] > 0)
          p.src[o++] = static_cast<int>(page);
        else
          p.remap[page] = -1;
      } else if (v[i] > 0) {
        p.remap[page] = static_cast<int>(page);
      } else {
        p.dst[h++] = static_cast<int>(page);
        p.remap[page] = -1;
      }
    }
    moved += n_both >> 16;
    holes += n_both & 0xffff;
  }
  __syncthreads();
  for (int k = tid; k < moved; k += kScanThreads) {
    const int s = __ldcg(p.src + k), d = __ldcg(p.dst + k);
    p.remap[s] = d;
    p.refs[d] = __ldcg(p.refs + s);
    p.refs[s] = 0;
  }
  if (tid == 0) {
    p.counts[0] = n_live;
    p.counts[1] = moved;
    p.counts[2] = 0;
  }
}

struct RemapParams {
  int32_t* tables;
  int64_t stride;
  int32_t width, batch, page_size;
  const int32_t* lens;
  const int32_t* remap;
  int64_t num_pages;
  int32_t* counts;
};

__global__ void __launch_bounds__(kReleaseThreads) remap_tables_kernel(const RemapParams p) {
  griddep_wait();
  griddep_launch_dependents();
  const int b = blockIdx.x;
  const int len = __ldg(p.lens + b);
  int32_t* row = p.tables + b * p.stride;
  // A length past the table is reported once, and the entries that there are
  // follow all the same: their pages have moved.
  const bool past = len > static_cast<int64_t>(p.width) * p.page_size;
  const int64_t held = (static_cast<int64_t>(len) + p.page_size - 1) / p.page_size;
  const int n = len < 0 ? 0 : past ? p.width : static_cast<int>(held);
  int errors = (len < 0 || past) && threadIdx.x == 0 ? 1 : 0;
  for (int j = threadIdx.x; j < n; j += kReleaseThreads) {
    const int page = row[j];
    if (page < 0) continue;
    const int to = page < p.num_pages ? __ldcg(p.remap + page) : -1;
    if (to < 0) {
      errors += !past;  // a page that nobody holds: the entry stays
      continue;
    }
    if (to != page) row[j] = to;
  }
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) errors += __shfl_xor_sync(0xffffffffu, errors, off);
  if ((threadIdx.x & 31) == 0 && errors) {
    atomicAdd(p.counts + 2, errors);
    set_status(PA_ERR_DEVICE_CHECK);
  }
}

}  // namespace pa
