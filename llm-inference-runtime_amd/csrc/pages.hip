// Page tables and pools kept on the device: pages for a step's new tokens with
// copy-on-write forks (todo.md:17-19 of the reference asks for those), sharing
// a sequence's pages with another row, releasing pages, and compaction of a
// scattered pool.  The engine does all of it on the host
// (src/engine/memory/allocator.py:52-87) and uploads the tables every step; here
// a captured step can do it.
//
// The state is one reference count per page, ref_counts [num_pages]: a page is
// free while it is 0.  Free pages are handed out in ascending order, so results
// do not depend on timing.  Finding them is a count per block of kPagesPerBlock
// pages and a rank by prefix sums, without a free list to keep in order;
// reading 4 bytes a page, 0.4 MB for 100 000 pages, costs less than a launch.
//
// Bounds: the metadata kernels by launch and load latency (two to four dependent
// loads each: 512 rows over 100 000 pages 7.0, 4.3, 5.2 us for reserve's three
// launches, 3.8 us for the release behind a window; 32 rows over 4000 pages 4.9
// and 5.7 us for its two, and 2.8 us), the copies by HBM bandwidth.
#include <algorithm>

#include "common.h"

namespace pa {

constexpr int kPagesPerBlock = 4096;
constexpr int kPageThreads = 256;
constexpr int kPageWaves = kPageThreads / kWave;
constexpr int kPageSteps = kPagesPerBlock / kPageThreads;

// Which of a block's pages are held.  Wave w has pages 1024 w to 1024 w + 1023 of
// it: bit `lane` of m[k] is page 1024 w + 64 k + lane.  Pages past the pool count
// as `past`.  One coalesced load a step, all in flight at once.
struct Held {
  uint64_t m[kPageSteps];
  int64_t page0;  // the wave's first page

  __device__ __forceinline__ void load(const int32_t* refs, int block, int num_pages, bool past) {
    const int lane = threadIdx.x & (kWave - 1);
    page0 = (int64_t)block * kPagesPerBlock +
            uniform((int)threadIdx.x >> 6) * (kPagesPerBlock / kPageWaves);
    int v[kPageSteps];
#pragma unroll
    for (int k = 0; k < kPageSteps; ++k) {
      const int64_t p = page0 + k * kWave + lane;
      v[k] = past ? 1 : 0;
      if (p < num_pages) v[k] = refs[p];
    }
#pragma unroll
    for (int k = 0; k < kPageSteps; ++k) m[k] = __builtin_amdgcn_ballot_w64(v[k] != 0);
  }
  __device__ __forceinline__ int count() const {
    int n = 0;
#pragma unroll
    for (int k = 0; k < kPageSteps; ++k) n += (int)__builtin_popcountll(m[k]);
    return n;
  }
  // those with a page id below `line`
  __device__ __forceinline__ int count_below(int64_t line) const {
    int n = 0;
#pragma unroll
    for (int k = 0; k < kPageSteps; ++k) {
      const int64_t d = line - (page0 + k * kWave);
      const uint64_t in = d >= kWave ? ~0ull : d > 0 ? (1ull << (int)d) - 1 : 0ull;
      n += (int)__builtin_popcountll(m[k] & in);
    }
    return n;
  }
};

// Bits of m below the lane's own.
__device__ __forceinline__ int bits_below(uint64_t m) {
  return (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32),
                                        __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0u));
}

// Sum of a wave-uniform value over the workgroup's waves; *before gets that of
// the waves before this one.
__device__ __forceinline__ int waves_sum(int v, int* red, int* before) {
  const int wave = uniform((int)threadIdx.x >> 6);
  __syncthreads();  // the last use of `red` is over
  if ((threadIdx.x & (kWave - 1)) == 0) red[wave] = v;
  __syncthreads();
  int all = 0, mine = 0;
#pragma unroll
  for (int w = 0; w < kPageWaves; ++w) {
    const int x = red[w];
    all += x;
    mine += w < wave ? x : 0;
  }
  *before = mine;
  return all;
}

__device__ __forceinline__ int block_sum(int v, int* red) {
#pragma unroll
  for (int o = kWave / 2; o > 0; o >>= 1) v += __shfl_xor(v, o);
  __syncthreads();  // the last use of `red` is over
  if ((threadIdx.x & (kWave - 1)) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  int s = 0;
#pragma unroll
  for (int i = 0; i < kPageThreads / kWave; ++i) s += red[i];
  return s;
}

// Sum of v[0, n) over the workgroup.
__device__ __forceinline__ int array_sum(const int32_t* v, int n, int* red) {
  int s = 0;
  for (int i = (int)threadIdx.x; i < n; i += kPageThreads) s += v[i];
  return block_sum(s, red);
}

// ----------------------------------------------------------------------------
// reserve: pages of the slots that a step's new tokens open, and a fresh page in
// place of a partial one that others hold.
struct ReserveArgs {
  int32_t* tables;
  int64_t stride;
  int32_t max_pages, batch;
  const int32_t* kv_lens;
  const int32_t* new_lens;  // null: one new token per sequence
  int32_t* refs;
  int32_t num_pages, n_blocks;
  int32_t* err;
  // scratch: pages wanted by each sequence (kForkBit: one of them for a fork),
  // the sum over those before it, free pages of each block, the pages taken in
  // order, and the forks: the page, the rank of the one that takes its rows, how many
  int32_t* need;
  int32_t* base;
  int32_t* free_cnt;
  int32_t* fresh;
  int32_t* n_forks;  // 0 where the pages do not suffice
  int32_t* fork_src;
  int32_t* fork_rank;
  int32_t* fork_rows;
  int32_t* short_of;  // pages missing; nothing is changed then
};
constexpr int32_t kForkBit = 1 << 30;

struct RowStep {
  bool ok;          // the row's lengths fit its table
  int first, last;  // slots the new tokens open
  int part;         // slot of the partial page they continue, or -1
  int rows;         // rows in it
};

__device__ __forceinline__ RowStep row_step(const ReserveArgs& a, int b) {
  const int len = a.kv_lens[b];
  const int n = a.new_lens ? a.new_lens[b] : 1;
  RowStep r{false, 0, 0, -1, 0};
  if (n < 0 || len < n) return r;
  const int held = len - n;
  r.last = (int)(((int64_t)len + kPage - 1) / kPage);
  if (r.last > a.max_pages) return r;
  r.ok = true;
  r.first = (int)(((int64_t)held + kPage - 1) / kPage);
  r.rows = held % kPage;
  if (n > 0 && r.rows) r.part = held / kPage;
  return r;
}

// Workgroups [0, n_blocks): free pages of a block.  The others: a wave per
// sequence counts the pages it wants.  The sequences of a call that append to one
// shared page fork in order while another holds it: sequence b forks where the
// page's count less the earlier ones is above 1.
__global__ void __launch_bounds__(kPageThreads) reserve_count_kernel(ReserveArgs a) {
  __shared__ int red[kPageThreads / kWave];
  const int lane = threadIdx.x & (kWave - 1);
  if ((int)blockIdx.x < a.n_blocks) {
    Held held;
    held.load(a.refs, (int)blockIdx.x, a.num_pages, true);
    int before;
    const int n = waves_sum(held.count(), red, &before);
    if (threadIdx.x == 0) a.free_cnt[blockIdx.x] = kPagesPerBlock - n;
    return;
  }
  const int b = ((int)blockIdx.x - a.n_blocks) * (kPageThreads / kWave) +
                uniform((int)threadIdx.x >> 6);
  if (b >= a.batch) return;
  const RowStep r = row_step(a, b);
  bool ok = r.ok;
  bool fork = false;
  if (ok && r.part >= 0) {
    const int page = a.tables[b * a.stride + r.part];
    ok = page >= 0 && page < a.num_pages && a.refs[page] > 0;
    if (ok && a.refs[page] > 1) {
      int earlier = 0;
      for (int i = lane; i < b; i += kWave) {
        const RowStep o = row_step(a, i);
        if (o.ok && o.part >= 0 && a.tables[i * a.stride + o.part] == page) ++earlier;
      }
#pragma unroll
      for (int o = kWave / 2; o > 0; o >>= 1) earlier += __shfl_xor(earlier, o);
      fork = a.refs[page] - earlier > 1;
    }
  }
  if (lane == 0) {
    a.need[b] = ok ? (r.last - r.first) + (fork ? 1 + kForkBit : 0) : 0;
    if (!ok && a.err) atomicAdd(a.err, 1);
  }
}

// What reserve_count_kernel counts for sequence threadIdx.x of at most kPageThreads,
// by a whole workgroup; *ok: the sequence is not skipped.
__device__ __forceinline__ int own_need(const ReserveArgs& a, int* part_page, bool* ok) {
  const int b = (int)threadIdx.x;
  RowStep r{true, 0, 0, -1, 0};
  int page = -1, held = 0;
  if (b < a.batch) {
    r = row_step(a, b);
    if (r.ok && r.part >= 0) {
      page = a.tables[b * a.stride + r.part];
      if (page >= 0 && page < a.num_pages) held = a.refs[page];
    }
  }
  part_page[b] = page;
  __syncthreads();
  *ok = r.ok && (r.part < 0 || held > 0);
  if (!*ok) return 0;
  bool fork = false;
  if (held > 1) {
    int earlier = 0;
    for (int i = 0; i < b; ++i) earlier += part_page[i] == page;
    fork = held - earlier > 1;
  }
  return (r.last - r.first) + (fork ? 1 + kForkBit : 0);
}

// COUNTS: the counts come from reserve_count_kernel.  Up to kOwnRows sequences over a
// pool of up to kReserveBlocks blocks are counted by every workgroup itself, which
// saves a launch.  Back to back on the GPU, us with and without it: 32 rows over 4000
// pages 8.1 and 6.2, 128 over 4000 8.4 and 7.5, over 8192 8.6 and 8.2; 256 over 4000
// 9.0 and 9.3, over 16384 9.5 and 11.5, 32 over 16384 8.5 both.
constexpr int kOwnRows = 128;
constexpr int kReserveBlocks = 2;
static_assert(kOwnRows <= kPageThreads, "a sequence per thread");

// Workgroups [0, n_blocks): the free pages of a block at their ranks, as far as
// they are wanted.  The last: the sequences' first ranks, the forks, and whether
// the pages suffice.
template <bool COUNTS>
__global__ void __launch_bounds__(kPageThreads) reserve_rank_kernel(ReserveArgs a) {
  __shared__ int red[kPageThreads / kWave];
  __shared__ int part_page[COUNTS ? 1 : kPageThreads];
  const int blk = (int)blockIdx.x;
  const bool last = blk == a.n_blocks;
  // the block's pages are on their way while the counts are summed
  Held held;
  if (!last) held.load(a.refs, blk, a.num_pages, true);
  // free pages before the block (the last workgroup: all), and those wanted
  int before, wanted, own = 0;
  if constexpr (COUNTS) {
    before = array_sum(a.free_cnt, blk, red);
  } else {
    int taken = 0;  // the wave's share of the blocks'
#pragma unroll
    for (int i = 0; i < kReserveBlocks; ++i)
      if (i < blk) {
        Held other;
        other.load(a.refs, i, a.num_pages, true);
        taken += other.count();
      }
    int unused;
    before = blk * kPagesPerBlock - waves_sum(taken, red, &unused);
    bool ok;
    own = own_need(a, part_page, &ok);
    if (last && !ok && a.err) atomicAdd(a.err, 1);
  }
  if (last) {
    int run = 0, forks = 0;
    for (int b0 = 0; b0 < a.batch; b0 += kPageThreads) {
      const int b = b0 + (int)threadIdx.x;
      int need = own;
      if constexpr (COUNTS) need = b < a.batch ? a.need[b] : 0;
      else if (b < a.batch) a.need[b] = need;
      const bool fork = need & kForkBit;
      int total, total_forks;
      __syncthreads();
      const int at = run + block_excl_scan<kPageThreads>(need & ~kForkBit, &total, red);
      const int f = forks + block_excl_scan<kPageThreads>(fork ? 1 : 0, &total_forks, red);
      if (b < a.batch) a.base[b] = at;
      if (fork) {
        const RowStep r = row_step(a, b);
        a.fork_src[f] = a.tables[b * a.stride + r.part];
        a.fork_rank[f] = at;
        a.fork_rows[f] = r.rows;
      }
      run += total;
      forks += total_forks;
    }
    if (threadIdx.x == 0) {
      const int missing = max(run - before, 0);
      *a.short_of = missing;
      *a.n_forks = missing > 0 ? 0 : forks;
      if (missing > 0 && a.err) atomicAdd(a.err + 1, missing);
    }
    return;
  }
  wanted = own & ~kForkBit;
  if constexpr (COUNTS) {
    wanted = 0;
    for (int b = (int)threadIdx.x; b < a.batch; b += kPageThreads) wanted += a.need[b] & ~kForkBit;
  }
  wanted = block_sum(wanted, red);
  if (before >= wanted) return;  // uniform
  int held_before;
  waves_sum(held.count(), red, &held_before);
  // free pages before the wave's first
  int rank = before + uniform((int)threadIdx.x >> 6) * (kPagesPerBlock / kPageWaves) - held_before;
  const int lane = threadIdx.x & (kWave - 1);
#pragma unroll
  for (int k = 0; k < kPageSteps; ++k) {
    const uint64_t open = ~held.m[k];
    const int at = rank + bits_below(open);
    if (((open >> lane) & 1) && at < wanted) a.fresh[at] = (int32_t)(held.page0 + k * kWave + lane);
    rank += (int)__builtin_popcountll(open);
  }
}

// ----------------------------------------------------------------------------
// Copies of pages in every layer: the page src[i] to dst[i], i < *count; forks
// (ROWS) the first rows[i] rows of each (K|V, head) block, to page
// dst[dst_at[i]].  No destination is a source.  Resident workgroups walk units of up to kCopyUnit
// bytes; a page's layer is one run of 2 Hkv 16 D elements.  Bound by HBM: every
// byte is read and written once.
struct CopyArgs {
  uint8_t* pool;
  float* scales;  // [L, P, 2, Hkv] or null
  const int32_t* count;
  const int32_t* src;
  const int32_t* dst;
  const int32_t* dst_at;
  const int32_t* rows;
  int32_t num_layers, num_pages, blocks;  // blocks: 2 Hkv
  int32_t block_bytes, row_bytes;
  int32_t units;  // of a page's layer
};
constexpr int kCopyLoads = 4;
constexpr int kCopyUnit = kPageThreads * 16 * kCopyLoads;

template <bool ROWS>
__device__ __forceinline__ void copy_pages(const CopyArgs& c, int64_t wg, int64_t n_wg) {
  const int page_bytes = c.blocks * c.block_bytes;
  const int64_t per_move = (int64_t)c.num_layers * c.units;
  const int64_t total = (int64_t)*c.count * per_move;
  for (int64_t u = wg; u < total; u += n_wg) {
    const int i = (int)(u / per_move);
    const int rem = (int)(u - i * per_move);
    const int layer = rem / c.units;
    const int part = rem - layer * c.units;
    const int64_t from = (int64_t)layer * c.num_pages + uniform(c.src[i]);
    const int64_t to = (int64_t)layer * c.num_pages + uniform(c.dst[ROWS ? c.dst_at[i] : i]);
    const int bytes = ROWS ? uniform(c.rows[i]) * c.row_bytes : c.block_bytes;
    const uint8_t* s = c.pool + from * page_bytes;
    uint8_t* d = c.pool + to * page_bytes;
    u32x4 x[kCopyLoads];
    int at[kCopyLoads];
    bool on[kCopyLoads];
#pragma unroll
    for (int k = 0; k < kCopyLoads; ++k) {
      at[k] = part * kCopyUnit + (k * kPageThreads + (int)threadIdx.x) * 16;
      on[k] = at[k] < page_bytes;
      if constexpr (ROWS) on[k] = on[k] && at[k] % c.block_bytes < bytes;
      x[k] = u32x4{0u, 0u, 0u, 0u};
      if (on[k]) x[k] = *reinterpret_cast<const u32x4*>(s + at[k]);
    }
#pragma unroll
    for (int k = 0; k < kCopyLoads; ++k)
      if (on[k]) {
        // a compacted pool is past the caches (a streamed store: 263 -> 252 us); a
        // fork's page is the next one written and read
        if constexpr (ROWS) *reinterpret_cast<u32x4*>(d + at[k]) = x[k];
        else __builtin_nontemporal_store(x[k], reinterpret_cast<u32x4*>(d + at[k]));
      }
    if (c.scales && part == 0)
      for (int j = (int)threadIdx.x; j < c.blocks; j += kPageThreads)
        c.scales[to * c.blocks + j] = c.scales[from * c.blocks + j];
  }
}

// A wave per sequence: its new table entries and their counts.  Every workgroup:
// its share of the forks' rows (the pages copied keep their rows, whoever
// appends to them comes later on the stream).
__global__ void __launch_bounds__(kPageThreads) reserve_assign_kernel(ReserveArgs a, CopyArgs c) {
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = uniform((int)threadIdx.x >> 6);
  if (*a.short_of > 0) return;
  for (int b = (int)blockIdx.x * (kPageThreads / kWave) + wave; b < a.batch;
       b += (int)gridDim.x * (kPageThreads / kWave)) {
    const int want = a.need[b];
    if (want == 0) continue;
    const RowStep r = row_step(a, b);
    const int fork = want & kForkBit ? 1 : 0;
    const int n = (want & ~kForkBit) - fork;
    const int32_t* got = a.fresh + a.base[b];
    int32_t* row = a.tables + b * a.stride;
    for (int i = lane; i < n; i += kWave) {
      const int page = got[fork + i];
      row[r.first + i] = page;
      a.refs[page] = 1;
    }
    if (fork && lane == 0) {
      atomicSub(a.refs + row[r.part], 1);
      row[r.part] = got[0];
      a.refs[got[0]] = 1;
    }
  }
  copy_pages<true>(c, blockIdx.x, gridDim.x);
}

// ----------------------------------------------------------------------------
// release: table slots [first, last) of every row give up their pages.  A page
// named more often than its count says is counted as an error and stays at 0.
struct ReleaseArgs {
  int32_t* tables;
  int64_t stride;
  int32_t max_pages, batch;
  int32_t* refs;
  int32_t num_pages;
  const int32_t* first;  // null: 0
  const int32_t* last;   // null: max_pages
  // window: the pages between the sinks' and the one that holds the first token
  // that the newest sees
  const int32_t* kv_lens;  // null: no window
  int32_t window_left, sinks;
  int32_t* err;
};

__global__ void __launch_bounds__(kPageThreads) release_pages_kernel(ReleaseArgs a) {
  const int b = blockIdx.y;
  int lo = 0, hi = a.max_pages;
  if (a.kv_lens) {
    const int64_t start = (int64_t)a.kv_lens[b] - 1 - a.window_left;
    lo = (int)(((int64_t)a.sinks + kPage - 1) / kPage);
    hi = start > 0 ? (int)min<int64_t>(start / kPage, a.max_pages) : 0;
  } else {
    if (a.first) lo = max(a.first[b], 0);
    if (a.last) hi = min(a.last[b], a.max_pages);
  }
  int32_t* row = a.tables + b * a.stride;
  const int step = (int)(gridDim.x * kPageThreads);
  for (int64_t s = (int64_t)lo + blockIdx.x * kPageThreads + threadIdx.x; s < hi; s += step) {
    const int page = row[s];
    bool bad = false;
    if (page >= 0) {
      bad = page >= a.num_pages;
      if (!bad && atomicSub(a.refs + page, 1) <= 0) {
        atomicAdd(a.refs + page, 1);
        bad = true;
      }
      row[s] = -1;
    }
    count_lanes(a.err, bad);
  }
}

// ----------------------------------------------------------------------------
// share: row dst[i] becomes a second holder of row src[i]'s pages.
struct ShareArgs {
  int32_t* tables;
  int64_t stride;
  int32_t max_pages, batch;
  int32_t* kv_lens;
  const int32_t* src;
  const int32_t* dst;
  int32_t n;
  int32_t* refs;
  int32_t num_pages;
  int32_t* err;
};

__global__ void __launch_bounds__(kPageThreads) share_pages_kernel(ShareArgs a) {
  __shared__ int red[kPageThreads / kWave];
  const int i = blockIdx.x;
  const int s = a.src[i], d = a.dst[i];
  // a destination is nobody's source, and nobody else's destination
  int clash = 0;
  for (int j = (int)threadIdx.x; j < a.n; j += kPageThreads)
    if (a.src[j] == d || (j < i && a.dst[j] == d)) ++clash;
  clash = block_sum(clash, red);
  if (clash > 0 || s < 0 || s >= a.batch || d < 0 || d >= a.batch) {
    if (threadIdx.x == 0) count_lanes(a.err, true);
    return;
  }
  const int len = max(a.kv_lens[s], 0);
  const int n = (int)min<int64_t>(((int64_t)len + kPage - 1) / kPage, a.max_pages);
  const int32_t* from = a.tables + s * a.stride;
  int32_t* to = a.tables + d * a.stride;
  for (int k = (int)threadIdx.x; k < a.max_pages; k += kPageThreads) {
    int page = k < n ? from[k] : -1;
    const bool bad = page >= a.num_pages;
    if (bad) page = -1;
    if (page >= 0) atomicAdd(a.refs + page, 1);
    to[k] = page;
    count_lanes(a.err, bad);
  }
  if (threadIdx.x == 0) a.kv_lens[d] = len;
}

// ----------------------------------------------------------------------------
// compact: the n live pages move to ids [0, n).  Those already there stay; the
// k-th live page at or past n goes to the k-th free page below n, so no
// destination is a source and one launch can copy them all.  4950 pages of 4 layers
// x 32 KiB, 1.3 GB read and written: 246 us, 5.3 TB/s (a large copy moves 4.8);
// the ranks before it 12 us.  Pages are copied layer by layer in units of 16 KiB, 4
// loads of 16 bytes a thread at once, by one resident set of workgroups.
struct CompactArgs {
  int32_t* refs;
  int32_t num_pages, n_blocks;
  int32_t* remap;
  int32_t* tables;
  int64_t stride;
  int32_t max_pages, batch;
  int32_t* err;
  // scratch: live pages of each block, the moves, each page's move (kStays, kFree)
  int32_t* live_cnt;
  int32_t* n_live;
  int32_t* n_moves;
  int32_t* src;
  int32_t* dst;
  int32_t* move;
};
constexpr int32_t kStays = -1, kFree = -2;

__global__ void __launch_bounds__(kPageThreads) compact_count_kernel(CompactArgs a) {
  __shared__ int red[kPageWaves];
  Held held;
  held.load(a.refs, (int)blockIdx.x, a.num_pages, false);
  int before;
  const int n = waves_sum(held.count(), red, &before);
  if (threadIdx.x == 0) a.live_cnt[blockIdx.x] = n;
}

// COUNTS: the blocks' counts come from compact_count_kernel.  Pools of up to
// kOwnBlocks blocks are counted by every workgroup itself, which saves a launch.
constexpr int kOwnBlocks = 4;

template <bool COUNTS>
__global__ void __launch_bounds__(kPageThreads) compact_rank_kernel(CompactArgs a) {
  __shared__ int red[kPageWaves];
  const int blk = (int)blockIdx.x;
  Held held;  // on its way while the counts are summed
  held.load(a.refs, blk, a.num_pages, false);
  // live pages in all, and in the blocks before this one
  int n_live, before_blk, unused;
  int own[kOwnBlocks];  // the wave's share of every block's
  if constexpr (COUNTS) {
    int all = 0, mine = 0;
    for (int i = (int)threadIdx.x; i < a.n_blocks; i += kPageThreads) {
      const int n = a.live_cnt[i];
      all += n;
      mine += i < blk ? n : 0;
    }
    n_live = block_sum(all, red);
    before_blk = block_sum(mine, red);
  } else {
    int all = 0, mine = 0;
#pragma unroll
    for (int i = 0; i < kOwnBlocks; ++i) {
      own[i] = 0;
      if (i < a.n_blocks) {
        Held other;
        other.load(a.refs, i, a.num_pages, false);
        own[i] = other.count();
      }
      all += own[i];
      mine += i < blk ? own[i] : 0;
    }
    n_live = waves_sum(all, red, &unused);
    before_blk = waves_sum(mine, red, &unused);
  }
  // live pages below n_live, which stay
  const int line_blk = min(n_live / kPagesPerBlock, a.n_blocks - 1);
  Held at_line;
  at_line.load(a.refs, line_blk, a.num_pages, false);
  int stay = at_line.count_below(n_live);
  if constexpr (COUNTS) {
    stay = waves_sum(stay, red, &unused);
    stay += array_sum(a.live_cnt, line_blk, red);
  } else {
#pragma unroll
    for (int i = 0; i < kOwnBlocks; ++i) stay += i < line_blk ? own[i] : 0;
    stay = waves_sum(stay, red, &unused);
  }
  if (blk == 0 && threadIdx.x == 0) {
    *a.n_live = n_live;
    *a.n_moves = n_live - stay;
  }
  int before;  // live pages before the wave's first, then before each step's
  waves_sum(held.count(), red, &before);
  before += before_blk;
  const int lane = threadIdx.x & (kWave - 1);
#pragma unroll
  for (int k = 0; k < kPageSteps; ++k) {
    const int64_t p = held.page0 + k * kWave + lane;
    const bool is_live = (held.m[k] >> lane) & 1;
    const int rank = before + bits_below(held.m[k]);
    before += (int)__builtin_popcountll(held.m[k]);
    if (p >= a.num_pages) continue;
    int move = is_live ? kStays : kFree;
    if (is_live && p >= n_live) {
      move = rank - stay;
      a.src[move] = (int32_t)p;
    } else if (!is_live && p < n_live) {
      a.dst[(int)p - rank] = (int32_t)p;
    }
    a.move[p] = move;
    if (move < 0) a.remap[p] = is_live ? (int32_t)p : -1;
  }
}

// The moves: counts and remap entries, the tables' entries, and the pages.
__global__ void __launch_bounds__(kPageThreads) compact_move_kernel(CompactArgs a, CopyArgs c) {
  const int64_t t = (int64_t)blockIdx.x * kPageThreads + threadIdx.x;
  const int64_t n_threads = (int64_t)gridDim.x * kPageThreads;
  const int n_moves = *a.n_moves;
  for (int64_t k = t; k < n_moves; k += n_threads) {
    const int s = a.src[k], d = a.dst[k];
    a.refs[d] = a.refs[s];
    a.refs[s] = 0;
    a.remap[s] = d;
  }
  const int64_t entries = (int64_t)a.batch * a.max_pages;
  for (int64_t e = t; e < entries; e += n_threads) {
    int32_t* at = a.tables + e / a.max_pages * a.stride + e % a.max_pages;
    const int page = *at;
    if (page < 0) continue;
    const int move = page < a.num_pages ? a.move[page] : kFree;
    if (move >= 0) *at = a.dst[move];
    count_lanes(a.err, move == kFree);
  }
  copy_pages<false>(c, blockIdx.x, gridDim.x);
}

// ----------------------------------------------------------------------------
// host side
static int64_t scratch_ints(int64_t n) { return (n + 63) / 64 * 64; }

static int page_blocks(int32_t num_pages) {
  return (int)std::max<int64_t>(1, ((int64_t)num_pages + kPagesPerBlock - 1) / kPagesPerBlock);
}

// Workgroups of a copy: one resident set, 8 of 256 threads a CU.
static unsigned copy_grid() {
  const int cus = device_cu_count();
  return (unsigned)(8 * (cus > 0 ? cus : 256));
}

static int check_pool(const char* who, const void* kv_pool, int32_t dtype, int32_t num_layers,
                      int32_t num_pages, int32_t hkv, int32_t d, int32_t page_size,
                      const float* scales, CopyArgs* c) {
  if (page_size != kPage)
    return set_error(PAGEDATTN_ERR_UNSUPPORTED, "%s: page_size %d not supported (16)", who,
                     page_size);
  const int esz = dtype == PAGEDATTN_BF16 || dtype == PAGEDATTN_F16 ? 2
                  : dtype == PAGEDATTN_E4M3                         ? 1
                                                                    : 0;
  if (!esz)
    return set_error(PAGEDATTN_ERR_UNSUPPORTED, "%s: pool dtype %d not supported", who, dtype);
  if (num_layers <= 0 || num_pages < 0 || hkv <= 0 || d <= 0 || (d * esz) % 16 ||
      (int64_t)hkv * d > INT32_MAX / 2 / (2 * kPage * esz))
    return set_error(PAGEDATTN_ERR_INVALID,
                     "%s: bad shape layers=%d pages=%d hkv=%d d=%d (rows must be a multiple of "
                     "16 bytes)",
                     who, num_layers, num_pages, hkv, d);
  if (dtype == PAGEDATTN_E4M3 && !scales)
    return set_error(PAGEDATTN_ERR_INVALID, "%s: an e4m3 pool needs kv_scales", who);
  if (num_pages > 0 && (!kv_pool || !aligned16(kv_pool)))
    return set_error(PAGEDATTN_ERR_INVALID, "%s: null or misaligned pool", who);
  *c = CopyArgs{};
  c->pool = static_cast<uint8_t*>(const_cast<void*>(kv_pool));
  c->scales = dtype == PAGEDATTN_E4M3 ? const_cast<float*>(scales) : nullptr;
  c->num_layers = num_layers;
  c->num_pages = num_pages;
  c->blocks = 2 * hkv;
  c->row_bytes = d * esz;
  c->block_bytes = kPage * d * esz;
  c->units = (int)(((int64_t)c->blocks * c->block_bytes + kCopyUnit - 1) / kCopyUnit);
  if ((int64_t)num_layers * c->units > INT32_MAX)
    return set_error(PAGEDATTN_ERR_UNSUPPORTED, "%s: %d layers are too many", who, num_layers);
  return PAGEDATTN_OK;
}

static int check_tables(const char* who, const int32_t* tables, int64_t stride, int32_t max_pages,
                        int32_t batch, const int32_t* refs, int32_t num_pages) {
  if (batch < 0 || max_pages < 0 || stride < max_pages || num_pages < 0)
    return set_error(PAGEDATTN_ERR_INVALID,
                     "%s: bad sizes batch=%d max_pages=%d stride=%lld pages=%d", who, batch,
                     max_pages, (long long)stride, num_pages);
  if (batch > 65535 || (int64_t)batch * ((int64_t)max_pages + 1) > INT32_MAX)
    return set_error(PAGEDATTN_ERR_UNSUPPORTED,
                     "%s: batch_size %d above 65535, or with %d pages a row past 2^31 - 1 entries",
                     who, batch, max_pages);
  if (batch > 0 && max_pages > 0 && !tables)
    return set_error(PAGEDATTN_ERR_INVALID, "%s: null block_tables", who);
  if (num_pages > 0 && !refs)
    return set_error(PAGEDATTN_ERR_INVALID, "%s: null ref_counts", who);
  return PAGEDATTN_OK;
}

static int check_page_scratch(const char* who, const void* scratch, size_t have, size_t want) {
  if (!scratch || ((uintptr_t)scratch & 255))
    return set_error(PAGEDATTN_ERR_INVALID, "%s: the scratch must be 256-byte aligned", who);
  if (have < want)
    return set_error(PAGEDATTN_ERR_WORKSPACE, "%s: needs %zu scratch bytes, %zu given", who, want,
                     have);
  return PAGEDATTN_OK;
}

static int release(const char* who, ReleaseArgs a, void* stream) {
  if (a.batch == 0 || a.max_pages == 0) return PAGEDATTN_OK;
  // few slots a row are walked by one workgroup, long rows by up to 16
  const unsigned gx =
      (unsigned)std::max(1, std::min(16, (a.max_pages + kPageThreads - 1) / kPageThreads));
  hipLaunchKernelGGL(release_pages_kernel, dim3(gx, (unsigned)a.batch), dim3(kPageThreads), 0,
                     (hipStream_t)stream, a);
  return check_launch(who);
}

}  // namespace pa

using namespace pa;

extern "C" {

size_t pagedattn_page_scratch_bytes(int32_t num_pages, int32_t batch_size, int32_t max_pages) {
  if (num_pages < 0 || batch_size < 0 || max_pages < 0) return 0;
  const int64_t blocks = scratch_ints(page_blocks(num_pages));
  const int64_t reserve =
      blocks + 5 * scratch_ints(batch_size) + 64 +
      scratch_ints(std::min<int64_t>(num_pages, (int64_t)batch_size * ((int64_t)max_pages + 1)));
  const int64_t compact = blocks + 3 * scratch_ints(num_pages) + 64;
  return sizeof(int32_t) * (size_t)std::max(reserve, compact);
}

int pagedattn_reserve_pages(void* kv_pool, int32_t pool_dtype, int32_t num_layers,
                            int32_t num_pages, int32_t num_kv_heads, int32_t head_dim,
                            int32_t page_size, float* kv_scales, int32_t* block_tables,
                            int64_t table_stride, int32_t max_pages, const int32_t* kv_lens,
                            const int32_t* new_lens, int32_t batch_size, int32_t* ref_counts,
                            int32_t* error_flag, void* scratch, size_t scratch_bytes,
                            void* stream) {
  const char* who = "reserve_pages";
  CopyArgs c;
  int rc = check_pool(who, kv_pool, pool_dtype, num_layers, num_pages, num_kv_heads, head_dim,
                      page_size, kv_scales, &c);
  if (!rc)
    rc = check_tables(who, block_tables, table_stride, max_pages, batch_size, ref_counts,
                      num_pages);
  if (rc) return rc;
  if (batch_size == 0) return PAGEDATTN_OK;
  if (!kv_lens) return set_error(PAGEDATTN_ERR_INVALID, "%s: null kv_lens", who);
  rc = check_page_scratch(who, scratch, scratch_bytes,
                          pagedattn_page_scratch_bytes(num_pages, batch_size, max_pages));
  if (rc) return rc;
  ReserveArgs a{};
  a.tables = block_tables;
  a.stride = table_stride;
  a.max_pages = max_pages;
  a.batch = batch_size;
  a.kv_lens = kv_lens;
  a.new_lens = new_lens;
  a.refs = ref_counts;
  a.num_pages = num_pages;
  a.n_blocks = page_blocks(num_pages);
  a.err = error_flag;
  int32_t* at = static_cast<int32_t*>(scratch);
  auto take = [&](int64_t n) {
    int32_t* p = at;
    at += scratch_ints(n);
    return p;
  };
  a.need = take(batch_size);
  a.base = take(batch_size);
  a.fork_src = take(batch_size);
  a.fork_rank = take(batch_size);
  a.fork_rows = take(batch_size);
  a.free_cnt = take(a.n_blocks);
  a.n_forks = take(64);
  a.short_of = a.n_forks + 1;
  a.fresh = at;
  hipStream_t s = (hipStream_t)stream;
  const bool counts = a.n_blocks > kReserveBlocks || batch_size > kOwnRows;
  if (counts) {
    const unsigned waves =
        (unsigned)((batch_size + kPageThreads / kWave - 1) / (kPageThreads / kWave));
    hipLaunchKernelGGL(reserve_count_kernel, dim3((unsigned)a.n_blocks + waves),
                       dim3(kPageThreads), 0, s, a);
    rc = check_launch(who);
    if (rc) return rc;
  }
  hipLaunchKernelGGL(counts ? reserve_rank_kernel<true> : reserve_rank_kernel<false>,
                     dim3((unsigned)a.n_blocks + 1), dim3(kPageThreads), 0, s, a);
  rc = check_launch(who);
  if (rc) return rc;
  c.count = a.n_forks;
  c.src = a.fork_src;
  c.dst = a.fresh;
  c.dst_at = a.fork_rank;
  c.rows = a.fork_rows;
  const int64_t units = (int64_t)batch_size * num_layers * c.units;
  hipLaunchKernelGGL(reserve_assign_kernel, dim3((unsigned)std::min<int64_t>(units, copy_grid())),
                     dim3(kPageThreads), 0, s, a, c);
  return check_launch(who);
}

int pagedattn_release_pages(int32_t* block_tables, int64_t table_stride, int32_t max_pages,
                            int32_t batch_size, int32_t* ref_counts, int32_t num_pages,
                            const int32_t* first_slots, const int32_t* last_slots,
                            int32_t* error_flag, void* stream) {
  const char* who = "release_pages";
  const int rc = check_tables(who, block_tables, table_stride, max_pages, batch_size, ref_counts,
                              num_pages);
  if (rc) return rc;
  return release(who,
                 ReleaseArgs{block_tables, table_stride, max_pages, batch_size, ref_counts,
                             num_pages, first_slots, last_slots, nullptr, 0, 0, error_flag},
                 stream);
}

int pagedattn_release_window_pages(int32_t* block_tables, int64_t table_stride, int32_t max_pages,
                                   const int32_t* kv_lens, int32_t batch_size,
                                   int32_t* ref_counts, int32_t num_pages, int32_t window_left,
                                   int32_t sinks, int32_t* error_flag, void* stream) {
  const char* who = "release_window_pages";
  const int rc = check_tables(who, block_tables, table_stride, max_pages, batch_size, ref_counts,
                              num_pages);
  if (rc) return rc;
  if (window_left < 0 || sinks < 0)
    return set_error(PAGEDATTN_ERR_INVALID, "%s: window_left %d and sinks %d must not be negative",
                     who, window_left, sinks);
  if (batch_size > 0 && !kv_lens)
    return set_error(PAGEDATTN_ERR_INVALID, "%s: null kv_lens", who);
  return release(who,
                 ReleaseArgs{block_tables, table_stride, max_pages, batch_size, ref_counts,
                             num_pages, nullptr, nullptr, kv_lens, window_left, sinks, error_flag},
                 stream);
}

int pagedattn_share_pages(int32_t* block_tables, int64_t table_stride, int32_t max_pages,
                          int32_t* kv_lens, int32_t batch_size, const int32_t* src_rows,
                          const int32_t* dst_rows, int32_t num_shares, int32_t* ref_counts,
                          int32_t num_pages, int32_t* error_flag, void* stream) {
  const char* who = "share_pages";
  const int rc = check_tables(who, block_tables, table_stride, max_pages, batch_size, ref_counts,
                              num_pages);
  if (rc) return rc;
  if (num_shares < 0)
    return set_error(PAGEDATTN_ERR_INVALID, "%s: num_shares %d < 0", who, num_shares);
  if (num_shares == 0) return PAGEDATTN_OK;
  if (!kv_lens || !src_rows || !dst_rows)
    return set_error(PAGEDATTN_ERR_INVALID, "%s: null pointer", who);
  ShareArgs a{block_tables, table_stride, max_pages, batch_size, kv_lens, src_rows,
              dst_rows, num_shares, ref_counts, num_pages, error_flag};
  hipLaunchKernelGGL(share_pages_kernel, dim3((unsigned)num_shares), dim3(kPageThreads), 0,
                     (hipStream_t)stream, a);
  return check_launch(who);
}

int pagedattn_compact_pages(void* kv_pool, int32_t pool_dtype, int32_t num_layers,
                            int32_t num_pages, int32_t num_kv_heads, int32_t head_dim,
                            int32_t page_size, float* kv_scales, int32_t* block_tables,
                            int64_t table_stride, int32_t max_pages, int32_t batch_size,
                            int32_t* ref_counts, int32_t* remap, int32_t* error_flag,
                            void* scratch, size_t scratch_bytes, void* stream) {
  const char* who = "compact_pages";
  CopyArgs c;
  int rc = check_pool(who, kv_pool, pool_dtype, num_layers, num_pages, num_kv_heads, head_dim,
                      page_size, kv_scales, &c);
  if (!rc)
    rc = check_tables(who, block_tables, table_stride, max_pages, batch_size, ref_counts,
                      num_pages);
  if (rc) return rc;
  if (num_pages == 0) return PAGEDATTN_OK;
  if (!remap) return set_error(PAGEDATTN_ERR_INVALID, "%s: null remap", who);
  rc = check_page_scratch(who, scratch, scratch_bytes,
                          pagedattn_page_scratch_bytes(num_pages, batch_size, max_pages));
  if (rc) return rc;
  CompactArgs a{};
  a.refs = ref_counts;
  a.num_pages = num_pages;
  a.n_blocks = page_blocks(num_pages);
  a.remap = remap;
  a.tables = block_tables;
  a.stride = table_stride;
  a.max_pages = max_pages;
  a.batch = batch_size;
  a.err = error_flag;
  int32_t* at = static_cast<int32_t*>(scratch);
  auto take = [&](int64_t n) {
    int32_t* p = at;
    at += scratch_ints(n);
    return p;
  };
  a.live_cnt = take(a.n_blocks);
  a.src = take(num_pages);
  a.dst = take(num_pages);
  a.move = take(num_pages);
  a.n_live = at;
  a.n_moves = at + 1;
  hipStream_t s = (hipStream_t)stream;
  const bool counts = a.n_blocks > kOwnBlocks;
  if (counts) {
    hipLaunchKernelGGL(compact_count_kernel, dim3((unsigned)a.n_blocks), dim3(kPageThreads), 0, s,
                       a);
    rc = check_launch(who);
    if (rc) return rc;
  }
  hipLaunchKernelGGL(counts ? compact_rank_kernel<true> : compact_rank_kernel<false>,
                     dim3((unsigned)a.n_blocks), dim3(kPageThreads), 0, s, a);
  rc = check_launch(who);
  if (rc) return rc;
  c.count = a.n_moves;
  c.src = a.src;
  c.dst = a.dst;
  hipLaunchKernelGGL(compact_move_kernel, dim3(copy_grid()), dim3(kPageThreads), 0, s, a, c);
  return check_launch(who);
}

}  // extern "C"
