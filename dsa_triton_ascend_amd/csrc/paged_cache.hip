// Pages of a cache: writing new tokens' rows, forking / releasing / extending
// the block table's rows, planning a step of rows of many lengths, finding the
// prefixes that rows share, and compaction.
//
// A cache is [pages, page_size, row]; several caches (latent, rope, indexer
// keys, of several layers) share one block table, and one call moves the rows
// of all of them.  Rows are moved as bytes, in the widest unit (16 bytes down
// to 1) that row sizes and addresses allow.
//
// All of it is planned on the device: lengths, counts and free pages are
// never read by the host, so a call can be captured into a graph.  Free pages
// are handed out in ascending order to rows in ascending order, integer
// counts are the only atomics, so results do not depend on timing.
//
// Bound by the launches for one step's tables (a fork of 16 rows: 3.8 + 4.8 us
// for its two kernels, a write of 32 rows 3.9, of 8192 rows 8.4), by memory
// where pages move (half of a 740 MB pool in use: 369 MB read and written in
// 76.5 us, 4.8 TB/s; a large copy reaches 4.9).  A plan of 256 rows over 85000
// pages takes 5.5 + 3.6 us, writing 8192 rows of a plan 6.9 (22 MB; one
// dependent read less than a write that searches the tables, 8.4).
#include "common.h"

namespace dsa {

constexpr int kPcMaxCaches = 32;  // caches of one launch; more take more launches
constexpr int kPcThreads = 256;
constexpr int kPcPlanThreads = 1024;
constexpr int kPcChunk = kPcThreads * 4;  // units of a copy block

struct PcCache {
  const unsigned char* src;      // new rows (write)
  unsigned char* dst;            // the cache
  int64_t src_sb, src_st;        // strides of the new rows in bytes: batch, token
  int64_t page_bytes;
  int row_bytes;
  int shift;                     // log2 of the unit
  int unit0;                     // first unit of this cache among a token's (write)
  int chunk0;                    // first chunk of this cache among a page's (copies)
};

// widest unit that divides all the given sizes and addresses
static int pc_shift(uint64_t bits) {
  int s = 4;
  while (s > 0 && (bits & ((1u << s) - 1))) --s;
  return s;
}

__device__ __forceinline__ void pc_move(unsigned char* dst, const unsigned char* src, int shift) {
  switch (shift) {
    case 4: *(u32x4*)dst = *(const u32x4*)src; break;
    case 3: *(uint64_t*)dst = *(const uint64_t*)src; break;
    case 2: *(uint32_t*)dst = *(const uint32_t*)src; break;
    case 1: *(uint16_t*)dst = *(const uint16_t*)src; break;
    default: *dst = *src;
  }
}

// ---------------------------------------------------------------------------
// write: one thread per unit of a token's rows
// ---------------------------------------------------------------------------
struct PcWriteParams {
  PcCache c[kPcMaxCaches];
  int n;
  const int32_t *table, *lens, *rows;  // rows: per-sequence counts (BSND, may be null) or cumulative (TND)
  int64_t tokens, pages;
  int batch, s, max_blocks, page, tnd, units;
};

__global__ __launch_bounds__(kPcThreads) void pc_write_kernel(PcWriteParams p) {
  const int64_t i = (int64_t)blockIdx.x * kPcThreads + threadIdx.x;
  const int64_t t = i >> 32 ? i / p.units : (int64_t)((unsigned)i / (unsigned)p.units);
  if (t >= p.tokens) return;
  const int u = (int)(i - t * p.units);
  int b, s;
  if (p.tnd) {
    int lo = 0, hi = p.batch;  // first b with rows[b] > t
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (p.rows[mid] > t) hi = mid; else lo = mid + 1;
    }
    if (lo == p.batch) return;  // rows behind the last sequence
    b = lo;
    s = (int)(t - (b ? p.rows[b - 1] : 0));
    if (s < 0) return;  // (a count of -2^31 before it)
  } else {
    b = (int)(t / p.s);
    s = (int)(t - (int64_t)b * p.s);
    if (p.rows && s >= p.rows[b]) return;
  }
  const unsigned pos = (unsigned)max(p.lens[b], 0) + (unsigned)s;  // both are below 2^31
  const unsigned slot = pos / (unsigned)p.page;
  int ci = 0;
  while (ci + 1 < p.n && u >= p.c[ci + 1].unit0) ++ci;
  const PcCache& c = p.c[ci];
  const int64_t off = (int64_t)(u - c.unit0) << c.shift;
  const unsigned char* src = (p.tnd ? c.src + t * c.src_st : c.src + b * c.src_sb + s * c.src_st) + off;
  // (the row is read beside the table, not behind it)
  const u32x4 wide = c.shift == 4 ? *(const u32x4*)src : u32x4{0, 0, 0, 0};
  if (slot >= (unsigned)p.max_blocks) return;
  const int blk = p.table[(int64_t)b * p.max_blocks + slot];
  if (blk < 0 || blk >= p.pages) return;
  unsigned char* dst = c.dst + blk * c.page_bytes + (int64_t)(pos - slot * (unsigned)p.page) * c.row_bytes + off;
  if (c.shift == 4) *(u32x4*)dst = wide;
  else pc_move(dst, src, c.shift);
}

int pc_write_run(int64_t n, const void* const* rows, void* const* caches, const int64_t* row_bytes,
                 const int64_t* row_sb, const int64_t* row_st, const int32_t* table, const int32_t* lens,
                 const int32_t* row_lengths, int64_t batch, int64_t s, int64_t tokens, int64_t max_blocks,
                 int64_t pages, int64_t page, int32_t layout, hipStream_t stream) {
  PcWriteParams p = {};
  p.table = table;
  p.lens = lens;
  p.rows = row_lengths;
  p.tokens = tokens;
  p.pages = pages;
  p.batch = (int)batch;
  p.s = (int)s;
  p.max_blocks = (int)max_blocks;
  p.page = (int)page;
  p.tnd = layout == DSA_LAYOUT_TND;
  // blocks of the launch for the caches from c0 on
  auto take = [&](int64_t c0) {
    p.n = (int)(n - c0 < kPcMaxCaches ? n - c0 : kPcMaxCaches);
    int64_t units = 0;
    for (int i = 0; i < p.n; ++i) {
      PcCache& c = p.c[i];
      const int64_t k = c0 + i;
      c.src = (const unsigned char*)rows[k];
      c.dst = (unsigned char*)caches[k];
      c.src_sb = row_sb[k];
      c.src_st = row_st[k];
      c.row_bytes = (int)row_bytes[k];
      c.page_bytes = row_bytes[k] * page;
      c.shift = pc_shift((uint64_t)(uintptr_t)c.src | (uintptr_t)c.dst | (uint64_t)row_bytes[k] |
                         (uint64_t)row_sb[k] | (uint64_t)row_st[k]);
      c.unit0 = (int)units;
      units += row_bytes[k] >> c.shift;
    }
    p.units = (int)units;  // (at most 32 rows of 2^24 bytes)
    return (tokens * units + kPcThreads - 1) / kPcThreads;
  };
  // (all of them before the first: a call that is refused has written nothing)
  for (int64_t c0 = n > kPcMaxCaches ? 0 : n; c0 < n; c0 += kPcMaxCaches)
    DSA_CHECK_SUPPORTED(launchable(take(c0), kPcThreads), "too many rows for one call");
  for (int64_t c0 = 0; c0 < n; c0 += kPcMaxCaches) {
    const int64_t grid = take(c0);
    DSA_CHECK_SUPPORTED(launchable(grid, kPcThreads), "too many rows for one call");
    pc_write_kernel<<<dim3((unsigned)grid), kPcThreads, 0, stream>>>(p);
    DSA_HIP(hipGetLastError());
  }
  return DSA_OK;
}

// ---------------------------------------------------------------------------
// page copies
// ---------------------------------------------------------------------------
struct PcCopySet {
  PcCache c[kPcMaxCaches];
  int n, chunks;  // chunks of a page over all caches
};

// One block's chunk of a copy of the first `tok` tokens of page src to dst.
__device__ __forceinline__ void pc_copy_chunk(const PcCopySet& s, int chunk, int64_t src, int64_t dst, int tok) {
  int ci = 0;
  while (ci + 1 < s.n && chunk >= s.c[ci + 1].chunk0) ++ci;
  const PcCache& c = s.c[ci];
  const int64_t units = ((int64_t)tok * c.row_bytes) >> c.shift;
  const int64_t u0 = (int64_t)(chunk - c.chunk0) * kPcChunk + threadIdx.x;
  const unsigned char* from = c.dst + src * c.page_bytes;
  unsigned char* to = c.dst + dst * c.page_bytes;
  if (c.shift == 4) {
    // all loads of the chunk before its stores: four in flight per lane
    u32x4 v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (u0 + j * kPcThreads < units) v[j] = *(const u32x4*)(from + ((u0 + j * kPcThreads) << 4));
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (u0 + j * kPcThreads < units) *(u32x4*)(to + ((u0 + j * kPcThreads) << 4)) = v[j];
    return;
  }
  for (int j = 0; j < 4; ++j) {
    const int64_t u = u0 + j * kPcThreads;
    if (u < units) pc_move(to + (u << c.shift), from + (u << c.shift), c.shift);
  }
}

static int64_t pc_copy_set(PcCopySet& s, int64_t c0, int64_t n, void* const* caches, const int64_t* row_bytes,
                           int64_t page) {
  s.n = (int)(n - c0 < kPcMaxCaches ? n - c0 : kPcMaxCaches);
  int64_t chunks = 0;
  for (int i = 0; i < s.n; ++i) {
    PcCache& c = s.c[i];
    c = {};
    c.dst = (unsigned char*)caches[c0 + i];
    c.row_bytes = (int)row_bytes[c0 + i];
    c.page_bytes = row_bytes[c0 + i] * page;
    c.shift = pc_shift((uint64_t)(uintptr_t)c.dst | (uint64_t)c.row_bytes);
    c.chunk0 = (int)chunks;
    chunks += ((c.page_bytes >> c.shift) + kPcChunk - 1) / kPcChunk;
  }
  s.chunks = (int)chunks;
  return chunks;
}

// inclusive sum over the threads of a block of W waves; *total gets all of it
template <int W>
__device__ __forceinline__ int pc_block_scan(int v, int* s_part, int* total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int x = wave_scan(v);
  __syncthreads();  // s_part of the scan before is read
  if (lane == 63) s_part[wave] = x;
  __syncthreads();
  int base = 0, all = 0;
#pragma unroll
  for (int w = 0; w < W; ++w) {
    const int q = s_part[w];
    base += w < wave ? q : 0;
    all += q;
  }
  *total = all;
  return base + x;
}

// ---------------------------------------------------------------------------
// fork
// ---------------------------------------------------------------------------
struct PcForkParams {
  PcCopySet set;
  const int32_t *table, *lens, *refs, *parents;  // parents null: row c continues row c
  int32_t *new_table, *new_lens, *new_refs;
  int32_t *first, *start, *flags, *freelist;     // workspace (first: for more rows than kPcRowsHere)
  int64_t pages, new_tokens;
  int rows, children, max_blocks, new_blocks, page;
  int table_blocks;                              // blocks of the tables in the second launch
};

struct PcChild {
  int parent, len, held, want;  // pages held by its tokens, pages wanted with room for the new ones
};

__device__ __forceinline__ PcChild pc_child(const PcForkParams& p, int c) {
  PcChild k = {p.parents ? p.parents[c] : c, 0, 0, 0};
  if (k.parent < 0 || k.parent >= p.rows) {
    k.parent = -1;
    return k;
  }
  // a length past the table's end is the table's end
  const int64_t room = (int64_t)p.max_blocks * p.page;
  k.len = (int)min((int64_t)max(p.lens[k.parent], 0), room);
  // (below 2^26 tokens, 2^31 new ones, 2^20 of a page: the sums fit 32 bits)
  const unsigned page = (unsigned)p.page;
  k.held = (int)(((unsigned)k.len + page - 1) / page);
  k.want = (int)min(((unsigned)k.len + (unsigned)p.new_tokens + page - 1) / page, 0x7fffffffu);
  return k;
}

// Last page of the child's tokens where it is partly filled and has to be
// copied, else -1: the first child of a row keeps the row's own page, where
// nothing else refers to it.
__device__ __forceinline__ int pc_copied_page(const PcForkParams& p, const PcChild& k, int c, int first) {
  if (k.parent < 0 || k.len % p.page == 0) return -1;
  const int e = p.table[(int64_t)k.parent * p.max_blocks + k.held - 1];
  if (e < 0 || e >= p.pages) return -1;
  return first == c && p.refs[e] == 1 ? -1 : e;
}

constexpr int kPcRowsHere = 4096;  // rows whose first children the plan finds in LDS

// Block 0 plans: which rows need how many pages, and which free ones those
// are.  The other blocks copy the counts for the second launch to change.
// One workgroup is enough for the rows of a batch, not for a table of many
// thousands: whole forks of rows of 32 pages, captured, take 7 to 8 us for 16
// rows, 8 to 9 for 256, 10 to 11 for 1024, 24 to 28 for 4096 and 400 to 630 for
// 65536 (rows that continue themselves, and four from one parent).
__global__ __launch_bounds__(kPcPlanThreads) void pc_fork_plan_kernel(PcForkParams p) {
  const int tid = threadIdx.x;
  if (blockIdx.x > 0) {
    for (int64_t i = (int64_t)(blockIdx.x - 1) * kPcPlanThreads + tid; i < p.pages;
         i += (int64_t)(gridDim.x - 1) * kPcPlanThreads)
      p.new_refs[i] = p.refs[i];
    return;
  }
  __shared__ int s_part[kPcPlanThreads / 64];
  __shared__ int s_first[kPcRowsHere];
  // (the first counts are on their way beside what follows)
  int early[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) early[j] = 4 * tid + j < p.pages ? p.refs[4 * tid + j] : 1;
  // the first child of each row
  const bool here = p.rows <= kPcRowsHere;
  if (here) {
    for (int b = tid; b < p.rows; b += kPcPlanThreads) s_first[b] = 0x7fffffff;
  } else {
    for (int b = tid; b < p.rows; b += kPcPlanThreads)
      __hip_atomic_store(p.first + b, 0x7fffffff, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  for (int c = tid; c < p.children; c += kPcPlanThreads) {
    const int par = p.parents ? p.parents[c] : c;
    if (par >= 0 && par < p.rows) {
      if (here) atomicMin(s_first + par, c);
      else atomicMin(p.first + par, c);
    }
  }
  __syncthreads();
  auto first_of = [&](int row) {
    if (row < 0) return -1;
    if (here) return s_first[row];
    return __hip_atomic_load(p.first + row, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  };
  // pages that the rows before each row take; a row that does not fit the
  // new table takes none and is marked
  int64_t taken = 0;
  for (int c0 = 0; c0 < p.children; c0 += kPcPlanThreads) {
    const int c = c0 + tid;
    int need = 0;
    if (c < p.children) {
      const PcChild k = pc_child(p, c);
      int copies = 0;
      if (k.want > p.new_blocks) need = -1;
      else if (k.parent >= 0) {
        copies = pc_copied_page(p, k, c, first_of(k.parent)) >= 0;
        need = copies + k.want - k.held;
      }
      p.flags[c] = need * 2 + copies;
    }
    int total;
    const int mine = max(need, 0);
    const int incl = pc_block_scan<kPcPlanThreads / 64>(mine, s_part, &total);
    if (c < p.children) p.start[c] = (int)min(taken + incl - mine, (int64_t)0x7fffffff);
    taken += total;
  }
  // free pages in ascending order until that many are found
  int64_t found = 0;
  for (int64_t i0 = 0; i0 < p.pages && found < taken; i0 += 4 * kPcPlanThreads) {
    int fr[4], n = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t i = i0 + 4 * tid + j;
      fr[j] = i0 == 0 ? early[j] == 0 : (i < p.pages ? p.refs[i] == 0 : 0);
      n += fr[j];
    }
    int total;
    int64_t at = found + pc_block_scan<kPcPlanThreads / 64>(n, s_part, &total) - n;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (fr[j]) p.freelist[at++] = (int)(i0 + 4 * tid + j);
    found += total;
  }
  // a row is served if it needs nothing, or if the free pages last for it
  // and all before it; flags: bit 0 served, bit 1 its last page is a copy
  for (int c = tid; c < p.children; c += kPcPlanThreads) {
    const int f = p.flags[c], need = f >> 1;
    const int served = need == 0 || (need > 0 && (int64_t)p.start[c] + need <= found);
    p.flags[c] = served | (f & 1) << 1;
  }
}

__global__ __launch_bounds__(kPcThreads) void pc_fork_kernel(PcForkParams p) {
  const int tid = threadIdx.x;
  if ((int)blockIdx.x < p.table_blocks) {
    const int64_t stride = (int64_t)p.table_blocks * kPcThreads, me = (int64_t)blockIdx.x * kPcThreads + tid;
    for (int64_t i = me; i < (int64_t)p.rows * p.max_blocks; i += stride) {
      const int e = p.table[i];
      if (e >= 0 && e < p.pages) atomicSub(p.new_refs + e, 1);
    }
    for (int64_t i = me; i < (int64_t)p.children * p.new_blocks; i += stride) {
      const int c = i >> 32 ? (int)(i / p.new_blocks) : (int)((unsigned)i / (unsigned)p.new_blocks);
      const int col = (int)(i - (int64_t)c * p.new_blocks);
      const PcChild k = pc_child(p, c);
      const int flags = p.flags[c];
      const bool served = k.parent >= 0 && (flags & 1);
      int e = -1;
      if (served && col < k.want) {
        const int copies = flags >> 1;
        if (col >= k.held) e = p.freelist[p.start[c] + copies + col - k.held];
        else if (copies && col == k.held - 1) e = p.freelist[p.start[c]];
        else e = p.table[(int64_t)k.parent * p.max_blocks + col];
        if (e < 0 || e >= p.pages) e = -1;
      }
      p.new_table[i] = e;
      if (e >= 0) atomicAdd(p.new_refs + e, 1);
    }
    for (int64_t c = me; c < p.children; c += stride) {
      const PcChild k = pc_child(p, (int)c);
      p.new_lens[c] = k.parent < 0 ? 0 : (p.flags[c] & 1 ? k.len : -1);
    }
    return;
  }
  const int64_t w = (int64_t)blockIdx.x - p.table_blocks;
  const int c = (int)((unsigned)w / (unsigned)p.set.chunks);  // (the grid is below 2^31)
  if (p.flags[c] != 3) return;
  const PcChild k = pc_child(p, c);
  const int src = p.table[(int64_t)k.parent * p.max_blocks + k.held - 1];
  pc_copy_chunk(p.set, (int)(w - (int64_t)c * p.set.chunks), src, p.freelist[p.start[c]], k.len % p.page);
}

size_t pc_fork_workspace_bytes(int64_t rows, int64_t children, int64_t pages) {
  return (size_t)(rows + 2 * children + pages) * sizeof(int32_t);
}

int pc_fork_run(int64_t n, void* const* caches, const int64_t* row_bytes, const int32_t* table, const int32_t* lens,
                const int32_t* refs, const int32_t* parents, int32_t* new_table, int32_t* new_lens,
                int32_t* new_refs, int64_t rows, int64_t children, int64_t max_blocks, int64_t new_blocks,
                int64_t pages, int64_t page, int64_t new_tokens, void* workspace, hipStream_t stream) {
  PcForkParams p = {};
  p.table = table;
  p.lens = lens;
  p.refs = refs;
  p.parents = parents;
  p.new_table = new_table;
  p.new_lens = new_lens;
  p.new_refs = new_refs;
  p.first = (int32_t*)workspace;
  p.start = p.first + rows;
  p.flags = p.start + children;
  p.freelist = p.flags + children;
  p.pages = pages;
  p.new_tokens = new_tokens;
  p.rows = (int)rows;
  p.children = (int)children;
  p.max_blocks = (int)max_blocks;
  p.new_blocks = (int)new_blocks;
  p.page = (int)page;
  int64_t copy_blocks = (pages + 4 * kPcPlanThreads - 1) / (4 * kPcPlanThreads);
  copy_blocks = copy_blocks > 64 ? 64 : copy_blocks;
  const int64_t entries = rows * max_blocks > children * new_blocks ? rows * max_blocks : children * new_blocks;
  int64_t tb = (entries + 2 * kPcThreads - 1) / (2 * kPcThreads);
  tb = tb < 1 ? 1 : (tb > 1024 ? 1024 : tb);
  // (all launches before the first: a call that is refused has changed no cache)
  for (int64_t c0 = n > kPcMaxCaches ? 0 : n; c0 < n; c0 += kPcMaxCaches)
    DSA_CHECK_SUPPORTED(launchable(tb + children * pc_copy_set(p.set, c0, n, caches, row_bytes, page), kPcThreads),
                        "too many rows and pages for one call");
  bool first = true;
  for (int64_t c0 = 0; first || c0 < n; c0 += kPcMaxCaches, first = false) {
    const int64_t chunks = pc_copy_set(p.set, c0, n, caches, row_bytes, page);  // (32 pages of 2^31 bytes: below 2^26)
    p.table_blocks = first ? (int)tb : 0;
    const int64_t grid = p.table_blocks + children * chunks;
    DSA_CHECK_SUPPORTED(launchable(grid, kPcThreads), "too many rows and pages for one call");
    if (first) pc_fork_plan_kernel<<<dim3((unsigned)(1 + copy_blocks)), kPcPlanThreads, 0, stream>>>(p);
    if (grid > 0) pc_fork_kernel<<<dim3((unsigned)grid), kPcThreads, 0, stream>>>(p);
    DSA_HIP(hipGetLastError());
  }
  return DSA_OK;
}

// ---------------------------------------------------------------------------
// compact: n live pages go to the ids below n.  The k-th live page at an id
// of n or above moves to the k-th free id below n, so no page is both read
// and written and the moves need no order.
// ---------------------------------------------------------------------------
// Up to this many pages every block of the rank kernel counts the live pages by
// itself: a block's 1024 threads read 16 counts each.  Whole calls, captured,
// without and with a launch that counts first: 8192 pages 9.9 and 11.8 us,
// 16384 11.4 and 12.3, 24576 13.2 and 13.9, 32768 15.3 and 15.9, 65536 25.4 and
// 22.6 (each block reads all counts, so what they read grows with the square).
constexpr int64_t kPcCountsHere = 16384;

struct PcCompactParams {
  PcCopySet set;
  const int32_t *table, *refs;
  int32_t *new_table, *new_refs, *page_map;
  // workspace: live pages of each chunk (where they are counted first), ranks, moved pages and their places
  int32_t *live, *rank, *high, *hole;
  int64_t pages, entries;
  int chunks;                          // chunks of kPcPlanThreads pages
  int table_blocks, copy_blocks;
  int counts_here;                     // the ranks are found without a launch that counts first
};

__global__ __launch_bounds__(kPcPlanThreads) void pc_count_kernel(PcCompactParams p) {
  const int64_t i = (int64_t)blockIdx.x * kPcPlanThreads + threadIdx.x;
  const int n = __syncthreads_count(i < p.pages && p.refs[i] > 0);
  if (threadIdx.x == 0) p.live[blockIdx.x] = n;
}

// live pages before chunk `upto` and in all
template <int W>
__device__ __forceinline__ void pc_live(const PcCompactParams& p, int upto, int* s_part, int* before, int* all) {
  int a = 0, b = 0;
  for (int i = threadIdx.x; i < p.chunks; i += W * 64) {
    const int v = p.live[i];
    b += v;
    a += i < upto ? v : 0;
  }
  pc_block_scan<W>(a, s_part, before);
  pc_block_scan<W>(b, s_part, all);
}

__global__ __launch_bounds__(kPcPlanThreads) void pc_rank_kernel(PcCompactParams p) {
  constexpr int W = kPcPlanThreads / 64;
  __shared__ int s_part[W];
  int before, n, low, total, dummy;
  if (p.counts_here) {
    // few pages: every block counts them all
    int a = 0, b = 0;
    const int pages = (int)p.pages, mine = (int)blockIdx.x * kPcPlanThreads;
#pragma unroll 8
    for (int i = threadIdx.x; i < pages; i += kPcPlanThreads) {
      const int v = p.refs[i] > 0;
      b += v;
      a += i < mine ? v : 0;
    }
    pc_block_scan<W>(a, s_part, &before);
    pc_block_scan<W>(b, s_part, &n);
    int c = 0;
#pragma unroll 8
    for (int i = threadIdx.x; i < n; i += kPcPlanThreads) c += p.refs[i] > 0;
    pc_block_scan<W>(c, s_part, &low);
  } else {
    pc_live<W>(p, blockIdx.x, s_part, &before, &n);
    // live pages below id n: the chunks before n's, and that chunk's own part
    const int nc = n / kPcPlanThreads;
    pc_live<W>(p, nc, s_part, &low, &dummy);
    const int64_t in = (int64_t)nc * kPcPlanThreads + threadIdx.x;
    pc_block_scan<W>(in < n && p.refs[in] > 0, s_part, &dummy);
    low += dummy;
  }
  const int64_t i = (int64_t)blockIdx.x * kPcPlanThreads + threadIdx.x;
  const int lv = i < p.pages && p.refs[i] > 0;
  const int at = before + pc_block_scan<W>(lv, s_part, &total) - lv;  // live pages before i
  // live pages and moved ones, for the next launch: at most half the pages
  // move, so the lists' last places are free
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    p.high[p.pages - 1] = n;
    p.hole[p.pages - 1] = n - low;
  }
  if (i >= p.pages) return;
  int k = -1;
  if (lv && i >= n) {
    k = at - low;
    p.high[k] = (int)i;
  } else if (!lv && i < n) {
    k = (int)i - at;
    p.hole[k] = (int)i;
  }
  p.rank[i] = k;
}

__device__ __forceinline__ int pc_place(const PcCompactParams& p, int64_t i, int n) {
  if (p.refs[i] <= 0) return -1;
  return i < n ? (int)i : p.hole[p.rank[i]];
}

__global__ __launch_bounds__(kPcThreads) void pc_compact_kernel(PcCompactParams p) {
  const int tid = threadIdx.x;
  const int n = p.high[p.pages - 1];
  if ((int)blockIdx.x < p.table_blocks) {
    const int64_t stride = (int64_t)p.table_blocks * kPcThreads, me = (int64_t)blockIdx.x * kPcThreads + tid;
    for (int64_t i = me; i < p.entries; i += stride) {
      const int e = p.table[i];
      p.new_table[i] = e >= 0 && e < p.pages ? pc_place(p, e, n) : -1;
    }
    for (int64_t i = me; i < p.pages; i += stride) {
      const int r = p.refs[i];
      p.page_map[i] = pc_place(p, i, n);
      p.new_refs[i] = i >= n ? 0 : (r > 0 ? r : p.refs[p.high[p.rank[i]]]);
    }
    return;
  }
  const int64_t work = (int64_t)p.hole[p.pages - 1] * p.set.chunks;
  for (int64_t w = (int64_t)blockIdx.x - p.table_blocks; w < work; w += p.copy_blocks) {
    const int k = (int)(w / p.set.chunks);
    const int64_t src = p.high[k], dst = p.hole[k];
    pc_copy_chunk(p.set, (int)(w - (int64_t)k * p.set.chunks), src, dst, p.set.n ? (int)(p.set.c[0].page_bytes / p.set.c[0].row_bytes) : 0);
  }
}

size_t pc_compact_workspace_bytes(int64_t pages) {
  const int64_t chunks = (pages + kPcPlanThreads - 1) / kPcPlanThreads;
  return (size_t)(chunks + 3 * pages) * sizeof(int32_t);
}

int pc_compact_run(int64_t n, void* const* caches, const int64_t* row_bytes, const int32_t* table,
                   const int32_t* refs, int32_t* new_table, int32_t* new_refs, int32_t* page_map, int64_t entries,
                   int64_t pages, int64_t page, void* workspace, hipStream_t stream) {
  PcCompactParams p = {};
  p.table = table;
  p.refs = refs;
  p.new_table = new_table;
  p.new_refs = new_refs;
  p.page_map = page_map;
  p.chunks = (int)((pages + kPcPlanThreads - 1) / kPcPlanThreads);
  p.live = (int32_t*)workspace;
  p.rank = p.live + p.chunks;
  p.high = p.rank + pages;
  p.hole = p.high + pages;
  p.pages = pages;
  p.entries = entries;
  p.counts_here = pages <= kPcCountsHere;
  int64_t tb = ((entries > pages ? entries : pages) + 4 * kPcThreads - 1) / (4 * kPcThreads);
  tb = tb < 1 ? 1 : (tb > 512 ? 512 : tb);
  bool first = true;
  for (int64_t c0 = 0; first || c0 < n; c0 += kPcMaxCaches, first = false) {
    const int64_t chunks = pc_copy_set(p.set, c0, n, caches, row_bytes, page);
    p.table_blocks = first ? (int)tb : 0;
    // at most half the pages move; blocks beyond a few rounds of the CUs loop
    const int64_t most = (pages / 2) * chunks;
    const int64_t cap = 16ll * device_cu_count();
    p.copy_blocks = (int)(most < cap ? most : cap);
    if (first) {
      if (!p.counts_here) pc_count_kernel<<<dim3((unsigned)p.chunks), kPcPlanThreads, 0, stream>>>(p);
      pc_rank_kernel<<<dim3((unsigned)p.chunks), kPcPlanThreads, 0, stream>>>(p);
    }
    const int64_t grid = p.table_blocks + p.copy_blocks;
    if (grid > 0) pc_compact_kernel<<<dim3((unsigned)grid), kPcThreads, 0, stream>>>(p);
    DSA_HIP(hipGetLastError());
  }
  return DSA_OK;
}

// ---------------------------------------------------------------------------
// plan: rows extended by numbers of tokens of their own, a slot and a position
// for each of the packed tokens
// ---------------------------------------------------------------------------
struct PcPlanParams {
  const int32_t *table, *lens, *refs, *more;  // more: new tokens of each row, negative: the row has ended
  int32_t *new_table, *new_lens, *new_refs, *slots, *positions, *ends;
  int32_t *start, *freelist;                  // workspace
  int64_t pages, tokens;
  int rows, max_blocks, page;
  int wide_refs;                              // refs may be read 16 bytes at a time
  int table_blocks;                           // blocks of the table in the second launch
};

// A row: its tokens, the pages that they hold, and the pages wanted with the
// new ones (-1 where they would outgrow the table, -2 where the row has ended).
struct PcRow {
  int len, held, want;
};

__device__ __forceinline__ PcRow pc_row(const PcPlanParams& p, int len, int more) {
  PcRow r;
  // (below 2^26 tokens, 2^31 new ones, 2^20 of a page: the sums fit 32 bits)
  const unsigned page = (unsigned)p.page, room = (unsigned)(p.max_blocks * p.page);
  r.len = (int)min((unsigned)max(len, 0), room);
  r.held = (int)(((unsigned)r.len + page - 1) / page);
  const unsigned all = (unsigned)r.len + (unsigned)max(more, 0);
  r.want = more < 0 ? -2 : (all > room ? -1 : (int)((all + page - 1) / page));
  return r;
}

// sums that stop at 2^32 - 1
__device__ __forceinline__ unsigned pc_add_sat(unsigned a, unsigned b) { return a + b < a ? ~0u : a + b; }

// inclusive such sum over the threads of a block of W waves
template <int W>
__device__ __forceinline__ unsigned pc_block_scan_sat(unsigned v, unsigned* s_part, unsigned* total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int o = 1; o < 64; o *= 2) {
    const unsigned x = __shfl_up(v, o);
    v = lane >= o ? pc_add_sat(v, x) : v;
  }
  __syncthreads();
  if (lane == 63) s_part[wave] = v;
  __syncthreads();
  unsigned base = 0, all = 0;
#pragma unroll
  for (int w = 0; w < W; ++w) {
    const unsigned q = s_part[w];
    if (w < wave) base = pc_add_sat(base, q);
    all = pc_add_sat(all, q);
  }
  *total = all;
  return pc_add_sat(base, v);
}

// Pages that a thread looks at for free ones at a time.  One block looks, a pass
// of the loop waits for its counts and for the scan: with 4, 8 and 16 pages a
// thread a plan over 85000 pages takes 6.3, 5.4 and 5.0 us, one over 8192 pages
// 2.9, 2.8 and 3.5.
constexpr int kPcFree = 8;

// Block 0 plans: the first of each row's new pages among the free ones (-1: it
// gets none), and which those are; the lengths and the ends of the rows' tokens.
// The other blocks copy the counts for the second launch to change.
__global__ __launch_bounds__(kPcPlanThreads) void pc_plan_kernel(PcPlanParams p) {
  constexpr int W = kPcPlanThreads / 64;
  const int tid = threadIdx.x;
  if (blockIdx.x > 0) {
    for (int64_t i = (int64_t)(blockIdx.x - 1) * kPcPlanThreads + tid; i < p.pages;
         i += (int64_t)(gridDim.x - 1) * kPcPlanThreads)
      p.new_refs[i] = p.refs[i];
    return;
  }
  __shared__ int s_part[W];
  __shared__ unsigned s_part2[W];
  // the counts of kPcFree pages of a thread (1 past the last); the first are on
  // their way beside what follows
  auto counts = [&](int64_t i0, int (&c)[kPcFree]) {
    const int64_t i = i0 + kPcFree * tid;
    if (p.wide_refs && i + kPcFree <= p.pages) {
#pragma unroll
      for (int j = 0; j < kPcFree; j += 4) *(i32x4*)(c + j) = *(const i32x4*)(p.refs + i + j);
    } else {
#pragma unroll
      for (int j = 0; j < kPcFree; ++j) c[j] = i + j < p.pages ? p.refs[i + j] : 1;
    }
  };
  int c[kPcFree];
  counts(0, c);
  int64_t taken = 0;
  unsigned end = 0;
  for (int r0 = 0; r0 < p.rows; r0 += kPcPlanThreads) {
    const int r = r0 + tid;
    int need = 0;
    unsigned more = 0;
    if (r < p.rows) {
      const int m = p.more[r];
      const PcRow k = pc_row(p, p.lens[r], m);
      need = max(k.want - k.held, 0);
      more = (unsigned)max(m, 0);
    }
    int total;
    const int incl = pc_block_scan<W>(need, s_part, &total);
    unsigned all;
    const unsigned to = pc_add_sat(end, pc_block_scan_sat<W>(more, s_part2, &all));
    if (r < p.rows) {
      p.start[r] = (int)min(taken + incl - need, (int64_t)0x7fffffff);
      p.ends[r] = (int)min(to, 0x7fffffffu);
    }
    taken += total;
    end = pc_add_sat(end, all);
  }
  // free pages in ascending order until that many are found
  int64_t found = 0;
  for (int64_t i0 = 0; i0 < p.pages && found < taken; i0 += kPcFree * kPcPlanThreads) {
    int free = 0;
#pragma unroll
    for (int j = 0; j < kPcFree; ++j) free |= (c[j] == 0) << j;
    if (i0 + kPcFree * kPcPlanThreads < p.pages) counts(i0 + kPcFree * kPcPlanThreads, c);
    const int n = __popc(free);
    int total;
    int64_t at = found + pc_block_scan<W>(n, s_part, &total) - n;
    for (; free && at < taken; free &= free - 1) p.freelist[at++] = (int)(i0 + kPcFree * tid + __ffs(free) - 1);
    found += total;
  }
  // a row is served if the free pages last for it and all before it (a thread
  // reads what it wrote itself)
  for (int r = tid; r < p.rows; r += kPcPlanThreads) {
    const int m = p.more[r];
    const PcRow k = pc_row(p, p.lens[r], m);
    const int need = max(k.want - k.held, 0);
    const bool served = k.want >= 0 && (need == 0 || (int64_t)p.start[r] + need <= found);
    if (!served) p.start[r] = -1;
    p.new_lens[r] = served ? k.len + m : (k.want == -2 ? 0 : k.len);
  }
}

constexpr int kPcEndsHere = 4096;  // rows whose ends a block of tokens keeps in LDS

__global__ __launch_bounds__(kPcThreads) void pc_plan_tables_kernel(PcPlanParams p) {
  __shared__ int s_ends[kPcEndsHere];
  const int tid = threadIdx.x;
  if ((int)blockIdx.x < p.table_blocks) {
    const int64_t stride = (int64_t)p.table_blocks * kPcThreads, me = (int64_t)blockIdx.x * kPcThreads + tid;
    for (int64_t i = me; i < (int64_t)p.rows * p.max_blocks; i += stride) {
      const int r = i >> 32 ? (int)(i / p.max_blocks) : (int)((unsigned)i / (unsigned)p.max_blocks);
      const int col = (int)(i - (int64_t)r * p.max_blocks);
      const int old = p.table[i], at = p.start[r];
      const PcRow k = pc_row(p, p.lens[r], p.more[r]);
      int e = -1;
      if (k.want != -2 && col < k.held) {
        e = old >= 0 && old < p.pages ? old : -1;
      } else {
        if (old >= 0 && old < p.pages) atomicSub(p.new_refs + old, 1);
        if (at >= 0 && col < k.want) {
          e = p.freelist[at + col - k.held];
          atomicAdd(p.new_refs + e, 1);
        }
      }
      p.new_table[i] = e;
    }
    return;
  }
  // a block's tokens find their rows by the ends
  const bool here = p.rows <= kPcEndsHere;
  if (here) {
    for (int i = tid; i < p.rows; i += kPcThreads) s_ends[i] = p.ends[i];
    __syncthreads();
  }
  const int64_t t = ((int64_t)blockIdx.x - p.table_blocks) * kPcThreads + tid;
  if (t >= p.tokens) return;
  int lo = 0, hi = p.rows;  // first r with ends[r] > t
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if ((here ? s_ends[mid] : p.ends[mid]) > t) hi = mid; else lo = mid + 1;
  }
  int slot = -1, pos = 0;
  if (lo < p.rows) {
    const int r = lo, first = r ? (here ? s_ends[r - 1] : p.ends[r - 1]) : 0;
    const int at = p.start[r];
    const PcRow k = pc_row(p, p.lens[r], p.more[r]);
    pos = k.len + (int)(t - first);
    if (at >= 0) {
      const int col = (int)((unsigned)pos / (unsigned)p.page);
      const int blk = col < k.held ? p.table[(int64_t)r * p.max_blocks + col] : p.freelist[at + col - k.held];
      if (blk >= 0 && blk < p.pages) slot = blk * p.page + (pos - col * p.page);
    }
  }
  p.slots[t] = slot;
  p.positions[t] = pos;
}

size_t pc_plan_workspace_bytes(int64_t rows, int64_t pages) { return (size_t)(rows + pages) * sizeof(int32_t); }

int pc_plan_run(const int32_t* table, const int32_t* lens, const int32_t* refs, const int32_t* more,
                int32_t* new_table, int32_t* new_lens, int32_t* new_refs, int32_t* slots, int32_t* positions,
                int32_t* ends, int64_t rows, int64_t max_blocks, int64_t pages, int64_t page, int64_t tokens,
                void* workspace, hipStream_t stream) {
  PcPlanParams p = {};
  p.table = table;
  p.lens = lens;
  p.refs = refs;
  p.more = more;
  p.new_table = new_table;
  p.new_lens = new_lens;
  p.new_refs = new_refs;
  p.slots = slots;
  p.positions = positions;
  p.ends = ends;
  p.start = (int32_t*)workspace;
  p.freelist = p.start + rows;
  p.wide_refs = ((uintptr_t)refs & 15) == 0;
  p.pages = pages;
  p.tokens = tokens;
  p.rows = (int)rows;
  p.max_blocks = (int)max_blocks;
  p.page = (int)page;
  int64_t copy_blocks = (pages + 4 * kPcPlanThreads - 1) / (4 * kPcPlanThreads);
  copy_blocks = copy_blocks > 64 ? 64 : copy_blocks;
  int64_t tb = (rows * max_blocks + 2 * kPcThreads - 1) / (2 * kPcThreads);
  tb = tb > 1024 ? 1024 : tb;
  p.table_blocks = (int)tb;
  const int64_t grid = tb + (tokens + kPcThreads - 1) / kPcThreads;
  DSA_CHECK_SUPPORTED(launchable(grid, kPcThreads), "too many tokens for one call");
  pc_plan_kernel<<<dim3((unsigned)(1 + copy_blocks)), kPcPlanThreads, 0, stream>>>(p);
  pc_plan_tables_kernel<<<dim3((unsigned)grid), kPcThreads, 0, stream>>>(p);
  DSA_HIP(hipGetLastError());
  return DSA_OK;
}

// ---------------------------------------------------------------------------
// write to slots: one thread per unit of a token's rows
// ---------------------------------------------------------------------------
struct PcSlotParams {
  PcCache c[kPcMaxCaches];
  const int32_t* at;
  int64_t tokens, slots;
  int n, s, units;
};

__global__ __launch_bounds__(kPcThreads) void pc_slots_kernel(PcSlotParams p) {
  const int64_t i = (int64_t)blockIdx.x * kPcThreads + threadIdx.x;
  const int64_t t = i >> 32 ? i / p.units : (int64_t)((unsigned)i / (unsigned)p.units);
  if (t >= p.tokens) return;
  const int u = (int)(i - t * p.units);
  int ci = 0;
  while (ci + 1 < p.n && u >= p.c[ci + 1].unit0) ++ci;
  const PcCache& c = p.c[ci];
  const int64_t off = (int64_t)(u - c.unit0) << c.shift;
  const int64_t b = p.s == p.tokens ? 0 : t / p.s;
  const unsigned char* src = c.src + b * c.src_sb + (t - b * p.s) * c.src_st + off;
  // (the row is read beside its slot, not behind it)
  const u32x4 wide = c.shift == 4 ? *(const u32x4*)src : u32x4{0, 0, 0, 0};
  const int slot = p.at[t];
  if (slot < 0 || slot >= p.slots) return;
  unsigned char* dst = c.dst + (int64_t)slot * c.row_bytes + off;
  if (c.shift == 4) *(u32x4*)dst = wide;
  else pc_move(dst, src, c.shift);
}

int pc_slots_run(int64_t n, const void* const* rows, void* const* caches, const int64_t* row_bytes,
                 const int64_t* row_sb, const int64_t* row_st, const int32_t* slots, int64_t batch, int64_t s,
                 int64_t pages, int64_t page, hipStream_t stream) {
  PcSlotParams p = {};
  p.at = slots;
  p.tokens = batch * s;
  p.slots = pages * page;
  p.s = (int)s;
  // blocks of the launch for the caches from c0 on
  auto take = [&](int64_t c0) {
    p.n = (int)(n - c0 < kPcMaxCaches ? n - c0 : kPcMaxCaches);
    int64_t units = 0;
    for (int i = 0; i < p.n; ++i) {
      PcCache& c = p.c[i];
      const int64_t k = c0 + i;
      c.src = (const unsigned char*)rows[k];
      c.dst = (unsigned char*)caches[k];
      c.src_sb = row_sb[k];
      c.src_st = row_st[k];
      c.row_bytes = (int)row_bytes[k];
      c.shift = pc_shift((uint64_t)(uintptr_t)c.src | (uintptr_t)c.dst | (uint64_t)row_bytes[k] |
                         (uint64_t)row_sb[k] | (uint64_t)row_st[k]);
      c.unit0 = (int)units;
      units += row_bytes[k] >> c.shift;
    }
    p.units = (int)units;  // (at most 32 rows of 2^24 bytes)
    return (p.tokens * units + kPcThreads - 1) / kPcThreads;
  };
  // (all of them before the first: a call that is refused has written nothing)
  for (int64_t c0 = n > kPcMaxCaches ? 0 : n; c0 < n; c0 += kPcMaxCaches)
    DSA_CHECK_SUPPORTED(launchable(take(c0), kPcThreads), "too many rows for one call");
  for (int64_t c0 = 0; c0 < n; c0 += kPcMaxCaches) {
    const int64_t grid = take(c0);
    DSA_CHECK_SUPPORTED(launchable(grid, kPcThreads), "too many rows for one call");
    pc_slots_kernel<<<dim3((unsigned)grid), kPcThreads, 0, stream>>>(p);
    DSA_HIP(hipGetLastError());
  }
  return DSA_OK;
}

// ---------------------------------------------------------------------------
// prefixes: neighbouring rows that begin with the same full pages
// ---------------------------------------------------------------------------
struct PcPrefixParams {
  const int32_t *table, *lens;
  int32_t *groups, *lengths;
  int rows, max_blocks, page, min_pages;
};

// First column in [c0, c1) where rows x and y of the table differ or name no
// page, 0x7fffffff if none does.  One wave; rows of `wide` columns.
__device__ __forceinline__ int pc_apart(const int32_t* x, const int32_t* y, int c0, int c1, int wide, int lane) {
  constexpr int kAhead = 8;  // columns of a lane on their way at a time
  int apart = 0x7fffffff;
  for (; c0 < c1 && apart == 0x7fffffff; c0 += 64 * kAhead) {
    int e[kAhead], f[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const int c = min(c0 + j * 64 + lane, wide - 1);
      e[j] = x[c];
      f[j] = y[c];
    }
#pragma unroll
    for (int j = kAhead - 1; j >= 0; --j) {
      const int c = c0 + j * 64 + lane;
      const unsigned long long m = __ballot(c < c1 && (e[j] != f[j] || e[j] < 0));
      if (m) apart = c0 + j * 64 + __ffsll(m) - 1;
    }
  }
  return apart;
}

// the full pages that row b shares, of those before column `apart`; 0 if too few to count
__device__ __forceinline__ int pc_shared(const PcPrefixParams& p, int l0, int l1, int apart) {
  const int n = min(min(max(min(l0, l1), 0) / p.page, p.max_blocks), apart);
  return n >= p.min_pages ? n : 0;
}

// A workgroup per row: leading full pages that it has in common with the row
// before it, to groups.  Its waves look at a quarter of the columns each (256
// rows of 2000 pages: 3.4 us, one wave a row 6.7), and do not wait for the
// lengths to know how many there are.
__global__ __launch_bounds__(kPcThreads) void pc_common_kernel(PcPrefixParams p) {
  constexpr int W = kPcThreads / 64;
  __shared__ int s_apart[W];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), b = blockIdx.x;
  if (b == 0) {
    if (threadIdx.x == 0) p.groups[0] = 0;
    return;
  }
  const int l0 = p.lens[b - 1], l1 = p.lens[b];
  const int32_t* x = p.table + (int64_t)b * p.max_blocks;
  const int part = (p.max_blocks + 64 * W - 1) / (64 * W) * 64, c0 = wave * part;
  const int mine = pc_apart(x, x - p.max_blocks, c0, min(c0 + part, p.max_blocks), p.max_blocks, threadIdx.x & 63);
  if ((threadIdx.x & 63) == 0) s_apart[wave] = mine;
  __syncthreads();
  if (threadIdx.x == 0) {
    int apart = s_apart[0];
#pragma unroll
    for (int w = 1; w < W; ++w) apart = min(apart, s_apart[w]);
    p.groups[b] = pc_shared(p, l0, l1, apart);
  }
}

// One workgroup: runs of linked rows and the least that they share.  ALL: it
// looks for what they have in common too, a wave a row.
template <bool ALL>
__global__ __launch_bounds__(kPcPlanThreads) void pc_groups_kernel(PcPrefixParams p) {
  constexpr int W = kPcPlanThreads / 64;
  __shared__ int s_last[W];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  if (ALL) {
    for (int b = __builtin_amdgcn_readfirstlane(wave); b < p.rows; b += W) {
      const int32_t* x = p.table + (int64_t)b * p.max_blocks;
      const int l0 = p.lens[max(b - 1, 0)], l1 = p.lens[b];
      const int apart = b ? pc_apart(x, x - p.max_blocks, 0, p.max_blocks, p.max_blocks, lane) : 0;
      if (lane == 0) p.groups[b] = pc_shared(p, l0, l1, apart);
    }
  }
  for (int b = tid; b < p.rows; b += kPcPlanThreads)
    __hip_atomic_store(p.lengths + b, 0x7fffffff, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __syncthreads();
  int before = 0;  // first row of the group that the chunk's first rows may belong to
  for (int b0 = 0; b0 < p.rows; b0 += kPcPlanThreads) {
    const int b = b0 + tid;
    const int common = b < p.rows ? p.groups[b] : 0;
    // first row of the group: the last row up to b that is not linked
    const unsigned long long starts = __ballot(common == 0);
    __syncthreads();
    if (lane == 0) s_last[wave] = starts ? b0 + wave * 64 + 63 - __clzll(starts) : -1;
    __syncthreads();
    const unsigned long long mine = starts & (~0ull >> (63 - lane));
    int first = -1, last = before;
    for (int w = 0; w < W; ++w) {
      const int x = s_last[w];
      if (w == wave) first = mine ? b0 + wave * 64 + 63 - __clzll(mine) : last;
      if (x >= 0) last = x;
    }
    before = last;
    if (b < p.rows) {
      if (common) atomicMin(p.lengths + first, common * p.page);
      p.groups[b] = first;
    }
  }
  __syncthreads();
  for (int b = tid; b < p.rows; b += kPcPlanThreads) {
    const int first = p.groups[b];
    const int n = __hip_atomic_load(p.lengths + first, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    // (a row alone writes its own; the others of a group write what its first row has)
    __hip_atomic_store(p.lengths + b, n == 0x7fffffff ? 0 : n, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
}

int pc_prefixes_run(const int32_t* table, const int32_t* lens, int32_t* groups, int32_t* lengths, int64_t rows,
                    int64_t max_blocks, int64_t page, int64_t min_tokens, hipStream_t stream) {
  PcPrefixParams p = {table, lens, groups, lengths, (int)rows, (int)max_blocks, (int)page, 1};
  const int64_t pages = (min_tokens + page - 1) / page;
  p.min_pages = (int)(pages < 1 ? 1 : pages);
  DSA_CHECK_SUPPORTED(launchable(rows, kPcThreads), "too many rows for one call");
  // In one launch where a wave has a row and looks at it once (a call for 16 rows
  // of 512 columns takes 3.9 us, replayed 3.7; in two launches 6.5, replayed 4.5;
  // for 32 rows, two a wave, 5.0 and 4.9 against 6.6 and 4.7).
  if (rows <= kPcPlanThreads / 64 && max_blocks <= 512) {
    pc_groups_kernel<true><<<dim3(1), kPcPlanThreads, 0, stream>>>(p);
  } else {
    pc_common_kernel<<<dim3((unsigned)rows), kPcThreads, 0, stream>>>(p);
    pc_groups_kernel<false><<<dim3(1), kPcPlanThreads, 0, stream>>>(p);
  }
  DSA_HIP(hipGetLastError());
  return DSA_OK;
}

}  // namespace dsa
