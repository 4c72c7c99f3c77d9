// Attention of the newest tokens over a paged cache: what the grouped-head
// and the shared-latent kernels have in common.
//
// Work.  A sequence's visible tokens are cut into tiles, the tiles of all
// sequences are laid end to end, and every worker (a wave or a workgroup)
// takes an equal run of them, whatever the lengths: no worker waits for a
// long sequence while others idle, and the host need not know the lengths.
// Where the workers suffice for it, each sequence starts a run of its own: a
// run that crosses from one sequence into the next fills its pipeline twice.
// A run that covers a sequence whole writes its output; every other run
// leaves its softmax sums and unnormalised output in the workspace, and
// paged_combine_kernel joins the runs of a sequence.
//
// Softmax.  Scores are in log2 units.  A row's numerators are
// 2^(score - ref), with ref 8 below the largest score when it was set and
// moved only when a score comes 14 above it, so the output accumulator is
// rescaled rarely; fp16 numerators (largest 2^14) then keep weights of
// 2^-22 of the largest at full precision.  Sums are in 32 bits.
//
// Visible tokens of a row follow sparse flash attention: token t of row s1
// is visible iff diag - pre_tokens <= t <= diag + next_tokens, t < act_k,
// and (mode 3) t <= diag; diag = s1 in mode 0, act_k - act_q + s1 in mode 3.
// A row without one gives zeros, statistics too.  A block-table entry
// outside the cache reads as zero rows.
#pragma once

#include "sfa_common.h"

#include <type_traits>

namespace dsa {

constexpr float kPaBelow = 8.f;   // ref is set this far below the largest score
constexpr float kPaAbove = 14.f;  // and moved when a score exceeds it by more than this

struct PagedAttnParams {
  const void *q, *qr, *k, *kr, *v;
  void* out;
  float *smax, *ssum;
  const int32_t *act_q, *act_k, *table;
  // Outputs of runs, unnormalised, [worker][2][lane group][rows][D], in 32
  // bits.  16 bits with a power of two per row would halve what is written and
  // read (134 MB at 128 heads, 352 us in place of 358 for 32 x 32K tokens), but
  // a column much larger than its row's others would take their bits: at 2^24
  // times their size they were off by a tenth of their values.
  float* part_o;
  f32x4* part_ml;  // [worker][2][lane group][rows] {ref, sum, largest score, divisor of the output}
  int64_t kv_rows, band_pre, band_next;
  int batch, s1, n1, n2, group, rows;  // group = n1 / n2 query heads of a key head; rows = s1 * group
  int max_blocks, page, mode, return_lse;
  int workers, min_tiles;              // workers of one lane group; fewest tiles of a worker
  int groups, row_groups, group_rows;  // lane groups (key head, row group); rows of a row group
  unsigned page_magic;                 // floor((2^32 - 1) / page)
  float scale_log2;
};

// With a prefix that sequences share (paged_prefix.h): these kernels take what
// is behind it, plan the work on the prefixes meanwhile, and the join takes
// both's parts.  A short prefix they take too, for each sequence, from the pages
// of its family's first.
struct PagedWhere {  // of a sequence, for the join
  int job0, blocks, parts, place;  // first job of its family, blocks of rows, parts (0: no family), its place there
  int run0, runs, slot0, unused;   // its runs and the slot of the first
};
struct PagedJob {  // rows of a family, and tokens tok0 .. tok1 of its prefix
  int first, row0, rows, lead;     // first sequence; rows from row0 on; the sequence whose pages hold the prefix
  int tok0, tok1;
  int all_lo, all_hi;              // tokens that all rows of the family see
};
struct PagedPrefixParams : PagedAttnParams {
  const int32_t *ids, *shared;  // per sequence: its family and the tokens that it shares
  int before;  // sequences of the call that come before this launch's, in all arrays (-before .. -1)
  PagedWhere* where;
  PagedJob* job;
  int* n_jobs;
  // rows of part_o / part_ml: behind those of the runs come, for each sequence,
  // one for what a run has of it if that is all of it, then those of the jobs
  int64_t whole0, part0;
  int least;  // tokens of a prefix from which on it is worked on for its family together
  int prefix_workers;           // jobs of one key head aimed at
  int job_shift;                // log2 of the rows of a block
  unsigned rows_magic, group_magic, heads_magic;  // floor((2^32 - 1) / rows), of group, of n2
};

template <typename P> constexpr bool kPrefixed = std::is_same<P, PagedPrefixParams>::value;

// whether sequence b has the family of the one before it
__device__ __forceinline__ bool paged_linked(const PagedPrefixParams& p, int b) {
  const int here = min(b, p.batch - 1), before = max(here - 1, -p.before), id = p.ids[here], n = p.shared[here];
  return b == here && b > -p.before && id >= 0 && n > 0 && p.ids[before] == id && p.shared[before] == n;
}

// the first sequence of the family that b is in, for a b that is the same on all lanes (all of them active)
__device__ __forceinline__ int paged_leader(const PagedPrefixParams& p, int b, int lane) {
  for (;; b -= 64) {
    const unsigned long long apart = ~__ballot(paged_linked(p, max(b - lane, -p.before)));
    if (apart) return b - (__ffsll(apart) - 1);
  }
}

// Whether the prefix of a family of `count` sequences is worked on for all of
// them together (paged_prefix.h).
__device__ __forceinline__ bool paged_together(const PagedPrefixParams& p, int tokens, int count) {
  return count > 1 && tokens >= p.least;
}

// Sequence b's family among the 64 sequences from a multiple of 64 on: where it
// starts and how many they are.  What is worked on together is cut there, so
// that a wave sees all of it at once.  b: the same on all lanes, or lane l's is
// the l-th of the 64; lanes may be missing only where no sequence is theirs.
struct PagedFamily {
  int first, count;
  bool linked;  // with any other, also of another 64
};
__device__ __forceinline__ PagedFamily paged_family(const PagedPrefixParams& p, int b) {
  const int c0 = b & ~63, l = b & 63;
  const unsigned long long all = __ballot(paged_linked(p, c0 + (int)(threadIdx.x & 63))), links = all & ~1ull;
  PagedFamily f;
  f.first = c0 + 63 - __clzll(~links & (~0ull >> (63 - l)));
  const unsigned long long after = l == 63 ? 0ull : links >> (l + 1);
  f.count = b - f.first + __ffsll(~after);
  f.linked = f.count > 1 || (l == 0 && (all & 1)) || (l == 63 && paged_linked(p, b + 1));
  return f;
}

// page and offset of a token.  t * magic / 2^32 is at most t / 2^32 below
// t / page, so its integer part is off by one at most.
__device__ __forceinline__ unsigned paged_split(const PagedAttnParams& p, unsigned t, unsigned* off) {
  unsigned q = __umulhi(t, p.page_magic);
  unsigned r = t - q * (unsigned)p.page;
  if (r >= (unsigned)p.page) {
    ++q;
    r -= (unsigned)p.page;
  }
  *off = r;
  return q;
}

// The tokens of a prefix that are worked on together: its whole pages, since a
// sequence may have the page in which it ends for itself; all of one that ends in
// its first page.
__device__ __forceinline__ int paged_whole_pages(const PagedAttnParams& p, int tokens) {
  if (tokens <= p.page) return tokens;
  unsigned off;
  paged_split(p, (unsigned)tokens, &off);
  return tokens - (int)off;
}

// How many of a prefix's tokens a sequence has in the pages of its family's first:
// all but those of the page in which the prefix ends, where its own row of the table
// (`own`) names the same page as the first's for the last whole one.  Then it has a
// page of its own there, as after a fork, which copies a page that is partly filled;
// rows that leave the prefix out hold anything else.
// The same on all lanes: the numbers of tiles come from it.
__device__ __forceinline__ int paged_given(const PagedAttnParams& p, int tokens, const int32_t* own,
                                           const int32_t* first) {
  tokens = __builtin_amdgcn_readfirstlane(tokens);
  const int whole = paged_whole_pages(p, tokens);
  if (whole == tokens) return tokens;
  unsigned off;
  const unsigned last = paged_split(p, (unsigned)whole, &off) - 1;
  const int e = __builtin_amdgcn_readfirstlane(own[last]);
  const bool named = e == __builtin_amdgcn_readfirstlane(first[last]) && e >= 0 && (int64_t)e * p.page < p.kv_rows;
  return named ? whole : tokens;
}

struct PagedSeq {
  int act_q, act_k, lo, hi;  // lo <= t < hi: tokens that any row sees (with a prefix: behind it)
};
struct PagedSeqBehind : PagedSeq {
  int shared;  // tokens of the prefix before it
  int given;   // where it reads some of the prefix itself: the prefix's tokens (paged_given)
};
template <typename P> using PagedSeqOf = std::conditional_t<kPrefixed<P>, PagedSeqBehind, PagedSeq>;
// whether a sequence has a prefix before it
__device__ __forceinline__ bool paged_behind(const PagedSeq&) { return false; }
__device__ __forceinline__ bool paged_behind(const PagedSeqBehind& s) { return s.shared != 0; }

// A row's output times the factor f, which is 0 where the row saw no token of
// the run: then the output is 0 too, also where another row's value beside it
// is not finite.
__device__ __forceinline__ float paged_scaled(float x, float f) { return f == 0.f ? 0.f : x * f; }
__device__ __forceinline__ f32x4 paged_scaled(f32x4 x, float f) {
  return f == 0.f ? f32x4{0.f, 0.f, 0.f, 0.f} : x * f;
}

// bounds of row s1
__device__ __forceinline__ void paged_bounds(const PagedAttnParams& p, int act_q, int act_k, int s1, int* lo, int* hi) {
  const int64_t diag = p.mode == 0 ? (int64_t)s1 : (int64_t)act_k - act_q + s1;
  const int64_t top = p.mode == 0 ? (int64_t)act_k : diag + 1;
  const int64_t h = min(min(top, (int64_t)act_k), diag + p.band_next + 1);
  const int64_t l = diag - p.band_pre;
  *hi = s1 < act_q ? (int)max(h, (int64_t)0) : 0;
  *lo = (int)min(max(l, (int64_t)0), (int64_t)0x7fffffff);
}

template <typename P>
__device__ __forceinline__ PagedSeqOf<P> paged_seq(const P& p, int b) {
  PagedSeqOf<P> s;
  s.act_k = min(max(p.act_k[b], 0), p.max_blocks * p.page);
  s.act_q = p.act_q ? min(max(p.act_q[b], 0), p.s1) : p.s1;
  int l, h;
  paged_bounds(p, s.act_q, s.act_k, 0, &s.lo, &h);
  paged_bounds(p, s.act_q, s.act_k, max(s.act_q - 1, 0), &l, &s.hi);
  if constexpr (kPrefixed<P>) {
    const PagedFamily f = paged_family(p, b);
    const int tokens = f.linked ? min(p.shared[b], p.max_blocks * p.page) : 0;
    const int whole = paged_whole_pages(p, tokens);
    s.shared = paged_together(p, whole, f.count) ? whole : 0;
    s.given = s.shared == tokens ? 0 : tokens;
    s.lo = max(s.lo, s.shared);
  }
  if (s.hi < s.lo) s.hi = s.lo;
  return s;
}

// sequence b, the same on all lanes (nothing past the last)
template <typename P>
__device__ __forceinline__ PagedSeqOf<P> paged_seq_uniform(const P& p, int b) {
  PagedSeqOf<P> s = paged_seq(p, min(b, p.batch - 1));
  s.lo = __builtin_amdgcn_readfirstlane(s.lo);
  s.hi = b < p.batch ? __builtin_amdgcn_readfirstlane(s.hi) : s.lo;
  return s;
}

__device__ __forceinline__ int paged_tiles(const PagedSeq& s, int tile) { return (s.hi - s.lo + tile - 1) / tile; }

// The tiles of all sequences end to end, as a wave sees them (every lane
// gets the same results); the tiles of a sequence are counted as a multiple
// of `grain`, what is behind its last tile is nobody's work.  grain is the
// length of a run, so that sequences start runs, if there are workers enough
// for runs of the balanced length or kPaSlack tiles more, and 1 otherwise.
// Lane l keeps sequence l of the first 64, so that up to 64 sequences are
// read once.  (The entry point refuses tables of more than 2^30 tiles, so all
// of this is in 32 bits: 64-bit quotients take a microsecond each.)
//
// A sequence more in a run costs some 2 to 4 tiles (its rows, pages and first
// tiles have to arrive, its output leaves): 4 sequences of 40 tokens at 128
// heads took 86 us in one run, 27 in four; one tile too many is cheaper.
constexpr int kPaSlack = 2;

// Fewest tiles of a run: fewer make more runs to join, more leave workers idle
// (16 latent heads, one sequence of 512 tokens: 17.3 us with 1, 17.1 with 2,
// 19.2 with 4, 23.4 with 8; of 8192: 27.5, 22.1, 21.4, 26.5; grouped heads alike).
constexpr int kPaMinTiles = 2;

template <typename P>
struct PagedPlan {
  int total, per;   // tiles, tiles of a worker
  int grain;
  PagedSeqOf<P> seq;  // of this lane
  int tiles, incl;  // its tiles, and those of the lanes up to it

  __device__ __forceinline__ int padded(int n) const {
    return grain == 1 ? n : (int)((unsigned)(n + grain - 1) / (unsigned)grain) * grain;
  }

  __device__ __forceinline__ void make(const P& p, int tile, int lane) {
    tiles = 0;
    if (lane < p.batch) {
      seq = paged_seq(p, lane);
      tiles = paged_tiles(seq, tile);
    }
    incl = wave_scan(tiles);
    total = __builtin_amdgcn_readlane(incl, 63);
    if (p.batch > 64) {
      int n = 0;
#pragma unroll (kPrefixed<P> ? 1 : 4)
      for (int b = 64 + lane; b < p.batch; b += 64) n += paged_tiles(paged_seq(p, b), tile);
      total += wave_total(n);
    }
    per = max((int)((unsigned)(total + p.workers - 1) / (unsigned)p.workers), p.min_tiles);
    grain = 1;
    if (p.batch > p.workers) return;
    for (int g = per; g <= per + kPaSlack; g += kPaSlack) {
      int n = (int)((unsigned)(tiles + g - 1) / (unsigned)g);
#pragma unroll (kPrefixed<P> ? 1 : 4)
      for (int b = 64 + lane; b < p.batch; b += 64)
        n += (int)((unsigned)(paged_tiles(paged_seq(p, b), tile) + g - 1) / (unsigned)g);
      const int runs = wave_total(n);
      if (runs <= p.workers) {
        grain = per = g;
        total = runs * g;
        tiles = padded(tiles);
        incl = wave_scan(tiles);
        break;
      }
    }
  }

  // sequence that holds tile `at` (< total), and the tiles before it
  __device__ __forceinline__ int find(const P& p, int tile, int lane, int at, int* before) const {
    int base = 0, n = tiles, in = incl;
    for (int b0 = 0; b0 < p.batch; b0 += 64) {
      const int b = b0 + 64 + lane;
      const int next = b < p.batch ? padded(paged_tiles(paged_seq(p, b), tile)) : 0;
      const unsigned long long m = __ballot(base + in > at);
      if (m) {
        const int first = __ffsll(m) - 1;
        *before = base + __builtin_amdgcn_readlane(in - n, first);
        return b0 + first;
      }
      base += __builtin_amdgcn_readlane(in, 63);
      n = next;
      in = wave_scan(n);
    }
    *before = base;
    return p.batch;
  }

  // sequence b (the same on all lanes)
  __device__ __forceinline__ PagedSeqOf<P> sequence(const P& p, int b) const {
    PagedSeqOf<P> s;
    if (b < 64) {
      s.act_q = __builtin_amdgcn_readlane(seq.act_q, b);
      s.act_k = __builtin_amdgcn_readlane(seq.act_k, b);
      s.lo = __builtin_amdgcn_readlane(seq.lo, b);
      s.hi = __builtin_amdgcn_readlane(seq.hi, b);
      if constexpr (kPrefixed<P>) {
        s.shared = __builtin_amdgcn_readlane(seq.shared, b);
        s.given = __builtin_amdgcn_readlane(seq.given, b);
      }
    } else {
      s = paged_seq(p, b);
      s.lo = __builtin_amdgcn_readfirstlane(s.lo);
      s.hi = __builtin_amdgcn_readfirstlane(s.hi);
    }
    return s;
  }

  __device__ __forceinline__ int worker_of(int at) const { return (int)((unsigned)at / (unsigned)per); }

  // tiles before sequence b
  __device__ __forceinline__ int start(const P& p, int tile, int lane, int b) const {
    static_assert(!kPrefixed<P>, "the lanes from b on stay away from the loop, so that families would end at b");
    if (b < 64) return b ? __builtin_amdgcn_readlane(incl, b - 1) : 0;
    int n = 0;
#pragma unroll 4
    for (int i = lane; i < b; i += 64) n += padded(paged_tiles(paged_seq(p, i), tile));
    return wave_total(n);
  }
};

// Row of part_o where a run that has all tokens of sequence b leaves its output
// for lane group g, if there is a prefix before them (a run may have several
// such sequences, where it has two parts of sequences at most).
__device__ __forceinline__ int64_t paged_whole_slot(const PagedAttnParams&, int, int) { return 0; }
__device__ __forceinline__ int64_t paged_whole_slot(const PagedPrefixParams& p, int b, int g) {
  return p.whole0 + ((int64_t)b * p.groups + g) * p.group_rows;
}

// workspace and launches of the two kernels (paged_attn.hip, paged_attn_latent.hip)
struct PagedShape {
  int workers, min_tiles, groups, row_groups, group_rows, tile;
};
size_t paged_part_bytes(const PagedShape& s, int64_t d);
int paged_workers(int64_t slots, int64_t groups, int64_t batch, int64_t tiles, int min_tiles);
int paged_combine_launch(const PagedAttnParams& p, int tile, int64_t d, int32_t dtype, hipStream_t stream);
bool paged_combine_launchable(int64_t workers, int64_t batch, int64_t s1, int64_t n1);
int paged_combine_launch(const PagedPrefixParams& p, int tile, int64_t d, int32_t dtype, hipStream_t stream);
// of either kind of work: its shape, its parameters, and the launch of all but the join
PagedShape paged_shape(int64_t batch, int64_t s1, int64_t n1, int64_t n2, int64_t d, bool latent, int64_t max_blocks,
                       int64_t page);
void paged_fill(PagedAttnParams& p, const PagedShape& s, const void* query, const void* query_rope, const void* key,
                const void* key_rope, const void* value, void* out, float* smax, float* ssum, const int32_t* act_q,
                const int32_t* act_k, const int32_t* table, int64_t batch, int64_t s1, int64_t n1, int64_t n2,
                int64_t num_blocks, int64_t page, int64_t max_blocks, int32_t mode, int64_t pre_tokens,
                int64_t next_tokens, float scale, int32_t return_lse);
int paged_grouped_launch(const PagedPrefixParams& p, int64_t d, int32_t dtype, hipStream_t stream);
PagedShape paged_latent_shape(int64_t batch, int64_t s1, int64_t n1, int64_t d, int64_t max_blocks, int64_t page);
bool paged_latent_launchable(int64_t workers, int64_t row_groups);
int paged_latent_launch(const PagedAttnParams& p, int64_t d, int32_t dtype, hipStream_t stream);
int paged_latent_launch(const PagedPrefixParams& p, int64_t d, int32_t dtype, hipStream_t stream);

}  // namespace dsa
