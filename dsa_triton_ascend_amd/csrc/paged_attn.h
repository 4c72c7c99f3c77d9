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

struct PagedSeq {
  int act_q, act_k, lo, hi;  // lo <= t < hi: tokens that any row sees
};

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

__device__ __forceinline__ PagedSeq paged_seq(const PagedAttnParams& p, int b) {
  PagedSeq s;
  s.act_k = min(max(p.act_k[b], 0), p.max_blocks * p.page);
  s.act_q = p.act_q ? min(max(p.act_q[b], 0), p.s1) : p.s1;
  int l, h;
  paged_bounds(p, s.act_q, s.act_k, 0, &s.lo, &h);
  paged_bounds(p, s.act_q, s.act_k, max(s.act_q - 1, 0), &l, &s.hi);
  if (s.hi < s.lo) s.hi = s.lo;
  return s;
}

// sequence b, the same on all lanes (nothing past the last)
__device__ __forceinline__ PagedSeq paged_seq_uniform(const PagedAttnParams& p, int b) {
  PagedSeq s = paged_seq(p, min(b, p.batch - 1));
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

struct PagedPlan {
  int total, per;   // tiles, tiles of a worker
  int grain;
  PagedSeq seq;     // of this lane
  int tiles, incl;  // its tiles, and those of the lanes up to it

  __device__ __forceinline__ int padded(int n) const {
    return grain == 1 ? n : (int)((unsigned)(n + grain - 1) / (unsigned)grain) * grain;
  }

  __device__ __forceinline__ void make(const PagedAttnParams& p, int tile, int lane) {
    tiles = 0;
    if (lane < p.batch) {
      seq = paged_seq(p, lane);
      tiles = paged_tiles(seq, tile);
    }
    incl = wave_scan(tiles);
    total = __builtin_amdgcn_readlane(incl, 63);
    if (p.batch > 64) {
      int n = 0;
#pragma unroll 4
      for (int b = 64 + lane; b < p.batch; b += 64) n += paged_tiles(paged_seq(p, b), tile);
      total += wave_total(n);
    }
    per = max((int)((unsigned)(total + p.workers - 1) / (unsigned)p.workers), p.min_tiles);
    grain = 1;
    if (p.batch > p.workers) return;
    for (int g = per; g <= per + kPaSlack; g += kPaSlack) {
      int n = (int)((unsigned)(tiles + g - 1) / (unsigned)g);
#pragma unroll 4
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
  __device__ __forceinline__ int find(const PagedAttnParams& p, int tile, int lane, int at, int* before) const {
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
  __device__ __forceinline__ PagedSeq sequence(const PagedAttnParams& p, int b) const {
    PagedSeq s;
    if (b < 64) {
      s.act_q = __builtin_amdgcn_readlane(seq.act_q, b);
      s.act_k = __builtin_amdgcn_readlane(seq.act_k, b);
      s.lo = __builtin_amdgcn_readlane(seq.lo, b);
      s.hi = __builtin_amdgcn_readlane(seq.hi, b);
    } else {
      s = paged_seq(p, b);
      s.lo = __builtin_amdgcn_readfirstlane(s.lo);
      s.hi = __builtin_amdgcn_readfirstlane(s.hi);
    }
    return s;
  }

  __device__ __forceinline__ int worker_of(int at) const { return (int)((unsigned)at / (unsigned)per); }

  // tiles before sequence b
  __device__ __forceinline__ int start(const PagedAttnParams& p, int tile, int lane, int b) const {
    if (b < 64) return b ? __builtin_amdgcn_readlane(incl, b - 1) : 0;
    int n = 0;
#pragma unroll 4
    for (int i = lane; i < b; i += 64) n += padded(paged_tiles(paged_seq(p, i), tile));
    return wave_total(n);
  }
};

// workspace and launches of the two kernels (paged_attn.hip, paged_attn_latent.hip)
struct PagedShape {
  int workers, min_tiles, groups, row_groups, group_rows, tile;
};
size_t paged_part_bytes(const PagedShape& s, int64_t d);
int paged_workers(int64_t slots, int64_t groups, int64_t batch, int64_t tiles, int min_tiles);
int paged_combine_launch(const PagedAttnParams& p, int tile, int64_t d, int32_t dtype, hipStream_t stream);
PagedShape paged_latent_shape(int64_t batch, int64_t s1, int64_t n1, int64_t d, int64_t max_blocks, int64_t page);
bool paged_latent_launchable(int64_t workers, int64_t row_groups);
int paged_latent_launch(const PagedAttnParams& p, int64_t d, int32_t dtype, hipStream_t stream);

}  // namespace dsa
