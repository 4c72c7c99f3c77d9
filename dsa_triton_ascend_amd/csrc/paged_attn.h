// Attention of the newest tokens over a paged cache: what the grouped-head
// and the shared-latent kernels have in common.
//
// Work.  A sequence's visible tokens are cut into tiles, the tiles of all
// sequences are laid end to end, and every worker (a wave or a workgroup)
// takes an equal run of them, whatever the lengths: no worker waits for a
// long sequence while others idle, and the host need not know the lengths.
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
  // Outputs of runs, [worker][2][lane group][rows][D]: unnormalised in 32
  // bits, or (half_parts) divided by their divisor and by a power of two above
  // their row's largest, in 16.  The latter are off by 2^-12 of the row's
  // largest value, a sixteenth of what the bf16 output rounds and as much as
  // the fp16 output does; they halve 134 MB written and read at 128 heads.
  void* part_o;
  float* part_scale;  // [worker][2][lane group][rows] those powers of two
  f32x4* part_ml;  // [worker][2][lane group][rows] {ref, sum, largest score, divisor of the output}
  int64_t kv_rows, band_pre, band_next;
  int batch, s1, n1, n2, group, rows;  // group = n1 / n2 query heads of a key head; rows = s1 * group
  int max_blocks, page, mode, return_lse;
  int half_parts;
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

__device__ __forceinline__ int paged_tiles(const PagedSeq& s, int tile) { return (s.hi - s.lo + tile - 1) / tile; }

// the first lane's value, for all (a scalar to the compiler)
__device__ __forceinline__ int64_t wave_first(int64_t v) {
  const unsigned lo = __builtin_amdgcn_readfirstlane((int)(unsigned)v);
  const int hi = __builtin_amdgcn_readfirstlane((int)(v >> 32));
  return ((int64_t)hi << 32) | lo;
}

// inclusive sum over the lanes of a wave
__device__ __forceinline__ int wave_scan(int v, int lane) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int y = __shfl_up(v, o);
    if (lane >= o) v += y;
  }
  return v;
}

// The tiles of all sequences end to end, as a wave sees them (every lane
// gets the same results).  Lane l keeps sequence l of the first 64, so that
// up to 64 sequences are read once.  (64 sequences have fewer than 2^31
// tiles.)
struct PagedPlan {
  int64_t total, per;  // tiles, tiles of a worker
  PagedSeq seq;        // of this lane
  int tiles, incl;     // its tiles, and those of the lanes up to it

  __device__ __forceinline__ void make(const PagedAttnParams& p, int tile, int lane) {
    tiles = 0;
    if (lane < p.batch) {
      seq = paged_seq(p, lane);
      tiles = paged_tiles(seq, tile);
    }
    incl = wave_scan(tiles, lane);
    total = __builtin_amdgcn_readlane(incl, 63);
    for (int b0 = 64; b0 < p.batch; b0 += 64) {
      const int b = b0 + lane;
      const int n = wave_scan(b < p.batch ? paged_tiles(paged_seq(p, b), tile) : 0, lane);
      total += __builtin_amdgcn_readlane(n, 63);
    }
    // (the quotient in 32 bits wherever it fits: a 64-bit one takes a microsecond)
    const int64_t sum = total + p.workers - 1;
    per = sum >> 32 ? sum / p.workers : (int64_t)((unsigned)sum / (unsigned)p.workers);
    per = max(per, (int64_t)p.min_tiles);
  }

  // sequence that holds tile `at` (< total), and the tiles before it
  __device__ __forceinline__ int find(const PagedAttnParams& p, int tile, int lane, int64_t at, int64_t* before) const {
    int64_t base = 0;
    for (int b0 = 0; b0 < p.batch; b0 += 64) {
      const int b = b0 + lane;
      int n = tiles, in = incl;
      if (b0) {
        n = b < p.batch ? paged_tiles(paged_seq(p, b), tile) : 0;
        in = wave_scan(n, lane);
      }
      const unsigned long long m = __ballot(base + in > at);
      if (m) {
        const int first = __ffsll(m) - 1;
        *before = base + __builtin_amdgcn_readlane(in - n, first);
        return b0 + first;
      }
      base += __builtin_amdgcn_readlane(in, 63);
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

  __device__ __forceinline__ int64_t worker_of(int64_t at) const {
    return (at | per) >> 32 ? at / per : (int64_t)((unsigned)at / (unsigned)per);
  }

  // tiles before sequence b
  __device__ __forceinline__ int64_t start(const PagedAttnParams& p, int tile, int lane, int b) const {
    if (b < 64) return b ? __builtin_amdgcn_readlane(incl, b - 1) : 0;
    int64_t n = 0;
    for (int i = lane; i < b; i += 64) n += paged_tiles(paged_seq(p, i), tile);
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) n += __shfl_xor(n, o);
    return wave_first(n);
  }
};

// workspace and launches of the two kernels (paged_attn.hip, paged_attn_latent.hip)
struct PagedShape {
  int workers, min_tiles, groups, row_groups, group_rows, tile, half_parts;
};
size_t paged_part_bytes(const PagedShape& s, int64_t d);
int paged_workers(int64_t slots, int64_t groups, int64_t tiles, int min_tiles);
int paged_combine_launch(const PagedAttnParams& p, int tile, int64_t d, int32_t dtype, hipStream_t stream);
PagedShape paged_latent_shape(int64_t batch, int64_t s1, int64_t n1, int64_t d, int64_t max_blocks, int64_t page);
int paged_latent_launch(const PagedAttnParams& p, int64_t d, int32_t dtype, hipStream_t stream);

}  // namespace dsa
