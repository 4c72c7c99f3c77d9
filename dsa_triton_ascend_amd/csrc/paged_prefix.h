// Attention over a paged cache of sequences that share a prefix: what the
// grouped-head and the shared-latent kernels have in common.
//
// A family is a run of neighbouring sequences with the same id and the same
// shared length; its prefix lies in the pages of its first sequence, but for the
// page in which it ends, which each sequence may have for itself (paged_given).  The
// queries of all of a family's sequences attend over the prefix together, so
// that a token of it is read once for all of them and the products have
// hundreds of rows; what each sequence has behind the prefix goes the way of
// paged_attn.h.  paged_combine_kernel joins both: every part i of a row comes as
// a reference, a sum and an unnormalised output, as the runs there,
//
//   O = (sum_i 2^(ref_i - m) O_i) / (sum_i 2^(ref_i - m) n_i),  m = max_i ref_i
//
// all in 32 bits (the parts in memory too).
//
// Which families.  Together costs a launch more, and outputs of 32 bits that are
// written and joined: 5 to 10 us with grouped heads, 15 to 20 over the latent
// cache.  Apart costs the reading of the prefix by every sequence (and every
// row group of one), from the caches for the most part.  So a prefix has to be
// so long that the whole batch would read 256 MB (latent: 320 MB) of it.
// Measured, us, apart and together, 200 tokens behind the prefix, 8 key heads of
// 128 columns and eight query heads on each: 32 sequences behind 2048 tokens 40
// and 43, behind 8192 95 and 52, behind 32768 324 and 83; 8 behind 2048 25 and 29,
// behind 8192 41 and 35; 16 families of two behind 4096 95 and 87, behind 16384
// 318 and 240; 16 new tokens of 16 sequences behind 2048 84 and 81.  16 latent
// heads: 32 sequences behind 8192 tokens 58 and 61, behind 32768 171 and 83; 64
// behind 8192 97 and 72; 16 families of two behind 16384 96 and 104.
// From 64 latent rows of a sequence on its own products bound it, and together
// is hardly faster or slower (32 sequences behind 32768 tokens: 128 heads 310 and
// 322; 64 heads 194 and 183).  The caller may set the length instead.
//
// The rule counts the batch, not what each family saves: near its border it takes
// the slower way by up to 8 % (the first of the grouped cases, the last of the
// latent ones), and one pair among many unrelated sequences may be worked on
// together for less than the launch costs.  Pools and tables of more than 256 MB of cache are loaded past the
// caches, as by paged_attention; prefixes that sequences read apart are then read
// from memory by each (32 behind 1024 tokens with 1024 of their own: 53 us, 40
// with loads that are kept, which take 202 in place of 182 for 32 unrelated
// sequences of 8000 tokens).
// What is not worked on together each sequence reads for itself (paged_attn.h),
// from the pages of the family's first: up to 2 us slower than paged_attention
// with grouped heads, 2 to 9 % over the latent cache (16 heads, 64 sequences
// behind 8192 tokens: 89 and 97 us; 128 heads, 32 behind 32768: 301 and 310), for
// the search for families in every worker.
//
// Work.  A job is a block of up to R rows of a family (over its sequences, new
// tokens and the query heads of one key head) and a part of its prefix.  Parts
// are as long as gives as many jobs as there are workgroups, whatever the
// families' sizes and lengths; the jobs of the same part, for other rows and key
// heads, run next to each other on one XCD, whose L2 they share.  All of it is
// found on the device from the ids and lengths, by one wave beside the kernel of
// paged_attn.h, which runs first: found by every workgroup for itself it took
// 8 us of each (most of it instructions that had to be fetched first).
// Families are cut at multiples of 64 sequences, so that a wave sees them whole.
#pragma once

#include "paged_attn.h"

namespace dsa {

constexpr int kPrefixTile = 32;  // tokens
constexpr int kPrefixMinTiles = 2;  // fewest tiles of a part
constexpr float kPrefixPartTiles = 18.f;  // jobs whose outputs cost what a tile of all of them does

// jobs of one key head for `m` blocks of rows: as many as there are workers, or
// (where the blocks alone are more than half of them) whole rounds of workers,
// with two jobs at least for a block of rows
__host__ __device__ __forceinline__ int prefix_jobs(int m, int workers) {
  return 2 * m <= workers ? workers : (2 * m + workers - 1) / workers * workers;
}

struct PrefixFamily {
  int first, count, tokens;  // sequences and shared tokens (0: none starts here)
};

// the families worked on together that start at sequences c0 .. c0 + 63, one per lane
__device__ __forceinline__ PrefixFamily prefix_families(const PagedPrefixParams& p, int c0, int lane) {
  const int b = c0 + lane;
  const PagedFamily f = paged_family(p, b);
  const int tokens = paged_whole_pages(p, min(p.shared[min(b, p.batch - 1)], p.max_blocks * p.page));
  const bool here = f.first == b && paged_together(p, tokens, f.count);
  return {b, here ? f.count : 0, here ? tokens : 0};
}

// n / d with magic = floor((2^32 - 1) / d): n * magic / 2^32 is at most
// n / 2^32 below n / d, so its integer part is off by one at most
__device__ __forceinline__ unsigned prefix_div(unsigned n, unsigned d, unsigned magic) {
  const unsigned q = __umulhi(n, magic);
  return q + (n - q * d >= d);
}

__device__ __forceinline__ int prefix_div_up(int a, int b) { return (int)((unsigned)(a + b - 1) / (unsigned)b); }

__device__ __forceinline__ int wave_min_int(int v) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) v = min(v, __shfl_xor(v, o));
  return v;
}

// The jobs of one key head, where the join finds a sequence's parts.  One wave.
struct PrefixPlan {
  int per;         // tiles of a part, at most
  int jobs;        // in all
  PrefixFamily f;  // of this lane among 64 sequences,
  int m, t;        // its blocks of rows and tiles

  __device__ __forceinline__ void families(const PagedPrefixParams& p, int c0, int lane) {
    f = prefix_families(p, c0, lane);
    m = (int)(((int64_t)f.count * p.rows + (1 << p.job_shift) - 1) >> p.job_shift);
    t = (f.tokens + kPrefixTile - 1) / kPrefixTile;
  }

  // Fewest tiles of a part.  J jobs of W tiles in all take about W / J tiles'
  // time, and the writing and joining of their outputs J / 18 of it (full
  // blocks): least for J = sqrt(18 W).  (16 latent heads, 8 sequences behind 8192
  // tokens: 51 us with 64 jobs, 57 with 128.)
  __device__ __forceinline__ int least(const PagedPrefixParams& p, int work, int blocks, int rows) const {
    const float fill = (float)rows / (float)(max(blocks, 1) << p.job_shift);
    const float tiles = __builtin_sqrtf((float)work * (float)p.n2 * fill * (1.f / kPrefixPartTiles) + 0.5f);
    return max((int)tiles, kPrefixMinTiles);
  }

  // sum m ceil(t / per) may be `most` jobs.  Up to 64 sequences the length of
  // the parts is fitted to the families; with more, which would be read again
  // for it, it is the shortest that has room for every rounding up, unless one
  // that has room for none happens to do.
  __device__ __forceinline__ void make(const PagedPrefixParams& p, int lane) {
    families(p, 0, lane);
    if (p.batch <= 64) {
      const int work = wave_total(m * t), blocks = wave_total(m), most = prefix_jobs(blocks, p.prefix_workers);
      per = max(prefix_div_up(work, most), least(p, work, blocks, wave_total(f.count * p.rows)));
      for (;;) {
        jobs = wave_total(m * prefix_div_up(t, per));
        if (jobs <= most) return;
        per += max(per >> 4, 1);
      }
    }
    int work = 0, rows = 0, all = 0;
    for (int c0 = 0; c0 < p.batch; c0 += 64) {
      families(p, c0, lane);
      work += m * t;
      rows += m;
      all += f.count * p.rows;
    }
    work = wave_total(work);
    rows = wave_total(rows);
    const int most = prefix_jobs(rows, p.prefix_workers), fewest = least(p, work, rows, wave_total(all));
    for (int room = 0;; room = rows) {
      per = max(prefix_div_up(work, most - room), fewest);
      int n = 0;
      for (int c0 = 0; c0 < p.batch; c0 += 64) {
        families(p, c0, lane);
        n += m * prefix_div_up(t, per);
      }
      jobs = wave_total(n);
      if (jobs <= most) return;
    }
  }

  // Writes the jobs, and for every sequence where its parts are; `runs` is the
  // plan of what is behind the prefixes.
  __device__ __forceinline__ void write(const PagedPrefixParams& p, const PagedPlan<PagedPrefixParams>& runs, int tile,
                                        int lane) {
    if (lane == 0) *p.n_jobs = jobs;
    int job_base = 0, run_base = 0;
    for (int c0 = 0; c0 < p.batch; c0 += 64) {
      if (p.batch > 64) families(p, c0, lane);
      // the sequences' runs
      const int b = c0 + lane;
      PagedSeqBehind seq = {};
      int nt = 0, padded = 0;
      if (b < p.batch) {
        seq = paged_seq(p, b);
        nt = paged_tiles(seq, tile);
        padded = runs.padded(nt);
      }
      const int upto = wave_scan(padded);
      PagedWhere w = {};
      if (nt) {
        const int first = run_base + upto - padded;
        w.run0 = runs.worker_of(first);
        w.runs = runs.worker_of(first + nt - 1) - w.run0 + 1;
        w.slot0 = first != w.run0 * runs.per;
      }
      if (b < p.batch) {  // (of a family's sequences the first half comes with the family)
        int* at = (int*)(p.where + b);
        at[4] = w.run0, at[5] = w.runs, at[6] = w.slot0;
        if (!seq.shared) at[0] = at[1] = at[2] = at[3] = 0;
      }
      run_base += __builtin_amdgcn_readlane(upto, 63);
      // what the rows of a sequence see: they rise with its new token
      int lo0, hi0, lo1, hi1;
      paged_bounds(p, seq.act_q, seq.act_k, 0, &lo0, &hi0);
      paged_bounds(p, seq.act_q, seq.act_k, max(p.s1 - 1, 0), &lo1, &hi1);
      int seen_lo = 0x7fffffff, seen_hi = 0;  // any of its rows
      if (seq.act_q > 0) {
        seen_lo = lo0;
        int l;
        paged_bounds(p, seq.act_q, seq.act_k, seq.act_q - 1, &l, &seen_hi);
      }
      const int all_lo = lo1, all_hi = seq.act_q == p.s1 ? hi0 : 0;
      // the families that start here
      const int parts = prefix_div_up(t, per), n = m * parts, incl = wave_scan(n);
      for (unsigned long long todo = __ballot(n > 0); todo; todo &= todo - 1) {
        const int l = __ffsll(todo) - 1;
        const int first = __builtin_amdgcn_readlane(f.first, l), count = __builtin_amdgcn_readlane(f.count, l);
        const int tokens = __builtin_amdgcn_readlane(f.tokens, l), blocks = __builtin_amdgcn_readlane(m, l);
        const int np = __builtin_amdgcn_readlane(parts, l), nj = __builtin_amdgcn_readlane(n, l);
        const int job0 = job_base + __builtin_amdgcn_readlane(incl, l) - nj;
        const bool in = lane >= l && lane < l + count;
        const int lo = wave_min_int(in ? seen_lo : 0x7fffffff), hi = min(-wave_min_int(in ? -seen_hi : 0), tokens);
        const int alo = -wave_min_int(in ? -all_lo : 0), ahi = wave_min_int(in ? all_hi : 0x7fffffff);
        const int lead = first == c0 ? paged_leader(p, first, lane) : first;
        // parts of equal numbers of whole tiles, cut to what is seen
        const int each = prefix_div_up((tokens + kPrefixTile - 1) / kPrefixTile, np) * kPrefixTile;
        for (int j = lane; j < nj; j += 64) {
          const int part = (int)((unsigned)j / (unsigned)blocks), block = j - part * blocks;
          PagedJob q;
          q.first = first;
          q.row0 = block << p.job_shift;
          q.rows = min(count * p.rows - q.row0, 1 << p.job_shift);
          q.lead = lead;
          q.tok0 = max(part * each, lo);
          q.tok1 = min(part * each + each, hi);
          q.all_lo = alo;
          q.all_hi = ahi;
          p.job[job0 + j] = q;
        }
        for (int i = lane; i < count; i += 64) {
          int* at = (int*)(p.where + first + i);
          at[0] = job0, at[1] = blocks, at[2] = np, at[3] = i;
        }
      }
      job_base += __builtin_amdgcn_readlane(incl, 63);
    }
  }
};

// A wave beside the runs plans the prefixes.
__device__ __forceinline__ void prefix_plan(const PagedPrefixParams& p, int tile, int lane) {
  PagedPlan<PagedPrefixParams> runs;
  runs.make(p, tile, lane);
  PrefixPlan plan;
  plan.make(p, lane);
  plan.write(p, runs, tile, lane);
}

// Which job, of which key head, workgroup `block` of `grid` has in round `round`:
// the jobs lie end to end over the XCDs (workgroup x runs on XCD x % 8), key
// heads next to each other.
__device__ __forceinline__ int prefix_job_of(const PagedPrefixParams& p, int block, int grid, int round, int* head) {
  const int at = round * grid + (block & 7) * (grid >> 3) + (block >> 3);
  const int job = p.n2 == 1 ? at : (int)prefix_div(at, p.n2, p.heads_magic);
  *head = at - job * p.n2;
  return job;
}

// The tokens that row `row` of a job sees of the prefix.
__device__ __forceinline__ void prefix_bounds(const PagedPrefixParams& p, const PagedJob& j, int row, int* lo, int* hi) {
  const unsigned vr = j.row0 + row, i = prefix_div(vr, p.rows, p.rows_magic);
  const int s = (int)prefix_div(vr - i * p.rows, p.group, p.group_magic), b = j.first + (int)i;
  const int act_k = min(max(p.act_k[b], 0), p.max_blocks * p.page);
  paged_bounds(p, p.act_q ? min(max(p.act_q[b], 0), p.s1) : p.s1, act_k, s, lo, hi);
  *hi = min(*hi, j.tok1);
}

// kernels of the two forms (paged_prefix.hip, paged_prefix_latent.hip)
int prefix_latent_launch(const PagedPrefixParams& p, int64_t d, int32_t dtype, unsigned grid, hipStream_t stream);
constexpr int kPrefixLatentRows = 128;

}  // namespace dsa
