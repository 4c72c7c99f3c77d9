// Attention over a paged cache of sequences that share a prefix: what the
// grouped-head and the shared-latent kernels have in common.
//
// A family is a run of neighbouring sequences with the same id and the same
// shared length; its prefix lies in the pages of its first sequence.  The
// queries of all of a family's sequences attend over the prefix together, so
// that a token of it is read once for all of them and the products have
// hundreds of rows; what each sequence has behind the prefix goes the way of
// paged_attn.h.  paged_combine_kernel joins both: every part of a row comes as
// a reference, a sum and an unnormalised output, as the runs there.
//
// Work.  A job is up to R rows of a family (over its sequences, new tokens and
// the query heads of one key head) and a part of its prefix.  Parts are as long
// as gives as many jobs as there are workgroups, whatever the families' sizes
// and lengths; the jobs of the same part, for other rows and key heads, run
// next to each other on one XCD, whose L2 they share.  All of it is found on
// the device from the ids and lengths, by every wave for itself.
#pragma once

#include "paged_attn.h"

namespace dsa {

constexpr int kPrefixTile = 32;  // tokens
constexpr int kPrefixMinTiles = 2;  // fewest tiles of a part

// jobs of one key head for `m` blocks of rows: as many as there are workers, or
// (where the blocks alone are more than half of them) whole rounds of workers,
// with two jobs at least for a block of rows
__host__ __device__ __forceinline__ int prefix_jobs(int m, int workers) {
  return 2 * m <= workers ? workers : (2 * m + workers - 1) / workers * workers;
}

struct PrefixFamily {
  int first, count, tokens;  // sequences and shared tokens (0: none starts here)
};

// the families that start at sequences c0 .. c0 + 63, one per lane (all loads of
// a lane at once: one after the other they take a microsecond each)
__device__ __forceinline__ PrefixFamily prefix_families(const PagedPrefixParams& p, int c0, int lane) {
  const int last = p.batch - 1, b = c0 + lane;
  const int i0 = min(max(b - 1, 0), last), i1 = min(b, last), i2 = min(b + 1, last);
  const int id0 = p.ids[i0], id1 = p.ids[i1], id2 = p.ids[i2];
  const int n0 = p.shared[i0], n1 = p.shared[i1], n2 = p.shared[i2];
  const bool shares = id1 >= 0 && n1 > 0;
  const bool mine = shares && b > 0 && b <= last && id0 == id1 && n0 == n1;  // linked to the sequence before it
  const bool next = shares && b < last && id1 == id2 && n1 == n2;
  const unsigned long long links = __ballot(mine);
  PrefixFamily f = {b, 0, 0};
  if (next && !mine) {
    const unsigned long long after = lane == 63 ? 0ull : links >> (lane + 1);
    f.count = __ffsll(~after);  // the links that follow, and the first sequence
    f.tokens = min(n1, p.max_blocks * p.page);
  }
  // a family that goes on behind these
  bool open = f.count > 0 && lane + f.count == 64 && b + f.count < p.batch;
  for (int e = c0 + 64; __any(open); e += 64) {
    const int j = min(e + lane, last), id = p.ids[j], n = p.shared[j];
    const bool linked = e + lane <= last && id >= 0 && n > 0 && id == p.ids[j - 1] && n == p.shared[j - 1];
    const unsigned long long more = __ballot(linked);
    const int k = ~more ? __ffsll(~more) - 1 : 64;
    if (open) f.count += k;
    open = open && k == 64;
  }
  return f;
}

// New and cached tokens of the sequences of a family's rows.  Lane l keeps
// those of sequence l, so that up to 64 sequences are read once, beside the
// families, and not behind them.
struct PrefixLengths {
  int act_q, act_k;
  __device__ __forceinline__ void load(const PagedPrefixParams& p, int lane) {
    const int b = min(lane, p.batch - 1);
    act_k = p.act_k[b];
    act_q = p.act_q ? p.act_q[b] : p.s1;
  }
  // the tokens of the family's prefix that new token s of sequence b sees
  __device__ __forceinline__ void bounds(const PagedPrefixParams& p, int b, int s, int tokens, int* lo, int* hi) const {
    int k, q;
    if (p.batch <= 64) {
      k = __shfl(act_k, b);
      q = __shfl(act_q, b);
    } else {
      k = p.act_k[b];
      q = p.act_q ? p.act_q[b] : p.s1;
    }
    paged_bounds(p, min(max(q, 0), p.s1), min(max(k, 0), p.max_blocks * p.page), s, lo, hi);
    *hi = min(*hi, tokens);
  }
};

// Jobs of one key head for blocks of R rows.
template <int R>
struct PrefixPlan {
  int per;           // tiles of a part, at most
  int jobs;          // in all
  PrefixFamily f;    // of this lane among the first 64 sequences,
  int m, t;          // its blocks of rows and tiles

  struct Job {
    PrefixFamily f;
    int job0, blocks, parts;  // of the family: its first job, blocks of rows, parts of its prefix
  };

  static __device__ __forceinline__ int div_up(int a, int b) { return (int)((unsigned)(a + b - 1) / (unsigned)b); }

  __device__ __forceinline__ void families(const PagedPrefixParams& p, int c0, int lane) {
    f = prefix_families(p, c0, lane);
    m = f.count ? (int)(((int64_t)f.count * p.rows + R - 1) / R) : 0;
    t = (f.tokens + kPrefixTile - 1) / kPrefixTile;
  }

  // sum m ceil(t / per) may be `most` jobs.  Up to 64 sequences the length of
  // the parts is fitted to the families; with more, which would be read again
  // for it, it is the shortest that has room for every rounding up, unless one
  // that has room for none happens to do.
  __device__ __forceinline__ void make(const PagedPrefixParams& p, int lane) {
    families(p, 0, lane);
    if (p.batch <= 64) {
      const int work = wave_total(m * t), most = prefix_jobs(wave_total(m), p.prefix_workers);
      per = max(div_up(work, most), kPrefixMinTiles);
      for (;;) {
        jobs = wave_total(m * div_up(t, per));
        if (jobs <= most) return;
        per += max(per >> 4, 1);
      }
    }
    int work = 0, rows = 0;
    for (int c0 = 0; c0 < p.batch; c0 += 64) {
      families(p, c0, lane);
      work += m * t;
      rows += m;
    }
    work = wave_total(work);
    rows = wave_total(rows);
    const int most = prefix_jobs(rows, p.prefix_workers);
    for (int room = 0;; room = rows) {
      per = max(div_up(work, most - room), kPrefixMinTiles);
      int n = 0;
      for (int c0 = 0; c0 < p.batch; c0 += 64) {
        families(p, c0, lane);
        n += m * div_up(t, per);
      }
      jobs = wave_total(n);
      if (jobs <= most) return;
    }
  }

  // job number `job` (below `jobs`)
  __device__ __forceinline__ Job find(const PagedPrefixParams& p, int lane, int job) {
    Job j = {{0, 0, 0}, 0, 1, 1};
    int base = 0;
    for (int c0 = 0; c0 < p.batch; c0 += 64) {
      if (p.batch > 64) families(p, c0, lane);
      const int parts = div_up(t, per), n = m * parts;
      const int incl = wave_scan(n);
      const unsigned long long hit = __ballot(base + incl > job);
      if (hit) {
        const int l = __ffsll(hit) - 1;
        j.f.first = __builtin_amdgcn_readlane(f.first, l);
        j.f.count = __builtin_amdgcn_readlane(f.count, l);
        j.f.tokens = __builtin_amdgcn_readlane(f.tokens, l);
        j.job0 = base + __builtin_amdgcn_readlane(incl - n, l);
        j.blocks = __builtin_amdgcn_readlane(m, l);
        j.parts = __builtin_amdgcn_readlane(parts, l);
        break;
      }
      base += __builtin_amdgcn_readlane(incl, 63);
    }
    return j;
  }
};

// n / d with magic = floor((2^32 - 1) / d): n * magic / 2^32 is at most
// n / 2^32 below n / d, so its integer part is off by one at most
__device__ __forceinline__ unsigned prefix_div(unsigned n, unsigned d, unsigned magic) {
  const unsigned q = __umulhi(n, magic);
  return q + (n - q * d >= d);
}

// Which job, of which key head, workgroup `block` of `grid` has in round `round`
// (-1: none): the jobs lie end to end over the XCDs (workgroup x runs on XCD
// x % 8), key head by key head.
__device__ __forceinline__ int prefix_job_of(int block, int grid, int round, int heads, int* head) {
  const int at = round * grid + (block & 7) * (grid >> 3) + (block >> 3);
  const int job = at / heads;
  *head = at - job * heads;
  return job;
}

// kernels of the two forms (paged_prefix.hip, paged_prefix_latent.hip)
int prefix_latent_launch(const PagedPrefixParams& p, int64_t d, int32_t dtype, unsigned grid, hipStream_t stream);
constexpr int kPrefixLatentRows = 128;

}  // namespace dsa
