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

// the families that start at sequences c0 .. c0 + 63, one per lane
__device__ __forceinline__ PrefixFamily prefix_families(const PagedPrefixParams& p, int c0, int lane) {
  auto linked = [&](int b) {  // to the sequence before it
    if (b <= 0 || b >= p.batch) return false;
    const int id = p.ids[b], n = p.shared[b];
    return id >= 0 && n > 0 && p.ids[b - 1] == id && p.shared[b - 1] == n;
  };
  const int b = c0 + lane;
  const bool mine = linked(b), next = linked(b + 1);
  const unsigned long long links = __ballot(mine);
  PrefixFamily f = {b, 0, 0};
  if (next && !mine) {
    const unsigned long long after = lane == 63 ? 0ull : links >> (lane + 1);
    f.count = __ffsll(~after);  // the links that follow, and the first sequence
    f.tokens = min(p.shared[b], p.max_blocks * p.page);
  }
  // a family that goes on behind these
  bool open = f.count > 0 && lane + f.count == 64 && b + f.count < p.batch;
  for (int e = c0 + 64; __any(open); e += 64) {
    const unsigned long long more = __ballot(linked(e + lane));
    const int n = ~more ? __ffsll(~more) - 1 : 64;
    if (open) f.count += n;
    open = open && n == 64;
  }
  return f;
}

// Jobs of one key head for blocks of R rows.
template <int R>
struct PrefixPlan {
  static constexpr int kHere = 4;  // batches of 64 sequences whose families stay in registers
  int per;                         // tiles of a part, at most
  int jobs;                        // in all

  static __device__ __forceinline__ int blocks(const PagedPrefixParams& p, const PrefixFamily& f) {
    return (int)(((int64_t)f.count * p.rows + R - 1) / R);
  }
  static __device__ __forceinline__ int tiles(const PrefixFamily& f) { return (f.tokens + kPrefixTile - 1) / kPrefixTile; }
  static __device__ __forceinline__ int div_up(int a, int b) { return (int)((unsigned)(a + b - 1) / (unsigned)b); }

  struct Job {
    PrefixFamily f;
    int job0, blocks, parts;  // of the family: its first job, blocks of rows, parts of its prefix
  };

  // The plan, and the job `job` of it (f.count 0 if there is none such).  Of
  // more than 64 * kHere sequences the parts are not fitted to the families.
  __device__ __forceinline__ Job make(const PagedPrefixParams& p, int lane, int job) {
    PrefixFamily f[kHere];
    int m[kHere], t[kHere];
    int work = 0, rows = 0;
#pragma unroll
    for (int i = 0; i < kHere; ++i) {
      m[i] = t[i] = 0;
      f[i] = {0, 0, 0};
      if (i * 64 < p.batch) {
        f[i] = prefix_families(p, i * 64, lane);
        m[i] = f[i].count ? blocks(p, f[i]) : 0;
        t[i] = tiles(f[i]);
        work += m[i] * t[i];
        rows += m[i];
      }
    }
    for (int c0 = kHere * 64; c0 < p.batch; c0 += 64) {
      const PrefixFamily g = prefix_families(p, c0, lane);
      const int n = g.count ? blocks(p, g) : 0;
      work += n * tiles(g);
      rows += n;
    }
    work = wave_total(work);
    rows = wave_total(rows);
    const int most = prefix_jobs(rows, p.prefix_workers);
    // sum m ceil(t / per) <= most: at least work / most; the rounding up costs `rows` jobs at most
    const bool here = p.batch <= kHere * 64;
    per = max(div_up(work, here ? most : most - rows), kPrefixMinTiles);
    for (;;) {
      int n = 0;
#pragma unroll
      for (int i = 0; i < kHere; ++i) n += m[i] * div_up(t[i], per);
      for (int c0 = kHere * 64; c0 < p.batch; c0 += 64) {
        const PrefixFamily g = prefix_families(p, c0, lane);
        if (g.count) n += blocks(p, g) * div_up(tiles(g), per);
      }
      jobs = wave_total(n);
      if (jobs <= most) break;
      per += max(per >> 4, 1);
    }
    return find(p, lane, job, f, m, t);
  }

  __device__ __forceinline__ Job find(const PagedPrefixParams& p, int lane, int job, const PrefixFamily (&f)[kHere],
                                      const int (&m)[kHere], const int (&t)[kHere]) const {
    Job j = {{0, 0, 0}, 0, 1, 1};
    if (job >= jobs) return j;
    int base = 0;
    auto here = [&](const PrefixFamily& g, int gm, int gt) {
      const int parts = div_up(gt, per), n = gm * parts;
      const int incl = wave_scan(n);
      const unsigned long long hit = __ballot(base + incl > job);
      if (!hit) {
        base += __builtin_amdgcn_readlane(incl, 63);
        return false;
      }
      const int l = __ffsll(hit) - 1;
      j.f.first = __builtin_amdgcn_readlane(g.first, l);
      j.f.count = __builtin_amdgcn_readlane(g.count, l);
      j.f.tokens = __builtin_amdgcn_readlane(g.tokens, l);
      j.job0 = base + __builtin_amdgcn_readlane(incl - n, l);
      j.blocks = __builtin_amdgcn_readlane(gm, l);
      j.parts = __builtin_amdgcn_readlane(parts, l);
      return true;
    };
#pragma unroll
    for (int i = 0; i < kHere; ++i)
      if (i * 64 < p.batch && here(f[i], m[i], t[i])) return j;
    for (int c0 = kHere * 64; c0 < p.batch; c0 += 64) {
      const PrefixFamily g = prefix_families(p, c0, lane);
      if (here(g, g.count ? blocks(p, g) : 0, tiles(g))) return j;
    }
    return j;
  }

  // another job of the plan
  __device__ __forceinline__ Job next(const PagedPrefixParams& p, int lane, int job) const {
    PrefixFamily f[kHere];
    int m[kHere], t[kHere];
#pragma unroll
    for (int i = 0; i < kHere; ++i) {
      f[i] = {0, 0, 0};
      m[i] = t[i] = 0;
      if (i * 64 < p.batch) {
        f[i] = prefix_families(p, i * 64, lane);
        m[i] = f[i].count ? blocks(p, f[i]) : 0;
        t[i] = tiles(f[i]);
      }
    }
    return find(p, lane, job, f, m, t);
  }
};

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
