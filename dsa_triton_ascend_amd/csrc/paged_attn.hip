// Attention of the newest tokens over paged key and value caches with grouped
// heads, and the join of the runs of a sequence (both described in
// paged_attn.h).
//
//   S^T = K Q^T,  P = 2^(S - ref),  O^T = V^T P^T
//
// Bound by the bytes of K and V: 2 (G / 2) flops per byte at G query heads
// per key head.  So every wave works alone, on its own run of tokens of one
// key head, with no LDS and no barrier; what it needs in flight sits in
// registers.  Neighbouring waves take neighbouring key heads of the same
// tokens, so that the rows of a page are read whole.  32 x 32K tokens of eight
// key heads of 128 columns, 4.3 GB: 650 us, 6.6 TB/s (a streaming read alone:
// 7.1); the join behind it takes 6 us.
//
// Per tile of 32 tokens: K goes straight into the A operand of 16x16x32
// (lane l: token l % 16, 16 bytes of 8 columns).  V is read a row at a time
// across 16 lanes, each lane 8 tokens x D/16 columns, and turned in the lane
// by byte permutes into V^T operands: the column a lane's MFMA row stands
// for, and the token its k slot stands for, are free to choose, and are
// chosen so that nothing crosses lanes.  Token 16 st + 4 g + r is k slot
// 8 g + 4 st + r of lane group g, which is also where S^T leaves its score,
// so P needs no shuffle either.  K of the next tile is loaded as soon as the
// scores are done, V of the next as soon as the output is.
//
// P is multiplied as a sum of two values of the input type (the MFMAs are
// idle otherwise), so the weights keep 16 bits and more.
#include "paged_attn.h"

namespace dsa {

__device__ __attribute__((aligned(16))) unsigned char g_paged_zero_row[1024];

constexpr int kPaTile = 32;
constexpr int kPaThreads = 256;

// Waves of a SIMD: as many as keep everything in registers, at most two.  At
// 128 columns three waves spill 12 registers, and each reload waits for the
// tile on its way too (32 x 32K tokens of eight key heads: 711 us against 663
// with two, 1350 with four); at 64 columns three fit and are slower (32 x 8K
// tokens of four key heads: 55 to 62 us against 51).
constexpr int pa_waves(int d, int mt) { return d <= 128 && mt <= 2 ? 2 : 1; }

// STREAM: loads that keep nothing in the caches, for more K and V than the
// caches hold from one call to the next.
template <typename T, int D, int MT, bool STREAM>
__global__ __launch_bounds__(kPaThreads, pa_waves(D, MT)) void paged_attn_kernel(PagedAttnParams p) {
  using E = Elem<T>;
  using V8 = typename E::v8;
  constexpr int KS = D / 32;   // k-steps of the scores
  constexpr int NJ = D / 16;   // output tiles
  constexpr int VC = D >= 128 ? D / 128 : 1;  // 16-byte pieces of a lane's V row
  constexpr int EPL = D / 16;  // V columns of a lane
  const int lane = threadIdx.x & 63;
  const int li = lane & 15, lg = lane >> 4;
  const int64_t wid = (int64_t)blockIdx.x * (kPaThreads / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int worker = (int)(wid / p.groups), ng = (int)(wid - (int64_t)worker * p.groups);
  if (worker >= p.workers) return;
  const int kvh = ng / p.row_groups, rg = ng - kvh * p.row_groups;

  PagedPlan plan;
  plan.make(p, kPaTile, lane);
  if (worker >= (plan.total + plan.per - 1) / plan.per) return;
  int at = worker * plan.per;
  const int end = min(at + plan.per, plan.total);
  int before;
  int b = plan.find(p, kPaTile, lane, at, &before);
  const int64_t row_bytes = (int64_t)p.n2 * D * 2;
  const unsigned char* kbase = (const unsigned char*)p.k + (int64_t)kvh * D * 2;
  const unsigned char* vbase = (const unsigned char*)p.v + (int64_t)kvh * D * 2;

  bool first_segment = true;
  b = __builtin_amdgcn_readfirstlane(b);
  PagedSeq seq = plan.sequence(p, b);  // (later ones are read again: the plan's do not stay in registers)
  while (at < end) {
    const int nt = paged_tiles(seq, kPaTile);
    if (nt == 0) {
      if (++b >= p.batch) break;
      seq = paged_seq_uniform(p, b);
      continue;
    }
    const int t0 = at - before, t1 = min(end - before, nt);
    const int tok0 = seq.lo + t0 * kPaTile, tok1 = min(seq.hi, seq.lo + t1 * kPaTile);
    const int32_t* tab = p.table + (int64_t)b * p.max_blocks;

    // rows of this lane's MFMA column: query head kvh * group + r % group of
    // token r / group
    V8 qf[MT][KS];
    int lo[MT], hi[MT];
    int64_t orow[MT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      const int r = rg * p.group_rows + mt * 16 + li;
      const bool live = r < p.rows;
      const int s = live ? r / p.group : 0;
      orow[mt] = live ? ((int64_t)b * p.s1 + s) * p.n1 + kvh * p.group + (r - s * p.group) : -1;
      paged_bounds(p, seq.act_q, seq.act_k, s, &lo[mt], &hi[mt]);
      if (!live) hi[mt] = 0;
      const u32x4 z = {0u, 0u, 0u, 0u};
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
        qf[mt][ks] = as_v8<V8>(live ? *(const u32x4*)((const T*)p.q + orow[mt] * D + ks * 32 + lg * 8) : z);
    }

    f32x4 acc[MT][NJ];
    float ref[MT], top[MT], sum[MT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      ref[mt] = top[mt] = -INFINITY;
      sum[mt] = 0.f;
#pragma unroll
      for (int j = 0; j < NJ; ++j) acc[mt][j] = {0.f, 0.f, 0.f, 0.f};
    }

    // cache row of token tile0 + lane % 32, -1 past the run's end or where
    // the table names no page
    auto page_of = [&](int tile0) {
      const int t = tile0 + (lane & 31);
      unsigned off;
      return t < tok1 ? tab[paged_split(p, (unsigned)t, &off)] : -1;
    };
    auto row_of = [&](int tile0, int blk) {
      unsigned off;
      paged_split(p, (unsigned)(tile0 + (lane & 31)), &off);
      const int64_t r = (int64_t)blk * p.page + (int)off;
      return blk < 0 || r >= p.kv_rows ? -1 : (int)r;
    };
    auto load = [](auto* at) {
      if constexpr (STREAM) return __builtin_nontemporal_load(at);
      else return *at;
    };
    u32x4 kf[2][KS];
    auto load_k = [&](int row) {
#pragma unroll
      for (int st = 0; st < 2; ++st) {
        const int r = __shfl(row, st * 16 + li);
        const unsigned char* src = r >= 0 ? kbase + r * row_bytes : g_paged_zero_row;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) kf[st][ks] = load((const u32x4*)(src + ks * 64 + lg * 16));
      }
    };
    typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
    unsigned vf[8][EPL / 2];
    auto load_v = [&](int row) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int r = __shfl(row, (i >> 2) * 16 + lg * 4 + (i & 3));
        const unsigned char* src = r >= 0 ? vbase + r * row_bytes : g_paged_zero_row;
        if constexpr (D == 64) {
          const u32x2 x = load((const u32x2*)(src + li * 8));
          vf[i][0] = x[0], vf[i][1] = x[1];
        } else {
#pragma unroll
          for (int c = 0; c < VC; ++c) {
            const u32x4 x = load((const u32x4*)(src + c * 256 + li * 16));
#pragma unroll
            for (int e = 0; e < 4; ++e) vf[i][c * 4 + e] = x[e];
          }
        }
      }
    };

    int row = row_of(tok0, page_of(tok0));
    load_k(row);
    load_v(row);
    int blk = page_of(tok0 + kPaTile);
    for (int tk = tok0; tk < tok1; tk += kPaTile) {
      const int next = row_of(tk + kPaTile, blk);
      blk = page_of(tk + 2 * kPaTile);
      f32x4 s[MT][2];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int st = 0; st < 2; ++st) {
          s[mt][st] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int ks = 0; ks < KS; ++ks) s[mt][st] = E::mfma(as_v8<V8>(kf[st][ks]), qf[mt][ks], s[mt][st]);
        }
      const bool more = tk + kPaTile < tok1;
      if (more) load_k(next);

      V8 ph[MT], pl[MT];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        float v[8], mx = -INFINITY;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int t = tk + (i >> 2) * 16 + lg * 4 + (i & 3);
          v[i] = t >= lo[mt] && t < hi[mt] ? s[mt][i >> 2][i & 3] * p.scale_log2 : -INFINITY;
          mx = fmaxf(mx, v[i]);
        }
        mx = xgroup_max(mx);
        top[mt] = fmaxf(top[mt], mx);
        if (__any(mx > ref[mt] + kPaAbove)) {
          const float nref = mx > ref[mt] + kPaAbove ? mx - kPaBelow : ref[mt];
          const float f = ref[mt] == -INFINITY ? 0.f : fast_exp2(ref[mt] - nref);
          ref[mt] = nref;
          sum[mt] *= f;
#pragma unroll
          for (int j = 0; j < NJ; ++j) acc[mt][j] *= f;
        }
        const float from = ref[mt] == -INFINITY ? 0.f : ref[mt];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float e = fast_exp2(v[i] - from);
          sum[mt] += e;
          ph[mt][i] = E::from_f32(e);
          pl[mt][i] = E::from_f32(e - E::to_f32(ph[mt][i]));
        }
      }
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        // columns EPL-major: piece j / 8 (or j / 4 at D = 64), element j % 8
        const int dw = j / 2;
        u32x4 w;
#pragma unroll
        for (int q2 = 0; q2 < 4; ++q2)
          w[q2] = __builtin_amdgcn_perm(vf[2 * q2 + 1][dw], vf[2 * q2][dw], j & 1 ? 0x07060302u : 0x05040100u);
        const V8 a = as_v8<V8>(w);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          acc[mt][j] = E::mfma(a, ph[mt], acc[mt][j]);
          acc[mt][j] = E::mfma(a, pl[mt], acc[mt][j]);
        }
      }
      if (more) load_v(next);
    }

    // MFMA j, register r of lane group g: column 8 (4 g + r) + j % 8 of piece
    // j / 8 (4 (4 g + r) + j at D = 64), so a lane holds whole chunks
    const bool whole = t0 == 0 && t1 == nt;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      const float l = xgroup_sum(sum[mt]);
      const float inv = l != 0.f ? 1.f / l : 0.f;
      constexpr int EC = D == 64 ? 4 : 8;  // elements of a chunk
      if (whole) {
        if (orow[mt] >= 0) {
          typedef T TC __attribute__((ext_vector_type(EC)));
#pragma unroll
          for (int c = 0; c < NJ / EC; ++c)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              TC o;
#pragma unroll
              for (int e = 0; e < EC; ++e) o[e] = E::from_f32(paged_scaled(acc[mt][c * EC + e][r], inv));
              *(TC*)((T*)p.out + orow[mt] * D + c * 128 + (lg * 4 + r) * EC) = o;
            }
          if (lg == 0 && p.smax) {
            // statistics are [B, N2, S1, G]
            const int rr = rg * p.group_rows + mt * 16 + li;
            const int64_t at2 = ((int64_t)b * p.n2 + kvh) * p.rows + rr;
            const bool any = p.return_lse && l != 0.f;
            p.smax[at2] = any ? top[mt] * kLn2 : 0.f;
            p.ssum[at2] = any ? l * fast_exp2(ref[mt] - top[mt]) : 0.f;
          }
        }
      } else {
        const int64_t slot = (((int64_t)worker * 2 + (first_segment ? 0 : 1)) * p.groups + ng) * p.group_rows +
                             mt * 16 + li;
        float* dst = p.part_o + slot * D;
        const float seen = l != 0.f ? 1.f : 0.f;
#pragma unroll
        for (int c = 0; c < NJ / EC; ++c)
#pragma unroll
          for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int e = 0; e < EC; e += 4) {
              const f32x4 o = {acc[mt][c * EC + e][r], acc[mt][c * EC + e + 1][r], acc[mt][c * EC + e + 2][r],
                               acc[mt][c * EC + e + 3][r]};
              *(f32x4*)(dst + c * 128 + (lg * 4 + r) * EC + e) = paged_scaled(o, seen);
            }
        if (lg == 0) p.part_ml[slot] = {ref[mt], l, top[mt], l};
      }
    }
    first_segment = false;
    at = before + t1;
    if (t1 == nt) {
      at = before += plan.padded(nt);
      if (at < end) seq = paged_seq_uniform(p, ++b);
    }
  }
}

// ---------------------------------------------------------------------------
// join: a workgroup takes `wg_rows` rows of a sequence.  With up to 64 runs a
// wave takes a row; with more (one row per workgroup, where the host expects
// them) the four waves share them.  A lane holds D / 64 columns and, for the
// weights, one run of 64.  Sequences without a visible token get their zeros
// here.
// ---------------------------------------------------------------------------
constexpr int kPcFewRuns = 64;

template <typename T, int D>
__global__ __launch_bounds__(256) void paged_combine_kernel(PagedAttnParams p, int tile, int wg_rows) {
  using E = Elem<T>;
  constexpr int EPL = D / 64;
  typedef T TV __attribute__((ext_vector_type(EPL)));
  typedef float FV __attribute__((ext_vector_type(EPL)));
  __shared__ FV s_o[4][64];
  __shared__ float s_l[4], s_n[4];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int per_seq = p.n2 * p.rows, groups = (per_seq + wg_rows - 1) / wg_rows;
  const int b = blockIdx.x / groups, row0 = (blockIdx.x - b * groups) * wg_rows;

  PagedPlan plan;
  plan.make(p, tile, lane);
  const int nt = paged_tiles(plan.sequence(p, b), tile);
  const int first = plan.start(p, tile, lane, b), last = first + nt - 1;
  const int w0 = nt ? plan.worker_of(first) : 0;
  const int runs = nt ? plan.worker_of(last) - w0 + 1 : 0;
  if (runs == 1) return;  // written whole by its worker
  const int slot0 = first != w0 * plan.per ? 1 : 0;  // of the first worker; the others' is 0

  // the runs i0 .. i1 of a row, summed relative to the largest reference of all
  auto row_of = [&](int row, int i0, int i1, float* big, float* top, FV* o, float* l, float* n) {
    const int kvh = row / p.rows, rr = row - kvh * p.rows;  // row rr = s * group + head
    const int rg = rr / p.group_rows;
    const int64_t in_group = (int64_t)(kvh * p.row_groups + rg) * p.group_rows + (rr - rg * p.group_rows);
    const int64_t span = (int64_t)p.groups * p.group_rows;
    auto slot = [&](int i) { return ((int64_t)(w0 + i) * 2 + (i == 0 ? slot0 : 0)) * span + in_group; };
    float m = -INFINITY, t = -INFINITY;
    for (int i = lane; i < runs; i += 64) {
      const f32x4 ml = p.part_ml[slot(i)];
      m = fmaxf(m, ml[0]);
      t = fmaxf(t, ml[2]);
    }
    *big = m = wave_max(m);
    *top = wave_max(t);
    FV acc = {};
    float la = 0.f, na = 0.f;
    if (m != -INFINITY)
      for (int c = i0; c < i1; c += 64) {
        const int mine = c + lane;
        float f = 0.f;
        if (mine < i1) {
          const f32x4 ml = p.part_ml[slot(mine)];
          f = fast_exp2(ml[0] - m);
          la += ml[1] * f;
          na += ml[3] * f;
        }
        const int cnt = min(64, i1 - c);
        for (int i = 0; i < cnt; i += 8) {
          // eight rows in flight (those past the last read it again, times zero)
          FV x[8];
#pragma unroll
          for (int u = 0; u < 8; ++u) x[u] = *((const FV*)p.part_o + slot(c + min(i + u, cnt - 1)) * 64 + lane);
#pragma unroll
          for (int u = 0; u < 8; ++u) {
            const float g =
                i + u < cnt ? __int_as_float(__builtin_amdgcn_readlane(__float_as_int(f), (i + u) & 63)) : 0.f;
#pragma unroll
            for (int e = 0; e < EPL; ++e) acc[e] += i + u < cnt ? x[u][e] * g : 0.f;
          }
        }
      }
    *o = acc;
    *l = wave_sum(la);
    *n = wave_sum(na);
  };
  auto write = [&](int row, FV o, float big, float top, float l, float n) {
    const int kvh = row / p.rows, rr = row - kvh * p.rows;
    const int s = rr / p.group;
    const int64_t orow = ((int64_t)b * p.s1 + s) * p.n1 + kvh * p.group + (rr - s * p.group);
    const float inv = n != 0.f ? 1.f / n : 0.f;
    TV r;
#pragma unroll
    for (int e = 0; e < EPL; ++e) r[e] = E::from_f32(paged_scaled(o[e], inv));
    *(TV*)((T*)p.out + orow * D + lane * EPL) = r;
    if (lane == 0 && p.smax) {
      const int64_t srow = (int64_t)b * per_seq + row;
      const bool any = p.return_lse && l != 0.f;
      p.smax[srow] = any ? top * kLn2 : 0.f;
      p.ssum[srow] = any ? l * fast_exp2(big - top) : 0.f;
    }
  };
  FV o;
  float big, top, l, n;
  if (runs <= kPcFewRuns && wg_rows > 1) {
    if (row0 + wave < per_seq) {
      row_of(row0 + wave, 0, runs, &big, &top, &o, &l, &n);
      write(row0 + wave, o, big, top, l, n);
    }
    return;
  }
  const int part = (runs + 3) / 4;
  for (int row = row0; row < min(row0 + wg_rows, per_seq); ++row) {
    row_of(row, min(wave * part, runs), min((wave + 1) * part, runs), &big, &top, &o, &l, &n);
    s_o[wave][lane] = o;
    if (lane == 0) s_l[wave] = l, s_n[wave] = n;
    __syncthreads();
    if (wave == 0) {
#pragma unroll
      for (int w = 1; w < 4; ++w) {
        o += s_o[w][lane];
        l += s_l[w];
        n += s_n[w];
      }
      write(row, o, big, top, l, n);
    }
    __syncthreads();
  }
}

template <typename T>
static void paged_combine_d(const PagedAttnParams& p, int tile, int wg_rows, int64_t d, unsigned grid, hipStream_t stream) {
  if (d == 64) paged_combine_kernel<T, 64><<<grid, 256, 0, stream>>>(p, tile, wg_rows);  // grouped form only
  else if (d == 128) paged_combine_kernel<T, 128><<<grid, 256, 0, stream>>>(p, tile, wg_rows);
  else if (d == 256) paged_combine_kernel<T, 256><<<grid, 256, 0, stream>>>(p, tile, wg_rows);
  else paged_combine_kernel<T, 512><<<grid, 256, 0, stream>>>(p, tile, wg_rows);
}

// rows of a workgroup of the join: four, one per wave, unless the average
// sequence has so many runs that the waves had better share them
static int paged_combine_rows(int64_t workers, int64_t batch) { return workers > 32 * batch ? 1 : 4; }
static int64_t paged_combine_grid(int64_t workers, int64_t batch, int64_t s1, int64_t n1) {
  const int wg_rows = paged_combine_rows(workers, batch);
  return batch * ((s1 * n1 + wg_rows - 1) / wg_rows);
}

int paged_combine_launch(const PagedAttnParams& p, int tile, int64_t d, int32_t dtype, hipStream_t stream) {
  const int wg_rows = paged_combine_rows(p.workers, p.batch);
  const unsigned grid = (unsigned)paged_combine_grid(p.workers, p.batch, p.s1, p.n1);
  if (dtype == DSA_DTYPE_BF16) paged_combine_d<bf16>(p, tile, wg_rows, d, grid, stream);
  else paged_combine_d<f16>(p, tile, wg_rows, d, grid, stream);
  DSA_HIP(hipGetLastError());
  return DSA_OK;
}

size_t paged_part_bytes(const PagedShape& s, int64_t d) {
  const size_t rows = (size_t)s.workers * 2 * s.groups * s.group_rows;
  return rows * (sizeof(f32x4) + d * sizeof(float));
}

// Workers of a lane group for `slots` workers resident at once.  As many as
// fill the slots once; where the lane groups alone come near that, so many
// that the last round of them is nearly full too.  Never more than sequences
// of the longest length, `tiles`, keep busy.
int paged_workers(int64_t slots, int64_t groups, int64_t batch, int64_t tiles, int min_tiles) {
  int64_t best = slots / groups;
  if (best < 8) {
    double best_fill = 0;
    const int64_t from = best < 1 ? 1 : best;
    for (int64_t w = from; w < from + 8; ++w) {
      const int64_t all = w * groups, rounds = (all + slots - 1) / slots;
      const double fill = (double)all / ((double)rounds * slots);
      if (fill > best_fill + 0.02) best = w, best_fill = fill;
    }
  }
  const int64_t most = batch * ((tiles + min_tiles - 1) / min_tiles);
  return (int)(best > most ? (most < 1 ? 1 : most) : best);
}

static PagedShape paged_grouped_shape(int64_t batch, int64_t s1, int64_t n1, int64_t n2, int64_t d,
                                      int64_t max_blocks, int64_t page) {
  PagedShape s;
  s.tile = kPaTile;
  const int64_t rows = s1 * (n1 / n2);
  int mt = rows <= 16 ? 1 : (rows <= 32 ? 2 : 4);
  if (d * mt > 512) mt = 2;
  s.group_rows = mt * 16;
  s.row_groups = (int)((rows + s.group_rows - 1) / s.group_rows);
  s.groups = (int)n2 * s.row_groups;
  s.min_tiles = kPaMinTiles;
  s.workers = paged_workers((int64_t)device_cu_count() * 4 * pa_waves((int)d, mt), s.groups, batch,
                            (max_blocks * page + kPaTile - 1) / kPaTile, s.min_tiles);
  return s;
}

static PagedShape paged_shape(int64_t batch, int64_t s1, int64_t n1, int64_t n2, int64_t d, bool latent,
                              int64_t max_blocks, int64_t page) {
  return latent ? paged_latent_shape(batch, s1, n1, d, max_blocks, page)
                : paged_grouped_shape(batch, s1, n1, n2, d, max_blocks, page);
}

static int64_t paged_grouped_grid(int64_t workers, int64_t groups) {
  return (workers * groups + kPaThreads / 64 - 1) / (kPaThreads / 64);
}

bool paged_attn_launchable(int64_t batch, int64_t s1, int64_t n1, int64_t n2, int64_t d, bool latent,
                           int64_t max_blocks, int64_t page) {
  const PagedShape s = paged_shape(batch, s1, n1, n2, d, latent, max_blocks, page);
  return (latent ? paged_latent_launchable(s.workers, s.row_groups)
                 : launchable(paged_grouped_grid(s.workers, s.groups), kPaThreads)) &&
         launchable(paged_combine_grid(s.workers, batch, s1, n1), 256);
}

size_t paged_attn_workspace_bytes(int64_t batch, int64_t s1, int64_t n1, int64_t n2, int64_t d, bool latent,
                                  int64_t max_blocks, int64_t page) {
  return paged_part_bytes(paged_shape(batch, s1, n1, n2, d, latent, max_blocks, page), d);
}

template <typename T, int D, int MT>
static void paged_launch_one(const PagedAttnParams& p, bool streaming, unsigned grid, hipStream_t stream) {
  if (streaming) paged_attn_kernel<T, D, MT, true><<<grid, kPaThreads, 0, stream>>>(p);
  else paged_attn_kernel<T, D, MT, false><<<grid, kPaThreads, 0, stream>>>(p);
}

template <typename T, int D>
static void paged_launch_mt(const PagedAttnParams& p, bool streaming, unsigned grid, hipStream_t stream) {
  if (p.group_rows == 16) paged_launch_one<T, D, 1>(p, streaming, grid, stream);
  else if (p.group_rows == 32) paged_launch_one<T, D, 2>(p, streaming, grid, stream);
  else if constexpr (D <= 128) paged_launch_one<T, D, 4>(p, streaming, grid, stream);
}

template <typename T>
static void paged_launch(const PagedAttnParams& p, int64_t d, bool streaming, unsigned grid, hipStream_t stream) {
  if (d == 64) paged_launch_mt<T, 64>(p, streaming, grid, stream);
  else if (d == 128) paged_launch_mt<T, 128>(p, streaming, grid, stream);
  else paged_launch_mt<T, 256>(p, streaming, grid, stream);
}

int paged_attn_run(const void* query, const void* query_rope, const void* key, const void* key_rope,
                   const void* value, void* out, float* smax, float* ssum, const int32_t* act_q,
                   const int32_t* act_k, const int32_t* table, int64_t batch, int64_t s1, int64_t n1, int64_t n2,
                   int64_t d, int64_t num_blocks, int64_t page, int64_t max_blocks, int32_t mode, int64_t pre_tokens,
                   int64_t next_tokens, int32_t dtype, float scale, int32_t return_lse, void* workspace,
                   hipStream_t stream) {
  const bool latent = value == nullptr;
  const PagedShape s = paged_shape(batch, s1, n1, n2, d, latent, max_blocks, page);
  PagedAttnParams p = {};
  p.q = query;
  p.qr = query_rope;
  p.k = key;
  p.kr = key_rope;
  p.v = value;
  p.out = out;
  p.smax = smax;
  p.ssum = ssum;
  p.act_q = act_q;
  p.act_k = act_k;
  p.table = table;
  const int64_t part_rows = (int64_t)s.workers * 2 * s.groups * s.group_rows;
  p.part_ml = (f32x4*)workspace;
  p.part_o = (float*)(p.part_ml + part_rows);
  p.kv_rows = num_blocks * page;
  p.band_pre = band_clamp(pre_tokens);
  p.band_next = band_clamp(next_tokens);
  p.batch = (int)batch;
  p.s1 = (int)s1;
  p.n1 = (int)n1;
  p.n2 = (int)n2;
  p.group = (int)(n1 / n2);
  p.rows = (int)(s1 * p.group);
  p.max_blocks = (int)max_blocks;
  p.page = (int)page;
  p.mode = mode;
  p.return_lse = return_lse;
  p.workers = s.workers;
  p.min_tiles = s.min_tiles;
  p.groups = s.groups;
  p.row_groups = s.row_groups;
  p.group_rows = s.group_rows;
  p.page_magic = 0xffffffffu / (unsigned)page;
  p.scale_log2 = scale * kLog2e;
  if (latent) {
    const int st = paged_latent_launch(p, d, dtype, stream);
    if (st != DSA_OK) return st;
  } else {
    const unsigned grid = (unsigned)paged_grouped_grid(s.workers, s.groups);
    // K and V that the caches could hold until the next call are kept there
    // (134 MB: 38 us, streaming 41; 537 MB: 115 us, streaming 104)
    const int64_t tokens = p.kv_rows < batch * max_blocks * page ? p.kv_rows : batch * max_blocks * page;
    const bool streaming = tokens * n2 * d * 4 > (256ll << 20);
    if (dtype == DSA_DTYPE_BF16) paged_launch<bf16>(p, d, streaming, grid, stream);
    else paged_launch<f16>(p, d, streaming, grid, stream);
    DSA_HIP(hipGetLastError());
  }
  return paged_combine_launch(p, s.tile, d, dtype, stream);
}

}  // namespace dsa
