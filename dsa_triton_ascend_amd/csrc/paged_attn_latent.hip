// Attention of the newest tokens over a paged latent cache (described in
// paged_attn.h): one key head of D + 64 columns, its first D the value too.
//
//   S^T = K Q^T,  P = 2^(S - ref),  O^T = V^T P^T,  V = K[:, :D]
//
// At 128 heads a token is 242 flops per byte, so bytes, matrix rate and LDS
// reads are all near their limits; below that the bytes are.  A token is
// read from memory once per workgroup and serves both products and every
// row (head, new token) of the workgroup.
//
// One workgroup of eight waves per CU owns a run of tokens for HG rows.
//  * Tiles of 32 tokens come by LDS-DMA into a ring, chunks swizzled so that
//    both products read them without bank conflicts.
//  * S^T: a wave takes 16 rows and all 32 tokens (HG = 128) or 16 of them.
//    Its Q stays in registers.
//  * P goes through LDS, 64 bytes per row: token 16 tt + 4 g + r in slot
//    8 g + 4 tt + r, chunk g at g ^ (row / 4 % 4).
//  * O^T: a wave owns D / 8 columns of all HG rows, so each V^T fragment is
//    read by one wave and serves all rows.
//  * The scores of tile t + 1 are computed in the same stretch as the output
//    of tile t, with two P buffers and one barrier per tile, so that a SIMD's
//    two waves can be in different products.
// The references (paged_attn.h) are looked at once per tile: a wave that
// sees a score too far above its row's raises a flag, and behind the barrier
// everyone takes the slow way for that tile (exchange of the maxima, new
// numerators, rescaled output).  That happens on a run's first tile and
// seldom after it.
//
// Up to 64 rows P is multiplied as a sum of two values of the input type.  At
// 128 rows the second product would take half of the time again, so P is
// rounded once there, and the output is divided by the sum of the rounded
// values: the weights still add up to one, and what is left is the rounding
// of single weights, below the rounding of the output.
#include "paged_attn.h"
#include "sfa_fwd.h"

namespace dsa {

__device__ __attribute__((aligned(16))) unsigned char g_latent_zero_row[1024];

constexpr int kPlTile = 32;
constexpr int kPlThreads = 512;
constexpr int kPlPages = 1024;  // block-table entries held in LDS

template <int D, typename T, int HG>
__global__ __launch_bounds__(kPlThreads, 1) void paged_latent_kernel(PagedAttnParams p) {
  using E = Elem<T>;
  using V8 = typename E::v8;
  typedef T T4 __attribute__((ext_vector_type(4)));
  constexpr int NW = kPlThreads / 64;
  constexpr int HGT = HG / 16;         // row tiles
  constexpr int TW = HG == 128 ? 1 : 2;  // waves that share a row tile's tokens
  constexpr int NTT = 2 / TW;          // 16-token sub-tiles of a wave's scores
  constexpr int NG1 = HGT * TW;        // waves that compute scores
  constexpr bool kLo = HG <= 64;       // P as two values
  constexpr int NPB = kLo ? 2 : 1;
  constexpr int DR = 64;
  constexpr int KS = (D + DR) / 32, KSN = D / 32;
  constexpr int NDW = D / NW / 16;     // output column tiles of a wave
  constexpr int TILE = kPlTile;
  constexpr int NOPE_BYTES = TILE * D * 2;
  constexpr int BUF_BYTES = NOPE_BYTES + TILE * DR * 2;
  constexpr int NBUF = HG <= 32 ? 4 : 3;  // what fits beside P
  constexpr int CPT = D / 8;           // 16-byte chunks of a token
  constexpr int TPI = 64 / CPT;        // tokens of one DMA
  constexpr int NIW = TILE / TPI / NW;  // DMAs of a wave per tile, beside the rope rows' (waves 0..3)
  constexpr int ROPE0 = NBUF * NOPE_BYTES;
  constexpr int PROW = TILE * 2;
  static_assert(NG1 <= NW && NIW * TPI * NW == TILE && NDW * 16 * NW == D, "tile split");
  // a token's row of buffer b; buffers alternate per DMA
  auto nope_off = [](int tk, int b) { return ((tk / TPI) * NBUF + b) * 1024 + (tk % TPI) * (D * 2); };
  auto rope_off = [](int tk, int b) { return ROPE0 + ((tk >> 3) * NBUF + b) * 1024 + (tk & 7) * (DR * 2); };

  __shared__ __attribute__((aligned(16))) unsigned char smem[NBUF * BUF_BYTES];
  __shared__ __attribute__((aligned(16))) unsigned char s_p[2 * NPB * HG * PROW];
  __shared__ int s_tab[kPlPages];
  __shared__ float s_mx[TW * HG], s_l[TW * HG], s_f[HG];
  __shared__ int s_flag[3];  // of a tile: its number modulo 3

  const int tid = threadIdx.x, lane = tid & 63;
  const int li = lane & 15, lg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const bool scores = wave < NG1;
  const int hq = wave % HGT, th = scores ? wave / HGT : 0;

  // the row groups of a worker read the same tokens: they share an XCD
  const int jj = blockIdx.x >> 3;
  const int rg = jj % p.row_groups;
  const int worker = (jj / p.row_groups) * 8 + (blockIdx.x & 7);
  if (worker >= p.workers) return;
  PagedPlan plan;
  plan.make(p, TILE, lane);
  int64_t at = (int64_t)worker * plan.per;
  const int64_t end = min(at + plan.per, plan.total);
  if (at >= end) return;
  int64_t before;
  int b = plan.find(p, TILE, lane, at, &before);

  const unsigned smem_base = (unsigned)(uintptr_t)smem;
  const bool rope_wave = wave < 4;
  const unsigned char* const kbase = (const unsigned char*)p.k;
  const unsigned char* const rbase = (const unsigned char*)p.kr;
  // this lane's addresses in the two products, made anew from the lane's
  // number in every step: kept, they would push Q or the output out of the
  // registers
  auto fresh_lane = []() {
    int ln = __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0u));
    asm volatile("" : "+v"(ln));
    return ln;
  };
  constexpr int G1_TT = ((16 / TPI) * NBUF) * 1024;
  constexpr int G1R_TT = 2 * NBUF * 1024;
  auto a1 = [&](int g1b, int g1rb, int ks, int tt) -> V8 {
    if (ks < KSN) return as_v8<V8>(*(const u32x4*)(smem + ((g1b ^ ((ks & 3) << 6)) + tt * G1_TT + (ks >> 2) * 256)));
    return as_v8<V8>(*(const u32x4*)(smem + ((g1rb ^ ((ks - KSN) << 6)) + tt * G1R_TT)));
  };
  auto a2 = [&](int g2b, int dt) -> V8 {
    const unsigned char* pp = smem + ((g2b ^ ((dt & 7) << 5)) + (dt >> 3) * 256);
    const bf16x4 v1 = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16x4*)pp);
    const bf16x4 v2 = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16x4*)(pp + G1_TT));
    const i16x4 w1 = __builtin_bit_cast(i16x4, v1), w2 = __builtin_bit_cast(i16x4, v2);
    const i16x8 w = {w1[0], w1[1], w1[2], w1[3], w2[0], w2[1], w2[2], w2[3]};
    return __builtin_bit_cast(V8, w);
  };

  bool first_segment = true;
  while (at < end) {
    b = __builtin_amdgcn_readfirstlane(b);
    PagedSeq seq = paged_seq(p, b);
    seq.lo = __builtin_amdgcn_readfirstlane(seq.lo);
    seq.hi = __builtin_amdgcn_readfirstlane(seq.hi);
    const int nt = paged_tiles(seq, TILE);
    if (nt == 0) {
      ++b;
      continue;
    }
    const int t0 = (int)(at - before), t1 = (int)min(end - before, (int64_t)nt);
    const int tok0 = seq.lo + t0 * TILE, tok1 = min(seq.hi, seq.lo + t1 * TILE);
    const int32_t* tab = p.table + (int64_t)b * p.max_blocks;

    // row of this lane's column of the scores: head rr % n1 of new token rr / n1
    const int rr = rg * HG + hq * 16 + li;
    const bool live = scores && rr < p.rows;
    int lo = 0, hi = 0;
    V8 qf[KS];
    {
      const int s = live ? rr / p.n1 : 0;
      const int64_t qrow = (int64_t)b * p.rows + (live ? rr : 0);
      // (rows that do not exist read row 0; what they compute is not stored)
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const T* src = ks < KSN ? (const T*)p.q + qrow * D + ks * 32 + lg * 8
                                : (const T*)p.qr + qrow * DR + (ks - KSN) * 32 + lg * 8;
        qf[ks] = as_v8<V8>(*(const u32x4*)src);
      }
      if (live) paged_bounds(p, seq.act_q, seq.act_k, s, &lo, &hi);
    }
    // the loads end here, not inside the tile loop, where a wait for them
    // would be one for the tiles in flight too
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) asm volatile("" : "+v"(qf[ks]));
    // tokens that all of the wave's rows see need no mask
    int all_lo = live ? lo : 0, all_hi = live ? hi : 0x7fffffff;
#pragma unroll
    for (int o = 8; o >= 1; o >>= 1) {
      all_lo = max(all_lo, __shfl_xor(all_lo, o));
      all_hi = min(all_hi, __shfl_xor(all_hi, o));
    }
    all_lo = __builtin_amdgcn_readfirstlane(all_lo);
    all_hi = __builtin_amdgcn_readfirstlane(all_hi);

    f32x4 acc[NDW][HGT];
#pragma unroll
    for (int j = 0; j < NDW; ++j)
#pragma unroll
      for (int ht = 0; ht < HGT; ++ht) acc[j][ht] = {0.f, 0.f, 0.f, 0.f};
    float ref = -INFINITY, top = -INFINITY, sum = 0.f, sum_p = 0.f;

    for (int ta = tok0; ta < tok1;) {
      // the run's pages, as many as the LDS holds at a time
      unsigned off0;
      const int pg0 = (int)paged_split(p, (unsigned)ta, &off0);
      const int tb = (int)min((int64_t)tok1, (int64_t)(pg0 + kPlPages) * p.page);
      const int npg = (int)(((int64_t)tb - 1) / p.page) - pg0 + 1;
      lds_barrier();  // the pages, tiles and numerators of the stretch before are read
      if (tid < 3) s_flag[tid] = 0;
      for (int i = tid; i < npg; i += kPlThreads) s_tab[i] = tab[pg0 + i];
      lds_barrier();
      const int n_tiles = (tb - ta + TILE - 1) / TILE;

      auto issue = [&](int t, int buf) {
        const int lane = fresh_lane();
        // lane l < 32 finds token l's row, -1 past the end or without a page
        const int tok = ta + t * TILE + (lane & 31);
        int row = -1;
        if (tok < tb) {
          unsigned off;
          const unsigned pg = paged_split(p, (unsigned)tok, &off);
          const int blk = s_tab[(int)pg - pg0];
          const int64_t r = (int64_t)blk * p.page + (int)off;
          row = blk < 0 || r >= p.kv_rows ? -1 : (int)r;
        }
#pragma unroll
        for (int j = 0; j < NIW; ++j) {
          const int tk = (j * NW + wave) * TPI + lane / CPT;
          const int ch = (lane % CPT) ^ nope_swz(tk);
          const int r = TPI == 1 ? __builtin_amdgcn_readlane(row, j * NW + wave) : __shfl(row, tk);
          dma_glb16(smem_base + nope_off((j * NW + wave) * TPI, buf),
                    r >= 0 ? kbase + (int64_t)r * (D * 2) + ch * 16 : g_latent_zero_row + ch * 16);
        }
        if (rope_wave) {
          const int tk = wave * 8 + (lane >> 3);
          const int ch = (lane & 7) ^ rope_swz(tk);
          const int r = __shfl(row, tk);
          dma_glb16(smem_base + rope_off(wave * 8, buf),
                    r >= 0 ? rbase + (int64_t)r * (DR * 2) + ch * 16 : g_latent_zero_row + ch * 16);
        }
      };
      f32x4 s[NTT];
      auto gemm1 = [&](int buf) {
        f32x4 a[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
        // two accumulators, so that neighbouring MFMAs are independent
        // (sub-tiles, or even and odd k-steps); PF fragments read ahead, and
        // no more (the accumulators leave few registers)
        constexpr int NS = KS * NTT, PF = 4;
        const int ln = fresh_lane(), l = ln & 15, g = ln >> 4;
        const int g1b = nope_off(l, 0) + ((g ^ nope_swz(l)) * 16) + buf * 1024;
        const int g1rb = rope_off(l, 0) + ((g ^ rope_swz(l)) * 16) + buf * 1024;
        auto read = [&](int st) { return a1(g1b, g1rb, st / NTT, NTT == 1 ? th : st % NTT); };
        V8 fa[PF];
#pragma unroll
        for (int i = 0; i < PF; ++i) fa[i] = read(i);
#pragma unroll
        for (int st = 0; st < NS; ++st) {
          const V8 f = fa[st % PF];
          if (st + PF < NS) fa[st % PF] = read(st + PF);
          a[st & 1] = E::mfma(f, qf[st / NTT], a[st & 1]);
          if constexpr (HG == 128) __builtin_amdgcn_sched_barrier(0);
        }
        if constexpr (NTT == 1) s[0] = a[0] + a[1];
        else s[0] = a[0], s[1] = a[1];
      };
      // numerators of the wave's scores into P buffer `par`; their sums
      float v[NTT * 4], tmax, es, eps;
      auto scale_mask = [&](int t) {
        const int tk = ta + t * TILE;
        tmax = -INFINITY;
        if (tk >= all_lo && tk + TILE <= min(all_hi, tb)) {
#pragma unroll
          for (int i = 0; i < NTT * 4; ++i) v[i] = s[i >> 2][i & 3] * p.scale_log2;
        } else {
#pragma unroll
          for (int i = 0; i < NTT * 4; ++i) {
            const int tok = tk + (NTT == 1 ? th : i >> 2) * 16 + lg * 4 + (i & 3);
            v[i] = tok >= lo && tok < min(hi, tb) ? s[i >> 2][i & 3] * p.scale_log2 : -INFINITY;
          }
        }
#pragma unroll
        for (int i = 0; i < NTT * 4; ++i) tmax = fmaxf(tmax, v[i]);
        tmax = xgroup_max(tmax);
      };
      auto numerators = [&](int par) {
        const float from = ref == -INFINITY ? 0.f : ref;
        const int ln = fresh_lane(), l = ln & 15, g = ln >> 4;
        unsigned char* dst = s_p + par * (NPB * HG * PROW) + (hq * 16 + l) * PROW + ((g ^ ((l >> 2) & 3)) * 16);
        es = 0.f;
        eps = 0.f;
#pragma unroll
        for (int u = 0; u < NTT; ++u) {
          T4 h, lw;
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float e = fast_exp2(v[u * 4 + r] - from);
            es += e;
            h[r] = E::from_f32(e);
            if constexpr (kLo) lw[r] = E::from_f32(e - E::to_f32(h[r]));
            else eps += E::to_f32(h[r]);
          }
          *(T4*)(dst + (NTT == 1 ? th : u) * 8) = h;
          if constexpr (kLo) *(T4*)(dst + HG * PROW + (NTT == 1 ? th : u) * 8) = lw;
        }
      };
      auto gemm2 = [&](int buf, int par) {
        const int ln = fresh_lane(), l = ln & 15, g = ln >> 4;
        const int r1 = g * 4 + (l >> 2);
        const int g2b = nope_off(r1, 0) + ((((l & 3) >> 1) ^ nope_swz(r1)) * 16) + (l & 1) * 8 + buf * 1024;
        V8 va[NDW];
#pragma unroll
        for (int j = 0; j < NDW; ++j) va[j] = a2(g2b, wave * NDW + j);
        const unsigned char* src = s_p + par * (NPB * HG * PROW) + l * PROW + ((g ^ ((l >> 2) & 3)) * 16);
        auto read = [&](int ht, int part) {
          return as_v8<V8>(*(const u32x4*)(src + part * HG * PROW + ht * 16 * PROW));
        };
        V8 nh = read(0, 0), nl = kLo ? read(0, 1) : nh;
#pragma unroll
        for (int ht = 0; ht < HGT; ++ht) {
          const V8 ph = nh, pl = nl;
          if (ht + 1 < HGT) {
            nh = read(ht + 1, 0);
            if constexpr (kLo) nl = read(ht + 1, 1);
          }
#pragma unroll
          for (int j = 0; j < NDW; ++j) acc[j][ht] = E::mfma(va[j], ph, acc[j][ht]);
          if constexpr (kLo) {
#pragma unroll
            for (int j = 0; j < NDW; ++j) acc[j][ht] = E::mfma(va[j], pl, acc[j][ht]);
          }
          if constexpr (HG == 128) __builtin_amdgcn_sched_barrier(0);
        }
      };

#pragma unroll
      for (int t = 0; t < NBUF - 1; ++t)
        if (t < n_tiles) issue(t, t);
      wait_vmcnt<0>();
      lds_barrier();
      // step t: scores of tile t + 1, output of tile t
      int buf = NBUF - 1;  // buffer of tile t
      int flag = 0;        // of tile t + 1
      for (int t = -1; t < n_tiles; ++t) {
        const int next = buf + 1 == NBUF ? 0 : buf + 1;
        const bool more = t + 1 < n_tiles;
        const bool loads = t >= 0 && t + NBUF - 1 < n_tiles;
        if (loads) issue(t + NBUF - 1, buf == 0 ? NBUF - 1 : buf - 1);
        auto score_tile = [&]() {
          gemm1(next);
          scale_mask(t + 1);
          numerators((t + 1) & 1);
          if (__any(tmax > ref + kPaAbove) && lane == 0) s_flag[flag] = 1;
        };
        // of the two waves of a SIMD one starts with the scores and one with
        // the output, so that one's MFMAs run beside the other's softmax
        if (more && scores && wave < 4) score_tile();
        if (t >= 0) gemm2(buf, t & 1);
        if (more && scores && wave >= 4) score_tile();
        // tile t + 2's flag, last read a barrier ago
        const int flag2 = flag == 2 ? 0 : flag + 1;
        if (tid == 0) s_flag[flag2] = 0;
        // tile t + 2 has landed: with four buffers the one after it may be
        // in flight
        if (NBUF == 3 || !loads) wait_vmcnt<0>();
        else if (rope_wave) wait_vmcnt<NIW + 1>();
        else wait_vmcnt<NIW>();
        lds_barrier();
        if (!more) break;
        const bool moved = __builtin_amdgcn_readfirstlane(s_flag[flag]) != 0;
        flag = flag2;
        if (moved) {
          if (scores && lg == 0) s_mx[th * HG + hq * 16 + li] = tmax;
          lds_barrier();
          if (scores) {
            float mx = s_mx[hq * 16 + li];
            if constexpr (TW == 2) mx = fmaxf(mx, s_mx[HG + hq * 16 + li]);
            const float nref = mx > ref + kPaAbove ? mx - kPaBelow : ref;
            const float f = ref == -INFINITY ? 0.f : fast_exp2(ref - nref);
            if (th == 0 && lg == 0) s_f[hq * 16 + li] = f;
            ref = nref;
            sum *= f;
            sum_p *= f;
            numerators((t + 1) & 1);
          }
          lds_barrier();
#pragma unroll
          for (int ht = 0; ht < HGT; ++ht) {
            const float f = s_f[ht * 16 + li];
#pragma unroll
            for (int j = 0; j < NDW; ++j) acc[j][ht] *= f;
          }
        }
        if (scores) {
          sum += es;
          sum_p += eps;
          top = fmaxf(top, tmax);
        }
        buf = next;
      }
      ta = tb;
    }

    // ---- the run's output ----
    const int ln = fresh_lane(), li = ln & 15, lg = ln >> 4;
    {
      const float l = xgroup_sum(sum), lp = xgroup_sum(kLo ? sum : sum_p);
      if (scores && lg == 0) {
        s_l[th * HG + hq * 16 + li] = l;
        s_mx[th * HG + hq * 16 + li] = top;
        if (th == 0) s_f[hq * 16 + li] = kLo ? 0.f : lp;
      }
    }
    lds_barrier();
    const bool whole = t0 == 0 && t1 == nt;
    const int64_t slot0 =
        (((int64_t)worker * 2 + (first_segment ? 0 : 1)) * p.groups + rg) * p.group_rows;
    // the statistics, by the waves that hold a row's reference
    if (scores && th == 0 && lg == 0 && live) {
      const int h = hq * 16 + li;
      float l = s_l[h], m = s_mx[h];
      if constexpr (TW == 2) l += s_l[HG + h], m = fmaxf(m, s_mx[HG + h]);
      if (whole) {
        if (p.smax) {
          const int64_t o = (int64_t)b * p.rows + rr;
          const bool any = p.return_lse && l > 0.f;
          // [B, 1, S1, N1], the order of the rows
          p.smax[o] = any ? m * kLn2 : 0.f;
          p.ssum[o] = any ? l * fast_exp2(ref - m) : 0.f;
        }
      } else {
        p.part_ml[slot0 + h] = {ref, l, m, kLo ? l : s_f[h]};
      }
    }
#pragma unroll
    for (int ht = 0; ht < HGT; ++ht) {
      const int h = ht * 16 + li;
      const int64_t r = (int64_t)rg * HG + h;
      float l = s_l[h];
      if constexpr (TW == 2) l += s_l[HG + h];
      if constexpr (!kLo) l = s_f[h];
      const float inv = l > 0.f ? 1.f / l : 0.f;
      if (r >= p.rows) continue;
#pragma unroll
      for (int j = 0; j < NDW; ++j) {
        const int col = (wave * NDW + j) * 16 + lg * 4;
        if (whole) {
          const f32x4 x = acc[j][ht] * inv;
          const T4 o = {E::from_f32(x[0]), E::from_f32(x[1]), E::from_f32(x[2]), E::from_f32(x[3])};
          *(T4*)((T*)p.out + ((int64_t)b * p.rows + r) * D + col) = o;
        } else {
          *(f32x4*)(p.part_o + (slot0 + h) * D + col) = acc[j][ht];
        }
      }
    }
    first_segment = false;
    at = before + t1;
    if (t1 == nt) {
      before += nt;
      ++b;
    }
    lds_barrier();  // s_l, s_mx and s_f are read
  }
}

PagedShape paged_latent_shape(int64_t batch, int64_t s1, int64_t n1, int64_t d, int64_t max_blocks, int64_t page) {
  PagedShape s;
  s.tile = kPlTile;
  const int64_t rows = s1 * n1;
  s.group_rows = rows <= 16 ? 16 : (rows <= 32 ? 32 : (rows <= 64 ? 64 : 128));
  s.row_groups = (int)((rows + s.group_rows - 1) / s.group_rows);
  s.groups = s.row_groups;
  s.min_tiles = 8;
  s.workers = paged_workers(device_cu_count(), s.groups, batch * ((max_blocks * page + s.tile - 1) / s.tile),
                            s.min_tiles);
  return s;
}

template <int D, typename T>
static void paged_latent_hg(const PagedAttnParams& p, unsigned grid, hipStream_t stream) {
  if (p.group_rows == 16) paged_latent_kernel<D, T, 16><<<grid, kPlThreads, 0, stream>>>(p);
  else if (p.group_rows == 32) paged_latent_kernel<D, T, 32><<<grid, kPlThreads, 0, stream>>>(p);
  else if (p.group_rows == 64) paged_latent_kernel<D, T, 64><<<grid, kPlThreads, 0, stream>>>(p);
  else paged_latent_kernel<D, T, 128><<<grid, kPlThreads, 0, stream>>>(p);
}

template <typename T>
static void paged_latent_d(const PagedAttnParams& p, int64_t d, unsigned grid, hipStream_t stream) {
  if (d == 128) paged_latent_hg<128, T>(p, grid, stream);
  else if (d == 256) paged_latent_hg<256, T>(p, grid, stream);
  else paged_latent_hg<512, T>(p, grid, stream);
}

int paged_latent_launch(const PagedAttnParams& p, int64_t d, int32_t dtype, hipStream_t stream) {
  const unsigned grid = (unsigned)(8ll * ((p.workers + 7) / 8) * p.row_groups);
  if (dtype == DSA_DTYPE_BF16) paged_latent_d<bf16>(p, d, grid, stream);
  else paged_latent_d<f16>(p, d, grid, stream);
  DSA_HIP(hipGetLastError());
  return DSA_OK;
}

}  // namespace dsa
