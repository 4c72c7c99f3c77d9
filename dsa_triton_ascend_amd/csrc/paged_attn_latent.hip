// Attention of the newest tokens over a paged latent cache (described in
// paged_attn.h): one key head of D + 64 columns, its first D the value too.
//
//   S^T = K Q^T,  P = 2^(S - ref),  O^T = V^T P^T,  V = K[:, :D]
//
// A token of 576 columns is 1152 bytes and 2176 flops a row.  Up to 32 rows
// the bytes bound it (16 heads, 32 x 32K tokens, 1.2 GB: 191 us, 6.3 TB/s in
// all and 7.4 TB/s between 16K and 32K); at 64 rows bytes and LDS reads are
// near each other (238 us); at 128 it is the LDS reads: 416 KB a tile of 32
// tokens (288 of them K, which each of eight waves reads for its 16 rows),
// 3250 of a tile's 5400 cycles, beside 2180 of MFMAs (360 us with the join of
// 14, 0.81 PFLOP/s, 44 % of the matrix pipes' cycles).
//
// One workgroup of eight waves per CU owns a run of tokens for HG rows; a
// token is read from memory once and serves both products and every row
// (head, new token) of the workgroup.
//  * Tiles of 32 tokens come by LDS-DMA into a ring of four (of three at 128
//    rows of 512 columns), 16-byte chunks swizzled so that both products read
//    them without bank conflicts.  Up to 64 rows the four waves without scores
//    fetch; at 128 all do, a DMA between every few score MFMAs.
//  * S^T: wave w < HG / 16 takes 16 rows and all 32 tokens, so a row's softmax
//    stays in one wave.  Its Q stays in registers, but for four k-steps at 128
//    rows of 512 columns, where the output takes half of the registers.
//  * P goes through LDS, 64 bytes per row: token 16 tt + 4 g + r in slot
//    8 g + 4 tt + r, chunk g at g ^ (row / 4 % 4).
//  * O^T: a wave owns D / 8 columns of all HG rows, so each V^T fragment is
//    read by one wave (transposed on its way out of the LDS) and serves all
//    rows.
//  * A step computes the scores of tile t + 1, then the output of tile t with
//    the softmax of tile t + 1 between its MFMAs; P has two buffers and a step
//    one barrier.
// A row's reference (paged_attn.h) is moved by the wave that owns the row: it
// leaves the factor in LDS and raises its bit of the tile's flags, and every
// wave scales that row's output before it multiplies the tile.  That happens on
// a run's first tile and seldom after it.
//
// Up to 32 rows P is multiplied as a sum of two values of the input type,
// which is free where the bytes bound.  With more rows the MFMAs and LDS reads
// of the second value are not (at 128 rows of 512 columns the LDS has no room
// for it either), so P is rounded once there, at any number of tokens, and the
// output is divided by the sum of the rounded values, so that the weights still
// add up to one.  What is left is the rounding of single weights: an output is
// off by up to eps sum w |v|, and for values that vary from token to token by
// about half of its own rounding.  Error against 64 bits over the output, both
// 2-norms, with P as two values and rounded: bf16 1.66e-3 and 1.73e-3 over 32K
// tokens, 1.66e-3 and 1.90e-3 over 60 to 1000, 1.66e-3 and 1.70e-3 over two;
// fp16 2.07e-4 and 2.17e-4, 2.38e-4, 2.13e-4.
#include "paged_prefix.h"
#include "sfa_fwd.h"

namespace dsa {

__device__ __attribute__((aligned(16))) unsigned char g_latent_zero_row[1024];

constexpr int kPlTile = 32;

// The LDS-DMAs of sfa_fwd.h, and the same with loads that keep nothing in
// the caches.
template <bool STREAM>
__device__ __forceinline__ void pl_dma_buf(unsigned lds_base, int voff, __amdgpu_buffer_rsrc_t rsrc) {
  if constexpr (STREAM)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen nt lds"
                 :: "s"(lds_base), "v"(voff), "s"(rsrc) : "memory");
  else dma_buf16(lds_base, voff, rsrc);
}
template <bool STREAM>
__device__ __forceinline__ void pl_dma_glb(unsigned lds_base, const void* gaddr) {
  if constexpr (STREAM)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off nt"
                 :: "s"(lds_base), "v"(gaddr) : "memory");
  else dma_glb16(lds_base, gaddr);
}
constexpr int kPlThreads = 512;
constexpr int kPlPages = 512;  // block-table entries held in LDS

template <int D, typename T, int HG, bool STREAM, typename P>
__global__ __launch_bounds__(kPlThreads, 1) void paged_latent_kernel(P p) {
  using E = Elem<T>;
  using V8 = typename E::v8;
  typedef T T4 __attribute__((ext_vector_type(4)));
  constexpr int NW = kPlThreads / 64;
  constexpr int HW = HG / 16;            // waves that compute scores, 16 rows each
  constexpr int NTT = 2;                 // 16-token sub-tiles
  constexpr bool kLo = HG <= 32;         // P as two values
  constexpr int NPB = kLo ? 2 : 1;
  constexpr int DR = 64;
  constexpr int KS = (D + DR) / 32, KSN = D / 32;
  constexpr int NDW = D / NW / 16;       // output column tiles of a wave
  constexpr int TILE = kPlTile;
  constexpr int NOPE_BYTES = TILE * D * 2;
  constexpr int BUF_BYTES = NOPE_BYTES + TILE * DR * 2;
  // at 128 rows of 512 columns the output takes half of the registers and Q
  // would take most of the rest: QL k-steps of it are kept in LDS, in the
  // place of a ring buffer
  constexpr int QL = HG == 128 && D == 512 ? 4 : 0;
  constexpr int KQR = KS - QL;
  constexpr int NBUF = QL ? 3 : 4, RBUF = 3;  // ring buffers: a tile's rope rows serve the scores only
  constexpr int CPT = D / 8;             // 16-byte chunks of a token
  constexpr int TPI = 64 / CPT;          // tokens of one DMA
  // waves that fetch: those without scores, where four are
  constexpr int NL = HW <= 4 ? 4 : 8;
  constexpr int NIW = TILE / TPI / NL;   // DMAs of a fetching wave per tile; four waves one more for rope rows
  constexpr int ROPE0 = NBUF * NOPE_BYTES;
  constexpr int PROW = TILE * 2;
  static_assert(HW <= NW && NIW * TPI * NL == TILE && NDW * 16 * NW == D, "tile split");
  // a token's row of buffer b; buffers alternate per DMA
  auto nope_off = [](int tk, int b) { return ((tk / TPI) * NBUF + b) * 1024 + (tk % TPI) * (D * 2); };
  auto rope_off = [](int tk, int b) { return ROPE0 + ((tk >> 3) * RBUF + b) * 1024 + (tk & 7) * (DR * 2); };

  __shared__ __attribute__((aligned(16))) unsigned char smem[NBUF * NOPE_BYTES + RBUF * TILE * DR * 2];
  __shared__ __attribute__((aligned(16))) unsigned char s_p[2 * NPB * HG * PROW];
  __shared__ __attribute__((aligned(16))) unsigned char s_q[QL ? HG * QL * 64 : 16];
  __shared__ int s_tab[kPlPages];
  __shared__ float s_f[2 * HG];  // by a tile's parity: factors of the rows whose reference moved
  __shared__ int s_flag[3];  // by a tile's number modulo 3: bits of the waves whose rows moved
  float* const s_n = (float*)s_p;  // of a finished run, in place of P: the rows' divisors

  const int tid = threadIdx.x, lane = tid & 63;
  const int li = lane & 15, lg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const bool scores = wave < HW;
  const bool fetches = NL == NW || wave >= NW - NL;
  const int lw = wave - (NW - NL);  // among the fetching waves
  const bool rope_wave = lw >= 0 && lw < 4;

  if constexpr (kPrefixed<P>) {
    // the last workgroup plans the work on the prefixes
    if (blockIdx.x == gridDim.x - 1) {
      if (wave == 0) prefix_plan(p, TILE, lane);
      return;
    }
  }
  // the row groups of a worker read the same tokens: they share an XCD
  const int jj = blockIdx.x >> 3;
  const int rg = jj % p.row_groups;
  const int worker = (jj / p.row_groups) * 8 + (blockIdx.x & 7);
  if (worker >= p.workers) return;
  PagedPlan<P> plan;
  plan.make(p, TILE, lane);
  if (worker >= (plan.total + plan.per - 1) / plan.per) return;
  int at = worker * plan.per;
  const int end = min(at + plan.per, plan.total);
  int before;
  int b = plan.find(p, TILE, lane, at, &before);

  // scores in log2 units are s * scale - ref, one operation each; for that
  // the scale is positive: Q takes its sign, and is zero where it is
  const float scale = p.scale_log2 == 0.f ? 1.f : fabsf(p.scale_log2);
  const unsigned flip = p.scale_log2 < 0.f ? 0x80008000u : 0u, keep = p.scale_log2 == 0.f ? 0u : ~0u;
  const unsigned smem_base = (unsigned)(uintptr_t)smem;
  const unsigned char* const kbase = (const unsigned char*)p.k;
  const unsigned char* const rbase = (const unsigned char*)p.kr;
  // a lane's addresses in the two products are made anew from its number in
  // every step: kept, they would push Q or the output out of the registers
  auto fresh_lane = []() {
    int ln = __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0u));
    asm volatile("" : "+v"(ln));
    return ln;
  };
  constexpr int G1_TT = ((16 / TPI) * NBUF) * 1024;
  constexpr int G1R_TT = 2 * RBUF * 1024;
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
  using Off = std::integral_constant<bool, false>;

  bool first_segment = true;
  // (what the plan keeps of the sequences does not stay in the registers
  // through the tiles: later ones are read again)
  b = __builtin_amdgcn_readfirstlane(b);
  PagedSeqOf<P> seq = plan.sequence(p, b);
  while (at < end) {
    const int ln = fresh_lane(), li = ln & 15, lg = ln >> 4, tid = wave * 64 + ln;
    const int nt = paged_tiles(seq, TILE);
    if (nt == 0) {
      if (++b >= p.batch) break;
      seq = paged_seq_uniform(p, b);
      continue;
    }
    const int t0 = at - before, t1 = min(end - before, nt);
    const int tok0 = seq.lo + t0 * TILE, tok1 = min(seq.hi, seq.lo + t1 * TILE);
    const int32_t *tab = p.table + (int64_t)b * p.max_blocks, *lead = tab;
    if constexpr (kPrefixed<P>)
      if (__any(seq.given)) {
        lead = p.table + (int64_t)paged_leader(p, b, ln) * p.max_blocks;
        seq.given = paged_given(p, seq.given, tab, lead);
      }

    // the run's pages, as many as the LDS holds at a time, a thread's each
    int ta = tok0, tb, pg0, page_entry;
    auto read_pages = [&]() {
      unsigned off0;
      pg0 = (int)paged_split(p, (unsigned)ta, &off0);
      tb = (int)min((int64_t)tok1, (int64_t)(pg0 + kPlPages) * p.page);
      const int32_t* from = tab;
      if constexpr (kPrefixed<P>)
        if (ta < seq.given) from = lead, tb = min(tb, seq.given);
      const int npg = (int)paged_split(p, (unsigned)tb - 1u, &off0) - pg0 + 1;
      page_entry = tid < npg ? from[pg0 + tid] : 0;
    };
    read_pages();

    // rows of the wave's scores: head rr % n1 of new token rr / n1 (those
    // that do not exist compute something, which is not stored).  Tokens that
    // all of them see need no mask; a row's bounds rise with its token.
    int all_lo = 0, all_hi = 0x7fffffff;
    const int first_row = rg * HG + wave * 16;
    if (scores && first_row < p.rows) {
      int l, h;
      const int s_first = p.s1 == 1 ? 0 : first_row / p.n1;
      const int s_last = p.s1 == 1 ? 0 : min(first_row + 15, p.rows - 1) / p.n1;
      paged_bounds(p, seq.act_q, seq.act_k, s_last, &all_lo, &h);
      paged_bounds(p, seq.act_q, seq.act_k, s_first, &l, &all_hi);
      all_lo = __builtin_amdgcn_readfirstlane(all_lo);
      all_hi = __builtin_amdgcn_readfirstlane(min(all_hi, h));
    }
    V8 qf[KQR];
    u32x4 ql_in[QL ? QL : 1];
    {
      // (bounds in the descriptors: rows that do not exist read zeros)
      const int rows_here = min(p.rows - rg * HG, HG);
      const int64_t row0 = (int64_t)b * p.rows + rg * HG;
      const __amdgpu_buffer_rsrc_t q_src =
          __builtin_amdgcn_make_buffer_rsrc((void*)((const T*)p.q + row0 * D), (short)0, rows_here * D * 2, 0x00020000);
      const __amdgpu_buffer_rsrc_t qr_src = __builtin_amdgcn_make_buffer_rsrc(
          (void*)((const T*)p.qr + row0 * DR), (short)0, rows_here * DR * 2, 0x00020000);
      const int r = wave * 16 + li;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        // (the empty asm gives waves without scores something in these registers:
        // left undefined, they cost 60 spilled ones)
        u32x4 x;
        asm volatile("" : "=v"(x));
        if (NL == NW || scores)
          x = ks < KSN ? __builtin_amdgcn_raw_buffer_load_b128(q_src, r * (D * 2) + lg * 16 + ks * 64, 0, 0)
                       : __builtin_amdgcn_raw_buffer_load_b128(qr_src, r * (DR * 2) + lg * 16 + (ks - KSN) * 64, 0, 0);
        if (ks < KQR) qf[ks < KQR ? ks : 0] = as_v8<V8>(x);
        else ql_in[ks < KQR ? 0 : ks - KQR] = x;
      }
      __builtin_amdgcn_sched_barrier(0);  // all on their way before the first is waited for
    }
    f32x4 acc[NDW][HW];
#pragma unroll
    for (int j = 0; j < NDW; ++j)
#pragma unroll
      for (int ht = 0; ht < HW; ++ht) acc[j][ht] = {0.f, 0.f, 0.f, 0.f};
    float ref = -INFINITY, top = -INFINITY, sum = 0.f, sum_p = 0.f;

    auto share_pages = [&]() {
      lds_barrier();  // the pages, tiles and numerators before are read
      if (tid < 3) s_flag[tid] = 0;
      s_tab[tid] = page_entry;
      lds_barrier();
    };
    share_pages();
    // Q's loads, on their way beside the pages', end here and not inside the
    // tile loop, where a wait for them would be one for the tiles in flight too
    {
#pragma unroll
      for (int ks = 0; ks < KQR; ++ks) {
        qf[ks] = as_v8<V8>((__builtin_bit_cast(u32x4, qf[ks]) & keep) ^ flip);
        asm volatile("" : "+v"(qf[ks]));
      }
#pragma unroll
      for (int i = 0; i < QL; ++i)
        *(u32x4*)(s_q + (((wave * 16 + li) * (QL * 64) + ((lg ^ nope_swz(li)) * 16)) ^ (i << 6))) = (ql_in[i] & keep) ^ flip;
    }

    for (;;) {
      const int n_tiles = (tb - ta + TILE - 1) / TILE;
      // cache row of token lane % 32 of tile t, -1 past the end or without a
      // page (both are read as zeros)
      auto tile_rows = [&](int t) -> int {
        const int tok = ta + t * TILE + (fresh_lane() & 31);
        if (tok >= tb) return -1;
        unsigned off;
        const unsigned pg = paged_split(p, (unsigned)tok, &off);
        const int blk = s_tab[(int)pg - pg0];
        const int64_t r = (int64_t)blk * p.page + (int)off;
        return blk < 0 || r >= p.kv_rows ? -1 : (int)r;
      };
      // the wave's DMA j of a tile into buffers buf and rbuf
      auto dma = [&](int j, int rows, int buf, int rbuf) {
        const int ln = fresh_lane();
        if (j < NIW) {
          const unsigned dst = smem_base + nope_off((j * NL + lw) * TPI, buf);
          if constexpr (TPI == 1) {
            // one row: its address goes into the descriptor, of no bytes
            // where there is no row
            const int r = __builtin_amdgcn_readlane(rows, j * NL + lw);
            const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc(
                (void*)(kbase + (int64_t)(r < 0 ? 0 : r) * (D * 2)), (short)0, r < 0 ? 0 : D * 2, 0x00020000);
            pl_dma_buf<STREAM>(dst, (ln ^ nope_swz(j * NL + lw)) * 16, rsrc);
          } else {
            const int tk = (j * NL + lw) * TPI + ((unsigned)ln / CPT);
            const int ch = ((unsigned)ln % CPT) ^ nope_swz(tk);
            const int r = __shfl(rows, tk);
            pl_dma_glb<STREAM>(dst, r >= 0 ? kbase + (int64_t)r * (D * 2) + ch * 16 : g_latent_zero_row + ch * 16);
          }
        } else if (rope_wave) {
          const int tk = lw * 8 + (ln >> 3);
          const int ch = (ln & 7) ^ rope_swz(tk);
          const int r = __shfl(rows, tk);
          pl_dma_glb<STREAM>(smem_base + rope_off(lw * 8, rbuf),
                    r >= 0 ? rbase + (int64_t)r * (DR * 2) + ch * 16 : g_latent_zero_row + ch * 16);
        }
      };

      // all but the last K tiles that this wave asked for have landed
      auto landed = [&](auto k) {
        constexpr int K = decltype(k)::value;
        if (rope_wave) wait_vmcnt<K * (NIW + 1)>();
        else wait_vmcnt<K * NIW>();
      };

      // ---- scores of a tile, with the DMAs of another between the MFMAs ----
      f32x4 s[NTT] = {};  // (these are set to something so that they do not stay alive from run to run)
      V8 va[NDW];
      auto read_v = [&](int buf) {
        const int ln = fresh_lane(), l = ln & 15, g = ln >> 4;
        const int r1 = g * 4 + (l >> 2);
        const int g2b = nope_off(r1, 0) + ((((l & 3) >> 1) ^ nope_swz(r1)) * 16) + (l & 1) * 8 + buf * 1024;
#pragma unroll
        for (int j = 0; j < NDW; ++j) va[j] = a2(g2b, wave * NDW + j);
      };
      auto gemm1 = [&](int kbuf, int krbuf, auto with_dma, int rows, int dbuf, int drbuf) {
        constexpr int PF = QL ? 2 : HG <= 32 && KS >= 8 ? 8 : 4;  // k-steps read ahead
        const int ln = fresh_lane(), l = ln & 15, g = ln >> 4;
        const int g1b = nope_off(l, 0) + ((g ^ nope_swz(l)) * 16) + kbuf * 1024;
        const int g1rb = rope_off(l, 0) + ((g ^ rope_swz(l)) * 16) + krbuf * 1024;
        const int qb = ((wave * 16 + l) * (QL * 64)) + ((g ^ nope_swz(l)) * 16);
        V8 fa[PF][NTT], ql[2];  // Q of a k-step in LDS is read two ahead
#pragma unroll
        for (int i = 0; i < PF; ++i)
#pragma unroll
          for (int u = 0; u < NTT; ++u) fa[i][u] = a1(g1b, g1rb, i, u);
#pragma unroll
        for (int u = 0; u < NTT; ++u) s[u] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          V8 f[NTT];
#pragma unroll
          for (int u = 0; u < NTT; ++u) {
            f[u] = fa[ks % PF][u];
            if (ks + PF < KS) fa[ks % PF][u] = a1(g1b, g1rb, ks + PF, u);
          }
          const V8 q = ks < KQR ? qf[ks < KQR ? ks : 0] : ql[ks & 1];
          if (QL > 0 && ks + 2 >= KQR && ks + 2 < KS)
            ql[ks & 1] = as_v8<V8>(*(const u32x4*)(s_q + (qb ^ ((ks + 2 - KQR) << 6))));
#pragma unroll
          for (int u = 0; u < NTT; ++u) s[u] = E::mfma(f[u], q, s[u]);
          if constexpr (decltype(with_dma)::value) {
            constexpr int kStep = KS / (NIW + 1);
            if (ks % kStep == 0 && ks / kStep <= NIW) dma(ks / kStep, rows, dbuf, drbuf);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      };

      // ---- softmax of the scores in eight stages, which go between the
      // groups of output MFMAs ----
      float es = 0.f, eps = 0.f;
      T4 ph[NTT] = {}, pl[NTT] = {};
      auto stage = [&](int k, int t, int flag) {
        if (k == 0) {
          const int tk = ta + t * TILE;
          if (tk < all_lo || tk + TILE > min(all_hi, tb)) {
            const int ln = fresh_lane();
            int lo, hi;
            const int r = min(rg * HG + wave * 16 + (ln & 15), p.rows - 1);
            paged_bounds(p, seq.act_q, seq.act_k, r / p.n1, &lo, &hi);
            hi = min(hi, tb);
#pragma unroll
            for (int i = 0; i < NTT * 4; ++i) {
              const int tok = tk + (i >> 2) * 16 + (ln >> 4) * 4 + (i & 3);
              s[i >> 2][i & 3] = tok >= lo && tok < hi ? s[i >> 2][i & 3] : -INFINITY;
            }
          }
        } else if (k == 1) {
          float m = s[0][0];
#pragma unroll
          for (int i = 1; i < NTT * 4; ++i) m = fmaxf(m, s[i >> 2][i & 3]);
          const float tmax = xgroup_max(m) * scale;
          top = fmaxf(top, tmax);
          es = eps = 0.f;
          const bool moves = tmax > ref + kPaAbove;
          if (__any(moves)) {
            // new references; whoever multiplies this tile's numerators
            // first scales these rows of its output
            const int ln = fresh_lane();
            const float nref = moves ? tmax - kPaBelow : ref;
            const float f = ref == -INFINITY ? 0.f : fast_exp2(ref - nref);
            ref = nref;
            sum *= f;
            sum_p *= f;
            if (ln < 16) s_f[(t & 1) * HG + wave * 16 + ln] = f;
            if (ln == 0) atomicOr(&s_flag[flag], 1 << wave);
          }
        } else if (k < 6) {
          // a quarter of the numerators
          const float from = ref == -INFINITY ? 0.f : ref;
#pragma unroll
          for (int i = (k - 2) * NTT; i < (k - 1) * NTT; ++i) {
            const float e = fast_exp2(__builtin_fmaf(s[i >> 2][i & 3], scale, -from));
            es += e;
            ph[i >> 2][i & 3] = E::from_f32(e);
            if constexpr (kLo) pl[i >> 2][i & 3] = E::from_f32(e - E::to_f32(ph[i >> 2][i & 3]));
            else eps += E::to_f32(ph[i >> 2][i & 3]);
          }
        } else if (k == 6) {
          sum += es;
          sum_p += eps;
        } else {
          const int ln = fresh_lane(), l = ln & 15, g = ln >> 4;
          unsigned char* dst = s_p + (t & 1) * (NPB * HG * PROW) + (wave * 16 + l) * PROW + ((g ^ ((l >> 2) & 3)) * 16);
#pragma unroll
          for (int u = 0; u < NTT; ++u) {
            *(T4*)(dst + u * 8) = ph[u];
            if constexpr (kLo) *(T4*)(dst + HG * PROW + u * 8) = pl[u];
          }
        }
      };

      // ---- output of tile t (V^T fragments in va), with the softmax of tile
      // t + 1 between the MFMAs ----
      auto gemm2 = [&](int t, int flag) {
        const int ln = fresh_lane(), l = ln & 15, g = ln >> 4;
        const unsigned char* src = s_p + (t & 1) * (NPB * HG * PROW) + l * PROW + ((g ^ ((l >> 2) & 3)) * 16);
        auto read = [&](int ht, int part) {
          return as_v8<V8>(*(const u32x4*)(src + part * HG * PROW + ht * 16 * PROW));
        };
        V8 nh = read(0, 0), nl = kLo ? read(0, 1) : nh;
#pragma unroll
        for (int ht = 0; ht < HW; ++ht) {
          const V8 bh = nh, bl = nl;
          if (ht + 1 < HW) {
            nh = read(ht + 1, 0);
            if constexpr (kLo) nl = read(ht + 1, 1);
          }
#pragma unroll
          for (int j = 0; j < NDW; ++j) acc[j][ht] = E::mfma(va[j], bh, acc[j][ht]);
          if constexpr (kLo) {
#pragma unroll
            for (int j = 0; j < NDW; ++j) acc[j][ht] = E::mfma(va[j], bl, acc[j][ht]);
          }
          if (scores) {
#pragma unroll
            for (int k = ht * 8 / HW; k < (ht + 1) * 8 / HW; ++k) stage(k, t + 1, flag);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      };

      // the first tiles (those past the end, here and below, read zeros, so
      // that the number of DMAs in flight is known)
      if (fetches) {
#pragma unroll
        for (int t = 0; t < NBUF - 1; ++t) {
          const int rows = tile_rows(t);
#pragma unroll
          for (int j = 0; j <= NIW; ++j) dma(j, rows, t, t);
        }
      }
      landed(std::integral_constant<int, NBUF - 2>{});
      lds_barrier();
      if (scores) {
        gemm1(0, 0, Off{}, 0, 0, 0);
#pragma unroll
        for (int k = 0; k < 8; ++k) stage(k, 0, 0);
      }
      landed(std::integral_constant<int, NBUF - 3>{});
      lds_barrier();
      // step t: scores of tile t + 1 (of no visible token after the last),
      // output of tile t, DMAs of tile t + NBUF - 1
      int buf = 0, rbuf = 0;  // buffers and flags of tile t
      for (int t = 0; t < n_tiles; ++t) {
        const int next = buf + 1 == NBUF ? 0 : buf + 1;
        const int rnext = rbuf + 1 == RBUF ? 0 : rbuf + 1;
        const int rlast = rnext + 1 == RBUF ? 0 : rnext + 1;  // of tile t + 2, and of tile t - 1
        const int dbuf = buf == 0 ? NBUF - 1 : buf - 1, drbuf = NBUF == 3 ? rlast : rbuf;
        const int moved_v = s_flag[rbuf];
        // flags of tile t + 2, last read a step ago
        if (tid == 0) s_flag[rlast] = 0;
        const int rows = fetches ? tile_rows(t + NBUF - 1) : -1;
        if (NL < NW && fetches) {
#pragma unroll
          for (int j = 0; j <= NIW; ++j) dma(j, rows, dbuf, drbuf);
        }
        if (scores) gemm1(next, rnext, std::integral_constant<bool, NL == NW>{}, rows, dbuf, drbuf);
        read_v(buf);
        const int moved = __builtin_amdgcn_readfirstlane(moved_v);
        if (moved) {
          const int l = fresh_lane() & 15;
#pragma unroll
          for (int w = 0; w < HW; ++w)
            if (moved >> w & 1) {
              const float f = s_f[(t & 1) * HG + w * 16 + l];
#pragma unroll
              for (int j = 0; j < NDW; ++j) acc[j][w] *= f;
            }
        }
        gemm2(t, rnext);
        landed(std::integral_constant<int, NBUF - 3>{});  // tile t + 2 has
        lds_barrier();
        buf = next;
        rbuf = rnext;
      }
      wait_vmcnt<0>();  // of the DMAs past the end too: the ring is theirs until then
      ta = tb;
      if (ta >= tok1) break;
      read_pages();
      share_pages();
    }

    // ---- the run's output ----
    // (a scope of its own: the lane's numbers are made anew here)
    [&](int ln) __attribute__((always_inline)) {
    const int li = ln & 15, lg = ln >> 4;
    const bool all = t0 == 0 && t1 == nt, whole = all && !paged_behind(seq);
    int64_t slot0 =
        (((int64_t)worker * 2 + (first_segment ? 0 : 1)) * p.groups + rg) * p.group_rows;
    if constexpr (kPrefixed<P>) slot0 = all ? paged_whole_slot(p, b, rg) : slot0;
    {
      const float l = xgroup_sum(sum), n = xgroup_sum(kLo ? sum : sum_p);
      const int r = wave * 16 + li, rr = rg * HG + r;
      if (scores && lg == 0) {
        s_n[r] = n;
        if (rr < p.rows) {
          if (!whole) {
            p.part_ml[slot0 + r] = {ref, l, top, n};
          } else if (p.smax) {
            const int64_t o = (int64_t)b * p.rows + rr;  // [B, 1, S1, N1], the order of the rows
            const bool any = p.return_lse && l != 0.f;
            p.smax[o] = any ? top * kLn2 : 0.f;
            p.ssum[o] = any ? l * fast_exp2(ref - top) : 0.f;
          }
        }
      }
    }
    lds_barrier();
    // By columns, as the waves hold it, the output would leave in pieces of
    // 32 bytes (9 to 19 thousand cycles at 128 rows of 512; a tile is 5): it goes through
    // the ring, which is free by now, and leaves as whole rows, which follow
    // each other in memory.
    auto put = [&](auto zero, void* to, auto value) {
      using O = decltype(zero);
      typedef O O4 __attribute__((ext_vector_type(4)));
      constexpr int ROW = D * (int)sizeof(O), PITCH = ROW + 16;  // (16 rows' chunks lie in 64 different banks)
      constexpr int FIT = 64 * PITCH <= (int)sizeof(smem) ? 64 : 32;
      constexpr int RP = HG < FIT ? HG : FIT;                    // rows of a pass
      constexpr int CHUNKS = RP * ROW / 16;
      static_assert(RP * PITCH <= (int)sizeof(smem), "output stage");
      const int col = (wave * NDW * 16 + lg * 4) * (int)sizeof(O);
#pragma unroll
      for (int h0 = 0; h0 < HW; h0 += RP / 16) {
        if (h0) lds_barrier();
#pragma unroll
        for (int h = 0; h < RP / 16; ++h)
#pragma unroll
          for (int j = 0; j < NDW; ++j) {
            const f32x4 x = value(h0 + h, j);
            *(O4*)(smem + (h * 16 + li) * PITCH + col + j * 16 * (int)sizeof(O)) =
                __builtin_convertvector(x, O4);
          }
        lds_barrier();
        const int bytes = min(p.rows - rg * HG - h0 * 16, RP) * ROW;  // (not positive without rows)
        unsigned char* const dst = (unsigned char*)to + h0 * 16 * ROW;
#pragma unroll
        for (int i = 0; i < (CHUNKS + kPlThreads - 1) / kPlThreads; ++i) {
          const int c = i * kPlThreads + wave * 64 + ln;
          if (c * 16 < bytes) *(u32x4*)(dst + c * 16) = *(const u32x4*)(smem + c * 16 / ROW * PITCH + c * 16 % ROW);
        }
      }
    };
    // rows that saw no token of the run: their output is zero, also where
    // another row's value beside it was not finite
    float n_row[HW];
    bool none = false;
#pragma unroll
    for (int ht = 0; ht < HW; ++ht) {
      n_row[ht] = s_n[ht * 16 + li];
      none |= n_row[ht] == 0.f;
    }
    if (__any(none)) {
#pragma unroll
      for (int ht = 0; ht < HW; ++ht)
#pragma unroll
        for (int j = 0; j < NDW; ++j)
          if (n_row[ht] == 0.f) acc[j][ht] = {0.f, 0.f, 0.f, 0.f};
    }
    if (whole) {
      float inv[HW];
#pragma unroll
      for (int ht = 0; ht < HW; ++ht) {
        inv[ht] = n_row[ht] != 0.f ? 1.f / n_row[ht] : 0.f;
      }
      put(T{}, (T*)p.out + ((int64_t)b * p.rows + rg * HG) * D, [&](int ht, int j) { return acc[j][ht] * inv[ht]; });
    } else {
      put(0.f, p.part_o + slot0 * D, [&](int ht, int j) { return acc[j][ht]; });
    }
    }(fresh_lane());
    first_segment = false;
    at = before + t1;
    if (t1 == nt) {
      at = before += plan.padded(nt);
      if (at < end) seq = paged_seq_uniform(p, ++b);
    }
  }
}

PagedShape paged_latent_shape(int64_t batch, int64_t s1, int64_t n1, int64_t d, int64_t max_blocks, int64_t page) {
  PagedShape s;
  s.tile = kPlTile;
  const int64_t rows = s1 * n1;
  s.group_rows = rows <= 16 ? 16 : (rows <= 32 ? 32 : (rows <= 64 ? 64 : 128));
  s.row_groups = (int)((rows + s.group_rows - 1) / s.group_rows);
  s.groups = s.row_groups;
  s.min_tiles = kPaMinTiles;
  s.workers = paged_workers(device_cu_count(), s.groups, batch, (max_blocks * page + s.tile - 1) / s.tile,
                            s.min_tiles);
  return s;
}

template <int D, typename T, bool STREAM, typename P>
static void paged_latent_hg(const P& p, unsigned grid, hipStream_t stream) {
  if (p.group_rows == 16) paged_latent_kernel<D, T, 16, STREAM><<<grid, kPlThreads, 0, stream>>>(p);
  else if (p.group_rows == 32) paged_latent_kernel<D, T, 32, STREAM><<<grid, kPlThreads, 0, stream>>>(p);
  else if (p.group_rows == 64) paged_latent_kernel<D, T, 64, STREAM><<<grid, kPlThreads, 0, stream>>>(p);
  else paged_latent_kernel<D, T, 128, STREAM><<<grid, kPlThreads, 0, stream>>>(p);
}

template <typename T, typename P>
static void paged_latent_d(const P& p, int64_t d, unsigned grid, hipStream_t stream) {
  // rows that the caches cannot hold until the next call, read by one row
  // group only, are not kept there (512 columns; 1.2 GB at 16 heads: 222 us,
  // streaming 192; 300 MB at 32 rows: 85 and 79; 75 MB at 16: 28 and 29)
  const int64_t tokens = p.kv_rows < (int64_t)p.batch * p.max_blocks * p.page
                             ? p.kv_rows : (int64_t)p.batch * p.max_blocks * p.page;
  const bool streaming = p.row_groups == 1 && tokens * (d + 64) * 2 > (256ll << 20);
  if (d == 128) paged_latent_hg<128, T, false>(p, grid, stream);
  else if (d == 256) paged_latent_hg<256, T, false>(p, grid, stream);
  else if (streaming) paged_latent_hg<512, T, true>(p, grid, stream);
  else paged_latent_hg<512, T, false>(p, grid, stream);
}

static int64_t paged_latent_grid(int64_t workers, int64_t row_groups) { return 8 * ((workers + 7) / 8) * row_groups; }
bool paged_latent_launchable(int64_t workers, int64_t row_groups) {
  return launchable(paged_latent_grid(workers, row_groups), kPlThreads);
}

template <typename P>
static int paged_latent(const P& p, int64_t d, int32_t dtype, hipStream_t stream) {
  const unsigned grid = (unsigned)paged_latent_grid(p.workers, p.row_groups) + (kPrefixed<P> ? 1 : 0);
  if (dtype == DSA_DTYPE_BF16) paged_latent_d<bf16>(p, d, grid, stream);
  else paged_latent_d<f16>(p, d, grid, stream);
  DSA_HIP(hipGetLastError());
  return DSA_OK;
}

int paged_latent_launch(const PagedAttnParams& p, int64_t d, int32_t dtype, hipStream_t stream) {
  return paged_latent(p, d, dtype, stream);
}
int paged_latent_launch(const PagedPrefixParams& p, int64_t d, int32_t dtype, hipStream_t stream) {
  return paged_latent(p, d, dtype, stream);
}

}  // namespace dsa
