// Attention over a prefix that sequences share, latent cache (described in
// paged_prefix.h): one key head of D + 64 columns, its first D the value too.
//
//   S^T = K Q^T,  P = 2^(S - ref),  O^T = V^T P^T,  V = K[:, :D]
//
// At 16 heads a sequence alone has 2 * 1088 * 16 flops for the 1152 bytes of a
// token; the rows of eight sequences together are 128, whose products bound it,
// and beside them the LDS, from which each of eight waves reads all of K for its
// 16 rows.  The split of the work in a workgroup is that of paged_attn_latent.hip at 128 rows: wave w has the
// scores and the softmax of rows 16 w on, P goes through LDS, and each wave has
// D / 8 columns of all rows' outputs.  What is a row's sequence, new token and
// head, and what it sees, differs from row to row here.
//
// P is rounded once, and the output divided by the sum of the rounded values,
// as there at 128 rows (with up to 32 it keeps two values there; 2-norms of the
// error, bf16, 1.66e-3 with two and 1.75e-3 with one, of which 1.66e-3 is the
// output's own rounding).  Measured, 512 columns: 2.3 us for a tile of 32 tokens of
// every CU's 128 rows (0.9 PFLOP/s; the matrix pipes, the LDS and the vector units
// each work 33 to 36 % of the cycles of a launch of some 25 tiles: what is lost is
// overlap), and 20 us for the start and the 32-bit outputs of 256
// jobs (67 MB): 16 heads, 32 sequences behind 32768 tokens 56 us, with what is
// behind the prefix and the join 81 (each sequence for itself 162).
#include "paged_prefix.h"
#include "sfa_fwd.h"

namespace dsa {

__device__ __attribute__((aligned(16))) unsigned char g_prefix_latent_zero_row[1024];

constexpr int kPxThreads = 512;
constexpr int kPxPages = 256;  // block-table entries held in LDS

template <int D, typename T>
__global__ __launch_bounds__(kPxThreads, 1) void prefix_latent_kernel(PagedPrefixParams p) {
  using E = Elem<T>;
  using V8 = typename E::v8;
  typedef T T4 __attribute__((ext_vector_type(4)));
  constexpr int HG = kPrefixLatentRows;
  constexpr int NW = kPxThreads / 64;
  constexpr int HW = HG / 16;            // (a wave's scores are of 16 rows)
  constexpr int NTT = 2;                 // 16-token sub-tiles
  constexpr int DR = 64;
  constexpr int KS = (D + DR) / 32, KSN = D / 32;
  constexpr int NDW = D / NW / 16;       // output column tiles of a wave
  constexpr int TILE = kPrefixTile;
  constexpr int NOPE_BYTES = TILE * D * 2;
  constexpr int BUF_BYTES = NOPE_BYTES + TILE * DR * 2;
  // at 128 rows of 512 columns the output takes half of the registers and Q
  // would take most of the rest: QL k-steps of it are kept in LDS, in the
  // place of a ring buffer
  constexpr int QL = D == 512 ? 4 : 0;
  constexpr int KQR = KS - QL;
  constexpr int NBUF = QL ? 3 : 4, RBUF = 3;  // ring buffers: a tile's rope rows serve the scores only
  constexpr int CPT = D / 8;             // 16-byte chunks of a token
  constexpr int TPI = 64 / CPT;          // tokens of one DMA
  constexpr int NIW = TILE / TPI / NW;   // DMAs of a wave per tile; four waves one more for rope rows
  constexpr int ROPE0 = NBUF * NOPE_BYTES;
  constexpr int PROW = TILE * 2;
  static_assert(HW == NW && NIW * TPI * NW == TILE && NDW * 16 * NW == D, "tile split");
  // a token's row of buffer b; buffers alternate per DMA
  auto nope_off = [](int tk, int b) { return ((tk / TPI) * NBUF + b) * 1024 + (tk % TPI) * (D * 2); };
  auto rope_off = [](int tk, int b) { return ROPE0 + ((tk >> 3) * RBUF + b) * 1024 + (tk & 7) * (DR * 2); };

  __shared__ __attribute__((aligned(16))) unsigned char smem[NBUF * NOPE_BYTES + RBUF * TILE * DR * 2];
  __shared__ __attribute__((aligned(16))) unsigned char s_p[2 * HG * PROW];
  __shared__ __attribute__((aligned(16))) unsigned char s_q[QL ? HG * QL * 64 : 16];
  __shared__ int s_tab[kPxPages];
  __shared__ int s_lo[HG], s_hi[HG];
  __shared__ float s_f[2 * HG];  // by a tile's parity: factors of the rows whose reference moved
  __shared__ int s_flag[3];  // by a tile's number modulo 3: bits of the waves whose rows moved
  float* const s_n = (float*)s_p;  // of a finished run, in place of P: the rows' divisors

  const int tid = threadIdx.x, lane = tid & 63;
  const int li = lane & 15, lg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const bool rope_wave = wave < 4;

  int head;
  int job = prefix_job_of(p, blockIdx.x, gridDim.x, 0, &head);
  const int jobs = *p.n_jobs;

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

  for (int round = 0; job < jobs;) {
    const PagedJob jb = p.job[job];
    const int ln = fresh_lane(), li = ln & 15, lg = ln >> 4, tid = wave * 64 + ln;
    const int first = jb.first, n_rows = jb.rows, tok0 = jb.tok0, tok1 = jb.tok1;
    const int64_t slot0 = p.part0 + (int64_t)job * HG;
    const bool masked = tok0 < jb.all_lo || tok1 > jb.all_hi;
    if (masked) {  // what the rows see, where it is not all of it
      lds_barrier();  // (the job before has read what it left)
      for (int r = tid; r < n_rows; r += kPxThreads) prefix_bounds(p, jb, r, s_lo + r, s_hi + r);
    }
    {
      if (tok1 <= tok0) {  // none of the block's rows sees any of it
        for (int r = tid; r < n_rows; r += kPxThreads) p.part_ml[slot0 + r] = {-INFINITY, 0.f, -INFINITY, 0.f};
        for (int c = tid; c < n_rows * (D / 4); c += kPxThreads)
          *((f32x4*)(p.part_o + slot0 * D) + c) = f32x4{0.f, 0.f, 0.f, 0.f};
        job = prefix_job_of(p, blockIdx.x, gridDim.x, ++round, &head);
        continue;
      }
    }
    const int32_t* tab = p.table + (int64_t)jb.lead * p.max_blocks;

    // the run's pages, as many as the LDS holds at a time, a thread's each
    int ta = tok0, tb, pg0, page_entry;
    auto read_pages = [&]() {
      unsigned off0;
      pg0 = (int)paged_split(p, (unsigned)ta, &off0);
      tb = (int)min((int64_t)tok1, (int64_t)(pg0 + kPxPages) * p.page);
      const int npg = (int)paged_split(p, (unsigned)tb - 1u, &off0) - pg0 + 1;
      page_entry = tid < npg ? tab[pg0 + tid] : 0;
    };
    read_pages();

    V8 qf[KQR];
    u32x4 ql_in[QL ? QL : 1];
    {
      // (bounds in the descriptors: rows that do not exist read zeros)
      const int64_t row0 = (int64_t)first * p.rows + jb.row0;
      const __amdgpu_buffer_rsrc_t q_src =
          __builtin_amdgcn_make_buffer_rsrc((void*)((const T*)p.q + row0 * D), (short)0, n_rows * D * 2, 0x00020000);
      const __amdgpu_buffer_rsrc_t qr_src = __builtin_amdgcn_make_buffer_rsrc(
          (void*)((const T*)p.qr + row0 * DR), (short)0, n_rows * DR * 2, 0x00020000);
      const int r = wave * 16 + li;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const u32x4 x = ks < KSN
                            ? __builtin_amdgcn_raw_buffer_load_b128(q_src, r * (D * 2) + lg * 16 + ks * 64, 0, 0)
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
      if (tid < kPxPages) s_tab[tid] = page_entry;
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
          const unsigned dst = smem_base + nope_off((j * NW + wave) * TPI, buf);
          if constexpr (TPI == 1) {
            // one row: its address goes into the descriptor, of no bytes
            // where there is no row
            const int r = __builtin_amdgcn_readlane(rows, j * NW + wave);
            const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc(
                (void*)(kbase + (int64_t)(r < 0 ? 0 : r) * (D * 2)), (short)0, r < 0 ? 0 : D * 2, 0x00020000);
            dma_buf16(dst, (ln ^ nope_swz(j * NW + wave)) * 16, rsrc);
          } else {
            const int tk = (j * NW + wave) * TPI + ((unsigned)ln / CPT);
            const int ch = ((unsigned)ln % CPT) ^ nope_swz(tk);
            const int r = __shfl(rows, tk);
            dma_glb16(dst, r >= 0 ? kbase + (int64_t)r * (D * 2) + ch * 16 : g_prefix_latent_zero_row + ch * 16);
          }
        } else if (rope_wave) {
          const int tk = wave * 8 + (ln >> 3);
          const int ch = (ln & 7) ^ rope_swz(tk);
          const int r = __shfl(rows, tk);
          dma_glb16(smem_base + rope_off(wave * 8, rbuf),
                    r >= 0 ? rbase + (int64_t)r * (DR * 2) + ch * 16 : g_prefix_latent_zero_row + ch * 16);
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
        constexpr int PF = QL ? 2 : 4;  // k-steps read ahead
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
      T4 ph[NTT] = {};
      auto stage = [&](int k, int t, int flag) {
        if (k == 0) {
          const int tk = ta + t * TILE;
          if (masked || tk + TILE > tb) {
            const int ln = fresh_lane();
            const int r = min(wave * 16 + (ln & 15), n_rows - 1);
            const int lo = masked ? s_lo[r] : 0, hi = masked ? min(s_hi[r], tb) : tb;
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
            eps += E::to_f32(ph[i >> 2][i & 3]);
          }
        } else if (k == 6) {
          sum += es;
          sum_p += eps;
        } else {
          const int ln = fresh_lane(), l = ln & 15, g = ln >> 4;
          unsigned char* dst = s_p + (t & 1) * (HG * PROW) + (wave * 16 + l) * PROW + ((g ^ ((l >> 2) & 3)) * 16);
#pragma unroll
          for (int u = 0; u < NTT; ++u) *(T4*)(dst + u * 8) = ph[u];
        }
      };

      // ---- output of tile t (V^T fragments in va), with the softmax of tile
      // t + 1 between the MFMAs ----
      auto gemm2 = [&](int t, int flag) {
        const int ln = fresh_lane(), l = ln & 15, g = ln >> 4;
        const unsigned char* src = s_p + (t & 1) * (HG * PROW) + l * PROW + ((g ^ ((l >> 2) & 3)) * 16);
        auto read = [&](int ht) { return as_v8<V8>(*(const u32x4*)(src + ht * 16 * PROW)); };
        V8 nh = read(0);
#pragma unroll
        for (int ht = 0; ht < HW; ++ht) {
          const V8 bh = nh;
          if (ht + 1 < HW) nh = read(ht + 1);
#pragma unroll
          for (int j = 0; j < NDW; ++j) acc[j][ht] = E::mfma(va[j], bh, acc[j][ht]);
#pragma unroll
          for (int k = ht * 8 / HW; k < (ht + 1) * 8 / HW; ++k) stage(k, t + 1, flag);
          __builtin_amdgcn_sched_barrier(0);
        }
      };

      // the first tiles (those past the end, here and below, read zeros, so
      // that the number of DMAs in flight is known)
#pragma unroll
      for (int t = 0; t < NBUF - 1; ++t) {
        const int rows = tile_rows(t);
#pragma unroll
        for (int j = 0; j <= NIW; ++j) dma(j, rows, t, t);
      }
      landed(std::integral_constant<int, NBUF - 2>{});
      lds_barrier();
      gemm1(0, 0, Off{}, 0, 0, 0);
#pragma unroll
      for (int k = 0; k < 8; ++k) stage(k, 0, 0);
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
        const int rows = tile_rows(t + NBUF - 1);
        gemm1(next, rnext, std::integral_constant<bool, true>{}, rows, dbuf, drbuf);
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
    {
      const float l = xgroup_sum(sum), n = xgroup_sum(sum_p);
      const int r = wave * 16 + li;
      if (lg == 0) {
        s_n[r] = n;
        if (r < n_rows) p.part_ml[slot0 + r] = {ref, l, top, n};
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
        const int bytes = min(n_rows - h0 * 16, RP) * ROW;  // (not positive without rows)
        unsigned char* const dst = (unsigned char*)to + h0 * 16 * ROW;
#pragma unroll
        for (int i = 0; i < (CHUNKS + kPxThreads - 1) / kPxThreads; ++i) {
          const int c = i * kPxThreads + wave * 64 + ln;
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
    put(0.f, p.part_o + slot0 * D, [&](int ht, int j) { return acc[j][ht]; });
    }(fresh_lane());
    job = prefix_job_of(p, blockIdx.x, gridDim.x, ++round, &head);
  }
}

template <typename T>
static void prefix_latent_d(const PagedPrefixParams& p, int64_t d, unsigned grid, hipStream_t stream) {
  if (d == 128) prefix_latent_kernel<128, T><<<grid, kPxThreads, 0, stream>>>(p);
  else if (d == 256) prefix_latent_kernel<256, T><<<grid, kPxThreads, 0, stream>>>(p);
  else prefix_latent_kernel<512, T><<<grid, kPxThreads, 0, stream>>>(p);
}

int prefix_latent_launch(const PagedPrefixParams& p, int64_t d, int32_t dtype, unsigned grid, hipStream_t stream) {
  if (dtype == DSA_DTYPE_BF16) prefix_latent_d<bf16>(p, d, grid, stream);
  else prefix_latent_d<f16>(p, d, grid, stream);
  DSA_HIP(hipGetLastError());
  return DSA_OK;
}

}  // namespace dsa
