// Attention over a prefix that sequences share, grouped heads (described in
// paged_prefix.h), and the launches of the whole operator.
//
//   S^T = K Q^T,  P = 2^(S - ref),  O^T = V^T P^T
//
// A family of 32 sequences with eight query heads per key head has 256 rows a
// key head, and a token of the prefix serves them all: 256 flops per byte of K
// and V, so the matrix instructions bound it, and beside them the vector unit,
// which has a softmax weight to make for every 4 D flops.
//
// A workgroup has up to 16 NW MR rows: wave w the 16 MR from 16 MR w on, in MR
// tiles of 16.  K and V come in tiles of 32 tokens by LDS-DMA into a ring,
// chunks of 16 bytes swizzled so that both products read them without bank
// conflicts; every wave reads the whole tile, so the rows of a wave set what the
// LDS has to give (at 32 rows a wave 128 KB a tile of 128 columns, 512 cycles of
// a CU's LDS beside 1536 of its MFMAs).
// S^T leaves a token's weight where the second product wants it: token 16 tt +
// 4 g + r is k slot 8 g + 4 tt + r of lane group g, and V^T is read transposed
// in that order, so P stays in its lanes.
//
// A step computes the scores of tile t + 1 with the second half of the softmax
// of tile t between its MFMAs, then the output of tile t with the first half of
// that of tile t + 1.  One barrier a step.
//
// P is multiplied as a sum of two values of the input type, as paged_attn.hip has
// it: half as many matrix instructions again, and the error of a call does not
// depend on which way its sizes choose.  Rounded once the kernel took 50 us in
// place of 63 behind 32768 tokens, and the error against 64 bits, both 2-norms,
// was 2.1e-3 with bf16 where the rounding of the output alone is 1.7e-3, as now.
//
// Measured, 8 key heads of 128 columns with eight query heads each, 32
// sequences: behind 32768 tokens 63 us, 0.55 PFLOP/s without counting weights
// twice, behind 131072 215 us, 0.64 (a large product of the library: 1.3 to 1.4).
// In the latter the matrix pipes work 49 % of the cycles, the vector units 46 %
// beside the issue of the MFMAs, the LDS 16 %; two waves of a SIMD overlap the
// two only in part.  10 us of a launch are its start and the 32-bit outputs of
// 256 jobs (34 MB).
// Steps, measured with weights in one value:
//  * All DMAs of a stage at once, where all waves wait for the issue: 200 us
//    behind 131072 tokens; one by one between the scores' MFMAs: 174; between
//    the output's: 184.
//  * Four waves of 64 rows with a barrier a tile of 32 tokens: 91 us behind
//    32768 tokens; eight waves of 32 rows, page rows of 32 stages in a register,
//    stages of 64 tokens (the barriers half): 60.
//  * D = 256 has room for 128 rows and for tiles of one stage.
#include "paged_prefix.h"
#include "sfa_fwd.h"

namespace dsa {

__device__ __attribute__((aligned(16))) unsigned char g_prefix_zero_row[1024];

constexpr int kPrefixPages = 1024;  // block-table entries held in LDS

// tiles of a stage of the ring, and stages: what 128 KB of LDS hold
template <int D> constexpr int kPrefixSub = D == 256 ? 1 : 2;
template <int D> constexpr int kPrefixRing = D == 64 ? 6 : 4;

// FAST: no DMA lies in two pages (jobs start at whole tiles: there is no band),
// and none of its rows' offsets needs more than 32 bits, so that one descriptor
// serves a DMA in place of an address per lane (32 sequences behind 32768
// tokens: 63 us against 75 at 8 key heads of 128 columns, 44.6 against 46.6
// at 8 of 64, 69 against 98 at 4 of 256).
template <typename T, int D, int NW, int MR, bool FAST>
__global__ __launch_bounds__(NW * 64, 1) void prefix_grouped_kernel(PagedPrefixParams p) {
  using E = Elem<T>;
  using V8 = typename E::v8;
  constexpr int R = NW * 16 * MR, NT = NW * 64, TILE = kPrefixTile;
  constexpr int KS = D / 32;                // k-steps of the scores
  constexpr int ND = D / 16;                // output tiles
  constexpr int ROW = D * 2;
  constexpr int CPT = D / 8;                // 16-byte chunks of a token
  constexpr int TPI = 64 / CPT;             // tokens of one DMA
  constexpr int SUB = kPrefixSub<D>, FETCH = TILE * SUB;   // tokens of a stage
  constexpr int NI = FETCH / TPI / NW;      // DMAs of a wave per stage of K, and of V
  constexpr int K_BYTES = FETCH * ROW, STAGE = 2 * K_BYTES, NB = kPrefixRing<D>;
  constexpr int kStages = 64 / NI;          // stages whose rows a register holds
  constexpr int HR = MR / 2;                // row tiles of the first half of a softmax
  static_assert(NI * NW * TPI == FETCH && MR % 2 == 0 && NB * STAGE <= 131072, "tile split");
  __shared__ __attribute__((aligned(16))) unsigned char smem[NB * STAGE];
  __shared__ int s_tab[kPrefixPages];
  __shared__ int s_lo[R], s_hi[R];  // tokens that the rows see

  const int tid = threadIdx.x, lane = tid & 63, li = lane & 15, lg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  auto swz_k = [](int t) { return D == 64 ? rope_swz(t) : nope_swz(t); };
  auto swz_v = [](int t) { return D == 64 ? ((t >> 1) & 3) << 1 : nope_swz(t); };

  const int64_t row_bytes = (int64_t)p.n2 * ROW;
  const float scale = p.scale_log2 == 0.f ? 1.f : fabsf(p.scale_log2);
  const unsigned flip = p.scale_log2 < 0.f ? 0x80008000u : 0u, keep = p.scale_log2 == 0.f ? 0u : ~0u;
  const unsigned smem_base = (unsigned)(uintptr_t)smem;
  // where a lane reads, and the wave's DMAs take from
  const int k_at = li * ROW + ((lg ^ swz_k(li)) * 16);
  const int v_tok = lg * 4 + (li >> 2);
  const int v_at = K_BYTES + v_tok * ROW + ((((li & 3) >> 1) ^ swz_v(v_tok)) * 16) + (li & 1) * 8;
  int k_from[NI], v_from[NI];
#pragma unroll
  for (int j = 0; j < NI; ++j) {
    const int tk = (j * NW + wave) * TPI + lane / CPT;
    k_from[j] = (int)((lane / CPT) * row_bytes) + ((lane % CPT) ^ swz_k(tk)) * 16;
    v_from[j] = (int)((lane / CPT) * row_bytes) + ((lane % CPT) ^ swz_v(tk)) * 16;
  }

  int head;
  int job = prefix_job_of(p, blockIdx.x, gridDim.x, 0, &head);
  const int jobs = *p.n_jobs;
  for (int round = 0; job < jobs;) {
    const PagedJob jb = p.job[job];
    const int first = jb.first, n_rows = jb.rows, tok0 = jb.tok0, tok1 = jb.tok1;
    const bool masked = tok0 < jb.all_lo || tok1 > jb.all_hi;
    if (masked) {  // what the rows see, where it is not all of it
      lds_barrier();  // (the job before has read what it left)
      for (int r = tid; r < n_rows; r += NT) prefix_bounds(p, jb, r, s_lo + r, s_hi + r);
    }
    const bool active = wave * 16 * MR < n_rows;
    V8 qf[MR][KS];
    auto load_q = [&]() {
      u32x4 x[MR][KS];
#pragma unroll
      for (int rt = 0; rt < MR; ++rt) {
        const int r = wave * 16 * MR + rt * 16 + li;
        const bool live = r < n_rows;
        const unsigned vr = jb.row0 + (live ? r : 0), i = prefix_div(vr, p.rows, p.rows_magic);
        const unsigned rr = vr - i * p.rows, s = prefix_div(rr, p.group, p.group_magic);
        const int64_t row = ((int64_t)(first + i) * p.s1 + s) * p.n1 + head * p.group + (rr - s * p.group);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
          x[rt][ks] = live ? *(const u32x4*)((const T*)p.q + row * D + ks * 32 + lg * 8) : u32x4{0u, 0u, 0u, 0u};
      }
#pragma unroll
      for (int rt = 0; rt < MR; ++rt)
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) qf[rt][ks] = as_v8<V8>((x[rt][ks] & keep) ^ flip);
    };
    f32x4 acc[ND][MR];
    float ref[MR], top[MR], sum[MR];
#pragma unroll
    for (int rt = 0; rt < MR; ++rt) {
      ref[rt] = top[rt] = -INFINITY;
      sum[rt] = 0.f;
#pragma unroll
      for (int j = 0; j < ND; ++j) acc[j][rt] = {0.f, 0.f, 0.f, 0.f};
    }
    const unsigned char* const kbase = (const unsigned char*)p.k + (int64_t)head * ROW;
    const unsigned char* const vbase = (const unsigned char*)p.v + (int64_t)head * ROW;
    const int32_t* const tab = p.table + (int64_t)jb.lead * p.max_blocks;

    for (int ta = tok0; ta < tok1;) {
      // the pages of as many tokens as the LDS holds entries for, in whole tiles
      unsigned off0;
      const int pg0 = (int)paged_split(p, (unsigned)ta, &off0);
      const int64_t reach = (int64_t)(pg0 + kPrefixPages) * p.page;
      const int tb = reach >= tok1 ? tok1 : (int)(reach / TILE * TILE);
      const int npg = (int)paged_split(p, (unsigned)tb - 1u, &off0) - pg0 + 1;
      lds_barrier();  // the entries and tiles before are read
      for (int i = tid; i < npg; i += NT) s_tab[i] = tab[pg0 + i];
      lds_barrier();
      const int n_tiles = (tb - ta + TILE - 1) / TILE;

      // cache row of a token, -1 outside the span or without a page (read as zeros)
      auto row_of = [&](int tok) -> int {
        if (tok >= tb) return -1;
        unsigned off;
        const unsigned pg = paged_split(p, (unsigned)tok, &off);
        const int blk = s_tab[(int)pg - pg0];
        const int64_t r = (int64_t)blk * p.page + (int)off;
        return blk < 0 || r >= p.kv_rows ? -1 : (int)r;
      };
      // DMA i (K and V in turn) of the f-th stage's tokens into the ring at `at`
      int rows = -1;  // lane e: first cache row of DMA pair e % NI of stage f0 + e / NI
      auto dma = [&](int f, int i, int at) {
        const int j = i >> 1, tok = ta + f * FETCH;
        const unsigned dst = smem_base + at + (j * NW + wave) * 1024 + (i & 1 ? K_BYTES : 0);
        if constexpr (FAST) {
          if (i == 0 && f % kStages == 0) rows = row_of(tok + lane / NI * FETCH + ((lane % NI) * NW + wave) * TPI);
          // (a row of -1: no bytes)
          const int r = __builtin_amdgcn_readlane(rows, (f % kStages) * NI + j);
          const int bytes = min(tb - tok - (j * NW + wave) * TPI, TPI) * (int)row_bytes & ~(r >> 31);
          const int64_t from = (int64_t)max(r, 0) * row_bytes;
          dma_buf16(dst, i & 1 ? v_from[j] : k_from[j],
                    __builtin_amdgcn_make_buffer_rsrc((void*)((i & 1 ? vbase : kbase) + from), (short)0, bytes, 0x00020000));
        } else {
          const int tk = (j * NW + wave) * TPI + lane / CPT;
          const int r = row_of(tok + tk), ch = ((lane % CPT) ^ (i & 1 ? swz_v(tk) : swz_k(tk))) * 16;
          dma_glb16(dst, r >= 0 ? (i & 1 ? vbase : kbase) + r * row_bytes + ch : g_prefix_zero_row + ch);
        }
      };
      auto fetch = [&](int f, int at) {
#pragma unroll
        for (int i = 0; i < 2 * NI; ++i) dma(f, i, at);
      };

      float f_moved[MR];
      bool moved = false;
      auto weights = [&](int rt, int tt, f32x4 (&s)[2][MR], V8 (&ph)[MR], V8 (&pl)[MR]) {
        const float from = ref[rt] == -INFINITY ? 0.f : ref[rt];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float e = fast_exp2(__builtin_fmaf(s[tt][rt][i], scale, -from));
          sum[rt] += e;
          ph[rt][tt * 4 + i] = E::from_f32(e);
          pl[rt][tt * 4 + i] = E::from_f32(e - E::to_f32(ph[rt][tt * 4 + i]));
        }
      };
      // the first half of the softmax of tile t, in NA slices
      constexpr int NA = 2 + 2 * HR, NBH = 2 * HR;
      auto soft_a = [&](int k, f32x4 (&s)[2][MR], V8 (&ph)[MR], V8 (&pl)[MR], int t) {
        if (k == 0) {
          const int tk = ta + t * TILE;
          if (masked || tk + TILE > tb) {
            const int mine = tk + lg * 4;
#pragma unroll
            for (int rt = 0; rt < MR; ++rt) {
              const int r = min(wave * 16 * MR + rt * 16 + li, n_rows - 1);
              const int lo = masked ? s_lo[r] : 0, hi = masked ? min(s_hi[r], tb) : tb;
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                const int tok = mine + (i >> 2) * 16 + (i & 3);
                s[i >> 2][rt][i & 3] = tok >= lo && tok < hi ? s[i >> 2][rt][i & 3] : -INFINITY;
              }
            }
          }
        } else if (k == 1) {
          float m[MR];
          bool moves = false;
#pragma unroll
          for (int rt = 0; rt < MR; ++rt) {
            m[rt] = s[0][rt][0];
#pragma unroll
            for (int i = 1; i < 8; ++i) m[rt] = fmaxf(m[rt], s[i >> 2][rt][i & 3]);
            top[rt] = fmaxf(top[rt], m[rt]);
            moves |= m[rt] * scale > ref[rt] + kPaAbove;
          }
          moved = __any(moves);
          if (moved) {
#pragma unroll
            for (int rt = 0; rt < MR; ++rt) {
              const float mx = xgroup_max(m[rt]) * scale;
              const float nref = mx > ref[rt] + kPaAbove ? mx - kPaBelow : ref[rt];
              const float f = ref[rt] == -INFINITY ? 0.f : fast_exp2(ref[rt] - nref);
              ref[rt] = nref;
              sum[rt] *= f;
              f_moved[rt] = f;
            }
          }
        } else if (k < NA) {
          weights((k - 2) >> 1, (k - 2) & 1, s, ph, pl);
        }
      };
      // the second half, in NBH slices
      auto soft_b = [&](int k, f32x4 (&s)[2][MR], V8 (&ph)[MR], V8 (&pl)[MR]) { weights(HR + (k >> 1), k & 1, s, ph, pl); };
      // The first fragments of a product are read while the one before it ends:
      // both tiles have landed by then.
      constexpr int PK = 2, PV = 2;
      V8 ka[PK][2], va[PV];
      auto read_k = [&](int base, int ks, int tt) {
        return as_v8<V8>(*(const u32x4*)(smem + (base ^ ((ks & 3) << 6)) + tt * 16 * ROW + (ks >> 2) * 256));
      };
      auto read_v = [&](int base, int dt) -> V8 {
        const unsigned char* pp = smem + (base ^ ((dt & 7) << 5)) + (dt >> 3) * 256;
        const bf16x4 v1 = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16x4*)pp);
        const bf16x4 v2 = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16x4*)(pp + 16 * ROW));
        const i16x4 w1 = __builtin_bit_cast(i16x4, v1), w2 = __builtin_bit_cast(i16x4, v2);
        const i16x8 w = {w1[0], w1[1], w1[2], w1[3], w2[0], w2[1], w2[2], w2[3]};
        return __builtin_bit_cast(V8, w);
      };
      auto first_k = [&](int at) {
#pragma unroll
        for (int i = 0; i < PK; ++i)
#pragma unroll
          for (int tt = 0; tt < 2; ++tt) ka[i][tt] = read_k(at + k_at, i, tt);
      };
      auto first_v = [&](int at) {
#pragma unroll
        for (int i = 0; i < PV; ++i) va[i] = read_v(at + v_at, i);
      };
      // scores of the tile at `at`; behind them the tile at `then` is multiplied
      auto gemm1 = [&](int at, int then, f32x4 (&s)[2][MR], auto&& between) {
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
#pragma unroll
          for (int tt = 0; tt < 2; ++tt) {
            const V8 f = ka[ks % PK][tt];
            if (ks + PK < KS) ka[ks % PK][tt] = read_k(at + k_at, ks + PK, tt);
            else if (ks + 1 == KS && tt == 0) first_v(then);
#pragma unroll
            for (int rt = 0; rt < MR; ++rt) {
              const f32x4 z = {0.f, 0.f, 0.f, 0.f};
              s[tt][rt] = E::mfma(f, qf[rt][ks], ks == 0 ? z : s[tt][rt]);
            }
            between(ks * 2 + tt);
            __builtin_amdgcn_sched_barrier(0);
          }
        }
      };
      // output of the tile at `at`; behind it come the scores of the tile at `then`
      auto gemm2 = [&](int at, int then, V8 (&ph)[MR], V8 (&pl)[MR], auto&& between) {
#pragma unroll
        for (int dt = 0; dt < ND; ++dt) {
          const V8 f = va[dt % PV];
          if (dt + PV < ND) va[dt % PV] = read_v(at + v_at, dt + PV);
          else if (SUB == 2 && dt + 1 == ND) first_k(then);
#pragma unroll
          for (int rt = 0; rt < MR; ++rt) acc[dt][rt] = E::mfma(f, ph[rt], acc[dt][rt]);
#pragma unroll
          for (int rt = 0; rt < MR; ++rt) acc[dt][rt] = E::mfma(f, pl[rt], acc[dt][rt]);
          between(dt);
          __builtin_amdgcn_sched_barrier(0);
        }
        if (moved) {  // for the tile after this one
#pragma unroll
          for (int rt = 0; rt < MR; ++rt) {
#pragma unroll
            for (int j = 0; j < ND; ++j) acc[j][rt] *= f_moved[rt];
          }
        }
      };

      // the first stage comes beside Q, whose loads end here, the others behind
      // (those past the end, here and below, read zeros, so that the number of
      // DMAs in flight is known)
      fetch(0, 0);
      if (ta == tok0) load_q();
      wait_vmcnt<0>();
#pragma unroll
      for (int rt = 0; rt < MR; ++rt)
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) asm volatile("" : "+v"(qf[rt][ks]));
#pragma unroll 1
      for (int f = 1; f < NB - 1; ++f) fetch(f, f * STAGE);
      lds_barrier();
      // step t: scores of tile t + 1 (of no visible token after the last) with the
      // second half of the softmax of tile t, then the output of tile t with the
      // first half of that of tile t + 1
      int at = 0;  // of the stage of tile t
      const int n_stages = (n_tiles + SUB - 1) / SUB;
      auto next_stage = [&](int x) { return x == (NB - 1) * STAGE ? 0 : x + STAGE; };
      auto open_stage = [&]() {
        wait_vmcnt<(NB - 3) * 2 * NI>();  // the stage after it has landed
        lds_barrier();
      };
      auto free_stage = [&]() { return at == 0 ? (NB - 1) * STAGE : at - STAGE; };
      if (active) {
        f32x4 s0[2][MR], s1[2][MR];
        V8 p0[MR], p1[MR], l0[MR], l1[MR];
        first_k(0);
        gemm1(0, 0, s0, [](int) {});
#pragma unroll
        for (int k = 0; k < NA; ++k) soft_a(k, s0, p0, l0, 0);
        if (moved) {
#pragma unroll
          for (int rt = 0; rt < MR; ++rt) {
#pragma unroll
            for (int j = 0; j < ND; ++j) acc[j][rt] *= f_moved[rt];
          }
        }
        // Tiles t, t + 1 and t + 2 lie at `cur`, `next` and `then`.  DMAs d0 .. d1 of
        // stage f go into the ring at `to`, between the scores: one after the
        // other they hold up the wave that asks for them (43 cycles each, when
        // all waves do).
        auto step = [&](int t, int cur, int next, int then, f32x4 (&s)[2][MR], f32x4 (&sn)[2][MR], V8 (&ph)[MR],
                        V8 (&pl)[MR], V8 (&pn)[MR], V8 (&ln)[MR], auto d0, auto d1, int f, int to) {
          gemm1(next, cur, sn, [&](int i) {
            // 2 KS places for NBH slices and the DMAs
#pragma unroll
            for (int k = i * NBH / (2 * KS); k < (i + 1) * NBH / (2 * KS); ++k) soft_b(k, s, ph, pl);
            constexpr int n = decltype(d1)::value - decltype(d0)::value;
#pragma unroll
            for (int k = i * n / (2 * KS); k < (i + 1) * n / (2 * KS); ++k) dma(f, decltype(d0)::value + k, to);
          });
          gemm2(cur, then, ph, pl, [&](int i) {
#pragma unroll
            for (int k = i * NA / ND; k < (i + 1) * NA / ND; ++k) soft_a(k, sn, pn, ln, t + 1);
          });
        };
        // (the first fragments of tile 1's scores: its stage has landed)
        if constexpr (SUB == 2) first_k(TILE * ROW);
        std::integral_constant<int, 0> none;
        std::integral_constant<int, NI> half;
        std::integral_constant<int, 2 * NI> all;
        for (int t = 0;;) {
          open_stage();
          int next = next_stage(at);
          asm volatile("" : "+s"(next));  // (so that each stage's offsets fit the instructions)
          if constexpr (SUB == 2) {
            const int here = at, to = free_stage(), f = t / 2 + NB - 1;
            step(t, here, here + TILE * ROW, next, s0, s1, p0, l0, p1, l1, none, half, f, to);
            at = next;  // (of tile t + 2)
            if (++t >= n_tiles) break;
            step(t, here + TILE * ROW, next, next + TILE * ROW, s1, s0, p1, l1, p0, l0, half, all, f, to);
            if (++t >= n_tiles) break;
          } else {
            first_k(next);
            step(t, at, next, next, s0, s1, p0, l0, p1, l1, none, all, t + NB - 1, free_stage());
            at = next;
            if (++t >= n_tiles) break;
            open_stage();
            int then = next_stage(next);
            asm volatile("" : "+s"(then));
            first_k(then);
            step(t, at, then, then, s1, s0, p1, l1, p0, l0, none, all, t + NB - 1, free_stage());
            at = then;
            if (++t >= n_tiles) break;
          }
        }
      } else {
        for (int f = 0; f < n_stages; ++f) {
          open_stage();
          fetch(f + NB - 1, free_stage());
          at = next_stage(at);
        }
      }
      wait_vmcnt<0>();  // of the DMAs past the end too: the ring is theirs until then
      ta = tb;
    }

    // the job's output
    const int64_t slot0 = p.part0 + ((int64_t)job * p.n2 + head) * R;
#pragma unroll
    for (int rt = 0; rt < MR; ++rt) {
      const int r = wave * 16 * MR + rt * 16 + li;
      const float l = xgroup_sum(sum[rt]), t = xgroup_max(top[rt]) * scale;
      if (r >= n_rows) continue;
      const float seen = l != 0.f ? 1.f : 0.f;
      float* dst = p.part_o + (slot0 + r) * D + lg * 4;
#pragma unroll
      for (int j = 0; j < ND; ++j) *(f32x4*)(dst + j * 16) = paged_scaled(acc[j][rt], seen);
      if (lg == 0) p.part_ml[slot0 + r] = {ref[rt], l, t, l};
    }
    job = prefix_job_of(p, blockIdx.x, gridDim.x, ++round, &head);
  }
}

// ---------------------------------------------------------------------------
// the operator: the prefixes, what is behind them, and the join
// ---------------------------------------------------------------------------
struct PrefixShape {
  PagedShape behind;
  int workers, shift;  // jobs of one key head aimed at; log2 of the rows of a block
  int64_t jobs, grid;  // at most
  int64_t run_rows, whole_rows, job_rows;  // of outputs: of runs, of sequences that a run has whole, of jobs
};

static int prefix_shift(int64_t d, bool latent) { return latent || d == 256 ? 7 : 8; }

// together: whether there may be jobs
static PrefixShape prefix_shape(int64_t batch, int64_t s1, int64_t n1, int64_t n2, int64_t d, bool latent,
                                int64_t max_blocks, int64_t page, bool together) {
  PrefixShape s;
  s.behind = paged_shape(batch, s1, n1, n2, d, latent, max_blocks, page);
  s.shift = prefix_shift(d, latent);
  const int64_t cus = device_cu_count();
  s.workers = (int)(cus / n2 < 1 ? 1 : cus / n2);
  const int64_t blocks = (batch * s1 * (n1 / n2) >> s.shift) + batch / 2 + 1;
  s.jobs = blocks >= (1ll << 30) ? 1ll << 31 : prefix_jobs((int)blocks, s.workers);
  s.grid = (cus + 7) / 8 * 8;
  if (!together) s.jobs = 0;
  s.run_rows = (int64_t)s.behind.workers * 2 * s.behind.groups * s.behind.group_rows;
  s.whole_rows = together ? batch * s.behind.groups * s.behind.group_rows : 0;
  s.job_rows = s.jobs * n2 << s.shift;
  return s;
}

bool paged_prefix_launchable(int64_t batch, int64_t s1, int64_t n1, int64_t n2, int64_t d, bool latent,
                             int64_t max_blocks, int64_t page) {
  const PrefixShape s = prefix_shape(batch, s1, n1, n2, d, latent, max_blocks, page, true);
  // (jobs, their places over all key heads, and the tiles of all blocks of rows are counted in 32 bits)
  return s.jobs < (1ll << 26) && s.jobs * n2 + s.grid < (1ll << 31) &&
         ((batch * s1 * (n1 / n2) >> s.shift) + batch) * ((max_blocks * page + kPrefixTile - 1) / kPrefixTile) < (1ll << 31);
}

// Tokens of a prefix from which on it is worked on for its family together
// (described in paged_prefix.h).
static int prefix_least(int64_t min_tokens, int64_t rows, int64_t readers, int64_t token_bytes, bool latent) {
  constexpr int64_t never = 0x7fffffff;
  if (min_tokens < 0)
    min_tokens = latent && rows >= 64 ? never : (latent ? 320 << 20 : 256 << 20) / (readers * token_bytes);
  return (int)(min_tokens < 1 ? 1 : (min_tokens < never ? min_tokens : never));
}

// How a call is worked on: which prefixes for their families together, and the
// sequences of a launch.  Together takes some three times the rows of the queries
// in 32 bits: up to 512 MB of it for all sequences at once, else for as many at a
// time (families that go on in the next launch are cut there, as at multiples of
// 64 sequences; with so many rows each has blocks of its own anyway), and for none
// where two would be too many.
constexpr int64_t kPrefixBytes = 1 << 29;

struct PrefixCall {
  int least;      // tokens, more than the table has where nothing is worked on together
  int64_t batch;  // sequences of a launch
  PrefixShape shape;
  size_t part_rows() const { return (size_t)(shape.run_rows + shape.whole_rows + shape.job_rows); }
};

static PrefixCall prefix_call(int64_t batch, int64_t s1, int64_t n1, int64_t n2, int64_t d, bool latent,
                              int64_t max_blocks, int64_t page, int64_t min_tokens) {
  PrefixCall c;
  const int64_t room = max_blocks * page;
  auto shape = [&](int64_t n, bool together) { return prefix_shape(n, s1, n1, n2, d, latent, max_blocks, page, together); };
  c.batch = batch;
  c.shape = shape(batch, true);
  c.least = prefix_least(min_tokens, s1 * (n1 / n2), batch * c.shape.behind.row_groups, (latent ? d + 64 : 2 * n2 * d) * 2,
                         latent);
  auto fits = [&](const PrefixShape& s) {
    return (s.whole_rows + s.job_rows) * (int64_t)(sizeof(f32x4) + d * sizeof(float)) <= kPrefixBytes;
  };
  if (c.least <= room && !fits(c.shape)) {
    int64_t most = 1, over = batch;
    while (over - most > 1) {
      const int64_t n = (most + over) / 2;
      (fits(shape(n, true)) ? most : over) = n;
    }
    if (most == 1) c.least = 0x7fffffff;
    const int64_t launches = (batch + most - 1) / most;
    if (most > 1) c.batch = (batch + launches - 1) / launches;
  }
  if (c.least > room || c.batch < batch) c.shape = shape(c.batch, c.least <= room);
  return c;
}

size_t paged_prefix_workspace_bytes(int64_t batch, int64_t s1, int64_t n1, int64_t n2, int64_t d, bool latent,
                                    int64_t max_blocks, int64_t page, int64_t min_tokens) {
  const PrefixCall c = prefix_call(batch, s1, n1, n2, d, latent, max_blocks, page, min_tokens);
  return c.part_rows() * (sizeof(f32x4) + d * sizeof(float)) + (size_t)c.batch * sizeof(PagedWhere) +
         (size_t)c.shape.jobs * sizeof(PagedJob) + 16;
}

template <typename T, bool FAST>
static void prefix_grouped_d(const PagedPrefixParams& p, int64_t d, unsigned grid, hipStream_t stream) {
  if (d == 64) prefix_grouped_kernel<T, 64, 8, 2, FAST><<<grid, 512, 0, stream>>>(p);
  else if (d == 128) prefix_grouped_kernel<T, 128, 8, 2, FAST><<<grid, 512, 0, stream>>>(p);
  else prefix_grouped_kernel<T, 256, 4, 2, FAST><<<grid, 256, 0, stream>>>(p);
}

static int prefix_grouped_launch(const PagedPrefixParams& p, int64_t d, int32_t dtype, unsigned grid, hipStream_t stream) {
  const int tokens = (int)(512 / d);  // of a DMA
  const bool fast = p.page % tokens == 0 && (int64_t)p.n2 * d * 2 * tokens < (1ll << 31) && p.band_pre >= (1ll << 31);
  if (dtype == DSA_DTYPE_BF16 && fast) prefix_grouped_d<bf16, true>(p, d, grid, stream);
  else if (dtype == DSA_DTYPE_BF16) prefix_grouped_d<bf16, false>(p, d, grid, stream);
  else if (fast) prefix_grouped_d<f16, true>(p, d, grid, stream);
  else prefix_grouped_d<f16, false>(p, d, grid, stream);
  DSA_HIP(hipGetLastError());
  return DSA_OK;
}

int paged_prefix_run(const void* query, const void* query_rope, const void* key, const void* key_rope,
                     const void* value, void* out, float* smax, float* ssum, const int32_t* act_q,
                     const int32_t* act_k, const int32_t* table, const int32_t* ids, const int32_t* shared,
                     int64_t batch, int64_t s1, int64_t n1, int64_t n2, int64_t d, int64_t num_blocks, int64_t page,
                     int64_t max_blocks, int32_t mode, int64_t pre_tokens, int64_t next_tokens, int64_t min_tokens,
                     int32_t dtype, float scale, int32_t return_lse, void* workspace, hipStream_t stream) {
  const bool latent = value == nullptr;
  const PrefixCall c = prefix_call(batch, s1, n1, n2, d, latent, max_blocks, page, min_tokens);
  const bool together = c.least <= max_blocks * page;
  auto at = [](const void* x, int64_t bytes) { return x ? (const unsigned char*)x + bytes : nullptr; };
  for (int64_t b0 = 0; b0 < batch; b0 += c.batch) {
    const int64_t n = batch - b0 < c.batch ? batch - b0 : c.batch, rows0 = b0 * s1 * n1;
    const PrefixShape s =
        n == c.batch ? c.shape : prefix_shape(n, s1, n1, n2, d, latent, max_blocks, page, together);
    PagedPrefixParams p = {};
    paged_fill(p, s.behind, at(query, rows0 * d * 2), at(query_rope, rows0 * 64 * 2), key, key_rope, value,
               (void*)at(out, rows0 * d * 2), (float*)at(smax, rows0 * 4), (float*)at(ssum, rows0 * 4),
               (const int32_t*)at(act_q, b0 * 4), act_k + b0, table + b0 * max_blocks, n, s1, n1, n2, num_blocks, page,
               max_blocks, mode, pre_tokens, next_tokens, scale, return_lse);
    const int64_t rows = s.run_rows + s.whole_rows + s.job_rows;
    p.part_ml = (f32x4*)workspace;
    p.part_o = (float*)(p.part_ml + rows);
    p.where = (PagedWhere*)(p.part_o + rows * d);
    p.job = (PagedJob*)(p.where + n);
    p.n_jobs = (int*)(p.job + s.jobs);
    p.whole0 = s.run_rows;
    p.part0 = p.whole0 + s.whole_rows;
    p.ids = ids + b0;
    p.shared = shared + b0;
    p.before = (int)b0;
    p.least = c.least;
    p.prefix_workers = s.workers;
    p.job_shift = s.shift;
    p.rows_magic = 0xffffffffu / (unsigned)p.rows;
    p.group_magic = 0xffffffffu / (unsigned)p.group;
    p.heads_magic = 0xffffffffu / (unsigned)p.n2;
    const int64_t most = (s.jobs * n2 + 7) / 8 * 8;
    const unsigned grid = (unsigned)(most < s.grid ? most : s.grid);
    int st = latent ? paged_latent_launch(p, d, dtype, stream) : paged_grouped_launch(p, d, dtype, stream);
    if (st == DSA_OK && together)
      st = latent ? prefix_latent_launch(p, d, dtype, grid, stream) : prefix_grouped_launch(p, d, dtype, grid, stream);
    if (st == DSA_OK) st = paged_combine_launch(p, s.behind.tile, d, dtype, stream);
    if (st != DSA_OK) return st;
  }
  return DSA_OK;
}

}  // namespace dsa
