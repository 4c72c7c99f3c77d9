// Rotary positions: the pairs (a, b) of a head's rotary slice turned by the
// angle position * inv_freq[i],
//   a' = s (a cos - b sin),  b' = s (a sin + b cos),
// with pairs of adjacent columns (interleaved) or of columns i and i + R/2
// (half).  The backward is the rotation by the opposite angle, the same
// kernel with the sine negated.
//
// The angle is formed in 64 bits, as turns: position * inv_freq / 2 pi less
// its nearest integer is exact to 2^-33 of a turn at position 2^20, where a
// 32-bit product is off by 0.06 rad.  The sine and cosine of what is left
// are taken in 32 bits, once per token and frequency, into LDS; all heads of
// the token share them.  No table of positions is read or kept.
//
// Bound by memory (3 flops per element), or by the launch for one decoding
// step.  A thread moves 16 bytes (two times 16 for pairs in the half layout),
// neighbouring threads neighbouring chunks of a head; heads and tokens are
// flattened, so that no lane idles at any head count.  Query and key go in
// one launch.  4096 tokens of 128 heads of 192 columns and a key, 403 MB read
// and written: 85 us, 4.7 TB/s (a large copy reaches 4.9).
#include "common.h"

namespace dsa {

struct RopeTensor {
  const void* in;
  void* out;
  int64_t in_sb, in_ss, in_sh;     // strides in elements: batch, token, head
  int64_t out_sb, out_ss, out_sh;
  int heads, d, start;             // head columns, first rotated column
  int units;                       // work units of a head
  int total;                       // heads * units
  unsigned magic;                  // of units
};

struct RopeParams {
  RopeTensor t[2];
  const void* pos;
  const double* inv_freq;
  int64_t tokens;
  int s;               // tokens of a sequence (BSND); tokens for packed rows
  int pos64, pos_per_seq;
  int rot, rot_units, interleaved;
  int tok_wg, parts, per_part;     // tokens of a workgroup; unit ranges they are cut into
  float scale, sign;
};

constexpr int kRopeThreads = 256;
constexpr int kRopeDeep = 3;
constexpr int kRopeTab = 4096;  // cos and sin values of a workgroup's tokens

template <typename T> struct RopeIo {
  static __device__ __forceinline__ float get(T x) { return Elem<T>::to_f32(x); }
  static __device__ __forceinline__ T put(float x) { return Elem<T>::from_f32(x); }
};
template <> struct RopeIo<float> {
  static __device__ __forceinline__ float get(float x) { return x; }
  static __device__ __forceinline__ float put(float x) { return x; }
};

// n / d with magic = floor((2^32 - 1) / d): n * magic / 2^32 is at most
// n / 2^32 below n / d, so its integer part is off by one at most
__device__ __forceinline__ int fast_div(unsigned n, unsigned d, unsigned magic) {
  const unsigned q = __umulhi(n, magic);
  return (int)(q + (n - q * d >= d));
}

// VEC elements per chunk: 16 bytes, or 1 where sizes, strides or addresses
// do not allow it.  A unit is one chunk of the output, so that lanes read and
// write memory in its order; in the half layout it reads the other member of
// its pairs too, which the cache holds (both members by one lane: a fifth of
// the lanes active in every second load and store, 117 against 99 us for 4096
// tokens of 128 heads of 128 + 64 columns).  In place and with VEC = 1 a unit
// is what one lane can turn alone: a pair of chunks or columns, or a copy.
template <typename T, int VEC, bool INPLACE, bool STREAM>
__global__ __launch_bounds__(kRopeThreads) void rope_kernel(RopeParams p) {
  typedef T Vec __attribute__((ext_vector_type(VEC)));
  // (a choice of two tensors' addresses is a flat address unless it is said
  // that both are global; flat accesses wait for LDS too)
  typedef __attribute__((address_space(1))) T GT;
  typedef __attribute__((address_space(1))) Vec GVec;
  using Io = RopeIo<T>;
  constexpr bool kPairs = INPLACE || VEC == 1;
  __shared__ float s_tab[kRopeTab];
  const int half = p.rot / 2;
  const int64_t tok0 = (int64_t)(blockIdx.x / p.parts) * p.tok_wg;
  const int ntok = (int)min((int64_t)p.tok_wg, p.tokens - tok0);
  for (int i = threadIdx.x; i < ntok * half; i += kRopeThreads) {
    const int tk = i / half, f = i - tk * half;
    const int64_t t = tok0 + tk;
    const int64_t pi = p.pos_per_seq ? t : t % p.s;
    const double pos = p.pos64 ? (double)((const int64_t*)p.pos)[pi] : (double)((const int32_t*)p.pos)[pi];
    const double turns = pos * (p.inv_freq[f] * 0.15915494309189533577);  // 1 / (2 pi)
    float sn, cs;
    sincospif(2.f * (float)(turns - rint(turns)), &sn, &cs);
    s_tab[2 * i] = cs * p.scale;
    s_tab[2 * i + 1] = sn * p.scale * p.sign;
  }
  __syncthreads();
  const int all = p.t[0].total + p.t[1].total;
  const int u0 = (blockIdx.x % p.parts) * p.per_part;
  const int u1 = min(u0 + p.per_part, all * ntok);
  auto put = [&](GT* at, Vec x) {
    if constexpr (STREAM) __builtin_nontemporal_store(x, (GVec*)at);
    else *(GVec*)at = x;
  };
  // kRopeDeep units of a thread at a time: all their loads go out before the
  // first is used
  for (int ub = u0 + threadIdx.x; ub < u1; ub += kRopeThreads * kRopeDeep) {
    Vec va[kRopeDeep], vb[kRopeDeep];
    GT* dst[kRopeDeep];
    int unit[kRopeDeep];  // chunk of the head; -1: none
    int tab[kRopeDeep];   // its token's sines and cosines
    int start[kRopeDeep];
#pragma unroll
    for (int j = 0; j < kRopeDeep; ++j) {
      const int u = ub + j * kRopeThreads;
      unit[j] = -1;
      if (u >= u1) continue;
      const int tk = ntok == 1 ? 0 : u / all;
      int r = u - tk * all;
      const bool key = r >= p.t[0].total;
      r -= key ? p.t[0].total : 0;
      const unsigned units = key ? p.t[1].units : p.t[0].units;
      const int h = fast_div((unsigned)r, units, key ? p.t[1].magic : p.t[0].magic), c = r - h * (int)units;
      const int64_t t = tok0 + tk, b = p.s == p.tokens ? 0 : t / p.s, s = t - b * p.s;
      const GT* in = (const GT*)(key ? p.t[1].in : p.t[0].in) + b * (key ? p.t[1].in_sb : p.t[0].in_sb) +
                    s * (key ? p.t[1].in_ss : p.t[0].in_ss) + h * (key ? p.t[1].in_sh : p.t[0].in_sh);
      dst[j] = (GT*)(key ? p.t[1].out : p.t[0].out) + b * (key ? p.t[1].out_sb : p.t[0].out_sb) +
               s * (key ? p.t[1].out_ss : p.t[0].out_ss) + h * (key ? p.t[1].out_sh : p.t[0].out_sh);
      unit[j] = c;
      tab[j] = tk * p.rot;
      start[j] = key ? p.t[1].start : p.t[0].start;
      if constexpr (kPairs) {
        // pairs c * VEC ..: columns i and i + R/2, or (VEC = 1) 2i and 2i + 1
        if (c >= p.rot_units) {  // a column outside the rotary slice
          int col = (c - p.rot_units) * VEC;
          if (col >= start[j]) col += p.rot;
          dst[j] += col;
          va[j] = *(const GVec*)(in + col);
        } else {
          const int ca = start[j] + (p.interleaved ? (VEC > 1 ? c * VEC : 2 * c) : c * VEC);
          dst[j] += ca;
          va[j] = *(const GVec*)(in + ca);
          if (VEC == 1 || !p.interleaved) vb[j] = *(const GVec*)(in + ca + (p.interleaved ? 1 : half));
        }
      } else {
        // chunk c of the head; unit: its place in the rotary slice, or past it
        const int col = c * VEC, i = col - start[j];
        dst[j] += col;
        va[j] = *(const GVec*)(in + col);
        unit[j] = i >= 0 && i < p.rot ? i / VEC : p.rot_units;
        if (!p.interleaved && unit[j] < p.rot_units) vb[j] = *(const GVec*)(in + col + (i < half ? half : -half));
      }
    }
#pragma unroll
    for (int j = 0; j < kRopeDeep; ++j) {
      const int c = unit[j];
      if (c < 0) continue;
      // one store for all lanes, turned or copied (stores of their own for
      // each took 10 us more of 94)
      Vec w = va[j];
      if (c < p.rot_units) {
        if (VEC > 1 && p.interleaved) {
#pragma unroll
          for (int i = 0; i < VEC / 2; ++i) {
            const float cs = s_tab[tab[j] + c * VEC + 2 * i], sn = s_tab[tab[j] + c * VEC + 2 * i + 1];
            const float a = Io::get(va[j][2 * i]), bb = Io::get(va[j][VEC > 1 ? 2 * i + 1 : 0]);
            w[2 * i] = Io::put(a * cs - bb * sn);
            w[VEC > 1 ? 2 * i + 1 : 0] = Io::put(a * sn + bb * cs);
          }
        } else if constexpr (!kPairs) {
          // the other member of each pair is in vb
          const bool first = c * VEC < half;
          const int t2 = tab[j] + 2 * (c * VEC - (first ? 0 : half));
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            const float cs = s_tab[t2 + 2 * i], s1 = s_tab[t2 + 2 * i + 1], sn = first ? -s1 : s1;
            w[i] = Io::put(Io::get(va[j][i]) * cs + Io::get(vb[j][i]) * sn);
          }
        } else {
          Vec wb;
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            const float cs = s_tab[tab[j] + 2 * (c * VEC + i)], sn = s_tab[tab[j] + 2 * (c * VEC + i) + 1];
            const float a = Io::get(va[j][i]), bb = Io::get(vb[j][i]);
            w[i] = Io::put(a * cs - bb * sn);
            wb[i] = Io::put(a * sn + bb * cs);
          }
          put(dst[j] + (p.interleaved ? 1 : half), wb);
        }
      }
      put(dst[j], w);
    }
  }
}

template <typename T>
static void rope_launch(const RopeParams& p, int vec, bool inplace, bool streaming, int64_t grid, hipStream_t stream) {
  constexpr int VEC = 16 / (int)sizeof(T);
  const dim3 g((unsigned)grid);
  if (vec == 1) rope_kernel<T, 1, true, false><<<g, kRopeThreads, 0, stream>>>(p);
  else if (inplace) rope_kernel<T, VEC, true, false><<<g, kRopeThreads, 0, stream>>>(p);
  else if (streaming) rope_kernel<T, VEC, false, true><<<g, kRopeThreads, 0, stream>>>(p);
  else rope_kernel<T, VEC, false, false><<<g, kRopeThreads, 0, stream>>>(p);
}

// strides: in (batch, token, head) then out, in elements
int rope_run(const void* const in[2], void* const out[2], const int64_t* const strides[2], const int64_t heads[2],
             const int64_t d[2], const int64_t start[2], int n, const void* positions, int32_t pos64,
             int32_t pos_per_seq, const double* inv_freq, int64_t tokens, int64_t s, int64_t rot, int32_t interleaved,
             int32_t inverse, int32_t dtype, float scale, hipStream_t stream) {
  const int es = dtype == DSA_DTYPE_FP32 ? 4 : 2;
  const int full = 16 / es;
  // 16-byte chunks: every column count, offset, stride and address a whole
  // number of them
  bool wide = (interleaved ? rot : rot / 2) % full == 0;
  for (int i = 0; i < n; ++i) {
    wide &= d[i] % full == 0 && start[i] % full == 0;
    wide &= (((uintptr_t)in[i] | (uintptr_t)out[i]) & 15) == 0;
    for (int j = 0; j < 6; ++j) wide &= strides[i][j] % full == 0;
  }
  const int vec = wide ? full : 1;
  RopeParams p = {};
  p.rot = (int)rot;
  p.interleaved = interleaved;
  // an output that is its input, of either tensor, takes the units that need
  // no other's input
  bool inplace = false;
  for (int i = 0; i < n; ++i) inplace |= in[i] == out[i];
  const bool pairs = inplace || !wide;
  p.rot_units = (int)(pairs ? (wide && interleaved ? rot / vec : rot / 2 / vec) : rot / vec);
  int64_t all = 0;
  for (int i = 0; i < n; ++i) {
    RopeTensor& x = p.t[i];
    x.in = in[i];
    x.out = out[i];
    x.in_sb = strides[i][0], x.in_ss = strides[i][1], x.in_sh = strides[i][2];
    x.out_sb = strides[i][3], x.out_ss = strides[i][4], x.out_sh = strides[i][5];
    x.heads = (int)heads[i];
    x.d = (int)d[i];
    x.start = (int)start[i];
    // in place, the columns outside the slice stay as they are
    x.units = pairs ? p.rot_units + (in[i] == out[i] ? 0 : (int)((d[i] - rot) / vec)) : (int)(d[i] / vec);
    x.total = x.heads * x.units;
    x.magic = 0xffffffffu / (unsigned)x.units;
    all += x.total;
  }
  p.pos = positions;
  p.inv_freq = inv_freq;
  p.tokens = tokens;
  p.s = (int)s;
  p.pos64 = pos64;
  p.pos_per_seq = pos_per_seq;
  p.scale = scale;
  p.sign = inverse ? -1.f : 1.f;
  // tokens of few units share a workgroup; tokens of many are cut into parts
  // where they alone would not give every CU a few workgroups
  p.tok_wg = 1;
  while (p.tok_wg < 16 && p.tok_wg * all < kRopeThreads && 2 * p.tok_wg * rot <= kRopeTab) p.tok_wg *= 2;
  // 201 MB of output: 93.5 us with such stores, 96.5 without (half layout;
  // interleaved 81.9 and 87.1)
  int64_t bytes = 0;
  for (int i = 0; i < n; ++i) bytes += tokens * heads[i] * d[i] * es;
  const bool streaming = bytes > (64ll << 20);  // more than the caches hold for whoever reads it
  const int64_t groups = (tokens + p.tok_wg - 1) / p.tok_wg;
  const int64_t units = p.tok_wg * all;
  int64_t parts = 4ll * device_cu_count() / groups;
  const int64_t most = (units + kRopeThreads - 1) / kRopeThreads;
  parts = parts < 1 ? 1 : (parts > most ? most : parts);
  p.per_part = (int)(((units + parts - 1) / parts + kRopeThreads - 1) / kRopeThreads * kRopeThreads);
  p.parts = (int)((units + p.per_part - 1) / p.per_part);
  const int64_t grid = groups * p.parts;
  DSA_CHECK_SUPPORTED(launchable(grid, kRopeThreads), "too many tokens for one launch");
  if (dtype == DSA_DTYPE_BF16) rope_launch<bf16>(p, vec, inplace, streaming, grid, stream);
  else if (dtype == DSA_DTYPE_FP16) rope_launch<f16>(p, vec, inplace, streaming, grid, stream);
  else rope_launch<float>(p, vec, inplace, streaming, grid, stream);
  DSA_HIP(hipGetLastError());
  return DSA_OK;
}

}  // namespace dsa
