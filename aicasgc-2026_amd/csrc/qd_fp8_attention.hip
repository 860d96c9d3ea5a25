// Attention over the 8-bit KV cache for gfx950: one query token or several per
// sequence, causal, with an optional sliding window and first tokens (sinks) that
// stay visible.
//
// Row r of a (sequence, kv head) is query token r / G, head kvh G + r % G, and
// sees cache rows t <= p (p its position) below the capacity; with a window W also
// t > p - W or t < sinks.  Out of a row that sees nothing come zeros.
//
// A 64-token tile of the cache carries one exponent for K and one for V.  K's goes
// into the score factor.  V's would scale the probabilities into their fp16
// operand's subnormals, so it joins the softmax's exponent instead: with
// s' = s + ev (log2 units) and the running maximum m' of s',
//   p' = 2^(s' - m'),   l = sum p' 2^-ev,   o = sum p' vq,   out = o / l,
// where vq are the stored values: p' is near its maximum for the rows that
// contribute most, whatever their blocks' exponents.
//
// Products run on the fp16 MFMAs with the cache's bytes converted exactly in
// registers and fp32 sums.  The probabilities, times 2^9, are rounded to fp16: at most
// 2^-11 of each, as the output's own rounding is of their sum, and of either sign, so
// that over N(0, 1) rows the result is 2.7e-4 from 64 bits where its rounding alone is
// 2.0e-4.  (The same MFMAs on two fp16 halves of each would cost as many again.)  l
// sums them unrounded.

#include <math.h>

#include <type_traits>

#include "qd_fp8.h"

namespace qd {

namespace {

typedef _Float16 h2v __attribute__((ext_vector_type(2)));

constexpr int kHD = 128;
constexpr int kTileBytes = kKvBlock * kHD;
constexpr float kProbExp = 9.f;
constexpr float kMaxLag = 6.f;   // 2^(9 + 6) is within fp16
constexpr float kLowest = -3.402823466e38f;   // running maximum of a row that has seen nothing

// The cache tiles that query tokens at [p_min, p_max] of a sequence see: the sink tiles
// [0, ns) and the tiles [first, first + n - ns); of those, [full0, full1) and [0, sink_full)
// are visible to every one of them as a whole.
struct TileRange {
  int first, ns, n, full0, full1, sink_full;
  __device__ __forceinline__ int tile(int v) const { return v < ns ? v : first + (v - ns); }
  __device__ __forceinline__ bool masked(int t) const { return !((t >= full0 && t < full1) || t < sink_full); }
};
__device__ __forceinline__ TileRange visible_tiles(long p_min, long p_max, const AttnFp8Args& a) {
  TileRange r{0, 0, 0, 0, 0, 0};
  const long hi = min(p_max + 1, (long)a.c.T);
  if (hi <= 0) return r;
  const int end = (int)((hi + kKvBlock - 1) >> 6);
  r.full1 = (int)(max(min(p_min + 1, (long)a.c.T), 0L) >> 6);
  if (a.window > 0) {
    r.first = (int)min(max(p_min - a.window + 1, 0L) >> 6, (long)end);
    r.ns = min((int)((min((long)a.sinks, hi) + kKvBlock - 1) >> 6), r.first);
    r.full0 = (int)min((max(p_max - a.window + 1, 0L) + kKvBlock - 1) >> 6, (long)end);
    r.sink_full = min(a.sinks >> 6, r.full1);
  }
  r.n = r.ns + end - r.first;
  return r;
}

// Maximum over the four lane groups g (v_permlane*_swap: no LDS round trip).  (The
// swapped pair goes through scalars: bit casts of a vector's elements are folded to
// its first one.)
__device__ __forceinline__ float max_groups(float x) {
  const unsigned u = __builtin_bit_cast(unsigned, x);
  const auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  const unsigned a0 = a[0], a1 = a[1];
  const unsigned v = __builtin_bit_cast(unsigned, fmaxf(__builtin_bit_cast(float, a0), __builtin_bit_cast(float, a1)));
  const auto b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  const unsigned b0 = b[0], b1 = b[1];
  return fmaxf(__builtin_bit_cast(float, b0), __builtin_bit_cast(float, b1));
}

// True where an e4m3 byte of v is NaN (0x7f or 0xff).
__device__ __forceinline__ unsigned nan_bytes(unsigned v) { return ((v & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }

// A wave's QT x 16 rows (one per column c of each tile, the same in the four
// lane groups g) and what they have accumulated, of 16 ND of the 128 dims.
template <int QT, int ND = 8>
struct Rows {
  long p_min, p_max;    // positions of all rows that share this wave's tiles
  int prow[QT];         // each row's, from p_min on (rows past the last repeat it)
  f32x4 o[QT][ND];      // O^T: dims 16 d + 4 g + j from the first of its own on
  float m[QT], l[QT];
};

template <int QT, int ND>
__device__ __forceinline__ void init_rows(Rows<QT, ND>& w, h8v (&q)[QT][4], const AttnFp8Args& a, int b, int kvh, long pos, int r0,
                                          int R, int c, int g) {
#pragma unroll
  for (int i = 0; i < QT; ++i) {
    const int r = min(r0 + 16 * i + c, R - 1), tok = r / a.G;
    w.prow[i] = (int)(pos + tok - w.p_min);
    const uint16_t* src = a.q + b * a.q_sb + (long)(kvh * a.G + r - tok * a.G) * a.q_sh + (long)tok * a.q_ss + 16 * g;
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) q[i][ks] = *reinterpret_cast<const h8v*>(src + 64 * (ks / 2) + 8 * (ks & 1));
    w.m[i] = kLowest;
    w.l[i] = 0.f;
#pragma unroll
    for (int d = 0; d < ND; ++d) w.o[i][d] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
}

// S^T of a tile; load(n, h) gives 16 bytes of this lane's K row of MFMA n, q(i, ks) the
// operand of row tile i.
template <int QT, typename F, typename Q>
__device__ __forceinline__ void scores(f32x4 (&s)[QT][4], Q q, F load) {
#pragma unroll
  for (int i = 0; i < QT; ++i)
#pragma unroll
    for (int n = 0; n < 4; ++n) s[i][n] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    u32x4 k[4];
#pragma unroll
    for (int n = 0; n < 4; ++n) k[n] = load(n, h);
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      h8v qf[QT];
#pragma unroll
      for (int i = 0; i < QT; ++i) qf[i] = q(i, 2 * h + u);
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        const h8v kf = fp8x8_to_f16(k[n][2 * u], k[n][2 * u + 1]);
#pragma unroll
        for (int i = 0; i < QT; ++i) s[i][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qf[i], s[i][n], 0, 0, 0);
      }
    }
  }
}

// Bit 4 n + j: this lane's token (n, j) of the tile at `base` is visible to its row i.
template <int QT, int ND>
__device__ __forceinline__ unsigned visible_bits(const Rows<QT, ND>& w, const int i, const long base, const AttnFp8Args& a, const int g) {
  // bits of the tokens below x of this lane's 16
  auto below = [&](long x) { return 0xffffu >> (16 - min(max((int)min(max(x - base, 0L), (long)kKvBlock) - 16 * g, 0), 16)); };
  const long p = w.p_min + w.prow[i];
  unsigned seen = below(p + 1);
  if (a.window > 0) seen &= ~below(p + 1 - a.window) | below(a.sinks);
  return seen;
}

// Masks a tile's scores and lets the rows' maxima follow them.
template <int QT, int ND>
__device__ __forceinline__ void mask_and_max(Rows<QT, ND>& w, f32x4 (&s)[QT][4], const float fac, const int ev, const bool masked,
                                             const long base, const AttnFp8Args& a, const int g) {
  if (masked) {
#pragma unroll
    for (int i = 0; i < QT; ++i) {
      const unsigned seen = visible_bits(w, i, base, a, g);
#pragma unroll
      for (int n = 0; n < 4; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) s[i][n][j] = (seen >> (4 * n + j)) & 1u ? s[i][n][j] : -INFINITY;
    }
  }
  // The running maximum follows only when some row's has grown by more than kMaxLag
  // (log2): until then the probabilities stay within fp16 and the accumulators as
  // they are.
  const float fev = (float)ev;
  float mx[QT];
  bool grow = false;
#pragma unroll
  for (int i = 0; i < QT; ++i) {
    float x = s[i][0][0];
#pragma unroll
    for (int n = 0; n < 4; ++n)
#pragma unroll
      for (int j = 0; j < 4; ++j) x = fmaxf(x, s[i][n][j]);
    mx[i] = __builtin_fmaf(max_groups(x), fac, fev);
    grow = grow || mx[i] > w.m[i] + kMaxLag;
  }
  if (__any(grow)) {
#pragma unroll
    for (int i = 0; i < QT; ++i) {
      const float mn = fmaxf(w.m[i], mx[i]);
      const float al = __builtin_amdgcn_exp2f(w.m[i] - mn);
      w.m[i] = mn;
      w.l[i] *= al;
#pragma unroll
      for (int d = 0; d < ND; ++d) w.o[i][d] *= al;
    }
  }
}

// The tile's probabilities in units of the rows' maxima, and their sums.
template <int QT, int ND>
__device__ __forceinline__ void probabilities(Rows<QT, ND>& w, const f32x4 (&s)[QT][4], const float fac, const int ev,
                                              h8v (&p)[QT][2]) {
  const float fev = (float)ev, inv = pow2i(-ev);
#pragma unroll
  for (int i = 0; i < QT; ++i) {
    const float sub = kProbExp + fev - w.m[i];
    float ps = 0.f;
#pragma unroll
    for (int n = 0; n < 4; ++n)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float y = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i][n][j], fac, sub));
        ps += y;
        p[i][n / 2][4 * (n & 1) + j] = (_Float16)y;
      }
    w.l[i] = __builtin_fmaf(ps, inv, w.l[i]);
  }
}

// O^T += V^T.P^T; load(d) gives 16 bytes of this lane's V row of dims 16 d.
template <int QT, int ND, typename F>
__device__ __forceinline__ void accumulate(Rows<QT, ND>& w, const h8v (&p)[QT][2], F load) {
#pragma unroll
  for (int d = 0; d < ND; ++d) {
    const u32x4 v = load(d);
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      const h8v vf = fp8x8_to_f16(v[2 * ks], v[2 * ks + 1]);
#pragma unroll
      for (int i = 0; i < QT; ++i) w.o[i][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, p[i][ks], w.o[i][d], 0, 0, 0);
    }
  }
}

// A NaN among the V rows must reach the rows that see it and no others, though a
// masked probability times it would be NaN.  A masked tile is multiplied with its NaN
// bytes as zeros (clean_nan), and after all tiles mark_nan reads the masked ones
// again and counts the NaNs that a row sees, per dim, by a product with the masks.
__device__ __forceinline__ u32x4 clean_nan(u32x4 v) {
#pragma unroll
  for (int x = 0; x < 4; ++x) v[x] &= ~((nan_bytes(v[x]) >> 7) * 0xffu);
  return v;
}

// tile(v): the v-th of the wave's tiles v, v + step, ... below v1; vp: this lane's V
// row of its first dims and token 16 g.
template <int QT, int ND>
__device__ __forceinline__ void mark_nan(Rows<QT, ND>& w, const TileRange& tr, int v, const int step, const int v1, const uint8_t* vp,
                                         const AttnFp8Args& a, const int g) {
#pragma unroll 1
  for (; v < v1; v += step) {
    if (!tr.masked(tr.tile(v))) continue;
    const long t = tr.tile(v), base = t * kKvBlock;
    unsigned any = 0u;
#pragma unroll
    for (int d = 0; d < ND; ++d) {
      const u32x4 x = ld16(vp + t * kTileBytes + 16 * d * kKvBlock);
      any |= nan_bytes(x.x) | nan_bytes(x.y) | nan_bytes(x.z) | nan_bytes(x.w);
    }
    if (!__any(any != 0u)) continue;
#pragma unroll
    for (int i = 0; i < QT; ++i) {
      const unsigned seen = visible_bits(w, i, base, a, g);
      h8v vis[2];
#pragma unroll
      for (int e = 0; e < 16; ++e) vis[e / 8][e % 8] = (seen >> e) & 1u ? (_Float16)1.f : (_Float16)0.f;
#pragma unroll
      for (int d = 0; d < ND; ++d) {
        const u32x4 x = ld16(vp + t * kTileBytes + 16 * d * kKvBlock);
        f32x4 cnt = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
          h8v f;
#pragma unroll
          for (int e = 0; e < 8; ++e)
            f[e] = (nan_bytes(x[2 * ks + e / 4]) >> (8 * (e & 3) + 7)) & 1u ? (_Float16)1.f : (_Float16)0.f;
          cnt = __builtin_amdgcn_mfma_f32_16x16x32_f16(f, vis[ks], cnt, 0, 0, 0);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (cnt[j] > 0.f) w.o[i][d][j] = NAN;
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  }
}

// Accumulated rows in LDS: row r's 16-byte chunk x at x ^ (r % 32).
__device__ __forceinline__ f32x4* row_chunk(char* slot, int r, int x) {
  return reinterpret_cast<f32x4*>(slot + r * (kHD * 4) + 16 * (x ^ (r & 31)));
}
// A wave's rows, chunk(r, x) the place of row r's chunk x.
template <int QT, int ND, typename F>
__device__ __forceinline__ void spill_rows(Rows<QT, ND>& w, F chunk, float (*sml)[2], int c, int g) {
#pragma unroll
  for (int i = 0; i < QT; ++i) {
    const int r = 16 * i + c;
    w.l[i] += __shfl_xor(w.l[i], 16);
    w.l[i] += __shfl_xor(w.l[i], 32);
    if (g == 0) {
      sml[r][0] = w.m[i];
      sml[r][1] = w.l[i];
    }
#pragma unroll
    for (int d = 0; d < ND; ++d) *chunk(r, 4 * d + g) = w.o[i][d];
  }
}

__device__ __forceinline__ void store_out(const AttnFp8Args& a, int b, int kvh, int r, int d, const f32x4 acc, const float l) {
  const float il = l == 0.f ? 0.f : 1.f / l;
  const long row = ((long)b * a.Sq + r / a.G) * a.c.Hkv * a.G + kvh * a.G + r % a.G;
  *reinterpret_cast<u32x2*>(a.out + row * kHD + d) = u32x2{pack2(acc.x * il, acc.y * il), pack2(acc.z * il, acc.w * il)};
}

// Joins NS waves' ROWS rows (fixed order), chunk(wave, r, x) the place of a chunk:
// the result's dims from d0 on, or a split's partial.
template <int NS, int ROWS, int NT, int ND, typename F>
__device__ __forceinline__ void join_rows(F chunk, float (*sml)[ROWS][2], const AttnFp8Args& a, int bh, int split, int r0, int R,
                                          int d0) {
  for (int n = threadIdx.x; n < ROWS * 4 * ND; n += NT) {
    const int rr = n / (4 * ND), x = n % (4 * ND), d = d0 + 4 * x, r = r0 + rr;
    if (r >= R) break;
    float mm = sml[0][rr][0];
#pragma unroll
    for (int y = 1; y < NS; ++y) mm = fmaxf(mm, sml[y][rr][0]);
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    float ll = 0.f;
#pragma unroll
    for (int y = 0; y < NS; ++y) {
      const float f = __builtin_amdgcn_exp2f(sml[y][rr][0] - mm);
      ll = __builtin_fmaf(sml[y][rr][1], f, ll);
      acc += *chunk(y, rr, x) * f;
    }
    if (a.n_split > 1) {
      const long pr = ((long)bh * a.n_split + split) * R + r;
      *reinterpret_cast<f32x4*>(a.part_o + pr * kHD + d) = acc;
      if (d == 0) {
        a.part_ml[2 * pr] = mm;
        a.part_ml[2 * pr + 1] = ll;
      }
    } else {
      store_out(a, bh / a.c.Hkv, bh % a.c.Hkv, r, d, acc, ll);
    }
  }
}

// (a scale that underflows to 0 would turn the masked -inf scores into NaN)
__device__ __forceinline__ float score_factor(const AttnFp8Args& a, int k_byte) {
  return fmaxf(a.scale2 * pow2i(k_byte - 127), 0x1p-120f);
}

// S^T = K.Q^T and O^T = V^T.P^T.  A lane's K row of MFMA n = 2 s + a is token
// 16 (c / 4) + 8 s + 4 a + c % 4, so that its results (one q row, tokens
// 16 g + 8 s + 4 a + i) are in order the second product's operand, whose k slots
// are the 16 consecutive tokens 16 g .. 16 g + 15 of the V row it loads: no lane
// exchange between the two products.
__device__ __forceinline__ int k_token(int c, int n) { return 16 * (c >> 2) + 4 * n + (c & 3); }

}  // namespace

// At most 16 rows of one (sequence, kv head): bound by the cache's bytes.  NW waves
// take the split's tiles in turn, each tile from memory to the MFMA without LDS,
// and their partial softmaxes are joined through LDS.  The scores of a wave's next
// tile are multiplied before the softmax of this one, and K two tiles and V one
// tile ahead are in flight meanwhile.
//
// One workgroup per CU (190 registers, eight waves).  Measured, two q rows of each of 8 kv
// heads: 30001 rows 14.4 us (61 MB, 4.3 TB/s) and 3 to 4 for the merge, 8 sequences of 2048 to
// 4096 rows 14.3 and the same, 1029 rows 8.6 in one launch, one tile 4.4.  (Four
// waves and twice the splits: 18.9 us in all for 17.5 at 30001 rows; V two tiles ahead as
// well, 228 registers: 17.4 for 17.1.)
//
// DS workgroups may share the dims (128 / DS each) and each read all of K: what one CU
// takes in, some 50 bytes a ns of what memory has to send, falls from 16 KB a tile to
// 8 + 8 / DS.
template <int NW, int DS>
__global__ __launch_bounds__(kWave * NW) void attention_fp8_kernel(const AttnFp8Args a) {
  constexpr int ND = 8 / DS;
  __shared__ __align__(16) char s_o[NW][16 * kHD * 4];
  __shared__ float s_ml[NW][16][2];
  const int lane = lane_id();
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int c = lane & 15, g = lane >> 4;
  const int bh = (int)blockIdx.x, b = bh / a.c.Hkv, kvh = bh % a.c.Hkv;
  const int split = (int)blockIdx.y, R = a.Sq * a.G, d0 = 16 * ND * (int)blockIdx.z;
  const long pos = a.cache_position[b];
  Rows<1, ND> rows;
  rows.p_min = pos;
  rows.p_max = pos + a.Sq - 1;
  const TileRange tr = visible_tiles(rows.p_min, rows.p_max, a);
  const int v0 = (int)((unsigned)tr.n * (unsigned)split / (unsigned)a.n_split);
  const int v1 = (int)((unsigned)tr.n * (unsigned)(split + 1) / (unsigned)a.n_split);
  const long off = b * a.c.stride_b + kvh * a.c.stride_h;
  const long so = b * a.c.scale_stride_b + kvh * a.c.scale_stride_h;
  const uint8_t* kp = a.c.k + off + k_token(c, 0) * kHD + 16 * g;
  const uint8_t* vp = a.c.v + off + (d0 + c) * kKvBlock + 16 * g;
  u32x4 kr[4][2], vr[ND];
  int ks_byte = 0, vs_byte = 0;   // scales of the tiles in kr and vr
  auto load_k = [&](long t) __attribute__((always_inline)) {
#pragma unroll
    for (int n = 0; n < 4; ++n)
#pragma unroll
      for (int h = 0; h < 2; ++h) kr[n][h] = ld16(kp + t * kTileBytes + 4 * n * kHD + 64 * h);
    ks_byte = a.c.k_scale[so + t];
  };
  auto load_v = [&](long t) __attribute__((always_inline)) {
#pragma unroll
    for (int d = 0; d < ND; ++d) vr[d] = ld16(vp + t * kTileBytes + 16 * d * kKvBlock);
    vs_byte = a.c.v_scale[so + t];
  };
  int v = v0 + w;
  if (v < v1) {
    load_k(tr.tile(v));
    load_v(tr.tile(v));
  }
  h8v q[1][4];
  init_rows<1, ND>(rows, q, a, b, kvh, pos, 0, R, c, g);
  f32x4 s[2][1][4];
  float fac[2];
  auto next_scores = [&](auto X) __attribute__((always_inline)) {
    constexpr int x = decltype(X)::value;
    scores<1>(s[x], [&](int i, int ks) { return q[i][ks]; }, [&](int n, int h) { return kr[n][h]; });
    fac[x] = score_factor(a, ks_byte);
  };
  auto body = [&](auto X, int v) __attribute__((always_inline)) {
    constexpr int x = decltype(X)::value;
    if (v + NW < v1) {
      next_scores(std::integral_constant<int, 1 - x>{});
      if (v + 2 * NW < v1) load_k(tr.tile(v + 2 * NW));
    }
    __builtin_amdgcn_sched_barrier(0);
    h8v p[1][2];
    const long base = tr.tile(v) * kKvBlock;
    const bool masked = tr.masked(tr.tile(v));
    mask_and_max<1, ND>(rows, s[x], fac[x], vs_byte - 127, masked, base, a, g);
    if (masked) {
#pragma unroll
      for (int d = 0; d < ND; ++d) vr[d] = clean_nan(vr[d]);
    }
    probabilities<1, ND>(rows, s[x], fac[x], vs_byte - 127, p);
    accumulate<1, ND>(rows, p, [&](int d) { return vr[d]; });
    if (v + NW < v1) load_v(tr.tile(v + NW));
  };
  if (v < v1) {
    next_scores(std::integral_constant<int, 0>{});
    if (v + NW < v1) load_k(tr.tile(v + NW));
  }
#pragma unroll 1
  for (; v < v1; v += 2 * NW) {
    body(std::integral_constant<int, 0>{}, v);
    if (v + NW >= v1) break;
    body(std::integral_constant<int, 1>{}, v + NW);
  }
  mark_nan<1, ND>(rows, tr, v0 + w, NW, v1, vp, a, g);
  auto chunk = [&](int x, int r, int y) { return row_chunk(s_o[x], r, y); };
  spill_rows<1, ND>(rows, [&](int r, int y) { return chunk(w, r, y); }, s_ml[w], c, g);
  __syncthreads();
  join_rows<NW, 16, kWave * NW, ND>(chunk, s_ml, a, bh, split, 0, R, d0);
}

namespace {

constexpr int kStreams = 4;      // tiles that a workgroup of many rows works on at once
constexpr int kManyRows = 64;    // its rows: two groups of 32
constexpr int kStageBytes = kStreams * 2 * kTileBytes;

__device__ __forceinline__ void load_lds16(const void* g, void* l) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)g,
                                   (__attribute__((address_space(3))) void*)l, 16, 0, 0);
}

// This wave's loads and LDS accesses are done, then the workgroup barrier.
__device__ __forceinline__ void wait_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_waitcnt(0x0070);   // vmcnt(0) lgkmcnt(0)
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("" ::: "memory");
}

// Separate variables: the compiler then knows that reading one stage does not
// depend on the loads in flight to the other.
template <int I>
__device__ __forceinline__ char* attention_stage() {
  __shared__ __align__(16) char buf[kStageBytes];
  return buf;
}

}  // namespace

// More rows, 64 per workgroup: bound by the products and the softmax's vector
// instructions.  Eight waves: 32 rows (wave % 2) of every fourth tile (wave / 2).
// V of a step's four tiles and K of the next step's lie in LDS, filled by asynchronous
// loads one step ahead (K by the even wave of a pair, V by the odd one), so that a tile
// is read from L2 once for 64 rows and converted once for 32, and the products of the
// next scores run beside this step's softmax.  q's operands lie in LDS too: registers
// for a step's two sets of scores.
//
// Measured, 16 heads over 8: 929 tokens, the last at row 4000, 48 to 51 us (0.55 PFLOP/s), a
// prompt of 4001 110 us (0.6).  The vector instructions (conversions of K and V, and per
// score a scaling, an exponential, a sum and a rounding) take 38 % of the cycles, the
// products 21 %; the rest are waits of the two waves a SIMD has.  (16 waves of 16 rows: 57 / 120 us; 96 rows in 12 waves 70 /
// 117; q in registers 53 / 118; the probabilities' sums through the matrix unit, or a raised
// wave priority: no change; tiles per wave without the barrier 54 / 112.)
//
// A tile in LDS: K's token row t has its 16-byte chunk c at c ^ f, f of t's bits
// 0, 1 and 4 (the rows of one fragment read differ in bits 0, 1, 4 and 5); V's dim row
// d (64 bytes) at c ^ (d / 2 % 4).
__global__ __launch_bounds__(512, 2) void attention_fp8_many_kernel(const AttnFp8Args a) {
  __shared__ h8v s_q[2][2][4][kWave];
  __shared__ float s_ml[kStreams][kManyRows][2];
  const int lane = lane_id();
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int c = lane & 15, g = lane >> 4, half = w & 1, stream = w >> 1;
  // (sequence, kv head) fastest: with 8 of them one head's row tiles share an XCD's L2
  const unsigned heads = (unsigned)(a.c.B * a.c.Hkv);
  const int bh = (int)(blockIdx.x % heads), b = bh / a.c.Hkv, kvh = bh % a.c.Hkv;
  // the tiles of the latest rows, which see the most, start first
  const int R = a.Sq * a.G, r0 = (int)(gridDim.x / heads - 1 - blockIdx.x / heads) * kManyRows;
  const int split = (int)blockIdx.y;
  const long pos = a.cache_position[b];
  Rows<2> rows;
  rows.p_min = pos + r0 / a.G;
  rows.p_max = pos + min(r0 + kManyRows - 1, R - 1) / a.G;
  const TileRange tr = visible_tiles(rows.p_min, rows.p_max, a);
  const int v0 = (int)((unsigned)tr.n * (unsigned)split / (unsigned)a.n_split);
  const int v1 = (int)((unsigned)tr.n * (unsigned)(split + 1) / (unsigned)a.n_split);
  const long off = b * a.c.stride_b + kvh * a.c.stride_h;
  const long so = b * a.c.scale_stride_b + kvh * a.c.scale_stride_h;
  const bool idle = r0 + 32 * half >= R;   // its rows are past the last

  // this lane's source in a tile: K rows 8 i + lane / 8, V rows 16 i + lane / 4
  const int kt = lane >> 3, vd = lane >> 2;
  const uint8_t* src = half == 0 ? a.c.k + off + kt * kHD : a.c.v + off + vd * kKvBlock + 16 * ((lane & 3) ^ ((vd >> 1) & 3));
  int ks_next = 0, vs_next = 0;
  // This wave's half of a stage: K of tile v + 4 (even wave) or V of tile v (odd wave)
  // of its stream; a stream without a tile loads the last one.
  auto issue = [&](auto S, int v) __attribute__((always_inline)) {
    const long tk = tr.tile(min(v + kStreams + stream, v1 - 1)), tv = tr.tile(min(max(v + stream, v0), v1 - 1));
    char* st = attention_stage<decltype(S)::value>() + stream * 2 * kTileBytes + half * kTileBytes;
    if (half == 0) {
      const int ch[2] = {16 * ((lane & 7) ^ (kt & 3)), 16 * ((lane & 7) ^ ((kt & 3) | 4))};   // by bit 4 of the token
#pragma unroll
      for (int i = 0; i < 8; ++i) load_lds16(src + tk * kTileBytes + i * 1024 + ch[(i >> 1) & 1], st + i * 1024);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) load_lds16(src + tv * kTileBytes + i * 1024, st + i * 1024);
    }
    ks_next = a.c.k_scale[so + tk];
    vs_next = a.c.v_scale[so + tv];
  };
  if (v0 < v1) issue(std::integral_constant<int, 1>{}, v0 - kStreams);   // the first tiles' K
  {
    h8v q[2][4];
    init_rows<2, 8>(rows, q, a, b, kvh, pos, r0 + 32 * half, R, c, g);
    if (stream < 2)   // one row tile each
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) s_q[half][stream][ks][lane] = stream == 0 ? q[0][ks] : q[1][ks];
  }
  // offsets of this lane's K chunks h = 0, 1 of token k_token(c, n) (n adds whole rows
  // and leaves f's bits) and of its V chunk
  const int fk = (c & 3) | ((c >> 2) & 1) << 2;
  const int ko = k_token(c, 0) * kHD + 16 * (g ^ fk);   // chunk 4 + g is at ko ^ 64
  const int vo = kTileBytes + c * kKvBlock + 16 * (g ^ ((c >> 1) & 3));
  auto qrow = [&](int i, int ks) { return s_q[half][i][ks][lane]; };
  f32x4 s[2][2][4];
  float fac_next = 0.f;
  auto next_scores = [&](auto S, auto X) __attribute__((always_inline)) {
    const char* st = attention_stage<decltype(S)::value>() + stream * 2 * kTileBytes;
    scores<2>(s[decltype(X)::value], qrow, [&](int n, int h) { return *reinterpret_cast<const u32x4*>(st + (ko ^ (64 * h)) + 4 * n * kHD); });
  };
  const std::integral_constant<int, 0> i0;
  const std::integral_constant<int, 1> i1;
  // stage S: K of tile v + 4, V of tile v, whose scores are in s[S]
  auto step = [&](auto S, int v) __attribute__((always_inline)) {
    constexpr int x = decltype(S)::value;
    const std::integral_constant<int, 1 - x> other;
    wait_barrier();
    // (opaque: what is computed from them is not moved up to their loads, where it
    // would wait for the tiles in flight)
    asm volatile("" : "+v"(ks_next), "+v"(vs_next));
    const float fac = fac_next;
    fac_next = score_factor(a, ks_next);
    const int ev = vs_next - 127;
    if (v + kStreams < v1) issue(other, v + kStreams);
    v += stream;
    if (v >= v1 || idle) return;
    char* st = attention_stage<x>() + stream * 2 * kTileBytes;
    auto vrow = [&](int d) { return reinterpret_cast<u32x4*>(st + vo + 16 * d * kKvBlock); };
    const long base = tr.tile(v) * kKvBlock;
    const bool masked = tr.masked(tr.tile(v));
    mask_and_max<2, 8>(rows, s[x], fac, ev, masked, base, a, g);
    if (masked) {   // (in place: the wave of the other rows does the same to the same tile)
#pragma unroll
      for (int d = 0; d < 8; ++d) *vrow(d) = clean_nan(*vrow(d));
    }
    // no branch from here on: the next scores' products run beside this softmax's vector
    // instructions (after the last tile they are of no use)
    h8v p[2][2];
    next_scores(S, other);
    probabilities<2, 8>(rows, s[x], fac, ev, p);
    accumulate<2, 8>(rows, p, [&](int d) { return *vrow(d); });
  };
  wait_barrier();
  if (v0 < v1) {
    asm volatile("" : "+v"(ks_next));
    fac_next = score_factor(a, ks_next);
    issue(i0, v0);
    next_scores(i1, i0);
  }
#pragma unroll 1
  for (int v = v0; v < v1; v += 2 * kStreams) {
    step(i0, v);
    if (v + kStreams < v1) step(i1, v + kStreams);
  }
  if (!idle) mark_nan<2, 8>(rows, tr, v0 + stream, kStreams, v1, a.c.v + off + c * kKvBlock + 16 * g, a, g);
  // join the four streams: the stages are free once every wave is past its last
  // step, each holds the rows of two
  wait_barrier();
  static_assert(kStageBytes == 2 * kManyRows * kHD * 4, "two streams' rows per stage");
  auto chunk = [&](int x, int r, int y) {
    return row_chunk((x < 2 ? attention_stage<0>() : attention_stage<1>()) + (x & 1) * kManyRows * kHD * 4, r, y);
  };
  spill_rows<2, 8>(rows, [&](int r, int y) { return chunk(stream, 32 * half + r, y); }, &s_ml[stream][32 * half], c, g);
  __syncthreads();
  join_rows<kStreams, kManyRows, 512, 8>(chunk, s_ml, a, bh, split, r0, R, 0);
}

// Joins the splits' partials of one row per workgroup, in a fixed order: lane s of a
// wave holds the weight of split s, eight groups of 32 lanes (4 dims each) sum an
// eighth of the splits and are added through LDS.  2.8 to 3.8 us: the launch and a
// read.
constexpr int kMaxSplits = 64;
template <int N>   // eights of splits
__global__ __launch_bounds__(256) void attention_fp8_merge_kernel(const AttnFp8Args a) {
  __shared__ __align__(16) f32x4 s_acc[8][32];
  const int R = a.Sq * a.G;
  const long bh = (long)blockIdx.x / R;
  const int r = (int)((long)blockIdx.x % R);
  const long p0 = bh * a.n_split * R + r;
  const int lane = lane_id(), grp = threadIdx.x / 32, d = 4 * (threadIdx.x & 31);
  // (the partials are loaded before their weights are known: one round trip to memory)
  f32x4 part[N];
#pragma unroll
  for (int i = 0; i < N; ++i)
    part[i] = *reinterpret_cast<const f32x4*>(a.part_o + (p0 + (long)min(8 * i + grp, a.n_split - 1) * R) * kHD + d);
  float m = kLowest, l = 0.f;
  if (lane < a.n_split) {
    m = a.part_ml[2 * (p0 + (long)lane * R)];
    l = a.part_ml[2 * (p0 + (long)lane * R) + 1];
  }
  const float wgt = __builtin_amdgcn_exp2f(m - wave_max(m));
  const float ll = wave_sum(l * wgt);
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int s = 8 * i + grp;
    const float f = __shfl(wgt, s);
    if (s < a.n_split) acc += part[i] * f;
  }
  s_acc[grp][threadIdx.x & 31] = acc;
  __syncthreads();
  if (grp != 0) return;
#pragma unroll
  for (int i = 1; i < 8; ++i) acc += s_acc[i][threadIdx.x & 31];
  store_out(a, (int)(bh / a.c.Hkv), (int)(bh % a.c.Hkv), r, d, acc, ll);
}

constexpr long kCUs = 256;

int attention_fp8_splits(int B, int Hkv, int Sq, int G, int T, int window, int sinks) {
  long tiles = T / kKvBlock;
  if (window > 0) tiles = min(tiles, ((long)window + Sq + 2 * kKvBlock) / kKvBlock + ((long)sinks + kKvBlock - 1) / kKvBlock);
  const long R = (long)Sq * G;
  const long units = (long)B * Hkv * (R <= 16 ? 1 : (R + kManyRows - 1) / kManyRows);
  // up to 1536 rows one launch is quicker than two (batch 1, us: 1029 rows 9.5 in one, 11.9
  // in two; 1536 rows 10.5 / 12.5; every 512 rows more add 2 us to one)
  if (tiles <= 24) return 1;
  // one workgroup per CU, a tile or two per wave at least
  const long n = min(kCUs / units, (tiles + 7) / 8);
  return (int)max(1L, min(n, (long)kMaxSplits));
}

int attention_fp8_launch(const AttnFp8Args& a, hipStream_t s) {
  const long R = (long)a.Sq * a.G, heads = (long)a.c.B * a.c.Hkv;
  if (R <= 16) {
    // the dims of few workgroups are shared while that gives every one a CU of its own (8 kv
    // heads, us, alone / shared by four: 1029 rows 10.4 / 8.6, 512 7.0 / 6.4, 64 4.6 / 4.4)
    const long n = heads * a.n_split;
    if (4 * n <= kCUs)
      hipLaunchKernelGGL((attention_fp8_kernel<8, 4>), dim3((unsigned)heads, (unsigned)a.n_split, 4), dim3(512), 0, s, a);
    else if (2 * n <= kCUs)
      hipLaunchKernelGGL((attention_fp8_kernel<8, 2>), dim3((unsigned)heads, (unsigned)a.n_split, 2), dim3(512), 0, s, a);
    else
      hipLaunchKernelGGL((attention_fp8_kernel<8, 1>), dim3((unsigned)heads, (unsigned)a.n_split), dim3(512), 0, s, a);
  } else {
    hipLaunchKernelGGL(attention_fp8_many_kernel, dim3((unsigned)(heads * ((R + kManyRows - 1) / kManyRows)), (unsigned)a.n_split),
                       dim3(512), 0, s, a);
  }
  const int st = qd_host::launch_status("attention_fp8_kernel");
  if (st != QD_OK || a.n_split == 1) return st;
  const dim3 grid((unsigned)(heads * R));
  if (a.n_split <= 8)
    hipLaunchKernelGGL(attention_fp8_merge_kernel<1>, grid, dim3(256), 0, s, a);
  else if (a.n_split <= 32)
    hipLaunchKernelGGL(attention_fp8_merge_kernel<4>, grid, dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL(attention_fp8_merge_kernel<kMaxSplits / 8>, grid, dim3(256), 0, s, a);
  return qd_host::launch_status("attention_fp8_merge_kernel");
}

}  // namespace qd
