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
// registers and fp32 sums; the probabilities, times 2^9, are rounded to fp16 (half
// a step, 2^-12 of each on average half that, where the output's own rounding is
// 2^-11 of the sum), l sums them unrounded.

#include <math.h>

#include "qd_fp8.h"

namespace qd {

namespace {

typedef _Float16 h2v __attribute__((ext_vector_type(2)));

constexpr int kHD = 128;
constexpr int kTileBytes = kKvBlock * kHD;
constexpr float kProbExp = 9.f;
constexpr float kLowest = -3.402823466e38f;   // running maximum of a row that has seen nothing

// The cache tiles that query tokens [t0, t1] of a sequence see: the sink tiles
// [0, ns) and the tiles [first, first + n - ns).
struct TileRange {
  long first;
  int ns, n;
  __device__ __forceinline__ long tile(int v) const { return v < ns ? v : first + (v - ns); }
};
__device__ __forceinline__ TileRange visible_tiles(long p_min, long p_max, const AttnFp8Args& a) {
  TileRange r{0, 0, 0};
  const long hi = min(p_max + 1, (long)a.c.T);
  if (hi <= 0) return r;
  const long end = (hi + kKvBlock - 1) >> 6;
  if (a.window > 0) {
    r.first = min(max(p_min - a.window + 1, 0L) >> 6, end);
    r.ns = (int)min((min((long)a.sinks, hi) + kKvBlock - 1) >> 6, r.first);
  }
  r.n = r.ns + (int)(end - r.first);
  return r;
}

// True where an e4m3 byte of v is NaN (0x7f or 0xff).
__device__ __forceinline__ unsigned nan_bytes(unsigned v) { return ((v & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }

}  // namespace

// NW waves per workgroup, QT x 16 rows of one (sequence, kv head); the waves take
// the split's tiles in turn and their partial softmaxes are joined through LDS.
//
// S^T = K.Q^T and O^T = V^T.P^T.  A lane's K row of MFMA (s, a) is token
// 16 (c / 4) + 8 s + 4 a + c % 4, so that its results (one q row, tokens
// 16 g + 8 s + 4 a + i) are in order the second product's operand, whose k slots
// are the 16 consecutive tokens 16 g .. 16 g + 15 of the V row it loaded: both
// tiles go from memory to the MFMA without LDS or lane exchange.
template <int QT, int NW>
__global__ __launch_bounds__(kWave * NW) void attention_fp8_kernel(const AttnFp8Args a) {
  __shared__ __align__(16) float s_o[NW][16 * QT][kHD + 4];
  __shared__ float s_ml[NW][16 * QT][2];
  const int lane = lane_id();
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int c = lane & 15, g = lane >> 4;
  const int bh = blockIdx.z, b = bh / a.c.Hkv, kvh = bh % a.c.Hkv;
  const int R = a.Sq * a.G, r0 = (int)blockIdx.y * 16 * QT;
  const long pos = a.cache_position[b];
  const int tok0 = r0 / a.G, tok1 = min(r0 + 16 * QT - 1, R - 1) / a.G;
  const TileRange tr = visible_tiles(pos + tok0, pos + tok1, a);
  const int v0 = (int)((long)tr.n * blockIdx.x / a.n_split), v1 = (int)((long)tr.n * (blockIdx.x + 1) / a.n_split);

  long prow[QT];   // each row's position (rows past the last repeat it)
  h8v q[QT][4];
#pragma unroll
  for (int i = 0; i < QT; ++i) {
    const int r = min(r0 + 16 * i + c, R - 1);
    prow[i] = pos + r / a.G;
    const uint16_t* src = a.q + b * a.q_sb + (long)(kvh * a.G + r % a.G) * a.q_sh + (long)(r / a.G) * a.q_ss + 16 * g;
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) q[i][ks] = *reinterpret_cast<const h8v*>(src + 64 * (ks / 2) + 8 * (ks & 1));
  }
  f32x4 o[QT][8];
  float m[QT], l[QT];
#pragma unroll
  for (int i = 0; i < QT; ++i) {
    m[i] = kLowest;
    l[i] = 0.f;
#pragma unroll
    for (int d = 0; d < 8; ++d) o[i][d] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  const long off = b * a.c.stride_b + kvh * a.c.stride_h;
  const long so = b * a.c.scale_stride_b + kvh * a.c.scale_stride_h;
  const uint8_t* kp = a.c.k + off + (16 * (c >> 2) + (c & 3)) * kHD + 16 * g;
  const uint8_t* vp = a.c.v + off + c * kKvBlock + 16 * g;

  for (int v = v0 + w; v < v1; v += NW) {
    const long t = tr.tile(v), base = t * kKvBlock;
    u32x4 kr[4][2], vr[8];
#pragma unroll
    for (int n = 0; n < 4; ++n)   // n = 2 s + a
#pragma unroll
      for (int h = 0; h < 2; ++h) kr[n][h] = ld16(kp + t * kTileBytes + 4 * n * kHD + 64 * h);
#pragma unroll
    for (int d = 0; d < 8; ++d) vr[d] = ld16(vp + t * kTileBytes + 16 * d * kKvBlock);
    // (a scale that underflows to 0 would turn the masked -inf scores into NaN)
    const float fac = fmaxf(a.scale2 * pow2i((int)a.c.k_scale[so + t] - 127), 0x1p-120f);
    const int ev = (int)a.c.v_scale[so + t] - 127;
    f32x4 s[QT][4];
#pragma unroll
    for (int i = 0; i < QT; ++i)
#pragma unroll
      for (int n = 0; n < 4; ++n) s[i][n] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int n = 0; n < 4; ++n)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const h8v kf = fp8x8_to_f16(kr[n][h][2 * u], kr[n][h][2 * u + 1]);
#pragma unroll
          for (int i = 0; i < QT; ++i)
            s[i][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, q[i][2 * h + u], s[i][n], 0, 0, 0);
        }
    const bool full = base + kKvBlock - 1 <= pos + tok0 &&
                      (a.window == 0 || base > pos + tok1 - a.window || base + kKvBlock <= a.sinks);
    unsigned seen[QT];   // bit 4 n + j: this lane's token (n, j) is visible to its row
    if (!full) {
#pragma unroll
      for (int i = 0; i < QT; ++i) {
        seen[i] = 0u;
#pragma unroll
        for (int n = 0; n < 4; ++n)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const long tok = base + 16 * g + 4 * n + j;
            const bool vis = tok <= prow[i] && (a.window == 0 || tok > prow[i] - a.window || tok < a.sinks);
            seen[i] |= vis ? 1u << (4 * n + j) : 0u;
            s[i][n][j] = vis ? s[i][n][j] : -INFINITY;
          }
      }
    }
    h8v p[QT][2];
    const float fev = (float)ev, inv = pow2i(-ev);
#pragma unroll
    for (int i = 0; i < QT; ++i) {
      float x = s[i][0][0];
#pragma unroll
      for (int n = 0; n < 4; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) x = fmaxf(x, s[i][n][j]);
      x = fmaxf(x, __shfl_xor(x, 16));
      x = fmaxf(x, __shfl_xor(x, 32));
      const float mn = fmaxf(m[i], __builtin_fmaf(x, fac, fev));
      const float al = __builtin_amdgcn_exp2f(m[i] - mn);
      m[i] = mn;
      const float sub = kProbExp + fev - mn;
      float ps = 0.f;
#pragma unroll
      for (int n = 0; n < 4; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float y = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i][n][j], fac, sub));
          ps += y;
          p[i][n / 2][4 * (n & 1) + j] = (_Float16)y;
        }
      l[i] = __builtin_fmaf(ps, inv, l[i] * al);
#pragma unroll
      for (int d = 0; d < 8; ++d) o[i][d] *= al;
    }
    // A NaN among the V rows must reach the rows that see it and no others,
    // though a masked probability times it would be NaN: such tiles (only masked
    // ones need it) multiply with the NaN bytes as zeros and mark afterwards.
    bool marked = false;
    if (!full) {
      unsigned any = 0u;
#pragma unroll
      for (int d = 0; d < 8; ++d)
#pragma unroll
        for (int x = 0; x < 4; ++x) any |= nan_bytes(vr[d][x]);
      marked = __any(any != 0u);
    }
    if (marked) {
      h8v vis[QT][2];
#pragma unroll
      for (int i = 0; i < QT; ++i)
#pragma unroll
        for (int n = 0; n < 4; ++n)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            vis[i][n / 2][4 * (n & 1) + j] = (seen[i] >> (4 * n + j)) & 1u ? (_Float16)1.f : (_Float16)0.f;
#pragma unroll
      for (int d = 0; d < 8; ++d) {
        f32x4 cnt[QT];
#pragma unroll
        for (int i = 0; i < QT; ++i) cnt[i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
          h8v f;
#pragma unroll
          for (int e = 0; e < 8; ++e)
            f[e] = (nan_bytes(vr[d][2 * ks + e / 4]) >> (8 * (e & 3) + 7)) & 1u ? (_Float16)1.f : (_Float16)0.f;
#pragma unroll
          for (int i = 0; i < QT; ++i) cnt[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f, vis[i][ks], cnt[i], 0, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < QT; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (cnt[i][j] > 0.f) o[i][d][j] = NAN;
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const unsigned nb = nan_bytes(vr[d][x]);
          vr[d][x] &= ~((nb >> 7) * 0xffu);
        }
      }
    }
#pragma unroll
    for (int d = 0; d < 8; ++d)
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
        const h8v vf = fp8x8_to_f16(vr[d][2 * ks], vr[d][2 * ks + 1]);
#pragma unroll
        for (int i = 0; i < QT; ++i) o[i][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, p[i][ks], o[i][d], 0, 0, 0);
      }
  }

  // join the waves (fixed order)
#pragma unroll
  for (int i = 0; i < QT; ++i) {
    l[i] += __shfl_xor(l[i], 16);
    l[i] += __shfl_xor(l[i], 32);
    if (g == 0) {
      s_ml[w][16 * i + c][0] = m[i];
      s_ml[w][16 * i + c][1] = l[i];
    }
#pragma unroll
    for (int d = 0; d < 8; ++d) *reinterpret_cast<f32x4*>(&s_o[w][16 * i + c][16 * d + 4 * g]) = o[i][d];
  }
  __syncthreads();
  for (int n = threadIdx.x; n < 16 * QT * (kHD / 4); n += kWave * NW) {
    const int rr = n / (kHD / 4), d = 4 * (n % (kHD / 4)), r = r0 + rr;
    if (r >= R) continue;
    float mm = s_ml[0][rr][0];
#pragma unroll
    for (int x = 1; x < NW; ++x) mm = fmaxf(mm, s_ml[x][rr][0]);
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    float ll = 0.f;
#pragma unroll
    for (int x = 0; x < NW; ++x) {
      const float f = __builtin_amdgcn_exp2f(s_ml[x][rr][0] - mm);
      ll = __builtin_fmaf(s_ml[x][rr][1], f, ll);
      acc += *reinterpret_cast<const f32x4*>(&s_o[x][rr][d]) * f;
    }
    if (a.n_split > 1) {
      const long pr = ((long)bh * a.n_split + blockIdx.x) * R + r;
      *reinterpret_cast<f32x4*>(a.part_o + pr * kHD + d) = acc;
      if (d == 0) {
        a.part_ml[2 * pr] = mm;
        a.part_ml[2 * pr + 1] = ll;
      }
      continue;
    }
    const float il = ll == 0.f ? 0.f : 1.f / ll;
    const long row = ((long)b * a.Sq + r / a.G) * a.c.Hkv * a.G + kvh * a.G + r % a.G;
    *reinterpret_cast<u32x2*>(a.out + row * kHD + d) = u32x2{pack2(acc.x * il, acc.y * il), pack2(acc.z * il, acc.w * il)};
  }
}

// The splits' partials of two rows per workgroup, in order.
__global__ __launch_bounds__(64) void attention_fp8_merge_kernel(const AttnFp8Args a) {
  const int R = a.Sq * a.G;
  const long idx = (long)blockIdx.x * 2 + threadIdx.x / 32;   // (bh, r)
  if (idx >= (long)a.c.B * a.c.Hkv * R) return;
  const long bh = idx / R;
  const int r = (int)(idx % R), d = 4 * (threadIdx.x & 31);
  const long p0 = bh * a.n_split * R + r;
  float mm = kLowest;
  for (int s = 0; s < a.n_split; ++s) mm = fmaxf(mm, a.part_ml[2 * (p0 + (long)s * R)]);
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  float ll = 0.f;
#pragma unroll 8
  for (int s = 0; s < a.n_split; ++s) {
    const long p = p0 + (long)s * R;
    const float f = __builtin_amdgcn_exp2f(a.part_ml[2 * p] - mm);
    ll = __builtin_fmaf(a.part_ml[2 * p + 1], f, ll);
    acc += *reinterpret_cast<const f32x4*>(a.part_o + p * kHD + d) * f;
  }
  const float il = ll == 0.f ? 0.f : 1.f / ll;
  const int b = (int)(bh / a.c.Hkv), kvh = (int)(bh % a.c.Hkv);
  const long row = ((long)b * a.Sq + r / a.G) * a.c.Hkv * a.G + kvh * a.G + r % a.G;
  *reinterpret_cast<u32x2*>(a.out + row * kHD + d) = u32x2{pack2(acc.x * il, acc.y * il), pack2(acc.z * il, acc.w * il)};
}

int attention_fp8_splits(int B, int Hkv, int Sq, int G, int T, int window, int sinks) {
  long tiles = T / kKvBlock;
  if (window > 0) tiles = min(tiles, ((long)window + Sq + 2 * kKvBlock) / kKvBlock + ((long)sinks + kKvBlock - 1) / kKvBlock);
  const long units = (long)B * Hkv * (((long)Sq * G + 15) / 16);
  long n = (512 + units - 1) / units;
  n = min(n, (tiles + 3) / 4);
  return (int)max(1L, min(n, 64L));
}

int attention_fp8_launch(const AttnFp8Args& a, hipStream_t s) {
  const int R = a.Sq * a.G;
  const dim3 grid((unsigned)a.n_split, (unsigned)((R + 15) / 16), (unsigned)(a.c.B * a.c.Hkv));
  hipLaunchKernelGGL((attention_fp8_kernel<1, 4>), grid, dim3(256), 0, s, a);
  int st = qd_host::launch_status("attention_fp8_kernel");
  if (st != QD_OK || a.n_split == 1) return st;
  const long rows = (long)a.c.B * a.c.Hkv * R;
  hipLaunchKernelGGL(attention_fp8_merge_kernel, dim3((unsigned)((rows + 1) / 2)), dim3(64), 0, s, a);
  return qd_host::launch_status("attention_fp8_merge_kernel");
}

}  // namespace qd
