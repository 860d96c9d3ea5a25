// Block-scaled 8-bit product for gfx950:
//   y[m][n] = sum over 128-column blocks b of 2^(ex[m][b] + ew[n / 128][b])
//             sum over k in b of x[m][k] w[n][k]
// with e4m3 values and power-of-two scales.
//
// Two kinds of sums.  The fp8 matrix instructions add the products of 8 neighbouring
// k with 14 bits: whatever lies below 2^-13 of the largest of the eight is cut
// (measured product by product; the groups' sums are fp32).  The fp16 ones, on the
// same values converted exactly in registers, sum in fp32 throughout, at half
// the rate.  So fp32 results, and few rows, where the weight's bytes are the bound
// anyway, take the fp16 ones; fp16 results of many rows the fp8 ones (error 4e-6 of
// the result on N(0, 1) operands, 2^-11 is half a step of the result's type), whose
// scaled form applies both block exponents by itself.  (151936 x 2048 by 8 rows: the
// same 58 us either way; 4001 x 12288 x 2048: 101 us, in fp32 sums 213.)
//
// The k order inside a block is free (both operands use the same one): a lane
// holds bytes [16 g, 16 g + 16) and [64 + 16 g, ...) of its row's block.  W is the MFMA's A
// operand, so a lane holds four consecutive outputs of one row of x.

#include <math.h>

#include <algorithm>
#include <type_traits>

#include "qd_fp8.h"

namespace qd {

namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));

// One 128-column block of a 16 x 16 tile in fp32 sums: four fp16 MFMAs.
__device__ __forceinline__ f32x4 block_f16(const h8v (&w)[4], const h8v (&x)[4]) {
  f32x4 t = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int ks = 0; ks < 4; ++ks) t = __builtin_amdgcn_mfma_f32_16x16x32_f16(w[ks], x[ks], t, 0, 0, 0);
  return t;
}
__device__ __forceinline__ void widen_block(const u32x4 lo, const u32x4 hi, h8v (&o)[4]) {
  o[0] = fp8x8_to_f16(lo.x, lo.y);
  o[1] = fp8x8_to_f16(lo.z, lo.w);
  o[2] = fp8x8_to_f16(hi.x, hi.y);
  o[3] = fp8x8_to_f16(hi.z, hi.w);
}
// 2^(a + b) of two E8M0 bytes (0 or infinity past fp32's range).
__device__ __forceinline__ float scale_of(int a, int b) { return ldexpf(1.f, a + b - 254); }

__device__ __forceinline__ void store4(float* y, long m, long N, int n, const f32x4 v) {
  if (n + 3 < N && (N & 3) == 0) {
    *reinterpret_cast<f32x4*>(y + m * N + n) = v;
    return;
  }
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (n + j < N) y[m * N + n + j] = v[j];
}
__device__ __forceinline__ void store4(uint16_t* y, long m, long N, int n, const f32x4 v) {
  if (n + 3 < N && (N & 3) == 0) {
    *reinterpret_cast<u32x2*>(y + m * N + n) = u32x2{pack2(v.x, v.y), pack2(v.z, v.w)};
    return;
  }
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (n + j < N) y[m * N + n + j] = f2h(v[j]);
}

}  // namespace

// ---------------------------------------------------------------- few rows

// Bound by the weight's bytes.  One workgroup of KS waves per 16 rows of W and 16 MT
// of x; the waves share the K blocks, U at a time in flight, and add up through
// LDS in order.  W goes from memory to the MFMA without LDS.
// 4096 x 2048 by one row: 3.8 us, of which the 8.4 MB are 1.7; the rest is the launch, the
// first loads and the join.
template <int MT, int KS, int U, typename TO>
__global__ __launch_bounds__(kWave * KS) void gemm_fp8_rows_kernel(const GemmFp8Args a) {
  const int lane = lane_id();
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int c = lane & 15, g = lane >> 4;
  const int n0 = (int)blockIdx.x * 16, m0 = (int)blockIdx.y * 16 * MT;
  const int kb_n = (a.K + kScaleCols - 1) / kScaleCols;
  const int kb0 = kb_n * w / KS, kb1 = kb_n * (w + 1) / KS;
  const uint8_t* wr = a.w + (long)min(n0 + c, a.N - 1) * a.K;
  const uint8_t* ws = a.w_scale + (long)(n0 / kScaleCols) * kb_n;
  const uint8_t* xr[MT];
  const uint8_t* xs[MT];
  f32x4 acc[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const long m = min(m0 + 16 * i + c, a.M - 1);
    xr[i] = a.x + m * a.K;
    xs[i] = a.x_scale + m * kb_n;
    acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  for (int kb = kb0; kb < kb1; kb += U) {
    u32x4 fw[U][2], fx[U][MT][2];
    int sw[U], sx[U][MT];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int b = min(kb + u, kb1 - 1);
      const int k = b * kScaleCols + 16 * g;
      // a chunk past K (a multiple of 16) repeats the row's last one, W's as zeros
      const int k0 = min(k, a.K - 16), k1 = min(k + 64, a.K - 16);
      fw[u][0] = ld16(wr + k0);
      fw[u][1] = ld16(wr + k1);
      sw[u] = ws[b];
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        fx[u][i][0] = ld16(xr[i] + k0);
        fx[u][i][1] = ld16(xr[i] + k1);
        sx[u][i] = xs[i][b];
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (kb + u >= kb1) break;
      const int k = (kb + u) * kScaleCols + 16 * g;
      const u32x4 zero = {0u, 0u, 0u, 0u};
      h8v hw[4];
      widen_block(k < a.K ? fw[u][0] : zero, k + 64 < a.K ? fw[u][1] : zero, hw);
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        h8v hx[4];
        widen_block(fx[u][i][0], fx[u][i][1], hx);
        acc[i] += block_f16(hw, hx) * scale_of(sw[u], sx[u][i]);
      }
    }
  }
  TO* y = reinterpret_cast<TO*>(a.y);
  if constexpr (KS > 1) {
    __shared__ f32x4 s_acc[KS][MT][kWave];
#pragma unroll
    for (int i = 0; i < MT; ++i) s_acc[w][i][lane] = acc[i];
    __syncthreads();
    for (int i = w; i < MT; i += KS) {
      f32x4 v = s_acc[0][i][lane];
#pragma unroll
      for (int x = 1; x < KS; ++x) v += s_acc[x][i][lane];
      const int m = m0 + 16 * i + c;
      if (m < a.M) store4(y, m, a.N, n0 + 4 * g, v);
    }
  } else {
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      const int m = m0 + 16 * i + c;
      if (m < a.M) store4(y, m, a.N, n0 + 4 * g, acc[i]);
    }
  }
}

// At most 16 rows of x and 8 KBW blocks of K: eight waves share the K blocks, each keeps
// its part of x in registers, converted, and the workgroup passes over the weight's
// rows, RG groups of 16 at a time, the next groups' bytes in flight.  (Reading x again
// for every 16 rows of W costs as many loads as W itself: 8 rows of the 151936 x 2048
// lm_head 69 us, kept in registers 58, 5.4 TB/s.)
template <int KBW, int RG, typename TO>
__global__ __launch_bounds__(512) void gemm_fp8_stream_kernel(const GemmFp8Args a) {
  constexpr int KS = 8;
  __shared__ f32x4 s_acc[2][RG][KS][kWave];
  const int lane = lane_id();
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int c = lane & 15, g = lane >> 4;
  const int kb_n = (a.K + kScaleCols - 1) / kScaleCols;
  const int kb0 = kb_n * w / KS, kb1 = kb_n * (w + 1) / KS;
  const int groups = (a.N + 16 * RG - 1) / (16 * RG);
  h8v hx[KBW][4];
  int sx[KBW];
  unsigned koff[KBW][2];
  int kbs[KBW];
#pragma unroll
  for (int u = 0; u < KBW; ++u) {
    // a block or chunk that the wave or the row does not have: zeros of x times
    // some other bytes of the same row of W
    const bool mine = kb0 + u < kb1;
    const int kb = min(kb0 + u, kb_n - 1), k = kb * kScaleCols + 16 * g;
    kbs[u] = kb;
    koff[u][0] = min(k, a.K - 16);
    koff[u][1] = min(k + 64, a.K - 16);
    const uint8_t* xr = a.x + (long)min(c, a.M - 1) * a.K;
    const u32x4 zero = {0u, 0u, 0u, 0u};
    widen_block(mine && k < a.K ? ld16(xr + koff[u][0]) : zero, mine && k + 64 < a.K ? ld16(xr + koff[u][1]) : zero, hx[u]);
    sx[u] = mine ? a.x_scale[(long)min(c, a.M - 1) * kb_n + kb] : -(1 << 20);   // (2^sx = 0)
  }
  u32x4 fw[2][RG][KBW][2];
  int sw[2][RG][KBW];
  auto load = [&](auto B, int grp) __attribute__((always_inline)) {
    constexpr int x = decltype(B)::value;
#pragma unroll
    for (int i = 0; i < RG; ++i) {
      const int n0 = min(grp, groups - 1) * 16 * RG + 16 * i;
      const uint8_t* wr = a.w + (long)min(n0 + c, a.N - 1) * a.K;
      const uint8_t* ws = a.w_scale + (long)(min(n0, a.N - 1) / kScaleCols) * kb_n;
#pragma unroll
      for (int u = 0; u < KBW; ++u) {
        fw[x][i][u][0] = ld16(wr + koff[u][0]);
        fw[x][i][u][1] = ld16(wr + koff[u][1]);
        sw[x][i][u] = ws[kbs[u]];
      }
    }
  };
  TO* y = reinterpret_cast<TO*>(a.y);
  auto pass = [&](auto B, int grp) __attribute__((always_inline)) {
    constexpr int x = decltype(B)::value;
    load(std::integral_constant<int, 1 - x>{}, grp + (int)gridDim.x);
#pragma unroll
    for (int i = 0; i < RG; ++i) {
      f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int u = 0; u < KBW; ++u) {
        h8v hw[4];
        widen_block(fw[x][i][u][0], fw[x][i][u][1], hw);
        acc += block_f16(hw, hx[u]) * scale_of(sw[x][i][u], sx[u]);
      }
      s_acc[x][i][w][lane] = acc;
    }
    __syncthreads();   // (the other buffer's readers are past the barrier before this one)
    if (w < RG) {
      f32x4 v = s_acc[x][w][0][lane];
#pragma unroll
      for (int z = 1; z < KS; ++z) v += s_acc[x][w][z][lane];
      const int n = grp * 16 * RG + 16 * w + 4 * g;
      if (c < a.M && n < a.N) store4(y, c, a.N, n, v);
    }
  };
  const std::integral_constant<int, 0> b0;
  const std::integral_constant<int, 1> b1;
  int grp = blockIdx.x;
  load(b0, grp);
#pragma unroll 1
  for (; grp < groups; grp += 2 * gridDim.x) {
    pass(b0, grp);
    if (grp + (int)gridDim.x >= groups) break;
    pass(b1, grp + gridDim.x);
  }
}

// ---------------------------------------------------------------- many rows

namespace {

// What the chunks of W past K read.
__device__ const u32x4 kZeros = {0u, 0u, 0u, 0u};

__device__ __forceinline__ void load_lds16(const void* g, void* l) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)g,
                                   (__attribute__((address_space(3))) void*)l, 16, 0, 0);
}

// At most N of this wave's loads are in flight and its LDS accesses are done, then
// the workgroup barrier.
template <int N>
__device__ __forceinline__ void wait_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | 0x0070);   // vmcnt(N) lgkmcnt(0)
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("" ::: "memory");
}

// The stages are separate variables: the compiler then knows that reading one does
// not depend on the loads in flight to another.
template <int I, int N>
__device__ __forceinline__ char* tile_stage() {
  __shared__ __align__(16) char buf[N];
  return buf;
}

// One tile per workgroup, tiles of one W band after another within an XCD: the m
// tiles of a band share its rows, which then come out of that XCD's L2.
__device__ __forceinline__ int tile_of_block() {
  const int q = (int)gridDim.x >> 3, r = (int)gridDim.x & 7, xcd = (int)blockIdx.x & 7, loc = (int)blockIdx.x >> 3;
  return xcd * q + min(xcd, r) + loc;
}

}  // namespace

// Tile BM (rows of x) x BN (rows of W), one K block of 128 bytes per row and stage,
// NS stages filled by asynchronous global-to-LDS loads NS - 1 steps ahead; WM x WN
// waves.  16-byte chunk c of row r sits at c ^ (r % 8); the permutation is applied to
// the source address, since the load's LDS side is contiguous.
//
// Scales come with their stage, as the aligned words that hold them (up to 3 bytes of a
// word are a neighbour's; a word never leaves its scale's allocation): each wave loads
// one word per lane, lane l < BM / waves the one of its l-th row of x, the others W's.
//
// TAIL: the last block is partial (K is a multiple of 16); a chunk past K repeats
// the row's last one, W's is zeros.
template <int BM, int BN, int WM, int WN, int NS, bool TAIL, bool F8, typename TO>
__global__ __launch_bounds__(kWave * WM * WN) void gemm_fp8_tile_kernel(const GemmFp8Args a) {
  constexpr int NW = WM * WN, TM = BM / WM, TN = BN / WN, I = TM / 16, J = TN / 16;
  constexpr int GA = BM / 8, GW = BN / 8, LA = GA / NW, LW = GW / NW, LOADS = LA + LW + 1;   // loads of 8 rows, per wave
  constexpr int SR = BM / NW;   // rows of x whose scales a wave loads
  constexpr int SCALES = (BM + BN) * kScaleCols, STAGE = SCALES + NW * kWave * 4;
  static_assert(GA % NW == 0 && GW % NW == 0 && TM % 16 == 0 && TN % 16 == 0 && SR < kWave && BN <= kScaleCols &&
                    LOADS * (NS - 2) < 64 && (NS == 2 || NS == 3 || NS == 4),
                "tile shape");
  const int lane = lane_id();
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int tiles_m = (a.M + BM - 1) / BM, t = tile_of_block();
  const int m0 = (t % tiles_m) * BM, n0 = (t / tiles_m) * BN;
  const int kb_n = (a.K + kScaleCols - 1) / kScaleCols;
  const int lr = lane >> 3, chunk = 16 * ((lane & 7) ^ lr);
  // 32-bit offsets from the tile's first row (BM rows of K <= 2^23 bytes)
  const uint8_t* xb = a.x + (long)m0 * a.K;
  const uint8_t* wb = a.w + (long)n0 * a.K;
  unsigned offA[LA], offW[LW];
#pragma unroll
  for (int i = 0; i < LA; ++i) offA[i] = (unsigned)min((i * NW + w) * 8 + lr, a.M - 1 - m0) * (unsigned)a.K + chunk;
#pragma unroll
  for (int i = 0; i < LW; ++i) offW[i] = (unsigned)min((i * NW + w) * 8 + lr, a.N - 1 - n0) * (unsigned)a.K + chunk;
  const uint8_t* sp = lane < SR ? a.x_scale + (long)min(m0 + w * SR + lane, a.M - 1) * kb_n
                                : a.w_scale + (long)(n0 / kScaleCols) * kb_n;
  // (a block past the last is loaded like the last one, so that every step issues the
  // same number, and not used)
  auto issue = [&](auto S, int block) __attribute__((always_inline)) {
    char* st = tile_stage<decltype(S)::value, STAGE>();
    const int kb = min(block, kb_n - 1);
    const unsigned k = (unsigned)kb * kScaleCols;
    const bool past = TAIL && (int)k + chunk >= a.K;
    const unsigned ka = past ? a.K - 16 - chunk : k;
#pragma unroll
    for (int i = 0; i < LA; ++i) load_lds16(xb + (offA[i] + ka), st + (i * NW + w) * 1024);
#pragma unroll
    for (int i = 0; i < LW; ++i)
      load_lds16(past ? reinterpret_cast<const uint8_t*>(&kZeros) : wb + (offW[i] + k), st + BM * kScaleCols + (i * NW + w) * 1024);
    const uintptr_t at = reinterpret_cast<uintptr_t>(sp + kb);
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(at & ~(uintptr_t)3),
                                     (__attribute__((address_space(3))) void*)(st + SCALES + w * kWave * 4), 4, 0, 0);
  };
  f32x4 acc[I][J];
#pragma unroll
  for (int i = 0; i < I; ++i)
#pragma unroll
    for (int j = 0; j < J; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int wm = w / WN, wn = w % WN, fr = lane & 15, fg = lane >> 4;
  // byte offsets of this lane's two chunks, opaque so that every fragment address
  // stays one base plus a constant
  unsigned bA[2], bW[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const unsigned co = ((4 * h + fg) ^ (fr & 7)) * 16;
    bA[h] = (wm * TM + fr) * kScaleCols + co;
    bW[h] = (BM + wn * TN + fr) * kScaleCols + co;
    asm("" : "+v"(bA[h]));
    asm("" : "+v"(bW[h]));
  }
  // where this lane's scales lie in their words: byte (address + block) % 4
  unsigned sx_at[I], sx_lo[I];
#pragma unroll
  for (int i = 0; i < I; ++i) {
    const int row = wm * TM + 16 * i + fr;
    sx_at[i] = SCALES + (row / SR) * kWave * 4 + (row % SR) * 4;
    sx_lo[i] = (unsigned)(reinterpret_cast<uintptr_t>(a.x_scale) + (uintptr_t)min(m0 + row, a.M - 1) * (uintptr_t)kb_n) & 3u;
  }
  const unsigned sw_lo = (unsigned)(reinterpret_cast<uintptr_t>(a.w_scale) + (uintptr_t)(n0 / kScaleCols) * (uintptr_t)kb_n) & 3u;
  auto compute = [&](auto S, int kb) __attribute__((always_inline)) {
    const char* st = tile_stage<decltype(S)::value, STAGE>();
    auto frag = [&](const unsigned (&b)[2], int tile, u32x4& lo, u32x4& hi) {
      lo = *reinterpret_cast<const u32x4*>(st + b[0] + tile * 16 * kScaleCols);
      hi = *reinterpret_cast<const u32x4*>(st + b[1] + tile * 16 * kScaleCols);
    };
    auto byte = [&](unsigned at, unsigned lo) {
      return (int)((*reinterpret_cast<const unsigned*>(st + at) >> (8 * ((lo + kb) & 3u))) & 0xffu);
    };
    const int sw = byte(SCALES + (kWave - 1) * 4, sw_lo);
    if constexpr (F8) {
      i32x8 fw[J];
#pragma unroll
      for (int j = 0; j < J; ++j) {
        u32x4 lo, hi;
        frag(bW, j, lo, hi);
        fw[j] = i32x8{(int)lo.x, (int)lo.y, (int)lo.z, (int)lo.w, (int)hi.x, (int)hi.y, (int)hi.z, (int)hi.w};
      }
#pragma unroll
      for (int i = 0; i < I; ++i) {
        u32x4 lo, hi;
        frag(bA, i, lo, hi);
        const i32x8 fx = {(int)lo.x, (int)lo.y, (int)lo.z, (int)lo.w, (int)hi.x, (int)hi.y, (int)hi.z, (int)hi.w};
        const int sx = byte(sx_at[i], sx_lo[i]);
#pragma unroll
        for (int j = 0; j < J; ++j)
          acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fw[j], fx, acc[i][j], 0, 0, 0, sw, 0, sx);
      }
    } else {
      h8v hw[J][4];
#pragma unroll
      for (int j = 0; j < J; ++j) {
        u32x4 lo, hi;
        frag(bW, j, lo, hi);
        widen_block(lo, hi, hw[j]);
      }
#pragma unroll
      for (int i = 0; i < I; ++i) {
        u32x4 lo, hi;
        frag(bA, i, lo, hi);
        h8v hx[4];
        widen_block(lo, hi, hx);
        const float f = scale_of(sw, byte(sx_at[i], sx_lo[i]));
        f32x4 blk[J];
#pragma unroll
        for (int j = 0; j < J; ++j) blk[j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < 4; ++ks)
#pragma unroll
          for (int j = 0; j < J; ++j) blk[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(hw[j][ks], hx[ks], blk[j], 0, 0, 0);
#pragma unroll
        for (int j = 0; j < J; ++j) acc[i][j] += blk[j] * f;
      }
    }
  };
  // (no branch inside a step: the compiler would move products past it, behind the
  // next wait)
  auto step = [&](auto S, int kb) __attribute__((always_inline)) {
    wait_barrier<LOADS*(NS - 2)>();   // block kb is there, the stage refilled next is read
    issue(std::integral_constant<int, (decltype(S)::value + NS - 1) % NS>{}, kb + NS - 1);
    compute(S, kb);
  };
  const std::integral_constant<int, 0> s0;
  const std::integral_constant<int, 1> s1;
  const std::integral_constant<int, NS == 2 ? 0 : 2> s2;   // (the second round of two)
  const std::integral_constant<int, NS == 2 ? 1 : NS - 1> s3;
  issue(s0, 0);
  if constexpr (NS > 2) issue(s1, 1);
  if constexpr (NS > 3) issue(s2, 2);
  constexpr int ROUND = NS == 3 ? 3 : 4;
  int kb = 0;
#pragma unroll 1
  for (; kb + ROUND <= kb_n; kb += ROUND) {
    step(s0, kb);
    step(s1, kb + 1);
    step(s2, kb + 2);
    if constexpr (ROUND == 4) step(s3, kb + 3);
  }
  if (kb < kb_n) step(s0, kb);
  if (kb + 1 < kb_n) step(s1, kb + 1);
  if (ROUND == 4 && kb + 2 < kb_n) step(s2, kb + 2);
  TO* y = reinterpret_cast<TO*>(a.y);
#pragma unroll
  for (int i = 0; i < I; ++i) {
    const int m = m0 + wm * TM + 16 * i + fr;
    if (m < a.M) {
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const int n = n0 + wn * TN + 16 * j + 4 * fg;
        if (n < a.N) store4(y, m, a.N, n, acc[i][j]);
      }
    }
  }
  wait_barrier<0>();   // (the loads past the last block go to LDS that is still this workgroup's)
}

// ---------------------------------------------------------------- large products, fp16 results

namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kBigK = 64;           // k per stage
constexpr int kBigMaxBlocks = 56;   // K blocks whose scales fit the LDS of two workgroups per CU

}  // namespace

// Tile BM x BN, four waves of BM / 2 x BN / 2, fp8 products of 32 x 32 x 64.
//
// Three stages of 64 k.  In step k the products use fragments that were read from LDS
// during step k - 1, the fragments of step k + 1 are read, stage k + 2 is in flight and
// stage k + 3 is issued into the place of stage k: neither loads nor LDS reads stand
// between two steps' products.  Scales lie in LDS, [block][row].
//
// 16-byte chunk c of row r (64 bytes) sits at c ^ (r / 2 % 4).  K is a multiple of 64.
//
// 4001 x 12288 x 2048 in 256 x 256: 101 us, 2.0 PFLOP/s, 81 % of an 8192-cubed library product
// here (2.46).  A step of 64 k takes 0.67 us, 3.2 PFLOP/s over the card; each of the three
// rounds of tiles adds some 9 us for its first loads and its results, which nothing
// overlaps.  (128 x 256 two per CU 116 us; 256 x 256 with W from memory to
// registers 137; the fp16 MFMAs 213.  One workgroup per CU for several tiles, the next one's
// stages loaded before this one's results are stored: 116, since a wave's loads
// complete behind its earlier stores, which a new workgroup's do not.)
template <int BM, int BN, int OCC>
__global__ __launch_bounds__(256, OCC) void gemm_fp8_big_kernel(const GemmFp8Args a) {
  constexpr int TM = BM / 2, TN = BN / 2, I = TM / 32, J = TN / 32;
  constexpr int LA = BM / 64, LW = BN / 64, LOADS = LA + LW;   // loads of 16 rows, per wave
  constexpr int STAGE = (BM + BN) * kBigK;
  static_assert(BM <= 256 && TN <= kScaleCols, "tile shape");
  __shared__ uint8_t s_sx[kBigMaxBlocks][BM];
  __shared__ uint8_t s_sw[kBigMaxBlocks][2];
  const int lane = lane_id();
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int tiles_m = (a.M + BM - 1) / BM, t = tile_of_block();
  const int m0 = (t % tiles_m) * BM, n0 = (t / tiles_m) * BN;
  const int kb_n = (a.K + kScaleCols - 1) / kScaleCols, steps = a.K / kBigK;
  const int lr = lane >> 2, chunk = 16 * ((lane & 3) ^ ((lr >> 2) & 3));
  const int wm = w >> 1, wn = w & 1, fr = lane & 31, fh = lane >> 5;
  // 32-bit offsets from the tile's first row
  const uint8_t* xb = a.x + (long)m0 * a.K;
  const uint8_t* wb = a.w + (long)n0 * a.K;
  unsigned offA[LA], offW[LW];
#pragma unroll
  for (int i = 0; i < LA; ++i) offA[i] = (unsigned)min((i * 4 + w) * 16 + lr, a.M - 1 - m0) * (unsigned)a.K + chunk;
#pragma unroll
  for (int i = 0; i < LW; ++i) offW[i] = (unsigned)min((i * 4 + w) * 16 + lr, a.N - 1 - n0) * (unsigned)a.K + chunk;
  // a stage past the last is loaded like the last one (so that every step issues the
  // same number) and not used
  auto issue = [&](auto S, int st) __attribute__((always_inline)) {
    char* p = tile_stage<8 + decltype(S)::value, STAGE>();
    const unsigned k = (unsigned)min(st, steps - 1) * kBigK;
#pragma unroll
    for (int i = 0; i < LA; ++i) load_lds16(xb + (offA[i] + k), p + (i * 4 + w) * 1024);
#pragma unroll
    for (int i = 0; i < LW; ++i) load_lds16(wb + (offW[i] + k), p + BM * kBigK + (i * 4 + w) * 1024);
  };
  const std::integral_constant<int, 0> s0;
  const std::integral_constant<int, 1> s1;
  const std::integral_constant<int, 2> s2;
  issue(s0, 0);
  issue(s1, 1);
  issue(s2, 2);
  {
    const int row = threadIdx.x;
    if (row < BM) {
      const uint8_t* sx = a.x_scale + (long)min(m0 + row, a.M - 1) * kb_n;
      int b = 0;
      if ((kb_n & 15) == 0 && (reinterpret_cast<uintptr_t>(a.x_scale) & 15) == 0) {
        for (; b < kb_n; b += 16) {
          const u32x4 v = ld16(sx + b);
#pragma unroll
          for (int e = 0; e < 16; ++e) s_sx[b + e][row] = (uint8_t)(v[e / 4] >> (8 * (e & 3)));
        }
      }
#pragma unroll 8
      for (; b < kb_n; ++b) s_sx[b][row] = sx[b];
    }
    // the two halves of the tile's W rows
    for (int b = row; b < 2 * kb_n; b += 256) {
      const int h = b / kb_n, n = min(n0 + h * TN, a.N - 1);
      s_sw[b - h * kb_n][h] = a.w_scale[(long)(n / kScaleCols) * kb_n + b - h * kb_n];
    }
  }

  // this lane's two chunks fh and 2 + fh of its row (the second at ^ 32)
  const unsigned co = 16 * (fh ^ ((fr >> 2) & 3));
  unsigned bA = (wm * TM + fr) * kBigK + co, bW = (BM + wn * TN + fr) * kBigK + co;
  asm("" : "+v"(bA));
  asm("" : "+v"(bW));
  f32x16 acc[I][J];
#pragma unroll
  for (int i = 0; i < I; ++i)
#pragma unroll
    for (int j = 0; j < J; ++j) {
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
      if constexpr (OCC == 1)
        asm volatile("" : "+a"(acc[i][j]));   // (cleared here, while the first loads are on their way)
      else
        asm volatile("" : "+v"(acc[i][j]));
    }
  i32x8 fx[2][I], fw[2][J];
  int sx[2][I], sw[2];
  auto read = [&](auto S, auto F, int st) __attribute__((always_inline)) {   // fragments and scales of step st
    const char* p = tile_stage<8 + decltype(S)::value, STAGE>();
    constexpr int f = decltype(F)::value;
    auto frag = [&](unsigned b, int tile) {
      const u32x4 lo = *reinterpret_cast<const u32x4*>(p + b + tile * 32 * kBigK);
      const u32x4 hi = *reinterpret_cast<const u32x4*>(p + (b ^ 32) + tile * 32 * kBigK);
      return i32x8{(int)lo.x, (int)lo.y, (int)lo.z, (int)lo.w, (int)hi.x, (int)hi.y, (int)hi.z, (int)hi.w};
    };
    const int kb = min(st, steps - 1) >> 1;
#pragma unroll
    for (int j = 0; j < J; ++j) fw[f][j] = frag(bW, j);
#pragma unroll
    for (int i = 0; i < I; ++i) {
      fx[f][i] = frag(bA, i);
      sx[f][i] = s_sx[kb][wm * TM + 32 * i + fr];
    }
    sw[f] = s_sw[kb][wn];
  };
  // stage N holds step st + 1; S, whose fragments are in F, is refilled
  auto step = [&](auto S, auto N, auto F, int st) __attribute__((always_inline)) {
    constexpr int f = decltype(F)::value;
    wait_barrier<LOADS>();   // stage st + 1 is there (st + 2 in flight), S is read
    issue(S, st + 3);
    read(N, std::integral_constant<int, 1 - f>{}, st + 1);
#pragma unroll
    for (int i = 0; i < I; ++i)
#pragma unroll
      for (int j = 0; j < J; ++j)
        acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(fw[f][j], fx[f][i], acc[i][j], 0, 0, 0, sw[f], 0, sx[f][i]);
    // products first, and between any two of them a load and one or two LDS reads: a
    // run of LDS reads would hold the wave, and its products, at the LDS queue
    // (256 x 256 tiles: 0.85 us a step, interleaved 0.67)
#pragma unroll
    for (int i = 0; i < I * J / 2; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);   // MFMA
      __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);   // LDS reads
      __builtin_amdgcn_sched_group_barrier(0x020, I * J >= 2 * LOADS ? 1 : 2, 0);   // global reads
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, I * J >= 16 ? 1 : 2, 0);
    }
  };
  wait_barrier<0>();   // the first three stages and the scales
  read(s0, s0, 0);
  int st = 0;
#pragma unroll 1
  for (; st + 5 < steps; st += 6) {
    step(s0, s1, s0, st);
    step(s1, s2, s1, st + 1);
    step(s2, s0, s0, st + 2);
    step(s0, s1, s1, st + 3);
    step(s1, s2, s0, st + 4);
    step(s2, s0, s1, st + 5);
  }
  if (st < steps) step(s0, s1, s0, st);
  if (st + 1 < steps) step(s1, s2, s1, st + 1);
  if (st + 2 < steps) step(s2, s0, s0, st + 2);
  if (st + 3 < steps) step(s0, s1, s1, st + 3);
  if (st + 4 < steps) step(s1, s2, s0, st + 4);
  uint16_t* y = reinterpret_cast<uint16_t*>(a.y);
  wait_barrier<0>();   // all fragments are read and the loads past the last stage are done
  if (a.N % 8 != 0) {
#pragma unroll
    for (int i = 0; i < I; ++i) {
      const int m = m0 + wm * TM + 32 * i + fr;
#pragma unroll
      for (int j = 0; j < J; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int n = n0 + wn * TN + 32 * j + 8 * e + 4 * fh;
          if (m < a.M && n < a.N)
            store4(y, m, a.N, n, f32x4{acc[i][j][4 * e], acc[i][j][4 * e + 1], acc[i][j][4 * e + 2], acc[i][j][4 * e + 3]});
        }
    }
    return;
  }
  // through LDS, 32 rows of the wave's at a time, so that stores are rows of 2 TN
  // bytes: chunk c of row r at c ^ (r % chunks)
  constexpr int C = TN / 8, RPS = kWave / C;   // chunks of a row, rows per store
  char* mine = (wm == 0 ? tile_stage<8, STAGE>() : tile_stage<9, STAGE>()) + wn * 32 * TN * 2;
  static_assert(2 * 32 * TN * 2 <= STAGE && C <= 16, "store staging");
#pragma unroll
  for (int i = 0; i < I; ++i) {
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const f32x16& v = acc[i][j];
        *reinterpret_cast<u32x2*>(mine + fr * (TN * 2) + 16 * ((4 * j + e) ^ (fr & (C - 1))) + 8 * fh) =
            u32x2{pack2(v[4 * e], v[4 * e + 1]), pack2(v[4 * e + 2], v[4 * e + 3])};
      }
    const int mr = m0 + wm * TM + 32 * i;
#pragma unroll
    for (int it = 0; it < 32 / RPS; ++it) {
      const int row = RPS * it + lane / C, c = (lane & (C - 1)) ^ (row & (C - 1));
      const u32x4 v = *reinterpret_cast<const u32x4*>(mine + row * (TN * 2) + 16 * (lane & (C - 1)));
      const int n = n0 + wn * TN + 8 * c;
      if (mr + row < a.M && n < a.N) *reinterpret_cast<u32x4*>(y + (long)(mr + row) * a.N + n) = v;
    }
  }
}

// ---------------------------------------------------------------- choice

namespace {

template <int MT, int KS, int U, typename TO>
int launch_rows(const GemmFp8Args& a, hipStream_t s) {
  hipLaunchKernelGGL((gemm_fp8_rows_kernel<MT, KS, U, TO>),
                     dim3((unsigned)((a.N + 15) / 16), (unsigned)((a.M + 16 * MT - 1) / (16 * MT))), dim3(kWave * KS), 0,
                     s, a);
  return qd_host::launch_status("gemm_fp8_rows_kernel");
}

template <int KBW, int RG, int WPC, typename TO>
int launch_stream(const GemmFp8Args& a, hipStream_t s) {
  const int groups = (a.N + 16 * RG - 1) / (16 * RG);
  hipLaunchKernelGGL((gemm_fp8_stream_kernel<KBW, RG, TO>), dim3((unsigned)std::min(groups, WPC * qd_host::cu_count())), dim3(512), 0, s, a);
  return qd_host::launch_status("gemm_fp8_stream_kernel");
}

template <int BM, int BN, int WM, int WN, int NS, typename TO>
int launch_tile(const GemmFp8Args& a, hipStream_t s) {
  const unsigned t = (unsigned)(((a.M + BM - 1) / BM) * (long)((a.N + BN - 1) / BN));
  constexpr bool F8 = sizeof(TO) == 2;
  if (a.K % kScaleCols)
    hipLaunchKernelGGL((gemm_fp8_tile_kernel<BM, BN, WM, WN, NS, true, F8, TO>), dim3(t), dim3(kWave * WM * WN), 0, s, a);
  else
    hipLaunchKernelGGL((gemm_fp8_tile_kernel<BM, BN, WM, WN, NS, false, F8, TO>), dim3(t), dim3(kWave * WM * WN), 0, s, a);
  return qd_host::launch_status("gemm_fp8_tile_kernel");
}

template <int BM, int BN, int OCC>
int launch_big(const GemmFp8Args& a, hipStream_t s) {
  const unsigned t = (unsigned)(((a.M + BM - 1) / BM) * (long)((a.N + BN - 1) / BN));
  hipLaunchKernelGGL((gemm_fp8_big_kernel<BM, BN, OCC>), dim3(t), dim3(256), 0, s, a);
  return qd_host::launch_status("gemm_fp8_big_kernel");
}

// Tile shapes and their cost in us: `base` per launch, `ramp` per round of one tile per
// CU, per 128 of K `lat` on a round that is the only one and `us` in a full one.
// Fitted to 63 products of 17 .. 4001 rows, 512 .. 6144 of K (5 to 16 % rms); the
// shape with the least cost is 0.4 % behind the best measured one on average.
// Measured, us, F8 of 512 x 2048 x 6144: 64 x 64 12.3, 128 x 128 (two stages) 42;
// of 4001 x 12288 x 2048: 225, 122, and 256 x 256 of three stages 101.
struct TileCost {
  int bm, bn;
  float base, ramp, us, lat;
};
constexpr TileCost kTilesF8[] = {
    {32, 64, 1.9f, 0.43f, 0.141f, 0.165f},  {64, 64, 1.9f, 0.58f, 0.223f, 0.205f},  {64, 128, 1.8f, 1.08f, 0.309f, 0.332f},
    {128, 128, 0.7f, 1.96f, 0.519f, 0.738f}, {128, 128, 1.9f, 1.17f, 0.553f, 0.438f}, {128, 256, 1.0f, 3.0f, 0.893f, 0.66f},
    {256, 256, 0.0f, 8.1f, 1.387f, 0.916f}};
constexpr TileCost kTilesF16[] = {
    {32, 16, 2.0f, 0.0f, 0.205f, 0.205f},   {64, 64, 1.8f, 0.88f, 0.337f, 0.428f},  {64, 128, 2.0f, 1.36f, 0.561f, 0.66f},
    {128, 128, 0.9f, 2.84f, 0.913f, 1.095f}};

template <int N>
int cheapest(const TileCost (&tiles)[N], int count, const GemmFp8Args& a) {
  const int cus = qd_host::cu_count();
  const float steps = (float)((a.K + kScaleCols - 1) / kScaleCols);
  int best = 0;
  float best_us = 0.f;
  for (int i = 0; i < count; ++i) {
    const TileCost& t = tiles[i];
    const long n = (long)((a.M + t.bm - 1) / t.bm) * ((a.N + t.bn - 1) / t.bn), rounds = (n + cus - 1) / cus;
    const float us = t.base + (rounds == 1 ? t.ramp + steps * t.lat : (float)rounds * (t.ramp + steps * t.us));
    if (i == 0 || us < best_us) {
      best = i;
      best_us = us;
    }
  }
  return best;
}

// Up to 16 rows.  Measured, us: 8 rows of 12288 x 2048 7.3 with x read again, 8.9 kept in
// registers; of 32768 x 2048 15.2 / 14.2, of 151936 x 2048 69 / 58 (4 rows 60 / 59, one 50
// / 58); below 1024 of K the waves have too little each (151936 x 1024, 16 rows: 40 / 42).
template <typename TO>
int launch_few(const GemmFp8Args& a, hipStream_t s) {
  const bool stream = a.K > 1024 && a.K <= 2048 && (long)a.M * a.N >= 250000;
  return stream ? launch_stream<2, 2, 1, TO>(a, s) : launch_rows<1, 8, 2, TO>(a, s);
}

int launch_f8(const GemmFp8Args& a, hipStream_t s) {
  const bool big = a.K % kBigK == 0 && a.K <= kBigMaxBlocks * kScaleCols;
  switch (cheapest(kTilesF8, big ? 7 : 4, a)) {
    case 0: return launch_tile<32, 64, 2, 2, 4, uint16_t>(a, s);
    case 1: return launch_tile<64, 64, 2, 2, 4, uint16_t>(a, s);
    case 2: return launch_tile<64, 128, 2, 2, 3, uint16_t>(a, s);
    case 3: return launch_tile<128, 128, 2, 2, 2, uint16_t>(a, s);
    case 4: return launch_big<128, 128, 2>(a, s);
    case 5: return launch_big<128, 256, 2>(a, s);
    default: return launch_big<256, 256, 1>(a, s);
  }
}

int launch_f16(const GemmFp8Args& a, hipStream_t s) {
  switch (cheapest(kTilesF16, 4, a)) {
    case 0: return launch_rows<2, 8, 2, float>(a, s);
    case 1: return launch_tile<64, 64, 2, 2, 4, float>(a, s);
    case 2: return launch_tile<64, 128, 2, 2, 3, float>(a, s);
    default: return launch_tile<128, 128, 2, 2, 2, float>(a, s);
  }
}

}  // namespace

int gemm_fp8_launch(const GemmFp8Args& a, hipStream_t s) {
  if (a.M <= 16) return a.y_f32 ? launch_few<float>(a, s) : launch_few<uint16_t>(a, s);
  return a.y_f32 ? launch_f16(a, s) : launch_f8(a, s);
}

}  // namespace qd
