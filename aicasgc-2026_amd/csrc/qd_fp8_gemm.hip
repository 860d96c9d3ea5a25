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
// scaled form applies both block exponents by itself.
//
// The k order inside a block is free (both operands use the same one): a lane
// holds bytes [16 g, 16 g + 16) and [64 + 16 g, ...) of its row's block.  W is the MFMA's A
// operand, so a lane holds four consecutive outputs of one row of x.

#include <math.h>

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

// ---------------------------------------------------------------- many rows

namespace {

// What the chunks of W past K read.
__device__ const u32x4 kZeros = {0u, 0u, 0u, 0u};

__device__ __forceinline__ void load_lds16(const void* g, void* l) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)g,
                                   (__attribute__((address_space(3))) void*)l, 16, 0, 0);
}

// This wave's loads and LDS reads are done, then the workgroup barrier.
__device__ __forceinline__ void wait_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_waitcnt(0x0070);   // vmcnt(0) lgkmcnt(0)
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("" ::: "memory");
}

// The two stages are separate variables: the compiler then knows that reading one
// does not depend on the loads in flight to the other.
template <int I, int N>
__device__ __forceinline__ char* tile_stage() {
  __shared__ __align__(16) char buf[N];
  return buf;
}

}  // namespace

// Tile BM (rows of x) x BN (rows of W), one K block of 128 bytes per row and stage,
// two stages filled by asynchronous global-to-LDS loads one step ahead; WM x WN
// waves.  16-byte chunk c of row r sits at c ^ (r % 8), so that the rows a fragment
// read touches spread over the banks; the permutation is applied to the source
// address, since the load's LDS side is contiguous.  Consecutive tiles of one
// XCD share their W rows (the m tiles of one n band), which then come out of its L2.
template <int BM, int BN, int WM, int WN, bool F8, typename TO>
__global__ __launch_bounds__(kWave * WM * WN) void gemm_fp8_tile_kernel(const GemmFp8Args a) {
  constexpr int NW = WM * WN, TM = BM / WM, TN = BN / WN;
  constexpr int GA = BM / 8, GW = BN / 8, LA = GA / NW, LW = GW / NW;   // loads of 8 rows, per wave
  constexpr int STAGE = (BM + BN) * kScaleCols;
  static_assert(GA % NW == 0 && GW % NW == 0 && TM % 16 == 0 && TN % 16 == 0 && kScaleCols % TN == 0, "tile shape");
  const int lane = lane_id();
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int tiles_m = (a.M + BM - 1) / BM;
  const int q = (int)gridDim.x >> 3, r = (int)gridDim.x & 7, xcd = (int)blockIdx.x & 7, loc = (int)blockIdx.x >> 3;
  const int t = xcd * q + min(xcd, r) + loc;
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
  const int wm = w / WN, wn = w % WN, fr = lane & 15, fg = lane >> 4;
  const uint8_t* sxb = a.x_scale + (long)m0 * kb_n;
  unsigned offS[TM / 16];
#pragma unroll
  for (int i = 0; i < TM / 16; ++i) offS[i] = (unsigned)min(wm * TM + 16 * i + fr, a.M - 1 - m0) * (unsigned)kb_n;
  const uint8_t* swp = a.w_scale + (long)(min(n0 + wn * TN, a.N - 1) / kScaleCols) * kb_n;
  int sx[TM / 16], sx_next[TM / 16], sw = 0, sw_next = 0;

  auto issue = [&](auto S, int kb) {
    char* st = tile_stage<decltype(S)::value, STAGE>();
    const int k = kb * kScaleCols;
    const bool tail = k + chunk >= a.K;   // only in a last, partial block
    const unsigned ka = tail ? a.K - 16 - chunk : k;
#pragma unroll
    for (int i = 0; i < LA; ++i) load_lds16(xb + (offA[i] + ka), st + (i * NW + w) * 1024);
#pragma unroll
    for (int i = 0; i < LW; ++i)
      load_lds16(tail ? reinterpret_cast<const uint8_t*>(&kZeros) : wb + (offW[i] + k), st + BM * kScaleCols + (i * NW + w) * 1024);
#pragma unroll
    for (int i = 0; i < TM / 16; ++i) sx_next[i] = sxb[offS[i] + kb];
    sw_next = swp[kb];
  };
  f32x4 acc[TM / 16][TN / 16];
#pragma unroll
  for (int i = 0; i < TM / 16; ++i)
#pragma unroll
    for (int j = 0; j < TN / 16; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
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
  auto compute = [&](auto S) {
    const char* st = tile_stage<decltype(S)::value, STAGE>();
    auto frag = [&](const unsigned (&b)[2], int tile, u32x4& lo, u32x4& hi) {
      lo = *reinterpret_cast<const u32x4*>(st + b[0] + tile * 16 * kScaleCols);
      hi = *reinterpret_cast<const u32x4*>(st + b[1] + tile * 16 * kScaleCols);
    };
    if constexpr (F8) {
      i32x8 fw[TN / 16];
#pragma unroll
      for (int j = 0; j < TN / 16; ++j) {
        u32x4 lo, hi;
        frag(bW, j, lo, hi);
        fw[j] = i32x8{(int)lo.x, (int)lo.y, (int)lo.z, (int)lo.w, (int)hi.x, (int)hi.y, (int)hi.z, (int)hi.w};
      }
#pragma unroll
      for (int i = 0; i < TM / 16; ++i) {
        u32x4 lo, hi;
        frag(bA, i, lo, hi);
        const i32x8 fx = {(int)lo.x, (int)lo.y, (int)lo.z, (int)lo.w, (int)hi.x, (int)hi.y, (int)hi.z, (int)hi.w};
#pragma unroll
        for (int j = 0; j < TN / 16; ++j)
          acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fw[j], fx, acc[i][j], 0, 0, 0, sw, 0, sx[i]);
      }
    } else {
      h8v hw[TN / 16][4];
#pragma unroll
      for (int j = 0; j < TN / 16; ++j) {
        u32x4 lo, hi;
        frag(bW, j, lo, hi);
        widen_block(lo, hi, hw[j]);
      }
#pragma unroll
      for (int i = 0; i < TM / 16; ++i) {
        u32x4 lo, hi;
        frag(bA, i, lo, hi);
        h8v hx[4];
        widen_block(lo, hi, hx);
        const float f = scale_of(sw, sx[i]);
        f32x4 blk[TN / 16];
#pragma unroll
        for (int j = 0; j < TN / 16; ++j) blk[j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < 4; ++ks)
#pragma unroll
          for (int j = 0; j < TN / 16; ++j) blk[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(hw[j][ks], hx[ks], blk[j], 0, 0, 0);
#pragma unroll
        for (int j = 0; j < TN / 16; ++j) acc[i][j] += blk[j] * f;
      }
    }
  };
  const std::integral_constant<int, 0> s0;
  const std::integral_constant<int, 1> s1;
  auto step = [&](auto S, int kb) {
    wait_barrier();
#pragma unroll
    for (int i = 0; i < TM / 16; ++i) sx[i] = sx_next[i];
    sw = sw_next;
    if (kb + 1 < kb_n) issue(std::integral_constant<int, 1 - decltype(S)::value>{}, kb + 1);
    compute(S);
  };
  issue(s0, 0);
  int kb = 0;
#pragma unroll 1
  for (; kb + 1 < kb_n; kb += 2) {
    step(s0, kb);
    step(s1, kb + 1);
  }
  if (kb < kb_n) step(s0, kb);
  TO* y = reinterpret_cast<TO*>(a.y);
#pragma unroll
  for (int i = 0; i < TM / 16; ++i) {
    const int m = m0 + wm * TM + 16 * i + fr;
    if (m < a.M) {
#pragma unroll
      for (int j = 0; j < TN / 16; ++j) {
        const int n = n0 + wn * TN + 16 * j + 4 * fg;
        if (n < a.N) store4(y, m, a.N, n, acc[i][j]);
      }
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

template <int BM, int BN, int WM, int WN, typename TO>
int launch_tile(const GemmFp8Args& a, hipStream_t s) {
  const unsigned t = (unsigned)(((a.M + BM - 1) / BM) * (long)((a.N + BN - 1) / BN));
  hipLaunchKernelGGL((gemm_fp8_tile_kernel<BM, BN, WM, WN, sizeof(TO) == 2, TO>), dim3(t), dim3(kWave * WM * WN), 0, s, a);
  return qd_host::launch_status("gemm_fp8_tile_kernel");
}

template <typename TO>
int launch(const GemmFp8Args& a, hipStream_t s) {
  if (a.M <= 16) return launch_rows<1, 4, 4, TO>(a, s);
  if (a.M <= 64) return launch_rows<2, 4, 2, TO>(a, s);
  if (a.M <= 256) return launch_tile<64, 128, 2, 2, TO>(a, s);
  return launch_tile<128, 256, 2, 4, TO>(a, s);
}

}  // namespace

int gemm_fp8_launch(const GemmFp8Args& a, hipStream_t s) {
  return a.y_f32 ? launch<float>(a, s) : launch<uint16_t>(a, s);
}

}  // namespace qd
