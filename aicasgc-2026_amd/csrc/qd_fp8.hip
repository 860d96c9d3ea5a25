// 8-bit quantisers for gfx950: activation rows (add + RMSNorm, SiLU * up, plain),
// weight blocks, and the KV cache written in 8 bits and read back.  All are bound by
// memory or, for a decode token, by their launch.  Sums and maxima are fp32; the one
// rounding of a stored value is its own to e4m3 (the scales are powers of two).

#include <math.h>

#include "qd_fp8.h"

namespace qd {

namespace {

constexpr int kHD = 128;
constexpr int kRowThreads = 256;
constexpr int kRowSpan = kRowThreads * 8;   // columns a workgroup passes over at once

// 8 consecutive fp16 values of a row of `cols`; VEC: the 16 bytes are aligned
// and lie inside the row wholly or not at all.
template <bool VEC>
__device__ __forceinline__ void load_row8(const uint16_t* p, long k, long cols, float* o) {
  if constexpr (VEC) {
    unpack8(ld16(p + k), o);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = k + e < cols ? h2f(p[k + e]) : 0.f;
  }
}
template <bool VEC>
__device__ __forceinline__ void store_row8(uint16_t* p, long k, long cols, const float* v) {
  if constexpr (VEC) {
    store_act8(p, k, v);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (k + e < cols) p[k + e] = f2h(v[e]);
  }
}
template <bool VEC>
__device__ __forceinline__ void store_q8(uint8_t* p, long k, long cols, const float* v, int e2) {
  const float s = pow2i(-e2);
  const unsigned lo = pack_fp8x4(v[0] * s, v[1] * s, v[2] * s, v[3] * s);
  const unsigned hi = pack_fp8x4(v[4] * s, v[5] * s, v[6] * s, v[7] * s);
  if constexpr (VEC) {
    *reinterpret_cast<u32x2*>(p + k) = u32x2{lo, hi};
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (k + e < cols) p[k + e] = (uint8_t)((e < 4 ? lo : hi) >> (8 * (e & 3)));
  }
}

__device__ __forceinline__ float amax8(const float* v) {
  float m = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) m = fmaxf(m, finite_abs(v[e]));
  return m;
}

// Quantises this thread's 8 values at column k; the 16 lanes of a row16 hold one
// 128-column block, so its amax is four DPP steps.  Lanes past the row's end hold
// zeros.
template <bool VEC>
__device__ __forceinline__ void quantize8(const RowQuantArgs& a, long row, long k, const float* v) {
  const int e2 = fp8_exp(row16_max(amax8(v)), kFp8Low);
  if (k < a.cols) {
    store_q8<VEC>(a.q + row * a.cols, k, a.cols, v, e2);
    if ((threadIdx.x & 15) == 0) a.scale[row * a.scale_cols + k / kScaleCols] = (uint8_t)(e2 + 127);
  }
}

// v / (1 + e^-v) within 4 * 2^-24 of itself: e^-v as 2^t (1 + lo ln 2), t + lo = -v log2(e) to
// twice fp32's digits, since t's rounding alone is |v| 2^-24 of the result.  From t = 100 on
// the 1 is nothing and the result is v e^v, with 2^64 taken out of e^v for as long as it would
// be denormal (64 - t is exact there), so that nothing overflows or is flushed.  (expf and a
// division, about 40 instructions a value, would bind the kernel instead of memory:
// 4001 x 6144 took 29.9 us with them and takes 22.5 without.)
__device__ __forceinline__ float silu(float v) {
  constexpr float kLog2e = 1.44269502162933349609f, kLog2eLow = 1.92596299112661746887e-8f, kLn2 = 0.69314718055994530942f;
  const float t = -v * kLog2e;
  const float c = __builtin_fmaf(-v, kLog2eLow, __builtin_fmaf(-v, kLog2e, -t)) * kLn2;
  const bool far = t > 100.0f;
  const float e = __builtin_amdgcn_exp2f(far ? 64.0f - t : t);
  const float r = __builtin_fmaf(e, far ? -c : c, e);   // 2^64 e^v, or e^-v
  return far ? v * 0x1p-64f * r : v * __builtin_amdgcn_rcpf(1.0f + r);
}

__device__ __forceinline__ void add_row8(float* v, const float* r) {
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] += r[e];
}

}  // namespace

// One row per workgroup: v = x (+ residual, also stored as fp16), RMSNorm of the
// fp32 sum, quantised.  C chunks of 2048 columns stay in registers between the two
// passes; C = 0 (longer rows) reads them again.  A row per workgroup: its sum needs one
// exchange of four waves, and 16 lanes hold a scale's 128 columns.  2048 columns with a
// residual: 4001 rows 12.2 us (4.7 TB/s; a copy of that size reaches 5.1), one row 2.0.
template <int C, bool VEC>
__global__ __launch_bounds__(kRowThreads) void add_rmsnorm_fp8_kernel(const RowQuantArgs a) {
  __shared__ float s_red[kRowThreads / kWave];
  const long row = blockIdx.x;
  const uint16_t* x = a.x + row * a.ldx;
  const uint16_t* r = a.x2 != nullptr ? a.x2 + row * a.ldx2 : nullptr;
  uint16_t* sum = a.sum != nullptr ? a.sum + row * a.cols : nullptr;
  const long k0 = threadIdx.x * 8;
  float u[C > 0 ? C : 1][8];
  float ss = 0.f;
  auto load = [&](long k, float* v) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = 0.f;
    if (k >= a.cols) return;
    load_row8<VEC>(x, k, a.cols, v);
    if (r != nullptr) {
      float t[8];
      load_row8<VEC>(r, k, a.cols, t);
      add_row8(v, t);
    }
  };
  auto square = [&](const float* v) {
#pragma unroll
    for (int e = 0; e < 8; ++e) ss = __builtin_fmaf(v[e], v[e], ss);
  };
  if constexpr (C > 0) {
#pragma unroll
    for (int c = 0; c < C; ++c) load(k0 + c * kRowSpan, u[c]);
#pragma unroll
    for (int c = 0; c < C; ++c) square(u[c]);
  } else {
    for (long k = k0; k < a.cols; k += kRowSpan) {
      load(k, u[0]);
      square(u[0]);
    }
  }
  ss = wave_sum(ss);
  if (lane_id() == 0) s_red[threadIdx.x / kWave] = ss;
  __syncthreads();
  ss = (s_red[0] + s_red[1]) + (s_red[2] + s_red[3]);
  const float rstd = rsqrtf(ss / (float)a.cols + a.eps);
  auto finish = [&](long k, float* v) {
    if (sum != nullptr && k < a.cols) store_row8<VEC>(sum, k, a.cols, v);
    float w[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (k < a.cols) load_row8<VEC>(a.weight, k, a.cols, w);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = k + e < a.cols ? (v[e] * rstd) * w[e] : 0.f;
    quantize8<VEC>(a, row, k, v);
  };
  if constexpr (C > 0) {
#pragma unroll
    for (int c = 0; c < C; ++c) finish(k0 + c * kRowSpan, u[c]);
  } else {
    // every lane of a 16-lane row runs the same number of rounds: the row is one block
    for (long k = k0; k / kScaleCols * kScaleCols < a.cols; k += kRowSpan) {
      load(k, u[0]);
      finish(k, u[0]);
    }
  }
}

// 2048 columns of one row per workgroup: x, or silu(x) * x2.  4001 rows: 2048 columns of x
// 5.3 us (4.6 TB/s), 6144 of silu(x) * x2 22.5 us (5.5 TB/s); one row of 6144 2.4 us.
template <bool SILU, bool VEC>
__global__ __launch_bounds__(kRowThreads) void quantize_rows_kernel(const RowQuantArgs a) {
  const long row = blockIdx.x, k = (long)blockIdx.y * kRowSpan + threadIdx.x * 8;
  float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (k < a.cols) {
    load_row8<VEC>(a.x + row * a.ldx, k, a.cols, v);
    if constexpr (SILU) {
      float u[8];
      load_row8<VEC>(a.x2 + row * a.ldx2, k, a.cols, u);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = silu(v[e]) * u[e];
    }
  }
  quantize8<VEC>(a, row, k, v);
}

// One 128 x 128 block of a weight per workgroup, in registers between its maximum and its
// rounding.  12288 x 2048: 15.6 us (4.8 TB/s).
template <bool VEC>
__global__ __launch_bounds__(kRowThreads) void quantize_blocks_kernel(const RowQuantArgs a) {
  __shared__ float s_red[kRowThreads / kWave];
  const long r0 = (long)blockIdx.x * kScaleCols + threadIdx.x / 16;
  const long k = (long)blockIdx.y * kScaleCols + (threadIdx.x & 15) * 8;
  float v[8][8];
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const long row = r0 + 16 * i;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[i][e] = 0.f;
    if (row < a.rows && k < a.cols) load_row8<VEC>(a.x + row * a.ldx, k, a.cols, v[i]);
    m = fmaxf(m, amax8(v[i]));
  }
  m = wave_max(m);
  if (lane_id() == 0) s_red[threadIdx.x / kWave] = m;
  __syncthreads();
  const int e2 = fp8_exp(fmaxf(fmaxf(s_red[0], s_red[1]), fmaxf(s_red[2], s_red[3])), kFp8Low);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const long row = r0 + 16 * i;
    if (row < a.rows && k < a.cols) store_q8<VEC>(a.q + row * a.cols, k, a.cols, v[i], e2);
  }
  if (threadIdx.x == 0) a.scale[(long)blockIdx.x * a.scale_cols + blockIdx.y] = (uint8_t)(e2 + 127);
}

namespace {

// 16-byte loads need aligned rows of whole 8-value chunks.
bool vec_ok(const RowQuantArgs& a) {
  const uintptr_t p = reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.x2) |
                      reinterpret_cast<uintptr_t>(a.weight) | reinterpret_cast<uintptr_t>(a.sum);
  return a.cols % 8 == 0 && a.ldx % 8 == 0 && a.ldx2 % 8 == 0 && (p & 15) == 0 &&
         (reinterpret_cast<uintptr_t>(a.q) & 7) == 0;
}

template <int C>
void launch_norm(const RowQuantArgs& a, hipStream_t s) {
  if (vec_ok(a))
    hipLaunchKernelGGL((add_rmsnorm_fp8_kernel<C, true>), dim3((unsigned)a.rows), dim3(kRowThreads), 0, s, a);
  else
    hipLaunchKernelGGL((add_rmsnorm_fp8_kernel<C, false>), dim3((unsigned)a.rows), dim3(kRowThreads), 0, s, a);
}

}  // namespace

int add_rmsnorm_fp8_launch(const RowQuantArgs& a, hipStream_t s) {
  const long chunks = (a.cols + kRowSpan - 1) / kRowSpan;
  if (chunks == 1)
    launch_norm<1>(a, s);
  else if (chunks <= 4)
    launch_norm<4>(a, s);
  else
    launch_norm<0>(a, s);
  return qd_host::launch_status("add_rmsnorm_fp8_kernel");
}

int quantize_rows_fp8_launch(const RowQuantArgs& a, bool silu, hipStream_t s) {
  const dim3 grid((unsigned)a.rows, (unsigned)((a.cols + kRowSpan - 1) / kRowSpan));
  const bool vec = vec_ok(a);
  if (silu && vec)
    hipLaunchKernelGGL((quantize_rows_kernel<true, true>), grid, dim3(kRowThreads), 0, s, a);
  else if (silu)
    hipLaunchKernelGGL((quantize_rows_kernel<true, false>), grid, dim3(kRowThreads), 0, s, a);
  else if (vec)
    hipLaunchKernelGGL((quantize_rows_kernel<false, true>), grid, dim3(kRowThreads), 0, s, a);
  else
    hipLaunchKernelGGL((quantize_rows_kernel<false, false>), grid, dim3(kRowThreads), 0, s, a);
  return qd_host::launch_status("quantize_rows_kernel");
}

int quantize_blocks_fp8_launch(const RowQuantArgs& a, hipStream_t s) {
  const dim3 grid((unsigned)((a.rows + kScaleCols - 1) / kScaleCols), (unsigned)a.scale_cols);
  if (vec_ok(a))
    hipLaunchKernelGGL((quantize_blocks_kernel<true>), grid, dim3(kRowThreads), 0, s, a);
  else
    hipLaunchKernelGGL((quantize_blocks_kernel<false>), grid, dim3(kRowThreads), 0, s, a);
  return qd_host::launch_status("quantize_blocks_kernel");
}

// ---------------------------------------------------------------- the cache, written

namespace {

// 4 fp16 values at an 8-byte aligned address.
__device__ __forceinline__ void load4(const uint16_t* p, float* o) {
  const u32x2 v = *reinterpret_cast<const u32x2*>(p);
  o[0] = lo_f(v.x); o[1] = hi_f(v.x); o[2] = lo_f(v.y); o[3] = hi_f(v.y);
}

// 4 e4m3 bytes times f (a power of two below 1).
__device__ __forceinline__ unsigned rescale4(unsigned v, float f) {
  float t[4];
  unpack_fp8x4(v, t);
  return pack_fp8x4(t[0] * f, t[1] * f, t[2] * f, t[3] * f);
}

__device__ __forceinline__ float block_max4(float m, float* s_red) {
  m = wave_max(m);
  if (lane_id() == 0) s_red[threadIdx.x / kWave] = m;
  __syncthreads();
  return fmaxf(fmaxf(s_red[0], s_red[1]), fmaxf(s_red[2], s_red[3]));
}

}  // namespace

// grid (blocks, 2 + G, B * Hkv), 256 threads.  Workgroup (j, 0 / 1, bh): the new K
// / V rows that fall into the j-th 64-row cache block from the first new row's on;
// (j, 2 + g, bh): q rows [64 j, 64 j + 64) of the group's head g.
//
// A block with rows from before keeps its exponent unless the new rows need a
// larger one; then the earlier rows are read, scaled down and written again (exact
// but for values that become subnormal).  One workgroup owns the block, so nobody
// else touches those bytes.  Rows behind the new ones keep their bytes.
//
// Bound by memory: 4001 tokens of 16 + 2 * 8 heads 14.1 us (60 MB, 4.2 TB/s).  One token of
// 8 sequences takes 5.7 us, the chain of dependent loads position, row, scale,
// earlier rows of the block.
__global__ __launch_bounds__(256) void kv_update_fp8_kernel(const KvUpdateFp8Args a) {
  __shared__ float s_red[4];
  const int b = (int)blockIdx.z / a.c.Hkv, kvh = (int)blockIdx.z % a.c.Hkv;
  const int role = (int)blockIdx.y;
  const int sub = threadIdx.x & 15, grp = threadIdx.x / 16;   // 16 lanes per row, 16 rows per pass
  const int d0 = 4 * sub;                                     // dims [d0, d0 + 4) and [64 + d0, ...)
  const long pos = a.cache_position[b];

  float w[8];   // this role's norm weights
  if (role != 1) {
    load4((role == 0 ? a.k_weight : a.q_weight) + d0, w);
    load4((role == 0 ? a.k_weight : a.q_weight) + 64 + d0, w + 4);
  }
  // rows of a head, normalised and rotated: 8 values of 4 rotary pairs
  auto load_rotated = [&](const uint16_t* src, long i, float* o) {
    float x[8], cs[8], sn[8];
    const long at = ((long)b * a.S + i) * kHD + d0;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      load4(src + 64 * h + d0, x + 4 * h);
      load4(a.cos + at + 64 * h, cs + 4 * h);
      load4(a.sin + at + 64 * h, sn + 4 * h);
    }
    float ss = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) ss = __builtin_fmaf(x[e], x[e], ss);
    const float rstd = rsqrtf(row16_sum(ss) / (float)kHD + a.eps);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float n0 = (x[e] * rstd) * w[e], n1 = (x[4 + e] * rstd) * w[4 + e];
      o[e] = n0 * cs[e] - n1 * sn[e];
      o[4 + e] = n1 * cs[4 + e] + n0 * sn[4 + e];
    }
  };

  if (role >= 2) {
    const int h = kvh * a.G + role - 2;
    for (int p = 0; p < 4; ++p) {
      const long i = (long)blockIdx.x * kKvBlock + 16 * p + grp;
      if (i >= a.S) break;   // uniform over the 16 lanes that share the row
      float o[8];
      load_rotated(a.q + b * a.q_sb + i * a.q_ss + h * a.q_sh, i, o);
      uint16_t* dst = a.q_out + (((long)b * a.S + i) * a.c.Hkv * a.G + h) * kHD + d0;
      *reinterpret_cast<u32x2*>(dst) = u32x2{pack2(o[0], o[1]), pack2(o[2], o[3])};
      *reinterpret_cast<u32x2*>(dst + 64) = u32x2{pack2(o[4], o[5]), pack2(o[6], o[7])};
    }
    return;
  }

  // this block's rows, and which of its slots [lo, hi) are new
  const long blk = (pos >> 6) + blockIdx.x, base = blk * kKvBlock;
  if (blk < 0 || base >= a.c.T) return;
  const int lo = (int)max(pos - base, 0L), hi = (int)min(pos + a.S - base, (long)kKvBlock);
  if (lo >= hi) return;
  const long so = b * a.c.scale_stride_b + kvh * a.c.scale_stride_h + blk;
  const long off = b * a.c.stride_b + kvh * a.c.stride_h + base * kHD;
  uint8_t* sp = (role == 0 ? a.c.k_scale : a.c.v_scale) + so;
  uint8_t* dst = (role == 0 ? a.c.k : a.c.v) + off;
  const int e_old = lo > 0 ? (int)*sp - 127 : -127;

  if (role == 0) {
    float o[4][8];
    float m = 0.f;
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      const int slot = 16 * p + grp;
      if (slot < lo || slot >= hi) continue;
      const long i = base + slot - pos;
      load_rotated(a.k + b * a.k_sb + i * a.k_ss + kvh * a.k_sh, i, o[p]);
      m = fmaxf(m, amax8(o[p]));
    }
    const int e2 = max(fp8_exp(block_max4(m, s_red), kFp8KvLow), e_old);
    const float f = pow2i(-e2);
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      const int slot = 16 * p + grp;
      if (slot < lo || slot >= hi) continue;
      unsigned* row = reinterpret_cast<unsigned*>(dst + slot * kHD) + sub;
      row[0] = pack_fp8x4(o[p][0] * f, o[p][1] * f, o[p][2] * f, o[p][3] * f);
      row[16] = pack_fp8x4(o[p][4] * f, o[p][5] * f, o[p][6] * f, o[p][7] * f);
    }
    if (lo > 0 && e2 > e_old) {
      unsigned* w = reinterpret_cast<unsigned*>(dst);
      const float g = pow2i(max(e_old - e2, -126));
      for (int n = threadIdx.x; n < lo * (kHD / 4); n += 256) w[n] = rescale4(w[n], g);
    }
    if (threadIdx.x == 0) *sp = (uint8_t)(e2 + 127);
    return;
  }

  // V: 4 dims of 8 consecutive slots per thread, so that the loads are rows of
  // 256 bytes and a thread's bytes of one dim are 8 consecutive ones
  const int dq = (threadIdx.x & 31) * 4, s0 = (threadIdx.x / 32) * 8;
  float o[8][4];
  float m = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int slot = s0 + e;
    u32x2 x = {0u, 0u};
    if (slot >= lo && slot < hi)
      x = *reinterpret_cast<const u32x2*>(a.v + b * a.v_sb + (base + slot - pos) * a.v_ss + kvh * a.v_sh + dq);
    o[e][0] = lo_f(x.x); o[e][1] = hi_f(x.x); o[e][2] = lo_f(x.y); o[e][3] = hi_f(x.y);
#pragma unroll
    for (int d = 0; d < 4; ++d) m = fmaxf(m, finite_abs(o[e][d]));
  }
  const int e2 = max(fp8_exp(block_max4(m, s_red), kFp8KvLow), e_old);
  const float f = pow2i(-e2);
  const bool again = lo > 0 && e2 > e_old && s0 < lo;   // holds earlier rows to be scaled down
  const bool whole = s0 >= lo && s0 + 8 <= hi;
  if (again || (s0 < hi && s0 + 8 > lo)) {
    const float g = pow2i(max(e_old - e2, -126));
#pragma unroll
    for (int d = 0; d < 4; ++d) {
      const unsigned n0 = pack_fp8x4(o[0][d] * f, o[1][d] * f, o[2][d] * f, o[3][d] * f);
      const unsigned n1 = pack_fp8x4(o[4][d] * f, o[5][d] * f, o[6][d] * f, o[7][d] * f);
      uint8_t* p = dst + (dq + d) * kKvBlock + s0;
      if (whole) {
        *reinterpret_cast<u32x2*>(p) = u32x2{n0, n1};
        continue;
      }
      u32x2 r = {0u, 0u};
      if (again) {
        r = *reinterpret_cast<const u32x2*>(p);
        r.x = rescale4(r.x, g);
        r.y = rescale4(r.y, g);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int slot = s0 + e;
        const unsigned sh = 8 * (e & 3);
        if (slot >= lo && slot < hi)
          p[e] = (uint8_t)((e < 4 ? n0 : n1) >> sh);
        else if (again && slot < lo)
          p[e] = (uint8_t)((e < 4 ? r.x : r.y) >> sh);
      }
    }
  }
  if (threadIdx.x == 0) *sp = (uint8_t)(e2 + 127);
}

int kv_update_fp8_launch(const KvUpdateFp8Args& a, hipStream_t s) {
  const dim3 grid((unsigned)((a.S + 126) / kKvBlock), (unsigned)(2 + a.G), (unsigned)(a.c.B * a.c.Hkv));
  hipLaunchKernelGGL(kv_update_fp8_kernel, grid, dim3(256), 0, s, a);
  return qd_host::launch_status("kv_update_fp8_kernel");
}

// ---------------------------------------------------------------- the cache, read back

// One (block, K or V, head) per workgroup: 8 KB in, 16 KB out.  V's 4 dims x 8
// slots per thread are transposed 4 x 4 bytes at a time, and a wave stores rows of
// 256 bytes.  30001 rows of 8 heads: 29.6 us for 184 MB, 6.2 TB/s.
__global__ __launch_bounds__(256) void kv_read_fp8_kernel(const KvReadFp8Args a) {
  const int b = (int)blockIdx.z / a.c.Hkv, kvh = (int)blockIdx.z % a.c.Hkv;
  const long base = (long)blockIdx.x * kKvBlock;
  const long off = b * a.c.stride_b + kvh * a.c.stride_h + base * kHD;
  const long so = b * a.c.scale_stride_b + kvh * a.c.scale_stride_h + blockIdx.x;
  const long rows = min(a.rows - base, (long)kKvBlock);
  const long out = (((long)b * a.c.Hkv + kvh) * a.rows + base) * kHD;
  if (blockIdx.y == 0) {
    const float f = pow2i((int)a.c.k_scale[so] - 127);
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      const int n = (p * 256 + threadIdx.x) * 16;   // byte of the block
      if (n / kHD >= rows) break;
      const u32x4 x = ld16(a.c.k + off + n);
      float v[16];
#pragma unroll
      for (int i = 0; i < 4; ++i) unpack_fp8x4(x[i], v + 4 * i);
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] *= f;
      store_act8(a.k + out, n, v);
      store_act8(a.k + out, n + 8, v + 8);
    }
    return;
  }
  const float f = pow2i((int)a.c.v_scale[so] - 127);
  const int dq = (threadIdx.x & 31) * 4, s0 = (threadIdx.x / 32) * 8;
  if (s0 >= rows) return;
  float t[4][8];
#pragma unroll
  for (int d = 0; d < 4; ++d) {
    const u32x2 x = *reinterpret_cast<const u32x2*>(a.c.v + off + (dq + d) * kKvBlock + s0);
    unpack_fp8x4(x.x, t[d]);
    unpack_fp8x4(x.y, t[d] + 4);
  }
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (s0 + e < rows)
      *reinterpret_cast<u32x2*>(a.v + out + (long)(s0 + e) * kHD + dq) =
          u32x2{pack2(t[0][e] * f, t[1][e] * f), pack2(t[2][e] * f, t[3][e] * f)};
}

int kv_read_fp8_launch(const KvReadFp8Args& a, hipStream_t s) {
  const dim3 grid((unsigned)((a.rows + kKvBlock - 1) / kKvBlock), 2u, (unsigned)(a.c.B * a.c.Hkv));
  hipLaunchKernelGGL(kv_read_fp8_kernel, grid, dim3(256), 0, s, a);
  return qd_host::launch_status("kv_read_fp8_kernel");
}

}  // namespace qd
