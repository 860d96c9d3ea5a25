// Shared by the 8-bit kernels: e4m3 values (OCP, gfx950's native conversions)
// with a power-of-two scale per block, stored as E8M0 bytes 2^(b - 127).
//
// A block's exponent e is the least integer with amax <= 448 * 2^e (448 is
// e4m3's largest value), amax taken over the finite values; NaN and infinities
// are stored as NaN.  e4m3 is a floating format, so against an fp32 scale a power
// of two costs at most one bit of underflow range and no precision of a normal
// value, and every scaling is exact: the only rounding is a value's own, half an
// e4m3 step.
#pragma once

#include "qd_common.h"

namespace qd {

typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8v __attribute__((ext_vector_type(8)));

constexpr int kFp8Low = -126;     // least exponent of an activation or weight block
constexpr int kFp8KvLow = -32;    // of a cache block: holds fp16's least subnormal, and keeps
                                  // the attention's sums over blocks of any exponents in range
constexpr int kScaleCols = 128;   // columns (of x, of W) per scale; also W rows per scale
constexpr int kKvBlock = 64;      // cache rows per scale

__device__ __forceinline__ float pow2i(int e) {   // -126 <= e <= 127
  return __builtin_bit_cast(float, (unsigned)(e + 127) << 23);
}

// 448 = 1.75 * 2^8.
__device__ __forceinline__ int fp8_exp(float amax, int low) {
  const unsigned u = __builtin_bit_cast(unsigned, amax);
  const int e = (int)(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
  return max(e, low);
}

// |v| where it counts for a block's amax, else 0.
__device__ __forceinline__ float finite_abs(float v) {
  const float a = fabsf(v);
  return a <= 3.402823466e38f ? a : 0.f;
}

// Four scaled values to e4m3 bytes (round to nearest even; NaN and infinities
// to NaN).
__device__ __forceinline__ unsigned pack_fp8x4(float a, float b, float c, float d) {
  int r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true);
}

// Four e4m3 bytes to fp32.
__device__ __forceinline__ void unpack_fp8x4(unsigned v, float* o) {
  typedef float f2 __attribute__((ext_vector_type(2)));
  const f2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)v, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)v, true);
  o[0] = a.x; o[1] = a.y; o[2] = b.x; o[3] = b.y;
}

// Eight e4m3 bytes to fp16, exact (every e4m3 value is an fp16 value).
template <bool HI>
__device__ __forceinline__ unsigned fp8x2_to_f16(unsigned v) {
  return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)v, 1.0f, HI));
}
__device__ __forceinline__ h8v fp8x8_to_f16(unsigned lo, unsigned hi) {
  return __builtin_bit_cast(h8v, u32x4{fp8x2_to_f16<false>(lo), fp8x2_to_f16<true>(lo), fp8x2_to_f16<false>(hi),
                                       fp8x2_to_f16<true>(hi)});
}

// ---------------------------------------------------------------- the 8-bit cache

// Rows in blocks of kKvBlock tokens per (sequence, kv head), one exponent per
// block of K and one per block of V.  K rows lie as [T][128], V transposed inside
// its block, [T / 64][128][64], so that a 64-token tile of either is 8 KB of
// consecutive bytes that an attention wave loads as matrix operands as they are.
struct Fp8Cache {
  uint8_t* k = nullptr;
  uint8_t* v = nullptr;
  uint8_t* k_scale = nullptr;   // [T / 64] per head
  uint8_t* v_scale = nullptr;
  long stride_b = 0, stride_h = 0;               // values, K and V alike
  long scale_stride_b = 0, scale_stride_h = 0;   // both scale arrays
  int T = 0;                    // capacity, a multiple of 64
  int B = 0, Hkv = 0;
};

// ---------------------------------------------------------------- launches

struct RowQuantArgs {
  const uint16_t* x = nullptr;        // [rows][cols], row stride ldx
  const uint16_t* x2 = nullptr;       // residual (norm, may be null) or up (SiLU), row stride ldx2
  const uint16_t* weight = nullptr;   // norm: [cols]
  uint16_t* sum = nullptr;            // norm with a residual: [rows][cols]
  uint8_t* q = nullptr;               // [rows][cols]
  uint8_t* scale = nullptr;           // [rows or ceil(rows / 128)][scale_cols]
  long ldx = 0, ldx2 = 0;
  long rows = 0, cols = 0;
  long scale_cols = 0;                // ceil(cols / 128)
  float eps = 0.f;
};
int add_rmsnorm_fp8_launch(const RowQuantArgs& a, hipStream_t s);
int quantize_rows_fp8_launch(const RowQuantArgs& a, bool silu, hipStream_t s);
int quantize_blocks_fp8_launch(const RowQuantArgs& a, hipStream_t s);

struct KvUpdateFp8Args {
  const uint16_t *q = nullptr, *k = nullptr, *v = nullptr;   // batch, token and head strides below
  long q_sb = 0, q_ss = 0, q_sh = 0, k_sb = 0, k_ss = 0, k_sh = 0, v_sb = 0, v_ss = 0, v_sh = 0;
  const uint16_t *q_weight = nullptr, *k_weight = nullptr;   // [128]
  const uint16_t *cos = nullptr, *sin = nullptr;             // [B][S][128]
  uint16_t* q_out = nullptr;                                 // [B][S][Hq][128]
  const int64_t* cache_position = nullptr;                   // [B]
  Fp8Cache c;
  long S = 0;
  int G = 0;                                                 // q heads per kv head
  float eps = 0.f;
};
int kv_update_fp8_launch(const KvUpdateFp8Args& a, hipStream_t s);

struct KvReadFp8Args {
  Fp8Cache c;
  uint16_t *k = nullptr, *v = nullptr;   // [B][Hkv][rows][128]
  long rows = 0;
};
int kv_read_fp8_launch(const KvReadFp8Args& a, hipStream_t s);

struct AttnFp8Args {
  const uint16_t* q = nullptr;           // batch, head and token strides below
  long q_sb = 0, q_sh = 0, q_ss = 0;
  uint16_t* out = nullptr;               // [B][Sq][Hq][128]
  const int64_t* cache_position = nullptr;   // [B], of the first query token
  Fp8Cache c;
  int Sq = 0, G = 0;
  float scale2 = 0.f;                    // score scale times log2(e)
  int window = 0, sinks = 0;             // window 0: none
  int n_split = 1;
  float* part_o = nullptr;               // [B * Hkv][n_split][Sq * G][128]
  float* part_ml = nullptr;              // [B * Hkv][n_split][Sq * G][2]
};
int attention_fp8_splits(int B, int Hkv, int Sq, int G, int T, int window, int sinks);
int attention_fp8_launch(const AttnFp8Args& a, hipStream_t s);

struct GemmFp8Args {
  const uint8_t* x = nullptr;            // [M][K]
  const uint8_t* x_scale = nullptr;      // [M][ceil(K / 128)]
  const uint8_t* w = nullptr;            // [N][K]
  const uint8_t* w_scale = nullptr;      // [ceil(N / 128)][ceil(K / 128)]
  void* y = nullptr;                     // [M][N]
  int y_f32 = 0;
  int M = 0, N = 0, K = 0;
};
int gemm_fp8_launch(const GemmFp8Args& a, hipStream_t s);

}  // namespace qd
