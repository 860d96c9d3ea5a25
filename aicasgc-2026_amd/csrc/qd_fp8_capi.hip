// C ABI of the 8-bit operators (see include/qwen3vl_decode.h): argument checks and
// dispatch.

#include <math.h>

#include "qd_fp8.h"

namespace {

using u16 = uint16_t;
using u8 = uint8_t;

inline hipStream_t S(void* s) { return reinterpret_cast<hipStream_t>(s); }
inline bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

constexpr long kMaxRows = 1L << 23;    // a row per workgroup of 256 threads: below 2^32 threads

int check_rows(const void* x, const void* q, const void* scale, long rows, long cols) {
  QD_REQUIRE(rows >= 0 && rows <= kMaxRows && cols >= 1 && cols <= (1L << 26), QD_ERR_SHAPE,
             "need 0 <= rows <= %ld and 1 <= cols <= 2^26 (rows=%ld cols=%ld)", kMaxRows, rows, cols);
  QD_REQUIRE(rows == 0 || (x && q && scale), QD_ERR_ARG, "null pointer");
  QD_REQUIRE(aligned(x, 2), QD_ERR_ARG, "fp16 rows must be 2-byte aligned");
  return QD_OK;
}

int check_cache(qd::Fp8Cache& c, void* k, void* v, void* ks, void* vs, long stride_b, long stride_h, long scale_stride_b,
                long scale_stride_h, int T, int B, int Hkv) {
  QD_REQUIRE(B >= 0 && Hkv >= 1 && (long)B * Hkv <= 65535, QD_ERR_SHAPE, "need B * Hkv in [0, 65535] (B=%d Hkv=%d)", B,
             Hkv);
  QD_REQUIRE(T >= 0 && T % qd::kKvBlock == 0, QD_ERR_SHAPE, "the capacity must be a multiple of %d (T=%d)", qd::kKvBlock,
             T);
  QD_REQUIRE(B == 0 || T == 0 || (k && v && ks && vs), QD_ERR_ARG, "null cache pointer");
  QD_REQUIRE(aligned(k, 16) && aligned(v, 16) && stride_b % 16 == 0 && stride_h % 16 == 0, QD_ERR_ARG,
             "cache heads must be 16-byte aligned");
  c.k = (u8*)k; c.v = (u8*)v; c.k_scale = (u8*)ks; c.v_scale = (u8*)vs;
  c.stride_b = stride_b; c.stride_h = stride_h; c.scale_stride_b = scale_stride_b; c.scale_stride_h = scale_stride_h;
  c.T = T; c.B = B; c.Hkv = Hkv;
  return QD_OK;
}

}  // namespace

#define QD_TRY(expr)                   \
  do {                                 \
    const int st_ = (expr);            \
    if (st_ != QD_OK) return st_;      \
  } while (0)

extern "C" {

int qd_quantize_fp8(const void* x, long ldx, void* q, void* scale, long rows, long cols, int block_rows, void* stream) {
  QD_REQUIRE(block_rows == 1 || block_rows == qd::kScaleCols, QD_ERR_ARG, "block_rows is 1 or 128 (got %d)", block_rows);
  QD_TRY(check_rows(x, q, scale, rows, cols));
  qd::RowQuantArgs a;
  a.x = (const u16*)x; a.ldx = ldx; a.q = (u8*)q; a.scale = (u8*)scale;
  a.rows = rows; a.cols = cols; a.scale_cols = (cols + qd::kScaleCols - 1) / qd::kScaleCols;
  QD_REQUIRE(block_rows == 1 || a.scale_cols <= 65535, QD_ERR_SHAPE, "too many columns (%ld)", cols);
  if (rows == 0) return QD_OK;
  return block_rows == 1 ? qd::quantize_rows_fp8_launch(a, false, S(stream)) : qd::quantize_blocks_fp8_launch(a, S(stream));
}

int qd_silu_mul_fp8(const void* gate, long ld_gate, const void* up, long ld_up, void* q, void* scale, long rows,
                    long cols, void* stream) {
  QD_TRY(check_rows(gate, q, scale, rows, cols));
  QD_REQUIRE((rows == 0 || up) && aligned(up, 2), QD_ERR_ARG, "up must be a 2-byte aligned pointer");
  if (rows == 0) return QD_OK;
  qd::RowQuantArgs a;
  a.x = (const u16*)gate; a.ldx = ld_gate; a.x2 = (const u16*)up; a.ldx2 = ld_up; a.q = (u8*)q; a.scale = (u8*)scale;
  a.rows = rows; a.cols = cols; a.scale_cols = (cols + qd::kScaleCols - 1) / qd::kScaleCols;
  return qd::quantize_rows_fp8_launch(a, true, S(stream));
}

int qd_add_rmsnorm_fp8(const void* residual, long ld_residual, const void* x, long ldx, const void* weight, void* out_sum,
                       void* q, void* scale, long rows, long cols, float eps, void* stream) {
  QD_TRY(check_rows(x, q, scale, rows, cols));
  QD_REQUIRE(rows == 0 || weight, QD_ERR_ARG, "null pointer");
  QD_REQUIRE(aligned(residual, 2) && aligned(weight, 2) && aligned(out_sum, 2), QD_ERR_ARG,
             "fp16 operands must be 2-byte aligned");
  if (rows == 0) return QD_OK;
  qd::RowQuantArgs a;
  a.x = (const u16*)x; a.ldx = ldx; a.x2 = (const u16*)residual; a.ldx2 = residual ? ld_residual : 0;
  a.weight = (const u16*)weight; a.sum = (u16*)out_sum; a.q = (u8*)q; a.scale = (u8*)scale;
  a.rows = rows; a.cols = cols; a.scale_cols = (cols + qd::kScaleCols - 1) / qd::kScaleCols; a.eps = eps;
  return qd::add_rmsnorm_fp8_launch(a, S(stream));
}

int qd_block_matmul_fp8(const void* x, const void* x_scale, const void* w, const void* w_scale, void* y, int y_dtype,
                        int M, int N, int K, void* stream) {
  QD_REQUIRE(y_dtype == QD_F16 || y_dtype == QD_F32, QD_ERR_ARG, "y_dtype is QD_F16 or QD_F32 (got %d)", y_dtype);
  QD_REQUIRE(M >= 0 && N >= 1 && K >= 16 && K % 16 == 0, QD_ERR_SHAPE,
             "need M >= 0, N >= 1 and K a positive multiple of 16 (M=%d N=%d K=%d)", M, N, K);
  QD_REQUIRE(N <= (1 << 24) && M <= (1 << 20) && K <= (1 << 23), QD_ERR_SHAPE,
             "need M <= 2^20, N <= 2^24 and K <= 2^23 (M=%d N=%d K=%d)", M, N, K);
  QD_REQUIRE((long)M * N <= (1L << 37), QD_ERR_SHAPE, "more than 2^37 results (M=%d N=%d)", M, N);
  if (M == 0) return QD_OK;
  QD_REQUIRE(x && x_scale && w && w_scale && y, QD_ERR_ARG, "null pointer");
  QD_REQUIRE(aligned(x, 16) && aligned(w, 16) && aligned(y, 16), QD_ERR_ARG, "x, w and y must be 16-byte aligned");
  qd::GemmFp8Args a;
  a.x = (const u8*)x; a.x_scale = (const u8*)x_scale; a.w = (const u8*)w; a.w_scale = (const u8*)w_scale; a.y = y;
  a.y_f32 = y_dtype == QD_F32; a.M = M; a.N = N; a.K = K;
  return qd::gemm_fp8_launch(a, S(stream));
}

int qd_q_rope_kv_update_fp8(const void* q, long q_sb, long q_ss, long q_sh, const void* k, long k_sb, long k_ss, long k_sh,
                            const void* v, long v_sb, long v_ss, long v_sh, const void* q_weight, const void* k_weight,
                            float eps, const void* cos, const void* sin, void* q_out, void* k_cache, void* v_cache,
                            void* k_scale, void* v_scale, long stride_b, long stride_h, long scale_stride_b,
                            long scale_stride_h, int T, const int64_t* cache_position, int B, int S_, int Hq, int Hkv,
                            void* stream) {
  qd::KvUpdateFp8Args a;
  QD_TRY(check_cache(a.c, k_cache, v_cache, k_scale, v_scale, stride_b, stride_h, scale_stride_b, scale_stride_h, T, B,
                     Hkv));
  QD_REQUIRE(S_ >= 0 && S_ <= (1 << 24), QD_ERR_SHAPE, "need 0 <= S <= 2^24 (S=%d)", S_);
  QD_REQUIRE(Hq >= Hkv && Hq % Hkv == 0 && Hq / Hkv <= 64, QD_ERR_SHAPE,
             "Hq must be 1 to 64 times Hkv (Hq=%d Hkv=%d)", Hq, Hkv);
  if (B == 0 || S_ == 0) return QD_OK;
  QD_REQUIRE(q && k && v && q_weight && k_weight && cos && sin && q_out && cache_position, QD_ERR_ARG, "null pointer");
  QD_REQUIRE(aligned(q, 8) && aligned(k, 8) && aligned(v, 8) && aligned(q_out, 8) && aligned(cos, 8) && aligned(sin, 8) &&
                 aligned(q_weight, 8) && aligned(k_weight, 8) && aligned(cache_position, 8),
             QD_ERR_ARG, "every operand must be 8-byte aligned");
  QD_REQUIRE(((q_sb | q_ss | q_sh | k_sb | k_ss | k_sh | v_sb | v_ss | v_sh) & 3) == 0, QD_ERR_ARG,
             "q, k and v strides must be multiples of 4 elements");
  a.q = (const u16*)q; a.q_sb = q_sb; a.q_ss = q_ss; a.q_sh = q_sh;
  a.k = (const u16*)k; a.k_sb = k_sb; a.k_ss = k_ss; a.k_sh = k_sh;
  a.v = (const u16*)v; a.v_sb = v_sb; a.v_ss = v_ss; a.v_sh = v_sh;
  a.q_weight = (const u16*)q_weight; a.k_weight = (const u16*)k_weight;
  a.cos = (const u16*)cos; a.sin = (const u16*)sin; a.q_out = (u16*)q_out; a.cache_position = cache_position;
  a.S = S_; a.G = Hq / Hkv; a.eps = eps;
  return qd::kv_update_fp8_launch(a, S(stream));
}

int qd_kv_read_fp8(const void* k_cache, const void* v_cache, const void* k_scale, const void* v_scale, long stride_b,
                   long stride_h, long scale_stride_b, long scale_stride_h, int T, void* k_out, void* v_out, int B, int Hkv,
                   int rows, void* stream) {
  qd::KvReadFp8Args a;
  QD_TRY(check_cache(a.c, const_cast<void*>(k_cache), const_cast<void*>(v_cache), const_cast<void*>(k_scale),
                     const_cast<void*>(v_scale), stride_b, stride_h, scale_stride_b, scale_stride_h, T, B, Hkv));
  QD_REQUIRE(rows >= 0 && rows <= T, QD_ERR_SHAPE, "need 0 <= rows <= the capacity %d (rows=%d)", T, rows);
  if (B == 0 || rows == 0) return QD_OK;
  QD_REQUIRE(k_out && v_out && aligned(k_out, 16) && aligned(v_out, 16), QD_ERR_ARG,
             "k_out and v_out must be 16-byte aligned pointers");
  a.k = (u16*)k_out; a.v = (u16*)v_out; a.rows = rows;
  return qd::kv_read_fp8_launch(a, S(stream));
}

size_t qd_attention_fp8_workspace_bytes(int B, int Sq, int Hq, int Hkv, int T, int window, int sinks) {
  if (B < 1 || Sq < 1 || Hkv < 1 || Hq < Hkv || Hq % Hkv || T < 1 || window < 0 || sinks < 0) return 0;
  const int n = qd::attention_fp8_splits(B, Hkv, Sq, Hq / Hkv, T, window, sinks);
  return n > 1 ? (size_t)B * Hq * Sq * n * 130 * sizeof(float) : 0;
}

int qd_attention_fp8(const void* q, long q_sb, long q_sh, long q_ss, const void* k_cache, const void* v_cache,
                     const void* k_scale, const void* v_scale, long stride_b, long stride_h, long scale_stride_b,
                     long scale_stride_h, int T, const int64_t* cache_position, float scale, int window, int sinks,
                     void* out, int B, int Sq, int Hq, int Hkv, void* workspace, size_t workspace_bytes, void* stream) {
  qd::AttnFp8Args a;
  QD_TRY(check_cache(a.c, const_cast<void*>(k_cache), const_cast<void*>(v_cache), const_cast<void*>(k_scale),
                     const_cast<void*>(v_scale), stride_b, stride_h, scale_stride_b, scale_stride_h, T, B, Hkv));
  QD_REQUIRE(Hq >= Hkv && Hq % Hkv == 0, QD_ERR_SHAPE, "Hq must be a multiple of Hkv (Hq=%d Hkv=%d)", Hq, Hkv);
  QD_REQUIRE(Sq >= 0 && (long)Sq * (Hq / Hkv) <= (1L << 22) && (long)B * Hkv * ((long)Sq * (Hq / Hkv) / 64 + 1) < (1L << 23),
             QD_ERR_SHAPE, "too many query rows (B=%d Sq=%d Hq=%d)", B, Sq, Hq);
  QD_REQUIRE(window >= 0 && sinks >= 0, QD_ERR_ARG, "window and sinks must not be negative (%d, %d)", window, sinks);
  QD_REQUIRE(scale > 0.f && scale <= 3.402823466e38f, QD_ERR_ARG, "scale must be positive and finite (%g)", (double)scale);
  if (B == 0 || Sq == 0) return QD_OK;
  QD_REQUIRE(q && out && cache_position, QD_ERR_ARG, "null pointer");
  QD_REQUIRE(aligned(q, 16) && aligned(out, 16) && aligned(cache_position, 8) && ((q_sb | q_sh | q_ss) & 7) == 0, QD_ERR_ARG,
             "q rows and out must be 16-byte aligned");
  a.q = (const u16*)q; a.q_sb = q_sb; a.q_sh = q_sh; a.q_ss = q_ss;
  a.out = (u16*)out; a.cache_position = cache_position;
  a.Sq = Sq; a.G = Hq / Hkv; a.scale2 = scale * 1.44269504088896340736f; a.window = window; a.sinks = sinks;
  a.n_split = T == 0 ? 1 : qd::attention_fp8_splits(B, Hkv, Sq, a.G, T, window, sinks);
  if (a.n_split > 1) {
    const size_t need = qd_attention_fp8_workspace_bytes(B, Sq, Hq, Hkv, T, window, sinks);
    QD_REQUIRE(workspace && workspace_bytes >= need && aligned(workspace, 16), QD_ERR_WORKSPACE,
               "needs a 16-byte aligned workspace of %zu bytes (got %zu)", need, workspace_bytes);
    a.part_o = (float*)workspace;
    a.part_ml = a.part_o + (size_t)B * Hq * Sq * a.n_split * 128;
  }
  return qd::attention_fp8_launch(a, S(stream));
}

}  // extern "C"
