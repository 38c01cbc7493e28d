// Argument checks of the e4m3 operators (f8.hip).  Plain host code: no HIP call and no context, so
// every refusal can be reached without a device.  Each check returns a status and, when it is not
// ANIMA_OK, writes the message.
#pragma once

#include <cstdint>
#include <cstdio>

#include "../../include/anima.h"

namespace anima {

constexpr int F8_MAX_K = 1 << 20;         // of a product: 256 rows of a tile stay below 2^31 bytes
constexpr int64_t F8_MAX_LDX = 1 << 22;   // bytes between e4m3 rows of a product's input, likewise
constexpr int F8_NORM_MAX_COLS = 16384;   // a row in one workgroup's registers
constexpr int F8_MAX_SIDE = 1 << 29;      // rows and outputs of a product: tiles of 256 x 128 stay below 2^32 threads

// A launch has fewer than 2^32 threads a dimension, so large calls are cut into several.
constexpr int64_t F8_MAX_THREADS = 0xffffffff;
// Rows of a launch of quant_rows_f8_kernel: up to 16 threads to a block of 128 columns, 2^27 blocks (which are counted
// in 31 bits).
inline int64_t f8_quant_part(int K) { return ((int64_t)1 << 27) / ((K - 1) / 128 + 1); }
// Rows of a launch of residual_norm_kernel, whose workgroups of `threads` take one each.
constexpr int64_t f8_norm_part(int threads) { return ((int64_t)1 << 31) / threads; }

struct F8Msg {
  char* buf;
  size_t len;
  template <class... A>
  int operator()(int code, const char* fmt, A... args) const {
    snprintf(buf, len, fmt, args...);
    return code;
  }
  int operator()(int code, const char* text) const {
    snprintf(buf, len, "%s", text);
    return code;
  }
};

inline bool f8_al(const void* p, int b) { return ((uintptr_t)p & (uintptr_t)(b - 1)) == 0; }

inline int check_quant_rows_f8(const void* x, int x_bf16, int64_t M, int K, int64_t ldx, const uint8_t* q, const float* s,
                               F8Msg fail) {
  if (M < 0 || M > 0x7fffffff || K < 1) return fail(ANIMA_E_ARG, "anima_quant_rows_f8: M=%lld K=%d", (long long)M, K);
  if (x_bf16 != 0 && x_bf16 != 1) return fail(ANIMA_E_ARG, "anima_quant_rows_f8: x_bf16=%d", x_bf16);
  if (M == 0) return ANIMA_OK;
  if (!x || !q || !s) return fail(ANIMA_E_ARG, "anima_quant_rows_f8: null pointer");
  const int64_t ld = ldx ? ldx : K;
  if (K % 16) return fail(ANIMA_E_ARG, "anima_quant_rows_f8: K=%d needs K %% 16 == 0", K);
  if (ld < K || ld % (x_bf16 ? 8 : 4) || !f8_al(x, 16) || !f8_al(q, 16) || !f8_al(s, 4))
    return fail(ANIMA_E_ARG, "anima_quant_rows_f8: rows of x and q on 16 bytes (ldx=%lld, K=%d)", (long long)ld, K);
  return ANIMA_OK;
}

inline int check_weight_quant_f8(const void* w, int w_bf16, int N, int K, const uint8_t* q, const float* scale, F8Msg fail) {
  if (N < 1 || K < 1 || K % 16) return fail(ANIMA_E_ARG, "anima_weight_quant_f8: N=%d K=%d (K %% 16 == 0)", N, K);
  if (w_bf16 != 0 && w_bf16 != 1) return fail(ANIMA_E_ARG, "anima_weight_quant_f8: w_bf16=%d", w_bf16);
  if (!w || !q || !scale) return fail(ANIMA_E_ARG, "anima_weight_quant_f8: null pointer");
  if (!f8_al(w, 16) || !f8_al(q, 16) || !f8_al(scale, 4)) return fail(ANIMA_E_ARG, "anima_weight_quant_f8: w and q on 16 bytes");
  if ((int64_t)((N - 1) / 128 + 1) * ((K - 1) / 128 + 1) > F8_MAX_THREADS / 256)
    return fail(ANIMA_E_UNSUPPORTED, "anima_weight_quant_f8: N=%d K=%d, 2^24 blocks and more", N, K);
  return ANIMA_OK;
}

// The weight and the input rows of a product: e4m3 rows xq, else fp32 rows x.
inline int check_f8_operands(const char* who, const anima_weight* W, int64_t M, const float* x, int64_t ldx, const void* xq, const float* xs,
                             F8Msg fail) {
  if (W->N < 1 || W->K < 1 || W->K % 16 || W->K > F8_MAX_K)
    return fail(ANIMA_E_ARG, "%s: an f8 weight needs K %% 16 == 0 and K <= %d (N=%d K=%d)", who, F8_MAX_K, W->N, W->K);
  if (M > F8_MAX_SIDE || W->N > F8_MAX_SIDE)
    return fail(ANIMA_E_UNSUPPORTED, "%s: M=%lld N=%d, more than %d rows or outputs", who, (long long)M, W->N, F8_MAX_SIDE);
  if (!W->w || !W->scale) return fail(ANIMA_E_ARG, "%s: an f8 weight needs its data and block scales", who);
  if (!f8_al(W->w, 16) || !f8_al(W->scale, 4) || !f8_al(W->bias, 4))
    return fail(ANIMA_E_ARG, "%s: the f8 weight's data on 16 bytes, its scales and bias on 4", who);
  const int64_t ld = ldx ? ldx : W->K;
  if (ld < W->K) return fail(ANIMA_E_ARG, "%s: ldx=%lld < K=%d", who, (long long)ld, W->K);
  if (xq) {
    if (!xs) return fail(ANIMA_E_ARG, "%s: e4m3 rows need their scales xs", who);
    if (ld % 16 || !f8_al(xq, 16) || !f8_al(xs, 4)) return fail(ANIMA_E_ARG, "%s: e4m3 rows on 16 bytes (ldx=%lld)", who, (long long)ld);
    if (ld > F8_MAX_LDX) return fail(ANIMA_E_UNSUPPORTED, "%s: ldx=%lld above %lld", who, (long long)ld, (long long)F8_MAX_LDX);
  } else {
    if (!x) return fail(ANIMA_E_ARG, "%s: needs fp32 rows x or e4m3 rows xq", who);
    if (ld % 4 || !f8_al(x, 16)) return fail(ANIMA_E_ARG, "%s: fp32 rows on 16 bytes (ldx=%lld)", who, (long long)ld);
  }
  return ANIMA_OK;
}

// The rest of anima_linear's checks for an f8 weight (linear_launch has made the common ones).
inline int check_linear_f8(const anima_linear_desc* d, F8Msg fail) {
  if (d->acc_out) return fail(ANIMA_E_UNSUPPORTED, "anima_linear: acc_out applies to i8/w4 weights only");
  if (d->precision != ANIMA_PREC_BF16 && d->precision != ANIMA_PREC_FP32)
    return fail(ANIMA_E_ARG, "anima_linear: unknown precision %d", d->precision);
  if (d->out_bf16 != 0 && d->out_bf16 != 1) return fail(ANIMA_E_ARG, "anima_linear: out_bf16=%d", d->out_bf16);
  if (d->out_bf16 && d->epilogue != ANIMA_EPI_STORE)
    return fail(ANIMA_E_UNSUPPORTED, "anima_linear: bf16 rows with the store epilogue only (%d)", d->epilogue);
  if (!f8_al(d->out, d->out_bf16 ? 2 : 4) || !f8_al(d->gate, 4) || !f8_al(d->add, 4))
    return fail(ANIMA_E_ARG, "anima_linear: out, gate or add off its element size");
  return check_f8_operands("anima_linear", d->W, d->M, d->x, d->ldx, d->xq, d->xs, fail);
}

inline int check_linear_glu(const anima_glu_desc* d, F8Msg fail) {
  if (!d) return fail(ANIMA_E_ARG, "anima_linear_glu: null descriptor");
  const anima_weight *G = d->gate, *U = d->up;
  if (!G || !U) return fail(ANIMA_E_ARG, "anima_linear_glu: null weight");
  if (G->kind != ANIMA_W_F8 || U->kind != ANIMA_W_F8)
    return fail(ANIMA_E_UNSUPPORTED, "anima_linear_glu: f8 weights only (kinds %d, %d)", G->kind, U->kind);
  if (G->N != U->N || G->K != U->K)
    return fail(ANIMA_E_ARG, "anima_linear_glu: gate [%d][%d] and up [%d][%d] differ", G->N, G->K, U->N, U->K);
  if (d->M < 0 || d->M > 0x7fffffff) return fail(ANIMA_E_ARG, "anima_linear_glu: M=%lld", (long long)d->M);
  if (d->act < ANIMA_ACT_NONE || d->act > ANIMA_ACT_SILU) return fail(ANIMA_E_ARG, "anima_linear_glu: unknown act %d", d->act);
  if (d->precision != ANIMA_PREC_BF16 && d->precision != ANIMA_PREC_FP32)
    return fail(ANIMA_E_ARG, "anima_linear_glu: unknown precision %d", d->precision);
  if (d->M == 0) return ANIMA_OK;
  int rc = check_f8_operands("anima_linear_glu", G, d->M, d->x, d->ldx, d->xq, d->xs, fail);
  if (rc == ANIMA_OK) rc = check_f8_operands("anima_linear_glu", U, d->M, d->x, d->ldx, d->xq, d->xs, fail);
  if (rc != ANIMA_OK) return rc;
  if (d->out_q) {
    if (d->out) return fail(ANIMA_E_ARG, "anima_linear_glu: fp32 rows or e4m3 rows, not both");
    if (!d->out_s || !f8_al(d->out_s, 4)) return fail(ANIMA_E_ARG, "anima_linear_glu: e4m3 rows need out_s");
    if (G->N % 16 || !f8_al(d->out_q, 16))
      return fail(ANIMA_E_ARG, "anima_linear_glu: e4m3 rows on 16 bytes need N %% 16 == 0 (N=%d)", G->N);
  } else {
    if (!d->out || !f8_al(d->out, 4)) return fail(ANIMA_E_ARG, "anima_linear_glu: null out, or off 4 bytes");
    if (d->out_s) return fail(ANIMA_E_ARG, "anima_linear_glu: out_s without out_q");
    if (d->ldc && d->ldc < G->N) return fail(ANIMA_E_ARG, "anima_linear_glu: ldc=%lld < N=%d", (long long)d->ldc, G->N);
  }
  return ANIMA_OK;
}

inline int check_residual_norm(const anima_resnorm_desc* d, F8Msg fail) {
  if (!d) return fail(ANIMA_E_ARG, "anima_residual_norm: null descriptor");
  const int64_t C = d->cols;
  if (d->rows < 0 || d->rows > 0x7fffffff || C < 1 || C % 4 || C > F8_NORM_MAX_COLS)
    return fail(ANIMA_E_ARG, "anima_residual_norm: rows=%lld cols=%d (cols %% 4 == 0, at most %d)", (long long)d->rows, d->cols,
                F8_NORM_MAX_COLS);
  if (d->norm != ANIMA_NORM_RMS && d->norm != ANIMA_NORM_LAYER) return fail(ANIMA_E_ARG, "anima_residual_norm: unknown norm %d", d->norm);
  if (d->rows == 0) return ANIMA_OK;
  if (!(d->eps >= 0.0f)) return fail(ANIMA_E_ARG, "anima_residual_norm: eps=%g", (double)d->eps);
  if (!d->x || (!d->h && !d->q)) return fail(ANIMA_E_ARG, "anima_residual_norm: needs x and an output (h, q)");
  if (d->y_bf16 != 0 && d->y_bf16 != 1) return fail(ANIMA_E_ARG, "anima_residual_norm: y_bf16=%d", d->y_bf16);
  if ((d->q != nullptr) != (d->s != nullptr)) return fail(ANIMA_E_ARG, "anima_residual_norm: q and s go together");
  if (d->q && C % 16) return fail(ANIMA_E_ARG, "anima_residual_norm: e4m3 rows need cols %% 16 == 0 (cols=%d)", d->cols);
  if (!d->y && (d->post_w || d->gate)) return fail(ANIMA_E_ARG, "anima_residual_norm: post_w and gate apply to y");
  if ((d->shift != nullptr) != (d->scale != nullptr)) return fail(ANIMA_E_ARG, "anima_residual_norm: shift and scale go together");
  if (d->group_rows < 0) return fail(ANIMA_E_ARG, "anima_residual_norm: group_rows=%lld", (long long)d->group_rows);
  const int64_t ldx = d->ldx ? d->ldx : C, ldy = d->ldy ? d->ldy : C, ldh = d->ldh ? d->ldh : C, ldm = d->mod_ld ? d->mod_ld : C,
                ldg = d->gate_ld ? d->gate_ld : C;
  if (ldx < C || ldx % 4 || ldy < C || ldy % 4 || ldh < C || ldh % 4 || ldm < C || ldm % 4 || ldg < C || ldg % 4)
    return fail(ANIMA_E_ARG, "anima_residual_norm: row strides of at least cols=%d, multiples of 4", d->cols);
  // (a row's h is written when its own y has been read, other rows' y not yet)
  if (d->h && (const void*)d->h == d->y && (d->y_bf16 || (d->rows > 1 && ldh != ldy)))
    return fail(ANIMA_E_ARG, "anima_residual_norm: h may be an fp32 y of its own stride (ldh=%lld ldy=%lld)", (long long)ldh, (long long)ldy);
  if (!f8_al(d->y, d->y_bf16 ? 8 : 16)) return fail(ANIMA_E_ARG, "anima_residual_norm: rows of y on four elements");
  if (!f8_al(d->s, 4)) return fail(ANIMA_E_ARG, "anima_residual_norm: s off 4 bytes");
  const void* const p[] = {d->x, d->post_w, d->gate, d->norm_w, d->shift, d->scale, d->h, d->q};
  for (const void* v : p)
    if (!f8_al(v, 16)) return fail(ANIMA_E_ARG, "anima_residual_norm: rows and vectors on 16 bytes");
  return ANIMA_OK;
}

}  // namespace anima
