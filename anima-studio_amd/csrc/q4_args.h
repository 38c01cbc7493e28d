// Argument checks of the 4-bit weights and of the embedding rows (q4.hip).  Plain host code: no HIP call and no
// context, so every refusal can be reached without a device.  Each check returns a status and, when it is not
// ANIMA_OK, writes the message.
#pragma once

#include <algorithm>
#include <cstdint>
#include <cstdio>

#include "../../include/anima.h"

namespace anima {

constexpr int Q4_MAX_K = 1 << 20;         // of a product
constexpr int Q4_MAX_SIDE = 1 << 29;      // rows and outputs of a product (cut into launches by q4_part)
constexpr int64_t Q4_MAX_LDX = 1 << 22;   // floats between rows of a product's input (the interface's bound: offsets have 64 bits)
constexpr int64_t Q4_MAX_QUANT = (int64_t)1 << 34;  // weights of one conversion

struct Q4Msg {
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

// The largest part of a product of M rows and N columns that its kernels are launched for: a launch has fewer than 2^32 threads a
// dimension, and the pass before takes 64 a row and a column, the kernels for few rows 16 a column, tiles of 64 x 64 one for 16
// outputs.  Columns in whole pieces of 2^24, so that the parts' codes and scales are aligned as the whole's.
struct Q4Part {
  int64_t rows, cols;
};
inline Q4Part q4_part(int64_t M, int64_t N) {
  const int64_t side = (int64_t)1 << 24, cols = std::min(N, side);
  return {std::min(std::min(M, side), ((int64_t)1 << 35) / cols), cols};
}

inline bool q4_al(const void* p, int b) { return ((uintptr_t)p & (uintptr_t)(b - 1)) == 0; }
inline bool q4_group(int g) { return g == 32 || g == 64 || g == 128; }

inline int check_weight_quant_q4(const void* w, int w_bf16, int N, int K, int group, const uint8_t* q, const uint16_t* scale,
                                 const uint16_t* mid, Q4Msg fail) {
  if (N < 1 || K < 1 || !q4_group(group) || K % group)
    return fail(ANIMA_E_ARG, "anima_weight_quant_q4: N=%d K=%d in groups of %d (32, 64 or 128, K a multiple)", N, K, group);
  if (w_bf16 != 0 && w_bf16 != 1) return fail(ANIMA_E_ARG, "anima_weight_quant_q4: w_bf16=%d", w_bf16);
  if (!w || !q || !scale) return fail(ANIMA_E_ARG, "anima_weight_quant_q4: null pointer");
  if (!q4_al(w, 16) || !q4_al(q, 16) || !q4_al(scale, 2) || !q4_al(mid, 2))
    return fail(ANIMA_E_ARG, "anima_weight_quant_q4: w and q on 16 bytes, scale and mid on 2");
  if ((int64_t)N * K >= Q4_MAX_QUANT) return fail(ANIMA_E_UNSUPPORTED, "anima_weight_quant_q4: N=%d K=%d, 2^34 weights and more", N, K);
  return ANIMA_OK;
}

// A q4 weight's own fields.
inline int check_q4_weight(const char* who, const anima_weight* W, Q4Msg fail) {
  if (W->N < 1 || W->K < 1 || !q4_group(W->group) || W->K % W->group)
    return fail(ANIMA_E_ARG, "%s: a q4 weight needs groups of 32, 64 or 128 that divide K (N=%d K=%d group=%d)", who, W->N, W->K, W->group);
  if (!W->w || !W->group_scale) return fail(ANIMA_E_ARG, "%s: a q4 weight needs its codes and group scales", who);
  if (!q4_al(W->w, 16) || !q4_al(W->group_scale, 2) || !q4_al(W->group_mid, 2))
    return fail(ANIMA_E_ARG, "%s: the q4 weight's codes on 16 bytes, its scales and middles on 2", who);
  return ANIMA_OK;
}

// The rest of anima_linear's checks for a q4 weight (linear_launch has made the common ones).
inline int check_linear_q4(const anima_linear_desc* d, Q4Msg fail) {
  const anima_weight* W = d->W;
  if (int rc = check_q4_weight("anima_linear", W, fail)) return rc;
  if (d->acc_out) return fail(ANIMA_E_UNSUPPORTED, "anima_linear: acc_out applies to i8/w4 weights only");
  if (d->xq || d->xs) return fail(ANIMA_E_ARG, "anima_linear: q4 weights take fp32 rows x");
  if (d->precision != ANIMA_PREC_BF16 && d->precision != ANIMA_PREC_FP32)
    return fail(ANIMA_E_ARG, "anima_linear: unknown precision %d", d->precision);
  if (d->out_bf16 != 0 && d->out_bf16 != 1) return fail(ANIMA_E_ARG, "anima_linear: out_bf16=%d", d->out_bf16);
  if (d->out_bf16 && d->epilogue != ANIMA_EPI_STORE)
    return fail(ANIMA_E_UNSUPPORTED, "anima_linear: bf16 rows with the store epilogue only (%d)", d->epilogue);
  if (!q4_al(d->out, d->out_bf16 ? 2 : 4) || !q4_al(d->gate, 4) || !q4_al(d->add, 4) || !q4_al(W->bias, 4))
    return fail(ANIMA_E_ARG, "anima_linear: out, gate, add or bias off its element size");
  const int64_t ldx = d->ldx ? d->ldx : W->K;
  if (!d->x) return fail(ANIMA_E_ARG, "anima_linear: q4 weights need fp32 rows x");
  if (ldx < W->K || ldx % 4 || !q4_al(d->x, 16))
    return fail(ANIMA_E_ARG, "anima_linear: fp32 rows of at least K on 16 bytes (ldx=%lld, K=%d)", (long long)ldx, W->K);
  if (d->M > Q4_MAX_SIDE || W->N > Q4_MAX_SIDE || W->K > Q4_MAX_K || ldx > Q4_MAX_LDX)
    return fail(ANIMA_E_UNSUPPORTED, "anima_linear: M=%lld N=%d K=%d ldx=%lld (q4: at most %d rows and outputs, K %d, ldx %lld)",
                (long long)d->M, W->N, W->K, (long long)ldx, Q4_MAX_SIDE, Q4_MAX_K, (long long)Q4_MAX_LDX);
  return ANIMA_OK;
}

inline int check_embed_rows(const anima_weight* W, const int32_t* ids, int64_t T, const float* weights, const float* out, int64_t ldo,
                            Q4Msg fail) {
  if (!W) return fail(ANIMA_E_ARG, "anima_embed_rows: null table");
  if (W->kind != ANIMA_W_F32 && W->kind != ANIMA_W_BF16 && W->kind != ANIMA_W_Q4)
    return fail(ANIMA_E_UNSUPPORTED, "anima_embed_rows: a table of kind f32, bf16 or q4 (kind %d)", W->kind);
  if (T < 0 || T > 0x7fffffff || W->N < 1 || W->K < 1)
    return fail(ANIMA_E_ARG, "anima_embed_rows: T=%lld N=%d K=%d", (long long)T, W->N, W->K);
  if (W->K % 4) return fail(ANIMA_E_ARG, "anima_embed_rows: K=%d needs K %% 4 == 0", W->K);
  if (W->kind == ANIMA_W_Q4)
    if (int rc = check_q4_weight("anima_embed_rows", W, fail)) return rc;
  if (T == 0) return ANIMA_OK;
  if (!W->w || !ids || !out) return fail(ANIMA_E_ARG, "anima_embed_rows: null pointer");
  if (!q4_al(W->w, W->kind == ANIMA_W_BF16 ? 8 : 16) || !q4_al(ids, 4) || !q4_al(weights, 4) || !q4_al(out, 16))
    return fail(ANIMA_E_ARG, "anima_embed_rows: out and the table's rows of four on their size, ids and weights on 4 bytes");
  const int64_t ld = ldo ? ldo : W->K;
  if (ld < W->K || ld % 4) return fail(ANIMA_E_ARG, "anima_embed_rows: ldo=%lld (at least K=%d, a multiple of 4)", (long long)ld, W->K);
  return ANIMA_OK;
}

}  // namespace anima
