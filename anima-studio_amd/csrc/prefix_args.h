// Argument checks of anima_attention_prefix (prefix.hip).  Plain host code: no HIP call and no context, so every
// refusal can be reached without a device.
#pragma once

#include <algorithm>
#include <cstdint>
#include <cstdio>

#include "../../include/anima.h"

namespace anima {

constexpr int64_t PREFIX_MAX_KEYS = 1 << 22;  // of the prefix and of a sequence, as anima_attention's Lk
constexpr int64_t PREFIX_MAX_ROWS = 1 << 28;  // of all sequences
constexpr int64_t PREFIX_MAX_LD = 1 << 20;    // elements between rows (the interface's bound: offsets have 64 bits)
constexpr int PREFIX_MAX_HEADS = 1 << 12;
constexpr int64_t PREFIX_MAX_VROWS = 1 << 30;  // rows times heads of a launch: 256 threads to 128 of them stay below 2^32

constexpr int PREFIX_BLOCK = 64;               // keys per block of the prepared layouts
constexpr int64_t PREFIX_MAX_PARTS = 1 << 26;  // rows of the parts of a split call: 32 threads each in the join

struct PrefixMsg {
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

// Bytes of a prefix's prepared K and V: rows in blocks of 64 (attention_kv_bytes of one batch element).
inline int64_t prefix_kv_bytes(int Hkv, int P, int precision) {
  return P < 1 ? 0 : 2 * (int64_t)Hkv * (((int64_t)P + 63) / 64 * 64) * 128 * (precision == ANIMA_PREC_BF16 ? 2 : 4);
}

// Tiles of 128 or 256 virtual rows (V = T * group of a kv head), and the parts that their key blocks are split into: what ends first
// by the times that a block of 64 keys, a workgroup's start and a join take, in us (fitted to 46 calls timed at all their plans: 1 to
// 17390 rows of 3 to 32 heads behind 0 to 8192 keys; this picks a plan within 2 % of the best on average).
// 266 rows of 32 heads behind 49 keys, bf16: 22.9 whole, 27.0 in three parts; 365 rows of 8 behind 467, fp32: 86 whole, 33 in 12.
struct PrefixPlan {
  int waves, nt, splits;  // of a tile; tiles of a kv head; parts
};
inline PrefixPlan prefix_plan(int num_cus, bool bf, int V, int group, int Hkv, int T, int P, int longest) {
  PrefixPlan plan{};
  double best = 0.0;
  const int64_t rows = (int64_t)Hkv * V;
  for (int nw = 4; nw <= 8; nw += 4) {
    const int nt = (int)(((int64_t)V + 32 * nw - 1) / (32 * nw));
    const int64_t span = std::min(T, (32 * nw + group - 1) / group + 1) + (int64_t)longest;  // own keys that a tile's rows see
    const int total = (P + PREFIX_BLOCK - 1) / PREFIX_BLOCK +
                      (int)std::min<int64_t>((T + PREFIX_BLOCK - 1) / PREFIX_BLOCK, (span + PREFIX_BLOCK - 1) / PREFIX_BLOCK + 1);
    for (int s = 1; s <= std::min(total, 64); s++) {
      if (s > 1 && s * rows > PREFIX_MAX_PARTS) break;
      const int64_t rounds = ((int64_t)nt * Hkv * s + num_cus - 1) / num_cus;
      const double block = !bf ? 6.0 : nw == 4 ? 1.2 : 1.4, start = bf ? 5.0 : 4.0, join = 2.0 + (double)s * rows * 1056 / 5e6;
      const double blocks = 0.5 * ((total + s - 1) / s) + 0.5 * total / s;  // (the longest part and the mean one)
      const double t = (double)rounds * (start + blocks * block) + (s > 1 ? join : 0.0);
      // (bf16, one wave of rows whose blocks are all copied at its start: whole.  1 to 30 rows behind 70 to 128 keys, at eight sizes of 3
      // to 32 heads: 14.4 to 16.4 us whole, 15.7 to 16.9 in two or three parts)
      if (plan.waves && (t >= best || (bf && s > 1 && V <= 32 && total <= 3))) continue;
      best = t;
      plan = {nw, nt, s};
    }
  }
  return plan;
}

// rows: the sum of the lengths; longest: the largest.
inline int check_attention_prefix(const anima_prefix_attn_desc* d, int64_t* rows, int* longest, PrefixMsg fail) {
  const char* const who = "anima_attention_prefix";
  const auto al = [](const void* p, int b) { return ((uintptr_t)p & (uintptr_t)(b - 1)) == 0; };
  *rows = 0;
  *longest = 0;
  if (!d) return fail(ANIMA_E_ARG, "%s: null descriptor", who);
  const int group = d->group == 0 ? 1 : d->group;
  if (d->D != 128) return fail(ANIMA_E_UNSUPPORTED, "%s: head dim %d (128)", who, d->D);
  if (d->B < 0 || (d->B > 0 && !d->len)) return fail(ANIMA_E_ARG, "%s: B=%d, or null len", who, d->B);
  if (d->H < 1 || group < 1 || d->H % group || d->H > PREFIX_MAX_HEADS)
    return fail(ANIMA_E_ARG, "%s: H=%d heads in groups of %d (at most %d heads)", who, d->H, d->group, PREFIX_MAX_HEADS);
  if (d->P < 0 || d->P > PREFIX_MAX_KEYS) return fail(ANIMA_E_ARG, "%s: P=%d outside [0, %lld]", who, d->P, (long long)PREFIX_MAX_KEYS);
  if (d->precision != ANIMA_PREC_BF16 && d->precision != ANIMA_PREC_FP32) return fail(ANIMA_E_ARG, "%s: unknown precision %d", who, d->precision);
  if (d->causal != 0 && d->causal != 1) return fail(ANIMA_E_ARG, "%s: causal=%d", who, d->causal);
  if (d->o_bf16 != 0 && d->o_bf16 != 1) return fail(ANIMA_E_ARG, "%s: o_bf16=%d", who, d->o_bf16);
  if (d->o_bf16 && d->precision != ANIMA_PREC_BF16) return fail(ANIMA_E_ARG, "%s: a bf16 O needs bf16 precision", who);
  for (int b = 0; b < d->B; b++) {
    if (d->len[b] < 0 || d->len[b] > PREFIX_MAX_KEYS)
      return fail(ANIMA_E_ARG, "%s: len[%d]=%d outside [0, %lld]", who, b, d->len[b], (long long)PREFIX_MAX_KEYS);
    if ((int64_t)d->len[b] * d->H > PREFIX_MAX_VROWS)
      return fail(ANIMA_E_UNSUPPORTED, "%s: len[%d]=%d rows of %d heads (at most 2^30 together)", who, b, d->len[b], d->H);
    *rows += d->len[b];
    if (d->len[b] > *longest) *longest = d->len[b];
    if (*rows > PREFIX_MAX_ROWS) return fail(ANIMA_E_UNSUPPORTED, "%s: more than %lld rows", who, (long long)PREFIX_MAX_ROWS);
  }
  if (*rows == 0) return ANIMA_OK;
  if (!d->q || !d->k || !d->v || !d->o) return fail(ANIMA_E_ARG, "%s: null q/k/v/o", who);
  const int64_t ld[4] = {d->ldq, d->ldk, d->ldv, d->ldo}, off[4] = {d->q_off, d->k_off, d->v_off, d->o_off};
  const int heads[4] = {d->H, d->H / group, d->H / group, d->H};
  const char* const nm[4] = {"q", "k", "v", "o"};
  for (int i = 0; i < 4; i++) {
    if (ld[i] % 4 || off[i] % 4 || off[i] < 0 || ld[i] < off[i] + (int64_t)heads[i] * 128)
      return fail(ANIMA_E_ARG, "%s: %s rows of %lld elements (a multiple of 4) cannot hold off %lld + %d heads x 128", who, nm[i],
                  (long long)ld[i], (long long)off[i], heads[i]);
    if (ld[i] > PREFIX_MAX_LD) return fail(ANIMA_E_UNSUPPORTED, "%s: %s rows %lld apart (at most %lld)", who, nm[i], (long long)ld[i], (long long)PREFIX_MAX_LD);
  }
  if (!al(d->q, 16) || !al(d->k, 16) || !al(d->v, 16) || !al(d->o, d->o_bf16 ? 8 : 16) || !al(d->q_norm, 16) || !al(d->k_norm, 16) ||
      !al(d->rope_cs, 16) || !al(d->prefix_kv, 16))
    return fail(ANIMA_E_ARG, "%s: q/k/v/o, prefix_kv, norms and rope_cs on 16 bytes (a bf16 o on 8)", who);
  if ((d->P > 0) != (d->prefix_kv != nullptr)) return fail(ANIMA_E_ARG, "%s: prefix_kv goes with P > 0 (P=%d)", who, d->P);
  const int64_t want = prefix_kv_bytes(d->H / group, d->P, d->precision);
  if (d->prefix_kv_bytes != want)
    return fail(ANIMA_E_ARG, "%s: prefix_kv_bytes=%lld, but %d kv heads and P=%d at this precision take %lld", who,
                (long long)d->prefix_kv_bytes, d->H / group, d->P, (long long)want);
  if (d->rope_cs) {
    const int64_t table = d->rope_sin_off / 64;
    if (d->rope_sin_off <= 0 || d->rope_sin_off % 64 || table < (int64_t)d->P + *longest)
      return fail(ANIMA_E_ARG, "%s: rope_sin_off=%lld must be rows*64 with rows >= P + longest = %lld", who, (long long)d->rope_sin_off,
                  (long long)d->P + *longest);
  }
  if (!(d->eps >= 0.0f)) return fail(ANIMA_E_ARG, "%s: eps=%g", who, (double)d->eps);
  return ANIMA_OK;
}

// One sequence's keys and values as a prefix: what anima_attention_prefix asks of them, at positions 0 ...
inline int check_attention_prefix_prepare(const anima_prefix_attn_desc* d, const void* out, int64_t bytes, PrefixMsg fail) {
  const char* const who = "anima_attention_prefix_prepare";
  if (!d || !out) return fail(ANIMA_E_ARG, "%s: null descriptor or output", who);
  if (d->B != 1 || !d->len || d->len[0] < 1) return fail(ANIMA_E_ARG, "%s: one sequence of rows (B=%d)", who, d->B);
  if (d->P || d->prefix_kv) return fail(ANIMA_E_ARG, "%s: P=%d, a prefix starts at 0 and has none before it", who, d->P);
  anima_prefix_attn_desc k = *d;  // (q and o take no part)
  k.q = d->k;
  k.ldq = (int64_t)d->H * 128;
  k.q_off = 0;
  k.q_norm = nullptr;
  k.o = (float*)out;
  k.ldo = k.ldq;
  k.o_off = 0;
  k.o_bf16 = 0;
  k.prefix_kv_bytes = 0;
  int64_t rows;
  int longest;
  if (int rc = check_attention_prefix(&k, &rows, &longest, fail)) return rc;
  const int Hkv = d->H / (d->group == 0 ? 1 : d->group);
  const int64_t want = prefix_kv_bytes(Hkv, d->len[0], d->precision);
  if (bytes != want)
    return fail(ANIMA_E_ARG, "%s: %lld bytes, but %d kv heads and %d rows at this precision take %lld", who, (long long)bytes, Hkv, d->len[0],
                (long long)want);
  return ANIMA_OK;
}

}  // namespace anima
