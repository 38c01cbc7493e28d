// Attention of many sequences behind one shared prefix (anima_attention_prefix).
//
//   o[i] = sum_j p_ij v_j,  p_ij = exp(scale q_i . k_j) / sum_j,  j over the P prefix keys and the row's own
//   sequence's keys (causal: up to itself)
//
// The sequences' rows are packed, so the prefix is one product for all of them: tiles of rows run over the prefix's key
// blocks whatever sequence the rows belong to, then over the packed keys of their own sequences, masked by each row's
// range of them.  The packed K (normed, rotated at P + place) and V are laid out as the prefix's are, in one pass.
#include <algorithm>

#include "common.h"
#include "internal.h"
#include "prefix_args.h"

namespace anima {

constexpr int PHD = 128;      // head dim
constexpr int PBK = 64;       // keys per block of the prepared layouts
constexpr int PSEQ = 256;     // sequences of one launch (their first rows go with the kernel's arguments)
constexpr float LOG2E = 1.4426950408889634f;

struct PrefixSeqs {
  int n;                // sequences
  int start[PSEQ + 1];  // first packed row of each, then the number of rows
};

// The sequence of packed row l (rows past the last count to the last one).
__device__ __forceinline__ int seq_of(const PrefixSeqs& s, int l) {
  int lo = 0, hi = s.n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (s.start[mid] <= l) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

struct PrefixArgs {
  const float* q;
  int64_t ldq;
  const float* k;
  int64_t ldk;
  const float* v;
  int64_t ldv;
  void* o;
  int64_t ldo;
  const void* pk;   // prefix: K [Hkv][Pp][128], V^T [Hkv][128][Pp]
  const void* pvt;
  void* ok;         // own: K [Hkv][Tp][128], V^T [Hkv][128][Tp]
  void* ovt;
  const float* qn;
  const float* kn;
  const float* cs;
  int64_t sin_off;
  float eps, c;     // c = scale * log2(e)
  int T, Tp, P, Pp, H, Hkv, group, causal, obf;
  PrefixSeqs seq;
};

// One packed row of q or k in a wave, lane l holding dims l and l + 64: RMS norm, then the rotation.
__device__ __forceinline__ void row_norm_rope(const PrefixArgs& a, const float* w, int pos, float& x0, float& x1) {
  const int lane = threadIdx.x & 63;
  if (w) {
    const float rn = 1.0f / sqrtf(wave_sum(x0 * x0 + x1 * x1) / 128.0f + a.eps);
    x0 = x0 * rn * w[lane];
    x1 = x1 * rn * w[lane + 64];
  }
  if (a.cs) {
    const float c = a.cs[(int64_t)pos * 64 + lane], s = a.cs[a.sin_off + (int64_t)pos * 64 + lane];
    const float y0 = x0 * c - x1 * s;
    x1 = x1 * c + x0 * s;
    x0 = y0;
  }
}

// place of key l in a V^T row: the bf16 form keeps each 16 keys as 0-3, 8-11, 4-7, 12-15
template <class T>
__device__ __forceinline__ int vt_place(int l) {
  if (sizeof(T) == 4) return l;
  const int r = l & 15;
  return (l & ~15) | (r & 3) | ((r & 4) << 1) | ((r & 8) >> 1);
}

// A wave per packed row and kv head; rows T .. Tp are zeros.  A key whose K or V is not finite gets a K of NaN and a V of
// zeros: every row that sees it becomes NaN, and where it is masked its weight of 0 meets no NaN in V.
template <class T>
__global__ __launch_bounds__(256) void prefix_prep_kernel(PrefixArgs a) {
  const int l = blockIdx.x * 4 + (threadIdx.x >> 6), hk = blockIdx.y, lane = threadIdx.x & 63;
  if (l >= a.Tp) return;
  float k0 = 0.0f, k1 = 0.0f, v0 = 0.0f, v1 = 0.0f;
  if (l < a.T) {
    const float* k = a.k + (int64_t)l * a.ldk + hk * PHD;
    const float* v = a.v + (int64_t)l * a.ldv + hk * PHD;
    k0 = k[lane];
    k1 = k[lane + 64];
    v0 = v[lane];
    v1 = v[lane + 64];
    row_norm_rope(a, a.kn, a.P + l - a.seq.start[seq_of(a.seq, l)], k0, k1);
  }
  k0 = (float)(T)k0;
  k1 = (float)(T)k1;
  v0 = (float)(T)v0;
  v1 = (float)(T)v1;
  if (__builtin_amdgcn_ballot_w64(!(fabsf(k0) < INFINITY && fabsf(k1) < INFINITY && fabsf(v0) < INFINITY && fabsf(v1) < INFINITY))) {
    k0 = k1 = __builtin_nanf("");
    v0 = v1 = 0.0f;
  }
  T* kd = (T*)a.ok + ((int64_t)hk * a.Tp + l) * PHD;
  kd[lane] = (T)k0;
  kd[lane + 64] = (T)k1;
  T* vd = (T*)a.ovt + (int64_t)hk * PHD * a.Tp + vt_place<T>(l);
  vd[(int64_t)lane * a.Tp] = (T)v0;
  vd[(int64_t)(lane + 64) * a.Tp] = (T)v1;
}

// A wave per packed row and head, one key at a time, running maximum and sum.
template <class T>
__global__ __launch_bounds__(256) void prefix_rows_kernel(PrefixArgs a) {
  const int64_t i = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const int l = (int)(i / a.H), h = (int)(i - (int64_t)l * a.H), hk = h / a.group;
  if (l >= a.T) return;
  const int b = seq_of(a.seq, l), lo = a.seq.start[b], hi = a.causal ? l + 1 : a.seq.start[b + 1];
  float q0 = a.q[(int64_t)l * a.ldq + h * PHD + lane], q1 = a.q[(int64_t)l * a.ldq + h * PHD + lane + 64];
  row_norm_rope(a, a.qn, a.P + l - lo, q0, q1);
  q0 = (float)(T)(q0 * a.c);
  q1 = (float)(T)(q1 * a.c);
  float m = -INFINITY, sum = 0.0f, o0 = 0.0f, o1 = 0.0f;
  auto keys = [&](const T* k, const T* vt, int64_t ld, int j0, int j1) {
    k += (int64_t)hk * ld * PHD;
    vt += (int64_t)hk * ld * PHD;
    for (int j = j0; j < j1; j++) {
      const float s = wave_sum(q0 * (float)k[(int64_t)j * PHD + lane] + q1 * (float)k[(int64_t)j * PHD + lane + 64]);
      if (s > m) {
        const float r = __builtin_amdgcn_exp2f(m - s);  // (0 at the first key)
        sum *= r;
        o0 *= r;
        o1 *= r;
        m = s;
      }
      const float p = __builtin_amdgcn_exp2f(s - m);
      const int jp = vt_place<T>(j);
      sum += p;
      o0 += p * (float)vt[lane * ld + jp];
      o1 += p * (float)vt[(lane + 64) * ld + jp];
    }
  };
  keys((const T*)a.pk, (const T*)a.pvt, a.Pp, 0, a.P);
  keys((const T*)a.ok, (const T*)a.ovt, a.Tp, lo, hi);
  const float inv = 1.0f / sum;
  if (a.obf) {
    bf16* o = (bf16*)a.o + (int64_t)l * a.ldo + h * PHD;
    o[lane] = to_bf16(o0 * inv);
    o[lane + 64] = to_bf16(o1 * inv);
  } else {
    float* o = (float*)a.o + (int64_t)l * a.ldo + h * PHD;
    o[lane] = o0 * inv;
    o[lane + 64] = o1 * inv;
  }
}

// ------------------------------------------------------------------ host

// The sequences of one launch, which the arguments describe: their keys and values into the workspace, then the rows.
template <class T>
static int prefix_part(anima_ctx* c, PrefixArgs& a) {
  void* ws = nullptr;
  const size_t plane = (size_t)a.Hkv * a.Tp * PHD * sizeof(T);
  if (int rc = workspace(c, 2 * plane, &ws)) return rc;
  a.ok = ws;
  a.ovt = (char*)ws + plane;
  {
    Launch L(c, "attn.prefix_prep", 0.0, (double)a.Hkv * a.T * PHD * (8.0 + 2 * sizeof(T)));
    hipLaunchKernelGGL(prefix_prep_kernel<T>, dim3((unsigned)(a.Tp / 4), (unsigned)a.Hkv), dim3(256), 0, c->stream, a);
    if (int rc = L.end()) return rc;
  }
  Launch L(c, "attn.prefix", 4.0 * a.T * a.H * PHD * a.P, 0.0);
  hipLaunchKernelGGL(prefix_rows_kernel<T>, dim3((unsigned)(((int64_t)a.T * a.H + 3) / 4)), dim3(256), 0, c->stream, a);
  return L.end();
}

int attention_prefix_launch(anima_ctx* c, const anima_prefix_attn_desc* d) {
  char msg[256];
  int64_t rows = 0;
  int longest = 0;
  if (int rc = check_attention_prefix(d, &rows, &longest, PrefixMsg{msg, sizeof msg})) return fail(c, rc, "%s", msg);
  if (rows == 0) return ANIMA_OK;
  OnDevice on(c);
  const bool bf = d->precision == ANIMA_PREC_BF16;
  PrefixArgs a;
  a.group = d->group == 0 ? 1 : d->group;
  a.H = d->H;
  a.Hkv = d->H / a.group;
  a.P = d->P;
  a.Pp = (d->P + PBK - 1) / PBK * PBK;
  a.pk = d->prefix_kv;
  a.pvt = (const char*)d->prefix_kv + (int64_t)a.Hkv * a.Pp * PHD * (bf ? 2 : 4);
  a.ldq = d->ldq;
  a.ldk = d->ldk;
  a.ldv = d->ldv;
  a.ldo = d->ldo;
  a.qn = d->q_norm;
  a.kn = d->k_norm;
  a.cs = d->rope_cs;
  a.sin_off = d->rope_sin_off;
  a.eps = d->eps;
  a.c = (d->scale != 0.0f ? d->scale : 1.0f / sqrtf((float)PHD)) * LOG2E;
  a.causal = d->causal;
  a.obf = d->o_bf16;
  int64_t row = 0;
  for (int b = 0; b < d->B;) {
    // the next sequences, as many as one launch describes and 2^22 rows hold
    a.seq.n = 0;
    int64_t t = 0;
    while (b < d->B && a.seq.n < PSEQ && t + d->len[b] <= PREFIX_MAX_KEYS) {
      if (d->len[b] > 0) {
        a.seq.start[a.seq.n++] = (int)t;
        t += d->len[b];
      }
      b++;
    }
    if (t == 0) continue;
    a.seq.start[a.seq.n] = (int)t;
    a.T = (int)t;
    a.Tp = (int)((t + PBK - 1) / PBK * PBK);
    a.q = d->q + d->q_off + row * d->ldq;
    a.k = d->k + d->k_off + row * d->ldk;
    a.v = d->v + d->v_off + row * d->ldv;
    a.o = (char*)d->o + (d->o_off + row * d->ldo) * (bf && d->o_bf16 ? 2 : 4);
    if (int rc = bf ? prefix_part<bf16>(c, a) : prefix_part<float>(c, a)) return rc;
    row += t;
  }
  return ANIMA_OK;
}

}  // namespace anima
