// 4-bit weights with group scales (ANIMA_W_Q4) and embedding rows.
//
//   w[n][k] = s[n][k / G] * (code - 8) + z[n][k / G]          G = 32, 64 or 128, s and z bf16
//
// s (code - 8) has at most 11 significant bits (8 of s, 3 of 1 .. 7, and 8 is a power of two), so it is exact in fp32,
// and w is one rounding away from it.
#include <algorithm>

#include "common.h"
#include "internal.h"
#include "q4_args.h"

namespace anima {

__device__ __forceinline__ float bf16_f(uint16_t b) { return __uint_as_float((uint32_t)b << 16); }

// ------------------------------------------------------------------ weights to 4 bits

template <class T>
__device__ __forceinline__ void ld8(const T* p, float (&v)[8]) {
  if constexpr (sizeof(T) == 2) {
    const uint4 r = *(const uint4*)p;
    const uint32_t u[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
      v[2 * i] = __uint_as_float(u[i] << 16);
      v[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
    }
  } else {
    const float4 a = *(const float4*)p, b = *(const float4*)(p + 4);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  }
}

// Eight weights a thread; the G / 8 neighbouring lanes of a group share its extremes.  One pass over the weight
// (a load-time conversion, bound by its bytes).
template <class T>
__global__ __launch_bounds__(256) void weight_quant_q4_kernel(const T* w, int64_t n8, int lanes, uint32_t* q, uint16_t* scale,
                                                              uint16_t* mid) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= n8) return;  // (whole groups: n8 is a multiple of `lanes`, a power of two)
  float v[8];
  ld8(w + 8 * i, v);
  float lo = v[0], hi = v[0];
  bool nan = v[0] != v[0];
#pragma unroll
  for (int j = 1; j < 8; j++) {
    lo = fminf(lo, v[j]);
    hi = fmaxf(hi, v[j]);
    nan |= v[j] != v[j];
  }
  if (nan) lo = hi = __builtin_nanf("");
  for (int s = 1; s < lanes; s <<= 1) {
    const float l2 = __shfl_xor(lo, s), h2 = __shfl_xor(hi, s);
    const bool bad = lo != lo || l2 != l2;
    lo = bad ? __builtin_nanf("") : fminf(lo, l2);
    hi = bad ? __builtin_nanf("") : fmaxf(hi, h2);
  }
  float s, z = 0.0f;
  if (mid) {
    s = (float)to_bf16((hi - lo) / 15.0f);
    z = (float)to_bf16(__builtin_fmaf(8.0f, s, lo));
  } else {
    s = (float)to_bf16((lo != lo ? lo : fmaxf(-lo, hi)) / 7.0f);
  }
  uint32_t codes = 0;
#pragma unroll
  for (int j = 0; j < 8; j++) {
    const float c = s == 0.0f ? 0.0f : fminf(fmaxf(rintf((v[j] - z) / s), -8.0f), 7.0f);
    codes |= (uint32_t)((int)c + 8) << (4 * j);
  }
  q[i] = codes;
  if ((i & (lanes - 1)) == 0) {
    scale[i / lanes] = __builtin_bit_cast(uint16_t, to_bf16(s));
    if (mid) mid[i / lanes] = __builtin_bit_cast(uint16_t, to_bf16(z));
  }
}

// ------------------------------------------------------------------ embedding rows

struct EmbedArgs {
  const void* w;
  const uint16_t* gs;
  const uint16_t* gz;
  const int32_t* ids;
  const float* weights;
  float* out;
  int64_t ldo;
  float scale;
  int N, K, G;
};

// four values of a table's row, from column k on
template <int KIND>
__device__ __forceinline__ f32x4 embed4(const EmbedArgs& a, int64_t row, int k) {
  if constexpr (KIND == ANIMA_W_F32) {
    return *(const f32x4*)((const float*)a.w + row * a.K + k);
  } else if constexpr (KIND == ANIMA_W_BF16) {
    const uint2 r = *(const uint2*)((const uint16_t*)a.w + row * a.K + k);
    return f32x4{__uint_as_float(r.x << 16), __uint_as_float(r.x & 0xffff0000u), __uint_as_float(r.y << 16),
                 __uint_as_float(r.y & 0xffff0000u)};
  } else {
    const int64_t g = row * (a.K / a.G) + k / a.G;
    const uint32_t c = *(const uint16_t*)((const uint8_t*)a.w + (row * a.K + k) / 2);
    const float s = bf16_f(a.gs[g]), z = a.gz ? bf16_f(a.gz[g]) : 0.0f;
    f32x4 v;
#pragma unroll
    for (int j = 0; j < 4; j++) v[j] = __builtin_fmaf((float)((int)((c >> (4 * j)) & 15) - 8), s, z);
    return v;
  }
}

// A workgroup of 256 threads per row, four columns a thread at a time.
template <int KIND>
__global__ __launch_bounds__(256) void embed_rows_kernel(EmbedArgs a) {
  const int64_t t = blockIdx.x;
  const int32_t id = a.ids[t];
  const bool in = id >= 0 && id < a.N;
  const float f = a.weights ? a.scale * a.weights[t] : a.scale;
  for (int k = 4 * threadIdx.x; k < a.K; k += 1024) {
    f32x4 v = {};
    if (in) v = embed4<KIND>(a, id, k) * f;
    *(f32x4*)(a.out + t * a.ldo + k) = v;
  }
}

// ------------------------------------------------------------------ products

struct Q4Args {
  const float* x;
  int64_t ldx;
  const uint8_t* w;
  const uint16_t* gs;
  const uint16_t* gz;
  const float* bias;
  void* out;
  int64_t ldc;
  float alpha;
  int act, epi;
  const float* gate;  // (at its offset)
  const float* add;
  int64_t ld_add;
  int M, N, K, G;
  int obf;
};

__device__ __forceinline__ float q4_act(float r, int act) {
  if (act == ANIMA_ACT_GELU) return gelu_erf(r);
  if (act == ANIMA_ACT_SILU) return silu_f(r);
  return r;
}

__device__ __forceinline__ void q4_store(const Q4Args& a, int64_t m, int n, float r) {
  r = r * a.alpha;
  if (a.bias) r = r + a.bias[n];
  if (a.add) r = r + a.add[m * a.ld_add + n];
  r = q4_act(r, a.act);
  if (a.obf) {
    ((bf16*)a.out)[m * a.ldc + n] = to_bf16(r);
    return;
  }
  float* c = (float*)a.out + m * a.ldc + n;
  if (a.epi == ANIMA_EPI_STORE) *c = r;
  else if (a.epi == ANIMA_EPI_RESID) *c = *c + r;
  else *c = __builtin_fmaf(a.gate[n], r, *c);
}

// One wave per output column and four rows, lanes striding k in pieces of eight, sums in fp32.
__global__ __launch_bounds__(256) void q4_rows_kernel(Q4Args a) {
  const int lane = threadIdx.x & 63;
  const int64_t n = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6), m0 = (int64_t)blockIdx.y * 4;
  if (n >= a.N) return;
  const int live = min(4, a.M - (int)m0);
  float acc[4] = {};
  for (int k = 8 * lane; k < a.K; k += 512) {
    const uint32_t c = *(const uint32_t*)(a.w + (n * a.K + k) / 2);
    const int64_t g = n * (a.K / a.G) + k / a.G;
    const float s = bf16_f(a.gs[g]), z = a.gz ? bf16_f(a.gz[g]) : 0.0f;
    float w[8];
#pragma unroll
    for (int j = 0; j < 8; j++) w[j] = __builtin_fmaf((float)((int)((c >> (4 * j)) & 15) - 8), s, z);
#pragma unroll
    for (int r = 0; r < 4; r++)
      if (r < live) {
        float x[8];
        ld8(a.x + (m0 + r) * a.ldx + k, x);
#pragma unroll
        for (int j = 0; j < 8; j++) acc[r] = __builtin_fmaf(x[j], w[j], acc[r]);
      }
  }
#pragma unroll
  for (int r = 0; r < 4; r++) {
    const float t = wave_sum(acc[r]);
    if (lane == 0 && r < live) q4_store(a, m0 + r, (int)n, t);
  }
}

// ------------------------------------------------------------------ host

namespace {
int refused(anima_ctx* c, int rc, const char* msg) { return fail(c, rc, "%s", msg); }
}  // namespace

int weight_quant_q4_launch(anima_ctx* c, const void* w, int w_bf16, int N, int K, int group, uint8_t* q, uint16_t* scale, uint16_t* mid) {
  char msg[256];
  if (int rc = check_weight_quant_q4(w, w_bf16, N, K, group, q, scale, mid, Q4Msg{msg, sizeof msg})) return refused(c, rc, msg);
  OnDevice on(c);
  const int64_t n8 = (int64_t)N * K / 8;
  const dim3 grid((unsigned)((n8 + 255) / 256));
  Launch L(c, "weight_quant.q4", 0.0, (double)N * K * (w_bf16 ? 2.5 : 4.5));
  if (w_bf16)
    hipLaunchKernelGGL(weight_quant_q4_kernel<uint16_t>, grid, dim3(256), 0, c->stream, (const uint16_t*)w, n8, group / 8, (uint32_t*)q, scale,
                       mid);
  else
    hipLaunchKernelGGL(weight_quant_q4_kernel<float>, grid, dim3(256), 0, c->stream, (const float*)w, n8, group / 8, (uint32_t*)q, scale, mid);
  return L.end();
}

int embed_rows_launch(anima_ctx* c, const anima_weight* W, const int32_t* ids, int64_t T, const float* weights, float scale, float* out,
                      int64_t ldo) {
  char msg[256];
  if (int rc = check_embed_rows(W, ids, T, weights, out, ldo, Q4Msg{msg, sizeof msg})) return refused(c, rc, msg);
  if (T == 0) return ANIMA_OK;
  OnDevice on(c);
  EmbedArgs a{W->w, W->group_scale, W->group_mid, ids, weights, out, ldo ? ldo : W->K, scale != 0.0f ? scale : 1.0f, W->N, W->K, W->group};
  Launch L(c, "embed_rows", 0.0, (double)T * W->K * (W->kind == ANIMA_W_F32 ? 8 : W->kind == ANIMA_W_BF16 ? 6 : 4.5));
  constexpr int64_t PART = 1 << 23;  // (a launch has fewer than 2^32 threads)
  for (int64_t t = 0; t < T; t += PART) {
    const dim3 grid((unsigned)std::min(PART, T - t));
    if (W->kind == ANIMA_W_F32) hipLaunchKernelGGL(embed_rows_kernel<ANIMA_W_F32>, grid, dim3(256), 0, c->stream, a);
    else if (W->kind == ANIMA_W_BF16) hipLaunchKernelGGL(embed_rows_kernel<ANIMA_W_BF16>, grid, dim3(256), 0, c->stream, a);
    else hipLaunchKernelGGL(embed_rows_kernel<ANIMA_W_Q4>, grid, dim3(256), 0, c->stream, a);
    a.ids += PART;
    if (a.weights) a.weights += PART;
    a.out += PART * a.ldo;
  }
  return L.end();
}

int linear_q4_launch(anima_ctx* c, const anima_linear_desc* d) {
  char msg[256];
  if (int rc = check_linear_q4(d, Q4Msg{msg, sizeof msg})) return refused(c, rc, msg);
  OnDevice on(c);
  const anima_weight* W = d->W;
  Q4Args a{d->x, d->ldx ? d->ldx : W->K, (const uint8_t*)W->w, W->group_scale, W->group_mid, W->bias, d->out, d->ldc ? d->ldc : W->N,
           d->alpha != 0.0f ? d->alpha : 1.0f, d->act, d->epilogue, d->epilogue == ANIMA_EPI_GATED ? d->gate + d->gate_off : nullptr, d->add,
           d->ld_add ? d->ld_add : W->N, (int)d->M, W->N, W->K, W->group, d->out_bf16};
  Launch L(c, "gemv.q4", 2.0 * a.M * a.N * a.K, 0.5 * a.N * a.K);
  constexpr int PART = 65535 * 4;  // (rows of a launch's grid)
  const int M = a.M;
  for (int m = 0; m < M; m += PART) {
    a.M = std::min(PART, M - m);
    hipLaunchKernelGGL(q4_rows_kernel, dim3((unsigned)((a.N + 3) / 4), (unsigned)((a.M + 3) / 4)), dim3(256), 0, c->stream, a);
    a.x += (int64_t)PART * a.ldx;
    if (a.add) a.add += (int64_t)PART * a.ld_add;
    a.out = (char*)a.out + (int64_t)PART * a.ldc * (a.obf ? 2 : 4);
  }
  return L.end();
}

}  // namespace anima
