// 4-bit weights with group scales (ANIMA_W_Q4) and embedding rows.
//
//   w[n][k] = s[n][k / G] * (code - 8) + z[n][k / G]          G = 32, 64 or 128, s and z bf16
//
// s (code - 8) has at most 11 significant bits (8 of s, 3 of 1 .. 7, and 8 is a power of two), so it is exact in fp32,
// and w is one rounding away from it.
#include <algorithm>
#include <type_traits>

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

// Eight weights a thread; the G / 8 neighbouring lanes of a group share its extremes.  One pass over the weight, a load-time
// conversion (151936 x 1024 from bf16: 132 us, 3.0 TB/s: the divisions, which the definition rounds, beside the bytes).
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

// A workgroup of 256 threads per row, four columns a thread at a time.  Bound by the rows' bytes: 8191 rows of 2048 from 4 bits 13.5
// us, 77 MB at 5.7 TB/s; one row of 1024 1.3 us.
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

// What an output's epilogue reads, asked for before its sum is there.
template <class V>
struct Q4Ends {
  V bias, add, gate, c;
};

__device__ __forceinline__ Q4Ends<float> q4_ask(const Q4Args& a, int64_t m, int n) {
  Q4Ends<float> e{};
  if (a.bias) e.bias = a.bias[n];
  if (a.add) e.add = a.add[m * a.ld_add + n];
  if (a.epi == ANIMA_EPI_GATED) e.gate = a.gate[n];
  if (a.epi != ANIMA_EPI_STORE) e.c = ((const float*)a.out)[m * a.ldc + n];
  return e;
}

__device__ __forceinline__ void q4_leave(const Q4Args& a, int64_t m, int n, float r, const Q4Ends<float>& e) {
  r = q4_act(r * a.alpha + e.bias + e.add, a.act);
  if (a.obf) {
    ((bf16*)a.out)[m * a.ldc + n] = to_bf16(r);
    return;
  }
  ((float*)a.out)[m * a.ldc + n] = a.epi == ANIMA_EPI_GATED ? __builtin_fmaf(e.gate, r, e.c) : r + e.c;
}

// The same for four columns from n (a multiple of 4) on, fewer at the row's end.  Rows may start anywhere: the memory takes 16 bytes
// of any four columns at once (2770 x 6019 x 256 in one term, a column at a time against so: 95 and 59 us by the largest tile,
// 52 and 39 by the smallest).
typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));
typedef __bf16 bf16x4_any __attribute__((ext_vector_type(4), aligned(2)));

__device__ __forceinline__ Q4Ends<f32x4> q4_ask4(const Q4Args& a, int64_t m, int n) {
  Q4Ends<f32x4> e{};
  if (n + 4 > a.N) return e;
  if (a.bias) e.bias = *(const f32x4_any*)(a.bias + n);
  if (a.add) e.add = *(const f32x4_any*)(a.add + m * a.ld_add + n);
  if (a.epi == ANIMA_EPI_GATED) e.gate = *(const f32x4_any*)(a.gate + n);
  if (a.epi != ANIMA_EPI_STORE) e.c = *(const f32x4_any*)((const float*)a.out + m * a.ldc + n);
  return e;
}

__device__ __forceinline__ void q4_leave4(const Q4Args& a, int64_t m, int n, f32x4 r, const Q4Ends<f32x4>& e) {
  if (n + 4 > a.N) {
#pragma unroll 1
    for (int i = 0; n + i < a.N; i++) q4_leave(a, m, n + i, i == 0 ? r[0] : i == 1 ? r[1] : r[2], q4_ask(a, m, n + i));
    return;
  }
  r = r * a.alpha + e.bias + e.add;
  if (a.act == ANIMA_ACT_GELU) {
#pragma unroll
    for (int i = 0; i < 4; i++) r[i] = gelu_erf(r[i]);
  } else if (a.act == ANIMA_ACT_SILU) {
#pragma unroll
    for (int i = 0; i < 4; i++) r[i] = silu_f(r[i]);
  }
  if (a.obf) {
    *(bf16x4_any*)((bf16*)a.out + m * a.ldc + n) = bf16x4_any{to_bf16(r[0]), to_bf16(r[1]), to_bf16(r[2]), to_bf16(r[3])};
    return;
  }
  if (a.epi == ANIMA_EPI_GATED) {
#pragma unroll
    for (int i = 0; i < 4; i++) r[i] = __builtin_fmaf(e.gate[i], r[i], e.c[i]);
  } else {
    r = r + e.c;
  }
  *(f32x4_any*)((float*)a.out + m * a.ldc + n) = r;
}

// One to four rows (a group of blockIdx.y) on the vector units, in fp32: a wave takes U columns, a lane 16 consecutive k of each 1024 (eight bytes of
// codes, one group).  x goes through LDS, quad j of lane l's 16 at [j][l], so that the reads touch every bank once.  A code with its
// highest bit turned is c - 8 in two's complement: in a byte's upper half 16 (c - 8), one conversion away from a
// float, and s takes the 16.
// Bound by its launch and one trip to memory for the codes: 1 x 4096 x 1024 3.6 us, 1 x 8192 x 2048 in groups of 32 5.2 us (10.6 MB).
// More columns a wave share x's way through LDS, fewer fill more CUs: four from N = 4096 on, two from 2048 (four rows of 8192 x 2048:
// 8.2 us, 13.7 a column a wave; one of 1024 x 8192: 5.7 a column a wave, 9.1 four).
template <int MR, int U>
__global__ __launch_bounds__(256) void q4_gemv_kernel(Q4Args a) {
  __shared__ f32x4 xs[2][MR][256];
  const int tid = threadIdx.x, lane = tid & 63, n0 = (blockIdx.x * 4 + (tid >> 6)) * U, KG = a.K / a.G, lg = 31 - __builtin_clz(a.G);
  if (const int64_t m0 = (int64_t)blockIdx.y * MR) {  // this group's rows
    a.x += m0 * a.ldx;
    a.out = (char*)a.out + m0 * a.ldc * (a.obf ? 2 : 4);
    if (a.add) a.add += m0 * a.ld_add;
    a.M -= (int)m0;
  }
  float acc[MR][U] = {};
  // the output that this lane ends with, if it has any
  int first = 0;
#pragma unroll
  for (int d = 32, cnt = U; cnt > 1; d >>= 1) {
    cnt >>= 1;
    if (lane & d) first += cnt;
  }
  const int no = n0 + first;
  const bool ends = (lane & (64 / U - 1)) == 0 && no < a.N;
  Q4Ends<float> ask[MR] = {};
  if (ends)
#pragma unroll
    for (int m = 0; m < MR; m++)
      if (m < a.M) ask[m] = q4_ask(a, m, no);
  const uint8_t* w[U];
  const uint16_t *gs[U], *gz[U];
#pragma unroll
  for (int u = 0; u < U; u++) {
    const int64_t n = min(n0 + u, a.N - 1);
    w[u] = a.w + n * (a.K / 2);
    gs[u] = a.gs + n * KG;
    gz[u] = a.gz ? a.gz + n * KG : gs[u];
  }
  for (int k0 = 0, p = 0; k0 < a.K; k0 += 1024, p ^= 1) {
    const int k = min(k0 + 16 * lane, a.K - 16);  // (past the row's end its last 16: they meet zeros of x)
    uint2 c[U];
    uint16_t s[U], z[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
      c[u] = *(const uint2*)(w[u] + k / 2);
      s[u] = gs[u][k >> lg];
      z[u] = gz[u][k >> lg];
    }
#pragma unroll
    for (int m = 0; m < MR; m++) {
      const int kq = k0 + 4 * tid;
      const f32x4 v = *(const f32x4*)(a.x + min(m, a.M - 1) * a.ldx + min(kq, a.K - 4));
      xs[p][m][(tid & 3) * 64 + (tid >> 2)] = kq < a.K ? v : f32x4{};
    }
    __syncthreads();  // (one a turn: the other buffer's readers are past it by the next)
#pragma unroll
    for (int m = 0; m < MR; m++) {
      float t[U] = {}, sx = 0.0f;
#pragma unroll
      for (int j = 0; j < 4; j++) {  // quad j: half a word of codes
        const f32x4 x = xs[p][m][j * 64 + lane];
        sx += (x[0] + x[1]) + (x[2] + x[3]);
#pragma unroll
        for (int u = 0; u < U; u++) {
          const uint32_t v = (j < 2 ? c[u].x : c[u].y) ^ 0x88888888u;
          const uint32_t half[2] = {(v << 4) & 0xf0f0f0f0u, v & 0xf0f0f0f0u};  // (even and odd k)
#pragma unroll
          for (int e = 0; e < 4; e++)
            t[u] = __builtin_fmaf(x[e], (float)(int8_t)(half[e & 1] >> (16 * (j & 1) + 8 * (e >> 1))), t[u]);
        }
      }
#pragma unroll
      for (int u = 0; u < U; u++) {
        acc[m][u] = __builtin_fmaf(bf16_f(s[u]) * 0.0625f, t[u], acc[m][u]);
        if (a.gz) acc[m][u] = __builtin_fmaf(bf16_f(z[u]), sx, acc[m][u]);
      }
    }
  }
  // The sums over the lanes: while a lane holds several outputs, the two of a pair keep half of them each.
#pragma unroll
  for (int m = 0; m < MR; m++) {
    int cnt = U;
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) {
      if (cnt > 1) {
        cnt >>= 1;
        const bool hi = lane & d;
#pragma unroll
        for (int u = 0; u < U / 2; u++)
          if (u < cnt) {
            const float send = hi ? acc[m][u] : acc[m][u + cnt], keep = hi ? acc[m][u + cnt] : acc[m][u];
            acc[m][u] = keep + __shfl_xor(send, d);
          }
      } else {
        acc[m][0] += __shfl_xor(acc[m][0], d);
      }
    }
    if (ends && m < a.M) q4_leave(a, m, no, acc[m][0], ask[m]);
  }
}

// ------------------------------------------------------------------ products of many rows
//
// On the f16 matrix cores.  A row of x, times a power of two that brings its largest value to 2^14 .. 2^15, is the sum of
// two f16 terms to 2^-23 of each value (or 2^-39 of the largest); ANIMA_PREC_BF16 keeps the first term, 11 bits (or 2^-39).
// s (c - 8), times a power of two for the whole column that brings its largest scale to 2^11 .. 2^12, is one f16 value: exact
// for scales from 2^-28 of the largest on; a smaller one is off by at most 2^-36 of the largest.  Both powers come off the sums at
// the end, so the k loop has nothing but matrix products and the codes' decode.  The middles' part, sum_g z[n][g] (sum of x
// over group g), is a small product of bf16 terms.

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// 2^e as a float, e from -126 to 127
__device__ __forceinline__ float pow2f(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// The exponent that brings a largest magnitude to [2^top, 2^(top + 1)); 0 for zeros, infinities and NaN.
__device__ __forceinline__ int q4_exp(float amax, int top) {
  const int b = (int)(__float_as_uint(amax) >> 23);
  return amax == 0.0f || b == 255 ? 0 : min(top + 127 - b, 120);
}

struct Q4Prep {
  const float* x;
  int64_t ldx;
  _Float16* xh;   // rows of Kp, ldp apart, each eight values in the order k 0 4 1 5 2 6 3 7 (the decode's), zeros from K on;
                  // or (frag) as the 32 x 32 x 16 products take them: [rows / 32][Kp / 16][k / 8 % 2][row % 32][8]
  _Float16* xl;   // the second terms, or NULL
  float* rm;      // [M] what x's power comes off with
  bf16* sx;       // [3][M][KGp] group sums of x with x's power, three terms each, or NULL
  bf16* zp;       // [N][KGp] the middles with the column's power, zeros from K / G on
  const uint16_t* gs;
  const uint16_t* gz;
  float* rn;      // [N] what the column's power comes off with
  int64_t ldp;    // values between the terms' rows
  int M, N, K, Kp, G, KGp, rows;  // rows: workgroups of x rows (four each), the rest are of columns
  int frag;
};

// A wave per row of x (NV: pieces of 512 k that a wave holds; 0: two passes over the row, the second from the caches), or per
// column's scales.  Bound by memory (8192 x 2048 into one term: 101 MB, 16 us), few rows by a launch and a trip (4 us).
template <int NV>
__global__ __launch_bounds__(256) void q4_prep_kernel(Q4Prep a) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if ((int)blockIdx.x >= a.rows) {
    const int64_t n = (int64_t)(blockIdx.x - a.rows) * 4 + wave;
    if (n >= a.N) return;
    const int KG = a.K / a.G;
    float m = 0.0f;
    for (int g = lane; g < KG; g += 64) m = fmaxf(m, fabsf(bf16_f(a.gs[n * KG + g])));
    m = wave_max(m);
    int e = a.rn ? q4_exp(m, 11) : 0;
    if (a.zp) {
      float mz = 0.0f;
      for (int g = lane; g < KG; g += 64) mz = fmaxf(mz, fabsf(bf16_f(a.gz[n * KG + g])));
      mz = wave_max(mz);
      // (beside middles of 2^78 scales these give way: 2^20 values of x below 2^15 and middles below 2^89 have finite sums)
      if (a.rn && mz != 0.0f) e = min(e, q4_exp(mz, 88));
      for (int g = lane; g < a.KGp; g += 64) a.zp[n * a.KGp + g] = to_bf16(g < KG ? bf16_f(a.gz[n * KG + g]) * pow2f(e) : 0.0f);
    }
    if (a.rn && lane == 0) a.rn[n] = pow2f(-e);
    return;
  }
  const int64_t m = (int64_t)blockIdx.x * 4 + wave;
  if (m >= a.M) return;
  const float* x = a.x + m * a.ldx;
  const auto piece = [&](int k, float (&v)[8]) __attribute__((always_inline)) {  // (past K: zeros)
    const bool in = k < a.K;
    ld8(x + (in ? k : 0), v);
    if (!in)
#pragma unroll
      for (int j = 0; j < 8; j++) v[j] = 0.0f;
  };
  const auto largest = [](const float (&v)[8], float mx) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < 8; j++) mx = fmaxf(mx, fabsf(v[j]));
    return mx;
  };
  const auto leave = [&](int k, const float (&v)[8], float f) __attribute__((always_inline)) {
    if (a.sx) {
      float t = ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
      for (int s = 1; s < a.G / 8; s <<= 1) t += __shfl_xor(t, s);
      if (k < a.K && k % a.G == 0) {
        t *= f;
#pragma unroll
        for (int c = 0; c < 3; c++) {
          const bf16 b = to_bf16(t);
          a.sx[((int64_t)c * a.M + m) * a.KGp + k / a.G] = b;
          t -= (float)b;
        }
      }
    }
    f16x8 h, l;
#pragma unroll
    for (int j = 0; j < 8; j++) {
      const float y = v[j] * f;
      const int o = 2 * (j & 3) + (j >> 2);
      h[o] = (_Float16)y;
      l[o] = (_Float16)(y - (float)h[o]);
    }
    if (k < a.Kp) {
      const int64_t at = a.frag ? (((m >> 5) * (a.Kp >> 4) + (k >> 4)) * 2 + (k >> 3 & 1)) * 256 + (m & 31) * 8 : m * a.ldp + k;
      *(f16x8*)(a.xh + at) = h;
      if (a.xl) *(f16x8*)(a.xl + at) = l;
    }
  };
  if (a.sx && a.K / a.G + lane < a.KGp)
#pragma unroll
    for (int c = 0; c < 3; c++) a.sx[((int64_t)c * a.M + m) * a.KGp + a.K / a.G + lane] = (bf16)0.0f;
  float mx = 0.0f;
  if constexpr (NV > 0) {
    float v[NV][8];
#pragma unroll
    for (int i = 0; i < NV; i++) piece(8 * lane + 512 * i, v[i]);
#pragma unroll
    for (int i = 0; i < NV; i++) mx = largest(v[i], mx);
    const int e = q4_exp(wave_max(mx), 14);
    if (lane == 0) a.rm[m] = pow2f(-e);
#pragma unroll
    for (int i = 0; i < NV; i++) leave(8 * lane + 512 * i, v[i], pow2f(e));
  } else {
    float v[8];
    for (int k = 8 * lane; k < a.K; k += 512) {
      piece(k, v);
      mx = largest(v, mx);
    }
    const int e = q4_exp(wave_max(mx), 14);
    if (lane == 0) a.rm[m] = pow2f(-e);
    for (int k = 8 * lane; k < (a.Kp + 511) / 512 * 512; k += 512) {
      piece(k, v);
      leave(k, v, pow2f(e));
    }
  }
}

// Eight codes, times the scale pair s, in the order 0 4 1 5 2 6 3 7.  A code's bits in the mantissa of 1024 are 1024 + c, four places
// further up in that of 64 they are 64 + c: less 1032, or 72, it is c - 8 exactly, and both meet the same s.
struct Q4Bits {  // (in registers: an instruction takes one constant of its own, and v_and_or two)
  uint32_t even = 0x000f000fu, odd = 0x00f000f0u, big = 0x64006400u, big_odd = 0x54005400u;
  __device__ __forceinline__ Q4Bits() { asm("" : "+s"(even), "+s"(odd), "+v"(big), "+v"(big_odd)); }
};
__device__ __forceinline__ f16x8 q4_decode(const Q4Bits& b, uint32_t c, f16x2 s) {
  const f16x2 off = {(_Float16)-1032.0f, (_Float16)-1032.0f}, off_odd = {(_Float16)-72.0f, (_Float16)-72.0f};
  f16x8 r;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const uint32_t v = i < 2 ? c : c >> 8;
    const f16x2 k = __builtin_bit_cast(f16x2, i & 1 ? (v & b.odd) | b.big_odd : (v & b.even) | b.big), w = (k + (i & 1 ? off_odd : off)) * s;
    r[2 * i] = w[0];
    r[2 * i + 1] = w[1];
  }
  return r;
}

typedef __attribute__((address_space(3))) void q4_lds_t;
#define Q4_WAIT_VM(n) __builtin_amdgcn_s_waitcnt(((n) & 15) | (7 << 4) | (15 << 8) | (((n) >> 4) << 14))

__device__ __forceinline__ void q4_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

__device__ __forceinline__ __amdgpu_buffer_rsrc_t q4_rsrc(const void* p, int64_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc((void*)p, (short)0, (int)bytes, 0x00020000);
}

// a wave's copy of 64 x 16 bytes into LDS
__device__ __forceinline__ void q4_copy16(__amdgpu_buffer_rsrc_t rs, char* dst, uint32_t off, uint32_t step) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (q4_lds_t*)dst, 16, off, step, 0, 0);
}

struct Q4Tile {
  Q4Args a;
  const _Float16* xh;
  const _Float16* xl;
  const float* rm;
  const float* rn;   // (readable to the next multiple of 256 columns)
  const bf16* sx;    // (as q4_prep_kernel leaves them)
  const bf16* zp;
  float* part;       // [splits][M][ldn] sums of a product split over k, or NULL
  int Kp, KGp, sps;  // k padded, groups padded to 16; steps of 64 k in a split
  int ldp;           // values between the terms' rows
  int ldn;           // N to the next multiple of 4
  int svec;          // four steps' scales are one aligned piece of a row
};

// ------------------------------------------------------------------ products of a few rows
//
// A workgroup takes 32 columns and 32 rows, its eight waves every eighth step of 64 k each, their sums joined in order
// through LDS.  The codes stay whole numbers (exact in f16), and each group's sums meet their scale in fp32; the scales lie
// in LDS as [group][column], and the middles' part is a small product of its own.  x comes from q4_prep_kernel in the order of
// the lanes (as rows, a load meets 32 lines and takes the address unit four times as long).  Bound by trips to memory, of which
// each wave has two steps' under way (four: no faster): 43 x 1024 x 2048 7.7 us, behind 4.8 for x.
constexpr int QF_WAVES = 8;

template <int TERMS, bool G32>
__global__ __launch_bounds__(64 * QF_WAVES, 2) void q4_few_kernel(Q4Tile q) {
  constexpr int NG = G32 ? 2 : 1;  // groups in a step (of 64 k; groups of 128 meet it in two)
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const Q4Args& a = q.a;
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, r = lane & 31, hf = lane >> 5;
  const int n0 = blockIdx.x * 32, m0 = blockIdx.y * 32, KG = a.K / a.G, steps = q.Kp / 64;
  float* const ss = (float*)smem;  // [KG][32]
  // a step's operands: codes 32 hf .. + 31 of column r; x's 16 i + 8 hf .. + 7 of row r
  struct Step {
    u32x4 w;
    f16x8 x[TERMS][4];
  } st[2];
  const uint8_t* wr = a.w + (int64_t)min(n0 + r, a.N - 1) * (a.K / 2);
  const int64_t mr = min(m0 + r, a.M - 1);
  const float rm = q.rm[mr];  // (a power of two)
  const int64_t xo = (int64_t)blockIdx.y * 32 * q.Kp + lane * 8;
  const auto load = [&](Step& v, int step) __attribute__((always_inline)) {  // (past the last step: that one again, unused)
    const int k = 64 * min(step, steps - 1);
    v.w = *(const u32x4*)(wr + min(k + 32 * hf, a.K - 32) / 2);  // (past the row's end its last 32: they meet zeros of x)
#pragma unroll
    for (int i = 0; i < 4; i++) {
      v.x[0][i] = *(const f16x8*)(q.xh + xo + (k + 16 * i) * 32);
      if (TERMS > 1) v.x[TERMS - 1][i] = *(const f16x8*)(q.xl + xo + (k + 16 * i) * 32);
    }
  };
  load(st[0], wave);
  load(st[1], wave + QF_WAVES);
  // what this thread's output reads at the end
  const int om = m0 + (lane & 31), on = n0 + 8 * wave + 4 * (lane >> 5);
  const bool out = wave < 4 && om < a.M && on < a.N;
  Q4Ends<f32x4> ask{};
  if (out) ask = q4_ask4(a, om, on);
  {
    const int64_t col = (int64_t)min(n0 + (tid >> 4), a.N - 1) * KG;
    for (int g0 = tid & 15; g0 < KG; g0 += 64) {
      uint16_t s[4];
#pragma unroll
      for (int i = 0; i < 4; i++) s[i] = a.gs[col + min(g0 + 16 * i, KG - 1)];
#pragma unroll
      for (int i = 0; i < 4; i++)
        if (g0 + 16 * i < KG) ss[(g0 + 16 * i) * 32 + (tid >> 4)] = bf16_f(s[i]);
    }
  }
  __builtin_amdgcn_s_waitcnt(0xc07f);
  q4_barrier();
  f32x16 acc = {};
  const f16x2 one = {(_Float16)1.0f, (_Float16)1.0f};
  const Q4Bits bits;
  const auto product = [&](const Step& v, int step) __attribute__((always_inline)) {
    // the halves' words exchanged, so that matrix step i covers k 16 i .. 16 i + 15: lane half hf word 2 i + hf of 8
    u32x4 w = v.w;
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
      const auto e = __builtin_amdgcn_permlane32_swap(w[i], w[i + 1], false, false);
      w[i] = e[0];      // k 8 i .. 8 i + 15
      w[i + 1] = e[1];  // k 32 + 8 i ..
    }
    f32x16 part[NG];
#pragma unroll
    for (int g = 0; g < NG; g++) part[g] = f32x16{};
#pragma unroll
    for (int i = 0; i < 4; i++) {
      f32x16& p = part[G32 ? i >> 1 : 0];
      const f16x8 wf = q4_decode(bits, w[i < 2 ? 2 * i : 2 * i - 3], one);
#pragma unroll
      for (int e = TERMS - 1; e >= 0; e--) p = __builtin_amdgcn_mfma_f32_32x32x16_f16(wf, v.x[e][i], p, 0, 0, 0);
    }
#pragma unroll
    for (int g = 0; g < NG; g++) {
      const int at = min((64 * step + 32 * g) / a.G, KG - 1) * 32 + 4 * hf;
#pragma unroll
      for (int c = 0; c < 4; c++) {
        const f32x4 s = *(const f32x4*)(ss + at + 8 * c);
#pragma unroll
        for (int e = 0; e < 4; e++) acc[4 * c + e] = __builtin_fmaf(part[g][4 * c + e], s[e], acc[4 * c + e]);
      }
    }
  };
  // the middles' part: sixteen groups a wave
  if (a.gz)
    for (int g = 16 * wave; g < q.KGp; g += 16 * QF_WAVES) {
      bf16x8 xs[3];
      const bf16x8 z = *(const bf16x8*)(q.zp + (int64_t)min(n0 + r, a.N - 1) * q.KGp + g + 8 * hf);
#pragma unroll
      for (int c = 0; c < 3; c++) xs[c] = *(const bf16x8*)(q.sx + ((int64_t)c * a.M + mr) * q.KGp + g + 8 * hf);
#pragma unroll
      for (int c = 2; c >= 0; c--) acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(z, xs[c], acc, 0, 0, 0);
    }
  for (int s = wave; s < steps; s += 2 * QF_WAVES) {
    product(st[0], s);
    load(st[0], s + 2 * QF_WAVES);
    if (s + QF_WAVES < steps) product(st[1], s + QF_WAVES);
    load(st[1], s + 3 * QF_WAVES);
  }
  __syncthreads();  // (the scales' place becomes the sums')
  f32x4* const sum = (f32x4*)smem;  // [wave][quad][lane]
#pragma unroll
  for (int c = 0; c < 4; c++) {
    f32x4 v;
#pragma unroll
    for (int e = 0; e < 4; e++) v[e] = acc[4 * c + e] * rm;
    sum[(wave * 4 + c) * 64 + lane] = v;
  }
  __syncthreads();
  if (!out) return;
  f32x4 v = sum[tid];
#pragma unroll
  for (int w = 1; w < QF_WAVES; w++) v = v + sum[w * 256 + tid];
  q4_leave4(a, om, on, v, ask);
}

// ------------------------------------------------------------------ tiles

// One BM x BN tile a workgroup, waves of WM rows x WN columns.  A step is 64 k: BM rows of x (128 bytes, each term) and BN columns'
// codes (32 bytes) in one of NST LDS stages, filled ahead by buffer_load ... lds.  x's units of 16 bytes lie at slot
// u ^ (row / 2 % 8) (sixteen rows' reads of one unit touch each bank once).  Lane (n, half) takes the 16 bytes of column n's 32 k of
// its half, so that matrix step i of a lane pair covers k 8 i .. 8 i + 7 of both halves; x's units follow.  The scales of four
// steps come in one load where rows of them allow it: each of a lane's own addresses costs the address unit as
// much as 64 neighbouring bytes.  The LDS is held to half of a CU's (three stages for the largest tiles), so that one workgroup's
// first copies and its epilogue pass under another's products: 8192 x 8192 x 2048, one term, gelu, 354 us by 256 x 256 tiles alone on
// their CU and 332 by two of 128 x 256 (828 TFLOP/s; a library product of f16 matrices reaches 1110).  The matrix cores are busy 45 %
// of the cycles at 1.75 GHz, the vector instructions (decode and gelu) take nearly as many.  2048 x 4096 x 1024 in two terms: 48 us,
// one round of tiles, of whose time the k loop takes 30 and the start and the epilogue the rest.
template <int BM, int BN, int WM, int WN, int TERMS, int NST>
__global__ __launch_bounds__(64 * (BM / WM) * (BN / WN), 2) void q4_tile_kernel(Q4Tile t) {
  constexpr int NWM = BM / WM, NW = NWM * (BN / WN), MT = WM / 32, NT = WN / 32;
  constexpr int XB = BM * 128, WO = XB * TERMS, SB = WO + BN * 32, CX = TERMS * BM / 8 / NW, CW = (BN / 32 + NW - 1) / NW, CPW = CX + CW;
  static_assert(CX * NW * 8 == TERMS * BM, "whole copies");
  constexpr int RS = WN + 4, EPL = NW * 32 * RS * 4;
  constexpr int LDS = NST * SB > EPL ? NST * SB : EPL;
  __shared__ __attribute__((aligned(1024))) char smem[LDS];
  const Q4Args& a = t.a;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, r = lane & 31, hf = lane >> 5;
  const int ntn = (a.N + BN - 1) / BN, ntm = (a.M + BM - 1) / BM;
  int tm, tn;
  {
    // XCD x takes a contiguous range of tiles, in groups of 8 row tiles, column-major inside a group
    const int total = ntn * ntm, q = total >> 3, rem = total & 7, x = blockIdx.x & 7;
    const int i = x * q + min(x, rem) + (int)(blockIdx.x >> 3);
    const int grp = i / (8 * ntn), row0 = 8 * grp, gm = min(8, ntm - row0), local = i - grp * 8 * ntn;
    tn = __builtin_amdgcn_readfirstlane(local / gm);
    tm = __builtin_amdgcn_readfirstlane(row0 + (local - tn * gm));
  }
  const int bm = tm * BM, bn = tn * BN, K = a.K, KG = __builtin_amdgcn_readfirstlane(K / a.G);
  const int wm = (wave % NWM) * WM, wn = (wave / NWM) * WN;
  const int s0 = blockIdx.y * t.sps, steps = min(t.sps, t.Kp / 64 - s0);

  const int mrows = min(BM, a.M - bm), ncols = min(BN, a.N - bn);
  const __amdgpu_buffer_rsrc_t rh = q4_rsrc(t.xh + (int64_t)bm * t.ldp, (int64_t)mrows * t.ldp * 2),
                               rl = q4_rsrc((TERMS > 1 ? t.xl : t.xh) + (int64_t)bm * t.ldp, (int64_t)mrows * t.ldp * 2),
                               rw = q4_rsrc(a.w + (int64_t)bn * (K / 2), (int64_t)ncols * (K / 2));
  // copies of this wave: eight rows of a term, or 32 columns' codes (past the tile's last: that one again)
  uint32_t xo[CX], wo[CW];
#pragma unroll
  for (int c = 0; c < CX; c++) {
    const int row = (8 * (wave * CX + c)) % BM + (lane >> 3);
    xo[c] = (uint32_t)row * (uint32_t)(t.ldp * 2) + 16 * ((lane & 7) ^ ((row >> 1) & 7)) + 128 * s0;
  }
#pragma unroll
  for (int c = 0; c < CW; c++) wo[c] = (uint32_t)(32 * min(wave * CW + c, BN / 32 - 1) + (lane >> 1)) * (uint32_t)(K / 2) + 16 * (lane & 1);
  const auto copies = [&](int step, int po) __attribute__((always_inline)) {  // into the stage at po
#pragma unroll
    for (int c = 0; c < CX; c++)
      q4_copy16(TERMS > 1 && wave * CX + c >= BM / 8 ? rl : rh, smem + po + (wave * CX + c) * 1024, xo[c], 128 * step);
    // (K of an odd number of 32: the last half is the next column's or past the end, and meets zeros of x)
#pragma unroll
    for (int c = 0; c < CW; c++) q4_copy16(rw, smem + po + WO + min(wave * CW + c, BN / 32 - 1) * 1024, wo[c], 32 * (s0 + step));
  };
  copies(0, 0);
  // The scales of steps s .. s + 3 (s % 4 == 0): as they lie, if four steps' are one aligned piece of the row, else one by one; then
  // each step's as a pair for the decode.
  const uint16_t* srow[NT];
  float fn[NT];
#pragma unroll
  for (int j = 0; j < NT; j++) {
    const int64_t n = min(bn + wn + 32 * j + r, a.N - 1);
    srow[j] = a.gs + n * KG;
    fn[j] = 1.0f / t.rn[n];
  }
  const int lg = 31 - __builtin_clz(a.G);
  u32x4 sc[NT];
  f16x2 sv[4][NT];
  const auto scales = [&](int step) __attribute__((always_inline)) {
    const int g = (s0 + step) * 64 >> lg;
#pragma unroll
    for (int j = 0; j < NT; j++) {
      if (t.svec) {
        const int at = min(g, KG - (256 >> lg));
        if (a.G == 32) {
          sc[j] = *(const u32x4*)(srow[j] + at);
        } else if (a.G == 64) {
          const uint2 v = *(const uint2*)(srow[j] + at);
          sc[j][0] = v.x;
          sc[j][1] = v.y;
        } else {
          sc[j][0] = *(const uint32_t*)(srow[j] + at);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 4; i++) sc[j][i] = srow[j][min(64 * (s0 + step + i) + 32 * hf, K - 32) >> lg];
      }
    }
  };
  const auto pairs = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < NT; j++) {
      u32x4 v = sc[j];
      if (t.svec) {
        if (a.G == 32) {
#pragma unroll
          for (int i = 0; i < 4; i++) v[i] = v[i] >> (16 * hf);
        } else if (a.G == 64) {
          v = u32x4{v[0], v[0] >> 16, v[1], v[1] >> 16};
        } else {
          v = u32x4{v[0], v[0], v[0] >> 16, v[0] >> 16};
        }
      }
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const _Float16 f = (_Float16)(__uint_as_float(v[i] << 16) * fn[j]);
        sv[i][j] = f16x2{f, f};
      }
    }
  };
  f32x16 acc[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; i++)
#pragma unroll
    for (int j = 0; j < NT; j++) acc[i][j] = f32x16{};
  scales(0);
  // The middles' part: z in bf16, the groups' sums of x as three bf16 terms, sixteen groups a matrix step, dealt to the parts of k.  The
  // first are asked for before the copies that the loop waits for.  (515 x 1316 x 1440 in groups of 32: 20.2 us without middles, 22.5
  // with them, 25.0 where every tile cut its rows' sums into terms and took all of them in the first part.)
  const int mids = a.gz ? t.KGp / 16 : 0;
  int mid = blockIdx.y;
  bf16x8 zf[NT], xs[MT][3];
  const auto ask_mids = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < NT; j++) zf[j] = *(const bf16x8*)(t.zp + (int64_t)min(bn + wn + 32 * j + r, a.N - 1) * t.KGp + 16 * mid + 8 * hf);
#pragma unroll
    for (int i = 0; i < MT; i++)
#pragma unroll
      for (int c = 0; c < 3; c++)
        xs[i][c] = *(const bf16x8*)(t.sx + ((int64_t)c * a.M + min(bm + wm + 32 * i + r, a.M - 1)) * t.KGp + 16 * mid + 8 * hf);
  };
  if (mid < mids) ask_mids();
#pragma unroll
  for (int p = 1; p < NST; p++) copies(p, p * SB);
  while (mid < mids) {
#pragma unroll
    for (int c = 2; c >= 0; c--)
#pragma unroll
      for (int i = 0; i < MT; i++)
#pragma unroll
        for (int j = 0; j < NT; j++) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(zf[j], xs[i][c], acc[i][j], 0, 0, 0);
    mid += gridDim.y;
    if (mid < mids) ask_mids();
  }
  int xa[4];  // unit 4 hf + i of row r
#pragma unroll
  for (int i = 0; i < 4; i++) xa[i] = (wm + r) * 128 + 16 * ((4 * hf + i) ^ ((r >> 1) & 7));
  const int wa = WO + (wn + r) * 32 + 16 * hf;

  // Fragments of matrix step i + 1 are read and decoded under step i's products.  Before the last of a stage's four, whose
  // fragments are in registers by then, a barrier ends every wave's reads of the stage (its buffer is refilled) and publishes
  // the next one: this wave's copies of it have arrived when at most those of the stages after it pend.
  f16x8 xf[2][MT][TERMS], wf[2][NT];
  u32x4 wr[NT];
  const Q4Bits bits;
  const auto xread = [&](int u, int po, int i) __attribute__((always_inline)) {
#pragma unroll
    for (int m = 0; m < MT; m++)
#pragma unroll
      for (int e = 0; e < TERMS; e++) xf[u][m][e] = *(const f16x8*)(smem + po + xa[i] + e * XB + m * 4096);
  };
  const auto wread = [&](int po) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < NT; j++) wr[j] = *(const u32x4*)(smem + po + wa + j * 1024);
  };
  const auto decode = [&](int u, int q, int i) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < NT; j++) wf[u][j] = q4_decode(bits, wr[j][i], sv[q][j]);
  };
  pairs();
  Q4_WAIT_VM((NST - 1) * CPW);
  q4_barrier();
  scales(4);
  wread(0);
  xread(0, 0, 0);
  decode(0, 0, 0);
  int po = 0;  // the stage's place
  const auto stage = [&](int step, auto quarter) __attribute__((always_inline)) {
    constexpr int q = decltype(quarter)::value, qn = (q + 1) % 4;  // of its four
    const int pn = po + SB == NST * SB ? 0 : po + SB;
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const int u = i & 1;
      if (i == 3) {
        __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0)
        Q4_WAIT_VM((NST - 2) * CPW);
        q4_barrier();
        copies(step + NST, po);
        wread(pn);
        xread(u ^ 1, pn, 0);
        if (q == 3) {
          pairs();
          scales(step + 5);
        }
        decode(u ^ 1, qn, 0);
      } else {
        xread(u ^ 1, po, i + 1);
        decode(u ^ 1, q, i + 1);
      }
#pragma unroll
      for (int e = TERMS - 1; e >= 0; e--)
#pragma unroll
        for (int m = 0; m < MT; m++)
#pragma unroll
          for (int j = 0; j < NT; j++) acc[m][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(wf[u][j], xf[u][m][e], acc[m][j], 0, 0, 0);
      __builtin_amdgcn_sched_barrier(0);
    }
    po = pn;
  };
  int s = 0;
  for (; s + 4 <= steps; s += 4) {
    stage(s, std::integral_constant<int, 0>{});
    stage(s + 1, std::integral_constant<int, 1>{});
    stage(s + 2, std::integral_constant<int, 2>{});
    stage(s + 3, std::integral_constant<int, 3>{});
  }
  if (s < steps) stage(s, std::integral_constant<int, 0>{});
  if (s + 1 < steps) stage(s + 1, std::integral_constant<int, 1>{});
  if (s + 2 < steps) stage(s + 2, std::integral_constant<int, 2>{});
  Q4_WAIT_VM(0);  // no copy into LDS outlives the loop
  q4_barrier();

  // Rows leave through LDS, 32 rows of a wave at a time, so that neighbouring lanes hold 16 bytes of one row each.
  float* rows = (float*)smem + wave * 32 * RS;
  constexpr int LR = WN / 4, PR = 64 / LR;
  const int n0 = bn + wn;
#pragma unroll
  for (int i = 0; i < MT; i++) {
    const int m = bm + wm + 32 * i + r, mc = min(m, a.M - 1);
    const float fm = t.rm[mc];
#pragma unroll
    for (int j = 0; j < NT; j++) {
#pragma unroll
      for (int q = 0; q < 4; q++) {
        const f32x4 f = *(const f32x4*)(t.rn + n0 + 32 * j + 8 * q + 4 * hf);
        f32x4 v;
#pragma unroll
        for (int e = 0; e < 4; e++) v[e] = acc[i][j][4 * q + e] * f[e] * fm;
        *(f32x4*)(rows + r * RS + 32 * j + 8 * q + 4 * hf) = v;
      }
    }
    __builtin_amdgcn_wave_barrier();
    const int n = n0 + 4 * (lane % LR);
    // (a loop with one body: unrolled, the epilogue is more code than the instruction cache holds beside the k loop)
#pragma unroll 1
    for (int q = 0; q < 32; q += 4 * PR) {
      const int64_t mo = bm + wm + 32 * i + q + lane / LR;
      f32x4 v[4];
      Q4Ends<f32x4> ask[4];
#pragma unroll
      for (int u = 0; u < 4; u++) {
        v[u] = *(const f32x4*)(rows + (q + u * PR + lane / LR) * RS + 4 * (lane % LR));
        if (!t.part && mo + u * PR < a.M && n < a.N) ask[u] = q4_ask4(a, mo + u * PR, n);
      }
#pragma unroll
      for (int u = 0; u < 4; u++) {
        const int64_t m = mo + u * PR;
        if (m >= a.M || n >= a.N) continue;
        if (t.part) *(f32x4*)(t.part + ((int64_t)blockIdx.y * a.M + m) * t.ldn + n) = v[u];
        else q4_leave4(a, m, n, v[u], ask[u]);
      }
    }
    __builtin_amdgcn_wave_barrier();
  }
}

// A split product's sums, added in order, and the epilogue.  Bound by a launch and a trip to memory (3 to 5 us).
constexpr int Q4_SPLITS = 16;
__global__ __launch_bounds__(256) void q4_join_kernel(Q4Tile t, int splits) {
  const Q4Args& a = t.a;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, m = i / (t.ldn / 4), plane = (int64_t)a.M * t.ldn;
  if (m >= a.M) return;
  const int n = (int)(4 * i - m * t.ldn);
  const Q4Ends<f32x4> ask = q4_ask4(a, m, n);
  f32x4 w[Q4_SPLITS], v = {};  // (all asked for before the first is added)
#pragma unroll
  for (int s = 0; s < Q4_SPLITS; s++) w[s] = s < splits ? *(const f32x4*)(t.part + s * plane + 4 * i) : f32x4{};
#pragma unroll
  for (int s = 0; s < Q4_SPLITS; s++) v = v + w[s];
  q4_leave4(a, m, n, v, ask);
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

constexpr int Q4_FEW_LDS = 65536;  // that a launch may ask for

static int q4_columns(const Q4Args& a) { return a.N >= 4096 ? 4 : a.N >= 2048 ? 2 : 1; }  // of a wave of the vector kernel

static void q4_gemv(anima_ctx* c, const Q4Args& a) {
#define GEMV(MR, U) hipLaunchKernelGGL((q4_gemv_kernel<MR, U>), dim3((unsigned)((a.N + 4 * U - 1) / (4 * U)), (unsigned)((a.M + MR - 1) / MR)), dim3(256), 0, c->stream, a)
#define GEMV_U(MR)                    \
  do {                                \
    if (q4_columns(a) == 4) GEMV(MR, 4);     \
    else if (q4_columns(a) == 2) GEMV(MR, 2); \
    else GEMV(MR, 1);                 \
  } while (0)
  if (a.M == 1) GEMV_U(1);
  else if (a.M == 2) GEMV_U(2);
  else GEMV_U(4);
#undef GEMV_U
#undef GEMV
}

// LDS of the kernel for few rows: the scales, then the waves' sums
static int64_t q4_few_lds(const Q4Args& a) {
  return std::max<int64_t>((int64_t)(a.K / a.G) * 128, QF_WAVES * 4096);
}

template <int BM, int BN, int WM, int WN, int TERMS, int NST>
static void q4_tile_launch(anima_ctx* c, const Q4Tile& t, int splits) {
  const dim3 grid((unsigned)(((t.a.N + BN - 1) / BN) * ((t.a.M + BM - 1) / BM)), (unsigned)splits), block(64 * (BM / WM) * (BN / WN));
  hipLaunchKernelGGL((q4_tile_kernel<BM, BN, WM, WN, TERMS, NST>), grid, block, 0, c->stream, t);
}

// Up to 64 rows by 32 x 32 tiles, but two terms of more than 32 rows with many steps, where x is read once more for every 32 rows
// (33 x 8192 x 4096: 29 us, 23 by the larger tiles; 64 x 4096 x 4096: 19 and 23).
static bool q4_few(const Q4Args& a, bool two) {
  const bool many = two && a.M > 32 && (a.K >= 8192 || (int64_t)a.N * a.K >= (int64_t)1 << 25);
  return a.M <= 64 && !many && q4_few_lds(a) <= Q4_FEW_LDS;
}

// Whether the vector kernel, four rows a group, ends before the matrix kernels, by times in us that were fitted to 70 sizes: it takes a
// launch, then a trip to memory for each 1024 of k, or its workgroups' shares (a start, and for each 1024 of k the rows of x and the
// columns' codes); they take a launch more, and k's steps one behind the other.  8 x 2048 x 1024: 5.8 us, 9.5 by 32 x 32 tiles
// (8 x 8192 x 2048: 13.2 and 11.2); 100 x 100 x 512: 5.5, 10.4 by tiles of 64 x 64 (1093 x 65 x 64: 20.8 and 8.6).
static bool q4_rows(const Q4Args& a, bool two) {
  if (a.M <= 4) return true;
  const int64_t groups = (a.M + 3) / 4, u = q4_columns(a), wgs = (a.N + 4 * u - 1) / (4 * u) * groups;
  if (groups > 65535) return false;
  const double k = a.K / 1024.0, turns = (a.K + 1023) / 1024, work = 1e-3 * (double)wgs * (1.6 + turns * (1.27 + 0.63 * (double)u));
  return 4.0 + std::max(1.24 * turns, work) < (!q4_few(a, two) ? 8.5 : two ? 7.0 + 2.0 * k : 6.6 + 1.4 * k);
}

// x into f16 terms (and the columns' powers), then the products, then, where k was split, the sums.
static int q4_matrix(anima_ctx* c, const Q4Args& a, bool two) {
  Q4Tile t{};
  t.a = a;
  t.Kp = (a.K + 63) / 64 * 64;
  // rows of the terms an odd number of lines of 128 bytes apart: at a power of two one step's rows meet in one memory channel
  t.ldp = t.Kp / 64 % 2 ? t.Kp : t.Kp + 64;
  t.ldn = (a.N + 3) / 4 * 4;
  const int steps = t.Kp / 64;
  t.KGp = (a.K / a.G + 15) / 16 * 16;
  const bool few = q4_few(a, two);
  const auto tiles = [&](int bm, int bn) { return (int64_t)((a.M + bm - 1) / bm) * ((a.N + bn - 1) / bn); };
  // The largest tile of which there are enough and that the columns fill by more than half; the smallest ends soonest (K = 256 in one term, 2770 x 6019: 39 us, 59 by the largest),
  // the largest read x least (8192 x 8192 x 2048: two terms 587, 636, 888 us from the largest down, one term 337, 392, 513).
  // Where there are too few, parts of k: of 16 steps and more on the CUs' second places (two terms, 644 x 1695 x 6912:
  // 82 us whole, 62 in parts), of three and more while CUs are idle (202 x 122 x 1792: 24 and 14; a join takes 3 us and more).
  const int rows = two ? 64 : 128;  // of the larger tiles
  const int64_t cus = c->num_cus, t0 = tiles(rows, 256), t1 = tiles(rows, 128), t2 = tiles(64, 64);
  int tile = 2, splits = 1;
  if (few) {
  } else if (a.N > 128 && t0 >= 2 * cus && (two ? steps >= 16 || t0 >= 4 * cus : steps >= 8)) {
    tile = 0;
  } else if (a.N > 64 && (two ? t1 >= cus : t1 >= 2 * cus && steps >= 8)) {
    tile = 1;
  } else {
    if (two) {
      while (t1 * splits < cus && splits < Q4_SPLITS) splits *= 2;
      if (t1 * splits >= cus && steps / splits >= 16) tile = 1;
      else splits = 1;
    } else {
      while (t2 * splits < 2 * cus && splits < Q4_SPLITS && steps / (2 * splits) >= 16) splits *= 2;
    }
    if (tile == 2 && steps >= 16)
      while (splits < Q4_SPLITS && t2 * splits * 2 <= cus && steps / (2 * splits) >= 3) splits *= 2;
  }
  t.sps = (steps + splits - 1) / splits;
  if (splits > 1) t.sps = (t.sps + 3) / 4 * 4;
  t.svec = a.K % 256 == 0 && q4_al(a.gs, 16);
  splits = (steps + t.sps - 1) / t.sps;
  // scratch: the terms, the powers, the group sums, the splits' sums
  size_t at = 0;
  const auto take = [&](size_t bytes) {
    const size_t o = at;
    at += (bytes + 255) / 256 * 256;
    return o;
  };
  const size_t plane = (few ? (size_t)(a.M + 31) / 32 * 32 * t.Kp : (size_t)a.M * t.ldp) * 2, oh = take(plane), ol = two ? take(plane) : 0, om = take((size_t)a.M * 4),
               on = few ? 0 : take(((size_t)a.N + 255) / 256 * 1024), os = a.gz ? take((size_t)a.M * t.KGp * 6) : 0, oz = a.gz ? take((size_t)a.N * t.KGp * 2) : 0,
               op = splits > 1 ? take((size_t)splits * a.M * t.ldn * 4) : 0;
  void* tmp = nullptr;
  if (int rc = anima_alloc(c, at, &tmp)) return rc;
  char* const b = (char*)tmp;
  Q4Prep p{a.x, a.ldx, (_Float16*)(b + oh), two ? (_Float16*)(b + ol) : nullptr, (float*)(b + om), a.gz ? (bf16*)(b + os) : nullptr,
           a.gz ? (bf16*)(b + oz) : nullptr, a.gs, a.gz, few ? nullptr : (float*)(b + on), t.ldp, a.M, a.N, a.K, t.Kp, a.G, t.KGp, (a.M + 3) / 4, few};
  t.xh = p.xh;
  t.xl = p.xl;
  t.rm = p.rm;
  t.rn = p.rn;
  t.sx = p.sx;
  t.zp = p.zp;
  t.part = splits > 1 ? (float*)(b + op) : nullptr;
  Launch L(c, few ? "gemm.q4.few" : tile == 0 ? "gemm.q4.256" : tile == 1 ? "gemm.q4.128" : "gemm.q4.64", 2.0 * a.M * a.N * a.K, 0.0);
  {
    const dim3 grid((unsigned)(p.rows + (few && !a.gz ? 0 : (a.N + 3) / 4))), block(256);
    if (a.K <= 1024) hipLaunchKernelGGL(q4_prep_kernel<2>, grid, block, 0, c->stream, p);
    else if (a.K <= 2048) hipLaunchKernelGGL(q4_prep_kernel<4>, grid, block, 0, c->stream, p);
    else if (a.K <= 8192) hipLaunchKernelGGL(q4_prep_kernel<16>, grid, block, 0, c->stream, p);
    else hipLaunchKernelGGL(q4_prep_kernel<0>, grid, block, 0, c->stream, p);
  }
  if (hipPeekAtLastError() != hipSuccess) {  // (no product of terms that were not written)
    const int rc = L.end();
    anima_free(c, tmp);
    return rc;
  }
  if (few) {
    const dim3 grid((unsigned)((a.N + 31) / 32), (unsigned)((a.M + 31) / 32)), block(64 * QF_WAVES);
    const int lds = (int)q4_few_lds(a);
    if (two && a.G == 32) hipLaunchKernelGGL((q4_few_kernel<2, true>), grid, block, lds, c->stream, t);
    else if (two) hipLaunchKernelGGL((q4_few_kernel<2, false>), grid, block, lds, c->stream, t);
    else if (a.G == 32) hipLaunchKernelGGL((q4_few_kernel<1, true>), grid, block, lds, c->stream, t);
    else hipLaunchKernelGGL((q4_few_kernel<1, false>), grid, block, lds, c->stream, t);
  } else if (two) {
    if (tile == 0) q4_tile_launch<64, 256, 64, 64, 2, 3>(c, t, splits);
    else if (tile == 1) q4_tile_launch<64, 128, 64, 32, 2, 4>(c, t, splits);
    else q4_tile_launch<64, 64, 32, 32, 2, 4>(c, t, splits);
  } else {
    if (tile == 0) q4_tile_launch<128, 256, 128, 64, 1, 3>(c, t, splits);
    else if (tile == 1) q4_tile_launch<128, 128, 64, 64, 1, 4>(c, t, splits);
    else q4_tile_launch<64, 64, 32, 32, 1, 4>(c, t, splits);
  }
  if (splits > 1)
    hipLaunchKernelGGL(q4_join_kernel, dim3((unsigned)(((int64_t)a.M * (t.ldn / 4) + 255) / 256)), dim3(256), 0, c->stream, t, splits);
  const int rc = L.end();
  anima_free(c, tmp);
  return rc;
}

static int q4_linear_part(anima_ctx* c, const Q4Args& a, bool two) {
  if (!q4_rows(a, two)) return q4_matrix(c, a, two);
  Launch L(c, "gemv.q4", 2.0 * a.M * a.N * a.K, 0.5 * a.N * a.K);
  q4_gemv(c, a);
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
  const bool two = d->precision == ANIMA_PREC_FP32;
  const Q4Part part = q4_part(d->M, W->N);
  for (int64_t n = 0; n < W->N; n += part.cols)
    for (int64_t m = 0; m < d->M; m += part.rows) {
      Q4Args p = a;
      p.M = (int)std::min(part.rows, d->M - m);
      p.N = (int)std::min(part.cols, W->N - n);
      p.x += m * a.ldx;
      p.w += n * (a.K / 2);
      p.gs += n * (a.K / a.G);
      if (a.gz) p.gz += n * (a.K / a.G);
      if (a.bias) p.bias += n;
      if (a.gate) p.gate += n;
      if (a.add) p.add += m * a.ld_add + n;
      p.out = (char*)a.out + (m * a.ldc + n) * (a.obf ? 2 : 4);
      if (int rc = q4_linear_part(c, p, two)) return rc;
    }
  return ANIMA_OK;
}

}  // namespace anima
