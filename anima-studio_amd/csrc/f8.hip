// The e4m3 operators for gfx950: rows and weights to 8-bit floating point with a scale per block of 128,
// the products of such rows and weights, the gated half of a feed-forward block, and the residual / norm
// seam that leaves e4m3 rows.  No reference counterpart (see anima.h).
//
// Quantization of a block with largest magnitude a: a' = max(a, 2^-100), scale = a' / 448,
// value = e4m3(x * (448 * (1 / a'))).  The maximum is taken on the bit patterns of |x| (as unsigned integers they
// order like the values, an infinity above every finite value and NaN above that), so a NaN reaches the
// scale.  |x| * (448 * (1 / a')) is at most 448 (1 + 2^-21) (1 / a' has 22 bits at the least, as a subnormal of
// the largest a'), which rounds to 448: no clamp.
//
// Products: D = sum over the 128 k of a block on the matrix cores, then acc = fma(xs * scale, D, acc) in fp32.
// ANIMA_PREC_BF16 takes v_mfma_f32_32x32x64_f8f6f4, two of them a block of k: within each eight k it aligns the
// products to the largest and drops what lies 2^-13 below (measured: 2^16 + 2^3 is exact, 2^16 + 2^2 gives 2^16;
// relative L2 error of a block of normal values 1.5e-5, mean 1e-7), between the eights it adds in 32 bits.
// ANIMA_PREC_FP32 widens e4m3 to bf16 (exact: 4 significant bits) and takes v_mfma_f32_32x32x16_bf16, whose
// products of such values are exact and sums 32 bits (error of a block 9e-9), at half the rate.  The weight is
// the first operand, so D's rows are outputs n and its columns rows m of x: a lane holds four consecutive n of
// one m, and its xs is one value.
#include <cmath>
#include <type_traits>

#include "common.h"
#include "f8_args.h"
#include "internal.h"

namespace anima {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr float F8_TOP = 448.0f;                     // largest e4m3 value
constexpr uint32_t F8_TINY = (127u - 100u) << 23;    // bits of 2^-100

struct F8Args {
  const uint8_t* xq;  // e4m3 rows, ldx bytes apart, and xs [KB][M]; or fp32 rows x, ldx floats apart
  const float* xs;
  const float* x;
  int64_t ldx;
  const uint8_t* w;   // [N][K], ws [ceil(N/128)][KB]; GLU: the gate's
  const float* ws;
  const float* bias;
  const uint8_t* w2;  // GLU: the up projection
  const float* ws2;
  const float* bias2;
  float* out;
  int64_t ldc;
  float alpha;
  int act, epi;
  const float* gate;  // [N]
  const float* add;
  int64_t ld_add;
  int M, N, K, KB;
  int kbs;            // f8_tile: blocks of k of a split (blockIdx.y), whose sums leave as fp32 rows [M][N] of their own
  int vec;            // four columns of out, add, bias and gate at a time
  int obf;            // out is bf16 rows
  uint8_t* oq;        // GLU: e4m3 rows [M][N] instead, and their scales
  float* os;
};

__device__ __forceinline__ uint32_t abs_bits(float v) { return __builtin_bit_cast(uint32_t, v) & 0x7fffffffu; }
__device__ __forceinline__ uint32_t umax(uint32_t a, uint32_t b) { return a > b ? a : b; }

// A block's scale and the factor its values are multiplied with, from the bits of its largest magnitude.
__device__ __forceinline__ void f8_scale(uint32_t amax, float& scale, float& mul) {
  const float a = __builtin_bit_cast(float, umax(amax, F8_TINY));
  // a / 448 rounded once: the product with 1 / 448 corrected by its exact remainder (equal to the quotient for all 2^23
  // fractions of a; a is no subnormal), an infinity or NaN as the quotient's
  constexpr float y = 1.0f / F8_TOP;
  const float q = a * y;
  scale = __builtin_amdgcn_div_fixupf(__builtin_fmaf(__builtin_fmaf(-F8_TOP, q, a), y, q), F8_TOP, a);
  mul = F8_TOP * (1.0f / a);
}

// four values to e4m3 bytes, the first in the lowest
__device__ __forceinline__ uint32_t f8_pack(f32x4 v, float mul) {
  int r = __builtin_amdgcn_cvt_pk_fp8_f32(v[0] * mul, v[1] * mul, 0, false);
  r = __builtin_amdgcn_cvt_pk_fp8_f32(v[2] * mul, v[3] * mul, r, true);
  return (uint32_t)r;
}

__device__ __forceinline__ uint32_t amax4(f32x4 v, uint32_t m) {
  return umax(umax(abs_bits(v[0]), abs_bits(v[1])), umax(umax(abs_bits(v[2]), abs_bits(v[3])), m));
}

__device__ __forceinline__ __amdgpu_buffer_rsrc_t f8_rsrc(const void* p, int64_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc((void*)p, (short)0, (int)bytes, 0x00020000);
}

// v of the lane that DPP control C names
template <int C>
__device__ __forceinline__ uint32_t dpp(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, C, 0xf, 0xf, false);
}
// DPP controls that exchange lanes 1, 2, then (the quads being equal) 4 and 8 apart
constexpr int X1 = 0xb1, X2 = 0x4e, X4 = 0x141, X8 = 0x140;

// maximum over the 32 lanes of a half wave, in every lane: 16 lanes with DPP, then both rows of 16
__device__ __forceinline__ uint32_t half_umax(uint32_t v) {
  v = umax(v, dpp<X1>(v));
  v = umax(v, dpp<X2>(v));
  v = umax(v, dpp<X4>(v));
  v = umax(v, dpp<X8>(v));
  const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  return umax(r[0], r[1]);
}

// maximum over the lanes with the same lane % 16, in every lane
__device__ __forceinline__ uint32_t cross_umax(uint32_t v) {
  const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  v = umax(r[0], r[1]);
  const auto q = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return umax(q[0], q[1]);
}

// SiLU as r * rcp(1 + 2^(-r log2 e)) on v_exp_f32 and v_rcp_f32 (1 ulp each): the exponent is off by 1.22 roundings of
// itself, the power, the sum, the reciprocal and the product by 2, 1, 2 and 1, so within 2^-22 (3/2 + |r| / 3) of itself for
// r from -87 to 0 and 1.3 2^-22 for others; below -87, where the power or its reciprocal leaves the range, it may be -0
// (within 1.5e-36).  5 instructions, where silu_f's expf and quotient take 40 (of a 256 x 256 tile's epilogue 25000 cycles,
// and 9000).
__device__ __forceinline__ float f8_silu(float r) {
  return r * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(r * -1.4426950408889634f));
}

__device__ __forceinline__ float f8_act(float r, int act) {
  if (act == ANIMA_ACT_GELU) return gelu_erf(r);
  if (act == ANIMA_ACT_SILU) return f8_silu(r);
  return r;
}

// ------------------------------------------------------------------ rows and weights to e4m3

__device__ __forceinline__ f32x4 ld4(const float* p) { return *(const f32x4*)p; }
__device__ __forceinline__ f32x4 ld4(const uint16_t* p) {
  const uint2 u = *(const uint2*)p;
  return f32x4{__builtin_bit_cast(float, u.x << 16), __builtin_bit_cast(float, u.x & 0xffff0000u),
               __builtin_bit_cast(float, u.y << 16), __builtin_bit_cast(float, u.y & 0xffff0000u)};
}

// n / d for n < 2^31 by a multiplication: d = 1, or (n * mul >> 32) >> shift with mul = floor(2^(32 + shift) / d) + 1 and
// 2^shift < d <= 2^(shift + 1), which is exact there (the excess, below n / 2^(32 + shift) < 1 / d, changes no quotient).
struct DivBy {
  uint32_t d, mul, shift;
};
static DivBy div_by(uint32_t d) {
  uint32_t l = 0;
  while ((2u << l) < d) l++;
  return d < 2 ? DivBy{1, 0, 0} : DivBy{d, (uint32_t)(((uint64_t)1 << (32 + l)) / d + 1), l};
}
__device__ __forceinline__ uint32_t div_u31(uint32_t n, const DivBy& d) { return d.d == 1 ? n : __umulhi(n, d.mul) >> d.shift; }

// eight values of a row
struct Eight {
  f32x4 lo, hi;
};
__device__ __forceinline__ Eight ld8(const float* p) { return {ld4(p), ld4(p + 4)}; }
__device__ __forceinline__ Eight ld8(const uint16_t* p) {
  const uint4 u = *(const uint4*)p;
  const auto two = [](uint32_t a, uint32_t b) {
    return f32x4{__builtin_bit_cast(float, a << 16), __builtin_bit_cast(float, a & 0xffff0000u), __builtin_bit_cast(float, b << 16),
                 __builtin_bit_cast(float, b & 0xffff0000u)};
  };
  return {two(u.x, u.y), two(u.z, u.w)};
}

// 16 lanes per block of 128 columns (a lane: eight of them, whose maximum takes four DPP steps), blocks in row
// order, U of them 16 workgroup threads' blocks apart so that their loads are in flight together.  Bound by the bytes:
// 8192 x 2048 bf16 rows (51 MB) 11.1 us, 4.6 TB/s (lanes of four values, one block each, 15.2); 43 rows 2.2 us in a
// graph, a launch and one trip to memory.
template <class T, int U>
__global__ __launch_bounds__(256) void quant_rows_f8_kernel(const T* X, int64_t ldx, uint32_t blocks, int K, int64_t M, DivBy KB, uint8_t* Q,
                                                            float* S) {
  const int l = threadIdx.x & 15;
  const uint32_t b0 = (uint32_t)xcd_remap(blockIdx.x, gridDim.x) * (16 * U) + (threadIdx.x >> 4);
  Eight v[U];
  uint32_t m[U], kb[U];
  bool in[U];
#pragma unroll
  for (int u = 0; u < U; u++) {
    const uint32_t b = b0 + 16 * u;
    m[u] = div_u31(b, KB);
    kb[u] = b - m[u] * KB.d;
    const int k = (int)kb[u] * 128 + 8 * l;
    in[u] = b < blocks && k < K;
    v[u] = in[u] ? ld8(X + (int64_t)m[u] * ldx + k) : Eight{};
  }
#pragma unroll
  for (int u = 0; u < U; u++) {
    uint32_t a = amax4(v[u].hi, amax4(v[u].lo, 0));
    a = umax(a, dpp<X1>(a));
    a = umax(a, dpp<X2>(a));
    a = umax(a, dpp<X4>(a));
    a = umax(a, dpp<X8>(a));
    float scale, mul;
    f8_scale(a, scale, mul);
    if (in[u]) {
      *(uint2*)(Q + (int64_t)m[u] * K + kb[u] * 128 + 8 * l) = make_uint2(f8_pack(v[u].lo, mul), f8_pack(v[u].hi, mul));
      if (l == 0) S[(int64_t)kb[u] * M + m[u]] = scale;
    }
  }
}

// A workgroup per 128 x 128 block (a checkpoint's conversion, once per weight): thread t holds columns 4 (t % 32) .. + 3 of
// rows t / 32 + 8 i.  Bound by the bytes: 8192 x 2048 from bf16 (50 MB) 10.4 us, 4.8 TB/s, from fp32 (84 MB) 14.6, 5.7.
template <class T>
__global__ __launch_bounds__(256) void weight_quant_f8_kernel(const T* W, int N, int K, int KB, uint8_t* Q, float* S) {
  __shared__ uint32_t red[8];
  const int kb = blockIdx.x % KB, nb = blockIdx.x / KB;
  const int k = kb * 128 + 4 * (threadIdx.x & 31), n0 = nb * 128 + (threadIdx.x >> 5);
  f32x4 v[16];
  uint32_t a = 0;
#pragma unroll
  for (int i = 0; i < 16; i++) {
    const int n = n0 + 8 * i;
    v[i] = n < N && k < K ? ld4(W + (int64_t)n * K + k) : f32x4{};
    a = amax4(v[i], a);
  }
  a = half_umax(a);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = a;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; i++) a = umax(a, red[i]);
  float scale, mul;
  f8_scale(a, scale, mul);
#pragma unroll
  for (int i = 0; i < 16; i++) {
    const int n = n0 + 8 * i;
    if (n < N && k < K) *(uint32_t*)(Q + (int64_t)n * K + k) = f8_pack(v[i], mul);
  }
  if (threadIdx.x == 0) S[(int64_t)nb * KB + kb] = scale;
}

// ------------------------------------------------------------------ residual + norm

struct NormArgs {
  float* x;
  const void* y;
  const float *post_w, *gate, *norm_w, *shift, *scale;
  float* h;
  uint8_t* q;
  float* s;
  int64_t ldx, ldy, ldh, gate_ld, mod_ld, group_rows;
  float res_scale, eps;
  int rows, cols, layer, y_bf16;
  uint32_t row0;  // of the launch
};

// Sum over a wave, in every lane: 16 lanes with DPP, then both halves of 32 and of 64.
__device__ __forceinline__ float wave_fsum(float v) {
  const auto bits = [](float f) { return __builtin_bit_cast(uint32_t, f); };
  const auto val = [](uint32_t u) { return __builtin_bit_cast(float, u); };
  v += val(dpp<X1>(bits(v)));
  v += val(dpp<X2>(bits(v)));
  v += val(dpp<X4>(bits(v)));
  v += val(dpp<X8>(bits(v)));
  const auto r = __builtin_amdgcn_permlane16_swap(bits(v), bits(v), false, false);
  v = val(r[0]) + val(r[1]);
  const auto q = __builtin_amdgcn_permlane32_swap(bits(v), bits(v), false, false);
  return val(q[0]) + val(q[1]);
}

// Sum over the workgroup of T threads; `red` holds T / 64 floats, of its own for each use.
template <int T>
__device__ __forceinline__ float group_sum(float v, float* red) {
  v = wave_fsum(v);
  if constexpr (T == 64) return v;
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  v = 0.0f;
#pragma unroll
  for (int i = 0; i < T / 64; i++) v += red[i];
  return v;
}

// A workgroup per row, the row in registers: thread t holds the four-column groups t + T i, i < NV.  EARLY: the vectors
// are asked for together with the row (few rows: one wait for memory instead of three); otherwise where they are
// needed, other rows' waves covering the wait.  Bound by the bytes: 8192 x 2048 with bf16 y, gate, modulation and
// e4m3 rows (185 MB) 40 us, 4.6 TB/s; one row of 1024 2.4 us in a graph, 512 rows of 1600 with both norms 3.9.
template <int T, int NV, bool EARLY>
__global__ __launch_bounds__(T, EARLY ? 1 : 4) void residual_norm_kernel(NormArgs a) {
  __shared__ float red[3][T / 64];
  const int t = threadIdx.x;
  const uint32_t row32 = a.row0 + (uint32_t)xcd_remap(blockIdx.x, gridDim.x);
  const int64_t row = row32, grp = a.group_rows >= a.rows ? 0 : row32 / (uint32_t)a.group_rows;
  const float inv = 1.0f / (float)a.cols;
  // every access through a resource of the row's bytes: past its end loads give zeros and stores nothing (the whole
  // offset in the lanes' part: the bound is of that part alone)
  const __amdgpu_buffer_rsrc_t rx = f8_rsrc(a.x + row * a.ldx, 4 * a.cols);
  const auto load = [&](__amdgpu_buffer_rsrc_t rs, int i) {
    return __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, 16 * t + 16 * T * i, 0, 0));
  };
  const auto vec = [&](const float* p, int i) { return p ? load(f8_rsrc(p, 4 * a.cols), i) : f32x4{}; };
  const float *gate = a.gate ? a.gate + grp * a.gate_ld : nullptr, *scale = a.scale ? a.scale + grp * a.mod_ld : nullptr,
              *shift = a.scale ? a.shift + grp * a.mod_ld : nullptr;
  f32x4 x[NV], y[NV];
#pragma unroll
  for (int i = 0; i < NV; i++) x[i] = load(rx, i);
  if (a.y) {
    if (a.y_bf16) {
      const __amdgpu_buffer_rsrc_t ry = f8_rsrc((const uint16_t*)a.y + row * a.ldy, 2 * a.cols);
#pragma unroll
      for (int i = 0; i < NV; i++) {
        const auto u = __builtin_amdgcn_raw_buffer_load_b64(ry, 8 * t + 8 * T * i, 0, 0);
        y[i] = f32x4{__builtin_bit_cast(float, u[0] << 16), __builtin_bit_cast(float, u[0] & 0xffff0000u), __builtin_bit_cast(float, u[1] << 16),
                     __builtin_bit_cast(float, u[1] & 0xffff0000u)};
      }
    } else {
      const __amdgpu_buffer_rsrc_t ry = f8_rsrc((const float*)a.y + row * a.ldy, 4 * a.cols);
#pragma unroll
      for (int i = 0; i < NV; i++) y[i] = load(ry, i);
    }
  }
  constexpr int E = EARLY ? NV : 1;
  f32x4 pe[E], ge[E], we[E], ce[E], se[E];
  if constexpr (EARLY) {
#pragma unroll
    for (int i = 0; i < NV; i++) {
      pe[i] = vec(a.post_w, i);
      ge[i] = vec(gate, i);
      we[i] = vec(a.norm_w, i);
      ce[i] = vec(scale, i);
      se[i] = vec(shift, i);
    }
  }
  if (a.y) {
    if (a.post_w) {
      float ss = 0.0f;
#pragma unroll
      for (int i = 0; i < NV; i++)
#pragma unroll
        for (int e = 0; e < 4; e++) ss = __builtin_fmaf(y[i][e], y[i][e], ss);
      const float r = 1.0f / sqrtf(group_sum<T>(ss, red[0]) * inv + a.eps);
#pragma unroll
      for (int i = 0; i < NV; i++) y[i] = y[i] * r * (EARLY ? pe[i % E] : vec(a.post_w, i));
    }
    if (gate) {
#pragma unroll
      for (int i = 0; i < NV; i++) y[i] = y[i] * (EARLY ? ge[i % E] : vec(gate, i));
    }
#pragma unroll
    for (int i = 0; i < NV; i++) {
#pragma unroll
      for (int e = 0; e < 4; e++) x[i][e] = __builtin_fmaf(a.res_scale, y[i][e], x[i][e]);
      __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, x[i]), rx, 16 * t + 16 * T * i, 0, 0);
    }
  }
  if (a.layer) {
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; i++) s += (x[i][0] + x[i][1]) + (x[i][2] + x[i][3]);
    const float mean = group_sum<T>(s, red[1]) * inv;
    const bool whole = a.cols == 4 * T * NV;  // (past the row x stays zero)
#pragma unroll
    for (int i = 0; i < NV; i++)
#pragma unroll
      for (int e = 0; e < 4; e++) x[i][e] -= whole || 4 * (t + T * i) < a.cols ? mean : 0.0f;
  }
  float ss = 0.0f;
#pragma unroll
  for (int i = 0; i < NV; i++)
#pragma unroll
    for (int e = 0; e < 4; e++) ss = __builtin_fmaf(x[i][e], x[i][e], ss);
  const float r = 1.0f / sqrtf(group_sum<T>(ss, red[2]) * inv + a.eps);
#pragma unroll
  for (int i = 0; i < NV; i++) x[i] = x[i] * r;
  if (a.norm_w) {
#pragma unroll
    for (int i = 0; i < NV; i++) x[i] = x[i] * (EARLY ? we[i % E] : vec(a.norm_w, i));
  }
  if (scale) {
#pragma unroll
    for (int i = 0; i < NV; i++) {
      const f32x4 sc = EARLY ? ce[i % E] : vec(scale, i), sh = EARLY ? se[i % E] : vec(shift, i);
#pragma unroll
      for (int e = 0; e < 4; e++) x[i][e] = __builtin_fmaf(x[i][e], 1.0f + sc[e], sh[e]);
    }
  }
  if (a.h) {
    const __amdgpu_buffer_rsrc_t rh = f8_rsrc(a.h + row * a.ldh, 4 * a.cols);
#pragma unroll
    for (int i = 0; i < NV; i++) __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, x[i]), rh, 16 * t + 16 * T * i, 0, 0);
  }
  if (a.q) {  // 32 lanes hold one block of 128 columns (zeros past the row)
    const __amdgpu_buffer_rsrc_t rq = f8_rsrc(a.q + row * a.cols, a.cols);
#pragma unroll
    for (int i = 0; i < NV; i++) {
      float sc, mul;
      f8_scale(half_umax(amax4(x[i], 0)), sc, mul);
      __builtin_amdgcn_raw_buffer_store_b32(f8_pack(x[i], mul), rq, 4 * t + 4 * T * i, 0, 0);
      const int c = 4 * (t + T * i);
      if ((t & 31) == 0 && c < a.cols) a.s[(int64_t)(c >> 7) * a.rows + row] = sc;
    }
  }
}

// ------------------------------------------------------------------ products

typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));

// eight e4m3 values as bf16
__device__ __forceinline__ bf16x8 widen8(int lo, int hi) {
  const bf16x2_t a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, true),
                 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, true);
  return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// 32 values of k of a lane as four fragments of v_mfma_f32_16x16x32_bf16 (any order of k that both operands share
// will do)
struct Wide {
  bf16x8 v[4];
};
__device__ __forceinline__ Wide widen(i32x8 a) {
  Wide w;
#pragma unroll
  for (int i = 0; i < 4; i++) w.v[i] = widen8(a[2 * i], a[2 * i + 1]);
  return w;
}
__device__ __forceinline__ f32x4 mfma_wide(const Wide& a, const Wide& b) {
  f32x4 d{};
#pragma unroll
  for (int i = 0; i < 4; i++) d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.v[i], b.v[i], d, 0, 0, 0);
  return d;
}

__device__ __forceinline__ f32x4 fma4(float s, f32x4 d, f32x4 c) {
#pragma unroll
  for (int e = 0; e < 4; e++) c[e] = __builtin_fmaf(s, d[e], c[e]);
  return c;
}

__device__ __forceinline__ uint32_t bf16_bits(float v) { return __builtin_bit_cast(uint16_t, to_bf16(v)); }

// Columns n .. n + 3 of a row of N values; zeros past it.
__device__ __forceinline__ f32x4 f8_ld4(const float* p, int n, int N, int vec) {
  if (vec) return n < N ? ld4(p + n) : f32x4{};
  f32x4 v{};
#pragma unroll
  for (int e = 0; e < 4; e++)
    if (n + e < N) v[e] = p[n + e];
  return v;
}

// What is in columns n .. n + 3 of row m of the output.
__device__ __forceinline__ f32x4 f8_ld_out(const F8Args& a, int m, int n) {
  return m < a.M ? f8_ld4(a.out + (int64_t)m * a.ldc, n, a.N, a.vec) : f32x4{};
}

// Columns n .. n + 3 of row m of a linear's output from their sums, bias, gate and what is there.
__device__ __forceinline__ void f8_store(const F8Args& a, int m, int n, f32x4 r, f32x4 bias, f32x4 gate, f32x4 c) {
  if (m >= a.M || n >= a.N) return;
  const int64_t at = (int64_t)m * a.ldc + n;
#pragma unroll
  for (int e = 0; e < 4; e++) r[e] = __builtin_fmaf(r[e], a.alpha, bias[e]);
  if (a.add) r = r + f8_ld4(a.add + (int64_t)m * a.ld_add, n, a.N, a.vec);
  if (a.act) {
#pragma unroll
    for (int e = 0; e < 4; e++) r[e] = f8_act(r[e], a.act);
  }
  if (a.epi == ANIMA_EPI_RESID) {
    r = r + c;
  } else if (a.epi == ANIMA_EPI_GATED) {
#pragma unroll
    for (int e = 0; e < 4; e++) r[e] = __builtin_fmaf(gate[e], r[e], c[e]);
  }
  uint16_t* ob = (uint16_t*)a.out + at;
  if (a.vec) {
    if (a.obf) *(uint2*)ob = make_uint2(bf16_bits(r[0]) | bf16_bits(r[1]) << 16, bf16_bits(r[2]) | bf16_bits(r[3]) << 16);
    else *(f32x4*)(a.out + at) = r;
    return;
  }
#pragma unroll
  for (int e = 0; e < 4; e++) {
    if (n + e >= a.N) return;
    if (a.obf) ob[e] = (uint16_t)bf16_bits(r[e]);
    else a.out[at + e] = r[e];
  }
}

// The biases of columns n .. n + 3 of both projections.
struct GluBias {
  f32x4 g, u;
};
__device__ __forceinline__ GluBias f8_glu_bias(const F8Args& a, int n) {
  GluBias b{};
#pragma unroll
  for (int e = 0; e < 4; e++) {
    if (a.bias && n + e < a.N) b.g[e] = a.bias[n + e];
    if (a.bias2 && n + e < a.N) b.u[e] = a.bias2[n + e];
  }
  return b;
}

// h = act(g + b_gate) * (u + b_up)
__device__ __forceinline__ f32x4 f8_glu(int act, const GluBias& b, f32x4 g, f32x4 u) {
  g = g + b.g;
  u = u + b.u;
#pragma unroll
  for (int e = 0; e < 4; e++) g[e] = f8_act(g[e], act) * u[e];
  return g;
}

// f(the activation as a constant)
template <class F>
__device__ __forceinline__ void f8_with_act(int act, const F& f) {
  if (act == ANIMA_ACT_SILU) f(std::integral_constant<int, ANIMA_ACT_SILU>{});
  else if (act == ANIMA_ACT_GELU) f(std::integral_constant<int, ANIMA_ACT_GELU>{});
  else f(std::integral_constant<int, ANIMA_ACT_NONE>{});
}

__device__ __forceinline__ void f8_glu_store(const F8Args& a, int m, int n, f32x4 h) {
  if (m >= a.M || n >= a.N) return;
  float* o = a.out + (int64_t)m * a.ldc + n;
  if (a.vec) {
    *(f32x4*)o = h;
    return;
  }
#pragma unroll
  for (int e = 0; e < 4; e++)
    if (n + e < a.N) o[e] = h[e];
}

// f8_skinny: 16 outputs of 16 rows per workgroup, up to 16 waves that share the blocks of k; operands straight
// from memory into the matrix cores' registers (a lane: 32 consecutive k of one row), the waves' sums
// added through LDS in wave order.  QX: fp32 rows, each wave quantizing the blocks that it multiplies.  Sums in
// 32 bits whatever the precision asked for: these products wait for the weight's bytes.  Everything a wave reads of
// a block is asked for before the first use, x (whose quantization runs while the weight arrives) first, and the
// next block's weight before this one's products.  1 x 4096 x 1024 3.8 us in a graph, of which a launch takes 2; gated
// 4.7 (8.4 MB, 1.8 TB/s): two trips to memory in a row, not its bandwidth.
constexpr int SKW = 16;
constexpr uint32_t F8_PAST = 0x80000000u;  // an offset past every resource's end: reads as zero

// 32 bytes at k of a row that starts at `row`, zeros past K
__device__ __forceinline__ i32x8 f8_frag(__amdgpu_buffer_rsrc_t rs, uint32_t row, int k, int K) {
  const u32x4 lo = __builtin_amdgcn_raw_buffer_load_b128(rs, k < K ? row + k : F8_PAST, 0, 0);
  const u32x4 hi = __builtin_amdgcn_raw_buffer_load_b128(rs, k + 16 < K ? row + k + 16 : F8_PAST, 0, 0);
  return i32x8{(int)lo[0], (int)lo[1], (int)lo[2], (int)lo[3], (int)hi[0], (int)hi[1], (int)hi[2], (int)hi[3]};
}

template <bool QX, bool GLU>
__global__ __launch_bounds__(64 * SKW) void f8_skinny(F8Args a) {
  constexpr int TT = GLU ? 2 : 1;
  __shared__ f32x4 part[SKW][TT][64];
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, nw = blockDim.x >> 6;
  const int r = lane & 15, g = lane >> 4;
  const int n0 = blockIdx.x * 16, m0 = blockIdx.y * 16, m = m0 + r, K = a.K, KB = a.KB;
  const int nr = min(16, a.N - n0), mr = min(16, a.M - m0);
  const __amdgpu_buffer_rsrc_t rw = f8_rsrc(a.w + (int64_t)n0 * K, nr * (int64_t)K),
                               rw2 = GLU ? f8_rsrc(a.w2 + (int64_t)n0 * K, nr * (int64_t)K) : rw,
                               rx = QX ? f8_rsrc(a.x + (int64_t)m0 * a.ldx, 4 * ((mr - 1) * a.ldx + K))
                                       : f8_rsrc(a.xq + (int64_t)m0 * a.ldx, (mr - 1) * a.ldx + K);
  const float* ws = a.ws + (int64_t)(n0 >> 7) * KB;
  const float* ws2 = GLU ? a.ws2 + (int64_t)(n0 >> 7) * KB : nullptr;
  f32x4 acc[TT];
#pragma unroll
  for (int t = 0; t < TT; t++) acc[t] = f32x4{};
  const float* xs = QX ? nullptr : a.xs + min(m, a.M - 1);
  i32x8 w[TT], x;
  float sx = 0.0f;
  for (int kb = wave; kb < KB; kb += nw) {
    const int k = kb * 128 + 32 * g;
    f32x4 v[QX ? 8 : 1];
    if constexpr (QX) {
#pragma unroll
      for (int i = 0; i < 8; i++) {  // lane g: four values of every 16 (whole sectors of the 16 rows an instruction)
        const int c = 128 * kb + 16 * i + 4 * g;
        const u32x4 u = __builtin_amdgcn_raw_buffer_load_b128(rx, c < K && r < mr ? 4 * (r * (uint32_t)a.ldx + c) : F8_PAST, 0, 0);
        v[i] = __builtin_bit_cast(f32x4, u);
      }
    }
    if (kb == wave) {
      if constexpr (!QX) {
        x = f8_frag(rx, r * (uint32_t)a.ldx, k, K);
        sx = xs[(int64_t)kb * a.M];
      }
      w[0] = f8_frag(rw, r * K, k, K);
      if constexpr (GLU) w[1] = f8_frag(rw2, r * K, k, K);
    }
    i32x8 next[TT], nx;
    float ns = 0.0f;
    if (kb + nw < KB) {
      next[0] = f8_frag(rw, r * K, k + 128 * nw, K);
      if constexpr (GLU) next[1] = f8_frag(rw2, r * K, k + 128 * nw, K);
      if constexpr (!QX) {
        nx = f8_frag(rx, r * (uint32_t)a.ldx, k + 128 * nw, K);
        ns = xs[(int64_t)(kb + nw) * a.M];
      }
    }
    const float s0 = ws[kb], s1 = GLU ? ws2[kb] : 0.0f;
    if constexpr (QX) {
      uint32_t am = 0;
#pragma unroll
      for (int i = 0; i < 8; i++) am = amax4(v[i], am);
      float mul;
      f8_scale(cross_umax(am), sx, mul);
      // dword i holds k = 16 i + 4 g ...: two 4 x 4 transposes over g give lane g its 32 consecutive ones
      uint32_t e[2][4];
#pragma unroll
      for (int i = 0; i < 8; i++) e[i & 1][i >> 1] = f8_pack(v[i], mul);
#pragma unroll
      for (int o = 0; o < 2; o++) {
#pragma unroll
        for (int j = 0; j < 2; j++) {
          const auto t = __builtin_amdgcn_permlane32_swap(e[o][j], e[o][j + 2], false, false);
          e[o][j] = t[0];
          e[o][j + 2] = t[1];
        }
#pragma unroll
        for (int j = 0; j < 4; j += 2) {
          const auto t = __builtin_amdgcn_permlane16_swap(e[o][j], e[o][j + 1], false, false);
          x[4 * o + j] = (int)t[0];
          x[4 * o + j + 1] = (int)t[1];
        }
      }
    }
    const Wide xw = widen(x);
    acc[0] = fma4(sx * s0, mfma_wide(widen(w[0]), xw), acc[0]);
    if constexpr (GLU) acc[1] = fma4(sx * s1, mfma_wide(widen(w[1]), xw), acc[1]);
#pragma unroll
    for (int t = 0; t < TT; t++) w[t] = next[t];
    if constexpr (!QX) {
      x = nx;
      sx = ns;
    }
  }
  const int n = n0 + 4 * g;
  // (what the first wave needs for the epilogue, asked for before the sums meet)
  f32x4 bias{}, gate{}, c{};
  if constexpr (!GLU) {
    if (wave == 0) {
      if (a.bias) bias = f8_ld4(a.bias, n, a.N, a.vec);
      if (a.epi == ANIMA_EPI_GATED) gate = f8_ld4(a.gate, n, a.N, a.vec);
      if (a.epi != ANIMA_EPI_STORE) c = f8_ld_out(a, m, n);
    }
  }
  if (wave > 0) {
#pragma unroll
    for (int t = 0; t < TT; t++) part[wave][t][lane] = acc[t];
  }
  __syncthreads();
  if (wave > 0) return;
#pragma unroll
  for (int t = 0; t < TT; t++)
    for (int o = 1; o < nw; o++) acc[t] = acc[t] + part[o][t][lane];
  if constexpr (GLU) f8_glu_store(a, m, n, f8_glu(a.act, f8_glu_bias(a, n), acc[0], acc[1]));
  else f8_store(a, m, n, acc[0], bias, gate, c);
}

// f8_tile: one BM x BN output tile per workgroup (GLU: BN / 2 columns of each projection), waves of WM x WN.
// A stage is one block of 128 k: BM rows of x, BN of the weight (128 bytes each) and BM scales, filled NST - 1
// stages ahead by buffer_load ... lds.  LDS row r holds eight 16-byte units, unit u at slot u ^ (r / 2 % 8): a copy
// (eight whole rows, 1 KiB) is contiguous in LDS as the instruction needs it, and sixteen consecutive rows' reads
// of one unit touch each of the 64 banks once (229 bytes per cycle and CU; 120 with r % 8).  Rows past M (N) lie past their resource's end and units past K are sent
// there: they read as zero.  GLU: each 64 rows of the weight tile are 32 of the gate and the same 32 of the up
// projection, so that a lane holds both values of an output.  Tiles and waves: a lane holds its outputs' sums (half of
// its registers at 128 x 64) beside the products that are being added (16 registers each, two in turn), and a
// wave's tile decides what each loaded fragment is used for; two waves a SIMD cover each other's waits.
// 8192 x 2048 x 8192 into bf16 rows 116 to 124 us (2370 to 2220 TFLOP/s; matrix cores 67% busy at 1.6 GHz, the power
// limit), gated 8192 x 8192 x 2048 with 32-bit sums 466 to 489 (1180 to 1125; 58% at 1.8 GHz, the widening and the
// additions beside them).
typedef __attribute__((address_space(3))) void f8_lds_t;
#define F8_WAIT_VM(n) __builtin_amdgcn_s_waitcnt(((n) & 15) | (7 << 4) | (15 << 8) | (((n) >> 4) << 14))

__device__ __forceinline__ void f8_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// a wave's copy of 64 x 16 (x 4) bytes into LDS
__device__ __forceinline__ void f8_copy16(__amdgpu_buffer_rsrc_t rs, char* dst, uint32_t off) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (f8_lds_t*)dst, 16, off, 0, 0, 0);
}
__device__ __forceinline__ void f8_copy4(__amdgpu_buffer_rsrc_t rs, char* dst, uint32_t off) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (f8_lds_t*)dst, 4, off, 0, 0, 0);
}

template <int BM, int BN, int WM, int WN, int NST, bool WIDE, bool GLU>
__global__ __launch_bounds__(64 * (BM / WM) * (BN / WN), 2) void f8_tile(F8Args a) {
  constexpr int NWM = BM / WM, NW = NWM * (BN / WN), MT = WM / 32, NT = WN / 32;
  // LDS: the stages' rows of x, then those of the weight, the scales of x, the scales of the weight; each address is
  // a lane's register plus a constant
  constexpr int XB = BM * 128, WB = BN * 128, SB = GLU ? 512 : 256;  // bytes of a stage
  constexpr int WO = NST * XB, XSO = WO + NST * WB, WSO = XSO + NST * BM * 4;
  constexpr int EPL = NW * 32 * (MT < 2 ? 1 : 2) * ((GLU ? WN / 2 : WN) + 4) * 4;  // the epilogue's rows
  constexpr int LDS = WSO + NST * SB > EPL ? WSO + NST * SB : EPL;
  constexpr int CPW = (BM + BN) / 8 / NW, SPW = BM / 64;  // copies per wave: rows; waves that copy 64 scales each
  constexpr int FN = GLU ? BN / 2 : BN;                   // output columns of a tile
  static_assert(CPW * NW * 8 == BM + BN && SPW + (GLU ? 1 : 0) < NW && WN <= 64 && (!GLU || WN == 64), "copies and waves");
  __shared__ __attribute__((aligned(1024))) char smem[LDS];
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int r = lane & 31, hf = lane >> 5;
  const int ntn = (a.N + FN - 1) / FN, ntm = (a.M + BM - 1) / BM;
  int tm, tn;
  {
    // XCD x takes a contiguous range of tiles (dispatch is round-robin over the 8 XCDs), in groups of 8 row
    // tiles, column-major inside a group: the tiles in flight on one XCD share rows of both operands in its L2
    const int total = ntn * ntm, q = total >> 3, rem = total & 7, x = blockIdx.x & 7;
    const int t = x * q + min(x, rem) + (int)(blockIdx.x >> 3);
    const int grp = t / (8 * ntn), row0 = 8 * grp, gm = min(8, ntm - row0), local = t - grp * 8 * ntn;
    tn = local / gm;
    tm = row0 + (local - tn * gm);
  }
  const int bm = tm * BM, bn = tn * FN, K = a.K, KB = a.KB;
  const int kb0 = blockIdx.y * a.kbs, nkb = min(a.kbs, KB - kb0);
  if (blockIdx.y > 0) a.out += (int64_t)blockIdx.y * a.M * a.N;
  const int wm = (wave % NWM) * WM, wn = (wave / NWM) * WN;

  const int mrows = min(BM, a.M - bm), nrows = min(FN, a.N - bn);
  const __amdgpu_buffer_rsrc_t rx = f8_rsrc(a.xq + (int64_t)bm * a.ldx, (mrows - 1) * a.ldx + K),
                               rw = f8_rsrc(a.w + (int64_t)bn * K, nrows * (int64_t)K),
                               rw2 = GLU ? f8_rsrc(a.w2 + (int64_t)bn * K, nrows * (int64_t)K) : rw;
  // copy c of this wave: eight rows of one operand, row lane / 8 at (lane / 8) * ld + 16 * unit past their start
  int src[CPW];        // 0: x, 1: the weight, 2: the up projection
  uint32_t roff[CPW];  // where the rows start
#pragma unroll
  for (int c = 0; c < CPW; c++) {
    const int row = 8 * (wave * CPW + c), b = row - BM;
    src[c] = b < 0 ? 0 : GLU && (b & 32) ? 2 : 1;
    roff[c] = b < 0 ? (uint32_t)row * (uint32_t)a.ldx : (uint32_t)(GLU ? (b >> 6) * 32 + (b & 31) : b) * (uint32_t)K;
  }
  // One more copy in every wave, so that the wait counts are the same: 64 scales of x each, then the block scales of
  // the tile's columns (even lanes the first block of 128, odd lanes the second) and of the up projection's.  No
  // branch: a stage is one basic block, or its sums would move behind it.
  const bool up = GLU && wave > SPW;
  const float* sbase = wave < SPW ? a.xs + bm : (up ? a.ws2 : a.ws) + (int64_t)(bn >> 7) * KB;
  const int64_t sstep = wave < SPW ? a.M : 1;
  const int srec = wave < SPW ? mrows * 4 : min((a.N + 127) / 128 - (bn >> 7), 2) * KB * 4;
  const int sdst = wave < SPW ? XSO + wave * 256 : WSO + (up ? 256 : 0), sdstep = wave < SPW ? BM * 4 : SB;
  // The lanes' parts of the addresses are formed again for every stage (the asm keeps them there): registers are
  // what the sums leave, and a spilled one waits for all copies in flight.
  int ikb = kb0;  // the next block to copy (into buffer p = (ikb - kb0) % NST)
  uint32_t lx[2], lw[2], soff;
  const auto lanes = [&]() __attribute__((always_inline)) {
    int l;
    asm volatile("v_mbcnt_lo_u32_b32 %0, -1, 0\n\tv_mbcnt_hi_u32_b32 %0, -1, %0" : "=v"(l));
    const int unit = (l & 7) ^ (l >> 4), k = ikb * 128;  // (rows of an odd eight: unit ^ 4)
#pragma unroll
    for (int o = 0; o < 2; o++) {
      const int kl = k + 16 * (unit ^ 4 * o);
      lx[o] = (uint32_t)(l >> 3) * (uint32_t)a.ldx + (kl < K ? (uint32_t)kl : F8_PAST);
      lw[o] = (uint32_t)(l >> 3) * (uint32_t)K + (kl < K ? (uint32_t)kl : F8_PAST);
    }
    soff = wave < SPW ? 4 * (64 * wave + l) : 4 * ((l & 1) * KB);
  };
  const auto copies = [&](int p, int c0, int c1) __attribute__((always_inline)) {
#pragma unroll
    for (int c = c0; c < c1 && c < CPW; c++) {
      const uint32_t even = src[c] ? lw[c & 1] : lx[c & 1], odd = src[c] ? lw[~c & 1] : lx[~c & 1];
      f8_copy16(src[c] == 0 ? rx : src[c] == 1 ? rw : rw2, smem + (wave * CPW + c) * 1024 + (src[c] ? WO - XB + p * WB : p * XB),
                (CPW % 2 && wave & 1 ? odd : even) + roff[c]);
    }
    if (c1 == CPW + 1) {
      const int kbc = min(ikb, KB - 1);  // (past the last block its scales again, unused)
      f8_copy4(f8_rsrc(sbase + kbc * sstep, srec - (wave < SPW ? 0 : 4 * kbc)), smem + sdst + p * sdstep, soff);
      ikb++;
    }
  };
  f32x16 acc[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; i++)
#pragma unroll
    for (int j = 0; j < NT; j++) acc[i][j] = f32x16{};
  // a fragment: units 2 c + hf (c = 0 .. 3) of row r, 64 of the block's k in 16 registers
  int xa[4], wa[4];
#pragma unroll
  for (int c = 0; c < 4; c++) {
    const int f = r * 128 + 16 * ((2 * c + hf) ^ (r >> 1 & 7));
    xa[c] = f + wm * 128;
    wa[c] = f + wn * 128 + WO;
  }
  const auto axpy = [](float s, const f32x16& d, f32x16& c, int e0, int e1) __attribute__((always_inline)) {
#pragma unroll
    for (int e = e0; e < e1; e++) c[e] = __builtin_fmaf(s, d[e], c[e]);
  };

  const int xsa = XSO + 4 * (wm + r), wsa = WSO + 4 * (((bn + (GLU ? wn / 2 : wn)) >> 7) - (bn >> 7));
  const auto wscale = [&](int p, int up) __attribute__((always_inline)) { return *(const float*)(smem + wsa + p * SB + 256 * up); };
  const auto xscale = [&](int p, int i) __attribute__((always_inline)) { return *(const float*)(smem + xsa + p * BM * 4 + 128 * i); };
  const auto xunit = [&](int p, int i, int c) __attribute__((always_inline)) { return *(const i32x4*)(smem + xa[c] + p * XB + 4096 * i); };
  const auto wunit = [&](int p, int j, int c) __attribute__((always_inline)) { return *(const i32x4*)(smem + wa[c] + p * WB + 4096 * j); };

  // The order of a stage is written out (sched_barrier): a tile's sums are scaled and added between the products of
  // the tiles after it.  A stage's copies are issued one by one between the products of the last tiles of one stage
  // and of the first ones of the next (slots): all at once, they would wait for each other at the CU's one address
  // unit (72 of 16 cycles each) and the products behind them (a stage of 256 x 256 3700 cycles, spread 2850, without
  // copies 2650; with 32-bit sums 6500, 6050 and 5600).
  constexpr int T = MT * NT;
  constexpr bool SPREAD = T >= 4 || (WIDE && T == 2 && NST == 3);  // (else the next stage's wait would meet the copies)
  constexpr int SLOTS = WIDE ? 16 : 4 * NT;
  const auto slot = [&](int p, int n) __attribute__((always_inline)) {
    if constexpr (SPREAD) copies(p, (CPW + 1) * n / SLOTS, (CPW + 1) * (n + 1) / SLOTS);
  };
  constexpr int FIRST = SPREAD ? (CPW + 1) / 2 : CPW + 1;  // of the last stage before the loop
#pragma unroll
  for (int p = 0; p < NST; p++) {
    lanes();
    copies(p, 0, p + 1 < NST ? CPW + 1 : FIRST);
  }
  const auto stages = [&](const auto& stage) __attribute__((always_inline)) {  // the buffer as a constant
    int kb = 0;
    for (; kb + NST <= nkb; kb += NST) {
      stage(std::integral_constant<int, 0>{});
      stage(std::integral_constant<int, 1>{});
      if constexpr (NST == 3) stage(std::integral_constant<int, 2>{});
    }
    if (kb < nkb) stage(std::integral_constant<int, 0>{});
    if constexpr (NST == 3)
      if (kb + 1 < nkb) stage(std::integral_constant<int, 1>{});
  };
  // Stages overlap: before the last tiles of stage kb, whose fragments are in registers by then, a barrier ends every
  // wave's reads of the stage (its buffer is refilled) and publishes stage kb + 1 (arrived once at most the copies of
  // the NST - 2 stages after it pend), whose first fragments are then read under those tiles' products.
  const auto turn = [&](int p) __attribute__((always_inline)) {
    __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0)
    F8_WAIT_VM((NST - 2) * (CPW + 1));
    f8_barrier();
    lanes();
    if constexpr (!SPREAD) copies(p, 0, CPW + 1);
  };
  F8_WAIT_VM((NST - 2) * (CPW + 1) + FIRST);
  f8_barrier();
  static_assert((MT == 1 || MT % 2 == 0) && (T == 1 || T % 2 == 0), "fragments and sums alternate");
  f32x16 d[2];
  float sp = 0.0f;  // the scale of the tile in the other d
  d[1] = f32x16{};
  if constexpr (WIDE) {
    // One column of tiles after the other, so that the widened weight is one fragment; x, where its fragments of all
    // rows find registers, is widened once (KEEP: 128 x 128 tiles 7 to 10% faster), else again for each column, and
    // the registers of its bytes take the next row's units one by one.
    i32x4 xr[4], wr[4];
    bf16x8 wf[8];
    constexpr bool KEEP = NT > 1 && MT <= 2;
    bf16x8 xk[KEEP ? MT : 1][8];
#pragma unroll
    for (int c = 0; c < 4; c++) {
      xr[c] = xunit(0, 0, c);
      wr[c] = wunit(0, 0, c);
    }
    stages([&](auto buffer) __attribute__((always_inline)) {
      constexpr int p = decltype(buffer)::value, pn = (p + 1) % NST;
#pragma unroll
      for (int t = 0; t < T; t++) {
        const int j = t / MT, i = t % MT, pt = (t + T - 1) % T;
        const bool last = t + 1 == T;
        const float s = xscale(p, i) * wscale(p, GLU && j >= NT / 2);
        if (last) turn(p);
#pragma unroll
        for (int q = 0; q < 8; q++) {
          bf16x8& xq = xk[KEEP ? i : 0][q];
          if (!KEEP || j == 0) xq = widen8(xr[q / 2][q % 2 * 2], xr[q / 2][q % 2 * 2 + 1]);
          if (i == 0) wf[q] = widen8(wr[q / 2][q % 2 * 2], wr[q / 2][q % 2 * 2 + 1]);
          if (q % 2 == 1) {  // the unit is done with
            if (!KEEP || last || (j == 0 && i + 1 < MT)) xr[q / 2] = xunit(last ? pn : p, (i + 1) % MT, q / 2);
            if (i + 1 == MT) wr[q / 2] = wunit(last ? pn : p, (j + 1) % NT, q / 2);
          }
          d[t & 1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(wf[q], xq, q ? d[t & 1] : f32x16{}, 0, 0, 0);
          if (t == 0) slot((p + NST - 1) % NST, 8 + q);
          if (last) slot(p, q);
          if constexpr (T > 1) axpy(sp, d[(t + 1) & 1], acc[pt % MT][pt / MT], 2 * q, 2 * q + 2);
          __builtin_amdgcn_sched_barrier(0);
        }
        sp = s;
        if constexpr (T == 1) axpy(sp, d[0], acc[0][0], 0, 16);
      }
    });
  } else {
    i32x8 wf[NT][2], xf[2][2];
    const auto two = [](i32x4 lo, i32x4 hi) __attribute__((always_inline)) { return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7); };
    const auto x64 = [&](int p, int i, int h) __attribute__((always_inline)) { return two(xunit(p, i, 2 * h), xunit(p, i, 2 * h + 1)); };
    const auto w64 = [&](int p, int j, int h) __attribute__((always_inline)) { return two(wunit(p, j, 2 * h), wunit(p, j, 2 * h + 1)); };
#pragma unroll
    for (int h = 0; h < 2; h++) {
      xf[0][h] = x64(0, 0, h);
#pragma unroll
      for (int j = 0; j < NT; j++) wf[j][h] = w64(0, j, h);
    }
    stages([&](auto buffer) __attribute__((always_inline)) {
      constexpr int p = decltype(buffer)::value, pn = (p + 1) % NST;
      float s[NT];
#pragma unroll
      for (int t = 0; t < T; t++) {
        const int i = t / NT, j = t % NT, pt = (t + T - 1) % T;
        if (j == 0) {
#pragma unroll
          for (int n = 0; n < NT; n++) s[n] = xscale(p, i) * wscale(p, GLU && n >= NT / 2);
          if (i + 1 == MT) turn(p);
          if constexpr (MT > 1) {  // (past the last row: the next stage's first)
#pragma unroll
            for (int h = 0; h < 2; h++) xf[(i + 1) & 1][h] = i + 1 == MT ? x64(pn, 0, h) : x64(p, i + 1, h);
          }
        }
#pragma unroll
        for (int h = 0; h < 2; h++) {
          d[t & 1] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wf[j][h], xf[i & 1][h], h ? d[t & 1] : f32x16{}, 0, 0, 0, 0, 0, 0);
          if (i == 0) slot((p + NST - 1) % NST, 2 * NT + 2 * j + h);
          if (i + 1 == MT) slot(p, 2 * j + h);
          if constexpr (T > 1) axpy(sp, d[(t + 1) & 1], acc[pt / NT][pt % NT], 8 * h, 8 * h + 8);
          __builtin_amdgcn_sched_barrier(0);
        }
        if (i + 1 == MT) {
#pragma unroll
          for (int h = 0; h < 2; h++) {
            wf[j][h] = w64(pn, j, h);
            if (MT == 1 && j + 1 == NT) xf[0][h] = x64(pn, 0, h);
          }
        }
        sp = s[j];
        if constexpr (T == 1) axpy(sp, d[0], acc[0][0], 0, 16);
      }
    });
  }
  if constexpr (T > 1) axpy(sp, d[1], acc[MT - 1][NT - 1], 0, 16);
  F8_WAIT_VM(0);  // no copy into LDS outlives the loop

  // fp32 (bf16) rows leave through LDS, 64 rows of a wave at a time: a loop with 16 bytes of one row in neighbouring
  // lanes (whole lines; the accumulators' layout has 16 bytes of 32 rows), a lane keeping its four columns.
  constexpr int OC = GLU ? WN / 2 : WN, RS = OC + 4, LR = OC / 4, PR = 64 / LR, HR = MT < 2 ? 1 : 2;
  static_assert(NW * 32 * HR * RS * 4 <= LDS && 32 * HR * LR % 256 == 0, "the waves' rows fit; four passes at a time");
  const int n0 = bn + (GLU ? wn / 2 : wn);
  const auto quad = [](const f32x16& v, int q) __attribute__((always_inline)) {
    return f32x4{v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]};
  };
  if constexpr (GLU) {  // (NT = 2: a lane's gate and up values of columns n0 + 8 q + 4 hf + e)
    GluBias b[4];
#pragma unroll
    for (int q = 0; q < 4; q++) b[q] = f8_glu_bias(a, n0 + 8 * q + 4 * hf);
    f8_with_act(a.act, [&](auto act) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < MT; i++)
#pragma unroll
        for (int q = 0; q < 4; q++) {
          const f32x4 h = f8_glu(decltype(act)::value, b[q], quad(acc[i][0], q), quad(acc[i][1], q));
#pragma unroll
          for (int e = 0; e < 4; e++) acc[i][0][4 * q + e] = h[e];
        }
    });
  }
  f8_barrier();  // every wave's reads of the last stage are done
  if (a.out) {
    float* rows = (float*)smem + wave * (32 * HR * RS);
    const int n = n0 + 4 * (lane % LR);
    const float* line = rows + (lane / LR) * RS + 4 * (lane % LR);
    // rows 32 i ... of the wave into LDS, and `pass` for each four of a lane's rows (row in the tile, their values)
    const auto leave = [&](const auto& pass) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < MT; i += HR) {
#pragma unroll
        for (int k = 0; k < HR; k++)
#pragma unroll
          for (int j = 0; j < OC / 32; j++)
#pragma unroll
            for (int q = 0; q < 4; q++) *(f32x4*)(rows + (32 * k + r) * RS + 32 * j + 8 * q + 4 * hf) = quad(acc[i + k][j], q);
        __builtin_amdgcn_wave_barrier();
#pragma unroll 1
        for (int q = 0; q < 32 * HR; q += 4 * PR) {
          f32x4 v[4];
#pragma unroll
          for (int u = 0; u < 4; u++) v[u] = *(const f32x4*)(line + (q + u * PR) * RS);
          pass(bm + wm + 32 * i + q + lane / LR, v);
        }
        __builtin_amdgcn_wave_barrier();
      }
    };
    if constexpr (GLU) {
      leave([&](int m, const f32x4 (&v)[4]) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < 4; u++) f8_glu_store(a, m + u * PR, n, v[u]);
      });
    } else {
      const f32x4 bias = a.bias ? f8_ld4(a.bias, n, a.N, a.vec) : f32x4{};
      const f32x4 gate = a.epi == ANIMA_EPI_GATED ? f8_ld4(a.gate, n, a.N, a.vec) : f32x4{};
      if (a.vec && !a.add) {
        // the plain rows, each kind with code of its own: four rows' loads before the first store, one address each
        const int64_t step = (int64_t)PR * a.ldc;
        int M = n < a.N ? a.M : 0;
        float alpha = a.alpha;
        const auto plain = [&](auto kind, auto act) __attribute__((always_inline)) {
          constexpr int E = decltype(kind)::value;  // ANIMA_EPI_*, 3: bf16 rows
          leave([&](int m, f32x4 (&v)[4]) __attribute__((always_inline)) {
            const int64_t at = (int64_t)m * a.ldc + n;
            f32x4 c[4];
            if constexpr (E == ANIMA_EPI_RESID || E == ANIMA_EPI_GATED) {
#pragma unroll
              for (int u = 0; u < 4; u++) c[u] = m + u * PR < M ? ld4(a.out + at + u * step) : f32x4{};
            }
#pragma unroll
            for (int u = 0; u < 4; u++)
#pragma unroll
              for (int e = 0; e < 4; e++) {
                const float t = f8_act(__builtin_fmaf(v[u][e], alpha, bias[e]), decltype(act)::value);
                v[u][e] = E == ANIMA_EPI_RESID ? t + c[u][e] : E == ANIMA_EPI_GATED ? __builtin_fmaf(gate[e], t, c[u][e]) : t;
              }
#pragma unroll
            for (int u = 0; u < 4; u++)
              if (m + u * PR < M) {
                if constexpr (E == 3)
                  *(uint2*)((uint16_t*)a.out + at + u * step) =
                      make_uint2(bf16_bits(v[u][0]) | bf16_bits(v[u][1]) << 16, bf16_bits(v[u][2]) | bf16_bits(v[u][3]) << 16);
                else
                  *(f32x4*)(a.out + at + u * step) = v[u];
              }
          });
        };
        f8_with_act(a.act, [&](auto act) __attribute__((always_inline)) {
          if (a.epi == ANIMA_EPI_RESID) plain(std::integral_constant<int, ANIMA_EPI_RESID>{}, act);
          else if (a.epi == ANIMA_EPI_GATED) plain(std::integral_constant<int, ANIMA_EPI_GATED>{}, act);
          else if (a.obf) plain(std::integral_constant<int, 3>{}, act);
          else plain(std::integral_constant<int, ANIMA_EPI_STORE>{}, act);
        });
      } else {
        leave([&](int m, const f32x4 (&v)[4]) __attribute__((always_inline)) {
#pragma unroll
          for (int u = 0; u < 4; u++)
            f8_store(a, m + u * PR, n, v[u], bias, gate, a.epi != ANIMA_EPI_STORE ? f8_ld_out(a, m + u * PR, n) : f32x4{});
        });
      }
    }
  }
  if constexpr (GLU && FN == 128) {
    if (a.oq) {  // a tile is one block of 128 columns: its waves' maxima meet in LDS
      uint32_t* red = (uint32_t*)smem;  // [NW / NWM][BM]
#pragma unroll
      for (int i = 0; i < MT; i++) {
        uint32_t m = 0;
#pragma unroll
        for (int q = 0; q < 4; q++) m = amax4(n0 + 8 * q + 4 * hf < a.N ? quad(acc[i][0], q) : f32x4{}, m);  // (N % 16 == 0)
        const auto o = __builtin_amdgcn_permlane32_swap(m, m, false, false);
        m = umax(o[0], o[1]);
        if (hf == 0) red[(wave / NWM) * BM + wm + 32 * i + r] = m;
      }
      __syncthreads();
#pragma unroll
      for (int i = 0; i < MT; i++) {
        const int ml = wm + 32 * i + r, m = bm + ml;
        uint32_t am = 0;
#pragma unroll
        for (int w = 0; w < NW / NWM; w++) am = umax(am, red[w * BM + ml]);
        float scale, mul;
        f8_scale(am, scale, mul);
        // lane hf of a row holds columns 8 q + 4 hf: it gives away two quads and stores 16 columns from 16 hf on
        uint32_t p[4];
#pragma unroll
        for (int q = 0; q < 4; q++) p[q] = f8_pack(quad(acc[i][0], q), mul);
        const uint32_t g0 = (uint32_t)__shfl_xor((int)(hf ? p[0] : p[2]), 32), g1 = (uint32_t)__shfl_xor((int)(hf ? p[1] : p[3]), 32);
        if (m >= a.M) continue;
        const u32x4 o = hf ? u32x4{g0, p[2], g1, p[3]} : u32x4{p[0], g0, p[1], g1};
        if (n0 + 16 * hf < a.N) *(u32x4*)(a.oq + (int64_t)m * a.N + n0 + 16 * hf) = o;
        if (wave < NWM && hf == 0) a.os[(int64_t)tn * a.M + m] = scale;
      }
    }
  }
}

// The sums of a product's splits, added in their order, and its epilogue: a thread holds four columns of a row.
// Bound by its launch and one trip to memory: 100 x 1300 in six splits (3.6 MB) 3.1 us, 512 x 1024 in four (10.5 MB) 4.1
// (the loads in turn 4.0 and 4.8).
constexpr int F8_SPLITS = 8;
__global__ __launch_bounds__(256) void f8_join(F8Args a, const float* part, int splits) {
  const uint32_t i = blockIdx.x * 256 + threadIdx.x, quads = (uint32_t)(a.N + 3) / 4, row = i / quads;
  const int m = (int)row, n = (int)(4 * (i - row * quads));
  if (m >= a.M) return;
  const float* p = part + (int64_t)m * a.N;
  f32x4 v[F8_SPLITS];  // (all asked for before the first is added)
#pragma unroll
  for (int s = 0; s < F8_SPLITS; s++) v[s] = s < splits ? f8_ld4(p + (int64_t)s * a.M * a.N, n, a.N, a.vec) : f32x4{};
  const f32x4 bias = a.bias ? f8_ld4(a.bias, n, a.N, a.vec) : f32x4{};
  const f32x4 gate = a.epi == ANIMA_EPI_GATED ? f8_ld4(a.gate, n, a.N, a.vec) : f32x4{};
  const f32x4 c = a.epi != ANIMA_EPI_STORE ? f8_ld_out(a, m, n) : f32x4{};
  f32x4 r = v[0];
#pragma unroll
  for (int s = 1; s < F8_SPLITS; s++) r = r + v[s];
  f8_store(a, m, n, r, bias, gate, c);
}

// ------------------------------------------------------------------ host

namespace {

int refused(anima_ctx* c, int rc, const char* msg) { return fail(c, rc, "%s", msg); }

}  // namespace

int quant_rows_f8_launch(anima_ctx* c, const void* x, int x_bf16, int64_t M, int K, int64_t ldx, uint8_t* q, float* s) {
  char msg[256];
  if (int rc = check_quant_rows_f8(x, x_bf16, M, K, ldx, q, s, F8Msg{msg, sizeof msg})) return refused(c, rc, msg);
  if (M == 0) return ANIMA_OK;
  OnDevice on(c);
  const int KB = (K - 1) / 128 + 1;
  const int64_t ld = ldx ? ldx : K;
  const DivBy div = div_by((uint32_t)KB);
  Launch L(c, x_bf16 ? "quant.f8.bf16" : "quant.f8", 0.0, (double)M * K * (x_bf16 ? 3 : 5));
  const int64_t part = f8_quant_part(K);
  for (int64_t m = 0; m < M; m += part) {
    const uint32_t blocks = (uint32_t)((M - m < part ? M - m : part) * KB);
    const bool many = blocks >= 65536;  // (two blocks in flight per thread once the workgroups fill the chip)
    const dim3 grid((blocks + (many ? 31 : 15)) / (many ? 32 : 16)), block(256);
#define QR(T, U)                                                                                                                   \
  hipLaunchKernelGGL((quant_rows_f8_kernel<T, U>), grid, block, 0, c->stream, (const T*)x + m * ld, ld, blocks, K, M, div, q + m * K, \
                     s + m)
    if (x_bf16) {
      if (many) QR(uint16_t, 2);
      else QR(uint16_t, 1);
    } else {
      if (many) QR(float, 2);
      else QR(float, 1);
    }
#undef QR
  }
  return L.end();
}

int weight_quant_f8_launch(anima_ctx* c, const void* w, int w_bf16, int N, int K, uint8_t* q, float* scale) {
  char msg[256];
  if (int rc = check_weight_quant_f8(w, w_bf16, N, K, q, scale, F8Msg{msg, sizeof msg})) return refused(c, rc, msg);
  OnDevice on(c);
  const int KB = (K - 1) / 128 + 1;
  const int64_t blocks = (int64_t)((N - 1) / 128 + 1) * KB;
  Launch L(c, "weight_quant.f8", 0.0, (double)N * K * (w_bf16 ? 3 : 5));
  if (w_bf16)
    hipLaunchKernelGGL(weight_quant_f8_kernel<uint16_t>, dim3((unsigned)blocks), dim3(256), 0, c->stream, (const uint16_t*)w, N, K, KB, q,
                       scale);
  else
    hipLaunchKernelGGL(weight_quant_f8_kernel<float>, dim3((unsigned)blocks), dim3(256), 0, c->stream, (const float*)w, N, K, KB, q, scale);
  return L.end();
}

int residual_norm_launch(anima_ctx* c, const anima_resnorm_desc* d) {
  char msg[256];
  if (int rc = check_residual_norm(d, F8Msg{msg, sizeof msg})) return refused(c, rc, msg);
  if (d->rows == 0) return ANIMA_OK;
  OnDevice on(c);
  const int64_t C = d->cols;
  const auto ld = [&](int64_t v) { return v ? v : C; };
  NormArgs a{d->x,
             d->y,
             d->post_w,
             d->gate,
             d->norm_w,
             d->shift,
             d->scale,
             d->h,
             d->q,
             d->s,
             ld(d->ldx),
             ld(d->ldy),
             ld(d->ldh),
             ld(d->gate_ld),
             ld(d->mod_ld),
             d->group_rows ? d->group_rows : d->rows,
             d->res_scale != 0.0f ? d->res_scale : 1.0f,
             d->eps,
             (int)d->rows,
             d->cols,
             d->norm == ANIMA_NORM_LAYER,
             d->y_bf16,
             0};
  Launch L(c, "residual_norm", 0.0, (double)d->rows * C * ((d->y ? d->y_bf16 ? 10.0 : 12.0 : 4.0) + (d->h ? 4 : 0) + (d->q ? 1 : 0)));
#define RN(T, NV, EARLY)                                                                                                     \
  for (int64_t r = 0, part = f8_norm_part(T); r < d->rows; r += part) {                                                      \
    a.row0 = (uint32_t)r;                                                                                                    \
    hipLaunchKernelGGL((residual_norm_kernel<T, NV, EARLY>), dim3((unsigned)(d->rows - r < part ? d->rows - r : part)), dim3(T), 0, \
                       c->stream, a);                                                                                        \
  }
  if (d->rows <= 4 * c->num_cus) {
    if (C <= 256) RN(64, 1, true)
    else if (C <= 512) RN(128, 1, true)
    else if (C <= 1024) RN(256, 1, true)
    else if (C <= 2048) RN(256, 2, true)
    else if (C <= 4096) RN(512, 2, true)
    else if (C <= 8192) RN(1024, 2, true)
    else RN(1024, 4, true)
  } else {
    if (C <= 256) RN(64, 1, false)
    else if (C <= 512) RN(64, 2, false)
    else if (C <= 1024) RN(64, 4, false)
    else if (C <= 2048) RN(64, 8, false)
    else if (C <= 4096) RN(128, 8, false)
    else if (C <= 8192) RN(256, 8, false)
    else RN(512, 8, false)
  }
#undef RN
  return L.end();
}

// The product's input as e4m3 rows: those given, or fp32 rows in `a` as they are.
static void f8_input(F8Args& a, const anima_weight* W, const float* x, int64_t ldx, const int8_t* xq, const float* xs) {
  a.xq = (const uint8_t*)xq;
  a.xs = xs;
  a.x = xq ? nullptr : x;
  a.ldx = ldx ? ldx : W->K;
  a.N = W->N;
  a.K = W->K;
  a.KB = (W->K + 127) / 128;
}

// The kernel for a product's sizes.
enum { F8_SKINNY, F8_256, F8_128, F8_MID, F8_64, F8_COUNT };  // (F8_MID: 128 x 64, gated 64 x 256)

static int64_t f8_tiles(int kind, bool glu, int64_t M, int64_t N) {
  static const int bm[2][F8_COUNT] = {{16, 256, 128, 128, 64}, {16, 256, 128, 64, 64}};
  static const int bn[2][F8_COUNT] = {{16, 256, 128, 64, 64}, {16, 128, 64, 128, 64}};  // (gated: columns of each projection)
  return (M + bm[glu][kind] - 1) / bm[glu][kind] * ((N + bn[glu][kind] - 1) / bn[glu][kind]);
}

// Microseconds of a product (f8_skinny: base + step for each block of k of a wave + work for each 4096 blocks that all
// its workgroups read; tiles: base + for each tile per CU step for each block of k, round for each tile after the first)
// + out for a million outputs.  Fitted to 3000 products of M = 1 .. 8192, N and K = 64 .. 8192: the choice takes
// 0.1 to 1.0% longer than the best kernel in the mean (the linear's 128 x 64 tiles with 32-bit sums as they were with
// two stages; their third took 4 to 5% off where the choice takes 128 x 128: 4096 x 1024 x 2048, 2048 x 2048 x 4096).
// Small products are bound by the depth of one workgroup's k loop, so they take the waves of f8_skinny or small tiles;
// large ones by the bytes that a tile's operands move per product (43 x 2048 x 1024: 4.6, 64x64 8.6, 256x256 33 us;
// 3013 x 1316 x 1424 gated with 32-bit sums: 64x64 26.2, 128x64 23.3; 8192 x 2048 x 8192: 64x64 220, 256x256 116).
// The gated form leaves e4m3 rows from the tiles of 128 columns; from the others they cost a pass.
// Where the tiles leave CUs idle, the k loop of a linear is split (*splits): each split's sums go through memory and
// f8_join (512 x 1024 x 8192 with 32-bit sums 32.7 us, split 20.0; 64 x 4096 x 4096 20.4, 12.5; 300 x 384 x 4096 10.9,
// 11.3: not taken).
static int f8_choose(anima_ctx* c, bool glu, bool f8_out, int64_t M, int64_t N, int K, int precision, int* splits) {
  struct Fit {
    float base, step, round, out;
  };
  static const Fit fit[2][2][F8_COUNT] = {
      {{{1.55f, 1.05f, 1.58f, 0.0f}, {6.95f, 1.20f, 1.40f, 0.66f}, {4.20f, 0.68f, 0.0f, 0.61f}, {3.59f, 0.40f, 0.1f, 0.76f}, {3.24f, 0.312f, 0.0f, 0.67f}},
       {{1.55f, 1.05f, 1.60f, 0.0f}, {6.75f, 2.58f, 2.0f, 0.72f}, {4.31f, 0.852f, 0.0f, 0.70f}, {3.51f, 0.625f, 0.0f, 0.53f}, {3.30f, 0.408f, 0.0f, 0.61f}}},
      {{{1.15f, 1.80f, 2.75f, 0.08f}, {7.80f, 1.34f, 5.96f, 0.92f}, {4.66f, 0.73f, 0.0f, 0.97f}, {4.82f, 0.78f, 3.04f, 1.25f}, {4.84f, 0.535f, 0.2f, 1.05f}},
       {{1.15f, 1.80f, 2.75f, 0.08f}, {7.50f, 2.61f, 5.70f, 0.85f}, {4.56f, 0.87f, 0.0f, 1.09f}, {4.83f, 1.07f, 2.65f, 1.23f}, {4.85f, 0.723f, 0.2f, 1.15f}}}};
  const int KB = (K + 127) / 128;
  int best = F8_256, sbest = F8_256, sn = 1;
  float bt = 0.0f, st = 0.0f;  // of the best kernel, of the best one with its k loop split
  for (int k = F8_COUNT - 1; k >= 0; k--) {
    const int64_t tiles = f8_tiles(k, glu, M, N);
    // the grid's second dimension, and its threads (512 a tile at the most); 256 x 256 tiles have room for every product
    // whose output finds memory
    if (k == F8_SKINNY ? M > 16 * 65535 || (N + 15) / 16 * 64 * SKW > F8_MAX_THREADS : tiles > F8_MAX_THREADS / 512) continue;
    const Fit& f = fit[glu][precision][k];
    const float rounds = (float)((tiles + c->num_cus - 1) / c->num_cus), mn = 1e-6f * (float)M * (float)N;
    const bool fused = k == F8_256 || k == F8_MID;
    float us = f.base + f.out * mn * (f8_out && fused ? 0.6f : 1.0f);
    if (k == F8_SKINNY) us += f.step * (float)((KB + SKW - 1) / SKW) + f.round * (float)tiles * (float)KB / 4096.0f;
    else us += f.step * (float)KB * rounds + f.round * (rounds - 1.0f);
    if (f8_out && !fused) us += 2.0f + 1.2f * mn;
    if (bt == 0.0f || us < bt) {
      best = k;
      bt = us;
    }
    if (glu || k == F8_SKINNY || tiles > 2 * c->num_cus || KB < 8) continue;
    for (int s = 2; s <= F8_SPLITS; s++) {
      const int kbs = (KB + s - 1) / s, n = (KB + kbs - 1) / kbs;
      if (kbs < 3 || M * N * n > (1 << 26)) break;
      const float rs = (float)((tiles * n + c->num_cus - 1) / c->num_cus);
      us = f.base + f.step * (float)kbs * rs + f.round * (rs - 1.0f) + f.out * mn * (float)n + 2.4f + mn * (1.6f + (float)n);
      if (st == 0.0f || us < st) {
        sbest = k;
        st = us;
        sn = n;
      }
    }
  }
  const bool split = st > 0.0f && st < 0.9f * bt;  // (what the model is sure of)
  *splits = split ? sn : 1;
  return split ? sbest : best;
}

// Whether fp32 rows are quantized inside f8_skinny (each workgroup quantizes its 16 rows again) instead of by a pass
// before the product (1.6 to 2.5 us): rows of x times blocks of one workgroup, and of all, below what a
// pass costs.  1 row of 1024 to 2048 outputs 3.8 us with the pass 5.1, of 8192 12.1 and 10.3; 16 rows of 1024 5.1 and 5.9,
// of 2048 7.4 and 6.9; 48 rows of 1024 7.4 and 6.8.
static bool f8_quantizes(const F8Args& a, int kind) {
  if (kind != F8_SKINNY || a.ldx >= (1 << 25)) return false;  // (16 rows within a resource's 2^31 bytes)
  const int64_t work = (4 + (a.M < 16 ? a.M : 16)) * (int64_t)a.KB;
  return work <= 240 && work * f8_tiles(F8_SKINNY, false, a.M, a.N) <= 50000;
}

template <int BM, int BN, int WM, int WN, int NST, bool GLU>
static void f8_tile_launch(anima_ctx* c, const F8Args& a, int precision) {
  constexpr int FN = GLU ? BN / 2 : BN;
  const dim3 grid((unsigned)((int64_t)((a.N + FN - 1) / FN) * ((a.M + BM - 1) / BM)), (unsigned)((a.KB + a.kbs - 1) / a.kbs)), block(64 * (BM / WM) * (BN / WN));
  if (precision == ANIMA_PREC_FP32) hipLaunchKernelGGL((f8_tile<BM, BN, WM, WN, NST, true, GLU>), grid, block, 0, c->stream, a);
  else hipLaunchKernelGGL((f8_tile<BM, BN, WM, WN, NST, false, GLU>), grid, block, 0, c->stream, a);
}

// Runs the product of a's rows, quantizing fp32 rows first where the kernel takes e4m3 rows.
template <bool GLU>
static int f8_product(anima_ctx* c, F8Args a, int kind, int precision, int splits) {
  static const char* const names[2][F8_COUNT] = {{"gemm.f8.skinny", "gemm.f8.256x256", "gemm.f8.128x128", "gemm.f8.128x64", "gemm.f8.64x64"},
                                                 {"glu.f8.skinny", "glu.f8.256x256", "glu.f8.128x128", "glu.f8.64x256", "glu.f8.64x128"}};
  void* scratch = nullptr;
  if (a.x && !f8_quantizes(a, kind)) {
    const size_t qb = ((size_t)a.M * a.K + 255) / 256 * 256;
    if (int rc = anima_alloc(c, qb + (size_t)a.M * a.KB * 4, &scratch)) return rc;
    a.xq = (const uint8_t*)scratch;
    a.xs = (const float*)((char*)scratch + qb);
    const int rc = quant_rows_f8_launch(c, a.x, 0, a.M, a.K, a.ldx, (uint8_t*)scratch, (float*)((char*)scratch + qb));
    if (rc != ANIMA_OK) {
      anima_free(c, scratch);
      return rc;
    }
    a.ldx = a.K;
    a.x = nullptr;
  }
  const F8Args whole = a;
  void* part = nullptr;
  a.kbs = (a.KB + splits - 1) / splits;
  if (splits > 1) {  // (a linear's tiles) the sums alone, into pooled scratch
    if (int rc = anima_alloc(c, (size_t)splits * a.M * a.N * 4, &part)) {
      if (scratch) anima_free(c, scratch);
      return rc;
    }
    a.out = (float*)part;
    a.ldc = a.N;
    a.alpha = 1.0f;
    a.bias = a.add = nullptr;
    a.act = ANIMA_ACT_NONE;
    a.epi = ANIMA_EPI_STORE;
    a.obf = 0;
    a.vec = a.N % 4 == 0;
  }
  Launch L(c, names[GLU][kind], (GLU ? 4.0 : 2.0) * a.M * a.N * a.K, (double)a.N * a.K * (GLU ? 2 : 1));
  if (kind == F8_SKINNY) {
    const dim3 grid((unsigned)((a.N + 15) / 16), (unsigned)((a.M + 15) / 16)), block(64 * (a.KB < SKW ? a.KB : SKW));
    if (a.x) hipLaunchKernelGGL((f8_skinny<true, GLU>), grid, block, 0, c->stream, a);
    else hipLaunchKernelGGL((f8_skinny<false, GLU>), grid, block, 0, c->stream, a);
  } else if (kind == F8_256) {
    f8_tile_launch<256, 256, 128, 64, 2, GLU>(c, a, precision);
  } else if (kind == F8_128) {
    f8_tile_launch<128, 128, 64, 64, 2, GLU>(c, a, precision);
  } else if (kind == F8_MID) {
    if constexpr (GLU) f8_tile_launch<64, 256, 32, 64, 2, GLU>(c, a, precision);
    else f8_tile_launch<128, 64, 64, 32, 3, GLU>(c, a, precision);  // (1024 x 2048 x 2048 with 2 stages 15.1 us, 3 12.4)
  } else {
    if constexpr (GLU) f8_tile_launch<64, 128, 32, 64, 3, GLU>(c, a, precision);
    else f8_tile_launch<64, 64, 32, 32, 3, GLU>(c, a, precision);
  }
  int rc = L.end();
  if (part) {
    if (rc == ANIMA_OK) {
      Launch J(c, "gemm.f8.join", 0.0, (double)a.M * a.N * 4 * (splits + 1));
      const int64_t quads = (int64_t)a.M * ((a.N + 3) / 4);
      hipLaunchKernelGGL(f8_join, dim3((unsigned)((quads + 255) / 256)), dim3(256), 0, c->stream, whole, (const float*)part, splits);
      rc = J.end();
    }
    anima_free(c, part);
  }
  if (scratch) anima_free(c, scratch);
  return rc;
}

int linear_f8_launch(anima_ctx* c, const anima_linear_desc* d) {
  char msg[256];
  if (int rc = check_linear_f8(d, F8Msg{msg, sizeof msg})) return refused(c, rc, msg);
  OnDevice on(c);
  const anima_weight* W = d->W;
  F8Args a{};
  f8_input(a, W, d->x, d->ldx, d->xq, d->xs);
  a.M = (int)d->M;
  a.w = (const uint8_t*)W->w;
  a.ws = W->scale;
  a.bias = W->bias;
  a.out = d->out;
  a.ldc = d->ldc ? d->ldc : W->N;
  a.alpha = d->alpha != 0.0f ? d->alpha : 1.0f;
  a.act = d->act;
  a.epi = d->epilogue;
  a.gate = d->gate ? d->gate + d->gate_off : nullptr;
  a.add = d->add;
  a.ld_add = d->ld_add ? d->ld_add : W->N;
  a.obf = d->out_bf16;
  a.vec = a.N % 4 == 0 && a.ldc % 4 == 0 && f8_al(a.out, a.obf ? 8 : 16) && f8_al(a.bias, 16) && (!a.add || (a.ld_add % 4 == 0 && f8_al(a.add, 16))) &&
          (a.epi != ANIMA_EPI_GATED || f8_al(a.gate, 16));
  int splits = 1;
  const int kind = f8_choose(c, false, false, a.M, a.N, a.K, d->precision, &splits);
  return f8_product<false>(c, a, kind, d->precision, splits);
}

int linear_glu_launch(anima_ctx* c, const anima_glu_desc* d) {
  char msg[256];
  if (int rc = check_linear_glu(d, F8Msg{msg, sizeof msg})) return refused(c, rc, msg);
  if (d->M == 0) return ANIMA_OK;
  OnDevice on(c);
  const anima_weight *G = d->gate, *U = d->up;
  F8Args a{};
  f8_input(a, G, d->x, d->ldx, d->xq, d->xs);
  a.M = (int)d->M;
  a.w = (const uint8_t*)G->w;
  a.ws = G->scale;
  a.bias = G->bias;
  a.w2 = (const uint8_t*)U->w;
  a.ws2 = U->scale;
  a.bias2 = U->bias;
  a.act = d->act;
  a.out = d->out;
  a.ldc = d->ldc ? d->ldc : a.N;
  void* tmp = nullptr;
  int splits = 1;
  const int kind = f8_choose(c, true, d->out_q != nullptr, a.M, a.N, a.K, d->precision, &splits);
  if (d->out_q && (kind == F8_256 || kind == F8_MID)) {  // a tile is one block of 128 columns
    a.oq = d->out_q;
    a.os = d->out_s;
    a.out = nullptr;
  } else if (d->out_q) {  // fp32 rows first (pooled scratch), then their e4m3 rows
    if (int rc = anima_alloc(c, (size_t)a.M * a.N * 4, &tmp)) return rc;
    a.out = (float*)tmp;
    a.ldc = a.N;
  }
  a.vec = a.N % 4 == 0 && a.ldc % 4 == 0 && f8_al(a.out, 16);
  int rc = f8_product<true>(c, a, kind, d->precision, splits);
  if (tmp) {
    if (rc == ANIMA_OK) rc = quant_rows_f8_launch(c, tmp, 0, a.M, a.N, 0, d->out_q, d->out_s);
    anima_free(c, tmp);
  }
  return rc;
}

}  // namespace anima
