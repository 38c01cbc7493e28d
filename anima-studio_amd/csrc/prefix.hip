// Attention of many sequences behind one shared prefix (anima_attention_prefix).
//
//   o[i] = sum_j p_ij v_j,  p_ij = exp(scale q_i . k_j) / sum_j,  j over the P prefix keys and the row's own
//   sequence's keys (causal: up to itself)
//
// The sequences' rows are packed, so the prefix is one product for all of them: tiles of rows run over the prefix's key
// blocks whatever sequence the rows belong to, then over the packed keys of their own sequences, masked by each row's
// range of them.  One pass before it norms and rotates q and the packed K (at P + place), and lays K and V out as the
// prefix's are.
#include <algorithm>
#include <type_traits>

#include "common.h"
#include "internal.h"
#include "prefix_args.h"

namespace anima {

constexpr int PHD = 128;      // head dim
constexpr int PBK = PREFIX_BLOCK;
constexpr int PSEQ = 256;     // sequences of one launch (their first rows go with the kernel's arguments)
constexpr float LOG2E = 1.4426950408889634f;

typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

struct PrefixSeqs {
  int n;                // sequences
  int start[PSEQ + 1];  // first packed row of each, then the number of rows
};

// The sequences' first rows in LDS: a search there is a few LDS reads, in the arguments as many trips to memory.
struct SeqStarts {
  int at[PSEQ + 1];
  __device__ __forceinline__ void fill(const PrefixSeqs& s) {  // (a barrier follows)
    for (int i = threadIdx.x; i <= s.n; i += blockDim.x) at[i] = s.start[i];
  }
  // the sequence of packed row l
  __device__ __forceinline__ int of(int n, int l) const {
    int lo = 0, hi = n - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (at[mid] <= l) lo = mid;
      else hi = mid - 1;
    }
    return lo;
  }
};

struct PrefixArgs {
  const float* q;
  int64_t ldq;
  const float* k;
  int64_t ldk;
  const float* v;
  int64_t ldv;
  void* o;
  int64_t ldo;
  const void* pk;   // prefix: K [Hkv][Pp][128], V^T [Hkv][Pp/64][128][64] (a block's rows in one piece: rows of all keys would
  const void* pvt;  // lie a power of two apart, in one memory channel)
  void* ok;         // own: the same of Tp keys
  void* ovt;
  void* pq;         // q [Hkv][V][128], ready to be multiplied: normed, rotated, times c
  int2* range;      // [T] own keys that a row sees: from, to
  const float* qn;
  const float* kn;
  const float* cs;
  int64_t sin_off;
  float eps, c;     // c = scale * log2(e)
  int T, Tp, P, Pp, H, Hkv, group, causal, obf;
  // tiles: virtual rows V = T * group of a kv head (row v / group, its head v % group), key blocks in `splits` parts
  int V, nt, splits;
  float* po;        // [splits][Hkv][V][128] sums, and
  float* pml;       // [splits][Hkv][V][2] maximum and sum of weights, of a split call
  PrefixSeqs seq;
};

// A workgroup barrier that waits for nothing: what it publishes has been waited for before it.
__device__ __forceinline__ void p_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// One workgroup per 64 packed rows and kv head (then, with a.pq, per q head); rows T .. Tp are zeros.  K: 16 lanes a row, lane q
// holding dims 4 q .. + 3 and 64 + the same (both of each rotated pair); V: wave w takes dims 32 w .. + 31 of all rows, lane
// (q, c) the eight keys of V^T chunk c at dims 4 q .. + 3, so that every load and store moves whole lines.  The bf16 form has K
// and q in f16 (their rounding to 8 bits alone would be 0.005 of a result) and keeps each 16 keys of a V^T row as 0-3, 8-11,
// 4-7, 12-15, as the matrix products take them.  Every part of a split call would norm and rotate q again: once here (64 rows behind
// 8192 keys 36 us with it in the tiles, 31 so).  Bound by memory (7741 rows of 16 and 8 heads: 190 MB, 36 us, 5.2 TB/s), few
// rows by a launch and three trips to memory, one behind the other (7 us).
// A key whose K or V is not finite (in its form) gets a K of NaN and a V of zeros: every row that sees it becomes NaN, and where it
// is masked its weight of 0 meets no NaN in V.
template <class T>
__global__ __launch_bounds__(256) void prefix_prep_kernel(PrefixArgs a) {
  constexpr bool BF = sizeof(T) == 2;
  typedef std::conditional_t<BF, _Float16, float> TK;
  __shared__ int bad[64], start[64];  // of the rows: whether they are not finite, their sequences' first rows
  __shared__ SeqStarts seq;
  const int t = threadIdx.x, w = t >> 6, lane = t & 63, kb0 = blockIdx.x * 64;
  const bool query = (int)blockIdx.y >= a.Hkv;
  const int hk = query ? blockIdx.y - a.Hkv : blockIdx.y;  // (its q head)
  const int q16 = lane & 15, rsub = lane >> 4, vq = lane & 7, vc = lane >> 3;
  const auto vkey = [&](int e) { return BF ? kb0 + 16 * (vc >> 1) + 4 * (vc & 1) + (e & 3) + 8 * (e >> 2) : kb0 + 8 * vc + e; };
  f32x4 klo[4], khi[4], ve[8], cv[4], sv[4], wl{}, wh{};
  const float* const x = query ? a.q : a.k;
  const int64_t ldx = query ? a.ldq : a.ldk;
  const float* const norm = query ? a.qn : a.kn;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const int l = min(kb0 + 16 * w + 4 * i + rsub, a.T - 1);
    const float* src = x + (int64_t)l * ldx + hk * PHD + 4 * q16;
    klo[i] = *(const f32x4*)src;
    khi[i] = *(const f32x4*)(src + 64);
  }
  if (!query) {
#pragma unroll
    for (int e = 0; e < 8; e++) ve[e] = *(const f32x4*)(a.v + (int64_t)min(vkey(e), a.T - 1) * a.ldv + hk * PHD + 32 * w + 4 * vq);
  }
  if (norm) {
    wl = *(const f32x4*)(norm + 4 * q16);
    wh = *(const f32x4*)(norm + 64 + 4 * q16);
  }
  if (t < 64) bad[t] = 0;
  seq.fill(a.seq);
  __builtin_amdgcn_s_waitcnt(0xc07f);  // (LDS alone: the loads above go on)
  p_barrier();
  if (t < 64) {
    const int l = min(kb0 + t, a.T - 1), b = seq.of(a.seq.n, l);
    start[t] = seq.at[b];
    if (a.range && blockIdx.y == 0 && kb0 + t < a.T) a.range[l] = make_int2(seq.at[b], a.causal ? l + 1 : seq.at[b + 1]);
  }
  __builtin_amdgcn_s_waitcnt(0xc07f);
  p_barrier();
  if (a.cs) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const int rl = 16 * w + 4 * i + rsub, l = min(kb0 + rl, a.T - 1);
      const float* cr = a.cs + (int64_t)(a.P + l - start[rl]) * 64 + 4 * q16;
      cv[i] = *(const f32x4*)cr;
      sv[i] = *(const f32x4*)(cr + a.sin_off);
    }
  }
  const auto finite = [](f32x4 v, auto as) {
    float m = 0.0f;
#pragma unroll
    for (int j = 0; j < 4; j++) m += (float)(decltype(as))v[j] * 0.0f;  // (0 of finite values, else NaN)
    return m == 0.0f;
  };
  const auto put = [](TK* d, f32x4 lo, f32x4 hi) {
    if constexpr (BF) {
      *(f16x4*)d = f16x4{(_Float16)lo[0], (_Float16)lo[1], (_Float16)lo[2], (_Float16)lo[3]};
      *(f16x4*)(d + 64) = f16x4{(_Float16)hi[0], (_Float16)hi[1], (_Float16)hi[2], (_Float16)hi[3]};
    } else {
      *(f32x4*)d = lo;
      *(f32x4*)(d + 64) = hi;
    }
  };
#pragma unroll
  for (int i = 0; i < 4; i++) {
    f32x4 lo = klo[i], hi = khi[i];
    if (norm) {
      float ss = 0.0f;
#pragma unroll
      for (int j = 0; j < 4; j++) ss += lo[j] * lo[j] + hi[j] * hi[j];
#pragma unroll
      for (int s = 1; s < 16; s <<= 1) ss += __shfl_xor(ss, s);
      const float rn = 1.0f / sqrtf(ss / 128.0f + a.eps);
      lo = lo * rn * wl;
      hi = hi * rn * wh;
    }
    if (a.cs) {
      const f32x4 x = lo;
      lo = x * cv[i] - hi * sv[i];
      hi = hi * cv[i] + x * sv[i];
    }
    klo[i] = lo;
    khi[i] = hi;
    if (!query && (!finite(lo, TK()) || !finite(hi, TK()))) bad[16 * w + 4 * i + rsub] = 1;
  }
  if (query) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const int l = kb0 + 16 * w + 4 * i + rsub;
      if (l < a.T) put((TK*)a.pq + ((int64_t)(hk / a.group) * a.V + (int64_t)l * a.group + hk % a.group) * PHD + 4 * q16, klo[i] * a.c, khi[i] * a.c);
    }
    return;
  }
#pragma unroll
  for (int e = 0; e < 8; e++)
    if (!finite(ve[e], T())) bad[vkey(e) - kb0] = 1;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const int r = 16 * w + 4 * i + rsub, l = kb0 + r;
    const float k = __builtin_nanf("");
    const f32x4 z = l < a.T ? f32x4{k, k, k, k} : f32x4{};
    const bool keep = l < a.T && !bad[r];
    put((TK*)a.ok + ((int64_t)hk * a.Tp + l) * PHD + 4 * q16, keep ? klo[i] : z, keep ? khi[i] : z);
  }
#pragma unroll
  for (int e = 0; e < 8; e++)
    if (vkey(e) >= a.T || bad[vkey(e) - kb0]) ve[e] = f32x4{};
  T* vd = (T*)a.ovt + ((int64_t)hk * a.Tp + kb0) * PHD + (32 * w + 4 * vq) * 64 + 8 * vc;
#pragma unroll
  for (int j = 0; j < 4; j++) {
    T* d = vd + j * 64;
    if constexpr (BF) {
      bf16x8 o;
#pragma unroll
      for (int e = 0; e < 8; e++) o[e] = to_bf16(ve[e][j]);
      *(bf16x8*)d = o;
    } else {
      *(f32x4*)d = f32x4{ve[0][j], ve[1][j], ve[2][j], ve[3][j]};
      *(f32x4*)(d + 4) = f32x4{ve[4][j], ve[5][j], ve[6][j], ve[7][j]};
    }
  }
}

// ------------------------------------------------------------------ bf16 tiles
//
// A workgroup takes 32 NW virtual rows of one kv head (a wave 32 of them) and a part of their key blocks of 64: first the
// blocks that every row sees whole (the prefix's, then own ones before all of the tile's rows), then the prefix's last
// part and the own blocks that the rows' ranges cut.  Keys in any order give the same softmax, so both kinds are one loop each.
//
// Scores transposed, S^T = K Q^T: lane (r, hf) of a 32 x 32 product owns row r, and each of its maxima and sums is a register.  q and k
// are in f16, 11 bits (in bf16 they would be 0.005 of a result off: more than its own rounding), the weights and V in bf16.
// p = 2^(s - m) with an integer m that only rises (a power of two, so no rounding depends on when it rose): in blocks that
// are seen whole without looking, as long as the weights' sum stays below 2^8, from -m in the scores' accumulators.  No key's weight is
// above 2^8, so n of them with values below 2^119 / n have finite sums.  Where m rises, it rises to 2^24 times the largest weight, so that
// it seldom does again (7741 rows of 16 heads behind 4096 keys, scores of a standard deviation of 8: 318 us without that, 296 so).
// Blocks are copied by buffer_load ... lds three ahead into four stages of LDS, so a barrier a block is all that waves share.
// 7741 rows of 16 heads behind 4096 keys: 264 GFLOP in 267 us, 990 TFLOP/s; the matrix cores are busy 56 % of the cycles at the 1.7
// GHz that the power limit leaves (a library product of 8192 x 8192 x 8192: 1150).  64 rows of 32 heads behind 8192: 33.6 MB of keys
// in 19 us, a start of 2, eleven until the last block is there, and the sums' way out.

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) void prefix_lds_t;
constexpr float P_LIMIT = 256.0f, P_HEAD = 24.0f;
constexpr float M_NONE = -3e38f;                    // no key so far (below every score)
constexpr int PKT = 64 * PHD * 2;                   // bytes of a block's K; its V^T follows
constexpr int PST = 2 * PKT;                        // of a stage
constexpr int PNST = 4;

#define P_WAIT_VM(n) __builtin_amdgcn_s_waitcnt(((n) & 15) | (7 << 4) | (15 << 8) | (((n) >> 4) << 14))
#define P_SB() __builtin_amdgcn_sched_barrier(0)

__device__ __forceinline__ __amdgpu_buffer_rsrc_t p_rsrc(const void* p, int64_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc((void*)p, (short)0, (int)bytes, 0x00020000);
}
__device__ __forceinline__ void p_copy16(__amdgpu_buffer_rsrc_t rs, char* dst, uint32_t off, uint32_t base) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (prefix_lds_t*)dst, 16, off, base, 0, 0);
}
// of a value over the lane pair (l, l ^ 32)
__device__ __forceinline__ float p_pair_max(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float p_pair_sum(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// a value that is the same in all lanes, in a scalar register (quotients are formed in vector ones)
__device__ __forceinline__ int p_same(int x) { return __builtin_amdgcn_readfirstlane(x); }

// The key blocks of a tile: `full` whole ones (nP of the prefix, then own ones from of0), then the cut ones (the
// prefix's last, then own ones from ob0 up to of0 and from of1 up to ob1).
struct PrefixBlocks {
  int nP, of0, full, tail, ob0, cut0, of1, total;
  __device__ __forceinline__ PrefixBlocks(const PrefixArgs& a, int row0, int row1) {  // rows row0 .. row1
    const int2 r0 = a.range[row0], r1 = a.range[row1];
    const int s0 = p_same(r0.x), end = p_same(r1.y), hi = p_same(r0.x == r1.x ? r0.y : 0);  // own keys s0 .. end, s0 .. hi of them seen by all
    nP = a.P / PBK;
    tail = a.P % PBK ? 1 : 0;
    ob0 = s0 / PBK;
    const int ob1 = (end + PBK - 1) / PBK;
    of0 = (s0 + PBK - 1) / PBK;
    of1 = hi / PBK;
    if (of1 <= of0) of0 = of1 = ob0;
    full = nP + of1 - of0;
    cut0 = of0 - ob0;
    total = full + tail + cut0 + ob1 - of1;
  }
  // block i: its number, and whether it is of the prefix
  __device__ __forceinline__ int at(int i, bool& prefix) const {
    if (i < full) {
      prefix = i < nP;
      return prefix ? i : of0 + i - nP;
    }
    i -= full;
    prefix = i < tail;
    if (prefix) return nP;
    i -= tail;
    return i < cut0 ? ob0 + i : of1 + i - cut0;
  }
};

// A wave's rows v0 ... (o of lane (r, hf) is row r's, register 4 g + e of o[i] its dim 32 i + 8 g + 4 hf + e; m, l: exponent and
// this lane's sum of the weights), divided, or as a part of a split call.  They leave through LDS in halves of 64 columns, so that
// every store writes 256 bytes of a row.
__device__ __forceinline__ void p_leave(const PrefixArgs& a, char* smem, int sp, int hk, int v0, int wave, int lane, f32x16 (&o)[4], float m, float l) {
  const int r = lane & 31, hf = lane >> 5, v = v0 + r;
  l = p_pair_sum(l);
  const bool part = a.splits > 1;
  const float inv = part ? 1.0f : 1.0f / l;
  const int64_t plane = ((int64_t)sp * a.Hkv + hk) * a.V;
  if (part && v < a.V && hf == 0) *(float2*)(a.pml + (plane + v) * 2) = make_float2(m, l);
  constexpr int RS = 64 + 4;
  float* ow = (float*)smem + wave * 32 * RS;
  const int rr = lane >> 4, cc = 4 * (lane & 15);
#pragma unroll
  for (int half = 0; half < 2; half++) {
#pragma unroll
    for (int d2 = 0; d2 < 2; d2++)
#pragma unroll
      for (int g = 0; g < 4; g++) {
        const f32x16& w = o[2 * half + d2];
        *(f32x4*)(ow + r * RS + 32 * d2 + 8 * g + 4 * hf) = f32x4{w[4 * g] * inv, w[4 * g + 1] * inv, w[4 * g + 2] * inv, w[4 * g + 3] * inv};
      }
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int k = 0; k < 8; k++) {
      const int q = 4 * k + rr, vo = v0 + q;
      const f32x4 w = *(const f32x4*)(ow + q * RS + cc);
      if (vo < a.V) {
        if (part) {
          *(f32x4*)(a.po + (plane + vo) * PHD + 64 * half + cc) = w;
        } else {
          const int64_t ro = vo / a.group, off = ro * a.ldo + (hk * a.group + vo - ro * a.group) * PHD + 64 * half + cc;
          if (a.obf) *(bf16x4*)((bf16*)a.o + off) = bf16x4{to_bf16(w[0]), to_bf16(w[1]), to_bf16(w[2]), to_bf16(w[3])};
          else *(f32x4*)((float*)a.o + off) = w;
        }
      }
    }
    __builtin_amdgcn_wave_barrier();
  }
}

template <int NW>
__global__ __launch_bounds__(64 * NW, NW / 4) void prefix_flash_bf16(PrefixArgs a) {
  constexpr int CPW = 16 / NW;  // copies of K, and of V^T, a wave and block
  // (one LDS object: beside a second one the compiler has every read of the stages wait for all copies in flight)
  __shared__ __attribute__((aligned(1024))) char smem[PNST * PST];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, r = lane & 31, hf = lane >> 5;
  // tiles of a head and split follow each other (on one XCD: they read the same blocks)
  const int id = xcd_remap(blockIdx.x, gridDim.x), hs = p_same(id / a.nt), tile = id - hs * a.nt, hk = p_same(hs / a.splits),
            sp = hs - hk * a.splits;
  const int v0 = tile * 32 * NW, v = v0 + 32 * wave + r, vc = min(v, a.V - 1);
  f16x8 qf[8];
#pragma unroll
  for (int ks = 0; ks < 8; ks++) qf[ks] = *(const f16x8*)((const _Float16*)a.pq + ((int64_t)hk * a.V + vc) * PHD + 16 * ks + 8 * hf);
  const int2 range = a.range[vc / a.group];
  const PrefixBlocks B(a, p_same(v0 / a.group), p_same((min(v0 + 32 * NW, a.V) - 1) / a.group));
  const int each = p_same(B.total / a.splits), more = B.total - each * a.splits;  // (blocks of a part: each, and one more of the first)
  const int i0 = sp * each + min(sp, more), nb = each + (sp < more ? 1 : 0), i1 = i0 + nb;
  // own keys that a row of the wave sees (its rows ascend; none without rows)
  const int wlo = __builtin_amdgcn_readfirstlane(range.x), whi = __builtin_amdgcn_readlane(range.y, 31);
  const bool live = v0 + 32 * wave < a.V;

  const int64_t pb = (int64_t)a.Pp * PHD * 2, ob = (int64_t)a.Tp * PHD * 2;
  const __amdgpu_buffer_rsrc_t rpk = p_rsrc((const char*)a.pk + hk * pb, a.P ? pb : 0), rpv = p_rsrc((const char*)a.pvt + hk * pb, a.P ? pb : 0),
                               rok = p_rsrc((const char*)a.ok + hk * ob, ob), rov = p_rsrc((const char*)a.ovt + hk * ob, ob);
  uint32_t ko[CPW], vo[CPW];
#pragma unroll
  for (int c = 0; c < CPW; c++) {
    const int row = 4 * (wave * CPW + c) + (lane >> 4), d = 8 * (wave * CPW + c) + (lane >> 3);
    ko[c] = row * 256 + 16 * ((lane & 15) ^ (row & 15));
    vo[c] = d * 128 + 16 * ((lane & 7) ^ ((d >> 1) & 7));
  }
  const auto load = [&](int j) __attribute__((always_inline)) {  // block j of the part, if there is one
    if (j >= nb) return;
    bool pre;
    const int blk = B.at(i0 + j, pre);
    char* st = smem + (j & 3) * PST;
#pragma unroll
    for (int c = 0; c < CPW; c++) p_copy16(pre ? rpk : rok, st + (wave * CPW + c) * 1024, ko[c], blk * (64 * 256));
#pragma unroll
    for (int c = 0; c < CPW; c++) p_copy16(pre ? rpv : rov, st + PKT + (wave * CPW + c) * 1024, vo[c], blk * (64 * 256));
  };
  load(0);
  load(1);
  load(2);

  f32x16 o[4];
#pragma unroll
  for (int i = 0; i < 4; i++) o[i] = f32x16{};
  float m = M_NONE, l = 0.0f;
  int kof[8], vof[4];
#pragma unroll
  for (int ks = 0; ks < 8; ks++) kof[ks] = r * 256 + 16 * ((2 * ks + hf) ^ (r & 15));
#pragma unroll
  for (int j = 0; j < 4; j++) vof[j] = PKT + r * 128 + 16 * ((2 * j + hf) ^ ((r >> 1) & 7));
  const bf16x2 ones = {(bf16)1.0f, (bf16)1.0f};

  // sets p (eight weights) and adds their sum
  const auto weights = [&](const f32x16& s, int u, bf16x8& p, float& sum) __attribute__((always_inline)) {
#pragma unroll
    for (int e = 0; e < 8; e++) p[e] = to_bf16(__builtin_amdgcn_exp2f(s[8 * u + e]));
#pragma unroll
    for (int e = 0; e < 4; e++) sum = __builtin_amdgcn_fdot2_f32_bf16(bf16x2{p[2 * e], p[2 * e + 1]}, ones, sum, false);
  };
  // A block with its maximum looked at.  Keys k0 + ... outside [lo, hi) are masked.
  const auto block = [&](const char* st, auto masked, int k0, int lo, int hi) __attribute__((always_inline)) {
    f32x16 s[2];
#pragma unroll
    for (int t = 0; t < 2; t++) {
      s[t] = f32x16{};
#pragma unroll
      for (int ks = 0; ks < 8; ks++) {
        s[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(*(const f16x8*)(st + kof[ks] + t * 8192), qf[ks], s[t], 0, 0, 0);
      }
    }
    if constexpr (decltype(masked)::value) {
      if (__builtin_amdgcn_ballot_w64(lo > k0 || hi < k0 + PBK)) {
        const uint32_t at = k0 + 4 * hf - lo, n = hi - lo;  // (below lo: a large number)
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
          for (int e = 0; e < 16; e++)
            if (at + (32 * t + 8 * (e >> 2) + (e & 3)) >= n) s[t][e] = -INFINITY;
      }
    }
    float bm = fmaxf(s[0][0], s[1][0]);
#pragma unroll
    for (int e = 1; e < 16; e++) bm = fmaxf(bm, fmaxf(s[0][e], s[1][e]));
    const float top = ceilf(p_pair_max(bm));
    if (__builtin_amdgcn_ballot_w64(top > m)) {
      const float mn = top > m ? top + P_HEAD : m, f = __builtin_amdgcn_exp2f(m - mn);
      m = mn;
      l *= f;
#pragma unroll
      for (int i = 0; i < 4; i++) o[i] *= f;
    }
#pragma unroll
    for (int t = 0; t < 2; t++) {
      s[t] -= m;
#pragma unroll
      for (int u = 0; u < 2; u++) {
        bf16x8 p;
        weights(s[t], u, p, l);
#pragma unroll
        for (int i = 0; i < 4; i++) o[i] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(*(const bf16x8*)(st + vof[2 * t + u] + i * 4096), p, o[i], 0, 0, 0);
      }
    }
  };
  // A block that every row sees whole, after another: the written order is kept (each product's fragment was read four
  // reads before it, one half's exponentials run beside the next products).
  f32x16 negm;
  bf16x8 f[4];  // the block's first fragments; at its end the next one's (st: the block, nx: the next)
  const auto whole = [&](const char* st, const char* nx) __attribute__((always_inline)) {
    const auto frag = [&](int i) __attribute__((always_inline)) {
      return i < 16 ? *(const bf16x8*)(st + kof[i & 7] + (i >> 3) * 8192)
                    : *(const bf16x8*)(st + vof[(i - 16) >> 3 << 1 | (i & 1)] + (((i - 16) & 7) >> 1) * 4096);
    };
    f32x16 s[2];
    bf16x8 p[4];
    float la = 0.0f, lb = 0.0f;
    const auto prob2 = [&](int t, int k) __attribute__((always_inline)) {
      bf16x8& q = p[2 * t + (k >> 2)];
      q[2 * (k & 3)] = to_bf16(__builtin_amdgcn_exp2f(s[t][2 * k]));
      q[2 * (k & 3) + 1] = to_bf16(__builtin_amdgcn_exp2f(s[t][2 * k + 1]));
      float& acc = k & 1 ? lb : la;
      acc = __builtin_amdgcn_fdot2_f32_bf16(bf16x2{q[2 * (k & 3)], q[2 * (k & 3) + 1]}, ones, acc, false);
    };
    // the rare case of a sum above 2^8: m rises to the half's largest score
    const auto settle = [&](int t) __attribute__((always_inline)) {
      float sum = la + lb;
      if (__builtin_expect(__builtin_amdgcn_ballot_w64(!(sum <= P_LIMIT)) != 0, 0)) {
        float bm = s[t][0];
#pragma unroll
        for (int e = 1; e < 16; e++) bm = fmaxf(bm, s[t][e]);
        const float top = ceilf(p_pair_max(bm)), d = top > 0.0f ? top + P_HEAD : 0.0f, g = __builtin_amdgcn_exp2f(-d);
        m += d;
        negm -= d;
        l *= g;
#pragma unroll
        for (int i = 0; i < 4; i++) o[i] *= g;
#pragma unroll
        for (int u = t; u < 2; u++) s[u] -= d;
        la = lb = 0.0f;
#pragma unroll
        for (int k = 0; k < 8; k++) prob2(t, k);
        sum = la + lb;
      }
      l += sum;
      la = lb = 0.0f;
    };
#pragma unroll
    for (int i = 0; i < 16; i++) {
      f32x16& d = s[i >> 3];
      d = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, f[i & 3]), qf[i & 7], (i & 7) == 0 ? negm : d, 0, 0, 0);
      f[i & 3] = frag(i + 4);
      if (i >= 8) prob2(0, i - 8);
      P_SB();
    }
    settle(0);
    P_SB();
#pragma unroll
    for (int j = 0; j < 16; j++) {
      if (j == 8) {
        settle(1);
        P_SB();
      }
      o[(j & 7) >> 1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f[j & 3], p[j >> 3 << 1 | (j & 1)], o[(j & 7) >> 1], 0, 0, 0);
      f[j & 3] = j < 12 ? frag(j + 20) : *(const bf16x8*)(nx + kof[j - 12]);
      if (j < 8) prob2(1, j);
      P_SB();
    }
  };

  // Block j in stage j % 4.  At the top of its turn this wave's copies of block j + 1 have arrived (those of the block after it
  // may pend); behind the barrier everyone's have, so that its first fragments are read under block j's last products, and the
  // stage of block j - 1 is refilled.
  const auto turn = [&](int j) __attribute__((always_inline)) {
    if (j + 2 < nb) P_WAIT_VM(2 * CPW);
    else P_WAIT_VM(0);
    p_barrier();
    load(j + 3);
    return (const char*)smem + (j & 3) * PST;
  };
  const auto after = [&](int j) __attribute__((always_inline)) { return (const char*)smem + ((j + 1) & 3) * PST; };
  const int nf = max(min(B.full, i1) - i0, 0);
  int j = 0;
  if (nf > 0) {
    const char* st = turn(0);
    if (live) {
      block(st, std::false_type{}, 0, 0, 0);
#pragma unroll
      for (int i = 0; i < 4; i++) f[i] = *(const bf16x8*)(after(0) + kof[i]);
    }
    negm = f32x16{} - m;
    for (j = 1; j < nf; j++) {
      st = turn(j);
      if (live) whole(st, after(j));
    }
  }
  for (; j < nb; j++) {
    const char* st = turn(j);
    bool pre;
    const int blk = B.at(i0 + j, pre);
    if (live && (pre || (blk * PBK < whi && blk * PBK + PBK > wlo)))
      block(st, std::true_type{}, blk * PBK, pre ? 0 : range.x, pre ? a.P : range.y);
  }
  p_barrier();  // (the stages become the rows')

  p_leave(a, smem, sp, hk, v0 + 32 * wave, wave, lane, o, m, l);
}

// ------------------------------------------------------------------ fp32 tiles
//
// The same parts in fp32 precision.  A value is three bf16 ones, x = x1 + x2 + x3 exactly (8 bits each, cut off and not rounded: x2 is
// below 2^-7 of x and x3 below 2^-15), and a product six on the bf16 matrix cores, x1 y1 + x1 y2 + x2 y1 + x2 y2 + x1 y3 + x3 y1.  What
// is left out, x2 y3 + x3 y2 + x3 y3, has the product's sign and is below 2^-21 of it.
// A step is 32 keys.  They come as fp32 by buffer_load ... lds into one of two stages, a step ahead are cut into their planes (once
// for all waves, under the products of the step before), and a step later are multiplied: one barrier a step.
// p = 2^(s - m) with m raised where a step's maximum passes it by more than 8.  A step's products of V are added by themselves first:
// chains of one step a sum across steps.
// 1265 rows of 15 heads behind 1000 keys: 79 us (131 by the fp32 matrix cores), 1000 TFLOP/s of bf16 products with the tiles' unseen
// keys, the matrix cores busy 54 % of the cycles at 1.5 GHz; LDS is full (raw keys and planes, two stages each).
constexpr int FRAW = 2 * 32 * PHD * 4;   // bytes of a step's K, then V^T, as they come
constexpr int FPL = 32 * PHD * 2;        // of one plane of its K or V^T
constexpr int FST = 6 * FPL;             // of its planes: three of K, three of V^T
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// Two values' terms, packed: bf16 is the upper half of an fp32.
__device__ __forceinline__ void p_terms(float x, float y, uint32_t (&t)[3]) {
#pragma unroll
  for (int i = 0; i < 3; i++) {
    const uint32_t a = __float_as_uint(x), b = __float_as_uint(y);
    t[i] = __builtin_amdgcn_perm(b, a, 0x07060302);
    x -= __uint_as_float(a & 0xffff0000u);
    y -= __uint_as_float(b & 0xffff0000u);
  }
}
__device__ __forceinline__ void p_terms8(const float* x, bf16x8 (&t)[3]) {
  uint32_t w[4][3];
#pragma unroll
  for (int i = 0; i < 4; i++) p_terms(x[2 * i], x[2 * i + 1], w[i]);
#pragma unroll
  for (int c = 0; c < 3; c++) t[c] = __builtin_bit_cast(bf16x8, u32x4{w[0][c], w[1][c], w[2][c], w[3][c]});
}
// c + x y of six terms, the smallest first
__device__ __forceinline__ f32x16 p_mfma6(const bf16x8 (&x)[3], const bf16x8 (&y)[3], f32x16 c) {
  c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x[2], y[0], c, 0, 0, 0);
  c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x[0], y[2], c, 0, 0, 0);
  c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x[1], y[1], c, 0, 0, 0);
  c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x[1], y[0], c, 0, 0, 0);
  c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x[0], y[1], c, 0, 0, 0);
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(x[0], y[0], c, 0, 0, 0);
}

template <int NW>
__global__ __launch_bounds__(64 * NW, NW / 4) void prefix_flash_fp32(PrefixArgs a) {
  constexpr int CP = 16 / NW;  // pieces of 16 bytes of a step's K, and of its V^T, a thread
  __shared__ __attribute__((aligned(1024))) char smem[2 * FRAW + 2 * FST];
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, r = lane & 31, hf = lane >> 5;
  const int id = xcd_remap(blockIdx.x, gridDim.x), hs = p_same(id / a.nt), tile = id - hs * a.nt, hk = p_same(hs / a.splits),
            sp = hs - hk * a.splits;
  const int v0 = tile * 32 * NW, v = v0 + 32 * wave + r, vc = min(v, a.V - 1);
  float x[64];
#pragma unroll
  for (int g = 0; g < 16; g++) {
    const f32x4 w = *(const f32x4*)((const float*)a.pq + ((int64_t)hk * a.V + vc) * PHD + 16 * (g >> 1) + 8 * hf + 4 * (g & 1));
#pragma unroll
    for (int e = 0; e < 4; e++) x[4 * g + e] = w[e];
  }
  const int2 range = a.range[vc / a.group];
  const PrefixBlocks B(a, p_same(v0 / a.group), p_same((min(v0 + 32 * NW, a.V) - 1) / a.group));
  const int each = p_same(B.total / a.splits), more = B.total - each * a.splits;
  const int i0 = sp * each + min(sp, more), ns = 2 * (each + (sp < more ? 1 : 0));  // steps: halves of blocks
  const int wlo = __builtin_amdgcn_readfirstlane(range.x), whi = __builtin_amdgcn_readlane(range.y, 31);
  const bool live = v0 + 32 * wave < a.V;

  const int64_t pb = (int64_t)a.Pp * PHD * 4, ob = (int64_t)a.Tp * PHD * 4;
  const __amdgpu_buffer_rsrc_t rpk = p_rsrc((const char*)a.pk + hk * pb, a.P ? pb : 0), rpv = p_rsrc((const char*)a.pvt + hk * pb, a.P ? pb : 0),
                               rok = p_rsrc((const char*)a.ok + hk * ob, ob), rov = p_rsrc((const char*)a.ovt + hk * ob, ob);
  // piece u = 64 (wave CP + c) + lane: K row u / 32, V^T row u / 8 (its 32 keys are 128 bytes of 256)
  uint32_t vo[CP];
#pragma unroll
  for (int c = 0; c < CP; c++) {
    const int u = 64 * (wave * CP + c) + lane;
    vo[c] = (u >> 3) * 256 + (u & 7) * 16;
  }
  const auto load = [&](int j) __attribute__((always_inline)) {  // step j of the part, if there is one
    if (j >= ns) return;
    bool pre;
    const uint32_t blk = B.at(i0 + (j >> 1), pre), half = j & 1;
    char* st = smem + half * FRAW;
#pragma unroll
    for (int c = 0; c < CP; c++) p_copy16(pre ? rpk : rok, st + (wave * CP + c) * 1024, lane * 16, blk * 32768 + half * 16384 + (wave * CP + c) * 1024);
#pragma unroll
    for (int c = 0; c < CP; c++) p_copy16(pre ? rpv : rov, st + FRAW / 2 + (wave * CP + c) * 1024, vo[c], blk * 32768 + half * 128);
  };
  // this thread's own pieces of step j (those of its own wave's copies) into planes
  const auto cut = [&](int j) __attribute__((always_inline)) {
    const char* st = smem + (j & 1) * FRAW;
    char* pl = smem + 2 * FRAW + (j & 1) * FST;
#pragma unroll
    for (int c = 0; c < 2 * CP; c++) {
      const bool key = c < CP;
      const int u = 64 * (wave * CP + (key ? c : c - CP)) + lane;
      const f32x4 w = *(const f32x4*)(st + (key ? 0 : FRAW / 2) + u * 16);
      uint32_t t0[3], t1[3];
      p_terms(w[0], w[1], t0);
      p_terms(w[2], w[3], t1);
      // K: dims 4 (u % 32) .. of row u / 32.  V^T: keys 4 q .. of row u / 8, each 16 of them kept as 0-3, 8-11, 4-7, 12-15
      const int row = key ? u >> 5 : u >> 3, q = key ? u & 31 : u & 7;
      const int at = key ? row * 256 + 16 * ((q >> 1) ^ (row & 15)) + 8 * (q & 1)
                         : 3 * FPL + row * 64 + 16 * ((2 * (q >> 2) + (q & 1)) ^ ((row >> 1) & 3)) + 8 * ((q >> 1) & 1);
#pragma unroll
      for (int p = 0; p < 3; p++) *(u32x2*)(pl + at + p * FPL) = u32x2{t0[p], t1[p]};
    }
  };
  load(0);
  load(1);
  bf16x8 qf[8][3];
#pragma unroll
  for (int ks = 0; ks < 8; ks++) p_terms8(x + 8 * ks, qf[ks]);
  f32x16 o[4];
#pragma unroll
  for (int i = 0; i < 4; i++) o[i] = f32x16{};
  float m = M_NONE, l = 0.0f;
  int kof[8], vof[2];
#pragma unroll
  for (int ks = 0; ks < 8; ks++) kof[ks] = r * 256 + 16 * ((2 * ks + hf) ^ (r & 15));
#pragma unroll
  for (int u = 0; u < 2; u++) vof[u] = 3 * FPL + r * 64 + 16 * ((2 * u + hf) ^ ((r >> 1) & 3));
  if (ns > 0) {
    if (ns > 1) P_WAIT_VM(2 * CP);
    else P_WAIT_VM(0);
    cut(0);
  }
  for (int j = 0; j < ns; j++) {
    // This wave's copies of step j + 1 have arrived and its planes of step j are written; behind the barrier everyone's are, and the
    // planes of step j - 1 and this wave's copies of step j are done with.
    P_WAIT_VM(0);
    __builtin_amdgcn_s_waitcnt(0xc07f);
    p_barrier();
    load(j + 2);
    bool pre;
    const int blk = B.at(i0 + (j >> 1), pre), k0 = blk * PBK + 32 * (j & 1);
    const bool cutting = j + 1 < ns;
    if (!live || (i0 + (j >> 1) >= B.full && !pre && (k0 >= whi || k0 + 32 <= wlo))) {
      if (cutting) cut(j + 1);
      continue;
    }
    const char* st = smem + 2 * FRAW + (j & 1) * FST;
    f32x16 s = {};
#pragma unroll
    for (int ks = 0; ks < 8; ks++) {
      bf16x8 kf[3];
#pragma unroll
      for (int p = 0; p < 3; p++) kf[p] = *(const bf16x8*)(st + kof[ks] + p * FPL);
      s = p_mfma6(kf, qf[ks], s);
    }
    if (cutting) cut(j + 1);
    if (i0 + (j >> 1) >= B.full) {
      const int lo = pre ? 0 : range.x, hi = pre ? a.P : range.y;
      if (__builtin_amdgcn_ballot_w64(lo > k0 || hi < k0 + 32)) {
        const uint32_t at = k0 + 4 * hf - lo, n = hi - lo;
#pragma unroll
        for (int e = 0; e < 16; e++)
          if (at + (8 * (e >> 2) + (e & 3)) >= n) s[e] = -INFINITY;
      }
    }
    float bm = s[0];
#pragma unroll
    for (int e = 1; e < 16; e++) bm = fmaxf(bm, s[e]);
    bm = p_pair_max(bm);
    const bool need = bm > m + 8.0f;
    if (__builtin_amdgcn_ballot_w64(need)) {
      const float mn = need ? ceilf(bm) : m, f = __builtin_amdgcn_exp2f(m - mn);
      m = mn;
      l *= f;
#pragma unroll
      for (int i = 0; i < 4; i++) o[i] *= f;
    }
    float w[16], bl = 0.0f;
#pragma unroll
    for (int e = 0; e < 16; e++) {
      w[e] = __builtin_amdgcn_exp2f(s[e] - m);
      bl += w[e];
    }
    l += bl;
    bf16x8 pf[2][3];
#pragma unroll
    for (int u = 0; u < 2; u++) p_terms8(w + 8 * u, pf[u]);
#pragma unroll
    for (int dt = 0; dt < 4; dt++) {
      f32x16 sum = {};
#pragma unroll
      for (int u = 0; u < 2; u++) {
        bf16x8 vf[3];
#pragma unroll
        for (int p = 0; p < 3; p++) vf[p] = *(const bf16x8*)(st + vof[u] + dt * 2048 + p * FPL);
        sum = p_mfma6(vf, pf[u], sum);
      }
      o[dt] += sum;
    }
  }
  p_barrier();  // (the planes become the rows')
  p_leave(a, smem, sp, hk, v0 + 32 * wave, wave, lane, o, m, l);
}

// The parts of a split call, a half wave per virtual row: o = sum 2^(m_s - m) o_s / sum 2^(m_s - m) l_s, eight parts asked for
// at a time.  Bound by the parts' bytes (1265 rows of 15 heads in three parts: 39 MB, 8.6 us), few rows by a launch (2.5 us).
__global__ __launch_bounds__(256) void prefix_join_kernel(PrefixArgs a) {
  const int64_t i = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5), n = (int64_t)a.Hkv * a.V;
  if (i >= n) return;
  const int d = 4 * (threadIdx.x & 31);
  float m = M_NONE, l = 0.0f;
  f32x4 o = {};
  for (int s0 = 0; s0 < a.splits; s0 += 8) {
    float2 ml[8];
    f32x4 w[8];
#pragma unroll
    for (int u = 0; u < 8; u++) {
      const int64_t p = min(s0 + u, a.splits - 1) * n + i;
      ml[u] = *(const float2*)(a.pml + p * 2);
      w[u] = *(const f32x4*)(a.po + p * PHD + d);
    }
    float mn = m;
#pragma unroll
    for (int u = 0; u < 8; u++) mn = fmaxf(mn, ml[u].x);
    const float g = __builtin_amdgcn_exp2f(m - mn);
    l *= g;
    o *= g;
    m = mn;
#pragma unroll
    for (int u = 0; u < 8; u++) {
      const float f = s0 + u < a.splits ? __builtin_amdgcn_exp2f(ml[u].x - m) : 0.0f;
      l += f * ml[u].y;
      if (f != 0.0f) o += f * w[u];
    }
  }
  o *= 1.0f / l;
  const int hk = (int)(i / a.V), v = (int)(i - (int64_t)hk * a.V);
  const int64_t row = v / a.group, off = row * a.ldo + (hk * a.group + v - row * a.group) * PHD + d;
  if (a.obf) *(bf16x4*)((bf16*)a.o + off) = bf16x4{to_bf16(o[0]), to_bf16(o[1]), to_bf16(o[2]), to_bf16(o[3])};
  else *(f32x4*)((float*)a.o + off) = o;
}

// ------------------------------------------------------------------ host

template <class T>
static int prefix_prep_launch(anima_ctx* c, const PrefixArgs& a) {
  Launch L(c, sizeof(T) == 2 ? "attn.prefix_prep_bf16" : "attn.prefix_prep_fp32", 0.0, (double)a.T * PHD * (a.Hkv * (8.0 + 2 * sizeof(T)) + (a.pq ? a.H * (4.0 + sizeof(T)) : 0.0)));
  hipLaunchKernelGGL(prefix_prep_kernel<T>, dim3((unsigned)(a.Tp / 64), (unsigned)(a.Hkv + (a.pq ? a.H : 0))), dim3(256), 0, c->stream, a);
  return L.end();
}

// The sequences of one launch, which the arguments describe: their keys and values into the workspace, then the rows.
template <class T>
static int prefix_part(anima_ctx* c, PrefixArgs& a, int longest) {
  constexpr bool BF = sizeof(T) == 2;
  a.V = a.T * a.group;
  const PrefixPlan plan = prefix_plan(c->num_cus, BF, a.V, a.group, a.Hkv, a.T, a.P, longest);
  const bool eight = plan.waves == 8;
  a.nt = plan.nt;
  a.splits = plan.splits;
  const size_t plane = (size_t)a.Hkv * a.Tp * PHD * sizeof(T), q = (size_t)a.Hkv * a.V * PHD * sizeof(T),
               n = a.splits > 1 ? (size_t)a.splits * a.Hkv * a.V : 0;
  void* ws = nullptr;
  if (int rc = workspace(c, 2 * plane + q + n * (PHD + 2) * 4 + (size_t)a.T * 8, &ws)) return rc;
  a.ok = ws;
  a.ovt = (char*)ws + plane;
  a.pq = (char*)ws + 2 * plane;
  a.po = (float*)((char*)a.pq + q);
  a.pml = a.po + n * PHD;
  a.range = (int2*)(a.pml + 2 * n);
  if (int rc = prefix_prep_launch<T>(c, a)) return rc;
  Launch L(c, BF ? "attn.prefix_bf16" : "attn.prefix_fp32", 4.0 * a.T * a.H * PHD * a.P, 0.0);
  const dim3 grid((unsigned)((int64_t)a.nt * a.Hkv * a.splits));
  if (!BF && eight) hipLaunchKernelGGL(prefix_flash_fp32<8>, grid, dim3(512), 0, c->stream, a);
  else if (!BF) hipLaunchKernelGGL(prefix_flash_fp32<4>, grid, dim3(256), 0, c->stream, a);
  else if (eight) hipLaunchKernelGGL(prefix_flash_bf16<8>, grid, dim3(512), 0, c->stream, a);
  else hipLaunchKernelGGL(prefix_flash_bf16<4>, grid, dim3(256), 0, c->stream, a);
  if (a.splits > 1)
    hipLaunchKernelGGL(prefix_join_kernel, dim3((unsigned)(((int64_t)a.Hkv * a.V + 7) / 8)), dim3(256), 0, c->stream, a);
  return L.end();
}

int attention_prefix_prepare_launch(anima_ctx* c, const anima_prefix_attn_desc* d, void* out, int64_t bytes) {
  char msg[256];
  if (int rc = check_attention_prefix_prepare(d, out, bytes, PrefixMsg{msg, sizeof msg})) return fail(c, rc, "%s", msg);
  OnDevice on(c);
  const bool bf = d->precision == ANIMA_PREC_BF16;
  PrefixArgs a{};
  a.group = d->group == 0 ? 1 : d->group;
  a.H = d->H;
  a.Hkv = d->H / a.group;
  a.T = d->len[0];
  a.Tp = (a.T + PBK - 1) / PBK * PBK;
  a.k = d->k + d->k_off;
  a.ldk = d->ldk;
  a.v = d->v + d->v_off;
  a.ldv = d->ldv;
  a.kn = d->k_norm;
  a.cs = d->rope_cs;
  a.sin_off = d->rope_sin_off;
  a.eps = d->eps;
  a.ok = out;
  a.ovt = (char*)out + bytes / 2;
  a.seq.n = 1;
  a.seq.start[1] = a.T;
  return bf ? prefix_prep_launch<bf16>(c, a) : prefix_prep_launch<float>(c, a);
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
    // the next sequences, as many as one launch describes, 2^22 keys and 2^30 rows of all heads hold
    a.seq.n = 0;
    int64_t t = 0;
    while (b < d->B && a.seq.n < PSEQ && t + d->len[b] <= PREFIX_MAX_KEYS && (t + d->len[b]) * d->H <= PREFIX_MAX_VROWS) {
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
    if (int rc = bf ? prefix_part<bf16>(c, a, longest) : prefix_part<float>(c, a, longest)) return rc;
    row += t;
  }
  return ANIMA_OK;
}

}  // namespace anima
