// Causal grouped-query attention over the 8-bit key / value cache, and the
// attention weight each slot receives.
//
//   s = scale q.k,  out = softmax(s) v,  lse = log sum exp(s)
//   weights[j] += sum over the new tokens and the heads of the group of
//                 exp(s_j - lse)     (slots of the new tokens start from 0)
//
// Tensor cores in fp32 accuracy.  An int8 value is exact in fp16, so only the
// other operand of each product is split: q (scaled by a power of two to
// magnitude 1..2 a row) and p (at most 1) into fp16 hi + lo, 22 bits in all,
// each product twice.  The scale of a 16-key tile (a block has at least 16
// keys) multiplies its scores, and its share of p: p v_scale / v_ref, v_ref
// the largest scale of the tiles in hand, keeps p within fp16's range.  The
// tail (fp32 rows) is split the same way on both sides: three products.
// Scores, sums and outputs are fp32; the products of a few tiles are summed
// by the tensor core, whose additions round towards zero, and then added to
// the running output in fp32.
#include <cooperative_groups.h>
#include <cuda_fp16.h>

#include "spx_internal.cuh"

namespace spx {
namespace {

namespace cg = cooperative_groups;

__device__ __forceinline__ int clamp_len(int v, int hi) { return v < 0 ? 0 : v > hi ? hi : v; }

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

struct AttnArgs {
  const float* q;
  spx_kv8_cache c;
  const int32_t* new_lens;
  int T, Hq;
  float scale;
  float* out;
  float* lse;
  float* weights;
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transposed8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ uint32_t as_u32(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }

// (x, y) as packed fp16 hi and lo parts.
__device__ __forceinline__ void split2(float x, float y, uint32_t& hi, uint32_t& lo) {
  const __half2 h = __floats2half2_rn(x, y);
  const float2 f = __half22float2(h);
  hi = as_u32(h);
  lo = as_u32(__floats2half2_rn(x - f.x, y - f.y));
}

// Two bytes (already flipped by 0x80: value + 128) to fp16: 0x6400 | u is
// 1024 + u, less 1152.
__device__ __forceinline__ uint32_t two_halves(uint32_t w, uint32_t sel) {
  uint32_t r = __byte_perm(w, 0x64646464u, sel);
  const __half2 v = __hsub2(*reinterpret_cast<__half2*>(&r),
                            __half2half2(__ushort_as_half((unsigned short)0x6480)));
  return as_u32(v);
}

// 2^-e and 2^e for a largest magnitude with these bits (finite).
__device__ __forceinline__ void pow2_scale(uint32_t amax_bits, float& down, float& up) {
  int e = (int)(amax_bits >> 23);
  e = e < 1 ? 1 : e > 253 ? 253 : e;
  down = __uint_as_float((uint32_t)(254 - e) << 23);
  up = __uint_as_float((uint32_t)e << 23);
}
__device__ __forceinline__ uint32_t finite_abs(float x) {
  const uint32_t b = __float_as_uint(x) & 0x7fffffffu;
  return b >= 0x7f800000u ? 0u : b;
}

// ---------------------------------------------------------------------------
// Few rows (decode, drafts).  A row is a (new token, head of the group) pair.
// Scores are held transposed, S^T = K Q^T: 16 keys are the M side of
// mma.m16n8k16 and 8 rows the N side, so that no lane is padding for a group
// of 8 heads.  Within a dot product the order of d is free: lane (g, t) reads
// 16 contiguous bytes of key row g and lets them be its four k-steps, straight
// from global memory in fragment order.  The output is held transposed too,
// O^T = V^T P^T: the lane's V bytes of four keys are interleaved into fp16
// pairs of keys, and the 8 x 8 blocks of P come from the scores' layout to the
// B operand's by movmatrix.  Each warp walks its own 16-key tiles with its own
// running maximum and sum; warps are joined in shared memory and the CTAs of a
// cluster, over which one sequence's keys are spread, through distributed
// shared memory: one launch, no workspace.
//
// What bounds it: the cache's bytes, 2 D + 8 / block a key and head; 16
// products of 4096 operations for 16 keys of D = 64 are a third of the tensor
// pipe's rate at full bandwidth.
template <int D>
struct Frag {                   // one 16-key tile of int8 K and V in registers
  uint4 k[2][D / 64];           // key rows g, g + 8
  uint32_t v[4][D / 32];        // keys 2t, 2t+1, 2t+8, 2t+9; d = D/8 g ...
  float ks, vs;
};

template <int NW>
__device__ __forceinline__ void load_words(uint32_t (&w)[NW], const void* p) {
  if constexpr (NW == 2) {
    const uint2 x = __ldg(reinterpret_cast<const uint2*>(p));
    w[0] = x.x;
    w[1] = x.y;
  } else {
    const uint4 x = __ldg(reinterpret_cast<const uint4*>(p));
    w[0] = x.x;
    w[1] = x.y;
    w[2] = x.z;
    w[3] = x.w;
  }
}

template <int D>
struct Keys {
  const int8_t* k8;
  const int8_t* v8;
  const float* ks;
  const float* vs;
  const float* kt;
  const float* vt;
  int shift;      // log2(block)
  __device__ __forceinline__ void load_k(Frag<D>& f, int tile, int g, int t) const {
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
      for (int h = 0; h < D / 64; ++h)
        f.k[r][h] = __ldg(reinterpret_cast<const uint4*>(
            k8 + ((int64_t)tile * 16 + g + 8 * r) * D + 64 * h + 16 * t));
    f.ks = __ldg(ks + ((tile * 16) >> shift));
  }
  __device__ __forceinline__ void load_v(Frag<D>& f, int tile, int g, int t) const {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      load_words(f.v[i], v8 + ((int64_t)tile * 16 + 2 * t + (i & 1) + 8 * (i >> 1)) * D + D / 8 * g);
    f.vs = __ldg(vs + ((tile * 16) >> shift));
  }
};

// Q of 8 rows as B fragments, hi and lo: [k-step][hi b0, b1, lo b0, b1], and
// for the lane's two columns (rows 2t, 2t + 1) the factor that takes a product
// to a score in units of log 2.
template <int D>
__device__ __forceinline__ void load_q(uint32_t (&qf)[D / 16][4], float (&qs)[2], const float* row,
                                       float scale, int t) {
  float x[D / 64][16];
  uint32_t mx = 0;
#pragma unroll
  for (int h = 0; h < D / 64; ++h)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float4 v = row ? __ldg(reinterpret_cast<const float4*>(row + 64 * h + 16 * t) + i)
                           : make_float4(0.f, 0.f, 0.f, 0.f);
      x[h][4 * i] = v.x;
      x[h][4 * i + 1] = v.y;
      x[h][4 * i + 2] = v.z;
      x[h][4 * i + 3] = v.w;
#pragma unroll
      for (int e = 0; e < 4; ++e) mx = max(mx, finite_abs(x[h][4 * i + e]));
    }
  mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
  mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
  float down, up;
  pow2_scale(mx, down, up);
#pragma unroll
  for (int h = 0; h < D / 64; ++h)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t* f = qf[4 * h + i];
      split2(x[h][4 * i] * down, x[h][4 * i + 1] * down, f[0], f[2]);
      split2(x[h][4 * i + 2] * down, x[h][4 * i + 3] * down, f[1], f[3]);
    }
  const float s = up * (scale * kLog2e);
  qs[0] = __shfl_sync(0xffffffffu, s, t * 8);
  qs[1] = __shfl_sync(0xffffffffu, s, t * 8 + 4);
}

// c += K Q^T of one int8 tile.
template <int D, int NT>
__device__ __forceinline__ void scores(float (&c)[NT][4], const Frag<D>& f,
                                       const uint32_t (&qf)[NT][D / 16][4]) {
#pragma unroll
  for (int h = 0; h < D / 64; ++h) {
    const uint32_t* r0 = reinterpret_cast<const uint32_t*>(&f.k[0][h]);
    const uint32_t* r1 = reinterpret_cast<const uint32_t*>(&f.k[1][h]);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t w0 = r0[i] ^ 0x80808080u, w1 = r1[i] ^ 0x80808080u;
      const uint32_t a[4] = {two_halves(w0, 0x4140), two_halves(w1, 0x4140),
                             two_halves(w0, 0x4342), two_halves(w1, 0x4342)};
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        mma16816(c[n], a, qf[n][4 * h + i][0], qf[n][4 * h + i][1]);
        mma16816(c[n], a, qf[n][4 * h + i][2], qf[n][4 * h + i][3]);
      }
    }
  }
}

// The running softmax of one warp: lane (g, t) holds rows (columns) 2t, 2t+1
// of each 8 and, of the output, d = D/8 g .. D/8 (g + 1) - 1.
template <int D, int NT>
struct Running {
  float m[NT][2], l[NT][2], o[NT][D / 16][4];
  __device__ __forceinline__ void init() {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        m[n][e] = -INFINITY;
        l[n][e] = 0.0f;
      }
#pragma unroll
      for (int i = 0; i < D / 16; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[n][i][e] = 0.0f;
    }
  }
  // New maxima for tile scores (log2 units); c becomes exp2(c - m), the sums
  // take them, and `corr` is what the outputs so far have to be scaled by.
  template <int KT>
  __device__ __forceinline__ void weigh(float (&c)[KT][NT][4], float (&corr)[NT][2]) {
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float mt = -INFINITY;
#pragma unroll
        for (int k = 0; k < KT; ++k) mt = fmaxf(mt, fmaxf(c[k][n][e], c[k][n][e + 2]));
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, x));
        const float mn = fmaxf(m[n][e], mt), base = mn == -INFINITY ? 0.0f : mn;
        corr[n][e] = ex2(m[n][e] - base);
        m[n][e] = mn;
        float sum = 0.0f;
#pragma unroll
        for (int k = 0; k < KT; ++k) {
          c[k][n][e] = ex2(c[k][n][e] - base);
          c[k][n][e + 2] = ex2(c[k][n][e + 2] - base);
          sum += c[k][n][e] + c[k][n][e + 2];
        }
        l[n][e] = fmaf(l[n][e], corr[n][e], sum);
      }
  }
};

// P (rows of 16 keys, already scaled) as B fragments: hi b0, b1, lo b0, b1.
__device__ __forceinline__ void p_frags(uint32_t (&pf)[4], const float (&p)[4]) {
  uint32_t h0, l0, h1, l1;
  split2(p[0], p[1], h0, l0);
  split2(p[2], p[3], h1, l1);
  pf[0] = transposed8x8(h0);
  pf[1] = transposed8x8(h1);
  pf[2] = transposed8x8(l0);
  pf[3] = transposed8x8(l1);
}

// One 16-key tile of the tail: fp32 rows, both operands split.
template <int D, int NT>
__device__ __forceinline__ void tail_tile(Running<D, NT>& run, const Keys<D>& kv,
                                          const uint32_t (&qf)[NT][D / 16][4],
                                          const float (&qs)[NT][2], const int (&last)[NT][2],
                                          int jb, int total, int g, int t) {
  const int blk_mask = (1 << kv.shift) - 1;
  // K rows g and g + 8
  float up_k, down;
  float c[1][NT][4] = {};
  {
    float x[2][D / 64][16];
    uint32_t mx = 0;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int j = jb + g + 8 * r;
      const float* row = kv.kt + (int64_t)(j & blk_mask) * D + 16 * t;
#pragma unroll
      for (int h = 0; h < D / 64; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float4 v = j < total ? *(reinterpret_cast<const float4*>(row + 64 * h) + i)
                                     : make_float4(0.f, 0.f, 0.f, 0.f);
          x[r][h][4 * i] = v.x;
          x[r][h][4 * i + 1] = v.y;
          x[r][h][4 * i + 2] = v.z;
          x[r][h][4 * i + 3] = v.w;
#pragma unroll
          for (int e = 0; e < 4; ++e) mx = max(mx, finite_abs(x[r][h][4 * i + e]));
        }
    }
    pow2_scale(__reduce_max_sync(0xffffffffu, mx), down, up_k);
#pragma unroll
    for (int h = 0; h < D / 64; ++h)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t a[4], al[4];
        split2(x[0][h][4 * i] * down, x[0][h][4 * i + 1] * down, a[0], al[0]);
        split2(x[1][h][4 * i] * down, x[1][h][4 * i + 1] * down, a[1], al[1]);
        split2(x[0][h][4 * i + 2] * down, x[0][h][4 * i + 3] * down, a[2], al[2]);
        split2(x[1][h][4 * i + 2] * down, x[1][h][4 * i + 3] * down, a[3], al[3]);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const uint32_t* q = qf[n][4 * h + i];
          mma16816(c[0][n], al, q[0], q[1]);
          mma16816(c[0][n], a, q[2], q[3]);
          mma16816(c[0][n], a, q[0], q[1]);
        }
      }
  }
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e)
      c[0][n][e] = jb + g + 8 * (e >> 1) <= last[n][e & 1] ? c[0][n][e] * (up_k * qs[n][e & 1])
                                                           : -INFINITY;
  float corr[NT][2];
  run.weigh(c, corr);
  // V rows 2t, 2t+1, 2t+8, 2t+9
  float y[4][D / 8];
  uint32_t mx = 0;
  uint32_t bad[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int j = jb + 2 * t + (i & 1) + 8 * (i >> 1);
    const float* row = kv.vt + (int64_t)(j & blk_mask) * D + D / 8 * g;
    bool odd = false;
#pragma unroll
    for (int e = 0; e < D / 32; ++e) {
      const float4 v = j < total ? *(reinterpret_cast<const float4*>(row) + e)
                                 : make_float4(0.f, 0.f, 0.f, 0.f);
      y[i][4 * e] = v.x;
      y[i][4 * e + 1] = v.y;
      y[i][4 * e + 2] = v.z;
      y[i][4 * e + 3] = v.w;
#pragma unroll
      for (int f = 0; f < 4; ++f) {
        // A NaN or infinity would reach rows that do not see this key: it
        // goes into the key's weight instead, where the mask stops it.
        float& z = y[i][4 * e + f];
        if ((__float_as_uint(z) & 0x7f800000u) == 0x7f800000u) {
          odd = true;
          z = 0.0f;
        }
        mx = max(mx, __float_as_uint(z) & 0x7fffffffu);
      }
    }
    bad[i] = __ballot_sync(0xffffffffu, odd);
  }
  float up_v;
  pow2_scale(__reduce_max_sync(0xffffffffu, mx), down, up_v);
  const uint32_t mine = 0x11111111u << (g >> 1);   // lanes with key g's (g + 8's) V
  const bool bad0 = (g & 1 ? bad[1] : bad[0]) & mine, bad1 = (g & 1 ? bad[3] : bad[2]) & mine;
#pragma unroll
  for (int n = 0; n < NT; ++n) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if ((e < 2 ? bad0 : bad1) && jb + g + 8 * (e >> 1) <= last[n][e & 1])
        c[0][n][e] = __int_as_float(0x7fc00000);
    uint32_t pf[4];
    p_frags(pf, c[0][n]);
#pragma unroll
    for (int i = 0; i < D / 16; ++i) {
      uint32_t a[4], al[4];
      split2(y[0][2 * i] * down, y[1][2 * i] * down, a[0], al[0]);
      split2(y[0][2 * i + 1] * down, y[1][2 * i + 1] * down, a[1], al[1]);
      split2(y[2][2 * i] * down, y[3][2 * i] * down, a[2], al[2]);
      split2(y[2][2 * i + 1] * down, y[3][2 * i + 1] * down, a[3], al[3]);
      float o[4] = {};
      mma16816(o, al, pf[0], pf[1]);
      mma16816(o, a, pf[2], pf[3]);
      mma16816(o, a, pf[0], pf[1]);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        run.o[n][i][e] = fmaf(run.o[n][i][e], corr[n][e & 1], up_v * o[e]);
    }
  }
}

constexpr int kFewMaxWarps = 8;

template <int D, int NT>
__global__ void __launch_bounds__(kFewMaxWarps * 32, 1)
    attention_kv8_few_kernel(const AttnArgs a, int groups, int cluster) {
  constexpr int KT = D == 64 ? 4 : 2;   // tiles in flight: 64 registers of K and V
  constexpr int R = 8 * NT;
  extern __shared__ __align__(16) float smem[];
  const int W = blockDim.x >> 5;
  float* part_m = smem;                 // [W][R]
  float* part_l = part_m + W * R;       // [W][R]
  float* cta_m = part_l + W * R;        // [R]
  float* cta_l = cta_m + R;             // [R]
  float* part_o = cta_l + R;            // [W][R][D]; the CTA's own sum goes to warp 0's
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int rank = blockIdx.x % cluster;
  const int unit = blockIdx.x / cluster, grp = unit % groups, h = unit / groups, b = blockIdx.y;
  const int S = a.c.max_seq, Hkv = a.c.kv_heads, G = a.Hq / Hkv;
  const int n_new = a.new_lens ? clamp_len(a.new_lens[b], a.T) : a.T;
  const int rows = n_new * G, r0 = grp * R;
  if (r0 >= rows) return;               // the whole cluster
  const int len = clamp_len(a.c.lens[b], S), total = min(len + n_new, S);
  const int shift = 31 - __clz(a.c.block);
  const int closed = total >> shift << shift;
  const int t_first = r0 / G, t_last = min(r0 + R, rows) - 1;   // rows; tokens below
  const int lim = min(len + t_last / G + 1, S);                 // slots that some row sees
  const int64_t bh = (int64_t)b * Hkv + h;
  Keys<D> kv;
  kv.k8 = a.c.k + bh * S * D;
  kv.v8 = a.c.v + bh * S * D;
  kv.ks = a.c.k_scale + bh * (S >> shift);
  kv.vs = a.c.v_scale + bh * (S >> shift);
  kv.kt = a.c.k_tail + bh * ((int64_t)D << shift);
  kv.vt = a.c.v_tail + bh * ((int64_t)D << shift);
  kv.shift = shift;

  uint32_t qf[NT][D / 16][4];
  float qs[NT][2];
  int last[NT][2];                      // the last slot that a column sees
  auto row_at = [&](int r) {            // [token][head] row of the group's row r
    return ((int64_t)b * a.T + r / G) * a.Hq + h * G + r % G;
  };
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int r = r0 + 8 * n + g;
    load_q<D>(qf[n], qs[n], r < rows ? a.q + row_at(r) * D : nullptr, a.scale, t);
#pragma unroll
    for (int e = 0; e < 2; ++e)
      last[n][e] = min(len + min(r0 + 8 * n + 2 * t + e, rows - 1) / G, total - 1);
  }
  Running<D, NT> run;
  run.init();

  const int tiles = (min(closed, lim) + 15) >> 4;
  const int first = (rank * W + warp) * KT, step = cluster * W * KT;
  Frag<D> f[KT];
  auto load_k = [&](int base) {
#pragma unroll
    for (int k = 0; k < KT; ++k) kv.load_k(f[k], min(base + k, tiles - 1), g, t);
  };
  auto load_v = [&](int base) {
#pragma unroll
    for (int k = 0; k < KT; ++k) kv.load_v(f[k], min(base + k, tiles - 1), g, t);
  };
  if (first < tiles) {
    load_k(first);
    load_v(first);
  }
  for (int base = first; base < tiles; base += step) {
    float c[KT][NT][4];
    // every key of these tiles is seen by every row of the group
    const bool all = (base + KT) * 16 <= len + t_first / G + 1 && base + KT <= tiles;
#pragma unroll
    for (int k = 0; k < KT; ++k) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) c[k][n][e] = 0.0f;
      scores<D, NT>(c[k], f[k], qf);
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) c[k][n][e] *= f[k].ks * qs[n][e & 1];
      if (!all) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (base + k >= tiles || (base + k) * 16 + g + 8 * (e >> 1) > last[n][e & 1])
              c[k][n][e] = -INFINITY;
      }
    }
    const bool more = base + step < tiles;
    if (more) load_k(base + step);
    // Rows that do not see a key have to weigh it 0 whatever its scale is.
    uint32_t hidden = 0;
    if (!all) {
#pragma unroll
      for (int k = 0; k < KT; ++k)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            hidden |= (c[k][n][e] == -INFINITY ? 1u : 0u) << ((k * NT + n) * 4 + e);
    }
    float corr[NT][2];
    run.weigh(c, corr);
    float ref = 0.0f;
#pragma unroll
    for (int k = 0; k < KT; ++k)
      if (f[k].vs <= 3.4028234663852886e38f) ref = fmaxf(ref, f[k].vs);
    const float inv = ref > 0.0f ? 1.0f / ref : 0.0f;
    float o[NT][D / 16][4];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < D / 16; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[n][i][e] = 0.0f;
#pragma unroll
    for (int k = 0; k < KT; ++k) {
      const float share = f[k].vs * inv;
      uint32_t pf[NT][4];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          c[k][n][e] = hidden >> ((k * NT + n) * 4 + e) & 1u ? 0.0f : c[k][n][e] * share;
        p_frags(pf[n], c[k][n]);
      }
#pragma unroll
      for (int w = 0; w < D / 32; ++w) {
        const uint32_t v0 = f[k].v[0][w] ^ 0x80808080u, v1 = f[k].v[1][w] ^ 0x80808080u;
        const uint32_t v2 = f[k].v[2][w] ^ 0x80808080u, v3 = f[k].v[3][w] ^ 0x80808080u;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t x = __byte_perm(v0, v1, i ? 0x7362 : 0x5140);
          const uint32_t y = __byte_perm(v2, v3, i ? 0x7362 : 0x5140);
          const uint32_t av[4] = {two_halves(x, 0x4140), two_halves(x, 0x4342),
                                  two_halves(y, 0x4140), two_halves(y, 0x4342)};
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            mma16816(o[n][2 * w + i], av, pf[n][0], pf[n][1]);
            mma16816(o[n][2 * w + i], av, pf[n][2], pf[n][3]);
          }
        }
      }
    }
    if (more) load_v(base + step);
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < D / 16; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          run.o[n][i][e] = fmaf(run.o[n][i][e], corr[n][e & 1], ref * o[n][i][e]);
  }
  for (int i = rank * W + warp; closed + 16 * i < lim; i += cluster * W)
    tail_tile<D, NT>(run, kv, qf, qs, last, closed + 16 * i, total, g, t);

  // Join the warps, then the CTAs of the cluster.
#pragma unroll
  for (int n = 0; n < NT; ++n) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float l = run.l[n][e];
#pragma unroll
      for (int x = 4; x < 32; x <<= 1) l += __shfl_xor_sync(0xffffffffu, l, x);
      if (g == 0) {
        part_m[warp * R + 8 * n + 2 * t + e] = run.m[n][e];
        part_l[warp * R + 8 * n + 2 * t + e] = l;
      }
#pragma unroll
      for (int i = 0; i < D / 16; ++i)
        *reinterpret_cast<float2*>(part_o + ((warp * R + 8 * n + 2 * t + e) * D + D / 8 * g +
                                             2 * i)) =
            make_float2(run.o[n][i][e], run.o[n][i][e + 2]);
    }
  }
  __syncthreads();
  auto joined = [](float m, float to) { return m == -INFINITY ? 0.0f : ex2(m - to); };
  for (int r = threadIdx.x; r < R; r += blockDim.x) {
    float m = -INFINITY, l = 0.0f;
    for (int w = 0; w < W; ++w) m = fmaxf(m, part_m[w * R + r]);
    for (int w = 0; w < W; ++w) l += part_l[w * R + r] * joined(part_m[w * R + r], m);
    cta_m[r] = m;
    cta_l[r] = l;
  }
  __syncthreads();
  for (int e = threadIdx.x; e < R * D; e += blockDim.x) {
    const int r = e / D;
    float o = 0.0f;
    for (int w = 0; w < W; ++w)
      o += part_o[w * R * D + e] * joined(part_m[w * R + r], cta_m[r]);
    part_o[e] = o;
  }
  auto emit = [&](int e, float o, float m, float l) {
    const int r = e / D, row = r0 + r;
    if (row >= rows) return;
    const int64_t at = row_at(row);
    a.out[at * D + e % D] = o / l;
    if (a.lse && e % D == 0) a.lse[at] = (m + log2f(l)) * kLn2;
  };
  if (cluster == 1) {
    for (int e = threadIdx.x; e < R * D; e += blockDim.x)   // the thread's own sums
      emit(e, part_o[e], cta_m[e / D], cta_l[e / D]);
    return;
  }
  cg::cluster_group cl = cg::this_cluster();
  cl.sync();
  const int share = R * D / cluster;
  for (int i = threadIdx.x; i < share; i += blockDim.x) {
    const int e = rank * share + i, r = e / D;
    float m = -INFINITY, l = 0.0f, o = 0.0f;
    for (int k = 0; k < cluster; ++k) m = fmaxf(m, *cl.map_shared_rank(cta_m + r, k));
    for (int k = 0; k < cluster; ++k) {
      const float f = joined(*cl.map_shared_rank(cta_m + r, k), m);
      l = fmaf(*cl.map_shared_rank(cta_l + r, k), f, l);
      o = fmaf(*cl.map_shared_rank(part_o + e, k), f, o);
    }
    emit(e, o, m, l);
  }
  cl.sync();
}

// ---------------------------------------------------------------------------
// Weights: S^T again, now with the softmax sums known.  A warp keeps the keys
// of one 16-key tile and walks the rows that see them.
template <int D>
__global__ void __launch_bounds__(128) kv8_weights_kernel(const AttnArgs a) {
  const int S = a.c.max_seq, G = a.Hq / a.c.kv_heads;
  const int bh = blockIdx.y, b = bh / a.c.kv_heads, h = bh % a.c.kv_heads;
  const int n_new = a.new_lens ? clamp_len(a.new_lens[b], a.T) : a.T;
  const int len = clamp_len(a.c.lens[b], S), total = min(len + n_new, S);
  const int shift = 31 - __clz(a.c.block), closed = total >> shift << shift;
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int tile = blockIdx.x * 4 + (threadIdx.x >> 5), jb = tile * 16;
  if (n_new == 0 || jb >= total) return;
  const bool tail = jb >= closed;
  uint32_t ka[D / 16][4], kl[D / 16][4];   // A fragments, hi and lo (tail only)
  float up;
  if (!tail) {
    Keys<D> kv;
    kv.k8 = a.c.k + (int64_t)bh * S * D;
    kv.ks = a.c.k_scale + (int64_t)bh * (S >> shift);
    kv.shift = shift;
    Frag<D> f;
    kv.load_k(f, tile, g, t);
    up = f.ks;
#pragma unroll
    for (int k = 0; k < D / 16; ++k) {
      const uint32_t w0 = reinterpret_cast<const uint32_t*>(&f.k[0][k / 4])[k % 4] ^ 0x80808080u;
      const uint32_t w1 = reinterpret_cast<const uint32_t*>(&f.k[1][k / 4])[k % 4] ^ 0x80808080u;
      ka[k][0] = two_halves(w0, 0x4140);
      ka[k][1] = two_halves(w1, 0x4140);
      ka[k][2] = two_halves(w0, 0x4342);
      ka[k][3] = two_halves(w1, 0x4342);
#pragma unroll
      for (int e = 0; e < 4; ++e) kl[k][e] = 0;
    }
  } else {
    const float* kt = a.c.k_tail + (int64_t)bh * ((int64_t)D << shift);
    float x[2][D / 64][16];
    uint32_t mx = 0;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int j = jb + g + 8 * r;
      const float* row = kt + (int64_t)(j & (a.c.block - 1)) * D + 16 * t;
#pragma unroll
      for (int hh = 0; hh < D / 64; ++hh)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          x[r][hh][i] = j < total ? row[64 * hh + i] : 0.0f;
          mx = max(mx, finite_abs(x[r][hh][i]));
        }
    }
    float down;
    pow2_scale(__reduce_max_sync(0xffffffffu, mx), down, up);
#pragma unroll
    for (int k = 0; k < D / 16; ++k) {
      const int hh = k / 4, i = 4 * (k % 4);
      split2(x[0][hh][i] * down, x[0][hh][i + 1] * down, ka[k][0], kl[k][0]);
      split2(x[1][hh][i] * down, x[1][hh][i + 1] * down, ka[k][1], kl[k][1]);
      split2(x[0][hh][i + 2] * down, x[0][hh][i + 3] * down, ka[k][2], kl[k][2]);
      split2(x[1][hh][i + 2] * down, x[1][hh][i + 3] * down, ka[k][3], kl[k][3]);
    }
  }
  const int rows = n_new * G;
  float w[2] = {0.0f, 0.0f};
  // rows of the tokens before the tile's first key see none of it
  for (int r0 = max(0, jb - len) * G / 8 * 8; r0 < rows; r0 += 8) {
    const int r = r0 + g;
    uint32_t qf[D / 16][4];
    float qs[2], z[2];
    int last[2];
    auto row_at = [&](int rr) { return ((int64_t)b * a.T + rr / G) * a.Hq + h * G + rr % G; };
    load_q<D>(qf, qs, r < rows ? a.q + row_at(r) * D : nullptr, a.scale, t);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int col = r0 + 2 * t + e;
      z[e] = col < rows ? a.lse[row_at(col)] * kLog2e : 0.0f;
      last[e] = col < rows ? min(len + col / G, total - 1) : -1;
    }
    float c[4] = {};
#pragma unroll
    for (int k = 0; k < D / 16; ++k) {
      if (tail) mma16816(c, kl[k], qf[k][0], qf[k][1]);
      mma16816(c, ka[k], qf[k][2], qf[k][3]);
      mma16816(c, ka[k], qf[k][0], qf[k][1]);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (jb + g + 8 * (e >> 1) <= last[e & 1])
        w[e >> 1] += ex2(fmaf(c[e], up * qs[e & 1], -z[e & 1]));
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    w[i] += __shfl_xor_sync(0xffffffffu, w[i], 1);
    w[i] += __shfl_xor_sync(0xffffffffu, w[i], 2);
    const int j = jb + g + 8 * i;
    if (t == 0 && j < total) {
      float* p = a.weights + (int64_t)bh * S + j;
      *p = (j < len ? *p : 0.0f) + w[i];
    }
  }
}

template <int D, int NT>
int launch_few(cudaStream_t s, const AttnArgs& a) {
  constexpr int R = 8 * NT;
  const int groups = (int)ceil_div((int64_t)a.T * (a.Hq / a.c.kv_heads), R);
  const int64_t units = (int64_t)groups * a.c.kv_heads * a.c.batch;
  // Spread a sequence's keys over warps while there are SMs without work and
  // a warp still has a step of tiles; over CTAs before warps.
  const int steps = (int)ceil_div(a.c.max_seq, D == 64 ? 64 : 32);
  int W = 4, C = 1;
  while (C < 16 && units * C * 2 <= 2 * kNumSms && C * 2 * W <= steps) C *= 2;
  while (W < kFewMaxWarps && units * C * W * 2 <= 16 * kNumSms && C * W * 2 <= steps) W *= 2;
  const size_t smem = sizeof(float) * ((size_t)W * R * (2 + D) + 2 * R);
  auto kern = attention_kv8_few_kernel<D, NT>;
  int rc;
  if (smem > 48 * 1024 &&
      (rc = check_cuda(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                            (int)smem),
                       "attention_kv8: smem attribute")))
    return rc;
  if (C > 8 && (rc = check_cuda(cudaFuncSetAttribute(
                                    kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1),
                                "attention_kv8: cluster attribute")))
    return rc;
  if ((int64_t)groups * a.c.kv_heads * C > INT32_MAX || a.c.batch > 65535)
    return fail(SPX_ERR_UNSUPPORTED, "attention_kv8: grid too large");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(groups * a.c.kv_heads * C), (unsigned)a.c.batch);
  cfg.blockDim = dim3((unsigned)W * 32);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)C;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return check_cuda(cudaLaunchKernelEx(&cfg, kern, a, groups, C), "attention_kv8");
}

}  // namespace

int launch_attention_kv8(cudaStream_t s, int64_t* cnt, const float* q, const spx_kv8_cache* c,
                         const int32_t* new_lens, int T, int Hq, float scale, float* out,
                         float* lse, float* weights) {
  int rc = kv8_check(c, "attention_kv8");
  if (rc) return rc;
  if (T <= 0 || Hq <= 0 || Hq % c->kv_heads)
    return fail(SPX_ERR_INVALID_ARGUMENT, "attention_kv8: bad shape");
  if (weights && !lse)
    return fail(SPX_ERR_INVALID_ARGUMENT, "attention_kv8: weights need an lse buffer");
  if (((uintptr_t)q & 15) || ((uintptr_t)out & 15))
    return fail(SPX_ERR_INVALID_ARGUMENT, "attention_kv8: q and out must be 16-byte aligned");
  const int64_t bh = (int64_t)c->batch * c->kv_heads;
  if ((int64_t)c->batch * T * Hq > INT32_MAX || bh > 65535)
    return fail(SPX_ERR_UNSUPPORTED, "attention_kv8: grid too large");
  const AttnArgs a{q, *c, new_lens, T, Hq, scale, out, lse, weights};
  const bool wide = (int64_t)T * (Hq / c->kv_heads) > 8;
  if (c->head_dim == 64)
    rc = wide ? launch_few<64, 2>(s, a) : launch_few<64, 1>(s, a);
  else
    rc = launch_few<128, 1>(s, a);
  if (rc) return rc;
  if ((rc = after_launch(cnt, "attention_kv8")) || !weights) return rc;
  const dim3 wg((unsigned)ceil_div(c->max_seq, 64), (unsigned)bh);
  if (c->head_dim == 64)
    kv8_weights_kernel<64><<<wg, 128, 0, s>>>(a);
  else
    kv8_weights_kernel<128><<<wg, 128, 0, s>>>(a);
  return after_launch(cnt, "attention_kv8: weights");
}

}  // namespace spx
