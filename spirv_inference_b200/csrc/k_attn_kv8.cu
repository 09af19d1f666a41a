// Causal grouped-query attention over the 8-bit key / value cache, and the
// attention weight each slot receives.
//
//   s = scale q.k,  out = softmax(s) v,  lse = log sum exp(s)
//   weights[j] += sum over the new tokens and the heads of the group of
//                 exp(s_j - lse)     (slots of the new tokens start from 0)
//
// Tensor cores in fp32 accuracy, with the int8 operand as it is.
//
// Scores: a row of q, scaled by a power of two to whole numbers below 2^30, is
// four digits of 8 bits, and the products of each digit with the int8 keys are
// exact in int32 (mma m16n8k32); the scale of the keys' block multiplies their
// sum.  An element of q keeps its 24 bits down to 2^-6 of the row's largest, and
// below that 2^-30 of it.
//
// Outputs: an int8 value is exact in fp16, p as fp16 hi + lo has 22 bits, and
// each product is taken twice with fp32 sums.  p is multiplied by its block's
// share v_scale / v_ref (v_ref the largest scale of the tiles in hand) and by
// 2^15, so that small p keep their low part.  The tensor core's additions
// round towards zero, so a few tiles' products are added to the running
// output in fp32.
//
// Rows of the tail are fp32: both operands are split into fp16 hi + lo, each row
// scaled by a power of two of its own, three products each.
#include <cooperative_groups.h>
#include <cuda_fp16.h>

#include <array>
#include <type_traits>

#include "attn_kv8.cuh"

namespace spx {
namespace {

namespace cg = cooperative_groups;

// d = a b + c.  (c apart from d: zeros and constants need no copy.)
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                         uint32_t b1, float c0, float c1, float c2, float c3) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%10, %11, %12, %13};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2),
        "f"(c3));
}
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                         uint32_t b1) {
  mma16816(c, a, b0, b1, c[0], c[1], c[2], c[3]);
}
__device__ __forceinline__ void mma16832(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                         uint32_t a3, uint32_t b0, uint32_t b1, int c0, int c1,
                                         int c2, int c3) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%10, %11, %12, %13};"
      : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "r"(c0), "r"(c1), "r"(c2), "r"(c3));
}
__device__ __forceinline__ void cluster_arrive() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() {
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// ---------------------------------------------------------------------------
// Few rows (decode, drafts).  A row is a (new token, head of the group) pair;
// a warp takes 8 of them, or 16, and walks its own groups of 16-key tiles with
// its own running maxima and sums.
//
// Scores, S = Q K^T: the 16 rows of the A operand are the first and the second
// digits of 8 rows of q, in another product the third and the fourth, the 8
// columns are keys.  Within a dot product the order of d is free, so lane (g, t) takes
// 16 contiguous bytes of a key, and they are its B operand as they come from
// memory.  Lane (g, t) then holds row g and two keys of eight, which is also
// how O^T = V^T P^T wants P as its B operand.  There the lane's V bytes of four
// keys become fp16 pairs of keys.
//
// A warp copies its next groups of 32 keys to shared memory for itself, three
// ahead (64 D bytes each, 192 KB an SM), with no barrier but its own.
//
// Warps are joined in shared memory and the CTAs of a cluster, over which one
// sequence's keys are spread, by stores into each other's shared memory: one
// launch, no workspace.
//
// What bounds it: the cache's bytes, 2 D + 8 / block a key and head, and close
// behind the instructions, about 150 for 16 keys of D = 64 and 8 rows (48 of
// them turn V into fp16); with sequences of unlike lengths, the longest one.  So
// tiles that every row sees in full take a path without masks, and the others, one
// by one, another.
// Which key of eight stands in column n: the order in which lanes' reads of K
// (keys_at(g), 16 bytes at t) and of V (keys_at(2t), keys_at(2t + 1), 8 bytes
// at g) meet no bank of shared memory twice.
__device__ __forceinline__ int key_at(int n) { return n & 1 ? ((n >> 1) ^ 1) + 4 : n >> 1; }
// The key of 16 that score e of a lane belongs to.
__device__ __forceinline__ int key_of(int e, int t) {
  return 8 * (e >> 1) + (e & 1 ? (t ^ 1) + 4 : t);
}
// 16-byte pieces of a row are exchanged by this in shared memory.
template <int D>
__device__ __forceinline__ int row_swap(int row) {
  return (D == 128 ? 4 * (row & 1) : 0) + (row & 2);
}

template <int D>
struct Frag {                   // one 16-key tile of int8 K and V in registers
  uint4 k[2][D / 64];           // keys key_at(g), + 8
  uint32_t v[4][D / 32];        // keys key_of(0 .. 3); d = D/8 g ...
  float ks, vs;
};

template <int NW>
__device__ __forceinline__ void put_words(uint32_t (&w)[NW], uint2 x) {
  w[0] = x.x;
  w[1] = x.y;
}
template <int NW>
__device__ __forceinline__ void put_words(uint32_t (&w)[NW], uint4 x) {
  w[0] = x.x;
  w[1] = x.y;
  w[2] = x.z;
  w[3] = x.w;
}

template <int D>
struct Keys {
  using Words = typename std::conditional<D == 64, uint2, uint4>::type;
  const int8_t* k8;
  const int8_t* v8;
  const float* ks;
  const float* vs;
  const float* kt;
  const float* vt;
  int shift;           // log2(block)
  __device__ __forceinline__ Keys(const spx_kv8_cache& c, int64_t bh) {
    shift = 31 - __clz(c.block);
    k8 = c.k + bh * c.max_seq * D;
    v8 = c.v + bh * c.max_seq * D;
    ks = c.k_scale + bh * (c.max_seq >> shift);
    vs = c.v_scale + bh * (c.max_seq >> shift);
    kt = c.k_tail + bh * ((int64_t)D << shift);
    vt = c.v_tail + bh * ((int64_t)D << shift);
  }
  // One tile from global memory.
  __device__ __forceinline__ void load_k(Frag<D>& f, int tile, int g, int t) const {
    const int8_t* p = k8 + (int64_t)tile * (16 * D) + key_at(g) * D + 16 * t;
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
      for (int h = 0; h < D / 64; ++h)
        f.k[r][h] = __ldg(reinterpret_cast<const uint4*>(p + 8 * r * D + 64 * h));
    f.ks = __ldg(ks + ((tile * 16) >> shift));
  }
  __device__ __forceinline__ void load_v(Frag<D>& f, int tile, int g, int t) const {
    const int8_t* p = v8 + (int64_t)tile * (16 * D) + D / 8 * g;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      put_words(f.v[e], __ldg(reinterpret_cast<const Words*>(p + key_of(e, t) * D)));
    f.vs = __ldg(vs + ((tile * 16) >> shift));
  }
};

// A warp's ring of groups of 32 keys in shared memory.
template <int D>
struct Ring {
  static constexpr int kSlots = 3, kGroup = 32 * D, kSlot = 2 * kGroup;   // bytes: K, then V
  uint32_t here;          // the lane's place in the ring, as it copies
  uint32_t k_at[D / 64];  // the lane's bytes of K and V in a slot
  uint32_t v_at[2];
  __device__ __forceinline__ Ring(uint8_t* mem, int lane, int g, int t) {
    const uint32_t base = (uint32_t)__cvta_generic_to_shared(mem);
    constexpr int kPieces = D / 16;
    const int row = lane / kPieces;
    here = base + row * D + ((lane % kPieces) ^ row_swap<D>(row)) * 16;
    const int k = key_at(g);
#pragma unroll
    for (int h = 0; h < D / 64; ++h)
      k_at[h] = base + k * D + ((t + 4 * h) ^ row_swap<D>(k)) * 16;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int v = key_of(e, t);
      v_at[e] = base + kGroup + v * D +
                (D == 64 ? ((g >> 1) ^ row_swap<D>(v)) * 16 + (g & 1) * 8
                         : (g ^ row_swap<D>(v)) * 16);
    }
  }
  // Starts the copies of the 32 keys from tile `tile` on, if any.
  __device__ __forceinline__ void start(int slot, const Keys<D>& kv, int tile, bool any,
                                        bool with_v, int lane) const {
    if (any) {
      const int64_t from = (int64_t)tile * (16 * D) + lane * 16;
      const uint32_t to = here + slot * kSlot;
#pragma unroll
      for (int i = 0; i < kGroup / 512; ++i)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + i * 512),
                     "l"(kv.k8 + from + i * 512)
                     : "memory");
      if (with_v) {
#pragma unroll
        for (int i = 0; i < kGroup / 512; ++i)
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + kGroup + i * 512),
                       "l"(kv.v8 + from + i * 512)
                       : "memory");
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  // Until the oldest of kSlots groups is there, for the whole warp.
  __device__ __forceinline__ void wait() const {
    asm volatile("cp.async.wait_group %0;" ::"n"(kSlots - 1) : "memory");
    __syncwarp();
  }
  __device__ __forceinline__ void drain() const {
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncwarp();
  }
  __device__ __forceinline__ void read_k(Frag<D>& f, int slot, int k) const {
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
      for (int h = 0; h < D / 64; ++h) {
        uint4& x = f.k[r][h];
        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w)
                     : "r"(k_at[h] + slot * kSlot + (16 * k + 8 * r) * D));
      }
  }
  __device__ __forceinline__ void read_v(Frag<D>& f, int slot, int k) const {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t at = v_at[e & 1] + slot * kSlot + (16 * k + 8 * (e >> 1)) * D;
      if constexpr (D == 64)
        asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];"
                     : "=r"(f.v[e][0]), "=r"(f.v[e][1])
                     : "r"(at));
      else
        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(f.v[e][0]), "=r"(f.v[e][1]), "=r"(f.v[e][2]), "=r"(f.v[e][3])
                     : "r"(at));
    }
  }
};

// The lane's 16 values in each 64 of a row of q, and the row's largest finite
// magnitude; `odd`: the row has a NaN or an infinity.
template <int D>
__device__ __forceinline__ uint32_t read_q(float (&x)[D / 64][16], bool& odd, const float* row,
                                           int t) {
  uint32_t mx = 0;
  odd = false;
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
      for (int e = 0; e < 4; ++e) {
        mx = max(mx, finite_abs(x[h][4 * i + e]));
        odd |= (__float_as_uint(x[h][4 * i + e]) & 0x7f800000u) == 0x7f800000u;
      }
    }
  mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
  mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
  odd = __ballot_sync(0xffffffffu, odd) >> ((threadIdx.x & 28)) & 15u;
  return mx;
}

// Digits of 8 rows of q as A fragments: [k-step][digit][4 + 4 values], and the
// factor that takes a product of row g to a score in units of log 2 (NaN for a
// row with a NaN or an infinity).
template <int D>
__device__ __forceinline__ void load_q(uint32_t (&qd)[D / 32][4][2], float& qs, const float* row,
                                       float scale, int t) {
  float x[D / 64][16];
  bool odd;
  int exp = (int)(read_q<D>(x, odd, row, t) >> 23);
  exp = exp < 30 ? 30 : exp;             // (a row below 2^-97 stays smaller)
  // the largest to 2^29 or above, below 2^30, and back
  float down = __uint_as_float((uint32_t)(283 - exp) << 23);
  if (scale < 0.0f) down = -down;
  qs = __uint_as_float((uint32_t)(exp - 29) << 23) * (fabsf(scale) * kLog2e);
  if (odd) qs = __int_as_float(0x7fc00000);
#pragma unroll
  for (int i = 0; i < D / 16; ++i) {     // four values: k-step i / 2, register i % 2
    uint32_t w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e)
      // digits in [-128, 127]: the bytes of v + 0x80808080, less 128 each (of a
      // NaN or an infinity, any)
      w[e] = ((uint32_t)__float2int_rn(x[i / 4][4 * (i % 4) + e] * down) + 0x80808080u) ^
             0x80808080u;
    const uint32_t a = __byte_perm(w[0], w[1], 0x5140), b = __byte_perm(w[2], w[3], 0x5140);
    const uint32_t c = __byte_perm(w[0], w[1], 0x7362), d = __byte_perm(w[2], w[3], 0x7362);
    qd[i / 2][0][i % 2] = __byte_perm(c, d, 0x7632);
    qd[i / 2][1][i % 2] = __byte_perm(c, d, 0x5410);
    qd[i / 2][2][i % 2] = __byte_perm(a, b, 0x7632);
    qd[i / 2][3][i % 2] = __byte_perm(a, b, 0x5410);
  }
}

// Q K^T of 8 NT rows and one int8 tile, before any scale, plus kBias: row g,
// keys key_of(0 .. 3).
constexpr float kBias = 12582912.0f;   // 1.5 2^23, of scores of about 2^36
template <int D, int NT>
__device__ __forceinline__ void products(float (&c)[NT][4], const Frag<D>& f,
                                         const uint32_t (&qd)[NT][D / 32][4][2]) {
  constexpr int kOne = 0x4b400000;     // as a float, kBias; plus a sum, kBias + the sum
#pragma unroll
  for (int b = 0; b < 2; ++b)
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      int hi[4], lo[4];
#pragma unroll
      for (int s = 0; s < D / 32; ++s) {
        const uint32_t* k = reinterpret_cast<const uint32_t*>(&f.k[b][s / 2]) + 2 * (s % 2);
        const uint32_t(&q)[4][2] = qd[n][s];
        if (s == 0) {
          mma16832(hi, q[0][0], q[1][0], q[0][1], q[1][1], k[0], k[1], 0, 0, 0, 0);
          mma16832(lo, q[2][0], q[3][0], q[2][1], q[3][1], k[0], k[1], kOne, kOne, kOne, kOne);
        } else {
          mma16832(hi, q[0][0], q[1][0], q[0][1], q[1][1], k[0], k[1], hi[0], hi[1], hi[2], hi[3]);
          mma16832(lo, q[2][0], q[3][0], q[2][1], q[3][1], k[0], k[1], lo[0], lo[1], lo[2], lo[3]);
        }
      }
      // the last two digits with one bias of two, then all (hi: below 2^29)
      const float2 third = add2(make_float2(__int_as_float(lo[0]), __int_as_float(lo[1])),
                                make_float2(-kBias, -kBias));
      const float2 low = fma2(third, make_float2(256.0f, 256.0f),
                              make_float2(__int_as_float(lo[2]), __int_as_float(lo[3])));
      const float2 sum = fma2(
          make_float2((float)(hi[0] * 256 + hi[2]), (float)(hi[1] * 256 + hi[3])),
          make_float2(65536.0f, 65536.0f), low);
      c[n][2 * b] = sum.x;
      c[n][2 * b + 1] = sum.y;
    }
}

// The running softmax of one warp: lane (g, t) holds maximum and sum of row g
// of each 8 and, of the output, rows 2t, 2t+1 and d = D/8 g .. D/8 (g + 1) - 1.
template <int D, int NT>
struct Running {
  float m[NT], l[NT], o[NT][D / 16][4];   // o in units of `ref` / 2^15
  float ref;                              // the largest v scale so far, or kMinRef
  __device__ __forceinline__ void init() {
    ref = kMinRef;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      m[n] = -INFINITY;
      l[n] = 0.0f;
#pragma unroll
      for (int i = 0; i < D / 16; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[n][i][e] = 0.0f;
    }
  }
  // New maxima for tile scores (c - bias) f (f >= 0 the tile's factor of row
  // g); c becomes exp2(score - m), 0 where hidden, the sums take them, and
  // `corr` is what the outputs of the lane's two rows have to be scaled by.
  template <int KT, bool MASK>
  __device__ __forceinline__ void weigh(float (&c)[KT][NT][4], const float (&f)[KT][NT],
                                        float bias, float (&corr)[NT][2], uint32_t hidden,
                                        int t) {
    auto hides = [&](int k, int n, int e) {
      return MASK && (hidden >> ((k * NT + n) * 4 + e) & 1u);
    };
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float mt = -INFINITY, off[KT];
#pragma unroll
      for (int k = 0; k < KT; ++k) {
        off[k] = -bias * f[k][n];
        if (MASK) {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (!hides(k, n, e)) mt = fmaxf(mt, fmaf(c[k][n][e], f[k][n], off[k]));
        } else {
          const float most = fmaxf(fmaxf(c[k][n][0], c[k][n][1]), fmaxf(c[k][n][2], c[k][n][3]));
          mt = fmaxf(mt, fmaf(most, f[k][n], off[k]));
        }
      }
      mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, 1));
      mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, 2));
      const float mn = fmaxf(m[n], mt), base = mn == -INFINITY ? 0.0f : mn;
      const float down = ex2(m[n] - base);
      m[n] = mn;
      float sum = 0.0f;
#pragma unroll
      for (int k = 0; k < KT; ++k) {
        const float to = off[k] - base;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          c[k][n][e] = hides(k, n, e) ? 0.0f : ex2(fmaf(c[k][n][e], f[k][n], to));
          sum += c[k][n][e];
        }
      }
      l[n] = fmaf(l[n], down, sum);
      corr[n][0] = __shfl_sync(0xffffffffu, down, t * 8);
      corr[n][1] = __shfl_sync(0xffffffffu, down, t * 8 + 4);
    }
  }
};

// P (row g, 16 keys, already scaled) as B fragments: hi b0, b1, lo b0, b1.
__device__ __forceinline__ void p_frags(uint32_t (&pf)[4], const float (&p)[4]) {
  split2(p[0], p[1], pf[0], pf[2]);
  split2(p[2], p[3], pf[1], pf[3]);
}

// The factor that takes a tile's v scale to its share of 2^15, after `ref` has
// grown to the largest (finite) scale of KT tiles; `corr` takes what the change
// means for the outputs so far.
template <int D, int NT>
__device__ __forceinline__ float share_of(Running<D, NT>& run, float largest,
                                          float (&corr)[NT][2]) {
  if (largest > run.ref) {               // the same in every lane
    const float down = run.ref / largest;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      corr[n][0] *= down;
      corr[n][1] *= down;
    }
    run.ref = largest;
  }
  return kPUp / run.ref;
}

// O^T += V^T P^T over KT int8 tiles; c: exp2(score - m), zero where MASK hides.
template <int D, int NT, int KT, bool MASK>
__device__ __forceinline__ void add_values(Running<D, NT>& run, const Frag<D> (&f)[KT],
                                           float (&c)[KT][NT][4], float (&corr)[NT][2],
                                           uint32_t hidden) {
  float most = 0.0f, sum = 0.0f;
#pragma unroll
  for (int k = 0; k < KT; ++k) {
    most = fmaxf(most, f[k].vs);
    sum += f[k].vs;
  }
  const bool odd = !(sum <= 3.4028234663852886e38f);   // a block with a NaN or an infinity
  if (odd) {
    most = 0.0f;
#pragma unroll
    for (int k = 0; k < KT; ++k)
      if (f[k].vs <= 3.4028234663852886e38f) most = fmaxf(most, f[k].vs);
  }
  const float inv = share_of<D, NT>(run, most, corr);
#pragma unroll
  for (int k = 0; k < KT; ++k) {
    const float share = f[k].vs * inv;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) c[k][n][e] *= share;
  }
  if (odd) {
    // The weights of that block's keys become NaN, hidden ones stay zero.
    asm volatile("");              // a branch, not selects
#pragma unroll
    for (int k = 0; k < KT; ++k)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (!(f[k].vs <= 3.4028234663852886e38f)) c[k][n][e] = __int_as_float(0x7fc00000);
          if (MASK && (hidden >> ((k * NT + n) * 4 + e) & 1u)) c[k][n][e] = 0.0f;
        }
  }
  uint32_t mask;
  asm volatile("mov.b32 %0, 0x00ff00ff;" : "=r"(mask));
  float o[NT][D / 16][4];
#pragma unroll
  for (int k = 0; k < KT; ++k) {
    uint32_t pf[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) p_frags(pf[n], c[k][n]);
#pragma unroll
    for (int w = 0; w < D / 32; ++w)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        // d = 2 (2w + i) and + 1 of keys key_of(0, 1) and key_of(2, 3)
        const uint32_t sel = i ? 0x7632 : 0x5410;
        const uint32_t x = __byte_perm(f[k].v[0][w], f[k].v[1][w], sel);
        const uint32_t y = __byte_perm(f[k].v[2][w], f[k].v[3][w], sel);
        const uint32_t av[4] = {even_bytes(x, mask), even_bytes(x >> 8, mask),
                                even_bytes(y, mask), even_bytes(y >> 8, mask)};
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float(&acc)[4] = o[n][2 * w + i];
          if (k == 0)
            mma16816(acc, av, pf[n][0], pf[n][1], 0.f, 0.f, 0.f, 0.f);
          else
            mma16816(acc, av, pf[n][0], pf[n][1]);
          mma16816(acc, av, pf[n][2], pf[n][3]);
        }
      }
  }
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int i = 0; i < D / 16; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        run.o[n][i][e] = fmaf(run.o[n][i][e], corr[n][e & 1], o[n][i][e]);
}

// Scores of one 16-key tile of the tail, in units of log 2: fp32 rows, both
// operands split, each row and each key by its own power of two.  The A operand's
// rows are q hi and q lo.  q: row g of each 8 (null: none).
template <int D, int NT>
__device__ __forceinline__ void tail_products(float (&c)[1][NT][4], const Keys<D>& kv,
                                              const float* const (&q)[NT], float scale, int jb,
                                              int total, int g, int t) {
  const int blk_mask = (1 << kv.shift) - 1;
  // All loads first: they do not move over the shuffles.
  float x[2][D / 64][16];                        // keys key_at(g), + 8
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int j = jb + key_at(g) + 8 * r;
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
      }
  }
  uint32_t a[NT][D / 16][4];
  float up[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    float y[D / 64][16], down;
    bool odd;
    pow2_scale(read_q<D>(y, odd, q[n], t), down, up[n]);
    up[n] *= fabsf(scale) * kLog2e;
    if (scale < 0.0f) down = -down;
#pragma unroll
    for (int k = 0; k < D / 16; ++k) {
      const int h = k / 4, i = 4 * (k % 4);
      split2(y[h][i] * down, y[h][i + 1] * down, a[n][k][0], a[n][k][1]);
      split2(y[h][i + 2] * down, y[h][i + 3] * down, a[n][k][2], a[n][k][3]);
    }
  }
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    float down, up_k;
    uint32_t mx = 0;
#pragma unroll
    for (int h = 0; h < D / 64; ++h)
#pragma unroll
      for (int i = 0; i < 16; ++i) mx = max(mx, finite_abs(x[r][h][i]));
    mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
    mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
    pow2_scale(mx, down, up_k);
    float s[NT][4] = {};
#pragma unroll
    for (int k = 0; k < D / 16; ++k) {
      const int h = k / 4, i = 4 * (k % 4);
      uint32_t hi[2], lo[2];
      split2(x[r][h][i] * down, x[r][h][i + 1] * down, hi[0], lo[0]);
      split2(x[r][h][i + 2] * down, x[r][h][i + 3] * down, hi[1], lo[1]);
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        mma16816(s[n], a[n][k], lo[0], lo[1]);
        mma16816(s[n], a[n][k], hi[0], hi[1]);
      }
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      // column 2t + e is key key_at(2t + e)
      const float by = __shfl_sync(0xffffffffu, up_k, t * 8 + 4 * e);
#pragma unroll
      for (int n = 0; n < NT; ++n)
        c[0][n][2 * r + e] = (s[n][e] + s[n][e + 2]) * up[n] * by;
    }
  }
}

// Which of a tile's scores their rows do not see.
template <int NT>
__device__ __forceinline__ uint32_t hidden_in(int jb, const int (&last)[NT], int t) {
  uint32_t hidden = 0;
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e)
      hidden |= (jb + key_of(e, t) > last[n] ? 1u : 0u) << (n * 4 + e);
  return hidden;
}

// One 16-key tile of the tail.
template <int D, int NT>
__device__ __forceinline__ void tail_tile(Running<D, NT>& run, const Keys<D>& kv,
                                          const float* const (&q)[NT], float scale,
                                          const int (&last)[NT], int jb, int total, int g,
                                          int t) {
  const int blk_mask = (1 << kv.shift) - 1;
  float c[1][NT][4], one[1][NT], corr[NT][2];
  tail_products<D, NT>(c, kv, q, scale, jb, total, g, t);
#pragma unroll
  for (int n = 0; n < NT; ++n) one[0][n] = 1.0f;
  const uint32_t hidden = hidden_in<NT>(jb, last, t);
  run.template weigh<1, true>(c, one, 0.0f, corr, hidden, t);
  // V of keys key_of(0 .. 3), each by its own power of two; rows of 128 are read
  // once more for the products, piece by piece (all at once took the loop over
  // whole groups registers).
  auto piece = [&](int i, int e) {       // NaNs and infinities as they are
    const int j = jb + key_of(i, t);
    return j < total ? *(reinterpret_cast<const float4*>(
                             kv.vt + (int64_t)(j & blk_mask) * D + D / 8 * g) +
                         e)
                     : make_float4(0.f, 0.f, 0.f, 0.f);
  };
  float up[4], down[4];
  float4 y[4][D / 32];
  uint32_t mx[4] = {}, any[4] = {};
#pragma unroll
  for (int i = 0; i < 4; ++i)            // (loads do not move over shuffles)
#pragma unroll
    for (int e = 0; e < D / 32; ++e) {
      const float4 v = y[i][e] = piece(i, e);
      mx[i] = max(max(mx[i], finite_abs(v.x)),
                  max(finite_abs(v.y), max(finite_abs(v.z), finite_abs(v.w))));
      any[i] = max(max(any[i], __float_as_uint(v.x) & 0x7fffffffu),
                   max(__float_as_uint(v.y) & 0x7fffffffu,
                       max(__float_as_uint(v.z) & 0x7fffffffu,
                           __float_as_uint(v.w) & 0x7fffffffu)));
    }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    // over the lanes that hold the key
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) mx[i] = max(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], o));
    pow2_scale(mx[i], down[i], up[i]);
    // A NaN or infinity would reach rows that do not see this key: it goes into
    // the key's weight instead, where the mask stops it.
    if (__ballot_sync(0xffffffffu, any[i] >= 0x7f800000u) >> t & 0x11111111u)
      up[i] = __int_as_float(0x7fc00000);
  }
  // The tile's sums of a row are in units of `most` / 2^15, the largest factor of
  // the keys that it sees (others, later ones, do not matter to it), the running
  // ones in units of ref / 2^15.
  uint32_t pf[NT][4];
  float most[NT], all = 0.0f, back[NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    most[n] = 0x1p-126f;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (!(hidden >> (n * 4 + e) & 1u)) most[n] = fmaxf(most[n], up[e]);
    most[n] = fmaxf(most[n], __shfl_xor_sync(0xffffffffu, most[n], 1));
    most[n] = fmaxf(most[n], __shfl_xor_sync(0xffffffffu, most[n], 2));
    all = fmaxf(all, most[n]);
    const float inv = __uint_as_float((254u << 23) - __float_as_uint(most[n]));   // exact
#pragma unroll
    for (int e = 0; e < 4; ++e)        // (a hidden key's factor may be NaN)
      c[0][n][e] = hidden >> (n * 4 + e) & 1u ? 0.0f : c[0][n][e] * (up[e] * inv) * kPUp;
    p_frags(pf[n], c[0][n]);
  }
#pragma unroll
  for (int o = 4; o < 32; o <<= 1) all = fmaxf(all, __shfl_xor_sync(0xffffffffu, all, o));
  const float unit = share_of<D, NT>(run, all, corr) * (1.0f / kPUp);
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int e = 0; e < 2; ++e)
      back[n][e] = __shfl_sync(0xffffffffu, most[n], t * 8 + 4 * e) * unit;
#pragma unroll
  for (int e = 0; e < D / 32; ++e) {
    float x[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float4 v = D == 64 ? y[i][e] : piece(i, e);
      x[i][0] = v.x;
      x[i][1] = v.y;
      x[i][2] = v.z;
      x[i][3] = v.w;
#pragma unroll
      for (int z = 0; z < 4; ++z)
        x[i][z] = (__float_as_uint(x[i][z]) & 0x7f800000u) == 0x7f800000u ? 0.0f
                                                                          : x[i][z] * down[i];
    }
#pragma unroll
    for (int z = 0; z < 4; z += 2) {     // d = 4 e + z and + 1 of the lane's
      uint32_t a[4], al[4];
      split2(x[0][z], x[1][z], a[0], al[0]);
      split2(x[0][z + 1], x[1][z + 1], a[1], al[1]);
      split2(x[2][z], x[3][z], a[2], al[2]);
      split2(x[2][z + 1], x[3][z + 1], a[3], al[3]);
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float o[4] = {};
        mma16816(o, al, pf[n][0], pf[n][1]);
        mma16816(o, a, pf[n][2], pf[n][3]);
        mma16816(o, a, pf[n][0], pf[n][1]);
        float(&to)[4] = run.o[n][2 * e + z / 2];
#pragma unroll
        for (int f = 0; f < 4; ++f) to[f] = fmaf(to[f], corr[n][f & 1], back[n][f & 1] * o[f]);
      }
    }
  }
}

// What this lane's key of a tile has gathered: nothing for a new token.
__device__ __forceinline__ int own_key(int jb, int g, int t) {
  return jb + key_of((g & 4 ? 2 : 0) + (g & 2 ? 1 : 0), t);
}
__device__ __forceinline__ float gathered(const float* out, int jb, int len, int g, int t) {
  const int j = own_key(jb, g, t);
  return !(g & 1) && j < len ? out[j] : 0.0f;
}
// Puts the weights of a tile's keys: w of keys key_of(0 .. 3), summed over the
// lanes with the same t (each step leaves a lane half of the values), and what
// they had.
__device__ __forceinline__ void put_weights(float* out, const float (&w)[4], float had, int jb,
                                            int total, int g, int t) {
  const bool up = g & 4, right = g & 2;
  const float a = (up ? w[2] : w[0]) + __shfl_xor_sync(0xffffffffu, up ? w[0] : w[2], 16);
  const float b = (up ? w[3] : w[1]) + __shfl_xor_sync(0xffffffffu, up ? w[1] : w[3], 16);
  float sum = (right ? b : a) + __shfl_xor_sync(0xffffffffu, right ? a : b, 8);
  sum += __shfl_xor_sync(0xffffffffu, sum, 4);
  const int j = own_key(jb, g, t);
  if (!(g & 1) && j < total) out[j] = had + sum;
}
// w += exp2((c - bias) f - z) of row g of each 8, where it sees the key.
template <int NT>
__device__ __forceinline__ void add_weights(float (&w)[4], const float (&c)[1][NT][4],
                                            const float (&f)[1][NT], float bias,
                                            const float (&z)[NT], uint32_t hidden) {
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const float to = fmaf(-bias, f[0][n], -z[n]);
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (!(hidden >> (n * 4 + e) & 1u)) w[e] += ex2(fmaf(c[0][n][e], f[0][n], to));
  }
}

constexpr int kFewMaxWarps = 8;
constexpr int kMaxCluster = 16;
constexpr int kBigClusters[] = {16, 14, 12, 10};

template <int D, int NT>
struct FewShape {
  static constexpr int KT = 2;          // tiles of a group of 32 keys
  static constexpr int R = 8 * NT;      // rows
  // Warps an SM that the rings leave room for: 16, or 8 of D = 128.
  static constexpr int kBlocks = D == 64 && NT == 1 ? 2 : 1;   // of 8 warps
  // Shared memory in floats: the warps' rings (later their partial outputs),
  // then what the others of the cluster send, then maxima and sums.
  static constexpr int kRing = Ring<D>::kSlots * Ring<D>::kSlot / 4;
  static_assert(R * D <= kRing, "partial outputs fit a ring");
  static constexpr size_t smem(int W) {
    return sizeof(float) *
           ((size_t)W * kRing + R * D + 4 * kMaxCluster + 2 * W * R + 2 * kMaxCluster * R);
  }
};

template <int D, int NT>
__global__ void __launch_bounds__(kFewMaxWarps * 32, FewShape<D, NT>::kBlocks)
    attention_kv8_few_kernel(const AttnArgs a, int groups, int cluster) {
  using Shape = FewShape<D, NT>;
  constexpr int KT = Shape::KT, R = Shape::R, kRing = Shape::kRing;
  constexpr int kSlots = Ring<D>::kSlots;
  extern __shared__ __align__(16) float smem[];
  const int W = blockDim.x >> 5;
  float* part_o = smem;                 // [W][kRing], the first R D of each
  float* recv_o = part_o + W * kRing;   // [cluster][share]: of this CTA's outputs
  float* part_m = recv_o + R * D + 4 * kMaxCluster;   // [W][R]
  float* part_l = part_m + W * R;       // [W][R]
  float* recv_m = part_l + W * R;       // [cluster][R]
  float* recv_l = recv_m + kMaxCluster * R;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int rank = blockIdx.x % cluster;
  const int unit = blockIdx.x / cluster, grp = unit % groups, h = unit / groups, b = blockIdx.y;
  const int S = a.c.max_seq, Hkv = a.c.kv_heads, G = a.Hq / Hkv;
  if (cluster > 1) cluster_arrive();    // waited for before stores into other CTAs
  // What does not depend on the lengths is on its way before they are known.
  const int n_arg = a.new_lens ? a.new_lens[b] : a.T, len_arg = a.c.lens[b];
  const Keys<D> kv(a.c, (int64_t)b * Hkv + h);
  const Ring<D> ring(reinterpret_cast<uint8_t*>(part_o + warp * kRing), lane, g, t);
  const int first = (rank * W + warp) * KT, step = cluster * W * KT;
#pragma unroll
  for (int s = 0; s < kSlots; ++s)
    ring.start(s, kv, first + s * step, (first + s * step + KT) * 16 <= S, true, lane);
  const int r0 = grp * R, all_rows = a.T * G;
  auto row_at = [&](int r) {            // [token][head] row of the group's row r
    const int tk = a.div_g(r);
    return ((int64_t)b * a.T + tk) * a.Hq + h * G + (r - tk * G);
  };
  uint32_t qd[NT][D / 32][4][2];
  float qs[NT];
  const float* q_row[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int r = r0 + 8 * n + g;
    q_row[n] = r < all_rows ? a.q + row_at(r) * D : nullptr;
    load_q<D>(qd[n], qs[n], q_row[n], a.scale, t);
  }
  const int n_new = clamp_len(n_arg, a.T), rows = n_new * G;
  if (r0 >= rows) {                     // the whole cluster
    ring.drain();
    if (cluster > 1) cluster_wait();
    return;
  }
  const int len = clamp_len(len_arg, S), total = min(len + n_new, S);
  const int closed = total >> kv.shift << kv.shift;
  // slots that some row sees
  const int lim = min(len + a.div_g(min(r0 + R - 1, rows - 1)) + 1, S);
  int last[NT];                         // the last slot that row g sees
#pragma unroll
  for (int n = 0; n < NT; ++n)
    last[n] = min(len + a.div_g(min(r0 + 8 * n + g, rows - 1)), total - 1);
  Running<D, NT> run;
  run.init();

  // Groups of tiles that every row sees in full.
  const int tiles = (min(closed, lim) + 15) >> 4;
  const int whole = min(closed, len + a.div_g(r0) + 1) / (16 * KT) * KT;
  // (a block of 32 keys or more holds both tiles of a group)
  const int second = kv.shift == 4 ? 1 : 0;
  auto scales = [&](float (&s)[2 * KT], int base) {
    if (base >= whole) return;
    const int blk = (base * 16) >> kv.shift;
    s[0] = __ldg(kv.ks + blk);
    s[1] = __ldg(kv.ks + blk + second);
    s[2] = __ldg(kv.vs + blk);
    s[3] = __ldg(kv.vs + blk + second);
  };
  float sc[2 * KT], sc_next[2 * KT] = {};
  scales(sc_next, first);
  int slot = 0;
  for (int base = first; base < whole; base += step) {
    float c[KT][NT][4], fk[KT][NT], corr[NT][2];
    Frag<D> f[KT];
#pragma unroll
    for (int i = 0; i < 2 * KT; ++i) sc[i] = sc_next[i];
    scales(sc_next, base + step);
    ring.wait();
#pragma unroll
    for (int k = 0; k < KT; ++k) {
      ring.read_k(f[k], slot, k);
      products<D, NT>(c[k], f[k], qd);
#pragma unroll
      for (int n = 0; n < NT; ++n) fk[k][n] = sc[k] * qs[n];
      f[k].vs = sc[KT + k];
    }
    run.template weigh<KT, false>(c, fk, kBias, corr, 0u, t);
#pragma unroll
    for (int k = 0; k < KT; ++k) ring.read_v(f[k], slot, k);
    add_values<D, NT, KT, false>(run, f, c, corr, 0u);
    __syncwarp();                       // all lanes have read the slot
    const int ahead = base + kSlots * step;
    ring.start(slot, kv, ahead, ahead < whole, true, lane);
    slot = slot == kSlots - 1 ? 0 : slot + 1;
  }
  ring.drain();
  // The other closed tiles, and the tail's, one by one, from the last warp on.
  const int mine = cluster * W - 1 - (rank * W + warp);
  for (int tile = whole + mine; tile < tiles; tile += cluster * W) {
    Frag<D> one[1];
    kv.load_k(one[0], tile, g, t);
    kv.load_v(one[0], tile, g, t);
    float c[1][NT][4], fk[1][NT], corr[NT][2];
    const uint32_t hidden = hidden_in<NT>(tile * 16, last, t);
    products<D, NT>(c[0], one[0], qd);
#pragma unroll
    for (int n = 0; n < NT; ++n) fk[0][n] = one[0].ks * qs[n];
    run.template weigh<1, true>(c, fk, kBias, corr, hidden, t);
    add_values<D, NT, 1, true>(run, one, c, corr, hidden);
  }
  for (int i = mine; closed + 16 * i < lim; i += cluster * W)
    tail_tile<D, NT>(run, kv, q_row, a.scale, last, closed + 16 * i, total, g, t);

  // Join the warps, then the CTAs of the cluster.
  const float o_unit = run.ref * (1.0f / kPUp);
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    float l = run.l[n];
    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);
    if (t == 0) {
      part_m[warp * R + 8 * n + g] = run.m[n];
      part_l[warp * R + 8 * n + g] = l;
    }
#pragma unroll
    for (int e = 0; e < 2; ++e)
#pragma unroll
      for (int i = 0; i < D / 16; ++i)
        *reinterpret_cast<float2*>(part_o + warp * kRing + (8 * n + 2 * t + e) * D + D / 8 * g +
                                   2 * i) =
            make_float2(run.o[n][i][e] * o_unit, run.o[n][i][e + 2] * o_unit);
  }
  __syncthreads();
  // Four outputs of one row from `parts` partial sums.
  auto join = [](const float* m, const float* l, int ml_step, const float* o, int o_step,
                 int parts, float& M, float& L) {
    M = -INFINITY;
    L = 0.0f;
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int w = 0; w < parts; ++w) M = fmaxf(M, m[w * ml_step]);
    for (int w = 0; w < parts; ++w) {
      const float mw = m[w * ml_step], x = mw == -INFINITY ? 0.0f : ex2(mw - M);
      const float4 v = *reinterpret_cast<const float4*>(o + w * o_step);
      L = fmaf(l[w * ml_step], x, L);
      sum.x = fmaf(v.x, x, sum.x);
      sum.y = fmaf(v.y, x, sum.y);
      sum.z = fmaf(v.z, x, sum.z);
      sum.w = fmaf(v.w, x, sum.w);
    }
    return sum;
  };
  auto emit = [&](int e, float4 o, float M, float L) {
    const int row = r0 + e / D;
    if (row >= rows) return;
    const int64_t at = row_at(row);
    const float inv = 1.0f / L;
    *reinterpret_cast<float4*>(a.out + at * D + e % D) =
        make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
    if (a.lse && e % D == 0) a.lse[at] = (M + log2f(L)) * kLn2;
  };
  const int share = (R * D / 4 + cluster - 1) / cluster * 4;
  const float *m_of = part_m, *l_of = part_l;
  int parts = W;
  if (cluster > 1) {
    cg::cluster_group cl = cg::this_cluster();
    cluster_wait();                     // every CTA of the cluster has started
    for (int e = threadIdx.x * 4; e < R * D; e += blockDim.x * 4) {
      float M, L;
      const float4 o = join(part_m + e / D, part_l + e / D, R, part_o + e, kRing, W, M, L);
      *reinterpret_cast<float4*>(cl.map_shared_rank(recv_o, e / share) + rank * share +
                                 e % share) = o;
      if (e % D == 0)
        for (int k = 0; k < cluster; ++k) {
          cl.map_shared_rank(recv_m, k)[rank * R + e / D] = M;
          cl.map_shared_rank(recv_l, k)[rank * R + e / D] = L;
        }
    }
    cl.sync();
    m_of = recv_m;
    l_of = recv_l;
    parts = cluster;
  }
  const float* o_of = cluster > 1 ? recv_o : part_o;
  const int o_step = cluster > 1 ? share : kRing;
  for (int i = threadIdx.x * 4; i < share && rank * share + i < R * D; i += blockDim.x * 4) {
    const int e = rank * share + i;
    float M, L;
    const float4 o = join(m_of + e / D, l_of + e / D, R, o_of + i, o_step, parts, M, L);
    emit(e, o, M, L);
  }
  if (!a.weights || groups > 1) return;
  // The weights of this warp's keys, which are in a cache near by, now that
  // the sums are known.
  float z[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int r = 8 * n + g;
    float M = -INFINITY, L = 0.0f;
    for (int w = 0; w < parts; ++w) M = fmaxf(M, m_of[w * R + r]);
    for (int w = 0; w < parts; ++w) {
      const float mw = m_of[w * R + r];
      L = fmaf(l_of[w * R + r], mw == -INFINITY ? 0.0f : ex2(mw - M), L);
    }
    z[n] = M + log2f(L);
    if (r >= rows) last[n] = -1;        // sees nothing
  }
  float* w_out = a.weights + ((int64_t)b * Hkv + h) * S;
  // (the partial outputs in the ring have been read: every thread of the CTA
  // is past its share before the next copies)
  __syncthreads();
#pragma unroll
  for (int s = 0; s < kSlots; ++s)
    ring.start(s, kv, first + s * step, first + s * step < whole, false, lane);
  float had_next[KT] = {};
  auto had_of = [&](int base) {
    if (base >= whole) return;
#pragma unroll
    for (int k = 0; k < KT; ++k) had_next[k] = gathered(w_out, (base + k) * 16, len, g, t);
  };
  scales(sc_next, first);
  had_of(first);
  slot = 0;
  for (int base = first; base < whole; base += step) {
    float keep[KT], had[KT];
#pragma unroll
    for (int k = 0; k < KT; ++k) {
      keep[k] = sc_next[k];
      had[k] = had_next[k];
    }
    scales(sc_next, base + step);
    had_of(base + step);
    ring.wait();
#pragma unroll
    for (int k = 0; k < KT; ++k) {
      Frag<D> one;
      ring.read_k(one, slot, k);
      float c[1][NT][4], fk[1][NT], w[4] = {};
      products<D, NT>(c[0], one, qd);
#pragma unroll
      for (int n = 0; n < NT; ++n) fk[0][n] = keep[k] * qs[n];
      // (rows past the last see nothing, the others all of a whole group)
      add_weights<NT>(w, c, fk, kBias, z, hidden_in<NT>((base + k) * 16, last, t));
      put_weights(w_out, w, had[k], (base + k) * 16, total, g, t);
    }
    __syncwarp();
    const int ahead = base + kSlots * step;
    ring.start(slot, kv, ahead, ahead < whole, false, lane);
    slot = slot == kSlots - 1 ? 0 : slot + 1;
  }
  ring.drain();
  for (int tile = whole + mine; tile < tiles; tile += cluster * W) {
    Frag<D> one;
    const float had = gathered(w_out, tile * 16, len, g, t);
    kv.load_k(one, tile, g, t);
    float c[1][NT][4], fk[1][NT], w[4] = {};
    products<D, NT>(c[0], one, qd);
#pragma unroll
    for (int n = 0; n < NT; ++n) fk[0][n] = one.ks * qs[n];
    add_weights<NT>(w, c, fk, kBias, z, hidden_in<NT>(tile * 16, last, t));
    put_weights(w_out, w, had, tile * 16, total, g, t);
  }
  for (int i = mine; closed + 16 * i < lim; i += cluster * W) {
    const float had = gathered(w_out, closed + 16 * i, len, g, t);
    float c[1][NT][4], fk[1][NT], w[4] = {};
    tail_products<D, NT>(c, kv, q_row, a.scale, closed + 16 * i, total, g, t);
#pragma unroll
    for (int n = 0; n < NT; ++n) fk[0][n] = 1.0f;
    add_weights<NT>(w, c, fk, 0.0f, z, hidden_in<NT>(closed + 16 * i, last, t));
    put_weights(w_out, w, had, closed + 16 * i, total, g, t);
  }
}

// ---------------------------------------------------------------------------
// Weights for more rows: a warp keeps the keys of two 16-key tiles, the CTA
// turns 64 rows of q at a time into digits in shared memory, eight a warp.
template <int D>
__global__ void __launch_bounds__(256, D == 64 ? 2 : 1) kv8_weights_kernel(const AttnArgs a) {
  __shared__ uint32_t q_s[8][D / 32][4][2][32];
  __shared__ float qs_s[8][8], z_s[8][8];
  __shared__ int last_s[8][8];
  const int S = a.c.max_seq, G = a.Hq / a.c.kv_heads;
  const int bh = blockIdx.y, b = bh / a.c.kv_heads, h = bh % a.c.kv_heads;
  const int n_new = a.new_lens ? clamp_len(a.new_lens[b], a.T) : a.T;
  const int len = clamp_len(a.c.lens[b], S), total = min(len + n_new, S);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int j0 = blockIdx.x * 256;
  if (n_new == 0 || j0 >= total) return;
  const Keys<D> kv(a.c, bh);
  const int closed = total >> kv.shift << kv.shift;
  const int rows = n_new * G;
  Frag<D> f[2];
  float w[2][4] = {};
  auto jb = [&](int k) { return j0 + (warp * 2 + k) * 16; };
#pragma unroll
  for (int k = 0; k < 2; ++k)
    if (jb(k) < closed) kv.load_k(f[k], jb(k) >> 4, g, t);
  float* out = a.weights + (int64_t)bh * S;
  float had[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) had[k] = gathered(out, jb(k), len, g, t);
  auto row_at = [&](int r) {
    const int tk = a.div_g(r);
    return ((int64_t)b * a.T + tk) * a.Hq + h * G + (r - tk * G);
  };
  // rows of the tokens before the chunk's first key see none of it
  for (int r0 = max(0, j0 - len) * G / 64 * 64; r0 < rows; r0 += 64) {
    __syncthreads();
    {
      const int r = r0 + 8 * warp + g;
      const float* row = r < rows ? a.q + row_at(r) * D : nullptr;
      uint32_t qd[D / 32][4][2];
      float qs;
      load_q<D>(qd, qs, row, a.scale, t);
#pragma unroll
      for (int s = 0; s < D / 32; ++s)
#pragma unroll
        for (int d = 0; d < 4; ++d)
#pragma unroll
          for (int i = 0; i < 2; ++i) q_s[warp][s][d][i][lane] = qd[s][d][i];
      if (t == 0) {
        qs_s[warp][g] = qs;
        z_s[warp][g] = r < rows ? a.lse[row_at(r)] * kLog2e : 0.0f;
        last_s[warp][g] = r < rows ? min(len + a.div_g(r), total - 1) : -1;
      }
    }
    __syncthreads();
    for (int grp = 0; grp < 8 && r0 + 8 * grp < rows; ++grp) {
      uint32_t qd[1][D / 32][4][2];
#pragma unroll
      for (int s = 0; s < D / 32; ++s)
#pragma unroll
        for (int d = 0; d < 4; ++d)
#pragma unroll
          for (int i = 0; i < 2; ++i) qd[0][s][d][i] = q_s[grp][s][d][i][lane];
      const float qs = qs_s[grp][g], z[1] = {z_s[grp][g]};
      const int last[1] = {last_s[grp][g]};
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        if (jb(k) >= total) continue;
        float c[1][1][4], fk[1][1];
        if (jb(k) < closed) {
          products<D, 1>(c[0], f[k], qd);
          fk[0][0] = f[k].ks * qs;
          add_weights<1>(w[k], c, fk, kBias, z, hidden_in<1>(jb(k), last, t));
        } else {
          const int r = r0 + 8 * grp + g;
          const float* const row[1] = {r < rows ? a.q + row_at(r) * D : nullptr};
          tail_products<D, 1>(c, kv, row, a.scale, jb(k), total, g, t);
          fk[0][0] = 1.0f;
          add_weights<1>(w[k], c, fk, 0.0f, z, hidden_in<1>(jb(k), last, t));
        }
      }
    }
  }
#pragma unroll
  for (int k = 0; k < 2; ++k)
    put_weights(out, w[k], had[k], jb(k), total, g, t);
}

// From so many rows of a sequence and kv head on, tcgen05.  In us, this file's
// kernels against those, with weights, 4 kv heads:
//                                        64 rows     80 rows     128 rows
//   64 values a head, tokens in the cache
//     32 to 64, 1 sequence                18, 24      21, 25       29, 26
//     32 to 64, 32                        33, 26      42, 27       61, 27
//     300 to 1500, 4                      36, 34      41, 35       54, 35
//     300 to 1500, 32                     60, 74      74, 75      107, 75
//     16 thousand, 1                      47, 71      52, 72       76, 72
//     16 thousand, 32                    497, 635    702, 646     952, 653
//     100 thousand, 1                    185, 324    200, 328     293, 331
//   128 values a head
//     300 to 1500, 4                      49, 47      55, 48       77, 49
//     300 to 1500, 32                    117, 131    146, 133     210, 140
//     16 thousand, 1                      75, 109     86, 110     103, 112
//     16 thousand, 32                    978, 1331  1245, 1355   1798, 1399
// The two cross between 64 and 128 rows in all of these; one long sequence of 80 to
// 127 rows is where the rule costs most (its tcgen05 row tile is one, on 8 CTAs a
// kv head).
constexpr int kTcRows = 80;

template <int D, int NT>
int launch_few(cudaStream_t s, const AttnArgs& a) {
  constexpr int R = 8 * NT;
  const int groups = (int)ceil_div((int64_t)a.T * (a.Hq / a.c.kv_heads), R);
  const int64_t units = (int64_t)groups * a.c.kv_heads * a.c.batch;
  // Spread a sequence's keys over a CTA's warps, then over CTAs, while that does
  // not make more warps than are resident at a time (16 an SM) and a warp still
  // has a group of tiles.  64 sequences of 611 to 4095, 4 kv heads, with weights: 8
  // warps 45 us, 4 warps 53, 2 CTAs of 8 warps 48.  One of 131 thousand tokens: 1,
  // 2, 4, 8 CTAs 632, 321, 166, 88.  One of 45: 4 warps 4.9, 8 warps 5.2, 2 CTAs 6.1.
  const int steps = (int)ceil_div(a.c.max_seq, 16 * FewShape<D, NT>::KT);
  int W = 4, C = 1;
  while (W < kFewMaxWarps && units * W * 2 <= 16 * kNumSms && W * 2 <= steps) W *= 2;
  while (C < 8 && units * C * W * 2 <= 16 * kNumSms && C * W * 2 <= steps) C *= 2;
  const size_t smem = FewShape<D, NT>::smem(W);
  auto kern = attention_kv8_few_kernel<D, NT>;
  int rc;
  // (the most that any call asks for: the attribute is the function's, and another
  // thread's smaller one must not come between this one and the launch)
  if ((rc = check_cuda(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                            (int)FewShape<D, NT>::smem(kFewMaxWarps)),
                       "attention_kv8: smem attribute")))
    return rc;
  if ((int64_t)groups * a.c.kv_heads * kMaxCluster > INT32_MAX || a.c.batch > 65535)
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
  if (C == 8 && units * 10 <= FewShape<D, NT>::kBlocks * kNumSms) {
    // Few sequences: larger clusters, of as many CTAs as the GPU has room for
    // at a time (a cluster's SMs are neighbours: 8 clusters of 16 may not fit).
    // At one sequence of 131 thousand tokens, 8 kv heads of 128, 8 CTAs a head
    // take 88 us, 10 take 74.
    if ((rc = check_cuda(
             cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1),
             "attention_kv8: cluster attribute")))
      return rc;
    static const std::array<int, 4> most = [&] {
      std::array<int, 4> n = {};
      for (size_t i = 0; i < n.size(); ++i) {
        cudaLaunchConfig_t big = cfg;
        cudaLaunchAttribute size = attr[0];
        size.val.clusterDim.x = kBigClusters[i];
        big.attrs = &size;
        big.gridDim = dim3(kBigClusters[i]);
        if (cudaOccupancyMaxActiveClusters(&n[i], kern, &big)) cudaGetLastError();
      }
      return n;
    }();
    for (size_t i = 0; i < most.size() && C == 8; ++i)
      if (most[i] >= units && kBigClusters[i] * W <= steps) C = kBigClusters[i];
    attr[0].val.clusterDim.x = (unsigned)C;
    cfg.gridDim.x = (unsigned)(groups * a.c.kv_heads * C);
  }
  return check_cuda(cudaLaunchKernelEx(&cfg, kern, a, groups, C), "attention_kv8");
}

}  // namespace

int launch_attention_kv8(cudaStream_t s, int64_t* cnt, const float* q, const spx_kv8_cache* c,
                         const int32_t* new_lens, int T, int Hq, float scale, float* out,
                         float* lse, float* weights, int* slot) {
  int rc = kv8_check(c, "attention_kv8");
  if (rc) return rc;
  if (T <= 0 || Hq <= 0 || Hq % c->kv_heads)
    return fail(SPX_ERR_INVALID_ARGUMENT, "attention_kv8: bad shape");
  if (weights && !lse)
    return fail(SPX_ERR_INVALID_ARGUMENT, "attention_kv8: weights need an lse buffer");
  if (((uintptr_t)q & 15) || ((uintptr_t)out & 15))
    return fail(SPX_ERR_INVALID_ARGUMENT, "attention_kv8: q and out must be 16-byte aligned");
  const int64_t bh = (int64_t)c->batch * c->kv_heads;
  const uint64_t bytes = (uint64_t)c->batch * T * Hq * c->head_dim * 4;   // q is read to the end
  if ((uintptr_t)q < (uintptr_t)out + bytes && (uintptr_t)out < (uintptr_t)q + bytes)
    return fail(SPX_ERR_INVALID_ARGUMENT, "attention_kv8: q and out share memory");
  if ((int64_t)c->batch * T * Hq > INT32_MAX || bh > 65535)
    return fail(SPX_ERR_UNSUPPORTED, "attention_kv8: grid too large");
  const int G = Hq / c->kv_heads;
  const int64_t rows = (int64_t)T * G;
  if (rows * G > UINT32_MAX) return fail(SPX_ERR_UNSUPPORTED, "attention_kv8: too many rows");
  const uint32_t g_mul = G > 1 ? (uint32_t)(((1ull << 32) + G - 1) / G) : 0u;
  if (rows >= kTcRows && *slot < 0) *slot = at_slot_get();
  const AttnArgs a{q, *c, new_lens, T, Hq, g_mul, scale, out, lse, weights, *slot};
  const bool wide = rows > 8;
  // A group of rows that is alone adds its weights itself.
  const bool apart = rows > (c->head_dim == 64 ? 16 : 8);
  if (rows >= kTcRows)
    rc = launch_attention_kv8_tc(s, a);
  else if (c->head_dim == 64)
    rc = wide ? launch_few<64, 2>(s, a) : launch_few<64, 1>(s, a);
  else
    rc = launch_few<128, 1>(s, a);
  if (rc) return rc;
  if ((rc = after_launch(cnt, "attention_kv8")) || !weights || !apart) return rc;
  if (rows >= kTcRows) {
    if ((rc = launch_weights_kv8_tc(s, a))) return rc;
  } else {
    const dim3 wg((unsigned)ceil_div(c->max_seq, 256), (unsigned)bh);
    if (c->head_dim == 64)
      kv8_weights_kernel<64><<<wg, 256, 0, s>>>(a);
    else
      kv8_weights_kernel<128><<<wg, 256, 0, s>>>(a);
  }
  return after_launch(cnt, "attention_kv8: weights");
}

}  // namespace spx
