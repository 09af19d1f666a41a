// The 8-bit key / value cache: append, read-back and eviction
// (the attention over it is in k_attn_kv8.cu).
//
// A cache of `max_seq` slots per sequence and kv head is held in blocks of
// `block` tokens.  A full block is int8 with one fp32 scale per head for K
// and one for V; the block that is still open is fp32 ("tail", `block` rows),
// and is quantised once, when its last token arrives.  So what the cache
// holds depends on the tokens alone and not on how calls cut them, and no
// value is rounded to 8 bits twice on its way in.
//
//   full block:  s = max|x| / 127,  q = x / s rounded half to even,  value q s
//
// max|x| below 127 * 2^-126 (s would be subnormal) is held as zero.  A block
// with a NaN or an infinity gets that as its scale, so all of it reads back
// as NaN: the fault stays visible.
#include <cooperative_groups.h>

#include "attn_kv8.cuh"

namespace spx {
namespace {

namespace cg = cooperative_groups;

constexpr float kTinyAmax = 127.0f * 1.17549435e-38f;

// x / s rounded to the nearest whole number, halves to even, for s a normal
// number and |x| <= 127 s: the product with 1 / s can fall on the wrong side
// of a half, the remainder (exact in fp32: both terms are multiples of the
// smaller one's last place and the difference is at most s) tells.
__device__ __forceinline__ int round_div(float x, float s, float inv) {
  float q = rintf(x * inv);
  const float r = fmaf(-q, s, x), half = 0.5f * s;
  if (fabsf(r) >= half) {
    const bool odd = ((int)q) & 1;
    if (fabsf(r) > half || odd) q += r > 0.0f ? 1.0f : -1.0f;
  }
  return (int)fminf(fmaxf(q, -127.0f), 127.0f);
}

__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// Scale of a block (or row) whose largest magnitude has these bits: NaN sorts
// above infinity above every number.
__device__ __forceinline__ float scale_of(uint32_t amax_bits) {
  const float a = __uint_as_float(amax_bits);
  if (amax_bits >= 0x7f800000u) return a;
  return a < kTinyAmax ? 0.0f : a / 127.0f;
}
__device__ __forceinline__ bool usable(float s) { return s > 0.0f && s <= 3.4028234663852886e38f; }

struct KvView {
  int8_t* q8;     // int8 blocks of this (sequence, head)
  float* scale;
  float* tail;
};
__device__ __forceinline__ KvView view_of(const spx_kv8_cache& c, int b, int h, bool is_v) {
  const int64_t bh = (int64_t)b * c.kv_heads + h;
  KvView v;
  v.q8 = (is_v ? c.v : c.k) + bh * c.max_seq * c.head_dim;
  v.scale = (is_v ? c.v_scale : c.k_scale) + bh * (c.max_seq / c.block);
  v.tail = (is_v ? c.v_tail : c.k_tail) + bh * c.block * c.head_dim;
  return v;
}

// ---------------------------------------------------------------------------
// Append.  Grid: one CTA per new token rotates that token's queries; each
// other CTA takes one block of one (sequence, head, K or V).  A thread works on
// four values of a row's lower half and the four of the upper half that RoPE
// turns with them, and keeps its part of a block in registers between the
// block's largest magnitude and its rounding.  A row that does not start on 16
// bytes is read value by value.  16 prompts of 117 to 1000 tokens, 32 heads of 64 on
// 4 kv heads: 55 us for 172 MB, 26 at the rate of a copy.  20 thousand CTAs of one
// short chain each: a token's CTA loads cos and sin and two items a thread, rotates
// and ends; a block's waits for its maximum with nothing else to load.
constexpr int kAppendThreads = 256;

struct AppendArgs {
  const float* qkv;
  int64_t ld;
  const float* cos_t;
  const float* sin_t;
  int table_rows;
  const int32_t* pos;
  const int32_t* new_lens;
  int T, Hq;
  float* q_out;
  spx_kv8_cache c;
  int blocks;     // blocks that one sequence's new tokens may touch
  int q_ctas;     // batch * T
  int vec;        // qkv rows and tables on 16 bytes
};

// Values i .. i + 3 and half + i .. half + i + 3 of a row.
struct Pair {
  float lo[4], hi[4];
};
__device__ __forceinline__ Pair load_pair(const float* p, int i, int half, bool vec) {
  Pair v;
  if (vec) {
    const float4 a = __ldg(reinterpret_cast<const float4*>(p + i));
    const float4 b = __ldg(reinterpret_cast<const float4*>(p + half + i));
    v = {{a.x, a.y, a.z, a.w}, {b.x, b.y, b.z, b.w}};
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v.lo[e] = __ldg(p + i + e);
      v.hi[e] = __ldg(p + half + i + e);
    }
  }
  return v;
}
// x * cos + rotate_half(x) * sin, each product and the sum rounded once; a
// position outside the tables gives NaN.
struct Turn {
  Pair c, s;
};
__device__ __forceinline__ Turn load_turn(const AppendArgs& a, int p, int i, int half) {
  Turn t;
  if (p >= 0 && p < a.table_rows) {
    t.c = load_pair(a.cos_t + (int64_t)p * 2 * half, i, half, a.vec);
    t.s = load_pair(a.sin_t + (int64_t)p * 2 * half, i, half, a.vec);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      t.c.lo[e] = t.c.hi[e] = t.s.lo[e] = t.s.hi[e] = __int_as_float(0x7fc00000);
  }
  return t;
}
__device__ __forceinline__ Pair turned(const Pair& x, const Turn& t) {
  Pair y;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    y.lo[e] = __fadd_rn(__fmul_rn(x.lo[e], t.c.lo[e]), __fmul_rn(-x.hi[e], t.s.lo[e]));
    y.hi[e] = __fadd_rn(__fmul_rn(x.hi[e], t.c.hi[e]), __fmul_rn(x.lo[e], t.s.hi[e]));
  }
  return y;
}
__device__ __forceinline__ void store_pair(float* p, int i, int half, const Pair& v) {
  *reinterpret_cast<float4*>(p + i) = make_float4(v.lo[0], v.lo[1], v.lo[2], v.lo[3]);
  *reinterpret_cast<float4*>(p + half + i) = make_float4(v.hi[0], v.hi[1], v.hi[2], v.hi[3]);
}
__device__ __forceinline__ char4 round4(const float (&x)[4], float s, float inv) {
  return make_char4((signed char)round_div(x[0], s, inv), (signed char)round_div(x[1], s, inv),
                    (signed char)round_div(x[2], s, inv), (signed char)round_div(x[3], s, inv));
}

// IPT: the items (eighths of a row of 64, sixteenths of 128) of a block that a
// thread holds.
template <int IPT>
__global__ void __launch_bounds__(kAppendThreads) rope_kv8_append_kernel(const AppendArgs a) {
  __shared__ uint32_t warp_max[kAppendThreads / 32];
  const int D = a.c.head_dim, half = D >> 1, Hkv = a.c.kv_heads, blk = a.c.block, T = a.T;
  const int per_row = D >> 3, log_items = 31 - __clz(per_row);
  if ((int)blockIdx.x < a.q_ctas) {
    const int b = blockIdx.x / T, tk = blockIdx.x - b * T;
    if (a.new_lens && tk >= a.new_lens[b]) return;
    const int i = (threadIdx.x & (per_row - 1)) * 4;   // the same for each of its heads
    const Turn turn = load_turn(a, a.pos[b] + tk, i, half);
    const float* src = a.qkv + (int64_t)blockIdx.x * a.ld;
    float* dst = a.q_out + (int64_t)blockIdx.x * a.Hq * D;
    for (int h = threadIdx.x >> log_items; h < a.Hq; h += kAppendThreads >> log_items)
      store_pair(dst + (int64_t)h * D, i, half,
                 turned(load_pair(src + (int64_t)h * D, i, half, a.vec), turn));
    return;
  }
  int w = (int)blockIdx.x - a.q_ctas;
  const int wb = w % a.blocks;
  w /= a.blocks;
  const bool is_v = w & 1;
  w >>= 1;
  const int h = w % Hkv, b = w / Hkv;
  const int n = a.new_lens ? clamp_len(a.new_lens[b], T) : T;
  const int len = clamp_len(a.c.lens[b], a.c.max_seq);
  const int total = min(len + n, a.c.max_seq);
  const int blk_i = len / blk + wb;            // from the block that is open before the call
  const int lo = blk_i * blk;
  if (n == 0 || lo >= total) return;
  const KvView kv = view_of(a.c, b, h, is_v);
  const float* src = a.qkv + (int64_t)b * T * a.ld + (int64_t)(a.Hq + (is_v ? Hkv : 0) + h) * D;
  const int pos = a.pos[b];
  auto fresh = [&](int slot, int i) {
    const int tk = slot - len;
    const Pair x = load_pair(src + tk * a.ld, i, half, a.vec);
    return is_v ? x : turned(x, load_turn(a, pos + tk, i, half));
  };
  auto to_tail = [&](int from, int to) {       // new tokens of an open block
    for (int e = threadIdx.x; e < (to - from) * per_row; e += kAppendThreads) {
      const int slot = from + (e >> log_items), i = (e & (per_row - 1)) * 4;
      store_pair(kv.tail + (slot & (blk - 1)) * D, i, half, fresh(slot, i));
    }
  };
  if (lo + blk > total) {
    // Open.  Where it is not the block that was open before, the CTA of that
    // block writes it, after it has read the tail.
    if (wb == 0) to_tail(max(lo, len), total);
    return;
  }
  Pair x[IPT];
  uint32_t mx = 0;
  const int items = blk * per_row;
#pragma unroll
  for (int k = 0; k < IPT; ++k) {
    const int e = threadIdx.x + k * kAppendThreads;
    if (e < items) {
      const int r = e >> log_items, i = (e & (per_row - 1)) * 4, slot = lo + r;
      if (slot < len) {   // not __ldg: this CTA writes the tail further down
        const float4 p = *reinterpret_cast<const float4*>(kv.tail + r * D + i);
        const float4 q = *reinterpret_cast<const float4*>(kv.tail + r * D + half + i);
        x[k] = {{p.x, p.y, p.z, p.w}, {q.x, q.y, q.z, q.w}};
      } else {
        x[k] = fresh(slot, i);
      }
#pragma unroll
      for (int f = 0; f < 4; ++f) mx = max(mx, max(abs_bits(x[k].lo[f]), abs_bits(x[k].hi[f])));
    }
  }
  mx = __reduce_max_sync(0xffffffffu, mx);
  if ((threadIdx.x & 31) == 0) warp_max[threadIdx.x >> 5] = mx;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kAppendThreads / 32; ++i) mx = max(mx, warp_max[i]);
  const float s = scale_of(mx);
  const bool ok = usable(s);
  const float inv = ok ? 1.0f / s : 0.0f;
  if (threadIdx.x == 0) kv.scale[blk_i] = s;
#pragma unroll
  for (int k = 0; k < IPT; ++k) {
    const int e = threadIdx.x + k * kAppendThreads;
    if (e < items) {
      const int i = (e & (per_row - 1)) * 4;
      int8_t* out = kv.q8 + (int64_t)(lo + (e >> log_items)) * D;
      const char4 zero = make_char4(0, 0, 0, 0);
      *reinterpret_cast<char4*>(out + i) = ok ? round4(x[k].lo, s, inv) : zero;
      *reinterpret_cast<char4*>(out + half + i) = ok ? round4(x[k].hi, s, inv) : zero;
    }
  }
  if (wb == 0) {
    const int open = total / blk * blk;
    if (open > lo && open < total) to_tail(open, total);
  }
}

// ---------------------------------------------------------------------------
// Read-back of `count` slots from starts[b] on, as fp32; 0 behind the end.  A
// CTA per 4096 values of one (sequence, head, K or V), 8 a thread at a time.
// Bound by the bytes it writes: 64 sequences of 2048, 4 kv heads of 64: 62 us,
// 5.4 TB/s (74 with four values a thread and conversion instructions).
constexpr int kReadValues = 4096;

__global__ void __launch_bounds__(256)
    kv8_read_kernel(const spx_kv8_cache c, const int32_t* __restrict__ new_lens, int q_len,
                    const int32_t* __restrict__ starts, int count, int chunks,
                    float* __restrict__ k_out, float* __restrict__ v_out) {
  const int D = c.head_dim, blk = c.block, shift = 31 - __clz(D);
  int u = blockIdx.x / chunks;
  const int chunk = blockIdx.x - u * chunks;
  const bool is_v = u & 1;
  u >>= 1;
  const int b = u / c.kv_heads, h = u - b * c.kv_heads;
  const int n = new_lens ? clamp_len(new_lens[b], q_len) : q_len;
  const int len = add_len(clamp_len(c.lens[b], c.max_seq), n, c.max_seq);
  const int closed = len / blk * blk;
  const int64_t start = starts ? starts[b] : 0;
  const KvView kv = view_of(c, b, h, is_v);
  float* out = (is_v ? v_out : k_out) + (int64_t)u * count * D;
  const int64_t all = (int64_t)count * D;
  constexpr int N = kReadValues / 2048;
  const int blk_shift = 31 - __clz(blk), d = threadIdx.x * 8 & (D - 1);
  const int64_t e0 = (int64_t)chunk * kReadValues + threadIdx.x * 8;
  uint2 q[N];
  float s[N];
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const int64_t e = e0 + k * 2048, slot = start + (e >> shift);
    q[k] = make_uint2(0x80808080u, 0x80808080u);
    s[k] = 0.0f;
    if (e < all && slot >= 0 && slot < closed) {
      q[k] = __ldg(reinterpret_cast<const uint2*>(kv.q8 + slot * D + d));
      q[k] = make_uint2(q[k].x ^ 0x80808080u, q[k].y ^ 0x80808080u);
      s[k] = __ldg(kv.scale + (slot >> blk_shift));
    }
  }
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const int64_t e = e0 + k * 2048, slot = start + (e >> shift);
    if (e >= all) continue;
    float4* to = reinterpret_cast<float4*>(out + e);
    if (slot >= closed && slot < len) {
      const float4* x =
          reinterpret_cast<const float4*>(kv.tail + (slot & (blk - 1)) * D + d);
      __stcs(to, __ldg(x));
      __stcs(to + 1, __ldg(x + 1));
      continue;
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t w = i ? q[k].y : q[k].x;
      float2 v[2];
#pragma unroll
      for (int j = 0; j < 2; ++j)          // 0x4b000000 | (value + 128) is 2^23 + 128 + value
        v[j] = mul2(add2(make_float2(__uint_as_float(__byte_perm(w, 0x4b000000u, 0x7550 | 2 * j)),
                                     __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7551 | 2 * j))),
                         make_float2(-8388736.0f, -8388736.0f)),
                    make_float2(s[k], s[k]));
      __stcs(to + i, make_float4(v[0].x, v[0].y, v[1].x, v[1].y));
    }
  }
}

// ---------------------------------------------------------------------------
// Eviction, part 1: which slots stay.  One CTA per (sequence, head).  The
// first `sink` and the last `recent` slots stay; of those between, the ones
// with the largest weight: their smallest key T by a radix select of four
// 8-bit digits, then every key above T and the first ones equal to it, in
// slot order.  Each warp owns a contiguous part of the slots, so two sweeps
// with ballots give every slot its place.
constexpr int kSelThreads = 1024;

// Order-preserving bits; NaN below everything, -0 equal to +0.
__device__ __forceinline__ uint32_t order_key(float w) {
  if (w != w) return 0u;
  const uint32_t u = __float_as_uint(w + 0.0f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

__global__ void __launch_bounds__(kSelThreads)
    kv8_select_kernel(const float* __restrict__ weights, const int32_t* __restrict__ lens, int Hkv,
                      int max_seq, int keep, int recent, int sink, int32_t* __restrict__ idx) {
  __shared__ uint32_t hist[256];
  __shared__ uint32_t prefix_s, need_s;
  __shared__ int gt_c[32], eq_c[32];
  const int bh = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int n = clamp_len(lens[bh / Hkv], max_seq);
  const float* w = weights + (int64_t)bh * max_seq;
  int32_t* out = idx + (int64_t)bh * keep;
  if (n <= keep) {
    for (int i = tid; i < keep; i += blockDim.x) out[i] = i < n ? i : -1;
    return;
  }
  const int need = keep - sink - recent, m0 = sink, m1 = n - recent;
  for (int i = tid; i < sink; i += blockDim.x) out[i] = i;
  for (int i = tid; i < recent; i += blockDim.x) out[sink + need + i] = m1 + i;
  if (need == 0) return;
  uint32_t prefix = 0, left = (uint32_t)need;
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int i = tid; i < 256; i += blockDim.x) hist[i] = 0;
    __syncthreads();
    for (int j = m0 + tid; j < m1; j += blockDim.x) {
      const uint32_t key = order_key(w[j]);
      if (shift == 24 || (key >> (shift + 8)) == (prefix >> (shift + 8)))
        atomicAdd(&hist[(key >> shift) & 255u], 1u);
    }
    __syncthreads();
    if (warp == 0) {
      // lane l sums bins 255 - 8 l .. 248 - 8 l, from the top down
      uint32_t c[8], s = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        c[i] = hist[255 - 8 * lane - i];
        s += c[i];
      }
      uint32_t inc = s;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t v = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += v;
      }
      uint32_t before = inc - s;
      if (before < left && left <= inc) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (before < left && left <= before + c[i]) {
            prefix_s = prefix | ((uint32_t)(255 - 8 * lane - i) << shift);
            need_s = left - before;
          }
          before += c[i];
        }
      }
    }
    __syncthreads();
    prefix = prefix_s;
    left = need_s;
  }
  // `left` slots with key == prefix stay, the first ones.
  const int span = ((m1 - m0 + 31) / 32 + 31) / 32 * 32;
  const int j0 = m0 + warp * span, j1 = min(j0 + span, m1);
  int gt = 0, eq = 0;
  for (int j = j0; j < j1; j += 32) {
    const uint32_t key = j + lane < j1 ? order_key(w[j + lane]) : 0u;
    const bool in = j + lane < j1;
    gt += __popc(__ballot_sync(0xffffffffu, in && key > prefix));
    eq += __popc(__ballot_sync(0xffffffffu, in && key == prefix));
  }
  if (lane == 0) {
    gt_c[warp] = gt;
    eq_c[warp] = eq;
  }
  __syncthreads();
  gt = 0;
  eq = 0;
  for (int i = 0; i < warp; ++i) {
    gt += gt_c[i];
    eq += eq_c[i];
  }
  const uint32_t below = (1u << lane) - 1u;
  for (int j = j0; j < j1; j += 32) {
    const bool in = j + lane < j1;
    const uint32_t key = in ? order_key(w[j + lane]) : 0u;
    const uint32_t bg = __ballot_sync(0xffffffffu, in && key > prefix);
    const uint32_t be = __ballot_sync(0xffffffffu, in && key == prefix);
    const int eq_before = eq + __popc(be & below);
    const bool take = in && (key > prefix || (key == prefix && eq_before < (int)left));
    if (take) out[sink + gt + __popc(bg & below) + min(eq_before, (int)left)] = j + lane;
    gt += __popc(bg);
    eq += __popc(be);
  }
}

// Part 2: the kept rows to the front, in order.  A full block of the result
// takes the largest scale of its members' (a row of the tail has the scale it
// would have alone) and rounds each value to it once; members with that scale
// keep their 8 bits.  A cluster of CTAs moves one (sequence, head, K or V), in
// chunks of 256 rows a CTA: all of a chunk into registers, a cluster barrier,
// then out.  Slot i of the result comes from a slot >= i, so in that order it
// also works in place, without a second buffer (into another there is no cluster
// barrier).  64 sequences of 1500 to 4096 cut to 2048, 4 kv heads of 64: 70 us
// into another cache, 92 in place, for 134 MB, 20 at the rate of a copy (clusters
// of 4 and 2 took 73 and 75 when the first took 75).  A chunk a CTA at a time is a
// chain of loads (slot, scale, row) and barriers between them, with nothing else
// in flight, and then the instructions of values that are rounded again.
constexpr int kGatherRows = 256;

// The int8 value nearest to q s / ns, halves to even, for |q s| <= 127 ns.
// ratio + rest = s / ns to 2^-48; a quotient that is no half is at least
// 2^-32 away from one.
__device__ __forceinline__ int requant(int q, float ratio, float rest) {
  const float fq = (float)q, p = fq * ratio;
  float k = rintf(p);
  const float e = fmaf(fq, rest, fmaf(fq, ratio, -p));
  const float dir = p - k + e >= 0.0f ? 1.0f : -1.0f;
  const float over = dir * ((p - k) - 0.5f * dir) + dir * e;   // past the half, if positive
  if (over > 0x1p-36f || (over >= -0x1p-36f && ((int)k & 1))) k += dir;
  return (int)k;
}

// Four values at once.  The product with the rounded ratio is within 2^-16 of
// the quotient: away from the halves it rounds as the quotient does.
__device__ __forceinline__ uint32_t requant4(uint32_t w, float ratio, float rest) {
  uint32_t r[4];
  float worst = 0.0f;
  const uint32_t x = w ^ 0x80808080u;
  const float2 by = make_float2(ratio, ratio);
#pragma unroll
  for (int i = 0; i < 4; i += 2) {
    // bytes to fp32: 0x4b000000 | (q + 128) is 2^23 + 128 + q
    const float2 q = add2(make_float2(__uint_as_float(__byte_perm(x, 0x4b000000u, 0x7550 | i)),
                                      __uint_as_float(__byte_perm(x, 0x4b000000u, 0x7551 | i))),
                          make_float2(-8388736.0f, -8388736.0f));
    // 1.5 2^23: rounds to a whole, half to even
    const float2 k = fma2(q, by, make_float2(12582912.0f, 12582912.0f));
    r[i] = __float_as_uint(k.x);
    r[i + 1] = __float_as_uint(k.y);
    const float2 whole = add2(k, make_float2(-12582912.0f, -12582912.0f));
    const float2 off = fma2(q, by, make_float2(-whole.x, -whole.y));
    worst = fmaxf(worst, fmaxf(fabsf(off.x), fabsf(off.y)));
  }
  if (worst > 0.4999f) {
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = (uint32_t)requant((int8_t)(w >> (8 * i)), ratio, rest);
  }
  return __byte_perm(__byte_perm(r[0], r[1], 0x0040), __byte_perm(r[2], r[3], 0x0040), 0x5410);
}

template <int D>
__global__ void __launch_bounds__(kGatherRows)
    kv8_gather_kernel(const spx_kv8_cache src, const spx_kv8_cache dst, const float* w_src,
                      float* w_dst, const int32_t* __restrict__ idx, int keep, int in_place,
                      int cluster) {
  constexpr int P = D / 16;                    // 16-byte pieces of a row
  extern __shared__ __align__(16) float open_rows[];   // [block][D], the open block
  __shared__ float row_scale[kGatherRows];
  __shared__ int row_src[kGatherRows];
  __shared__ uint32_t blk_scale[kGatherRows / 16];
  __shared__ float2 row_by[kGatherRows];       // the new scale into the row's: ratio, rest
  const int blk = src.block, shift = 31 - __clz(blk);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = blockIdx.x % cluster, unit = blockIdx.x / cluster;
  const int bh = unit >> 1, b = bh / src.kv_heads, h = bh % src.kv_heads;
  const bool is_v = unit & 1;
  const int n = clamp_len(src.lens[b], src.max_seq);
  const int kept = min(n, keep), full = kept >> shift << shift;
  if (in_place && n <= keep) return;           // the whole cluster
  const KvView s = view_of(src, b, h, is_v), d = view_of(dst, b, h, is_v);
  const int closed = n >> shift << shift;
  const int32_t* from = idx + (int64_t)bh * keep;
  for (int base = 0; base < kept; base += cluster * kGatherRows) {
    const int lo = base + rank * kGatherRows;  // this CTA's rows, whole blocks
    const int rows = max(0, min(full - lo, kGatherRows));
    float wv = 0.0f;
    const bool has_w = !is_v && lo + tid < kept;
    if (tid < kGatherRows / 16) blk_scale[tid] = 0;
    __syncthreads();
    int j = 0;
    bool in_tail = false;
    if (lo + tid < kept) j = from[lo + tid];
    if (has_w) wv = w_src[(int64_t)bh * src.max_seq + j];
    if (tid < rows) {
      row_src[tid] = j;
      in_tail = j >= closed;
      if (!in_tail) {
        const float sc = s.scale[j >> shift];
        row_scale[tid] = sc;
        atomicMax(&blk_scale[tid >> shift], abs_bits(sc));
      }
    }
    for (uint32_t todo = __ballot_sync(0xffffffffu, in_tail); todo; todo &= todo - 1) {
      const int r = warp * 32 + __ffs(todo) - 1;
      const int jr = __shfl_sync(0xffffffffu, j, r & 31);
      uint32_t mx = 0;
#pragma unroll
      for (int e = 0; e < D; e += 32)
        mx = max(mx, abs_bits(s.tail[(jr & (blk - 1)) * D + e + lane]));
      const float sc = scale_of(__reduce_max_sync(0xffffffffu, mx));
      if (lane == 0) {
        row_scale[r] = sc;
        atomicMax(&blk_scale[r >> shift], abs_bits(sc));
      }
    }
    __syncthreads();
    uint4 out[P];
#pragma unroll
    for (int k = 0; k < P; ++k) {
      const int e = tid + k * kGatherRows, r = e / P, at = (e % P) * 16;
      out[k] = make_uint4(0, 0, 0, 0);
      if (r < rows && row_src[r] < closed)
        out[k] = *reinterpret_cast<const uint4*>(s.q8 + (int64_t)row_src[r] * D + at);
    }
    if (tid < rows) {
      // (far from subnormal remainders)
      const float ns = __uint_as_float(blk_scale[tid >> shift]), sc = row_scale[tid];
      const float up = ns < 0x1p-60f ? 0x1p64f : 1.0f, sn = sc * up, nn = ns * up;
      const float ratio = sn / nn;
      row_by[tid] = make_float2(ratio, fmaf(-ratio, nn, sn) / nn);
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < P; ++k) {
      const int e = tid + k * kGatherRows, r = e / P, at = (e % P) * 16;
      if (r >= rows) continue;
      const float ns = __uint_as_float(blk_scale[r >> shift]);
      uint32_t* o = reinterpret_cast<uint32_t*>(&out[k]);
      if (!usable(ns)) {
        out[k] = make_uint4(0, 0, 0, 0);
      } else if (row_src[r] >= closed) {
        const float* x = s.tail + (row_src[r] & (blk - 1)) * D + at;
        const float inv = 1.0f / ns;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float4 v = *reinterpret_cast<const float4*>(x + 4 * i);
          const char4 q = make_char4(
              (signed char)round_div(v.x, ns, inv), (signed char)round_div(v.y, ns, inv),
              (signed char)round_div(v.z, ns, inv), (signed char)round_div(v.w, ns, inv));
          o[i] = *reinterpret_cast<const uint32_t*>(&q);
        }
      } else if (row_by[r].x != 1.0f) {        // (of 1, each value is its own quotient)
        const float2 by = row_by[r];
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = requant4(o[i], by.x, by.y);
      }
    }
    if (in_place) {
      if (cluster > 1)
        cg::this_cluster().sync();
      else
        __syncthreads();
    }
    if (has_w) w_dst[(int64_t)bh * dst.max_seq + lo + tid] = wv;
    if (tid < rows && (tid & (blk - 1)) == 0)
      d.scale[(lo + tid) >> shift] = __uint_as_float(blk_scale[tid >> shift]);
#pragma unroll
    for (int k = 0; k < P; ++k) {
      const int e = tid + k * kGatherRows;
      if (e / P < rows)
        *reinterpret_cast<uint4*>(d.q8 + (int64_t)lo * D + (int64_t)e * 16) = out[k];
    }
    __syncthreads();
  }
  // The open block, by one CTA: every row that others take from the tail has
  // been read by now.
  if (rank != 0 || full == kept) return;
  for (int e = tid; e < (kept - full) * D; e += kGatherRows) {
    const int j = from[full + e / D], x = e % D;
    open_rows[e] = j < closed ? s.q8[(int64_t)j * D + x] * s.scale[j >> shift]
                              : s.tail[(j & (blk - 1)) * D + x];
  }
  __syncthreads();
  for (int e = tid; e < (kept - full) * D; e += kGatherRows) d.tail[e] = open_rows[e];
}

__global__ void kv8_advance_kernel(int32_t* lens, int32_t* pos, const int32_t* new_lens, int batch,
                                   int q_len, int limit) {
  for (int b = blockIdx.x * blockDim.x + threadIdx.x; b < batch; b += gridDim.x * blockDim.x) {
    const int n = new_lens ? clamp_len(new_lens[b], q_len) : q_len;
    if (lens) lens[b] = add_len(clamp_len(lens[b], limit), n, limit);
    if (pos) pos[b] += n;
  }
}

bool al16(const void* p) { return ((uintptr_t)p & 15) == 0; }

}  // namespace

int kv8_check(const spx_kv8_cache* c, const char* what) {
  if (!c || !c->k || !c->v || !c->k_scale || !c->v_scale || !c->k_tail || !c->v_tail || !c->lens)
    return fail(SPX_ERR_INVALID_ARGUMENT, "%s: null cache buffer", what);
  if (c->batch <= 0 || c->kv_heads <= 0 || c->max_seq <= 0)
    return fail(SPX_ERR_INVALID_ARGUMENT, "%s: bad cache shape", what);
  if (c->head_dim != 64 && c->head_dim != 128)
    return fail(SPX_ERR_UNSUPPORTED, "%s: head_dim must be 64 or 128", what);
  if (c->block != 16 && c->block != 32 && c->block != 64 && c->block != 128)
    return fail(SPX_ERR_UNSUPPORTED, "%s: block must be 16, 32, 64 or 128", what);
  if (c->max_seq % c->block)
    return fail(SPX_ERR_INVALID_ARGUMENT, "%s: max_seq %d is not a whole number of blocks", what,
                c->max_seq);
  if (c->max_seq > (1 << 30) || (int64_t)c->batch * c->kv_heads > (1 << 20))
    return fail(SPX_ERR_UNSUPPORTED, "%s: cache too large", what);
  if (!al16(c->k) || !al16(c->v) || !al16(c->k_tail) || !al16(c->v_tail))
    return fail(SPX_ERR_INVALID_ARGUMENT, "%s: cache buffers must be 16-byte aligned", what);
  return SPX_OK;
}

int launch_rope_kv8_append(cudaStream_t s, int64_t* cnt, const float* qkv, int64_t ld_qkv,
                           const float* cos_t, const float* sin_t, int table_rows,
                           const int32_t* pos, const int32_t* new_lens, int T, int Hq,
                           float* q_out, const spx_kv8_cache* c) {
  int rc = kv8_check(c, "rope_kv8_append");
  if (rc) return rc;
  if (T <= 0 || Hq <= 0 || table_rows <= 0 ||
      ld_qkv < (int64_t)(Hq + 2 * c->kv_heads) * c->head_dim)
    return fail(SPX_ERR_INVALID_ARGUMENT, "rope_kv8_append: bad shape");
  if (!al16(q_out))
    return fail(SPX_ERR_INVALID_ARGUMENT, "rope_kv8_append: q_out must be 16-byte aligned");
  const uint64_t rows = (uint64_t)c->batch * T, row = (uint64_t)(Hq + 2 * c->kv_heads) * c->head_dim;
  const uintptr_t in = (uintptr_t)qkv, out = (uintptr_t)q_out;   // one's rows, others still read
  if (in < out + rows * Hq * c->head_dim * 4 && out < in + ((rows - 1) * ld_qkv + row) * 4)
    return fail(SPX_ERR_INVALID_ARGUMENT, "rope_kv8_append: qkv and q_out share memory");
  AppendArgs a;
  a.qkv = qkv;
  a.ld = ld_qkv;
  a.cos_t = cos_t;
  a.sin_t = sin_t;
  a.table_rows = table_rows;
  a.pos = pos;
  a.new_lens = new_lens;
  a.T = T;
  a.Hq = Hq;
  a.q_out = q_out;
  a.c = *c;
  // the open block and what follows
  const int64_t blocks = ((int64_t)T + 2 * c->block - 2) / c->block;
  const int64_t q_ctas = (int64_t)c->batch * T;
  const int64_t grid = q_ctas + (int64_t)c->batch * c->kv_heads * 2 * blocks;
  if (grid > INT32_MAX) return fail(SPX_ERR_UNSUPPORTED, "rope_kv8_append: grid too large");
  a.blocks = (int)blocks;
  a.q_ctas = (int)q_ctas;
  a.vec = al16(qkv) && ld_qkv % 4 == 0 && al16(cos_t) && al16(sin_t);
  const int items = c->block * c->head_dim / 8;
  if (items <= kAppendThreads)
    rope_kv8_append_kernel<1><<<(int)grid, kAppendThreads, 0, s>>>(a);
  else if (items == 2 * kAppendThreads)
    rope_kv8_append_kernel<2><<<(int)grid, kAppendThreads, 0, s>>>(a);
  else if (items == 4 * kAppendThreads)
    rope_kv8_append_kernel<4><<<(int)grid, kAppendThreads, 0, s>>>(a);
  else
    rope_kv8_append_kernel<8><<<(int)grid, kAppendThreads, 0, s>>>(a);
  return after_launch(cnt, "rope_kv8_append");
}

int launch_kv8_read(cudaStream_t s, int64_t* cnt, const spx_kv8_cache* c, const int32_t* new_lens,
                    int q_len, const int32_t* starts, int count, float* k_out, float* v_out) {
  int rc = kv8_check(c, "kv8_read");
  if (rc) return rc;
  if (q_len < 0 || count <= 0) return fail(SPX_ERR_INVALID_ARGUMENT, "kv8_read: bad shape");
  if (!al16(k_out) || !al16(v_out))
    return fail(SPX_ERR_INVALID_ARGUMENT, "kv8_read: outputs must be 16-byte aligned");
  const int64_t chunks = ceil_div((int64_t)count * c->head_dim, kReadValues);
  const int64_t grid = (int64_t)c->batch * c->kv_heads * 2 * chunks;
  if (grid > INT32_MAX) return fail(SPX_ERR_UNSUPPORTED, "kv8_read: grid too large");
  kv8_read_kernel<<<(int)grid, 256, 0, s>>>(*c, new_lens, q_len, starts, count, (int)chunks, k_out,
                                            v_out);
  return after_launch(cnt, "kv8_read");
}

int launch_kv8_evict(cudaStream_t s, int64_t* cnt, const spx_kv8_cache* src, const float* weights,
                     int keep, int recent, int sink, int32_t* idx, const spx_kv8_cache* dst,
                     float* dst_weights) {
  int rc = kv8_check(src, "kv8_evict");
  if (!rc) rc = kv8_check(dst, "kv8_evict");
  if (rc) return rc;
  if (keep <= 0 || recent < 0 || sink < 0 || recent > keep || sink > keep - recent)
    return fail(SPX_ERR_INVALID_ARGUMENT, "kv8_evict: sink + recent must fit in keep");
  if (keep > dst->max_seq || src->batch != dst->batch || src->kv_heads != dst->kv_heads ||
      src->head_dim != dst->head_dim || src->block != dst->block)
    return fail(SPX_ERR_INVALID_ARGUMENT, "kv8_evict: the two caches do not fit each other");
  // Either the same cache or nothing in common.
  const int64_t bh = (int64_t)src->batch * src->kv_heads;
  const bool same = src->k == dst->k && src->v == dst->v && src->k_scale == dst->k_scale &&
                    src->v_scale == dst->v_scale && src->k_tail == dst->k_tail &&
                    src->v_tail == dst->v_tail && weights == dst_weights &&
                    src->max_seq == dst->max_seq;
  if (!same) {
    auto span = [&](const spx_kv8_cache* c, const float* w, int i, const char** p, int64_t* n) {
      const int64_t q = bh * c->max_seq * c->head_dim, sc = bh * (c->max_seq / c->block) * 4,
                    t = bh * c->block * c->head_dim * 4;
      const void* ps[7] = {c->k, c->v, c->k_scale, c->v_scale, c->k_tail, c->v_tail, w};
      const int64_t ns[7] = {q, q, sc, sc, t, t, bh * c->max_seq * 4};
      *p = (const char*)ps[i];
      *n = ns[i];
    };
    for (int i = 0; i < 7; ++i)
      for (int j = 0; j < 7; ++j) {
        const char *p, *q;
        int64_t np, nq;
        span(src, weights, i, &p, &np);
        span(dst, dst_weights, j, &q, &nq);
        if (p < q + nq && q < p + np)
          return fail(SPX_ERR_INVALID_ARGUMENT,
                      "kv8_evict: source and result overlap without being the same cache");
      }
  }
  kv8_select_kernel<<<(int)bh, kSelThreads, 0, s>>>(weights, src->lens, src->kv_heads,
                                                    src->max_seq, keep, recent, sink, idx);
  if ((rc = after_launch(cnt, "kv8_evict: select"))) return rc;
  // CTAs enough to take all kept rows at once, a portable cluster at most.
  int cluster = 1;
  while (cluster < 8 && cluster * kGatherRows < keep) cluster *= 2;
  if (2 * bh * cluster > INT32_MAX) return fail(SPX_ERR_UNSUPPORTED, "kv8_evict: grid too large");
  const size_t smem = (size_t)src->block * src->head_dim * sizeof(float);
  auto kern = src->head_dim == 64 ? kv8_gather_kernel<64> : kv8_gather_kernel<128>;
  if (smem > 40 * 1024) {
    rc = check_cuda(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         (int)smem),
                    "kv8_evict: smem attribute");
    if (rc) return rc;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(2 * bh * cluster));
  cfg.blockDim = dim3(kGatherRows);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)cluster;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  rc = check_cuda(cudaLaunchKernelEx(&cfg, kern, *src, *dst, weights, dst_weights,
                                     (const int32_t*)idx, keep, same ? 1 : 0, cluster),
                  "kv8_evict: gather");
  return rc ? rc : after_launch(cnt, "kv8_evict: gather");
}

int launch_kv8_advance(cudaStream_t s, int64_t* cnt, int32_t* lens, int32_t* pos,
                       const int32_t* new_lens, int batch, int q_len, int limit) {
  if (batch <= 0 || q_len < 0 || limit <= 0)
    return fail(SPX_ERR_INVALID_ARGUMENT, "kv8_advance: bad shape");
  kv8_advance_kernel<<<grid_for(batch, 128), 128, 0, s>>>(lens, pos, new_lens, batch, q_len, limit);
  return after_launch(cnt, "kv8_advance");
}

}  // namespace spx
