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
#include "spx_internal.cuh"

namespace spx {
namespace {

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

__device__ __forceinline__ int clamp_len(int v, int hi) { return v < 0 ? 0 : v > hi ? hi : v; }

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
// Append.  Grid: the first `q_ctas` CTAs rotate the queries (elementwise);
// each other CTA takes one block of one (sequence, head, K or V): its values
// into shared memory (rotated where they are keys), the largest magnitude,
// then the int8 block, or the tail while the block stays open.
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
  int blocks;   // blocks that one sequence's new tokens may touch
  int64_t q_ctas;
};

// x * cos + rotate_half(x) * sin, each product and the sum rounded once; a
// position outside the tables gives NaN.
__device__ __forceinline__ float rotated(const AppendArgs& a, const float* src, int d, int p) {
  const int D = a.c.head_dim, half = D >> 1;
  if (p < 0 || p >= a.table_rows) return __int_as_float(0x7fc00000);
  const float x = src[d];
  const float o = d < half ? -src[d + half] : src[d - half];
  return __fadd_rn(__fmul_rn(x, a.cos_t[(int64_t)p * D + d]),
                   __fmul_rn(o, a.sin_t[(int64_t)p * D + d]));
}

__global__ void __launch_bounds__(kAppendThreads) rope_kv8_append_kernel(const AppendArgs a) {
  extern __shared__ float vals[];   // [block][D]
  __shared__ uint32_t warp_max[kAppendThreads / 32];
  const int D = a.c.head_dim, Hkv = a.c.kv_heads, blk = a.c.block, T = a.T;
  if ((int64_t)blockIdx.x < a.q_ctas) {
    const int64_t total = (int64_t)a.c.batch * T * a.Hq * D;
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total;
         i += a.q_ctas * blockDim.x) {
      const int d = (int)(i % D);
      const int64_t rh = i / D;
      const int h = (int)(rh % a.Hq);
      const int64_t r = rh / a.Hq;
      const int t = (int)(r % T), b = (int)(r / T);
      if (a.new_lens && t >= a.new_lens[b]) continue;
      a.q_out[i] = rotated(a, a.qkv + r * a.ld + (int64_t)h * D, d, a.pos[b] + t);
    }
    return;
  }
  int64_t w = (int64_t)blockIdx.x - a.q_ctas;
  const int wb = (int)(w % a.blocks);
  w /= a.blocks;
  const bool is_v = w & 1;
  w >>= 1;
  const int h = (int)(w % Hkv), b = (int)(w / Hkv);
  const int n = a.new_lens ? clamp_len(a.new_lens[b], T) : T;
  const int len = clamp_len(a.c.lens[b], a.c.max_seq);
  const int total = min(len + n, a.c.max_seq);
  const int first = len / blk;                 // the block that is open before the call
  const int blk_i = first + wb;
  const int lo = blk_i * blk;
  if (n == 0 || lo >= total) return;
  const KvView kv = view_of(a.c, b, h, is_v);
  const int64_t col = (int64_t)(a.Hq + (is_v ? Hkv : 0) + h) * D;
  const int pos = a.pos[b];
  auto fresh = [&](int slot, int d) {
    const int t = slot - len;
    const float* src = a.qkv + ((int64_t)b * T + t) * a.ld + col;
    return is_v ? src[d] : rotated(a, src, d, pos + t);
  };
  auto to_tail = [&](int from, int to) {       // new tokens of an open block
    for (int e = threadIdx.x; e < (to - from) * D; e += blockDim.x) {
      const int slot = from + e / D, d = e % D;
      kv.tail[(slot % blk) * D + d] = fresh(slot, d);
    }
  };
  if (lo + blk > total) {
    // Open.  Where it is not the block that was open before, the CTA of that
    // block writes it, after it has read the tail.
    if (wb == 0) to_tail(max(lo, len), total);
    return;
  }
  uint32_t mx = 0;
  for (int e = threadIdx.x; e < blk * D; e += blockDim.x) {
    const int slot = lo + e / D, d = e % D;
    const float x = slot < len ? kv.tail[e] : fresh(slot, d);
    vals[e] = x;
    mx = max(mx, abs_bits(x));
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
  char4* out = reinterpret_cast<char4*>(kv.q8 + (int64_t)lo * D);
  for (int e = threadIdx.x; e < blk * D / 4; e += blockDim.x) {
    const float4 x = reinterpret_cast<const float4*>(vals)[e];
    char4 q = make_char4(0, 0, 0, 0);
    if (ok)
      q = make_char4((signed char)round_div(x.x, s, inv), (signed char)round_div(x.y, s, inv),
                     (signed char)round_div(x.z, s, inv), (signed char)round_div(x.w, s, inv));
    out[e] = q;
  }
  if (wb == 0) {
    const int open = total / blk * blk;
    if (open > lo && open < total) to_tail(open, total);
  }
}

// ---------------------------------------------------------------------------
// Read-back of `count` slots from starts[b] on, as fp32; 0 behind the end.
__global__ void kv8_read_kernel(const spx_kv8_cache c, const int32_t* __restrict__ new_lens,
                                int q_len, const int32_t* __restrict__ starts, int count,
                                float* __restrict__ k_out, float* __restrict__ v_out) {
  const int D = c.head_dim, blk = c.block;
  const int64_t per = (int64_t)c.batch * c.kv_heads * count * (D / 4);
  const int64_t total = per * 2;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total;
       i += (int64_t)gridDim.x * blockDim.x) {
    const bool is_v = i >= per;
    const int64_t e = is_v ? i - per : i;
    const int d = (int)(e % (D / 4)) * 4;
    int64_t r = e / (D / 4);
    const int at = (int)(r % count);
    r /= count;
    const int h = (int)(r % c.kv_heads), b = (int)(r / c.kv_heads);
    const int n = new_lens ? clamp_len(new_lens[b], q_len) : q_len;
    const int len = min(clamp_len(c.lens[b], c.max_seq) + n, c.max_seq);
    const int64_t slot = (starts ? (int64_t)starts[b] : 0) + at;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    if (slot >= 0 && slot < len) {
      const KvView kv = view_of(c, b, h, is_v);
      if (slot < len / blk * blk) {
        const char4 q = *reinterpret_cast<const char4*>(kv.q8 + slot * D + d);
        const float s = kv.scale[slot / blk];
        x = make_float4(q.x * s, q.y * s, q.z * s, q.w * s);
      } else {
        x = *reinterpret_cast<const float4*>(kv.tail + (slot % blk) * D + d);
      }
    }
    reinterpret_cast<float4*>(is_v ? v_out : k_out)[e] = x;
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
// keep their 8 bits.  Slot i of the result comes from a slot >= i, so walking
// the blocks upwards and reading a block's rows before writing it also works
// in place.  One CTA per (sequence, head, K or V).
constexpr int kGatherThreads = 256;

__global__ void __launch_bounds__(kGatherThreads)
    kv8_gather_kernel(const spx_kv8_cache src, const spx_kv8_cache dst, const float* w_src,
                      float* w_dst, const int32_t* __restrict__ idx, int keep, int in_place) {
  extern __shared__ float vals[];   // [block][D] values
  __shared__ float row_scale[128];
  __shared__ int row_src[128];
  const int D = src.head_dim, blk = src.block;
  const int bh = blockIdx.x >> 1, b = bh / src.kv_heads, h = bh % src.kv_heads;
  const bool is_v = blockIdx.x & 1;
  const int n = clamp_len(src.lens[b], src.max_seq);
  const int kept = min(n, keep);
  if (in_place && n <= keep) return;
  const KvView s = view_of(src, b, h, is_v), d = view_of(dst, b, h, is_v);
  const int closed = n / blk * blk;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  for (int lo = 0; lo < kept; lo += blk) {
    const int rows = min(blk, kept - lo);
    float wv = 0.0f;
    for (int r = warp; r < rows; r += kGatherThreads / 32) {
      const int j = idx[(int64_t)bh * keep + lo + r];
      float sc;
      if (j < closed) {
        sc = s.scale[j / blk];
        for (int e = lane; e < D; e += 32) vals[r * D + e] = s.q8[(int64_t)j * D + e] * sc;
      } else {
        uint32_t mx = 0;
        for (int e = lane; e < D; e += 32) {
          const float x = s.tail[(j % blk) * D + e];
          vals[r * D + e] = x;
          mx = max(mx, abs_bits(x));
        }
        sc = scale_of(__reduce_max_sync(0xffffffffu, mx));
      }
      if (lane == 0) {
        row_scale[r] = sc;
        row_src[r] = j;
      }
    }
    __syncthreads();
    if (tid < rows && !is_v) wv = w_src[(int64_t)bh * src.max_seq + row_src[tid]];
    uint32_t mx = 0;
    for (int r = 0; r < rows; ++r) mx = max(mx, __float_as_uint(row_scale[r]) & 0x7fffffffu);
    const float ns = __uint_as_float(mx);
    __syncthreads();
    if (tid < rows && !is_v) w_dst[(int64_t)bh * dst.max_seq + lo + tid] = wv;
    if (rows < blk) {
      for (int e = tid; e < rows * D; e += blockDim.x) d.tail[e] = vals[e];
    } else {
      const bool ok = usable(ns);
      if (tid == 0) d.scale[lo / blk] = ns;
      for (int e = tid; e < rows * D; e += blockDim.x) {
        int q = 0;
        if (ok) {
          const int j = row_src[e / D];
          // exact value of an int8 row: q * scale needs more bits than fp32 has
          const double x = j < closed ? (double)rint(vals[e] / row_scale[e / D]) * row_scale[e / D]
                                      : (double)vals[e];
          const double v = row_scale[e / D] > 0.0f || j >= closed ? x / ns : 0.0;
          q = (int)rint(fmin(fmax(v, -127.0), 127.0));
        }
        d.q8[(int64_t)lo * D + e] = (int8_t)q;
      }
    }
    __syncthreads();
  }
}

__global__ void kv8_advance_kernel(int32_t* lens, int32_t* pos, const int32_t* new_lens, int batch,
                                   int q_len, int limit) {
  for (int b = blockIdx.x * blockDim.x + threadIdx.x; b < batch; b += gridDim.x * blockDim.x) {
    const int n = new_lens ? clamp_len(new_lens[b], q_len) : q_len;
    if (lens) lens[b] = min(clamp_len(lens[b], limit) + n, limit);
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
  a.blocks = (T + 2 * c->block - 2) / c->block;   // the open block and what follows
  a.q_ctas = grid_for((int64_t)c->batch * T * Hq * c->head_dim, kAppendThreads);
  const int64_t grid = a.q_ctas + (int64_t)c->batch * c->kv_heads * 2 * a.blocks;
  if (grid > INT32_MAX) return fail(SPX_ERR_UNSUPPORTED, "rope_kv8_append: grid too large");
  const size_t smem = (size_t)c->block * c->head_dim * sizeof(float);
  if (smem > 48 * 1024) {
    rc = check_cuda(cudaFuncSetAttribute(rope_kv8_append_kernel,
                                         cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem),
                    "rope_kv8_append: smem attribute");
    if (rc) return rc;
  }
  rope_kv8_append_kernel<<<(int)grid, kAppendThreads, smem, s>>>(a);
  return after_launch(cnt, "rope_kv8_append");
}

int launch_kv8_read(cudaStream_t s, int64_t* cnt, const spx_kv8_cache* c, const int32_t* new_lens,
                    int q_len, const int32_t* starts, int count, float* k_out, float* v_out) {
  int rc = kv8_check(c, "kv8_read");
  if (rc) return rc;
  if (q_len < 0 || count <= 0) return fail(SPX_ERR_INVALID_ARGUMENT, "kv8_read: bad shape");
  if (!al16(k_out) || !al16(v_out))
    return fail(SPX_ERR_INVALID_ARGUMENT, "kv8_read: outputs must be 16-byte aligned");
  const int64_t work = (int64_t)c->batch * c->kv_heads * count * (c->head_dim / 4) * 2;
  kv8_read_kernel<<<grid_for(work, 256, 16), 256, 0, s>>>(*c, new_lens, q_len, starts, count, k_out,
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
  const size_t smem = (size_t)src->block * src->head_dim * sizeof(float);
  if (smem > 40 * 1024) {
    rc = check_cuda(cudaFuncSetAttribute(kv8_gather_kernel,
                                         cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem),
                    "kv8_evict: smem attribute");
    if (rc) return rc;
  }
  kv8_gather_kernel<<<(int)(2 * bh), kGatherThreads, smem, s>>>(*src, *dst, weights, dst_weights,
                                                                idx, keep, same ? 1 : 0);
  return after_launch(cnt, "kv8_evict: gather");
}

int launch_kv8_advance(cudaStream_t s, int64_t* cnt, int32_t* lens, int32_t* pos,
                       const int32_t* new_lens, int batch, int q_len, int limit) {
  if (batch <= 0 || q_len < 0 || limit <= 0)
    return fail(SPX_ERR_INVALID_ARGUMENT, "kv8_advance: bad shape");
  kv8_advance_kernel<<<grid_for(batch, 128), 128, 0, s>>>(lens, pos, new_lens, batch, q_len, limit);
  return after_launch(cnt, "kv8_advance");
}

}  // namespace spx
