// Causal grouped-query attention over the 8-bit key / value cache, and the
// attention weight each slot receives.
//
//   s = scale q.k,  out = softmax(s) v,  lse = log sum exp(s)
//   weights[j] += sum over the new tokens and the heads of the group of
//                 exp(s_j - lse)     (slots of the new tokens start from 0)
#include "spx_internal.cuh"

namespace spx {
namespace {

__device__ __forceinline__ int clamp_len(int v, int hi) { return v < 0 ? 0 : v > hi ? hi : v; }

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

// One value of a cached row.
__device__ __forceinline__ float cached(const int8_t* q8, const float* scale, const float* tail,
                                        int j, int d, int closed, int blk, int D) {
  return j < closed ? q8[(int64_t)j * D + d] * scale[j / blk] : tail[(j % blk) * D + d];
}

// A warp per (token, head).
template <int D>
__global__ void __launch_bounds__(128) attention_kv8_kernel(const AttnArgs a) {
  constexpr int E = D / 32;
  const int lane = threadIdx.x & 31;
  const int64_t item = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (item >= (int64_t)a.c.batch * a.T * a.Hq) return;
  const int hq = (int)(item % a.Hq);
  const int64_t row = item / a.Hq;
  const int t = (int)(row % a.T), b = (int)(row / a.T);
  const int S = a.c.max_seq, blk = a.c.block;
  const int n = a.new_lens ? clamp_len(a.new_lens[b], a.T) : a.T;
  if (t >= n) return;
  const int len = clamp_len(a.c.lens[b], S), total = min(len + n, S);
  const int closed = total / blk * blk, seen = min(len + t + 1, S);
  const int64_t bh = (int64_t)b * a.c.kv_heads + hq / (a.Hq / a.c.kv_heads);
  const int8_t *k8 = a.c.k + bh * S * D, *v8 = a.c.v + bh * S * D;
  const float *ks = a.c.k_scale + bh * (S / blk), *vs = a.c.v_scale + bh * (S / blk);
  const float *kt = a.c.k_tail + bh * blk * D, *vt = a.c.v_tail + bh * blk * D;
  float q[E], o[E], m = -INFINITY, l = 0.0f;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    q[e] = a.q[item * D + e * 32 + lane] * a.scale;
    o[e] = 0.0f;
  }
  for (int j = 0; j < seen; ++j) {
    float s = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e)
      s = fmaf(q[e], cached(k8, ks, kt, j, e * 32 + lane, closed, blk, D), s);
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
    const float mn = fmaxf(m, s), f = expf(m - mn), p = expf(s - mn);
    l = l * f + p;
#pragma unroll
    for (int e = 0; e < E; ++e)
      o[e] = fmaf(p, cached(v8, vs, vt, j, e * 32 + lane, closed, blk, D), o[e] * f);
    m = mn;
  }
#pragma unroll
  for (int e = 0; e < E; ++e) a.out[item * D + e * 32 + lane] = o[e] / l;
  if (a.lse && lane == 0) a.lse[item] = m + logf(l);
}

// A thread per slot.
template <int D>
__global__ void __launch_bounds__(128) kv8_weights_kernel(const AttnArgs a) {
  const int S = a.c.max_seq, blk = a.c.block, G = a.Hq / a.c.kv_heads;
  const int bh = blockIdx.y, b = bh / a.c.kv_heads, h = bh % a.c.kv_heads;
  const int n = a.new_lens ? clamp_len(a.new_lens[b], a.T) : a.T;
  const int len = clamp_len(a.c.lens[b], S), total = min(len + n, S);
  const int j = blockIdx.x * blockDim.x + threadIdx.x;
  if (n == 0 || j >= total) return;
  const int closed = total / blk * blk;
  const int8_t* k8 = a.c.k + (int64_t)bh * S * D;
  const float* ks = a.c.k_scale + (int64_t)bh * (S / blk);
  const float* kt = a.c.k_tail + (int64_t)bh * blk * D;
  float w = 0.0f;
  for (int t = 0; t < n; ++t) {
    if (j >= min(len + t + 1, S)) continue;
    for (int g = 0; g < G; ++g) {
      const int64_t item = ((int64_t)b * a.T + t) * a.Hq + h * G + g;
      float s = 0.0f;
      for (int d = 0; d < D; ++d)
        s = fmaf(a.q[item * D + d] * a.scale, cached(k8, ks, kt, j, d, closed, blk, D), s);
      w += expf(s - a.lse[item]);
    }
  }
  float* wp = a.weights + (int64_t)bh * S + j;
  *wp = (j < len ? *wp : 0.0f) + w;
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
  const int64_t items = (int64_t)c->batch * T * Hq;
  const int64_t bh = (int64_t)c->batch * c->kv_heads;
  if (items > INT32_MAX || bh > 65535)
    return fail(SPX_ERR_UNSUPPORTED, "attention_kv8: grid too large");
  const AttnArgs a{q, *c, new_lens, T, Hq, scale, out, lse, weights};
  const int grid = (int)ceil_div(items, 4);
  if (c->head_dim == 64)
    attention_kv8_kernel<64><<<grid, 128, 0, s>>>(a);
  else
    attention_kv8_kernel<128><<<grid, 128, 0, s>>>(a);
  if ((rc = after_launch(cnt, "attention_kv8")) || !weights) return rc;
  const dim3 wg((unsigned)ceil_div(c->max_seq, 128), (unsigned)bh);
  if (c->head_dim == 64)
    kv8_weights_kernel<64><<<wg, 128, 0, s>>>(a);
  else
    kv8_weights_kernel<128><<<wg, 128, 0, s>>>(a);
  return after_launch(cnt, "attention_kv8: weights");
}

}  // namespace spx
