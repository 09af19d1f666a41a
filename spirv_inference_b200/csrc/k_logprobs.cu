// Log probabilities of given tokens from rows of logits, with the entropy of
// the row, the token's rank and the top alternatives:
//
//   m = max x,  l = sum e^(x - m),  log p_i = x_i - m - log l
//   entropy = log l - sum e^(x - m) (x - m) / l
//   rank = 1 + #{x_j > x_id},  ties among the top k go to the lowest index
//
// One pass over the logits.  A cluster of CTAs shares a row (one CTA when
// there are rows enough); a CTA walks its part in tiles of 4096 values, 16 a
// thread, in registers.  Maximum, sum and sum e^(x-m) (x-m) run per thread and
// are joined at the end.  For the top k a CTA keeps a list of candidates in
// shared memory: of its first tile each warp takes the k-th largest of its
// lanes' maxima (so k values are at least that), the largest of these over
// the warps is the threshold, and only values that reach it enter the list,
// about a dozen of 4096; the list is cut to its k best when it grows.  A tile
// that would overflow it (rising logits, ties) takes its k best one by one.
// Bound by the logits' bytes.
#include <cooperative_groups.h>

#include "spx_internal.cuh"

namespace spx {
namespace {

namespace cg = cooperative_groups;

constexpr int kLpThreads = 256;
constexpr int kLpWarps = kLpThreads / 32;
constexpr int kLpQuads = 4;                              // float4 a thread and tile
constexpr int kLpTile = kLpThreads * kLpQuads * 4;
constexpr int kLpCap = 512;                              // candidates
constexpr int kLpMaxTop = 64;
constexpr float kLog2e = 1.4426950408889634f;

// Order-preserving bits; NaN below everything, -0 equal to +0.
__device__ __forceinline__ uint32_t order_key(float x) {
  if (x != x) return 0u;
  const uint32_t u = __float_as_uint(x + 0.0f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
  if (k == 0u) return __int_as_float(0x7fc00000);
  return __uint_as_float((k & 0x80000000u) ? (k ^ 0x80000000u) : ~k);
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

struct LpArgs {
  const float* x;
  int64_t ld;
  int cols;
  const int32_t* ids;
  float* logprobs;
  float* entropy;
  int32_t* rank;
  int top_k;
  int32_t* top_ids;
  float* top_logprobs;
};

struct Stats {          // of some values: maximum, sum e^(x-m), sum e^(x-m) (x-m)
  float m, l, t;
  int above;
  __device__ __forceinline__ void rebase(float to) {   // to >= m
    if (m == to || m == -INFINITY) {
      m = to;
      return;
    }
    const float d = m - to, f = ex2(d * kLog2e);
    t = f == 0.0f ? 0.0f : f * fmaf(l, d, t);
    l *= f;
    m = to;
  }
  __device__ __forceinline__ void join(Stats o) {
    const float to = fmaxf(m, o.m);
    rebase(to);
    o.rebase(to);
    l += o.l;
    t += o.t;
    above += o.above;
  }
};

// The k best of n <= kLpCap distinct keys, in falling order, to the front.
__device__ __forceinline__ void keep_best(unsigned long long* list, int n, int k) {
  unsigned long long key[kLpCap / kLpThreads];
  int at[kLpCap / kLpThreads];
#pragma unroll
  for (int i = 0; i < kLpCap / kLpThreads; ++i) {
    const int e = threadIdx.x + i * kLpThreads;
    at[i] = k;
    if (e < n) {
      key[i] = list[e];
      int larger = 0;
      for (int j = 0; j < n; ++j) larger += list[j] > key[i];
      at[i] = larger;
    }
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kLpCap / kLpThreads; ++i)
    if (at[i] < k) list[at[i]] = key[i];
  __syncthreads();
}

__global__ void __launch_bounds__(kLpThreads, 4)
    token_logprobs_kernel(const LpArgs a, int cluster, int seg) {
  __shared__ unsigned long long list[kLpCap];
  __shared__ unsigned long long warp_best[kLpWarps];
  __shared__ uint32_t warp_thr[kLpWarps];
  __shared__ Stats warp_stats[kLpWarps];
  __shared__ Stats cta_stats;
  __shared__ int count[3], cta_count;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int r = blockIdx.x / cluster, rank = blockIdx.x - r * cluster;
  const float* x = a.x + (int64_t)r * a.ld;
  // Positions count from the 16-byte boundary at or before the row's start.
  const int shift = (int)(((uintptr_t)x >> 2) & 3);
  const int v0 = rank * seg, v1 = min(v0 + seg, a.cols + shift);
  const int id = a.ids ? a.ids[r] : -1;
  const bool has = id >= 0 && id < a.cols;
  const float one = has ? __ldg(x + id) : 0.0f;
  const int k = a.top_k;
  if (tid == 0) count[0] = 0;
  Stats st = {-INFINITY, 0.0f, 0.0f, 0};
  uint32_t thr = 0;                  // the key that a candidate has to reach
  int held = 0, slot = 0;            // candidates before this tile; its counter
  for (int base = v0; base < v1; base += kLpTile) {
    float v[kLpQuads * 4];
    uint32_t in = 0;                 // which of them are values of the row
#pragma unroll
    for (int q = 0; q < kLpQuads; ++q) {
      const int p = base + (q * kLpThreads + tid) * 4;
      if (p >= shift && p + 4 <= v1) {
        const float4 f = __ldg(reinterpret_cast<const float4*>(x + (p - shift)));
        v[4 * q] = f.x;
        v[4 * q + 1] = f.y;
        v[4 * q + 2] = f.z;
        v[4 * q + 3] = f.w;
        in |= 15u << (4 * q);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const bool ok = p + e >= shift && p + e < v1;
          v[4 * q + e] = ok ? __ldg(x + (p + e - shift)) : -INFINITY;
          in |= (ok ? 1u : 0u) << (4 * q + e);
        }
      }
    }
    // What lies outside is -inf and adds nothing to the sums or the rank.
    float mt = -INFINITY;
#pragma unroll
    for (int i = 0; i < kLpQuads * 4; ++i) mt = fmaxf(mt, v[i]);
    const float to = fmaxf(st.m, mt);
    st.rebase(to);
    const float zero = to == -INFINITY ? 0.0f : to;
#pragma unroll
    for (int i = 0; i < kLpQuads * 4; ++i) {
      const float d = v[i] - zero, e = ex2(d * kLog2e);
      st.l += e;
      st.t = fmaf(e, fmaxf(d, -3.4e38f), st.t);
      st.above += v[i] > one;
    }
    if (k == 0) continue;
    uint32_t best = in ? order_key(mt) : 0u;
    if (st.l != st.l) {              // a NaN may be all that a thread has
      best = 0u;
#pragma unroll
      for (int i = 0; i < kLpQuads * 4; ++i)
        if (in >> i & 1u) best = max(best, order_key(v[i]));
    }
    if (base == v0) {
      // k2 lanes of each of one warp, or of two, reach the threshold.
      const int k2 = k > 32 ? (k + 1) / 2 : k;
      uint32_t left = best, kth = 0;
      for (int i = 0; i < k2; ++i) {
        kth = __reduce_max_sync(0xffffffffu, left);
        const uint32_t who = __ballot_sync(0xffffffffu, left == kth);
        if (lane == __ffs(who) - 1) left = 0;
      }
      if (lane == 0) warp_thr[warp] = kth;
      __syncthreads();
      if (k > 32) {
        for (int w = 0; w < kLpWarps; w += 2) thr = max(thr, min(warp_thr[w], warp_thr[w + 1]));
      } else {
        for (int w = 0; w < kLpWarps; ++w) thr = max(thr, warp_thr[w]);
      }
    }
    if (in && best >= thr) {
#pragma unroll
      for (int i = 0; i < kLpQuads * 4; ++i) {
        const uint32_t key = order_key(v[i]);
        if (key >= thr && (in >> i & 1u)) {
          const int at = held + atomicAdd(&count[slot], 1);
          const uint32_t j = base + ((i >> 2) * kLpThreads + tid) * 4 + (i & 3) - shift;
          if (at < kLpCap) list[at] = ((unsigned long long)key << 32) | (0xffffffffu - j);
        }
      }
    }
    // Three counters in turn: this tile's, the next one's, which nobody reads
    // any more, and the last one's, which slower threads may still read.
    if (tid == 0) count[slot == 2 ? 0 : slot + 1] = 0;
    __syncthreads();
    int n = held + count[slot];
    slot = slot == 2 ? 0 : slot + 1;
    if (n > kLpCap) {
      // Too many: the tile's k best, each the largest below the one before.
      unsigned long long below = ~0ull;
      for (int i = 0; i < k; ++i) {
        unsigned long long b = 0;
#pragma unroll
        for (int e = 0; e < kLpQuads * 4; ++e) {
          const uint32_t j = base + ((e >> 2) * kLpThreads + tid) * 4 + (e & 3) - shift;
          const unsigned long long key =
              ((unsigned long long)order_key(v[e]) << 32) | (0xffffffffu - j);
          if ((in >> e & 1u) && key < below && key > b) b = key;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
          const unsigned long long other = __shfl_xor_sync(0xffffffffu, b, o);
          b = other > b ? other : b;
        }
        if (lane == 0) warp_best[warp] = b;
        __syncthreads();
        for (int w = 0; w < kLpWarps; ++w) b = warp_best[w] > b ? warp_best[w] : b;
        below = b;
        if (tid == 0) list[held + i] = b;   // 0 where the tile has no more
        __syncthreads();
      }
      n = held + k;
    }
    if (n > kLpCap / 2) {
      keep_best(list, n, k);
      n = k;
      thr = max(thr, (uint32_t)(list[k - 1] >> 32));
    }
    held = n;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    Stats s;
    s.m = __shfl_xor_sync(0xffffffffu, st.m, o);
    s.l = __shfl_xor_sync(0xffffffffu, st.l, o);
    s.t = __shfl_xor_sync(0xffffffffu, st.t, o);
    s.above = __shfl_xor_sync(0xffffffffu, st.above, o);
    st.join(s);
  }
  if (lane == 0) warp_stats[warp] = st;
  __syncthreads();
  if (cluster > 1) {
    if (k && held > k) {
      keep_best(list, held, k);
      held = k;
    }
    if (tid == 0) {
      for (int w = 1; w < kLpWarps; ++w) st.join(warp_stats[w]);
      cta_stats = st;
      cta_count = held;
    }
    cg::cluster_group cl = cg::this_cluster();
    cl.sync();
    if (rank == 0) {
      for (int c = 1; c < cluster; ++c) {
        const int n = *cl.map_shared_rank(&cta_count, c);
        const unsigned long long* theirs = cl.map_shared_rank(&list[0], c);
        for (int i = tid; i < n; i += kLpThreads) list[held + i] = theirs[i];
        held += n;
        if (tid == 0) st.join(*cl.map_shared_rank(&cta_stats, c));
      }
      __syncthreads();
    }
    cl.sync();
    if (rank != 0) return;
  } else if (tid == 0) {
    for (int w = 1; w < kLpWarps; ++w) st.join(warp_stats[w]);
  }
  if (tid == 0) cta_stats = st;
  __syncthreads();
  if (k) keep_best(list, held, k);
  st = cta_stats;
  const bool empty = st.m == -INFINITY && st.l == 0.0f;   // every token is masked
  const float log_l = empty ? 0.0f : logf(st.l);
  auto logp = [&](float v) { return empty ? -INFINITY : (v - st.m) - log_l; };
  if (tid == 0) {
    if (a.logprobs)
      a.logprobs[r] = has ? logp(one) : id < 0 ? 0.0f : __int_as_float(0x7fc00000);
    if (a.entropy) a.entropy[r] = empty ? 0.0f : log_l - st.t / st.l;
    if (a.rank) a.rank[r] = has ? st.above + 1 : 0;
  }
  if (tid < k) {
    const unsigned long long b = list[tid];
    a.top_ids[(int64_t)r * k + tid] = (int32_t)(0xffffffffu - (uint32_t)b);
    a.top_logprobs[(int64_t)r * k + tid] = logp(key_value((uint32_t)(b >> 32)));
  }
}

}  // namespace

int launch_token_logprobs(cudaStream_t s, int64_t* cnt, const float* x, int64_t ld, int rows,
                          int cols, const int32_t* ids, float* logprobs, float* entropy,
                          int32_t* rank, int top_k, int32_t* top_ids, float* top_logprobs) {
  if (rows <= 0 || cols <= 0 || ld < cols)
    return fail(SPX_ERR_INVALID_ARGUMENT, "token_logprobs: bad shape");
  if ((logprobs || rank) && !ids)
    return fail(SPX_ERR_INVALID_ARGUMENT, "token_logprobs: logprobs and rank need token ids");
  if (top_k < 0 || top_k > kLpMaxTop || top_k > cols)
    return fail(SPX_ERR_INVALID_ARGUMENT, "token_logprobs: top_k must be 0..64 and at most cols");
  if (top_k && (!top_ids || !top_logprobs))
    return fail(SPX_ERR_INVALID_ARGUMENT, "token_logprobs: top_k needs both outputs");
  if (cols > INT32_MAX - 2 * kLpTile)
    return fail(SPX_ERR_UNSUPPORTED, "token_logprobs: too many columns");
  // Rows over several CTAs while there are fewer than two CTAs an SM and a
  // part stays half a tile.
  int cluster = 1;
  while (cluster < 8 && (int64_t)rows * cluster < 2 * kNumSms && cols / cluster > kLpTile / 2)
    cluster *= 2;
  const int seg = (int)ceil_div(ceil_div(cols + 3, cluster), 4) * 4;
  if ((int64_t)rows * cluster > INT32_MAX)
    return fail(SPX_ERR_UNSUPPORTED, "token_logprobs: grid too large");
  const LpArgs a{x, ld, cols, ids, logprobs, entropy, rank, top_k, top_ids, top_logprobs};
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(rows * cluster));
  cfg.blockDim = dim3(kLpThreads);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)cluster;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const int rc = check_cuda(cudaLaunchKernelEx(&cfg, token_logprobs_kernel, a, cluster, seg),
                            "token_logprobs");
  return rc ? rc : after_launch(cnt, "token_logprobs");
}

}  // namespace spx
