// Log probabilities of given tokens from rows of logits, with the entropy of
// the row, the token's rank and the top alternatives:
//
//   m = max x,  l = sum e^(x - m),  log p_i = x_i - m - log l
//   entropy = log l - sum e^(x - m) (x - m) / l
//   rank = 1 + #{x_j > x_id},  ties among the top k go to the lowest index
#include "spx_internal.cuh"

namespace spx {
namespace {

constexpr int kLpThreads = 512;

// Order-preserving bits; NaN below everything, -0 equal to +0.
__device__ __forceinline__ uint32_t order_key(float x) {
  if (x != x) return 0u;
  const uint32_t u = __float_as_uint(x + 0.0f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
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

__global__ void __launch_bounds__(kLpThreads) token_logprobs_kernel(const LpArgs a) {
  __shared__ float red[3][kLpThreads / 32];
  __shared__ int cnt[kLpThreads / 32];
  __shared__ unsigned long long best[kLpThreads / 32];
  const int r = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const float* x = a.x + (int64_t)r * a.ld;
  const int id = a.ids ? a.ids[r] : -1;
  const bool has = id >= 0 && id < a.cols;
  const float one = has ? x[id] : 0.0f;
  float m = -INFINITY;
  bool nan = false;
  int above = 0;
  for (int j = tid; j < a.cols; j += kLpThreads) {
    const float v = x[j];
    m = fmaxf(m, v);
    nan |= v != v;
    above += v > one;
  }
  for (int o = 16; o > 0; o >>= 1) {
    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    above += __shfl_xor_sync(0xffffffffu, above, o);
  }
  if (lane == 0) {
    red[0][warp] = m;
    cnt[warp] = above;
  }
  nan = __syncthreads_or(nan);
  m = -INFINITY;
  above = 0;
  for (int i = 0; i < kLpThreads / 32; ++i) {
    m = fmaxf(m, red[0][i]);
    above += cnt[i];
  }
  float l = 0.0f, t = 0.0f;
  for (int j = tid; j < a.cols; j += kLpThreads) {
    const float d = x[j] - m;
    if (x[j] == -INFINITY) continue;   // nothing of either sum
    const float e = expf(d);
    l += e;
    t += e * d;
  }
  for (int o = 16; o > 0; o >>= 1) {
    l += __shfl_xor_sync(0xffffffffu, l, o);
    t += __shfl_xor_sync(0xffffffffu, t, o);
  }
  if (lane == 0) {
    red[1][warp] = l;
    red[2][warp] = t;
  }
  __syncthreads();
  l = 0.0f;
  t = 0.0f;
  for (int i = 0; i < kLpThreads / 32; ++i) {
    l += red[1][i];
    t += red[2][i];
  }
  const bool empty = m == -INFINITY && !nan;   // every token is masked
  const float log_l = empty ? 0.0f : logf(l);
  auto logp = [&](float v) { return empty ? -INFINITY : nan ? NAN : v - m - log_l; };
  if (tid == 0) {
    if (a.logprobs) a.logprobs[r] = has ? logp(one) : id < 0 ? 0.0f : NAN;
    if (a.entropy) a.entropy[r] = empty ? 0.0f : nan ? NAN : log_l - t / l;
    if (a.rank) a.rank[r] = has ? above + 1 : 0;
  }
  unsigned long long last = ~0ull;
  for (int k = 0; k < a.top_k; ++k) {
    unsigned long long b = 0;
    for (int j = tid; j < a.cols; j += kLpThreads) {
      const unsigned long long key =
          ((unsigned long long)order_key(x[j]) << 32) | (0xffffffffu - (uint32_t)j);
      if (key < last && key > b) b = key;
    }
    for (int o = 16; o > 0; o >>= 1) {
      const unsigned long long v = __shfl_xor_sync(0xffffffffu, b, o);
      b = v > b ? v : b;
    }
    __syncthreads();
    if (lane == 0) best[warp] = b;
    __syncthreads();
    for (int i = 0; i < kLpThreads / 32; ++i) b = best[i] > b ? best[i] : b;
    last = b;
    if (tid == 0) {
      const int j = (int)(0xffffffffu - (uint32_t)(b & 0xffffffffull));
      a.top_ids[(int64_t)r * a.top_k + k] = j;
      a.top_logprobs[(int64_t)r * a.top_k + k] = logp(x[j]);
    }
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
  if (top_k < 0 || top_k > 64 || top_k > cols)
    return fail(SPX_ERR_INVALID_ARGUMENT, "token_logprobs: top_k must be 0..64 and at most cols");
  if (top_k && (!top_ids || !top_logprobs))
    return fail(SPX_ERR_INVALID_ARGUMENT, "token_logprobs: top_k needs both outputs");
  const LpArgs a{x, ld, cols, ids, logprobs, entropy, rank, top_k, top_ids, top_logprobs};
  token_logprobs_kernel<<<rows, kLpThreads, 0, s>>>(a);
  return after_launch(cnt, "token_logprobs");
}

}  // namespace spx
