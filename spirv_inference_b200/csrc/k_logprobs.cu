// Log probabilities of given tokens from rows of logits, with the entropy of
// the row, the token's rank and the top alternatives:
//
//   m = max x,  l = sum e^(x - m),  log p_i = x_i - m - log l
//   entropy = log l - sum e^(x - m) (x - m) / l
//   rank = 1 + #{x_j > x_id},  ties among the top k go to the lowest index
//
// One pass over the logits.  With rows enough for every SM a warp takes a row;
// else the eight warps of a CTA, and with few rows a cluster of CTAs, share
// one.  A warp walks tiles of 512 values, 16 a lane, which each lane copies to
// shared memory for itself two tiles ahead (32 KB a CTA in flight, four CTAs an
// SM, no barrier).  Maximum, sum and sum e^(x-m) (x-m) run per lane.
//
// For the top k a warp keeps a list of candidates in shared memory: the k-th
// largest of its lanes' maxima in its first tile is a threshold that k values
// reach, and only values that reach it enter the list; when the list grows it
// is cut to its k best, and values then have to exceed the last of them.  A
// tile that would overflow it (rising logits, ties) gives its k best one by
// one.  Warps' and CTAs' lists are merged by binary searches.
//
// 4096 rows of 32000: 102 us, 5.1 TB/s.  Bound by the logits' bytes;
// instructions come next (a maximum, a difference, a product, ex2 and two sums a
// value), so pairs of values go through the packed fp32 operations, and the rank
// is counted only in lanes whose maximum exceeds the token's logit.
#include <cooperative_groups.h>

#include "spx_internal.cuh"

namespace spx {
namespace {

namespace cg = cooperative_groups;

constexpr int kLpWarps = 8;
constexpr int kLpPerSm = 4;                    // CTAs an SM
constexpr int kLpQuads = 4;                    // float4 a lane and tile
constexpr int kLpTile = 32 * kLpQuads * 4;
constexpr int kLpSlots = 2;                    // tiles of a warp in flight
constexpr int kLpCap = 120;                    // candidates of a warp
constexpr size_t kLpRing = sizeof(float) * kLpWarps * kLpSlots * kLpTile;
constexpr int kLpMaxTop = 64;
constexpr int kLpMaxCluster = 8;               // (merge_lists takes eight lists)
static_assert(kLpWarps == 8 && kLpMaxCluster == 8 && kLpQuads == 4, "lists and maxima a lane");
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

__device__ __forceinline__ void cluster_arrive() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() {
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

struct LpArgs {
  const float* x;
  int64_t ld;
  int rows, cols;
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
  // Of the warp's lanes together, to all of them.
  __device__ __forceinline__ void join_lanes() {
    const uint32_t u = __float_as_uint(m);
    const uint32_t key = __reduce_max_sync(0xffffffffu, u & 0x80000000u ? ~u : u | 0x80000000u);
    rebase(__uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key));
    above = __reduce_add_sync(0xffffffffu, above);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      l += __shfl_xor_sync(0xffffffffu, l, o);
      t += __shfl_xor_sync(0xffffffffu, t, o);
    }
  }
};

// Two fp32 operations in one instruction, each rounded as the single one is.
__device__ __forceinline__ unsigned long long f2_bits(float2 v) {
  return *reinterpret_cast<unsigned long long*>(&v);
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  unsigned long long d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(f2_bits(a)), "l"(f2_bits(b)));
  return *reinterpret_cast<float2*>(&d);
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  unsigned long long d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(f2_bits(a)), "l"(f2_bits(b)));
  return *reinterpret_cast<float2*>(&d);
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  unsigned long long d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(d)
      : "l"(f2_bits(a)), "l"(f2_bits(b)), "l"(f2_bits(c)));
  return *reinterpret_cast<float2*>(&d);
}

// The k best of a warp's n <= kLpCap distinct keys, in falling order, to the
// front of the list.
__device__ __forceinline__ void keep_best(unsigned long long* list, int n, int k, int lane) {
  unsigned long long key[4];
  int at[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int e = lane + 32 * i;
    key[i] = e < n ? list[e] : 0ull;
    at[i] = e < n ? 0 : k;
    if (32 * i < n) {
#pragma unroll 8
      for (int j = 0; j < n; ++j) at[i] += list[j] > key[i];
    }
  }
  __syncwarp();
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (at[i] < k) list[at[i]] = key[i];
  __syncwarp();
}

// The k best of eight lists in falling order (counts[i] <= k keys, at lists +
// i * stride), to `out`; of the CTA.  A key's place is its own plus the number
// of larger keys in the seven others, by seven binary searches side by side.
__device__ __forceinline__ void merge_lists(const unsigned long long* lists, int stride,
                                            const int* counts, int k, unsigned long long* out,
                                            int warp, int lane) {
  const int first_step = 1 << (31 - __clz(k));
  for (int i = lane; i < counts[warp]; i += 32) {
    const unsigned long long key = lists[warp * stride + i];
    int pos[kLpWarps] = {};
#pragma unroll 1
    for (int s = first_step; s > 0; s >>= 1) {
#pragma unroll
      for (int w = 0; w < kLpWarps; ++w)
        if (pos[w] + s <= counts[w] && lists[w * stride + pos[w] + s - 1] > key) pos[w] += s;
    }
    int at = 0;
#pragma unroll
    for (int w = 0; w < kLpWarps; ++w) at += w == warp ? i : pos[w];
    if (at < k) out[at] = key;
  }
}

// The largest value that k >= 1 of 32 lanes' keys reach.
__device__ __forceinline__ uint32_t kth_largest(uint32_t x, int k, int lane) {
#pragma unroll
  for (int size = 2; size <= 32; size <<= 1)       // bitonic, falling
#pragma unroll
    for (int d = size >> 1; d > 0; d >>= 1) {
      const uint32_t y = __shfl_xor_sync(0xffffffffu, x, d);
      const bool low = !(lane & d), falls = !(lane & size) || size == 32;
      x = low == falls ? max(x, y) : min(x, y);
    }
  return __shfl_sync(0xffffffffu, x, k - 1);
}

__device__ __forceinline__ unsigned long long packed(float v, uint32_t j) {
  return ((unsigned long long)order_key(v) << 32) | (0xffffffffu - j);
}

__device__ __forceinline__ void copy_async(void* to, const float* from, bool quad) {
  const uint32_t s = (uint32_t)__cvta_generic_to_shared(to);
  if (quad)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(s), "l"(from) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(s), "l"(from) : "memory");
}

// Starts the copies of a tile (positions base ..) into the lane's places of a
// slot.  Positions outside [shift, v1) are not read.
__device__ __forceinline__ void start_tile(float4* slot, const float* x, int base, int shift,
                                           int v1, int lane) {
  if (base >= shift && base + kLpTile <= v1) {
    const float* from = x + (base - shift) + lane * 4;
#pragma unroll
    for (int q = 0; q < kLpQuads; ++q) copy_async(slot + q * 32 + lane, from + q * 128, true);
  } else if (base < v1) {
    for (int q = 0; q < kLpQuads; ++q) {
      const int p = base + (q * 32 + lane) * 4;
      float* to = reinterpret_cast<float*>(slot + q * 32 + lane);
      if (p >= shift && p + 4 <= v1) {
        copy_async(to, x + (p - shift), true);
      } else {
        for (int e = 0; e < 4; ++e)
          if (p + e >= shift && p + e < v1) copy_async(to + e, x + (p + e - shift), false);
      }
    }
  }
  asm volatile("cp.async.commit_group;" ::: "memory");
}

// A row's results, by `threads` threads of which this is number `me`.
__device__ __forceinline__ void emit(const LpArgs& a, int r, const Stats& st,
                                     const unsigned long long* top, int me, int threads, float one,
                                     int id, bool has) {
  const bool empty = st.m == -INFINITY && st.l == 0.0f;   // every token is masked
  const float log_l = empty ? 0.0f : logf(st.l);
  auto logp = [&](float v) { return empty ? -INFINITY : (v - st.m) - log_l; };
  if (me == 0) {
    if (a.logprobs)
      a.logprobs[r] = has ? logp(one) : id < 0 ? 0.0f : __int_as_float(0x7fc00000);
    if (a.entropy) a.entropy[r] = empty ? 0.0f : log_l - st.t / st.l;
    if (a.rank) a.rank[r] = has ? st.above + 1 : 0;
  }
  for (int i = me; i < a.top_k; i += threads) {
    const unsigned long long b = top[i];
    a.top_ids[(int64_t)r * a.top_k + i] = (int32_t)(0xffffffffu - (uint32_t)b);
    a.top_logprobs[(int64_t)r * a.top_k + i] = logp(key_value((uint32_t)(b >> 32)));
  }
}

template <bool ROW_PER_WARP>
__global__ void __launch_bounds__(kLpWarps * 32, kLpPerSm)
    token_logprobs_kernel(const LpArgs a, int cluster, int seg) {
  __shared__ unsigned long long lists[kLpWarps][kLpCap];
  __shared__ unsigned long long joined[ROW_PER_WARP ? 1 : kLpMaxTop];
  __shared__ unsigned long long theirs[ROW_PER_WARP ? 1 : kLpMaxCluster][kLpMaxTop];
  __shared__ Stats parts[kLpWarps], cta_parts[kLpMaxCluster];
  __shared__ int counts[kLpWarps], cta_counts[kLpMaxCluster];
  extern __shared__ float4 ring_all[];         // [warp][slot][quad][lane]
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  float4* ring = ring_all + warp * (kLpSlots * kLpQuads * 32);
  const int warps = blockDim.x >> 5;           // kLpWarps unless a warp has a row
  int r = ROW_PER_WARP ? warp * gridDim.x + blockIdx.x : blockIdx.x / cluster;
  const int rank = ROW_PER_WARP ? 0 : blockIdx.x - r * cluster;
  if (ROW_PER_WARP && r >= a.rows) return;
  cg::cluster_group cl = cg::this_cluster();
  if (!ROW_PER_WARP && cluster > 1) cluster_arrive();
  constexpr int kStep = ROW_PER_WARP ? kLpTile : kLpWarps * kLpTile;
  const int k = a.top_k;
  unsigned long long* list = lists[warp];
  // The row: positions count from the 16-byte boundary at or before its start.
  const float* x;
  int shift, v1, base, id;
  float one;
  bool has;
  auto take_row = [&]() {
    x = a.x + (int64_t)r * a.ld;
    shift = (int)(((uintptr_t)x >> 2) & 3);
    v1 = min(rank * seg + seg, a.cols + shift);
    base = rank * seg + (ROW_PER_WARP ? 0 : warp * kLpTile);
    for (int s = 0; s < kLpSlots; ++s)
      start_tile(ring + s * (kLpQuads * 32), x, base + s * kStep, shift, v1, lane);
    id = a.ids ? a.ids[r] : -1;
    has = id >= 0 && id < a.cols;
    one = has ? __ldg(x + id) : 0.0f;
  };
  take_row();
  for (;;) {                         // one row, or a warp's rows
    Stats st = {-INFINITY, 0.0f, 0.0f, 0};
    float thr = -INFINITY;             // what a candidate has to reach
    int held = 0;
    bool first = true;
    float2 l2 = make_float2(0.f, 0.f), t2 = make_float2(0.f, 0.f);
    int slot = 0;
    for (; base < v1; base += kStep) {
      asm volatile("cp.async.wait_group %0;" ::"n"(kLpSlots - 1) : "memory");
      float4* here = ring + slot * (kLpQuads * 32);
      slot = slot == kLpSlots - 1 ? 0 : slot + 1;
      float v[kLpQuads * 4];
#pragma unroll
      for (int q = 0; q < kLpQuads; ++q) {
        const float4 f = here[q * 32 + lane];   // the lane's own copies
        v[4 * q] = f.x;
        v[4 * q + 1] = f.y;
        v[4 * q + 2] = f.z;
        v[4 * q + 3] = f.w;
      }
      // Bit i: v[i] is a value of the row.  What lies outside is -inf and adds
      // nothing to the sums or the rank.
      uint32_t in = 0xffffffffu >> (32 - kLpQuads * 4);
      if (base < shift || base + kLpTile > v1) {
#pragma unroll
        for (int i = 0; i < kLpQuads * 4; ++i) {
          const int p = base + ((i >> 2) * 32 + lane) * 4 + (i & 3);
          if (p < shift || p >= v1) {
            v[i] = -INFINITY;
            in &= ~(1u << i);
          }
        }
      }
      float top[kLpQuads];
#pragma unroll
      for (int q = 0; q < kLpQuads; ++q)
        top[q] = fmaxf(fmaxf(v[4 * q], v[4 * q + 1]), fmaxf(v[4 * q + 2], v[4 * q + 3]));
      float mt = top[0];
#pragma unroll
      for (int q = 1; q < kLpQuads; ++q) mt = fmaxf(mt, top[q]);
      if (mt > st.m) {
        if (st.m != -INFINITY) {
          const float d = st.m - mt, f = ex2(d * kLog2e);
          const float2 f2 = make_float2(f, f);
          t2 = f == 0.0f ? make_float2(0.f, 0.f) : mul2(fma2(l2, make_float2(d, d), t2), f2);
          l2 = mul2(l2, f2);
        }
        st.m = mt;
      }
      const float zero = st.m == -INFINITY ? 0.0f : -st.m;
#pragma unroll
      for (int i = 0; i < kLpQuads * 2; ++i) {
        float2 d = add2(make_float2(v[2 * i], v[2 * i + 1]), make_float2(zero, zero));
        const float2 p = mul2(d, make_float2(kLog2e, kLog2e));
        const float2 e = make_float2(ex2(p.x), ex2(p.y));
        l2 = add2(l2, e);
        d = make_float2(fmaxf(d.x, -3.4e38f), fmaxf(d.y, -3.4e38f));   // 0 * -inf
        t2 = fma2(e, d, t2);
      }
      if (mt > one) {
#pragma unroll
        for (int i = 0; i < kLpQuads * 4; ++i) st.above += v[i] > one;
      }
      const bool nan = l2.x != l2.x || l2.y != l2.y;   // a NaN may be all that a lane has
      if (k) {
        if (first) {
          // Two maxima of eight values a lane; k values reach the k-th of 32
          // lanes' larger ones, or half of k of each kind the lower half-k-th.
          uint32_t best[2];
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            best[q] = in >> (8 * q) & 255u ? order_key(fmaxf(top[2 * q], top[2 * q + 1])) : 0u;
            if (nan) {               // a NaN may be all that there is
              best[q] = 0u;
#pragma unroll
              for (int i = 8 * q; i < 8 * q + 8; ++i)
                if (in >> i & 1u) best[q] = max(best[q], order_key(v[i]));
            }
          }
          uint32_t kth;
          if (k <= 32)
            kth = kth_largest(max(best[0], best[1]), k, lane);
          else
            kth = min(kth_largest(best[0], (k + 1) / 2, lane),
                      kth_largest(best[1], (k + 1) / 2, lane));
          // (below -inf there is NaN only)
          thr = kth > 0x007fffffu ? key_value(kth) : -INFINITY;
          first = false;
        }
        // (a NaN is not below the threshold, and is sorted out by its key)
        int n = held;
        if (__any_sync(0xffffffffu, !(mt < thr) || nan)) {
#pragma unroll
          for (int q = 0; q < kLpQuads; ++q)
            if (__any_sync(0xffffffffu, !(top[q] < thr) || nan)) {
#pragma unroll
              for (int i = 4 * q; i < 4 * q + 4; ++i) {
                const bool hit = !(v[i] < thr) && (in >> i & 1u);
                const uint32_t who = __ballot_sync(0xffffffffu, hit);
                const int at = n + __popc(who & ((1u << lane) - 1u));
                if (hit && at < kLpCap)
                  list[at] = packed(v[i], base + (q * 32 + lane) * 4 + (i & 3) - shift);
                n += __popc(who);
              }
            }
          __syncwarp();
        }
        if (n > kLpCap || (n >= 32 && n >= 2 * k)) {
          if (n > kLpCap) {
            // The tile's k best, each the largest below the one before.
            unsigned long long below = ~0ull;
            n = held;
#pragma unroll 1
            for (int i = 0; i < k; ++i) {
              unsigned long long b = 0;
#pragma unroll 1
              for (int q = 0; q < kLpQuads; ++q) {
                const float4 f = here[q * 32 + lane];
                const float u[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  const unsigned long long key =
                      packed(u[e], base + (q * 32 + lane) * 4 + e - shift);
                  if ((in >> (4 * q + e) & 1u) && key < below && key > b) b = key;
                }
              }
#pragma unroll 1
              for (int o = 16; o > 0; o >>= 1) {
                const unsigned long long other = __shfl_xor_sync(0xffffffffu, b, o);
                b = other > b ? other : b;
              }
              if (b == 0) break;
              below = b;
              if (n == kLpCap) {
                __syncwarp();
                keep_best(list, n, k, lane);
                n = k;
              }
              if (lane == 0) list[n] = b;
              ++n;
            }
            __syncwarp();
          }
          if (n > k) {
            keep_best(list, n, k, lane);
            n = k;
          }
          // Full and in order: what comes later loses a tie, so it has to be
          // larger than the last.
          const uint32_t kth = (uint32_t)(list[k - 1] >> 32);
          if (n == k && kth) thr = fmaxf(thr, key_value(kth + 1));
        }
        held = n;
      }
      start_tile(here, x, base + kLpSlots * kStep, shift, v1, lane);
    }
    st.l = l2.x + l2.y;
    st.t = t2.x + t2.y;
    st.join_lanes();
    if (k) keep_best(list, held, k, lane);
    if constexpr (ROW_PER_WARP) {
      const int done = r, done_id = id;
      const float done_one = one;
      const bool done_has = has;
      const int step = warps * gridDim.x;
      const bool more = step < a.rows - r;   // (r + step may pass 2^31)
      r += more ? step : 0;
      if (more) take_row();            // its copies start before this row's results
      emit(a, done, st, list, lane, 32, done_one, done_id, done_has);
      __syncwarp();
      if (!more) return;
      continue;
    }
    if (lane == 0) {
      parts[warp] = st;
      counts[warp] = min(held, k);
    }
    __syncthreads();
    auto join_parts = [&](const Stats* p, int n) {   // by every warp
      st = {-INFINITY, 0.0f, 0.0f, 0};
      if (lane < n) st = p[lane];
      st.join_lanes();
    };
    join_parts(parts, kLpWarps);
    if (cluster > 1) {
      // Into the first CTA's shared memory.
      if (k) {
        merge_lists(lists[0], kLpCap, counts, k, joined, warp, lane);
        __syncthreads();
      }
      int n = 0;
      for (int w = 0; w < kLpWarps; ++w) n += counts[w];
      n = min(n, k);
      cluster_wait();                  // every CTA of the cluster has started
      unsigned long long* to = cl.map_shared_rank(&theirs[0][0], 0) + rank * kLpMaxTop;
      if (tid < n) to[tid] = joined[tid];
      if (tid == 0) {
        *cl.map_shared_rank(&cta_parts[rank], 0) = st;
        *cl.map_shared_rank(&cta_counts[rank], 0) = n;
      }
      cl.sync();
      if (rank != 0) return;
      join_parts(cta_parts, cluster);
      if (tid >= cluster && tid < kLpMaxCluster) cta_counts[tid] = 0;
      __syncthreads();
    }
    if (k) {
      if (cluster > 1)
        merge_lists(theirs[0], kLpMaxTop, cta_counts, k, joined, warp, lane);
      else
        merge_lists(lists[0], kLpCap, counts, k, joined, warp, lane);
      __syncthreads();
    }
    emit(a, r, st, joined, tid, kLpWarps * 32, one, id, has);
    return;
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
  if (cols > INT32_MAX - 16 * kLpWarps * kLpTile)
    return fail(SPX_ERR_UNSUPPORTED, "token_logprobs: too many columns");
  // A warp a row from two warps a CTA on, four CTAs an SM: as few warps as take
  // the same number of rounds, so that they end together.  Of 32000 columns, us
  // with a CTA and with a warp a row: 600 rows 39, 56; 1200: 62, 59; 2368: 109,
  // 71; 4096: 182, 102.  Else a CTA a row, or several while that makes no more
  // than three an SM and half of a CTA's warps still have a tile: 1 row with 1,
  // 2, 4, 8 CTAs: 14.5, 12.0, 8.2, 6.5; 64 rows: 15.9, 12.7, 9.8, 11.2; 148 rows:
  // 16.3, 14.4, 17.5, 21.2; 200 rows: 19.1, 17.5, 20.4, 27.4.
  const bool row_per_warp = rows >= kLpPerSm * kNumSms * 2;
  const int rounds = (int)ceil_div(rows, kLpPerSm * kNumSms * kLpWarps);
  const int warps = row_per_warp ? (int)ceil_div(rows, kLpPerSm * kNumSms * rounds) : kLpWarps;
  int cluster = 1;
  while (cluster < kLpMaxCluster && (int64_t)rows * cluster * 2 <= 3 * kNumSms &&
         cols / cluster > kLpWarps * kLpTile / 2)
    cluster *= 2;
  const int seg = (int)ceil_div(ceil_div(cols + 3, cluster), 4) * 4;
  const LpArgs a{x, ld, rows, cols, ids, logprobs, entropy, rank, top_k, top_ids, top_logprobs};
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(row_per_warp ? kLpPerSm * kNumSms : rows * cluster));
  cfg.blockDim = dim3((unsigned)warps * 32);
  cfg.dynamicSmemBytes = kLpRing;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)cluster;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  auto kern = row_per_warp ? token_logprobs_kernel<true> : token_logprobs_kernel<false>;
  int rc = check_cuda(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                           (int)kLpRing),
                      "token_logprobs: smem attribute");
  if (rc) return rc;
  rc = check_cuda(cudaLaunchKernelEx(&cfg, kern, a, cluster, seg), "token_logprobs");
  return rc ? rc : after_launch(cnt, "token_logprobs");
}

}  // namespace spx
