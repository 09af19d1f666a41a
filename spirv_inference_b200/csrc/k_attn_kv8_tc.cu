// Attention over the 8-bit cache for many rows (prompts), on tcgen05.
//
// A CTA takes 128 rows, (new token, head of the group) pairs of one sequence
// and kv head, and walks the keys they see in tiles of 64:
//
//   two warps turn a tile's K and V into fp16 (int8 is exact there) in shared
//     memory, 16 bytes of a row a thread;
//   S = Q K^T goes into TMEM, q as fp16 hi + lo, two products;
//   four warps, one row a thread, read S, take the softmax step, and write P,
//     as fp16 hi + lo, over S;
//   O = P V, two products with P from TMEM, each tile into a fresh accumulator;
//   the row's thread adds O to its output in registers, in fp32 (the tensor
//     core's sums round towards zero: over a whole prompt that shows).
//
// S and O have two buffers each, so that the products of a tile run under the
// softmax of its neighbours; one more warp issues them.  (With tiles of 128
// keys, one buffer and the issue on a softmax thread, 128 keys took 10.7
// thousand cycles, 3.3 of them issuing and 5.3 of softmax.)  With few row tiles
// the keys go to the CTAs of a cluster, which join their outputs at the end.
//
// K and V rows are 128 bytes of 64 values under the 128-byte swizzle: K is a
// K-major operand, V, whose keys are the reduction, an MN-major one of the same
// layout.  Turning bytes into fp16 leaves each four values in the order 0, 2,
// 1, 3: q is stored in that order too, and the output comes out in it.
//
// A tile with rows of the tail (fp32) is two tiles: the hi parts, each row scaled
// by a power of two, and the lo parts, whose products with the hi parts of q and p
// are added.
//
// Four prompts of 777 to 1024 tokens onto 0 to 1000, 32 heads of 64 on 4 kv
// heads: 128 us, 0.45 PFLOP/s of fp16 products, the weights another 104.  What
// bounds it: no unit (issue slots 45 % of the active cycles, exponentials 25,
// tensor pipe 24), but a chain in too few warps.  Two CTAs an SM (D = 64) are two
// softmax warps a scheduler, and each of them, for every 64 keys, waits for O, then
// for S, and takes the maximum, the exponentials, the split and the store in turn.
#include <cooperative_groups.h>
#include <cuda.h>

#include <mutex>
#include <type_traits>

#include "attn_kv8.cuh"
#include "sm100_prims.cuh"

namespace spx {

// Of each graph that runs these kernels, a word that a wait which gave up sets.
constexpr int kAtSlots = 1024;
__device__ int g_at_status[kAtSlots];

namespace {

__device__ __forceinline__ int* status_of(const AttnArgs& a) { return g_at_status + a.slot; }

using namespace sm100;
namespace cg = cooperative_groups;

constexpr int kRows = 128, kTile = 64, kGroups = kTile / 16;
constexpr int kThreads = 256;             // softmax, conversion
constexpr int kMaxSplit = 8;              // CTAs that share a row tile's keys
constexpr uint32_t kAtom = 128 * 128;     // 128 rows of 128 bytes
constexpr unsigned long long kWaitNs = 2000000000ull;
constexpr float kMaxFloat = 3.4028234663852886e38f;

template <int D>
struct TcShape {
  static constexpr int kAtoms = D / 64;
  static constexpr int kSlots = 4;
  static constexpr uint32_t kQ = kAtoms * kAtom;         // hi or lo
  static constexpr uint32_t kHalf = kAtoms * kTile * 128;  // K or V of a slot
  static constexpr uint32_t kSlot = 2 * kHalf;
  static constexpr uint32_t kTmem = D == 64 ? 256 : 512;   // S / P: 2 x 64 columns, O: 2 x D
  static constexpr int kBlocks = D == 64 ? 2 : 1;        // CTAs an SM
  // Two CTAs an SM leave 128 registers a thread; the conversion warps give
  // some of theirs to the softmax warps, which hold a row of the output.
  static constexpr int kRegs = 128, kSoftmaxRegs = 168, kConvertRegs = 88;
  static_assert(kSoftmaxRegs + kConvertRegs <= 2 * kRegs, "within what the launch has");
};

struct Aux {                   // of the slots
  // Closed blocks: of 16 keys the scales (NaN: V has a NaN or an infinity), and
  // the share of V's in the tile's largest.
  float k_scale[4][kGroups], v_scale[4][kGroups];
  float share[4][kGroups];
  float back[4];
  // A tile with rows of the tail: the same of each key.
  alignas(16) float k_key[4][kTile];
  alignas(16) float v_key[4][kTile];
  uint64_t full[4], empty[4], q_full, s_ready[2], p_ready[2], done;
  uint32_t tmem;
  int abort_flag;
};

// fp16 A and B, fp32 sums; b_mn: B's rows are the reduction.
__host__ __device__ constexpr uint32_t idesc_f16(int m, int n, int b_mn) {
  return (1u << 4) | ((uint32_t)b_mn << 16) | ((uint32_t)(n >> 3) << 17) |
         ((uint32_t)(m >> 4) << 24);
}
__device__ __forceinline__ void mma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                        uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate));
}
// The same with A in TMEM.
__device__ __forceinline__ void mma_f16_ta(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc,
                                           uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(accumulate));
}
// MN-major operand in the same layout as sw128_desc's: 64 values a row, 8-row
// groups of the reduction 1024 bytes apart, the next 64 values an atom away.
__device__ __forceinline__ uint64_t mn_desc(uint32_t saddr) {
  return (sw128_desc(saddr) & ~(0x3fffull << 16)) | ((uint64_t)((kTile * 128) >> 4) << 16);
}
// What k-step i of a K-major operand of `rows` rows adds to its descriptor.
__host__ __device__ constexpr uint64_t k_step(int i, int rows) {
  return ((uint64_t)(i >> 2) * rows * 128 + (i & 3) * 32) >> 4;
}
__device__ __forceinline__ void tmem_st_32x32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31};" ::"r"(
          r[0]),
      "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
      "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]),
      "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]),
      "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]),
      "r"(r[30]), "r"(r[31]), "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_wait_st() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

// Of a warp that goes together, the lane that issues.
__device__ __forceinline__ bool first_lane() { return (threadIdx.x & 31) == 0; }

// 16 bytes of piece `c` (eight values) of row `r` of an operand of ROWS rows.
template <int ROWS>
__device__ __forceinline__ uint4* piece(uint8_t* base, int r, int c) {
  return reinterpret_cast<uint4*>(base + (c >> 3) * (ROWS * 128) + r * 128 +
                                  (((c & 7) ^ (r & 7)) << 4));
}
// Eight int8 values as fp16, each four in the order 0, 2, 1, 3.
__device__ __forceinline__ uint4 eight(uint32_t a, uint32_t b, uint32_t mask) {
  return make_uint4(even_bytes(a, mask), even_bytes(a >> 8, mask), even_bytes(b, mask),
                    even_bytes(b >> 8, mask));
}
// Eight fp32 values times `by` as fp16 hi and lo, in that order.
__device__ __forceinline__ void eight_split(const float4 x, const float4 y, float by, uint4& hi,
                                            uint4& lo) {
  split2(x.x * by, x.z * by, hi.x, lo.x);
  split2(x.y * by, x.w * by, hi.y, lo.y);
  split2(y.x * by, y.z * by, hi.z, lo.z);
  split2(y.y * by, y.w * by, hi.w, lo.w);
}
__device__ __forceinline__ bool odd_bits(float x) {
  return (__float_as_uint(x) & 0x7f800000u) == 0x7f800000u;
}
__device__ __forceinline__ float4 finite4(float4 v, bool& odd) {
  if (odd_bits(v.x)) odd = true, v.x = 0.f;
  if (odd_bits(v.y)) odd = true, v.y = 0.f;
  if (odd_bits(v.z)) odd = true, v.z = 0.f;
  if (odd_bits(v.w)) odd = true, v.w = 0.f;
  return v;
}

// What every role knows of the CTA's work.
template <int D>
struct Unit {
  int h, b, r0, rows, len, total, closed, lim, first, tiles, G;
  int all_see;           // the last slot that every row sees
  __device__ __forceinline__ Unit(const AttnArgs& a, int cluster) {
    G = a.Hq / a.c.kv_heads;
    // the last rows see the most keys: first, and those of all heads
    const int heads = a.c.batch * a.c.kv_heads, unit = blockIdx.x / cluster;
    const int at = unit / heads, bh = unit - at * heads;
    b = bh / a.c.kv_heads;
    h = bh - b * a.c.kv_heads;
    r0 = (int)(gridDim.x / cluster / heads - 1 - at) * kRows;
    const int n_new = a.new_lens ? clamp_len(a.new_lens[b], a.T) : a.T;
    rows = n_new * G;
    len = clamp_len(a.c.lens[b], a.c.max_seq);
    total = min(len + n_new, a.c.max_seq);
    closed = total / a.c.block * a.c.block;
    lim = min(len + a.div_g(min(r0 + kRows, rows) - 1) + 1, a.c.max_seq);
    all_see = min(len + a.div_g(r0), total - 1);
    // this CTA's tiles, `tiles` from `first` on
    const int all = (lim + kTile - 1) / kTile, rank = blockIdx.x % cluster;
    first = (int)((int64_t)all * rank / cluster);
    tiles = (int)((int64_t)all * (rank + 1) / cluster) - first;
  }
  __device__ __forceinline__ int64_t row_at(const AttnArgs& a, int r) const {
    const int tk = a.div_g(r);
    return ((int64_t)b * a.T + tk) * a.Hq + h * G + (r - tk * G);
  }
  __device__ __forceinline__ bool has_tail(int tile) const {
    return closed < lim && (first + tile + 1) * kTile > closed;
  }
  // how many tiles have no rows of the tail; the others come behind them
  __device__ __forceinline__ int plain() const {
    return closed < lim ? max(0, min(tiles, closed / kTile - first)) : tiles;
  }
};

// ---- conversion of rows of q -----------------------------------------------------
// kRows rows by 128 threads.  Threads next to each other take 8 values each of
// one row, so that a warp reads whole lines (a row a thread took four times as
// long for the loads: each touched 32 lines).
template <int D, int PARTS>
struct Rows {                  // 1 / PARTS of them at a time
  static constexpr int L = D / 8, PER = 128 / L, N = kRows / PER / PARTS;
  float4 v[N][2];
  // row_of: the row's values, or null for zeros
  template <class F>
  __device__ __forceinline__ void load(int x, int part, F row_of) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float* row = row_of((part * N + i) * PER + x / L);
      const float4* from = reinterpret_cast<const float4*>(row) + x % L * 2;
      const bool is = row != nullptr;
      v[i][0] = is ? __ldg(from) : make_float4(0.f, 0.f, 0.f, 0.f);
      v[i][1] = is ? __ldg(from + 1) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
  }
  // put(row, the factor that takes its products to scores in units of log 2:
  // NaN for a row with a NaN or an infinity)
  template <class F>
  __device__ __forceinline__ void convert(int x, int part, float scale, uint8_t* hi_to,
                                          uint8_t* lo_to, F put) const {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      uint32_t mx = 0;
#pragma unroll
      for (int e = 0; e < 2; ++e)
        mx = max(max(max(__float_as_uint(v[i][e].x) & 0x7fffffffu,
                         __float_as_uint(v[i][e].y) & 0x7fffffffu),
                     max(__float_as_uint(v[i][e].z) & 0x7fffffffu,
                         __float_as_uint(v[i][e].w) & 0x7fffffffu)),
                 mx);
#pragma unroll
      for (int o = 1; o < L; o <<= 1) mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, o));
      const bool odd = mx >= 0x7f800000u;
      float down, up;
      pow2_scale(odd ? 0x3f800000u : mx, down, up);
      if (scale < 0.0f) down = -down;
      uint4 hi, lo;
      eight_split(v[i][0], v[i][1], down, hi, lo);
      const int r = (part * N + i) * PER + x / L;
      *piece<kRows>(hi_to, r, x % L) = hi;
      *piece<kRows>(lo_to, r, x % L) = lo;
      if (x % L == 0) put(r, odd ? __int_as_float(0x7fc00000) : up * (fabsf(scale) * kLog2e));
    }
  }
};

// ---- products, issued by a warp ---------------------------------------------------
template <int D>
struct Issue {
  using S = TcShape<D>;
  static constexpr uint32_t kS = idesc_f16(kRows, kTile, 0), kO = idesc_f16(kRows, D, 1);
  uint64_t q_hi, q_lo, k, v;     // descriptors; k and v of slot 0
  uint32_t tmem;
  __device__ __forceinline__ Issue(uint32_t q_hi_at, uint32_t q_lo_at, uint32_t slots, uint32_t t)
      : q_hi(sw128_desc(q_hi_at)), q_lo(sw128_desc(q_lo_at)), k(sw128_desc(slots)),
        v(mn_desc(slots + S::kHalf)), tmem(t) {}
  // Q (from q) K^T (from a slot's k) over D, to the S buffer at `to`.
  template <bool MORE>
  static __device__ __forceinline__ void scores(uint64_t q, uint64_t from, uint32_t to) {
#pragma unroll
    for (int i = 0; i < D / 16; ++i)
      mma_f16(to, q + k_step(i, kRows), from + k_step(i, kTile), kS,
              MORE || i ? 1u : 0u);
  }
  // P (at `p`; hi: PART 0, lo: PART 16 columns into each 32) V (from a slot's v)
  // over the keys, to the O buffer at `to`.
  template <int PART, bool MORE>
  static __device__ __forceinline__ void values(uint32_t p, uint64_t from, uint32_t to) {
#pragma unroll
    for (int i = 0; i < kTile / 16; ++i)
      mma_f16_ta(to, p + (i >> 1) * 32 + PART + (i & 1) * 8,
                 from + i * (2048 >> 4), kO, MORE || i ? 1u : 0u);
  }
  static __device__ __forceinline__ bool wait(const AttnArgs& a, Aux& aux, uint64_t* bar,
                                              int parity) {
    const bool ok = mb_wait(bar, parity, &aux.abort_flag, status_of(a), kWaitNs, 32);
    if (!__all_sync(0xffffffffu, ok)) return false;
    tc_after();
    return true;
  }
  // S of a tile whose rows are in slot n (and n + 1), once they are there.
  __device__ __forceinline__ bool tile_scores(const AttnArgs& a, Aux& aux, int tile, int n,
                                              bool tail) const {
    const int s = n & 3, s2 = (n + 1) & 3, j = tile & 1;
    const uint64_t from = k + (uint64_t)s * (S::kSlot >> 4);
    const uint64_t from2 = k + (uint64_t)s2 * (S::kSlot >> 4);
    const uint32_t to = tmem + j * kTile;
    if (!wait(a, aux, &aux.full[s], (n >> 2) & 1)) return false;
    if (first_lane()) {
      scores<false>(q_lo, from, to);
      scores<true>(q_hi, from, to);
      if (!tail) mma_commit(&aux.s_ready[j]);
    }
    __syncwarp();
    if (!tail) return true;
    if (!wait(a, aux, &aux.full[s2], ((n + 1) >> 2) & 1)) return false;
    if (first_lane()) {
      scores<true>(q_hi, from2, to);
      mma_commit(&aux.s_ready[j]);
    }
    __syncwarp();
    return true;
  }
  // O of a tile, once P is there.
  __device__ __forceinline__ bool tile_values(const AttnArgs& a, Aux& aux, int tile, int n,
                                              bool tail) const {
    const int s = n & 3, s2 = (n + 1) & 3, j = tile & 1;
    const uint64_t from = v + (uint64_t)s * (S::kSlot >> 4);
    const uint64_t from2 = v + (uint64_t)s2 * (S::kSlot >> 4);
    const uint32_t p = tmem + j * kTile, to = tmem + 2 * kTile + j * D;
    if (!wait(a, aux, &aux.p_ready[j], (tile >> 1) & 1)) return false;
    if (first_lane()) {
      values<16, false>(p, from, to);
      values<0, true>(p, from, to);
      if (tail) values<0, true>(p, from2, to);
      mma_commit(&aux.empty[s]);
      if (tail) mma_commit(&aux.empty[s2]);
    }
    __syncwarp();
    return true;
  }
};

// All products of the tiles, by one lane: a commit follows all issued before it.
template <int D>
__device__ __forceinline__ void issue_tiles(const AttnArgs& a, const Unit<D>& u, Aux& aux,
                                            const Issue<D>& issue) {
  bool ok = Issue<D>::wait(a, aux, &aux.q_full, 0);
  int n = 0, n1 = 0, n2 = 0;   // the slots of tiles j, j - 1, j - 2
  for (int j = 0; ok && j < u.tiles + 2; ++j) {
    if (j >= 2) ok = issue.tile_values(a, aux, j - 2, n2, u.has_tail(j - 2));
    n2 = n1;
    if (!ok || j >= u.tiles) continue;
    const bool tail = u.has_tail(j);
    ok = issue.tile_scores(a, aux, j, n, tail);
    n1 = n;
    n += tail ? 2 : 1;
  }
  if (first_lane()) {
    mma_commit(&aux.done);
    if (!ok) {
      // The products in flight end before shared memory and TMEM are given up.
      volatile int never = 0;
      mb_wait(&aux.done, 0, &never, status_of(a), 200000000ull, 64);
    }
  }
  __syncwarp();
}

// ---- conversion of keys and values ------------------------------------------------
// 16 rows of the tail, `n` of them there, as hi and lo parts of the operand's
// rows r0 on, by a warp: a row's lanes next to each other, four loads at a time
// (more cost the loop over closed tiles its registers).  Each row is scaled by a
// power of two of its own, which goes to `factor`.  V: a NaN or an infinity
// becomes zero and makes its key's factor NaN.
template <int D, bool V>
__device__ __forceinline__ void tail_group(uint8_t* hi_to, uint8_t* lo_to, int r0,
                                           const float* rows, int n, float* factor, int lane) {
  constexpr int L = D / 4, PER = 32 / L, N = 16 / PER;
  const int c = lane % L, r = lane / L;
#pragma unroll 1
  for (int from = 0; from < N; from += 4) {
    float4 v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = (from + i) * PER + r;
      v[i] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (row < n) v[i] = reinterpret_cast<const float4*>(rows)[row * L + c];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      bool odd = false;
      if (V) v[i] = finite4(v[i], odd);
      uint32_t mx = max(max(finite_abs(v[i].x), finite_abs(v[i].y)),
                        max(finite_abs(v[i].z), finite_abs(v[i].w)));
#pragma unroll
      for (int o = 1; o < L; o <<= 1) mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, o));
      const uint32_t who = __ballot_sync(0xffffffffu, odd);
      float down, up;
      pow2_scale(mx, down, up);
      if (V) {
        // To 2^10, between the 2^14 that would suit the values and the 2^7 of int8
        // ones: a tile's keys share the unit of their weights, whose low halves
        // are multiples of 2^-24, and both then lose 2^-36 of the largest at most.
        down *= 0x1p-4f;
        up *= 0x1p4f;
      }
      uint2 hi, lo;
      split2(v[i].x * down, v[i].z * down, hi.x, lo.x);
      split2(v[i].y * down, v[i].w * down, hi.y, lo.y);
      const int to = r0 + (from + i) * PER + r;
      reinterpret_cast<uint2*>(piece<kTile>(hi_to, to, c >> 1))[c & 1] = hi;
      reinterpret_cast<uint2*>(piece<kTile>(lo_to, to, c >> 1))[c & 1] = lo;
      if (c == 0)
        factor[to] = (L == 32 ? who : who >> (r * L) & 0xffffu) ? __int_as_float(0x7fc00000) : up;
    }
  }
}

template <int D>
__device__ __forceinline__ void convert_tiles(const AttnArgs& a, const Unit<D>& u, uint8_t* slots,
                                              Aux& aux, int r) {
  using S = TcShape<D>;
  // (few values are kept: registers are short)
  const int64_t bh = (int64_t)u.b * a.c.kv_heads + u.h;
  const int shift = 31 - __clz(a.c.block);
  uint32_t mask;
  asm volatile("mov.b32 %0, 0x00ff00ff;" : "=r"(mask));
  // Rows of closed blocks: 16 bytes of a row a thread, a warp's next to each
  // other.  Scales: by the first four lanes, of a group each.
  constexpr int L = D / 16, PER = kTile / L;
  const int r16 = r / L, c16 = r % L;
  uint4 kr[L], vr[L];
  float k_sc = 0.0f, v_sc = 0.0f;
  auto load = [&](int tile) {
    const int j0 = (u.first + tile) * kTile, left = u.closed - j0 - r16;
    const int64_t at = (bh * a.c.max_seq + j0 + r16) * D + c16 * 16;
#pragma unroll
    for (int i = 0; i < L; ++i)
      if (i * PER < left) kr[i] = __ldg(reinterpret_cast<const uint4*>(a.c.k + at) + i * PER * L);
#pragma unroll
    for (int i = 0; i < L; ++i)
      if (i * PER < left) vr[i] = __ldg(reinterpret_cast<const uint4*>(a.c.v + at) + i * PER * L);
    const int key = j0 + r * 16;
    k_sc = v_sc = 0.0f;
    if (r < kGroups && key < u.closed) {
      const int64_t blk = ((bh * a.c.max_seq) >> shift) + (key >> shift);
      k_sc = __ldg(a.c.k_scale + blk);
      v_sc = __ldg(a.c.v_scale + blk);
    }
  };
  auto store = [&](uint8_t* k_to, uint8_t* v_to, int left) {
#pragma unroll
    for (int i = 0; i < L; ++i) {
      const int to = i * PER + r16;
      if (to >= left) break;
      *piece<kTile>(k_to, to, 2 * c16) = eight(kr[i].x, kr[i].y, mask);
      *piece<kTile>(k_to, to, 2 * c16 + 1) = eight(kr[i].z, kr[i].w, mask);
      *piece<kTile>(v_to, to, 2 * c16) = eight(vr[i].x, vr[i].y, mask);
      *piece<kTile>(v_to, to, 2 * c16 + 1) = eight(vr[i].z, vr[i].w, mask);
    }
  };
  auto shares = [&](int s) {                 // by the first warp, lane i with group i's v_sc
    float ref = v_sc <= kMaxFloat ? fmaxf(v_sc, kMinRef) : kMinRef;
#pragma unroll
    for (int o = 1; o < kGroups; o <<= 1) ref = fmaxf(ref, __shfl_xor_sync(0xffffffffu, ref, o));
    if (r < kGroups) aux.share[s][r] = v_sc * (kPUp / ref);
    if (r == 0) aux.back[s] = ref * (1.0f / kPUp);
  };
  auto put_scales = [&](int s) {             // by lane i of the first warp, group i's
    aux.k_scale[s][r] = k_sc;
    aux.v_scale[s][r] = v_sc <= kMaxFloat ? v_sc : __int_as_float(0x7fc00000);
  };
  auto drained = [&](int slot, int m) {
    return mb_wait(&aux.empty[slot], ((m >> 2) & 1) ^ 1, &aux.abort_flag, status_of(a), kWaitNs,
                   64);
  };
  // (Apart from the others, whose code cost this loop its registers: 32 us when
  // four prompts took 172.)
  // Tiles of closed blocks only, each one's bytes on their way while the one
  // before drains.
  const int whole = max(0, min(u.tiles, u.closed / kTile - u.first));
  if (whole > 0) load(0);
  int n = 0;                   // the tile's slot
  for (; n < whole; ++n) {
    const int s = n & 3;
    if (!__all_sync(0xffffffffu, drained(s, n))) return;
    uint8_t* k_to = slots + s * S::kSlot;
    store(k_to, k_to + S::kHalf, kTile);
    if (r < 32) {
      if (r < kGroups) put_scales(s);
      shares(s);
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    mb_arrive(&aux.full[s]);
    if (n + 1 < whole) load(n + 1);
  }
  // The others.
  for (int tile = whole; tile < u.tiles; ++tile) {
    const int j0 = (u.first + tile) * kTile;
    const bool tail = u.has_tail(tile);
    const int s = n & 3, s2 = (n + 1) & 3;
    load(tile);
    bool ok = drained(s, n);
    if (tail) ok = ok && drained(s2, n + 1);
    if (!__all_sync(0xffffffffu, ok)) return;
    uint8_t* k_to = slots + s * S::kSlot;
    uint8_t* v_to = k_to + S::kHalf;
    uint8_t* k_lo = slots + s2 * S::kSlot;
    uint8_t* v_lo = k_lo + S::kHalf;
    if (tail) {                // the keys of closed blocks
      const int key = j0 + r;
      if (key < u.closed) {
        const int64_t blk = ((bh * a.c.max_seq) >> shift) + (key >> shift);
        const float v = __ldg(a.c.v_scale + blk);
        aux.k_key[s][r] = __ldg(a.c.k_scale + blk);
        aux.v_key[s][r] = v <= kMaxFloat ? v : __int_as_float(0x7fc00000);
      }
    } else if (r < kGroups) {  // (no row sees a key behind the closed ones)
      put_scales(s);
    }
    store(k_to, v_to, u.closed - j0);
    __syncwarp();
    // Groups of 16 keys, two of the tile's four a warp: closed ones have no
    // lo part; the others come from the tail if some row sees it.
#pragma unroll 1
    for (int grp = r >> 5 << 1; grp < (r >> 5 << 1) + kGroups / 2; ++grp) {
      const int key = j0 + grp * 16;
      if (key < u.closed || !tail) {
        if (tail || key >= u.closed)
          for (int i = r & 31; i < D * 2; i += 32) {
            const int row = grp * 16 + i / (D / 8), c = i % (D / 8);
            *piece<kTile>(tail ? k_lo : k_to, row, c) = make_uint4(0, 0, 0, 0);
            *piece<kTile>(tail ? v_lo : v_to, row, c) = make_uint4(0, 0, 0, 0);
          }
        continue;
      }
      const int64_t at = ((bh << shift) + (key & (a.c.block - 1))) * D;
      const int rows = max(0, min(u.total - key, 16));
      tail_group<D, false>(k_to, k_lo, grp * 16, a.c.k_tail + at, rows, aux.k_key[s], r & 31);
      tail_group<D, true>(v_to, v_lo, grp * 16, a.c.v_tail + at, rows, aux.v_key[s], r & 31);
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    mb_arrive(&aux.full[s]);
    if (tail) mb_arrive(&aux.full[s2]);
    n += tail ? 2 : 1;
  }
}

// ---- softmax: one row a thread -------------------------------------------------
template <int D>
__device__ __forceinline__ bool softmax_tiles(const AttnArgs& a, const Unit<D>& u, Aux& aux,
                                              const float* q_scale, uint32_t tmem, int x,
                                              float (&o)[D], float& m, float& l) {
  const uint32_t lanes = tmem + ((uint32_t)((x >> 5) * 32) << 16);
  auto wait = [&](uint64_t* b, int parity) {
    const bool ok = mb_wait(b, parity, &aux.abort_flag, status_of(a), kWaitNs, 32);
    return __all_sync(0xffffffffu, ok) != 0;   // a warp goes on or ends as one
  };
  if (!wait(&aux.q_full, 0)) return false;
  const float qs = q_scale[x];
  const int last = min(u.len + a.div_g(min(u.r0 + x, u.rows - 1)), u.total - 1);
  m = -INFINITY;
  l = 0.0f;
  // of the tile before, and of the one before that, whose output comes next
  float corr1 = 0.0f, back1 = 0.0f, corr2 = 0.0f, back2 = 0.0f;
  // o = o corr + back * (P V of `tile`)
  auto take_output = [&](int tile, float corr, float back) {
#pragma unroll
    for (int c = 0; c < D / 32; ++c) {
      float v[32];
      tmem_ld_32x32(lanes + 2 * kTile + (tile & 1) * D + c * 32, v);
#pragma unroll
      for (int e = 0; e < 32; e += 2) {
        const float2 r = fma2(make_float2(o[c * 32 + e], o[c * 32 + e + 1]),
                              make_float2(corr, corr),
                              mul2(make_float2(v[e], v[e + 1]), make_float2(back, back)));
        o[c * 32 + e] = r.x;
        o[c * 32 + e + 1] = r.y;
      }
    }
  };
  // A tile's S and the slot of its scales, `n`, are there, and O of two tiles back,
  // which is taken.
  auto begin = [&](int tile, int n) {
    if (!wait(&aux.full[n & 3], (n >> 2) & 1)) return false;
    if (!wait(&aux.s_ready[tile & 1], (tile >> 1) & 1)) return false;
    tc_after();
    // The products before this tile's S are done, P V of two tiles back too.
    if (tile >= 2) take_output(tile - 2, corr2, back2);
    return true;
  };
  // A tile's P is there: its part of the sum, what it does to the outputs before
  // it, and what takes its output to its size.
  auto end = [&](int tile, float2 sum, float corr, float back) {
    l = fmaf(l, corr, sum.x + sum.y);
    corr2 = corr1;
    back2 = back1;
    corr1 = corr;
    back1 = back;
    tmem_wait_st();
    tc_before();
    mb_arrive(&aux.p_ready[tile & 1]);
  };
  const int plain = u.plain();
  for (int tile = 0; tile < plain; ++tile) {
    const int s = tile & 3, j0 = (u.first + tile) * kTile;
    if (!begin(tile, tile)) return false;
    const uint32_t t_s = lanes + (tile & 1) * kTile;
    const bool mask = j0 + kTile - 1 > u.all_see;
    const int seen = last - j0;         // the last column that the row sees
    float v[kTile];
#pragma unroll
    for (int c = 0; c < kTile / 32; ++c)
      tmem_ld_32x32_async(t_s + c * 32, reinterpret_cast<uint32_t(&)[32]>(v[c * 32]));
    tmem_wait_ld();
    settled(v);
    float f[kGroups], mt = -INFINITY;
    if (mask) {
#pragma unroll
      for (int e = 0; e < kTile; ++e)
        if (e > seen) v[e] = -INFINITY;
    }
#pragma unroll
    for (int i = 0; i < kGroups; ++i) {
      f[i] = aux.k_scale[s][i] * qs;
      float top = v[i * 16];
#pragma unroll
      for (int e = 1; e < 16; ++e) top = fmaxf(top, v[i * 16 + e]);
      // (a factor of 0 or NaN would make NaN of -inf, which fmaxf passes over)
      mt = fmaxf(mt, top * f[i]);
    }
    const float mn = fmaxf(m, mt), base = mn == -INFINITY ? 0.0f : mn;
    const float corr = ex2(m - base);
    m = mn;
    float2 sum = make_float2(0.f, 0.f);
    auto weigh = [&](auto tag, float by) {
      constexpr bool masked = decltype(tag)::value;
#pragma unroll
      for (int c = 0; c < kTile / 32; ++c) {
        uint32_t p[32];
#pragma unroll
        for (int e = 0; e < 32; e += 2) {
          const int k = c * 32 + e;
          const float share = masked ? aux.v_scale[s][k / 16] * by : aux.share[s][k / 16];
          float2 w = fma2(make_float2(v[k], v[k + 1]), make_float2(f[k / 16], f[k / 16]),
                          make_float2(-base, -base));
          w = make_float2(ex2(w.x), ex2(w.y));
          if (masked) {
            if (k > seen) w.x = 0.0f;
            if (k + 1 > seen) w.y = 0.0f;
          }
          sum = add2(sum, w);
          w = mul2(w, make_float2(share, share));
          if (masked) {                // (a share may be NaN)
            if (k > seen) w.x = 0.0f;
            if (k + 1 > seen) w.y = 0.0f;
          }
          split2(w.x, w.y, p[e / 2], p[16 + e / 2]);
        }
        tmem_st_32x32(t_s + c * 32, p);
      }
    };
    float back;
    if (mask) {
      // Values are taken beside the largest that the row sees: others, later ones,
      // do not matter to it.
      float most = kMinRef;
#pragma unroll
      for (int i = 0; i < kGroups; ++i)
        if (i * 16 <= seen) most = fmaxf(most, aux.v_scale[s][i]);
      weigh(std::true_type(), kPUp / most);
      back = most * (1.0f / kPUp);
    } else {
      weigh(std::false_type(), 0.0f);
      back = aux.back[s];
    }
    end(tile, sum, corr, back);
  }
  // Tiles with rows of the tail, by each key's own factors: apart, and in halves
  // with S read twice, since their code and their registers in the other loop's way
  // took 128 to 143 us over four prompts of 1024.
#pragma unroll 1
  for (int tile = plain; tile < u.tiles; ++tile) {
    const int n = 2 * tile - plain, s = n & 3, seen = last - (u.first + tile) * kTile;
    if (!begin(tile, n)) return false;
    const uint32_t t_s = lanes + (tile & 1) * kTile;
    float mt = -INFINITY, most = kMinRef;
    // a half's scores, in units of log 2
    auto scores = [&](int c, float (&v)[32]) {
      tmem_ld_32x32(t_s + c * 32, v);
#pragma unroll
      for (int e = 0; e < 32; ++e)
        v[e] = c * 32 + e > seen ? -INFINITY : v[e] * (aux.k_key[s][c * 32 + e] * qs);
    };
#pragma unroll 1
    for (int c = 0; c < kTile / 32; ++c) {
      float v[32];
      scores(c, v);
#pragma unroll
      for (int e = 0; e < 32; ++e) {
        mt = fmaxf(mt, v[e]);
        if (c * 32 + e <= seen) most = fmaxf(most, aux.v_key[s][c * 32 + e]);
      }
    }
    const float mn = fmaxf(m, mt), base = mn == -INFINITY ? 0.0f : mn;
    const float corr = ex2(m - base), by = kPUp / most;
    m = mn;
    float2 sum = make_float2(0.f, 0.f);
#pragma unroll 1
    for (int c = 0; c < kTile / 32; ++c) {
      float v[32];
      uint32_t p[32];
      scores(c, v);
#pragma unroll
      for (int e = 0; e < 32; e += 2) {
        const int k = c * 32 + e;
        float2 w = make_float2(ex2(v[e] - base), ex2(v[e + 1] - base));
        sum = add2(sum, w);
        w.x = k > seen ? 0.0f : w.x * (aux.v_key[s][k] * by);   // (a factor may be NaN)
        w.y = k + 1 > seen ? 0.0f : w.y * (aux.v_key[s][k + 1] * by);
        split2(w.x, w.y, p[e / 2], p[16 + e / 2]);
      }
      tmem_st_32x32(t_s + c * 32, p);
    }
    end(tile, sum, corr, most * (1.0f / kPUp));
  }
  if (!wait(&aux.done, 0)) return false;
  tc_after();
  if (u.tiles >= 2) take_output(u.tiles - 2, corr2, back2);
  if (u.tiles >= 1) take_output(u.tiles - 1, corr1, back1);
  return true;
}

// Joins the outputs that a cluster's CTAs have of the same 128 rows: each gets
// an equal share of the rows from all, where its keys and values were.  By the
// softmax threads; the others take part in the two barriers.
template <int D>
__device__ __forceinline__ void join(const AttnArgs& a, const Unit<D>& u, uint8_t* slots,
                                     int cluster, int x, const float (&o)[D], float m, float l) {
  static_assert(kRows * (D + 2) * 4 <= TcShape<D>::kSlots * TcShape<D>::kSlot, "fits");
  cg::cluster_group cl = cg::this_cluster();
  const int rank = blockIdx.x % cluster, per = kRows / cluster;
  float* got = reinterpret_cast<float*>(slots);        // [CTA][row][D]
  float2* got_ml = reinterpret_cast<float2*>(got + kRows * D);
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  const int at = rank * per + x % per;
  float4* to = reinterpret_cast<float4*>(cl.map_shared_rank(got, x / per) + at * D);
#pragma unroll
  for (int i = 0; i < D / 4; ++i)     // each four came as 0, 2, 1, 3
    to[i] = make_float4(o[4 * i], o[4 * i + 2], o[4 * i + 1], o[4 * i + 3]);
  cl.map_shared_rank(got_ml, x / per)[at] = make_float2(m, m == m ? l : NAN);
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  const int row = x / cluster, part = x % cluster, r = u.r0 + rank * per + row;
  if (r >= u.rows) return;
  float most = -INFINITY, sum = 0.0f;
  for (int k = 0; k < cluster; ++k) most = fmaxf(most, got_ml[k * per + row].x);
  for (int k = 0; k < cluster; ++k) {
    const float2 ml = got_ml[k * per + row];
    sum = fmaf(ml.y, ml.x == -INFINITY ? 0.0f : ex2(ml.x - most), sum);
  }
  const int64_t out_row = u.row_at(a, r);
  const float inv = 1.0f / sum;
  for (int e = part * (D / cluster); e < (part + 1) * (D / cluster); e += 4) {
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int k = 0; k < cluster; ++k) {
      const float mk = got_ml[k * per + row].x, f = mk == -INFINITY ? 0.0f : ex2(mk - most);
      const float4 w = *reinterpret_cast<const float4*>(got + (k * per + row) * D + e);
      v = make_float4(fmaf(w.x, f, v.x), fmaf(w.y, f, v.y), fmaf(w.z, f, v.z), fmaf(w.w, f, v.w));
    }
    *reinterpret_cast<float4*>(a.out + out_row * D + e) =
        make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv);
  }
  if (a.lse && part == 0) a.lse[out_row] = (most + log2f(sum)) * kLn2;
}

// SPLIT: the keys are dealt to a cluster.  (Apart: the join costs the others
// registers; when four prompts of 1024 took 168 us, they took 180 with it.)
template <int D, bool SPLIT>
__global__ void __launch_bounds__(kThreads, TcShape<D>::kBlocks)
    attention_kv8_tc_kernel(const AttnArgs a, int ctas) {
  using S = TcShape<D>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* q_hi = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint8_t* q_lo = q_hi + S::kQ;
  uint8_t* slots = q_lo + S::kQ;
  __shared__ Aux aux;
  __shared__ float q_scale[kRows];
  const int warp = threadIdx.x >> 5;
  const int cluster = SPLIT ? ctas : 1;
  const Unit<D> u(a, cluster);
  if (u.r0 >= u.rows) return;                 // the whole cluster
  if (threadIdx.x == 0) {
    for (int i = 0; i < S::kSlots; ++i) {
      mb_init(&aux.full[i], kTile);
      mb_init(&aux.empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mb_init(&aux.s_ready[i], 1);
      mb_init(&aux.p_ready[i], 128);
    }
    mb_init(&aux.q_full, 128);
    mb_init(&aux.done, 1);
    aux.abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 4) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     sa(&aux.tmem)),
                 "r"(S::kTmem));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  tc_before();
  __syncthreads();
  tc_after();
  const uint32_t tmem = aux.tmem;
  if (warp < 4) {
    if constexpr (D == 64)
      asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(S::kSoftmaxRegs));
    const int x = threadIdx.x;
    float o[D], m, l;
#pragma unroll
    for (int i = 0; i < D; ++i) o[i] = 0.0f;
    const bool ok = softmax_tiles<D>(a, u, aux, q_scale, tmem, x, o, m, l);
    const int r = u.r0 + x;
    if (SPLIT) {
      join<D>(a, u, slots, cluster, x, o, ok ? m : NAN, l);
    } else if (ok && r < u.rows) {
      const int64_t at = u.row_at(a, r);
      const float inv = 1.0f / l;
      float4* out = reinterpret_cast<float4*>(a.out + at * D);
#pragma unroll
      for (int i = 0; i < D / 4; ++i)   // each four came as 0, 2, 1, 3
        out[i] = make_float4(o[4 * i] * inv, o[4 * i + 2] * inv, o[4 * i + 1] * inv,
                             o[4 * i + 3] * inv);
      if (a.lse) a.lse[at] = (m + log2f(l)) * kLn2;
    }
  } else {
    const int x = threadIdx.x - 128;
    {
      Rows<D, 1> rows;
      rows.load(x, 0, [&](int r) {
        return u.r0 + r < u.rows ? a.q + u.row_at(a, u.r0 + r) * D : nullptr;
      });
      rows.convert(x, 0, a.scale, q_hi, q_lo, [&](int r, float f) { q_scale[r] = f; });
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    mb_arrive(&aux.q_full);
    if constexpr (D == 64)
      asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(S::kConvertRegs));
    if (warp < 6) {
      convert_tiles<D>(a, u, slots, aux, x);
    } else if (warp == 6) {
      const Issue<D> issue(sa(q_hi), sa(q_lo), sa(slots), tmem);
      issue_tiles<D>(a, u, aux, issue);
    }
    if (SPLIT) {                              // (of join)
      __syncwarp();
      for (int i = 0; i < 2; ++i) {
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
      }
    }
  }
  tc_before();
  __syncthreads();
  if (warp == 4) {
    tc_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem),
                 "r"(S::kTmem));
  }
}

// ---------------------------------------------------------------------------
// Weights for many rows: S^T = K Q^T, 128 keys on the lanes, which stay, and
// 128 rows at a time on the columns.  Four warps turn rows of q into operands
// one tile ahead; two groups of four take every other tile, each with a half of
// TMEM, issue its products themselves and add exp(score - lse) over its rows, a
// key a thread: while one waits for its products, the other adds.  The row
// tiles are dealt to a cluster's CTAs, whose sums are added in order.  About 3
// instructions a score, and 4 a value of q, which is turned into operands again for
// every 128 keys.  Four prompts as above: 104 us (one group adding and two
// converting: 4 % more; clusters of 2 and 8 in place of 4, when this took 137: 141
// and 162).
constexpr int kWeightCluster = 4, kKeys = 128, kWeightThreads = 384;

struct WeightAux {
  alignas(16) float2 row[2][kRows];   // the row's factor, and its lse in units of log 2
  float got[kWeightCluster][kKeys];
  float k_scale[kKeys], odd_tiles[kKeys];
  uint64_t full[2], empty[2], k_full, s_ready[2], done[2];
  uint32_t tmem;
  int abort_flag;
};

template <int D>
struct WeightShape {
  static constexpr uint32_t kK = D / 64 * kAtom;       // hi or lo
  static constexpr uint32_t kSlot = 2 * D / 64 * kAtom;  // q hi, lo
  static constexpr size_t kSmem = 1024 + 2 * kK + 2 * kSlot;
};

template <int D>
__global__ void __launch_bounds__(kWeightThreads, TcShape<D>::kBlocks)
    kv8_weights_tc_kernel(const AttnArgs a, int cluster) {
  using S = WeightShape<D>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* k_hi = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint8_t* k_lo = k_hi + S::kK;
  uint8_t* slots = k_lo + S::kK;
  __shared__ WeightAux aux;
  const int warp = threadIdx.x >> 5, x = threadIdx.x & 127;   // of the first four: a key
  // the first keys are seen by the most rows: first, and those of all heads
  const int heads = a.c.batch * a.c.kv_heads, rank = blockIdx.x % cluster;
  const int unit = blockIdx.x / cluster, j0 = unit / heads * kKeys, bh = unit % heads;
  const int b = bh / a.c.kv_heads, h = bh - b * a.c.kv_heads;
  const int G = a.Hq / a.c.kv_heads, blk = a.c.block;
  const int n_new = a.new_lens ? clamp_len(a.new_lens[b], a.T) : a.T;
  const int len = clamp_len(a.c.lens[b], a.c.max_seq), total = min(len + n_new, a.c.max_seq);
  if (n_new == 0 || j0 >= total) return;      // the whole cluster
  const int closed = total / blk * blk, rows = n_new * G;
  const bool tail = j0 + kKeys > closed && closed < total;
  // Rows of tokens before the first key see none of these.
  const int first = max(0, j0 - len) * G / kRows, last = (rows + kRows - 1) / kRows;
  const int tiles = max(0, (last - first - rank + cluster - 1) / cluster);
  auto row0 = [&](int i) { return (first + rank + i * cluster) * kRows; };
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mb_init(&aux.full[i], 128);
      mb_init(&aux.empty[i], 129);     // the products, and the threads that read `row`
      mb_init(&aux.s_ready[i], 1);
      mb_init(&aux.done[i], 1);
    }
    mb_init(&aux.k_full, 128);
    aux.abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 4) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     sa(&aux.tmem)),
                 "r"(256));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  tc_before();
  __syncthreads();
  tc_after();
  if (cluster > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  const uint32_t tmem = aux.tmem;
  auto wait = [&](uint64_t* bar, int parity) {
    return mb_wait(bar, parity, &aux.abort_flag, status_of(a), kWaitNs, 32);
  };
  float w = 0.0f;
  if (warp >= 8) {
    auto row_at = [&](int r) {
      const int tk = a.div_g(r);
      return ((int64_t)b * a.T + tk) * a.Hq + h * G + (r - tk * G);
    };
    // (rows of q in two parts: all at once took registers that were not there)
    Rows<D, 2> q;
    float z = INFINITY;                // (a row that is none weighs nothing)
    auto load = [&](int i, int part) {
      if (i >= tiles) return;
      const int r0 = row0(i);
      q.load(x, part, [&](int r) { return r0 + r < rows ? a.q + row_at(r0 + r) * D : nullptr; });
      if (part == 0) z = r0 + x < rows ? a.lse[row_at(r0 + x)] : INFINITY;
    };
    load(0, 0);
    for (int i = 0; i < tiles; ++i) {
      const int s = i & 1;
      uint8_t* to = slots + s * S::kSlot;
      auto put = [&](int r, float f) { aux.row[s][r].x = f; };
      const bool drained = mb_wait(&aux.empty[s], ((i >> 1) & 1) ^ 1, &aux.abort_flag,
                                   status_of(a), kWaitNs, 128);
      if (!__all_sync(0xffffffffu, drained)) break;
      q.convert(x, 0, a.scale, to, to + S::kSlot / 2, put);
      load(i, 1);
      aux.row[s][x].y = z * kLog2e;
      q.convert(x, 1, a.scale, to, to + S::kSlot / 2, put);
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      mb_arrive(&aux.full[s]);
      load(i + 1, 0);                  // on its way while the slot is used
    }
  } else {
    if (warp < 4) {
      // The key's row, and its scale.
      const int key = j0 + x;
      float ks = 0.0f;
      if (key < closed) {
        const uint4* kp =
            reinterpret_cast<const uint4*>(a.c.k + ((int64_t)bh * a.c.max_seq + key) * D);
        uint32_t mask;
        asm volatile("mov.b32 %0, 0x00ff00ff;" : "=r"(mask));
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
          const uint4 v = __ldg(kp + i);
          *piece<kKeys>(k_hi, x, 2 * i) = eight(v.x, v.y, mask);
          *piece<kKeys>(k_hi, x, 2 * i + 1) = eight(v.z, v.w, mask);
          *piece<kKeys>(k_lo, x, 2 * i) = make_uint4(0, 0, 0, 0);
          *piece<kKeys>(k_lo, x, 2 * i + 1) = make_uint4(0, 0, 0, 0);
        }
        ks = __ldg(a.c.k_scale + (int64_t)bh * (a.c.max_seq / blk) + key / blk);
      } else {
        // a row of the tail on its own: any power of two does
        const float* row =
            key < total ? a.c.k_tail + ((int64_t)bh * blk + (key & (blk - 1))) * D : nullptr;
        const float4* from = reinterpret_cast<const float4*>(row);
        const float4 zero = make_float4(0.f, 0.f, 0.f, 0.f);
        uint32_t mx = 0;
        for (int i = 0; i < D / 4; ++i) {
          const float4 v = row ? from[i] : zero;
          mx = max(max(mx, finite_abs(v.x)),
                   max(finite_abs(v.y), max(finite_abs(v.z), finite_abs(v.w))));
        }
        float down;
        pow2_scale(mx, down, ks);
        for (int c = 0; c < D / 8; ++c) {
          uint4 hi, lo;
          eight_split(row ? from[2 * c] : zero, row ? from[2 * c + 1] : zero, down, hi, lo);
          *piece<kKeys>(k_hi, x, c) = hi;
          *piece<kKeys>(k_lo, x, c) = lo;
        }
      }
      aux.k_scale[x] = ks;
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      mb_arrive(&aux.k_full);
    }
    const uint64_t kh = sw128_desc(sa(k_hi)), kl = sw128_desc(sa(k_lo));
    const uint64_t q0 = sw128_desc(sa(slots));
    constexpr uint32_t kDesc = idesc_f16(kKeys, kRows, 0);
    auto products = [&](uint64_t k, uint64_t q, uint32_t to, uint32_t more) {
#pragma unroll
      for (int i = 0; i < D / 16; ++i)
        mma_f16(to, k + k_step(i, kKeys), q + k_step(i, kRows), kDesc, i ? 1u : more);
    };
    const int s = warp >> 2, key = j0 + x;
    const uint64_t qh = q0 + (uint64_t)s * (S::kSlot >> 4), ql = qh + (S::kSlot >> 5);
    const uint32_t to = tmem + s * kRows;
    auto hold = [&](uint64_t* bar, int parity) {     // a warp goes on or ends as one
      return __all_sync(0xffffffffu, wait(bar, parity)) != 0;
    };
    bool ok = hold(&aux.k_full, 0);
    const float ks = aux.k_scale[x];
    // The key's first row, and whether a tile has any before that of some key.
    const int r_min = max(0, key - len) * G, r_all = max(0, j0 + kKeys - 1 - len) * G;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    for (int i = s; ok && i < tiles; i += 2) {
      // (a slot is filled anew after the group has read its half of TMEM)
      if (!(ok = hold(&aux.full[s], (i >> 1) & 1))) break;
      if ((warp & 3) == 0) {
        tc_after();
        if (first_lane()) {
          products(kh, ql, to, 0u);
          if (tail) products(kl, qh, to, 1u);
          products(kh, qh, to, 1u);
          mma_commit(&aux.empty[s]);
          mma_commit(&aux.s_ready[s]);
        }
        __syncwarp();
      }
      if (!(ok = hold(&aux.s_ready[s], (i >> 1) & 1))) break;
      tc_after();
      const bool mask = row0(i) < r_all;
      const int from = r_min - row0(i);       // the first column that the key is seen by
      auto add = [&](auto tag) {
        constexpr bool masked = decltype(tag)::value;
#pragma unroll
        for (int c = 0; c < kRows / 32; ++c) {
          float v[32];
          tmem_ld_32x32(tmem + s * kRows + lanes + c * 32, v);
          float2 part = make_float2(0.f, 0.f);
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            // factor and lse of two rows
            const float4 r = *reinterpret_cast<const float4*>(&aux.row[s][c * 32 + e]);
            float2 p = fma2(make_float2(v[e], v[e + 1]),
                            mul2(make_float2(r.x, r.z), make_float2(ks, ks)),
                            make_float2(-r.y, -r.w));
            p = make_float2(ex2(p.x), ex2(p.y));
            if (masked) {
              if (c * 32 + e < from) p.x = 0.0f;
              if (c * 32 + e + 1 < from) p.y = 0.0f;
            }
            part = add2(part, p);
          }
          w += part.x + part.y;
        }
      };
      if (mask)
        add(std::true_type());
      else
        add(std::false_type());
      tc_before();
      mb_arrive(&aux.empty[s]);
    }
    if (!ok && (warp & 3) == 0 && first_lane()) {
      // The products in flight end before shared memory and TMEM are given up.
      volatile int never = 0;
      mma_commit(&aux.done[s]);
      mb_wait(&aux.done[s], 0, &never, status_of(a), 200000000ull, 64);
    }
    if (s == 1) aux.odd_tiles[x] = w;
  }
  __syncthreads();
  if (warp < 4) w += aux.odd_tiles[x];
  const bool good = !aux.abort_flag;
  if (cluster > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  cg::cluster_group cl = cg::this_cluster();
  if (warp < 4) cl.map_shared_rank(&aux.got[rank][0], 0)[x] = good ? w : __int_as_float(0x7fc00000);
  if (cluster > 1)
    cl.sync();
  else
    __syncthreads();
  if (rank == 0 && warp < 4 && j0 + x < total) {
    float sum = 0.0f;
    for (int i = 0; i < cluster; ++i) sum += aux.got[i][x];
    float* out = a.weights + ((int64_t)b * a.c.kv_heads + h) * a.c.max_seq + j0 + x;
    *out = (j0 + x < len ? *out : 0.0f) + sum;
  }
  tc_before();
  __syncthreads();
  if (warp == 4) {
    tc_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(256));
  }
}

template <int D>
int launch_tc(cudaStream_t s, const AttnArgs& a) {
  using S = TcShape<D>;
  const int64_t row_tiles = ceil_div((int64_t)a.T * (a.Hq / a.c.kv_heads), kRows);
  // Few rows: their keys go to the CTAs of a cluster, as long as there are SMs
  // without work and four tiles each.  16 tokens of 4 sequences of 300 to 1500,
  // 4 kv heads of 64, with weights: 42 us, 63 without a cluster (now 35).
  const int64_t units = row_tiles * a.c.kv_heads * a.c.batch;
  int cluster = 1;
  while (cluster < kMaxSplit && units * cluster * 2 <= S::kBlocks * kNumSms &&
         cluster * 2 * 4 <= a.c.max_seq / kTile)
    cluster *= 2;
  const int64_t grid = units * cluster;
  if (grid > INT32_MAX) return fail(SPX_ERR_UNSUPPORTED, "attention_kv8: grid too large");
  const size_t smem = 1024 + 2 * S::kQ + S::kSlots * S::kSlot;
  auto kern = cluster > 1 ? attention_kv8_tc_kernel<D, true> : attention_kv8_tc_kernel<D, false>;
  int rc = check_cuda(
      cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem),
      "attention_kv8: smem attribute");
  if (rc) return rc;
  if constexpr (D == 64) {
    // setmaxnreg draws on the registers that the launch has: with fewer than
    // it was written for, it would wait for good.
    cudaFuncAttributes f;
    if ((rc = check_cuda(cudaFuncGetAttributes(&f, kern), "attention_kv8: attributes"))) return rc;
    if (f.numRegs < S::kRegs)
      return fail(SPX_ERR_UNSUPPORTED, "attention_kv8: built with %d registers a thread",
                  f.numRegs);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)cluster;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return check_cuda(cudaLaunchKernelEx(&cfg, kern, a, cluster), "attention_kv8");
}

template <int D>
int launch_weights_tc(cudaStream_t s, const AttnArgs& a) {
  const int64_t row_tiles = ceil_div((int64_t)a.T * (a.Hq / a.c.kv_heads), kRows);
  int cluster = 1;
  while (cluster < kWeightCluster && cluster * 2 <= row_tiles) cluster *= 2;
  const int64_t grid = ceil_div(a.c.max_seq, kKeys) * cluster * a.c.batch * a.c.kv_heads;
  if (grid > INT32_MAX) return fail(SPX_ERR_UNSUPPORTED, "attention_kv8: grid too large");
  auto kern = kv8_weights_tc_kernel<D>;
  constexpr size_t smem = WeightShape<D>::kSmem;
  int rc = check_cuda(
      cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem),
      "attention_kv8: smem attribute");
  if (rc) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(kWeightThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)cluster;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return check_cuda(cudaLaunchKernelEx(&cfg, kern, a, cluster), "attention_kv8: weights");
}

}  // namespace

int launch_weights_kv8_tc(cudaStream_t s, const AttnArgs& a) {
  return a.c.head_dim == 64 ? launch_weights_tc<64>(s, a) : launch_weights_tc<128>(s, a);
}

int launch_attention_kv8_tc(cudaStream_t s, const AttnArgs& a) {
  return a.c.head_dim == 64 ? launch_tc<64>(s, a) : launch_tc<128>(s, a);
}

namespace {
std::mutex g_slot_mu;
bool g_slot_used[kAtSlots - 1];
}  // namespace

int at_slot_get() {
  std::lock_guard<std::mutex> lock(g_slot_mu);
  for (int i = 0; i < kAtSlots - 1; ++i)
    if (!g_slot_used[i]) {
      g_slot_used[i] = true;
      return i;
    }
  return kAtSlots - 1;         // shared by all that come later
}

void at_slot_put(int slot) {
  std::lock_guard<std::mutex> lock(g_slot_mu);
  if (slot >= 0 && slot < kAtSlots - 1) g_slot_used[slot] = false;
}

int at_take_status(int slot) {
  const int from = slot < 0 ? 0 : slot, n = slot < 0 ? kAtSlots : 1;
  int v[kAtSlots] = {}, any = 0;
  if (cudaMemcpyFromSymbol(v, g_at_status, n * sizeof(int), from * sizeof(int)) != cudaSuccess) {
    cudaGetLastError();
    return 0;
  }
  for (int i = 0; i < n; ++i) {
    any |= v[i];
    v[i] = 0;
  }
  if (any) cudaMemcpyToSymbol(g_at_status, v, n * sizeof(int), from * sizeof(int));
  return any;
}

}  // namespace spx
