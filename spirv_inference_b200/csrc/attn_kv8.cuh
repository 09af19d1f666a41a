// What the kernels of attention over the 8-bit key / value cache share.
#pragma once

#include <cuda_fp16.h>

#include "spx_internal.cuh"

namespace spx {

struct AttnArgs {
  const float* q;
  spx_kv8_cache c;
  const int32_t* new_lens;
  int T, Hq;
  uint32_t g_mul;   // ceil(2^32 / heads of a group)
  float scale;
  float* out;
  float* lse;
  float* weights;
  int slot;         // of the graph's status word (many rows)
  // r / (heads of a group), exact while r times those is below 2^32
  __device__ __forceinline__ int div_g(int r) const {
    return g_mul ? (int)__umulhi((uint32_t)r, g_mul) : r;
  }
};

namespace {

__device__ __forceinline__ int clamp_len(int v, int hi) { return v < 0 ? 0 : v > hi ? hi : v; }
// len + n, at most hi, for 0 <= len <= hi and any n >= 0.
__device__ __forceinline__ int add_len(int len, int n, int hi) {
  return n > hi - len ? hi : len + n;
}

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

constexpr float kPUp = 32768.0f;   // 2^15
// v scales are taken against a reference of at least this: kPUp over it, and it
// over kPUp, are normal numbers (a smaller one's quotient would be infinite, and
// times values of zero NaN).
constexpr float kMinRef = 0x1p-111f;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t as_u32(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }

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
// (x, y) as packed fp16 hi and lo parts.
__device__ __forceinline__ void split2(float x, float y, uint32_t& hi, uint32_t& lo) {
  const __half2 h = __floats2half2_rn(x, y);
  const float2 f = __half22float2(h), d = add2(make_float2(x, y), make_float2(-f.x, -f.y));
  hi = as_u32(h);
  lo = as_u32(__floats2half2_rn(d.x, d.y));
}

// 2^-e and 2^e that take a largest magnitude with these bits (finite) to 2^14 or
// above, below 2^15, and back.  fp16 hi + lo then hold what is 2^-39 of it or more
// with the full 22 bits, and nothing to worse than 2^-39 of it (with the largest
// at 1, values 1000 times smaller kept 15 bits).  Below 2^-112 it stays smaller.
__device__ __forceinline__ void pow2_scale(uint32_t amax_bits, float& down, float& up) {
  int e = (int)(amax_bits >> 23);
  e = e < 15 ? 15 : e > 253 ? 253 : e;
  down = __uint_as_float((uint32_t)(268 - e) << 23);
  up = __uint_as_float((uint32_t)(e - 14) << 23);
}
__device__ __forceinline__ uint32_t finite_abs(float x) {
  const uint32_t b = __float_as_uint(x) & 0x7fffffffu;
  return b >= 0x7f800000u ? 0u : b;
}

// Bytes 0 and 2 of a word of two's complement bytes to fp16: with the sign bit
// flipped under 0x64, they are 1024 + 128 + value.  (mask: 0x00ff00ff in a
// register, for one instruction: a lop3 takes one constant of its own.)
__device__ __forceinline__ uint32_t even_bytes(uint32_t w, uint32_t mask) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, 0x64806480, 0x6a;" : "=r"(r) : "r"(w), "r"(mask));   // (w & mask) ^ c
  const __half2 v = __hsub2(*reinterpret_cast<__half2*>(&r),
                            __half2half2(__ushort_as_half((unsigned short)0x6480)));
  return as_u32(v);
}

}  // namespace

// Many rows (k_attn_kv8_tc.cu).
int launch_attention_kv8_tc(cudaStream_t s, const AttnArgs& a);
int launch_weights_kv8_tc(cudaStream_t s, const AttnArgs& a);

}  // namespace spx
