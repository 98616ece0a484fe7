// logprobs.cuh -- softmax statistics of a row, kept by a running maximum: shared by the operators on logits
// (logprobs.cu) and the head product that never stores them (head_logprobs.cu).
#pragma once
#include <cmath>

#include "common.cuh"

namespace zl {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kFloor = -1000.f;  // a log2 probability this low has p = 0; stands for -inf in products

inline bool bad_scale(float s) { return !(s >= 1e-4f && s <= 1e4f); }

__device__ __forceinline__ float ex2(float t) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(t));
  return r;
}

// ------------------------------------------------------------------ running softmax statistics
// c = scale * log2(e).  A masked logit (-inf) has e = 0; its exponent is kept off -inf before it is
// multiplied with e.  A NaN or +inf logit makes s0 and s1 NaN.
struct Stats {
  float m = -INFINITY, s0 = 0.f, s1 = 0.f;
  // statistics of the same elements about the larger maximum M
  __device__ __forceinline__ void rebase(float M, float c) {
    const float d = m == -INFINITY ? kFloor : fmaxf((m - M) * c, kFloor);
    const float f = ex2(d);
    s1 = f * fmaf(d, s0, s1);
    s0 *= f;
    m = M;
  }
  template <int N> __device__ __forceinline__ void add(const float (&v)[N], float c) {
    float b = v[0];
#pragma unroll
    for (int j = 1; j < N; ++j) b = fmaxf(b, v[j]);
    if (b > m) rebase(b, c);
    add_below(v, c);
  }
  // elements none of which is above m
  template <int N> __device__ __forceinline__ void add_below(const float (&v)[N], float c) {
    const float base = m == -INFINITY ? 0.f : m;
    if constexpr (N % 4 == 0) {
      // two pairs of partial sums: four chains of N / 4 additions, paired fp32 instructions
      const uint64_t nb = f2_pack(-base, -base), c2 = f2_pack(c, c);
      uint64_t a0[2] = {0, 0}, a1[2] = {0, 0};
#pragma unroll
      for (int j = 0; j < N; j += 2) {
        float t0, t1;
        f2_unpack(mul2(add2(f2_pack(v[j], v[j + 1]), nb), c2), t0, t1);
        const uint64_t e = f2_pack(ex2(t0), ex2(t1));
        a0[j / 2 & 1] = add2(a0[j / 2 & 1], e);
        a1[j / 2 & 1] = fma2(e, f2_pack(fmaxf(t0, kFloor), fmaxf(t1, kFloor)), a1[j / 2 & 1]);
      }
      float x, y;
      f2_unpack(add2(a0[0], a0[1]), x, y);
      s0 += x + y;
      f2_unpack(add2(a1[0], a1[1]), x, y);
      s1 += x + y;
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const float t = (v[j] - base) * c, e = ex2(t);
        s0 += e;
        s1 = fmaf(e, fmaxf(t, kFloor), s1);
      }
    }
  }
  __device__ __forceinline__ void join(const Stats& o, float c) {
    Stats a = o;
    const float M = fmaxf(m, o.m);
    rebase(M, c);
    a.rebase(M, c);
    s0 += a.s0;
    s1 += a.s1;
  }
  __device__ __forceinline__ void join_warp(float c) {
    float M = m;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
    rebase(M, c);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      s0 += __shfl_xor_sync(0xffffffffu, s0, o);
      s1 += __shfl_xor_sync(0xffffffffu, s1, o);
    }
  }
};
// ln p of a logit from a row's statistics; a row without a finite logit (s0 = 0) has ln p = -inf everywhere.
__device__ __forceinline__ float log_prob(float x, const Stats& s, float ln_s0, float scale) {
  return s.s0 == 0.f ? -INFINITY : fmaf(x - s.m, scale, -ln_s0);
}


}  // namespace zl
