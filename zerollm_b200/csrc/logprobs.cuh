// logprobs.cuh -- softmax statistics of a row, kept by a running maximum: shared by the operators on logits
// (logprobs.cu) and the head product that never stores them (head_logprobs.cu).
#pragma once
#include <cmath>

#include "common.cuh"

namespace zl {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kFloor = -1000.f;  // a log2 probability this low has p = 0; stands for -inf in products

inline bool bad_scale(float s) { return !(s >= 1e-4f && s <= 1e4f); }

// A kernel launched by launch_after() may start while the one before it in the stream still runs; follows() waits
// until that one is done and its results are seen.  let_follow(): this kernel's successor may start from here on.
__device__ __forceinline__ void follows() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_follow() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
// The status of a launch or of a call before it; its error is not left behind for a later call to report.
inline zl_status launched(const char* what, cudaError_t e) {
  if (e == cudaSuccess) return ZL_OK;
  cudaGetLastError();
  return set_error(ZL_ECUDA, "%s: %s", what, cudaGetErrorString(e));
}
template <typename K, typename... A>
zl_status launch_after(const char* what, K kern, int blocks, int threads, cudaStream_t st, A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(blocks, 1, 1);
  cfg.blockDim = dim3(threads, 1, 1);
  cfg.stream = st;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return launched(what, cudaLaunchKernelEx(&cfg, kern, args...));
}

__device__ __forceinline__ float ex2(float t) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(t));
  return r;
}

// ------------------------------------------------------------------ running softmax statistics
// c = scale * log2(e).  Sums of e = 2^((x - m) c) and e (x - m) c about the running maximum m.  A masked logit
// (-inf) has e = 0; it is kept off -inf before anything is multiplied with e.  A NaN or +inf logit makes s0 and
// s1 NaN.  While |m c| <= kNear the exponent is one fused product x c - fl(m c): the running sums are about fl(m c), whose
// rounding off = m c - fl(m c), at most 2^-7 there, is taken out of them when they leave the thread.  Beyond it (large
// logits, masks of finite values) the exponent is (x - m) c, of a difference that is exact where x is near m.
constexpr float kNear = 0x1p18f;  // (rows about -1e5, or masked with it, at the full rate)
// 2^-off of such a rounding, to second order (the third is below 2^-25)
__device__ __forceinline__ float take_out(float off) {
  const float x = off * kLn2;
  return fmaf(x, fmaf(x, 0.5f, -1.f), 1.f);
}
constexpr float kClamp = -0x1p96f;   // masked logits in fused products: e = 0 beside any |m c| <= kNear
constexpr uint32_t kClampBf16 = 0xef80ef80u;
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ uint32_t max2_nan(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// Maximum over a warp, NaN aside (-inf where every lane has NaN or -inf).
__device__ __forceinline__ float max_warp(float v) {
  float r;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}

// Statistics of some elements, exact about m.
struct Stats {
  float m = -INFINITY, s0 = 0.f, s1 = 0.f;
  __device__ Stats() {}
  __device__ explicit Stats(const float3& v) : m(v.x), s0(v.y), s1(v.z) {}
  __device__ float3 pack() const { return make_float3(m, s0, s1); }
  // the same about the larger maximum M
  __device__ __forceinline__ void rebase(float M, float c) {
    const float d = m == -INFINITY ? kFloor : fmaxf((m - M) * c, kFloor);
    const float f = ex2(d);
    s1 = f * fmaf(d, s0, s1);
    s0 *= f;
    m = M;
  }
  __device__ __forceinline__ void join_warp(float c) {
    rebase(max_warp(m), c);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      s0 += __shfl_xor_sync(0xffffffffu, s0, o);
      s1 += __shfl_xor_sync(0xffffffffu, s1, o);
    }
  }
};

// A thread's running statistics.
template <bool ENTROPY> struct RunningT {
  float m = -INFINITY, mc = 0.f, s0 = 0.f, s1 = 0.f;
  // whether the fused product holds about m (also before any logit, mc = 0: nothing but masks adds to the sums then)
  __device__ __forceinline__ bool near() const { return fabsf(mc) <= kNear; }
  __device__ __forceinline__ Stats sums(float c) const {
    Stats s;
    s.m = m; s.s0 = s0; s.s1 = s1;
    if (near() && m != -INFINITY) {  // m c - fl(m c), exact
      const float off = fmaf(m, c, -mc), f = take_out(off);
      s.s1 = f * fmaf(-off, s.s0, s.s1);
      s.s0 *= f;
    }
    return s;
  }
  // a maximum above m of elements to come: the sums go from fl(m c) (or m c) to fl(most c) (or most c)
  __device__ __forceinline__ void raise(float most, float c) {
    const float most_c = most * c;
    float d = (m - most) * c;
    if (near()) d -= fmaf(m, c, -mc);
    if (fabsf(most_c) <= kNear) d += fmaf(most, c, -most_c);
    d = fmaxf(d, kFloor);  // (also where m = -inf)
    const float f = ex2(d);
    s1 = f * fmaf(d, s0, s1);
    s0 *= f;
    m = most; mc = most_c;
  }
  // sums of N elements about m, none above it: pairs of partial sums (paired fp32 instructions).  NEAR: by the fused
  // product, which has to hold, and none below kClamp; otherwise by whichever holds, of any values
  template <bool NEAR, int N> __device__ __forceinline__ void fold(const float (&v)[N], float c, float& x0, float& x1) const {
    const float sub = NEAR || near() ? 0.f : -m, add = NEAR || near() ? -mc : 0.f;
    const uint64_t c2 = f2_pack(c, c), n2 = f2_pack(add, add), s2 = f2_pack(sub, sub);
    uint64_t a0[2] = {0, 0}, a1[2] = {0, 0};
#pragma unroll
    for (int j = 0; j < N; j += 2) {
      uint64_t t = f2_pack(v[j], v[j + 1]);
      if (!NEAR) t = add2(t, s2);
      t = fma2(t, c2, n2);
      float t0, t1;
      f2_unpack(t, t0, t1);
      const uint64_t e = f2_pack(ex2(t0), ex2(t1));
      if (!NEAR) t = f2_pack(fmaxf(t0, kFloor), fmaxf(t1, kFloor));
      a0[j / 2 & 1] = add2(a0[j / 2 & 1], e);
      if (ENTROPY) a1[j / 2 & 1] = fma2(e, t, a1[j / 2 & 1]);
    }
    float x, y;
    f2_unpack(add2(a0[0], a0[1]), x, y);
    x0 = x + y;
    if (ENTROPY) {
      f2_unpack(add2(a1[0], a1[1]), x, y);
      x1 = x + y;
    }
  }
  // N elements, none above m (NEAR: as for fold())
  template <bool NEAR, int N> __device__ __forceinline__ void add(const float (&v)[N], float c) {
    float x0, x1 = 0.f;
    fold<NEAR>(v, c, x0, x1);
    s0 += x0;
    s1 += x1;
  }
  // N elements, whose maximum is only looked for where their sum says that it lies well above m (by 3 at least, in powers
  // of two): m need not be the maximum for the sums to be exact, only near enough to it that neither they nor
  // ln S0 - S1 / S0 lose digits.  (x1 is NaN beside -inf, which the fused product does not take.)
  template <int N> __device__ __forceinline__ void add_near(const float (&v)[N], float c) {
    float x0 = INFINITY, x1 = 0.f;
    if (near() && m != -INFINITY) fold<true>(v, c, x0, x1);
    if (x0 <= 8.f * N && x1 == x1) {
      s0 += x0;
      s1 += x1;
    } else {
      add_any(v, c);
    }
  }
  // one element of any value
  __device__ __forceinline__ void add_one(float v, float c) {
    if (v > m) raise(v, c);
    const float t = near() ? fmaf(v, c, -mc) : (v - m) * c, e = ex2(t);
    s0 += e;
    if (ENTROPY) s1 = fmaf(e, fmaxf(t, kFloor), s1);
  }
  // N elements of any values
  template <int N> __device__ __forceinline__ void add_any(const float (&v)[N], float c) {
    float b = v[0];
#pragma unroll
    for (int j = 1; j < N; ++j) b = fmaxf(b, v[j]);
    if (b > m) raise(b, c);
    add<false>(v, c);
  }
};
using Running = RunningT<true>;
// ln p of a logit from a row's statistics; a row without a finite logit (s0 = 0) has ln p = -inf everywhere.
__device__ __forceinline__ float log_prob(float x, const Stats& s, float ln_s0, float scale) {
  return s.s0 == 0.f ? -INFINITY : fmaf(x - s.m, scale, -ln_s0);
}


}  // namespace zl
