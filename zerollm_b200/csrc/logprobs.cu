// logprobs.cu -- operators on next-token distributions: log probabilities of given tokens with entropy
// and top alternatives, their gradient, and distillation from a teacher's top logits.
//
// All work on rows of logits x (bf16 or fp32, any row stride and alignment) with y = scale * x:
//   m = max x,  S0 = sum_j e^(y_j - y_max),  S1 = sum_j e^(y_j - y_max) (y_j - y_max)
//   lse = y_max + ln S0,  ln p_t = y_t - lse,  H = ln S0 - S1 / S0
// kept in fp32 by a running maximum per thread (one pass over the row, one exponential per logit), joined
// over a block and, where there are few rows, over the cluster of blocks that shares a row.
// The reference has no counterpart: its loss takes softmax probabilities (cross_entropy.cpp:23-79).
#include <cooperative_groups.h>
#include <cfloat>
#include <cmath>
#include <cstdint>

#include "logprobs.cuh"

namespace cg = cooperative_groups;

namespace zl {
int sm_count_current();  // gemm.cu

namespace {
constexpr int kTopMax = 128;   // most alternatives of a row
constexpr int kCand = 512;     // candidates ranked at once; more (long runs of equal values) go the slow way
constexpr int kMaxParts = 8;   // blocks of a cluster that share a row

// ------------------------------------------------------------------ elements
template <typename T> struct Elt;
template <> struct Elt<float> {
  static constexpr int VEC = 4;
  static __device__ __forceinline__ float get(const float* p) { return *p; }
  static __device__ __forceinline__ void put(float* p, float v) { *p = v; }
  static __device__ __forceinline__ void unpack(const uint4& u, float (&v)[4]) {
    v[0] = __uint_as_float(u.x); v[1] = __uint_as_float(u.y); v[2] = __uint_as_float(u.z); v[3] = __uint_as_float(u.w);
  }
  static __device__ __forceinline__ uint4 pack(const float (&v)[4]) {
    return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
  }
};
template <> struct Elt<__nv_bfloat16> {
  static constexpr int VEC = 8;
  static __device__ __forceinline__ float get(const __nv_bfloat16* p) { return __bfloat162float(*p); }
  static __device__ __forceinline__ void put(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
  static __device__ __forceinline__ void unpack(const uint4& u, float (&v)[8]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ uint4 pack(const float (&v)[8]) {
    return make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
  }
};

// Plain (coherent) 16-byte load: distillation may write its gradient over the logits.
__device__ __forceinline__ uint4 load16(const void* p) {
  uint4 u;
  asm volatile("ld.global.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w) : "l"(p));
  return u;
}
// A row as elements [0, head) before its first 16-byte boundary, nv whole vectors, and the rest [tail, V).
// Block `part` of the `parts` that share the row takes the vectors [lo, hi); the first block takes the
// head and the last one the rest, one element per thread.
template <typename T> struct Span {
  int head, lo, hi, tail;
  __device__ Span(const T* x, int V, int part, int parts) {
    constexpr int VEC = Elt<T>::VEC;
    const int mis = (int)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
    head = mis ? min(VEC - mis, V) : 0;
    const int nv = (V - head) / VEC;
    lo = (int)((int64_t)nv * part / parts);
    hi = (int)((int64_t)nv * (part + 1) / parts);
    tail = head + nv * VEC;
  }
  // the element outside whole vectors that this thread has, or -1
  __device__ int single(int V, int part, int parts) const {
    const int t = threadIdx.x;
    if (part == 0 && t < head) return t;
    if (part == parts - 1 && t >= 8 && t < 16 && tail + t - 8 < V) return tail + t - 8;
    return -1;
  }
  // whether block `part` has element i
  __device__ bool has(int i, int part, int parts) const {
    constexpr int VEC = Elt<T>::VEC;
    if (i < head) return part == 0;
    if (i >= tail) return part == parts - 1;
    const int v = (i - head) / VEC;
    return v >= lo && v < hi;
  }
};

// Statistics of this block's part of a row, the same in every thread (two block barriers).
template <typename T, int NT>
__device__ __forceinline__ Stats block_stats(const T* x, const Span<T>& sp, int single, float c, float& thread_max,
                                             Stats* red) {
  constexpr int VEC = Elt<T>::VEC, U = 4;
  Stats s;
  for (int v = sp.lo + (int)threadIdx.x; v < sp.hi; v += NT * U) {
    uint4 u[U];
#pragma unroll
    for (int i = 0; i < U; ++i)
      if (v + i * NT < sp.hi) u[i] = load16(x + sp.head + (int64_t)(v + i * NT) * VEC);
#pragma unroll
    for (int i = 0; i < U; ++i)
      if (v + i * NT < sp.hi) {
        float f[VEC];
        Elt<T>::unpack(u[i], f);
        s.add(f, c);
      }
  }
  if (single >= 0) {
    const float f[1] = {Elt<T>::get(x + single)};
    s.add(f, c);
  }
  thread_max = s.m;
  s.join_warp(c);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = s;
  __syncthreads();
  s = red[0];
#pragma unroll
  for (int w = 1; w < NT / 32; ++w) s.join(red[w], c);
  __syncthreads();
  return s;
}

// ------------------------------------------------------------------ top alternatives
// Order-preserving key: larger values have larger keys, -0 and +0 the same one, NaN the lowest (0).
__device__ __forceinline__ uint32_t order_key(float x) {
  if (x != x) return 0u;
  const uint32_t b = __float_as_uint(x + 0.f);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
constexpr uint32_t kKeyMasked = 0x007fffffu;  // of -inf
__device__ __forceinline__ float key_value(uint32_t k) {
  return k == 0u ? __uint_as_float(0x7fffffffu) : __uint_as_float((k & 0x80000000u) ? (k ^ 0x80000000u) : ~k);
}
// A candidate: larger key first, then the lower index.
__device__ __forceinline__ unsigned long long candidate(uint32_t key, int i) {
  return ((unsigned long long)key << 32) | (0xffffffffu - (uint32_t)i);
}

struct TopShared {
  unsigned long long cand[kCand];
  uint32_t group[256];
  int col[256];
  int n, ncol;
  uint32_t tau;
};

// Count of the row's elements with key >= k, the same in every thread (one block, the whole row).
template <typename T, int NT>
__device__ int count_from(const T* x, int V, uint32_t k, int* slots) {
  int n = 0;
  for (int i = threadIdx.x; i < V; i += NT) n += order_key(Elt<T>::get(x + i)) >= k;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) slots[threadIdx.x >> 5] = n;
  __syncthreads();
  n = 0;
#pragma unroll
  for (int w = 0; w < NT / 32; ++w) n += slots[w];
  return n;
}

// The candidates of a row in which more than kCand elements are at least tau (long runs of equal values:
// masked vocabularies, constant rows): the exact key K of the k-th largest element, every element above it
// (fewer than k) and the lowest-indexed ones equal to it.
template <typename T, int NT>
__device__ void select_slow(const T* x, int V, int k, uint32_t tau, TopShared& sh, int* slots) {
  if (tau == 0 && count_from<T, NT>(x, V, kKeyMasked, slots) >= k) tau = kKeyMasked;
  uint32_t K = tau;
  if (tau != 0xffffffffu && count_from<T, NT>(x, V, tau + 1, slots) >= k) {
    K = 0;
    for (int b = 31; b >= 0; --b) {
      const uint32_t t = K | (1u << b);
      if (count_from<T, NT>(x, V, t, slots) >= k) K = t;
    }
  }
  __syncthreads();
  if (threadIdx.x == 0) sh.n = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < V; i += NT) {
    const uint32_t q = order_key(Elt<T>::get(x + i));
    if (q > K) sh.cand[atomicAdd(&sh.n, 1)] = candidate(q, i);
  }
  __syncthreads();
  int n = sh.n;  // < k <= kTopMax
  // equal ones in index order, NT elements at a time
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  for (int i0 = 0; i0 < V && n < k; i0 += NT) {
    const int i = i0 + threadIdx.x;
    const bool eq = i < V && order_key(Elt<T>::get(x + i)) == K;
    const uint32_t vote = __ballot_sync(0xffffffffu, eq);
    __syncthreads();
    if (lane == 0) slots[w] = __popc(vote);
    __syncthreads();
    int at = n, all = 0;
#pragma unroll
    for (int j = 0; j < NT / 32; ++j) {
      if (j < w) at += slots[j];
      all += slots[j];
    }
    at += __popc(vote & ((1u << lane) - 1u));
    if (eq && at < k) sh.cand[at] = candidate(K, i);
    n = min(k, n + all);
  }
  __syncthreads();
  if (threadIdx.x == 0) sh.n = n;
  __syncthreads();
}

struct LogprobArgs {
  const void* logits;
  int64_t stride;
  const int32_t* targets;
  int rows, vocab, k, groups, parts;
  float scale;
  float *logp, *entropy, *lse, *top_logp;
  int32_t* top_ids;
};

// One row per block, or per cluster of `parts` blocks.  Top alternatives: the k-th largest of the maxima of
// `groups` disjoint sets of elements (a thread's elements, or those of some neighbouring threads) is a bound
// tau that at least k elements reach; only threads whose own maximum reaches it have candidates, and a warp
// reads such a thread's elements again (from L2).  For values in any order about k * 1.15 elements reach tau.
template <typename T, int NT>
__global__ void __launch_bounds__(NT) logprobs_kernel(const LogprobArgs a) {
  constexpr int VEC = Elt<T>::VEC, NW = NT / 32;
  __shared__ Stats red[NW];
  __shared__ Stats parts_st[kMaxParts];
  __shared__ int slots[NW];
  __shared__ TopShared sh;
  const int parts = a.parts, part = parts > 1 ? (int)(blockIdx.x % parts) : 0;
  const int64_t r = blockIdx.x / parts;
  const int V = a.vocab, tid = threadIdx.x, lane = tid & 31;
  const T* x = static_cast<const T*>(a.logits) + r * a.stride;
  const float c = a.scale * kLog2e;
  const Span<T> sp(x, V, part, parts);
  const int single = sp.single(V, part, parts);
  if (tid == 0) { sh.n = 0; sh.ncol = 0; }
  if (parts > 1) cg::this_cluster().barrier_arrive();
  float tmax;
  Stats s = block_stats<T, NT>(x, sp, single, c, tmax, red);
  // a maximum of -inf may stand for -inf, for NaN or for no element at all: below every bound
  const uint32_t tkey = tmax == -INFINITY ? 0u : order_key(tmax);
  if (parts > 1) cg::this_cluster().barrier_wait();  // every block of the cluster runs: its shared memory may be written
  if (a.k > 0) {
    // NT * parts / groups threads to a group (a power of two, at most 32)
    const int per = NT * parts / a.groups;
    uint32_t g = tkey;
    for (int o = per >> 1; o > 0; o >>= 1) g = max(g, __shfl_xor_sync(0xffffffffu, g, o));
    if ((tid & (per - 1)) == 0) {
      const int at = part * (a.groups / parts) + tid / per;
      if (parts == 1) sh.group[at] = g;
      else
        for (int q = 0; q < parts; ++q) *cg::this_cluster().map_shared_rank(&sh.group[at], q) = g;
    }
  }
  if (parts > 1) {
    if (tid < parts) *cg::this_cluster().map_shared_rank(&parts_st[part], tid) = s;
    cg::this_cluster().sync();
    s = parts_st[0];
    for (int q = 1; q < parts; ++q) s.join(parts_st[q], c);
  } else {
    __syncthreads();
  }
  const float ln_s0 = logf(s.s0);
  if (part == 0 && tid == 0) {
    const int t = a.targets ? a.targets[r] : -1;
    const float h = fmaf(-kLn2, s.s1 / s.s0, ln_s0);
    if (a.lse) a.lse[r] = s.s0 == 0.f ? -INFINITY : fmaf(s.m, a.scale, ln_s0);
    if (a.entropy) a.entropy[r] = (s.s0 == 0.f || h < 0.f) ? 0.f : h;
    if (a.logp) a.logp[r] = (t >= 0 && t < V) ? log_prob(Elt<T>::get(x + t), s, ln_s0, a.scale) : 0.f;
  }
  if (a.k == 0) return;

  // tau: the k-th largest group maximum, bit by bit over one warp's ballots
  if (tid < 32) {
    uint32_t g[8], tau = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) g[i] = i * 32 + lane < a.groups ? sh.group[i * 32 + lane] : 0u;
    for (int b = 31; b >= 0; --b) {
      const uint32_t t = tau | (1u << b);
      int n = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i * 32 < a.groups) n += __popc(__ballot_sync(0xffffffffu, g[i] >= t));
      if (n >= a.k) tau = t;
    }
    if (lane == 0) sh.tau = tau;
  }
  __syncthreads();
  const uint32_t tau = sh.tau;
  if (tkey >= tau) sh.col[atomicAdd(&sh.ncol, 1)] = tid;
  TopShared& first = parts > 1 ? *cg::this_cluster().map_shared_rank(&sh, 0) : sh;
  auto offer = [&](float f, int i) {
    const uint32_t q = order_key(f);
    if (q >= tau) {
      const int n = atomicAdd(&first.n, 1);
      if (n < kCand) first.cand[n] = candidate(q, i);
    }
  };
  if (single >= 0) offer(Elt<T>::get(x + single), single);
  __syncthreads();
  const int ncol = sh.ncol;
  for (int i = tid >> 5; i < ncol; i += NW) {
    for (int v = sp.lo + sh.col[i] + lane * NT; v < sp.hi; v += 32 * NT) {
      float f[VEC];
      Elt<T>::unpack(load16(x + sp.head + (int64_t)v * VEC), f);
#pragma unroll
      for (int j = 0; j < VEC; ++j) offer(f[j], sp.head + v * VEC + j);
    }
  }
  if (parts > 1) cg::this_cluster().sync();
  else __syncthreads();
  if (part != 0) return;
  if (sh.n > kCand) select_slow<T, NT>(x, V, a.k, tau, sh, slots);
  const int n = sh.n;
  for (int i = tid; i < n; i += NT) {
    const unsigned long long me = sh.cand[i];
    int rank = 0;
    for (int j = 0; j < n; ++j) rank += sh.cand[j] > me;
    if (rank < a.k) {
      const int64_t o = r * a.k + rank;
      if (a.top_logp) a.top_logp[o] = log_prob(key_value((uint32_t)(me >> 32)), s, ln_s0, a.scale);
      a.top_ids[o] = (int32_t)(0xffffffffu - (uint32_t)me);
    }
  }
}

// ------------------------------------------------------------------ gradient of the log probabilities
struct LogprobBwdArgs {
  const void* logits;
  int64_t stride;
  const int32_t* targets;
  const float *lse, *entropy, *g_logp, *g_entropy;
  int rows, vocab;
  float scale;
  void* d;
  int64_t d_stride;
};

// d_j = scale [ g (1[j = t] - p_j) - h p_j (ln p_j + H) ], element by element from the row's saved statistics.
// One block per (row, slice of the vocabulary); elements one at a time where logits and gradient rows do not
// share their place within 16 bytes.
template <typename T, int NT>
__global__ void __launch_bounds__(NT) logprobs_bwd_kernel(const LogprobBwdArgs a, int slices) {
  constexpr int VEC = Elt<T>::VEC;
  const int64_t r = blockIdx.x / slices;
  const int part = (int)(blockIdx.x % slices);
  const int V = a.vocab, tid = threadIdx.x;
  const T* x = static_cast<const T*>(a.logits) + r * a.stride;
  T* d = static_cast<T*>(a.d) + r * a.d_stride;
  const float lse = a.lse[r];
  // a row masked wholly has no gradient: with -inf, or with the type's lowest value, beside which its saved
  // lse cannot hold the ln V that its p would need
  const bool none = lse < -1e30f;
  int t = (a.g_logp && a.targets) ? a.targets[r] : -1;
  if (t >= V) t = -1;
  const float g = t >= 0 ? a.g_logp[r] : 0.f;
  const float h = a.g_entropy ? a.g_entropy[r] : 0.f, H = a.g_entropy ? a.entropy[r] : 0.f;
  const float scale = a.scale;
  auto grad = [&](float f, int i) {
    if (none) return 0.f;
    const float l = fmaf(f, scale, -lse), p = ex2(l * kLog2e);
    // -p (g + h (ln p + H)), ln p kept off -inf where p = 0
    float v = -p * fmaf(h, fmaxf(l, kFloor) + H, g);
    if (i == t) v += g;
    return v * scale;
  };
  if (((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(d)) & 15) == 0) {
    const Span<T> sp(x, V, part, slices);
    const int single = sp.single(V, part, slices);
    for (int v = sp.lo + tid; v < sp.hi; v += NT) {
      float f[VEC];
      const int i0 = sp.head + v * VEC;
      Elt<T>::unpack(load16(x + i0), f);
#pragma unroll
      for (int j = 0; j < VEC; ++j) f[j] = grad(f[j], i0 + j);
      *reinterpret_cast<uint4*>(d + i0) = Elt<T>::pack(f);
    }
    if (single >= 0) Elt<T>::put(d + single, grad(Elt<T>::get(x + single), single));
  } else {
    const int lo = (int)((int64_t)V * part / slices), hi = (int)((int64_t)V * (part + 1) / slices);
    for (int i = lo + tid; i < hi; i += NT) Elt<T>::put(d + i, grad(Elt<T>::get(x + i), i));
  }
}

// ------------------------------------------------------------------ distillation
struct DistillArgs {
  const void* logits;
  int64_t stride;
  const int32_t* ids;
  const float* values;
  const int32_t* targets;
  const float* row_weight;
  int rows, vocab, k, parts;
  zl_distill_options opt;
  void* d;
  int64_t d_stride;
  float* loss_rows;
};

__device__ __forceinline__ float block_sum(float v, float* slots, int warps) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) slots[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0.f;
  for (int w = 0; w < warps; ++w) v += slots[w];
  return v;
}

// Loss and gradient of one row per block (or cluster): the statistics of s x (and of x, for the hard target,
// where s != 1) in one pass, then the dense part p of the gradient in a second one over the row (from L2),
// then the at most k + 1 elements that also have a teacher's or target's share.  The logits are read before
// any of this row's gradient is written, so the gradient may take their place.
template <typename T, int NT>
__global__ void __launch_bounds__(NT) distill_kernel(const DistillArgs a) {
  constexpr int VEC = Elt<T>::VEC, NW = NT / 32;
  __shared__ Stats red[NW];
  __shared__ Stats parts_st[kMaxParts], parts_st1[kMaxParts];
  __shared__ float slots[NW];
  __shared__ int s_id[kTopMax + 1];
  __shared__ float s_q[kTopMax + 1];
  __shared__ float s_sum[2];  // sum q, sum q ln q
  __shared__ float part_loss[kMaxParts];
  const int parts = a.parts, part = parts > 1 ? (int)(blockIdx.x % parts) : 0;
  const int64_t r = blockIdx.x / parts;
  const int V = a.vocab, tid = threadIdx.x, lane = tid & 31, k = a.k;
  const T* x = static_cast<const T*>(a.logits) + r * a.stride;
  T* d = a.d ? static_cast<T*>(a.d) + r * a.d_stride : nullptr;
  const float w = a.row_weight ? a.row_weight[r] : 1.f;
  const bool same = d && ((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(d)) & 15) == 0;
  const Span<T> sp(x, V, part, parts);
  const int single = sp.single(V, part, parts);
  // d[i] = f(x[i], i) over this block's part of the row
  auto fill = [&](auto f) {
    for (int v = sp.lo + tid; v < sp.hi; v += NT) {
      float e[VEC];
      const int i0 = sp.head + v * VEC;
      Elt<T>::unpack(load16(x + i0), e);
#pragma unroll
      for (int j = 0; j < VEC; ++j) e[j] = f(e[j]);
      if (same) {
        *reinterpret_cast<uint4*>(d + i0) = Elt<T>::pack(e);
      } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j) Elt<T>::put(d + i0 + j, e[j]);
      }
    }
    if (single >= 0) Elt<T>::put(d + single, f(Elt<T>::get(x + single)));
  };
  if (w == 0.f) {  // a row without weight has no part in the loss, whatever its logits hold
    if (d) fill([](float) { return 0.f; });
    if (part == 0 && tid == 0) a.loss_rows[r] = 0.f;
    return;
  }
  const float s = a.opt.scale, c = s * kLog2e, kd = a.opt.distill_weight;
  int t = a.targets ? a.targets[r] : -1;
  if (t >= V || a.opt.target_weight == 0.f) t = -1;
  const float ce = t >= 0 ? a.opt.target_weight : 0.f;
  const bool hard = t >= 0 && s != 1.f;  // needs the statistics at scale 1 too

  // the teacher's distribution, four alternatives to a lane
  if (tid < 32) {
    float y[kTopMax / 32], mx = -INFINITY;
    int id[kTopMax / 32];
#pragma unroll
    for (int i = 0; i < kTopMax / 32; ++i) {
      const int j = i * 32 + lane;
      id[i] = j < k ? a.ids[r * k + j] : -1;
      if (id[i] >= V) id[i] = -1;
      y[i] = id[i] >= 0 ? a.values[r * k + j] * a.opt.teacher_scale : -INFINITY;
      if (id[i] < 0) id[i] = -1;
      mx = fmaxf(mx, y[i]);
    }
    float ln_n = 0.f;
    if (a.opt.normalize) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
      if (mx == -INFINITY) mx = 0.f;
      float n = 0.f;
#pragma unroll
      for (int i = 0; i < kTopMax / 32; ++i) n += expf(y[i] - mx);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
      ln_n = n == 0.f ? 0.f : mx + logf(n);
    }
    float sum = 0.f, ent = 0.f;
#pragma unroll
    for (int i = 0; i < kTopMax / 32; ++i) {
      const int j = i * 32 + lane;
      const float lq = y[i] - ln_n, q = id[i] >= 0 ? expf(lq) : 0.f;
      sum += q;
      ent += q == 0.f ? 0.f : q * lq;
      s_id[j] = id[i];
      s_q[j] = q;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      sum += __shfl_xor_sync(0xffffffffu, sum, o);
      ent += __shfl_xor_sync(0xffffffffu, ent, o);
    }
    if (lane == 0) {
      s_sum[0] = sum; s_sum[1] = ent;
      s_id[kTopMax] = t; s_q[kTopMax] = 0.f;
    }
  }
  if (parts > 1) cg::this_cluster().barrier_arrive();
  float tmax;
  Stats st = block_stats<T, NT>(x, sp, single, c, tmax, red), st1 = st;
  if (hard) st1 = block_stats<T, NT>(x, sp, single, kLog2e, tmax, red);
  if (parts > 1) {
    cg::this_cluster().barrier_wait();  // every block of the cluster runs: its shared memory may be written
    if (tid < parts) {
      *cg::this_cluster().map_shared_rank(&parts_st[part], tid) = st;
      *cg::this_cluster().map_shared_rank(&parts_st1[part], tid) = st1;
    }
    cg::this_cluster().sync();
    st = parts_st[0];
    st1 = parts_st1[0];
    for (int q = 1; q < parts; ++q) { st.join(parts_st[q], c); if (hard) st1.join(parts_st1[q], kLog2e); }
    if (!hard) st1 = st;
  }
  const bool none = st.s0 == 0.f;  // nothing left of the student's row: no loss, no gradient
  const float ln_s0 = logf(st.s0), ln_s1 = hard ? logf(st1.s0) : ln_s0;
  // this thread's alternative (or the hard target), where it lies in this block's part of the row
  float ej = 0.f, xj = 0.f;
  const int idx = tid <= kTopMax ? s_id[tid] : -1;
  static_assert(NT > kTopMax, "a thread for each alternative and the target");
  const bool mine = idx >= 0 && sp.has(idx, part, parts);
  if (mine) {
    xj = Elt<T>::get(x + idx);
    const float q = s_q[tid];
    if (tid < kTopMax && q != 0.f && kd != 0.f) ej = -kd * q * log_prob(xj, st, ln_s0, s);
    if (tid == kTopMax) ej = -ce * log_prob(xj, st1, ln_s1, hard ? 1.f : s);
  }
  const float loss = block_sum(ej, slots, NW);
  if (parts > 1 && tid == 0) *cg::this_cluster().map_shared_rank(&part_loss[part], 0) = loss;

  if (d) {
    const float gs = a.opt.grad_scale * w;
    const float wp = gs * kd * s * s_sum[0], wq = gs * kd * s, wc = gs * ce;
    const float is0 = 1.f / st.s0, is1 = 1.f / st1.s0;
    const float m = st.m;
    auto dense = [&](float f) {
      if (none) return 0.f;
      const float p = ex2((f - m) * c) * is0;
      const float p1 = hard ? ex2((f - m) * kLog2e) * is1 : p;
      return fmaf(wp, p, wc * p1);
    };
    fill(dense);
    __syncthreads();  // the elements below are written a second time, by other threads
    if (mine && !none) {
      float q = 0.f;
      for (int j = 0; j < k; ++j) q += s_id[j] == idx ? s_q[j] : 0.f;
      Elt<T>::put(d + idx, dense(xj) - wq * q - (idx == t ? wc : 0.f));
    }
  }
  float all = loss;
  if (parts > 1) {
    cg::this_cluster().sync();
    all = 0.f;
    for (int q = 0; q < parts; ++q) all += part_loss[q];
  }
  if (part == 0 && tid == 0) a.loss_rows[r] = none ? 0.f : w * fmaf(kd, s_sum[1], all);
}

// *out = scale * sum(v), summed in 64 bits in a fixed order (one block).
__global__ void __launch_bounds__(1024) scaled_sum_kernel(const float* __restrict__ v, int n, float scale,
                                                          float* __restrict__ out) {
  __shared__ double red[32];
  double s = 0.0;
  for (int i = threadIdx.x; i < n; i += 1024) s += v[i];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = s;
  __syncthreads();
  if (threadIdx.x < 32) {
    s = red[threadIdx.x];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (threadIdx.x == 0) *out = (float)(s * scale);
  }
}

// ------------------------------------------------------------------ host side
// Blocks that share a row: more while the rows alone leave SMs idle and each block keeps at least 2048 logits.
int row_parts(int rows, int vocab) {
  int p = 1;
  while (p < kMaxParts && (int64_t)rows * p < 2 * sm_count_current() && vocab / (2 * p) >= 2048) p *= 2;
  return p;
}

template <typename K, typename... A>
zl_status launch_parts(const char* what, K kern, int64_t blocks, int threads, int parts, zl_stream s, A... args) {
  if (blocks > 0x7fffffff) return set_error(ZL_EUNSUPPORTED, "%s: too many rows", what);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)blocks, 1, 1);
  cfg.blockDim = dim3(threads, 1, 1);
  cfg.stream = (cudaStream_t)s;
  cudaLaunchAttribute attr[1];
  if (parts > 1) {
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = parts;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
  }
  cudaError_t e = cudaLaunchKernelEx(&cfg, kern, args...);
  if (e != cudaSuccess) return set_error(ZL_ECUDA, "%s: %s", what, cudaGetErrorString(e));
  return ZL_OK;
}

template <typename T> bool off_element(const void* p) { return (reinterpret_cast<uintptr_t>(p) % sizeof(T)) != 0; }

template <typename T>
zl_status check_rows(const char* what, const void* logits, int64_t stride, int rows, int vocab, float scale) {
  if (rows < 0 || vocab <= 0) return set_error(ZL_EINVAL, "%s: sizes must be positive", what);
  if (stride < vocab) return set_error(ZL_EINVAL, "%s: the row stride is below the vocabulary size", what);
  if (bad_scale(scale)) return set_error(ZL_EINVAL, "%s: scale must be in [1e-4, 1e4]", what);
  if (rows > 0 && !logits) return set_error(ZL_EINVAL, "%s: null logits", what);
  if (off_element<T>(logits)) return set_error(ZL_EINVAL, "%s: logits off an element boundary", what);
  return ZL_OK;
}

template <typename T>
zl_status token_logprobs(const T* logits, int64_t stride, const int32_t* targets, int rows, int vocab, float scale,
                         int top_k, float* logp, float* entropy, float* lse, float* top_logp, int32_t* top_ids,
                         zl_stream s) {
  zl_status st = check_rows<T>("token_logprobs", logits, stride, rows, vocab, scale);
  if (st != ZL_OK) return st;
  if (logp && !targets) return set_error(ZL_EINVAL, "token_logprobs: log probabilities need targets");
  if (top_k < 0 || top_k > vocab) return set_error(ZL_EINVAL, "token_logprobs: top_k must be in [0, vocab]");
  if (top_k > kTopMax) return set_error(ZL_EUNSUPPORTED, "token_logprobs: top_k is at most %d", kTopMax);
  if (top_k > 0 && !top_ids) return set_error(ZL_EINVAL, "token_logprobs: null top_ids");
  if (rows == 0) return ZL_OK;
  constexpr int NT = 256;
  LogprobArgs a{logits, stride, targets, rows, vocab, top_k, 0, row_parts(rows, vocab), scale,
                logp, entropy, lse, top_logp, top_ids};
  a.groups = NT;
  return launch_parts("token_logprobs", logprobs_kernel<T, NT>, (int64_t)rows * a.parts, NT, a.parts, s, a);
}

template <typename T>
zl_status token_logprobs_backward(const T* logits, int64_t stride, const int32_t* targets, const float* lse,
                                  const float* entropy, const float* g_logp, const float* g_entropy, int rows, int vocab,
                                  float scale, T* d, int64_t d_stride, zl_stream s) {
  const char* what = "token_logprobs_backward";
  zl_status st = check_rows<T>(what, logits, stride, rows, vocab, scale);
  if (st != ZL_OK) return st;
  if (d_stride < vocab) return set_error(ZL_EINVAL, "%s: the gradient's row stride is below the vocabulary size", what);
  if (rows == 0) return ZL_OK;
  if (!d || !lse) return set_error(ZL_EINVAL, "%s: null gradient or lse", what);
  if (off_element<T>(d)) return set_error(ZL_EINVAL, "%s: gradient off an element boundary", what);
  if (g_logp && !targets) return set_error(ZL_EINVAL, "%s: a gradient of log probabilities needs targets", what);
  if (g_entropy && !entropy) return set_error(ZL_EINVAL, "%s: a gradient of entropies needs the entropies", what);
  if ((const void*)d == (const void*)logits && d_stride != stride)
    return set_error(ZL_EINVAL, "%s: a gradient in the logits' place has their row stride", what);
  constexpr int NT = 256;
  const int per = NT * Elt<T>::VEC * 4;
  const int slices = (vocab + per - 1) / per;
  LogprobBwdArgs a{logits, stride, targets, lse, entropy, g_logp, g_entropy, rows, vocab, scale, d, d_stride};
  return launch_parts(what, logprobs_bwd_kernel<T, NT>, (int64_t)rows * slices, NT, 1, s, a, slices);
}

template <typename T>
zl_status distill_topk(const T* logits, int64_t stride, const int32_t* ids, const float* values, int k,
                       const int32_t* targets, const float* row_weight, const zl_distill_options* opt, int rows,
                       int vocab, T* d, int64_t d_stride, float* loss_rows, float* loss_out, zl_stream s) {
  const char* what = "distill_topk";
  if (!opt) return set_error(ZL_EINVAL, "%s: null options", what);
  zl_status st = check_rows<T>(what, logits, stride, rows, vocab, opt->scale);
  if (st != ZL_OK) return st;
  if (bad_scale(opt->teacher_scale)) return set_error(ZL_EINVAL, "%s: teacher_scale must be in [1e-4, 1e4]", what);
  if (!std::isfinite(opt->distill_weight) || !std::isfinite(opt->target_weight) || !std::isfinite(opt->grad_scale))
    return set_error(ZL_EINVAL, "%s: weights must be finite", what);
  if (k < 0) return set_error(ZL_EINVAL, "%s: top_k must not be negative", what);
  if (k > kTopMax) return set_error(ZL_EUNSUPPORTED, "%s: top_k is at most %d", what, kTopMax);
  if (rows > 0 && k > 0 && (!ids || !values)) return set_error(ZL_EINVAL, "%s: null teacher_ids or teacher_logits", what);
  if (opt->target_weight != 0.f && !targets) return set_error(ZL_EINVAL, "%s: a target weight needs targets", what);
  if (d && d_stride < vocab) return set_error(ZL_EINVAL, "%s: the gradient's row stride is below the vocabulary size", what);
  if (off_element<T>(d)) return set_error(ZL_EINVAL, "%s: gradient off an element boundary", what);
  if (d && (const void*)d == (const void*)logits && d_stride != stride)
    return set_error(ZL_EINVAL, "%s: a gradient in the logits' place has their row stride", what);
  if (rows > 0 && !loss_rows) return set_error(ZL_EINVAL, "%s: null loss_rows", what);
  if (rows > 0) {
    constexpr int NT = 256;
    DistillArgs a{logits, stride, ids, values, targets, row_weight, rows, vocab, k, row_parts(rows, vocab), *opt, d,
                  d_stride, loss_rows};
    st = launch_parts(what, distill_kernel<T, NT>, (int64_t)rows * a.parts, NT, a.parts, s, a);
    if (st != ZL_OK) return st;
  }
  if (!loss_out) return ZL_OK;
  scaled_sum_kernel<<<1, 1024, 0, (cudaStream_t)s>>>(loss_rows, rows, opt->grad_scale, loss_out);
  return check_launch("distill_topk loss");
}
const __nv_bfloat16* B(const zl_bf16* p) { return reinterpret_cast<const __nv_bfloat16*>(p); }
__nv_bfloat16* B(zl_bf16* p) { return reinterpret_cast<__nv_bfloat16*>(p); }
}  // namespace
}  // namespace zl

// ============================================================== C ABI
using namespace zl;

extern "C" zl_status zl_token_logprobs_bf16(const zl_bf16* logits, int64_t row_stride, const int32_t* targets, int rows,
                                            int vocab, float scale, int top_k, float* logp, float* entropy, float* lse,
                                            float* top_logp, int32_t* top_ids, zl_stream s) {
  return token_logprobs(B(logits), row_stride, targets, rows, vocab, scale, top_k, logp, entropy, lse, top_logp, top_ids, s);
}
extern "C" zl_status zl_token_logprobs_f32(const float* logits, int64_t row_stride, const int32_t* targets, int rows,
                                           int vocab, float scale, int top_k, float* logp, float* entropy, float* lse,
                                           float* top_logp, int32_t* top_ids, zl_stream s) {
  return token_logprobs(logits, row_stride, targets, rows, vocab, scale, top_k, logp, entropy, lse, top_logp, top_ids, s);
}
extern "C" zl_status zl_token_logprobs_backward_bf16(const zl_bf16* logits, int64_t row_stride, const int32_t* targets,
                                                     const float* lse, const float* entropy, const float* g_logp,
                                                     const float* g_entropy, int rows, int vocab, float scale,
                                                     zl_bf16* d_logits, int64_t d_row_stride, zl_stream s) {
  return token_logprobs_backward(B(logits), row_stride, targets, lse, entropy, g_logp, g_entropy, rows, vocab, scale,
                                 B(d_logits), d_row_stride, s);
}
extern "C" zl_status zl_token_logprobs_backward_f32(const float* logits, int64_t row_stride, const int32_t* targets,
                                                    const float* lse, const float* entropy, const float* g_logp,
                                                    const float* g_entropy, int rows, int vocab, float scale,
                                                    float* d_logits, int64_t d_row_stride, zl_stream s) {
  return token_logprobs_backward(logits, row_stride, targets, lse, entropy, g_logp, g_entropy, rows, vocab, scale,
                                 d_logits, d_row_stride, s);
}
extern "C" zl_status zl_distill_topk_bf16(const zl_bf16* logits, int64_t row_stride, const int32_t* teacher_ids,
                                          const float* teacher_logits, int top_k, const int32_t* targets,
                                          const float* row_weight, const zl_distill_options* opt, int rows, int vocab,
                                          zl_bf16* d_logits, int64_t d_row_stride, float* loss_rows, float* loss_out,
                                          zl_stream s) {
  return distill_topk(B(logits), row_stride, teacher_ids, teacher_logits, top_k, targets, row_weight, opt, rows, vocab,
                      B(d_logits), d_row_stride, loss_rows, loss_out, s);
}
extern "C" zl_status zl_distill_topk_f32(const float* logits, int64_t row_stride, const int32_t* teacher_ids,
                                         const float* teacher_logits, int top_k, const int32_t* targets,
                                         const float* row_weight, const zl_distill_options* opt, int rows, int vocab,
                                         float* d_logits, int64_t d_row_stride, float* loss_rows, float* loss_out,
                                         zl_stream s) {
  return distill_topk(logits, row_stride, teacher_ids, teacher_logits, top_k, targets, row_weight, opt, rows, vocab,
                      d_logits, d_row_stride, loss_rows, loss_out, s);
}
