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
#include <algorithm>
#include <atomic>
#include <cfloat>
#include <cmath>
#include <cstdint>
#include <initializer_list>
#include <type_traits>

#include "logprobs.cuh"

namespace cg = cooperative_groups;

namespace zl {
int sm_count_current();  // gemm.cu

namespace {
constexpr int kTopMax = 128;   // most alternatives of a row
constexpr int kMaxParts = 8;   // blocks of a cluster that share a row

// ------------------------------------------------------------------ elements
template <typename T> struct Elt;
template <> struct Elt<float> {
  static constexpr int VEC = 4;
  static constexpr float MAX = FLT_MAX;
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
  static constexpr float MAX = 0x1.fep127f;
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
// Block `part` of the `parts` (a power of two) that share the row takes the vectors [lo, hi); the first block takes the
// head and the last one the rest, one element per thread.
template <typename T> struct Span {
  int head, lo, hi, tail;
  __device__ Span(const T* x, int V, int part, int parts) {
    constexpr int VEC = Elt<T>::VEC;
    const int mis = (int)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
    head = mis ? min(VEC - mis, V) : 0;
    const int nv = (V - head) / VEC;
    lo = 0;
    hi = nv;
    if (parts > 1) {
      const int sh = __ffs(parts) - 1;
      lo = (int)(((int64_t)nv * part) >> sh);
      hi = (int)(((int64_t)nv * (part + 1)) >> sh);
    }
    tail = head + nv * VEC;
  }
  // the element outside whole vectors that thread t has, or -1
  __device__ int single(int V, int part, int parts, int t) const {
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

// ------------------------------------------------------------------ rows through shared memory
// A row's vectors are cut into pieces of 128 (four to a lane).  A warp takes every NW-th piece and has up to
// kDepth of them on the way from device memory (cp.async.bulk into its own ring), so that loads run on while
// it computes, and into its next row.
constexpr int kLaneVecs = 4, kPieceVecs = 32 * kLaneVecs, kPieceBytes = kPieceVecs * 16, kDepth = 2;
constexpr int kRowBlocks = 6;  // blocks of four single-warp teams on an SM

// The source of a warp's pieces: rows r, r + step, ... of the matrix, of each the pieces first, first + NW, ...
// of the part [lo, hi) of its vectors.
template <typename T, int NW> struct Feed {
  const T* base;
  int64_t stride;
  int rows, V, part, parts, first, row_step;
  int64_t row;
  const uint8_t* src;
  int left;  // vectors from src to the end of the part
  bool twice, again;  // every row comes twice; this is the second time
  uint32_t issued;
  uint8_t* buf;
  uint64_t* bar;
  __device__ void open() {
    for (left = 0; row < rows; row += row_step) {
      const T* x = base + row * stride;
      const Span<T> sp(x, V, NW == 1 ? 0 : part, NW == 1 ? 1 : parts);
      left = sp.hi - sp.lo - first * kPieceVecs;
      src = reinterpret_cast<const uint8_t*>(x + sp.head) + (int64_t)(sp.lo + first * kPieceVecs) * 16;
      if (left > 0) return;
    }
    left = 0;
  }
  // the next piece on its way (one lane copies); nothing once the rows are through
  __device__ __forceinline__ void issue(int lane) {
    if (left <= 0) return;
    const uint32_t s = issued % kDepth;
    const uint32_t bytes = min(left, kPieceVecs) * 16;
    if (lane == 0) {
      mbar_arrive_expect_tx(&bar[s], bytes);
      bulk_copy_g2s(buf + s * kPieceBytes, src, bytes, &bar[s]);
    }
    ++issued;
    left -= NW * kPieceVecs;
    src += NW * kPieceBytes;
    if (left <= 0) {
      again = twice && !again;
      if (!again) row += row_step;
      open();
    }
  }
  __device__ void init(const T* x, int64_t x_stride, int n_rows, int vocab, int p, int ps, int warp, int64_t row0, int step,
                       bool both, uint8_t* ring, uint64_t* bars, int lane) {
    base = x; stride = x_stride; rows = n_rows; V = vocab; part = p; parts = ps;
    first = warp; row = row0; row_step = step; twice = both; again = false; issued = 0;
    buf = ring; bar = bars;
    if (lane == 0) {
      for (int i = 0; i < kDepth; ++i) mbar_init(&bar[i], 1);
      fence_mbar_init();
      fence_proxy_async_smem();
    }
    __syncwarp();
    open();
    for (int i = 0; i < kDepth; ++i) issue(lane);
  }
  // piece n (of those issued) has arrived, in the slot returned
  __device__ __forceinline__ const uint8_t* wait(uint32_t n) {
    const uint32_t s = n % kDepth;
    bounded_wait(&bar[s], (n / kDepth) & 1u, DEV_TIMEOUT_FULL);  // (a lost copy: its error is recorded, nobody hangs)
    return buf + s * kPieceBytes;
  }
};

// A lane's vectors of a consumed piece (every 32nd one); those past its end are -inf.
template <typename T, int NW>
__device__ __forceinline__ void take_piece(Feed<T, NW>& feed, uint32_t n, int vecs, int lane, uint4 (&u)[kLaneVecs]) {
  const uint4* p = reinterpret_cast<const uint4*>(feed.wait(n)) + lane;
  constexpr uint32_t NI = sizeof(T) == 2 ? 0xff80ff80u : 0xff800000u;
  if (vecs >= kPieceVecs) {
#pragma unroll
    for (int j = 0; j < kLaneVecs; ++j) u[j] = p[j * 32];
  } else {
#pragma unroll
    for (int j = 0; j < kLaneVecs; ++j) u[j] = j * 32 + lane < vecs ? p[j * 32] : make_uint4(NI, NI, NI, NI);
  }
  __syncwarp();
  feed.issue(lane);
}

// Maxima of a lane's vectors, NaN aside: of each for the piece, and of four classes over all its pieces.
__device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ float lo_bf16(uint32_t a) { return __uint_as_float(a << 16); }
__device__ __forceinline__ float hi_bf16(uint32_t a) { return __uint_as_float(a & 0xffff0000u); }
__device__ __forceinline__ float max_of(const float4& v) { return fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)); }
template <typename T> struct Maxima;
template <> struct Maxima<__nv_bfloat16> {
  struct __align__(kLaneVecs * 2) Store {
    uint32_t v[kLaneVecs / 2];
    __device__ __forceinline__ float most() const {
      uint32_t a = v[0];
#pragma unroll
      for (int j = 1; j < kLaneVecs / 2; ++j) a = max2(a, v[j]);
      return fmaxf(lo_bf16(a), hi_bf16(a));
    }
    // which of them are >= least (a bf16 value), a bit each
    __device__ __forceinline__ uint32_t reaching(float least) const {
      const __nv_bfloat162 l = __float2bfloat162_rn(least);
      uint32_t b = 0;
#pragma unroll
      for (int j = 0; j < kLaneVecs / 2; ++j)
        b |= __hge2_mask(reinterpret_cast<const __nv_bfloat162&>(v[j]), l) & (0x00020001u << (2 * j));
      return (b | (b >> 16)) & ((1u << kLaneVecs) - 1u);
    }
  };
  uint32_t m[2] = {0xff80ff80u, 0xff80ff80u};
  __device__ __forceinline__ Store take(const uint4 (&u)[kLaneVecs]) {
    uint32_t h[kLaneVecs];
    Store s;
#pragma unroll
    for (int j = 0; j < kLaneVecs; ++j) h[j] = max2(max2(u[j].x, u[j].y), max2(u[j].z, u[j].w));
#pragma unroll
    for (int j = 0; j < kLaneVecs / 2; ++j) {
      s.v[j] = max2(__byte_perm(h[2 * j], h[2 * j + 1], 0x5410), __byte_perm(h[2 * j], h[2 * j + 1], 0x7632));
      m[j & 1] = max2(m[j & 1], s.v[j]);
    }
    return s;
  }
  __device__ __forceinline__ float4 all() const { return make_float4(lo_bf16(m[0]), hi_bf16(m[0]), lo_bf16(m[1]), hi_bf16(m[1])); }
};
template <> struct Maxima<float> {
  struct __align__(16) Store {
    float v[kLaneVecs];
    __device__ __forceinline__ float most() const {
      float a = v[0];
#pragma unroll
      for (int j = 1; j < kLaneVecs; ++j) a = fmaxf(a, v[j]);
      return a;
    }
    __device__ __forceinline__ uint32_t reaching(float least) const {
      uint32_t b = 0;
#pragma unroll
      for (int j = 0; j < kLaneVecs; ++j) b |= v[j] >= least ? 1u << j : 0u;
      return b;
    }
  };
  float m[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
  __device__ __forceinline__ Store take(const uint4 (&u)[kLaneVecs]) {
    Store s;
#pragma unroll
    for (int j = 0; j < kLaneVecs; ++j) {
      s.v[j] = fmaxf(fmaxf(__uint_as_float(u[j].x), __uint_as_float(u[j].y)), fmaxf(__uint_as_float(u[j].z), __uint_as_float(u[j].w)));
      m[j & 3] = fmaxf(m[j & 3], s.v[j]);
    }
    return s;
  }
  __device__ __forceinline__ float4 all() const { return make_float4(m[0], m[1], m[2], m[3]); }
};

// Maximum of a lane's vectors, NaN aside.
template <typename T> __device__ __forceinline__ float max_vecs(const uint4 (&u)[kLaneVecs]) {
  if constexpr (sizeof(T) == 2) {
    uint32_t a = max2(max2(u[0].x, u[0].y), max2(u[0].z, u[0].w));
#pragma unroll
    for (int j = 1; j < kLaneVecs; ++j) a = max2(a, max2(max2(u[j].x, u[j].y), max2(u[j].z, u[j].w)));
    return fmaxf(lo_bf16(a), hi_bf16(a));
  } else {
    float a = -INFINITY;
#pragma unroll
    for (int j = 0; j < kLaneVecs; ++j)
      a = fmaxf(a, fmaxf(fmaxf(__uint_as_float(u[j].x), __uint_as_float(u[j].y)), fmaxf(__uint_as_float(u[j].z), __uint_as_float(u[j].w))));
    return a;
  }
}

// N of a lane's vectors, none of whose elements is above the running maximum.
template <typename T, int N, bool E> __device__ __forceinline__ void add_vecs(RunningT<E>& s, const uint4* u, float c) {
  constexpr int VEC = Elt<T>::VEC;
  float f[N * VEC];
#pragma unroll
  for (int j = 0; j < N; ++j) {
    float e[VEC];
    if constexpr (sizeof(T) == 2) {
      Elt<T>::unpack(make_uint4(max2_nan(u[j].x, kClampBf16), max2_nan(u[j].y, kClampBf16), max2_nan(u[j].z, kClampBf16),
                                max2_nan(u[j].w, kClampBf16)), e);
    } else {
      Elt<T>::unpack(u[j], e);
#pragma unroll
      for (int i = 0; i < VEC; ++i) e[i] = max_nan(e[i], kClamp);
    }
#pragma unroll
    for (int i = 0; i < VEC; ++i) f[j * VEC + i] = e[i];
  }
  s.template add<true>(f, c);
}
// A lane's vectors of a piece, the maximum of which is known.
template <typename T, bool E>
__device__ __forceinline__ void add_piece(RunningT<E>& s, const uint4 (&u)[kLaneVecs], int vecs, float most, float c) {
  constexpr int VEC = Elt<T>::VEC;
  if (most > s.m) s.raise(most, c);
  if (__any_sync(0xffffffffu, !s.near())) {
#pragma unroll 1
    for (int j = 0; j < kLaneVecs; ++j) {  // (by elements, in a short loop: in pairs, or unrolled, it cost other rows 2%, 3%)
      uint4 w = u[0];
#pragma unroll
      for (int i = 1; i < kLaneVecs; ++i) w = i == j ? u[i] : w;
      float f[VEC];
      Elt<T>::unpack(w, f);
#pragma unroll
      for (int i = 0; i < VEC; ++i) s.add_one(f[i], c);
    }
  } else if (vecs >= kPieceVecs) {
    add_vecs<T, kLaneVecs>(s, u, c);
  } else {
#pragma unroll
    for (int j = 0; j < kLaneVecs; j += 2)
      if (vecs > j * 32) add_vecs<T, 2>(s, u + j, c);
  }
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
// key of a maximum: -inf may stand for -inf, for NaN or for no element at all, so it is below every bound
__device__ __forceinline__ uint32_t max_key(float m) { return m == -INFINITY ? 0u : order_key(m); }
// A candidate: larger key first, then the lower index.
__device__ __forceinline__ unsigned long long candidate(uint32_t key, int i) {
  return ((unsigned long long)key << 32) | (0xffffffffu - (uint32_t)i);
}

// Threads of the NW warps that share a row (or a part of one).
template <int NW> __device__ __forceinline__ void team_sync() {
  if (NW == 1) __syncwarp();
  else __syncthreads();
}
template <int NW> __device__ __forceinline__ int team_thread() { return NW == 1 ? (threadIdx.x & 31) : threadIdx.x; }

template <int NW> struct TopShared {
  static constexpr int CAP = NW == 1 ? 192 : 512;  // candidates ranked at once; more go the slow way
  unsigned long long cand[CAP];
  int vec[CAP];
  float group[NW == 1 ? 1 : 256];
  int slots[NW];
  int n, nvec;
};

// Disjoint sets of elements whose maxima bound the top k: with G of them about -G ln(1 - k / G) elements reach the
// k-th largest maximum (1.1 to 2 k here).
__host__ __device__ inline int group_count(int k, int least) {
  const int g = k <= 24 ? 32 : k <= 48 ? 64 : k <= 96 ? 128 : 256;
  return g < least ? least : g;
}

// The k-th largest of a warp's 32 values, one to a lane (none NaN): a bitonic sort.
__device__ __forceinline__ float kth_of_32(float v, int k) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int size = 2; size <= 32; size *= 2)
#pragma unroll
    for (int d = size / 2; d > 0; d /= 2) {
      const float o = __shfl_xor_sync(0xffffffffu, v, d);
      v = ((lane & size) == 0) == ((lane & d) == 0) ? fmaxf(v, o) : fminf(v, o);
    }
  return __shfl_sync(0xffffffffu, v, k - 1);
}
// The largest t, its bits from hi to lo beside those of t0, such that at least k of a warp's keys (R to a lane) are
// >= t, given that at least k are >= t0.
template <int R> __device__ __forceinline__ uint32_t kth_key(const uint32_t (&g)[R], int k, uint32_t t0, int hi, int lo) {
  uint32_t tau = t0;
#pragma unroll 1
  for (int b = hi; b >= lo; --b) {
    const uint32_t t = tau | (1u << b);
    int n = 0;
#pragma unroll
    for (int i = 0; i < R; ++i) n += g[i] >= t;
    if (__reduce_add_sync(0xffffffffu, n) >= k) tau = t;
  }
  return tau;
}
template <int R> __device__ __forceinline__ uint32_t kth_key(const float* group, int k, uint32_t t0, int hi, int lo) {
  uint32_t g[R];
#pragma unroll
  for (int i = 0; i < R; ++i) g[i] = max_key(group[i * 32 + (threadIdx.x & 31)]);
  return kth_key(g, k, t0, hi, lo);
}

// Appends a value of each lane that has one; n counts them all, those past CAP are dropped.  The counter of a
// single warp's list is a register of all lanes, that of several warps (or blocks) is in shared memory.
template <typename V> __device__ __forceinline__ void push(bool yes, V v, V* list, int& n, int cap) {
  const uint32_t vote = __ballot_sync(0xffffffffu, yes);
  const int at = n + __popc(vote & ((1u << (threadIdx.x & 31)) - 1u));
  if (yes && at < cap) list[at] = v;
  n += __popc(vote);
}
template <typename V> __device__ __forceinline__ void push(bool yes, V v, V* list, int* n, int cap) {
  const uint32_t vote = __ballot_sync(0xffffffffu, yes);
  if (vote == 0) return;
  const int lane = threadIdx.x & 31, first = __ffs(vote) - 1;
  int at = 0;
  if (lane == first) at = atomicAdd(n, __popc(vote));
  at = __shfl_sync(0xffffffffu, at, first) + __popc(vote & ((1u << lane) - 1u));
  if (yes && at < cap) list[at] = v;
}

// Count of the row's elements with key >= t, the same in every thread of the team.
template <typename T, int NW> __device__ int count_from(const T* x, int V, uint32_t t, TopShared<NW>& sh) {
  int n = 0;
#pragma unroll 4
  for (int i = team_thread<NW>(); i < V; i += NW * 32) n += order_key(Elt<T>::get(x + i)) >= t;
  n = __reduce_add_sync(0xffffffffu, n);
  if (NW == 1) return n;
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sh.slots[threadIdx.x >> 5] = n;
  __syncthreads();
  n = 0;
#pragma unroll
  for (int w = 0; w < NW; ++w) n += sh.slots[w];
  return n;
}

// Appends to the n candidates the lowest-indexed elements of key K, up to k candidates; returns their number.
template <typename T, int NW> __device__ int append_equal(const T* x, int V, uint32_t K, int n, int k, TopShared<NW>& sh) {
  const int tid = team_thread<NW>(), lane = tid & 31, w = tid >> 5;
  for (int i0 = 0; i0 < V && n < k; i0 += NW * 32) {
    const int i = i0 + tid;
    const bool eq = i < V && order_key(Elt<T>::get(x + i)) == K;
    const uint32_t vote = __ballot_sync(0xffffffffu, eq);
    int at = n, all = __popc(vote);
    if (NW > 1) {
      __syncthreads();
      if (lane == 0) sh.slots[w] = all;
      __syncthreads();
      all = 0;
#pragma unroll
      for (int j = 0; j < NW; ++j) {
        if (j < w) at += sh.slots[j];
        all += sh.slots[j];
      }
    }
    at += __popc(vote & ((1u << lane) - 1u));
    if (eq && at < k) sh.cand[at] = candidate(K, i);
    n = min(k, n + all);
  }
  team_sync<NW>();
  return n;
}

// The candidates of a row in which more than CAP elements reach the bound (long runs of equal values, as in
// constant rows and rows masked with a finite value): every element above the key K of the k-th largest one
// (fewer than k), then the lowest-indexed ones equal to it.  tau is the k-th largest group maximum, so K >= tau, and
// K = tau unless k elements are above it.
template <typename T, int NW> __device__ int select_slow(const T* x, int V, int k, uint32_t tau, TopShared<NW>& sh) {
  uint32_t K = tau;
  if (count_from<T, NW>(x, V, tau + 1, sh) >= k) {
    K = 0;
#pragma unroll 1
    for (int b = 31; b >= 0; --b) {
      const uint32_t t = K | (1u << b);
      if (count_from<T, NW>(x, V, t, sh) >= k) K = t;
    }
  }
  team_sync<NW>();
  if (team_thread<NW>() == 0) sh.n = 0;
  team_sync<NW>();
#pragma unroll 4
  for (int i = team_thread<NW>(); i < V; i += NW * 32) {
    const uint32_t q = order_key(Elt<T>::get(x + i));
    if (q > K) sh.cand[atomicAdd(&sh.n, 1)] = candidate(q, i);
  }
  team_sync<NW>();
  const int n = sh.n;
  team_sync<NW>();
  return append_equal<T, NW>(x, V, K, n, k, sh);
}

// The candidates of a short row (one warp): its keys in registers, the k-th largest found bit by bit, every element
// above it and the lowest-indexed ones equal to it.
constexpr int kShortRow = 1024;
template <typename T> __device__ int select_short(const T* x, int V, int k, TopShared<1>& sh) {
  constexpr int R = kShortRow / 32;
  const int lane = threadIdx.x & 31;
  uint32_t q[R];
#pragma unroll
  for (int i = 0; i < R; ++i) q[i] = i * 32 + lane < V ? order_key(Elt<T>::get(x + i * 32 + lane)) : 0u;
  uint32_t K = 0;
#pragma unroll 1
  for (int b = 31; b >= 0; --b) {
    const uint32_t t = K | (1u << b);
    int n = 0;
#pragma unroll
    for (int i = 0; i < R; ++i)
      if (i * 32 < V) n += q[i] >= t;
    if (__reduce_add_sync(0xffffffffu, n) >= k) K = t;
  }
  int n = 0;  // (fewer than k are above K)
#pragma unroll
  for (int i = 0; i < R; ++i)
    if (i * 32 < V) push(q[i] > K, candidate(q[i], i * 32 + lane), sh.cand, n, k);
#pragma unroll
  for (int i = 0; i < R; ++i)
    if (i * 32 < V && n < k) push(q[i] == K && i * 32 + lane < V, candidate(K, i * 32 + lane), sh.cand, n, k);
  __syncwarp();
  return min(n, k);
}

struct LogprobArgs {
  const void* logits;
  int64_t stride;
  const int32_t* targets;
  int rows, vocab, k, parts, pieces;  // pieces: most of a part
  float scale;
  float *logp, *entropy, *lse, *top_logp;
  int32_t* top_ids;
};
// dynamic shared memory: rings, then per team the vectors' maxima
template <typename T, int NW, int TEAMS> size_t logprobs_smem(const LogprobArgs& a) {
  return (size_t)NW * TEAMS * kDepth * kPieceBytes +
         (a.k ? (size_t)TEAMS * a.pieces * 32 * sizeof(typename Maxima<T>::Store) : 0);
}

// NW warps to a row (TEAMS rows to a block), or a cluster of `parts` blocks of NW warps.  A single warp goes on to further
// rows; the grid has a block (or cluster) for every row of several warps.  Top alternatives: the
// k-th largest of the maxima of 32 to 256 disjoint sets of elements is a bound that at least k elements reach, and
// few more where values come in any order; the maxima of the single vectors, kept in shared memory, say which
// vectors to read again (from L2).  The candidates' ranks are counted.
// Measured: 32768 x 6400 bf16 118 us with 16 alternatives, 91 us without (419 MB, 64 us at the copy rate; the ring
// alone, without arithmetic, takes 64 us).  Bound by instructions: about 270 for a lane's 32 logits of a piece
// (unpacking, maxima, clamp, exponential, two sums) and 700 for a row's alternatives fill 2/3 of the issue slots and
// half of the exponential units.  With 7/8 of each row masked 115 us by -inf or -1e4, 176 us by -1e9, whose pieces are
// added element by element.  1021 x 50001 38 us, 1 x 32000 with 20 about 8.5 us (8 of them the host's call).
//
// LOOSE (one warp to a row): a short row with too few vectors for its groups to bound anything, or a large k with
// fewer than 256 groups.  All of its elements are ranked, or where those are too many none is found by a bound and
// select_short is asked: 32768 rows of 300 with 64 alternatives 243 us (364 by the bound), of 900 with 128 366 us
// (1011 by a whole block to a row), of 64 with 30 76 us (86).  A kernel of its own, since the code costs the other 3%.
template <typename T, int NW, int TEAMS, bool LOOSE = false>
__global__ void __launch_bounds__(NW * TEAMS * 32, NW == 1 ? kRowBlocks : 24 / NW) logprobs_kernel(const LogprobArgs a) {
  constexpr int VEC = Elt<T>::VEC, CAP = TopShared<NW>::CAP;
  using Store = typename Maxima<T>::Store;
  extern __shared__ __align__(128) uint8_t dyn[];
  __shared__ TopShared<NW> top[TEAMS];
  __shared__ float3 red[NW], parts_st[kMaxParts];  // (Stats)
  __shared__ uint64_t bars[NW * TEAMS * kDepth];
  static_assert(NW == 1 || TEAMS == 1, "a block barrier serves one team");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, team = NW == 1 ? warp : 0, tid = team_thread<NW>();
  const int parts = NW == 1 ? 1 : a.parts, part = parts > 1 ? (int)(blockIdx.x & (parts - 1)) : 0;
  const int V = a.vocab, k = a.k, groups = group_count(k, NW * parts);
  const float c = a.scale * kLog2e;
  TopShared<NW>& sh = top[team];
  Store* vmax = reinterpret_cast<Store*>(dyn + NW * TEAMS * kDepth * kPieceBytes) + (int64_t)team * a.pieces * 32;
  const int64_t row0 = parts > 1 ? blockIdx.x / parts : (int64_t)blockIdx.x * TEAMS + team;
  const int row_step = parts > 1 ? (int)(gridDim.x / parts) : (int)gridDim.x * TEAMS;

  Feed<T, NW> feed;
  feed.init(static_cast<const T*>(a.logits), a.stride, a.rows, V, part, parts, NW == 1 ? 0 : warp, row0, row_step, false,
            dyn + warp * kDepth * kPieceBytes, bars + warp * kDepth, lane);
  if (parts > 1) cg::this_cluster().barrier_arrive();
  uint32_t taken = 0;
  bool entered = parts == 1;

  for (int64_t r = row0; r < a.rows; r += row_step) {
    const T* x = feed.base + r * a.stride;
    const Span<T> sp(x, V, part, parts);
    // the target's logit, asked for early
    int t = -1;
    float xt = 0.f;
    if (a.logp && part == 0 && tid == 0) {
      t = a.targets[r];
      if (t >= V) t = -1;
      if (t >= 0) xt = Elt<T>::get(x + t);
    }
    const int single = (NW == 1 || tid < 32) ? sp.single(V, part, parts, tid) : -1;
    const float xs = single >= 0 ? Elt<T>::get(x + single) : -INFINITY;
    if (k > 0 && tid == 0) { sh.n = 0; sh.nvec = 0; }

    Running run;
    Maxima<T> mx;
    for (int v = sp.lo + (NW == 1 ? 0 : warp) * kPieceVecs, i = NW == 1 ? 0 : warp; v < sp.hi; v += NW * kPieceVecs, i += NW) {
      uint4 u[kLaneVecs];
      take_piece(feed, taken++, sp.hi - v, lane, u);
      const Store m = mx.take(u);
      if (k > 0) vmax[i * 32 + lane] = m;
      add_piece<T>(run, u, sp.hi - v, m.most(), c);
    }
    if (single >= 0) run.add_one(xs, c);
    Stats s = run.sums(c);
    float4 g4 = mx.all();
    g4.x = fmaxf(g4.x, xs);
    s.join_warp(c);
    if constexpr (NW > 1) {
      if (k > 0) {
        if (!entered) { cg::this_cluster().barrier_wait(); entered = true; }  // the other blocks run: their memory may be written
        const int mine = groups / (NW * parts), at = (part * NW + warp) * mine;  // this warp's groups
        auto put = [&](int i, float v) {
          if (parts == 1) sh.group[i] = v;
          else
            for (int q = 0; q < parts; ++q) *cg::this_cluster().map_shared_rank(&sh.group[i], q) = v;
        };
        if (mine == 128) {
          put(at + lane, g4.x); put(at + 32 + lane, g4.y); put(at + 64 + lane, g4.z); put(at + 96 + lane, g4.w);
        } else if (mine == 64) {
          put(at + lane, fmaxf(g4.x, g4.y)); put(at + 32 + lane, fmaxf(g4.z, g4.w));
        } else {
          float g = max_of(g4);
          const int per = 32 / mine;
          for (int o = per >> 1; o > 0; o >>= 1) g = fmaxf(g, __shfl_xor_sync(0xffffffffu, g, o));
          if ((lane & (per - 1)) == 0) put(at + lane / per, g);
        }
      }
      if (lane == 0) red[warp] = s.pack();
      __syncthreads();
      s = lane < NW ? Stats(red[lane]) : Stats();
      s.join_warp(c);
      if (parts > 1) {
        if (!entered) { cg::this_cluster().barrier_wait(); entered = true; }
        if (tid < parts) *cg::this_cluster().map_shared_rank(&parts_st[part], tid) = s.pack();
        cg::this_cluster().sync();
        s = lane < parts ? Stats(parts_st[lane]) : Stats();
        s.join_warp(c);
      }
    }
    const float ln_s0 = logf(s.s0);
    if (part == 0 && tid == 0) {
      const float h = fmaf(-kLn2, __fdividef(s.s1, s.s0), ln_s0);
      if (a.lse) a.lse[r] = s.s0 == 0.f ? -INFINITY : fmaf(s.m, a.scale, ln_s0);
      if (a.entropy) a.entropy[r] = (s.s0 == 0.f || h < 0.f) ? 0.f : h;
      if (a.logp) a.logp[r] = t >= 0 ? log_prob(xt, s, ln_s0, a.scale) : 0.f;
    }
    if (k > 0) {
      if (NW == 1) __syncwarp();
      // every warp finds the bound: a value that at least k elements reach (0: fewer than k groups have a finite
      // maximum, and every finite logit is a candidate).  Keys are cut to their upper half at first.
      auto bound = [&](uint32_t t0, int hi, int lo) -> uint32_t {
        if constexpr (NW == 1) {
          if (groups == 64) {
            const uint32_t g[2] = {max_key(fmaxf(g4.x, g4.y)), max_key(fmaxf(g4.z, g4.w))};
            return kth_key(g, k, t0, hi, lo);
          }
          const uint32_t g[4] = {max_key(g4.x), max_key(g4.y), max_key(g4.z), max_key(g4.w)};
          return kth_key(g, k, t0, hi, lo);
        } else {
          return groups == 64 ? kth_key<2>(sh.group, k, t0, hi, lo)
                 : groups == 128 ? kth_key<4>(sh.group, k, t0, hi, lo) : kth_key<8>(sh.group, k, t0, hi, lo);
        }
      };
      const uint32_t tau = LOOSE ? 0u
                           : groups == 32 ? max_key(kth_of_32(NW == 1 ? max_of(g4) : sh.group[lane % 256], k)) : bound(0u, 31, 16);
      // as a logit: of a cut bf16 key the value itself (below zero a bf16 value's key ends in ones), so that vectors and
      // their elements are compared with the same number and -inf, which also stands for no element, never reaches it
      const uint32_t exact = sizeof(T) == 2 && tau < 0x80000000u ? tau | 0xffffu : tau;
      const float least = LOOSE && V > CAP ? NAN : tau == 0 ? -Elt<T>::MAX : key_value(exact);
      TopShared<NW>& first = parts > 1 ? *cg::this_cluster().map_shared_rank(&sh, 0) : sh;
      int own_n = 0, own_vec = 0;  // the counters of a single warp
      auto push_cand = [&](bool yes, float v, int i) {
        if constexpr (NW == 1) push(yes, candidate(order_key(v), i), sh.cand, own_n, CAP);
        else push(yes, candidate(order_key(v), i), first.cand, &first.n, CAP);
      };
      if (__any_sync(0xffffffffu, xs >= least)) push_cand(xs >= least, xs, single);
      // the vectors that reach it, as many pieces at a time as a lane's word has bits for
      constexpr int PW = 32 / kLaneVecs;
      const int p0 = NW == 1 ? 0 : warp;
      for (int v0 = sp.lo + p0 * kPieceVecs, i0 = p0; v0 < sp.hi; v0 += PW * NW * kPieceVecs, i0 += PW * NW) {
        uint32_t bits = 0;
        const int n = min(PW, (sp.hi - v0 + NW * kPieceVecs - 1) / (NW * kPieceVecs));
        for (int i = 0; i < n; ++i) bits |= vmax[(i0 + i * NW) * 32 + lane].reaching(least) << (kLaneVecs * i);
        while (__any_sync(0xffffffffu, bits != 0)) {
          const int b = __ffs(bits) - 1;
          const int v = v0 + b / kLaneVecs * NW * kPieceVecs + b % kLaneVecs * 32 + lane;
          const bool in = bits != 0 && v < sp.hi;
          if constexpr (NW == 1) push(in, v, sh.vec, own_vec, CAP);
          else push(in, v, sh.vec, &sh.nvec, CAP);
          bits &= bits - 1;
        }
      }
      team_sync<NW>();
      const int nvec = NW == 1 ? own_vec : sh.nvec;
      for (int i0 = warp * 32 * (NW > 1); i0 < min(nvec, CAP); i0 += NW * 32) {
        float f[VEC];
        int at = 0;
        uint32_t bits = 0;
        if (i0 + lane < min(nvec, CAP)) {
          at = sp.head + sh.vec[i0 + lane] * VEC;
          Elt<T>::unpack(load16(x + at), f);
#pragma unroll
          for (int j = 0; j < VEC; ++j) bits |= f[j] >= least ? 1u << j : 0u;
        }
        while (__any_sync(0xffffffffu, bits != 0)) {
          const int b = __ffs(bits) - 1;
          float v = 0.f;
#pragma unroll
          for (int j = 0; j < VEC; ++j) v = b == j ? f[j] : v;
          push_cand(bits != 0, v, at + b);
          bits &= bits - 1;
        }
      }
      if (nvec > CAP) {  // vectors were dropped: the slow way
        own_n += CAP + 1;
        if (NW > 1 && tid == 0) atomicAdd(&first.n, CAP + 1);
      }
      if (parts > 1) cg::this_cluster().sync();
      else team_sync<NW>();
      if (part == 0) {
        int n = NW == 1 ? own_n : sh.n;
        team_sync<NW>();
        if (LOOSE && V > CAP) {
          if constexpr (LOOSE) n = select_short<T>(x, V, k, sh);
        } else if (n > CAP) {
          n = select_slow<T, NW>(x, V, k, groups == 32 || tau == 0 ? tau : bound(tau, 15, 0), sh);
        } else if (n < k) {  // (tau = 0) masked logits, then NaN ones, by their index
          n = append_equal<T, NW>(x, V, kKeyMasked, n, k, sh);
          n = append_equal<T, NW>(x, V, 0u, n, k, sh);
        }
        for (int i = tid; i < n; i += NW * 32) {
          const unsigned long long me = sh.cand[i];
          int rank = 0;
#pragma unroll 4
          for (int j = 0; j < n; ++j) rank += sh.cand[j] > me;
          if (rank < k) {
            const int64_t o = r * k + rank;
            if (a.top_logp) a.top_logp[o] = log_prob(key_value((uint32_t)(me >> 32)), s, ln_s0, a.scale);
            a.top_ids[o] = (int32_t)(0xffffffffu - (uint32_t)me);
          }
        }
        team_sync<NW>();
      }
    }
    if (NW > 1) break;  // one row: red, parts_st and the groups have no barrier between a row's reads and the next one's writes
  }
  if (!entered) cg::this_cluster().barrier_wait();
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

// A row whose lse is so far from 0 that its rounding shows in p (kFarLse on, at most 2^-17 of p below it; a row masked with -1e9,
// whose lse holds nothing of ln V, at the far end): one block finds the row's maximum and sum again and has all of its
// gradient, read a second time after the whole row was read once (it may lie in the logits' place).  32768 x 6400 bf16
// of such rows 215 us, 130 us of others.
constexpr float kFarLse = 256.f;
template <typename T, int NT>
__device__ __forceinline__ void far_row(const T* x, T* d, int V, float scale, int t, float g, float h, float gh, bool same) {
  constexpr int VEC = Elt<T>::VEC;
  __shared__ float3 red[NT / 32];
  const int tid = threadIdx.x, lane = tid & 31;
  const float c = scale * kLog2e;
  const Span<T> sp(x, V, 0, 1);
  RunningT<false> run;
  for (int v = tid; v < sp.hi; v += NT) {
    float f[VEC];
    Elt<T>::unpack(load16(x + sp.head + (int64_t)v * VEC), f);
    run.add_any(f, c);
  }
  const int single = sp.single(V, 0, 1, tid);
  if (single >= 0) run.add_one(Elt<T>::get(x + single), c);
  Stats s = run.sums(c);
  s.join_warp(c);
  if (lane == 0) red[tid >> 5] = s.pack();
  __syncthreads();
  s = lane < NT / 32 ? Stats(red[lane]) : Stats();
  s.join_warp(c);
  const float ln_s0 = logf(s.s0);
  auto grad = [&](float f, int i) {
    if (s.s0 == 0.f) return 0.f;
    const float l = fmaf(f - s.m, scale, -ln_s0), p = ex2(l * kLog2e);
    return p * fmaf(-h, fmaxf(l, kFloor), -gh) + (i == t ? g : 0.f);
  };
  if (same) {
    for (int v = tid; v < sp.hi; v += NT) {
      const int i0 = sp.head + v * VEC;
      float f[VEC];
      Elt<T>::unpack(load16(x + i0), f);
#pragma unroll
      for (int j = 0; j < VEC; ++j) f[j] = grad(f[j], i0 + j);
      *reinterpret_cast<uint4*>(d + i0) = Elt<T>::pack(f);
    }
    if (single >= 0) Elt<T>::put(d + single, grad(Elt<T>::get(x + single), single));
  } else {
    for (int i = tid; i < V; i += NT) Elt<T>::put(d + i, grad(Elt<T>::get(x + i), i));
  }
}

// d_j = scale [ g (1[j = t] - p_j) - h p_j (ln p_j + H) ], element by element from the row's saved statistics.  One
// block per (row, slice of the vocabulary); a thread has four vectors on the way at once, or, where logits and gradient
// rows do not share their place within 16 bytes, that many bytes' worth of single elements.
// With l = scale x - lse: d = p (-scale h l - scale (g + h H)), one exponential and paired fp32 instructions.  Masked
// logits are kept at -2^40 (l finite, p = 0).
template <typename T, int NT>
__global__ void __launch_bounds__(NT) logprobs_bwd_kernel(const LogprobBwdArgs a, int slices) {
  constexpr int VEC = Elt<T>::VEC, U = 4;
  constexpr float FLOOR = -0x1p40f;
  const int64_t r = blockIdx.x / slices;
  const int part = (int)(blockIdx.x % slices);
  const int V = a.vocab, tid = threadIdx.x;
  const T* x = static_cast<const T*>(a.logits) + r * a.stride;
  T* d = static_cast<T*>(a.d) + r * a.d_stride;
  const bool same = ((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(d)) & 15) == 0;
  const Span<T> sp(x, V, 0, 1);
  // this thread's first vectors, asked for before the row's statistics
  uint4 u[U];
  const int v0 = part * NT * U + tid;
  if (same) {
#pragma unroll
    for (int i = 0; i < U; ++i)
      if (v0 + i * NT < sp.hi) u[i] = load16(x + sp.head + (int64_t)(v0 + i * NT) * VEC);
  }
  const float lse = a.lse[r], scale = a.scale;
  // a row masked wholly (with -inf, or with the type's lowest value) or with a token forced by the highest value has
  // no gradient: beside a mask's value the saved lse cannot hold what its p would need
  const bool none = fabsf(lse) > 1e30f;
  int t = (a.g_logp && a.targets) ? a.targets[r] : -1;
  if (t >= V) t = -1;
  const float g = t >= 0 ? a.g_logp[r] * scale : 0.f;
  const float h = a.g_entropy ? a.g_entropy[r] * scale : 0.f, H = a.g_entropy ? a.entropy[r] : 0.f;
  const float gh = fmaf(h, H, g);
  // fp32 rows at another place than their gradient's ask about far ones only once their loads are on their way: asked here
  // 8000 x 6400 takes 83 us instead of 70, where bf16 takes 60 instead of 64.
  const bool far = fabsf(lse) > kFarLse && !none;
  constexpr bool LATE = sizeof(T) == 4;
  if (!LATE && far) {
    if (part == 0) far_row<T, NT>(x, d, V, scale, t, g, h, gh, same);
    return;
  }
  auto grad = [&](float f, int i) {
    if (none) return 0.f;
    const float l = fmaf(f, scale, -lse), p = ex2(l * kLog2e);
    return p * fmaf(-h, fmaxf(l, kFloor), -gh) + (i == t ? g : 0.f);  // (ln p kept off -inf where p = 0)
  };
  if (same) {
    if (LATE && far) {
      if (part == 0) far_row<T, NT>(x, d, V, scale, t, g, h, gh, true);
      return;
    }
    const bool fast = fabsf(lse) <= kFarLse;  // (not NaN, not beyond 1e30)
    const uint64_t s2 = f2_pack(scale, scale), n2 = f2_pack(-lse, -lse), e2 = f2_pack(kLog2e, kLog2e), h2 = f2_pack(-h, -h),
                   g2 = f2_pack(-gh, -gh);
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int v = v0 + i * NT;
      if (v >= sp.hi) break;
      const int i0 = sp.head + v * VEC;
      float f[VEC];
      if (fast) {
        if constexpr (sizeof(T) == 2) {
          constexpr uint32_t F = 0xd380d380u;  // -2^40 twice
          Elt<T>::unpack(make_uint4(max2_nan(u[i].x, F), max2_nan(u[i].y, F), max2_nan(u[i].z, F), max2_nan(u[i].w, F)), f);
        } else {
          Elt<T>::unpack(u[i], f);
#pragma unroll
          for (int j = 0; j < VEC; ++j) f[j] = max_nan(f[j], FLOOR);
        }
#pragma unroll
        for (int j = 0; j < VEC; j += 2) {
          const uint64_t l = fma2(f2_pack(f[j], f[j + 1]), s2, n2);
          float a0, a1;
          f2_unpack(mul2(l, e2), a0, a1);
          f2_unpack(mul2(f2_pack(ex2(a0), ex2(a1)), fma2(h2, l, g2)), f[j], f[j + 1]);
        }
        if (t >= i0 && t < i0 + VEC) {
#pragma unroll
          for (int j = 0; j < VEC; ++j) f[j] += t == i0 + j ? g : 0.f;
        }
      } else {
        Elt<T>::unpack(u[i], f);
#pragma unroll
        for (int j = 0; j < VEC; ++j) f[j] = grad(f[j], i0 + j);
      }
      *reinterpret_cast<uint4*>(d + i0) = Elt<T>::pack(f);
    }
    const int single = part == 0 ? sp.single(V, 0, 1, tid) : -1;
    if (single >= 0) Elt<T>::put(d + single, grad(Elt<T>::get(x + single), single));
  } else {
    constexpr int E = VEC * 2;
    const int hi = min((int64_t)V, (int64_t)(part + 1) * NT * U * VEC);  // (vectors of a slice, in elements)
    const int end = LATE && far ? 0 : hi;
    for (int i0 = part * NT * U * VEC + tid; i0 < hi; i0 += NT * E) {
      float f[E];
#pragma unroll
      for (int j = 0; j < E; ++j) f[j] = i0 + j * NT < hi ? Elt<T>::get(x + i0 + j * NT) : 0.f;
#pragma unroll
      for (int j = 0; j < E; ++j)
        if (i0 + j * NT < end) Elt<T>::put(d + i0 + j * NT, grad(f[j], i0 + j * NT));
    }
    if (LATE && far && part == 0) far_row<T, NT>(x, d, V, scale, t, g, h, gh, false);
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

// How the second exponential, e1 = 2^((x - m) log2 e) beside e = 2^((x - m) s log2 e), is had: not at all (no
// hard targets, or s = 1), as the square of the first (s = 1/2), as the fourth power (s = 1/4), or by itself.  A power has
// twice or four times the first one's relative error (2^-22 of the instruction): 1e-6 at most.
enum Second { kNone, kSquare, kFourth, kOwn };

// Sums of both exponentials about a maximum.
struct Sums2 {
  float m = -INFINITY, s = 0.f, h = 0.f;
  __device__ Sums2() {}
  __device__ explicit Sums2(const float3& v) : m(v.x), s(v.y), h(v.z) {}
  __device__ float3 pack() const { return make_float3(m, s, h); }
  __device__ __forceinline__ void rebase(float M, float c) {
    const float d = m == -INFINITY ? kFloor : m - M;
    s *= ex2(fmaxf(d * c, kFloor));
    h *= ex2(fmaxf(d * kLog2e, kFloor));
    m = M;
  }
  __device__ __forceinline__ void join_warp(float c) {
    rebase(max_warp(m), c);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      s += __shfl_xor_sync(0xffffffffu, s, o);
      h += __shfl_xor_sync(0xffffffffu, h, o);
    }
  }
};

// A thread's exponentials about a maximum m: x c - fl(m c), the rounding of m c taken out by settle() (as in RunningT)
// while |m| times the larger of both factors is at most kNear (the fourth power's rounding is then four times 2^-9);
// (x - m) c beyond it.
template <int SECOND> struct Exponent {
  float m, c, sub, mc, mc1;  // sub: -m where the difference is formed first (mc and mc1 are 0 then), else 0
  __device__ __forceinline__ void at(float M, float scale_c) {
    m = M; c = scale_c;
    const float most = SECOND == kNone ? c : fmaxf(c, kLog2e);
    const bool near = fabsf(m) * most <= kNear;
    sub = near || m == -INFINITY ? 0.f : -m;
    mc = near ? m * c : 0.f;
    mc1 = near ? m * kLog2e : 0.f;
  }
  __device__ __forceinline__ bool far() const { return sub != 0.f; }
  // what m c and m log2 e lost to rounding where they are used
  __device__ __forceinline__ float off() const { return far() ? 0.f : fmaf(m, c, -mc); }
  __device__ __forceinline__ float off1() const { return far() ? 0.f : fmaf(m, kLog2e, -mc1); }
  // factors that make sums of e and e1 exact about m
  __device__ __forceinline__ void settle(float& f, float& f1) const {
    f = f1 = 1.f;
    if (m != -INFINITY) {
      f = take_out(off());
      f1 = SECOND == kSquare ? take_out(2.f * off()) : SECOND == kFourth ? take_out(4.f * off())
           : SECOND == kOwn ? take_out(off1()) : 1.f;
    }
  }
  // a larger maximum M, and the factors that take sums of e and e1 there
  __device__ __forceinline__ void raise(float M, float& f, float& f1) {
    const Exponent was = *this;
    at(M, c);
    f = ex2(fmaxf((was.m - M) * c + (off() - was.off()), kFloor));  // (also where m was -inf)
    f1 = SECOND == kSquare ? f * f : SECOND == kFourth ? (f * f) * (f * f)
         : SECOND == kOwn ? ex2(fmaxf((was.m - M) * kLog2e + (off1() - was.off1()), kFloor)) : 1.f;
  }
  // of a pair; its difference to m where that is formed first (FAR: it may be)
  template <bool FAR> __device__ __forceinline__ uint64_t about(uint64_t x) const { return FAR ? add2(x, f2_pack(sub, sub)) : x; }
  __device__ __forceinline__ uint64_t first2(uint64_t x) const {
    float a, b;
    f2_unpack(fma2(x, f2_pack(c, c), f2_pack(-mc, -mc)), a, b);
    return f2_pack(ex2(a), ex2(b));
  }
  __device__ __forceinline__ uint64_t second2(uint64_t x, uint64_t e) const {
    if (SECOND == kSquare) return mul2(e, e);
    if (SECOND == kFourth) { const uint64_t q = mul2(e, e); return mul2(q, q); }
    float a, b;
    f2_unpack(fma2(x, f2_pack(kLog2e, kLog2e), f2_pack(-mc1, -mc1)), a, b);
    return f2_pack(ex2(a), ex2(b));
  }
  // one element of any value
  __device__ __forceinline__ void one(float x, float& e, float& e1) const {
    if (far()) x += sub;
    e = ex2(fmaf(x, c, -mc));
    if (SECOND == kSquare) e1 = e * e;
    else if (SECOND == kFourth) e1 = (e * e) * (e * e);
    else if (SECOND == kOwn) e1 = ex2(fmaf(x, kLog2e, -mc1));
    else e1 = 0.f;
  }
  // wf e + wc e1, of a pair (m not far) and of one element, rounded alike
  __device__ __forceinline__ uint64_t grad2(uint64_t x, uint64_t wf, uint64_t wc) const {
    const uint64_t e = first2(x);
    if (SECOND == kNone) return mul2(e, wf);
    if (SECOND == kSquare) return mul2(e, fma2(e, wc, wf));
    return fma2(wc, second2(x, e), mul2(wf, e));
  }
  __device__ __forceinline__ float grad(float x, float wf, float wc) const {
    float e, e1;
    one(x, e, e1);
    if (SECOND == kNone) return __fmul_rn(e, wf);
    if (SECOND == kSquare) return __fmul_rn(e, fmaf(e, wc, wf));
    return fmaf(wc, e1, __fmul_rn(wf, e));
  }
};

template <int NW> struct DistillShared {
  __align__(16) int id[kTopMax + 4];  // the teacher's alternatives, then the hard target
  __align__(16) float q[kTopMax + 4];
  float x[kTopMax + 4];     // the student's logits there
  int next_id[kTopMax];     // as given, of the next row
  float next_val[kTopMax];
  float sum, ent;    // sum q, sum q ln q
  float3 red[NW], part[kMaxParts];  // (Sums2)
};
// 4 bytes on their way to shared memory; all of the thread's have arrived
__device__ __forceinline__ void copy4(void* to, const void* from) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(to)), "l"(from) : "memory");
}
__device__ __forceinline__ void copies_done() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// A warp's sums of its pieces of a row and of its single element xs.
template <int SECOND, typename T, int NW>
__device__ __forceinline__ Sums2 distill_sums(Feed<T, NW>& feed, uint32_t& taken, const Span<T>& sp, float xs, bool single, float c,
                                              int lane) {
  constexpr int VEC = Elt<T>::VEC;
  Sums2 t;
  Exponent<SECOND> ex;
  ex.at(-INFINITY, c);
  float s = 0.f, h = 0.f;  // about ex
  auto raise = [&](float most) {
    float f, f1;
    ex.raise(most, f, f1);
    s *= f;
    h *= f1;
  };
  auto one = [&](float x) {
    if (x > ex.m) raise(x);
    float e, e1;
    ex.one(x, e, e1);
    s += e;
    h += e1;
  };
  for (int v = sp.lo + feed.first * kPieceVecs; v < sp.hi; v += NW * kPieceVecs) {
    uint4 u[kLaneVecs];
    const int vecs = sp.hi - v;
    take_piece(feed, taken++, vecs, lane, u);
    const float most = max_vecs<T>(u);
    if (most > ex.m) raise(most);
    uint64_t b0[2] = {0, 0}, b1[2] = {0, 0};
    auto add = [&](const uint4& w, auto far) {
      float f[VEC];
      Elt<T>::unpack(w, f);
#pragma unroll
      for (int l = 0; l < VEC; l += 2) {
        const uint64_t x = ex.template about<far.value>(f2_pack(f[l], f[l + 1])), e = ex.first2(x);
        b0[l / 2 & 1] = add2(b0[l / 2 & 1], e);
        if (SECOND == kSquare) b1[l / 2 & 1] = fma2(e, e, b1[l / 2 & 1]);
        else if (SECOND != kNone) b1[l / 2 & 1] = add2(b1[l / 2 & 1], ex.second2(x, e));
      }
    };
    if (__any_sync(0xffffffffu, ex.far())) {
#pragma unroll 1
      for (int j = 0; j < kLaneVecs; ++j) {  // (a short loop, as in add_piece())
        uint4 w = u[0];
#pragma unroll
        for (int i = 1; i < kLaneVecs; ++i) w = i == j ? u[i] : w;
        if constexpr (SECOND == kOwn) {  // (by elements: in pairs it cost other rows 281 instead of 277 us at 32768 x 6400)
          float f[VEC];
          Elt<T>::unpack(w, f);
#pragma unroll
          for (int l = 0; l < VEC; ++l) one(f[l]);
        } else {
          add(w, std::true_type());
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < kLaneVecs; ++j) {
        add(u[j], std::false_type());
        if (vecs <= (j + 1) * 32) break;
      }
    }
    float p, q;
    f2_unpack(add2(b0[0], b0[1]), p, q);
    s += p + q;
    if (SECOND != kNone) {
      f2_unpack(add2(b1[0], b1[1]), p, q);
      h += p + q;
    }
  }
  if (single) one(xs);
  float f, f1;
  ex.settle(f, f1);
  t.m = ex.m; t.s = s * f; t.h = h * f1;
  return t;
}

// d = wf e + wc e1 over a warp's pieces of a row.
template <int SECOND, typename T, int NW>
__device__ __forceinline__ void distill_gradient(Feed<T, NW>& feed, uint32_t& taken, const Span<T>& sp, const T* x, T* d, bool zero,
                                                 const Exponent<SECOND>& ex, float wf, float wc, int lane) {
  constexpr int VEC = Elt<T>::VEC;
  const bool plain = !zero && !ex.far() && ((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(d)) & 15) == 0;
  const uint64_t wf2 = f2_pack(wf, wf), wc2 = f2_pack(wc, wc);
  for (int v = sp.lo + feed.first * kPieceVecs; v < sp.hi; v += NW * kPieceVecs) {
    const int vecs = sp.hi - v;
    if (plain) {
      uint4 u[kLaneVecs];
      take_piece(feed, taken++, vecs, lane, u);
      T* o = d + sp.head + (int64_t)(v + lane) * VEC;
#pragma unroll
      for (int j = 0; j < kLaneVecs; ++j) {
        float f[VEC];
        Elt<T>::unpack(u[j], f);
#pragma unroll
        for (int l = 0; l < VEC; l += 2) f2_unpack(ex.grad2(f2_pack(f[l], f[l + 1]), wf2, wc2), f[l], f[l + 1]);
        if (j * 32 + lane < vecs) *reinterpret_cast<uint4*>(o + j * 32 * VEC) = Elt<T>::pack(f);
        if (vecs <= (j + 1) * 32) break;
      }
    } else {
      // one element at a time: rows without part in the loss, of masks only, or of another place within 16 bytes
      const T* e = reinterpret_cast<const T*>(feed.wait(taken++));
      T* o = d + sp.head + (int64_t)v * VEC;
#pragma unroll 4
      for (int l = lane; l < min(vecs, kPieceVecs) * VEC; l += 32) Elt<T>::put(o + l, zero ? 0.f : ex.grad(Elt<T>::get(e + l), wf, wc));
      __syncwarp();
      feed.issue(lane);
    }
  }
}

// Loss and gradient, a row to NW warps (TEAMS rows to a block) or to a cluster of `parts` blocks: the sums of both
// exponentials from one reading of the row, the dense part of the gradient from a second one (out of L2, and already
// under way while the sums are joined), then the at most k + 1 elements with a teacher's or target's share.  An element
// is read for the last time before its gradient is written, so the gradient may take its place.
// Measured, in a burst of 30 passes: 32768 x 6400 bf16 with 16 alternatives and hard targets at scale 1/2 198 us (209 us
// over seconds, under the power cap), 188 us at scale 1 without targets, 277 us at scale 0.7 with them (839 MB, 128 us at
// the copy rate); 2048 x 32000 63 us (262 MB), 64 x 262139 fp32 39 us (134 MB).  Bound by instructions (two
// exponentials a logit, about 1000 instructions a row beside them).
// Rows kept in shared memory from their sums to their gradient ran at 233 us: fewer warps fit.
template <typename T, int NW, int TEAMS, int SECOND>
__global__ void __launch_bounds__(NW * TEAMS * 32, 24 / (NW * TEAMS)) distill_kernel(const DistillArgs a) {
  extern __shared__ __align__(128) uint8_t dyn[];
  __shared__ DistillShared<NW> shared[TEAMS];
  __shared__ uint64_t bars[NW * TEAMS * kDepth];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, team = NW == 1 ? warp : 0, tid = team_thread<NW>();
  const bool lead = NW == 1 || warp == 0;  // the team's first warp
  const int parts = NW == 1 ? 1 : a.parts, part = parts > 1 ? (int)(blockIdx.x & (parts - 1)) : 0;
  const int V = a.vocab, k = a.k;
  DistillShared<NW>& sh = shared[team];
  const int64_t row0 = parts > 1 ? blockIdx.x / parts : (int64_t)blockIdx.x * TEAMS + team;
  const int step = parts > 1 ? (int)(gridDim.x / parts) : (int)gridDim.x * TEAMS;
  Feed<T, NW> feed;
  feed.init(static_cast<const T*>(a.logits), a.stride, a.rows, V, part, parts, NW == 1 ? 0 : warp, row0, step, a.d != nullptr,
            dyn + warp * kDepth * kPieceBytes, bars + warp * kDepth, lane);
  uint32_t taken = 0;
  if (parts > 1) cg::this_cluster().barrier_arrive();
  bool entered = parts == 1;

  const float s = a.opt.scale, c = s * kLog2e, kd = a.opt.distill_weight;
  // What a row needs beside its logits is asked for one row ahead: the teacher's alternatives, weight and target.
  int t = -1;
  float weight = 1.f;
  auto fetch = [&](int64_t r, int& t, float& weight) {
    if (r >= a.rows) return;
    if (lead)
      for (int j = lane; j < k; j += 32) {
        copy4(&sh.next_id[j], a.ids + r * k + j);
        copy4(&sh.next_val[j], a.values + r * k + j);
      }
    if (a.targets && a.opt.target_weight != 0.f) t = a.targets[r];
    if (a.row_weight) weight = a.row_weight[r];
  };
  fetch(row0, t, weight);
  for (int64_t r = row0; r < a.rows; r += step) {
    const T* x = static_cast<const T*>(a.logits) + r * a.stride;
    T* d = a.d ? static_cast<T*>(a.d) + r * a.d_stride : nullptr;
    const Span<T> sp(x, V, part, parts);
    const int single = (NW == 1 || tid < 32) ? sp.single(V, part, parts, tid) : -1;
    const float xs = single >= 0 ? Elt<T>::get(x + single) : -INFINITY;
    if (t >= V) t = -1;
    const float ce = t >= 0 ? a.opt.target_weight : 0.f;
    int t_n = -1;
    float weight_n = 1.f;
    if (lead) {
      // the alternatives, and the student's logits at them and at the target
      copies_done();  // (each lane's own)
      float mx = -INFINITY;
      for (int j = lane; j < k; j += 32) {
        int id = sh.next_id[j];
        if (id >= V) id = -1;
        if (id >= 0) sh.x[j] = Elt<T>::get(x + id);
        const float v = id >= 0 ? sh.next_val[j] * a.opt.teacher_scale : -INFINITY;
        sh.id[j] = id;
        sh.q[j] = v;
        mx = fmaxf(mx, v);
      }
      // normalised: q = e^(y - mx) / n and ln q = y - mx - ln n; as given: mx = ln n = 0, n = 1
      mx = a.opt.normalize ? max_warp(mx) : 0.f;
      if (mx == -INFINITY) mx = 0.f;
      float n = 0.f, dot = 0.f;
      for (int j = lane; j < k; j += 32) {
        const float y = sh.q[j] - mx, e = sh.id[j] >= 0 ? expf(y) : 0.f;
        n += e;
        dot += e == 0.f ? 0.f : e * y;
        sh.q[j] = e;
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        n += __shfl_xor_sync(0xffffffffu, n, o);
        dot += __shfl_xor_sync(0xffffffffu, dot, o);
      }
      if (a.opt.normalize) {
        const float inv = n == 0.f ? 0.f : __fdividef(1.f, n);
        for (int j = lane; j < k; j += 32) sh.q[j] *= inv;
        dot = n == 0.f ? 0.f : fmaf(dot, inv, -logf(n));
        n *= inv;
      }
      if (lane < 4) {  // the entry after the last is the hard target; then none, up to a multiple of four
        sh.id[k + lane] = lane == 0 ? t : -1;
        sh.q[k + lane] = 0.f;
      }
      if (lane == 0) {
        if (t >= 0) sh.x[k] = Elt<T>::get(x + t);
        sh.sum = n;
        sh.ent = dot;
      }
    }
    fetch(r + step, t_n, weight_n);

    Sums2 st = distill_sums<SECOND>(feed, taken, sp, xs, single >= 0, c, lane);
    st.join_warp(c);
    if constexpr (NW > 1) {
      if (lane == 0) sh.red[warp] = st.pack();
      __syncthreads();
      st = lane < NW ? Sums2(sh.red[lane]) : Sums2();
      st.join_warp(c);
      if (parts > 1) {
        if (!entered) { cg::this_cluster().barrier_wait(); entered = true; }  // the other blocks run: their memory may be written
        if (tid < parts) *cg::this_cluster().map_shared_rank(&sh.part[part], tid) = st.pack();
        cg::this_cluster().sync();  // (also: every block has read its logits at the alternatives)
        st = lane < parts ? Sums2(sh.part[lane]) : Sums2();
        st.join_warp(c);
      }
    } else {
      __syncwarp();
    }
    // a row without weight, or with nothing left, has no part in the loss, whatever else it holds
    const bool none = weight == 0.f || st.s == 0.f;
    if (SECOND == kNone) st.h = st.s;
    if (part == 0 && lead) {
      const float ln_s = logf(st.s), ln_h = SECOND == kNone ? ln_s : logf(st.h);
      float loss = 0.f;
      for (int j = lane; j <= k; j += 32) {
        const bool hard = j == k;
        if (sh.id[j] < 0 || (hard ? false : sh.q[j] == 0.f || kd == 0.f)) continue;
        const float w = hard ? ce : kd * sh.q[j];
        loss -= w * fmaf(sh.x[j] - st.m, hard && SECOND != kNone ? 1.f : s, -(hard ? ln_h : ln_s));
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) loss += __shfl_xor_sync(0xffffffffu, loss, o);
      if (lane == 0) a.loss_rows[r] = none ? 0.f : weight * fmaf(kd, sh.ent, loss);
    }
    const float gs = a.opt.grad_scale * weight, wq = gs * kd * s, wc = gs * ce;
    if (d) {
      Exponent<SECOND> ex;
      ex.at(st.m, c);
      float f, f1;
      ex.settle(f, f1);
      const float ff = (SECOND == kNone ? fmaf(wq, sh.sum, wc) : wq * sh.sum) * __fdividef(f, st.s), fc = SECOND == kNone ? 0.f : wc * __fdividef(f1, st.h);
      distill_gradient<SECOND>(feed, taken, sp, x, d, none, ex, ff, fc, lane);
      if (single >= 0) Elt<T>::put(d + single, none ? 0.f : ex.grad(xs, ff, fc));
      team_sync<NW>();  // the elements below are written a second time, by other threads
      for (int j = tid; j <= k && !none; j += NW * 32) {
        const int i = sh.id[j];
        if (i < 0 || !sp.has(i, part, parts)) continue;
        float q = 0.f;
        for (int l = 0; l < k; l += 4) {  // (the target's q is 0)
          const int4 ids = *reinterpret_cast<const int4*>(&sh.id[l]);
          const float4 qs = *reinterpret_cast<const float4*>(&sh.q[l]);
          q += (ids.x == i ? qs.x : 0.f) + (ids.y == i ? qs.y : 0.f) + (ids.z == i ? qs.z : 0.f) + (ids.w == i ? qs.w : 0.f);
        }
        Elt<T>::put(d + i, ex.grad(sh.x[j], ff, fc) - wq * q - (i == t ? wc : 0.f));
      }
    }
    t = t_n;
    weight = weight_n;
    team_sync<NW>();
    if (parts > 1) cg::this_cluster().sync();  // this row's sums are read: the next row's may come
  }
  if (!entered) cg::this_cluster().barrier_wait();
}

// *out = scale * sum(v), summed in 64 bits in a fixed order (one block).
__global__ void __launch_bounds__(1024) scaled_sum_kernel(const float* __restrict__ v, int n, float scale,
                                                          float* __restrict__ out) {
  __shared__ double red[32];
  double s = 0.0;
  follows();
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
// Warps to a row: as many as let all rows run at once (24 warps on an SM), if each has a piece of its own; with
// more rows than that one warp where a row is short, four where it is 16 pieces or longer, whose rows would leave
// SMs idle at the end.  Measured, log probabilities: 2400 x 6400 17 us with one, 22 / 25 / 41 us with 2 / 4 / 8;
// 600 x 1100 9 us with one, 27 us with two, of which the second has nine vectors;
// 1021 x 50001 35 us with two, 39 / 41 us with 4 / 8; 600 x 50001 25 us with four, 29 us with 2 or 8; 2048 x 32000
// 45 us with four, 56 us with one.  Distillation: 32768 x 6400 201 us with one, 280 / 303 us with 2 / 4; 2048 x
// 32000 66 us with four, 84 / 74 us with 1 / 8; 500 x 50001 39 us with four, 54 / 42 us with 2 / 8.
int team_warps(int rows, int pieces) {
  const int64_t room = 24 * (int64_t)sm_count_current();
  if (rows > room / 2) return pieces >= 16 ? 4 : 1;
  int nw = 1;
  while (nw < 8 && (int64_t)rows * 2 * nw <= room && pieces > 2 * nw) nw *= 2;  // (a whole piece for each)
  return nw;
}
// Blocks of eight warps to a row: more while all still run at once and each warp has a piece.  Log probabilities:
// 64 x 131072 21 / 15 / 13 / 22 us with 1 / 2 / 4 / 8; 1 x 131072 19 / 15 / 13 / 11 us.  Distillation: 64 x 262139
// fp32 82 / 54 / 42 / 50 us; 100 x 100003 31 / 27 / 24 / 35 us.
int team_parts(int rows, int pieces) {
  int p = 1;
  while (p < kMaxParts && (int64_t)rows * 2 * p * 8 <= 24 * (int64_t)sm_count_current() && pieces >= 14 * p) p *= 2;
  return p;
}

constexpr size_t kMaxDynamic = 200 * 1024;
// Lets a kernel have that much dynamic shared memory, once per device.
template <typename K> cudaError_t allow_dynamic(K kern, std::atomic<uint64_t>& done) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess || (dev < 64 && (done.load() >> dev & 1))) return e;
  e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kMaxDynamic);
  if (e == cudaSuccess && dev < 64) done.fetch_or(1ull << dev);
  return e;
}
template <typename K, typename... A>
zl_status launch(const char* what, K kern, int64_t blocks, int threads, int parts, size_t smem, zl_stream s, A... args) {
  if (blocks > 0x7fffffff) return set_error(ZL_EUNSUPPORTED, "%s: too many rows", what);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)blocks, 1, 1);
  cfg.blockDim = dim3(threads, 1, 1);
  cfg.dynamicSmemBytes = smem;
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
  return launched(what, cudaLaunchKernelEx(&cfg, kern, args...));
}
// Teams of NW warps to a row, or clusters of `parts` blocks; single warps go on to further rows, no more blocks of
// them than run at once.
template <typename T, int NW, int TEAMS, bool LOOSE = false>
zl_status launch_rows(const char* what, int rows, int parts, zl_stream s, const LogprobArgs& a) {
  static std::atomic<uint64_t> done{0};
  const auto kern = logprobs_kernel<T, NW, TEAMS, LOOSE>;
  const size_t smem = logprobs_smem<T, NW, TEAMS>(a);
  const cudaError_t e = allow_dynamic(kern, done);
  if (e != cudaSuccess) return launched(what, e);
  int64_t blocks = ((int64_t)rows + TEAMS - 1) / TEAMS * parts;
  if (NW == 1) {
    const int64_t per_sm = std::min<int64_t>(kRowBlocks, (227 * 1024) / (smem + sizeof(TopShared<NW>) * TEAMS + 2048));
    blocks = std::min(blocks, per_sm * sm_count_current());
  }
  return launch(what, kern, blocks, NW * TEAMS * 32, parts, smem, s, a);
}

// Teams (or clusters) that run at once, each of which goes on to further rows.
template <typename T, int NW, int TEAMS, int SECOND> zl_status launch_distill(const char* what, zl_stream s, const DistillArgs& a) {
  static std::atomic<uint64_t> done{0};
  const auto kern = distill_kernel<T, NW, TEAMS, SECOND>;
  const size_t smem = (size_t)TEAMS * NW * kDepth * kPieceBytes;
  const cudaError_t e = allow_dynamic(kern, done);
  if (e != cudaSuccess) return launched(what, e);
  const int64_t rows = ((int64_t)a.rows + TEAMS - 1) / TEAMS;
  const int64_t room = std::max<int64_t>(1, 24 / (NW * TEAMS) * sm_count_current() / a.parts);
  return launch(what, kern, std::min(rows, room) * a.parts, NW * TEAMS * 32, a.parts, smem, s, a);
}
template <typename T, int SECOND> zl_status launch_distill(const char* what, int nw, zl_stream s, const DistillArgs& a) {
  return nw == 1 ? launch_distill<T, 1, 4, SECOND>(what, s, a) : nw == 2 ? launch_distill<T, 2, 1, SECOND>(what, s, a)
         : nw == 4 ? launch_distill<T, 4, 1, SECOND>(what, s, a) : launch_distill<T, 8, 1, SECOND>(what, s, a);
}

constexpr int kVocabMax = 1 << 30;  // (column arithmetic is 32-bit)
// Most logits of a row with alternatives: the maxima of kMaxParts parts beside the rings of eight warps.
template <typename T> constexpr int top_vocab() {
  constexpr int pieces = (int)((kMaxDynamic - 8 * kDepth * kPieceBytes) / (32 * sizeof(typename Maxima<T>::Store)));
  constexpr int vecs = kMaxParts * (pieces * kPieceVecs - 1) + kMaxParts - 1;
  return (vecs - 1) * Elt<T>::VEC + Elt<T>::VEC - 1;
}
static_assert(top_vocab<__nv_bfloat16>() == 5505015 && top_vocab<float>() == 1376251, "as the header says");
bool off_words(std::initializer_list<const void*> ps) {
  for (const void* p : ps)
    if (reinterpret_cast<uintptr_t>(p) & 3) return true;
  return false;
}
template <typename T> bool off_element(const void* p) { return (reinterpret_cast<uintptr_t>(p) % sizeof(T)) != 0; }

template <typename T>
zl_status check_rows(const char* what, const void* logits, int64_t stride, int rows, int vocab, float scale) {
  if (rows < 0 || vocab <= 0) return set_error(ZL_EINVAL, "%s: sizes must be positive", what);
  if (vocab > kVocabMax) return set_error(ZL_EUNSUPPORTED, "%s: at most 2^30 logits to a row", what);
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
  if (off_words({targets, logp, entropy, lse, top_logp, top_ids}))
    return set_error(ZL_EINVAL, "token_logprobs: a target or output array off a 4-byte boundary");
  // (the vectors' maxima of a row fit into the shared memory of a cluster)
  if (top_k > 0 && vocab > top_vocab<T>())
    return set_error(ZL_EUNSUPPORTED, "token_logprobs: top alternatives of at most %d logits", top_vocab<T>());
  if (rows == 0) return ZL_OK;
  LogprobArgs a{logits, stride, targets, rows, vocab, top_k, 1, 0, scale, logp, entropy, lse, top_logp, top_ids};
  const int vecs = vocab / Elt<T>::VEC + 1;
  a.pieces = (vecs + kPieceVecs - 1) / kPieceVecs;
  int nw = team_warps(rows, a.pieces);
  // the vectors' maxima of a row fit beside the rings, and a single warp has 128 groups (or the row is short)
  while (nw < 8 && (vecs > 4096 * nw || (nw == 1 && top_k > 96 && vocab > kShortRow))) nw *= 2;
  const bool loose = vocab <= kShortRow && (3 * (vocab / Elt<T>::VEC) < 4 * top_k || top_k > 96);
  if (nw == 1 && loose) return launch_rows<T, 1, 4, true>("token_logprobs", rows, 1, s, a);
  if (nw == 1) return launch_rows<T, 1, 4>("token_logprobs", rows, 1, s, a);
  if (nw == 2) return launch_rows<T, 2, 1>("token_logprobs", rows, 1, s, a);
  if (nw == 4) return launch_rows<T, 4, 1>("token_logprobs", rows, 1, s, a);
  a.parts = team_parts(rows, a.pieces);
  for (;; a.parts *= 2) {  // (ends at kMaxParts at the latest)
    a.pieces = (vecs / a.parts + 1 + kPieceVecs - 1) / kPieceVecs;
    if (logprobs_smem<T, 8, 1>(a) <= kMaxDynamic) break;
  }
  return launch_rows<T, 8, 1>("token_logprobs", rows, a.parts, s, a);
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
  if (off_words({targets, lse, entropy, g_logp, g_entropy})) return set_error(ZL_EINVAL, "%s: an input array off a 4-byte boundary", what);
  if (g_logp && !targets) return set_error(ZL_EINVAL, "%s: a gradient of log probabilities needs targets", what);
  if (g_entropy && !entropy) return set_error(ZL_EINVAL, "%s: a gradient of entropies needs the entropies", what);
  if ((const void*)d == (const void*)logits && d_stride != stride)
    return set_error(ZL_EINVAL, "%s: a gradient in the logits' place has their row stride", what);
  // (128 threads to a block: 32768 x 6400 bf16 130 us in a burst, 134 / 241 us with 256 / 512; 839 MB, 128 us at the copy
  // rate; 138 us over seconds)
  constexpr int NT = 128;
  constexpr int per = NT * Elt<T>::VEC * 4;
  const int slices = (int)(((int64_t)vocab + per - 1) / per);
  LogprobBwdArgs a{logits, stride, targets, lse, entropy, g_logp, g_entropy, rows, vocab, scale, d, d_stride};
  return launch(what, logprobs_bwd_kernel<T, NT>, (int64_t)rows * slices, NT, 1, 0, s, a, slices);
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
  if (off_words({ids, values, targets, row_weight, loss_rows, loss_out}))
    return set_error(ZL_EINVAL, "%s: an array of 4-byte values off a 4-byte boundary", what);
  if (rows > 0) {
    // (without weight the teacher's record is not read: whatever it holds, 0 times it is 0)
    const int used = opt->distill_weight == 0.f ? 0 : k;
    DistillArgs a{logits, stride, ids, values, targets, row_weight, rows, vocab, used, 1, *opt, d, d_stride, loss_rows};
    const int pieces = (vocab / Elt<T>::VEC + kPieceVecs) / kPieceVecs;
    const int nw = team_warps(rows, pieces);
    if (nw == 8) a.parts = team_parts(rows, pieces);
    const float sc = opt->scale;
    const Second second = opt->target_weight == 0.f || sc == 1.f ? kNone : sc == 0.5f ? kSquare : sc == 0.25f ? kFourth : kOwn;
    st = second == kNone ? launch_distill<T, kNone>(what, nw, s, a) : second == kSquare ? launch_distill<T, kSquare>(what, nw, s, a)
         : second == kFourth ? launch_distill<T, kFourth>(what, nw, s, a) : launch_distill<T, kOwn>(what, nw, s, a);
    if (st != ZL_OK) return st;
  }
  if (!loss_out) return ZL_OK;
  return launch_after(what, scaled_sum_kernel, 1, 1024, (cudaStream_t)s, (const float*)loss_rows, rows, opt->grad_scale, loss_out);
}
}  // namespace

int logprobs_dev_error_read_and_clear() {
  int v = 0;
  cudaMemcpyFromSymbol(&v, zl_dev_error, sizeof(int));
  if (v) {
    int z = 0;
    cudaMemcpyToSymbol(zl_dev_error, &z, sizeof(int));
  }
  return v;
}

namespace {
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
