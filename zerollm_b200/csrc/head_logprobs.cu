// head_logprobs.cu -- log probabilities of given tokens straight from hidden states and the output head's
// weight: logits = hidden weight^T stay in tensor memory, where each tile's epilogue folds them into the
// running softmax statistics of its rows.  Neither logits nor probabilities reach device memory (the
// reference's head writes them, zerollm.cpp:150-195).
//
// A CTA pair (cta_group::2) computes tiles of 256 rows x 256 vocabulary entries as the pair GEMM does
// (gemm.cu): each CTA loads its 128 rows of hidden and its half of the weight tile by TMA, the even CTA
// issues the products for both, each CTA's eight epilogue warps read their 128 x 256 half of the accumulator
// (two in tensor memory, so products and epilogue overlap).  A thread keeps (m, S0, S1, target logit) of one
// row and half of the tile's columns over the consecutive tiles of a work segment and writes them once, as a
// partial; a second small kernel joins a row's partials in a fixed order.
//
// Measured (2 T V d flops at the measured 1.63 PFLOP/s burst / 1.39 PFLOP/s sustained rates): 16384 x 2048 x 32000
// 1.27 to 1.38 ms in a burst of 30 passes, 1.48 to 1.54 ms over seconds (floor 1.32 / 1.54 ms): the tensor cores bind.
// 32768 x 512 x 6400 154 to 158 / 177 to 184 us (floor 133 / 154 us); without the epilogue's arithmetic 136 us, so there
// the epilogue's exponentials cost the rest; sixteen epilogue warps in place of eight gained 1 % there and lost 4 % on the
// long reduction.  With the weight and hidden both streamed and a row tile's vocabulary walked by one pair the same took
// 2.60 ms and 209 us.
#include <algorithm>
#include <atomic>
#include <cstdio>

#include "logprobs.cuh"

namespace zl {
int sm_count_current();  // gemm.cu
bool make_tma_map(CUtensorMap* map, const void* ptr, bool is_f32, uint64_t inner, uint64_t rows, uint32_t box_inner,
                  uint32_t box_rows, int swizzle_bytes, uint64_t row_stride);


namespace {
constexpr int BM = 128, BN = 256, BK = 64;   // rows of a CTA, vocabulary entries of a tile, reduction block
constexpr int kEpiWarps = 8, kShares = kEpiWarps / 4;  // epilogue warps; those that share a row, each its columns of a tile
constexpr int kThreads = 64 + kEpiWarps * 32;
constexpr int kTileBytes = BM * BK * 2;      // a CTA's share of hidden, and of the weight, in one reduction block
// A short reduction (up to kHeld blocks) keeps the row tile of hidden in shared memory from one vocabulary tile to the
// next; its ring holds weight blocks.  A longer one streams both through a ring of pairs.
constexpr int kHeld = 8;
// Most reduction blocks that the tensor core sums at once; a longer reduction is cut into chunks alike, added in fp32 by
// the epilogue.  Each step of 16 products is cut to fp32 toward zero, so a sum comes out too small in magnitude by 0.1 to
// 0.9 of 2^-24 for every step behind it, which like a temperature moves a row's entropy (of 16384 x 2048 x 32000,
// undivided: 1.7e-6 of it).  Chunks of up to 48 steps bound that for any length (6e-7 there).  Reading an accumulator takes
// 1800 cycles, about what tensor memory gives beside the products, and a tile's statistics 3200; the products of two chunks
// have to last as long: undivided, or in three chunks of 11, 1.31 ms there, in four of 8 1.36 ms, in seven of 5 a third
// more; 8192 x 1024 x 16000 171 us undivided, 176 us in two chunks.
constexpr int kChunk = 12;
static_assert(kHeld <= kChunk, "a reduction that is held is one chunk");
template <bool HELD> struct Smem {
  static constexpr int STAGES = HELD ? 5 : 6;
  static constexpr int STAGE_BYTES = HELD ? kTileBytes : 2 * kTileBytes;
  static constexpr int RING = HELD ? kHeld * kTileBytes : 0;  // offset of the ring
  static constexpr int BARS = RING + STAGES * STAGE_BYTES;
  static constexpr int TOTAL = BARS + 512 + 1024;  // barriers, alignment slack
};

int pair_slots();  // CTA pairs that the current device runs at once

// Work: (row tile, vocabulary tile) steps in segments of one row tile and some consecutive vocabulary tiles; each
// segment leaves one partial per row.
//  * group = 0 (the weight fits into L2): steps are numbered row tile by row tile and pair p takes the steps
//    [p per, (p + 1) per), the same number each; a row tile's steps fall to the pairs first .. last, slot p - first.
//  * group > 0 (it does not): segments of `group` vocabulary tiles, row tiles running fastest, pair p takes every
//    pairs-th.  All pairs work on the same few vocabulary tiles at a time, so the weight comes from memory once, not
//    once per row tile (16384 x 2048 x 32000: see below).  Slot: the group.
struct Plan {
  int row_tiles, n_tiles, pairs, slots, group;
  int64_t steps, per;
};
Plan make_plan(int rows, int dim, int vocab) {
  Plan p;
  p.row_tiles = (rows + 2 * BM - 1) / (2 * BM);
  p.n_tiles = (vocab + BN - 1) / BN;
  p.steps = (int64_t)p.row_tiles * p.n_tiles;
  p.pairs = (int)std::min<int64_t>(p.steps, pair_slots());
  p.per = (p.steps + p.pairs - 1) / p.pairs;
  p.group = 0;
  if ((int64_t)vocab * dim * 2 > (int64_t)40 << 20 && p.row_tiles > 1) {
    // rounds of segments, a segment's steps and a tenth for its partials
    double best = 1e30;
    for (int g = 1; g <= std::min(p.n_tiles, 16); ++g) {
      const int64_t units = (int64_t)p.row_tiles * ((p.n_tiles + g - 1) / g);
      const double t = (double)((units + p.pairs - 1) / p.pairs) * (g + 0.1);
      if (t < best) { best = t; p.group = g; }
    }
  }
  p.slots = p.group ? (p.n_tiles + p.group - 1) / p.group : (int)std::min<int64_t>(p.pairs, (p.n_tiles - 1) / p.per + 2);
  return p;
}

struct HeadArgs {
  const int32_t* targets;
  int rows, vocab, k_blocks, row_tiles, n_tiles, slots, group;
  int64_t steps, per;
  float c;  // scale * log2(e)
  int chunk;  // reduction blocks of a chunk (at most kChunk, alike)
  int few;    // few rows: partials of a row, one of each block
  float4* partials;  // [row][slot][share] (m, S0, S1, target logit)
};

// The segments of a pair, one after the other.
struct Segments {
  int64_t at, end;
  int pair, pairs;
  int rt, nt0, nt1, slot;
  __device__ __forceinline__ Segments(const HeadArgs& a, int p, int n) : pair(p), pairs(n) {
    at = a.group ? p : p * a.per;
    end = a.group ? (int64_t)a.row_tiles * a.slots : min(a.steps, (p + 1) * a.per);
  }
  __device__ __forceinline__ bool next(const HeadArgs& a) {
    if (at >= end) return false;
    if (a.group) {
      rt = (int)(at % a.row_tiles);
      slot = (int)(at / a.row_tiles);
      nt0 = slot * a.group;
      nt1 = min(a.n_tiles, nt0 + a.group);
      at += pairs;
    } else {
      rt = (int)(at / a.n_tiles);
      slot = pair - (int)((int64_t)rt * a.n_tiles / a.per);
      nt0 = (int)(at % a.n_tiles);
      nt1 = (int)min((int64_t)a.n_tiles, nt0 + (end - at));
      at += nt1 - nt0;
    }
    return true;
  }
};

template <bool HELD>
__global__ void __launch_bounds__(kThreads, 1)
    head_logprobs_kernel(const __grid_constant__ CUtensorMap tmH, const __grid_constant__ CUtensorMap tmW,
                         const HeadArgs a) {
  using L = Smem<HELD>;
  constexpr int STAGES = L::STAGES;
  constexpr uint32_t IDESC = make_idesc(1, 2 * BM, BN, 0, 0);
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  uint8_t* smem = smem_raw + (((raw + 1023u) & ~1023u) - raw);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::BARS);
  uint64_t* empty = full + STAGES;
  uint64_t* acc_full = empty + STAGES;
  uint64_t* acc_empty = acc_full + 2;
  uint64_t* h_full = acc_empty + 2;  // [kHeld] the held blocks of hidden
  uint64_t* h_empty = h_full + kHeld;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(h_empty + kHeld);
  static_assert((2 * STAGES + 4 + 2 * kHeld + 1) * 8 <= 512, "barrier area");

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;
  Segments seg(a, (int)(blockIdx.x >> 1), (int)(gridDim.x >> 1));

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
    for (int b = 0; b < 2; ++b) { mbar_init(&acc_full[b], 1); mbar_init(&acc_empty[b], 2 * kEpiWarps * 32); }
    for (int i = 0; i < kHeld; ++i) { mbar_init(&h_full[i], 1); mbar_init(&h_empty[i], 1); }
    fence_mbar_init();
    tma_prefetch_desc(&tmH);
    tma_prefetch_desc(&tmW);
  }
  if (warp == 1) {
    tmem_alloc_pair(tmem_holder, 2 * BN);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  __syncwarp();
  cluster_sync_all();  // barriers of both CTAs initialised, tensor memory allocated in both
  tc_fence_after();
  const uint32_t tmem_base = *tmem_holder;

  if (warp == 0) {
    // ------------------------------------------------ TMA producer (both CTAs)
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0, h_phase = 0;
      bool ok = true;
      while (ok && seg.next(a)) {
        const int m0 = seg.rt * (2 * BM) + (int)rank * BM;
        for (int nt = seg.nt0; nt < seg.nt1 && ok; ++nt) {
          const int n0 = nt * BN + (int)rank * (BN / 2);
          for (int kb = 0; kb < a.k_blocks; ++kb) {
            if (HELD && nt == seg.nt0) {
              // block kb of the new row tile, as soon as the last product with the old one is done
              if (!bounded_wait(&h_empty[kb], h_phase ^ 1u, DEV_TIMEOUT_EMPTY)) { ok = false; break; }
              if (leader) mbar_arrive_expect_tx(&h_full[kb], 2 * kTileBytes);
              tma_load_2d_pair(smem + kb * kTileBytes, &tmH, mapa_shared(smem_u32(&h_full[kb]), 0), kb * BK, m0);
            }
            if (!bounded_wait(&empty[stage], phase ^ 1u, DEV_TIMEOUT_EMPTY)) { ok = false; break; }
            uint8_t* st = smem + L::RING + stage * L::STAGE_BYTES;
            const uint32_t bar = mapa_shared(smem_u32(&full[stage]), 0);  // the even CTA's barrier
            if (leader) mbar_arrive_expect_tx(&full[stage], 2 * L::STAGE_BYTES);
            if (!HELD) tma_load_2d_pair(st + kTileBytes, &tmH, bar, kb * BK, m0);
            tma_load_2d_pair(st, &tmW, bar, kb * BK, n0);
            if (++stage == STAGES) { stage = 0; phase ^= 1u; }
          }
        }
        h_phase ^= 1u;
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------ MMA issuer (even CTA only)
    if (leader) {
      int stage = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0, h_phase = 0;
      bool ok = true;
      while (ok && seg.next(a)) {
        for (int nt = seg.nt0; nt < seg.nt1 && ok; ++nt) {
          for (int k0 = 0; k0 < a.k_blocks && ok; k0 += a.chunk) {
            // both CTAs' epilogues have drained accumulator `acc`
            if (!__all_sync(0xffffffffu, bounded_wait_cluster(&acc_empty[acc], acc_phase ^ 1u, DEV_TIMEOUT_ACC))) { ok = false; break; }
            tc_fence_after();
            const uint32_t d_tmem = tmem_base + (uint32_t)(acc * BN);
            const int k1 = HELD ? a.k_blocks : min(a.k_blocks, k0 + a.chunk);
            for (int kb = k0; kb < k1; ++kb) {
              if (HELD && nt == seg.nt0 && !bounded_wait_warp(&h_full[kb], h_phase, DEV_TIMEOUT_FULL)) { ok = false; break; }
              if (!bounded_wait_warp(&full[stage], phase, DEV_TIMEOUT_FULL)) { ok = false; break; }
              tc_fence_after();
              const uint32_t w_base = smem_u32(smem + L::RING + stage * L::STAGE_BYTES);
              const uint32_t h_base = HELD ? smem_u32(smem + kb * kTileBytes) : w_base + kTileBytes;
#pragma unroll
              for (int k = 0; k < BK / 16; ++k)
                umma_f16_pair_w(d_tmem, smem_desc_sw128(h_base + k * 32, 16, 1024), smem_desc_sw128(w_base + k * 32, 16, 1024),
                                IDESC, (kb > k0 || k > 0) ? 1u : 0u);
              umma_commit_pair_w(&empty[stage], 0x3);
              if (HELD && nt + 1 == seg.nt1) umma_commit_pair_w(&h_empty[kb], 0x3);
              if (++stage == STAGES) { stage = 0; phase ^= 1u; }
            }
            if (!ok) break;
            umma_commit_pair_w(&acc_full[acc], 0x3);
            if (++acc == 2) { acc = 0; acc_phase ^= 1u; }
          }
        }
        h_phase ^= 1u;
      }
    }
  } else {
    // ------------------------------------------------ epilogue (both CTAs, own half of the rows)
    const int quarter = warp & 3, share = (warp - 2) >> 2;
    const uint32_t acc_empty_leader[2] = {mapa_shared(smem_u32(&acc_empty[0]), 0), mapa_shared(smem_u32(&acc_empty[1]), 0)};
    int acc = 0;
    uint32_t acc_phase = 0;
    bool ok = true;
    while (ok && seg.next(a)) {
      const int row = seg.rt * (2 * BM) + (int)rank * BM + quarter * 32 + lane;
      const int t = (a.targets && row < a.rows) ? a.targets[row] : -1;
      Running run;
      float xt = 0.f;
      // 32 columns of the tile, from column n of the vocabulary on
      auto fold = [&](float (&v)[32], int n) {
        if (n >= a.vocab) return;
        if (n + 32 > a.vocab) {  // the last tile: entries past the vocabulary have p = 0
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = n + j < a.vocab ? v[j] : -INFINITY;
        }
        if (t >= n && t < n + 32 && t < a.vocab) {
#pragma unroll
          for (int j = 0; j < 32; ++j) xt = t == n + j ? v[j] : xt;
        }
        run.add_near(v, a.c);
      };
      auto drained = [&] {
        tc_fence_before();
        mbar_arrive_cluster(acc_empty_leader[acc]);
        if (++acc == 2) { acc = 0; acc_phase ^= 1u; }
      };
      constexpr int COLS = BN / kShares;  // this warp's columns of a tile
      for (int nt = seg.nt0; nt < seg.nt1 && ok; ++nt) {
        const uint32_t t_row = tmem_base + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(share * COLS);
        const int n0 = nt * BN + share * COLS;
        if constexpr (HELD) {  // one chunk: from tensor memory
          if (!bounded_wait_warp(&acc_full[acc], acc_phase, DEV_TIMEOUT_ACC)) { ok = false; break; }
          tc_fence_after();
#pragma unroll 1
          for (int c = 0; c < COLS && n0 + c < a.vocab; c += 32) {
            uint32_t u[32];
            tmem_ld32(t_row + (uint32_t)(acc * BN + c), u);
            tmem_ld_wait();
            float v[32];
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(u[j]);
            fold(v, n0 + c);
          }
          drained();
        } else {  // the sum of the chunks in registers; the last accumulator is free before its logits are folded
          uint32_t v[COLS / 8][8];  // (the first chunk comes straight into them)
          if (!bounded_wait_warp(&acc_full[acc], acc_phase, DEV_TIMEOUT_ACC)) { ok = false; break; }
          tc_fence_after();
#pragma unroll
          for (int c = 0; c < COLS / 8; ++c) tmem_ld8(t_row + (uint32_t)(acc * BN + c * 8), v[c]);
          tmem_ld_wait();
          drained();
          for (int kb = a.chunk; kb < a.k_blocks; kb += a.chunk) {
            if (!bounded_wait_warp(&acc_full[acc], acc_phase, DEV_TIMEOUT_ACC)) { ok = false; break; }
            tc_fence_after();
#pragma unroll
            for (int c = 0; c < COLS / 8; c += 2) {
              uint32_t u[2][8];
#pragma unroll
              for (int p = 0; p < 2; ++p) tmem_ld8(t_row + (uint32_t)(acc * BN + (c + p) * 8), u[p]);
              tmem_ld_wait();
#pragma unroll
              for (int p = 0; p < 2; ++p)
#pragma unroll
                for (int j = 0; j < 8; ++j) v[c + p][j] = __float_as_uint(__uint_as_float(v[c + p][j]) + __uint_as_float(u[p][j]));
            }
            drained();
          }
          if (!ok) break;
#pragma unroll
          for (int c = 0; c < COLS / 32; ++c) {
            float x[32];
#pragma unroll
            for (int j = 0; j < 32; ++j) x[j] = __uint_as_float(v[(c * 32 + j) / 8][j % 8]);
            fold(x, n0 + c * 32);
          }
        }
      }
      if (ok && row < a.rows) {  // this pair's partial of the row
        const Stats st = run.sums(a.c);
        a.partials[((int64_t)row * a.slots + seg.slot) * kShares + share] = make_float4(st.m, st.s0, st.s1, xt);
      }
    }
  }
  // The even CTA's products read both CTAs' shared memory and write both tensor memories: neither CTA may
  // leave (or free its tensor memory) before both are done.
  tc_fence_before();
  __syncwarp();
  cluster_sync_all();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, 2 * BN);
  }
}

cudaLaunchConfig_t pair_config(int pairs, size_t smem, cudaStream_t st, cudaLaunchAttribute* attr) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(2 * pairs, 1, 1);
  cfg.blockDim = dim3(kThreads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  attr->id = cudaLaunchAttributeClusterDimension;
  attr->val.clusterDim.x = 2;
  attr->val.clusterDim.y = 1;
  attr->val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cfg;
}

int pair_slots() {
  static std::atomic<int> found[64];
  const int sms = std::max(1, sm_count_current() / 2);
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) {
    cudaGetLastError();
    return sms;  // no device: the plan of a full one
  }
  int n = found[dev].load();
  if (n == 0) {
    cudaLaunchAttribute attr;
    cudaLaunchConfig_t cfg = pair_config(sms, Smem<true>::TOTAL, nullptr, &attr);
    if (cudaFuncSetAttribute(head_logprobs_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, Smem<true>::TOTAL) != cudaSuccess ||
        cudaFuncSetAttribute(head_logprobs_kernel<false>, cudaFuncAttributeMaxDynamicSharedMemorySize, Smem<false>::TOTAL) != cudaSuccess ||
        cudaOccupancyMaxActiveClusters(&n, head_logprobs_kernel<true>, &cfg) != cudaSuccess || n <= 0) {
      cudaGetLastError();
      return sms;
    }
    n = std::min(n, sms);
    found[dev].store(n);
  }
  return n;
}

// ------------------------------------------------------------------ few rows
// Up to 8 rows: the weight is read once, at the rate of device memory, and tensor-core tiles of 256 rows would be
// empty.  Every warp takes tiles of 16 vocabulary entries: mma.m16n8k16 with the weight's rows as A, straight from
// device memory to registers, and the rows of hidden as B, from shared memory.  The order of the reduction index is
// free as long as both operands use the same one, so a lane's 16-byte load of 8 consecutive elements of one weight row
// serves as its A registers of two products.  A lane has the logits of 2 entries x 2 rows and folds them into the
// statistics of these rows; a block leaves one partial per row.  Measured: one row of 2048 x 32000 28.7 us with the
// join (131 MB, 20 us at the copy rate), of 2048 x 128000 84 to 87 us (92 to 95 % of it); nine rows, on the tensor-core tiles, 39 us.  Eight
// loads of a weight row in flight per lane; four of them with 3 or 4 blocks an SM took 34 / 37 us.
constexpr int kFewRows = 8, kFewWarps = 8, kFewBlocks = 2, kFewDim = 8192;  // (hidden: up to 128 KB of shared memory)

__device__ __forceinline__ void mma_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__global__ void __launch_bounds__(kFewWarps * 32, kFewBlocks)
    head_few_kernel(const __nv_bfloat16* __restrict__ hidden, const __nv_bfloat16* __restrict__ weight, int dim, const HeadArgs a) {
  extern __shared__ uint8_t smem_raw[];
  uint4* h = reinterpret_cast<uint4*>(smem_raw);  // [block of 32][row of 8][quad of 4]: 8 elements each, 0 past the ends
  __shared__ float4 part[kFewWarps][kFewRows];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, q = lane & 3;
  const int blocks = (dim + 31) / 32, vecs = dim / 8;
  for (int i = threadIdx.x; i < blocks * 32; i += kFewWarps * 32) {
    const int r = (i >> 2) & 7, v = (i >> 5) * 4 + (i & 3);
    h[i] = r < a.rows && v < vecs ? __ldg(reinterpret_cast<const uint4*>(hidden + (int64_t)r * dim) + v) : make_uint4(0, 0, 0, 0);
  }
  int t[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) t[i] = a.targets && 2 * q + i < a.rows ? a.targets[2 * q + i] : -1;
  __syncthreads();
  Running run[2];
  float xt[2] = {0.f, 0.f};
  let_follow();
  const int tiles = (a.vocab + 15) / 16, step = gridDim.x * kFewWarps;
  for (int tile = warp * gridDim.x + blockIdx.x; tile < tiles; tile += step) {  // (spread over all SMs)
    const int n0 = tile * 16 + g, n1 = n0 + 8;  // this lane's weight rows (the last one again past the end)
    const uint4* w0 = reinterpret_cast<const uint4*>(weight + (int64_t)min(n0, a.vocab - 1) * dim) + q;
    const uint4* w1 = reinterpret_cast<const uint4*>(weight + (int64_t)min(n1, a.vocab - 1) * dim) + q;
    float d[4][4] = {}, sum[4] = {};  // (sums of a few products each, joined in fp32: few steps that cut one)
    auto join = [&] {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        sum[j] += (d[0][j] + d[1][j]) + (d[2][j] + d[3][j]);
        d[0][j] = d[1][j] = d[2][j] = d[3][j] = 0.f;
      }
    };
    auto product = [&](const uint4& u0, const uint4& u1, int b, int half) {
      const uint4 x = h[(b * 8 + g) * 4 + q];
      mma_16816(d[half], u0.x, u1.x, u0.y, u1.y, x.x, x.y);
      mma_16816(d[half + 1], u0.z, u1.z, u0.w, u1.w, x.z, x.w);
    };
    constexpr int U = 8;
    const int whole = vecs / 4;  // blocks of 32 elements without an end inside
    int b = 0;
    for (; b + U <= whole; b += U) {
      uint4 u0[U], u1[U];
#pragma unroll
      for (int i = 0; i < U; ++i) {
        u0[i] = __ldg(w0 + (b + i) * 4);
        u1[i] = __ldg(w1 + (b + i) * 4);
      }
#pragma unroll
      for (int i = 0; i < U; ++i) product(u0[i], u1[i], b + i, i % 2 * 2);
      join();
    }
    for (; b < blocks; ++b) {
      const bool in = b * 4 + q < vecs;
      product(in ? __ldg(w0 + b * 4) : make_uint4(0, 0, 0, 0), in ? __ldg(w1 + b * 4) : make_uint4(0, 0, 0, 0), b, 0);
    }
    join();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float x0 = sum[i], x1 = sum[2 + i];
      if (n0 < a.vocab) {
        run[i].add_one(x0, a.c);
        if (t[i] == n0) xt[i] = x0;
      }
      if (n1 < a.vocab) {
        run[i].add_one(x1, a.c);
        if (t[i] == n1) xt[i] = x1;
      }
    }
  }
  // a row's statistics are in the eight lanes of one q
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    Stats s = run[i].sums(a.c);
    float M = s.m;  // (one common maximum, then one rescaling: each costs an exponential's rounding)
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
    s.rebase(M, a.c);
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) {
      s.s0 += __shfl_xor_sync(0xffffffffu, s.s0, o);
      s.s1 += __shfl_xor_sync(0xffffffffu, s.s1, o);
      xt[i] += __shfl_xor_sync(0xffffffffu, xt[i], o);
    }
    if (g == 0) part[warp][2 * q + i] = make_float4(s.m, s.s0, s.s1, xt[i]);
  }
  __syncthreads();
  if (threadIdx.x < kFewRows && threadIdx.x < a.rows) {
    Stats s;
    float x = 0.f;
    for (int w = 0; w < kFewWarps; ++w) s.m = fmaxf(s.m, part[w][threadIdx.x].x);
    for (int w = 0; w < kFewWarps; ++w) {
      const float4 p = part[w][threadIdx.x];
      Stats o(make_float3(p.x, p.y, p.z));
      o.rebase(s.m, a.c);
      s.s0 += o.s0;
      s.s1 += o.s1;
      x += p.w;
    }
    a.partials[(int64_t)threadIdx.x * gridDim.x + blockIdx.x] = make_float4(s.m, s.s0, s.s1, x);
  }
}
int few_blocks(int vocab) {
  return std::min((vocab + 16 * kFewWarps - 1) / (16 * kFewWarps), kFewBlocks * sm_count_current());
}

// One warp per row: its partials joined in a fixed order.
__global__ void __launch_bounds__(256) head_join_kernel(const HeadArgs a, float scale, float* __restrict__ logp,
                                                        float* __restrict__ entropy, float* __restrict__ lse) {
  const int row = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  follows();
  if (row >= a.rows) return;
  const int64_t rt = row / (2 * BM);
  const int n = a.few ? a.few : kShares * (a.group ? a.slots : (int)(((rt + 1) * a.n_tiles - 1) / a.per - rt * a.n_tiles / a.per + 1));
  const float4* parts = a.partials + (int64_t)row * (a.few ? a.few : a.slots * kShares);
  Stats s;
  float xt = 0.f;
  for (int i = lane; i < n; i += 32) s.m = fmaxf(s.m, parts[i].x);
  s.m = max_warp(s.m);
  for (int i = lane; i < n; i += 32) {
    const float4 p = parts[i];
    Stats o(make_float3(p.x, p.y, p.z));
    o.rebase(s.m, a.c);
    s.s0 += o.s0;
    s.s1 += o.s1;
    xt += p.w;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    s.s0 += __shfl_xor_sync(0xffffffffu, s.s0, o);
    s.s1 += __shfl_xor_sync(0xffffffffu, s.s1, o);
    xt += __shfl_xor_sync(0xffffffffu, xt, o);
  }
  if (lane) return;
  const float ln_s0 = logf(s.s0), h = fmaf(-kLn2, s.s1 / s.s0, ln_s0);
  const int t = a.targets ? a.targets[row] : -1;
  if (lse) lse[row] = s.s0 == 0.f ? -INFINITY : fmaf(s.m, scale, ln_s0);
  if (entropy) entropy[row] = (s.s0 == 0.f || h < 0.f) ? 0.f : h;
  if (logp) logp[row] = (t >= 0 && t < a.vocab) ? log_prob(xt, s, ln_s0, scale) : 0.f;
}
}  // namespace

int head_dev_error_read_and_clear() {
  int v = 0;
  cudaMemcpyFromSymbol(&v, zl_dev_error, sizeof(int));
  if (v) {
    int z = 0;
    cudaMemcpyToSymbol(zl_dev_error, &z, sizeof(int));
  }
  return v;
}
}  // namespace zl

// ============================================================== C ABI
using namespace zl;

extern "C" int64_t zl_linear_logprobs_workspace_floats(int rows, int dim, int vocab) {
  if (rows <= 0 || dim <= 0 || vocab <= 0 || rows > (1 << 30) || vocab > (1 << 30)) return 0;
  if (rows <= kFewRows && dim <= kFewDim) return (int64_t)rows * few_blocks(vocab) * 4;
  return (int64_t)rows * make_plan(rows, dim, vocab).slots * kShares * 4;
}

extern "C" zl_status zl_linear_logprobs_bf16(const zl_bf16* hidden, const zl_bf16* weight, const int32_t* targets, int rows,
                                             int dim, int vocab, float scale, float* logp, float* entropy, float* lse,
                                             float* workspace, zl_stream stream) {
  const char* what = "linear_logprobs";
  if (rows < 0 || dim <= 0 || vocab <= 0) return set_error(ZL_EINVAL, "%s: sizes must be positive", what);
  if (rows > (1 << 30) || vocab > (1 << 30)) return set_error(ZL_EUNSUPPORTED, "%s: at most 2^30 rows and vocabulary entries", what);
  if (dim % 8) return set_error(ZL_EUNSUPPORTED, "%s: dim %% 8 != 0", what);
  if (bad_scale(scale)) return set_error(ZL_EINVAL, "%s: scale must be in [1e-4, 1e4]", what);
  if (logp && !targets) return set_error(ZL_EINVAL, "%s: log probabilities need targets", what);
  if (rows == 0) return ZL_OK;
  if (!hidden || !weight || !workspace) return set_error(ZL_EINVAL, "%s: null hidden, weight or workspace", what);
  if ((reinterpret_cast<uintptr_t>(hidden) | reinterpret_cast<uintptr_t>(weight) | reinterpret_cast<uintptr_t>(workspace)) & 15)
    return set_error(ZL_EINVAL, "%s: hidden, weight and workspace must be 16-byte aligned", what);
  if ((reinterpret_cast<uintptr_t>(targets) | reinterpret_cast<uintptr_t>(logp) | reinterpret_cast<uintptr_t>(entropy) |
       reinterpret_cast<uintptr_t>(lse)) & 3)
    return set_error(ZL_EINVAL, "%s: a target or output array off a 4-byte boundary", what);
  if (rows <= kFewRows && dim <= kFewDim) {
    HeadArgs a{targets, rows, vocab, 0, 0, 0, 0, 0, 0, 0, scale * kLog2e, 0, few_blocks(vocab), reinterpret_cast<float4*>(workspace)};
    const size_t smem = (size_t)(dim + 31) / 32 * 512;
    cudaError_t e = cudaFuncSetAttribute(head_few_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kFewDim / 32 * 512);
    if (e != cudaSuccess) return launched(what, e);
    head_few_kernel<<<a.few, kFewWarps * 32, smem, (cudaStream_t)stream>>>(reinterpret_cast<const __nv_bfloat16*>(hidden),
                                                                           reinterpret_cast<const __nv_bfloat16*>(weight), dim, a);
    const zl_status st = check_launch(what);
    return st != ZL_OK ? st : launch_after(what, head_join_kernel, 1, 256, (cudaStream_t)stream, a, scale, logp, entropy, lse);
  }
  const Plan p = make_plan(rows, dim, vocab);
  CUtensorMap mh, mw;
  if (!make_tma_map(&mh, hidden, false, dim, rows, BK, BM, 128, 0) ||
      !make_tma_map(&mw, weight, false, dim, vocab, BK, BN / 2, 128, 0))
    return set_error(ZL_ECUDA, "%s: cuTensorMapEncodeTiled failed", what);
  HeadArgs a{targets, rows, vocab, (dim + BK - 1) / BK, p.row_tiles, p.n_tiles, p.slots, p.group, p.steps, p.per,
             scale * kLog2e, 0, 0, reinterpret_cast<float4*>(workspace)};
  const int chunks = (a.k_blocks + kChunk - 1) / kChunk;
  a.chunk = (a.k_blocks + chunks - 1) / chunks;
  const bool held = a.k_blocks <= kHeld;
  cudaLaunchAttribute attr;
  const cudaLaunchConfig_t cfg = pair_config(p.pairs, held ? Smem<true>::TOTAL : Smem<false>::TOTAL, (cudaStream_t)stream, &attr);
  // (make_plan has set the kernels' shared-memory attributes)
  cudaError_t e = held ? cudaLaunchKernelEx(&cfg, head_logprobs_kernel<true>, mh, mw, a)
                       : cudaLaunchKernelEx(&cfg, head_logprobs_kernel<false>, mh, mw, a);
  if (e != cudaSuccess) return launched(what, e);
  return launch_after(what, head_join_kernel, (rows + 7) / 8, 256, (cudaStream_t)stream, a, scale, logp, entropy, lse);
}
