// gemm_blk.cuh — tcgen05 products of the 8-bit float operators: block-scaled
// e4m3, and products grouped by expert (e4m3, f16 or bf16).
//
// For the rows i of group g (offsets[g] ≤ i < offsets[g+1]; one group of m
// rows when there are no offsets) and the weight matrix B_g [n, k]:
//     D[i, j] = Σ_kb sa[i, kb] · sb_g[j / 128, kb] · Σ_{k in kb} A[i, k] · B_g[j, k]
//               + bias_g[j]
// with kb running over k in blocks of 128. The inner sum is one tensor-core
// accumulation (f32, in TMEM); the outer one runs in f32 registers, because
// the scales are arbitrary f32 numbers and change with every kb. 16-bit
// operands have no scales: all of k accumulates in TMEM.
//
// One persistent CTA per SM (BlkCfg::kThreads threads):
//   warp 0   TMA producer: 128-byte-swizzled k-blocks of both operands into a
//            ring of shared-memory stages
//   warp 1   lane 0 issues tcgen05.mma into one of kNumAcc TMEM accumulators,
//            one k-block each (e4m3) or one tile each (16-bit)
//   warp 2   e4m3: copies the scales of each k-block into a ring of its own
//            (cp.async, arriving on the ring's barriers)
//   warp 3   allocates TMEM, lays out the groups' tiles
//   warps 4- accumulate: TMEM → registers, times the scales, and at the end
//            of the tile the store
// Two forms:
//   SWAP = false  128 tokens (MMA rows) × BN weight rows: a thread holds one
//                 token's row, so a k-block's scale is one number per thread
//                 and each accumulator element costs one fused multiply-add.
//   SWAP = true   128 weight rows (MMA rows) × BN ≤ 64 tokens: for few tokens
//                 per group, where the weights are the traffic and a 128-row
//                 token tile would be mostly padding. The k-blocks may be
//                 split over the CTAs of a cluster; the partial tiles meet in
//                 distributed shared memory and are added in rank order, so
//                 the result does not depend on timing and no workspace is
//                 needed.
#pragma once

#include <cuda_fp16.h>

#include "common.cuh"
#include "mathf32.cuh"

namespace futon {

constexpr int kBlkMaxGroups = 1024;
constexpr int kBlkRing = 8;   // k-blocks of scales in flight
constexpr int kBlkBand = 16;  // row tiles that share a weight tile before the next one

enum BlkOut : int { kBlkOutF32 = 0, kBlkOutF16 = 1, kBlkOutBf16 = 2 };

struct BlkParams {
  int m, n, k;
  int groups;
  const int* offsets;    // [groups + 1] or null: one group of m rows
  const float* a_scale;  // e4m3: [m, ceil(k / 128)]
  const float* b_scale;  // e4m3: [groups, ceil(n / 128), ceil(k / 128)]
  const float* bias;     // [groups, n] or null
  void* out;             // row stride ldo elements
  long long ldo;
  int out_kind;          // BlkOut
  int out_vec;           // rows of out start at multiples of 16 bytes
  int split;             // SWAP: CTAs of a cluster that share a tile's k-blocks
  int ab_format;         // 16-bit operands: 0 = f16, 1 = bf16
  int* err;              // device error word
};

template <bool F8, bool SWAP, int BN>
struct BlkCfg {
  static constexpr int kTokens = SWAP ? BN : 128;   // rows of A per tile
  static constexpr int kWeights = SWAP ? 128 : BN;  // rows of B per tile
  static constexpr int kBK = F8 ? 128 : 64;         // k elements of a 128-byte row
  static constexpr int kXBytes = 128 * 128;
  static constexpr int kYBytes = BN * 128;
  static constexpr int kStageBytes = kXBytes + kYBytes;
  static constexpr int kEpiWarps = SWAP ? 4 : 8;
  static constexpr int kParts = kEpiWarps / 4;  // warps that share a TMEM lane quarter
  static constexpr int kCols = BN / kParts;     // accumulator columns of one thread
  static constexpr int kThreads = 128 + 32 * kEpiWarps;
  static constexpr uint32_t kAccStride = BN < 32 ? 32 : BN;
  static constexpr int kNumAcc = BN == 256 ? 2 : 4;
  static constexpr uint32_t kTmemCols = kNumAcc * kAccStride;
  static constexpr int kSlotFloats = kTokens + 4;  // a scales, then up to two b scales
  static constexpr int kRingBytes = F8 ? (kBlkRing * kSlotFloats * 4 + 1023) / 1024 * 1024 : 0;
  static constexpr int kSchedBytes = (2 * (kBlkMaxGroups + 1) * 4 + 1023) / 1024 * 1024;
  // Partial tiles from the cluster's CTAs, by tile parity; BN tokens cut into
  // `split` runs of ceil(BN / split) tokens need up to BN + 7 columns.
  static constexpr int kXchCols = SWAP ? BN + 8 : 0;
  static constexpr int kXchBytes = 2 * kXchCols * 128 * 4;
  static constexpr int kFixed = 1024 /*align*/ + 1024 /*barriers*/ + kSchedBytes + kRingBytes + kXchBytes;
  static constexpr int kBudget = 227 * 1024;
  static constexpr int kFit = (kBudget - kFixed) / kStageBytes;
  static constexpr int kStages = kFit > 10 ? 10 : kFit;
  static constexpr int kSmemBytes = kFixed + kStages * kStageBytes;
  static_assert(kStages >= 4 && kSmemBytes <= kBudget, "shared-memory budget");
  static_assert(kTmemCols <= 512 && (kTmemCols & (kTmemCols - 1)) == 0, "TMEM columns");
};

// tcgen05.mma with 8-bit float operands (kind::f8f6f4), f32 accumulation.
__device__ __forceinline__ void mma_f8(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc,
                                       uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// 16 consecutive columns of this thread's TMEM lane.
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}

// Asynchronous 4-byte copy; `ok` false writes 0 and reads nothing.
__device__ __forceinline__ void cp_async4(uint32_t dst, const float* src, bool ok) {
  const int n = ok ? 4 : 0;
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(n)
               : "memory");
}
// Arrives on `bar` (one of its expected arrivals) once this thread's earlier
// cp.async copies have landed.
__device__ __forceinline__ void cp_async_arrive(uint32_t bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared.b64 [%0];" ::"r"(bar) : "memory");
}

__device__ __forceinline__ void st_cluster_f32(uint32_t caddr, float v) {
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(caddr), "f"(v) : "memory");
}

// One value in the output's type, rounded to nearest even.
__device__ __forceinline__ void blk_store1(void* out, int kind, size_t i, float v) {
  if (kind == kBlkOutF32) reinterpret_cast<float*>(out)[i] = v;
  else if (kind == kBlkOutF16) reinterpret_cast<__half*>(out)[i] = __float2half_rn(v);
  else reinterpret_cast<__nv_bfloat16*>(out)[i] = __float2bfloat16_rn(v);
}

// Eight consecutive values of a row.
template <int KIND>
__device__ __forceinline__ void blk_store8(void* out, size_t i, const float* v) {
  if constexpr (KIND == kBlkOutF32) {
    float4* d = reinterpret_cast<float4*>(reinterpret_cast<float*>(out) + i);
    d[0] = make_float4(v[0], v[1], v[2], v[3]);
    d[1] = make_float4(v[4], v[5], v[6], v[7]);
  } else {
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (KIND == kBlkOutF16) {
        const __half2 h = __floats2half2_rn(v[2 * j], v[2 * j + 1]);
        w[j] = *reinterpret_cast<const uint32_t*>(&h);
      } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
        w[j] = *reinterpret_cast<const uint32_t*>(&h);
      }
    }
    *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(out) + i) =
        make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// The NC columns [col, col + NC) of one output row.
template <int KIND, int NC>
__device__ __forceinline__ void blk_store_row(const BlkParams& p, int row, int col,
                                              const uint64_t (&acc)[NC / 2], const float* bias) {
#pragma unroll
  for (int c = 0; c < NC; c += 8) {
    float v[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) f2_unpack(acc[c / 2 + j], v[2 * j], v[2 * j + 1]);
    if (bias) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (col + c + j < p.n) v[j] += __ldg(bias + col + c + j);
    }
    const size_t at = (size_t)row * p.ldo + col + c;
    if (p.out_vec && col + c + 8 <= p.n) {
      blk_store8<KIND>(p.out, at, v);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (col + c + j < p.n) blk_store1(p.out, KIND, at + j, v[j]);
    }
  }
}

// A tile: rows [row0, row_end) of A (at most kTokens of them are its own)
// with the weight tile nt of group g.
struct BlkTile {
  int g, row0, row_end, nt;
};

// Tiles run group by group; inside a group in bands of kBlkBand row tiles,
// row tiles fastest, so CTAs running together share weight tiles through L2.
__device__ __forceinline__ BlkTile blk_tile(int t, const int* goff, const int* gtile, int groups,
                                            int ntn, int tokens) {
  int lo = 0, hi = groups;  // the last group whose first tile is ≤ t
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if ((long long)gtile[mid] * ntn <= t) lo = mid; else hi = mid;
  }
  const int mt = gtile[lo + 1] - gtile[lo];
  const int local = t - gtile[lo] * ntn;
  const int band = local / (kBlkBand * ntn), in = local - band * (kBlkBand * ntn);
  const int rows = min(kBlkBand, mt - band * kBlkBand);
  BlkTile r;
  r.g = lo;
  r.nt = in / rows;
  r.row0 = goff[lo] + (band * kBlkBand + in - r.nt * rows) * tokens;
  r.row_end = goff[lo + 1];
  return r;
}

template <bool F8, bool SWAP, int BN>
__global__ void __launch_bounds__(BlkCfg<F8, SWAP, BN>::kThreads, 1)
    gemm_blk_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                    const __grid_constant__ BlkParams p) {
  using C = BlkCfg<F8, SWAP, BN>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~uintptr_t(1023));
  uint8_t* fixed = smem + C::kStages * C::kStageBytes;
  uint64_t* bars = reinterpret_cast<uint64_t*>(fixed);
  uint64_t* full_bar = bars;                      // [kStages] TMA → MMA
  uint64_t* empty_bar = full_bar + C::kStages;    // [kStages] MMA → TMA
  uint64_t* accf_bar = empty_bar + C::kStages;    // [kNumAcc] MMA → accumulate
  uint64_t* acce_bar = accf_bar + C::kNumAcc;     // [kNumAcc] accumulate → MMA
  uint64_t* sfull_bar = acce_bar + C::kNumAcc;    // [kBlkRing] scales → accumulate
  uint64_t* sempty_bar = sfull_bar + kBlkRing;    // [kBlkRing] accumulate → scales
  uint64_t* xfull_bar = sempty_bar + kBlkRing;    // [2] partial tiles of the cluster
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(xfull_bar + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* goff = reinterpret_cast<int*>(fixed + 1024);  // [groups + 1] clamped offsets
  int* gtile = goff + kBlkMaxGroups + 1;             // [groups + 1] row tiles before a group
  float* ring = reinterpret_cast<float*>(fixed + 1024 + C::kSchedBytes);
  float* xch = reinterpret_cast<float*>(fixed + 1024 + C::kSchedBytes + C::kRingBytes);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int split = SWAP ? p.split : 1;
  const int crank = split > 1 ? (int)cluster_ctarank() : 0;
  const int nkb = (p.k + C::kBK - 1) / C::kBK;
  const int kb0 = (int)((long long)crank * nkb / split);
  const int kb1 = (int)((long long)(crank + 1) * nkb / split);
  const int ntn = (p.n + C::kWeights - 1) / C::kWeights;

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(smem_u32(&full_bar[s]), 1);
      mbar_init(smem_u32(&empty_bar[s]), 1);
    }
    for (int a = 0; a < C::kNumAcc; ++a) {
      mbar_init(smem_u32(&accf_bar[a]), 1);
      mbar_init(smem_u32(&acce_bar[a]), C::kEpiWarps);
    }
    for (int s = 0; s < kBlkRing; ++s) {
      mbar_init(smem_u32(&sfull_bar[s]), 32);
      mbar_init(smem_u32(&sempty_bar[s]), C::kEpiWarps);
    }
    for (int x = 0; x < 2; ++x) mbar_init(smem_u32(&xfull_bar[x]), (uint32_t)(split * C::kEpiWarps));
    *abort_flag = 0;
    fence_barrier_init();
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmB);
  }
  if (warp == 3) {
    tmem_alloc(smem_u32(tmem_slot), C::kTmemCols);
    tmem_relinquish();
  }
  pdl_wait();
  pdl_trigger();
  if (p.offsets)
    for (int i = threadIdx.x; i <= p.groups; i += C::kThreads) goff[i] = __ldg(p.offsets + i);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 3) {
    if (p.offsets) {
      // Offsets outside [0, m] or falling below an earlier one are clamped
      // (so no row outside the buffers is touched) and reported.
      int top = 0, tiles = 0;
      bool bad = false;
      for (int base = 0; base <= p.groups; base += 32) {
        const int i = base + lane;
        const int raw = i <= p.groups ? goff[i] : 0;
        int v = min(max(raw, 0), p.m);
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int u = __shfl_up_sync(0xffffffffu, v, o);
          if (lane >= o) v = max(v, u);
        }
        v = max(v, top);
        int before = __shfl_up_sync(0xffffffffu, v, 1);
        if (lane == 0) before = base ? top : v;
        int tl = i <= p.groups ? (v - before + C::kTokens - 1) / C::kTokens : 0;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int u = __shfl_up_sync(0xffffffffu, tl, o);
          if (lane >= o) tl += u;
        }
        tl += tiles;
        if (i <= p.groups) {
          bad |= raw != v;
          goff[i] = v;
          gtile[i] = tl;
        }
        top = __shfl_sync(0xffffffffu, v, 31);
        tiles = __shfl_sync(0xffffffffu, tl, 31);
      }
      if (bad) atomicCAS(p.err, 0, (int)kDevBadInput);
    } else if (lane == 0) {
      goff[0] = 0;
      goff[1] = p.m;
      gtile[0] = 0;
      gtile[1] = (p.m + C::kTokens - 1) / C::kTokens;
    }
  }
  // Peers' barriers exist before any remote arrive.
  if (split > 1) cluster_sync_all();
  else __syncthreads();
  const uint32_t tmem_base = *tmem_slot;
  const int num_tiles = gtile[p.groups] * ntn;
  const int first = (int)blockIdx.x / split;
  const int stride = (int)gridDim.x / split;
  auto tile_at = [&](int t) { return blk_tile(t, goff, gtile, p.groups, ntn, C::kTokens); };

  if (warp == 0) {
    if (lane == 0) {
      // ---------------- TMA producer ----------------
      int stage = 0;
      uint32_t phase = 0;
      int issued = 0;
      for (int tile = first; tile < num_tiles; tile += stride) {
        const BlkTile t = tile_at(tile);
        const int arow = t.row0, brow = t.g * p.n + t.nt * C::kWeights;
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!mbar_wait_bounded(smem_u32(&empty_bar[stage]), phase ^ 1u, p.err,
                                 kDevTimeoutSmemEmpty, abort_flag))
            goto producer_done;
          const uint32_t sx = smem_u32(smem + stage * C::kStageBytes);
          const uint32_t fb = smem_u32(&full_bar[stage]);
          mbar_arrive_expect_tx(fb, C::kStageBytes);
          tma_load_2d(sx, SWAP ? &tmB : &tmA, fb, kb * C::kBK, SWAP ? brow : arow);
          tma_load_2d(sx + C::kXBytes, SWAP ? &tmA : &tmB, fb, kb * C::kBK, SWAP ? arow : brow);
          ++issued;
          if (++stage == C::kStages) { stage = 0; phase ^= 1u; }
        }
      }
    producer_done:
      // This thread's own copies have landed before the CTA exits.
      const int n = issued < C::kStages ? issued : C::kStages;
      for (int i = 0; i < n; ++i) {
        if (--stage < 0) { stage = C::kStages - 1; phase ^= 1u; }
        const uint64_t t0 = globaltimer_ns();
        while (!mbar_try_wait(smem_u32(&full_bar[stage]), phase)) {
          if (globaltimer_ns() - t0 > kWaitLimitNs) break;
        }
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      // ---------------- MMA issuer ----------------
      // kind::f8f6f4: e4m3 is format 0; kind::f16: f16 0, bf16 1.
      const uint32_t idesc = make_idesc(1u, F8 ? 0u : (uint32_t)p.ab_format, 128u, (uint32_t)BN);
      int stage = 0;
      uint32_t phase = 0;
      int it = 0;  // accumulations begun
      bool ok = true;
      for (int tile = first; tile < num_tiles && ok; tile += stride) {
        for (int kb = kb0; kb < kb1; ++kb) {
          const bool fresh = F8 || kb == kb0;
          const int cur = fresh ? it : it - 1;
          const int acc = cur % C::kNumAcc;
          if (fresh) {
            if (!mbar_wait_bounded(smem_u32(&acce_bar[acc]),
                                   ((uint32_t)(it / C::kNumAcc) & 1u) ^ 1u, p.err,
                                   kDevTimeoutAccEmpty, abort_flag)) {
              ok = false;
              break;
            }
            ++it;
          }
          if (!mbar_wait_bounded(smem_u32(&full_bar[stage]), phase, p.err, kDevTimeoutTmaFull,
                                 abort_flag)) {
            ok = false;
            // The accumulation begun above still commits, for the drain below.
            mma_commit(smem_u32(&accf_bar[acc]));
            break;
          }
          tc_fence_after();
          const uint32_t sx = smem_u32(smem + stage * C::kStageBytes);
          const uint64_t xdesc = smem_desc_k_sw128(sx);
          const uint64_t ydesc = smem_desc_k_sw128(sx + C::kXBytes);
          const uint32_t d = tmem_base + (uint32_t)acc * C::kAccStride;
#pragma unroll
          for (int ks = 0; ks < 4; ++ks) {
            const uint64_t koff = (uint64_t)(ks * 2);  // 32 bytes along k, encoded >> 4
            const uint32_t on = (!fresh || ks) ? 1u : 0u;
            if constexpr (F8) mma_f8(d, xdesc + koff, ydesc + koff, idesc, on);
            else mma_f16kind(d, xdesc + koff, ydesc + koff, idesc, on);
          }
          mma_commit(smem_u32(&empty_bar[stage]));
          if (F8 || kb + 1 == kb1) mma_commit(smem_u32(&accf_bar[acc]));
          if (++stage == C::kStages) { stage = 0; phase ^= 1u; }
        }
      }
      // The last committed MMAs are done before TMEM is freed (bounded).
      if (it > 0) {
        const uint64_t t0 = globaltimer_ns();
        const int acc = (it - 1) % C::kNumAcc;
        while (!mbar_try_wait(smem_u32(&accf_bar[acc]), (uint32_t)((it - 1) / C::kNumAcc) & 1u)) {
          if (globaltimer_ns() - t0 > kWaitLimitNs) break;
        }
      }
    }
  } else if (warp == 2) {
    if constexpr (F8) {
      // ---------------- scales ----------------
      const int nnb = (p.n + 127) / 128;
      int slot = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int tile = first; tile < num_tiles && ok; tile += stride) {
        const BlkTile t = tile_at(tile);
        const int nb0 = t.nt * (C::kWeights / 128);
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!mbar_wait_bounded(smem_u32(&sempty_bar[slot]), phase ^ 1u, p.err,
                                 kDevTimeoutSmemEmpty, abort_flag)) {
            ok = false;
            break;
          }
          const uint32_t dst = smem_u32(ring + slot * C::kSlotFloats);
#pragma unroll
          for (int i = lane; i < C::kTokens; i += 32) {
            const bool in = t.row0 + i < t.row_end;
            cp_async4(dst + 4u * (uint32_t)i,
                      p.a_scale + (in ? (size_t)(t.row0 + i) * nkb + kb : 0), in);
          }
          if (lane < C::kWeights / 128) {
            const bool in = nb0 + lane < nnb;
            cp_async4(dst + 4u * (uint32_t)(C::kTokens + lane),
                      p.b_scale + (in ? ((size_t)t.g * nnb + nb0 + lane) * nkb + kb : 0), in);
          }
          cp_async_arrive(smem_u32(&sfull_bar[slot]));
          if (++slot == kBlkRing) { slot = 0; phase ^= 1u; }
        }
      }
      asm volatile("cp.async.wait_all;" ::: "memory");
    }
  } else if (warp >= 4) {
    // ---------------- accumulate and store ----------------
    const int quarter = warp & 3;
    const int part = (warp - 4) >> 2;
    int it = 0, slot = 0, done = 0;
    uint32_t sphase = 0;
    bool ok = true;
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
    for (int tile = first; tile < num_tiles; tile += stride, ++done) {
      const BlkTile t = tile_at(tile);
      uint64_t acc[C::kCols / 2];
#pragma unroll
      for (int i = 0; i < C::kCols / 2; ++i) acc[i] = 0;
      const int steps = F8 ? kb1 - kb0 : 1;
      for (int s = 0; s < steps; ++s, ++it) {
        const int a = it % C::kNumAcc;
        const float* sc = ring + slot * C::kSlotFloats;
        if (F8)
          ok = mbar_wait_bounded(smem_u32(&sfull_bar[slot]), sphase, p.err, kDevTimeoutTmaFull,
                                 abort_flag);
        ok = ok && mbar_wait_bounded(smem_u32(&accf_bar[a]), (uint32_t)(it / C::kNumAcc) & 1u,
                                     p.err, kDevTimeoutAccFull, abort_flag);
        // The whole warp goes on or leaves (tcgen05.ld is warp-wide).
        if (!__all_sync(0xffffffffu, ok)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t taddr =
            tmem_base + (uint32_t)a * C::kAccStride + lanes + (uint32_t)(part * C::kCols);
        if constexpr (SWAP) {
          const float sb = F8 ? sc[C::kTokens] : 1.0f;
          const uint64_t sb2 = f2_pack(sb, sb);
          constexpr int kChunks = C::kCols / 16;
#pragma unroll
          for (int c = 0; c < kChunks; ++c) {
            uint32_t u[16];
            tmem_ld16(taddr + 16 * c, u);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              uint64_t s0 = 0, s1 = 0;
              if constexpr (F8) {
                const float4 q = *reinterpret_cast<const float4*>(sc + 16 * c + 4 * i);
                s0 = f2_mul(f2_pack(q.x, q.y), sb2);
                s1 = f2_mul(f2_pack(q.z, q.w), sb2);
              }
              const uint64_t d0 = f2_pack(__uint_as_float(u[4 * i]), __uint_as_float(u[4 * i + 1]));
              const uint64_t d1 =
                  f2_pack(__uint_as_float(u[4 * i + 2]), __uint_as_float(u[4 * i + 3]));
              uint64_t& x0 = acc[8 * c + 2 * i];
              uint64_t& x1 = acc[8 * c + 2 * i + 1];
              x0 = F8 ? f2_fma(d0, s0, x0) : d0;
              x1 = F8 ? f2_fma(d1, s1, x1) : d1;
            }
          }
        } else {
          const float sv = F8 ? sc[quarter * 32 + lane] *
                                    sc[C::kTokens + (C::kWeights > 128 ? part : 0)]
                              : 1.0f;
          const uint64_t s2 = f2_pack(sv, sv);
          constexpr int kChunks = C::kCols / 32;
#pragma unroll
          for (int c = 0; c < kChunks; ++c) {
            uint32_t u[32];
            tmem_ld32(taddr + 32 * c, u);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const uint64_t d = f2_pack(__uint_as_float(u[2 * i]), __uint_as_float(u[2 * i + 1]));
              acc[16 * c + i] = F8 ? f2_fma(d, s2, acc[16 * c + i]) : d;
            }
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(smem_u32(&acce_bar[a]));
          if (F8) mbar_arrive(smem_u32(&sempty_bar[slot]));
        }
        if (F8 && ++slot == kBlkRing) { slot = 0; sphase ^= 1u; }
      }
      if (!ok) break;

      if constexpr (!SWAP) {
        const int row = t.row0 + quarter * 32 + lane;
        const int col = t.nt * C::kWeights + part * C::kCols;
        const float* bias = p.bias ? p.bias + (size_t)t.g * p.n : nullptr;
        if (row < t.row_end) {
          if (p.out_kind == kBlkOutF32) blk_store_row<kBlkOutF32, C::kCols>(p, row, col, acc, bias);
          else if (p.out_kind == kBlkOutF16) blk_store_row<kBlkOutF16, C::kCols>(p, row, col, acc, bias);
          else blk_store_row<kBlkOutBf16, C::kCols>(p, row, col, acc, bias);
        }
      } else {
        const int line = quarter * 32 + lane;  // weight row of the tile
        const int col = t.nt * 128 + line;
        const float bv = p.bias && col < p.n ? __ldg(p.bias + (size_t)t.g * p.n + col) : 0.0f;
        float v[BN];
#pragma unroll
        for (int j = 0; j < BN / 2; ++j) f2_unpack(acc[j], v[2 * j], v[2 * j + 1]);
        if (split == 1) {
          if (col < p.n) {
#pragma unroll
            for (int j = 0; j < BN; ++j)
              if (t.row0 + j < t.row_end)
                blk_store1(p.out, p.out_kind, (size_t)(t.row0 + j) * p.ldo + col, v[j] + bv);
          }
        } else {
          // Token j goes to rank j / each, which adds the ranks' partial sums
          // in rank order. Buffers alternate by tile: a peer sends its sums
          // of tile t only after it has read those of tile t - 2, and its
          // sums of tile t - 1 have been waited for here.
          const int each = (BN + split - 1) / split;
          const int par = done & 1;
          const uint32_t base =
              smem_u32(xch + ((size_t)par * C::kXchCols + crank * each) * 128 + line);
#pragma unroll
          for (int j = 0; j < BN; ++j) {
            const int owner = j / each;
            st_cluster_f32(mapa_shared(base + (uint32_t)(j - owner * each) * 512u, (uint32_t)owner),
                           v[j]);
          }
          asm volatile("fence.acq_rel.cluster;" ::: "memory");
          __syncwarp();
          if (lane < split)
            mbar_arrive_cluster(mapa_shared(smem_u32(&xfull_bar[par]), (uint32_t)lane));
          ok = mbar_wait_cluster_bounded(smem_u32(&xfull_bar[par]), (uint32_t)(done >> 1) & 1u,
                                         p.err, kDevTimeoutLnPeer, abort_flag);
          if (!__all_sync(0xffffffffu, ok)) break;
          const float* mine = xch + (size_t)par * C::kXchCols * 128 + line;
          for (int j = 0; j < each; ++j) {
            const int row = t.row0 + crank * each + j;
            if (crank * each + j >= BN || row >= t.row_end || col >= p.n) break;
            float sum = 0.0f;
            for (int q = 0; q < split; ++q) sum += mine[(q * each + j) * 128];
            blk_store1(p.out, p.out_kind, (size_t)row * p.ldo + col, sum + bv);
          }
        }
      }
    }
  }

  __syncthreads();
  // No CTA of a cluster leaves while a peer may still store into its shared
  // memory (every wait above is bounded, so all CTAs get here).
  if (split > 1) cluster_sync_all();
  if (warp == 3) {
    tc_fence_after();
    tmem_dealloc(tmem_base, C::kTmemCols);
  }
}

}  // namespace futon
