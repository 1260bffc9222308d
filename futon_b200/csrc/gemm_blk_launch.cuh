// gemm_blk_launch.cuh — host-side launch of the gemm_blk_kernel instantiations.
#pragma once

#include <algorithm>
#include <atomic>

#include "gemm_blk.cuh"

namespace futon {

struct BlkLaunch {
  const CUtensorMap* ta;  // A: box kTokens (≤ 128) × 128 bytes
  const CUtensorMap* tb;  // B: box kYRows × 128 bytes
  const CUtensorMap* to;  // output (p.out_tma), or any other map
  BlkParams p;
  bool swap;
  bool ragged;  // rows of the output are not made of whole 16-byte pieces
  int bn;
  long long tiles;  // at most this many tiles
  int device;
  int num_sms;
  cudaStream_t stream;
};

// Defined in gemm_f8.cu and gemm_grouped16.cu.
cudaError_t launch_blk_f8(const BlkLaunch& g);
cudaError_t launch_blk_16(const BlkLaunch& g);

template <bool F8, bool SWAP, int BN, bool PAIR = false, bool SPLITK = SWAP, bool RAG = false>
cudaError_t launch_blk_inst(const BlkLaunch& g) {
  using C = BlkCfg<F8, SWAP, BN, PAIR, SPLITK>;
  auto kern = gemm_blk_kernel<F8, SWAP, BN, PAIR, SPLITK, RAG>;
  static std::atomic<uint64_t> attr_done{0};  // one bit per device
  const uint64_t bit = 1ull << (g.device & 63);
  if (!(attr_done.load() & bit)) {
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         C::kSmemBytes);
    if (e != cudaSuccess) return e;
    // setmaxnreg.inc would wait for registers that the launch does not hold.
    cudaFuncAttributes fa;
    if ((e = cudaFuncGetAttributes(&fa, kern)) != cudaSuccess) return e;
    if (fa.numRegs < C::kRegsNeeded) return cudaErrorLaunchOutOfResources;
    attr_done.fetch_or(bit);
  }
  const int split = SPLITK ? g.p.split : PAIR ? 2 : 1;  // CTAs of a cluster
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  int na = 0;
  attr[na].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[na].val.programmaticStreamSerializationAllowed = 1;
  ++na;
  if (split > 1) {
    attr[na].id = cudaLaunchAttributeClusterDimension;
    attr[na].val.clusterDim.x = (unsigned)split;
    attr[na].val.clusterDim.y = 1;
    attr[na].val.clusterDim.z = 1;
    ++na;
  }
  const long long wave = std::max(1, g.num_sms / split);
  cfg.gridDim = dim3((unsigned)(std::min(g.tiles, wave) * split));
  cfg.blockDim = dim3(C::kThreads);
  cfg.dynamicSmemBytes = C::kSmemBytes;
  cfg.stream = g.stream;
  cfg.attrs = attr;
  cfg.numAttrs = (unsigned)na;
  return cudaLaunchKernelEx(&cfg, kern, *g.ta, *g.tb, *g.to, g.p);
}

template <bool F8, bool RAG>
cudaError_t launch_blk_rows(const BlkLaunch& g) {
  if (g.bn == 256) return launch_blk_inst<F8, false, 256, true, false, RAG>(g);
  if (g.p.split > 1) return launch_blk_inst<F8, false, 128, false, true, RAG>(g);
  return launch_blk_inst<F8, false, 128, false, false, RAG>(g);
}

template <bool F8>
cudaError_t launch_blk_any(const BlkLaunch& g) {
  if (g.swap) {
    if (g.bn == 16) return launch_blk_inst<F8, true, 16>(g);
    if (g.bn == 32) return launch_blk_inst<F8, true, 32>(g);
    return launch_blk_inst<F8, true, 64>(g);
  }
  return g.ragged ? launch_blk_rows<F8, true>(g) : launch_blk_rows<F8, false>(g);
}

}  // namespace futon
