// Instantiations of the many-row attention kernel of one query type.
#pragma once

#include "attn_tiles.cuh"

namespace llg {

template <typename T, bool FP8, int D>
cudaError_t attn_tiles_start(const AttnDev& p, const CUtensorMap& k, const CUtensorMap& v, const CUtensorMap& q, int ctas, bool pdl, cudaStream_t s) {
  constexpr int smem = TilesCfg<T, FP8, D>::kSmem;
  static std::atomic<uint64_t> done{0};
  const cudaError_t e = allow_smem(reinterpret_cast<const void*>(attn_tiles_kernel<T, FP8, D>), smem, done);
  if (e != cudaSuccess) return e;
  return launch_ex(attn_tiles_kernel<T, FP8, D>, dim3(ctas), dim3(kTilesThreads), smem, s, pdl, dim3(1, 1, 1), p, k, v, q);
}

template <typename T>
cudaError_t attn_tiles_dispatch(const AttnDev& p, const CUtensorMap& k, const CUtensorMap& v, const CUtensorMap& q, bool fp8, int ctas, bool pdl, cudaStream_t s) {
  if (p.c.head_dim == 128) return fp8 ? attn_tiles_start<T, true, 128>(p, k, v, q, ctas, pdl, s) : attn_tiles_start<T, false, 128>(p, k, v, q, ctas, pdl, s);
  return fp8 ? attn_tiles_start<T, true, 64>(p, k, v, q, ctas, pdl, s) : attn_tiles_start<T, false, 64>(p, k, v, q, ctas, pdl, s);
}

}  // namespace llg
