// Instantiations of the few-row attention kernel of one query type.
#pragma once

#include "attn_rows.cuh"

namespace llg {

template <typename T, bool FP8, int D, int NB>
cudaError_t attn_rows_start(const AttnDev& p, const CUtensorMap& k, const CUtensorMap& v, int ctas, bool pdl, cudaStream_t s) {
  constexpr int smem = RowsCfg<T, FP8, D, NB>::kSmem;
  static std::atomic<uint64_t> done{0};
  const cudaError_t e = allow_smem(reinterpret_cast<const void*>(attn_rows_kernel<T, FP8, D, NB>), smem, done);
  if (e != cudaSuccess) return e;
  return launch_ex(attn_rows_kernel<T, FP8, D, NB>, dim3(ctas), dim3(kRowsThreads), smem, s, pdl, dim3(1, 1, 1), p, k, v);
}

template <typename T, bool FP8, int D>
cudaError_t attn_rows_blocks(const AttnDev& p, const CUtensorMap& k, const CUtensorMap& v, int blocks, int ctas, bool pdl, cudaStream_t s) {
  switch (blocks) {
    case 1: return attn_rows_start<T, FP8, D, 1>(p, k, v, ctas, pdl, s);
    case 2: return attn_rows_start<T, FP8, D, 2>(p, k, v, ctas, pdl, s);
    case 3: return attn_rows_start<T, FP8, D, 3>(p, k, v, ctas, pdl, s);
    default: return attn_rows_start<T, FP8, D, D == 64 ? 4 : 3>(p, k, v, ctas, pdl, s);  // head_dim 128 has no more than 24 rows here
  }
}

// blocks: 1 to 4 blocks of eight rows per tile.
template <typename T>
cudaError_t attn_rows_dispatch(const AttnDev& p, const CUtensorMap& k, const CUtensorMap& v, bool fp8, int blocks, int ctas, bool pdl, cudaStream_t s) {
  if (p.c.head_dim == 128) return fp8 ? attn_rows_blocks<T, true, 128>(p, k, v, blocks, ctas, pdl, s) : attn_rows_blocks<T, false, 128>(p, k, v, blocks, ctas, pdl, s);
  return fp8 ? attn_rows_blocks<T, true, 64>(p, k, v, blocks, ctas, pdl, s) : attn_rows_blocks<T, false, 64>(p, k, v, blocks, ctas, pdl, s);
}

}  // namespace llg
