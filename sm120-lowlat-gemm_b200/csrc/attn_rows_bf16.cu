// Few-row attention over a paged cache, bf16 queries (see attn_rows.cuh).
#include "attn_rows_launch.cuh"

namespace llg {
cudaError_t attn_rows_launch_bf16(const AttnDev& p, const CUtensorMap& k, const CUtensorMap& v, bool fp8, int blocks, int ctas, bool pdl, cudaStream_t s) {
  return attn_rows_dispatch<__nv_bfloat16>(p, k, v, fp8, blocks, ctas, pdl, s);
}
}  // namespace llg
