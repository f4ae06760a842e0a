// Few-row attention over a paged cache, f16 queries (see attn_rows.cuh).
#include "attn_rows_launch.cuh"

namespace llg {
cudaError_t attn_rows_launch_f16(const AttnDev& p, const CUtensorMap& k, const CUtensorMap& v, bool fp8, int blocks, int ctas, bool pdl, cudaStream_t s) {
  return attn_rows_dispatch<__half>(p, k, v, fp8, blocks, ctas, pdl, s);
}
}  // namespace llg
