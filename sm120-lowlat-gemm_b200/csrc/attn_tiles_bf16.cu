// Many-row attention over a paged cache, bf16 queries (see attn_tiles.cuh).
#include "attn_tiles_launch.cuh"

namespace llg {
cudaError_t attn_tiles_launch_bf16(const AttnDev& p, const CUtensorMap& k, const CUtensorMap& v, const CUtensorMap& q, bool fp8, int ctas, bool pdl, cudaStream_t s) {
  return attn_tiles_dispatch<__nv_bfloat16>(p, k, v, q, fp8, ctas, pdl, s);
}
}  // namespace llg
