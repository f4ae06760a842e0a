// Attention over a paged cache: what is launched for a call, and where its scratch lies.
#include "paged_kv.cuh"

namespace llg {
namespace {

constexpr int kRowsMax = 32;  // rows of a few-row tile

struct Plan {
  int blocks;      // few-row kernel: blocks of eight rows per tile
  int rows_ctas;
  int64_t split, part_o, part_ml, bytes;  // scratch offsets
};

int64_t pad(int64_t v) { return (v + 255) / 256 * 256; }

// Depends on numbers the host has - never on lengths or offsets, which only the device reads.
Plan plan_of(const llg_attn_args& a) {
  const llg_paged_kv& c = a.kv;
  Plan p{};
  const int group = a.heads / c.kv_heads;
  // Rows per tile: a sequence's rows when all have the same number of new tokens, as wide as it gets when they may differ.
  const int64_t rows = c.q_starts ? (int64_t)c.tokens * group : (int64_t)(c.tokens / c.batch) * group;
  p.blocks = rows <= 8 ? 1 : rows <= 16 ? 2 : 4;
  if (group > 8 * p.blocks) p.blocks = group <= 16 ? 2 : 4;
  const int tile = p.blocks * 8;
  const int tok_tile = tile / group;
  const int64_t tiles = (c.tokens + tok_tile - 1) / tok_tile + c.batch;
  const int64_t units = tiles * c.kv_heads * (((int64_t)c.table_width * c.page_size + 63) / 64 + 1);
  p.rows_ctas = (int)(units < 2 * sm_count() ? units : 2 * sm_count());
  p.split = 0;
  p.part_ml = pad((int64_t)p.rows_ctas * 16);
  p.part_o = p.part_ml + pad((int64_t)p.rows_ctas * 2 * tile * 8);
  p.bytes = p.part_o + (int64_t)p.rows_ctas * 2 * tile * c.head_dim * 4;
  return p;
}

}  // namespace

int64_t attn_workspace(const llg_attn_args& a) {
  if (a.kv.batch == 0 || a.kv.tokens == 0) return 0;
  return plan_of(a).bytes;
}

cudaError_t attn_launch(const llg_attn_args& a, unsigned* status, cudaStream_t s) {
  const Plan plan = plan_of(a);
  AttnDev p{};
  p.c = paged_view(a.kv, status);
  p.q = static_cast<const unsigned char*>(a.q);
  p.q_tok = a.q_stride[0] * 2; p.q_head = a.q_stride[1] * 2;
  p.out = static_cast<unsigned char*>(a.out);
  p.o_tok = a.out_stride[0] * 2; p.o_head = a.out_stride[1] * 2;
  p.lse = a.lse;
  p.lse_tok = a.lse_stride;
  p.group = a.heads / a.kv.kv_heads;
  p.causal = a.causal != 0;
  p.window = a.window;
  p.scale_log2 = a.scale * 1.44269504088896341f;
  p.row_min = 0;
  p.row_max = INT32_MAX;
  p.tok_tile = plan.blocks * 8 / p.group;
  unsigned char* const ws = static_cast<unsigned char*>(a.ws);
  p.split = reinterpret_cast<int4*>(ws + plan.split);
  p.part_ml = reinterpret_cast<float*>(ws + plan.part_ml);
  p.part_o = reinterpret_cast<float*>(ws + plan.part_o);
  const bool fp8 = a.kv.dtype == LLG_DT_E4M3, f16 = a.q_dtype == LLG_DT_F16;
  const cudaError_t e = f16 ? attn_rows_launch_f16(p, fp8, plan.blocks, plan.rows_ctas, pdl_on(), s)
                            : attn_rows_launch_bf16(p, fp8, plan.blocks, plan.rows_ctas, pdl_on(), s);
  if (e != cudaSuccess) return e;
  return attn_combine_launch(p, f16, plan.rows_ctas, plan.blocks * 8, s);
}

}  // namespace llg
