// Attention over a paged cache: what is launched for a call, and where its scratch lies.
#include <cmath>

#include "paged_kv.cuh"

namespace llg {
namespace {

constexpr int kTileRows = 256;

struct Part {  // one kernel's CTAs and scratch
  int ctas, rows, tok_tile;
  int row_max;     // query rows per kv head of the sequences it serves
  int64_t split, first, part_ml, part_o;  // offsets
};
struct Plan {
  bool few, many;
  Part f, m;
  int64_t units;  // no more key tiles than this
  int64_t bytes;
};

int64_t pad(int64_t v) { return (v + 255) / 256 * 256; }

void lay_out(Part* q, int64_t units, int ctas, int rows, int head_dim, int64_t* at) {
  q->ctas = (int)(units < ctas ? units : ctas);
  q->rows = rows;
  q->split = *at;
  q->first = q->split + pad((int64_t)q->ctas * 32);
  q->part_ml = q->first + pad((int64_t)q->ctas * 4);
  q->part_o = q->part_ml + pad((int64_t)q->ctas * 2 * rows * 8);
  *at = q->part_o + pad((int64_t)q->ctas * 2 * rows * head_dim * 4);
}

// Depends on numbers the host has - never on lengths or offsets, which only the device reads. Without offsets every sequence
// has the same number of rows and one kernel serves them all; with offsets both are launched and each takes its own.
Plan plan_of(const llg_attn_args& a) {
  const llg_paged_kv& c = a.kv;
  Plan p{};
  const int group = a.heads / c.kv_heads, sms = sm_count();
  const int64_t most = c.q_starts ? (int64_t)c.tokens * group : (int64_t)(c.tokens / c.batch) * group;
  const int64_t keys = (int64_t)c.table_width * c.page_size;
  // Rows per kv head that the few-row kernel takes. 25 to 32 rows of head_dim 128 fill its registers and run faster as tiles, fewer
  // and narrower ones do not (16 sequences of 1.2k to 2.5k keys, few-row kernel against tiles, us: 32 rows of 128 16-bit values 76
  // and 50.5, e4m3 78 and 69; 24 rows 44 and 50.5, 46 and 69; 32 rows of 64 values 38 and 41, 42 and 51).
  const int64_t fit = c.head_dim == 128 ? 24 : 32;
  // With offsets it takes the sequences of one token (of a few, where the group is small), in tiles no wider than that: wider ones
  // would hold registers that decoding sequences do not use. Without, tiles as wide as the rows. (Eight heads per kv head, tiles of
  // 8 rows against 24, us: 32 decoding sequences over e4m3 72 and 120, over bf16 103 and 111; 16 sequences of 1 to 5 drafted tokens 64 and
  // 71, 58 and 66; of 1 to 3, all of which the wider tiles take, 62 and 48, 58 and 48. Calls of equal counts without offsets: 62 and 93 for
  // the 32, 39 and 36 for 16 of two tokens.)
  const int64_t widest = c.q_starts ? (group <= 8 ? 8 : group <= 16 ? 16 : fit) : fit;
  p.few = group <= widest && (c.q_starts || most <= widest);
  p.many = most > widest;
  if (p.few) {
    const int64_t rows = most < widest ? most : widest;
    const int blocks = (int)(rows + 7) / 8;
    p.f.row_max = (int)widest;
    p.f.tok_tile = blocks * 8 / group;
    p.units = (int64_t)c.batch * c.kv_heads * ((keys + 63) / 64 + 1);  // one tile per sequence
    lay_out(&p.f, p.units, rows_ctas_per_sm(c.dtype == LLG_DT_E4M3, c.head_dim, blocks) * sms, blocks * 8, c.head_dim, &p.bytes);
  }
  if (p.many) {
    p.m.tok_tile = kTileRows / group;
    const int64_t tiles = (c.tokens + p.m.tok_tile - 1) / p.m.tok_tile + c.batch;
    const int64_t units = tiles * c.kv_heads * ((keys + 127) / 128 + 1);
    if (units > p.units) p.units = units;
    lay_out(&p.m, units, sms, kTileRows, c.head_dim, &p.bytes);
  }
  return p;
}

}  // namespace

int64_t attn_workspace(const llg_attn_args& a) {
  if (a.kv.batch == 0 || a.kv.tokens == 0) return 0;
  const Plan p = plan_of(a);
  return p.units < INT32_MAX / 2 ? p.bytes : -1;  // the kernels count key tiles in 32 bits
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
  p.window = a.window < (1 << 30) ? a.window : 1 << 30;  // no cache is longer, and positions less this stay in 32 bits
  const bool fp8 = a.kv.dtype == LLG_DT_E4M3, f16 = a.q_dtype == LLG_DT_F16;
  const float scale_log2 = a.scale * 1.44269504088896341f;
  unsigned char* const ws = static_cast<unsigned char*>(a.ws);
  auto use = [&](const Part& q) {
    p.tok_tile = q.tok_tile;
    p.split = reinterpret_cast<int4*>(ws + q.split);
    p.first = reinterpret_cast<int*>(ws + q.first);
    p.part_ml = reinterpret_cast<float*>(ws + q.part_ml);
    p.part_o = reinterpret_cast<float*>(ws + q.part_o);
  };
  auto lined_up = [](const unsigned char* base, int64_t page, int64_t head, int64_t slot) {
    return reinterpret_cast<uintptr_t>(base) % 16 == 0 && page % 16 == 0 && head % 16 == 0 && slot == 1;
  };
  p.scale16 = fp8 && lined_up(p.c.ks, p.c.ks_page, p.c.ks_head, p.c.ks_slot) && lined_up(p.c.vs, p.c.vs_page, p.c.vs_head, p.c.vs_slot);
  CUtensorMap mk{}, mv{};
  auto maps = [&](int box, bool swizzle) {
    const int es = fp8 ? 1 : 2;
    const int64_t ks[3] = {p.c.k_page, p.c.k_head, p.c.k_slot}, vs[3] = {p.c.v_page, p.c.v_head, p.c.v_slot};
    return p.c.pages > 0 && make_paged_map(&mk, p.c.k, p.c.head_dim, es, p.c.page_size, p.c.kv_heads, p.c.pages, ks, box, swizzle) &&
           make_paged_map(&mv, p.c.v, p.c.head_dim, es, p.c.page_size, p.c.kv_heads, p.c.pages, vs, box, swizzle);
  };
  if (plan.many) {
    use(plan.m);
    p.row_min = plan.few ? plan.f.row_max : 0;
    p.row_max = INT32_MAX;
    // the tile kernel takes the maximum of unscaled scores: a positive scale (1e-30 for 0), the sign goes to q
    p.negate = scale_log2 < 0.f;
    p.scale_log2 = fmaxf(fabsf(scale_log2), 1e-30f);
    // boxes of rows that share a page, at most a loader warp's 32 and at least the 8 of a swizzle atom
    int box = 32;
    while (p.c.page_size % box) box /= 2;
    p.box = box >= 8 && maps(box, !fp8) ? box : 0;
    // queries: a stream's 128 rows are a box of whole tokens where the group divides them
    CUtensorMap mq{};
    const int64_t qs[3] = {p.q_tok * a.kv.tokens, p.q_tok, p.q_head};
    p.q_box = 128 % p.group == 0 && make_paged_map(&mq, a.q, p.c.head_dim, 2, a.heads, a.kv.tokens, 1, qs, p.group, true, 128 / p.group);
    const cudaError_t e = f16 ? attn_tiles_launch_f16(p, mk, mv, mq, fp8, plan.m.ctas, pdl_on(), s)
                              : attn_tiles_launch_bf16(p, mk, mv, mq, fp8, plan.m.ctas, pdl_on(), s);
    if (e != cudaSuccess) return e;
  }
  const AttnDev many = p;
  if (plan.few) {
    use(plan.f);
    p.row_min = 0;
    p.row_max = plan.f.row_max;
    p.negate = 0;
    p.scale_log2 = scale_log2;
    p.box = p.c.page_size % 16 == 0 && maps(16, true) ? 16 : 0;  // a warp's 16 keys
    const int blocks = plan.f.rows / 8;
    const bool early = plan.many || pdl_on();  // behind the tile kernel the launch overlaps its end; the kernel waits for it
    const cudaError_t e = f16 ? attn_rows_launch_f16(p, mk, mv, fp8, blocks, plan.f.ctas, early, s)
                              : attn_rows_launch_bf16(p, mk, mv, fp8, blocks, plan.f.ctas, early, s);
    if (e != cudaSuccess) return e;
  }
  return attn_combine_launch(plan.many ? many : p, p, f16, plan.many ? plan.m.ctas : 0, plan.few ? plan.f.ctas : 0, plan.few ? plan.f.rows : 0, s);
}

}  // namespace llg
