// What the cache writer, the cache reader and the attention kernels share: the device view of a paged key/value cache and the
// split of a ragged attention problem into equal shares of key tiles.
//
// Cache rows: token j of sequence i is row (page_table[i, j / page_size], head, j % page_size) of k and v. Page, head and slot
// strides are 64-bit byte offsets. An e4m3 cache holds beside each row of head_dim values one e8m0 byte b, the row's power of
// two 2^(b - 127): e4m3 has the same relative step at every scale inside its normal range, so a power of two loses nothing
// against an amax / 448 scale, and value * 2^(b - 127) is exact in bf16 and fp32.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "llg_internal.h"
#include "ptx_sm100.cuh"

namespace llg {

struct PagedKV {
  unsigned char *k, *v;
  int64_t k_page, k_head, k_slot, v_page, v_head, v_slot;          // bytes
  unsigned char *ks, *vs;
  int64_t ks_page, ks_head, ks_slot, vs_page, vs_head, vs_slot;    // bytes
  const int* table;
  int64_t table_stride;
  const int* lens;
  const int* starts;  // or null: every sequence has q_len new tokens
  int pages, kv_heads, page_size, head_dim, table_width, batch, tokens, q_len;
  int page_shift;     // log2 of a page size that is a power of two, else -1
  unsigned* status;
};

struct SeqView {
  int t0, n;       // first row of its new tokens in q / k / v, their number
  int pos;         // position of the first one: the length as it is given, less n
  int len;         // tokens that the cache holds: no more than the page table can name
};

// Offsets that point outside the call's tensors are cut to them. Tokens behind the end of the page table are not in the cache, but
// the new ones before them stand where they would without that end.
__device__ __forceinline__ SeqView seq_view(const PagedKV& c, int i) {
  SeqView s;
  if (c.starts) {
    s.t0 = min(max(c.starts[i], 0), c.tokens);
    s.n = min(max(c.starts[i + 1], s.t0), c.tokens) - s.t0;
  } else {
    s.t0 = i * c.q_len;
    s.n = c.q_len;
  }
  const int len = max(c.lens[i], 0);
  s.pos = len - s.n;
  s.len = (int)min((int64_t)len, (int64_t)c.table_width * c.page_size);
  return s;
}

// Block (index into the page table's row) and slot of token j.
__device__ __forceinline__ void split_key(const PagedKV& c, int j, int& block, int& slot) {
  if (c.page_shift >= 0) {
    block = j >> c.page_shift;
    slot = j & (c.page_size - 1);
  } else {
    block = j / c.page_size;
    slot = j - block * c.page_size;
  }
}

// Page of token j, or -1 (recorded in the status word) when the table's entry names no page of the cache.
__device__ __forceinline__ int page_of(const PagedKV& c, int seq, int block) {
  const int pg = c.table[(int64_t)seq * c.table_stride + block];
  if ((unsigned)pg < (unsigned)c.pages) return pg;
  atomicCAS(c.status, 0u, (unsigned)ST_BAD_PAGE);
  return -1;
}

// 2^(b - 127), NaN for 255.
__device__ __forceinline__ float e8m0_value(uint32_t b) {
  return __uint_as_float(b == 0u ? 0x00400000u : b == 255u ? 0x7fffffffu : b << 23);
}

__device__ __forceinline__ float least_of_both(float a, float b) {  // NaN if either is
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// A product of two factors, no larger than the largest float (a product of 0 with it stays 0).
__device__ __forceinline__ float finite_product(float a, float b) { return least_of_both(a * b, 3.40282347e38f); }

// Two of them at a time by one conversion (selects for 0 and 255 cost the few-row kernel 1.5 us of 66).
__device__ __forceinline__ void e8m0_values(uint32_t b0, uint32_t b1, float& f0, float& f1) {
  uint32_t r;
  asm("cvt.rn.bf16x2.ue8m0x2 %0, %1;" : "=r"(r) : "h"((uint16_t)(b0 | b1 << 8)));
  f0 = __uint_as_float(r << 16);
  f1 = __uint_as_float(r & 0xffff0000u);
}
// Probabilities carry the power of two of V's row, 2^(score + e - m): its byte as carried (255, no number, is the values' affair), e, and
// 2^-e, which takes it out of the row sum again. That the sum adds up the very exponentials that the values are multiplied with is
// what keeps them in step where a large score swallows e.
__device__ __forceinline__ uint32_t carried(uint32_t b, uint32_t least) { return b == 255u ? least : max(b, least); }
__device__ __forceinline__ float power_of(uint32_t c) { return __uint_as_float(0x4b000000u + c) - 8388735.f; }  // bits of 2^23 + c, less 2^23 + 127
__device__ __forceinline__ float power_out(uint32_t c) { return __uint_as_float(c == 254u ? 0x00400000u : (254u - c) << 23); }

// ---- attention ---------------------------------------------------------------------------------------------------
// Rows of a sequence are packed token-major over the query heads that share a key/value head: row = token * group + head in
// group. An item is (sequence, kv head, tile of whole tokens); it walks the key tiles that any of its rows sees. All items'
// key tiles, counted through, are cut into equal shares, one per CTA: every CTA streams the same number of tiles whatever the
// lengths are. An item that a share boundary cuts leaves one partial result per CTA (unnormalised sums in fp32, row maximum,
// row sum); attn_combine_kernel adds them in order of the CTAs, so results do not depend on timing.
struct AttnDev {
  PagedKV c;
  const unsigned char* q;
  int64_t q_tok, q_head;  // bytes
  unsigned char* out;
  int64_t o_tok, o_head;  // bytes
  float* lse;
  int64_t lse_tok;        // elements; heads are contiguous
  int group;              // query heads per kv head
  int causal, window;
  float scale_log2;       // softmax scale * log2(e); its magnitude in the tile kernel ...
  int negate;             // ... which turns the signs of q around for a negative scale
  int row_min, row_max;   // this launch serves sequences with row_min < new tokens * group <= row_max
  int scale16;            // 16 scale bytes of a page from a multiple of 16 on lie together, 16-byte aligned
  int tok_tile;           // whole tokens per row tile
  int box;                // rows of a TMA box (16, or a divisor of 32 and of the page size in the tile kernel), 0: no tensor maps
  int q_box;              // tile kernel: queries by TMA, 128 rows to a box
  float* part_o;          // [slots][rows per tile][head_dim]; tile kernel: [slots][head_dim / 4][256 rows][4]
  float* part_ml;         // [slots][rows per tile][2]: maximum (log2 domain), sum
  int4* split;            // [CTAs][2]: the cut item that goes on at the beginning of a CTA's share, and the one that starts at its
                          // end: {CTAs that share it (0: none), first token, kv head, rows}; 1 << 16 in the last: every CTA left
                          // two parts, the second 128 rows behind the first
  int* first;             // [CTAs]: the CTA in which the item that goes on started
};

// Probabilities are 2^(score - m) with m kHead below the largest score that moved it, and m moves when a score exceeds it by 2^15: the
// largest of a row lies between 2^7 and 2^15. f16 ends at 2^15.99 and, with full accuracy, at 2^-14, so keys down to 2^-21 of the
// largest keep their bits and keys down to 2^-32 are counted (a largest probability of 1 to 2^8 lost 131k keys 2^-25.3 below one).
constexpr float kHead = 7.f, kMove = 15.f;
// Least power of two of a row of V (biased by 127) that the probabilities carry: row sums, up to 2^(15 + 88) a key, stay in fp32. What
// smaller rows have below it stays with their values.
constexpr uint32_t kLeastV = 39;
// Scores of 2^22 and more have a last bit of half a power of two and more: there products are rounded before m, which was, is taken off
// (a multiply-add would be off by powers of two, and f16 ends from scores of 2^27 on).
constexpr float kHuge = 4194304.f;

// CTAs of the few-row kernel that fit an SM: as many as its registers and rings of two to three tiles let in, which hides the chain
// from a load to the next product better than longer rings (8 rows, decode batch over e4m3: two 74.5 us, three 65.3; 16-bit 51.8, 50.4;
// 20 rows of 64 values: two of 32 rows 32.9, three of 24 29.4). Not where registers would spill: 16 rows of 128 e4m3 values three 39.1, two 36.3.
__host__ __device__ constexpr int rows_ctas_per_sm(bool fp8, int head_dim, int blocks) {
  return blocks == 4 ? 2 : blocks == 3 ? (head_dim == 64 ? 3 : 2) : blocks == 2 ? (head_dim == 64 ? 3 : 2) : fp8 || head_dim == 128 ? 3 : 4;
}

// Keys [lo, hi) that any row of token tile [tf, tf + cnt) sees.
struct KeyRange {
  int lo, hi;
};
__device__ __forceinline__ KeyRange key_range(const AttnDev& p, const SeqView& s, int tf, int cnt) {
  KeyRange r;
  r.hi = p.causal ? min(max(s.pos + tf + cnt, 0), s.len) : s.len;
  r.lo = p.window > 0 ? max(s.pos + tf + 1 - p.window, 0) : 0;
  r.lo = min(r.lo, r.hi);
  return r;
}
template <int KT>
__device__ __forceinline__ int key_tiles(const KeyRange& r) {
  return max((r.hi + KT - 1) / KT - r.lo / KT, 1);  // an item without keys still writes its rows
}

__device__ __forceinline__ int token_tiles(const AttnDev& p, const SeqView& s) {
  const int64_t rows = (int64_t)s.n * p.group;
  return rows > p.row_min && rows <= p.row_max ? (s.n + p.tok_tile - 1) / p.tok_tile : 0;
}

// Key tiles of token tile r.
template <int KT>
__device__ __forceinline__ int tile_units(const AttnDev& p, const SeqView& s, int r) {
  const int tf = r * p.tok_tile;
  return key_tiles<KT>(key_range(p, s, tf, min(p.tok_tile, s.n - tf)));
}

// Key tiles of one kv head of a sequence, over all of its token tiles, by one thread or by a warp. (The host refuses calls whose
// key tiles might not fit 31 bits: 64-bit divisions in every CTA's start cost a microsecond.)
template <int KT>
__device__ __forceinline__ int seq_units(const AttnDev& p, const SeqView& s) {
  int u = 0;
  const int nt = token_tiles(p, s);
  for (int r = 0; r < nt; ++r) u += tile_units<KT>(p, s, r);
  return u;
}
template <int KT>
__device__ __forceinline__ int seq_units_warp(const AttnDev& p, const SeqView& s) {
  const int nt = token_tiles(p, s);
  if (nt <= 1) return nt == 0 ? 0 : tile_units<KT>(p, s, 0);
  int u = 0;
  for (int r = threadIdx.x & 31; r < nt; r += 32) u += tile_units<KT>(p, s, r);
  return __reduce_add_sync(0xffffffffu, u);
}

// A CTA's share of the key tiles and its place in the walk.
struct Share {
  int u, end, per;  // next unit, end of the share, units per CTA
  int seq, off;     // units of `seq` (over all kv heads) before u
  int known;        // sequence whose units of one kv head `per_head` holds
  int per_head;
};

// Every thread of the CTA takes part. scratch: NT / 32 + 2 ints of shared memory. Up to NT / 32 sequences are counted by a warp each
// (a prompt chunk has many tiles), more by a thread each.
template <int KT, int NT>
__device__ __forceinline__ Share find_share(const AttnDev& p, int* scratch) {
  constexpr int W = NT / 32;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int* const part = scratch;       // warp sums
  int* const found = scratch + W;  // {seq, units before u}
  // one prefix sum over the first NT sequences, and the total of all
  int x = 0, rest = 0;
  if (p.c.batch <= W) {
    if (warp < p.c.batch) {
      const int u = seq_units_warp<KT>(p, seq_view(p.c, warp)) * p.c.kv_heads;
      if (lane == 0) part[warp] = u;
    }
    __syncthreads();
    if (tid < p.c.batch) x = part[tid];
    __syncthreads();
  } else {
    for (int i = tid; i < p.c.batch; i += NT) {
      const int u = seq_units<KT>(p, seq_view(p.c, i)) * p.c.kv_heads;
      if (i == tid) x = u;
      else rest += u;
    }
  }
  int inc = x;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += y;
  }
  if (lane == 31) part[warp] = inc;
  const int beyond = p.c.batch > NT ? __syncthreads_or(rest != 0) : (__syncthreads(), 0);
  int before = 0, chunk = 0;
#pragma unroll
  for (int w = 0; w < W; ++w) {
    if (w < warp) before += part[w];
    chunk += part[w];
  }
  int total = chunk;
  if (beyond) {  // more sequences than threads
    __syncthreads();
    if (tid == 0) found[0] = 0;
    __syncthreads();
    atomicAdd(&found[0], rest);
    __syncthreads();
    total += found[0];
  }
  Share sh;
  sh.per = (total + (int)gridDim.x - 1) / (int)gridDim.x;
  sh.u = sh.per * (int)blockIdx.x;
  sh.end = min(total, sh.u + sh.per);
  sh.known = -1;
  sh.per_head = sh.seq = sh.off = 0;
  if (sh.u >= sh.end) return sh;
  __syncthreads();
  int base = 0;
  for (int c0 = 0;; c0 += NT) {
    const int lo = base + before + inc - x;
    if (x > 0 && lo <= sh.u && sh.u < lo + x) {
      found[0] = c0 + tid;
      found[1] = sh.u - lo;
    }
    if (sh.u < base + chunk || c0 + NT >= p.c.batch) break;
    // not among these: the next NT sequences
    base += chunk;
    const int i = c0 + NT + tid;
    x = i < p.c.batch ? seq_units<KT>(p, seq_view(p.c, i)) * p.c.kv_heads : 0;
    inc = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += y;
    }
    __syncthreads();
    if (lane == 31) part[warp] = inc;
    __syncthreads();
    before = chunk = 0;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      if (w < warp) before += part[w];
      chunk += part[w];
    }
  }
  __syncthreads();
  sh.seq = found[0];
  sh.off = found[1];
  return sh;
}

// The next piece of the walk: key tiles [tile0, tile1) of one item.
struct Segment {
  int seq, head, tok0, toks;   // sequence, kv head, first token within the sequence's new ones, tokens
  SeqView s;
  KeyRange keys;
  int tile0, tile1;            // key tiles, counted from key 0
  bool starts, whole;          // the segment begins its item / is all of it
  int first, parts;            // the item's first CTA, and how many share it
};

// Whole warps take part.
template <int KT>
__device__ __forceinline__ bool next_segment(const AttnDev& p, Share& sh, Segment& g) {
  if (sh.u >= sh.end) return false;
  int per_head;
  for (;;) {
    if (sh.seq >= p.c.batch) return false;
    g.s = seq_view(p.c, sh.seq);
    if (sh.known != sh.seq) {
      sh.per_head = seq_units_warp<KT>(p, g.s);
      sh.known = sh.seq;
    }
    per_head = sh.per_head;
    if (per_head > 0) break;
    ++sh.seq;  // nothing of this sequence belongs to this launch
    sh.off = 0;
  }
  g.seq = sh.seq;
  g.head = sh.off / per_head;
  int rem = sh.off - g.head * per_head;
  int tile = 0;
  const int nt = token_tiles(p, g.s);
  if (nt > 1) {  // 32 token tiles at a time
    const int lane = threadIdx.x & 31;
    for (int r0 = 0;; r0 += 32) {
      const int x = r0 + lane < nt ? tile_units<KT>(p, g.s, r0 + lane) : 0;
      int inc = x;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += y;
      }
      const uint32_t hit = __ballot_sync(0xffffffffu, rem < inc);
      if (hit != 0u || r0 + 32 >= nt) {
        const int at = hit ? __ffs(hit) - 1 : min(31, nt - 1 - r0);
        rem -= __shfl_sync(0xffffffffu, inc - x, at);
        tile = r0 + at;
        break;
      }
      rem -= __shfl_sync(0xffffffffu, inc, 31);
    }
  }
  g.tok0 = tile * p.tok_tile;
  g.toks = min(p.tok_tile, g.s.n - g.tok0);
  g.keys = key_range(p, g.s, g.tok0, g.toks);
  const int units = key_tiles<KT>(g.keys);
  const int take = min(units - rem, sh.end - sh.u);
  g.tile0 = g.keys.lo / KT + rem;
  g.tile1 = g.tile0 + take;
  g.starts = rem == 0;
  g.whole = g.starts && take == units;
  g.first = g.parts = 0;
  if (!g.whole) {
    g.first = (sh.u - rem) / sh.per;
    g.parts = (sh.u - rem + units - 1) / sh.per - g.first + 1;
  }
  sh.u += take;
  sh.off += take;
  if (sh.off == per_head * p.c.kv_heads) {
    ++sh.seq;
    sh.off = 0;
  }
  return true;
}

// Notes a cut item for the kernel that adds its parts up. One thread.
__device__ __forceinline__ void note_split(const AttnDev& p, const Segment& g, int rows) {
  p.split[2 * blockIdx.x + (g.starts ? 1 : 0)] = make_int4(g.parts, g.s.t0 + g.tok0, g.head, rows);
  if (!g.starts) p.first[blockIdx.x] = g.first;
}
__device__ __forceinline__ void clear_splits(const AttnDev& p) {
  p.split[2 * blockIdx.x] = p.split[2 * blockIdx.x + 1] = make_int4(0, 0, 0, 0);
}

// A cut item's part of this CTA: slot 1 when the CTA begins the item (at the end of its share), else slot 0.
__device__ __forceinline__ int part_slot(int cta, bool starts) { return 2 * cta + (starts ? 1 : 0); }

}  // namespace llg
