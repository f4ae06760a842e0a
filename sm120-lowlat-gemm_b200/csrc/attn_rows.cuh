// Attention of few query rows per key/value head over a paged cache (one token, drafted tokens): bound by the bytes of K and V.
//
//   s = scale * q . k,  m = max s,  l = sum exp(s - m),  o = sum exp(s - m) v / l       one pass, running m, l and o
//
// Key tiles of 64 tokens (128: e4m3, up to 8 rows, which halves what is spent per key beside the products); each of the CTA's four
// warps owns 16 (32) of them with its own ring of stages, softmax state and accumulators, so nothing between the loads and the last
// merge synchronises more than a warp. Sixteen rows that are all there and share a page come by TMA, swizzled; others are gathered
// with cp.async, zeros for the missing. The products are taken transposed, S^T[16 keys x rows] = K Q^T and
// O^T[head_dim x rows] = V^T P^T, so that the rows - 8 for a group of eight heads and one token - are the narrow side (8) of
// mma.m16n8k16 and no row of the tensor-core tile is padding.
//   16-bit cache: K by ldmatrix, V by ldmatrix.trans.
//   e4m3 cache: 16-byte reads of a row give a thread 16 neighbouring values; the order of head_dim inside a product is free, so
//     they serve four consecutive k steps of K Q^T (Q is read in the same order) and eight row blocks of V^T without any
//     transposition, and so are the orders of the keys and of head_dim's blocks among the lanes, which keep the reads of the
//     TMA's swizzle free of bank conflicts. One cvt makes two f16 of two values, exactly, so both products run in f16 whatever q's
//     type is: a bf16 row of q is brought to f16 by a power of two (its largest value to 2^14; values 2^-28 below that and less
//     lose bits). The scores take the powers of two of q's and K's rows in fp32; V's goes to the probability, 2^(s + e - m) with m
//     following the maximum of s + e, which is at most 2^15 and keeps f16's 11 bits where it matters; l takes it times 2^-e.
// P is rounded to the operand type of the second product (bf16 2^-8, f16 2^-11 relative); l sums the unrounded fp32 values.
// Measured: 32 sequences of 0.9k to 8.2k keys, 64 heads over 8, e4m3, 65.7 us (4.4 TB/s); 4 of 50k to 65k, bf16, 50.4 us (5.2 TB/s).
// m moves only when a score exceeds the largest so far by more than 2^8, so the shuffles and the rescaling of O are skipped for almost
// every tile; kHead, kMove: where p lies.
#pragma once

#include <climits>
#include <type_traits>

#include "paged_kv.cuh"

namespace llg {

constexpr int kRowsWarps = 4;
constexpr int kRowsThreads = 32 * kRowsWarps;

// Box of a page: x = element, then slot, head, page.
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* m, uint32_t bar, int x, int slot, int head, int page) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst),
      "l"(m), "r"(bar), "r"(x), "r"(slot), "r"(head), "r"(page)
      : "memory");
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ void ldsm_x4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm_x4_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ uint4 lds16(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ uint2 lds8(uint32_t addr) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <typename T>
struct Mma;
template <>
struct Mma<__nv_bfloat16> {
  static __device__ __forceinline__ void run(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
  }
};
template <>
struct Mma<__half> {
  static __device__ __forceinline__ void run(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
  }
};

// e4m3 bytes as pairs of f16, which holds every one of their values.
__device__ __forceinline__ uint32_t widen2(uint32_t v) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((uint16_t)v));
  return r;
}
__device__ __forceinline__ void widen4(uint32_t w, uint32_t& lo, uint32_t& hi) {
  lo = widen2(w & 0xffffu);
  hi = widen2(w >> 16);
}
// (a.b0, b.b0) (a.b1, b.b1) (a.b2, b.b2) (a.b3, b.b3)
__device__ __forceinline__ void widen_cross(uint32_t a, uint32_t b, uint32_t (&o)[4]) {
  const uint32_t x = __byte_perm(a, b, 0x5140), y = __byte_perm(a, b, 0x7362);
  o[0] = widen2(x & 0xffffu);
  o[1] = widen2(x >> 16);
  o[2] = widen2(y & 0xffffu);
  o[3] = widen2(y >> 16);
}

__device__ __forceinline__ float pow2_of(uint32_t biased) { return __uint_as_float(biased << 23); }

template <typename T, bool FP8, int D, int NB>
struct RowsCfg {
  using Op = typename std::conditional<FP8, __half, T>::type;   // operand type of the products
  static constexpr int kCtas = rows_ctas_per_sm(FP8, D, NB);
  static constexpr int kRowBytes = D * (FP8 ? 1 : 2);
  static constexpr int kChunks = kRowBytes / 16;      // 16-byte pieces per row
  static constexpr int kParts = kRowBytes > 128 ? 2 : 1;            // a row lies in pieces of at most 128 bytes ...
  static constexpr int kPitch = kRowBytes / kParts;                 // ... of this size, 16 rows of a piece together
  static constexpr int kSub = FP8 && NB == 1 ? 2 : 1; // groups of 16 keys per warp and tile
  static constexpr int kKeys = 16 * kSub * kRowsWarps;
  static constexpr int kGroup = 2 * 16 * kRowBytes;   // bytes of a group: K, V
  static constexpr int kStage = kSub * kGroup;        // per warp
  static constexpr int kStages = [] {
    const int n = (226 * 1024 / kCtas - 4096) / kRowsWarps / (kStage + 32 * kSub);
    return n > 8 ? 8 : n;
  }();
  static constexpr int kRing = kStages * kStage;      // per warp
  static constexpr int kRows = NB * 8;
  static constexpr int kPad = D + 4;                  // floats between rows of the merge buffer
  static constexpr int kMerge = kRowsWarps * kRows * (kPad + 2) * 4;
  static constexpr int kSmem = (kRowsWarps * kRing > kMerge ? kRowsWarps * kRing : kMerge) + 1024;  // + alignment slack
};

// Place of 16-byte piece `ch` of row `row` (< 16) of K or V in a stage: what the TMA's swizzle makes of it.
template <typename Cfg>
__device__ __forceinline__ uint32_t rows_at(int row, int ch) {
  if constexpr (Cfg::kPitch == 128) return (ch >> 3) * 2048 + row * 128 + (((ch & 7) ^ (row & 7)) << 4);
  else return row * 64 + ((ch ^ ((row >> 1) & 3)) << 4);
}

template <typename T, bool FP8, int D, int NB>
__global__ void __launch_bounds__(kRowsThreads, (RowsCfg<T, FP8, D, NB>::kCtas))
    attn_rows_kernel(const __grid_constant__ AttnDev p, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v) {
  using Cfg = RowsCfg<T, FP8, D, NB>;
  using Op = typename Cfg::Op;
  constexpr bool kToF16 = FP8 && std::is_same<T, __nv_bfloat16>::value;
  constexpr int KT = Cfg::kKeys, SUB = Cfg::kSub;
  constexpr int S = Cfg::kStages, CH = Cfg::kChunks, KS = D / 16, MB = D / 16;
  extern __shared__ unsigned char smem_raw[];
  __shared__ int scratch[kRowsWarps + 2];
  __shared__ __align__(8) unsigned long long bars[kRowsWarps * S];
  __shared__ __align__(16) unsigned char scales[FP8 ? kRowsWarps * S * 32 * Cfg::kSub : 1];
  __shared__ volatile uint32_t abort_word;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int quad = lane & 3, oct = lane >> 2;  // fragment coordinates
  // e4m3, 128-byte rows: which key a fragment's row `oct` is, and which 16 values of head_dim a lane's V fragments hold
  constexpr bool kMixed = FP8 && D == 128;
  const int krow = kMixed ? (oct >> 1) + 4 * (oct & 1) : oct;
  const int vrow0 = kMixed ? quad : 2 * quad, vrow1 = kMixed ? quad + 4 : 2 * quad + 1;  // keys of k steps 2 quad, 2 quad + 1
  unsigned char* const smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  if (tid < kRowsWarps * S) {
    mbar_init(smem_u32(&bars[tid]), 32);
    mbar_fence_init();
  }
  if (tid == 0) {
    abort_word = 0u;
    tma_prefetch_desc(&map_k);
    tma_prefetch_desc(&map_v);
  }
  pdl_trigger();
  pdl_wait();
  if (tid == 0) clear_splits(p);
  Share share = find_share<KT, kRowsThreads>(p, scratch);
  const uint32_t ring = smem_u32(smem) + warp * Cfg::kRing, bar = smem_u32(&bars[warp * S]);
  const uint32_t scale_at = smem_u32(scales) + warp * S * 32 * SUB;
  int put = 0, get = 0;         // stages filled next / read next
  uint32_t get_phase = 0;
  bool gathered = false;        // copies of cp.async went into the ring since the last proxy fence
  bool ok_all = true;
  const PagedKV& c = p.c;
  // row / group for rows of a tile: exact while row * group < 2^16
  const uint32_t group_inv = (65535u + p.group) / p.group;
  auto token_of = [&](int row) { return (int)((uint32_t)row * group_inv >> 16); };
  const bool one_page = c.page_size % 16 == 0;  // 16 keys from a multiple of 16 on share a page

  Segment g;
  while (next_segment<KT>(p, share, g)) {
    const int rows = g.toks * p.group;
    const int nb_used = (rows + 7) >> 3;
    const int pos0 = g.s.pos + g.tok0;  // position of the tile's first token

    // ---- the warp's ring: tile t holds the warp's groups of 16 keys, from key_of(t) on
    const int nt = g.tile1 - g.tile0;
    const int head = g.head;
    const int* const table_row = c.table + (int64_t)g.seq * c.table_stride;
    // keys that every row of the tile sees: tiles inside need no mask
    const int all_hi = p.causal ? min(pos0, g.s.len - 1) : g.s.len - 1;
    const int all_lo = p.window > 0 ? pos0 + g.toks - p.window : 0;
    auto key_of = [&](int t) { return (g.tile0 + t) * KT + warp * (16 * SUB); };
    // Where 16 keys from a multiple of 16 on share a page: page table entries of the warp's next 32 groups, one per lane, and of the
    // 32 behind them, on their way. A request per tile would make a chain of them: filling a ring of seven stages took 3 us.
    constexpr int kLook = 32 / SUB;             // tiles
    auto look_up = [&](int t0) {
      const int t = t0 + lane / SUB, k0 = key_of(t) + 16 * (lane % SUB);
      int block, slot;
      split_key(c, k0, block, slot);
      return t < nt && k0 < g.keys.hi && k0 + 16 > g.keys.lo ? table_row[block] : INT_MIN;
    };
    int entries = INT_MIN, ahead = INT_MIN;
    if (one_page) {
      entries = look_up(0);
      ahead = look_up(kLook);
    }
    // the tile located last: the lane's group (lane % SUB), its page (-1: none) and first slot; tiles are located in order
    const int sub = lane % SUB;
    int pg = -1, at = 0;
    auto locate = [&](int t) {
      if (!one_page) return;
      if (t % kLook == 0 && t > 0) {
        entries = ahead;
        ahead = look_up(t + kLook);
      }
      int block;
      split_key(c, key_of(t) + 16 * sub, block, at);
      pg = __shfl_sync(0xffffffffu, entries, t % kLook * SUB + sub);
      if ((unsigned)pg >= (unsigned)c.pages) {
        if (pg != INT_MIN) atomicCAS(c.status, 0u, (unsigned)ST_BAD_PAGE);
        pg = -1;
      }
    };

    // ---- queries: B fragments of K Q^T, row oct of each block; requested before the ring is filled
    uint32_t qf[NB][KS][2];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      const int row = nb * 8 + oct;
      const int tok = token_of(row), hh = row - tok * p.group;
      const unsigned char* src = p.q + (int64_t)(g.s.t0 + g.tok0 + tok) * p.q_tok + (int64_t)(g.head * p.group + hh) * p.q_head;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        uint2 v = make_uint2(0u, 0u);
        if (row < rows) {
          if constexpr (FP8) {  // the order in which a thread holds a row of K: 16 * (quad + 4 i) + 4 j
            const int i = ks >> 2, j = ks & 3;
            v = *reinterpret_cast<const uint2*>(src + 2 * (16 * (quad + 4 * i) + 4 * j));
          } else {
            v.x = *reinterpret_cast<const uint32_t*>(src + 2 * (16 * ks + 2 * quad));
            v.y = *reinterpret_cast<const uint32_t*>(src + 2 * (16 * ks + 2 * quad + 8));
          }
        }
        qf[nb][ks][0] = v.x;
        qf[nb][ks][1] = v.y;
      }
    }
    const bool by_tma = one_page && p.box != 0;
    auto issue = [&](int t) {  // starts the copies of tile t, located by the call before, into stage `put`
      if (t >= nt) return;
      const uint32_t dst = ring + put * Cfg::kStage, full = bar + 8u * put, sdst = scale_at + put * 32 * SUB;
      const int k0 = key_of(t);
      if (by_tma && k0 >= g.keys.lo && k0 + 16 * SUB <= g.keys.hi && __all_sync(0xffffffffu, pg >= 0)) {
        if (gathered) {
          fence_async_shared();
          __syncwarp();
          gathered = false;
        }
        if (FP8 && !p.scale16) {  // scale bytes that do not lie together: one per lane
          for (int q = 0; q < SUB; ++q) {
            const int64_t x = __shfl_sync(0xffffffffu, pg, q), y = __shfl_sync(0xffffffffu, at, q) + (lane & 15);
            const uint32_t v = lane < 16 ? c.ks[x * c.ks_page + head * c.ks_head + y * c.ks_slot] : c.vs[x * c.vs_page + head * c.vs_head + y * c.vs_slot];
            asm volatile("st.shared.u8 [%0], %1;" ::"r"(sdst + q * 32 + lane), "r"(v) : "memory");
          }
        }
        if (lane < SUB) {
          mbar_expect_tx(full, Cfg::kGroup);
#pragma unroll
          for (int h = 0; h < Cfg::kParts; ++h) {
            tma_load_4d(dst + sub * Cfg::kGroup + h * 2048, &map_k, full, h * 64, at, head, pg);
            tma_load_4d(dst + sub * Cfg::kGroup + 16 * Cfg::kRowBytes + h * 2048, &map_v, full, h * 64, at, head, pg);
          }
        } else if (FP8 && p.scale16 && lane < 3 * SUB) {  // a group's 16 scale bytes of K, of V
          const bool is_v = lane >= 2 * SUB;
          cp_async16(sdst + sub * 32 + (is_v ? 16 : 0), is_v ? c.vs + pg * c.vs_page + head * c.vs_head + at : c.ks + pg * c.ks_page + head * c.ks_head + at, 16u);
          cp_async_arrive_noinc(full);
        } else {
          mbar_arrive(full);
        }
      } else {
        // row by row, zeros for rows that are not there; lanes 0-15: rows of K, 16-31: of V
        const bool is_v = lane >= 16;
#pragma unroll 1
        for (int q = 0; q < SUB; ++q) {
          const int key = k0 + 16 * q + (lane & 15);
          int64_t page = -1, slot = 0;
          if (one_page) {
            const int x = __shfl_sync(0xffffffffu, pg, q), y = __shfl_sync(0xffffffffu, at, q);
            if (key >= g.keys.lo && key < g.keys.hi) page = x;
            slot = y + (lane & 15);
          } else if (key >= g.keys.lo && key < g.keys.hi) {
            int block, y;
            split_key(c, key, block, y);
            page = page_of(c, g.seq, block);
            slot = y;
          }
          int64_t off = -1;
          uint32_t scale = 0u;
          if (page >= 0) {
            off = is_v ? page * c.v_page + head * c.v_head + slot * c.v_slot : page * c.k_page + head * c.k_head + slot * c.k_slot;
            if constexpr (FP8)
              scale = is_v ? c.vs[page * c.vs_page + head * c.vs_head + slot * c.vs_slot] : c.ks[page * c.ks_page + head * c.ks_head + slot * c.ks_slot];
          }
#pragma unroll 2
          for (int i = 0; i < CH / 2; ++i) {
            const int row = lane / CH + i * (32 / CH), ch = lane % CH;
            const int64_t ko = __shfl_sync(0xffffffffu, off, row), vo = __shfl_sync(0xffffffffu, off, 16 + row);
            const uint32_t to = dst + q * Cfg::kGroup + rows_at<Cfg>(row, ch);
            cp_async16(to, c.k + (ko >= 0 ? ko + ch * 16 : 0), ko >= 0 ? 16u : 0u);
            cp_async16(to + 16 * Cfg::kRowBytes, c.v + (vo >= 0 ? vo + ch * 16 : 0), vo >= 0 ? 16u : 0u);
          }
          if constexpr (FP8) asm volatile("st.shared.u8 [%0], %1;" ::"r"(sdst + q * 32 + lane), "r"(scale) : "memory");
        }
        cp_async_arrive_noinc(full);
        gathered = true;
      }
      put = put + 1 == S ? 0 : put + 1;
    };
#pragma unroll 1
    for (int t = 0; t < S - 1; ++t) {
      locate(t);
      issue(t);
    }
    locate(S - 1);

    // ---- what the rows see, and bf16 queries to f16
    float row_f[NB][2];                     // what turns a product of those rows into log2 units
    int first_key[NB][2], last_key[NB][2];  // keys that rows 2 * quad, 2 * quad + 1 of a block see: [first, last]
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      float mine = p.scale_log2;              // of row oct
      if constexpr (kToF16) {
        float top = 0.f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float2 f = __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&qf[nb][ks][h]));
            top = fmaxf(top, fmaxf(fabsf(f.x), fabsf(f.y)));
          }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const uint32_t e = max(__float_as_uint(top) >> 23, 20u);
        const float up = __uint_as_float((268u - e) << 23);  // 2^(14 - exponent of the row's largest value)
        mine *= __uint_as_float((e - 14u) << 23);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float2 f = __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&qf[nb][ks][h]));
            qf[nb][ks][h] = Mma<__half>::pack(f.x * up, f.y * up);
          }
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        row_f[nb][e] = __shfl_sync(0xffffffffu, mine, (2 * quad + e) * 4);
        const int r = nb * 8 + 2 * quad + e;
        const int pos = pos0 + token_of(r);
        last_key[nb][e] = r < rows ? (p.causal ? min(pos, g.s.len - 1) : g.s.len - 1) : -1;
        first_key[nb][e] = p.window > 0 ? pos - p.window + 1 : 0;
      }
    }

    float o[NB][MB][4];
    float m[NB][2], l[NB][2];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
      for (int mb = 0; mb < MB; ++mb) o[nb][mb][0] = o[nb][mb][1] = o[nb][mb][2] = o[nb][mb][3] = 0.f;
      m[nb][0] = m[nb][1] = -INFINITY;
      l[nb][0] = l[nb][1] = 0.f;
    }

    for (int t = 0; t < nt; ++t) {
      const uint32_t stage = ring + get * Cfg::kStage, sb = scale_at + get * 32 * SUB;
      if (ok_all && !mbar_wait(bar + 8u * get, get_phase, &abort_word)) {
        ok_all = false;
        atomicCAS(c.status, 0u, (unsigned)ST_CONVERT_WAIT);
      }
      if (++get == S) {
        get = 0;
        get_phase ^= 1u;
      }
      __syncwarp();
      issue(t + S - 1);  // into the stage that the warp finished reading one tile ago

      // ---- S^T = K Q^T: thread holds keys oct, oct + 8 of rows 2 * quad, 2 * quad + 1 of each block
      float s[SUB][NB][4];
#pragma unroll
      for (int u = 0; u < SUB; ++u) {
        const uint32_t kb = stage + u * Cfg::kGroup;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) s[u][nb][0] = s[u][nb][1] = s[u][nb][2] = s[u][nb][3] = 0.f;
        if constexpr (FP8) {
#pragma unroll
          for (int i = 0; i < D / 64; ++i) {
            const int ch = quad + 4 * i;
            const uint4 r0 = lds16(kb + rows_at<Cfg>(krow, ch)), r1 = lds16(kb + rows_at<Cfg>(krow + 8, ch));
            const uint32_t w0[4] = {r0.x, r0.y, r0.z, r0.w}, w1[4] = {r1.x, r1.y, r1.z, r1.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              uint32_t a[4];
              widen4(w0[j], a[0], a[2]);
              widen4(w1[j], a[1], a[3]);
#pragma unroll
              for (int nb = 0; nb < NB; ++nb)
                if (nb < nb_used) Mma<Op>::run(s[u][nb], a, qf[nb][4 * i + j][0], qf[nb][4 * i + j][1]);
            }
          }
        } else {
#pragma unroll
          for (int ks = 0; ks < KS; ++ks) {
            uint32_t a[4];
            const int row = lane & 15, ch = 2 * ks + (lane >> 4);
            ldsm_x4(kb + rows_at<Cfg>(row, ch), a);
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
              if (nb < nb_used) Mma<Op>::run(s[u][nb], a, qf[nb][ks][0], qf[nb][ks][1]);
          }
        }
      }

      // ---- softmax
      const int key0 = key_of(t);
      const bool inner = key0 >= all_lo && key0 + 16 * SUB - 1 <= all_hi;
      float kf[SUB][2], ve[SUB][2], out[SUB][2], left[SUB][2];  // keys krow, krow + 8 of a group: 2^e of K; of V: e, 2^-e, what is left
#pragma unroll
      for (int u = 0; u < SUB; ++u) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          kf[u][e] = out[u][e] = left[u][e] = 1.f;
          ve[u][e] = 0.f;
        }
        if constexpr (FP8) {
          uint32_t bk[2], bv[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            asm volatile("ld.shared.u8 %0, [%1];" : "=r"(bk[e]) : "r"(sb + 32 * u + krow + 8 * e) : "memory");
            asm volatile("ld.shared.u8 %0, [%1];" : "=r"(bv[e]) : "r"(sb + 32 * u + 16 + krow + 8 * e) : "memory");
          }
          e8m0_values(bk[0], bk[1], kf[u][0], kf[u][1]);
          float vf[2];
          e8m0_values(bv[0], bv[1], vf[0], vf[1]);
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const uint32_t c = carried(bv[e], kLeastV);
            ve[u][e] = power_of(c);
            out[u][e] = power_out(c);
            left[u][e] = least_of_both(vf[e] * 0x1p88f, 1.f);  // 2^(127 - kLeastV)
          }
        }
      }
      uint32_t pf[SUB][NB][2];
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        if (nb >= nb_used) continue;
        float x[SUB][4];
        bool more = false;
#pragma unroll
        for (int u = 0; u < SUB; ++u)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if constexpr (FP8) x[u][e] = s[u][nb][e] * finite_product(row_f[nb][e & 1], kf[u][e >> 1]) + ve[u][e >> 1];
            else x[u][e] = s[u][nb][e] * row_f[nb][e & 1];
            if (!inner) {
              const int key = key0 + 16 * u + krow + (e >> 1) * 8;
              if (key > last_key[nb][e & 1] || key < first_key[nb][e & 1]) x[u][e] = -INFINITY;
            }
            more |= x[u][e] > m[nb][e & 1] + kMove;
          }
        if (__any_sync(0xffffffffu, more)) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float mx = -INFINITY;
#pragma unroll
            for (int u = 0; u < SUB; ++u) mx = fmaxf(mx, fmaxf(x[u][e], x[u][e + 2]));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
            const float top = fmaxf(m[nb][e], mx - kHead);
            const float keep = m[nb][e] == -INFINITY ? 0.f : exp2_fast(m[nb][e] - top);
            m[nb][e] = top;
            l[nb][e] *= keep;
#pragma unroll
            for (int mb = 0; mb < MB; ++mb) {
              o[nb][mb][e] *= keep;
              o[nb][mb][e + 2] *= keep;
            }
          }
        }
        const float base[2] = {m[nb][0] == -INFINITY ? 0.f : m[nb][0], m[nb][1] == -INFINITY ? 0.f : m[nb][1]};
#pragma unroll
        for (int u = 0; u < SUB; ++u) {
          float pr[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            pr[e] = exp2_fast(x[u][e] - base[e & 1]);
            if constexpr (FP8) l[nb][e & 1] = fmaf(pr[e], out[u][e >> 1], l[nb][e & 1]);
            else l[nb][e & 1] += pr[e];
          }
          pf[u][nb][0] = transpose8x8(Mma<Op>::pack(pr[0] * left[u][0], pr[1] * left[u][0]));
          pf[u][nb][1] = transpose8x8(Mma<Op>::pack(pr[2] * left[u][1], pr[3] * left[u][1]));
        }
      }

      // ---- O^T += V^T P^T
#pragma unroll
      for (int u = 0; u < SUB; ++u) {
        const uint32_t vb = stage + u * Cfg::kGroup + 16 * Cfg::kRowBytes;
        if constexpr (FP8) {
          constexpr int W = D / 32;  // 4-byte words of a row that a thread holds (of head_dim: 16 * krow + ..., or 8 * oct + ...)
          uint32_t w[4][W];
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int row = ((r & 1) ? vrow1 : vrow0) + (r >> 1) * 8;
            if constexpr (D == 128) {
              const uint4 v = lds16(vb + rows_at<Cfg>(row, krow));
              w[r][0] = v.x; w[r][1] = v.y; w[r][2] = v.z; w[r][3] = v.w;
            } else {
              const uint2 v = lds8(vb + rows_at<Cfg>(row, oct >> 1) + (oct & 1) * 8);
              w[r][0] = v.x; w[r][1] = v.y;
            }
          }
#pragma unroll
          for (int j = 0; j < W; ++j) {
            uint32_t lo[4], hi[4];
            widen_cross(w[0][j], w[1][j], lo);
            widen_cross(w[2][j], w[3][j], hi);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const uint32_t a[4] = {lo[2 * h], lo[2 * h + 1], hi[2 * h], hi[2 * h + 1]};
#pragma unroll
              for (int nb = 0; nb < NB; ++nb)
                if (nb < nb_used) Mma<Op>::run(o[nb][2 * j + h], a, pf[u][nb][0], pf[u][nb][1]);
            }
          }
        } else {
#pragma unroll
          for (int mb = 0; mb < MB; ++mb) {
            uint32_t a[4];
            const int row = (lane & 7) + ((lane >> 4) << 3), ch = 2 * mb + ((lane >> 3) & 1);
            ldsm_x4_t(vb + rows_at<Cfg>(row, ch), a);
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
              if (nb < nb_used) Mma<Op>::run(o[nb][mb], a, pf[u][nb][0], pf[u][nb][1]);
          }
        }
      }
      __syncwarp();          // every lane has read the stage before the next issue overwrites it
      locate(t + S);
    }
    // ---- the four warps' states become one
    __syncthreads();
    float* const mo = reinterpret_cast<float*>(smem);                      // [warp][row][kPad]
    float* const mm = mo + kRowsWarps * Cfg::kRows * Cfg::kPad;             // [warp][row]
    float* const ml = mm + kRowsWarps * Cfg::kRows;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      if (nb >= nb_used) continue;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int row = nb * 8 + 2 * quad + e;
        float sum = l[nb][e];
        sum += __shfl_xor_sync(0xffffffffu, sum, 4);
        sum += __shfl_xor_sync(0xffffffffu, sum, 8);
        sum += __shfl_xor_sync(0xffffffffu, sum, 16);
        if (oct == 0) {
          mm[warp * Cfg::kRows + row] = m[nb][e];
          ml[warp * Cfg::kRows + row] = sum;
        }
        float* const dst = mo + (warp * Cfg::kRows + row) * Cfg::kPad;
#pragma unroll
        for (int mb = 0; mb < MB; ++mb) {
          const int d0 = FP8 ? (D / 8) * krow + 2 * mb : 16 * mb + oct, d1 = FP8 ? d0 + 1 : d0 + 8;
          dst[d0] = o[nb][mb][e];
          dst[d1] = o[nb][mb][e + 2];
        }
      }
    }
    __syncthreads();
    const int slot = part_slot(blockIdx.x, g.starts);
    for (int i = tid; i < rows * (D / 4); i += kRowsThreads) {
      const int row = i / (D / 4), d = (i % (D / 4)) * 4;
      float top = -INFINITY;
#pragma unroll
      for (int w = 0; w < kRowsWarps; ++w) top = fmaxf(top, mm[w * Cfg::kRows + row]);
      const float base = top == -INFINITY ? 0.f : top;
      float sum = 0.f;
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kRowsWarps; ++w) {
        const float f = exp2_fast(mm[w * Cfg::kRows + row] - base);
        sum += f * ml[w * Cfg::kRows + row];
        const float4 v = *reinterpret_cast<const float4*>(mo + (w * Cfg::kRows + row) * Cfg::kPad + d);
        acc.x += f * v.x; acc.y += f * v.y; acc.z += f * v.z; acc.w += f * v.w;
      }
      if (g.whole) {
        const float inv = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
        const int tok = token_of(row), head = g.head * p.group + row - tok * p.group;
        const int64_t t = g.s.t0 + g.tok0 + tok;
        *reinterpret_cast<uint2*>(p.out + t * p.o_tok + head * p.o_head + 2 * d) =
            make_uint2(Mma<T>::pack(acc.x * inv, acc.y * inv), Mma<T>::pack(acc.z * inv, acc.w * inv));
        if (p.lse && d == 0) p.lse[t * p.lse_tok + head] = sum > 0.f || sum != sum ? (base + log2f(sum)) * 0.693147180559945309f : -INFINITY;
      } else {
        *reinterpret_cast<float4*>(p.part_o + ((int64_t)slot * Cfg::kRows + row) * D + d) = acc;
        if (d == 0) *reinterpret_cast<float2*>(p.part_ml + ((int64_t)slot * Cfg::kRows + row) * 2) = make_float2(top, sum);
      }
    }
    if (!g.whole && tid == 0) note_split(p, g, rows);
    fence_async_shared();  // the next segment's TMA writes where the merge was
    __syncthreads();
    gathered = false;
  }
}

}  // namespace llg
