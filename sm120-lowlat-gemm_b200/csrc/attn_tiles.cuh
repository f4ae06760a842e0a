// Attention of many query rows per key/value head over a paged cache (prompt chunks): bound by the tensor cores.
//
// One persistent CTA per SM walks its share of (item, 128-key tile) units; an item is up to 256 packed query rows of one
// sequence and kv head, held as two 128-row streams A and B.
//   S = Q K^T   tcgen05.mma 128 x 128, both operands in shared memory (K-major, 128-byte swizzle)
//   P           softmax in registers, one thread per row: no shuffles; P goes back over S in tensor memory, 16 bit
//   O += P V    tcgen05.mma 128 x head_dim, P from tensor memory, V as it lies in the cache (rows of head_dim: MN-major B)
// Tensor memory: S_A, S_B (128 columns each), O_A, O_B (head_dim columns each). Warps 0-3 and 4-7: softmax of A and B; 8-11: loaders;
// 12: MMA issue; 13: the walk, published as segments in shared memory; 14, 15: fetch e4m3 rows for the loaders to widen, or fill the
// warpgroup: registers move between warpgroups, so that a row of 128 scores stays in the softmax threads. While one stream's softmax
// runs, the other stream's products do: per key tile and stream the tensor core needs 2 x 128 x 128 x head_dim / 4096 cycles (1024 at
// head_dim 128) and the exponentials 128 x 128 / 16 = 1024, so the two streams alternate between units that are equally busy.
// Items of at most 128 rows that several CTAs share (few rows, long cache) give both streams the same queries: A takes the
// even key tiles, B the odd ones, and each leaves a partial result of its own.
// m moves (and O is rescaled, from and to tensor memory) only when a row's score exceeds the largest so far by 2^8.
// Loaders: each of four warps fills a quarter of a 16-bit tile, by TMA in boxes of rows that share a page (page sizes that are a multiple
// of 8), row by row with cp.async and zeros where a quarter has rows outside the item's keys. e4m3 tiles come the same way, whole,
// into a staging ring; the loaders widen them into the swizzled tile. Queries: a stream's rows are one box of whole tokens where the
// group is a power of two (a ragged windowed batch 73.9 us with 32 cp.async per thread and item instead, 70.8 so);
// other groups are gathered.
// e4m3 caches are multiplied in f16 whatever q's type is: one conversion makes two values, exactly. The rows of a quarter tile (32
// keys) keep their powers of two relative to the quarter's largest, 2^E of K and 2^F of V, in the f16 values, which is exact down to
// 2^-15 (4 of 11 bits); rows of bf16 queries are brought to f16 by a power of two each. The softmax threads
// put the rest back where it costs nothing: score * (2^E, q's power) is the factor their multiply-add has anyway, and the
// probability is 2^(s + F - m) with m following the maximum of s + F, so that P 2^-F V is what the product sums; the row sum takes
// its quarters (an own tile's: its keys) times 2^-F.
// The quarter's largest may be a row that a query does not see, so a tile with rows further apart than that (V: 2^-7, the room that m
// leaves above) is an own one: its values are widened as they are, and the softmax threads, which find every row's two powers in
// shared memory, multiply each score by its own and take s + e of the keys that they see. A tile of that kind takes four times as
// long (a chunk of 512 behind 8192 of nothing else 675 us instead of 169): its code stays small, since code beside the loop that
// always runs slows that down (176 and 183 us with the whole tile unrolled).
// (Gathering every tile with cp.async was measured first: the proxy fence between a thread's copies and the tensor core's reads
// waits for all of the thread's copies in flight, 2600 cycles per 32 KB tile.)
// Measured, 64 heads over 8, head_dim 128: 2048 tokens behind 14k keys, bf16, 937 us (1.10 PFLOP/s, at the power cap); 512 behind
// 8192, e4m3, 169 us (0.84 PFLOP/s: the loaders' conversions and their shared-memory traffic).
// P is rounded to 16 bits (bf16 2^-8, f16 2^-11 relative); statistics and O stay in fp32, l sums the unrounded values.
#pragma once

#include <climits>
#include <type_traits>

#include "attn_rows.cuh"

namespace llg {

constexpr int kTilesKT = 128;     // keys per unit
constexpr int kTilesRows = 256;   // rows per item
constexpr int kTilesThreads = 512;

template <typename T, bool FP8, int D>
struct TilesCfg {
  using Op = typename std::conditional<FP8, __half, T>::type;  // operand type of the products
  static constexpr int kHalf = 128 * 128;                 // 128 rows x 64 elements, one swizzle-atom column
  static constexpr int kHalves = D / 64;
  static constexpr int kTile = kHalves * kHalf;           // a 128-row tile of Q, K or V
  static constexpr int kSlots = FP8 ? 3 : 4;              // ring of K and V tiles
  static constexpr int kStageRing = FP8 ? 3 : 0;          // staged e4m3 tiles
  static constexpr int kStage = 128 * D;
  static constexpr int kQ = 1024;                         // header before
  static constexpr int kRing = kQ + 2 * kTile;
  static constexpr int kStageAt = kRing + kSlots * kTile;
  static constexpr int kScaleAt = kStageAt + kStageRing * kStage;  // [kStageRing][128] f16: a staged row's factor
  static constexpr int kRefAt = kScaleAt + kStageRing * 256;       // [8 key tiles][8] bytes: biased E and F of the quarters; F 0: an own tile
  static constexpr int kQFacAt = kRefAt + (FP8 ? 64 : 0);          // [2 items][256] floats: the power of two of a row of q
  static constexpr int kOwnAt = kQFacAt + (FP8 ? 2048 : 0);        // [8 key tiles][2][128] bytes: powers of two of an own tile's rows of K, of V
  static constexpr int kSmem = kOwnAt + (FP8 ? 2048 : 0) + 1024;   // + alignment slack
};

// How far below a quarter's largest power of two its other rows may lie (see above).
constexpr uint32_t kSpreadK = 15, kSpreadV = 7;

// Shared-memory descriptor of V: rows of 64 elements (128 bytes, 128-byte swizzle) along K, 8 rows every 1024 bytes, the next
// 64 columns `half` bytes on (MN-major operand).
__device__ __forceinline__ uint64_t umma_desc_mn128(uint32_t addr, uint32_t half) {
  uint64_t d = 0;
  d |= (uint64_t)((addr & 0x3ffffu) >> 4);
  d |= (uint64_t)(half >> 4) << 16;
  d |= (uint64_t)(1024u >> 4) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}

__device__ __forceinline__ void tmem_ld32(uint32_t taddr, float (&v)[32]) {
  uint32_t* r = reinterpret_cast<uint32_t*>(v);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, "
      "%18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
        "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
        "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}
// Waits for the tensor-memory loads issued so far; naming the values keeps their uses behind the wait.
__device__ __forceinline__ void tmem_wait_ld32(float (&v)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]), "+f"(v[8]), "+f"(v[9]),
                 "+f"(v[10]), "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]), "+f"(v[15])
               :
               : "memory");
  asm volatile(""
               : "+f"(v[16]), "+f"(v[17]), "+f"(v[18]), "+f"(v[19]), "+f"(v[20]), "+f"(v[21]), "+f"(v[22]), "+f"(v[23]), "+f"(v[24]),
                 "+f"(v[25]), "+f"(v[26]), "+f"(v[27]), "+f"(v[28]), "+f"(v[29]), "+f"(v[30]), "+f"(v[31])
               :
               : "memory");
}
__device__ __forceinline__ void tmem_wait_ld16(uint32_t (&v)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]), "+r"(v[8]), "+r"(v[9]),
                 "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15])
               :
               : "memory");
}
// Moves registers between the warpgroups of a CTA. All four warps of a warpgroup execute it; the counts of all warpgroups
// together stay within what the CTA was launched with.
template <int N>
__device__ __forceinline__ void regs_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void regs_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ uint64_t pack_f32x2(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void unpack_f32x2(uint64_t v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ uint64_t fma_f32x2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add_f32x2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// Byte i of sixteen.
__device__ __forceinline__ uint32_t byte_of(const uint4& v, int i) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  return (w[i >> 2] >> (8 * (i & 3))) & 0xffu;
}

// Ring of mbarrier phases: slot i of n, used round after round.
struct Ring {
  int slot = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ void next(int n) {
    if (++slot == n) {
      slot = 0;
      phase ^= 1u;
    }
  }
};

// Barriers in the header: word offsets of 8 bytes from the start of shared memory.
enum : int { BAR_KV_FULL = 0, BAR_KV_EMPTY = 8, BAR_Q_FULL = 16, BAR_Q_EMPTY = 17, BAR_S_FULL = 18, BAR_P_FULL = 20, BAR_PV_DONE = 22, BAR_DONE = 24,
             BAR_SEG_FULL = 25, BAR_SEG_EMPTY = 29, BAR_RAW_FULL = 33, BAR_RAW_EMPTY = 37, BAR_Q_RAW = 41 };
constexpr int kSegRing = 4;        // segments published ahead of the roles that work on them

// How an item uses the two streams.
enum : int { MODE_ROWS = 0, MODE_ONE = 1, MODE_KEYS = 2 };  // B: rows 128 and on / idle / odd key tiles
__device__ __forceinline__ int tiles_mode(const Segment& g, int group) {
  return g.toks * group > 128 ? MODE_ROWS : g.whole ? MODE_ONE : MODE_KEYS;
}

template <typename T, bool FP8, int D>
__global__ void __launch_bounds__(kTilesThreads, 1) attn_tiles_kernel(const __grid_constant__ AttnDev p, const __grid_constant__ CUtensorMap map_k,
                                                                        const __grid_constant__ CUtensorMap map_v,
                                                                        const __grid_constant__ CUtensorMap map_q) {
  using Cfg = TilesCfg<T, FP8, D>;
  using Op = typename Cfg::Op;
  constexpr bool kBf16 = std::is_same<Op, __nv_bfloat16>::value;
  constexpr bool kToF16 = FP8 && std::is_same<T, __nv_bfloat16>::value;
  extern __shared__ unsigned char smem_raw[];
  __shared__ int scratch[kTilesThreads / 32 + 2];
  __shared__ uint32_t tmem_holder;
  __shared__ Segment segments[kSegRing];
  __shared__ volatile uint32_t abort_word, drain_word;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  auto bar = [&](int i) { return base + 8u * i; };
  if (tid == 0) {
    abort_word = drain_word = 0u;
    for (int i = 0; i < Cfg::kSlots; ++i) {
      mbar_init(bar(BAR_KV_FULL + i), 4);
      mbar_init(bar(BAR_KV_EMPTY + i), 1);
    }
    mbar_init(bar(BAR_Q_FULL), 128);
    mbar_init(bar(BAR_Q_EMPTY), 1);
    mbar_init(bar(BAR_Q_RAW), 1);
    for (int s = 0; s < 2; ++s) {
      mbar_init(bar(BAR_S_FULL + s), 1);
      mbar_init(bar(BAR_P_FULL + s), 128);
      mbar_init(bar(BAR_PV_DONE + s), 1);
    }
    mbar_init(bar(BAR_DONE), 1);
    for (int i = 0; i < Cfg::kStageRing; ++i) {
      mbar_init(bar(BAR_RAW_FULL + i), 32);
      mbar_init(bar(BAR_RAW_EMPTY + i), 4);
    }
    for (int i = 0; i < kSegRing; ++i) {
      mbar_init(bar(BAR_SEG_FULL + i), 1);
      mbar_init(bar(BAR_SEG_EMPTY + i), FP8 ? 15 : 13);  // the warps that read a segment
    }
    mbar_fence_init();
  }
  if (tid == 32) {
    tma_prefetch_desc(&map_k);
    tma_prefetch_desc(&map_v);
    tma_prefetch_desc(&map_q);
  }
  if (warp == 12) {
    tmem_alloc(smem_u32(&tmem_holder), 512);
    tmem_relinquish();
  }
  pdl_trigger();
  pdl_wait();
  if (tid == 0) clear_splits(p);
  tc_fence_before();
  Share share = find_share<kTilesKT, kTilesThreads>(p, scratch);  // synchronises the CTA
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_holder;
  const PagedKV& c = p.c;
  volatile uint32_t* const abort_at = &abort_word;
  bool ok = true;
  auto wait = [&](int b, uint32_t parity, uint32_t code) {
    if (!ok) return;
    if (!mbar_wait(bar(b), parity, abort_at)) {
      ok = false;
      atomicCAS(c.status, 0u, code);
    }
  };
  // The segments that warp 13 publishes, in order: next_item() waits for one (null behind the last), done_item() hands it back.
  Ring items;
  auto next_item = [&]() -> const Segment* {
    wait(BAR_SEG_FULL + items.slot, items.phase, ST_MMA_FULL_WAIT);
    return ok && segments[items.slot].tile0 >= 0 ? &segments[items.slot] : nullptr;
  };
  auto done_item = [&]() {
    __syncwarp();
    if (lane == 0) mbar_arrive(bar(BAR_SEG_EMPTY + items.slot));
    items.next(kSegRing);
  };

  if (warp >= 8 && warp < 12) {
    // ================================================================================================ loaders
    regs_down<64>();  // 512 threads start with 128 each: 2 x 200 (softmax) + 64 + 48, or 2 x 192 + 64 + 64 for e4m3 = 4 x 128
    const int lt = tid - 256, lw = warp - 8;                       // this warp fills rows 32 lw .. 32 lw + 31 of every tile
    Ring ring;
    uint32_t q_phase = 1;  // the first wait for an empty Q passes
    // The segment at hand. Its fields are copied: the tensor core's operand reads fill the shared-memory pipe, and every load from
    // there costs the loaders hundreds of cycles.
    int tile0 = 0, tile1 = 0, key_lo = 0, key_hi = 0, kv_head = 0;
    const int* table_row = nullptr;
    // A tile's row 32 lw + lane: its page (-1: no row, reads as zeros) and slot. The page table's entry is requested a tile ahead.
    struct Row {
      int pg, slot;
    };
    int entry = 0;
    auto in_use = [&](int j) {
      const int key = j * kTilesKT + lt;
      return j < tile1 && key >= key_lo && key < key_hi;
    };
    auto look_up = [&](int j) {
      int block, slot;
      split_key(c, j * kTilesKT + lt, block, slot);
      if (in_use(j)) entry = table_row[block];
    };
    auto locate = [&](int j) {
      Row r{-1, 0};
      const int pg = entry;
      look_up(j + 1);
      if (in_use(j)) {
        int block;
        split_key(c, j * kTilesKT + lt, block, r.slot);
        if ((unsigned)pg >= (unsigned)c.pages) {
          atomicCAS(c.status, 0u, (unsigned)ST_BAD_PAGE);
        } else {
          r.pg = pg;
        }
      }
      return r;
    };
    // byte offset of a row of K or V, -1 for none
    auto offset = [&](const Row& r, bool is_v) -> int64_t {
      if (r.pg < 0) return -1;
      return is_v ? r.pg * c.v_page + kv_head * c.v_head + r.slot * c.v_slot : r.pg * c.k_page + kv_head * c.k_head + r.slot * c.k_slot;
    };
    const int box = p.box;                                         // rows of a TMA box, 0: gather every row
    // Whole quarter tiles come by TMA, boxes of rows that lie in one page; quarters with rows that are not there are gathered.
    auto by_tma = [&](const Row& r) { return box > 0 && __all_sync(0xffffffffu, r.pg >= 0); };
    // 16-bit rows: straight into slot `ring.slot`, swizzled
    auto copy16 = [&](const Row& r, bool is_v) {
      wait(BAR_KV_EMPTY + ring.slot, ring.phase ^ 1u, ST_PRODUCER_EMPTY_WAIT);
      if (!ok) return;
      const uint32_t dst = base + Cfg::kRing + ring.slot * Cfg::kTile, full = bar(BAR_KV_FULL + ring.slot);
      if (by_tma(r)) {
        if (lane == 0) mbar_expect_tx(full, 32 * D * 2);
        const int at = (lane / Cfg::kHalves) * box, half = lane % Cfg::kHalves;
        const int pg = __shfl_sync(0xffffffffu, r.pg, at & 31), slot = __shfl_sync(0xffffffffu, r.slot, at & 31);
        if (at < 32) tma_load_4d(dst + half * Cfg::kHalf + (lw * 32 + at) * 128, is_v ? &map_v : &map_k, full, half * 64, slot, kv_head, pg);
      } else {
        const int64_t off = offset(r, is_v);
        const unsigned char* const src = is_v ? c.v : c.k;
        constexpr int CH = D / 8, RP = 32 / CH;                    // 16-byte pieces per row, rows per warp instruction
#pragma unroll 4
        for (int i = 0; i < 32 / RP; ++i) {
          const int q = i * RP + lane / CH, ch = lane % CH, row = lw * 32 + q;
          const int64_t o = __shfl_sync(0xffffffffu, off, q);
          cp_async16(dst + (ch >> 3) * Cfg::kHalf + row * 128 + (((ch & 7) ^ (row & 7)) << 4), src + (o >= 0 ? o + ch * 16 : 0), o >= 0 ? 16u : 0u);
        }
        cp_async_commit();
        cp_async_wait<0>();
        fence_async_shared();
        __syncwarp();
        if (lane == 0) mbar_arrive(full);
      }
      __syncwarp();
      ring.next(Cfg::kSlots);
    };
    // e4m3 rows: warps 14 and 15 fetch them as they are, `widen` converts the warp's quarter into the ring
    constexpr int CH8 = D / 16, RP8 = 32 / CH8, IT8 = 32 / RP8;    // 16-byte pieces per row, rows per warp instruction, instructions
    Ring raw;
    auto widen = [&]() {
      wait(BAR_RAW_FULL + raw.slot, raw.phase, ST_CONVERT_WAIT);
      wait(BAR_KV_EMPTY + ring.slot, ring.phase ^ 1u, ST_CONVERT_WAIT);
      if (!ok) return;
      const uint32_t src = base + Cfg::kStageAt + raw.slot * Cfg::kStage + lw * (32 * D) + lane * 16;
      const uint32_t scales = base + Cfg::kScaleAt + raw.slot * 256 + lw * 64;
      const uint32_t dst = base + Cfg::kRing + ring.slot * Cfg::kTile;
#pragma unroll 4
      for (int i = 0; i < IT8; ++i) {
        const int q = i * RP8 + lane / CH8, ch = lane % CH8, row = lw * 32 + q;
        const uint4 v = lds16(src + i * 512);
        uint32_t b;
        asm volatile("ld.shared.u16 %0, [%1];" : "=r"(b) : "r"(scales + q * 2) : "memory");
        b |= b << 16;
        const __half2 f = *reinterpret_cast<const __half2*>(&b);
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
        uint32_t o[8];
#pragma unroll
        for (int j = 0; j < 4; ++j) widen4(w[j], o[2 * j], o[2 * j + 1]);
#pragma unroll
        for (int j = 0; j < 8; ++j) *reinterpret_cast<__half2*>(&o[j]) = __hmul2(*reinterpret_cast<__half2*>(&o[j]), f);
        const uint32_t at0 = dst + (ch >> 2) * Cfg::kHalf + row * 128;
        const int c0 = 2 * (ch & 3);
        // lanes of the two halves write alternate pieces first: eight lanes then fall on eight different bank groups
        const bool odd = (ch >> 2) & 1;
        const uint32_t a0 = at0 + (((c0 + (odd ? 1 : 0)) ^ (row & 7)) << 4), a1 = at0 + (((c0 + (odd ? 0 : 1)) ^ (row & 7)) << 4);
        const uint4 lo = make_uint4(o[0], o[1], o[2], o[3]), hi = make_uint4(o[4], o[5], o[6], o[7]);
        const uint4 x = odd ? hi : lo, y = odd ? lo : hi;
        asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(a0), "r"(x.x), "r"(x.y), "r"(x.z), "r"(x.w) : "memory");
        asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(a1), "r"(y.x), "r"(y.y), "r"(y.z), "r"(y.w) : "memory");
      }
      fence_async_shared();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(bar(BAR_KV_FULL + ring.slot));
        mbar_arrive(bar(BAR_RAW_EMPTY + raw.slot));
      }
      ring.next(Cfg::kSlots);
      raw.next(Cfg::kStageRing);
    };
    int item_parity = 0;
    uint32_t q_raw_phase = 0;
    const bool remake = kToF16 || p.negate;                        // queries are not multiplied as they are
    auto q_free = [&]() { return mbar_try(bar(BAR_Q_EMPTY), q_phase); };
    auto start_q = [&](const Segment& g) {  // copies under way
      wait(BAR_Q_EMPTY, q_phase, ST_PRODUCER_EMPTY_WAIT);
      q_phase ^= 1u;
      if (!ok) return;
      if (p.q_box) {  // rows of no token of the tile get other tokens' queries, or zeros behind the last: nobody reads their results
        if (lt == 0) {
          const uint32_t there = bar(remake ? BAR_Q_RAW : BAR_Q_FULL);
          mbar_expect_tx(there, 2 * Cfg::kTile);
          for (int i = 0; i < 2 * Cfg::kHalves; ++i) {
            const int half = i % Cfg::kHalves, stream = i / Cfg::kHalves;
            tma_load_4d(base + Cfg::kQ + stream * Cfg::kTile + half * Cfg::kHalf, &map_q, there, half * 64, kv_head * p.group,
                        g.s.t0 + g.tok0 + stream * (p.tok_tile / 2), 0);
          }
        }
        return;
      }
      const int rows = g.toks * p.group;
      const int64_t first = g.s.t0 + g.tok0;
      constexpr int CH = D / 8;
      // 32 (16) copies of 16 bytes per thread, all in flight at once
      const int ch = lt % CH;
      int row = lt / CH, tok = row / p.group, hh = row - tok * p.group;
#pragma unroll 4
      for (int i = 0; i < kTilesRows * CH / 128; ++i) {
        const bool there = row < rows;
        const unsigned char* const src = p.q + (first + tok) * p.q_tok + (int64_t)(kv_head * p.group + hh) * p.q_head + ch * 16;
        cp_async16(base + Cfg::kQ + (row >> 7) * Cfg::kTile + (ch >> 3) * Cfg::kHalf + (row & 127) * 128 + (((ch & 7) ^ (row & 7)) << 4),
                   there ? src : p.q, there ? 16u : 0u);
        row += 128 / CH;
        for (hh += 128 / CH; hh >= p.group; hh -= p.group) ++tok;
      }
      cp_async_commit();
    };
    auto finish_q = [&]() {                 // copies there, and in the form the products take
      if (!ok) return;
      if (p.q_box && !remake) {  // thread 0 arrived when it announced the copies' bytes
        if (lt != 0) mbar_arrive(bar(BAR_Q_FULL));
        return;
      }
      constexpr int CH = D / 8;
      const int ch = lt % CH;
      if (p.q_box) {
        wait(BAR_Q_RAW, q_raw_phase, ST_PRODUCER_EMPTY_WAIT);
        q_raw_phase ^= 1u;
        if (!ok) return;
      } else {
        cp_async_wait<0>();
      }
      if (remake) {  // bf16 rows to f16 in place, and the sign of a negative softmax scale: each thread what it copied itself, or what TMA did
        const uint32_t flip = p.negate ? 0x80008000u : 0u;
#pragma unroll 4
        for (int r = lt / CH; r < kTilesRows; r += 128 / CH) {     // CH neighbouring lanes hold a row
          const uint32_t at = base + Cfg::kQ + (r >> 7) * Cfg::kTile + (ch >> 3) * Cfg::kHalf + (r & 127) * 128 + (((ch & 7) ^ (r & 7)) << 4);
          const uint4 v = lds16(at);
          uint32_t w[4] = {v.x, v.y, v.z, v.w};
          if constexpr (kToF16) {
            // largest magnitude: bf16 bits without the sign are ordered like integers
            uint32_t top = __vmaxu2(__vmaxu2(w[0] & 0x7fff7fffu, w[1] & 0x7fff7fffu), __vmaxu2(w[2] & 0x7fff7fffu, w[3] & 0x7fff7fffu));
#pragma unroll
            for (int o = CH / 2; o >= 1; o >>= 1) top = __vmaxu2(top, __shfl_xor_sync(0xffffffffu, top, o));
            const uint32_t e = max(max(top & 0xffffu, top >> 16) >> 7, 20u);
            const float up = __uint_as_float((268u - e) << 23);    // 2^(14 - exponent of the row's largest value)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float2 f = __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&w[j]));
              w[j] = Mma<__half>::pack(f.x * up, f.y * up);
            }
            if (ch == 0) asm volatile("st.shared.u32 [%0], %1;" ::"r"(base + Cfg::kQFacAt + item_parity * 1024 + r * 4), "r"((e - 14u) << 23) : "memory");
          }
          asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(w[0] ^ flip), "r"(w[1] ^ flip), "r"(w[2] ^ flip), "r"(w[3] ^ flip)
                       : "memory");
        }
        item_parity ^= 1;
      }
      fence_async_shared();
      mbar_arrive(bar(BAR_Q_FULL));
    };
    while (const Segment* const seg = next_item()) {
      tile0 = seg->tile0;
      tile1 = seg->tile1;
      key_lo = seg->keys.lo;
      key_hi = seg->keys.hi;
      kv_head = seg->head;
      table_row = c.table + (int64_t)seg->seq * c.table_stride;
      const bool keys = tiles_mode(*seg, p.group) == MODE_KEYS;
      // queries first when their place is free already (the first item), else behind the first tiles
      const bool early = __all_sync(0xffffffffu, q_free());
      if (early) start_q(*seg);
      auto load_q = [&]() {
        if (!early) start_q(*seg);
        finish_q();
      };
      // order in which the MMA warp takes them: K0 V0 K1 V1 ..., or K0 K1 V0 K2 V1 ... when the streams take turns
      if constexpr (!FP8) {
        look_up(tile0);
        Row next = locate(tile0), held{};
        for (int j = tile0; j < tile1; ++j) {
          const Row row = next;
          next = locate(j + 1);
          copy16(row, false);
          if (keys && j == tile0 + 1) load_q();
          if (!keys) copy16(row, true);
          else if (j > tile0) copy16(held, true);
          if (!keys && j == tile0) load_q();  // behind two tiles that travel meanwhile
          held = row;
        }
        if (keys && tile1 - tile0 == 1) load_q();
        if (keys) copy16(held, true);
      } else {
        load_q();
        for (int n = 2 * (tile1 - tile0); n > 0 && ok; --n) widen();
      }
      done_item();
    }
  } else if (warp >= 12) {
    regs_down<FP8 ? 64 : 48>();
    if (warp == 12) {
    // ================================================================================================ MMA issue
    constexpr uint32_t kFmt = kBf16 ? 1u : 0u;
    constexpr uint32_t kIdescS = umma_idesc(1, kFmt, kFmt, 128, 128);
    constexpr uint32_t kIdescO = umma_idesc(1, kFmt, kFmt, 128, D) | (1u << 16);  // B is MN-major
    Ring ring;
    uint32_t q_phase = 0, p_phase[2] = {0u, 0u};
    const bool leader = elect_one();
    auto scores = [&](int s, int qt, uint32_t kslot) {  // S_s = Q_qt K^T
      if (leader) {
        // descriptors differ in the low word's address only; opaque, so that no call site keeps its sixteen of them
        uint32_t qa = (base + Cfg::kQ + qt * Cfg::kTile) >> 4, ka = (base + Cfg::kRing + kslot * Cfg::kTile) >> 4;
        asm volatile("" : "+r"(qa), "+r"(ka));
        const uint64_t hi = umma_desc_sw128(0);
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
          const uint32_t off = ((ks >> 2) * Cfg::kHalf + (ks & 3) * 32) >> 4;
          mma_ss_f16(tmem + s * 128, hi | (qa + off), hi | (ka + off), kIdescS, ks > 0);
        }
        umma_commit(bar(BAR_S_FULL + s));
      }
      __syncwarp();
    };
    auto values = [&](int s, uint32_t vslot, bool first) {  // O_s (+)= P_s V
      wait(BAR_P_FULL + s, p_phase[s], ST_MMA_FULL_WAIT);
      p_phase[s] ^= 1u;
      if (!ok) return;
      tc_fence_after();
      if (leader) {
        uint32_t va = (base + Cfg::kRing + vslot * Cfg::kTile) >> 4;
        asm volatile("" : "+r"(va));
        const uint64_t hi = umma_desc_mn128(0, Cfg::kHalf);
#pragma unroll
        for (int ks = 0; ks < 8; ++ks)
          mma_ts_f16(tmem + 256 + s * D, tmem + s * 128 + ks * 8, hi | (va + ks * 128), kIdescO, !first || ks > 0);
        umma_commit(bar(BAR_PV_DONE + s));
      }
      __syncwarp();
    };
    auto full = [&]() -> int {  // waits for the next tile of the ring
      wait(BAR_KV_FULL + ring.slot, ring.phase, ST_MMA_FULL_WAIT);
      if (ok) tc_fence_after();
      const int s = ring.slot;
      ring.next(Cfg::kSlots);
      return s;
    };
    auto release = [&](int b) {
      if (leader) umma_commit(bar(b));
      __syncwarp();
    };
    while (const Segment* seg = next_item()) {
      const int mode = tiles_mode(*seg, p.group);
      const int nt = seg->tile1 - seg->tile0;
      done_item();
      int k = full();
      wait(BAR_Q_FULL, q_phase, ST_MMA_FULL_WAIT);
      q_phase ^= 1u;
      if (!ok) break;
      tc_fence_after();
      scores(0, 0, k);
      if (mode == MODE_ROWS) scores(1, 1, k);
      release(BAR_KV_EMPTY + k);
      if (mode == MODE_KEYS && nt > 1) {
        k = full();
        if (!ok) break;
        scores(1, 0, k);
        release(BAR_KV_EMPTY + k);
      }
      if (nt == 1 || (mode == MODE_KEYS && nt == 2)) release(BAR_Q_EMPTY);
      for (int j = 0; j < nt && ok; ++j) {
        const int v = full();
        if (!ok) break;
        if (mode == MODE_KEYS) {
          const int s = j & 1;
          const bool more = j + 2 < nt;
          if (more) k = full();
          if (!ok) break;
          values(s, v, j < 2);
          if (!ok) break;
          if (more) scores(s, 0, k);
          release(BAR_KV_EMPTY + v);
          if (more) release(BAR_KV_EMPTY + k);
          if (j + 3 == nt) release(BAR_Q_EMPTY);
        } else {
          // both tiles are waited for ahead of P: between the products a barrier's latency would leave the tensor core idle
          const bool more = j + 1 < nt;
          if (more) k = full();
          if (!ok) break;
          values(0, v, j == 0);
          if (!ok) break;
          if (more) scores(0, 0, k);
          if (mode == MODE_ROWS) {
            values(1, v, j == 0);
            if (!ok) break;
            if (more) scores(1, 1, k);
          }
          release(BAR_KV_EMPTY + v);
          if (more) release(BAR_KV_EMPTY + k);
          if (j + 2 == nt) release(BAR_Q_EMPTY);
        }
      }
    }
    // nothing of this CTA may be in flight when its tensor memory goes
    release(BAR_DONE);
    mbar_wait(bar(BAR_DONE), 0, &drain_word);
    } else if (warp == 13) {
    // ================================================================================================ schedule
    while (ok) {
      wait(BAR_SEG_EMPTY + items.slot, items.phase ^ 1u, ST_PRODUCER_EMPTY_WAIT);
      Segment g;
      const bool more = ok && next_segment<kTilesKT>(p, share, g);
      if (!more) g.tile0 = -1;
      if (lane == 0) {
        segments[items.slot] = g;
        mbar_arrive(bar(BAR_SEG_FULL + items.slot));
      }
      __syncwarp();
      items.next(kSegRing);
      if (!more) break;
    }
    } else if (FP8) {
    // ================================================================================================ e4m3 fetch
    // Tiles as they lie in the cache, in the order in which the loaders widen them - warp 14 those of K, warp 15 those of V - with
    // what their rows' powers of two become: each row's factor relative to its quarter's largest, and the quarters' largest of K
    // and V for the softmax. Where scale bytes lie row by row and all of a tile's rows exist, a lane has the four rows from 4 * lane
    // on - one page table entry, requested a tile ahead, and one word of scales; else it has row `lane` of each quarter.
    const bool is_v = warp == 15;
    Ring raw;
    int tiles_in = 0;            // key tiles fetched
    while (const Segment* const seg = next_item()) {
      const int tile0 = seg->tile0, tile1 = seg->tile1, key_lo = seg->keys.lo, key_hi = seg->keys.hi, kv_head = seg->head;
      const int* const table_row = c.table + (int64_t)seg->seq * c.table_stride;
      const bool keys = tiles_mode(*seg, p.group) == MODE_KEYS;
      const int n = 2 * (tile1 - tile0);
      int j = tile0, entry = INT_MIN;
      const unsigned char *const ks = c.ks + kv_head * c.ks_head, *const vs = c.vs + kv_head * c.vs_head;
      const bool words = p.scale16 && p.box > 0;
      // Scale bytes are worked on four at a time. Are any of them further below their quarters' largest (`high`) than may be, or beyond
      // what the softmax's factors can take? Then the tile is an own one. Rows of zeros and others of the smallest power that the cache's
      // writer knows, 2^-100, do not ask for that: beside larger ones they count as zeros.
      const uint32_t spread = (is_v ? kSpreadV : kSpreadK) * 0x01010101u, least = (is_v ? kLeastV : 27u) * 0x01010101u;
      auto far_apart = [&](uint32_t w, uint32_t high, uint32_t by) {
        w |= __vcmpleu4(w, 27u * 0x01010101u);
        return __any_sync(0xffffffffu, __vmaxu4(w, __vsubus4(high, by)) != w || __vmaxu4(high, 0xfdfdfdfdu) != 0xfdfdfdfdu);
      };
      // by how many powers of two the rows' values go down: an own tile's only where m takes no account of them
      auto shifts = [&](bool own, uint32_t w, uint32_t top) { return !own ? top - w : is_v ? __vsubus4(least, w) : 0u; };
      auto down16 = [&](uint32_t d4) {  // 2^-d as f16, d the lowest byte
        const uint32_t d = d4 & 0xffu;
        return d < 15u ? (15u - d) << 10 : d <= 24u ? 1u << (24u - d) : 0u;
      };
      auto whole = [&](int t) { return words && t * kTilesKT >= key_lo && (t + 1) * kTilesKT <= key_hi; };
      auto look_up = [&](int t) {
        int block, slot;
        split_key(c, t * kTilesKT + 4 * lane, block, slot);
        if (t < tile1 && whole(t)) entry = table_row[block];
      };
      look_up(j);
      for (int i = 0; i < n && ok; ++i) {
        const bool of_v = keys ? !(i == 0 || ((i & 1) && i < n - 1)) : (i & 1) != 0;
        if (of_v != is_v) {      // the other warp's
          raw.next(Cfg::kStageRing);
          continue;
        }
        const int tile = j++, fast_pg = entry;
        look_up(j);
        if (whole(tile) && __all_sync(0xffffffffu, (unsigned)fast_pg < (unsigned)c.pages)) {
          int block, slot;
          split_key(c, tile * kTilesKT + 4 * lane, block, slot);
          const uint32_t sv = *reinterpret_cast<const uint32_t*>(vs + fast_pg * c.vs_page + slot);
          const uint32_t sc = is_v ? sv : *reinterpret_cast<const uint32_t*>(ks + fast_pg * c.ks_page + slot);
          wait(BAR_RAW_EMPTY + raw.slot, raw.phase ^ 1u, ST_PRODUCER_EMPTY_WAIT);
          if (!ok) break;
          const uint32_t dst = base + Cfg::kStageAt + raw.slot * Cfg::kStage, full = bar(BAR_RAW_FULL + raw.slot);
          if (lane == 0) mbar_expect_tx_only(full, 128 * D);
          __syncwarp();
          const int at = lane * p.box;   // boxes of rows that share a page
          const int bp = __shfl_sync(0xffffffffu, fast_pg, (at >> 2) & 31), bs = __shfl_sync(0xffffffffu, slot, (at >> 2) & 31);
          if (at < 128) tma_load_4d(dst + at * D, is_v ? &map_v : &map_k, full, 0, bs, kv_head, bp);
          // largest of the quarter's bytes: of the word's four, then of the quarter's eight lanes
          auto quarter_top = [&](uint32_t w) {
            w = __vmaxu4(w, w >> 16);
            w = max(w & 0xffu, (w >> 8) & 0xffu);
#pragma unroll
            for (int d = 1; d < 8; d <<= 1) w = max(w, __shfl_xor_sync(0xffffffffu, w, d));
            return w;
          };
          const uint32_t high = quarter_top(sc) * 0x01010101u;
          const bool own = far_apart(sc, high, spread);
          const uint32_t top = __vmaxu4(high, least), d4 = shifts(own, sc, top);
          asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(base + Cfg::kScaleAt + raw.slot * 256 + lane * 8), "r"(down16(d4) | down16(d4 >> 8) << 16),
                       "r"(down16(d4 >> 16) | down16(d4 >> 24) << 16) : "memory");
          if (!is_v) {
            const uint32_t v_high = quarter_top(sv) * 0x01010101u, v_top = __vmaxu4(v_high, kLeastV * 0x01010101u);
            const bool v_own = far_apart(sv, v_high, kSpreadV * 0x01010101u), any_own = own || v_own;
            if (any_own) {
              const uint32_t to = base + Cfg::kOwnAt + (tiles_in & 7) * 256 + lane * 4;
              asm volatile("st.shared.u32 [%0], %1;" ::"r"(to), "r"(own ? sc : top) : "memory");
              asm volatile("st.shared.u32 [%0], %1;" ::"r"(to + 128), "r"(v_own ? sv : v_top) : "memory");
            }
            if ((lane & 7) == 0) {
              const uint32_t ref = base + Cfg::kRefAt + (tiles_in & 7) * 8 + (lane >> 3);
              asm volatile("st.shared.u8 [%0], %1;" ::"r"(ref), "r"(top) : "memory");
              asm volatile("st.shared.u8 [%0], %1;" ::"r"(ref + 4), "r"(any_own ? 0u : v_top) : "memory");
            }
            ++tiles_in;
          }
          mbar_arrive(full);
          raw.next(Cfg::kStageRing);
          continue;
        }
        int pg[4], slot[4];
        bool all = true;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int key = tile * kTilesKT + 32 * q + lane;
          int block;
          split_key(c, key, block, slot[q]);
          pg[q] = key >= key_lo && key < key_hi ? table_row[block] : INT_MIN;
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          if ((unsigned)pg[q] >= (unsigned)c.pages) {
            if (pg[q] != INT_MIN) atomicCAS(c.status, 0u, (unsigned)ST_BAD_PAGE);
            pg[q] = -1;
            all = false;
          }
        }
        all = __all_sync(0xffffffffu, all) && p.box > 0;
        uint32_t sc[4], other[4] = {0u, 0u, 0u, 0u};
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          sc[q] = 0u;
          if (pg[q] >= 0) {
            const uint32_t of_values = vs[pg[q] * c.vs_page + slot[q] * c.vs_slot];
            sc[q] = is_v ? of_values : ks[pg[q] * c.ks_page + slot[q] * c.ks_slot];
            other[q] = of_values;
          }
        }
        wait(BAR_RAW_EMPTY + raw.slot, raw.phase ^ 1u, ST_PRODUCER_EMPTY_WAIT);
        if (!ok) break;
        const uint32_t dst = base + Cfg::kStageAt + raw.slot * Cfg::kStage, full = bar(BAR_RAW_FULL + raw.slot);
        if (all) {
          if (lane == 0) mbar_expect_tx_only(full, 128 * D);
          __syncwarp();
          const int at = lane * p.box;   // boxes of rows that share a page
          int bp = 0, bs = 0;
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const int x = __shfl_sync(0xffffffffu, pg[q], at & 31), y = __shfl_sync(0xffffffffu, slot[q], at & 31);
            if ((at >> 5) == q) {
              bp = x;
              bs = y;
            }
          }
          if (at < 128) tma_load_4d(dst + at * D, is_v ? &map_v : &map_k, full, 0, bs, kv_head, bp);
        } else {
          constexpr int CH = D / 16, RP = 32 / CH;
          const unsigned char* const src = is_v ? c.v : c.k;
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            int64_t off = -1;
            if (pg[q] >= 0)
              off = is_v ? pg[q] * c.v_page + kv_head * c.v_head + slot[q] * c.v_slot : pg[q] * c.k_page + kv_head * c.k_head + slot[q] * c.k_slot;
#pragma unroll 2
            for (int r = 0; r < CH; ++r) {
              const int64_t o = __shfl_sync(0xffffffffu, off, r * RP + lane / CH);
              cp_async16(dst + q * (32 * D) + r * 512 + lane * 16, src + (o >= 0 ? o + (lane % CH) * 16 : 0), o >= 0 ? 16u : 0u);
            }
          }
          cp_async_commit();
          cp_async_wait<0>();
          fence_async_shared();  // a later TMA writes here
        }
        uint32_t w = 0u, v = 0u, high = 0u, v_high = 0u;  // a byte of each word per quarter; rows that are not there have none
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          w |= sc[q] << (8 * q);
          v |= other[q] << (8 * q);
          high |= __reduce_max_sync(0xffffffffu, sc[q]) << (8 * q);
          v_high |= __reduce_max_sync(0xffffffffu, other[q]) << (8 * q);
        }
        const bool own = far_apart(w, high, spread);
        const uint32_t top = __vmaxu4(high, least), d4 = shifts(own, w, top);
#pragma unroll
        for (int q = 0; q < 4; ++q)
          asm volatile("st.shared.u16 [%0], %1;" ::"r"(base + Cfg::kScaleAt + raw.slot * 256 + (32 * q + lane) * 2), "h"((uint16_t)down16(d4 >> (8 * q))) : "memory");
        if (!is_v) {
          const bool v_own = far_apart(v, v_high, kSpreadV * 0x01010101u), any_own = own || v_own;
          const uint32_t v_top = __vmaxu4(v_high, kLeastV * 0x01010101u);
          if (any_own) {  // rows that are not there are zeros: any power will do
            const uint32_t to = base + Cfg::kOwnAt + (tiles_in & 7) * 256 + lane, k4 = own ? w : top, v4 = v_own ? v : v_top;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              asm volatile("st.shared.u8 [%0], %1;" ::"r"(to + 32 * q), "r"(k4 >> (8 * q)) : "memory");
              asm volatile("st.shared.u8 [%0], %1;" ::"r"(to + 128 + 32 * q), "r"(v4 >> (8 * q)) : "memory");
            }
          }
          if (lane == 0)
            asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(base + Cfg::kRefAt + (tiles_in & 7) * 8), "r"(top), "r"(any_own ? 0u : v_top) : "memory");
          ++tiles_in;
        }
        mbar_arrive(full);
        raw.next(Cfg::kStageRing);
      }
      done_item();
    }
    }
  } else {
    // ================================================================================================ softmax
    regs_up<FP8 ? 192 : 200>();
    const int s = warp >> 2;                                   // stream
    const int row_in = (warp & 3) * 32 + lane;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t tS = tmem + lanes + s * 128, tO = tmem + lanes + 256 + s * D;
    uint32_t s_phase = 0, pv_phase = 0;
    int item_parity = 0, tile_base = 0;                            // e4m3: which q factors and which references are this item's
    while (const Segment* seg = next_item()) {
      const Segment& g = *seg;
      const int mode = tiles_mode(g, p.group);
      const int my_parity = item_parity, my_base = tile_base - g.tile0;
      item_parity ^= 1;
      tile_base += g.tile1 - g.tile0;
      if (mode == MODE_ONE && s == 1) {
        done_item();
        continue;
      }
      const int rows = g.toks * p.group;
      const int row = mode == MODE_ROWS ? s * 128 + row_in : row_in;
      const int step = mode == MODE_KEYS ? 2 : 1;
      const bool live = row < rows;
      const int tok = row / p.group;
      const int pos = g.s.pos + g.tok0 + tok;
      // rows of no token see everything: they keep no tile from the unmasked path, and nobody reads them
      const int last = !live ? INT_MAX : p.causal ? min(pos, g.s.len - 1) : g.s.len - 1;
      const int first = live && p.window > 0 ? pos - p.window + 1 : 0;
      float m = -INFINITY;                                       // reference of the probabilities: scores in log2 units (+ F)
      bool huge = false;                                         // kHuge, in a row of the warp
      float c_row = p.scale_log2;
      uint64_t l2 = 0;                                           // two partial row sums
      int done = 0;                                              // key tiles of this stream behind us
      const int tile1 = g.tile1;
      for (int j = g.tile0 + (mode == MODE_KEYS ? s : 0); j < tile1 && ok; j += step, ++done) {
        wait(BAR_S_FULL + s, s_phase, ST_EPILOGUE_WAIT);
        s_phase ^= 1u;
        if (!ok) break;
        tc_fence_after();
        // what turns a quarter's products into log2 units, and its F
        float cq[4], fq[4];
        uint32_t f_bytes = 0;
        if constexpr (FP8) {
          if (kToF16 && done == 0) {
            float f;
            asm volatile("ld.shared.f32 %0, [%1];" : "=f"(f) : "r"(base + Cfg::kQFacAt + my_parity * 1024 + row * 4) : "memory");
            c_row *= f;
          }
          const uint2 ref = lds8(base + Cfg::kRefAt + ((my_base + j) & 7) * 8);
          f_bytes = ref.y;
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            // not 0, which would make NaN of a masked column's -inf (a row of zeros against rows of zeros: 2^-121 * 2^-100), nor infinite,
            // which would of a product of 0
            cq[q] = fminf(fmaxf(c_row * pow2_of((ref.x >> (8 * q)) & 0xffu), 1.17549435e-38f), 3.40282347e38f);
            fq[q] = __uint_as_float(0x4b000000u + ((ref.y >> (8 * q)) & 0xffu)) - 8388735.f;  // F: bits of 2^23 + byte, less 2^23 + 127
          }
        } else {
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            cq[q] = c_row;
            fq[q] = 0.f;
          }
        }
        const int key0 = j * kTilesKT;
        // does any row of the warp see only a part of the tile?
        const bool edge = __any_sync(0xffffffffu, key0 + kTilesKT - 1 > last || key0 < first);
        const int hi = last - key0, lo = first - key0;           // columns [lo, hi] are seen
        // the reference follows a row's largest score; what has been added up so far is rescaled
        auto follow = [&](float top) {
          const bool move = top > m + kMove || (m == -INFINITY && top > m);
          if (!__any_sync(0xffffffffu, move)) return;
          const float now = move ? top - kHead : m;
          const float keep = m == -INFINITY ? 0.f : exp2_fast(m - now);
          if (done > 0) {
            wait(BAR_PV_DONE + s, pv_phase ^ 1u, ST_EPILOGUE_WAIT);
            if (!ok) return;
            tc_fence_after();
#pragma unroll 1
            for (int q = 0; q < D / 16; ++q) {
              uint32_t o[16];
              tmem_ld16(tO + 16 * q, o);
              tmem_wait_ld16(o);
#pragma unroll
              for (int i = 0; i < 16; ++i) o[i] = keep == 0.f ? 0u : __float_as_uint(__uint_as_float(o[i]) * keep);
              tmem_st16(tO + 16 * q, o);
            }
            float a, b;
            unpack_f32x2(l2, a, b);
            l2 = pack_f32x2(a * keep, b * keep);
          }
          m = now;
          huge = __any_sync(0xffffffffu, fabsf(m) > kHuge && m > -INFINITY);
        };
        float x[4][32];
#pragma unroll
        for (int q = 0; q < 4; ++q) tmem_ld32(tS + 32 * q, x[q]);
#pragma unroll
        for (int q = 0; q < 4; ++q) tmem_wait_ld32(x[q]);
        if (FP8 && __builtin_expect(__any_sync(0xffffffffu, f_bytes == 0u), 0)) {
          // an own tile, 16 columns at a time: scores in log2 units, masked, go back to where they came from, then become P
          const uint32_t powers = base + Cfg::kOwnAt + ((my_base + j) & 7) * 256;
          float top = -INFINITY;
#pragma unroll 1
          for (int c16 = 0; c16 < 128; c16 += 16) {
            uint32_t y[16];
            tmem_ld16(tS + c16, y);
            tmem_wait_ld16(y);
            const uint4 kb = lds16(powers + c16), vb = lds16(powers + 128 + c16);
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const float score = __uint_as_float(y[i]) * finite_product(c_row, e8m0_value(byte_of(kb, i))) + power_of(carried(byte_of(vb, i), kLeastV));
              const float z = c16 + i <= hi && c16 + i >= lo ? score : -INFINITY;
              top = fmaxf(top, z);
              y[i] = __float_as_uint(z);
            }
            tmem_st16(tS + c16, y);
          }
          tmem_wait_st();
          follow(top);
          if (!ok) break;
          const float base_m = m == -INFINITY ? 0.f : m;
#pragma unroll 1
          for (int c16 = 0; c16 < 128; c16 += 16) {
            uint32_t y[16], w[8];
            tmem_ld16(tS + c16, y);
            tmem_wait_ld16(y);
            const uint4 vb = lds16(powers + 128 + c16);
#pragma unroll
            for (int i = 0; i < 16; i += 2) {
              float pr[2], out[2], pv[2];
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const uint32_t b = byte_of(vb, i + e);
                pr[e] = exp2_fast(__uint_as_float(y[i + e]) - base_m);
                out[e] = power_out(carried(b, kLeastV));
                pv[e] = b == 255u && pr[e] != 0.f ? __uint_as_float(0x7fffffffu) : pr[e];
              }
              l2 = fma_f32x2(pack_f32x2(pr[0], pr[1]), pack_f32x2(out[0], out[1]), l2);
              w[i / 2] = Mma<Op>::pack(pv[0], pv[1]);
            }
            tmem_st8(tS + c16 / 2, w);  // over columns that have been read
          }
        } else {
          if (edge) {
#pragma unroll
            for (int q = 0; q < 4; ++q)
#pragma unroll
              for (int i = 0; i < 32; ++i) x[q][i] = 32 * q + i <= hi && 32 * q + i >= lo ? x[q][i] : -INFINITY;
          }
          float part[4];
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            part[q] = fmaxf(x[q][0], x[q][1]);
#pragma unroll
            for (int i = 2; i < 32; i += 2) part[q] = fmaxf(part[q], fmaxf(x[q][i], x[q][i + 1]));
          }
          if constexpr (FP8) {
#pragma unroll
            for (int q = 0; q < 4; ++q) part[q] = fmaf(part[q], cq[q], fq[q]);
            follow(fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3])));
          } else {
            follow(fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3])) * c_row);
          }
          if (!ok) break;
          if (__builtin_expect(huge, 0)) {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const uint64_t c2 = pack_f32x2(cq[q], cq[q]), f2 = pack_f32x2(fq[q], fq[q]);
#pragma unroll
              for (int i = 0; i < 32; i += 2) unpack_f32x2(fma_f32x2(pack_f32x2(x[q][i], x[q][i + 1]), c2, f2), x[q][i], x[q][i + 1]);
              cq[q] = 1.f;
              fq[q] = 0.f;
            }
          }
          const float base_m = m == -INFINITY ? 0.f : m;
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const uint64_t c2 = pack_f32x2(cq[q], cq[q]), neg = pack_f32x2(fq[q] - base_m, fq[q] - base_m);
            uint64_t quarter = 0;
            uint32_t w[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              float a, b;
              unpack_f32x2(fma_f32x2(pack_f32x2(x[q][2 * i], x[q][2 * i + 1]), c2, neg), a, b);
              a = exp2_fast(a);
              b = exp2_fast(b);
              if constexpr (FP8) quarter = add_f32x2(quarter, pack_f32x2(a, b));
              else l2 = add_f32x2(l2, pack_f32x2(a, b));
              w[i] = Mma<Op>::pack(a, b);
            }
            if constexpr (FP8) {
              const float down = pow2_of(254u - ((f_bytes >> (8 * q)) & 0xffu));  // 2^-F
              l2 = fma_f32x2(quarter, pack_f32x2(down, down), l2);
            }
            tmem_st16(tS + 16 * q, w);  // P lies over the first half of S, which this thread holds in registers
          }
        }
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(bar(BAR_P_FULL + s));
        pv_phase ^= 1u;
      }
      if (!ok) break;
      // ---- the row's result
      float sum0, sum1;
      unpack_f32x2(l2, sum0, sum1);
      const float sum = sum0 + sum1;
      const int tok_row = tok;
      const int head = g.head * p.group + row - tok_row * p.group;
      const int64_t t = g.s.t0 + g.tok0 + tok_row;
      const float inv = g.whole ? (sum > 0.f || sum != sum ? 1.f / sum : 0.f) : 1.f;
      const int slot = part_slot(blockIdx.x, g.starts), part_row = mode == MODE_KEYS ? s * 128 + row_in : row;
      if (done > 0) {
        wait(BAR_PV_DONE + s, pv_phase ^ 1u, ST_EPILOGUE_WAIT);
        if (!ok) break;
        tc_fence_after();
#pragma unroll 1
        for (int q = 0; q < D / 32; ++q) {
          float x[32];
          tmem_ld32(tO + 32 * q, x);
          tmem_wait_ld32(x);
          if (!live) continue;
          if (g.whole) {
            uint4* const dst = reinterpret_cast<uint4*>(p.out + t * p.o_tok + head * p.o_head + 64 * q);
#pragma unroll
            for (int i = 0; i < 4; ++i)
              dst[i] = make_uint4(Mma<T>::pack(x[8 * i] * inv, x[8 * i + 1] * inv), Mma<T>::pack(x[8 * i + 2] * inv, x[8 * i + 3] * inv),
                                  Mma<T>::pack(x[8 * i + 4] * inv, x[8 * i + 5] * inv), Mma<T>::pack(x[8 * i + 6] * inv, x[8 * i + 7] * inv));
          } else {
            // [slot][head_dim / 4][row][4]: a warp's rows lie side by side
            float4* const dst = reinterpret_cast<float4*>(p.part_o) + ((int64_t)slot * (D / 4) + 8 * q) * kTilesRows + part_row;
#pragma unroll
            for (int i = 0; i < 8; ++i) dst[i * kTilesRows] = make_float4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
          }
        }
        tc_fence_before();
      }
      if (live) {
        if (!g.whole) *reinterpret_cast<float2*>(p.part_ml + ((int64_t)slot * kTilesRows + part_row) * 2) = make_float2(done > 0 ? m : -INFINITY, sum);
        else if (p.lse) p.lse[t * p.lse_tok + head] = sum > 0.f || sum != sum ? (m + log2f(sum)) * 0.693147180559945309f : -INFINITY;
      }
      if (tid == 0 && !g.whole) note_split(p, g, rows | (mode == MODE_KEYS ? 1 << 16 : 0));
      done_item();
    }
  }
  __syncthreads();
  if (warp == 12) tmem_dealloc(tmem, 512);
}

}  // namespace llg
