// Writing new tokens' keys and values into a paged cache, and reading cached rows back.
//
// Writing. Row x of head_dim values: a = max |x|, e = smallest integer with a * 2^-e <= 448 (clamped to [-100, 119], -100 for a
// zero row), stored e4m3(x * 2^-e), round to nearest even, saturating, and the byte e + 127. The multiply by a power of two is
// exact, so the one rounding is the conversion's. An infinity saturates to 448 * 2^119, a NaN stays one. A 16-bit cache is a copy.
// Reading. value * 2^e (NaN for byte 255), one rounding to the output type (none for bf16 and fp32 from byte 27 on: four significant
// bits fit).
//
// Both move bytes. A CTA takes a few tokens: a thread per token finds its page and slot once, then the rows of all heads go
// through, 16 values (append: of K's row and of V's) or 8 (read) per lane, a row on 4 to 32 lanes so that a row's maximum is a
// shuffle, several rows requested before the first is written. Measured: 8192 tokens of 8 kv heads, bf16 into e4m3, 12.3 us
// (4.1 TB/s of read and written bytes; conversions and maxima fill 60% of the issue slots); 8 x 8192 tokens back to bf16 72 us (5.4 TB/s; 80
// with 16 values per lane, whose two stores each touched half of every sector).
#include <type_traits>

#include "paged_kv.cuh"

namespace llg {
namespace {

constexpr int kThreads = 256;

// Sequence of token t: the number of entries of starts[1..batch] that are <= t, by 32-way search; every lane of the warp takes part.
__device__ __forceinline__ int seq_of(const PagedKV& c, int t, int lane) {
  int lo = 0, n = c.batch;  // the answer lies in [lo, lo + n]
  while (n > 0) {
    const int step = (n + 31) >> 5;
    const int at = lo + (lane + 1) * step;  // entries of blocks up to this lane's are all <= t when entry `at` is
    const bool le = (lane + 1) * step <= n && c.starts[at] <= t;
    const int full = __popc(__ballot_sync(0xffffffffu, le));
    lo += full * step;
    n = min(n - full * step, step - 1);
  }
  return lo;
}

// 16 values of type T held in raw words.
template <typename T>
__device__ __forceinline__ void as_floats(const uint4* raw, float (&f)[16]) {
  const uint32_t* const w = reinterpret_cast<const uint32_t*>(raw);
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 16; ++i) f[i] = __uint_as_float(w[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float2 v;
      if constexpr (std::is_same<T, __half>::value) v = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      else v = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w[i]));
      f[2 * i] = v.x;
      f[2 * i + 1] = v.y;
    }
  }
}

struct AppendDev {
  PagedKV c;
  const unsigned char *k, *v;
  int64_t k_tok, k_head, v_tok, v_head;  // bytes
};

// Smallest e with a * 2^-e <= 448 = 1.75 * 2^8, from the bits of a.
__device__ __forceinline__ int row_exponent(float a) {
  const uint32_t bits = __float_as_uint(a);
  const int e = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  return min(max(e, -100), 119);
}

// Where a token lies in the cache; pg < 0: nowhere.
struct Place {
  int pg, slot;
};
constexpr int kMaxTokens = 32;  // tokens per CTA at most

// One row of K or V, 16 of its values per lane.
template <typename T, bool FP8, int LPR>
__device__ __forceinline__ void put_row(const uint4* raw, unsigned char* dst, unsigned char* scale, int sub, bool ok) {
  if constexpr (FP8) {
    float f[16];
    as_floats<T>(raw, f);
    float a = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) a = fmaxf(a, fabsf(f[i]));
#pragma unroll
    for (int o = LPR / 2; o >= 1; o >>= 1) a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, o));
    const int e = row_exponent(a);
    const float inv = __uint_as_float((uint32_t)(127 - e) << 23);
    if (!ok) return;
    uint32_t q[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      q[i] = cvt_e4m3x2(f[4 * i] * inv, f[4 * i + 1] * inv) | (cvt_e4m3x2(f[4 * i + 2] * inv, f[4 * i + 3] * inv) << 16);
    *reinterpret_cast<uint4*>(dst + sub * 16) = make_uint4(q[0], q[1], q[2], q[3]);
    if (sub == 0) *scale = (unsigned char)(e + 127);
  } else {
    if (!ok) return;
    reinterpret_cast<uint4*>(dst + sub * 32)[0] = raw[0];
    reinterpret_cast<uint4*>(dst + sub * 32)[1] = raw[1];
  }
}

// LPR lanes per row; tokens [blockIdx.x * per, + per).
template <typename T, bool FP8, int LPR>
__global__ void __launch_bounds__(kThreads) kv_append_kernel(const __grid_constant__ AppendDev p, int per) {
  __shared__ Place where[kMaxTokens];
  pdl_trigger();
  pdl_wait();
  const PagedKV& c = p.c;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = threadIdx.x % LPR;
  const int t0 = blockIdx.x * per, count = min(per, c.tokens - t0);
  for (int i = warp; i < count; i += kThreads / 32) {  // a warp per token: its sequence by 32-way search
    const int t = t0 + i;
    const int seq = c.starts ? seq_of(c, t, lane) : t / c.q_len;
    Place w{-1, 0};
    if (lane == 0) {
      if (seq < c.batch && (!c.starts || t >= c.starts[seq])) {  // seq == batch: behind the last sequence
        const int end = c.starts ? min(c.starts[seq + 1], c.tokens) : (seq + 1) * c.q_len;
        const int pos = max(c.lens[seq], 0) - end + t;
        if (pos >= 0) {
          int block;
          split_key(c, pos, block, w.slot);
          if (block < c.table_width) w.pg = page_of(c, seq, block);
        }
      }
      where[i] = w;
    }
  }
  __syncthreads();
  const int rows = count * c.kv_heads;
  constexpr int kRowsPass = kThreads / LPR, kAhead = sizeof(T) == 4 ? 1 : 2, W = sizeof(T);  // 16-byte words per lane and row
  const bool in_row = sub * 16 < c.head_dim;
  const int mine = threadIdx.x / LPR;
  for (int r0 = 0; r0 < rows; r0 += kRowsPass * kAhead) {  // the same for every lane: rows' maxima are shuffles
    uint4 k[kAhead][W], v[kAhead][W];
    Place at[kAhead];
    int head[kAhead];
#pragma unroll
    for (int a = 0; a < kAhead; ++a) {
      const int r = r0 + a * kRowsPass + mine;
      at[a] = Place{-1, 0};
      head[a] = 0;
#pragma unroll
      for (int w = 0; w < W; ++w) k[a][w] = v[a][w] = make_uint4(0u, 0u, 0u, 0u);
      if (r < rows) {
        const int i = r / c.kv_heads;
        head[a] = r - i * c.kv_heads;
        at[a] = where[i];
        if (at[a].pg >= 0 && in_row) {
          const int64_t t = t0 + i;
          const uint4* const ks = reinterpret_cast<const uint4*>(p.k + t * p.k_tok + head[a] * p.k_head) + sub * W;
          const uint4* const vs = reinterpret_cast<const uint4*>(p.v + t * p.v_tok + head[a] * p.v_head) + sub * W;
#pragma unroll
          for (int w = 0; w < W; ++w) {
            k[a][w] = ks[w];
            v[a][w] = vs[w];
          }
        }
      }
    }
#pragma unroll
    for (int a = 0; a < kAhead; ++a) {
      const bool ok = at[a].pg >= 0 && in_row;
      const int64_t pg = at[a].pg, slot = at[a].slot, h = head[a];
      put_row<T, FP8, LPR>(k[a], c.k + pg * c.k_page + h * c.k_head + slot * c.k_slot,
                           c.ks + (pg * c.ks_page + h * c.ks_head + slot * c.ks_slot), sub, ok);
      put_row<T, FP8, LPR>(v[a], c.v + pg * c.v_page + h * c.v_head + slot * c.v_slot,
                           c.vs + (pg * c.vs_page + h * c.vs_head + slot * c.vs_slot), sub, ok);
    }
  }
}

struct ReadDev {
  PagedKV c;
  unsigned char *k, *v;                        // [batch, max_len, kv_heads, head_dim], contiguous
  int max_len;
};

__device__ __forceinline__ float2 e4m3x2_to_f32(uint32_t v) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)v));
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

// LPR lanes per row, 8 values per lane, so that a 16-bit row is written 16 bytes by 16 bytes without gaps; tokens [blockIdx.x * per,
// + per) of sequence blockIdx.y; blockIdx.z: K or V. Rows go through in the order of the output.
template <typename T, bool FP8, int LPR>
__global__ void __launch_bounds__(kThreads) kv_read_kernel(const __grid_constant__ ReadDev p, int per) {
  __shared__ Place where[kMaxTokens];
  pdl_trigger();
  pdl_wait();
  const PagedKV& c = p.c;
  const int seq = blockIdx.y, t0 = blockIdx.x * per, count = min(per, p.max_len - t0);
  const bool is_v = blockIdx.z != 0;
  const int sub = threadIdx.x % LPR;
  constexpr int kValues = 8;  // per lane
  using Raw = typename std::conditional<FP8, uint2, uint4>::type;
  if (threadIdx.x < count) {
    const int pos = t0 + threadIdx.x;
    Place w{-1, 0};
    if (pos < c.lens[seq]) {
      int block;
      split_key(c, pos, block, w.slot);
      if (block < c.table_width) w.pg = page_of(c, seq, block);
    }
    where[threadIdx.x] = w;
  }
  __syncthreads();
  if (sub * kValues >= c.head_dim) return;
  const unsigned char* const base = is_v ? c.v : c.k;
  const unsigned char* const scales = is_v ? c.vs : c.ks;
  const int64_t s_page = is_v ? c.v_page : c.k_page, s_head = is_v ? c.v_head : c.k_head, s_slot = is_v ? c.v_slot : c.k_slot;
  const int64_t c_page = is_v ? c.vs_page : c.ks_page, c_head = is_v ? c.vs_head : c.ks_head, c_slot = is_v ? c.vs_slot : c.ks_slot;
  unsigned char* const out = (is_v ? p.v : p.k) + ((int64_t)seq * p.max_len + t0) * c.kv_heads * c.head_dim * (int64_t)sizeof(T);
  const int rows = count * c.kv_heads;
  constexpr int kRowsPass = kThreads / LPR, kAhead = FP8 ? 8 : 4;
  for (int r0 = threadIdx.x / LPR; r0 < rows; r0 += kRowsPass * kAhead) {
    Raw raw[kAhead];
    uint32_t b[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int r = r0 + k * kRowsPass;
      raw[k] = Raw{};
      b[k] = 0u;
      if (r < rows) {
        const int i = r / c.kv_heads, head = r - i * c.kv_heads;
        const Place w = where[i];
        if (w.pg >= 0) {
          raw[k] = *reinterpret_cast<const Raw*>(base + w.pg * s_page + head * s_head + w.slot * s_slot + sub * (int)sizeof(Raw));
          if constexpr (FP8) b[k] = scales[w.pg * c_page + head * c_head + w.slot * c_slot];
        }
      }
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int r = r0 + k * kRowsPass;
      if (r >= rows) break;
      unsigned char* const dst = out + ((int64_t)r * c.head_dim + sub * kValues) * (int64_t)sizeof(T);
      if constexpr (FP8) {
        const float up = e8m0_value(b[k]);
        const float2 x[4] = {e4m3x2_to_f32(raw[k].x & 0xffffu), e4m3x2_to_f32(raw[k].x >> 16), e4m3x2_to_f32(raw[k].y & 0xffffu),
                             e4m3x2_to_f32(raw[k].y >> 16)};
        float f[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          f[2 * i] = x[i].x * up;
          f[2 * i + 1] = x[i].y * up;
        }
        if constexpr (sizeof(T) == 4) {
#pragma unroll
          for (int i = 0; i < 2; ++i) __stcs(reinterpret_cast<float4*>(dst) + i, make_float4(f[4 * i], f[4 * i + 1], f[4 * i + 2], f[4 * i + 3]));
        } else {
          alignas(16) T o[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            if constexpr (std::is_same<T, __half>::value) o[i] = __float2half_rn(f[i]);
            else o[i] = __float2bfloat16_rn(f[i]);
          }
          __stcs(reinterpret_cast<uint4*>(dst), *reinterpret_cast<const uint4*>(o));
        }
      } else {
        __stcs(reinterpret_cast<uint4*>(dst), raw[k]);
      }
    }
  }
}

int lanes_for(int pieces) { return pieces <= 4 ? 4 : pieces <= 8 ? 8 : pieces <= 16 ? 16 : 32; }

// Tokens per CTA: as many as keep `ahead` rows per lane group in flight, fewer while that leaves SMs without a CTA.
int tokens_per_cta(long long tokens, int heads, int lpr, int ahead) {
  int per = ahead * (kThreads / lpr) / heads;
  per = per < 1 ? 1 : per > kMaxTokens ? kMaxTokens : per;
  while (per > 1 && (tokens + per - 1) / per < 2 * sm_count()) per /= 2;
  return per;
}

template <typename T, bool FP8>
cudaError_t append(const AppendDev& p, cudaStream_t s) {
  const int lpr = lanes_for(p.c.head_dim / 16);
  const int per = tokens_per_cta(p.c.tokens, p.c.kv_heads, lpr, sizeof(T) == 4 ? 1 : 2);
  const dim3 grid((unsigned)((p.c.tokens + per - 1) / per)), block(kThreads), one(1, 1, 1);
  switch (lpr) {
    case 4: return launch_ex(kv_append_kernel<T, FP8, 4>, grid, block, 0, s, pdl_on(), one, p, per);
    case 8: return launch_ex(kv_append_kernel<T, FP8, 8>, grid, block, 0, s, pdl_on(), one, p, per);
    default: return launch_ex(kv_append_kernel<T, FP8, 16>, grid, block, 0, s, pdl_on(), one, p, per);
  }
}

template <typename T, bool FP8>
cudaError_t read(const ReadDev& p, cudaStream_t s) {
  const int lpr = lanes_for(p.c.head_dim / 8);
  const int per = tokens_per_cta((long long)p.c.batch * p.max_len * 2, p.c.kv_heads, lpr, FP8 ? 8 : 4);
  const dim3 grid((unsigned)((p.max_len + per - 1) / per), (unsigned)p.c.batch, 2), block(kThreads), one(1, 1, 1);
  switch (lpr) {
    case 4: return launch_ex(kv_read_kernel<T, FP8, 4>, grid, block, 0, s, pdl_on(), one, p, per);
    case 8: return launch_ex(kv_read_kernel<T, FP8, 8>, grid, block, 0, s, pdl_on(), one, p, per);
    case 16: return launch_ex(kv_read_kernel<T, FP8, 16>, grid, block, 0, s, pdl_on(), one, p, per);
    default: return launch_ex(kv_read_kernel<T, FP8, 32>, grid, block, 0, s, pdl_on(), one, p, per);
  }
}

int esize(int dt) { return dt == LLG_DT_F32 ? 4 : dt == LLG_DT_E4M3 ? 1 : 2; }

}  // namespace

PagedKV paged_view(const llg_paged_kv& a, unsigned* status) {
  PagedKV c{};
  const int64_t es = esize(a.dtype);
  c.k = static_cast<unsigned char*>(a.k);
  c.v = static_cast<unsigned char*>(a.v);
  c.k_page = a.k_stride[0] * es; c.k_head = a.k_stride[1] * es; c.k_slot = a.k_stride[2] * es;
  c.v_page = a.v_stride[0] * es; c.v_head = a.v_stride[1] * es; c.v_slot = a.v_stride[2] * es;
  c.ks = static_cast<unsigned char*>(a.k_scale);
  c.vs = static_cast<unsigned char*>(a.v_scale);
  c.ks_page = a.k_scale_stride[0]; c.ks_head = a.k_scale_stride[1]; c.ks_slot = a.k_scale_stride[2];
  c.vs_page = a.v_scale_stride[0]; c.vs_head = a.v_scale_stride[1]; c.vs_slot = a.v_scale_stride[2];
  c.table = a.page_table;
  c.table_stride = a.table_stride;
  c.lens = a.kv_lens;
  c.starts = a.q_starts;
  c.pages = a.pages; c.kv_heads = a.kv_heads; c.page_size = a.page_size; c.head_dim = a.head_dim;
  c.table_width = a.table_width; c.batch = a.batch; c.tokens = a.tokens;
  c.q_len = a.batch > 0 ? a.tokens / a.batch : 0;
  c.page_shift = (a.page_size & (a.page_size - 1)) == 0 ? __builtin_ctz(a.page_size) : -1;
  c.status = status;
  return c;
}

cudaError_t kv_append_launch(const llg_kv_append_args& a, unsigned* status, cudaStream_t s) {
  AppendDev p{};
  p.c = paged_view(a.kv, status);
  const int64_t es = esize(a.in_dtype);
  p.k = static_cast<const unsigned char*>(a.k_in);
  p.v = static_cast<const unsigned char*>(a.v_in);
  p.k_tok = a.k_in_stride[0] * es; p.k_head = a.k_in_stride[1] * es;
  p.v_tok = a.v_in_stride[0] * es; p.v_head = a.v_in_stride[1] * es;
  if (a.kv.dtype != LLG_DT_E4M3) return append<__half, false>(p, s);  // a copy: the type does not matter
  switch (a.in_dtype) {
    case LLG_DT_BF16: return append<__nv_bfloat16, true>(p, s);
    case LLG_DT_F16: return append<__half, true>(p, s);
    default: return append<float, true>(p, s);
  }
}

cudaError_t kv_read_launch(const llg_kv_read_args& a, unsigned* status, cudaStream_t s) {
  ReadDev p{};
  p.c = paged_view(a.kv, status);
  p.k = static_cast<unsigned char*>(a.k_out);
  p.v = static_cast<unsigned char*>(a.v_out);
  p.max_len = a.max_len;
  if (a.kv.dtype != LLG_DT_E4M3) return read<__half, false>(p, s);
  switch (a.out_dtype) {
    case LLG_DT_BF16: return read<__nv_bfloat16, true>(p, s);
    case LLG_DT_F16: return read<__half, true>(p, s);
    default: return read<float, true>(p, s);
  }
}

}  // namespace llg
