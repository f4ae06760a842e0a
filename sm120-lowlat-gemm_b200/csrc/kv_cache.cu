// Writing new tokens' keys and values into a paged cache, and reading cached rows back.
//
// Writing. Row x of head_dim values: a = max |x|, e = smallest integer with a * 2^-e <= 448 (clamped to [-100, 119], -100 for a
// zero row), stored e4m3(x * 2^-e), round to nearest even, saturating, and the byte e + 127. The multiply by a power of two is
// exact, so the one rounding is the conversion's. An infinity saturates to 448 * 2^119, a NaN stays one. A 16-bit cache is a copy.
// Reading. value * 2^e, one rounding to the output type (none for bf16 and fp32: four significant bits fit).
//
// Both move bytes: 16-byte loads and 8- to 16-byte stores, a row per 8, 16 or 32 lanes, so that a token's heads - one
// contiguous run of the qkv projection - are read by neighbouring lanes, and a row's maximum is a shuffle over its lanes.
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

template <typename T>
__device__ __forceinline__ void load8(const unsigned char* p, float (&f)[8]) {
  if constexpr (sizeof(T) == 4) {
    const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 16);
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w; f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
  } else {
    const uint4 raw = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
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

// LPR lanes per row, 8 values per lane.
template <typename T, bool FP8, int LPR>
__global__ void __launch_bounds__(kThreads) kv_append_kernel(const __grid_constant__ AppendDev p) {
  pdl_trigger();
  pdl_wait();
  const PagedKV& c = p.c;
  const int lane = threadIdx.x & 31, sub = lane % LPR;
  const long long per_tok = 2ll * c.kv_heads;
  const long long rows = per_tok * c.tokens;
  const long long row0 = ((long long)blockIdx.x * kThreads + (threadIdx.x & ~31)) / LPR;  // the warp's first row
  if (row0 >= rows) return;
  const long long row = row0 + lane / LPR;
  const bool there = row < rows;
  const int t = (int)((there ? row : rows - 1) / per_tok);
  int seq;
  if (c.starts) {
    // the rows of a warp belong to at most two tokens unless there are fewer than 32 / LPR rows per token
    const int t_first = __shfl_sync(0xffffffffu, t, 0), t_last = __shfl_sync(0xffffffffu, t, 31);
    seq = 0;
    for (int x = t_first; x <= t_last; ++x) {
      const int s = seq_of(c, x, lane);
      if (x == t) seq = s;
    }
  } else {
    seq = t / c.q_len;
  }
  const int r = (int)((there ? row : rows - 1) - t * per_tok);
  const bool is_v = r >= c.kv_heads;
  const int head = is_v ? r - c.kv_heads : r;
  bool ok = there && sub * 8 < c.head_dim && seq < c.batch;  // seq == batch: a token behind the last sequence
  int pos = 0;
  if (seq < c.batch) {
    const int end = c.starts ? min(c.starts[seq + 1], c.tokens) : (seq + 1) * c.q_len;
    pos = c.lens[seq] - end + t;
    ok = ok && pos >= 0 && pos / c.page_size < c.table_width && (!c.starts || t >= c.starts[seq]);
  } else {
    ok = false;
  }
  int pg = -1;
  if (ok) pg = page_of(c, seq, pos / c.page_size);
  ok = ok && pg >= 0;
  const int slot = pos % c.page_size;
  const unsigned char* src = is_v ? p.v + t * p.v_tok + head * p.v_head : p.k + t * p.k_tok + head * p.k_head;
  src += sub * 8 * sizeof(T);
  unsigned char* const dst = is_v ? c.v + pg * c.v_page + head * c.v_head + slot * c.v_slot
                                  : c.k + pg * c.k_page + head * c.k_head + slot * c.k_slot;
  if constexpr (FP8) {
    float f[8] = {};
    if (ok) load8<T>(src, f);
    float a = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) a = fmaxf(a, fabsf(f[i]));
#pragma unroll
    for (int o = LPR / 2; o >= 1; o >>= 1) a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, o));
    const int e = row_exponent(a);
    const float inv = __uint_as_float((uint32_t)(127 - e) << 23);
    if (!ok) return;
    uint2 q;
    q.x = cvt_e4m3x2(f[0] * inv, f[1] * inv) | (cvt_e4m3x2(f[2] * inv, f[3] * inv) << 16);
    q.y = cvt_e4m3x2(f[4] * inv, f[5] * inv) | (cvt_e4m3x2(f[6] * inv, f[7] * inv) << 16);
    *reinterpret_cast<uint2*>(dst + sub * 8) = q;
    if (sub == 0) {
      unsigned char* const s = is_v ? c.vs + pg * c.vs_page + head * c.vs_head + slot * c.vs_slot
                                    : c.ks + pg * c.ks_page + head * c.ks_head + slot * c.ks_slot;
      *s = (unsigned char)(e + 127);
    }
  } else {
    if (ok) *reinterpret_cast<uint4*>(dst + sub * 16) = *reinterpret_cast<const uint4*>(src);
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

// LPR lanes per row, 8 values per lane; rows in the order of the output.
template <typename T, bool FP8, int LPR>
__global__ void __launch_bounds__(kThreads) kv_read_kernel(const __grid_constant__ ReadDev p) {
  pdl_trigger();
  pdl_wait();
  const PagedKV& c = p.c;
  const int sub = threadIdx.x % LPR;
  const long long rows = (long long)c.batch * p.max_len * c.kv_heads;
  const long long row = ((long long)blockIdx.x * kThreads + threadIdx.x) / LPR;
  if (row >= rows || sub * 8 >= c.head_dim) return;
  const bool is_v = blockIdx.y != 0;
  const int head = (int)(row % c.kv_heads);
  const long long bt = row / c.kv_heads;
  const int seq = (int)(bt / p.max_len), pos = (int)(bt - (long long)seq * p.max_len);
  unsigned char* const dst = (is_v ? p.v : p.k) + (row * c.head_dim + sub * 8) * (int64_t)sizeof(T);
  int pg = -1;
  if (pos < c.lens[seq] && pos / c.page_size < c.table_width) pg = page_of(c, seq, pos / c.page_size);
  const int slot = pos % c.page_size;
  const unsigned char* const src = is_v ? c.v + pg * c.v_page + head * c.v_head + slot * c.v_slot
                                        : c.k + pg * c.k_page + head * c.k_head + slot * c.k_slot;
  if constexpr (FP8) {
    float f[8] = {};
    if (pg >= 0) {
      const unsigned char* const s = is_v ? c.vs + pg * c.vs_page + head * c.vs_head + slot * c.vs_slot
                                          : c.ks + pg * c.ks_page + head * c.ks_head + slot * c.ks_slot;
      const uint2 q = *reinterpret_cast<const uint2*>(src + sub * 8);
      const float up = __uint_as_float((uint32_t)*s << 23);
      const float2 a = e4m3x2_to_f32(q.x & 0xffffu), b = e4m3x2_to_f32(q.x >> 16);
      const float2 d = e4m3x2_to_f32(q.y & 0xffffu), e = e4m3x2_to_f32(q.y >> 16);
      f[0] = a.x * up; f[1] = a.y * up; f[2] = b.x * up; f[3] = b.y * up;
      f[4] = d.x * up; f[5] = d.y * up; f[6] = e.x * up; f[7] = e.y * up;
    }
    if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<float4*>(dst) = make_float4(f[0], f[1], f[2], f[3]);
      *reinterpret_cast<float4*>(dst + 16) = make_float4(f[4], f[5], f[6], f[7]);
    } else {
      T o[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if constexpr (std::is_same<T, __half>::value) o[i] = __float2half_rn(f[i]);
        else o[i] = __float2bfloat16_rn(f[i]);
      }
      *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(o);
    }
  } else {
    *reinterpret_cast<uint4*>(dst) = pg >= 0 ? *reinterpret_cast<const uint4*>(src + sub * 16) : make_uint4(0u, 0u, 0u, 0u);
  }
}

int lanes_of(int head_dim) { return head_dim <= 64 ? 8 : head_dim <= 128 ? 16 : 32; }

template <typename T, bool FP8>
cudaError_t append(const AppendDev& p, cudaStream_t s) {
  const int lpr = lanes_of(p.c.head_dim);
  const long long threads = 2ll * p.c.kv_heads * p.c.tokens * lpr;
  const dim3 grid((unsigned)((threads + kThreads - 1) / kThreads)), block(kThreads), one(1, 1, 1);
  switch (lpr) {
    case 8: return launch_ex(kv_append_kernel<T, FP8, 8>, grid, block, 0, s, pdl_on(), one, p);
    case 16: return launch_ex(kv_append_kernel<T, FP8, 16>, grid, block, 0, s, pdl_on(), one, p);
    default: return launch_ex(kv_append_kernel<T, FP8, 32>, grid, block, 0, s, pdl_on(), one, p);
  }
}

template <typename T, bool FP8>
cudaError_t read(const ReadDev& p, cudaStream_t s) {
  const int lpr = lanes_of(p.c.head_dim);
  const long long threads = (long long)p.c.batch * p.max_len * p.c.kv_heads * lpr;
  const dim3 grid((unsigned)((threads + kThreads - 1) / kThreads), 2), block(kThreads), one(1, 1, 1);
  switch (lpr) {
    case 8: return launch_ex(kv_read_kernel<T, FP8, 8>, grid, block, 0, s, pdl_on(), one, p);
    case 16: return launch_ex(kv_read_kernel<T, FP8, 16>, grid, block, 0, s, pdl_on(), one, p);
    default: return launch_ex(kv_read_kernel<T, FP8, 32>, grid, block, 0, s, pdl_on(), one, p);
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
