// Adds the partial results of items that several CTAs shared: o = sum_i 2^(m_i - M) o_i / sum_i 2^(m_i - M) l_i, in the order
// of the CTAs. Bound by the latency of reading a few kilobytes back from L2; a row's parts are spread over the warps of a CTA
// (a long sequence of few heads leaves one part per SM) and every warp keeps four of its parts in flight.
#include "paged_kv.cuh"

namespace llg {
namespace {

template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

constexpr int kWarps = 8;

// blockIdx.x: the main kernel's CTA whose share ends inside an item. SPREAD warps work on one row, blockIdx.y counts groups of
// kWarps / SPREAD rows.
template <typename T, int D, int SPREAD>
__global__ void __launch_bounds__(32 * kWarps) attn_combine_kernel(const __grid_constant__ AttnDev p, int tile_rows) {
  constexpr int V = D / 32;  // values per lane
  __shared__ float part[kWarps][D + 2];
  pdl_trigger();
  pdl_wait();
  int4 item = p.split[blockIdx.x];
  if (item.x == 0) return;
  const int twice = item.w >> 16;  // two parts per CTA
  item.w &= 0xffff;
  item.x <<= twice;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, share = warp % SPREAD;
  const int row = blockIdx.y * (kWarps / SPREAD) + warp / SPREAD;
  const bool live = row < item.w;
  float top = -INFINITY, sum = 0.f, acc[V] = {};
  if (live) {
    // parts share, share + SPREAD, ...: 32 of them at a time, one per lane
    for (int i0 = share; i0 < item.x; i0 += 32 * SPREAD) {
      const int i = i0 + lane * SPREAD;
      float2 ml = make_float2(-INFINITY, 0.f);
      int64_t at = 0;
      if (i < item.x) {
        const int cta = i >> twice;
        at = (int64_t)part_slot(blockIdx.x + cta, cta == 0) * tile_rows + row + (twice & i ? 128 : 0);
        ml = *reinterpret_cast<const float2*>(p.part_ml + at * 2);
      }
      float mx = ml.x;
#pragma unroll
      for (int o = 16; o >= 1; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
      const float now = fmaxf(top, mx);
      const float keep = top == -INFINITY ? 0.f : exp2f(top - now);
      const float w = ml.x == -INFINITY ? 0.f : exp2f(ml.x - now);
      top = now;
      sum = sum * keep + w * ml.y;  // this lane's parts only
#pragma unroll
      for (int v = 0; v < V; ++v) acc[v] *= keep;
      const int n = min(32, (item.x - i0 + SPREAD - 1) / SPREAD);
#pragma unroll 4
      for (int j = 0; j < n; ++j) {
        const float f = __shfl_sync(0xffffffffu, w, j);
        const int64_t a = __shfl_sync(0xffffffffu, at, j);
        if (f == 0.f) continue;  // a part without keys has no sums
        const float* const src = p.part_o + a * D + lane * V;
        if constexpr (V == 4) {
          const float4 x = *reinterpret_cast<const float4*>(src);
          acc[0] += f * x.x; acc[1] += f * x.y; acc[2] += f * x.z; acc[3] += f * x.w;
        } else {
          const float2 x = *reinterpret_cast<const float2*>(src);
          acc[0] += f * x.x; acc[1] += f * x.y;
        }
      }
    }
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  }
  if constexpr (SPREAD > 1) {
#pragma unroll
    for (int v = 0; v < V; ++v) part[warp][lane * V + v] = acc[v];
    if (lane == 0) {
      part[warp][D] = top;
      part[warp][D + 1] = sum;
    }
    __syncthreads();
    if (share != 0 || !live) return;
    float all = top;
#pragma unroll
    for (int s = 1; s < SPREAD; ++s) all = fmaxf(all, part[warp + s][D]);
    const float base = all == -INFINITY ? 0.f : all;
    sum = 0.f;
#pragma unroll
    for (int v = 0; v < V; ++v) acc[v] = 0.f;
#pragma unroll
    for (int s = 0; s < SPREAD; ++s) {
      const float f = exp2f(part[warp + s][D] - base);
      sum += f * part[warp + s][D + 1];
#pragma unroll
      for (int v = 0; v < V; ++v) acc[v] += f * part[warp + s][lane * V + v];
    }
    top = base;
  }
  if (!live) return;
  const float inv = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
  const int tok = row / p.group, head = item.z * p.group + row - tok * p.group;
  const int64_t t = item.y + tok;
  unsigned char* const dst = p.out + t * p.o_tok + head * p.o_head + 2 * V * lane;
  if constexpr (V == 4)
    *reinterpret_cast<uint2*>(dst) = make_uint2(pack2<T>(acc[0] * inv, acc[1] * inv), pack2<T>(acc[2] * inv, acc[3] * inv));
  else
    *reinterpret_cast<uint32_t*>(dst) = pack2<T>(acc[0] * inv, acc[1] * inv);
  if (p.lse && lane == 0) p.lse[t * p.lse_tok + head] = sum > 0.f || sum != sum ? (top + log2f(sum)) * 0.693147180559945309f : -INFINITY;
}

template <typename T, int D>
cudaError_t combine(const AttnDev& p, int ctas, int tile_rows, cudaStream_t s) {
  const dim3 block(32 * kWarps), one(1, 1, 1);
  // Few rows per item come with many parts (a long cache), many rows with two or three: one row per CTA or one per warp.
  if (tile_rows <= 32) return launch_ex(attn_combine_kernel<T, D, kWarps>, dim3(ctas, tile_rows), block, 0, s, true, one, p, tile_rows);
  return launch_ex(attn_combine_kernel<T, D, 1>, dim3(ctas, tile_rows / kWarps), block, 0, s, true, one, p, tile_rows);
}

}  // namespace

cudaError_t attn_combine_launch(const AttnDev& p, bool f16, int ctas, int tile_rows, cudaStream_t s) {
  if (p.c.head_dim == 128)
    return f16 ? combine<__half, 128>(p, ctas, tile_rows, s) : combine<__nv_bfloat16, 128>(p, ctas, tile_rows, s);
  return f16 ? combine<__half, 64>(p, ctas, tile_rows, s) : combine<__nv_bfloat16, 64>(p, ctas, tile_rows, s);
}

}  // namespace llg
