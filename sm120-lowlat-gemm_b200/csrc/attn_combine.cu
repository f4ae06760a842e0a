// Adds the partial results of items that several CTAs shared: o = sum_i 2^(m_i - M) o_i / sum_i 2^(m_i - M) l_i, in the order
// of the CTAs. Bound by the latency of reading a few kilobytes back from L2. The CTAs of the main kernel that shared an item are
// also the indexes of those that add it up here, each its part of the rows: a long sequence of few heads, with a part from every
// SM, so has all SMs at work, two parts have two. A CTA with fewer rows than warps puts several warps on a row. One launch serves both
// kernels (two cost a ragged batch 2.5 us), in 64 registers: four CTAs per SM took 1.5 us less than three behind 296 CTAs.
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

// Running sum of one row's parts, as one warp holds it: V values of head_dim per lane.
template <int V>
struct RowSum {
  float top = -INFINITY, sum = 0.f, acc[V] = {};
};

// Parts share, share + spread, ... of the row: 32 of them at a time, one per lane, then one after the other.
template <int V>
__device__ __forceinline__ void add_parts(const AttnDev& p, RowSum<V>& s, int parts, int first, int tile_rows, int row, int share,
                                          int spread, int lane) {
  for (int i0 = share; i0 < parts; i0 += 32 * spread) {
    const int i = i0 + lane * spread;
    float2 ml = make_float2(-INFINITY, 0.f);
    int64_t at = 0;
    if (i < parts) {
      at = (int64_t)part_slot(first + i, i == 0) * tile_rows + row;
      ml = *reinterpret_cast<const float2*>(p.part_ml + at * 2);
    }
    // the first sums are requested before their weights are known
    const int n = min(32, (parts - i0 + spread - 1) / spread);
    float x[4][V];
    auto get = [&](int j, float (&v)[V]) {
      const int64_t a = __shfl_sync(0xffffffffu, at, j);
      const float* const src = p.part_o + a * (32 * V) + lane * V;
      if constexpr (V == 4) *reinterpret_cast<float4*>(v) = *reinterpret_cast<const float4*>(src);
      else *reinterpret_cast<float2*>(v) = *reinterpret_cast<const float2*>(src);
    };
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j < n) get(j, x[j]);
    float mx = ml.x;
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    const float now = fmaxf(s.top, mx);
    const float keep = s.top == -INFINITY ? 0.f : exp2f(s.top - now);
    const float w = ml.x == -INFINITY ? 0.f : exp2f(ml.x - now);
    s.top = now;
    s.sum = s.sum * keep + w * ml.y;  // this lane's parts only
#pragma unroll
    for (int v = 0; v < V; ++v) s.acc[v] *= keep;
    for (int j0 = 0; j0 < n; j0 += 4) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float f = __shfl_sync(0xffffffffu, w, j0 + j);
        if (j0 + j < n && f != 0.f) {  // a part without keys has no sums
#pragma unroll
          for (int v = 0; v < V; ++v) s.acc[v] += f * x[j][v];
        }
      }
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (j0 + 4 + j < n) get(j0 + 4 + j, x[j]);
    }
  }
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) s.sum += __shfl_xor_sync(0xffffffffu, s.sum, o);
}

// One CTA for each of the two items that CTA `cta` of the few-row kernel may share with others.
template <typename T, int D>
__device__ __forceinline__ void combine_rows(const AttnDev& p, int cta, int e, int tile_rows, float (*part)[D + 2]) {
  constexpr int V = D / 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int4 item = p.split[2 * cta + e];
  const int went_on = p.first[cta];  // only looked at when an item went on
  if (item.x == 0) return;
  {
    const int rows = item.w;
    const int first = e == 0 ? went_on : cta;
    // this CTA's rows: worker, worker + workers, ...
    const int workers = item.x, worker = cta - first;
    const int mine = worker < rows ? (rows - worker + workers - 1) / workers : 0;
    const int spread = mine >= kWarps ? 1 : mine >= 4 ? 2 : mine >= 2 ? 4 : kWarps;  // warps per row
    const int share = warp % spread;
    for (int r0 = 0; r0 < mine; r0 += kWarps / spread) {
      const int index = r0 + warp / spread;
      const bool live = index < mine;
      const int row = worker + index * workers;
      RowSum<V> s;
      if (live) add_parts<V>(p, s, item.x, first, tile_rows, row, share, spread, lane);
      if (spread > 1) {
        __syncthreads();
#pragma unroll
        for (int v = 0; v < V; ++v) part[warp][lane * V + v] = s.acc[v];
        if (lane == 0) {
          part[warp][D] = s.top;
          part[warp][D + 1] = s.sum;
        }
        __syncthreads();
        float all = -INFINITY;
        for (int q = 0; q < spread; ++q) all = fmaxf(all, part[warp - share + q][D]);
        s.top = all == -INFINITY ? 0.f : all;
        s.sum = 0.f;
#pragma unroll
        for (int v = 0; v < V; ++v) s.acc[v] = 0.f;
        for (int q = 0; q < spread; ++q) {
          const float* const from = part[warp - share + q];
          const float f = exp2f(from[D] - s.top);
          s.sum += f * from[D + 1];
#pragma unroll
          for (int v = 0; v < V; ++v) s.acc[v] += f * from[lane * V + v];
        }
      }
      if (!live || share != 0) continue;
      const float inv = s.sum > 0.f || s.sum != s.sum ? 1.f / s.sum : 0.f;
      const int tok = row / p.group, head = item.z * p.group + row - tok * p.group;
      const int64_t t = item.y + tok;
      unsigned char* const dst = p.out + t * p.o_tok + head * p.o_head + 2 * V * lane;
      if constexpr (V == 4)
        *reinterpret_cast<uint2*>(dst) = make_uint2(pack2<T>(s.acc[0] * inv, s.acc[1] * inv), pack2<T>(s.acc[2] * inv, s.acc[3] * inv));
      else
        *reinterpret_cast<uint32_t*>(dst) = pack2<T>(s.acc[0] * inv, s.acc[1] * inv);
      if (p.lse && lane == 0)
        p.lse[t * p.lse_tok + head] = s.sum > 0.f || s.sum != s.sum ? (s.top + log2f(s.sum)) * 0.693147180559945309f : -INFINITY;
    }
  }
}

// Parts of the tile kernel, [slot][head_dim / 4][256 rows][4]: a warp takes 32 rows, one per lane, and eight values of each. With
// many parts (few rows of a long cache) the CTA's warps share that work, each every eighth part. kTileShare CTAs for each of the
// two items that CTA `cta` of the tile kernel may share with others; this is number `nth`.
constexpr int kTileShare = 4;
template <typename T, int D>
__device__ __forceinline__ void combine_tiles(const AttnDev& p, int cta, int e, int nth, float (*state)[10][32]) {
  constexpr int kRows = 256;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int4 item = p.split[2 * cta + e];
  const int went_on = p.first[cta];
  if (item.x == 0) return;
  const int twice = item.w >> 16, rows = item.w & 0xffff, parts = item.x << twice;
  const int first = e == 0 ? went_on : cta;
  const bool shared = parts > 2 * kWarps;  // by the whole CTA
  const int lanes = shared ? 1 : kWarps;
  const int workers = item.x * kTileShare * lanes;
  const int worker = ((cta - first) * kTileShare + nth) * lanes + (shared ? 0 : warp);
  const int units = (rows + 31) / 32 * (D / 8);
  const int from = shared ? warp : 0, stride = shared ? kWarps : 1;
  const float4* const o = reinterpret_cast<const float4*>(p.part_o);
  for (int u = worker; u < units; u += workers) {
    const int row = u / (D / 8) * 32 + lane, c = u % (D / 8);
    const bool live = row < rows;
    float top = -INFINITY, sum = 0.f, acc[8] = {};
    auto add = [&](float m, float l, const float (&v)[8]) {
      const float now = fmaxf(top, m);
      const float keep = top == -INFINITY ? 0.f : exp2f(top - now), w = exp2f(m - now);
      top = now;
      sum = sum * keep + w * l;
#pragma unroll
      for (int d = 0; d < 8; ++d) acc[d] = acc[d] * keep + w * v[d];
    };
    for (int i0 = from; i0 < parts; i0 += 4 * stride) {
      float2 ml[4];
      float4 x[4][2];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int i = i0 + k * stride, of = i >> twice;
        ml[k] = make_float2(-INFINITY, 0.f);
        if (i < parts && live) {
          const int slot = part_slot(first + of, of == 0), r = row + (twice & i ? 128 : 0);
          ml[k] = *reinterpret_cast<const float2*>(p.part_ml + ((int64_t)slot * kRows + r) * 2);
          const float4* const src = o + ((int64_t)slot * (D / 4) + 2 * c) * kRows + r;
          x[k][0] = src[0];
          x[k][1] = src[kRows];
        }
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (ml[k].x == -INFINITY && ml[k].y == 0.f) continue;  // no keys: the part has no sums (without a maximum but with a sum: NaN)
        const float v[8] = {x[k][0].x, x[k][0].y, x[k][0].z, x[k][0].w, x[k][1].x, x[k][1].y, x[k][1].z, x[k][1].w};
        add(ml[k].x, ml[k].y, v);
      }
    }
    if (shared) {
      __syncthreads();  // the state of the unit before has been read
      state[warp][8][lane] = top;
      state[warp][9][lane] = sum;
#pragma unroll
      for (int d = 0; d < 8; ++d) state[warp][d][lane] = acc[d];
      __syncthreads();
      if (warp != 0) continue;
      for (int w = 1; w < kWarps; ++w) {
        if (state[w][8][lane] == -INFINITY && state[w][9][lane] == 0.f) continue;
        float v[8];
#pragma unroll
        for (int d = 0; d < 8; ++d) v[d] = state[w][d][lane];
        add(state[w][8][lane], state[w][9][lane], v);
      }
    }
    if (!live) continue;
    const float inv = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
    const int tok = row / p.group, head = item.z * p.group + row - tok * p.group;
    const int64_t t = item.y + tok;
    *reinterpret_cast<uint4*>(p.out + t * p.o_tok + head * p.o_head + 16 * c) =
        make_uint4(pack2<T>(acc[0] * inv, acc[1] * inv), pack2<T>(acc[2] * inv, acc[3] * inv), pack2<T>(acc[4] * inv, acc[5] * inv),
                   pack2<T>(acc[6] * inv, acc[7] * inv));
    if (p.lse && c == 0) p.lse[t * p.lse_tok + head] = sum > 0.f || sum != sum ? (top + log2f(sum)) * 0.693147180559945309f : -INFINITY;
  }
}

// Both kernels' items in one launch: first those of the tile kernel's CTAs, then those of the few-row kernel's.
template <typename T, int D>
__global__ void __launch_bounds__(32 * kWarps, 4) attn_combine_kernel(const __grid_constant__ AttnDev many, const __grid_constant__ AttnDev few,
                                                                   int many_blocks, int few_rows) {
  __shared__ union {
    float part[kWarps][D + 2];
    float state[kWarps][10][32];
  } sh;
  pdl_trigger();
  pdl_wait();
  const int b = blockIdx.x;
  if (b < many_blocks) combine_tiles<T, D>(many, b / (2 * kTileShare), b & 1, (b >> 1) % kTileShare, sh.state);
  else combine_rows<T, D>(few, (b - many_blocks) >> 1, (b - many_blocks) & 1, few_rows, sh.part);
}

template <typename T, int D>
cudaError_t combine(const AttnDev& many, const AttnDev& few, int many_ctas, int few_ctas, int few_rows, cudaStream_t s) {
  const int many_blocks = many_ctas * 2 * kTileShare;
  return launch_ex(attn_combine_kernel<T, D>, dim3(many_blocks + 2 * few_ctas), dim3(32 * kWarps), 0, s, true, dim3(1, 1, 1), many, few,
                   many_blocks, few_rows);
}

}  // namespace

cudaError_t attn_combine_launch(const AttnDev& many, const AttnDev& few, bool f16, int many_ctas, int few_ctas, int few_rows, cudaStream_t s) {
  if (many.c.head_dim == 128)
    return f16 ? combine<__half, 128>(many, few, many_ctas, few_ctas, few_rows, s) : combine<__nv_bfloat16, 128>(many, few, many_ctas, few_ctas, few_rows, s);
  return f16 ? combine<__half, 64>(many, few, many_ctas, few_ctas, few_rows, s) : combine<__nv_bfloat16, 64>(many, few, many_ctas, few_ctas, few_rows, s);
}

}  // namespace llg
