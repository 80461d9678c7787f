// Decode attention over the 4-bit paged cache (row format: kv4_format.cuh).
//
//   out[b, h] = sum_t p_t v_t / sum_t p_t,  p_t = 2^(qscale q . k_t - m),  t < seq_lens[b]
//
// in one pass with a running maximum m and sum. The sequence is cut into
// `splits` ranges of pages; each CTA takes one range of one (request, KV head,
// up to 8 query heads) and the ranges' (m, l, acc) are merged at the end.
#pragma once

#include "common.cuh"
#include "kv4_format.cuh"

namespace kvbm {
namespace kv4 {

struct AttnParams {
  Cache cache;
  const __nv_bfloat16* q;
  int64_t q_stride;
  const int32_t* table;
  int64_t table_stride;
  int max_blocks;
  const int32_t* seq_lens;
  int hq, group;
  float qscale;
  float* part_acc;
  float* part_ml;
  unsigned int* counters;
  __nv_bfloat16* out;
  FastDiv page_div;
};

constexpr int kHeads = 8;  // query heads a CTA takes at most
constexpr int kAttnWarps = 4;

// Merges the splits of one query head's row: thread d of HD.
template <int HD>
__device__ __forceinline__ void merge_row(const AttnParams& P, int64_t bh, int splits, int d) {
  float M = -INFINITY;
  for (int s = 0; s < splits; ++s) M = fmaxf(M, __ldcg(&P.part_ml[(bh * splits + s) * 2]));
  float l = 0.f, a = 0.f;
  for (int s = 0; s < splits; ++s) {
    const float ls = __ldcg(&P.part_ml[(bh * splits + s) * 2 + 1]);
    if (ls == 0.f) continue;  // no tokens (a NaN goes on)
    const float f = exp2f(__ldcg(&P.part_ml[(bh * splits + s) * 2]) - M);
    l += f * ls;
    a += f * __ldcg(&P.part_acc[(bh * splits + s) * HD + d]);
  }
  P.out[bh * HD + d] = __float2bfloat16(l == 0.f ? 0.f : a / l);
}

template <int HD>
__global__ void __launch_bounds__(HD) kv4_merge_kernel(const __grid_constant__ AttnParams P, int splits) {
  merge_row<HD>(P, blockIdx.x, splits, threadIdx.x);
}

// A warp takes every 4th token of the range; lane l holds elements [l E, l E + E).
template <int HD>
__global__ void __launch_bounds__(kAttnWarps * 32) kv4_decode_kernel(const __grid_constant__ AttnParams P) {
  constexpr int E = HD / 32, NG = HD / kGroup;
  const int splits = gridDim.x, split = blockIdx.x, b = blockIdx.z;
  const int chunks = (P.group + kHeads - 1) / kHeads;
  const int kvh = blockIdx.y / chunks, h0 = (blockIdx.y - kvh * chunks) * kHeads;
  const int heads = min(kHeads, P.group - h0);
  const int64_t bh0 = static_cast<int64_t>(b) * P.hq + kvh * P.group + h0;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  __shared__ float red[kAttnWarps][kHeads][HD + 2];

  float q[kHeads][E], acc[kHeads][E], m[kHeads], l[kHeads];
#pragma unroll
  for (int h = 0; h < kHeads; ++h) {
    m[h] = -INFINITY;
    l[h] = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      acc[h][e] = 0.f;
      q[h][e] = h < heads ? __bfloat162float(P.q[b * P.q_stride + (kvh * P.group + h0 + h) * static_cast<int64_t>(HD) +
                                                 lane * E + e]) * P.qscale
                          : 0.f;
    }
  }
  const int64_t seq = min(static_cast<int64_t>(max(P.seq_lens[b], 0)),
                          static_cast<int64_t>(P.max_blocks) * P.cache.page);
  const int64_t per = ((seq + P.cache.page - 1) / P.cache.page + splits - 1) / splits * P.cache.page;
  const int64_t t1 = min(seq, (split + 1) * per);
  for (int64_t t = split * per + warp; t < t1; t += kAttnWarps) {
    const uint32_t col = P.page_div.div(static_cast<uint32_t>(t));
    const int32_t blk = P.table[b * P.table_stride + col];
    if (blk < 0 || blk >= P.cache.num_blocks) continue;  // a page that is not there holds no tokens
    const uint8_t* k = P.cache.base + blk * P.cache.block_stride +
                       static_cast<int64_t>(P.page_div.mod(static_cast<uint32_t>(t), col)) * P.cache.token_stride +
                       static_cast<int64_t>(kvh) * P.cache.head_stride;
    const uint8_t* v = k + P.cache.outer_stride;
    float kd[E], vd[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int d = lane * E + e, g = d / kGroup, n = 4 * (NG * (d % kGroup / 4) + g) + d % 4;
      const uint32_t ks = reinterpret_cast<const uint32_t*>(k + HD / 2)[g];
      const uint32_t vs = reinterpret_cast<const uint32_t*>(v + HD / 2)[g];
      kd[e] = fmaf(static_cast<float>((k[d / 2] >> (4 * (d & 1))) & 15), bf_lo(ks), bf_hi(ks));
      vd[e] = fmaf(static_cast<float>((v[n / 2] >> (4 * (n & 1))) & 15), bf_lo(vs), bf_hi(vs));
    }
#pragma unroll
    for (int h = 0; h < kHeads; ++h) {
      if (h >= heads) break;
      float s = 0.f;
#pragma unroll
      for (int e = 0; e < E; ++e) s = fmaf(q[h][e], kd[e], s);
      s = warp_sum(s);
      const float m_new = fmaxf(m[h], s);
      const float alpha = m[h] == -INFINITY ? 0.f : exp2f(m[h] - m_new);
      const float p = exp2f(s - m_new);
      m[h] = m_new;
      l[h] = l[h] * alpha + p;
#pragma unroll
      for (int e = 0; e < E; ++e) acc[h][e] = acc[h][e] * alpha + p * vd[e];
    }
  }
#pragma unroll
  for (int h = 0; h < kHeads; ++h) {
#pragma unroll
    for (int e = 0; e < E; ++e) red[warp][h][lane * E + e] = acc[h][e];
    if (lane == 0) {
      red[warp][h][HD] = m[h];
      red[warp][h][HD + 1] = l[h];
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < heads * HD; i += kAttnWarps * 32) {
    const int h = i / HD, d = i - h * HD;
    float M = -INFINITY, L = 0.f, A = 0.f;
#pragma unroll
    for (int w = 0; w < kAttnWarps; ++w) M = fmaxf(M, red[w][h][HD]);
#pragma unroll
    for (int w = 0; w < kAttnWarps; ++w) {
      if (red[w][h][HD + 1] == 0.f) continue;
      const float f = exp2f(red[w][h][HD] - M);
      L += f * red[w][h][HD + 1];
      A += f * red[w][h][d];
    }
    if (splits == 1) {
      P.out[(bh0 + h) * HD + d] = __float2bfloat16(L == 0.f ? 0.f : A / L);
    } else {
      const int64_t row = (bh0 + h) * splits + split;
      P.part_acc[row * HD + d] = A;
      if (d == 0) {
        P.part_ml[row * 2] = M;
        P.part_ml[row * 2 + 1] = L;
      }
    }
  }
  if (splits == 1 || P.counters == nullptr) return;
  __shared__ unsigned int ticket;
  __threadfence();
  __syncthreads();
  unsigned int* counter = &P.counters[static_cast<int64_t>(b) * gridDim.y + blockIdx.y];
  if (threadIdx.x == 0) ticket = atomicAdd(counter, 1u);
  __syncthreads();
  if (ticket != static_cast<unsigned int>(splits - 1)) return;
  __threadfence();
  for (int i = threadIdx.x; i < heads * HD; i += kAttnWarps * 32) merge_row<HD>(P, bh0 + i / HD, splits, i % HD);
  if (threadIdx.x == 0) *counter = 0u;
}

template <int HD>
cudaError_t launch_decode_hd(const AttnParams& P, int batch, int splits, cudaStream_t stream) {
  const int chunks = (P.group + kHeads - 1) / kHeads;
  const int64_t y = static_cast<int64_t>(P.cache.heads) * chunks;
  if (y > 65535) return cudaErrorInvalidValue;
  kv4_decode_kernel<HD><<<dim3(splits, static_cast<unsigned>(y), batch), kAttnWarps * 32, 0, stream>>>(P);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess || splits == 1 || P.counters != nullptr) return e;
  kv4_merge_kernel<HD><<<static_cast<unsigned>(batch) * P.hq, HD, 0, stream>>>(P, splits);
  return cudaGetLastError();
}

inline cudaError_t launch_decode(const AttnParams& P, int batch, int hd, int splits, cudaStream_t stream) {
  switch (hd) {
    case 64: return launch_decode_hd<64>(P, batch, splits, stream);
    case 128: return launch_decode_hd<128>(P, batch, splits, stream);
    case 256: return launch_decode_hd<256>(P, batch, splits, stream);
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace kv4
}  // namespace kvbm
