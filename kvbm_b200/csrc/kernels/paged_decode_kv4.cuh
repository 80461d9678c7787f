// Decode attention over the 4-bit paged cache (row format: kv4_format.cuh).
//
//   out[b, h] = sum_t p_t v_t / sum_t p_t,  p_t = 2^(s_t - m),  s_t = qscale q . k_t,  t < seq_lens[b]
//
// in one pass with a running maximum m and sum. The sequence is cut into
// `splits` ranges; a CTA takes one range of one (request, KV head, up to 8 query
// heads), its 4 warps every 4th tile of 32 tokens, and the (m, l, acc) of warps
// and ranges are merged at the end.
//
// What bounds it: at the HBM rate an SM gets the 160 bytes of a (token, KV head)
// of 128 elements every 7 cycles, so about 28 warp instructions are all there is
// for unpacking 256 codes, both products and the softmax. Hence warp-level
// mma.sync with the codes turned into operands in registers, rather than
// tcgen05, whose operands would have to be written back to shared memory first
// (and whose block scales run along the contraction, which for P V is the
// tokens: the wrong way). The arithmetic is arranged so that no element is
// dequantised:
//
// Scores. A nibble c read as an e4m3 byte is c 2^-9, exactly (0..7 are its
// subnormals, 8..15 its first binade). q is split into two e4m3 parts
// q 2^k = hi + lo, which together hold a bf16's 8 bits (exact for elements down
// to 2^-9 of the head's largest; below, off by at most 2^-18 of it). One
// m16n8k32 product covers one group of 32, and its scale and zero are applied to
// the fp32 sums:  q . k = sum_g s_g (c . q_g) + z_g (sum of q_g).
//
// P V. A nibble c or'ed into 0x4300 is the bf16 128 + c. Codes of two tokens are
// paired by one byte permute, the V scale goes into the weight, p' = bf16(p s):
//
//   acc = sum p' (128 + c),  W = sum p' (a product with ones),  Z = sum p (z + 8 s)
//   sum p v = acc - 136 W + Z
//
// so p' only multiplies c - 8, never the offset. Products of 32 tokens are folded
// into fp32 accumulators, since the tensor core's own accumulation truncates.
//
// With up to 4 query heads (PAIR) the 8 columns of a product hold hi and lo of
// 4 heads for the scores, and for P V the p' of 4 heads for two groups: tile
// rows 0-7 are elements of the even group, rows 8-15 of the odd one, half of the
// outputs have no meaning. With 5 to 8 heads hi and lo are two products and a
// tile lies in one group.
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
constexpr int kUnit = 16;  // tokens a stage of the ring holds
constexpr int kTile = 32;  // tokens a warp takes between two updates of its accumulators

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

// ---- instructions ----------------------------------------------------------
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void mma_e4m3(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Transposes the 8x8 matrix of 16-bit elements whose row lane / 4 this lane holds in columns 2 (lane % 4) + {0, 1}.
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ void copy16(uint32_t smem, const void* gmem) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem), "l"(gmem) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
template <int WORDS>
__device__ __forceinline__ void lds(uint32_t (&x)[WORDS], uint32_t addr) {
  if constexpr (WORDS == 1)
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(x[0]) : "r"(addr));
  else if constexpr (WORDS == 2)
    asm volatile("ld.shared.v2.b32 {%0,%1}, [%2];" : "=r"(x[0]), "=r"(x[1]) : "r"(addr));
  else
#pragma unroll
    for (int i = 0; i < WORDS; i += 4)
      asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];"
                   : "=r"(x[i]), "=r"(x[i + 1]), "=r"(x[i + 2]), "=r"(x[i + 3])
                   : "r"(addr + 4 * i));
}
__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
  return lo | (hi << 16);
}
__device__ __forceinline__ float e4m3_part(float x, bool low) {
  __nv_fp8_e4m3 h(x);
  return low ? x - static_cast<float>(h) : x;
}
// Code i of two tokens' packed codes y (one token a half word) as the bf16 pair 128 + c.
__device__ __forceinline__ uint32_t code_pair(uint32_t y, int i) { return ((y >> (4 * i)) & 0x000f000fu) | 0x43004300u; }

template <int HD>
struct Geometry {
  static constexpr int NG = HD / kGroup;
  static constexpr int kRow = row_bytes(HD);
  static constexpr int kChunks = kRow / 16;                  // 16-byte pieces a row; also copies a lane per unit
  static constexpr int kSmemRow = kRow + (HD == 256 ? 16 : 0);  // rows 8 apart in banks of 4 words: no conflicts
  static constexpr int kUnitBytes = 2 * kUnit * kSmemRow;    // K rows, then V rows
  static constexpr int kStages = 4;
  static constexpr int kCtasPerSm = HD == 256 ? 2 : 4;
  static constexpr int kSmem = kAttnWarps * kStages * kUnitBytes;
};

template <int HD, bool PAIR, bool SMALL_PAGE>
__global__ void __launch_bounds__(kAttnWarps * 32, Geometry<HD>::kCtasPerSm)
    kv4_decode_kernel(const __grid_constant__ AttnParams P) {
  using G = Geometry<HD>;
  constexpr int NG = G::NG;
  constexpr int NH = PAIR ? 1 : 2;             // query heads whose scores a lane holds
  constexpr int NW = NG / 2;                   // words of V codes a lane takes from a row
  extern __shared__ __align__(128) uint8_t smem[];
  const int splits = gridDim.x, split = blockIdx.x, b = blockIdx.z;
  const int chunks = (P.group + kHeads - 1) / kHeads;
  const int kvh = blockIdx.y / chunks, h0 = (blockIdx.y - kvh * chunks) * kHeads;
  const int heads = min(kHeads, P.group - h0);
  const int64_t bh0 = static_cast<int64_t>(b) * P.hq + kvh * P.group + h0;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int gid = lane >> 2, tig = lane & 3;

  const int64_t seq = min(static_cast<int64_t>(max(P.seq_lens[b], 0)),
                          static_cast<int64_t>(P.max_blocks) * P.cache.page);
  // ranges of whole rounds of the 4 warps, so that no warp of a long range idles
  constexpr int kRound = kAttnWarps * kTile;
  const int64_t per = ((seq + splits - 1) / splits + kRound - 1) / kRound * kRound;
  const int64_t t_begin = min(seq, split * per);
  const int count = static_cast<int>(min(seq, t_begin + per) - t_begin);  // tokens of this range
  const int tiles = (count + kTile - 1) / kTile;
  const int mine = tiles > warp ? (tiles - warp + kAttnWarps - 1) / kAttnWarps : 0;

  // ---- q as e4m3 operands: column gid is head gid / 2, part gid % 2 (PAIR) or head gid
  uint32_t bq[PAIR ? 1 : 2][NG][2];
  float factor[NH], qsum[NH][NG];
  {
    const int h = PAIR ? gid >> 1 : gid;
    float x[NG][8];
    float top = 0.f;
    bool bad = false;
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      int4 w = make_int4(0, 0, 0, 0);
      if (h < heads)
        w = *reinterpret_cast<const int4*>(P.q + b * P.q_stride + (kvh * P.group + h0 + h) * static_cast<int64_t>(HD) +
                                           g * kGroup + tig * 8);
      const uint32_t ww[4] = {(uint32_t)w.x, (uint32_t)w.y, (uint32_t)w.z, (uint32_t)w.w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        x[g][2 * k] = bf_lo(ww[k]);
        x[g][2 * k + 1] = bf_hi(ww[k]);
        top = fmaxf(top, fmaxf(fabsf(x[g][2 * k]), fabsf(x[g][2 * k + 1])));
        bad |= (ww[k] & 0x7f80u) == 0x7f80u || (ww[k] & 0x7f800000u) == 0x7f800000u;
      }
    }
    int flag = bad;
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      flag |= __shfl_xor_sync(0xffffffffu, flag, o);
    }
    // a power of two that brings the largest element to [128, 256)
    const int e = max(static_cast<int>(__float_as_uint(top) >> 23) - 127, -100);
    const float up = flag ? 0.f : __uint_as_float(static_cast<uint32_t>(127 + 7 - e) << 23);
    const float f = flag ? __uint_as_float(0x7fc00000u) : ldexpf(P.qscale, 9 + e - 7);
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      float s = 0.f;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        x[g][k] = flag ? 0.f : x[g][k] * up;
        s += x[g][k];
      }
      s += __shfl_xor_sync(0xffffffffu, s, 1);
      s += __shfl_xor_sync(0xffffffffu, s, 2);
#pragma unroll
      for (int n = 0; n < NH; ++n)
        qsum[n][g] = 0.001953125f * __shfl_sync(0xffffffffu, s, 8 * tig + 4 * n);  // 2^-9, the codes' unit
#pragma unroll
      for (int part = 0; part < (PAIR ? 1 : 2); ++part) {
        const bool low = PAIR ? (gid & 1) != 0 : part == 1;
#pragma unroll
        for (int odd = 0; odd < 2; ++odd)  // even elements meet the low nibbles, odd ones the high
          bq[part][g][odd] = e4m3x4(e4m3_part(x[g][odd], low), e4m3_part(x[g][2 + odd], low),
                                    e4m3_part(x[g][4 + odd], low), e4m3_part(x[g][6 + odd], low));
      }
    }
#pragma unroll
    for (int n = 0; n < NH; ++n) factor[n] = __shfl_sync(0xffffffffu, f, 8 * tig + 4 * n);
  }

  // ---- the ring: every lane copies kChunks pieces of a unit
  const uint32_t ring = smem_u32(smem) + warp * (G::kStages * G::kUnitBytes);
  int64_t from[G::kChunks];
  uint32_t to[G::kChunks];
#pragma unroll
  for (int i = 0; i < G::kChunks; ++i) {
    const int c = lane + 32 * i, v = c >= kUnit * G::kChunks;
    const int r = c / G::kChunks - (v ? kUnit : 0), piece = c % G::kChunks;
    from[i] = (v ? P.cache.outer_stride : 0) + (SMALL_PAGE ? 0 : r * P.cache.token_stride) + piece * 16;
    to[i] = (v * kUnit + r) * G::kSmemRow + piece * 16;
  }
  const int32_t* table = P.table + b * P.table_stride;
  const uint8_t* base = P.cache.base + static_cast<int64_t>(kvh) * P.cache.head_stride;
  // block ids of the next 32 units, one a lane (-1: no tokens there)
  int32_t ids = -1;
  auto fetch_ids = [&](int tile) {  // for local tiles [tile, tile + 16)
    const int64_t t = static_cast<int64_t>(warp + (tile + (lane >> 1)) * kAttnWarps) * kTile + (lane & 1) * kUnit;
    ids = -1;
    if (t < count) {
      ids = table[P.page_div.div(static_cast<uint32_t>(t_begin + t))];
      if (static_cast<uint32_t>(ids) >= static_cast<uint32_t>(P.cache.num_blocks)) ids = -1;
    }
  };
  // tokens of unit 0 / 1 of the tile in flight that count, a bit each (16 of each)
  uint32_t live_next = 0u;
  auto issue = [&](int tile) {
    uint32_t live = 0u;
    if (tile < mine) {
      if (!SMALL_PAGE && (tile & 15) == 0) fetch_ids(tile);
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int t = (warp + tile * kAttnWarps) * kTile + u * kUnit;
        const uint32_t st = ring + ((2 * tile + u) % G::kStages) * G::kUnitBytes;
        if constexpr (!SMALL_PAGE) {
          const int32_t id = __shfl_sync(0xffffffffu, ids, 2 * (tile & 15) + u);
          if (id >= 0) {
            const uint32_t tok = static_cast<uint32_t>(t_begin + t);
            const uint8_t* src = base + id * P.cache.block_stride +
                                 static_cast<int64_t>(P.page_div.mod(tok, P.page_div.div(tok))) * P.cache.token_stride;
#pragma unroll
            for (int i = 0; i < G::kChunks; ++i) copy16(st + to[i], src + from[i]);
            const int n = min(kUnit, count - t);
            live |= ((1u << n) - 1u) << (16 * u);
          }
        } else {  // pages that a unit does not fit into: every row looks up its own
          const int n = min(kUnit, count - t);
          int32_t id = -1;
          if ((lane & 15) < n) {
            id = table[P.page_div.div(static_cast<uint32_t>(t_begin + t + (lane & 15)))];
            if (static_cast<uint32_t>(id) >= static_cast<uint32_t>(P.cache.num_blocks)) id = -1;
          }
          live |= (__ballot_sync(0xffffffffu, id >= 0) & 0xffffu) << (16 * u);
#pragma unroll
          for (int i = 0; i < G::kChunks; ++i) {
            const int c = lane + 32 * i;
            const int r = (c / G::kChunks) & (kUnit - 1);
            const int32_t row_id = __shfl_sync(0xffffffffu, id, r);
            if (row_id >= 0) {
              const uint32_t tok = static_cast<uint32_t>(t_begin + t + r);
              copy16(st + to[i], base + row_id * P.cache.block_stride +
                                     static_cast<int64_t>(P.page_div.mod(tok, P.page_div.div(tok))) *
                                         P.cache.token_stride +
                                     from[i]);
            }
          }
        }
      }
    }
    copy_commit();
    return live;
  };

  // ---- running state: of query head tig (PAIR) or 2 tig + n
  float m[NH], l[NH], z[NH][NG], w[NH][NG];
  float acc[NG][4][NH];  // element 32 g + 4 gid + i
#pragma unroll
  for (int n = 0; n < NH; ++n) {
    m[n] = -INFINITY;
    l[n] = 0.f;
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      z[n][g] = w[n][g] = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[g][i][n] = 0.f;
    }
  }

  live_next = issue(0);
  for (int tile = 0; tile < mine; ++tile) {
    const uint32_t live = live_next;
    live_next = issue(tile + 1);
    copy_wait<1>();
    __syncwarp();
    const uint32_t st = ring + ((2 * tile) % G::kStages) * G::kUnitBytes;
    const bool whole = live == 0xffffffffu;

    // ---- scores of tokens gid, gid + 8 of both units
    float s[2][2][NH];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const uint32_t k0 = st + u * G::kUnitBytes + gid * G::kSmemRow, k1 = k0 + 8 * G::kSmemRow;
      uint32_t par[2][NG];
      lds(par[0], k0 + HD / 2);
      lds(par[1], k1 + HD / 2);
#pragma unroll
      for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int n = 0; n < NH; ++n) s[u][r][n] = 0.f;
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        uint32_t x0[1], x1[1];
        lds(x0, k0 + g * 16 + tig * 4);
        lds(x1, k1 + g * 16 + tig * 4);
        const uint32_t a[4] = {x0[0] & 0x0f0f0f0fu, x1[0] & 0x0f0f0f0fu, (x0[0] >> 4) & 0x0f0f0f0fu,
                               (x1[0] >> 4) & 0x0f0f0f0fu};
        float c[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int part = 0; part < (PAIR ? 1 : 2); ++part) mma_e4m3(c, a, bq[part][g][0], bq[part][g][1]);
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const float scale = bf_lo(par[r][g]), zero = bf_hi(par[r][g]);
          if constexpr (PAIR) {
            s[u][r][0] = fmaf(scale, c[2 * r] + c[2 * r + 1], fmaf(zero, qsum[0][g], s[u][r][0]));
          } else {
#pragma unroll
            for (int n = 0; n < NH; ++n) s[u][r][n] = fmaf(scale, c[2 * r + n], fmaf(zero, qsum[n][g], s[u][r][n]));
          }
        }
      }
    }
    // ---- softmax
    float alpha[NH];
#pragma unroll
    for (int n = 0; n < NH; ++n) {
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int r = 0; r < 2; ++r) s[u][r][n] *= factor[n];
      if (!whole) {
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int r = 0; r < 2; ++r)
            if (!((live >> (16 * u + 8 * r + gid)) & 1u)) s[u][r][n] = -INFINITY;
      }
      float top = fmaxf(fmaxf(s[0][0][n], s[0][1][n]), fmaxf(s[1][0][n], s[1][1][n]));
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      top = fmaxf(m[n], top);
      const float ref = top == -INFINITY ? 0.f : top;
      alpha[n] = ex2(m[n] - ref);
      m[n] = top;
      l[n] *= alpha[n];
#pragma unroll
      for (int g = 0; g < NG; ++g) z[n][g] *= alpha[n];
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          s[u][r][n] = ex2(s[u][r][n] - ref);
          l[n] += s[u][r][n];
        }
    }
    // ---- weights times V scales, as operands: PAIR columns are (head, group parity)
    constexpr int NB = PAIR ? NG / 2 : NG;
    uint32_t bp[2][NB][2];
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        uint32_t par[NG];
        lds(par, st + u * G::kUnitBytes + (kUnit + gid + 8 * r) * G::kSmemRow + HD / 2);
        if (!whole && !((live >> (16 * u + 8 * r + gid)) & 1u)) {
#pragma unroll
          for (int g = 0; g < NG; ++g) par[g] = 0u;  // what lies behind the last token may be a NaN
        }
        float ps[NG][NH];
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          const float scale = bf_lo(par[g]), mid = fmaf(8.f, scale, bf_hi(par[g]));
#pragma unroll
          for (int n = 0; n < NH; ++n) {
            z[n][g] = fmaf(s[u][r][n], mid, z[n][g]);
            ps[g][n] = s[u][r][n] * scale;
          }
        }
#pragma unroll
        for (int k = 0; k < NB; ++k)
          bp[u][k][r] = transpose8x8(PAIR ? pack2(ps[2 * k][0], ps[2 * k + 1][0]) : pack2(ps[k][0], ps[k][NH - 1]));
      }
    // ---- W = sum p'
#pragma unroll
    for (int k = 0; k < NB; ++k) {
      float c[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int u = 0; u < 2; ++u)
        mma_bf16(c, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u, bp[u][k][0], bp[u][k][1]);
      if constexpr (PAIR) {
        w[0][2 * k] = fmaf(w[0][2 * k], alpha[0], c[0]);
        w[0][2 * k + 1] = fmaf(w[0][2 * k + 1], alpha[0], c[1]);
      } else {
#pragma unroll
        for (int n = 0; n < NH; ++n) w[n][k] = fmaf(w[n][k], alpha[n], c[n]);
      }
    }
    // ---- acc += sum p' (128 + c): this lane's codes of tokens 2 tig, 2 tig + 1 and those 8 further
    uint32_t x[2][4][NW];
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int t = 0; t < 4; ++t)
        lds(x[u][t], st + u * G::kUnitBytes + (kUnit + 2 * tig + (t & 1) + 8 * (t >> 1)) * G::kSmemRow + gid * NW * 4);
#pragma unroll
    for (int k = 0; k < NW; ++k) {  // groups 2 k and 2 k + 1
      uint32_t y[2][2][2];          // [unit][group][tokens 2 tig.. / 8 further]
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          y[u][0][r] = __byte_perm(x[u][2 * r][k], x[u][2 * r + 1][k], 0x5410);
          y[u][1][r] = __byte_perm(x[u][2 * r][k], x[u][2 * r + 1][k], 0x7632);
        }
      if constexpr (PAIR) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float c[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int u = 0; u < 2; ++u)
            mma_bf16(c, code_pair(y[u][0][0], i), code_pair(y[u][1][0], i), code_pair(y[u][0][1], i),
                     code_pair(y[u][1][1], i), bp[u][k][0], bp[u][k][1]);
          acc[2 * k][i][0] = fmaf(acc[2 * k][i][0], alpha[0], c[0]);
          acc[2 * k + 1][i][0] = fmaf(acc[2 * k + 1][i][0], alpha[0], c[3]);
        }
      } else {
#pragma unroll
        for (int p = 0; p < 2; ++p)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const int g = 2 * k + p;
            float c[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int u = 0; u < 2; ++u)
              mma_bf16(c, code_pair(y[u][p][0], 2 * j), code_pair(y[u][p][0], 2 * j + 1),
                       code_pair(y[u][p][1], 2 * j), code_pair(y[u][p][1], 2 * j + 1), bp[u][g][0], bp[u][g][1]);
#pragma unroll
            for (int n = 0; n < NH; ++n) {
              acc[g][2 * j][n] = fmaf(acc[g][2 * j][n], alpha[n], c[n]);
              acc[g][2 * j + 1][n] = fmaf(acc[g][2 * j + 1][n], alpha[n], c[2 + n]);
            }
          }
      }
    }
    __syncwarp();
  }
  copy_wait<0>();

  // ---- sums over the lanes that share a head, then the 4 warps
#pragma unroll
  for (int n = 0; n < NH; ++n)
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) {
      l[n] += __shfl_xor_sync(0xffffffffu, l[n], o);
#pragma unroll
      for (int g = 0; g < NG; ++g) z[n][g] += __shfl_xor_sync(0xffffffffu, z[n][g], o);
    }
  __shared__ float red_m[kAttnWarps][kHeads], red_l[kAttnWarps][kHeads];
  float* red = reinterpret_cast<float*>(smem);  // [warps][heads][HD], in the ring's place
  __syncthreads();
#pragma unroll
  for (int n = 0; n < NH; ++n) {
    const int h = NH * tig + n;
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      const float off = fmaf(-136.f, w[n][g], z[n][g]);
      *reinterpret_cast<float4*>(red + (warp * kHeads + h) * HD + g * kGroup + gid * 4) =
          make_float4(acc[g][0][n] + off, acc[g][1][n] + off, acc[g][2][n] + off, acc[g][3][n] + off);
    }
    if (gid == 0) {
      red_m[warp][h] = m[n];
      red_l[warp][h] = l[n];
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < heads * HD; i += kAttnWarps * 32) {
    const int h = i / HD, d = i - h * HD;
    float M = -INFINITY, L = 0.f, A = 0.f;
#pragma unroll
    for (int k = 0; k < kAttnWarps; ++k) M = fmaxf(M, red_m[k][h]);
#pragma unroll
    for (int k = 0; k < kAttnWarps; ++k) {
      if (red_l[k][h] == 0.f) continue;
      const float f = exp2f(red_m[k][h] - M);
      L += f * red_l[k][h];
      A += f * red[(k * kHeads + h) * HD + d];
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

template <int HD, bool PAIR, bool SMALL_PAGE>
cudaError_t launch_decode_kernel(const AttnParams& P, dim3 grid, cudaStream_t stream) {
  auto kernel = kv4_decode_kernel<HD, PAIR, SMALL_PAGE>;
  constexpr int kSmem = Geometry<HD>::kSmem > kAttnWarps * kHeads * HD * 4 ? Geometry<HD>::kSmem
                                                                          : kAttnWarps * kHeads * HD * 4;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
  if (e != cudaSuccess) return e;
  kernel<<<grid, kAttnWarps * 32, kSmem, stream>>>(P);
  return cudaGetLastError();
}

template <int HD>
cudaError_t launch_decode_hd(const AttnParams& P, int batch, int splits, cudaStream_t stream) {
  const int chunks = (P.group + kHeads - 1) / kHeads;
  const int64_t y = static_cast<int64_t>(P.cache.heads) * chunks;
  if (y > 65535) return cudaErrorInvalidValue;
  const dim3 grid(splits, static_cast<unsigned>(y), batch);
  const bool small = P.cache.page % kUnit != 0;
  cudaError_t e;
  if (P.group <= 4)
    e = small ? launch_decode_kernel<HD, true, true>(P, grid, stream)
              : launch_decode_kernel<HD, true, false>(P, grid, stream);
  else
    e = small ? launch_decode_kernel<HD, false, true>(P, grid, stream)
              : launch_decode_kernel<HD, false, false>(P, grid, stream);
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
