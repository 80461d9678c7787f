// Decode attention over the 4-bit paged cache (row format: kv4_format.cuh).
//
//   out[b, h] = sum_t p_t v_t / sum_t p_t,  p_t = 2^(s_t - m),  s_t = qscale q . k_t,  t < seq_lens[b]
//
// in one pass with a running maximum m and sum.
//
// What bounds it: at the HBM rate an SM gets the 160 bytes of a (token, KV head)
// of 128 elements every 7 cycles, in which it issues 28 warp instructions, 14 of
// them on the integer pipe. That is all there is for unpacking 256 codes, both
// products and the softmax. Hence warp-level mma.sync with the codes turned into
// operands in registers, rather than tcgen05, whose operands would have to be
// written back to shared memory first (and whose block scales run along the
// contraction, which for P V is the tokens: the wrong way). No element is
// dequantised:
//
// A nibble masked in place is a subnormal fp16: c 2^-24 in bits 0-3, c 2^-20 in
// bits 4-7, both exact, and so is a whole byte, (c0 + 16 c1) 2^-24. A word of 8
// codes becomes 4 operand registers, c0 and c0 + 16 c1 of its even and of its odd
// bytes, with three ands and one byte permute; what multiplies or follows them
// takes the two apart: a c0 + b c1 = (a - b / 16) c0 + (b / 16) (c0 + 16 c1).
//
// Scores. q 2^k is put in fp16, k bringing the head's largest element to 2^13.
// (a - b / 16) of two q needs more bits than fp16 has: with up to 4 query heads on
// a KV head (PAIR) it goes in two parts, in two of the 8 columns of a product, and
// 2^-22 of it is lost at most; with 5 to 8 there are no columns to spare, and c1 is
// taken alone at one shift more a word. Each group of 32 is two m16n8k16 products,
// whose fp32 sums take the group's scale; the zeros' part, sum over g of z_g (sum
// of q_g), is one bf16 product more with the sums of q in three bf16 parts.
//
// P V. Codes of two tokens are paired by one byte permute. The V scale goes into
// the weight: p' = fp16(p s f), f a power of two. When sums of p' come out infinite,
// as they do in a first tile, f is set so that the largest p s lies at [2^10, 2^11)
// (2^9 with the most operands), and the sums of products go along. Then
// sum p v = sum p' c / f + sum p z.
// p' is off by up to 2^-11 of itself, or by 2^-25 / f. So the largest weight that a
// query head has given a group of V has to lie at 2 or more, where the latter is
// 2^-26 of it: a tile in which the head's maximum m rises, or in which f falls, has
// to bring each group such a weight. Where one does not (V whose scales differ by a
// factor of 2^9 or so), share_in_fp32 does the warp's tiles of this request again,
// element by element. (A factor for each head and group took 4 to 22 % more time in
// registers or in shared memory, with all tiles.) 11 bits are enough for the others:
// a second fp16 part would double the products with 5 to 8 heads, and an average of
// weights so rounded is nearer than the bf16 of the result.
// The same goes for scores above 2^12: p comes from one multiply-add with the rounded
// m, which is off by 2^-24 of it, and s from sums that are off by about as much.
// Products of 32 tokens are folded into fp32 accumulators, since the tensor
// core's own accumulation truncates.
//
// In PAIR the 8 columns of a P V product hold p' of 4 heads for two groups: tile rows 0-7 are elements of the even
// group, rows 8-15 of the odd one, half of the outputs have no meaning. With 5
// to 8 heads a column is a head and a tile lies in one group.
//
// Work. A warp takes one (KV head, up to 8 query heads) and tiles of 32 tokens;
// the warps of a CTA take different KV heads of the same tokens (with fewer than
// 8, several streams of tokens), so that what lies together in a token-first pool
// is read together. All requests' tiles are laid end to end and cut into equal
// ranges, one for each CTA the GPU holds at a time, so ragged batches and odd
// numbers of heads cost no idle SMs; a cut that falls into a short request moves
// to its end. A CTA meets at most two requests that are not its own alone; their
// partial results (m, l, acc) are merged by a second kernel, whose launch overlaps
// the first's end and is left out where the table holds short requests only.
//
// Copies. Each warp has its own ring of two tiles. A unit of 16 tokens, K and V
// rows of one KV head, is one TMA box of the five-dimensional pool, issued by the
// lane that looked the unit's page up (32 units at a time); where a page is not a
// multiple of 16 tokens, rows are copied one by one with cp.async. What limits the
// copies is the number of contiguous runs, of 80 bytes with 128 elements a head:
// in a head-first pool the 16 rows are one run, and in a token-first one two warps
// share the rows of two neighbouring heads (SHARED), one of them issuing, with a
// barrier of the two where a tile's stage is given back.
//
// Measured, pages of 16 tokens, heads of 128, 32 on 8 KV heads: 32 requests of
// 8,448 tokens 65.6 us = 5.3 TB/s, one of 131,072 38.0 us = 4.4 TB/s, one of 300
// 7.9 us; each further byte costs what it costs in a copy (1.03 of it token-first,
// 1.02 head-first), the rest is the start, the last round and the merge, about 11
// us. Heads of 64, 28 on 4: 61 requests of up to 9,000 tokens 33.9 us = 3.1 TB/s,
// where 520 instructions a tile are the bound (1.3 of a copy a further byte, as at
// 128 with 5 to 8 heads on one). Pages that are not a multiple of 16 tokens, whose
// rows are copied one by one, cost 1.6 to 1.8.
#pragma once

#include "common.cuh"
#include "kv4_format.cuh"

#include <cuda.h>
#include <cudaTypedefs.h>

#include <algorithm>

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
  int batch, hq, group, chunks;  // chunks: groups of up to 8 query heads on a KV head
  int y_total, y_cta, streams;   // (KV head, chunk) pairs: in all, a CTA; streams of tokens a CTA
  float qscale;
  float* part_acc;  // [cta][2][hq][HD]
  float* part_ml;   // [cta][2][hq][2]
  int2* parts;      // [batch], null if no request can be cut: a request's first slot of partial results (2 cta, + 1: not its CTA's first), and how many
  __nv_bfloat16* out;
  int* status;       // where a launch that gives a copy up says so
  uint64_t wait_ns;  // after which a warp gives a copy up; 0: at once
  bool flat;  // a head's rows in a page are contiguous: the copies take them as one
};

// A kernel launched by launch_overlapped reads and writes nothing before wait_before, the end of the kernel before;
// release_next lets the next one be put in place.
__device__ __forceinline__ void wait_before() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void release_next() { asm volatile("griddepcontrol.launch_dependents;"); }

constexpr int kHeads = 8;       // query heads a warp takes at most
constexpr int kMaxWarps = 8;
enum Copies { kRows, kTma, kTmaShared };
constexpr int kUnit = 16;       // tokens a stage of the ring holds
constexpr int kTile = 32;       // tokens a warp takes between two updates of its accumulators
constexpr int kMinRounds = 2;   // a CTA takes at least so many tiles a warp: below, merging costs more than it saves
constexpr int kWhole = 6;       // requests of up to so many rounds (kStart among them) are not cut
constexpr float kLargeScore = 4096.f;  // of log2 of p: above, fp32 products of scores are not near enough
constexpr uint64_t kWaitNs = 1000000000ull;  // limit of a wait for a copy

// ---- instructions ----------------------------------------------------------
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// d = a b + c; the first product of a chain takes zeros for c, which costs no registers.
#define KVBM_KV4_MMA(NAME, TYPE)                                                                                     \
  __device__ __forceinline__ void NAME(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,            \
                                       uint32_t b0, uint32_t b1, float c0, float c1, float c2, float c3) {           \
    asm("mma.sync.aligned.m16n8k16.row.col.f32." TYPE "." TYPE                                                       \
        ".f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"                                             \
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])                                                             \
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));                 \
  }
KVBM_KV4_MMA(mma_f16, "f16")
KVBM_KV4_MMA(mma_bf16, "bf16")
#undef KVBM_KV4_MMA
// Transposes the 8x8 matrix of 16-bit elements whose row lane / 4 this lane holds in columns 2 (lane % 4) + {0, 1}.
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
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
// K and V rows of `kUnit` tokens of one KV head: coordinates (byte / 8, head, token in the page, K / V, block).
__device__ __forceinline__ void copy_unit(uint32_t smem, const CUtensorMap* map, int word, int head, int token, int block,
                                          uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, %6}], "
      "[%7];" ::"r"(smem),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(word), "r"(head), "r"(token), "r"(0), "r"(block), "r"(smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ uint32_t half2(float lo, float hi) {
  __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}
// A word's nibbles i and i + 4 as fp16 pairs in units of 2^-24: i even c_i; i odd c_{i-1} + 16 c_i.
__device__ __forceinline__ void code_pairs(uint32_t (&a)[4], uint32_t x) {
  a[1] = x & 0x00ff00ffu;
  a[0] = x & 0x000f000fu;
  a[3] = __byte_perm(x, 0, 0x4341);
  a[2] = a[3] & 0x000f000fu;
}
// The same with i odd 16 c_i alone.
__device__ __forceinline__ void code_pairs_alone(uint32_t (&a)[4], uint32_t x) {
  a[0] = x & 0x000f000fu;
  a[1] = x & 0x00f000f0u;
  x >>= 8;
  a[2] = x & 0x000f000fu;
  a[3] = x & 0x00f000f0u;
}
__device__ __forceinline__ uint32_t add_half2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("add.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
__device__ __forceinline__ float pow2(int e) { return __uint_as_float(static_cast<uint32_t>(127 + e) << 23); }
__device__ __forceinline__ int exponent(float x) { return static_cast<int>((__float_as_uint(x) >> 23) & 255u) - 127; }

// The same value, for a branch that is seldom taken: what is computed from it there is not moved in front of the branch.
__device__ __forceinline__ uint32_t seldom(uint32_t x) {
  asm volatile("" : "+r"(x));
  return x;
}

__device__ __forceinline__ int tokens_of(const AttnParams& P, int b) {
  return static_cast<int>(min(static_cast<int64_t>(max(P.seq_lens[b], 0)),
                              min(static_cast<int64_t>(P.max_blocks) * P.cache.page, static_cast<int64_t>(0x7ffff000))));
}
// Rounds of streams x 32 tokens that a request counts for: its own, and kStart in front of them in which nothing
// is done, for what it costs a CTA to begin a request.
constexpr int kStart = 2;
__device__ __forceinline__ int rounds_of(int tokens, int streams) {
  return kStart + (tokens + kTile * streams - 1) / (kTile * streams);
}
// Merges the partial results of each request that several CTAs worked on. Part i of a request that begins in
// CTA c lies in CTA c + i, in the slot of that CTA's first request (0), or of a later one (1: only its last can go
// on). A warp reads 32 parts' (m, l), a lane each, together with 64 / E parts' acc, of which lane l has elements
// l E .. (E = HD / 32): the bound is the latency of that one round of loads. A CTA takes 8 query heads of a request,
// a warp each, or (many parts, or heads too few to fill the GPU) one at a time, its warps sharing the parts.
constexpr int kMergeWarps = 8;
template <int HD>
__device__ __forceinline__ void merge_parts(const AttnParams& P, int64_t row0, int64_t slot0, int begin, int end,
                                            float& m, float& l, float (&acc)[HD / 32]) {
  constexpr int E = HD / 32, V = E < 4 ? E : 4, kFly = 64 / E;
  const int lane = threadIdx.x & 31;
  auto row = [&](int i) { return row0 + static_cast<int64_t>(i) * 2 * P.hq + (i == 0 ? slot0 : 0); };
  float x[kFly][E];
  auto load = [&](int i0, int n) {
#pragma unroll
    for (int k = 0; k < kFly; ++k) {
      if (k >= n) break;
      const float* src = P.part_acc + row(i0 + k) * HD + lane * E;
#pragma unroll
      for (int e = 0; e < E; e += V) {
        if constexpr (V == 2)
          *reinterpret_cast<float2*>(&x[k][e]) = __ldcg(reinterpret_cast<const float2*>(src + e));
        else
          *reinterpret_cast<float4*>(&x[k][e]) = __ldcg(reinterpret_cast<const float4*>(src + e));
      }
    }
  };
  m = -INFINITY;
  l = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) acc[e] = 0.f;
  for (int i0 = begin; i0 < end; i0 += 32) {
    const int here = min(32, end - i0);
    float2 ml = make_float2(-INFINITY, 0.f);
    if (lane < here) ml = __ldcg(reinterpret_cast<const float2*>(P.part_ml) + row(i0 + lane));
    load(i0, here);
    const float top = fmaxf(m, warp_max(ml.x));
    const float down = l == 0.f ? 0.f : exp2f(m - top);
    const float f = ml.y == 0.f ? 0.f : exp2f(ml.x - top);  // no tokens: nothing (a NaN goes on)
    l = fmaf(l, down, warp_sum(f * ml.y));
    m = top;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] *= down;
    for (int j = 0; j < here; j += kFly) {
      if (j > 0) load(i0 + j, here - j);
#pragma unroll
      for (int k = 0; k < kFly; ++k) {
        if (j + k >= here) break;
        const float fk = __shfl_sync(0xffffffffu, f, j + k);
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] = fmaf(fk, x[k][e], acc[e]);
      }
    }
  }
}

template <int HD>
__global__ void __launch_bounds__(kMergeWarps * 32) kv4_merge_kernel(const __grid_constant__ AttnParams P,
                                                                     int heads_cta) {
  constexpr int E = HD / 32;
  __shared__ float red[kMergeWarps][HD + 2];
  const int b = blockIdx.y, h_begin = blockIdx.x * heads_cta, h_end = min(P.hq, h_begin + heads_cta);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  release_next();
  wait_before();
  const int2 parts = __ldcg(&P.parts[b]);
  const int n = parts.y;
  if (n == 1) return;  // written by its one CTA
  const int64_t row0 = static_cast<int64_t>(parts.x & ~1) * P.hq, slot0 = (parts.x & 1) * P.hq;
  const bool apart = heads_cta > 1 && n <= 64;
  const int each = apart ? n : (n + kMergeWarps - 1) / kMergeWarps;
  const int begin = apart ? 0 : warp * each, end = min(n, begin + each);
  for (int h = h_begin + (apart ? warp : 0); h < h_end; h += apart ? kMergeWarps : 1) {
    float m, l, acc[E];
    merge_parts<HD>(P, row0 + h, slot0, begin, end, m, l, acc);
    if (!apart) {
      __syncthreads();
#pragma unroll
      for (int e = 0; e < E; ++e) red[warp][lane * E + e] = acc[e];
      if (lane == 0) {
        red[warp][HD] = m;
        red[warp][HD + 1] = l;
      }
      __syncthreads();
      if (warp != 0) continue;
      m = -INFINITY;
#pragma unroll
      for (int w = 0; w < kMergeWarps; ++w) m = fmaxf(m, red[w][HD]);
      l = 0.f;
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] = 0.f;
#pragma unroll
      for (int w = 0; w < kMergeWarps; ++w) {
        const float lw = red[w][HD + 1];
        const float f = lw == 0.f ? 0.f : exp2f(red[w][HD] - m);
        l = fmaf(f, lw, l);
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] = fmaf(f, red[w][lane * E + e], acc[e]);
      }
    }
    const float r = l == 0.f ? 0.f : 1.f / l;
    uint32_t* dst = reinterpret_cast<uint32_t*>(P.out + (static_cast<int64_t>(b) * P.hq + h) * HD + lane * E);
#pragma unroll
    for (int e = 0; e < E; e += 2) dst[e / 2] = pack2(acc[e] * r, acc[e + 1] * r);
  }
}

template <int HD>
struct Geometry {
  static constexpr int NG = HD / kGroup;
  static constexpr int kRow = row_bytes(HD);
  static constexpr int kChunks = kRow / 16;        // 16-byte pieces a row; also copies a lane for a unit
  static constexpr int kCtasPerSm = HD == 256 ? 1 : 2;  // of 8 warps
  static constexpr int kRingBytes = 4 * 2 * kUnit * kRow;  // a warp: two tiles of two units, K and V
};

// The K row (the V row is outer_stride behind it) of token t of a request, or null for a page outside the pool.
__device__ __forceinline__ const uint8_t* row_of(const AttnParams& P, const int32_t* table, int t, int kvh) {
  const uint32_t col = P.cache.page_div.div(static_cast<uint32_t>(t));
  const int32_t id = table[col];
  if (static_cast<uint32_t>(id) >= static_cast<uint32_t>(P.cache.num_blocks)) return nullptr;
  return P.cache.base + id * P.cache.block_stride +
         P.cache.page_div.mod(static_cast<uint32_t>(t), col) * P.cache.token_stride + kvh * P.cache.head_stride;
}
// Whether one of the groups (a bit each) has elements that differ in one of a warp's tokens: groups of equal elements, as
// in padding, take no weights (with one such group in four 105 us in place of 75).
template <int HD>
__device__ __forceinline__ bool any_scale(const AttnParams& P, int b, int kvh, int seq, int t_begin, int tiles,
                                          int round_tokens, uint32_t groups) {
  constexpr int NG = HD / kGroup;
  const int32_t* table = P.table + b * P.table_stride;
  bool found = false;
  for (int tile = 0; tile < tiles; ++tile) {
    const int t = t_begin + tile * round_tokens + static_cast<int>(threadIdx.x & 31);
    const uint8_t* k = t < seq ? row_of(P, table, t, kvh) : nullptr;
    if (k == nullptr) continue;
    for (int g = 0; g < NG; ++g) {
      if ((groups >> g) & 1u)
        found |= (*reinterpret_cast<const uint32_t*>(k + P.cache.outer_stride + HD / 2 + 4 * g) & 0xffffu) != 0u;
    }
  }
  return __any_sync(0xffffffffu, found);
}
// A warp's tiles of a request once more, from the pool and in fp32 alone: a token at a time, each element taken apart.
// Lane (gid, tig) has elements 32 g + 4 gid + i of query heads NH tig + n, as in the loop that it replaces (32
// requests of 8,448 tokens, all of them again: 1.0 ms in place of 0.07. With the next token's rows under way it took
// 0.8, and the registers for that 2 to 8 % of the other's time).
template <int HD, int NH>
__device__ __forceinline__ void share_in_fp32(const AttnParams& P, int b, int kvh, int head0, int heads, int seq,
                                              int t_begin, int tiles, int round_tokens, float (&m)[NH], float (&l)[NH],
                                              float (&acc)[HD / kGroup][4][NH]) {
  constexpr int NG = HD / kGroup;
  const int lane = threadIdx.x & 31, gid = lane >> 2, tig = lane & 3;
  float q[NH][NG][4];
#pragma unroll
  for (int n = 0; n < NH; ++n) {
    m[n] = -INFINITY;
    l[n] = 0.f;
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      uint2 w = make_uint2(0u, 0u);
      if (NH * tig + n < heads)
        w = *reinterpret_cast<const uint2*>(P.q + b * P.q_stride + (head0 + NH * tig + n) * static_cast<int64_t>(HD) +
                                            g * kGroup + gid * 4);
      q[n][g][0] = bf_lo(w.x), q[n][g][1] = bf_hi(w.x), q[n][g][2] = bf_lo(w.y), q[n][g][3] = bf_hi(w.y);
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[g][i][n] = 0.f;
    }
  }
  const int32_t* table = P.table + b * P.table_stride;
  for (int tile = 0; tile < tiles; ++tile) {
    const int t0 = t_begin + tile * round_tokens;
    for (int t = t0; t < min(seq, t0 + kTile); ++t) {
      const uint8_t* k = row_of(P, table, t, kvh);
      if (k == nullptr) continue;
      const uint8_t* v = k + P.cache.outer_stride;
      float score[NH], x[NG][4];
#pragma unroll
      for (int n = 0; n < NH; ++n) score[n] = 0.f;
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        const uint32_t kc = *reinterpret_cast<const uint16_t*>(k + 16 * g + 2 * gid);
        const uint32_t kp = *reinterpret_cast<const uint32_t*>(k + HD / 2 + 4 * g);
        const uint32_t vc = *reinterpret_cast<const uint16_t*>(v + 2 * (NG * gid + g));
        const uint32_t vp = *reinterpret_cast<const uint32_t*>(v + HD / 2 + 4 * g);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float y = fmaf(static_cast<float>((kc >> (4 * i)) & 15u), bf_lo(kp), bf_hi(kp));
          x[g][i] = fmaf(static_cast<float>((vc >> (4 * i)) & 15u), bf_lo(vp), bf_hi(vp));
#pragma unroll
          for (int n = 0; n < NH; ++n) score[n] = fmaf(q[n][g][i], y, score[n]);
        }
      }
#pragma unroll
      for (int n = 0; n < NH; ++n) {
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) score[n] += __shfl_xor_sync(0xffffffffu, score[n], o);
        score[n] *= P.qscale;
        const float top = fmaxf(m[n], score[n]), ref = top == -INFINITY ? 0.f : top;
        const float down = exp2f(m[n] - ref), p = exp2f(score[n] - ref);
        m[n] = top;
        l[n] = fmaf(l[n], down, p);
#pragma unroll
        for (int g = 0; g < NG; ++g)
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[g][i][n] = fmaf(p, x[g][i], acc[g][i][n] * down);
      }
    }
  }
}

template <int HD, bool PAIR, Copies COPIES>
__global__ void __launch_bounds__(kMaxWarps * 32, Geometry<HD>::kCtasPerSm)
    kv4_decode_kernel(const __grid_constant__ AttnParams P, const __grid_constant__ CUtensorMap map) {
  using G = Geometry<HD>;
  constexpr bool TMA = COPIES != kRows, SHARED = COPIES == kTmaShared;
  constexpr int kStride = SHARED ? 2 * G::kRow : G::kRow;  // between rows in shared memory
  constexpr int kStage = 2 * kUnit * kStride;              // a unit's K rows, then its V rows
  constexpr int NG = G::NG;
  constexpr int NH = PAIR ? 1 : 2;       // query heads whose scores a lane holds
  constexpr int NW = NG / 2;             // words of V codes a lane takes from a row
  constexpr int NZ = (NG + 3) / 4;       // products for the zeros of K
  constexpr int NB = PAIR ? NG / 2 : NG; // operands of weights a unit
  constexpr int kBest = NB < 8 ? 10 : 9; // exponent of a tile's largest weight when f is set: 4 NB such add up to less than 2^16
  extern __shared__ __align__(128) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int gid = lane >> 2, tig = lane & 3;
  release_next();  // the merge
  __shared__ uint64_t full[kMaxWarps][2];  // a warp's two tiles
  if constexpr (TMA) {
    if (lane < 2) mbar_init(&full[warp][lane], 2);  // the two lanes that issue its units
    fence_mbar_init();
    if (threadIdx.x == 0) asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&map)) : "memory");
  }

  // What is above overlaps the end of the kernel before; nothing that it may have written is read above.
  wait_before();
  // ---- this CTA's range of rounds, and the request it begins in
  __shared__ int64_t warp_sum[kMaxWarps];
  __shared__ int64_t cut_at[2], cut_first;
  __shared__ int cut_b;
  int64_t per;
  {
    const int each = (P.batch + blockDim.x - 1) / blockDim.x;
    const int b0 = min(P.batch, static_cast<int>(threadIdx.x) * each), b1 = min(P.batch, b0 + each);
    int64_t sum = 0;
    for (int b = b0; b < b1; ++b) sum += rounds_of(tokens_of(P, b), P.streams);
    int64_t run = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t x = __shfl_up_sync(0xffffffffu, run, o);
      if (lane >= o) run += x;
    }
    if (lane == 31) warp_sum[warp] = run;
    if (threadIdx.x < 2) cut_at[threadIdx.x] = INT64_MAX;
    __syncthreads();
    int64_t before = run - sum, total = 0;
    for (int w = 0; w < static_cast<int>(blockDim.x >> 5); ++w) {
      if (w < warp) before += warp_sum[w];
      total += warp_sum[w];
    }
    per = max((total + gridDim.x - 1) / gridDim.x, static_cast<int64_t>(kMinRounds));
#pragma unroll
    for (int i = 0; i < 2; ++i) {  // where this CTA begins, and where the next one does
      int64_t cut = (blockIdx.x + i) * per, at = before;
      if (at <= cut && cut < before + sum) {
        int b = b0, n = rounds_of(tokens_of(P, b), P.streams);
        while (cut >= at + n) {
          at += n;
          n = rounds_of(tokens_of(P, ++b), P.streams);
        }
        if (cut > at && n <= kWhole) {  // into a short request: behind it
          cut = at += n;
          ++b;
        }
        cut_at[i] = cut;
        if (i == 0) {
          cut_b = b;
          cut_first = at;
        }
      }
    }
    __syncthreads();
    if (threadIdx.x < 2) cut_at[threadIdx.x] = min(cut_at[threadIdx.x], total);
    __syncthreads();
  }
  int64_t f = cut_at[0];
  const int64_t f_begin = f, f_end = cut_at[1];
  if (f >= f_end) return;
  int b = cut_b;
  int64_t first = cut_first;
  const int yw = warp % P.y_cta, stream = warp / P.y_cta;
  const int y = blockIdx.y * P.y_cta + yw;
  const bool active = y < P.y_total;
  const int kvh = active ? y / P.chunks : 0;
  const int h0 = active ? (y - kvh * P.chunks) * kHeads : 0;
  const int heads = active ? min(kHeads, P.group - h0) : 0;
  const int head0 = kvh * P.group + h0;  // first query head

  // Two warps that share copies are 2 k and 2 k + 1; they have both their rings and one set of barriers.
  const bool leads = !SHARED || (warp & 1) == 0;
  const int owner = SHARED ? warp & ~1 : warp;
  const uint32_t ring = smem_u32(smem) + owner * G::kRingBytes;
  const uint32_t mine_at = SHARED ? (warp & 1) * G::kRow : 0;  // this warp's head in a row
  auto give_back = [&] {  // the stage just read may be written
    if constexpr (SHARED)
      asm volatile("bar.sync %0, 64;" ::"r"(1 + (warp >> 1)) : "memory");
    else
      __syncwarp();
  };
  const int round_tokens = kTile * P.streams;
  uint32_t phases = 0u;  // of full[warp][0], [1]
  bool given_up = false;

  while (f < f_end) {
    const int seq = tokens_of(P, b);
    const int rounds = rounds_of(seq, P.streams);
    const int r_begin = static_cast<int>(f - first);
    const int r_end = static_cast<int>(min(static_cast<int64_t>(rounds), f_end - first));
    const bool whole_request = r_begin == 0 && r_end == rounds;
    const int r0 = max(r_begin - kStart, 0);
    const int mine = r_end - kStart - r0;  // tiles of this warp here (not positive: only the request's start is)
    const int t_begin = r0 * round_tokens + stream * kTile;  // tile i begins at t_begin + i round_tokens
    const int32_t* table = P.table + b * P.table_stride;

    // Starts the copies of a tile. TMA: returns a bit for each of its two units that is there; by rows: one for
    // each of its tokens.
    int32_t id = -1, at = 0;    // block of the unit that this lane looked up and its first token there
    uint32_t there = 0u;        // which of the 32 units have a block
    auto issue = [&](int tile) {
      if (tile >= mine || !active) {
        if constexpr (!TMA) copy_commit();
        return 0u;
      }
      const int t0 = t_begin + tile * round_tokens;
      const uint32_t st = ring + (tile & 1) * 2 * kStage;
      if constexpr (TMA) {
        if ((tile & 15) == 0) {  // the next 32 units, one a lane
          const int t = t_begin + (tile + (lane >> 1)) * round_tokens + (lane & 1) * kUnit;
          id = -1;
          if (tile + (lane >> 1) < mine && t < seq) {
            const uint32_t col = P.cache.page_div.div(static_cast<uint32_t>(t));
            at = P.cache.page_div.mod(static_cast<uint32_t>(t), col);
            id = table[col];
            if (static_cast<uint32_t>(id) >= static_cast<uint32_t>(P.cache.num_blocks)) id = -1;
          }
          there = __ballot_sync(0xffffffffu, id >= 0);
        }
        const uint32_t two = (there >> (2 * (tile & 15))) & 3u;
        if (two != 0u && leads && !given_up && (lane >> 1) == (tile & 15)) {
          uint64_t* bar = &full[owner][tile & 1];
          mbar_arrive_expect_tx(bar, id >= 0 ? kStage : 0);
          if (id >= 0)
            copy_unit(st + (lane & 1) * kStage, &map, P.flat ? at * (G::kRow / 8) : 0, SHARED ? kvh >> 1 : kvh,
                      P.flat ? 0 : at, id, bar);
        }
        return two;
      } else {  // every row looks its own page up
        int32_t row_block = -1, row_at = 0;
        if (t0 + lane < seq) {
          const uint32_t col = P.cache.page_div.div(static_cast<uint32_t>(t0 + lane));
          row_at = P.cache.page_div.mod(static_cast<uint32_t>(t0 + lane), col);
          row_block = table[col];
          if (static_cast<uint32_t>(row_block) >= static_cast<uint32_t>(P.cache.num_blocks)) row_block = -1;
        }
        const uint32_t live = __ballot_sync(0xffffffffu, row_block >= 0);
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int i = 0; i < G::kChunks; ++i) {
            const int c = lane + 32 * i, v = c >= kUnit * G::kChunks;
            const int r = c / G::kChunks - (v ? kUnit : 0), piece = c % G::kChunks;
            const int32_t blk = __shfl_sync(0xffffffffu, row_block, u * kUnit + r);
            const int32_t off = __shfl_sync(0xffffffffu, row_at, u * kUnit + r);
            if (blk >= 0)
              copy16(st + u * kStage + c * 16,
                     P.cache.base + blk * P.cache.block_stride + (v ? P.cache.outer_stride : 0) +
                         off * P.cache.token_stride + kvh * P.cache.head_stride + piece * 16);
          }
        copy_commit();
        return live;
      }
    };
    // ---- q as operands: column gid is head gid / 2, odd columns the second parts (PAIR), or head gid
    uint32_t next;
    uint32_t bq[NG][2][2], bz[NZ][2];
    float factor[NH];
    {
      const int h = PAIR ? gid >> 1 : gid;
      const bool second = PAIR && (gid & 1) != 0;
      uint32_t xw[NG][4];
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        int4 w = make_int4(0, 0, 0, 0);
        if (h < heads)
          w = *reinterpret_cast<const int4*>(P.q + b * P.q_stride + (head0 + h) * static_cast<int64_t>(HD) +
                                             g * kGroup + tig * 8);
        xw[g][0] = w.x, xw[g][1] = w.y, xw[g][2] = w.z, xw[g][3] = w.w;
      }
      next = issue(0);  // behind the loads of q: both are under way together
      float top = 0.f;
      bool bad = false;
#pragma unroll
      for (int g = 0; g < NG; ++g)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          top = fmaxf(top, fmaxf(fabsf(bf_lo(xw[g][k])), fabsf(bf_hi(xw[g][k]))));
          bad |= (xw[g][k] & 0x7f80u) == 0x7f80u || (xw[g][k] & 0x7f800000u) == 0x7f800000u;
        }
      int flag = bad;
#pragma unroll
      for (int o = 1; o < 4; o <<= 1) {
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        flag |= __shfl_xor_sync(0xffffffffu, flag, o);
      }
      const int e = max(exponent(top), -100);  // the largest element comes to [2^13, 2^14)
      const float up = flag ? 0.f : copysignf(pow2(13 - e), P.qscale);  // a negative scale turns q: factor is positive
      float fac = flag ? __uint_as_float(0x7fc00000u) : ldexpf(fabsf(P.qscale), 24 + e - 13);
      if (fac < 1e-36f) fac = 1e-36f;  // (times -infinity is to be -infinity, and times 0 to be 0)
      if (fac > 3.4e38f) fac = 3.4e38f;
      float qs[NG];
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        float x[8];
        qs[g] = 0.f;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          x[2 * k] = flag ? 0.f : bf_lo(xw[g][k]) * up;
          x[2 * k + 1] = flag ? 0.f : bf_hi(xw[g][k]) * up;
          qs[g] += x[2 * k] + x[2 * k + 1];
        }
        qs[g] += __shfl_xor_sync(0xffffffffu, qs[g], 1);
        qs[g] += __shfl_xor_sync(0xffffffffu, qs[g], 2);
        // register i of a word has to do with elements i and i + 4
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float even[2], odd[2];
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            odd[k] = 0.0625f * x[2 * j + 1 + 4 * k];  // exact in fp16, but for the smallest elements
            even[k] = x[2 * j + 4 * k] - (PAIR ? odd[k] : 0.f);
            if (second) {
              even[k] -= __half2float(__float2half_rn(even[k]));
              odd[k] -= __half2float(__float2half_rn(odd[k]));
            }
          }
          bq[g][j][0] = half2(even[0], even[1]);
          bq[g][j][1] = half2(odd[0], odd[1]);
        }
      }
      // sums of q of group tig (+ 4) in the codes' unit 2^-24: three bf16 parts in k slots 2 tig, + 1, + 8 (the fourth: 0)
#pragma unroll
      for (int j = 0; j < NZ; ++j) {
        float s = 0.f;
#pragma unroll
        for (int g = 4 * j; g < 4 * j + 4 && g < NG; ++g) s = (g & 3) == tig ? qs[g] : s;
        s *= pow2(-24);
        const float s1 = __bfloat162float(__float2bfloat16(s)), s2 = __bfloat162float(__float2bfloat16(s - s1));
        bz[j][0] = second ? 0u : pack2(s1, s2);
        bz[j][1] = second ? 0u : pack2(s - s1 - s2, 0.f);
      }
#pragma unroll
      for (int n = 0; n < NH; ++n) factor[n] = __shfl_sync(0xffffffffu, fac, 8 * tig + 4 * n);
    }

    // ---- running state: of query head tig (PAIR) or 2 tig + n; m in the scores' unit before factor
    float m[NH], ref[NH], l[NH], z[NH][NG];  // ref = m factor, 0 before there is an m
    float acc[NG][4][NH];  // element 32 g + 4 gid + i, times f 2^-24; odd i: that of i - 1 and 16 times i's
    float vf = pow2(100);  // f; the first tile sets it
    constexpr int kWords = (NB + 3) / 4;
    uint32_t lacking[kWords] = {};         // the lane's heads' groups that have not been given a large weight where they should
#pragma unroll
    for (int n = 0; n < NH; ++n) {
      m[n] = -INFINITY;
      ref[n] = l[n] = 0.f;
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        z[n][g] = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[g][i][n] = 0.f;
      }
    }

    for (int tile = 0; tile < mine; ++tile) {
      const uint32_t here = next;
      next = issue(tile + 1);
      if constexpr (!TMA) {
        copy_wait<1>();
        __syncwarp();
      }
      if (here == 0u) continue;
      if constexpr (TMA) {
        if (!given_up) {
          uint64_t* bar = &full[owner][tile & 1];
          const uint32_t phase = (phases >> (tile & 1)) & 1u;
          bool ok = P.wait_ns != 0 && mbar_try_wait(bar, phase);
          if (!__all_sync(0xffffffffu, ok)) {
            ok = P.wait_ns != 0 && mbar_wait_bounded(bar, phase, P.wait_ns);
            if (!__all_sync(0xffffffffu, ok)) {  // the launch is given up when both copies in flight have had their time
              given_up = true;
              report_status(P.status, kStatusPipelineTimeout);
              mbar_wait_bounded(bar, phase, kWaitNs);
              if (next != 0u) mbar_wait_bounded(&full[owner][~tile & 1], (phases >> (~tile & 1)) & 1u, kWaitNs);
            }
          }
          phases ^= 1u << (tile & 1);
        }
        if (given_up) {  // no more copies, no more waiting; the results are NaN
          give_back();
          continue;
        }
      }
      const uint32_t st = ring + (tile & 1) * 2 * kStage + mine_at;
      const int left = seq - (t_begin + tile * round_tokens);  // tokens from this tile's first on, at least 1
      const bool whole = here == (TMA ? 3u : 0xffffffffu) && left >= kTile;
      uint32_t live = 0xffffffffu;
      if (!whole) {  // a bit for each token that counts; V of the others, which may hold anything, becomes zeros
        live = TMA ? (here & 1u ? 0xffffu : 0u) | (here & 2u ? 0xffff0000u : 0u) : here;
        if (left < kTile) live &= (1u << left) - 1u;
        if (!((live >> lane) & 1u)) {
          const uint32_t par = st + (lane >> 4) * kStage + (kUnit + (lane & 15)) * kStride + HD / 2;
#pragma unroll
          for (int g = 0; g < NG; ++g) asm volatile("st.shared.b32 [%0], %1;" ::"r"(par + 4 * g), "r"(0) : "memory");
        }
        if constexpr (TMA) fence_proxy_async_smem();  // the next copy into this place comes behind
        __syncwarp();
      }

      // ---- scores of tokens gid, gid + 8 of both units
      float s[2][2][NH];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const uint32_t k0 = st + u * kStage + gid * kStride, k1 = k0 + 8 * kStride;
        float c[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < NZ; ++j) {
          uint32_t z0[1], z1[1];  // (lanes without a group of their own meet zeros of bz)
          lds(z0, k0 + HD / 2 + 16 * j + 4 * (NG < 4 ? tig % NG : tig));
          lds(z1, k1 + HD / 2 + 16 * j + 4 * (NG < 4 ? tig % NG : tig));
          z0[0] = __byte_perm(z0[0], 0, 0x3232);
          z1[0] = __byte_perm(z1[0], 0, 0x3232);
          mma_bf16(c, z0[0], z1[0], z0[0], z1[0], bz[j][0], bz[j][1], c[0], c[1], c[2], c[3]);
        }
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
          for (int n = 0; n < NH; ++n) s[u][r][n] = c[2 * r + n];
        uint32_t par[2][NG];
        lds(par[0], k0 + HD / 2);
        lds(par[1], k1 + HD / 2);
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          uint32_t x0[1], x1[1];
          lds(x0, k0 + g * 16 + tig * 4);
          lds(x1, k1 + g * 16 + tig * 4);
          uint32_t a0[4], a1[4];
          if constexpr (PAIR) {
            code_pairs(a0, x0[0]);
            code_pairs(a1, x1[0]);
          } else {
            code_pairs_alone(a0, x0[0]);
            code_pairs_alone(a1, x1[0]);
          }
          mma_f16(c, a0[0], a1[0], a0[1], a1[1], bq[g][0][0], bq[g][0][1], 0.f, 0.f, 0.f, 0.f);
          mma_f16(c, a0[2], a1[2], a0[3], a1[3], bq[g][1][0], bq[g][1][1], c[0], c[1], c[2], c[3]);
#pragma unroll
          for (int r = 0; r < 2; ++r)
#pragma unroll
            for (int n = 0; n < NH; ++n)
              s[u][r][n] = fmaf(bf_lo(par[r][g]), PAIR ? c[2 * r] + c[2 * r + 1] : c[2 * r + n], s[u][r][n]);
        }
      }
      // ---- softmax. A tile without a new maximum, as most are after the first few, needs no sums scaled.
      float alpha[NH];
      bool higher = false;
#pragma unroll
      for (int n = 0; n < NH; ++n) {
        if (!whole) {
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int r = 0; r < 2; ++r)
              if (!((live >> (16 * u + 8 * r + gid)) & 1u)) s[u][r][n] = -INFINITY;
        }
        alpha[n] = fmaxf(fmaxf(s[0][0][n], s[0][1][n]), fmaxf(s[1][0][n], s[1][1][n]));
        higher |= alpha[n] > m[n];
      }
      higher = __any_sync(0xffffffffu, higher);
      if (higher) {
#pragma unroll
        for (int n = 0; n < NH; ++n) {
          float top = alpha[n];
#pragma unroll
          for (int o = 4; o < 32; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
          const bool rises = top > m[n];
          top = fmaxf(m[n], top);
          ref[n] = top == -INFINITY ? 0.f : top * factor[n];
          alpha[n] = rises ? ex2(fmaf(m[n], factor[n], -ref[n])) : 1.f;
          m[n] = top;
          l[n] *= alpha[n];
#pragma unroll
          for (int g = 0; g < NG; ++g) z[n][g] *= alpha[n];
        }
      } else {
#pragma unroll
        for (int n = 0; n < NH; ++n) alpha[n] = 1.f;
      }
#pragma unroll
      for (int n = 0; n < NH; ++n)
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            s[u][r][n] = ex2(fmaf(s[u][r][n], factor[n], -ref[n]));
            l[n] += s[u][r][n];
          }
      // ---- weights times V scales, as operands: PAIR columns are (head, group parity)
      uint32_t par[2][2][NG], bp[2][NB][2];
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          lds(par[u][r], st + u * kStage + (kUnit + gid + 8 * r) * kStride + HD / 2);
#pragma unroll
          for (int n = 0; n < NH; ++n)
#pragma unroll
            for (int g = 0; g < NG; ++g) z[n][g] = fmaf(s[u][r][n], bf_hi(par[u][r][g]), z[n][g]);
        }
      bool set = false;
      while (true) {
        uint32_t sum = 0u;  // infinite (or a NaN) if a weight is, or all are near it
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            float ps[NG][NH];
#pragma unroll
            for (int n = 0; n < NH; ++n) {
              const float pf = s[u][r][n] * vf;
#pragma unroll
              for (int g = 0; g < NG; ++g) ps[g][n] = pf * bf_lo(par[u][r][g]);
            }
#pragma unroll
            for (int k = 0; k < NB; ++k) {
              const uint32_t p = PAIR ? half2(ps[2 * k][0], ps[2 * k + 1][0]) : half2(ps[k][0], ps[k][NH - 1]);
              sum = add_half2(sum, p);
              bp[u][k][r] = p;
            }
          }
        const bool over = (sum & 0x7c00u) == 0x7c00u || (sum & 0x7c000000u) == 0x7c000000u;
        if (set || !__any_sync(0xffffffffu, over)) break;
        set = true;
        float top = 0.f;
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int r = 0; r < 2; ++r)
#pragma unroll
            for (int n = 0; n < NH; ++n)
#pragma unroll
              for (int g = 0; g < NG; ++g) top = fmaxf(top, s[u][r][n] * bf_lo(seldom(par[u][r][g])));
        const int old = exponent(vf), now = min(old, kBest - exponent(warp_max(top)));
        vf = pow2(now);
#pragma unroll
        for (int n = 0; n < NH; ++n) alpha[n] *= pow2(max(now - old, -126));
      }
      if (higher || set) {  // has each group that needs it been given a weight of 2 or more, bit 14 of an fp16?
        // operand k of lanes tig at bits 15 - (4 tig + k) and 16 above, four operands a word
        constexpr int kOps = NB < 4 ? NB : 4;
        constexpr uint32_t kMine = 0x8000u / (1u << (kOps - 1)) * ((1u << kOps) - 1u);
        constexpr uint32_t kAll = (kMine | kMine >> 4 | kMine >> 8 | kMine >> 12) * 0x10001u;
        // (from 128 on made anew each time: 1.3 % with 4 heads of 128; at 64 kept in registers, there are some: 1.3 %)
        const uint32_t at = 4 * (HD < 128 ? tig : seldom(tig)), own = (kMine >> at) * 0x10001u;
        const uint32_t exempt = (alpha[0] == 1.f ? own & 0xffffu : 0u) | (alpha[NH - 1] == 1.f ? own & 0xffff0000u : 0u);
#pragma unroll
        for (int w = 0; w < kWords; ++w) {
          uint32_t have = 0u;
#pragma unroll
          for (int k = 4 * w; k < 4 * w + kOps; ++k)
            have |= ((bp[0][k][0] | bp[0][k][1] | bp[1][k][0] | bp[1][k][1]) & 0x40004000u) >> (k & 3);
          have = __reduce_or_sync(0xffffffffu, ((have << 1) >> at) | exempt);
          lacking[w] |= kAll & ~have;
        }
      }
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int k = 0; k < NB; ++k)
#pragma unroll
          for (int r = 0; r < 2; ++r) bp[u][k][r] = transpose8x8(bp[u][k][r]);
      // ---- acc += sum p' c: this lane's codes of tokens 2 tig, 2 tig + 1 and those 8 further
      uint32_t x[2][4][NW];
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int t = 0; t < 4; ++t)
          lds(x[u][t], st + u * kStage + (kUnit + 2 * tig + (t & 1) + 8 * (t >> 1)) * kStride + gid * NW * 4);
#pragma unroll
      for (int k = 0; k < NW; ++k) {  // groups 2 k and 2 k + 1
        uint32_t w[2][2][2][4];       // [unit][group][tokens 2 tig.. / 8 further][register]
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            code_pairs(w[u][0][r], __byte_perm(x[u][2 * r][k], x[u][2 * r + 1][k], 0x5410));
            code_pairs(w[u][1][r], __byte_perm(x[u][2 * r][k], x[u][2 * r + 1][k], 0x7632));
          }
        if constexpr (PAIR) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float c[4];
            mma_f16(c, w[0][0][0][i], w[0][1][0][i], w[0][0][1][i], w[0][1][1][i], bp[0][k][0], bp[0][k][1], 0.f, 0.f,
                    0.f, 0.f);
            mma_f16(c, w[1][0][0][i], w[1][1][0][i], w[1][0][1][i], w[1][1][1][i], bp[1][k][0], bp[1][k][1], c[0], c[1],
                    c[2], c[3]);
            acc[2 * k][i][0] = fmaf(acc[2 * k][i][0], alpha[0], c[0]);
            acc[2 * k + 1][i][0] = fmaf(acc[2 * k + 1][i][0], alpha[0], c[3]);
          }
        } else {
#pragma unroll
          for (int p = 0; p < 2; ++p)
#pragma unroll
            for (int j = 0; j < 2; ++j) {  // rows 0-7: register 2 j, rows 8-15: register 2 j + 1
              const int g = 2 * k + p;
              float c[4];
              mma_f16(c, w[0][p][0][2 * j], w[0][p][0][2 * j + 1], w[0][p][1][2 * j], w[0][p][1][2 * j + 1], bp[0][g][0],
                      bp[0][g][1], 0.f, 0.f, 0.f, 0.f);
              mma_f16(c, w[1][p][0][2 * j], w[1][p][0][2 * j + 1], w[1][p][1][2 * j], w[1][p][1][2 * j + 1], bp[1][g][0],
                      bp[1][g][1], c[0], c[1], c[2], c[3]);
#pragma unroll
              for (int n = 0; n < NH; ++n) {
                acc[g][2 * j][n] = fmaf(acc[g][2 * j][n], alpha[n], c[n]);
                acc[g][2 * j + 1][n] = fmaf(acc[g][2 * j + 1][n], alpha[n], c[2 + n]);
              }
            }
        }
      }
      give_back();
    }
    if constexpr (!TMA) copy_wait<0>();
    __syncwarp();
    if (given_up) {
#pragma unroll
      for (int n = 0; n < NH; ++n) l[n] = __uint_as_float(0x7fc00000u);
    }

#pragma unroll
    for (int n = 0; n < NH; ++n) m[n] = m[n] == -INFINITY ? m[n] : m[n] * factor[n];
    // ---- sums over the lanes that share a head; codes' unit and f out of the sums, zeros' part in
#pragma unroll
    for (int n = 0; n < NH; ++n) {
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) {
        l[n] += __shfl_xor_sync(0xffffffffu, l[n], o);
#pragma unroll
        for (int g = 0; g < NG; ++g) z[n][g] += __shfl_xor_sync(0xffffffffu, z[n][g], o);
      }
#pragma unroll
      for (int g = 0; g < NG; ++g)
#pragma unroll
        for (int i = 0; i < 4; i += 2) {
          acc[g][i + 1][n] = fmaf((acc[g][i + 1][n] - acc[g][i][n]) * 1048576.f, 1.f / vf, z[n][g]);
          acc[g][i][n] = fmaf(acc[g][i][n] * 16777216.f, 1.f / vf, z[n][g]);
        }
    }
    bool large = false;  // (m large and negative at first, and higher later, has left an infinite l or a NaN, or nothing)
#pragma unroll
    for (int n = 0; n < NH; ++n)
      large |= fabsf(ref[n]) > kLargeScore || !(l[n] < INFINITY);
    uint32_t groups = 0u;
#pragma unroll
    for (int w = 0; w < kWords; ++w)
#pragma unroll
      for (int k = 4 * w; k < 4 * w + 4 && k < NB; ++k) {
        if (lacking[w] & (0x8888u >> (k & 3))) groups |= 1u << (PAIR ? 2 * k : k);
        if (lacking[w] & (0x88880000u >> (k & 3))) groups |= 1u << (PAIR ? 2 * k + 1 : k);
      }
    large = __any_sync(0xffffffffu, large);
    if ((large || groups != 0u) && !given_up &&
        (large || any_scale<HD>(P, b, kvh, seq, t_begin, mine, round_tokens, groups)))
      share_in_fp32<HD, NH>(P, b, kvh, head0, heads, seq, t_begin, mine, round_tokens, m, l, acc);
    if constexpr (SHARED) give_back();  // a warp's limited waits are for copies, not for the other's second go
    // ---- streams of this CTA: the first one's warp takes the others' results, lane by lane
    if (P.streams > 1) {
      constexpr int kVals = NH * (2 + 4 * NG);
      float* red = reinterpret_cast<float*>(smem) + warp * kVals * 32 + lane;
      __syncthreads();
      if (stream > 0) {
#pragma unroll
        for (int n = 0; n < NH; ++n) {
          red[(2 * n) * 32] = m[n];
          red[(2 * n + 1) * 32] = l[n];
#pragma unroll
          for (int k = 0; k < 4 * NG; ++k) red[(2 * NH + n * 4 * NG + k) * 32] = acc[k / 4][k % 4][n];
        }
      }
      __syncthreads();
      if (stream == 0) {
        for (int t = 1; t < P.streams; ++t) {
          const float* o = red + t * P.y_cta * kVals * 32;
#pragma unroll
          for (int n = 0; n < NH; ++n) {
            const float mo = o[(2 * n) * 32], lo = o[(2 * n + 1) * 32];
            const float top = fmaxf(m[n], mo);
            const float f0 = l[n] == 0.f ? 0.f : exp2f(m[n] - top), f1 = lo == 0.f ? 0.f : exp2f(mo - top);
            m[n] = top;
            l[n] = f0 * l[n] + f1 * lo;
#pragma unroll
            for (int k = 0; k < 4 * NG; ++k)
              acc[k / 4][k % 4][n] = f0 * acc[k / 4][k % 4][n] + f1 * o[(2 * NH + n * 4 * NG + k) * 32];
          }
        }
      }
      if constexpr (TMA) fence_proxy_async_smem();  // the next request's copies come behind
      __syncthreads();
    }
    // ---- to the output, or to this CTA's slot of partial results
    if (stream == 0 && active) {
      const int64_t slot_row = (static_cast<int64_t>(blockIdx.x) * 2 + (f == f_begin ? 0 : 1)) * P.hq + head0;
#pragma unroll
      for (int n = 0; n < NH; ++n) {
        const int h = NH * tig + n;
        if (h >= heads) continue;
        const float r = whole_request ? (l[n] == 0.f ? 0.f : 1.f / l[n]) : 1.f;
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          const int d = g * kGroup + gid * 4;
          if (whole_request)
            *reinterpret_cast<uint2*>(P.out + (static_cast<int64_t>(b) * P.hq + head0 + h) * HD + d) =
                make_uint2(pack2(acc[g][0][n] * r, acc[g][1][n] * r), pack2(acc[g][2][n] * r, acc[g][3][n] * r));
          else
            *reinterpret_cast<float4*>(P.part_acc + (slot_row + h) * HD + d) =
                make_float4(acc[g][0][n], acc[g][1][n], acc[g][2][n], acc[g][3][n]);
        }
        if (!whole_request && gid == 0) {
          P.part_ml[(slot_row + h) * 2] = m[n];
          P.part_ml[(slot_row + h) * 2 + 1] = l[n];
        }
      }
      if (P.parts != nullptr && r_begin == 0 && y == 0 && lane == 0)
        P.parts[b] = make_int2(2 * blockIdx.x + (f == f_begin ? 0 : 1),
                               whole_request ? 1 : static_cast<int>((first + rounds - 1) / per) - static_cast<int>(blockIdx.x) + 1);
    }
    f = first + r_end;
    if (r_end == rounds) {
      first += rounds;
      ++b;
    }
  }
}

// How a launch is laid out: (KV head, chunk) pairs and streams a CTA, CTAs along the work.
struct Plan {
  int chunks, y_total, y_cta, y_ctas, streams, ctas, sms;
  bool cut;  // whether a request may be cut, and the merge is to follow
};
inline Plan plan_decode(int batch, int hq, int hkv, int hd, int64_t max_tokens, int ctas, int sm_count) {
  Plan p{};
  p.sms = sm_count;
  p.chunks = (hq / hkv + kHeads - 1) / kHeads;
  p.y_total = hkv * p.chunks;
  // Where requests are short and few, one KV head a CTA: its 8 streams of tokens take a request's 1,024 tokens in 4
  // rounds, and nothing is cut (600 tokens of one request, 8 KV heads: 8.8 us in place of 10.5). Else as many as it
  // has warps, an even number so that pairs can share copies, unless requests are so few that each would be cut into
  // more than 80 parts (131,072 tokens of one request, 8 KV heads: 296 parts of 8 heads 40 us, 74 of two 37 us, 37 of
  // one 47 us).
  const int most = (hd == 256 ? 8 : 16) / kMaxWarps;  // registers allow 16 warps an SM (8 with 256 elements a head)
  const bool short_few = kStart + (max_tokens + 8 * kTile - 1) / (8 * kTile) <= kWhole &&
                         static_cast<int64_t>(batch) * p.y_total <= 2 * most * sm_count;
  for (int n = (p.y_total + kMaxWarps - 1) / kMaxWarps;; ++n) {
    const int y = short_few ? 1 : (p.y_total + n - 1) / n;
    if (y > 1 && y % 2 != 0 && y < kMaxWarps && p.y_total % 2 == 0) continue;
    p.y_cta = y;
    p.y_ctas = (p.y_total + y - 1) / y;
    p.streams = kMaxWarps / y;
    const int per_sm = std::max(1, most * kMaxWarps / (y * p.streams));
    p.ctas = ctas > 0 ? ctas : std::max(1, sm_count * per_sm / p.y_ctas);
    if (p.ctas / batch <= 80 || y <= 2) break;
  }
  const int64_t rounds = (max_tokens + kTile * p.streams - 1) / (kTile * p.streams);
  p.ctas = static_cast<int>(std::min<int64_t>(p.ctas, std::max<int64_t>(1, (batch * (rounds + kStart) + kMinRounds - 1) / kMinRounds)));
  p.cut = p.ctas > 1 && rounds + kStart > kWhole;
  return p;
}

// The pool as a tensor of 8-byte words [block][K / V][token][head][row], boxes of a unit's rows of one head. Where a
// head's rows of a page are contiguous (head-first pools) and a unit's are no longer than a box may be, the tokens
// are part of the innermost dimension: 2 runs a box instead of 32. `shared`, if asked for and the pool is
// token-first with an even number of heads: a box has the rows of two heads.
inline bool make_map(CUtensorMap* map, const Cache& c, int row, bool* flat, bool* shared) {
  static const PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    const bool ok = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
                    q == cudaDriverEntryPointSuccess;
    return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(ok ? p : nullptr);
  }();
  if (!fn || c.num_blocks < 1) return false;
  *flat = c.token_stride == row && kUnit * row / 8 <= 256;
  *shared = *shared && !*flat && c.head_stride == row && c.heads % 2 == 0;
  const int64_t head_stride = *shared ? 2 * c.head_stride : c.head_stride;
  const int heads = *shared ? c.heads / 2 : c.heads;
  const cuuint64_t words = static_cast<cuuint64_t>(row) / 8 * (*shared ? 2 : 1);
  const cuuint64_t dims[5] = {*flat ? words * c.page : words, static_cast<cuuint64_t>(heads),
                              *flat ? 1 : static_cast<cuuint64_t>(c.page), 2, static_cast<cuuint64_t>(c.num_blocks)};
  // a dimension of one may come with any stride
  const cuuint64_t strides[4] = {static_cast<cuuint64_t>(heads > 1 ? head_stride : row),
                                 static_cast<cuuint64_t>(c.token_stride), static_cast<cuuint64_t>(c.outer_stride),
                                 static_cast<cuuint64_t>(c.num_blocks > 1 ? c.block_stride : row)};
  const cuuint32_t box[5] = {static_cast<cuuint32_t>(*flat ? words * kUnit : words), 1,
                             static_cast<cuuint32_t>(*flat ? 1 : kUnit), 2, 1};
  const cuuint32_t step[5] = {1, 1, 1, 1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT64, 5, c.base, dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) ==
         CUDA_SUCCESS;
}

// Lets a kernel be put in place before the one in front of it has ended; it waits for that itself.
template <typename K, typename... A>
cudaError_t launch_overlapped(K kernel, dim3 grid, int threads, int smem, cudaStream_t stream, const A&... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

template <int HD, bool PAIR, Copies COPIES>
cudaError_t launch_decode_kernel(const AttnParams& P, const CUtensorMap& map, const Plan& plan, cudaStream_t stream) {
  auto kernel = kv4_decode_kernel<HD, PAIR, COPIES>;
  const int warps = plan.y_cta * plan.streams;
  constexpr int kVals = (PAIR ? 1 : 2) * (2 + 4 * (HD / kGroup));  // merging streams, in the ring's place
  constexpr int kWarpBytes = std::max(Geometry<HD>::kRingBytes, kVals * 128);
  // what any launch may take: another thread's launch of this kernel may stand between this call and the next
  const cudaError_t e =
      cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxWarps * kWarpBytes);
  if (e != cudaSuccess) return e;
  return launch_overlapped(kernel, dim3(plan.ctas, plan.y_ctas), warps * 32, warps * kWarpBytes, stream, P, map);
}

template <int HD>
cudaError_t launch_decode_hd(AttnParams& P, const Plan& plan, cudaStream_t stream) {
  CUtensorMap map{};
  bool shared = HD < 256 && plan.chunks == 1 && plan.y_cta % 2 == 0;
  const bool tma = P.cache.page % kUnit == 0 && make_map(&map, P.cache, row_bytes(HD), &P.flat, &shared);
  cudaError_t e;
  if constexpr (HD == 256) {
    if (P.group <= 4)
      e = tma ? launch_decode_kernel<HD, true, kTma>(P, map, plan, stream)
              : launch_decode_kernel<HD, true, kRows>(P, map, plan, stream);
    else
      e = tma ? launch_decode_kernel<HD, false, kTma>(P, map, plan, stream)
              : launch_decode_kernel<HD, false, kRows>(P, map, plan, stream);
  } else {
    if (P.group <= 4)
      e = !tma     ? launch_decode_kernel<HD, true, kRows>(P, map, plan, stream)
          : shared ? launch_decode_kernel<HD, true, kTmaShared>(P, map, plan, stream)
                   : launch_decode_kernel<HD, true, kTma>(P, map, plan, stream);
    else
      e = !tma     ? launch_decode_kernel<HD, false, kRows>(P, map, plan, stream)
          : shared ? launch_decode_kernel<HD, false, kTmaShared>(P, map, plan, stream)
                   : launch_decode_kernel<HD, false, kTma>(P, map, plan, stream);
  }
  if (e != cudaSuccess || !plan.cut) return e;
  const int heads_cta = static_cast<int64_t>(P.batch) * P.hq <= 2 * plan.sms ? 1 : kMergeWarps;
  return launch_overlapped(kv4_merge_kernel<HD>, dim3((P.hq + heads_cta - 1) / heads_cta, P.batch), kMergeWarps * 32, 0,
                           stream, P, heads_cta);
}

inline cudaError_t launch_decode(AttnParams& P, int hd, const Plan& plan, cudaStream_t stream) {
  switch (hd) {
    case 64: return launch_decode_hd<64>(P, plan, stream);
    case 128: return launch_decode_hd<128>(P, plan, stream);
    case 256: return launch_decode_hd<256>(P, plan, stream);
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace kv4
}  // namespace kvbm
