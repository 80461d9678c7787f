// Operators of the 4-bit paged KV cache (row format: kv4_format.cuh): head norms
// + RoPE + cache write, rows back to bf16, decode attention.
#include "common.cuh"
#include "kv4_format.cuh"
#include "kvbm_kernels.h"
#include "paged_decode_kv4.cuh"

#include <algorithm>

using namespace kvbm;
using kvbm::kv4::Cache;

namespace {

constexpr int kThreads = 256;

// ---------------------------------------------------------------------------
// q/k head norms + RoPE + paged cache write, one pass over a packed qkv.
//
//   y = w x / sqrt(mean(x^2) + eps)          (left out without a weight)
//   out[i] = y[i] cos - y[i + R/2] sin, out[i + R/2] = y[i + R/2] cos + y[i] sin,  i < R/2; the rest as it is
//
// all in fp32 and rounded to bf16 once. The cache takes that bf16 k and the bf16
// v, so quantising a 16-bit cache later gives the same codes.
//
// A row of HD elements is held by HD/8 lanes, 16 bytes each. The rotation
// partner's input (not its normalised value) comes by shuffle: both lanes know
// the row's 1/rms, so exchanging 4 packed registers does.
// ---------------------------------------------------------------------------
struct WriteParams {
  __nv_bfloat16* qkv;
  int64_t qkv_stride;  // elements between tokens
  int64_t tokens;
  int hq, hkv, rot, max_pos;
  const int32_t* positions;
  const float* cos_sin;
  const __nv_bfloat16* q_weight;
  const __nv_bfloat16* k_weight;
  float eps;
  const int64_t* slots;
  Cache cache;
  FastDiv page_div, heads_div;
  __nv_bfloat16* q_out;
  __nv_bfloat16* k_out;
};

template <int HD, bool KV4>
__global__ void __launch_bounds__(kThreads) qk_norm_rope_kv_write_kernel(const __grid_constant__ WriteParams P) {
  constexpr int L = HD / 8;  // lanes a row
  const int H = P.hq + 2 * P.hkv;
  const int l = threadIdx.x % L;
  const int64_t item = (static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x) / L;
  const int64_t t = item / H;
  const int h = static_cast<int>(item - t * H);
  const bool live = t < P.tokens;
  const int32_t pos = live ? P.positions[t] : -1;
  const bool ok = pos >= 0 && pos < P.max_pos;  // a token outside the table is left alone
  const bool is_q = h < P.hq, is_v = h >= P.hq + P.hkv;
  __nv_bfloat16* row = P.qkv + t * P.qkv_stride + static_cast<int64_t>(h) * HD + 8 * l;
  int4 x4 = make_int4(0, 0, 0, 0);
  if (ok) x4 = *reinterpret_cast<const int4*>(row);
  uint32_t x[4] = {(uint32_t)x4.x, (uint32_t)x4.y, (uint32_t)x4.z, (uint32_t)x4.w};

  float ss = 0.f;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float a = kv4::bf_lo(x[k]), b = kv4::bf_hi(x[k]);
    ss = fmaf(a, a, fmaf(b, b, ss));
  }
#pragma unroll
  for (int o = 1; o < L; o <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  const int half = P.rot / 16;  // lanes that hold one half of the rotated elements
  const int partner = l < half ? l + half : l < 2 * half ? l - half : l;
  uint32_t xp[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) xp[k] = __shfl_sync(0xffffffffu, x[k], partner, L);

  if (ok && !is_v) {
    const __nv_bfloat16* w = is_q ? P.q_weight : P.k_weight;
    float inv = 1.f;
    uint32_t wm[4] = {0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u}, wp[4] = {wm[0], wm[0], wm[0], wm[0]};
    if (w != nullptr) {
      inv = rsqrtf(ss / HD + P.eps);
      const int4 a = reinterpret_cast<const int4*>(w)[l], b = reinterpret_cast<const int4*>(w)[partner];
      wm[0] = a.x, wm[1] = a.y, wm[2] = a.z, wm[3] = a.w;
      wp[0] = b.x, wp[1] = b.y, wp[2] = b.z, wp[3] = b.w;
    }
    float c[8], s[8];
    if (l < 2 * half) {
      const float* cs = P.cos_sin + static_cast<int64_t>(pos) * P.rot + (l < half ? l : l - half) * 8;
      const float sign = l < half ? -1.f : 1.f;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        c[k] = cs[k];
        s[k] = sign * cs[P.rot / 2 + k];
      }
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) c[k] = 1.f, s[k] = 0.f;
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float m0 = kv4::bf_lo(x[k]) * inv * kv4::bf_lo(wm[k]), m1 = kv4::bf_hi(x[k]) * inv * kv4::bf_hi(wm[k]);
      const float p0 = kv4::bf_lo(xp[k]) * inv * kv4::bf_lo(wp[k]), p1 = kv4::bf_hi(xp[k]) * inv * kv4::bf_hi(wp[k]);
      x[k] = kv4::pack2(m0 * c[2 * k] + p0 * s[2 * k], m1 * c[2 * k + 1] + p1 * s[2 * k + 1]);
    }
    const int4 y = make_int4(x[0], x[1], x[2], x[3]);
    if (P.q_out == nullptr)
      *reinterpret_cast<int4*>(row) = y;
    else if (is_q)
      *reinterpret_cast<int4*>(P.q_out + (t * P.hq + h) * HD + 8 * l) = y;
    else if (P.k_out != nullptr)
      *reinterpret_cast<int4*>(P.k_out + (t * P.hkv + h - P.hq) * HD + 8 * l) = y;
  }
  const int64_t slot = ok ? P.slots[t] : -1;
  const bool store = !is_q && slot >= 0 && slot < static_cast<int64_t>(P.cache.num_blocks) * P.cache.page;
  uint8_t* dst = nullptr;
  if (store) {
    const int64_t blk = slot / P.cache.page, off = slot - blk * P.cache.page;
    dst = P.cache.base + blk * P.cache.block_stride + (is_v ? P.cache.outer_stride : 0) + off * P.cache.token_stride +
          static_cast<int64_t>(h - P.hq - (is_v ? P.hkv : 0)) * P.cache.head_stride;
  }
  if constexpr (KV4) {
    uint32_t scale_zero;
    const uint32_t codes = kv4::quantise8(x, &scale_zero);
    if (store) {
      kv4::store_codes<HD>(dst, l, is_v, codes);
      if ((l & 3) == 0) reinterpret_cast<uint32_t*>(dst + HD / 2)[l >> 2] = scale_zero;
      constexpr int kUsed = HD / 2 + HD / 8;
      if constexpr (kUsed < kv4::row_bytes(HD))
        if (l < (kv4::row_bytes(HD) - kUsed) / 4) reinterpret_cast<uint32_t*>(dst + kUsed)[l] = 0u;
    }
  } else if (store) {
    reinterpret_cast<int4*>(dst)[l] = make_int4(x[0], x[1], x[2], x[3]);
  }
}

// ---------------------------------------------------------------------------
// Rows of the cache back to bf16: k_out[t][h] / v_out[t][h] = z + s c of slot
// slots[t] (zeros for a slot outside the pool).
// ---------------------------------------------------------------------------
struct GatherParams {
  Cache cache;
  const int64_t* slots;
  int64_t tokens;
  __nv_bfloat16* k_out;
  __nv_bfloat16* v_out;
};

template <int HD>
__global__ void __launch_bounds__(kThreads) kv4_gather_kernel(const __grid_constant__ GatherParams P) {
  constexpr int L = HD / 8;
  const int l = threadIdx.x % L;
  const int64_t item = (static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x) / L;
  const int64_t t = item / (2 * P.cache.heads);
  if (t >= P.tokens) return;
  const int r = static_cast<int>(item - t * 2 * P.cache.heads);
  const bool value = r >= P.cache.heads;
  const int h = value ? r - P.cache.heads : r;
  const int64_t slot = P.slots[t];
  int4 o = make_int4(0, 0, 0, 0);
  if (slot >= 0 && slot < static_cast<int64_t>(P.cache.num_blocks) * P.cache.page) {
    const int64_t blk = slot / P.cache.page, off = slot - blk * P.cache.page;
    const uint8_t* row = P.cache.base + blk * P.cache.block_stride + (value ? P.cache.outer_stride : 0) +
                         off * P.cache.token_stride + static_cast<int64_t>(h) * P.cache.head_stride;
    o = kv4::dequantise8(kv4::load_codes<HD>(row, l, value), reinterpret_cast<const uint32_t*>(row + HD / 2)[l >> 2]);
  }
  reinterpret_cast<int4*>((value ? P.v_out : P.k_out) + (t * P.cache.heads + h) * HD)[l] = o;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

bool cache_ok(const Cache& c) {
  return c.base != nullptr && aligned16(c.base) && c.block_stride % 16 == 0 && c.outer_stride % 16 == 0 &&
         c.token_stride % 16 == 0 && c.head_stride % 16 == 0 && c.page > 0 && c.num_blocks >= 0 && c.heads > 0;
}

}  // namespace

extern "C" int kvbm_qk_norm_rope_kv_write(void* qkv, int64_t qkv_stride, int64_t tokens, int hq, int hkv, int hd,
                                          int rot, const int32_t* positions, const float* cos_sin, int max_pos,
                                          const void* q_weight, const void* k_weight, float eps, int bits, void* kv,
                                          int64_t block_stride, int64_t outer_stride, int64_t token_stride,
                                          int64_t head_stride, int page, int num_blocks, const int64_t* slots,
                                          void* q_out, void* k_out, cudaStream_t stream) {
  if (tokens == 0) return cudaSuccess;
  WriteParams P{};
  P.cache = Cache{static_cast<uint8_t*>(kv), block_stride, outer_stride, token_stride, head_stride, page, num_blocks, hkv};
  if (tokens < 0 || hq < 0 || !cache_ok(P.cache) || !qkv || !positions || !cos_sin || !slots || !aligned16(qkv) ||
      qkv_stride % 8 != 0 || !aligned16(cos_sin) || !aligned16(q_out) || !aligned16(k_out) || !aligned16(q_weight) ||
      !aligned16(k_weight) || rot <= 0 || rot > hd || rot % 16 != 0 || max_pos < 0 || (bits != 4 && bits != 16) ||
      (k_out && !q_out))
    return cudaErrorInvalidValue;
  P.qkv = static_cast<__nv_bfloat16*>(qkv);
  P.qkv_stride = qkv_stride;
  P.tokens = tokens;
  P.hq = hq;
  P.hkv = hkv;
  P.rot = rot;
  P.max_pos = max_pos;
  P.positions = positions;
  P.cos_sin = cos_sin;
  P.q_weight = static_cast<const __nv_bfloat16*>(q_weight);
  P.k_weight = static_cast<const __nv_bfloat16*>(k_weight);
  P.eps = eps;
  P.slots = slots;
  P.q_out = static_cast<__nv_bfloat16*>(q_out);
  P.k_out = static_cast<__nv_bfloat16*>(k_out);
  const int64_t ctas = (tokens * (hq + 2 * hkv) * (hd / 8) + kThreads - 1) / kThreads;
  if (ctas > 0x7fffffff) return cudaErrorInvalidValue;
  const unsigned grid = static_cast<unsigned>(ctas);
#define KVBM_WRITE(HD)                                                                           \
  case HD:                                                                                       \
    if (bits == 4)                                                                               \
      qk_norm_rope_kv_write_kernel<HD, true><<<grid, kThreads, 0, stream>>>(P);                  \
    else                                                                                         \
      qk_norm_rope_kv_write_kernel<HD, false><<<grid, kThreads, 0, stream>>>(P);                 \
    break;
  switch (hd) {
    KVBM_WRITE(64)
    KVBM_WRITE(128)
    KVBM_WRITE(256)
    default: return cudaErrorInvalidValue;
  }
#undef KVBM_WRITE
  return cudaGetLastError();
}

extern "C" int kvbm_kv4_gather(const void* kv, int64_t block_stride, int64_t outer_stride, int64_t token_stride,
                               int64_t head_stride, int page, int num_blocks, int heads, int hd, const int64_t* slots,
                               int64_t tokens, void* k_out, void* v_out, cudaStream_t stream) {
  if (tokens == 0) return cudaSuccess;
  GatherParams P{};
  P.cache = Cache{static_cast<uint8_t*>(const_cast<void*>(kv)), block_stride, outer_stride, token_stride, head_stride,
                  page, num_blocks, heads};
  if (tokens < 0 || !cache_ok(P.cache) || !slots || !k_out || !v_out || !aligned16(k_out) || !aligned16(v_out))
    return cudaErrorInvalidValue;
  P.slots = slots;
  P.tokens = tokens;
  P.k_out = static_cast<__nv_bfloat16*>(k_out);
  P.v_out = static_cast<__nv_bfloat16*>(v_out);
  const int64_t ctas = (tokens * 2 * heads * (hd / 8) + kThreads - 1) / kThreads;
  if (ctas > 0x7fffffff) return cudaErrorInvalidValue;
  const unsigned grid = static_cast<unsigned>(ctas);
  switch (hd) {
    case 64: kv4_gather_kernel<64><<<grid, kThreads, 0, stream>>>(P); break;
    case 128: kv4_gather_kernel<128><<<grid, kThreads, 0, stream>>>(P); break;
    case 256: kv4_gather_kernel<256><<<grid, kThreads, 0, stream>>>(P); break;
    default: return cudaErrorInvalidValue;
  }
  return cudaGetLastError();
}

// How a launch of the decode attention is laid out: out[0] floats of scratch, out[1]
// CTAs along the work. `ctas` 0: one for each the GPU holds at a time.
extern "C" int kvbm_paged_decode_attn_kv4_plan(int batch, int hq, int hkv, int hd, int64_t max_tokens, int ctas,
                                               int sm_count, int64_t* out) {
  if (!out || batch <= 0 || hkv <= 0 || hq <= 0 || hq % hkv != 0 || max_tokens < 0 || ctas < 0 || sm_count <= 0)
    return cudaErrorInvalidValue;
  const kv4::Plan p = kv4::plan_decode(batch, hq, hkv, hd, max_tokens, ctas, sm_count);
  out[0] = static_cast<int64_t>(p.ctas) * 2 * hq * (hd + 2) + 2 * (static_cast<int64_t>(batch) + 1);
  out[1] = p.ctas;
  return cudaSuccess;
}

// `scratch`: 16-byte aligned floats as the plan says.
extern "C" int kvbm_paged_decode_attn_kv4(const void* q, int64_t q_stride, const void* kv, int64_t block_stride,
                                          int64_t outer_stride, int64_t token_stride, int64_t head_stride, int page,
                                          int num_blocks, const int32_t* block_table, int64_t table_stride,
                                          int max_blocks, const int32_t* seq_lens, int batch, int hq, int hkv, int hd,
                                          float softmax_scale, int ctas, int sm_count, float* scratch, void* out,
                                          cudaStream_t stream) {
  if (batch == 0) return cudaSuccess;
  kv4::AttnParams P{};
  P.cache = Cache{static_cast<uint8_t*>(const_cast<void*>(kv)), block_stride, outer_stride, token_stride, head_stride,
                  page, num_blocks, hkv};
  if (batch < 0 || batch > 65535 || hkv <= 0 || hq <= 0 || hq % hkv != 0 || !cache_ok(P.cache) || !q || !aligned16(q) ||
      q_stride % 8 != 0 || !out || !aligned16(out) || !seq_lens || max_blocks < 0 || (max_blocks > 0 && !block_table) ||
      ctas < 0 || sm_count <= 0 || !scratch || !aligned16(scratch))
    return cudaErrorInvalidValue;
  const kv4::Plan plan =
      kv4::plan_decode(batch, hq, hkv, hd, static_cast<int64_t>(max_blocks) * page, ctas, sm_count);
  if (plan.y_ctas > 65535 || static_cast<int64_t>(batch) * hq > 0x7fffffff) return cudaErrorInvalidValue;
  P.q = static_cast<const __nv_bfloat16*>(q);
  P.q_stride = q_stride;
  P.table = block_table;
  P.table_stride = table_stride;
  P.max_blocks = max_blocks;
  P.seq_lens = seq_lens;
  P.batch = batch;
  P.hq = hq;
  P.group = hq / hkv;
  P.chunks = plan.chunks;
  P.y_total = plan.y_total;
  P.y_cta = plan.y_cta;
  P.streams = plan.streams;
  P.qscale = softmax_scale * 1.4426950408889634f;  // log2(e)
  const int64_t rows = static_cast<int64_t>(plan.ctas) * 2 * hq;
  P.part_acc = scratch;
  P.part_ml = scratch + rows * hd;
  P.first = reinterpret_cast<int64_t*>(scratch + rows * (hd + 2));
  P.out = static_cast<__nv_bfloat16*>(out);
  P.page_div = FastDiv(static_cast<uint32_t>(page));
  return kv4::launch_decode(P, hd, plan, stream);
}

// 0, or the status a launch recorded (3 = a wait for a copy gave up); synchronizes.
extern "C" int kvbm_kv4_status(int reset) {
  int v = -1;
  if (cudaMemcpyFromSymbol(&v, kv4::g_kv4_status, sizeof(int)) != cudaSuccess) return -1;
  if (reset) {
    const int zero = 0;
    cudaMemcpyToSymbol(kv4::g_kv4_status, &zero, sizeof(int));
  }
  return v;
}
