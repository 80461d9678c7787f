// The 4-bit KV cache row, and what the kernels that write and read it share.
//
// One row holds the K or the V of one (token, KV head), HD = 64, 128 or 256
// elements in groups of 32 (NG = HD / 32):
//
//   bytes [0, HD/2)            codes c, 4 bits each
//   bytes [HD/2, HD/2 + 4 NG)  per group (scale s, zero z), bf16 each
//   padding to a multiple of 16 bytes: 48, 80 or 160 bytes a row
//
// and stands for z + s c. K keeps the code of element d in nibble d. V keeps
// the code of element 32 g + 4 b + i in nibble 4 (NG b + g) + i: the P V product
// wants, in one lane, the same few elements of every group of many tokens, and
// in this order those are HD/16 contiguous bytes.
//
// Quantising a bf16 group: z = min (a bf16 value, so exact), s = (max - min) / 15
// rounded UP to bf16 (so that z + 15 s reaches max), c = the code nearest to
// (x - z) / s, ties to even. The error is at most s / 2. A range below 15 x
// 2^-126 gives s = 0. A group that holds an infinity or a NaN gets s = NaN and
// reads back as NaN: a poisoned row shows instead of turning into numbers.
// A row costs 5 bits an element (6 with HD = 64's padding) where bf16 costs 16.
#pragma once

#include "common.cuh"

namespace kvbm {
namespace kv4 {

constexpr int kGroup = 32;

__host__ __device__ constexpr int row_bytes(int hd) { return (hd / 2 + hd / kGroup * 4 + 15) / 16 * 16; }

// Where a paged pool keeps its rows: pool[block][outer][token][head], byte strides.
struct Cache {
  uint8_t* base;
  int64_t block_stride, outer_stride, token_stride, head_stride;
  int page, num_blocks, heads;
};

__device__ __forceinline__ float bf_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf_hi(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}

// Quantises the 8 bf16 values `x` (packed pairs) of this lane; the 4 lanes that
// share lane / 4 hold one group. Returns the 8 codes (value k in nibble k) and
// the group's (scale | zero << 16).
//
// The code is the correctly rounded quotient (x - z) / s, then rint: bf16 inputs
// hit the midpoint between two codes exactly in about 1 of 500 elements, where a
// product with 1 / s would round either way. The quotient is Markstein's
// ("Computation of elementary functions on the IBM RISC System/6000", 1990):
// with y = 1 / s correctly rounded, q0 = a y, q = q0 + (a - q0 s) y in fused
// multiply-adds is a / s correctly rounded. Halves keep x - z from overflowing.
__device__ __forceinline__ uint32_t quantise8(const uint32_t (&x)[4], uint32_t* scale_zero) {
  float v[8];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    v[2 * k] = bf_lo(x[k]);
    v[2 * k + 1] = bf_hi(x[k]);
  }
  float lo = v[0], hi = v[0];
  bool bad = false;
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    lo = fminf(lo, v[k]);
    hi = fmaxf(hi, v[k]);
    bad |= (__float_as_uint(v[k]) & 0x7f800000u) == 0x7f800000u;
  }
  int flag = bad;
#pragma unroll
  for (int o = 1; o < 4; o <<= 1) {
    lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    flag |= __shfl_xor_sync(0xffffffffu, flag, o);
  }
  if (flag) {
    *scale_zero = 0x7fc0u;
    return 0u;
  }
  const float half_lo = 0.5f * lo;
  const float s = __fdiv_rn(fmaf(0.5f, hi, -half_lo), 7.5f);
  const uint32_t up = s < 1.17549435e-38f ? 0u : (__float_as_uint(s) + 0xffffu) & 0xffff0000u;
  *scale_zero = (up >> 16) | (__float_as_uint(lo) & 0xffff0000u);
  if (up == 0u) return 0u;
  const float half_s = 0.5f * __uint_as_float(up);
  const float y = __frcp_rn(half_s);
  uint32_t codes = 0u;
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const float a = fmaf(0.5f, v[k], -half_lo);
    const float q0 = a * y;
    const float q = fmaf(fmaf(-q0, half_s, a), y, q0);
    codes |= static_cast<uint32_t>(min(__float2int_rn(q), 15)) << (4 * k);
  }
  return codes;
}

// 8 codes (nibble k -> value k) of one group back to bf16 pairs, one rounding.
__device__ __forceinline__ int4 dequantise8(uint32_t codes, uint32_t scale_zero) {
  const float s = bf_lo(scale_zero), z = bf_hi(scale_zero);
  uint32_t o[4];
#pragma unroll
  for (int k = 0; k < 4; ++k)
    o[k] = pack2(fmaf(static_cast<float>((codes >> (8 * k)) & 15u), s, z),
                 fmaf(static_cast<float>((codes >> (8 * k + 4)) & 15u), s, z));
  return make_int4(o[0], o[1], o[2], o[3]);
}

// Lane l (0 .. HD/8) of a row holds elements [8 l, 8 l + 8): group l / 4. K: word
// l. V: two 16-bit pieces, b = 2 (l % 4) and the next.
template <int HD>
__device__ __forceinline__ void store_codes(uint8_t* row, int l, bool value, uint32_t codes) {
  constexpr int NG = HD / kGroup;
  if (!value) {
    reinterpret_cast<uint32_t*>(row)[l] = codes;
  } else {
    uint16_t* p = reinterpret_cast<uint16_t*>(row);
    const int b = 2 * (l & 3), g = l >> 2;
    p[NG * b + g] = static_cast<uint16_t>(codes);
    p[NG * (b + 1) + g] = static_cast<uint16_t>(codes >> 16);
  }
}
template <int HD>
__device__ __forceinline__ uint32_t load_codes(const uint8_t* row, int l, bool value) {
  constexpr int NG = HD / kGroup;
  if (!value) return reinterpret_cast<const uint32_t*>(row)[l];
  const uint16_t* p = reinterpret_cast<const uint16_t*>(row);
  const int b = 2 * (l & 3), g = l >> 2;
  return p[NG * b + g] | (static_cast<uint32_t>(p[NG * (b + 1) + g]) << 16);
}

}  // namespace kv4
}  // namespace kvbm
