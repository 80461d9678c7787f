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
  FastDiv page_div;
  // First byte of a slot's K row of head 0, or null outside the pool.
  __device__ __forceinline__ uint8_t* row(int64_t slot) const {
    if (slot < 0 || slot >= static_cast<int64_t>(num_blocks) * page) return nullptr;
    int64_t blk;
    if (slot < 0x7fffffff)
      blk = page_div.div(static_cast<uint32_t>(slot));
    else
      blk = slot / page;
    return base + blk * block_stride + (slot - blk * page) * token_stride;
  }
};

__device__ __forceinline__ float bf_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf_hi(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}

// Two fp32 in a register pair: Blackwell's packed fp32 arithmetic, two results an instruction.
using f32x2 = unsigned long long;
__device__ __forceinline__ f32x2 make2(float lo, float hi) {
  f32x2 d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(lo), "f"(hi));
  return d;
}
__device__ __forceinline__ void split2(f32x2 x, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(x));
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
  f32x2 d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
  f32x2 d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ f32x2 widen(uint32_t bf16x2) { return make2(bf_lo(bf16x2), bf_hi(bf16x2)); }
// NaN if either is.
__device__ __forceinline__ uint32_t min_bf16x2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
__device__ __forceinline__ uint32_t max_bf16x2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}

// Quantises the 8 bf16 values `x` (packed pairs) of this lane; the 4 lanes that
// share lane / 4 hold one group between them. Returns the 8 codes (value k in nibble k) and
// the group's (scale | zero << 16).
//
// The code is the quotient (x - z) / s rounded to an integer, and the quotient
// has to be right where it lies on the midpoint of two codes: bf16 inputs do so
// exactly in about 1 of 500 elements, and a product with 1 / s would fall either
// way. Two multiply-adds after Markstein ("Computation of elementary functions on
// the IBM RISC System/6000", 1990) see to it: q0 = a y with y near 1 / s, then
// q0 + (a - q0 s) y, whose error is the square of y's, so a quotient that fp32
// holds (a midpoint) comes out as it is, and any other lies 2^-9 from one. Halves
// keep x - z from overflowing.
__device__ __forceinline__ uint32_t quantise8(const uint32_t (&x)[4], uint32_t* scale_zero) {
  uint32_t lo = min_bf16x2(min_bf16x2(x[0], x[1]), min_bf16x2(x[2], x[3]));
  uint32_t hi = max_bf16x2(max_bf16x2(x[0], x[1]), max_bf16x2(x[2], x[3]));
  lo = min_bf16x2(lo, __byte_perm(lo, 0, 0x1032));
  hi = max_bf16x2(hi, __byte_perm(hi, 0, 0x1032));
  uint32_t range = __byte_perm(lo, hi, 0x5410);  // least | largest << 16
#pragma unroll
  for (int o = 1; o < 4; o <<= 1) {
    const uint32_t other = __shfl_xor_sync(0xffffffffu, range, o);
    range = __byte_perm(min_bf16x2(range, other), max_bf16x2(range, other), 0x7610);
  }
  if ((range & 0x7f80u) == 0x7f80u || (range & 0x7f800000u) == 0x7f800000u) {  // an infinity or a NaN among them
    *scale_zero = 0x7fc0u;
    return 0u;
  }
  const float half_lo = 0.5f * bf_lo(range);
  // by 7.5 in the same way; its reciprocal is a constant
  const float width = fmaf(0.5f, bf_hi(range), -half_lo);
  constexpr float kInv = 1.f / 7.5f;
  const float w0 = width * kInv;
  const float s = fmaf(fmaf(-w0, 7.5f, width), kInv, w0);
  const uint32_t up = s < 1.17549435e-38f ? 0u : (__float_as_uint(s) + 0xffffu) & 0xffff0000u;
  *scale_zero = (up >> 16) | (range << 16);
  if (up == 0u) return 0u;
  const float half_s = 0.5f * __uint_as_float(up);
  float y;
  asm("rcp.approx.f32 %0, %1;" : "=f"(y) : "f"(half_s));
  // q is at most 15 (s is not below range / 15 but by the rounding of one fp32 quotient). Adding 1.5 x 2^23 rounds
  // to an integer, ties to even; codes are put together as fp32 integers and converted four at a time, since
  // conversions are the slowest instructions here.
  const f32x2 half = make2(0.5f, 0.5f), lo2 = make2(-half_lo, -half_lo), y2 = make2(y, y);
  const f32x2 s2 = make2(-half_s, -half_s), round = make2(12582912.f, 12582912.f), back = make2(-12582912.f, -12582912.f);
  uint32_t packed[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    float c[4];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const f32x2 a = fma2(half, widen(x[2 * k + j]), lo2);
      const f32x2 q0 = mul2(a, y2);
      split2(add2(add2(fma2(fma2(q0, s2, a), y2, q0), round), back), c[2 * j], c[2 * j + 1]);
    }
    packed[k] = static_cast<uint32_t>(fmaf(fmaf(fmaf(c[3], 16.f, c[2]), 16.f, c[1]), 16.f, c[0]));
  }
  return packed[0] | (packed[1] << 16);
}

// 8 codes (nibble k -> value k) of one group back to bf16. A code or'ed into 0x4300 is the bf16 128 + c; z + s c is
// one bf16 fused multiply-add, rounded once.
__device__ __forceinline__ int4 dequantise8(uint32_t codes, uint32_t scale_zero) {
  const uint32_t s2 = __byte_perm(scale_zero, 0, 0x1010), z2 = __byte_perm(scale_zero, 0, 0x3232);
  uint32_t r[4];  // elements k and k + 4
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const uint32_t c = ((codes >> (4 * k)) & 0x000f000fu) | 0x43004300u;
    asm("{\n\t.reg .b32 t;\n\t"
        "sub.rn.bf16x2 t, %1, %2;\n\t"
        "fma.rn.bf16x2 %0, t, %3, %4;\n\t}"
        : "=r"(r[k])
        : "r"(c), "r"(0x43004300u), "r"(s2), "r"(z2));
  }
  return make_int4(__byte_perm(r[0], r[1], 0x5410), __byte_perm(r[2], r[3], 0x5410), __byte_perm(r[0], r[1], 0x7632),
                   __byte_perm(r[2], r[3], 0x7632));
}

// Unit u (0 .. HD/8) of a row is elements [8 u, 8 u + 8), of group u / 4. K: word u. V: two 16-bit pieces,
// b = 2 (u % 4) and the next.
template <int HD>
__device__ __forceinline__ void store_codes(uint8_t* row, int u, bool value, uint32_t codes) {
  constexpr int NG = HD / kGroup;
  if (!value) {
    reinterpret_cast<uint32_t*>(row)[u] = codes;
  } else {
    uint16_t* p = reinterpret_cast<uint16_t*>(row) + 2 * NG * (u & 3) + (u >> 2);
    p[0] = static_cast<uint16_t>(codes);
    p[NG] = static_cast<uint16_t>(codes >> 16);
  }
}
template <int HD>
__device__ __forceinline__ uint32_t load_codes(const uint8_t* row, int u, bool value) {
  constexpr int NG = HD / kGroup;
  if (!value) return reinterpret_cast<const uint32_t*>(row)[u];
  const uint16_t* p = reinterpret_cast<const uint16_t*>(row) + 2 * NG * (u & 3) + (u >> 2);
  return p[0] | (static_cast<uint32_t>(p[NG]) << 16);
}

}  // namespace kv4
}  // namespace kvbm
