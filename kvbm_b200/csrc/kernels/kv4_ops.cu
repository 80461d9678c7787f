// Operators of the 4-bit paged KV cache (row format: kv4_format.cuh): head norms
// + RoPE + cache write, rows back to bf16, decode attention.
#include "common.cuh"
#include "kv4_format.cuh"
#include "kvbm_kernels.h"
#include "paged_decode_kv4.cuh"

#include <algorithm>
#include <atomic>
#include <cstring>
#include <mutex>

using namespace kvbm;
using kvbm::kv4::Cache;
using kvbm::kv4::f32x2;

namespace {

constexpr int kWriteThreads = 64;  // small blocks: their warps' places are taken up again sooner
constexpr int kReadThreads = 128;

// ---------------------------------------------------------------------------
// q/k head norms + RoPE + paged cache write, one pass over a packed qkv.
//
//   y = w x / sqrt(mean(x^2) + eps)          (left out without a weight)
//   out[i] = y[i] cos - y[i + R/2] sin, out[i + R/2] = y[i + R/2] cos + y[i] sin,  i < R/2; the rest as it is
//
// all in fp32 and rounded to bf16 once. The cache takes that bf16 k and the bf16
// v, so quantising a 16-bit cache that this kernel has written gives the same codes.
// (The 16-bit write of models without head norms, rope_kv_write, fuses a product and
// a sum of the rotation: its k may be a bf16 step away, and a code with it.)
//
// A row of HD elements is held by HD/16 lanes, each with 8 elements of the first
// half and the 8 that lie HD/2 behind them, so with rot = HD both elements of a
// rotation are in one lane (with a smaller rot the other comes by shuffle), and
// a warp takes 512 / HD rows a step. Every product is rounded to fp32 by itself in
// the order of the formula, and the squares are summed in the order in which PyTorch's
// reductions sum a row (sum_squares). Nothing else in this library computes k so: it
// makes k, and the codes, the same bit for bit as the formula's operations one after
// another, which is how they are checked, where one fp32 step moves a code that lies
// next to a border by a fifteenth of its group's range (folding w into cos and sin,
// two of five products less an element, moved 4 codes in a chunk of 8,192 tokens).
// What bounds it is HBM for a prefill (the rows go in and out once), nearly
// matched by the instructions of the norm, the rotation and the quantising (250 a
// step; at the HBM rate an SM issues 340): hence the packed arithmetic, and copies
// of three steps in flight. For a decode step it is the latency of one token, so
// there a token's rows are spread over warps. Rows are taken by kind (q, k, v),
// which keeps branches uniform. Measured at 32 + 16 heads of 128, 4 bits: 8,192
// tokens, 195 MB, 38.0 us = 5.1 TB/s (a plain copy of as many bytes: 32 us); 32
// tokens 2.6 us.
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
  int steps_q, steps_kv, steps_item;  // steps of a token's q rows, of its k (v) rows, of one warp
  FastDiv items_div;                  // divides by the items of a token
  __nv_bfloat16* q_out;
  __nv_bfloat16* k_out;
  f32x2 one, minus_one;  // pairs of them
  bool release;          // let the next kernel be put in place beside this one
};

__device__ __forceinline__ void words(uint32_t (&x)[4], int4 v) { x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w; }
// A unit's 8 bf16 values in fp32, elements k and k + 4 a pair, and back.
__device__ __forceinline__ void widen8(f32x2 (&y)[4], const uint32_t (&x)[4]) {
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    y[2 * k] = kv4::make2(kv4::bf_lo(x[k]), kv4::bf_lo(x[k + 2]));
    y[2 * k + 1] = kv4::make2(kv4::bf_hi(x[k]), kv4::bf_hi(x[k + 2]));
  }
}
__device__ __forceinline__ void narrow8(uint32_t (&x)[4], const f32x2 (&y)[4]) {
  float lo[4], hi[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) kv4::split2(y[k], lo[k], hi[k]);
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    x[k] = kv4::pack2(lo[2 * k], lo[2 * k + 1]);
    x[k + 2] = kv4::pack2(hi[2 * k], hi[2 * k + 1]);
  }
}

enum Kind { kQ, kK, kV };

// Sum of the squares of a row's HD values; this lane has units l and l + HD/16. The order: at 256, the two halves of
// the row are added element by element first; at 128 and 256, each four neighbours one after another; then the upper
// half of what is left is added to the lower half until one value is left. Squares of bf16 values are exact in fp32,
// so a fused multiply-add is a rounded sum of squares.
template <int HD>
__device__ __forceinline__ float sum_squares(const f32x2 (&a)[4], const f32x2 (&b)[4]) {
  f32x2 h[4];
  constexpr int kLeft = HD == 64 ? 4 : 1;  // pairs a lane has left before lanes are added
  if constexpr (HD == 128) {
    f32x2 qb = kv4::mul2(b[0], b[0]);
    h[0] = kv4::mul2(a[0], a[0]);
#pragma unroll
    for (int k = 1; k < 4; ++k) {
      h[0] = kv4::fma2(a[k], a[k], h[0]);
      qb = kv4::fma2(b[k], b[k], qb);
    }
    h[0] = kv4::add2(h[0], qb);
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) h[k] = kv4::fma2(b[k], b[k], kv4::mul2(a[k], a[k]));
    if constexpr (HD == 256) h[0] = kv4::add2(kv4::add2(kv4::add2(h[0], h[1]), h[2]), h[3]);
  }
#pragma unroll
  for (int o = HD / 32; o > 0; o >>= 1)
#pragma unroll
    for (int k = 0; k < kLeft; ++k) {
      float lo, hi;
      kv4::split2(h[k], lo, hi);
      h[k] = kv4::add2(h[k], kv4::make2(__shfl_xor_sync(0xffffffffu, lo, o), __shfl_xor_sync(0xffffffffu, hi, o)));
    }
  float s[kLeft];
#pragma unroll
  for (int k = 0; k < kLeft; ++k) {
    float lo, hi;
    kv4::split2(h[k], lo, hi);
    s[k] = lo + hi;
  }
#pragma unroll
  for (int n = kLeft / 2; n > 0; n >>= 1)
#pragma unroll
    for (int k = 0; k < n; ++k) s[k] += s[k + n];
  return s[0];
}

// Where a warp's steps find their rows: copies of the next kRing - 1 steps are in flight, across the borders of the
// kinds too. A lane reads what it copied itself.
constexpr int kRing = 4;
struct Rows {
  const WriteParams& P;
  const __nv_bfloat16* token;
  int4* ring;  // this lane's first piece; [kRing][2][32]
  int end;
  template <int HD>
  __device__ __forceinline__ void load(int step) const {
    constexpr int L = HD / 16, R = 32 / L;
    const int lane = threadIdx.x & 31, l = lane % L, r = lane / L;
    if (step < end) {
      int first = 0, rows = P.hq, at = step;
      if (at >= P.steps_q) {
        at -= P.steps_q, first = P.hq, rows = P.hkv;
        if (at >= P.steps_kv) at -= P.steps_kv, first += P.hkv;
      }
      const int h = at * R + r;
      if (h < rows) {
        const __nv_bfloat16* src = token + static_cast<int64_t>(first + h) * HD + 8 * l;
        int4* dst = ring + (step % kRing) * 64;
        kv4::copy16(smem_u32(dst), src);
        kv4::copy16(smem_u32(dst + 32), src + HD / 2);
      }
    }
    kv4::copy_commit();
  }
  template <int HD>
  __device__ __forceinline__ void take(int step, uint32_t (&x)[2][4]) const {
    load<HD>(step + kRing - 1);
    kv4::copy_wait<kRing - 1>();
    words(x[0], ring[(step % kRing) * 64]);
    words(x[1], ring[(step % kRing) * 64 + 32]);
  }
};

template <int HD, bool KV4, bool FULL, Kind KIND>
__device__ __forceinline__ void write_rows(const WriteParams& P, const Rows& from, int64_t t, int first, int begin,
                                           int end, int32_t pos, uint8_t* cache_row) {
  constexpr int L = HD / 16, R = 32 / L;  // lanes a row, rows a step
  const int lane = threadIdx.x & 31, l = lane % L, r = lane / L;
  const int rows = KIND == kQ ? P.hq : P.hkv;

  // With y = x / rms w and, for unit i of this lane, y' the unit `other[i]` of the row: out = y cs[i] + y' sn[i]. With
  // all elements rotated the other unit is the lane's own, and cos and sin are the same for both: out[0] = y[0] cs[0]
  // - y[1] sn[0], out[1] = y[1] cs[0] + y[0] sn[0].
  constexpr int U = FULL ? 1 : 2;
  f32x2 cs[U][4], sn[U][4];
  uint32_t wt[2][4], wt_other[2][4];  // bf16 pairs
  int other[2];
  bool turned[2];
  const __nv_bfloat16* w = KIND == kQ ? P.q_weight : P.k_weight;
  if constexpr (KIND != kV) {
    const int half = FULL ? L : P.rot / 16;  // units that hold one half of the rotated elements
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int u = l + i * L;
      other[i] = u < half ? u + half : u < 2 * half ? u - half : u;
      turned[i] = u < 2 * half;
      if (i < U) {
#pragma unroll
        for (int k = 0; k < 4; ++k) cs[i][k] = sn[i][k] = 0;
        if (FULL || turned[i]) {
          const float* at = P.cos_sin + static_cast<int64_t>(pos) * (FULL ? HD : P.rot) + (u < half ? u : u - half) * 8;
          const float sign = FULL || u >= half ? 1.f : -1.f;
          const float4 a = reinterpret_cast<const float4*>(at)[0], b = reinterpret_cast<const float4*>(at)[1];
          const float4 c = reinterpret_cast<const float4*>(at + 8 * half)[0], d = reinterpret_cast<const float4*>(at + 8 * half)[1];
          cs[i][0] = kv4::make2(a.x, b.x), cs[i][1] = kv4::make2(a.y, b.y);
          cs[i][2] = kv4::make2(a.z, b.z), cs[i][3] = kv4::make2(a.w, b.w);
          sn[i][0] = kv4::make2(sign * c.x, sign * d.x), sn[i][1] = kv4::make2(sign * c.y, sign * d.y);
          sn[i][2] = kv4::make2(sign * c.z, sign * d.z), sn[i][3] = kv4::make2(sign * c.w, sign * d.w);
        }
      }
      if (w != nullptr) {
        words(wt[i], reinterpret_cast<const int4*>(w)[u]);
        if constexpr (!FULL) words(wt_other[i], reinterpret_cast<const int4*>(w)[other[i]]);
      }
    }
  }
  for (int step = begin; step < end; ++step) {
    const int h = step * R + r;
    uint32_t x[2][4];
    from.take<HD>(first + step, x);
    if constexpr (KIND != kV) {
      f32x2 y[2][4], p[2][4];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        widen8(y[i], x[i]);
        if constexpr (!FULL) {  // the other unit lies in lane other % L, as its first or its second
          uint32_t theirs[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint32_t a = __shfl_sync(0xffffffffu, x[0][k], other[i] % L, L);
            const uint32_t b = __shfl_sync(0xffffffffu, x[1][k], other[i] % L, L);
            theirs[k] = other[i] < L ? a : b;
          }
          widen8(p[i], theirs);
        }
      }
      if (w != nullptr) {
        const float inv = rsqrtf(fmaf(sum_squares<HD>(y[0], y[1]), 1.f / HD, P.eps));
        const f32x2 inv2 = kv4::make2(inv, inv);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          f32x2 wide[4];
          widen8(wide, wt[i]);
#pragma unroll
          for (int k = 0; k < 4; ++k) y[i][k] = kv4::mul2(kv4::mul2(y[i][k], inv2), wide[k]);
          if constexpr (!FULL) {
            widen8(wide, wt_other[i]);
#pragma unroll
            for (int k = 0; k < 4; ++k) p[i][k] = kv4::mul2(kv4::mul2(p[i][k], inv2), wide[k]);
          }
        }
      }
      // Products are added by an fma with a factor of one that the compiler does not know: it would fuse a packed
      // product and a packed sum.
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if constexpr (FULL) {
          const f32x2 a = y[0][k], b = y[1][k];
          y[0][k] = kv4::fma2(kv4::mul2(b, sn[0][k]), P.minus_one, kv4::mul2(a, cs[0][k]));
          y[1][k] = kv4::fma2(kv4::mul2(a, sn[0][k]), P.one, kv4::mul2(b, cs[0][k]));
        } else {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const f32x2 o = kv4::fma2(kv4::mul2(p[i][k], sn[i][k]), P.one, kv4::mul2(y[i][k], cs[i][k]));
            y[i][k] = turned[i] ? o : y[i][k];
          }
        }
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) narrow8(x[i], y[i]);
      __nv_bfloat16* dst = nullptr;
      if (P.q_out == nullptr)
        dst = P.qkv + t * P.qkv_stride + static_cast<int64_t>((KIND == kQ ? 0 : P.hq) + h) * HD + 8 * l;
      else if (KIND == kQ)
        dst = P.q_out + (t * P.hq + h) * HD + 8 * l;
      else if (P.k_out != nullptr)
        dst = P.k_out + (t * P.hkv + h) * HD + 8 * l;
      if (dst != nullptr && h < rows) {
        *reinterpret_cast<int4*>(dst) = make_int4(x[0][0], x[0][1], x[0][2], x[0][3]);
        *reinterpret_cast<int4*>(dst + HD / 2) = make_int4(x[1][0], x[1][1], x[1][2], x[1][3]);
      }
    }
    if constexpr (KIND != kQ) {
      if (cache_row != nullptr) {  // the whole warp's: one token
        uint8_t* dst = cache_row + (KIND == kV ? P.cache.outer_stride : 0) + h * P.cache.head_stride;
        if constexpr (KV4) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            uint32_t scale_zero;
            const uint32_t codes = kv4::quantise8(x[i], &scale_zero);
            if (h < rows) {
              kv4::store_codes<HD>(dst, l + i * L, KIND == kV, codes);
              if ((l & 3) == 0) reinterpret_cast<uint32_t*>(dst + HD / 2)[(l + i * L) >> 2] = scale_zero;
            }
          }
          constexpr int kUsed = HD / 2 + HD / 8;
          if constexpr (kUsed < kv4::row_bytes(HD))
            if (h < rows && l < (kv4::row_bytes(HD) - kUsed) / 4) reinterpret_cast<uint32_t*>(dst + kUsed)[l] = 0u;
        } else if (h < rows) {
          reinterpret_cast<int4*>(dst)[l] = make_int4(x[0][0], x[0][1], x[0][2], x[0][3]);
          reinterpret_cast<int4*>(dst)[l + L] = make_int4(x[1][0], x[1][1], x[1][2], x[1][3]);
        }
      }
    }
  }
}

// Warps an SM holds: registers are for so many (80 and 128 a thread).
constexpr int write_warps_sm(bool full) { return full ? 24 : 16; }

template <int HD, bool KV4, bool FULL>
__global__ void __launch_bounds__(kWriteThreads, write_warps_sm(FULL) * 32 / kWriteThreads)
    qk_norm_rope_kv_write_kernel(const __grid_constant__ WriteParams P) {
  __shared__ int4 ring[kWriteThreads / 32][kRing * 2 * 32];
  const int64_t item = static_cast<int64_t>(blockIdx.x) * (kWriteThreads / 32) + (threadIdx.x >> 5);
  kv4::wait_before();
  if (P.release) kv4::release_next();
  if (item >= P.tokens * P.items_div.d) return;
  const int64_t t = P.items_div.div(static_cast<uint32_t>(item));
  const int begin = static_cast<int>(item - t * P.items_div.d) * P.steps_item;
  const int k0 = P.steps_q, v0 = k0 + P.steps_kv, end = min(begin + P.steps_item, v0 + P.steps_kv);
  const Rows from{P, P.qkv + t * P.qkv_stride, ring[threadIdx.x >> 5] + (threadIdx.x & 31), end};
#pragma unroll
  for (int i = 0; i < kRing - 1; ++i) from.load<HD>(begin + i);
  const int32_t pos = P.positions[t];
  if (pos >= 0 && pos < P.max_pos) {  // a token outside the table is left alone
    uint8_t* cache_row = nullptr;
    if (end > k0) cache_row = P.cache.row(P.slots[t]);
    if (begin < k0) write_rows<HD, KV4, FULL, kQ>(P, from, t, 0, begin, min(end, k0), pos, nullptr);
    if (begin < v0 && end > k0)
      write_rows<HD, KV4, FULL, kK>(P, from, t, k0, max(begin, k0) - k0, min(end, v0) - k0, pos, cache_row);
    if (end > v0) write_rows<HD, KV4, FULL, kV>(P, from, t, v0, max(begin, v0) - v0, end - v0, pos, cache_row);
  }
  kv4::copy_wait<0>();
}

// ---------------------------------------------------------------------------
// Rows of the cache back to bf16: k_out[t][h] / v_out[t][h] = z + s c of slot
// slots[t] (zeros for a slot outside the pool). HBM bounds it, 5 bits an element
// in and 16 out: lanes hold rows as in the write, and a warp has kReadFly steps of
// 512 / HD rows in flight. Measured at 8 heads of 128: 16,384 tokens, 88 MB, 14.0
// us = 6.3 TB/s; 77 tokens 1.7 us.
// ---------------------------------------------------------------------------
constexpr int kReadFly = 2;
struct GatherParams {
  Cache cache;
  const int64_t* slots;
  int64_t tokens;
  FastDiv items_div;  // divides by the items of a token: groups of kReadFly steps of its K rows, then of its V rows
  __nv_bfloat16* k_out;
  __nv_bfloat16* v_out;
};

template <int HD>
__global__ void __launch_bounds__(kReadThreads) kv4_gather_kernel(const __grid_constant__ GatherParams P) {
  constexpr int L = HD / 16, R = 32 / L;
  const int lane = threadIdx.x & 31, l = lane % L, r = lane / L;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * (kReadThreads / 32) + (threadIdx.x >> 5);
  kv4::wait_before();
  if (item >= P.tokens * P.items_div.d) return;
  const int64_t t = P.items_div.div(static_cast<uint32_t>(item));
  int group = static_cast<int>(item - t * P.items_div.d);
  const bool value = group >= static_cast<int>(P.items_div.d / 2);
  if (value) group -= P.items_div.d / 2;
  const uint8_t* row = P.cache.row(P.slots[t]);
  __nv_bfloat16* out = (value ? P.v_out : P.k_out) + t * P.cache.heads * HD;
  uint32_t codes[kReadFly][2], par[kReadFly][2];
#pragma unroll
  for (int u = 0; u < kReadFly; ++u) {
    const int h = (group * kReadFly + u) * R + r;
#pragma unroll
    for (int i = 0; i < 2; ++i) codes[u][i] = par[u][i] = 0u;
    if (row != nullptr && h < P.cache.heads) {
      const uint8_t* src = row + (value ? P.cache.outer_stride : 0) + h * P.cache.head_stride;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        codes[u][i] = kv4::load_codes<HD>(src, l + i * L, value);
        par[u][i] = reinterpret_cast<const uint32_t*>(src + HD / 2)[(l + i * L) >> 2];
      }
    }
  }
#pragma unroll
  for (int u = 0; u < kReadFly; ++u) {
    const int h = (group * kReadFly + u) * R + r;
    if (h < P.cache.heads) {
#pragma unroll
      for (int i = 0; i < 2; ++i)
        reinterpret_cast<int4*>(out + h * HD)[l + i * L] = kv4::dequantise8(codes[u][i], par[u][i]);
    }
  }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

bool cache_ok(const Cache& c) {
  return (c.base != nullptr || c.num_blocks == 0) && aligned16(c.base) && c.block_stride % 16 == 0 && c.outer_stride % 16 == 0 &&
         c.token_stride % 16 == 0 && c.head_stride % 16 == 0 && c.page > 0 && c.num_blocks >= 0 && c.heads > 0;
}

// One status word a device in mapped host memory: the host reads it without waiting for the device.
constexpr int kMaxDevices = 64;
std::mutex g_status_lock;
std::atomic<int*> g_status_host{nullptr};
std::atomic<uint64_t> g_wait_ns{kv4::kWaitNs};

int* status_word() {
  int* host = g_status_host;
  if (host == nullptr) {
    std::lock_guard<std::mutex> lock(g_status_lock);
    host = g_status_host;
    if (host == nullptr) {
      cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;  // the first call may be one that is captured
      cudaThreadExchangeStreamCaptureMode(&mode);
      void* p = nullptr;
      const cudaError_t e = cudaHostAlloc(&p, sizeof(int) * kMaxDevices, cudaHostAllocMapped | cudaHostAllocPortable);
      cudaThreadExchangeStreamCaptureMode(&mode);
      if (e != cudaSuccess) return nullptr;
      host = static_cast<int*>(p);
      std::memset(host, 0, sizeof(int) * kMaxDevices);
      g_status_host = host;
    }
  }
  int dev = 0;
  void* d = nullptr;
  if (cudaGetDevice(&dev) != cudaSuccess || dev >= kMaxDevices ||
      cudaHostGetDevicePointer(&d, host + dev, 0) != cudaSuccess)
    return nullptr;
  return static_cast<int*>(d);
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
  P.cache = Cache{static_cast<uint8_t*>(kv), block_stride, outer_stride, token_stride, head_stride, page, num_blocks, hkv,
                  FastDiv(static_cast<uint32_t>(page > 0 ? page : 1))};
  if (tokens < 0 || hq < 0 || !cache_ok(P.cache) || !qkv || !positions || !cos_sin || !slots || !aligned16(qkv) ||
      (tokens > 1 && qkv_stride % 8 != 0) || !aligned16(cos_sin) || !aligned16(q_out) || !aligned16(k_out) || !aligned16(q_weight) ||
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
  P.one = 0x3f8000003f800000ull;
  P.minus_one = 0xbf800000bf800000ull;
  P.q_out = static_cast<__nv_bfloat16*>(q_out);
  P.k_out = static_cast<__nv_bfloat16*>(k_out);
  if (hd != 64 && hd != 128 && hd != 256) return cudaErrorInvalidValue;
  const int rows_step = 512 / hd;
  P.steps_q = (hq + rows_step - 1) / rows_step;
  P.steps_kv = (hkv + rows_step - 1) / rows_step;
  // A token's rows are spread over as many warps as find a place at the same time, and a warp has the whole token if
  // tokens alone take all places (2,048 tokens of 32 + 16 heads of 128: whole tokens 13.6 us, two warps a token, of
  // which the last ones wait for a place, 16.0; 512 tokens: six warps a token 5.1, four 5.6).
  const int steps = P.steps_q + 2 * P.steps_kv;
  const int64_t places = static_cast<int64_t>(kvbm_sm_count()) * write_warps_sm(rot == hd);
  const int64_t items = std::clamp<int64_t>(places / tokens, 1, steps);
  P.steps_item = static_cast<int>((steps + items - 1) / items);
  P.items_div = FastDiv(static_cast<uint32_t>((steps + P.steps_item - 1) / P.steps_item));
  const int64_t warps = tokens * P.items_div.d;
  if (warps > 0x7fffffff) return cudaErrorInvalidValue;
  // The next kernel (a decode step's attention) is let in early only where this one leaves most places free: 3 us a
  // layer of a decode step of 32 requests; filling the places beside 200 tokens' 2,400 warps cost 0.3 us, since the
  // blocks that found none were placed unevenly.
  P.release = warps * 4 <= places;
  const unsigned grid = static_cast<unsigned>((warps + kWriteThreads / 32 - 1) / (kWriteThreads / 32));
#define KVBM_WRITE(HD, KV4, FULL) \
  kv4::launch_overlapped(qk_norm_rope_kv_write_kernel<HD, KV4, FULL>, dim3(grid), kWriteThreads, 0, stream, P)
#define KVBM_WRITE_HD(HD)                                                                    \
  case HD:                                                                                   \
    return bits == 4 ? (rot == HD ? KVBM_WRITE(HD, true, true) : KVBM_WRITE(HD, true, false)) \
                     : (rot == HD ? KVBM_WRITE(HD, false, true) : KVBM_WRITE(HD, false, false));
  switch (hd) {
    KVBM_WRITE_HD(64)
    KVBM_WRITE_HD(128)
    KVBM_WRITE_HD(256)
    default: return cudaErrorInvalidValue;
  }
#undef KVBM_WRITE_HD
#undef KVBM_WRITE
}

extern "C" int kvbm_kv4_gather(const void* kv, int64_t block_stride, int64_t outer_stride, int64_t token_stride,
                               int64_t head_stride, int page, int num_blocks, int heads, int hd, const int64_t* slots,
                               int64_t tokens, void* k_out, void* v_out, cudaStream_t stream) {
  if (tokens == 0) return cudaSuccess;
  GatherParams P{};
  P.cache = Cache{static_cast<uint8_t*>(const_cast<void*>(kv)), block_stride, outer_stride, token_stride, head_stride,
                  page, num_blocks, heads, FastDiv(static_cast<uint32_t>(page > 0 ? page : 1))};
  if (tokens < 0 || !cache_ok(P.cache) || !slots || !k_out || !v_out || !aligned16(k_out) || !aligned16(v_out))
    return cudaErrorInvalidValue;
  P.slots = slots;
  P.tokens = tokens;
  P.k_out = static_cast<__nv_bfloat16*>(k_out);
  P.v_out = static_cast<__nv_bfloat16*>(v_out);
  if (hd != 64 && hd != 128 && hd != 256) return cudaErrorInvalidValue;
  const int steps = (heads * (hd / 16) + 31) / 32;  // of a token's K (V) rows
  P.items_div = FastDiv(2 * static_cast<uint32_t>((steps + kReadFly - 1) / kReadFly));
  const int64_t warps = tokens * P.items_div.d;
  if (warps > 0x7fffffff) return cudaErrorInvalidValue;
  const unsigned grid = static_cast<unsigned>((warps + kReadThreads / 32 - 1) / (kReadThreads / 32));
  switch (hd) {
    case 64: return kv4::launch_overlapped(kv4_gather_kernel<64>, dim3(grid), kReadThreads, 0, stream, P);
    case 128: return kv4::launch_overlapped(kv4_gather_kernel<128>, dim3(grid), kReadThreads, 0, stream, P);
    case 256: return kv4::launch_overlapped(kv4_gather_kernel<256>, dim3(grid), kReadThreads, 0, stream, P);
    default: return cudaErrorInvalidValue;
  }
}

// How a launch of the decode attention is laid out: out[0] floats of scratch, out[1]
// CTAs along the work. `ctas` 0: one for each the GPU holds at a time.
extern "C" int kvbm_paged_decode_attn_kv4_plan(int batch, int hq, int hkv, int hd, int64_t max_tokens, int ctas,
                                               int sm_count, int64_t* out) {
  if (!out || batch <= 0 || hkv <= 0 || hq <= 0 || hq % hkv != 0 || max_tokens < 0 || ctas < 0 || sm_count <= 0)
    return cudaErrorInvalidValue;
  const kv4::Plan p = kv4::plan_decode(batch, hq, hkv, hd, max_tokens, ctas, sm_count);
  out[0] = p.cut ? static_cast<int64_t>(p.ctas) * 2 * hq * (hd + 2) + 2 * static_cast<int64_t>(batch) : 0;
  out[1] = p.ctas;
  return cudaSuccess;
}

// `scratch`: 16-byte aligned floats as the plan says, null for none.
extern "C" int kvbm_paged_decode_attn_kv4(const void* q, int64_t q_stride, const void* kv, int64_t block_stride,
                                          int64_t outer_stride, int64_t token_stride, int64_t head_stride, int page,
                                          int num_blocks, const int32_t* block_table, int64_t table_stride,
                                          int max_blocks, const int32_t* seq_lens, int batch, int hq, int hkv, int hd,
                                          float softmax_scale, int ctas, int sm_count, float* scratch, void* out,
                                          cudaStream_t stream) {
  if (batch == 0) return cudaSuccess;
  kv4::AttnParams P{};
  P.cache = Cache{static_cast<uint8_t*>(const_cast<void*>(kv)), block_stride, outer_stride, token_stride, head_stride,
                  page, num_blocks, hkv, FastDiv(static_cast<uint32_t>(page > 0 ? page : 1))};
  if (batch < 0 || batch > 65535 || hkv <= 0 || hq <= 0 || hq % hkv != 0 || !cache_ok(P.cache) || !q || !aligned16(q) ||
      (batch > 1 && q_stride % 8 != 0) || !out || !aligned16(out) || !seq_lens || max_blocks < 0 || (max_blocks > 0 && !block_table) ||
      ctas < 0 || sm_count <= 0 || !aligned16(scratch))
    return cudaErrorInvalidValue;
  const kv4::Plan plan =
      kv4::plan_decode(batch, hq, hkv, hd, static_cast<int64_t>(max_blocks) * page, ctas, sm_count);
  if (plan.y_ctas > 65535 || static_cast<int64_t>(batch) * hq > 0x7fffffff || (plan.cut && !scratch)) return cudaErrorInvalidValue;
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
  if (plan.cut) {
    P.part_acc = scratch;
    P.part_ml = scratch + rows * hd;
    P.parts = reinterpret_cast<int2*>(scratch + rows * (hd + 2));
  }
  P.out = static_cast<__nv_bfloat16*>(out);
  P.status = status_word();
  P.wait_ns = g_wait_ns;
  if (P.status == nullptr) return cudaErrorMemoryAllocation;
  return kv4::launch_decode(P, hd, plan, stream);
}

extern "C" int kvbm_kv4_status(int device, int reset) {
  if (device < 0 || device >= kMaxDevices || g_status_host == nullptr) return 0;
  volatile int* word = g_status_host + device;
  const int v = *word;
  if (reset) *word = 0;
  return v;
}

extern "C" void kvbm_kv4_set_wait_limit_ns(int64_t ns) { g_wait_ns = ns < 0 ? kv4::kWaitNs : static_cast<uint64_t>(ns); }
