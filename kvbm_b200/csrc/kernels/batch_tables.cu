// Block tables, positions and cache slots of a batch, from its request lengths.
//
// Request b brings q = query_lens[b] new tokens behind c = context_lens[b] cached
// ones and owns n = block_counts[b] (or ceil((c + q) / page)) blocks, listed one
// request after another in block_ids:
//
//   cu[b] = sum of q before b,  first[b] = sum of n before b
//   table[b][j] = block_ids[first[b] + j] for j < n, else the pad value
//   token cu[b] + i: position c + i, slot = table[b][(c + i) / page] * page + (c + i) % page
//
// The bound is latency: one launch in place of a dozen small ones. Every CTA
// scans all lengths itself in shared memory (256 requests: one each thread, two
// barriers), because a CTA that waited for another's scan would wait longer than
// the scan takes; then rows and tokens are spread over the grid, and a token
// finds its request by bisection in the scanned sums. Measured: 256 requests with
// 8,192 tokens and rows of 1,024 blocks 4.0 us, 4 with 64 tokens 2.6 us; slots of
// 32 tokens from a table 1.4 us.
#include "common.cuh"
#include "kvbm_kernels.h"

#include <algorithm>

using namespace kvbm;

namespace {

constexpr int kThreads = 256;
constexpr int kMaxBatch = 8192;  // two 64-bit sums a request in shared memory: 128 KiB

struct TablesParams {
  const int32_t* query_lens;
  const int32_t* context_lens;
  const int32_t* block_counts;
  const int32_t* block_ids;
  int64_t num_ids, tokens;
  int batch, max_blocks, pad, num_rows;
  int32_t* table;
  int64_t table_stride;
  const int32_t* rows;
  int32_t* seq_lens;
  int32_t* cu_query;
  int32_t* positions;
  int64_t* slots;
  int page;
  FastDiv page_div;
};

__device__ __forceinline__ int64_t blocks_of(const TablesParams& P, int b, int64_t seq) {
  if (P.block_counts != nullptr) return max(P.block_counts[b], 0);
  return (seq + P.page - 1) / P.page;
}

__global__ void __launch_bounds__(kThreads) batch_tables_kernel(const __grid_constant__ TablesParams P) {
  extern __shared__ int64_t sums[];
  int64_t* cu = sums;                      // [batch + 1]
  int64_t* first = sums + P.batch + 1;     // [batch + 1]
  __shared__ int64_t warp_q[kThreads / 32], warp_n[kThreads / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

  // ---- scan: thread t owns `per` consecutive requests
  const int per = (P.batch + kThreads - 1) / kThreads;
  const int b0 = min(P.batch, tid * per), b1 = min(P.batch, b0 + per);
  int64_t q_sum = 0, n_sum = 0;
  for (int b = b0; b < b1; ++b) {
    const int64_t q = max(P.query_lens[b], 0), seq = q + max(P.context_lens[b], 0);
    q_sum += q;
    n_sum += blocks_of(P, b, seq);
    if (blockIdx.x == 0 && P.seq_lens != nullptr)
      P.seq_lens[b] = static_cast<int32_t>(seq < 0x7fffffff ? seq : 0x7fffffff);
  }
  int64_t q_run = q_sum, n_run = n_sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t q = __shfl_up_sync(0xffffffffu, q_run, o), n = __shfl_up_sync(0xffffffffu, n_run, o);
    if (lane >= o) {
      q_run += q;
      n_run += n;
    }
  }
  if (lane == 31) {
    warp_q[warp] = q_run;
    warp_n[warp] = n_run;
  }
  __syncthreads();
  int64_t q_at = q_run - q_sum, n_at = n_run - n_sum;
  for (int w = 0; w < warp; ++w) {
    q_at += warp_q[w];
    n_at += warp_n[w];
  }
  for (int b = b0; b < b1; ++b) {
    cu[b] = q_at;
    first[b] = n_at;
    const int64_t q = max(P.query_lens[b], 0);
    q_at += q;
    n_at += blocks_of(P, b, q + max(P.context_lens[b], 0));
  }
  if (b1 == P.batch && (b0 < b1 || (P.batch == 0 && tid == 0))) {  // whoever owns the last request closes the sums
    cu[P.batch] = q_at;
    first[P.batch] = n_at;
  }
  __syncthreads();
  if (blockIdx.x == 0)
    for (int b = tid; b <= P.batch; b += kThreads)
      P.cu_query[b] = static_cast<int32_t>(cu[b] < 0x7fffffff ? cu[b] : 0x7fffffff);

  // ---- table rows
  if (P.table != nullptr) {
    for (int b = blockIdx.x; b < P.batch; b += gridDim.x) {
      const int r = P.rows != nullptr ? P.rows[b] : b;
      if (r < 0 || r >= P.num_rows) continue;
      const int64_t at = first[b];
      const int64_t have = min(min(first[b + 1], P.num_ids) - at, static_cast<int64_t>(P.max_blocks));
      int32_t* row = P.table + r * P.table_stride;
      for (int j = tid; j < P.max_blocks; j += kThreads) row[j] = j < have ? P.block_ids[at + j] : P.pad;
    }
  }

  // ---- tokens
  const int64_t total = cu[P.batch];
  for (int64_t t = static_cast<int64_t>(blockIdx.x) * kThreads + tid; t < P.tokens;
       t += static_cast<int64_t>(gridDim.x) * kThreads) {
    int32_t pos = 0;
    int64_t slot = -1;
    if (t < total) {
      int lo = 0, hi = P.batch - 1;  // the last b with cu[b] <= t
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (cu[mid] <= t)
          lo = mid;
        else
          hi = mid - 1;
      }
      const int64_t p = max(P.context_lens[lo], 0) + (t - cu[lo]);
      if (p <= 0x7fffffff) {
        pos = static_cast<int32_t>(p);
        const uint32_t col = P.page_div.div(static_cast<uint32_t>(pos));
        const int64_t at = first[lo] + col;
        if (col < static_cast<uint32_t>(P.max_blocks) && at < first[lo + 1] && at < P.num_ids) {
          const int32_t id = P.block_ids[at];
          if (id >= 0)
            slot = static_cast<int64_t>(id) * P.page + P.page_div.mod(static_cast<uint32_t>(pos), col);
        }
      }
    }
    P.positions[t] = pos;
    P.slots[t] = slot;
  }
}

__global__ void __launch_bounds__(kThreads) slot_map_kernel(const int32_t* __restrict__ table, int64_t row_stride,
                                                            int max_blocks, const int32_t* __restrict__ positions,
                                                            int64_t tokens, int page, FastDiv page_div,
                                                            int64_t* __restrict__ slots) {
  const int64_t t = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (t >= tokens) return;
  const int32_t pos = positions[t];
  int64_t slot = -1;
  if (pos >= 0) {
    const uint32_t col = page_div.div(static_cast<uint32_t>(pos));
    if (col < static_cast<uint32_t>(max_blocks)) {
      const int32_t id = table[t * row_stride + col];
      if (id >= 0) slot = static_cast<int64_t>(id) * page + page_div.mod(static_cast<uint32_t>(pos), col);
    }
  }
  slots[t] = slot;
}

}  // namespace

extern "C" int kvbm_batch_tables(const int32_t* query_lens, const int32_t* context_lens, const int32_t* block_counts,
                                 const int32_t* block_ids, int64_t num_ids, int batch, int page, int max_blocks,
                                 int pad, int32_t* table, int64_t table_stride, const int32_t* rows, int num_rows,
                                 int32_t* seq_lens, int32_t* cu_query, int32_t* positions, int64_t* slots,
                                 int64_t tokens, cudaStream_t stream) {
  if (batch < 0 || batch > kMaxBatch || page <= 0 || max_blocks < 0 || num_ids < 0 || tokens < 0)
    return cudaErrorInvalidValue;
  if (!cu_query || (batch > 0 && (!query_lens || !context_lens)) || (num_ids > 0 && !block_ids) ||
      (tokens > 0 && (!positions || !slots)))
    return cudaErrorInvalidValue;
  TablesParams P{};
  P.query_lens = query_lens;
  P.context_lens = context_lens;
  P.block_counts = block_counts;
  P.block_ids = block_ids;
  P.num_ids = num_ids;
  P.tokens = tokens;
  P.batch = batch;
  P.max_blocks = max_blocks;
  P.pad = pad;
  P.num_rows = num_rows;
  P.table = table;
  P.table_stride = table_stride;
  P.rows = rows;
  P.seq_lens = seq_lens;
  P.cu_query = cu_query;
  P.positions = positions;
  P.slots = slots;
  P.page = page;
  P.page_div = FastDiv(static_cast<uint32_t>(page));
  const size_t smem = 2 * sizeof(int64_t) * (static_cast<size_t>(batch) + 1);
  if (smem > 48 * 1024) {  // for the largest batch: another thread's launch may stand between this call and the launch
    const cudaError_t e = cudaFuncSetAttribute(batch_tables_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               static_cast<int>(2 * sizeof(int64_t) * (kMaxBatch + 1)));
    if (e != cudaSuccess) return e;
  }
  // a row or 256 tokens a CTA, up to four CTAs on each SM
  const int64_t ctas = std::max<int64_t>(table ? batch : 0, (tokens + kThreads - 1) / kThreads);
  const unsigned grid = static_cast<unsigned>(std::max<int64_t>(1, std::min<int64_t>(ctas, 4 * kvbm_sm_count())));
  batch_tables_kernel<<<grid, kThreads, smem, stream>>>(P);
  return cudaGetLastError();
}

// Slots of tokens from a table that exists: token t uses row t, or row 0 for all with row_stride 0.
extern "C" int kvbm_slot_map(const int32_t* table, int64_t row_stride, int max_blocks, const int32_t* positions,
                             int64_t tokens, int page, int64_t* slots, cudaStream_t stream) {
  if (tokens == 0) return cudaSuccess;
  if (tokens < 0 || page <= 0 || max_blocks < 0 || !positions || !slots || (max_blocks > 0 && !table))
    return cudaErrorInvalidValue;
  const int64_t grid = (tokens + kThreads - 1) / kThreads;
  if (grid > 0x7fffffff) return cudaErrorInvalidValue;
  slot_map_kernel<<<static_cast<unsigned>(grid), kThreads, 0, stream>>>(table, row_stride, max_blocks, positions,
                                                                       tokens, page,
                                                                       FastDiv(static_cast<uint32_t>(page)), slots);
  return cudaGetLastError();
}
