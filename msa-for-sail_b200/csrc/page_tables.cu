// The page table, the slots and the positions of a step, from the lengths of its requests.
//
//   n_b      = ceil(kv_b / page_size)            pages of request b
//   indptr   = exclusive scan of n               where its entries start in the flat page table
//   new_b    = max(0, n_b - held_b)              pages it needs beyond those in its row of the block table
//   page(b, p) = table[b, p]  for p < held_b,  else free[num_free - 1 - (scan of new)_b - (p - held_b)]
//   position = kv_b - qo_b + i,  slot = page(b, position / page_size) * page_size + position % page_size   for token i
//
// One CTA scans the batch (three sums at once), then every entry of the flat table and every token finds its request by a
// binary search of the scans and is computed on its own: neither one very long request nor many short ones leave
// threads without work.  Pages are handed out in the order of the requests, whatever the order of the threads.
//
// Bound by launches and by dependent reads (lengths, scans, the table, the slots): 8 requests 4.2 us in one launch, 2 048 requests of up to
// 32 768 keys with 263 113 pages 13 us in two; their bytes would take 0.1.
#include <algorithm>

#include "common.cuh"
#include "nvtx_range.h"

namespace msa {
namespace {

constexpr int kScanThreads = 1024;

// The scans, in the caller's workspace.
struct Scans {
  int32_t* qo_start;   // [batch + 1]
  int32_t* held;       // [batch] pages of the row that were there before
  int32_t* rank;       // [batch] pages taken from the stack by the requests before
  int32_t* num_free;   // [1] pages on the stack (the caller's count may be overwritten in place)
};
__host__ __device__ inline Scans scans_of(const MsaPageTablesArgs& a) {
  return {a.workspace, a.workspace + a.batch + 1, a.workspace + 2 * a.batch + 1, a.workspace + 3 * a.batch + 1};
}

__device__ __forceinline__ int free_count(const MsaPageTablesArgs& a) {
  return a.num_free ? min(max(*a.num_free, 0), a.free_capacity) : 0;
}

// Last b in [0, batch) with start[b] <= x; start[0] = 0 <= x < start[batch].
__device__ __forceinline__ int request_of(const int32_t* start, int batch, int x) {
  int lo = 0, hi = batch;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (start[mid] <= x) lo = mid; else hi = mid;
  }
  return lo;
}

// Physical page of logical page p of request b, -1 if there is none (or sums of the lengths passed 32 bits and p is one of no request).
__device__ __forceinline__ int page_of(const MsaPageTablesArgs& a, const Scans& s, int b, int p, int num_free) {
  if (static_cast<unsigned>(p) >= static_cast<unsigned>(a.table_width)) return -1;
  const int held = s.held[b];
  if (p < held) return a.block_table[b * a.table_stride + p];
  const int r = s.rank[b] + p - held;
  return static_cast<unsigned>(r) < static_cast<unsigned>(num_free) ? a.free_pages[num_free - 1 - r] : -1;
}

// Entries [first, .) of the flat table and of the tokens, `step` apart.
__device__ void fill(const MsaPageTablesArgs& a, int num_free, int64_t first, int64_t step) {
  const Scans s = scans_of(a);
  const int pages = a.kv_page_indptr[a.batch];               // more than the flat table holds: their rows are completed all the same
  for (int64_t e = first; e < max(pages, a.max_total_pages); e += step) {
    int page = -1;
    if (e < pages) {
      const int b = request_of(a.kv_page_indptr, a.batch, static_cast<int>(e));
      const int p = static_cast<int>(e) - a.kv_page_indptr[b];
      page = page_of(a, s, b, p, num_free);
      if (p >= s.held[b] && p < a.table_width) a.block_table[b * a.table_stride + p] = page;
      page = max(page, 0);      // a page that is missing (and counted): what reads the table stays in bounds
    }
    if (e < a.max_total_pages) a.kv_indices[e] = page;
  }
  const int tokens = min(s.qo_start[a.batch], a.max_total_q);
  for (int64_t t = first; t < a.max_total_q; t += step) {
    int slot = -1, pos = 0;
    if (t < tokens) {
      const int b = request_of(s.qo_start, a.batch, static_cast<int>(t));
      pos = a.kv_len[b] - (s.qo_start[b + 1] - static_cast<int>(t));
      const int page = pos >= 0 ? page_of(a, s, b, pos / a.page_size, num_free) : -1;
      const int64_t at = static_cast<int64_t>(page) * a.page_size + pos % a.page_size;
      if (page >= 0 && at <= 0x7fffffff) slot = static_cast<int>(at);
      pos = max(pos, 0);
    }
    a.slot_map[t] = slot;
    a.positions[t] = pos;
  }
}

__global__ void __launch_bounds__(kScanThreads) page_tables_scan_kernel(const MsaPageTablesArgs a, bool fill_too) {
  chain_begin();
  const Scans s = scans_of(a);
  const int num_free = free_count(a);
  __shared__ int s_sum[kScanThreads / 32][3];
  __shared__ int s_missing;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (threadIdx.x == 0) s_missing = 0;
  int carry[3] = {0, 0, 0};                                  // pages, tokens, new pages of the requests before
  int missing = 0;
  for (int b0 = 0; b0 < a.batch; b0 += kScanThreads) {
    const int b = b0 + static_cast<int>(threadIdx.x);
    int own[3] = {0, 0, 0}, held = 0, held_was = 0;
    if (b < a.batch) {
      own[0] = static_cast<int>((static_cast<int64_t>(max(a.kv_len[b], 0)) + a.page_size - 1) / a.page_size);
      own[1] = max(a.qo_len[b], 0);
      held_was = a.num_held ? a.num_held[b] : own[0];
      held = min(max(held_was, 0), a.table_width);
      own[2] = max(0, min(own[0], a.table_width) - held);
    }
    int incl[3];
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      incl[i] = own[i];
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, incl[i], d);
        if (lane >= d) incl[i] += v;
      }
      if (lane == 31) s_sum[warp][i] = incl[i];
    }
    __syncthreads();
    // every warp scans the sums of the warps
    int start[3];
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      const int mine = s_sum[lane][i];
      int scan = mine;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, scan, d);
        if (lane >= d) scan += v;
      }
      start[i] = carry[i] + __shfl_sync(0xffffffffu, scan - mine, warp) + incl[i] - own[i];
      carry[i] += __shfl_sync(0xffffffffu, scan, 31);
    }
    if (b < a.batch) {
      a.kv_page_indptr[b] = start[0];
      s.qo_start[b] = start[1];
      s.held[b] = held;
      s.rank[b] = start[2];
      const int got = min(own[2], max(0, num_free - start[2]));
      missing += own[2] - got + max(0, own[0] - a.table_width);
      if (a.num_held_out) a.num_held_out[b] = max(held_was, held + got);
    }
    __syncthreads();
  }
  if (missing) atomicAdd(&s_missing, missing);               // a sum of integers: the order does not matter
  __syncthreads();
  if (threadIdx.x == 0) {
    a.kv_page_indptr[a.batch] = carry[0];
    s.qo_start[a.batch] = carry[1];
    *s.num_free = num_free;
    if (a.num_free_out) *a.num_free_out = max(0, num_free - carry[2]);
    if (a.num_missing) *a.num_missing = s_missing + max(0, carry[0] - a.max_total_pages) + max(0, carry[1] - a.max_total_q);
  }
  if (!fill_too) return;
  __syncthreads();
  fill(a, num_free, threadIdx.x, kScanThreads);
}

__global__ void __launch_bounds__(256) page_tables_fill_kernel(const MsaPageTablesArgs a) {
  chain_begin();
  fill(a, *scans_of(a).num_free, static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x, static_cast<int64_t>(gridDim.x) * 256);
}

}  // namespace
}  // namespace msa

extern "C" int64_t msa_page_tables_workspace_bytes(int32_t batch) {
  return batch < 0 ? MSA_ERR_BAD_ARG : 4 * (3 * static_cast<int64_t>(batch) + 2);
}

extern "C" int msa_page_tables(const MsaPageTablesArgs* pa, msa_stream_t stream) {
  if (!pa) return MSA_ERR_BAD_ARG;
  const MsaPageTablesArgs& a = *pa;
  if (a.batch < 0 || a.table_width < 0 || a.page_size < 1 || a.max_total_q < 0 || a.max_total_pages < 0 || a.table_stride < a.table_width)
    return MSA_ERR_BAD_ARG;
  if (!a.kv_page_indptr || !a.workspace) return MSA_ERR_BAD_ARG;
  if (a.batch > 0 && (!a.qo_len || !a.kv_len || (a.table_width > 0 && !a.block_table))) return MSA_ERR_BAD_ARG;
  if ((a.max_total_pages > 0 && !a.kv_indices) || (a.max_total_q > 0 && (!a.slot_map || !a.positions))) return MSA_ERR_BAD_ARG;
  // pages are taken from the stack only where it is known which ones a request holds, and the other way round
  if (a.free_capacity < 0) return MSA_ERR_BAD_ARG;
  if (a.num_free) {
    if ((a.batch > 0 && !a.num_held) || (a.free_capacity > 0 && !a.free_pages)) return MSA_ERR_BAD_ARG;
  } else if (a.num_held || a.free_pages || a.num_held_out || a.num_free_out) {
    return MSA_ERR_BAD_ARG;
  }
  msa::NvtxRange range("msa_page_tables");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  // The scanning CTA also writes the entries where they are few.  In one launch against two: 64 requests with 2 218 pages 6.3 and
  // 6.7 us, 128 with 4 315 pages 9.0 and 7.6 us, 2 048 with 263 113 pages 300 and 12 us.
  const int64_t entries = static_cast<int64_t>(a.max_total_pages) + a.max_total_q;
  const bool one = entries <= 3 * msa::kScanThreads;
  if (msa::launch_chained(msa::page_tables_scan_kernel, 1, msa::kScanThreads, 0, st, a, one) != cudaSuccess) return MSA_ERR_LAUNCH;
  if (one) return MSA_OK;
  const unsigned blocks = static_cast<unsigned>(std::min<int64_t>((std::max(a.max_total_pages, a.max_total_q) + 255) / 256, 148 * 8));
  return msa::launch_chained(msa::page_tables_fill_kernel, blocks, 256, 0, st, a) == cudaSuccess ? MSA_OK : MSA_ERR_LAUNCH;
}
