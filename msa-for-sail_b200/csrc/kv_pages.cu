// Pages of a cache: copies, rows of the block table that share pages, pages given back, pages in use moved together.
//
// A block table has a row for each request; entry c of a row is the page of its tokens c * page_size .., -1 where that page was given
// back.  Free pages are a stack.  shares[p] counts the rows that hold page p beyond the first, so that a page taken from the stack needs
// no entry there.  What several threads could do in either order is made a sum of integers, a bit of a set, or goes to the first entry in the
// order of the table: results do not depend on how threads are scheduled.
//
// The tables are small: launches and chains of dependent reads bound these passes.  The copies are bound by memory.
#include <cooperative_groups.h>

#include <algorithm>
#include <climits>

#include "common.cuh"
#include "nvtx_range.h"

namespace msa {
namespace pages {
namespace {

constexpr int kThreads = 256;
constexpr int kScanThreads = 1024;
constexpr int kChunk = 16384;                  // bytes of a piece of a page that a CTA copies at a time
constexpr int kMaxCaches = 64;                 // of one launch
constexpr int kCopyCtas = 148 * 8;
constexpr int kMostIndex = INT_MAX - (1 << 20);               // of rows, columns, pages: the kernels' loops step by less than 2^20 beyond it, in 32 bits

// ---------------------------------------------------------------------------------------------------------------------------
// copies
// ---------------------------------------------------------------------------------------------------------------------------

// One cache as the copying CTAs see it: a page is `parts` pieces of `part_bytes`, stride_part apart.
struct Cache {
  char* base;
  int64_t stride_page, stride_part;
  int32_t parts, part_bytes, token_bytes;      // token_bytes: of one token in a piece (0: pieces are copied whole, -1: each is a token)
  int32_t chunks;                              // of a piece
  int32_t unit0;                               // first unit of the cache among those of an entry
  int32_t width;                               // bytes of a load: all addresses and sizes are multiples of it
};
struct Copies {
  Cache cache[kMaxCaches];
  int32_t n;
  int32_t units;                               // (cache, piece, chunk) of an entry
  int32_t num_pages;
  int32_t page_size;
  int32_t entries;                             // of the list
  const int32_t* src;
  const int32_t* dst;
  const int32_t* tokens;                       // of each entry to copy, or NULL: whole pages
  const int32_t* count;                        // entries that count, or NULL: all
  int32_t* status;
};

template <typename V>
__device__ __forceinline__ void copy_bytes(const char* src, char* dst, int bytes) {
  const V* s = reinterpret_cast<const V*>(src);
  V* d = reinterpret_cast<V*>(dst);
  const int n = bytes / static_cast<int>(sizeof(V));
  constexpr int U = 4;                         // loads on their way
  for (int i = threadIdx.x; i < n; i += U * kThreads) {
    V x[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (i + u * kThreads < n) x[u] = s[i + u * kThreads];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (i + u * kThreads < n) d[i + u * kThreads] = x[u];
  }
}

// Page src[e] to page dst[e] for every entry, by all CTAs of the grid.  An entry with a number that is no page is not copied.
__device__ __forceinline__ void copy_pages(const Copies& c) {
  const int entries = c.count ? min(max(*c.count, 0), c.entries) : c.entries;
  const int64_t all = static_cast<int64_t>(entries) * c.units;
  for (int64_t u = blockIdx.x; u < all; u += gridDim.x) {
    const int e = static_cast<int>(u / c.units);
    int unit = static_cast<int>(u % c.units);
    const int src = c.src[e], dst = c.dst[e];
    if (src < 0 || dst < 0) continue;
    if (src >= c.num_pages || dst >= c.num_pages) {
      if (threadIdx.x == 0) { chk(src, 0, c.num_pages, c.status); chk(dst, 0, c.num_pages, c.status); }
      continue;
    }
    int k = 0;
    while (k + 1 < c.n && unit >= c.cache[k + 1].unit0) ++k;
    const Cache& h = c.cache[k];
    unit -= h.unit0;
    const int part = unit / h.chunks, at = (unit % h.chunks) * kChunk;
    int all_bytes = h.part_bytes;
    if (c.tokens && h.token_bytes) {
      const int tokens = min(max(c.tokens[e], 0), c.page_size);
      all_bytes = h.token_bytes > 0 ? tokens * h.token_bytes : part < tokens ? h.part_bytes : 0;
    }
    const int bytes = min(kChunk, all_bytes - at);
    if (bytes <= 0) continue;
    const int64_t off = part * h.stride_part + at;
    const char* s = h.base + src * h.stride_page + off;
    char* d = h.base + dst * h.stride_page + off;
    if (h.width == 16) copy_bytes<uint4>(s, d, bytes);
    else if (h.width == 8) copy_bytes<uint2>(s, d, bytes);
    else if (h.width == 4) copy_bytes<uint32_t>(s, d, bytes);
    else copy_bytes<unsigned char>(s, d, bytes);
  }
}

__global__ void __launch_bounds__(kThreads) pages_copy_kernel(const __grid_constant__ Copies c) {
  chain_begin();
  copy_pages(c);
}

// ---------------------------------------------------------------------------------------------------------------------------
// scans of a CTA
// ---------------------------------------------------------------------------------------------------------------------------

// Exclusive prefix of x over the CTA, and the sum of all; s_sum has a word for each warp.  All threads take part.
template <int THREADS, typename T>
__device__ __forceinline__ T block_scan(T x, T* s_sum, T& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  constexpr int WARPS = THREADS / 32;
  T incl = x;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const T v = __shfl_up_sync(0xffffffffu, incl, d);
    if (lane >= d) incl += v;
  }
  if (lane == 31) s_sum[warp] = incl;
  __syncthreads();
  const T mine = lane < WARPS ? s_sum[lane] : T(0);
  T scan = mine;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const T v = __shfl_up_sync(0xffffffffu, scan, d);
    if (lane >= d) scan += v;
  }
  total = __shfl_sync(0xffffffffu, scan, 31);
  const T before = __shfl_sync(0xffffffffu, scan - mine, warp);
  __syncthreads();                             // s_sum may be written again
  return before + incl - x;
}

// One cluster.
template <typename... P, typename... A>
cudaError_t launch_cluster(void (*kernel)(P...), int ctas, int threads, cudaStream_t stream, A&&... args) {
  if (ctas > 8) {                              // more than every device of the architecture has to take
    const cudaError_t rc = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (rc != cudaSuccess) return rc;
  }
  return launch_chained_clusters(kernel, static_cast<unsigned>(ctas), ctas, threads, 0, stream, args...);
}

__device__ __forceinline__ int stack_size(const int32_t* num_free, int capacity) { return min(max(__ldcg(num_free), 0), capacity); }

// ---------------------------------------------------------------------------------------------------------------------------
// forks
// ---------------------------------------------------------------------------------------------------------------------------

// Workspace: claim [batch], then for each entry its child (-1: no fork), the pages it shares, the page that is copied, the page it is copied to
// (-1: none), the tokens of that, and the pages and the length that the child gets.
struct Forks {
  int32_t *claim, *child, *full, *src, *dst, *tokens, *held, *len;
};
__host__ __device__ inline Forks forks_of(const MsaPagesForkArgs& a) {
  int32_t* w = a.workspace + a.batch;
  const int64_t n = a.count;
  return {a.workspace, w, w + n, w + 2 * n, w + 3 * n, w + 4 * n, w + 5 * n, w + 6 * n};
}

__global__ void __launch_bounds__(kScanThreads) pages_fork_plan_kernel(const MsaPagesForkArgs a) {
  chain_begin();
  const Forks f = forks_of(a);
  __shared__ int s_sum[32];
  __shared__ int s_missing;
  const int tid = threadIdx.x;
  const int num_free = stack_size(a.num_free, a.free_capacity);
  auto is_row = [&](int r) { return static_cast<unsigned>(r) < static_cast<unsigned>(a.batch); };
  if (tid == 0) s_missing = 0;
  // the first of the entries that name a child has it (one with a negative parent does nothing, whatever its child)
  for (int i = tid; i < a.count; i += kScanThreads)
    if (is_row(a.children[i])) f.claim[a.children[i]] = INT_MAX;
  __syncthreads();
  for (int i = tid; i < a.count; i += kScanThreads)
    if (is_row(a.children[i]) && a.parents[i] >= 0) atomicMin(&f.claim[a.children[i]], i);
  __syncthreads();
  int taken = 0, missing = 0;                  // pages that the entries before need
  for (int i0 = 0; i0 < a.count; i0 += kScanThreads) {
    const int i = i0 + tid;
    int child = -1, full = 0, src = -1, part = 0, held = 0, len = 0;
    if (i < a.count) {
      const int p = a.parents[i], c = a.children[i];
      if (p >= 0 && c >= 0) {
        if (is_row(p) && is_row(c) && p != c && __ldcg(&f.claim[c]) == i && a.num_held[c] == 0) {
          child = c;
          const int pages = min(max(a.num_held[p], 0), a.table_width);
          len = static_cast<int>(min(static_cast<int64_t>(max(a.kv_len[p], 0)), static_cast<int64_t>(pages) * a.page_size));
          full = len / a.page_size;
          part = len - full * a.page_size;
          held = full + (part > 0);
          if (part > 0) {
            src = a.block_table[p * a.table_stride + full];
            if (static_cast<unsigned>(src) >= static_cast<unsigned>(a.num_pages)) { src = -1; part = 0; }     // the parent has none either
          }
        } else {
          ++missing;
        }
      }
    }
    int total;
    const int rank = taken + block_scan<kScanThreads>(part > 0 ? 1 : 0, s_sum, total);
    taken += total;
    int dst = -1;
    if (part > 0) {
      dst = rank < num_free ? a.free_pages[num_free - 1 - rank] : -1;
      if (static_cast<unsigned>(dst) >= static_cast<unsigned>(a.num_pages)) {                                 // it ends with its last full page
        ++missing;
        dst = src = -1;
        held = full;
        len = full * a.page_size;
      }
    }
    if (i < a.count) {
      f.child[i] = child; f.full[i] = full; f.src[i] = src; f.dst[i] = dst; f.tokens[i] = part; f.held[i] = held; f.len[i] = len;
    }
  }
  if (missing) atomicAdd(&s_missing, missing);
  __syncthreads();                             // a row may be the parent of another entry, which has read what was there before
  for (int i = tid; i < a.count; i += kScanThreads) {
    const int c = f.child[i];
    if (c < 0) continue;
    a.num_held[c] = f.held[i];
    a.kv_len[c] = f.len[i];
  }
  if (tid == 0) {
    *a.num_free = num_free - min(taken, num_free);
    if (a.num_missing) *a.num_missing = s_missing;
  }
}

__global__ void __launch_bounds__(kThreads) pages_fork_apply_kernel(const __grid_constant__ MsaPagesForkArgs a, const __grid_constant__ Copies c) {
  chain_begin();
  const Forks f = forks_of(a);
  const int chunks = (a.table_width + kThreads - 1) / kThreads;
  for (int64_t u = blockIdx.x; u < static_cast<int64_t>(a.count) * chunks; u += gridDim.x) {
    const int i = static_cast<int>(u / chunks), col = static_cast<int>(u % chunks) * kThreads + threadIdx.x;
    const int child = f.child[i];
    if (child < 0) continue;
    const int full = f.full[i];
    int32_t* row = a.block_table + child * a.table_stride;
    if (col < full) {
      const int page = a.block_table[a.parents[i] * a.table_stride + col];
      row[col] = page;
      if (static_cast<unsigned>(page) < static_cast<unsigned>(a.num_pages)) atomicAdd(&a.shares[page], 1);
    } else if (col == full && col < a.num_held[child]) {
      row[col] = f.dst[i];
    }
  }
  copy_pages(c);
}

// ---------------------------------------------------------------------------------------------------------------------------
// pages given back
// ---------------------------------------------------------------------------------------------------------------------------

// Entry (b, col) is given back: it is behind the pages that the length needs, or before all that a later query's window can see and not among
// the sinks.  The next query stands at place kv_len or later, so it sees no key below kv_len - window + 1.
struct Kept { int end, hole0, hole1, held; };                 // kept are [0, end) without [hole0, hole1)
__device__ __forceinline__ Kept kept_of(const MsaPagesFreeArgs& a, int b) {
  const int len = max(a.kv_len[b], 0), held = min(max(a.num_held[b], 0), a.table_width);
  Kept k;
  k.held = held;
  k.end = min(len / a.page_size + (len % a.page_size != 0), held);
  k.hole0 = k.hole1 = 0;
  if (a.window > 0) {
    const long long first = static_cast<long long>(len) - a.window + 1;
    k.hole0 = a.sink_tokens / a.page_size + (a.sink_tokens % a.page_size != 0);
    k.hole1 = static_cast<int>(min(static_cast<long long>(k.end), first > 0 ? first / a.page_size : 0));
  }
  return k;
}
__device__ __forceinline__ bool given_back(const Kept& k, int col) {
  return (col >= k.end && col < k.held) || (col >= k.hole0 && col < k.hole1);
}

// Page of entry (b, col) if it is given back, else -1.  Numbers that are no pages go nowhere.
__device__ __forceinline__ int page_back(const MsaPagesFreeArgs& a, const Kept& k, int b, int col) {
  if (!given_back(k, col)) return -1;
  const int page = a.block_table[b * a.table_stride + col];
  return page >= 0 && page < a.num_pages ? page : -1;
}
// The three steps for a page of an entry with number `order`.  Shares go down by one for each entry; below zero nobody holds the page, and the
// first of its entries, whose number is put in the place of the share, gives it back.
__device__ __forceinline__ void release(const MsaPagesFreeArgs& a, int page) {
  if (page >= 0 && a.shares) atomicSub(&a.shares[page], 1);
}
__device__ __forceinline__ void claim(const MsaPagesFreeArgs& a, int page, int order) {
  if (page >= 0 && a.shares && __ldcg(&a.shares[page]) < 0) atomicMin(&a.shares[page], INT_MIN + order);
}
__device__ __forceinline__ bool gives(const MsaPagesFreeArgs& a, int page, int order) {
  return page >= 0 && (!a.shares || __ldcg(&a.shares[page]) == INT_MIN + order);
}
__device__ __forceinline__ void push(const MsaPagesFreeArgs& a, int page, int place) {
  if (place < a.free_capacity) a.free_pages[place] = page;
  if (a.shares) a.shares[page] = 0;
}

// Tables of up to 2^18 entries: the CTAs of one cluster, K entries a thread that stay in registers from step to step; between the steps are
// barriers of the cluster.  (8 rows of 257 pages: 5.2 us, 8.3 in launches of their own.  512 rows that share pages: 20.5 us in a captured graph
// against 17.5, but 27 a call against 36, whose launches the host cannot keep up with.)
constexpr int kClusterCtas = 16;

template <int K>
__global__ void __launch_bounds__(kScanThreads) pages_free_cluster_kernel(const MsaPagesFreeArgs a, const int span) {
  // span: entries of a thread, at most K
  chain_begin();
  auto cluster = cooperative_groups::this_cluster();
  __shared__ int s_sum[32];
  __shared__ int s_warps[K * 32];              // pages that a warp's entries give back, then those of the entries before it in this CTA
  __shared__ int s_total;
  __shared__ Kept s_kept[kScanThreads];        // of the rows that this CTA has entries of
  const int ctas = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int entries = a.batch * a.table_width, e0 = rank * span * kScanThreads + tid;
  const int num_free = stack_size(a.num_free, a.free_capacity);
  // (the divisions of a row's limits, made for each entry, would take longest of all)
  const int row0 = min(e0 - tid, entries) / max(a.table_width, 1);
  const bool few_rows = span * kScanThreads / max(a.table_width, 1) + 2 <= kScanThreads;
  if (few_rows && row0 + tid < a.batch) s_kept[tid] = kept_of(a, row0 + tid);
  __syncthreads();
  int page[K];
  unsigned back = 0, own = 0;                  // bit k: entry e0 + k * kScanThreads is given back, and its page goes onto the stack
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int e = e0 + k * kScanThreads;
    page[k] = -1;
    if (k < span && e < entries) {
      const int b = e / a.table_width, col = e - b * a.table_width;
      if (given_back(few_rows ? s_kept[b - row0] : kept_of(a, b), col)) {
        back |= 1u << k;
        page[k] = a.block_table[b * a.table_stride + col];
      }
    }
  }
#pragma unroll
  for (int k = 0; k < K; ++k)
    if (page[k] >= a.num_pages) page[k] = -1;
  if (a.shares) {
#pragma unroll
    for (int k = 0; k < K; ++k) release(a, page[k]);
    cluster.sync();
    int share[K];
#pragma unroll
    for (int k = 0; k < K; ++k) share[k] = page[k] >= 0 ? __ldcg(&a.shares[page[k]]) : 0;
#pragma unroll
    for (int k = 0; k < K; ++k)
      if (share[k] < 0) atomicMin(&a.shares[page[k]], INT_MIN + e0 + k * kScanThreads);
    cluster.sync();
#pragma unroll
    for (int k = 0; k < K; ++k) share[k] = page[k] >= 0 ? __ldcg(&a.shares[page[k]]) : 0;
#pragma unroll
    for (int k = 0; k < K; ++k) own |= static_cast<unsigned>(share[k] == INT_MIN + e0 + k * kScanThreads) << k;
  } else {
#pragma unroll
    for (int k = 0; k < K; ++k) own |= static_cast<unsigned>(page[k] >= 0) << k;
  }
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const unsigned who = __ballot_sync(0xffffffffu, (own >> k) & 1);
    if (lane == 0) s_warps[k * 32 + warp] = __popc(who);
  }
  __syncthreads();
  int total;
  const int mine = tid < K * 32 ? s_warps[tid] : 0;
  const int before = block_scan<kScanThreads>(mine, s_sum, total);
  if (tid < K * 32) s_warps[tid] = before;
  if (tid == 0) s_total = total;
  cluster.sync();
  int at = num_free, all = 0;
  for (int c = 0; c < ctas; ++c) {
    const int n = *cluster.map_shared_rank(&s_total, c);
    if (c < rank) at += n;
    all += n;
  }
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const unsigned who = __ballot_sync(0xffffffffu, (own >> k) & 1);
    if ((own >> k) & 1) push(a, page[k], at + s_warps[k * 32 + warp] + __popc(who & ((1u << lane) - 1)));
    if ((back >> k) & 1) {
      const int e = e0 + k * kScanThreads, b = e / a.table_width;
      a.block_table[b * a.table_stride + e - b * a.table_width] = -1;
    }
  }
  for (int b = rank * kScanThreads + tid; b < a.batch; b += ctas * kScanThreads) a.num_held[b] = kept_of(a, b).end;
  if (rank == 0 && tid == 0) {
    *a.num_free = min(num_free + all, a.free_capacity);
    if (a.num_freed) *a.num_freed = all;
  }
  cluster.sync();                              // nobody leaves while its s_total may be read
}

// Long rows, or many: a CTA for 1 024 columns of a row, a kernel for each step.  Workspace: pages given back by each of these chunks, then the size of
// the stack.
constexpr int kCols = 4 * kThreads;
__device__ __forceinline__ int chunks_of(const MsaPagesFreeArgs& a) { return (a.table_width + kCols - 1) / kCols; }

template <int STEP>                            // 0 release, 1 claim, 2 count
__global__ void __launch_bounds__(kThreads) pages_free_step_kernel(const MsaPagesFreeArgs a) {
  chain_begin();
  __shared__ int s_sum[32];
  const int chunks = chunks_of(a);
  for (int u = blockIdx.x; u < a.batch * chunks; u += gridDim.x) {
    const int b = u / chunks, col0 = (u % chunks) * kCols + threadIdx.x;
    const Kept k = kept_of(a, b);
    int count = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int col = col0 + i * kThreads;
      if (col >= a.table_width) continue;
      const int page = page_back(a, k, b, col), order = b * a.table_width + col;
      if (STEP == 0) release(a, page);
      if (STEP == 1) claim(a, page, order);
      if (STEP == 2) count += gives(a, page, order);
    }
    if (STEP == 2) {
      int total;
      block_scan<kThreads>(count, s_sum, total);
      if (threadIdx.x == 0) a.workspace[u] = total;
    }
  }
  if (STEP == 2 && blockIdx.x == 0 && threadIdx.x == 0) a.workspace[a.batch * chunks] = stack_size(a.num_free, a.free_capacity);
}

// Counts become the sums of those before.
__global__ void __launch_bounds__(kScanThreads) pages_free_scan_kernel(const MsaPagesFreeArgs a) {
  chain_begin();
  __shared__ int s_sum[32];
  const int n = a.batch * chunks_of(a);
  int at = a.workspace[n];
  for (int i0 = 0; i0 < n; i0 += kScanThreads) {
    const int i = i0 + static_cast<int>(threadIdx.x);
    int total;
    const int before = block_scan<kScanThreads>(i < n ? a.workspace[i] : 0, s_sum, total);
    if (i < n) a.workspace[i] = at + before;
    at += total;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    if (a.num_freed) *a.num_freed = at - a.workspace[n];
    *a.num_free = min(at, a.free_capacity);
  }
}

__global__ void __launch_bounds__(kThreads) pages_free_push_kernel(const MsaPagesFreeArgs a) {
  chain_begin();
  __shared__ int s_sum[32];
  const int chunks = chunks_of(a);
  for (int u = blockIdx.x; u < a.batch * chunks; u += gridDim.x) {
    const int b = u / chunks, col0 = (u % chunks) * kCols;
    const Kept k = kept_of(a, b);
    int at = a.workspace[u];
#pragma unroll 1
    for (int i = 0; i < 4; ++i) {
      const int col = col0 + i * kThreads + static_cast<int>(threadIdx.x);
      int page = -1;
      bool mine = false;
      if (col < a.table_width) {
        page = page_back(a, k, b, col);
        mine = gives(a, page, b * a.table_width + col);
        if (given_back(k, col)) a.block_table[b * a.table_stride + col] = -1;
      }
      int total;
      const int rank = block_scan<kThreads>(mine ? 1 : 0, s_sum, total);
      if (mine) push(a, page, at + rank);
      at += total;
    }
    if (chunks == 1 && threadIdx.x == 0) a.num_held[b] = k.end;
  }
}

// Rows of several chunks, each of which reads what the row held before.
__global__ void __launch_bounds__(kThreads) pages_free_held_kernel(const MsaPagesFreeArgs a) {
  chain_begin();
  for (int b = blockIdx.x * kThreads + threadIdx.x; b < a.batch; b += gridDim.x * kThreads) a.num_held[b] = kept_of(a, b).end;
}

// Rows that were cut back into a page that other rows hold (see kept_of: entry len / page_size, partly used).  By one CTA, after all of the above.
// Workspace, behind the counts: the page of each such row (-1: none), its number among those that go to another page (-1: it does not), then the moves
// (from, to, tokens), then their number.  shares[p] goes down by one for each such row of p; below zero nobody else holds p, and the last row, whose
// number is put in the place of the share, keeps it.  (512 rows of 17 pages, 8 of them so: 8 us with the copy's launch, in a captured graph.)
struct Cut {
  int32_t *page, *rank, *src, *dst, *tokens, *moves;
};
__host__ __device__ inline int64_t counts_of(int batch, int width) { return static_cast<int64_t>(batch) * ((static_cast<int64_t>(width) + kCols - 1) / kCols) + 1; }
__host__ __device__ inline Cut cut_of(const MsaPagesFreeArgs& a) {
  int32_t* w = a.workspace + counts_of(a.batch, a.table_width);
  const int64_t n = a.batch;
  return {w, w + n, w + 2 * n, w + 3 * n, w + 4 * n, w + 5 * n};
}
__global__ void __launch_bounds__(kScanThreads) pages_cut_kernel(const MsaPagesFreeArgs a) {
  chain_begin();
  const Cut w = cut_of(a);
  __shared__ int s_sum[32];
  __shared__ int s_left;
  const int tid = threadIdx.x;
  const bool moves = a.num_caches > 0;
  if (tid == 0) s_left = 0;
  for (int b = tid; b < a.batch; b += kScanThreads) {
    const int len = max(a.kv_len[b], 0), col = len / a.page_size;
    int page = -1;
    if (len % a.page_size > 0 && col < min(a.num_held[b], a.table_width)) {
      page = a.block_table[b * a.table_stride + col];
      if (page < 0 || page >= a.num_pages || __ldcg(&a.shares[page]) <= 0) page = -1;
    }
    w.page[b] = page;
  }
  __syncthreads();
  if (moves) {
    for (int b = tid; b < a.batch; b += kScanThreads)
      if (w.page[b] >= 0) atomicSub(&a.shares[w.page[b]], 1);
    __syncthreads();
    for (int b = tid; b < a.batch; b += kScanThreads)
      if (w.page[b] >= 0 && __ldcg(&a.shares[w.page[b]]) < 0) atomicMin(&a.shares[w.page[b]], INT_MIN + (a.batch - 1 - b));
    __syncthreads();
    const int num_free = stack_size(a.num_free, a.free_capacity);
    int taken = 0;
    for (int b0 = 0; b0 < a.batch; b0 += kScanThreads) {
      const int b = b0 + tid, page = b < a.batch ? w.page[b] : -1;
      const bool keeps = page >= 0 && __ldcg(&a.shares[page]) == INT_MIN + (a.batch - 1 - b), goes = page >= 0 && !keeps;
      int total;
      const int rank = taken + block_scan<kScanThreads>(goes ? 1 : 0, s_sum, total);
      taken += total;
      if (b < a.batch) w.rank[b] = goes ? rank : keeps ? -2 : -1;
    }
    __syncthreads();
    for (int b = tid; b < a.batch; b += kScanThreads)
      if (w.rank[b] == -2) a.shares[w.page[b]] = 0;
    __syncthreads();
    for (int b = tid; b < a.batch; b += kScanThreads) {
      const int rank = w.rank[b];
      if (rank < 0) continue;
      const int len = a.kv_len[b];
      int to = rank < num_free ? a.free_pages[num_free - 1 - rank] : -1;
      if (static_cast<unsigned>(to) >= static_cast<unsigned>(a.num_pages)) to = -1;
      w.src[rank] = w.page[b]; w.dst[rank] = to; w.tokens[rank] = len % a.page_size;
      if (to >= 0) {
        a.block_table[b * a.table_stride + len / a.page_size] = to;
        w.page[b] = -1;                        // (it is not counted)
      } else {
        atomicAdd(&a.shares[w.page[b]], 1);
      }
    }
    __syncthreads();
    if (tid == 0) {
      *w.moves = taken;
      *a.num_free = num_free - min(taken, num_free);
    }
  }
  if (a.num_shared) {
    int left = 0;
    for (int b = tid; b < a.batch; b += kScanThreads) left += w.page[b] >= 0 && __ldcg(&a.shares[w.page[b]]) > 0;
    if (left) atomicAdd(&s_left, left);
    __syncthreads();
    if (tid == 0) *a.num_shared = s_left;
  }
}

// ---------------------------------------------------------------------------------------------------------------------------
// pages in use moved together
// ---------------------------------------------------------------------------------------------------------------------------

// Sets of pages as bits.  Managed are the pages that a row holds and those on the stack; of them, in ascending order, the first as many as rows
// hold are where the pages in use go: those above them (from `line` on) move into the free ones below, lowest to lowest.
// Workspace: live [words], free [words], then for each word the moving, the receiving and the staying-free pages in the words before, then
// {line, moving, free pages afterwards}.
struct Sets {
  uint32_t *live, *free;
  int32_t *moving, *holes, *rest, *sums;
};
__host__ __device__ inline int words_of(int num_pages) { return num_pages / 32 + (num_pages % 32 != 0); }
__host__ __device__ inline Sets sets_of(const MsaPagesCompactArgs& a) {
  const int64_t w = words_of(a.num_pages);
  int32_t* s = a.workspace;
  return {reinterpret_cast<uint32_t*>(s), reinterpret_cast<uint32_t*>(s + w), s + 2 * w, s + 3 * w, s + 4 * w, s + 5 * w};
}

// Steps, for thread `first` of `step`.
__device__ __forceinline__ void mark_pages(const MsaPagesCompactArgs& a, int64_t first, int64_t step) {
  const Sets s = sets_of(a);
  const int num_free = stack_size(a.num_free, a.free_capacity);
  auto mark = [&](uint32_t* set, int page) {
    if (static_cast<unsigned>(page) < static_cast<unsigned>(a.num_pages)) atomicOr(&set[page >> 5], 1u << (page & 31));
  };
  for (int64_t i = first; i < num_free; i += step) mark(s.free, a.free_pages[i]);
  constexpr int U = 4;                         // entries on their way
  const int64_t entries = static_cast<int64_t>(a.batch) * a.table_width;
  for (int64_t e0 = first; e0 < entries; e0 += U * step) {
    int page[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t e = e0 + u * step;
      page[u] = -1;
      if (e < entries) {
        const int b = static_cast<int>(e / a.table_width), col = static_cast<int>(e % a.table_width);
        if (col < a.num_held[b]) page[u] = a.block_table[b * a.table_stride + col];
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) mark(s.live, page[u]);
  }
}

// Bits of word w from page `line` on.
__device__ __forceinline__ uint32_t from_line(int w, int line) {
  const int d = line - 32 * w;
  return d <= 0 ? 0xffffffffu : d >= 32 ? 0u : 0xffffffffu << d;
}

// By one CTA of kScanThreads.
__device__ __forceinline__ void rank_pages(const MsaPagesCompactArgs& a) {
  // Several counts go through a scan at once, in fields that the pages of one scan (2^15) do not fill.
  using u64 = unsigned long long;
  const Sets s = sets_of(a);
  __shared__ u64 s_sum[32];
  __shared__ int s_line;
  const int tid = threadIdx.x, words = words_of(a.num_pages);
  u64 total;
  int used = 0, before = 0, mine = 0;          // pages in use; managed ones in the words before this scan's, before this thread's
  uint32_t managed = 0;
  for (int w0 = 0; w0 < words; w0 += kScanThreads) {
    const int w = w0 + tid;
    const uint32_t live = w < words ? __ldcg(&s.live[w]) : 0u;
    managed = w < words ? live | __ldcg(&s.free[w]) : 0u;
    mine = before + static_cast<int>(block_scan<kScanThreads>(static_cast<u64>(__popc(live)) << 32 | __popc(managed), s_sum, total) & 0xffffffffu);
    used += static_cast<int>(total >> 32);
    before += static_cast<int>(total & 0xffffffffu);
  }
  if (tid == 0) s_line = a.num_pages;          // (nothing is free below it: nothing moves)
  __syncthreads();
  // the managed page with number `used` (from 0) is the first one that does not stay in use
  auto find = [&](int w) {
    if (mine <= used && used < mine + __popc(managed)) {
      uint32_t m = managed;
      for (int n = used - mine; n > 0; --n) m &= m - 1;
      s_line = 32 * w + __ffs(m) - 1;
    }
  };
  if (words <= kScanThreads) {
    find(tid);
  } else {
    before = 0;
    for (int w0 = 0; w0 < words && before <= used; w0 += kScanThreads) {
      const int w = w0 + tid;
      managed = w < words ? __ldcg(&s.live[w]) | __ldcg(&s.free[w]) : 0u;
      mine = before + static_cast<int>(block_scan<kScanThreads>(static_cast<u64>(__popc(managed)), s_sum, total));
      before += static_cast<int>(total);
      find(w);
    }
  }
  __syncthreads();
  const int line = s_line;
  int sums[3] = {0, 0, 0};
  for (int w0 = 0; w0 < words; w0 += kScanThreads) {
    const int w = w0 + tid;
    u64 own = 0;
    if (w < words) {
      const uint32_t live = __ldcg(&s.live[w]), all = live | __ldcg(&s.free[w]), above = from_line(w, line);
      own = static_cast<u64>(__popc(live & above)) | static_cast<u64>(__popc(all & ~live & ~above)) << 20 | static_cast<u64>(__popc(all & above)) << 40;
    }
    const u64 at = block_scan<kScanThreads>(own, s_sum, total);
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      if (w < words) (i == 0 ? s.moving : i == 1 ? s.holes : s.rest)[w] = sums[i] + static_cast<int>(at >> (20 * i) & 0xfffff);
      sums[i] += static_cast<int>(total >> (20 * i) & 0xfffff);
    }
  }
  if (tid == 0) {
    s.sums[0] = line; s.sums[1] = sums[0]; s.sums[2] = sums[2];
    *a.num_moved = sums[0];
  }
}

// The list of moves, and the stack: the lowest page on top.
__device__ __forceinline__ void list_pages(const MsaPagesCompactArgs& a, int first, int step) {
  const Sets s = sets_of(a);
  const int line = __ldcg(&s.sums[0]), moved = __ldcg(&s.sums[1]), left = __ldcg(&s.sums[2]);
  for (int p = first; p < a.num_pages; p += step) {
    const int w = p >> 5;
    const uint32_t bit = 1u << (p & 31), live = __ldcg(&s.live[w]), managed = live | __ldcg(&s.free[w]), above = from_line(w, line);
    if (live & above & bit) a.src[__ldcg(&s.moving[w]) + __popc(live & above & (bit - 1))] = p;
    if (managed & ~live & ~above & bit) a.dst[__ldcg(&s.holes[w]) + __popc(managed & ~live & ~above & (bit - 1))] = p;
    if (managed & above & bit) a.free_pages[left - 1 - __ldcg(&s.rest[w]) - __popc(managed & above & (bit - 1))] = p;
    if (p >= moved) a.src[p] = a.dst[p] = -1;  // (the lists have a place for every page; moves come before)
  }
  if (first == 0) *a.num_free = left;
}

// Ordinary pools: the CTAs of one cluster.  (8 192 pages, nothing to copy: 14.4 us in a captured graph; 15.5 before the counts shared a scan,
// when a memset and three launches took 17.4.)
__global__ void __launch_bounds__(kScanThreads) pages_compact_cluster_kernel(const MsaPagesCompactArgs a) {
  chain_begin();
  auto cluster = cooperative_groups::this_cluster();
  const int first = static_cast<int>(cluster.block_rank()) * kScanThreads + threadIdx.x, step = static_cast<int>(cluster.num_blocks()) * kScanThreads;
  uint32_t* words = sets_of(a).live;           // and the free ones behind them
  for (int w = first; w < 2 * words_of(a.num_pages); w += step) words[w] = 0;
  cluster.sync();
  mark_pages(a, first, step);
  cluster.sync();
  if (cluster.block_rank() == 0) rank_pages(a);
  cluster.sync();
  list_pages(a, first, step);
}

__global__ void __launch_bounds__(kThreads) pages_mark_kernel(const MsaPagesCompactArgs a) {
  chain_begin();
  mark_pages(a, static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x, static_cast<int64_t>(gridDim.x) * kThreads);
}
__global__ void __launch_bounds__(kScanThreads) pages_rank_kernel(const MsaPagesCompactArgs a) {
  chain_begin();
  rank_pages(a);
}
__global__ void __launch_bounds__(kThreads) pages_list_kernel(const MsaPagesCompactArgs a) {
  chain_begin();
  list_pages(a, blockIdx.x * kThreads + threadIdx.x, gridDim.x * kThreads);
}

__global__ void __launch_bounds__(kThreads) pages_move_kernel(const __grid_constant__ MsaPagesCompactArgs a, const __grid_constant__ Copies c) {
  chain_begin();
  const Sets s = sets_of(a);
  const int line = s.sums[0], moved = s.sums[1];
  const int64_t first = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x, step = static_cast<int64_t>(gridDim.x) * kThreads;
  for (int64_t e = first; moved > 0 && e < static_cast<int64_t>(a.batch) * a.table_width; e += step) {
    const int b = static_cast<int>(e / a.table_width), col = static_cast<int>(e % a.table_width);
    if (col >= a.num_held[b]) continue;
    int32_t* entry = a.block_table + b * a.table_stride + col;
    const int p = *entry;
    if (p < line || p >= a.num_pages) continue;
    const int w = p >> 5;
    *entry = a.dst[s.moving[w] + __popc(s.live[w] & from_line(w, line) & ((1u << (p & 31)) - 1))];
  }
  if (a.shares)
    for (int64_t i = first; i < moved; i += step) {
      a.shares[a.dst[i]] = a.shares[a.src[i]];
      a.shares[a.src[i]] = 0;
    }
  copy_pages(c);
}

// ---------------------------------------------------------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------------------------------------------------------

// Caches [first, first + kMaxCaches) for a launch; `tokens_count`: entries may copy part of a page.
int make_copies(Copies& c, const MsaPageCache* caches, int num_caches, int first, int num_pages, int page_size, bool tokens_count) {
  c = {};
  c.num_pages = num_pages;
  c.page_size = page_size;
  for (int i = first; i < std::min(num_caches, first + kMaxCaches); ++i) {
    const MsaPageCache& m = caches[i];
    if (!m.base || m.parts < 1 || m.part_bytes < 1 || m.token_bytes < -1) return MSA_ERR_BAD_ARG;
    if (m.token_bytes > 0 && static_cast<int64_t>(m.token_bytes) * page_size > m.part_bytes) return MSA_ERR_BAD_ARG;
    Cache& h = c.cache[c.n];
    h.base = static_cast<char*>(m.base);
    h.stride_page = m.stride_page; h.stride_part = m.stride_part;
    h.parts = m.parts; h.part_bytes = m.part_bytes; h.token_bytes = tokens_count ? m.token_bytes : 0;
    if (h.token_bytes == 0 && m.stride_part == m.part_bytes && static_cast<int64_t>(m.parts) * m.part_bytes <= INT_MAX) {     // one piece
      h.part_bytes *= h.parts;
      h.parts = 1;
    }
    uint64_t bits = reinterpret_cast<uint64_t>(h.base) | static_cast<uint64_t>(h.stride_page) | static_cast<uint64_t>(h.part_bytes) |
                    static_cast<uint64_t>(std::max(h.token_bytes, 0)) | (h.parts > 1 ? static_cast<uint64_t>(h.stride_part) : 0);
    h.width = bits % 16 == 0 ? 16 : bits % 8 == 0 ? 8 : bits % 4 == 0 ? 4 : 1;
    h.chunks = (h.part_bytes + kChunk - 1) / kChunk;
    h.unit0 = c.units;
    const int64_t units = c.units + static_cast<int64_t>(h.parts) * h.chunks;
    if (units > INT_MAX) return MSA_ERR_TOO_LARGE;
    c.units = static_cast<int>(units);
    ++c.n;
  }
  return MSA_OK;
}

unsigned copy_grid(const Copies& c) {
  return static_cast<unsigned>(std::max<int64_t>(1, std::min<int64_t>(static_cast<int64_t>(c.entries) * c.units, kCopyCtas)));
}

// The launches of a copy of all caches; `first(copies, grid)` in the place of the first of them, where a kernel does more.
template <typename F>
int launch_copies(const MsaPageCache* caches, int num_caches, int num_pages, int page_size, const Copies& list, unsigned least, cudaStream_t st, F&& first) {
  for (int i = 0; i == 0 || i < num_caches; i += kMaxCaches) {
    Copies c;
    if (const int rc = make_copies(c, caches, num_caches, i, num_pages, page_size, list.tokens != nullptr)) return rc;
    c.entries = list.entries; c.src = list.src; c.dst = list.dst; c.tokens = list.tokens; c.count = list.count; c.status = list.status;
    const unsigned grid = copy_grid(c);
    const cudaError_t rc = i == 0 ? first(c, std::max(grid, least)) : launch_chained(pages_copy_kernel, grid, kThreads, 0, st, c);
    if (rc != cudaSuccess) return MSA_ERR_LAUNCH;
  }
  return MSA_OK;
}

int check_caches(const MsaPageCache* caches, int num_caches, int num_pages, int page_size) {
  if (num_caches < 0 || (num_caches > 0 && !caches) || num_pages < 0 || page_size < 1) return MSA_ERR_BAD_ARG;
  for (int i = 0; i < num_caches; i += kMaxCaches) {
    Copies c;
    if (const int rc = make_copies(c, caches, num_caches, i, num_pages, page_size, true)) return rc;
  }
  return MSA_OK;
}

// The pages that rows give back.
int give_back(const MsaPagesFreeArgs& a, int64_t entries, cudaStream_t st) {
  if (entries <= 16 * kClusterCtas * kScanThreads) {
    const int k = entries <= kClusterCtas * kScanThreads ? 1 : entries <= 4 * kClusterCtas * kScanThreads ? 4 : 16;
    int ctas = 1;
    while (ctas < kClusterCtas && static_cast<int64_t>(ctas) * kScanThreads < entries) ctas *= 2;
    const int span = static_cast<int>((entries + ctas * kScanThreads - 1) / (ctas * kScanThreads));
    const auto kernel = k == 1 ? pages_free_cluster_kernel<1> : k == 4 ? pages_free_cluster_kernel<4> : pages_free_cluster_kernel<16>;
    return launch_cluster(kernel, ctas, kScanThreads, st, a, span) == cudaSuccess ? MSA_OK : MSA_ERR_LAUNCH;
  }
  const int64_t units = static_cast<int64_t>(a.batch) * ((a.table_width + kCols - 1) / kCols);
  const unsigned grid = static_cast<unsigned>(std::min<int64_t>(units, kCopyCtas));
  cudaError_t rc = cudaSuccess;
  if (a.shares) {
    rc = msa::launch_chained(pages_free_step_kernel<0>, grid, kThreads, 0, st, a);
    if (rc == cudaSuccess) rc = msa::launch_chained(pages_free_step_kernel<1>, grid, kThreads, 0, st, a);
  }
  if (rc == cudaSuccess) rc = msa::launch_chained(pages_free_step_kernel<2>, grid, kThreads, 0, st, a);
  if (rc == cudaSuccess) rc = msa::launch_chained(pages_free_scan_kernel, 1, kScanThreads, 0, st, a);
  if (rc == cudaSuccess) rc = msa::launch_chained(pages_free_push_kernel, grid, kThreads, 0, st, a);
  if (rc == cudaSuccess && a.table_width > kCols)
    rc = msa::launch_chained(pages_free_held_kernel, static_cast<unsigned>(std::min((a.batch + kThreads - 1) / kThreads, 148)), kThreads, 0, st, a);
  return rc == cudaSuccess ? MSA_OK : MSA_ERR_LAUNCH;
}

}  // namespace
}  // namespace pages
}  // namespace msa

extern "C" int msa_pages_copy(const MsaPagesCopyArgs* pa, msa_stream_t stream) {
  using namespace msa::pages;
  if (!pa) return MSA_ERR_BAD_ARG;
  const MsaPagesCopyArgs& a = *pa;
  if (const int rc = check_caches(a.caches, a.num_caches, a.num_pages, a.page_size)) return rc;
  if (a.count < 0 || (a.count > 0 && (!a.src || !a.dst))) return MSA_ERR_BAD_ARG;
  if (a.count == 0 || a.num_caches == 0) return MSA_OK;
  msa::NvtxRange range("msa_pages_copy");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  Copies list = {};
  list.entries = a.count; list.src = a.src; list.dst = a.dst; list.status = a.status;
  return launch_copies(a.caches, a.num_caches, a.num_pages, a.page_size, list, 1, st, [&](const Copies& c, unsigned grid) {
    return msa::launch_chained(pages_copy_kernel, grid, kThreads, 0, st, c);
  });
}

extern "C" int64_t msa_pages_fork_workspace_bytes(int32_t batch, int32_t count) {
  return batch < 0 || count < 0 ? MSA_ERR_BAD_ARG : 4 * (static_cast<int64_t>(batch) + 7 * static_cast<int64_t>(count));
}

extern "C" int msa_pages_fork(const MsaPagesForkArgs* pa, msa_stream_t stream) {
  using namespace msa::pages;
  if (!pa) return MSA_ERR_BAD_ARG;
  const MsaPagesForkArgs& a = *pa;
  if (const int rc = check_caches(a.caches, a.num_caches, a.num_pages, a.page_size)) return rc;
  if (a.batch < 0 || a.table_width < 0 || a.table_stride < a.table_width || a.count < 0 || a.free_capacity < 0) return MSA_ERR_BAD_ARG;
  if (!a.num_free || !a.workspace || (a.count > 0 && (!a.parents || !a.children))) return MSA_ERR_BAD_ARG;
  if (a.batch > 0 && (!a.num_held || !a.kv_len || (a.table_width > 0 && !a.block_table))) return MSA_ERR_BAD_ARG;
  if ((a.free_capacity > 0 && !a.free_pages) || (a.num_pages > 0 && !a.shares)) return MSA_ERR_BAD_ARG;
  if (a.count > (1 << 24) || a.table_width > kMostIndex) return MSA_ERR_TOO_LARGE;
  msa::NvtxRange range("msa_pages_fork");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (msa::launch_chained(pages_fork_plan_kernel, 1, kScanThreads, 0, st, a) != cudaSuccess) return MSA_ERR_LAUNCH;
  if (a.count == 0) return MSA_OK;
  const Forks f = forks_of(a);
  Copies list = {};
  list.entries = a.count; list.src = f.src; list.dst = f.dst; list.tokens = f.tokens;
  const int64_t rows = static_cast<int64_t>(a.count) * ((a.table_width + kThreads - 1) / kThreads);
  return launch_copies(a.caches, a.num_caches, a.num_pages, a.page_size, list, static_cast<unsigned>(std::min<int64_t>(std::max<int64_t>(rows, 1), kCopyCtas)), st,
                       [&](const Copies& c, unsigned grid) { return msa::launch_chained(pages_fork_apply_kernel, grid, kThreads, 0, st, a, c); });
}

extern "C" int64_t msa_pages_free_workspace_bytes(int32_t batch, int32_t table_width) {
  if (batch < 0 || table_width < 0) return MSA_ERR_BAD_ARG;
  return 4 * (msa::pages::counts_of(batch, table_width) + 5 * static_cast<int64_t>(batch) + 1);
}

extern "C" int msa_pages_free(const MsaPagesFreeArgs* pa, msa_stream_t stream) {
  using namespace msa::pages;
  if (!pa) return MSA_ERR_BAD_ARG;
  const MsaPagesFreeArgs& a = *pa;
  if (a.batch < 0 || a.table_width < 0 || a.table_stride < a.table_width || a.page_size < 1 || a.free_capacity < 0 || a.num_pages < 0) return MSA_ERR_BAD_ARG;
  if (a.window < 0 || a.sink_tokens < 0 || (a.sink_tokens > 0 && a.window == 0)) return MSA_ERR_BAD_ARG;
  if (!a.num_free || !a.workspace || (a.free_capacity > 0 && !a.free_pages)) return MSA_ERR_BAD_ARG;
  if (a.batch > 0 && (!a.num_held || !a.kv_len || (a.table_width > 0 && !a.block_table))) return MSA_ERR_BAD_ARG;
  if (const int rc = check_caches(a.caches, a.num_caches, a.num_pages, a.page_size)) return rc;
  if ((a.num_caches > 0 || a.num_shared) && !a.shares) return MSA_ERR_BAD_ARG;
  const int64_t entries = static_cast<int64_t>(a.batch) * a.table_width;
  if (entries > INT_MAX / 2 || a.batch > kMostIndex) return MSA_ERR_TOO_LARGE;
  msa::NvtxRange range("msa_pages_free");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (const int rc = give_back(a, entries, st)) return rc;
  if (a.num_caches == 0 && !a.num_shared) return MSA_OK;
  if (msa::launch_chained(pages_cut_kernel, 1, kScanThreads, 0, st, a) != cudaSuccess) return MSA_ERR_LAUNCH;
  if (a.num_caches == 0 || a.batch == 0) return MSA_OK;
  const Cut w = cut_of(a);
  Copies list = {};
  list.entries = a.batch; list.src = w.src; list.dst = w.dst; list.tokens = w.tokens; list.count = w.moves;
  return launch_copies(a.caches, a.num_caches, a.num_pages, a.page_size, list, 1, st, [&](const Copies& c, unsigned grid) {
    return msa::launch_chained(pages_copy_kernel, grid, kThreads, 0, st, c);
  });
}

extern "C" int64_t msa_pages_compact_workspace_bytes(int32_t num_pages) {
  return num_pages < 0 ? MSA_ERR_BAD_ARG : 4 * (5 * static_cast<int64_t>(msa::pages::words_of(num_pages)) + 3);
}

extern "C" int msa_pages_compact(const MsaPagesCompactArgs* pa, msa_stream_t stream) {
  using namespace msa::pages;
  if (!pa) return MSA_ERR_BAD_ARG;
  const MsaPagesCompactArgs& a = *pa;
  if (const int rc = check_caches(a.caches, a.num_caches, a.num_pages, a.page_size)) return rc;
  if (a.batch < 0 || a.table_width < 0 || a.table_stride < a.table_width || a.free_capacity < 0) return MSA_ERR_BAD_ARG;
  if (!a.num_free || !a.workspace || !a.num_moved || (a.free_capacity > 0 && !a.free_pages) || (a.num_pages > 0 && (!a.src || !a.dst))) return MSA_ERR_BAD_ARG;
  if (a.batch > 0 && (!a.num_held || (a.table_width > 0 && !a.block_table))) return MSA_ERR_BAD_ARG;
  if (a.num_pages > kMostIndex || a.batch > kMostIndex || a.table_width > kMostIndex) return MSA_ERR_TOO_LARGE;
  msa::NvtxRange range("msa_pages_compact");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const Sets s = sets_of(a);
  const int64_t entries = static_cast<int64_t>(a.batch) * a.table_width;
  auto grid = [](int64_t n) { return static_cast<unsigned>(std::max<int64_t>(1, std::min<int64_t>((n + kThreads - 1) / kThreads, kCopyCtas))); };
  cudaError_t rc = cudaSuccess;
  if (entries <= (1 << 17) && a.num_pages <= (1 << 17)) {
    rc = launch_cluster(pages_compact_cluster_kernel, kClusterCtas, kScanThreads, st, a);
  } else {
    rc = cudaMemsetAsync(s.live, 0, 8 * static_cast<size_t>(words_of(a.num_pages)), st);
    if (rc == cudaSuccess) rc = msa::launch_chained(pages_mark_kernel, grid(std::max<int64_t>(entries, a.free_capacity)), kThreads, 0, st, a);
    if (rc == cudaSuccess) rc = msa::launch_chained(pages_rank_kernel, 1, kScanThreads, 0, st, a);
    if (rc == cudaSuccess) rc = msa::launch_chained(pages_list_kernel, grid(a.num_pages), kThreads, 0, st, a);
  }
  if (rc != cudaSuccess) return MSA_ERR_LAUNCH;
  Copies list = {};
  list.entries = a.num_pages; list.src = a.src; list.dst = a.dst; list.count = a.num_moved;
  return launch_copies(a.caches, a.num_caches, a.num_pages, a.page_size, list, grid(entries), st,
                       [&](const Copies& c, unsigned g) { return msa::launch_chained(pages_move_kernel, g, kThreads, 0, st, a, c); });
}
