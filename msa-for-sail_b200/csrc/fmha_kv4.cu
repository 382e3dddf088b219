// Attention of a few query rows over a cache held in 4 bits (layout in kv4.cuh).
//
// Per key and KV head 144 bytes are read and 4 * 128 multiplications are made for every row, so the pass should be bound by memory;
// what is in the way is the conversion of two 4-bit elements a byte into operands of the tensor cores.  So the products are
// arranged such that codes go from shared memory to registers, are converted there, and are operands as they are:
//
//   S^T = K Q^T   A = 16 keys x 16 elements of K, B = Q^T (rows in registers for the whole item)
//   O^T = V^T P^T A = 16 elements x 16 keys of V^T, B = P^T (S^T through a transposing register move)
//
// (mma.sync.m16n8k16, f16 operands, f32 accumulators.)  The order of the contraction is free, so thread t of a group of four takes
// elements 32 t .. 32 t + 31 of its keys: 16 contiguous bytes.  For V^T thread group g holds elements 16 g .. 16 g + 15, the 16 that
// share a scale, of the keys 2 t, 2 t + 1, 2 t + 8, 2 t + 9 of a step.  tcgen05 would take its operands from shared memory, where
// the converted tiles (64 KB a page, in and out again) cost more than the pages' share of the memory bandwidth.
//
// e2m1 x e4m3 is exact in f16 (6 significant bits, at most 2688, a multiple of 2^-10).  A query row is multiplied by a power of two that
// brings its largest element to [2^14, 2^15): exact in f16 down to 2^-28 of the largest.  P is written as 2^(x - m + 7), with m at
// most 8 behind the true maximum: at most 2^15, 11 bits down to 2^-21 of the largest weight.  O is divided by the sum of the
// rounded P, the LSE comes from the sum before rounding.
//
// A CTA has four warps that multiply (warp w has keys 32 w .. 32 w + 31 of every page, with a softmax of its own; the four states are
// joined at the end) and one that fetches: a page and head is one bulk copy each for K and V.  Three CTAs share an SM: one item's
// first pages and epilogue come under the others' work.
#include <algorithm>

#include "kv4.cuh"
#include "nvtx_range.h"
#include "tc_ptx.cuh"

namespace msa {
namespace kv4 {
namespace {

using namespace tc;

constexpr int kWarps = 4;                                    // that multiply
constexpr int kThreads = 32 * (kWarps + 1);
constexpr int kStages = 4;
constexpr int kStageBytes = 2 * kKv4TileBytes;
constexpr int kOffFull = kStages * kStageBytes;
constexpr int kOffEmpty = kOffFull + 8 * kStages;
constexpr int kOffKey = kOffEmpty + 8 * kStages;             // first key of the page in a stage, -1: no more pages
constexpr int kOffAbort = kOffKey + 4 * kStages;
constexpr int kSmemBytes = kOffAbort + 16 + 128;             // + slack to align the base
constexpr int kLdO = kHeadDim + 4;                           // floats of a row of O in shared memory
constexpr float kPOffset = 7.f;
constexpr float kRescale = 8.f;

// Key of a 16-key step that stands at place j (0..7) of an operand: a quarter-warp's 16-byte reads of K rows fall into all banks.
__device__ __forceinline__ int key_at(int j) { return (j & 4) | ((j & 2) ? 3 - (j & 1) : (j & 1)); }

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  const uint32_t a[4] = {a0, a1, a2, a3};
  mma_16816<true>(d, a, b0, b1);
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
               ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
  return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t addr) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr));
  return v;
}
__device__ __forceinline__ uint32_t lds16(uint32_t addr) {
  uint16_t v;
  asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(addr));
  return v;
}
__device__ __forceinline__ uint32_t lds8(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared.u8 %0, [%1];" : "=r"(v) : "r"(addr));
  return v;
}

// The item of a CTA: rows of one KV head against a list of pages.
struct Item {
  int b, kvh, split;
  int row0, nrows;                 // packed rows (token, head) of this CTA
  int head0, pack, tok0;           // row r: token tok0 + r / pack of the sequence, head head0 + r % pack
  int qo_base, kv_len, off, page_base;
  int first, last;                 // entries of the page list: logical pages, or places of the selection
  const int32_t* blocks;           // selection, or nullptr
};

template <int NT>
__global__ void __launch_bounds__(kThreads, 3) kv4_decode_kernel(const __grid_constant__ MsaFmhaParams p) {
  extern __shared__ unsigned char smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 127u) & ~127u;
  unsigned char* smem = smem_raw + (base - smem_u32(smem_raw));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  auto full = [&](int s) -> uint32_t { return base + kOffFull + 8 * s; };
  auto empty = [&](int s) -> uint32_t { return base + kOffEmpty + 8 * s; };
  volatile int* s_key = reinterpret_cast<volatile int*>(smem + kOffKey);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + kOffAbort);
  volatile int* skip_flag = abort_flag + 1;
  chain_begin();

  // ---------------- the item ----------------
  const bool sparse = (p.flags & MSA_FLAG_SPARSE) != 0;
  const int h_r = p.num_qo_heads / p.num_kv_heads;
  const int rg = blockIdx.y * (8 * NT);                      // first row of this CTA's group
  Item it;
  if (!sparse) {
    const MsaWorkItem w = p.work[blockIdx.x];
    it.b = chk(w.batch, 0, p.batch, p.status);
    it.head0 = chk(w.head0, 0, p.num_qo_heads, p.status);
    it.split = chk(w.split, 0, p.num_splits, p.status);
    it.pack = p.pack; it.tok0 = 0;
    it.row0 = w.row0 + rg; it.nrows = min(8 * NT, w.num_rows - rg);
    it.first = w.kv_tile_begin; it.last = w.kv_tile_end;
    it.blocks = nullptr;
    it.kvh = it.head0 / h_r;
  } else {
    int idx = blockIdx.x;
    it.split = idx % p.num_splits; idx /= p.num_splits;
    it.kvh = idx % p.num_kv_heads;
    const int t = idx / p.num_kv_heads;
    it.b = chk(p.token_batch[t], 0, p.batch, p.status);
    it.head0 = it.kvh * h_r; it.pack = h_r;
    it.tok0 = t - p.qo_start[it.b];
    it.row0 = rg; it.nrows = min(8 * NT, h_r - rg);
    const int per = (p.kv_block_num + p.num_splits - 1) / p.num_splits;
    it.first = it.split * per;
    it.last = min(p.kv_block_num, it.first + per);
    it.blocks = p.kv_block_indexes + t * p.kbi_stride_tok + it.kvh * p.kbi_stride_head;
  }
  if (it.nrows <= 0) return;
  it.qo_base = p.qo_start[it.b];
  it.kv_len = p.kv_len[it.b];
  it.off = p.qo_offset[it.b];
  it.page_base = p.kv_page_indptr[it.b];
  // keys that rows may see: row r sees keys below lim(r), which grows with r
  auto lim = [&](int r) -> int { return min(it.kv_len, it.tok0 + (it.row0 + min(r, it.nrows - 1)) / it.pack + it.off + 1); };
  const int lim_first = lim(0), lim_last = lim(it.nrows - 1);

  if (threadIdx.x == kThreads - 1)
    *skip_flag = (p.status != nullptr && *reinterpret_cast<const volatile int32_t*>(p.status) != 0) ? 1 : 0;
  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) { mbar_init(full(s), 1); mbar_init(empty(s), kWarps); }
    *abort_flag = 0;
    mbar_fence_init();
  }
  __syncthreads();
  if (*skip_flag) return;

  float m[NT][2], l_round[NT][2], l_sum[NT][2];
  float o[8][NT][4];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
#pragma unroll
    for (int c = 0; c < 2; ++c) { m[n][c] = -INFINITY; l_round[n][c] = l_sum[n][c] = 0.f; }
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int c = 0; c < 4; ++c) o[i][n][c] = 0.f;
  }
  const int g = lane >> 2, t4 = lane & 3;

  if (warp == kWarps) {
    // =========================== fetching ===========================
    int stage = 0;
    uint32_t phase = 0;
    bool alive = true;
    for (int j0 = it.first; j0 < it.last && alive; j0 += 32) {
      const int j = j0 + lane;
      int blk = -1, phys = 0;
      if (j < it.last) blk = it.blocks ? it.blocks[j] : j;
      const bool seen = blk >= 0 && blk * static_cast<int64_t>(kKvTile) < lim_last;
      if (seen) phys = min(max(chk(p.kv_indices[it.page_base + blk], 0, static_cast<int>(p.kv_extent), p.status), 0), static_cast<int>(p.kv_extent) - 1);
      for (uint32_t todo = __ballot_sync(0xffffffffu, seen); todo && alive; todo &= todo - 1) {
        const int src = __ffs(todo) - 1;
        const int page = __shfl_sync(0xffffffffu, phys, src), lp = __shfl_sync(0xffffffffu, blk, src);
        alive = mbar_wait_warp(empty(stage), phase ^ 1, abort_flag);
        if (!alive) break;
        if (elect_one()) {
          s_key[stage] = lp * kKvTile;
          mbar_arrive_expect_tx(full(stage), kStageBytes);
          const uint32_t dst = base + stage * kStageBytes;
          bulk_load(dst, static_cast<const unsigned char*>(p.k) + page * p.k_stride_page + it.kvh * p.k_stride_head, kKv4TileBytes, full(stage));
          bulk_load(dst + kKv4TileBytes, static_cast<const unsigned char*>(p.v) + page * p.v_stride_page + it.kvh * p.v_stride_head, kKv4TileBytes,
                    full(stage));
        }
        __syncwarp();
        if (++stage == kStages) { stage = 0; phase ^= 1; }
      }
    }
    if (alive) alive = mbar_wait_warp(empty(stage), phase ^ 1, abort_flag);
    if (alive && elect_one()) { s_key[stage] = -1; mbar_arrive(full(stage)); }
    __syncwarp();
  } else {
    // =========================== multiplying ===========================
    uint32_t qf[NT][16];
    float fac[NT][2];                                        // score * fac = exponent of two
    int limit[NT][2];
    const float scale = p.sm_scale * (p.k_scale_head ? p.k_scale_head[it.kvh] : 1.f) * kLog2e;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int r = 8 * n + g;
      const int row = it.row0 + min(r, it.nrows - 1);
      const int64_t at = (it.qo_base + it.tok0 + row / it.pack) * p.q_stride_tok + (it.head0 + row % it.pack) * p.q_stride_head + 32 * t4;
      float x[32];
      if (p.q_dtype == MSA_DT_E4M3) {
        const uint4* src = reinterpret_cast<const uint4*>(static_cast<const unsigned char*>(p.q) + at);
#pragma unroll
        for (int v = 0; v < 2; ++v) {
          const uint4 raw = src[v];
          const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            const uint32_t h = kv4_scales_to_half(static_cast<uint16_t>(w[c >> 1] >> (16 * (c & 1))));
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
            x[16 * v + 2 * c] = f.x; x[16 * v + 2 * c + 1] = f.y;
          }
        }
      } else {
        const uint4* src = reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(p.q) + at);
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          const uint4 raw = src[v];
          const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            x[8 * v + 2 * c] = __uint_as_float(w[c] << 16); x[8 * v + 2 * c + 1] = __uint_as_float(w[c] & 0xffff0000u);
          }
        }
      }
      float top = 0.f;
#pragma unroll
      for (int c = 0; c < 32; ++c) top = fmaxf(top, fabsf(x[c]));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      // exponent of the largest element; a row of zeros or with an infinity is taken as it is
      int e = static_cast<int>(__float_as_uint(top) >> 23) - 127 - 14;
      if (top == 0.f || !(top < INFINITY)) e = 0;
      e = max(e, -126);                                      // 2^-e is a normal number
      const float up = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
#pragma unroll
      for (int c = 0; c < 16; ++c) qf[n][c] = pack2<true>(x[2 * c] * up, x[2 * c + 1] * up);
      const float back = scale * __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
      // this thread's columns of S^T are rows 8 n + 2 t4 and the next one
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        fac[n][c] = __shfl_sync(0xffffffffu, back, 4 * (2 * t4 + c));
        limit[n][c] = lim(8 * n + 2 * t4 + c);
      }
    }
    const uint32_t k_code = 64 * (32 * warp + key_at(g)) + 16 * t4;
    const uint32_t k_scale = kKv4ScaleOffset + 8 * (32 * warp + key_at(g)) + 2 * t4;
    const int v_key[2] = {32 * warp + key_at(2 * t4), 32 * warp + key_at(2 * t4 + 1)};

    int stage = 0;
    uint32_t phase = 0;
    while (true) {
      if (!mbar_wait_warp(full(stage), phase, abort_flag)) break;
      const int key0 = s_key[stage];
      if (key0 < 0) break;
      const uint32_t kt = base + stage * kStageBytes, vt = kt + kKv4TileBytes;
      // ---- S^T: two steps of 16 keys ----
      float s[2][NT][4];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int c = 0; c < 4; ++c) s[u][n][c] = 0.f;
        uint4 code[2];
        uint32_t sc[2][2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          code[r] = lds128(kt + k_code + 64 * (16 * u + 8 * r));
          const uint32_t both = kv4_scales_to_half(static_cast<uint16_t>(lds16(kt + k_scale + 8 * (16 * u + 8 * r))));
          sc[r][0] = __byte_perm(both, 0, 0x1010);
          sc[r][1] = __byte_perm(both, 0, 0x3232);
        }
        const uint32_t w0[4] = {code[0].x, code[0].y, code[0].z, code[0].w}, w1[4] = {code[1].x, code[1].y, code[1].z, code[1].w};
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t a[4], b[4];
          kv4_to_half(w0[c], a);
          kv4_to_half(w1[c], b);
#pragma unroll
          for (int i = 0; i < 4; ++i) { a[i] = half2_mul(a[i], sc[0][c >> 1]); b[i] = half2_mul(b[i], sc[1][c >> 1]); }
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            mma_f16(s[u][n], a[0], b[0], a[1], b[1], qf[n][4 * c], qf[n][4 * c + 1]);
            mma_f16(s[u][n], a[2], b[2], a[3], b[3], qf[n][4 * c + 2], qf[n][4 * c + 3]);
          }
        }
      }
      // ---- softmax: exponents, mask, maximum that may lag ----
      bool raise = false;
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int c = 0; c < 4; ++c) s[u][n][c] *= fac[n][c & 1];
      if (key0 + kKvTile > lim_first) {
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int c = 0; c < 4; ++c)
              if (key0 + 32 * warp + 16 * u + 8 * (c >> 1) + key_at(g) >= limit[n][c & 1]) s[u][n][c] = -INFINITY;
      }
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int c = 0; c < 4; ++c) raise |= s[u][n][c] > m[n][c & 1] + kRescale;
      if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float top = fmaxf(fmaxf(s[0][n][c], s[0][n][c + 2]), fmaxf(s[1][n][c], s[1][n][c + 2]));
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
            top = fmaxf(top, m[n][c]);
            const float keep = top == -INFINITY ? 1.f : exp2_fast(m[n][c] - top);
            m[n][c] = top;
            l_round[n][c] *= keep; l_sum[n][c] *= keep;
#pragma unroll
            for (int i = 0; i < 8; ++i) { o[i][n][c] *= keep; o[i][n][c + 2] *= keep; }
          }
      }
      uint32_t pt[2][NT][2];                                 // P^T as an operand: [step][rows][keys 0-7, keys 8-15]
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float shift[2];
#pragma unroll
        for (int c = 0; c < 2; ++c) shift[c] = m[n][c] == -INFINITY ? 0.f : m[n][c] - kPOffset;
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float p0 = exp2_fast(s[u][n][2 * h] - shift[0]), p1 = exp2_fast(s[u][n][2 * h + 1] - shift[1]);
            const uint32_t pk = pack2<true>(p0, p1);
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&pk));
            l_sum[n][0] += p0; l_sum[n][1] += p1;
            l_round[n][0] += f.x; l_round[n][1] += f.y;
            pt[u][n][h] = transpose8x8(pk);
          }
      }
      // ---- O^T ----
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        uint2 code[4];
        uint32_t sb[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int key = v_key[r & 1] + 16 * u + 8 * (r >> 1);
          code[r] = lds64(vt + 64 * key + 8 * g);
          sb[r] = lds8(vt + kKv4ScaleOffset + 8 * key + g);
          if (key0 + key >= it.kv_len) sb[r] = 0;            // nobody wrote there: a scale may be NaN, and 0 x NaN is not 0
        }
        const uint32_t s01 = kv4_scales_to_half(static_cast<uint16_t>(sb[0] | (sb[1] << 8)));
        const uint32_t s23 = kv4_scales_to_half(static_cast<uint16_t>(sb[2] | (sb[3] << 8)));
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          uint32_t x[4][4];
#pragma unroll
          for (int r = 0; r < 4; ++r) kv4_to_half(w ? code[r].y : code[r].x, x[r]);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t a0 = half2_mul(__byte_perm(x[0][i], x[1][i], 0x5410), s01);
            const uint32_t a1 = half2_mul(__byte_perm(x[0][i], x[1][i], 0x7632), s01);
            const uint32_t a2 = half2_mul(__byte_perm(x[2][i], x[3][i], 0x5410), s23);
            const uint32_t a3 = half2_mul(__byte_perm(x[2][i], x[3][i], 0x7632), s23);
#pragma unroll
            for (int n = 0; n < NT; ++n) mma_f16(o[4 * w + i][n], a0, a1, a2, a3, pt[u][n][0], pt[u][n][1]);
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(empty(stage));
      if (++stage == kStages) { stage = 0; phase ^= 1; }
    }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) {
          l_round[n][c] += __shfl_xor_sync(0xffffffffu, l_round[n][c], d);
          l_sum[n][c] += __shfl_xor_sync(0xffffffffu, l_sum[n][c], d);
        }
  }
  __syncthreads();                                           // the ring is no longer read, and no copy is on its way
  if (*abort_flag) {
    outlast_async_work();
    if (threadIdx.x == 0 && p.status) *p.status = MSA_STATUS_TIMEOUT;
    return;
  }
  // ---------------- the four states of a row become one ----------------
  float* s_o = reinterpret_cast<float*>(smem);               // [warp][row][kLdO]
  float* s_m = s_o + kWarps * 8 * NT * kLdO;                 // [warp][row][3]: maximum, sum of rounded P, sum of P
  static_assert((kWarps * 16 * (kLdO + 3)) * 4 <= kStages * kStageBytes, "states fit the ring");
  if (warp < kWarps) {
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int r = warp * 8 * NT + 8 * n + 2 * t4 + c;
#pragma unroll
        for (int i = 0; i < 8; i += 2)
          *reinterpret_cast<float4*>(s_o + r * kLdO + 16 * g + 2 * i) = make_float4(o[i][n][c], o[i][n][c + 2], o[i + 1][n][c], o[i + 1][n][c + 2]);
        if (g == 0) { s_m[3 * r] = m[n][c]; s_m[3 * r + 1] = l_round[n][c]; s_m[3 * r + 2] = l_sum[n][c]; }
      }
  }
  __syncthreads();
  if (warp == kWarps) return;
  // 16 threads a row, 8 columns each
  const int c16 = threadIdx.x & 15;
#pragma unroll
  for (int r0 = 0; r0 < 8 * NT; r0 += 8) {
    const int r = r0 + (threadIdx.x >> 4);
    if (r >= it.nrows) continue;
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) top = fmaxf(top, s_m[3 * (w * 8 * NT + r)]);
    float sum = 0.f, total = 0.f, acc[8];
#pragma unroll
    for (int c = 0; c < 8; ++c) acc[c] = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const int at = w * 8 * NT + r;
      const float mw = s_m[3 * at];
      // a warp that saw no number has weight 0, unless what it saw was NaN
      const float f = mw == -INFINITY ? (s_m[3 * at + 1] == 0.f ? 0.f : s_m[3 * at + 1]) : exp2_fast(mw - top);
      sum += f * s_m[3 * at + 1];
      total += f * s_m[3 * at + 2];
#pragma unroll
      for (int c = 0; c < 8; ++c) acc[c] += f * s_o[at * kLdO + 8 * c16 + c];
    }
    const int row = it.row0 + r;
    const int64_t tok = it.qo_base + it.tok0 + row / it.pack;
    const int head = it.head0 + row % it.pack;
    const bool none = sum == 0.f;
    const float vs = p.v_scale_head ? p.v_scale_head[it.kvh] : 1.f;
    const float inv = none ? 0.f : vs / sum;
    const float lse = none ? -INFINITY : ((top == -INFINITY ? 0.f : top) - kPOffset + log2f(total)) * kLn2;
    if (p.partial_o) {
      const int64_t at = (static_cast<int64_t>(it.split) * p.total_q + tok) * p.num_qo_heads + head;
      float* dst = p.partial_o + at * kHeadDim + 8 * c16;
      *reinterpret_cast<float4*>(dst) = make_float4(acc[0] * inv, acc[1] * inv, acc[2] * inv, acc[3] * inv);
      *reinterpret_cast<float4*>(dst + 4) = make_float4(acc[4] * inv, acc[5] * inv, acc[6] * inv, acc[7] * inv);
      if (c16 == 0) p.partial_lse[at] = lse;
    } else {
      const float f = inv * p.out_scale;
      const uint4 pk = make_uint4(pack2<false>(acc[0] * f, acc[1] * f), pack2<false>(acc[2] * f, acc[3] * f),
                                  pack2<false>(acc[4] * f, acc[5] * f), pack2<false>(acc[6] * f, acc[7] * f));
      *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(p.out) + tok * p.out_stride_tok + head * p.out_stride_head + 8 * c16) = pk;
      if (p.lse && c16 == 0) p.lse[tok * p.num_qo_heads + head] = lse;
    }
  }
}

template <int NT>
int launch(const MsaFmhaParams& p, int rows, cudaStream_t stream) {
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess) return MSA_ERR_LAUNCH;
  static bool ready[64] = {};
  if (device < 0 || device >= 64 || !ready[device]) {
    if (cudaFuncSetAttribute(kv4_decode_kernel<NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes) != cudaSuccess) return MSA_ERR_LAUNCH;
    if (device >= 0 && device < 64) ready[device] = true;
  }
  const int64_t items = (p.flags & MSA_FLAG_SPARSE) ? static_cast<int64_t>(p.total_q) * p.num_kv_heads * p.num_splits : p.num_work;
  if (items > 0x7fffffffLL) return MSA_ERR_TOO_LARGE;
  if (items == 0) return MSA_OK;
  const dim3 grid(static_cast<unsigned>(items), (rows + 8 * NT - 1) / (8 * NT));
  return launch_chained(kv4_decode_kernel<NT>, grid, kThreads, kSmemBytes, stream, p) == cudaSuccess ? MSA_OK : MSA_ERR_LAUNCH;
}

}  // namespace
}  // namespace kv4

// Checks of the fields that the 4-bit pass reads, and the launch.  Nothing here touches the device before the checks are through.
int fmha_kv4_fwd(const MsaFmhaParams& p, cudaStream_t stream) {
  const bool sparse = (p.flags & MSA_FLAG_SPARSE) != 0;
  if (!(p.flags & MSA_FLAG_OUT_O)) return (p.flags & MSA_FLAG_OUT_SCORE) ? MSA_ERR_UNSUPPORTED : MSA_ERR_BAD_ARG;
  if (p.flags & MSA_FLAG_OUT_SCORE) return MSA_ERR_UNSUPPORTED;
  if (!p.q || !p.k || !p.v || !p.qo_start || !p.kv_len || !p.qo_offset || !p.kv_page_indptr || !p.kv_indices) return MSA_ERR_BAD_ARG;
  if (p.total_q < 0 || p.batch < 0 || p.kv_extent < 0 || (!p.out && !p.partial_o)) return MSA_ERR_BAD_ARG;
  if (p.partial_o ? (!p.partial_lse || p.num_splits < 1) : p.num_splits != 1) return MSA_ERR_BAD_ARG;
  if (p.num_qo_heads <= 0 || p.num_kv_heads <= 0 || p.num_qo_heads % p.num_kv_heads) return MSA_ERR_BAD_ARG;
  const int h_r = p.num_qo_heads / p.num_kv_heads;
  if (p.pack < 1 || h_r % p.pack) return MSA_ERR_BAD_ARG;
  if (p.page_size != kKvTile) return MSA_ERR_UNSUPPORTED;
  if (p.q_dtype != MSA_DT_BF16 && p.q_dtype != MSA_DT_E4M3) return MSA_ERR_UNSUPPORTED;
  int rows;
  if (sparse) {
    if (!p.kv_block_indexes || !p.token_batch || p.kv_block_num <= 0 || p.pack != h_r) return MSA_ERR_BAD_ARG;
    rows = h_r;
  } else {
    if (p.num_work < 0 || (p.num_work > 0 && !p.work)) return MSA_ERR_BAD_ARG;
    if (p.block_m != 16 && p.block_m != 64 && p.block_m != 128) return MSA_ERR_UNSUPPORTED;
    if (p.pack > p.block_m) return MSA_ERR_BAD_ARG;
    rows = p.decode_rows > 0 ? std::min(p.decode_rows, p.block_m) : p.block_m;
  }
  auto al = [](const void* ptr) { return (reinterpret_cast<uintptr_t>(ptr) & 15) == 0; };
  const int qe = p.q_dtype == MSA_DT_E4M3 ? 1 : 2;
  if (!al(p.q) || !al(p.k) || !al(p.v) || !al(p.out) || !al(p.partial_o)) return MSA_ERR_BAD_ARG;
  if ((p.q_stride_tok * qe) % 16 || (p.q_stride_head * qe) % 16 || p.k_stride_page % 16 || p.k_stride_head % 16 || p.v_stride_page % 16 ||
      p.v_stride_head % 16 || (p.out && ((p.out_stride_tok * 2) % 16 || (p.out_stride_head * 2) % 16)))
    return MSA_ERR_BAD_ARG;
  if (p.total_q == 0 || p.kv_extent == 0) return p.total_q == 0 ? MSA_OK : MSA_ERR_BAD_ARG;
  return rows <= 8 ? kv4::launch<1>(p, rows, stream) : kv4::launch<2>(p, rows, stream);
}
}  // namespace msa
