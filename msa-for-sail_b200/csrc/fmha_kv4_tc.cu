// Attention of 17 to 128 query rows over a cache held in 4 bits (layout in kv4.cuh): several tokens of a sequence, or many heads.
//
// With so many rows to a KV head the products outgrow mma.sync, and the conversion of a page should be shared by all of them.  One CTA =
// one work item; its packed rows are the rows of a 128-row MMA tile.
//
//   warps 0-3    softmax and epilogue: thread r owns row r; at first they convert Q into TMEM.  With at most 128 / F rows (F = 2, 4) the rows stand
//                F times in the tile, and copy f has keys 128 / F * f .. of every page, with a maximum and a sum of its own and zeros in
//                P elsewhere: all four warps work on a page (32 sequences x 4 tokens x 16 heads: 94 us with half of the threads idle).
//                The F states of a row are joined at the end
//   warp 4       issues S[j & 1] = Q K_j^T (tcgen05, f16 operands, Q and accumulators in TMEM; Q in shared memory costs 1.4 us more
//                of 32 sequences x 4 tokens x 64 heads)
//   warp 5       issues O += P_j V_j (P from TMEM).  (One warp for both took 2 150 clocks a page: 1 350 to issue, which is what
//                the tensor pipe takes, and 250 for each of three waits, ready or not.)
//   warps 8-23   conversion, eight warps for K and eight for V: warp w has keys 16 w .. 16 w + 15 of every page.  16-byte copies bring
//                codes and scales into a ring of the warp's own, three pages deep; converted rows go to the 128-byte-swizzled
//                tiles of K and V (two each), which the MMAs read.  (Eight warps in all took 2 100 clocks a page, of which each wait
//                for a tile and each fence between the proxies was 200.)
//
// Registers move from the converting warpgroups to the softmax one (setmaxnreg).
//
// Numbers as in fmha_kv4.cu: codes times scales are exact in f16, Q rows are scaled by a power of two, P = 2^(x - m + 7) with a maximum that
// lags by at most 8.
//
// A page costs 64 KB written to shared memory and as much read by the MMAs, about 1 000 clocks of its bandwidth, 500 clocks of conversions
// per scheduler, and with 128 rows 1 000 clocks of exponentials; its 18 KB from memory are 810.  Measured: 32 sequences of 131 to
// 16 384 keys x 4 tokens, 64 / 4 heads, 64 rows to a head: 67 us and 4 for the merge, 2 100 clocks a page (149 us in groups of 16 rows on
// fmha_kv4.cu, which convert every page four times); with 128 rows 2 600, with 32 rows 1 900.  From 64 rows on the softmax
// warpgroup bounds it, which is never without work: 550 clocks to read S, take the maximum and vote, 1 100 for exponentials and P; below that the
// converting warps: 600 clocks to read codes and order more, 400 for a free tile, 650 to convert and fence.  Two softmax warpgroups that take
// turns (one buffer of S each, or registers run out), one warp that hands over K and V together, a fourth page on its way: slower or no gain.
// Every wait is bounded (tc_ptx.cuh).
#include <algorithm>

#include "kv4.cuh"
#include "nvtx_range.h"
#include "tc_ptx.cuh"

namespace msa {
namespace kv4_tc {
namespace {

using namespace tc;

constexpr int BM = 128, BN = 128;
constexpr int SUB_BYTES = BM * 128;                          // one [128 rows][64 f16] swizzled sub-tile
constexpr int TILE_BYTES = 2 * SUB_BYTES;
constexpr int MMA_WARP = 4, PV_WARP = 5, CONVERT_WARP0 = 8, CONVERT_WARPS = 8;       // of K; as many of V follow
constexpr int NTHREADS = 32 * (CONVERT_WARP0 + 2 * CONVERT_WARPS);
// What the launch allocates (threads x compiled registers) must cover the registers after the moves, or the increase never
// completes: the launcher checks it.
constexpr int REGS_SOFTMAX = 208, REGS_MMA = 40, REGS_CONVERT = 56;
constexpr int REGS_NEEDED = 128 * (REGS_SOFTMAX + REGS_MMA + 4 * REGS_CONVERT);
static_assert(NTHREADS == 6 * 128, "warpgroups");
constexpr int STAGES = 2;                                    // tiles of K and of V
constexpr int RING = 3;                                      // pages on their way
constexpr int KEYS = BN / CONVERT_WARPS;                     // of a page that a warp converts
constexpr int CODE_BYTES = KEYS * kKv4CodeBytes, SCALE_BYTES = KEYS * kKv4ScaleBytes;
constexpr int HALF = CODE_BYTES + SCALE_BYTES;               // of a warp's keys

constexpr int OFF_K = 0;
constexpr int OFF_V = OFF_K + STAGES * TILE_BYTES;
constexpr int OFF_RING = OFF_V + STAGES * TILE_BYTES;
constexpr int OFF_BAR = OFF_RING + 2 * CONVERT_WARPS * RING * HALF;
enum Bar { Q_FULL = 0, K_FULL = 1, K_EMPTY = 3, V_FULL = 5, V_EMPTY = 7, S_FULL = 9, P_FULL = 11, O_DONE = 13, NUM_BARS = 14 };
constexpr int OFF_NAN = OFF_BAR + NUM_BARS * 8 + 16;          // per 16 elements of V: first key with a NaN that not all rows see
constexpr int SMEM_BYTES = OFF_NAN + 32 + 1024;           // + slack to align the base to 1 KB
static_assert(SMEM_BYTES <= 227 * 1024 && HALF % 16 == 0 && OFF_BAR % 16 == 0, "shared memory");
constexpr int TMEM_COLS = 512, O_COL = 256, Q_COL = 384;        // S twice, O, Q
constexpr float kPOffset = 7.f, kRescale = 8.f, kNoMax = -3e38f;

// kind::f16 with f16 operands and f32 accumulation
constexpr uint32_t idesc_f16(int m, int n, bool b_mn_major) {
  return (1u << 4) | (static_cast<uint32_t>(b_mn_major) << 16) | (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24);
}
// 16-byte chunk c (0..15) of row r of a tile
__device__ __forceinline__ int tile_at(int r, int c) { return (c >> 3) * SUB_BYTES + r * 128 + (((c & 7) ^ (r & 7)) << 4); }
// 16-byte chunk q (0..3) of row r of the codes in a warp's ring: eight rows' chunks q fall into different banks
__device__ __forceinline__ int code_at(int r, int q) { return r * kKv4CodeBytes + ((q ^ ((r >> 1) & 3)) << 4); }

__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}

template <int F>
__global__ void __launch_bounds__(NTHREADS, 1) kv4_tc_kernel(const __grid_constant__ MsaFmhaParams p) {
  extern __shared__ unsigned char smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  unsigned char* smem = smem_raw + (base - smem_u32(smem_raw));
  const uint32_t bars = base + OFF_BAR;
  auto bar = [&](int i) -> uint32_t { return bars + 8u * i; };
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + OFF_BAR + NUM_BARS * 8);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + OFF_BAR + NUM_BARS * 8 + 4);
  volatile int* skip_flag = abort_flag + 1;
  int* const nan_key = reinterpret_cast<int*>(smem + OFF_NAN);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  // ---------------- the item ----------------
  const MsaWorkItem w = p.work[blockIdx.x];
  const int b = chk(w.batch, 0, p.batch, p.status), head0 = chk(w.head0, 0, p.num_qo_heads, p.status), split = chk(w.split, 0, p.num_splits, p.status);
  constexpr int ROWS = BM / F, COLS = BN / F;                // rows of a copy, keys of a page that one has
  const int nrows = min(w.num_rows, ROWS);
  if (nrows <= 0) return;
  const int G = p.pack, kvh = head0 / (p.num_qo_heads / p.num_kv_heads);
  const int qo_base = p.qo_start[b], kv_len = p.kv_len[b], off = min(p.qo_offset[b], kv_len), page_base = p.kv_page_indptr[b];
  // row r sees keys below lim(r), which grows with r
  auto lim = [&](int r) -> int { return min(kv_len, (w.row0 + r) / G + off + 1); };
  const int lim_first = lim(0), lim_last = lim(nrows - 1);
  const int first = w.kv_tile_begin;
  // (none where the table is empty: the conversion then has nothing to read)
  const int n_tiles = p.num_logical_pages <= 0 ? 0 : max(0, min(w.kv_tile_end, (lim_last + BN - 1) / BN) - first);
  const int n_active = F == 1 ? (nrows + 31) / 32 : 4;       // warps that have rows

  // a timeout reported earlier on this device (status word not cleared yet): do not start
  if (threadIdx.x == NTHREADS - 1)
    *skip_flag = (p.status != nullptr && *reinterpret_cast<const volatile int32_t*>(p.status) != 0) ? 1 : 0;
  if (threadIdx.x == 0) {
    mbar_init(bar(Q_FULL), 32 * n_active);
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(bar(K_FULL + s), CONVERT_WARPS); mbar_init(bar(K_EMPTY + s), 1);
      mbar_init(bar(V_FULL + s), CONVERT_WARPS); mbar_init(bar(V_EMPTY + s), 1);
      mbar_init(bar(S_FULL + s), 1); mbar_init(bar(P_FULL + s), 32 * n_active);
    }
    mbar_init(bar(O_DONE), 1);
    *abort_flag = 0;
    for (int i = 0; i < 8; ++i) nan_key[i] = 0x7fffffff;
    mbar_fence_init();
  }
  if (warp == MMA_WARP) {
    tmem_alloc(smem_u32(tmem_slot), TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (*skip_flag != 0) {
    // nothing: fall through to the teardown
  } else if (warp >= CONVERT_WARP0) {
    // =========================== conversion ===========================
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS_CONVERT));
    const int cw = (warp - CONVERT_WARP0) % CONVERT_WARPS;
    const bool is_v = warp >= CONVERT_WARP0 + CONVERT_WARPS;
    unsigned char* ring = smem + OFF_RING + (warp - CONVERT_WARP0) * RING * HALF;
    const unsigned char* const cache = (is_v ? static_cast<const unsigned char*>(p.v) + kvh * p.v_stride_head
                                             : static_cast<const unsigned char*>(p.k) + kvh * p.k_stride_head) + 16 * lane;
    const int64_t stride = is_v ? p.v_stride_page : p.k_stride_page;
    auto physical = [&](int j) -> int {
      if (j >= n_tiles) return 0;
      const int at = min(chk(page_base + first + j, 0, p.num_logical_pages, p.status), p.num_logical_pages - 1);
      return min(max(chk(p.kv_indices[at], 0, static_cast<int>(p.kv_extent), p.status), 0), static_cast<int>(p.kv_extent) - 1);
    };
    int phys = physical(lane), next = physical(32 + lane);   // page-table entries, one a lane
    const uint32_t code_dst = smem_u32(ring) + code_at(lane >> 2, lane & 3), scale_dst = smem_u32(ring) + CODE_BYTES + 16 * lane;
    static_assert(CODE_BYTES == 1024 && SCALE_BYTES == 128, "two copies of 16 bytes a lane, and one of the first eight lanes");
    auto fetch = [&](int j, int place) {                     // page j into a place of the ring that no lane reads any more
      if (j > 0 && (j & 31) == 0) { phys = next; next = physical(j + 32 + lane); }
      const int64_t page = __shfl_sync(0xffffffffu, phys, j & 31);
      const unsigned char* src = cache + page * stride;
      copy16(code_dst + place * HALF, src + cw * CODE_BYTES);
      copy16(code_dst + place * HALF + 512, src + cw * CODE_BYTES + 512);       // eight rows on: the same place within the row
      if (lane < 8) copy16(scale_dst + place * HALF, src + kKv4ScaleOffset + cw * SCALE_BYTES);
    };
#pragma unroll
    for (int j = 0; j < RING; ++j) {
      if (j < n_tiles) fetch(j, j);
      cp_async_commit();
    }
    const int r8 = lane & 7, q = lane >> 3;                  // rows r8 and 8 + r8 of this warp's keys, elements 32 q .. 32 q + 31
    unsigned char* const tiles = smem + (is_v ? OFF_V : OFF_K);
    const int full = is_v ? V_FULL : K_FULL, empty = is_v ? V_EMPTY : K_EMPTY;
    int place = 0;
    for (int j = 0; j < n_tiles; ++j) {
      const int st = j % STAGES;
      cp_async_wait<RING - 1>();
      __syncwarp();
      uint4 code[KEYS / 8];
      uint32_t scale[KEYS / 8];
      const int key0 = (first + j) * BN + cw * KEYS + r8;
#pragma unroll
      for (int i = 0; i < KEYS / 8; ++i) {
        const unsigned char* src = ring + place * HALF;
        code[i] = *reinterpret_cast<const uint4*>(src + code_at(8 * i + r8, q));
        scale[i] = *reinterpret_cast<const uint16_t*>(src + CODE_BYTES + (8 * i + r8) * kKv4ScaleBytes + 2 * q);
        // P is 0 where a row does not see a key, but 0 x NaN is not.  Behind the last row's keys, where maybe nobody wrote, V becomes
        // zero; a NaN that some of the rows see is taken out, and they get it at the end.
        if (is_v && key0 + 8 * i >= lim_first) {
          if (key0 + 8 * i >= lim_last) scale[i] = 0;
#pragma unroll
          for (int h = 0; h < 2; ++h)
            if ((scale[i] >> (8 * h) & 0x7f) == 0x7f) {
              atomicMin(nan_key + 2 * q + h, key0 + 8 * i);  // a minimum: the order does not matter
              scale[i] &= ~(0xffu << (8 * h));
            }
        }
      }
      __syncwarp();                                          // all lanes have read this place of the ring
      if (j + RING < n_tiles) fetch(j + RING, place);
      cp_async_commit();                                     // an empty group at the end: the wait above counts groups
      if (++place == RING) place = 0;
      if (!mbar_wait_warp(bar(empty + st), ((j / STAGES) & 1) ^ 1, abort_flag)) break;
      unsigned char* tile = tiles + st * TILE_BYTES;
#pragma unroll
      for (int i = 0; i < KEYS / 8; ++i) {
        const uint32_t both = kv4_scales_to_half(static_cast<uint16_t>(scale[i]));
        const uint32_t words[4] = {code[i].x, code[i].y, code[i].z, code[i].w};
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t h[4];
          kv4_to_half(words[c], h);
          const uint32_t s = __byte_perm(both, 0, c < 2 ? 0x1010 : 0x3232);
#pragma unroll
          for (int e = 0; e < 4; ++e) h[e] = half2_mul(h[e], s);
          *reinterpret_cast<uint4*>(tile + tile_at(cw * KEYS + 8 * i + r8, 4 * q + c)) = make_uint4(h[0], h[1], h[2], h[3]);
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(full + st));
    }
    cp_async_wait<0>();                                      // nothing is on its way when the CTA ends
  } else if (warp >= MMA_WARP) {
    // =========================== MMA issuers ===========================
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS_MMA));
    const uint64_t dk_hi = smem_desc(0, 16, 1024) & 0xFFFFFFFFFFFF0000ull;
    const uint64_t dv_hi = smem_desc(0, SUB_BYTES, 1024) & 0xFFFFFFFFFFFF0000ull;
    if (warp == MMA_WARP) {
      constexpr uint32_t IDESC_QK = idesc_f16(BM, BN, false);
      bool alive = n_tiles > 0 && mbar_wait_warp(bar(Q_FULL), 0, abort_flag);
      tc_fence_after();
      for (int j = 0; j < n_tiles && alive; ++j) {
        const int st = j % STAGES;
        // V_EMPTY: P_{j-2} V_{j-2} is done, which read P from this buffer of S
        alive = mbar_wait_warp(bar(K_FULL + st), (j / STAGES) & 1, abort_flag);
        if (alive) alive = mbar_wait_warp(bar(V_EMPTY + st), ((j / STAGES) & 1) ^ 1, abort_flag);
        if (!alive) break;
        tc_fence_after();
        if (elect_one()) {
          const uint32_t ka = (base + OFF_K + st * TILE_BYTES) >> 4;
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const uint32_t o = ((k >> 2) * SUB_BYTES + (k & 3) * 32) >> 4;
            mma_ts(tmem + st * BN, tmem + Q_COL + k * 8, dk_hi | ((ka + o) & 0x3FFF), IDESC_QK, k > 0);
          }
          mma_commit(bar(S_FULL + st));
          mma_commit(bar(K_EMPTY + st));
        }
        __syncwarp();
      }
    } else if (warp == PV_WARP) {
      constexpr uint32_t IDESC_PV = idesc_f16(BM, kHeadDim, true);
      bool alive = true;
      for (int j = 0; j < n_tiles && alive; ++j) {
        const int st = j % STAGES;
        alive = mbar_wait_warp(bar(V_FULL + st), (j / STAGES) & 1, abort_flag);
        if (alive) alive = mbar_wait_warp(bar(P_FULL + st), (j / STAGES) & 1, abort_flag);
        if (!alive) break;
        tc_fence_after();
        if (elect_one()) {
          const uint32_t va = (base + OFF_V + st * TILE_BYTES) >> 4;
#pragma unroll
          for (int k = 0; k < 8; ++k)
            mma_ts(tmem + O_COL, tmem + st * BN + k * 8, dv_hi | ((va + k * (16 * 128 >> 4)) & 0x3FFF), IDESC_PV, (j > 0 || k > 0) ? 1u : 0u);
          mma_commit(bar(V_EMPTY + st));
          if (j == n_tiles - 1) mma_commit(bar(O_DONE));
        }
        __syncwarp();
      }
    }
  } else {
    // =========================== softmax / epilogue ===========================
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REGS_SOFTMAX));
    if (warp < n_active) {
      const int trow = (warp << 5) | lane;                     // row of the tile, TMEM lane
      const int r = trow % ROWS, part = trow / ROWS;           // row of the item, copy
      const uint32_t lane_addr = static_cast<uint32_t>(warp << 5) << 16;
      const uint32_t tO = tmem + O_COL + lane_addr;
      const bool row_ok = r < nrows;
      const int row = w.row0 + min(r, nrows - 1);
      const int64_t tok = qo_base + row / G;
      const int head = head0 + row % G;
      const int limit = lim(min(r, nrows - 1));
      float fac = 1.f;
      {
        const float scale = p.sm_scale * (p.k_scale_head ? p.k_scale_head[kvh] : 1.f) * kLog2e;
        const int64_t at = tok * p.q_stride_tok + head * p.q_stride_head;
        const bool e4m3 = p.q_dtype == MSA_DT_E4M3;
        auto load8 = [&](int c, float (&x)[8]) {               // elements 8 c .. 8 c + 7
          if (e4m3) {
            const uint2 raw = *reinterpret_cast<const uint2*>(static_cast<const unsigned char*>(p.q) + at + 8 * c);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint32_t h = kv4_scales_to_half(static_cast<uint16_t>((i < 2 ? raw.x : raw.y) >> (16 * (i & 1))));
              const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
              x[2 * i] = f.x; x[2 * i + 1] = f.y;
            }
          } else {
            const uint4 raw = *reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(p.q) + at + 8 * c);
            const uint32_t v[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) { x[2 * i] = __uint_as_float(v[i] << 16); x[2 * i + 1] = __uint_as_float(v[i] & 0xffff0000u); }
          }
        };
        float top = 0.f;
#pragma unroll 4
        for (int c = 0; c < 16; ++c) {
          float x[8];
          load8(c, x);
#pragma unroll
          for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(x[i]));
        }
        // exponent of the largest element; a row of zeros or with an infinity is taken as it is.  The factor of the scores is made
        // positive (its sign goes to Q), so that the largest score has the largest exponent.
        int e = static_cast<int>(__float_as_uint(top) >> 23) - 127 - 14;
        if (top == 0.f || !(top < INFINITY)) e = 0;
        e = max(e, -126);
        const float up = copysignf(scale == 0.f ? 0.f : __uint_as_float(static_cast<uint32_t>(127 - e) << 23), scale);
        if (scale != 0.f) fac = fabsf(scale) * __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t pk[16];
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            float x[8];
            load8(4 * i + c, x);
#pragma unroll
            for (int e = 0; e < 4; ++e) pk[4 * c + e] = pack2<true>(x[2 * e] * up, x[2 * e + 1] * up);
          }
          tmem_st16(tmem + Q_COL + 16 * i + lane_addr, pk);
        }
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(bar(Q_FULL));
      }
      float m = kNoMax, l = 0.f;                               // maximum - kPOffset, sum of P
      bool alive = true;
      for (int j = 0; j < n_tiles && alive; ++j) {
        const uint32_t tS = tmem + (j & 1) * BN + lane_addr;
        alive = mbar_wait_warp(bar(S_FULL + j % STAGES), (j / STAGES) & 1, abort_flag);
        if (!alive) break;
        tc_fence_after();
        const int key0 = (first + j) * BN + part * COLS;       // of this thread
        const bool edge = (first + j) * BN + BN > lim_first;
        constexpr int CH = COLS / 32;
        uint32_t sv[CH][32];
#pragma unroll
        for (int c = 0; c < CH; ++c) tmem_ld32(tS + part * COLS + 32 * c, sv[c]);
        tmem_wait_ld();
        if (edge) {
#pragma unroll
          for (int c = 0; c < CH; ++c)
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (key0 + 32 * c + e >= limit) sv[c][e] = 0xff800000u;
        }
        float top = -INFINITY, t2 = -INFINITY;
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
          for (int e = 0; e < 32; e += 4) {
            top = max3(top, __uint_as_float(sv[c][e]), __uint_as_float(sv[c][e + 1]));
            t2 = max3(t2, __uint_as_float(sv[c][e + 2]), __uint_as_float(sv[c][e + 3]));
          }
        top = fmaxf(top, t2) * fac;
        const bool raise = top > m + (kPOffset + kRescale);
        if (__any_sync(0xffffffffu, raise)) {
          const float now = raise ? top - kPOffset : m;
          const float keep = exp2_fast(m - now);
          m = now;
          l *= keep;
          if (j > 0) {                                         // O may still be the target of P_{j-1} V_{j-1}
            // (V_EMPTY of tile j - 3 was seen before S_{j-1} was computed: the phase is this one)
            alive = mbar_wait_warp(bar(V_EMPTY + (j - 1) % STAGES), ((j - 1) / STAGES) & 1, abort_flag);
            if (!alive) break;
            tc_fence_after();
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              uint32_t v[32];
              tmem_ld32(tO + c * 32, v);
              tmem_wait_ld();
#pragma unroll
              for (int e = 0; e < 32; ++e) v[e] = __float_as_uint(__uint_as_float(v[e]) * keep);
              tmem_st32(tO + c * 32, v);
            }
          }
        }
        const uint64_t f2 = f2_pack(fac, fac), shift = f2_pack(-m, -m);
        uint64_t l2 = 0;
#pragma unroll
        for (int c = 0; c < CH; ++c) {                         // P overwrites the first half of S
          uint32_t pk[16];
          const uint32_t (&x)[32] = sv[c];
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            float x0, x1;
            f2_unpack(f2_fma(f2_pack(__uint_as_float(x[e]), __uint_as_float(x[e + 1])), f2, shift), x0, x1);
            const float p0 = exp2_fast(x0), p1 = exp2_fast(x1);
            l2 = f2_add(l2, f2_pack(p0, p1));
            pk[e >> 1] = pack2<true>(p0, p1);
          }
          tmem_st16(tS + part * (COLS / 2) + c * 16, pk);
        }
        if constexpr (F > 1) {                                 // the keys of the other copies
          uint32_t zero[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) zero[e] = 0u;
#pragma unroll
          for (int c = 0; c < 4; ++c)
            if (c / CH != part) tmem_st16(tS + c * 16, zero);
        }
        float la, lb;
        f2_unpack(l2, la, lb);
        l += la + lb;
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(bar(P_FULL + j % STAGES));
      }
      // ---- epilogue ----
      if (alive && n_tiles > 0) alive = mbar_wait_warp(bar(O_DONE), 0, abort_flag);
      // (it has completed: the wait makes what the converting warps wrote into nan_key visible)
      if (alive && n_tiles > 0) alive = mbar_wait_warp(bar(V_FULL + (n_tiles - 1) % STAGES), ((n_tiles - 1) / STAGES) & 1, abort_flag);
      const float vs = p.v_scale_head ? p.v_scale_head[kvh] : 1.f;
      const int64_t prow = (static_cast<int64_t>(split) * p.total_q + tok) * p.num_qo_heads + head;
      // columns c0 .. c0 + 7 of a row of the result; tok_, head_, prow_: the row
      auto store8 = [&](const float (&v)[8], int c0, int64_t tok_, int head_, int64_t prow_) {
        if (p.partial_o) {
          float* dst = p.partial_o + prow_ * kHeadDim + c0;
          *reinterpret_cast<float4*>(dst) = make_float4(v[0], v[1], v[2], v[3]);
          *reinterpret_cast<float4*>(dst + 4) = make_float4(v[4], v[5], v[6], v[7]);
        } else {
          *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(p.out) + tok_ * p.out_stride_tok + head_ * p.out_stride_head + c0) =
              make_uint4(pack2<false>(v[0], v[1]), pack2<false>(v[2], v[3]), pack2<false>(v[4], v[5]), pack2<false>(v[6], v[7]));
        }
      };
      auto store_lse = [&](float lse, int64_t tok_, int head_, int64_t prow_) {
        if (p.partial_o) p.partial_lse[prow_] = lse;
        else if (p.lse) p.lse[tok_ * p.num_qo_heads + head_] = lse;
      };
      const float to_out = p.partial_o ? vs : vs * p.out_scale;
      // F > 1: every MMA and conversion of the CTA is done, the tiles of K and V hold the F results of a row
      float* stage = reinterpret_cast<float*>(smem + OFF_K);   // [128 rows of the tile][LD_O], then maximum and sum of each
      constexpr int LD_O = kHeadDim + 4;
      float* st_m = stage + BM * LD_O;
      static_assert(BM * (LD_O + 2) * 4 <= 2 * STAGES * TILE_BYTES, "results fit the tiles");
      if (alive) {
        tc_fence_after();
        const bool none = l == 0.f;
        const float inv = F > 1 ? 1.f : (none ? 0.f : to_out / l);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t v[32];
          if (n_tiles > 0) {
            tmem_ld32(tO + c * 32, v);
            tmem_wait_ld();
          } else {
#pragma unroll
            for (int e = 0; e < 32; ++e) v[e] = 0u;
          }
          if (!row_ok) continue;
#pragma unroll
          for (int e = 0; e < 32; e += 8) {
            float x[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = __uint_as_float(v[e + i]) * inv;
            if (F == 1 && nan_key[2 * c + e / 16] < limit) {
#pragma unroll
              for (int i = 0; i < 8; ++i) x[i] = __int_as_float(0x7fc00000);
            }
            if constexpr (F > 1) {
              float* dst = stage + trow * LD_O + c * 32 + e;
              *reinterpret_cast<float4*>(dst) = make_float4(x[0], x[1], x[2], x[3]);
              *reinterpret_cast<float4*>(dst + 4) = make_float4(x[4], x[5], x[6], x[7]);
            } else {
              store8(x, c * 32 + e, tok, head, prow);
            }
          }
        }
        if constexpr (F > 1) { st_m[trow] = m; st_m[BM + trow] = l; }
        else if (row_ok) store_lse(none ? -INFINITY : (m + log2f(l)) * kLn2, tok, head, prow);
      }
      if constexpr (F > 1) {
        asm volatile("bar.sync 1, 128;" ::: "memory");         // whatever came of the waits, all four warps come here
        if (*abort_flag == 0) {
          const int c8 = (trow & 15) * 8;                      // 16 threads a row, 8 columns each
          for (int rr = trow >> 4; rr < nrows; rr += 8) {
            float top = kNoMax, sum = 0.f, f[F], acc[8];
#pragma unroll
            for (int k = 0; k < F; ++k) top = fmaxf(top, st_m[k * ROWS + rr]);
#pragma unroll
            for (int k = 0; k < F; ++k) { f[k] = exp2_fast(st_m[k * ROWS + rr] - top); sum += f[k] * st_m[BM + k * ROWS + rr]; }
            const bool none = sum == 0.f;
            const float inv = none ? 0.f : to_out / sum;
#pragma unroll
            for (int i = 0; i < 8; ++i) acc[i] = 0.f;
#pragma unroll
            for (int k = 0; k < F; ++k)
#pragma unroll
              for (int i = 0; i < 8; ++i) acc[i] += f[k] * stage[(k * ROWS + rr) * LD_O + c8 + i];
#pragma unroll
            for (int i = 0; i < 8; ++i) acc[i] = nan_key[c8 / 16] < lim(rr) ? __int_as_float(0x7fc00000) : acc[i] * inv;
            const int row2 = w.row0 + rr;
            const int64_t tok2 = qo_base + row2 / G;
            const int head2 = head0 + row2 % G;
            const int64_t prow2 = (static_cast<int64_t>(split) * p.total_q + tok2) * p.num_qo_heads + head2;
            store8(acc, c8, tok2, head2, prow2);
            if (c8 == 0) store_lse(none ? -INFINITY : (top + log2f(sum)) * kLn2, tok2, head2, prow2);
          }
        }
      }
    }
  }

  // ---------------- teardown ----------------
  tc_fence_before();
  __syncthreads();
  if (*abort_flag) {
    if (threadIdx.x == 0 && p.status) atomicExch(p.status, MSA_STATUS_TIMEOUT);
    outlast_async_work();
  }
  if (warp == MMA_WARP) {
    tc_fence_after();
    tmem_dealloc(tmem, TMEM_COLS);
  }
}

}  // namespace
}  // namespace kv4_tc

namespace kv4_tc {
template <int F>
int launch(const MsaFmhaParams& p, cudaStream_t stream) {
  static bool ready[64] = {};
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess) return MSA_ERR_LAUNCH;
  if (device < 0 || device >= 64 || !ready[device]) {
    cudaFuncAttributes fa;
    if (cudaFuncGetAttributes(&fa, kv4_tc_kernel<F>) != cudaSuccess || fa.numRegs * NTHREADS < REGS_NEEDED) return MSA_ERR_LAUNCH;
    if (cudaFuncSetAttribute(kv4_tc_kernel<F>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_BYTES) != cudaSuccess) return MSA_ERR_LAUNCH;
    if (device >= 0 && device < 64) ready[device] = true;
  }
  if (p.num_work == 0) return MSA_OK;
  kv4_tc_kernel<F><<<static_cast<unsigned>(p.num_work), NTHREADS, SMEM_BYTES, stream>>>(p);
  return cudaGetLastError() == cudaSuccess ? MSA_OK : MSA_ERR_LAUNCH;
}
}  // namespace kv4_tc

// Checked by fmha_kv4_fwd; dense items of at most `rows` (128) rows.
int fmha_kv4_tc_launch(const MsaFmhaParams& p, int rows, cudaStream_t stream) {
  return rows <= 32 ? kv4_tc::launch<4>(p, stream) : rows <= 64 ? kv4_tc::launch<2>(p, stream) : kv4_tc::launch<1>(p, stream);
}

}  // namespace msa
