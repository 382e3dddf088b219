// Windowed attention of up to 32 rows, 8 or 16 over an e4m3 cache (decode: tokens x query heads of a KV head), streamed at the rate of the memory.
//
// Per key and KV head 4 * 128 multiplications are made for each row, so memory is the bound, and what has to be short is the chain from a
// key's arrival to its place in the sums.  In the tcgen05 decode kernel that chain (load, Q K^T, commit, softmax, store, P V) takes 1 100
// clocks for 64 keys whatever they hold, most of it hand-overs between warps, and two CTAs of it share an SM: 71 us for 64 sequences x 8
// heads x 2 100 e4m3 keys, 41 would be the memory's.  Here a warp does all of it itself, on mma.sync, and there are eight warps an SM at
// different points of it:
//
//   S^T = K Q^T     A = 16 keys x 16 elements of K from shared memory, B = Q^T, in registers for the whole item
//   O^T = V^T P^T   A = 16 elements x 16 keys of V^T, B = P^T: S^T through a transposing register move
//
// A warp has a ring of its own, filled by TMA (128-byte swizzle: every read below is free of bank conflicts) with units of 16 bf16 or 32 e4m3
// keys, 4 KB each of K and V; unit n of an item is warp n % 4's.  It has a softmax of its own; the four states are joined at the end.
// Units that no row sees are not loaded, so a window costs its keys and at most two units' edges.
//
// Where items are few, the CTAs of a cluster share one: unit n is warp n % (4 S)'s of S CTAs, and the S states of a row are joined through
// distributed shared memory.  There are no partials in memory and no merge to launch.
//
// bf16: P is rounded to bf16 (2^-8), its sum is that of the unrounded weights.
// e4m3: m16n8k32 on the bytes as they are (with K and V converted to f16 the conversions alone took 55 % of the ALU pipe, and an m16n8k16 of f16
// takes 2.1 clocks an SM where an m16n8k32 of e4m3 takes 1.2).  Q and P are pairs of e4m3 values, hi + lo, both multiplied: 8 bits (e4m3_pair).  A query
// row is multiplied by a power of two that brings its largest element to [2^7, 2^8), P is 2^(x - m + 5) and at most 2^8.8.  The order of
// a contraction is free: thread t of a group of four takes elements 32 t .. 32 t + 31 of its keys (K), thread group g elements 16 g .. 16 g + 15 of
// the keys 2 t, 2 t + 8, 2 t + 1, 2 t + 9 (V; four bytes of a key each become four keys of an element by eight byte permutations),
// which is the order that the transposed bytes of P come in.
#include <cooperative_groups.h>

#include <algorithm>

#include "tc_ptx.cuh"

namespace msa {
int make_tma_map_bf16(CUtensorMap* m, const void* base, int rank, const uint64_t* dims, const uint64_t* strides_bytes, const uint32_t* box);
int make_tma_map_u8(CUtensorMap* m, const void* base, int rank, const uint64_t* dims, const uint64_t* strides_bytes, const uint32_t* box);

namespace window {
namespace {

using namespace tc;

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr int kHalf = 4096;                                  // K of a unit; V follows
constexpr int kLdO = kHeadDim + 4;                           // floats of a row of O in shared memory
constexpr float kNoMax = -3e38f;                             // maximum of a row that has seen no key
constexpr int kMaxCluster = 16;

template <bool F8>
__host__ __device__ constexpr int unit_keys() { return F8 ? 32 : 16; }

template <int NT>
struct Cfg {
  // (8 rows leave registers for three CTAs with two stages, 64 e4m3 sequences x 8 heads: 66 us instead of 61)
  static constexpr int CTAS = 2;                             // that share an SM
  static constexpr int STAGES = 3;
  static constexpr int OFF_BAR = kWarps * STAGES * 2 * kHalf;        // [warp][stage] full
  static constexpr int OFF_FAC = OFF_BAR + kWarps * STAGES * 8;      // [8 NT] factor of a row's scores
  static constexpr int OFF_LIM = OFF_FAC + 32 * NT;                  // [8 NT] first key that a row does not see any more, first key of its window
                                                                     // (in the end, in a cluster: maximum - kPOffset, sum of the CTA's state)
  static constexpr int OFF_FLAG = OFF_LIM + 64 * NT;                 // abort, skip, state is good
  // 32 rows: Q^T in shared memory, [step][8 rows][lane] x 8 bytes, or registers run out
  static constexpr bool Q_SHARED = NT == 4;
  static constexpr int OFF_Q = OFF_FLAG + 16;
  static constexpr int SMEM_BYTES = OFF_Q + (Q_SHARED ? NT * 2048 : 0) + 1024;      // + slack to align the base to 1 KB
  static_assert(OFF_FAC % 16 == 0 && OFF_Q % 16 == 0, "alignment");
  static_assert(CTAS * (SMEM_BYTES + 1024) <= 228 * 1024, "they fit an SM");
  static_assert(kWarps * 8 * NT * (kLdO + 2) * 4 <= OFF_BAR, "states fit the rings");
};

__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
// 16 bytes of a row of a swizzled tile of 128-byte rows
__device__ __forceinline__ uint32_t swizzled(int row, int chunk) { return static_cast<uint32_t>(row * 128 + ((chunk ^ (row & 7)) << 4)); }
__device__ __forceinline__ void mma_e4m3(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Bytes i of four words, as word i.
__device__ __forceinline__ void transpose_bytes(uint32_t w0, uint32_t w1, uint32_t w2, uint32_t w3, uint32_t (&d)[4]) {
  const uint32_t a = __byte_perm(w0, w1, 0x5140), b = __byte_perm(w2, w3, 0x5140), c = __byte_perm(w0, w1, 0x7362), e = __byte_perm(w2, w3, 0x7362);
  d[0] = __byte_perm(a, b, 0x5410); d[1] = __byte_perm(a, b, 0x7632);
  d[2] = __byte_perm(c, e, 0x5410); d[3] = __byte_perm(c, e, 0x7632);
}
__device__ __forceinline__ void load_words(const unsigned char* at, uint32_t* w) {
  const uint4 v = *reinterpret_cast<const uint4*>(at);
  w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
}

template <int NT, bool F8>
__global__ void __launch_bounds__(kThreads, Cfg<NT>::CTAS)
window_decode_kernel(const __grid_constant__ MsaFmhaParams p, const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v) {
  using C = Cfg<NT>;
  constexpr int OFF_BAR = C::OFF_BAR, OFF_FAC = C::OFF_FAC, OFF_LIM = C::OFF_LIM, OFF_FLAG = C::OFF_FLAG, kStages = C::STAGES;
  constexpr int UK = unit_keys<F8>(), STEPS = UK / 16;
  constexpr int SUB = UK * 128;                              // a half of head_dim of a bf16 unit, all of it in e4m3
  constexpr float kPOffset = F8 ? kPairOffset : 0.f, kRescale = F8 ? kPairRescale : 8.f;      // P is at most 2^8, 2^8.8 in e4m3
  extern __shared__ unsigned char smem_raw[];
  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  unsigned char* smem = smem_raw + (smem_base - smem_u32(smem_raw));
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + OFF_FLAG);
  volatile int* skip_flag = abort_flag + 1;
  const auto cluster = cooperative_groups::this_cluster();
  const int S = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
  unsigned char* ring = smem + warp * kStages * 2 * kHalf;
  const uint32_t ring_u = smem_base + warp * kStages * 2 * kHalf, bars = smem_base + OFF_BAR + warp * kStages * 8;

  // a timeout reported earlier on this device (status word not cleared yet): do not start
  if (threadIdx.x == kThreads - 1) *skip_flag = (p.status != nullptr && *reinterpret_cast<const volatile int32_t*>(p.status) != 0) ? 1 : 0;
  if (threadIdx.x == 0) {
    *abort_flag = 0;
    for (int s = 0; s < kWarps * kStages; ++s) mbar_init(smem_base + OFF_BAR + 8 * s, 1);
    mbar_fence_init();
  }

  // ---------------- the item ----------------
  const MsaWorkItem w = p.work[blockIdx.x / S];
  const int b = chk(w.batch, 0, p.batch, p.status), head0 = chk(w.head0, 0, p.num_qo_heads, p.status), split = chk(w.split, 0, p.num_splits, p.status);
  const int G = p.pack, kvh = head0 / (p.num_qo_heads / p.num_kv_heads);
  const int qo_base = p.qo_start[b], kv_len = p.kv_len[b], off = p.qo_offset[b];
  const bool paged = p.page_size > 0;
  const int kv0 = paged ? p.kv_page_indptr[b] : p.kv_start[b];
  const int ntok = min(p.qo_start[b + 1] - qo_base, p.decode_rows / G);      // (lengths on the device may outgrow the rows there are)
  const int nrows = ntok * G;
  // Units are numbered without those that no row sees: number n stands for unit n of the keys below sink_u, for n + skip_u from there on.
  const int first_key = window_first(off, kv_len, p.window);                 // of the first row's window
  const int end_key = max(0, min(kv_len, off + ntok));                       // behind what the last row sees
  const int sink_u = p.sink_tokens / UK + (p.sink_tokens % UK != 0), skip_u = max(0, first_key / UK - sink_u);
  auto number = [&](int u) { return u < sink_u ? u : max(sink_u, u - skip_u); };
  auto real_tile = [&](int t) { return t < sink_tiles(p.sink_tokens) ? t : t + w.kv_tile_skip; };
  int begin = 0, end = 0;
  if (w.kv_tile_begin < w.kv_tile_end && nrows > 0) {
    begin = number(real_tile(w.kv_tile_begin) * (kKvTile / UK));
    end = number(min((real_tile(w.kv_tile_end - 1) + 1) * (kKvTile / UK), (end_key + UK - 1) / UK));
  }
  const int step = kWarps * S;
  begin += kWarps * rank + warp;                             // this warp's: every step-th
  const int n_units = end > begin ? (end - begin + step - 1) / step : 0;
  auto key_of = [&](int i) { const int n = begin + step * i; return (n < sink_u ? n : n + skip_u) * UK; };

  // ---------------- loads ----------------
  int phys = 0, row = 0;                                     // lane i: where this warp's unit 32 k + i is, its page and its first row there
  auto load_pages = [&](int i0) {
    if (i0 + lane >= n_units) return;
    const int key0 = key_of(i0 + lane);
    row = kv0 + key0;
    if (paged) {
      const int c = key0 / p.page_size;
      phys = page_entry(p, kv0 + c);
      row = key0 - c * p.page_size;
    }
  };
  auto fetch = [&](int i, int stage) {                       // unit i into a stage that no lane reads any more
    if ((i & 31) == 0) { load_pages(i); __syncwarp(); }
    const int page = __shfl_sync(0xffffffffu, phys, i & 31), first = __shfl_sync(0xffffffffu, row, i & 31);
    if (elect_one()) {
      const uint32_t bar = bars + 8 * stage, dst = ring_u + stage * 2 * kHalf;
      mbar_arrive_expect_tx(bar, 2 * kHalf);
      // (both halves of head_dim in one copy: its tensor has them as a dimension)
      if (paged) {
        tma_load_5d(dst, &tm_k, bar, 0, first, 0, kvh, page);
        tma_load_5d(dst + kHalf, &tm_v, bar, 0, first, 0, kvh, page);
      } else {
        tma_load_4d(dst, &tm_k, bar, 0, first, 0, kvh);
        tma_load_4d(dst + kHalf, &tm_v, bar, 0, first, 0, kvh);
      }
    }
    __syncwarp();
  };
  __syncthreads();
  const bool run = *skip_flag == 0;
  bool alive = run;
  if (run) {
#pragma unroll
    for (int s = 0; s < kStages; ++s)
      if (s < n_units) fetch(s, s);
  }

  // ---------------- Q^T: row 8 n + g, as operands ----------------
  // The factor of the scores is made positive, its sign goes to Q, so that the largest score has the largest exponent; a factor of 0 makes Q 0.
  const float signed_scale = p.sm_scale * kLog2e * (p.k_scale_head ? p.k_scale_head[kvh] : 1.f);
  const float scale = signed_scale == 0.f ? 1.f : fabsf(signed_scale);
  [[maybe_unused]] const uint32_t flip = signed_scale < 0.f ? 0x80008000u : 0u, keep = signed_scale == 0.f ? 0u : 0xffffffffu;
  uint32_t qf[C::Q_SHARED ? 1 : NT][8][2];                   // bf16: [step of 16 elements]; e4m3: [step of 32 elements, + 4: lo]
  [[maybe_unused]] const bool pair_q = F8 && p.q_dtype == MSA_DT_BF16;
  float* s_fac = reinterpret_cast<float*>(smem + OFF_FAC);
  // (in shared memory: warp n makes those of rows 8 n .. 8 n + 7)
#pragma unroll
  for (int n_ = 0; n_ < (C::Q_SHARED ? 1 : NT); ++n_) {
    const int n = C::Q_SHARED ? warp : n_;
    const int row = min(8 * n + g, max(nrows, 1) - 1);       // rows that are none repeat the last one and are not written
    const int64_t at = static_cast<int64_t>(qo_base + row / G) * p.q_stride_tok + static_cast<int64_t>(head0 + row % G) * p.q_stride_head;
    if constexpr (!F8) {
      const uint32_t* src = reinterpret_cast<const uint32_t*>(static_cast<const __nv_bfloat16*>(p.q) + at);
#pragma unroll
      for (int s = 0; s < 8; ++s) {
        qf[n_][s][0] = nrows > 0 ? (src[8 * s + t4] ^ flip) & keep : 0u;
        qf[n_][s][1] = nrows > 0 ? (src[8 * s + 4 + t4] ^ flip) & keep : 0u;
      }
    } else {
      int e = 0;                                             // exponent that the row is divided by
      if (!pair_q) {
        uint32_t v[8] = {};
        if (nrows > 0) {
          load_words(static_cast<const unsigned char*>(p.q) + at + 32 * t4, v);
          load_words(static_cast<const unsigned char*>(p.q) + at + 32 * t4 + 16, v + 4);
        }
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          qf[n_][c >> 1][c & 1] = (v[c] ^ (flip | (flip >> 8))) & keep;
          qf[n_][4 + (c >> 1)][c & 1] = 0;
        }
      } else {
        uint32_t v[16] = {};                                 // elements 32 t .. 32 t + 31
        if (nrows > 0) {
#pragma unroll
          for (int c = 0; c < 4; ++c) load_words(reinterpret_cast<const unsigned char*>(static_cast<const __nv_bfloat16*>(p.q) + at + 32 * t4) + 16 * c, v + 4 * c);
        }
        uint32_t top = 0;                                    // magnitudes order as their bits do
#pragma unroll
        for (int c = 0; c < 16; ++c) top = max(top, max(v[c] & 0x7fffu, (v[c] >> 16) & 0x7fffu));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        // (a row of zeros, or with an infinity or NaN, is taken as it is; the factors are normal numbers)
        e = static_cast<int>(top >> 7) - 127 - 7;
        if (top == 0 || top >= 0x7f80u) e = 0;
        e = min(max(e, -126), 126);
        const float up = copysignf(signed_scale == 0.f ? 0.f : __uint_as_float(static_cast<uint32_t>(127 - e) << 23), signed_scale);
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          uint32_t hi[2], lo[2];
#pragma unroll
          for (int h = 0; h < 2; ++h)
            e4m3_pair(__uint_as_float(v[2 * c + h] << 16) * up, __uint_as_float(v[2 * c + h] & 0xffff0000u) * up, hi[h], lo[h]);
          qf[n_][c >> 1][c & 1] = hi[0] | (hi[1] << 16);
          qf[n_][4 + (c >> 1)][c & 1] = lo[0] | (lo[1] << 16);
        }
      }
      if ((C::Q_SHARED || warp == 0) && t4 == 0) s_fac[8 * n + g] = signed_scale == 0.f ? 1.f : scale * __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
    }
  }
  uint2* s_q = reinterpret_cast<uint2*>(smem + C::OFF_Q) + lane;
  if constexpr (C::Q_SHARED) {
#pragma unroll
    for (int s = 0; s < 8; ++s) s_q[(s * NT + warp) * 32] = make_uint2(qf[0][s][0], qf[0][s][1]);
  }
  auto q_of = [&](int n, int s) -> uint2 {
    if constexpr (C::Q_SHARED) return s_q[(s * NT + n) * 32];
    else return make_uint2(qf[n][s][0], qf[n][s][1]);
  };
  int2* s_lim = reinterpret_cast<int2*>(smem + OFF_LIM);
  if (threadIdx.x < 8 * NT) {
    const int tok = min(static_cast<int>(threadIdx.x), max(nrows, 1) - 1) / G;
    s_lim[threadIdx.x] = make_int2(max(0, min(kv_len, tok + off + 1)), window_first(tok + off, kv_len, p.window));
  }
  __syncthreads();

  float fac[NT][2];                                          // of rows 8 n + 2 t4 + c: factor of the scores
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int c = 0; c < 2; ++c) fac[n][c] = F8 ? s_fac[8 * n + 2 * t4 + c] : scale;
  const int lim_first = max(0, min(kv_len, off + 1)), from_last = window_first(off + ntok - 1, kv_len, p.window);

  float m[NT][2];                                            // maximum - kPOffset
  uint64_t l[NT];                                            // sums of the weights, two floats
  float o[8][NT][4];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    m[n][0] = m[n][1] = kNoMax;
    l[n] = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int c = 0; c < 4; ++c) o[i][n][c] = 0.f;
  }

  int stage = 0, parity = 0;
  [[maybe_unused]] bool settled = !F8;
#pragma unroll 1
  for (int i = 0; i < n_units && alive; ++i) {
    const int key0 = key_of(i);
    unsigned char* kt = ring + stage * 2 * kHalf;
    unsigned char* vt = kt + kHalf;
    const uint32_t kt_u = ring_u + stage * 2 * kHalf, vt_u = kt_u + kHalf;
    alive = mbar_wait_warp(bars + 8 * stage, parity, abort_flag);
    if (!alive) break;
    // Keys that no row sees read as 0 in V: the weight of 0 that they have does not take a NaN out.
    const bool unseen = key0 + UK > end_key || (key0 < first_key && key0 + UK > p.sink_tokens);
    if (unseen) {
      for (int c = lane; c < UK * (F8 ? 8 : 16); c += 32) {
        const int r = c / (F8 ? 8 : 16), ch = c % (F8 ? 8 : 16), key = key0 + r;
        if (key >= end_key || (key < first_key && key >= p.sink_tokens))
          *reinterpret_cast<uint4*>(vt + (ch >> 3) * SUB + r * 128 + (ch & 7) * 16) = make_uint4(0, 0, 0, 0);
      }
      fence_proxy_async_smem();                              // before the next copy into these bytes
      __syncwarp();
    }
    // ---- S^T ----
    float s[STEPS][NT][4];
#pragma unroll
    for (int u = 0; u < STEPS; ++u) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int c = 0; c < 4; ++c) s[u][n][c] = 0.f;
      if constexpr (!F8) {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          uint32_t a[4];
          const int ch = 2 * k + (lane >> 4);
          ldmatrix_x4(kt_u + (ch >> 3) * SUB + swizzled(lane & 15, ch & 7), a[0], a[1], a[2], a[3]);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            const uint2 q = q_of(n, k);
            mma_16816<false>(s[u][n], a, q.x, q.y);
          }
        }
      } else {
        uint32_t lo[8], hi[8];                               // keys g and g + 8
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          load_words(kt + swizzled(16 * u + g, 2 * t4 + h), lo + 4 * h);
          load_words(kt + swizzled(16 * u + 8 + g, 2 * t4 + h), hi + 4 * h);
        }
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            const uint2 q = q_of(n, k);
            mma_e4m3(s[u][n], lo[2 * k], hi[2 * k], lo[2 * k + 1], hi[2 * k + 1], q.x, q.y);
          }
        if (pair_q) {                                        // sums of their own: chains half as long
          float s2[NT][4] = {};
#pragma unroll
          for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              const uint2 q = q_of(n, 4 + k);
              mma_e4m3(s2[n], lo[2 * k], hi[2 * k], lo[2 * k + 1], hi[2 * k + 1], q.x, q.y);
            }
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int c = 0; c < 4; ++c) s[u][n][c] += s2[n][c];
        }
      }
    }
    // ---- softmax: mask, a maximum that may lag, exponents ----
    if (key0 + UK > lim_first || (key0 < from_last && key0 + UK > p.sink_tokens)) {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const int4 r = *reinterpret_cast<const int4*>(s_lim + 8 * n + 2 * t4);       // of two rows
#pragma unroll
        for (int u = 0; u < STEPS; ++u)
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const int key = key0 + 16 * u + 8 * (c >> 1) + g;
            if (key >= (c & 1 ? r.z : r.x) || (key < (c & 1 ? r.w : r.y) && key >= p.sink_tokens)) s[u][n][c] = -INFINITY;
          }
      }
    }
    bool raise = false;
    float top[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float x = fmaxf(s[0][n][c], s[0][n][c + 2]);
        if constexpr (STEPS == 2) x = max3(x, s[STEPS - 1][n][c], s[STEPS - 1][n][c + 2]);
        top[n][c] = x * fac[n][c];
        raise |= top[n][c] > m[n][c] + (kPOffset + kRescale);
      }
    if (!settled || __any_sync(0xffffffffu, raise)) {
      bool enough = true;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float k2[2];
        [[maybe_unused]] float sum[2];
        if constexpr (F8) f2_unpack(l[n], sum[0], sum[1]);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float x = top[n][c];
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, d));
          float now;
          if constexpr (F8) {
            // pairs: up, or down where the row's sums do not allow small weights to get lost (pair_lowers; all units' keys count from the start,
            // which takes no registers); the unit's sum is that of the largest weights of four keys at least
            const bool up = x > m[n][c] + (kPOffset + kRescale);
            now = up ? x - (m[n][c] == kNoMax ? kPOffset : kPOffset + kPairRise) : m[n][c];
            float tile = exp2_fast(top[n][c] - now);
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) {
              tile += __shfl_xor_sync(0xffffffffu, tile, d);
              sum[c] += __shfl_xor_sync(0xffffffffu, sum[c], d);
            }
            const float row = sum[c] * exp2_fast(m[n][c] - now), all = static_cast<float>(UK) * static_cast<float>(n_units);
            if (pair_lowers(now + kPOffset, x, tile, row, UK, all - UK)) now = x - kPOffset;
            enough &= row >= kPairEnough * all;
          } else {
            now = fmaxf(x - kPOffset, m[n][c]);
          }
          k2[c] = exp2_fast(m[n][c] - now);
          m[n][c] = now;
#pragma unroll
          for (int j = 0; j < 8; ++j) { o[j][n][c] *= k2[c]; o[j][n][c + 2] *= k2[c]; }
        }
        l[n] = f2_fma(l[n], f2_pack(k2[0], k2[1]), 0);
      }
      if constexpr (F8) settled = __all_sync(0xffffffffu, enough);     // once all rows have enough for all units, only a maximum that rises asks again
    }
    uint32_t pt[STEPS][NT][2];                               // P^T as an operand: keys 0-7, keys 8-15; e4m3: hi, lo of the step's 16 keys
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const uint64_t f = f2_pack(fac[n][0], fac[n][1]), shift = f2_pack(-m[n][0], -m[n][1]);
#pragma unroll
      for (int u = 0; u < STEPS; ++u) {
        float w0[2], w1[2];                                  // keys g and g + 8 of the rows 2 t, 2 t + 1
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float x0, x1;
          f2_unpack(f2_fma(f2_pack(s[u][n][2 * h], s[u][n][2 * h + 1]), f, shift), x0, x1);
          w0[h] = exp2_fast(x0); w1[h] = exp2_fast(x1);
          l[n] = f2_add(l[n], f2_pack(w0[h], w1[h]));
          if constexpr (!F8) pt[u][n][h] = transpose8x8(pack2<false>(w0[h], w1[h]));
        }
        if constexpr (F8) {
          uint32_t h0, l0, h1, l1;
          e4m3_pair(w0[0], w0[1], h0, l0);
          e4m3_pair(w1[0], w1[1], h1, l1);
          pt[u][n][0] = transpose8x8(h0 | (h1 << 16));
          pt[u][n][1] = transpose8x8(l0 | (l1 << 16));
        }
      }
    }
    // ---- O^T ----
    if constexpr (!F8) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        uint32_t a[4];
        const int ch = 2 * j + ((lane >> 3) & 1), r = (lane & 7) + ((lane >> 4) << 3);
        ldmatrix_x4_trans(vt_u + (ch >> 3) * SUB + swizzled(r, ch & 7), a[0], a[1], a[2], a[3]);
#pragma unroll
        for (int n = 0; n < NT; ++n) mma_16816<false>(o[j][n], a, pt[0][n][0], pt[0][n][1]);
      }
    } else {
      uint32_t v[2][4][4];                                   // [step][key 2 t, 2 t + 8, 2 t + 1, 2 t + 9][4 elements]
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int r = 0; r < 4; ++r) load_words(vt + swizzled(16 * u + 2 * t4 + (r >> 1) + 8 * (r & 1), g), v[u][r]);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        uint32_t a[2][4];                                    // elements 4 j .. 4 j + 3 of four keys
#pragma unroll
        for (int u = 0; u < 2; ++u) transpose_bytes(v[u][0][j], v[u][1][j], v[u][2][j], v[u][3][j], a[u]);
#pragma unroll
        for (int part = 0; part < 2; ++part)                 // hi, lo
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int n = 0; n < NT; ++n)
              mma_e4m3(o[2 * j + h][n], a[0][2 * h], a[0][2 * h + 1], a[1][2 * h], a[1][2 * h + 1], pt[0][n][part], pt[STEPS - 1][n][part]);
      }
    }
    __syncwarp();                                            // all lanes have read the stage
    if (i + kStages < n_units) fetch(i + kStages, stage);
    if (++stage == kStages) { stage = 0; parity ^= 1; }
  }
  float sums[NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    f2_unpack(l[n], sums[n][0], sums[n][1]);
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int d = 4; d < 32; d <<= 1) sums[n][c] += __shfl_xor_sync(0xffffffffu, sums[n][c], d);
  }
  __syncthreads();                                           // the rings are no longer read, and no copy is on its way (but after a timeout)
  bool good = run;
  if (*abort_flag) {
    if (threadIdx.x == 0 && p.status) atomicExch(p.status, MSA_STATUS_TIMEOUT);
    outlast_async_work();
    good = false;
  }
  if (nrows <= 0 || (S == 1 && !good)) return;               // (all CTAs of a cluster, or one without any)
  // ---------------- the four states of a row become one ----------------
  float* s_o = reinterpret_cast<float*>(smem);               // [warp][row][kLdO]
  float* s_m = s_o + kWarps * 8 * NT * kLdO;                 // [warp][row][2]: maximum - kPOffset, sum
  float2* s_c = reinterpret_cast<float2*>(smem + OFF_LIM);
  int* s_good = reinterpret_cast<int*>(smem + OFF_FLAG) + 2;
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int r = warp * 8 * NT + 8 * n + 2 * t4 + c;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if constexpr (F8) {
          *reinterpret_cast<float2*>(s_o + r * kLdO + 16 * g + 2 * j) = make_float2(o[j][n][c], o[j][n][c + 2]);
        } else {
          s_o[r * kLdO + 16 * j + g] = o[j][n][c];
          s_o[r * kLdO + 16 * j + g + 8] = o[j][n][c + 2];
        }
      }
      if (g == 0) { s_m[2 * r] = m[n][c]; s_m[2 * r + 1] = sums[n][c]; }
    }
  __syncthreads();
  // 16 threads a row, 8 columns each
  const int c16 = threadIdx.x & 15;
#pragma unroll
  for (int r0 = 0; r0 < 8 * NT; r0 += 8) {
    const int r = r0 + (threadIdx.x >> 4);
    if (r >= nrows) continue;
    float top = kNoMax;
#pragma unroll
    for (int v = 0; v < kWarps; ++v) top = fmaxf(top, s_m[2 * (v * 8 * NT + r)]);
    float sum = 0.f, acc[8];
#pragma unroll
    for (int c = 0; c < 8; ++c) acc[c] = 0.f;
#pragma unroll
    for (int v = 0; v < kWarps; ++v) {
      const int at = v * 8 * NT + r;
      const float f = exp2_fast(s_m[2 * at] - top);
      sum += f * s_m[2 * at + 1];
#pragma unroll
      for (int c = 0; c < 8; ++c) acc[c] += f * s_o[at * kLdO + 8 * c16 + c];
    }
    if (S > 1) {                                             // in the place of warp 0's, which no other thread reads
      *reinterpret_cast<float4*>(s_o + r * kLdO + 8 * c16) = make_float4(acc[0], acc[1], acc[2], acc[3]);
      *reinterpret_cast<float4*>(s_o + r * kLdO + 8 * c16 + 4) = make_float4(acc[4], acc[5], acc[6], acc[7]);
      if (c16 == 0) s_c[r] = make_float2(top, sum);
      continue;
    }
    const int64_t tok = qo_base + r / G;
    const int head = head0 + r % G;
    const bool none = sum == 0.f;
    const float inv = none ? 0.f : (p.v_scale_head ? p.v_scale_head[kvh] : 1.f) / sum;
    const float lse = none ? -INFINITY : (top + log2f(sum)) * kLn2;
    if (p.partial_o) {
      const int64_t at = (static_cast<int64_t>(split) * p.total_q + tok) * p.num_qo_heads + head;
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
  if (S == 1) return;
  // ---------------- the S states of a row become one ----------------
  if (threadIdx.x == 0) *s_good = good;
  cluster.sync();
  const int q = min(lane, S - 1);                            // lane q has what CTA q has of a row
  if (__all_sync(0xffffffffu, *cluster.map_shared_rank(s_good, q) != 0)) {
    for (int r = rank + S * warp; r < nrows; r += step) {
      const float2 c = *cluster.map_shared_rank(s_c + r, q);
      float top = c.x;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
      const float weight = exp2_fast(c.x - top);
      float sum = lane < S ? weight * c.y : 0.f;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
      for (int i = 0; i < S; ++i) {
        const float4 x = *cluster.map_shared_rank(reinterpret_cast<const float4*>(s_o + r * kLdO + 4 * lane), i);
        const float f = __shfl_sync(0xffffffffu, weight, i);
        acc.x = fmaf(f, x.x, acc.x); acc.y = fmaf(f, x.y, acc.y); acc.z = fmaf(f, x.z, acc.z); acc.w = fmaf(f, x.w, acc.w);
      }
      const int64_t tok = qo_base + r / G;
      const int head = head0 + r % G;
      const bool none = sum == 0.f;
      const float f = none ? 0.f : (p.v_scale_head ? p.v_scale_head[kvh] : 1.f) * p.out_scale / sum;
      *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(p.out) + tok * p.out_stride_tok + head * p.out_stride_head + 4 * lane) =
          make_uint2(pack2<false>(acc.x * f, acc.y * f), pack2<false>(acc.z * f, acc.w * f));
      if (p.lse && lane == 0) p.lse[tok * p.num_qo_heads + head] = none ? -INFINITY : (top + log2f(sum)) * kLn2;
    }
  }
  cluster.sync();                                            // until nobody reads this CTA's memory
}

// CTAs that share an item: the most with which all items are on the GPU at once, and with a unit for each warp.
template <int NT, bool F8>
int cluster_of(const MsaFmhaParams& p, cudaLaunchConfig_t config, int device) {
  if (p.partial_o || device < 0 || device >= 64) return 1;
  static int fit[64][kMaxCluster + 1] = {};                  // clusters of a size that a device holds, + 1
  const int64_t keys = static_cast<int64_t>(p.window) + p.sink_tokens + p.decode_rows / p.pack;
  const int64_t most = std::min<int64_t>(kMaxCluster, (keys + kWarps * unit_keys<F8>() - 1) / (kWarps * unit_keys<F8>()));
  for (int s = static_cast<int>(most); s > 1; --s) {
    if (static_cast<int64_t>(p.num_work) * s > sms_of(p) * Cfg<NT>::CTAS) continue;
    if (!fit[device][s]) {
      cudaLaunchAttribute attr = {};
      attr.id = cudaLaunchAttributeClusterDimension;
      attr.val.clusterDim.x = s; attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
      config.gridDim = dim3(s);
      config.attrs = &attr; config.numAttrs = 1;
      int n = 0;
      if (cudaOccupancyMaxActiveClusters(&n, window_decode_kernel<NT, F8>, &config) != cudaSuccess) { cudaGetLastError(); n = 0; }
      fit[device][s] = n + 1;
    }
    if (p.num_work < fit[device][s]) return s;
  }
  return 1;
}

template <int NT, bool F8>
int launch(const MsaFmhaParams& p, cudaStream_t stream) {
  constexpr int UK = unit_keys<F8>();
  const uint64_t e = F8 ? 1 : 2;
  CUtensorMap tk, tv;
  for (int i = 0; i < 2; ++i) {
    const void* base = i ? p.v : p.k;
    const uint64_t tok = (i ? p.v_stride_tok : p.k_stride_tok) * e, head = (i ? p.v_stride_head : p.k_stride_head) * e,
                   page = (i ? p.v_stride_page : p.k_stride_page) * e;
    const uint32_t cols = F8 ? 128 : 64, halves = F8 ? 1 : 2;          // of head_dim: 128 bytes each, a swizzled tile of its own
    const auto make = F8 ? make_tma_map_u8 : make_tma_map_bf16;
    int rc;
    if (p.page_size > 0) {
      const uint64_t dims[5] = {cols, static_cast<uint64_t>(p.page_size), halves, static_cast<uint64_t>(p.num_kv_heads), static_cast<uint64_t>(p.kv_extent)};
      const uint64_t str[4] = {tok, 128, head, page};
      const uint32_t box[5] = {cols, UK, halves, 1, 1};
      rc = make(i ? &tv : &tk, base, 5, dims, str, box);
    } else {
      const uint64_t dims[4] = {cols, static_cast<uint64_t>(p.kv_extent), halves, static_cast<uint64_t>(p.num_kv_heads)};
      const uint64_t str[3] = {tok, 128, head};
      const uint32_t box[4] = {cols, UK, halves, 1};
      rc = make(i ? &tv : &tk, base, 4, dims, str, box);
    }
    if (rc != MSA_OK) return MSA_ERR_LAUNCH;
  }
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess) return MSA_ERR_LAUNCH;
  static bool ready[64] = {};
  if (device < 0 || device >= 64 || !ready[device]) {
    if (cudaFuncSetAttribute(window_decode_kernel<NT, F8>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<NT>::SMEM_BYTES) != cudaSuccess ||
        cudaFuncSetAttribute(window_decode_kernel<NT, F8>, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared) != cudaSuccess ||
        cudaFuncSetAttribute(window_decode_kernel<NT, F8>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess)
      return MSA_ERR_LAUNCH;
    if (device >= 0 && device < 64) ready[device] = true;
  }
  cudaLaunchConfig_t config = {};
  config.blockDim = dim3(kThreads);
  config.dynamicSmemBytes = Cfg<NT>::SMEM_BYTES;
  config.stream = stream;
  const int s = cluster_of<NT, F8>(p, config, device);
  config.gridDim = dim3(static_cast<unsigned>(p.num_work) * s);
  cudaLaunchAttribute attr = {};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = s; attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  if (s > 1) { config.attrs = &attr; config.numAttrs = 1; }
  return cudaLaunchKernelEx(&config, window_decode_kernel<NT, F8>, p, tk, tv) == cudaSuccess ? MSA_OK : MSA_ERR_LAUNCH;
}

}  // namespace
}  // namespace window

// Windowed items of few packed rows; pages of whole units, or ragged keys.  Here and on the tcgen05 decode kernel (pages of 128 keys), one token a
// sequence: bf16, 32 rows, 64 sequences x 2 heads x 2 048 keys 34 and 34 us, 128 x 8 x 4 096 326 and 366; e4m3, 8 rows, 64 x 1 x 2 048 15.2 and 22.3,
// 128 x 8 x 4 096 186 and 285.  16 rows over an e4m3 cache (255 registers) pay while items are few and three CTAs or more share one: windows of 1 024 keys, 32
// items 14.1 and 16.4 us, 80 17.6 and 19.7, 96 21.8 and 20.3, 512 61 and 55; of 4 096, 32 21.6 and 33.6, 80 36.5 and 43.9, 96 51 and 45, 512 166 and 148;
// of 512, within 5 % from 64 items on.  With 32 rows registers run out.
int fmha_window_rows(const MsaFmhaParams& p) {
  if (p.kv_dtype != MSA_DT_E4M3) return 32;
  return p.page_size == kKvTile && 128 % p.pack == 0 && p.num_work > sms_of(p) * 3 / 5 ? 8 : 16;
}
int fmha_window_supported(const MsaFmhaParams& p) {
  if (p.window <= 0 || (p.flags & MSA_FLAG_SPARSE) || p.decode_rows < 1 || p.decode_rows > fmha_window_rows(p)) return 0;
  if (p.pack != p.num_qo_heads / p.num_kv_heads) return 0;
  const bool f8 = p.kv_dtype == MSA_DT_E4M3;
  if (p.q_dtype != MSA_DT_BF16 && !(f8 && p.q_dtype == MSA_DT_E4M3)) return 0;
  if (p.page_size > 0 && p.page_size % (f8 ? window::unit_keys<true>() : window::unit_keys<false>())) return 0;
  return p.kv_extent > 0;
}

int fmha_window_launch(const MsaFmhaParams& p, cudaStream_t stream) {
  using namespace window;
  if (p.num_work <= 0) return MSA_OK;
  const bool f8 = p.kv_dtype == MSA_DT_E4M3;
  if (p.decode_rows <= 8) return f8 ? launch<1, true>(p, stream) : launch<1, false>(p, stream);
  if (p.decode_rows <= 16) return f8 ? launch<2, true>(p, stream) : launch<2, false>(p, stream);
  return launch<4, false>(p, stream);
}

}  // namespace msa
