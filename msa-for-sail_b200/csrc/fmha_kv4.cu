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
// most 8 behind the true maximum: at most 2^15, 11 bits down to 2^-21 of the largest weight.
//
// A CTA has four warps.  Warp w has keys 32 w .. 32 w + 31 of every page, a ring of its own that it fills with 16-byte copies, and a
// softmax of its own; the four states are joined at the end.  So the warps of an SM run past one another without barriers.  (Rings
// filled by bulk copies, sixteen small ones a page and warp: 281 us instead of 246 for a million keys; one ring a CTA with a warp
// that loads: 250.)
//
// Up to 8 rows to a head (NT = 1): four CTAs an SM, two pages in a ring; to 16 (NT = 2): three CTAs with three, or registers run out.
// More rows: fmha_kv4_tc.cu, or, where a selection is a token's own, groups of 16.
//
// Measured: one sequence of 1 048 576 keys, 64 / 8 heads: 219 us and 5 for the merge, 5.5 TB/s of codes and scales.  The copies alone take 186 us,
// the conversions and products alone 213: the issue slots (55 % used, a conversion is an instruction of two clocks on the ALU
// pipe) bound it, together with what the two leave one another.  (Under the 1 000 W cap, after some hundreds of passes, 260 at 1.68 GHz.)  24 ragged sequences, 64 / 4 heads (NT = 2): 56 us, 3.4 TB/s; a page
// takes an SM 1 300 clocks, 830 would be the memory's (its two steps of 16 keys one after the other, which spares registers: 62 us with
// three CTAs an SM, 67 with four).  32 x 16 selected pages of 1 024, 64 / 8 heads: 22 us, 3.4 TB/s; index
// loads, first page and epilogue of one wave of CTAs.
#include <algorithm>

#include "kv4.cuh"
#include "nvtx_range.h"

namespace msa {
namespace kv4 {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr int kKeys = kKvTile / kWarps;                      // of a page that a warp has
constexpr int kCodeBytes = kKeys * kKv4CodeBytes, kScaleBytes = kKeys * kKv4ScaleBytes;

// Shared memory of a CTA for 8 NT rows.
template <int NT>
struct Cfg {
  static constexpr int CTAS = NT == 1 ? 4 : 3;               // that share an SM
  static constexpr int STAGES = NT == 1 ? 2 : 3;
  static constexpr int HALF = kCodeBytes + kScaleBytes;      // K of a warp's keys; V follows
  static constexpr int OFF_Q = kWarps * STAGES * 2 * HALF;   // Q^T as the operands of a warp's lanes: [word][8 rows][lane] x 16 bytes
  static constexpr int OFF_FAC = OFF_Q + 4 * NT * 512;       // [8 NT] factor of a row's scores
  static constexpr int OFF_LIM = OFF_FAC + 32 * NT;          // [8 NT] first key that a row may not see
  static constexpr int BYTES = OFF_LIM + 32 * NT;
  static_assert(HALF % 16 == 0 && OFF_Q % 16 == 0 && OFF_FAC % 16 == 0 && OFF_LIM % 16 == 0, "alignment");
  static_assert(CTAS * (BYTES + 1024) <= 228 * 1024, "they fit an SM");
};

constexpr int kLdO = kHeadDim + 4;                           // floats of a row of O in shared memory
constexpr float kPOffset = 7.f;
constexpr float kRescale = 8.f;
constexpr float kNoMax = -3e38f;                             // maximum of a row that has seen no key

// Key of a 16-key step that stands at place j (0..7) of an operand: a quarter-warp's 16-byte reads of K rows fall into all banks.
__device__ __forceinline__ int key_at(int j) { return (j & 4) | ((j & 2) ? 3 - (j & 1) : (j & 1)); }

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  const uint32_t a[4] = {a0, a1, a2, a3};
  mma_16816<true>(d, a, b0, b1);
}
// Without a sum to add to.
__device__ __forceinline__ void mma_f16_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};\n"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
// Both halves of x times one half of s.
__device__ __forceinline__ uint32_t half2_mul_by(uint32_t x, uint32_t s, bool high) {
  const __half2 f = *reinterpret_cast<const __half2*>(&s);
  const __half2 d = __hmul2(*reinterpret_cast<const __half2*>(&x), high ? __high2half2(f) : __low2half2(f));
  return *reinterpret_cast<const uint32_t*>(&d);
}
// Four or two words of shared memory.
__device__ __forceinline__ void load_words(const unsigned char* at, uint32_t (&w)[4]) {
  const uint4 v = *reinterpret_cast<const uint4*>(at);
  w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
}
__device__ __forceinline__ void load_words(const unsigned char* at, uint32_t (&w)[2]) {
  const uint2 v = *reinterpret_cast<const uint2*>(at);
  w[0] = v.x; w[1] = v.y;
}

// 0xff for each byte that is an e4m3 NaN.
__device__ __forceinline__ uint32_t nan_bytes(uint32_t x) { return __vcmpeq4(x & 0x7f7f7f7fu, 0x7f7f7f7fu); }

// The item of a CTA: rows of one KV head against a list of pages.
struct Item {
  int b, kvh, split;
  int row0, nrows;                 // packed rows (token, head) of this CTA
  int head0, pack, tok0;           // row r: token tok0 + r / pack of the sequence, head head0 + r % pack
  int qo_base, kv_len, off, page_base;
  int first, last;                 // entries of the page list: logical pages, or places of the selection
  const int32_t* blocks;           // selection
};

template <int NT, bool SPARSE>
__global__ void __launch_bounds__(kThreads, Cfg<NT>::CTAS) kv4_decode_kernel(const __grid_constant__ MsaFmhaParams p) {
  using C = Cfg<NT>;
  extern __shared__ __align__(16) unsigned char smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  unsigned char* ring = smem + warp * C::STAGES * 2 * C::HALF;

  // ---------------- the item ----------------
  const int h_r = p.num_qo_heads / p.num_kv_heads;
  const int rg = blockIdx.y * (8 * NT);                      // first row of this CTA's group
  Item it;
  int first_blocks = -1;                                     // this lane's entry of a selection: on its way before the loads that depend on the batch item
  if constexpr (!SPARSE) {
    const MsaWorkItem w = p.work[blockIdx.x];
    it.b = chk(w.batch, 0, p.batch, p.status);
    it.head0 = chk(w.head0, 0, p.num_qo_heads, p.status);
    it.split = chk(w.split, 0, p.num_splits, p.status);
    it.pack = p.pack; it.tok0 = 0;
    it.row0 = w.row0 + rg; it.nrows = min(8 * NT, w.num_rows - rg);
    it.first = w.kv_tile_begin; it.last = w.kv_tile_end;
    it.kvh = it.head0 / h_r;
  } else {
    int idx = blockIdx.x;
    it.split = idx % p.num_splits; idx /= p.num_splits;
    it.kvh = idx % p.num_kv_heads;
    const int t = idx / p.num_kv_heads;
    const int per = (p.kv_block_num + p.num_splits - 1) / p.num_splits;
    it.first = it.split * per;
    it.last = min(p.kv_block_num, it.first + per);
    it.blocks = p.kv_block_indexes + t * p.kbi_stride_tok + it.kvh * p.kbi_stride_head;
    if (it.first + lane < it.last) first_blocks = it.blocks[it.first + lane];
    if (t >= p.qo_start[p.batch]) return;                    // a padded row, behind the last sequence: left as it was
    it.b = chk(p.token_batch[t], 0, p.batch, p.status);
    it.head0 = it.kvh * h_r; it.pack = h_r;
    it.tok0 = t - p.qo_start[it.b];
    it.row0 = rg; it.nrows = min(8 * NT, h_r - rg);
  }
  if (it.nrows <= 0) return;
  it.qo_base = p.qo_start[it.b];
  it.kv_len = p.kv_len[it.b];
  it.off = min(p.qo_offset[it.b], it.kv_len);                // (no sum below passes 32 bits)
  it.page_base = p.kv_page_indptr[it.b];
  // keys that rows may see: row r sees keys below lim(r), which grows with r
  auto lim = [&](int r) -> int { return min(it.kv_len, it.tok0 + (it.row0 + min(r, it.nrows - 1)) / it.pack + it.off + 1); };
  const int lim_first = lim(0), lim_last = lim(it.nrows - 1);

  // ---------------- this warp's list of pages, and the copies ----------------
  // (none where the table is empty: `physical` then has nothing to read)
  const int n_tiles = p.num_logical_pages <= 0 ? 0 : max(0, SPARSE ? it.last - it.first : min(it.last, (lim_last + kKvTile - 1) / kKvTile) - it.first);
  // entries of the list, one a lane: physical pages, and logical pages of a selection or the next physical pages
  auto physical = [&](int lp) -> int {                       // in bounds whatever the table holds, and however short it is
    const int at = chk(it.page_base + lp, 0, p.num_logical_pages, p.status);
    return min(max(chk(p.kv_indices[min(at, p.num_logical_pages - 1)], 0, static_cast<int>(p.kv_extent), p.status), 0), static_cast<int>(p.kv_extent) - 1);
  };
  const unsigned char* const k_head = static_cast<const unsigned char*>(p.k) + it.kvh * p.k_stride_head + warp * kCodeBytes + 16 * lane;
  const unsigned char* const v_head = static_cast<const unsigned char*>(p.v) + it.kvh * p.v_stride_head + warp * kCodeBytes + 16 * lane;
  int phys = -1, aux = -1;
  auto load_entries = [&](int j0) {
    if constexpr (SPARSE) {
      aux = j0 == 0 ? first_blocks : (j0 + lane < n_tiles ? it.blocks[it.first + j0 + lane] : -1);
      phys = aux >= 0 && aux < (lim_last + kKvTile - 1) / kKvTile ? physical(aux) : -1;
    } else {
      phys = j0 > 0 ? aux : (lane < n_tiles ? physical(it.first + lane) : -1);
      aux = j0 + 32 + lane < n_tiles ? physical(it.first + j0 + 32 + lane) : -1;
    }
  };
  // Page j of the list into a stage that no lane reads any more; its first key (of this warp), negative if none of it is seen.
  auto fetch = [&](int j, int stage) {
    if ((j & 31) == 0) load_entries(j);
    const int page = __shfl_sync(0xffffffffu, phys, j & 31);
    const int lp = SPARSE ? __shfl_sync(0xffffffffu, aux, j & 31) : it.first + j;
    if (page >= 0) {
      const uint32_t dst = smem_u32(ring) + stage * 2 * C::HALF + 16 * lane;
      const unsigned char* k = k_head + page * p.k_stride_page;
      const unsigned char* v = v_head + page * p.v_stride_page;
#pragma unroll
      for (int i = 0; i < kCodeBytes / 512; ++i) cp_async16(dst + 512 * i, k + 512 * i);
#pragma unroll
      for (int i = 0; i < kCodeBytes / 512; ++i) cp_async16(dst + C::HALF + 512 * i, v + 512 * i);
      // scales: K by the first half of the warp, V by the second
      cp_async16(dst + kCodeBytes + (lane < 16 ? 0 : C::HALF - 256), (lane < 16 ? k : v - 256) + (kKv4ScaleOffset - warp * (kCodeBytes - kScaleBytes)));
    }
    return page >= 0 ? lp * kKvTile + kKeys * warp : -1;
  };
  int keys[C::STAGES];
#pragma unroll
  for (int j = 0; j < C::STAGES; ++j) {
    keys[j] = j < n_tiles ? fetch(j, j) : -1;
    cp_async_commit();                                       // of fewer pages too: the waits below count groups
  }

  // Q^T: warp n converts rows 8 n .. 8 n + 7 for all warps.
  const int g = lane >> 2, t4 = lane & 3;
  if (warp < NT) {
    const int r = 8 * warp + g;
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
    e = max(e, -126);                                        // 2^-e is a normal number
    // The factor of the scores is made positive (its sign goes to Q), so that the largest score has the largest exponent.
    const float scale = p.sm_scale * (p.k_scale_head ? p.k_scale_head[it.kvh] : 1.f) * kLog2e;
    const float up = copysignf(scale == 0.f ? 0.f : __uint_as_float(static_cast<uint32_t>(127 - e) << 23), scale);
    uint32_t h[16];
#pragma unroll
    for (int c = 0; c < 16; ++c) h[c] = pack2<true>(x[2 * c] * up, x[2 * c + 1] * up);
#pragma unroll
    for (int c = 0; c < 4; ++c)
      *reinterpret_cast<uint4*>(smem + C::OFF_Q + ((c * NT + warp) * 32 + lane) * 16) = make_uint4(h[4 * c], h[4 * c + 1], h[4 * c + 2], h[4 * c + 3]);
    if (t4 == 0) {
      reinterpret_cast<int*>(smem + C::OFF_LIM)[r] = lim(r);
      reinterpret_cast<float*>(smem + C::OFF_FAC)[r] = scale == 0.f ? 1.f : fabsf(scale) * __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
    }
  }
  __syncthreads();

  float m[NT][2];                                            // of rows 8 n + 2 t4 and the next one: maximum - kPOffset,
  uint64_t l[NT];                                            // sums of P, two floats
  float o[8][NT][4];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
#pragma unroll
    for (int c = 0; c < 2; ++c) m[n][c] = kNoMax;
    l[n] = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int c = 0; c < 4; ++c) o[i][n][c] = 0.f;
  }

  const unsigned char* q_at = smem + C::OFF_Q + 16 * lane;
  const int k_code = 64 * key_at(g) + 16 * t4;
  const int k_scale = kCodeBytes + 8 * key_at(g) + 2 * t4;
  const int v_key[2] = {key_at(2 * t4), key_at(2 * t4 + 1)};

  int stage = 0;
#pragma unroll 1
  for (int j = 0; j < n_tiles; ++j) {
    cp_async_wait<C::STAGES - 1>();
    __syncwarp();
    const int key0 = keys[0];
    const unsigned char* kt = ring + stage * 2 * C::HALF;
    unsigned char* vt = ring + stage * 2 * C::HALF + C::HALF;
    if (key0 >= 0) {
      // ---- S^T: two steps of 16 keys ----
      float s[2][NT][4];
      // 16 rows: half of a thread's codes of a key at a time, or there are too few registers
      constexpr int W = NT == 1 ? 4 : 2;
      uint32_t code[2][2][W];
      uint32_t sc[2][2];                                     // scales of this thread's two blocks of a key
#pragma unroll
      for (int u = 0; u < 2; ++u) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          sc[u][r] = kv4_scales_to_half(*reinterpret_cast<const uint16_t*>(kt + k_scale + 8 * (16 * u + 8 * r)));
        }
      }
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        if (c % W == 0) {
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int r = 0; r < 2; ++r) load_words(kt + k_code + 64 * (16 * u + 8 * r) + 4 * c, code[u][r]);
        }
        uint4 qf[NT];
#pragma unroll
        for (int n = 0; n < NT; ++n) qf[n] = *reinterpret_cast<const uint4*>(q_at + (c * NT + n) * 512);
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          uint32_t a[4], b[4];
          kv4_to_half(code[u][0][c % W], a);
          kv4_to_half(code[u][1][c % W], b);
#pragma unroll
          for (int i = 0; i < 4; ++i) { a[i] = half2_mul_by(a[i], sc[u][0], c >= 2); b[i] = half2_mul_by(b[i], sc[u][1], c >= 2); }
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            if (c == 0) mma_f16_first(s[u][n], a[0], b[0], a[1], b[1], qf[n].x, qf[n].y);
            else mma_f16(s[u][n], a[0], b[0], a[1], b[1], qf[n].x, qf[n].y);
          }
#pragma unroll
          for (int n = 0; n < NT; ++n) mma_f16(s[u][n], a[2], b[2], a[3], b[3], qf[n].z, qf[n].w);
        }
      }
      // ---- softmax: mask, exponents, a maximum that may lag ----
      float fac[NT][2];                                      // score * factor = exponent of two
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const float2 f = *reinterpret_cast<const float2*>(smem + C::OFF_FAC + 4 * (8 * n + 2 * t4));
        fac[n][0] = f.x; fac[n][1] = f.y;
      }
      if (key0 + kKeys > lim_first) {
        uint32_t nx = 0, ny = 0;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const int2 f = *reinterpret_cast<const int2*>(smem + C::OFF_LIM + 4 * (8 * n + 2 * t4));
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int c = 0; c < 4; ++c)
              if (key0 + 16 * u + 8 * (c >> 1) + key_at(g) >= (c & 1 ? f.y : f.x)) s[u][n][c] = -INFINITY;
        }
        // P is 0 where a row does not see a key, but 0 x NaN is not.  Behind the last row's keys, where maybe nobody wrote, V becomes
        // zero; a NaN that some of the rows see is taken out of V and put into their sums.
        uint2* vs = reinterpret_cast<uint2*>(vt + kCodeBytes + 8 * lane);
        if (key0 + lane >= lim_last) *vs = make_uint2(0, 0);
        else if (lim_first < lim_last && key0 + lane >= lim_first) nx = nan_bytes(vs->x), ny = nan_bytes(vs->y);
        if (__any_sync(0xffffffffu, nx | ny)) {
          if (nx | ny) *vs = make_uint2(vs->x & ~nx, vs->y & ~ny);
          uint32_t at = 0;                                   // keys with a NaN in this thread's 16 elements
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const uint32_t v = __ballot_sync(0xffffffffu, ((i < 4 ? nx : ny) >> (8 * (i & 3))) & 1);
            if (i == g) at = v;
          }
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              const int seen = reinterpret_cast<const int*>(smem + C::OFF_LIM)[8 * n + 2 * t4 + c] - key0;
              if (seen > 0 && (at & (0xffffffffu >> (32 - min(seen, 32)))) != 0) {
#pragma unroll
                for (int i = 0; i < 8; ++i) o[i][n][c] = o[i][n][c + 2] = __int_as_float(0x7fc00000);
              }
            }
        }
        __syncwarp();
      }
      bool raise = false;
      float top[NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          top[n][c] = fmaxf(max3(s[0][n][c], s[0][n][c + 2], s[1][n][c]), s[1][n][c + 2]) * fac[n][c];
          raise |= top[n][c] > m[n][c] + (kPOffset + kRescale);
        }
      if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float k2[2];
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float x = top[n][c];
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, d));
            x = fmaxf(x - kPOffset, m[n][c]);
            const float keep = exp2_fast(m[n][c] - x);
            m[n][c] = x;
            k2[c] = keep;
#pragma unroll
            for (int i = 0; i < 8; ++i) { o[i][n][c] *= keep; o[i][n][c + 2] *= keep; }
          }
          l[n] = f2_fma(l[n], f2_pack(k2[0], k2[1]), 0);
        }
      }
      uint32_t pt[2][NT][2];                                 // P^T as an operand: [step][rows][keys 0-7, keys 8-15]
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const uint64_t f = f2_pack(fac[n][0], fac[n][1]), shift = f2_pack(-m[n][0], -m[n][1]);
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float x0, x1;
            f2_unpack(f2_fma(f2_pack(s[u][n][2 * h], s[u][n][2 * h + 1]), f, shift), x0, x1);
            const float p0 = exp2_fast(x0), p1 = exp2_fast(x1);
            l[n] = f2_add(l[n], f2_pack(p0, p1));
            pt[u][n][h] = transpose8x8(pack2<true>(p0, p1));
          }
      }
      // ---- O^T ----
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        uint32_t code[4][2], sb[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int key = v_key[r & 1] + 16 * u + 8 * (r >> 1);
          load_words(vt + 64 * key + 8 * g, code[r]);
          sb[r] = vt[kCodeBytes + 8 * key + g];
        }
        const uint32_t s01 = kv4_scales_to_half(static_cast<uint16_t>(__byte_perm(sb[0], sb[1], 0x0040)));
        const uint32_t s23 = kv4_scales_to_half(static_cast<uint16_t>(__byte_perm(sb[2], sb[3], 0x0040)));
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          // the codes of two keys side by side in a byte: even elements, odd elements
          uint32_t x[4][4];
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const uint32_t ca = code[2 * r][w], cb = code[2 * r + 1][w];
            kv4_to_half((ca & 0x0f0f0f0fu) | ((cb << 4) & 0xf0f0f0f0u), x[2 * r]);
            kv4_to_half(((ca >> 4) & 0x0f0f0f0fu) | (cb & 0xf0f0f0f0u), x[2 * r + 1]);
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t a0 = half2_mul(x[0][i], s01), a1 = half2_mul(x[1][i], s01);
            const uint32_t a2 = half2_mul(x[2][i], s23), a3 = half2_mul(x[3][i], s23);
#pragma unroll
            for (int n = 0; n < NT; ++n) mma_f16(o[4 * w + i][n], a0, a1, a2, a3, pt[u][n][0], pt[u][n][1]);
          }
        }
      }
    }
    __syncwarp();                                          // all lanes have read the stage
#pragma unroll
    for (int i = 0; i + 1 < C::STAGES; ++i) keys[i] = keys[i + 1];
    if (j + C::STAGES < n_tiles) keys[C::STAGES - 1] = fetch(j + C::STAGES, stage);
    cp_async_commit();                                       // an empty group at the end
    if (++stage == C::STAGES) stage = 0;
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
  __syncthreads();                                           // the ring is no longer read, and no copy is on its way
  // ---------------- the four states of a row become one ----------------
  float* s_o = reinterpret_cast<float*>(smem);               // [warp][row][kLdO]
  float* s_m = s_o + kWarps * 8 * NT * kLdO;                 // [warp][row][2]: maximum - kPOffset, sum of P
  static_assert((kWarps * 8 * NT * (kLdO + 2)) * 4 <= C::OFF_Q, "states fit the ring");
  {
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int r = warp * 8 * NT + 8 * n + 2 * t4 + c;
#pragma unroll
        for (int i = 0; i < 8; i += 2)
          *reinterpret_cast<float4*>(s_o + r * kLdO + 16 * g + 2 * i) = make_float4(o[i][n][c], o[i][n][c + 2], o[i + 1][n][c], o[i + 1][n][c + 2]);
        if (g == 0) { s_m[2 * r] = m[n][c]; s_m[2 * r + 1] = sums[n][c]; }
      }
  }
  __syncthreads();
  // 16 threads a row, 8 columns each
  const int c16 = threadIdx.x & 15;
#pragma unroll
  for (int r0 = 0; r0 < 8 * NT; r0 += 8) {
    const int r = r0 + (threadIdx.x >> 4);
    if (r >= it.nrows) continue;
    float top = kNoMax;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) top = fmaxf(top, s_m[2 * (w * 8 * NT + r)]);
    float sum = 0.f, acc[8];
#pragma unroll
    for (int c = 0; c < 8; ++c) acc[c] = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const int at = w * 8 * NT + r;
      const float f = exp2_fast(s_m[2 * at] - top);
      sum += f * s_m[2 * at + 1];
#pragma unroll
      for (int c = 0; c < 8; ++c) acc[c] += f * s_o[at * kLdO + 8 * c16 + c];
    }
    const int row = it.row0 + r;
    const int64_t tok = it.qo_base + it.tok0 + row / it.pack;
    const int head = it.head0 + row % it.pack;
    const bool none = sum == 0.f;
    const float vs = p.v_scale_head ? p.v_scale_head[it.kvh] : 1.f;
    const float inv = none ? 0.f : vs / sum;
    const float lse = none ? -INFINITY : (top + log2f(sum)) * kLn2;
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

template <int NT, bool SPARSE>
int launch(const MsaFmhaParams& p, int rows, cudaStream_t stream) {
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess) return MSA_ERR_LAUNCH;
  static bool ready[64] = {};
  if (device < 0 || device >= 64 || !ready[device]) {
    if (cudaFuncSetAttribute(kv4_decode_kernel<NT, SPARSE>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<NT>::BYTES) != cudaSuccess) return MSA_ERR_LAUNCH;
    if (device >= 0 && device < 64) ready[device] = true;
  }
  const int64_t items = SPARSE ? static_cast<int64_t>(p.total_q) * p.num_kv_heads * p.num_splits : p.num_work;
  if (items > 0x7fffffffLL) return MSA_ERR_TOO_LARGE;
  if (items == 0) return MSA_OK;
  const dim3 grid(static_cast<unsigned>(items), (rows + 8 * NT - 1) / (8 * NT));
  // A plain launch, and the next kernel comes up at the end of this one: CTAs that came up while the kernel before ends would fill
  // the SMs that are free first, three or four of the longest items on one (24 ragged sequences x 4 heads: 116 us instead of
  // 89), and a merge that came up early would take the place of CTAs here (82 us instead of 62, finer cut).
  kv4_decode_kernel<NT, SPARSE><<<grid, kThreads, Cfg<NT>::BYTES, stream>>>(p);
  return cudaGetLastError() == cudaSuccess ? MSA_OK : MSA_ERR_LAUNCH;
}

}  // namespace
}  // namespace kv4

int fmha_kv4_tc_launch(const MsaFmhaParams& p, int rows, cudaStream_t stream);

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
  if (p.total_q == 0) return MSA_OK;
  if (p.kv_extent == 0 || p.num_logical_pages < 0) return MSA_ERR_BAD_ARG;
  if (!sparse && rows > 16) return fmha_kv4_tc_launch(p, rows, stream);
  if (sparse) return rows <= 8 ? kv4::launch<1, true>(p, rows, stream) : kv4::launch<2, true>(p, rows, stream);
  return rows <= 8 ? kv4::launch<1, false>(p, rows, stream) : kv4::launch<2, false>(p, rows, stream);
}
}  // namespace msa
