// Norm of every query and key head, rotation, and the write of keys and values into the paged cache, in one pass.
//
//   y = x / sqrt(mean(x^2) + eps) * w                                        over the 128 elements of a head
//   (y_i, y_j) -> (y_i cos t - y_j sin t, y_j cos t + y_i sin t)            for pair n of the rotary elements,
//   t = position[axis_n] * inv_freq_n;  j = i + rotary / 2, or i + 1 (interleaved)
//
// Angles: the frequencies come as fractions of a turn in 64-bit fixed point, so position * frequency modulo a turn is one
// wrapping integer product, exact to 2^-64 turns times the position at any position; the cosine and sine of what is left
// are taken once per token and pair and shared by all heads.
//
// Keys that go into a cache are normed and rotated in 64 bits, rounded to 32 bits, from there to bf16 (the two steps of a cast of a
// 64-bit tensor; a key within 2^-24 of itself of a border of two bf16 values may become the border and go to the even one), and
// quantised from there: which bf16, e4m3 or e2m1 value a key next to a border gets does not depend on the order of a sum.  (They are
// a tenth of the rows or less.)  All else is computed in 32 bits and rounded to bf16; queries in e4m3 are divided by their scale and
// rounded from there, as a call that quantises bf16 queries does.
//
// 4-bit rows: 16 elements share an e4m3 scale s = round(max|x| / 6), at least 2^-9; the codes are the e2m1 roundings of x / s
// (divisions as IEEE has them: an x on a border goes to the even code).  A NaN makes the scale of its 16 elements NaN.
//
// A warp works on four heads at a time, 8 lanes each.  A lane has eight pairs: two chunks of eight elements (16 bytes), rotary / 2
// apart (one after the other if interleaved, and in what is not rotated), so that a rotation needs no other lane.
#include <algorithm>

#include <cuda_fp4.h>

#include "common.cuh"
#include "kv4.cuh"
#include "nvtx_range.h"

namespace msa {
namespace {

// Elements of a row that a lane has: x[0..7] at a, x[8..15] at b.
struct Lane {
  int a, b;
  bool rotary;
};
template <bool PAIRS>
__device__ __forceinline__ Lane lane_of(int l, int rotary) {
  Lane v;
  v.rotary = 16 * l < rotary;
  v.a = v.rotary && !PAIRS ? 8 * l : 16 * l;
  v.b = v.rotary && !PAIRS ? rotary / 2 + 8 * l : 16 * l + 8;
  return v;
}

__device__ __forceinline__ void unpack8(const uint4& r, float* x) {
  const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) { x[2 * i] = __uint_as_float(w[i] << 16); x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
}
__device__ __forceinline__ uint4 pack8(const float* x) {
  return make_uint4(pack2<false>(x[0], x[1]), pack2<false>(x[2], x[3]), pack2<false>(x[4], x[5]), pack2<false>(x[6], x[7]));
}
__device__ __forceinline__ float to_bf16(float x) { return __bfloat162float(__float2bfloat16_rn(x)); }
__device__ __forceinline__ uint2 pack8_e4m3(const float* x, float scale) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    w[i] = __nv_cvt_float2_to_fp8x2(make_float2(__fdiv_rn(x[2 * i], scale), __fdiv_rn(x[2 * i + 1], scale)), __NV_SATFINITE, __NV_E4M3);
  return make_uint2(w[0] | (w[1] << 16), w[2] | (w[3] << 16));
}

// A lane's elements of the weight of a head, 1 without one.
__device__ __forceinline__ void load_weight(const void* w, int dtype, int64_t row, const Lane& v, float (&x)[16]) {
  if (!w) {
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = 1.f;
  } else if (dtype == MSA_DT_F32) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float4 f = *reinterpret_cast<const float4*>(static_cast<const float*>(w) + row + (i < 2 ? v.a : v.b) + 4 * (i & 1));
      x[4 * i] = f.x; x[4 * i + 1] = f.y; x[4 * i + 2] = f.z; x[4 * i + 3] = f.w;
    }
  } else {
    const __nv_bfloat16* p = static_cast<const __nv_bfloat16*>(w) + row;
    unpack8(*reinterpret_cast<const uint4*>(p + v.a), x);
    unpack8(*reinterpret_cast<const uint4*>(p + v.b), x + 8);
  }
}

// Norm and rotation of the head that 8 lanes hold.  The factor of the norm is the same for all elements, so it comes last and the
// rotation does not wait for the sum.  32 bits: packed pairs, x[0..3] the first and x[4..7] the second elements of the pairs to turn.
struct TurnF { uint64_t c[4], s[4]; };                     // cosines and sines
__device__ __forceinline__ uint64_t f2_mul(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
template <bool NORM>
__device__ __forceinline__ void norm_rotate_f(uint64_t (&x)[8], const uint64_t (&w)[8], float eps, bool turn, const TurnF& t) {
  float r = 1.f;
  if (NORM) {
    uint64_t s0 = f2_mul(x[0], x[0]), s1 = f2_mul(x[1], x[1]);
#pragma unroll
    for (int i = 2; i < 8; i += 2) { s0 = f2_fma(x[i], x[i], s0); s1 = f2_fma(x[i + 1], x[i + 1], s1); }
    float lo, hi;
    f2_unpack(f2_add(s0, s1), lo, hi);
    float sum = lo + hi;
#pragma unroll
    for (int d = 4; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d, 8);
    r = rsqrtf(sum * (1.f / kHeadDim) + eps);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = f2_mul(x[i], w[i]);
  }
  if (turn) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint64_t p = x[i], q = x[i + 4];
      x[i] = f2_fma(q, t.s[i] ^ 0x8000000080000000ull, f2_mul(p, t.c[i]));
      x[i + 4] = f2_fma(p, t.s[i], f2_mul(q, t.c[i]));
    }
  }
  if (NORM) {
    const uint64_t rr = f2_pack(r, r);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = f2_mul(x[i], rr);
  }
}

// 64 bits, rounded to 32 and to bf16.  cs: of pair i of this lane at 8 i.
template <bool PAIRS>
__device__ __forceinline__ void norm_rotate_d(float (&x)[16], const float (&w)[16], bool norm, float eps, bool turn, const double2* cs) {
  double z[16], r = 1.0;
#pragma unroll
  for (int i = 0; i < 16; ++i) z[i] = x[i];
  if (norm) {
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < 16; ++i) sum += z[i] * z[i];
#pragma unroll
    for (int d = 4; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d, 8);
    r = rsqrt(sum * (1.0 / kHeadDim) + static_cast<double>(eps));
#pragma unroll
    for (int i = 0; i < 16; ++i) z[i] *= static_cast<double>(w[i]);
  }
  if (turn) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const double2 t = cs[8 * i];
      double& p = z[PAIRS ? 2 * i : i];
      double& q = z[PAIRS ? 2 * i + 1 : i + 8];
      const double p0 = p, q0 = q;
      p = p0 * t.x - q0 * t.y;
      q = q0 * t.x + p0 * t.y;
    }
  }
#pragma unroll
  for (int i = 0; i < 16; ++i) x[i] = to_bf16(static_cast<float>(z[i] * r));
}

// Eight elements of a block of 16 as codes, and the block's scale; top: its largest magnitude.  `short_y`: the y have 8
// significant bits.  Then y / s is a border of two codes or at least 2^-8 of it away (borders times scales have 7 bits), and the
// product with 1 / s, rounded to 16 bits, is on the same side of it or on it: a third of the time of a division.
__device__ __forceinline__ uint32_t codes8(const float* y, uint32_t top, bool short_y, __nv_fp8_storage_t& sb) {
  float s = __fdiv_rn(__uint_as_float(top), 6.f);
  s = s < kKv4MinScale ? kKv4MinScale : s;
  sb = __nv_cvt_float_to_fp8(s, __NV_SATFINITE, __NV_E4M3);
  const __half_raw sh = __nv_cvt_fp8_to_halfraw(sb, __NV_E4M3);
  const float sf = __half2float(*reinterpret_cast<const __half*>(&sh));
  float q[8];
  if (short_y) {
    const float inv = __frcp_rn(sf);
#pragma unroll
    for (int i = 0; i < 8; ++i) q[i] = __uint_as_float((__float_as_uint(y[i] * inv) + 0x40u) & ~0x7fu);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) q[i] = __fdiv_rn(y[i], sf);
  }
  uint32_t codes = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    codes |= static_cast<uint32_t>(__nv_cvt_float2_to_fp4x2(make_float2(q[2 * i], q[2 * i + 1]), __NV_E2M1, cudaRoundNearest)) << (8 * i);
  return codes;
}

// Writes a lane's bf16-valued elements of a row of the cache.  All lanes of the warp take part.
__device__ __forceinline__ void store_row(void* cache, int dtype, int64_t at, int64_t stride_tok, int r, const Lane& v, int l, const float (&x)[16],
                                          float scale, bool write) {
  if (dtype == MSA_DT_KV4) {
    float y[16];
    uint32_t top[2] = {0, 0};                                // as integers: a NaN is above every number
#pragma unroll
    for (int i = 0; i < 16; ++i) y[i] = x[i];
    // a power of two (that has a reciprocal): the division is a product, and exact
    const uint32_t se = __float_as_uint(scale);
    const bool two = (se & 0x807fffffu) == 0 && se >= 0x01000000u && se <= 0x7e000000u;
    if (two) {
      const float inv = __uint_as_float(0x7f000000u - se);
#pragma unroll
      for (int i = 0; i < 16; ++i) y[i] *= inv;
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) y[i] = __fdiv_rn(y[i], scale);
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) top[i >> 3] = max(top[i >> 3], __float_as_uint(y[i]) & 0x7fffffffu);
    // 16 elements that share a scale: one chunk of two lanes, or both chunks of this one
    const bool apart = v.b != v.a + 8;
    const uint32_t far0 = __shfl_xor_sync(0xffffffffu, top[0], 1), far1 = __shfl_xor_sync(0xffffffffu, top[1], 1);
    if (apart) { top[0] = max(top[0], far0); top[1] = max(top[1], far1); }
    else top[0] = top[1] = max(top[0], top[1]);
    __nv_fp8_storage_t sa, sb;
    const uint32_t ca = codes8(y, top[0], two, sa), cb = codes8(y + 8, top[1], two, sb);
    if (write) {
      unsigned char* tile = static_cast<unsigned char*>(cache) + at;
      unsigned char* code = tile + r * kKv4CodeBytes;
      unsigned char* sc = tile + kKv4ScaleOffset + r * kKv4ScaleBytes;
      *reinterpret_cast<uint32_t*>(code + v.a / 2) = ca;
      *reinterpret_cast<uint32_t*>(code + v.b / 2) = cb;
      if (!apart || !(l & 1)) sc[v.a / 16] = sa;
      if (apart && !(l & 1)) sc[v.b / 16] = sb;
    }
  } else if (write && dtype == MSA_DT_E4M3) {
    unsigned char* row = static_cast<unsigned char*>(cache) + at + r * stride_tok;
    *reinterpret_cast<uint2*>(row + v.a) = pack8_e4m3(x, scale);
    *reinterpret_cast<uint2*>(row + v.b) = pack8_e4m3(x + 8, scale);
  } else if (write) {
    __nv_bfloat16* row = static_cast<__nv_bfloat16*>(cache) + at + r * stride_tok;
    *reinterpret_cast<uint4*>(row + v.a) = pack8(x);
    *reinterpret_cast<uint4*>(row + v.b) = pack8(x + 8);
  }
}

// Elements of the two chunks <-> packed pairs, the first elements of the pairs to turn in x[0..3].
template <bool PAIRS>
__device__ __forceinline__ void pairs_of(const float (&y)[16], uint64_t (&x)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (PAIRS) { x[i] = f2_pack(y[4 * i], y[4 * i + 2]); x[i + 4] = f2_pack(y[4 * i + 1], y[4 * i + 3]); }
    else { x[i] = f2_pack(y[2 * i], y[2 * i + 1]); x[i + 4] = f2_pack(y[2 * i + 8], y[2 * i + 9]); }
  }
}
template <bool PAIRS>
__device__ __forceinline__ void elements_of(const uint64_t (&x)[8], float (&y)[16]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (PAIRS) { f2_unpack(x[i], y[4 * i], y[4 * i + 2]); f2_unpack(x[i + 4], y[4 * i + 1], y[4 * i + 3]); }
    else { f2_unpack(x[i], y[2 * i], y[2 * i + 1]); f2_unpack(x[i + 4], y[2 * i + 8], y[2 * i + 9]); }
  }
}

// A warp has one of `parts` parts of a token's heads, four heads (a unit) at a time: units part, part + parts, ... of the queries,
// then of the keys, then of the values.  The next kBatch query units are on their way while as many are worked on.
//
// Bound by memory, and by what its instructions leave of that: 8 192 tokens of 64 + 8 heads, 302 MB, 60 us, where a copy of as
// many bytes takes 50 and this kernel without norm and rotation 52.  CTAs of one warp, so that a warp that is through makes place for the next one:
// 62 us with four (32 768 tokens of 64 + 2 x 4 heads into a 4-bit cache: 231 and 247 us).  More units on their way by fewer
// warps, or more warps with fewer registers: 63 to 70 us.
constexpr int kBatch = 2;
constexpr int kCtas = 20;                                    // of an SM

template <bool PAIRS, bool NORM, bool Q8>
__global__ void __launch_bounds__(32, kCtas) norm_rope_kernel(const __grid_constant__ MsaNormRopeArgs a, int parts) {
  chain_begin();
  __shared__ double2 s_cs[kHeadDim / 2];
  const int lane = threadIdx.x, l = lane & 7, sub = lane >> 3;
  const int t = blockIdx.x / parts, part = blockIdx.x % parts;
  const Lane v = lane_of<PAIRS>(l, a.rotary);
  const int off = v.b - v.a;
  const int q_units = a.q ? (a.num_qo_heads + 3) / 4 : 0, kv_units = (a.num_kv_heads + 3) / 4;
  const int q_whole = a.q ? a.num_qo_heads / 4 : 0;          // units of four heads
  const __nv_bfloat16* q_at = static_cast<const __nv_bfloat16*>(a.q) + t * a.q_stride_tok + (4 * part + sub) * a.q_stride_head + v.a;
  const int64_t q_step = 4 * parts * a.q_stride_head;
  uint4 raw[kBatch][2];
  auto load_q = [&](const __nv_bfloat16* p, uint4 (&r)[kBatch][2]) {
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      r[i][0] = *reinterpret_cast<const uint4*>(p + i * q_step);
      r[i][1] = *reinterpret_cast<const uint4*>(p + i * q_step + off);
    }
  };
  if (part + (kBatch - 1) * parts < q_whole) load_q(q_at, raw);
  const int slot = a.slot_map ? a.slot_map[t] : -1;
  TurnF turn = {};
  if (a.rotary > 0) {
    for (int n = lane; n < a.rotary / 2; n += 32) {
      const int64_t at = a.axis[n] * a.pos_stride_axis + t;
      const int64_t pos = a.pos_int64 ? static_cast<const int64_t*>(a.positions)[at] : static_cast<const int32_t*>(a.positions)[at];
      const int64_t turns = static_cast<int64_t>(static_cast<uint64_t>(pos) * static_cast<uint64_t>(a.turns[n]));   // modulo a turn
      double2 d;
      sincospi(static_cast<double>(turns) * 0x1p-63, &d.y, &d.x);
      s_cs[(n & 7) * 8 + (n >> 3)] = d;                      // pair i of lane l at 8 i + l
    }
    __syncwarp();
    if (v.rotary) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const double2 d = s_cs[16 * i + l], e = s_cs[16 * i + 8 + l];
        turn.c[i] = f2_pack(static_cast<float>(d.x), static_cast<float>(e.x));
        turn.s[i] = f2_pack(static_cast<float>(d.y), static_cast<float>(e.y));
      }
    }
  }
  uint64_t w8[8] = {};
  auto load_w8 = [&](const void* weight, int64_t row) {
    float w[16];
    load_weight(weight, a.weight_dtype, row, v, w);
    pairs_of<PAIRS>(w, w8);
  };
  auto turned = [&](const uint4 (&r)[2], float (&y)[16]) {
    uint64_t x[8];
    unpack8(r[0], y);
    unpack8(r[1], y + 8);
    pairs_of<PAIRS>(y, x);
    norm_rotate_f<NORM>(x, w8, a.eps, v.rotary, turn);
    elements_of<PAIRS>(x, y);
  };
  const int64_t out_at = t * a.q_out_stride_tok + (4 * part + sub) * a.q_out_stride_head + v.a;
  const int64_t out_step = 4 * parts * a.q_out_stride_head;
  auto store_q = [&](int64_t at, float (&y)[16]) {
    if (Q8) {
#pragma unroll
      for (int n = 0; n < 16; ++n) y[n] = to_bf16(y[n]);
      unsigned char* out = static_cast<unsigned char*>(a.q_out) + at;
      *reinterpret_cast<uint2*>(out) = pack8_e4m3(y, a.q_scale);
      *reinterpret_cast<uint2*>(out + off) = pack8_e4m3(y + 8, a.q_scale);
    } else {
      __nv_bfloat16* out = static_cast<__nv_bfloat16*>(a.q_out) + at;
      *reinterpret_cast<uint4*>(out) = pack8(y);
      *reinterpret_cast<uint4*>(out + off) = pack8(y + 8);
    }
  };
  const bool w_head = NORM && a.q_weight_stride != 0;        // a weight for each head
  if (NORM && a.q) load_w8(a.q_weight, 0);
  int u = part, n_done = 0;                                  // n_done: units of this warp that are through
  for (; u + (kBatch - 1) * parts < q_whole; u += kBatch * parts, n_done += kBatch) {
    uint4 next[kBatch][2] = {};
    const bool more = u + (2 * kBatch - 1) * parts < q_whole;
    if (more) load_q(q_at + (n_done + kBatch) * q_step, next);
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      float y[16];
      if (w_head) load_w8(a.q_weight, (4 * (u + i * parts) + sub) * a.q_weight_stride);
      turned(raw[i], y);
      store_q(out_at + (n_done + i) * out_step, y);
    }
#pragma unroll
    for (int i = 0; i < kBatch; ++i) { raw[i][0] = next[i][0]; raw[i][1] = next[i][1]; }
  }
#pragma unroll 1
  for (; u < q_units; u += parts, ++n_done) {                // what is left; lanes past the last head have that one once more
    const int h = min(4 * u + sub, a.num_qo_heads - 1);
    const bool real = 4 * u + sub < a.num_qo_heads;
    const __nv_bfloat16* p = static_cast<const __nv_bfloat16*>(a.q) + t * a.q_stride_tok + h * a.q_stride_head + v.a;
    const uint4 r[2] = {*reinterpret_cast<const uint4*>(p), *reinterpret_cast<const uint4*>(p + off)};
    float y[16];
    if (w_head) load_w8(a.q_weight, h * a.q_weight_stride);
    turned(r, y);
    if (real) store_q(out_at + n_done * out_step, y);
  }
  if (!a.k && !a.v) return;
  const int page_size = max(a.page_size, 1), page = slot / page_size, row = slot - page * page_size;
  const bool has_slot = slot >= 0 && page < a.num_pages;
#ifdef MSA_BOUNDS_CHECK
  if (slot >= 0 && a.slot_map && !has_slot) chk(slot, 0, 0, a.status);
#endif
  const bool fine = a.k_cache != nullptr;                    // keys in 64 bits
  if (a.k && NORM && !fine) load_w8(a.k_weight, 0);
#pragma unroll 1
  for (u -= q_units; a.k && u < kv_units; u += parts) {
    const int h = min(4 * u + sub, a.num_kv_heads - 1);
    const bool real = 4 * u + sub < a.num_kv_heads;
    const __nv_bfloat16* p = static_cast<const __nv_bfloat16*>(a.k) + t * a.k_stride_tok + h * a.k_stride_head + v.a;
    const uint4 r[2] = {*reinterpret_cast<const uint4*>(p), *reinterpret_cast<const uint4*>(p + off)};
    float x[16];
    if (!fine && (NORM || a.rotary > 0)) {
      if (NORM && a.k_weight_stride) load_w8(a.k_weight, h * a.k_weight_stride);
      turned(r, x);
    } else {
      unpack8(r[0], x);
      unpack8(r[1], x + 8);
      if (NORM || a.rotary > 0) {
        float w[16];
        if (NORM) load_weight(a.k_weight, a.weight_dtype, h * a.k_weight_stride, v, w);
        norm_rotate_d<PAIRS>(x, w, NORM, a.eps, v.rotary, s_cs + l);
      }
    }
    if (a.k_out && real) {
      __nv_bfloat16* out = static_cast<__nv_bfloat16*>(a.k_out) + t * a.k_out_stride_tok + h * a.k_out_stride_head + v.a;
      *reinterpret_cast<uint4*>(out) = pack8(x);
      *reinterpret_cast<uint4*>(out + off) = pack8(x + 8);
    }
    if (a.k_cache)
      store_row(a.k_cache, a.cache_dtype, page * a.k_cache_stride_page + h * a.k_cache_stride_head, a.k_cache_stride_tok, row, v, l, x,
                a.k_scale * (a.k_scale_head ? a.k_scale_head[h] : 1.f), has_slot && real);
  }
#pragma unroll 1
  for (u -= a.k ? kv_units : 0; a.v && u < kv_units; u += parts) {
    const int h = min(4 * u + sub, a.num_kv_heads - 1);
    const __nv_bfloat16* p = static_cast<const __nv_bfloat16*>(a.v) + t * a.v_stride_tok + h * a.v_stride_head + v.a;
    float x[16];
    unpack8(*reinterpret_cast<const uint4*>(p), x);
    unpack8(*reinterpret_cast<const uint4*>(p + off), x + 8);
    store_row(a.v_cache, a.cache_dtype, page * a.v_cache_stride_page + h * a.v_cache_stride_head, a.v_cache_stride_tok, row, v, l, x,
              a.v_scale * (a.v_scale_head ? a.v_scale_head[h] : 1.f), has_slot && 4 * u + sub < a.num_kv_heads);
  }
}

// Rows of a 4-bit cache as bf16 (exact: a code has two significant bits, a scale four): 16 lanes a row.
__global__ void __launch_bounds__(256) kv4_read_kernel(const MsaKv4ReadArgs a) {
  chain_begin();
  const int l = threadIdx.x & 15;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 16 + (threadIdx.x >> 4);
  if (row >= static_cast<int64_t>(a.rows) * a.num_kv_heads) return;
  const int i = static_cast<int>(row / a.num_kv_heads), h = static_cast<int>(row % a.num_kv_heads);
  const int slot = a.slot_map[i];
  uint4 out = make_uint4(0, 0, 0, 0);
  if (slot >= 0 && slot / kKvTile < a.num_pages) {
    const unsigned char* tile = static_cast<const unsigned char*>(a.cache) + (slot / kKvTile) * a.stride_page + h * a.stride_head;
    const int r = slot % kKvTile;
    const uint32_t codes = *reinterpret_cast<const uint32_t*>(tile + r * kKv4CodeBytes + 4 * l);
    out = kv4_to_bf16(codes, tile[kKv4ScaleOffset + r * kKv4ScaleBytes + (l >> 1)]);
  }
#ifdef MSA_BOUNDS_CHECK
  else if (slot >= 0) chk(slot, 0, 0, a.status);
#endif
  *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(a.out) + row * kHeadDim + 8 * l) = out;
}

// Whole pages, in the order of a page table: out[e, head, 128, 128] = page kv_indices[e].  A block has a (page, head), 16 lanes a row as
// above, so that the writes of a warp are 512 contiguous bytes; memory bounds it.  A number that is no page is the nearest one, as in
// the kernels that read 4 bits: what is attended to was written.
__global__ void __launch_bounds__(256) kv4_unpack_kernel(const MsaKv4ReadArgs a) {
  chain_begin();
  const int l = threadIdx.x & 15;
  const int e = blockIdx.x, h = blockIdx.y;
  const int entry = a.slot_map[e], used = a.num_used ? *a.num_used : a.rows;         // (on their way together)
  if (e >= used || a.num_pages == 0) return;                 // behind the last page of a table that is longer than its use
  const int page = min(max(chk(entry, 0, a.num_pages, a.status), 0), a.num_pages - 1);
  const unsigned char* tile = static_cast<const unsigned char*>(a.cache) + page * a.stride_page + h * a.stride_head;
  __nv_bfloat16* out = static_cast<__nv_bfloat16*>(a.out) + (static_cast<int64_t>(e) * a.num_kv_heads + h) * (kKvTile * kHeadDim) + 8 * l;
#pragma unroll
  for (int r = threadIdx.x >> 4; r < kKvTile; r += 16) {
    const uint32_t codes = *reinterpret_cast<const uint32_t*>(tile + r * kKv4CodeBytes + 4 * l);
    *reinterpret_cast<uint4*>(out + r * kHeadDim) = kv4_to_bf16(codes, tile[kKv4ScaleOffset + r * kKv4ScaleBytes + (l >> 1)]);
  }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Rows of `bytes`-wide elements that are read or written 8 elements at a time.
bool rows_ok(const void* p, int64_t stride_tok, int64_t stride_head, int bytes) {
  const int unit = 8 * bytes;
  return (reinterpret_cast<uintptr_t>(p) % unit) == 0 && (stride_tok * bytes) % unit == 0 && (stride_head * bytes) % unit == 0;
}

bool cache_ok(const void* p, int dtype, int64_t page, int64_t head, int64_t tok) {
  if (dtype == MSA_DT_KV4) return aligned16(p) && page % 16 == 0 && head % 16 == 0;
  const int bytes = dtype == MSA_DT_E4M3 ? 1 : 2;
  return rows_ok(p, tok, head, bytes) && (page * bytes) % (8 * bytes) == 0;
}

}  // namespace
}  // namespace msa

extern "C" int msa_norm_rope(const MsaNormRopeArgs* pa, msa_stream_t stream) {
  using namespace msa;
  if (!pa) return MSA_ERR_BAD_ARG;
  const MsaNormRopeArgs& a = *pa;
  if (a.tokens < 0 || a.num_qo_heads < 0 || a.num_kv_heads < 0 || (!a.q && !a.k && !a.v)) return MSA_ERR_BAD_ARG;
  if (a.rotary < 0 || a.rotary > kHeadDim || a.rotary % 32) return MSA_ERR_UNSUPPORTED;
  if (a.rotary > 0 && (!a.positions || !a.turns || !a.axis)) return MSA_ERR_BAD_ARG;
  if (a.q) {
    if (!a.q_out || a.num_qo_heads < 1 || !rows_ok(a.q, a.q_stride_tok, a.q_stride_head, 2)) return MSA_ERR_BAD_ARG;
    if (a.q_out_dtype != MSA_DT_BF16 && a.q_out_dtype != MSA_DT_E4M3) return MSA_ERR_UNSUPPORTED;
    if (!rows_ok(a.q_out, a.q_out_stride_tok, a.q_out_stride_head, a.q_out_dtype == MSA_DT_E4M3 ? 1 : 2)) return MSA_ERR_BAD_ARG;
  }
  if ((a.k || a.v) && a.num_kv_heads < 1) return MSA_ERR_BAD_ARG;
  if (a.k) {
    if (!a.k_out && !a.k_cache) return MSA_ERR_BAD_ARG;
    if (!rows_ok(a.k, a.k_stride_tok, a.k_stride_head, 2)) return MSA_ERR_BAD_ARG;
    if (a.k_out && !rows_ok(a.k_out, a.k_out_stride_tok, a.k_out_stride_head, 2)) return MSA_ERR_BAD_ARG;
  }
  if (a.v && (!a.v_cache || !rows_ok(a.v, a.v_stride_tok, a.v_stride_head, 2))) return MSA_ERR_BAD_ARG;
  if (a.k_cache || a.v_cache) {
    if (!a.slot_map || a.page_size < 1 || a.num_pages < 0) return MSA_ERR_BAD_ARG;
    if (a.cache_dtype != MSA_DT_BF16 && a.cache_dtype != MSA_DT_E4M3 && a.cache_dtype != MSA_DT_KV4) return MSA_ERR_UNSUPPORTED;
    if (a.cache_dtype == MSA_DT_KV4 && a.page_size != kKvTile) return MSA_ERR_UNSUPPORTED;
    if (a.k_cache && (!a.k || !cache_ok(a.k_cache, a.cache_dtype, a.k_cache_stride_page, a.k_cache_stride_head, a.k_cache_stride_tok))) return MSA_ERR_BAD_ARG;
    if (a.v_cache && (!a.v || !cache_ok(a.v_cache, a.cache_dtype, a.v_cache_stride_page, a.v_cache_stride_head, a.v_cache_stride_tok))) return MSA_ERR_BAD_ARG;
  }
  if (!aligned16(a.q_weight) || !aligned16(a.k_weight) || a.q_weight_stride % 8 || a.k_weight_stride % 8) return MSA_ERR_BAD_ARG;
  if (a.weight_dtype != MSA_DT_F32 && a.weight_dtype != MSA_DT_BF16) return MSA_ERR_UNSUPPORTED;
  if (a.tokens == 0) return MSA_OK;
  NvtxRange range("msa_norm_rope");
  const int kv_units = (a.num_kv_heads + 3) / 4;
  const int units = (a.q ? (a.num_qo_heads + 3) / 4 : 0) + (a.k ? kv_units : 0) + (a.v ? kv_units : 0);
  // few tokens: the heads of one go to several warps, until the SMs have 16 each or a warp has one unit.  777 tokens of 16 + 2 x 2
  // heads in 3 parts 8.3 us, in one 11.7, in 6 11.2; 32 of 64 + 2 x 4 in 18 parts 5.8 us less than in
  // one.
  const int parts = std::max(1, std::min(units, 148 * 16 / a.tokens));
  const unsigned blocks = static_cast<unsigned>(a.tokens) * static_cast<unsigned>(parts);      // 148 x 16, or a.tokens, at most
  const bool q8 = a.q && a.q_out_dtype == MSA_DT_E4M3;
#define MSA_ROPE_CASE(PAIRS) \
  (a.norm ? (q8 ? norm_rope_kernel<PAIRS, true, true> : norm_rope_kernel<PAIRS, true, false>) \
          : (q8 ? norm_rope_kernel<PAIRS, false, true> : norm_rope_kernel<PAIRS, false, false>))
  return launch_chained(a.interleaved ? MSA_ROPE_CASE(true) : MSA_ROPE_CASE(false), dim3(blocks), 32, 0,
                        static_cast<cudaStream_t>(stream), a, parts) == cudaSuccess ? MSA_OK : MSA_ERR_LAUNCH;
#undef MSA_ROPE_CASE
}

extern "C" int msa_kv4_read(const MsaKv4ReadArgs* pa, msa_stream_t stream) {
  using namespace msa;
  if (!pa) return MSA_ERR_BAD_ARG;
  const MsaKv4ReadArgs& a = *pa;
  if (!a.cache || !a.out || !a.slot_map || a.rows < 0 || a.num_kv_heads < 1 || a.num_pages < 0) return MSA_ERR_BAD_ARG;
  if (!aligned16(a.cache) || !aligned16(a.out) || a.stride_page % 16 || a.stride_head % 16) return MSA_ERR_BAD_ARG;
  if (a.num_kv_heads > 65535) return MSA_ERR_TOO_LARGE;
  if (a.rows == 0) return MSA_OK;
  NvtxRange range("msa_kv4_read");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (a.whole_pages)
    return launch_chained(kv4_unpack_kernel, dim3(a.rows, a.num_kv_heads), 256, 0, st, a) == cudaSuccess ? MSA_OK : MSA_ERR_LAUNCH;
  const int64_t blocks = (static_cast<int64_t>(a.rows) * a.num_kv_heads + 15) / 16;
  if (blocks > 0x7fffffffLL) return MSA_ERR_TOO_LARGE;
  return launch_chained(kv4_read_kernel, dim3(static_cast<unsigned>(blocks)), 256, 0, st, a) == cudaSuccess ? MSA_OK : MSA_ERR_LAUNCH;
}
