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
// Keys are normed and rotated in 64 bits and rounded to bf16 once, then quantised from there: which e4m3 or e2m1 value a key
// next to a border gets does not depend on the order of a sum.  (They are a tenth of the rows or less; the pass is bound
// by memory.)  Queries are computed in 32 bits.
//
// 4-bit rows: 16 elements share an e4m3 scale s = round(max|x| / 6), at least 2^-9; the codes are the e2m1 roundings of x / s
// (divisions as IEEE has them: an x on a border goes to the even code).  A NaN makes the scale of its 16 elements NaN.
//
// A row of 128 bf16 is read by 16 lanes, 16 bytes each; a warp works on two heads at a time.
#include <algorithm>

#include <cuda_fp4.h>

#include "common.cuh"
#include "kv4.cuh"
#include "nvtx_range.h"

namespace msa {
namespace {

constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;

__device__ __forceinline__ void load8(const __nv_bfloat16* p, float (&x)[8]) {
  const uint4 r = *reinterpret_cast<const uint4*>(p);
  const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) { x[2 * i] = __uint_as_float(w[i] << 16); x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
}
__device__ __forceinline__ uint4 pack8(const float (&x)[8]) {
  return make_uint4(pack2<false>(x[0], x[1]), pack2<false>(x[2], x[3]), pack2<false>(x[4], x[5]), pack2<false>(x[6], x[7]));
}
__device__ __forceinline__ float to_bf16(float x) { return __bfloat162float(__float2bfloat16_rn(x)); }
__device__ __forceinline__ uint2 pack8_e4m3(const float (&x)[8], float scale) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    w[i] = __nv_cvt_float2_to_fp8x2(make_float2(__fdiv_rn(x[2 * i], scale), __fdiv_rn(x[2 * i + 1], scale)), __NV_SATFINITE, __NV_E4M3);
  return make_uint2(w[0] | (w[1] << 16), w[2] | (w[3] << 16));
}

// Elements 8 * l .. + 7 of the weight of a head, 1 without one.
__device__ __forceinline__ void load_weight(const void* w, int dtype, int64_t at, float (&x)[8]) {
  if (!w) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = 1.f;
  } else if (dtype == MSA_DT_F32) {
    const float4 a = *reinterpret_cast<const float4*>(static_cast<const float*>(w) + at);
    const float4 b = *reinterpret_cast<const float4*>(static_cast<const float*>(w) + at + 4);
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
  } else {
    load8(static_cast<const __nv_bfloat16*>(w) + at, x);
  }
}

__device__ __forceinline__ float rsqrt_of(float x) { return rsqrtf(x); }
__device__ __forceinline__ double rsqrt_of(double x) { return rsqrt(x); }

// Norm and rotation of one head held by 16 lanes (lane l: elements 8 l .. 8 l + 7); cs: cosine and sine of every pair.
template <typename F, typename F2>
__device__ __forceinline__ void norm_rotate(F (&x)[8], const float (&w)[8], bool norm, float eps, const F2* cs, int rotary, bool interleaved,
                                            int l) {
  if (norm) {
    F sum = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) sum += x[i] * x[i];
#pragma unroll
    for (int d = 8; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d, 16);
    const F r = rsqrt_of(sum * F(1.0 / kHeadDim) + F(eps));
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = x[i] * r * F(w[i]);
  }
  if (interleaved) {
    if (8 * l < rotary) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const F2 t = cs[4 * l + i];
        const F a = x[2 * i], b = x[2 * i + 1];
        x[2 * i] = a * t.x - b * t.y;
        x[2 * i + 1] = b * t.x + a * t.y;
      }
    }
    return;
  }
  const int off = rotary >> 4;                               // lanes from one half of the pairs to the other
  const bool first = l < off, second = !first && l < 2 * off;
  const int partner = first ? l + off : (second ? l - off : l);
  const int pair0 = 8 * (first ? l : (second ? l - off : 0));
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const F other = __shfl_sync(0xffffffffu, x[i], partner, 16);
    const F2 t = cs[pair0 + i];
    if (first) x[i] = x[i] * t.x - other * t.y;
    else if (second) x[i] = x[i] * t.x + other * t.y;
  }
}

// Writes 8 bf16-valued elements of a row of the cache.
__device__ __forceinline__ void store_row(void* cache, int dtype, int64_t stride_page, int64_t stride_head, int64_t stride_tok, int page_size,
                                          int slot, int head, int l, const float (&x)[8], float scale, bool write) {
  const int page = slot / page_size, r = slot - page * page_size;
  const int64_t at = page * stride_page + head * stride_head;
  if (dtype == MSA_DT_KV4) {
    float y[8];
    uint32_t top = 0;                                        // as integers: a NaN is above every number
#pragma unroll
    for (int i = 0; i < 8; ++i) { y[i] = __fdiv_rn(x[i], scale); top = max(top, __float_as_uint(y[i]) & 0x7fffffffu); }
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    float s = __fdiv_rn(__uint_as_float(top), 6.f);
    s = s < kKv4MinScale ? kKv4MinScale : s;
    const __nv_fp8_storage_t sb = __nv_cvt_float_to_fp8(s, __NV_SATFINITE, __NV_E4M3);
    const __half_raw sh = __nv_cvt_fp8_to_halfraw(sb, __NV_E4M3);
    const float sf = __half2float(*reinterpret_cast<const __half*>(&sh));
    uint32_t codes = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      codes |= static_cast<uint32_t>(__nv_cvt_float2_to_fp4x2(make_float2(__fdiv_rn(y[2 * i], sf), __fdiv_rn(y[2 * i + 1], sf)), __NV_E2M1,
                                                              cudaRoundNearest)) << (8 * i);
    if (write) {
      unsigned char* tile = static_cast<unsigned char*>(cache) + at;
      *reinterpret_cast<uint32_t*>(tile + r * kKv4CodeBytes + 4 * l) = codes;
      if (!(l & 1)) tile[kKv4ScaleOffset + r * kKv4ScaleBytes + (l >> 1)] = sb;
    }
  } else if (write && dtype == MSA_DT_E4M3) {
    *reinterpret_cast<uint2*>(static_cast<unsigned char*>(cache) + at + r * stride_tok + 8 * l) = pack8_e4m3(x, scale);
  } else if (write) {
    *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(cache) + at + r * stride_tok + 8 * l) = pack8(x);
  }
}

__global__ void __launch_bounds__(kThreads) norm_rope_kernel(const MsaNormRopeArgs a) {
  chain_begin();
  __shared__ double2 s_cs[kHeadDim / 2];
  __shared__ float2 s_csf[kHeadDim / 2];
  const int t = blockIdx.x;
  const int lane = threadIdx.x & 31, l = lane & 15, half = lane >> 4;
  if (a.rotary > 0) {
    const int n = threadIdx.x;
    if (n < a.rotary / 2) {
      const int64_t at = a.axis[n] * a.pos_stride_axis + t;
      const int64_t pos = a.pos_int64 ? static_cast<const int64_t*>(a.positions)[at] : static_cast<const int32_t*>(a.positions)[at];
      const int64_t turns = static_cast<int64_t>(static_cast<uint64_t>(pos) * static_cast<uint64_t>(a.turns[n]));   // modulo a turn
      double2 cs;
      sincospi(static_cast<double>(turns) * 0x1p-63, &cs.y, &cs.x);
      s_cs[n] = cs;
      s_csf[n] = make_float2(static_cast<float>(cs.x), static_cast<float>(cs.y));
    }
    __syncthreads();
  }
  const int slot = a.slot_map ? a.slot_map[t] : -1;
  const bool has_slot = slot >= 0 && slot / a.page_size < a.num_pages;
#ifdef MSA_BOUNDS_CHECK
  if (slot >= 0 && !has_slot) chk(slot, 0, 0, a.status);
#endif
  const int slot_in = has_slot ? slot : 0;
  const int q_units = a.q ? (a.num_qo_heads + 1) / 2 : 0, kv_units = (a.num_kv_heads + 1) / 2;
  const int k_end = q_units + (a.k ? kv_units : 0), v_end = k_end + (a.v ? kv_units : 0);
  for (int u = blockIdx.y * kWarps + (threadIdx.x >> 5); u < v_end; u += gridDim.y * kWarps) {
    float x[8], w[8];
    if (u < q_units) {
      const int head = 2 * u + half;
      const bool real = head < a.num_qo_heads;
      const int h = real ? head : head - 1;
      load8(static_cast<const __nv_bfloat16*>(a.q) + t * a.q_stride_tok + h * a.q_stride_head + 8 * l, x);
      load_weight(a.q_weight, a.weight_dtype, h * a.q_weight_stride + 8 * l, w);
      norm_rotate(x, w, a.norm, a.eps, s_csf, a.rotary, a.interleaved, l);
      if (real) {
        const int64_t at = t * a.q_out_stride_tok + h * a.q_out_stride_head + 8 * l;
        if (a.q_out_dtype == MSA_DT_E4M3) {
#pragma unroll
          for (int i = 0; i < 8; ++i) x[i] = to_bf16(x[i]);
          *reinterpret_cast<uint2*>(static_cast<unsigned char*>(a.q_out) + at) = pack8_e4m3(x, a.q_scale);
        } else {
          *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(a.q_out) + at) = pack8(x);
        }
      }
    } else if (u < k_end) {
      const int head = 2 * (u - q_units) + half;
      const bool real = head < a.num_kv_heads;
      const int h = real ? head : head - 1;
      load8(static_cast<const __nv_bfloat16*>(a.k) + t * a.k_stride_tok + h * a.k_stride_head + 8 * l, x);
      if (a.norm || a.rotary > 0) {
        load_weight(a.k_weight, a.weight_dtype, h * a.k_weight_stride + 8 * l, w);
        double z[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) z[i] = x[i];
        norm_rotate(z, w, a.norm, a.eps, s_cs, a.rotary, a.interleaved, l);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = to_bf16(static_cast<float>(z[i]));
      }
      if (a.k_out && real)
        *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(a.k_out) + t * a.k_out_stride_tok + h * a.k_out_stride_head + 8 * l) = pack8(x);
      if (a.k_cache)
        store_row(a.k_cache, a.cache_dtype, a.k_cache_stride_page, a.k_cache_stride_head, a.k_cache_stride_tok, a.page_size, slot_in, h, l, x,
                  a.k_scale * (a.k_scale_head ? a.k_scale_head[h] : 1.f), has_slot && real);
    } else {
      const int head = 2 * (u - k_end) + half;
      const bool real = head < a.num_kv_heads;
      const int h = real ? head : head - 1;
      load8(static_cast<const __nv_bfloat16*>(a.v) + t * a.v_stride_tok + h * a.v_stride_head + 8 * l, x);
      store_row(a.v_cache, a.cache_dtype, a.v_cache_stride_page, a.v_cache_stride_head, a.v_cache_stride_tok, a.page_size, slot_in, h, l, x,
                a.v_scale * (a.v_scale_head ? a.v_scale_head[h] : 1.f), has_slot && real);
    }
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

// Whole pages, in the order of a page table: out[e, head, 128, 128] = page kv_indices[e].  A warp takes a row of 4 tokens ... of
// one (page, head): 8 lanes per row would leave scales to be loaded twice; 16 lanes a row as above, 16 rows a block step.
__global__ void __launch_bounds__(256) kv4_unpack_kernel(const MsaKv4ReadArgs a) {
  chain_begin();
  const int l = threadIdx.x & 15;
  const int e = blockIdx.x, h = blockIdx.y;
  const int page = a.slot_map[e];
  if (page < 0 || page >= a.num_pages) return;               // behind the last page of a table that is longer than its use
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
  if (a.rotary < 0 || a.rotary > kHeadDim || a.rotary % 16) return MSA_ERR_UNSUPPORTED;
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
  const int kv_units = (a.num_kv_heads + 1) / 2;
  const int units = (a.q ? (a.num_qo_heads + 1) / 2 : 0) + (a.k ? kv_units : 0) + (a.v ? kv_units : 0);
  // few tokens: the heads of one go to several CTAs, so that a warp has one unit
  const int most = (units + kWarps - 1) / kWarps;
  const int y = std::max(1, std::min(most, 2 * 148 / std::max(1, a.tokens)));
  return launch_chained(norm_rope_kernel, dim3(a.tokens, y), kThreads, 0, static_cast<cudaStream_t>(stream), a) == cudaSuccess ? MSA_OK
                                                                                                                           : MSA_ERR_LAUNCH;
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
