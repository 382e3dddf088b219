// The 4-bit cache: layout and conversions.
//
// The tile of one (page, KV head) is 9 216 contiguous bytes: 128 rows of 64 bytes, two e2m1 codes a byte (element 2 i in the low
// half of byte i), then 128 rows of eight e4m3 scales, one for each 16 elements.  An element is code * scale; a scale per KV
// head (the k_scale / v_scale of the attention call) comes on top.  Codes before scales, so that both are read in 16-byte pieces;
// 16 elements a scale, 72 bytes a row: 0.56 of an e4m3 row.
#pragma once

#include "common.cuh"

namespace msa {

constexpr int kKv4CodeBytes = kHeadDim / 2;                   // of a row
constexpr int kKv4ScaleBytes = kHeadDim / 16;
constexpr int kKv4ScaleOffset = kKvTile * kKv4CodeBytes;
constexpr float kKv4MinScale = 0x1p-9f;                       // the smallest e4m3 number: no block of small values is lost to a scale of zero

// Four bytes of codes (8 elements) -> four f16 pairs, the low half of a byte in the low half of a pair.
__device__ __forceinline__ void kv4_to_half(uint32_t codes, uint32_t (&out)[4]) {
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "mov.b32 {b0, b1, b2, b3}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, b2;\n\t"
      "cvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
      : "=r"(out[0]), "=r"(out[1]), "=r"(out[2]), "=r"(out[3]) : "r"(codes));
}

// Two e4m3 scales -> an f16 pair (exact).
__device__ __forceinline__ uint32_t kv4_scales_to_half(uint16_t x) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(x), __NV_E4M3);
  return static_cast<uint32_t>(h.x) | (static_cast<uint32_t>(h.y) << 16);
}

__device__ __forceinline__ uint32_t half2_mul(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}

// 8 elements as bf16.  The product of a code (2 significant bits) and a scale (4) is exact in f16, 2688 at most and a multiple of
// 2^-10, and in bf16.
__device__ __forceinline__ uint4 kv4_to_bf16(uint32_t codes, uint32_t scale) {
  uint32_t h[4];
  kv4_to_half(codes, h);
  const uint32_t s = kv4_scales_to_half(static_cast<uint16_t>(scale | (scale << 8)));
  uint32_t b[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t p = half2_mul(h[i], s);
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&p));
    b[i] = pack2<false>(f.x, f.y);
  }
  return make_uint4(b[0], b[1], b[2], b[3]);
}

}  // namespace msa
