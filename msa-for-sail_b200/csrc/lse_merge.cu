// Split-KV merge for sm_100a: combines normalised partial outputs with their LSEs.
//
//   out[t,h,:] = sum_s w_s * partial_o[s,t,h,:] / sum_s w_s,   w_s = exp(lse_s - max_s lse_s)
//
// A split whose LSE is -inf contributes nothing and its partial is never multiplied in (it may
// hold NaN or stale bytes).  Same contract as the upstream reduction
// (csrc/include/sm80_fmha_reduction.hpp:133-215); partials here are fp32 or bf16 and the LSE
// is a natural logarithm.  Half a warp handles one (token, head).
#include "common.cuh"
#include "nvtx_range.h"

namespace msa {
namespace {

// Half a warp per (token, head) row: lane l of the half owns columns 8l..8l+7.  Loads of up to
// eight splits are issued back to back before they are consumed.
template <bool PBF16, bool OF32>
__global__ void __launch_bounds__(256)
lse_merge_kernel(const void* po_, const float* pl, const int32_t* spr,
                 void* out_, float* lse_out, int num_splits, int total_q,
                 int num_heads, int64_t o_split_stride, int64_t l_split_stride, int64_t out_stride_tok,
                 int64_t out_stride_head, float out_scale) {
  chain_begin();
  const int l16 = threadIdx.x & 15;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (blockDim.x >> 4) + (threadIdx.x >> 4);   // t * H + h
  const int64_t rows = static_cast<int64_t>(total_q) * num_heads;
  if (row >= rows) return;
  const int t = static_cast<int>(row / num_heads), h = static_cast<int>(row % num_heads);
  const int S = spr ? min(spr[t], num_splits) : num_splits;

  float mx = -INFINITY;
  for (int s = 0; s < S; ++s) mx = fmaxf(mx, pl[static_cast<int64_t>(s) * l_split_stride + row]);
  const float mxs = (mx == -INFINITY) ? 0.f : mx;

  float acc[8];
#pragma unroll
  for (int c = 0; c < 8; ++c) acc[c] = 0.f;
  float sw = 0.f;
  constexpr int U = 8;
  for (int s0 = 0; s0 < S; s0 += U) {
    float w[U];
    uint4 raw[U][PBF16 ? 1 : 2];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int s = min(s0 + u, S - 1);                         // clamped: always a readable slot
      const int64_t base = static_cast<int64_t>(s) * o_split_stride + row * kHeadDim + l16 * 8;
      if constexpr (PBF16) {
        raw[u][0] = *reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(po_) + base);
      } else {
        raw[u][0] = *reinterpret_cast<const uint4*>(static_cast<const float*>(po_) + base);
        raw[u][1] = *reinterpret_cast<const uint4*>(static_cast<const float*>(po_) + base + 4);
      }
      const float l = pl[static_cast<int64_t>(s) * l_split_stride + row];
      w[u] = (s0 + u < S && l != -INFINITY) ? __expf(l - mxs) : 0.f;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (w[u] != 0.f) {                                        // value select after an unconditional load
        sw += w[u];
        if constexpr (PBF16) {
          const uint32_t* r4 = reinterpret_cast<const uint32_t*>(&raw[u][0]);
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            acc[2 * c] = fmaf(w[u], bf16_bits_to_float(r4[c] & 0xffff), acc[2 * c]);
            acc[2 * c + 1] = fmaf(w[u], bf16_bits_to_float(r4[c] >> 16), acc[2 * c + 1]);
          }
        } else {
          const float* f = reinterpret_cast<const float*>(&raw[u][0]);
#pragma unroll
          for (int c = 0; c < 8; ++c) acc[c] = fmaf(w[u], f[c], acc[c]);
        }
      }
    }
  }
  const float inv = sw > 0.f ? out_scale / sw : 0.f;
  if (out_ && OF32) {
    float* dst = static_cast<float*>(out_) + static_cast<int64_t>(t) * out_stride_tok + static_cast<int64_t>(h) * out_stride_head + l16 * 8;
    *reinterpret_cast<float4*>(dst) = make_float4(acc[0] * inv, acc[1] * inv, acc[2] * inv, acc[3] * inv);
    *reinterpret_cast<float4*>(dst + 4) = make_float4(acc[4] * inv, acc[5] * inv, acc[6] * inv, acc[7] * inv);
  } else if (out_) {
    __nv_bfloat16* dst = static_cast<__nv_bfloat16*>(out_) + static_cast<int64_t>(t) * out_stride_tok + static_cast<int64_t>(h) * out_stride_head + l16 * 8;
    uint4 pk;
    pk.x = pack2<false>(acc[0] * inv, acc[1] * inv);
    pk.y = pack2<false>(acc[2] * inv, acc[3] * inv);
    pk.z = pack2<false>(acc[4] * inv, acc[5] * inv);
    pk.w = pack2<false>(acc[6] * inv, acc[7] * inv);
    *reinterpret_cast<uint4*>(dst) = pk;
  }
  if (lse_out && l16 == 0) lse_out[row] = sw > 0.f ? mxs + __logf(sw) : -INFINITY;
}

// A CTA per row, for many splits of few rows: half a warp would take eight splits after eight.  Warp w has splits w, w + 4, ...,
// eight of them on their way at a time, a lane four columns; the four sums are added in their order.  Bound by the latency of
// three dependent reads (weights, partials, sums of the warps).
constexpr int kManyWarps = 4, kManyChunk = 128;               // splits whose weights are in shared memory at a time
template <bool OF32>
__global__ void __launch_bounds__(32 * kManyWarps)
lse_merge_many_kernel(const float* po, const float* pl, const int32_t* spr, void* out_, float* lse_out, int num_splits, int64_t rows,
                      int num_heads, int64_t out_stride_tok, int64_t out_stride_head, float out_scale) {
  chain_begin();
  __shared__ float s_w[kManyChunk];
  __shared__ float s_red[2][kManyWarps];
  __shared__ float4 s_acc[kManyWarps][32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t row = blockIdx.x;
  const int t = static_cast<int>(row / num_heads), h = static_cast<int>(row % num_heads);
  const int S = spr ? min(spr[t], num_splits) : num_splits;
  float first = -INFINITY, mx = -INFINITY;
  for (int s = threadIdx.x; s < S; s += 32 * kManyWarps) {
    const float l = pl[s * rows + row];
    if (s < kManyChunk) first = l;
    mx = fmaxf(mx, l);
  }
#pragma unroll
  for (int d = 16; d; d >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
  if (lane == 0) s_red[0][warp] = mx;
  __syncthreads();
  mx = fmaxf(fmaxf(s_red[0][0], s_red[0][1]), fmaxf(s_red[0][2], s_red[0][3]));
  const float mxs = mx == -INFINITY ? 0.f : mx;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  float sw = 0.f;
  for (int c0 = 0; c0 < S; c0 += kManyChunk) {
    const int n = min(kManyChunk, S - c0);
    if (c0 > 0) __syncthreads();                               // the weights before these are no longer read
    if (threadIdx.x < n) {
      const float l = c0 == 0 ? first : pl[(c0 + threadIdx.x) * rows + row];
      const float w = l != -INFINITY ? __expf(l - mxs) : 0.f;
      s_w[threadIdx.x] = w;
      sw += w;
    }
    __syncthreads();
    const float* src = po + (c0 * rows + row) * kHeadDim + 4 * lane;
    constexpr int U = 8;
    for (int s0 = warp; s0 < n; s0 += kManyWarps * U) {
      float4 x[U];
#pragma unroll
      for (int u = 0; u < U; ++u) x[u] = *reinterpret_cast<const float4*>(src + min(s0 + kManyWarps * u, n - 1) * rows * kHeadDim);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const float w = s0 + kManyWarps * u < n ? s_w[s0 + kManyWarps * u] : 0.f;
        if (w != 0.f) {                                        // the partial of an empty split is not looked at
          acc.x = fmaf(w, x[u].x, acc.x); acc.y = fmaf(w, x[u].y, acc.y);
          acc.z = fmaf(w, x[u].z, acc.z); acc.w = fmaf(w, x[u].w, acc.w);
        }
      }
    }
  }
#pragma unroll
  for (int d = 16; d; d >>= 1) sw += __shfl_xor_sync(0xffffffffu, sw, d);
  if (lane == 0) s_red[1][warp] = sw;
  s_acc[warp][lane] = acc;
  __syncthreads();
  if (warp != 0) return;
  sw = (s_red[1][0] + s_red[1][1]) + (s_red[1][2] + s_red[1][3]);
  const float inv = sw > 0.f || isnan(sw) ? out_scale / sw : 0.f;
#pragma unroll
  for (int w = 1; w < kManyWarps; ++w) {
    const float4 o = s_acc[w][lane];
    acc.x += o.x; acc.y += o.y; acc.z += o.z; acc.w += o.w;
  }
  const int64_t at = t * out_stride_tok + h * out_stride_head + 4 * lane;
  if (OF32) *reinterpret_cast<float4*>(static_cast<float*>(out_) + at) = make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
  else *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(out_) + at) = make_uint2(pack2<false>(acc.x * inv, acc.y * inv), pack2<false>(acc.z * inv, acc.w * inv));
  if (lse_out && lane == 0) lse_out[row] = sw > 0.f || isnan(sw) ? mxs + __logf(sw) : -INFINITY;
}

// A warp per row, for many rows or few splits: lane l has the weight of split l of every 32, and four columns.  The first partials
// are on their way while the weights are, and none is read twice: 8 192 rows x 4 splits 4.0 us, 6.0 with half a warp per row above.
template <bool OF32>
__global__ void __launch_bounds__(128)
lse_merge_rows_kernel(const float* po, const float* pl, const int32_t* spr, void* out_, float* lse_out, int num_splits, int64_t rows,
                      int num_heads, int64_t out_stride_tok, int64_t out_stride_head, float out_scale) {
  chain_begin();
  const int lane = threadIdx.x & 31;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 5);
  if (row >= rows) return;
  const int t = static_cast<int>(row / num_heads), h = static_cast<int>(row % num_heads);
  const int S = spr ? min(spr[t], num_splits) : num_splits;
  constexpr int U = 4;
  const float* src = po + row * kHeadDim + 4 * lane;
  float4 x[U];
  auto load = [&](int s0) {
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (s0 + u < S) x[u] = *reinterpret_cast<const float4*>(src + (s0 + u) * rows * kHeadDim);
  };
  load(0);
  const float first = lane < S ? pl[lane * rows + row] : -INFINITY;
  float mx = first;
  for (int s = 32 + lane; s < S; s += 32) mx = fmaxf(mx, pl[s * rows + row]);
#pragma unroll
  for (int d = 16; d; d >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
  const float mxs = mx == -INFINITY ? 0.f : mx;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  float sw = 0.f, w_lane = 0.f;
  for (int s0 = 0; s0 < S; s0 += U) {
    if ((s0 & 31) == 0) {
      const float l = s0 == 0 ? first : (s0 + lane < S ? pl[(s0 + lane) * rows + row] : -INFINITY);
      w_lane = l != -INFINITY ? __expf(l - mxs) : 0.f;
      sw += w_lane;
    }
    if (s0 > 0) load(s0);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const float w = __shfl_sync(0xffffffffu, w_lane, (s0 + u) & 31);
      if (s0 + u < S && w != 0.f) {                            // the partial of an empty split is not looked at
        acc.x = fmaf(w, x[u].x, acc.x); acc.y = fmaf(w, x[u].y, acc.y);
        acc.z = fmaf(w, x[u].z, acc.z); acc.w = fmaf(w, x[u].w, acc.w);
      }
    }
  }
#pragma unroll
  for (int d = 16; d; d >>= 1) sw += __shfl_xor_sync(0xffffffffu, sw, d);
  const float inv = sw > 0.f || isnan(sw) ? out_scale / sw : 0.f;
  const int64_t at = t * out_stride_tok + h * out_stride_head + 4 * lane;
  if (OF32) *reinterpret_cast<float4*>(static_cast<float*>(out_) + at) = make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
  else *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(out_) + at) = make_uint2(pack2<false>(acc.x * inv, acc.y * inv), pack2<false>(acc.z * inv, acc.w * inv));
  if (lse_out && lane == 0) lse_out[row] = sw > 0.f || isnan(sw) ? mxs + __logf(sw) : -INFINITY;
}

}  // namespace
}  // namespace msa

extern "C" int msa_lse_merge_many(const float* partial_o, const float* partial_lse, const int32_t* splits_per_row, void* out,
                                  int32_t out_dtype, float* lse_out, int32_t num_splits, int32_t total_q, int32_t num_heads,
                                  int64_t out_stride_tok, int64_t out_stride_head, float out_scale, msa_stream_t stream) {
  if (!partial_o || !partial_lse || !out || num_splits < 1 || total_q < 0 || num_heads <= 0) return MSA_ERR_BAD_ARG;
  if (out_dtype != MSA_DT_F32 && out_dtype != MSA_DT_BF16) return MSA_ERR_UNSUPPORTED;
  const int64_t rows = static_cast<int64_t>(total_q) * num_heads;
  if (rows == 0) return MSA_OK;
  if (rows > 0x7fffffffLL) return MSA_ERR_TOO_LARGE;
  // rows of partials are read 16 bytes at a time, those of the result written 16 or 8
  const int oe = out_dtype == MSA_DT_BF16 ? 2 : 4;
  if ((reinterpret_cast<uintptr_t>(partial_o) & 15) || reinterpret_cast<uintptr_t>(out) % (4 * oe) || out_stride_tok % 4 || out_stride_head % 4)
    return MSA_ERR_BAD_ARG;
  msa::NvtxRange range("msa_lse_merge_many");
  // 64 rows x 72 splits: 3.8 us with a CTA each, 7.4 with a warp; 512 x 16 3.0 and 3.0, 1 536 x 37 7.0 and 5.6, 8 192 x 4 14.8 and 4.0
  const bool wide = num_splits > 16 && rows <= 1024;
  const auto kernel = wide ? (out_dtype == MSA_DT_F32 ? msa::lse_merge_many_kernel<true> : msa::lse_merge_many_kernel<false>)
                           : (out_dtype == MSA_DT_F32 ? msa::lse_merge_rows_kernel<true> : msa::lse_merge_rows_kernel<false>);
  return msa::launch_chained(kernel, dim3(static_cast<unsigned>(wide ? rows : (rows + 3) / 4)), 128, 0, static_cast<cudaStream_t>(stream), partial_o,
                             partial_lse, splits_per_row, out, lse_out, num_splits, rows, num_heads, out_stride_tok, out_stride_head,
                             out_scale) == cudaSuccess ? MSA_OK : MSA_ERR_LAUNCH;
}

extern "C" int msa_lse_merge_ex(const void* partial_o, int32_t partial_dtype, const float* partial_lse,
                                const int32_t* splits_per_row, void* out, int32_t out_dtype, float* lse_out,
                                int32_t num_splits, int32_t total_q, int32_t num_heads, int64_t o_split_stride,
                                int64_t lse_split_stride, int64_t out_stride_tok, int64_t out_stride_head,
                                float out_scale, msa_stream_t stream) {
  if (!partial_o || !partial_lse || (!out && !lse_out) || num_splits < 1 || total_q < 0 || num_heads <= 0)
    return MSA_ERR_BAD_ARG;
  msa::NvtxRange range("msa_lse_merge");
  const int64_t rows = static_cast<int64_t>(total_q) * num_heads;
  if (rows == 0) return MSA_OK;
  const int64_t blocks = (rows + 15) / 16;
  if (blocks > 0x7fffffffLL) return MSA_ERR_TOO_LARGE;
  if (partial_dtype != MSA_DT_F32 && partial_dtype != MSA_DT_BF16) return MSA_ERR_UNSUPPORTED;
  if (out_dtype != MSA_DT_F32 && out_dtype != MSA_DT_BF16) return MSA_ERR_UNSUPPORTED;
  if (o_split_stride <= 0) o_split_stride = rows * msa::kHeadDim;
  if (lse_split_stride <= 0) lse_split_stride = rows;
  // rows are read and written 16 bytes at a time
  const int pe = partial_dtype == MSA_DT_BF16 ? 2 : 4, oe = out_dtype == MSA_DT_BF16 ? 2 : 4;
  auto al = [](const void* ptr) { return (reinterpret_cast<uintptr_t>(ptr) & 15) == 0; };
  if (!al(partial_o) || (o_split_stride * pe) % 16 || (out && (!al(out) || (out_stride_tok * oe) % 16 ||
                                                                (out_stride_head * oe) % 16)))
    return MSA_ERR_BAD_ARG;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const unsigned nb = static_cast<unsigned>(blocks);
#define MSA_MERGE_CASE(PB, OF)                                                                                       \
  msa::launch_chained(msa::lse_merge_kernel<PB, OF>, nb, 256, 0, st, partial_o, partial_lse, splits_per_row, out, lse_out, num_splits, \
                                                    total_q, num_heads, o_split_stride, lse_split_stride,           \
                                                    out_stride_tok, out_stride_head, out_scale)
  if (partial_dtype == MSA_DT_BF16) { if (out_dtype == MSA_DT_F32) MSA_MERGE_CASE(true, true); else MSA_MERGE_CASE(true, false); }
  else { if (out_dtype == MSA_DT_F32) MSA_MERGE_CASE(false, true); else MSA_MERGE_CASE(false, false); }
#undef MSA_MERGE_CASE
  return cudaGetLastError() == cudaSuccess ? MSA_OK : MSA_ERR_LAUNCH;
}

extern "C" int msa_lse_merge(const void* partial_o, int32_t partial_dtype, const float* partial_lse,
                             const int32_t* splits_per_row, void* out, float* lse_out, int32_t num_splits,
                             int32_t total_q, int32_t num_heads, int64_t out_stride_tok, int64_t out_stride_head,
                             float out_scale, msa_stream_t stream) {
  return msa_lse_merge_ex(partial_o, partial_dtype, partial_lse, splits_per_row, out, MSA_DT_BF16, lse_out, num_splits,
                          total_q, num_heads, 0, 0, out_stride_tok, out_stride_head, out_scale, stream);
}
