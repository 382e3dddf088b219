// Shared device helpers for the sm_100a MSA kernels.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "msa_b200.h"

namespace msa {

constexpr int kHeadDim = 128;   // upstream fixes D = 128 (jit.py:117-121)
constexpr int kKvTile = 128;    // keys per KV tile == max_score granularity
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// Range check of an index that a kernel read from a caller's table and is about to turn into an address
// (upstream: FMHA_GMEM_CHECK=1, csrc/gmem_bounds_check.h:27-69, which prints and returns 0).  In the
// bounds-checked build (-DMSA_BOUNDS_CHECK, libmsa_b200_check.so) a value outside [lo, hi) is clamped
// into the range and the first violation is recorded in the caller's status word -- no printf, no trap,
// the launch completes; in the shipped build the function is the identity.
#ifdef MSA_BOUNDS_CHECK
__device__ __forceinline__ int chk(int v, int lo, int hi, int32_t* status) {
  if (v >= lo && v < hi) return v;
  if (status) atomicCAS(status, MSA_STATUS_OK, MSA_STATUS_BOUNDS);
  return hi > lo ? min(max(v, lo), hi - 1) : lo;
}
#else
__device__ __forceinline__ int chk(int v, int, int, int32_t*) { return v; }
#endif

// Entry `at` of the flat page table.  Lengths that live on the device may outgrow the table: the places behind its end are its last
// entry, and nothing behind it is read.  (num_page_entries = 0: the caller did not say how long it is.)
__device__ __forceinline__ int page_entry(const MsaFmhaParams& p, int at) {
#ifdef MSA_BOUNDS_CHECK
  if (p.num_page_entries > 0) at = chk(at, 0, p.num_page_entries, p.status);
#endif
  const unsigned place = min(static_cast<unsigned>(at), static_cast<unsigned>(p.num_page_entries) - 1u);
  return chk(p.kv_indices[place], 0, static_cast<int>(p.kv_extent), p.status);
}

// ---- windows ----
// With a window W and S sink tokens a row at place t of its sequence sees key j <= t iff j > t - W or j < S.  The tiles that any of a row
// tile's rows sees are those of the sinks and those from the first key of its first row's window on: the ones between are left out
// of its work item, so that one range of numbers [0, count) stands for both.  Sums are taken in 64 bits: places may lie far behind the keys.
struct WindowSpan {
  int count;                    // tiles of the row tile
  int skip;                     // tiles left out behind those of the sinks
};
__host__ __device__ inline int sink_tiles(int sink_tokens) { return sink_tokens / kKvTile + (sink_tokens % kKvTile != 0); }
__host__ __device__ inline WindowSpan window_span(long long first_place, long long last_place, int kv_len, int window, int sink_tokens) {
  long long end = last_place + 1 < kv_len ? last_place + 1 : kv_len;
  if (end < 0) end = 0;
  const int tiles = static_cast<int>((end + kKvTile - 1) / kKvTile);
  if (window <= 0) return {tiles, 0};
  long long lo = (first_place - window + 1) / kKvTile;
  if (lo > tiles) lo = tiles;
  const int skip = lo > sink_tiles(sink_tokens) ? static_cast<int>(lo) - sink_tiles(sink_tokens) : 0;
  return {tiles - skip, skip};
}
// First key of the window of a row at place t, at most `kv_len`.
__device__ __forceinline__ int window_first(int place, int kv_len, int window) {
  const long long lo = static_cast<long long>(place) - window + 1;
  return lo < 0 ? 0 : lo < kv_len ? static_cast<int>(lo) : kv_len;
}
// SMs that the CTAs of a call may be spread over.
inline int sms_of(const MsaFmhaParams& p) { return p.num_sms > 0 && p.num_sms < 148 ? p.num_sms : 148; }
// Factor of the scores where masked ones are -inf, a positive number: -inf * 0 is no number, the smallest one changes no score by as much as its last
// bit.  The sign of a negative one (a head's own scale) goes to Q, or to the scores before they are masked and the largest is sought.
__device__ __forceinline__ float masked_scale(float scale) { return scale == 0.f ? 1.17549435e-38f : fabsf(scale); }
template <int N>
__device__ __forceinline__ void turn_scores(uint32_t (&s)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) s[i] ^= 0x80000000u;
}

// ---- kernels of one stream without a gap between them ----
// A kernel launched with launch_chained() may start while the kernel before it in the stream still runs: once every CTA of
// that one has called chain_begin() or ended.  chain_begin() comes before anything that touches global memory: it waits
// until the kernel before has completed and its writes are visible (at once if there is nothing to wait for), then
// lets the next kernel of the stream come up in the same way.  So the order of all memory accesses is that of the
// stream, and only the launch and the start of the CTAs overlap.
// What such a kernel reads may still be written while it starts, so it reads global memory with ordinary loads only: no
// __ldg, ld.global.nc or __restrict__, which promise data that does not change during the kernel, and would allow a load
// above the wait or a line of L1 from before it.
__device__ __forceinline__ void chain_begin() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}
template <typename... P, typename... A>
inline cudaError_t launch_chained_clusters(void (*kernel)(P...), unsigned cluster, dim3 grid, dim3 block, size_t smem, cudaStream_t stream, A&&... args) {
  // Under capture the launches stay plain: with programmatic edges the replay of a six-kernel decode graph took 86.5 us
  // against 77 us.
  cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
  cudaStreamIsCapturing(stream, &capture);
  cudaLaunchAttribute attr[2] = {};
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = capture == cudaStreamCaptureStatusNone ? 1 : 0;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid; cfg.blockDim = block; cfg.dynamicSmemBytes = smem; cfg.stream = stream;
  cfg.attrs = attr; cfg.numAttrs = cluster > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, P(args)...);
}
template <typename... P, typename... A>
inline cudaError_t launch_chained(void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream, A&&... args) {
  return launch_chained_clusters(kernel, 1, grid, block, smem, stream, args...);
}

__device__ __forceinline__ uint32_t smem_u32(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}

// 16-byte async copy global -> shared; `valid == false` writes zeros and reads nothing.
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool valid) {
  const int sz = valid ? 16 : 0;
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(dst), "l"(src), "r"(sz)
               : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;\n" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;\n" ::"n"(N) : "memory");
}

__device__ __forceinline__ void ldmatrix_x4(uint32_t addr, uint32_t& r0, uint32_t& r1, uint32_t& r2,
                                            uint32_t& r3) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];\n"
               : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3)
               : "r"(addr));
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t addr, uint32_t& r0, uint32_t& r1,
                                                  uint32_t& r2, uint32_t& r3) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];\n"
               : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3)
               : "r"(addr));
}

// D(16x8,f32) += A(16x16) * B(16x8); bf16 or fp16 operands.
template <bool kHalf>
__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                          uint32_t b1) {
  if constexpr (kHalf) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%0,%1,%2,%3};\n"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  } else {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%0,%1,%2,%3};\n"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
}

template <bool kHalf>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (kHalf) {
    __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&h);
  } else {
    __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&h);
  }
}

// three-input maximum (one instruction on sm_100)
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;\n" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// ---- packed fp32 pairs (one instruction, two lanes; sm_100) ----
__device__ __forceinline__ uint64_t f2_pack(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};\n" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void f2_unpack(uint64_t v, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;\n" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ uint64_t f2_fma(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;\n" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t f2_add(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;\n" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

// Two values as pairs of e4m3 values, hi and lo (low 16 bits each).  hi is the value rounded to 4 significant bits: with t = (2^20 + 1) x,
// t - (t - x) (Veltkamp's splitting); what it leaves is exact.  No conversion back from e4m3 is needed.  A pair is within 2^-8 x + 1.5 * 2^-10 of x: below
// e4m3's normal numbers, 2^-6, hi rounds by up to 2^-10, what is left of it by 2^-11, and a weight below 2^-10 is gone.
//
// So what weights are relative to must not lie far above most of a row's mass: one heavy key (a sink) with weight 2^4 would leave nothing of thousands
// of keys ten nats below it, 16 % of the mass with 4 096 of them.  It follows a tile's largest score down as well as up (pair_lowers).  Of a tile of n keys
// 1.5 * 2^-10 n is lost at most.  That is left so where the tile's weights have a sum of n / 4, or the row's have one of a quarter of its keys so far; else
// it goes down to the tile's largest score.  Either way all that is lost of a row is 1.5 * 2^-8 of its sum at most.  A row of scores that lie within a few
// nats has such a sum throughout.
__device__ __forceinline__ void e4m3_pair(float a, float b, uint32_t& hi, uint32_t& lo) {
  const uint64_t x = f2_pack(a, b), t = f2_fma(x, f2_pack(1048577.f, 1048577.f), 0), minus = f2_pack(-1.f, -1.f);
  const uint64_t h = f2_fma(f2_fma(x, minus, t), minus, t), rest = f2_fma(h, minus, x);
  float h0, h1, l0, l1;
  f2_unpack(h, h0, h1);
  f2_unpack(rest, l0, l1);
  hi = __nv_cvt_float2_to_fp8x2(make_float2(h0, h1), __NV_SATFINITE, __NV_E4M3);
  lo = __nv_cvt_float2_to_fp8x2(make_float2(l0, l1), __NV_SATFINITE, __NV_E4M3);
}

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}

// What a row's weights are relative to, for pairs of e4m3 values (e4m3_pair): a score equal to it has weight 2^kPairOffset, one kPairRescale (log2)
// above it raises it, to kPairRise below that score.
constexpr float kPairOffset = 5.f, kPairRescale = 3.8f, kPairRise = 2.8f;
constexpr float kPairEnough = 0.25f;                         // sum of weights, for each key, of which the loss is small enough
// It goes down to a tile's largest score where neither `tile`, (a lower bound of) the sum of the tile's n weights, is enough for the tile's keys, nor that
// and `row`, the sum of the row's weights before, for these and `lossy` keys before.  Nothing 2^60 below is looked at: fewer than 2^31 keys have no weight
// there, and sums and O stay finite.  (A tile without a key has top -inf.)
__device__ __forceinline__ bool pair_lowers(float ref, float top, float tile, float row, int n, float lossy) {
  const float down = ref - top;
  return tile < kPairEnough * static_cast<float>(n) && row + tile < kPairEnough * (lossy + static_cast<float>(n)) && down > 0.f && down <= 60.f;
}
// The next `ref` of a row, by a thread that has all of it: `top` are the largest scores of N parts of the tile, to be multiplied by `scale`, `sum` is
// the row's so far, relative to `ref`.  lossy: keys so far, as far as what they lost weighs now (it moves with the sum).  settled: all rows of the warp
// have enough for what they lost and for the `left` keys from this tile on, which only a rise of `ref` changes.
template <int N>
__device__ __forceinline__ float pair_reference(float ref, float sum, float& lossy, const float (&top)[N], float scale, int n, int left, bool exists, bool& settled) {
  float best = top[0];
#pragma unroll
  for (int i = 1; i < N; ++i) best = fmaxf(best, top[i]);
  best *= scale;
  const bool up = best - ref > kPairRescale;
  float now = up ? (ref == -INFINITY ? best : best - kPairRise) : ref;
  if (!settled || __any_sync(0xffffffffu, up)) {
    const float f = up ? exp2_fast(ref - now) : 1.f, row = sum * f;
    lossy *= f;
    settled = __all_sync(0xffffffffu, row >= kPairEnough * (lossy + static_cast<float>(left)) || !exists);
    if (!settled && !__all_sync(0xffffffffu, row >= kPairEnough * (lossy + static_cast<float>(n)) || !exists)) {
      float tile = 0.f;
#pragma unroll
      for (int i = 0; i < N; ++i) tile += exp2_fast(fmaf(top[i], scale, kPairOffset - now));
      if (pair_lowers(now, best, tile, row, n, lossy)) {
        lossy *= exp2_fast(now - best);
        now = best;
      }
    }
  }
  lossy += static_cast<float>(n);
  return now;
}

// Row tile [rows][128 x 16-bit]: 16 chunks of 16 bytes per row, chunk index XOR-ed with
// (row & 7) so that ldmatrix reads and 16-byte row writes are bank-conflict free.
__device__ __forceinline__ uint32_t swz_off(int row, int chunk) {
  return static_cast<uint32_t>(row * 256 + ((chunk ^ (row & 7)) << 4));
}

// two e4m3 bytes (low 16 bits of x) -> packed pair of compute-type values
template <bool kHalf>
__device__ __forceinline__ uint32_t cvt_e4m3x2(uint16_t x) {
  __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(x), __NV_E4M3);
  if constexpr (kHalf) {
    return static_cast<uint32_t>(h.x) | (static_cast<uint32_t>(h.y) << 16);
  } else {
    __half2 hh = *reinterpret_cast<__half2*>(&h);
    float2 f = __half22float2(hh);
    return pack2<false>(f.x, f.y);
  }
}

__device__ __forceinline__ float bf16_bits_to_float(uint16_t b) {
  return __uint_as_float(static_cast<uint32_t>(b) << 16);
}

}  // namespace msa
