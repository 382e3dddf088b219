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
inline cudaError_t launch_chained(void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream, A&&... args) {
  // Under capture the launches stay plain: with programmatic edges the replay of a six-kernel decode graph took 86.5 us
  // against 77 us.
  cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
  cudaStreamIsCapturing(stream, &capture);
  cudaLaunchAttribute attr = {};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = capture == cudaStreamCaptureStatusNone ? 1 : 0;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid; cfg.blockDim = block; cfg.dynamicSmemBytes = smem; cfg.stream = stream;
  cfg.attrs = &attr; cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, P(args)...);
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

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
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
