// What the two attention kernels of the paged cache share: cp.async, the
// batch's geometry, the layout of partial results and the kernel that joins
// them.
#pragma once

#include <atomic>
#include <type_traits>

#include "paged_common.cuh"

namespace persona {

constexpr float kNegInf = -INFINITY;

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool live) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src, bool live) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(live ? 4 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float log2_approx(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp_approx(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// log2 of how far a row's maximum may outgrow the one its weights are taken
// against before they are rescaled: weights up to 2^8 round as well as those
// up to 1 do, and a rescaling of all outputs becomes rare.
constexpr float kGrow = 8.f;
// Smallest v scale the kernels compute with (its logarithm and reciprocal).
constexpr float kLeastScale = 8.673617379884035e-19f;  // 2^-60

// A sequence as the kernels see it.
struct Seq {
  int row0, n, len;  // first row, new tokens, cached positions (new ones among them)
};
__device__ __forceinline__ Seq load_seq(const PagedAttention& a, int b) {
  Seq s;
  const int r0 = a.c.indptr[b], r1 = a.c.indptr[b + 1];
  const int64_t cap = static_cast<int64_t>(a.c.max_pages) * a.c.page_size;
  const int len = a.c.lengths[b];
  const bool bad = r0 < 0 || r1 < r0 || r1 > a.rows;
  s.row0 = r0;
  s.n = bad ? 0 : r1 - r0;
  s.len = len < 0 ? 0 : len > cap ? static_cast<int>(cap) : len;
  if (bad) raise_error(a.err, PERSONA_DEV_ERR_SEGMENT);
  if (s.n > 0 && len > cap) raise_error(a.err, PERSONA_DEV_ERR_PAGE);
  return s;
}
template <int TR, int D> struct Part {  // one piece: TR x D outputs, TR maxima, TR sums
  static constexpr int kFloats = TR * D + 2 * TR;
};

// A CTA notes the tile whose first piece it leaves unfinished, for the kernel
// below: {part slot of that piece, last CTA with a piece, first row of the
// tile, rows} and {first row of the sequence, kv head, -, -}; no rows: none.
__device__ __forceinline__ void note_cut(const PagedAttention& a, int cta, bool first_piece, int last_cta, int m0, int mrows,
                                         int row0, int h) {
  a.desc[2 * cta] = make_int4(2 * cta + (first_piece ? 0 : 1), last_cta, m0, mrows);
  a.desc[2 * cta + 1] = make_int4(row0, h, 0, 0);
}

// Joins the pieces of one cut tile: CTA c looks after the tile whose first
// piece CTA c of the attention left.  A warp per row; gridDim.y CTAs share the
// rows.  The weights of up to 32 pieces sit in the lanes, so that the pieces'
// rows are read without waiting for one another, and are added in order.
template <typename T, int D, int TR>
__global__ void __launch_bounds__(256) paged_combine_kernel(const __grid_constant__ PagedAttention a) {
  pdl_wait();
  pdl_launch();
  const int4 d = a.desc[2 * blockIdx.x];
  if (d.w == 0) return;
  const int4 e = a.desc[2 * blockIdx.x + 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int first = blockIdx.x, pieces = d.y - first + 1, m0 = d.z, mrows = d.w;
  constexpr int kF = Part<TR, D>::kFloats, kV = D / 32;
  // piece i > 0 is the first piece of CTA first + i
  auto piece = [&](int i) { return a.part + static_cast<int64_t>(i == 0 ? d.x : 2 * (first + i)) * kF; };
  for (int m = blockIdx.y * 8 + warp; m < mrows; m += 8 * gridDim.y) {
    float mx = kNegInf, l = 0.f, o[kV];
#pragma unroll
    for (int x = 0; x < kV; ++x) o[x] = 0.f;
    for (int i0 = 0; i0 < pieces; i0 += 32) {
      const int n = min(32, pieces - i0);
      float pm = kNegInf, pl = 0.f;
      if (lane < n) {
        const float* p = piece(i0 + lane) + TR * D + m;
        pm = p[0];
        pl = p[TR];
      }
      float top = pm;
#pragma unroll
      for (int s = 16; s > 0; s >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, s));
      top = fmaxf(top, mx);
      if (top == kNegInf) continue;  // nothing seen so far
      const float f = exp2_approx(pm - top), old = exp2_approx(mx - top);
      mx = top;
      pl *= f;
#pragma unroll
      for (int s = 16; s > 0; s >>= 1) pl += __shfl_xor_sync(0xffffffffu, pl, s);
      l = fmaf(l, old, pl);
#pragma unroll
      for (int x = 0; x < kV; ++x) o[x] *= old;
#pragma unroll 4
      for (int i = 0; i < n; ++i) {
        const float* p = piece(i0 + i) + m * D + lane * kV;
        const float fi = __shfl_sync(0xffffffffu, f, i);
        if constexpr (kV == 4) {
          const float4 v = *reinterpret_cast<const float4*>(p);
          o[0] = fmaf(fi, v.x, o[0]);
          o[1] = fmaf(fi, v.y, o[1]);
          o[2] = fmaf(fi, v.z, o[2]);
          o[3] = fmaf(fi, v.w, o[3]);
        } else {
          const float2 v = *reinterpret_cast<const float2*>(p);
          o[0] = fmaf(fi, v.x, o[0]);
          o[1] = fmaf(fi, v.y, o[1]);
        }
      }
    }
    const float inv = l > 0.f ? 1.f / l : 0.f;
    const int mm = m0 + m, tok = mm / a.G;
    T* dst = static_cast<T*>(a.out.p) + static_cast<int64_t>(e.x + tok) * a.out.row_stride +
             static_cast<int64_t>(e.y * a.G + mm - tok * a.G) * a.out.head_stride + lane * kV;
#pragma unroll
    for (int x = 0; x < kV; x += 2)
      *reinterpret_cast<uint32_t*>(dst + x) = Mma<T>::pack(o[x] * inv, o[x + 1] * inv);
  }
}

// A kernel's attributes, set once per device: allows `smem` bytes of dynamic
// shared memory and, where regs > 0, checks that the kernel is launched with
// that many registers a thread.  `done`: one flag per device, static at the
// caller.
template <typename K> cudaError_t prepare_kernel(std::atomic<bool> (&done)[64], K kernel, int smem, int regs) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 64 && done[dev].load(std::memory_order_acquire)) return cudaSuccess;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return e;
  if (regs > 0) {
    cudaFuncAttributes attr;
    e = cudaFuncGetAttributes(&attr, kernel);
    if (e != cudaSuccess) return e;
    if (attr.numRegs != regs) return cudaErrorInvalidConfiguration;
  }
  if (dev < 64) done[dev].store(true, std::memory_order_release);
  return cudaSuccess;
}

}  // namespace persona
