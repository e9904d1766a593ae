// What the two attention kernels of the paged cache share: cp.async, the
// batch's geometry, the layout of partial results and the kernel that joins
// them.
#pragma once

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

// Position p of sequence b: its offset (elements) in the pages of head 0 and
// of the scales.
struct Pager {
  const int32_t* row;  // the sequence's page table
  int page_size, max_pages, num_pages;
  int32_t* err;
  __device__ __forceinline__ int page_of(int p, int& at) const {
    const int pi = p / page_size;
    at = p - pi * page_size;
    const int pg = pi < max_pages ? row[pi] : -1;
    if (pg < 0 || pg >= num_pages) {
      raise_error(err, PERSONA_DEV_ERR_PAGE);
      return -1;
    }
    return pg;
  }
};

// Joins the pieces of one cut tile: CTA c looks after the tile whose first
// piece CTA c of the attention left.  A warp per row, pieces in order;
// gridDim.y CTAs share the rows.
template <typename T, int D, int TR>
__global__ void __launch_bounds__(256) paged_combine_kernel(const __grid_constant__ PagedAttention a) {
  pdl_wait();
  pdl_launch();
  const int4 d = a.desc[blockIdx.x];
  if (d.w == 0) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int b = d.x, tile = d.y / a.c.Hkv, h = d.y % a.c.Hkv, first = blockIdx.x, pieces = d.z - first + 1;
  const Seq seq = load_seq(a, b);
  const int m0 = tile * TR, mrows = min(TR, seq.n * a.G - m0);
  constexpr int kF = Part<TR, D>::kFloats, kV = D / 32;
  const float* p0 = a.part + static_cast<int64_t>(2 * first + d.w - 1) * kF;
  // piece i > 0 is the first piece of CTA first + i
  auto piece = [&](int i) { return i == 0 ? p0 : a.part + static_cast<int64_t>(2 * (first + i)) * kF; };
  for (int m = blockIdx.y * 8 + warp; m < mrows; m += 8 * gridDim.y) {
    float mx = kNegInf;
    for (int i = lane; i < pieces; i += 32) mx = fmaxf(mx, piece(i)[TR * D + m]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    float l = 0.f, o[kV];
#pragma unroll
    for (int x = 0; x < kV; ++x) o[x] = 0.f;
    if (mx != kNegInf) {
#pragma unroll 4
      for (int i = 0; i < pieces; ++i) {
        const float* p = piece(i);
        const float f = exp2_approx(p[TR * D + m] - mx);
        l = fmaf(f, p[TR * D + TR + m], l);
#pragma unroll
        for (int x = 0; x < kV; ++x) o[x] = fmaf(f, p[m * D + lane * kV + x], o[x]);
      }
    }
    const float inv = l > 0.f ? 1.f / l : 0.f;
    const int mm = m0 + m, tok = mm / a.G;
    T* dst = static_cast<T*>(a.out.p) + static_cast<int64_t>(seq.row0 + tok) * a.out.row_stride +
             static_cast<int64_t>(h * a.G + mm - tok * a.G) * a.out.head_stride + lane * kV;
#pragma unroll
    for (int x = 0; x < kV; x += 2)
      *reinterpret_cast<uint32_t*>(dst + x) = Mma<T>::pack(o[x] * inv, o[x + 1] * inv);
  }
}

inline int sm_count() {
  int dev = 0, n = 148;
  if (cudaGetDevice(&dev) != cudaSuccess) return n;
  if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 148;
  return n;
}

}  // namespace persona
