// Device helpers shared by the paged KV cache kernels.
#pragma once

#include <atomic>

#include "common.cuh"
#include "paged_args.h"

namespace persona {

__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void pdl_launch() { asm volatile("griddepcontrol.launch_dependents;"); }

// Page of a position.
__device__ __forceinline__ int page_index(const PagedCache& c, int p) {
  return c.page_shift >= 0 ? p >> c.page_shift : p / c.page_size;
}

// The sequence that row r belongs to: the largest b in [0, B) with
// indptr[b] <= r, or -1.  Warp-wide: 32 probes per step, so one step up to
// 32 sequences and two up to 1024.  Whatever indptr holds, b stays in range.
__device__ __forceinline__ int find_seq(const int32_t* indptr, int B, int r) {
  const int lane = threadIdx.x & 31;
  int lo = 0, n = B;
  while (true) {
    const int step = (n + 31) / 32;
    const int i = lane * step;
    const bool le = i < n && indptr[lo + i] <= r;
    const int cnt = __popc(__ballot_sync(0xffffffffu, le));
    if (cnt == 0) return -1;
    lo += (cnt - 1) * step;
    n = min(step, n - (cnt - 1) * step);
    if (step == 1) return lo;
  }
}

// Where row r's token sits in the cache: its position, page and place in the
// page.  False for a row of no sequence and for one before position 0 (left
// alone), and, with PERSONA_DEV_ERR_PAGE raised, for a position behind the
// page table or a page outside the cache.  Warp-wide.
__device__ __forceinline__ bool locate_row(const PagedCache& c, int r, int32_t* err, int& pos, int64_t& page, int& at) {
  const int b = find_seq(c.indptr, c.B, r);
  if (b < 0) return false;
  const int end = c.indptr[b + 1];
  if (r >= end) return false;
  const int64_t p = static_cast<int64_t>(c.lengths[b]) - (static_cast<int64_t>(end) - r);
  if (p < 0) return false;
  const int64_t pi = p < 2147483647 ? page_index(c, static_cast<int>(p)) : p / c.page_size;
  const int pg = pi < c.max_pages ? c.table[b * c.table_stride + pi] : -1;
  if (pg < 0 || pg >= c.num_pages) {
    if ((threadIdx.x & 31) == 0) raise_error(err, PERSONA_DEV_ERR_PAGE);
    return false;
  }
  pos = static_cast<int>(p);
  page = pg;
  at = static_cast<int>(p - pi * c.page_size);
  return true;
}

// Four e4m3 codes of a word as two pairs of fp16 (exact: every e4m3 value is
// an fp16 value).
__device__ __forceinline__ void e4m3x4_to_half(uint32_t w, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
      : "=r"(lo), "=r"(hi)
      : "r"(w));
}

// Two fp32 as e4m3 codes, `lo` in the low byte, round to nearest even,
// saturating.
__device__ __forceinline__ uint16_t to_e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}

constexpr float kE4m3Max = 448.f;
// Smallest scale written: 2^-40 keeps 1 / scale and scale * 448 far inside
// fp32 and lies below what the smallest fp16 value needs (2^-24 / 448).
constexpr float kMinScale = 9.094947017729282e-13f;

// SMs of the current device.
inline int sm_count() {
  static std::atomic<int> known[64];
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
  n = known[dev].load(std::memory_order_relaxed);
  if (n > 0) return n;
  if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 148;
  known[dev].store(n, std::memory_order_relaxed);
  return n;
}

// Launches `kern`, as a programmatic dependent of the kernel before it if
// `early`.  A kernel that takes most of an SM's shared memory is not launched
// early: the SM keeps the division of its memory for as long as the kernel
// before is resident, and a grid that is meant to be resident as a whole gets
// fewer blocks per SM (three blocks of 68 KB became two: 77 us instead of 55).
template <typename... KArgs, typename... Args>
cudaError_t launch_paged(void (*kern)(KArgs...), dim3 grid, dim3 block, size_t smem, int cluster_x, bool early,
                         cudaStream_t st, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  if (early) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (cluster_x > 1) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
    attr[cfg.numAttrs].val.clusterDim.x = cluster_x;
    attr[cfg.numAttrs].val.clusterDim.y = 1;
    attr[cfg.numAttrs++].val.clusterDim.z = 1;
  }
  cfg.attrs = attr;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, static_cast<KArgs>(args)...);
  if (e != cudaSuccess) return e;
  return cudaGetLastError();
}

}  // namespace persona
