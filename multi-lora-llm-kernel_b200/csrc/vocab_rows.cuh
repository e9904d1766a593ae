// Rows over the vocabulary as the draft verification and the sampling read
// them: eight elements a lane, and sums over a warp.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "paged_common.cuh"

namespace persona {

// Elements [x, x + 8) of a row of V as they are stored; 0 outside of it.
// 16-byte loads where the address allows.
template <typename T> struct Raw {
  static constexpr bool kWide = sizeof(T) == 4;
  uint32_t u[kWide ? 8 : 4];
  __device__ __forceinline__ void load(const void* base, int64_t row, int x, int V) {
    const char* p = static_cast<const char*>(base) + (row + x) * (kWide ? 4 : 2);
    if (x >= 0 && x + 8 <= V && (reinterpret_cast<uintptr_t>(p) & 15) == 0) {
#pragma unroll
      for (int i = 0; i < (kWide ? 2 : 1); ++i) {
        const uint4 a = __ldg(reinterpret_cast<const uint4*>(p) + i);
        u[4 * i] = a.x;
        u[4 * i + 1] = a.y;
        u[4 * i + 2] = a.z;
        u[4 * i + 3] = a.w;
      }
    } else if (x + 8 <= 0 || x >= V) {
      zero();
    } else if constexpr (kWide) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        u[i] = x + i >= 0 && x + i < V ? static_cast<const uint32_t*>(base)[row + x + i] : 0u;
    } else {
      const uint16_t* h = static_cast<const uint16_t*>(base) + row + x;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        u[i] = (x + 2 * i >= 0 && x + 2 * i < V ? h[2 * i] : 0u) |
               (x + 2 * i + 1 >= 0 && x + 2 * i + 1 < V ? static_cast<uint32_t>(h[2 * i + 1]) << 16 : 0u);
    }
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < (kWide ? 8 : 4); ++i) u[i] = 0u;
  }
  __device__ __forceinline__ void values(float (&f)[8]) const {
    if constexpr (kWide) {
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = __uint_as_float(u[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 v = Cvt<T>::to2(u[i]);
        f[2 * i] = v.x;
        f[2 * i + 1] = v.y;
      }
    }
  }
};

__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// Sum over the lanes up to and with this one.
__device__ __forceinline__ double warp_scan(double v) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double up = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += up;
  }
  return v;
}

// Sums over the warp of kN values (a power of two) at once: every exchange halves how
// many a lane still carries.  Value i ends in the lanes whose top bits are i.
template <int kN> __device__ __forceinline__ double warp_sums(double (&s)[kN]) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 16, k = kN / 2; k > 0; o >>= 1, k >>= 1) {
    const bool up = (lane & o) != 0;
#pragma unroll
    for (int i = 0; i < k; ++i) {
      const double keep = up ? s[k + i] : s[i], send = up ? s[i] : s[k + i];
      s[i] = keep + __shfl_xor_sync(0xffffffffu, send, o);
    }
  }
  double v = s[0];
#pragma unroll
  for (int o = 16 / kN; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

}  // namespace persona
