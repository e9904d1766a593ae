// Paged KV cache: rotary embedding and page write of a ragged batch of new
// tokens, and the read of cached positions back into dense rows.
//
// Both are bound by HBM at prompt sizes and by the latency of their chain of
// small reads (indptr, length, page table) at decode sizes.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "paged_common.cuh"

namespace persona {
namespace {

constexpr int kWriteThreads = 128;

// 8 16-bit values <-> fp32.
template <typename T>
__device__ __forceinline__ void unpack8(const uint4& w, float (&f)[8]) {
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 p = Cvt<T>::to2(u[i]);
    f[2 * i] = p.x;
    f[2 * i + 1] = p.y;
  }
}
template <typename T>
__device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
  return make_uint4(Mma<T>::pack(f[0], f[1]), Mma<T>::pack(f[2], f[3]), Mma<T>::pack(f[4], f[5]),
                    Mma<T>::pack(f[6], f[7]));
}
// Codes of f / scale.  The product with 1 / scale can lie on the wrong side of a
// tie between two codes (16-bit values and their maximum's 448th part make ties
// common), so it takes one step of its remainder (Markstein 1990): that leaves an
// error of 2^-23 of an fp32 step, so a quotient which is an fp32 number, as every
// tie is, comes out exact.  16384 rows: 71 us by the product alone, 72 with the
// step, 77 by division.
__device__ __forceinline__ float quotient(float x, float scale, float inv) {
  const float q = x * inv;
  return fmaf(fmaf(-q, scale, x), inv, q);
}
__device__ __forceinline__ uint2 pack8_e4m3(const float (&f)[8], float scale, float inv) {
  uint32_t w[2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
    w[i] = static_cast<uint32_t>(to_e4m3x2(quotient(f[4 * i], scale, inv), quotient(f[4 * i + 1], scale, inv))) |
           static_cast<uint32_t>(to_e4m3x2(quotient(f[4 * i + 2], scale, inv), quotient(f[4 * i + 3], scale, inv))) << 16;
  return make_uint2(w[0], w[1]);
}

// One CTA per row.  D / 16 lanes take one head: lane i holds dims [8i, 8i + 8)
// and their partners D / 2 further on, which are one rotation's two sides, so
// a head is two 16-byte loads and two stores per lane and no lane needs
// another's values but for the maximum of an e4m3 row.  The sines and cosines
// of the row's position are made once by the first D / 2 threads: position
// times turns in 64 bits, whose fraction carries the angle of a far position
// that a 32-bit product loses.
// Measured: 16384 rows of 32 + 2 x 8 heads into 8-bit pages 72 us among other
// calls, 0.79 of the measured HBM rate, into 16-bit pages 67 us, 0.92.  Twelve
// CTAs per SM (40 registers) were 6 % faster than the nine that 56 registers
// leave room for, and fourteen spill.
template <typename T, int D, bool kE4m3>
__global__ void __launch_bounds__(kWriteThreads, 12) paged_write_kernel(const __grid_constant__ PagedWrite a, int32_t* err) {
  constexpr int kLanes = D / 16;
  __shared__ float s_cos[D / 2], s_sin[D / 2];
  pdl_wait();
  pdl_launch();
  const int r = blockIdx.x;
  int pos, at;
  int64_t page;
  if (!locate_row(a.c, r, err, pos, page, at)) return;  // the same for every warp of the CTA
  if (threadIdx.x < D / 2) {
    const double t = static_cast<double>(pos) * a.turns[threadIdx.x];
    float sn, cs;
    sincospif(2.f * static_cast<float>(t - rint(t)), &sn, &cs);
    s_cos[threadIdx.x] = cs;
    s_sin[threadIdx.x] = sn;
  }
  __syncthreads();
  const int i = threadIdx.x % kLanes;
  float c[8], s[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    c[j] = s_cos[8 * i + j];
    s[j] = s_sin[8 * i + j];
  }
  const int Hq = a.Hq, Hkv = a.c.Hkv, heads = Hq + 2 * Hkv;
  const int64_t slot = page * a.c.page_stride + at * a.c.pos_stride;
  const int64_t sslot = page * a.c.scale_page_stride + at;
  for (int h0 = 0; h0 < heads; h0 += kWriteThreads / kLanes) {  // uniform trips: the lanes of a warp shuffle together
    const int hh = h0 + threadIdx.x / kLanes;
    const bool live = hh < heads;
    const bool is_q = hh < Hq, is_v = hh >= Hq + Hkv;
    const int kh = is_v ? hh - Hq - Hkv : hh - Hq;
    const PagedRows& src = is_q ? a.q : is_v ? a.v : a.k;
    const T* x = static_cast<const T*>(src.p) + static_cast<int64_t>(r) * src.row_stride +
                 static_cast<int64_t>(is_q ? hh : kh) * src.head_stride;
    float lo[8], hi[8];
    if (live) {
      unpack8<T>(*reinterpret_cast<const uint4*>(x + 8 * i), lo);
      unpack8<T>(*reinterpret_cast<const uint4*>(x + D / 2 + 8 * i), hi);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) lo[j] = hi[j] = 0.f;
    }
    if (!is_v) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float x1 = lo[j], x2 = hi[j];
        lo[j] = fmaf(x1, c[j], -x2 * s[j]);
        hi[j] = fmaf(x2, c[j], x1 * s[j]);
      }
    }
    float amax = 0.f;
    if (kE4m3) {
#pragma unroll
      for (int j = 0; j < 8; ++j) amax = fmaxf(amax, fmaxf(fabsf(lo[j]), fabsf(hi[j])));
#pragma unroll
      for (int o = kLanes / 2; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    }
    if (!live) continue;
    if (is_q) {
      T* o = static_cast<T*>(a.q_out.p) + static_cast<int64_t>(r) * a.q_out.row_stride +
             static_cast<int64_t>(hh) * a.q_out.head_stride;
      *reinterpret_cast<uint4*>(o + 8 * i) = pack8<T>(lo);
      *reinterpret_cast<uint4*>(o + D / 2 + 8 * i) = pack8<T>(hi);
    } else if (!kE4m3) {
      T* o = static_cast<T*>(is_v ? a.c.v : a.c.k) + slot + static_cast<int64_t>(kh) * a.c.head_stride;
      *reinterpret_cast<uint4*>(o + 8 * i) = pack8<T>(lo);
      *reinterpret_cast<uint4*>(o + D / 2 + 8 * i) = pack8<T>(hi);
    } else {
      // k is quantised from the fp32 rotation, not from a 16-bit rounding of it
      const float scale = fmaxf(amax / kE4m3Max, kMinScale), inv = 1.f / scale;
      uint8_t* o = static_cast<uint8_t*>(is_v ? a.c.v : a.c.k) + slot + static_cast<int64_t>(kh) * a.c.head_stride;
      *reinterpret_cast<uint2*>(o + 8 * i) = pack8_e4m3(lo, scale, inv);
      *reinterpret_cast<uint2*>(o + D / 2 + 8 * i) = pack8_e4m3(hi, scale, inv);
      if (i == 0) (is_v ? a.c.v_scale : a.c.k_scale)[sslot + static_cast<int64_t>(kh) * a.c.scale_head_stride] = scale;
    }
  }
}

// One warp per row: the position's k and v of every head, 16 bytes of the cache
// a lane and step.  Codes times scale are rounded once, to the rows' 16-bit
// type.  (Two to eight rows a warp, to share the search for the sequence, took
// as long at 36213 rows and 1.3 to 2.7 times as long at 1999.)
template <typename T, int D, bool kE4m3>
__global__ void __launch_bounds__(128) paged_read_kernel(const __grid_constant__ PagedRead a, int32_t* err) {
  pdl_wait();
  pdl_launch();
  const int r = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (r >= a.rows) return;
  int pos, at;
  int64_t page;
  if (!locate_row(a.c, r, err, pos, page, at)) return;
  const int64_t from = page * a.c.page_stride + at * a.c.pos_stride;
  const int64_t sfrom = page * a.c.scale_page_stride + at;
  constexpr int kEach = kE4m3 ? 16 : 8;  // elements of 16 bytes in the cache
  constexpr int kChunks = D / kEach;
  const int n = 2 * a.c.Hkv * kChunks;
#pragma unroll 4
  for (int x = lane; x < n; x += 32) {
    const int hh = x / kChunks, d = (x % kChunks) * kEach;
    const bool is_v = hh >= a.c.Hkv;
    const int64_t kh = is_v ? hh - a.c.Hkv : hh;
    const PagedRows& dst = is_v ? a.v : a.k;
    T* o = static_cast<T*>(dst.p) + static_cast<int64_t>(r) * dst.row_stride + kh * dst.head_stride + d;
    const char* src = static_cast<const char*>(is_v ? a.c.v : a.c.k) + (from + kh * a.c.head_stride + d) * (kE4m3 ? 1 : 2);
    const uint4 w = __ldg(reinterpret_cast<const uint4*>(src));
    if (!kE4m3) {
      *reinterpret_cast<uint4*>(o) = w;
    } else {
      const float sc = __ldg((is_v ? a.c.v_scale : a.c.k_scale) + sfrom + kh * a.c.scale_head_stride);
      const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        uint32_t h[4];
        e4m3x4_to_half(u[2 * y], h[0], h[1]);
        e4m3x4_to_half(u[2 * y + 1], h[2], h[3]);
        float f[8];
#pragma unroll
        for (int z = 0; z < 4; ++z) {
          const float2 p = Cvt<__half>::to2(h[z]);
          f[2 * z] = p.x * sc;
          f[2 * z + 1] = p.y * sc;
        }
        *reinterpret_cast<uint4*>(o + 8 * y) = pack8<T>(f);
      }
    }
  }
}

template <typename T>
cudaError_t write_for(const PagedWrite& a, int32_t* err, cudaStream_t st) {
  const bool e = a.c.k_scale != nullptr;
  auto k = a.c.D == 128 ? (e ? paged_write_kernel<T, 128, true> : paged_write_kernel<T, 128, false>)
                        : (e ? paged_write_kernel<T, 64, true> : paged_write_kernel<T, 64, false>);
  return launch_paged(k, dim3(a.rows), dim3(kWriteThreads), 0, 1, true, st, a, err);
}
template <typename T>
cudaError_t read_for(const PagedRead& a, int32_t* err, cudaStream_t st) {
  const bool e = a.c.k_scale != nullptr;
  auto k = a.c.D == 128 ? (e ? paged_read_kernel<T, 128, true> : paged_read_kernel<T, 128, false>)
                        : (e ? paged_read_kernel<T, 64, true> : paged_read_kernel<T, 64, false>);
  return launch_paged(k, dim3((a.rows + 3) / 4), dim3(128), 0, 1, true, st, a, err);
}

}  // namespace

cudaError_t launch_paged_write(const PagedWrite& a, int dtype, int32_t* err, cudaStream_t st) {
  return dtype == PERSONA_DTYPE_BF16 ? write_for<__nv_bfloat16>(a, err, st) : write_for<__half>(a, err, st);
}
cudaError_t launch_paged_read(const PagedRead& a, int dtype, int32_t* err, cudaStream_t st) {
  return dtype == PERSONA_DTYPE_BF16 ? read_for<__nv_bfloat16>(a, err, st) : read_for<__half>(a, err, st);
}

}  // namespace persona
