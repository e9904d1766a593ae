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

// ---- 8-bit pages with a scale per block ----
constexpr int kMostHeads = 1024;  // kv heads that the entry point lets through

// The smallest power of two s with amax <= 448 s (448 = 1.75 2^8), from
// kMinScale up to 2^120.
__device__ __forceinline__ float two_power(float amax) {
  const uint32_t u = __float_as_uint(amax);
  const int e = static_cast<int>(u >> 23) - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
  return __uint_as_float(static_cast<uint32_t>(min(max(e, 127 - 40), 247)) << 23);
}

// The new rows that fall into one block of one sequence are a run.  Sequence
// b has the runs [(indptr[b] >> shift) + 2 b, the same of b + 1): at least as
// many as blocks that it touches, so no scan is needed to number them, and
// those behind the last one have nothing to do.  This finds the sequence of a
// run, like find_seq.
__device__ __forceinline__ int find_run_seq(const int32_t* indptr, int B, int shift, int64_t run) {
  const int lane = threadIdx.x & 31;
  int lo = 0, n = B;
  while (true) {
    const int step = (n + 31) / 32;
    const int i = lane * step;
    const bool le = i < n && (indptr[lo + i] >> shift) + 2 * static_cast<int64_t>(lo + i) <= run;
    const int cnt = __popc(__ballot_sync(0xffffffffu, le));
    if (cnt == 0) return -1;
    lo += (cnt - 1) * step;
    n = min(step, n - (cnt - 1) * step);
    if (step == 1) return lo;
  }
}

// One CTA per run and slice of the heads (gridDim.y of them).  D / 16 lanes
// take one row of one head as in paged_write_kernel.  k and v are gone over
// twice: for the block's maxima, and to write the codes (the second read comes
// out of the caches).  The scale is a power of two, so codes lose nothing by it
// (8-bit floats), it can grow with the block, and the codes of the block's
// earlier tokens move to the larger one exactly unless they fall below the
// smallest normal code.  The angles of every row are made once per CTA.
// Measured: 7982 rows of 32 + 2 x 8 heads 49 to 52 us in blocks of 2 to 64, 54 in
// blocks of 128 (0.53 of the measured HBM rate; 16000 rows 0.61): every CTA
// is resident at once, so all of them wait for the same chain of reads, then
// for the angles.  With 40 registers a thread 72 us, with 100 64.
template <typename T, int D, int kThreads>
__global__ void __launch_bounds__(kThreads, 1024 / kThreads) paged_block_write_kernel(const __grid_constant__ PagedWrite a, int32_t* err) {
  constexpr int kLanes = D / 16, kGroups = kThreads / kLanes;
  extern __shared__ float2 s_turn[];  // [rows of the run][D / 2]: cosine and sine; then by k and v head of the slice:
  int* const s_amax = reinterpret_cast<int*>(s_turn + (D / 2 << a.c.scale_shift));  // maximum, as bits
  float2* const s_scale = s_turn + (D / 2 << a.c.scale_shift) + a.c.Hkv;            // new scale, and old over new
  pdl_wait();
  pdl_launch();
  const PagedCache& c = a.c;
  const int b = find_run_seq(c.indptr, c.B, c.scale_shift, blockIdx.x);
  if (b < 0) return;
  const int start = c.indptr[b], end = c.indptr[b + 1];
  const int64_t ctx = static_cast<int64_t>(c.lengths[b]) - (static_cast<int64_t>(end) - start);
  const int64_t run = blockIdx.x - ((start >> c.scale_shift) + 2 * static_cast<int64_t>(b));
  const int64_t p_new = ctx > 0 ? ctx : 0;  // the first new position
  const int64_t blk0 = ((p_new >> c.scale_shift) + run) << c.scale_shift;
  // new positions [p0, p1) of the block, rows from r0 on; rows outside of the activations are left out
  int64_t p0 = blk0 > p_new ? blk0 : p_new, p1 = blk0 + (int64_t{1} << c.scale_shift);
  if (p1 > c.lengths[b]) p1 = c.lengths[b];
  const int64_t row_of = static_cast<int64_t>(start) - ctx;  // row of position p: p + row_of
  if (p0 + row_of < 0) p0 = -row_of;
  if (p1 + row_of > a.rows) p1 = a.rows - row_of;
  if (p0 >= p1) return;
  const int64_t pi = p0 / c.page_size;
  const int pg = pi < c.max_pages ? c.table[b * c.table_stride + pi] : -1;
  if (pg < 0 || pg >= c.num_pages) {
    if (threadIdx.x == 0) raise_error(err, PERSONA_DEV_ERR_PAGE);
    return;
  }
  const int cnt = static_cast<int>(p1 - p0), at = static_cast<int>(p0 - pi * c.page_size);
  const int older = static_cast<int>(p0 - blk0);  // tokens of the block from before the call
  const int64_t r0 = p0 + row_of;
  const int slices = static_cast<int>(gridDim.y), slice = blockIdx.y;
  const int units = 2 * c.Hkv, mine = (units - slice + slices - 1) / slices;  // k and v heads: slice, slice + slices, ...
  {
    // Sines and cosines in 64 bits, rounded once: a code flips where k is nearer to
    // a tie than its error.  A thread has one frequency and a few rows: the first
    // one's angle by the function, the next ones' by a turn of one position each.
    constexpr int kParts = kThreads / (D / 2);
    const int f = threadIdx.x % (D / 2), each = (cnt + kParts - 1) / kParts;
    const int j0 = threadIdx.x / (D / 2) * each, j1 = min(cnt, j0 + each);
    if (j0 < j1) {
      const double t = static_cast<double>(p0 + j0) * a.turns[f];
      double sn, cs, s1 = 0.0, c1 = 1.0;
      sincospi(2.0 * (t - rint(t)), &sn, &cs);
      if (j0 + 1 < j1) sincospi(2.0 * a.turns[f], &s1, &c1);
      for (int j = j0; j < j1; ++j) {
        s_turn[j * (D / 2) + f] = make_float2(static_cast<float>(cs), static_cast<float>(sn));
        const double c = cs * c1 - sn * s1;
        sn = sn * c1 + cs * s1;
        cs = c;
      }
    }
  }
  for (int x = threadIdx.x; x < mine; x += kThreads) s_amax[x] = 0;
  __syncthreads();
  const int i = threadIdx.x % kLanes, group = threadIdx.x / kLanes;
  auto load = [&](const PagedRows& src, int j, int h, bool turn, float (&lo)[8], float (&hi)[8]) {
    const T* x = static_cast<const T*>(src.p) + (r0 + j) * src.row_stride + static_cast<int64_t>(h) * src.head_stride;
    unpack8<T>(*reinterpret_cast<const uint4*>(x + 8 * i), lo);
    unpack8<T>(*reinterpret_cast<const uint4*>(x + D / 2 + 8 * i), hi);
    if (turn) {
#pragma unroll
      for (int z = 0; z < 8; z += 2) {
        const float4 w = *reinterpret_cast<const float4*>(&s_turn[j * (D / 2) + 8 * i + z]);
        const float x1 = lo[z], x2 = hi[z], y1 = lo[z + 1], y2 = hi[z + 1];
        lo[z] = fmaf(x1, w.x, -x2 * w.y);
        hi[z] = fmaf(x2, w.x, x1 * w.y);
        lo[z + 1] = fmaf(y1, w.z, -y2 * w.w);
        hi[z + 1] = fmaf(y2, w.z, y1 * w.w);
      }
    }
  };
  float lo[8], hi[8];
  // ---- the maxima of the block's new rows ----
#pragma unroll 2
  for (int x0 = 0; x0 < mine * cnt; x0 += kGroups) {  // uniform trips: the lanes of a warp shuffle together
    const int x = x0 + group, u = x / cnt, j = x - u * cnt, uu = slice + u * slices;
    const bool live = x < mine * cnt, is_v = uu >= c.Hkv;
    float amax = 0.f;
    if (live) {
      load(is_v ? a.v : a.k, j, is_v ? uu - c.Hkv : uu, !is_v, lo, hi);
#pragma unroll
      for (int z = 0; z < 8; ++z) amax = fmaxf(amax, fmaxf(fabsf(lo[z]), fabsf(hi[z])));
    }
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    if (live && i == 0) atomicMax(&s_amax[u], __float_as_int(amax));
  }
  __syncthreads();
  const int64_t scale_at = pg * c.scale_page_stride + (at >> c.scale_shift);
  bool grown = false;
  for (int u = threadIdx.x; u < mine; u += kThreads) {
    const int uu = slice + u * slices;
    const bool is_v = uu >= c.Hkv;
    float* const sc = (is_v ? c.v_scale : c.k_scale) + scale_at + static_cast<int64_t>(is_v ? uu - c.Hkv : uu) * c.scale_head_stride;
    const float old = older > 0 ? *sc : 0.f, scale = fmaxf(old, two_power(__int_as_float(s_amax[u])));
    *sc = scale;
    s_scale[u] = make_float2(scale, older > 0 && scale > old ? old / scale : 1.f);
    grown |= older > 0 && scale > old;
  }
  const bool again = __syncthreads_or(grown);
  uint8_t *const k_at = static_cast<uint8_t*>(c.k) + static_cast<int64_t>(pg) * c.page_stride + at * c.pos_stride + 8 * i,
          *const v_at = static_cast<uint8_t*>(c.v) + static_cast<int64_t>(pg) * c.page_stride + at * c.pos_stride + 8 * i;
  // ---- the codes of the new rows ----
#pragma unroll 2
  for (int x = group; x < mine * cnt; x += kGroups) {
    const int u = x / cnt, j = x - u * cnt, uu = slice + u * slices;
    const bool is_v = uu >= c.Hkv;
    const int h = is_v ? uu - c.Hkv : uu;
    load(is_v ? a.v : a.k, j, h, !is_v, lo, hi);
    const float scale = s_scale[u].x, inv = 1.f / scale;
    uint8_t* o = (is_v ? v_at : k_at) + static_cast<int64_t>(h) * c.head_stride + j * c.pos_stride;
    *reinterpret_cast<uint2*>(o) = pack8_e4m3(lo, scale, inv);
    *reinterpret_cast<uint2*>(o + D / 2) = pack8_e4m3(hi, scale, inv);
  }
  // ---- those of the block's earlier tokens, where its scale has grown ----
  for (int x = group; again && x < mine * older; x += kGroups) {
    const int u = x / older, j = x - u * older - older, uu = slice + u * slices;
    const float ratio = s_scale[u].y;
    if (ratio == 1.f) continue;
    const bool is_v = uu >= c.Hkv;
    uint8_t* o = (is_v ? v_at : k_at) + static_cast<int64_t>(is_v ? uu - c.Hkv : uu) * c.head_stride + j * c.pos_stride;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      uint2* w = reinterpret_cast<uint2*>(o + half * (D / 2));
      const uint2 v = *w;
      uint32_t y[4];
      e4m3x4_to_half(v.x, y[0], y[1]);
      e4m3x4_to_half(v.y, y[2], y[3]);
#pragma unroll
      for (int z = 0; z < 4; ++z) {
        const float2 f = Cvt<__half>::to2(y[z]);
        lo[2 * z] = f.x * ratio;
        lo[2 * z + 1] = f.y * ratio;
      }
      *w = make_uint2(to_e4m3x2(lo[0], lo[1]) | static_cast<uint32_t>(to_e4m3x2(lo[2], lo[3])) << 16,
                      to_e4m3x2(lo[4], lo[5]) | static_cast<uint32_t>(to_e4m3x2(lo[6], lo[7])) << 16);
    }
  }
  // ---- q ----
  const int heads = (a.Hq - slice + slices - 1) / slices;
#pragma unroll 2
  for (int x = group; x < heads * cnt; x += kGroups) {
    const int j = x / heads, h = slice + (x - j * heads) * slices;
    load(a.q, j, h, true, lo, hi);
    T* o = static_cast<T*>(a.q_out.p) + (r0 + j) * a.q_out.row_stride + static_cast<int64_t>(h) * a.q_out.head_stride;
    *reinterpret_cast<uint4*>(o + 8 * i) = pack8<T>(lo);
    *reinterpret_cast<uint4*>(o + D / 2 + 8 * i) = pack8<T>(hi);
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
  const int64_t sfrom = page * a.c.scale_page_stride + (at >> a.c.scale_shift);
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
template <typename T, int D, int kThreads>
cudaError_t block_write_launch(const PagedWrite& a, int slices, int32_t* err, cudaStream_t st) {
  auto k = paged_block_write_kernel<T, D, kThreads>;
  // angles; maxima, scales and ratios by head
  const int smem = ((D / 2 << a.c.scale_shift) + 3 * a.c.Hkv) * static_cast<int>(sizeof(float2));
  static std::atomic<bool> done[64];
  const cudaError_t e = prepare_kernel(done, k, ((64 << 7) + 3 * kMostHeads) * static_cast<int>(sizeof(float2)), 0);
  if (e != cudaSuccess) return e;
  const int64_t runs = (a.rows >> a.c.scale_shift) + 2 * static_cast<int64_t>(a.c.B);
  return launch_paged(k, dim3(static_cast<unsigned>(runs), slices), dim3(kThreads), smem, 1, true, st, a, err);
}
template <typename T, int D>
cudaError_t block_write_dim(const PagedWrite& a, int32_t* err, cudaStream_t st) {
  // Threads by the block's size, and few slices, since each makes the angles anew.
  // 7982 prompt rows of 32 + 2 x 8 heads, threads x slices as chosen and beside it, us:
  // blocks of 2 128 x 1 49 (x 2 54, 256 x 1 55), of 8 128 x 1 51 (x 2 50, 256 x 1 52), of 16
  // 128 x 2 52 (x 1 66, x 4 50), of 32 128 x 4 52 (x 2 67, 256 x 2 52), of 64 512 x 2 52 (x 1
  // 93, x 4 56, 128 x 4 75), of 128 512 x 4 54 (x 2 93, 256 x 8 72).  64 single tokens take
  // 5.6 to 5.8 in any of these, but 7.8 with 512 x 4.
  const int block = 1 << a.c.scale_shift;
  return block < 32   ? block_write_launch<T, D, 128>(a, block < 16 ? 1 : 2, err, st)
         : block < 64 ? block_write_launch<T, D, 128>(a, 4, err, st)
                      : block_write_launch<T, D, 512>(a, block < 128 ? 2 : 4, err, st);
}
template <typename T>
cudaError_t block_write_for(const PagedWrite& a, int32_t* err, cudaStream_t st) {
  return a.c.D == 128 ? block_write_dim<T, 128>(a, err, st) : block_write_dim<T, 64>(a, err, st);
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
cudaError_t launch_paged_block_write(const PagedWrite& a, int dtype, int32_t* err, cudaStream_t st) {
  return dtype == PERSONA_DTYPE_BF16 ? block_write_for<__nv_bfloat16>(a, err, st) : block_write_for<__half>(a, err, st);
}
cudaError_t launch_paged_read(const PagedRead& a, int dtype, int32_t* err, cudaStream_t st) {
  return dtype == PERSONA_DTYPE_BF16 ? read_for<__nv_bfloat16>(a, err, st) : read_for<__half>(a, err, st);
}

}  // namespace persona
