// Verification of drafted tokens against the target's probabilities from
// given random numbers (speculative sampling, Leviathan et al. 2023 and Chen
// et al. 2023): draft i is kept while u_i q_i(d_i) < p_i(d_i); the first one
// that is not is replaced by a draw from max(p - q, 0), and a sequence that
// keeps all of its drafts draws one more token from its last row of p.
//
// What it must read is one row of each distribution per sequence, so it is
// bound by HBM for a full batch and by its chain of dependent steps for a
// few sequences.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "paged_common.cuh"

namespace persona {
namespace cg = cooperative_groups;
namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kSplit = 8;        // CTAs (one cluster) per sequence
constexpr int kTile = 256;       // elements of one tile: 8 a lane
constexpr int kMaxTiles = 1024;  // tiles of one CTA: V up to kSplit * kMaxTiles * kTile

template <typename T> __device__ __forceinline__ float prob(const void* p, int64_t i) {
  return Cvt<T>::to1(static_cast<const uint16_t*>(p)[i]);
}
template <> __device__ __forceinline__ float prob<float>(const void* p, int64_t i) {
  return static_cast<const float*>(p)[i];
}

// The weight of token t: max(p - q, 0), or p (mode 0), or p without token
// `skip` (the residual of a draft that was certain of it).  A weight that is
// not positive, a NaN among them, counts as none.
template <typename T>
__device__ __forceinline__ double weight(const void* p, const void* q, int64_t prow, int64_t qrow, int t, int skip) {
  const double x = prob<T>(p, prow + t);
  const double w = q != nullptr ? x - static_cast<double>(prob<T>(q, qrow + t)) : t == skip ? 0.0 : x;
  return w > 0.0 ? w : 0.0;
}

__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// One cluster per sequence; CTA c sums the weights of its eighth of the
// vocabulary tile by tile, in 64 bits (the draw compares sums of up to 2^21
// terms with a number that falls between two of them), the CTAs exchange
// their sums, and the one whose range the number falls in finds the tile and
// then the token.
template <typename T>
__global__ void __launch_bounds__(kThreads) verify_draft_kernel(const __grid_constant__ VerifyDraft a) {
  cg::cluster_group cluster = cg::this_cluster();
  pdl_wait();
  pdl_launch();
  __shared__ double s_tile[kMaxTiles];
  __shared__ double s_sum;
  __shared__ double s_warp[kWarps];
  __shared__ int s_acc;
  const int b = blockIdx.x / kSplit, rank = blockIdx.x % kSplit;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int r0 = a.indptr[b], r1 = a.indptr[b + 1];
  const int n = r1 - r0;
  // the same in every CTA of the cluster, which therefore leaves together
  if (r0 < 0 || r1 > a.rows || n < 0) {
    if (rank == 0 && tid == 0) {
      raise_error(a.err, PERSONA_DEV_ERR_SEGMENT);
      a.accepted[b] = 0;
    }
    return;
  }
  if (n == 0) {
    if (rank == 0 && tid == 0) a.accepted[b] = 0;
    return;
  }
  // drafts kept: the first 32 judged rows at once, then the next 32
  if (warp == 0) {
    int kept = 0;
    while (kept < n - 1) {
      const int i = kept + lane;
      bool ok = false;
      if (i < n - 1) {
        const int64_t r = r0 + i, d = a.draft_tokens[r];
        if (d < 0 || d >= a.V) {
          if (rank == 0) raise_error(a.err, PERSONA_DEV_ERR_TOKEN);
        } else {
          const double p = prob<T>(a.target, r * a.ld_target + d);
          const double q = a.draft != nullptr ? prob<T>(a.draft, r * a.ld_draft + d) : 1.0;
          ok = static_cast<double>(a.u_accept[r]) * q < p;
        }
      }
      const unsigned no = ~__ballot_sync(0xffffffffu, ok);
      const int run = no == 0 ? 32 : __ffs(no) - 1;
      kept += run;
      if (run < 32) break;
    }
    if (lane == 0) s_acc = kept;
  }
  __syncthreads();
  const int acc = s_acc;
  const int64_t row = r0 + acc;
  const bool rejected = acc < n - 1;
  const int per = ((a.V + kSplit - 1) / kSplit + kTile - 1) / kTile * kTile;
  const int lo = min(a.V, rank * per), hi = min(a.V, lo + per);
  const int tiles = (hi - lo + kTile - 1) / kTile;
  // mode 1: the residual of a rejected draft; mode 0: p itself, also where
  // the residual has no weight left (p and q equal up to rounding)
  double total = 0.0, before = 0.0;
  const void* q = nullptr;
  int skip = -1, last = -1;  // last: the last CTA with weight
  for (int mode = rejected ? 1 : 0; mode >= 0; --mode) {
    q = mode == 1 ? a.draft : nullptr;
    skip = mode == 1 && a.draft == nullptr ? static_cast<int>(a.draft_tokens[row]) : -1;
    const int64_t prow = row * a.ld_target, qrow = row * a.ld_draft;
    double sum = 0.0;
    for (int t = warp; t < tiles; t += kWarps) {
      double s = 0.0;
#pragma unroll
      for (int j = 0; j < kTile / 32; ++j) {
        const int x = lo + t * kTile + j * 32 + lane;
        if (x < hi) s += weight<T>(a.target, q, prow, qrow, x, skip);
      }
      s = warp_sum(s);
      if (lane == 0) s_tile[t] = s;
      sum += s;
    }
    if (lane == 0) s_warp[warp] = sum;
    __syncthreads();
    if (tid == 0) {
      double s = 0.0;
      for (int w = 0; w < kWarps; ++w) s += s_warp[w];
      s_sum = s;
    }
    cluster.sync();
    total = before = 0.0;
    for (int c = 0; c < kSplit; ++c) {
      const double s = *cluster.map_shared_rank(&s_sum, c);
      if (c < rank) before += s;
      total += s;
      if (s > 0.0) last = c;
    }
    cluster.sync();  // nobody overwrites or leaves while its sum is read
    if (total > 0.0) break;
  }
  const int i0 = rank == 0 ? tid : n;  // the accepted drafts, and -1 behind the drawn token
  for (int i = i0; i < n; i += kThreads)
    if (i != acc) a.tokens[r0 + i] = i < acc ? a.draft_tokens[r0 + i] : -1;
  if (rank == 0 && tid == 0) a.accepted[b] = acc;
  if (!(total > 0.0)) {  // not one positive weight: no token can be drawn
    if (rank == 0 && tid == 0) a.tokens[row] = -1;
    return;
  }
  // The number falls into the first tile whose running sum exceeds it; where
  // rounding (or a number of 1) leaves none, the last tile with weight has it.
  const double target = static_cast<double>(a.u_sample[b]) * total;
  const double mine = s_sum;
  // (before + mine is the next CTA's `before` to the bit, so one CTA goes on.)
  const bool chosen = total > target ? before + mine > target && !(before > target) : rank == last;
  if (!chosen || warp != 0) return;
  // Running sums over the tiles, 32 at a time; `at`: the tile, `run`: the sum before it.
  int at = -1;
  double run = before, at_run = before;
  for (int t0 = 0; t0 < tiles; t0 += 32) {
    const double s = t0 + lane < tiles ? s_tile[t0 + lane] : 0.0;
    double inc = s;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double up = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += up;
    }
    const unsigned over = __ballot_sync(0xffffffffu, s > 0.0 && run + inc > target);
    const unsigned some = __ballot_sync(0xffffffffu, s > 0.0);
    if (over != 0 || some != 0) {
      const int l = over != 0 ? __ffs(over) - 1 : 31 - __clz(some);
      at = t0 + l;
      at_run = run + __shfl_sync(0xffffffffu, inc - s, l);
    }
    if (over != 0) break;
    run += __shfl_sync(0xffffffffu, inc, 31);
  }
  if (at < 0) return;  // cannot be: this CTA's sum is positive
  // Inside the tile: 8 consecutive tokens a lane.
  const int64_t prow = row * a.ld_target, qrow = row * a.ld_draft;
  const int x0 = lo + at * kTile + lane * 8;
  double w[8], s = 0.0;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    w[j] = x0 + j < hi ? weight<T>(a.target, q, prow, qrow, x0 + j, skip) : 0.0;
    s += w[j];
  }
  double inc = s;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double up = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += up;
  }
  double sum = at_run + (inc - s);
  int first = -1, tail = -1;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    sum += w[j];
    if (w[j] > 0.0) {
      tail = x0 + j;
      if (first < 0 && sum > target) first = x0 + j;
    }
  }
  const unsigned over = __ballot_sync(0xffffffffu, first >= 0), some = __ballot_sync(0xffffffffu, tail >= 0);
  const int l = over != 0 ? __ffs(over) - 1 : 31 - __clz(some | 1u);
  const int tok = __shfl_sync(0xffffffffu, over != 0 ? first : tail, l);
  if (lane == 0) a.tokens[row] = tok;
}

}  // namespace

cudaError_t launch_verify_draft(const VerifyDraft& a, int type, cudaStream_t st) {
  auto k = type == 2 ? verify_draft_kernel<float> : type == 1 ? verify_draft_kernel<__nv_bfloat16> : verify_draft_kernel<__half>;
  return launch_paged(k, dim3(a.B * kSplit), dim3(kThreads), 0, kSplit, st, a);
}

}  // namespace persona
