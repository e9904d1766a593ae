// Verification of drafted tokens against the target's probabilities from
// given random numbers (speculative sampling, Leviathan et al. 2023 and Chen
// et al. 2023): draft i is kept while u_i q_i(d_i) < p_i(d_i); the first one
// that is not is replaced by a draw from max(p - q, 0), and a sequence that
// keeps all of its drafts draws one more token from its last row of p.
//
// What it must read is one row of each distribution per sequence, so it is
// bound by its chain of dependent steps (rows, tokens, their probabilities, the
// row, the sums, the tile): 8 sequences of 4 drafts over 32000 tokens take 5.6
// us, 256 of up to 7 over 50257 16 us in fp16 (0.48 of the measured HBM
// rate; 17 in a graph), 21 us in bf16 and 23 in fp32 (0.69 of it), whose sums
// take more conversions to 64 bits.
#include <cooperative_groups.h>
#include <type_traits>

#include "vocab_rows.cuh"

namespace persona {
namespace cg = cooperative_groups;
namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kTile = 256;        // elements of one tile: 8 a lane
constexpr int kMaxSplit = 8;      // CTAs (one cluster) per sequence
constexpr int kMaxTiles = 1040;   // tiles of one CTA: the largest vocabulary over kMaxSplit CTAs, and a start off by a tile
static_assert(static_cast<int64_t>(kMaxTiles - 2) * kTile * kMaxSplit >= PERSONA_VERIFY_MAX_VOCAB, "tiles");

template <typename T> __device__ __forceinline__ float prob(const void* p, int64_t i) {
  return Cvt<T>::to1(static_cast<const uint16_t*>(p)[i]);
}
template <> __device__ __forceinline__ float prob<float>(const void* p, int64_t i) {
  return static_cast<const float*>(p)[i];
}

// The weight of one token: max(p - q, 0), exact in 64 bits but for a last
// rounding; one that is not positive, a NaN among them, counts as none.
__device__ __forceinline__ double weight(float p, float q) {
  return p > q ? static_cast<double>(p) - static_cast<double>(q) : 0.0;
}

// One cluster per sequence.  Every warp finds the kept drafts for itself (no
// barrier); CTA c sums the weights of its part of the vocabulary tile by
// tile, in 64 bits (the draw compares sums of up to 2^21 terms with a number
// that falls between two of them), the CTAs exchange their sums, and the one
// whose range the number falls in finds the tile and then the token.
template <typename T>
__global__ void __launch_bounds__(kThreads, 4) verify_draft_kernel(const __grid_constant__ VerifyDraft a) {
  cg::cluster_group cluster = cg::this_cluster();
  __shared__ double s_tile[kMaxTiles];
  __shared__ double s_warp[kWarps];
  __shared__ double s_sum[2];  // by mode
  const int split = static_cast<int>(cluster.num_blocks());
  const int b = blockIdx.x / split, rank = static_cast<int>(cluster.block_rank());
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  pdl_wait();
  pdl_launch();
  const int r0 = a.indptr[b], r1 = a.indptr[b + 1];
  const int n = r1 - r0;
  // the same in every CTA of the cluster, which therefore leaves together
  if (r0 < 0 || r1 > a.rows || n <= 0) {
    if (rank == 0 && tid == 0) {
      if (r0 < 0 || r1 > a.rows || n < 0) raise_error(a.err, PERSONA_DEV_ERR_SEGMENT);
      a.accepted[b] = 0;
    }
    return;
  }
  const float us = a.u_sample[b];
  // drafts kept: the first 32 judged rows at once, then the next 32
  int acc = 0;
  while (acc < n - 1) {
    const int i = acc + lane;
    bool ok = false;
    if (i < n - 1) {
      const int64_t r = r0 + i, d = a.draft_tokens[r];
      const double u = a.u_accept[r];
      if (d < 0 || d >= a.V) {
        if (rank == 0 && warp == 0) raise_error(a.err, PERSONA_DEV_ERR_TOKEN);
      } else {
        const double p = prob<T>(a.target, r * a.ld_target + d);
        const double q = a.draft != nullptr ? prob<T>(a.draft, r * a.ld_draft + d) : 1.0;
        ok = u * q < p;
      }
    }
    const unsigned no = ~__ballot_sync(0xffffffffu, ok);
    const int run = no == 0 ? 32 : __ffs(no) - 1;
    acc += run;
    if (run < 32) break;
  }
  const int64_t row = r0 + acc;
  const bool rejected = acc < n - 1;
  const int64_t prow = row * a.ld_target, qrow = row * a.ld_draft;
  if (rank == 0) {  // the kept drafts, and -1 behind the drawn token
    for (int i = tid; i < n; i += kThreads)
      if (i != acc) a.tokens[r0 + i] = i < acc ? a.draft_tokens[r0 + i] : -1;
    if (tid == 0) a.accepted[b] = acc;
  }
  // Tiles start `lead` elements before the row, on a 16-byte boundary.
  constexpr int kSize = sizeof(T) == 4 ? 4 : 2;
  const int lead =
      static_cast<int>(((reinterpret_cast<uintptr_t>(a.target) + static_cast<uint64_t>(prow) * kSize) & 15) / kSize);
  const int all = (a.V + lead + kTile - 1) / kTile, per = (all + split - 1) / split;
  const int t0 = min(all, rank * per), tiles = min(all, t0 + per) - t0;
  const int x0 = t0 * kTile - lead;  // first element of this CTA's first tile
  // Mode 1: the residual of a rejected draft; mode 0: p itself, also where
  // the residual has no weight left (p and q equal up to rounding).
  const void* q = nullptr;
  int skip = -1;
  auto weights = [&](const Raw<T>& rp, const Raw<T>& rq, int x, double (&w)[8]) {  // returns their sum
    float p[8], f[8];
    rp.values(p);
    rq.values(f);
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = x + i == skip ? 0.0 : weight(p[i], f[i]);
    return ((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7]));
  };
  // The sum alone.  fp16: differences of two numbers are multiples of 2^-24, and
  // fp32 holds those below 1 exactly, so a sum of such weights that comes out
  // below 1 had no larger part and no rounding: one conversion to 64 bits for
  // eight tokens instead of sixteen, which the SM makes 16 of per cycle.
  auto weight_sum = [&](const Raw<T>& rp, const Raw<T>& rq, int x) {
    if constexpr (std::is_same<T, __half>::value) {
      float p[8], f[8];
      rp.values(p);
      rq.values(f);
#pragma unroll
      for (int i = 0; i < 8; ++i) p[i] = p[i] > f[i] ? p[i] - f[i] : 0.f;
      const float s = ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
      if (s < 1.f && static_cast<unsigned>(skip - x) >= 8u) return static_cast<double>(s);
    }
    double w[8];
    return weights(rp, rq, x, w);
  };
  // tiles of a warp's step, all of whose loads are under way at once (256
  // sequences: four of fp16 take 18.9 us, two 17.1; of bf16 23.5 and 21.0)
  constexpr int kStep = 2;
  double total = 0.0, before = 0.0;
  int last = -1;  // the last CTA with weight
  int mode = rejected ? 1 : 0;
  while (true) {
    q = mode == 1 ? a.draft : nullptr;
    // a draft that was certain of its token: it is the only one with q > 0 (one
    // outside the vocabulary is no token of the row, whatever its low 32 bits)
    skip = -1;
    if (mode == 1 && a.draft == nullptr) {
      const int64_t d = a.draft_tokens[row];
      if (d >= 0 && d < a.V) skip = static_cast<int>(d);
    }
    double sum = 0.0;
    const int end = tiles * (warp + 1) / kWarps;
    for (int t = tiles * warp / kWarps; t < end; t += kStep) {
      Raw<T> rp[kStep], rq[kStep];
#pragma unroll
      for (int i = 0; i < kStep; ++i) {
        const int x = t + i < end ? x0 + (t + i) * kTile + lane * 8 : a.V;
        rp[i].load(a.target, prow, x, a.V);
        if (q != nullptr) {
          rq[i].load(q, qrow, x, a.V);
        } else {
          rq[i].zero();
        }
      }
      double s[kStep];
#pragma unroll
      for (int i = 0; i < kStep; ++i) s[i] = weight_sum(rp[i], rq[i], x0 + (t + i) * kTile + lane * 8);
      const double v = warp_sums<kStep>(s);
      const int i = lane / (32 / kStep);
      if (lane % (32 / kStep) == 0 && t + i < end) s_tile[t + i] = v;
      if (lane % (32 / kStep) == 0) sum += v;
    }
    sum = warp_sum(sum);
    if (lane == 0) s_warp[warp] = sum;
    __syncthreads();
    if (warp == 0) {
      const double s = warp_sum(lane < kWarps ? s_warp[lane] : 0.0);
      if (lane == 0) s_sum[mode] = s;
    }
    cluster.sync();
    // every lane reads one CTA's sum; they are added in the CTAs' order
    const double mine = lane < split ? *cluster.map_shared_rank(&s_sum[mode], lane) : 0.0;
    total = before = 0.0;
    last = -1;
    for (int c = 0; c < split; ++c) {
      const double s = __shfl_sync(0xffffffffu, mine, c);
      if (c < rank) before += s;
      total += s;
      if (s > 0.0) last = c;
    }
    if (total > 0.0 || mode == 0) break;
    mode = 0;
  }
  cluster.barrier_arrive();  // this CTA has read the others' sums; nobody leaves before all have
  if (!(total > 0.0)) {      // not one positive weight: no token can be drawn
    if (rank == 0 && tid == 0) a.tokens[row] = -1;
  } else if (warp == 0) {
    // The number falls into the first tile whose running sum exceeds it; where
    // rounding (or a number of 1) leaves none, the last tile with weight has it.
    // (before + s_sum is the next CTA's `before` to the bit, so one CTA goes on.)
    // A number below 0, or a NaN, counts as 0: no CTA's sums lie below 0.
    const double target = fmax(static_cast<double>(us) * total, 0.0);
    const bool chosen = total > target ? before + s_sum[mode] > target && !(before > target) : rank == last;
    if (chosen) {
      int at = -1;  // the tile, and the sum before it
      double run = before, at_run = before;
      for (int i = 0; i < tiles; i += 32) {
        const double s = i + lane < tiles ? s_tile[i + lane] : 0.0;
        const double inc = warp_scan(s);
        const unsigned over = __ballot_sync(0xffffffffu, s > 0.0 && run + inc > target);
        const unsigned some = __ballot_sync(0xffffffffu, s > 0.0);
        if (some != 0) {
          const int l = over != 0 ? __ffs(over) - 1 : 31 - __clz(some);
          at = i + l;
          at_run = run + __shfl_sync(0xffffffffu, inc - s, l);
        }
        if (over != 0) break;
        run += __shfl_sync(0xffffffffu, inc, 31);
      }
      if (at >= 0) {  // inside the tile: 8 consecutive tokens a lane
        const int x = x0 + at * kTile + lane * 8;
        Raw<T> rp, rq;
        rp.load(a.target, prow, x, a.V);
        if (q != nullptr) {
          rq.load(q, qrow, x, a.V);
        } else {
          rq.zero();
        }
        double w[8];
        const double s = weights(rp, rq, x, w);
        double sum = at_run + (warp_scan(s) - s);
        int first = -1, tail = -1;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          sum += w[i];
          if (w[i] > 0.0) {
            tail = x + i;
            if (first < 0 && sum > target) first = x + i;
          }
        }
        const unsigned over = __ballot_sync(0xffffffffu, first >= 0), some = __ballot_sync(0xffffffffu, tail >= 0);
        const int l = over != 0 ? __ffs(over) - 1 : 31 - __clz(some | 1u);
        const int tok = __shfl_sync(0xffffffffu, over != 0 ? first : tail, l);
        if (lane == 0) a.tokens[row] = tok;
      }
    }
  }
  cluster.barrier_wait();
}

}  // namespace

cudaError_t launch_verify_draft(const VerifyDraft& a, int type, cudaStream_t st) {
  auto k = type == 2 ? verify_draft_kernel<float> : type == 1 ? verify_draft_kernel<__nv_bfloat16> : verify_draft_kernel<__half>;
  // As many CTAs per sequence as keep the batch within about four per SM (one
  // wave), and no fewer than the tile table allows.
  int split = kMaxSplit;
  while (split > 1 && static_cast<int64_t>(a.B) * split > 4 * sm_count() &&
         a.V <= static_cast<int64_t>(kMaxTiles - 2) * kTile * (split / 2))
    split /= 2;
  return launch_paged(k, dim3(a.B * split), dim3(kThreads), 0, split, true, st, a);
}

}  // namespace persona
