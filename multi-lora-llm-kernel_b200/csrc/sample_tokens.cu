// The next token of every row of logits, drawn with a given number:
//
//   w_i = exp((x_i - max x) / T)
//   order: larger x first, equal ones by their index
//   kept by top-k: the first k of the order; by top-p: those whose weights
//   before them sum to at most p of top-k's whole sum; by min-p: w_i >= min_p
//   token = the first i, by index, whose running sum of kept weights exceeds u
//   times their whole sum
//
// Weights, sums and comparisons are in 64 bits: the draw, and the end of the
// nucleus, compare a sum over up to 2^21 tokens with a number that falls
// between two of them.
//
// Every condition but the draw keeps a beginning of the order, so a row is cut
// at one (value, index) pair: a 64-bit number `pair` whose high half orders the
// floats and whose low half is the index, counted down.  The pair is found by
// counts of tokens in 2048 classes, first by distance from the maximum (1/64
// of a power of two of weight each), then by pair: for top-k the class of the
// k-th token; for top-p the classes in which the sum can pass its mark, by the
// least and the largest weight that a class can have.  Once the tokens down to
// the cut (or those of its classes alone) fit into a list, that is sorted and
// the cut read off.  A list that holds all kept tokens also gives the draw;
// else a last pass sums the kept weights tile by tile.
#include <cooperative_groups.h>

#include "vocab_rows.cuh"

namespace persona {
namespace cg = cooperative_groups;
namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kTile = 256;      // elements of one tile: 8 a lane
constexpr int kMaxSplit = 8;    // CTAs (one cluster) per row
constexpr int kMaxTiles = 1040;
constexpr int kBins = 2048, kBinsEach = kBins / kThreads;
constexpr int kList = 2048;
static_assert(static_cast<int64_t>(kMaxTiles - 2) * kTile * kMaxSplit >= PERSONA_VERIFY_MAX_VOCAB, "tiles");

using u64 = unsigned long long;

// Orders floats as unsigned numbers (none of them NaN or -0).
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t u = __float_as_uint(x);
  return u ^ (static_cast<uint32_t>(static_cast<int32_t>(u) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}
__device__ __forceinline__ u64 pair_of(float x, int i) {
  return static_cast<u64>(key_of(x)) << 32 | (0xffffffffu - static_cast<uint32_t>(i));
}
__device__ __forceinline__ int index_of(u64 p) { return static_cast<int>(0xffffffffu - static_cast<uint32_t>(p)); }

struct Shared {
  union {
    uint32_t bins[kBins];
    double tile[kMaxTiles];
  };
  u64 list[kList];
  double wt[kList];
  double dsum[kWarps], part[2];
  u64 top[kWarps], best;
  int isum[kWarps], lo, hi, count, at;
};

template <typename T>
__global__ void __launch_bounds__(kThreads) sample_tokens_kernel(const __grid_constant__ SampleTokens a) {
  cg::cluster_group cluster = cg::this_cluster();
  __shared__ Shared sh;
  const int split = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
  const int b = blockIdx.x / split;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  pdl_wait();
  pdl_launch();
  const float temp = a.temperature != nullptr ? a.temperature[b] : 1.f;
  const int want_k = a.top_k != nullptr ? a.top_k[b] : 0;
  const float want_p = a.top_p != nullptr ? a.top_p[b] : 1.f, want_m = a.min_p != nullptr ? a.min_p[b] : 0.f;
  const int64_t row = static_cast<int64_t>(b) * a.ld;

  // Tiles start `lead` elements before the row, on a 16-byte boundary; a warp
  // has a run of this CTA's tiles.
  constexpr int kSize = sizeof(T) == 4 ? 4 : 2;
  const int lead =
      static_cast<int>(((reinterpret_cast<uintptr_t>(a.logits) + static_cast<uint64_t>(row) * kSize) & 15) / kSize);
  const int all = (a.V + lead + kTile - 1) / kTile, per = (all + split - 1) / split;
  const int t0 = min(all, rank * per), tiles = min(all, t0 + per) - t0;
  const int x0 = t0 * kTile - lead;
  const int w0 = tiles * warp / kWarps, w1 = tiles * (warp + 1) / kWarps;
  // fn(tile, index of the first, values): eight tokens a lane; what is no token
  // of the row, a NaN among them, is -infinity
  auto load = [&](int t, float (&f)[8]) {
    const int x = x0 + t * kTile + lane * 8;
    Raw<T> r;
    r.load(a.logits, row, x, a.V);
    r.values(f);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const bool real = x + i >= 0 && x + i < a.V && f[i] == f[i];
      f[i] = real ? f[i] + 0.f : -INFINITY;  // (-0 is 0)
    }
    return x;
  };
  auto each = [&](auto fn) {
    for (int t = w0; t < w1; ++t) {
      float f[8];
      const int x = load(t, f);
      fn(t, x, f);
    }
  };

  // ---- the largest ----
  u64 best = 0;
  each([&](int, int x, const float (&f)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const u64 p = f[i] > -INFINITY ? pair_of(f[i], x + i) : 0;
      best = p > best ? p : best;
    }
  });
  auto block_max = [&](u64 v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const u64 w = __shfl_xor_sync(0xffffffffu, v, o);
      v = w > v ? w : v;
    }
    if (lane == 0) sh.top[warp] = v;
    __syncthreads();
    v = sh.top[lane % kWarps];
#pragma unroll
    for (int o = kWarps / 2; o > 0; o >>= 1) {
      const u64 w = __shfl_xor_sync(0xffffffffu, v, o);
      v = w > v ? w : v;
    }
    return v;
  };
  best = block_max(best);
  if (tid == 0) sh.best = best;
  cluster.sync();
  for (int c = 0; c < split; ++c) {
    const u64 w = *cluster.map_shared_rank(&sh.best, c);
    best = w > best ? w : best;
  }
  // (the next cluster barrier comes before anybody leaves)
  const bool greedy = !(temp > 0.f);
  if (best == 0 || greedy) {
    if (rank == 0 && tid == 0) a.tokens[b] = best == 0 ? -1 : index_of(best);
    cluster.sync();
    return;
  }
  const float top = value_of(static_cast<uint32_t>(best >> 32));
  const double rate = 1.4426950408889634074 / static_cast<double>(temp);  // log2(e) / T
  // Weights relative to the largest, which has exactly 1.
  auto weight = [&](float x) {
    if (x == top) return 1.0;
    const double t = (static_cast<double>(x) - static_cast<double>(top)) * rate;
    return t > -1000.0 ? exp2(t) : 0.0;
  };
  const double min_w = want_m > 0.f ? fmin(static_cast<double>(want_m), 1.0) : 0.0;
  const double least = min_w > 0.0 ? min_w : 4.9406564584124654e-324;  // a weight of zero is never drawn
  const double u = static_cast<double>(a.u[b]);

  auto block_sum = [&](double v) {  // in the order of the warps
    v = warp_sum(v);
    __syncthreads();
    if (lane == 0) sh.dsum[warp] = v;
    __syncthreads();
    double s = 0.0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) s += sh.dsum[w];
    return s;
  };
  auto cluster_sum = [&](double v) {
    v = block_sum(v);
    if (split == 1) return v;
    cluster.sync();  // the one before has been read
    if (tid == 0) sh.part[0] = v;
    cluster.sync();
    v = 0.0;
    for (int c = 0; c < split; ++c) v += *cluster.map_shared_rank(&sh.part[0], c);
    return v;
  };
  // Sorts n <= kList entries, the largest first.
  auto sort = [&](int n) {
    int m = 1;
    while (m < n) m *= 2;
    for (int i = n + tid; i < m; i += kThreads) sh.list[i] = 0;
    __syncthreads();
    for (int k = 2; k <= m; k *= 2)
      for (int j = k / 2; j > 0; j /= 2) {
        for (int x = tid; x < m / 2; x += kThreads) {
          const int i = (x / j) * 2 * j + x % j;
          const u64 p = sh.list[i], q = sh.list[i + j];
          if ((p < q) == ((i & k) == 0)) {
            sh.list[i] = q;
            sh.list[i + j] = p;
          }
        }
        __syncthreads();
      }
  };
  // Running sums of wt[0 .. n) in place (every entry the sum up to and with it).
  auto running = [&](int n) {
    const int len = (n + kThreads - 1) / kThreads, i0 = min(n, tid * len), i1 = min(n, i0 + len);
    double s = 0.0;
    for (int i = i0; i < i1; ++i) s += sh.wt[i];
    const double inc = warp_scan(s);
    __syncthreads();
    if (lane == 31) sh.dsum[warp] = inc;
    __syncthreads();
    double run = inc - s;
    for (int w = 0; w < warp; ++w) run += sh.dsum[w];
    for (int i = i0; i < i1; ++i) {
      run += sh.wt[i];
      sh.wt[i] = run;
    }
    __syncthreads();
  };
  // How many of n entries are true, where the true ones come first.
  auto first_ones = [&](int n, auto test) {
    __syncthreads();
    if (tid == 0) sh.at = n;
    __syncthreads();
    for (int i = tid; i < n; i += kThreads)
      if (!test(i)) atomicMin(&sh.at, i);
    __syncthreads();
    return sh.at;
  };

  // ---- the cut: tokens of pair >= cut are kept ----
  u64 cut = 0;
  bool need_k = want_k > 0 && want_k < a.V, need_p = want_p < 1.f;
  double whole = 0.0;    // for top-p: the sum of what top-k keeps
  bool whole_known = false;
  const double p_of = fmax(static_cast<double>(want_p), 0.0);
  while (need_k || need_p) {
    const bool by_k = need_k;
    // Where the cut can lie: pairs [lo, hi].  `above`, `mass`: tokens and weight over it.
    u64 lo = cut, hi = best;
    bool linear = true, found = false;
    // classes by distance from the maximum: 1/64 of a power of two of weight
    const float inv_width = static_cast<float>(fmin(64.0 * rate, 1e30));
    for (int round = 0; !found; ++round) {
      int sh_bits = 0;
      while (((hi - lo) >> sh_bits) >= kBins) ++sh_bits;
      __syncthreads();
      for (int i = tid; i < kBins; i += kThreads) sh.bins[i] = 0;
      __syncthreads();
      double sum_all = 0.0, sum_above = 0.0;
      int over = 0;
      each([&](int, int x, const float (&f)[8]) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (!(f[i] > -INFINITY)) continue;
          const u64 p = pair_of(f[i], x + i);
          if (p < cut) continue;
          if (!by_k && !whole_known) sum_all += weight(f[i]);
          if (p > hi) {
            ++over;
            if (!by_k) sum_above += weight(f[i]);
          } else if (p >= lo) {
            int c;
            if (linear) {
              const float d = (top - f[i]) * inv_width;
              c = f[i] == top ? 0 : d < static_cast<float>(kBins - 1) ? static_cast<int>(d) : kBins - 1;
            } else {
              c = static_cast<int>((hi - p) >> sh_bits);
            }
            atomicAdd(&sh.bins[c], 1u);
          }
        }
      });
      if (!by_k && !whole_known) {
        whole = cluster_sum(sum_all);
        whole_known = true;
      }
      const double mass = by_k || linear ? 0.0 : cluster_sum(sum_above);
      const int above = linear ? 0 : static_cast<int>(cluster_sum(static_cast<double>(over)));
      cluster.sync();  // every CTA's counts are complete
      uint32_t cnt[kBinsEach];
#pragma unroll
      for (int i = 0; i < kBinsEach; ++i) cnt[i] = 0;
      for (int c = 0; c < split; ++c) {
        const uint32_t* from = cluster.map_shared_rank(&sh.bins[0], c) + tid * kBinsEach;
#pragma unroll
        for (int i = 0; i < kBinsEach; ++i) cnt[i] += from[i];
      }
      uint32_t mine = 0;
#pragma unroll
      for (int i = 0; i < kBinsEach; ++i) mine += cnt[i];
      // tokens before this thread's classes
      uint32_t inc = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t up = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += up;
      }
      if (lane == 31) sh.isum[warp] = static_cast<int>(inc);
      if (tid == 0) {
        sh.lo = kBins;
        sh.hi = kBins;
      }
      __syncthreads();
      uint32_t before = inc - mine;
      for (int w = 0; w < warp; ++w) before += sh.isum[w];
      uint32_t total = 0;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) total += sh.isum[w];
      // pairs of a class: (upper, lower)
      auto upper = [&](int c) -> u64 {
        if (!linear) return hi - (static_cast<u64>(c) << sh_bits);
        if (c == 0) return hi;
        // the classes' borders are known to a few roundings of the distance
        const double width = 1.0 / static_cast<double>(inv_width);
        const float x = __double2float_ru(static_cast<double>(top) - (c - 0.01) * width);
        const u64 p = static_cast<u64>(key_of(x + 0.f)) << 32 | 0xffffffffu;
        return p < hi ? p : hi;
      };
      auto lower = [&](int c) -> u64 {
        if (!linear) {
          const u64 span = (static_cast<u64>(c) + 1) << sh_bits;
          return span > hi - lo ? lo : hi - span + 1;
        }
        if (c == kBins - 1) return lo;
        const double width = 1.0 / static_cast<double>(inv_width);
        const double v = static_cast<double>(top) - (c + 1.01) * width;
        const float x = v > -3.4e38 ? __double2float_rd(v) : -3.4028234663852886e38f;
        const u64 p = static_cast<u64>(key_of(x + 0.f)) << 32;
        return p > lo ? p : lo;
      };
      int c_lo = kBins, c_hi = kBins;  // the classes that hold the cut
      if (by_k) {
        const uint32_t k = static_cast<uint32_t>(want_k - above);
        uint32_t run = before;
#pragma unroll
        for (int i = 0; i < kBinsEach; ++i) {
          if (c_lo == kBins && run < k && run + cnt[i] >= k) c_lo = c_hi = tid * kBinsEach + i;
          run += cnt[i];
        }
      } else {
        // sums of the largest and of the least weights that the classes can have
        double up = 0.0, dn = 0.0, w_up[kBinsEach], w_dn[kBinsEach];
#pragma unroll
        for (int i = 0; i < kBinsEach; ++i) {
          const int c = tid * kBinsEach + i;
          w_up[i] = w_dn[i] = 0.0;
          if (cnt[i] != 0) {
            w_up[i] = weight(value_of(static_cast<uint32_t>(upper(c) >> 32))) * cnt[i] * (1.0 + 1e-12);
            w_dn[i] = weight(value_of(static_cast<uint32_t>(lower(c) >> 32))) * cnt[i] * (1.0 - 1e-12);
          }
          up += w_up[i];
          dn += w_dn[i];
        }
        const double up_inc = warp_scan(up), dn_inc = warp_scan(dn);
        __syncthreads();
        if (lane == 31) {
          sh.dsum[warp] = up_inc;
          sh.wt[warp] = dn_inc;
        }
        __syncthreads();
        double run_up = mass * (1.0 + 1e-12) + (up_inc - up), run_dn = mass * (1.0 - 1e-12) + (dn_inc - dn);
        for (int w = 0; w < warp; ++w) {
          run_up += sh.dsum[w];
          run_dn += sh.wt[w];
        }
        const double mark = p_of * whole;
#pragma unroll
        for (int i = 0; i < kBinsEach; ++i) {
          run_up += w_up[i];
          run_dn += w_dn[i];
          if (cnt[i] == 0) continue;
          if (c_lo == kBins && run_up > mark * (1.0 - 1e-12)) c_lo = tid * kBinsEach + i;
          if (c_hi == kBins && run_dn > mark * (1.0 + 1e-12)) c_hi = tid * kBinsEach + i;
        }
      }
      if (c_lo < kBins) atomicMin(&sh.lo, c_lo);
      if (c_hi < kBins) atomicMin(&sh.hi, c_hi);
      __syncthreads();
      c_lo = sh.lo;
      c_hi = sh.hi;
      if (by_k && c_lo == kBins) {  // fewer tokens than k
        found = true;
        __syncthreads();
        cluster.sync();  // the counts have been read
        break;
      }
      // (no class where rounding leaves the sum below its mark: the cut lies behind all of them)
      if (c_lo == kBins) c_lo = kBins - 1;
      if (c_hi == kBins) c_hi = kBins - 1;
      // tokens down to the last of these classes, and in them
      if (tid == c_hi / kBinsEach) {
        uint32_t run = before;
        for (int i = 0; i <= c_hi % kBinsEach; ++i) run += cnt[i];
        sh.count = static_cast<int>(run);
      }
      if (tid == c_lo / kBinsEach) {
        uint32_t run = before;
        for (int i = 0; i < c_lo % kBinsEach; ++i) run += cnt[i];
        sh.at = static_cast<int>(run);
      }
      __syncthreads();
      const int down = sh.count, inside = down - sh.at;
      u64 nlo = lower(c_hi), nhi = upper(c_lo);
      __syncthreads();
      cluster.sync();  // the counts have been read
      const bool from_top = above + down <= kList;
      if (from_top || inside <= kList) {
        // ---- the list: all pairs down to nlo, or those of the classes alone ----
        const u64 ghi = from_top ? best : nhi;
        if (tid == 0) sh.count = 0;
        cluster.sync();
        int* const count = cluster.map_shared_rank(&sh.count, 0);
        u64* const list = cluster.map_shared_rank(&sh.list[0], 0);
        double heavy = 0.0;
        int over2 = 0;
        each([&](int, int x, const float (&f)[8]) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            if (!(f[i] > -INFINITY)) continue;
            const u64 p = pair_of(f[i], x + i);
            if (p > ghi) {
              ++over2;
              if (!by_k) heavy += weight(f[i]);
            } else if (p >= nlo && p >= cut) {
              const int at = atomicAdd(count, 1);
              if (at < kList) list[at] = p;
            }
          }
        });
        const double over_mass = by_k || from_top ? 0.0 : cluster_sum(heavy);
        const int over_count = from_top ? 0 : static_cast<int>(cluster_sum(static_cast<double>(over2)));
        cluster.sync();  // the list is complete
        const int n = *count;
        if (n <= kList) {
          if (rank == 0) {
            sort(n);
            if (from_top) {
              // all of it: top-k, top-p, min-p and the draw on the list
              int m = need_k ? min(n, want_k) : n;
              for (int i = tid; i < n; i += kThreads) sh.wt[i] = weight(value_of(static_cast<uint32_t>(sh.list[i] >> 32)));
              __syncthreads();
              const int by_min = min_w > 0.0 ? first_ones(m, [&](int i) { return sh.wt[i] >= least; }) : m;
              __syncthreads();
              running(m);
              if (need_p) {
                const double mark = p_of * (need_k ? sh.wt[m - 1] : whole);
                m = first_ones(m, [&](int i) { return i == 0 || sh.wt[i - 1] <= mark; });
              }
              m = min(m, by_min);
              // the kept ones by their index, with their place in the order
              __syncthreads();
              for (int i = tid; i < m; i += kThreads) {
                const u64 p = sh.list[i];
                sh.wt[i] = weight(value_of(static_cast<uint32_t>(p >> 32)));
                sh.list[i] = (p & 0xffffffffu) << 32 | static_cast<uint32_t>(i);
              }
              __syncthreads();
              sort(m);  // the largest low half, the smallest index, first
              double w[kList / kThreads];
#pragma unroll
              for (int i = 0; i < kList / kThreads; ++i) {
                const int x = tid + i * kThreads;
                w[i] = x < m ? sh.wt[static_cast<uint32_t>(sh.list[x])] : 0.0;
              }
              __syncthreads();
#pragma unroll
              for (int i = 0; i < kList / kThreads; ++i)
                if (tid + i * kThreads < m) sh.wt[tid + i * kThreads] = w[i];
              __syncthreads();
              running(m);
              const double target = fmax(u * sh.wt[m - 1], 0.0);
              const int at = first_ones(m, [&](int i) { return !(sh.wt[i] > target); });
              if (tid == 0)
                a.tokens[b] = static_cast<int>(0xffffffffu - static_cast<uint32_t>(sh.list[min(at, m - 1)] >> 32));
            } else if (by_k) {
              if (tid == 0) sh.best = sh.list[min(n, want_k - over_count) - 1];
            } else {
              for (int i = tid; i < n; i += kThreads) sh.wt[i] = weight(value_of(static_cast<uint32_t>(sh.list[i] >> 32)));
              __syncthreads();
              running(n);
              const double mark = p_of * whole;
              const int m = first_ones(n, [&](int i) { return over_mass + (i == 0 ? 0.0 : sh.wt[i - 1]) <= mark; });
              if (tid == 0) sh.best = m > 0 ? sh.list[m - 1] : ghi + 1;
            }
            __syncthreads();
          }
          cluster.sync();
          if (from_top) return;  // drawn
          cut = *cluster.map_shared_rank(&sh.best, 0);
          cluster.sync();
          found = true;
          break;
        }
      }
      nlo = nlo > cut ? nlo : cut;
      if (!by_k && !linear && nhi - nlo > (hi - lo) / 2) {
        // Classes so wide that their bounds say little (a tiny temperature): one
        // step by the exact sum over the middle, so that the range always shrinks.
        const u64 mid = nlo + (nhi - nlo) / 2;
        double s = 0.0;
        each([&](int, int x, const float (&f)[8]) {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (f[i] > -INFINITY && pair_of(f[i], x + i) > mid) s += weight(f[i]);
        });
        if (cluster_sum(s) > p_of * whole) {
          nlo = mid + 1;
        } else {
          nhi = mid;
        }
      }
      linear = false;
      lo = nlo;
      hi = nhi;
    }
    if (by_k) {
      need_k = false;
    } else {
      need_p = false;
    }
  }

  // ---- the draw over the kept tokens ----
  auto weight_of = [&](float x, int i) {
    if (!(x > -INFINITY) || pair_of(x, i) < cut) return 0.0;
    const double w = weight(x);
    return w >= least ? w : 0.0;
  };
  __syncthreads();
  double sum = 0.0;
  each([&](int t, int x, const float (&f)[8]) {
    double s = 0.0;
#pragma unroll
    for (int i = 0; i < 8; ++i) s += weight_of(f[i], x + i);
    s = warp_sum(s);
    if (lane == 0) sh.tile[t] = s;
    sum += s;
  });
  if (lane == 0) sh.dsum[warp] = sum;
  __syncthreads();
  if (tid == 0) {
    double s = 0.0;
    for (int w = 0; w < kWarps; ++w) s += sh.dsum[w];
    sh.part[1] = s;
  }
  cluster.sync();
  double total = 0.0, before = 0.0;
  int last = -1;
  for (int c = 0; c < split; ++c) {
    const double s = *cluster.map_shared_rank(&sh.part[1], c);
    if (c < rank) before += s;
    total += s;
    if (s > 0.0) last = c;
  }
  cluster.barrier_arrive();  // this CTA has read the others' sums; nobody leaves before all have
  if (warp == 0) {
    // as in verify_draft.cu: the first tile whose running sum exceeds the number, or
    // the last with weight where rounding leaves none
    const double target = fmax(u * total, 0.0);
    const bool chosen = total > target ? before + sh.part[1] > target && !(before > target) : rank == last;
    if (chosen) {
      int at = -1;
      double run = before, at_run = before;
      for (int i = 0; i < tiles; i += 32) {
        const double s = i + lane < tiles ? sh.tile[i + lane] : 0.0;
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
      if (at >= 0) {
        float f[8];
        const int x = load(at, f);
        double w[8], s = 0.0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          w[i] = weight_of(f[i], x + i);
          s += w[i];
        }
        double acc = at_run + (warp_scan(s) - s);
        int first = -1, tail = -1;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          acc += w[i];
          if (w[i] > 0.0) {
            tail = x + i;
            if (first < 0 && acc > target) first = x + i;
          }
        }
        const unsigned over = __ballot_sync(0xffffffffu, first >= 0), some = __ballot_sync(0xffffffffu, tail >= 0);
        const int l = over != 0 ? __ffs(over) - 1 : 31 - __clz(some | 1u);
        const int tok = __shfl_sync(0xffffffffu, over != 0 ? first : tail, l);
        if (lane == 0) a.tokens[b] = tok;
      }
    }
  }
  cluster.barrier_wait();
}

}  // namespace

cudaError_t launch_sample_tokens(const SampleTokens& a, int type, cudaStream_t st) {
  auto k = type == 2 ? sample_tokens_kernel<float> : type == 1 ? sample_tokens_kernel<__nv_bfloat16> : sample_tokens_kernel<__half>;
  int split = kMaxSplit;
  while (split > 1 && static_cast<int64_t>(a.B) * split > 4 * sm_count() &&
         a.V <= static_cast<int64_t>(kMaxTiles - 2) * kTile * (split / 2))
    split /= 2;
  return launch_paged(k, dim3(a.B * split), dim3(kThreads), 0, split, true, st, a);
}

}  // namespace persona
