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
// between two of them.  A weight below 2^-1000 counts as none: it changes no sum
// that holds the largest weight, 1, and would be drawn by a number of 0 alone.
//
// Every condition but the draw keeps a beginning of the order, so a row is cut
// at one (value, index) pair: a 64-bit number `pair` whose high half orders the
// floats and whose low half is the index, counted down.  The pair is found by
// counts of tokens in 2048 classes, first by distance from the maximum (1/64
// of a power of two of weight each), then by pair: for top-k the class of the
// k-th token; for top-p the classes in which the sum can pass its mark, by the
// least and the largest weight that a class can have.  The tokens of those
// classes are sorted and the cut read off.  Where all tokens down to it are
// few, the list is of them all and gives the draw too; else the kept weights
// are summed tile by tile, over copies of the tokens down to the cut where
// those fit into shared memory (a twentieth of a language model's row, say:
// weights of all tokens would cost as much again), else over the row.
// What it must read is the logits, once.  What bounds it is instructions: 25 to
// 30 a token and pass with a weight (ten of them in 64 bits), and for few rows
// the chain of passes, exchanges between the CTAs of a cluster, and the list.
// Measured, with inputs that change from call to call: 8 rows of 32000 tokens,
// fp16: 4.9 us greedy, 8.7 by temperature, 8.9 by min-p, 24 by top-k, 29 by top-p;
// 256 of 50257: 14 (0.28 of the measured HBM rate), 35, 36, 56 and 122 us, 104 with
// every row a rule of its own; 64 fp32 rows of 130001: 14 (0.36), 31, 32, 50, 105, 86.
#include <cooperative_groups.h>

#include <type_traits>

#include "vocab_rows.cuh"

namespace persona {
namespace cg = cooperative_groups;
namespace {

constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int kTile = 256;      // elements of one tile: 8 a lane
constexpr int kMaxSplit = 8;    // CTAs (one cluster) per row
constexpr int kMaxTiles = 1040;
constexpr int kBins = 1 << 11, kBinsEach = kBins / kThreads;
constexpr int kList = 1024;     // pairs that are sorted at most
constexpr int kWhole = 512;     // and of which the list is to hold all that are kept
static_assert(static_cast<int64_t>(kMaxTiles - 2) * kTile * kMaxSplit >= PERSONA_VERIFY_MAX_VOCAB, "tiles");
constexpr int kStepBits = 9, kSteps = 1 << kStepBits;  // of the table of powers, per power of two
constexpr int kPerClass = 8;   // steps of a class: 1/64 of a power of two
constexpr int kCopies = 320;     // tokens that a warp can copy
static_assert(kSteps == kThreads && kWarps >= 2 * (kMaxSplit - 1), "a thread makes one power, two warps fetch a list");
static_assert(kBinsEach == 4, "a thread reads its classes at once");

using u64 = unsigned long long;

// Orders floats as unsigned numbers (none of them NaN; -0 is below 0).
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t u = __float_as_uint(x);
  return u ^ (static_cast<uint32_t>(static_cast<int32_t>(u) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}
__device__ __forceinline__ u64 pair_of(float x, int i) {
  return static_cast<u64>(key_of(x + 0.f)) << 32 | (0xffffffffu - static_cast<uint32_t>(i));  // (-0 is 0)
}
__device__ __forceinline__ int index_of(u64 p) { return static_cast<int>(0xffffffffu - static_cast<uint32_t>(p)); }

// 2^t for t in [-1000, 0]: the power of two next to it, and the Taylor series
// of exp(f ln 2) for the rest, |f| <= 1/2, whose terms from the twelfth on are
// below 7e-15.
__device__ __forceinline__ double exp2_of(double t) {
  constexpr double kShift = 6755399441055744.0;  // 1.5 2^52: the integer next to t in the low bits
  const double m = t + kShift, f = (t - (m - kShift)) * 0.69314718055994530942;
  double p = 1.0 / 39916800;
  p = fma(p, f, 1.0 / 3628800);
  p = fma(p, f, 1.0 / 362880);
  p = fma(p, f, 1.0 / 40320);
  p = fma(p, f, 1.0 / 5040);
  p = fma(p, f, 1.0 / 720);
  p = fma(p, f, 1.0 / 120);
  p = fma(p, f, 1.0 / 24);
  p = fma(p, f, 1.0 / 6);
  p = fma(p, f, 0.5);
  p = fma(p, f, 1.0);
  p = fma(p, f, 1.0);
  return __hiloint2double(__double2hiint(p) + (__double2loint(m) << 20), __double2loint(p));
}

// A row as a CTA reads it: tiles start `lead` elements before the row, on a
// 16-byte boundary; a warp has a run of the CTA's tiles.
struct Row {
  const void* logits;
  int64_t at;  // element of the row's first logit
  int V, x0, w0, w1;  // w0, w1: the warp's tiles
  bool inf;    // a logit is +infinity: those that are count as 0, all others as none
  float top, least;  // the largest; the last one whose weight is a normal number
  double rate, unit;  // log2(e) / T, and one over it
};

struct Shared {
  double power[kSteps];  // 2^(-i / kSteps)
  union {
    alignas(16) uint32_t bins[kBins];
    double tile[kMaxTiles];
  };
  alignas(16) uint32_t slice[kBins / 2];  // this CTA's classes, over the cluster
  alignas(16) u64 list[kList];   // this CTA's pairs; in the first CTA then all
  alignas(16) u64 sorted[kList];
  double wt[kList];
  double dsum[kWarps], part;
  u64 best, cut;
  u64 copy[kWarps][kCopies];     // values and indexes, tile by tile
  uint16_t copied[kMaxTiles];    // and how many of the warp's up to and with a tile
  Row row[kWarps];
  float fmax[kWarps], top;
  int isum[kWarps], copies[kWarps], lo, hi, count, at, over, down, from;
};

// (Every function finds it for itself: through a reference its atomics would
// be those of any memory, several times as slow.)
__device__ __forceinline__ Shared& shared() {
  extern __shared__ __align__(16) uint8_t smem[];
  return *reinterpret_cast<Shared*>(smem);
}

// Weights of four logits relative to the largest, which has exactly 1, and how
// far below it they are in steps of the table (n): 2^t is a power of the table,
// a power of two and 1 + r (..), the Taylor series of 2^r to the third power,
// |r| <= 1/1024 (the rest is below 9e-15).  Not for logits below r.least.
// Four at once, since each is a chain of ten 64-bit operations.
__device__ __forceinline__ void steps4(const Row& r, const float* f, double (&t)[4], double (&m)[4], int (&n)[4]) {
  constexpr double kShift = 6755399441055744.0;  // 1.5 2^52: integers in the low bits
#pragma unroll
  for (int i = 0; i < 4; ++i) t[i] = (static_cast<double>(f[i]) - static_cast<double>(r.top)) * r.rate;
#pragma unroll
  for (int i = 0; i < 4; ++i) m[i] = fma(t[i], -static_cast<double>(kSteps), kShift);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    n[i] = __double2loint(m[i]);
    m[i] -= kShift;
  }
}
__device__ __forceinline__ void weights4(const Row& r, const double* power, const float* f, double (&w)[4], int (&n)[4]) {
  constexpr double kLn2 = 0.69314718055994530942;
  double t[4], m[4], p[4];
  steps4(r, f, t, m, n);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    p[i] = power[n[i] & (kSteps - 1)];
    t[i] = fma(m[i], 1.0 / kSteps, t[i]);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) m[i] = fma(t[i], kLn2 * kLn2 * kLn2 / 6, kLn2 * kLn2 / 2);
#pragma unroll
  for (int i = 0; i < 4; ++i) m[i] = fma(t[i], m[i], kLn2);
#pragma unroll
  for (int i = 0; i < 4; ++i) m[i] = m[i] * t[i];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const double v = fma(p[i], m[i], p[i]);
    w[i] = __hiloint2double(__double2hiint(v) - ((n[i] >> kStepBits) << 20), __double2loint(v));
  }
}
// One weight by itself.
__device__ __forceinline__ double weight(const Row& r, const double* power, float x) {
  constexpr double kShift = 6755399441055744.0, kLn2 = 0.69314718055994530942;
  const double t = (static_cast<double>(x) - static_cast<double>(r.top)) * r.rate;
  const double m = fma(t, -static_cast<double>(kSteps), kShift);
  const int n = __double2loint(m);
  const double p = power[n & (kSteps - 1)], f = fma(m - kShift, 1.0 / kSteps, t);
  const double v = fma(p, fma(f, fma(f, kLn2 * kLn2 * kLn2 / 6, kLn2 * kLn2 / 2), kLn2) * f, p);
  return x >= r.least ? __hiloint2double(__double2hiint(v) - ((n >> kStepBits) << 20), __double2loint(v)) : 0.0;
}

// fn(tile, index of the first, values) for the eight tokens a lane has of each
// of the warp's tiles, two tiles' loads under way at once.  What is no token of
// the row is -infinity; a NaN stays one, which no comparison lets through.
template <typename T, typename F> __device__ __forceinline__ void each(const Row& r, F fn) {
  for (int t = r.w0; t < r.w1; t += 2) {
    const int x0 = r.x0 + t * kTile + (threadIdx.x & 31) * 8;
    Raw<T> raw[2];
    raw[0].load(r.logits, r.at, x0, r.V);
    raw[1].load(r.logits, r.at, t + 1 < r.w1 ? x0 + kTile : r.V, r.V);
#pragma unroll 1
    for (int k = 0; k < 2; ++k) {
      if (t + k >= r.w1) break;
      const int x = x0 + k * kTile;
      float f[8];
      raw[0].values(f);
      if (__any_sync(0xffffffffu, r.inf || x < 0 || x + 8 > r.V)) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (!(x + i >= 0 && x + i < r.V)) f[i] = -INFINITY;
          if (r.inf) f[i] = f[i] == INFINITY ? 0.f : -INFINITY;
        }
      }
      fn(t + k, x, f);
      raw[0] = raw[1];
    }
  }
}

// The largest of a lane's eight (a NaN is none of them).
template <typename T> __device__ __forceinline__ float largest(const Raw<T>& raw) {
  if constexpr (sizeof(T) == 4) {
    float f[8];
    raw.values(f);
    return fmaxf(fmaxf(fmaxf(f[0], f[1]), fmaxf(f[2], f[3])), fmaxf(fmaxf(f[4], f[5]), fmaxf(f[6], f[7])));
  } else {
    using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
    const T2* h = reinterpret_cast<const T2*>(raw.u);
    const T2 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
    const float2 f = Cvt<T>::to2(*reinterpret_cast<const uint32_t*>(&m));
    return fmaxf(f.x, f.y);
  }
}

template <typename T> __device__ __forceinline__ float value_at(const Row& r, int i) {
  if constexpr (sizeof(T) == 4) {
    return __ldg(static_cast<const float*>(r.logits) + r.at + i);
  } else {
    return Cvt<T>::to1(__ldg(static_cast<const uint16_t*>(r.logits) + r.at + i));
  }
}

// A comparison with a pair, most of it with its value.
struct Border {
  float x;
  unsigned at;
  __device__ __forceinline__ explicit Border(u64 p)
      : x(value_of(static_cast<uint32_t>(p >> 32))), at(0xffffffffu - static_cast<uint32_t>(p)) {
    const uint32_t key = static_cast<uint32_t>(p >> 32);
    if (key >= 0xff800000u) x = INFINITY;                                  // above all tokens
    if (key < 0x00800000u) x = -3.4028234663852886e38f, at = 0xffffffffu;  // below them
    if (key == 0x7fffffffu) x = 0.f, at = 0xffffffffu;                     // (that of -0, which no token has)
  }
  // whether the pair of (f, i) is at least this one (never for -infinity)
  __device__ __forceinline__ bool upto(float f, int i) const { return f >= x && (f > x || static_cast<unsigned>(i) <= at); }
};

// ---- passes over the row; their sums are the warp's ----
// Counts tokens of pair >= lo by distance from the maximum, those of the last
// class in `tail` (many there may be, and they would queue for one word), and
// sums their weights.
template <typename T, bool kWeighed>
__device__ __noinline__ void count_pass(u64 lo_pair, double& sum_out, int& tail_out) {
  Shared& sh = shared();
  const Row r = sh.row[threadIdx.x >> 5];
  const Border lo(lo_pair);
  const bool ties = lo.at < static_cast<unsigned>(r.V);
  // What is further than 2046.9 classes from the maximum is in the last one.  Steps are
  // rounded, so class 2046 by them ends at 2046.94; the last class has its upper border
  // at 2046.85 (upper) and its largest weight at 2046.875 (by_mass), both above these tokens.
  const float least = fmaxf(r.least, __double2float_ru(static_cast<double>(r.top) - (kBins - 1.1) * kPerClass / kSteps * r.unit));
  const uint32_t bins = smem_u32(sh.bins);
  double sum = 0.0;
  int tail = 0;
  each<T>(r, [&](int, int x, const float (&f)[8]) {
#pragma unroll
    for (int h = 0; h < 8; h += 4) {
      double t[4], w[4];
      int n[4];
      if (kWeighed) {
        weights4(r, sh.power, f + h, w, n);
      } else {
        steps4(r, f + h, t, w, n);
      }
      bool in[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) in[j] = f[h + j] >= lo.x;
      if (ties) {
#pragma unroll
        for (int j = 0; j < 4; ++j) in[j] = lo.upto(f[h + j], x + h + j);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float v = in[j] ? f[h + j] : -INFINITY;
        if (kWeighed && v >= r.least) sum += w[j];
        // (a predicated instruction: a branch for each costs more than the count)
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ge.f32 p, %0, %1;\n\t@p red.shared.add.u32 [%2], 1;\n\t}" ::"f"(v), "f"(least),
                     "r"(bins + 4u * (static_cast<unsigned>(n[j]) / kPerClass))
                     : "memory");
        tail += in[j] && v < least ? 1 : 0;
      }
    }
  });
  sum_out = warp_sum(sum);
  tail_out = __reduce_add_sync(0xffffffffu, tail);
}
// Sums of weights of tokens of pair >= heavy and logit >= least, tile by tile.
template <typename T>
__device__ __noinline__ void draw_pass(u64 heavy, float least, double& sum_out) {
  Shared& sh = shared();
  const Row r = sh.row[threadIdx.x >> 5];
  const Border lo(heavy);
  const bool ties = lo.at < static_cast<unsigned>(r.V);
  const float end = fmaxf(fmaxf(least, r.least), lo.x);
  const int lane = threadIdx.x & 31;
  double sum = 0.0;
  each<T>(r, [&](int t, int x, const float (&f)[8]) {
    double s = 0.0;
#pragma unroll
    for (int h = 0; h < 8; h += 4) {
      double w[4];
      int n[4];
      weights4(r, sh.power, f + h, w, n);
      bool in[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) in[j] = f[h + j] >= end;
      if (ties) {
#pragma unroll
        for (int j = 0; j < 4; ++j) in[j] = in[j] && lo.upto(f[h + j], x + h + j);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (in[j]) s += w[j];
    }
    s = warp_sum(s);
    if (lane == 0) sh.tile[t] = s;
    sum += s;
  });
  sum_out = sum;
}
// Copies tokens of pair >= lo, tile by tile in a fixed order; how many the warp
// has (none copied behind its kCopies).
template <typename T> __device__ __noinline__ int copy_pass(u64 lo_pair) {
  Shared& sh = shared();
  const Row r = sh.row[threadIdx.x >> 5];
  const Border lo(lo_pair);
  const bool ties = lo.at < static_cast<unsigned>(r.V);
  const int lane = threadIdx.x & 31;
  u64* const to = sh.copy[threadIdx.x >> 5];
  int n = 0;
  each<T>(r, [&](int t, int x, const float (&f)[8]) {
    // lane after lane, each lane's in the order of the row
    unsigned mine = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) mine |= f[i] >= lo.x ? 1u << i : 0u;
    if (ties) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (!lo.upto(f[i], x + i)) mine &= ~(1u << i);
    }
    int inc = __popc(mine);
    const int own = inc;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += up;
    }
    int at = n + inc - own;
    for (; mine != 0; mine &= mine - 1, ++at) {  // two or three rounds; the values once more, out of the caches
      const int i = x + __ffs(mine) - 1;
      if (at < kCopies) to[at] = static_cast<u64>(__float_as_uint(r.inf ? 0.f : value_at<T>(r, i))) << 32 | static_cast<uint32_t>(i);
    }
    n += __shfl_sync(0xffffffffu, inc, 31);
    if (lane == 0) sh.copied[t] = static_cast<uint16_t>(min(n, kCopies));
  });
  return n;
}
// Of the warp's copies: counts those of pair > hi and, if weighed, sums their
// weights; lists the others.
__device__ __noinline__ void split_copies(u64 hi, bool weighed, int n, double& sum_out, int& over_out) {
  Shared& sh = shared();
  const Row r = sh.row[threadIdx.x >> 5];
  const u64* const from = sh.copy[threadIdx.x >> 5];
  double sum = 0.0;
  int over = 0;
  for (int i = threadIdx.x & 31; i < n; i += 32) {
    const float x = __uint_as_float(static_cast<uint32_t>(from[i] >> 32));
    const u64 p = pair_of(x, static_cast<int>(from[i]));
    if (p > hi) {
      ++over;
      if (weighed) sum += weight(r, sh.power, x);
    } else {
      const int at = atomicAdd(&sh.count, 1);
      if (at < kList) sh.list[at] = p;
    }
  }
  sum_out = warp_sum(sum);
  over_out = __reduce_add_sync(0xffffffffu, over);
}
// draw_pass over the copies.
__device__ __noinline__ void draw_copies(u64 heavy, float least, double& sum_out) {
  Shared& sh = shared();
  const Row r = sh.row[threadIdx.x >> 5];
  const Border lo(heavy);
  const int lane = threadIdx.x & 31;
  const u64* const from = sh.copy[threadIdx.x >> 5];
  double sum = 0.0;
  for (int t = r.w0, i0 = 0; t < r.w1; ++t) {
    const int i1 = sh.copied[t];
    double s = 0.0;
    for (int i = i0 + lane; i < i1; i += 32) {
      const float x = __uint_as_float(static_cast<uint32_t>(from[i] >> 32));
      if (x >= least && lo.upto(x, static_cast<int>(from[i]))) s += weight(r, sh.power, x);
    }
    i0 = i1;
    s = warp_sum(s);
    if (lane == 0) sh.tile[t] = s;
    sum += s;
  }
  sum_out = sum;
}
// What else there is, seldom or for small lists: counts tokens of pair > hi and
// sums their weights if weighed; counts those in [lo, hi] by pair, or lists them.
template <typename T>
__device__ __noinline__ void pair_pass(u64 lo_pair, u64 hi, bool weighed, bool append, int bits,
                                       double& sum_out, int& over_out) {
  Shared& sh = shared();
  const Row r = sh.row[threadIdx.x >> 5];
  const Border lo(lo_pair), above(hi + 1 != 0 ? hi + 1 : hi);
  double sum = 0.0;
  int over = 0;
  each<T>(r, [&](int, int x, const float (&f)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (!(f[i] >= lo.x) || !lo.upto(f[i], x + i)) continue;
      if (above.upto(f[i], x + i)) {
        ++over;
        if (weighed) sum += weight(r, sh.power, f[i]);
      } else if (append) {
        const int at = atomicAdd(&sh.count, 1);
        if (at < kList) sh.list[at] = pair_of(f[i], x + i);
      } else {
        atomicAdd(&sh.bins[static_cast<int>((hi - pair_of(f[i], x + i)) >> bits)], 1u);
      }
    }
  });
  sum_out = warp_sum(sum);
  over_out = __reduce_add_sync(0xffffffffu, over);
}

// Sorts n <= kList pairs, the largest first, from list to sorted.  Few by
// counting the larger ones of each (no two are equal), many by a network.
__device__ __noinline__ void sort_list(int n) {
  Shared& sh = shared();
  u64 *const list = sh.list, *const sorted = sh.sorted;
  const int tid = threadIdx.x;
  if (n <= kThreads) {
    // as many threads an element as there are, each for a part of the others
    int* const rank = reinterpret_cast<int*>(sh.wt);
    const int share = n <= 64 ? 8 : n <= 128 ? 4 : n <= 256 ? 2 : 1, own = kThreads / share;
    if (tid < n) rank[tid] = 0;
    if (tid == 0 && (n & 1)) list[n] = 0;  // (n < kList)
    __syncthreads();
    const int e = tid % own, part = tid / own, pairs = (n + 1) / 2;
    const u64 p = e < n ? list[e] : 0;
    if (e < n) {
      int larger = 0;
#pragma unroll 4
      for (int j = pairs * part / share; j < pairs * (part + 1) / share; ++j) {
        const ulonglong2 q = *reinterpret_cast<const ulonglong2*>(list + 2 * j);
        larger += (q.x > p ? 1 : 0) + (q.y > p ? 1 : 0);
      }
      if (share == 1) {
        rank[e] = larger;
      } else {
        atomicAdd(&rank[e], larger);
      }
    }
    __syncthreads();
    if (tid < n) sorted[rank[tid]] = p;
    __syncthreads();
    return;
  }
  int m = 1;
  while (m < n) m *= 2;
  for (int i = tid; i < m; i += kThreads) sorted[i] = i < n ? list[i] : 0;
  __syncthreads();
  for (int k = 2; k <= m; k *= 2)
    for (int j = k / 2; j > 0; j /= 2) {
      for (int x = tid; x < m / 2; x += kThreads) {
        const int i = 2 * x - (x & (j - 1));
        const u64 p = sorted[i], q = sorted[i + j];
        if ((p < q) == ((i & k) == 0)) {
          sorted[i] = q;
          sorted[i + j] = p;
        }
      }
      if (j > 32) {
        __syncthreads();
      } else {  // pairs of 64 neighbours stay with a warp
        __syncwarp();
        if (j == 1) __syncthreads();
      }
    }
}
// Sum over the lanes up to and with this one.
template <typename F> __device__ __forceinline__ F scan_lanes(F v) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const F up = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += up;
  }
  return v;
}
// Running sums of wt[0 .. n) in place (every entry the sum up to and with it).
__device__ __noinline__ void running_sums(int n) {
  Shared& sh = shared();
  double *const wt = sh.wt, *const warps = sh.dsum;
  const int tid = threadIdx.x, warp = tid >> 5;
  const int len = (n + kThreads - 1) / kThreads, i0 = min(n, tid * len), i1 = min(n, i0 + len);
  double s = 0.0;
  for (int i = i0; i < i1; ++i) s += wt[i];
  const double inc = warp_scan(s);
  if ((tid & 31) == 31) warps[warp] = inc;
  __syncthreads();
  const double to = warp_scan((tid & 31) < kWarps ? warps[tid & 31] : 0.0);
  double run = inc - s + (warp > 0 ? __shfl_sync(0xffffffffu, to, max(warp - 1, 0)) : 0.0);
  for (int i = i0; i < i1; ++i) {
    run += wt[i];
    wt[i] = run;
  }
  __syncthreads();
}
// The weights of n sorted pairs whose value is in the bits from `shift` on.
__device__ __noinline__ void list_weights(int n, int shift) {
  Shared& sh = shared();
  const Row r = sh.row[threadIdx.x >> 5];
  for (int i = threadIdx.x; i < n; i += kThreads) sh.wt[i] = weight(r, sh.power, value_of(static_cast<uint32_t>(sh.sorted[i] >> shift)));
  __syncthreads();
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 2) sample_tokens_kernel(const __grid_constant__ SampleTokens a) {
  cg::cluster_group cluster = cg::this_cluster();
  Shared& sh = shared();
  const int split = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
  const int b = blockIdx.x / split;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  sh.power[tid] = exp2_of(static_cast<double>(tid) * (-1.0 / kSteps));
  for (int i = tid; i < kBins; i += kThreads) sh.bins[i] = 0;
  for (int i = tid; i < kBins / 2; i += kThreads) sh.slice[i] = 0;
  if (tid == 0) sh.count = 0;
  pdl_wait();
  pdl_launch();
  const float temp = a.temperature != nullptr ? a.temperature[b] : 1.f;
  const int want_k = a.top_k != nullptr ? a.top_k[b] : 0;
  const float want_p = a.top_p != nullptr ? a.top_p[b] : 1.f, want_m = a.min_p != nullptr ? a.min_p[b] : 0.f;
  const double u = static_cast<double>(a.u[b]);
  const int64_t row = static_cast<int64_t>(b) * a.ld;

  constexpr int kSize = sizeof(T) == 4 ? 4 : 2;
  const int lead =
      static_cast<int>(((reinterpret_cast<uintptr_t>(a.logits) + static_cast<uint64_t>(row) * kSize) & 15) / kSize);
  const int all = (a.V + lead + kTile - 1) / kTile, per = (all + split - 1) / split;
  const int t0 = min(all, rank * per), tiles = min(all, t0 + per) - t0;
  Row r{a.logits, row, a.V, t0 * kTile - lead, tiles * warp / kWarps, tiles * (warp + 1) / kWarps, false, 0.f, 0.f, 0.0, 0.0};
  auto barrier = [&] {
    if (split > 1) {
      cluster.sync();
    } else {
      __syncthreads();
    }
  };
  // fn of every CTA's number at p (lane c has CTA c's; lanes from split on `none`)
  auto of_all = [&](auto* p, auto none) { return lane < split ? *cluster.map_shared_rank(p, lane) : none; };

  // ---- the largest ----
  float top = -INFINITY;
  for (int t = r.w0; t < r.w1; t += 2) {
    const int x = r.x0 + t * kTile + lane * 8;
    Raw<T> raw[2];
    raw[0].load(r.logits, r.at, x, r.V);
    raw[1].load(r.logits, r.at, t + 1 < r.w1 ? x + kTile : r.V, r.V);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int xi = i == 0 || t + 1 < r.w1 ? x + i * kTile : r.V;
      if (xi >= 0 && xi + 8 <= r.V) {
        top = fmaxf(top, largest<T>(raw[i]));
      } else {
        float f[8];
        raw[i].values(f);
#pragma unroll
        for (int z = 0; z < 8; ++z)
          if (xi + z >= 0 && xi + z < r.V) top = fmaxf(top, f[z]);
      }
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (lane == 0) sh.fmax[warp] = top;
  __syncthreads();
  top = sh.fmax[lane % kWarps];
#pragma unroll
  for (int o = kWarps / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (split > 1) {
    if (tid == 0) sh.top = top;
    cluster.sync();
    top = of_all(&sh.top, -INFINITY);
#pragma unroll
    for (int o = kMaxSplit / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    top = __shfl_sync(0xffffffffu, top, 0);
  }
  r.inf = top == INFINITY;
  top = r.inf ? 0.f : top + 0.f;
  if (top == -INFINITY || !(temp > 0.f)) {
    // the first index of the largest logit
    unsigned at = 0xffffffffu;
    if (top > -INFINITY)
      each<T>(r, [&](int, int x, const float (&f)[8]) {
#pragma unroll
        for (int i = 7; i >= 0; --i)  // (0 is -0 here)
          if (f[i] == top) at = min(at, static_cast<unsigned>(x + i));
      });
    at = __reduce_min_sync(0xffffffffu, at);
    if (lane == 0) sh.isum[warp] = static_cast<int>(at);
    __syncthreads();
    at = __reduce_min_sync(0xffffffffu, static_cast<unsigned>(sh.isum[lane % kWarps]));
    if (tid == 0) sh.at = static_cast<int>(at);
    barrier();
    if (rank == 0 && warp == 0) {
      at = __reduce_min_sync(0xffffffffu, static_cast<unsigned>(of_all(&sh.at, -1)));
      if (lane == 0) a.tokens[b] = static_cast<int>(at);
    }
    barrier();  // nobody leaves before all have read
    return;
  }
  const double top64 = top, rate = 1.4426950408889634074 / static_cast<double>(temp);  // log2(e) / T
  r.top = top;
  r.rate = rate;
  const double unit = static_cast<double>(temp) * 0.69314718055994530942;  // logits to half the weight: 1 / rate
  r.least = fmaxf(__double2float_ru(top64 - 1000.0 * unit), -3.4028234663852886e38f);
  r.unit = unit;
  // (field by field: nvcc 12.9 leaves a copy of the whole unset, since the functions
  // above capture r)
  if (lane == 0) {
    Row& to = sh.row[warp];
    to.logits = r.logits;
    to.at = r.at;
    to.V = r.V;
    to.x0 = r.x0;
    to.w0 = r.w0;
    to.w1 = r.w1;
    to.inf = r.inf;
    to.top = top;
    to.least = r.least;
    to.rate = rate;
    to.unit = unit;
  }
  __syncwarp();
  const u64 best = static_cast<u64>(key_of(top)) << 32 | 0xffffffffu;  // no pair is larger
  // min-p as the smallest logit whose weight suffices: a search over the floats,
  // as many at once as there are threads.
  float x_min = -3.4028234663852886e38f;
  if (want_m > 0.f) {
    const double min_w = fmin(static_cast<double>(want_m), 1.0);
    u64 lo = 0, hi = key_of(top);  // in keys: too light, heavy enough
    {
      const double about = top64 + log2(min_w) * unit, off = (fabs(about) + fabs(top64)) * 1e-6 + 1e-6 * unit;
      const float x0 = __double2float_rd(about - off), x1 = __double2float_ru(about + off);
      if (x0 > -3.4e38f && x0 < top) lo = key_of(x0 + 0.f);
      if (x1 < top) hi = key_of(x1 + 0.f);
    }
    while (hi - lo > 1) {
      const u64 step = (hi - lo + kThreads - 1) / kThreads, k = lo + step * tid;
      const float x = value_of(static_cast<uint32_t>(k));
      // (the first thread's is too light by itself, keys from hi on are heavy enough)
      const bool light = tid == 0 || (k < hi && !(x >= r.least && weight(r, sh.power, x + 0.f) >= min_w));
      const int n = __syncthreads_count(light);
      hi = n < kThreads ? min(hi, lo + step * n) : hi;
      lo += step * (n - 1);
    }
    x_min = fmaxf(x_min, value_of(static_cast<uint32_t>(hi)));
  }

  // The warps' sums of a pass: over the CTA in part, over and tail, for all to
  // read after the barrier.
  auto publish = [&](double sum, int over, int tail) {
    if (lane == 0) {
      sh.dsum[warp] = sum;
      sh.isum[warp] = over;
      if (tail != 0) atomicAdd(&sh.bins[kBins - 1], static_cast<uint32_t>(tail));
    }
    __syncthreads();
    if (warp == 0) {
      const double s = warp_sum(lane < kWarps ? sh.dsum[lane] : 0.0);
      const int n = __reduce_add_sync(0xffffffffu, lane < kWarps ? sh.isum[lane] : 0);
      if (lane == 0) {
        sh.part = s;
        sh.over = n;
        sh.lo = sh.hi = kBins;
      }
    }
  };
  // Sums over the CTAs, the same bits in all of them.
  auto all_parts = [&] { return warp_sum(of_all(&sh.part, 0.0)); };
  auto all_of = [&](int* p) { return __reduce_add_sync(0xffffffffu, of_all(p, 0)); };
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
  int copies = -1;      // tokens that this warp has copied,
  bool copied = false;  // and whether those of the CTA are all down to the cut
  bool need_k = want_k > 0 && want_k < a.V, need_p = want_p < 1.f;
  double whole = 0.0;  // for top-p: the sum of what top-k keeps
  const double p_of = fmax(static_cast<double>(want_p), 0.0);
  while (need_k || need_p) {
    const bool by_k = need_k;
    u64 lo = cut != 0 ? cut : 1, hi = best;  // where the cut can lie (0 is no token)
    bool linear = true;
    const double width = static_cast<double>(kPerClass) / kSteps * unit;  // of a linear class, in logits
    while (true) {
      const int bits = max(0, 64 - __clzll(static_cast<long long>(hi - lo)) - 11);  // (hi - lo) >> bits < 2^11

      // ---- counts of the classes; tokens and weight above them ----
      {
        double sum = 0.0;
        int over = 0, tail = 0;
        if (!linear) {
          pair_pass<T>(lo, hi, !by_k, false, bits, sum, over);
        } else if (by_k) {
          count_pass<T, false>(lo, sum, tail);
        } else {
          count_pass<T, true>(lo, sum, tail);
        }
        publish(sum, over, tail);
      }
      barrier();
      // Every CTA adds up a slice of the classes over the cluster and hands it on
      // (all of them by every CTA would be eight times the traffic).
      const int quads = kThreads / split;
      if (split > 1) {
        const uint4 v = reinterpret_cast<const uint4*>(cluster.map_shared_rank(&sh.bins[0], tid / quads))[rank * quads + tid % quads];
        uint32_t* const to = sh.slice + 4 * (tid % quads);
        if (v.x) atomicAdd(to, v.x);
        if (v.y) atomicAdd(to + 1, v.y);
        if (v.z) atomicAdd(to + 2, v.z);
        if (v.w) atomicAdd(to + 3, v.w);
        cluster.sync();
      }
      const uint4 got = reinterpret_cast<const uint4*>(split > 1 ? cluster.map_shared_rank(&sh.slice[0], tid / quads)
                                                                 : &sh.bins[0])[tid % quads];
      const uint32_t cnt[kBinsEach] = {got.x, got.y, got.z, got.w};
      double mass = all_parts();
      const int above = all_of(&sh.over);
      if (linear && !by_k) {
        whole = mass;
        mass = 0.0;
      }
      const uint32_t mine = (cnt[0] + cnt[1]) + (cnt[2] + cnt[3]);
      uint32_t inc = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t n = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += n;
      }
      barrier();  // the counts have been read
      if (lane == 31) sh.isum[warp] = static_cast<int>(inc);
      for (int i = tid; i < kBins; i += kThreads) sh.bins[i] = 0;  // for the next time
      for (int i = tid; i < kBins / 2; i += kThreads) sh.slice[i] = 0;
      // Pairs of a class, largest and least.  The linear ones end half a step off
      // their distances; a little more allows for roundings.
      const int end_class = linear ? kBins - 1 : static_cast<int>((hi - lo) >> bits);
      auto upper = [&](int c) -> u64 {
        if (!linear) return hi - (static_cast<u64>(c) << bits);
        if (c == 0) return hi;
        const u64 p = static_cast<u64>(key_of(__double2float_ru(top64 - (c - 0.15) * width) + 0.f)) << 32 | 0xffffffffu;
        return p < hi ? p : hi;
      };
      auto lower = [&](int c) -> u64 {
        if (!linear) return c >= end_class ? lo : hi - ((static_cast<u64>(c) + 1) << bits) + 1;
        if (c == kBins - 1) return lo;
        const double v = top64 - (c + 1.0) * width;
        const u64 p = static_cast<u64>(key_of((v > -3.4e38 ? __double2float_rd(v) : -3.4028234663852886e38f) + 0.f)) << 32;
        return p > lo ? p : lo;
      };
      // ---- the classes that hold the cut ----
      const double mark = p_of * whole;
      __syncthreads();
      const int to_warp = scan_lanes(lane < kWarps ? sh.isum[lane] : 0);
      const uint32_t before = inc - mine + (warp > 0 ? __shfl_sync(0xffffffffu, to_warp, max(warp - 1, 0)) : 0);
      int c_lo = kBins, c_hi = kBins;
      if (by_k) {
        const uint32_t k = static_cast<uint32_t>(want_k - above);
        uint32_t run = before;
#pragma unroll
        for (int i = 0; i < kBinsEach; ++i) {
          if (run < k && run + cnt[i] >= k) c_lo = c_hi = tid * kBinsEach + i;
          run += cnt[i];
        }
      } else {
        // sums of the largest and of the least weights that the classes can have
        const auto by_mass = [&](auto zero, auto slack, auto bounds) {
          using F = decltype(zero);
          F up = 0, dn = 0, w_up[kBinsEach], w_dn[kBinsEach];
#pragma unroll
          for (int i = 0; i < kBinsEach; ++i) {
            w_up[i] = w_dn[i] = 0;
            if (cnt[i] != 0) bounds(tid * kBinsEach + i, static_cast<F>(cnt[i]), w_up[i], w_dn[i]);
            up += w_up[i];
            dn += w_dn[i];
          }
          const F su = scan_lanes(up), sd = scan_lanes(dn);
          F* const sums = reinterpret_cast<F*>(sh.wt);
          if (lane == 31) {
            sums[warp] = su;
            sums[kWarps + warp] = sd;
          }
          __syncthreads();
          const F wu = scan_lanes(lane < kWarps ? sums[lane] : F(0)), wd = scan_lanes(lane < kWarps ? sums[kWarps + lane] : F(0));
          F run_up = static_cast<F>(mass) + (su - up), run_dn = static_cast<F>(mass) + (sd - dn);
          if (warp > 0) {
            run_up += __shfl_sync(0xffffffffu, wu, max(warp - 1, 0));
            run_dn += __shfl_sync(0xffffffffu, wd, max(warp - 1, 0));
          }
          // What the classes behind hold bounds it too, where those are all there
          // is (a mark near the whole: the error is that of the rest)
          const F all_up = __shfl_sync(0xffffffffu, wu, 31), all_dn = __shfl_sync(0xffffffffu, wd, 31), sum = static_cast<F>(whole);
          const F low = static_cast<F>(mark) * (1 - slack), high = static_cast<F>(mark) * (1 + slack);
#pragma unroll
          for (int i = 0; i < kBinsEach; ++i) {
            run_up += w_up[i];
            run_dn += w_dn[i];
            if (cnt[i] == 0) continue;
            if (c_lo == kBins && run_up > low && (!linear || sum - (all_dn - run_dn) > low)) c_lo = tid * kBinsEach + i;
            if (c_hi == kBins && (run_dn > high || (linear && sum - (all_up - run_up) > high))) c_hi = tid * kBinsEach + i;
          }
        };
        if (linear) {
          // powers of two by distance, which end half a step above it; fp32 does
          // (sums of 2048 terms, to 2^-16: a class is 2^-6 of its weight wide)
          by_mass(0.f, 1.f / 65536, [&](int c, float n, float& u, float& d) {
            u = exp2f(static_cast<float>(c) * (-1.f * kPerClass / kSteps) + 1.f / kSteps) * n;
            d = c == kBins - 1 ? 0.f : exp2f(static_cast<float>(c + 1) * (-1.f * kPerClass / kSteps)) * n;
          });
        } else {
          by_mass(0.0, 1e-12, [&](int c, double n, double& u, double& d) {
            u = weight(r, sh.power, value_of(static_cast<uint32_t>(upper(c) >> 32))) * n;
            d = weight(r, sh.power, value_of(static_cast<uint32_t>(lower(c) >> 32))) * n;
          });
        }
      }
      if (c_lo < kBins) atomicMin(&sh.lo, c_lo);
      if (c_hi < kBins) atomicMin(&sh.hi, c_hi);
      __syncthreads();
      c_lo = sh.lo;
      c_hi = sh.hi;
      if (by_k && c_lo == kBins) break;  // fewer tokens than k: all are kept
      // (no class where the sum stays below its mark: the cut lies behind all of them)
      if (c_lo == kBins) c_lo = end_class;
      if (c_hi == kBins) c_hi = end_class;
      // tokens down to the last of these classes, and before the first
      if (tid == c_hi / kBinsEach) {
        uint32_t run = before;
#pragma unroll
        for (int i = 0; i < kBinsEach; ++i) run += i <= c_hi % kBinsEach ? cnt[i] : 0;
        sh.down = static_cast<int>(run);
      }
      if (tid == c_lo / kBinsEach) {
        uint32_t run = before;
#pragma unroll
        for (int i = 0; i < kBinsEach; ++i) run += i < c_lo % kBinsEach ? cnt[i] : 0;
        sh.from = static_cast<int>(run);
      }
      __syncthreads();
      const int down = sh.down, inside = down - sh.from;
      u64 nlo = lower(c_hi), nhi = upper(c_lo);
      nlo = nlo > cut ? nlo : cut;
      const bool from_top = above + down <= kWhole;
      if (from_top || inside <= kList) {
        // ---- the list: all pairs down to nlo, or those of the classes alone ----
        const u64 ghi = from_top ? best : nhi;
        {
          double sum = 0.0;
          int over = 0;
          copies = -1;
          if (!from_top && (!by_k || !need_p) && above + down <= kCopies * kWarps * split) {
            copies = copy_pass<T>(nlo);
            sh.copies[warp] = copies;
            __syncthreads();
            // (whether any warp of the CTA has more than it could copy)
            copied = __reduce_max_sync(0xffffffffu, sh.copies[lane % kWarps]) <= kCopies;
          }
          if (copies >= 0 && copied) {
            split_copies(ghi, !by_k, copies, sum, over);
          } else {
            copied = false;
            double above_mass = 0.0;
            if (!by_k && !from_top) draw_pass<T>(ghi + 1, -3.4028234663852886e38f, above_mass);
            pair_pass<T>(nlo, ghi, false, true, 0, sum, over);
            sum = above_mass;
          }
          publish(sum, over, 0);
        }
        barrier();
        const int n = all_of(&sh.count), over_count = all_of(&sh.over);
        const double over_mass = all_parts();
        if (n <= kList) {
          if (rank == 0) {
            // the other CTAs' pairs behind this one's: lane c knows where CTA c's start
            const int of_c = of_all(&sh.count, 0);
            int at_c = of_c;
#pragma unroll
            for (int o = 1; o < kMaxSplit; o <<= 1) {
              const int m = __shfl_up_sync(0xffffffffu, at_c, o);
              if (lane >= o) at_c += m;
            }
            const int c = 1 + warp / 2;  // two warps for each
            if (c < split) {
              const int m = __shfl_sync(0xffffffffu, of_c, c), at = __shfl_sync(0xffffffffu, at_c, c) - m;
              const u64* from = cluster.map_shared_rank(&sh.list[0], c);
              for (int i = lane + 32 * (warp % 2); i < m; i += 64) sh.list[at + i] = from[i];
            }
            __syncthreads();
            sort_list(n);
            if (from_top) {
              // all of it: top-k, top-p, min-p and the draw on the list
              int m = need_k ? min(n, want_k) : n;
              list_weights(n, 32);
              const int by_min =
                  want_m > 0.f ? first_ones(m, [&](int i) { return value_of(static_cast<uint32_t>(sh.sorted[i] >> 32)) >= x_min; }) : m;
              if (need_p) {
                __syncthreads();
                running_sums(m);
                const double end = p_of * (need_k ? sh.wt[m - 1] : whole);
                m = first_ones(m, [&](int i) { return i == 0 || sh.wt[i - 1] <= end; });
              }
              m = min(m, by_min);
              // the kept ones by their index, each with its value
              for (int i = tid; i < m; i += kThreads) sh.list[i] = sh.sorted[i] << 32 | sh.sorted[i] >> 32;
              __syncthreads();
              sort_list(m);  // the largest high half, the smallest index, first
              list_weights(m, 0);
              running_sums(m);
              const double target = fmax(u * sh.wt[m - 1], 0.0);
              const int pick = first_ones(m, [&](int i) { return !(sh.wt[i] > target); });
              // (none where rounding, or a number of 1, leaves none: the last with weight)
              const int some = pick < m ? 0 : first_ones(m, [&](int i) { return sh.wt[i] < sh.wt[m - 1]; });
              if (tid == 0) a.tokens[b] = index_of(sh.sorted[pick < m ? pick : some] >> 32);
            } else if (by_k) {
              if (tid == 0) sh.cut = sh.sorted[min(n, want_k - over_count) - 1];
            } else {
              list_weights(n, 32);
              running_sums(n);
              const double end = p_of * whole;
              const int m = first_ones(n, [&](int i) { return over_mass + (i == 0 ? 0.0 : sh.wt[i - 1]) <= end; });
              if (tid == 0) sh.cut = m > 0 ? sh.sorted[m - 1] : ghi + 1;
            }
          }
          barrier();
          if (from_top) return;  // drawn
          cut = *cluster.map_shared_rank(&sh.cut, 0);
          if (tid == 0) sh.count = 0;  // (the other CTAs have read it)
          break;
        }
        barrier();  // the counts have been read
        if (tid == 0) sh.count = 0;
        for (int i = tid; i < kBins; i += kThreads) sh.bins[i] = 0;  // (tiles lie over them)
      }
      if (!by_k && !linear && nhi - nlo > (hi - lo) / 2) {
        // Classes so wide that their bounds say little (a tiny temperature): one
        // step by the exact sum over the middle, so that the range always shrinks.
        const u64 mid = nlo + (nhi - nlo) / 2;
        barrier();
        double sum;
        int over;
        pair_pass<T>(mid + 1, mid, true, false, 0, sum, over);
        publish(sum, over, 0);
        barrier();
        const double s = all_parts();
        barrier();
        if (s > mark) {
          nlo = mid + 1;
        } else {
          nhi = mid;
        }
      }
      linear = false;
      lo = nlo;
      hi = nhi;
      __syncthreads();
    }
    if (by_k) {
      need_k = false;
      if (need_p) copied = false;
    } else {
      need_p = false;
    }
    __syncthreads();
  }

  // ---- the draw over the kept tokens ----
  {
    double sum;
    const u64 heavy = cut != 0 ? cut : 1;
    if (copied) {
      draw_copies(heavy, x_min, sum);
    } else {
      draw_pass<T>(heavy, x_min, sum);
    }
    publish(lane == 0 ? sum : 0.0, 0, 0);
  }
  barrier();
  double total = 0.0, before = 0.0;
  int last = -1;
  {
    const double mine = of_all(&sh.part, 0.0);
#pragma unroll
    for (int c = 0; c < kMaxSplit; ++c) {  // in the order of the CTAs
      const double s = __shfl_sync(0xffffffffu, mine, c);
      if (c < rank) before += s;
      total += s;
      if (s > 0.0) last = c;
    }
  }
  cluster.barrier_arrive();  // this CTA has read the others' sums; nobody leaves before all have
  if (warp == 0) {
    // as in verify_draft.cu: the first tile whose running sum exceeds the number, or
    // the last with weight where rounding leaves none
    const double target = fmax(u * total, 0.0);
    const bool chosen = total > target ? before + sh.part > target && !(before > target) : rank == last;
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
        const int x = r.x0 + at * kTile + lane * 8;
        Row one = sh.row[0];
        one.w0 = at;
        one.w1 = at + 1;
        double w[8], s = 0.0;
        each<T>(one, [&](int, int x, const float (&f)[8]) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const bool kept = f[i] >= r.least && f[i] >= x_min && pair_of(f[i], x + i) >= cut;
            w[i] = kept ? weight(r, sh.power, f[i]) : 0.0;
            s += w[i];
          }
        });
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
  static std::atomic<bool> done[3][64];
  auto k = type == 2 ? sample_tokens_kernel<float> : type == 1 ? sample_tokens_kernel<__nv_bfloat16> : sample_tokens_kernel<__half>;
  const cudaError_t e = prepare_kernel(done[type], k, static_cast<int>(sizeof(Shared)), 0);
  if (e != cudaSuccess) return e;
  int split = kMaxSplit;
  while (split > 1 && static_cast<int64_t>(a.B) * split > 2 * sm_count() &&
         a.V <= static_cast<int64_t>(kMaxTiles - 2) * kTile * (split / 2))
    split /= 2;
  return launch_paged(k, dim3(a.B * split), dim3(kThreads), sizeof(Shared), split, true, st, a);
}

}  // namespace persona
