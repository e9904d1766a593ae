// Causal attention of each sequence's new tokens over its paged KV cache, for
// many query rows per kv head (prompt chunks): the same result as
// paged_attention.cu, on the tensor cores' tcgen05 path.
//
// A tile is up to 256 query rows (token, head of the group) of one sequence
// and kv head, in two halves A and B of 128 rows; a unit is one block of 128
// positions of a tile.  The units of all tiles lie in one line (sequence,
// tile, kv head, block), cut into equal ranges, one per CTA and SM; tiles end
// at their last row's position, so a range of units is a range of work.  Cut
// tiles leave pieces that a second kernel joins in order.
//
// Per block and half: S = Q K^T (operands in shared memory, 128 x 128 fp32
// accumulator in tensor memory), softmax with one thread per row, P written
// back over S as 16 bits, O += P V (P from tensor memory, V from shared
// memory).  While one half is in its softmax the tensor cores work on the
// other.  512 columns of tensor memory: S/P and O of both halves.
//
// Warps: 0-3 and 4-7 softmax of halves A and B (thread = row), 8-11 load
// (pages to swizzled shared memory), 12 issues the MMAs.  Rows are loaded by
// cp.async from per-position offsets, so pages may end anywhere in a block.
//
// The running maximum is only moved, and O only rescaled, once a row's new
// maximum exceeds it by 2^8: until then the weights may grow to 256, which
// fp16, bf16 and the fp32 sums hold as exactly as weights up to 1.
//
// What bounds it: per block and both halves 2048 cycles of tensor work against
// 3400 of the chain scores - softmax - products of each half; the exponentials
// (128 x 128 a half, 16 per cycle and SM) are not it: an eighth of them by a
// polynomial on the FMA units took 4 % longer.  Measured (f16, 32 heads over 8,
// D = 128, calls in a row): 4096 new tokens over 16384 positions 919 us, 1.05
// PFLOP/s, 0.75 of the measured sustained bf16 rate (792 us in bursts, 0.73 of
// the burst rate).  At D = 64 655 us: half the products, the same chain.  32
// prompts of 512 with nothing cached 174 us: 35 blocks per SM are 62 us of it,
// most of the rest is starting and ending fourteen tiles.
//
// 8-bit pages: codes become fp16 in shared memory, exactly; the k scale
// multiplies the fp32 score and log2 of the v scale joins its exponent (see
// paged_attention.cu).  The same chunk then takes 1.41 ms: the codes are
// converted once per tile of 256 rows, and each row reads every column's
// scales.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "paged_attention.cuh"
#include "tcgen05.cuh"

namespace persona {
namespace {

constexpr int kThreads = 512;
constexpr int kBlock = 128;  // positions of a unit
constexpr int kTile = 256;   // rows of a tile
constexpr int kLoaders = 128;
// Registers per thread after the split: two softmax warpgroups, loaders, MMA.
// 2 x 184 + 96 + 48 = 512 <= 4 x 128, what the block is launched with.
constexpr int kRegsSoftmax = 184, kRegsLoad = 96, kRegsMma = 48, kRegsLaunch = 128;
static_assert(2 * kRegsSoftmax + kRegsLoad + kRegsMma <= 4 * kRegsLaunch, "register split");

template <int D> struct Cfg {
  static constexpr int kStages = 256 / D;              // k and v slots
  static constexpr int kHalfBytes = 128 * 128;         // 128 rows of 64 16-bit elements
  static constexpr int kSlot = kHalfBytes * (D / 64);  // 128 x D, 64-element columns side by side
  static constexpr int kScales = kStages + 1;          // slots of scales: the softmax may be one block behind the k slots
  static constexpr int kSmem = 1024 + kSlot * (2 + 2 * kStages);
};

struct Shared {
  uint64_t q_full, q_empty;
  uint64_t k_full[4], k_empty[4], v_full[4], v_empty[4];
  uint64_t s_full[2], p_ready[2], p_rest[2], pv_done[2], drained;
  uint32_t tmem;
  int abort;
  int b, tile;
  long long off, begin, end, sum[16], items[16];
  long long at[2][kBlock];   // page offset (bytes) of each position of a block, -1: none
  alignas(16) float ks[5][kBlock];  // read four at a time
  alignas(16) float lv[5][kBlock];
  alignas(16) float rv[5][kBlock];
  long long q_at[2][kTile];  // offset (elements) of each row of a tile, -1: none; by piece
  alignas(16) uint8_t stage[8][2048];  // finished rows on their way out, by softmax warp
  float qmul[2][kTile];      // by piece: the next one's rows are loaded while this one's are read
};

// What starting and ending a tile costs, in units: so many stand before its
// first one in the line.  None where every unit has a CTA of its own.
constexpr int kPieceUnits = 2;

struct TileGeo {
  int m0, mrows, first, per, pbegin, pend;  // per: with the `lead` units above
};
__device__ __forceinline__ TileGeo tile_geo(const Seq& s, int window, int G, int t, int lead) {
  TileGeo g;
  g.m0 = t * kTile;
  g.mrows = min(kTile, s.n * G - g.m0);
  const int ctx = s.len - s.n, tok0 = g.m0 / G, tok1 = (g.m0 + g.mrows - 1) / G;
  g.pend = max(0, min(s.len, ctx + tok1 + 1));
  g.pbegin = window > 0 ? max(0, ctx + tok0 + 1 - window) : 0;
  g.first = g.pbegin / kBlock;
  g.per = max(1, (g.pend + kBlock - 1) / kBlock - g.first) + lead;
  return g;
}
__device__ __forceinline__ int seq_tiles(const Seq& s, int G) { return (s.n * G + kTile - 1) / kTile; }

// The pieces of a CTA's range of units, walked alike by every role.
struct Walk {
  const PagedAttention& a;
  int lead;
  int b, t, h;
  long long left;
  Seq seq;
  TileGeo g;
  int k0, k1;
  bool first;
  __device__ __forceinline__ Walk(const PagedAttention& a_, int lead_, int b_, int t_, long long off, long long left_)
      : a(a_), lead(lead_), b(b_), t(t_), left(left_), first(true) {
    seq = load_seq(a, b);
    g = tile_geo(seq, a.window, a.G, t, lead);
    h = static_cast<int>(off / g.per);
    k1 = static_cast<int>(off - static_cast<long long>(h) * g.per);
    k0 = k1;
  }
  // to the next piece: tile (t, h) of sequence b, blocks [k0, k1)
  __device__ __forceinline__ bool next() {
    if (left <= 0) return false;
    if (k0 != k1) first = false;
    if (k1 == g.per) {
      k1 = 0;
      if (++h == a.c.Hkv) {
        h = 0;
        ++t;
        while (t >= seq_tiles(seq, a.G)) {
          if (++b >= a.c.B) return false;
          seq = load_seq(a, b);
          t = 0;
        }
        g = tile_geo(seq, a.window, a.G, t, lead);
      }
    }
    k0 = k1;
    k1 = static_cast<int>(min(static_cast<long long>(g.per), k0 + left));
    left -= k1 - k0;
    return true;
  }
  __device__ __forceinline__ int block0() const { return g.first + max(k0 - lead, 0); }
  __device__ __forceinline__ int blocks() const { return g.pend > 0 ? max(k1 - lead, 0) - max(k0 - lead, 0) : 0; }
  __device__ __forceinline__ bool has_b() const { return g.mrows > 128; }
};

// Two fp32 operations in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, c, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
      "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
      "mul.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
      "add.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
template <int N> __device__ __forceinline__ void regs_inc() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void regs_dec() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

template <typename T, int D, bool kE4m3>
__global__ void __launch_bounds__(kThreads, 1) paged_chunk_kernel(const __grid_constant__ PagedAttention a) {
  using C = Cfg<D>;
  using PT = typename std::conditional<kE4m3, __half, T>::type;  // type of the products
  constexpr bool kScaleQ = kE4m3 && !std::is_same<T, __half>::value;
  constexpr int kSt = C::kStages;
  constexpr int kFirstPart = kE4m3 ? 2 : 3;  // quarters of P that the first products take (8-bit: registers)
  extern __shared__ uint8_t smem_raw[];
  __shared__ Shared sh;
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t s_q = base, s_k = base + 2 * C::kSlot, s_v = s_k + kSt * C::kSlot;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int cta = blockIdx.x, G = a.G;
  // Wait before anything else, the allocation of tensor memory included: a
  // kernel before this one may still hold some.
  pdl_wait();
  if (warp == 12) {
    tc::tmem_alloc(&sh.tmem, 512);
    tc::tmem_relinquish();
  }
  if (tid == 0) {
    mbar_init(&sh.q_full, kLoaders);
    mbar_init(&sh.q_empty, 1);
    for (int i = 0; i < kSt; ++i) {
      mbar_init(&sh.k_full[i], kLoaders);
      mbar_init(&sh.v_full[i], kLoaders);
      mbar_init(&sh.k_empty[i], 1);
      mbar_init(&sh.v_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sh.s_full[i], 1);
      mbar_init(&sh.p_ready[i], 128);
      mbar_init(&sh.p_rest[i], 128);
      mbar_init(&sh.pv_done[i], 1);
    }
    mbar_init(&sh.drained, 1);
    sh.abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    a.desc[2 * cta] = make_int4(0, 0, 0, 0);
  }

  // ---- this CTA's range of units ----
  auto seq_sum = [&](int b, int& items) -> long long {  // units without the lead, and tiles times heads
    items = 0;
    if (b >= a.c.B) return 0;
    const Seq s = load_seq(a, b);
    long long u = 0;
    const int tiles = seq_tiles(s, G);
    for (int t = 0; t < tiles; ++t) u += tile_geo(s, a.window, G, t, 0).per;
    items = tiles * a.c.Hkv;
    return u * a.c.Hkv;
  };
  long long total = 0, all_items = 0, mine = 0;
  int my_items = 0;
  for (int b0 = 0; b0 < a.c.B; b0 += kThreads) {
    int n;
    const long long u = seq_sum(b0 + tid, n);
    if (b0 == 0) {
      mine = u;
      my_items = n;
    }
    long long w = u, v = n;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      w += __shfl_xor_sync(0xffffffffu, w, o);
      v += __shfl_xor_sync(0xffffffffu, v, o);
    }
    if (lane == 0) {
      sh.sum[warp] = w;
      sh.items[warp] = v;
    }
    __syncthreads();
    for (int i = 0; i < 16; ++i) {
      total += sh.sum[i];
      all_items += sh.items[i];
    }
    __syncthreads();
  }
  const int lead = total <= gridDim.x ? 0 : kPieceUnits;
  total += lead * all_items;
  // no more CTAs than units, so that every range (before the move below) has one
  const int ctas = static_cast<int>(min(total, static_cast<long long>(gridDim.x)));
  if (tid == 0) sh.begin = sh.end = cta < ctas ? total * (cta + 1) / ctas : 0;
  if (cta < ctas) {
    const long long raw0 = total * cta / ctas, raw1 = total * (cta + 1) / ctas;
    long long run = 0;
    for (int b0 = 0; b0 < a.c.B && run <= raw1; b0 += kThreads) {
      int n = my_items;
      long long u = b0 == 0 ? mine : seq_sum(b0 + tid, n);
      u += static_cast<long long>(n) * lead;
      long long inc = u;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long up = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += up;
      }
      if (lane == 31) sh.sum[warp] = inc;
      __syncthreads();
      long long lo = run + inc - u;
      for (int i = 0; i < warp; ++i) lo += sh.sum[i];
#pragma unroll 1
      for (int side = 0; side < 2; ++side) {  // both ends: tile, and offset in its units
        const long long raw = side == 0 ? raw0 : raw1;
        if (raw < lo || raw >= lo + u) continue;
        long long off = raw - lo;
        const Seq s = load_seq(a, b0 + tid);
        const int tiles = seq_tiles(s, G);
        int t = 0, per = 1;
        for (; t < tiles; ++t) {
          per = tile_geo(s, a.window, G, t, lead).per;
          const long long c = static_cast<long long>(per) * a.c.Hkv;
          if (off < c || t == tiles - 1) break;
          off -= c;
        }
        // a cut inside what a tile costs to start is moved before it
        const int k = static_cast<int>(off % per), back = k < lead ? k : 0;
        if (side == 0) {
          sh.b = b0 + tid;
          sh.tile = t;
          sh.off = off - back;
          sh.begin = raw - back;
        } else {
          sh.end = raw - back;
        }
      }
      for (int i = 0; i < 16; ++i) run += sh.sum[i];
      __syncthreads();
    }
  }
  __syncthreads();
  const long long u0 = sh.begin, u1 = sh.end;
  const bool works = u0 < u1;
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  pdl_launch();  // after the allocation: a dependent that takes tensor memory must find ours taken
  const uint32_t tmem = sh.tmem;
  int* const abort = &sh.abort;
  int32_t* const err = a.err;

  if (warp < 8) {
    // ------------------------------------------------------------ softmax --
    regs_inc<kRegsSoftmax>();
    const int half = warp >> 2;
    const int r = half * 128 + (warp & 3) * 32 + lane;  // row of the tile
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t t_s = tmem + lanes + half * 128, t_o = tmem + lanes + 256 + half * D;
    int n_s = 0, n_pv = 0, n_sc = 0, n_q = 0;  // blocks so far: of this half, and of all (the scales' slots); pieces
    bool ok = true;
    auto wait = [&](uint64_t* bar, int n) {  // the same answer in the whole warp, as the tensor memory loads need
      ok = __all_sync(0xffffffffu, mbar_wait_abortable(bar, n & 1, err, abort));
      tc::fence_after_sync();
      return ok;
    };
    if (works) {
      Walk w(a, lead, sh.b, sh.tile, sh.off, u1 - u0);
      while (ok && w.next()) {
        const int nb = w.blocks();
        const bool act = half == 0 || w.has_b();
        const int ctx = w.seq.len - w.seq.n;
        const bool live = r < w.g.mrows;
        const int mm = w.g.m0 + (live ? r : 0), tok = mm / G, hg = mm - tok * G;
        const int hi = live ? ctx + tok : -1;                        // last position this row sees
        const int lo = a.window > 0 ? max(0, hi - a.window + 1) : 0;  // and the first
        // positions that every row of the tile sees
        const int all_hi = ctx + w.g.m0 / G;
        const int all_lo = a.window > 0 ? ctx + (w.g.m0 + w.g.mrows - 1) / G - a.window + 1 : 0;
        float m = kNegInf, l = 0.f, qm = a.scale_log2;
        for (int j = 0; act && j < nb; ++j) {
          if (!wait(&sh.s_full[half], n_s)) break;
          ++n_s;
          if (kScaleQ && j == 0) qm = sh.qmul[n_q & 1][r];
          float s[kBlock];
#pragma unroll
          for (int c = 0; c < 4; ++c) tc::ld32(t_s + 32 * c, reinterpret_cast<uint32_t*>(s) + 32 * c);
          tc::wait_ld();
          const int p0 = (w.block0() + j) * kBlock;
          const int sc = (n_sc + j) % C::kScales;
          if (kE4m3) {
            const float4* ks = reinterpret_cast<const float4*>(sh.ks[sc]);
            const float4* lv = reinterpret_cast<const float4*>(sh.lv[sc]);
#pragma unroll
            for (int c = 0; c < kBlock; c += 4) {
              if (c % 16 == 0) asm volatile("" ::: "memory");  // keeps the loads near their use, in few registers
              const float4 k4 = ks[c / 4], l4 = lv[c / 4];
              const float2 x = fma2(mul2(make_float2(s[c], s[c + 1]), make_float2(k4.x, k4.y)), both(qm), make_float2(l4.x, l4.y));
              const float2 y = fma2(mul2(make_float2(s[c + 2], s[c + 3]), make_float2(k4.z, k4.w)), both(qm), make_float2(l4.z, l4.w));
              s[c] = x.x;
              s[c + 1] = x.y;
              s[c + 2] = y.x;
              s[c + 3] = y.y;
            }
          }
          if (p0 + kBlock - 1 > all_hi || p0 < all_lo) {
#pragma unroll
            for (int x = 0; x < kBlock / 32; ++x) {
              // bits of the positions that this row sees
              const int n1 = min(max(hi - p0 + 1 - 32 * x, 0), 32), n0 = min(max(lo - p0 - 32 * x, 0), 32);
              const uint32_t keep = static_cast<uint32_t>((1ull << n1) - 1) & ~static_cast<uint32_t>((1ull << n0) - 1);
#pragma unroll
              for (int c = 0; c < 32; ++c) s[32 * x + c] = (keep & (1u << c)) != 0 ? s[32 * x + c] : kNegInf;
            }
          }
          float mxs[8];
#pragma unroll
          for (int c = 0; c < 8; ++c) mxs[c] = fmaxf(s[c], s[c + 8]);
#pragma unroll
          for (int c = 16; c < kBlock; c += 16)
#pragma unroll
            for (int x = 0; x < 8; ++x) mxs[x] = max3(mxs[x], s[c + x], s[c + 8 + x]);
          const float mul = kE4m3 ? 1.f : a.scale_log2;
          const float mx = mul * fmaxf(max3(max3(mxs[0], mxs[1], mxs[2]), mxs[3], mxs[4]), max3(mxs[5], mxs[6], mxs[7]));
          const bool grow = j > 0 && mx > m + kGrow;
          const float shrink = grow ? exp2_approx(m - mx) : 1.f;
          if (j == 0 || grow) m = mx;
          const float2 neg = both(m == kNegInf ? 0.f : -m);
          float2 sum[2] = {both(0.f), both(0.f)};
          const float4* rv = reinterpret_cast<const float4*>(sh.rv[sc]);
          // The weights go back over S, 32 positions at a time, and the tensor
          // cores start on the first of them.
          auto weights = [&](auto from, auto to) {
            constexpr int kFrom = decltype(from)::value, kTo = decltype(to)::value;
            uint32_t pk[(kTo - kFrom) / 2];
#pragma unroll
            for (int c = kFrom; c < kTo; c += 4) {
              float2 x = make_float2(s[c], s[c + 1]), y = make_float2(s[c + 2], s[c + 3]);
              x = kE4m3 ? add2(x, neg) : fma2(x, both(a.scale_log2), neg);
              y = kE4m3 ? add2(y, neg) : fma2(y, both(a.scale_log2), neg);
              x = make_float2(exp2_approx(x.x), exp2_approx(x.y));
              y = make_float2(exp2_approx(y.x), exp2_approx(y.y));
              if (kE4m3) {
                if (c % 16 == 0) asm volatile("" ::: "memory");
                const float4 r4 = rv[c / 4];
                sum[0] = fma2(x, make_float2(r4.x, r4.y), sum[0]);
                sum[1] = fma2(y, make_float2(r4.z, r4.w), sum[1]);
              } else {
                sum[0] = add2(sum[0], x);
                sum[1] = add2(sum[1], y);
              }
              pk[(c - kFrom) / 2] = Mma<PT>::pack(x.x, x.y);
              pk[(c - kFrom) / 2 + 1] = Mma<PT>::pack(y.x, y.y);
            }
#pragma unroll
            for (int c = 0; c < (kTo - kFrom) / 32; ++c) tc::st16(t_s + kFrom / 2 + 16 * c, pk + 16 * c);
          };
          weights(std::integral_constant<int, 0>(), std::integral_constant<int, 32 * kFirstPart>());
          if (__any_sync(0xffffffffu, grow)) {
            // the products before this block have to be in O first
            if (!wait(&sh.pv_done[half], n_pv + j - 1)) break;
#pragma unroll 1
            for (int c = 0; c < D / 32; ++c) {
              uint32_t o[32];
              tc::ld32(t_o + 32 * c, o);
              tc::wait_ld();
#pragma unroll
              for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * shrink);
              tc::st32(t_o + 32 * c, o);
            }
          }
          tc::wait_st();
          tc::fence_before_sync();
          mbar_arrive(&sh.p_ready[half]);
          weights(std::integral_constant<int, 32 * kFirstPart>(), std::integral_constant<int, kBlock>());
          l = fmaf(l, shrink, (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y));
          tc::wait_st();
          tc::fence_before_sync();
          mbar_arrive(&sh.p_rest[half]);
        }
        if (!ok) break;
        n_sc += nb;
        if (nb > 0) ++n_q;
        if (!act) continue;
        // ---- this piece's rows ----
        if (nb > 0) {
          if (!wait(&sh.pv_done[half], n_pv + nb - 1)) break;
          n_pv += nb;
        }
        const bool complete = w.k0 == 0 && w.k1 == w.g.per;
        const float inv = l > 0.f && m != kNegInf ? 1.f / l : 0.f;
        float* part = a.part + static_cast<int64_t>(2 * cta + (w.first ? 0 : 1)) * Part<kTile, D>::kFloats;
        // Finished rows go through 2 KB of shared memory per warp, 32 columns at
        // a time, so that four lanes write 64 bytes of a row side by side;
        // pieces are kept four columns by four, a lane per row.
        const long long mine = live ? static_cast<int64_t>(w.seq.row0 + tok) * a.out.row_stride +
                                          static_cast<int64_t>(w.h * G + hg) * a.out.head_stride
                                    : -1;
        long long to[4];
        if (complete) {
#pragma unroll
          for (int i = 0; i < 4; ++i) to[i] = __shfl_sync(0xffffffffu, mine, 8 * i + (lane >> 2));
        }
        const uint32_t stage = smem_u32(sh.stage[warp]);
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
          float o[32];
          if (nb > 0) {
            tc::ld32(t_o + 32 * c, reinterpret_cast<uint32_t*>(o));
            tc::wait_ld();
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = 0.f;
          }
          if (complete) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
              asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(stage + lane * 64 + ((i ^ ((lane >> 1) & 3)) << 4)),
                           "r"(Mma<T>::pack(o[8 * i] * inv, o[8 * i + 1] * inv)), "r"(Mma<T>::pack(o[8 * i + 2] * inv, o[8 * i + 3] * inv)),
                           "r"(Mma<T>::pack(o[8 * i + 4] * inv, o[8 * i + 5] * inv)), "r"(Mma<T>::pack(o[8 * i + 6] * inv, o[8 * i + 7] * inv))
                           : "memory");
            __syncwarp();
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int row = 8 * i + (lane >> 2);
              const uint4 v = lds128(stage + row * 64 + (((lane & 3) ^ ((row >> 1) & 3)) << 4));
              if (to[i] >= 0) *reinterpret_cast<uint4*>(static_cast<T*>(a.out.p) + to[i] + 32 * c + 8 * (lane & 3)) = v;
            }
            __syncwarp();
          } else {
#pragma unroll
            for (int i = 0; i < 32; i += 4)
              *reinterpret_cast<float4*>(part + (8 * c + i / 4) * (4 * kTile) + 4 * r) = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
          }
        }
        if (!complete) {
          part[kTile * D + r] = m;
          part[kTile * D + kTile + r] = l;
        }
        // O is read: the first product of the next piece waits for this
        // half's next p_ready, which comes after
        tc::fence_before_sync();
        if (r == 0 && w.k0 == 0 && w.k1 < w.g.per) {
          const long long end = u1 - w.left - w.k1 + w.g.per - 1;  // the tile's last unit
          long long c = end * ctas / total;
          while (total * (c + 1) / ctas <= end) ++c;
          while (total * c / ctas > end) --c;
          note_cut(a, cta, w.first, static_cast<int>(c), w.g.m0, w.g.mrows, w.seq.row0, w.h);
        }
      }
    }
  } else if (warp < 12) {
    // -------------------------------------------------------------- loads --
    regs_dec<kRegsLoad>();
    const int t = tid - 256;
    int n_k = 0, n_q = 0, n_at = 0;  // blocks, pieces and published blocks so far
    bool ok = true;
    uint64_t* pending = nullptr;  // loads under way whose arrival is due
    auto flush = [&]() {
      if (pending != nullptr) {
        cp_wait<0>();
        tc::fence_proxy_async();
        mbar_arrive(pending);
        pending = nullptr;
      }
    };
    auto issued = [&](uint64_t* bar) {
      cp_commit();
      if (pending != nullptr) {
        cp_wait<1>();
        tc::fence_proxy_async();
        mbar_arrive(pending);
      }
      pending = bar;
    };
    auto acquire = [&](uint64_t* bar, uint32_t parity) {
      if (mbar_try_wait(bar, parity)) return true;
      flush();  // nobody waits for what this thread holds back
      return mbar_wait_abortable(bar, parity, err, abort);
    };
    if (works) {
      Walk w(a, lead, sh.b, sh.tile, sh.off, u1 - u0);
      // A wait that gave up (ok) ends the loads but not the walk: the barrier
      // of the four warps needs them all.
      while (w.next()) {
        const int nb = w.blocks();
        if (nb == 0) continue;
        // ---- q rows ----
        if (n_q > 0) ok = ok && acquire(&sh.q_empty, (n_q - 1) & 1);
        if (ok) {
          // thread t works out where rows t and 128 + t are
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const int i = t + 128 * x, mm = w.g.m0 + i, tok = mm / G;
            sh.q_at[n_q & 1][i] = i < w.g.mrows ? static_cast<int64_t>(tok) * a.q.row_stride +
                                                      static_cast<int64_t>(mm - tok * G) * a.q.head_stride
                                                : -1;
          }
        }
        named_sync(1, kLoaders);
        if (ok) {
          constexpr int kCh = D / 8, kPer = kLoaders / kCh, kAhead = 8;
          const int c = t % kCh, rows = w.has_b() ? 256 : 128;
          const T* qb = static_cast<const T*>(a.q.p) + static_cast<int64_t>(w.seq.row0) * a.q.row_stride +
                        static_cast<int64_t>(w.h * G) * a.q.head_stride + c * 8;
          for (int i0 = t / kCh; i0 < rows; i0 += kPer * kAhead) {
            long long from[kAhead];
#pragma unroll
            for (int x = 0; x < kAhead; ++x) from[x] = sh.q_at[n_q & 1][i0 + x * kPer];
            auto place = [&](int i) {
              return s_q + (i >> 7) * C::kSlot + (c >> 3) * C::kHalfBytes + (i & 127) * 128 + (((c & 7) ^ (i & 7)) << 4);
            };
            if constexpr (!kScaleQ) {
#pragma unroll
              for (int x = 0; x < kAhead; ++x) cp_async16(place(i0 + x * kPer), qb + (from[x] < 0 ? 0 : from[x]), from[x] >= 0);
            } else {
              // bf16 row -> fp16, scaled by the power of two that brings its
              // largest element into [1, 2)
              uint4 v[kAhead];
#pragma unroll
              for (int x = 0; x < kAhead; ++x)
                v[x] = from[x] >= 0 ? __ldg(reinterpret_cast<const uint4*>(qb + from[x])) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
              for (int x = 0; x < kAhead; ++x) {
                const int i = i0 + x * kPer;
                const uint32_t u[4] = {v[x].x, v[x].y, v[x].z, v[x].w};
                float f[8], mx = 0.f;
#pragma unroll
                for (int y = 0; y < 4; ++y) {
                  const float2 p = Cvt<T>::to2(u[y]);
                  f[2 * y] = p.x;
                  f[2 * y + 1] = p.y;
                  mx = fmaxf(mx, fmaxf(fabsf(p.x), fabsf(p.y)));
                }
#pragma unroll
                for (int o = kCh / 2; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
                const int e = min(max(static_cast<int>(__float_as_uint(mx) >> 23), 2), 252);
                const float down = __uint_as_float(static_cast<uint32_t>(254 - e) << 23);
                if (c == 0) sh.qmul[n_q & 1][i] = a.scale_log2 * __uint_as_float(static_cast<uint32_t>(e) << 23);
                asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(place(i)), "r"(Mma<__half>::pack(f[0] * down, f[1] * down)),
                             "r"(Mma<__half>::pack(f[2] * down, f[3] * down)), "r"(Mma<__half>::pack(f[4] * down, f[5] * down)),
                             "r"(Mma<__half>::pack(f[6] * down, f[7] * down))
                             : "memory");
              }
            }
          }
        }
        if (ok) issued(&sh.q_full);
        ++n_q;
        // ---- blocks ----
        const int32_t* row = a.c.table + w.b * a.c.table_stride;
        const int first = w.block0();
        // Thread t looks up position t of a block, one block ahead: the page
        // is read here and used when the block is due.
        int pg = -1, at = 0;
        bool seen = false;
        auto fetch = [&](int j) {
          const int p = (first + j) * kBlock + t, pi = page_index(a.c, p);
          at = p - pi * a.c.page_size;
          // (what lies before the window may be in a page that was given back)
          seen = p >= w.g.pbegin && p < w.g.pend;
          pg = -1;
          if (seen && pi < a.c.max_pages) pg = row[pi];
        };
        fetch(0);
        constexpr int kElt = kE4m3 ? 1 : 2, kCh = D * kElt / 16, kPer = kLoaders / kCh;  // 16-byte chunks of a position
        const int c = t % kCh, r0 = t / kCh;
        const uint8_t* kb = static_cast<const uint8_t*>(a.c.k) + static_cast<int64_t>(w.h) * a.c.head_stride * kElt + c * 16;
        const uint8_t* vb = static_cast<const uint8_t*>(a.c.v) + static_cast<int64_t>(w.h) * a.c.head_stride * kElt + c * 16;
        float k_sc = 0.f, v_sc = 0.f;
        long long place[kBlock / kPer];  // bytes, of this thread's rows
        auto publish = [&](int j) {      // of block j, and its scales
          const bool there = pg >= 0 && pg < a.c.num_pages;
          if (seen && !there) raise_error(err, PERSONA_DEV_ERR_PAGE);
          if (kE4m3) {
            k_sc = v_sc = 0.f;
            if (there) {
              const int64_t so = pg * a.c.scale_page_stride + (at >> a.c.scale_shift) + static_cast<int64_t>(w.h) * a.c.scale_head_stride;
              k_sc = a.c.k_scale[so];
              v_sc = a.c.v_scale[so];
            }
          }
          long long* const places = sh.at[n_at & 1];
          ++n_at;
          places[t] = there ? (pg * a.c.page_stride + at * a.c.pos_stride) * kElt : -1;
          named_sync(1, kLoaders);
          if (j + 1 < nb) fetch(j + 1);
#pragma unroll
          for (int i = 0; i < kBlock / kPer; ++i) place[i] = places[r0 + i * kPer];
        };
        publish(0);
        if constexpr (!kE4m3) {
          for (int j = 0; j < nb; ++j) {
            const int st = n_k % kSt;
            const uint32_t parity = (n_k / kSt - 1) & 1;
            for (int kv = 0; kv < 2; ++kv) {
              if (n_k >= kSt) ok = ok && acquire(kv == 0 ? &sh.k_empty[st] : &sh.v_empty[st], parity);
              if (!ok) continue;
              const uint8_t* src = kv == 0 ? kb : vb;
              const uint32_t slot = (kv == 0 ? s_k : s_v) + st * C::kSlot;
#pragma unroll
              for (int i = 0; i < kBlock / kPer; ++i) {
                const int r = r0 + i * kPer;
                cp_async16(slot + (c >> 3) * C::kHalfBytes + r * 128 + (((c & 7) ^ (r & 7)) << 4),
                           src + (place[i] < 0 ? 0 : place[i]), place[i] >= 0);
              }
              issued(kv == 0 ? &sh.k_full[st] : &sh.v_full[st]);
            }
            ++n_k;
            if (j + 1 < nb) publish(j + 1);
          }
        } else {
          // Codes go through registers: while one tile's are converted and
          // stored, the next tile's (k, v, the next block's k, ...) are loaded
          // into the registers that this frees.
          uint4 x[kBlock / kPer];
          auto load = [&](int i, const uint8_t* src) {
            x[i] = place[i] >= 0 ? __ldg(reinterpret_cast<const uint4*>(src + place[i])) : make_uint4(0u, 0u, 0u, 0u);
          };
          auto convert = [&](uint32_t slot, const uint8_t* next) {
#pragma unroll
            for (int i = 0; i < kBlock / kPer; ++i) {
              const int r = r0 + i * kPer;
              const uint32_t u[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
              if (next != nullptr) load(i, next);
#pragma unroll
              for (int y = 0; y < 2; ++y) {
                const int cc = 2 * c + y;
                uint32_t hh[4];
                e4m3x4_to_half(u[2 * y], hh[0], hh[1]);
                e4m3x4_to_half(u[2 * y + 1], hh[2], hh[3]);
                asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(
                                 slot + (cc >> 3) * C::kHalfBytes + r * 128 + (((cc & 7) ^ (r & 7)) << 4)),
                             "r"(hh[0]), "r"(hh[1]), "r"(hh[2]), "r"(hh[3])
                             : "memory");
              }
            }
          };
#pragma unroll
          for (int i = 0; i < kBlock / kPer; ++i) load(i, kb);
          for (int j = 0; j < nb; ++j) {
            const int st = n_k % kSt;
            const uint32_t parity = (n_k / kSt - 1) & 1;
            if (n_k >= kSt) ok = ok && acquire(&sh.k_empty[st], parity);
            if (ok) {
              const int sc = n_k % C::kScales;
              const float vs = fmaxf(v_sc, kLeastScale);
              sh.ks[sc][t] = k_sc;
              sh.lv[sc][t] = log2_approx(vs);
              sh.rv[sc][t] = rcp_approx(vs);
              convert(s_k + st * C::kSlot, vb);
              flush();
              tc::fence_proxy_async();
              mbar_arrive(&sh.k_full[st]);
            }
            if (j + 1 < nb) publish(j + 1);
            if (n_k >= kSt) ok = ok && acquire(&sh.v_empty[st], parity);
            if (ok) {
              convert(s_v + st * C::kSlot, j + 1 < nb ? kb : nullptr);
              tc::fence_proxy_async();
              mbar_arrive(&sh.v_full[st]);
            }
            ++n_k;
          }
        }
      }
      flush();
    }
  } else {
    // ---------------------------------------------------------------- MMA --
    regs_dec<kRegsMma>();
    if (warp == 12 && works) {
      const bool one = tc::elect_one();
      const uint32_t tm = tc::uniform(tmem);
      constexpr uint32_t kFmt = std::is_same<PT, __nv_bfloat16>::value ? 1u : 0u;
      constexpr uint32_t kIdescS = tc::idesc_f16(kFmt, 128, kBlock);
      constexpr uint32_t kIdescO = tc::idesc_f16(kFmt, 128, D) | tc::kIdescBMnMajor;
      int n_k = 0, n_q = 0, n_p[2] = {0, 0};
      bool ok = true;
      auto wait = [&](uint64_t* bar, int n) {
        if (ok && !mbar_wait_abortable(bar, n & 1, err, abort)) ok = false;
        if (ok) tc::fence_after_sync();
        return ok;
      };
      // Descriptors differ in the start address alone (bits 0-13, units of 16
      // bytes, below 2^14 for any shared address): the rest is added once.
      const uint32_t dq = tc::uniform(static_cast<uint32_t>(tc::smem_desc(s_q, 1024, tc::kLayoutSw128)));
      const uint32_t dk = tc::uniform(static_cast<uint32_t>(tc::smem_desc(s_k, 1024, tc::kLayoutSw128)));
      const uint32_t dv = tc::uniform(static_cast<uint32_t>(tc::smem_desc_mn128(s_v, C::kHalfBytes, 1024)));
      const uint32_t hk = static_cast<uint32_t>(tc::smem_desc(s_k, 1024, tc::kLayoutSw128) >> 32);
      const uint32_t hv = static_cast<uint32_t>(tc::smem_desc_mn128(s_v, C::kHalfBytes, 1024) >> 32);
      auto mma_s = [&](int half, uint32_t st) {  // S = Q K^T
        if (one) {
          const uint32_t q = dq + half * (C::kSlot >> 4), k = dk + st * (C::kSlot >> 4);
#pragma unroll
          for (int ks = 0; ks < D / 16; ++ks) {
            constexpr int kHalf16 = C::kHalfBytes >> 4;
            const int in = (ks >> 2) * kHalf16 + (ks & 3) * 2;
            tc::mma_f16_lo(tm + half * 128, q, k, hk, in, kIdescS, ks > 0 ? 1u : 0u);
          }
          tc::commit(&sh.s_full[half]);
        }
      };
      auto mma_o = [&](int half, uint32_t st, bool first) {  // O += P V, as the halves of P come
        if (!wait(&sh.p_ready[half], n_p[half])) return;
        const uint32_t v = dv + st * (C::kSlot >> 4);
        if (one) {
#pragma unroll
          for (int ks = 0; ks < 2 * kFirstPart; ++ks)
            tc::mma_f16_ts_lo(tm + 256 + half * D, tm + half * 128, ks * 8, v, hv, ks * (2048 >> 4), kIdescO,
                              first && ks == 0 ? 0u : 1u);
        }
        if (!wait(&sh.p_rest[half], n_p[half]++)) return;
        if (one) {
#pragma unroll
          for (int ks = 2 * kFirstPart; ks < 8; ++ks)
            tc::mma_f16_ts_lo(tm + 256 + half * D, tm + half * 128, ks * 8, v, hv, ks * (2048 >> 4), kIdescO, 1u);
          tc::commit(&sh.pv_done[half]);
        }
      };
      Walk w(a, lead, sh.b, sh.tile, sh.off, u1 - u0);
      while (ok && w.next()) {
        const int nb = w.blocks();
        if (nb == 0) continue;
        const bool two = w.has_b();
        if (!wait(&sh.q_full, n_q)) break;
        if (!wait(&sh.k_full[n_k % kSt], n_k / kSt)) break;
        const uint32_t st0 = tc::uniform(n_k % kSt);
        mma_s(0, st0);
        if (two) mma_s(1, st0);
        if (one) {
          tc::commit(&sh.k_empty[n_k % kSt]);
          if (nb == 1) tc::commit(&sh.q_empty);
        }
        for (int j = 0; j < nb; ++j) {
          const uint32_t st = tc::uniform(n_k % kSt), nst = tc::uniform((n_k + 1) % kSt);
          const bool more = j + 1 < nb;
          if (!wait(&sh.v_full[st], n_k / kSt)) break;
          if (more && !wait(&sh.k_full[nst], (n_k + 1) / kSt)) break;
          mma_o(0, st, j == 0);
          if (!ok) break;
          // S of the next block may be written over P: the tensor cores take
          // the products in the order of their issue
          if (more) mma_s(0, nst);
          if (two) {
            mma_o(1, st, j == 0);
            if (!ok) break;
          }
          if (one) tc::commit(&sh.v_empty[st]);
          if (more) {
            if (two) mma_s(1, nst);
            if (one) {
              tc::commit(&sh.k_empty[nst]);
              if (j + 2 == nb) tc::commit(&sh.q_empty);
            }
          }
          ++n_k;
        }
        ++n_q;
      }
      if (!ok && one) {  // gave up: nothing of ours may be under way when the memory goes
        tc::commit(&sh.drained);
        mbar_wait(&sh.drained, 0, err);
      }
    }
    __syncwarp();
  }
  // ---- end: every product has been waited for by its softmax rows ----
  tc::fence_before_sync();
  __syncthreads();
  if (warp == 12) {
    tc::fence_after_sync();
    tc::tmem_dealloc(tmem, 512);
  }
}

// Joins the pieces of one cut tile, which lie four columns by four: CTA (c, y)
// looks after rows [32 y, 32 y + 32) of the tile whose first piece CTA c left;
// a lane is a row, a warp an eighth of the columns.  Pieces in order.
template <typename T, int D>
__global__ void __launch_bounds__(256) paged_chunk_join_kernel(const __grid_constant__ PagedAttention a) {
  pdl_wait();
  pdl_launch();
  const int4 d = a.desc[2 * blockIdx.x];
  const int r = blockIdx.y * 32 + (threadIdx.x & 31);
  if (static_cast<int>(blockIdx.y) * 32 >= d.w) return;
  const int4 e = a.desc[2 * blockIdx.x + 1];
  constexpr int kF = Part<kTile, D>::kFloats, kV = D / 8;
  const int first = blockIdx.x, pieces = d.y - first + 1, c0 = (threadIdx.x >> 5) * kV;
  auto piece = [&](int i) { return a.part + static_cast<int64_t>(i == 0 ? d.x : 2 * (first + i)) * kF; };
  float mx = kNegInf, l = 0.f, o[kV];
#pragma unroll
  for (int x = 0; x < kV; ++x) o[x] = 0.f;
#pragma unroll 4
  for (int i = 0; i < pieces; ++i) mx = fmaxf(mx, piece(i)[kTile * D + r]);
  const float neg = mx == kNegInf ? 0.f : -mx;  // a row that saw nothing: weights of 0
#pragma unroll 2
  for (int i = 0; i < pieces; ++i) {
    const float* p = piece(i);
    const float f = exp2_approx(p[kTile * D + r] + neg);
    l = fmaf(f, p[kTile * D + kTile + r], l);
#pragma unroll
    for (int x = 0; x < kV; x += 4) {
      const float4 v = *reinterpret_cast<const float4*>(p + (c0 + x) * kTile + 4 * r);
      o[x] = fmaf(f, v.x, o[x]);
      o[x + 1] = fmaf(f, v.y, o[x + 1]);
      o[x + 2] = fmaf(f, v.z, o[x + 2]);
      o[x + 3] = fmaf(f, v.w, o[x + 3]);
    }
  }
  if (r >= d.w) return;
  const float inv = l > 0.f ? 1.f / l : 0.f;
  const int mm = d.z + r, tok = mm / a.G;
  T* dst = static_cast<T*>(a.out.p) + static_cast<int64_t>(e.x + tok) * a.out.row_stride +
           static_cast<int64_t>(e.y * a.G + mm - tok * a.G) * a.out.head_stride + c0;
#pragma unroll
  for (int x = 0; x < kV; x += 8)
    *reinterpret_cast<uint4*>(dst + x) =
        make_uint4(Mma<T>::pack(o[x] * inv, o[x + 1] * inv), Mma<T>::pack(o[x + 2] * inv, o[x + 3] * inv),
                   Mma<T>::pack(o[x + 4] * inv, o[x + 5] * inv), Mma<T>::pack(o[x + 6] * inv, o[x + 7] * inv));
}

template <typename T, int D, bool kE4m3>
cudaError_t chunk_launch(const PagedAttention& a, cudaStream_t st) {
  auto k = paged_chunk_kernel<T, D, kE4m3>;
  static std::atomic<bool> done[64];
  // the register split above draws on kRegsLaunch registers a thread
  cudaError_t e = prepare_kernel(done, k, Cfg<D>::kSmem, kRegsLaunch);
  if (e != cudaSuccess) return e;
  const int ctas = sm_count();
  e = launch_paged(k, dim3(ctas), dim3(kThreads), Cfg<D>::kSmem, 1, false, st, a);
  if (e != cudaSuccess) return e;
  return launch_paged(paged_chunk_join_kernel<T, D>, dim3(ctas, kTile / 32), dim3(256), 0, 1, true, st, a);
}
template <typename T>
cudaError_t chunk_for(const PagedAttention& a, cudaStream_t st) {
  const bool e = a.c.k_scale != nullptr;
  if (a.c.D == 128) return e ? chunk_launch<T, 128, true>(a, st) : chunk_launch<T, 128, false>(a, st);
  return e ? chunk_launch<T, 64, true>(a, st) : chunk_launch<T, 64, false>(a, st);
}

}  // namespace

size_t paged_chunk_ws_bytes(int D) {
  const size_t ctas = sm_count();
  return ctas * 2 * sizeof(int4) + ctas * 2 * (kTile * static_cast<size_t>(D) + 2 * kTile) * sizeof(float);
}

cudaError_t launch_paged_chunk(PagedAttention a, int dtype, void* workspace, cudaStream_t st) {
  a.desc = static_cast<int4*>(workspace);
  a.part = reinterpret_cast<float*>(static_cast<char*>(workspace) + sm_count() * 2 * sizeof(int4));
  return dtype == PERSONA_DTYPE_BF16 ? chunk_for<__nv_bfloat16>(a, st) : chunk_for<__half>(a, st);
}

}  // namespace persona
