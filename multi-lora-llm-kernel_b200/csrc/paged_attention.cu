// Causal attention of each sequence's new tokens over its paged KV cache, for
// few query rows per kv head: single tokens and drafted ones.
//
//   out[r, h] = sum_j p_j v[j, h / G],  p = softmax_j(scale q[r, h] . k[j, h / G])
//
// over the positions j <= pos(r) (and j > pos(r) - window).  At these sizes
// the kernel is bound by the pages it has to read once.
//
// Work.  A tile is TR = 16 MT query rows (token, head of the group) that
// share a kv head; a unit is 64 positions of one tile's keys.  The units of
// all tiles lie in one line (sequence, tile, kv head, position), which is cut
// into equal ranges, one per CTA, so lengths may differ as they like.  A
// range that starts or ends inside a tile's units leaves a piece (running
// maximum, sum and unnormalised output, fp32) that paged_combine_kernel
// joins, always in the order of the positions.  Small batches take a cluster
// per tile instead, whose CTAs hold equal parts of its units and join them
// through distributed shared memory, in one launch.
//
// Measured (32 heads over 8, D = 128, a call among others): 64 sequences of 500
// to 8192 positions, bf16, 119 us, 0.90 of the measured HBM rate; over 8-bit
// pages 100 us, 0.55 of it.  32 x 5 drafted tokens over 300 to 6000 positions of
// 16-bit pages 67 us, 0.64; of 8-bit ones 70 us, 0.32: no unit is full there
// (issue slots 37 %, tensor 25 %, exponentials 10 %).  An SM's registers hold
// eight warps, two per scheduler, too few to cover the latency of each one's
// chain of loads, conversions, products and exponentials; and of the products'
// 32 rows 12 are not there (20 rows; with one token 12 of 16).
//
// A CTA.  Four warps; warp w takes positions [16 w, 16 w + 16) of every unit
// through a ring of its own shared memory filled with cp.async, so no warp
// waits for another inside a piece: scores by mma.sync m16n8k16 (q fragments
// in registers), one pass with a running maximum per row, and the
// probabilities, rounded to 16 bits, go from the accumulators' layout
// straight into the operand's for the second product.  The warps' results
// are joined in shared memory at the end of a piece.
//
// 8-bit pages.  The codes become fp16 in registers, exactly, and the products
// run in fp16 for either type of q (a bf16 row is first scaled by a power of
// two into fp16's range).  The k scale multiplies the fp32 score.  The v scale
// goes into the exponent: the running maximum is taken over x + log2(vs), so
// that p vs is at most 2^kGrow whatever the scales' range, and the sum of p is
// accumulated as (p vs) / vs.  Scales are not negative; a v scale below
// kLeastScale counts as that.
//
// mma.sync, not tcgen05: a tile has 16 or 32 rows, a quarter or half of
// tcgen05's smallest M (64), and the tensor work per byte of pages is far below
// what the warp-level product delivers.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cooperative_groups.h>

#include "paged_attention.cuh"

namespace persona {
namespace cg = cooperative_groups;
namespace {

constexpr int kWarps = 4, kThreads = 32 * kWarps;
constexpr int kPos = 16;              // positions of one warp step
constexpr int kUnit = kPos * kWarps;  // positions of one unit
// What starting and ending a tile costs, in units: so many stand before its
// first one in the line.  None where every unit has a CTA of its own.
constexpr int kPieceUnits = 3;

__device__ __forceinline__ void ldsm_x4_trans(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
// Units of one tile (the same for all tiles of a sequence; a tile that ends
// before the sequence does leaves its last ones empty) and the first one.
__device__ __forceinline__ void seq_units(const Seq& s, int window, int TR, int G, int& tiles, int& first, int& per) {
  tiles = (s.n * G + TR - 1) / TR;
  const int ctx = s.len - s.n;
  const int begin = window > 0 ? max(0, ctx + 1 - window) : 0;
  first = begin / kUnit;
  per = max(1, (s.len + kUnit - 1) / kUnit - first);
}

// Shared memory of the ring, which also holds the warps' results at a piece's end.
template <int D, int MT, bool kE4m3, int kStages> struct RingBytes {
  static constexpr int kSlot = 2 * kPos * D * (kE4m3 ? 1 : 2) + (kE4m3 ? 2 * kPos * 4 : 0);
  static constexpr int kRing = kWarps * kStages * kSlot, kWarpOut = kWarps * 16 * MT * D * 4;
  static constexpr int kJoin = kWarpOut + 16 * MT * D * 4;  // the warps' results, and a cluster's share of them
  static constexpr int kBytes = kRing > kJoin ? kRing : kJoin;
};

template <typename T, int D, int MT, bool kE4m3, int kStages, bool kCluster>
__global__ void __launch_bounds__(kThreads) paged_attention_kernel(const __grid_constant__ PagedAttention a) {
  using MT16 = typename std::conditional<kE4m3, __half, T>::type;  // type of the products
  constexpr int TR = 16 * MT;
  constexpr int kElt = kE4m3 ? 1 : 2;
  constexpr int kRowBytes = D * kElt;                  // one position in a ring slot
  constexpr int kChunks = kRowBytes / 16;
  constexpr int kHalf = kPos * kRowBytes;              // k (or v) of one warp step
  constexpr int kSlot = 2 * kHalf + (kE4m3 ? 2 * kPos * 4 : 0);
  constexpr int kSteps = D / 16;
  constexpr int kQAt = RingBytes<D, MT, kE4m3, kStages>::kBytes;  // q fragments behind the ring (MT = 2)
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ long long s_scan[kWarps], s_items[kWarps], s_begin;
  __shared__ int s_b;
  __shared__ long long s_off, s_end;
  __shared__ float s_m[kWarps][TR], s_l[kWarps][TR];
  __shared__ float s_cm[kCluster ? TR : 1], s_cl[kCluster ? TR : 1];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, t = lane & 3;
  const int cta = blockIdx.x;
  const int Hkv = a.c.Hkv, G = a.G;
  pdl_wait();
  pdl_launch();

  // ---- this CTA's range of units ----
  // A cluster takes one tile after another and cuts each into equal parts;
  // otherwise the CTA has a range of the line of all units.
  const int split = kCluster ? a.split : 1, rank = kCluster ? cta % split : 0;
  const int index = cta / split;  // cluster: sequence, first tile, kv head
  int b = kCluster ? index / (Hkv * a.tile_step) : 0, next_tile = kCluster ? index / Hkv % a.tile_step : 0;
  int lead = 0, ctas = 0;
  long long total = 0, u1 = 0, off = 0, left = 0;
  if constexpr (!kCluster) {
    auto count = [&](int b, int& per) -> int {  // tiles times heads, units of each
      if (b >= a.c.B) return 0;
      int tiles, first;
      seq_units(load_seq(a, b), a.window, TR, G, tiles, first, per);
      return tiles * Hkv;
    };
    long long items = 0;
    int my_items = 0, my_per = 0;
    for (int b0 = 0; b0 < a.c.B; b0 += kThreads) {
      int per = 0;
      const int n = count(b0 + tid, per);
      if (b0 == 0) {
        my_items = n;
        my_per = per;
      }
      long long u = static_cast<long long>(n) * per, v = n;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        u += __shfl_xor_sync(0xffffffffu, u, o);
        v += __shfl_xor_sync(0xffffffffu, v, o);
      }
      if (lane == 0) {
        s_scan[warp] = u;
        s_items[warp] = v;
      }
      __syncthreads();
      for (int w = 0; w < kWarps; ++w) {
        total += s_scan[w];
        items += s_items[w];
      }
      __syncthreads();
    }
    lead = total <= gridDim.x ? 0 : kPieceUnits;
    total += lead * items;
    if (tid == 0) a.desc[2 * cta] = make_int4(0, 0, 0, 0);
    // no more CTAs than units, so that every range (before the move below) has one
    ctas = static_cast<int>(min(total, static_cast<long long>(gridDim.x)));
    if (cta >= ctas) return;
    // a cut inside what a tile costs to start is moved before it
    const long long raw0 = total * cta / ctas, raw1 = total * (cta + 1) / ctas;
    auto start_of = [&](long long off, int per) {
      const int k = static_cast<int>(off % per);
      return k < lead ? off - k : off;
    };
    if (tid == 0) {
      s_b = 0;
      s_off = 0;
      s_begin = s_end = raw1;
    }
    {
      long long run = 0;
      for (int b0 = 0; b0 < a.c.B && run <= raw1; b0 += kThreads) {
        int per = my_per;
        const int n = b0 == 0 ? my_items : count(b0 + tid, per);
        per += lead;
        const long long u = static_cast<long long>(n) * per;
        long long inc = u;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const long long up = __shfl_up_sync(0xffffffffu, inc, o);
          if (lane >= o) inc += up;
        }
        if (lane == 31) s_scan[warp] = inc;
        __syncthreads();
        long long lo = run + inc - u;
        for (int w = 0; w < warp; ++w) lo += s_scan[w];
        if (raw0 >= lo && raw0 < lo + u) {
          s_b = b0 + tid;
          s_off = start_of(raw0 - lo, per);
          s_begin = lo + s_off;
        }
        if (raw1 >= lo && raw1 < lo + u) s_end = lo + start_of(raw1 - lo, per);
        for (int w = 0; w < kWarps; ++w) run += s_scan[w];
        __syncthreads();
      }
    }
    u1 = s_end;
    if (s_begin >= u1) return;
    b = s_b;
    off = s_off;
    left = u1 - s_begin;
  }
  bool first_piece = true;
  const uint32_t ring = smem_u32(smem) + warp * kStages * kSlot;

  Seq seq = load_seq(a, b);
  int tiles, kfirst, per;
  seq_units(seq, a.window, TR, G, tiles, kfirst, per);
  per += lead;
  while (true) {
    int item, k0, k1;
    if constexpr (kCluster) {
      if (next_tile >= tiles) break;
      item = next_tile * Hkv + index % Hkv;
      next_tile += a.tile_step;
      k0 = per * rank / split;
      k1 = per * (rank + 1) / split;
    } else {
      if (left <= 0) break;
      while (off >= static_cast<long long>(tiles) * per * Hkv) {  // the next sequence with units
        off -= static_cast<long long>(tiles) * per * Hkv;
        if (++b >= a.c.B) return;  // the arrays changed under the call
        seq = load_seq(a, b);
        seq_units(seq, a.window, TR, G, tiles, kfirst, per);
        per += lead;
      }
      item = static_cast<int>(off / per);
      k0 = static_cast<int>(off - static_cast<long long>(item) * per);
      k1 = static_cast<int>(min(static_cast<long long>(per), k0 + left));
    }
    const int tile = item / Hkv, h = item - tile * Hkv;
    const int ctx = seq.len - seq.n;
    const int m0 = tile * TR, mrows = min(TR, seq.n * G - m0);
    const int tok0 = m0 / G, tok1 = (m0 + mrows - 1) / G;  // first and last token of the tile
    const int pend = max(0, min(seq.len, ctx + tok1 + 1));  // keys of the tile end here
    const int pbegin = a.window > 0 ? max(0, ctx + tok0 + 1 - a.window) : 0;
    // positions of the steps of this piece that have any key
    const int p_lo = max((kfirst + max(k0 - lead, 0)) * kUnit, pbegin / kUnit * kUnit);
    const int p_hi = min((kfirst + max(k1 - lead, 0)) * kUnit, pend);
    const int steps = p_hi > p_lo ? (p_hi - p_lo + kUnit - 1) / kUnit : 0;

    // ---- loads ----
    const int32_t* const pages = a.c.table + b * a.c.table_stride;
    auto page_of = [&](int p, int& at) {
      const int pi = page_index(a.c, p);
      at = p - pi * a.c.page_size;
      const int pg = pi < a.c.max_pages ? pages[pi] : -1;
      if (pg >= 0 && pg < a.c.num_pages) return pg;
      raise_error(a.err, PERSONA_DEV_ERR_PAGE);
      return -1;
    };
    const uint8_t* kb = static_cast<const uint8_t*>(a.c.k) + static_cast<int64_t>(h) * a.c.head_stride * kElt;
    const uint8_t* vb = static_cast<const uint8_t*>(a.c.v) + static_cast<int64_t>(h) * a.c.head_stride * kElt;
    const bool whole = a.c.page_size % kPos == 0;  // a step's positions share a page
    constexpr int kRowsPer = 32 / kChunks;
    const int ch = lane % kChunks, lr = lane / kChunks;  // this lane's chunk, and its row among kRowsPer
    const uint8_t* const kl = kb + lr * a.c.pos_stride * kElt + ch * 16;
    const uint8_t* const vl = vb + lr * a.c.pos_stride * kElt + ch * 16;
    const int64_t row_step = kRowsPer * a.c.pos_stride * kElt;
    const float* const sl = kE4m3 ? (lane < 16 ? a.c.k_scale : a.c.v_scale) + static_cast<int64_t>(h) * a.c.scale_head_stride : nullptr;
    // 16-byte chunks are XORed by the row so that the fragment reads below touch
    // every bank once (8-bit: k reads two rows of four chunks, v reads even rows
    // of two chunks, per quarter warp).  A lane's row is lr plus a multiple of
    // kRowsPer, whose bits do not meet.
    constexpr int kMask = kChunks - 1;
    const int ck0 = kE4m3 ? ch ^ ((lr & 1) << 2) : ch ^ (lr & 7), cv0 = kE4m3 ? ch ^ (((lr >> 1) & 3) << 1) : ck0;
    // Where a step's positions share a page, the pages of 32 steps are read at
    // once, one a lane.
    int pages32 = -1;
    auto load = [&](int s) {
      const int p0 = p_lo + s * kUnit + warp * kPos;
      const uint32_t dst = ring + (s % kStages) * kSlot;
      if (whole) {
        if ((s & 31) == 0) {
          const int p = p0 + lane * kUnit, pi = page_index(a.c, p);
          pages32 = p < pend && pi < a.c.max_pages ? pages[pi] : -1;
        }
        const int pg = __shfl_sync(0xffffffffu, pages32, s & 31);
        // positions of this step: those from `skip` on, `rem` of them (what lies
        // before the window may be in a page that was given back)
        const int skip = max(pbegin - p0, 0);
        int rem = min(pend - p0, kPos) - skip;
        if (rem > 0 && (pg < 0 || pg >= a.c.num_pages)) {
          raise_error(a.err, PERSONA_DEV_ERR_PAGE);
          rem = 0;
        }
        rem = max(rem, 0);
        const int lrs = lr - skip;
        const int at = p0 - page_index(a.c, p0) * a.c.page_size;
        const int64_t base = rem > 0 ? (pg * a.c.page_stride + at * a.c.pos_stride) * kElt : 0;
        const uint8_t *kp = kl + base, *vp = vl + base;
#pragma unroll
        for (int i = 0; i < kPos / kRowsPer; ++i, kp += row_step, vp += row_step) {
          constexpr int kStep = kRowsPer;
          const int ck = kE4m3 ? ck0 : ck0 ^ ((i * kStep) & 7), cv = kE4m3 ? cv0 ^ (((i * kStep / 2) & 3) << 1) : ck;
          const bool live = static_cast<uint32_t>(lrs + i * kStep) < static_cast<uint32_t>(rem);
          const uint32_t to = dst + (lr + i * kStep) * kRowBytes;
          cp_async16(to + (ck & kMask) * 16, live ? kp : kl, live);
          cp_async16(to + kHalf + (cv & kMask) * 16, live ? vp : vl, live);
        }
        if (kE4m3) {
          const int r = lane & 15;
          const bool live = static_cast<uint32_t>(r - skip) < static_cast<uint32_t>(rem);
          cp_async4(dst + 2 * kHalf + lane * 4, live ? sl + (pg * a.c.scale_page_stride + at + r) : sl, live);
        }
      } else {
#pragma unroll
        for (int i = 0; i < kPos / kRowsPer; ++i) {
          const int r = lr + i * kRowsPer;
          const int ck = kE4m3 ? ck0 : ck0 ^ ((i * kRowsPer) & 7), cv = kE4m3 ? cv0 ^ (((i * kRowsPer / 2) & 3) << 1) : ck;
          int at = 0;
          const int pg = p0 + r >= pbegin && p0 + r < pend ? page_of(p0 + r, at) : -1;
          const bool live = pg >= 0;
          const int64_t src = live ? (pg * a.c.page_stride + at * a.c.pos_stride) * kElt : 0;
          const uint32_t to = dst + r * kRowBytes;
          cp_async16(to + (ck & kMask) * 16, kb + src + ch * 16, live);
          cp_async16(to + kHalf + (cv & kMask) * 16, vb + src + ch * 16, live);
        }
        if (kE4m3) {
          const int p = p0 + (lane & 15);
          int at = 0;
          const int pg = p >= pbegin && p < pend ? page_of(p, at) : -1;
          cp_async4(dst + 2 * kHalf + lane * 4, pg >= 0 ? sl + (pg * a.c.scale_page_stride + at) : sl, pg >= 0);
        }
      }
    };
#pragma unroll
    for (int s = 0; s < kStages - 1; ++s) {
      if (s < steps) load(s);
      cp_commit();
    }

    // ---- q fragments ----
    // 16-bit pages: the operand's own order of d.  8-bit pages: a lane reads
    // 16 consecutive codes of k, [64 blk + 16 t, ...), so step (blk, s) takes
    // d = 64 blk + 16 t + 4 s + {0, 1} and {2, 3} where the operand has
    // k = 2 t + {0, 1} and 2 t + 8 + {0, 1}.
    uint32_t qf[MT][kSteps][4];
    float qmul[MT][2];
    int hi_pos[MT][2];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int m = mt * 16 + half * 8 + g;
        const bool live = m < mrows;
        const int mm = m0 + (live ? m : 0);
        const int tok = mm / G, hg = mm - tok * G;
        const T* qp = static_cast<const T*>(a.q.p) + static_cast<int64_t>(seq.row0 + tok) * a.q.row_stride +
                      static_cast<int64_t>(h * G + hg) * a.q.head_stride;
        hi_pos[mt][half] = live ? ctx + tok : -1;
        qmul[mt][half] = a.scale_log2;
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
          if (!kE4m3) {
            qf[mt][s][half] = live ? *reinterpret_cast<const uint32_t*>(qp + 16 * s + 2 * t) : 0u;
            qf[mt][s][half + 2] = live ? *reinterpret_cast<const uint32_t*>(qp + 16 * s + 8 + 2 * t) : 0u;
          } else {
            const int d = 64 * (s / 4) + 16 * t + 4 * (s % 4);
            const uint2 w = live ? *reinterpret_cast<const uint2*>(qp + d) : make_uint2(0u, 0u);
            qf[mt][s][half] = w.x;
            qf[mt][s][half + 2] = w.y;
          }
        }
        if (kE4m3 && !std::is_same<T, __half>::value) {
          // bf16 row -> fp16: scaled by the power of two that brings its
          // largest element into [1, 2); elements 2^-24 below that vanish
          float mx = 0.f;
#pragma unroll
          for (int s = 0; s < kSteps; ++s)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              const float2 f = Cvt<T>::to2(qf[mt][s][half + 2 * x]);
              mx = fmaxf(mx, fmaxf(fabsf(f.x), fabsf(f.y)));
            }
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
          // exponent field of mx, kept where both powers are normal numbers
          const int e = min(max(static_cast<int>(__float_as_uint(mx) >> 23), 2), 252);
          const float down = __uint_as_float(static_cast<uint32_t>(254 - e) << 23);
          qmul[mt][half] = a.scale_log2 * __uint_as_float(static_cast<uint32_t>(e) << 23);
#pragma unroll
          for (int s = 0; s < kSteps; ++s)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              const float2 f = Cvt<T>::to2(qf[mt][s][half + 2 * x]);
              qf[mt][s][half + 2 * x] = Mma<__half>::pack(f.x * down, f.y * down);
            }
        }
      }

    // With two row tiles the fragments would take 64 registers beside 128 of
    // outputs: they go to shared memory, one 16-byte read a lane, row tile and step.
    const uint32_t s_qf = smem_u32(smem) + kQAt + lane * 16;
    if constexpr (MT == 2) {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int ks = 0; ks < kSteps; ++ks)
          if (ks / (kSteps / kWarps) == warp)
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(s_qf + (mt * kSteps + ks) * 512), "r"(qf[mt][ks][0]),
                         "r"(qf[mt][ks][1]), "r"(qf[mt][ks][2]), "r"(qf[mt][ks][3])
                         : "memory");
      __syncthreads();
    }
    auto q_of = [&](int mt, int ks, uint32_t (&f)[4]) {
      if constexpr (MT == 2) {
        const uint4 v = lds128(s_qf + (mt * kSteps + ks) * 512);
        f[0] = v.x;
        f[1] = v.y;
        f[2] = v.z;
        f[3] = v.w;
      } else {
#pragma unroll
        for (int x = 0; x < 4; ++x) f[x] = qf[mt][ks][x];
      }
    };

    // ---- one pass over the piece's positions ----
    float acc[MT][D / 8][4];
    float m_run[MT][2], l_run[MT][2];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
      for (int i = 0; i < D / 8; ++i)
#pragma unroll
        for (int x = 0; x < 4; ++x) acc[mt][i][x] = 0.f;
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        m_run[mt][x] = kNegInf;
        l_run[mt][x] = 0.f;
      }
    }
    const int full_hi = ctx + tok0;                                          // positions all rows see: <= this
    const int full_lo = a.window > 0 ? ctx + tok1 - a.window + 1 : 0;       // and >= this
    for (int s = 0; s < steps; ++s) {
      cp_wait<kStages - 2>();
      __syncwarp();
      if (s + kStages - 1 < steps) load(s + kStages - 1);
      cp_commit();
      const int p0 = p_lo + s * kUnit + warp * kPos;
      if (p0 >= pend) continue;
      const uint32_t slot = ring + (s % kStages) * kSlot;

      float sc[MT][2][4];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int x = 0; x < 4; ++x) sc[mt][n][x] = 0.f;
      if (!kE4m3) {
        const int r = (lane & 7) + ((lane >> 4) << 3);  // matrices 0, 1: rows 0-7; 2, 3: rows 8-15
        const uint32_t rowaddr = slot + r * kRowBytes;
#pragma unroll
        for (int ks = 0; ks < kSteps; ++ks) {
          const int ch = (2 * ks + ((lane >> 3) & 1)) ^ (r & 7);
          uint32_t kf[4];
          ldsm_x4(rowaddr + (ch & (kChunks - 1)) * 16, kf);
          const uint32_t b0[2] = {kf[0], kf[1]}, b1[2] = {kf[2], kf[3]};
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
            uint32_t f[4];
            q_of(mt, ks, f);
            Mma<MT16>::k16(sc[mt][0], f, b0);
            Mma<MT16>::k16(sc[mt][1], f, b1);
          }
        }
      } else {
#pragma unroll
        for (int blk = 0; blk < D / 64; ++blk) {
          uint32_t u[2][4];
#pragma unroll
          for (int n = 0; n < 2; ++n) {
            const int r = n * 8 + g;
            const uint4 w = lds128(slot + r * kRowBytes + (((4 * blk + t) ^ ((r & 1) << 2)) & (kChunks - 1)) * 16);
            u[n][0] = w.x;
            u[n][1] = w.y;
            u[n][2] = w.z;
            u[n][3] = w.w;
          }
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            uint32_t b0[2], b1[2];
            e4m3x4_to_half(u[0][x], b0[0], b0[1]);
            e4m3x4_to_half(u[1][x], b1[0], b1[1]);
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
              uint32_t f[4];
              q_of(mt, 4 * blk + x, f);
              Mma<MT16>::k16(sc[mt][0], f, b0);
              Mma<MT16>::k16(sc[mt][1], f, b1);
            }
          }
        }
      }

      // scores in the log2 domain, masked
      float lv[2][2], rv[2][2];
      if (kE4m3) {
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          const uint32_t sa = slot + 2 * kHalf + (8 * n + 2 * t) * 4;
          float ks2[2] = {__uint_as_float(lds32(sa)), __uint_as_float(lds32(sa + 4))};
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const float vs = fmaxf(__uint_as_float(lds32(sa + kPos * 4 + 4 * x)), kLeastScale);
            lv[n][x] = log2_approx(vs);
            rv[n][x] = rcp_approx(vs);
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
              sc[mt][n][x] *= ks2[x];
              sc[mt][n][2 + x] *= ks2[x];
            }
          }
        }
      }
      const bool need_mask = p0 + kPos - 1 > full_hi || p0 < full_lo;
      bool grow = false;
      float m_new[MT][2];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          float mx = kNegInf;
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              float& v = sc[mt][n][2 * half + x];
              v = kE4m3 ? fmaf(v, qmul[mt][half], lv[n][x]) : v * a.scale_log2;
              if (need_mask) {
                const int p = p0 + 8 * n + 2 * t + x;
                const bool seen = p <= hi_pos[mt][half] && (a.window == 0 || p > hi_pos[mt][half] - a.window);
                v = seen ? v : kNegInf;
              }
              mx = fmaxf(mx, v);
            }
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
          // the maximum moves at the first key and when outgrown by 2^8
          const bool up = mx > (m_run[mt][half] == kNegInf ? kNegInf : m_run[mt][half] + kGrow);
          m_new[mt][half] = up ? mx : m_run[mt][half];
          grow |= up;
        }
      if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          float f[2];
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            f[half] = m_new[mt][half] != m_run[mt][half] ? exp2_approx(m_run[mt][half] - m_new[mt][half]) : 1.f;
            l_run[mt][half] *= f[half];
            m_run[mt][half] = m_new[mt][half];
          }
#pragma unroll
          for (int i = 0; i < D / 8; ++i) {
            acc[mt][i][0] *= f[0];
            acc[mt][i][1] *= f[0];
            acc[mt][i][2] *= f[1];
            acc[mt][i][3] *= f[1];
          }
        }
      }
      uint32_t pf[MT][4];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const float mm = m_run[mt][half] == kNegInf ? 0.f : m_run[mt][half];
#pragma unroll
          for (int n = 0; n < 2; ++n) {
            const float e0 = exp2_approx(sc[mt][n][2 * half] - mm), e1 = exp2_approx(sc[mt][n][2 * half + 1] - mm);
            l_run[mt][half] += kE4m3 ? fmaf(e0, rv[n][0], e1 * rv[n][1]) : e0 + e1;
            // 16 bits for the product: half a step, 2^-11 (fp16) or 2^-8
            // (bf16) of a weight, the precision of v itself
            pf[mt][half + 2 * n] = Mma<MT16>::pack(e0, e1);
          }
        }

      // ---- P V ----
      const uint32_t vslot = slot + kHalf;
      if (!kE4m3) {
        const int r = (lane & 7) + (((lane >> 3) & 1) << 3);  // matrices 0, 2: positions 0-7; 1, 3: 8-15
        const uint32_t rowaddr = vslot + r * kRowBytes;
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
          const int ch = (2 * i + (lane >> 4)) ^ (r & 7);
          uint32_t vf[4];
          ldsm_x4_trans(rowaddr + (ch & (kChunks - 1)) * 16, vf);
          const uint32_t b0[2] = {vf[0], vf[1]}, b1[2] = {vf[2], vf[3]};
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
            Mma<MT16>::k16(acc[mt][2 * i], pf[mt], b0);
            Mma<MT16>::k16(acc[mt][2 * i + 1], pf[mt], b1);
          }
        }
      } else {
        // A lane holds D / 8 consecutive dims, [g D / 8, ...), of positions
        // 2 t, 2 t + 1, 2 t + 8, 2 t + 9: column g of n-tile i is dim g D / 8 + i.
        constexpr int kW = D / 32;  // words of a lane and position
        uint32_t w[4][kW];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const int r = 2 * t + (x & 1) + 8 * (x >> 1);
          if (D == 128) {
            const uint4 v = lds128(vslot + r * kRowBytes + ((g ^ (((r >> 1) & 3) << 1)) & (kChunks - 1)) * 16);
            w[x][0] = v.x;
            w[x][1] = v.y;
            w[x][kW - 2] = v.z;
            w[x][kW - 1] = v.w;
          } else {
            const uint32_t ad = vslot + r * kRowBytes + (((g >> 1) ^ (((r >> 1) & 3) << 1)) & (kChunks - 1)) * 16 + (g & 1) * 8;
            w[x][0] = lds32(ad);
            w[x][1] = lds32(ad + 4);
          }
        }
#pragma unroll
        for (int j = 0; j < kW; ++j) {
          uint32_t bfr[4][2];
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            // bytes (p, p + 1) side by side, then two conversions of pairs
            const uint32_t ab = __byte_perm(w[2 * x][j], w[2 * x + 1][j], 0x5140);
            const uint32_t cd = __byte_perm(w[2 * x][j], w[2 * x + 1][j], 0x7362);
            e4m3x4_to_half(ab, bfr[0][x], bfr[1][x]);
            e4m3x4_to_half(cd, bfr[2][x], bfr[3][x]);
          }
#pragma unroll
          for (int x = 0; x < 4; ++x)
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) Mma<MT16>::k16(acc[mt][4 * j + x], pf[mt], bfr[x]);
        }
      }
      __syncwarp();
    }
    cp_wait<0>();
    __syncthreads();  // every warp is done with the ring, which now takes the warps' results

    // ---- join the warps ----
    float* accs = reinterpret_cast<float*>(smem);  // [kWarps][TR][D]
    // Where dim d of row m is: 8-dim chunks XORed by the row, or (8-bit pages,
    // whose lanes hold D / 8 dims in a row) those dims turned by row and lane.
    auto join_at = [&](int m, int d) {
      if (!kE4m3) return d ^ ((m & 7) << 3);
      constexpr int kW = D / 8;
      const int blk = d / kW;
      return blk * kW + ((d + 2 * (m & 7) + (blk >> 2)) & (kW - 1));
    };
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int m = mt * 16 + half * 8 + g;
        float l = l_run[mt][half];
        l += __shfl_xor_sync(0xffffffffu, l, 1);
        l += __shfl_xor_sync(0xffffffffu, l, 2);
        if (t == 0) {
          s_m[warp][m] = m_run[mt][half];
          s_l[warp][m] = l;
        }
        if (mt * 16 + half * 8 >= mrows) continue;  // no such rows
        float* dst = accs + (warp * TR + m) * D;
#pragma unroll
        for (int i = 0; i < D / 8; ++i) {
          const float x0 = acc[mt][i][2 * half], x1 = acc[mt][i][2 * half + 1];
          if (!kE4m3) {
            *reinterpret_cast<float2*>(dst + join_at(m, 8 * i + 2 * t)) = make_float2(x0, x1);
          } else {  // the odd lanes the other way round: 32 lanes, 32 banks
            const int a0 = join_at(m, 2 * t * (D / 8) + i), a1 = join_at(m, (2 * t + 1) * (D / 8) + i);
            dst[(t & 1) == 0 ? a0 : a1] = (t & 1) == 0 ? x0 : x1;
            dst[(t & 1) == 0 ? a1 : a0] = (t & 1) == 0 ? x1 : x0;
          }
        }
      }
    __syncthreads();
    const bool complete = !kCluster && k0 == 0 && k1 == per;
    float* const mine = reinterpret_cast<float*>(smem + RingBytes<D, MT, kE4m3, kStages>::kWarpOut);  // [TR][D], cluster
    float* part = a.part + static_cast<int64_t>(2 * cta + (first_piece ? 0 : 1)) * Part<TR, D>::kFloats;
    for (int i = tid; i < mrows * (D / 8); i += kThreads) {
      const int m = i / (D / 8), d = (i % (D / 8)) * 8;
      float mx = kNegInf;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) mx = fmaxf(mx, s_m[w][m]);
      float l = 0.f, o[8];
#pragma unroll
      for (int x = 0; x < 8; ++x) o[x] = 0.f;
      if (mx != kNegInf) {
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          const float f = exp2_approx(s_m[w][m] - mx);
          l = fmaf(f, s_l[w][m], l);
          const float* src = accs + (w * TR + m) * D;
#pragma unroll
          for (int x = 0; x < 8; ++x) o[x] = fmaf(f, src[kE4m3 ? join_at(m, d + x) : join_at(m, d) + x], o[x]);
        }
      }
      if (complete) {
        const float inv = l > 0.f ? 1.f / l : 0.f;
        const int mm = m0 + m, tok = mm / G;
        T* dst = static_cast<T*>(a.out.p) + static_cast<int64_t>(seq.row0 + tok) * a.out.row_stride +
                 static_cast<int64_t>(h * G + mm - tok * G) * a.out.head_stride + d;
        *reinterpret_cast<uint4*>(dst) = make_uint4(Mma<T>::pack(o[0] * inv, o[1] * inv), Mma<T>::pack(o[2] * inv, o[3] * inv),
                                                    Mma<T>::pack(o[4] * inv, o[5] * inv), Mma<T>::pack(o[6] * inv, o[7] * inv));
      } else {
        float4* dst = reinterpret_cast<float4*>((kCluster ? mine : part) + m * D + d);
        dst[0] = make_float4(o[0], o[1], o[2], o[3]);
        dst[1] = make_float4(o[4], o[5], o[6], o[7]);
        if (kCluster && d == 0) {
          s_cm[m] = mx;
          s_cl[m] = l;
        } else if (d == 0) {
          part[TR * D + m] = mx;
          part[TR * D + TR + m] = l;
        }
      }
    }
    if constexpr (kCluster) {
      // every CTA of the cluster has its part of the tile: each writes a slice
      // of the rows, joined over the parts in order
      cg::cluster_group cluster = cg::this_cluster();
      cluster.sync();
      for (int i = rank * kThreads + tid; i < mrows * (D / 8); i += kThreads * split) {
        const int m = i / (D / 8), d = (i % (D / 8)) * 8;
        float mx = kNegInf;
        for (int c = 0; c < split; ++c) mx = fmaxf(mx, *cluster.map_shared_rank(&s_cm[m], c));
        float l = 0.f, o[8];
#pragma unroll
        for (int x = 0; x < 8; ++x) o[x] = 0.f;
        for (int c = 0; mx != kNegInf && c < split; ++c) {
          const float f = exp2_approx(*cluster.map_shared_rank(&s_cm[m], c) - mx);
          l = fmaf(f, *cluster.map_shared_rank(&s_cl[m], c), l);
          const float4* src = reinterpret_cast<const float4*>(cluster.map_shared_rank(mine + m * D + d, c));
          const float4 v0 = src[0], v1 = src[1];
          o[0] = fmaf(f, v0.x, o[0]);
          o[1] = fmaf(f, v0.y, o[1]);
          o[2] = fmaf(f, v0.z, o[2]);
          o[3] = fmaf(f, v0.w, o[3]);
          o[4] = fmaf(f, v1.x, o[4]);
          o[5] = fmaf(f, v1.y, o[5]);
          o[6] = fmaf(f, v1.z, o[6]);
          o[7] = fmaf(f, v1.w, o[7]);
        }
        const float inv = l > 0.f ? 1.f / l : 0.f;
        const int mm = m0 + m, tok = mm / G;
        T* dst = static_cast<T*>(a.out.p) + static_cast<int64_t>(seq.row0 + tok) * a.out.row_stride +
                 static_cast<int64_t>(h * G + mm - tok * G) * a.out.head_stride + d;
        *reinterpret_cast<uint4*>(dst) = make_uint4(Mma<T>::pack(o[0] * inv, o[1] * inv), Mma<T>::pack(o[2] * inv, o[3] * inv),
                                                    Mma<T>::pack(o[4] * inv, o[5] * inv), Mma<T>::pack(o[6] * inv, o[7] * inv));
      }
      cluster.sync();  // the parts have been read: they may go
      continue;
    }
    if (tid == 0 && k0 == 0 && k1 < per) {
      // the first piece of a tile that goes on in later CTAs: the last of
      // them is the one whose range holds the tile's last unit
      const long long end = u1 - left - k0 + per - 1;
      long long c = end * ctas / total;
      while (total * (c + 1) / ctas <= end) ++c;
      while (total * c / ctas > end) --c;
      note_cut(a, cta, first_piece, static_cast<int>(c), m0, mrows, seq.row0, h);
    }
    __syncthreads();  // the ring is free again
    off += k1 - k0;
    left -= k1 - k0;
    first_piece = false;
  }
}

constexpr int kCtasPerSm = 2;

template <typename T, int D, int MT, bool kE4m3>
cudaError_t attention_launch(const PagedAttention& a, int max_new, cudaStream_t st) {
  // Ring slots of 8 KB (16-bit) or 4.1 KB (8-bit) per warp at D = 128, two CTAs
  // per SM: 3 and 6 (96 KB a CTA); with two row tiles over 8-bit pages 4 (77.7
  // against 81.3 us for 32 x 5 rows).
  constexpr int kStages = (kE4m3 ? (MT == 2 ? 4 : 6) : 3) * (128 / D);
  constexpr int kSmem = RingBytes<D, MT, kE4m3, kStages>::kBytes + (MT == 2 ? MT * (D / 16) * 512 : 0);
  const int sms = sm_count();
  // Where the page table cannot hold long sequences: a cluster per tile, in one
  // launch, as many CTAs as keep every cluster resident.  8 sequences of up to
  // 255 positions take 7.1 us so in a graph (8.2 as calls), and 10.2 by ranges of
  // the line and the join that goes with them; 4 of up to 8000 15.8 and 19.0.  A CTA takes at most 16
  // units so: from 32 on longer sequences are balanced better by the line (one
  // of 16000: 32.3 and 27.5).
  const int64_t units = (static_cast<int64_t>(a.c.max_pages) * a.c.page_size + kUnit - 1) / kUnit;
  const int64_t most = (static_cast<int64_t>(max_new) * a.G + 16 * MT - 1) / (16 * MT);  // tiles of a sequence
  const int64_t items = most * a.c.Hkv * a.c.B;
  int split = 8;
  while (split > 1 && (items * split > kCtasPerSm * sms || split / 2 >= units)) split /= 2;
  if (items * split <= kCtasPerSm * sms && units <= 16 * split) {
    PagedAttention c = a;
    c.split = split;
    c.tile_step = static_cast<int>(most);
    auto k = paged_attention_kernel<T, D, MT, kE4m3, kStages, true>;
    static std::atomic<bool> done[64];
    const cudaError_t e = prepare_kernel(done, k, kSmem, 0);
    if (e != cudaSuccess) return e;
    return launch_paged(k, dim3(static_cast<unsigned>(items * split)), dim3(kThreads), kSmem, split, false, st, c);
  }
  auto k = paged_attention_kernel<T, D, MT, kE4m3, kStages, false>;
  static std::atomic<bool> done[64];
  cudaError_t e = prepare_kernel(done, k, kSmem, 0);
  if (e != cudaSuccess) return e;
  const int ctas = kCtasPerSm * sms;
  e = launch_paged(k, dim3(ctas), dim3(kThreads), kSmem, 1, false, st, a);
  if (e != cudaSuccess) return e;
  return launch_paged(paged_combine_kernel<T, D, 16 * MT>, dim3(ctas, 2 * MT), dim3(256), 0, 1, true, st, a);
}
template <typename T, int D, int MT>
cudaError_t attention_pages(const PagedAttention& a, int max_new, cudaStream_t st) {
  return a.c.k_scale != nullptr ? attention_launch<T, D, MT, true>(a, max_new, st)
                                : attention_launch<T, D, MT, false>(a, max_new, st);
}
template <typename T, int D>
cudaError_t attention_rows(const PagedAttention& a, int max_new, cudaStream_t st) {
  return static_cast<int64_t>(max_new) * a.G <= 16 ? attention_pages<T, D, 1>(a, max_new, st)
                                                  : attention_pages<T, D, 2>(a, max_new, st);
}
template <typename T>
cudaError_t attention_dim(const PagedAttention& a, int max_new, cudaStream_t st) {
  return a.c.D == 128 ? attention_rows<T, 128>(a, max_new, st) : attention_rows<T, 64>(a, max_new, st);
}

}  // namespace

size_t paged_attention_ws_bytes(int D) {
  const size_t ctas = static_cast<size_t>(kCtasPerSm) * sm_count();
  return ctas * 2 * sizeof(int4) + ctas * 2 * (32 * static_cast<size_t>(D) + 64) * sizeof(float);
}

cudaError_t launch_paged_attention(PagedAttention a, int dtype, int max_new, void* workspace, cudaStream_t st) {
  const size_t ctas = static_cast<size_t>(kCtasPerSm) * sm_count();
  a.desc = static_cast<int4*>(workspace);
  a.part = reinterpret_cast<float*>(static_cast<char*>(workspace) + ctas * 2 * sizeof(int4));
  return dtype == PERSONA_DTYPE_BF16 ? attention_dim<__nv_bfloat16>(a, max_new, st) : attention_dim<__half>(a, max_new, st);
}

}  // namespace persona
