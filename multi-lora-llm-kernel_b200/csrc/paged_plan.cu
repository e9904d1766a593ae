// The plan of a step over a paged cache, made on the device from the lengths
// of its sequences: pages given back and taken, row offsets, and for every new
// row its place in the cache and its adapter slot.
//
//   held = ceil(lengths / page), kept = ceil(keep / page), need = ceil((keep + new) / page)
//   free list: push pages [kept, held) of every sequence, the last sequence's
//   last page first; then pop pages [kept, need), the first sequence's first
//   page first (so a step that is taken back and made again gets its old pages)
//   indptr = running sums of new;  places[r] = page(p) * page_size + p % page_size
//
// It reads a few numbers per sequence and writes twelve bytes per row: bound
// by the launch and its chain of reads, scan, stores: 4.8 us for 8 sequences,
// 6.2 for 256 whose drafts are cut back, 7.3 for 48 with 14700 new rows.
#include <cooperative_groups.h>

#include "paged_common.cuh"

namespace persona {
namespace cg = cooperative_groups;
namespace {

constexpr int kThreads = 1024, kWarps = kThreads / 32;

// The last i in [0, n) with from[i] <= x (from[0] <= x, not decreasing).
__device__ __forceinline__ int last_at_most(const int* from, int n, int x) {
  int lo = 0;
  while (n > 1) {
    const int half = n / 2;
    if (from[lo + half] <= x) {
      lo += half;
      n -= half;
    } else {
      n = half;
    }
  }
  return lo;
}

// One cluster.  Every CTA scans all sequences for itself, so that none waits
// for another's sums; then they share the pages and the rows.
__global__ void __launch_bounds__(kThreads, 1) paged_plan_kernel(const __grid_constant__ PagedPlan a) {
  cg::cluster_group cluster = cg::this_cluster();
  extern __shared__ int s_seq[];
  __shared__ long long s_sum[3][kWarps];
  __shared__ int s_bad[kWarps];
  const int B = a.B, ps = a.page_size;
  // of every sequence: first row, pages taken and given back before it, tokens kept, pages kept
  int* const s_row = s_seq;
  int* const s_take = s_row + B;
  int* const s_back = s_take + B;
  int* const s_keep = s_back + B;
  int* const s_kept = s_keep + B;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int ctas = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
  pdl_wait();
  pdl_launch();

  // ---- scan: a thread has a run of neighbouring sequences ----
  const int each = (B + kThreads - 1) / kThreads, b0 = min(B, tid * each), b1 = min(B, b0 + each);
  const int num_free = *a.num_free;
  long long sum[3] = {0, 0, 0};  // rows, pages taken, pages given back
  int bad = num_free < 0 || num_free > a.pool ? PERSONA_DEV_ERR_PAGE : 0;
  for (int b = b0; b < b1; ++b) {
    const int len = a.lengths[b], keep = a.keep != nullptr ? a.keep[b] : len, add = a.add[b];
    const long long want = static_cast<long long>(keep) + add;
    if (keep < 0 || keep > len || add < 0) {
      bad |= PERSONA_DEV_ERR_SEGMENT;
      continue;
    }
    const int held = (static_cast<long long>(len) + ps - 1) / ps, kept = (static_cast<long long>(keep) + ps - 1) / ps;
    const long long need = (want + ps - 1) / ps;
    if (held > a.max_pages) bad |= PERSONA_DEV_ERR_PAGE;
    if (need > a.max_pages || want > 2147483647) bad |= PERSONA_DEV_ERR_FULL;
    s_row[b] = add;
    s_take[b] = static_cast<int>(need - kept);
    s_back[b] = held - kept;
    s_keep[b] = keep;
    s_kept[b] = kept;
    sum[0] += add;
    sum[1] += need - kept;
    sum[2] += held - kept;
  }
  long long before[3], total[3];
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    long long inc = sum[i];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long up = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += up;
    }
    if (lane == 31) s_sum[i][warp] = inc;
    before[i] = inc - sum[i];
  }
  bad = static_cast<int>(__reduce_or_sync(0xffffffffu, static_cast<unsigned>(bad)));
  if (lane == 0) s_bad[warp] = bad;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    const long long s = s_sum[i][lane];
    long long inc = s;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long up = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += up;
    }
    total[i] = __shfl_sync(0xffffffffu, inc, 31);
    before[i] += __shfl_sync(0xffffffffu, inc - s, warp);
  }
  const long long top = num_free + total[2];  // pages in the list once all are given back
  int bits = static_cast<int>(__reduce_or_sync(0xffffffffu, static_cast<unsigned>(s_bad[lane])));
  if (total[0] > a.rows) bits |= PERSONA_DEV_ERR_SEGMENT;
  if (bits == 0 && top > a.pool) bits |= PERSONA_DEV_ERR_PAGE;  // more pages than the list has room for
  if (bits == 0 && total[1] > top) bits |= PERSONA_DEV_ERR_FULL;
  const int first = rank * kThreads + tid, step = ctas * kThreads;
  cluster.sync();  // every CTA has read what follows changes
  if (bits != 0) {  // the same in all CTAs: nothing changes, and no row belongs to a sequence
    if (first == 0) raise_error(a.err, bits);
    for (int b = first; b <= B; b += step) a.indptr[b] = 0;
    for (int r = first; r < a.rows; r += step) {
      a.places[r] = -1;
      if (a.row_slots != nullptr) a.row_slots[r] = -1;
    }
    return;
  }
  for (int b = b0; b < b1; ++b) {  // sums before each sequence in place of its own numbers
    const int n[3] = {s_row[b], s_take[b], s_back[b]};
    s_row[b] = static_cast<int>(before[0]);
    s_take[b] = static_cast<int>(before[1]);
    s_back[b] = static_cast<int>(before[2]);
#pragma unroll
    for (int i = 0; i < 3; ++i) before[i] += n[i];
  }
  __syncthreads();

  // ---- pages given back ----
  const int back = static_cast<int>(total[2]);
  if (back > 0) {
    for (int x = first; x < back; x += step) {
      const int b = last_at_most(s_back, B, x);
      const int j = s_kept[b] + (x - s_back[b]);
      a.free_pages[num_free + (back - 1 - x)] = a.table[b * a.table_stride + j];
    }
    cluster.sync();  // the list is complete
  }
  // ---- pages taken, rows ----
  const int last = static_cast<int>(top) - 1;
  for (int x = first; x < static_cast<int>(total[1]); x += step) {
    const int b = last_at_most(s_take, B, x);
    a.table[b * a.table_stride + s_kept[b] + (x - s_take[b])] = a.free_pages[last - x];
  }
  const int rows = static_cast<int>(total[0]);
  for (int r = first; r < a.rows; r += step) {
    int64_t place = -1;
    int slot = -1;
    if (r < rows) {
      const int b = last_at_most(s_row, B, r);
      const int p = s_keep[b] + (r - s_row[b]), j = p / ps;
      const int page = j < s_kept[b] ? a.table[b * a.table_stride + j] : a.free_pages[last - (s_take[b] + j - s_kept[b])];
      place = static_cast<int64_t>(page) * ps + (p - j * ps);
      if (a.row_slots != nullptr) slot = a.seq_slots[b];
    }
    a.places[r] = place;
    if (a.row_slots != nullptr) a.row_slots[r] = slot;
  }
  for (int b = first; b < B; b += step) {
    const int next = b + 1 < B ? s_row[b + 1] : rows;
    a.indptr[b + 1] = next;
    a.lengths[b] = s_keep[b] + next - s_row[b];
  }
  if (first == 0) {
    a.indptr[0] = 0;
    *a.num_free = static_cast<int>(top - total[1]);
  }
}

constexpr int kSeqBytes = 5 * sizeof(int);
static_assert(PERSONA_PLAN_MAX_SEQS * kSeqBytes <= 200 * 1024, "shared memory");

}  // namespace

cudaError_t launch_paged_plan(const PagedPlan& a, cudaStream_t st) {
  static std::atomic<bool> done[64];
  const cudaError_t e = prepare_kernel(done, paged_plan_kernel, PERSONA_PLAN_MAX_SEQS * kSeqBytes, 0);
  if (e != cudaSuccess) return e;
  // One CTA for few rows, which has no cluster barriers: 512 rows 4.9 us (eight CTAs
  // 5.5), 1024 5.1 (5.9), 2048 5.8 (5.8), 4096 7.4 (6.0), 14700 16.7 (7.5).  Pages given
  // back, which the host does not know, are not in the rule: 3000 of them cost one CTA
  // 4.4 us (4.7), 32000, sequences of half a million tokens that end together, 17.7 (4.7).
  const int ctas = a.rows <= 2048 ? 1 : 8;
  return launch_paged(paged_plan_kernel, dim3(ctas), dim3(kThreads), static_cast<size_t>(a.B) * kSeqBytes, ctas, true, st, a);
}

}  // namespace persona
