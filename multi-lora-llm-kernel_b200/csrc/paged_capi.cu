// extern "C" entry points of the paged KV cache operators and of the draft
// verification: argument checks, then one enqueue.  Nothing here synchronises
// with the device or allocates device memory.
#include <cmath>

#include "overlap.h"
#include "paged_args.h"
#include "persona_bgmv.h"

namespace persona {
namespace {

constexpr int64_t kI32Max = 2147483647;
constexpr int64_t kMaxHeads = 1024;
constexpr int64_t kMaxPositions = int64_t{1} << 30;
constexpr float kLog2E = 1.4426950408889634f;
// Most query rows per kv head (new tokens times heads of a group) for the
// warp-level kernel, which reads the pages once per 32 rows.  Measured with 32
// sequences of up to 6000 tokens: over 16-bit pages 36 rows take it 118 us and
// the tcgen05 kernel 77 (20 rows: 66 and 77); over 8-bit pages, whose codes the
// tcgen05 kernel has to convert for each of its tiles, 64 rows take 129 and 149.
constexpr int64_t kFewRows16 = 32, kFewRows8 = 64;

bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }
int status(cudaError_t e) { return e == cudaSuccess ? PERSONA_OK : PERSONA_ERR_CUDA; }

int check_cache(const persona_paged_cache* c, int dtype, PagedCache& out) {
  if (c == nullptr) return PERSONA_ERR_INVALID_ARG;
  if (dtype != PERSONA_DTYPE_F16 && dtype != PERSONA_DTYPE_BF16) return PERSONA_ERR_DTYPE;
  const bool e4m3 = c->kind == PERSONA_PAGES_E4M3;
  if (!e4m3 && c->kind != PERSONA_PAGES_16BIT) return PERSONA_ERR_DTYPE;
  // (arrays without an element may be null: no sequences, or a table without columns)
  if (c->k == nullptr || c->v == nullptr || (c->B != 0 && (c->indptr == nullptr || c->lengths == nullptr)) ||
      (c->B != 0 && c->max_pages != 0 && c->page_table == nullptr))
    return PERSONA_ERR_INVALID_ARG;
  if (e4m3 != (c->k_scale != nullptr) || e4m3 != (c->v_scale != nullptr)) return PERSONA_ERR_INVALID_ARG;
  if ((c->D != 64 && c->D != 128) || c->Hkv <= 0 || c->Hkv > kMaxHeads || c->num_pages <= 0 || c->num_pages > kI32Max ||
      c->page_size <= 0 || c->page_size > kI32Max || c->max_pages < 0 || c->max_pages > kI32Max || c->B < 0 ||
      c->B > kI32Max / 2 || c->table_stride < c->max_pages)
    return PERSONA_ERR_SHAPE;
  const int64_t unit = e4m3 ? 16 : 8;  // elements of 16 bytes
  if (c->page_stride < 0 || c->head_stride < 0 || c->pos_stride < c->D) return PERSONA_ERR_SHAPE;
  if (!aligned(c->k, 16) || !aligned(c->v, 16) || c->page_stride % unit || c->head_stride % unit || c->pos_stride % unit)
    return PERSONA_ERR_ALIGNMENT;
  if (e4m3 && (c->scale_page_stride < 0 || c->scale_head_stride < 0)) return PERSONA_ERR_SHAPE;
  if (!aligned(c->k_scale, 4) || !aligned(c->v_scale, 4) || !aligned(c->page_table, 4) || !aligned(c->indptr, 4) ||
      !aligned(c->lengths, 4))
    return PERSONA_ERR_ALIGNMENT;
  out = PagedCache{c->k, c->v, c->k_scale, c->v_scale, c->page_stride, c->head_stride, c->pos_stride,
                   c->scale_page_stride, c->scale_head_stride, c->page_table, c->table_stride, c->indptr, c->lengths,
                   static_cast<int>(c->num_pages), static_cast<int>(c->page_size), static_cast<int>(c->max_pages),
                   static_cast<int>(c->Hkv), static_cast<int>(c->D), static_cast<int>(c->B), -1};
  if ((c->page_size & (c->page_size - 1)) == 0)
    for (out.page_shift = 0; (int64_t{1} << out.page_shift) < c->page_size;) ++out.page_shift;
  return PERSONA_OK;
}

int check_rows(const persona_rows* r, PagedRows& out) {
  if (r == nullptr || r->p == nullptr) return PERSONA_ERR_INVALID_ARG;
  if (r->row_stride < 0 || r->head_stride < 0) return PERSONA_ERR_SHAPE;
  if (!aligned(r->p, 16) || r->row_stride % 8 || r->head_stride % 8) return PERSONA_ERR_ALIGNMENT;
  out = PagedRows{r->p, r->row_stride, r->head_stride};
  return PERSONA_OK;
}

// ---- what a call writes ----
using overlap::View;

View rows_view(const PagedRows& r, int64_t rows, int64_t heads, int64_t D) {
  return View{r.p, D * 2, {rows, heads, 1}, {r.row_stride * 2, r.head_stride * 2, 0}};
}
template <typename T> View array_view(const T* p, int64_t n) {
  return View{p, static_cast<int64_t>(sizeof(T)) * n, {1, 1, 1}, {0, 0, 0}};
}
// The memory of a cache and of the int32 arrays that go with it.
struct CacheViews {
  const PagedCache& c;
  const int64_t e;
  const View k, v, k_scale, v_scale, table, indptr, lengths;
  explicit CacheViews(const PagedCache& a)
      : c(a), e(a.k_scale != nullptr ? 1 : 2), k(pages(a.k)), v(pages(a.v)), k_scale(scales(a.k_scale)),
        v_scale(scales(a.v_scale)), table(a.table, int64_t{4} * a.max_pages, {a.B, 1, 1}, {a.table_stride * 4, 0, 0}),
        indptr(array_view(a.indptr, int64_t{a.B} + 1)), lengths(array_view(a.lengths, a.B)) {}
  View pages(const void* p) const {
    return View{p, c.D * e, {c.num_pages, c.Hkv, c.page_size}, {c.page_stride * e, c.head_stride * e, c.pos_stride * e}};
  }
  View scales(const void* p) const {
    return View{p, p != nullptr ? int64_t{4} * c.page_size : 0, {c.num_pages, c.Hkv, 1},
                {c.scale_page_stride * 4, c.scale_head_stride * 4, 0}};
  }
  // Whether the address range of x meets that of the page table, indptr or lengths,
  bool meet_index(const View& x) const {
    return overlap::ranges_meet(x, table) || overlap::ranges_meet(x, indptr) || overlap::ranges_meet(x, lengths);
  }
  // or that of the pages or scales.
  bool meet_pages(const View& x) const {
    return overlap::ranges_meet(x, k) || overlap::ranges_meet(x, v) || overlap::ranges_meet(x, k_scale) ||
           overlap::ranges_meet(x, v_scale);
  }
  // Rows that a call writes: none twice, and nothing that it reads of the cache.
  bool apart(const View& x) const { return overlap::nested(x) && !meet_pages(x) && !meet_index(x); }
  // Pages and scales that a call writes.  (The scales may lie inside the pool
  // of the pages, so those two are not compared.)
  bool writable() const {
    if (!overlap::nested(k) || overlap::share(k, v) || meet_index(k) || meet_index(v)) return false;
    return c.k_scale == nullptr || (overlap::nested(k_scale) && !overlap::share(k_scale, v_scale) &&
                                    !meet_index(k_scale) && !meet_index(v_scale));
  }
};

}  // namespace
}  // namespace persona

using namespace persona;

#define PERSONA_TRY(x)                      \
  do {                                      \
    const int st_ = (x);                    \
    if (st_ != PERSONA_OK) return st_;      \
  } while (0)

extern "C" {

int persona_paged_rope_cache(const persona_paged_cache* cache, const persona_rows* q, const persona_rows* q_out,
                             const persona_rows* k, const persona_rows* v, int64_t rows, int64_t Hq, float theta,
                             int dtype, int32_t* dev_err, cudaStream_t stream) {
  PagedWrite a;
  PERSONA_TRY(check_cache(cache, dtype, a.c));
  if (rows < 0 || rows > kI32Max || Hq <= 0 || Hq > kMaxHeads || !(theta > 1.f) || !std::isfinite(theta))
    return PERSONA_ERR_SHAPE;
  if (rows == 0 || cache->B == 0) return PERSONA_OK;
  PERSONA_TRY(check_rows(q, a.q));
  PERSONA_TRY(check_rows(q_out, a.q_out));
  PERSONA_TRY(check_rows(k, a.k));
  PERSONA_TRY(check_rows(v, a.v));
  a.rows = static_cast<int>(rows);
  a.Hq = static_cast<int>(Hq);
  const int D = a.c.D;
  const CacheViews m(a.c);
  const View vq = rows_view(a.q, rows, Hq, D), vo = rows_view(a.q_out, rows, Hq, D), vk = rows_view(a.k, rows, a.c.Hkv, D),
             vv = rows_view(a.v, rows, a.c.Hkv, D);
  const bool in_place = a.q.p == a.q_out.p && a.q.row_stride == a.q_out.row_stride && a.q.head_stride == a.q_out.head_stride;
  if (!m.writable() || !m.apart(vo) || (!in_place && overlap::share(vq, vo)) || overlap::share(vk, vo) ||
      overlap::share(vv, vo) || m.meet_pages(vq) || m.meet_pages(vk) || m.meet_pages(vv))
    return PERSONA_ERR_OVERLAP;
  // theta^(-2j / D) / (2 pi) by multiplication: 63 roundings of 2^-53
  const double ratio = std::pow(static_cast<double>(theta), -2.0 / D);
  double f = 1.0 / 6.283185307179586476925;
  for (int j = 0; j < 64; ++j, f *= ratio) a.turns[j] = j < D / 2 ? f : 0.0;
  return status(launch_paged_write(a, dtype, dev_err, stream));
}

int persona_paged_cache_read(const persona_paged_cache* cache, const persona_rows* k, const persona_rows* v,
                             int64_t rows, int dtype, int32_t* dev_err, cudaStream_t stream) {
  PagedRead a;
  PERSONA_TRY(check_cache(cache, dtype, a.c));
  if (rows < 0 || rows > kI32Max) return PERSONA_ERR_SHAPE;
  if (rows == 0 || cache->B == 0) return PERSONA_OK;
  PERSONA_TRY(check_rows(k, a.k));
  PERSONA_TRY(check_rows(v, a.v));
  const View vk = rows_view(a.k, rows, a.c.Hkv, a.c.D), vv = rows_view(a.v, rows, a.c.Hkv, a.c.D);
  const CacheViews m(a.c);
  if (!m.apart(vk) || !m.apart(vv) || overlap::share(vk, vv)) return PERSONA_ERR_OVERLAP;
  a.rows = static_cast<int>(rows);
  return status(launch_paged_read(a, dtype, dev_err, stream));
}

size_t persona_paged_attention_workspace_size(int64_t D) {
  if (D != 64 && D != 128) return 0;
  const size_t few = paged_attention_ws_bytes(static_cast<int>(D)), many = paged_chunk_ws_bytes(static_cast<int>(D));
  return few > many ? few : many;
}

int persona_paged_attention(const persona_paged_cache* cache, const persona_rows* q, const persona_rows* out,
                            int64_t rows, int64_t Hq, float scale, int64_t window, int64_t max_new, int dtype,
                            void* workspace, size_t workspace_bytes, int32_t* dev_err, cudaStream_t stream) {
  PagedAttention a;
  PERSONA_TRY(check_cache(cache, dtype, a.c));
  if (rows < 0 || Hq <= 0 || Hq > kMaxHeads || Hq % cache->Hkv || rows > kI32Max / Hq || window < 0 || max_new < 1 ||
      !(scale > 0.f) || !std::isfinite(scale * kLog2E))
    return PERSONA_ERR_SHAPE;
  // positions of a sequence, and what the kernels add to and take from them
  // (blocks ahead, a window), are 32-bit numbers
  if (cache->max_pages > kMaxPositions / cache->page_size) return PERSONA_ERR_SHAPE;
  if (rows == 0 || cache->B == 0) return PERSONA_OK;
  PERSONA_TRY(check_rows(q, a.q));
  PERSONA_TRY(check_rows(out, a.out));
  if (workspace == nullptr || workspace_bytes < persona_paged_attention_workspace_size(a.c.D)) return PERSONA_ERR_WORKSPACE;
  if (!aligned(workspace, 16)) return PERSONA_ERR_ALIGNMENT;
  // a row's q is read again by the CTAs that share its positions
  const View vq = rows_view(a.q, rows, Hq, a.c.D), vo = rows_view(a.out, rows, Hq, a.c.D);
  const View ws = array_view(static_cast<const char*>(workspace), static_cast<int64_t>(persona_paged_attention_workspace_size(a.c.D)));
  const CacheViews m(a.c);
  if (!m.apart(vo) || overlap::share(vq, vo) || overlap::ranges_meet(ws, vo) || overlap::ranges_meet(ws, vq) ||
      m.meet_pages(ws) || m.meet_index(ws))
    return PERSONA_ERR_OVERLAP;
  a.rows = static_cast<int>(rows);
  a.G = static_cast<int>(Hq / cache->Hkv);
  a.window = window >= kMaxPositions ? 0 : static_cast<int>(window);  // wider than any sequence
  a.scale_log2 = scale * kLog2E;
  a.err = dev_err;
  a.split = a.tile_step = 1;
  const int most = static_cast<int>(max_new > rows ? rows : max_new);
  if (static_cast<int64_t>(most) * a.G > (a.c.k_scale != nullptr ? kFewRows8 : kFewRows16))
    return status(launch_paged_chunk(a, dtype, workspace, stream));
  return status(launch_paged_attention(a, dtype, most, workspace, stream));
}

int persona_verify_draft(const void* target, int64_t ld_target, const void* draft, int64_t ld_draft, int prob_type,
                         const int64_t* draft_tokens, const int32_t* indptr, const float* u_accept,
                         const float* u_sample, int64_t* tokens, int32_t* accepted, int64_t rows, int64_t B, int64_t V,
                         int32_t* dev_err, cudaStream_t stream) {
  if (prob_type < PERSONA_DTYPE_F16 || prob_type > PERSONA_DTYPE_F32) return PERSONA_ERR_DTYPE;
  if (rows < 0 || rows > kI32Max || B < 0 || B > kI32Max / 8 || V <= 0 || V > PERSONA_VERIFY_MAX_VOCAB || ld_target < V ||
      (draft != nullptr && ld_draft < V))
    return PERSONA_ERR_SHAPE;
  if (B == 0) return PERSONA_OK;
  if (indptr == nullptr || u_sample == nullptr || accepted == nullptr) return PERSONA_ERR_INVALID_ARG;
  if (rows > 0 && (target == nullptr || draft_tokens == nullptr || u_accept == nullptr || tokens == nullptr))
    return PERSONA_ERR_INVALID_ARG;
  const uintptr_t e = prob_type == PERSONA_DTYPE_F32 ? 4 : 2;
  if (!aligned(target, e) || !aligned(draft, e) || !aligned(draft_tokens, 8) || !aligned(tokens, 8) || !aligned(indptr, 4) ||
      !aligned(u_accept, 4) || !aligned(u_sample, 4) || !aligned(accepted, 4))
    return PERSONA_ERR_ALIGNMENT;
  // the CTAs of a cluster, and those of other sequences, read the inputs at any time
  const View out = array_view(tokens, rows), kept = array_view(accepted, B);
  const View in[] = {View{target, V * static_cast<int64_t>(e), {rows, 1, 1}, {ld_target * static_cast<int64_t>(e), 0, 0}},
                     View{draft, draft != nullptr ? V * static_cast<int64_t>(e) : 0, {rows, 1, 1}, {ld_draft * static_cast<int64_t>(e), 0, 0}},
                     array_view(draft_tokens, rows), array_view(indptr, B + 1), array_view(u_accept, rows), array_view(u_sample, B)};
  if (overlap::ranges_meet(out, kept)) return PERSONA_ERR_OVERLAP;
  for (const View& v : in)
    if (overlap::ranges_meet(out, v) || overlap::ranges_meet(kept, v)) return PERSONA_ERR_OVERLAP;
  const VerifyDraft a{target, draft, ld_target, ld_draft, draft_tokens, indptr, u_accept, u_sample, tokens, accepted,
                      static_cast<int>(rows), static_cast<int>(B), static_cast<int>(V), dev_err};
  return status(launch_verify_draft(a, prob_type, stream));
}

}  // extern "C"
