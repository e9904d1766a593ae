// Arguments and launchers of the paged KV cache operators and of the draft
// verification.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

namespace persona {

// A paged cache and the ragged batch that uses it, as the kernels read it.
// k and v share their shape and strides (in elements); the scales (e4m3
// only) have unit position stride.  Sequence b's new tokens are rows
// [indptr[b], indptr[b + 1]) and sit at its last positions, the last one at
// lengths[b] - 1.
struct PagedCache {
  void* k;
  void* v;
  float* k_scale;  // nullptr: 16-bit pages
  float* v_scale;
  int64_t page_stride, head_stride, pos_stride;
  int64_t scale_page_stride, scale_head_stride;
  const int32_t* table;
  int64_t table_stride;
  const int32_t* indptr;
  const int32_t* lengths;
  int num_pages, page_size, max_pages, Hkv, D, B;
  int page_shift;  // log2(page_size), -1 if it is no power of two
};

// One [rows, heads, D] activation: unit inner stride, others in elements.
struct PagedRows {
  void* p;
  int64_t row_stride, head_stride;
};

struct PagedWrite {
  PagedCache c;
  PagedRows q, q_out, k, v;
  int rows, Hq;
  double turns[64];  // inverse frequencies of the rotary embedding, in turns per position
};

struct PagedRead {
  PagedCache c;
  PagedRows k, v;
  int rows;
};

struct PagedAttention {
  PagedCache c;
  PagedRows q, out;
  int rows, G;         // q heads per kv head
  int window;          // 0: none
  float scale_log2;    // softmax scale times log2(e)
  int split, tile_step;  // a cluster per tile: its CTAs, and the first tiles taken per sequence and head
  float* part;         // partial results, see paged_attention.cuh
  int4* desc;          // two per CTA
  int32_t* err;
};

cudaError_t launch_paged_write(const PagedWrite& a, int dtype, int32_t* err, cudaStream_t st);
cudaError_t launch_paged_read(const PagedRead& a, int dtype, int32_t* err, cudaStream_t st);
// Bytes of part and desc for any call with this head size on the current device.
size_t paged_attention_ws_bytes(int D);
cudaError_t launch_paged_attention(PagedAttention a, int dtype, int max_new, void* workspace, cudaStream_t st);
// The same for many rows per kv head (paged_chunk.cu).
size_t paged_chunk_ws_bytes(int D);
cudaError_t launch_paged_chunk(PagedAttention a, int dtype, void* workspace, cudaStream_t st);

struct VerifyDraft {
  const void* target;  // [rows, V], row stride ld_target
  const void* draft;   // [rows, V] or nullptr
  int64_t ld_target, ld_draft;
  const int64_t* draft_tokens;
  const int32_t* indptr;
  const float* u_accept;
  const float* u_sample;
  int64_t* tokens;
  int32_t* accepted;
  int rows, B, V;
  int32_t* err;
};
// type: 0 fp16, 1 bf16, 2 fp32
cudaError_t launch_verify_draft(const VerifyDraft& a, int type, cudaStream_t st);

}  // namespace persona
