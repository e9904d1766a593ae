// torch.ops.persona registration over the C ABI of libpersona_bgmv.so.
//
// The three reference schemas are registered byte-identically on the CUDA
// dispatch key (reference csrc/bindings.cpp:19-29), with the same C++ host
// symbols (bgmv_shrink_cuda, bgmv_expand_cuda, persona::gemv_fp16_cuda) and
// the same TORCH_CHECK messages.  New ops (fused, planned variants, plan)
// are registered beside them.  Python module persona._C keeps `noop`
// (reference csrc/bindings.cpp:31-33) and adds the device error word
// helpers.
//
// Slot validation: the reference syncs with the host once per row
// (csrc/bgmv_shrink.cu:106-109).  Here the device flags an out-of-range
// slot in a per-device error word held in mapped pinned host memory; every
// op first reads that word (no sync) and raises RuntimeError if an earlier
// call flagged it, and PERSONA_STRICT_SLOTS=1 makes each op synchronise and
// raise on its own call instead.
#include <ATen/PythonTorchFunctionTLS.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>
#include <torch/library.h>

#include <algorithm>
#include <cstdlib>
#include <mutex>
#include <sstream>
#include <vector>

#include "overlap.h"
#include "persona_bgmv.h"

namespace {

constexpr int kMaxDevices = 64;

struct ErrorWords {
  std::mutex mu;
  int32_t* host[kMaxDevices] = {};
};
ErrorWords& error_words() {
  static ErrorWords w;
  return w;
}

// Mapped pinned int32 of `device` (allocated on first use), host view.
int32_t* error_word_host(int device) {
  TORCH_CHECK(device >= 0 && device < kMaxDevices, "persona: device index out of range");
  auto& w = error_words();
  std::lock_guard<std::mutex> lock(w.mu);
  if (w.host[device] == nullptr) {
    void* p = nullptr;
    C10_CUDA_CHECK(cudaHostAlloc(&p, sizeof(int32_t), cudaHostAllocMapped | cudaHostAllocPortable));
    *static_cast<volatile int32_t*>(p) = 0;
    w.host[device] = static_cast<int32_t*>(p);
  }
  return w.host[device];
}

int32_t* error_word_device(int device) {
  static int32_t* dev_ptr[kMaxDevices] = {};
  if (dev_ptr[device] == nullptr) {
    int32_t* h = error_word_host(device);
    void* d = nullptr;
    C10_CUDA_CHECK(cudaHostGetDevicePointer(&d, h, 0));
    dev_ptr[device] = static_cast<int32_t*>(d);
  }
  return dev_ptr[device];
}

std::string describe_error(int bits) {
  std::ostringstream os;
  os << "persona: a BGMV/SGMV call on this device flagged an error (bits 0x" << std::hex << bits
     << std::dec << "):";
  if (bits & PERSONA_DEV_ERR_SLOT) os << " slot out of range;";
  if (bits & PERSONA_DEV_ERR_TIMEOUT) os << " device wait timed out;";
  if (bits & PERSONA_DEV_ERR_SEGMENT) os << " invalid segment table;";
  if (bits & PERSONA_DEV_ERR_PLAN) os << " reused plan does not match the call;";
  if (bits & PERSONA_DEV_ERR_PAGE) os << " page or position outside the paged cache;";
  if (bits & PERSONA_DEV_ERR_TOKEN) os << " drafted token outside the vocabulary;";
  if (bits & PERSONA_DEV_ERR_FULL) os << " no room for a planned step in the free pages or the page table;";
  return os.str();
}

// Raise (and clear) an error flagged by an earlier call on `device`.
void raise_pending(int device, const char* op) {
  volatile int32_t* h = error_word_host(device);
  const int bits = *h;
  if (bits != 0) {
    *h = 0;
    TORCH_CHECK(false, op, ": ", describe_error(bits));
  }
}

bool strict_slots() {
  static const bool strict = [] {
    const char* e = std::getenv("PERSONA_STRICT_SLOTS");
    return e != nullptr && e[0] == '1';
  }();
  return strict;
}

void after_launch(int device, const char* op, cudaStream_t stream) {
  if (!strict_slots()) return;
  C10_CUDA_CHECK(cudaStreamSynchronize(stream));
  volatile int32_t* h = error_word_host(device);
  const int bits = *h;
  if (bits & PERSONA_DEV_ERR_SLOT) {
    *h = 0;
    TORCH_CHECK(false, op, ": slot out of range");
  }
  raise_pending(device, op);
}

void check_status(int st, const char* op) {
  TORCH_CHECK(st == PERSONA_OK, op, ": ", persona_status_string(st));
}

int dtype_code(const at::Tensor& t, const char* op) {
  if (t.scalar_type() == at::kHalf) return PERSONA_DTYPE_F16;
  if (t.scalar_type() == at::kBFloat16) return PERSONA_DTYPE_BF16;
  TORCH_CHECK(false, op, ": only float16 and bfloat16 supported");
  return -1;
}

// Row-major [rows, cols] with unit inner stride (a view of a wider buffer is
// fine); returns the row stride in elements.
int64_t row_stride(const at::Tensor& t) { return t.size(0) <= 1 ? t.size(1) : t.stride(0); }

// Sized for a multi-projection launch, so that any plan serves every op.
at::Tensor workspace_for(int64_t T, const at::Tensor& like) {
  const size_t bytes = persona_bgmv_multi_workspace_size(T, PERSONA_MAX_PROBLEMS);
  return at::empty({static_cast<int64_t>(bytes)}, like.options().dtype(at::kByte));
}

void check_pool_a(const at::Tensor& a_pool, const char* op) {
  TORCH_CHECK(a_pool.dim() == 3, op, ": a_pool must be [S, R, K]");
  TORCH_CHECK(a_pool.stride(2) == 1, op, ": tensors must be contiguous");
}

void check_pool_b(const at::Tensor& b_pool, const char* op) {
  TORCH_CHECK(b_pool.dim() == 3, op, ": b_pool must be [S, N, R]");
  TORCH_CHECK(b_pool.stride(2) == 1 && b_pool.stride(1) == b_pool.size(2), op,
              ": tensors must be contiguous");
}

void shrink_impl(const at::Tensor& x, const at::Tensor& a_pool, const at::Tensor& slots,
                 at::Tensor& v, const c10::optional<at::Tensor>& plan) {
  const char* op = "bgmv_shrink";
  TORCH_CHECK(x.is_cuda() && a_pool.is_cuda() && slots.is_cuda() && v.is_cuda(),
              "bgmv_shrink: all tensors must be CUDA");
  TORCH_CHECK(x.dim() == 2 && x.stride(1) == 1 && slots.is_contiguous() && v.is_contiguous(),
              "bgmv_shrink: tensors must be contiguous");
  check_pool_a(a_pool, op);
  TORCH_CHECK(slots.scalar_type() == at::kInt, "bgmv_shrink: slots must be int32");
  TORCH_CHECK(v.scalar_type() == at::kFloat, "bgmv_shrink: v must be float32");
  const int64_t T = x.size(0), K = x.size(1), S = a_pool.size(0), R = a_pool.size(1);
  TORCH_CHECK(a_pool.size(2) == K, "bgmv_shrink: a_pool shape mismatch");
  TORCH_CHECK(slots.dim() == 1 && slots.size(0) == T, "bgmv_shrink: slots length must match T");
  TORCH_CHECK(v.dim() == 2 && v.size(0) == T && v.size(1) == R, "bgmv_shrink: v shape mismatch");
  TORCH_CHECK(K % 8 == 0, "bgmv_shrink: K must be a multiple of 8");
  TORCH_CHECK(reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 == 0, "bgmv_shrink: x must be 16-byte aligned");
  TORCH_CHECK(reinterpret_cast<uintptr_t>(a_pool.data_ptr()) % 16 == 0,
              "bgmv_shrink: a_pool must be 16-byte aligned");
  const int dt = dtype_code(x, op);
  TORCH_CHECK(a_pool.scalar_type() == x.scalar_type(), "bgmv_shrink: dtype mismatch");
  const at::cuda::OptionalCUDAGuard guard(x.device());
  const int dev = x.get_device();
  raise_pending(dev, op);
  if (T == 0) return;
  cudaStream_t stream = at::cuda::getCurrentCUDAStream();
  at::Tensor ws = plan.has_value() ? *plan : workspace_for(T, x);
  const int flags = plan.has_value() ? PERSONA_REUSE_PLAN : 0;
  TORCH_CHECK(static_cast<size_t>(ws.numel()) >= persona_bgmv_workspace_size(T),
              "bgmv_shrink: plan was built for fewer rows");
  const int st = persona_bgmv_shrink(x.data_ptr(), row_stride(x), a_pool.data_ptr(), a_pool.stride(0),
                                     a_pool.stride(1), slots.data_ptr<int32_t>(), v.data_ptr<float>(), T,
                                     K, R, S, dt, ws.data_ptr(), ws.numel(), flags,
                                     error_word_device(dev), stream);
  check_status(st, op);
  after_launch(dev, op, stream);
}

void expand_impl(const at::Tensor& v, const at::Tensor& b_pool, const at::Tensor& slots, at::Tensor& y,
                 const c10::optional<at::Tensor>& plan) {
  const char* op = "bgmv_expand";
  TORCH_CHECK(v.is_cuda() && b_pool.is_cuda() && slots.is_cuda() && y.is_cuda(),
              "bgmv_expand: all tensors must be CUDA");
  TORCH_CHECK(v.is_contiguous() && slots.is_contiguous() && y.dim() == 2 && y.stride(1) == 1,
              "bgmv_expand: tensors must be contiguous");
  check_pool_b(b_pool, op);
  TORCH_CHECK(slots.scalar_type() == at::kInt, "bgmv_expand: slots must be int32");
  TORCH_CHECK(v.scalar_type() == at::kFloat, "bgmv_expand: v must be float32");
  const int64_t T = v.size(0), R = v.size(1), S = b_pool.size(0), N = b_pool.size(1);
  TORCH_CHECK(b_pool.size(2) == R, "bgmv_expand: b_pool rank dim mismatch");
  TORCH_CHECK(slots.dim() == 1 && slots.size(0) == T, "bgmv_expand: slots length must match T");
  TORCH_CHECK(y.size(0) == T && y.size(1) == N, "bgmv_expand: y shape mismatch");
  TORCH_CHECK(N % 8 == 0, "bgmv_expand: N must be a multiple of 8");
  TORCH_CHECK(reinterpret_cast<uintptr_t>(b_pool.data_ptr()) % 16 == 0,
              "bgmv_expand: b_pool must be 16-byte aligned");
  TORCH_CHECK(reinterpret_cast<uintptr_t>(y.data_ptr()) % 16 == 0, "bgmv_expand: y must be 16-byte aligned");
  TORCH_CHECK(R == 8 || R == 16 || R == 32 || R == 64, "bgmv_expand: R must be 8, 16, 32, or 64");
  const int dt = dtype_code(y, op);
  TORCH_CHECK(b_pool.scalar_type() == y.scalar_type(), "bgmv_expand: dtype mismatch");
  const at::cuda::OptionalCUDAGuard guard(v.device());
  const int dev = v.get_device();
  raise_pending(dev, op);
  if (T == 0) return;
  cudaStream_t stream = at::cuda::getCurrentCUDAStream();
  at::Tensor ws = plan.has_value() ? *plan : workspace_for(T, v);
  const int flags = plan.has_value() ? PERSONA_REUSE_PLAN : 0;
  TORCH_CHECK(static_cast<size_t>(ws.numel()) >= persona_bgmv_workspace_size(T),
              "bgmv_expand: plan was built for fewer rows");
  const int st = persona_bgmv_expand(v.data_ptr<float>(), b_pool.data_ptr(), b_pool.stride(0),
                                     slots.data_ptr<int32_t>(), y.data_ptr(), row_stride(y), T, N, R, S,
                                     dt, ws.data_ptr(), ws.numel(), flags, error_word_device(dev), stream);
  check_status(st, op);
  after_launch(dev, op, stream);
}

void fused_impl(const at::Tensor& x, const at::Tensor& a_pool, const at::Tensor& b_pool,
                const at::Tensor& slots, at::Tensor& y, const c10::optional<at::Tensor>& plan) {
  const char* op = "bgmv_fused";
  TORCH_CHECK(x.is_cuda() && a_pool.is_cuda() && b_pool.is_cuda() && slots.is_cuda() && y.is_cuda(),
              "bgmv_fused: all tensors must be CUDA");
  TORCH_CHECK(x.dim() == 2 && x.stride(1) == 1 && slots.is_contiguous() && y.dim() == 2 &&
                  y.stride(1) == 1,
              "bgmv_fused: tensors must be contiguous");
  check_pool_a(a_pool, op);
  check_pool_b(b_pool, op);
  TORCH_CHECK(slots.scalar_type() == at::kInt, "bgmv_fused: slots must be int32");
  const int64_t T = x.size(0), K = x.size(1), S = a_pool.size(0), R = a_pool.size(1), N = b_pool.size(1);
  TORCH_CHECK(a_pool.size(2) == K, "bgmv_fused: a_pool shape mismatch");
  TORCH_CHECK(b_pool.size(0) == S && b_pool.size(2) == R, "bgmv_fused: b_pool shape mismatch");
  TORCH_CHECK(slots.dim() == 1 && slots.size(0) == T, "bgmv_fused: slots length must match T");
  TORCH_CHECK(y.size(0) == T && y.size(1) == N, "bgmv_fused: y shape mismatch");
  const int dt = dtype_code(x, op);
  TORCH_CHECK(a_pool.scalar_type() == x.scalar_type() && b_pool.scalar_type() == x.scalar_type() &&
                  y.scalar_type() == x.scalar_type(),
              "bgmv_fused: dtype mismatch");
  const at::cuda::OptionalCUDAGuard guard(x.device());
  const int dev = x.get_device();
  raise_pending(dev, op);
  if (T == 0) return;
  cudaStream_t stream = at::cuda::getCurrentCUDAStream();
  at::Tensor ws = plan.has_value() ? *plan : workspace_for(T, x);
  const int flags = plan.has_value() ? PERSONA_REUSE_PLAN : 0;
  TORCH_CHECK(static_cast<size_t>(ws.numel()) >= persona_bgmv_workspace_size(T),
              "bgmv_fused: plan was built for fewer rows");
  const int st = persona_bgmv_fused(x.data_ptr(), row_stride(x), a_pool.data_ptr(), a_pool.stride(0),
                                    a_pool.stride(1), b_pool.data_ptr(), b_pool.stride(0),
                                    slots.data_ptr<int32_t>(), y.data_ptr(), row_stride(y), T, K, N, R,
                                    S, dt, ws.data_ptr(), ws.numel(), flags, error_word_device(dev),
                                    stream);
  check_status(st, op);
  after_launch(dev, op, stream);
}

void fused_multi_impl(at::TensorList xs, at::TensorList a_pools, at::TensorList b_pools, const at::Tensor& slots,
                      at::TensorList ys, const c10::optional<at::Tensor>& plan) {
  const char* op = "bgmv_fused_multi";
  const int P = static_cast<int>(xs.size());
  TORCH_CHECK(P >= 1 && P <= PERSONA_MAX_PROBLEMS, op, ": 1 to ", PERSONA_MAX_PROBLEMS, " projections");
  TORCH_CHECK(a_pools.size() == xs.size() && b_pools.size() == xs.size() && ys.size() == xs.size(), op,
              ": xs, a_pools, b_pools and ys must have the same length");
  TORCH_CHECK(slots.is_cuda() && slots.is_contiguous() && slots.dim() == 1 && slots.scalar_type() == at::kInt, op,
              ": slots must be a contiguous int32 CUDA vector");
  const int64_t T = slots.size(0);
  const int64_t S = a_pools[0].size(0), R = a_pools[0].size(1);
  const int dt = dtype_code(xs[0], op);
  persona_bgmv_problem probs[PERSONA_MAX_PROBLEMS];
  for (int p = 0; p < P; ++p) {
    const at::Tensor &x = xs[p], &a = a_pools[p], &b = b_pools[p], &y = ys[p];
    TORCH_CHECK(x.is_cuda() && a.is_cuda() && b.is_cuda() && y.is_cuda(), op, ": all tensors must be CUDA");
    TORCH_CHECK(x.dim() == 2 && x.stride(1) == 1 && y.dim() == 2 && y.stride(1) == 1, op,
                ": tensors must be contiguous");
    check_pool_a(a, op);
    check_pool_b(b, op);
    TORCH_CHECK(x.size(0) == T && y.size(0) == T, op, ": x / y rows must match slots");
    TORCH_CHECK(a.size(0) == S && a.size(1) == R && a.size(2) == x.size(1), op, ": a_pool shape mismatch");
    TORCH_CHECK(b.size(0) == S && b.size(2) == R && b.size(1) == y.size(1), op, ": b_pool shape mismatch");
    TORCH_CHECK(x.scalar_type() == xs[0].scalar_type() && a.scalar_type() == x.scalar_type() &&
                    b.scalar_type() == x.scalar_type() && y.scalar_type() == x.scalar_type(),
                op, ": dtype mismatch");
    TORCH_CHECK(x.get_device() == slots.get_device() && y.get_device() == slots.get_device(), op,
                ": tensors on different devices");
    probs[p] = persona_bgmv_problem{x.data_ptr(), row_stride(x), a.data_ptr(), a.stride(0), a.stride(1),
                                    b.data_ptr(), b.stride(0),   y.data_ptr(), row_stride(y), x.size(1),
                                    y.size(1)};
  }
  const at::cuda::OptionalCUDAGuard guard(slots.device());
  const int dev = slots.get_device();
  raise_pending(dev, op);
  if (T == 0) return;
  cudaStream_t stream = at::cuda::getCurrentCUDAStream();
  at::Tensor ws = plan.has_value() ? *plan : workspace_for(T, slots);
  const int flags = plan.has_value() ? PERSONA_REUSE_PLAN : 0;
  TORCH_CHECK(static_cast<size_t>(ws.numel()) >= persona_bgmv_multi_workspace_size(T, P), op,
              ": plan was built for fewer rows");
  check_status(persona_bgmv_fused_multi(probs, P, slots.data_ptr<int32_t>(), T, R, S, dt, ws.data_ptr(),
                                        ws.numel(), flags, error_word_device(dev), stream),
               op);
  after_launch(dev, op, stream);
}

at::Tensor plan_impl(const at::Tensor& slots, int64_t S) {
  const char* op = "bgmv_plan";
  TORCH_CHECK(slots.is_cuda(), "bgmv_plan: all tensors must be CUDA");
  TORCH_CHECK(slots.is_contiguous() && slots.dim() == 1, "bgmv_plan: tensors must be contiguous");
  TORCH_CHECK(slots.scalar_type() == at::kInt, "bgmv_plan: slots must be int32");
  const at::cuda::OptionalCUDAGuard guard(slots.device());
  const int dev = slots.get_device();
  raise_pending(dev, op);
  const int64_t T = slots.size(0);
  at::Tensor ws = workspace_for(T, slots);
  if (T == 0) return ws;
  cudaStream_t stream = at::cuda::getCurrentCUDAStream();
  check_status(persona_bgmv_plan(slots.data_ptr<int32_t>(), T, S, ws.data_ptr(), ws.numel(),
                                 error_word_device(dev), stream),
               op);
  after_launch(dev, op, stream);
  return ws;
}

}  // namespace

// Same C++ host symbols as the reference (csrc/bgmv_shrink.cu:81, csrc/bgmv_expand.cu:88).
void bgmv_shrink_cuda(const at::Tensor& x, const at::Tensor& a_pool, const at::Tensor& slots, at::Tensor& v) {
  shrink_impl(x, a_pool, slots, v, c10::nullopt);
}

void bgmv_expand_cuda(const at::Tensor& v, const at::Tensor& b_pool, const at::Tensor& slots, at::Tensor& y) {
  expand_impl(v, b_pool, slots, y, c10::nullopt);
}

namespace persona {
// Reference csrc/gemv_fp16.cu:33-50.
void gemv_fp16_cuda(const at::Tensor& x, const at::Tensor& W, at::Tensor& y) {
  TORCH_CHECK(x.is_cuda() && W.is_cuda() && y.is_cuda(), "gemv_fp16: CUDA only");
  TORCH_CHECK(x.dim() == 1 && W.dim() == 2 && y.dim() == 1, "gemv_fp16: shape");
  const int64_t K = x.size(0), N = W.size(0);
  TORCH_CHECK(W.size(1) == K && y.size(0) == N, "gemv_fp16: mismatch");
  TORCH_CHECK(x.scalar_type() == at::kHalf && W.scalar_type() == at::kHalf && y.scalar_type() == at::kHalf,
              "gemv_fp16: half only in v1 scaffold");
  TORCH_CHECK(x.is_contiguous() && W.is_contiguous() && y.is_contiguous(), "gemv_fp16: contiguous only");
  const at::cuda::OptionalCUDAGuard guard(x.device());
  check_status(persona_gemv_fp16(x.data_ptr(), W.data_ptr(), y.data_ptr(), K, N,
                                 at::cuda::getCurrentCUDAStream()),
               "gemv_fp16");
}
}  // namespace persona

namespace {
void shrink_with_plan(const at::Tensor& x, const at::Tensor& a_pool, const at::Tensor& slots,
                      const at::Tensor& plan, at::Tensor& v) {
  shrink_impl(x, a_pool, slots, v, plan);
}
void expand_with_plan(const at::Tensor& v, const at::Tensor& b_pool, const at::Tensor& slots,
                      const at::Tensor& plan, at::Tensor& y) {
  expand_impl(v, b_pool, slots, y, plan);
}
void fused_noplan(const at::Tensor& x, const at::Tensor& a_pool, const at::Tensor& b_pool,
                  const at::Tensor& slots, at::Tensor& y) {
  fused_impl(x, a_pool, b_pool, slots, y, c10::nullopt);
}
void fused_with_plan(const at::Tensor& x, const at::Tensor& a_pool, const at::Tensor& b_pool,
                     const at::Tensor& slots, const at::Tensor& plan, at::Tensor& y) {
  fused_impl(x, a_pool, b_pool, slots, y, plan);
}
}  // namespace

namespace {
void check_segments(const at::Tensor& indptr, const at::Tensor& seg_slots, const char* op) {
  TORCH_CHECK(indptr.is_cuda() && seg_slots.is_cuda(), op, ": all tensors must be CUDA");
  TORCH_CHECK(indptr.dim() == 1 && seg_slots.dim() == 1 && indptr.size(0) == seg_slots.size(0) + 1, op,
              ": seg_indptr must have one more entry than seg_slots");
  TORCH_CHECK(indptr.is_contiguous() && seg_slots.is_contiguous(), op, ": tensors must be contiguous");
  TORCH_CHECK(indptr.scalar_type() == at::kInt && seg_slots.scalar_type() == at::kInt, op,
              ": seg_indptr and seg_slots must be int32");
}

at::Tensor sgmv_workspace(int64_t T, const at::Tensor& like) {
  return at::empty({static_cast<int64_t>(persona_sgmv_workspace_size(T))}, like.options().dtype(at::kByte));
}

void sgmv_shrink_op(const at::Tensor& x, const at::Tensor& a_pool, const at::Tensor& indptr,
                    const at::Tensor& seg_slots, at::Tensor& v) {
  const char* op = "sgmv_shrink";
  check_segments(indptr, seg_slots, op);
  TORCH_CHECK(x.is_cuda() && a_pool.is_cuda() && v.is_cuda(), "sgmv_shrink: all tensors must be CUDA");
  TORCH_CHECK(x.dim() == 2 && x.stride(1) == 1 && v.is_contiguous(), "sgmv_shrink: tensors must be contiguous");
  check_pool_a(a_pool, op);
  TORCH_CHECK(v.scalar_type() == at::kFloat, "sgmv_shrink: v must be float32");
  const int64_t T = x.size(0), K = x.size(1), S = a_pool.size(0), R = a_pool.size(1);
  TORCH_CHECK(a_pool.size(2) == K, "sgmv_shrink: a_pool shape mismatch");
  TORCH_CHECK(v.dim() == 2 && v.size(0) == T && v.size(1) == R, "sgmv_shrink: v shape mismatch");
  const int dt = dtype_code(x, op);
  TORCH_CHECK(a_pool.scalar_type() == x.scalar_type(), "sgmv_shrink: dtype mismatch");
  const at::cuda::OptionalCUDAGuard guard(x.device());
  const int dev = x.get_device();
  raise_pending(dev, op);
  if (T == 0) return;
  at::Tensor ws = sgmv_workspace(T, x);
  cudaStream_t stream = at::cuda::getCurrentCUDAStream();
  check_status(persona_sgmv_shrink(x.data_ptr(), row_stride(x), a_pool.data_ptr(), a_pool.stride(0),
                                   a_pool.stride(1), indptr.data_ptr<int32_t>(), seg_slots.data_ptr<int32_t>(),
                                   seg_slots.size(0), v.data_ptr<float>(), T, K, R, S, dt, ws.data_ptr(),
                                   ws.numel(), error_word_device(dev), stream),
               op);
  after_launch(dev, op, stream);
}

void sgmv_expand_op(const at::Tensor& v, const at::Tensor& b_pool, const at::Tensor& indptr,
                    const at::Tensor& seg_slots, at::Tensor& y) {
  const char* op = "sgmv_expand";
  check_segments(indptr, seg_slots, op);
  TORCH_CHECK(v.is_cuda() && b_pool.is_cuda() && y.is_cuda(), "sgmv_expand: all tensors must be CUDA");
  TORCH_CHECK(v.is_contiguous() && y.dim() == 2 && y.stride(1) == 1, "sgmv_expand: tensors must be contiguous");
  check_pool_b(b_pool, op);
  TORCH_CHECK(v.scalar_type() == at::kFloat, "sgmv_expand: v must be float32");
  const int64_t T = v.size(0), R = v.size(1), S = b_pool.size(0), N = b_pool.size(1);
  TORCH_CHECK(b_pool.size(2) == R, "sgmv_expand: b_pool rank dim mismatch");
  TORCH_CHECK(y.size(0) == T && y.size(1) == N, "sgmv_expand: y shape mismatch");
  const int dt = dtype_code(y, op);
  TORCH_CHECK(b_pool.scalar_type() == y.scalar_type(), "sgmv_expand: dtype mismatch");
  const at::cuda::OptionalCUDAGuard guard(v.device());
  const int dev = v.get_device();
  raise_pending(dev, op);
  if (T == 0) return;
  at::Tensor ws = sgmv_workspace(T, v);
  cudaStream_t stream = at::cuda::getCurrentCUDAStream();
  check_status(persona_sgmv_expand(v.data_ptr<float>(), b_pool.data_ptr(), b_pool.stride(0),
                                   indptr.data_ptr<int32_t>(), seg_slots.data_ptr<int32_t>(), seg_slots.size(0),
                                   y.data_ptr(), row_stride(y), T, N, R, S, dt, ws.data_ptr(), ws.numel(),
                                   error_word_device(dev), stream),
               op);
  after_launch(dev, op, stream);
}

void sgmv_fused_op(const at::Tensor& x, const at::Tensor& a_pool, const at::Tensor& b_pool,
                   const at::Tensor& indptr, const at::Tensor& seg_slots, at::Tensor& y) {
  const char* op = "sgmv_fused";
  check_segments(indptr, seg_slots, op);
  TORCH_CHECK(x.is_cuda() && a_pool.is_cuda() && b_pool.is_cuda() && y.is_cuda(),
              "sgmv_fused: all tensors must be CUDA");
  TORCH_CHECK(x.dim() == 2 && x.stride(1) == 1 && y.dim() == 2 && y.stride(1) == 1,
              "sgmv_fused: tensors must be contiguous");
  check_pool_a(a_pool, op);
  check_pool_b(b_pool, op);
  const int64_t T = x.size(0), K = x.size(1), S = a_pool.size(0), R = a_pool.size(1), N = b_pool.size(1);
  TORCH_CHECK(a_pool.size(2) == K && b_pool.size(0) == S && b_pool.size(2) == R, "sgmv_fused: pool shape mismatch");
  TORCH_CHECK(y.size(0) == T && y.size(1) == N, "sgmv_fused: y shape mismatch");
  const int dt = dtype_code(x, op);
  TORCH_CHECK(a_pool.scalar_type() == x.scalar_type() && b_pool.scalar_type() == x.scalar_type() &&
                  y.scalar_type() == x.scalar_type(),
              "sgmv_fused: dtype mismatch");
  const at::cuda::OptionalCUDAGuard guard(x.device());
  const int dev = x.get_device();
  raise_pending(dev, op);
  if (T == 0) return;
  at::Tensor ws = sgmv_workspace(T, x);
  cudaStream_t stream = at::cuda::getCurrentCUDAStream();
  check_status(persona_sgmv_fused(x.data_ptr(), row_stride(x), a_pool.data_ptr(), a_pool.stride(0),
                                  a_pool.stride(1), b_pool.data_ptr(), b_pool.stride(0), indptr.data_ptr<int32_t>(),
                                  seg_slots.data_ptr<int32_t>(), seg_slots.size(0), y.data_ptr(), row_stride(y), T,
                                  K, N, R, S, dt, ws.data_ptr(), ws.numel(), error_word_device(dev), stream),
               op);
  after_launch(dev, op, stream);
}
}  // namespace

namespace {
// ------------------------------------------------------------------ NF4 ---
// Base linears of the end-to-end decode (persona_nf4_* in the C ABI).
std::tuple<at::Tensor, at::Tensor> nf4_quantize_op(const at::Tensor& w) {
  const char* op = "nf4_quantize";
  TORCH_CHECK(w.is_cuda() && w.dim() == 2 && w.stride(1) == 1, op, ": w must be a CUDA [N, K] matrix");
  TORCH_CHECK(w.scalar_type() == at::kHalf, op, ": w must be float16");
  const int64_t N = w.size(0), K = w.size(1);
  TORCH_CHECK(N % 128 == 0 && K % 128 == 0 && N > 0 && K > 0, op, ": N and K must be multiples of 128");
  const at::cuda::OptionalCUDAGuard guard(w.device());
  auto u8 = w.options().dtype(at::kByte);
  at::Tensor packed = at::empty({N / 128, K / 128, PERSONA_NF4_CHUNK_BYTES}, u8);
  at::Tensor offset = at::empty({1}, w.options().dtype(at::kFloat));
  at::Tensor ws = at::empty({static_cast<int64_t>(persona_nf4_quantize_workspace_size(N, K))}, u8);
  cudaStream_t stream = at::cuda::getCurrentCUDAStream();
  check_status(persona_nf4_quantize(w.data_ptr(), row_stride(w), N, K, packed.data_ptr(), offset.data_ptr<float>(),
                                    ws.data_ptr(), ws.numel(), stream),
               op);
  after_launch(w.get_device(), op, stream);
  return {packed, offset};
}

void check_nf4_weight(const at::Tensor& packed, const at::Tensor& offset, int64_t N, int64_t K, const char* op) {
  TORCH_CHECK(packed.is_cuda() && offset.is_cuda(), op, ": tensors must be CUDA");
  TORCH_CHECK(packed.scalar_type() == at::kByte && packed.is_contiguous() && packed.dim() == 3 &&
                  packed.size(0) * 128 == N && packed.size(1) * 128 == K && packed.size(2) == PERSONA_NF4_CHUNK_BYTES,
              op, ": packed must be uint8 [N/128, K/128, ", PERSONA_NF4_CHUNK_BYTES, "]");
  TORCH_CHECK(offset.scalar_type() == at::kFloat && offset.numel() == 1, op, ": offset must be one float32");
}

at::Tensor nf4_dequantize_op(const at::Tensor& packed, const at::Tensor& offset, int64_t N, int64_t K) {
  const char* op = "nf4_dequantize";
  check_nf4_weight(packed, offset, N, K, op);
  const at::cuda::OptionalCUDAGuard guard(packed.device());
  at::Tensor w = at::empty({N, K}, packed.options().dtype(at::kHalf));
  cudaStream_t stream = at::cuda::getCurrentCUDAStream();
  check_status(persona_nf4_dequantize(packed.data_ptr(), offset.data_ptr<float>(), N, K, w.data_ptr(), K, stream),
               op);
  after_launch(packed.get_device(), op, stream);
  return w;
}

// Workspace of the NF4 linear on a stream, whose counters are zeroed when it is
// made (the kernel leaves them at zero).  Calls on two streams never share one,
// nor do two captured graphs: each capture makes its own, in the graph's memory,
// zeroed once per replay (64 KB and more of counters, so that it is made once).
// Kept for the streams used last; what is freed stays its stream's until the
// launches there have run, so a stream that comes back just makes another.
at::Tensor nf4_workspace(const persona_nf4_problem* probs, int n, const at::Tensor& like, cudaStream_t stream) {
  struct Entry {
    cudaStream_t stream;
    unsigned long long capture;  // 0: none
    at::Tensor t;
  };
  static std::mutex mu;
  static auto* const made = new std::vector<Entry>[kMaxDevices];  // (lives on: no tensor is freed behind the context)
  const int dev = like.get_device();
  TORCH_CHECK(dev >= 0 && dev < kMaxDevices, "nf4_linear: device index out of range");
  const int64_t bytes = static_cast<int64_t>(persona_nf4_linear_workspace_size(probs, n));
  cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
  unsigned long long capture = 0;
  C10_CUDA_CHECK(cudaStreamGetCaptureInfo(stream, &status, &capture));
  if (status == cudaStreamCaptureStatusNone) capture = 0;
  std::lock_guard<std::mutex> lock(mu);
  std::vector<Entry>& list = made[dev];
  if (capture != 0)  // those of a graph that has been captured belong to it alone
    list.erase(std::remove_if(list.begin(), list.end(),
                              [&](const Entry& e) { return e.capture != 0 && e.capture != capture; }),
               list.end());
  auto e = std::find_if(list.begin(), list.end(),
                        [&](const Entry& x) { return x.stream == stream && x.capture == capture; });
  if (e == list.end()) {
    constexpr size_t kStreams = 8;  // 19 MB each
    if (list.size() >= kStreams) list.erase(list.begin());
    list.push_back(Entry{stream, capture, at::Tensor()});
  } else {
    std::rotate(e, e + 1, list.end());  // (the one used last is the last)
  }
  e = list.end() - 1;
  if (!e->t.defined() || e->t.numel() < bytes) {
    const int64_t from = static_cast<int64_t>(persona_nf4_linear_counter_offset());
    e->t = at::Tensor();
    e->t = at::empty({std::max(bytes, from + 65536)}, like.options().dtype(at::kByte));
    e->t.narrow(0, from, e->t.numel() - from).zero_();
  }
  return e->t;
}

void nf4_linear_op(const at::Tensor& x, at::TensorList packed, at::TensorList offsets, at::TensorList ys) {
  const char* op = "nf4_linear";
  const int n = static_cast<int>(packed.size());
  TORCH_CHECK(n >= 1 && n <= PERSONA_NF4_MAX_PROBLEMS, op, ": 1 to ", PERSONA_NF4_MAX_PROBLEMS, " weights");
  TORCH_CHECK(static_cast<int>(offsets.size()) == n && static_cast<int>(ys.size()) == n, op,
              ": one offset and one y per weight");
  TORCH_CHECK(x.is_cuda() && x.dim() == 2 && x.stride(1) == 1 && x.scalar_type() == at::kHalf, op,
              ": x must be a CUDA float16 [M, K] matrix with unit inner stride");
  const int64_t M = x.size(0), K = x.size(1);
  persona_nf4_problem probs[PERSONA_NF4_MAX_PROBLEMS];
  for (int i = 0; i < n; ++i) {
    const at::Tensor& y = ys[i];
    TORCH_CHECK(y.is_cuda() && y.dim() == 2 && y.stride(1) == 1 && y.scalar_type() == at::kHalf && y.size(0) == M,
                op, ": y must be a CUDA float16 [M, N] matrix with unit inner stride");
    const int64_t N = y.size(1);
    check_nf4_weight(packed[i], offsets[i], N, K, op);
    TORCH_CHECK(packed[i].get_device() == x.get_device() && y.get_device() == x.get_device(), op,
                ": tensors must be on one device");
    probs[i] = persona_nf4_problem{packed[i].data_ptr(), offsets[i].data_ptr<float>(), x.data_ptr(), row_stride(x),
                                   y.data_ptr(), row_stride(y), N, K};
  }
  const at::cuda::OptionalCUDAGuard guard(x.device());
  const int dev = x.get_device();
  raise_pending(dev, op);
  if (M == 0) return;
  cudaStream_t stream = at::cuda::getCurrentCUDAStream();
  at::Tensor ws = nf4_workspace(probs, n, x, stream);
  check_status(persona_nf4_linear(probs, n, M, ws.data_ptr(), ws.numel(), error_word_device(dev), stream), op);
  after_launch(dev, op, stream);
}
}  // namespace

namespace {
// ---------------------------------------------------- decode helpers ----
void check_half_cuda(const at::Tensor& t, const char* op) {
  TORCH_CHECK(t.is_cuda() && t.scalar_type() == at::kHalf && t.is_contiguous(), op,
              ": tensors must be contiguous CUDA float16");
}

void add_rmsnorm_op(at::Tensor& h, const c10::optional<at::Tensor>& delta, const at::Tensor& w, at::Tensor& out,
                    double eps) {
  const char* op = "add_rmsnorm";
  check_half_cuda(h, op);
  check_half_cuda(w, op);
  check_half_cuda(out, op);
  const int64_t D = h.size(-1), rows = h.numel() / D;
  TORCH_CHECK(w.numel() == D && out.numel() == h.numel(), op, ": shape mismatch");
  if (delta.has_value()) {
    check_half_cuda(*delta, op);
    TORCH_CHECK(delta->numel() == h.numel(), op, ": delta shape mismatch");
  }
  const at::cuda::OptionalCUDAGuard guard(h.device());
  cudaStream_t stream = at::cuda::getCurrentCUDAStream();
  check_status(persona_add_rmsnorm(h.data_ptr(), delta.has_value() ? delta->data_ptr() : nullptr, w.data_ptr(),
                                   out.data_ptr(), rows, D, static_cast<float>(eps), stream),
               op);
}

void rope_cache_op(at::Tensor& q, at::Tensor& k, const at::Tensor& v, at::Tensor& k_cache, at::Tensor& v_cache,
                   const at::Tensor& start, int64_t per_seq, double theta) {
  const char* op = "rope_cache";
  for (const at::Tensor* t : std::initializer_list<const at::Tensor*>{&q, &k, &v, &k_cache, &v_cache})
    check_half_cuda(*t, op);
  TORCH_CHECK(q.dim() == 3 && k.dim() == 3 && v.sizes() == k.sizes() && q.size(2) == 128 && k.size(2) == 128 &&
                  q.size(0) == k.size(0),
              op, ": q [rows, Hq, 128], k / v [rows, Hkv, 128]");
  TORCH_CHECK(k_cache.dim() == 4 && v_cache.sizes() == k_cache.sizes() && k_cache.size(1) == k.size(1) &&
                  k_cache.size(3) == 128 && k_cache.size(0) * per_seq == q.size(0),
              op, ": caches [B, Hkv, L, 128] with B * per_seq rows");
  TORCH_CHECK(start.is_cuda() && start.scalar_type() == at::kInt && start.numel() >= 1, op,
              ": start must be a CUDA int32 scalar");
  const at::cuda::OptionalCUDAGuard guard(q.device());
  cudaStream_t stream = at::cuda::getCurrentCUDAStream();
  check_status(persona_rope_cache(q.data_ptr(), k.data_ptr(), v.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(),
                                  start.data_ptr<int32_t>(), q.size(0), per_seq, q.size(1), k.size(1),
                                  k_cache.size(2), static_cast<float>(theta), stream),
               op);
}

void silu_mul_op(const at::Tensor& g, const at::Tensor& u, at::Tensor& out) {
  const char* op = "silu_mul";
  check_half_cuda(g, op);
  check_half_cuda(u, op);
  check_half_cuda(out, op);
  TORCH_CHECK(g.numel() == u.numel() && out.numel() == g.numel(), op, ": shape mismatch");
  const at::cuda::OptionalCUDAGuard guard(g.device());
  cudaStream_t stream = at::cuda::getCurrentCUDAStream();
  check_status(persona_silu_mul(g.data_ptr(), u.data_ptr(), out.data_ptr(), g.numel(), stream), op);
}

void rope_decode_attention_op(at::Tensor& q, at::Tensor& k, const at::Tensor& v, at::Tensor& k_cache,
                              at::Tensor& v_cache, const at::Tensor& pos, const at::Tensor& len, at::Tensor& out,
                              double theta, double scale) {
  const char* op = "rope_decode_attention";
  for (const at::Tensor* t : std::initializer_list<const at::Tensor*>{&q, &k, &v, &k_cache, &v_cache, &out})
    check_half_cuda(*t, op);
  TORCH_CHECK(q.dim() == 3 && q.size(2) == 128 && out.sizes() == q.sizes() && k.dim() == 3 && v.sizes() == k.sizes() &&
                  k.size(2) == 128 && k.size(0) == q.size(0),
              op, ": q, out [B, Hq, 128], k / v [B, Hkv, 128]");
  TORCH_CHECK(k_cache.dim() == 4 && v_cache.sizes() == k_cache.sizes() && k_cache.size(0) == q.size(0) &&
                  k_cache.size(1) == k.size(1) && k_cache.size(3) == 128,
              op, ": caches [B, Hkv, L, 128]");
  TORCH_CHECK(pos.is_cuda() && pos.scalar_type() == at::kInt && pos.numel() >= 1 && len.is_cuda() &&
                  len.scalar_type() == at::kInt && len.numel() >= 1,
              op, ": pos and len must be CUDA int32 scalars");
  const at::cuda::OptionalCUDAGuard guard(q.device());
  cudaStream_t stream = at::cuda::getCurrentCUDAStream();
  check_status(persona_rope_decode_attention(q.data_ptr(), k.data_ptr(), v.data_ptr(), k_cache.data_ptr(),
                                             v_cache.data_ptr(), pos.data_ptr<int32_t>(), len.data_ptr<int32_t>(),
                                             out.data_ptr(), q.size(0), q.size(1), k.size(1), k_cache.size(2),
                                             static_cast<float>(theta), static_cast<float>(scale), stream),
               op);
}

void decode_attention_op(const at::Tensor& q, const at::Tensor& k_cache, const at::Tensor& v_cache,
                         const at::Tensor& len, at::Tensor& out, double scale) {
  const char* op = "decode_attention";
  for (const at::Tensor* t : std::initializer_list<const at::Tensor*>{&q, &k_cache, &v_cache, &out})
    check_half_cuda(*t, op);
  TORCH_CHECK(q.dim() == 3 && q.size(2) == 128 && out.sizes() == q.sizes(), op, ": q, out [B, Hq, 128]");
  TORCH_CHECK(k_cache.dim() == 4 && v_cache.sizes() == k_cache.sizes() && k_cache.size(0) == q.size(0) &&
                  k_cache.size(3) == 128,
              op, ": caches [B, Hkv, L, 128]");
  TORCH_CHECK(len.is_cuda() && len.scalar_type() == at::kInt && len.numel() >= 1, op,
              ": len must be a CUDA int32 scalar");
  const at::cuda::OptionalCUDAGuard guard(q.device());
  cudaStream_t stream = at::cuda::getCurrentCUDAStream();
  check_status(persona_decode_attention(q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), len.data_ptr<int32_t>(),
                                        out.data_ptr(), q.size(0), q.size(1), k_cache.size(1), k_cache.size(2),
                                        static_cast<float>(scale), stream),
               op);
}
}  // namespace

namespace {
// LoRA term alone at decode sizes (persona_bgmv_lora_delta_multi): deltas[i]
// is fp32 [T, N_i]; the base projection adds it (nf4_linear_add).
void lora_delta_multi_op(at::TensorList xs, at::TensorList a_pools, at::TensorList b_pools, const at::Tensor& slots,
                         at::TensorList deltas) {
  const char* op = "bgmv_lora_delta_multi";
  const int P = static_cast<int>(xs.size());
  TORCH_CHECK(P >= 1 && P <= PERSONA_MAX_PROBLEMS, op, ": 1 to ", PERSONA_MAX_PROBLEMS, " projections");
  TORCH_CHECK(a_pools.size() == xs.size() && b_pools.size() == xs.size() && deltas.size() == xs.size(), op,
              ": xs, a_pools, b_pools and deltas must have the same length");
  TORCH_CHECK(slots.is_cuda() && slots.is_contiguous() && slots.dim() == 1 && slots.scalar_type() == at::kInt, op,
              ": slots must be a contiguous int32 CUDA vector");
  const int64_t T = slots.size(0);
  const int64_t S = a_pools[0].size(0), R = a_pools[0].size(1);
  const int dt = dtype_code(xs[0], op);
  persona_bgmv_problem probs[PERSONA_MAX_PROBLEMS];
  float* dptr[PERSONA_MAX_PROBLEMS];
  int64_t dld[PERSONA_MAX_PROBLEMS];
  for (int p = 0; p < P; ++p) {
    const at::Tensor &x = xs[p], &a = a_pools[p], &b = b_pools[p], &d = deltas[p];
    TORCH_CHECK(x.is_cuda() && a.is_cuda() && b.is_cuda() && d.is_cuda(), op, ": all tensors must be CUDA");
    TORCH_CHECK(x.dim() == 2 && x.stride(1) == 1 && d.dim() == 2 && d.stride(1) == 1, op,
                ": tensors must be contiguous");
    TORCH_CHECK(d.scalar_type() == at::kFloat, op, ": deltas must be float32");
    check_pool_a(a, op);
    check_pool_b(b, op);
    TORCH_CHECK(x.size(0) == T && d.size(0) == T, op, ": x / delta rows must match slots");
    TORCH_CHECK(a.size(0) == S && a.size(1) == R && a.size(2) == x.size(1), op, ": a_pool shape mismatch");
    TORCH_CHECK(b.size(0) == S && b.size(2) == R && b.size(1) == d.size(1), op, ": b_pool shape mismatch");
    TORCH_CHECK(x.scalar_type() == xs[0].scalar_type() && a.scalar_type() == x.scalar_type() &&
                    b.scalar_type() == x.scalar_type(),
                op, ": dtype mismatch");
    probs[p] = persona_bgmv_problem{x.data_ptr(), row_stride(x), a.data_ptr(), a.stride(0), a.stride(1),
                                    b.data_ptr(), b.stride(0),   nullptr,      0,            x.size(1),
                                    d.size(1)};
    dptr[p] = d.data_ptr<float>();
    dld[p] = row_stride(d);
  }
  const at::cuda::OptionalCUDAGuard guard(slots.device());
  const int dev = slots.get_device();
  raise_pending(dev, op);
  cudaStream_t stream = at::cuda::getCurrentCUDAStream();
  check_status(persona_bgmv_lora_delta_multi(probs, P, dptr, dld, slots.data_ptr<int32_t>(), T, R, S, dt,
                                             error_word_device(dev), stream),
               op);
  after_launch(dev, op, stream);
}

void nf4_linear_add_op(const at::Tensor& x, at::TensorList packed, at::TensorList offsets, at::TensorList addends,
                       at::TensorList ys) {
  const char* op = "nf4_linear_add";
  const int n = static_cast<int>(packed.size());
  TORCH_CHECK(n >= 1 && n <= PERSONA_NF4_MAX_PROBLEMS, op, ": 1 to ", PERSONA_NF4_MAX_PROBLEMS, " weights");
  TORCH_CHECK(static_cast<int>(offsets.size()) == n && static_cast<int>(ys.size()) == n &&
                  static_cast<int>(addends.size()) == n,
              op, ": one offset, one addend and one y per weight");
  TORCH_CHECK(x.is_cuda() && x.dim() == 2 && x.stride(1) == 1 && x.scalar_type() == at::kHalf, op,
              ": x must be a CUDA float16 [M, K] matrix with unit inner stride");
  const int64_t M = x.size(0), K = x.size(1);
  persona_nf4_problem probs[PERSONA_NF4_MAX_PROBLEMS];
  const float* add[PERSONA_NF4_MAX_PROBLEMS];
  int64_t ldadd[PERSONA_NF4_MAX_PROBLEMS];
  for (int i = 0; i < n; ++i) {
    const at::Tensor& y = ys[i];
    const at::Tensor& d = addends[i];
    TORCH_CHECK(y.is_cuda() && y.dim() == 2 && y.stride(1) == 1 && y.scalar_type() == at::kHalf && y.size(0) == M,
                op, ": y must be a CUDA float16 [M, N] matrix with unit inner stride");
    const int64_t N = y.size(1);
    TORCH_CHECK(d.is_cuda() && d.dim() == 2 && d.stride(1) == 1 && d.scalar_type() == at::kFloat &&
                    d.size(0) == M && d.size(1) == N,
                op, ": addend must be a CUDA float32 [M, N] matrix with unit inner stride");
    check_nf4_weight(packed[i], offsets[i], N, K, op);
    probs[i] = persona_nf4_problem{packed[i].data_ptr(), offsets[i].data_ptr<float>(), x.data_ptr(), row_stride(x),
                                   y.data_ptr(), row_stride(y), N, K};
    add[i] = d.data_ptr<float>();
    ldadd[i] = row_stride(d);
  }
  const at::cuda::OptionalCUDAGuard guard(x.device());
  const int dev = x.get_device();
  raise_pending(dev, op);
  if (M == 0) return;
  cudaStream_t stream = at::cuda::getCurrentCUDAStream();
  at::Tensor ws = nf4_workspace(probs, n, x, stream);
  check_status(persona_nf4_linear_add(probs, n, add, ldadd, M, ws.data_ptr(), ws.numel(), error_word_device(dev),
                                      stream),
               op);
  after_launch(dev, op, stream);
}
}  // namespace

namespace {
// ------------------------------------------- paged cache, draft checks ----
void check_index(const at::Tensor& t, int64_t dim, const at::Tensor& like, const char* op, const char* name) {
  TORCH_CHECK(t.is_cuda() && t.scalar_type() == at::kInt && t.dim() == dim && (t.numel() == 0 || t.stride(dim - 1) == 1),
              op, ": ", name, " must be a CUDA int32 tensor with ", dim, " dimension(s) and unit inner stride");
  TORCH_CHECK(t.get_device() == like.get_device(), op, ": tensors on different devices");
}

// A [rows, heads, D] activation of the batch; sizes already checked.
persona_rows rows_of(const at::Tensor& t, const at::Tensor& like, const char* op, const char* name, bool written) {
  TORCH_CHECK(t.is_cuda() && t.dim() == 3 && t.stride(2) == 1, op, ": ", name,
              " must be a CUDA [rows, heads, D] tensor with unit inner stride");
  TORCH_CHECK(t.scalar_type() == like.scalar_type(), op, ": dtype mismatch");
  TORCH_CHECK(t.get_device() == like.get_device(), op, ": tensors on different devices");
  TORCH_CHECK(t.size(0) == like.size(0) && t.size(2) == like.size(2), op, ": ", name, " shape mismatch");
  TORCH_CHECK(!written || ((t.size(0) <= 1 || t.stride(0) >= t.size(2)) && (t.size(1) <= 1 || t.stride(1) >= t.size(2))),
              op, ": ", name, " is written and must not overlap itself");
  return persona_rows{t.data_ptr(), t.size(0) <= 1 ? 0 : t.stride(0), t.size(1) <= 1 ? 0 : t.stride(1)};
}

// Whether two [rows, heads, D] activations share an element: exact where they
// step alike, as slices of one buffer do, elsewhere whether their ranges meet.
bool rows_meet(const at::Tensor& a, const at::Tensor& b) {
  const auto view = [](const at::Tensor& t) {
    const int64_t e = t.element_size();
    return persona::overlap::View{t.data_ptr(), t.size(2) * e, {t.size(0), t.size(1), 1}, {t.stride(0) * e, t.stride(1) * e, 0}};
  };
  return persona::overlap::share(view(a), view(b));
}

bool same_rows(const at::Tensor& a, const at::Tensor& b) {
  return a.data_ptr() == b.data_ptr() && a.sizes() == b.sizes() && a.strides() == b.strides();
}

persona_paged_cache cache_of(const at::Tensor& k_cache, const at::Tensor& v_cache, const c10::optional<at::Tensor>& k_scale,
                             const c10::optional<at::Tensor>& v_scale, const at::Tensor& table, const at::Tensor& indptr,
                             const at::Tensor& lengths, const at::Tensor& like, const char* op) {
  TORCH_CHECK(k_cache.is_cuda() && v_cache.is_cuda() && k_cache.dim() == 4 && k_cache.stride(3) == 1, op,
              ": caches must be CUDA [pages, kv heads, page size, D] tensors with unit inner stride");
  TORCH_CHECK(v_cache.sizes() == k_cache.sizes() && v_cache.strides() == k_cache.strides() &&
                  v_cache.scalar_type() == k_cache.scalar_type(),
              op, ": k and v caches must have the same type, shape and strides");
  TORCH_CHECK(k_cache.get_device() == like.get_device() && v_cache.get_device() == like.get_device(), op,
              ": tensors on different devices");
  TORCH_CHECK(k_cache.size(3) == like.size(2), op, ": cache head size mismatch");
  TORCH_CHECK(like.size(2) == 64 || like.size(2) == 128, op, ": head size must be 64 or 128");
  const bool e4m3 = k_cache.scalar_type() == at::kFloat8_e4m3fn;
  TORCH_CHECK(e4m3 || k_cache.scalar_type() == like.scalar_type(), op,
              ": caches must have the activations' type or be float8_e4m3fn");
  TORCH_CHECK(k_scale.has_value() == e4m3 && v_scale.has_value() == e4m3, op,
              ": k_scale and v_scale go with float8_e4m3fn caches, and only with them");
  persona_paged_cache c = {};
  c.k = k_cache.data_ptr();
  c.v = v_cache.data_ptr();
  c.num_pages = k_cache.size(0);
  c.Hkv = k_cache.size(1);
  c.page_size = k_cache.size(2);
  c.D = k_cache.size(3);
  // the stride of a dimension of one is never used
  c.page_stride = c.num_pages <= 1 ? 0 : k_cache.stride(0);
  c.head_stride = c.Hkv <= 1 ? 0 : k_cache.stride(1);
  c.pos_stride = c.page_size <= 1 ? c.D : k_cache.stride(2);
  c.kind = e4m3 ? PERSONA_PAGES_E4M3 : PERSONA_PAGES_16BIT;
  if (e4m3) {
    const int64_t n = k_scale->dim() == 3 ? k_scale->size(2) : 0;  // scales of a page
    for (const at::Tensor* t : {&*k_scale, &*v_scale}) {
      TORCH_CHECK(t->is_cuda() && t->scalar_type() == at::kFloat && t->dim() == 3 && t->size(0) == c.num_pages &&
                      t->size(1) == c.Hkv && t->size(2) == n && (n <= 1 || t->stride(2) == 1) &&
                      t->strides() == k_scale->strides() && t->get_device() == like.get_device(),
                  op, ": scales must be float32 [pages, kv heads, page size or blocks of a page] with unit inner stride, "
                      "strides alike");
    }
    int shift = 0;
    while (shift < 7 && (n << shift) < c.page_size) ++shift;
    TORCH_CHECK(n << shift == c.page_size, op,
                ": a page has a scale per position, or per block of 2, 4, ... 128 of them");
    c.kind = PERSONA_PAGES_E4M3_BLOCK(shift);
    c.k_scale = k_scale->data_ptr<float>();
    c.v_scale = v_scale->data_ptr<float>();
    c.scale_page_stride = c.num_pages <= 1 ? 0 : k_scale->stride(0);
    c.scale_head_stride = c.Hkv <= 1 ? 0 : k_scale->stride(1);
  }
  check_index(table, 2, like, op, "page_table");
  check_index(indptr, 1, like, op, "indptr");
  check_index(lengths, 1, like, op, "lengths");
  c.B = lengths.size(0);
  TORCH_CHECK(indptr.size(0) == c.B + 1 && table.size(0) == c.B, op,
              ": indptr [B + 1], lengths [B] and page_table [B, max pages] do not agree");
  c.page_table = table.data_ptr<int32_t>();
  c.max_pages = table.size(1);
  c.table_stride = c.B <= 1 ? c.max_pages : table.stride(0);
  c.indptr = indptr.data_ptr<int32_t>();
  c.lengths = lengths.data_ptr<int32_t>();
  return c;
}

void paged_rope_cache_op(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, at::Tensor& q_out,
                         at::Tensor& k_cache, at::Tensor& v_cache, const at::Tensor& page_table, const at::Tensor& indptr,
                         const at::Tensor& lengths, double theta, const c10::optional<at::Tensor>& k_scale,
                         const c10::optional<at::Tensor>& v_scale) {
  const char* op = "paged_rope_cache";
  const persona_rows qr = rows_of(q, q, op, "q", false), kr = rows_of(k, q, op, "k", false),
                     vr = rows_of(v, q, op, "v", false), qo = rows_of(q_out, q, op, "q_out", true);
  const int dt = dtype_code(q, op);
  const persona_paged_cache c = cache_of(k_cache, v_cache, k_scale, v_scale, page_table, indptr, lengths, q, op);
  TORCH_CHECK(k.size(1) == c.Hkv && v.size(1) == c.Hkv && q_out.size(1) == q.size(1), op, ": head count mismatch");
  TORCH_CHECK((c.num_pages <= 1 || c.page_stride >= c.D) && (c.Hkv <= 1 || c.head_stride >= c.D), op,
              ": caches are written and must not overlap themselves");
  const at::cuda::OptionalCUDAGuard guard(q.device());
  const int dev = q.get_device();
  raise_pending(dev, op);
  if (q.size(0) == 0) return;
  cudaStream_t stream = at::cuda::getCurrentCUDAStream();
  const int st = persona_paged_rope_cache(&c, &qr, &qo, &kr, &vr, q.size(0), q.size(1), static_cast<float>(theta), dt,
                                          error_word_device(dev), stream);
  if (st == PERSONA_ERR_OVERLAP) {  // which
    TORCH_CHECK(same_rows(q, q_out) || !rows_meet(q, q_out), op, ": q_out must be q or not overlap it");
    TORCH_CHECK(!rows_meet(k, q_out) && !rows_meet(v, q_out), op, ": q_out must not overlap k or v");
  }
  check_status(st, op);
  after_launch(dev, op, stream);
}

void paged_cache_read_op(const at::Tensor& k_cache, const at::Tensor& v_cache, const at::Tensor& page_table,
                         const at::Tensor& indptr, const at::Tensor& lengths, at::Tensor& k_out, at::Tensor& v_out,
                         const c10::optional<at::Tensor>& k_scale, const c10::optional<at::Tensor>& v_scale) {
  const char* op = "paged_cache_read";
  const persona_rows kr = rows_of(k_out, k_out, op, "k_out", true), vr = rows_of(v_out, k_out, op, "v_out", true);
  const int dt = dtype_code(k_out, op);
  const persona_paged_cache c = cache_of(k_cache, v_cache, k_scale, v_scale, page_table, indptr, lengths, k_out, op);
  TORCH_CHECK(k_out.size(1) == c.Hkv && v_out.size(1) == c.Hkv, op, ": head count mismatch");
  const at::cuda::OptionalCUDAGuard guard(k_out.device());
  const int dev = k_out.get_device();
  raise_pending(dev, op);
  if (k_out.size(0) == 0) return;
  cudaStream_t stream = at::cuda::getCurrentCUDAStream();
  const int st = persona_paged_cache_read(&c, &kr, &vr, k_out.size(0), dt, error_word_device(dev), stream);
  TORCH_CHECK(st != PERSONA_ERR_OVERLAP || !rows_meet(k_out, v_out), op, ": k_out and v_out must not overlap");
  check_status(st, op);
  after_launch(dev, op, stream);
}

void paged_attention_op(const at::Tensor& q, const at::Tensor& k_cache, const at::Tensor& v_cache,
                        const at::Tensor& page_table, const at::Tensor& indptr, const at::Tensor& lengths, at::Tensor& out,
                        double scale, int64_t window, int64_t max_new, const c10::optional<at::Tensor>& k_scale,
                        const c10::optional<at::Tensor>& v_scale) {
  const char* op = "paged_attention";
  const persona_rows qr = rows_of(q, q, op, "q", false), orow = rows_of(out, q, op, "out", true);
  const int dt = dtype_code(q, op);
  const persona_paged_cache c = cache_of(k_cache, v_cache, k_scale, v_scale, page_table, indptr, lengths, q, op);
  TORCH_CHECK(out.size(1) == q.size(1) && c.Hkv > 0 && q.size(1) % c.Hkv == 0, op,
              ": the heads of q and out must be a multiple of the kv heads");
  TORCH_CHECK(window >= 0, op, ": window must not be negative (0: none)");
  TORCH_CHECK(max_new >= 1, op, ": max_new must be positive");
  const at::cuda::OptionalCUDAGuard guard(q.device());
  const int dev = q.get_device();
  raise_pending(dev, op);
  if (q.size(0) == 0 || c.B == 0) return;
  cudaStream_t stream = at::cuda::getCurrentCUDAStream();
  // a buffer of this call's own (from the graph's pool under capture)
  at::Tensor ws = at::empty({static_cast<int64_t>(persona_paged_attention_workspace_size(c.D))},
                            q.options().dtype(at::kByte));
  const int st = persona_paged_attention(&c, &qr, &orow, q.size(0), q.size(1), static_cast<float>(scale), window, max_new,
                                         dt, ws.data_ptr(), ws.numel(), error_word_device(dev), stream);
  TORCH_CHECK(st != PERSONA_ERR_OVERLAP || !rows_meet(q, out), op, ": out must not overlap q");
  check_status(st, op);
  after_launch(dev, op, stream);
}

void paged_plan_op(const at::Tensor& add, at::Tensor& lengths, at::Tensor& page_table, at::Tensor& free_pages,
                   at::Tensor& num_free, int64_t page_size, at::Tensor& indptr, at::Tensor& places,
                   const c10::optional<at::Tensor>& keep, const c10::optional<at::Tensor>& seq_slots,
                   const c10::optional<at::Tensor>& row_slots) {
  const char* op = "paged_plan";
  const int64_t B = lengths.dim() == 1 ? lengths.size(0) : -1;
  auto vec = [&](const at::Tensor& t, at::ScalarType ty, int64_t n, const char* name, const char* want) {
    TORCH_CHECK(t.is_cuda() && t.is_contiguous() && t.dim() == 1 && t.scalar_type() == ty && (n < 0 || t.size(0) == n) &&
                    t.get_device() == add.get_device(),
                op, ": ", name, " must be a contiguous CUDA ", want);
  };
  TORCH_CHECK(B >= 0, op, ": lengths must be a contiguous CUDA int32 [B] tensor");
  TORCH_CHECK(B <= PERSONA_PLAN_MAX_SEQS, op, ": at most ", PERSONA_PLAN_MAX_SEQS, " sequences");
  vec(add, at::kInt, B, "new", "int32 [B] tensor");
  vec(lengths, at::kInt, B, "lengths", "int32 [B] tensor");
  vec(free_pages, at::kInt, -1, "free_pages", "int32 vector");
  vec(num_free, at::kInt, 1, "num_free", "int32 tensor of one element");
  vec(indptr, at::kInt, B + 1, "indptr", "int32 [B + 1] tensor");
  vec(places, at::kLong, -1, "places", "int64 [rows] tensor");
  if (keep.has_value()) vec(*keep, at::kInt, B, "keep", "int32 [B] tensor");
  TORCH_CHECK(seq_slots.has_value() == row_slots.has_value(), op, ": seq_slots and row_slots go together");
  if (row_slots.has_value()) {
    vec(*seq_slots, at::kInt, B, "seq_slots", "int32 [B] tensor");
    vec(*row_slots, at::kInt, places.size(0), "row_slots", "int32 [rows] tensor");
  }
  check_index(page_table, 2, add, op, "page_table");
  TORCH_CHECK(page_table.size(0) == B && (B <= 1 || page_table.stride(0) >= page_table.size(1)), op,
              ": page_table must be [B, max pages] and not overlap itself");
  TORCH_CHECK(page_size >= 1, op, ": page_size must be positive");
  const at::cuda::OptionalCUDAGuard guard(add.device());
  const int dev = add.get_device();
  raise_pending(dev, op);
  cudaStream_t stream = at::cuda::getCurrentCUDAStream();
  auto ptr = [](const c10::optional<at::Tensor>& t) { return t.has_value() ? t->data_ptr<int32_t>() : nullptr; };
  check_status(persona_paged_plan(add.data_ptr<int32_t>(), ptr(keep), lengths.data_ptr<int32_t>(), B,
                                  page_table.data_ptr<int32_t>(), B <= 1 ? page_table.size(1) : page_table.stride(0),
                                  page_table.size(1), free_pages.data_ptr<int32_t>(), free_pages.size(0),
                                  num_free.data_ptr<int32_t>(), page_size, indptr.data_ptr<int32_t>(),
                                  places.data_ptr<int64_t>(), ptr(seq_slots), ptr(row_slots), places.size(0),
                                  error_word_device(dev), stream),
               op);
  after_launch(dev, op, stream);
}

void sample_tokens_op(const at::Tensor& logits, const at::Tensor& u, at::Tensor& tokens,
                      const c10::optional<at::Tensor>& temperature, const c10::optional<at::Tensor>& top_k,
                      const c10::optional<at::Tensor>& top_p, const c10::optional<at::Tensor>& min_p) {
  const char* op = "sample_tokens";
  TORCH_CHECK(logits.is_cuda() && logits.dim() == 2 && (logits.size(1) <= 1 || logits.stride(1) == 1), op,
              ": logits must be a CUDA [B, V] matrix with unit inner stride");
  const int64_t B = logits.size(0), V = logits.size(1);
  const int type = logits.scalar_type() == at::kFloat ? PERSONA_DTYPE_F32 : logits.scalar_type() == at::kHalf
                       ? PERSONA_DTYPE_F16 : PERSONA_DTYPE_BF16;
  TORCH_CHECK(type != PERSONA_DTYPE_BF16 || logits.scalar_type() == at::kBFloat16, op,
              ": logits must be float32, float16 or bfloat16");
  TORCH_CHECK(V >= 1 && V <= PERSONA_VERIFY_MAX_VOCAB, op, ": vocabulary of 1 to ", PERSONA_VERIFY_MAX_VOCAB, " tokens");
  auto vec = [&](const at::Tensor& t, at::ScalarType ty, const char* name, const char* want) {
    TORCH_CHECK(t.is_cuda() && t.is_contiguous() && t.dim() == 1 && t.scalar_type() == ty && t.size(0) == B &&
                    t.get_device() == logits.get_device(),
                op, ": ", name, " must be a contiguous CUDA ", want);
  };
  vec(u, at::kFloat, "u", "float32 [B] tensor");
  vec(tokens, at::kLong, "tokens", "int64 [B] tensor");
  if (temperature.has_value()) vec(*temperature, at::kFloat, "temperature", "float32 [B] tensor");
  if (top_k.has_value()) vec(*top_k, at::kInt, "top_k", "int32 [B] tensor");
  if (top_p.has_value()) vec(*top_p, at::kFloat, "top_p", "float32 [B] tensor");
  if (min_p.has_value()) vec(*min_p, at::kFloat, "min_p", "float32 [B] tensor");
  const at::cuda::OptionalCUDAGuard guard(logits.device());
  const int dev = logits.get_device();
  raise_pending(dev, op);
  if (B == 0) return;
  cudaStream_t stream = at::cuda::getCurrentCUDAStream();
  auto f32 = [](const c10::optional<at::Tensor>& t) { return t.has_value() ? t->data_ptr<float>() : nullptr; };
  check_status(persona_sample_tokens(logits.data_ptr(), B <= 1 ? V : logits.stride(0), type, u.data_ptr<float>(),
                                     f32(temperature), top_k.has_value() ? top_k->data_ptr<int32_t>() : nullptr, f32(top_p),
                                     f32(min_p), tokens.data_ptr<int64_t>(), B, V, stream),
               op);
  after_launch(dev, op, stream);
}

void verify_draft_op(const at::Tensor& target, const at::Tensor& draft_tokens, const c10::optional<at::Tensor>& draft,
                     const at::Tensor& indptr, const at::Tensor& u_accept, const at::Tensor& u_sample,
                     at::Tensor& tokens, at::Tensor& accepted) {
  const char* op = "verify_draft";
  TORCH_CHECK(target.is_cuda() && target.dim() == 2 && (target.size(1) <= 1 || target.stride(1) == 1), op,
              ": target_probs must be a CUDA [rows, V] matrix with unit inner stride");
  const int64_t rows = target.size(0), V = target.size(1);
  const int type = target.scalar_type() == at::kFloat ? PERSONA_DTYPE_F32 : target.scalar_type() == at::kHalf
                       ? PERSONA_DTYPE_F16 : PERSONA_DTYPE_BF16;
  TORCH_CHECK(type != PERSONA_DTYPE_BF16 || target.scalar_type() == at::kBFloat16, op,
              ": probabilities must be float32, float16 or bfloat16");
  TORCH_CHECK(V >= 1 && V <= PERSONA_VERIFY_MAX_VOCAB, op, ": vocabulary of 1 to ", PERSONA_VERIFY_MAX_VOCAB, " tokens");
  if (draft.has_value())
    TORCH_CHECK(draft->is_cuda() && draft->scalar_type() == target.scalar_type() && draft->sizes() == target.sizes() &&
                    (V <= 1 || draft->stride(1) == 1) && draft->get_device() == target.get_device(),
                op, ": draft_probs must match target_probs");
  check_index(indptr, 1, target, op, "indptr");
  const int64_t B = indptr.size(0) - 1;
  TORCH_CHECK(B >= 0, op, ": indptr must have B + 1 entries");
  auto vec = [&](const at::Tensor& t, at::ScalarType ty, int64_t n, const char* name, const char* want) {
    TORCH_CHECK(t.is_cuda() && t.is_contiguous() && t.dim() == 1 && t.scalar_type() == ty && t.size(0) == n &&
                    t.get_device() == target.get_device(),
                op, ": ", name, " must be a contiguous CUDA ", want);
  };
  vec(draft_tokens, at::kLong, rows, "draft_tokens", "int64 [rows] tensor");
  vec(u_accept, at::kFloat, rows, "u_accept", "float32 [rows] tensor");
  vec(u_sample, at::kFloat, B, "u_sample", "float32 [B] tensor");
  vec(tokens, at::kLong, rows, "tokens", "int64 [rows] tensor");
  vec(accepted, at::kInt, B, "accepted", "int32 [B] tensor");
  TORCH_CHECK(rows == 0 || tokens.data_ptr<int64_t>() + rows <= draft_tokens.data_ptr<int64_t>() ||
                  draft_tokens.data_ptr<int64_t>() + rows <= tokens.data_ptr<int64_t>(),
              op, ": tokens must not overlap draft_tokens");
  const at::cuda::OptionalCUDAGuard guard(target.device());
  const int dev = target.get_device();
  raise_pending(dev, op);
  if (B == 0) return;
  cudaStream_t stream = at::cuda::getCurrentCUDAStream();
  check_status(persona_verify_draft(target.data_ptr(), rows <= 1 ? V : target.stride(0),
                                    draft.has_value() ? draft->data_ptr() : nullptr,
                                    draft.has_value() && rows > 1 ? draft->stride(0) : V, type,
                                    draft_tokens.data_ptr<int64_t>(), indptr.data_ptr<int32_t>(),
                                    u_accept.data_ptr<float>(), u_sample.data_ptr<float>(), tokens.data_ptr<int64_t>(),
                                    accepted.data_ptr<int32_t>(), rows, B, V, error_word_device(dev), stream),
               op);
  after_launch(dev, op, stream);
}
}  // namespace

TORCH_LIBRARY(persona, m) {
  // Reference schemas, unchanged (csrc/bindings.cpp:19-23).
  m.def("bgmv_shrink(Tensor x, Tensor a_pool, Tensor slots, Tensor(a!) v) -> ()");
  m.def("bgmv_expand(Tensor v, Tensor b_pool, Tensor slots, Tensor(a!) y) -> ()");
  m.def("gemv_fp16(Tensor x, Tensor W, Tensor(a!) y) -> ()");
  // New in this build.
  m.def("bgmv_plan(Tensor slots, int S) -> Tensor");
  m.def("bgmv_shrink_with_plan(Tensor x, Tensor a_pool, Tensor slots, Tensor plan, Tensor(a!) v) -> ()");
  m.def("bgmv_expand_with_plan(Tensor v, Tensor b_pool, Tensor slots, Tensor plan, Tensor(a!) y) -> ()");
  m.def("bgmv_fused(Tensor x, Tensor a_pool, Tensor b_pool, Tensor slots, Tensor(a!) y) -> ()");
  m.def("bgmv_fused_with_plan(Tensor x, Tensor a_pool, Tensor b_pool, Tensor slots, Tensor plan, "
        "Tensor(a!) y) -> ()");
  m.def("bgmv_fused_multi(Tensor[] xs, Tensor[] a_pools, Tensor[] b_pools, Tensor slots, Tensor(a!)[] ys, "
        "Tensor? plan=None) -> ()");
  m.def("sgmv_shrink(Tensor x, Tensor a_pool, Tensor seg_indptr, Tensor seg_slots, Tensor(a!) v) -> ()");
  m.def("sgmv_expand(Tensor v, Tensor b_pool, Tensor seg_indptr, Tensor seg_slots, Tensor(a!) y) -> ()");
  m.def("sgmv_fused(Tensor x, Tensor a_pool, Tensor b_pool, Tensor seg_indptr, Tensor seg_slots, "
        "Tensor(a!) y) -> ()");
  m.def("nf4_quantize(Tensor w) -> (Tensor, Tensor)");
  m.def("nf4_dequantize(Tensor packed, Tensor offset, int N, int K) -> Tensor");
  m.def("nf4_linear(Tensor x, Tensor[] packed, Tensor[] offsets, Tensor(a!)[] ys) -> ()");
  m.def("nf4_linear_add(Tensor x, Tensor[] packed, Tensor[] offsets, Tensor[] addends, Tensor(a!)[] ys) -> ()");
  m.def("bgmv_lora_delta_multi(Tensor[] xs, Tensor[] a_pools, Tensor[] b_pools, Tensor slots, "
        "Tensor(a!)[] deltas) -> ()");
  m.def("add_rmsnorm(Tensor(a!) h, Tensor? delta, Tensor w, Tensor(b!) out, float eps) -> ()");
  m.def("rope_cache(Tensor(a!) q, Tensor(b!) k, Tensor v, Tensor(c!) k_cache, Tensor(d!) v_cache, Tensor start, "
        "int per_seq, float theta) -> ()");
  m.def("silu_mul(Tensor g, Tensor u, Tensor(a!) out) -> ()");
  m.def("decode_attention(Tensor q, Tensor k_cache, Tensor v_cache, Tensor len, Tensor(a!) out, float scale) -> ()");
  m.def("rope_decode_attention(Tensor(a!) q, Tensor(b!) k, Tensor v, Tensor(c!) k_cache, Tensor(d!) v_cache, "
        "Tensor pos, Tensor len, Tensor(e!) out, float theta, float scale) -> ()");
  // q_out may be q itself: both carry the same alias set.
  m.def("paged_rope_cache(Tensor(a!) q, Tensor k, Tensor v, Tensor(a!) q_out, Tensor(b!) k_cache, Tensor(c!) v_cache, "
        "Tensor page_table, Tensor indptr, Tensor lengths, float theta, Tensor(d!)? k_scale=None, "
        "Tensor(e!)? v_scale=None) -> ()");
  m.def("paged_cache_read(Tensor k_cache, Tensor v_cache, Tensor page_table, Tensor indptr, Tensor lengths, "
        "Tensor(a!) k_out, Tensor(b!) v_out, Tensor? k_scale=None, Tensor? v_scale=None) -> ()");
  m.def("paged_attention(Tensor q, Tensor k_cache, Tensor v_cache, Tensor page_table, Tensor indptr, Tensor lengths, "
        "Tensor(a!) out, float scale, int window, int max_new, Tensor? k_scale=None, Tensor? v_scale=None) -> ()");
  m.def("verify_draft(Tensor target_probs, Tensor draft_tokens, Tensor? draft_probs, Tensor indptr, Tensor u_accept, "
        "Tensor u_sample, Tensor(a!) tokens, Tensor(b!) accepted) -> ()");
  m.def("paged_plan(Tensor new, Tensor(a!) lengths, Tensor(b!) page_table, Tensor(c!) free_pages, Tensor(d!) num_free, "
        "int page_size, Tensor(e!) indptr, Tensor(f!) places, Tensor? keep=None, Tensor? seq_slots=None, "
        "Tensor(g!)? row_slots=None) -> ()");
  m.def("sample_tokens(Tensor logits, Tensor u, Tensor(a!) tokens, Tensor? temperature=None, Tensor? top_k=None, "
        "Tensor? top_p=None, Tensor? min_p=None) -> ()");
}

TORCH_LIBRARY_IMPL(persona, CUDA, m) {
  m.impl("nf4_quantize", &nf4_quantize_op);
  m.impl("nf4_dequantize", &nf4_dequantize_op);
  m.impl("nf4_linear", &nf4_linear_op);
  m.impl("nf4_linear_add", &nf4_linear_add_op);
  m.impl("bgmv_lora_delta_multi", &lora_delta_multi_op);
  m.impl("add_rmsnorm", &add_rmsnorm_op);
  m.impl("rope_cache", &rope_cache_op);
  m.impl("silu_mul", &silu_mul_op);
  m.impl("decode_attention", &decode_attention_op);
  m.impl("rope_decode_attention", &rope_decode_attention_op);
  m.impl("paged_rope_cache", &paged_rope_cache_op);
  m.impl("paged_cache_read", &paged_cache_read_op);
  m.impl("paged_attention", &paged_attention_op);
  m.impl("verify_draft", &verify_draft_op);
  m.impl("paged_plan", &paged_plan_op);
  m.impl("sample_tokens", &sample_tokens_op);
  m.impl("bgmv_shrink", &bgmv_shrink_cuda);
  m.impl("bgmv_expand", &bgmv_expand_cuda);
  m.impl("gemv_fp16", &persona::gemv_fp16_cuda);
  m.impl("bgmv_plan", &plan_impl);
  m.impl("bgmv_shrink_with_plan", &shrink_with_plan);
  m.impl("bgmv_expand_with_plan", &expand_with_plan);
  m.impl("bgmv_fused", &fused_noplan);
  m.impl("bgmv_fused_with_plan", &fused_with_plan);
  m.impl("bgmv_fused_multi", &fused_multi_impl);
  m.impl("sgmv_shrink", &sgmv_shrink_op);
  m.impl("sgmv_expand", &sgmv_expand_op);
  m.impl("sgmv_fused", &sgmv_fused_op);
}

namespace {
// Tensor-parallel segmented fused op (persona_sgmv_fused_tp); `peers` are the
// other ranks' y buffers mapped into this process, as integers.
void sgmv_fused_tp_op(const at::Tensor& x, const at::Tensor& a_pool, const at::Tensor& b_pool,
                      const at::Tensor& indptr, const at::Tensor& seg_slots, at::Tensor& y,
                      const std::vector<int64_t>& peers, int64_t n0, int64_t n1) {
  const char* op = "sgmv_fused_tp";
  check_segments(indptr, seg_slots, op);
  TORCH_CHECK(x.is_cuda() && a_pool.is_cuda() && b_pool.is_cuda() && y.is_cuda(), op, ": all tensors must be CUDA");
  TORCH_CHECK(x.dim() == 2 && x.stride(1) == 1 && y.dim() == 2 && y.stride(1) == 1, op,
              ": tensors must be contiguous");
  check_pool_a(a_pool, op);
  check_pool_b(b_pool, op);
  const int64_t T = x.size(0), K = x.size(1), S = a_pool.size(0), R = a_pool.size(1), N = b_pool.size(1);
  TORCH_CHECK(a_pool.size(2) == K && b_pool.size(0) == S && b_pool.size(2) == R, op, ": pool shape mismatch");
  TORCH_CHECK(y.size(0) == T && y.size(1) == N, op, ": y shape mismatch");
  TORCH_CHECK(peers.size() <= PERSONA_MAX_TP_PEERS, op, ": too many peers");
  const int dt = dtype_code(x, op);
  TORCH_CHECK(a_pool.scalar_type() == x.scalar_type() && b_pool.scalar_type() == x.scalar_type() &&
                  y.scalar_type() == x.scalar_type(),
              op, ": dtype mismatch");
  const at::cuda::OptionalCUDAGuard guard(x.device());
  const int dev = x.get_device();
  raise_pending(dev, op);
  if (T == 0) return;
  void* pp[PERSONA_MAX_TP_PEERS];
  for (size_t i = 0; i < peers.size(); ++i) pp[i] = reinterpret_cast<void*>(peers[i]);
  at::Tensor ws = sgmv_workspace(T, x);
  cudaStream_t stream = at::cuda::getCurrentCUDAStream();
  check_status(persona_sgmv_fused_tp(x.data_ptr(), row_stride(x), a_pool.data_ptr(), a_pool.stride(0),
                                     a_pool.stride(1), b_pool.data_ptr(), b_pool.stride(0),
                                     indptr.data_ptr<int32_t>(), seg_slots.data_ptr<int32_t>(), seg_slots.size(0),
                                     y.data_ptr(), row_stride(y), pp, static_cast<int>(peers.size()), n0, n1, T, K,
                                     N, R, S, dt, ws.data_ptr(), ws.numel(), error_word_device(dev), stream),
               op);
  after_launch(dev, op, stream);
}
}  // namespace

namespace {
// Whether a dispatch or function mode, or the subclass of a tensor, has to see
// a call (a fake tensor among them, which has no memory to hand to a kernel).
bool watched(const at::Tensor& t) { return t.key_set().has(c10::DispatchKey::Python); }
bool watched(const c10::optional<at::Tensor>& t) { return t.has_value() && watched(*t); }
template <typename T> bool watched(const T&) { return false; }
// Gives Python's lock up for its lifetime.
struct Unlocked {
  PyThreadState* const thread = PyEval_SaveThread();
  ~Unlocked() { PyEval_RestoreThread(thread); }
};
template <typename... A> void def_direct(pybind11::module& m, const char* name, void (*op)(A...)) {
  m.def(name, [name, op](A... a) {
    if (C10_UNLIKELY(c10::impl::TorchDispatchModeTLS::any_modes_set() || at::impl::torch_function_mode_enabled() ||
                     (watched(a) || ...))) {
      pybind11::module_::import("torch").attr("ops").attr("persona").attr(name)(a...);
      return;
    }
    const Unlocked others;  // as torch.ops does: the call may wait for its stream, or for room in it
    op(a...);
  });
}
}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  // The paged-cache ops for persona.ops, past the dispatcher: half of a small
  // call's time on the host is spent there.  The same functions are registered
  // as torch.ops.persona.*.
  def_direct(m, "paged_rope_cache", &paged_rope_cache_op);
  def_direct(m, "paged_cache_read", &paged_cache_read_op);
  def_direct(m, "paged_attention", &paged_attention_op);
  def_direct(m, "verify_draft", &verify_draft_op);
  def_direct(m, "paged_plan", &paged_plan_op);
  def_direct(m, "sample_tokens", &sample_tokens_op);
  m.def("sgmv_fused_tp", &sgmv_fused_tp_op,
        "Tensor-parallel segmented fused LoRA: columns [n0, n1) of y, every finished tile also stored into the "
        "peers' y (pointers from ipc_import).");
  m.def(
      "ipc_export",
      [](const at::Tensor& t) {
        TORCH_CHECK(t.is_cuda(), "ipc_export: CUDA tensor expected");
        const at::cuda::OptionalCUDAGuard guard(t.device());
        char handle[64];
        size_t offset = 0;
        check_status(persona_ipc_export(t.data_ptr(), handle, &offset), "ipc_export");
        return pybind11::make_tuple(pybind11::bytes(handle, sizeof(handle)), static_cast<int64_t>(offset));
      },
      "64-byte CUDA IPC handle of the allocation holding `t`, and t's offset in it.");
  m.def(
      "ipc_import",
      [](const std::string& handle, int64_t offset, int device) {
        TORCH_CHECK(handle.size() == 64, "ipc_import: 64-byte handle expected");
        const at::cuda::OptionalCUDAGuard guard(at::Device(at::kCUDA, device));
        void* ptr = nullptr;
        void* base = nullptr;
        check_status(persona_ipc_import(handle.data(), static_cast<size_t>(offset), &ptr, &base), "ipc_import");
        return pybind11::make_tuple(reinterpret_cast<int64_t>(ptr), reinterpret_cast<int64_t>(base));
      },
      "Map another process's buffer: returns (pointer, mapping base).");
  m.def(
      "ipc_close", [](int64_t base, int device) {
        const at::cuda::OptionalCUDAGuard guard(at::Device(at::kCUDA, device));
        check_status(persona_ipc_close(reinterpret_cast<void*>(base)), "ipc_close");
      },
      "Unmap a buffer mapped by ipc_import (its mapping base).");
  m.def("noop", []() { return 0; });
  m.def("abi_version", []() { return persona_abi_version(); });
  m.def("workspace_size", [](int64_t T) { return persona_bgmv_workspace_size(T); });
  m.def(
      "take_device_error",
      [](int device) {
        volatile int32_t* h = error_word_host(device);
        const int bits = *h;
        *h = 0;
        return bits;
      },
      "Read and clear the device error word of `device` (no synchronisation).");
}
