// What the operators of the serving kernels share: workspaces, checks of
// arguments, errors.
#pragma once

#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/AutogradState.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/library.h>

#include <map>
#include <mutex>
#include <tuple>
#include <utility>
#include <vector>

#include "tensorshrink_b200.h"

namespace ts_torch {

using OptTensor = c10::optional<at::Tensor>;

struct Workspace {
  std::mutex mu;                    // see Scratch
  at::Tensor t;
  unsigned long long capture = 0;   // of the graph that it belongs to
};

inline std::mutex g_mu;                    // of the maps; entries stay where they are
inline std::map<std::pair<int, cudaStream_t>, Workspace> g_ws, g_captured;

// A stream's workspace in the hands of one call. Kernels of a call pass data to
// one another through it, so the call holds it from before its first launch to
// behind its last: another host thread's launches on the same stream come
// before or behind them, never between.
struct Scratch {
  std::unique_lock<std::mutex> held;
  at::Tensor t;
  void* data() const { return t.defined() ? t.data_ptr() : nullptr; }
  size_t bytes() const { return t.defined() ? (size_t)t.numel() : 0; }
};

// A workspace of at least `bytes`, its counters zero. A captured stream has
// its own, from the graph's memory, and the graph zeroes it: neither the
// graph's replays on another stream nor calls outside of it meet the other's
// counters, and no warm-up has to come before the capture. Buffers are used on
// the stream that they were allocated on, so a superseded one can be freed.
inline Scratch workspace(const at::Device& dev, cudaStream_t s, size_t bytes) {
  cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
  unsigned long long id = 0;
  if (cudaStreamGetCaptureInfo(s, &status, &id) != cudaSuccess) (void)cudaGetLastError();
  const bool captured = status == cudaStreamCaptureStatusActive;
  Workspace* w;
  {
    std::lock_guard<std::mutex> lk(g_mu);
    w = &(captured ? g_captured : g_ws)[{dev.index(), s}];
  }
  Scratch r;
  r.held = std::unique_lock<std::mutex>(w->mu);
  if (!w->t.defined() || (captured && w->capture != id) || (size_t)w->t.numel() < bytes) {
    w->t = at::empty({(int64_t)std::max<size_t>(bytes, 1 << 20)}, at::TensorOptions().dtype(at::kByte).device(dev));
    w->t.slice(0, 0, (int64_t)ts_serving_counter_bytes()).zero_();
    w->capture = id;
  }
  r.t = w->t;
  return r;
}

inline bool has(const OptTensor& t) { return t.has_value() && t->defined(); }
template <typename T = void>
T* ptr(const OptTensor& t) { return has(t) ? static_cast<T*>(t->data_ptr()) : nullptr; }

// An uninitialised tensor on the current device, without a dispatcher call.
inline at::Tensor fresh(at::IntArrayRef shape, at::ScalarType type, const at::Device& dev) {
  return at::Tensor(at::detail::empty_cuda(shape, type, dev, c10::nullopt));
}

inline bool known(at::ScalarType t) { return t == at::kHalf || t == at::kBFloat16 || t == at::kFloat; }

inline int code_of(at::ScalarType t, const char* what) {
  switch (t) {
    case at::kHalf: return TS_F16;
    case at::kBFloat16: return TS_BF16;
    case at::kFloat: return TS_F32;
    default: TORCH_CHECK_NOT_IMPLEMENTED(false, what, ": dtype ", t, " is not supported");
  }
  return -1;
}

inline void on(const at::Tensor& t, const at::Device& dev, const char* name) {
  TORCH_CHECK(t.device() == dev, name, " is on ", t.device(), ", expected ", dev);
}
inline void on(const OptTensor& t, const at::Device& dev, const char* name) {
  if (has(t)) on(*t, dev, name);
}

// The operators compute no gradients. A floating-point result of inputs that want
// them says so when a backward pass reaches it, instead of ending it silently;
// the forward pass is the same. Inputs with tangents (derivatives in forward mode) are
// refused at once, as the result would come without one. (Codes are integers, and what is
// quantised or written into a cache or a given result is held without its history.)
inline const at::Tensor* in(const OptTensor& t) { return has(t) ? &*t : nullptr; }
inline bool has_tangent(const at::Tensor& t) {
  return c10::AutogradState::get_tls_state().get_fw_grad_mode() && t._fw_grad(0).defined();
}
// (By itself in front of what writes into a cache.)
inline void no_tangents(const char* name, std::initializer_list<const at::Tensor*> of) {
  for (const at::Tensor* t : of)
    TORCH_CHECK_NOT_IMPLEMENTED(t == nullptr || !has_tangent(*t), "tensorshrink::", name,
                                " has no derivative in forward mode, and an input has a tangent");
}
inline at::Tensor forward_only(at::Tensor y, const char* name, std::initializer_list<const at::Tensor*> of) {
  no_tangents(name, of);
  if (!at::GradMode::is_enabled()) return y;
  std::vector<at::Tensor> in;
  for (const at::Tensor* t : of)
    if (t != nullptr && t->requires_grad()) in.push_back(*t);
  if (!in.empty())
    torch::autograd::set_history(
        y, std::make_shared<torch::autograd::NotImplemented>(std::string("tensorshrink::") + name,
                                                             torch::autograd::collect_next_edges(in)));
  return y;
}

// Refuses an `out` whose rows share memory with one another, or with rows of x that kernels read
// where they lie: but for the same columns of the same rows, some warps may have yet to read
// what others write. Both are matrices with as many rows, of contiguous elements of one size. (ATen's own check passes
// over tensors with gaps between their rows.)
inline void apart(const at::Tensor& out, const at::Tensor& x, const char* what) {
  const int64_t rows = out.size(0), item = out.element_size(), width = out.size(1) * item, x_width = x.size(1) * item;
  if (rows == 0 || width == 0 || x_width == 0) return;
  const int64_t step = out.stride(0) * item, x_step = x.stride(0) * item;
  TORCH_CHECK_VALUE(rows == 1 || step >= width, what, ": the rows of out overlap");
  const auto at = reinterpret_cast<intptr_t>(out.data_ptr()), x_at = reinterpret_cast<intptr_t>(x.data_ptr());
  if (at + (rows - 1) * step + width <= x_at || x_at + (rows - 1) * x_step + x_width <= at) return;
  if (rows == 1 || step == x_step) {
    if (at == x_at && width <= x_width) return;
    const int64_t gap = rows == 1 ? 0 : ((at - x_at) % step + step) % step;   // from a row of x to the next of out
    if (rows > 1 && gap >= x_width && gap + width <= step) return;
  }
  TORCH_CHECK(false, what, ": out overlaps the input");
}

// What is written into a given result has no history: one that wants a gradient, or has a tangent, is refused.
inline void no_history(const at::Tensor& out, const char* what) {
  TORCH_CHECK(!at::GradMode::is_enabled() || !out.requires_grad(), what, ": out wants a gradient, and there is none");
  TORCH_CHECK_NOT_IMPLEMENTED(!has_tangent(out), what, ": out has a tangent, and there is no derivative in forward mode");
}

// Raises the exception that the library's status stands for.
inline void done(int rc, const char* what) {
  if (rc == TS_OK) return;
  TORCH_CHECK_VALUE(rc != TS_ERR_INVALID, what, ": ", ts_last_error());
  TORCH_CHECK_NOT_IMPLEMENTED(rc != TS_ERR_UNSUPPORTED, what, ": ", ts_last_error());
  TORCH_CHECK(false, what, ": ", ts_last_error());
}

inline int check_bias(const OptTensor& bias, int64_t n, const at::Device& dev, const char* what) {
  if (!has(bias)) return 0;
  on(*bias, dev, "bias");
  TORCH_CHECK_VALUE(bias->numel() == n && known(bias->scalar_type()) && bias->is_contiguous(), what, ": bias must be ", n,
                    " contiguous fp16, bf16 or fp32 values");
  return code_of(bias->scalar_type(), what);
}

// What can be said of a cache without its memory.
inline void cache_fits(const at::Tensor& k, const at::Tensor& v, const at::Tensor& table, const at::Tensor& lens,
                const OptTensor& scores, const OptTensor& slot_pos) {
  const at::Device dev = k.device();
  TORCH_CHECK_VALUE(k.dim() == 4 && v.sizes() == k.sizes(),
                    "k_pages and v_pages must both be [num_pages, n_kv, page_size, head_dim]");
  TORCH_CHECK_NOT_IMPLEMENTED(k.scalar_type() == at::kHalf || k.scalar_type() == at::kBFloat16,
                              "the cache holds fp16 or bf16");
  TORCH_CHECK_VALUE(v.scalar_type() == k.scalar_type(), "k_pages and v_pages differ in type");
  TORCH_CHECK_VALUE(v.strides() == k.strides() && k.stride(3) == 1,
                    "k_pages and v_pages must share their strides and have contiguous rows");
  TORCH_CHECK_VALUE(table.scalar_type() == at::kInt && table.dim() == 2 && (table.stride(1) == 1 || table.size(1) <= 1),
                    "page_table must be int32 [batch, max_pages] with contiguous rows");
  TORCH_CHECK_VALUE(lens.scalar_type() == at::kInt && lens.dim() == 1 && lens.size(0) == table.size(0) && lens.is_contiguous(),
                    "seq_lens must be contiguous int32 [batch]");
  on(v, dev, "v_pages");
  on(table, dev, "page_table");
  on(lens, dev, "seq_lens");
  for (const auto& [t, type, name] : {std::make_tuple(&scores, at::kFloat, "scores"),
                                      std::make_tuple(&slot_pos, at::kInt, "slot_pos")}) {
    if (!has(*t)) continue;
    on(**t, dev, name);
    TORCH_CHECK_VALUE((*t)->scalar_type() == type && (*t)->sizes() == k.sizes().slice(0, 3) && (*t)->is_contiguous(), name,
                      " must be contiguous ", type, " [num_pages, n_kv, page_size]");
  }
}

inline ts_paged_cache cache_view(const at::Tensor& k, const at::Tensor& v, const at::Tensor& table, const at::Tensor& lens,
                          const OptTensor& scores, const OptTensor& slot_pos) {
  TORCH_CHECK(k.is_cuda(), "PagedKVCache: tensorshrink_b200 runs on CUDA tensors only (got ", k.device(), ")");
  cache_fits(k, v, table, lens, scores, slot_pos);
  ts_paged_cache c{};
  c.k_pages = k.data_ptr();
  c.v_pages = v.data_ptr();
  c.page_stride = k.stride(0);
  c.head_stride = k.stride(1);
  c.token_stride = k.stride(2);
  c.page_table = static_cast<const int32_t*>(table.data_ptr());
  c.table_stride = table.stride(0);
  c.seq_lens = static_cast<int32_t*>(lens.data_ptr());
  c.scores = ptr<float>(scores);
  c.slot_pos = ptr<int32_t>(slot_pos);
  c.dtype = k.scalar_type() == at::kHalf ? TS_F16 : TS_BF16;
  c.batch = (int32_t)table.size(0);
  c.n_kv = (int32_t)k.size(1);
  c.head_dim = (int32_t)k.size(3);
  c.page_size = (int32_t)k.size(2);
  c.num_pages = (int32_t)k.size(0);
  c.max_pages = (int32_t)table.size(1);
  return c;
}

inline int64_t rope_rows(const ts_paged_cache& c, const OptTensor& cos, const OptTensor& sin, const at::Device& dev,
                  const char* what) {
  TORCH_CHECK_VALUE(has(cos) == has(sin), what, ": rope_cos and rope_sin come both or neither");
  if (!has(cos)) return 0;
  for (const at::Tensor* t : {&*cos, &*sin}) {
    on(*t, dev, "a rotary table");
    TORCH_CHECK_VALUE(t->scalar_type() == at::kFloat && t->dim() == 2 && t->size(1) == c.head_dim / 2 && t->is_contiguous(),
                      what, ": the rotary tables must be contiguous fp32 [positions, head_dim / 2]");
  }
  // (the library takes the NULL that an empty table's data is for no table)
  TORCH_CHECK_VALUE(cos->size(0) == sin->size(0) && cos->size(0) > 0, what, ": the rotary tables are empty or differ in length");
  return cos->size(0);
}

inline void per_sequence(const OptTensor& t, const ts_paged_cache& c, at::ScalarType type, const at::Device& dev, const char* name) {
  if (!has(t)) return;
  on(*t, dev, name);
  TORCH_CHECK_VALUE(t->scalar_type() == type && t->dim() == 1 && t->size(0) == c.batch && t->is_contiguous(), name,
                    " must be contiguous ", type, " [batch]");
}

}  // namespace ts_torch
