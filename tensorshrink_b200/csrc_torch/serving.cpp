// torch.ops.tensorshrink operators of the serving kernels: microscaled 4-bit
// floating point and the paged key-value cache (C ABI: ts_fp4_*, ts_paged_*).
//
// As for qlinear, each call is one dispatcher call with no Python-side
// workspace lookup or struct packing. Arguments are checked here (ValueError
// and NotImplementedError as the Python wrappers document them); launches go
// to the current stream of the tensors' device. One workspace per (device,
// stream) serves all of them, and one per graph while the stream is captured;
// calls of several host threads take turns at it.
#include "serving_common.h"

namespace {

using namespace ts_torch;

// ---- microscaled 4-bit ----------------------------------------------------------

int64_t padded(int64_t cols) { return (cols + 63) / 64 * 64; }

// What can be said of a tensor's description without its memory.
void fp4_fits(const at::Tensor& codes, const at::Tensor& scales, const OptTensor& g, int64_t rows, int64_t cols,
              int64_t format, const char* what) {
  TORCH_CHECK_NOT_IMPLEMENTED(format == TS_NVFP4 || format == TS_MXFP4, what, ": unknown format");
  TORCH_CHECK_VALUE(rows >= 0 && cols > 0, what, ": bad shape [", rows, ", ", cols, "]");
  TORCH_CHECK_VALUE(codes.scalar_type() == at::kByte && scales.scalar_type() == at::kByte && codes.is_contiguous() &&
                        scales.is_contiguous(),
                    what, ": codes and scales must be contiguous uint8");
  TORCH_CHECK_VALUE(codes.numel() == rows * (padded(cols) / 2), what, ": codes hold ", codes.numel(), " bytes, [", rows,
                    ", ", padded(cols) / 2, "] wanted");
  TORCH_CHECK_VALUE((size_t)scales.numel() >= ts_fp4_scales_bytes(rows, cols, (int)format), what, ": scales hold ",
                    scales.numel(), " bytes, ", ts_fp4_scales_bytes(rows, cols, (int)format), " wanted");
  on(scales, codes.device(), "scales");
  if (has(g)) {
    TORCH_CHECK_VALUE(format == TS_NVFP4, what, ": only nvfp4 has a tensor scale");
    TORCH_CHECK_VALUE(g->scalar_type() == at::kFloat && g->numel() == 1, what, ": the tensor scale must be one fp32 value");
    on(*g, codes.device(), "the tensor scale");
  }
}

ts_fp4_tensor fp4_view(const at::Tensor& codes, const at::Tensor& scales, const OptTensor& g, int64_t rows, int64_t cols,
                       int64_t format, const char* what) {
  TORCH_CHECK(codes.is_cuda(), what, ": tensorshrink_b200 runs on CUDA tensors only (got ", codes.device(), ")");
  fp4_fits(codes, scales, g, rows, cols, format, what);
  ts_fp4_tensor t{};
  t.codes = static_cast<uint8_t*>(codes.data_ptr());
  t.scales = static_cast<uint8_t*>(scales.data_ptr());
  t.global_scale = ptr<float>(g);
  t.rows = rows;
  t.cols = cols;
  t.format = (int32_t)format;
  return t;
}

void fp4_check(const at::Tensor& codes, const at::Tensor& scales, const OptTensor& g, int64_t rows, int64_t cols,
               int64_t format) {
  fp4_view(codes, scales, g, rows, cols, format, "Fp4Tensor");
}

// Codes, scales and the tensor scale where it was found (a given one is the caller's).
std::tuple<at::Tensor, at::Tensor, OptTensor> fp4_quantize(const at::Tensor& x_in, int64_t format, const OptTensor& scale) {
  TORCH_CHECK(x_in.is_cuda(), "fp4_quantize: tensorshrink_b200 runs on CUDA tensors only (got ", x_in.device(), ")");
  const at::Device dev = x_in.device();
  c10::cuda::CUDAGuard guard(dev);
  TORCH_CHECK_VALUE(x_in.dim() == 2 && x_in.size(1) > 0, "fp4_quantize takes a [rows, cols] tensor, got ", x_in.sizes());
  const int dt = code_of(x_in.scalar_type(), "fp4_quantize");
  const at::Tensor x = x_in.stride(1) == 1 || x_in.size(1) == 1 ? x_in : x_in.contiguous();
  const int64_t rows = x.size(0), cols = x.size(1), kb = padded(cols) / 2;
  const bool find = format == TS_NVFP4 && !has(scale);
  at::Tensor g;
  if (find) g = rows ? fresh({1}, at::kFloat, dev) : at::ones({1}, at::TensorOptions().dtype(at::kFloat).device(dev));
  else if (has(scale)) g = *scale;
  at::Tensor codes = fresh({rows, kb}, at::kByte, dev);
  at::Tensor scales = fresh({(int64_t)ts_fp4_scales_bytes(rows, cols, (int)format)}, at::kByte, dev);
  const ts_fp4_tensor t = fp4_view(codes, scales, g.defined() ? OptTensor(g) : c10::nullopt, rows, cols, format, "fp4_quantize");
  cudaStream_t s = at::cuda::getCurrentCUDAStream(dev.index()).stream();
  Scratch ws;
  if (find) ws = workspace(dev, s, ts_fp4_quantize_workspace_size());
  done(ts_fp4_quantize(x.data_ptr(), dt, x.stride(0), &t, find, ws.data(), ws.bytes(), s), "fp4_quantize");
  return {codes, scales, find ? OptTensor(g) : c10::nullopt};
}

at::Tensor fp4_dequantize(const at::Tensor& codes, const at::Tensor& scales, const OptTensor& g, int64_t rows,
                          int64_t cols, int64_t format, at::ScalarType dtype) {
  const ts_fp4_tensor t = fp4_view(codes, scales, g, rows, cols, format, "fp4_dequantize");
  const int dt = code_of(dtype, "fp4_dequantize");
  c10::cuda::CUDAGuard guard(codes.device());
  at::Tensor out = fresh({rows, cols}, dtype, codes.device());
  done(ts_fp4_dequantize(&t, out.data_ptr(), dt, cols, at::cuda::getCurrentCUDAStream(codes.device().index()).stream()),
       "fp4_dequantize");
  return forward_only(std::move(out), "fp4_dequantize", {in(g)});
}

at::Tensor fp4_matmul(const at::Tensor& ac, const at::Tensor& as, const OptTensor& ag, int64_t m, const at::Tensor& bc,
                      const at::Tensor& bs, const OptTensor& bg, int64_t n, int64_t cols, int64_t format,
                      const OptTensor& bias, at::ScalarType out_dtype) {
  const ts_fp4_tensor a = fp4_view(ac, as, ag, m, cols, format, "fp4_matmul"),
                      b = fp4_view(bc, bs, bg, n, cols, format, "fp4_matmul");
  const at::Device dev = ac.device();
  on(bc, dev, "b");
  c10::cuda::CUDAGuard guard(dev);
  const int bdt = check_bias(bias, n, dev, "fp4_matmul"), dt = code_of(out_dtype, "fp4_matmul");
  at::Tensor out = fresh({m, n}, out_dtype, dev);
  cudaStream_t s = at::cuda::getCurrentCUDAStream(dev.index()).stream();
  const Scratch ws = workspace(dev, s, ts_fp4_matmul_workspace_size(m, n, cols, (int)format));
  done(ts_fp4_matmul(&a, &b, ptr(bias), bdt, out.data_ptr(), dt, n, ws.data(), ws.bytes(), s), "fp4_matmul");
  return forward_only(std::move(out), "fp4_matmul", {in(ag), in(bg), in(bias)});
}

at::Tensor fp4_linear(const at::Tensor& x, const at::Tensor& codes, const at::Tensor& scales, const OptTensor& g,
                      int64_t rows, int64_t cols, int64_t format, const OptTensor& bias, const OptTensor& input_scale,
                      c10::optional<at::ScalarType> out_dtype) {
  const ts_fp4_tensor w = fp4_view(codes, scales, g, rows, cols, format, "fp4_linear");
  const at::Device dev = codes.device();
  on(x, dev, "x");
  c10::cuda::CUDAGuard guard(dev);
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) == cols, "fp4_linear: x has ", x.dim() ? x.size(-1) : 0,
                    " features, the weight ", cols);
  if (has(input_scale)) {
    TORCH_CHECK_VALUE(format == TS_NVFP4, "fp4_linear: only nvfp4 has an input_scale");
    TORCH_CHECK_VALUE(input_scale->scalar_type() == at::kFloat && input_scale->numel() == 1,
                      "fp4_linear: input_scale must be one fp32 value");
    on(*input_scale, dev, "input_scale");
  }
  const int xdt = code_of(x.scalar_type(), "fp4_linear");
  const at::ScalarType odt = out_dtype.value_or(x.scalar_type());
  const int dt = code_of(odt, "fp4_linear"), bdt = check_bias(bias, rows, dev, "fp4_linear");
  at::Tensor x2d = x.dim() == 2 ? x : x.reshape({-1, cols});
  if (x2d.stride(1) != 1 && cols != 1) x2d = x2d.contiguous();
  std::vector<int64_t> shape(x.sizes().begin(), x.sizes().end());
  shape.back() = rows;
  at::Tensor out = fresh(shape, odt, dev);
  const int64_t m = x2d.size(0);
  cudaStream_t s = at::cuda::getCurrentCUDAStream(dev.index()).stream();
  const Scratch ws = workspace(dev, s, ts_fp4_linear_workspace_size(m, rows, cols, (int)format));
  done(ts_fp4_linear(x2d.data_ptr(), xdt, m, x2d.stride(0), ptr<float>(input_scale), &w, ptr(bias), bdt, out.data_ptr(), dt,
                     rows, ws.data(), ws.bytes(), s), "fp4_linear");
  return forward_only(std::move(out), "fp4_linear", {&x, in(g), in(bias), in(input_scale)});
}

// ---- paged cache ------------------------------------------------------------------

void paged_check(const at::Tensor& k, const at::Tensor& v, const at::Tensor& table, const at::Tensor& lens,
                 const OptTensor& scores, const OptTensor& slot_pos) {
  cache_view(k, v, table, lens, scores, slot_pos);
}

void paged_append(const at::Tensor& k_in, const at::Tensor& v_in, const at::Tensor& kp, const at::Tensor& vp,
                  const at::Tensor& table, const at::Tensor& lens, const OptTensor& scores, const OptTensor& slot_pos,
                  const OptTensor& positions, const OptTensor& cos, const OptTensor& sin, const OptTensor& n_new,
                  const OptTensor& new_scores) {
  const ts_paged_cache c = cache_view(kp, vp, table, lens, scores, slot_pos);
  const at::Device dev = kp.device();
  c10::cuda::CUDAGuard guard(dev);
  on(k_in, dev, "k");
  on(v_in, dev, "v");
  TORCH_CHECK_VALUE(k_in.dim() == 4 && v_in.sizes() == k_in.sizes() && k_in.size(0) == c.batch && k_in.size(2) == c.n_kv &&
                        k_in.size(3) == c.head_dim,
                    "k and v must be [batch, tokens, n_kv, head_dim], got ", k_in.sizes(), " and ", v_in.sizes());
  TORCH_CHECK_VALUE(k_in.scalar_type() == kp.scalar_type() && v_in.scalar_type() == kp.scalar_type(),
                    "k and v must have the cache's type");
  const int64_t rows = rope_rows(c, cos, sin, dev, "paged_append");
  per_sequence(positions, c, at::kLong, dev, "positions");
  per_sequence(n_new, c, at::kInt, dev, "n_new");
  // rows as the kernel reads them: contiguous and 16-byte aligned
  auto fit = [](const at::Tensor& t) {
    bool ok = t.stride(3) == 1 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
    for (int i = 0; i < 3; ++i) ok = ok && t.stride(i) % 8 == 0;
    return ok ? t : t.clone(at::MemoryFormat::Contiguous);
  };
  const at::Tensor k = fit(k_in), v = fit(v_in);
  int64_t ss[3] = {0, 0, 0};
  if (has(new_scores)) {
    on(*new_scores, dev, "scores");
    TORCH_CHECK_VALUE(has(scores), "scores were given for a cache that keeps none");
    TORCH_CHECK_VALUE(new_scores->scalar_type() == at::kFloat && new_scores->dim() == 3 && new_scores->size(0) == c.batch &&
                          new_scores->size(1) == c.n_kv && new_scores->size(2) == k.size(1),
                      "scores must be fp32 [batch, n_kv, tokens]");
    for (int i = 0; i < 3; ++i) ss[i] = new_scores->stride(i);
  }
  const int64_t ks[3] = {k.stride(0), k.stride(1), k.stride(2)}, vs[3] = {v.stride(0), v.stride(1), v.stride(2)};
  done(ts_paged_append(k.data_ptr(), ks, v.data_ptr(), vs, (int)k.size(1), ptr<int32_t>(n_new), &c, ptr<int64_t>(positions),
                       ptr<float>(cos), ptr<float>(sin), rows, ptr<float>(new_scores), ss,
                       at::cuda::getCurrentCUDAStream(dev.index()).stream()), "paged_append");
}

at::Tensor attend(const at::Tensor& qkv, int64_t n_q, const at::Tensor& kp, const at::Tensor& vp, const at::Tensor& table,
                  const at::Tensor& lens, const OptTensor& scores, const OptTensor& slot_pos, const OptTensor& positions,
                  const OptTensor& cos, const OptTensor& sin, c10::optional<double> scale, bool accumulate,
                  const OptTensor& out_) {
  const ts_paged_cache c = cache_view(kp, vp, table, lens, scores, slot_pos);
  const at::Device dev = kp.device();
  c10::cuda::CUDAGuard guard(dev);
  on(qkv, dev, "qkv");
  TORCH_CHECK_VALUE(n_q > 0 && n_q % c.n_kv == 0, n_q, " query heads over ", c.n_kv, " kv heads");
  const int64_t width = (n_q + 2 * (int64_t)c.n_kv) * c.head_dim, owidth = n_q * c.head_dim;
  TORCH_CHECK_VALUE(qkv.dim() == 2 && qkv.size(0) == c.batch && qkv.size(1) == width && qkv.stride(1) == 1,
                    "qkv must be [batch, (n_q + 2 n_kv) head_dim] with contiguous rows, got ", qkv.sizes());
  TORCH_CHECK_VALUE(qkv.scalar_type() == kp.scalar_type(), "qkv must have the cache's type");
  const int64_t rows = rope_rows(c, cos, sin, dev, "paged_decode_attention");
  per_sequence(positions, c, at::kLong, dev, "positions");
  TORCH_CHECK_VALUE(has(positions) || (rows == 0 && !has(slot_pos)),
                    "positions are needed for the rotation and for slot_pos");
  TORCH_CHECK_VALUE(!accumulate || has(scores), "the cache has no scores to accumulate into");
  at::Tensor out;
  if (has(out_)) {
    out = *out_;
    on(out, dev, "out");
    TORCH_CHECK_VALUE(out.dim() == 2 && out.size(0) == c.batch && out.size(1) == owidth &&
                          out.scalar_type() == qkv.scalar_type() && out.stride(1) == 1,
                      "out must be [batch, n_q head_dim] of qkv's type with contiguous rows");
    no_history(out, "paged_decode_attention");
    apart(out, qkv, "paged_decode_attention");
  } else {
    out = fresh({c.batch, owidth}, qkv.scalar_type(), dev);
  }
  cudaStream_t s = at::cuda::getCurrentCUDAStream(dev.index()).stream();
  const Scratch ws = workspace(dev, s, ts_paged_attention_workspace_size(&c, (int)n_q, accumulate));
  const float sc = scale.has_value() ? (float)*scale : 1.0f / std::sqrt((float)c.head_dim);
  done(ts_paged_decode_attention(qkv.data_ptr(), qkv.stride(0), (int)n_q, &c, ptr<int64_t>(positions), ptr<float>(cos),
                                 ptr<float>(sin), rows, sc, accumulate, out.data_ptr(), out.stride(0), ws.data(),
                                 ws.bytes(), s), "paged_decode_attention");
  return out;
}

at::Tensor paged_decode_attention(const at::Tensor& qkv, int64_t n_q, const at::Tensor& kp, const at::Tensor& vp,
                                  const at::Tensor& table, const at::Tensor& lens, const OptTensor& scores,
                                  const OptTensor& slot_pos, const OptTensor& positions, const OptTensor& cos,
                                  const OptTensor& sin, c10::optional<double> scale, bool accumulate) {
  no_tangents("paged_decode_attention", {&qkv});
  return forward_only(attend(qkv, n_q, kp, vp, table, lens, scores, slot_pos, positions, cos, sin, scale, accumulate,
                             c10::nullopt), "paged_decode_attention", {&qkv});
}
at::Tensor& paged_decode_attention_out(const at::Tensor& qkv, int64_t n_q, const at::Tensor& kp, const at::Tensor& vp,
                                       const at::Tensor& table, const at::Tensor& lens, const OptTensor& scores,
                                       const OptTensor& slot_pos, const OptTensor& positions, const OptTensor& cos,
                                       const OptTensor& sin, c10::optional<double> scale, bool accumulate, at::Tensor& out) {
  attend(qkv, n_q, kp, vp, table, lens, scores, slot_pos, positions, cos, sin, scale, accumulate, out);
  return out;
}

void paged_evict(const at::Tensor& kp, const at::Tensor& vp, const at::Tensor& table, const at::Tensor& lens,
                 const OptTensor& scores, const OptTensor& slot_pos, int64_t budget, int64_t recent) {
  const ts_paged_cache c = cache_view(kp, vp, table, lens, scores, slot_pos);
  TORCH_CHECK_VALUE(has(scores) && has(slot_pos), "eviction needs the cache's scores and slot_pos");
  TORCH_CHECK_VALUE(budget > 0 && budget <= INT32_MAX && recent >= 0 && recent <= budget,
                    "budget must be positive and recent in [0, budget], got ", budget, " and ", recent);
  const at::Device dev = kp.device();
  c10::cuda::CUDAGuard guard(dev);
  cudaStream_t s = at::cuda::getCurrentCUDAStream(dev.index()).stream();
  const Scratch ws = workspace(dev, s, ts_paged_evict_workspace_size(&c, (int)budget));
  done(ts_paged_evict(&c, (int)budget, (int)recent, ws.data(), ws.bytes(), s), "paged_evict");
}

// Raises if a bounded wait in a kernel ran out since the last check: of the
// current stream, which is waited for, and of what other streams have finished.
// With `clear`, after such a failure, the whole device is waited for, so that
// no kernel of any stream is on its way, and nobody launches until the flag
// and the counters that CTAs which gave up may have left non-zero are zero
// again (a graph zeroes its own).
void serving_status(int64_t device, bool clear) {
  c10::cuda::CUDAGuard guard((c10::DeviceIndex)device);
  cudaStream_t s = at::cuda::getCurrentCUDAStream((c10::DeviceIndex)device).stream();
  int rc = TS_OK;
  const char* what = "serving_status";
  auto ask = [&](int clear_flags) {
    rc = TS_OK;
    auto one = [&](int r, const char* name) {   // (waits for the stream)
      if (r == TS_OK) return;
      rc = r;
      what = name;
    };
    one(ts_fp4_status(nullptr, 0, clear_flags, s), "ts_fp4_status");
    one(ts_int8_status(clear_flags, s), "ts_int8_status");
    one(ts_paged8_status(clear_flags, s), "ts_paged8_status");
  };
  ask(0);
  if (rc == TS_ERR_TIMEOUT && clear) {
    std::lock_guard<std::mutex> lk(g_mu);
    std::vector<std::unique_lock<std::mutex>> held;
    for (auto& kv : g_ws)
      if (kv.first.first == device) held.emplace_back(kv.second.mu);
    C10_CUDA_CHECK(cudaDeviceSynchronize());
    for (auto& kv : g_ws)
      if (kv.first.first == device && kv.second.t.defined())
        C10_CUDA_CHECK(cudaMemsetAsync(kv.second.t.data_ptr(), 0, ts_serving_counter_bytes(), s));
    ask(1);
  }
  done(rc, what);
}

// ---- shapes for tracing -------------------------------------------------------
//
// The operators on tensors without memory: the outputs' shapes and types, after
// those checks that do not need numbers a tracer may not have.

using c10::SymInt;

SymInt padded(const SymInt& cols) { return (cols + 63) / 64 * 64; }

void fp4_check_meta(const at::Tensor& codes, const at::Tensor& scales, const OptTensor& g, int64_t rows, int64_t cols,
                    int64_t format) {
  fp4_fits(codes, scales, g, rows, cols, format, "Fp4Tensor");
}

std::tuple<at::Tensor, at::Tensor, OptTensor> fp4_quantize_meta(const at::Tensor& x, int64_t format, const OptTensor& scale) {
  TORCH_CHECK_VALUE(x.dim() == 2, "fp4_quantize takes a [rows, cols] tensor, got ", x.dim(), " dimensions");
  code_of(x.scalar_type(), "fp4_quantize");
  TORCH_CHECK_NOT_IMPLEMENTED(format == TS_NVFP4 || format == TS_MXFP4, "fp4_quantize: unknown format");
  TORCH_CHECK_VALUE(!has(scale) || format == TS_NVFP4, "fp4_quantize: only nvfp4 has a tensor scale");
  const SymInt rows = x.sym_size(0), cols = padded(x.sym_size(1));
  const SymInt tiles = (rows + 127) / 128 * ((cols / (format == TS_NVFP4 ? 16 : 32) + 3) / 4);
  const auto bytes = x.options().dtype(at::kByte);
  return {at::empty_symint({rows, cols / 2}, bytes), at::empty_symint({tiles * 512}, bytes),
          format == TS_NVFP4 && !has(scale) ? OptTensor(at::empty({1}, x.options().dtype(at::kFloat))) : c10::nullopt};
}

at::Tensor fp4_dequantize_meta(const at::Tensor& codes, const at::Tensor& scales, const OptTensor& g, int64_t rows,
                               int64_t cols, int64_t format, at::ScalarType dtype) {
  fp4_fits(codes, scales, g, rows, cols, format, "fp4_dequantize");
  code_of(dtype, "fp4_dequantize");
  return forward_only(at::empty({rows, cols}, codes.options().dtype(dtype)), "fp4_dequantize", {in(g)});
}

at::Tensor fp4_matmul_meta(const at::Tensor& ac, const at::Tensor& as, const OptTensor& ag, int64_t m, const at::Tensor& bc,
                           const at::Tensor& bs, const OptTensor& bg, int64_t n, int64_t cols, int64_t format,
                           const OptTensor& bias, at::ScalarType out_dtype) {
  fp4_fits(ac, as, ag, m, cols, format, "fp4_matmul");
  fp4_fits(bc, bs, bg, n, cols, format, "fp4_matmul");
  check_bias(bias, n, bc.device(), "fp4_matmul");
  code_of(out_dtype, "fp4_matmul");
  return forward_only(at::empty({m, n}, ac.options().dtype(out_dtype)), "fp4_matmul", {in(ag), in(bg), in(bias)});
}

at::Tensor fp4_linear_meta(const at::Tensor& x, const at::Tensor& codes, const at::Tensor& scales, const OptTensor& g,
                           int64_t rows, int64_t cols, int64_t format, const OptTensor& bias, const OptTensor& input_scale,
                           c10::optional<at::ScalarType> out_dtype) {
  fp4_fits(codes, scales, g, rows, cols, format, "fp4_linear");
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.sym_size(-1) == cols, "fp4_linear: x has ", x.dim() ? x.sym_size(-1) : SymInt(0),
                    " features, the weight ", cols);
  TORCH_CHECK_VALUE(!has(input_scale) || format == TS_NVFP4, "fp4_linear: only nvfp4 has an input_scale");
  check_bias(bias, rows, codes.device(), "fp4_linear");
  code_of(x.scalar_type(), "fp4_linear");
  const at::ScalarType odt = out_dtype.value_or(x.scalar_type());
  code_of(odt, "fp4_linear");
  c10::SymDimVector shape(x.sym_sizes().begin(), x.sym_sizes().end());
  shape.back() = rows;
  return forward_only(at::empty_symint(shape, x.options().dtype(odt)), "fp4_linear", {&x, in(g), in(bias), in(input_scale)});
}

void paged_check_meta(const at::Tensor& k, const at::Tensor& v, const at::Tensor&, const at::Tensor&, const OptTensor&,
                      const OptTensor&) {
  TORCH_CHECK_VALUE(k.dim() == 4 && v.dim() == 4, "k_pages and v_pages must both be [num_pages, n_kv, page_size, head_dim]");
  TORCH_CHECK_NOT_IMPLEMENTED(k.scalar_type() == at::kHalf || k.scalar_type() == at::kBFloat16,
                              "the cache holds fp16 or bf16");
}

void paged_append_meta(const at::Tensor& k, const at::Tensor& v, const at::Tensor& kp, const at::Tensor&, const at::Tensor&,
                       const at::Tensor&, const OptTensor&, const OptTensor&, const OptTensor&, const OptTensor&,
                       const OptTensor&, const OptTensor&, const OptTensor&) {
  TORCH_CHECK_VALUE(k.dim() == 4 && v.dim() == 4, "k and v must be [batch, tokens, n_kv, head_dim]");
  TORCH_CHECK_VALUE(k.scalar_type() == kp.scalar_type() && v.scalar_type() == kp.scalar_type(),
                    "k and v must have the cache's type");
}

at::Tensor paged_decode_attention_meta(const at::Tensor& qkv, int64_t n_q, const at::Tensor& kp, const at::Tensor&,
                                       const at::Tensor&, const at::Tensor&, const OptTensor& scores, const OptTensor&,
                                       const OptTensor&, const OptTensor&, const OptTensor&, c10::optional<double>,
                                       bool accumulate) {
  TORCH_CHECK_VALUE(n_q > 0 && qkv.dim() == 2 && kp.dim() == 4 && qkv.scalar_type() == kp.scalar_type(),
                    "qkv must be [batch, (n_q + 2 n_kv) head_dim] of the cache's type");
  TORCH_CHECK_VALUE(!accumulate || has(scores), "the cache has no scores to accumulate into");
  return forward_only(at::empty_symint({qkv.sym_size(0), kp.sym_size(3) * n_q}, qkv.options()), "paged_decode_attention",
                      {&qkv});
}
at::Tensor& paged_decode_attention_out_meta(const at::Tensor& qkv, int64_t n_q, const at::Tensor& kp, const at::Tensor& vp,
                                            const at::Tensor& table, const at::Tensor& lens, const OptTensor& scores,
                                            const OptTensor& slot_pos, const OptTensor& positions, const OptTensor& cos,
                                            const OptTensor& sin, c10::optional<double> scale, bool accumulate,
                                            at::Tensor& out) {
  paged_decode_attention_meta(qkv, n_q, kp, vp, table, lens, scores, slot_pos, positions, cos, sin, scale, accumulate);
  no_history(out, "paged_decode_attention");
  return out;
}

void paged_evict_meta(const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&, const OptTensor& scores,
                      const OptTensor& slot_pos, int64_t, int64_t) {
  TORCH_CHECK_VALUE(has(scores) && has(slot_pos), "eviction needs the cache's scores and slot_pos");
}

}  // namespace

#define TS_CACHE(lens) "Tensor(a!) k_pages, Tensor(b!) v_pages, Tensor page_table, " lens " seq_lens, " \
                       "Tensor(d!)? scores, Tensor(e!)? slot_pos"
#define TS_ATTEND "Tensor qkv, int n_q, " TS_CACHE("Tensor") ", Tensor? positions, Tensor? rope_cos, Tensor? rope_sin, " \
                  "float? scale, bool accumulate"

TORCH_LIBRARY_FRAGMENT(tensorshrink, m) {
  m.def("serving_status(int device, bool clear=True) -> ()", &serving_status);
  m.def("fp4_check(Tensor codes, Tensor scales, Tensor? global_scale, int rows, int cols, int format) -> ()");
  m.def("fp4_quantize(Tensor x, int format, Tensor? global_scale) -> (Tensor, Tensor, Tensor?)");
  m.def("fp4_dequantize(Tensor codes, Tensor scales, Tensor? global_scale, int rows, int cols, int format, "
        "ScalarType dtype) -> Tensor");
  m.def("fp4_matmul(Tensor a_codes, Tensor a_scales, Tensor? a_scale, int m, Tensor b_codes, Tensor b_scales, "
        "Tensor? b_scale, int n, int cols, int format, Tensor? bias, ScalarType out_dtype) -> Tensor");
  m.def("fp4_linear(Tensor x, Tensor codes, Tensor scales, Tensor? global_scale, int rows, int cols, int format, "
        "Tensor? bias, Tensor? input_scale, ScalarType? out_dtype=None) -> Tensor");
  m.def("paged_check(Tensor k_pages, Tensor v_pages, Tensor page_table, Tensor seq_lens, Tensor? scores, "
        "Tensor? slot_pos) -> ()");
  m.def("paged_append(Tensor k, Tensor v, " TS_CACHE("Tensor") ", Tensor? positions, Tensor? rope_cos, Tensor? rope_sin, "
        "Tensor? n_new, Tensor? new_scores) -> ()");
  m.def("paged_decode_attention(" TS_ATTEND ") -> Tensor");
  m.def("paged_decode_attention.out(" TS_ATTEND ", *, Tensor(f!) out) -> Tensor(f!)");
  m.def("paged_evict(" TS_CACHE("Tensor(c!)") ", int budget, int recent) -> ()");
}

// (On the CPU the operators say that they do not run there.)
#define TS_IMPL(m, suffix)                                                     \
  m.impl("fp4_check", &fp4_check##suffix);                                     \
  m.impl("fp4_quantize", &fp4_quantize##suffix);                               \
  m.impl("fp4_dequantize", &fp4_dequantize##suffix);                           \
  m.impl("fp4_matmul", &fp4_matmul##suffix);                                   \
  m.impl("fp4_linear", &fp4_linear##suffix);                                   \
  m.impl("paged_check", &paged_check##suffix);                                 \
  m.impl("paged_append", &paged_append##suffix);                               \
  m.impl("paged_decode_attention", &paged_decode_attention##suffix);           \
  m.impl("paged_decode_attention.out", &paged_decode_attention_out##suffix);   \
  m.impl("paged_evict", &paged_evict##suffix);

TORCH_LIBRARY_IMPL(tensorshrink, CUDA, m) { TS_IMPL(m, ) }
TORCH_LIBRARY_IMPL(tensorshrink, CPU, m) { TS_IMPL(m, ) }
TORCH_LIBRARY_IMPL(tensorshrink, Meta, m) { TS_IMPL(m, _meta) }
// (See forward_only: the dispatcher has nothing to do for gradients.)
TORCH_LIBRARY_IMPL(tensorshrink, Autograd, m) {
  for (const char* name : {"fp4_check", "fp4_quantize", "fp4_dequantize", "fp4_matmul", "fp4_linear", "paged_check",
                           "paged_append", "paged_decode_attention", "paged_decode_attention.out", "paged_evict"})
    m.impl(name, torch::CppFunction::makeFallthrough());
}
