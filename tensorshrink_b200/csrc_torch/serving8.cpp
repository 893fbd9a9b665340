// torch.ops.tensorshrink operators of a decoder served in 8 bits: the 8-bit integer
// product, norms of queries and keys, the paged cache of 8 bits and the page
// tables (C ABI: ts_int8_*, ts_qk_norm_rope, ts_paged8_*, ts_paged_reserve,
// ts_paged_release). Conventions as in serving.cpp.
#include "serving_common.h"

namespace {

using namespace ts_torch;

cudaStream_t stream_of(const at::Device& dev) { return at::cuda::getCurrentCUDAStream(dev.index()).stream(); }

void cuda_only(const at::Tensor& t, const char* what) {
  TORCH_CHECK(t.is_cuda(), what, ": tensorshrink_b200 runs on CUDA tensors only (got ", t.device(), ")");
}

// Rows as the kernels read them: contiguous and 16-byte aligned (16-bit elements).
at::Tensor fit_rows(const at::Tensor& t) {
  bool ok = t.stride(-1) == 1 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
  for (int64_t i = 0; i + 1 < t.dim(); ++i) ok = ok && t.stride(i) % 8 == 0;
  return ok ? t : t.clone(at::MemoryFormat::Contiguous);
}

// ---- 8-bit integers -----------------------------------------------------------

int64_t padded16(int64_t cols) { return (cols + 15) / 16 * 16; }

// What can be said of a tensor's description without its memory.
void int8_fits(const at::Tensor& codes, const at::Tensor& scales, int64_t cols, const char* what) {
  TORCH_CHECK_VALUE(codes.scalar_type() == at::kChar && codes.dim() == 2 && scales.scalar_type() == at::kFloat &&
                        scales.dim() == 1 && scales.is_contiguous(),
                    what, ": codes must be int8 [rows, columns], scales contiguous fp32 [rows]");
  TORCH_CHECK_VALUE(cols > 0 && codes.size(1) >= padded16(cols), what, ": rows of codes hold ", codes.size(1), " columns, ",
                    padded16(cols), " wanted (", cols, " padded to 16)");
  TORCH_CHECK_VALUE(scales.size(0) == codes.size(0), what, ": ", scales.size(0), " scales for ", codes.size(0), " rows");
  TORCH_CHECK_VALUE(codes.stride(1) == 1 && (codes.size(0) <= 1 || codes.stride(0) % 16 == 0), what,
                    ": rows of codes must be contiguous and start on 16 bytes");
  on(scales, codes.device(), "scales");
}

ts_int8_tensor int8_view(const at::Tensor& codes, const at::Tensor& scales, int64_t cols, const char* what) {
  cuda_only(codes, what);
  int8_fits(codes, scales, cols, what);
  ts_int8_tensor t{};
  t.codes = static_cast<int8_t*>(codes.data_ptr());
  t.row_stride = codes.size(0) > 1 ? codes.stride(0) : padded16(cols);
  t.scales = static_cast<float*>(scales.data_ptr());
  t.rows = codes.size(0);
  t.cols = cols;
  return t;
}

void int8_check(const at::Tensor& codes, const at::Tensor& scales, int64_t cols) { int8_view(codes, scales, cols, "Int8Tensor"); }

std::tuple<at::Tensor, at::Tensor> int8_quantize(const at::Tensor& x_in) {
  cuda_only(x_in, "int8_quantize");
  const at::Device dev = x_in.device();
  c10::cuda::CUDAGuard guard(dev);
  TORCH_CHECK_VALUE(x_in.dim() == 2 && x_in.size(1) > 0, "int8_quantize takes a [rows, cols] tensor, got ", x_in.sizes());
  const int dt = code_of(x_in.scalar_type(), "int8_quantize");
  const at::Tensor x = x_in.stride(1) == 1 || x_in.size(1) == 1 ? x_in : x_in.contiguous();
  at::Tensor codes = fresh({x.size(0), padded16(x.size(1))}, at::kChar, dev), scales = fresh({x.size(0)}, at::kFloat, dev);
  const ts_int8_tensor t = int8_view(codes, scales, x.size(1), "int8_quantize");
  done(ts_int8_quantize(x.data_ptr(), dt, x.stride(0), &t, stream_of(dev)), "int8_quantize");
  return {codes, scales};
}

at::Tensor int8_dequantize(const at::Tensor& codes, const at::Tensor& scales, int64_t cols, at::ScalarType dtype) {
  const ts_int8_tensor t = int8_view(codes, scales, cols, "int8_dequantize");
  const int dt = code_of(dtype, "int8_dequantize");
  c10::cuda::CUDAGuard guard(codes.device());
  at::Tensor out = fresh({t.rows, cols}, dtype, codes.device());
  done(ts_int8_dequantize(&t, out.data_ptr(), dt, cols, stream_of(codes.device())), "int8_dequantize");
  return forward_only(std::move(out), "int8_dequantize", {&scales});
}

at::Tensor int8_matmul(const at::Tensor& ac, const at::Tensor& as, const at::Tensor& bc, const at::Tensor& bs, int64_t cols,
                       const OptTensor& bias, at::ScalarType out_dtype) {
  const ts_int8_tensor a = int8_view(ac, as, cols, "int8_matmul"), b = int8_view(bc, bs, cols, "int8_matmul");
  const at::Device dev = ac.device();
  on(bc, dev, "b");
  c10::cuda::CUDAGuard guard(dev);
  const int bdt = check_bias(bias, b.rows, dev, "int8_matmul"), dt = code_of(out_dtype, "int8_matmul");
  at::Tensor out = fresh({a.rows, b.rows}, out_dtype, dev);
  cudaStream_t s = stream_of(dev);
  const Scratch ws = workspace(dev, s, ts_int8_matmul_workspace_size(a.rows, b.rows, cols));
  done(ts_int8_matmul(&a, &b, ptr(bias), bdt, out.data_ptr(), dt, b.rows, ws.data(), ws.bytes(), s), "int8_matmul");
  return forward_only(std::move(out), "int8_matmul", {&as, &bs, in(bias)});
}

at::Tensor int8_linear(const at::Tensor& x, const at::Tensor& codes, const at::Tensor& scales, int64_t cols,
                       const OptTensor& bias, c10::optional<at::ScalarType> out_dtype) {
  const ts_int8_tensor w = int8_view(codes, scales, cols, "int8_linear");
  const at::Device dev = codes.device();
  on(x, dev, "x");
  c10::cuda::CUDAGuard guard(dev);
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) == cols, "int8_linear: x has ", x.dim() ? x.size(-1) : 0,
                    " features, the weight ", cols);
  const int xdt = code_of(x.scalar_type(), "int8_linear");
  const at::ScalarType odt = out_dtype.value_or(x.scalar_type());
  const int dt = code_of(odt, "int8_linear"), bdt = check_bias(bias, w.rows, dev, "int8_linear");
  at::Tensor x2d = x.dim() == 2 ? x : x.reshape({-1, cols});
  if (x2d.stride(1) != 1 && cols != 1) x2d = x2d.contiguous();
  std::vector<int64_t> shape(x.sizes().begin(), x.sizes().end());
  shape.back() = w.rows;
  at::Tensor out = fresh(shape, odt, dev);
  const int64_t m = x2d.size(0);
  cudaStream_t s = stream_of(dev);
  const Scratch ws = workspace(dev, s, ts_int8_linear_workspace_size(m, w.rows, cols));
  done(ts_int8_linear(x2d.data_ptr(), xdt, m, x2d.stride(0), &w, ptr(bias), bdt, out.data_ptr(), dt, w.rows, ws.data(),
                      ws.bytes(), s), "int8_linear");
  return forward_only(std::move(out), "int8_linear", {&x, &scales, in(bias)});
}

// ---- norms of queries and keys --------------------------------------------------

void norm_fits(const at::Tensor& x, int64_t n_q, int64_t n_kv, int64_t d, const OptTensor& qw, const OptTensor& kw) {
  for (const OptTensor* w : {&qw, &kw}) {
    if (!has(*w)) continue;
    on(**w, x.device(), "a norm's weight");
    TORCH_CHECK_VALUE((*w)->dim() == 1 && (*w)->size(0) == d && (*w)->is_contiguous() &&
                          ((*w)->scalar_type() == at::kFloat || (*w)->scalar_type() == x.scalar_type()),
                      "qk_norm_rope: weights must be contiguous [head_dim] of fp32 or of x's type");
    TORCH_CHECK_VALUE(!has(qw) || !has(kw) || qw->scalar_type() == kw->scalar_type(),
                      "qk_norm_rope: the weights differ in type");
  }
}

at::Tensor norm_rope(const at::Tensor& x_in, int64_t n_q, int64_t n_kv, const OptTensor& qw_in, const OptTensor& kw_in,
                     const OptTensor& positions, const OptTensor& cos, const OptTensor& sin, double eps, const OptTensor& out_,
                     const ts_paged_cache* cache, const OptTensor& slots) {
  cuda_only(x_in, "qk_norm_rope");
  const at::Device dev = x_in.device();
  c10::cuda::CUDAGuard guard(dev);
  TORCH_CHECK_NOT_IMPLEMENTED(x_in.scalar_type() == at::kHalf || x_in.scalar_type() == at::kBFloat16,
                              "qk_norm_rope: x must be fp16 or bf16");
  TORCH_CHECK_VALUE(n_q >= 0 && n_kv >= 0 && n_q + n_kv > 0 && n_q <= INT16_MAX && n_kv <= INT16_MAX, n_q,
                    " query heads and ", n_kv, " kv heads");
  const int64_t heads = n_q + 2 * n_kv;
  TORCH_CHECK_VALUE(x_in.dim() == 2 && x_in.size(1) > 0 && x_in.size(1) % heads == 0,
                    "qk_norm_rope takes x [tokens, (n_q + 2 n_kv) head_dim], got ", x_in.sizes());
  const int64_t tokens = x_in.size(0), d = x_in.size(1) / heads;
  norm_fits(x_in, n_q, n_kv, d, qw_in, kw_in);
  TORCH_CHECK_VALUE(has(cos) == has(sin), "qk_norm_rope: rope_cos and rope_sin come both or neither");
  int64_t rows = 0;
  if (has(cos)) {
    ts_paged_cache c{};
    c.head_dim = (int32_t)d;
    rows = rope_rows(c, cos, sin, dev, "qk_norm_rope");
    TORCH_CHECK_VALUE(has(positions), "positions are needed for the rotation");
  }
  for (const auto& [t, name] : {std::make_pair(&positions, "positions"), std::make_pair(&slots, "slots")}) {
    if (!has(*t)) continue;
    on(**t, dev, name);
    TORCH_CHECK_VALUE((*t)->scalar_type() == at::kLong && (*t)->dim() == 1 && (*t)->size(0) == tokens && (*t)->is_contiguous(),
                      name, " must be contiguous int64 [tokens]");
  }
  // (weights and tables that do not start on 16 bytes are copied)
  auto aligned = [](const OptTensor& t) {
    return has(t) && reinterpret_cast<uintptr_t>(t->data_ptr()) % 16 != 0 ? OptTensor(t->clone()) : t;
  };
  const OptTensor qw = aligned(qw_in), kw = aligned(kw_in), ct = aligned(cos), st = aligned(sin);
  at::Tensor out, x = x_in;
  if (has(out_)) {
    out = *out_;
    on(out, dev, "out");
    TORCH_CHECK_VALUE(out.sizes() == x.sizes() && out.scalar_type() == x.scalar_type() && out.stride(1) == 1 &&
                          out.stride(0) % 8 == 0 && reinterpret_cast<uintptr_t>(out.data_ptr()) % 16 == 0,
                      "out must have x's shape and type, and contiguous rows that start on 16 bytes");
    no_history(out, "qk_norm_rope");
  } else {
    out = fresh(x.sizes(), x.scalar_type(), dev);
  }
  x = fit_rows(x);
  if (has(out_)) apart(out, x, "qk_norm_rope");
  const int wdt = has(qw) ? code_of(qw->scalar_type(), "qk_norm_rope") : has(kw) ? code_of(kw->scalar_type(), "qk_norm_rope") : 0;
  done(ts_qk_norm_rope(x.data_ptr(), code_of(x.scalar_type(), "qk_norm_rope"), x.stride(0), tokens, (int)n_q, (int)n_kv, (int)d,
                       ptr(qw), ptr(kw), wdt, (float)eps, ptr<int64_t>(positions), ptr<float>(ct), ptr<float>(st), rows,
                       out.data_ptr(), out.stride(0), cache, ptr<int64_t>(slots), stream_of(dev)), "qk_norm_rope");
  return out;
}

at::Tensor qk_norm_rope(const at::Tensor& x, int64_t n_q, int64_t n_kv, const OptTensor& qw, const OptTensor& kw,
                        const OptTensor& positions, const OptTensor& cos, const OptTensor& sin, double eps) {
  return forward_only(norm_rope(x, n_q, n_kv, qw, kw, positions, cos, sin, eps, c10::nullopt, nullptr, c10::nullopt),
                      "qk_norm_rope", {&x, in(qw), in(kw)});
}
at::Tensor& qk_norm_rope_out(const at::Tensor& x, int64_t n_q, int64_t n_kv, const OptTensor& qw, const OptTensor& kw,
                             const OptTensor& positions, const OptTensor& cos, const OptTensor& sin, double eps,
                             at::Tensor& out) {
  norm_rope(x, n_q, n_kv, qw, kw, positions, cos, sin, eps, out, nullptr, c10::nullopt);
  return out;
}

at::Tensor store(const at::Tensor& x, int64_t n_q, int64_t n_kv, const OptTensor& qw, const OptTensor& kw,
                 const OptTensor& positions, const OptTensor& cos, const OptTensor& sin, double eps, const at::Tensor& kp,
                 const at::Tensor& vp, const at::Tensor& table, const at::Tensor& lens, const OptTensor& scores,
                 const OptTensor& slot_pos, const at::Tensor& slots, const OptTensor& out) {
  const ts_paged_cache c = cache_view(kp, vp, table, lens, scores, slot_pos);
  on(x, kp.device(), "x");
  TORCH_CHECK_VALUE(x.scalar_type() == kp.scalar_type() && x.dim() == 2 && c.n_kv == n_kv &&
                        x.size(1) == (n_q + 2 * n_kv) * c.head_dim,
                    "qk_norm_rope: the cache's heads or type differ from x's");
  TORCH_CHECK_VALUE(!has(slot_pos) || has(positions), "positions are needed for slot_pos");
  return norm_rope(x, n_q, n_kv, qw, kw, positions, cos, sin, eps, out, &c, slots);
}
at::Tensor qk_norm_rope_store(const at::Tensor& x, int64_t n_q, int64_t n_kv, const OptTensor& qw, const OptTensor& kw,
                              const OptTensor& positions, const OptTensor& cos, const OptTensor& sin, double eps,
                              const at::Tensor& kp, const at::Tensor& vp, const at::Tensor& table, const at::Tensor& lens,
                              const OptTensor& scores, const OptTensor& slot_pos, const at::Tensor& slots) {
  no_tangents("qk_norm_rope_store", {&x, in(qw), in(kw)});
  return forward_only(store(x, n_q, n_kv, qw, kw, positions, cos, sin, eps, kp, vp, table, lens, scores, slot_pos, slots,
                            c10::nullopt), "qk_norm_rope_store", {&x, in(qw), in(kw)});
}
at::Tensor& qk_norm_rope_store_out(const at::Tensor& x, int64_t n_q, int64_t n_kv, const OptTensor& qw, const OptTensor& kw,
                                   const OptTensor& positions, const OptTensor& cos, const OptTensor& sin, double eps,
                                   const at::Tensor& kp, const at::Tensor& vp, const at::Tensor& table, const at::Tensor& lens,
                                   const OptTensor& scores, const OptTensor& slot_pos, const at::Tensor& slots,
                                   at::Tensor& out) {
  store(x, n_q, n_kv, qw, kw, positions, cos, sin, eps, kp, vp, table, lens, scores, slot_pos, slots, out);
  return out;
}

// ---- paged cache of 8 bits --------------------------------------------------------

void cache8_types(const at::Tensor& k, const at::Tensor& v) {
  TORCH_CHECK_VALUE(k.dim() == 4 && v.dim() == 4, "k_pages and v_pages must both be [num_pages, n_kv, page_size, head_dim]");
  TORCH_CHECK_NOT_IMPLEMENTED(k.scalar_type() == at::kChar || k.scalar_type() == at::kFloat8_e4m3fn,
                              "the cache holds int8 or float8_e4m3fn");
  TORCH_CHECK_VALUE(v.scalar_type() == k.scalar_type(), "k_pages and v_pages differ in type");
}

ts_paged_cache8 cache8_view(const at::Tensor& k, const at::Tensor& v, const at::Tensor& ks, const at::Tensor& vs,
                            const at::Tensor& table, const at::Tensor& lens) {
  cuda_only(k, "PagedKVCache8");
  const at::Device dev = k.device();
  cache8_types(k, v);
  TORCH_CHECK_VALUE(v.sizes() == k.sizes(), "k_pages and v_pages must both be [num_pages, n_kv, page_size, head_dim]");
  TORCH_CHECK_VALUE(v.strides() == k.strides() && k.stride(3) == 1,
                    "k_pages and v_pages must share their strides and have contiguous rows");
  for (const auto& [t, name] : {std::make_pair(&ks, "k_scales"), std::make_pair(&vs, "v_scales")}) {
    on(*t, dev, name);
    TORCH_CHECK_VALUE(t->scalar_type() == at::kFloat && t->dim() == 3 && t->is_contiguous() && t->size(0) == k.size(0) &&
                          t->size(1) == k.size(1) && t->size(2) > 0 && k.size(2) % t->size(2) == 0 && t->sizes() == ks.sizes(),
                      name, " must be contiguous fp32 [num_pages, n_kv, page_size / block]");
  }
  TORCH_CHECK_VALUE(table.scalar_type() == at::kInt && table.dim() == 2 && (table.stride(1) == 1 || table.size(1) <= 1),
                    "page_table must be int32 [batch, max_pages] with contiguous rows");
  TORCH_CHECK_VALUE(lens.scalar_type() == at::kInt && lens.dim() == 1 && lens.size(0) == table.size(0) && lens.is_contiguous(),
                    "seq_lens must be contiguous int32 [batch]");
  on(v, dev, "v_pages");
  on(table, dev, "page_table");
  on(lens, dev, "seq_lens");
  ts_paged_cache8 c{};
  c.k_pages = k.data_ptr();
  c.v_pages = v.data_ptr();
  c.page_stride = k.stride(0);
  c.head_stride = k.stride(1);
  c.token_stride = k.stride(2);
  c.k_scales = static_cast<float*>(ks.data_ptr());
  c.v_scales = static_cast<float*>(vs.data_ptr());
  c.page_table = static_cast<const int32_t*>(table.data_ptr());
  c.table_stride = table.stride(0);
  c.seq_lens = static_cast<int32_t*>(lens.data_ptr());
  c.code = k.scalar_type() == at::kChar ? TS_CACHE_INT8 : TS_CACHE_E4M3;
  c.batch = (int32_t)table.size(0);
  c.n_kv = (int32_t)k.size(1);
  c.head_dim = (int32_t)k.size(3);
  c.page_size = (int32_t)k.size(2);
  c.num_pages = (int32_t)k.size(0);
  c.max_pages = (int32_t)table.size(1);
  c.block = (int32_t)(k.size(2) / ks.size(2));
  TORCH_CHECK_NOT_IMPLEMENTED(c.block % 16 == 0, "a block of ", c.block, " tokens: a multiple of 16 is wanted");
  TORCH_CHECK_NOT_IMPLEMENTED(c.head_dim % 16 == 0 && c.head_dim > 0 && c.head_dim <= 256,
                              "head_dim must be a multiple of 16, <= 256");
  return c;
}

void paged8_check(const at::Tensor& k, const at::Tensor& v, const at::Tensor& ks, const at::Tensor& vs, const at::Tensor& table,
                  const at::Tensor& lens) {
  cache8_view(k, v, ks, vs, table, lens);
}

// A cache's sizes as the helpers of the 16-bit cache take them.
ts_paged_cache sizes_of(const ts_paged_cache8& c) {
  ts_paged_cache r{};
  r.batch = c.batch;
  r.head_dim = c.head_dim;
  return r;
}

void check_16bit(const at::Tensor& t, const char* name) {
  TORCH_CHECK_NOT_IMPLEMENTED(t.scalar_type() == at::kHalf || t.scalar_type() == at::kBFloat16, name, " must be fp16 or bf16");
}

void paged8_append(const at::Tensor& k_in, const at::Tensor& v_in, const at::Tensor& kp, const at::Tensor& vp,
                   const at::Tensor& ks, const at::Tensor& vs, const at::Tensor& table, const at::Tensor& lens,
                   const OptTensor& positions, const OptTensor& cos, const OptTensor& sin, const OptTensor& n_new,
                   const OptTensor& offsets) {
  const ts_paged_cache8 c = cache8_view(kp, vp, ks, vs, table, lens);
  const at::Device dev = kp.device();
  c10::cuda::CUDAGuard guard(dev);
  on(k_in, dev, "k");
  on(v_in, dev, "v");
  const bool packed = has(offsets);
  const int64_t lead = packed ? 1 : 2;
  TORCH_CHECK_VALUE(k_in.dim() == lead + 2 && v_in.sizes() == k_in.sizes() && (packed || k_in.size(0) == c.batch) &&
                        k_in.size(lead) == c.n_kv && k_in.size(lead + 1) == c.head_dim,
                    "k and v must be ", packed ? "[tokens, n_kv, head_dim]" : "[batch, tokens, n_kv, head_dim]", ", got ",
                    k_in.sizes(), " and ", v_in.sizes());
  check_16bit(k_in, "k");
  TORCH_CHECK_VALUE(v_in.scalar_type() == k_in.scalar_type(), "k and v differ in type");
  const ts_paged_cache sz = sizes_of(c);
  const int64_t rows = rope_rows(sz, cos, sin, dev, "paged_append");
  per_sequence(positions, sz, at::kLong, dev, "positions");
  per_sequence(n_new, sz, at::kInt, dev, "n_new");
  if (packed) {
    on(*offsets, dev, "offsets");
    TORCH_CHECK_VALUE(offsets->scalar_type() == at::kInt && offsets->dim() == 1 && offsets->size(0) == c.batch + 1 &&
                          offsets->is_contiguous(),
                      "offsets must be contiguous int32 [batch + 1]");
  }
  const at::Tensor k = fit_rows(k_in), v = fit_rows(v_in);
  const int64_t ks3[3] = {packed ? 0 : k.stride(0), k.stride(lead - 1), k.stride(lead)};
  const int64_t vs3[3] = {packed ? 0 : v.stride(0), v.stride(lead - 1), v.stride(lead)};
  done(ts_paged8_append(k.data_ptr(), ks3, v.data_ptr(), vs3, code_of(k.scalar_type(), "paged_append"), k.size(lead - 1),
                        ptr<int32_t>(offsets), ptr<int32_t>(n_new), &c, ptr<int64_t>(positions), ptr<float>(cos),
                        ptr<float>(sin), rows, stream_of(dev)), "paged_append");
}

std::tuple<at::Tensor, at::Tensor> paged8_dequantize(const at::Tensor& kp, const at::Tensor& vp, const at::Tensor& ks,
                                                     const at::Tensor& vs, const at::Tensor& table, const at::Tensor& lens,
                                                     at::ScalarType dtype) {
  const ts_paged_cache8 c = cache8_view(kp, vp, ks, vs, table, lens);
  const at::Device dev = kp.device();
  c10::cuda::CUDAGuard guard(dev);
  const int dt = code_of(dtype, "paged_dequantize");
  at::Tensor k = fresh(kp.sizes(), dtype, dev), v = fresh(kp.sizes(), dtype, dev);
  done(ts_paged8_dequantize(&c, k.data_ptr(), v.data_ptr(), dt, stream_of(dev)), "paged_dequantize");
  return {forward_only(std::move(k), "paged_dequantize", {&ks}), forward_only(std::move(v), "paged_dequantize", {&vs})};
}

// The output of an attention call: the caller's, or a new one.
// (q: the queries, or their projection, as they are read)
at::Tensor attend_out(const OptTensor& out_, const ts_paged_cache8& c, int64_t width, const at::Tensor& q, const char* what) {
  if (!has(out_)) return fresh({c.batch, width}, q.scalar_type(), q.device());
  on(*out_, q.device(), "out");
  TORCH_CHECK_VALUE(out_->dim() == 2 && out_->size(0) == c.batch && out_->size(1) == width &&
                        out_->scalar_type() == q.scalar_type() && out_->stride(1) == 1,
                    "out must be [batch, n_q head_dim] of the queries' type with contiguous rows");
  no_history(*out_, what);
  apart(*out_, q, what);
  return *out_;
}

float scale_or(c10::optional<double> scale, int d) { return scale.has_value() ? (float)*scale : 1.0f / std::sqrt((float)d); }

at::Tensor attend8(const at::Tensor& q, const at::Tensor& kp, const at::Tensor& vp, const at::Tensor& ks, const at::Tensor& vs,
                   const at::Tensor& table, const at::Tensor& lens, const OptTensor& positions, const OptTensor& cos,
                   const OptTensor& sin, c10::optional<double> scale, const OptTensor& out_) {
  const ts_paged_cache8 c = cache8_view(kp, vp, ks, vs, table, lens);
  const at::Device dev = kp.device();
  c10::cuda::CUDAGuard guard(dev);
  on(q, dev, "q");
  check_16bit(q, "q");
  TORCH_CHECK_VALUE(q.dim() == 2 && q.size(0) == c.batch && q.size(1) > 0 && q.size(1) % ((int64_t)c.n_kv * c.head_dim) == 0 &&
                        q.stride(1) == 1,
                    "q must be [batch, n_q head_dim] with contiguous rows and n_q a multiple of n_kv, got ", q.sizes());
  const ts_paged_cache sz = sizes_of(c);
  const int64_t rows = rope_rows(sz, cos, sin, dev, "paged_attention");
  per_sequence(positions, sz, at::kLong, dev, "positions");
  TORCH_CHECK_VALUE(has(positions) || rows == 0, "positions are needed for the rotation");
  const int64_t n_q = q.size(1) / c.head_dim;
  at::Tensor out = attend_out(out_, c, q.size(1), q, "paged_attention");
  cudaStream_t s = stream_of(dev);
  const Scratch ws = workspace(dev, s, ts_paged8_attention_workspace_size(&c, (int)n_q));
  done(ts_paged8_attention(q.data_ptr(), code_of(q.scalar_type(), "paged_attention"), q.stride(0), (int)n_q, &c,
                           ptr<int64_t>(positions), ptr<float>(cos), ptr<float>(sin), rows, scale_or(scale, c.head_dim),
                           out.data_ptr(), out.stride(0), ws.data(), ws.bytes(), s), "paged_attention");
  return out;
}
at::Tensor paged8_attention(const at::Tensor& q, const at::Tensor& kp, const at::Tensor& vp, const at::Tensor& ks,
                            const at::Tensor& vs, const at::Tensor& table, const at::Tensor& lens, const OptTensor& positions,
                            const OptTensor& cos, const OptTensor& sin, c10::optional<double> scale) {
  return forward_only(attend8(q, kp, vp, ks, vs, table, lens, positions, cos, sin, scale, c10::nullopt), "paged_attention", {&q});
}
at::Tensor& paged8_attention_out(const at::Tensor& q, const at::Tensor& kp, const at::Tensor& vp, const at::Tensor& ks,
                                 const at::Tensor& vs, const at::Tensor& table, const at::Tensor& lens,
                                 const OptTensor& positions, const OptTensor& cos, const OptTensor& sin,
                                 c10::optional<double> scale, at::Tensor& out) {
  attend8(q, kp, vp, ks, vs, table, lens, positions, cos, sin, scale, out);
  return out;
}

at::Tensor decode8(const at::Tensor& qkv_in, int64_t n_q, const at::Tensor& kp, const at::Tensor& vp, const at::Tensor& ks,
                   const at::Tensor& vs, const at::Tensor& table, const at::Tensor& lens, const OptTensor& positions,
                   const OptTensor& cos, const OptTensor& sin, c10::optional<double> scale, const OptTensor& out_) {
  const ts_paged_cache8 c = cache8_view(kp, vp, ks, vs, table, lens);
  const at::Device dev = kp.device();
  c10::cuda::CUDAGuard guard(dev);
  on(qkv_in, dev, "qkv");
  check_16bit(qkv_in, "qkv");
  TORCH_CHECK_VALUE(n_q > 0 && n_q % c.n_kv == 0, n_q, " query heads over ", c.n_kv, " kv heads");
  const int64_t width = (n_q + 2 * (int64_t)c.n_kv) * c.head_dim;
  TORCH_CHECK_VALUE(qkv_in.dim() == 2 && qkv_in.size(0) == c.batch && qkv_in.size(1) == width && qkv_in.stride(1) == 1,
                    "qkv must be [batch, (n_q + 2 n_kv) head_dim] with contiguous rows, got ", qkv_in.sizes());
  const ts_paged_cache sz = sizes_of(c);
  const int64_t rows = rope_rows(sz, cos, sin, dev, "paged_decode_attention");
  per_sequence(positions, sz, at::kLong, dev, "positions");
  TORCH_CHECK_VALUE(has(positions) || rows == 0, "positions are needed for the rotation");
  const at::Tensor qkv = fit_rows(qkv_in);
  at::Tensor out = attend_out(out_, c, n_q * c.head_dim, qkv, "paged_decode_attention");
  cudaStream_t s = stream_of(dev);
  const Scratch ws = workspace(dev, s, ts_paged8_attention_workspace_size(&c, (int)n_q));
  done(ts_paged8_decode_attention(qkv.data_ptr(), code_of(qkv.scalar_type(), "paged_decode_attention"), qkv.stride(0), (int)n_q,
                                  &c, ptr<int64_t>(positions), ptr<float>(cos), ptr<float>(sin), rows,
                                  scale_or(scale, c.head_dim), out.data_ptr(), out.stride(0), ws.data(), ws.bytes(), s),
       "paged_decode_attention");
  return out;
}
at::Tensor paged8_decode_attention(const at::Tensor& qkv, int64_t n_q, const at::Tensor& kp, const at::Tensor& vp,
                                   const at::Tensor& ks, const at::Tensor& vs, const at::Tensor& table, const at::Tensor& lens,
                                   const OptTensor& positions, const OptTensor& cos, const OptTensor& sin,
                                   c10::optional<double> scale) {
  no_tangents("paged_decode_attention", {&qkv});
  return forward_only(decode8(qkv, n_q, kp, vp, ks, vs, table, lens, positions, cos, sin, scale, c10::nullopt),
                      "paged_decode_attention", {&qkv});
}
at::Tensor& paged8_decode_attention_out(const at::Tensor& qkv, int64_t n_q, const at::Tensor& kp, const at::Tensor& vp,
                                        const at::Tensor& ks, const at::Tensor& vs, const at::Tensor& table,
                                        const at::Tensor& lens, const OptTensor& positions, const OptTensor& cos,
                                        const OptTensor& sin, c10::optional<double> scale, at::Tensor& out) {
  decode8(qkv, n_q, kp, vp, ks, vs, table, lens, positions, cos, sin, scale, out);
  return out;
}

// ---- page tables -----------------------------------------------------------------

void pool_fits(const at::Tensor& free, const at::Tensor& n_free) {
  TORCH_CHECK_VALUE(free.scalar_type() == at::kInt && free.dim() == 1 && free.is_contiguous() &&
                        n_free.scalar_type() == at::kInt && n_free.numel() == 1,
                    "PagePool: free must be contiguous int32 [pages], n_free one int32 value");
}

void pool_check(const at::Tensor& free, const at::Tensor& n_free) {
  cuda_only(free, "PagePool");
  pool_fits(free, n_free);
  on(n_free, free.device(), "n_free");
}

void table_views(const at::Tensor& free, const at::Tensor& n_free, const at::Tensor& table, const at::Tensor& lens,
                 int64_t page_size, int64_t num_pages, const at::Tensor& per_sequence, const char* name, ts_page_pool* p,
                 ts_page_table* t) {
  pool_check(free, n_free);
  const at::Device dev = free.device();
  on(table, dev, "page_table");
  on(lens, dev, "seq_lens");
  on(per_sequence, dev, name);
  TORCH_CHECK_VALUE(table.scalar_type() == at::kInt && table.dim() == 2 && (table.stride(1) == 1 || table.size(1) <= 1),
                    "page_table must be int32 [batch, max_pages] with contiguous rows");
  TORCH_CHECK_VALUE(lens.scalar_type() == at::kInt && lens.dim() == 1 && lens.size(0) == table.size(0) && lens.is_contiguous(),
                    "seq_lens must be contiguous int32 [batch]");
  TORCH_CHECK_VALUE(per_sequence.scalar_type() == at::kInt && per_sequence.dim() == 1 &&
                        per_sequence.size(0) == table.size(0) && per_sequence.is_contiguous(),
                    name, " must be contiguous int32 [batch]");
  TORCH_CHECK_VALUE(page_size > 0 && page_size <= INT32_MAX && num_pages >= 0 && num_pages <= INT32_MAX, "bad page_size or num_pages");
  // (rows that share memory would be written by several sequences)
  TORCH_CHECK_VALUE(table.size(0) <= 1 || table.stride(0) >= table.size(1), "the rows of page_table overlap");
  *p = ts_page_pool{static_cast<int32_t*>(free.data_ptr()), static_cast<int32_t*>(n_free.data_ptr()), (int32_t)free.size(0), 0};
  *t = ts_page_table{static_cast<int32_t*>(table.data_ptr()), table.stride(0), static_cast<int32_t*>(lens.data_ptr()),
                     (int32_t)table.size(0), (int32_t)table.size(1), (int32_t)page_size, (int32_t)num_pages};
}

using Slots = std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor>;

Slots paged_reserve(const at::Tensor& free, const at::Tensor& n_free, const at::Tensor& table, const at::Tensor& lens,
                    int64_t page_size, int64_t num_pages, const at::Tensor& n_new, const OptTensor& first, int64_t tokens) {
  ts_page_pool p;
  ts_page_table t;
  table_views(free, n_free, table, lens, page_size, num_pages, n_new, "n_new", &p, &t);
  const at::Device dev = free.device();
  c10::cuda::CUDAGuard guard(dev);
  TORCH_CHECK_VALUE(tokens >= 0 && tokens <= INT32_MAX - 1, "paged_reserve: bad number of tokens ", tokens);
  if (has(first)) {
    on(*first, dev, "positions");
    TORCH_CHECK_VALUE(first->scalar_type() == at::kLong && first->dim() == 1 && first->size(0) == t.batch && first->is_contiguous(),
                      "positions must be contiguous int64 [batch]");
  }
  at::Tensor granted = fresh({t.batch}, at::kInt, dev), offsets = fresh({t.batch + 1}, at::kInt, dev),
             slots = fresh({tokens}, at::kLong, dev), positions = fresh({tokens}, at::kLong, dev),
             sequences = fresh({tokens}, at::kInt, dev);
  if (t.batch == 0) {
    offsets.zero_();
    slots.fill_(-1);
    positions.zero_();
    sequences.fill_(-1);
  } else {
    done(ts_paged_reserve(&p, &t, static_cast<const int32_t*>(n_new.data_ptr()), ptr<int64_t>(first), tokens,
                          static_cast<int32_t*>(granted.data_ptr()), static_cast<int32_t*>(offsets.data_ptr()),
                          static_cast<int64_t*>(slots.data_ptr()), static_cast<int64_t*>(positions.data_ptr()),
                          static_cast<int32_t*>(sequences.data_ptr()), stream_of(dev)), "paged_reserve");
  }
  return {granted, offsets, slots, positions, sequences};
}

void paged_release(const at::Tensor& free, const at::Tensor& n_free, const at::Tensor& table, const at::Tensor& lens,
                   int64_t page_size, int64_t num_pages, const at::Tensor& keep) {
  ts_page_pool p;
  ts_page_table t;
  table_views(free, n_free, table, lens, page_size, num_pages, keep, "keep", &p, &t);
  c10::cuda::CUDAGuard guard(free.device());
  done(ts_paged_release(&p, &t, static_cast<const int32_t*>(keep.data_ptr()), stream_of(free.device())), "paged_release");
}

// ---- shapes for tracing -------------------------------------------------------

using c10::SymInt;

void int8_check_meta(const at::Tensor& codes, const at::Tensor& scales, int64_t cols) { int8_fits(codes, scales, cols, "Int8Tensor"); }

std::tuple<at::Tensor, at::Tensor> int8_quantize_meta(const at::Tensor& x) {
  TORCH_CHECK_VALUE(x.dim() == 2, "int8_quantize takes a [rows, cols] tensor, got ", x.dim(), " dimensions");
  code_of(x.scalar_type(), "int8_quantize");
  return {at::empty_symint({x.sym_size(0), (x.sym_size(1) + 15) / 16 * 16}, x.options().dtype(at::kChar)),
          at::empty_symint({x.sym_size(0)}, x.options().dtype(at::kFloat))};
}

at::Tensor int8_dequantize_meta(const at::Tensor& codes, const at::Tensor& scales, int64_t cols, at::ScalarType dtype) {
  code_of(dtype, "int8_dequantize");
  return forward_only(at::empty_symint({codes.sym_size(0), cols}, codes.options().dtype(dtype)), "int8_dequantize", {&scales});
}

at::Tensor int8_matmul_meta(const at::Tensor& ac, const at::Tensor& as, const at::Tensor& bc, const at::Tensor& bs, int64_t,
                            const OptTensor& bias, at::ScalarType out_dtype) {
  code_of(out_dtype, "int8_matmul");
  return forward_only(at::empty_symint({ac.sym_size(0), bc.sym_size(0)}, ac.options().dtype(out_dtype)), "int8_matmul",
                      {&as, &bs, in(bias)});
}

at::Tensor int8_linear_meta(const at::Tensor& x, const at::Tensor& codes, const at::Tensor& scales, int64_t cols,
                            const OptTensor& bias, c10::optional<at::ScalarType> out_dtype) {
  int8_fits(codes, scales, cols, "int8_linear");
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.sym_size(-1) == cols, "int8_linear: x has ", x.dim() ? x.sym_size(-1) : SymInt(0),
                    " features, the weight ", cols);
  check_bias(bias, codes.size(0), codes.device(), "int8_linear");
  code_of(x.scalar_type(), "int8_linear");
  const at::ScalarType odt = out_dtype.value_or(x.scalar_type());
  code_of(odt, "int8_linear");
  c10::SymDimVector shape(x.sym_sizes().begin(), x.sym_sizes().end());
  shape.back() = codes.sym_size(0);
  return forward_only(at::empty_symint(shape, x.options().dtype(odt)), "int8_linear", {&x, &scales, in(bias)});
}

at::Tensor qk_norm_rope_meta(const at::Tensor& x, int64_t n_q, int64_t n_kv, const OptTensor& qw, const OptTensor& kw,
                             const OptTensor& positions, const OptTensor& cos, const OptTensor& sin, double) {
  TORCH_CHECK_VALUE(x.dim() == 2 && n_q >= 0 && n_kv >= 0 && n_q + n_kv > 0,
                    "qk_norm_rope takes x [tokens, (n_q + 2 n_kv) head_dim]");
  check_16bit(x, "x");
  TORCH_CHECK_VALUE(has(cos) == has(sin), "qk_norm_rope: rope_cos and rope_sin come both or neither");
  TORCH_CHECK_VALUE(has(positions) || !has(cos), "positions are needed for the rotation");
  return forward_only(at::empty_symint(x.sym_sizes(), x.options()), "qk_norm_rope", {&x, in(qw), in(kw)});
}
at::Tensor& qk_norm_rope_out_meta(const at::Tensor& x, int64_t n_q, int64_t n_kv, const OptTensor& qw, const OptTensor& kw,
                                  const OptTensor& positions, const OptTensor& cos, const OptTensor& sin, double eps,
                                  at::Tensor& out) {
  qk_norm_rope_meta(x, n_q, n_kv, qw, kw, positions, cos, sin, eps);
  no_history(out, "qk_norm_rope");
  return out;
}
at::Tensor qk_norm_rope_store_meta(const at::Tensor& x, int64_t n_q, int64_t n_kv, const OptTensor& qw, const OptTensor& kw,
                                   const OptTensor& positions, const OptTensor& cos, const OptTensor& sin, double eps,
                                   const at::Tensor& kp, const at::Tensor&, const at::Tensor&, const at::Tensor&,
                                   const OptTensor&, const OptTensor&, const at::Tensor&) {
  TORCH_CHECK_VALUE(x.scalar_type() == kp.scalar_type(), "qk_norm_rope: the cache's heads or type differ from x's");
  return qk_norm_rope_meta(x, n_q, n_kv, qw, kw, positions, cos, sin, eps);
}
at::Tensor& qk_norm_rope_store_out_meta(const at::Tensor& x, int64_t n_q, int64_t n_kv, const OptTensor& qw, const OptTensor& kw,
                                        const OptTensor& positions, const OptTensor& cos, const OptTensor& sin, double eps,
                                        const at::Tensor& kp, const at::Tensor&, const at::Tensor&, const at::Tensor&,
                                        const OptTensor&, const OptTensor&, const at::Tensor&, at::Tensor& out) {
  TORCH_CHECK_VALUE(x.scalar_type() == kp.scalar_type(), "qk_norm_rope: the cache's heads or type differ from x's");
  qk_norm_rope_meta(x, n_q, n_kv, qw, kw, positions, cos, sin, eps);
  no_history(out, "qk_norm_rope");
  return out;
}

void paged8_check_meta(const at::Tensor& k, const at::Tensor& v, const at::Tensor&, const at::Tensor&, const at::Tensor&,
                       const at::Tensor&) {
  cache8_types(k, v);
}

void paged8_append_meta(const at::Tensor& k, const at::Tensor& v, const at::Tensor& kp, const at::Tensor& vp, const at::Tensor&,
                        const at::Tensor&, const at::Tensor&, const at::Tensor&, const OptTensor&, const OptTensor&,
                        const OptTensor&, const OptTensor&, const OptTensor& offsets) {
  cache8_types(kp, vp);
  const int64_t dims = has(offsets) ? 3 : 4;
  TORCH_CHECK_VALUE(k.dim() == dims && v.dim() == dims, "k and v must be ",
                    has(offsets) ? "[tokens, n_kv, head_dim]" : "[batch, tokens, n_kv, head_dim]");
  check_16bit(k, "k");
  TORCH_CHECK_VALUE(v.scalar_type() == k.scalar_type(), "k and v differ in type");
}

std::tuple<at::Tensor, at::Tensor> paged8_dequantize_meta(const at::Tensor& kp, const at::Tensor& vp, const at::Tensor&,
                                                          const at::Tensor&, const at::Tensor&, const at::Tensor&,
                                                          at::ScalarType dtype) {
  cache8_types(kp, vp);
  code_of(dtype, "paged_dequantize");
  return {at::empty_symint(kp.sym_sizes(), kp.options().dtype(dtype)), at::empty_symint(kp.sym_sizes(), kp.options().dtype(dtype))};
}

at::Tensor paged8_attention_meta(const at::Tensor& q, const at::Tensor& kp, const at::Tensor& vp, const at::Tensor&,
                                 const at::Tensor&, const at::Tensor&, const at::Tensor&, const OptTensor&, const OptTensor&,
                                 const OptTensor&, c10::optional<double>) {
  cache8_types(kp, vp);
  check_16bit(q, "q");
  TORCH_CHECK_VALUE(q.dim() == 2, "q must be [batch, n_q head_dim]");
  return forward_only(at::empty_symint(q.sym_sizes(), q.options()), "paged_attention", {&q});
}
at::Tensor& paged8_attention_out_meta(const at::Tensor& q, const at::Tensor& kp, const at::Tensor& vp, const at::Tensor& ks,
                                      const at::Tensor& vs, const at::Tensor& table, const at::Tensor& lens,
                                      const OptTensor& positions, const OptTensor& cos, const OptTensor& sin,
                                      c10::optional<double> scale, at::Tensor& out) {
  paged8_attention_meta(q, kp, vp, ks, vs, table, lens, positions, cos, sin, scale);
  no_history(out, "paged_attention");
  return out;
}

at::Tensor paged8_decode_attention_meta(const at::Tensor& qkv, int64_t n_q, const at::Tensor& kp, const at::Tensor& vp,
                                        const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&,
                                        const OptTensor&, const OptTensor&, const OptTensor&, c10::optional<double>) {
  cache8_types(kp, vp);
  check_16bit(qkv, "qkv");
  TORCH_CHECK_VALUE(n_q > 0 && qkv.dim() == 2, "qkv must be [batch, (n_q + 2 n_kv) head_dim]");
  return forward_only(at::empty_symint({qkv.sym_size(0), kp.sym_size(3) * n_q}, qkv.options()), "paged_decode_attention", {&qkv});
}
at::Tensor& paged8_decode_attention_out_meta(const at::Tensor& qkv, int64_t n_q, const at::Tensor& kp, const at::Tensor& vp,
                                             const at::Tensor& ks, const at::Tensor& vs, const at::Tensor& table,
                                             const at::Tensor& lens, const OptTensor& positions, const OptTensor& cos,
                                             const OptTensor& sin, c10::optional<double> scale, at::Tensor& out) {
  paged8_decode_attention_meta(qkv, n_q, kp, vp, ks, vs, table, lens, positions, cos, sin, scale);
  no_history(out, "paged_decode_attention");
  return out;
}

void pool_check_meta(const at::Tensor& free, const at::Tensor& n_free) { pool_fits(free, n_free); }

Slots paged_reserve_meta(const at::Tensor& free, const at::Tensor&, const at::Tensor&, const at::Tensor& lens, int64_t, int64_t,
                         const at::Tensor&, const OptTensor&, SymInt tokens) {
  TORCH_CHECK_VALUE(!tokens.maybe_as_int() || *tokens.maybe_as_int() >= 0, "paged_reserve: bad number of tokens ", tokens);
  const auto i32 = free.options().dtype(at::kInt), i64 = free.options().dtype(at::kLong);
  return {at::empty_symint({lens.sym_size(0)}, i32), at::empty_symint({lens.sym_size(0) + 1}, i32), at::empty_symint({tokens}, i64),
          at::empty_symint({tokens}, i64), at::empty_symint({tokens}, i32)};
}

void paged_release_meta(const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&, int64_t, int64_t,
                        const at::Tensor&) {}

}  // namespace

#define TS_CACHE "Tensor(a!) k_pages, Tensor(b!) v_pages, Tensor page_table, Tensor seq_lens, Tensor(d!)? scores, " \
                 "Tensor(e!)? slot_pos"
#define TS_CACHE8_READ "Tensor k_pages, Tensor v_pages, Tensor k_scales, Tensor v_scales, Tensor page_table, Tensor seq_lens"
#define TS_CACHE8_WRITE "Tensor(a!) k_pages, Tensor(b!) v_pages, Tensor(c!) k_scales, Tensor(d!) v_scales, " \
                        "Tensor page_table, Tensor seq_lens"
#define TS_NORM "Tensor x, int n_q, int n_kv, Tensor? q_weight, Tensor? k_weight, Tensor? positions, Tensor? rope_cos, " \
                "Tensor? rope_sin, float eps"
#define TS_ROPE "Tensor? positions, Tensor? rope_cos, Tensor? rope_sin"

TORCH_LIBRARY_FRAGMENT(tensorshrink, m) {
  m.def("int8_check(Tensor codes, Tensor scales, int cols) -> ()");
  m.def("int8_quantize(Tensor x) -> (Tensor, Tensor)");
  m.def("int8_dequantize(Tensor codes, Tensor scales, int cols, ScalarType dtype) -> Tensor");
  m.def("int8_matmul(Tensor a_codes, Tensor a_scales, Tensor b_codes, Tensor b_scales, int cols, Tensor? bias, "
        "ScalarType out_dtype) -> Tensor");
  m.def("int8_linear(Tensor x, Tensor codes, Tensor scales, int cols, Tensor? bias, ScalarType? out_dtype=None) -> Tensor");
  m.def("qk_norm_rope(" TS_NORM ") -> Tensor");
  m.def("qk_norm_rope.out(" TS_NORM ", *, Tensor(f!) out) -> Tensor(f!)");
  m.def("qk_norm_rope_store(" TS_NORM ", " TS_CACHE ", Tensor slots) -> Tensor");
  m.def("qk_norm_rope_store.out(" TS_NORM ", " TS_CACHE ", Tensor slots, *, Tensor(f!) out) -> Tensor(f!)");
  m.def("paged8_check(" TS_CACHE8_READ ") -> ()");
  m.def("paged8_append(Tensor k, Tensor v, " TS_CACHE8_WRITE ", " TS_ROPE ", Tensor? n_new, Tensor? offsets) -> ()");
  m.def("paged8_dequantize(" TS_CACHE8_READ ", ScalarType dtype) -> (Tensor, Tensor)");
  m.def("paged8_attention(Tensor q, " TS_CACHE8_READ ", " TS_ROPE ", float? scale) -> Tensor");
  m.def("paged8_attention.out(Tensor q, " TS_CACHE8_READ ", " TS_ROPE ", float? scale, *, Tensor(f!) out) -> Tensor(f!)");
  m.def("paged8_decode_attention(Tensor qkv, int n_q, " TS_CACHE8_WRITE ", " TS_ROPE ", float? scale) -> Tensor");
  m.def("paged8_decode_attention.out(Tensor qkv, int n_q, " TS_CACHE8_WRITE ", " TS_ROPE ", float? scale, *, "
        "Tensor(f!) out) -> Tensor(f!)");
  m.def("pool_check(Tensor free, Tensor n_free) -> ()");
  m.def("paged_reserve(Tensor free, Tensor(a!) n_free, Tensor(b!) page_table, Tensor seq_lens, int page_size, int num_pages, "
        "Tensor n_new, Tensor? positions, SymInt tokens) -> (Tensor, Tensor, Tensor, Tensor, Tensor)");
  m.def("paged_release(Tensor(a!) free, Tensor(b!) n_free, Tensor(c!) page_table, Tensor(d!) seq_lens, int page_size, "
        "int num_pages, Tensor keep) -> ()");
}

// (On the CPU the operators say that they do not run there.)
#define TS_IMPL8(m, suffix)                                                        \
  m.impl("int8_check", &int8_check##suffix);                                       \
  m.impl("int8_quantize", &int8_quantize##suffix);                                 \
  m.impl("int8_dequantize", &int8_dequantize##suffix);                             \
  m.impl("int8_matmul", &int8_matmul##suffix);                                     \
  m.impl("int8_linear", &int8_linear##suffix);                                     \
  m.impl("qk_norm_rope", &qk_norm_rope##suffix);                                   \
  m.impl("qk_norm_rope.out", &qk_norm_rope_out##suffix);                           \
  m.impl("qk_norm_rope_store", &qk_norm_rope_store##suffix);                       \
  m.impl("qk_norm_rope_store.out", &qk_norm_rope_store_out##suffix);               \
  m.impl("paged8_check", &paged8_check##suffix);                                   \
  m.impl("paged8_append", &paged8_append##suffix);                                 \
  m.impl("paged8_dequantize", &paged8_dequantize##suffix);                         \
  m.impl("paged8_attention", &paged8_attention##suffix);                           \
  m.impl("paged8_attention.out", &paged8_attention_out##suffix);                   \
  m.impl("paged8_decode_attention", &paged8_decode_attention##suffix);             \
  m.impl("paged8_decode_attention.out", &paged8_decode_attention_out##suffix);     \
  m.impl("pool_check", &pool_check##suffix);                                       \
  m.impl("paged_reserve", &paged_reserve##suffix);                                 \
  m.impl("paged_release", &paged_release##suffix);

TORCH_LIBRARY_IMPL(tensorshrink, CUDA, m) { TS_IMPL8(m, ) }
TORCH_LIBRARY_IMPL(tensorshrink, CPU, m) { TS_IMPL8(m, ) }
TORCH_LIBRARY_IMPL(tensorshrink, Meta, m) { TS_IMPL8(m, _meta) }
// (The operators have no gradients: the dispatcher has nothing to do for them.)
TORCH_LIBRARY_IMPL(tensorshrink, Autograd, m) {
  for (const char* name : {"int8_check", "int8_quantize", "int8_dequantize", "int8_matmul", "int8_linear", "qk_norm_rope",
                           "qk_norm_rope.out", "qk_norm_rope_store", "qk_norm_rope_store.out", "paged8_check", "paged8_append",
                           "paged8_dequantize", "paged8_attention", "paged8_attention.out", "paged8_decode_attention",
                           "paged8_decode_attention.out", "pool_check", "paged_reserve", "paged_release"})
    m.impl(name, torch::CppFunction::makeFallthrough());
}
