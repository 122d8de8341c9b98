// The torch side of the serving operators (kv_append, packed_attention, paged_attention, quantize_rows, linear_i8_rows,
// sample_tokens of ops.py): the tensors' checks, the outputs and the call of the C ABI.  In C++ because a single token's operators take less time on the GPU than an
// interpreter needs to look at a dozen tensors: an append of one token, called again and again, takes 5.9 us, 12.5 with the
// checks in Python and the call through ctypes (attention of one token 6.0 and 11.0).
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/extension.h>

#include <cstdint>
#include <limits>
#include <optional>
#include <string>

#include "../../include/svla.h"

namespace {

using at::Tensor;
using Opt = std::optional<Tensor>;

// entry points of libsvla.so as loaded by _lib.py
struct {
  decltype(&svla_kv_append) append = nullptr;
  decltype(&svla_packed_attention) packed = nullptr;
  decltype(&svla_paged_attention) paged = nullptr;
  decltype(&svla_paged_attention_workspace_size) paged_workspace = nullptr;
  decltype(&svla_quant_rows) quant_rows = nullptr;
  decltype(&svla_linear_i8) linear = nullptr;
  decltype(&svla_sample_tokens) sample = nullptr;
} calls;

void bind(uintptr_t append, uintptr_t packed, uintptr_t paged, uintptr_t paged_workspace, uintptr_t quant_rows, uintptr_t linear,
          uintptr_t sample) {
  calls.append = reinterpret_cast<decltype(calls.append)>(append);
  calls.packed = reinterpret_cast<decltype(calls.packed)>(packed);
  calls.paged = reinterpret_cast<decltype(calls.paged)>(paged);
  calls.paged_workspace = reinterpret_cast<decltype(calls.paged_workspace)>(paged_workspace);
  calls.quant_rows = reinterpret_cast<decltype(calls.quant_rows)>(quant_rows);
  calls.linear = reinterpret_cast<decltype(calls.linear)>(linear);
  calls.sample = reinterpret_cast<decltype(calls.sample)>(sample);
}

// a message's pieces; no streams, whose state belongs to the C++ library that a process loaded
std::string text(const char* s) { return s; }
std::string text(int64_t x) { return std::to_string(x); }
std::string text(int x) { return std::to_string(x); }
std::string text(at::ScalarType t) { return c10::toString(t); }
std::string text(c10::Device d) { return d.str(); }
std::string text(at::IntArrayRef a) {
  std::string s = "[";
  for (size_t i = 0; i < a.size(); ++i) s += (i ? ", " : "") + std::to_string(a[i]);
  return s + "]";
}

template <typename... A>
[[noreturn]] void refuse(const A&... a) {
  throw py::value_error((text(a) + ...));
}

// the library's own refusals and CUDA errors, as SvlaError with its message
void check(int32_t rc, const char* who) {
  if (rc) py::module_::import("smolvla_mujoco_libero_b200._lib").attr("check")(rc, who);
}

// a caller's tensor that a kernel writes has a new version, as after torch's own in-place operations: a graph that saved it notices
void written(const Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}
void written(const Opt& t) {
  if (t) written(*t);
}

int32_t i32(int64_t x, const char* what) {
  if (x > std::numeric_limits<int32_t>::max()) refuse(what, " does not fit 31 bits (", x, ")");
  return static_cast<int32_t>(x);
}

// a number that is not 0 must not become the 0 that stands for head_dim^-1/2
float f32_scale(double x) {
  const float f = static_cast<float>(x);
  if (f == 0.f && x != 0.0) refuse("scale is too small for fp32");
  return f;
}

// what the call's tensors share, taken from its first one
struct Call {
  at::ScalarType dtype;
  int dev;
  int64_t d;

  Call(const Tensor& t, const char* name) : dtype(t.scalar_type()), dev(-1), d(0) {
    if (!t.is_cuda()) refuse(name, " must be a CUDA tensor (there is no CPU path)");
    dev = t.get_device();
    if (t.dim() != 3 || (dtype != at::kBFloat16 && dtype != at::kHalf))
      refuse(name, " must be bf16 or fp16 [rows, heads, head_dim], got ", dtype, " ", t.sizes());
    const int now = c10::cuda::current_device();
    if (dev != now) refuse(name, " is on cuda:", dev, ", the current device is cuda:", now);
    d = t.size(2);
  }
  bool here(const Tensor& t) const { return t.is_cuda() && t.get_device() == dev; }
  int32_t code() const { return dtype == at::kHalf ? SVLA_DT_HALF : SVLA_DT_BF16; }
  svla_stream_t stream() const { return c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(dev)).stream(); }
};

// [rows, heads, d], the heads of a row next to each other, any row stride (a single row's does not matter to torch, so
// it is not taken from it)
struct Rows {
  int64_t rows, heads, rs;

  Rows(const Call& c, const Tensor& t, const char* name) {
    if (t.scalar_type() != c.dtype || !c.here(t) || t.dim() != 3)
      refuse(name, " must be ", c.dtype, " [rows, heads, ", c.d, "] on cuda:", c.dev, ", got ", t.scalar_type(), " ", t.sizes(),
             " on ", t.device());
    rows = t.size(0), heads = t.size(1);
    if (t.size(2) != c.d || (rows && (t.stride(2) != 1 || (t.stride(1) != c.d && heads > 1))))
      refuse(name, " must be [rows, heads, ", c.d, "] with the heads of a row next to each other, got ", t.sizes(),
             " with strides ", t.strides());
    rs = rows > 1 ? t.stride(0) : heads * c.d;
  }
};

const int32_t* ints(const Call& c, const Tensor& t, const char* name, int64_t n) {
  if (t.scalar_type() != at::kInt || !c.here(t) || t.dim() != 1 || t.numel() != n || !t.is_contiguous())
    refuse(name, " must be contiguous int32 [", n, "] on cuda:", c.dev, ", got ", t.scalar_type(), " ", t.sizes(), " on ",
           t.device());
  return static_cast<const int32_t*>(t.const_data_ptr());
}

// starts of a batch's sequences: [batch + 1]
int32_t batch_of(const Call& c, const Tensor& cu, const char* name) {
  ints(c, cu, name, cu.numel() ? cu.numel() : 1);
  return i32(cu.numel() - 1, name);
}

struct Cache {
  int32_t bits, page, n_pages, heads, max_pages;
  int64_t table_rs;

  Cache(const Call& c, const Tensor& cache, const Tensor& table, int64_t batch) {
    if (cache.dim() == 5 && cache.scalar_type() == c.dtype && cache.size(2) == 2 && cache.size(4) == c.d) {
      bits = 16, page = i32(cache.size(3), "page_size");
    } else if (cache.dim() == 4 && cache.scalar_type() == at::kByte && cache.size(3) == c.d + c.d / 4) {
      bits = 4, page = i32(cache.size(2), "page_size");
    } else {
      refuse("cache ", cache.scalar_type(), " ", cache.sizes(), " does not hold entries of ", c.dtype, " [", c.d, "] (see kv_cache)");
    }
    if (!c.here(cache) || !cache.is_contiguous()) refuse("cache must be contiguous on cuda:", c.dev);
    n_pages = i32(cache.size(0), "the number of pages"), heads = i32(cache.size(1), "kv heads");
    if (table.scalar_type() != at::kInt || !c.here(table) || table.dim() != 2 || table.size(0) != batch)
      refuse("page_table must be int32 [", batch, ", max_pages] on cuda:", c.dev, ", got ", table.scalar_type(), " ",
             table.sizes(), " on ", table.device());
    max_pages = i32(table.size(1), "max_pages");
    if (table.stride(1) != 1 && max_pages > 1) refuse("page_table must have unit column stride, got strides ", table.strides());
    table_rs = batch > 1 ? table.stride(0) : max_pages;
  }
};

// the caller's output, or a new one; -> row stride
int64_t output(const Call& c, Opt& out, const Tensor& like, const Rows& r, const char* name, const char* whose) {
  if (!out) {
    out = like.new_empty({r.rows, r.heads, c.d});
    return r.heads * c.d;
  }
  const Rows o(c, *out, name);
  if (o.rows != r.rows || o.heads != r.heads) refuse(name, " must have ", whose, "'s shape");
  return o.rs;
}

py::object kv_append(const Tensor& cache, const Tensor& k, const Tensor& v, const Tensor& cu_q, const Tensor& kv_len,
                     const Tensor& page_table, const Opt& q, const Opt& rope_cs, const Opt& pos, Opt q_out, bool want_rows,
                     Opt k_out, Opt v_out) {
  const Call c(k, "k");
  const Rows rk(c, k, "k"), rv(c, v, "v");
  if (rv.rows != rk.rows || rv.heads != rk.heads) refuse("k and v must have one shape, got ", k.sizes(), " and ", v.sizes());
  svla_kv_append_desc d = {};
  d.batch = batch_of(c, cu_q, "cu_q");
  const Cache ca(c, cache, page_table, d.batch);
  if (ca.heads != rk.heads) refuse("the cache holds ", ca.heads, " kv heads, k has ", rk.heads);
  d.kv_len = ints(c, kv_len, "kv_len", d.batch);
  if (q) {
    const Rows rq(c, *q, "q");
    if (rq.rows != rk.rows) refuse("q has ", rq.rows, " rows, k ", rk.rows);
    d.q_out_rs = output(c, q_out, *q, rq, "q_out", "q");
    d.q = q->const_data_ptr(), d.q_out = q_out->data_ptr(), d.q_rs = rq.rs, d.hq = i32(rq.heads, "query heads");
  } else if (q_out) {
    refuse("q_out without q");
  }
  if (want_rows || k_out) d.k_out_rs = output(c, k_out, k, rk, "k_out", "k"), d.k_out = k_out->data_ptr();
  if (want_rows || v_out) d.v_out_rs = output(c, v_out, v, rv, "v_out", "v"), d.v_out = v_out->data_ptr();
  if (rope_cs) {
    const Tensor& t = *rope_cs;
    if (t.scalar_type() != at::kFloat || !c.here(t) || t.dim() != 3 || t.size(1) != c.d / 2 || t.size(2) != 2 || !t.is_contiguous())
      refuse("rope_cs must be contiguous fp32 [max_pos, ", c.d / 2, ", 2] on cuda:", c.dev);
    if (t.size(0) == 0) refuse("rope_cs holds no positions");  // (its null pointer would stand for no rotation)
    d.max_pos = i32(t.size(0), "max_pos"), d.rope_cs = static_cast<const float*>(t.const_data_ptr());
  }
  if (pos) d.pos = ints(c, *pos, "pos", rk.rows);
  d.total_q = i32(rk.rows, "the number of rows");
  if (d.total_q) {
    d.k = k.const_data_ptr(), d.v = v.const_data_ptr(), d.k_rs = rk.rs, d.v_rs = rv.rs;
    d.cache = cache.data_ptr(), d.cu_q = static_cast<const int32_t*>(cu_q.const_data_ptr());
    d.page_table = static_cast<const int32_t*>(page_table.const_data_ptr()), d.page_table_rs = ca.table_rs;
    d.hkv = ca.heads, d.head_dim = i32(c.d, "head_dim"), d.dtype = c.code();
    d.bits = ca.bits, d.page_size = ca.page, d.n_pages = ca.n_pages, d.max_pages = ca.max_pages;
    check(calls.append(&d, c.stream()), "svla_kv_append");
    written(cache), written(q_out), written(k_out), written(v_out);
  }
  if (want_rows) return py::make_tuple(q_out, *k_out, *v_out);
  return py::cast(q_out);
}

Tensor packed_attention(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& cu_q, const Opt& cu_k, bool causal,
                        double scale, Opt out, int impl) {
  const Call c(q, "q");
  const Rows rq(c, q, "q"), rk(c, k, "k"), rv(c, v, "v");
  if (rv.rows != rk.rows || rv.heads != rk.heads) refuse("k and v must have one shape, got ", k.sizes(), " and ", v.sizes());
  svla_packed_attn_desc d = {};
  d.batch = batch_of(c, cu_q, "cu_q");
  d.cu_q = static_cast<const int32_t*>(cu_q.const_data_ptr());
  d.cu_k = cu_k ? ints(c, *cu_k, "cu_k", static_cast<int64_t>(d.batch) + 1) : d.cu_q;
  d.o_rs = output(c, out, q, rq, "out", "q");
  d.q = q.const_data_ptr(), d.k = k.const_data_ptr(), d.v = v.const_data_ptr(), d.o = out->data_ptr();
  d.q_rs = rq.rs, d.k_rs = rk.rs, d.v_rs = rv.rs;
  d.total_q = i32(rq.rows, "the number of rows"), d.total_k = i32(rk.rows, "the number of rows");
  d.hq = i32(rq.heads, "query heads"), d.hkv = i32(rk.heads, "kv heads");
  d.head_dim = i32(c.d, "head_dim"), d.dtype = c.code(), d.causal = causal;
  d.scale = f32_scale(scale), d.impl = impl;
  check(calls.packed(&d, c.stream()), "svla_packed_attention");
  written(out);
  return *out;
}

Tensor paged_attention(const Tensor& q, const Tensor& cache, const Tensor& cu_q, const Tensor& kv_len,
                       const Tensor& page_table, double scale, Opt out, Opt workspace) {
  const Call c(q, "q");
  const Rows rq(c, q, "q");
  svla_paged_attn_desc d = {};
  d.batch = batch_of(c, cu_q, "cu_q");
  const Cache ca(c, cache, page_table, d.batch);
  d.kv_len = ints(c, kv_len, "kv_len", d.batch);
  d.o_rs = output(c, out, q, rq, "out", "q");
  d.total_q = i32(rq.rows, "the number of rows");
  d.hq = i32(rq.heads, "query heads"), d.hkv = ca.heads;
  d.head_dim = i32(c.d, "head_dim"), d.dtype = c.code();
  d.bits = ca.bits, d.page_size = ca.page, d.n_pages = ca.n_pages, d.max_pages = ca.max_pages;
  if (!workspace) {
    const size_t need = calls.paged_workspace(d.batch, d.total_q, d.hq, d.hkv, d.head_dim, static_cast<int64_t>(ca.max_pages) * ca.page);
    if (need) workspace = at::empty({static_cast<int64_t>(need)}, q.options().dtype(at::kByte));
  } else if (!c.here(*workspace) || workspace->scalar_type() != at::kByte || !workspace->is_contiguous()) {
    refuse("workspace must be contiguous uint8 on cuda:", c.dev);
  }
  if (workspace) d.workspace = workspace->data_ptr(), d.workspace_bytes = static_cast<size_t>(workspace->numel());
  d.q = q.const_data_ptr(), d.cache = cache.const_data_ptr(), d.o = out->data_ptr();
  d.cu_q = static_cast<const int32_t*>(cu_q.const_data_ptr());
  d.page_table = static_cast<const int32_t*>(page_table.const_data_ptr()), d.page_table_rs = ca.table_rs;
  d.q_rs = rq.rs, d.scale = f32_scale(scale);
  check(calls.paged(&d, c.stream()), "svla_paged_attention");
  written(out), written(workspace);
  return *out;
}

// ---------------------------------------------------------------- rows and products in 8 bits, tokens

// the device that a call's tensors share: the first one's, which has to be the current one
struct Where {
  int dev;

  Where(const Tensor& t, const char* name) : dev(-1) {
    if (!t.is_cuda()) refuse(name, " must be a CUDA tensor (there is no CPU path)");
    dev = t.get_device();
    const int now = c10::cuda::current_device();
    if (dev != now) refuse(name, " is on cuda:", dev, ", the current device is cuda:", now);
  }
  bool here(const Tensor& t) const { return t.is_cuda() && t.get_device() == dev; }
  svla_stream_t stream() const { return c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(dev)).stream(); }

  // a matrix [rows, cols] whose rows are contiguous; -> row stride (a single row's does not matter to torch: `one` then)
  int64_t matrix(const Tensor& t, const char* name, at::ScalarType dtype, int64_t rows, int64_t cols, int64_t one) const {
    if (t.scalar_type() != dtype || !here(t) || t.dim() != 2 || t.size(0) != rows || t.size(1) != cols || (cols > 1 && rows && t.stride(1) != 1))
      refuse(name, " must be ", dtype, " [", rows, ", ", cols, "] with contiguous rows on cuda:", dev, ", got ", t.scalar_type(), " ",
             t.sizes(), " with strides ", t.strides(), " on ", t.device());
    if (rows > 1 && t.stride(0) < cols) refuse(name, " has overlapping rows: strides ", t.strides());
    return rows > 1 ? t.stride(0) : one;
  }
  const void* vector(const Tensor& t, const char* name, at::ScalarType dtype, int64_t n) const {
    if (t.scalar_type() != dtype || !here(t) || t.dim() != 1 || t.size(0) != n || !t.is_contiguous())
      refuse(name, " must be contiguous ", dtype, " [", n, "] on cuda:", dev, ", got ", t.scalar_type(), " ", t.sizes(), " on ", t.device());
    return t.const_data_ptr();
  }
};

// an output from torch's allocator, without the dispatcher's way there (half a microsecond each)
Tensor fresh(const Where& w, at::IntArrayRef sizes, at::ScalarType dtype) {
  return Tensor(at::detail::empty_cuda(sizes, dtype, c10::Device(c10::kCUDA, static_cast<c10::DeviceIndex>(w.dev)), std::nullopt));
}

// Outputs of one call.  Small ones share an allocation (one row of 960 with four outputs: 4.6 us a call on the host, 5.9 with
// an allocation each); large ones do not, so that none keeps another's memory.
class Outputs {
 public:
  Outputs(const Where& w, int64_t bytes) : w_(w) {
    if (bytes > 0 && bytes + 4 * kAlign <= kShared) shared_ = fresh(w, {bytes + 4 * kAlign}, at::kByte);
  }
  // [rows, cols], rows `stride` elements apart
  Tensor matrix(int64_t rows, int64_t cols, int64_t stride, at::ScalarType dtype) {
    const int64_t size = static_cast<int64_t>(c10::elementSize(dtype));
    if (!shared_.defined()) {
      const Tensor t = fresh(w_, {rows, stride}, dtype);
      return stride == cols ? t : t.narrow(1, 0, cols);
    }
    Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(shared_.storage()), shared_.key_set(), c10::scalarTypeToTypeMeta(dtype));
    t.unsafeGetTensorImpl()->set_storage_offset(at_ / size);
    const int64_t sizes[2] = {rows, cols}, strides[2] = {stride, 1};
    t.unsafeGetTensorImpl()->set_sizes_and_strides(at::IntArrayRef(sizes, 2), at::IntArrayRef(strides, 2));
    at_ += (rows * stride * size + kAlign - 1) / kAlign * kAlign;
    return t;
  }
  Tensor vector(int64_t n, at::ScalarType dtype) {
    if (!shared_.defined()) return fresh(w_, {n}, dtype);
    Tensor t = matrix(1, n, n, dtype);
    t.unsafeGetTensorImpl()->set_sizes_contiguous(at::IntArrayRef(&n, 1));
    return t;
  }

 private:
  static constexpr int64_t kAlign = 256, kShared = 65536;
  const Where& w_;
  Tensor shared_;
  int64_t at_ = 0;
};

int32_t dtype_code(at::ScalarType t) {
  return t == at::kHalf ? SVLA_DT_HALF : t == at::kBFloat16 ? SVLA_DT_BF16 : t == at::kFloat ? SVLA_DT_FLOAT : -1;
}

py::tuple quantize_rows(const Tensor& x, const Opt& weight, const Opt& bias, double eps, const Opt& residual, const Opt& smooth,
                        bool want_values, Opt codes, Opt scale, Opt sum, Opt values) {
  const Where w(x, "x");
  const at::ScalarType t = x.scalar_type();
  if ((t != at::kBFloat16 && t != at::kHalf) || x.dim() != 2) refuse("x must be bf16 or fp16 [rows, k], got ", t, " ", x.sizes());
  const int64_t m = x.size(0), k = x.size(1);
  svla_quant_rows_desc d = {};
  d.x_rs = w.matrix(x, "x", t, m, k, k);
  if (residual) d.residual_rs = w.matrix(*residual, "residual", t, m, k, k), d.residual = residual->const_data_ptr();
  if (weight) d.weight = w.vector(*weight, "weight", t, k);
  if (bias) d.bias = w.vector(*bias, "bias", t, k);
  if (smooth) d.smooth = static_cast<const float*>(w.vector(*smooth, "smooth", at::kFloat, k));
  const int64_t padded = (k + 15) / 16 * 16;  // rows 16 bytes apart, as the product takes them
  const bool new_sum = !sum && residual, new_values = !values && want_values;
  Outputs made(w, (codes ? 0 : m * padded) + (scale ? 0 : 4 * m) + ((new_sum ? 2 : 0) + (new_values ? 2 : 0)) * m * k);
  d.codes_rs = codes ? w.matrix(*codes, "codes", at::kChar, m, k, k) : padded;
  if (!codes) codes = made.matrix(m, k, padded, at::kChar);
  if (scale) w.vector(*scale, "scale", at::kFloat, m);
  else scale = made.vector(m, at::kFloat);
  if (sum) d.sum_rs = w.matrix(*sum, "sum", t, m, k, k);
  else if (new_sum) sum = made.matrix(m, k, k, t), d.sum_rs = k;
  if (values) d.values_rs = w.matrix(*values, "values", t, m, k, k);
  else if (new_values) values = made.matrix(m, k, k, t), d.values_rs = k;
  d.x = x.const_data_ptr(), d.codes = static_cast<int8_t*>(codes->data_ptr()), d.scale = static_cast<float*>(scale->data_ptr());
  if (sum) d.sum = sum->data_ptr();
  if (values) d.values = values->data_ptr();
  d.m = i32(m, "the number of rows"), d.k = i32(k, "k"), d.dtype = dtype_code(t), d.eps = static_cast<float>(eps);
  check(calls.quant_rows(&d, w.stream()), "svla_quant_rows");
  written(codes), written(scale), written(sum), written(values);
  return py::make_tuple(*codes, *scale, sum, values);
}

Tensor linear_i8_rows(const Tensor& x, const Tensor& xscale, const Tensor& weight, const Tensor& wscale, const Opt& bias,
                      const Opt& residual, bool gated, at::ScalarType dtype, Opt out, int impl) {
  const Where w(x, "x");
  if (x.dim() != 2 || weight.dim() != 2) refuse("x and weight must be matrices, got ", x.sizes(), " and ", weight.sizes());
  const int64_t m = x.size(0), k = x.size(1), rows = weight.size(0), padded = (k + 15) / 16 * 16;
  if (gated && rows % 2) refuse("a gated product's weight holds gate and up rows, got ", rows, " rows");
  const int64_t n = gated ? rows / 2 : rows;
  if (out) dtype = out->scalar_type();
  if (dtype_code(dtype) < 0) refuse("dtype must be bf16, fp16 or fp32, got ", dtype);
  svla_linear_i8_desc d = {};
  d.x_rs = w.matrix(x, "x", at::kChar, m, k, padded);
  d.w_rs = w.matrix(weight, "weight", at::kChar, rows, k, padded);
  d.xscale = static_cast<const float*>(w.vector(xscale, "x_scale", at::kFloat, m));
  d.wscale = static_cast<const float*>(w.vector(wscale, "wscale", at::kFloat, rows));
  if (bias) d.bias = static_cast<const float*>(w.vector(*bias, "bias", at::kFloat, n));
  if (residual) d.residual_rs = w.matrix(*residual, "residual", dtype, m, n, n), d.residual = residual->const_data_ptr();
  if (out) d.out_rs = w.matrix(*out, "out", dtype, m, n, n);
  else out = fresh(w, {m, n}, dtype), d.out_rs = n;
  d.x = static_cast<const int8_t*>(x.const_data_ptr()), d.w = static_cast<const int8_t*>(weight.const_data_ptr());
  d.out = out->data_ptr();
  d.m = i32(m, "the number of rows"), d.n = i32(n, "n"), d.k = i32(k, "k");
  d.dtype = dtype_code(dtype), d.gated = gated, d.impl = impl;
  check(calls.linear(&d, w.stream()), "svla_linear_i8");
  written(out);
  return *out;
}

// a setting of sample_tokens: a tensor with a value per row, a number for all rows, or None
template <typename V>
void setting(const Where& w, const py::object& o, const char* name, at::ScalarType dtype, int64_t batch, const V** rows, V* value) {
  if (o.is_none()) return;
  if (THPVariable_Check(o.ptr())) *rows = static_cast<const V*>(w.vector(THPVariable_Unpack(o.ptr()), name, dtype, batch));
  else *value = o.cast<V>();
}

py::tuple sample_tokens(const Tensor& logits, const Tensor& u, const py::object& temperature, const py::object& top_k,
                        const py::object& top_p, const py::object& min_p, Opt tokens, Opt logprob) {
  const Where w(logits, "logits");
  const at::ScalarType t = logits.scalar_type();
  if (dtype_code(t) < 0 || logits.dim() != 2) refuse("logits must be bf16, fp16 or fp32 [batch, vocab], got ", t, " ", logits.sizes());
  const int64_t batch = logits.size(0), vocab = logits.size(1);
  svla_sample_desc d = {};
  d.logits_rs = w.matrix(logits, "logits", t, batch, vocab, vocab);
  d.u = static_cast<const float*>(w.vector(u, "u", at::kFloat, batch));
  d.temperature_value = 1.f, d.top_p_value = 1.f;
  setting(w, temperature, "temperature", at::kFloat, batch, &d.temperature, &d.temperature_value);
  setting(w, top_k, "top_k", at::kInt, batch, &d.top_k, &d.top_k_value);
  setting(w, top_p, "top_p", at::kFloat, batch, &d.top_p, &d.top_p_value);
  setting(w, min_p, "min_p", at::kFloat, batch, &d.min_p, &d.min_p_value);
  if (tokens) w.vector(*tokens, "tokens", at::kInt, batch);
  else tokens = fresh(w, {batch}, at::kInt);
  if (logprob) w.vector(*logprob, "logprob", at::kFloat, batch);
  else logprob = fresh(w, {batch}, at::kFloat);
  d.logits = logits.const_data_ptr();
  d.tokens = static_cast<int32_t*>(tokens->data_ptr()), d.logprob = static_cast<float*>(logprob->data_ptr());
  d.batch = i32(batch, "the number of rows"), d.vocab = i32(vocab, "vocab"), d.dtype = dtype_code(t);
  check(calls.sample(&d, w.stream()), "svla_sample_tokens");
  written(tokens), written(logprob);
  return py::make_tuple(*tokens, *logprob);
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.attr("__doc__") = SVLA_TORCH_TAG;  // build.py looks for it in the file
  m.def("bind", &bind);
  m.def("kv_append", &kv_append);
  m.def("packed_attention", &packed_attention);
  m.def("paged_attention", &paged_attention);
  m.def("quantize_rows", &quantize_rows);
  m.def("linear_i8_rows", &linear_i8_rows);
  m.def("sample_tokens", &sample_tokens);
}
