// The torch side of the serving operators (kv_append, packed_attention, paged_attention of ops.py): the tensors' checks,
// the outputs and the call of the C ABI.  In C++ because a single token's operators take less time on the GPU than an
// interpreter needs to look at a dozen tensors: an append of one token, called again and again, takes 5.9 us, 12.5 with the
// checks in Python and the call through ctypes (attention of one token 6.0 and 11.0).
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
} calls;

void bind(uintptr_t append, uintptr_t packed, uintptr_t paged, uintptr_t paged_workspace) {
  calls.append = reinterpret_cast<decltype(calls.append)>(append);
  calls.packed = reinterpret_cast<decltype(calls.packed)>(packed);
  calls.paged = reinterpret_cast<decltype(calls.paged)>(paged);
  calls.paged_workspace = reinterpret_cast<decltype(calls.paged_workspace)>(paged_workspace);
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
  return *out;
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.attr("__doc__") = SVLA_TORCH_TAG;  // build.py looks for it in the file
  m.def("bind", &bind);
  m.def("kv_append", &kv_append);
  m.def("packed_attention", &packed_attention);
  m.def("paged_attention", &paged_attention);
}
