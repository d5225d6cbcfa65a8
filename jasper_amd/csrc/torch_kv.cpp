// torch_kv.cpp -- the paged cache's calls (include/jasper_amd.h) as a Python
// module that takes torch tensors: argument checks, outputs, scratch, the
// current stream, and the rotary positions' gradient. They are called once or
// twice per layer and token, and a small one's kernels take 4 to 10 us: through
// ctypes its host side took 15 to 20 us, here 4 to 8.
#include <torch/extension.h>

#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>

#include <algorithm>
#include <cmath>
#include <optional>
#include <string>
#include <vector>

#include "../../include/jasper_amd.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;
namespace py = pybind11;

// A failure that is not the caller's: jasper_amd.JasperError in Python.
struct Failure : std::runtime_error {
  using std::runtime_error::runtime_error;
};

void check(int64_t r) {
  if (r >= 0) return;
  const std::string text = jasper_last_error();
  for (const char* caller : {"must be", "too large", "out of range"})
    TORCH_CHECK_VALUE(text.find(caller) == std::string::npos, text);
  throw Failure(text);
}

void* current_stream(int64_t device) { return c10::hip::getCurrentHIPStream((c10::DeviceIndex)device).stream(); }

// 0 fp16, 1 bf16, 2 e4m3, -1 others
int32_t type_of(const Tensor& t) {
  const auto s = t.scalar_type();
  return s == at::kHalf ? 0 : s == at::kBFloat16 ? 1 : s == at::kFloat8_e4m3fn ? 2 : -1;
}

bool is_row_type(const Tensor& t) { return type_of(t) == 0 || type_of(t) == 1; }

const float* scale_ptr(const char* name, const OptTensor& t, int64_t heads, const Tensor& pages) {
  if (!t) return nullptr;
  TORCH_CHECK_VALUE(pages.scalar_type() == at::kFloat8_e4m3fn, name, " needs float8_e4m3fn pages");
  TORCH_CHECK_VALUE(t->scalar_type() == at::kFloat && t->dim() == 1 && t->size(0) == heads && t->is_contiguous() &&
                        t->device() == pages.device(),
                    name, " must be a contiguous float32 [", heads, "] tensor on the pages' device");
  return (const float*)t->data_ptr();
}

jasperx_kv_pages pages_of(const Tensor& k, const Tensor& v, const OptTensor& k_scale, const OptTensor& v_scale,
                          bool layers) {
  jasperx_kv_pages p{};
  p.type = type_of(k);
  TORCH_CHECK_VALUE(p.type >= 0, "pages must be float16, bfloat16 or float8_e4m3fn, got ", k.dtype());
  TORCH_CHECK_VALUE(v.scalar_type() == k.scalar_type() && v.sizes() == k.sizes() && v.strides() == k.strides() &&
                        v.device() == k.device(),
                    "k_pages and v_pages must have the same type, shape, strides and device");
  TORCH_CHECK_VALUE(k.is_cuda(), "k_pages must be a CUDA tensor");
  const int first = layers && k.dim() == 5 ? 1 : 0;
  TORCH_CHECK_VALUE(k.dim() == 4 + first, "pages must be [", layers ? "layers, " : "",
                    "n_pages, kv_heads, page_size, dim], got ", k.dim(), "D");
  const auto size = k.sizes().slice(first), stride = k.strides().slice(first);
  TORCH_CHECK_VALUE(stride[3] == 1, "the last dimension of the pages must be contiguous");
  for (int i = 0; i < 4; ++i) TORCH_CHECK_VALUE(size[i] <= INT32_MAX, "pages are too large");
  p.k = k.data_ptr(), p.v = v.data_ptr();
  p.layers = first ? (int32_t)k.size(0) : 1, p.layer_stride = first ? k.stride(0) : 0;
  p.pages = (int32_t)size[0], p.heads = (int32_t)size[1], p.page_size = (int32_t)size[2], p.dim = (int32_t)size[3];
  p.page_stride = stride[0], p.head_stride = stride[1], p.row_stride = stride[2];
  p.k_scale = scale_ptr("k_scale", k_scale, p.heads, k), p.v_scale = scale_ptr("v_scale", v_scale, p.heads, k);
  return p;
}

Tensor indexes(const char* name, const Tensor& t, const Tensor& like) {
  TORCH_CHECK_VALUE(t.scalar_type() == at::kLong || t.scalar_type() == at::kInt, name,
                    " must be int32 or int64, got ", t.dtype());
  TORCH_CHECK_VALUE(t.device() == like.device(), name, " must be on ", like.device(), ", is on ", t.device());
  return t.contiguous();
}

struct Table {
  const float *cos = nullptr, *sin = nullptr;
  int64_t rows = 0, rot = 0;
};

Table table_of(const OptTensor& cos, const OptTensor& sin, const Tensor& like) {
  if (!cos && !sin) return {};
  TORCH_CHECK_VALUE(cos && sin && cos->scalar_type() == at::kFloat && sin->scalar_type() == at::kFloat &&
                        cos->dim() == 2 && cos->sizes() == sin->sizes() && cos->is_contiguous() &&
                        sin->is_contiguous() && cos->device() == like.device() && sin->device() == like.device(),
                    "cos and sin must be contiguous float32 [n_positions, rot_dim / 2] tensors on ", like.device());
  return {(const float*)cos->data_ptr(), (const float*)sin->data_ptr(), cos->size(0), 2 * cos->size(1)};
}

// [..., heads, dim] as rows [n][heads][dim] with contiguous values; `held`
// keeps what had to be copied.
jasperx_head_rows rows_of(const Tensor& t, Tensor& held) {
  held = t;
  if (held.dim() != 3) held = held.dim() > 3 ? held.flatten(0, -3) : held.unsqueeze(0);
  if (held.stride(2) != 1) held = held.contiguous();
  return {held.data_ptr(), held.stride(0), held.stride(1), held.size(1)};
}

void check_alike(const char* name, const Tensor& t, const Tensor& like) {
  TORCH_CHECK_VALUE(t.scalar_type() == like.scalar_type() && t.device() == like.device() && t.dim() == like.dim() &&
                        t.sizes().slice(0, t.dim() - 2) == like.sizes().slice(0, like.dim() - 2) &&
                        t.size(-1) == like.size(-1),
                    name, " must match the other rows in type, device, leading sizes and dim");
}

bool wants_grad(const Tensor& t) { return t.defined() && t.requires_grad(); }

bool wants_grad(const OptTensor& t) { return t && wants_grad(*t); }

// Forward mode: a tensor that carries a tangent (it need not require a gradient).
bool has_tangent(const Tensor& t) { return t.defined() && t._fw_grad(0).defined(); }
bool has_tangent(const OptTensor& t) { return t && has_tangent(*t); }

// What has no gradient is refused where one is asked for, rather than taken as a constant.
template <typename... Ts>
bool asks_grad(const Ts&... given) {
  return (at::GradMode::is_enabled() && (wants_grad(given) || ...)) || (has_tangent(given) || ...);
}

// A tensor was written in place: autograd refuses what it saved of it before
// (inference tensors keep no count).
void mark_written(const Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// ---- rotary positions ----

// q and k turned; either may be undefined. The arguments are checked.
std::pair<Tensor, Tensor> rotate(const Tensor& q, const Tensor& k, const Tensor& positions, const Tensor& cos,
                                 const Tensor& sin, bool interleaved, bool back) {
  const Tensor& first = q.defined() ? q : k;
  const c10::DeviceGuard guard(first.device());
  const Table table = table_of(cos, sin, first);
  Tensor q_out, k_out, q_held, k_held;
  jasperx_head_rows q_rows{}, k_rows{};
  if (q.defined()) q_out = at::empty(q.sizes(), q.options()), q_rows = rows_of(q, q_held);
  if (k.defined()) k_out = at::empty(k.sizes(), k.options()), k_rows = rows_of(k, k_held);
  const int64_t n = positions.numel();
  if (n)
    check(jasperx_rotary(&q_rows, &k_rows, type_of(first), n, first.size(-1), positions.data_ptr(),
                         (int32_t)positions.element_size(), table.cos, table.sin, table.rows, table.rot,
                         (interleaved ? JASPERX_ROTARY_INTERLEAVED : 0u) | (back ? JASPERX_ROTARY_INVERSE : 0u),
                         q.defined() ? q_out.data_ptr() : nullptr, k.defined() ? k_out.data_ptr() : nullptr,
                         current_stream(first.get_device())));
  return {q_out, k_out};
}

// Linear in q and k: the gradient is the rotation by the opposite angles,
// which is differentiated the same way.
struct Rotary : torch::autograd::Function<Rotary> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const OptTensor& q,
                                                const OptTensor& k, const Tensor& positions, const Tensor& cos,
                                                const Tensor& sin, bool interleaved, bool back) {
    ctx->save_for_backward({positions, cos, sin});
    ctx->saved_data["interleaved"] = interleaved;
    ctx->saved_data["back"] = back;
    ctx->saved_data["q"] = q.has_value();
    ctx->saved_data["k"] = k.has_value();
    ctx->set_materialize_grads(false);
    const auto [q_out, k_out] = rotate(q.value_or(Tensor()), k.value_or(Tensor()), positions, cos, sin, interleaved, back);
    torch::autograd::variable_list out;
    if (q) out.push_back(q_out);
    if (k) out.push_back(k_out);
    return out;
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    const bool has_q = ctx->saved_data["q"].toBool(), has_k = ctx->saved_data["k"].toBool();
    const size_t at_k = has_q ? 1 : 0;  // what was not given has no place among the inputs
    Tensor gq, gk;
    if (has_q && ctx->needs_input_grad(0)) gq = grads[0];
    if (has_k && ctx->needs_input_grad(at_k)) gk = grads[at_k];
    torch::autograd::variable_list out(7);
    if (!gq.defined() && !gk.defined()) return out;
    const auto saved = ctx->get_saved_variables();
    const bool interleaved = ctx->saved_data["interleaved"].toBool(), back = ctx->saved_data["back"].toBool();
    std::tie(out[0], out[1]) = turn(gq, gk, saved[0], saved[1], saved[2], interleaved, !back);
    return out;
  }

  // differentiable where something asks for it; the tangents are turned like the rows
  static std::pair<Tensor, Tensor> turn(const Tensor& q, const Tensor& k, const Tensor& positions, const Tensor& cos,
                                        const Tensor& sin, bool interleaved, bool back) {
    if (has_tangent(q) || has_tangent(k)) {
      const auto value = [](const Tensor& t) { return t.defined() ? t._fw_primal(0) : t; };
      const auto tangent = [](const Tensor& t) { return t.defined() ? t._fw_grad(0) : t; };
      const auto out = turn(value(q), value(k), positions, cos, sin, interleaved, back);
      const auto moved = turn(tangent(q), tangent(k), positions, cos, sin, interleaved, back);
      if (moved.first.defined()) out.first._set_fw_grad(moved.first, 0, false);
      if (moved.second.defined()) out.second._set_fw_grad(moved.second, 0, false);
      return out;
    }
    if (!at::GradMode::is_enabled() || !(wants_grad(q) || wants_grad(k)))
      return rotate(q, k, positions, cos, sin, interleaved, back);
    const auto given = [](const Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); };
    const auto out = Rotary::apply(given(q), given(k), positions, cos, sin, interleaved, back);
    return {q.defined() ? out[0] : Tensor(), k.defined() ? out[q.defined() ? 1 : 0] : Tensor()};
  }
};

py::tuple rotary(const Tensor& q, const OptTensor& k, const Tensor& positions, const OptTensor& cos,
                 const OptTensor& sin, bool interleaved) {
  TORCH_CHECK_VALUE(is_row_type(q), "q must be float16 or bfloat16, got ", q.dtype());
  TORCH_CHECK_VALUE(q.is_cuda(), "q must be a CUDA tensor");
  TORCH_CHECK_VALUE(q.dim() >= 2 && q.size(-1) % 2 == 0, "q must be [..., heads, dim] with an even dim");
  if (k) check_alike("k", *k, q);
  const Tensor at = indexes("positions", positions, q);
  TORCH_CHECK_VALUE(at.sizes() == q.sizes().slice(0, q.dim() - 2), "positions must be ",
                    q.sizes().slice(0, q.dim() - 2), ", got ", at.sizes());
  TORCH_CHECK_VALUE(cos && sin, "cos and sin are needed");
  TORCH_CHECK_VALUE(!asks_grad(cos, sin), "rotary has no gradient for cos and sin: detach them");
  TORCH_CHECK_VALUE(table_of(cos, sin, q).rot <= q.size(-1), "the tables rotate more values than a head has");
  const auto [q_out, k_out] = Rotary::turn(q, k ? *k : Tensor(), at, *cos, *sin, interleaved, false);
  return py::make_tuple(q_out, k ? py::cast(k_out) : py::none());
}

// ---- the cache ----

OptTensor append_tokens(const OptTensor& q, const Tensor& k, const Tensor& v, const OptTensor& positions,
                        const Tensor& slots, const OptTensor& cos, const OptTensor& sin, const Tensor& k_pages,
                        const Tensor& v_pages, bool interleaved, const OptTensor& k_scale, const OptTensor& v_scale) {
  const jasperx_kv_pages pages = pages_of(k_pages, v_pages, k_scale, v_scale, false);
  TORCH_CHECK_VALUE(is_row_type(k) && (pages.type == 2 || pages.type == type_of(k)),
                    "k must be float16 or bfloat16 and the pages of its type or float8_e4m3fn, got ", k.dtype(), " and ",
                    k_pages.dtype());
  TORCH_CHECK_VALUE(k.dim() == 3 && k.size(1) == pages.heads && k.size(2) == pages.dim && k.device() == k_pages.device(),
                    "k must be [n, ", pages.heads, ", ", pages.dim, "] on ", k_pages.device());
  check_alike("v", v, k);
  TORCH_CHECK_VALUE(v.size(1) == pages.heads, "v must be [n, ", pages.heads, ", ", pages.dim, "]");
  if (q) check_alike("q", *q, k);
  TORCH_CHECK_VALUE(!asks_grad(q, k, v, cos, sin, k_pages, v_pages, k_scale, v_scale),
                    "append_tokens has no gradient: use rotary, or detached tensors or torch.no_grad()");
  const int64_t n = k.size(0);
  Tensor rows = indexes("slots", slots, k), at;
  TORCH_CHECK_VALUE(rows.dim() == 1 && rows.size(0) == n, "slots must be [", n, "]");
  const Table table = table_of(cos, sin, k);
  TORCH_CHECK_VALUE(table.rot <= pages.dim, "the tables rotate more values than a head has");
  if (table.rot) {
    TORCH_CHECK_VALUE(positions, "positions are needed with cos and sin");
    at = indexes("positions", *positions, k);
    TORCH_CHECK_VALUE(at.dim() == 1 && at.size(0) == n, "positions must be [", n, "]");
    if (at.scalar_type() != rows.scalar_type()) at = at.to(at::kLong), rows = rows.to(at::kLong);
  }
  const c10::DeviceGuard guard(k.device());
  OptTensor out;
  Tensor q_held, k_held, v_held;
  jasperx_head_rows q_rows{};
  if (q) out = at::empty(q->sizes(), q->options()), q_rows = rows_of(*q, q_held);
  const jasperx_head_rows k_rows = rows_of(k, k_held), v_rows = rows_of(v, v_held);
  if (n) {
    check(jasperx_append_tokens(&q_rows, &k_rows, &v_rows, type_of(k), n, table.rot ? at.data_ptr() : nullptr,
                                rows.data_ptr(), (int32_t)rows.element_size(), table.cos, table.sin, table.rows,
                                table.rot, interleaved ? JASPERX_ROTARY_INTERLEAVED : 0u, &pages,
                                out ? out->data_ptr() : nullptr, current_stream(k.get_device())));
    mark_written(k_pages), mark_written(v_pages);
  }
  return out;
}

void copy_pages(const Tensor& k_pages, const Tensor& v_pages, const Tensor& src, const Tensor& dst,
                const OptTensor& tables) {
  const jasperx_kv_pages pages = pages_of(k_pages, v_pages, {}, {}, true);
  TORCH_CHECK_VALUE(!asks_grad(k_pages, v_pages), "copy_pages has no gradient: use detached tensors or torch.no_grad()");
  for (const Tensor* t : {&src, &dst})
    TORCH_CHECK_VALUE(t->scalar_type() == at::kInt && t->dim() == 1 && t->device() == k_pages.device() &&
                          t->is_contiguous(),
                      "src and dst must be contiguous 1D int32 tensors on ", k_pages.device());
  TORCH_CHECK_VALUE(src.size(0) == dst.size(0), "src and dst must have the same length");
  TORCH_CHECK_VALUE(!tables || (tables->scalar_type() == at::kInt && tables->is_contiguous() &&
                                tables->device() == k_pages.device()),
                    "tables must be a contiguous int32 tensor on ", k_pages.device());
  const c10::DeviceGuard guard(k_pages.device());
  if (src.size(0)) {
    check(jasperx_copy_pages(&pages, (const int32_t*)src.data_ptr(), (const int32_t*)dst.data_ptr(), src.size(0),
                             tables ? (int32_t*)tables->data_ptr() : nullptr, tables ? tables->numel() : 0,
                             current_stream(k_pages.get_device())));
    mark_written(k_pages), mark_written(v_pages);
    if (tables) mark_written(*tables);
  }
}

// ---- attention of one new token ----

// One call's queries, tables and outputs, checked and allocated.
struct Attention {
  jasperx_kv_pages pages;
  Tensor q, lens, out, lse, scratch;
  jasperx_head_rows rows;
  int64_t batch;
  double scale;

  Attention(const Tensor& q_in, const Tensor& k_pages, const Tensor& v_pages, const Tensor& tables,
            const Tensor& lens_in, std::optional<double> scale_in, const OptTensor& k_scale, const OptTensor& v_scale)
      : pages(pages_of(k_pages, v_pages, k_scale, v_scale, false)), q(q_in), lens(lens_in) {
    TORCH_CHECK_VALUE(is_row_type(q) && (pages.type == 2 || pages.type == type_of(q)),
                      "q must be float16 or bfloat16 and the pages of its type or float8_e4m3fn, got ", q.dtype(),
                      " and ", k_pages.dtype());
    const c10::Device device = k_pages.device();
    TORCH_CHECK_VALUE(q.dim() == 3 && q.size(2) == pages.dim && q.size(1) > 0 && pages.heads > 0 &&
                          q.size(1) % pages.heads == 0 && q.device() == device,
                      "q must be [batch, a multiple of ", pages.heads, " heads, ", pages.dim, "] on ", device);
    TORCH_CHECK_VALUE(!asks_grad(q, k_pages, v_pages, k_scale, v_scale),
                      "attention over the cache has no gradient: use detached tensors or torch.no_grad()");
    batch = q.size(0);
    TORCH_CHECK_VALUE(tables.scalar_type() == at::kInt && tables.dim() == 2 && tables.size(0) == batch &&
                          tables.device() == device && (tables.size(1) <= 1 || tables.stride(1) == 1),
                      "tables must be int32 [", batch, ", pages] with contiguous rows, on ", device);
    TORCH_CHECK_VALUE(lens.scalar_type() == at::kInt && lens.dim() == 1 && lens.size(0) == batch &&
                          lens.device() == device,
                      "lens must be int32 [", batch, "] on ", device);
    lens = lens.contiguous();
    if (q.stride(2) != 1 || q.stride(0) % 8 || q.stride(1) % 8 || (uintptr_t)q.data_ptr() % 16)
      q = q.clone(at::MemoryFormat::Contiguous);
    rows = {q.data_ptr(), q.stride(0), q.stride(1), q.size(1)};
    scale = scale_in ? *scale_in : 1.0 / std::sqrt((double)pages.dim);
  }

  int64_t allocate(bool return_lse, int64_t max_tokens, int64_t lists) {
    out = at::empty(q.sizes(), q.options());
    if (return_lse) lse = at::empty({batch, q.size(1)}, q.options().dtype(at::kFloat));
    int64_t size = 0;
    if (batch) {
      size = jasperx_attention_workspace(batch, q.size(1), &pages, max_tokens, lists);
      check(size);
      scratch = at::empty({size}, q.options().dtype(at::kByte));
    }
    return size;
  }

  float* lse_ptr() { return lse.defined() ? (float*)lse.data_ptr() : nullptr; }

  py::object result() {
    if (!lse.defined()) return py::cast(out);
    return py::make_tuple(out, lse);
  }
};

py::object decode_attention(const Tensor& q, const Tensor& k_pages, const Tensor& v_pages, const Tensor& tables,
                            const Tensor& lens, std::optional<double> scale, int64_t window, const OptTensor& k_scale,
                            const OptTensor& v_scale, std::optional<int64_t> max_len, bool return_lse) {
  Attention a(q, k_pages, v_pages, tables, lens, scale, k_scale, v_scale);
  TORCH_CHECK_VALUE(window >= 0 && (!max_len || *max_len >= 0), "window and max_len must be at least 0");
  const c10::DeviceGuard guard(k_pages.device());
  int64_t most = tables.size(1) * a.pages.page_size;
  if (max_len) most = std::min(most, *max_len);
  const int64_t size = a.allocate(return_lse, window ? std::min(window, most) : most, 0);
  if (a.batch)
    check(jasperx_decode_attention(&a.rows, type_of(a.q), a.batch, &a.pages, (const int32_t*)tables.data_ptr(),
                                   tables.stride(0), tables.size(1), (const int32_t*)a.lens.data_ptr(), most, a.scale,
                                   window, a.out.data_ptr(), a.lse_ptr(), a.scratch.data_ptr(), size,
                                   current_stream(k_pages.get_device())));
  return a.result();
}

py::object retrieved_attention(const Tensor& q, const Tensor& k_pages, const Tensor& v_pages, const Tensor& tables,
                               const Tensor& lens, const Tensor& ids, int64_t first, int64_t last,
                               std::optional<double> scale, const OptTensor& k_scale, const OptTensor& v_scale,
                               bool return_lse) {
  Attention a(q, k_pages, v_pages, tables, lens, scale, k_scale, v_scale);
  TORCH_CHECK_VALUE(ids.scalar_type() == at::kInt && ids.dim() == 3 && ids.size(0) == a.batch &&
                        (ids.size(1) == q.size(1) || ids.size(1) == a.pages.heads) && ids.device() == k_pages.device(),
                    "ids must be int32 [", a.batch, ", ", q.size(1), " or ", a.pages.heads, ", count] on ",
                    k_pages.device());
  const int64_t lists = ids.size(1), count = ids.size(2), most = INT64_C(1) << 30;
  TORCH_CHECK_VALUE(first >= 0 && last >= 0 && first < most && last < most && first + last + count < most,
                    "first, last and count must be at least 0, and below 2^30 in sum");
  const c10::DeviceGuard guard(k_pages.device());
  const Tensor held = ids.contiguous();
  const int64_t size = a.allocate(return_lse, first + last + count, lists);
  if (a.batch)
    check(jasperx_retrieved_attention(&a.rows, type_of(a.q), a.batch, &a.pages, (const int32_t*)tables.data_ptr(),
                                      tables.stride(0), tables.size(1), (const int32_t*)a.lens.data_ptr(),
                                      (const int32_t*)held.data_ptr(), lists, count, first, last, a.scale,
                                      a.out.data_ptr(), a.lse_ptr(), a.scratch.data_ptr(), size,
                                      current_stream(k_pages.get_device())));
  return a.result();
}

}  // namespace

PYBIND11_MODULE(_kv, m) {
  py::register_exception_translator([](std::exception_ptr e) {
    try {
      if (e) std::rethrow_exception(e);
    } catch (const Failure& f) {
      PyErr_SetString(py::module_::import("jasper_amd").attr("JasperError").ptr(), f.what());
    }
  });
  m.def("rotary", &rotary);
  m.def("append_tokens", &append_tokens);
  m.def("copy_pages", &copy_pages);
  m.def("decode_attention", &decode_attention);
  m.def("retrieved_attention", &retrieved_attention);
}
