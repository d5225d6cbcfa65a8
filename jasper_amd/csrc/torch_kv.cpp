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

// Positions of several axes: the pairs of each; none: one position for all.
struct Axes {
  std::vector<int32_t> sections;
  bool cyclic = false;
  int64_t count() const { return (int64_t)sections.size(); }
};

Axes axes_of(const std::optional<std::vector<int64_t>>& sections, bool cyclic, int64_t rot) {
  Axes a;
  a.cyclic = cyclic;
  if (!sections) {
    TORCH_CHECK_VALUE(!cyclic, "cyclic needs sections");
    return a;
  }
  TORCH_CHECK_VALUE(!sections->empty() && sections->size() <= 4, "sections must be of 1 to 4 axes, got ", sections->size());
  int64_t pairs = 0;
  for (const int64_t s : *sections) {
    TORCH_CHECK_VALUE(s >= 0 && s <= 1024, "a section must be of 0 to 1024 pairs, got ", s);
    a.sections.push_back((int32_t)s), pairs += s;
  }
  TORCH_CHECK_VALUE(2 * pairs == rot, "sections must be ", rot / 2, " pairs in sum (half of what the tables rotate), got ", pairs);
  return a;
}

// The sizes of positions for rows with these leading sizes.
std::vector<int64_t> position_sizes(const Axes& axes, at::IntArrayRef leading) {
  std::vector<int64_t> r;
  if (axes.count()) r.push_back(axes.count());
  r.insert(r.end(), leading.begin(), leading.end());
  return r;
}

// q and k turned; either may be undefined. The arguments are checked.
std::pair<Tensor, Tensor> rotate(const Tensor& q, const Tensor& k, const Tensor& positions, const Tensor& cos,
                                 const Tensor& sin, bool interleaved, bool back, const Axes& axes) {
  const Tensor& first = q.defined() ? q : k;
  const c10::DeviceGuard guard(first.device());
  const Table table = table_of(cos, sin, first);
  Tensor q_out, k_out, q_held, k_held;
  jasperx_head_rows q_rows{}, k_rows{};
  if (q.defined()) q_out = at::empty(q.sizes(), q.options()), q_rows = rows_of(q, q_held);
  if (k.defined()) k_out = at::empty(k.sizes(), k.options()), k_rows = rows_of(k, k_held);
  const int64_t n = positions.numel() / std::max<int64_t>(1, axes.count());
  if (n) {
    const uint32_t flags = (interleaved ? JASPERX_ROTARY_INTERLEAVED : 0u) | (back ? JASPERX_ROTARY_INVERSE : 0u);
    void* const q_to = q.defined() ? q_out.data_ptr() : nullptr;
    void* const k_to = k.defined() ? k_out.data_ptr() : nullptr;
    const int32_t type = type_of(first), bytes = (int32_t)positions.element_size();
    void* const stream = current_stream(first.get_device());
    if (axes.count())
      check(jasperx_rotary_by_axes(&q_rows, &k_rows, type, n, first.size(-1), positions.data_ptr(), bytes,
                                   axes.sections.data(), (int32_t)axes.count(), axes.cyclic, table.cos, table.sin,
                                   table.rows, table.rot, flags, q_to, k_to, stream));
    else
      check(jasperx_rotary(&q_rows, &k_rows, type, n, first.size(-1), positions.data_ptr(), bytes, table.cos, table.sin,
                           table.rows, table.rot, flags, q_to, k_to, stream));
  }
  return {q_out, k_out};
}

// Linear in q and k: the gradient is the rotation by the opposite angles,
// which is differentiated the same way.
struct Rotary : torch::autograd::Function<Rotary> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const OptTensor& q,
                                                const OptTensor& k, const Tensor& positions, const Tensor& cos,
                                                const Tensor& sin, bool interleaved, bool back, Axes axes) {
    ctx->save_for_backward({positions, cos, sin});
    ctx->saved_data["interleaved"] = interleaved;
    ctx->saved_data["back"] = back;
    ctx->saved_data["q"] = q.has_value();
    ctx->saved_data["k"] = k.has_value();
    if (axes.count()) {
      ctx->saved_data["sections"] = std::vector<int64_t>(axes.sections.begin(), axes.sections.end());
      ctx->saved_data["cyclic"] = axes.cyclic;
    }
    ctx->set_materialize_grads(false);
    const auto [q_out, k_out] = rotate(q.value_or(Tensor()), k.value_or(Tensor()), positions, cos, sin, interleaved, back, axes);
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
    torch::autograd::variable_list out(8);
    if (!gq.defined() && !gk.defined()) return out;
    const auto saved = ctx->get_saved_variables();
    const bool interleaved = ctx->saved_data["interleaved"].toBool(), back = ctx->saved_data["back"].toBool();
    Axes axes;
    const auto sections = ctx->saved_data.find("sections");
    if (sections != ctx->saved_data.end()) {
      for (const int64_t s : sections->second.toIntVector()) axes.sections.push_back((int32_t)s);
      axes.cyclic = ctx->saved_data["cyclic"].toBool();
    }
    std::tie(out[0], out[1]) = turn(gq, gk, saved[0], saved[1], saved[2], interleaved, !back, axes);
    return out;
  }

  // differentiable where something asks for it; the tangents are turned like the rows
  static std::pair<Tensor, Tensor> turn(const Tensor& q, const Tensor& k, const Tensor& positions, const Tensor& cos,
                                        const Tensor& sin, bool interleaved, bool back, const Axes& axes) {
    if (has_tangent(q) || has_tangent(k)) {
      const auto value = [](const Tensor& t) { return t.defined() ? t._fw_primal(0) : t; };
      const auto tangent = [](const Tensor& t) { return t.defined() ? t._fw_grad(0) : t; };
      const auto out = turn(value(q), value(k), positions, cos, sin, interleaved, back, axes);
      const auto moved = turn(tangent(q), tangent(k), positions, cos, sin, interleaved, back, axes);
      if (moved.first.defined()) out.first._set_fw_grad(moved.first, 0, false);
      if (moved.second.defined()) out.second._set_fw_grad(moved.second, 0, false);
      return out;
    }
    if (!at::GradMode::is_enabled() || !(wants_grad(q) || wants_grad(k)))
      return rotate(q, k, positions, cos, sin, interleaved, back, axes);
    const auto given = [](const Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); };
    const auto out = Rotary::apply(given(q), given(k), positions, cos, sin, interleaved, back, axes);
    return {q.defined() ? out[0] : Tensor(), k.defined() ? out[q.defined() ? 1 : 0] : Tensor()};
  }
};

py::tuple rotary(const Tensor& q, const OptTensor& k, const Tensor& positions, const OptTensor& cos,
                 const OptTensor& sin, bool interleaved, const std::optional<std::vector<int64_t>>& sections, bool cyclic) {
  TORCH_CHECK_VALUE(is_row_type(q), "q must be float16 or bfloat16, got ", q.dtype());
  TORCH_CHECK_VALUE(q.is_cuda(), "q must be a CUDA tensor");
  TORCH_CHECK_VALUE(q.dim() >= 2 && q.size(-1) % 2 == 0, "q must be [..., heads, dim] with an even dim");
  if (k) check_alike("k", *k, q);
  const Tensor at = indexes("positions", positions, q);
  TORCH_CHECK_VALUE(cos && sin, "cos and sin are needed");
  TORCH_CHECK_VALUE(!asks_grad(cos, sin), "rotary has no gradient for cos and sin: detach them");
  const int64_t rot = table_of(cos, sin, q).rot;
  TORCH_CHECK_VALUE(rot <= q.size(-1), "the tables rotate more values than a head has");
  const Axes axes = axes_of(sections, cyclic, rot);
  const auto sizes = position_sizes(axes, q.sizes().slice(0, q.dim() - 2));
  TORCH_CHECK_VALUE(at.sizes() == at::IntArrayRef(sizes), "positions must be ", at::IntArrayRef(sizes), ", got ", at.sizes());
  const auto [q_out, k_out] = Rotary::turn(q, k ? *k : Tensor(), at, *cos, *sin, interleaved, false, axes);
  return py::make_tuple(q_out, k ? py::cast(k_out) : py::none());
}

// ---- the cache ----

OptTensor append_tokens(const OptTensor& q, const Tensor& k, const Tensor& v, const OptTensor& positions,
                        const Tensor& slots, const OptTensor& cos, const OptTensor& sin, const Tensor& k_pages,
                        const Tensor& v_pages, bool interleaved, const OptTensor& k_scale, const OptTensor& v_scale,
                        const std::optional<std::vector<int64_t>>& sections, bool cyclic) {
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
  const Axes axes = axes_of(sections, cyclic, table.rot);
  if (table.rot) {
    TORCH_CHECK_VALUE(positions, "positions are needed with cos and sin");
    at = indexes("positions", *positions, k);
    const auto sizes = position_sizes(axes, {n});
    TORCH_CHECK_VALUE(at.sizes() == at::IntArrayRef(sizes), "positions must be ", at::IntArrayRef(sizes), ", got ", at.sizes());
    if (at.scalar_type() != rows.scalar_type()) at = at.to(at::kLong), rows = rows.to(at::kLong);
  }
  const c10::DeviceGuard guard(k.device());
  OptTensor out;
  Tensor q_held, k_held, v_held;
  jasperx_head_rows q_rows{};
  if (q) out = at::empty(q->sizes(), q->options()), q_rows = rows_of(*q, q_held);
  const jasperx_head_rows k_rows = rows_of(k, k_held), v_rows = rows_of(v, v_held);
  if (n) {
    const void* const at_ptr = table.rot ? at.data_ptr() : nullptr;
    const uint32_t flags = interleaved ? JASPERX_ROTARY_INTERLEAVED : 0u;
    const int32_t bytes = (int32_t)rows.element_size();
    void* const q_to = out ? out->data_ptr() : nullptr;
    void* const stream = current_stream(k.get_device());
    if (axes.count())
      check(jasperx_append_tokens_by_axes(&q_rows, &k_rows, &v_rows, type_of(k), n, at_ptr, rows.data_ptr(), bytes,
                                          axes.sections.data(), (int32_t)axes.count(), axes.cyclic, table.cos, table.sin,
                                          table.rows, table.rot, flags, &pages, q_to, stream));
    else
      check(jasperx_append_tokens(&q_rows, &k_rows, &v_rows, type_of(k), n, at_ptr, rows.data_ptr(), bytes, table.cos,
                                  table.sin, table.rows, table.rot, flags, &pages, q_to, stream));
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

// ---- page tables on the GPU ----

void check_ints(const char* name, const Tensor& t, int64_t dims, c10::Device device) {
  TORCH_CHECK_VALUE(t.scalar_type() == at::kInt && t.dim() == dims && t.is_contiguous() && t.device() == device, name,
                    " must be a contiguous ", dims, "D int32 tensor on ", device);
}

struct PageTable {
  jasperx_page_table table{};
  c10::Device device;

  PageTable(const Tensor& tables, const Tensor& lens, const Tensor& refs, const Tensor& free, int64_t page_size)
      : device(tables.device()) {
    TORCH_CHECK_VALUE(tables.is_cuda(), "tables must be a CUDA tensor");
    check_ints("tables", tables, 2, device), check_ints("lens", lens, 1, device);
    check_ints("refs", refs, 1, device), check_ints("free", free, 1, device);
    for (const Tensor* t : {&tables, &lens, &refs, &free})
      for (const int64_t size : t->sizes()) TORCH_CHECK_VALUE(size <= INT32_MAX, "the page table is too large");
    TORCH_CHECK_VALUE(lens.size(0) == tables.size(0), "lens must be [", tables.size(0), "], a length for each table");
    TORCH_CHECK_VALUE(free.size(0) == (refs.size(0) + 31) / 32, "free must be [", (refs.size(0) + 31) / 32,
                      "], a bit for each of ", refs.size(0), " pages");
    TORCH_CHECK_VALUE(page_size > 0 && page_size <= 256, "page_size must be a power of two from 8 to 256, got ", page_size);
    table.tables = (int32_t*)tables.data_ptr(), table.lens = (int32_t*)lens.data_ptr();
    table.refs = (int32_t*)refs.data_ptr(), table.free_bits = (uint32_t*)free.data_ptr();
    table.sequences = (int32_t)tables.size(0), table.width = (int32_t)tables.size(1);
    table.pages = (int32_t)refs.size(0), table.page_size = (int32_t)page_size;
  }

  void pair(const char* name_a, const Tensor& a, const char* name_b, const Tensor& b) const {
    check_ints(name_a, a, 1, device), check_ints(name_b, b, 1, device);
    TORCH_CHECK_VALUE(a.size(0) == b.size(0), name_a, " and ", name_b, " must have the same length");
  }
};

py::tuple extend_tables(const Tensor& tables, const Tensor& lens, const Tensor& refs, const Tensor& free,
                        const Tensor& seqs, const Tensor& counts, int64_t page_size, int64_t n_tokens,
                        std::optional<int64_t> width) {
  const PageTable t(tables, lens, refs, free, page_size);
  t.pair("seqs", seqs, "counts", counts);
  const int64_t wide = width.value_or(tables.size(1)), n = seqs.size(0);
  TORCH_CHECK_VALUE(n_tokens >= 0 && wide >= 0 && n_tokens <= INT32_MAX && wide <= INT32_MAX,
                    "n_tokens and width must be at least 0 and below 2^31");
  const c10::DeviceGuard guard(t.device);
  const auto longs = tables.options().dtype(at::kLong);
  const Tensor positions = at::empty({n_tokens}, longs), slots = at::empty({n_tokens}, longs);
  const Tensor starts = at::empty({n + 1}, tables.options()), step = at::empty({n, wide}, tables.options());
  const Tensor step_lens = at::empty({n}, tables.options()), src = at::empty({n}, tables.options());
  const Tensor dst = at::empty({n}, tables.options()), missing = at::empty({1}, tables.options());
  const int64_t size = jasperx_extend_workspace(n, refs.size(0));
  check(size);
  const Tensor scratch = at::empty({std::max<int64_t>(size, 16)}, tables.options().dtype(at::kByte));
  const auto ints = [](const Tensor& x) { return (int32_t*)x.data_ptr(); };
  check(jasperx_extend_tables(&t.table, ints(seqs), ints(counts), n, n_tokens, wide, (int64_t*)positions.data_ptr(),
                              (int64_t*)slots.data_ptr(), ints(starts), ints(step), ints(step_lens), ints(src), ints(dst),
                              ints(missing), scratch.data_ptr(), size, current_stream(tables.get_device())));
  for (const Tensor* x : {&tables, &lens, &refs, &free}) mark_written(*x);
  return py::make_tuple(positions, slots, starts, step, step_lens, src, dst, missing);
}

void truncate_tables(const Tensor& tables, const Tensor& lens, const Tensor& refs, const Tensor& free,
                     const Tensor& seqs, const Tensor& to, int64_t page_size) {
  const PageTable t(tables, lens, refs, free, page_size);
  t.pair("seqs", seqs, "to", to);
  const c10::DeviceGuard guard(t.device);
  check(jasperx_truncate_tables(&t.table, (const int32_t*)seqs.data_ptr(), (const int32_t*)to.data_ptr(), seqs.size(0),
                                current_stream(tables.get_device())));
  for (const Tensor* x : {&tables, &lens, &refs, &free}) mark_written(*x);
}

void fork_tables(const Tensor& tables, const Tensor& lens, const Tensor& refs, const Tensor& free, const Tensor& seqs,
                 const Tensor& into, int64_t page_size) {
  const PageTable t(tables, lens, refs, free, page_size);
  t.pair("seqs", seqs, "into", into);
  const c10::DeviceGuard guard(t.device);
  check(jasperx_fork_tables(&t.table, (const int32_t*)seqs.data_ptr(), (const int32_t*)into.data_ptr(), seqs.size(0),
                            current_stream(tables.get_device())));
  for (const Tensor* x : {&tables, &lens, &refs}) mark_written(*x);
}

py::tuple shared_prefixes(const Tensor& tables, const Tensor& lens, int64_t page_size, int64_t least) {
  TORCH_CHECK_VALUE(tables.is_cuda() && tables.scalar_type() == at::kInt && tables.dim() == 2 &&
                        (tables.size(1) <= 1 || tables.stride(1) == 1),
                    "tables must be a CUDA int32 [batch, pages] tensor with contiguous rows");
  TORCH_CHECK_VALUE(lens.scalar_type() == at::kInt && lens.dim() == 1 && lens.size(0) == tables.size(0) &&
                        lens.device() == tables.device(),
                    "lens must be int32 [", tables.size(0), "] on ", tables.device());
  const c10::DeviceGuard guard(tables.device());
  const int64_t n = tables.size(0);
  const Tensor held = lens.contiguous();
  const Tensor groups = at::empty({n + 1}, held.options()), shared = at::empty({n}, held.options());
  const int64_t size = jasperx_prefixes_workspace(n);
  check(size);
  const Tensor scratch = at::empty({size}, held.options().dtype(at::kByte));
  check(jasperx_shared_prefixes((const int32_t*)tables.data_ptr(), tables.stride(0), tables.size(1),
                                (const int32_t*)held.data_ptr(), n, page_size, least, (int32_t*)groups.data_ptr(),
                                (int32_t*)shared.data_ptr(), scratch.data_ptr(), size, current_stream(tables.get_device())));
  return py::make_tuple(groups, shared);
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

  void allocate_outputs(bool return_lse) {
    out = at::empty(q.sizes(), q.options());
    if (return_lse) lse = at::empty({batch, q.size(1)}, q.options().dtype(at::kFloat));
  }

  int64_t allocate(bool return_lse, int64_t max_tokens, int64_t lists) {
    allocate_outputs(return_lse);
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

py::object shared_attention(const Tensor& q, const Tensor& k_pages, const Tensor& v_pages, const Tensor& tables,
                            const Tensor& lens, const Tensor& groups, const Tensor& shared, std::optional<double> scale,
                            const OptTensor& k_scale, const OptTensor& v_scale, std::optional<int64_t> max_len,
                            bool return_lse) {
  Attention a(q, k_pages, v_pages, tables, lens, scale, k_scale, v_scale);
  TORCH_CHECK_VALUE(!max_len || *max_len >= 0, "max_len must be at least 0");
  check_ints("groups", groups, 1, k_pages.device()), check_ints("shared", shared, 1, k_pages.device());
  const int64_t n = shared.size(0);
  TORCH_CHECK_VALUE(groups.size(0) == n + 1 && n <= a.batch, "groups must be [n_groups + 1] and shared [n_groups], of at most ",
                    a.batch, " groups, got ", groups.size(0), " and ", n);
  const c10::DeviceGuard guard(k_pages.device());
  int64_t most = tables.size(1) * a.pages.page_size;
  if (max_len) most = std::min(most, *max_len);
  a.allocate_outputs(return_lse);
  if (a.batch) {
    const int64_t size = jasperx_shared_workspace(a.batch, q.size(1), &a.pages, most, n);
    check(size);
    a.scratch = at::empty({size}, a.q.options().dtype(at::kByte));
    check(jasperx_shared_attention(&a.rows, type_of(a.q), a.batch, &a.pages, (const int32_t*)tables.data_ptr(),
                                   tables.stride(0), tables.size(1), (const int32_t*)a.lens.data_ptr(), most,
                                   (const int32_t*)groups.data_ptr(), (const int32_t*)shared.data_ptr(), n, a.scale,
                                   a.out.data_ptr(), a.lse_ptr(), a.scratch.data_ptr(), size,
                                   current_stream(k_pages.get_device())));
  }
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
  m.def("extend_tables", &extend_tables);
  m.def("truncate_tables", &truncate_tables);
  m.def("fork_tables", &fork_tables);
  m.def("shared_prefixes", &shared_prefixes);
  m.def("decode_attention", &decode_attention);
  m.def("retrieved_attention", &retrieved_attention);
  m.def("shared_attention", &shared_attention);
}
