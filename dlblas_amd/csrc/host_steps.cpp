// The steps around the products of a decoder block as native calls, under the same rules as host_calls.cpp: a function does the
// whole call or returns None without a trace, and the Python function then takes its own path.  Where a gradient is wanted the call
// becomes a node of the graph here too: through Python's autograd.Function and custom ops a forward and backward pass of a norm took 200
// us of host time, more than the kernels of 1237 x 2050 rows several times over.
#include "host_tensors.h"

#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>

#include <optional>

namespace {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

struct StepAbi {
  decltype(&dlb_last_error) last_error;
  decltype(&dlb_rms_norm_backward_workspace_bytes) norm_backward_ws;
  decltype(&dlb_rms_norm_backward) norm_backward;
  decltype(&dlb_moe_unpermute_backward) unpermute_backward;
  decltype(&dlb_rms_norm) norm;
  decltype(&dlb_rms_norm_quant) norm_quant;
  decltype(&dlb_moe_permute_workspace_bytes) permute_ws;
  decltype(&dlb_moe_permute) permute;
  decltype(&dlb_moe_unpermute) unpermute;
  decltype(&dlb_w4_gemm_workspace_bytes) w4_ws;
  decltype(&dlb_w4_gemm) w4;
} abi;

constexpr int64_t kMaxTopk = 64, kMaxExperts = DLB_SORT_MAX_EXPERTS;

// The tensors of a call, None (nullptr) where `optional` allows it; all plain and on the device of the first.  *grad: plain().
template <size_t N>
bool take(PyObject* const* args, const at::Tensor* (&out)[N], uint64_t optional, bool* grad = nullptr) {
  if (!no_modes()) return false;
  for (size_t i = 0; i < N; ++i) {
    out[i] = nullptr;
    if (args[i] == Py_None && (optional >> i & 1)) continue;
    out[i] = plain(args[i], grad);
    if (!out[i] || out[i]->get_device() != out[0]->get_device()) return false;
  }
  return true;
}

bool integer(PyObject* o, int64_t* v) {
  if (!PyLong_CheckExact(o)) return false;
  *v = PyLong_AsLongLong(o);
  if (!PyErr_Occurred()) return true;
  PyErr_Clear();
  return false;
}

void* optr(const at::Tensor* t) { return t ? ptr(*t) : nullptr; }

// [rows, H] of contiguous columns without a copy: the row stride, or -1.
int64_t row_stride(const at::Tensor& t) {
  if (t.dim() == 2 && t.stride(1) == 1) return t.stride(0);
  return t.is_contiguous() ? t.size(-1) : -1;
}

bool norm_operands(const at::Tensor& x, const at::Tensor& w, const at::Tensor* res) {
  if (in_code(x.scalar_type()) < 0 || x.dim() < 1 || x.numel() == 0 || x.size(-1) > DLB_NORM_MAX_COLUMNS || row_stride(x) < 0) return false;
  if ((w.scalar_type() != x.scalar_type() && !is_f32(w)) || w.dim() != 1 || w.size(0) != x.size(-1) || !w.is_contiguous()) return false;
  return !res || (res->scalar_type() == x.scalar_type() && res->sizes() == x.sizes() && row_stride(*res) >= 0);
}

bool index_of_rows(const at::Tensor& t, int64_t n) { return t.scalar_type() == at::kInt && t.dim() == 1 && t.size(0) == n && t.is_contiguous(); }

PyObject* tuple_of(std::initializer_list<at::Tensor*> tensors) {
  PyObject* out = PyTuple_New(static_cast<Py_ssize_t>(tensors.size()));
  if (!out) return nullptr;
  Py_ssize_t i = 0;
  for (at::Tensor* t : tensors) {
    PyObject* item = nullptr;
    if (t->defined()) {
      item = THPVariable_Wrap(std::move(*t));
    } else {
      item = Py_None;
      Py_INCREF(item);
    }
    if (!item) {
      Py_DECREF(out);
      return nullptr;
    }
    PyTuple_SET_ITEM(out, i++, item);
  }
  return out;
}

// ---- graph nodes ------------------------------------------------------------------------------------------------------

struct Failed : std::runtime_error {
  using std::runtime_error::runtime_error;
};
// A refused call enqueues nothing: an entry point leaves it to the Python path and its messages (DECLINE_FAILED), a node of the graph
// raises.
void must(int rc) {
  if (rc != DLB_OK) throw Failed(std::string("dlblas fp8_gemm error ") + std::to_string(rc) + ": " + abi.last_error());
}

// Gradients that cannot be differentiated again: in a graph of a graph they raise when somebody does.
variable_list once(variable_list grads) {
  if (!c10::GradMode::is_enabled()) return grads;
  variable_list through;
  for (at::Tensor& g : grads)
    if (g.defined()) through.push_back(g.detach().requires_grad_(true));
  const auto error = std::make_shared<torch::autograd::DelayedError>("a gradient of dlblas_amd was differentiated again, which is not implemented",
                                                                     static_cast<int64_t>(through.size()));
  through = (*error)(std::move(through));
  size_t i = 0;
  for (at::Tensor& g : grads)
    if (g.defined()) g = through[i++];
  return grads;
}

// Nor in forward mode: the kernels write into outputs that no tangent follows.
void no_tangent(const at::Tensor& grad) {
  TORCH_CHECK_NOT_IMPLEMENTED(!grad.defined() || !grad._fw_grad(0).defined(),
                              "forward-mode derivatives of the steps around the products are not implemented");
}

// A saved tensor as a hook on saved tensors gave it back.  Its layout may be another one; the kernels are told nothing but its address, so
// its device, type and sizes may not.
const at::Tensor& given_back(const at::Tensor& t, at::ScalarType type, at::IntArrayRef size, const at::Tensor& grad) {
  TORCH_CHECK(t.defined() && t.device() == grad.device() && t.scalar_type() == type && t.sizes() == size,
              "a tensor saved for a gradient of dlblas_amd came back from its hook on another device, of another type or with other sizes");
  return t;
}

at::Tensor whole_columns(const at::Tensor& t) { return row_stride(t) < 0 ? t.contiguous() : t; }
std::optional<at::Tensor> optional_of(const at::Tensor* t) { return t ? std::optional<at::Tensor>(*t) : std::nullopt; }

// {y} or {y, h}
variable_list norm_forward(const at::Tensor& x, const at::Tensor& w, const at::Tensor* res, double eps) {
  const int64_t H = x.size(-1), rows = x.numel() / H;
  at::Tensor y = empty(x.sizes(), x.scalar_type(), x), sum;
  if (res) sum = empty(x.sizes(), x.scalar_type(), x);
  must(abi.norm(ptr(x), row_stride(x), optr(res), res ? row_stride(*res) : 0, in_code(x.scalar_type()), ptr(w), in_code(w.scalar_type()), ptr(y), H,
                res ? ptr(sum) : nullptr, H, rows, H, static_cast<float>(eps), stream_of(x)));
  return res ? variable_list{y, sum} : variable_list{y};
}

struct RmsNorm : torch::autograd::Function<RmsNorm> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& w, const std::optional<at::Tensor>& res, double eps) {
    variable_list out = norm_forward(x, w, res ? &*res : nullptr, eps);
    ctx->set_materialize_grads(false);
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["res"] = res.has_value();
    ctx->save_for_backward({res ? out[1] : x, w});
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    const bool with_res = ctx->saved_data["res"].toBool();
    const at::Tensor dsum_given = with_res ? grads[1] : at::Tensor();
    no_tangent(grads[0]), no_tangent(dsum_given);
    if (!grads[0].defined()) return once({dsum_given, {}, with_res ? dsum_given : at::Tensor(), {}});  // only the sum went on, or nothing
    const at::Tensor& g = grads[0];
    DeviceScope scope(g);
    const int64_t H = g.size(-1), rows = g.numel() / H;
    const at::Tensor h = whole_columns(given_back(saved[0], g.scalar_type(), g.sizes(), g));
    const at::Tensor w = given_back(saved[1], is_f32(saved[1]) ? at::kFloat : g.scalar_type(), {H}, g).contiguous();
    const at::Tensor dy = whole_columns(g), dsum = dsum_given.defined() ? whole_columns(dsum_given) : dsum_given;
    at::Tensor dx = empty(h.sizes(), h.scalar_type(), h), dw, shares;
    size_t need = 0;
    if (ctx->needs_input_grad(1)) {
      dw = empty(w.sizes(), w.scalar_type(), w);
      need = abi.norm_backward_ws(rows, H);
      shares = empty({static_cast<int64_t>(need)}, at::kByte, h);
    }
    must(abi.norm_backward(ptr(dy), row_stride(dy), dsum.defined() ? ptr(dsum) : nullptr, dsum.defined() ? row_stride(dsum) : 0, ptr(h), row_stride(h),
                           in_code(h.scalar_type()), ptr(w), in_code(w.scalar_type()), ptr(dx), H, dw.defined() ? ptr(dw) : nullptr, rows, H,
                           static_cast<float>(ctx->saved_data["eps"].toDouble()), need > 0 ? ptr(shares) : nullptr, need, stream_of(h)));
    return once({dx, dw, with_res ? dx : at::Tensor(), {}});
  }
};

// A view of `size` ints from the offset-th on, without a trip through the dispatcher.
at::Tensor part_of(const at::Tensor& base, int64_t* offset, at::IntArrayRef size) {
  at::Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(base.storage()), base.key_set(), base.dtype());
  t.unsafeGetTensorImpl()->set_storage_offset(*offset);
  t.unsafeGetTensorImpl()->set_sizes_contiguous(size);
  *offset += t.numel();
  return t;
}

// {rows, row_index, source, m_indices, row_start, row_end}, behind them the rows' scales
variable_list permute_forward(const at::Tensor& x, const at::Tensor* x_s, const at::Tensor& ids, int64_t E, int64_t align, int64_t R) {
  const int64_t T = x.size(0), H = x.size(1), topk = ids.size(1);
  const hipStream_t stream = stream_of(x);
  at::Tensor rows = empty({R, H}, x.scalar_type(), x), rows_s, scratch;
  if (x_s) rows_s = empty({R, H / kBlock}, at::kFloat, x);
  const at::Tensor tables = empty({T * topk + 2 * R + 2 * E}, at::kInt, x);
  int64_t at = 0;
  variable_list out{rows, part_of(tables, &at, {T, topk}), part_of(tables, &at, {R}), part_of(tables, &at, {R}), part_of(tables, &at, {E}), part_of(tables, &at, {E})};
  const size_t need = abi.permute_ws(T, topk, E);
  if (need > 0) scratch = empty({static_cast<int64_t>(need)}, at::kByte, x);
  must(abi.permute(ptr(ids), idx_code(ids.scalar_type()), ids.stride(0), ids.stride(1), ptr(x), x.stride(0), x_s ? DLB_ROWS_E4M3 : in_code(x.scalar_type()),
                   x_s ? fptr(*x_s) : nullptr, x_s ? x_s->stride(0) : 0, x_s ? x_s->stride(1) : 0, iptr(out[1]), iptr(out[2]), iptr(out[3]), iptr(out[4]),
                   iptr(out[5]), ptr(rows), x_s ? fptr(rows_s) : nullptr, T, H, topk, E, align, R, need > 0 ? ptr(scratch) : nullptr, need, stream));
  if (x_s) out.push_back(rows_s);
  return out;
}

at::Tensor unpermute_forward(const at::Tensor& rows, const at::Tensor& index, const at::Tensor* w) {
  const int64_t T = index.size(0), H = rows.size(1);
  at::Tensor out = empty({T, H}, rows.scalar_type(), rows);
  must(abi.unpermute(ptr(rows), rows.stride(0), in_code(rows.scalar_type()), iptr(index), w ? fptr(*w) : nullptr, ptr(out), H, T, H, index.size(1), rows.size(0),
                     stream_of(rows)));
  return out;
}

struct Permute : torch::autograd::Function<Permute> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& ids, int64_t E, int64_t align, int64_t R) {
    variable_list out = permute_forward(x, nullptr, ids, E, align, R);
    ctx->save_for_backward({out[1]});
    ctx->saved_data["topk"] = ids.size(1);
    ctx->saved_data["tokens"] = ids.size(0);
    ctx->mark_non_differentiable({out.begin() + 1, out.end()});
    ctx->set_materialize_grads(false);
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    if (!grads[0].defined()) return {{}, {}, {}, {}, {}};
    no_tangent(grads[0]);
    const variable_list saved = ctx->get_saved_variables();
    DeviceScope scope(grads[0]);
    const at::Tensor index = given_back(saved[0], at::kInt, {ctx->saved_data["tokens"].toInt(), ctx->saved_data["topk"].toInt()}, grads[0]).contiguous();
    return once({unpermute_forward(whole_columns(grads[0]), index, nullptr), {}, {}, {}, {}});
  }
};

struct Unpermute : torch::autograd::Function<Unpermute> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& rows, const std::optional<at::Tensor>& w, const at::Tensor& index, const at::Tensor& source) {
    ctx->saved_data["rows"] = rows.size(0);
    ctx->saved_data["topk"] = index.size(1);
    // the rows themselves are needed for the gradient of the weights alone
    ctx->save_for_backward({w && w->requires_grad() ? rows : at::Tensor(), w ? *w : at::Tensor(), index, source});
    ctx->set_materialize_grads(false);
    return unpermute_forward(rows, index, w ? &*w : nullptr);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    if (!grads[0].defined()) return {{}, {}, {}, {}};
    no_tangent(grads[0]);
    const variable_list saved = ctx->get_saved_variables();
    DeviceScope scope(grads[0]);
    const at::Tensor dout = whole_columns(grads[0]);
    const int64_t R = ctx->saved_data["rows"].toInt(), topk = ctx->saved_data["topk"].toInt(), T = dout.size(0), H = dout.size(1);
    const bool want_w = saved[1].defined() && saved[0].defined() && ctx->needs_input_grad(1);
    const at::Tensor rows = want_w ? whole_columns(given_back(saved[0], dout.scalar_type(), {R, H}, dout)) : at::Tensor();
    const at::Tensor w = saved[1].defined() ? given_back(saved[1], at::kFloat, {T, topk}, dout).contiguous() : at::Tensor();
    const at::Tensor index = given_back(saved[2], at::kInt, {T, topk}, dout).contiguous(), source = given_back(saved[3], at::kInt, {R}, dout).contiguous();
    at::Tensor drows = empty({R, H}, dout.scalar_type(), dout), dw;
    if (want_w) dw = empty(w.sizes(), at::kFloat, dout);
    must(abi.unpermute_backward(ptr(dout), row_stride(dout), want_w ? ptr(rows) : nullptr, want_w ? rows.stride(0) : 0, in_code(dout.scalar_type()), iptr(index),
                                iptr(source), w.defined() ? fptr(w) : nullptr, ptr(drows), H, want_w ? fptr(dw) : nullptr, T, H, topk, R, stream_of(dout)));
    return once({drows, dw, {}, {}});
  }
};

#define DECLINE_FAILED       \
  }                          \
  catch (const Failed&) {    \
    NOT_PLAIN;

// ---- the entry points -------------------------------------------------------------------------------------------------

// rms_norm(x, weight, eps, residual) -> y, or (y, h)
PyObject* rms_norm(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_EXCEPTIONS_BEGIN
  if (n != 4 || !PyFloat_CheckExact(args[2])) NOT_PLAIN;
  PyObject* const given[] = {args[0], args[1], args[3]};
  const at::Tensor* t[3];
  bool grad = false;
  if (!take(given, t, 4, &grad)) NOT_PLAIN;
  const at::Tensor &x = *t[0], &w = *t[1];
  const at::Tensor* res = t[2];
  const double eps = PyFloat_AS_DOUBLE(args[2]);
  if (!norm_operands(x, w, res) || !(eps >= 0)) NOT_PLAIN;
  const OpRecord record("dlblas::rms_norm", t);
  DeviceScope scope(x);
  variable_list out;
  {
    const NoGil nogil;
    out = grad ? RmsNorm::apply(x, w, optional_of(res), eps) : norm_forward(x, w, res, eps);
  }
  return res ? tuple_of({&out[0], &out[1]}) : THPVariable_Wrap(std::move(out[0]));
  DECLINE_FAILED
  HANDLE_EXCEPTIONS_END
}

// rms_norm_quant(x, weight, eps, residual, group_size, quant_eps, column_major_scales) -> (q, s), or (q, s, h)
PyObject* rms_norm_quant(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_EXCEPTIONS_BEGIN
  int64_t group;
  if (n != 7 || !PyFloat_CheckExact(args[2]) || !integer(args[4], &group) || !PyFloat_CheckExact(args[5]) || !PyBool_Check(args[6])) NOT_PLAIN;
  PyObject* const given[] = {args[0], args[1], args[3]};
  const at::Tensor* t[3];
  if (!take(given, t, 4)) NOT_PLAIN;
  const at::Tensor &x = *t[0], &w = *t[1];
  const at::Tensor* res = t[2];
  const double eps = PyFloat_AS_DOUBLE(args[2]), quant_eps = PyFloat_AS_DOUBLE(args[5]);
  if (!norm_operands(x, w, res) || !(eps >= 0) || group != kBlock || x.size(-1) % kBlock != 0) NOT_PLAIN;
  const OpRecord record("dlblas::rms_norm_quant", t);
  const int64_t H = x.size(-1), rows = x.numel() / H, groups = H / kBlock;
  const bool col_major = args[6] == Py_True;
  DeviceScope scope(x);
  at::Tensor q, s, sum;
  at::DimVector size(x.sizes());
  size.back() = groups;
  int rc;
  {
    const NoGil nogil;
    q = empty(x.sizes(), at::kFloat8_e4m3fn, x);
    if (col_major) {
      // a [groups, rows...] buffer viewed with the group axis last
      at::DimVector stride(x.dim(), 1);
      for (int64_t d = x.dim() - 3; d >= 0; --d) stride[d] = stride[d + 1] * size[d + 1];
      stride.back() = rows;
      s = empty_strided(size, stride, at::kFloat, x);
    } else {
      s = empty(size, at::kFloat, x);
    }
    if (res) sum = empty(x.sizes(), x.scalar_type(), x);
    rc = abi.norm_quant(ptr(x), row_stride(x), optr(res), res ? row_stride(*res) : 0, in_code(x.scalar_type()), ptr(w), in_code(w.scalar_type()), ptr(q),
                        fptr(s), col_major ? 1 : groups, col_major ? rows : 1, res ? ptr(sum) : nullptr, H, rows, H, static_cast<float>(eps),
                        static_cast<float>(quant_eps), stream_of(x));
  }
  if (rc != DLB_OK) NOT_PLAIN;
  return res ? tuple_of({&q, &s, &sum}) : tuple_of({&q, &s});
  HANDLE_EXCEPTIONS_END
}

// moe_permute(x, x_s, topk_ids, num_experts, alignment, num_rows) -> (rows, rows_s, row_index, source, m_indices, row_start, row_end)
PyObject* moe_permute(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_EXCEPTIONS_BEGIN
  int64_t E, align, R = -1;
  if (n != 6 || !integer(args[3], &E) || !integer(args[4], &align) || (args[5] != Py_None && !integer(args[5], &R))) NOT_PLAIN;
  const at::Tensor* t[3];
  bool grad = false;
  if (!take(args, t, 2, &grad)) NOT_PLAIN;
  const at::Tensor &x = *t[0], &ids = *t[2];
  const at::Tensor* x_s = t[1];
  if (x.dim() != 2 || ids.dim() != 2 || x.numel() == 0 || ids.size(0) != x.size(0) || x.stride(1) != 1 || idx_code(ids.scalar_type()) < 0) NOT_PLAIN;
  const int64_t T = x.size(0), H = x.size(1), topk = ids.size(1), slots = T * topk;
  if (topk < 1 || topk > kMaxTopk || E < 1 || E > kMaxExperts || align < 1 || align > (1 << 20) || slots >= (1ll << 31)) NOT_PLAIN;
  if (args[5] == Py_None) R = ceil_div(slots + std::min(E, slots) * (align - 1), align) * align;
  if (R < 1 || R >= (1ll << 31)) NOT_PLAIN;
  if (x_s) {
    if (grad || !is_f8(x) || !is_f32(*x_s) || x_s->dim() != 2 || H % kBlock != 0 || x_s->size(0) != T || x_s->size(1) != H / kBlock || x.stride(0) % 16 != 0 ||
        reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 != 0)
      NOT_PLAIN;
  } else if (in_code(x.scalar_type()) < 0) {
    NOT_PLAIN;
  }
  const OpRecord record("dlblas::moe_permute", t);
  DeviceScope scope(x);
  variable_list out;
  {
    const NoGil nogil;
    out = grad ? Permute::apply(x, ids, E, align, R) : permute_forward(x, x_s, ids, E, align, R);
  }
  at::Tensor none;
  return tuple_of({&out[0], x_s ? &out[6] : &none, &out[1], &out[2], &out[3], &out[4], &out[5]});
  DECLINE_FAILED
  HANDLE_EXCEPTIONS_END
}

// moe_unpermute(rows, row_index, weights, source) -> out; source None: no gradient
PyObject* moe_unpermute(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_EXCEPTIONS_BEGIN
  const at::Tensor* t[4];
  bool grad = false;
  if (n != 4 || !take(args, t, 12, &grad)) NOT_PLAIN;
  const at::Tensor &rows = *t[0], &index = *t[1];
  const at::Tensor *w = t[2], *source = t[3];
  if (rows.dim() != 2 || index.dim() != 2 || rows.numel() == 0 || index.numel() == 0 || rows.stride(1) != 1 || in_code(rows.scalar_type()) < 0 ||
      index.scalar_type() != at::kInt || !index.is_contiguous() || index.size(1) > kMaxTopk)
    NOT_PLAIN;
  if (w && (!is_f32(*w) || w->sizes() != index.sizes() || !w->is_contiguous())) NOT_PLAIN;
  if (grad && (!source || !index_of_rows(*source, rows.size(0)) || rows.size(1) > DLB_NORM_MAX_COLUMNS)) NOT_PLAIN;
  const OpRecord record("dlblas::moe_unpermute", t);
  DeviceScope scope(rows);
  at::Tensor out;
  {
    const NoGil nogil;
    out = grad ? Unpermute::apply(rows, optional_of(w), index, *source) : unpermute_forward(rows, index, w);
  }
  return THPVariable_Wrap(std::move(out));
  DECLINE_FAILED
  HANDLE_EXCEPTIONS_END
}

// Group size of the weights of a product, 0: not plain ones.
int64_t w4_group(const at::Tensor& x, const at::Tensor& q, const at::Tensor& s, const at::Tensor* z, int64_t dims) {
  const at::ScalarType type = x.scalar_type();
  if ((type != at::kBFloat16 && type != at::kHalf) || q.scalar_type() != at::kByte || in_code(s.scalar_type()) < 0 || q.dim() != dims || s.dim() != dims) return 0;
  for (int64_t d = 0; d + 1 < dims; ++d)
    if (q.size(d) != s.size(d)) return 0;
  if (!q.is_contiguous() || !s.is_contiguous() || q.numel() == 0 || s.numel() == 0 || x.numel() == 0 || x.size(-1) != 2 * q.size(-1)) return 0;
  if (z && (z->scalar_type() != at::kByte || z->sizes() != s.sizes() || !z->is_contiguous())) return 0;
  const int64_t K = x.size(-1), groups = s.size(-1), stride = row_stride(x);
  if (stride < 0 || stride % 2 != 0 || stride > (1 << 24) || reinterpret_cast<uintptr_t>(x.data_ptr()) % 4 != 0) return 0;
  return K % groups == 0 ? K / groups : 0;  // the library refuses other sizes than its own
}

// w4_gemm(x, w_q, w_s, w_z) -> y
PyObject* w4_gemm(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_EXCEPTIONS_BEGIN
  const at::Tensor* t[4];
  if (n != 4 || !take(args, t, 8)) NOT_PLAIN;
  const at::Tensor &x = *t[0], &q = *t[1], &s = *t[2];
  if (x.dim() < 1) NOT_PLAIN;
  const int64_t group = w4_group(x, q, s, t[3], 2);
  if (group == 0) NOT_PLAIN;
  const OpRecord record("dlblas::w4_gemm", t);
  const int64_t K = x.size(-1), M = x.numel() / K, N = q.size(0);
  at::DimVector size(x.sizes());
  size.back() = N;
  DeviceScope scope(x);
  at::Tensor y, sums;
  int rc;
  {
    const NoGil nogil;
    y = empty(size, x.scalar_type(), x);
    const size_t need = abi.w4_ws(M, N, K, 0);
    if (need > 0) sums = empty({static_cast<int64_t>(need)}, at::kByte, x);
    rc = abi.w4(ptr(x), row_stride(x), in_code(x.scalar_type()), ptr(q), ptr(s), in_code(s.scalar_type()), optr(t[3]), ptr(y), N, nullptr, nullptr, M, N, K,
                group, 1, need > 0 ? ptr(sums) : nullptr, need, stream_of(x));
  }
  if (rc != DLB_OK) NOT_PLAIN;
  return THPVariable_Wrap(std::move(y));
  HANDLE_EXCEPTIONS_END
}

// w4_gemm_grouped(x, w_q, w_s, row_start, row_end, w_z) -> y
PyObject* w4_gemm_grouped(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_EXCEPTIONS_BEGIN
  const at::Tensor* t[6];
  if (n != 6 || !take(args, t, 32)) NOT_PLAIN;
  const at::Tensor &x = *t[0], &q = *t[1], &s = *t[2], &start = *t[3], &end = *t[4];
  if (x.dim() != 2 || x.stride(1) != 1) NOT_PLAIN;
  const int64_t group = w4_group(x, q, s, t[5], 3);
  if (group == 0) NOT_PLAIN;
  const int64_t E = q.size(0), N = q.size(1), K = x.size(1), R = x.size(0);
  for (const at::Tensor* r : {&start, &end})
    if (r->scalar_type() != at::kInt || r->dim() != 1 || r->size(0) != E || !r->is_contiguous()) NOT_PLAIN;
  const OpRecord record("dlblas::w4_gemm_grouped", t);
  DeviceScope scope(x);
  at::Tensor y;
  int rc;
  {
    const NoGil nogil;
    y = empty({R, N}, x.scalar_type(), x);
    rc = abi.w4(ptr(x), x.stride(0), in_code(x.scalar_type()), ptr(q), ptr(s), in_code(s.scalar_type()), optr(t[5]), ptr(y), N, iptr(start), iptr(end), R, N,
                K, group, E, nullptr, 0, stream_of(x));
  }
  if (rc != DLB_OK) NOT_PLAIN;
  return THPVariable_Wrap(std::move(y));
  HANDLE_EXCEPTIONS_END
}

// init_steps(addresses): in the order of StepAbi's members
PyObject* init_steps(PyObject*, PyObject* list) {
  void* slots[sizeof(StepAbi) / sizeof(void*)];
  if (!PyList_Check(list) || PyList_GET_SIZE(list) != static_cast<Py_ssize_t>(sizeof(slots) / sizeof(void*)))
    return PyErr_Format(PyExc_ValueError, "a list of %zu addresses expected", sizeof(slots) / sizeof(void*));
  for (size_t i = 0; i < sizeof(slots) / sizeof(void*); ++i) {
    slots[i] = PyLong_AsVoidPtr(PyList_GET_ITEM(list, i));
    if (!slots[i]) return PyErr_Occurred() ? nullptr : PyErr_Format(PyExc_ValueError, "address %zu is NULL", i);
  }
  memcpy(&abi, slots, sizeof(abi));
  Py_RETURN_NONE;
}

}  // namespace

#define FAST(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(name)), METH_FASTCALL, nullptr}
PyMethodDef host_step_methods[] = {FAST(rms_norm), FAST(rms_norm_quant), FAST(moe_permute), FAST(moe_unpermute), FAST(w4_gemm), FAST(w4_gemm_grouped),
                                   {"init_steps", init_steps, METH_O, nullptr}, {nullptr, nullptr, 0, nullptr}};
