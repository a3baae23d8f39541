// The steps around the products of a decoder block as native calls, under the same rules as host_calls.cpp: a function does the
// whole call or returns None without a trace, and the Python function then takes its own path.
#include "host_tensors.h"

namespace {

struct StepAbi {
  decltype(&dlb_rms_norm) norm;
  decltype(&dlb_rms_norm_quant) norm_quant;
  decltype(&dlb_moe_sort_workspace_bytes) sort_ws;
  decltype(&dlb_moe_sort) sort;
  decltype(&dlb_moe_permute) permute;
  decltype(&dlb_moe_unpermute) unpermute;
  decltype(&dlb_w4_gemm) w4;
} abi;

constexpr int64_t kMaxTopk = 64, kMaxExperts = DLB_SORT_MAX_EXPERTS;

// The tensors of a call, None (nullptr) where `optional` allows it; all plain and on the device of the first.
template <size_t N>
bool take(PyObject* const* args, const at::Tensor* (&out)[N], uint64_t optional) {
  if (!no_modes()) return false;
  for (size_t i = 0; i < N; ++i) {
    out[i] = nullptr;
    if (args[i] == Py_None && (optional >> i & 1)) continue;
    out[i] = plain(args[i]);
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

// rms_norm(x, weight, eps, residual) -> y, or (y, h)
PyObject* rms_norm(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_EXCEPTIONS_BEGIN
  if (n != 4 || !PyFloat_CheckExact(args[2])) NOT_PLAIN;
  PyObject* const given[] = {args[0], args[1], args[3]};
  const at::Tensor* t[3];
  if (!take(given, t, 4)) NOT_PLAIN;
  const at::Tensor &x = *t[0], &w = *t[1];
  const at::Tensor* res = t[2];
  const double eps = PyFloat_AS_DOUBLE(args[2]);
  if (!norm_operands(x, w, res) || !(eps >= 0)) NOT_PLAIN;
  const OpRecord record("dlblas::rms_norm", t);
  const int64_t H = x.size(-1), rows = x.numel() / H;
  DeviceScope scope(x);
  at::Tensor y, sum;
  int rc;
  {
    const NoGil nogil;
    y = empty(x.sizes(), x.scalar_type(), x);
    if (res) sum = empty(x.sizes(), x.scalar_type(), x);
    rc = abi.norm(ptr(x), row_stride(x), optr(res), res ? row_stride(*res) : 0, in_code(x.scalar_type()), ptr(w), in_code(w.scalar_type()), ptr(y), H,
                  res ? ptr(sum) : nullptr, H, rows, H, static_cast<float>(eps), stream_of(x));
  }
  if (rc != DLB_OK) NOT_PLAIN;
  return res ? tuple_of({&y, &sum}) : THPVariable_Wrap(std::move(y));
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
  if (!take(args, t, 2)) NOT_PLAIN;
  const at::Tensor &x = *t[0], &ids = *t[2];
  const at::Tensor* x_s = t[1];
  if (x.dim() != 2 || ids.dim() != 2 || x.numel() == 0 || ids.size(0) != x.size(0) || x.stride(1) != 1 || idx_code(ids.scalar_type()) < 0) NOT_PLAIN;
  const int64_t T = x.size(0), H = x.size(1), topk = ids.size(1), slots = T * topk;
  if (topk < 1 || topk > kMaxTopk || E < 1 || E > kMaxExperts || align < 1 || align > (1 << 20)) NOT_PLAIN;
  if (args[5] == Py_None) R = ceil_div(slots + std::min(E, slots) * (align - 1), align) * align;
  if (R < 1 || R >= (1ll << 31)) NOT_PLAIN;
  int code = in_code(x.scalar_type());
  if (x_s) {
    if (!is_f8(x) || !is_f32(*x_s) || x_s->dim() != 2 || H % kBlock != 0 || x_s->size(0) != T || x_s->size(1) != H / kBlock || x.stride(0) % 16 != 0) NOT_PLAIN;
    code = DLB_ROWS_E4M3;
  }
  if (code < 0) NOT_PLAIN;
  const OpRecord record("dlblas::moe_permute", t);
  DeviceScope scope(x);
  const hipStream_t stream = stream_of(x);
  at::Tensor rows, rows_s, row_index, source, m_indices, start, end, scratch;
  int rc;
  {
    const NoGil nogil;
    rows = empty({R, H}, x.scalar_type(), x);
    if (x_s) rows_s = empty({R, H / kBlock}, at::kFloat, x);
    row_index = empty({T, topk}, at::kInt, x);
    source = empty({R}, at::kInt, x);
    m_indices = empty({R}, at::kInt, x);
    start = empty({E}, at::kInt, x);
    end = empty({E}, at::kInt, x);
    const size_t need = abi.sort_ws(T, topk, E);
    if (need > 0) scratch = empty({static_cast<int64_t>(need)}, at::kByte, x);
    rc = abi.sort(ptr(ids), idx_code(ids.scalar_type()), ids.stride(0), ids.stride(1), iptr(row_index), iptr(source), iptr(m_indices), iptr(start),
                  iptr(end), T, topk, E, align, R, need > 0 ? ptr(scratch) : nullptr, need, stream);
    if (rc == DLB_OK)
      rc = abi.permute(ptr(x), x.stride(0), code, x_s ? fptr(*x_s) : nullptr, x_s ? x_s->stride(0) : 0, x_s ? x_s->stride(1) : 0, ptr(rows),
                       x_s ? fptr(rows_s) : nullptr, iptr(row_index), iptr(source), T, H, topk, R, stream);
  }
  if (rc != DLB_OK) NOT_PLAIN;  // the Python path starts over in buffers of its own
  return tuple_of({&rows, &rows_s, &row_index, &source, &m_indices, &start, &end});
  HANDLE_EXCEPTIONS_END
}

// moe_unpermute(rows, row_index, weights) -> out
PyObject* moe_unpermute(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_EXCEPTIONS_BEGIN
  const at::Tensor* t[3];
  if (n != 3 || !take(args, t, 4)) NOT_PLAIN;
  const at::Tensor &rows = *t[0], &index = *t[1];
  const at::Tensor* w = t[2];
  if (rows.dim() != 2 || index.dim() != 2 || rows.numel() == 0 || index.numel() == 0 || rows.stride(1) != 1 || in_code(rows.scalar_type()) < 0 ||
      index.scalar_type() != at::kInt || !index.is_contiguous() || index.size(1) > kMaxTopk)
    NOT_PLAIN;
  if (w && (!is_f32(*w) || w->sizes() != index.sizes() || !w->is_contiguous())) NOT_PLAIN;
  const OpRecord record("dlblas::moe_unpermute", t);
  const int64_t T = index.size(0), H = rows.size(1);
  DeviceScope scope(rows);
  at::Tensor out;
  int rc;
  {
    const NoGil nogil;
    out = empty({T, H}, rows.scalar_type(), rows);
    rc = abi.unpermute(ptr(rows), rows.stride(0), in_code(rows.scalar_type()), iptr(index), w ? fptr(*w) : nullptr, ptr(out), H, T, H, index.size(1),
                       rows.size(0), stream_of(rows));
  }
  if (rc != DLB_OK) NOT_PLAIN;
  return THPVariable_Wrap(std::move(out));
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
  const int64_t K = x.size(-1), groups = s.size(-1);
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
  if (group == 0 || row_stride(x) < 0) NOT_PLAIN;
  const OpRecord record("dlblas::w4_gemm", t);
  const int64_t K = x.size(-1), M = x.numel() / K, N = q.size(0);
  at::DimVector size(x.sizes());
  size.back() = N;
  DeviceScope scope(x);
  at::Tensor y;
  int rc;
  {
    const NoGil nogil;
    y = empty(size, x.scalar_type(), x);
    rc = abi.w4(ptr(x), row_stride(x), in_code(x.scalar_type()), ptr(q), ptr(s), in_code(s.scalar_type()), optr(t[3]), ptr(y), N, nullptr, nullptr, M, N, K,
                group, 1, stream_of(x));
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
                K, group, E, stream_of(x));
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
