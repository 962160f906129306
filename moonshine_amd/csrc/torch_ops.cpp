// The serving operators (include/moonshine_hip.h) on torch tensors: what moonshine_amd/ops.py documents.  A call is a check of its
// tensors, the allocation of its outputs and the C entry: a module of its own, because the same in Python takes longer than the
// smallest kernels run.  Plain C API functions (no binding library); linked against libmoonshine.so, built by moonshine_amd/build.py.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/EmptyTensor.h>
#include <ATen/hip/impl/HIPCachingAllocatorMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/AutogradState.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/GradMode.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <stdexcept>
#include <optional>
#include <string>

#include "moonshine_hip.h"

namespace {

PyObject* g_error = nullptr;    // MshError(code, message)

struct Refused {
  int code;
  std::string what;
};
[[noreturn]] void refuse(const std::string& what) { throw Refused{MSH_ERR_INVALID_ARGUMENT, what}; }
struct PyFailed {};

int64_t check(int64_t rc) {
  if (rc < 0) throw Refused{(int)rc, msh_op_last_error()};
  return rc;
}

std::string shape_of(const at::Tensor& t) {
  std::string s = c10::toString(t.scalar_type()) + std::string(" (");
  for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
  return s + ")";
}

const at::Tensor& tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) refuse(std::string(name) + ": a tensor is wanted");
  const at::Tensor& t = THPVariable_Unpack(o);
  if (t.is_neg() || t.is_conj()) refuse(std::string(name) + ": a view whose sign torch has not applied yet (x.conj().imag); give x.resolve_neg()");
  return t;
}
int64_t integer(PyObject* o, const char* name) {
  const int64_t v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    refuse(std::string(name) + ": an integer is wanted");
  }
  return v;
}

bool truth(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw PyFailed{};
  return v != 0;
}

// the device that all tensors share, current for the call's allocations, and torch's current stream there
struct Place {
  int32_t device;
  void* stream;
  c10::Device where;
  c10::OptionalDeviceGuard guard;

  explicit Place(const at::Tensor& first) : device(0), stream(nullptr), where(first.device()) {
    if (!where.is_cuda()) refuse("tensors must be on the GPU, not on " + where.str() + ": there is no CPU fallback");
    guard.reset_device(where);
    device = where.index();
    stream = (void*)c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(where.index()).stream();
  }
  const Place& same(const at::Tensor& t) const {
    if (t.device() != where) refuse("tensors on " + where.str() + " and " + t.device().str() + ": one call, one device");
    return *this;
  }
};

void no_grad(const at::Tensor& t) {
  if (t.requires_grad() && c10::GradMode::is_enabled())
    refuse("an input requires a gradient: this operator has no backward pass (call it under torch.no_grad())");
  // (torch.no_grad() does not end forward differentiation)
  if (c10::AutogradState::get_tls_state().get_fw_grad_mode() && t._fw_grad(0).defined())
    refuse("an input has a tangent: this operator has no forward derivative");
}

// a tensor that the call writes in place counts as changed, so that a backward pass that saved it says so.  (One made under inference mode has no count.)
void written(const at::Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

int32_t dtype_of(const at::Tensor& t, const char* name) {
  switch (t.scalar_type()) {
    case at::kFloat: return MSH_F32;
    case at::kBFloat16: return MSH_BF16;
    case at::kHalf: return MSH_F16;
    default: refuse(std::string(name) + ": fp32, bf16 or fp16 is wanted, not " + c10::toString(t.scalar_type()));
  }
}

// address of a contiguous tensor of this type and shape
void* array(const at::Tensor& t, const char* name, at::ScalarType type, at::IntArrayRef shape) {
  if (t.scalar_type() != type || t.sizes() != shape || !t.is_contiguous()) {
    std::string want = c10::toString(type) + std::string(" (");
    for (size_t i = 0; i < shape.size(); ++i) want += (i ? ", " : "") + std::to_string(shape[i]);
    refuse(std::string(name) + ": a contiguous tensor " + want + ") is wanted, not " + shape_of(t));
  }
  return t.data_ptr();
}

// Outputs and workspaces come from torch's allocator without the dispatcher, which takes longer than the allocation (0.5 us each of a call's 5 to 10).
c10::Allocator* allocator() { return c10::hip::HIPCachingAllocatorMasqueradingAsCUDA::get(); }
at::Tensor make(const Place&, at::IntArrayRef shape, at::ScalarType type) {
  return at::detail::empty_generic(shape, allocator(), c10::DispatchKeySet(c10::DispatchKey::CUDA), type, std::nullopt);
}

msh_kv4_cache cache_of(const at::Tensor& t, int64_t head_dim) {
  if (t.scalar_type() != at::kByte || t.dim() != 4 || !t.is_contiguous())
    refuse("cache: the contiguous uint8 tensor [pages, heads, page_size / 32, bytes] of kv4_cache() is wanted");
  if (head_dim < 1 || head_dim > 256 || t.size(3) != 1088 * ((head_dim + 31) / 32))
    refuse("cache: its blocks of " + std::to_string(t.size(3)) + " bytes are not those of head_dim " + std::to_string(head_dim));
  if (t.size(1) > 1024 || t.size(2) > 2048) refuse("cache: too many heads or blocks a page");
  return msh_kv4_cache{t.data_ptr(), t.size(0), (int32_t)t.size(1), (int32_t)t.size(2) * 32, (int32_t)head_dim};
}

int32_t small(int64_t v, const char* name) {
  if (v < INT32_MIN || v > INT32_MAX) refuse(std::string(name) + ": too large");
  return (int32_t)v;
}

PyObject* wrap(std::initializer_list<at::Tensor> list) {
  PyObject* out = PyTuple_New((Py_ssize_t)list.size());
  if (out == nullptr) throw PyFailed{};
  Py_ssize_t i = 0;
  for (const at::Tensor& t : list) {
    PyObject* o = THPVariable_Wrap(t);
    if (o == nullptr) {
      Py_DECREF(out);
      throw PyFailed{};
    }
    PyTuple_SET_ITEM(out, i++, o);
  }
  return out;
}

// ---- the operators ------------------------------------------------------------------------------------------------------
PyObject* page_plan(PyObject* const* a) {
  const at::Tensor &table = tensor(a[0], "block_table"), &kv = tensor(a[1], "kv_lens"), &fresh = tensor(a[2], "new_lens"),
                   &start = tensor(a[3], "row_start"), &free_pages = tensor(a[5], "free_pages");
  const int64_t rows = integer(a[4], "rows"), page = integer(a[6], "page_size");
  const Place p(table);
  p.same(kv).same(fresh).same(start).same(free_pages);
  if (table.dim() != 2 || free_pages.dim() != 1) refuse("block_table: [batch, width]; free_pages: [n]");
  if (rows < 0) refuse("rows: not negative");
  const int64_t batch = table.size(0), width = table.size(1), n_free = free_pages.size(0);
  auto* tp = (int32_t*)array(table, "block_table", at::kInt, {batch, width});
  auto* kp = (const int32_t*)array(kv, "kv_lens", at::kInt, {batch});
  auto* fp = (const int32_t*)array(fresh, "new_lens", at::kInt, {batch});
  auto* sp = (const int32_t*)array(start, "row_start", at::kInt, {batch});
  auto* pp = (const int32_t*)array(free_pages, "free_pages", at::kInt, {n_free});
  at::Tensor slots = make(p, {rows}, at::kLong), used = make(p, {1}, at::kInt);
  check(msh_page_plan(p.device, p.stream, tp, small(batch, "batch"), small(width, "width"), kp, fp, sp, rows, pp, n_free, small(page, "page_size"),
                      (int64_t*)slots.data_ptr(), (int32_t*)used.data_ptr()));
  written(table);
  return wrap({slots, used});
}

PyObject* kv4_write(PyObject* const* a) {
  const at::Tensor &cache = tensor(a[0], "cache"), &k = tensor(a[1], "k"), &v = tensor(a[2], "v"), &slots = tensor(a[3], "slots");
  const Place p(cache);
  p.same(k).same(v).same(slots);
  no_grad(k);
  no_grad(v);
  if (k.dim() != 3 || k.sizes() != v.sizes() || k.scalar_type() != v.scalar_type()) refuse("k and v: [rows, heads, head_dim], of one type");
  const int32_t type = dtype_of(k, "k and v");
  const int64_t rows = k.size(0);
  const msh_kv4_cache c = cache_of(cache, k.size(2));
  if (k.size(1) != c.heads) refuse("k and v have " + std::to_string(k.size(1)) + " heads, the cache " + std::to_string(c.heads));
  auto* sp = (const int64_t*)array(slots, "slots", at::kLong, {rows});
  const int64_t ks[3] = {k.stride(0), k.stride(1), k.stride(2)}, vs[3] = {v.stride(0), v.stride(1), v.stride(2)};
  check(msh_kv4_write(p.device, p.stream, &c, k.data_ptr(), ks, v.data_ptr(), vs, type, rows, sp));
  written(cache);
  Py_RETURN_NONE;
}

PyObject* kv4_read(PyObject* const* a) {
  const at::Tensor &cache = tensor(a[0], "cache"), &slots = tensor(a[1], "slots");
  const int64_t head_dim = integer(a[2], "head_dim"), type = integer(a[3], "dtype");
  const Place p(cache);
  p.same(slots);
  if (slots.dim() != 1) refuse("slots: [rows]");
  const int64_t rows = slots.size(0);
  const msh_kv4_cache c = cache_of(cache, head_dim);
  auto* sp = (const int64_t*)array(slots, "slots", at::kLong, {rows});
  const at::ScalarType t = type == MSH_F32 ? at::kFloat : type == MSH_BF16 ? at::kBFloat16 : at::kHalf;
  at::Tensor k = make(p, {rows, c.heads, head_dim}, t), v = make(p, {rows, c.heads, head_dim}, t);
  check(msh_kv4_read(p.device, p.stream, &c, sp, rows, k.data_ptr(), v.data_ptr(), (int32_t)type));
  return wrap({k, v});
}

// q, cache, block_table, kv_lens, q_start | None, max_q | None, scale | None, causal, window, return_lse, out | None
PyObject* kv4_attention(PyObject* const* a) {
  const at::Tensor &q = tensor(a[0], "q"), &cache = tensor(a[1], "cache"), &table = tensor(a[2], "block_table"), &lens = tensor(a[3], "kv_lens");
  const bool ragged = a[4] != Py_None;
  const Place p(q);
  p.same(cache).same(table).same(lens);
  no_grad(q);
  if (q.dim() != 3 || (q.stride(2) != 1 && q.size(2) > 1)) refuse("q: [rows, heads, head_dim] with a contiguous last dimension");
  if (table.dim() != 2) refuse("block_table: [batch, width]");
  msh_kv4_attention_args x{};
  x.dtype = dtype_of(q, "q");
  x.cache = cache_of(cache, q.size(2));
  x.rows = q.size(0), x.heads = small(q.size(1), "heads");
  int64_t batch = table.size(0), max_q = a[5] != Py_None ? integer(a[5], "max_q") : -1;
  x.table_width = small(table.size(1), "width");
  x.block_table = (const int32_t*)array(table, "block_table", at::kInt, {batch, table.size(1)});
  x.kv_lens = (const int32_t*)array(lens, "kv_lens", at::kInt, {batch});
  if (ragged) {
    const at::Tensor& start = tensor(a[4], "q_start");
    p.same(start);
    if (a[5] == Py_None) refuse("max_q: the most rows of a sequence (q_start is on the device)");
    x.q_start = (const int32_t*)array(start, "q_start", at::kInt, {batch + 1});
  } else {
    if (a[5] == Py_None) max_q = batch > 0 ? x.rows / batch : 1;
    if (x.rows != batch * max_q) refuse(std::to_string(x.rows) + " rows are not " + std::to_string(max_q) + " for each of " + std::to_string(batch) + " sequences: give q_start");
    if (x.rows == 0) batch = 0, max_q = 1;
  }
  x.batch = small(batch, "batch"), x.max_q = small(max_q, "max_q");
  x.causal = truth(a[7]) ? 1 : 0;
  x.window = small(integer(a[8], "window"), "window");
  if (a[6] == Py_None) {
    x.scale = (float)(1.0 / std::sqrt((double)q.size(2)));
  } else {
    const double s = PyFloat_AsDouble(a[6]);
    if (s == -1.0 && PyErr_Occurred()) throw PyFailed{};
    x.scale = (float)s;
  }
  at::Tensor out;
  if (a[10] != Py_None) {
    out = tensor(a[10], "out");
    p.same(out);
    if (out.sizes() != q.sizes() || out.scalar_type() != q.scalar_type() || (out.stride(2) != 1 && q.size(2) > 1))
      refuse("out: q's shape and type, with a contiguous last dimension");
    no_grad(out);
    const int64_t rows = out.size(0), heads = out.size(1), width = out.size(2), r = out.stride(0), h = out.stride(1);
    const bool by_row = (heads == 1 || h >= width) && (rows == 1 || r >= (heads - 1) * h + width);
    const bool by_head = (rows == 1 || r >= width) && (heads == 1 || h >= (rows - 1) * r + width);
    if (rows > 0 && !by_row && !by_head) refuse("out: its rows overlap");
  } else {
    out = make(p, q.sizes(), q.scalar_type());
  }
  at::Tensor lse;
  const bool with_lse = truth(a[9]);
  if (with_lse) lse = make(p, {x.rows, q.size(1)}, at::kFloat);
  x.q = q.data_ptr(), x.out = out.data_ptr(), x.lse = with_lse ? (float*)lse.data_ptr() : nullptr;
  x.q_row_stride = q.stride(0), x.q_head_stride = q.stride(1), x.out_row_stride = out.stride(0), x.out_head_stride = out.stride(1);
  const int64_t size = check(msh_kv4_attention_workspace(&x));
  const c10::DataPtr work = size > 0 ? allocator()->allocate((size_t)size) : c10::DataPtr();
  check(msh_kv4_attention(p.device, p.stream, &x, work.get(), size));
  if (a[10] != Py_None) written(out);
  if (with_lse) return wrap({out, lse});
  return THPVariable_Wrap(out);
}

PyObject* beam_select(PyObject* const* a) {
  const at::Tensor &logits = tensor(a[0], "logits"), &scores = tensor(a[1], "scores"), &finished = tensor(a[2], "finished");
  const int64_t eos = integer(a[3], "eos");
  const Place p(logits);
  p.same(scores).same(finished);
  no_grad(logits);
  no_grad(scores);
  if (logits.dim() != 3 || (logits.stride(2) != 1 && logits.size(2) > 1)) refuse("logits: [batch, beams, vocab] with a contiguous last dimension");
  const int32_t type = dtype_of(logits, "logits");
  const int64_t batch = logits.size(0), beams = logits.size(1), vocab = logits.size(2);
  int64_t row = logits.stride(1);
  if (beams == 1) row = logits.stride(0);
  else if (batch > 1 && logits.stride(0) != beams * row) refuse("logits: the rows of all beams must be evenly spaced");
  const at::ScalarType flag = finished.scalar_type();
  if (flag != at::kByte && flag != at::kBool) refuse("finished: uint8 or bool");
  auto* sp = (const float*)array(scores, "scores", at::kFloat, {batch, beams});
  auto* fp = (const uint8_t*)array(finished, "finished", flag, {batch, beams});
  const int64_t size = check(msh_beam_select_workspace(small(batch, "batch"), small(beams, "beams"), small(vocab, "vocab")));
  at::Tensor next = make(p, {batch, beams}, at::kFloat), parents = make(p, {batch, beams}, at::kInt), tokens = make(p, {batch, beams}, at::kInt),
             ended = make(p, {batch, beams}, flag);
  const c10::DataPtr work = allocator()->allocate((size_t)size);
  check(msh_beam_select(p.device, p.stream, logits.data_ptr(), type, row, (int32_t)batch, (int32_t)beams, (int32_t)vocab, sp, fp, small(eos, "eos"),
                        (float*)next.data_ptr(), (int32_t*)parents.data_ptr(), (int32_t*)tokens.data_ptr(), (uint8_t*)ended.data_ptr(),
                        work.get(), size));
  return wrap({next, parents, tokens, ended});
}

// several dimensions walked as one: (count, stride in elements)
std::pair<int64_t, int64_t> merge(at::IntArrayRef sizes, at::IntArrayRef strides, int64_t from, int64_t to, const char* what) {
  int64_t n = 1, step = 0;
  for (int64_t i = to - 1; i >= from; --i) {
    if (sizes[i] == 1) continue;
    if (n == 1) step = strides[i];
    else if (strides[i] != n * step) refuse(std::string("state: its ") + what + " dimensions cannot be walked as one");
    n *= sizes[i];
  }
  return {n, step};
}

// states (sequence), parents, lengths | None, batch_dims (sequence), row_dims (sequence)
PyObject* beam_reorder(PyObject* const* a) {
  const at::Tensor& parents = tensor(a[1], "parents");
  const Place p(parents);
  if (!PyList_Check(a[0]) || !PyList_Check(a[3]) || !PyList_Check(a[4])) refuse("states, batch_dims and row_dims: lists");
  const Py_ssize_t n = PyList_GET_SIZE(a[0]);
  if (parents.dim() != 2 || n < 1 || n > 4 || PyList_GET_SIZE(a[3]) != n || PyList_GET_SIZE(a[4]) != n)
    refuse("parents: [batch, beams]; one to four states, each with a batch and a row dimension");
  const int64_t batch = parents.size(0), beams = parents.size(1);
  auto* pp = (const int32_t*)array(parents, "parents", at::kInt, {batch, beams});
  msh_beam_state states[4];
  for (Py_ssize_t i = 0; i < n; ++i) {
    const at::Tensor& t = tensor(PyList_GET_ITEM(a[0], i), "state");
    const int64_t b = integer(PyList_GET_ITEM(a[3], i), "batch_dims"), r = integer(PyList_GET_ITEM(a[4], i), "row_dims");
    p.same(t);
    no_grad(t);
    const at::IntArrayRef shape = t.sizes(), strides = t.strides();
    if (b < 0 || r <= b + 1 || r >= t.dim() || shape[b] != batch || shape[b + 1] != beams)
      refuse("state " + shape_of(t) + ": dimensions " + std::to_string(b) + " and " + std::to_string(b + 1) + " are not the " + std::to_string(batch) +
             " entries and " + std::to_string(beams) + " beams, or dimension " + std::to_string(r) + " does not follow them");
    const auto outer = merge(shape, strides, 0, b, "outer"), inner = merge(shape, strides, b + 2, r, "inner"), row = merge(shape, strides, r + 1, t.dim(), "last");
    if (row.first > 1 && row.second != 1) refuse("state: what follows the row dimension must be contiguous");
    if (shape[r] > 1 && strides[r] != row.first) refuse("state: its rows must be contiguous");
    const int64_t beam = beams > 1 ? strides[b + 1] : strides[b];
    if (batch > 1 && strides[b] != beams * beam) refuse("state: its beams must be evenly spaced over all entries");
    const int64_t size = (int64_t)t.element_size();
    states[i] = msh_beam_state{t.data_ptr(), outer.first, outer.second * size, beam * size, inner.first, inner.second * size, row.first * size, shape[r]};
  }
  const int32_t* lp = nullptr;
  int32_t each = 0;
  if (a[2] != Py_None) {
    const at::Tensor& lengths = tensor(a[2], "lengths");
    p.same(lengths);
    if (lengths.dim() != 1 || (lengths.size(0) != 1 && lengths.size(0) != batch)) refuse("lengths: int32 [batch] or [1]");
    lp = (const int32_t*)array(lengths, "lengths", at::kInt, {lengths.size(0)});
    each = lengths.size(0) == batch ? 1 : 0;
  }
  check(msh_beam_reorder(p.device, p.stream, states, (int32_t)n, small(batch, "batch"), small(beams, "beams"), pp, lp, each));
  for (Py_ssize_t i = 0; i < n; ++i) written(tensor(PyList_GET_ITEM(a[0], i), "state"));
  Py_RETURN_NONE;
}

// ---- module -------------------------------------------------------------------------------------------------------------
template <PyObject* (*F)(PyObject* const*), int N>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != N) {
    PyErr_Format(PyExc_TypeError, "%d arguments are wanted", N);
    return nullptr;
  }
  try {
    return F(args);
  } catch (const Refused& r) {
    PyObject* v = Py_BuildValue("(is)", r.code, r.what.c_str());
    if (v != nullptr) PyErr_SetObject(g_error, v);
    Py_XDECREF(v);
  } catch (const PyFailed&) {
  } catch (const std::exception& e) {   // torch's own: an allocation that does not fit
    PyErr_SetString(PyExc_RuntimeError, e.what());
  } catch (...) {
    PyErr_SetString(PyExc_RuntimeError, "unknown error");
  }
  return nullptr;
}

PyObject* set_up(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 1) {
    PyErr_SetString(PyExc_TypeError, "set_up(error class)");
    return nullptr;
  }
  Py_INCREF(args[0]);
  g_error = args[0];
  Py_RETURN_NONE;
}

#define MSH_METHOD(name, fn) {name, (PyCFunction)(void (*)(void))(fn), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {
    MSH_METHOD("set_up", set_up),
    MSH_METHOD("page_plan", (entry<page_plan, 7>)),
    MSH_METHOD("kv4_write", (entry<kv4_write, 4>)),
    MSH_METHOD("kv4_read", (entry<kv4_read, 4>)),
    MSH_METHOD("kv4_attention", (entry<kv4_attention, 11>)),
    MSH_METHOD("beam_select", (entry<beam_select, 4>)),
    MSH_METHOD("beam_reorder", (entry<beam_reorder, 5>)),
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "msh_torch_ops", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

extern "C" __attribute__((visibility("default"))) PyObject* PyInit_msh_torch_ops() {
  PyObject* m = PyModule_Create(&module);
  if (m != nullptr && PyModule_AddStringConstant(m, "torch_version", MSH_TORCH_VERSION) != 0) {
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
