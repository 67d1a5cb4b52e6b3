// The short way from a PyTorch caller to the paged-cache and beam entries of libcv3cuda.so.
//
// A decode step's small operators take a few microseconds on the GPU; fetching shapes and strides,
// checking them and packing the parameter block in Python takes ten.  Each function here does the same
// for plain calls -- CUDA tensors of the current device, types and shapes as documented -- in one, and
// returns None for every other call, which paged.py then handles or refuses with its message.  The
// entries' addresses and the result classes come from Python (setup), so this module links nothing of
// the library.
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <utility>

#include "../../../include/cv3cuda.h"

namespace {

using at::Tensor;

struct Entries {
  int (*extend)(const cv3_paged_extend_params*, void*);
  int (*append)(const cv3_paged_append_params*, void*);
  int (*attention)(const cv3_paged_attention_params*, void*);
  int64_t (*attention_workspace)(int64_t, int64_t, int64_t, int64_t, int, int64_t);
  int (*beam)(const cv3_beam_params*, void*);
  int64_t (*beam_workspace)(int64_t, int64_t, int64_t);
  int (*reorder)(const cv3_paged_reorder_params*, void*);
} cv3;
PyObject *step_class, *beam_class;  // PagedStep, BeamStep

// The call's device and arguments; `ok` turns false on the first that is not plain.
struct Call {
  PyObject* const* args;
  int device = -1;
  bool ok = true;

  explicit Call(PyObject* const* a) : args(a) {}
  bool none(int i) const { return args[i] == Py_None; }
  void need(bool c) { ok = ok && c; }
  const Tensor& tensor(int i) {
    static const Tensor nothing;
    if (!ok || !THPVariable_Check(args[i])) {
      ok = false;
      return nothing;
    }
    const Tensor& t = THPVariable_Unpack(args[i]);
    if (!t.is_cuda()) {
      ok = false;
      return nothing;
    }
    if (device < 0) {
      device = t.get_device();
      ok = device == c10::cuda::current_device();
    } else {
      ok = t.get_device() == device;
    }
    return ok ? t : nothing;
  }
  int64_t integer(int i) {
    if (!ok || !PyLong_Check(args[i])) {
      ok = false;
      return 0;
    }
    const long long v = PyLong_AsLongLong(args[i]);
    if (v == -1 && PyErr_Occurred()) {
      PyErr_Clear();
      ok = false;
    }
    return v;
  }
  double real(int i) {
    if (!ok) return 0.0;
    const double v = PyFloat_AsDouble(args[i]);
    if (v == -1.0 && PyErr_Occurred()) {
      PyErr_Clear();
      ok = false;
    }
    return v;
  }
  // n contiguous values of a type; nullptr for None where that is allowed
  void* values(int i, at::ScalarType type, int64_t n, bool optional = false) {
    if (optional && none(i)) return nullptr;
    const Tensor& t = tensor(i);
    if (!ok) return nullptr;
    need(t.scalar_type() == type && t.numel() == n && t.is_contiguous());
    return t.data_ptr();
  }
  int* ints(int i, int64_t n, bool optional = false) {
    return static_cast<int*>(values(i, at::kInt, n, optional));
  }
  void* stream() const { return c10::cuda::getCurrentCUDAStream(device).stream(); }
};

int type_of(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return CV3_TYPE_F32;
    case at::kHalf: return CV3_TYPE_F16;
    case at::kBFloat16: return CV3_TYPE_BF16;
    default: return -1;
  }
}

// an int32 block table with contiguous rows
void table_of(Call& c, int i, int64_t rows, int*& p, int64_t& ld, int64_t& cols) {
  const Tensor& t = c.tensor(i);
  if (!c.ok) return;
  c.need(t.dim() == 2 && t.scalar_type() == at::kInt && t.size(0) == rows && rows > 0 && t.size(1) > 0 && t.stride(1) == 1);
  if (!c.ok) return;
  p = t.data_ptr<int>();
  cols = t.size(1);
  ld = rows > 1 ? t.stride(0) : std::max(t.stride(0), cols);
}

// a pair of page pools with contiguous rows
void pools_of(Call& c, const Tensor& k, const Tensor& v, int dims, bool written = false) {
  if (!c.ok) return;
  c.need(k.dim() == dims && k.sizes() == v.sizes() && k.scalar_type() == v.scalar_type() && type_of(k) >= 0);
  if (!c.ok) return;
  c.need(k.stride(dims - 1) == 1 && v.stride(dims - 1) == 1 && k.size(dims - 2) > 0 && k.size(dims - 3) > 0 &&
         k.size(dims - 1) > 0);
  if (written)  // (no expanded views)
    for (int i = 0; i < dims; ++i) c.need(k.size(i) <= 1 || (k.stride(i) && v.stride(i)));
}

bool alike(const Tensor& t, at::IntArrayRef sizes, at::ScalarType type) {
  return t.sizes() == sizes && t.scalar_type() == type && t.is_contiguous();
}

// A contiguous uninitialised tensor, and n elements of one from `at` on (past the dispatcher, whose 0.4 us a
// tensor are a third of such a call).
Tensor fresh(at::IntArrayRef sizes, at::ScalarType type, const Tensor& like) {
  return Tensor(at::detail::empty_cuda(sizes, type, like.device(), std::nullopt));
}
Tensor part_of(const Tensor& all, int64_t at, int64_t n) {
  Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(all.storage()), all.key_set(), all.dtype());
  t.unsafeGetTensorImpl()->set_storage_offset(at);
  t.unsafeGetTensorImpl()->set_sizes_contiguous({n});
  return t;
}

// an instance of a named tuple class, as its _make gives it
PyObject* made(PyObject* cls, std::initializer_list<Tensor> parts) {
  PyObject* v = PyTuple_New((Py_ssize_t)parts.size());
  Py_ssize_t n = 0;
  for (const Tensor& t : parts) PyTuple_SET_ITEM(v, n++, THPVariable_Wrap(t));
  PyObject* args = PyTuple_Pack(1, v);
  PyObject* r = PyTuple_Type.tp_new(reinterpret_cast<PyTypeObject*>(cls), args, nullptr);
  Py_DECREF(args);
  Py_DECREF(v);
  return r;
}

// (lens, new_lens, block_tables, free_pages, free_count, page_size, max_tokens, release)
PyObject* extend(PyObject*, PyObject* const* args, Py_ssize_t) {
  Call c(args);
  const Tensor& lens = c.tensor(0);
  if (!c.ok || lens.dim() != 1) Py_RETURN_NONE;
  cv3_paged_extend_params p = {sizeof(p)};
  p.batch = lens.size(0);
  p.lens = c.ints(0, p.batch);
  p.new_lens = c.ints(1, p.batch);
  table_of(c, 2, p.batch, p.block_tables, p.table_ld, p.max_blocks);
  const Tensor& free = c.tensor(3);
  if (!c.ok) Py_RETURN_NONE;
  p.free_cap = free.numel();
  p.free_pages = c.ints(3, p.free_cap);
  p.free_count = c.ints(4, 1);
  p.page_size = c.integer(5);
  p.max_tokens = c.integer(6);
  p.release = c.ints(7, p.batch, true);
  const int64_t T = p.max_tokens, n = p.batch;
  if (!c.ok || T < 0 || T > INT32_MAX) Py_RETURN_NONE;
  const Tensor slots = fresh({T}, at::kLong, lens), all = fresh({2 * T + 3 * n + 3}, at::kInt, lens);
  int64_t at = 0;
  auto part = [&](int64_t m) { return part_of(all, std::exchange(at, at + m), m); };
  const Tensor seq = part(T), pos = part(T), offsets = part(n + 1), lens_out = part(n), count = part(1);
  p.slots = slots.data_ptr<int64_t>();
  p.seq = seq.data_ptr<int>();
  p.pos = pos.data_ptr<int>();
  p.offsets = offsets.data_ptr<int>();
  p.lens_out = lens_out.data_ptr<int>();
  p.free_count_out = count.data_ptr<int>();
  p.scratch = all.data_ptr<int>() + at;
  if (cv3.extend(&p, c.stream())) Py_RETURN_NONE;
  return made(step_class, {slots, seq, pos, offsets, lens_out, count});
}

// (qkv, slots, pos, k_pages, v_pages, heads, cos, sin, out, bad)
PyObject* append(PyObject*, PyObject* const* args, Py_ssize_t) {
  Call c(args);
  const Tensor &qkv = c.tensor(0), &k = c.tensor(3), &v = c.tensor(4);
  pools_of(c, k, v, 4, true);
  cv3_paged_append_params p = {sizeof(p)};
  p.heads = c.integer(5);
  if (!c.ok || qkv.dim() != 2 || type_of(qkv) < 0 || p.heads <= 0) Py_RETURN_NONE;
  p.kv_heads = k.size(1);
  p.head_dim = k.size(3);
  const int64_t width = (p.heads + 2 * p.kv_heads) * p.head_dim;
  c.need(qkv.size(1) == width && qkv.stride(1) == 1);
  if (!c.ok) Py_RETURN_NONE;
  p.qkv = qkv.data_ptr();
  p.type = type_of(qkv);
  p.rows = qkv.size(0);
  p.ldq = p.rows > 1 ? qkv.stride(0) : width;
  p.slots = static_cast<int64_t*>(c.values(1, at::kLong, p.rows));
  p.pos = c.ints(2, p.rows, true);
  if (!c.none(6)) {
    const Tensor &cos = c.tensor(6), &sin = c.tensor(7);
    if (!c.ok || cos.dim() != 2 || !p.pos) Py_RETURN_NONE;
    c.need(alike(cos, {cos.size(0), p.head_dim}, at::kFloat) && alike(sin, cos.sizes(), at::kFloat));
    if (!c.ok) Py_RETURN_NONE;
    p.cos_table = cos.data_ptr<float>();
    p.sin_table = sin.data_ptr<float>();
    p.positions = cos.size(0);
  } else {
    c.need(c.none(7));
  }
  p.bad = c.ints(9, 1, true);
  if (!c.ok) Py_RETURN_NONE;
  Tensor out;
  if (c.none(8)) {
    out = fresh({p.rows, p.heads, p.head_dim}, qkv.scalar_type(), qkv);
  } else {
    out = c.tensor(8);
    if (!c.ok || !alike(out, {p.rows, p.heads, p.head_dim}, qkv.scalar_type())) Py_RETURN_NONE;
  }
  p.q_out = out.data_ptr();
  p.k_pages = k.data_ptr();
  p.v_pages = v.data_ptr();
  p.kv_type = type_of(k);
  p.ksp = k.stride(0), p.ksh = k.stride(1), p.kst = k.stride(2);
  p.vsp = v.stride(0), p.vsh = v.stride(1), p.vst = v.stride(2);
  p.num_pages = k.size(0);
  p.page_size = k.size(2);
  if (cv3.append(&p, c.stream())) Py_RETURN_NONE;
  return THPVariable_Wrap(out);
}

// (q, k_pages, v_pages, block_tables, lens, scale, window, out, return_lse, bad)
PyObject* attention(PyObject*, PyObject* const* args, Py_ssize_t) {
  Call c(args);
  const Tensor &q = c.tensor(0), &k = c.tensor(1), &v = c.tensor(2);
  pools_of(c, k, v, 4);
  if (!c.ok || q.dim() != 3 || type_of(q) < 0) Py_RETURN_NONE;
  cv3_paged_attention_params p = {sizeof(p)};
  p.batch = q.size(0), p.heads = q.size(1), p.kv_heads = k.size(1), p.head_dim = k.size(3);
  c.need(q.size(2) == p.head_dim && q.stride(2) == 1 && p.heads > 0 && p.heads % p.kv_heads == 0);
  int* tables = nullptr;
  table_of(c, 3, p.batch, tables, p.table_ld, p.max_blocks);
  p.block_tables = tables;
  p.lens = c.ints(4, p.batch);
  p.window = c.integer(6);
  p.bad = c.ints(9, 1, true);
  c.need(p.window >= 0);
  if (!c.ok) Py_RETURN_NONE;
  p.scale = c.none(5) ? 1.0 / std::sqrt((double)p.head_dim) : c.real(5);
  if (!c.ok) Py_RETURN_NONE;
  Tensor out;
  if (c.none(7)) {
    out = fresh({p.batch, p.heads, p.head_dim}, q.scalar_type(), q);
  } else {
    out = c.tensor(7);
    if (!c.ok || !alike(out, q.sizes(), q.scalar_type())) Py_RETURN_NONE;
  }
  const bool want_lse = args[8] == Py_True;
  if (!want_lse && args[8] != Py_False) Py_RETURN_NONE;
  Tensor lse, ws;
  if (want_lse) {
    lse = fresh({p.batch, p.heads}, at::kFloat, q);
    p.lse = lse.data_ptr<float>();
  }
  p.q = q.data_ptr();
  p.q_type = type_of(q), p.qsb = q.stride(0), p.qsh = q.stride(1);
  p.k_pages = k.data_ptr(), p.v_pages = v.data_ptr();
  p.kv_type = type_of(k);
  p.ksp = k.stride(0), p.ksh = k.stride(1), p.kst = k.stride(2);
  p.vsp = v.stride(0), p.vsh = v.stride(1), p.vst = v.stride(2);
  p.num_pages = k.size(0), p.page_size = k.size(2);
  p.out = out.data_ptr();
  p.osb = p.heads * p.head_dim, p.osh = p.head_dim;
  p.workspace_floats = cv3.attention_workspace(p.batch, p.heads, p.kv_heads, p.head_dim, (int)p.kv_type,
                                               p.max_blocks * p.page_size);
  if (p.workspace_floats) {
    ws = fresh({p.workspace_floats}, at::kFloat, q);
    p.workspace = ws.data_ptr<float>();
  }
  if (cv3.attention(&p, c.stream())) Py_RETURN_NONE;
  PyObject* o = THPVariable_Wrap(out);
  if (!want_lse) return o;
  PyObject* pair = PyTuple_New(2);
  PyTuple_SET_ITEM(pair, 0, o);
  PyTuple_SET_ITEM(pair, 1, THPVariable_Wrap(lse));
  return pair;
}

// (logits, scores, counts, done, stop, min_len, length_penalty)
PyObject* beam(PyObject*, PyObject* const* args, Py_ssize_t) {
  Call c(args);
  const Tensor &x = c.tensor(0), &scores = c.tensor(1), &counts = c.tensor(2), &done = c.tensor(3);
  if (!c.ok || x.dim() != 3 || type_of(x) < 0) Py_RETURN_NONE;
  cv3_beam_params p = {sizeof(p)};
  p.groups = x.size(0), p.beams = x.size(1), p.vocab = x.size(2);
  const int64_t n = p.groups * p.beams, shape[2] = {p.groups, p.beams};
  c.need(n > 0 && p.vocab > 0 && x.stride(2) == 1 && (p.groups == 1 || p.beams == 1 || x.stride(0) == p.beams * x.stride(1)) &&
         alike(scores, shape, at::kFloat) && alike(counts, shape, at::kInt) && alike(done, shape, at::kInt));
  p.min_len = c.ints(5, p.groups, true);
  p.length_penalty = c.real(6);
  if (!c.ok) Py_RETURN_NONE;
  if (!c.none(4)) {
    if (!PyTuple_Check(args[4]) || PyTuple_GET_SIZE(args[4]) != 2) Py_RETURN_NONE;
    Call pair(&PyTuple_GET_ITEM(args[4], 0));
    p.stop_lo = pair.integer(0), p.stop_hi = pair.integer(1);
    if (!pair.ok || p.stop_lo < 0 || p.stop_lo > p.stop_hi || p.stop_hi > p.vocab) Py_RETURN_NONE;
  }
  p.logits = x.data_ptr();
  p.type = type_of(x);
  p.ld = n == 1 ? p.vocab : p.beams > 1 ? x.stride(1) : x.stride(0);
  p.scores = scores.data_ptr<float>(), p.counts = counts.data_ptr<int>(), p.done = done.data_ptr<int>();
  const Tensor tokens = fresh(shape, at::kLong, x), parents = fresh(shape, at::kInt, x), s = fresh(shape, at::kFloat, x),
               cnt = fresh(shape, at::kInt, x), fin = fresh(shape, at::kInt, x);
  p.tokens = tokens.data_ptr<int64_t>(), p.parents = parents.data_ptr<int>(), p.scores_out = s.data_ptr<float>();
  p.counts_out = cnt.data_ptr<int>(), p.done_out = fin.data_ptr<int>();
  p.workspace_bytes = cv3.beam_workspace(p.groups, p.beams, p.vocab);
  Tensor ws;
  if (p.workspace_bytes) {
    ws = fresh({p.workspace_bytes / 8}, at::kLong, x);
    p.workspace = ws.data_ptr();
  }
  if (cv3.beam(&p, c.stream())) Py_RETURN_NONE;
  return made(beam_class, {tokens, parents, s, cnt, fin});
}

// (k_pages, v_pages, block_tables, parents, lens): True when done
PyObject* reorder(PyObject*, PyObject* const* args, Py_ssize_t) {
  Call c(args);
  const Tensor &k = c.tensor(0), &v = c.tensor(1), &parents = c.tensor(3);
  if (!c.ok || (k.dim() != 4 && k.dim() != 5) || parents.dim() != 2) Py_RETURN_NONE;
  const int d = (int)k.dim() - 4;
  pools_of(c, k, v, 4 + d, true);
  cv3_paged_reorder_params p = {sizeof(p)};
  p.groups = parents.size(0), p.beams = parents.size(1);
  const int64_t n = p.groups * p.beams;
  table_of(c, 2, n, p.block_tables, p.table_ld, p.max_blocks);
  p.parents = c.ints(3, n);
  p.lens = c.ints(4, n);
  if (!c.ok) Py_RETURN_NONE;
  p.k_pages = k.data_ptr(), p.v_pages = v.data_ptr();
  p.kv_type = type_of(k);
  p.layers = d ? k.size(0) : 1;
  p.ksl = d ? k.stride(0) : 0, p.vsl = d ? v.stride(0) : 0;
  p.num_pages = k.size(d), p.kv_heads = k.size(d + 1), p.page_size = k.size(d + 2), p.head_dim = k.size(d + 3);
  p.ksp = k.stride(d), p.ksh = k.stride(d + 1), p.kst = k.stride(d + 2);
  p.vsp = v.stride(d), p.vsh = v.stride(d + 1), p.vst = v.stride(d + 2);
  if (cv3.reorder(&p, c.stream())) Py_RETURN_NONE;
  Py_RETURN_TRUE;
}

// An exception of the tensor library (an allocation that fails) ends the short way: the long one meets and reports it.
template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t), int N>
PyObject* guarded(PyObject* self, PyObject* const* args, Py_ssize_t n) {
  if (n != N) {
    PyErr_Format(PyExc_TypeError, "%d arguments expected, got %zd", N, n);
    return nullptr;
  }
  try {
    return F(self, args, n);
  } catch (...) {
    PyErr_Clear();
    Py_RETURN_NONE;
  }
}

// (seven addresses, PagedStep, BeamStep)
PyObject* setup(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 9) {
    PyErr_SetString(PyExc_TypeError, "seven addresses and two classes expected");
    return nullptr;
  }
  void* at[7];
  for (int i = 0; i < 7; ++i) {
    at[i] = PyLong_AsVoidPtr(args[i]);
    if (!at[i]) {
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "null address");
      return nullptr;
    }
  }
  cv3.extend = reinterpret_cast<decltype(cv3.extend)>(at[0]);
  cv3.append = reinterpret_cast<decltype(cv3.append)>(at[1]);
  cv3.attention = reinterpret_cast<decltype(cv3.attention)>(at[2]);
  cv3.attention_workspace = reinterpret_cast<decltype(cv3.attention_workspace)>(at[3]);
  cv3.beam = reinterpret_cast<decltype(cv3.beam)>(at[4]);
  cv3.beam_workspace = reinterpret_cast<decltype(cv3.beam_workspace)>(at[5]);
  cv3.reorder = reinterpret_cast<decltype(cv3.reorder)>(at[6]);
  Py_INCREF(args[7]);
  Py_INCREF(args[8]);
  step_class = args[7];
  beam_class = args[8];
  Py_RETURN_NONE;
}

template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyCFunction fast() {
  return reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(F));
}

PyMethodDef methods[] = {{"setup", fast<setup>(), METH_FASTCALL, nullptr},
                         {"extend", fast<guarded<extend, 8>>(), METH_FASTCALL, nullptr},
                         {"append", fast<guarded<append, 10>>(), METH_FASTCALL, nullptr},
                         {"attention", fast<guarded<attention, 10>>(), METH_FASTCALL, nullptr},
                         {"beam", fast<guarded<beam, 7>>(), METH_FASTCALL, nullptr},
                         {"reorder", fast<guarded<reorder, 5>>(), METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module_def = {PyModuleDef_HEAD_INIT, "_paged_bind", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__paged_bind(void) { return PyModule_Create(&module_def); }
