// Python entries of the tree operators (myinfer_b200.tree): the checks of their
// arguments, their results and workspaces, and the call of the C entry points.
//
// A small call's kernels take 2 us (accepting a path) to 13 us (attention over a
// short cache), so what the host does before them is the call's time: accepting
// took 13.0 us a call with ctypes and takes 6.4-6.9, a commit of 28 layers 11.0 and 7.2-7.8
// (of a table already made), one row of logits 12.7 and 8.2, attention over 512 keys 22.2 and 13.3 (its kernels).
// The kernels and the C ABI are libm5cuda.so's, whose addresses `bind` receives.  Errors
// are ValueError for what a tensor must be, and the library's status through the
// `check` that `bind` receives too.
#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "m5cuda.h"

namespace {

struct {
  decltype(&m5_tree_plan) plan;
  decltype(&m5_tree_attention_workspace) workspace;
  decltype(&m5_tree_attention) attention;
  decltype(&m5_process_logits) logits;
  decltype(&m5_tree_accept) accept;
  decltype(&m5_tree_commit) commit;
  PyObject* check = nullptr;
} fn;

constexpr int64_t kMaxNodes = 64;

struct Unlocked {  // the interpreter's lock is given up while this lives
  PyThreadState* state = PyEval_SaveThread();
  ~Unlocked() { PyEval_RestoreThread(state); }
};

// Runs a C entry point on a device's current stream without the interpreter's lock.
// False: it failed and a Python exception is set.
template <typename F>
bool launch(int dev, F call) {
  TORCH_CHECK(fn.check, "the tree operators are not bound to libm5cuda.so");
  int rc;
  {
    c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(dev));
    void* stream = c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(dev)).stream();
    Unlocked unlocked;
    rc = call(stream);
  }
  if (rc == M5_OK) return true;
  PyObject* r = PyObject_CallFunction(fn.check, "i", rc);  // raises with the library's message
  if (r) {
    Py_DECREF(r);
    PyErr_Format(PyExc_RuntimeError, "libm5cuda status %d", rc);
  }
  return false;
}

const at::Tensor& tensor(PyObject* o, const char* what) {
  TORCH_CHECK_VALUE(THPVariable_Check(o), what, " must be a tensor");
  return THPVariable_Unpack(o);
}

// Pointer of a contiguous tensor of this shape and type on device `dev`.
void* whole(PyObject* o, at::IntArrayRef shape, const char* what, int dev, at::ScalarType type = at::kInt) {
  const at::Tensor& t = tensor(o, what);
  TORCH_CHECK_VALUE(t.scalar_type() == type && t.sizes() == shape && t.is_cuda() && t.get_device() == dev && t.is_contiguous(),
                    what, " must be a contiguous ", type, " tensor of shape ", shape, " on cuda:", dev);
  return t.data_ptr();
}

int64_t integer(PyObject* o) {
  PyObject* n = PyNumber_Long(o);
  if (!n) throw python_error();
  const int64_t v = PyLong_AsLongLong(n);
  Py_DECREF(n);
  if (v == -1 && PyErr_Occurred()) throw python_error();
  return v;
}

void expect(Py_ssize_t got, Py_ssize_t want) {
  TORCH_CHECK_TYPE(got == want, "expected ", want, " arguments, got ", got);
}

// An uninitialised tensor on a device, past the operator dispatch (0.3 us of a call each).
at::Tensor empty(at::IntArrayRef shape, at::ScalarType type, int dev) {
  return at::detail::empty_cuda(shape, type, c10::Device(c10::DeviceType::CUDA, static_cast<c10::DeviceIndex>(dev)), std::nullopt);
}

const at::Tensor& trees(PyObject* o) {
  const at::Tensor& t = tensor(o, "parents");
  TORCH_CHECK_VALUE(t.dim() == 2 && t.scalar_type() == at::kInt && t.is_cuda() && t.is_contiguous(),
                    "parents must be a contiguous int32 CUDA tensor [batch, nodes]");
  TORCH_CHECK_VALUE(t.size(1) >= 1 && t.size(1) <= kMaxNodes, "a tree has 1 to ", kMaxNodes, " nodes, got ", t.size(1));
  return t;
}

int small(int64_t v) {
  TORCH_CHECK_VALUE(v >= 0 && v <= INT32_MAX, "dimension ", v, " is out of range");
  return static_cast<int>(v);
}

PyObject* result(std::initializer_list<at::Tensor> ts) {
  PyObject* r = PyTuple_New(ts.size());
  if (!r) throw python_error();
  Py_ssize_t i = 0;
  for (const at::Tensor& t : ts) PyTuple_SET_ITEM(r, i++, THPVariable_Wrap(t));
  return r;
}

// bind([addresses, in the order of `fn`], check)
PyObject* bind(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  expect(n, 7);
  void* p[6];
  for (int i = 0; i < 6; ++i) {
    p[i] = PyLong_AsVoidPtr(args[i]);
    if (!p[i]) {
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "null entry point");
      return nullptr;
    }
  }
  fn.plan = reinterpret_cast<decltype(fn.plan)>(p[0]);
  fn.workspace = reinterpret_cast<decltype(fn.workspace)>(p[1]);
  fn.attention = reinterpret_cast<decltype(fn.attention)>(p[2]);
  fn.logits = reinterpret_cast<decltype(fn.logits)>(p[3]);
  fn.accept = reinterpret_cast<decltype(fn.accept)>(p[4]);
  fn.commit = reinterpret_cast<decltype(fn.commit)>(p[5]);
  Py_INCREF(args[6]);
  Py_XDECREF(fn.check);
  fn.check = args[6];
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

// plan(parents)
PyObject* plan(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  expect(n, 1);
  const at::Tensor& parents = trees(args[0]);
  const int B = small(parents.size(0)), T = small(parents.size(1)), dev = parents.get_device();
  at::Tensor anc = empty({B, T}, at::kLong, dev), depth = empty({B, T}, at::kInt, dev);
  if (!launch(dev, [&](void* st) {
        return fn.plan((const int32_t*)parents.data_ptr(), B, T, (int64_t*)anc.data_ptr(), (int32_t*)depth.data_ptr(), st);
      }))
    return nullptr;
  return result({anc, depth});
  END_HANDLE_TH_ERRORS
}

// A K or V operand over the whole cache: its view, and [batch, kv heads, rows].
m5_kv_view kv_view(PyObject* o, int bits, int64_t D, int dev, const char* what, int64_t (&shape)[3]) {
  const at::Tensor *data, *sc[2] = {nullptr, nullptr};
  if (bits) {
    const bool three = (PyTuple_Check(o) || PyList_Check(o)) && PySequence_Fast_GET_SIZE(o) == 3;
    TORCH_CHECK_VALUE(three, what, " of a quantized cache are (wq, scales, biases)");
    data = &tensor(PySequence_Fast_GET_ITEM(o, 0), what);
    for (int i = 0; i < 2; ++i) sc[i] = &tensor(PySequence_Fast_GET_ITEM(o, i + 1), what);
  } else {
    TORCH_CHECK_VALUE(THPVariable_Check(o), what, " of an unquantized cache are one bf16 tensor");
    data = &THPVariable_Unpack(o);
  }
  const int64_t width = bits ? D * bits / 32 : D;
  const auto type = bits ? at::kInt : at::kBFloat16;
  TORCH_CHECK_VALUE(data->dim() == 4 && data->scalar_type() == type && data->size(3) == width && data->is_cuda() &&
                        data->get_device() == dev,
                    what, " must be ", type, " [batch, kv heads, rows, ", width, "] on cuda:", dev);
  const auto size = data->sizes();
  // a dimension of size 1 may have any stride: it is never stepped over
  const int64_t sb = size[0] == 1 ? 0 : data->stride(0), sh = size[1] == 1 ? 0 : data->stride(1);
  TORCH_CHECK_VALUE((data->stride(3) == 1 || width == 1) && (size[2] == 1 || data->stride(2) == width) && sh % width == 0 &&
                        sb % width == 0,
                    what, ": a head's rows must be contiguous");
  for (int i = 0; i < 3; ++i) shape[i] = size[i];
  m5_kv_view v{data->data_ptr(), nullptr, nullptr, sb / width, sh / width};
  if (!bits) return v;
  const int64_t G = D / 64, want[4] = {size[0], size[1], size[2], G}, lay[4] = {v.batch_stride * G, v.head_stride * G, G, 1};
  for (const at::Tensor* x : sc) {
    TORCH_CHECK_VALUE(x->scalar_type() == at::kBFloat16 && x->sizes() == at::IntArrayRef(want) && x->is_cuda() &&
                          x->get_device() == dev,
                      what, ": scales and biases must be bf16 [batch, kv heads, rows, ", G, "] on cuda:", dev);
    for (int i = 0; i < 4; ++i)
      TORCH_CHECK_VALUE(want[i] == 1 || x->stride(i) == lay[i], what, ": scales and biases must be laid out like the rows");
  }
  v.scales = sc[0]->data_ptr();
  v.biases = sc[1]->data_ptr();
  return v;
}

struct Strides {
  int64_t s[3];
  explicit Strides(const at::Tensor& t) {
    for (int i = 0; i < 3; ++i) s[i] = t.size(i) == 1 ? 0 : t.stride(i);
  }
  bool aligned() const { return (s[0] | s[1] | s[2]) % 8 == 0; }
};
bool on16(const at::Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; }

// attention(queries, keys, values, lengths, ancestors, scale, tree_len or None, group_size, bits, out or None)
PyObject* attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  expect(n, 10);
  at::Tensor q = tensor(args[0], "queries");
  TORCH_CHECK_VALUE(q.dim() == 4 && q.scalar_type() == at::kBFloat16 && q.is_cuda(),
                    "queries must be bf16 CUDA [batch, heads, nodes, dim]");
  const int64_t B = q.size(0), Hq = q.size(1), L = q.size(2), D = q.size(3), T = args[6] == Py_None ? L : integer(args[6]);
  const int dev = q.get_device();
  TORCH_CHECK_VALUE(D == 64 || D == 128, "head_dim must be 64 or 128, got ", D);
  TORCH_CHECK_VALUE(L >= 1 && L <= kMaxNodes && T >= 1 && T <= kMaxNodes, "a tree has 1 to ", kMaxNodes, " nodes, got ", L,
                    " queries and ", T, " tree keys");
  const int64_t bits = integer(args[8]), group = integer(args[7]);
  TORCH_CHECK_VALUE((bits == 0 || bits == 4 || bits == 8) && (bits == 0 || group == 64),
                    "tree_attention supports bits 4/8 with group_size 64, or bits 0 (bf16)");
  int64_t shape[3], vshape[3];
  const m5_kv_view k = kv_view(args[1], bits, D, dev, "keys", shape), v = kv_view(args[2], bits, D, dev, "values", vshape);
  TORCH_CHECK_VALUE(at::IntArrayRef(shape) == at::IntArrayRef(vshape) && shape[0] == B, "keys ", at::IntArrayRef(shape),
                    " and values ", at::IntArrayRef(vshape), " must agree and have batch ", B);
  const int64_t Hkv = shape[1], rows = shape[2];
  TORCH_CHECK_VALUE(Hkv > 0 && Hq % Hkv == 0, "number of query heads must be a multiple of kv heads");
  const auto* lengths = (const int32_t*)whole(args[3], {B}, "lengths", dev);
  const auto* anc = (const int64_t*)whole(args[4], {B, L}, "ancestors", dev, at::kLong);
  const double scale = PyFloat_AsDouble(args[5]);
  if (scale == -1.0 && PyErr_Occurred()) return nullptr;
  Strides qs(q);
  if (q.stride(3) != 1 || !qs.aligned() || !on16(q)) {
    q = q.contiguous();
    if (!on16(q)) q = q.clone();
    qs = Strides(q);
  }
  at::Tensor out;
  if (args[9] == Py_None) {
    out = empty({B, Hq, L, D}, at::kBFloat16, dev);
  } else {
    out = tensor(args[9], "out");
    TORCH_CHECK_VALUE(out.dim() == 4 && out.scalar_type() == at::kBFloat16 && out.sizes() == q.sizes() && out.is_cuda() &&
                          out.get_device() == dev && out.stride(3) == 1,
                      "out must be bf16 of the queries' shape with contiguous dims");
  }
  const Strides os(out);
  at::Tensor ws;  // from the stream's own pool: calls on other streams never share it
  if (!launch(dev, [&](void* st) {
        size_t need = 0;
        if (int rc = fn.workspace(small(B), small(Hq), small(Hkv), small(L), small(D), &need)) return rc;
        ws = empty({(int64_t)need}, at::kByte, dev);
        return fn.attention(q.data_ptr(), qs.s, small(B), small(Hq), small(L), small(D), k, v, small(Hkv), rows, lengths,
                            small(T), anc, L, (float)scale, (int)group, (int)bits, out.data_ptr(), os.s, ws.data_ptr(), need, st);
      }))
    return nullptr;
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

// logits(logits, batch, counts, penalties, tokens, ancestors, bias_ids, bias_values, mask, out), all but the first or None
PyObject* logits(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  expect(n, 10);
  const at::Tensor& x = tensor(args[0], "logits");
  TORCH_CHECK_VALUE(x.dim() == 2 && (x.scalar_type() == at::kBFloat16 || x.scalar_type() == at::kFloat) && x.is_cuda(),
                    "logits must be bf16 or fp32 CUDA [rows, vocab]");
  const bool have_batch = args[1] != Py_None, counts = args[2] != Py_None, pen = args[3] != Py_None, toks = args[4] != Py_None,
             ids = args[6] != Py_None;
  const int64_t R = x.size(0), V = x.size(1), B = have_batch ? integer(args[1]) : R;
  const int dev = x.get_device();
  TORCH_CHECK_VALUE(B >= 1 && R % B == 0, R, " logits rows are no multiple of batch ", B);
  const int64_t T = R / B;
  TORCH_CHECK_VALUE(T <= kMaxNodes, "a tree has 1 to ", kMaxNodes, " nodes, got ", T);
  TORCH_CHECK_VALUE(x.stride(1) == 1 || V == 1, "logits rows must be contiguous");
  at::Tensor out;
  if (args[9] == Py_None) {
    out = empty({R, V}, x.scalar_type(), dev);
  } else {
    out = tensor(args[9], "out");
    TORCH_CHECK_VALUE(out.sizes() == x.sizes() && out.scalar_type() == x.scalar_type() && out.device() == x.device() &&
                          (out.stride(1) == 1 || V == 1),
                      "out must have the logits' shape and type, with contiguous rows");
  }
  TORCH_CHECK_VALUE(pen || !(counts || toks), "counts and tokens need penalties");
  TORCH_CHECK_VALUE(toks == (args[5] != Py_None) && ids == (args[7] != Py_None),
                    "tokens come with ancestors, and bias_ids with bias_values");
  const void* cp = counts ? whole(args[2], {B, V}, "counts", dev) : nullptr;
  const void* pp = pen ? whole(args[3], {B, 3}, "penalties", dev, at::kFloat) : nullptr;
  const void* tp = toks ? whole(args[4], {B, T}, "tokens", dev) : nullptr;
  const void* ap = toks ? whole(args[5], {B, T}, "ancestors", dev, at::kLong) : nullptr;
  auto last = [](PyObject* o, const char* what) {
    const at::Tensor& t = tensor(o, what);
    return t.dim() ? t.size(t.dim() - 1) : int64_t(0);
  };
  int64_t nb = 0, mld = 0;
  const void *ip = nullptr, *vp = nullptr, *mp = nullptr;
  if (ids) {
    nb = last(args[6], "bias_ids");
    ip = whole(args[6], {B, nb}, "bias_ids", dev);
    vp = whole(args[7], {B, nb}, "bias_values", dev, at::kFloat);
  }
  if (args[8] != Py_None) {
    mld = last(args[8], "mask");
    mp = whole(args[8], {R, mld}, "mask", dev);
  }
  at::Tensor choices = empty({R}, at::kInt, dev);
  // a single row's stride is meaningless (torch keeps any stride on a size-1 dimension)
  const int64_t ld = R > 1 ? x.stride(0) : V, old = R > 1 ? out.stride(0) : V;
  const int dt = x.scalar_type() == at::kBFloat16 ? M5_DTYPE_BF16 : M5_DTYPE_F32;
  if (!launch(dev, [&](void* st) {
        return fn.logits(x.data_ptr(), ld, out.data_ptr(), old, dt, small(B), small(T), V, (const int32_t*)cp, V,
                         (const float*)pp, (const int32_t*)tp, (const int64_t*)ap, (const int32_t*)ip, (const float*)vp,
                         small(nb), (const int32_t*)mp, mld, (int32_t*)choices.data_ptr(), st);
      }))
    return nullptr;
  return result({out, choices});
  END_HANDLE_TH_ERRORS
}

// accept(parents, tokens, picks, counts or None)
PyObject* accept(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  expect(n, 4);
  const at::Tensor& parents = trees(args[0]);
  const int64_t B = parents.size(0), T = parents.size(1);
  const int dev = parents.get_device();
  const auto* tp = (const int32_t*)whole(args[1], {B, T}, "tokens", dev);
  const auto* pp = (const int32_t*)whole(args[2], {B, T}, "picks", dev);
  int32_t* cp = nullptr;
  int64_t V = 0;
  if (args[3] != Py_None) {
    const at::Tensor& counts = tensor(args[3], "counts");
    TORCH_CHECK_VALUE(counts.dim() == 2, "counts must be int32 [batch, vocab]");
    V = counts.size(1);
    cp = (int32_t*)whole(args[3], {B, V}, "counts", dev);
  }
  at::Tensor path = empty({B, T}, at::kInt, dev), count = empty({B}, at::kInt, dev),
             next = empty({B}, at::kInt, dev);
  if (!launch(dev, [&](void* st) {
        return fn.accept((const int32_t*)parents.data_ptr(), tp, pp, small(B), small(T), (int32_t*)path.data_ptr(),
                         (int32_t*)count.data_ptr(), (int32_t*)next.data_ptr(), cp, V, V, st);
      }))
    return nullptr;
  return result({path, count, next});
  END_HANDLE_TH_ERRORS
}

// commit(address of the layers' table, layers, batch, kv heads, head_dim, device, lengths, path, accepted)
PyObject* commit(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  expect(n, 9);
  const auto* layers = static_cast<const m5_layer_kv*>(PyLong_AsVoidPtr(args[0]));
  if (!layers && PyErr_Occurred()) return nullptr;
  const int64_t count = integer(args[1]), B = integer(args[2]), H = integer(args[3]), D = integer(args[4]);
  const int dev = (int)integer(args[5]);
  const at::Tensor& path = tensor(args[7], "path");
  TORCH_CHECK_VALUE(path.dim() == 2 && path.size(0) == B && path.size(1) >= 1 && path.size(1) <= kMaxNodes,
                    "path must be int32 [", B, ", 1 to ", kMaxNodes, " nodes]");
  const int64_t T = path.size(1);
  const auto* lengths = (const int32_t*)whole(args[6], {B}, "lengths", dev);
  const auto* pp = (const int32_t*)whole(args[7], {B, T}, "path", dev);
  const auto* ap = (const int32_t*)whole(args[8], {B}, "accepted", dev);
  if (!launch(dev, [&](void* st) {
        return fn.commit(layers, small(count), small(B), small(H), small(D), lengths, pp, small(T), ap, st);
      }))
    return nullptr;
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

#define M5_METHOD(f) {#f, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {M5_METHOD(bind),   M5_METHOD(plan),   M5_METHOD(attention), M5_METHOD(logits),
                         M5_METHOD(accept), M5_METHOD(commit), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_tree_binding", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__tree_binding() { return PyModule_Create(&module); }
