// Native side of the Python binding: the calls a decode step or a prompt chunk makes by the dozen.
//
// A ctypes call through the public C ABI costs about 14 us of host time in Python (a dozen argument conversions, the
// stream lookup through torch.cuda, torch.empty per output), more than most decode kernels run: a layer of a small model
// (eight calls) took 114 us on the host and 35 us on the GPU.  Here a call takes the tensors as they are, reads pointers
// and strides from them, allocates its outputs from torch's caching allocator and calls the same C entry point with the
// current stream: about 1 us beside the launch itself.
//
// The module holds no state but the entry points' addresses: bind() receives them from the loaded libizb200.so, so the
// one library (also a build named by IZB200_LIB) serves both the ctypes and the native calls.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/izb200.h"

namespace {

#define IZB_PY_CALLS(X) \
  X(izb_quantize_act) X(izb_swiglu_quant) X(izb_rmsnorm_quant) X(izb_add_norm_quant) X(izb_softcap_rows) X(izb_matmul) X(izb_quant_matmul) \
  X(izb_gemv) X(izb_gemm) X(izb_moe_route_ex) X(izb_moe_sort_ex) X(izb_moe_gateup) X(izb_moe_down) X(izb_moe_combine_ex) \
  X(izb_moe_layer) X(izb_moe_layer_scratch) X(izb_lora_add) X(izb_lora_scratch) X(izb_logits_process)

struct Calls {
#define X(name) decltype(&name) name##_ = nullptr;
  IZB_PY_CALLS(X)
#undef X
} g;
PyObject* g_fail = nullptr;     // Python callable(status): raises
PyObject* g_address = nullptr;  // Python callable(object): the address of what is no torch tensor (a numpy array over pinned memory, ...)

// ---- arguments
const at::Tensor& tensor(PyObject* o) {
  if (!THPVariable_Check(o)) throw torch::TypeError(std::string("expected a torch tensor, got ") + Py_TYPE(o)->tp_name);
  return THPVariable_Unpack(o);
}
template <class T>
T* ptr(PyObject* o) {  // None = NULL
  if (o == Py_None) return nullptr;
  if (THPVariable_Check(o)) return static_cast<T*>(THPVariable_Unpack(o).data_ptr());
  PyObject* v = PyObject_CallOneArg(g_address, o);
  if (!v) throw python_error();
  void* p = PyLong_AsVoidPtr(v);
  Py_DECREF(v);
  if (!p && PyErr_Occurred()) throw python_error();
  return static_cast<T*>(p);
}
int extent(PyObject* o, int d) {  // o.shape[d]
  if (THPVariable_Check(o)) return (int)THPVariable_Unpack(o).size(d);
  PyObject* shape = PyObject_GetAttrString(o, "shape");
  PyObject* v = shape ? PySequence_GetItem(shape, d) : nullptr;
  Py_XDECREF(shape);
  if (!v) throw python_error();
  const long n = PyLong_AsLong(v);
  Py_DECREF(v);
  if (n == -1 && PyErr_Occurred()) throw python_error();
  return (int)n;
}
// rows and columns, as `rows, columns = x.shape` unpacks them: other numbers of dimensions are a ValueError
const at::Tensor& matrix(PyObject* o) {
  const at::Tensor& t = tensor(o);
  TORCH_CHECK_VALUE(t.dim() == 2, "expected two dimensions, got ", t.dim());
  return t;
}
int num(PyObject* o) {
  const long v = PyLong_AsLong(o);
  if (v == -1 && PyErr_Occurred()) throw python_error();
  if (v != (int)v) throw torch::TypeError("integer argument out of range: " + std::to_string(v));
  return (int)v;
}
float real(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw python_error();
  return (float)v;
}
izb_weight* weight(PyObject* o) {  // the handle's address, None = NULL
  if (o == Py_None) return nullptr;
  void* p = PyLong_AsVoidPtr(o);
  if (!p && PyErr_Occurred()) throw python_error();
  return static_cast<izb_weight*>(p);
}
void count(Py_ssize_t n, Py_ssize_t want) {
  if (n != want) throw torch::TypeError(std::to_string(n) + " arguments, " + std::to_string(want) + " expected");
}

at::Tensor empty(std::initializer_list<int64_t> size, at::ScalarType type, c10::Device dev) {
  if (dev.is_cuda()) return at::detail::empty_cuda(at::IntArrayRef(size), type, dev, std::nullopt);
  return at::empty(at::IntArrayRef(size), at::TensorOptions().dtype(type).device(dev));
}
// rows of the reference engine's padding (zero/engine.h:521-522)
int pad_rows(int m) { return m >= 128 ? (m + 127) / 128 * 128 : (m + 15) / 16 * 16; }
int rows_or_pad(PyObject* o, int64_t m) {
  const int v = o == Py_None ? 0 : num(o);
  return v ? v : pad_rows((int)m);
}

// ---- the call itself: without the interpreter lock, on the current stream of the current device
template <class F, class... A>
void call(F f, A... args) {
  void* st = c10::cuda::getCurrentCUDAStream().stream();
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = f(args..., st);
  Py_END_ALLOW_THREADS
  if (rc != 0) {
    PyObject* r = PyObject_CallFunction(g_fail, "i", rc);
    Py_XDECREF(r);
    if (!PyErr_Occurred()) PyErr_Format(PyExc_RuntimeError, "izb200 status %d", rc);
    throw python_error();
  }
}

PyObject* own(PyObject* o) { Py_INCREF(o); return o; }
PyObject* wrap(at::Tensor t) { return THPVariable_Wrap(std::move(t)); }
PyObject* tuple(std::initializer_list<PyObject*> items) {  // takes the references over
  PyObject* t = PyTuple_New((Py_ssize_t)items.size());
  Py_ssize_t i = 0;
  for (PyObject* o : items) PyTuple_SET_ITEM(t, i++, o);
  return t;
}

struct Quantised {
  at::Tensor aq, asc;
  // (one allocation for both: an allocator round trip is half a microsecond of a call's four)
  Quantised(int Mp, int64_t K, c10::Device dev) {
    const int64_t q_bytes = (Mp * K + 15) / 16 * 16;
    const at::Tensor both = empty({q_bytes + K / 32 * Mp * 4}, at::kByte, dev);
    auto part = [&](caffe2::TypeMeta type, int64_t rows, int64_t cols, int64_t first) {
      at::Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(both.storage()), both.key_set(), type);
      t.unsafeGetTensorImpl()->set_storage_offset(first);
      t.unsafeGetTensorImpl()->set_sizes_contiguous({rows, cols});
      return t;
    };
    aq = part(caffe2::TypeMeta::Make<int8_t>(), Mp, K, 0);
    asc = part(caffe2::TypeMeta::Make<float>(), K / 32, Mp, q_bytes / 4);
  }
  int8_t* q() { return static_cast<int8_t*>(aq.data_ptr()); }
  float* s() { return static_cast<float*>(asc.data_ptr()); }
};

#define FN(name) PyObject* name(PyObject*, PyObject* const* a, Py_ssize_t n)

// (x, Mp, want_absum, aq, asc, absum): aq None = allocate
FN(quantize_act) {
  HANDLE_TH_ERRORS
  count(n, 6);
  const at::Tensor& x = matrix(a[0]);
  const int M = (int)x.size(0), K = (int)x.size(1), Mp = rows_or_pad(a[1], M);
  if (a[3] != Py_None) {
    call(g.izb_quantize_act_, ptr<float>(a[0]), (int)x.stride(0), M, Mp, K, ptr<int8_t>(a[3]), ptr<float>(a[4]), ptr<int16_t>(a[5]));
    return tuple({own(a[3]), own(a[4]), own(a[5])});
  }
  Quantised o(Mp, K, x.device());
  at::Tensor sums;
  if (PyObject_IsTrue(a[2])) sums = empty({K / 16, Mp}, at::kShort, x.device());
  int16_t* ps = sums.defined() ? static_cast<int16_t*>(sums.data_ptr()) : nullptr;
  call(g.izb_quantize_act_, ptr<float>(a[0]), (int)x.stride(0), M, Mp, K, o.q(), o.s(), ps);
  return tuple({wrap(o.aq), wrap(o.asc), ps ? wrap(sums) : own(Py_None)});
  END_HANDLE_TH_ERRORS
}

// (gu, F, Mp, want_h)
FN(swiglu_quant) {
  HANDLE_TH_ERRORS
  count(n, 4);
  const at::Tensor& gu = tensor(a[0]);
  const int M = (int)gu.size(0), F = num(a[1]), Mp = rows_or_pad(a[2], M);
  Quantised o(Mp, F, gu.device());
  at::Tensor h;
  if (PyObject_IsTrue(a[3])) h = empty({M, F}, at::kFloat, gu.device());
  float* ph = h.defined() ? static_cast<float*>(h.data_ptr()) : nullptr;
  call(g.izb_swiglu_quant_, ptr<float>(a[0]), (int)gu.stride(0), 1, M, Mp, F, ph, o.q(), o.s(), nullptr);
  return tuple({wrap(o.aq), wrap(o.asc), ph ? wrap(h) : own(Py_None)});
  END_HANDLE_TH_ERRORS
}

// (x, w, eps, Mp, want_h)
FN(rmsnorm_quant) {
  HANDLE_TH_ERRORS
  count(n, 5);
  const at::Tensor& x = matrix(a[0]);
  const int M = (int)x.size(0), K = (int)x.size(1), Mp = rows_or_pad(a[3], M);
  const float eps = real(a[2]);
  Quantised o(Mp, K, x.device());
  at::Tensor h;
  if (PyObject_IsTrue(a[4])) h = empty({M, K}, at::kFloat, x.device());
  float* ph = h.defined() ? static_cast<float*>(h.data_ptr()) : nullptr;
  call(g.izb_rmsnorm_quant_, ptr<float>(a[0]), (int)x.stride(0), ptr<float>(a[1]), eps, M, Mp, K, ph, o.q(), o.s(), nullptr);
  return tuple({wrap(o.aq), wrap(o.asc), ph ? wrap(h) : own(Py_None)});
  END_HANDLE_TH_ERRORS
}

// (x, t, w, eps, s, w2, Mp)
FN(add_norm_quant) {
  HANDLE_TH_ERRORS
  count(n, 7);
  const at::Tensor& x = matrix(a[0]);
  const int M = (int)x.size(0), K = (int)x.size(1), Mp = rows_or_pad(a[6], M);
  const float eps = real(a[3]), s = real(a[4]);
  Quantised o(Mp, K, x.device());
  call(g.izb_add_norm_quant_, ptr<float>(a[0]), ptr<float>(a[1]), ptr<float>(a[2]), eps, s, ptr<float>(a[5]), M, Mp, K, o.q(), o.s(), nullptr);
  return tuple({wrap(o.aq), wrap(o.asc)});
  END_HANDLE_TH_ERRORS
}

// (c, rows, N, cap, off)
FN(softcap_rows) {
  HANDLE_TH_ERRORS
  count(n, 5);
  const at::Tensor& c = tensor(a[0]);
  const int rows = num(a[1]), N = num(a[2]), off = num(a[4]);
  const float cap = real(a[3]);
  call(g.izb_softcap_rows_, ptr<float>(a[0]), rows, (int)c.stride(0), off, N, cap);
  return own(a[0]);
  END_HANDLE_TH_ERRORS
}

// the output of a product: the caller's, or a new one of `rows` x `cols`
struct Out {
  at::Tensor made;
  PyObject* given;
  float* p;
  int ld;
  Out(PyObject* o, int rows, int cols, PyObject* like) : given(o) {  // (`like`: on whose device)
    if (o == Py_None) {
      made = empty({rows, cols}, at::kFloat, tensor(like).device());
      p = static_cast<float*>(made.data_ptr());
      ld = cols;
    } else {
      const at::Tensor& t = tensor(o);
      p = static_cast<float*>(t.data_ptr());
      ld = (int)t.stride(0);
    }
  }
  PyObject* result() { return given == Py_None ? wrap(made) : own(given); }
};

// (weight, N, mat, aq, asc, T, out, c_off, acc)
FN(matmul) {
  HANDLE_TH_ERRORS
  count(n, 9);
  izb_weight* w = weight(a[0]);
  const int mat = num(a[2]), T = num(a[5]), c_off = num(a[7]), acc = num(a[8]), Mp = extent(a[4], 1);
  Out o(a[6], Mp, num(a[1]), a[3]);
  call(g.izb_matmul_, w, mat, ptr<int8_t>(a[3]), ptr<float>(a[4]), nullptr, T, Mp, o.p, o.ld, c_off, acc);
  return o.result();
  END_HANDLE_TH_ERRORS
}

// (weight, N_out, K, x, T, Mp, out, c_off, acc, mat, aq, asc): aq None = allocate
FN(quant_matmul) {
  HANDLE_TH_ERRORS
  count(n, 12);
  izb_weight* w = weight(a[0]);
  const at::Tensor& x = tensor(a[3]);
  const int K = num(a[2]), T = num(a[4]), Mp = rows_or_pad(a[5], T), c_off = num(a[7]), acc = num(a[8]), mat = num(a[9]);
  at::Tensor aq, asc;
  if (a[10] == Py_None) {
    Quantised q(Mp, K, x.device());
    aq = q.aq;
    asc = q.asc;
  }
  Out o(a[6], Mp, num(a[1]), a[3]);
  int8_t* pq = aq.defined() ? static_cast<int8_t*>(aq.data_ptr()) : ptr<int8_t>(a[10]);
  float* ps = asc.defined() ? static_cast<float*>(asc.data_ptr()) : ptr<float>(a[11]);
  call(g.izb_quant_matmul_, w, mat, ptr<float>(a[3]), (int)x.stride(0), T, Mp, pq, ps, o.p, o.ld, c_off, acc);
  return tuple({o.result(), a[10] == Py_None ? wrap(aq) : own(a[10]), a[10] == Py_None ? wrap(asc) : own(a[11])});
  END_HANDLE_TH_ERRORS
}

// (weight, N, mat, aq, asc, T, out, c_off, acc)
FN(gemv) {
  HANDLE_TH_ERRORS
  count(n, 9);
  izb_weight* w = weight(a[0]);
  const int mat = num(a[2]), T = num(a[5]), c_off = num(a[7]), acc = num(a[8]), Mp = extent(a[4], 1);
  Out o(a[6], T, num(a[1]), a[3]);
  call(g.izb_gemv_, w, mat, ptr<int8_t>(a[3]), ptr<float>(a[4]), T, Mp, o.p, o.ld, c_off, acc);
  return o.result();
  END_HANDLE_TH_ERRORS
}

// (weight, N_out, mat, aq, asc, M, out, c_off, acc, impl): M 0 = all padded rows
FN(gemm) {
  HANDLE_TH_ERRORS
  count(n, 10);
  izb_weight* w = weight(a[0]);
  const int mat = num(a[2]), c_off = num(a[7]), acc = num(a[8]), impl = num(a[9]), Mp = extent(a[4], 1);
  const int m = a[5] == Py_None ? 0 : num(a[5]), M = m ? m : Mp;
  Out o(a[6], Mp, num(a[1]), a[3]);
  call(g.izb_gemm_, w, mat, ptr<int8_t>(a[3]), ptr<float>(a[4]), M, Mp, o.p, o.ld, c_off, acc, impl);
  return o.result();
  END_HANDLE_TH_ERRORS
}

// (logits, NU, shared_gate)
FN(moe_route) {
  HANDLE_TH_ERRORS
  count(n, 3);
  const at::Tensor& l = tensor(a[0]);
  const bool shared = PyObject_IsTrue(a[2]);
  const int T = (int)l.size(0), NE = (int)l.size(1) - (shared ? 1 : 0), NU = num(a[1]);
  const c10::Device dev = l.device();
  at::Tensor ids = empty({T, NU}, at::kInt, dev), wts = empty({T, NU}, at::kFloat, dev), counts = empty({NE}, at::kInt, dev), gate;
  if (shared) gate = empty({T}, at::kFloat, dev);
  float* pg = shared ? static_cast<float*>(gate.data_ptr()) : nullptr;
  call(g.izb_moe_route_ex_, ptr<float>(a[0]), (int)l.stride(0), T, NE, NU, static_cast<int32_t*>(ids.data_ptr()), static_cast<float*>(wts.data_ptr()),
                               static_cast<int32_t*>(counts.data_ptr()), pg);
  if (shared) return tuple({wrap(ids), wrap(wts), wrap(counts), wrap(gate)});
  return tuple({wrap(ids), wrap(wts), wrap(counts)});
  END_HANDLE_TH_ERRORS
}

// (ids, wts, counts, TM, e0, e1)
FN(moe_sort) {
  HANDLE_TH_ERRORS
  count(n, 6);
  const at::Tensor& ids = matrix(a[0]);
  const c10::Device dev = ids.device();
  const int T = (int)ids.size(0), NU = (int)ids.size(1), NE = extent(a[2], 0), TM = num(a[3]), e0 = num(a[4]), e1 = num(a[5]);
  const int S = T * NU, max_tiles = (TM > 0 ? (S + TM - 1) / TM : 0) + NE;
  at::Tensor offs = empty({NE + 1}, at::kInt, dev), tiles = empty({1 + 3 * (int64_t)max_tiles}, at::kInt, dev), stok = empty({S}, at::kInt, dev),
             swt = empty({S}, at::kFloat, dev), inv = empty({S}, at::kInt, dev);
  auto pi = [](at::Tensor& t) { return static_cast<int32_t*>(t.data_ptr()); };
  call(g.izb_moe_sort_ex_, ptr<int32_t>(a[0]), ptr<float>(a[1]), ptr<int32_t>(a[2]), T, NE, NU, TM, e0, e1, pi(offs), pi(tiles), max_tiles, pi(stok),
                              static_cast<float*>(swt.data_ptr()), pi(inv));
  return tuple({wrap(offs), wrap(tiles), PyLong_FromLong(max_tiles), wrap(stok), wrap(swt), wrap(inv)});
  END_HANDLE_TH_ERRORS
}

// (wg, wu, N_out, aq, asc, tiles, max_tiles, TM, stok, S)
FN(moe_gateup) {
  HANDLE_TH_ERRORS
  count(n, 10);
  izb_weight *wg = weight(a[0]), *wu = weight(a[1]);
  const int N = num(a[2]), Mp = extent(a[4], 1), max_tiles = num(a[6]), TM = num(a[7]), S = num(a[9]);
  at::Tensor h = empty({S, N}, at::kFloat, tensor(a[3]).device());
  float* ph = static_cast<float*>(h.data_ptr());
  call(g.izb_moe_gateup_, wg, wu, ptr<int8_t>(a[3]), ptr<float>(a[4]), Mp, ptr<int32_t>(a[5]), max_tiles, TM, ptr<int32_t>(a[8]), ph);
  return wrap(h);
  END_HANDLE_TH_ERRORS
}

// (wd, N, hq, hsc, tiles, max_tiles, TM, swt, S)
FN(moe_down) {
  HANDLE_TH_ERRORS
  count(n, 9);
  izb_weight* w = weight(a[0]);
  const int N = num(a[1]), Sp = extent(a[3], 1), max_tiles = num(a[5]), TM = num(a[6]), S = num(a[8]);
  at::Tensor y = empty({S, N}, at::kFloat, tensor(a[2]).device());
  float* py = static_cast<float*>(y.data_ptr());
  call(g.izb_moe_down_, w, ptr<int8_t>(a[2]), ptr<float>(a[3]), Sp, ptr<int32_t>(a[4]), max_tiles, TM, ptr<float>(a[7]), py);
  return wrap(y);
  END_HANDLE_TH_ERRORS
}

// (x, y, inv, NU, sh, sgate, partial)
FN(moe_combine) {
  HANDLE_TH_ERRORS
  count(n, 7);
  const at::Tensor& x = matrix(a[0]);
  const int T = (int)x.size(0), E = (int)x.size(1), NU = num(a[3]), partial = PyObject_IsTrue(a[6]) ? 1 : 0;
  call(g.izb_moe_combine_ex_, ptr<float>(a[0]), ptr<float>(a[1]), ptr<int32_t>(a[2]), T, NU, E, ptr<float>(a[4]), ptr<float>(a[5]), partial);
  return own(a[0]);
  END_HANDLE_TH_ERRORS
}

// ---- calls that check their tensors: on the current device, of the type, the number of dimensions and the strides that the call reads
const at::Tensor& checked(PyObject* o, const char* name, std::initializer_list<at::ScalarType> types, int dims) {
  const at::Tensor& t = tensor(o);
  bool ok = false;
  for (at::ScalarType s : types) ok = ok || t.scalar_type() == s;
  if (!ok) throw torch::TypeError(std::string(name) + ": a tensor of type " + c10::toString(*types.begin()) + " expected, got " + c10::toString(t.scalar_type()));
  TORCH_CHECK_VALUE(t.dim() == dims, name, ": ", dims, " dimensions expected, got ", t.dim());
  TORCH_CHECK_VALUE(t.is_cuda(), name, ": a tensor on the GPU expected, got one on ", t.device());
  TORCH_CHECK_VALUE(t.device().index() == c10::cuda::current_device(), name, ": on ", t.device(), ", but device ", (int)c10::cuda::current_device(), " is current");
  return t;
}
const at::Tensor& whole(PyObject* o, const char* name, std::initializer_list<at::ScalarType> types, int dims) {
  const at::Tensor& t = checked(o, name, types, dims);
  TORCH_CHECK_VALUE(t.is_contiguous(), name, ": not contiguous");
  return t;
}
// rows of f32, each contiguous; the row stride
const at::Tensor& rows_of(PyObject* o, const char* name, int* ld) {
  const at::Tensor& t = checked(o, name, {at::kFloat}, 2);
  TORCH_CHECK_VALUE(t.size(1) < 2 || t.stride(1) == 1, name, ": the values of a row are not contiguous");
  TORCH_CHECK_VALUE(t.size(0) < 2 || (t.stride(0) >= t.size(1) && t.stride(0) <= INT32_MAX), name, ": row stride ", t.stride(0));
  *ld = t.size(0) < 2 ? (int)t.size(1) : (int)t.stride(0);
  return t;
}
int int32_size(int64_t v, const char* name) {
  TORCH_CHECK_VALUE(v <= INT32_MAX, name, ": ", v, " is too many");
  return (int)v;
}
// quantised rows: aq [Mp, K] int8, asc [K / 32, Mp] f32
void quantised_rows(PyObject* aq, PyObject* asc, int64_t K, int64_t T) {
  const at::Tensor &q = whole(aq, "aq", {at::kChar}, 2), &s = whole(asc, "asc", {at::kFloat}, 2);
  TORCH_CHECK_VALUE(q.size(1) == K && q.size(0) >= T && s.size(0) == K / 32 && s.size(1) >= T, "aq ", q.sizes(), " and asc ", s.sizes(), " for ", T, " rows of ", K);
}

// (logits, out, params, hist, hist_off, bias_ids, bias, bias_off, mask, mask_row, want_best): out None = in place
FN(logits_process) {
  HANDLE_TH_ERRORS
  count(n, 11);
  int ldl = 0, ldo = 0;
  const at::Tensor& l = rows_of(a[0], "logits", &ldl);
  PyObject* po = a[1] == Py_None ? a[0] : a[1];
  const at::Tensor& o = rows_of(po, "out", &ldo);
  const int64_t rows = l.size(0);
  const int V = int32_size(l.size(1), "logits");
  TORCH_CHECK_VALUE(o.size(0) == rows && o.size(1) == V, "out ", o.sizes(), " for logits ", l.sizes());
  if (a[2] != Py_None) {
    const at::Tensor& p = whole(a[2], "params", {at::kFloat}, 2);
    TORCH_CHECK_VALUE(p.size(0) == rows && p.size(1) == 4, "params ", p.sizes(), " for ", rows, " rows ([rows, 4] expected)");
  }
  int n_hist = 0, n_bias = 0, words = 0, n_masks = 0;
  auto offsets = [&](PyObject* o, const char* name) {
    TORCH_CHECK_VALUE(whole(o, name, {at::kInt}, 1).size(0) == rows + 1, name, ": ", rows + 1, " offsets expected");
  };
  if (a[3] != Py_None) {
    n_hist = int32_size(whole(a[3], "hist", {at::kInt}, 1).size(0), "hist");
    offsets(a[4], "history offsets");
  }
  if (a[5] != Py_None) {
    n_bias = int32_size(whole(a[5], "bias ids", {at::kInt}, 1).size(0), "bias ids");
    TORCH_CHECK_VALUE(whole(a[6], "biases", {at::kFloat}, 1).size(0) == n_bias, "as many biases as bias ids expected");
    offsets(a[7], "bias offsets");
  }
  if (a[8] != Py_None) {
    const at::Tensor& m = whole(a[8], "mask", {at::kInt}, 2);
    n_masks = int32_size(m.size(0), "mask");
    words = int32_size(m.size(1), "mask");
  }
  if (a[9] != Py_None) TORCH_CHECK_VALUE(whole(a[9], "mask_row", {at::kInt}, 1).size(0) == rows, "mask_row: one per row expected");
  at::Tensor best, logz;
  if (PyObject_IsTrue(a[10])) {
    best = empty({rows}, at::kInt, l.device());
    logz = empty({rows}, at::kFloat, l.device());
  }
  int32_t* pb = best.defined() ? static_cast<int32_t*>(best.data_ptr()) : nullptr;
  float* pz = logz.defined() ? static_cast<float*>(logz.data_ptr()) : nullptr;
  call(g.izb_logits_process_, ptr<float>(a[0]), ldl, ptr<float>(po), ldo, int32_size(rows, "logits"), V, ptr<float>(a[2]), ptr<int32_t>(a[3]), ptr<int32_t>(a[4]),
       n_hist, ptr<int32_t>(a[5]), ptr<float>(a[6]), ptr<int32_t>(a[7]), n_bias, ptr<uint32_t>(a[8]), words, n_masks, ptr<int32_t>(a[9]), pb, pz);
  return tuple({own(po), pb ? wrap(best) : own(Py_None), pz ? wrap(logz) : own(Py_None)});
  END_HANDLE_TH_ERRORS
}

// (A, B, scales, aq, asc, T, seg, adapter, out, base, c_off, ranks): base None = out
FN(lora_add) {
  HANDLE_TH_ERRORS
  count(n, 12);
  const at::Tensor &A = whole(a[0], "A", {at::kHalf, at::kBFloat16}, 3), &B = whole(a[1], "B", {A.scalar_type()}, 3);
  const int n_ad = int32_size(A.size(0), "A"), R = int32_size(A.size(1), "A"), K = int32_size(A.size(2), "A"), N = int32_size(B.size(1), "B");
  TORCH_CHECK_VALUE(B.size(0) == n_ad && B.size(2) == R, "A ", A.sizes(), " and B ", B.sizes(), " ([n, R, K] and [n, N, R] expected)");
  TORCH_CHECK_VALUE(whole(a[2], "scales", {at::kFloat}, 1).size(0) == n_ad, "scales: one per adapter expected");
  const int T = num(a[5]), c_off = num(a[10]);
  quantised_rows(a[3], a[4], K, T);
  const int n_seg = int32_size(whole(a[7], "adapter", {at::kInt}, 1).size(0), "adapter");
  TORCH_CHECK_VALUE(whole(a[6], "seg", {at::kInt}, 1).size(0) == (int64_t)n_seg + 1, "seg: ", (int64_t)n_seg + 1, " offsets expected");
  int ldc = 0, ldb = 0;
  const at::Tensor& C = rows_of(a[8], "out", &ldc);
  TORCH_CHECK_VALUE(C.size(0) >= T && c_off >= 0 && C.size(1) >= (int64_t)c_off + N, "out ", C.sizes(), " for ", T, " rows of ", N, " at column ", c_off);
  const float* base = static_cast<const float*>(C.data_ptr()) + c_off;
  ldb = ldc;
  if (a[9] != Py_None) {
    const at::Tensor& b = rows_of(a[9], "base", &ldb);
    TORCH_CHECK_VALUE(b.size(0) >= T && b.size(1) >= N, "base ", b.sizes(), " for ", T, " rows of ", N);
    base = static_cast<const float*>(b.data_ptr());
  }
  if (a[11] != Py_None) TORCH_CHECK_VALUE(whole(a[11], "ranks", {at::kInt}, 1).size(0) == n_ad, "ranks: one per adapter expected");
  const int dtype = A.scalar_type() == at::kHalf ? IZB_F16 : IZB_BF16;
  at::Tensor scratch;
  const size_t bytes = g.izb_lora_scratch_(dtype, R, T, n_seg);
  if (bytes) scratch = empty({(int64_t)bytes}, at::kByte, A.device());
  call(g.izb_lora_add_, dtype, (const void*)A.data_ptr(), (const void*)B.data_ptr(), n_ad, R, ptr<int32_t>(a[11]), ptr<float>(a[2]), N, K,
       ptr<int8_t>(a[3]), ptr<float>(a[4]), T, extent(a[4], 1), ptr<int32_t>(a[6]), ptr<int32_t>(a[7]), n_seg, base, ldb, static_cast<float*>(C.data_ptr()), ldc, c_off,
       bytes ? scratch.data_ptr() : nullptr);
  return own(a[8]);
  END_HANDLE_TH_ERRORS
}

// (wg, wu, wd, E, F, aq, asc, logits, NU, x, out, sh, e0): out None = allocate
FN(moe_layer) {
  HANDLE_TH_ERRORS
  count(n, 13);
  izb_weight *wg = weight(a[0]), *wu = weight(a[1]), *wd = weight(a[2]);
  const int E = num(a[3]), F = num(a[4]), NU = num(a[8]), e0 = num(a[12]);
  int ldl = 0;
  const at::Tensor& l = rows_of(a[7], "logits", &ldl);
  const int T = int32_size(l.size(0), "logits"), NE = int32_size(l.size(1), "logits") - (a[11] != Py_None ? 1 : 0);
  quantised_rows(a[5], a[6], E, T);
  auto block = [&](PyObject* o, const char* name) {
    const at::Tensor& t = whole(o, name, {at::kFloat}, 2);
    TORCH_CHECK_VALUE(t.size(0) == T && t.size(1) == E, name, " ", t.sizes(), " ([", T, ", ", E, "] expected)");
  };
  if (a[9] != Py_None) block(a[9], "x");
  if (a[11] != Py_None) block(a[11], "sh");
  at::Tensor made;
  if (a[10] == Py_None) made = empty({T, E}, at::kFloat, l.device());
  else block(a[10], "out");
  // (the scratch goes back to torch's allocator when this returns, which gives it to later work of this stream only)
  const at::Tensor scratch = empty({(int64_t)g.izb_moe_layer_scratch_(T, NU, F)}, at::kByte, l.device());
  call(g.izb_moe_layer_, wg, wu, wd, ptr<int8_t>(a[5]), ptr<float>(a[6]), T, extent(a[6], 1), ptr<float>(a[7]), ldl, NE, NU, e0, ptr<float>(a[11]), ptr<float>(a[9]),
       made.defined() ? static_cast<float*>(made.data_ptr()) : ptr<float>(a[10]), scratch.data_ptr());
  return made.defined() ? wrap(made) : own(a[10]);
  END_HANDLE_TH_ERRORS
}

// bind(fail, address, {"izb_...": address})
FN(bind) {
  HANDLE_TH_ERRORS
  count(n, 3);
#define X(name)                                                                    \
  {                                                                                \
    PyObject* v = PyDict_GetItemString(a[2], #name);                               \
    if (!v) throw torch::TypeError("bind: no address for " #name);             \
    g.name##_ = reinterpret_cast<decltype(&name)>(PyLong_AsVoidPtr(v));            \
    if (!g.name##_) throw torch::TypeError("bind: null address for " #name);   \
  }
  IZB_PY_CALLS(X)
#undef X
  Py_INCREF(a[0]);
  Py_INCREF(a[1]);
  g_fail = a[0];
  g_address = a[1];
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

// names(): the entry points bind() wants
PyObject* names(PyObject*, PyObject*) {
  PyObject* l = PyList_New(0);
#define X(name)                                   \
  {                                               \
    PyObject* s = PyUnicode_FromString(#name);    \
    PyList_Append(l, s);                          \
    Py_DECREF(s);                                 \
  }
  IZB_PY_CALLS(X)
#undef X
  return l;
}

#define M(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {M(bind), M(quantize_act), M(swiglu_quant), M(rmsnorm_quant), M(add_norm_quant), M(softcap_rows), M(matmul), M(quant_matmul), M(gemv),
                         M(gemm), M(moe_route), M(moe_sort), M(moe_gateup), M(moe_down), M(moe_combine), M(moe_layer), M(lora_add),
                         M(logits_process), {"names", names, METH_NOARGS, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_izb_py", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__izb_py(void) { return PyModule_Create(&module); }
