// The way from Python to a kernel's entry point: an ``Entry`` is called with tensors and numbers, turns them into the
// C arguments that its signature names, adds the current stream and calls.  Built as an extension module (it takes a
// tensor's pointer from the tensor itself), so that a launch costs the host little more than the launch: through ctypes
// objects made one by one a decoded token's product cost 13 us, 3 of them cudaLaunchKernelEx.
//
// Signature letters: p a CUDA tensor or None (its address or null), i int, l long long, f float.  Every entry point
// takes its stream last and returns an int: 0, a CUDA error (> 0) or a refusal (< 0).  As with ctypes, numbers are
// narrowed without a check and the interpreter's lock is released during the call.
//
// ``product(x, w, out_f32, silu, limit, slope, shift)``: x . w^T for the plain cases of the bfloat16 kernels (see
// rllm_b200/kernels/ops.py, small_m_takes and tcgen05_takes, which hold the same rule), or None: the caller's own path.
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <ATen/ATen.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cstdlib>
#include <cstring>
#include <tuple>
#include <utility>

namespace {

PyObject* g_error = nullptr;        // the exception class of the kernels' refusals
PyObject* g_launches = nullptr;     // a list of one int: entry points called so far

template <char C> struct Arg;
template <> struct Arg<'p'> {
  typedef void* type;
  static type get(PyObject* o, bool& bad) {
    if (o == Py_None) return nullptr;
    if (!THPVariable_Check(o)) {
      bad = true;
      PyErr_Format(PyExc_TypeError, "a tensor or None is wanted, not %s", Py_TYPE(o)->tp_name);
      return nullptr;
    }
    const at::Tensor& t = THPVariable_Unpack(o);
    if (!t.is_cuda()) {
      bad = true;
      PyErr_SetString(g_error, "the engine's kernels run on CUDA tensors only; there is no CPU path");
      return nullptr;
    }
    return t.data_ptr();
  }
};
inline long long whole(PyObject* o, bool& bad) {
  const long long v = PyLong_AsLongLong(o);        // True, 3, and what has __index__
  if (v == -1 && PyErr_Occurred()) bad = true;
  return v;
}
template <> struct Arg<'i'> {
  typedef int type;
  static type get(PyObject* o, bool& bad) { return (int)whole(o, bad); }
};
template <> struct Arg<'l'> {
  typedef long long type;
  static type get(PyObject* o, bool& bad) { return whole(o, bad); }
};
template <> struct Arg<'f'> {
  typedef float type;
  static type get(PyObject* o, bool& bad) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) bad = true;
    return (float)v;
  }
};

// the current device's current stream
cudaStream_t stream_now() { return c10::cuda::getCurrentCUDAStream().stream(); }

typedef int (*Invoke)(void* fn, PyObject* const* args, bool& bad);

template <typename Ch, Ch... C> struct Signature {
  static constexpr char text[] = {C..., 0};
  template <std::size_t... I>
  static int run(void* fn, PyObject* const* a, bool& bad, std::index_sequence<I...>) {
    const std::tuple<typename Arg<C>::type...> v{(bad ? typename Arg<C>::type() : Arg<C>::get(a[I], bad))...};
    if (bad) return 0;
    const cudaStream_t stream = stream_now();
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = reinterpret_cast<int (*)(typename Arg<C>::type..., cudaStream_t)>(fn)(std::get<I>(v)..., stream);
    Py_END_ALLOW_THREADS
    return rc;
  }
  static int invoke(void* fn, PyObject* const* a, bool& bad) {
    return run(fn, a, bad, std::make_index_sequence<sizeof...(C)>());
  }
};
template <typename Ch, Ch... C> constexpr Signature<Ch, C...> operator""_sig() { return {}; }

struct Row { const char* text; Invoke invoke; };
#define ROW(s) {s, decltype(s##_sig)::invoke}
const Row kSignatures[] = {
    ROW("piiiiippfpppipppfiiiiiip"), ROW("piiippipp"), ROW("piiippp"), ROW("piiippppp"), ROW("piiippppppp"),
    ROW("piiipppppppi"), ROW("piippifpppfippppiiiiiippip"), ROW("piippippppiiipiiip"),
    ROW("piippppifpippiiiiiiipiiippififiip"), ROW("piippppippiiiiiiiiifiifppiipp"), ROW("piippppippiiiiiiiiifpi"),
    ROW("piipppppipipppippiiiiiiiiipp"), ROW("piplpppipiippppiiiiiip"), ROW("pppiippppppiiiiiip"), ROW("pipppppipippiiiiiiiiifp"),
    ROW("pipppppipippiiiiiiiiiifip"), ROW("pippiiipppppppiiiiiip"), ROW("pippppppippiiiiiiiiiifip"), ROW("piippppippiiiiiiifp"), ROW("piippppppppiiiiff"), ROW("piiipppppppppiiipiiiip"), ROW("pipifpipiiiiifff"),
    ROW("pipipiiii"), ROW("pipipiiiiifff"), ROW("pipipiiiiifffp"), ROW("pipipippipippiii"), ROW("pippifpppfipppppiiiiiiipp"),
    ROW("pippiiipppiiiiiiiifpp"), ROW("pippippppipppppppiiiiiiiiiiiiifffip"), ROW("pipppipippiiiiiiifp"),
    ROW("pipppipippiiiiiiiifiifppiipiip"), ROW("pipppipippiiiiiiip"), ROW("pipppippiiiiiiiiifpp"),
    ROW("pippppffpppiiiippiiiip"), ROW("pippppipiiiiiiiifiifppiipiipfpppp"), ROW("pippppipiiiiiiiifpiippp"),
    ROW("pippppippiiiiiiiiifiifppiipp"), ROW("pippppippiiiiiiiiifp"), ROW("pippppippiiiiiiiiiiiifp"), ROW("pipppppipiiiip"),
    ROW("pipppppipiiipiip"), ROW("plf"), ROW("plipppppfiiii"), ROW("pllplliplliiiii"), ROW("pllpllpiliiiip"), ROW("ppffpil"),
    ROW("ppfppiii"), ROW("ppiii"), ROW("ppiiifff"), ROW("ppiiii"), ROW("ppiip"), ROW("ppil"), ROW("ppili"), ROW("ppipiii"),
    ROW("ppipiiifip"), ROW("ppipipiiif"), ROW("ppipipiiiif"), ROW("ppippiiiif"), ROW("ppipppppppippili"), ROW("ppl"),
    ROW("pppffpffpiiii"), ROW("pppiiiiii"), ROW("pppiiippi"), ROW("pppiipppffppppiiiiiiippp"), ROW("pppiiippppppiiipiiip"),
    ROW("pppipippiiiiiiifpp"), ROW("pppippippfppfplippiiii"), ROW("ppppfiiiiiii"), ROW("ppppiii"), ROW("ppppiiiii"),
    ROW("ppppiiipppiiipppppiiipiip"), ROW("ppppipiiif"), ROW("ppppipiiifi"), ROW("ppppippiiiiiiiifpiipp"),
    ROW("ppppippiippfiiiiiiiiiiip"), ROW("pppppiipppiipiiiip"), ROW("pppppippiiiiiiiiiiifiipp"), ROW("ppppppipiiii"),
    ROW("ppppppipiilii"), ROW("ppppppppiiifi"), ROW("ppppppppppiiiiifffi"), ROW("ppppppppppiiiiiifffp"),
};

struct Entry {
  PyObject_HEAD
  vectorcallfunc vectorcall;
  Invoke invoke;
  Py_ssize_t count;
  void* fn;
  PyObject* find;                   // () -> the entry point's address; called once, by the first call
  PyObject* what;
};

bool ready(Entry* e) {
  if (e->fn) return true;
  PyObject* at = PyObject_CallNoArgs(e->find);
  if (!at) return false;
  e->fn = PyLong_AsVoidPtr(at);
  Py_DECREF(at);
  return e->fn != nullptr || (PyErr_Occurred() ? false : (PyErr_SetString(g_error, "an entry point without an address"), false));
}

bool finish(int rc, PyObject* what) {
  PyObject* n = PyList_GET_ITEM(g_launches, 0);
  PyObject* more = PyLong_FromLongLong(PyLong_AsLongLong(n) + 1);
  if (!more || PyList_SetItem(g_launches, 0, more)) return false;
  if (rc == 0) return true;
  if (rc == -1) PyErr_Format(g_error, "%U: refused its arguments (bad size or pointer)", what);
  else if (rc == -2) PyErr_Format(g_error, "%U: this size is legal but no kernel of this build takes it", what);
  else PyErr_Format(g_error, "%U: CUDA error %d", what, rc);
  return false;
}

// What ATen throws (no strides, no memory) becomes the exception that PyTorch makes of it: nothing of C++ may leave a function
// that the interpreter calls.
template <typename F> PyObject* guarded(F&& body) {
  try {
    return body();
  } catch (const std::exception&) {
    torch::translate_exception_to_python(std::current_exception());
    return nullptr;
  }
}

PyObject* entry_call(PyObject* self, PyObject* const* args, size_t nargsf, PyObject* names) {
  Entry* e = (Entry*)self;
  if ((names && PyTuple_GET_SIZE(names)) || PyVectorcall_NARGS(nargsf) != e->count)
    return PyErr_Format(PyExc_TypeError, "%U takes %zd arguments, by position", e->what, e->count);
  if (!ready(e)) return nullptr;
  return guarded([&]() -> PyObject* {
    bool bad = false;
    const int rc = e->invoke(e->fn, args, bad);
    if (bad || !finish(rc, e->what)) return nullptr;
    Py_RETURN_NONE;
  });
}

void entry_free(PyObject* self) {
  Py_XDECREF(((Entry*)self)->find);
  Py_XDECREF(((Entry*)self)->what);
  Py_TYPE(self)->tp_free(self);
}

PyTypeObject EntryType = {PyVarObject_HEAD_INIT(nullptr, 0) "rllm_launch.Entry"};

// entry(signature, find, what)
PyObject* make_entry(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 3 || !PyUnicode_Check(args[0]) || !PyUnicode_Check(args[2])) return PyErr_Format(PyExc_TypeError, "entry(signature, find, what)");
  const char* text = PyUnicode_AsUTF8(args[0]);
  if (!text) return nullptr;
  for (const Row& row : kSignatures) {
    if (std::strcmp(row.text, text)) continue;
    Entry* e = PyObject_New(Entry, &EntryType);
    if (!e) return nullptr;
    e->vectorcall = entry_call;
    e->invoke = row.invoke;
    e->count = (Py_ssize_t)std::strlen(text);
    e->fn = nullptr;
    e->find = Py_NewRef(args[1]);
    e->what = Py_NewRef(args[2]);
    return (PyObject*)e;
  }
  return PyErr_Format(PyExc_ValueError, "no signature %s among those that were compiled", text);
}

// ---------------------------------------------------------------------------------------------------------------
// products
// ---------------------------------------------------------------------------------------------------------------
Entry *g_small = nullptr, *g_tcgen05 = nullptr;
long long g_small_rows = 0, g_min_tiles = 0;
void* g_error_word[64] = {};        // by device; null: ask Python

// products(small_m entry, tcgen05 entry, most rows of the first, fewest tiles of the second)
PyObject* set_products(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 4 || Py_TYPE(args[0]) != &EntryType || Py_TYPE(args[1]) != &EntryType) return PyErr_Format(PyExc_TypeError, "products(entry, entry, rows, tiles)");
  g_small = (Entry*)Py_NewRef(args[0]);
  g_tcgen05 = (Entry*)Py_NewRef(args[1]);
  g_small_rows = PyLong_AsLongLong(args[2]);
  g_min_tiles = PyLong_AsLongLong(args[3]);
  if (PyErr_Occurred()) return nullptr;
  Py_RETURN_NONE;
}

// error_word(device index, tensor): the word that the tcgen05 product reports to on that device (the caller keeps it)
PyObject* set_error_word(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    const long long d = n == 2 ? PyLong_AsLongLong(args[0]) : -1;
    if (d < 0 || d >= 64 || !THPVariable_Check(args[1])) return PyErr_Occurred() ? nullptr : PyErr_Format(PyExc_TypeError, "error_word(device index, tensor)");
    g_error_word[d] = THPVariable_Unpack(args[1]).data_ptr();
    Py_RETURN_NONE;
  });
}

bool is(const char* value, const char* text) { return value && !std::strcmp(value, text); }

PyObject* checked_product(PyObject* const* args) {
  const at::Tensor &x = THPVariable_Unpack(args[0]), &w = THPVariable_Unpack(args[1]);
  const bool f32 = args[2] == Py_True, silu = args[3] == Py_True;
  if (!x.is_cuda() || !w.is_cuda() || x.dim() != 2 || w.dim() != 2 || x.scalar_type() != at::kBFloat16 || w.scalar_type() != at::kBFloat16)
    Py_RETURN_NONE;
  const long long M = x.size(0), K = x.size(1), N = silu ? w.size(0) / 2 : w.size(0), lda = x.stride(0), ldw = w.stride(0);
  if (M <= 0 || N <= 0 || w.size(1) != K || x.stride(1) != 1 || w.stride(1) != 1 || K % 8 || lda % 8 || ldw % 8 || (silu && w.size(0) != 2 * N))
    Py_RETURN_NONE;
  const char* mode = std::getenv("RLLM_GEMM");
  if (is(mode, "library")) Py_RETURN_NONE;
  const bool small = M <= g_small_rows;
  if (small) {
    if (!silu && w.size(0) > 65536 && (M > 8 || is(std::getenv("RLLM_HEAD"), "library"))) Py_RETURN_NONE;
  } else {
    if (is(mode, "no_tcgen05") || (((uintptr_t)x.data_ptr() | (uintptr_t)w.data_ptr()) & 15)) Py_RETURN_NONE;
    const long long cols = silu ? 128 : 256, tiles = (M + 127) / 128 * ((N + cols - 1) / cols);
    if (!is(mode, "tcgen05") && tiles < g_min_tiles) Py_RETURN_NONE;
  }
  const int device = x.get_device();
  Entry* e = small ? g_small : g_tcgen05;
  if (!small && (device < 0 || device >= 64 || !g_error_word[device])) Py_RETURN_NONE;
  if (!ready(e)) return nullptr;
  at::Tensor out = at::empty({M, N}, x.options().dtype(f32 ? at::kFloat : at::kBFloat16));
  bool bad = false;
  const float limit = Arg<'f'>::get(args[4], bad), slope = Arg<'f'>::get(args[5], bad), shift = Arg<'f'>::get(args[6], bad);
  if (bad) return nullptr;
  void *px = x.data_ptr(), *pw = w.data_ptr(), *po = out.data_ptr();
  const int code = silu ? 2 : (f32 ? 1 : 0);
  const cudaStream_t stream = stream_now();
  int rc;
  Py_BEGIN_ALLOW_THREADS
  if (small)
    rc = reinterpret_cast<int (*)(void*, int, void*, int, void*, int, int, int, int, int, float, float, float, cudaStream_t)>(e->fn)(
        px, (int)lda, pw, (int)ldw, po, (int)N, (int)M, (int)N, (int)K, code, limit, slope, shift, stream);
  else
    rc = reinterpret_cast<int (*)(void*, int, void*, int, void*, int, int, int, int, int, float, float, float, void*, cudaStream_t)>(e->fn)(
        px, (int)lda, pw, (int)ldw, po, (int)N, (int)M, (int)N, (int)K, code, limit, slope, shift, g_error_word[device], stream);
  Py_END_ALLOW_THREADS
  if (!finish(rc, e->what)) return nullptr;
  return THPVariable_Wrap(std::move(out));
}

PyObject* product(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 7) return PyErr_Format(PyExc_TypeError, "product(x, w, out_f32, silu, limit, slope, shift)");
  if (!g_small || !THPVariable_CheckExact(args[0]) || !THPVariable_CheckExact(args[1])) Py_RETURN_NONE;      // tensors and parameters
  return guarded([&] { return checked_product(args); });
}

// ---------------------------------------------------------------------------------------------------------------
// a cache kept in 8 bits
// ---------------------------------------------------------------------------------------------------------------
// e4m3_ready(kcache, vcache, kscale, vscale, block_table, nkv, d, *vectors): whether these are what the operators over such a
// cache take (see rllm_b200/kernels/ops.py, _e4m3_cache, which holds the same rules and says what is wrong): all on the current
// device, the vectors contiguous, one-dimensional and int32.  In Python these checks cost as much as the launch three times over.
bool vector_of_ints(const at::Tensor& t, int device) {
  return t.is_cuda() && t.get_device() == device && t.scalar_type() == at::kInt && t.dim() == 1 && t.is_contiguous();
}

bool e4m3_cache(PyObject* const* args, long long nkv, long long d, int device) {      // kcache, vcache, kscale, vscale, block_table
  const at::Tensor &k = THPVariable_Unpack(args[0]), &v = THPVariable_Unpack(args[1]), &ks = THPVariable_Unpack(args[2]),
                   &vs = THPVariable_Unpack(args[3]), &table = THPVariable_Unpack(args[4]);
  if (k.scalar_type() != at::kFloat8_e4m3fn || v.scalar_type() != at::kFloat8_e4m3fn || ks.scalar_type() != at::kFloat8_e8m0fnu ||
      vs.scalar_type() != at::kFloat8_e8m0fnu || table.scalar_type() != at::kInt)
    return false;
  if (k.dim() != 4 || k.size(1) != nkv || k.size(3) != d || k.size(2) > 0x7fffffffLL || v.sizes() != k.sizes() || ks.sizes() != k.sizes().slice(0, 3) ||
      vs.sizes() != ks.sizes() || table.dim() != 2)
    return false;
  for (int i = 0; i < 5; ++i) {
    const at::Tensor& t = THPVariable_Unpack(args[i]);
    if (!t.is_cuda() || t.get_device() != device || !t.is_contiguous()) return false;
  }
  return true;
}

// The entry points count in 32 bits: a bound that is larger than what it bounds can be becomes the largest such number, never its low bits.
long long in_32_bits(long long x) { return std::min(x, 0x7fffffffLL); }

// all of args[0 .. n - 1] are tensors on CUDA devices (asked before CUDA is asked for its current one)
bool cuda_tensors(PyObject* const* args, Py_ssize_t n) {
  for (Py_ssize_t i = 0; i < n; ++i)
    if (!THPVariable_Check(args[i]) || !THPVariable_Unpack(args[i]).is_cuda()) return false;
  return true;
}

PyObject* e4m3_ready(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n < 7) return PyErr_Format(PyExc_TypeError, "e4m3_ready(kcache, vcache, kscale, vscale, block_table, nkv, d, *vectors)");
  if (!cuda_tensors(args, 5) || !cuda_tensors(args + 7, n - 7)) Py_RETURN_FALSE;
  return guarded([&]() -> PyObject* {
    const long long nkv = PyLong_AsLongLong(args[5]), d = PyLong_AsLongLong(args[6]);
    if (PyErr_Occurred()) return nullptr;
    const int device = c10::cuda::current_device();
    if (!e4m3_cache(args, nkv, d, device)) Py_RETURN_FALSE;
    for (Py_ssize_t i = 7; i < n; ++i)
      if (!vector_of_ints(THPVariable_Unpack(args[i]), device)) Py_RETURN_FALSE;
    Py_RETURN_TRUE;
  });
}

// The operators' calls, checked and launched in one go: True, or False where Python has to look (and refuse, or take the call its
// own way).  Each is given its entry points first.
int float_code(const at::Tensor& t) { return t.scalar_type() == at::kBFloat16 ? 1 : t.scalar_type() == at::kFloat ? 0 : -1; }

// e4m3_write(entry, qkv, q_out or None, positions, token_seq, err, kcache, vcache, kscale, vscale, block_table, inv_freq or None, rotary_dim,
//            nq, nkv, d)
PyObject* e4m3_write(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 16 || Py_TYPE(args[0]) != &EntryType) return PyErr_Format(PyExc_TypeError, "e4m3_write(entry, ... 15 arguments)");
  const bool in_place = args[2] == Py_None;
  if (!cuda_tensors(args + 1, 1) || !(in_place || cuda_tensors(args + 2, 1)) || !cuda_tensors(args + 3, 8)) Py_RETURN_FALSE;
  return guarded([&]() -> PyObject* {
    bool bad = false;
    const long long rot = whole(args[12], bad), nq = whole(args[13], bad), nkv = whole(args[14], bad), d = whole(args[15], bad);
    if (bad) return nullptr;
    Entry* e = (Entry*)args[0];
    if (!ready(e)) return nullptr;
    const at::Tensor &qkv = THPVariable_Unpack(args[1]), &q = THPVariable_Unpack(args[in_place ? 1 : 2]);
    const int device = c10::cuda::current_device(), dt = float_code(qkv);
    if (dt < 0 || qkv.dim() != 2 || qkv.size(1) != (nq + 2 * nkv) * d || !qkv.is_contiguous() || qkv.get_device() != device ||
        q.dim() != 2 || q.size(0) != qkv.size(0) || (!in_place && q.size(1) != nq * d) || q.stride(1) != 1 || q.scalar_type() != qkv.scalar_type() ||
        q.get_device() != device || !e4m3_cache(args + 6, nkv, d, device))
      Py_RETURN_FALSE;
    const long long T = qkv.size(0), stride = T > 1 ? q.stride(0) : q.size(1);
    for (int i = 3; i < 6; ++i)
      if (!vector_of_ints(THPVariable_Unpack(args[i]), device)) Py_RETURN_FALSE;
    if (THPVariable_Unpack(args[3]).numel() != T || THPVariable_Unpack(args[4]).numel() != T) Py_RETURN_FALSE;
    void* freq = nullptr;
    if (rot) {
      if (!cuda_tensors(args + 11, 1)) Py_RETURN_FALSE;
      const at::Tensor& f = THPVariable_Unpack(args[11]);
      if (f.scalar_type() != at::kDouble || f.numel() != rot / 2 || !f.is_contiguous() || f.get_device() != device) Py_RETURN_FALSE;
      freq = f.data_ptr();
    }
    const at::Tensor &k = THPVariable_Unpack(args[6]), &table = THPVariable_Unpack(args[10]);
    auto at_ = [&](int i) { return THPVariable_Unpack(args[i]).data_ptr(); };
    const cudaStream_t stream = stream_now();
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = reinterpret_cast<int (*)(void*, int, void*, long long, void*, void*, void*, int, void*, int, int, void*, void*, void*, void*, int, int,
                                  int, int, int, int, void*, cudaStream_t)>(e->fn)(
        qkv.data_ptr(), dt, q.data_ptr(), stride, at_(3), at_(4), freq, (int)rot, table.data_ptr(), (int)table.size(1), (int)table.size(0),
        at_(6), at_(7), at_(8), at_(9), (int)T, (int)nq, (int)nkv, (int)d, (int)k.size(2), (int)in_32_bits(k.size(0)), at_(5), stream);
    Py_END_ALLOW_THREADS
    if (!finish(rc, e->what)) return nullptr;
    Py_RETURN_TRUE;
  });
}

// e4m3_read(entry, out_k, out_v, positions, token_seq, err, kcache, vcache, kscale, vscale, block_table)
PyObject* e4m3_read(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 11 || Py_TYPE(args[0]) != &EntryType) return PyErr_Format(PyExc_TypeError, "e4m3_read(entry, ... 10 arguments)");
  if (!cuda_tensors(args + 1, 10)) Py_RETURN_FALSE;
  return guarded([&]() -> PyObject* {
    Entry* e = (Entry*)args[0];
    if (!ready(e)) return nullptr;
    const at::Tensor &ok = THPVariable_Unpack(args[1]), &ov = THPVariable_Unpack(args[2]), &k = THPVariable_Unpack(args[6]),
                     &table = THPVariable_Unpack(args[10]);
    const int device = c10::cuda::current_device(), dt = float_code(ok);
    if (dt < 0 || k.dim() != 4 || !e4m3_cache(args + 6, k.size(1), k.size(3), device)) Py_RETURN_FALSE;
    for (int i = 3; i < 6; ++i)
      if (!vector_of_ints(THPVariable_Unpack(args[i]), device)) Py_RETURN_FALSE;
    const long long T = THPVariable_Unpack(args[3]).numel();
    if (THPVariable_Unpack(args[4]).numel() != T || ok.dim() != 2 || ok.size(0) != T || ok.size(1) != k.size(1) * k.size(3) ||
        ov.sizes() != ok.sizes() || ov.scalar_type() != ok.scalar_type() || !ok.is_contiguous() || !ov.is_contiguous() ||
        ok.get_device() != device || ov.get_device() != device)
      Py_RETURN_FALSE;
    auto at_ = [&](int i) { return THPVariable_Unpack(args[i]).data_ptr(); };
    const cudaStream_t stream = stream_now();
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = reinterpret_cast<int (*)(void*, void*, void*, int, int, void*, void*, void*, void*, void*, void*, int, int, int, int, int, int, void*,
                                  cudaStream_t)>(e->fn)(
        at_(3), at_(4), table.data_ptr(), (int)table.size(1), (int)table.size(0), at_(6), at_(7), at_(8), at_(9), ok.data_ptr(), ov.data_ptr(), dt,
        (int)T, (int)k.size(1), (int)k.size(3), (int)k.size(2), (int)in_32_bits(k.size(0)), at_(5), stream);
    Py_END_ALLOW_THREADS
    if (!finish(rc, e->what)) return nullptr;
    Py_RETURN_TRUE;
  });
}

// Which kernel takes an attention over such a cache: the rule of ops.attention_e4m3_form, whose text has both sides of every limit
// as measured.
enum Form { kRows, kColumns, kTcgen05, kDense, kSimt, kForms };
const char* const kFormNames[kForms] = {"rows", "columns", "tcgen05", "dense", "simt"};

Form e4m3_rule(bool bf16, long long nq, long long nkv, long long d, long long page, double scale, long long max_q_len, long long seqs,
               long long keys) {
  const char* forced = std::getenv("RLLM_ATTENTION");
  const long long g = nq / nkv, rows = max_q_len * g;
  const bool simt = is(forced, "simt"), in_16s = page % 16 == 0 && !simt, heads = d == 64 || d == 128;
  const bool rows_take = in_16s && (heads || d == 256) && (rows + 7) / 8 * nkv <= 65535;
  if (bf16 && heads && !simt && !is(forced, "mma")) {
    const long long tiles = (rows + 31) / 32;
    const bool few = tiles == 1 || seqs * nkv * tiles <= 32;
    if (few && in_16s && (tiles == 1 || d == 128) && tiles * nkv <= 65535 && keys >= 768 && seqs * nkv * tiles * keys >= (d == 64 ? 1 << 16 : 1 << 14))
      return kColumns;
    if (!(few && rows_take) && g <= 128 && scale > 0) {
      const long long tokens = 128 / g;                    // of a tile of 128 rows
      return (max_q_len + tokens - 1) / tokens <= 4 ? kTcgen05 : kDense;
    }
  }
  return rows_take ? kRows : kSimt;
}

// Whether a kernel takes a call at all: its grid's places, and what it reads or stores 16 bytes at a time.  The CUDA-core one takes every call.
bool e4m3_takes(Form form, long long nq, long long nkv, long long d, long long page, long long max_q_len, long long seqs, bool scales_on_16,
                bool queries_on_16, bool results_on_16) {
  if (form == kSimt) return true;
  const long long g = nq / nkv, places = 65535;
  if (!results_on_16 || (form != kDense && seqs > places)) return false;
  const long long rows = max_q_len * g, tile = form == kColumns ? std::min((rows + 7) / 8 * 8, 32LL) : 8;
  if (form == kRows || form == kColumns) return scales_on_16 && page % 16 == 0 && (rows + tile - 1) / tile * nkv <= places;
  if (!queries_on_16 || g > 128) return false;
  const long long tokens = 128 / g;
  return form == kDense ? nkv <= places : (max_q_len + tokens - 1) / tokens * nkv <= places;
}

// e4m3_form(bfloat16, nq, nkv, d, page_size, scale, max_q_len, num_seqs, max_keys)
PyObject* e4m3_form(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 9) return PyErr_Format(PyExc_TypeError, "e4m3_form(bfloat16, nq, nkv, d, page_size, scale, max_q_len, num_seqs, max_keys)");
  bool bad = false;
  long long v[9];
  for (int i = 0; i < 9; ++i) v[i] = i == 5 || bad ? 0 : whole(args[i], bad);
  const double scale = bad ? 0. : PyFloat_AsDouble(args[5]);
  if (bad || PyErr_Occurred()) return nullptr;
  if (v[1] <= 0 || v[2] <= 0 || v[1] % v[2]) return PyErr_Format(g_error, "%lld query heads over %lld kv heads", v[1], v[2]);
  return PyUnicode_FromString(kFormNames[e4m3_rule(v[0] != 0, v[1], v[2], v[3], v[4], scale, v[6], v[7], v[8])]);
}

// e4m3_attention(entries, q, out, q_start, seq_lens, err, kcache, vcache, kscale, vscale, block_table, num_decode, max_q_len,
//                max_seq_len, nq, nkv, window, scale, scratch, forms, lengths_ready): checked and launched.  entries: (rows, columns,
// tcgen05, simt, widen, dense); scratch: bytes of widened keys and values at a time; forms: None, or two names (for the single tokens, for
// the others) in place of the rule's.  False: a call that has to be refused, ops.attention_e4m3 says why.
enum Known { kAny = 0, kBeside = 1, kLengths = 2 };        // what the kernels are told of the one ahead: kernels/csrc/kv_e4m3.cuh
PyObject* e4m3_attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
  enum { kEntries = 6 };
  if (n != 21 || !PyTuple_Check(args[0]) || PyTuple_GET_SIZE(args[0]) != kEntries || !PyBool_Check(args[20]))
    return PyErr_Format(PyExc_TypeError, "e4m3_attention((entries), ... 20 arguments)");
  Entry* e[kEntries];
  for (int i = 0; i < kEntries; ++i) {
    PyObject* x = PyTuple_GET_ITEM(args[0], i);
    if (Py_TYPE(x) != &EntryType) return PyErr_Format(PyExc_TypeError, "entries are wanted first");
    e[i] = (Entry*)x;
  }
  int named[2] = {-1, -1};
  if (args[19] != Py_None) {
    if (!PyTuple_Check(args[19]) || PyTuple_GET_SIZE(args[19]) != 2) return PyErr_Format(PyExc_TypeError, "forms: None or two names");
    for (int i = 0; i < 2; ++i) {
      const char* text = PyUnicode_Check(PyTuple_GET_ITEM(args[19], i)) ? PyUnicode_AsUTF8(PyTuple_GET_ITEM(args[19], i)) : nullptr;
      for (int f = 0; text && f < kForms; ++f)
        if (!std::strcmp(text, kFormNames[f])) named[i] = f;
      if (named[i] < 0) return PyErr_Occurred() ? nullptr : PyErr_Format(g_error, "no form of that name");
    }
  }
  if (!cuda_tensors(args + 1, 10)) Py_RETURN_FALSE;
  return guarded([&]() -> PyObject* {
    bool bad = false;
    long long v[8];                                        // num_decode, max_q_len, max_seq_len, nq, nkv, window, -, scratch
    for (int i = 0; i < 8 && !bad; ++i) v[i] = i == 6 ? 0 : whole(args[11 + i], bad);
    const double scale = bad ? 0. : PyFloat_AsDouble(args[17]);
    if (bad || PyErr_Occurred()) return nullptr;
    const long long decode = v[0], nq = v[3], nkv = v[4], window = in_32_bits(v[5]), scratch = v[7];
    const at::Tensor &q = THPVariable_Unpack(args[1]), &out = THPVariable_Unpack(args[2]), &k = THPVariable_Unpack(args[6]),
                     &table = THPVariable_Unpack(args[10]);
    const int device = c10::cuda::current_device(), dt = float_code(q);
    if (dt < 0 || k.dim() != 4 || nq <= 0 || nkv <= 0 || nq % nkv || nq > 0x7fffffffLL || window < 0) Py_RETURN_FALSE;
    const long long d = k.size(3), page = k.size(2), pages = in_32_bits(k.size(0));
    if (!e4m3_cache(args + 6, nkv, d, device)) Py_RETURN_FALSE;
    for (int i = 3; i < 6; ++i)
      if (!vector_of_ints(THPVariable_Unpack(args[i]), device)) Py_RETURN_FALSE;
    const long long S = THPVariable_Unpack(args[4]).numel(), blocks = table.size(1);
    if (THPVariable_Unpack(args[3]).numel() != S + 1 || decode < 0 || decode > S || table.size(0) < S || v[1] < 0 || v[2] < 0 ||
        v[2] > blocks * page || q.dim() != 2 || out.dim() != 2 || out.scalar_type() != q.scalar_type() || q.stride(1) != 1 ||
        out.size(1) != nq * d || q.size(1) < nq * d || q.size(0) < out.size(0) || !out.is_contiguous() || q.get_device() != device ||
        out.get_device() != device)
      Py_RETURN_FALSE;
    // a single row may have any stride; no sequence has more tokens than out has rows, nor more keys than its length, an int, says
    const long long T = in_32_bits(out.size(0)), stride = q.size(0) > 1 ? q.stride(0) : nq * d, max_q = std::min(v[1], T), most = in_32_bits(v[2]);
    if (stride > 0x7fffffffLL) Py_RETURN_FALSE;
    if (T == 0 || S == 0) Py_RETURN_TRUE;
    const long long keys = window > 0 && window + max_q < most ? window + max_q : most;
    void *pq = q.data_ptr(), *po = out.data_ptr(), *pqs = THPVariable_Unpack(args[3]).data_ptr(), *psl = THPVariable_Unpack(args[4]).data_ptr(),
         *pe = THPVariable_Unpack(args[5]).data_ptr(), *pk = k.data_ptr(), *pv = THPVariable_Unpack(args[7]).data_ptr(),
         *pks = THPVariable_Unpack(args[8]).data_ptr(), *pvs = THPVariable_Unpack(args[9]).data_ptr(), *pt = table.data_ptr();
    const cudaStream_t stream = stream_now();
    // Where no fewer sequences bring several tokens than one, and all of them few, they go together: one launch behind another costs
    // more than the rows that single tokens leave empty (32/8 heads of 64, behind 4,000: 4 of one token and 4 of 5 25.6 -> 18.7 us; 16
    // and 16 of 8 behind 2,000, more tiles of 32 rows than SMs, would be 30 -> 35).
    const long long few = max_q * (nq / nkv);
    const bool together_all = args[19] == Py_None && decode > 0 && S - decode >= decode && (few <= 16 || (few <= 32 && S * nkv <= 148));
    const int ahead = args[20] == Py_True ? kLengths : kAny;
    int before = -1;                                       // the form of the call's first launch
    for (int group = together_all ? 1 : 0; group < 2; ++group) {
      const long long first = group && !together_all ? decode : 0, end = group ? S : decode, longest = group ? max_q : 1;
      if (first == end || longest == 0) continue;
      // behind the single tokens' kernel, of which it reads nothing and overwrites nothing (widened tiles come from memory that the first's
      // widened tiles may just have left)
      const int known = group && before >= 0 && before != kDense ? kBeside : ahead;
      Form form = named[group] >= 0 ? (Form)named[group] : e4m3_rule(dt == 1, nq, nkv, d, page, (float)scale, longest, end - first, keys);
      // off 16 bytes, or too many for its grid: the kernel that reads queries one by one, or the one that takes everything
      auto takes = [&](Form f) {
        return e4m3_takes(f, nq, nkv, d, page, longest, end - first, (((uintptr_t)pks | (uintptr_t)pvs) & 15) == 0,
                          (((uintptr_t)pq | (uintptr_t)stride * 2) & 15) == 0, ((uintptr_t)po & 15) == 0);
      };
      if (!takes(form)) form = form != kRows && (d == 64 || d == 128) && takes(kRows) ? kRows : kSimt;
      before = form;
      Entry* at_ = e[form == kRows ? 0 : form == kColumns ? 1 : form == kTcgen05 ? 2 : form == kSimt ? 3 : 5];
      if (!ready(at_)) return nullptr;
      int rc = 0;
      if (form == kColumns || form == kTcgen05) {
        Py_BEGIN_ALLOW_THREADS
        rc = reinterpret_cast<int (*)(void*, int, void*, void*, void*, void*, void*, void*, int, void*, void*, int, int, int, int, int, int, int,
                                      int, int, int, float, int, void*, cudaStream_t)>(at_->fn)(
            pq, (int)stride, po, pk, pv, pks, pvs, pt, (int)blocks, pqs, psl, (int)first, (int)end, (int)longest, (int)keys, (int)nq, (int)nkv,
            (int)d, (int)page, (int)pages, (int)window, (float)scale, known, pe, stream);
        Py_END_ALLOW_THREADS
      } else if (form == kRows) {
        Py_BEGIN_ALLOW_THREADS
        rc = reinterpret_cast<int (*)(void*, int, void*, void*, void*, void*, void*, int, void*, int, void*, void*, int, int, int, int, int, int,
                                      int, int, int, int, float, int, void*, cudaStream_t)>(at_->fn)(
            pq, (int)stride, po, pk, pv, pks, pvs, dt, pt, (int)blocks, pqs, psl, (int)first, (int)end, (int)longest, (int)keys, (int)nq, (int)nkv,
            (int)d, (int)page, (int)pages, (int)window, (float)scale, known, pe, stream);
        Py_END_ALLOW_THREADS
      } else if (form == kSimt) {
        const long long tokens = std::min(T, (end - first) * longest);
        Py_BEGIN_ALLOW_THREADS
        rc = reinterpret_cast<int (*)(void*, int, void*, void*, void*, void*, void*, int, void*, int, void*, void*, int, int, int, int, int, int,
                                      int, int, int, float, void*, cudaStream_t)>(at_->fn)(
            pq, (int)stride, po, pk, pv, pks, pvs, dt, pt, (int)blocks, pqs, psl, (int)first, (int)end, (int)tokens, (int)nq, (int)nkv, (int)d,
            (int)page, (int)pages, (int)window, (float)scale, pe, stream);
        Py_END_ALLOW_THREADS
      } else {
        const long long bn = 8192 / d, tiles = keys / bn + 2, a_sequence = 2 * tiles * nkv * bn * d;      // bytes
        const long long together = std::max(1LL, std::min(std::min(end - first, scratch / (2 * a_sequence)), 65535LL));
        const at::Tensor dense = at::empty({2 * together * a_sequence}, k.options().dtype(at::kByte));
        const at::Tensor marks = at::empty({together * tiles * nkv * 8}, table.options());
        char* const pd = (char*)dense.data_ptr();
        void* const pm = marks.data_ptr();
        if (!ready(e[4])) return nullptr;
        for (long long s = first; s < end; s += together) {
          const long long m = std::min(together, end - s);
          Py_BEGIN_ALLOW_THREADS
          rc = reinterpret_cast<int (*)(void*, int, void*, void*, int, int, int, void*, void*, void*, void*, void*, void*, void*, int, int, int, int,
                                        int, int, void*, cudaStream_t)>(e[4]->fn)(
              pt, (int)blocks, pqs, psl, (int)s, (int)m, (int)tiles, pk, pv, pks, pvs, pd, pd + together * a_sequence, pm, (int)nkv, (int)d,
              (int)page, (int)pages, (int)window, s == first ? known : kLengths, pe, stream);
          Py_END_ALLOW_THREADS
          if (!finish(rc, at_->what)) return nullptr;
          Py_BEGIN_ALLOW_THREADS
          rc = reinterpret_cast<int (*)(void*, int, int, void*, void*, void*, void*, int, void*, void*, int, int, int, int, int, int, int, float,
                                        void*, cudaStream_t)>(at_->fn)(
              pq, (int)stride, (int)q.size(0), po, pd, pd + together * a_sequence, pm, (int)tiles, pqs, psl, (int)s, (int)m,
              (int)std::min(T, m * longest), (int)nq, (int)nkv, (int)d, (int)window, (float)scale, pe, stream);
          Py_END_ALLOW_THREADS
          if (!finish(rc, at_->what)) return nullptr;
        }
        continue;
      }
      if (!finish(rc, at_->what)) return nullptr;
    }
    Py_RETURN_TRUE;
  });
}

// setup(exception class, list of one int)
PyObject* setup(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 2 || !PyList_Check(args[1]) || PyList_GET_SIZE(args[1]) != 1) return PyErr_Format(PyExc_TypeError, "setup(exception, [count])");
  g_error = Py_NewRef(args[0]);
  g_launches = Py_NewRef(args[1]);
  Py_RETURN_NONE;
}

PyMethodDef kMethods[] = {{"setup", (PyCFunction)(void*)setup, METH_FASTCALL, nullptr},
                          {"entry", (PyCFunction)(void*)make_entry, METH_FASTCALL, nullptr},
                          {"products", (PyCFunction)(void*)set_products, METH_FASTCALL, nullptr},
                          {"error_word", (PyCFunction)(void*)set_error_word, METH_FASTCALL, nullptr},
                          {"product", (PyCFunction)(void*)product, METH_FASTCALL, nullptr},
                          {"e4m3_ready", (PyCFunction)(void*)e4m3_ready, METH_FASTCALL, nullptr},
                          {"e4m3_write", (PyCFunction)(void*)e4m3_write, METH_FASTCALL, nullptr},
                          {"e4m3_read", (PyCFunction)(void*)e4m3_read, METH_FASTCALL, nullptr},
                          {"e4m3_form", (PyCFunction)(void*)e4m3_form, METH_FASTCALL, nullptr},
                          {"e4m3_attention", (PyCFunction)(void*)e4m3_attention, METH_FASTCALL, nullptr},
                          {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "launch", nullptr, -1, kMethods};

}  // namespace

extern "C" __attribute__((visibility("default"))) PyObject* PyInit_launch() {
  EntryType.tp_basicsize = sizeof(Entry);
  EntryType.tp_flags = Py_TPFLAGS_DEFAULT | Py_TPFLAGS_HAVE_VECTORCALL;
  EntryType.tp_vectorcall_offset = offsetof(Entry, vectorcall);
  EntryType.tp_call = PyVectorcall_Call;
  EntryType.tp_dealloc = entry_free;
  if (PyType_Ready(&EntryType) < 0) return nullptr;
  return PyModule_Create(&kModule);
}
