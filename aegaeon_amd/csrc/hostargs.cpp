// aegaeon_amd._hostargs: the argument tables of a move, read from Python
// objects in one pass, and the calls over a quantised cache.
//
// A copy over 72 backing tensors asks each for its device, layout, size and
// address. Asked from Python one attribute at a time that is 50 us, several
// times what the copy of one block takes; here it is 2. Both functions return
// None for anything but the plain case (a list of dense device tensors, a
// list of Python integers), and the caller then takes the general path, which
// names what is wrong or converts other kinds of sequences.
//
// A decode step makes two calls a layer over a quantised cache. Their tensors
// checked and their C arguments made in Python, they took the host 7.4 us
// (write) and 14 (attend), 3 to 6 of which are the launches; here 3.8 and 8.3.
// These functions too take the plain case only: None, with nothing enqueued,
// for anything else. What the library itself answers is the answer: its status, if
// it refused the call or failed in it, as a number. (A call made a second time
// could take what the first one wrote for its input.)

#include <torch/csrc/autograd/python_variable.h>
#include <ATen/ATen.h>
#include <c10/core/GradMode.h>

#include <cstdint>
#include <cstring>

namespace {

struct Ref {  // owned reference
  PyObject* p;
  explicit Ref(PyObject* o) : p(o) {}
  ~Ref() { Py_XDECREF(p); }
  PyObject* release() {
    PyObject* o = p;
    p = nullptr;
    return o;
  }
  Ref(const Ref&) = delete;
  Ref& operator=(const Ref&) = delete;
};

// A list or tuple, whose items stay where they are while none of the code
// here runs Python code.
bool plain_sequence(PyObject* o) { return PyList_CheckExact(o) || PyTuple_CheckExact(o); }

// segment_table(segments, num_blocks) -> (device index, num_blocks, addresses,
// page bytes), the last two as packed 8-byte values, or None. num_blocks None:
// the first tensor's leading size. A page is a tensor's bytes / num_blocks.
PyObject* segment_table(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  if (nargs != 2) {
    PyErr_SetString(PyExc_TypeError, "segment_table(segments, num_blocks)");
    return nullptr;
  }
  PyObject* seq = args[0];
  if (!plain_sequence(seq)) Py_RETURN_NONE;
  const Py_ssize_t n = PySequence_Fast_GET_SIZE(seq);
  PyObject** items = PySequence_Fast_ITEMS(seq);
  if (n == 0) Py_RETURN_NONE;
  int64_t blocks = 0;
  if (args[1] != Py_None) {
    if (!PyLong_CheckExact(args[1])) Py_RETURN_NONE;
    int overflow = 0;
    blocks = PyLong_AsLongLongAndOverflow(args[1], &overflow);
    if (overflow) Py_RETURN_NONE;
  }
  Ref bases(PyBytes_FromStringAndSize(nullptr, n * 8));
  Ref pages(PyBytes_FromStringAndSize(nullptr, n * 8));
  if (!bases.p || !pages.p) return nullptr;
  int device = -1;
  try {
    for (Py_ssize_t i = 0; i < n; ++i) {
      if (!THPVariable_CheckExact(items[i])) Py_RETURN_NONE;
      const at::Tensor& t = THPVariable_Unpack(items[i]);
      if (!t.defined() || !t.is_cuda() || t.layout() != at::kStrided || !t.is_contiguous())
        Py_RETURN_NONE;
      const int on = static_cast<int>(t.get_device());
      if (i == 0) {
        device = on;
        if (args[1] == Py_None) {
          if (t.dim() == 0) Py_RETURN_NONE;
          blocks = t.size(0);
        }
        if (blocks <= 0) Py_RETURN_NONE;
      }
      if (on != device) Py_RETURN_NONE;
      const int64_t page = static_cast<int64_t>(t.nbytes()) / blocks;
      const void* base = t.data_ptr();
      std::memcpy(PyBytes_AS_STRING(bases.p) + 8 * i, &base, 8);
      std::memcpy(PyBytes_AS_STRING(pages.p) + 8 * i, &page, 8);
    }
  } catch (...) {
    Py_RETURN_NONE;  // the general path meets the same error and reports it
  }
  return Py_BuildValue("iLNN", device, static_cast<long long>(blocks), bases.release(),
                       pages.release());
}

// pack_ids(ids) -> the packed 8-byte values of a list of Python integers, or None.
PyObject* pack_ids(PyObject*, PyObject* seq) {
  if (!plain_sequence(seq)) Py_RETURN_NONE;
  const Py_ssize_t n = PySequence_Fast_GET_SIZE(seq);
  PyObject** items = PySequence_Fast_ITEMS(seq);
  Ref out(PyBytes_FromStringAndSize(nullptr, n * 8));
  if (!out.p) return nullptr;
  char* to = PyBytes_AS_STRING(out.p);
  for (Py_ssize_t i = 0; i < n; ++i) {
    if (!PyLong_CheckExact(items[i])) Py_RETURN_NONE;  // booleans and numpy integers too
    int overflow = 0;
    const long long v = PyLong_AsLongLongAndOverflow(items[i], &overflow);
    if (overflow) Py_RETURN_NONE;
    std::memcpy(to + 8 * i, &v, 8);
  }
  return out.release();
}

// pack_ids32(ids, limit) -> the packed 4-byte values of a list of Python
// integers, each in [0, limit), or None.
PyObject* pack_ids32(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  if (nargs != 2) {
    PyErr_SetString(PyExc_TypeError, "pack_ids32(ids, limit)");
    return nullptr;
  }
  const int64_t limit = PyLong_AsLongLong(args[1]);
  if (limit == -1 && PyErr_Occurred()) return nullptr;
  PyObject* seq = args[0];
  if (!plain_sequence(seq)) Py_RETURN_NONE;
  const Py_ssize_t n = PySequence_Fast_GET_SIZE(seq);
  PyObject** items = PySequence_Fast_ITEMS(seq);
  Ref out(PyBytes_FromStringAndSize(nullptr, n * 4));
  if (!out.p) return nullptr;
  char* to = PyBytes_AS_STRING(out.p);
  for (Py_ssize_t i = 0; i < n; ++i) {
    if (!PyLong_CheckExact(items[i])) Py_RETURN_NONE;
    int overflow = 0;
    const long long v = PyLong_AsLongLongAndOverflow(items[i], &overflow);
    if (overflow || v < 0 || v >= limit || v > INT32_MAX) Py_RETURN_NONE;
    const int32_t x = static_cast<int32_t>(v);
    std::memcpy(to + 4 * i, &x, 4);
  }
  return out.release();
}

// What QuantCache and CacheBatch keep for these calls, packed by _lib.
struct CacheArgs {
  int64_t write, read, attend;   // addresses of the C entry points
  int64_t format, head_dim, k_pages, v_pages;
  int64_t kv_heads, block_size, num_blocks, device;
};
struct BatchArgs {
  int64_t host_plan, device_plan, stream;
  int64_t kv_heads, heads, block_size, num_blocks, device;
  int64_t num_tokens, read_tokens;
  int64_t workspace[3];          // bytes for heads 64, 128 and 256 wide
};

typedef int (*WriteFn)(const void*, const void*, int, int32_t, void*, void*, const void*, int64_t,
                       int64_t, const void*, int64_t, int64_t, int64_t, int, void*);
typedef int (*ReadFn)(const void*, const void*, int, int32_t, const void*, const void*, int, void*,
                      int64_t, int64_t, void*, int64_t, int64_t, int64_t, int, void*);
typedef int (*AttendFn)(const void*, const void*, int, int32_t, const void*, const void*,
                        const void*, int64_t, int64_t, void*, int64_t, int64_t, int64_t, int,
                        double, void*, int64_t, void*);

template <typename P>
P* at_address(int64_t a) {
  return reinterpret_cast<P*>(static_cast<intptr_t>(a));
}

// AEGKV_DTYPE_* of a type, 0 for others
int dtype_code(at::ScalarType t) {
  return t == at::kBFloat16 ? 1 : t == at::kHalf ? 2 : t == at::kFloat ? 3 : 0;
}

// The arguments of one call: cache, batch, raw stream, current device.
struct QuantArgs {
  CacheArgs c;
  BatchArgs b;
  void* stream;

  bool take(PyObject* cache, PyObject* batch, PyObject* raw, PyObject* current) {
    if (!PyBytes_CheckExact(cache) || !PyBytes_CheckExact(batch) || !PyLong_CheckExact(raw) ||
        !PyLong_CheckExact(current) || PyBytes_GET_SIZE(cache) != sizeof c ||
        PyBytes_GET_SIZE(batch) != sizeof b)
      return false;
    std::memcpy(&c, PyBytes_AS_STRING(cache), sizeof c);
    std::memcpy(&b, PyBytes_AS_STRING(batch), sizeof b);
    const int64_t s = PyLong_AsLongLong(raw);
    stream = at_address<void>(s);
    return s == b.stream && PyLong_AsLongLong(current) == c.device && b.device == c.device &&
           b.kv_heads == c.kv_heads && b.block_size == c.block_size &&
           b.num_blocks <= c.num_blocks && !PyErr_Occurred();
  }

  // A [tokens, heads, head_dim] tensor of the cache's device.
  const at::Tensor* rows(PyObject* o, int64_t heads) const {
    if (!THPVariable_CheckExact(o)) return nullptr;
    const at::Tensor& t = THPVariable_Unpack(o);
    if (!t.defined() || !t.is_cuda() || t.get_device() != c.device ||
        t.layout() != at::kStrided || t.dim() != 3 || t.size(1) != heads ||
        t.size(2) != c.head_dim || !dtype_code(t.scalar_type()) || t.stride(2) != 1 ||
        t.size(0) == 0 || (t.requires_grad() && c10::GradMode::is_enabled()) ||
        t._fw_grad(0).defined())
      return nullptr;
    return &t;
  }
};

bool alike(const at::Tensor& a, const at::Tensor& b) {
  return a.scalar_type() == b.scalar_type() && a.size(0) == b.size(0);
}

// quant_write(cache, batch, k, v, stream, device) -> True, a status, or None
PyObject* quant_write(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  QuantArgs q;
  if (nargs != 6 || !q.take(args[0], args[1], args[4], args[5])) Py_RETURN_NONE;
  try {
    const at::Tensor* k = q.rows(args[2], q.c.kv_heads);
    const at::Tensor* v = q.rows(args[3], q.c.kv_heads);
    if (!k || !v || !alike(*k, *v)) Py_RETURN_NONE;
    const int status = at_address<std::remove_pointer_t<WriteFn>>(q.c.write)(
            at_address<void>(q.b.host_plan), at_address<void>(q.b.device_plan),
            static_cast<int>(q.c.format), static_cast<int32_t>(q.c.head_dim),
            at_address<void>(q.c.k_pages), at_address<void>(q.c.v_pages), k->data_ptr(),
            k->stride(0), k->stride(1), v->data_ptr(), v->stride(0), v->stride(1), k->size(0),
            dtype_code(k->scalar_type()), q.stream);
    if (status) return PyLong_FromLong(status);
    Py_RETURN_TRUE;
  } catch (...) {
    Py_RETURN_NONE;
  }
}

// quant_read(cache, batch, new tokens, out or dtype code, stream, device) -> (k, v), a
// status, or None
PyObject* quant_read(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  QuantArgs q;
  if (nargs != 6 || !q.take(args[0], args[1], args[4], args[5])) Py_RETURN_NONE;
  try {
    const bool fresh = args[2] == Py_True;
    Ref made(nullptr);
    PyObject* out = args[3];
    if (PyLong_CheckExact(out)) {
      const long code = PyLong_AsLong(out);
      const int64_t tokens = fresh ? q.b.num_tokens : q.b.read_tokens;
      if (tokens <= 0 || code < 1 || code > 3) Py_RETURN_NONE;
      const auto options =
          at::TensorOptions()
              .dtype(code == 1 ? at::kBFloat16 : code == 2 ? at::kHalf : at::kFloat)
              .device(at::kCUDA, static_cast<c10::DeviceIndex>(q.c.device));
      at::Tensor k = at::empty({tokens, q.c.kv_heads, q.c.head_dim}, options);
      at::Tensor v = at::empty({tokens, q.c.kv_heads, q.c.head_dim}, options);
      made.p = PyTuple_New(2);
      if (!made.p) return nullptr;
      for (int i = 0; i < 2; ++i) {
        PyObject* wrapped = THPVariable_Wrap(i ? v : k);
        if (!wrapped) return nullptr;
        PyTuple_SET_ITEM(made.p, i, wrapped);
      }
      out = made.p;
    }
    if (!PyTuple_CheckExact(out) || PyTuple_GET_SIZE(out) != 2) Py_RETURN_NONE;
    const at::Tensor* k = q.rows(PyTuple_GET_ITEM(out, 0), q.c.kv_heads);
    const at::Tensor* v = q.rows(PyTuple_GET_ITEM(out, 1), q.c.kv_heads);
    if (!k || !v || !alike(*k, *v)) Py_RETURN_NONE;
    const int status = at_address<std::remove_pointer_t<ReadFn>>(q.c.read)(
            at_address<void>(q.b.host_plan), at_address<void>(q.b.device_plan),
            static_cast<int>(q.c.format), static_cast<int32_t>(q.c.head_dim),
            at_address<void>(q.c.k_pages), at_address<void>(q.c.v_pages), fresh, k->data_ptr(),
            k->stride(0), k->stride(1), v->data_ptr(), v->stride(0), v->stride(1), k->size(0),
            dtype_code(k->scalar_type()), q.stream);
    if (status) return PyLong_FromLong(status);
    if (made.p) return made.release();
    Py_INCREF(out);
    return out;
  } catch (...) {
    Py_RETURN_NONE;
  }
}

// quant_attend(cache, batch, q, out or None, scale or None, stream, device) -> out, a
// status, or None
PyObject* quant_attend(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  QuantArgs q;
  if (nargs != 7 || !q.take(args[0], args[1], args[5], args[6])) Py_RETURN_NONE;
  try {
    const at::Tensor* query = q.rows(args[2], q.b.heads);
    if (!query || query->scalar_type() == at::kFloat) Py_RETURN_NONE;
    double scale = q.c.head_dim == 64 ? 0.125 : q.c.head_dim == 256 ? 0.0625 : 0.08838834764831845;
    if (args[4] != Py_None) {
      if (!PyFloat_CheckExact(args[4])) Py_RETURN_NONE;
      scale = PyFloat_AS_DOUBLE(args[4]);
    }
    Ref result(nullptr);
    if (args[3] == Py_None) {
      result.p = THPVariable_Wrap(
          at::empty(query->sizes(), query->options().requires_grad(false)));
      if (!result.p) return nullptr;
    } else {
      Py_INCREF(args[3]);
      result.p = args[3];
    }
    const at::Tensor* out = q.rows(result.p, q.b.heads);
    if (!out || !alike(*query, *out)) Py_RETURN_NONE;
    const int64_t bytes = q.b.workspace[q.c.head_dim == 64 ? 0 : q.c.head_dim == 128 ? 1 : 2];
    at::Tensor work;   // goes back to the stream's pool, behind the call
    if (bytes) work = at::empty({bytes}, query->options().dtype(at::kByte).requires_grad(false));
    const int status = at_address<std::remove_pointer_t<AttendFn>>(q.c.attend)(
            at_address<void>(q.b.host_plan), at_address<void>(q.b.device_plan),
            static_cast<int>(q.c.format), static_cast<int32_t>(q.c.head_dim),
            at_address<void>(q.c.k_pages), at_address<void>(q.c.v_pages), query->data_ptr(),
            query->stride(0), query->stride(1), out->data_ptr(), out->stride(0), out->stride(1),
            query->size(0), dtype_code(query->scalar_type()), scale,
            bytes ? work.data_ptr() : nullptr, bytes, q.stream);
    return status ? PyLong_FromLong(status) : result.release();
  } catch (...) {
    Py_RETURN_NONE;
  }
}

template <typename F>
PyCFunction as_method(F* f) {
  return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f));
}

PyMethodDef methods[] = {
    {"segment_table", as_method(segment_table), METH_FASTCALL, nullptr},
    {"pack_ids32", as_method(pack_ids32), METH_FASTCALL, nullptr},
    {"pack_ids", pack_ids, METH_O, nullptr},
    {"quant_write", as_method(quant_write), METH_FASTCALL, nullptr},
    {"quant_read", as_method(quant_read), METH_FASTCALL, nullptr},
    {"quant_attend", as_method(quant_attend), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_hostargs", nullptr, -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

// torch_version: the torch whose tensor layout this was compiled against.
PyMODINIT_FUNC PyInit__hostargs() {
  PyObject* m = PyModule_Create(&module);
  if (m && PyModule_AddStringConstant(m, "torch_version", AEGKV_TORCH_VERSION) != 0) {
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
