// Argument checks of the post-training operators at C++ speed (the Python checks of native.py take longer than the
// smallest calls' kernels). pack(kinds, tensors) returns the tensors' part of an entry point's argument list, in order,
// or None when anything is not as the entry point wants it; native.py then goes through its own checks, which say what.
//
//   kind  tensor                                              becomes
//   L     logits [B, T, V] or [M, V], bf16 / fp16 / fp32      address, type, batch stride, token stride, B, T, V
//   G     gradient rows for L, or None                        address, batch stride, token stride
//   X     bf16 matrix [rows, K], unit stride along K          address, row stride (the first one's rows are M)
//   y f   int64 / fp32 of L's (X's) leading shape             address
//   b h c fp32 [B] / fp32 [B / 2] / int32 [B]                 address
//   a     fp32 [B], or of the leading shape                   address, 1 for the leading shape
//   1 4   fp32 [1] / [4]                                      address
//   u s   uint8 [n] / fp32 [ceil(n / 256)]                    address
//   F R   as f, b, or None                                    address or None
//   W     fp64 of the leading shape; None: allocated          address
//   P     fp32, 4 M ceil(V / 128) at least; None: allocated   address, their number
//   z     fp32, contiguous: gives N its shape, and n          nothing
//   N     None: fp32 of z's shape is allocated                address
// All tensors are on one GPU, whose index follows the arguments; behind it stand the tensors allocated here, which live
// as long as the list.
#define PY_SSIZE_T_CLEAN
#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstdint>

namespace {

struct Pack {
  PyObject* out;  // list under construction
  int64_t B = 0, T = 1, V = 0, M = 0, K = 0, n = -1;
  int lead = 0;  // leading dimensions: 1 or 2
  int64_t device = -1;
  const at::Tensor* logits = nullptr;
  const at::Tensor* like = nullptr;  // the first tensor: what is allocated goes where it is
  const at::Tensor* shape = nullptr;  // z
  at::Tensor made[2];
  int n_made = 0;
  bool ok = true;

  void put(int64_t v) {
    PyObject* o = PyLong_FromLongLong(v);
    if (o == nullptr || PyList_Append(out, o) != 0) ok = false;
    Py_XDECREF(o);
  }
  void put_none() {
    if (PyList_Append(out, Py_None) != 0) ok = false;
  }
  void put_address(const at::Tensor& t) { put((int64_t) reinterpret_cast<uintptr_t>(t.unsafeGetTensorImpl()->data())); }
  bool here(const at::Tensor& t) {
    if (!t.defined() || !t.is_cuda()) return false;
    const int64_t d = t.get_device();
    if (device < 0) device = d, like = &t;
    return d == device;
  }
  bool is(const at::Tensor& t, at::ScalarType s) { return t.scalar_type() == s && here(t) && t.is_contiguous(); }
  bool leading(const at::Tensor& t) {
    return lead == 2 ? t.dim() == 2 && t.size(0) == B && t.size(1) == T : t.dim() == 1 && t.size(0) == B;
  }
  bool vec(const at::Tensor& t, int64_t n_) { return t.dim() == 1 && t.size(0) == n_; }

  static int dtype(const at::Tensor& t) {
    switch (t.scalar_type()) {
      case at::kBFloat16: return 0;
      case at::kHalf: return 1;
      case at::kFloat: return 2;
      default: return -1;
    }
  }
  // strides of logits or their gradient; false for shapes and strides that are not rows
  static bool rows(const at::Tensor& t, int64_t* sb, int64_t* st) {
    const int64_t d = t.dim();
    if ((d != 2 && d != 3) || t.size(d - 1) < 1 || (t.size(d - 1) > 1 && t.stride(d - 1) != 1)) return false;
    *sb = t.stride(0);
    *st = d == 3 ? t.stride(1) : 0;
    return true;
  }
  static int64_t end(const at::Tensor& t) {
    int64_t last = 1;
    for (int64_t i = 0; i < t.dim(); ++i) last += (t.size(i) - 1) * t.stride(i);
    return (int64_t) reinterpret_cast<uintptr_t>(t.unsafeGetTensorImpl()->data()) + last * (int64_t)t.element_size();
  }

  bool add(char kind, const at::Tensor* tp) {
    if (tp == nullptr) {  // None
      if (kind == 'G') {
        put_none(), put(0), put(0);
        return ok;
      }
      if (kind == 'F' || kind == 'R') {
        put_none();
        return ok;
      }
      if ((kind == 'W' || kind == 'P' || kind == 'N') && like != nullptr && n_made < 2) {
        const int64_t floats = 4 * M * ((V + 127) / 128);
        if (kind == 'N' && shape == nullptr) return false;
        at::Tensor& t = made[n_made++];
        t = kind == 'P'   ? at::empty({floats}, like->options().dtype(at::kFloat))
            : kind == 'N' ? at::empty(shape->sizes(), like->options().dtype(at::kFloat))
                          : at::empty({B * T}, like->options().dtype(at::kDouble));
        put_address(t);
        if (kind == 'P') put(floats);
        return ok;
      }
      return false;
    }
    const at::Tensor& t = *tp;
    switch (kind) {
      case 'L': {
        int64_t sb, st;
        if (dtype(t) < 0 || !here(t) || !rows(t, &sb, &st)) return false;
        lead = (int)t.dim() - 1;
        B = t.size(0), T = lead == 2 ? t.size(1) : 1, V = t.size(lead);
        if (B < 1 || T < 1 || B > INT32_MAX || T > INT32_MAX || B * T > INT32_MAX || V > (1 << 30)) return false;
        logits = tp;
        put_address(t), put(dtype(t)), put(sb), put(st), put(B), put(T), put(V);
        return ok;
      }
      case 'G': {
        int64_t sb, st;
        if (logits == nullptr || t.scalar_type() != logits->scalar_type() || !here(t) || t.sizes() != logits->sizes() ||
            !rows(t, &sb, &st))
          return false;
        if (!t.is_contiguous() && !((T == 1 || st >= V) && (B == 1 || sb >= (T - 1) * st + V)) &&
            !(sb >= V && st >= (B - 1) * sb + V))
          return false;
        const int64_t at = (int64_t) reinterpret_cast<uintptr_t>(t.unsafeGetTensorImpl()->data());
        const int64_t of = (int64_t) reinterpret_cast<uintptr_t>(logits->unsafeGetTensorImpl()->data());
        if ((at != of || t.strides() != logits->strides()) && at < end(*logits) && of < end(t)) return false;
        put(at), put(sb), put(st);
        return ok;
      }
      case 'X': {
        if (t.scalar_type() != at::kBFloat16 || !here(t) || t.dim() != 2 || t.size(0) < 1 || t.size(1) < 1 ||
            t.size(0) > INT32_MAX || t.size(1) > INT32_MAX || t.stride(1) != 1 || t.stride(0) % 8 != 0 ||
            t.stride(0) < t.size(1))
          return false;
        if (M == 0) {
          M = B = t.size(0), K = t.size(1), lead = 1;
        } else {
          V = t.size(0);
          if (t.size(1) != K) return false;
        }
        put_address(t), put(t.stride(0));
        return ok;
      }
      case 'y': if (!is(t, at::kLong) || !leading(t)) return false; break;
      case 'f': case 'F': if (!is(t, at::kFloat) || !leading(t)) return false; break;
      case 'W': if (!is(t, at::kDouble) || !leading(t)) return false; break;
      case 'b': case 'R': if (!is(t, at::kFloat) || !vec(t, B)) return false; break;
      case 'h': if (!is(t, at::kFloat) || B % 2 != 0 || !vec(t, B / 2)) return false; break;
      case 'c': if (!is(t, at::kInt) || !vec(t, B)) return false; break;
      case '1': if (!is(t, at::kFloat) || !vec(t, 1)) return false; break;
      case '4': if (!is(t, at::kFloat) || !vec(t, 4)) return false; break;
      case 'a': {
        const bool per_sequence = vec(t, B);
        if (!is(t, at::kFloat) || !(per_sequence || leading(t))) return false;
        put_address(t), put(per_sequence ? 0 : 1);
        return ok;
      }
      case 'P':
        if (!is(t, at::kFloat) || t.numel() < 4 * M * ((V + 127) / 128)) return false;
        put_address(t), put(t.numel());
        return ok;
      case 'z':
        if (!is(t, at::kFloat)) return false;
        shape = tp, n = t.numel();
        return true;
      case 'u':
        if (!is(t, at::kByte) || !vec(t, n) || n < 1) return false;
        break;
      case 's': if (!is(t, at::kFloat) || !vec(t, (n + 255) / 256)) return false; break;
      default: return false;
    }
    put_address(t);
    return ok;
  }
};

PyObject* pack(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  if (nargs != 2 || !PyUnicode_Check(args[0]) || !PyTuple_Check(args[1])) {
    PyErr_SetString(PyExc_TypeError, "pack(kinds, tensors)");
    return nullptr;
  }
  Py_ssize_t len = 0;
  const char* kinds = PyUnicode_AsUTF8AndSize(args[0], &len);
  if (kinds == nullptr) return nullptr;
  if (len != PyTuple_GET_SIZE(args[1])) {
    PyErr_SetString(PyExc_ValueError, "pack: one kind a tensor");
    return nullptr;
  }
  Pack p;
  p.out = PyList_New(0);
  if (p.out == nullptr) return nullptr;
  bool good = true;
  try {
    for (Py_ssize_t i = 0; i < len && good; ++i) {
      PyObject* o = PyTuple_GET_ITEM(args[1], i);
      if (o == Py_None) good = p.add(kinds[i], nullptr);
      else if (THPVariable_Check(o)) good = p.add(kinds[i], &THPVariable_Unpack(o));
      else good = false;
    }
  } catch (const std::exception&) {  // a tensor without storage or strides: the Python checks name it
    good = false;
  }
  if (good) {
    p.put(p.device);
    for (int i = 0; i < p.n_made; ++i) {
      PyObject* o = THPVariable_Wrap(p.made[i]);
      if (o != nullptr) PyList_Append(p.out, o);
      Py_XDECREF(o);
    }
  }
  if (PyErr_Occurred()) {
    Py_DECREF(p.out);
    return nullptr;
  }
  if (!good) {
    Py_DECREF(p.out);
    Py_RETURN_NONE;
  }
  return p.out;
}

PyMethodDef methods[] = {{"pack", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(pack)), METH_FASTCALL,
                          "pack(kinds, tensors): the tensors' part of an entry point's arguments, or None"},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module_def = {PyModuleDef_HEAD_INIT, "_fastargs", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__fastargs(void) { return PyModule_Create(&module_def); }
