// omni_tensors: what the Python mirror asks of a call's tensors, in one call.
//
// take(kinds, names, device, ...) checks each tensor and answers with its pointer
// (and stride or format) as a flat tuple; the first one that does not fit raises the
// mirror's error. A tensor asked in Python costs 0.28 us (type, size, contiguity,
// device, pointer: a method call each), so that the row tables' 13 cost more
// than their kernel's launch; here they cost 0.4 us together.
//
// One letter of `kinds` each, a capital where None will do, and what follows it:
//   i tensor, least           contiguous int32 of at least `least`   -> pointer
//   b tensor, least           the same of bf16                       -> pointer
//   r tensor, rows, width     bf16 [>= rows][width], elements of a row adjacent -> pointer, row stride
//   c kv, kv_scale, 2 hk      the 8-bit cache and its exponents      -> pointer, pointer, format
//   p kv, kv_scale, page      a cache of one layer or several, 8-bit or (kv_scale None) bf16 slots or bytes [slots][bytes of one]
//                             -> pointer, pointer, layers, blocks (slots), bytes and exponents of one, and how many a page has
#include <Python.h>
#include <torch/csrc/autograd/python_variable.h>

#include <string>

namespace {

PyObject* g_error = nullptr;  // the mirror's error class
long g_code = 0;              // its code for a bad argument

struct Bad {
  std::string what;
};

const at::Tensor& tensor_of(PyObject* o, const char* what) {
  if (!THPVariable_Check(o)) throw Bad{std::string(what) + " must be a tensor"};
  return THPVariable_Unpack(o);
}

int64_t int_of(PyObject* o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    throw Bad{": a count is not an integer"};
  }
  return v;
}

void check_device(const at::Tensor& t, int64_t device) {
  if (t.is_cuda() && t.get_device() == device) return;
  throw Bad{" must lie on the current device, with the other tensors"};
}

struct Answer {
  PyObject* tuple;
  Py_ssize_t n = 0;
  void put(PyObject* o) {
    if (!o) throw std::bad_alloc();
    PyTuple_SET_ITEM(tuple, n++, o);
  }
  void put_ptr(const at::Tensor& t) { put(PyLong_FromVoidPtr(t.mutable_data_ptr())); }
};

// Letter `kind` with its arguments a[0 ..], `left` of them; how many it took.
int take_one(char kind, PyObject* const* a, Py_ssize_t left, int64_t device, Answer& out) {
  const char k = kind | 0x20;
  const int args = k == 'i' || k == 'b' ? 2 : 3;
  if (left < args) throw Bad{": too few arguments"};
  if (kind != k && a[0] == Py_None) {
    out.put(Py_NewRef(Py_None));
    if (k == 'r') out.put(PyLong_FromLong(0));
    return args;
  }
  const at::Tensor& t = tensor_of(a[0], "");
  if (k == 'i' || k == 'b') {
    const int64_t least = int_of(a[1]);
    if (t.scalar_type() != (k == 'i' ? at::kInt : at::kBFloat16) || t.numel() < least || !t.is_contiguous())
      throw Bad{std::string(" must be a contiguous ") + (k == 'i' ? "int32" : "bf16") + " tensor of at least " +
                std::to_string(least)};
    check_device(t, device);
    out.put_ptr(t);
  } else if (k == 'r') {
    const int64_t rows = int_of(a[1]), width = int_of(a[2]);
    if (t.scalar_type() != at::kBFloat16 || t.dim() != 2 || t.size(0) < rows || t.size(1) != width)
      throw Bad{" must be bf16 rows [" + std::to_string(rows) + "][" + std::to_string(width) + "]"};
    if (t.stride(1) != 1) throw Bad{": the elements of a row must be adjacent"};
    check_device(t, device);
    out.put_ptr(t);
    out.put(PyLong_FromLongLong(t.size(0) > 1 ? t.stride(0) : width));
  } else if (k == 'c') {
    const at::Tensor& s = tensor_of(a[1], "");
    const int64_t heads = int_of(a[2]);
    const auto type = t.scalar_type(), exps = s.scalar_type();
    const int format = type == at::kFloat8_e4m3fn ? 0 : type == at::kChar ? 1 : -1;
    if (format < 0 || t.dim() != 3 || t.size(1) != heads || t.size(2) != 2048)
      throw Bad{" must be float8_e4m3fn or int8 [blocks][" + std::to_string(heads) + "][2048]"};
    if ((exps != at::kByte && exps != at::kFloat8_e8m0fnu) || s.dim() != 2 || s.size(0) != t.size(0) || s.size(1) != heads)
      throw Bad{"'s kv_scale must be uint8 or float8_e8m0fnu [" + std::to_string(t.size(0)) + "][" + std::to_string(heads) + "]"};
    if (!t.is_contiguous() || !s.is_contiguous()) throw Bad{" and kv_scale must be contiguous"};
    check_device(t, device);
    check_device(s, device);
    out.put_ptr(t);
    out.put_ptr(s);
    out.put(PyLong_FromLong(format));
  } else if (k == 'p') {
    const int64_t page = int_of(a[2]);
    const bool slots = a[1] == Py_None;
    const auto type = t.scalar_type();
    if (slots && type == at::kByte) {  // FP8 slots, or any of so many bytes
      if (t.dim() != 2 && t.dim() != 3) throw Bad{" must be uint8 slots [slots][bytes], or layers of them"};
      const int64_t layers = t.dim() == 3 ? t.size(0) : 1, units = t.size(t.dim() - 2);
      if (page <= 0) throw Bad{": page=" + std::to_string(page)};
      if (units % page != 0) throw Bad{" must hold whole pages"};
      if (!t.is_contiguous()) throw Bad{" must be contiguous"};
      check_device(t, device);
      out.put_ptr(t);
      out.put(Py_NewRef(Py_None));
      for (const int64_t v : {layers, units, t.size(t.dim() - 1), (int64_t)0, page}) out.put(PyLong_FromLongLong(v));
      return args;
    }
    const int64_t lead = t.dim() - 3;  // layers before the blocks
    const bool shaped = (lead == 0 || lead == 1) && t.size(lead + 1) > 0 && t.size(lead + 1) % 2 == 0;
    if (slots ? type != at::kBFloat16 || !shaped || t.size(lead + 2) != 128
              : (type != at::kFloat8_e4m3fn && type != at::kChar) || !shaped || t.size(lead + 2) != 2048)
      throw Bad{slots ? " must be bf16 slots [slots][2 hk][128] or uint8 slots [slots][bytes], or layers of them"
                      : " must be float8_e4m3fn or int8 [blocks][2 hk][2048], or layers of it"};
    const int64_t units = t.size(lead), heads = t.size(lead + 1), layers = lead ? t.size(0) : 1;
    if (page <= 0 || (!slots && page % 16 != 0)) throw Bad{": page=" + std::to_string(page)};
    const int64_t per = slots ? page : page / 16;
    if (units % per != 0) throw Bad{" must hold whole pages"};
    if (!t.is_contiguous()) throw Bad{" must be contiguous"};
    check_device(t, device);
    out.put_ptr(t);
    if (slots) {
      out.put(Py_NewRef(Py_None));
    } else {
      const at::Tensor& s = tensor_of(a[1], "");
      const auto exps = s.scalar_type();
      if ((exps != at::kByte && exps != at::kFloat8_e8m0fnu) || s.dim() != t.dim() - 1 || s.size(lead) != units ||
          s.size(lead + 1) != heads || (lead && s.size(0) != layers) || !s.is_contiguous())
        throw Bad{"'s kv_scale must be contiguous uint8 or float8_e8m0fnu of its shape without the last dimension"};
      check_device(s, device);
      out.put_ptr(s);
    }
    for (const int64_t v : {layers, units, heads * (slots ? 256 : 2048), slots ? 0 : heads, per}) out.put(PyLong_FromLongLong(v));
  } else {
    throw Bad{": no such kind"};
  }
  return args;
}

// The which-th of `names`, words with a space between two.
std::string name_of(const char* names, int which) {
  const char* at = names;
  for (; which > 0 && *at; ++at) which -= *at == ' ';
  const char* end = at;
  while (*end && *end != ' ') ++end;
  return std::string(at, end);
}

PyObject* take(PyObject*, PyObject* const* a, Py_ssize_t n) {
  Py_ssize_t letters = 0;
  const char* kinds = n >= 3 ? PyUnicode_AsUTF8AndSize(a[0], &letters) : nullptr;
  const char* names = kinds ? PyUnicode_AsUTF8(a[1]) : nullptr;
  if (!names) {
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_TypeError, "take(kinds, names, device, ...)");
    return nullptr;
  }
  Py_ssize_t values = 0;
  for (Py_ssize_t i = 0; i < letters; ++i) values += (kinds[i] | 0x20) == 'p' ? 7 : (kinds[i] | 0x20) == 'c' ? 3 : (kinds[i] | 0x20) == 'r' ? 2 : 1;
  PyObject* tuple = PyTuple_New(values);
  if (!tuple) return nullptr;
  Answer out{tuple};
  Py_ssize_t i = 0;
  std::string what;
  try {
    const int64_t device = int_of(a[2]);
    Py_ssize_t at = 3;
    for (; i < letters; ++i) at += take_one(kinds[i], a + at, n - at, device, out);
    if (at != n) throw Bad{": too many arguments"};
    return tuple;
  } catch (const Bad& bad) {
    what = bad.what;
  } catch (const std::exception& e) {
    what = std::string(": ") + e.what();
  }
  Py_DECREF(tuple);
  what = name_of(names, (int)i) + what;
  PyObject* args = Py_BuildValue("(ls)", g_code, what.c_str());
  if (args) PyErr_SetObject(g_error ? g_error : PyExc_ValueError, args);
  Py_XDECREF(args);
  return nullptr;
}

PyObject* set_error(PyObject*, PyObject* args) {
  PyObject* cls;
  long code;
  if (!PyArg_ParseTuple(args, "Ol", &cls, &code)) return nullptr;
  Py_INCREF(cls);
  Py_XSETREF(g_error, cls);
  g_code = code;
  Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"take", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(take)), METH_FASTCALL, "take(kinds, names, device, ...) -> tuple"},
    {"set_error", set_error, METH_VARARGS, "set_error(class, code): what take raises, as class(code, text)"},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "omni_tensors", "The Python mirror's checks of a call's tensors.", -1, methods};

}  // namespace

// The torch and Python whose headers it was compiled with: it reads their objects, so the mirror loads it beside no other.
#ifndef OMNI_BUILT_FOR
#error "build.py names the versions"
#endif

PyMODINIT_FUNC PyInit_omni_tensors() {
  PyObject* m = PyModule_Create(&module);
  if (m && PyModule_AddStringConstant(m, "built_for", OMNI_BUILT_FOR) != 0) Py_CLEAR(m);
  return m;
}
