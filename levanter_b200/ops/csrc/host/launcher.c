// Calls a launcher of the kernel library with numbers from Python: what ctypes does, in a tenth of its time (20 arguments: 2.3 -> 0.3 us), which counts
// where a step's kernels are shorter than the calls that launch them.
//
// call(address, kinds, ...): `kinds` has a letter per argument, 'f' for a float and anything else for a pointer or a whole number.  In the calling conventions
// of 64-bit Linux (System V x86-64, AAPCS64) whole numbers and floats are passed in two sequences that do not depend on each other, a whole number of 32 bits takes
// the place of one of 64, and arguments that the callee does not have are not looked at; so one type of function serves for all of them.
#define Py_LIMITED_API 0x030A0000  // one library for all Pythons from 3.10 on
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <limits.h>
#include <stdint.h>

#if !(defined(__linux__) && (defined(__x86_64__) || defined(__aarch64__)))
#error "the calling convention is not known to pass whole numbers and floats in sequences of their own"
#endif

enum { kWhole = 24, kFloats = 8 };
typedef int (*Launcher)(long, long, long, long, long, long, long, long, long, long, long, long, long, long, long, long, long, long, long, long, long, long, long, long,
                        float, float, float, float, float, float, float, float);

static PyObject* call(PyObject* self, PyObject* const* args, Py_ssize_t n) {
  (void)self;
  const char* kinds;
  Py_ssize_t count;
  if (n < 2 || (kinds = PyUnicode_AsUTF8AndSize(args[1], &count)) == NULL) {
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_TypeError, "call(address, kinds, ...)");
    return NULL;
  }
  if (count != n - 2) return PyErr_Format(PyExc_TypeError, "%zd arguments expected, got %zd", count, n - 2);
  const unsigned long long address = PyLong_AsUnsignedLongLong(args[0]);
  if (PyErr_Occurred()) return NULL;
  long a[kWhole] = {0};
  float f[kFloats] = {0};
  int whole = 0, floats = 0;
  for (Py_ssize_t i = 0; i < count; ++i) {
    if (kinds[i] == 'f') {
      const double v = PyFloat_AsDouble(args[i + 2]);
      if ((v == -1.0 && PyErr_Occurred()) || floats == kFloats) goto refuse;
      f[floats++] = (float)v;
    } else {
      const long v = PyLong_AsLong(args[i + 2]);
      if ((v == -1 && PyErr_Occurred()) || whole == kWhole) goto refuse;
      if (kinds[i] == 'i' && (v < INT_MIN || v > INT_MAX)) return PyErr_Format(PyExc_OverflowError, "argument %zd does not fit into 32 bits", i);
      a[whole++] = v;
    }
  }
  int rc;
  Py_BEGIN_ALLOW_THREADS  // a launch may wait for room in the stream, and what it waits for may need the interpreter
  rc = ((Launcher)(uintptr_t)address)(a[0], a[1], a[2], a[3], a[4], a[5], a[6], a[7], a[8], a[9], a[10], a[11], a[12], a[13], a[14], a[15], a[16], a[17], a[18], a[19],
                                      a[20], a[21], a[22], a[23], f[0], f[1], f[2], f[3], f[4], f[5], f[6], f[7]);
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(rc);
refuse:
  if (!PyErr_Occurred()) PyErr_SetString(PyExc_TypeError, "too many arguments");
  return NULL;
}

static PyMethodDef methods[] = {{"call", (PyCFunction)(void (*)(void))call, METH_FASTCALL, "call(address, kinds, ...) -> int"}, {NULL, NULL, 0, NULL}};
static struct PyModuleDef module = {PyModuleDef_HEAD_INIT, "_lvb_launcher", NULL, -1, methods, NULL, NULL, NULL, NULL};
PyMODINIT_FUNC PyInit__lvb_launcher(void) { return PyModule_Create(&module); }
