/* CPython binding of the C-ABI entries that are called once per operator call: first
 * avo_b200_attn_fwd_ws, for attention(); the entries of the training side follow below.
 * Small problems are bound by host time per call (the B1 H4 S512 case of the scorer runs
 * ~15 us of GPU work per launch); a ctypes call with fifteen arguments costs ~2 us of argument
 * conversion, a METH_FASTCALL function a fraction of that.  The function address comes from
 * the library ctypes already loaded (bind), so this module links to nothing but Python and
 * calls exactly the same native entry.
 *
 * fwd_ws(q, k, v, o, lse_or_None, batch, heads, seq, head_dim, causal, scale,
 *        workspace, workspace_bytes, status, stream) -> int status code
 * Pointer arguments are integers (tensor.data_ptr()), lse may be None; the return value is
 * the entry's own status code. */
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <stddef.h>
#include <string.h>

typedef int (*fwd_ws_fn)(const void*, const void*, const void*, void*, float*, int, int, int, int, int, float,
                         void*, size_t, int*, void*);

static fwd_ws_fn g_fwd_ws = NULL;

static PyObject* bind(PyObject* self, PyObject* addr) {
  (void)self;
  void* fn = PyLong_AsVoidPtr(addr);
  if (fn == NULL) {
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "null function address");
    return NULL;
  }
  g_fwd_ws = (fwd_ws_fn)fn;
  Py_RETURN_NONE;
}

static int as_ptr(PyObject* obj, void** out) {
  if (obj == Py_None) {
    *out = NULL;
    return 0;
  }
  *out = PyLong_AsVoidPtr(obj);
  return (*out == NULL && PyErr_Occurred()) ? -1 : 0;
}

static int as_int(PyObject* obj, int* out) {
  long v = PyLong_AsLong(obj);
  if (v == -1 && PyErr_Occurred()) return -1;
  if (v < -2147483647L - 1L || v > 2147483647L) {
    PyErr_SetString(PyExc_OverflowError, "argument out of int range");
    return -1;
  }
  *out = (int)v;
  return 0;
}

static PyObject* fwd_ws(PyObject* self, PyObject* const* args, Py_ssize_t nargs) {
  (void)self;
  if (nargs != 15) {
    PyErr_SetString(PyExc_TypeError, "fwd_ws takes 15 arguments");
    return NULL;
  }
  if (g_fwd_ws == NULL) {
    PyErr_SetString(PyExc_RuntimeError, "fwd_ws is not bound to the library yet");
    return NULL;
  }
  void *q, *k, *v, *o, *lse, *ws, *status, *stream;
  int batch, heads, seq, head_dim, causal;
  if (as_ptr(args[0], &q) || as_ptr(args[1], &k) || as_ptr(args[2], &v) || as_ptr(args[3], &o) ||
      as_ptr(args[4], &lse) || as_int(args[5], &batch) || as_int(args[6], &heads) || as_int(args[7], &seq) ||
      as_int(args[8], &head_dim) || as_int(args[9], &causal))
    return NULL;
  const double scale = PyFloat_AsDouble(args[10]);
  if (scale == -1.0 && PyErr_Occurred()) return NULL;
  if (as_ptr(args[11], &ws)) return NULL;
  const size_t ws_bytes = PyLong_AsSize_t(args[12]);
  if (ws_bytes == (size_t)-1 && PyErr_Occurred()) return NULL;
  if (as_ptr(args[13], &status) || as_ptr(args[14], &stream)) return NULL;
  const int rc = g_fwd_ws(q, k, v, o, (float*)lse, batch, heads, seq, head_dim, causal, (float)scale, ws, ws_bytes,
                          (int*)status, stream);
  return PyLong_FromLong(rc);
}

/* ---------------------------------------------------------------- training entries
 * bind_entry(index, address) and call(index, args...) for the entries in `entries`; the
 * arguments are the entry's own, pointers as integers (0 or None: null). */
typedef union {
  void* p;
  int i;
  long long l;
  float f;
  size_t z;
} arg_t;

/* p pointer, i int, l long long, f float, z size_t */
#define ROPE_ARGS "iiiii" "ppippiii" "pilll" "ipf"
enum { FWD_GROUPED, BWD, ROPE, ROPE_BWD, N_ENTRIES };
static const char* const entries[N_ENTRIES] = {
    "pppppiiiiiiifpzpp",                       /* avo_b200_attn_fwd_grouped */
    "pppppppppiiiiiiifpzpp",                   /* avo_b200_attn_bwd */
    "pllppp" ROPE_ARGS "pp",                   /* avo_b200_qkv_norm_rope */
    "ppppllppp" ROPE_ARGS "pzpp",              /* avo_b200_qkv_norm_rope_bwd */
};
#define MAX_ARGS 40
static void* g_entry[N_ENTRIES];

static PyObject* bind_entry(PyObject* self, PyObject* const* args, Py_ssize_t nargs) {
  (void)self;
  int index;
  void* fn;
  if (nargs != 2) {
    PyErr_SetString(PyExc_TypeError, "bind_entry takes an index and an address");
    return NULL;
  }
  if (as_int(args[0], &index) || as_ptr(args[1], &fn)) return NULL;
  if (index < 0 || index >= N_ENTRIES || fn == NULL) {
    PyErr_SetString(PyExc_ValueError, "no such entry, or a null address");
    return NULL;
  }
  g_entry[index] = fn;
  Py_RETURN_NONE;
}

static int parse(const char* fmt, PyObject* const* in, arg_t* out) {
  for (; *fmt != 0; ++fmt, ++in, ++out) {
    switch (*fmt) {
      case 'p':
        if (as_ptr(*in, &out->p)) return -1;
        break;
      case 'i':
        if (as_int(*in, &out->i)) return -1;
        break;
      case 'l':
        out->l = PyLong_AsLongLong(*in);
        if (out->l == -1 && PyErr_Occurred()) return -1;
        break;
      case 'z':
        out->z = PyLong_AsSize_t(*in);
        if (out->z == (size_t)-1 && PyErr_Occurred()) return -1;
        break;
      default: {
        const double v = PyFloat_AsDouble(*in);
        if (v == -1.0 && PyErr_Occurred()) return -1;
        out->f = (float)v;
      }
    }
  }
  return 0;
}

typedef int (*grouped_fn)(const void*, const void*, const void*, void*, float*, int, int, int, int, int, int, int,
                          float, void*, size_t, int*, void*);
typedef int (*bwd_fn)(const void*, const void*, const void*, const void*, const void*, const float*, void*, void*,
                      void*, int, int, int, int, int, int, int, float, void*, size_t, int*, void*);
typedef int (*rope_fn)(const void*, long long, long long, void*, void*, void*, int, int, int, int, int, const void*,
                       const void*, int, const float*, const float*, int, int, int, const void*, int, long long,
                       long long, long long, int, const int*, float, int*, void*);
typedef int (*rope_bwd_fn)(const void*, const void*, const void*, const void*, long long, long long, void*, float*,
                           float*, int, int, int, int, int, const void*, const void*, int, const float*, const float*,
                           int, int, int, const void*, int, long long, long long, long long, int, const int*, float,
                           void*, size_t, int*, void*);

static PyObject* call(PyObject* self, PyObject* const* args, Py_ssize_t nargs) {
  (void)self;
  int index;
  if (nargs < 1) {
    PyErr_SetString(PyExc_TypeError, "call takes an entry index and its arguments");
    return NULL;
  }
  if (as_int(args[0], &index)) return NULL;
  if (index < 0 || index >= N_ENTRIES || g_entry[index] == NULL) {
    PyErr_SetString(PyExc_RuntimeError, "the entry is not bound to the library");
    return NULL;
  }
  const char* fmt = entries[index];
  if ((size_t)(nargs - 1) != strlen(fmt)) {
    PyErr_SetString(PyExc_TypeError, "wrong number of arguments for the entry");
    return NULL;
  }
  arg_t a[MAX_ARGS];
  if (parse(fmt, args + 1, a)) return NULL;
  int rc = 0;
  switch (index) {
    case FWD_GROUPED:
      rc = ((grouped_fn)g_entry[index])(a[0].p, a[1].p, a[2].p, a[3].p, a[4].p, a[5].i, a[6].i, a[7].i, a[8].i,
                                        a[9].i, a[10].i, a[11].i, a[12].f, a[13].p, a[14].z, a[15].p, a[16].p);
      break;
    case BWD:
      rc = ((bwd_fn)g_entry[index])(a[0].p, a[1].p, a[2].p, a[3].p, a[4].p, a[5].p, a[6].p, a[7].p, a[8].p, a[9].i,
                                    a[10].i, a[11].i, a[12].i, a[13].i, a[14].i, a[15].i, a[16].f, a[17].p, a[18].z,
                                    a[19].p, a[20].p);
      break;
    case ROPE:
      rc = ((rope_fn)g_entry[index])(a[0].p, a[1].l, a[2].l, a[3].p, a[4].p, a[5].p, a[6].i, a[7].i, a[8].i, a[9].i,
                                     a[10].i, a[11].p, a[12].p, a[13].i, a[14].p, a[15].p, a[16].i, a[17].i, a[18].i,
                                     a[19].p, a[20].i, a[21].l, a[22].l, a[23].l, a[24].i, a[25].p, a[26].f, a[27].p,
                                     a[28].p);
      break;
    default:
      rc = ((rope_bwd_fn)g_entry[index])(a[0].p, a[1].p, a[2].p, a[3].p, a[4].l, a[5].l, a[6].p, a[7].p, a[8].p,
                                         a[9].i, a[10].i, a[11].i, a[12].i, a[13].i, a[14].p, a[15].p, a[16].i,
                                         a[17].p, a[18].p, a[19].i, a[20].i, a[21].i, a[22].p, a[23].i, a[24].l,
                                         a[25].l, a[26].l, a[27].i, a[28].p, a[29].f, a[30].p, a[31].z, a[32].p,
                                         a[33].p);
  }
  return PyLong_FromLong(rc);
}

static PyMethodDef methods[] = {
    {"bind_entry", (PyCFunction)(void (*)(void))bind_entry, METH_FASTCALL, "bind_entry(index, address)"},
    {"call", (PyCFunction)(void (*)(void))call, METH_FASTCALL, "call(index, the entry's arguments...)"},
    {"bind", (PyCFunction)bind, METH_O, "bind(address of avo_b200_attn_fwd_ws)"},
    {"fwd_ws", (PyCFunction)(void (*)(void))fwd_ws, METH_FASTCALL, "avo_b200_attn_fwd_ws through the bound address"},
    {NULL, NULL, 0, NULL},
};

static struct PyModuleDef module = {PyModuleDef_HEAD_INIT, "_avo_b200_fast", NULL, -1, methods,
                                    NULL, NULL, NULL, NULL};

PyMODINIT_FUNC PyInit__avo_b200_fast(void) { return PyModule_Create(&module); }
