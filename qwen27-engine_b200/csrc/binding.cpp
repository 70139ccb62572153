// CPython binding of the entry points that an engine calls once per layer and step.
//
// A decode call behind a short context takes about ten microseconds on the GPU; the same call through ctypes
// takes longer than that on the host (a Python-level check and a ctypes object per tensor argument): prologue and
// decode of one token behind 256, 33.5 us a pass through ctypes, 9.3 through this binding. Here the
// arguments are read natively: same checks, same order, same errors. Anything that is not exactly a torch.Tensor
// or an nn.Parameter (a raw address, None, a subclass) goes through the module's Python-level check. The library
// stays the one that the Python module has loaded: it hands over the addresses of its functions.
#include <torch/csrc/autograd/python_variable.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>

#include <cstdint>

#include "q27b_attn.h"

namespace {

enum Fn { PREP, DECODE, PREP_PAGED, DECODE_PAGED, PREFILL, TREE, TREE_PAGED, COMMIT, COMMIT_PAGED, BOUNDS, BOUNDS_PAGED,
          SELECT, SELECT_PAGED, BLOCKS, BLOCKS_PAGED, N_FN };
// One per module object: the package may be loaded under two names, each with its own library and error class.
struct State {
  void* fn[N_FN];
  PyObject* ptr;    // _ptr(tensor, dtype, optional, numel) -> ctypes.c_void_p
  PyObject* check;  // _check(return code): raises
  PyObject *f32, *i32, *i8, *f16, *i64;  // torch.float32, int32, int8, float16, int64 as Python objects, for ptr
};
PyObject* dtype_object(const State* st, c10::ScalarType t) {
  return t == c10::kFloat ? st->f32 : t == c10::kInt ? st->i32 : t == c10::kChar ? st->i8
         : t == c10::kHalf ? st->f16 : t == c10::kLong ? st->i64 : Py_None;
}

// Device address of one tensor argument. want = Undefined: any dtype. least > 0: a tensor on the current device of at least
// that many elements (any dtype: bytes).
bool ptr(const State* st, PyObject* o, c10::ScalarType want, bool optional, void** out, int64_t least = 0) {
  if (THPVariable_CheckExact(o)) {
    const at::Tensor& t = THPVariable_Unpack(o);
    if (t.is_cuda() && t.is_contiguous() && (want == c10::ScalarType::Undefined || t.scalar_type() == want) &&
        (least <= 0 || ((want == c10::ScalarType::Undefined ? (int64_t)t.nbytes() : t.numel()) >= least && t.get_device() == c10::cuda::current_device()))) {
      *out = t.data_ptr();
      return true;
    }
  }
  PyObject* n = PyLong_FromLongLong(least);
  if (!n) return false;
  PyObject* r = PyObject_CallFunctionObjArgs(st->ptr, o, dtype_object(st, want), optional ? Py_True : Py_False, n, nullptr);
  Py_DECREF(n);
  if (!r) return false;
  PyObject* v = PyObject_GetAttrString(r, "value");
  Py_DECREF(r);
  if (!v) return false;
  *out = v == Py_None ? nullptr : PyLong_AsVoidPtr(v);
  Py_DECREF(v);
  return !PyErr_Occurred();
}

bool num(PyObject* o, int* out) {  // int(o), as ctypes takes it: the low 32 bits
  PyObject* l = PyLong_CheckExact(o) ? Py_NewRef(o) : PyObject_CallOneArg((PyObject*)&PyLong_Type, o);
  if (!l) return false;
  *out = (int)PyLong_AsUnsignedLongMask(l);
  Py_DECREF(l);
  return !PyErr_Occurred();
}
bool flt(PyObject* o, float* out) {
  *out = (float)PyFloat_AsDouble(o);
  return !PyErr_Occurred();
}
bool flag(PyObject* o, int* out) {
  const int t = PyObject_IsTrue(o);
  *out = t;
  return t >= 0;
}

PyObject* done(const State* st, int rc) {
  if (rc == 0) Py_RETURN_NONE;
  return PyObject_CallFunction(st->check, "i", rc);
}

constexpr c10::ScalarType F32 = c10::kFloat, I32 = c10::kInt, I8 = c10::kChar, F16 = c10::kHalf, I64 = c10::kLong, ANY = c10::ScalarType::Undefined;

// Runs `body`, turning C++ exceptions of torch into Python errors.
template <class B>
PyObject* guarded(PyObject* self, Py_ssize_t n, Py_ssize_t want, B body) {
  const State* st = (const State*)PyModule_GetState(self);
  if (!st || !st->ptr) return PyErr_Format(PyExc_RuntimeError, "q27b_binding is not bound");
  if (n != want) return PyErr_Format(PyExc_TypeError, "expected %zd arguments, got %zd", want, n);
  try {
    return body(st);
  } catch (const std::exception& e) {
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}
void* stream() { return (void*)c10::cuda::getCurrentCUDAStream().stream(); }

template <c10::ScalarType T> struct Elem { using type = void; };
template <> struct Elem<F32> { using type = float; };
template <> struct Elem<I32> { using type = int; };
template <> struct Elem<I8> { using type = int8_t; };
template <> struct Elem<I64> { using type = uint64_t; };

#define PTR(i, kind, opt, name)                            \
  void* name##_p;                                          \
  if (!ptr(st, a[i], kind, opt, &name##_p)) return nullptr; \
  Elem<kind>::type* name = static_cast<Elem<kind>::type*>(name##_p)
// The same with the number of elements that the call reads or writes there.
#define SIZED(i, kind, opt, name, n)                               \
  void* name##_p;                                                  \
  if (!ptr(st, a[i], kind, opt, &name##_p, (n))) return nullptr;   \
  Elem<kind>::type* name = static_cast<Elem<kind>::type*>(name##_p)
#define NUM(i, name) \
  int name;          \
  if (!num(a[i], &name)) return nullptr
#define FLT(i, name) \
  float name;        \
  if (!flt(a[i], &name)) return nullptr
#define FLAG(i, name) \
  int name;           \
  if (!flag(a[i], &name)) return nullptr
// The signature is the header's: a parameter added, taken out or of another type there does not compile here.
#define CALL(which, entry, ...)                                        \
  void* s = stream();                                                  \
  int rc;                                                              \
  Py_BEGIN_ALLOW_THREADS                                               \
  rc = reinterpret_cast<decltype(&entry)>(st->fn[which])(__VA_ARGS__); \
  Py_END_ALLOW_THREADS                                                 \
  return done(st, rc)

// qg, k, v, q_norm, k_norm, qn, kcache, vcache, pos0, T, eps, theta_scale, nqh, nkvh, n_ctx, q8, rope3, rdelta
PyObject* attn_prep(PyObject* self, PyObject* const* a, Py_ssize_t n) {
  return guarded(self, n, 18, [&](const State* st) -> PyObject* {
    PTR(0, F32, false, qg); PTR(1, F32, false, k); PTR(2, F32, false, v); PTR(3, F32, false, qw); PTR(4, F32, false, kw);
    PTR(5, F32, false, qn); PTR(6, ANY, false, kc); PTR(7, ANY, false, vc); PTR(8, I32, false, pos0);
    NUM(9, T); FLT(10, eps); FLT(11, theta); NUM(12, nqh); NUM(13, nkvh); NUM(14, n_ctx); FLAG(15, q8);
    PTR(16, I32, true, rope3); PTR(17, I32, true, rdelta);
    CALL(PREP, q27b_attn_prep, qg, k, v, qw, kw, qn, kc, vc, pos0, T, eps, theta, nqh, nkvh, n_ctx, q8, s, rope3, rdelta);
  });
}

// qn, qg, kcache, vcache, o, xq, xd, pos0, T, kq_scale, nqh, nkvh, n_ctx, q8
PyObject* attn_decode(PyObject* self, PyObject* const* a, Py_ssize_t n) {
  return guarded(self, n, 14, [&](const State* st) -> PyObject* {
    PTR(0, F32, false, qn); PTR(1, F32, false, qg); PTR(2, ANY, false, kc); PTR(3, ANY, false, vc); PTR(4, F32, true, o);
    PTR(5, I8, true, xq); PTR(6, F32, true, xd); PTR(7, I32, false, pos0);
    NUM(8, T); FLT(9, scale); NUM(10, nqh); NUM(11, nkvh); NUM(12, n_ctx); FLAG(13, q8);
    CALL(DECODE, q27b_attn_decode, qn, qg, kc, vc, o, xq, xd, pos0, T, scale, nqh, nkvh, n_ctx, q8, s);
  });
}

// qg, k, v, q_norm, k_norm, qn, kpool, vpool, page_table, seq_len, B, T, eps, theta_scale, nqh, nkvh, n_pages, max_pages, rope3, rdelta
PyObject* attn_prep_paged(PyObject* self, PyObject* const* a, Py_ssize_t n) {
  return guarded(self, n, 20, [&](const State* st) -> PyObject* {
    PTR(0, F32, true, qg); PTR(1, F32, false, k); PTR(2, F32, false, v); PTR(3, F32, true, qw); PTR(4, F32, true, kw);
    PTR(5, F32, true, qn); PTR(6, ANY, false, kp); PTR(7, ANY, false, vp); PTR(8, I32, false, table); PTR(9, I32, false, lens);
    NUM(10, B); NUM(11, T); FLT(12, eps); FLT(13, theta); NUM(14, nqh); NUM(15, nkvh); NUM(16, n_pages); NUM(17, max_pages);
    PTR(18, I32, true, rope3); PTR(19, I32, true, rdelta);
    CALL(PREP_PAGED, q27b_attn_prep_paged, qg, k, v, qw, kw, qn, kp, vp, table, lens, B, T, eps, theta, nqh, nkvh, n_pages, max_pages, s, rope3, rdelta);
  });
}

// qn, qg, kpool, vpool, page_table, seq_len, o, B, T, kq_scale, nqh, nkvh, n_pages, max_pages, max_seq_len
PyObject* attn_decode_paged(PyObject* self, PyObject* const* a, Py_ssize_t n) {
  return guarded(self, n, 15, [&](const State* st) -> PyObject* {
    PTR(0, F32, false, qn); PTR(1, F32, false, qg); PTR(2, ANY, false, kp); PTR(3, ANY, false, vp); PTR(4, I32, false, table);
    PTR(5, I32, false, lens); PTR(6, F32, false, o);
    NUM(7, B); NUM(8, T); FLT(9, scale); NUM(10, nqh); NUM(11, nkvh); NUM(12, n_pages); NUM(13, max_pages); NUM(14, max_len);
    CALL(DECODE_PAGED, q27b_attn_decode_paged, qn, qg, kp, vp, table, lens, o, B, T, scale, nqh, nkvh, n_pages, max_pages, max_len, s);
  });
}

// qn, qg, kcache, vcache, o, pos0, M, kq_scale, nqh, nkvh, n_ctx, q8, depth_hint
PyObject* attn_prefill(PyObject* self, PyObject* const* a, Py_ssize_t n) {
  return guarded(self, n, 13, [&](const State* st) -> PyObject* {
    PTR(0, F32, false, qn); PTR(1, F32, false, qg); PTR(2, ANY, false, kc); PTR(3, ANY, false, vc); PTR(4, F32, false, o);
    PTR(5, I32, false, pos0);
    NUM(6, M); FLT(7, scale); NUM(8, nqh); NUM(9, nkvh); NUM(10, n_ctx); FLAG(11, q8); NUM(12, depth);
    CALL(PREFILL, q27b_attn_prefill, qn, qg, kc, vc, o, pos0, M, scale, nqh, nkvh, n_ctx, q8, s, depth);
  });
}

// Sizes of the arguments that several calls share; a shape that the library refuses gives numbers that refuse nothing.
int64_t count(int64_t a, int64_t b = 1, int64_t c = 1, int64_t d = 1) {
  int64_t n = 1;
  for (int64_t x : {a, b, c, d})
    if (x < 1 || __builtin_mul_overflow(n, x, &n)) return 0;
  return n;
}
constexpr int DIM = Q27B_HEAD_DIM;
int64_t cache_bytes(int nkvh, int n_ctx, int q8) { return count(nkvh, n_ctx, q8 ? DIM + 16 : 2 * DIM); }
int64_t pool_bytes(int nkvh, int n_pages) { return count(n_pages, nkvh, Q27B_PAGE, DIM + 16); }

// qn, qg, kcache, vcache, o, xq, xd, pos0, mask, T, kq_scale, nqh, nkvh, n_ctx, q8
PyObject* attn_decode_tree(PyObject* self, PyObject* const* a, Py_ssize_t n) {
  return guarded(self, n, 15, [&](const State* st) -> PyObject* {
    NUM(9, T); FLT(10, scale); NUM(11, nqh); NUM(12, nkvh); NUM(13, n_ctx); FLAG(14, q8);
    const int64_t rows = count(T, nqh);
    SIZED(0, F32, false, qn, rows * DIM); SIZED(1, F32, false, qg, rows * 2 * DIM); SIZED(2, ANY, false, kc, cache_bytes(nkvh, n_ctx, q8));
    SIZED(3, ANY, false, vc, cache_bytes(nkvh, n_ctx, q8)); SIZED(4, F16, true, o, rows * DIM); SIZED(5, I8, true, xq, rows * DIM);
    SIZED(6, F32, true, xd, rows * DIM / 32); SIZED(7, I32, false, pos0, 1); SIZED(8, I64, false, mask, count(T));
    CALL(TREE, q27b_attn_decode_tree, qn, qg, kc, vc, o, xq, xd, pos0, mask, T, scale, nqh, nkvh, n_ctx, q8, s);
  });
}

// qn, qg, kpool, vpool, page_table, seq_len, mask, o, xq, xd, B, T, kq_scale, nqh, nkvh, n_pages, max_pages, max_seq_len
PyObject* attn_decode_tree_paged(PyObject* self, PyObject* const* a, Py_ssize_t n) {
  return guarded(self, n, 18, [&](const State* st) -> PyObject* {
    NUM(10, B); NUM(11, T); FLT(12, scale); NUM(13, nqh); NUM(14, nkvh); NUM(15, n_pages); NUM(16, max_pages); NUM(17, max_len);
    const int64_t rows = count(B, T, nqh);
    SIZED(0, F32, false, qn, rows * DIM); SIZED(1, F32, false, qg, rows * 2 * DIM); SIZED(2, ANY, false, kp, pool_bytes(nkvh, n_pages));
    SIZED(3, ANY, false, vp, pool_bytes(nkvh, n_pages)); SIZED(4, I32, false, table, count(B, max_pages)); SIZED(5, I32, false, lens, count(B));
    SIZED(6, I64, false, mask, count(B, T)); SIZED(7, F16, true, o, rows * DIM); SIZED(8, I8, true, xq, rows * DIM);
    SIZED(9, F32, true, xd, rows * DIM / 32);
    CALL(TREE_PAGED, q27b_attn_decode_tree_paged, qn, qg, kp, vp, table, lens, mask, o, xq, xd, B, T, scale, nqh, nkvh, n_pages,
         max_pages, max_len, s);
  });
}

// kcache, vcache, pos0, path, count, T, nkvh, n_ctx, q8
PyObject* kv_commit(PyObject* self, PyObject* const* a, Py_ssize_t n) {
  return guarded(self, n, 9, [&](const State* st) -> PyObject* {
    NUM(5, T); NUM(6, nkvh); NUM(7, n_ctx); FLAG(8, q8);
    SIZED(0, ANY, false, kc, cache_bytes(nkvh, n_ctx, q8)); SIZED(1, ANY, false, vc, cache_bytes(nkvh, n_ctx, q8)); SIZED(2, I32, false, pos0, 1); SIZED(3, I32, false, path, count(T));
    SIZED(4, I32, false, cnt, 1);
    CALL(COMMIT, q27b_kv_commit, kc, vc, pos0, path, cnt, T, nkvh, n_ctx, q8, s);
  });
}

// kpool, vpool, page_table, seq_len, path, count, B, T, nkvh, n_pages, max_pages
PyObject* kv_commit_paged(PyObject* self, PyObject* const* a, Py_ssize_t n) {
  return guarded(self, n, 11, [&](const State* st) -> PyObject* {
    NUM(6, B); NUM(7, T); NUM(8, nkvh); NUM(9, n_pages); NUM(10, max_pages);
    SIZED(0, ANY, false, kp, pool_bytes(nkvh, n_pages)); SIZED(1, ANY, false, vp, pool_bytes(nkvh, n_pages)); SIZED(2, I32, false, table, count(B, max_pages));
    SIZED(3, I32, false, lens, count(B)); SIZED(4, I32, false, path, count(B, T)); SIZED(5, I32, false, cnt, count(B));
    CALL(COMMIT_PAGED, q27b_kv_commit_paged, kp, vp, table, lens, path, cnt, B, T, nkvh, n_pages, max_pages, s);
  });
}

// kcache, bounds, pos0, T, nkvh, n_ctx, q8
PyObject* kv_bounds(PyObject* self, PyObject* const* a, Py_ssize_t n) {
  return guarded(self, n, 7, [&](const State* st) -> PyObject* {
    NUM(3, T); NUM(4, nkvh); NUM(5, n_ctx); FLAG(6, q8);
    SIZED(0, ANY, false, kc, cache_bytes(nkvh, n_ctx, q8)); SIZED(1, F16, false, bounds, count(nkvh, ((int64_t)n_ctx + 63) / 64, 2 * DIM));
    SIZED(2, I32, false, pos0, 1);
    CALL(BOUNDS, q27b_kv_bounds, kc, bounds, pos0, T, nkvh, n_ctx, q8, s);
  });
}

// kpool, bounds, page_table, seq_len, B, T, nkvh, n_pages, max_pages
PyObject* kv_bounds_paged(PyObject* self, PyObject* const* a, Py_ssize_t n) {
  return guarded(self, n, 9, [&](const State* st) -> PyObject* {
    NUM(4, B); NUM(5, T); NUM(6, nkvh); NUM(7, n_pages); NUM(8, max_pages);
    SIZED(0, ANY, false, kp, pool_bytes(nkvh, n_pages)); SIZED(1, F16, false, bounds, count(n_pages, nkvh, 4, 2 * DIM));
    SIZED(2, I32, false, table, count(B, max_pages)); SIZED(3, I32, false, lens, count(B));
    CALL(BOUNDS_PAGED, q27b_kv_bounds_paged, kp, bounds, table, lens, B, T, nkvh, n_pages, max_pages, s);
  });
}

// qn, bounds, sel, pos0, T, k, n_sink, n_recent, nqh, nkvh, n_ctx
PyObject* select_blocks(PyObject* self, PyObject* const* a, Py_ssize_t n) {
  return guarded(self, n, 11, [&](const State* st) -> PyObject* {
    NUM(4, T); NUM(5, k); NUM(6, n_sink); NUM(7, n_recent); NUM(8, nqh); NUM(9, nkvh); NUM(10, n_ctx);
    SIZED(0, F32, false, qn, count(T, nqh, DIM)); SIZED(1, F16, false, bounds, count(nkvh, ((int64_t)n_ctx + 63) / 64, 2 * DIM));
    SIZED(2, I32, false, sel, count(T, nkvh, k)); SIZED(3, I32, false, pos0, 1);
    CALL(SELECT, q27b_select_blocks, qn, bounds, sel, pos0, T, k, n_sink, n_recent, nqh, nkvh, n_ctx, s);
  });
}

// qn, bounds, sel, page_table, seq_len, B, T, k, n_sink, n_recent, nqh, nkvh, n_pages, max_pages, max_seq_len
PyObject* select_blocks_paged(PyObject* self, PyObject* const* a, Py_ssize_t n) {
  return guarded(self, n, 15, [&](const State* st) -> PyObject* {
    NUM(5, B); NUM(6, T); NUM(7, k); NUM(8, n_sink); NUM(9, n_recent); NUM(10, nqh); NUM(11, nkvh); NUM(12, n_pages);
    NUM(13, max_pages); NUM(14, max_len);
    SIZED(0, F32, false, qn, count(B, T, nqh, DIM)); SIZED(1, F16, false, bounds, count(n_pages, nkvh, 4, 2 * DIM));
    SIZED(2, I32, false, sel, count(B, T, nkvh, k)); SIZED(3, I32, false, table, count(B, max_pages));
    SIZED(4, I32, false, lens, count(B));
    CALL(SELECT_PAGED, q27b_select_blocks_paged, qn, bounds, sel, table, lens, B, T, k, n_sink, n_recent, nqh, nkvh, n_pages,
         max_pages, max_len, s);
  });
}

// qn, qg, kcache, vcache, o, xq, xd, pos0, sel, T, k, kq_scale, nqh, nkvh, n_ctx, q8
PyObject* attn_decode_blocks(PyObject* self, PyObject* const* a, Py_ssize_t n) {
  return guarded(self, n, 16, [&](const State* st) -> PyObject* {
    NUM(9, T); NUM(10, k); FLT(11, scale); NUM(12, nqh); NUM(13, nkvh); NUM(14, n_ctx); FLAG(15, q8);
    const int64_t rows = count(T, nqh);
    SIZED(0, F32, false, qn, rows * DIM); SIZED(1, F32, false, qg, rows * 2 * DIM); SIZED(2, ANY, false, kc, cache_bytes(nkvh, n_ctx, q8));
    SIZED(3, ANY, false, vc, cache_bytes(nkvh, n_ctx, q8)); SIZED(4, F16, true, o, rows * DIM); SIZED(5, I8, true, xq, rows * DIM);
    SIZED(6, F32, true, xd, rows * DIM / 32); SIZED(7, I32, false, pos0, 1); SIZED(8, I32, false, sel, count(T, nkvh, k));
    CALL(BLOCKS, q27b_attn_decode_blocks, qn, qg, kc, vc, o, xq, xd, pos0, sel, T, k, scale, nqh, nkvh, n_ctx, q8, s);
  });
}

// qn, qg, kpool, vpool, page_table, seq_len, sel, o, xq, xd, B, T, k, kq_scale, nqh, nkvh, n_pages, max_pages
PyObject* attn_decode_blocks_paged(PyObject* self, PyObject* const* a, Py_ssize_t n) {
  return guarded(self, n, 18, [&](const State* st) -> PyObject* {
    NUM(10, B); NUM(11, T); NUM(12, k); FLT(13, scale); NUM(14, nqh); NUM(15, nkvh); NUM(16, n_pages); NUM(17, max_pages);
    const int64_t rows = count(B, T, nqh);
    SIZED(0, F32, false, qn, rows * DIM); SIZED(1, F32, false, qg, rows * 2 * DIM); SIZED(2, ANY, false, kp, pool_bytes(nkvh, n_pages));
    SIZED(3, ANY, false, vp, pool_bytes(nkvh, n_pages)); SIZED(4, I32, false, table, count(B, max_pages)); SIZED(5, I32, false, lens, count(B));
    SIZED(6, I32, false, sel, count(B, T, nkvh, k)); SIZED(7, F16, true, o, rows * DIM); SIZED(8, I8, true, xq, rows * DIM);
    SIZED(9, F32, true, xd, rows * DIM / 32);
    CALL(BLOCKS_PAGED, q27b_attn_decode_blocks_paged, qn, qg, kp, vp, table, lens, sel, o, xq, xd, B, T, k, scale, nqh, nkvh,
         n_pages, max_pages, s);
  });
}

// addresses (tuple of N_FN ints), _ptr, _check, torch.float32, torch.int32, torch.int8, torch.float16, torch.int64
PyObject* bind(PyObject* self, PyObject* args) {
  PyObject *fns, *p, *c, *f32, *i32, *i8, *f16, *i64;
  if (!PyArg_ParseTuple(args, "O!OOOOOOO", &PyTuple_Type, &fns, &p, &c, &f32, &i32, &i8, &f16, &i64)) return nullptr;
  if (PyTuple_GET_SIZE(fns) != N_FN) return PyErr_Format(PyExc_ValueError, "expected %d addresses", (int)N_FN);
  State* st = (State*)PyModule_GetState(self);
  for (int i = 0; i < N_FN; i++) st->fn[i] = PyLong_AsVoidPtr(PyTuple_GET_ITEM(fns, i));
  if (PyErr_Occurred()) return nullptr;
  Py_XSETREF(st->ptr, Py_NewRef(p)); Py_XSETREF(st->check, Py_NewRef(c));
  Py_XSETREF(st->f32, Py_NewRef(f32)); Py_XSETREF(st->i32, Py_NewRef(i32)); Py_XSETREF(st->i8, Py_NewRef(i8));
  Py_XSETREF(st->f16, Py_NewRef(f16)); Py_XSETREF(st->i64, Py_NewRef(i64));
  Py_RETURN_NONE;
}

#define FAST(name) {#name, (PyCFunction)(void (*)(void))name, METH_FASTCALL, nullptr}
PyMethodDef g_methods[] = {{"bind", bind, METH_VARARGS, nullptr}, FAST(attn_prep), FAST(attn_decode), FAST(attn_prep_paged),
                           FAST(attn_decode_paged), FAST(attn_prefill), FAST(attn_decode_tree), FAST(attn_decode_tree_paged),
                           FAST(kv_commit), FAST(kv_commit_paged), FAST(kv_bounds), FAST(kv_bounds_paged), FAST(select_blocks),
                           FAST(select_blocks_paged), FAST(attn_decode_blocks), FAST(attn_decode_blocks_paged), {nullptr, nullptr, 0, nullptr}};
// The objects of the state belong to the package that holds this module: a cycle for the collector.
int traverse(PyObject* self, visitproc visit, void* arg) {
  State* st = (State*)PyModule_GetState(self);
  if (!st) return 0;
  Py_VISIT(st->ptr); Py_VISIT(st->check); Py_VISIT(st->f32); Py_VISIT(st->i32); Py_VISIT(st->i8); Py_VISIT(st->f16); Py_VISIT(st->i64);
  return 0;
}
int clear(PyObject* self) {
  State* st = (State*)PyModule_GetState(self);
  if (!st) return 0;
  Py_CLEAR(st->ptr); Py_CLEAR(st->check); Py_CLEAR(st->f32); Py_CLEAR(st->i32); Py_CLEAR(st->i8); Py_CLEAR(st->f16); Py_CLEAR(st->i64);
  return 0;
}
void release(void* self) { clear((PyObject*)self); }

PyModuleDef_Slot g_slots[] = {{0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "q27b_binding", nullptr, sizeof(State), g_methods, g_slots, traverse, clear, release};

}  // namespace

PyMODINIT_FUNC PyInit_q27b_binding(void) { return PyModuleDef_Init(&g_module); }
