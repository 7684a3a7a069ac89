// Short way from torch tensors to the paged operators' C entries.
//
// A serving step makes these calls for every layer, and marshalling some
// twenty arguments through ctypes after checking a dozen tensors one attribute
// at a time took 6 to 10 us a call, two to four times the launch.  Here the
// checks and the call are one function: it returns the entry's status, or -1
// if an argument is not what the fast way takes (a tensor of another device
// than the current one, of another type or size, not contiguous, not a tensor
// at all).  The Python wrapper then finds out which and raises, or makes the
// call through ctypes.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>

#include "../../include/sc_b200.h"

namespace {

// The arguments of one call: tensors are taken only if they are contiguous, on
// the current device and of the type asked for.
struct Args {
  PyObject* const* a;
  int dev;
  bool ok = true;

  const at::Tensor* tensor(int i) {
    if (!ok || !THPVariable_Check(a[i])) return fail();
    const at::Tensor& t = THPVariable_Unpack(a[i]);
    if (!t.is_cuda() || t.get_device() != dev || !t.is_contiguous()) return fail();
    return &t;
  }
  int32_t* ints(int i, int64_t n) {  // n < 0: any number
    const at::Tensor* t = tensor(i);
    if (!t || t->scalar_type() != at::kInt || (n >= 0 && t->numel() != n)) {
      ok = false;
      return nullptr;
    }
    return static_cast<int32_t*>(t->data_ptr());
  }
  int32_t* ints_or_none(int i, int64_t n) { return a[i] == Py_None ? nullptr : ints(i, n); }
  long long number(int i) {
    const long long v = PyLong_Check(a[i]) ? PyLong_AsLongLong(a[i]) : (ok = false, 0);
    if (PyErr_Occurred()) {
      PyErr_Clear();
      ok = false;
    }
    if (v < INT32_MIN || v > INT32_MAX) ok = false;
    return v;
  }
  int64_t size(int i, int d) { return THPVariable_Unpack(a[i]).size(d); }
  int64_t numel(int i) { return THPVariable_Unpack(a[i]).numel(); }
  // [B, columns]
  int32_t* table(int i, int64_t rows) {
    int32_t* p = ints(i, -1);
    if (p && (THPVariable_Unpack(a[i]).dim() != 2 || size(i, 0) != rows)) ok = false;
    return p;
  }

 private:
  const at::Tensor* fail() {
    ok = false;
    return nullptr;
  }
};

bool float_code(const at::Tensor* t, int* code) {
  if (!t) return false;
  *code = t->scalar_type() == at::kHalf ? SC_F16 : SC_F32;
  return t->scalar_type() == at::kHalf || t->scalar_type() == at::kFloat;
}

template <typename F>
PyObject* guarded(PyObject* const* args, Py_ssize_t n, Py_ssize_t want, F f) {
  if (n != want || !THPVariable_Check(args[0])) return PyLong_FromLong(-1);
  int st = -1;
  try {
    const at::Tensor& t = THPVariable_Unpack(args[0]);
    if (t.is_cuda() && t.get_device() == c10::cuda::current_device()) {
      Args a{args, (int)t.get_device()};
      st = f(a, c10::cuda::getCurrentCUDAStream(t.get_device()).stream());
    }
  } catch (...) {
    st = -1;
  }
  return PyLong_FromLong(st);
}

// The entry, without the interpreter's lock.
template <typename F>
int call(F f) {
  int st;
  Py_BEGIN_ALLOW_THREADS;
  st = f();
  Py_END_ALLOW_THREADS;
  return st;
}

// lens, new_lens, block_table, free_pages, free_count, page_size, rows, prefix_len | None, kv_lens, q_start, slots, positions,
// free_count_out, status
PyObject* paged_reserve(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(args, n, 14, [](Args& a, cudaStream_t s) {
    const int32_t* lens = a.ints(0, -1);
    if (!a.ok) return -1;
    const int64_t B = a.numel(0), rows = a.number(6);
    const int page = (int)a.number(5);
    const int32_t* add = a.ints(1, B);
    int32_t *table = a.table(2, B), *free = a.ints(3, -1), *count = a.ints(4, 1), *prefix = a.ints_or_none(7, 1), *kv = a.ints(8, B),
            *start = a.ints(9, B + 1), *slots = a.ints(10, -1), *pos = a.ints(11, -1), *left = a.ints(12, 1), *status = a.ints(13, 1);
    if (!a.ok || a.numel(10) < rows || a.numel(11) < rows) return -1;
    const int64_t blocks = a.size(2, 1), nf = a.numel(3);
    if (B > INT32_MAX || blocks > INT32_MAX || nf > INT32_MAX) return -1;
    return call([&] {
      return sc_paged_reserve(lens, add, (int)B, prefix, table, (int)blocks, free, (int)nf, count, page, (int)rows, kv, start, slots, pos,
                              left, status, s);
    });
  });
}

// lens, keep, block_table, free_pages, free_count, page_size, lens_out, free_count_out, status
PyObject* paged_truncate(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(args, n, 9, [](Args& a, cudaStream_t s) {
    const int32_t* lens = a.ints(0, -1);
    if (!a.ok) return -1;
    const int64_t B = a.numel(0);
    const int page = (int)a.number(5);
    const int32_t* keep = a.ints(1, B);
    int32_t *table = a.table(2, B), *free = a.ints(3, -1), *count = a.ints(4, 1), *out = a.ints(6, B), *left = a.ints(7, 1),
            *status = a.ints(8, 1);
    if (!a.ok) return -1;
    const int64_t blocks = a.size(2, 1), nf = a.numel(3);
    if (B > INT32_MAX || blocks > INT32_MAX || nf > INT32_MAX) return -1;
    return call([&] { return sc_paged_truncate(lens, keep, (int)B, table, (int)blocks, free, (int)nf, count, page, out, left, status, s); });
  });
}

// qkv, q_start, slots, positions, cos_tab, sin_tab, q_out, k_pages, v_pages
PyObject* paged_rope_append(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(args, n, 9, [](Args& a, cudaStream_t s) {
    const at::Tensor *x = a.tensor(0), *cos = a.tensor(4), *sin = a.tensor(5), *q = a.tensor(6), *k = a.tensor(7), *v = a.tensor(8);
    const int32_t *start = a.ints(1, -1), *slots = a.ints(2, -1), *pos = a.ints(3, -1);
    int xc, kc;
    if (!a.ok || !float_code(x, &xc) || !float_code(k, &kc) || k->dim() != 4 || k->sizes() != v->sizes() || x->dim() != 2) return -1;
    if (v->scalar_type() != k->scalar_type() || q->scalar_type() != k->scalar_type()) return -1;
    const int64_t pages = k->size(0), Hkv = k->size(1), page = k->size(2), hd = k->size(3), T = x->size(0), width = x->size(1);
    if (T < 1 || hd < 1 || width % hd || width / hd <= 2 * Hkv) return -1;
    const int64_t Hq = width / hd - 2 * Hkv;
    if (q->numel() != T * Hq * hd || a.numel(1) < 1 || a.numel(2) < T || a.numel(3) < T) return -1;
    if (cos->scalar_type() != at::kFloat || sin->scalar_type() != at::kFloat || cos->dim() != 2 || cos->size(1) * 2 != hd ||
        cos->sizes() != sin->sizes())
      return -1;
    if (T > INT32_MAX || pages > INT32_MAX || page > INT32_MAX || Hq > INT32_MAX || cos->size(0) > INT32_MAX) return -1;
    return call([&] {
      return sc_paged_rope_append(x->data_ptr(), xc, (int)T, start + a.numel(1) - 1, slots, pos, static_cast<const float*>(cos->data_ptr()),
                                  static_cast<const float*>(sin->data_ptr()), (int)cos->size(0), (int)Hq, (int)Hkv, (int)hd, q->data_ptr(),
                                  k->data_ptr(), v->data_ptr(), kc, (int)pages, (int)page, s);
    });
  });
}

// q, k_pages, v_pages, q_start, kv_lens, block_table, prefix_table | None, prefix_len | None, out, scale | None, workspace | None
PyObject* prefix_attn(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(args, n, 11, [](Args& a, cudaStream_t s) {
    const at::Tensor *q = a.tensor(0), *k = a.tensor(1), *v = a.tensor(2), *out = a.tensor(8);
    const int32_t *start = a.ints(3, -1), *lens = a.ints(4, -1);
    int code;
    if (!a.ok || !float_code(k, &code) || k->dim() != 4 || k->sizes() != v->sizes() || q->dim() < 1) return -1;
    if (v->scalar_type() != k->scalar_type() || q->scalar_type() != k->scalar_type() || out->scalar_type() != k->scalar_type()) return -1;
    const int64_t pages = k->size(0), Hkv = k->size(1), page = k->size(2), hd = k->size(3), T = q->size(0), B = a.numel(4), nq = q->numel();
    if (T < 1 || B < 1 || hd < 1 || out->numel() != nq || nq % (T * hd) || a.numel(3) != B + 1) return -1;
    const int64_t Hq = nq / (T * hd);
    const int32_t* table = a.table(5, B);
    if ((a.a[6] == Py_None) != (a.a[7] == Py_None)) return -1;
    const int32_t *ptab = a.ints_or_none(6, -1), *plen = a.ints_or_none(7, 1);
    if (!a.ok) return -1;
    const int64_t blocks = a.size(5, 1), pblocks = ptab ? a.numel(6) : 0;
    if (T > INT32_MAX || B > INT32_MAX || pages > INT32_MAX || page > INT32_MAX || Hq > INT32_MAX || blocks > INT32_MAX || pblocks > INT32_MAX)
      return -1;
    double scale = 1.0 / std::sqrt((double)hd);
    if (a.a[9] != Py_None) {
      if (!PyFloat_Check(a.a[9])) return -1;
      scale = PyFloat_AS_DOUBLE(a.a[9]);
    }
    at::Tensor scratch;
    void* ws = nullptr;
    size_t bytes = 0;
    if (a.a[10] != Py_None) {
      const at::Tensor* w = a.tensor(10);
      if (!w || w->scalar_type() != at::kByte) return -1;
      ws = w->data_ptr();
      bytes = (size_t)w->numel();
    } else {
      bytes = sc_prefix_attn_workspace_bytes((int)T, (int)B, (int)Hq, (int)Hkv, (int)hd, (int)blocks, (int)pblocks, (int)page, code);
      if (bytes) {
        scratch = at::empty({(int64_t)bytes}, q->options().dtype(at::kByte));
        ws = scratch.data_ptr();
      }
    }
    return call([&] {
      return sc_prefix_attn(q->data_ptr(), k->data_ptr(), v->data_ptr(), code, (int)T, start, lens, table, (int)B, (int)blocks, ptab, plen,
                            (int)pblocks, (int)Hq, (int)Hkv, (int)hd, (int)pages, (int)page, (float)scale, out->data_ptr(), ws, bytes, s);
    });
  });
}

// A pool in 8 or 4 bits (arguments i .. i + 4: data, head_dim, page_size, bits, group): uint8 [n_pages, Hkv, bytes of a page].
struct QuantPool {
  void* data = nullptr;
  int64_t pages = 0, Hkv = 0;
  int hd = 0, page = 0, bits = 0, group = 0;
};
bool quant_pool(Args& a, int i, QuantPool* p) {
  const at::Tensor* t = a.tensor(i);
  p->hd = (int)a.number(i + 1);
  p->page = (int)a.number(i + 2);
  p->bits = (int)a.number(i + 3);
  p->group = (int)a.number(i + 4);
  if (!a.ok || t->scalar_type() != at::kByte || t->dim() != 3) return a.ok = false;
  const size_t n = sc_quant_page_bytes(p->page, p->hd, p->bits, p->group);
  if (!n || (size_t)t->size(2) != n || t->size(0) > INT32_MAX || t->size(1) > INT32_MAX) return a.ok = false;
  p->data = t->data_ptr();
  p->pages = t->size(0);
  p->Hkv = t->size(1);
  return true;
}

// qkv, q_start, slots, positions, cos_tab, sin_tab, q_out, pool (5)
PyObject* paged_rope_append_q(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(args, n, 12, [](Args& a, cudaStream_t s) {
    const at::Tensor *x = a.tensor(0), *cos = a.tensor(4), *sin = a.tensor(5), *q = a.tensor(6);
    const int32_t *start = a.ints(1, -1), *slots = a.ints(2, -1), *pos = a.ints(3, -1);
    QuantPool k;
    int xc;
    if (!quant_pool(a, 7, &k) || !float_code(x, &xc) || x->dim() != 2 || q->scalar_type() != at::kHalf) return -1;
    const int64_t T = x->size(0), width = x->size(1);
    if (T < 1 || width % k.hd || width / k.hd <= 2 * k.Hkv) return -1;
    const int64_t Hq = width / k.hd - 2 * k.Hkv;
    if (q->numel() != T * Hq * k.hd || a.numel(1) < 1 || a.numel(2) < T || a.numel(3) < T) return -1;
    if (cos->scalar_type() != at::kFloat || sin->scalar_type() != at::kFloat || cos->dim() != 2 || cos->size(1) * 2 != k.hd ||
        cos->sizes() != sin->sizes())
      return -1;
    if (T > INT32_MAX || Hq > INT32_MAX || cos->size(0) > INT32_MAX) return -1;
    return call([&] {
      return sc_paged_rope_append_q(x->data_ptr(), xc, (int)T, start + a.numel(1) - 1, slots, pos, static_cast<const float*>(cos->data_ptr()),
                                    static_cast<const float*>(sin->data_ptr()), (int)cos->size(0), (int)Hq, (int)k.Hkv, k.hd, q->data_ptr(),
                                    k.data, k.bits, k.group, (int)k.pages, k.page, s);
    });
  });
}

// slots, pool (5), q_start | None, k_out, v_out
PyObject* paged_read_q(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(args, n, 9, [](Args& a, cudaStream_t s) {
    const int32_t *slots = a.ints(0, -1), *start = a.ints_or_none(6, -1);
    const at::Tensor *k_out = a.tensor(7), *v_out = a.tensor(8);
    QuantPool k;
    int code;
    if (!quant_pool(a, 1, &k) || !float_code(k_out, &code) || v_out->scalar_type() != k_out->scalar_type()) return -1;
    const int64_t T = a.numel(0), m = start ? a.numel(6) : 1;
    if (T < 1 || T > INT32_MAX || m < 1 || k_out->numel() != T * k.Hkv * k.hd || v_out->numel() != k_out->numel()) return -1;
    return call([&] {
      return sc_paged_read_q(k.data, k.bits, k.group, (int)k.pages, k.page, (int)k.Hkv, k.hd, slots, (int)T, start ? start + m - 1 : nullptr,
                             k_out->data_ptr(), v_out->data_ptr(), code, s);
    });
  });
}

// q, pool (5), q_start, kv_lens, block_table, prefix_table | None, prefix_len | None, out, scale | None, workspace | None
PyObject* prefix_attn_q(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(args, n, 14, [](Args& a, cudaStream_t s) {
    const at::Tensor *q = a.tensor(0), *out = a.tensor(11);
    const int32_t *start = a.ints(6, -1), *lens = a.ints(7, -1);
    QuantPool k;
    if (!quant_pool(a, 1, &k) || q->scalar_type() != at::kHalf || out->scalar_type() != at::kHalf || q->dim() < 1) return -1;
    const int64_t T = q->size(0), B = a.numel(7), nq = q->numel();
    if (T < 1 || B < 1 || out->numel() != nq || nq % (T * k.hd) || a.numel(6) != B + 1) return -1;
    const int64_t Hq = nq / (T * k.hd);
    const int32_t* table = a.table(8, B);
    if ((a.a[9] == Py_None) != (a.a[10] == Py_None)) return -1;
    const int32_t *ptab = a.ints_or_none(9, -1), *plen = a.ints_or_none(10, 1);
    if (!a.ok) return -1;
    const int64_t blocks = a.size(8, 1), pblocks = ptab ? a.numel(9) : 0;
    if (T > INT32_MAX || B > INT32_MAX || Hq > INT32_MAX || blocks > INT32_MAX || pblocks > INT32_MAX) return -1;
    double scale = 1.0 / std::sqrt((double)k.hd);
    if (a.a[12] != Py_None) {
      if (!PyFloat_Check(a.a[12])) return -1;
      scale = PyFloat_AS_DOUBLE(a.a[12]);
    }
    at::Tensor scratch;
    void* ws = nullptr;
    size_t bytes = 0;
    if (a.a[13] != Py_None) {
      const at::Tensor* w = a.tensor(13);
      if (!w || w->scalar_type() != at::kByte) return -1;
      ws = w->data_ptr();
      bytes = (size_t)w->numel();
    } else {
      bytes = sc_prefix_attn_q_workspace_bytes((int)T, (int)B, (int)Hq, (int)k.Hkv, k.hd, k.bits, k.group, (int)blocks, (int)pblocks, k.page);
      if (bytes) {
        scratch = at::empty({(int64_t)bytes}, q->options().dtype(at::kByte));
        ws = scratch.data_ptr();
      }
    }
    return call([&] {
      return sc_prefix_attn_q(q->data_ptr(), k.data, k.bits, k.group, (int)T, start, lens, table, (int)B, (int)blocks, ptab, plen, (int)pblocks,
                              (int)Hq, (int)k.Hkv, k.hd, (int)k.pages, k.page, (float)scale, out->data_ptr(), ws, bytes, s);
    });
  });
}

PyMethodDef methods[] = {
    {"paged_reserve", (PyCFunction)(void (*)(void))paged_reserve, METH_FASTCALL, nullptr},
    {"paged_truncate", (PyCFunction)(void (*)(void))paged_truncate, METH_FASTCALL, nullptr},
    {"paged_rope_append", (PyCFunction)(void (*)(void))paged_rope_append, METH_FASTCALL, nullptr},
    {"prefix_attn", (PyCFunction)(void (*)(void))prefix_attn, METH_FASTCALL, nullptr},
    {"paged_rope_append_q", (PyCFunction)(void (*)(void))paged_rope_append_q, METH_FASTCALL, nullptr},
    {"paged_read_q", (PyCFunction)(void (*)(void))paged_read_q, METH_FASTCALL, nullptr},
    {"prefix_attn_q", (PyCFunction)(void (*)(void))prefix_attn_q, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_native", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__native(void) { return PyModule_Create(&module); }
