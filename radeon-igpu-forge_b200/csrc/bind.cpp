// The generation operators' way from Python: one call that reads the tensors,
// checks that they fit, makes what is returned and launches. A decoding step
// makes these calls once a layer for a few microseconds of GPU work, and the
// same from Python, attribute by attribute, was what bounded small calls (host
// time of one token's attention 14.1 us, now 6.1; of a commit 11.4, now 4.5; of
// a chain's verification 12.4, now 6.6).
//
// A function returns its result, None when an argument does not fit (the caller
// then looks for the reason and raises), or the library's error code. The
// library itself stays free of torch: its functions come in as addresses.
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/object_ptr.h>

#include <ATen/core/grad_mode.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/empty_like.h>
#include <c10/cuda/CUDAStream.h>

#include <climits>
#include <cmath>
#include <initializer_list>

#include "fxb200.h"

namespace {

struct {
  decltype(&fxb_tree_attn) tree_attn;
  decltype(&fxb_tree_attn_workspace) tree_attn_workspace, tree_attn_zeroed;
  decltype(&fxb_verify_tree) verify_tree;
  decltype(&fxb_kv_commit) kv_commit;
  decltype(&fxb_kv_fork) kv_fork;
  decltype(&fxb_kv_fork_workspace) kv_fork_workspace;
} lib;
PyObject* workspace_of;  // fxb200.ops.stream_workspace
PyObject* tree_kind;     // the kind of workspace of tree_attention

constexpr int kMaxNodes = 64;

bool ints(std::initializer_list<int64_t> sizes) {  // the C structs take 32 bits
  for (int64_t x : sizes)
    if (x > INT_MAX) return false;
  return true;
}

const at::Tensor* tensor(PyObject* x) { return THPVariable_Check(x) ? &THPVariable_Unpack(x) : nullptr; }

// on the GPU of this index: a kernel runs on one, and would take another's address for its own
bool on(const at::Tensor& t, int64_t device) { return t.is_cuda() && t.get_device() == device; }

// a contiguous int32 tensor of this shape on this GPU
int32_t* i32(const at::Tensor* t, at::IntArrayRef shape, int64_t device) {
  if (!t || t->scalar_type() != at::kInt || !on(*t, device) || t->sizes() != shape || !t->is_contiguous()) return nullptr;
  return static_cast<int32_t*>(t->data_ptr());
}

struct Table {
  int32_t* p;
  int64_t rows, entries, stride;
};
bool table(const at::Tensor* t, Table* out, int64_t device) {
  if (!t || t->scalar_type() != at::kInt || !on(*t, device) || t->dim() != 2 || t->stride(1) != 1) return false;
  *out = {static_cast<int32_t*>(t->data_ptr()), t->size(0), t->size(1), t->size(0) > 1 ? t->stride(0) : t->size(1)};
  return true;
}

int dtype_code(at::ScalarType t) {
  return t == at::kFloat ? FXB_DTYPE_F32 : t == at::kHalf ? FXB_DTYPE_F16 : t == at::kBFloat16 ? FXB_DTYPE_BF16 : -1;
}

cudaStream_t stream_of(const at::Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.get_device()).stream(); }

template <typename F> int without_gil(F launch) {
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = launch();
  Py_END_ALLOW_THREADS
  return rc;
}

PyObject* init(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 9) return PyErr_Format(PyExc_TypeError, "init: 9 arguments");
  void* p[7];
  for (int i = 0; i < 7; ++i)
    if (!(p[i] = PyLong_AsVoidPtr(a[i])) && PyErr_Occurred()) return nullptr;
  lib = {reinterpret_cast<decltype(lib.tree_attn)>(p[0]),
         reinterpret_cast<decltype(lib.tree_attn_workspace)>(p[1]),
         reinterpret_cast<decltype(lib.tree_attn_zeroed)>(p[2]),
         reinterpret_cast<decltype(lib.verify_tree)>(p[3]),
         reinterpret_cast<decltype(lib.kv_commit)>(p[4]),
         reinterpret_cast<decltype(lib.kv_fork)>(p[5]),
         reinterpret_cast<decltype(lib.kv_fork_workspace)>(p[6])};
  workspace_of = Py_NewRef(a[7]);
  tree_kind = Py_NewRef(a[8]);
  Py_RETURN_NONE;
}

// q, k, v, k_pages, v_pages, page_table, ctx_lens, n_nodes, tree_mask, scale, out
PyObject* tree_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 11) return PyErr_Format(PyExc_TypeError, "tree_attention: 11 arguments");
  const at::Tensor* t[9];
  for (int i = 0; i < 9; ++i)
    if (!(t[i] = tensor(a[i]))) Py_RETURN_NONE;
  const at::Tensor &q = *t[0], &mask = *t[8];
  const auto type = q.scalar_type();
  const int code = dtype_code(type);
  if (code < 0) Py_RETURN_NONE;
  const int64_t dev = q.get_device();
  for (int i = 0; i < 5; ++i)
    if (t[i]->dim() != 4 || t[i]->scalar_type() != type || !on(*t[i], dev) || t[i]->stride(3) != 1) Py_RETURN_NONE;
  const auto s = q.sizes(), sp = t[3]->sizes();
  const int64_t B = s[0], T = s[1], Hq = s[2], D = s[3], Hkv = t[1]->size(2), page = sp[2];
  if (at::GradMode::is_enabled())  // no backward pass: a result without one would cut gradients silently
    for (int i = 0; i < 5; ++i)
      if (t[i]->requires_grad()) Py_RETURN_NONE;
  const int64_t node_shape[4] = {B, T, Hkv, D}, page_shape[4] = {sp[0], Hkv, page, D};
  if ((D != 64 && D != 128) || T > kMaxNodes || Hkv < 1 || Hq % Hkv || t[1]->sizes() != at::IntArrayRef(node_shape) ||
      t[2]->sizes() != at::IntArrayRef(node_shape) || sp != at::IntArrayRef(page_shape) || t[4]->sizes() != sp)
    Py_RETURN_NONE;
  Table tab;
  const int64_t rows[1] = {B};
  const int32_t *lens = i32(t[6], rows, dev), *nodes = i32(t[7], rows, dev);
  if (!table(t[5], &tab, dev) || tab.rows != B || mask.scalar_type() != at::kLong || !on(mask, dev) || mask.dim() != 2 ||
      mask.size(0) != B || mask.size(1) != T || (T > 1 && mask.stride(1) != 1))
    Py_RETURN_NONE;
  if ((B && (!lens || !nodes)) || !ints({B, Hq, page, sp[0], tab.entries})) Py_RETURN_NONE;
  double scale = 1 / std::sqrt((double)D);
  if (a[9] != Py_None && (scale = PyFloat_AsDouble(a[9])) == -1 && PyErr_Occurred()) return nullptr;
  at::Tensor out;
  if (a[10] == Py_None) {
    out = at::empty(s, q.options());
  } else {
    const at::Tensor* o = tensor(a[10]);
    if (!o || o->sizes() != s || o->scalar_type() != type || !on(*o, dev) || o->stride(3) != 1) Py_RETURN_NONE;
    out = *o;
  }
  if (B && T) {
    fxb_tree_attn_args x;
    x.dtype = code;
    x.B = (int)B;
    x.T = (int)T;
    x.Hq = (int)Hq;
    x.Hkv = (int)Hkv;
    x.D = (int)D;
    x.page = (int)page;
    x.P = (int)sp[0];
    x.W = (int)tab.entries;
    x.scale = (float)scale;
    x.q = q.data_ptr();
    x.q_sb = q.stride(0), x.q_st = q.stride(1), x.q_sh = q.stride(2);
    x.k = t[1]->data_ptr();
    x.k_sb = t[1]->stride(0), x.k_st = t[1]->stride(1), x.k_sh = t[1]->stride(2);
    x.v = t[2]->data_ptr();
    x.v_sb = t[2]->stride(0), x.v_st = t[2]->stride(1), x.v_sh = t[2]->stride(2);
    x.o = out.data_ptr();
    x.o_sb = out.stride(0), x.o_st = out.stride(1), x.o_sh = out.stride(2);
    x.k_pages = t[3]->data_ptr();
    x.kp_sp = t[3]->stride(0), x.kp_sh = t[3]->stride(1), x.kp_st = t[3]->stride(2);
    x.v_pages = t[4]->data_ptr();
    x.vp_sp = t[4]->stride(0), x.vp_sh = t[4]->stride(1), x.vp_st = t[4]->stride(2);
    x.table = tab.p;
    x.table_sb = tab.stride;
    x.lens = lens;
    x.n_nodes = nodes;
    x.mask = mask.const_data_ptr<int64_t>();
    x.mask_sb = B > 1 ? mask.stride(0) : T;
    const cudaStream_t stream = stream_of(q);
    const size_t bytes = lib.tree_attn_workspace(code, x.B, x.T, x.Hq, x.Hkv, x.D);
    THPObjectPtr device(PyLong_FromLong(dev)), handle(PyLong_FromVoidPtr(stream)),
        size(PyLong_FromSize_t(bytes)),
        zeroed(PyLong_FromSize_t(lib.tree_attn_zeroed(code, x.B, x.T, x.Hq, x.Hkv, x.D)));
    PyObject* const w[5] = {tree_kind, device.get(), handle.get(), size.get(), zeroed.get()};
    THPObjectPtr ws(PyObject_Vectorcall(workspace_of, w, 5, nullptr));
    if (!ws) return nullptr;
    x.workspace = THPVariable_Unpack(ws.get()).data_ptr();
    x.workspace_bytes = (int64_t)bytes;
    if (const int rc = without_gil([&] { return lib.tree_attn(&x, stream); })) return PyLong_FromLong(rc);
  }
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

// tokens, parents, n_nodes, target_probs, u, draft_probs
PyObject* verify_tree(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 6) return PyErr_Format(PyExc_TypeError, "verify_tree: 6 arguments");
  const at::Tensor* t[6] = {};
  for (int i = 0; i < 6; ++i)
    if (!(t[i] = tensor(a[i])) && !(i == 5 && a[i] == Py_None)) Py_RETURN_NONE;
  const at::Tensor &tokens = *t[0], &p = *t[3], &u = *t[4];
  if (tokens.dim() != 2 || tokens.scalar_type() != at::kLong || !tokens.is_cuda() || !tokens.is_contiguous() ||
      p.dim() != 3)
    Py_RETURN_NONE;
  const int64_t B = tokens.size(0), T = tokens.size(1), V = p.size(2);
  if (T < 1 || T > kMaxNodes || !ints({B, V})) Py_RETURN_NONE;
  const int64_t shape[3] = {B, T, V}, rows[1] = {B}, dev = tokens.get_device();
  const at::IntArrayRef nodes(shape, 2);
  for (const at::Tensor* x : {t[3], t[5]})
    if (x && (x->scalar_type() != at::kFloat || !on(*x, dev) || x->sizes() != at::IntArrayRef(shape) ||
              (V > 1 && x->stride(2) != 1)))
      Py_RETURN_NONE;
  const int32_t *parents = i32(t[1], nodes, dev), *count = i32(t[2], rows, dev);
  if (B && (!parents || !count)) Py_RETURN_NONE;
  if (u.scalar_type() != at::kFloat || !on(u, dev) || u.sizes() != nodes || !u.is_contiguous()) Py_RETURN_NONE;
  at::Tensor path = at::empty_like(*t[1]), n_path = at::empty_like(*t[2]), next = at::empty(rows, tokens.options());
  if (B) {
    const cudaStream_t stream = stream_of(tokens);
    const int rc = without_gil([&] {
      return lib.verify_tree(tokens.const_data_ptr<int64_t>(), parents, count, p.const_data_ptr<float>(), p.stride(0),
                             p.stride(1), t[5] ? t[5]->const_data_ptr<float>() : nullptr, t[5] ? t[5]->stride(0) : 0,
                             t[5] ? t[5]->stride(1) : 0, u.const_data_ptr<float>(),
                             static_cast<int32_t*>(path.data_ptr()), static_cast<int32_t*>(n_path.data_ptr()),
                             static_cast<int64_t*>(next.data_ptr()), (int)B, (int)T, (int)V, stream);
    });
    if (rc) return PyLong_FromLong(rc);
  }
  THPObjectPtr x(THPVariable_Wrap(path)), y(THPVariable_Wrap(n_path)), z(THPVariable_Wrap(next));
  return PyTuple_Pack(3, x.get(), y.get(), z.get());
  END_HANDLE_TH_ERRORS
}

// The cache's arguments k, v, page_table, n_pages, lens, ref (k and v None: the table alone)
bool cache(PyObject* const* a, int page, fxb_kv_args* x, const at::Tensor** lens) {
  Table tab;
  const at::Tensor* ref = tensor(a[5]);
  *lens = tensor(a[4]);
  const at::Tensor* pages = tensor(a[2]);
  const int64_t dev = pages ? pages->get_device() : -1;
  if (!table(pages, &tab, dev) || !ref || ref->dim() != 1 || !ints({tab.rows, tab.entries, ref->size(0)})) return false;
  const int64_t S[1] = {tab.rows}, P[1] = {ref->size(0)};
  *x = {};
  x->S = (int)tab.rows;
  x->W = (int)tab.entries;
  x->P = (int)P[0];
  x->page = page;
  x->table = tab.p;
  x->table_ss = tab.stride;
  x->n_pages = i32(tensor(a[3]), S, dev);
  x->lens = i32(*lens, S, dev);
  x->ref = i32(ref, P, dev);
  if (S[0] && (!x->n_pages || !x->lens)) return false;
  if (P[0] && !x->ref) return false;
  if (a[0] == Py_None) return true;
  const at::Tensor *k = tensor(a[0]), *v = tensor(a[1]);
  if (!k || !v || k->dim() != 5 || v->sizes() != k->sizes() || k->size(1) != P[0] || dtype_code(k->scalar_type()) < 0 ||
      v->scalar_type() != k->scalar_type() || !on(*k, dev) || !on(*v, dev) || k->stride(4) != 1 || v->stride(4) != 1)
    return false;
  x->elem_size = (int)k->element_size();
  x->L = (int)k->size(0);
  x->H = (int)k->size(2);
  x->page = (int)k->size(3);
  x->D = (int)k->size(4);
  x->k = k->data_ptr();
  x->k_sl = k->stride(0), x->k_sp = k->stride(1), x->k_sh = k->stride(2), x->k_st = k->stride(3);
  x->v = v->data_ptr();
  x->v_sl = v->stride(0), x->v_sp = v->stride(1), x->v_sh = v->stride(2), x->v_st = v->stride(3);
  return true;
}

// k, v, page_table, n_pages, lens, ref, path, n_path, room, out, page (path None: no path, page as given)
PyObject* kv_commit(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 11) return PyErr_Format(PyExc_TypeError, "kv_commit: 11 arguments");
  fxb_kv_args x;
  const at::Tensor* lens;
  const long page = PyLong_AsLong(a[10]);
  if (page == -1 && PyErr_Occurred()) return nullptr;
  if (!cache(a, (int)page, &x, &lens)) Py_RETURN_NONE;
  const int64_t S[1] = {x.S}, dev = lens->get_device();
  const int32_t *path = nullptr, *n_path = nullptr, *room = nullptr;
  int64_t T = 0;
  if (a[6] != Py_None) {
    const at::Tensor* t = tensor(a[6]);
    if (!t || t->dim() != 2 || (T = t->size(1)) < 1 || T > kMaxNodes) Py_RETURN_NONE;
    const int64_t shape[2] = {S[0], T};
    path = i32(t, shape, dev);
    n_path = i32(tensor(a[7]), S, dev);
    if (S[0] && (!path || !n_path)) Py_RETURN_NONE;
  }
  if (a[8] != Py_None && !(room = i32(tensor(a[8]), S, dev)) && S[0]) Py_RETURN_NONE;
  at::Tensor out;
  if (a[9] == Py_None) {
    out = at::empty_like(*lens);
  } else {
    const at::Tensor* o = tensor(a[9]);
    if (!o || (!i32(o, S, dev) && S[0])) Py_RETURN_NONE;
    out = *o;
  }
  if (S[0]) {
    const cudaStream_t stream = stream_of(*lens);
    int32_t* to = static_cast<int32_t*>(out.data_ptr());
    if (const int rc = without_gil([&] { return lib.kv_commit(&x, path, T, (int)T, n_path, room, to, stream); }))
      return PyLong_FromLong(rc);
  }
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

// k, v, page_table, n_pages, lens, ref, parents; returns True
PyObject* kv_fork(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 7) return PyErr_Format(PyExc_TypeError, "kv_fork: 7 arguments");
  fxb_kv_args x;
  const at::Tensor* lens;
  if (!cache(a, 0, &x, &lens)) Py_RETURN_NONE;
  const int64_t S[1] = {x.S};
  const int32_t* parents = i32(tensor(a[6]), S, lens->get_device());
  if (S[0] && !parents) Py_RETURN_NONE;
  if (S[0]) {
    const int64_t words[1] = {(int64_t)((lib.kv_fork_workspace(x.S, x.W) + 3) / 4)};
    const at::Tensor ws = at::empty(words, lens->options());
    const cudaStream_t stream = stream_of(*lens);
    void* w = ws.data_ptr();
    if (const int rc = without_gil([&] { return lib.kv_fork(&x, parents, w, stream); })) return PyLong_FromLong(rc);
  }
  Py_RETURN_TRUE;
  END_HANDLE_TH_ERRORS
}

#define FAST(name, f) {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {FAST("init", init),           FAST("tree_attention", tree_attention),
                         FAST("verify_tree", verify_tree), FAST("kv_commit", kv_commit),
                         FAST("kv_fork", kv_fork),     {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_fxbind", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__fxbind() { return PyModule_Create(&module); }
