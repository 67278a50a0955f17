// Python entry points of the speculative-decoding calls on torch CUDA tensors: argument checks, the current stream and the
// call into the C ABI, without a Python-level step per tensor.  These calls run once a layer or once a step and often
// eagerly; through ctypes and Python checks a call took 9 to 17 us of the host, more than most of them take on the GPU.
//
// Wrong types, extents, strides or devices raise ValueError; a non-zero status of the C entry raises the package's error;
// errors of torch (memory for a result) keep their type.
// No C++ exception leaves a function.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <stdexcept>
#include <string>

#include "../../../include/wukong_b200.h"

namespace {

PyObject* g_error = nullptr;      // the package's exception, handed over at import

struct Refused : std::runtime_error {
  using std::runtime_error::runtime_error;
};
struct PyRaised {};      // a Python exception is set

struct Call {
  PyObject* const* args;
  int device;

  Call(PyObject* const* a, Py_ssize_t n, Py_ssize_t want) : args(a), device(-1) {
    if (n != want) throw Refused("wrong number of arguments");
  }
  bool none(int i) const { return args[i] == Py_None; }
  const at::Tensor& tensor(int i, const char* what) const {
    if (!THPVariable_Check(args[i])) throw Refused(std::string(what) + " must be a tensor");
    return THPVariable_Unpack(args[i]);
  }
  int64_t integer(int i) const {
    const int64_t v = PyLong_AsLongLong(args[i]);
    if (v == -1 && PyErr_Occurred()) throw PyRaised();
    return v;
  }
  double real(int i) const {
    const double v = PyFloat_AsDouble(args[i]);
    if (v == -1.0 && PyErr_Occurred()) throw PyRaised();
    return v;
  }
  // the tensor whose device the call runs on: it has to be the current one
  void here(const at::Tensor& t) {
    if (!t.is_cuda() || t.get_device() != c10::cuda::current_device()) throw Refused("every tensor must lie on the current CUDA device");
    device = (int)t.get_device();
  }
  void on_device(const at::Tensor& t, const char* what) const {
    if (!t.is_cuda() || t.get_device() != device) throw Refused(std::string(what) + " must lie on the current CUDA device");
  }
  // address of a contiguous tensor of n values
  void* values(int i, int64_t n, at::ScalarType type, const char* what) const {
    const at::Tensor& t = tensor(i, what);
    on_device(t, what);
    if (t.scalar_type() != type || t.numel() != n || !t.is_contiguous())
      throw Refused(std::string(what) + " must be a contiguous " + c10::toString(type) + " tensor of " + std::to_string(n) + " values");
    return t.data_ptr();
  }
  void* stream() const { return (void*)c10::cuda::getCurrentCUDAStream(device).stream(); }
};

// row pitch of a matrix whose rows hold `cols` values
int64_t pitch(const at::Tensor& t, int64_t cols, const char* what) {
  if (t.dim() != 2 || t.size(1) < cols || t.stride(1) != 1) throw Refused(std::string(what) + " must be a matrix of at least " + std::to_string(cols) + " columns with unit column stride");
  return t.size(0) > 1 ? t.stride(0) : std::max(t.stride(0), t.size(1));
}
// rows of dense values, `stride` apart: [n], [rows, values] or [rows, heads, values], from which any number of values is used
void dense_rows(const at::Tensor& t, int64_t rows, int64_t stride, int64_t width, const char* what) {
  int64_t dense = 1;
  for (int64_t d = t.dim() - 1; d >= (t.dim() > 1 ? 1 : 0); --d) {
    if (t.size(d) != 1 && t.stride(d) != dense) throw Refused(std::string(what) + " must hold the values of a row one behind the other");
    dense *= t.size(d);
  }
  constexpr int64_t MOST = (int64_t)1 << 31;      // (no product wraps around)
  if (rows > 0 && (t.dim() == 0 || rows > MOST || width > MOST || stride < 0 || stride > MOST ||
                   (t.storage_offset() + (rows - 1) * stride + width) * (int64_t)t.element_size() > (int64_t)t.storage().nbytes()))
    throw Refused(std::string(what) + " does not hold " + std::to_string(rows) + " rows of pitch " + std::to_string(stride));
}
int float_code(const at::Tensor& t, const char* what) {
  if (t.scalar_type() == at::kFloat) return 0;
  if (t.scalar_type() == at::kBFloat16) return 1;
  throw Refused(std::string(what) + " must be f32 or bf16");
}
int64_t table_width(const Call& c, int i, int64_t mbps, int64_t trees) {
  const at::Tensor& t = c.tensor(i, "block_table");
  c.on_device(t, "block_table");
  if (t.scalar_type() != at::kInt || mbps < 1 || t.numel() % mbps || !t.is_contiguous()) throw Refused("block_table must be a contiguous int32 [slots, mbps]");
  if (trees > 0 && t.numel() == 0) throw Refused("block_table has no rows");
  return mbps;
}
struct Cache {
  int64_t layers, pages, kv_heads, page_tokens, head_dim, layer_stride;
  char *k, *v;
};
// k, v, layers, num_pages, kv_heads, page_tokens, head_dim from argument i on
Cache cache_of(const Call& c, int i) {
  const at::Tensor &k = c.tensor(i, "the cache"), &v = c.tensor(i + 1, "the cache");
  Cache s{c.integer(i + 2), c.integer(i + 3), c.integer(i + 4), c.integer(i + 5), c.integer(i + 6), 0, nullptr, nullptr};
  const int64_t want[5] = {s.layers, s.pages, s.kv_heads, s.page_tokens, s.head_dim};
  for (const at::Tensor* t : {&k, &v}) {
    c.on_device(*t, "the cache");
    if (t->scalar_type() != at::kBFloat16 || !t->is_contiguous() || t->sizes() != c10::IntArrayRef(want, 5))
      throw Refused("the cache must be contiguous bf16 [layers, pages, kv_heads, page_tokens, head_dim]");
  }
  s.layer_stride = s.pages * s.kv_heads * s.page_tokens * s.head_dim;
  s.k = static_cast<char*>(k.data_ptr());
  s.v = static_cast<char*>(v.data_ptr());
  return s;
}
void check(int rc, const char* what) {
  if (rc == 0) return;
  PyErr_Format(g_error ? g_error : PyExc_RuntimeError, "%s failed with status %d", what, rc);
  throw PyRaised();
}
// A C entry without the interpreter lock: a launch waits while the GPU's queue is full, and other threads (a host function of
// the stream among them, which the queue may be waiting for) have to go on.
template <typename... P, typename... A>
int unlocked(int (*entry)(P...), A... args) {
  PyThreadState* state = PyEval_SaveThread();
  const int rc = entry(static_cast<P>(args)...);
  PyEval_RestoreThread(state);
  return rc;
}
template <typename F>
PyObject* guarded(F&& f) {
  try {
    return f();
  } catch (const PyRaised&) {
  } catch (const Refused& e) {
    PyErr_SetString(PyExc_ValueError, e.what());
  } catch (...) {
    torch::translate_exception_to_python(std::current_exception());
  }
  return nullptr;
}
PyObject* same(PyObject* o) {
  Py_INCREF(o);
  return o;
}

// q, q_row_stride, k, v, layers, num_pages, kv_heads, page_tokens, head_dim, layer, block_table, tree_slot, tree_ctx, tree_row0,
// tree_mask, out, q_heads, mbps, max_nodes, scale, scratch -> out
PyObject* paged_attn_tree(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&] {
    Call c(args, n, 21);
    const at::Tensor &q = c.tensor(0, "q"), &out = c.tensor(15, "out"), &mask = c.tensor(14, "tree_mask"), &scratch = c.tensor(20, "scratch");
    c.here(out);
    const Cache kv = cache_of(c, 2);
    const int64_t stride = c.integer(1), layer = c.integer(9), q_heads = c.integer(16);
    if (q_heads < 1 || q_heads > 1 << 20) throw Refused("q_heads must be positive");
    const int64_t width = q_heads * kv.head_dim;
    const int64_t rows = out.dim() == 2 ? out.size(0) : 0, trees = c.tensor(11, "tree_slot").numel();
    const int q_code = float_code(q, "q"), out_code = float_code(out, "out");
    if (layer < 0 || layer >= kv.layers) throw Refused("no such layer");
    c.on_device(q, "q");
    dense_rows(q, rows, stride, width, "q");
    if (mask.dim() != 2 || mask.size(0) < rows) throw Refused("tree_mask must have a row for each row of out");
    const int64_t ldo = pitch(out, width, "out"), mbps = table_width(c, 10, c.integer(17), trees);
    const int64_t at_layer = layer * kv.layer_stride * 2;
    check(unlocked(wkb_paged_attn_tree, q.data_ptr(), q_code, stride, kv.k + at_layer, kv.v + at_layer, kv.pages, (const uint32_t*)c.tensor(10, "block_table").data_ptr(),
                              (const int*)c.values(11, trees, at::kInt, "tree_slot"), (const int*)c.values(12, trees, at::kInt, "tree_ctx"),
                              (const int*)c.values(13, trees + 1, at::kInt, "tree_row0"), (const uint32_t*)c.values(14, mask.numel(), at::kInt, "tree_mask"), mask.size(1),
                              out.data_ptr(), out_code, ldo, rows, trees, c.integer(18), q_heads, kv.kv_heads, kv.head_dim, kv.page_tokens, mbps, (float)c.real(19),
                              c.values(20, scratch.numel(), at::kByte, "scratch"), scratch.numel(), c.stream()),
          "wkb_paged_attn_tree");
    return same(args[15]);
  });
}

// logits, temperature or None, out or None -> out
PyObject* token_probs(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Call c(args, n, 3);
    const at::Tensor& x = c.tensor(0, "logits");
    c.here(x);
    if (x.dim() != 2) throw Refused("logits must be a matrix");
    const int64_t rows = x.size(0), cols = x.size(1), ld = pitch(x, cols, "logits");
    const int code = float_code(x, "logits");
    at::Tensor made;
    if (c.none(2)) made = at::empty({rows, cols}, x.options().dtype(at::kFloat));
    const at::Tensor& out = c.none(2) ? made : c.tensor(2, "out");
    c.on_device(out, "out");
    if (out.scalar_type() != at::kFloat || out.sizes() != x.sizes()) throw Refused("out must be f32 of the logits' shape");
    check(unlocked(wkb_token_probs, x.data_ptr(), code, ld, c.none(1) ? nullptr : (const float*)c.values(1, rows, at::kFloat, "temperature"), (float*)out.data_ptr(),
                          pitch(out, cols, "out"), rows, cols, c.stream()),
          "wkb_token_probs");
    return c.none(2) ? THPVariable_Wrap(std::move(made)) : same(args[2]);
  });
}

// probs, draft or None, token, parent, tree_row0, u_node, u_final, max_nodes, max_path, path, n_path, tokens (three None: made
// here) -> (path, n_path, tokens)
PyObject* tree_verify(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Call c(args, n, 12);
    const at::Tensor& p = c.tensor(0, "probs");
    c.here(p);
    if (p.dim() != 2 || p.scalar_type() != at::kFloat) throw Refused("probs must be f32 [rows, vocabulary]");
    const int64_t rows = p.size(0), cols = p.size(1), trees = c.tensor(4, "tree_row0").numel() - 1, max_nodes = c.integer(7), max_path = c.integer(8);
    const float* draft = nullptr;
    int64_t ldq = 0;
    if (!c.none(1)) {
      const at::Tensor& d = c.tensor(1, "draft");
      c.on_device(d, "draft");
      if (d.scalar_type() != at::kFloat || d.sizes() != p.sizes()) throw Refused("probs and draft must be f32 of one shape");
      ldq = pitch(d, cols, "draft");
      draft = (const float*)d.data_ptr();
    }
    if (trees < 0 || max_path < 1) throw Refused("tree_row0 must hold one entry more than trees, max_path must be positive");
    const bool make = c.none(9) && c.none(10) && c.none(11);
    at::Tensor path, n_path, tokens;
    int *pp, *pn, *pt;
    if (make) {
      const auto opt = p.options().dtype(at::kInt);
      path = at::empty({trees, max_path}, opt);
      n_path = at::empty({trees}, opt);
      tokens = at::empty({trees, max_path}, opt);
      pp = (int*)path.data_ptr(); pn = (int*)n_path.data_ptr(); pt = (int*)tokens.data_ptr();
    } else {
      pp = (int*)c.values(9, trees * max_path, at::kInt, "path");
      pn = (int*)c.values(10, trees, at::kInt, "n_path");
      pt = (int*)c.values(11, trees * max_path, at::kInt, "tokens");
    }
    check(unlocked(wkb_tree_verify, (const float*)p.data_ptr(), pitch(p, cols, "probs"), draft, ldq, (const int*)c.values(2, rows, at::kInt, "token"),
                          (const int*)c.values(3, rows, at::kInt, "parent"), (const int*)c.values(4, trees + 1, at::kInt, "tree_row0"), rows, trees, max_nodes, cols,
                          (const float*)c.values(5, rows, at::kFloat, "u_node"), (const float*)c.values(6, trees, at::kFloat, "u_final"), pp, pt, pn, max_path,
                          c.stream()),
          "wkb_tree_verify");
    if (!make) return PyTuple_Pack(3, args[9], args[10], args[11]);
    PyObject* r = PyTuple_New(3);
    if (!r) throw PyRaised();
    PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(std::move(path)));
    PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(std::move(n_path)));
    PyTuple_SET_ITEM(r, 2, THPVariable_Wrap(std::move(tokens)));
    return r;
  });
}

// k, v, layers, num_pages, kv_heads, page_tokens, head_dim, block_table, tree_slot, tree_ctx, path, n_path, mbps, new_ctx or None
PyObject* paged_kv_commit(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Call c(args, n, 14);
    const at::Tensor &slot = c.tensor(8, "tree_slot"), &path = c.tensor(10, "path");
    c.here(slot);
    const int64_t trees = slot.numel();
    const Cache kv = cache_of(c, 0);
    if (path.dim() != 2 || path.size(0) != trees) throw Refused("path must be int32 [n, max_path]");
    const int64_t mbps = table_width(c, 7, c.integer(12), trees);
    check(unlocked(wkb_paged_kv_commit, kv.k, kv.v, kv.layers, kv.layer_stride, kv.pages, (const uint32_t*)c.tensor(7, "block_table").data_ptr(),
                              (const int*)c.values(8, trees, at::kInt, "tree_slot"), (const int*)c.values(9, trees, at::kInt, "tree_ctx"),
                              (const int*)c.values(10, path.numel(), at::kInt, "path"), (const int*)c.values(11, trees, at::kInt, "n_path"), path.size(1), trees,
                              kv.kv_heads, kv.head_dim, kv.page_tokens, mbps, c.none(13) ? nullptr : (int*)c.values(13, trees, at::kInt, "new_ctx"), c.stream()),
          "wkb_paged_kv_commit");
    Py_RETURN_NONE;
  });
}

PyObject* set_error(PyObject*, PyObject* cls) {
  Py_INCREF(cls);
  Py_XSETREF(g_error, cls);
  Py_RETURN_NONE;
}

template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyMethodDef fast(const char* name) {
  return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(F)), METH_FASTCALL, nullptr};
}
PyMethodDef methods[] = {fast<paged_attn_tree>("paged_attn_tree"), fast<token_probs>("token_probs"),          fast<tree_verify>("tree_verify"),
                         fast<paged_kv_commit>("paged_kv_commit"), {"set_error", set_error, METH_O, nullptr}, {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_torch_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__torch_calls(void) {
  PyObject* m = PyModule_Create(&module);
  if (m && PyModule_AddStringConstant(m, "torch_version", WKB_TORCH_VERSION) != 0) Py_CLEAR(m);
  return m;
}
