// Python binding of the paged-cache entries (kta_b200.ops): tensor checks, output allocation and
// the call of the C ABI in native code.
//
// A decode step's small calls run for 2 to 5 us on the GPU. The same checks in Python with a ctypes
// call took 18.5 us (rope), 21 us (cache_slots), 26 us (rope_cache) and 30 us (tree_attn) of host
// time a call; here they take 3.8, 4.4, 5.0 and 10 (two launches and three tensor maps). Every function takes all its arguments by
// position (ops.py holds the signatures and documents them), raises ValueError for tensors that do
// not fit and kta_b200.lib.KtaError for a status code, launches on the current stream of the
// tensors' device with that device current, and allocates what was not given with torch.
#include <cmath>
#include <string>

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "kta_b200.h"

namespace {

struct Refused {  // becomes a ValueError
  std::string why;
};

[[noreturn]] void refuse(const std::string& why) { throw Refused{why}; }

PyObject* g_check = nullptr;  // kta_b200.lib.check, set by the module's user
PyObject* g_rope = nullptr;   // rope() as a node of autograd's graph, set by kta_b200.ops

// Raises KtaError for a status code.
bool passed(const char* entry, int status) {
  if (status == KTA_OK) return true;
  PyObject* r = PyObject_CallFunction(g_check, "si", entry, status);
  Py_XDECREF(r);
  if (!PyErr_Occurred()) PyErr_Format(PyExc_RuntimeError, "%s: status %d", entry, status);
  return false;
}

struct Args {
  PyObject* const* at;

  const at::Tensor& tensor(int i, const char* name) const {
    if (!THPVariable_Check(at[i])) refuse(std::string(name) + " must be a tensor");
    return THPVariable_Unpack(at[i]);
  }
  bool given(int i) const { return at[i] != Py_None; }
  int64_t integer(int i) const {
    const long long v = PyLong_AsLongLong(at[i]);
    if (v == -1 && PyErr_Occurred()) throw python_error();
    return v;
  }
  double real(int i) const {
    const double v = PyFloat_AsDouble(at[i]);
    if (v == -1.0 && PyErr_Occurred()) throw python_error();
    return v;
  }
  bool truth(int i) const {
    const int v = PyObject_IsTrue(at[i]);
    if (v < 0) throw python_error();
    return v != 0;
  }
};

// The one CUDA device of a call's tensors; it is current while this lives.
class On {
 public:
  explicit On(const at::Tensor& first) : device_(first.device()) {
    if (!device_.is_cuda()) refuse("libkta_b200 operates on CUDA tensors only");
    guard_.reset_device(device_);
  }
  void also(const at::Tensor& t) const {
    if (t.device() != device_) {
      refuse("tensors on " + t.device().str() + " and " + device_.str() + ": one device is needed");
    }
  }
  at::Tensor empty(at::IntArrayRef size, at::ScalarType type) const {
    return at::detail::empty_cuda(size, type, device_, c10::nullopt);  // without the dispatcher
  }
  // A tensor of n elements in `whole`, from byte `at` on; the next one starts on a 16-byte boundary.
  static at::Tensor part(const at::Tensor& whole, int64_t& at, int64_t n, at::ScalarType type) {
    const auto meta = c10::scalarTypeToTypeMeta(type);
    at::Tensor t = at::detail::make_tensor<c10::TensorImpl>(
        c10::Storage(whole.storage()), c10::DispatchKeySet(c10::DispatchKey::CUDA), meta);
    t.unsafeGetTensorImpl()->set_storage_offset(at / static_cast<int64_t>(meta.itemsize()));
    t.unsafeGetTensorImpl()->generic_set_sizes_contiguous(at::IntArrayRef(&n, 1));
    at += bytes_of(n, type);
    return t;
  }
  static int64_t bytes_of(int64_t n, at::ScalarType type) {
    return (n * static_cast<int64_t>(c10::elementSize(type)) + 15) / 16 * 16;
  }
  void* stream() const { return c10::cuda::getCurrentCUDAStream(device_.index()).stream(); }

 private:
  c10::Device device_;
  c10::cuda::OptionalCUDAGuard guard_;
};

// Counts a call's write to a tensor of the caller: autograd compares versions before it uses what it kept.
void written(const at::Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// A contiguous 1-D tensor of `type`, of n elements where n >= 0.
void vector(const at::Tensor& t, at::ScalarType type, int64_t n, const char* name) {
  if (t.scalar_type() != type || t.dim() != 1 || !t.is_contiguous() || (n >= 0 && t.size(0) != n)) {
    refuse(std::string(name) + " must be a contiguous " + c10::toString(type) + " vector" +
           (n >= 0 ? " of " + std::to_string(n) + " elements" : ""));
  }
}

void block_tables(const at::Tensor& t, int64_t batch) {
  if (t.scalar_type() != at::kInt || t.dim() != 2 || t.size(0) != batch ||
      (t.size(1) > 1 && t.stride(1) != 1)) {
    refuse("block_tables must be int32 [B, max_blocks] with unit column stride");
  }
}

bool is_bf16(const at::Tensor& t, const char* name) {
  if ((t.scalar_type() != at::kHalf && t.scalar_type() != at::kBFloat16) || t.dim() != 3) {
    refuse(std::string(name) + " must be an f16 or bf16 [tokens, heads, D] tensor");
  }
  return t.scalar_type() == at::kBFloat16;
}

// [tokens, heads, D] like q, with unit stride in D.
void rows_like(const at::Tensor& t, const at::Tensor& q, const char* name) {
  if (t.scalar_type() != q.scalar_type() || t.dim() != 3 || t.size(0) != q.size(0) ||
      t.size(2) != q.size(2) || (t.size(2) > 1 && t.stride(2) != 1)) {
    refuse(std::string(name) + " must be a " + c10::toString(q.scalar_type()) +
           " tensor [tokens, heads, D] with the tokens and D of the other rows and unit stride in D");
  }
}

// Token (0) or head (1) stride; torch leaves that of a dimension of size one open.
int64_t row_stride(const at::Tensor& t, int dim) {
  if (t.size(dim) > 1) return t.stride(dim);
  return dim == 0 ? t.size(1) * t.size(2) : t.size(2);
}

// Bytes of a position.
int64_t angles(const at::Tensor& positions, const at::Tensor& freqs, int64_t tokens) {
  const bool wide = positions.scalar_type() == at::kLong;
  if (!wide && positions.scalar_type() != at::kInt) refuse("positions must be int32 or int64");
  vector(positions, positions.scalar_type(), tokens, "positions");
  vector(freqs, at::kDouble, -1, "freqs");
  return wide ? 8 : 4;
}

void caches(const at::Tensor& k, const at::Tensor& v, const at::Tensor& q) {
  if (k.dim() != 4 || k.sizes() != v.sizes() || k.size(3) != q.size(2) ||
      k.scalar_type() != q.scalar_type() || v.scalar_type() != q.scalar_type()) {
    refuse("K and V caches must be [num_blocks, block_size, Hkv, D] of Q's type and D");
  }
  if (!k.is_contiguous() || !v.is_contiguous()) refuse("K and V caches must be contiguous");
}

// The lock is taken again on the way out of an exception too: a tensor without memory (a sparse one, one
// that a tracer made) throws from data_ptr().
template <typename F>
int without_gil(F&& call) {
  struct Released {
    PyThreadState* state = PyEval_SaveThread();
    ~Released() { PyEval_RestoreThread(state); }
  } released;
  return call();
}

// Runs `body` with `n` arguments; a refusal becomes a ValueError, any other C++ exception the
// Python error that torch makes of it.
template <typename F>
PyObject* guarded(PyObject* const* args, Py_ssize_t got, Py_ssize_t n, F&& body) {
  HANDLE_TH_ERRORS
  if (got != n) {
    PyErr_Format(PyExc_TypeError, "%zd arguments, %zd given", n, got);
    return nullptr;
  }
  try {
    return body(Args{args});
  } catch (const Refused& r) {
    PyErr_SetString(PyExc_ValueError, r.why.c_str());
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

// (context_lens, new_lens, block_tables, free_blocks, block_size, max_tokens, slots, positions,
//  offsets, used)
PyObject* cache_slots(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(args, n, 10, [](const Args& a) -> PyObject* {
    const at::Tensor& ctx = a.tensor(0, "context_lens");
    const at::Tensor& fresh = a.tensor(1, "new_lens");
    const at::Tensor& tables = a.tensor(2, "block_tables");
    const at::Tensor& pool = a.tensor(3, "free_blocks");
    const int64_t block = a.integer(4), rows = a.integer(5);
    On dev(ctx);
    dev.also(fresh);
    dev.also(tables);
    dev.also(pool);
    vector(ctx, at::kInt, -1, "context_lens");
    const int64_t batch = ctx.size(0);
    vector(fresh, at::kInt, batch, "new_lens");
    vector(pool, at::kInt, -1, "free_blocks");
    block_tables(tables, batch);
    if (rows <= 0) refuse("max_tokens must be positive");
    // What is not given is one allocation: with four a call takes 6.9 us of host time, so 4.4, and 3.0
    // where all are given.
    at::Tensor whole;
    int64_t at = 0;
    auto made = [&](int i, int64_t size, at::ScalarType type, const char* name) -> at::Tensor {
      if (!a.given(i)) {
        if (!whole.defined()) {
          whole = dev.empty({On::bytes_of(rows, at::kLong) + On::bytes_of(rows, at::kInt) +
                             On::bytes_of(batch + 1, at::kInt) + On::bytes_of(1, at::kInt)}, at::kByte);
        }
        return On::part(whole, at, size, type);
      }
      const at::Tensor& t = a.tensor(i, name);
      dev.also(t);
      vector(t, type, size, name);
      return t;
    };
    const at::Tensor slots = made(6, rows, at::kLong, "slots");
    const at::Tensor positions = made(7, rows, at::kInt, "positions");
    const at::Tensor offsets = made(8, batch + 1, at::kInt, "offsets");
    const at::Tensor used = made(9, 1, at::kInt, "used");
    const int64_t stride = batch > 1 ? tables.stride(0) : tables.size(1);
    const int status = without_gil([&] {
      return kta_cache_slots(ctx.data_ptr(), fresh.data_ptr(), tables.data_ptr(), pool.data_ptr(),
                             slots.data_ptr(), positions.data_ptr(), offsets.data_ptr(),
                             used.data_ptr(), batch, tables.size(1), stride, pool.size(0), block, rows,
                             dev.stream());
    });
    if (!passed("kta_cache_slots", status)) return nullptr;
    for (const at::Tensor* t : {&tables, &slots, &positions, &offsets, &used}) written(*t);
    PyObject* r = PyTuple_New(4);
    if (r == nullptr) return nullptr;
    PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(slots));
    PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(positions));
    PyTuple_SET_ITEM(r, 2, THPVariable_Wrap(offsets));
    PyTuple_SET_ITEM(r, 3, THPVariable_Wrap(used));
    return r;
  });
}

// (x, positions, freqs, interleaved, inverse, scale, out)
PyObject* rope(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(args, n, 7, [](const Args& a) -> PyObject* {
    const at::Tensor& x = a.tensor(0, "X");
    const at::Tensor& positions = a.tensor(1, "positions");
    const at::Tensor& freqs = a.tensor(2, "freqs");
    const bool bf16 = is_bf16(x, "X");
    rows_like(x, x, "X");
    const int64_t size = angles(positions, freqs, x.size(0));
    if (a.given(6)) {
      const at::Tensor& out = a.tensor(6, "out");
      rows_like(out, x, "out");
      if (out.size(1) != x.size(1)) refuse("out must have X's heads");
    }
    if (c10::GradMode::is_enabled() &&
        (x.requires_grad() || freqs.requires_grad() || (a.given(6) && a.tensor(6, "out").requires_grad()))) {
      if (freqs.requires_grad()) refuse("there is no gradient of freqs: detach them");
      if (a.given(6)) refuse("out cannot carry a gradient: leave it out, or use torch.no_grad()");
      if (g_rope == nullptr) refuse("kta_b200.ops is not loaded");
      return PyObject_Vectorcall(g_rope, a.at, 6, nullptr);  // which comes back with gradients off
    }
    On dev(x);
    dev.also(positions);
    dev.also(freqs);
    const at::Tensor out = a.given(6) ? a.tensor(6, "out") : dev.empty(x.sizes(), x.scalar_type());
    dev.also(out);
    const int inter = a.truth(3), inverse = a.truth(4);
    const float scale = static_cast<float>(a.real(5));
    auto* entry = bf16 ? kta_rope_bf16 : kta_rope_f16;
    const int status = without_gil([&] {
      return entry(x.data_ptr(), positions.data_ptr(), size, freqs.data_ptr(), out.data_ptr(), x.size(0),
                   x.size(1), x.size(2), 2 * freqs.size(0), row_stride(x, 0), row_stride(x, 1),
                   row_stride(out, 0), row_stride(out, 1), inter, inverse, scale, dev.stream());
    });
    if (!passed(bf16 ? "kta_rope_bf16" : "kta_rope_f16", status)) return nullptr;
    written(out);
    return THPVariable_Wrap(out);
  });
}

// (q, k, v, positions, slots, freqs, k_cache, v_cache, interleaved, scale, out)
PyObject* rope_cache(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(args, n, 11, [](const Args& a) -> PyObject* {
    const at::Tensor& q = a.tensor(0, "Q");
    const at::Tensor& k = a.tensor(1, "K");
    const at::Tensor& v = a.tensor(2, "V");
    const at::Tensor& positions = a.tensor(3, "positions");
    const at::Tensor& slots = a.tensor(4, "slots");
    const at::Tensor& freqs = a.tensor(5, "freqs");
    const at::Tensor& kc = a.tensor(6, "k_cache");
    const at::Tensor& vc = a.tensor(7, "v_cache");
    const bool bf16 = is_bf16(q, "Q");
    rows_like(q, q, "Q");
    rows_like(k, q, "K");
    rows_like(v, q, "V");
    caches(kc, vc, q);
    const int64_t tokens = q.size(0), hkv = k.size(1);
    if (v.size(1) != hkv || kc.size(2) != hkv) refuse("K, V and the caches must have the same heads");
    const int64_t size = angles(positions, freqs, tokens);
    vector(slots, at::kLong, tokens, "slots");
    if (a.given(10)) {
      const at::Tensor& out = a.tensor(10, "out");
      rows_like(out, q, "out");
      if (out.size(1) != q.size(1)) refuse("out must have Q's heads");
    }
    On dev(q);
    for (const at::Tensor* t : {&k, &v, &positions, &slots, &freqs, &kc, &vc}) dev.also(*t);
    const at::Tensor out = a.given(10) ? a.tensor(10, "out") : dev.empty(q.sizes(), q.scalar_type());
    dev.also(out);
    const int inter = a.truth(8);
    const float scale = static_cast<float>(a.real(9));
    const int64_t strides[8] = {row_stride(q, 0), row_stride(q, 1), row_stride(k, 0),   row_stride(k, 1),
                                row_stride(v, 0), row_stride(v, 1), row_stride(out, 0), row_stride(out, 1)};
    auto* entry = bf16 ? kta_rope_cache_bf16 : kta_rope_cache_f16;
    const int status = without_gil([&] {
      return entry(q.data_ptr(), k.data_ptr(), v.data_ptr(), positions.data_ptr(), size, slots.data_ptr(),
                   freqs.data_ptr(), out.data_ptr(), kc.data_ptr(), vc.data_ptr(), tokens, q.size(1), hkv,
                   q.size(2), 2 * freqs.size(0), strides, kc.size(0) * kc.size(1), inter, scale,
                   dev.stream());
    });
    if (!passed(bf16 ? "kta_rope_cache_bf16" : "kta_rope_cache_f16", status)) return nullptr;
    for (const at::Tensor* t : {&kc, &vc, &out}) written(*t);
    return THPVariable_Wrap(out);
  });
}

// (q, k_cache, v_cache, block_tables, context_lens, offsets, max_new, tree, scale, out, lse,
//  workspace)
PyObject* tree_attn(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(args, n, 12, [](const Args& a) -> PyObject* {
    const at::Tensor& q = a.tensor(0, "Q");
    const at::Tensor& kc = a.tensor(1, "k_cache");
    const at::Tensor& vc = a.tensor(2, "v_cache");
    const at::Tensor& tables = a.tensor(3, "block_tables");
    const at::Tensor& ctx = a.tensor(4, "context_lens");
    const at::Tensor& offsets = a.tensor(5, "offsets");
    const int64_t max_new = a.integer(6);
    const bool bf16 = is_bf16(q, "Q");
    const int64_t tokens = q.size(0), hq = q.size(1), d = q.size(2);
    if (d > 1 && (q.stride(2) != 1 || (hq > 1 && q.stride(1) != d))) {
      refuse("Q must be [tokens, Hq, D] with contiguous heads");
    }
    caches(kc, vc, q);
    const int64_t hkv = kc.size(2);
    vector(ctx, at::kInt, -1, "context_lens");
    const int64_t batch = ctx.size(0);
    vector(offsets, at::kInt, batch + 1, "offsets");
    block_tables(tables, batch);
    On dev(q);
    for (const at::Tensor* t : {&kc, &vc, &tables, &ctx, &offsets}) dev.also(*t);
    const void* tree = nullptr;
    if (a.given(7)) {
      const at::Tensor& t = a.tensor(7, "tree");
      dev.also(t);
      vector(t, at::kLong, tokens, "tree");
      tree = t.data_ptr();
    }
    const float scale = static_cast<float>(a.given(8) ? a.real(8) : 1.0 / std::sqrt(static_cast<double>(d)));
    const at::Tensor out = a.given(9) ? a.tensor(9, "out") : dev.empty(q.sizes(), q.scalar_type());
    if (out.sizes() != q.sizes() || out.scalar_type() != q.scalar_type() || !out.is_contiguous()) {
      refuse("out must be a contiguous tensor of Q's shape and type");
    }
    const at::Tensor lse = a.given(10) ? a.tensor(10, "lse") : dev.empty({tokens, hq}, at::kFloat);
    if (lse.dim() != 2 || lse.size(0) != tokens || lse.size(1) != hq || lse.scalar_type() != at::kFloat ||
        !lse.is_contiguous()) {
      refuse("lse must be a contiguous fp32 [tokens, Hq] tensor");
    }
    const at::Tensor ws =
        a.given(11) ? a.tensor(11, "workspace")
                    : dev.empty({static_cast<int64_t>(kta_tree_attn_workspace_bytes(max_new, hq, hkv, d))},
                                at::kByte);
    if (!ws.is_contiguous()) refuse("workspace must be contiguous");
    dev.also(out);
    dev.also(lse);
    dev.also(ws);
    const int64_t stride = batch > 1 ? tables.stride(0) : tables.size(1);
    auto* entry = bf16 ? kta_tree_attn_bf16 : kta_tree_attn_f16;
    const int status = without_gil([&] {
      return entry(q.data_ptr(), kc.data_ptr(), vc.data_ptr(), tables.data_ptr(), ctx.data_ptr(),
                   offsets.data_ptr(), tree, out.data_ptr(), lse.data_ptr(), tokens, batch, hq, hkv, d,
                   row_stride(q, 0), kc.size(0), kc.size(1), tables.size(1), stride, max_new, scale,
                   ws.data_ptr(), ws.nbytes(), dev.stream());
    });
    if (!passed(bf16 ? "kta_tree_attn_bf16" : "kta_tree_attn_f16", status)) return nullptr;
    for (const at::Tensor* t : {&out, &lse}) written(*t);
    PyObject* r = PyTuple_New(2);
    if (r == nullptr) return nullptr;
    PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(out));
    PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(lse));
    return r;
  });
}

// What the functions above call.
template <PyObject*& F>
PyObject* set_call(PyObject*, PyObject* f) {
  Py_INCREF(f);
  Py_XDECREF(F);
  F = f;
  Py_RETURN_NONE;
}

#define FAST(f) reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL

PyMethodDef g_methods[] = {
    {"cache_slots", FAST(cache_slots), nullptr}, {"rope", FAST(rope), nullptr},
    {"rope_cache", FAST(rope_cache), nullptr},   {"tree_attn", FAST(tree_attn), nullptr},
    {"set_check", set_call<g_check>, METH_O, nullptr},
    {"set_rope", set_call<g_rope>, METH_O, nullptr},
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_binding", nullptr, -1, g_methods,
                        nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__binding() { return PyModule_Create(&g_module); }
