// Native binding of the 8-bit page cache operators: the argument checks of ops.py's wrappers, the outputs, and the call of the C ABI, for
// calls whose kernels take a few microseconds.  Through ctypes and checks in Python such a call costs the host 8 to 15 us, most of it
// reading tensor attributes and converting 20 arguments one by one; here 3 to 7, most of it launches.
//
// The C ABI stays the only way to the kernels: ops.py hands over the addresses of its entry points (bind), so that this module
// has no library of its own to find and follows whichever one _lib.py loaded.

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <stdexcept>
#include <string>

#include "b200_decode.h"

namespace {

struct Refused : std::runtime_error {
  using std::runtime_error::runtime_error;
};
[[noreturn]] void refuse(const std::string& why) { throw Refused(why); }
std::string shape_of(const at::Tensor& t) {
  std::string s = "[";
  for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
  return s + "]";
}

// Entry points of the loaded library and what raises their errors, from bind().
decltype(&b200_kv_slot_map) p_slot_map;
decltype(&b200_kv8_append) p_append;
decltype(&b200_kv8_attn_workspace_bytes) p_decode_bytes;
decltype(&b200_kv8_attn_decode) p_decode;
decltype(&b200_kv8_attn_prefill_workspace_bytes) p_prefill_bytes;
decltype(&b200_kv8_attn_prefill) p_prefill;
PyObject* p_check;

const at::Tensor& tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) refuse(std::string(name) + " must be a tensor");
  return THPVariable_Unpack(o);
}
void need(const at::Tensor& t, const char* name, at::ScalarType dtype) {
  if (t.scalar_type() != dtype) refuse(std::string(name) + " must be " + c10::toString(dtype) + ", got " + c10::toString(t.scalar_type()));
  if (!t.is_contiguous()) refuse(std::string(name) + " must be contiguous");
}
// The device that all operands are on, which has to be the current one: operands of another are an error and not a fault.
int device_of(std::initializer_list<const at::Tensor*> operands) {
  const int here = (*operands.begin())->get_device();
  for (const at::Tensor* t : operands) {
    if (!t->is_cuda()) refuse("operands must be CUDA tensors (this path has no CPU implementation)");
    if (t->get_device() != here) refuse("operands are on cuda:" + std::to_string(here) + " and cuda:" + std::to_string(t->get_device()));
  }
  const int current = c10::cuda::current_device();
  if (here != current) refuse("operands are on cuda:" + std::to_string(here) + ", the current device is cuda:" + std::to_string(current));
  return here;
}
void* stream_of(int device) { return c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(device)).stream(); }
int whole(PyObject* o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw python_error();
  if (v < INT_MIN || v > INT_MAX) refuse("a number of " + std::to_string(v) + " does not fit 32 bits");
  return static_cast<int>(v);
}
int narrow(int64_t v, const char* what) {
  if (v > INT_MAX) refuse(std::string(what) + " of " + std::to_string(v) + " does not fit 32 bits");
  return static_cast<int>(v);
}
// An uninitialised tensor of the type and on the device of `like`, from the caching allocator without a detour through the dispatcher.
at::Tensor fresh_tensor(at::IntArrayRef sizes, const at::Tensor& like) {
  return at::detail::empty_cuda(sizes, like.scalar_type(), like.device(), std::nullopt);
}
// Numbers offset .. offset + n - 1 of a row of whole numbers, as a tensor on the same memory (six of them by way of the dispatcher: 2 us).
at::Tensor part_of(const at::Tensor& all, int64_t offset, int64_t n) {
  at::Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::TensorImpl::VIEW, c10::Storage(all.storage()), all.key_set(), all.dtype());
  t.unsafeGetTensorImpl()->set_storage_offset(offset);
  t.unsafeGetTensorImpl()->set_sizes_contiguous({n});
  return t;
}
// An optional status word on `device`.
void* status_word(PyObject* o, int device) {
  if (o == Py_None) return nullptr;
  const at::Tensor& t = tensor(o, "status");
  if (t.get_device() != device || !t.is_cuda() || !t.is_contiguous()) refuse("status must be a contiguous CUDA tensor beside the operands");
  if (t.nbytes() < 4) refuse("status holds less than a 4-byte word");
  return t.data_ptr();
}
template <typename F>
int without_gil(F&& f) {
  struct Released {
    PyThreadState* state = PyEval_SaveThread();
    ~Released() { PyEval_RestoreThread(state); }
  } released;
  return f();
}
// Raises what the library says about rc.
PyObject* failed(int rc, const char* where) {
  PyObject* r = PyObject_CallFunction(p_check, "is", rc, where);
  Py_XDECREF(r);
  if (!PyErr_Occurred()) PyErr_Format(PyExc_RuntimeError, "%s: code %d", where, rc);
  return nullptr;
}

struct Cache {
  const at::Tensor &k, &v, &ks, &vs;
  int blocks, heads, dim;
};
Cache cache_of(PyObject* const* args) {
  const at::Tensor &k = tensor(args[0], "k_pool"), &v = tensor(args[1], "v_pool"), &ks = tensor(args[2], "k_scale"), &vs = tensor(args[3], "v_scale");
  need(k, "k_pool", at::kFloat8_e4m3fn);
  need(v, "v_pool", at::kFloat8_e4m3fn);
  need(ks, "k_scale", at::kFloat8_e8m0fnu);
  need(vs, "v_scale", at::kFloat8_e8m0fnu);
  if (k.dim() != 4 || k.size(2) != 16) refuse("k_pool must be [num_blocks, kv_heads, 16, head_dim], got " + shape_of(k));
  if (v.sizes() != k.sizes() || ks.sizes() != k.sizes().slice(0, 2) || vs.sizes() != k.sizes().slice(0, 2))
    refuse("pools and scales do not match each other");
  return {k, v, ks, vs, narrow(k.size(0), "num_blocks"), narrow(k.size(1), "kv_heads"), narrow(k.size(3), "head_dim")};
}
// Query rows, the output (made here unless given) and the index tensor of an attention call.
struct Queries {
  const at::Tensor &q, &index;
  at::Tensor out;
  int rows, heads;
};
Queries queries_of(PyObject* q_arg, PyObject* out_arg, PyObject* index_arg, const char* index_name, int dim) {
  const at::Tensor &q = tensor(q_arg, "q"), &index = tensor(index_arg, index_name);
  need(q, "q", at::kBFloat16);
  need(index, index_name, at::kInt);
  if (q.dim() != 3 || q.size(2) != dim) refuse("q must be [rows, heads, " + std::to_string(dim) + "], got " + shape_of(q));
  Queries r{q, index, {}, narrow(q.size(0), "rows"), narrow(q.size(1), "heads")};
  if (out_arg != Py_None) {
    r.out = tensor(out_arg, "out");
    need(r.out, "out", at::kBFloat16);
    if (r.out.sizes() != q.sizes()) refuse("out does not match q");
  }
  return r;
}
// The workspace of an attention call.  Without one of the caller's it is made here, all of it uninitialised but the status word, which takes what the
// caller's status word says and is handed back to it (done): findings of such a call are not lost with its workspace.
struct Workspace {
  at::Tensor all, word, status;
  Workspace(PyObject* o, PyObject* status_arg, size_t (*bytes)(int, int, int, int, int, int), const int (&a)[6], const at::Tensor& q) {
    void* at = status_word(status_arg, q.get_device());
    if (o != Py_None) {
      if (at != nullptr) refuse("a call with a workspace records findings in its first word: status goes with workspace=None");
      all = tensor(o, "workspace");
      need(all, "workspace", at::kByte);
      device_of({&q, &all});
      return;
    }
    all = at::empty({static_cast<int64_t>(bytes(a[0], a[1], a[2], a[3], a[4], a[5]))}, q.options().dtype(at::kByte));
    word = all.narrow(0, 0, 4);
    if (at == nullptr) {
      word.zero_();
    } else {
      status = at::from_blob(at, {4}, word.options());
      word.copy_(status);
    }
  }
  void done() {
    if (status.defined()) status.copy_(word);
  }
};
size_t prefill_bytes(int tokens, int first, int hq, int hkv, int dim, int) { return p_prefill_bytes(tokens, first, hq, hkv, dim); }

// Turns what a body throws into Python errors.
template <typename F>
PyObject* guarded(Py_ssize_t given, Py_ssize_t wanted, F&& body) {
  HANDLE_TH_ERRORS
  try {
    if (given != wanted) refuse("expected " + std::to_string(wanted) + " arguments");
    return body();
  } catch (const Refused& e) {
    PyErr_SetString(PyExc_ValueError, e.what());
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

// (ctx_lens, new_lens, block_table, supply, supply_used, num_rows, num_blocks, status) -> six tensors
PyObject* slot_map(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(n, 8, [&]() -> PyObject* {
    const at::Tensor &ctx = tensor(args[0], "ctx_lens"), &fresh = tensor(args[1], "new_lens"), &table = tensor(args[2], "block_table"),
                     &supply = tensor(args[3], "supply"), &used = tensor(args[4], "supply_used");
    need(ctx, "ctx_lens", at::kInt);
    need(fresh, "new_lens", at::kInt);
    need(table, "block_table", at::kInt);
    need(supply, "supply", at::kInt);
    need(used, "supply_used", at::kInt);
    const int device = device_of({&ctx, &fresh, &table, &supply, &used});
    void* status = status_word(args[7], device);
    if (table.dim() != 2 || ctx.dim() != 1 || ctx.size(0) != table.size(0) || fresh.sizes() != ctx.sizes() || used.numel() != 1)
      refuse("lengths, block table or supply_used do not match");
    const int B = narrow(ctx.size(0), "sequences"), R = whole(args[5]), blocks = whole(args[6]);
    const int pages = narrow(supply.numel(), "supply"), width = narrow(table.size(1), "block table");
    if (R < 0) refuse(std::to_string(R) + " rows");
    // one allocation; every output is a part of it
    const int64_t sizes[6] = {B, B + int64_t(1), R, R, R, 1};
    at::Tensor all = fresh_tensor({2 * int64_t(B) + 2 + 3 * int64_t(R)}, ctx);
    int32_t* at[6];
    int32_t* next = all.data_ptr<int32_t>();
    for (int i = 0; i < 6; ++i) {
      at[i] = next;
      next += sizes[i];
    }
    const int rc = without_gil([&] {
      return p_slot_map(ctx.data_ptr<int32_t>(), fresh.data_ptr<int32_t>(), table.data_ptr<int32_t>(), supply.data_ptr<int32_t>(),
                        used.data_ptr<int32_t>(), pages, at[0], at[1], at[2], at[3], at[4], at[5], status, B, R, blocks, width,
                        stream_of(device));
    });
    if (rc) return failed(rc, "b200_kv_slot_map");
    PyObject* result = PyTuple_New(6);
    if (result == nullptr) throw python_error();
    int64_t offset = 0;
    for (int i = 0; i < 6; ++i) {
      PyTuple_SET_ITEM(result, i, THPVariable_Wrap(part_of(all, offset, sizes[i])));
      offset += sizes[i];
    }
    return result;
  });
}

// (k_new, v_new, k_pool, v_pool, k_scale, v_scale, slots, status)
PyObject* append(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(n, 8, [&]() -> PyObject* {
    const Cache c = cache_of(args + 2);
    const at::Tensor &k = tensor(args[0], "k_new"), &v = tensor(args[1], "v_new"), &slots = tensor(args[6], "slots");
    need(slots, "slots", at::kInt);
    const at::ScalarType dtype = k.scalar_type();
    if ((dtype != at::kBFloat16 && dtype != at::kFloat) || v.scalar_type() != dtype)
      refuse(std::string("k_new and v_new must be bfloat16 or float32, got ") + c10::toString(dtype) + " and " + c10::toString(v.scalar_type()));
    const int64_t want[3] = {slots.numel(), c.heads, c.dim};
    if (k.sizes() != at::IntArrayRef(want, 3) || v.sizes() != k.sizes())
      refuse("k_new and v_new must be [" + std::to_string(want[0]) + ", " + std::to_string(c.heads) + ", " + std::to_string(c.dim) + "], got " + shape_of(k) +
             " and " + shape_of(v));
    const int device = device_of({&c.k, &c.v, &c.ks, &c.vs, &k, &v, &slots});
    void* status = status_word(args[7], device);
    const int R = narrow(want[0], "rows");
    if (R == 0) Py_RETURN_NONE;
    for (const at::Tensor* t : {&k, &v})
      if (!t->is_contiguous() && (t->stride(2) != 1 || (c.heads > 1 && t->stride(1) != c.dim) || (R > 1 && t->stride(0) < int64_t(c.heads) * c.dim)))
        refuse("k_new and v_new may be strided in their rows only");
    const int64_t row = int64_t(c.heads) * c.dim;  // the stride of a single row says nothing
    const int rc = without_gil([&] {
      return p_append(k.data_ptr(), v.data_ptr(), R > 1 ? k.stride(0) : row, R > 1 ? v.stride(0) : row, c.k.data_ptr(), c.v.data_ptr(), c.ks.data_ptr(), c.vs.data_ptr(),
                      slots.data_ptr<int32_t>(), status, R, c.heads, c.dim, c.blocks, dtype == at::kBFloat16 ? B200_DTYPE_BF16 : B200_DTYPE_F32,
                      stream_of(device));
    });
    if (rc) return failed(rc, "b200_kv8_append");
    Py_RETURN_NONE;
  });
}

// (q, k_pool, v_pool, k_scale, v_scale, block_table, ctx_lens, scale, split_tokens, workspace, out, status) -> out
PyObject* decode(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(n, 12, [&]() -> PyObject* {
    const Cache c = cache_of(args + 1);
    Queries x = queries_of(args[0], args[10], args[5], "block_table", c.dim);
    const at::Tensor& ctx = tensor(args[6], "ctx_lens");
    need(ctx, "ctx_lens", at::kInt);
    if (x.index.dim() != 2 || x.index.size(0) != x.rows || ctx.dim() != 1 || ctx.size(0) != x.rows) refuse("block_table / ctx_lens batch mismatch");
    const int device = device_of({&x.q, &c.k, &c.v, &c.ks, &c.vs, &x.index, &ctx, x.out.defined() ? &x.out : &x.q});
    const double scale = PyFloat_AsDouble(args[7]);
    if (scale == -1.0 && PyErr_Occurred()) throw python_error();
    const int split = whole(args[8]), width = narrow(x.index.size(1), "block table");
    if (!x.out.defined()) x.out = fresh_tensor(x.q.sizes(), x.q);
    if (x.rows > 0) {
      Workspace ws(args[9], args[11], p_decode_bytes, {x.rows, x.heads, c.heads, c.dim, width, split}, x.q);
      const int rc = without_gil([&] {
        return p_decode(x.q.data_ptr(), c.k.data_ptr(), c.v.data_ptr(), c.ks.data_ptr(), c.vs.data_ptr(), x.index.data_ptr<int32_t>(),
                        ctx.data_ptr<int32_t>(), x.out.data_ptr(), ws.all.data_ptr(), ws.all.nbytes(), x.rows, x.heads, c.heads, c.dim, c.blocks, width,
                        static_cast<float>(scale), split, stream_of(device));
      });
      if (rc) return failed(rc, "b200_kv8_attn_decode");
      ws.done();
    }
    return THPVariable_Wrap(x.out);
  });
}

// (q, k_pool, v_pool, k_scale, v_scale, table_row, first_pos, scale, workspace, out, status) -> out
PyObject* prefill(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(n, 11, [&]() -> PyObject* {
    const Cache c = cache_of(args + 1);
    Queries x = queries_of(args[0], args[9], args[5], "table_row", c.dim);
    if (x.index.dim() != 1) refuse("table_row must be one row of a block table");
    const int device = device_of({&x.q, &c.k, &c.v, &c.ks, &c.vs, &x.index, x.out.defined() ? &x.out : &x.q});
    const int first = whole(args[6]), width = narrow(x.index.numel(), "table row");
    const double scale = PyFloat_AsDouble(args[7]);
    if (scale == -1.0 && PyErr_Occurred()) throw python_error();
    if (!x.out.defined()) x.out = fresh_tensor(x.q.sizes(), x.q);
    if (x.rows > 0) {
      Workspace ws(args[8], args[10], prefill_bytes, {x.rows, first, x.heads, c.heads, c.dim, 0}, x.q);
      const int rc = without_gil([&] {
        return p_prefill(x.q.data_ptr(), c.k.data_ptr(), c.v.data_ptr(), c.ks.data_ptr(), c.vs.data_ptr(), x.index.data_ptr<int32_t>(),
                         x.out.data_ptr(), ws.all.data_ptr(), ws.all.nbytes(), x.rows, first, x.heads, c.heads, c.dim, c.blocks, width,
                         static_cast<float>(scale), stream_of(device));
      });
      if (rc) return failed(rc, "b200_kv8_attn_prefill");
      ws.done();
    }
    return THPVariable_Wrap(x.out);
  });
}

// (check, addresses of the six entry points in the order above)
PyObject* bind(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(n, 7, [&]() -> PyObject* {
    void* at[6];
    for (int i = 0; i < 6; ++i) {
      at[i] = PyLong_AsVoidPtr(args[1 + i]);
      if (at[i] == nullptr) {
        if (PyErr_Occurred()) throw python_error();
        refuse("an entry point is null");
      }
    }
    p_slot_map = reinterpret_cast<decltype(p_slot_map)>(at[0]);
    p_append = reinterpret_cast<decltype(p_append)>(at[1]);
    p_decode_bytes = reinterpret_cast<decltype(p_decode_bytes)>(at[2]);
    p_decode = reinterpret_cast<decltype(p_decode)>(at[3]);
    p_prefill_bytes = reinterpret_cast<decltype(p_prefill_bytes)>(at[4]);
    p_prefill = reinterpret_cast<decltype(p_prefill)>(at[5]);
    Py_INCREF(args[0]);
    Py_XSETREF(p_check, args[0]);
    Py_RETURN_NONE;
  });
}

#define B200_METHOD(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {B200_METHOD(bind), B200_METHOD(slot_map), B200_METHOD(append), B200_METHOD(decode), B200_METHOD(prefill), {}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_kv8", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__kv8() { return PyModule_Create(&module); }
