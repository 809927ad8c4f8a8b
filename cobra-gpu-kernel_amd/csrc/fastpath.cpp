// Native steady-state calls of CobraAttentionSublayer.forward (cobra_amd/layer.py),
// of CobraTransformer.forward in its one-kernel-per-block mode (cobra_amd/model.py) and
// of the key/value cache's operators (cobra_amd/ops.py).
//
// At the small shapes one sublayer forward is a single ~7 us kernel, and the Python
// around its launch (signature and parameter-version checks, the output allocation,
// the ctypes call) took about as long as the kernel, so back-to-back forwards were
// bound by the host.  BoundForward holds one bound launch (cobra_layer_bind) and does
// those steps in C++: for an input of the bound signature, with the module's
// parameters and LayerNorm epsilon unchanged since the bind, it allocates y with the
// caching allocator, launches on the device's current stream and returns y; for any
// other call it returns None and the module takes its general path.  It never
// computes anything itself: the launch is the library's (libcobra_amd.so).
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/extension.h>

#include <ATen/hip/EmptyTensor.h>
#include <c10/hip/HIPStream.h>

#include <string>
#include <utility>
#include <vector>

#include "cobra_amd.h"

namespace {

class BoundForward {
 public:
  // handle: a cobra_layer_launch* from cobra_layer_bind (owned by the caller, which
  // keeps it and every buffer it names alive as long as this object).  like: an input
  // of the bound signature.  params / snapshot: the tensors the bound weights were
  // packed from, and for each its version counter (or, for an inference tensor, which
  // keeps none, its data pointer) at packing time.  norm: the module whose `eps`
  // attribute was bound (its value must still equal eps).  masked: the launch was bound
  // with a token mask, which every call must then pass ([B, S] bool or uint8 on the
  // device, 0 = padded), and a call without one must not.  on_error(name, code) raises
  // the library's error.
  BoundForward(int64_t handle, const at::Tensor& like, std::vector<at::Tensor> params,
               std::vector<int64_t> snapshot, py::object norm, double eps, bool masked, py::object on_error)
      : handle_(reinterpret_cast<const cobra_layer_launch*>(handle)),
        sizes_(like.sizes().vec()),
        dtype_(like.scalar_type()),
        device_(like.device()),
        params_(std::move(params)),
        snapshot_(std::move(snapshot)),
        norm_(std::move(norm)),
        eps_(eps),
        masked_(masked),
        on_error_(std::move(on_error)) {
    TORCH_CHECK(handle_ != nullptr, "BoundForward: null launch handle");
    TORCH_CHECK(params_.size() == snapshot_.size(), "BoundForward: one snapshot value per parameter");
    TORCH_CHECK(device_.is_cuda(), "BoundForward: the bound input must be a device tensor");
  }

  py::object call(const at::Tensor& x, const c10::optional<at::Tensor>& mask) const {
    if (!x.defined() || x.device() != device_ || x.scalar_type() != dtype_ || x.sizes() != sizes_ ||
        !x.is_contiguous())
      return py::none();
    const uint8_t* m = nullptr;
    if (mask.has_value() != masked_) return py::none();
    if (masked_) {
      const at::Tensor& t = *mask;
      if (!t.defined() || t.device() != device_ || (t.scalar_type() != at::kBool && t.scalar_type() != at::kByte) ||
          t.dim() != 2 || t.size(0) != sizes_[0] || t.size(1) != sizes_[1] || !t.is_contiguous())
        return py::none();
      m = static_cast<const uint8_t*>(t.data_ptr());
    }
    for (size_t i = 0; i < params_.size(); ++i) {
      const at::Tensor& p = params_[i];
      const int64_t now = p.is_inference() ? reinterpret_cast<int64_t>(p.data_ptr()) : p._version();
      if (now != snapshot_[i]) return py::none();
    }
    if (norm_.attr("eps").cast<double>() != eps_) return py::none();
    // The device allocator directly (the caching allocator, as empty_like reaches it
    // after two dispatcher round trips); x is contiguous, so y has x's layout.
    at::Tensor y = at::detail::empty_cuda(sizes_, dtype_, device_, c10::nullopt);
    const hipStream_t s = c10::hip::getCurrentHIPStream(device_.index()).stream();
    const int code = cobra_layer_run(handle_, x.data_ptr(), m, y.data_ptr(), nullptr, s);
    if (code != 0) {
      on_error_("cobra_layer_run", code);  // raises
      throw std::runtime_error("cobra_layer_run failed");
    }
    return py::cast(std::move(y));
  }

 private:
  const cobra_layer_launch* handle_;
  std::vector<int64_t> sizes_;
  at::ScalarType dtype_;
  at::Device device_;
  std::vector<at::Tensor> params_;
  std::vector<int64_t> snapshot_;
  py::object norm_;
  double eps_;
  bool masked_;
  py::object on_error_;
};

// Steady state of CobraTransformer.forward (cobra_amd/model.py) where every block runs
// as one whole-block kernel: layer 0's norm1 (which also widens x into the fp32
// residual), then one cobra_block_fwd per block, h ping-ponging between two buffers and
// the residual updated in place, the last block writing final_norm's output.  Same
// contract as BoundForward: an input of the bound signature with the parameters and
// epsilon unchanged gets the output; any other call returns None.
class BoundStack {
 public:
  // blocks: per block, in order, w_qkv, b_qkv, w_o, b_o, ln2_w, ln2_b, w1, b1, w2, b2 and
  // the next norm's weight and bias (the next block's norm1, final_norm after the last).
  BoundStack(const at::Tensor& like, std::vector<at::Tensor> params, std::vector<int64_t> snapshot,
             py::object norm, double eps, at::Tensor ln1_w, at::Tensor ln1_b, std::vector<at::Tensor> blocks,
             int64_t heads, int64_t ffn_dim, bool causal, py::object on_error)
      : sizes_(like.sizes().vec()),
        dtype_(like.scalar_type()),
        device_(like.device()),
        params_(std::move(params)),
        snapshot_(std::move(snapshot)),
        norm_(std::move(norm)),
        eps_(eps),
        ln1_w_(std::move(ln1_w)),
        ln1_b_(std::move(ln1_b)),
        blocks_(std::move(blocks)),
        heads_(heads),
        ffn_dim_(ffn_dim),
        causal_(causal),
        on_error_(std::move(on_error)) {
    TORCH_CHECK(params_.size() == snapshot_.size(), "BoundStack: one snapshot value per parameter");
    TORCH_CHECK(device_.is_cuda() && sizes_.size() == 3, "BoundStack: the bound input must be a [B, S, D] device tensor");
    TORCH_CHECK(dtype_ == at::kHalf || dtype_ == at::kFloat, "BoundStack: fp16 or fp32 activations");
    TORCH_CHECK(!blocks_.empty() && blocks_.size() % kPerBlock == 0, "BoundStack: 12 tensors per block");
  }

  py::object call(const at::Tensor& x) const {
    if (!x.defined() || x.device() != device_ || x.scalar_type() != dtype_ || x.sizes() != sizes_ ||
        !x.is_contiguous())
      return py::none();
    for (size_t i = 0; i < params_.size(); ++i) {
      const at::Tensor& p = params_[i];
      const int64_t now = p.is_inference() ? reinterpret_cast<int64_t>(p.data_ptr()) : p._version();
      if (now != snapshot_[i]) return py::none();
    }
    if (norm_.attr("eps").cast<double>() != eps_) return py::none();
    const int64_t B = sizes_[0], S = sizes_[1], D = sizes_[2], T = B * S;
    const int xdt = dtype_ == at::kHalf ? COBRA_F16 : COBRA_F32;
    const float eps = static_cast<float>(eps_);
    const size_t n = blocks_.size() / kPerBlock;
    at::Tensor r = at::detail::empty_cuda({T, D}, at::kFloat, device_, c10::nullopt);
    at::Tensor h = at::detail::empty_cuda({T, D}, at::kHalf, device_, c10::nullopt);
    at::Tensor hn = n > 1 ? at::detail::empty_cuda({T, D}, at::kHalf, device_, c10::nullopt) : at::Tensor();
    at::Tensor out = at::detail::empty_cuda(sizes_, dtype_, device_, c10::nullopt);
    const hipStream_t s = c10::hip::getCurrentHIPStream(device_.index()).stream();
    check("cobra_ln_fwd", cobra_ln_fwd(x.data_ptr(), xdt, nullptr, 0, ln1_w_.data_ptr<float>(),
                                       ln1_b_.data_ptr<float>(), nullptr, 0, r.data_ptr<float>(), h.data_ptr(),
                                       COBRA_F16, T, D, eps, s));
    for (size_t i = 0; i < n; ++i) {
      const at::Tensor* b = &blocks_[kPerBlock * i];
      const bool last = i + 1 == n;
      void* o = last ? out.data_ptr() : hn.data_ptr();
      check("cobra_block_fwd",
            cobra_block_fwd(h.data_ptr(), r.data_ptr<float>(), nullptr, b[0].data_ptr(), b[1].data_ptr<float>(),
                            b[2].data_ptr(), b[3].data_ptr<float>(), b[4].data_ptr<float>(), b[5].data_ptr<float>(),
                            b[6].data_ptr(), b[7].data_ptr<float>(), b[8].data_ptr(), b[9].data_ptr<float>(),
                            b[10].data_ptr<float>(), b[11].data_ptr<float>(), r.data_ptr<float>(), o,
                            last ? xdt : COBRA_F16, 0, B, S, D, heads_, ffn_dim_, causal_ ? 1 : 0, eps, s));
      if (!last) std::swap(h, hn);
    }
    return py::cast(std::move(out));
  }

 private:
  static constexpr size_t kPerBlock = 12;

  void check(const char* fn, int code) const {
    if (code != 0) {
      on_error_(fn, code);  // raises
      throw std::runtime_error(std::string(fn) + " failed");
    }
  }

  std::vector<int64_t> sizes_;
  at::ScalarType dtype_;
  at::Device device_;
  std::vector<at::Tensor> params_;
  std::vector<int64_t> snapshot_;
  py::object norm_;
  double eps_;
  at::Tensor ln1_w_, ln1_b_;
  std::vector<at::Tensor> blocks_;
  int64_t heads_, ffn_dim_;
  bool causal_;
  py::object on_error_;
};

// -- key/value cache ------------------------------------------------------------------
//
// The calls of cobra_amd/ops.py's cache_* functions in C++: a decode step's kernels take a few
// microseconds each, about what the checks and allocations of one call take in Python.  Same
// contract as above: a call whose tensors are all as they should be, on the current device, is
// made here, once, and raises the library's error; for any other these return None before the
// library is asked, and Python's own checks name what is wrong (or make the call on another
// device).  Arguments come by position (the vector-call protocol);
// what is not of the expected Python type makes a call "any other" too.

bool py_int(PyObject* o, int64_t* v) {
  if (!PyLong_Check(o)) return false;
  *v = PyLong_AsLongLong(o);
  if (*v == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    return false;
  }
  return true;
}

// A dense tensor on device `dev` of type `dt`, or null.
const at::Tensor* dev_tensor(PyObject* o, int dev, at::ScalarType dt) {
  if (!THPVariable_Check(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.is_cuda() || t.device().index() != dev || t.scalar_type() != dt || !t.is_contiguous()) return nullptr;
  return &t;
}

bool shape_is(const at::Tensor* t, std::initializer_list<int64_t> want) {
  return t && t->sizes() == at::IntArrayRef(want);
}

at::Tensor new_tensor(at::IntArrayRef sizes, at::ScalarType dt, const at::Device& dev) {
  return at::detail::empty_cuda(sizes, dt, dev, c10::nullopt);
}

// The current device, if it is a tensor's.
int device_of(PyObject* o) {
  if (!THPVariable_Check(o)) return -1;
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.is_cuda()) return -1;
  const int dev = t.device().index();
  return dev == c10::hip::current_device() ? dev : -1;
}

// A call that is not made here.
PyObject* none() { Py_RETURN_NONE; }

// A call that failed: it may have changed something (a reserve is two launches), so it is not
// left to the general path to be made again.
void check(const char* fn, int code) {
  if (code == 0) return;
  py::module_::import("cobra_amd._lib").attr("check")(fn, code);  // raises
  throw std::runtime_error(std::string(fn) + " failed");
}

bool block_ok(int64_t n) { return n == 16 || n == 32 || n == 64 || n == 128; }

// Exceptions as torch raises them (out of memory is its own type).
template <typename F>
PyObject* guarded(F&& f) {
  HANDLE_TH_ERRORS
  return f();
  END_HANDLE_TH_ERRORS
}

struct Tables {
  const at::Tensor *lens, *change, *table, *free_list, *count;
  int64_t batch, block;
  int dev;
  bool read(PyObject* const* a) {
    dev = device_of(a[0]);
    if (dev < 0) return false;
    lens = dev_tensor(a[0], dev, at::kInt);
    change = dev_tensor(a[1], dev, at::kInt);
    table = dev_tensor(a[2], dev, at::kInt);
    free_list = dev_tensor(a[3], dev, at::kInt);
    count = dev_tensor(a[4], dev, at::kInt);
    if (!lens || lens->dim() != 1 || !table || table->dim() != 2 || !free_list || free_list->dim() != 1) return false;
    batch = lens->size(0);
    return batch > 0 && shape_is(change, {batch}) && table->size(0) == batch && shape_is(count, {1}) &&
           py_int(a[5], &block) && block_ok(block);
  }
};

// (lens, new_lens, block_table, free_list, free_count, block_size, tokens) -> (slots, cu, missing) | None
PyObject* cache_reserve(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Tables t;
    int64_t tokens;
    if (n != 7 || !t.read(a) || !py_int(a[6], &tokens) || tokens < 0 || tokens > 0x7fffffff) return none();
    const at::Device dev = t.lens->device();
    at::Tensor slots = new_tensor({tokens}, at::kLong, dev), cu = new_tensor({t.batch + 1}, at::kInt, dev);
    at::Tensor missing = new_tensor({1}, at::kInt, dev), ws = new_tensor({t.batch + 1}, at::kInt, dev);
    const int code = cobra_cache_reserve(
        t.lens->data_ptr<int>(), t.change->data_ptr<int>(), t.table->data_ptr<int>(), t.table->size(1),
        t.free_list->data_ptr<int>(), t.free_list->size(0), t.count->data_ptr<int>(), slots.data_ptr<int64_t>(), tokens,
        cu.data_ptr<int>(), missing.data_ptr<int>(), ws.data_ptr<int>(), t.batch, t.block,
        c10::hip::getCurrentHIPStream(t.dev).stream());
    check("cobra_cache_reserve", code);
    PyObject* got = PyTuple_New(3);
    if (!got) return nullptr;
    PyTuple_SET_ITEM(got, 0, THPVariable_Wrap(std::move(slots)));
    PyTuple_SET_ITEM(got, 1, THPVariable_Wrap(std::move(cu)));
    PyTuple_SET_ITEM(got, 2, THPVariable_Wrap(std::move(missing)));
    return got;
  });
}

// (lens, keep_lens, block_table, free_list, free_count, block_size) -> refused | None
PyObject* cache_trim(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Tables t;
    if (n != 6 || !t.read(a)) return none();
    const at::Device dev = t.lens->device();
    at::Tensor refused = new_tensor({1}, at::kInt, dev), ws = new_tensor({t.batch}, at::kInt, dev);
    const int code = cobra_cache_trim(t.lens->data_ptr<int>(), t.change->data_ptr<int>(), t.table->data_ptr<int>(),
                                      t.table->size(1), t.free_list->data_ptr<int>(), t.free_list->size(0),
                                      t.count->data_ptr<int>(), refused.data_ptr<int>(), ws.data_ptr<int>(), t.batch,
                                      t.block, c10::hip::getCurrentHIPStream(t.dev).stream());
    check("cobra_cache_trim", code);
    return THPVariable_Wrap(std::move(refused));
  });
}

struct Pool {
  const at::Tensor *k, *v, *k_scale, *v_scale;
  int64_t blocks, kv_heads, block;
  int cache;
  bool read(PyObject* const* a, int dev, int64_t heads, int64_t head_dim) {
    if (!THPVariable_Check(a[0])) return false;
    const at::ScalarType dt = THPVariable_Unpack(a[0]).scalar_type();
    if (dt != at::kFloat8_e4m3fn && dt != at::kChar) return false;
    cache = dt == at::kChar ? COBRA_CACHE_I8 : COBRA_CACHE_E4M3;
    k = dev_tensor(a[0], dev, dt);
    v = dev_tensor(a[1], dev, dt);
    k_scale = dev_tensor(a[2], dev, at::kFloat);
    v_scale = dev_tensor(a[3], dev, at::kFloat);
    if (!k || k->dim() != 4) return false;
    blocks = k->size(0);
    kv_heads = k->size(1);
    block = k->size(2);
    const int64_t width = k->size(3);
    return block_ok(block) && width == cobra_cache_width(head_dim) &&
           shape_is(v, {blocks, kv_heads, width, block}) && shape_is(k_scale, {blocks, kv_heads}) &&
           shape_is(v_scale, {blocks, kv_heads}) && kv_heads > 0 && heads > 0 && heads % kv_heads == 0;
  }
};

// 16-bit activations on the current device, or null; dt: the C ABI's code.
const at::Tensor* rows16(PyObject* o, int* dt) {
  const int dev = device_of(o);
  if (dev < 0) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  if (t.dim() != 2 || !t.is_contiguous()) return nullptr;
  if (t.scalar_type() == at::kHalf)
    *dt = COBRA_F16;
  else if (t.scalar_type() == at::kBFloat16)
    *dt = COBRA_BF16;
  else
    return nullptr;
  return &t;
}

// (qkv, slots, heads, head_dim, k, v, k_scale, v_scale) -> True | None
PyObject* cache_append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    int dt;
    int64_t heads, hd;
    const at::Tensor* x = n == 8 ? rows16(a[0], &dt) : nullptr;
    if (!x || !py_int(a[2], &heads) || !py_int(a[3], &hd)) return none();
    const int dev = x->device().index();
    const at::Tensor* slots = dev_tensor(a[1], dev, at::kLong);
    Pool p;
    if (!slots || !p.read(a + 4, dev, heads, hd) || !shape_is(slots, {x->size(0)}) ||
        x->size(1) != (heads + 2 * p.kv_heads) * hd)
      return none();
    const int code = cobra_cache_append(x->data_ptr(), dt, x->size(1), slots->data_ptr<int64_t>(), p.k->data_ptr(),
                                        p.v->data_ptr(), p.k_scale->data_ptr<float>(), p.v_scale->data_ptr<float>(),
                                        p.cache, x->size(0), p.blocks, p.block, heads, p.kv_heads, hd,
                                        c10::hip::getCurrentHIPStream(dev).stream());
    check("cobra_cache_append", code);
    Py_RETURN_TRUE;
  });
}

// (q, cu, lens, block_table, heads, head_dim, scale, k, v, k_scale, v_scale, causal, max_new | None,
// max_len | None, out | None) -> ctx | None
PyObject* cache_attn(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    int dt;
    int64_t heads, hd;
    const at::Tensor* q = n == 15 ? rows16(a[0], &dt) : nullptr;
    if (!q || !py_int(a[4], &heads) || !py_int(a[5], &hd) || !PyFloat_Check(a[6])) return none();
    const int dev = q->device().index();
    const at::Tensor *cu = dev_tensor(a[1], dev, at::kInt), *lens = dev_tensor(a[2], dev, at::kInt),
                     *table = dev_tensor(a[3], dev, at::kInt);
    Pool p;
    if (!cu || !lens || !table || !p.read(a + 7, dev, heads, hd) || lens->dim() != 1 || table->dim() != 2) return none();
    const int64_t T = q->size(0), B = lens->size(0), W = table->size(1);
    if (!PyBool_Check(a[11]) || T == 0 || B == 0 || W == 0 || p.blocks == 0 || !shape_is(cu, {B + 1}) ||
        table->size(0) != B || q->size(1) < heads * hd || q->size(1) % 8 || !(PyFloat_AS_DOUBLE(a[6]) > 0.0))
      return none();
    int64_t new_most = T - B + 1, len_most = W * p.block;
    if (a[12] != Py_None && !py_int(a[12], &new_most)) return none();
    if (a[13] != Py_None && !py_int(a[13], &len_most)) return none();
    if (new_most < 1) new_most = 1;
    if (len_most < 1) len_most = 1;
    at::Tensor out;
    if (a[14] == Py_None) {
      out = new_tensor({T, heads * hd}, q->scalar_type(), q->device());
    } else {
      const at::Tensor* o = dev_tensor(a[14], dev, q->scalar_type());
      if (!shape_is(o, {T, heads * hd})) return none();
      out = *o;
    }
    const int64_t need = cobra_cache_attn_workspace_bytes(T, B, heads, p.kv_heads, hd, new_most, len_most);
    if (need < 0) return none();
    at::Tensor ws;
    if (need > 0) ws = new_tensor({need}, at::kByte, q->device());
    const int code = cobra_cache_attn_fwd(
        q->data_ptr(), dt, q->size(1), cu->data_ptr<int>(), lens->data_ptr<int>(), table->data_ptr<int>(), W,
        p.k->data_ptr(), p.v->data_ptr(), p.k_scale->data_ptr<float>(), p.v_scale->data_ptr<float>(), p.cache,
        out.data_ptr(), need > 0 ? ws.data_ptr() : nullptr, need, T, B, p.blocks, p.block, heads, p.kv_heads, hd,
        new_most, len_most, static_cast<float>(PyFloat_AS_DOUBLE(a[6])), a[11] == Py_True ? 1 : 0,
        c10::hip::getCurrentHIPStream(dev).stream());
    check("cobra_cache_attn_fwd", code);
    if (a[14] != Py_None) {
      Py_INCREF(a[14]);
      return a[14];
    }
    return THPVariable_Wrap(std::move(out));
  });
}

PyMethodDef kCacheCalls[] = {
    {"cache_reserve", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(cache_reserve)), METH_FASTCALL, nullptr},
    {"cache_trim", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(cache_trim)), METH_FASTCALL, nullptr},
    {"cache_append", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(cache_append)), METH_FASTCALL, nullptr},
    {"cache_attn", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(cache_attn)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  PyModule_AddFunctions(m.ptr(), kCacheCalls);
  m.doc() = "Native steady-state forward of the cobra_amd attention sublayer";
  py::class_<BoundForward>(m, "BoundForward")
      .def(py::init<int64_t, const at::Tensor&, std::vector<at::Tensor>, std::vector<int64_t>, py::object, double,
                    bool, py::object>())
      .def("__call__", &BoundForward::call, py::arg("x"), py::arg("mask") = py::none());
  py::class_<BoundStack>(m, "BoundStack")
      .def(py::init<const at::Tensor&, std::vector<at::Tensor>, std::vector<int64_t>, py::object, double, at::Tensor,
                    at::Tensor, std::vector<at::Tensor>, int64_t, int64_t, bool, py::object>())
      .def("__call__", &BoundStack::call);
}
