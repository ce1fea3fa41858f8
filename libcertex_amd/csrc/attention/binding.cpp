// Python binding of the attention operators over their C API (certex_attention.h).
//
// A decoding step calls operators whose kernels take a few microseconds each; their arguments are up to nine
// tensors. Checking and describing those in Python and calling through ctypes took longer than the kernels, so this
// extension does it: it checks, allocates outputs and workspaces from torch, and calls the C entry points on torch's
// current stream with resources of that stream that all threads share. The rotation's gradient is here too, so that
// a backward pass does not wait for the interpreter.
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/ops/empty.h>
#include <ATen/ops/empty_like.h>
#include <c10/hip/HIPStream.h>

#include <cuvs/neighbors/certex_attention.h>

#include <map>
#include <mutex>
#include <optional>
#include <string>

namespace {

using at::Tensor;
using maybe = std::optional<Tensor>;

/** An argument that is refused (a ValueError), and an error of the device (the package's CertexError). */
struct refusal : std::runtime_error {
  using std::runtime_error::runtime_error;
};
struct device_error : std::runtime_error {
  using std::runtime_error::runtime_error;
};
/** A Python error that is already set. */
struct python_error {};

#define EXPECTS(ok, message)              \
  do {                                    \
    if (!(ok)) { throw refusal(message); } \
  } while (0)

PyObject* g_device_error  = nullptr;  // CertexError
PyObject* g_out_of_memory = nullptr;  // torch.OutOfMemoryError

/** Raises the C API's last error, of the kind that ctypes callers raise (_capi.check). */
void check(cuvsError_t status)
{
  if (status == CUVS_SUCCESS) { return; }
  const char* text      = cuvsGetLastErrorText();
  const std::string all = text != nullptr ? text : "unknown error";
  if (all.find("HIP error") != std::string::npos || all.find("out of memory") != std::string::npos) {
    throw device_error(all);
  }
  throw refusal(all);
}

/** The resources of torch's current stream: made once per stream, which allocates nothing, and shared by all threads
 *  (the calls here only queue kernels on it). */
auto resources() -> cuvsResources_t
{
  static std::mutex mutex;
  static auto* made = new std::map<std::pair<int, void*>, cuvsResources_t>();  // never destroyed
  const auto stream = c10::hip::getCurrentHIPStream();
  const std::pair<int, void*> key{int(stream.device_index()), stream.stream()};
  std::lock_guard lk(mutex);
  auto it = made->find(key);
  if (it == made->end()) {
    cuvsResources_t res = 0;
    check(cuvsResourcesCreateOnStream(&res, key.second));
    it = made->emplace(key, res).first;
  }
  return it->second;
}

/** "torch.float32" */
auto name_of(at::ScalarType t) -> std::string
{
  switch (t) {
    case at::kFloat: return "torch.float32";
    case at::kHalf: return "torch.float16";
    case at::kBFloat16: return "torch.bfloat16";
    case at::kDouble: return "torch.float64";
    case at::kInt: return "torch.int32";
    case at::kLong: return "torch.int64";
    default: return std::string("torch.") + c10::toString(t);
  }
}

auto shape_of(at::IntArrayRef s) -> std::string
{
  std::string text = "(";
  for (size_t i = 0; i < s.size(); ++i) { text += (i > 0 ? ", " : "") + std::to_string(s[i]); }
  return text + (s.size() == 1 ? ",)" : ")");
}

/** The borrowed DLPack form of a tensor, for the time of a call. */
struct view {
  DLManagedTensor m{};
  view() = default;
  explicit view(Tensor const& t)
  {
    DLTensor& l = m.dl_tensor;
    switch (t.scalar_type()) {
      case at::kFloat: l.dtype = {kDLFloat, 32, 1}; break;
      case at::kHalf: l.dtype = {kDLFloat, 16, 1}; break;
      case at::kBFloat16: l.dtype = {kDLBfloat, 16, 1}; break;
      case at::kInt: l.dtype = {kDLInt, 32, 1}; break;
      case at::kLong: l.dtype = {kDLInt, 64, 1}; break;
      case at::kByte: l.dtype = {kDLUInt, 8, 1}; break;
      default: throw refusal("unsupported element type " + name_of(t.scalar_type()));
    }
    l.data    = t.data_ptr();
    l.device  = {t.is_cuda() ? kDLROCM : kDLCPU, t.is_cuda() ? int32_t(t.get_device()) : 0};
    l.ndim    = int32_t(t.dim());
    l.shape   = const_cast<int64_t*>(t.sizes().data());
    l.strides = const_cast<int64_t*>(t.strides().data());
  }
  explicit view(maybe const& t)
  {
    if (t) { *this = view(*t); }
  }
  /** NULL for no tensor. */
  auto operator&() -> DLManagedTensor* { return m.dl_tensor.dtype.lanes != 0 ? &m : nullptr; }
};

/** A row tensor on the GPU of one of the element types (of `like`'s, if given). */
auto rows(Tensor const& t, const char* what, int ndim, Tensor const* like = nullptr) -> Tensor const&
{
  const std::string name = what;
  EXPECTS(t.is_cuda() && t.layout() == at::kStrided, name + " must be a GPU tensor");
  const auto type = t.scalar_type();
  if (like == nullptr) {
    EXPECTS(type == at::kFloat || type == at::kHalf || type == at::kBFloat16,
            name + " must be float32, float16 or bfloat16, not " + name_of(type));
  } else {
    EXPECTS(type == like->scalar_type(),
            name + " must be " + name_of(like->scalar_type()) + " as the other tensors, not " + name_of(type));
  }
  EXPECTS(t.dim() == ndim,
          name + " must have " + std::to_string(ndim) + " dimensions, not shape " + shape_of(t.sizes()));
  return t;
}

/** A row tensor that is only read: one whose last dimension has gaps is copied. */
auto read(Tensor const& t, const char* what, int ndim, Tensor const* like = nullptr) -> Tensor
{
  rows(t, what, ndim, like);
  return t.stride(-1) == 1 || t.size(-1) <= 1 ? t : t.contiguous();
}

auto ints(Tensor const& t, const char* what, bool narrow = false) -> Tensor
{
  EXPECTS(t.is_cuda() && t.layout() == at::kStrided &&
            (t.scalar_type() == at::kInt || (!narrow && t.scalar_type() == at::kLong)),
          std::string(what) + " must be a GPU tensor of torch.int32" + (narrow ? "" : " or torch.int64"));
  EXPECTS(t.dim() <= 4, std::string(what) + " must have at most 4 dimensions, not shape " + shape_of(t.sizes()));
  return t.is_contiguous() ? t : t.contiguous();
}

/** The kernels read and write values alone: a tensor that carries a tangent of forward-mode differentiation is refused,
 *  or the result would pass for a constant. */
void no_tangent(std::initializer_list<Tensor const*> tensors)
{
  if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) { return; }
  for (Tensor const* t : tensors) {
    EXPECTS(t == nullptr || !t->_fw_grad(0).defined(), "this operator has no forward-mode derivative");
  }
}

void no_gradient(std::initializer_list<Tensor const*> tensors)
{
  no_tangent(tensors);
  if (!at::GradMode::is_enabled()) { return; }
  for (Tensor const* t : tensors) {
    EXPECTS(t == nullptr || !t->requires_grad(), "this operator has no gradient: call it under torch.no_grad()");
  }
}

/** Tells autograd that a call has written t through its address: a backward pass that saved t before raises, as after
 *  torch's in-place operators. (Tensors of inference mode are saved by none and have no version.) */
void wrote(Tensor const& t)
{
  if (!t.is_inference()) { t.unsafeGetTensorImpl()->bump_version(); }
}

/** Workspace of a call (none where it needs none). */
auto workspace(int64_t bytes, Tensor const& like) -> maybe
{
  if (bytes == 0) { return std::nullopt; }
  return at::empty({bytes}, like.options().dtype(at::kByte));
}

// ---- rotation ----

/** A rotation's frequencies on one GPU, freed with the last user: the Rotary, or a graph that awaits its backward. */
struct rotary : torch::CustomClassHolder {
  cuvsCertexRotary_t handle;
  explicit rotary(cuvsCertexRotary_t h) : handle(h) {}
  ~rotary() override { (void)cuvsCertexRotaryDestroy(handle); }
};
using rotary_ptr = c10::intrusive_ptr<rotary>;

auto turned(Tensor const& x_, Tensor const& positions_, rotary_ptr const& r, bool transpose, maybe const& out) -> Tensor
{
  no_tangent({&x_, out ? &*out : nullptr});
  const Tensor x = read(x_, "x", int(x_.dim())), positions = ints(positions_, "positions");
  EXPECTS(positions.sizes() == x.sizes().slice(0, x.dim() - 2),
          "positions must have shape " + shape_of(x.sizes().slice(0, x.dim() - 2)) + ", one entry per token");
  Tensor y;
  if (out) {
    y = rows(*out, "out", int(x.dim()), &x);
    EXPECTS(y.sizes() == x.sizes(), "out must have the shape of x");
  } else {
    y = at::empty_like(x);
    if (y.stride(-1) != 1) { y = at::empty(x.sizes(), x.options()); }  // dense in another order of dimensions
  }
  view xv(x), pv(positions), yv(y);
  check(cuvsCertexRotate(resources(), r->handle, &xv, &pv, &yv, transpose));
  if (out) { wrote(y); }
  return y;
}

/** The rotation is linear, and its matrix over the magnitude orthogonal: the gradient is the transposed rotation of the
 *  output's gradient. */
struct rotation : torch::autograd::Function<rotation> {
  static Tensor forward(torch::autograd::AutogradContext* ctx, Tensor const& x, Tensor const& positions, rotary_ptr r,
                        bool transpose)
  {
    ctx->save_for_backward({positions});
    ctx->saved_data["transpose"] = transpose;
    ctx->saved_data["rotary"]    = c10::IValue::make_capsule(r);
    return turned(x, positions, r, transpose, std::nullopt);
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list dy)
  {
    const bool transpose   = !ctx->saved_data["transpose"].toBool();
    const auto r           = c10::static_intrusive_pointer_cast<rotary>(ctx->saved_data["rotary"].toCapsule());
    const Tensor positions = ctx->get_saved_variables()[0];
    // with a gradient of the gradient, or without
    Tensor dx = at::GradMode::is_enabled() ? apply(dy[0], positions, r, transpose)
                                           : turned(dy[0], positions, r, transpose, std::nullopt);
    return {dx, Tensor(), Tensor(), Tensor()};
  }
};

constexpr const char* kCapsule = "libcertex_amd.rotary";

void free_capsule(PyObject* c) { delete static_cast<rotary_ptr*>(PyCapsule_GetPointer(c, kCapsule)); }

auto rotary_of(PyObject* o) -> rotary_ptr
{
  auto* p = static_cast<rotary_ptr*>(PyCapsule_GetPointer(o, kCapsule));
  if (p == nullptr) { throw python_error{}; }
  return *p;
}

// ---- Python ----

auto tensor(PyObject* o, const char* what) -> Tensor const&
{
  EXPECTS(THPVariable_Check(o), std::string(what) + " must be a GPU tensor");
  return THPVariable_Unpack(o);
}

auto maybe_tensor(PyObject* o, const char* what) -> maybe
{
  if (o == Py_None) { return std::nullopt; }
  return tensor(o, what);
}

auto wrap(Tensor const& t) -> PyObject*
{
  PyObject* o = THPVariable_Wrap(t);
  if (o == nullptr) { throw python_error{}; }
  return o;
}

/** f(), its exceptions as Python's. */
template <typename F>
PyObject* guarded(F f)
{
  try {
    return f();
  } catch (python_error const&) {
  } catch (refusal const& e) {
    PyErr_SetString(PyExc_ValueError, e.what());
  } catch (device_error const& e) {
    PyErr_SetString(g_device_error, e.what());
  } catch (c10::OutOfMemoryError const& e) {
    PyErr_SetString(g_out_of_memory, e.what_without_backtrace());
  } catch (c10::Error const& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
  } catch (std::exception const& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}

bool counted(Py_ssize_t n, Py_ssize_t want)
{
  if (n == want) { return true; }
  PyErr_SetString(PyExc_TypeError, "wrong number of arguments");
  return false;
}

/** The interpreter lock, given up for the rest of a scope: allocations and launches may wait for others. */
struct unlocked {
  PyThreadState* state = PyEval_SaveThread();
  unlocked()           = default;
  unlocked(unlocked const&) = delete;
  unlocked& operator=(unlocked const&) = delete;
  ~unlocked() { PyEval_RestoreThread(state); }
};

/** (CertexError, torch.OutOfMemoryError) */
PyObject* init(PyObject*, PyObject* const* a, Py_ssize_t n)
{
  if (!counted(n, 2)) { return nullptr; }
  Py_INCREF(a[0]);
  Py_INCREF(a[1]);
  Py_XSETREF(g_device_error, a[0]);
  Py_XSETREF(g_out_of_memory, a[1]);
  Py_RETURN_NONE;
}

/** (handle of cuvsCertexRotaryCreate): a capsule that owns it. */
PyObject* own(PyObject*, PyObject* handle)
{
  const size_t h = PyLong_AsSize_t(handle);
  if (PyErr_Occurred()) { return nullptr; }
  auto* p     = new rotary_ptr(c10::make_intrusive<rotary>(h));
  PyObject* c = PyCapsule_New(p, kCapsule, free_capsule);
  if (c == nullptr) { delete p; }
  return c;
}

/** (capsule, head_dim, x, positions, transpose, out) */
PyObject* rotate(PyObject*, PyObject* const* a, Py_ssize_t n)
{
  if (!counted(n, 6)) { return nullptr; }
  return guarded([&] {
    const auto r          = rotary_of(a[0]);
    const int64_t dim     = PyLong_AsLongLong(a[1]);
    Tensor const& x       = tensor(a[2], "x");
    Tensor const& p       = tensor(a[3], "positions");
    const bool transpose  = PyObject_IsTrue(a[4]) == 1;
    const maybe out       = maybe_tensor(a[5], "out");
    EXPECTS((x.dim() == 3 || x.dim() == 4) && x.size(-1) == dim,
            "x must be a tensor (tokens, heads, " + std::to_string(dim) + ") or (batch, tokens, heads, " +
              std::to_string(dim) + ")");
    const bool differentiated = x.requires_grad() && at::GradMode::is_enabled();
    EXPECTS(!differentiated || !out, "a rotation that is differentiated takes no out");
    EXPECTS(!out || !out->requires_grad() || !at::GradMode::is_enabled(),
            "out must not require a gradient: call the rotation without it, or under torch.no_grad()");
    Tensor y;
    {
      unlocked u;
      y = differentiated ? rotation::apply(x, p, r, transpose) : turned(x, p, r, transpose, out);
    }
    return wrap(y);
  });
}

/** (capsule or None, head_dim, k, v, k_pages, v_pages, page_table, positions, sequences, q) */
PyObject* append(PyObject*, PyObject* const* a, Py_ssize_t n)
{
  if (!counted(n, 10)) { return nullptr; }
  return guarded([&]() -> PyObject* {
    const rotary_ptr r      = a[0] != Py_None ? rotary_of(a[0]) : rotary_ptr();
    const Tensor k          = read(tensor(a[2], "k"), "k", 3);
    const Tensor v          = read(tensor(a[3], "v"), "v", 3, &k);
    Tensor const& k_pages   = rows(tensor(a[4], "k_pages"), "k_pages", 4, &k);
    Tensor const& v_pages   = rows(tensor(a[5], "v_pages"), "v_pages", 4, &k);
    const Tensor table      = ints(tensor(a[6], "page_table"), "page_table", true);
    const Tensor positions  = ints(tensor(a[7], "positions"), "positions");
    maybe sequences = maybe_tensor(a[8], "sequences"), q = maybe_tensor(a[9], "q"), out;
    if (sequences) { sequences = ints(*sequences, "sequences"); }
    no_gradient({&k, &v, &k_pages, &v_pages, q ? &*q : nullptr});
    if (q) {
      q   = read(*q, "q", 3, &k);
      out = at::empty(q->sizes(), q->options());
    }
    if (r) {
      const int64_t dim = PyLong_AsLongLong(a[1]);
      EXPECTS(dim == k.size(-1), "this rotation is of heads of " + std::to_string(dim) + ", not " + std::to_string(k.size(-1)));
    }
    view kv(k), vv(v), kp(k_pages), vp(v_pages), tv(table), pv(positions), sv(sequences), qv(q), ov(out);
    {
      unlocked u;
      check(cuvsCertexAppendPages(resources(), r ? r->handle : 0, &kv, &vv, &kp, &vp, &tv, &pv, &sv, &qv, &ov));
      wrote(k_pages);
      wrote(v_pages);
    }
    if (!out) { Py_RETURN_NONE; }
    return wrap(*out);
  });
}

auto with_lse(Tensor const& out, maybe const& lse) -> PyObject*
{
  if (!lse) { return wrap(out); }
  PyObject* o = wrap(out);
  PyObject* l = THPVariable_Wrap(*lse);
  PyObject* t = l != nullptr ? PyTuple_Pack(2, o, l) : nullptr;
  Py_DECREF(o);
  Py_XDECREF(l);
  if (t == nullptr) { throw python_error{}; }
  return t;
}

/** (q, k_pages, v_pages, page_table, lengths, scale or None, window or None, return_lse) */
PyObject* attend(PyObject*, PyObject* const* a, Py_ssize_t n)
{
  if (!counted(n, 8)) { return nullptr; }
  return guarded([&] {
    const Tensor q        = read(tensor(a[0], "q"), "q", 3);
    Tensor const& k_pages = rows(tensor(a[1], "k_pages"), "k_pages", 4, &q);
    Tensor const& v_pages = rows(tensor(a[2], "v_pages"), "v_pages", 4, &q);
    no_gradient({&q, &k_pages, &v_pages});
    const Tensor table   = ints(tensor(a[3], "page_table"), "page_table", true);
    const Tensor lengths = ints(tensor(a[4], "lengths"), "lengths");
    const double scale   = a[5] != Py_None ? PyFloat_AsDouble(a[5]) : 1.0 / std::sqrt(double(q.size(2)));
    const int64_t window = a[6] != Py_None ? PyLong_AsLongLong(a[6]) : 0;
    if (PyErr_Occurred()) { throw python_error{}; }
    EXPECTS(a[6] == Py_None || window >= 1, "the window must be at least 1, not " + std::to_string(window));
    const bool want = PyObject_IsTrue(a[7]) == 1;
    Tensor out;
    maybe lse;
    {
      unlocked u;
      out = at::empty({q.size(0), q.size(1), v_pages.size(3)}, q.options());
      if (want) { lse = at::empty({q.size(0), q.size(1)}, q.options().dtype(at::kFloat)); }
      view qv(q), kv(k_pages), vv(v_pages), tv(table), lv(lengths), ov(out), ev(lse);
      int64_t bytes = 0;
      check(cuvsCertexPagedAttentionWorkspace(&qv, &kv, &vv, &tv, window, &bytes));
      const maybe work = workspace(bytes, q);
      view wv(work);
      check(cuvsCertexPagedAttention(resources(), &qv, &kv, &vv, &tv, &lv, float(scale), window, &wv, &ov, &ev));
    }
    return with_lse(out, lse);
  });
}

/** (scores, ids, values, scale, page_table or None, return_lse) */
PyObject* select(PyObject*, PyObject* const* a, Py_ssize_t n)
{
  if (!counted(n, 6)) { return nullptr; }
  return guarded([&] {
    Tensor scores = tensor(a[0], "scores"), ids = ints(tensor(a[1], "ids"), "ids");
    EXPECTS(scores.is_cuda() && scores.scalar_type() == at::kFloat, "scores must be a float32 GPU tensor");
    EXPECTS((scores.dim() == 2 || scores.dim() == 3) && scores.sizes() == ids.sizes(),
            "scores and ids must have one shape (n_heads, queries, k) or (n_heads, k), not " + shape_of(scores.sizes()) +
              " and " + shape_of(ids.sizes()));
    maybe table         = maybe_tensor(a[4], "page_table");
    const Tensor values = read(tensor(a[2], "values"), "values", table ? 4 : 3);
    no_gradient({&scores, &values});
    const double scale = PyFloat_AsDouble(a[3]);
    if (PyErr_Occurred()) { throw python_error{}; }
    if (table) {
      table = ints(*table, "page_table", true);
      EXPECTS(table->dim() == 1, "page_table must be one sequence's pages, of shape (n,)");
    }
    const bool single = scores.dim() == 2, want = PyObject_IsTrue(a[5]) == 1;
    Tensor out;
    maybe lse;
    {
      unlocked u;
      if (single) {
        scores = scores.unsqueeze(1);
        ids    = ids.unsqueeze(1);
      }
      if (!scores.is_contiguous()) { scores = scores.contiguous(); }
      out = at::empty({scores.size(0), scores.size(1), values.size(-1)}, values.options());
      if (want) { lse = at::empty({scores.size(0), scores.size(1)}, values.options().dtype(at::kFloat)); }
      view sv(scores), iv(ids), vv(values), tv(table), ov(out), ev(lse);
      int64_t bytes = 0;
      check(cuvsCertexSelectedAttentionWorkspace(&sv, &vv, &tv, &bytes));
      const maybe work = workspace(bytes, values);
      view wv(work);
      check(cuvsCertexSelectedAttention(resources(), &sv, &iv, &vv, &tv, float(scale), &wv, &ov, &ev));
      if (single) {
        out = out.select(1, 0);
        if (lse) { lse = lse->select(1, 0); }
      }
    }
    return with_lse(out, lse);
  });
}

/** (tensor): refuses one that is differentiated, for callers whose first step is not of this extension. */
PyObject* undifferentiated(PyObject*, PyObject* t)
{
  return guarded([&] {
    no_gradient({&tensor(t, "the tensor")});
    Py_INCREF(Py_None);
    return Py_None;
  });
}

template <typename F>
constexpr PyCFunction fast(F f)
{
  return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f));
}

PyMethodDef methods[] = {{"init", fast(init), METH_FASTCALL, "(CertexError, torch.OutOfMemoryError)"},
                         {"own", own, METH_O, "(rotary handle) -> capsule that owns it"},
                         {"rotate", fast(rotate), METH_FASTCALL, "(capsule, head_dim, x, positions, transpose, out)"},
                         {"append", fast(append), METH_FASTCALL,
                          "(capsule, head_dim, k, v, k_pages, v_pages, page_table, positions, sequences, q)"},
                         {"attend", fast(attend), METH_FASTCALL,
                          "(q, k_pages, v_pages, page_table, lengths, scale, window, return_lse)"},
                         {"select", fast(select), METH_FASTCALL, "(scores, ids, values, scale, page_table, return_lse)"},
                         {"undifferentiated", undifferentiated, METH_O, "(tensor): refuses one that is differentiated"},
                         {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_attention", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__attention() { return PyModule_Create(&module); }
