// Python binding of the decoding operators (decode.py) over the C ABI of w8a8_b200.h.
//
// A decode step makes many short calls: checking a dozen tensors and packing their pointers
// in Python costs more than the kernels run.  This module does what decode.py's functions
// promise (dtype, shape, layout and device checks, outputs and workspaces from torch's
// allocator, torch's current stream of the tensors' device) and calls the C ABI, whose entry
// points it takes from the loaded library; it holds no kernel and no state of its own.
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <dlfcn.h>
#include <torch/csrc/autograd/python_variable.h>

#include <set>
#include <stdexcept>
#include <string>
#include <vector>

#include "../../include/w8a8_b200.h"

namespace {

using at::Tensor;

// Entry points, resolved by bind().
decltype(&w8_attention_tree) fn_tree = nullptr;
decltype(&w8_attention_tree_workspace_bytes) fn_tree_ws = nullptr;
decltype(&w8_cache_append) fn_append = nullptr;
decltype(&w8_cache_evict) fn_evict = nullptr;
decltype(&w8_cache_evict_workspace_bytes) fn_evict_ws = nullptr;
decltype(&w8_beam_select) fn_select = nullptr;
decltype(&w8_beam_select_workspace_bytes) fn_select_ws = nullptr;
decltype(&w8_cache_reorder) fn_reorder = nullptr;
decltype(&w8_attention_paged) fn_paged = nullptr;
decltype(&w8_attention_paged_workspace_bytes) fn_paged_ws = nullptr;
decltype(&w8_paged_append) fn_paged_append = nullptr;
decltype(&w8_page_assign) fn_assign = nullptr;
decltype(&w8_page_assign_workspace_bytes) fn_assign_ws = nullptr;
decltype(&w8_draft_verify) fn_verify = nullptr;
PyObject* check_status = nullptr;  // _lib.check(status, name): raises

struct Refused : std::runtime_error {  // ValueError
  using std::runtime_error::runtime_error;
};
struct Raised {};  // a Python exception is set

// Pieces of a message, without iostreams (whose number formatting needs the locale of the one
// libstdc++ that every library of the process must then share).
std::string text(const char* s) { return s; }
std::string text(const std::string& s) { return s; }
std::string text(int64_t v) { return std::to_string(v); }
std::string text(at::ScalarType t) { return c10::toString(t); }
std::string text(const at::Device& d) { return d.str(); }
std::string text(at::IntArrayRef s) {
  std::string o = "(";
  for (size_t i = 0; i < s.size(); ++i) o += (i ? ", " : "") + std::to_string(s[i]);
  return o + (s.size() == 1 ? ",)" : ")");
}

template <typename... A>
[[noreturn]] void refuse(const A&... a) {
  throw Refused((text(a) + ...));
}
#define NEED(cond, ...)            \
  do {                             \
    if (!(cond)) refuse(__VA_ARGS__); \
  } while (0)

bool is_none(PyObject* o) { return o == nullptr || o == Py_None; }

const Tensor& tensor(PyObject* o, const char* name) {
  NEED(o != nullptr && THPVariable_Check(o), name, " must be a tensor");
  return THPVariable_Unpack(o);
}
const Tensor& cuda_tensor(PyObject* o, const char* name) {
  NEED(o != nullptr && THPVariable_Check(o) && THPVariable_Unpack(o).is_cuda(), name,
       " must be a CUDA tensor; there is no CPU path");
  return THPVariable_Unpack(o);
}
int64_t integer(PyObject* o, const char* name) {
  NEED(PyLong_Check(o), name, " must be an integer");
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    refuse(name, " is out of range");
  }
  return v;
}
double real(PyObject* o, const char* name) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) {
    PyErr_Clear();
    refuse(name, " must be a number");
  }
  return v;
}

void expect(const Tensor& t, const char* name, at::ScalarType dtype, at::Device dev) {
  NEED(t.scalar_type() == dtype, name, " must be ", dtype, " (got ", t.scalar_type(), ")");
  NEED(t.device() == dev, name, " must be on ", dev, " (got ", t.device(), ")");
}
void expect_shape(const Tensor& t, const char* name, at::IntArrayRef shape) {
  NEED(t.sizes() == shape, name, " must have shape ", text(shape), " (got ", text(t.sizes()), ")");
}
const Tensor& vector(PyObject* o, const char* name, at::IntArrayRef shape, at::ScalarType dtype, at::Device dev) {
  const Tensor& t = tensor(o, name);
  expect(t, name, dtype, dev);
  expect_shape(t, name, shape);
  NEED(t.is_contiguous(), name, " must be contiguous");
  return t;
}
void unit_last(const Tensor& t, const char* name) {
  const int64_t d = t.dim() - 1;
  NEED(t.stride(d) == 1 || t.size(d) <= 1, name, " must have unit stride along its last dimension");
}
// What is written must not overlap itself along its first n dimensions.
void disjoint(const Tensor& t, const char* name, int n) {
  for (int i = 0; i < n; ++i)
    NEED(t.size(i) <= 1 || t.stride(i) != 0, name, " is written and must not be an expanded view");
}
// [batch, kv_heads, n] per slot: its first two strides.
const Tensor& per_slot(PyObject* o, const char* name, at::IntArrayRef shape, at::ScalarType dtype, at::Device dev,
                       int64_t* strides) {
  const Tensor& t = tensor(o, name);
  expect(t, name, dtype, dev);
  expect_shape(t, name, shape);
  unit_last(t, name);
  strides[0] = t.stride(0), strides[1] = t.stride(1);
  return t;
}
// A 4-D tensor of rows: its other strides times `scale`.  The stride of a dimension of one
// element is arbitrary and never used: 0 satisfies every alignment rule.
const Tensor& rows4(PyObject* o, const char* name, at::ScalarType dtype, at::Device dev, int64_t* strides, int64_t scale) {
  NEED(o != nullptr && THPVariable_Check(o) && THPVariable_Unpack(o).dim() == 4, name, " must be a 4-D tensor");
  const Tensor& t = THPVariable_Unpack(o);
  expect(t, name, dtype, dev);
  unit_last(t, name);
  for (int i = 0; i < 3; ++i) strides[i] = t.size(i) > 1 ? t.stride(i) * scale : 0;
  return t;
}

Tensor make(at::IntArrayRef shape, at::ScalarType dtype, at::Device dev) {
  return at::detail::empty_cuda(shape, dtype, dev, std::nullopt);
}
Tensor workspace(int64_t bytes, at::Device dev) {  // (a negative size is a shape that the call refuses)
  return make({bytes > 0 ? bytes : 0}, at::kByte, dev);
}
w8_stream_t stream_of(at::Device dev) {
  return reinterpret_cast<w8_stream_t>(c10::cuda::getCurrentCUDAStream(dev.index()).stream());
}
void check(int status, const char* name) {
  if (status == W8_OK) return;
  PyObject* r = PyObject_CallFunction(check_status, "is", status, name);
  Py_XDECREF(r);
  if (PyErr_Occurred()) throw Raised();
  refuse(name, ": status ", static_cast<int64_t>(status));
}

int type_code(at::ScalarType t) {
  return t == at::kBFloat16 ? W8_BF16 : t == at::kHalf ? W8_FP16 : t == at::kFloat ? W8_FP32 : -1;
}

PyObject* tuple_of(std::initializer_list<PyObject*> items) {  // steals the references
  PyObject* t = PyTuple_New(static_cast<Py_ssize_t>(items.size()));
  Py_ssize_t i = 0;
  for (PyObject* o : items) PyTuple_SET_ITEM(t, i++, o);
  return t;
}
PyObject* wrap(const Tensor& t) { return THPVariable_Wrap(t); }
PyObject* same(PyObject* o) {
  Py_INCREF(o);
  return o;
}

#define ENTRY(count)                                                              \
  NEED(check_status != nullptr, "the binding is not bound to the library");       \
  NEED(nargs == (count), "wrong number of arguments");

// A drafted tree's mask and its tokens' depths, each for all sequences or one for each.
template <typename Args>
void tree_depth(PyObject* tree, PyObject* depth, Args& a, int64_t B, int64_t N, at::Device dev) {
  if (!is_none(tree)) {
    const Tensor& t = tensor(tree, "tree");
    NEED(t.dim() == 2 || t.dim() == 3, "tree must be [N, N] or [B, N, N]");
    expect(t, "tree", at::kBool, dev);
    if (t.dim() == 2)
      expect_shape(t, "tree", {N, N});
    else
      expect_shape(t, "tree", {B, N, N});
    unit_last(t, "tree");
    a.tree = static_cast<const uint8_t*>(t.const_data_ptr());
    a.tree_stride[0] = t.dim() == 3 ? t.stride(0) : 0;
    a.tree_stride[1] = t.stride(t.dim() - 2);
  }
  if (!is_none(depth)) {
    const Tensor& t = tensor(depth, "depth");
    NEED(t.dim() == 1 || t.dim() == 2, "depth must be [N] or [B, N]");
    expect(t, "depth", at::kInt, dev);
    if (t.dim() == 1)
      expect_shape(t, "depth", {N});
    else
      expect_shape(t, "depth", {B, N});
    unit_last(t, "depth");
    a.depth = t.const_data_ptr<int32_t>();
    a.depth_stride = t.dim() == 2 ? t.stride(0) : 0;
  }
}

// q, k, v, lens, k_new, v_new, tree, depth, window, scale, out, weights, weights_out, draft_weights
PyObject* attention_tree(PyObject* const* arg, Py_ssize_t nargs) {
  ENTRY(14)
  w8_attention_tree_args a = {};
  const Tensor& q = cuda_tensor(arg[0], "q");
  const at::Device dev = q.device();
  const at::ScalarType dt = q.scalar_type();
  NEED(dt == at::kBFloat16 || dt == at::kHalf, "q must be bfloat16 or float16 (got ", dt, ")");
  rows4(arg[0], "q", dt, dev, a.q_stride, 1);
  const Tensor& k = rows4(arg[1], "k", dt, dev, a.k_stride, 1);
  const Tensor& v = rows4(arg[2], "v", dt, dev, a.v_stride, 1);
  const Tensor& kn = rows4(arg[4], "k_new", dt, dev, a.k_new_stride, 1);
  const Tensor& vn = rows4(arg[5], "v_new", dt, dev, a.v_new_stride, 1);
  const int64_t B = q.size(0), H = q.size(1), N = q.size(2), D = q.size(3), KV = k.size(1), S = k.size(2);
  NEED(k.size(0) == B && k.size(3) == D && v.sizes() == k.sizes(), "k and v must be [B, KV, S, D] with q's B and D");
  const int64_t new_shape[4] = {B, KV, N, D};
  NEED(kn.sizes() == at::IntArrayRef(new_shape) && vn.sizes() == kn.sizes(), "k_new and v_new must be [B, KV, N, D]");
  NEED(KV >= 1 && H % KV == 0, "H = ", H, " must be a multiple of KV = ", KV);
  a.lens = vector(arg[3], "lens", {B}, at::kInt, dev).const_data_ptr<int32_t>();
  a.window = integer(arg[8], "window");
  a.scale = real(arg[9], "scale");
  tree_depth(arg[6], arg[7], a, B, N, dev);
  NEED(a.tree == nullptr || a.window == 0 || a.depth != nullptr || N == 0, "a tree with a window needs the tokens' depths");
  Tensor out;
  if (is_none(arg[10])) {
    out = make({B, H, N, D}, dt, dev);
    a.out_stride[0] = H * N * D, a.out_stride[1] = N * D, a.out_stride[2] = D;
  } else {
    out = rows4(arg[10], "out", dt, dev, a.out_stride, 1);
    expect_shape(out, "out", q.sizes());
    disjoint(out, "out", 3);
  }
  Tensor draft;
  PyObject* w_out = nullptr;
  if (!is_none(arg[11])) {
    const Tensor& w = per_slot(arg[11], "weights", {B, KV, S}, at::kFloat, dev, a.weights_stride);
    w_out = is_none(arg[12]) ? arg[11] : arg[12];
    const Tensor& to = per_slot(w_out, "weights_out", {B, KV, S}, at::kFloat, dev, a.weights_out_stride);
    disjoint(to, "weights_out", 2);
    draft = is_none(arg[13]) ? make({B, KV, N}, at::kFloat, dev) : vector(arg[13], "draft_weights", {B, KV, N}, at::kFloat, dev);
    a.weights = static_cast<const float*>(w.const_data_ptr());
    a.weights_out = static_cast<float*>(to.data_ptr());
    a.draft_weights = static_cast<float*>(draft.data_ptr());
  } else {
    NEED(is_none(arg[12]) && is_none(arg[13]), "weights_out and draft_weights go with weights");
  }
  a.q = q.const_data_ptr(), a.k = k.const_data_ptr(), a.v = v.const_data_ptr();
  a.k_new = kn.const_data_ptr(), a.v_new = vn.const_data_ptr(), a.out = out.data_ptr();
  a.batch = B, a.heads = H, a.kv_heads = KV, a.head_dim = D, a.slots = S, a.n_new = N, a.dtype = type_code(dt);
  {
    const c10::cuda::CUDAGuard guard(dev);
    const int64_t bytes = fn_tree_ws(B, H, KV, D, S, N, a.window, w_out != nullptr);
    const Tensor ws = workspace(bytes, dev);
    check(fn_tree(&a, ws.data_ptr(), ws.numel(), stream_of(dev)), "w8_attention_tree");
  }
  PyObject* o = is_none(arg[10]) ? wrap(out) : same(arg[10]);
  if (w_out == nullptr) return o;
  return tuple_of({o, same(w_out), is_none(arg[13]) ? wrap(draft) : same(arg[13])});
}

// k, v, k_new, v_new, lens, path, weights, draft_weights, positions, seen, lens_out
PyObject* cache_append(PyObject* const* arg, Py_ssize_t nargs) {
  ENTRY(11)
  w8_cache_append_args a = {};
  const Tensor& k = cuda_tensor(arg[0], "k");
  const at::Device dev = k.device();
  const at::ScalarType dt = k.scalar_type();
  const int64_t e = k.element_size();
  rows4(arg[0], "k", dt, dev, a.k_stride, e);
  const Tensor& v = rows4(arg[1], "v", dt, dev, a.v_stride, e);
  const Tensor& kn = rows4(arg[2], "k_new", dt, dev, a.k_new_stride, e);
  const Tensor& vn = rows4(arg[3], "v_new", dt, dev, a.v_new_stride, e);
  const int64_t B = k.size(0), KV = k.size(1), S = k.size(2), D = k.size(3), N = kn.size(2);
  NEED(v.sizes() == k.sizes(), "v must have the shape of k");
  const int64_t new_shape[4] = {B, KV, N, D};
  NEED(kn.sizes() == at::IntArrayRef(new_shape) && vn.sizes() == kn.sizes(), "k_new and v_new must be [B, KV, N, D]");
  disjoint(k, "k", 3);
  disjoint(v, "v", 3);
  a.lens = vector(arg[4], "lens", {B}, at::kInt, dev).const_data_ptr<int32_t>();
  a.steps = N;
  if (!is_none(arg[5])) {
    const Tensor& p = tensor(arg[5], "path");
    NEED(p.dim() == 2, "path must be [B, P]");
    expect(p, "path", at::kInt, dev);
    a.steps = p.size(1);
    expect_shape(p, "path", {B, a.steps});
    unit_last(p, "path");
    // An empty path is a path: nothing is appended and nothing of it is read.
    a.path = a.steps > 0 ? p.const_data_ptr<int32_t>() : a.lens;
    a.path_stride = p.stride(0);
  }
  if (!is_none(arg[6])) {
    const Tensor& w = per_slot(arg[6], "weights", {B, KV, S}, at::kFloat, dev, a.weights_stride);
    disjoint(w, "weights", 2);
    a.weights = static_cast<float*>(w.data_ptr());
    if (!is_none(arg[7]))
      a.draft_weights = static_cast<const float*>(
          per_slot(arg[7], "draft_weights", {B, KV, N}, at::kFloat, dev, a.draft_weights_stride).const_data_ptr());
  } else {
    NEED(is_none(arg[7]), "draft_weights go with weights");
  }
  if (!is_none(arg[8])) {
    NEED(!is_none(arg[9]), "positions go with seen");
    const Tensor& p = per_slot(arg[8], "positions", {B, KV, S}, at::kInt, dev, a.positions_stride);
    disjoint(p, "positions", 2);
    a.positions = p.data_ptr<int32_t>();
    a.seen = vector(arg[9], "seen", {B}, at::kInt, dev).const_data_ptr<int32_t>();
  }
  const Tensor to = is_none(arg[10]) ? make({B}, at::kInt, dev) : vector(arg[10], "lens_out", {B}, at::kInt, dev);
  a.k = k.data_ptr(), a.v = v.data_ptr(), a.k_new = kn.const_data_ptr(), a.v_new = vn.const_data_ptr();
  a.lens_out = to.data_ptr<int32_t>();
  a.batch = B, a.kv_heads = KV, a.slots = S, a.n_new = N, a.row_bytes = D * e;
  {
    const c10::cuda::CUDAGuard guard(dev);
    check(fn_append(&a, stream_of(dev)), "w8_cache_append");
  }
  return is_none(arg[10]) ? wrap(to) : same(arg[10]);
}

// k, v, weights, positions, lens, budget, sink, recent, weights_out, positions_out, lens_out
PyObject* cache_evict(PyObject* const* arg, Py_ssize_t nargs) {
  ENTRY(11)
  w8_cache_evict_args a = {};
  const Tensor& k = cuda_tensor(arg[0], "k");
  const at::Device dev = k.device();
  const int64_t e = k.element_size();
  rows4(arg[0], "k", k.scalar_type(), dev, a.k_stride, e);
  const Tensor& v = rows4(arg[1], "v", k.scalar_type(), dev, a.v_stride, e);
  const int64_t B = k.size(0), KV = k.size(1), S = k.size(2), D = k.size(3);
  NEED(v.sizes() == k.sizes(), "v must have the shape of k");
  disjoint(k, "k", 3);
  disjoint(v, "v", 3);
  a.lens = vector(arg[4], "lens", {B}, at::kInt, dev).const_data_ptr<int32_t>();
  a.weights = static_cast<const float*>(per_slot(arg[2], "weights", {B, KV, S}, at::kFloat, dev, a.weights_stride).const_data_ptr());
  a.positions = per_slot(arg[3], "positions", {B, KV, S}, at::kInt, dev, a.positions_stride).const_data_ptr<int32_t>();
  a.budget = integer(arg[5], "budget"), a.sink = integer(arg[6], "sink"), a.recent = integer(arg[7], "recent");
  Tensor w, p, l;
  if (is_none(arg[8])) {
    w = make({B, KV, S}, at::kFloat, dev);
    a.weights_out_stride[0] = KV * S, a.weights_out_stride[1] = S;
  } else {
    w = per_slot(arg[8], "weights_out", {B, KV, S}, at::kFloat, dev, a.weights_out_stride);
    disjoint(w, "weights_out", 2);
  }
  if (is_none(arg[9])) {
    p = make({B, KV, S}, at::kInt, dev);
    a.positions_out_stride[0] = KV * S, a.positions_out_stride[1] = S;
  } else {
    p = per_slot(arg[9], "positions_out", {B, KV, S}, at::kInt, dev, a.positions_out_stride);
    disjoint(p, "positions_out", 2);
  }
  l = is_none(arg[10]) ? make({B}, at::kInt, dev) : vector(arg[10], "lens_out", {B}, at::kInt, dev);
  a.k = k.data_ptr(), a.v = v.data_ptr();
  a.weights_out = static_cast<float*>(w.data_ptr()), a.positions_out = p.data_ptr<int32_t>(), a.lens_out = l.data_ptr<int32_t>();
  a.batch = B, a.kv_heads = KV, a.slots = S, a.row_bytes = D * e;
  {
    const c10::cuda::CUDAGuard guard(dev);
    const Tensor ws = workspace(fn_evict_ws(B, KV, S, a.budget), dev);
    check(fn_evict(&a, ws.data_ptr(), ws.numel(), stream_of(dev)), "w8_cache_evict");
  }
  return tuple_of({is_none(arg[8]) ? wrap(w) : same(arg[8]), is_none(arg[9]) ? wrap(p) : same(arg[9]),
                   is_none(arg[10]) ? wrap(l) : same(arg[10])});
}

// logits, scores, finished, pad, n, cap, order
PyObject* beam_select(PyObject* const* arg, Py_ssize_t nargs) {
  ENTRY(7)
  const Tensor& x = cuda_tensor(arg[0], "logits");
  const at::Device dev = x.device();
  const int dt = type_code(x.scalar_type());
  NEED(dt >= 0, "logits must be float32, bfloat16 or float16 (got ", x.scalar_type(), ")");
  NEED(x.dim() == 3, "logits must be [B, K, V]");
  const int64_t B = x.size(0), K = x.size(1), V = x.size(2);
  unit_last(x, "logits");
  const float* scores = static_cast<const float*>(vector(arg[1], "scores", {B, K}, at::kFloat, dev).const_data_ptr());
  const uint8_t* finished =
      is_none(arg[2]) ? nullptr
                      : static_cast<const uint8_t*>(vector(arg[2], "finished", {B, K}, at::kBool, dev).const_data_ptr());
  const int64_t pad = integer(arg[3], "pad"), n = is_none(arg[4]) ? K : integer(arg[4], "n");
  const double cap = is_none(arg[5]) ? 0.0 : real(arg[5], "cap");
  // (checked here too: a double outside fp32's range would become another cap)
  NEED(cap <= 0.0 || (cap >= 1e-30 && cap <= 1e30), "cap must be 0 (none) or between 1e-30 and 1e30");
  NEED(n >= 1, "n = ", n, " must be positive");
  const auto is = [&](const char* s) { return PyUnicode_Check(arg[6]) && PyUnicode_CompareWithASCIIString(arg[6], s) == 0; };
  const bool slot = is("slot");
  NEED(slot || is("score"), "order must be one of ('score', 'slot')");
  const Tensor out = make({B, n}, at::kFloat, dev), beam = make({B, n}, at::kLong, dev), token = make({B, n}, at::kLong, dev);
  if (B > 0) {
    const c10::cuda::CUDAGuard guard(dev);
    const Tensor ws = workspace(fn_select_ws(B, K, V, n), dev);
    check(fn_select(x.const_data_ptr(), dt, x.stride(0), x.stride(1), scores, finished, pad, cap > 0.0 ? static_cast<float>(cap) : 0.f, B, K,
                    V, n, slot, static_cast<float*>(out.data_ptr()), beam.data_ptr<int64_t>(), token.data_ptr<int64_t>(),
                    ws.data_ptr(), ws.numel(), stream_of(dev)),
          "w8_beam_select");
  }
  return tuple_of({wrap(out), wrap(beam), wrap(token)});
}

// caches (a sequence of tensors), beam, lens
PyObject* cache_reorder(PyObject* const* arg, Py_ssize_t nargs) {
  ENTRY(3)
  PyObject* seq = PySequence_Fast(arg[0], "caches must be a tensor or a sequence of tensors");
  if (seq == nullptr) throw Raised();
  struct Release {
    PyObject* o;
    ~Release() { Py_DECREF(o); }
  } release{seq};
  const Py_ssize_t count = PySequence_Fast_GET_SIZE(seq);
  if (count == 0) Py_RETURN_NONE;
  PyObject** items = PySequence_Fast_ITEMS(seq);
  const Tensor& first = cuda_tensor(items[0], "caches");
  const at::Device dev = first.device();
  const Tensor& beam = tensor(arg[1], "beam");
  NEED(beam.dim() == 2 && (beam.scalar_type() == at::kLong || beam.scalar_type() == at::kInt),
       "beam must be int64 or int32 [B, K]");
  const int64_t B = beam.size(0), K = beam.size(1);
  vector(arg[1], "beam", {B, K}, beam.scalar_type(), dev);
  int64_t strides[3];
  rows4(items[0], "caches", first.scalar_type(), dev, strides, first.element_size());
  NEED(first.size(0) == B * K, "caches must have B * K = ", B * K, " states (got ", first.size(0), ")");
  disjoint(first, "caches", 3);
  std::vector<void*> ptrs;
  ptrs.reserve(static_cast<size_t>(count));
  for (Py_ssize_t i = 0; i < count; ++i) {
    const Tensor& t = tensor(items[i], "caches");
    NEED(t.sizes() == first.sizes() && t.scalar_type() == first.scalar_type() && t.device() == dev,
         "caches must share one shape, layout, dtype and device");
    int64_t own[3];  // (a dimension of one element has no stride to speak of: 0 in both)
    rows4(items[i], "caches", first.scalar_type(), dev, own, first.element_size());
    NEED(own[0] == strides[0] && own[1] == strides[1] && own[2] == strides[2],
         "caches must share one shape, layout, dtype and device");
    ptrs.push_back(t.data_ptr());
  }
  if (first.numel() > 0 && count > 1)
    NEED(std::set<void*>(ptrs.begin(), ptrs.end()).size() == ptrs.size(), "caches must be distinct tensors");
  const int32_t* lens = is_none(arg[2]) ? nullptr : vector(arg[2], "lens", {B * K}, at::kInt, dev).const_data_ptr<int32_t>();
  if (B > 0 && K > 0 && first.size(1) > 0) {
    const c10::cuda::CUDAGuard guard(dev);
    check(fn_reorder(ptrs.data(), count, strides, beam.const_data_ptr(), beam.scalar_type() == at::kLong, lens, B, K,
                     first.size(1), first.size(2), first.size(3) * first.element_size(), stream_of(dev)),
          "w8_cache_reorder");
  }
  Py_RETURN_NONE;
}

// The pool, tails and table of a paged cache as the C ABI takes them: arg k, v, k_scale, v_scale,
// k_tail, v_tail, table, lens.
template <typename Args>
void paged_cache(PyObject* const* arg, Args& a, at::ScalarType dt, at::Device dev, bool written) {
  const Tensor& k = rows4(arg[0], "k", at::kChar, dev, a.k_stride, 1);
  const Tensor& v = rows4(arg[1], "v", at::kChar, dev, a.v_stride, 1);
  const int64_t pages = k.size(0), KV = k.size(1), P = k.size(2), D = k.size(3);
  NEED(v.sizes() == k.sizes(), "v must have the shape of k");
  NEED(KV >= 1, "pages have no heads");
  const char* scale_names[2] = {"k_scale", "v_scale"};
  const char* tail_names[2] = {"k_tail", "v_tail"};
  int64_t* scale_strides[2] = {a.k_scale_stride, a.v_scale_stride};
  int64_t* tail_strides[2] = {a.k_tail_stride, a.v_tail_stride};
  const Tensor* scales[2];
  const Tensor* tails[2];
  for (int i = 0; i < 2; ++i) {
    const Tensor& s = tensor(arg[2 + i], scale_names[i]);
    expect(s, scale_names[i], at::kFloat, dev);
    expect_shape(s, scale_names[i], {pages, KV});
    scale_strides[i][0] = s.stride(0), scale_strides[i][1] = s.stride(1);
    scales[i] = &s;
    const Tensor& t = rows4(arg[4 + i], tail_names[i], dt, dev, tail_strides[i], 1);
    tails[i] = &t;
    NEED(t.size(1) == KV && t.size(2) == P && t.size(3) == D, tail_names[i], " must be [B, KV, P, D] with the pages' KV, P and D");
    if (written) {
      disjoint(s, scale_names[i], 2);
      disjoint(t, tail_names[i], 3);
    }
  }
  const int64_t B = tails[0]->size(0);
  NEED(tails[1]->size(0) == B, "v_tail must have the shape of k_tail");
  if (written) {
    disjoint(k, "k", 3);
    disjoint(v, "v", 3);
  }
  const Tensor& table = tensor(arg[6], "table");
  expect(table, "table", at::kInt, dev);
  NEED(table.dim() == 2 && table.size(0) == B, "table must be [B, pages of a sequence]");
  unit_last(table, "table");
  a.table = table.const_data_ptr<int32_t>();
  a.table_stride = table.stride(0);
  a.table_pages = table.size(1);
  a.lens = vector(arg[7], "lens", {B}, at::kInt, dev).const_data_ptr<int32_t>();
  // (written only where `written` is true: the two structs differ in const)
  a.k = static_cast<int8_t*>(const_cast<void*>(k.const_data_ptr()));
  a.v = static_cast<int8_t*>(const_cast<void*>(v.const_data_ptr()));
  a.k_scale = static_cast<float*>(const_cast<void*>(scales[0]->const_data_ptr()));
  a.v_scale = static_cast<float*>(const_cast<void*>(scales[1]->const_data_ptr()));
  a.k_tail = const_cast<void*>(tails[0]->const_data_ptr());
  a.v_tail = const_cast<void*>(tails[1]->const_data_ptr());
  a.batch = B, a.kv_heads = KV, a.head_dim = D, a.pages = pages, a.page = P, a.dtype = type_code(dt);
}

// q, k, v, k_scale, v_scale, k_tail, v_tail, table, lens, k_new, v_new, tree, depth, window, sink, scale, out
PyObject* attention_paged(PyObject* const* arg, Py_ssize_t nargs) {
  ENTRY(17)
  w8_attention_paged_args a = {};
  const Tensor& q = cuda_tensor(arg[0], "q");
  const at::Device dev = q.device();
  const at::ScalarType dt = q.scalar_type();
  NEED(dt == at::kBFloat16 || dt == at::kHalf, "q must be bfloat16 or float16 (got ", dt, ")");
  rows4(arg[0], "q", dt, dev, a.q_stride, 1);
  paged_cache(arg + 1, a, dt, dev, false);
  const int64_t B = q.size(0), H = q.size(1), N = q.size(2), D = q.size(3);
  NEED(a.batch == B && a.head_dim == D, "pages and tails must have q's batch and head size");
  NEED(H % a.kv_heads == 0, "H = ", H, " must be a multiple of KV = ", a.kv_heads);
  const Tensor& kn = rows4(arg[9], "k_new", dt, dev, a.k_new_stride, 1);
  const Tensor& vn = rows4(arg[10], "v_new", dt, dev, a.v_new_stride, 1);
  const int64_t new_shape[4] = {B, a.kv_heads, N, D};
  NEED(kn.sizes() == at::IntArrayRef(new_shape) && vn.sizes() == kn.sizes(), "k_new and v_new must be [B, KV, N, D]");
  a.window = integer(arg[13], "window");
  a.sink = integer(arg[14], "sink");
  a.scale = real(arg[15], "scale");
  tree_depth(arg[11], arg[12], a, B, N, dev);
  NEED(a.tree == nullptr || a.window == 0 || a.depth != nullptr || N == 0, "a tree with a window needs the tokens' depths");
  Tensor out;
  if (is_none(arg[16])) {
    out = make({B, H, N, D}, dt, dev);
    a.out_stride[0] = H * N * D, a.out_stride[1] = N * D, a.out_stride[2] = D;
  } else {
    out = rows4(arg[16], "out", dt, dev, a.out_stride, 1);
    expect_shape(out, "out", q.sizes());
    disjoint(out, "out", 3);
  }
  a.q = q.const_data_ptr(), a.k_new = kn.const_data_ptr(), a.v_new = vn.const_data_ptr(), a.out = out.data_ptr();
  a.heads = H, a.n_new = N;
  {
    const c10::cuda::CUDAGuard guard(dev);
    const Tensor ws = workspace(fn_paged_ws(&a), dev);
    check(fn_paged(&a, ws.data_ptr(), ws.numel(), stream_of(dev)), "w8_attention_paged");
  }
  return is_none(arg[16]) ? wrap(out) : same(arg[16]);
}

// k, v, k_scale, v_scale, k_tail, v_tail, table, lens, k_new, v_new, path, count, lens_out
PyObject* paged_append(PyObject* const* arg, Py_ssize_t nargs) {
  ENTRY(13)
  w8_paged_append_args a = {};
  const Tensor& kn = cuda_tensor(arg[8], "k_new");
  const at::Device dev = kn.device();
  const at::ScalarType dt = kn.scalar_type();
  NEED(dt == at::kBFloat16 || dt == at::kHalf, "k_new must be bfloat16 or float16 (got ", dt, ")");
  rows4(arg[8], "k_new", dt, dev, a.k_new_stride, 1);
  const Tensor& vn = rows4(arg[9], "v_new", dt, dev, a.v_new_stride, 1);
  paged_cache(arg, a, dt, dev, true);
  const int64_t B = a.batch, N = kn.size(2);
  const int64_t new_shape[4] = {B, a.kv_heads, N, a.head_dim};
  NEED(kn.sizes() == at::IntArrayRef(new_shape) && vn.sizes() == kn.sizes(), "k_new and v_new must be [B, KV, N, D]");
  a.n_new = a.steps = N;
  if (!is_none(arg[10])) {
    const Tensor& p = tensor(arg[10], "path");
    NEED(p.dim() == 2, "path must be [B, steps]");
    expect(p, "path", at::kInt, dev);
    a.steps = p.size(1);
    expect_shape(p, "path", {B, a.steps});
    unit_last(p, "path");
    // An empty path is a path: nothing is appended and nothing of it is read.
    a.path = a.steps > 0 ? p.const_data_ptr<int32_t>() : a.lens;
    a.path_stride = p.stride(0);
  }
  if (!is_none(arg[11])) a.count = vector(arg[11], "count", {B}, at::kInt, dev).const_data_ptr<int32_t>();
  const Tensor to = is_none(arg[12]) ? make({B}, at::kInt, dev) : vector(arg[12], "lens_out", {B}, at::kInt, dev);
  a.k_new = kn.const_data_ptr(), a.v_new = vn.const_data_ptr();
  a.lens_out = to.data_ptr<int32_t>();
  {
    const c10::cuda::CUDAGuard guard(dev);
    check(fn_paged_append(&a, stream_of(dev)), "w8_paged_append");
  }
  return is_none(arg[12]) ? wrap(to) : same(arg[12]);
}

// table, lens, free, top, page, room, active, window, sink
PyObject* page_assign(PyObject* const* arg, Py_ssize_t nargs) {
  ENTRY(9)
  w8_page_assign_args a = {};
  const Tensor& table = cuda_tensor(arg[0], "table");
  const at::Device dev = table.device();
  expect(table, "table", at::kInt, dev);
  NEED(table.dim() == 2, "table must be [B, pages of a sequence]");
  unit_last(table, "table");
  disjoint(table, "table", 1);
  const int64_t B = table.size(0);
  a.table = table.data_ptr<int32_t>();
  a.table_stride = table.stride(0);
  a.batch = B, a.table_pages = table.size(1);
  a.lens = vector(arg[1], "lens", {B}, at::kInt, dev).const_data_ptr<int32_t>();
  const Tensor& free = tensor(arg[2], "free");
  NEED(free.dim() == 1, "free must be one-dimensional");
  vector(arg[2], "free", {free.size(0)}, at::kInt, dev);
  a.free = free.data_ptr<int32_t>();
  a.free_pages = free.size(0);
  a.top = vector(arg[3], "top", {1}, at::kInt, dev).data_ptr<int32_t>();
  a.page = integer(arg[4], "page");
  a.room = integer(arg[5], "room");
  if (!is_none(arg[6]))
    a.active = static_cast<const uint8_t*>(vector(arg[6], "active", {B}, at::kBool, dev).const_data_ptr());
  a.window = integer(arg[7], "window");
  a.sink = integer(arg[8], "sink");
  const Tensor ok = make({B}, at::kBool, dev);
  a.ok = static_cast<uint8_t*>(ok.data_ptr());
  {
    const c10::cuda::CUDAGuard guard(dev);
    const Tensor ws = workspace(fn_assign_ws(B, a.table_pages), dev);
    check(fn_assign(&a, ws.data_ptr(), ws.numel(), stream_of(dev)), "w8_page_assign");
  }
  return wrap(ok);
}

// logits, tokens, uniform, parent, draft, temperature, cap
PyObject* draft_verify(PyObject* const* arg, Py_ssize_t nargs) {
  ENTRY(7)
  w8_draft_verify_args a = {};
  const Tensor& x = cuda_tensor(arg[0], "logits");
  const at::Device dev = x.device();
  const at::ScalarType dt = x.scalar_type();
  NEED(type_code(dt) >= 0, "logits must be float32, bfloat16 or float16 (got ", dt, ")");
  NEED(x.dim() == 3, "logits must be [B, N, V]");
  const int64_t B = x.size(0), N = x.size(1), V = x.size(2);
  unit_last(x, "logits");
  a.logits = x.const_data_ptr();
  a.logits_stride[0] = x.stride(0), a.logits_stride[1] = x.stride(1);
  a.tokens = vector(arg[1], "tokens", {B, N}, at::kLong, dev).const_data_ptr<int64_t>();
  a.temperature = real(arg[5], "temperature");
  a.cap = is_none(arg[6]) ? 0.0 : real(arg[6], "cap");
  if (!is_none(arg[2]))
    a.uniform = static_cast<const float*>(vector(arg[2], "uniform", {B, N}, at::kFloat, dev).const_data_ptr());
  else
    NEED(a.temperature == 0.0, "uniform is needed but at temperature 0");
  if (!is_none(arg[3])) {
    const Tensor& t = tensor(arg[3], "parent");
    NEED(t.dim() == 1 || t.dim() == 2, "parent must be [N] or [B, N]");
    expect(t, "parent", at::kInt, dev);
    if (t.dim() == 1)
      expect_shape(t, "parent", {N});
    else
      expect_shape(t, "parent", {B, N});
    unit_last(t, "parent");
    a.parent = t.const_data_ptr<int32_t>();
    a.parent_stride = t.dim() == 2 ? t.stride(0) : 0;
  }
  if (!is_none(arg[4])) {
    const Tensor& t = tensor(arg[4], "draft");
    expect(t, "draft", dt, dev);
    expect_shape(t, "draft", x.sizes());
    unit_last(t, "draft");
    a.draft = t.const_data_ptr();
    a.draft_stride[0] = t.stride(0), a.draft_stride[1] = t.stride(1);
  }
  const Tensor path = make({B, N}, at::kInt, dev), taken = make({B}, at::kInt, dev), token = make({B}, at::kLong, dev);
  a.path = path.data_ptr<int32_t>(), a.taken = taken.data_ptr<int32_t>(), a.token = token.data_ptr<int64_t>();
  a.batch = B, a.n_new = N, a.vocab = V, a.dtype = type_code(dt);
  {
    const c10::cuda::CUDAGuard guard(dev);
    check(fn_verify(&a, stream_of(dev)), "w8_draft_verify");
  }
  return tuple_of({wrap(path), wrap(taken), wrap(token)});
}

// bind(library path, check): take the entry points from the loaded library.
PyObject* bind(PyObject* const* arg, Py_ssize_t nargs) {
  NEED(nargs == 2 && PyUnicode_Check(arg[0]) && PyCallable_Check(arg[1]), "bind(path, check)");
  PyObject* name = nullptr;  // the path's bytes, which need not be UTF-8
  if (!PyUnicode_FSConverter(arg[0], &name)) throw Raised();
  const std::string path = PyBytes_AS_STRING(name);
  Py_DECREF(name);
  void* lib = dlopen(path.c_str(), RTLD_NOW);
  NEED(lib != nullptr, "cannot load ", path);
  auto get = [&](auto& fn, const char* name) {
    fn = reinterpret_cast<std::remove_reference_t<decltype(fn)>>(dlsym(lib, name));
    NEED(fn != nullptr, name, " is missing from the library");
  };
  get(fn_tree, "w8_attention_tree");
  get(fn_tree_ws, "w8_attention_tree_workspace_bytes");
  get(fn_append, "w8_cache_append");
  get(fn_evict, "w8_cache_evict");
  get(fn_evict_ws, "w8_cache_evict_workspace_bytes");
  get(fn_select, "w8_beam_select");
  get(fn_select_ws, "w8_beam_select_workspace_bytes");
  get(fn_reorder, "w8_cache_reorder");
  get(fn_paged, "w8_attention_paged");
  get(fn_paged_ws, "w8_attention_paged_workspace_bytes");
  get(fn_paged_append, "w8_paged_append");
  get(fn_assign, "w8_page_assign");
  get(fn_assign_ws, "w8_page_assign_workspace_bytes");
  get(fn_verify, "w8_draft_verify");
  check_status = same(arg[1]);
  Py_RETURN_NONE;
}

// (A message may quote a path, which need not be UTF-8.)
void raise(PyObject* type, const char* what) {
  PyObject* text = PyUnicode_DecodeUTF8(what, static_cast<Py_ssize_t>(std::char_traits<char>::length(what)), "replace");
  if (text == nullptr) return;
  PyErr_SetObject(type, text);
  Py_DECREF(text);
}

// No C++ exception passes into Python.
template <PyObject* (*F)(PyObject* const*, Py_ssize_t)>
PyObject* entry(PyObject*, PyObject* const* arg, Py_ssize_t nargs) {
  try {
    return F(arg, nargs);
  } catch (const Raised&) {
  } catch (const Refused& x) {
    raise(PyExc_ValueError, x.what());
  } catch (const std::exception& x) {  // torch's own, out of memory among them
    raise(PyExc_RuntimeError, x.what());
  } catch (...) {
    PyErr_SetString(PyExc_RuntimeError, "unknown C++ exception");
  }
  return nullptr;
}

}  // namespace

PyMODINIT_FUNC PyInit__decode(void) {
  static PyMethodDef methods[] = {
      {"bind", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&entry<bind>)), METH_FASTCALL, nullptr},
      {"attention_tree", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&entry<attention_tree>)), METH_FASTCALL, nullptr},
      {"cache_append", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&entry<cache_append>)), METH_FASTCALL, nullptr},
      {"cache_evict", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&entry<cache_evict>)), METH_FASTCALL, nullptr},
      {"beam_select", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&entry<beam_select>)), METH_FASTCALL, nullptr},
      {"attention_paged", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&entry<attention_paged>)), METH_FASTCALL, nullptr},
      {"paged_append", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&entry<paged_append>)), METH_FASTCALL, nullptr},
      {"page_assign", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&entry<page_assign>)), METH_FASTCALL, nullptr},
      {"draft_verify", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&entry<draft_verify>)), METH_FASTCALL, nullptr},
      {"cache_reorder", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&entry<cache_reorder>)), METH_FASTCALL, nullptr},
      {nullptr, nullptr, 0, nullptr}};
  static PyModuleDef module = {PyModuleDef_HEAD_INIT, "_decode", "Binding of the decoding operators.", -1, methods,
                               nullptr, nullptr, nullptr, nullptr};
  return PyModule_Create(&module);
}
