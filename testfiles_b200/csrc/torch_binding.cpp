// torch_binding.cpp — the Python module testfiles_b200._welm_torch: the
// multi-axis rotary embedding, the rotating cache append and the paged
// attention on torch tensors, over the library's C entries.
//
// A small launch takes the GPU about 2 us.  The same checks and call through
// Python and ctypes took 12 us (multi-axis, 16 tokens), 16 us (append, 32
// tokens) and 23 us (attention, one request), and the differentiable form 147 us,
// so these operators check their arguments, allocate and record gradients here.  Python's wrappers (paged.py) carry the signatures
// and the documentation.

#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/utils/object_ptr.h>

#include <ATen/ATen.h>
#include <ATen/core/grad_mode.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>

#include <array>
#include <cmath>
#include <limits>
#include <memory>
#include <mutex>
#include <stdexcept>
#include <string>

#include "rope_rows.h"
#include "welm_rope.h"

namespace {

using at::Tensor;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

constexpr int64_t kHeadDim = WELM_ROPE_HEAD_DIM, kRopeDim = WELM_ROPE_ROPE_DIM, kPairs = kRopeDim / 2;

// A library entry's non-zero status, raised as testfiles_b200.WelmRopeError
// (from a backward pass, whose errors torch's engine carries, as RuntimeError).
struct LibraryError : std::runtime_error {
  const char* entry;
  int status;
  LibraryError(const char* e, int s)
      : std::runtime_error(std::string(e) + " failed: " + welm_rope_status_string(s)), entry(e), status(s) {}
};

// ---------------------------------------------------------------------------
// Checks.
// ---------------------------------------------------------------------------
const char* dtype_name(at::ScalarType t) {
  switch (t) {
    case at::kBFloat16: return "torch.bfloat16";
    case at::kHalf: return "torch.float16";
    case at::kFloat: return "torch.float32";
    case at::kDouble: return "torch.float64";
    case at::kInt: return "torch.int32";
    case at::kLong: return "torch.int64";
    default: return c10::toString(t);
  }
}

void check(const Tensor& t, const char* name, at::ScalarType dtype, c10::DeviceIndex index) {
  TORCH_CHECK_VALUE(t.defined(), name, " is required");
  TORCH_CHECK_TYPE(t.scalar_type() == dtype, name, " must be ", dtype_name(dtype), ", got ",
                   dtype_name(t.scalar_type()));
  TORCH_CHECK_VALUE(t.is_cuda() && t.get_device() == index, name, " is on ", t.device(), ", expected cuda:",
                    int(index));
}

c10::DeviceIndex device_index(const Tensor& t) {
  TORCH_CHECK_VALUE(t.defined() && t.is_cuda(),
                    "query must be a CUDA tensor (the op runs only on the sm_100a library)");
  return t.get_device();
}

bool vectors(const Tensor& t, std::initializer_list<int64_t> strides) {  // 16-byte accesses reach every element
  int64_t bits = 0, low = 0;
  for (const int64_t s : strides) {
    bits |= s;
    low = std::min(low, s);
  }
  return low >= 0 && (bits & 7) == 0 && (reinterpret_cast<uintptr_t>(t.const_data_ptr()) & 15u) == 0;
}

struct Rows {
  int64_t tokens, heads, token, head;
};

Rows rows_of(const Tensor& t, const char* name) {
  TORCH_CHECK_VALUE(t.dim() == 3 && t.size(2) == kHeadDim, name, " must have shape [tokens, heads, ", kHeadDim,
                    "], got ", t.sizes());
  Rows r{t.size(0), t.size(1), 0, 0};
  if (r.tokens == 0 || r.heads == 0) return r;
  r.token = t.stride(0);
  r.head = t.stride(1);
  TORCH_CHECK_VALUE(t.stride(2) == 1 && vectors(t, {r.token, r.head}), name,
                    " must have lane stride 1, other strides that are multiples of 8, and a 16-byte aligned start");
  return r;
}

// A tensor that the call writes and one that it reads or writes must not share a
// row.  The library refuses that; only then is it looked up here which they are.
RowSet row_set(const Tensor& t, const Rows& r) {
  return {reinterpret_cast<uintptr_t>(t.const_data_ptr()), {r.tokens, r.heads, 1}, {r.token, r.head, 0}};
}

void check_apart(const RowSet& a, const char* a_name, const RowSet& b, const char* b_name) {
  TORCH_CHECK_VALUE(!rows_meet(a, b), a_name, " and ", b_name, " must not overlap");
}

void check_vector(const Tensor& t, const char* name, int64_t size) {
  TORCH_CHECK_VALUE(t.dim() == 1 && t.size(0) == size && (size <= 1 || t.stride(0) == 1), name,
                    " must be a contiguous 1-D tensor of ", size, " entries, got ", t.sizes());
}

struct Sections {
  int32_t pairs[WELM_ROPE_MAX_AXES] = {kPairs, 0, 0, 0};
  int64_t axes = 1;
  bool given = false;  // positions are [axes, tokens], else [tokens]
};

Sections sections_of(const std::vector<int64_t>& values) {
  Sections s;
  int64_t sum = 0;
  bool ok = !values.empty() && values.size() <= WELM_ROPE_MAX_AXES;
  for (size_t i = 0; ok && i < values.size(); ++i) {
    ok = values[i] >= 0 && values[i] <= kPairs;
    s.pairs[i] = int32_t(values[i]);
    sum += values[i];
  }
  TORCH_CHECK_VALUE(ok && sum == kPairs, "sections must be 1 to ", WELM_ROPE_MAX_AXES,
                    " counts of pairs that add up to ", kPairs, ", got ", values);
  s.axes = int64_t(values.size());
  s.given = true;
  return s;
}

// Position stride of `positions` for these sections.
int64_t check_positions(const Tensor& positions, const Sections& s, int64_t tokens, c10::DeviceIndex index) {
  check(positions, "positions", at::kLong, index);
  if (!s.given) {
    check_vector(positions, "positions", tokens);
    return 0;
  }
  TORCH_CHECK_VALUE(positions.dim() == 2 && positions.size(0) == s.axes && positions.size(1) == tokens &&
                        (tokens <= 1 || positions.stride(1) == 1),
                    "positions must have shape [", s.axes, ", ", tokens,
                    "] (axes, tokens) and contiguous rows, got ", positions.sizes(), " with strides ",
                    positions.strides());
  return positions.stride(0);
}

int64_t check_cos_sin(const Tensor& cache, c10::DeviceIndex index) {
  check(cache, "cos_sin_cache", at::kFloat, index);
  TORCH_CHECK_VALUE(cache.dim() == 2 && cache.size(1) == kRopeDim && cache.is_contiguous() &&
                        (reinterpret_cast<uintptr_t>(cache.const_data_ptr()) & 15u) == 0,
                    "cos_sin_cache must be a contiguous, 16-byte aligned [max_position, ", kRopeDim,
                    "] float32 tensor");
  return cache.size(0);
}

std::array<int64_t, 3> check_cache(const Tensor& cache, const char* name, c10::DeviceIndex index) {
  check(cache, name, at::kBFloat16, index);
  TORCH_CHECK_VALUE(cache.dim() == 4 && cache.size(3) == kHeadDim, name,
                    " must have shape [num_blocks, block_size, heads, ", kHeadDim, "], got ", cache.sizes());
  const std::array<int64_t, 3> s{cache.stride(0), cache.stride(1), cache.stride(2)};
  TORCH_CHECK_VALUE(cache.stride(3) == 1 && vectors(cache, {s[0], s[1], s[2]}), name,
                    " must have lane stride 1, other strides that are multiples of 8, and a 16-byte aligned start");
  return s;
}

RowSet page_set(const Tensor& cache, const std::array<int64_t, 3>& s) {
  return {reinterpret_cast<uintptr_t>(cache.const_data_ptr()), {cache.size(0), cache.size(1), cache.size(2)},
          {s[0], s[1], s[2]}};
}

int32_t* status_of(const OptTensor& status, c10::DeviceIndex index) {
  if (!status) return nullptr;
  check(*status, "status", at::kInt, index);
  TORCH_CHECK_VALUE(status->numel() >= 1, "status must hold at least one int32");
  return static_cast<int32_t*>(status->data_ptr());
}

// Refuses a tensor whose tangent the call would lose or leave behind.
void no_tangent(const char* entry, const Tensor& t) {
  TORCH_CHECK_NOT_IMPLEMENTED(!(t.defined() && t._fw_grad(0).defined()), entry, " has no forward-mode derivative");
}

// Refuses a tensor whose gradient or tangent the call would lose.
void no_grad(const char* entry, const Tensor& t) {
  no_tangent(entry, t);
  TORCH_CHECK_VALUE(!(t.defined() && t.requires_grad() && at::GradMode::is_enabled()), entry,
                    " has no backward pass: call it under torch.no_grad() or on detached tensors");
}

// Tells autograd that a tensor was written in place.
void written(const Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

void* stream_of(c10::DeviceIndex index) { return c10::cuda::getCurrentCUDAStream(index).stream(); }

void done(const char* entry, int status) {
  if (status != WELM_ROPE_OK) throw LibraryError(entry, status);
}

// ---------------------------------------------------------------------------
// Rotary embedding with several axes.
// ---------------------------------------------------------------------------
struct Turn {
  Sections sections;
  bool interleaved, inverse;
};

// welm_rope_multi_axis of x and, where given, y into x_out and y_out (which may be x and y).
void rotate(const Tensor& x, const Tensor& x_out, const char* x_name, const OptTensor& y, const OptTensor& y_out,
            const Tensor& positions, const Tensor& cos_sin, const Turn& turn, const OptTensor& status) {
  const c10::DeviceIndex index = device_index(x);
  check(x, x_name, at::kBFloat16, index);
  const Rows a = rows_of(x, x_name), a_out = rows_of(x_out, x_name);
  Rows b{a.tokens, 0, 0, 0}, b_out = b;
  if (y) {
    check(*y, "key", at::kBFloat16, index);
    b = rows_of(*y, "key");
    b_out = rows_of(*y_out, "key");
    TORCH_CHECK_VALUE(b.tokens == a.tokens, "query and key need the same number of tokens");
  }
  const int64_t position_stride = check_positions(positions, turn.sections, a.tokens, index);
  const int64_t max_position = check_cos_sin(cos_sin, index);
  int32_t* const device_status = status_of(status, index);
  const c10::cuda::CUDAGuard guard(index);
  const int result =
      welm_rope_multi_axis(x.const_data_ptr(), x_out.data_ptr(), y ? y->const_data_ptr() : nullptr,
                           y ? y_out->data_ptr() : nullptr, positions.const_data_ptr<int64_t>(),
                           cos_sin.const_data_ptr<float>(), turn.sections.pairs, turn.sections.axes, turn.interleaved,
                           turn.inverse, a.tokens, a.heads, b.heads, a.token, a.head, a_out.token, a_out.head, b.token,
                           b.head, b_out.token, b_out.head, position_stride, max_position, device_status,
                           stream_of(index));
  if (result == WELM_ROPE_ERR_BAD_STRIDE && y) check_apart(row_set(x_out, a_out), x_name, row_set(*y_out, b_out), "key");
  done("welm_rope_multi_axis", result);
}

// x in a layout that the kernel reads.
Tensor readable(const Tensor& x) {
  if (!x.defined() || x.dim() != 3 || x.numel() == 0) return x;
  if (x.stride(2) == 1 && vectors(x, {x.stride(0), x.stride(1)})) return x;
  return x.clone(at::MemoryFormat::Contiguous);
}

variable_list rotated(const Tensor& x, const char* x_name, const OptTensor& y, const Tensor& positions,
                      const Tensor& cos_sin, const Turn& turn, const OptTensor& status) {
  const Tensor from_x = readable(x);
  const OptTensor from_y = y ? OptTensor(readable(*y)) : std::nullopt;
  const Tensor x_out = at::empty(x.sizes(), x.options());
  const OptTensor y_out = y ? OptTensor(at::empty(y->sizes(), y->options())) : std::nullopt;
  rotate(from_x, x_out, x_name, from_y, y_out, positions, cos_sin, turn, status);
  if (y) return {x_out, *y_out};
  return {x_out};
}

variable_list differentiable(const Tensor& x, const char* x_name, const OptTensor& y, const Tensor& positions,
                             const Tensor& cos_sin, const Turn& turn, const OptTensor& status);

// The gradient of a rotation is the inverse rotation.  A node of its own holds
// what that needs as it is: a forward and a backward pass take 61 us of host time
// (35 us of a view's, with no kernel at all), and 67 through torch's custom
// functions, which box and look up every argument.
struct MultiAxisBackward : torch::autograd::Node {
  torch::autograd::SavedVariable positions, cos_sin;
  Turn turn;

  variable_list apply(variable_list&& grads) override {
    const std::lock_guard<std::mutex> lock(mutex_);
    const Tensor at = positions.unpack(), rows = cos_sin.unpack();
    const Turn back_turn{turn.sections, turn.interleaved, !turn.inverse};
    Tensor dx = task_should_compute_output(0) ? grads[0] : Tensor();
    Tensor dy = num_outputs() > 1 && task_should_compute_output(1) ? grads[1] : Tensor();
    if (dx.defined() || dy.defined()) {
      const bool both = dx.defined() && dy.defined();
      const variable_list back = differentiable(dx.defined() ? dx : dy, "gradient", both ? OptTensor(dy) : std::nullopt,
                                                at, rows, back_turn, std::nullopt);
      (dx.defined() ? dx : dy) = back[0];
      if (both) dy = back[1];
    }
    if (num_outputs() == 1) return {dx};
    return {dx, dy};
  }

  void release_variables() override {
    const std::lock_guard<std::mutex> lock(mutex_);
    positions.reset_data();
    cos_sin.reset_data();
  }

  std::string name() const override { return "MultiAxisBackward"; }
};

// Rotated copies of x and y, with their history where gradients are wanted.
variable_list differentiable(const Tensor& x, const char* x_name, const OptTensor& y, const Tensor& positions,
                             const Tensor& cos_sin, const Turn& turn, const OptTensor& status) {
  no_tangent("rope_multi_axis", x);
  if (y) no_tangent("rope_multi_axis", *y);
  std::shared_ptr<MultiAxisBackward> node;
  if (at::GradMode::is_enabled() && (x.requires_grad() || (y && y->requires_grad()))) {
    node = std::shared_ptr<MultiAxisBackward>(new MultiAxisBackward(), torch::autograd::deleteNode);
    node->set_next_edges(y ? torch::autograd::collect_next_edges(x, *y) : torch::autograd::collect_next_edges(x));
    node->positions = torch::autograd::SavedVariable(positions, false);
    node->cos_sin = torch::autograd::SavedVariable(cos_sin, false);
    node->turn = turn;
  }
  variable_list out;
  {
    const at::NoGradGuard no_grad;
    out = rotated(x, x_name, y, positions, cos_sin, turn, status);
  }
  if (node)
    for (const Tensor& t : out) torch::autograd::set_history(t, node);
  return out;
}

// ---------------------------------------------------------------------------
// Python's arguments and results.
// ---------------------------------------------------------------------------
Tensor tensor_arg(PyObject* o, const char* name) {
  TORCH_CHECK_VALUE(o != Py_None, name, " is required");
  TORCH_CHECK_TYPE(THPVariable_Check(o), name, " must be a torch.Tensor");
  return THPVariable_Unpack(o);
}
OptTensor opt_tensor_arg(PyObject* o, const char* name) {
  return o == Py_None ? std::nullopt : OptTensor(tensor_arg(o, name));
}
Tensor query_arg(PyObject* o) {  // decides the device, so what is no tensor is refused in the same words
  TORCH_CHECK_VALUE(THPVariable_Check(o), "query must be a CUDA tensor (the op runs only on the sm_100a library)");
  return THPVariable_Unpack(o);
}
bool bool_arg(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw python_error();
  return v != 0;
}
int64_t int_arg(PyObject* o) {
  const int64_t v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw python_error();
  return v;
}
std::vector<int64_t> ints_arg(PyObject* o) {
  THPObjectPtr list(PySequence_Fast(o, "sections must be a sequence of integers"));
  if (!list) throw python_error();
  std::vector<int64_t> v;
  const Py_ssize_t n = PySequence_Fast_GET_SIZE(list.get());
  for (Py_ssize_t i = 0; i < n; ++i) v.push_back(int_arg(PySequence_Fast_GET_ITEM(list.get(), i)));
  return v;
}

void arity(Py_ssize_t got, Py_ssize_t want) {
  TORCH_CHECK_TYPE(got == want, "expected ", want, " arguments, got ", got);
}

// testfiles_b200.WelmRopeError(entry, status)
void raise_library_error(const LibraryError& e) {
  THPObjectPtr module(PyImport_ImportModule("testfiles_b200._native"));
  if (!module) return;
  THPObjectPtr cls(PyObject_GetAttrString(module.get(), "WelmRopeError"));
  if (!cls) return;
  THPObjectPtr error(PyObject_CallFunction(cls.get(), "si", e.entry, e.status));
  if (error) PyErr_SetObject(cls.get(), error.get());
}

#define WELM_BEGIN HANDLE_TH_ERRORS try {
#define WELM_END                   \
  }                                \
  catch (const LibraryError& e) {  \
    raise_library_error(e);        \
    return nullptr;                \
  }                                \
  END_HANDLE_TH_ERRORS

PyObject* multi_axis_inplace(PyObject*, PyObject* const* args, Py_ssize_t n) {
  WELM_BEGIN
  arity(n, 8);
  const Tensor q = query_arg(args[0]), k = tensor_arg(args[1], "key");
  device_index(q);
  no_grad("rope_multi_axis_inplace", q);
  no_grad("rope_multi_axis_inplace", k);
  const Tensor cos_sin = tensor_arg(args[3], "cos_sin_cache");
  no_grad("rope_multi_axis_inplace", cos_sin);
  rotate(q, q, "query", k, k, tensor_arg(args[2], "positions"), cos_sin,
         {sections_of(ints_arg(args[4])), bool_arg(args[5]), bool_arg(args[6])}, opt_tensor_arg(args[7], "status"));
  written(q);
  written(k);
  Py_RETURN_NONE;
  WELM_END
}

PyObject* multi_axis(PyObject*, PyObject* const* args, Py_ssize_t n) {
  WELM_BEGIN
  arity(n, 8);
  const Tensor q = query_arg(args[0]), k = tensor_arg(args[1], "key");
  device_index(q);
  const Tensor cos_sin = tensor_arg(args[3], "cos_sin_cache");
  no_grad("the cos_sin_cache of rope_multi_axis", cos_sin);
  const variable_list out =
      differentiable(q, "query", k, tensor_arg(args[2], "positions"), cos_sin,
                     {sections_of(ints_arg(args[4])), bool_arg(args[5]), bool_arg(args[6])},
                     opt_tensor_arg(args[7], "status"));
  return PyTuple_Pack(2, THPObjectPtr(THPVariable_Wrap(out[0])).get(), THPObjectPtr(THPVariable_Wrap(out[1])).get());
  WELM_END
}

PyObject* kv_append(PyObject*, PyObject* const* args, Py_ssize_t n) {
  WELM_BEGIN
  arity(n, 11);
  const OptTensor q = opt_tensor_arg(args[0], "query");
  const Tensor k = query_arg(args[1]), v = tensor_arg(args[2], "v");
  const Tensor positions = tensor_arg(args[3], "positions"), cos_sin = tensor_arg(args[4], "cos_sin_cache");
  const Tensor slots = tensor_arg(args[5], "slot_mapping");
  const Tensor key_cache = tensor_arg(args[6], "key_cache"), value_cache = tensor_arg(args[7], "value_cache");
  const Sections sections = args[8] == Py_None ? Sections() : sections_of(ints_arg(args[8]));
  const bool interleaved = bool_arg(args[9]);
  const OptTensor status = opt_tensor_arg(args[10], "status");
  const c10::DeviceIndex index = device_index(k);
  if (q) no_grad("rope_kv_append", *q);
  no_grad("rope_kv_append", k);
  no_grad("rope_kv_append", v);
  no_grad("rope_kv_append", cos_sin);
  no_grad("rope_kv_append", key_cache);
  no_grad("rope_kv_append", value_cache);
  check(k, "key", at::kBFloat16, index);
  check(v, "v", at::kBFloat16, index);
  const Rows kr = rows_of(k, "key"), vr = rows_of(v, "v");
  TORCH_CHECK_VALUE(vr.tokens == kr.tokens && vr.heads == kr.heads, "key and v need the same tokens and heads");
  Rows qr{kr.tokens, 0, 0, 0};
  if (q) {
    check(*q, "query", at::kBFloat16, index);
    qr = rows_of(*q, "query");
    TORCH_CHECK_VALUE(qr.tokens == kr.tokens, "query and key need the same number of tokens");
  }
  const int64_t position_stride = check_positions(positions, sections, kr.tokens, index);
  const int64_t max_position = check_cos_sin(cos_sin, index);
  check(slots, "slot_mapping", at::kLong, index);
  check_vector(slots, "slot_mapping", kr.tokens);
  const auto key_strides = check_cache(key_cache, "key_cache", index);
  const auto value_strides = check_cache(value_cache, "value_cache", index);
  TORCH_CHECK_VALUE(value_cache.sizes() == key_cache.sizes() && key_cache.size(2) == kr.heads,
                    "key_cache and value_cache need the same shape, with the heads of key and v");
  int32_t* const device_status = status_of(status, index);
  const c10::cuda::CUDAGuard guard(index);
  const int result =
      welm_rope_kv_append(q ? q->data_ptr() : nullptr, k.const_data_ptr(), v.const_data_ptr(),
                          positions.const_data_ptr<int64_t>(), cos_sin.const_data_ptr<float>(), sections.pairs,
                          sections.axes, interleaved, slots.const_data_ptr<int64_t>(), key_cache.data_ptr(),
                          value_cache.data_ptr(), kr.tokens, qr.heads, kr.heads, qr.token, qr.head, kr.token, kr.head,
                          vr.token, vr.head, key_cache.size(0), key_cache.size(1), key_strides.data(),
                          value_strides.data(), position_stride, max_position, device_status, stream_of(index));
  if (result == WELM_ROPE_ERR_BAD_STRIDE) {
    const RowSet keys = page_set(key_cache, key_strides), values = page_set(value_cache, value_strides);
    if (q) {
      const RowSet q_rows = row_set(*q, qr);
      check_apart(q_rows, "query", row_set(k, kr), "key");
      check_apart(q_rows, "query", row_set(v, vr), "v");
      check_apart(q_rows, "query", keys, "key_cache");
      check_apart(q_rows, "query", values, "value_cache");
    }
    check_apart(keys, "key_cache", values, "value_cache");
  }
  done("welm_rope_kv_append", result);
  if (q) written(*q);
  written(key_cache);
  written(value_cache);
  Py_RETURN_NONE;
  WELM_END
}

int64_t workspace_bytes(int64_t tokens, int64_t batch, int64_t q_heads, int64_t k_heads, int64_t prefix_len,
                        c10::DeviceIndex index) {
  int64_t bytes = 0;
  const c10::cuda::CUDAGuard guard(index);
  done("welm_rope_attend_workspace",
       welm_rope_attend_workspace(tokens, batch, q_heads, k_heads, prefix_len, &bytes));
  return bytes;
}

PyObject* attend_workspace_bytes(PyObject*, PyObject* const* args, Py_ssize_t n) {
  WELM_BEGIN
  arity(n, 6);
  return PyLong_FromLongLong(workspace_bytes(int_arg(args[0]), int_arg(args[1]), int_arg(args[2]), int_arg(args[3]),
                                             int_arg(args[4]), c10::DeviceIndex(int_arg(args[5]))));
  WELM_END
}

PyObject* attend(PyObject*, PyObject* const* args, Py_ssize_t n) {
  WELM_BEGIN
  arity(n, 13);
  const Tensor q = query_arg(args[0]);
  const c10::DeviceIndex index = device_index(q);
  const Tensor key_cache = tensor_arg(args[1], "key_cache"), value_cache = tensor_arg(args[2], "value_cache");
  const Tensor table = tensor_arg(args[3], "block_table"), lens = tensor_arg(args[4], "seq_lens");
  const OptTensor starts = opt_tensor_arg(args[5], "query_starts");
  const OptTensor prefix_table = opt_tensor_arg(args[6], "prefix_table");
  const int64_t prefix_len = int_arg(args[7]);
  const double scale = args[8] == Py_None ? 1.0 / std::sqrt(double(kHeadDim)) : PyFloat_AsDouble(args[8]);
  if (PyErr_Occurred()) throw python_error();
  OptTensor out = opt_tensor_arg(args[9], "out");
  const bool return_lse = bool_arg(args[10]);
  OptTensor workspace = opt_tensor_arg(args[11], "workspace");
  const OptTensor status = opt_tensor_arg(args[12], "status");
  no_grad("attend_shared_prefix", q);
  no_grad("attend_shared_prefix", key_cache);
  no_grad("attend_shared_prefix", value_cache);
  check(q, "query", at::kBFloat16, index);
  const Rows qr = rows_of(q, "query");
  const auto key_strides = check_cache(key_cache, "key_cache", index);
  const auto value_strides = check_cache(value_cache, "value_cache", index);
  TORCH_CHECK_VALUE(value_cache.sizes() == key_cache.sizes(), "key_cache and value_cache need the same shape");
  const int64_t blocks = key_cache.size(0), block_size = key_cache.size(1), k_heads = key_cache.size(2);
  TORCH_CHECK_VALUE(k_heads >= 1 && qr.heads >= 1 && qr.heads % k_heads == 0, "query heads (", qr.heads,
                    ") must be a multiple of the cache's heads (", k_heads, ")");
  TORCH_CHECK_VALUE(block_size >= 1 && block_size % 8 == 0, "block_size must be a multiple of 8, got ", block_size);
  check(table, "block_table", at::kInt, index);
  TORCH_CHECK_VALUE(table.dim() == 2 && (table.size(1) <= 1 || table.stride(1) == 1),
                    "block_table must be a [batch, blocks] int32 tensor with contiguous rows");
  const int64_t batch = table.size(0), width = table.size(1);
  check(lens, "seq_lens", at::kLong, index);
  check_vector(lens, "seq_lens", batch);
  if (starts) {
    check(*starts, "query_starts", at::kLong, index);
    check_vector(*starts, "query_starts", batch + 1);
  } else {
    TORCH_CHECK_VALUE(qr.tokens == batch,
                      "without query_starts every request has one query token: q rows must equal block_table rows");
  }
  TORCH_CHECK_VALUE(prefix_len >= 0, "prefix_len must not be negative");
  if (prefix_len > 0) {
    check(prefix_table ? *prefix_table : Tensor(), "prefix_table", at::kInt, index);
    TORCH_CHECK_VALUE(prefix_table->dim() == 1 && prefix_table->size(0) >= (prefix_len - 1) / block_size + 1 &&
                          (prefix_table->size(0) <= 1 || prefix_table->stride(0) == 1),
                      "prefix_table must be a contiguous 1-D int32 tensor with a block for every prefix key");
  }
  // the kernels multiply by scale log2(e) in FP32
  TORCH_CHECK_VALUE(float(scale) > 0.0f && std::isfinite(float(scale) * 1.4426950408889634f),
                    "scale must be positive and finite in FP32, log2(e) times as much too, got ", scale);
  const bool fill = !out;
  if (out) {
    check(*out, "out", at::kBFloat16, index);
    TORCH_CHECK_VALUE(out->sizes() == q.sizes(), "out must have the shape of q, got ", out->sizes());
    no_grad("attend_shared_prefix", *out);
  } else {
    out = at::empty(q.sizes(), q.options());
  }
  const Rows outr = rows_of(*out, "out");
  Tensor lse;
  if (return_lse) lse = at::empty({qr.tokens, qr.heads}, q.options().dtype(at::kFloat));
  int32_t* const device_status = status_of(status, index);
  if (qr.tokens > 0 && batch > 0) {
    TORCH_CHECK_VALUE(blocks > 0, "the cache has no blocks");
    const int64_t need = workspace_bytes(qr.tokens, batch, qr.heads, k_heads, prefix_len, index);
    if (!workspace) workspace = at::empty({need}, q.options().dtype(at::kByte));
    TORCH_CHECK_VALUE(workspace->is_cuda() && workspace->get_device() == index,
                      "workspace must be a tensor on the device of q");
    const int64_t size = workspace->numel() * int64_t(workspace->element_size());
    TORCH_CHECK_VALUE(size >= need && workspace->is_contiguous() &&
                          (reinterpret_cast<uintptr_t>(workspace->data_ptr()) & 31u) == 0,
                      "workspace must be contiguous, 32-byte aligned and hold ", need, " bytes");
    const c10::cuda::CUDAGuard guard(index);
    const int result =
        welm_rope_attend(q.const_data_ptr(), out->data_ptr(), return_lse ? lse.data_ptr<float>() : nullptr,
                         key_cache.const_data_ptr(), value_cache.const_data_ptr(), table.const_data_ptr<int32_t>(),
                         lens.const_data_ptr<int64_t>(), starts ? starts->const_data_ptr<int64_t>() : nullptr,
                         prefix_len > 0 ? prefix_table->const_data_ptr<int32_t>() : nullptr, prefix_len, qr.tokens,
                         batch, qr.heads, k_heads, qr.token, qr.head, outr.token, outr.head, width, table.stride(0),
                         blocks, block_size, key_strides.data(), value_strides.data(), float(scale), fill,
                         workspace->data_ptr(), size, device_status, stream_of(index));
    if (result == WELM_ROPE_ERR_BAD_STRIDE) {
      const RowSet out_rows = row_set(*out, outr);
      check_apart(out_rows, "out", row_set(q, qr), "query");
      check_apart(out_rows, "out", page_set(key_cache, key_strides), "key_cache");
      check_apart(out_rows, "out", page_set(value_cache, value_strides), "value_cache");
    }
    done("welm_rope_attend", result);
  } else {  // no request
    if (fill) out->zero_();
    if (return_lse) lse.fill_(-std::numeric_limits<float>::infinity());
  }
  if (!fill) written(*out);
  if (!return_lse) return THPVariable_Wrap(*out);
  return PyTuple_Pack(2, THPObjectPtr(THPVariable_Wrap(*out)).get(), THPObjectPtr(THPVariable_Wrap(lse)).get());
  WELM_END
}

PyMethodDef methods[] = {
    {"multi_axis_inplace", reinterpret_cast<PyCFunction>(multi_axis_inplace), METH_FASTCALL, nullptr},
    {"multi_axis", reinterpret_cast<PyCFunction>(multi_axis), METH_FASTCALL, nullptr},
    {"kv_append", reinterpret_cast<PyCFunction>(kv_append), METH_FASTCALL, nullptr},
    {"attend", reinterpret_cast<PyCFunction>(attend), METH_FASTCALL, nullptr},
    {"attend_workspace_bytes", reinterpret_cast<PyCFunction>(attend_workspace_bytes), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_welm_torch", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

extern "C" __attribute__((visibility("default"))) PyObject* PyInit__welm_torch() {
  if (welm_rope_abi_version() != WELM_ROPE_ABI_VERSION) {
    PyErr_SetString(PyExc_RuntimeError,
                    "_welm_torch and libwelm_rope_b200 are of different versions: rebuild both with `python -m "
                    "testfiles_b200.build`");
    return nullptr;
  }
  return PyModule_Create(&module);
}
