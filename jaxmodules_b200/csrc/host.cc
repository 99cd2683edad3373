// The host side of one attention or mask call: arguments, allocations, launches, one call per step from Python.
//
// A small call is bound by its host path: the passes of 2 x 128 float32 tokens of 8 heads take 43 us of the device, and took 200 us
// of the host with the argument structures filled in, and the tensors allocated, from Python (136 - 147 us now; create_block_mask of
// 16 x 16 blocks 48 -> 22).  Everything is built for one call and dropped with it; the library's entry points are those of include/bma.h, handed over as addresses by jaxmodules_b200/_native.py,
// so that both sides use the one library that is loaded.
#include <cuda_runtime_api.h>
#include <nvtx3/nvToolsExt.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/utils/pybind.h>
#include <torch/csrc/autograd/custom_function.h>
#include <ATen/ATen.h>
#include <ATen/EmptyTensor.h>
#include <c10/core/Allocator.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/VirtualGuardImpl.h>

#include <algorithm>
#include <cmath>
#include <optional>
#include <string>

#include "../../include/bma.h"

namespace {

namespace py = pybind11;
using at::Tensor;
using OptTensor = std::optional<Tensor>;

// ---- the library ------------------------------------------------------------------------------------------------
#define BMA_FUNCTIONS(X)                                                                                                      \
  X(bma_mask_compile_workspace_bytes) X(bma_mask_compile) X(bma_attn_plan) X(bma_attn_bwd_plan) X(bma_attn_fwd_implies_lists) X(bma_attn_fwd_workspace_bytes) \
  X(bma_attn_fwd_uses_workspace) X(bma_attn_fwd_ws) X(bma_attn_f32_workspace_bytes) X(bma_attn_fwd_f32) X(bma_attn_bwd_f32) X(bma_attn_bwd_f32_o) X(bma_attn_bwd_preprocess)       \
  X(bma_attn_bwd_workspace_bytes) X(bma_attn_bwd_scratch_bytes) X(bma_attn_bwd_scratch_min_bytes) X(bma_attn_bwd) X(bma_attn_bwd_o) \
  X(bma_error_string) X(bma_rotate) X(bma_rotate_bwd_workspace_bytes) X(bma_rotate_bwd) X(bma_append_kv) X(bma_read_kv) X(bma_paged_attn_workspace_bytes) X(bma_paged_attn)
struct Library {
#define X(name) decltype(&::name) name = nullptr;
  BMA_FUNCTIONS(X)
#undef X
} lib;
PyObject* error_class = nullptr;   // _native.BmaError, which lives as long as the process

void bind(const py::dict& addresses, py::object error) {
#define X(name) lib.name = reinterpret_cast<decltype(&::name)>(addresses[#name].cast<uintptr_t>());
  BMA_FUNCTIONS(X)
#undef X
  Py_XDECREF(error_class);
  error_class = error.release().ptr();
}

void check(int status, const char* where) {
  if (status == BMA_OK) return;
  py::object e = py::reinterpret_borrow<py::object>(error_class)(status, where);
  PyErr_SetObject(error_class, e.ptr());
  throw py::error_already_set();
}

// One launch group: a range named after it, visible in a timeline profiler and free otherwise; other Python threads run meanwhile.
struct Group {
  explicit Group(const char* name) { nvtxRangePushA(name); }
  ~Group() { nvtxRangePop(); }
  py::gil_scoped_release no_gil;
};

// ---- arguments --------------------------------------------------------------------------------------------------
template <typename T>
T* at_address(uintptr_t p) { return reinterpret_cast<T*>(p); }

bma_tensor describe(const Tensor& t) {
  TORCH_CHECK_VALUE(t.dim() == 4 && t.stride(3) == 1, "innermost dimension must be contiguous");
  bma_tensor r{};
  r.ptr = t.data_ptr();
  r.stride_b = t.stride(0); r.stride_l = t.stride(1); r.stride_h = t.stride(2);
  TORCH_CHECK_TYPE(t.scalar_type() == at::kFloat || t.scalar_type() == at::kBFloat16, "float32 or bfloat16 expected");
  r.dtype = t.scalar_type() == at::kFloat ? BMA_DTYPE_F32 : BMA_DTYPE_BF16;
  return r;
}

bma_attn_args arguments(const Tensor& q, const Tensor& k, const Tensor& v, const OptTensor& key_bias, std::optional<double> scale, int backend) {
  bma_attn_args a{};
  a.q = describe(q); a.k = describe(k); a.v = describe(v);
  a.B = (int32_t)q.size(0); a.N = (int32_t)q.size(1); a.Hq = (int32_t)q.size(2); a.d = (int32_t)q.size(3);
  a.L = (int32_t)k.size(1); a.Hkv = (int32_t)k.size(2);
  a.scale = (float)(scale ? *scale : 1.0 / std::sqrt((double)k.size(3)));
  a.backend = backend;
  if (key_bias) a.key_bias = static_cast<const float*>(key_bias->data_ptr());   // [Hq] float32 on the device
  return a;
}

Tensor bytes_on(const Tensor& like, size_t n) { return at::empty({(int64_t)n}, like.options().dtype(at::kByte).requires_grad(false)); }

struct Route {
  int32_t backend = 0, q_tile = 0, kv_tile = 0;
  size_t f32_bytes = 0;
};
// The kernels of one pass: those of the float32 tensor-core entry points where these cover the request, else what the plan says.
Route route_of(const bma_attn_args& a, bool backward) {
  Route r;
  if (a.q.dtype == BMA_DTYPE_F32 && (r.f32_bytes = lib.bma_attn_f32_workspace_bytes(&a, backward))) {
    r.backend = BMA_BACKEND_SIMT;
    r.q_tile = r.kv_tile = BMA_F32_TILE;
    return r;
  }
  check((backward ? lib.bma_attn_bwd_plan : lib.bma_attn_plan)(&a, &r.backend, &r.q_tile, &r.kv_tile), "bma_attn_plan");
  return r;
}

// (backend, q_tile, kv_tile, workspace bytes of the float32 kernels) of the forward pass and, `backward`, of the backward pass
py::tuple routes(const Tensor& q, const Tensor& k, const Tensor& v, const OptTensor& key_bias, std::optional<double> scale, int backend,
                 bool forward, bool backward) {
  const bma_attn_args a = arguments(q, k, v, key_bias, scale, backend);
  auto one = [&](bool wanted, bool bwd) -> py::object {
    if (!wanted) return py::none();
    const Route r = route_of(a, bwd);
    return py::make_tuple(r.backend, r.q_tile, r.kv_tile, r.f32_bytes);
  };
  return py::make_tuple(one(forward, false), one(backward, true));
}

bool implies_lists(const Tensor& q, const Tensor& k, const Tensor& v, const OptTensor& key_bias, std::optional<double> scale, int backend, uintptr_t spec_at) {
  const bma_attn_args a = arguments(q, k, v, key_bias, scale, backend);
  return lib.bma_attn_fwd_implies_lists(&a, at_address<bma_mask_spec>(spec_at));
}

// ---- block lists ------------------------------------------------------------------------------------------------
// Compiles the lists that `lists` describes by its sizes; returns the tensors that hold them, in the order kv_num, kv_idx,
// full_kv_num, full_kv_idx [, q_num, q_idx, full_q_num, full_q_idx], workspace.  Without `views` the arrays lie in one buffer with the
// workspace.  `flags` are added to those of the mask; the valid lengths are cut at `q_valid`, `k_valid`.
std::vector<Tensor> compile_lists(uintptr_t spec_at, uintptr_t lists_at, int B, int H, bool q_side, bool views, int flags, int q_valid, int k_valid,
                                  int device, uintptr_t stream) {
  bma_mask_spec spec = *at_address<bma_mask_spec>(spec_at);
  bma_block_lists& l = *at_address<bma_block_lists>(lists_at);
  spec.flags |= flags;
  spec.q_valid = std::min(spec.q_valid, q_valid);
  spec.k_valid = std::min(spec.k_valid, k_valid);
  const size_t ws_bytes = lib.bma_mask_compile_workspace_bytes(&spec, B, H, l.NQ, l.NKV);
  const at::TensorOptions on = at::TensorOptions().device(at::kCUDA, (c10::DeviceIndex)device);
  std::vector<Tensor> out;
  uint8_t* ws;
  if (views) {
    const at::TensorOptions i32 = on.dtype(at::kInt);
    auto side = [&](int rows, int cols, int32_t*& num, int32_t*& idx, int32_t*& full_num, int32_t*& full_idx) {
      auto array = [&](at::IntArrayRef shape) {
        out.push_back(at::empty(shape, i32));
        return out.back().data_ptr<int32_t>();
      };
      num = array({l.B, l.H, rows});
      idx = array({l.B, l.H, rows, cols});
      full_num = array({l.B, l.H, rows});
      full_idx = array({l.B, l.H, rows, cols});
    };
    side(l.NQ, l.NKV, l.kv_num, l.kv_idx, l.full_kv_num, l.full_kv_idx);
    if (q_side) side(l.NKV, l.NQ, l.q_num, l.q_idx, l.full_q_num, l.full_q_idx);
    out.push_back(at::empty({(int64_t)std::max<size_t>(ws_bytes, 1)}, on.dtype(at::kByte)));
    ws = out.back().data_ptr<uint8_t>();
  } else {
    auto pad = [](int64_t n) { return (4 * n + 255) / 256 * 256; };   // bytes of n int32, every array on a 256-byte boundary
    const int64_t heads = (int64_t)l.B * l.H, rows = pad(heads * l.NQ), cols = pad(heads * l.NKV), cells = pad(heads * l.NQ * l.NKV);
    const int64_t total = 2 * (rows + cells) + (q_side ? 2 * (cols + cells) : 0);
    out.push_back(at::empty({total + (int64_t)ws_bytes + 1}, on.dtype(at::kByte)));
    uint8_t* at = out.back().data_ptr<uint8_t>();
    auto array = [&](int64_t bytes) {
      int32_t* r = reinterpret_cast<int32_t*>(at);
      at += bytes;
      return r;
    };
    l.kv_num = array(rows); l.kv_idx = array(cells); l.full_kv_num = array(rows); l.full_kv_idx = array(cells);
    if (q_side) { l.q_num = array(cols); l.q_idx = array(cells); l.full_q_num = array(cols); l.full_q_idx = array(cells); }
    ws = at;
  }
  int rc;
  {
    Group group("bma.mask_compile");
    rc = lib.bma_mask_compile(&spec, B, H, &l, ws, ws_bytes, reinterpret_cast<bma_stream_t>(stream));
  }
  check(rc, "bma_mask_compile");
  return out;
}

// ---- attention --------------------------------------------------------------------------------------------------
// `f32_bytes`: workspace of the float32 kernels, 0 for the others; `planes` is that workspace, None where there is no room for it.
std::tuple<Tensor, Tensor> forward(const Tensor& q, const Tensor& k, const Tensor& v, const OptTensor& key_bias, std::optional<double> scale, int backend,
                                   uintptr_t spec_at, uintptr_t lists_at, size_t f32_bytes, const OptTensor& planes, bool bf16_out, uintptr_t stream) {
  bma_attn_args a = arguments(q, k, v, key_bias, scale, backend);
  const bma_mask_spec* spec = at_address<bma_mask_spec>(spec_at);
  const bma_block_lists* lists = at_address<bma_block_lists>(lists_at);
  const at::TensorOptions f32 = q.options().dtype(at::kFloat).requires_grad(false);
  Tensor o = at::empty({a.B, a.N, a.Hq, a.d}, bf16_out ? f32.dtype(at::kBFloat16) : f32), lse = at::empty({a.B, a.Hq, a.N}, f32), ws;
  a.o = describe(o);
  a.lse = lse.data_ptr<float>();
  size_t ws_bytes = 0;
  if (!f32_bytes && lib.bma_attn_fwd_uses_workspace(&a, lists)) ws = bytes_on(q, ws_bytes = lib.bma_attn_fwd_workspace_bytes(&a, lists));
  int rc;
  {
    Group group("bma.fwd");
    const bma_stream_t st = reinterpret_cast<bma_stream_t>(stream);
    if (f32_bytes) rc = lib.bma_attn_fwd_f32(&a, spec, lists, planes ? planes->data_ptr() : nullptr, planes ? f32_bytes : 0, st);
    else rc = lib.bma_attn_fwd_ws(&a, spec, lists, ws_bytes ? ws.data_ptr() : nullptr, ws_bytes, st);
  }
  check(rc, f32_bytes ? "bma_attn_fwd_f32" : "bma_attn_fwd");
  return {o, lse};
}

// (delta, bf16 copy of the cotangent or None)
std::tuple<Tensor, OptTensor> preprocess(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& o, const Tensor& d_o, const OptTensor& key_bias,
                                        std::optional<double> scale, int backend, bool bf16_copy, uintptr_t stream) {
  bma_attn_args a = arguments(q, k, v, key_bias, scale, backend);
  const at::TensorOptions f32 = q.options().dtype(at::kFloat).requires_grad(false);
  Tensor delta = at::empty({a.B, a.Hq, a.N}, f32);
  OptTensor copy;
  if (bf16_copy) copy = at::empty({a.B, a.N, a.Hq, a.d}, f32.dtype(at::kBFloat16));
  a.o = describe(o);
  a.d_o = describe(d_o);
  a.delta = delta.data_ptr<float>();
  int rc;
  {
    Group group("bma.bwd_preprocess");
    rc = lib.bma_attn_bwd_preprocess(&a, copy ? copy->data_ptr() : nullptr, reinterpret_cast<bma_stream_t>(stream));
  }
  check(rc, "bma_attn_bwd_preprocess");
  return {delta, copy};
}

// Bytes of the tensor-core backward: (workspace without hand-over, hand-over of everything, of the largest unit); `visited`: host array of
// visited blocks per list head, 0 where the dS tiles cannot be handed over.
std::tuple<size_t, size_t, size_t> backward_bytes(const Tensor& q, const Tensor& k, const Tensor& v, const OptTensor& key_bias, std::optional<double> scale,
                                                  int backend, uintptr_t lists_at, uintptr_t visited) {
  const bma_attn_args a = arguments(q, k, v, key_bias, scale, backend);
  const bma_block_lists* lists = at_address<bma_block_lists>(lists_at);
  const int64_t* counts = at_address<const int64_t>(visited);
  return {lib.bma_attn_bwd_workspace_bytes(&a), counts ? lib.bma_attn_bwd_scratch_bytes(&a, lists, counts) : 0,
          counts ? lib.bma_attn_bwd_scratch_min_bytes(&a, lists, counts) : 0};
}

// Where `delta` is left out the pass takes it itself, from `d_o` as it came.
std::tuple<Tensor, Tensor, Tensor> backward(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& o, const Tensor& lse, const Tensor& d_o,
                                            OptTensor delta, const OptTensor& key_bias, std::optional<double> scale, int backend, uintptr_t spec_at,
                                            uintptr_t lists_at, size_t f32_bytes, const OptTensor& workspace, size_t ws_bytes, uintptr_t visited,
                                            uintptr_t mid_event, uintptr_t stream) {
  bma_attn_args a = arguments(q, k, v, key_bias, scale, backend);
  const bma_mask_spec* spec = at_address<bma_mask_spec>(spec_at);
  const bma_block_lists* lists = at_address<bma_block_lists>(lists_at);
  Tensor dq = at::empty_like(q), dk = at::empty_like(k), dv = at::empty_like(v);
  a.o = describe(o); a.d_o = describe(d_o);
  const bool own_delta = !delta;
  Tensor copy;
  if (own_delta && !f32_bytes && d_o.scalar_type() != at::kBFloat16) copy = at::empty({a.B, a.N, a.Hq, a.d}, q.options().dtype(at::kBFloat16).requires_grad(false));
  if (own_delta) delta = at::empty({a.B, a.Hq, a.N}, q.options().dtype(at::kFloat).requires_grad(false));
  a.lse = lse.data_ptr<float>(); a.delta = delta->data_ptr<float>();
  a.dq = describe(dq); a.dk = describe(dk); a.dv = describe(dv);
  Tensor small;
  void* ws = workspace ? workspace->data_ptr() : nullptr;
  if (!f32_bytes && !ws) {
    small = bytes_on(q, std::max<size_t>(ws_bytes, 1));
    ws = small.data_ptr();
  }
  int rc;
  {
    Group group("bma.bwd");
    const bma_stream_t st = reinterpret_cast<bma_stream_t>(stream);
    if (f32_bytes) rc = (own_delta ? lib.bma_attn_bwd_f32_o : lib.bma_attn_bwd_f32)(&a, spec, lists, ws, ws ? f32_bytes : 0, st);
    else if (own_delta)
      rc = lib.bma_attn_bwd_o(&a, copy.defined() ? copy.data_ptr() : nullptr, spec, lists, ws, ws_bytes, at_address<const int64_t>(visited), at_address<void>(mid_event), st);
    else rc = lib.bma_attn_bwd(&a, spec, lists, ws, ws_bytes, at_address<const int64_t>(visited), at_address<void>(mid_event), st);
  }
  check(rc, f32_bytes ? "bma_attn_bwd_f32" : "bma_attn_bwd");
  return {dq, dk, dv};
}

// ---- heads and the paged cache ------------------------------------------------------------------------------------
// These check their arguments and find their stream here: a small call takes as long on the host as on the device.
int dtype_of(const Tensor& t, const char* name) {
  TORCH_CHECK_TYPE(t.scalar_type() == at::kFloat || t.scalar_type() == at::kBFloat16, name, " must be float32 or bfloat16, not ", t.scalar_type());
  return t.scalar_type() == at::kFloat ? BMA_DTYPE_F32 : BMA_DTYPE_BF16;
}

// The tensors of a call, which have to lie on the device of the first: looked at when everything else has been.
struct Devices {
  const Tensor* at[16];
  const char* names[16];
  int n = 0;
  void add(const Tensor& t, const char* name) {
    at[n] = &t;
    names[n++] = name;
  }
  void check() const {
    for (int i = 0; i < n; ++i) {
      TORCH_CHECK(at[i]->is_cuda(), names[i], " must be a CUDA tensor; there is no CPU path");
      TORCH_CHECK_VALUE(at[i]->device() == at[0]->device(), names[i], " is on ", at[i]->device().str(), ", not on ", at[0]->device().str());
    }
  }
};

// The device of a call, made current, and its stream there.
struct Place {
  c10::DeviceGuard guard;
  bma_stream_t stream;
  explicit Place(const Tensor& t) : guard(t.device()), stream(c10::impl::VirtualGuardImpl(at::kCUDA).getStream(t.device()).native_handle()) {}
};

// at::empty on the current CUDA device (which Place has made the call's), without the dispatcher: 0.5 us less.
Tensor fresh(at::IntArrayRef sizes, at::ScalarType dtype) {
  return at::detail::empty_generic(sizes, c10::GetAllocator(at::kCUDA), c10::DispatchKeySet(c10::DispatchKey::CUDA), dtype, std::nullopt);
}

bool wants_gradient(std::initializer_list<const Tensor*> tensors) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : tensors)
    if (t && t->requires_grad()) return true;
  return false;
}
// Forward mode hands its tangents along beside the values, and a result without one counts as a constant there: none is dropped in silence.
void no_tangents(std::initializer_list<const Tensor*> tensors, const char* name) {
  for (const Tensor* t : tensors) TORCH_CHECK_VALUE(!t || !t->defined() || !t->_fw_grad(/*level=*/0).defined(), name, " has no derivatives in forward mode");
}
const Tensor* pointer(const OptTensor& t) { return t ? &*t : nullptr; }

// [B, L, H, d] heads; copied only where the components of a head do not lie side by side
Tensor heads_of(const Tensor& t, const char* name) {
  TORCH_CHECK_VALUE(t.dim() == 4, name, " must be [batch, length, heads, components]");
  TORCH_CHECK_VALUE(t.size(0) > 0 && t.size(1) > 0 && t.size(2) > 0 && t.size(3) > 0, name, " is empty");
  TORCH_CHECK_VALUE(t.size(0) <= INT32_MAX && t.size(1) <= INT32_MAX && t.size(2) <= 65535, name, " is too large");
  if (t.stride(3) == 1) return t;
  return t.size(3) == 1 ? t.as_strided(t.sizes(), {t.stride(0), t.stride(1), t.stride(2), 1}) : t.contiguous();
}

bma_rotary rotary_of(Devices& on, int64_t d, const OptTensor& frequencies, int layout, double magnitude, const OptTensor& q_weight, const OptTensor& k_weight,
                     double eps) {
  bma_rotary r{};
  r.layout = layout;
  r.magnitude = (float)magnitude;
  r.eps = (float)eps;
  if (frequencies) {
    TORCH_CHECK_TYPE(frequencies->scalar_type() == at::kDouble, "frequencies must be float64");
    TORCH_CHECK_VALUE(frequencies->dim() == 1 && frequencies->is_contiguous(), "frequencies must be a contiguous vector");
    TORCH_CHECK_VALUE(frequencies->numel() > 0 && 2 * frequencies->numel() <= d, "frequencies must have between 1 and " + std::to_string(d / 2) + " values");
    on.add(*frequencies, "frequencies");
    r.frequencies = frequencies->data_ptr<double>();
    r.dim = (int32_t)(2 * frequencies->numel());
  }
  const Tensor* first = nullptr;
  auto weight = [&](const OptTensor& w, const char* name) -> const void* {
    if (!w) return nullptr;
    r.weight_dtype = dtype_of(*w, name);
    TORCH_CHECK_VALUE(w->dim() == 1 && w->numel() == d && w->is_contiguous(), name, " must be a contiguous vector of " + std::to_string(d) + " values");
    TORCH_CHECK_TYPE(!first || first->scalar_type() == w->scalar_type(), "q_weight and k_weight must share a dtype");
    on.add(*w, name);
    first = &*w;
    return w->data_ptr();
  };
  r.q_weight = weight(q_weight, "q_weight");
  r.k_weight = weight(k_weight, "k_weight");
  TORCH_CHECK_VALUE(!first || eps >= 0, "eps must not be negative");
  return r;
}

bma_rotate_args rotate_args(Devices& on, const Tensor& q, const OptTensor& k, const OptTensor& positions, const OptTensor& frequencies, int layout, double magnitude,
                            const OptTensor& q_weight, const OptTensor& k_weight, double eps) {
  bma_rotate_args a{};
  a.B = (int32_t)q.size(0); a.L = (int32_t)q.size(1); a.Hq = (int32_t)q.size(2); a.d = (int32_t)q.size(3);
  dtype_of(q, "q");
  TORCH_CHECK_VALUE(a.d <= 256, "heads of at most 256 components");
  if (k) {
    TORCH_CHECK_VALUE(k->size(0) == a.B && k->size(1) == a.L && k->size(3) == a.d, "k must have the batch, length and components of q");
    TORCH_CHECK_TYPE(k->scalar_type() == q.scalar_type(), "q and k must share a dtype");
    a.Hkv = (int32_t)k->size(2);
  }
  TORCH_CHECK_VALUE(k || !k_weight, "k_weight without k");
  TORCH_CHECK_VALUE(frequencies || q_weight || k_weight, "neither frequencies nor weights: there is nothing to do");
  on.add(q, "q");
  if (k) on.add(*k, "k");
  a.rotary = rotary_of(on, a.d, frequencies, layout, magnitude, q_weight, k_weight, eps);
  if (positions) {
    const Tensor& p = *positions;
    TORCH_CHECK_TYPE(p.scalar_type() == at::kInt || p.scalar_type() == at::kLong, "positions must be int32 or int64");
    TORCH_CHECK_VALUE((p.dim() == 1 && p.size(0) == a.L) || (p.dim() == 2 && p.size(0) == a.B && p.size(1) == a.L), "positions must be [length] or [batch, length]");
    on.add(p, "positions");
    a.positions = p.data_ptr();
    a.position_bytes = p.scalar_type() == at::kInt ? 4 : 8;
    a.position_stride_b = p.dim() == 2 ? p.stride(0) : 0;
    a.position_stride_l = p.stride(p.dim() - 1);
  }
  return a;
}

struct Rotation {
  OptTensor positions, frequencies;
  int layout;
  double magnitude;
  OptTensor q_weight, k_weight;
  double eps;
};

// (both ways here come from Python and hold its lock)
std::tuple<Tensor, OptTensor> rotate_forward(const Tensor& q_in, const OptTensor& k_in, const Rotation& r) {
  const Tensor q = heads_of(q_in, "q");
  OptTensor k, k_out;
  if (k_in) k = heads_of(*k_in, "k");
  Devices on;
  bma_rotate_args a = rotate_args(on, q, k, r.positions, r.frequencies, r.layout, r.magnitude, r.q_weight, r.k_weight, r.eps);
  on.check();
  const Place place(q);
  Tensor q_out = fresh(q.sizes(), q.scalar_type());
  a.q = describe(q); a.q_out = describe(q_out);
  if (k) {
    k_out = fresh(k->sizes(), k->scalar_type());
    a.k = describe(*k); a.k_out = describe(*k_out);
  }
  int rc;
  {
    Group group("bma.rotate");
    rc = lib.bma_rotate(&a, place.stream);
  }
  check(rc, "bma_rotate");
  return {q_out, k_out};
}

// Gradients of (q, k, q_weight, k_weight), as far as they are there.  Runs on a thread of the autograd engine, without Python.
std::tuple<Tensor, OptTensor, OptTensor, OptTensor> rotate_backward(const Tensor& q_in, const OptTensor& k_in, const Rotation& r, const Tensor& g_q_in, const OptTensor& g_k_in) {
  const Tensor q = heads_of(q_in, "q"), g_q = heads_of(g_q_in, "the cotangent of q");
  OptTensor k, g_k, dk, dqw, dkw;
  if (k_in) {
    k = heads_of(*k_in, "k");
    g_k = heads_of(*g_k_in, "the cotangent of k");
  }
  Devices on;
  bma_rotate_args a = rotate_args(on, q, k, r.positions, r.frequencies, r.layout, r.magnitude, r.q_weight, r.k_weight, r.eps);
  TORCH_CHECK_VALUE(g_q.sizes() == q.sizes() && (!k || g_k->sizes() == k->sizes()), "the cotangents must have the shapes of the results");
  TORCH_CHECK_TYPE(g_q.scalar_type() == q.scalar_type() && (!k || g_k->scalar_type() == q.scalar_type()), "the cotangents must have the dtype of the results");
  on.add(g_q, "the cotangent of q");
  if (k) on.add(*g_k, "the cotangent of k");
  on.check();
  const Place place(q);
  Tensor dq = fresh(q.sizes(), q.scalar_type());
  a.q = describe(q); a.q_out = describe(g_q); a.dq = describe(dq);
  if (k) {
    dk = fresh(k->sizes(), k->scalar_type());
    a.k = describe(*k); a.k_out = describe(*g_k); a.dk = describe(*dk);
  }
  if (r.q_weight) a.dq_weight = (dqw = fresh(r.q_weight->sizes(), r.q_weight->scalar_type()))->data_ptr();
  if (r.k_weight) a.dk_weight = (dkw = fresh(r.k_weight->sizes(), r.k_weight->scalar_type()))->data_ptr();
  const size_t ws_bytes = lib.bma_rotate_bwd_workspace_bytes(&a);
  Tensor ws;
  if (ws_bytes) ws = fresh({(int64_t)ws_bytes}, at::kByte);
  nvtxRangePushA("bma.rotate_bwd");
  const int rc = lib.bma_rotate_bwd(&a, ws_bytes ? ws.data_ptr() : nullptr, ws_bytes, place.stream);
  nvtxRangePop();
  TORCH_CHECK(rc == BMA_OK, "bma_rotate_bwd: status ", std::to_string(rc), ": ", lib.bma_error_string(rc));
  return {dq, dk, dqw, dkw};
}

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
struct RotateNode : torch::autograd::Function<RotateNode> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const OptTensor& k, const OptTensor& positions, const OptTensor& frequencies, int64_t layout,
                               double magnitude, const OptTensor& q_weight, const OptTensor& k_weight, double eps) {
    at::AutoDispatchBelowADInplaceOrView below;
    const auto or_none = [](const OptTensor& t) { return t ? *t : Tensor(); };
    auto [q_out, k_out] = rotate_forward(q, k, {positions, frequencies, (int)layout, magnitude, q_weight, k_weight, eps});
    // a rotation alone is undone without its input: only the shape, the dtype and the device are kept
    ctx->save_for_backward({q_weight ? q : Tensor(), k && k_weight ? *k : Tensor(), or_none(positions), or_none(frequencies), or_none(q_weight), or_none(k_weight)});
    ctx->saved_data["layout"] = layout;
    ctx->saved_data["magnitude"] = magnitude;
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["q"] = at::empty({0}, q.options().requires_grad(false));
    ctx->saved_data["q_sizes"] = q.sizes().vec();
    if (k) ctx->saved_data["k_sizes"] = k->sizes().vec();
    ctx->set_materialize_grads(false);
    variable_list out{q_out};
    if (k_out) out.push_back(*k_out);
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    TORCH_CHECK(!at::GradMode::is_enabled(), "rotate_heads has no second derivatives: do not ask for create_graph");
    for (const Tensor& g : grads) no_tangents({&g}, "the backward pass of rotate_heads");
    const variable_list saved = ctx->get_saved_variables();
    const auto optional = [](const Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); };
    const Rotation r{optional(saved[2]), optional(saved[3]), (int)ctx->saved_data["layout"].toInt(), ctx->saved_data["magnitude"].toDouble(), optional(saved[4]),
                     optional(saved[5]), ctx->saved_data["eps"].toDouble()};
    const bool keys = grads.size() > 1;
    const Tensor like = ctx->saved_data["q"].toTensor();
    // an undefined cotangent stands for zeros
    const Tensor g_q = grads[0].defined() ? grads[0] : at::zeros(ctx->saved_data["q_sizes"].toIntVector(), like.options());
    OptTensor g_k;
    if (keys) g_k = grads[1].defined() ? grads[1] : at::zeros(ctx->saved_data["k_sizes"].toIntVector(), like.options());
    const auto [dq, dk, dqw, dkw] = rotate_backward(saved[0].defined() ? saved[0] : g_q, keys ? (saved[1].defined() ? OptTensor(saved[1]) : g_k) : OptTensor(), r, g_q, g_k);
    const auto or_none = [](const OptTensor& t) { return t ? *t : Tensor(); };
    return {dq, or_none(dk), Tensor(), Tensor(), Tensor(), Tensor(), or_none(dqw), or_none(dkw), Tensor()};
  }
};

std::tuple<Tensor, OptTensor> rotate(const Tensor& q, const OptTensor& k, const OptTensor& positions, const OptTensor& frequencies, int layout, double magnitude,
                                     const OptTensor& q_weight, const OptTensor& k_weight, double eps) {
  no_tangents({&q, pointer(k), pointer(q_weight), pointer(k_weight), pointer(frequencies)}, "rotate_heads");
  TORCH_CHECK_VALUE(!wants_gradient({pointer(frequencies)}), "rotate_heads is not differentiable in frequencies: detach them");
  if (!wants_gradient({&q, pointer(k), pointer(q_weight), pointer(k_weight)})) return rotate_forward(q, k, {positions, frequencies, layout, magnitude, q_weight, k_weight, eps});
  const variable_list out = RotateNode::apply(q, k, positions, frequencies, (int64_t)layout, magnitude, q_weight, k_weight, eps);
  return {out[0], out.size() > 1 ? OptTensor(out[1]) : OptTensor()};
}

bma_paged_cache cache_of(Devices& on, const Tensor& k, const Tensor& v, const Tensor& table, const OptTensor& k_scale, const OptTensor& v_scale) {
  bma_paged_cache c{};
  on.add(k, "the pages of keys");
  on.add(v, "the pages of values");
  on.add(table, "the page table");
  TORCH_CHECK_VALUE(k.dim() == 4 && v.dim() == 4, "the pages must be [pages, page_size, heads, components]");
  TORCH_CHECK_VALUE(k.sizes() == v.sizes() && k.strides() == v.strides(), "the pages of keys and of values must have the same shape and strides");
  TORCH_CHECK_TYPE(k.scalar_type() == v.scalar_type(), "the pages of keys and of values must share a dtype");
  TORCH_CHECK_VALUE(k.numel() > 0, "the pages are empty");
  TORCH_CHECK_VALUE(k.stride(3) == 1, "the components of a head must lie side by side in a page");
  TORCH_CHECK_VALUE(k.size(0) <= INT32_MAX && k.size(1) <= INT32_MAX && k.size(2) <= 65535, "too many pages, slots or heads");
  c.pages = (int32_t)k.size(0); c.page_size = (int32_t)k.size(1); c.Hkv = (int32_t)k.size(2); c.d = (int32_t)std::min<int64_t>(k.size(3), 1 << 20);
  c.stride_page = k.stride(0); c.stride_slot = k.stride(1); c.stride_head = k.stride(2);
  int64_t unit = 16;                     // values of 16 bytes
  if (k.scalar_type() == at::kByte) {
    c.dtype = BMA_DTYPE_MXFP4;
    c.d *= 2;
    TORCH_CHECK_VALUE(k_scale && v_scale, "a 4-bit cache has k_scale and v_scale");
    TORCH_CHECK_VALUE(c.d % 32 == 0 && c.d <= 128, "a 4-bit cache has heads of 32, 64, 96 or 128 components");
    for (const OptTensor* s : {&k_scale, &v_scale}) {
      const Tensor& t = **s;
      TORCH_CHECK_TYPE(t.scalar_type() == at::kByte, "the scales must be uint8");
      TORCH_CHECK_VALUE(t.dim() == 4 && t.size(0) == k.size(0) && t.size(1) == k.size(1) && t.size(2) == k.size(2) && t.size(3) * 32 == c.d,
                        "the scales must be [pages, page_size, heads, components / 32]");
      TORCH_CHECK_VALUE(t.stride(3) == 1 || t.size(3) == 1, "the scales of a head must lie side by side");
      TORCH_CHECK_VALUE(t.strides() == k_scale->strides(), "the scales of keys and of values must have the same strides");
      on.add(t, "the scales");
    }
    c.k_scale = k_scale->data_ptr<uint8_t>(); c.v_scale = v_scale->data_ptr<uint8_t>();
    c.scale_stride_page = k_scale->stride(0); c.scale_stride_slot = k_scale->stride(1); c.scale_stride_head = k_scale->stride(2);
  } else {
    c.dtype = dtype_of(k, "pages (of other than 4-bit caches)");
    unit = c.dtype == BMA_DTYPE_F32 ? 4 : 8;
    TORCH_CHECK_VALUE(!k_scale && !v_scale, "only a 4-bit cache (uint8 pages) has scales");
    TORCH_CHECK_VALUE(c.d % 8 == 0 && c.d <= 128, "a cache has heads of a multiple of 8 components, at most 128");
  }
  TORCH_CHECK_VALUE((reinterpret_cast<uintptr_t>(k.data_ptr()) | reinterpret_cast<uintptr_t>(v.data_ptr())) % 16 == 0 && c.stride_page % unit == 0 &&
                        c.stride_slot % unit == 0 && c.stride_head % unit == 0,
                    "every head of every slot must start on 16 bytes");
  c.k = k.data_ptr(); c.v = v.data_ptr();
  TORCH_CHECK_TYPE(table.scalar_type() == at::kInt, "the page table must be int32");
  TORCH_CHECK_VALUE(table.dim() == 2 && table.numel() > 0 && (table.stride(1) == 1 || table.size(1) == 1), "the page table must be [batch, width], its rows contiguous");
  TORCH_CHECK_VALUE(table.size(0) <= 65535, "a batch of at most 65535 sequences");
  TORCH_CHECK_VALUE(table.size(1) * (int64_t)c.page_size < (1ll << 31) - 4096, "the page table covers too many positions");
  c.page_table = table.data_ptr<int32_t>();
  c.table_stride = table.stride(0);
  c.B = (int32_t)table.size(0); c.width = (int32_t)table.size(1);
  return c;
}

const int32_t* counts_of(Devices& on, const Tensor& t, const bma_paged_cache& c, const char* name) {
  TORCH_CHECK_TYPE(t.scalar_type() == at::kInt, name, " must be int32");
  TORCH_CHECK_VALUE(t.dim() == 1 && t.size(0) == c.B && t.is_contiguous(), name, " must be a contiguous vector with a value for each row of the page table");
  on.add(t, name);
  return t.data_ptr<int32_t>();
}

void fits_cache(Devices& on, const Tensor& t, const bma_paged_cache& c, int64_t heads, const char* name) {
  TORCH_CHECK_VALUE(t.size(0) == c.B && t.size(3) == c.d && (heads < 0 || t.size(2) == heads), name, " does not fit the cache");
  const int dtype = dtype_of(t, name);
  TORCH_CHECK_TYPE(c.dtype == BMA_DTYPE_MXFP4 || dtype == c.dtype, name, " must have the dtype of the cache");
  on.add(t, name);
}

OptTensor append(const Tensor& pages_k, const Tensor& pages_v, const Tensor& table, const OptTensor& k_scale, const OptTensor& v_scale, const Tensor& k_in,
                 const Tensor& v_in, const Tensor& lengths, const OptTensor& new_lengths, const OptTensor& q_in, const OptTensor& frequencies, int layout, double magnitude,
                 const OptTensor& q_weight, const OptTensor& k_weight, double eps) {
  no_tangents({&k_in, &v_in, pointer(q_in), pointer(q_weight), pointer(k_weight), pointer(frequencies), &pages_k, &pages_v}, "append_kv");
  TORCH_CHECK_VALUE(!wants_gradient({&k_in, &v_in, pointer(q_in), pointer(q_weight), pointer(k_weight), pointer(frequencies), &pages_k, &pages_v}),
                    "append_kv is not differentiable: call it under torch.no_grad()");
  Devices on;
  const bma_paged_cache c = cache_of(on, pages_k, pages_v, table, k_scale, v_scale);
  const Tensor k = heads_of(k_in, "k"), v = heads_of(v_in, "v");
  OptTensor q, q_out;
  if (q_in) q = heads_of(*q_in, "q");
  bma_append_args a{};
  a.T = (int32_t)k.size(1);
  fits_cache(on, k, c, c.Hkv, "k");
  fits_cache(on, v, c, c.Hkv, "v");
  TORCH_CHECK_VALUE(v.size(1) == a.T && (!q || q->size(1) == a.T), "q, k and v must have the same number of tokens");
  TORCH_CHECK_TYPE(v.scalar_type() == k.scalar_type() && (!q || q->scalar_type() == k.scalar_type()), "q, k and v must share a dtype");
  TORCH_CHECK_VALUE(q || !q_weight, "q_weight without q");
  TORCH_CHECK_VALUE(!q || frequencies || q_weight, "neither frequencies nor q_weight: there is nothing to do with q");
  a.lengths = counts_of(on, lengths, c, "lengths");
  if (new_lengths) a.new_lengths = counts_of(on, *new_lengths, c, "new_lengths");
  a.rotary = rotary_of(on, c.d, frequencies, layout, magnitude, q_weight, k_weight, eps);
  if (q) fits_cache(on, *q, c, -1, "q");
  on.check();
  const Place place(pages_k);
  a.k = describe(k); a.v = describe(v);
  if (q) {
    q_out = fresh(q->sizes(), q->scalar_type());
    a.Hq = (int32_t)q->size(2);
    a.q = describe(*q); a.q_out = describe(*q_out);
  }
  int rc;
  {
    Group group("bma.append_kv");
    rc = lib.bma_append_kv(&c, &a, place.stream);
  }
  check(rc, "bma_append_kv");
  // a graph that has saved pages has to notice (tensors made in inference mode have no version, and no graph)
  for (const Tensor* t : {&pages_k, &pages_v, pointer(k_scale), pointer(v_scale)})
    if (t && !t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
  return q_out;
}

std::tuple<Tensor, Tensor> read_pages(const Tensor& pages_k, const Tensor& pages_v, const Tensor& table, const OptTensor& k_scale, const OptTensor& v_scale,
                                const Tensor& lengths, int64_t L) {
  Devices on;
  const bma_paged_cache c = cache_of(on, pages_k, pages_v, table, k_scale, v_scale);
  no_tangents({&pages_k, &pages_v}, "read_kv");
  TORCH_CHECK_VALUE(!wants_gradient({&pages_k, &pages_v}), "read_kv is not differentiable: call it under torch.no_grad()");
  TORCH_CHECK_VALUE(L > 0 && L < (1ll << 31) - 4096, "max_length must be positive, and below 2^31 - 4096");
  const int32_t* at_lengths = counts_of(on, lengths, c, "lengths");
  on.check();
  const Place place(pages_k);
  const at::ScalarType dtype = c.dtype == BMA_DTYPE_F32 ? at::kFloat : at::kBFloat16;
  Tensor k = fresh({c.B, L, c.Hkv, c.d}, dtype), v = fresh({c.B, L, c.Hkv, c.d}, dtype);
  const bma_tensor dk = describe(k), dv = describe(v);
  int rc;
  {
    Group group("bma.read_kv");
    rc = lib.bma_read_kv(&c, at_lengths, (int32_t)L, &dk, &dv, place.stream);
  }
  check(rc, "bma_read_kv");
  return {k, v};
}

std::tuple<Tensor, OptTensor> paged(const Tensor& pages_k, const Tensor& pages_v, const Tensor& table, const OptTensor& k_scale, const OptTensor& v_scale,
                                    const Tensor& q_in, const Tensor& lengths, const OptTensor& new_lengths, std::optional<double> scale,
                                    std::optional<int64_t> window, bool bf16_out, bool with_lse) {
  no_tangents({&q_in, &pages_k, &pages_v}, "paged_attention");
  TORCH_CHECK_VALUE(!wants_gradient({&q_in, &pages_k, &pages_v}), "paged_attention is not differentiable: call it under torch.no_grad()");
  Devices on;
  const bma_paged_cache c = cache_of(on, pages_k, pages_v, table, k_scale, v_scale);
  Tensor q = heads_of(q_in, "q");
  const int64_t bytes = q.element_size();
  if (reinterpret_cast<uintptr_t>(q.data_ptr()) % 16 || q.stride(0) * bytes % 16 || q.stride(1) * bytes % 16 || q.stride(2) * bytes % 16) q = q.clone(at::MemoryFormat::Contiguous);
  fits_cache(on, q, c, -1, "q");
  TORCH_CHECK_TYPE(c.dtype != BMA_DTYPE_MXFP4 || q.scalar_type() == at::kBFloat16, "q must be bfloat16 for a 4-bit cache");
  TORCH_CHECK_VALUE(q.size(2) % c.Hkv == 0, "the heads of the cache must divide those of q");
  TORCH_CHECK_VALUE(!window || (*window >= 0 && *window <= INT32_MAX), "window must not be negative");
  bma_paged_attn_args a{};
  a.T = (int32_t)q.size(1); a.Hq = (int32_t)q.size(2);
  a.lengths = counts_of(on, lengths, c, "lengths");
  if (new_lengths) a.new_lengths = counts_of(on, *new_lengths, c, "new_lengths");
  a.scale = (float)(scale ? *scale : 1.0 / std::sqrt((double)c.d));
  a.window = window ? (int32_t)*window : -1;
  on.check();
  const Place place(pages_k);
  Tensor o = fresh(q.sizes(), bf16_out ? at::kBFloat16 : at::kFloat);
  OptTensor lse;
  if (with_lse) lse = fresh({c.B, a.Hq, a.T}, at::kFloat);
  a.q = describe(q); a.o = describe(o);
  a.lse = lse ? lse->data_ptr<float>() : nullptr;
  const size_t ws_bytes = lib.bma_paged_attn_workspace_bytes(&c, &a);
  Tensor ws;
  if (ws_bytes) ws = fresh({(int64_t)ws_bytes}, at::kByte);
  int rc;
  {
    Group group("bma.paged_attn");
    rc = lib.bma_paged_attn(&c, &a, ws_bytes ? ws.data_ptr() : nullptr, ws_bytes, place.stream);
  }
  check(rc, "bma_paged_attn");
  return {o, lse};
}

}  // namespace

PYBIND11_MODULE(_host, m) {
  m.attr("torch_version") = BMA_TORCH_VERSION;   // the one whose headers this was built with
  m.def("bind", &bind);
  m.def("routes", torch::wrap_pybind_function(routes));
  m.def("implies_lists", torch::wrap_pybind_function(implies_lists));
  m.def("compile_lists", torch::wrap_pybind_function(compile_lists));
  m.def("forward", torch::wrap_pybind_function(forward));
  m.def("preprocess", torch::wrap_pybind_function(preprocess));
  m.def("backward_bytes", torch::wrap_pybind_function(backward_bytes));
  m.def("backward", torch::wrap_pybind_function(backward));
  m.def("rotate", torch::wrap_pybind_function(rotate));
  m.def("append", torch::wrap_pybind_function(append));
  m.def("read", torch::wrap_pybind_function(read_pages));
  m.def("paged", torch::wrap_pybind_function(paged));
}
