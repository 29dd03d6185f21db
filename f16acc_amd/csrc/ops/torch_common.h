// What the operators' torch sides share: argument checks, allocation, the bias's gradient.
#pragma once

#include <ATen/MemoryOverlap.h>
#include <c10/core/AutogradState.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/extension.h>
#include <torch/version.h>

#include <initializer_list>
#include <tuple>
#include <vector>

#include "f16acc_ops.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
typedef std::optional<Tensor> Maybe;

constexpr int64_t kBlock = 128;
constexpr auto kF8 = at::kFloat8_e4m3fn;

#define REQUIRE(cond, ...) TORCH_CHECK_VALUE(cond, __VA_ARGS__)

int64_t up(int64_t v, int64_t m) { return (v + m - 1) / m * m; }
int64_t blocks(int64_t v) { return (v + kBlock - 1) / kBlock; }

bool is_type(at::ScalarType t) { return t == at::kHalf || t == at::kBFloat16 || t == at::kFloat; }
int type_of(const Tensor& t) {
  return t.scalar_type() == at::kHalf ? F16ACC_TYPE_F16
         : t.scalar_type() == at::kBFloat16 ? F16ACC_TYPE_BF16 : F16ACC_TYPE_F32;
}

// Whether torch records the calls (torch.jit.trace, make_fx and export) or runs them on
// stand-ins (fake and functional tensors, torch.func's transforms).  The kernels write
// through pointers, which none of these sees: what it replays would hold the allocation
// alone and return uninitialised memory.
bool recorded() {
  using Modes = c10::impl::TorchDispatchModeTLS;
  using Key = c10::impl::TorchDispatchModeKey;
  if (torch::jit::tracer::isTracing()) return true;
  const c10::DispatchKeySet in = c10::impl::tls_local_dispatch_key_set().included_;
  if (in.has(c10::DispatchKey::FuncTorchDynamicLayerFrontMode) || in.has(c10::DispatchKey::PreDispatch)) return true;
  return Modes::any_modes_set() &&
         (Modes::get_mode(Key::FAKE) || Modes::get_mode(Key::PROXY) || Modes::get_mode(Key::FUNCTIONAL));
}

bool has_tangent(const Tensor& t) { return t.defined() && t._fw_grad(0).defined(); }

// Refuses a call whose result torch would take for something that it is not.
void check_call(const char* name, std::initializer_list<const Tensor*> tensors) {
  TORCH_CHECK_NOT_IMPLEMENTED(!recorded(), name,
                              " cannot be traced: its kernels write through pointers, which no trace records");
  if (c10::AutogradState::get_tls_state().get_fw_grad_mode())
    for (const Tensor* t : tensors)
      TORCH_CHECK_NOT_IMPLEMENTED(!t || !has_tangent(*t), name, " has no forward-mode derivative");
}

// A tensor that is nothing but strided memory: no wrapper around another, no lazily negated view.
void check_plain(const char* name, const Tensor& t) {
  using Key = c10::DispatchKey;
  static const uint64_t allowed = c10::DispatchKeySet({Key::CUDA, Key::HIP, Key::ADInplaceOrView, Key::AutogradCUDA,
                                                       Key::AutogradHIP, Key::AutocastCUDA})
                                      .raw_repr();
  REQUIRE((t.key_set().raw_repr() & ~allowed) == 0 && t.layout() == at::kStrided, name,
          " needs plain strided tensors, got one with ", t.key_set());
}
void check_device(const char* name, const Tensor& t, const Tensor& u) {
  REQUIRE(t.is_cuda() && u.device() == t.device(), name, " needs tensors on one GPU");
  check_plain(name, u);
}
void check_float(const char* name, const Tensor& t) {
  check_device(name, t, t);
  REQUIRE(is_type(t.scalar_type()), name, " needs torch.float16, bfloat16 or float32, not ", t.scalar_type());
}
const Tensor* maybe(const Maybe& t) { return t ? &*t : nullptr; }

// A gradient that autograd hands over, as plain memory.
Tensor check_grad(const char* name, const Tensor& grad) {
  check_call(name, {&grad});
  const Tensor g = grad.resolve_neg();  // (torch may negate lazily what came through complex numbers)
  check_plain(name, g);
  return g;
}

// The device of a tensor made current, and its current stream.
struct On {
  c10::DeviceGuard guard;
  void* stream;
  explicit On(const Tensor& t)
      : guard(t.device()), stream(c10::hip::getCurrentHIPStream(t.device().index()).stream()) {}
};

void check_rc(int rc) {
  REQUIRE(rc != F16ACC_OPS_E_ARG, f16acc_ops_strerror(rc));
  TORCH_CHECK(rc == 0, f16acc_ops_strerror(rc));
}

Tensor empty(at::IntArrayRef sizes, const Tensor& like, at::ScalarType t) {
  return at::empty(sizes, like.options().dtype(t).requires_grad(false));
}

uint8_t* bytes(const Tensor& t) { return t.defined() ? (uint8_t*)t.data_ptr() : nullptr; }
float* floats(const Tensor& t) { return t.defined() ? (float*)t.data_ptr() : nullptr; }
const void* data(const Maybe& t) { return t && t->defined() ? t->const_data_ptr() : nullptr; }

// t as [rows, last dimension]: a view, or a copy where its leading dimensions do not merge.
Tensor rows_of(const Tensor& t) {
  if (t.dim() == 2) return t;
  const int64_t last = t.size(-1);
  int64_t rows = 1;
  for (int64_t i = 0; i + 1 < t.dim(); ++i) rows *= t.size(i);
  return t.reshape({rows, last});
}

std::vector<int64_t> with_last(const Tensor& t, int64_t last) {
  std::vector<int64_t> s(t.sizes().begin(), t.sizes().end());
  s.back() = last;
  return s;
}

// The products address a tile's rows by 31-bit offsets: rows of an operand, and of its scales, may be
// this many bytes apart.  What lies further apart is copied.
constexpr int64_t kMaxRow = 1 << 22;

// An 8- or 4-bit operand and the bytes between its rows.
struct Operand {
  Tensor q;
  int64_t ld;
};

// The gradient of a bias.  (Not torch's sum: recorded in a graph, it clears its counters by a
// node that replays do not run right, and was wrong from the second replay on.)
Tensor column_sums(const Tensor& dy) {
  const int64_t M = dy.size(0), N = dy.size(1);
  const size_t n = f16acc_column_sums_workspace(M, N);
  Tensor ws, out = empty({N}, dy, dy.scalar_type());
  if (n) ws = empty({(int64_t)n}, dy, at::kByte);
  const On on(dy);
  check_rc(f16acc_column_sums(dy.const_data_ptr(), type_of(dy), M, N, dy.stride(0), dy.stride(1), out.data_ptr(),
                              bytes(ws), n, on.stream));
  return out;
}

void first_derivative_only() {
  TORCH_CHECK(!c10::GradMode::is_enabled(), "f16acc: there is no second derivative (create_graph)");
}

}  // namespace
