// What the operators' torch sides share: argument checks, the call into the kernels' library on the current stream, and what
// autograd nodes refuse. Each file that includes this has its own entries of that library, and its own `bound`.
#pragma once
#include <ATen/ATen.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/DeviceGuard.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

#include <algorithm>
#include <atomic>
#include <sstream>
#include <string>
#include <vector>

#include "policy_sizes.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

bool bound = false;  // whether the entries are there

#define POL "nablaengine_amd.policy: "
#define CHECK_TYPE(cond, ...) TORCH_CHECK_TYPE(cond, POL, __VA_ARGS__)
#define CHECK_VALUE(cond, ...) TORCH_CHECK_VALUE(cond, POL, __VA_ARGS__)

// what a message says of a tensor
std::string described(const Tensor& x) {
  std::ostringstream s;
  s << x.scalar_type() << " " << x.sizes() << " with strides " << x.strides() << " on " << x.device();
  return s.str();
}

int type_of(const Tensor& x) {
  switch (x.scalar_type()) {
    case at::kFloat: return 0;
    case at::kBFloat16: return 1;
    case at::kHalf: return 2;
    default: return -1;
  }
}
void check_device(const char* name, const Tensor& x, const Tensor& like) {
  CHECK_TYPE(x.defined() && x.device().type() == at::kCUDA, name, " must be a torch.Tensor on a ROCm device, got ",
             x.defined() ? x.device().str() : "none");
  CHECK_TYPE(x.device() == like.device(), name, " is on ", x.device(), ", the first tensor on ", like.device());
}
// on `like`'s device, of that type and shape
void check_as(const char* name, const Tensor& x, const Tensor& like, at::ScalarType type, at::IntArrayRef shape) {
  check_device(name, x, like);
  CHECK_TYPE(x.scalar_type() == type && x.sizes() == shape, name, ": expected ", type, " ", shape, ", got ", described(x));
}

void check_bound() {
  TORCH_CHECK(bound, POL "the kernels' library is not loaded (call nablaengine_amd.torch_ffi.init()), or was built before this operator");
}
// the kernels are built for one architecture: asked once a device
void check_arch(int device) {
  constexpr int MOST = 64;
  static std::atomic<bool> known[MOST];
  if (device < MOST && known[device].load(std::memory_order_relaxed)) return;
  hipDeviceProp_t p;
  TORCH_CHECK(hipGetDeviceProperties(&p, device) == hipSuccess, POL "no properties of device ", device);
  TORCH_CHECK(std::string(p.gcnArchName).rfind("gfx950", 0) == 0, POL "cuda:", device, " is ", p.gcnArchName,
              "; the library holds gfx950 code only");
  if (device < MOST) known[device].store(true, std::memory_order_relaxed);
}

// A library call on x's device and its current stream; a nonzero return is a RuntimeError naming `what`.
template <typename F>
void call(const char* what, const Tensor& x, F f) {
  check_bound();
  check_arch(x.device().index());
  const c10::DeviceGuard guard(x.device());
  const int rc = f(c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(x.device().index()).stream());
  TORCH_CHECK(rc == 0, POL, what, " failed (HIP error ", rc, ")");
}
Tensor work_of(const Tensor& x, long long bytes) { return at::empty({bytes}, x.options().dtype(at::kByte)); }
const void* in(const OptTensor& x) { return x && x->defined() ? x->data_ptr() : nullptr; }

// Elements from row to row of x seen as rows of its last dimension, or -1: its rows' elements are not neighbours, or its
// rows are not evenly spaced.
int64_t row_stride(const Tensor& x) {
  const int64_t d = x.dim(), n = x.size(d - 1);
  if (x.numel() == 0) return n;
  if (n > 1 && x.stride(d - 1) != 1) return -1;
  int64_t stride = n, size = 0;  // of the last dimension seen that has several rows
  for (int64_t i = d - 2; i >= 0; --i) {
    if (x.size(i) == 1) continue;
    if (size == 0) stride = x.stride(i), size = x.size(i);
    else if (x.stride(i) == stride * size) size *= x.size(i);
    else return -1;
  }
  return stride;
}

// attention's heads
struct Heads { int type, heads, kv, dim; };
// q (.., heads, dim), k and v of `dims` dimensions ending in (kv_heads, dim)
Heads heads_checks(const Tensor& q, const Tensor& k, const Tensor& v, int64_t dims) {
  check_device("q", q, q);
  CHECK_TYPE((q.scalar_type() == at::kBFloat16 || q.scalar_type() == at::kHalf) && q.dim() == 3,
             "q: expected bfloat16 or float16 of 3 dimensions, got ", described(q));
  check_device("k", k, q);
  CHECK_TYPE(k.scalar_type() == q.scalar_type() && k.dim() == dims, "k: expected ", q.scalar_type(), " of ", dims,
             " dimensions, got ", described(k));
  check_as("v", v, q, q.scalar_type(), k.sizes());
  const int64_t heads = q.size(1), dim = q.size(2), kv = k.size(-2);
  CHECK_TYPE(k.size(-1) == dim && dim % 8 == 0 && dim >= 8 && dim <= 128,
             "q and k need heads of one size, a multiple of 8 up to 128, got ", dim, " and ", k.size(-1));
  CHECK_TYPE(kv >= 1 && heads >= 1 && heads % kv == 0 && heads < 1 << 20, "q's heads must be a multiple of k's, got ",
             heads, " and ", kv);
  for (const auto& [name, x] : {std::pair<const char*, const Tensor&>{"q", q}, {"k", k}, {"v", v}})
    CHECK_TYPE(x.numel() == 0 || x.stride(-1) == 1, name, ": a head's elements must be neighbours, got ", described(x));
  return {type_of(q), (int)heads, (int)kv, (int)dim};
}

int sequences_checks(const Tensor& q, const Tensor& k, const Tensor& starts_q, const Tensor& starts_k, const Heads& h) {
  for (const auto& [name, x] : {std::pair<const char*, const Tensor&>{"starts_q", starts_q}, {"starts_k", starts_k}}) {
    check_device(name, x, q);
    CHECK_TYPE(x.scalar_type() == at::kInt && x.dim() == 1 && x.is_contiguous() && x.numel() >= 1 &&
                   x.numel() == starts_q.numel(),
               name, ": expected contiguous int32 offsets, one more than sequences in both, got ", described(x));
  }
  const int64_t seqs = starts_q.numel() - 1, most = 1 << 30;
  CHECK_VALUE(q.size(0) < most && k.size(0) < most && seqs < most &&
                  pol::attention_sizes(h.heads, h.kv, (int)seqs, (int)q.size(0), (int)k.size(0)),
              q.size(0), " queries of ", h.heads, " heads and ", k.size(0), " keys of ", h.kv, " in ", seqs,
              " sequences exceed one launch");
  return (int)seqs;
}

bool wants(const Tensor& x) { return x.defined() && x.requires_grad(); }
bool wants(const OptTensor& x) { return x && wants(*x); }

// There are gradients of first order by reverse mode, and no others: a tangent that reaches an operator (forward mode), or a
// gradient that is differentiated again, is an error, where below autograd it would be lost.
bool dual(const Tensor& x) { return x.defined() && x._fw_grad(/*level=*/0).defined(); }
bool dual(const OptTensor& x) { return x && dual(*x); }
bool dual(at::TensorList xs) { return std::any_of(xs.begin(), xs.end(), [](const Tensor& x) { return dual(x); }); }
template <typename... Xs>
void no_tangents(const char* what, const Xs&... xs) {
  TORCH_CHECK(!(dual(xs) || ...), POL, what, " has no forward-mode derivative");
}
// a gradient's operator as a node, for graphs of gradients (create_graph), that raises when it is run backward
#define FIRST_ORDER(what)                                                          \
  static variable_list backward(AutogradContext*, variable_list) {                 \
    TORCH_CHECK(false, POL what "'s gradients cannot be differentiated again");    \
  }

// The dispatcher's operators (a node calls them rather than the functions above, so that torch.compile sees them).
#define OP(name)                                                                                                        \
  const auto& name##_op() {                                                                                             \
    static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow("nablaengine::" #name, "").typed<decltype(name)>(); \
    return op;                                                                                                          \
  }

// the nodes' operators, where they are called above autograd: by name, or at a transform's inner level
void inner_autograd(const c10::OperatorHandle& op, torch::jit::Stack* stack) {
  const std::string& name = op.schema().name();
  const size_t count = op.schema().arguments().size();
  for (size_t i = stack->size() - count; i < stack->size(); ++i) {
    if (!(*stack)[i].isTensor()) continue;
    const Tensor& x = (*stack)[i].toTensor();
    no_tangents(name.c_str(), x);
    TORCH_CHECK(!at::GradMode::is_enabled() || !wants(x), POL, name, " has no gradient: call the operator that it is a part of");
  }
  at::AutoDispatchBelowADInplaceOrView below;
  op.callBoxed(stack);
}

}  // namespace
