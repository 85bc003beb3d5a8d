// The policy operators as operators of torch: argument checks, outputs and work memory from torch's allocator, the call
// into libnablaengine_g1.so on the current stream, and the gradients' autograd nodes. Native because the small calls are
// host time: with the same checks, ctypes call and autograd node in Python a layer norm of 4096 x 512 with its gradients
// took 177 us of host time a pass (110 us of it the backward, which a Python node runs on the engine's thread in turn
// with the caller's interpreter lock), where it takes 74 us now and its kernels 18 us.
//
// The kernels' library is loaded once per process by torch_ffi, which may be told another file: it hands the entries'
// addresses over (dk_policy_torch_bind), so that this library depends on torch alone.
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

#include "../../include/nablaengine_policy.h"
#include "policy_sizes.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

#define ENTRIES(X)                                                                                             \
  X(dk_layer_norm) X(dk_layer_norm_vjp) X(dk_layer_norm_work_bytes) X(dk_clip) X(dk_clip_work_bytes)           \
  X(dk_attention) X(dk_attention_vjp) X(dk_attention_work_bytes) X(dk_attention_scratch_bytes)                  \
  X(dk_attention_step) X(dk_attention_step_work_bytes)
struct Entries {
#define X(name) decltype(&::name) name;
  ENTRIES(X)
#undef X
} lib = {};
bool bound = false;

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
  TORCH_CHECK(bound, POL "the kernels' library is not loaded: call nablaengine_amd.torch_ffi.init()");
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

// ---- layer norm -----------------------------------------------------------------------------------------------------

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

struct Norm {
  int64_t n, rows, stride;
  int type, param_type;
  at::ScalarType params;
};
Norm norm_checks(const Tensor& x, const OptTensor& weight, const OptTensor& bias) {
  check_device("x", x, x);
  Norm r = {};
  r.type = type_of(x);
  CHECK_TYPE(r.type >= 0, "x: expected float32, bfloat16 or float16, got ", described(x));
  CHECK_TYPE(x.dim() >= 1 && x.size(-1) >= 1 && x.size(-1) < 1LL << 31,
             "x needs a last dimension of 1 to 2^31 - 1 elements, got ", described(x));
  r.n = x.size(-1), r.rows = x.numel() / r.n, r.params = at::kFloat;
  const Tensor* first = nullptr;
  for (const auto& [name, p] : {std::pair<const char*, const OptTensor&>{"weight", weight}, {"bias", bias}}) {
    if (!in(p)) continue;
    check_device(name, *p, x);
    CHECK_TYPE((p->scalar_type() == at::kFloat || p->scalar_type() == x.scalar_type()) && p->dim() == 1 &&
                   p->size(0) == r.n && p->is_contiguous(),
               name, ": expected ", r.n, " contiguous elements of float32 or ", x.scalar_type(), ", got ", described(*p));
    CHECK_TYPE(!first || first->scalar_type() == p->scalar_type(), "weight and bias must have one type");
    first = &*p, r.params = p->scalar_type(), r.param_type = type_of(*p);
  }
  r.stride = row_stride(x);
  CHECK_TYPE(r.stride >= 0, "x: expected evenly spaced rows of neighbouring elements, got ", described(x));
  return r;
}

std::vector<Tensor> layer_norm_forward(const Tensor& x, const OptTensor& weight, const OptTensor& bias, double eps,
                                       bool stats) {
  const Norm a = norm_checks(x, weight, bias);
  const Tensor y = at::empty(x.sizes(), x.options());
  const Tensor s = at::empty({2, stats ? a.rows : 0}, x.options().dtype(at::kFloat));
  call("the layer norm launch", x, [&](hipStream_t st) {
    return lib.dk_layer_norm(st, a.rows, (int)a.n, a.type, x.data_ptr(), a.stride, a.param_type, in(weight), in(bias),
                             (float)eps, y.data_ptr(), stats ? s.data_ptr<float>() : nullptr);
  });
  return {y, s};
}

// dy: any strides (a cotangent is what torch makes it; the node, which may hold tensors of symbolic sizes, does not look)
std::vector<Tensor> layer_norm_backward(const Tensor& grad, const Tensor& x, const OptTensor& weight, const OptTensor& bias,
                                        const Tensor& stats, bool want_x, bool want_weight, bool want_bias) {
  const Norm a = norm_checks(x, weight, bias);
  check_as("dy", grad, x, x.scalar_type(), x.sizes());
  const Tensor dy = row_stride(grad) < 0 ? grad.contiguous() : grad;
  const int64_t dy_stride = row_stride(dy);
  check_as("stats", stats, x, at::kFloat, {2, a.rows});
  const Tensor dx = at::empty(want_x ? x.sizes() : at::IntArrayRef{0}, x.options());
  const auto params = x.options().dtype(a.params);
  const Tensor dw = at::empty({want_weight ? a.n : 0}, params), db = at::empty({want_bias ? a.n : 0}, params);
  Tensor work;
  if (bound && (want_weight || want_bias)) work = work_of(x, lib.dk_layer_norm_work_bytes(a.rows, (int)a.n, a.type));
  call("the layer norm VJP launch", x, [&](hipStream_t st) {
    return lib.dk_layer_norm_vjp(st, a.rows, (int)a.n, a.type, x.data_ptr(), a.stride, dy.data_ptr(), dy_stride,
                                 a.param_type, in(weight), stats.data_ptr<float>(), want_x ? dx.data_ptr() : nullptr,
                                 want_weight ? dw.data_ptr() : nullptr, want_bias ? db.data_ptr() : nullptr,
                                 work.defined() ? work.data_ptr() : nullptr);
  });
  return {dx, dw, db};
}

// ---- the global gradient norm, and clipping -------------------------------------------------------------------------

// whether x's elements fill one stretch of memory, each once (in any order of its dimensions)
bool dense(const Tensor& x) { return x.is_contiguous() || x.is_non_overlapping_and_dense(); }

Tensor clip(at::TensorList grads, const at::TensorList* out, double limit) {
  TORCH_CHECK_VALUE(grads.size() > 0, POL "no gradients");
  const Tensor& like = grads[0];
  const size_t count = grads.size();
  std::vector<const void*> g;
  std::vector<void*> o;
  std::vector<long long> n;
  std::vector<int> types, out_types;
  struct Span { uintptr_t from, to; bool written; };
  std::vector<Span> spans;
  g.reserve(count), n.reserve(count), types.reserve(count);
  if (out) {
    CHECK_VALUE(out->size() == count, count, " gradients, but ", out->size(), " outputs");
    o.reserve(count), out_types.reserve(count), spans.reserve(2 * count);
  }
  for (size_t i = 0; i < count; ++i) {
    const Tensor& x = grads[i];
    check_device("a gradient", x, like);
    const int type = type_of(x);
    CHECK_TYPE(type >= 0, "gradient ", i, ": expected float32, bfloat16 or float16, got ", described(x));
    CHECK_TYPE(dense(x), "gradient ", i, ": expected a tensor that fills its memory, got ", described(x));
    if (out) {
      const Tensor& y = (*out)[i];
      check_device("an output", y, like);
      CHECK_TYPE((y.scalar_type() == at::kFloat || y.scalar_type() == x.scalar_type()) && y.sizes() == x.sizes(),
                 "output ", i, ": expected float32 or ", x.scalar_type(), " ", x.sizes(), ", got ", described(y));
      CHECK_TYPE(y.strides() == x.strides() || (y.is_contiguous() && x.is_contiguous()), "output ", i,
                 ": expected gradient ", i, "'s strides ", x.strides(), ", got ", described(y));
    }
    if (x.numel() == 0) continue;
    g.push_back(x.data_ptr()), n.push_back(x.numel()), types.push_back(type);
    if (out) {
      const Tensor& y = (*out)[i];
      o.push_back(y.data_ptr()), out_types.push_back(type_of(y));
      const uintptr_t from = (uintptr_t)x.data_ptr(), to = (uintptr_t)y.data_ptr();
      spans.push_back({to, to + y.numel() * y.element_size(), true});
      if (from != to || x.scalar_type() != y.scalar_type())
        spans.push_back({from, from + x.numel() * x.element_size(), false});
    }
  }
  std::sort(spans.begin(), spans.end(), [](const Span& a, const Span& b) { return a.from < b.from; });
  uintptr_t any_end = 0, out_end = 0;
  for (const Span& s : spans) {
    CHECK_VALUE(s.from >= (s.written ? any_end : out_end), "a tensor that is written overlaps another one");
    any_end = std::max(any_end, s.to);
    if (s.written) out_end = std::max(out_end, s.to);
  }
  const Tensor norm = at::empty({}, like.options().dtype(at::kFloat));
  const Tensor work = bound ? work_of(like, lib.dk_clip_work_bytes((int)g.size())) : Tensor();
  call("the gradient norm launch", like, [&](hipStream_t st) {
    return lib.dk_clip(st, (int)g.size(), g.data(), n.data(), types.data(), out ? o.data() : nullptr,
                       out ? out_types.data() : nullptr, (float)limit, norm.data_ptr<float>(), work.data_ptr());
  });
  if (out)  // a graph that saved one of them notices
    for (const Tensor& y : *out)
      if (!y.is_inference()) y.unsafeGetTensorImpl()->bump_version();
  return norm;
}
Tensor grad_norm(at::TensorList grads) { return clip(grads, nullptr, 0.0); }
Tensor clip_grads_(at::TensorList grads, double max_norm) { return clip(grads, &grads, max_norm); }
Tensor clip_grads_out(at::TensorList grads, at::TensorList out, double max_norm) { return clip(grads, &out, max_norm); }

// ---- attention ------------------------------------------------------------------------------------------------------

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
long long order_words(const Heads& h, int seqs, const Tensor& q, const Tensor& k) {
  return lib.dk_attention_work_bytes(h.heads, h.kv, h.dim, seqs, (int)q.size(0), (int)k.size(0)) / 4;
}

// what a call's kernels hand to one another, or an undefined tensor where they hand nothing
Tensor attention_scratch(const Heads& h, int seqs, const Tensor& q, const Tensor& k, int vjp) {
  const long long bytes =
      lib.dk_attention_scratch_bytes(h.heads, h.kv, h.dim, seqs, (int)q.size(0), (int)k.size(0), vjp);
  return bytes ? at::empty({bytes}, q.options().dtype(at::kByte)) : Tensor();
}

std::vector<Tensor> attention_forward(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& starts_q,
                                      const Tensor& starts_k, double scale, bool train) {
  const Heads h = heads_checks(q, k, v, 3);
  const int seqs = sequences_checks(q, k, starts_q, starts_k, h);
  check_bound();
  const Tensor out = at::empty(q.sizes(), q.options());
  const Tensor lse = at::empty({h.heads, train ? q.size(0) : 0}, q.options().dtype(at::kFloat));
  const Tensor work = at::empty({order_words(h, seqs, q, k)}, q.options().dtype(at::kInt));
  const Tensor scratch = attention_scratch(h, seqs, q, k, 0);
  call("the attention launch", q, [&](hipStream_t st) {
    return lib.dk_attention(st, h.type, h.heads, h.kv, h.dim, seqs, (int)q.size(0), (int)k.size(0), q.data_ptr(), q.stride(0),
                            q.stride(1), k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0), v.stride(1),
                            starts_q.data_ptr<int>(), starts_k.data_ptr<int>(), (float)scale, out.data_ptr(),
                            train ? lse.data_ptr<float>() : nullptr, work.data_ptr(),
                            scratch.defined() ? scratch.data_ptr() : nullptr);
  });
  return {out, lse, work};
}

// dout: any strides, as layer_norm_backward's
std::vector<Tensor> attention_backward(const Tensor& grad, const Tensor& q, const Tensor& k, const Tensor& v,
                                       const Tensor& starts_q, const Tensor& starts_k, const Tensor& out,
                                       const Tensor& lse, const Tensor& work, double scale) {
  const Heads h = heads_checks(q, k, v, 3);
  const int seqs = sequences_checks(q, k, starts_q, starts_k, h);
  check_bound();
  check_as("dout", grad, q, q.scalar_type(), q.sizes());
  check_as("out", out, q, q.scalar_type(), q.sizes());
  const Tensor dout = grad.numel() && grad.stride(2) != 1 ? grad.contiguous() : grad;
  check_as("lse", lse, q, at::kFloat, {h.heads, q.size(0)});
  check_as("work", work, q, at::kInt, {order_words(h, seqs, q, k)});
  CHECK_TYPE(out.is_contiguous() && lse.is_contiguous() && work.is_contiguous(), "out, lse and work must be contiguous");
  const Tensor delta = at::empty(lse.sizes(), lse.options());
  const Tensor dq = at::empty(q.sizes(), q.options()), dk = at::empty(k.sizes(), q.options()),
               dv = at::empty(k.sizes(), q.options());
  const Tensor scratch = attention_scratch(h, seqs, q, k, 1);
  call("the attention VJP launch", q, [&](hipStream_t st) {
    return lib.dk_attention_vjp(st, h.type, h.heads, h.kv, h.dim, seqs, (int)q.size(0), (int)k.size(0), q.data_ptr(),
                                q.stride(0), q.stride(1), k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0),
                                v.stride(1), starts_q.data_ptr<int>(), starts_k.data_ptr<int>(), (float)scale,
                                out.data_ptr(), lse.data_ptr<float>(), work.data_ptr(), dout.data_ptr(), dout.stride(0),
                                dout.stride(1), delta.data_ptr<float>(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(),
                                scratch.defined() ? scratch.data_ptr() : nullptr);
  });
  return {dq, dk, dv};
}

Tensor attention_step(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& lengths, double scale) {
  const Heads h = heads_checks(q, k, v, 4);
  const int64_t worlds = q.size(0), capacity = k.size(1);
  CHECK_TYPE(k.size(0) == worlds, "q has ", worlds, " worlds, the cache ", k.size(0));
  check_as("lengths", lengths, q, at::kInt, {worlds});
  CHECK_TYPE(lengths.is_contiguous(), "lengths must be contiguous, got ", described(lengths));
  CHECK_VALUE(worlds * h.heads < 1 << 24 && capacity < 1 << 30, worlds, " worlds of ", h.heads, " heads and a cache of ",
              capacity, " tokens exceed one launch");
  check_bound();
  const Tensor out = at::empty(q.sizes(), q.options());
  const long long bytes = lib.dk_attention_step_work_bytes((int)worlds, h.heads, h.kv, h.dim, (int)capacity);
  const Tensor work = bytes ? work_of(q, bytes) : Tensor();
  call("the attention step launch", q, [&](hipStream_t st) {
    return lib.dk_attention_step(st, h.type, (int)worlds, h.heads, h.kv, h.dim, (int)capacity, q.data_ptr(), q.stride(0),
                                 q.stride(1), k.data_ptr(), k.stride(0), k.stride(1), k.stride(2), v.data_ptr(),
                                 v.stride(0), v.stride(1), v.stride(2), lengths.data_ptr<int>(), (float)scale,
                                 out.data_ptr(), bytes ? work.data_ptr() : nullptr);
  });
  return out;
}

// ---- autograd -------------------------------------------------------------------------------------------------------

// The dispatcher's operators (a node calls them rather than the functions above, so that torch.compile sees them).
#define OP(name)                                                                                                        \
  const auto& name##_op() {                                                                                             \
    static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow("nablaengine::" #name, "").typed<decltype(name)>(); \
    return op;                                                                                                          \
  }
OP(layer_norm_forward) OP(layer_norm_backward) OP(grad_norm) OP(clip_grads_) OP(clip_grads_out)
OP(attention_forward) OP(attention_backward) OP(attention_step)
#undef OP

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
struct LayerNormBackward : torch::autograd::Function<LayerNormBackward> {
  static variable_list forward(AutogradContext*, const Tensor& dy, const Tensor& x, const OptTensor& weight,
                               const OptTensor& bias, const Tensor& stats, bool want_x, bool want_weight, bool want_bias) {
    at::AutoDispatchBelowADInplaceOrView below;
    return layer_norm_backward_op().call(dy, x, weight, bias, stats, want_x, want_weight, want_bias);
  }
  FIRST_ORDER("layer_norm")
};
struct AttentionBackward : torch::autograd::Function<AttentionBackward> {
  static variable_list forward(AutogradContext*, const Tensor& dout, const Tensor& q, const Tensor& k, const Tensor& v,
                               const Tensor& starts_q, const Tensor& starts_k, const Tensor& out, const Tensor& lse,
                               const Tensor& work, double scale) {
    at::AutoDispatchBelowADInplaceOrView below;
    return attention_backward_op().call(dout, q, k, v, starts_q, starts_k, out, lse, work, scale);
  }
  FIRST_ORDER("attention")
};
#undef FIRST_ORDER

struct LayerNorm : torch::autograd::Function<LayerNorm> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const OptTensor& weight, const OptTensor& bias, double eps) {
    at::AutoDispatchBelowADInplaceOrView below;
    auto r = layer_norm_forward_op().call(x, weight, bias, eps, true);
    ctx->saved_data["want"] = std::vector<int64_t>{wants(x), wants(weight), wants(bias)};
    ctx->save_for_backward({x, weight ? *weight : Tensor(), bias ? *bias : Tensor(), r[1]});
    return r[0];
  }
  static variable_list backward(AutogradContext* ctx, variable_list grad) {
    const auto saved = ctx->get_saved_variables();
    const auto want = ctx->saved_data["want"].toIntVector();
    if (!grad[0].defined()) return {Tensor(), Tensor(), Tensor(), Tensor()};
    const Tensor& dy = grad[0];
    auto param = [](const Tensor& p) { return p.defined() ? OptTensor(p) : OptTensor(); };
    no_tangents("layer_norm's gradient", dy, saved[0], saved[1], saved[2]);
    auto run = [&] {
      if (at::GradMode::is_enabled())
        return LayerNormBackward::apply(dy, saved[0], param(saved[1]), param(saved[2]), saved[3], !!want[0], !!want[1], !!want[2]);
      at::AutoDispatchBelowADInplaceOrView below;
      return layer_norm_backward_op().call(dy, saved[0], param(saved[1]), param(saved[2]), saved[3], want[0], want[1], want[2]);
    };
    const variable_list r = run();
    return {want[0] ? r[0] : Tensor(), want[1] ? r[1] : Tensor(), want[2] ? r[2] : Tensor(), Tensor()};
  }
};
Tensor layer_norm_autograd(const Tensor& x, const OptTensor& weight, const OptTensor& bias, double eps) {
  no_tangents("layer_norm", x, weight, bias);
  if (at::GradMode::is_enabled() && (wants(x) || wants(weight) || wants(bias)))
    return LayerNorm::apply(x, weight, bias, eps);
  at::AutoDispatchBelowADInplaceOrView below;
  return layer_norm_forward_op().call(x, weight, bias, eps, false)[0];
}
Tensor layer_norm(const Tensor& x, const OptTensor& weight, const OptTensor& bias, double eps) {
  return layer_norm_forward_op().call(x, weight, bias, eps, false)[0];
}

struct Attention : torch::autograd::Function<Attention> {
  static Tensor forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& starts_q,
                        const Tensor& starts_k, double scale) {
    at::AutoDispatchBelowADInplaceOrView below;
    auto r = attention_forward_op().call(q, k, v, starts_q, starts_k, scale, true);
    ctx->saved_data["scale"] = scale;
    ctx->save_for_backward({q, k, v, starts_q, starts_k, r[0], r[1], r[2]});
    return r[0];
  }
  static variable_list backward(AutogradContext* ctx, variable_list grad) {
    const auto s = ctx->get_saved_variables();
    if (!grad[0].defined()) return variable_list(6);
    const Tensor& dout = grad[0];
    no_tangents("attention's gradient", dout, s[0], s[1], s[2]);
    const double scale = ctx->saved_data["scale"].toDouble();
    auto run = [&] {
      if (at::GradMode::is_enabled())
        return AttentionBackward::apply(dout, s[0], s[1], s[2], s[3], s[4], s[5], s[6], s[7], scale);
      at::AutoDispatchBelowADInplaceOrView below;
      return attention_backward_op().call(dout, s[0], s[1], s[2], s[3], s[4], s[5], s[6], s[7], scale);
    };
    const variable_list r = run();
    return {r[0], r[1], r[2], Tensor(), Tensor(), Tensor()};
  }
};
Tensor attention_autograd(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& starts_q,
                          const Tensor& starts_k, double scale) {
  no_tangents("attention", q, k, v);
  if (at::GradMode::is_enabled() && (wants(q) || wants(k) || wants(v)))
    return Attention::apply(q, k, v, starts_q, starts_k, scale);
  at::AutoDispatchBelowADInplaceOrView below;
  return attention_forward_op().call(q, k, v, starts_q, starts_k, scale, false)[0];
}
Tensor attention(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& starts_q, const Tensor& starts_k,
                 double scale) {
  return attention_forward_op().call(q, k, v, starts_q, starts_k, scale, false)[0];
}

Tensor grad_norm_autograd(at::TensorList grads) {
  no_tangents("grad_norm", grads);
  at::AutoDispatchBelowADInplaceOrView below;
  return grad_norm_op().call(grads);
}
Tensor clip_grads_autograd(at::TensorList grads, double max_norm) {
  no_tangents("clip_grads_", grads);
  at::AutoDispatchBelowADInplaceOrView below;
  return clip_grads__op().call(grads, max_norm);
}
Tensor clip_grads_out_autograd(at::TensorList grads, at::TensorList out, double max_norm) {
  no_tangents("clip_grads_", grads, out);
  at::AutoDispatchBelowADInplaceOrView below;
  return clip_grads_out_op().call(grads, out, max_norm);
}
Tensor attention_step_autograd(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& lengths, double scale) {
  no_tangents("attention_step", q, k, v);
  TORCH_CHECK(!at::GradMode::is_enabled() || !(wants(q) || wants(k) || wants(v)), POL "attention_step has no gradient");
  at::AutoDispatchBelowADInplaceOrView below;
  return attention_step_op().call(q, k, v, lengths, scale);
}
// the nodes' operators, where they are called above autograd: by name, or at a transform's inner level
void inner_autograd(const c10::OperatorHandle& op, torch::jit::Stack* stack) {
  const std::string& name = op.schema().name();
  const size_t count = op.schema().arguments().size();
  for (size_t i = stack->size() - count; i < stack->size(); ++i) {
    if (!(*stack)[i].isTensor()) continue;
    const Tensor& x = (*stack)[i].toTensor();
    no_tangents(name.c_str(), x);
    TORCH_CHECK(!at::GradMode::is_enabled() || !wants(x), POL, name, " has no gradient: call layer_norm or attention");
  }
  at::AutoDispatchBelowADInplaceOrView below;
  op.callBoxed(stack);
}

}  // namespace

// the entries' names, in the order in which dk_policy_torch_bind takes their addresses
extern "C" const char* dk_policy_torch_entries() {
#define X(name) #name " "
  return ENTRIES(X);
#undef X
}
extern "C" void dk_policy_torch_bind(void* const* addresses) {
  size_t i = 0;
#define X(name) lib.name = (decltype(lib.name))addresses[i++];
  ENTRIES(X)
#undef X
  bound = true;
}

TORCH_LIBRARY_FRAGMENT(nablaengine, m) {
  m.def("layer_norm(Tensor x, Tensor? weight, Tensor? bias, float eps) -> Tensor");
  m.def("layer_norm_forward(Tensor x, Tensor? weight, Tensor? bias, float eps, bool stats) -> Tensor[]");
  m.def("layer_norm_backward(Tensor dy, Tensor x, Tensor? weight, Tensor? bias, Tensor stats, bool want_x, "
        "bool want_weight, bool want_bias) -> Tensor[]");
  m.def("grad_norm(Tensor[] grads) -> Tensor");
  m.def("clip_grads_(Tensor(a!)[] grads, float max_norm) -> Tensor");
  m.def("clip_grads_out(Tensor[] grads, Tensor(a!)[] out, float max_norm) -> Tensor");
  m.def("attention(Tensor q, Tensor k, Tensor v, Tensor starts_q, Tensor starts_k, float scale) -> Tensor");
  m.def("attention_forward(Tensor q, Tensor k, Tensor v, Tensor starts_q, Tensor starts_k, float scale, bool train) "
        "-> Tensor[]");
  m.def("attention_backward(Tensor dout, Tensor q, Tensor k, Tensor v, Tensor starts_q, Tensor starts_k, Tensor out, "
        "Tensor lse, Tensor work, float scale) -> Tensor[]");
  m.def("attention_step(Tensor q, Tensor k, Tensor v, Tensor lengths, float scale) -> Tensor");
}
// for every backend: a tensor that is not on a ROCm device reaches the checks and raises TypeError
TORCH_LIBRARY_IMPL(nablaengine, CompositeExplicitAutograd, m) {
  m.impl("layer_norm", layer_norm);
  m.impl("layer_norm_forward", layer_norm_forward);
  m.impl("layer_norm_backward", layer_norm_backward);
  m.impl("grad_norm", grad_norm);
  m.impl("clip_grads_", clip_grads_);
  m.impl("clip_grads_out", clip_grads_out);
  m.impl("attention", attention);
  m.impl("attention_forward", attention_forward);
  m.impl("attention_backward", attention_backward);
  m.impl("attention_step", attention_step);
}
TORCH_LIBRARY_IMPL(nablaengine, Autograd, m) {
  m.impl("layer_norm", layer_norm_autograd);
  m.impl("attention", attention_autograd);
  m.impl("grad_norm", grad_norm_autograd);
  m.impl("clip_grads_", clip_grads_autograd);
  m.impl("clip_grads_out", clip_grads_out_autograd);
  m.impl("attention_step", attention_step_autograd);
  for (const char* name : {"layer_norm_forward", "layer_norm_backward", "attention_forward", "attention_backward"})
    m.impl(name, torch::CppFunction::makeFromBoxedFunction<&inner_autograd>());
}
