// The torch side of the operators of nablaengine_memory.h, as policy_torch.cpp is of nablaengine_policy.h's. Their entries are
// handed over apart (dk_memory_torch_bind): a kernels' library built before them still has the others.
#include "policy_torch.h"

#include "../../include/nablaengine_memory.h"
#include "policy_sizes.h"

namespace {

#define ENTRIES(X)                                                                                                    \
  X(dk_recurrence) X(dk_recurrence_vjp) X(dk_recurrence_carry_bytes) X(dk_recurrence_work_bytes) X(dk_recurrence_step)
struct Entries {
#define X(name) decltype(&::name) name;
  ENTRIES(X)
#undef X
} lib = {};

template <typename T>
T* out_of(const Tensor& x) { return x.defined() ? (T*)x.data_ptr() : nullptr; }

// ---- recurrence -----------------------------------------------------------------------------------------------------

struct Sequences { int type, tokens, channels, seqs; };
// x: (tokens, channels) of a float type, each token's elements neighbours
int tokens_checks(const Tensor& x) {
  check_device("x", x, x);
  const int type = type_of(x);
  CHECK_TYPE(type >= 0 && x.dim() == 2 && x.size(1) >= 1, "x: expected float32, bfloat16 or float16 of 2 dimensions, got ", described(x));
  return type;
}
void neighbours(const char* name, const Tensor& x) {
  CHECK_TYPE(x.numel() == 0 || x.size(-1) == 1 || x.stride(-1) == 1, name, ": a row's elements must be neighbours, got ", described(x));
}
Sequences recurrence_checks(const Tensor& x, const Tensor& gate, const Tensor& starts, const OptTensor& initial) {
  Sequences r = {};
  r.type = tokens_checks(x);
  check_as("gate", gate, x, x.scalar_type(), x.sizes());
  check_device("starts", starts, x);
  CHECK_TYPE(starts.scalar_type() == at::kInt && starts.dim() == 1 && starts.is_contiguous() && starts.numel() >= 1,
             "starts: expected contiguous int32 offsets, one more than sequences, got ", described(starts));
  const int64_t seqs = starts.numel() - 1, most = 0x7fffffff;
  CHECK_VALUE(x.size(0) < most && x.size(1) < most && seqs < most && pol::scan_sizes((int)x.size(0), (int)x.size(1), (int)seqs),
              x.size(0), " tokens of ", x.size(1), " channels in ", seqs, " sequences exceed one launch");
  neighbours("x", x), neighbours("gate", gate);
  if (in(initial)) {
    check_as("initial", *initial, x, at::kFloat, {seqs, x.size(1)});
    CHECK_TYPE(initial->is_contiguous(), "initial must be contiguous, got ", described(*initial));
  }
  r.tokens = (int)x.size(0), r.channels = (int)x.size(1), r.seqs = (int)seqs;
  return r;
}
const float* floats(const OptTensor& x) { return (const float*)in(x); }

std::vector<Tensor> recurrence_forward(const Tensor& x, const Tensor& gate, const Tensor& starts, const OptTensor& initial) {
  const Sequences s = recurrence_checks(x, gate, starts, initial);
  check_bound();
  const auto f32 = x.options().dtype(at::kFloat);
  const Tensor h = at::empty(x.sizes(), x.options()), last = at::empty({s.seqs, s.channels}, f32);
  const Tensor carry = at::empty({lib.dk_recurrence_carry_bytes(s.tokens, s.channels) / 4}, f32);
  const Tensor work = work_of(x, lib.dk_recurrence_work_bytes(s.tokens, s.channels, 0));
  call("the recurrence launch", x, [&](hipStream_t st) {
    return lib.dk_recurrence(st, s.type, s.tokens, s.channels, s.seqs, x.data_ptr(), x.stride(0), gate.data_ptr(), gate.stride(0),
                             starts.data_ptr<int>(), floats(initial), h.data_ptr(), last.data_ptr<float>(),
                             carry.data_ptr<float>(), work.data_ptr());
  });
  return {h, last, carry};
}

// a cotangent, in any strides: rows of neighbouring elements
Tensor rows_of(const OptTensor& grad) {
  if (!in(grad)) return Tensor();
  return grad->numel() && grad->size(-1) > 1 && grad->stride(-1) != 1 ? grad->contiguous() : *grad;
}

std::vector<Tensor> recurrence_backward(const OptTensor& dh, const OptTensor& dlast, const Tensor& x, const Tensor& gate,
                                        const Tensor& starts, const OptTensor& initial, const Tensor& carry, bool want_x,
                                        bool want_gate, bool want_initial) {
  const Sequences s = recurrence_checks(x, gate, starts, initial);
  check_bound();
  if (dh && dh->defined()) check_as("dh", *dh, x, x.scalar_type(), x.sizes());
  if (dlast && dlast->defined()) check_as("dlast", *dlast, x, at::kFloat, {s.seqs, s.channels});
  check_as("carry", carry, x, at::kFloat, {lib.dk_recurrence_carry_bytes(s.tokens, s.channels) / 4});
  const Tensor d = rows_of(dh), l = in(dlast) ? dlast->contiguous() : Tensor();
  const Tensor dx = at::empty(want_x ? x.sizes() : at::IntArrayRef{0}, x.options());
  const Tensor dg = at::empty(want_gate ? x.sizes() : at::IntArrayRef{0}, x.options());
  const auto f32 = x.options().dtype(at::kFloat);
  const Tensor di = want_initial ? at::empty({s.seqs, s.channels}, f32) : at::empty({0}, f32);
  const Tensor work = work_of(x, lib.dk_recurrence_work_bytes(s.tokens, s.channels, 1));
  call("the recurrence VJP launch", x, [&](hipStream_t st) {
    return lib.dk_recurrence_vjp(st, s.type, s.tokens, s.channels, s.seqs, x.data_ptr(), x.stride(0), gate.data_ptr(),
                                 gate.stride(0), starts.data_ptr<int>(), floats(initial), carry.data_ptr<float>(),
                                 out_of<void>(d), d.defined() ? d.stride(0) : 0, out_of<float>(l), want_x ? dx.data_ptr() : nullptr,
                                 want_gate ? dg.data_ptr() : nullptr, want_initial ? di.data_ptr<float>() : nullptr, work.data_ptr());
  });
  return {dx, dg, di};
}

std::tuple<Tensor, Tensor> recurrence_step(const Tensor& x, const Tensor& gate, const Tensor& state) {
  const int type = tokens_checks(x);
  check_as("gate", gate, x, x.scalar_type(), x.sizes());
  check_as("state", state, x, at::kFloat, x.sizes());
  neighbours("x", x), neighbours("gate", gate), neighbours("state", state);
  CHECK_VALUE(x.size(1) < 1 << 30, x.size(1), " channels exceed one launch");
  const Tensor h = at::empty(x.sizes(), x.options()), next = at::empty(x.sizes(), state.options());
  call("the recurrence step launch", x, [&](hipStream_t st) {
    return lib.dk_recurrence_step(st, type, x.size(0), (int)x.size(1), x.data_ptr(), x.stride(0), gate.data_ptr(), gate.stride(0),
                                  state.data_ptr<float>(), state.stride(0), h.data_ptr(), next.data_ptr<float>());
  });
  return {h, next};
}

// ---- autograd -------------------------------------------------------------------------------------------------------

OP(recurrence_forward) OP(recurrence_backward) OP(recurrence_step)

OptTensor given(const Tensor& x) { return x.defined() ? OptTensor(x) : OptTensor(); }
bool wants_any(at::TensorList xs) { return std::any_of(xs.begin(), xs.end(), [](const Tensor& x) { return wants(x); }); }

struct RecurrenceBackward : torch::autograd::Function<RecurrenceBackward> {
  static variable_list forward(AutogradContext*, const OptTensor& dh, const OptTensor& dlast, const Tensor& x, const Tensor& gate,
                               const Tensor& starts, const OptTensor& initial, const Tensor& carry, bool want_x, bool want_gate,
                               bool want_initial) {
    at::AutoDispatchBelowADInplaceOrView below;
    return recurrence_backward_op().call(dh, dlast, x, gate, starts, initial, carry, want_x, want_gate, want_initial);
  }
  FIRST_ORDER("recurrence")
};
struct Recurrence : torch::autograd::Function<Recurrence> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& gate, const Tensor& starts,
                               const OptTensor& initial) {
    at::AutoDispatchBelowADInplaceOrView below;
    auto r = recurrence_forward_op().call(x, gate, starts, initial);
    ctx->set_materialize_grads(false);
    ctx->saved_data["want"] = std::vector<int64_t>{wants(x), wants(gate), wants(initial)};
    ctx->save_for_backward({x, gate, starts, initial ? *initial : Tensor(), r[2]});
    return {r[0], r[1]};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grad) {
    const auto s = ctx->get_saved_variables();
    const auto want = ctx->saved_data["want"].toIntVector();
    if (!grad[0].defined() && !grad[1].defined()) return variable_list(4);
    no_tangents("recurrence's gradient", grad[0], grad[1], s[0], s[1], s[3]);
    auto run = [&] {
      const OptTensor dh = given(grad[0]), dlast = given(grad[1]), initial = given(s[3]);
      if (at::GradMode::is_enabled())
        return RecurrenceBackward::apply(dh, dlast, s[0], s[1], s[2], initial, s[4], !!want[0], !!want[1], !!want[2]);
      at::AutoDispatchBelowADInplaceOrView below;
      return recurrence_backward_op().call(dh, dlast, s[0], s[1], s[2], initial, s[4], want[0], want[1], want[2]);
    };
    const variable_list r = run();
    return {want[0] ? r[0] : Tensor(), want[1] ? r[1] : Tensor(), Tensor(), want[2] ? r[2] : Tensor()};
  }
};
std::tuple<Tensor, Tensor> recurrence_autograd(const Tensor& x, const Tensor& gate, const Tensor& starts, const OptTensor& initial) {
  no_tangents("recurrence", x, gate, initial);
  if (at::GradMode::is_enabled() && (wants(x) || wants(gate) || wants(initial))) {
    const variable_list r = Recurrence::apply(x, gate, starts, initial);
    return {r[0], r[1]};
  }
  at::AutoDispatchBelowADInplaceOrView below;
  const auto r = recurrence_forward_op().call(x, gate, starts, initial);
  return {r[0], r[1]};
}
std::tuple<Tensor, Tensor> recurrence(const Tensor& x, const Tensor& gate, const Tensor& starts, const OptTensor& initial) {
  const auto r = recurrence_forward_op().call(x, gate, starts, initial);
  return {r[0], r[1]};
}
std::tuple<Tensor, Tensor> recurrence_step_autograd(const Tensor& x, const Tensor& gate, const Tensor& state) {
  no_tangents("recurrence_step", x, gate, state);
  TORCH_CHECK(!at::GradMode::is_enabled() || !wants_any({x, gate, state}), POL "recurrence_step has no gradient");
  at::AutoDispatchBelowADInplaceOrView below;
  return recurrence_step_op().call(x, gate, state);
}

}  // namespace

// the entries' names, in the order in which dk_memory_torch_bind takes their addresses
extern "C" const char* dk_memory_torch_entries() {
#define X(name) #name " "
  return ENTRIES(X);
#undef X
}
extern "C" void dk_memory_torch_bind(void* const* addresses) {
  size_t i = 0;
#define X(name) lib.name = (decltype(lib.name))addresses[i++];
  ENTRIES(X)
#undef X
  bound = true;
}

TORCH_LIBRARY_FRAGMENT(nablaengine, m) {
  m.def("recurrence(Tensor x, Tensor gate, Tensor starts, Tensor? initial) -> (Tensor, Tensor)");
  m.def("recurrence_forward(Tensor x, Tensor gate, Tensor starts, Tensor? initial) -> Tensor[]");
  m.def("recurrence_backward(Tensor? dh, Tensor? dlast, Tensor x, Tensor gate, Tensor starts, Tensor? initial, Tensor carry, "
        "bool want_x, bool want_gate, bool want_initial) -> Tensor[]");
  m.def("recurrence_step(Tensor x, Tensor gate, Tensor state) -> (Tensor, Tensor)");
}
TORCH_LIBRARY_IMPL(nablaengine, CompositeExplicitAutograd, m) {
  m.impl("recurrence", recurrence);
  m.impl("recurrence_forward", recurrence_forward);
  m.impl("recurrence_backward", recurrence_backward);
  m.impl("recurrence_step", recurrence_step);
}
TORCH_LIBRARY_IMPL(nablaengine, Autograd, m) {
  m.impl("recurrence", recurrence_autograd);
  m.impl("recurrence_step", recurrence_step_autograd);
  for (const char* name : {"recurrence_forward", "recurrence_backward"})
    m.impl(name, torch::CppFunction::makeFromBoxedFunction<&inner_autograd>());
}
