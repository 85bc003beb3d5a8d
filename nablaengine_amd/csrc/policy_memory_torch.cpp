// The torch side of the operators of nablaengine_memory.h, as policy_torch.cpp is of nablaengine_policy.h's. Their entries are
// handed over apart (dk_memory_torch_bind): a kernels' library built before them still has the others.
#include "policy_torch.h"

#include <ATen/MemoryOverlap.h>

#include "../../include/nablaengine_memory.h"
#include "../../include/nablaengine_policy.h"

namespace {

#define ENTRIES(X)                                                                                                    \
  X(dk_recurrence) X(dk_recurrence_vjp) X(dk_recurrence_carry_bytes) X(dk_recurrence_work_bytes) X(dk_recurrence_step) \
  X(dk_gated_residual) X(dk_gated_residual_vjp) X(dk_gated_residual_work_bytes)             \
  X(dk_attention_paged) X(dk_attention_paged_work_bytes) X(dk_cache_append)                             \
  X(dk_attention_window) X(dk_attention_window_vjp) X(dk_attention_window_scratch_bytes) X(dk_attention_work_bytes)
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

// ---- gated residual -------------------------------------------------------------------------------------------------

struct Rows {
  int64_t n, rows, x, u, gate;  // elements from row to row
  int type, param_type;
  at::ScalarType params;
};
Rows residual_checks(const Tensor& x, const Tensor& u, const OptTensor& weight, const OptTensor& next_weight, const OptTensor& gate,
                     const OptTensor& scale) {
  check_device("x", x, x);
  Rows r = {};
  r.type = type_of(x);
  CHECK_TYPE(r.type >= 0 && x.dim() >= 1 && x.size(-1) >= 1 && x.size(-1) < 1LL << 31,
             "x: expected float32, bfloat16 or float16 with a last dimension of 1 to 2^31 - 1 elements, got ", described(x));
  check_as("u", u, x, x.scalar_type(), x.sizes());
  if (in(gate)) check_as("gate", *gate, x, x.scalar_type(), x.sizes());
  r.n = x.size(-1), r.rows = x.numel() / r.n, r.params = at::kFloat;
  const Tensor* first = nullptr;
  for (const auto& [name, p] : {std::pair<const char*, const OptTensor&>{"weight", weight}, {"next_weight", next_weight}, {"scale", scale}}) {
    if (!in(p)) continue;
    check_device(name, *p, x);
    CHECK_TYPE((p->scalar_type() == at::kFloat || p->scalar_type() == x.scalar_type()) && p->dim() == 1 && p->size(0) == r.n &&
                   p->is_contiguous(),
               name, ": expected ", r.n, " contiguous elements of float32 or ", x.scalar_type(), ", got ", described(*p));
    CHECK_TYPE(!first || first->scalar_type() == p->scalar_type(), "weight, next_weight and scale must have one type");
    first = &*p, r.params = p->scalar_type(), r.param_type = type_of(*p);
  }
  r.x = row_stride(x), r.u = row_stride(u), r.gate = in(gate) ? row_stride(*gate) : 0;
  CHECK_TYPE(r.x >= 0 && r.u >= 0 && r.gate >= 0, "x, u and gate: expected evenly spaced rows of neighbouring elements, got ",
             described(x), ", ", described(u), in(gate) ? ", " + described(*gate) : "");
  return r;
}

std::vector<Tensor> gated_residual_forward(const Tensor& x, const Tensor& u, const OptTensor& weight, const OptTensor& next_weight,
                                           const OptTensor& gate, const OptTensor& scale, double eps, bool stats) {
  const Rows a = residual_checks(x, u, weight, next_weight, gate, scale);
  const Tensor y = at::empty(x.sizes(), x.options()), z = at::empty(x.sizes(), x.options());
  const Tensor s = at::empty({2, stats ? a.rows : 0}, x.options().dtype(at::kFloat));
  call("the gated residual launch", x, [&](hipStream_t st) {
    return lib.dk_gated_residual(st, a.rows, (int)a.n, a.type, x.data_ptr(), a.x, u.data_ptr(), a.u, in(gate), a.gate, a.param_type,
                                 in(weight), in(next_weight), in(scale), (float)eps, y.data_ptr(), z.data_ptr(),
                                 stats ? s.data_ptr<float>() : nullptr);
  });
  return {y, z, s};
}

// want: a bit for each of x, u, weight, next_weight, gate, scale
std::vector<Tensor> gated_residual_backward(const OptTensor& dy, const OptTensor& dz, const Tensor& x, const Tensor& u,
                                            const OptTensor& weight, const OptTensor& next_weight, const OptTensor& gate,
                                            const OptTensor& scale, const Tensor& stats, int64_t want) {
  const Rows a = residual_checks(x, u, weight, next_weight, gate, scale);
  Tensor cots[2];
  int64_t strides[2] = {};
  for (const auto& [i, name, g] : {std::tuple<int, const char*, const OptTensor&>{0, "dy", dy}, {1, "dz", dz}}) {
    if (!g || !g->defined()) continue;
    check_as(name, *g, x, x.scalar_type(), x.sizes());
    cots[i] = row_stride(*g) < 0 ? g->contiguous() : *g;
    strides[i] = row_stride(cots[i]);
  }
  check_as("stats", stats, x, at::kFloat, {2, a.rows});
  CHECK_TYPE(stats.is_contiguous(), "stats must be contiguous");
  const auto params = x.options().dtype(a.params);
  std::vector<Tensor> r;
  void* to[6];
  for (int i = 0; i < 6; ++i) {
    const bool row = i == 0 || i == 1 || i == 4, wanted = want >> i & 1;
    r.push_back(row ? at::empty(wanted ? x.sizes() : at::IntArrayRef{0}, x.options()) : at::empty({wanted ? a.n : 0}, params));
    to[i] = wanted ? r.back().data_ptr() : nullptr;
  }
  Tensor work;
  if (bound && (to[2] || to[3] || to[5])) work = work_of(x, lib.dk_gated_residual_work_bytes(a.rows, (int)a.n, a.type));
  call("the gated residual VJP launch", x, [&](hipStream_t st) {
    return lib.dk_gated_residual_vjp(st, a.rows, (int)a.n, a.type, x.data_ptr(), a.x, u.data_ptr(), a.u, in(gate), a.gate,
                                     a.param_type, in(weight), in(next_weight), in(scale), stats.data_ptr<float>(),
                                     out_of<void>(cots[0]), strides[0], out_of<void>(cots[1]), strides[1], to[0], to[1], to[4], to[2],
                                     to[3], to[5], work.defined() ? work.data_ptr() : nullptr);
  });
  return r;
}

// ---- paged histories ------------------------------------------------------------------------------------------------

struct Pool { int count, page, most; };
// a pool of pages (count, page, kv_heads, dim), and the worlds' tables and lengths
Pool pool_checks(const Tensor& k_pages, const Tensor& pages, const Tensor& lengths, int64_t worlds) {
  const int64_t count = k_pages.size(0), page = k_pages.size(1);
  CHECK_VALUE(page >= 1 && !(page & (page - 1)), "a page holds a power of two of tokens, not ", page);
  check_device("pages", pages, k_pages);
  CHECK_TYPE(pages.scalar_type() == at::kInt && pages.dim() == 2 && pages.size(0) == worlds &&
                 (pages.numel() == 0 || pages.size(1) == 1 || pages.stride(1) == 1),
             "pages: expected int32 page numbers of ", worlds, " worlds, each world's neighbours, got ", described(pages));
  check_as("lengths", lengths, k_pages, at::kInt, {worlds});
  CHECK_TYPE(lengths.is_contiguous(), "lengths must be contiguous, got ", described(lengths));
  const int64_t most = 1 << 30;
  CHECK_VALUE(count < most && page < most && pages.size(1) < most && pages.size(1) * page < most, count, " pages of ", page,
              " tokens, ", pages.size(1), " a world, exceed one launch");
  return {(int)count, (int)page, (int)pages.size(1)};
}

Tensor attention_paged(const Tensor& q, const Tensor& k_pages, const Tensor& v_pages, const Tensor& pages, const Tensor& lengths,
                       double scale, int64_t window, int64_t sinks) {
  const Heads h = heads_checks(q, k_pages, v_pages, 4);
  const int64_t worlds = q.size(0);
  const Pool p = pool_checks(k_pages, pages, lengths, worlds);
  CHECK_VALUE(worlds * h.heads < 1 << 24, worlds, " worlds of ", h.heads, " heads exceed one launch");
  CHECK_VALUE(window >= 0 && sinks >= 0, "window and sinks must not be negative, got ", window, " and ", sinks);
  const int w = (int)std::min<int64_t>(window, 1 << 30), s = (int)std::min<int64_t>(sinks, 1 << 30);
  check_bound();
  const Tensor out = at::empty(q.sizes(), q.options());
  const long long bytes = lib.dk_attention_paged_work_bytes((int)worlds, h.heads, h.kv, h.dim, p.page, p.most, w, s);
  const Tensor work = bytes ? work_of(q, bytes) : Tensor();
  const Tensor &k = k_pages, &v = v_pages;
  call("the paged attention launch", q, [&](hipStream_t st) {
    return lib.dk_attention_paged(st, h.type, (int)worlds, h.heads, h.kv, h.dim, p.count, p.page, p.most, q.data_ptr(), q.stride(0),
                                  q.stride(1), k.data_ptr(), k.stride(0), k.stride(1), k.stride(2), v.data_ptr(), v.stride(0),
                                  v.stride(1), v.stride(2), pages.data_ptr<int>(), pages.stride(0), lengths.data_ptr<int>(), w, s,
                                  (float)scale, out.data_ptr(), bytes ? work.data_ptr() : nullptr);
  });
  return out;
}

void cache_append_(const Tensor& k_pages, const Tensor& v_pages, const Tensor& k, const Tensor& v, const Tensor& pages,
                   const Tensor& lengths, const OptTensor& starts) {
  const Heads h = heads_checks(k, k_pages, v_pages, 4);
  CHECK_TYPE(h.heads == h.kv, "k has ", h.heads, " heads, the pages ", h.kv);
  check_as("v", v, k, k.scalar_type(), k.sizes());
  CHECK_TYPE(v.numel() == 0 || v.stride(2) == 1, "v: a head's elements must be neighbours, got ", described(v));
  for (const auto& [name, x] : {std::pair<const char*, const Tensor&>{"k_pages", k_pages}, {"v_pages", v_pages}})
    for (int64_t i = 0; i < 4; ++i)
      CHECK_TYPE(x.size(i) <= 1 || x.stride(i) != 0, name, " is written: expected no expanded tensor, got ", described(x));
  const int64_t tokens = k.size(0), worlds = lengths.dim() == 1 ? lengths.size(0) : -1;
  CHECK_TYPE(worlds >= 0, "lengths: expected one dimension, got ", described(lengths));
  const Pool p = pool_checks(k_pages, pages, lengths, worlds);
  if (in(starts)) {
    check_as("starts", *starts, k, at::kInt, {worlds + 1});
    CHECK_TYPE(starts->is_contiguous(), "starts must be contiguous, got ", described(*starts));
  } else {
    CHECK_TYPE(tokens == worlds, "without starts there is one token a world: ", tokens, " tokens, ", worlds, " worlds");
  }
  CHECK_VALUE(tokens < 1 << 30 && worlds < 1 << 24 && worlds * h.kv * (h.dim / 8) < 1LL << 30, tokens, " tokens of ", worlds,
              " worlds exceed one launch");
  // what is read beside what is written, where it can be told (pages of keys and values side by side in one buffer are apart)
  const auto apart = [](const char* a, const Tensor& x, const char* b, const Tensor& y) {
    const auto o = at::get_overlap_status(x, y);
    CHECK_VALUE(x.numel() == 0 || y.numel() == 0 || (o != at::MemOverlapStatus::Full && o != at::MemOverlapStatus::Partial), a, " and ",
                b, " lie over one another in memory");
  };
  apart("k_pages", k_pages, "v_pages", v_pages);
  apart("k", k, "k_pages", k_pages), apart("k", k, "v_pages", v_pages);
  apart("v", v, "k_pages", k_pages), apart("v", v, "v_pages", v_pages);
  call("the cache append launch", k, [&](hipStream_t st) {
    return lib.dk_cache_append(st, h.type, (int)worlds, (int)tokens, h.kv, h.dim, p.count, p.page, p.most, k.data_ptr(), k.stride(0),
                               k.stride(1), v.data_ptr(), v.stride(0), v.stride(1), (const int*)in(starts), k_pages.data_ptr(),
                               k_pages.stride(0), k_pages.stride(1), k_pages.stride(2), v_pages.data_ptr(), v_pages.stride(0),
                               v_pages.stride(1), v_pages.stride(2), pages.data_ptr<int>(), pages.stride(0), lengths.data_ptr<int>());
  });
  for (const Tensor& y : {k_pages, v_pages})  // a graph that saved one of them notices
    if (!y.is_inference()) y.unsafeGetTensorImpl()->bump_version();
}

// ---- attention with a window ----------------------------------------------------------------------------------------

struct Sight { int window, sinks; };
Sight sight_checks(int64_t window, int64_t sinks) {
  CHECK_VALUE(window >= 1 && sinks >= 0, "window must be at least 1 and sinks at least 0, got ", window, " and ", sinks);
  return {(int)std::min<int64_t>(window, 1 << 30), (int)std::min<int64_t>(sinks, 1 << 30)};
}
Tensor window_scratch(const Heads& h, int seqs, const Tensor& q, const Tensor& k, const Sight& s, int vjp) {
  const long long bytes = lib.dk_attention_window_scratch_bytes(h.heads, h.kv, h.dim, seqs, (int)q.size(0), (int)k.size(0), s.window,
                                                                s.sinks, vjp);
  return bytes ? work_of(q, bytes) : Tensor();
}
long long order_words(const Heads& h, int seqs, const Tensor& q, const Tensor& k) {
  return lib.dk_attention_work_bytes(h.heads, h.kv, h.dim, seqs, (int)q.size(0), (int)k.size(0)) / 4;
}

// out, lse, work and rest (what the output's rounding took off, for narrow windows)
std::vector<Tensor> attention_window_forward(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& starts_q,
                                             const Tensor& starts_k, double scale, int64_t window, int64_t sinks, bool train) {
  const Heads h = heads_checks(q, k, v, 3);
  const int seqs = sequences_checks(q, k, starts_q, starts_k, h);
  const Sight s = sight_checks(window, sinks);
  check_bound();
  const Tensor out = at::empty(q.sizes(), q.options());
  const Tensor lse = at::empty({h.heads, train ? q.size(0) : 0}, q.options().dtype(at::kFloat));
  const Tensor work = at::empty({order_words(h, seqs, q, k)}, q.options().dtype(at::kInt));
  const Tensor rest = at::empty(train && (int64_t)s.window + s.sinks <= pol::NARROW ? q.sizes() : at::IntArrayRef{0}, q.options());
  const Tensor scratch = window_scratch(h, seqs, q, k, s, 0);
  call("the windowed attention launch", q, [&](hipStream_t st) {
    return lib.dk_attention_window(st, h.type, h.heads, h.kv, h.dim, seqs, (int)q.size(0), (int)k.size(0), q.data_ptr(), q.stride(0),
                                   q.stride(1), k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0), v.stride(1),
                                   starts_q.data_ptr<int>(), starts_k.data_ptr<int>(), (float)scale, s.window, s.sinks, out.data_ptr(),
                                   rest.numel() ? rest.data_ptr() : nullptr, train ? lse.data_ptr<float>() : nullptr, work.data_ptr(),
                                   out_of<void>(scratch));
  });
  return {out, lse, work, rest};
}

// dout: any strides
std::vector<Tensor> attention_window_backward(const Tensor& grad, const Tensor& q, const Tensor& k, const Tensor& v,
                                              const Tensor& starts_q, const Tensor& starts_k, const Tensor& out, const Tensor& lse,
                                              const Tensor& work, const Tensor& rest, double scale, int64_t window, int64_t sinks) {
  const Heads h = heads_checks(q, k, v, 3);
  const int seqs = sequences_checks(q, k, starts_q, starts_k, h);
  const Sight s = sight_checks(window, sinks);
  check_bound();
  check_as("dout", grad, q, q.scalar_type(), q.sizes());
  check_as("out", out, q, q.scalar_type(), q.sizes());
  if (rest.numel()) check_as("rest", rest, q, q.scalar_type(), q.sizes());
  const Tensor dout = grad.numel() && grad.stride(2) != 1 ? grad.contiguous() : grad;
  check_as("lse", lse, q, at::kFloat, {h.heads, q.size(0)});
  check_as("work", work, q, at::kInt, {order_words(h, seqs, q, k)});
  CHECK_TYPE(out.is_contiguous() && lse.is_contiguous() && work.is_contiguous() && rest.is_contiguous(),
             "out, lse, work and rest must be contiguous");
  const Tensor delta = at::empty(lse.sizes(), lse.options());
  const Tensor dq = at::empty(q.sizes(), q.options()), dk = at::empty(k.sizes(), q.options()), dv = at::empty(k.sizes(), q.options());
  const Tensor scratch = window_scratch(h, seqs, q, k, s, 1);
  call("the windowed attention VJP launch", q, [&](hipStream_t st) {
    return lib.dk_attention_window_vjp(
        st, h.type, h.heads, h.kv, h.dim, seqs, (int)q.size(0), (int)k.size(0), q.data_ptr(), q.stride(0), q.stride(1), k.data_ptr(),
        k.stride(0), k.stride(1), v.data_ptr(), v.stride(0), v.stride(1), starts_q.data_ptr<int>(), starts_k.data_ptr<int>(),
        (float)scale, s.window, s.sinks, out.data_ptr(), rest.numel() ? rest.data_ptr() : nullptr, lse.data_ptr<float>(),
        work.data_ptr(), dout.data_ptr(), dout.stride(0), dout.stride(1), delta.data_ptr<float>(), dq.data_ptr(), dk.data_ptr(),
        dv.data_ptr(), out_of<void>(scratch));
  });
  return {dq, dk, dv};
}

// ---- autograd -------------------------------------------------------------------------------------------------------

OP(recurrence_forward) OP(recurrence_backward) OP(recurrence_step) OP(gated_residual_forward) OP(gated_residual_backward)
OP(attention_paged) OP(cache_append_) OP(attention_window_forward) OP(attention_window_backward)

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

struct GatedResidualBackward : torch::autograd::Function<GatedResidualBackward> {
  static variable_list forward(AutogradContext*, const OptTensor& dy, const OptTensor& dz, const Tensor& x, const Tensor& u,
                               const OptTensor& weight, const OptTensor& next_weight, const OptTensor& gate, const OptTensor& scale,
                               const Tensor& stats, int64_t want) {
    at::AutoDispatchBelowADInplaceOrView below;
    return gated_residual_backward_op().call(dy, dz, x, u, weight, next_weight, gate, scale, stats, want);
  }
  FIRST_ORDER("gated_residual")
};
struct GatedResidual : torch::autograd::Function<GatedResidual> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& u, const OptTensor& weight,
                               const OptTensor& next_weight, const OptTensor& gate, const OptTensor& scale, double eps) {
    at::AutoDispatchBelowADInplaceOrView below;
    auto r = gated_residual_forward_op().call(x, u, weight, next_weight, gate, scale, eps, true);
    ctx->set_materialize_grads(false);
    int64_t want = 0, bit = 1;
    for (bool w : {wants(x), wants(u), wants(weight), wants(next_weight), wants(gate), wants(scale)}) want |= w ? bit : 0, bit *= 2;
    ctx->saved_data["want"] = want;
    auto tensor = [](const OptTensor& p) { return p ? *p : Tensor(); };
    ctx->save_for_backward({x, u, tensor(weight), tensor(next_weight), tensor(gate), tensor(scale), r[2]});
    return {r[0], r[1]};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grad) {
    const auto s = ctx->get_saved_variables();
    const int64_t want = ctx->saved_data["want"].toInt();
    if (!grad[0].defined() && !grad[1].defined()) return variable_list(7);
    no_tangents("gated_residual's gradient", grad[0], grad[1], s[0], s[1], s[2], s[3], s[4], s[5]);
    auto run = [&] {
      const OptTensor dy = given(grad[0]), dz = given(grad[1]);
      if (at::GradMode::is_enabled())
        return GatedResidualBackward::apply(dy, dz, s[0], s[1], given(s[2]), given(s[3]), given(s[4]), given(s[5]), s[6], want);
      at::AutoDispatchBelowADInplaceOrView below;
      return gated_residual_backward_op().call(dy, dz, s[0], s[1], given(s[2]), given(s[3]), given(s[4]), given(s[5]), s[6], want);
    };
    variable_list r = run();
    for (int i = 0; i < 6; ++i)
      if (!(want >> i & 1)) r[i] = Tensor();
    r.push_back(Tensor());
    return r;
  }
};
std::tuple<Tensor, Tensor> gated_residual_autograd(const Tensor& x, const Tensor& u, const OptTensor& weight,
                                                   const OptTensor& next_weight, const OptTensor& gate, const OptTensor& scale,
                                                   double eps) {
  no_tangents("gated_residual", x, u, weight, next_weight, gate, scale);
  if (at::GradMode::is_enabled() &&
      (wants(x) || wants(u) || wants(weight) || wants(next_weight) || wants(gate) || wants(scale))) {
    const variable_list r = GatedResidual::apply(x, u, weight, next_weight, gate, scale, eps);
    return {r[0], r[1]};
  }
  at::AutoDispatchBelowADInplaceOrView below;
  const auto r = gated_residual_forward_op().call(x, u, weight, next_weight, gate, scale, eps, false);
  return {r[0], r[1]};
}
std::tuple<Tensor, Tensor> gated_residual(const Tensor& x, const Tensor& u, const OptTensor& weight, const OptTensor& next_weight,
                                          const OptTensor& gate, const OptTensor& scale, double eps) {
  const auto r = gated_residual_forward_op().call(x, u, weight, next_weight, gate, scale, eps, false);
  return {r[0], r[1]};
}

Tensor attention_paged_autograd(const Tensor& q, const Tensor& k_pages, const Tensor& v_pages, const Tensor& pages,
                                const Tensor& lengths, double scale, int64_t window, int64_t sinks) {
  no_tangents("attention_paged", q, k_pages, v_pages);
  TORCH_CHECK(!at::GradMode::is_enabled() || !wants_any({q, k_pages, v_pages}), POL "attention_paged has no gradient");
  at::AutoDispatchBelowADInplaceOrView below;
  return attention_paged_op().call(q, k_pages, v_pages, pages, lengths, scale, window, sinks);
}
void cache_append_autograd(const Tensor& k_pages, const Tensor& v_pages, const Tensor& k, const Tensor& v, const Tensor& pages,
                           const Tensor& lengths, const OptTensor& starts) {
  no_tangents("cache_append_", k_pages, v_pages, k, v);
  TORCH_CHECK(!at::GradMode::is_enabled() || !wants_any({k_pages, v_pages, k, v}), POL "cache_append_ has no gradient");
  at::AutoDispatchBelowADInplaceOrView below;
  cache_append__op().call(k_pages, v_pages, k, v, pages, lengths, starts);
}

struct WindowBackward : torch::autograd::Function<WindowBackward> {
  static variable_list forward(AutogradContext*, const Tensor& dout, const Tensor& q, const Tensor& k, const Tensor& v,
                               const Tensor& starts_q, const Tensor& starts_k, const Tensor& out, const Tensor& lse,
                               const Tensor& work, const Tensor& rest, double scale, int64_t window, int64_t sinks) {
    at::AutoDispatchBelowADInplaceOrView below;
    return attention_window_backward_op().call(dout, q, k, v, starts_q, starts_k, out, lse, work, rest, scale, window, sinks);
  }
  FIRST_ORDER("attention")
};
struct Window : torch::autograd::Function<Window> {
  static Tensor forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& starts_q,
                        const Tensor& starts_k, double scale, int64_t window, int64_t sinks) {
    at::AutoDispatchBelowADInplaceOrView below;
    auto r = attention_window_forward_op().call(q, k, v, starts_q, starts_k, scale, window, sinks, true);
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["window"] = window;
    ctx->saved_data["sinks"] = sinks;
    ctx->save_for_backward({q, k, v, starts_q, starts_k, r[0], r[1], r[2], r[3]});
    return r[0];
  }
  static variable_list backward(AutogradContext* ctx, variable_list grad) {
    const auto s = ctx->get_saved_variables();
    if (!grad[0].defined()) return variable_list(8);
    const Tensor& dout = grad[0];
    no_tangents("attention's gradient", dout, s[0], s[1], s[2]);
    const double scale = ctx->saved_data["scale"].toDouble();
    const int64_t window = ctx->saved_data["window"].toInt(), sinks = ctx->saved_data["sinks"].toInt();
    auto run = [&] {
      if (at::GradMode::is_enabled())
        return WindowBackward::apply(dout, s[0], s[1], s[2], s[3], s[4], s[5], s[6], s[7], s[8], scale, window, sinks);
      at::AutoDispatchBelowADInplaceOrView below;
      return attention_window_backward_op().call(dout, s[0], s[1], s[2], s[3], s[4], s[5], s[6], s[7], s[8], scale, window, sinks);
    };
    const variable_list r = run();
    return {r[0], r[1], r[2], Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};
Tensor attention_window_autograd(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& starts_q, const Tensor& starts_k,
                                 double scale, int64_t window, int64_t sinks) {
  no_tangents("attention", q, k, v);
  if (at::GradMode::is_enabled() && (wants(q) || wants(k) || wants(v)))
    return Window::apply(q, k, v, starts_q, starts_k, scale, window, sinks);
  at::AutoDispatchBelowADInplaceOrView below;
  return attention_window_forward_op().call(q, k, v, starts_q, starts_k, scale, window, sinks, false)[0];
}
Tensor attention_window(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& starts_q, const Tensor& starts_k,
                        double scale, int64_t window, int64_t sinks) {
  return attention_window_forward_op().call(q, k, v, starts_q, starts_k, scale, window, sinks, false)[0];
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
  m.def("gated_residual(Tensor x, Tensor u, Tensor? weight, Tensor? next_weight, Tensor? gate, Tensor? scale, float eps) "
        "-> (Tensor, Tensor)");
  m.def("gated_residual_forward(Tensor x, Tensor u, Tensor? weight, Tensor? next_weight, Tensor? gate, Tensor? scale, float eps, "
        "bool stats) -> Tensor[]");
  m.def("gated_residual_backward(Tensor? dy, Tensor? dz, Tensor x, Tensor u, Tensor? weight, Tensor? next_weight, Tensor? gate, "
        "Tensor? scale, Tensor stats, int want) -> Tensor[]");
  m.def("attention_paged(Tensor q, Tensor k_pages, Tensor v_pages, Tensor pages, Tensor lengths, float scale, int window, "
        "int sinks) -> Tensor");
  m.def("cache_append_(Tensor(a!) k_pages, Tensor(b!) v_pages, Tensor k, Tensor v, Tensor pages, Tensor lengths, Tensor? starts) "
        "-> ()");
  m.def("attention_window(Tensor q, Tensor k, Tensor v, Tensor starts_q, Tensor starts_k, float scale, int window, int sinks) "
        "-> Tensor");
  m.def("attention_window_forward(Tensor q, Tensor k, Tensor v, Tensor starts_q, Tensor starts_k, float scale, int window, "
        "int sinks, bool train) -> Tensor[]");
  m.def("attention_window_backward(Tensor dout, Tensor q, Tensor k, Tensor v, Tensor starts_q, Tensor starts_k, Tensor out, "
        "Tensor lse, Tensor work, Tensor rest, float scale, int window, int sinks) -> Tensor[]");
}
TORCH_LIBRARY_IMPL(nablaengine, CompositeExplicitAutograd, m) {
  m.impl("attention_window", attention_window);
  m.impl("attention_window_forward", attention_window_forward);
  m.impl("attention_window_backward", attention_window_backward);
  m.impl("attention_paged", attention_paged);
  m.impl("cache_append_", cache_append_);
  m.impl("recurrence", recurrence);
  m.impl("recurrence_forward", recurrence_forward);
  m.impl("recurrence_backward", recurrence_backward);
  m.impl("recurrence_step", recurrence_step);
  m.impl("gated_residual", gated_residual);
  m.impl("gated_residual_forward", gated_residual_forward);
  m.impl("gated_residual_backward", gated_residual_backward);
}
TORCH_LIBRARY_IMPL(nablaengine, Autograd, m) {
  m.impl("recurrence", recurrence_autograd);
  m.impl("recurrence_step", recurrence_step_autograd);
  m.impl("gated_residual", gated_residual_autograd);
  m.impl("attention_paged", attention_paged_autograd);
  m.impl("attention_window", attention_window_autograd);
  m.impl("cache_append_", cache_append_autograd);
  for (const char* name : {"recurrence_forward", "recurrence_backward", "gated_residual_forward", "gated_residual_backward",
                           "attention_window_forward", "attention_window_backward"})
    m.impl(name, torch::CppFunction::makeFromBoxedFunction<&inner_autograd>());
}
