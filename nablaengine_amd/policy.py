"""Operators of the policies that are trained through the control step, as hand-written kernels beside the step's own:

  layer_norm(x, weight=None, bias=None, *, eps=1e-5) -> y
  grad_norm(grads) -> norm
  clip_grads_(grads, max_norm, *, out=None) -> norm;  clip_grad_norm_(parameters, max_norm) -> norm
  attention(q, k, v, starts_q, starts_k=None, *, scale=None) -> out
  attention_step(q, k, v, lengths, *, scale=None) -> out

A policy's hidden layers are normed over thousands of worlds (layer_norm, with its gradients); one that remembers
attends over its own past: over whole episodes of different lengths, packed one after another, in training (attention,
with its gradients), and over each world's cached history in the control loop (attention_step). Backpropagation
through time gives large gradients now and then, which are clipped by their global norm before the optimizer's step
(clip_grad_norm_).

Conventions are torch_ffi's: tensors lie on one ROCm device and are never cast, copied or moved: another type, shape or
device is a TypeError, a bad option a ValueError, a failed library call a RuntimeError; there is no CPU path. Calls only
launch kernels on the device's current stream and take memory from torch's caching allocator: nothing synchronizes, so
they may be captured in a HIP graph, and each is an operator of the ``nablaengine`` namespace with a fake
implementation, which torch.compile keeps as one node. A tensor made on another stream than the call's is the caller's
to synchronize and to keep alive (Tensor.record_stream), as with torch's own operators. Results are bitwise the same on
every run. Gradients are first order only.
"""
import ctypes
import math

import torch
from torch import Tensor
from torch.autograd.function import once_differentiable

from . import torch_ffi
from .torch_ffi import _stream, _wants_grad

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
EPS = 1e-5
MAX_DIM = 128  # attention: elements of a head


def _err(msg, kind=TypeError):
    return kind(f"nablaengine_amd.policy: {msg}")


def _P(x):
    return None if x is None else ctypes.c_void_p(x.data_ptr())


def _describe(x):
    return f"{x.dtype} {tuple(x.shape)} with strides {x.stride()} on {x.device}" if isinstance(x, Tensor) else type(x).__name__


def _check(name, x, like, dtypes, dims=None, shape=None):
    """x is a tensor on `like`'s device (None: any ROCm device) of one of the types and of that rank or shape."""
    if not isinstance(x, Tensor) or x.device.type != "cuda":
        raise _err(f"{name} must be a torch.Tensor on a ROCm device, got {x.device if isinstance(x, Tensor) else type(x).__name__}")
    if like is not None and x.device != like.device:
        raise _err(f"{name} is on {x.device}, the first tensor on {like.device}")
    if x.dtype not in dtypes or (dims is not None and x.dim() != dims) or (shape is not None and tuple(x.shape) != shape):
        want = " or ".join(str(d) for d in dtypes)
        raise _err(f"{name}: expected {want}{'' if shape is None else f' of shape {shape}'}"
                   f"{'' if dims is None else f' of {dims} dimensions'}, got {_describe(x)}")


def _call(what, entry, dev, *args):
    nat = torch_ffi._ready(dev)
    with torch.cuda.device(dev):
        nat.run(what, entry, _stream(dev), *args)


def _dll(dev):
    return torch_ffi._ready(dev).dll


# ---- layer norm -----------------------------------------------------------------------------------------------------

def _row_stride(x):
    """Elements from row to row of x seen as rows of its last dimension, or None: its rows' elements are not
    neighbours, or its rows are not evenly spaced."""
    n = x.shape[-1]
    if x.numel() == 0:
        return n
    if n > 1 and x.stride(-1) != 1:
        return None
    lead = [(size, stride) for size, stride in zip(x.shape[:-1], x.stride()[:-1]) if size > 1]
    for (_, outer), (size, inner) in zip(lead, lead[1:]):
        if outer != size * inner:
            return None
    return lead[-1][1] if lead else n


def _norm_checks(x, weight, bias):
    _check("x", x, None, _TYPES)
    if x.dim() < 1 or x.shape[-1] < 1 or x.shape[-1] >= 2 ** 31:
        raise _err(f"x needs a last dimension of 1 to 2^31 - 1 elements, got {_describe(x)}")
    params = [(name, p) for name, p in (("weight", weight), ("bias", bias)) if p is not None]
    for name, p in params:
        _check(name, p, x, {torch.float32: 0, x.dtype: 0}, shape=(x.shape[-1],))
        if not p.is_contiguous():
            raise _err(f"{name} must be contiguous, got {_describe(p)}")
    if len(params) == 2 and weight.dtype != bias.dtype:
        raise _err(f"weight and bias must have one type, got {weight.dtype} and {bias.dtype}")
    stride = _row_stride(x)
    if stride is None:
        raise _err(f"x: expected evenly spaced rows of neighbouring elements, got {_describe(x)}")
    return stride, params[0][1].dtype if params else torch.float32


def _layer_norm_call(x, weight, bias, eps, stats):
    stride, ptype = _norm_checks(x, weight, bias)
    n = x.shape[-1]
    rows = x.numel() // n
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    st = torch.empty((2, rows if stats else 0), dtype=torch.float32, device=x.device)
    _call("the layer norm launch", "dk_layer_norm", x.device.index, rows, n, _TYPES[x.dtype], _P(x), stride,
          _TYPES[ptype], _P(weight), _P(bias), eps, _P(y), _P(st) if stats else None)
    return [y, st]


def _layer_norm_backward_call(dy, x, weight, bias, stats, want_x, want_weight, want_bias):
    stride, ptype = _norm_checks(x, weight, bias)
    _check("dy", dy, x, {x.dtype: 0}, shape=tuple(x.shape))
    dstride = _row_stride(dy)
    if dstride is None:
        raise _err(f"dy: expected evenly spaced rows of neighbouring elements, got {_describe(dy)}")
    n = x.shape[-1]
    rows = x.numel() // n
    _check("stats", stats, x, {torch.float32: 0}, shape=(2, rows))
    dev = x.device.index
    dx = torch.empty(x.shape if want_x else (0,), dtype=x.dtype, device=x.device)
    dw, db = (torch.empty((n if want else 0,), dtype=ptype, device=x.device) for want in (want_weight, want_bias))
    work = None
    if want_weight or want_bias:
        work = torch.empty((int(_dll(dev).dk_layer_norm_work_bytes(rows, n, _TYPES[x.dtype])),), dtype=torch.uint8,
                           device=x.device)
    _call("the layer norm VJP launch", "dk_layer_norm_vjp", dev, rows, n, _TYPES[x.dtype], _P(x), stride, _P(dy), dstride,
          _TYPES[ptype], _P(weight), _P(stats), _P(dx) if want_x else None, _P(dw) if want_weight else None,
          _P(db) if want_bias else None, _P(work))
    return [dx, dw, db]


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, stats = _ops().layer_norm(x, weight, bias, eps, True)
        ctx.save_for_backward(x, weight, bias, stats)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, bias, stats = ctx.saved_tensors
        want = ctx.needs_input_grad
        if _row_stride(dy) is None:
            dy = dy.contiguous()
        dx, dw, db = _ops().layer_norm_backward(dy, x, weight, bias, stats, want[0], want[1], want[2])
        return dx if want[0] else None, dw if want[1] else None, db if want[2] else None, None


def layer_norm(x, weight=None, bias=None, *, eps=EPS):
    """(x - mean) / sqrt(var + eps) * weight + bias over x's last dimension, differentiable in x, weight and bias.

    x: float32, bfloat16 or float16, of any shape whose rows are evenly spaced (a contiguous tensor, or a slice of a
    wider one's columns); weight, bias: float32 or x's type, or None. y is contiguous and has x's type; mean, variance
    and every sum are float32, and the gradients have their inputs' types."""
    e = float(eps)
    if not (math.isfinite(e) and e >= 0.0):
        raise _err(f"eps must be finite and >= 0, got {eps}", ValueError)
    if _wants_grad(x, weight, bias):
        return _LayerNorm.apply(x, weight, bias, e)
    return _ops().layer_norm(x, weight, bias, e, False)[0]


# ---- the global gradient norm, and clipping -------------------------------------------------------------------------

def _dense(x):
    """Whether x's elements fill one stretch of memory, each once (in any order of its dimensions)."""
    if x.is_contiguous():
        return True
    expect = 1
    for stride, size in sorted((s, n) for s, n in zip(x.stride(), x.shape) if n > 1):
        if stride != expect:
            return False
        expect *= size
    return True


def _grads_checks(grads, out):
    """The non-empty gradients and their outputs (None without `out`), after the checks."""
    for i, g in enumerate(grads):
        _check(f"gradient {i}", g, grads[0], _TYPES)
        if not _dense(g):
            raise _err(f"gradient {i}: expected a tensor that fills its memory, got {_describe(g)}")
    if out is None:
        return [g for g in grads if g.numel()], None
    if len(out) != len(grads):
        raise _err(f"{len(grads)} gradients, but {len(out)} outputs", ValueError)
    for i, (g, o) in enumerate(zip(grads, out)):
        _check(f"output {i}", o, g, {torch.float32: 0, g.dtype: 0}, shape=tuple(g.shape))
        if o.stride() != g.stride() and not (o.is_contiguous() and g.is_contiguous()):
            raise _err(f"output {i}: expected gradient {i}'s strides {g.stride()}, got {_describe(o)}")
    pairs = [(g, o) for g, o in zip(grads, out) if g.numel()]
    spans = []
    for g, o in pairs:
        at, to = g.data_ptr(), o.data_ptr()
        spans.append((to, to + o.numel() * o.element_size(), True))
        if at != to or g.dtype != o.dtype:
            spans.append((at, at + g.numel() * g.element_size(), False))
    any_end = out_end = 0
    for start, end, written in sorted(spans):
        if start < (any_end if written else out_end):
            raise _err("a tensor that is written overlaps another one", ValueError)
        any_end = max(any_end, end)
        if written:
            out_end = max(out_end, end)
    return [g for g, _ in pairs], [o for _, o in pairs]


def _clip(grads, out, max_norm):
    like = grads[0]
    grads, out = _grads_checks(grads, out)
    dev, n = like.device.index, len(grads)
    norm = torch.empty((), dtype=torch.float32, device=like.device)
    work = torch.empty((int(_dll(dev).dk_clip_work_bytes(n)),), dtype=torch.uint8, device=like.device)
    types = (ctypes.c_int * n)(*[_TYPES[g.dtype] for g in grads])
    _call("the gradient norm launch", "dk_clip", dev, n, (ctypes.c_void_p * n)(*[g.data_ptr() for g in grads]),
          (ctypes.c_longlong * n)(*[g.numel() for g in grads]), types,
          None if out is None else (ctypes.c_void_p * n)(*[o.data_ptr() for o in out]),
          None if out is None else (ctypes.c_int * n)(*[_TYPES[o.dtype] for o in out]), max_norm, _P(norm),
          _P(work) if n else None)
    return norm


def _grad_norm_call(grads):
    return _clip(grads, None, 0.0)


def _clip_grads__call(grads, max_norm):
    return _clip(grads, grads, max_norm)


def _clip_grads_out_call(grads, out, max_norm):
    return _clip(grads, out, max_norm)


def _tensors(xs, what):
    xs = [xs] if isinstance(xs, Tensor) else list(xs)
    for i, x in enumerate(xs):
        if not isinstance(x, Tensor):
            raise _err(f"{what} {i} must be a torch.Tensor, got {type(x).__name__}")
    return xs


def _gradients(grads):
    grads = _tensors(grads, "gradient")
    if any(g.requires_grad for g in grads):
        raise _err("a gradient that requires grad itself: the norm and clipping are not differentiable")
    return grads


def _max_norm(max_norm):
    limit = float(max_norm)
    if not limit >= 0.0:
        raise _err(f"max_norm must be >= 0, got {max_norm}", ValueError)
    return limit


def grad_norm(grads):
    """The 2-norm of all gradients' elements together: a float32 tensor without dimensions on their device. grads: a
    tensor or an iterable of them, float32, bfloat16 and float16 in any mixture, of any shapes and dense layouts. The
    squares are summed in float64: gradients of 1e30 or 1e-30 have their norm too."""
    grads = _gradients(grads)
    return _ops().grad_norm(grads) if grads else torch.zeros(())


def clip_grads_(grads, max_norm, *, out=None):
    """Multiply the gradients by min(1, max_norm / (norm + 1e-6)), norm = grad_norm(grads), which is returned (before
    clipping; nothing waits for it). In place, or into `out`: as many tensors, shaped and laid out as the gradients, of
    their types or float32 (an optimizer's buffers), which must not overlap one another or other gradients. An infinite
    norm gives zeros (NaN where the gradient is infinite), a norm that is NaN gives NaN everywhere."""
    limit = _max_norm(max_norm)
    grads = _gradients(grads)
    if out is None:
        return _ops().clip_grads_(grads, limit) if grads else torch.zeros(())
    out = _tensors(out, "output")
    if any(o.requires_grad for o in out):
        raise _err("an output that requires grad: clipping is not differentiable")
    if not grads:
        if out:
            raise _err(f"0 gradients, but {len(out)} outputs", ValueError)
        return torch.zeros(())
    return _ops().clip_grads_out(grads, out, limit)


def clip_grad_norm_(parameters, max_norm):
    """clip_grads_ of the gradients of `parameters` (those that have one), in place."""
    parameters = [parameters] if isinstance(parameters, Tensor) else list(parameters)
    return clip_grads_([p.grad for p in parameters if p.grad is not None], max_norm)


# ---- attention ------------------------------------------------------------------------------------------------------

_HALF = {torch.bfloat16: 0, torch.float16: 0}


def _heads_checks(q, k, v, dims):
    _check("q", q, None, _HALF, dims=3)
    _check("k", k, q, {q.dtype: 0}, dims=dims)
    _check("v", v, q, {q.dtype: 0}, shape=tuple(k.shape))
    heads, dim, kv = q.shape[1], q.shape[2], k.shape[-2]
    if k.shape[-1] != dim or dim % 8 or not 8 <= dim <= MAX_DIM:
        raise _err(f"q and k need heads of one size, a multiple of 8 up to {MAX_DIM}, got {dim} and {k.shape[-1]}")
    if kv < 1 or heads < 1 or heads % kv:
        raise _err(f"q's heads must be a multiple of k's, got {heads} and {kv}")
    for name, x in (("q", q), ("k", k), ("v", v)):
        if x.numel() and x.stride(-1) != 1:
            raise _err(f"{name}: a head's elements must be neighbours, got {_describe(x)}")
    return heads, kv, dim


def _attention_checks(q, k, v, starts_q, starts_k):
    heads, kv, dim = _heads_checks(q, k, v, 3)
    for name, x in (("starts_q", starts_q), ("starts_k", starts_k)):
        _check(name, x, q, {torch.int32: 0}, dims=1)
        if not x.is_contiguous() or x.numel() != starts_q.numel() or x.numel() < 1:
            raise _err(f"{name}: expected contiguous offsets, one more than sequences in both, got {_describe(x)}")
    seqs = starts_q.numel() - 1
    if (q.shape[0] * (heads // kv) >= 2 ** 30 or k.shape[0] >= 2 ** 30
            or max(q.shape[0] * (heads // kv) // 128, k.shape[0] // 128) + seqs + 1 >= 2 ** 24 // kv):
        raise _err(f"{q.shape[0]} queries of {heads} heads and {k.shape[0]} keys of {kv} in {seqs} sequences exceed one "
                   "launch", ValueError)
    return [_TYPES[q.dtype], heads, kv, dim, seqs, q.shape[0], k.shape[0], _P(q), q.stride(0), q.stride(1), _P(k),
            k.stride(0), k.stride(1), _P(v), v.stride(0), v.stride(1), _P(starts_q), _P(starts_k)]


def _attention_call(q, k, v, starts_q, starts_k, scale, train):
    args = _attention_checks(q, k, v, starts_q, starts_k)
    dev = q.device.index
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    lse = torch.empty((q.shape[1], q.shape[0] if train else 0), dtype=torch.float32, device=q.device)
    work = torch.empty((_order_words(q, k, starts_q),), dtype=torch.int32, device=q.device)
    _call("the attention launch", "dk_attention", dev, *args, scale, _P(out), _P(lse) if train else None, _P(work))
    return [out, lse, work]


def _order_words(q, k, starts_q):
    return int(torch_ffi._load().dll.dk_attention_work_bytes(q.shape[1], k.shape[1], starts_q.shape[0] - 1, q.shape[0],
                                                             k.shape[0])) // 4


def _attention_backward_call(dout, q, k, v, starts_q, starts_k, out, lse, work, scale):
    args = _attention_checks(q, k, v, starts_q, starts_k)
    dev = q.device.index
    for name, x in (("dout", dout), ("out", out)):
        _check(name, x, q, {q.dtype: 0}, shape=tuple(q.shape))
    if dout.numel() and dout.stride(2) != 1 or not out.is_contiguous():
        raise _err(f"dout: a head's elements must be neighbours, got {_describe(dout)}; out must be contiguous")
    _check("lse", lse, q, {torch.float32: 0}, shape=(q.shape[1], q.shape[0]))
    _check("work", work, q, {torch.int32: 0}, shape=(_order_words(q, k, starts_q),))
    delta = torch.empty_like(lse)
    dq, dk, dv = (torch.empty(x.shape, dtype=q.dtype, device=q.device) for x in (q, k, v))
    _call("the attention VJP launch", "dk_attention_vjp", dev, *args, scale, _P(out), _P(lse), _P(work), _P(dout),
          dout.stride(0), dout.stride(1), _P(delta), _P(dq), _P(dk), _P(dv))
    return [dq, dk, dv]


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, starts_q, starts_k, scale):
        out, lse, work = _ops().attention(q, k, v, starts_q, starts_k, scale, True)
        ctx.save_for_backward(q, k, v, starts_q, starts_k, out, lse, work)
        ctx.scale = scale
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        if dout.numel() and dout.stride(2) != 1:
            dout = dout.contiguous()
        dq, dk, dv = _ops().attention_backward(dout, *ctx.saved_tensors, ctx.scale)
        return dq, dk, dv, None, None, None


def _scale(scale, q):
    if scale is None:
        if not isinstance(q, Tensor) or q.dim() != 3 or q.shape[2] < 1:
            raise _err(f"q must have 3 dimensions, got {_describe(q)}")
        return 1.0 / math.sqrt(q.shape[2])
    s = float(scale)
    if not (math.isfinite(s) and s > 0.0):
        raise _err(f"scale must be finite and > 0, got {scale}", ValueError)
    return s


def attention(q, k, v, starts_q, starts_k=None, *, scale=None):
    """Causal attention over packed sequences (episodes of different lengths, one after another), differentiable in q, k
    and v: out = softmax(scale q k^T) v within each sequence, in q's type.

    q: (queries, heads, dim), k, v: (keys, kv_heads, dim), bfloat16 or float16; heads a multiple of kv_heads, each key
    head serving heads / kv_heads neighbouring query heads; dim a multiple of 8 up to 128, its elements neighbours, tokens
    and heads any distance apart (slices of one projection's output). starts_q, starts_k (default: starts_q): int32
    offsets on the device, 0 first, sequence s being tokens starts[s] .. starts[s + 1] - 1. Of nq queries and nk keys,
    query i sees keys 0 .. i + nk - nq: the last query sees every key, so that nk > nq gives the queries earlier keys
    (nq = 1: one new query over a history). A query that sees no key gives zeros, and so do tokens past the last
    sequence (padding), whose gradients are zero too. scale (> 0) defaults to 1 / sqrt(dim).

    Scores, softmax statistics and all sums are float32; probabilities and score gradients are rounded to q's type for
    the matrix instructions, as the inputs are."""
    starts_k = starts_q if starts_k is None else starts_k
    s = _scale(scale, q)
    if _wants_grad(q, k, v):
        return _Attention.apply(q, k, v, starts_q, starts_k, s)
    return _ops().attention(q, k, v, starts_q, starts_k, s, False)[0]


def _attention_step_call(q, k, v, lengths, scale):
    heads, kv, dim = _heads_checks(q, k, v, 4)
    worlds, capacity = q.shape[0], k.shape[1]
    if k.shape[0] != worlds:
        raise _err(f"q has {worlds} worlds, the cache {k.shape[0]}")
    _check("lengths", lengths, q, {torch.int32: 0}, shape=(worlds,))
    if not lengths.is_contiguous():
        raise _err(f"lengths must be contiguous, got {_describe(lengths)}")
    dev = q.device.index
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    size = int(_dll(dev).dk_attention_step_work_bytes(worlds, heads, kv, dim, capacity))
    work = torch.empty((size,), dtype=torch.uint8, device=q.device) if size else None
    _call("the attention step launch", "dk_attention_step", dev, _TYPES[q.dtype], worlds, heads, kv, dim, capacity, _P(q),
          q.stride(0), q.stride(1), _P(k), *k.stride()[:3], _P(v), *v.stride()[:3], _P(lengths), scale, _P(out), _P(work))
    return out


def attention_step(q, k, v, lengths, *, scale=None):
    """The control loop's attention: each world's one new query over its own cached history, without gradients.

    q: (worlds, heads, dim); k, v: (worlds, capacity, kv_heads, dim), the cache, of which the first lengths[w] tokens of
    world w count (lengths: (worlds,) int32 on the device, moved into 0 .. capacity; what lies past them is not read);
    types, heads, dim, strides and scale as attention's. A world without history gives zeros."""
    if _wants_grad(q, k, v):
        raise _err("attention_step has no gradient: use attention (one query a sequence), or torch.no_grad()", RuntimeError)
    return _ops().attention_step(q, k, v, lengths, _scale(scale, q))


# ---- the operators (torch.library) ----------------------------------------------------------------------------------

_SCHEMAS = {
    "layer_norm": "layer_norm(Tensor x, Tensor? weight, Tensor? bias, float eps, bool stats) -> Tensor[]",
    "layer_norm_backward": "layer_norm_backward(Tensor dy, Tensor x, Tensor? weight, Tensor? bias, Tensor stats, "
                           "bool want_x, bool want_weight, bool want_bias) -> Tensor[]",
    "grad_norm": "grad_norm(Tensor[] grads) -> Tensor",
    "clip_grads_": "clip_grads_(Tensor(a!)[] grads, float max_norm) -> Tensor",
    "clip_grads_out": "clip_grads_out(Tensor[] grads, Tensor(a!)[] out, float max_norm) -> Tensor",
    "attention": "attention(Tensor q, Tensor k, Tensor v, Tensor starts_q, Tensor starts_k, float scale, bool train) "
                 "-> Tensor[]",
    "attention_backward": "attention_backward(Tensor dout, Tensor q, Tensor k, Tensor v, Tensor starts_q, "
                          "Tensor starts_k, Tensor out, Tensor lse, Tensor work, float scale) -> Tensor[]",
    "attention_step": "attention_step(Tensor q, Tensor k, Tensor v, Tensor lengths, float scale) -> Tensor",
}


def _fake_layer_norm(x, weight, bias, eps, stats):
    rows = x.numel() // x.shape[-1] if stats else 0
    return [x.new_empty(x.shape), x.new_empty((2, rows), dtype=torch.float32)]


def _fake_layer_norm_backward(dy, x, weight, bias, stats, want_x, want_weight, want_bias):
    n, ptype = x.shape[-1], next((p.dtype for p in (weight, bias) if p is not None), torch.float32)
    return [x.new_empty(x.shape if want_x else (0,))] + [x.new_empty((n if want else 0,), dtype=ptype)
                                                         for want in (want_weight, want_bias)]


def _fake_norm(grads, *_):
    return grads[0].new_empty((), dtype=torch.float32)


def _fake_attention(q, k, v, starts_q, starts_k, scale, train):
    return [q.new_empty(q.shape), q.new_empty((q.shape[1], q.shape[0] if train else 0), dtype=torch.float32),
            starts_q.new_empty((_order_words(q, k, starts_q),))]


def _fake_attention_backward(dout, q, k, v, *_):
    return [q.new_empty(x.shape) for x in (q, k, v)]


def _fake_attention_step(q, k, v, lengths, scale):
    return q.new_empty(q.shape)


_KERNELS = {"layer_norm": (_layer_norm_call, _fake_layer_norm),
            "layer_norm_backward": (_layer_norm_backward_call, _fake_layer_norm_backward),
            "grad_norm": (_grad_norm_call, _fake_norm), "clip_grads_": (_clip_grads__call, _fake_norm),
            "clip_grads_out": (_clip_grads_out_call, _fake_norm), "attention": (_attention_call, _fake_attention),
            "attention_backward": (_attention_backward_call, _fake_attention_backward),
            "attention_step": (_attention_step_call, _fake_attention_step)}
_library_defs = []


def _ops():
    """torch.ops.nablaengine with this module's operators."""
    if not _library_defs:
        _register_ops()
    return torch.ops.nablaengine


def _register_ops():
    torch_ffi._register_ops()
    with torch_ffi._lock:
        if not _library_defs:
            lib = torch.library.Library("nablaengine", "FRAGMENT")
            for name, schema in _SCHEMAS.items():
                call, fake = _KERNELS[name]
                lib.define(schema)
                lib.impl(name, call, "CompositeExplicitAutograd")
                torch.library.register_fake(f"nablaengine::{name}", fake, lib=lib)
            _library_defs.append(lib)


_register_ops()  # at import: defining operators inside a torch.compile trace is not traceable
