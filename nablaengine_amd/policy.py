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
implementation, which torch.compile keeps as one node (torch_ffi.init() first, as for the step: a trace cannot load the
library). A tensor made on another stream than the call's is the caller's to synchronize and to keep alive
(Tensor.record_stream), as with torch's own operators. Results are bitwise the same on every run. Gradients are first order
by reverse mode: forward mode, the backward of a gradient and torch.func's derivatives raise RuntimeError.
"""
import ctypes
import math
import os

import torch
from torch import Tensor

from . import torch_ffi
from .torch_ffi import _wants_grad

EPS = 1e-5
TORCH_LIB = os.path.join(torch_ffi.HERE, "libnablaengine_policy_torch.so")


def _err(msg, kind=TypeError):
    return kind(f"nablaengine_amd.policy: {msg}")


def _tensor(name, x):
    if not isinstance(x, Tensor):
        raise _err(f"{name} must be a torch.Tensor on a ROCm device, got {type(x).__name__}")
    return x


# ---- the operators (csrc/policy_torch.cpp defines them, with their autograd nodes) ------------------------------------

_bound = []  # the operators' library, once it has the kernels' entries


def _ops():
    """torch.ops.nablaengine with this module's operators, bound to the kernels' library (torch_ffi's, one a process)."""
    if not _bound:
        _bind()
    return torch.ops.nablaengine


def _define():
    """Load the operators' definitions and give them their fake implementations (no kernel library yet)."""
    torch.ops.load_library(TORCH_LIB)
    for name, fake in _FAKES.items():
        torch.library.register_fake(f"nablaengine::{name}", fake)


def _bind():
    with torch_ffi._lock:
        if _bound:
            return
        if not os.path.exists(TORCH_LIB):
            raise _err(f"{TORCH_LIB} is missing: build it with `python -m nablaengine_amd.build`", RuntimeError)
        if not hasattr(torch.ops.nablaengine, "attention_step"):
            _define()
        native = torch_ffi._load()
        lib = ctypes.CDLL(TORCH_LIB)
        lib.dk_policy_torch_entries.restype, lib.dk_policy_torch_bind.restype = ctypes.c_char_p, None
        names = lib.dk_policy_torch_entries().decode().split()
        missing = [n for n in names if not hasattr(native.dll, n)]
        if missing:
            raise _err(f"{native.path} has no {missing[0]}: a build from before the policy operators", RuntimeError)
        entries = (ctypes.c_void_p * len(names))(*(ctypes.cast(getattr(native.dll, n), ctypes.c_void_p).value for n in names))
        lib.dk_policy_torch_bind(entries)
        _bound.append(lib)


def _fake_layer_norm_forward(x, weight, bias, eps, stats):
    rows = x.numel() // x.shape[-1] if stats else 0
    return [x.new_empty(x.shape), x.new_empty((2, rows), dtype=torch.float32)]


def _fake_layer_norm_backward(dy, x, weight, bias, stats, want_x, want_weight, want_bias):
    n, ptype = x.shape[-1], next((p.dtype for p in (weight, bias) if p is not None), torch.float32)
    return [x.new_empty(x.shape if want_x else (0,))] + [x.new_empty((n if want else 0,), dtype=ptype)
                                                         for want in (want_weight, want_bias)]


def _fake_norm(grads, *_):
    return grads[0].new_empty((), dtype=torch.float32)


def _order_words(group, dim, seqs, tq, tk):
    """dk_attention_work_bytes / 4, written out so that sizes may be symbolic (the library's own takes numbers only): a
    head of 16, and two words each of the query tiles of 128 rows and of the key tiles of 128 or 32 keys."""
    keys = 32 if dim <= 64 and tk <= 96 * seqs else 128
    return 16 + 2 * (tq * group // 128 + tk // keys + 2 * (seqs + 1))


def _fake_attention_forward(q, k, v, starts_q, starts_k, scale, train):
    words = _order_words(q.shape[1] // k.shape[1], q.shape[2], starts_q.shape[0] - 1, q.shape[0], k.shape[0])
    return [q.new_empty(q.shape), q.new_empty((q.shape[1], q.shape[0] if train else 0), dtype=torch.float32),
            starts_q.new_empty((words,))]


_FAKES = {"layer_norm": lambda x, *_: x.new_empty(x.shape), "layer_norm_forward": _fake_layer_norm_forward,
          "layer_norm_backward": _fake_layer_norm_backward, "grad_norm": _fake_norm, "clip_grads_": _fake_norm,
          "clip_grads_out": _fake_norm, "attention": lambda q, *_: q.new_empty(q.shape),
          "attention_forward": _fake_attention_forward,
          "attention_backward": lambda dout, q, k, v, *_: [q.new_empty(x.shape) for x in (q, k, v)],
          "attention_step": lambda q, *_: q.new_empty(q.shape)}


# ---- layer norm -----------------------------------------------------------------------------------------------------

def layer_norm(x, weight=None, bias=None, *, eps=EPS):
    """(x - mean) / sqrt(var + eps) * weight + bias over x's last dimension, differentiable in x, weight and bias.

    x: float32, bfloat16 or float16, of any shape whose rows are evenly spaced (a contiguous tensor, or a slice of a
    wider one's columns); weight, bias: float32 or x's type, or None. y is contiguous and has x's type; mean, variance
    and every sum are float32, and the gradients have their inputs' types."""
    e = float(eps)
    if not 0.0 <= e < math.inf:
        raise _err(f"eps must be finite and >= 0, got {eps}", ValueError)
    return _ops().layer_norm(_tensor("x", x), weight, bias, e)


# ---- the global gradient norm, and clipping -------------------------------------------------------------------------

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

def _scale(scale, q):
    if _tensor("q", q).dim() != 3 or q.shape[2] < 1:
        raise _err(f"q must have 3 dimensions, got {tuple(q.shape)}")
    if scale is None:
        return 1.0 / math.sqrt(q.shape[2])
    s = float(scale)
    if not 0.0 < s < math.inf:
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
    the matrix instructions, as the inputs are (float16: brought inside its range first). A query whose every score is -inf
    gives NaN."""
    starts_k = starts_q if starts_k is None else starts_k
    s = _scale(scale, q)
    return _ops().attention(q, _tensor("k", k), _tensor("v", v), _tensor("starts_q", starts_q),
                            _tensor("starts_k", starts_k), s)


def attention_step(q, k, v, lengths, *, scale=None):
    """The control loop's attention: each world's one new query over its own cached history, without gradients.

    q: (worlds, heads, dim); k, v: (worlds, capacity, kv_heads, dim), the cache, of which the first lengths[w] tokens of
    world w count (lengths: (worlds,) int32 on the device, moved into 0 .. capacity; what lies past them is not read);
    types, heads, dim, strides and scale as attention's. A world without history gives zeros."""
    if _wants_grad(q, k, v):
        raise _err("attention_step has no gradient: use attention (one query a sequence), or torch.no_grad()", RuntimeError)
    return _ops().attention_step(q, _tensor("k", k), _tensor("v", v), _tensor("lengths", lengths), _scale(scale, q))


def _bind_loaded():
    try:
        _bind()
    except Exception:  # a library without the operators: their first call says so, and the step needs none of them
        pass


if os.path.exists(TORCH_LIB):
    _define()  # at import: defining operators inside a torch.compile trace is not traceable, nor is binding them
    torch_ffi._on_load.append(_bind_loaded)
    if torch_ffi._native is not None:
        _bind_loaded()
