"""Operators of the policies that are trained through the control step, as hand-written kernels beside the step's own:

  layer_norm(x, weight=None, bias=None, *, eps=1e-5) -> y
  grad_norm(grads) -> norm
  clip_grads_(grads, max_norm, *, out=None) -> norm;  clip_grad_norm_(parameters, max_norm) -> norm
  attention(q, k, v, starts_q, starts_k=None, *, scale=None, window=None, sinks=0) -> out
  attention_step(q, k, v, lengths, *, scale=None) -> out
  cache_append_(k_pages, v_pages, k, v, pages, lengths, starts=None)
  attention_paged(q, k_pages, v_pages, pages, lengths, *, scale=None, window=None, sinks=0) -> out
  recurrence(x, gate, starts, initial=None) -> (h, last);  recurrence_step(x, gate, state) -> (h, state)
  gated_residual(x, u, weight=None, next_weight=None, *, gate=None, scale=None, eps=1e-5) -> (y, z)

A policy's hidden layers are normed over thousands of worlds (layer_norm, with its gradients); one that remembers
attends over its own past: over whole episodes of different lengths, packed one after another, in training (attention,
with its gradients), and over each world's cached history in the control loop (attention_step). One that remembers
longer carries a state (recurrence, with its gradients; recurrence_step in the control loop) beside attention that sees
a window of the last steps and a few first ones: over episodes in training, over pages of a shared pool in the control
loop (attention_paged, which cache_append_ fills), so that a world needs no more than its window's pages however long it
runs. Between its blocks lies gated_residual: a block's output normed, gated and scaled onto the residual stream, and
that normed for the next block. Backpropagation through time gives large gradients now and then, which are clipped by
their global norm before the optimizer's step (clip_grad_norm_).

Conventions are torch_ffi's: tensors lie on one ROCm device and are never cast, copied or moved: another type, shape or
device is a TypeError, a bad option a ValueError, a failed library call a RuntimeError; there is no CPU path. Calls only
launch kernels on the device's current stream and take memory from torch's caching allocator: nothing synchronizes, so
they may be captured in a HIP graph (a backward pass as torch captures any: with no eager graph of the same leaves left
alive), and each is an operator of the ``nablaengine`` namespace with a fake implementation, which torch.compile keeps
as one node (torch_ffi.init() first, as for the step: a trace cannot load the library). A tensor made on another stream
than the call's is the caller's to synchronize and to keep alive (Tensor.record_stream), as with torch's own operators.
Results are bitwise the same on every run. Gradients are first order by reverse mode: forward mode, the backward of a
gradient and torch.func's derivatives raise RuntimeError.
"""
import ctypes
import math
import operator
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
_later = []  # those of the operators from recurrence on that the kernels' library does not have


def _ops(later=False):
    """torch.ops.nablaengine with this module's operators, bound to the kernels' library (torch_ffi's, one a process);
    later: for one of the operators from recurrence on."""
    if not _bound:
        _bind()
    if later and _later:
        raise _err(f"{torch_ffi._load().path} has no {_later[0]}: a build from before this operator", RuntimeError)
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
        missing = _hand_over(native, lib.dk_policy_torch_entries, lib.dk_policy_torch_bind)
        if missing:
            raise _err(f"{native.path} has no {missing[0]}: a build from before the policy operators", RuntimeError)
        _later[:] = _hand_over(native, lib.dk_memory_torch_entries, lib.dk_memory_torch_bind)
        _bound.append(lib)


def _hand_over(native, entries, bind):
    """Give the operators the addresses of their entries, or return those that the kernels' library does not have."""
    entries.restype, bind.restype = ctypes.c_char_p, None
    names = entries().decode().split()
    missing = [n for n in names if not hasattr(native.dll, n)]
    if not missing:
        bind((ctypes.c_void_p * len(names))(*(ctypes.cast(getattr(native.dll, n), ctypes.c_void_p).value for n in names)))
    return missing


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


def _fake_attention_window_forward(q, k, v, starts_q, starts_k, scale, window, sinks, train):
    rest = q.new_empty(q.shape if train and window + sinks <= 64 else (0,))
    return _fake_attention_forward(q, k, v, starts_q, starts_k, scale, train) + [rest]


def _fake_recurrence(x, gate, starts, initial):
    return x.new_empty(x.shape), x.new_empty((starts.shape[0] - 1, x.shape[1]), dtype=torch.float32)


def _carry_words(tokens, channels):
    """dk_recurrence_carry_bytes / 4, of symbolic sizes too: a row for each chunk of 64 tokens."""
    return (tokens + 63) // 64 * channels


def _fake_recurrence_forward(x, gate, starts, initial):
    return [*_fake_recurrence(x, gate, starts, initial), x.new_empty((_carry_words(*x.shape),), dtype=torch.float32)]


def _fake_recurrence_backward(dh, dlast, x, gate, starts, initial, carry, want_x, want_gate, want_initial):
    seqs = starts.shape[0] - 1
    return [x.new_empty(x.shape if want else (0,)) for want in (want_x, want_gate)] + [
        x.new_empty((seqs, x.shape[1]) if want_initial else (0,), dtype=torch.float32)]


def _fake_gated_residual_backward(dy, dz, x, u, weight, next_weight, gate, scale, stats, want):
    n, ptype = x.shape[-1], next((p.dtype for p in (weight, next_weight, scale) if p is not None), torch.float32)
    row = lambda bit: x.new_empty(x.shape if want >> bit & 1 else (0,))  # noqa: E731
    param = lambda bit: x.new_empty((n if want >> bit & 1 else 0,), dtype=ptype)  # noqa: E731
    return [row(0), row(1), param(2), param(3), row(4), param(5)]


_FAKES = {"layer_norm": lambda x, *_: x.new_empty(x.shape), "layer_norm_forward": _fake_layer_norm_forward,
          "layer_norm_backward": _fake_layer_norm_backward, "grad_norm": _fake_norm, "clip_grads_": _fake_norm,
          "clip_grads_out": _fake_norm, "attention": lambda q, *_: q.new_empty(q.shape),
          "attention_forward": _fake_attention_forward,
          "attention_backward": lambda dout, q, k, v, *_: [q.new_empty(x.shape) for x in (q, k, v)],
          "attention_step": lambda q, *_: q.new_empty(q.shape),
          "recurrence": _fake_recurrence, "recurrence_forward": _fake_recurrence_forward,
          "recurrence_backward": _fake_recurrence_backward,
          "gated_residual": lambda x, *_: (x.new_empty(x.shape), x.new_empty(x.shape)),
          "gated_residual_forward": lambda x, u, w, w2, gate, scale, eps, stats: [
              x.new_empty(x.shape), x.new_empty(x.shape), x.new_empty((2, x.numel() // x.shape[-1] if stats else 0), dtype=torch.float32)],
          "gated_residual_backward": _fake_gated_residual_backward,
          "attention_window": lambda q, *_: q.new_empty(q.shape), "attention_window_forward": _fake_attention_window_forward,
          "attention_window_backward": lambda dout, q, k, v, *_: [q.new_empty(x.shape) for x in (q, k, v)],
          "attention_paged": lambda q, *_: q.new_empty(q.shape), "cache_append_": lambda *_: None,
          "recurrence_step": lambda x, gate, state: (x.new_empty(x.shape), state.new_empty(x.shape))}


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


def _sight(window, sinks):
    """window (0: none) and sinks as numbers."""
    w, s = 0 if window is None else operator.index(window), operator.index(sinks)
    if w < (0 if window is None else 1) or s < 0:
        raise _err(f"window must be None or at least 1 and sinks at least 0, got {window} and {sinks}", ValueError)
    most = 1 << 30  # more tokens than any sequence has
    return min(w, most), min(s, most)


def attention(q, k, v, starts_q, starts_k=None, *, scale=None, window=None, sinks=0):
    """Causal attention over packed sequences (episodes of different lengths, one after another), differentiable in q, k
    and v: out = softmax(scale q k^T) v within each sequence, in q's type.

    q: (queries, heads, dim), k, v: (keys, kv_heads, dim), bfloat16 or float16; heads a multiple of kv_heads, each key
    head serving heads / kv_heads neighbouring query heads; dim a multiple of 8 up to 128, its elements neighbours, tokens
    and heads any distance apart (slices of one projection's output). starts_q, starts_k (default: starts_q): int32
    offsets on the device, 0 first, sequence s being tokens starts[s] .. starts[s + 1] - 1. Of nq queries and nk keys,
    query i sees keys 0 .. i + nk - nq: the last query sees every key, so that nk > nq gives the queries earlier keys
    (nq = 1: one new query over a history). A query that sees no key gives zeros, and so do tokens past the last
    sequence (padding), whose gradients are zero too. scale (> 0) defaults to 1 / sqrt(dim).

    window: of those keys a query sees the `window` last ones only, and the `sinks` first ones of its sequence; the time goes by
    the keys in sight then, but with more than 128 sinks the gradients of the first keys by all of a sequence's rows. A window that no sequence is longer than hides nothing; without one, sinks have no part.

    Scores, softmax statistics and all sums are float32; probabilities and score gradients are rounded to q's type for
    the matrix instructions, as the inputs are (float16: brought inside its range first). A query whose every score is -inf
    gives NaN."""
    starts_k = starts_q if starts_k is None else starts_k
    s, (w, first) = _scale(scale, q), _sight(window, sinks)
    if w:
        return _ops(True).attention_window(q, _tensor("k", k), _tensor("v", v), _tensor("starts_q", starts_q),
                                           _tensor("starts_k", starts_k), s, w, first)
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


# ---- recurrence -----------------------------------------------------------------------------------------------------

def recurrence(x, gate, starts, initial=None):
    """A gated linear recurrence over packed sequences (episodes of different lengths, one after another): h_t = a_t h_{t-1} +
    (1 - a_t) x_t with a = sigmoid(gate), a channel at a time, differentiable in x, gate and initial. Returns h and each
    sequence's state after its last token, to be carried on.

    x, gate: (tokens, channels), float32, bfloat16 or float16, each token's elements neighbours, tokens any distance apart
    (slices of one projection's output; a gate of one row for all, expanded). starts: int32 offsets on the device, 0 first, not
    falling, sequence s being tokens starts[s] .. starts[s + 1] - 1. initial: (sequences, channels) float32, contiguous, the
    states before the first tokens, or None for zeros. h has x's type and is zero behind the last sequence (padding, whose gradients are zero
    too); the last states are float32, those of sequences without tokens their initial ones.

    The gate is given before its sigmoid, since 16 bits do not tell long memories apart after it: the smaller of a and 1 - a is
    computed of it directly, within 7 2^-24 of itself for float32 gates and 1.3 |gate| 2^-24 more for those of 16 bits. States and
    all sums are float32 and each output is rounded once. What steps are off by does not add up token by token: a state that its
    inputs repeat stays itself within 2^-18, whatever the gate and the tokens' number. Infinities and NaN stay in their channel and
    sequence; whether an infinite state or input gives infinities or NaN further on depends on where in a chunk it lies."""
    return _ops(True).recurrence(_tensor("x", x), _tensor("gate", gate), _tensor("starts", starts), initial)


def recurrence_step(x, gate, state):
    """One token of every world: (h, next state) with next = a state + (1 - a) x, a = sigmoid(gate), float32 as state is, and h
    its value in x's type; without gradients. x, gate, state: (worlds, channels), rows any distance apart. The control loop's
    form of recurrence."""
    if _wants_grad(x, gate, state):
        raise _err("recurrence_step has no gradient: use recurrence (one token a sequence), or torch.no_grad()", RuntimeError)
    return _ops(True).recurrence_step(_tensor("x", x), _tensor("gate", gate), _tensor("state", state))


# ---- gated residual -------------------------------------------------------------------------------------------------

def gated_residual(x, u, weight=None, next_weight=None, *, gate=None, scale=None, eps=EPS):
    """What lies between two blocks of a policy: (y, z) with y = x + scale sigmoid(gate) rms(u) weight, the residual stream x
    with a block's output u normed, gated and scaled onto it, and z = rms(y) next_weight, the next block's input (or the head's,
    behind the last block); rms(v) = v / sqrt(mean v^2 + eps) over the last dimension. Differentiable in all but eps.

    x, u, gate: float32, bfloat16 or float16, one type and shape, rows evenly spaced (as layer_norm's x); weight, next_weight,
    scale: vectors of float32 or x's type, one type. Without a gate it is open (1), without scale and weights they are ones. y
    and z are contiguous and have x's type. All is computed in float32: z comes of the y that is not rounded yet, and so do the
    gradients."""
    e = float(eps)
    if not 0.0 <= e < math.inf:
        raise _err(f"eps must be finite and >= 0, got {eps}", ValueError)
    return _ops(True).gated_residual(_tensor("x", x), _tensor("u", u), weight, next_weight, gate, scale, e)


# ---- paged histories ------------------------------------------------------------------------------------------------

def cache_append_(k_pages, v_pages, k, v, pages, lengths, starts=None):
    """Write new keys and values into the pages: one token a world, k and v (worlds, kv_heads, dim), or with starts (int32
    offsets on the device, one more than worlds) any number of each, packed (tokens, kv_heads, dim). The i-th of world w becomes
    its token lengths[w] + i, lengths being those without the new ones; adding them to lengths is the caller's.

    k_pages, v_pages: (pool, page, kv_heads, dim), bfloat16 or float16, page a power of two; pages: (worlds, most) int32 on the
    device, the numbers of each world's pages in order. A page that is written belongs to one world alone, and the pages, k and
    v lie apart in memory. A token that has no place, past the `most` pages or on a page whose number is none of the pool's
    (-1, say), is dropped. No gradients."""
    for name, x in (("k_pages", k_pages), ("v_pages", v_pages), ("k", k), ("v", v), ("pages", pages), ("lengths", lengths)):
        _tensor(name, x)
    if _wants_grad(k_pages, v_pages, k, v):
        raise _err("cache_append_ has no gradient: call it under torch.no_grad()", RuntimeError)
    _ops(True).cache_append_(k_pages, v_pages, k, v, pages, lengths, starts)


def attention_paged(q, k_pages, v_pages, pages, lengths, *, scale=None, window=None, sinks=0):
    """The control loop's attention over histories in pages: each world's one new query over its lengths[w] tokens, its newest
    one among them, without gradients. With a window the query sees the `window` last tokens and the `sinks` first ones, as
    attention's with the same window; pages that hold neither are not read and may serve others (their entries in `pages` may
    hold anything).

    q: (worlds, heads, dim); k_pages, v_pages, pages: as cache_append_'s; lengths: (worlds,) int32 on the device, moved into 0 ..
    most * page; heads, dim, strides and scale as attention's. A world without tokens gives zeros, one with a page in sight
    whose number is none of the pool's NaN. Worlds may share pages."""
    s = _scale(scale, q)
    for name, x in (("k_pages", k_pages), ("v_pages", v_pages), ("pages", pages), ("lengths", lengths)):
        _tensor(name, x)
    if _wants_grad(q, k_pages, v_pages):
        raise _err("attention_paged has no gradient: use attention (one query a sequence), or torch.no_grad()", RuntimeError)
    return _ops(True).attention_paged(q, k_pages, v_pages, pages, lengths, s, *_sight(window, sinks))


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
