"""The operators of policies with a longer memory without a GPU: the library exports every entry of
include/nablaengine_memory.h, the C entries refuse bad arguments before any launch, the Python calls refuse what is not on a ROCm
device, and the operators' fake implementations give the library's output shapes and types."""
import os
import re
import subprocess
import sys

import pytest
import torch

from nablaengine_amd import policy, torch_ffi

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
F32, BF16, I32 = torch.float32, torch.bfloat16, torch.int32


def _prototypes(header):
    """{name: result and arguments, one letter a value} of the header's declarations."""
    txt = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", header)).read(), flags=re.S)
    letter = lambda a: "p" if "*" in a or "hipStream_t" in a else {"long long": "q", "int": "i", "float": "f"}[  # noqa: E731
        a.rsplit(" ", 1)[0]]
    return {m[2]: {"long long": "q", "int": "i"}[m[1]] + ":" + "".join(letter(" ".join(a.split())) for a in m[3].split(","))
            for m in re.finditer(r"(long long|int) (dk_\w+)\(([^;]*?)\);", txt, re.S)}


def test_bindings_are_the_headers():
    protos = _prototypes("nablaengine_memory.h")
    assert protos == torch_ffi._MEMORY_PROTOTYPES
    dll = torch_ffi.load_library()
    for name in protos:
        assert hasattr(dll, name)


def test_c_entries_refuse_before_any_launch():
    dll = torch_ffi.load_library()
    X = 0x1000  # never dereferenced

    def recur(t=1, tokens=300, channels=8, seqs=2, x=X, gate=X, starts=X, h=X, last=X, carry=X, work=X):
        return dll.dk_recurrence(None, t, tokens, channels, seqs, x, 8, gate, 8, starts, None, h, last, carry, work)
    for bad in (dict(t=3), dict(t=-1), dict(tokens=-1), dict(channels=0), dict(seqs=-1), dict(x=None), dict(gate=None), dict(starts=None),
                dict(h=None), dict(last=None), dict(carry=None), dict(work=None), dict(tokens=2 ** 31 - 1), dict(tokens=2 ** 28, channels=1000)):
        assert recur(**bad) == 1, bad

    def recur_vjp(t=1, tokens=300, channels=8, seqs=2, x=X, starts=X, carry=X, work=X):
        return dll.dk_recurrence_vjp(None, t, tokens, channels, seqs, x, 8, X, 8, starts, None, carry, None, 0, None, X, X, X, work)
    for bad in (dict(t=3), dict(tokens=-1), dict(channels=0), dict(x=None), dict(starts=None), dict(carry=None), dict(work=None)):
        assert recur_vjp(**bad) == 1, bad
    assert dll.dk_recurrence_carry_bytes(0, 8) == 0 and dll.dk_recurrence_carry_bytes(1, 8) == 32
    assert dll.dk_recurrence_work_bytes(1, 8, 1) == 96
    tick = lambda t=0, worlds=3, c=8, x=X, s=X, to=X: dll.dk_recurrence_step(None, t, worlds, c, x, c, X, c, s, c, X, to)  # noqa: E731
    assert tick(worlds=0) == 0
    assert tick(t=3) == tick(worlds=-1) == tick(c=0) == tick(x=None) == tick(s=None) == tick(to=None) == 1

    def residual(rows=3, n=8, t=0, wt=0, x=X, u=X, y=X, z=X):
        return dll.dk_gated_residual(None, rows, n, t, x, n, u, n, None, 0, wt, None, None, None, 1e-5, y, z, None)
    assert residual(rows=0) == 0
    for bad in (dict(rows=-1), dict(n=0), dict(t=3), dict(t=1, wt=2), dict(x=None), dict(u=None), dict(y=None), dict(z=None)):
        assert residual(**bad) == 1, bad

    def residual_vjp(rows=3, n=8, t=0, x=X, stats=X, dw=X, work=X):
        return dll.dk_gated_residual_vjp(None, rows, n, t, x, n, X, n, None, 0, 0, None, None, None, stats, None, 0, None, 0, X, X, None,
                                         dw, None, None, work)
    for bad in (dict(rows=-1), dict(n=0), dict(t=3), dict(x=None), dict(stats=None), dict(work=None)):
        assert residual_vjp(**bad) == 1, bad
    assert dll.dk_gated_residual_work_bytes(0, 8, 0) == 0 and dll.dk_gated_residual_work_bytes(3, 8, 0) >= 64

    def paged(t=1, worlds=2, heads=4, kv=2, dim=64, count=9, page=16, most=3, q=X, k=X, pages=X, n=X, window=0, sinks=0, scale=0.1, out=X,
              work=X):
        return dll.dk_attention_paged(None, t, worlds, heads, kv, dim, count, page, most, q, 1, 1, k, 1, 1, 1, X, 1, 1, 1, pages, 1, n,
                                      window, sinks, scale, out, work)
    assert paged(worlds=0) == 0
    for bad in (dict(t=0), dict(worlds=-1), dict(heads=3), dict(kv=0), dict(dim=9), dict(dim=136), dict(count=-1), dict(page=0), dict(page=12),
                dict(most=-1), dict(most=2 ** 28), dict(q=None), dict(k=None), dict(pages=None), dict(n=None), dict(window=-1), dict(sinks=-1),
                dict(scale=0.0), dict(scale=float("nan")), dict(out=None), dict(most=5000, work=None)):
        assert paged(**bad) == 1, bad
    size = dll.dk_attention_paged_work_bytes
    assert size(2, 4, 2, 64, 16, 3, 0, 0) == 0 and size(2, 4, 2, 64, 16, 5000, 0, 0) > 0 and size(2, 4, 2, 64, 16, 5000, 100, 4) == 0

    def append(t=1, worlds=3, tokens=3, kv=2, dim=64, count=9, page=16, most=3, k=X, starts=None, kp=X, pages=X, n=X):
        return dll.dk_cache_append(None, t, worlds, tokens, kv, dim, count, page, most, k, 1, 1, X, 1, 1, starts, kp, 1, 1, 1, X, 1, 1, 1,
                                   pages, 1, n)
    assert append(worlds=0, tokens=0) == append(count=0) == append(most=0) == append(tokens=0, starts=X) == 0
    for bad in (dict(t=0), dict(worlds=-1), dict(tokens=-1), dict(tokens=4), dict(kv=0), dict(dim=9), dict(page=12), dict(k=None), dict(kp=None),
                dict(pages=None), dict(n=None), dict(worlds=2 ** 30, tokens=2 ** 30)):
        assert append(**bad) == 1, bad

    def window(t=1, heads=4, kv=2, dim=64, tq=5, tk=5, q=X, starts=X, scale=0.1, w=3, s=0, work=X, scratch=None, seqs=1):
        return dll.dk_attention_window(None, t, heads, kv, dim, seqs, tq, tk, q, 1, 1, X, 1, 1, X, 1, 1, starts, X, scale, w, s, X, None, None,
                                       work, scratch)
    for bad in (dict(t=0), dict(heads=3), dict(kv=0), dict(dim=7), dict(tq=-1), dict(tk=1 << 30), dict(q=None), dict(starts=None),
                dict(scale=0.0), dict(w=-1), dict(s=-1), dict(work=None), dict(tq=300, tk=5000, w=2000)):
        assert window(**bad) == 1, bad
    size = dll.dk_attention_window_scratch_bytes
    assert size(4, 2, 64, 1, 300, 5000, 0, 0, 1) == dll.dk_attention_scratch_bytes(4, 2, 64, 1, 300, 5000, 1)
    assert size(4, 2, 64, 1, 300, 5000, 6000, 4, 1) == size(4, 2, 64, 1, 300, 5000, 0, 0, 1)  # a window as long as the keys
    assert size(4, 2, 64, 9, 5000, 5000, 50, 4, 1) > 0 == size(4, 2, 64, 9, 5000, 5000, 50, 0, 1)


def test_next_states_lie_over_the_states_row_by_row_or_apart():
    dll = torch_ffi.load_library()

    def step(state, next_, worlds=3, channels=8, state_w=8):
        return dll.dk_recurrence_step(None, 0, worlds, channels, 0x100000, 8, 0x200000, 8, state, state_w, 0x300000, next_)
    at = 0x400000  # never dereferenced
    for args in (dict(state=at, next_=at, state_w=9), dict(state=at, next_=at, state_w=0), dict(state=at, next_=at + 4), dict(state=at, next_=at - 92),
                 dict(state=at, next_=at + 92), dict(state=at, next_=at - 4, worlds=1)):
        assert step(**args) == 1, args


def _cpu():
    """(x, gate, starts, states), heads of queries and keys, pages with their table and lengths, on the CPU or fake"""
    x, f, a, s = torch.randn(10, 6), torch.randn(10, 6), torch.tensor([0, 4, 10], dtype=I32), torch.randn(2, 6)
    q, k = torch.randn(10, 4, 64).bfloat16(), torch.randn(10, 2, 64).bfloat16()
    pages, table, n = torch.randn(7, 16, 2, 64).bfloat16(), torch.zeros((10, 3), dtype=I32), torch.zeros(10, dtype=I32)
    return (x, f, a, s), (q, k), (pages, table, n)


def test_no_cpu_path():
    (x, f, a, s), (q, k), (pages, table, n) = _cpu()
    for call in (lambda: policy.recurrence(x, f, a, s), lambda: policy.recurrence(x.requires_grad_(), f, a),
                 lambda: policy.recurrence_step(x.detach(), f, x.detach()), lambda: policy.gated_residual(x.detach(), f),
                 lambda: policy.attention(q, k, k, a, window=3), lambda: policy.attention_paged(q, pages, pages, table, n),
                 lambda: policy.cache_append_(pages, pages.clone(), k, k, table, n), lambda: policy.recurrence(None, f, a),
                 lambda: policy.recurrence_step(x.detach(), f, None), lambda: policy.gated_residual(x.detach(), None),
                 lambda: policy.attention_paged(None, pages, pages, table, n), lambda: policy.cache_append_(pages, None, k, k, table, n)):
        with pytest.raises(TypeError):
            call()
    for call in (lambda: policy.attention(q, k, k, a, window=0), lambda: policy.attention(q, k, k, a, window=4, sinks=-1),
                 lambda: policy.attention_paged(q, pages, pages, table, n, window=-2),
                 lambda: policy.gated_residual(x.detach(), f, eps=float("nan"))):
        with pytest.raises(ValueError):
            call()


def test_fake_shapes():
    from torch._subclasses.fake_tensor import FakeTensorMode
    ops = policy._ops(True)
    with FakeTensorMode():
        (x, f, a, s), (q, k), (pages, table, n) = _cpu()
        x, f = x.bfloat16(), f.bfloat16()
        h, last = ops.recurrence(x, f, a, s)
        assert h.shape == x.shape and h.dtype == BF16 and last.shape == (2, 6) and last.dtype == F32
        h, last, carry = ops.recurrence_forward(x, f, a, None)
        assert carry.dtype == F32 and last.shape == (2, 6)
        dx, df, di = ops.recurrence_backward(h, None, x, f, a, s, carry, True, False, True)
        assert dx.shape == x.shape and dx.dtype == BF16 and df.shape == (0,) and di.shape == (2, 6) and di.dtype == F32
        h, new = ops.recurrence_step(x, f, torch.randn(10, 6))
        assert h.dtype == BF16 and new.dtype == F32 and h.shape == new.shape == x.shape
        w = torch.randn(6)
        y, z, stats = ops.gated_residual_forward(x, f, w, None, f, None, 1e-5, True)
        assert y.shape == z.shape == x.shape and z.dtype == BF16 and stats.shape == (2, 10) and stats.dtype == F32
        assert ops.gated_residual_forward(x, f, w, None, f, None, 1e-5, False)[2].shape == (2, 0)
        g = ops.gated_residual_backward(y, None, x, f, w, None, f, None, stats, 0b010101)
        assert [t.shape for t in g] == [x.shape, (0,), (6,), (0,), x.shape, (0,)] and g[0].dtype == BF16 and g[2].dtype == F32
        out, lse, work, rest = ops.attention_window_forward(q, k, k, a, a, 0.125, 30, 4, True)
        assert out.shape == rest.shape == q.shape and lse.shape == (4, 10) and work.dtype == I32
        assert ops.attention_window_forward(q, k, k, a, a, 0.125, 100, 4, True)[3].shape == (0,)
        assert [t.shape for t in ops.attention_window_backward(q, q, k, k, a, a, out, lse, work, rest, 0.125, 30, 4)] == [
            q.shape, k.shape, k.shape]
        assert ops.attention_paged(q, pages, pages, table, n, 0.125, 0, 0).shape == q.shape
        assert ops.cache_append_(pages, pages, k, k, table, n, None) is None


def test_windows_of_any_length_are_taken():
    """A window or sinks past what an operator's integers hold are more than any sequence has."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    ops = policy._ops(True)
    with FakeTensorMode():
        (_, _, a, _), (q, k), (pages, table, n) = _cpu()
        for window, sinks in ((2 ** 63 - 1, 4), (2 ** 70, 0), (5, 2 ** 70), (2 ** 70, 2 ** 70)):
            w, s = policy._sight(window, sinks)
            out, _, _, rest = ops.attention_window_forward(q, k, k, a, a, 0.125, w, s, True)
            assert out.shape == q.shape and rest.shape == (0,)
            assert ops.attention_paged(q, pages, pages, table, n, 0.125, w, s).shape == q.shape


def test_fake_carry_is_the_librarys():
    dll = torch_ffi.load_library()
    for tokens in (0, 1, 63, 64, 65, 1000, 2 ** 30):
        for channels in (1, 64, 1000):
            assert 4 * policy._carry_words(tokens, channels) == dll.dk_recurrence_carry_bytes(tokens, channels)


def _differentiable():
    """(call, its first argument) of the operators with gradients, on what is made under a FakeTensorMode"""
    (x, f, a, s), (q, k), _ = _cpu()
    w = torch.randn(6)
    return ((lambda x: policy.recurrence(x, f, a, s)[0], x), (lambda s: policy.recurrence(x, f, a, s)[1], s),
            (lambda x: policy.gated_residual(x, f, w, w, gate=f, scale=w)[1], x), (lambda g: policy.gated_residual(x, f, gate=g)[0], x.clone()),
            (lambda q: policy.attention(q, k, k, a, window=3, sinks=1), q))


def test_forward_mode_raises():
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.autograd import forward_ad
    ops = policy._ops(True)
    with FakeTensorMode():
        (x, f, a, s), (q, k), (pages, table, n) = _cpu()
        others = ((lambda x: policy.recurrence_step(x, f, f)[0], x), (lambda q: policy.attention_paged(q, pages, pages, table, n), q),
                  (lambda k: policy.cache_append_(pages, pages.clone(), k, k, table, n), k),
                  (lambda x: ops.recurrence_forward(x, f, a, None)[0], x))
        for call, at in (*_differentiable(), *others):
            with forward_ad.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
                call(forward_ad.make_dual(at.clone(), at))
        for call, at in _differentiable():
            y = call(at.clone().requires_grad_())
            with forward_ad.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
                y.backward(forward_ad.make_dual(torch.ones_like(y), torch.ones_like(y)))


def test_second_order_raises():
    from torch._subclasses.fake_tensor import FakeTensorMode
    policy._ops(True)
    with FakeTensorMode():
        for call, at in _differentiable():
            x = at.clone().requires_grad_()
            g, = torch.autograd.grad(call(x).float().sum(), x, create_graph=True)
            assert g.requires_grad
            with pytest.raises(RuntimeError, match="differentiated again"):
                (g.float().square().sum() + x.float().sum()).backward()
            assert not torch.autograd.grad(call(x).float().sum(), x)[0].requires_grad


def test_what_has_no_gradient():
    from torch._subclasses.fake_tensor import FakeTensorMode
    ops = policy._ops(True)
    with FakeTensorMode():
        (x, f, a, s), (q, k), (pages, table, n) = _cpu()
        for call, at in ((lambda x: policy.recurrence_step(x, f, f), x), (lambda q: policy.attention_paged(q, pages, pages, table, n), q),
                         (lambda k: policy.cache_append_(pages, pages.clone(), k, k, table, n), k),
                         (lambda x: ops.recurrence_forward(x, f, a, None), x), (lambda x: ops.recurrence_step(x, f, f), x),
                         (lambda q: ops.attention_window_forward(q, k, k, a, a, 0.1, 3, 0, True), q),
                         (lambda q: ops.attention_paged(q, pages, pages, table, n, 0.1, 0, 0), q),
                         (lambda k: ops.cache_append_(pages, pages.clone(), k, k, table, n, None), k)):
            with pytest.raises(RuntimeError, match="no gradient"):
                call(at.clone().requires_grad_())
            with torch.no_grad():
                call(at.clone().requires_grad_())


def _compiles(call, inputs, dynamic):
    """How often torch.compile compiles call for the inputs, one list of arguments after another. Compilation needs no GPU; each
    call then ends in the operators' TypeError."""
    from torch._dynamo.backends.debugging import aot_eager
    count = []

    def backend(graph, example):
        count.append(1)
        return aot_eager(graph, example)
    torch._dynamo.reset()
    compiled = torch.compile(call, backend=backend, fullgraph=True, dynamic=dynamic)
    for args in inputs:
        with pytest.raises(TypeError, match="ROCm device"):
            compiled(*args)
    return len(count)


@pytest.mark.parametrize("dynamic", [None, True])
def test_compiled_once_for_all_sizes(dynamic):
    """After the first size torch.compile takes sizes as symbols: two graphs at most (numbers, then symbols; or symbols, and
    again with an option as a number), and one more for attention's short sequences."""
    leaf = lambda *shape, dtype=F32: torch.randn(shape).to(dtype).requires_grad_()  # noqa: E731
    rows = [(leaf(n, 8), leaf(n, 8), torch.zeros(3, dtype=I32), leaf(2, 8)) for n in (4, 60, 900, 7, 11, 3000)]
    assert _compiles(lambda x, f, a, s: sum(t.sum() for t in policy.recurrence(torch.sin(x), f, a, s)), rows, dynamic) <= 2
    rows = [(leaf(n, 5, 8), leaf(n, 5, 8), leaf(8)) for n in (4, 6, 9, 11, 700)]
    assert _compiles(lambda x, u, w: sum(t.sum() for t in policy.gated_residual(torch.sin(x), u, w, w, gate=u)), rows, dynamic) <= 2
    packed = [(leaf(n, 4, 64, dtype=BF16), leaf(n + 1, 2, 64, dtype=BF16), torch.zeros(3, dtype=I32)) for n in (4, 60, 900, 7, 11, 3000, 5000)]
    assert _compiles(lambda q, k, a: policy.attention(q * 2, k, k, a, window=50, sinks=4).float().sum(), packed, dynamic) <= 3
    worlds = [(torch.randn(n, 4, 64).bfloat16(), torch.randn(n + 3, 16, 2, 64).bfloat16(), torch.zeros((n, 5), dtype=I32),
               torch.zeros(n, dtype=I32)) for n in (4, 60, 900, 7)]
    assert _compiles(lambda q, p, t, n: policy.attention_paged(q * 2, p, p, t, n, window=9), worlds, dynamic) <= 2
    assert _compiles(lambda q, p, t, n: policy.recurrence_step(q[:, 0] * 2, q[:, 1], q[:, 2].float()), worlds, dynamic) <= 2


def test_a_library_from_before_these_operators(tmp_path):
    """A library with the other policy operators alone still has those; these raise RuntimeError."""
    old = [n for n in torch_ffi._PROTOTYPES if n not in torch_ffi._MEMORY_PROTOTYPES]
    (tmp_path / "old.c").write_text("".join(f"void {n}(void) {{}}\n" for n in old))
    lib = tmp_path / "old.so"
    subprocess.run(["gcc", "-shared", "-fPIC", "-o", lib, tmp_path / "old.c"], check=True)
    code = ("import pytest, torch\n"
            "from nablaengine_amd import policy, torch_ffi\n"
            "x, a = torch.zeros(2, 3), torch.zeros(2, dtype=torch.int32)\n"
            "with pytest.raises(TypeError, match='ROCm device'):\n"
            "    policy.layer_norm(x)\n"
            "for call in (lambda: policy.recurrence(x, x, a), lambda: policy.gated_residual(x, x)):\n"
            "    with pytest.raises(RuntimeError, match='before this operator'):\n"
            "        call()\n")
    subprocess.run([sys.executable, "-c", code], check=True, cwd=ROOT, env={**os.environ, "DK_TORCH_ARTIFACT": str(lib)})
