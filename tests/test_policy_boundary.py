"""The policy operators without a GPU: the library exports every entry of include/nablaengine_policy.h, the C entries
refuse bad arguments before any launch, the Python calls refuse what is not on a ROCm device, and the operators' fake
implementations give the library's output shapes and types."""
import ctypes
import os
import re
import subprocess
import sys

import pytest
import torch

from nablaengine_amd import policy, torch_ffi

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "nablaengine_policy.h")


def _prototypes():
    """{name: result and arguments, one letter a value} of the header's declarations."""
    txt = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    letter = lambda a: "p" if "*" in a or "hipStream_t" in a else {"long long": "q", "int": "i", "float": "f"}[  # noqa: E731
        a.rsplit(" ", 1)[0]]
    return {m[2]: {"long long": "q", "int": "i"}[m[1]] + ":" + "".join(letter(" ".join(a.split())) for a in m[3].split(","))
            for m in re.finditer(r"(long long|int) (dk_\w+)\(([^;]*?)\);", txt, re.S)}


def test_bindings_are_the_headers():
    protos = _prototypes()
    assert len(protos) == 11
    for name, proto in protos.items():
        assert torch_ffi._PROTOTYPES[name] == proto, name
    dll = torch_ffi.load_library()
    for name in protos:
        assert hasattr(dll, name)


def test_c_entries_refuse_before_any_launch():
    dll = torch_ffi.load_library()
    X = 0x1000  # never dereferenced
    norm = lambda rows=3, n=8, t=0, wt=0, x=X, y=X: dll.dk_layer_norm(None, rows, n, t, x, n, wt, None, None, 1e-5, y, None)  # noqa: E731
    assert norm(rows=0) == 0
    assert norm(rows=-1) == norm(n=0) == norm(t=3) == norm(t=1, wt=2) == norm(x=None) == norm(y=None) == 1
    vjp = lambda rows=3, n=8, t=0, stats=X, dw=X, work=X: dll.dk_layer_norm_vjp(  # noqa: E731
        None, rows, n, t, X, n, X, n, 0, None, stats, None, dw, None, work)
    assert vjp(rows=-1) == vjp(n=0) == vjp(t=-1) == vjp(stats=None) == vjp(work=None) == 1
    assert dll.dk_layer_norm_work_bytes(0, 8, 0) == 0 and dll.dk_layer_norm_work_bytes(3, 8, 0) >= 2 * 8 * 4

    def clip(n=(5,), types=(0,), outs=(0,), g=X, norm=X, work=X, out=X):
        k = len(n)
        ptr = (ctypes.c_void_p * k)(*[g] * k)
        return dll.dk_clip(None, k, ptr, (ctypes.c_longlong * k)(*n), (ctypes.c_int * k)(*types),
                           (ctypes.c_void_p * k)(*[out] * k), (ctypes.c_int * k)(*outs), 1.0, norm, work)
    assert clip(n=(-1,)) == clip(types=(3,)) == clip(outs=(1,)) == clip(g=None) == clip(norm=None) == clip(work=None) == 1
    assert clip(out=None) == clip(n=(5, 5), types=(1, 1), outs=(1, 2)) == 1
    assert dll.dk_clip(None, -1, None, None, None, None, None, 1.0, X, X) == 1

    def attention(t=1, heads=4, kv=2, dim=64, seqs=1, tq=5, tk=5, q=X, starts=X, scale=0.1, work=X, scratch=None):
        return dll.dk_attention(None, t, heads, kv, dim, seqs, tq, tk, q, 1, 1, X, 1, 1, X, 1, 1, starts, X, scale, X, None, work,
                                scratch)
    for bad in (dict(t=0), dict(heads=3), dict(kv=0), dict(dim=7), dict(dim=136), dict(seqs=-1), dict(tq=-1), dict(tk=1 << 30),
                dict(tq=1 << 29), dict(q=None), dict(starts=None), dict(scale=0.0), dict(scale=float("nan")), dict(work=None), dict(tq=300, tk=3000)):
        assert attention(**bad) == 1, bad
    assert dll.dk_attention_work_bytes(4, 2, 64, 1, 5, 5) > 0 and dll.dk_attention_scratch_bytes(4, 2, 64, 1, 5, 5, 1) == 0
    assert dll.dk_attention_scratch_bytes(4, 2, 64, 1, 300, 5000, 0) > 0

    def step(t=1, worlds=2, heads=4, kv=2, dim=64, cap=9, q=X, lengths=X, scale=0.1, work=X):
        return dll.dk_attention_step(None, t, worlds, heads, kv, dim, cap, q, 1, 1, X, 1, 1, 1, X, 1, 1, 1, lengths, scale, X, work)
    assert step(worlds=0) == 0
    for bad in (dict(t=0), dict(worlds=-1), dict(heads=3), dict(dim=9), dict(cap=-1), dict(q=None), dict(lengths=None),
                dict(scale=-1.0), dict(cap=100000, work=None)):
        assert step(**bad) == 1, bad


def test_no_cpu_path():
    x = torch.randn(3, 8)
    a = torch.tensor([0, 3], dtype=torch.int32)
    h = torch.randn(3, 2, 8).bfloat16()
    for call in (lambda: policy.layer_norm(x), lambda: policy.layer_norm(x.requires_grad_()), lambda: policy.grad_norm([a.float()]),
                 lambda: policy.clip_grads_([a.float()], 1.0), lambda: policy.attention(h, h, h, a),
                 lambda: policy.attention_step(h, h[:, None], h[:, None], a[:1]), lambda: policy.layer_norm(None),
                 lambda: policy.grad_norm([None]), lambda: policy.attention(None, h, h, a)):
        with pytest.raises(TypeError):
            call()
    for eps in (-1.0, float("nan"), float("inf")):
        with pytest.raises(ValueError):
            policy.layer_norm(x, eps=eps)


def test_fake_shapes():
    from torch._subclasses.fake_tensor import FakeTensorMode
    ops = policy._ops()
    with FakeTensorMode():
        x, w = torch.empty((4, 5, 9), dtype=torch.bfloat16), torch.empty(9)
        assert ops.layer_norm(x, w, None, 1e-5).shape == x.shape
        y, stats = ops.layer_norm_forward(x, w, None, 1e-5, True)
        assert y.shape == x.shape and y.dtype == x.dtype and stats.shape == (2, 20) and stats.dtype == torch.float32
        assert ops.layer_norm_forward(x, w, None, 1e-5, False)[1].shape == (2, 0)
        dx, dw, db = ops.layer_norm_backward(x, x, w, None, stats, True, True, False)
        assert dx.shape == x.shape and dw.shape == (9,) and dw.dtype == torch.float32 and db.shape == (0,)
        assert ops.grad_norm([x, w]).shape == () and ops.clip_grads_out([x], [x.float()], 1.0).dtype == torch.float32
        q, k = torch.empty((7, 4, 64), dtype=torch.float16), torch.empty((9, 2, 64), dtype=torch.float16)
        a = torch.empty(4, dtype=torch.int32)
        out, lse, work = ops.attention_forward(q, k, k, a, a, 0.125, True)
        assert out.shape == q.shape and lse.shape == (4, 7) and work.dtype == torch.int32
        assert [t.shape for t in ops.attention_backward(q, q, k, k, a, a, out, lse, work, 0.125)] == [q.shape, k.shape, k.shape]
        assert ops.attention_step(q, k[:7, None], k[:7, None], a, 0.125).shape == q.shape


def _differentiable():
    """(call, its first argument) of the operators with gradients, on what is made under a FakeTensorMode"""
    x, w, b = torch.randn(4, 8), torch.randn(8), torch.randn(8)
    q, k, a = torch.randn(5, 2, 8).bfloat16(), torch.randn(5, 1, 8).bfloat16(), torch.zeros(2, dtype=torch.int32)
    return ((lambda x: policy.layer_norm(x, w, b), x), (lambda q: policy.attention(q, k, k, a), q))


def test_forward_mode_raises():
    """A tangent is never dropped: not by an operator without gradients, not by a tensor that does not require grad, not in
    the backward."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.autograd import forward_ad
    ops = policy._ops()
    with FakeTensorMode():
        x, n = torch.randn(4, 8), torch.zeros(5, dtype=torch.int32)
        q, k = torch.randn(5, 2, 8).bfloat16(), torch.randn(5, 3, 1, 8).bfloat16()
        others = ((lambda g: policy.grad_norm([g]), x), (lambda g: policy.clip_grads_([g], 1.0), x),
                  (lambda g: policy.clip_grads_([g], 1.0, out=[x.clone()]), x), (lambda q: policy.attention_step(q, k, k, n), q),
                  (lambda x: ops.layer_norm_forward(x, None, None, 1e-5, True)[0], x))
        for call, at in (*_differentiable(), *others):
            with pytest.raises(RuntimeError, match="forward-mode"):
                torch.func.jvp(call, (at,), (at.clone(),))
            with forward_ad.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
                call(forward_ad.make_dual(at.clone(), at))
        for call, at in _differentiable():
            y = call(at.clone().requires_grad_())
            with forward_ad.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
                y.backward(forward_ad.make_dual(torch.ones_like(y), torch.ones_like(y)))


def test_second_order_raises():
    """A gradient that is differentiated again raises, also where the loss reaches the input on another path; without
    create_graph it is a plain tensor, and under it one of inputs that need none."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    policy._ops()
    with FakeTensorMode():
        for call, at in _differentiable():
            x = at.clone().requires_grad_()
            g, = torch.autograd.grad(call(x).float().sum(), x, create_graph=True)
            assert g.requires_grad
            with pytest.raises(RuntimeError, match="differentiated again"):
                (g.float().square().sum() + x.float().sum()).backward()
            dy = at.clone().requires_grad_()
            g, = torch.autograd.grad(call(x), x, dy, create_graph=True)
            with pytest.raises(RuntimeError, match="differentiated again"):
                torch.autograd.grad(g.float().sum(), dy)
            assert not torch.autograd.grad(call(x).float().sum(), x)[0].requires_grad


def test_the_nodes_operators_have_no_gradient():
    from torch._subclasses.fake_tensor import FakeTensorMode
    ops = policy._ops()
    with FakeTensorMode():
        x = torch.randn(4, 8, requires_grad=True)
        with pytest.raises(RuntimeError, match="no gradient"):
            ops.layer_norm_forward(x, None, None, 1e-5, True)
        with torch.no_grad():
            ops.layer_norm_forward(x, None, None, 1e-5, True)
        q, k, n = torch.randn(5, 2, 8).bfloat16(), torch.randn(5, 3, 1, 8).bfloat16(), torch.zeros(5, dtype=torch.int32)
        with pytest.raises(RuntimeError, match="no gradient"):
            ops.attention_step(q.requires_grad_(), k, k, n, 0.5)


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
    """After the first size torch.compile takes sizes as symbols: the operators, their nodes and their fake implementations
    read none of them as a number. Two graphs at most (numbers, then symbols; or symbols, and again with layer_norm's eps as
    a number), and one more for attention's short sequences."""
    leaf = lambda *shape, dtype=torch.float32: torch.randn(shape).to(dtype).requires_grad_()  # noqa: E731
    half = torch.bfloat16
    rows = [(leaf(n, 5, 8), leaf(8), leaf(8)) for n in (4, 6, 9, 11, 700)]
    assert _compiles(lambda x, w, b: policy.layer_norm(torch.sin(x), w, b).sum(), rows, dynamic) <= 2
    packed = [(leaf(n, 4, 64, dtype=half), leaf(n + 1, 2, 64, dtype=half), torch.zeros(3, dtype=torch.int32))
              for n in (4, 60, 900, 7, 11, 3000, 5000)]
    assert _compiles(lambda q, k, a: policy.attention(q * 2, k, k, a).float().sum(), packed, dynamic) <= 3
    worlds = [(torch.randn(n, 4, 64).bfloat16(), torch.randn(n, 9, 2, 64).bfloat16(), torch.zeros(n, dtype=torch.int32))
              for n in (4, 60, 900, 7)]
    assert _compiles(lambda q, k, n: policy.attention_step(q * 2, k, k, n), worlds, dynamic) <= 2
    assert _compiles(lambda g: policy.clip_grads_([g], 0.5), [(torch.randn(n, 3),) for n in (4, 60, 900)], dynamic) <= 2


def test_options_that_change_under_compile():
    x, h = torch.randn(4, 8, requires_grad=True), torch.randn(4, 2, 8).bfloat16()
    a = torch.zeros(2, dtype=torch.int32)
    for dynamic in (None, True):
        for call, at in ((lambda x, o: policy.layer_norm(torch.sin(x), eps=o).sum(), x),
                         (lambda h, o: policy.attention(h * 2, h, h, a, scale=o), h), (lambda g, o: policy.clip_grads_([g], o), h)):
            _compiles(call, [(at, o) for o in (0.1, 0.25, 0.5)], dynamic)


def test_fake_order_is_the_librarys():
    dll = torch_ffi.load_library()
    for heads, kv in ((1, 1), (8, 2), (6, 2), (70, 1)):
        for dim in (8, 64, 72, 128):
            for seqs, tq, tk in ((0, 0, 0), (0, 5, 9), (1, 1, 1), (1, 300, 5000), (3, 96, 288), (3, 96, 289), (4096, 70001, 130000),
                                 (1 << 20, 1 << 24, 1 << 27)):
                want = dll.dk_attention_work_bytes(heads, kv, dim, seqs, tq, tk)
                assert 4 * policy._order_words(heads // kv, dim, seqs, tq, tk) == want, (heads, kv, dim, seqs, tq, tk)


def test_a_library_without_the_policy_entries(tmp_path):
    """A library built before these operators still runs the step; the operators raise RuntimeError."""
    step = [n for n in torch_ffi._PROTOTYPES if n not in _prototypes()]
    (tmp_path / "old.c").write_text("".join(f"void {n}(void) {{}}\n" for n in step))
    lib = tmp_path / "old.so"
    subprocess.run(["gcc", "-shared", "-fPIC", "-o", lib, tmp_path / "old.c"], check=True)
    code = ("import pytest, torch\n"
            "from nablaengine_amd import policy, torch_ffi\n"
            "assert torch_ffi.load_library().dk_fwd_forward and torch_ffi.rec_words() == 0\n"
            "for call in (lambda: policy.layer_norm(torch.zeros(2, 3)), lambda: policy.grad_norm([torch.zeros(3)])):\n"
            "    with pytest.raises(RuntimeError, match='before the policy operators'):\n"
            "        call()\n")
    subprocess.run([sys.executable, "-c", code], check=True, cwd=ROOT, env={**os.environ, "DK_TORCH_ARTIFACT": str(lib)})


@pytest.mark.parametrize("order", ["policy, torch_ffi\ntorch_ffi.load_library()", "torch_ffi\ntorch_ffi.load_library()\n"
                                   "from nablaengine_amd import policy"])
def test_ready_with_the_library(order):
    """The operators are ready once the library is loaded, before or after their module: the first call may be a compiled
    one, or one by the operator's name."""
    code = (f"import pytest, torch\nfrom nablaengine_amd import {order}\n"
            "f = torch.compile(lambda x: policy.layer_norm(x) * 2, fullgraph=True, backend='aot_eager')\n"
            "with pytest.raises(TypeError, match='ROCm device'):\n"
            "    f(torch.zeros(2, 3))\n"
            "assert policy._bound\n")
    subprocess.run([sys.executable, "-c", code], check=True, cwd=ROOT)


def test_both_libraries_are_readable_alike():
    """What one user builds another may load: the torch side has the kernels' library's permissions."""
    mode = lambda path: os.stat(path).st_mode & 0o555  # noqa: E731
    assert mode(policy.TORCH_LIB) == mode(torch_ffi.LIB_PATH)
