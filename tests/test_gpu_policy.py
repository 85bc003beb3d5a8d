"""The policy operators on a GPU against their definitions in float64, at the sizes, strides and masks where they can go
wrong. Tolerances follow from the operators' roundings: U[type] is half a unit in the last place relative to the value
(2^-24, 2^-8, 2^-11); an output is rounded once; sums in float32 of n terms are off by at most about (terms a lane + log2
lanes) 2^-24 of the sum of magnitudes, for which SUM = 64 2^-24 stands at every size here; attention's probabilities and
score gradients are rounded to the inputs' type before they are multiplied, which the bounds carry through."""
import math
import random

import pytest
import torch

from nablaengine_amd import policy

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
U = {F32: 2.0 ** -24, BF16: 2.0 ** -8, F16: 2.0 ** -11}
SUM = 64 * 2.0 ** -24
TINY = {F32: 1e-37, BF16: 1e-37, F16: 2.0 ** -24}  # a value rounded to the type's smallest steps


@pytest.fixture(autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.fail("no GPU visible")


def rand(shape, dtype=F32, seed=0, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda", dtype=torch.float64) * scale).to(dtype)


def within(name, got, want, bound):
    got, want = got.double(), want.double()
    assert torch.isfinite(got).all(), f"{name}: not finite"
    over = (got - want).abs() - bound
    assert (over <= 0).all(), f"{name}: {int((over > 0).sum())} values off, the worst {over.max().item():.3g} over its bound"


# ---- layer norm -----------------------------------------------------------------------------------------------------

def norm64(x, w, b, eps):
    x = x.double()
    mean = x.mean(-1, keepdim=True)
    r = 1 / ((x - mean).square().mean(-1, keepdim=True) + eps).sqrt()
    xh = (x - mean) * r
    return xh * (1 if w is None else w.double()) + (0 if b is None else b.double()), xh, r, mean


def check_norm(x, w, b, dy, eps=1e-5):
    leaves = [t.detach().requires_grad_() for t in (x, w, b) if t is not None]
    xl = leaves[0]
    wl = leaves[1] if w is not None else None
    bl = leaves[-1] if b is not None else None
    y = policy.layer_norm(xl, wl, bl, eps=eps)
    grads = dict(zip([n for n, t in (("x", x), ("w", w), ("b", b)) if t is not None],
                     torch.autograd.grad(y, leaves, dy)))
    with torch.no_grad():
        assert torch.equal(y, policy.layer_norm(x, w, b, eps=eps))
    want, xh, r, mean = norm64(x, w, b, eps)
    u = U[x.dtype]
    wd = 1.0 if w is None else w.double()
    # xh from a mean that is off by SUM of the row's mean magnitude
    dxh = SUM * (r * x.double().abs().mean(-1, keepdim=True) + xh.abs() + 1)
    within("y", y, want, u * want.abs() + dxh * (wd if w is None else wd.abs()) + SUM * want.abs() + TINY[x.dtype])
    g, d = dy.double() * wd, dy.double()
    q = (g * xh).mean(-1, keepdim=True)
    dx = r * (g - g.mean(-1, keepdim=True) - xh * q)
    size = r * (g.abs() + g.abs().mean(-1, keepdim=True) + xh.abs() * (g * xh).abs().mean(-1, keepdim=True))
    rough = r * ((g.abs() * dxh).mean(-1, keepdim=True) * xh.abs() + q.abs() * dxh)
    within("dx", grads["x"], dx, u * dx.abs() + 2 * SUM * size + 2 * rough + TINY[x.dtype])
    n = x.shape[-1]
    if w is not None:
        dw = (d * xh).reshape(-1, n).sum(0)
        within("dw", grads["w"], dw, U[w.dtype] * dw.abs() + (SUM * (d * xh).abs() + d.abs() * dxh).reshape(-1, n).sum(0)
               + TINY[w.dtype])
    if b is not None:
        db = d.reshape(-1, n).sum(0)
        within("db", grads["b"], db, U[b.dtype] * db.abs() + SUM * d.abs().reshape(-1, n).sum(0) + TINY[b.dtype])


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("width", [1, 2, 7, 8, 9, 31, 32, 33, 63, 64, 65, 99, 127, 128, 129, 255, 257, 511, 512, 513, 1023,
                                   1025, 2047, 2049, 4095, 4097, 8191, 8193, 16385])
def test_norm_widths(dtype, width):
    """Every group size and both sides of each change between them, the wide rows' kernels among them."""
    print("norm", dtype, width, flush=True)
    rows = 37 if width < 4096 else 5
    x = rand((rows, width), dtype, width, 2.0) + 0.5
    check_norm(x, rand((width,), F32, 1), rand((width,), F32, 2), rand((rows, width), dtype, 3))


@pytest.mark.parametrize("rows,width", [(1, 99), (2, 512), (3000, 99), (9000, 16), (20000, 64), (2100, 256), (1100, 1000),
                                        (700, 2050)])
def test_norm_rows(rows, width):
    """From one row to more than the backward's workgroups take at once."""
    print("norm rows", rows, width, flush=True)
    check_norm(rand((rows, width), F32, rows), rand((width,), F32, 1), rand((width,), F32, 2), rand((rows, width), F32, 3))


@pytest.mark.parametrize("params", ["none", "weight", "bias", "both", "half"])
def test_norm_parameters(params):
    w = rand((77,), BF16 if params == "half" else F32, 1) if params in ("weight", "both", "half") else None
    b = rand((77,), BF16 if params == "half" else F32, 2) if params in ("bias", "both", "half") else None
    check_norm(rand((65, 77), BF16, 4), w, b, rand((65, 77), BF16, 5))


def test_norm_strides_and_alignments():
    """Slices of wider buffers at odd offsets, more dimensions, cotangents with their own strides; what is not evenly
    spaced is refused."""
    for dtype in (F32, BF16, F16):
        wide = rand((50, 131), dtype, 6)
        for off in (0, 1, 3, 8):
            check_norm(wide[:, off:off + 99], rand((99,), F32, 1), rand((100,), F32, 2)[1:], rand((50, 104), dtype, 7)[:, 5:])
    check_norm(rand((4, 9, 3, 40), F32, 8), rand((40,), F32, 1), None, rand((4, 9, 3, 40), F32, 9))
    check_norm(rand((4, 9, 48), F32, 8)[..., :40], rand((40,), F32, 1), None, rand((4, 9, 40), F32, 9))
    check_norm(rand((1, 24), F32, 8).expand(7, 24), None, None, rand((7, 24), F32, 9))  # one row, seven times
    dy = rand((24, 30), F32, 10).t()  # columns apart: the backward takes a contiguous copy
    x = rand((30, 24), F32, 11).requires_grad_()
    g = torch.autograd.grad(policy.layer_norm(x), x, dy)[0]
    assert torch.equal(g, torch.autograd.grad(policy.layer_norm(x), x, dy.contiguous())[0])
    with pytest.raises(TypeError):
        policy.layer_norm(rand((24, 30)).t())
    with pytest.raises(TypeError):
        policy.layer_norm(rand((4, 6, 10)).transpose(0, 1))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("rows", [1, 2, 3, 16385, 16387, 40001])
def test_norm_groups_of_two_waves(dtype, rows):
    """16-bit rows of 513 to 1024 elements share a workgroup of two groups, which meet at barriers: odd numbers of rows, fewer
    than the launch's groups and more, leave the last workgroup's second group without a row."""
    for width in (520, 777, 1024):
        print("norm two waves", dtype, rows, width, flush=True)
        x = rand((rows, width), dtype, rows + width, 2.0) + 0.5
        y, stats = policy._ops().layer_norm_forward(x, None, None, 1e-5, True)
        want, xh, r, mean = norm64(x, None, None, 1e-5)
        dxh = SUM * (r * x.double().abs().mean(-1, keepdim=True) + xh.abs() + 1)
        within("y", y, want, U[dtype] * want.abs() + dxh + SUM * want.abs() + TINY[dtype])
        within("mean", stats[0], mean[:, 0], SUM * x.double().abs().mean(-1))
        within("deviation", stats[1], r[:, 0], 4 * SUM * r[:, 0])


@pytest.mark.parametrize("width,rows", [(2 ** 31 - 1, 1), (2 ** 30 + 5, 1), (2 ** 27 + 3, 2)])
def test_norm_widest_rows(width, rows):
    """Rows up to the longest that is taken. Of alternating 1 and -1 with whole-number parameters and cotangents: each sum of
    x, of its squares and of g is of whole numbers that float32 holds, the outputs but dx are exact after rounding to
    bfloat16. The sum of g xh takes a thread 2^18 steps at most, each off by half a unit of what it has so far."""
    print("norm widest", width, rows, flush=True)
    one = torch.ones((rows, width), dtype=BF16, device="cuda")
    x, dy, w, b = one.clone(), one.clone(), one[0].clone(), one[0].clone()
    x[:, 1::2], dy[:, ::5], w[::3] = -1, 3, 2
    b[:] = 8  # no sum near zero
    b[::7] = 16
    del one
    leaves = [t.requires_grad_() for t in (x, w, b)]
    y = policy.layer_norm(*leaves)
    dx, dw, db = torch.autograd.grad(y, leaves, dy)
    x, w, b, y = (t.detach() for t in (x, w, b, y))
    for i in range(0, width, 2 ** 28):
        c = slice(i, min(i + 2 ** 28, width))
        assert torch.equal(y[:, c], x[:, c] * w[c] + b[c]), c
        assert torch.equal(dw[c], (dy[:, c] * x[:, c]).sum(0)) and torch.equal(db[c], dy[:, c].sum(0)), c
    sums = [[0.0] * rows for _ in range(3)]
    for i in range(0, width, 2 ** 28):
        c = slice(i, min(i + 2 ** 28, width))
        for r in range(rows):
            g = dy[r, c].double() * w[c].double()
            for s, t in zip(sums, (g, g * x[r, c].double(), g.abs())):
                s[r] += t.sum().item() / width
    for i in range(0, width, 2 ** 28):
        c = slice(i, min(i + 2 ** 28, width))
        for r in range(rows):
            xh = x[r, c].double() / math.sqrt(1 + 1e-5)
            g = dy[r, c].double() * w[c].double()
            want = (g - sums[0][r] - xh * sums[1][r]) / math.sqrt(1 + 1e-5)
            within("dx", dx[r, c], want, U[BF16] * want.abs() + 2.0 ** -6 * sums[2][r] + 1e-4)


def test_norm_extremes():
    """Constant rows (variance 0), a large mean, large and small values, rows that hold inf or NaN and their neighbours."""
    x = torch.full((3, 100), 7.25, device="cuda")
    assert torch.equal(policy.layer_norm(x, None, rand((100,), F32, 1)), rand((100,), F32, 1).expand(3, 100))
    big = rand((16, 333), F32, 2) + 1000.0  # the squares about the mean: no cancellation of mean squares
    want, xh, r, _ = norm64(big, None, None, 1e-5)
    within("offset rows", policy.layer_norm(big), want, SUM * (r * 1000 + 1 + xh.abs()))
    for scale in (1e-12, 1e12):
        z = rand((16, 333), F32, 3, scale)
        want, xh, r, _ = norm64(z, None, None, 0.0)
        within("scaled rows", policy.layer_norm(z, eps=0.0), want, 2 * SUM * (1 + xh.abs()))
    bad = rand((5, 70), F32, 4)
    bad[1, 3], bad[3, 69] = math.inf, math.nan
    y = policy.layer_norm(bad)
    assert torch.isnan(y[[1, 3]]).all() and torch.equal(y[[0, 2, 4]], policy.layer_norm(bad[[0, 2, 4]]))


def test_norm_empty_and_partial_gradients():
    w, b = rand((9,), F32, 1).requires_grad_(), rand((9,), F32, 2).requires_grad_()
    x = torch.empty((0, 9), device="cuda", requires_grad=True)
    y = policy.layer_norm(x, w, b)
    gx, gw, gb = torch.autograd.grad(y, (x, w, b), torch.empty_like(y))
    assert y.shape == gx.shape == (0, 9) and not gw.any() and not gb.any()
    x = rand((40, 9), F32, 3)
    full = torch.autograd.grad(policy.layer_norm(x.clone().requires_grad_(), w, b).sum(), (w, b))
    only = torch.autograd.grad(policy.layer_norm(x, w, b.detach()).sum(), w)[0]
    assert torch.equal(full[0], only)
    xr = x.clone().requires_grad_()
    assert torch.autograd.grad(policy.layer_norm(xr, w.detach(), b.detach()).square().sum(), xr)[0].shape == x.shape


def test_norm_gradient_is_the_slope():
    """The gradients against central differences of the definition in float64, along random directions."""
    x, w, b, dy = rand((33, 50), F32, 1), rand((50,), F32, 2), rand((50,), F32, 3), rand((33, 50), F32, 4)
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    grads = torch.autograd.grad(policy.layer_norm(*leaves), leaves, dy)
    dirs = [rand(t.shape, torch.float64, 5 + i) for i, t in enumerate((x, w, b))]
    h = 1e-6
    value = lambda s: (norm64(*(t.double() + s * h * d for t, d in zip((x, w, b), dirs)), 1e-5)[0] * dy.double()).sum()  # noqa: E731
    slope = (value(1) - value(-1)) / (2 * h)
    got = sum((g.double() * d).sum() for g, d in zip(grads, dirs))
    size = sum((g.double() * d).abs().sum() for g, d in zip(grads, dirs))
    assert abs(slope - got) <= 1e-6 * size, (slope.item(), got.item())


# ---- the global gradient norm ---------------------------------------------------------------------------------------

def check_clip(grads, limit, out=None):
    want = torch.sqrt(sum(g.double().square().sum() for g in grads)) if grads else 0.0
    factor = min(1.0, limit / (float(want) + 1e-6))
    ref = [g.double() * factor for g in grads]
    n = policy.grad_norm(grads)
    if out is None:
        norm, res = policy.clip_grads_(grads, limit), grads
    else:
        keep = [g.clone() for g in grads]
        norm, res = policy.clip_grads_(grads, limit, out=out), out
        assert all(torch.equal(a, b) for a, b in zip(keep, grads))
    assert torch.equal(n, norm) and norm.dtype == F32 and norm.shape == ()
    assert abs(norm.double() - want) <= 2 * U[F32] * want
    for i, (r, t) in enumerate(zip(res, ref)):
        within(f"gradient {i}", r, t, (U[r.dtype] + 4 * U[F32]) * t.abs() + TINY[r.dtype])


SIZES = [(), (1,), (3,), (0,), (255,), (257,), (4095,), (4096,), (4097,), (64, 65), (3, 0, 2), (100, 123), (70000,), (33, 7, 5)]


@pytest.mark.parametrize("limit", [0.0, 0.5, 1e9])
@pytest.mark.parametrize("types", [(F32,), (BF16,), (F16,), (F32, BF16, F16)])
def test_clip(types, limit):
    grads = [rand(s, types[i % len(types)], i, 0.3) for i, s in enumerate(SIZES)]
    check_clip([g.clone() for g in grads], limit)
    check_clip(grads, limit, out=[torch.full(g.shape, math.nan, device="cuda") for g in grads])
    check_clip(grads, limit, out=[torch.full(g.shape, math.nan, dtype=g.dtype, device="cuda") for g in grads])


def test_clip_many_views():
    """More tensors than a launch takes, views of one flat buffer at odd offsets, transposed ones."""
    n = [(i * 37) % 900 for i in range(700)]
    for dtype in (F32, BF16):
        flat = rand((sum(n) + 1,), dtype, 1)
        grads, at = [], 1
        for k in n:
            grads.append(flat[at:at + k])
            at += k
        copy = [g.clone() for g in grads]
        check_clip(grads, 2.0, out=copy)
        check_clip(grads, 2.0)
    g = rand((60, 50), F32, 2).t()
    check_clip([g], 0.5, out=[torch.empty((60, 50), device="cuda").t()])
    check_clip([rand((40, 6, 5), F32, 3).permute(2, 0, 1)], 0.5)


def test_clip_is_the_same_every_time():
    grads = [rand((3000, 101), F32, i) for i in range(8)]
    outs = [[torch.empty_like(g) for g in grads] for _ in range(2)]
    norms = [policy.clip_grads_(grads, 1.0, out=o) for o in outs]
    assert torch.equal(norms[0], norms[1]) and all(torch.equal(a, b) for a, b in zip(*outs))


def test_clip_of_values_whose_squares_float32_cannot_hold():
    """Exploded and vanished gradients: their norm is that of the definition, and the clipped ones are finite."""
    for scale in (1e30, 1e-30):
        g = [rand((1000,), F32, 1, scale), rand((37,), F32, 2, scale)]
        check_clip([x.clone() for x in g], 1.0)
    g = [torch.full((100,), 3e38, device="cuda")]  # the norm itself is past float32
    assert policy.clip_grads_(g, 1.0).isinf() and abs(g[0].double().norm() - 1) < 1e-5


def test_clip_of_values_that_are_not_finite():
    """As the definition's products: an infinite norm gives zeros, NaN where the gradient is infinite; NaN gives NaN."""
    a, b = rand((300,), F32, 1), rand((5000,), BF16, 2)
    a[7] = -math.inf
    assert policy.clip_grads_([a, b], 1.0).isinf()
    assert torch.isnan(a[7]) and not a[:7].any() and not a[8:].any() and not b.any()
    b[9] = math.nan
    c = rand((300,), F32, 1)
    assert policy.clip_grads_([c, b], 1.0).isnan() and torch.isnan(c).all() and torch.isnan(b).all()


def test_clip_of_parameters():
    ps = [torch.nn.Parameter(rand((50, 3), F32, i)) for i in range(4)]
    for p in ps[:3]:
        p.grad = rand((50, 3), F32, 9)
    want = torch.sqrt(3 * rand((50, 3), F32, 9).double().square().sum())
    assert abs(policy.clip_grad_norm_(iter(ps), 1.0).double() - want) < 1e-5
    assert abs(policy.grad_norm([p.grad for p in ps[:3]]) - 1.0) < 1e-5 and ps[3].grad is None
    assert policy.clip_grad_norm_([ps[3]], 1.0) == 0


def test_clip_past_32_bits():
    n = 2 ** 31 + 4099
    g = torch.full((n,), 2.0, dtype=BF16, device="cuda")
    norm = policy.clip_grads_([g], 1.0)
    assert abs(norm.item() / (2 * math.sqrt(n)) - 1) < 1e-6
    want = torch.tensor(1 / math.sqrt(n)).to(BF16)
    assert (g[:5] == want).all() and (g[-4200:] == want).all() and (g[2 ** 31 - 3:2 ** 31 + 3] == want).all()


def test_clip_refusals():
    g = rand((10,), F32, 1)
    for bad in (-1.0, math.nan):
        with pytest.raises(ValueError):
            policy.clip_grads_([g], bad)
    for grads in ([g.double()], [g, rand((4, 4))[:, :2]], [g[:1].expand(4)], [g.cpu()], [g, 3.0],
                  [g.clone().requires_grad_()]):
        with pytest.raises(TypeError):
            policy.clip_grads_(grads, 1.0)
    with pytest.raises(ValueError):
        policy.clip_grads_([g, g], 1.0)  # written twice
    with pytest.raises(ValueError):
        policy.clip_grads_([g[:6], g[4:]], 1.0)
    with pytest.raises(ValueError):
        policy.clip_grads_([g[:5], g[5:]], 1.0, out=[g[5:], g[:5]])
    with pytest.raises(ValueError):
        policy.clip_grads_([g], 1.0, out=[])
    with pytest.raises(TypeError):
        policy.clip_grads_([g], 1.0, out=[torch.empty(10, dtype=F16, device="cuda")])
    assert policy.clip_grads_([], 1.0) == 0 and policy.grad_norm([]) == 0


# ---- attention ------------------------------------------------------------------------------------------------------

EXP = 2.0 ** -12  # what float32 scores (|s| < 20 here, sums of at most 128 products) put on a probability


def starts(lengths):
    return torch.tensor([0] + list(lengths), dtype=torch.int64).cumsum(0).to(torch.int32).cuda()


def attend64(q, k, v, lq, lk, scale, dout=None):
    """The definition in float64, and the bounds of each output's error: {name: (value, bound)}."""
    u, tiny = U[q.dtype], TINY[q.dtype]
    q, k, v = (x.double() for x in (q, k, v))
    G = q.shape[1] // k.shape[1]
    r = {n: (torch.zeros_like(x), torch.zeros_like(x)) for n, x in (("out", q), ("dq", q), ("dk", k), ("dv", v))}
    aq = ak = 0
    for nq, nk in zip(lq, lk):
        sq, sk = slice(aq, aq + nq), slice(ak, ak + nk)
        aq, ak = aq + nq, ak + nk
        mask = torch.ones(nq, nk, dtype=torch.bool, device=q.device).tril(nk - nq)
        for h in range(q.shape[1]):
            Q, K, V = q[sq, h], k[sk, h // G], v[sk, h // G]
            s = (Q @ K.t() * scale).masked_fill(~mask, -math.inf)
            some = mask.any(1, keepdim=True)
            p = torch.where(some, torch.softmax(torch.where(some, s, 0.0), 1), 0.0) * mask
            o = p @ V
            ob = (u + 2 * EXP) * (p @ V.abs())
            r["out"][0][sq, h], r["out"][1][sq, h] = o, u * o.abs() + ob + tiny
            if dout is None:
                continue
            d = dout.double()[sq, h]
            r["dv"][0][sk, h // G] += p.t() @ d
            r["dv"][1][sk, h // G] += (u + 2 * EXP) * (p.t() @ d.abs())
            dp, delta = d @ V.t(), (d * o).sum(1, keepdim=True)
            ds = p * (dp - delta)
            doff = (d.abs() * (u * o.abs() + ob)).sum(1, keepdim=True) + 2 * SUM * (d.abs() @ V.abs().t())
            dsb = (u + 2 * EXP) * ds.abs() + p * doff
            r["dq"][0][sq, h], r["dq"][1][sq, h] = ds @ K * scale, dsb @ K.abs() * scale
            r["dk"][0][sk, h // G] += ds.t() @ Q * scale
            r["dk"][1][sk, h // G] += dsb.t() @ Q.abs() * scale
    return {n: (x, b + u * x.abs() + tiny if n != "out" else b) for n, (x, b) in r.items()}


def check_attention(q, k, v, lq, lk, scale=None, dout=None, same=False):
    leaves = [x.detach().requires_grad_() for x in (q, k, v)]
    dout = rand(q.shape, q.dtype, 99) if dout is None else dout
    a, b = starts(lq), starts(lk)
    out = policy.attention(*leaves, a, None if same else b, scale=scale)
    grads = torch.autograd.grad(out, leaves, dout)
    with torch.no_grad():
        assert torch.equal(out, policy.attention(q, k, v, a, b, scale=scale))
    want = attend64(q, k, v, lq, lk, 1 / math.sqrt(q.shape[2]) if scale is None else scale, dout)
    for name, got in zip(("out", "dq", "dk", "dv"), (out, *grads)):
        within(name, got, *want[name])


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("heads,kv,dim", [(1, 1, 64), (4, 2, 64), (6, 2, 128), (5, 5, 40), (8, 1, 8), (3, 1, 72), (7, 1, 120), (70, 1, 64),
                                           (130, 1, 128)])
def test_attention_heads(dtype, heads, kv, dim):
    print("attention", dtype, heads, kv, dim, flush=True)
    lq = [1, 33, 70, 0, 129, 5]
    q, k, v = rand((sum(lq), heads, dim), dtype, 1), rand((sum(lq), kv, dim), dtype, 2), rand((sum(lq), kv, dim), dtype, 3)
    check_attention(q, k, v, lq, lq, same=True)


@pytest.mark.parametrize("lq,lk", [([1], [1]), ([1], [300]), ([0], [5]), ([5], [0]), ([300], [1]), ([70, 3], [20, 200]),
                                   ([64], [64]), ([65], [64]), ([64], [65]), ([31, 32, 33], [31, 32, 33]),
                                   ([128], [128]), ([127], [257]), ([129, 1], [127, 640]), ([700], [700]), ([1] * 90, [7] * 90),
                                   ([2, 0, 0, 4], [0, 9, 0, 4]), ([513], [520])])
def test_attention_lengths(lq, lk):
    """One token to several tiles, queries with earlier keys, queries without keys (zeros), keys without queries, ends
    inside and on the tiles' edges."""
    print("attention lengths", lq[:4], lk[:4], flush=True)
    for dim, heads in ((64, 2), (128, 6)):
        q = rand((sum(lq), heads, dim), BF16, 1)
        k, v = rand((sum(lk), 2, dim), BF16, 2), rand((sum(lk), 2, dim), BF16, 3)
        check_attention(q, k, v, lq, lk)


def test_attention_drawn_lengths():
    rng = random.Random(5)
    for seed in range(4):
        lq = [rng.choice([0, 1, 2, 30, 32, 64, 100, rng.randint(1, 400)]) for _ in range(rng.randint(1, 30))]
        lk = [max(0, n + rng.choice([0, 0, 5, 100, -3])) for n in lq]
        print("attention drawn", seed, flush=True)
        q = rand((sum(lq), 4, 64), F16, seed)
        k, v = rand((sum(lk), 2, 64), F16, seed + 10), rand((sum(lk), 2, 64), F16, seed + 20)
        check_attention(q, k, v, lq, lk, scale=0.3)


@pytest.mark.parametrize("dtype,dim,heads", [(BF16, 64, 2), (F16, 128, 6), (BF16, 40, 8)])
@pytest.mark.parametrize("lq,lk", [([1], [4000]), ([5, 60], [1800, 2100]), ([70, 0, 9], [1100, 900, 0]), ([1500], [1500]),
                                   ([1300, 700], [257, 1900]), ([300], [256]), ([129], [5000])])
def test_attention_few_sequences(dtype, dim, heads, lq, lk):
    """Few tiles, long sequences: a tile's keys (rows) are split among workgroups, whose sums a second kernel adds."""
    print("attention few", dtype, dim, heads, lq, lk, flush=True)
    q = rand((sum(lq), heads, dim), dtype, 1)
    k, v = rand((sum(lk), 2, dim), dtype, 2), rand((sum(lk), 2, dim), dtype, 3)
    check_attention(q, k, v, lq, lk)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_attention_few_sequences_what_the_mask_hides(dim, bad):
    """As below for a tile's parts: the last key, which the last row alone sees, and the first row, which sees one key. The
    last row sees every key: what the last key holds reaches every key's gradient, so those are read without it."""
    print("attention few hidden", dim, bad, flush=True)
    n = 1200
    q, dout = rand((n, 2, dim), BF16, 1), rand((n, 2, dim), BF16, 4)
    k, v = rand((n, 1, dim), BF16, 2), rand((n, 1, dim), BF16, 3)
    want = attend64(q, k, v, [n], [n], 1 / math.sqrt(dim), dout)
    q[0], dout[0] = bad, bad

    def check(names):
        leaves = [x.detach().requires_grad_() for x in (q, k, v)]
        out = policy.attention(*leaves, starts([n]))
        got = dict(zip(("out", "dq", "dk", "dv"), (out, *torch.autograd.grad(out, leaves, dout))))
        for name in names:
            within(name, got[name][1:n - 1], want[name][0][1:n - 1], want[name][1][1:n - 1])
    check(("out", "dq", "dk", "dv"))
    k[-1], v[-1] = bad, bad
    check(("out", "dq"))


@pytest.mark.parametrize("dim", [64, 128])
def test_attention_long_sequences(dim):
    """Sequences long enough that their tiles are listed one by one, and enough of them that none is split."""
    print("attention long", dim, flush=True)
    lq, lk = [2500, 1900], [2500, 2100]
    q = rand((sum(lq), 16, dim), BF16, 1)
    k, v = rand((sum(lk), 8, dim), BF16, 2), rand((sum(lk), 8, dim), BF16, 3)
    check_attention(q, k, v, lq, lk)


def test_attention_one_long_among_short():
    """The mean length chooses the key tiles and the order: one sequence far above it, by either rule."""
    for dtype, dim, heads in ((BF16, 64, 8), (F16, 40, 2), (BF16, 128, 4)):
        print("attention one long", dtype, dim, heads, flush=True)
        lq, lk = [3, 0, 1] * 20 + [700] + [2] * 30, [3, 2, 1] * 20 + [900] + [40] * 30
        q = rand((sum(lq), heads, dim), dtype, 1)
        k, v = rand((sum(lk), 2, dim), dtype, 2), rand((sum(lk), 2, dim), dtype, 3)
        check_attention(q, k, v, lq, lk)


def test_attention_strides():
    """Slices of one projection at odd offsets, heads before tokens, a cotangent with its own strides."""
    lq = [40, 0, 77]
    for off in (0, 1, 3):
        both = rand((117, 8 * 64 + 5), BF16, 1)[:, off:off + 512].unflatten(1, (8, 64))
        check_attention(both[:, :4], both[:, 4:6], both[:, 6:], lq, lq, dout=rand((4, 117, 64), BF16, 2).transpose(0, 1))
    q, k = rand((2, 117, 64), BF16, 3).transpose(0, 1), rand((1, 117, 64), BF16, 4).transpose(0, 1)
    check_attention(q, k, k, lq, lq)
    check_attention(q, k.expand(117, 2, 64), k.expand(117, 2, 64), lq, lq)
    x = q.detach().requires_grad_()
    g = torch.autograd.grad(policy.attention(x, k, k, starts(lq)).sum(), x)[0]  # an expanded cotangent
    want = attend64(q, k, k, lq, lq, 0.125, torch.ones_like(q))["dq"]
    within("dq", g, *want)


def test_attention_padding():
    """Tokens past the last sequence: zeros out, zero gradients, and no part in the sequences; no sequences at all."""
    lq = [50, 20]
    q, k, v = (rand((100, n, 64), BF16, n) for n in (4, 2, 2))
    v[70:], k[75:] = math.nan, math.inf
    leaves = [x.detach().requires_grad_() for x in (q, k, v)]
    out = policy.attention(*leaves, starts(lq))
    grads = torch.autograd.grad(out, leaves, rand(q.shape, BF16, 9))
    assert not out[70:].any() and not any(g[70:].any() for g in grads)
    want = attend64(q[:70], k[:70], v[:70], lq, lq, 0.125, rand(q.shape, BF16, 9)[:70])
    for name, got in zip(("out", "dq", "dk", "dv"), (out, *grads)):
        within(name, got[:70], *want[name])
    assert not policy.attention(q, k, v, starts([])).any()
    empty = policy.attention(q[:0], k[:0], v[:0], starts([0, 0]))
    assert empty.shape == (0, 4, 64)


def test_attention_offsets_that_are_wrong_stay_in_bounds():
    """Offsets past the tokens, falling or negative: whatever comes out, it is computed from the tokens alone."""
    q, k, v = (rand((90, n, 64), BF16, n) for n in (2, 1, 1))
    for bad in ([0, 500], [0, 60, 30, 90], [0, -5, 90], [7, 2 ** 31 - 1, -2 ** 31, 3], [0, 90, 0, 90, 0, 90]):
        print("offsets", bad, flush=True)
        leaves = [x.detach().requires_grad_() for x in (q, k, v)]
        out = policy.attention(*leaves, torch.tensor(bad, dtype=torch.int32, device="cuda"))
        torch.autograd.grad(out, leaves, q)
        torch.cuda.synchronize()


@pytest.mark.parametrize("pairs,tq", [(3 << 19, 1 << 18), (1 << 20, 1 << 19)])
def test_attention_offsets_whose_tiles_pass_32_bits(pairs, tq):
    """Offsets that go back and forth over all queries: 3 and 4 times 2^30 tiles where the list holds 3 million. Without
    keys every query's output is zero, whichever of the tiles are computed."""
    print("offsets past 32 bits", pairs, tq, flush=True)
    q, k = rand((tq, 1, 8), BF16, 1), rand((64, 1, 8), BF16, 2)
    a = torch.zeros(2 * pairs + 1, dtype=torch.int32, device="cuda")
    a[1::2] = tq
    out, _, work = policy._ops().attention_forward(q, k, k, a, torch.zeros_like(a), 0.5, True)
    torch.cuda.synchronize()
    entries = work[16:16 + 2 * int(work[0])].view(-1, 2)
    assert 0 <= int(work[0]) <= tq // 128 + 2 * pairs + 1 and 0 <= int(work[1]) <= 64 // 32 + 2 * pairs + 1
    assert ((entries[:, 0] >= 0) & (entries[:, 0] <= 2 * pairs)).all()
    assert ((entries[:, 1] >= 0) & (entries[:, 1] < tq // 128)).all() and not out[:128].any()


def test_attention_sharp_and_equal_scores():
    """Scores far apart (one key takes all), all equal (the mean), and too large for float16's range when exponentiated."""
    lq = [200]
    q, k, v = (rand((200, 1, 64), F16, n) for n in (1, 2, 3))
    out = policy.attention(q * 30, k * 30, v, starts(lq), scale=1.0)
    s = (q[:, 0].double() * 30).to(F16).double() @ (k[:, 0].double() * 30).to(F16).double().t()
    s = s.masked_fill(~torch.ones_like(s, dtype=torch.bool).tril(), -math.inf)
    want = torch.softmax(s, 1) @ v[:, 0].double()
    top = s.sort(1, descending=True).values
    clear = (top[:, 0] - top[:, 1] > 40) | torch.isinf(top[:, 1])
    assert clear.float().mean() > 0.9
    within("sharp", out[clear, 0], want[clear], 2 * U[F16] * want[clear].abs() + 1e-6)
    out = policy.attention(torch.zeros_like(q), k, v, starts(lq))
    want = v[:, 0].double().cumsum(0) / torch.arange(1, 201, device="cuda")[:, None]
    mean = v[:, 0].double().abs().cumsum(0) / torch.arange(1, 201, device="cuda")[:, None]
    within("equal", out[:, 0], want, U[F16] * want.abs() + (U[F16] + EXP) * mean + 1e-7)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("lq,lk,heads", [([1], [100000], 1), ([7] * 40, [3000] * 40, 8), ([7] * 400, [500] * 400, 8)])
def test_attention_many_small_beside_a_large_one(dim, lq, lk, heads):
    """One key whose score is far above all others', whose probabilities are 2^-26 of its own: together they have a part in
    the output (values of 0 there and about 1 at the others), in float16 too, whose smallest step is 2^-24."""
    for dtype in (BF16, F16):
        print("small beside large", dtype, dim, lq[0], lk[0], flush=True)
        q = torch.zeros((sum(lq), heads, dim), dtype=dtype, device="cuda")
        k = torch.zeros((sum(lk), 1, dim), dtype=dtype, device="cuda")
        v = 1 + rand((sum(lk), 1, dim), dtype, 3, 0.1)
        q[..., 0] = 1.0
        first = starts(lk)[:-1].long()
        k[first, :, 0], v[first] = 26.0, 0.0
        out = policy.attention(q, k, v, starts(lq), starts(lk), scale=math.log(2))
        want, bound = attend64(q, k, v, lq, lk, math.log(2))["out"]
        within("out", out, want, bound)
        assert want.abs().min() > 4 * bound.max()  # it is not the bound that hides them


@pytest.mark.parametrize("heads,kv,dim", [(2, 1, 64), (4, 2, 128), (1, 1, 40)])
@pytest.mark.parametrize("lq,lk", [([3000, 40, 1, 0, 700], [3000, 40, 1, 3, 700]), ([1], [20000]), ([30] * 100, [30] * 100),
                                   ([150] * 150, [170] * 150)])
@pytest.mark.parametrize("size", ["2^-18", "2^-10", "1", "2^12", "rising", "falling"])
def test_attention_float16_gradients_of_any_size(size, lq, lk, heads, kv, dim):
    """Cotangents from float16's smallest (a mean loss) to its largest (a scaled one), and of all sizes in one sequence: the
    score gradients, a probability times them, are far outside float16's range. Queries and keys are small and the scale is
    large where cotangents are small, so that the results are inside it."""
    print("float16 gradients", size, lq[:3], heads, dim, flush=True)
    q, k = rand((sum(lq), heads, dim), F16, 1, 0.02), rand((sum(lk), kv, dim), F16, 2, 0.02)
    v, dout = rand((sum(lk), kv, dim), F16, 3), rand(q.shape, torch.float64, 4)
    if size in ("rising", "falling"):
        at = torch.cat([torch.arange(n, device="cuda") / max(n - 1, 1) for n in lq])
        at = 1 - at if size == "falling" else at
        dout = dout * torch.exp2(-16 + 26 * at)[:, None, None]
    else:
        dout = dout * 2.0 ** (0 if size == "1" else int(size[2:]))
    scale = 64.0 if size in ("2^-18", "2^-10") else 1.0
    check_attention(q, k, v, lq, lk, scale=scale, dout=dout.clamp(-6e4, 6e4).to(F16))


def test_attention_keeps_sequences_apart():
    """inf and NaN in one sequence reach no other sequence."""
    lq = [40, 40, 100]
    q, k, v = (rand((180, n, 64), BF16, n) for n in (4, 2, 2))
    dout = rand(q.shape, BF16, 9)

    def run(*xs):
        leaves = [x.detach().clone().requires_grad_() for x in xs]
        out = policy.attention(*leaves, starts(lq))
        return [out, *torch.autograd.grad(out, leaves, dout)]
    clean = run(q, k, v)
    q[50], k[60], v[70], dout[45] = math.nan, math.inf, -math.inf, math.nan
    for a, b in zip(clean, run(q, k, v)):
        assert torch.equal(a[:40], b[:40]) and torch.equal(a[80:], b[80:])


@pytest.mark.parametrize("dtype,dim,heads", [(BF16, 64, 2), (F16, 64, 6), (BF16, 128, 4), (F16, 40, 2)])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_attention_what_the_mask_hides(dtype, dim, heads, bad):
    """A value, key, query or cotangent that is not finite reaches the rows and keys that the mask lets see it, and no
    other of its sequence; an infinite value element reaches its own column only, as itself."""
    print("hidden", dtype, dim, heads, bad, flush=True)
    lq, lk = [150, 70], [150, 75]
    q, dout = rand((220, heads, dim), dtype, 1), rand((220, heads, dim), dtype, 4)
    k, v = rand((225, 2, dim), dtype, 2), rand((225, 2, dim), dtype, 3)
    want = attend64(q, k, v, lq, lk, 1 / math.sqrt(dim), dout)

    def run(q, k, v, dout):
        leaves = [x.detach().requires_grad_() for x in (q, k, v)]
        out = policy.attention(*leaves, starts(lq), starts(lk))
        return dict(zip(("out", "dq", "dk", "dv"), (out, *torch.autograd.grad(out, leaves, dout))))

    def same(got, name, rows, cols=slice(None)):
        w, b = want[name]
        within(f"{name} {rows}", got[name][rows, :, cols], w[rows, :, cols], b[rows, :, cols])
    early, late, other = slice(0, 100), slice(100, 150), slice(150, None)
    v2 = v.clone()
    v2[100, :, 7] = bad
    got = run(q, k, v2, dout)
    for name in ("out", "dq"):
        same(got, name, early), same(got, name, other)
    same(got, "out", late, slice(0, 7)), same(got, "out", late, slice(8, None))
    late7 = got["out"][late, :, 7]
    assert torch.isnan(late7).all() if math.isnan(bad) else (late7 == bad).all()
    same(got, "dv", slice(None))  # no value has a part in the values' gradient
    same(got, "dk", other)
    k2 = k.clone()
    k2[100] = bad
    got = run(q, k2, v, dout)
    for name in ("out", "dq"):
        same(got, name, early), same(got, name, other)
    for name in ("dk", "dv"):
        same(got, name, other)
    d2 = dout.clone()
    d2[40, :, 5] = bad  # row 40 sees keys 0 to 40
    got = run(q, k, v, d2)
    same(got, "out", slice(None))
    for name, rows in (("dq", slice(0, 40)), ("dq", slice(41, None)), ("dk", slice(41, None)), ("dv", slice(41, None))):
        same(got, name, rows)
    same(got, "dv", slice(0, 41), slice(0, 5)), same(got, "dv", slice(0, 41), slice(6, None))
    seen = got["dv"][0:41, :, 5]
    assert torch.isnan(seen).all() if math.isnan(bad) else (seen == bad).all()
    q2 = q.clone()
    q2[40] = bad
    got = run(q2, k, v, dout)
    for name in ("out", "dq"):
        same(got, name, slice(0, 40)), same(got, name, slice(41, None))
    for name in ("dk", "dv"):
        same(got, name, slice(41, None))


def test_attention_is_the_same_every_time():
    lq = [300, 7, 512, 64, 1]
    q, k, v = (rand((sum(lq), n, 64), BF16, n) for n in (4, 2, 2))

    def run():
        leaves = [x.detach().requires_grad_() for x in (q, k, v)]
        out = policy.attention(*leaves, starts(lq))
        return [out, *torch.autograd.grad(out, leaves, q)]
    assert all(torch.equal(a, b) for a, b in zip(run(), run()))


def test_attention_gradient_is_the_slope():
    lq, lk = [20, 45], [33, 45]
    q, k, v = rand((65, 4, 64), F16, 1), rand((78, 2, 64), F16, 2), rand((78, 2, 64), F16, 3)
    dout = rand(q.shape, F16, 4)
    leaves = [x.detach().requires_grad_() for x in (q, k, v)]
    grads = torch.autograd.grad(policy.attention(*leaves, starts(lq), starts(lk)), leaves, dout)
    want = attend64(q, k, v, lq, lk, 0.125, dout)
    for i, name in enumerate(("dq", "dk", "dv")):
        d = rand(leaves[i].shape, torch.float64, 7)
        xs = [x.double() for x in (q, k, v)]

        def value(s):
            ys = list(xs)
            ys[i] = ys[i] + s * d
            return (attend64_out(*ys, lq, lk, 0.125) * dout.double()).sum()
        slope = (value(1e-5) - value(-1e-5)) / 2e-5
        got = (grads[i].double() * d).sum()
        assert abs(slope - got) <= (want[name][1] * d.abs()).sum() + 1e-6 * abs(slope), name


def attend64_out(q, k, v, lq, lk, scale):
    out, aq, ak, G = torch.zeros_like(q), 0, 0, q.shape[1] // k.shape[1]
    for nq, nk in zip(lq, lk):
        mask = torch.ones(nq, nk, dtype=torch.bool, device=q.device).tril(nk - nq)
        for h in range(q.shape[1]):
            s = q[aq:aq + nq, h] @ k[ak:ak + nk, h // G].t() * scale
            out[aq:aq + nq, h] = torch.softmax(s.masked_fill(~mask, -math.inf), 1) @ v[ak:ak + nk, h // G]
        aq, ak = aq + nq, ak + nk
    return out


def test_attention_past_32_bits():
    """Tokens 2^20 elements apart: offsets past 2^31 elements."""
    big = torch.zeros((2200, 2 ** 20), dtype=BF16, device="cuda")
    q, k, v = (rand((2200, 1, 64), BF16, n) for n in (1, 2, 3))
    views = []
    for i, x in enumerate((q, k, v)):
        view = big[:, 64 * i:64 * i + 64].unflatten(1, (1, 64))
        view.copy_(x)
        views.append(view)
    lq = [1000, 1200]

    def run(*xs):
        leaves = [x.detach().requires_grad_() for x in xs]
        out = policy.attention(*leaves, starts(lq))
        return [out, *torch.autograd.grad(out, leaves, q)]
    assert all(torch.equal(a, b) for a, b in zip(run(q, k, v), run(*views)))


def test_attention_refusals():
    q, k, v, a = rand((10, 4, 64), BF16), rand((10, 2, 64), BF16), rand((10, 2, 64), BF16), starts([10])
    for args in ((q.float(), k.float(), v.float(), a), (q, k.half(), v, a), (q, k, v[:9], a), (q, k[:, :, :32], v[:, :, :32], a),
                 (q[:, :3], k, v, a), (q[..., :20], k[..., :20], v[..., :20], a), (q, k, v, a.long()), (q, k, v, a.cpu()),
                 (q, k, v, a, starts([5, 5])), (q, k, v, a[:0]), (q.transpose(1, 2), k, v, a), (q[0], k, v, a), (q.cpu(), k, v, a),
                 (q[..., ::2], k[..., ::2], v[..., ::2], a), (rand((10, 4, 136), BF16), rand((10, 2, 136), BF16),
                                                             rand((10, 2, 136), BF16), a)):
        with pytest.raises(TypeError):
            policy.attention(*args)
    for scale in (0.0, -1.0, math.nan, math.inf):
        with pytest.raises(ValueError):
            policy.attention(q, k, v, a, scale=scale)


def test_attention_sizes_past_one_launch():
    """ValueError, before anything is allocated, for each of the limits (strides of 0: the tensors are small)."""
    def of(tq, tk, kv, seqs, heads=None):
        q, k = (torch.zeros((1, 1, 8), dtype=BF16, device="cuda").expand(n, h, 8) for n, h in ((tq, heads or kv), (tk, kv)))
        a = torch.zeros(seqs + 1, dtype=torch.int32, device="cuda")
        before = torch.cuda.memory_allocated()
        with pytest.raises(ValueError, match="exceed one launch"):
            policy.attention(q, k, k, a)
        assert torch.cuda.memory_allocated() == before
    of(8, 2 ** 27, 1, 1)
    of(8, 2 ** 24, 8, 1)
    of(8, 8, 1, 2 ** 22)
    of(2 ** 29, 8, 1, 1)
    of(2 ** 28, 8, 1, 1, heads=4)
    of(8, 2 ** 30, 1, 1)
    of(2 ** 32 + 5, 8, 1, 1)


# ---- one new token --------------------------------------------------------------------------------------------------

def check_step(q, k, v, lengths, scale=None):
    out = policy.attention_step(q, k, v, torch.tensor(lengths, dtype=torch.int32, device="cuda"), scale=scale)
    scale = 1 / math.sqrt(q.shape[2]) if scale is None else scale
    G, u = q.shape[1] // k.shape[2], U[q.dtype]
    for w, n in enumerate(min(max(n, 0), k.shape[1]) for n in lengths):
        if n == 0:
            assert not out[w].any()
            continue
        K, V = (x[w, :n].double().repeat_interleave(G, 1).transpose(0, 1) for x in (k, v))
        p = torch.softmax((K @ q[w].double()[..., None])[..., 0] * scale, 1)
        want = (p[:, None] @ V)[:, 0]
        within(f"world {w}", out[w], want, u * want.abs() + EXP * (p[:, None] @ V.abs())[:, 0] + TINY[q.dtype])


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("heads,kv,dim", [(1, 1, 64), (8, 2, 64), (6, 2, 128), (5, 5, 40), (16, 1, 8), (3, 1, 72), (9, 1, 128),
                                          (4, 2, 120)])
def test_step_heads(dtype, heads, kv, dim):
    print("step", dtype, heads, kv, dim, flush=True)
    lengths = [0, 1, 31, 32, 33, 127, 128, 129, 300, 301, -4, 9999]
    k, v = rand((12, 301, kv, dim), dtype, 2), rand((12, 301, kv, dim), dtype, 3)
    check_step(rand((12, heads, dim), dtype, 1), k, v, lengths)


@pytest.mark.parametrize("worlds,capacity", [(1, 1), (1, 257), (3, 5000), (2, 40001), (700, 3), (1, 0), (0, 8)])
def test_step_capacities(worlds, capacity):
    """A cache from nothing to one that is cut into many stretches, full, short and empty histories in it."""
    lengths = [[capacity, capacity // 2 + 1, 0, 1][w % 4] for w in range(worlds)]
    k, v = rand((worlds, capacity, 2, 64), BF16, 2), rand((worlds, capacity, 2, 64), BF16, 3)
    check_step(rand((worlds, 4, 64), BF16, 1), k, v, lengths, scale=0.2)


@pytest.mark.parametrize("heads,kv,dim,capacity", [(1, 1, 64, 50), (4, 2, 64, 130), (6, 2, 40, 33), (8, 1, 128, 20), (24, 2, 8, 9)])
def test_step_many_worlds(heads, kv, dim, capacity):
    """Enough worlds that a wave takes each alone."""
    print("step many", heads, kv, dim, capacity, flush=True)
    W = 2049
    q, k, v = (rand((W, *s, dim), BF16, i) for i, s in enumerate(((heads,), (capacity, kv), (capacity, kv))))
    lengths = torch.tensor([(37 * w) % (capacity + 1) for w in range(W)], dtype=torch.int32, device="cuda")
    out = policy.attention_step(q, k, v, lengths)
    K, V = (x.double().repeat_interleave(heads // kv, 2).permute(0, 2, 1, 3) for x in (k, v))
    s = (K * q.double()[:, :, None]).sum(3) / math.sqrt(dim)
    seen = (torch.arange(capacity, device="cuda") < lengths[:, None])[:, None].expand_as(s)
    some = lengths[:, None, None] > 0
    p = torch.softmax(s.masked_fill(~seen & some, -math.inf), 2) * (seen & some)
    want, size = (p[..., None] * V).sum(2), (p[..., None] * V.abs()).sum(2)
    within("out", out, want, U[BF16] * want.abs() + EXP * size + TINY[BF16])


def test_step_reads_only_the_history():
    """What lies past a history (never written memory, NaN, inf) has no part."""
    k, v = rand((5, 900, 2, 64), F16, 2), rand((5, 900, 2, 64), F16, 3)
    lengths = [0, 1, 77, 600, 899]
    for w, n in enumerate(lengths):
        k[w, n:], v[w, n:] = math.nan, math.inf
    check_step(rand((5, 4, 64), F16, 1), k, v, lengths)


def test_step_strides():
    """Keys and values in one buffer at odd offsets, heads before tokens, a query slice."""
    both = rand((6, 70, 4 * 64 + 3), BF16, 2)[..., 3:].unflatten(2, (4, 64))
    q = rand((6, 12, 64), BF16, 1)[:, 2:6]
    check_step(q, both[:, :, :2], both[:, :, 2:], [70, 3, 0, 64, 69, 12])
    k = rand((6, 2, 70, 64), BF16, 4).transpose(1, 2)
    check_step(q, k, k[:1].expand(6, 70, 2, 64), [70, 3, 0, 64, 69, 12])


def test_step_is_attentions_last_row():
    lk = [5, 300, 64]
    q, k, v = rand((3, 4, 64), F16, 1), rand((3, 300, 2, 64), F16, 2), rand((3, 300, 2, 64), F16, 3)
    a = policy.attention_step(q, k, v, torch.tensor(lk, dtype=torch.int32, device="cuda"))
    packed = [torch.cat([x[w, :n] for w, n in enumerate(lk)]) for x in (k, v)]
    b = policy.attention(q, *packed, starts([1, 1, 1]), starts(lk))
    assert (a - b).abs().max() < 4 * U[F16]


def test_scores_that_are_all_minus_infinity():
    """Softmax over scores that are all -inf is 0 / 0: NaN, from an infinite key or from a product past float32, in the rows
    that see no other score and the keys they see; not zeros, which stand for rows without keys."""
    for dtype, dim, low in ((BF16, 64, -math.inf), (BF16, 128, -3e30), (F16, 40, -math.inf)):
        q, k, v = rand((240, 2, dim), dtype, 1), rand((240, 1, dim), dtype, 2), rand((240, 1, dim), dtype, 3)
        lq = [100, 140]
        clean = policy.attention(q, k, v, starts(lq))
        q[:100, :, 0], q[:100, :, 1:] = 3e30 if dtype == BF16 else 1.0, 0.0
        k[:30, :, 0], k[30:100, :, 0] = low, 0.0
        leaves = [x.detach().requires_grad_() for x in (q, k, v)]
        out = policy.attention(*leaves, starts(lq))
        dq, dk, dv = torch.autograd.grad(out, leaves, rand(q.shape, dtype, 4))
        assert torch.isnan(out[:30]).all() and torch.isfinite(out[30:]).all() and torch.equal(out[100:], clean[100:])
        assert torch.isnan(dv[0]).all() and torch.isnan(dq[:30, :, 0]).all()
        assert all(torch.isfinite(g[100:]).all() for g in (dq, dk, dv))
        rows = torch.arange(30, 100, device="cuda")
        mean = v[30:100, 0].double().cumsum(0) / (rows - 29)[:, None]  # the seen keys' scores are 0, the first 30 have no part
        size = v[30:100, 0].double().abs().cumsum(0) / (rows - 29)[:, None]
        within("rows", out[30:100, 0], mean, U[dtype] * mean.abs() + (U[dtype] + EXP) * size + TINY[dtype])
        for capacity in (30, 3000):  # whole, and in stretches
            cache = torch.zeros((3, capacity, 1, dim), dtype=dtype, device="cuda")
            cache[..., 0], cache[2, -1] = low, 0.0
            values = torch.ones_like(cache)
            n = torch.tensor([0, capacity, capacity], dtype=torch.int32, device="cuda")
            got = policy.attention_step(q[:3], cache, values, n)
            assert not got[0].any() and torch.isnan(got[1]).all() and torch.equal(got[2], torch.ones_like(got[2]))


def test_step_past_32_bits():
    cap, worlds = 2 ** 22, 5
    k = torch.zeros((worlds, cap, 1, 128), dtype=BF16, device="cuda")
    v = torch.zeros((worlds, cap, 1, 128), dtype=BF16, device="cuda")
    q = torch.ones((worlds, 2, 128), dtype=BF16, device="cuda")
    k[4, cap - 1], v[4, cap - 1] = 4.0, rand((1, 128), BF16, 1)  # its score, 45, against 0 for the 4 million others
    lengths = torch.tensor([0, 3, 0, 1, cap], dtype=torch.int32, device="cuda")
    out = policy.attention_step(q, k, v, lengths)
    assert torch.equal(out[4, 0], v[4, cap - 1, 0]) and torch.equal(out[4, 1], v[4, cap - 1, 0]) and not out[:4].any()


def test_step_refusals():
    q, k, n = rand((3, 4, 64), BF16), rand((3, 9, 2, 64), BF16), torch.zeros(3, dtype=torch.int32, device="cuda")
    for args in ((q.float(), k.float(), k.float(), n), (q, k, k[:, :8], n), (q[:2], k, k, n[:2]), (q, k, k, n.long()),
                 (q, k, k, n[:2]), (q, k, k, n.cpu()), (q[:, :3], k, k, n), (q, k[..., :60], k[..., :60], n), (q, k[0], k[0], n)):
        with pytest.raises(TypeError):
            policy.attention_step(*args)
    with pytest.raises(RuntimeError):
        policy.attention_step(q.requires_grad_(), k, k, n)
    with torch.no_grad():
        policy.attention_step(q, k, k, n)


# ---- streams, graphs, compilation -----------------------------------------------------------------------------------

def _all_operators():
    x, w, b = rand((300, 99), F32, 1), rand((99,), F32, 2), rand((99,), F32, 3)
    lq = [70, 3, 190]
    q, k, v = (rand((263, n, 64), BF16, n) for n in (4, 2, 2))
    cache, n = rand((6, 600, 2, 64), BF16, 5), torch.tensor([0, 1, 600, 33, 599, 2], dtype=torch.int32, device="cuda")
    a, dout, qs = starts(lq), rand((263, 4, 64), BF16, 6), rand((6, 4, 64), BF16, 7)
    grads = [rand((700, 99), F32, 8), rand((5000,), BF16, 9)]
    out = [torch.empty((700, 99), device="cuda"), torch.empty((5000,), device="cuda")]

    def run():
        xs = [t.detach().requires_grad_() for t in (x, w, b)]
        y = policy.layer_norm(*xs)
        res = [y, *torch.autograd.grad(y, xs, x)]
        ls = [t.detach().requires_grad_() for t in (q, k, v)]
        o = policy.attention(*ls, a)
        res += [o, *torch.autograd.grad(o, ls, dout), policy.attention_step(qs, cache, cache, n)]
        res += [policy.clip_grads_(grads, 0.5, out=out), policy.grad_norm(grads)] + [t.clone() for t in out]
        return [t.detach() for t in res]
    return run, (x, w, b, q, k, v, cache, dout, qs, *grads)


def test_operators_on_another_stream():
    run, _ = _all_operators()
    want = run()
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = run()
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_operators_in_a_graph():
    """Captured once, replayed over new inputs with eager work between the replays."""
    run, inputs = _all_operators()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        run()
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        held = run()
    for turn in range(4):
        for i, t in enumerate(inputs):
            t.copy_(rand(t.shape, t.dtype, 100 * turn + i))
        want = [t.clone() for t in run()]
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        for i, (a, b) in enumerate(zip(want, held)):
            assert torch.equal(a, b), (turn, i)


def test_operators_compiled():
    """torch.compile keeps each operator as one node of a full graph, forward and backward, with eager's results."""
    x, w, b = rand((300, 64), F32, 1), rand((64,), F32, 2), rand((64,), F32, 3)
    lq = [20, 0, 44, 11]
    a, heads = starts(lq), rand((75, 6, 64), BF16, 4)

    def loss(x, w, b, heads):
        y = policy.layer_norm(torch.sin(x), w, b)
        o = policy.attention(heads[:, :2], heads[:, 2:4], heads[:, 4:], a)
        return (y * y).sum() + (o.float() * 3).sum()

    def run(f):
        leaves = [t.detach().requires_grad_() for t in (x, w, b, heads)]
        value = f(*leaves)
        return [value.detach(), *torch.autograd.grad(value, leaves)]
    eager, compiled = run(loss), run(torch.compile(loss, fullgraph=True, backend="aot_eager"))
    for i, (e, c) in enumerate(zip(eager, compiled)):
        assert torch.equal(e, c), i
    grads = [rand((50, 3), F32, 5), rand((7,), F32, 6)]
    clip = torch.compile(lambda g: policy.clip_grads_(g, 0.5) * 2, fullgraph=True, backend="aot_eager")
    one, two = [g.clone() for g in grads], [g.clone() for g in grads]
    assert torch.equal(clip(one), policy.clip_grads_(two, 0.5) * 2) and all(torch.equal(p, q) for p, q in zip(one, two))


def test_operators_compiled_over_sizes():
    """One compiled function over several batches, cotangents in their own strides: eager's results for each."""
    w, b = rand((64,), F32, 2), rand((64,), F32, 3)

    def loss(x, w, b, heads, a):
        y = policy.layer_norm(torch.sin(x), w, b)
        o = policy.attention(heads[:, :2], heads[:, 2:4], heads[:, 4:], a)
        return (y.t() @ y).sum() + (o.float().transpose(0, 2) * 3).cumsum(0).sum()

    def run(f, rows, lq):
        leaves = [t.detach().requires_grad_() for t in (rand((rows, 64), F32, 1), w, b, rand((sum(lq), 6, 64), BF16, 4))]
        value = f(*leaves, starts(lq))
        return [value.detach(), *torch.autograd.grad(value, leaves)]
    torch._dynamo.reset()
    compiled = torch.compile(loss, fullgraph=True, backend="aot_eager")
    for rows, lq in ((300, [20, 0, 44, 11]), (301, [7, 300]), (4, [1]), (77, [500, 900, 2, 2, 2]), (5000, [33] * 40)):
        for i, (e, c) in enumerate(zip(run(loss, rows, lq), run(compiled, rows, lq))):
            assert torch.equal(e, c), (rows, i)


def test_gradients_in_a_graph_of_gradients():
    """Under create_graph the gradients are those without it, and differentiating them again raises."""
    x, w, b, dy = rand((40, 99), F32, 1), rand((99,), F32, 2), rand((99,), F32, 3), rand((40, 99), F32, 4)
    q, k, v = (rand((90, n, 64), BF16, n) for n in (4, 2, 2))
    a, dout = starts([20, 70]), rand((90, 4, 64), BF16, 9)
    for call, at, cot in ((policy.layer_norm, (x, w, b), dy), (lambda *t: policy.attention(*t, a), (q, k, v), dout)):
        leaves = [t.detach().requires_grad_() for t in at]
        want = torch.autograd.grad(call(*leaves), leaves, cot)
        got = torch.autograd.grad(call(*leaves), leaves, cot, create_graph=True)
        assert all(torch.equal(p, r) and r.requires_grad and not p.requires_grad for p, r in zip(want, got))
        with pytest.raises(RuntimeError, match="differentiated again"):
            sum(g.float().square().sum() for g in got).backward()


def test_clipping_marks_what_it_writes():
    """A graph that saved a tensor which clipping then overwrites notices."""
    w = rand((8,), F32, 1).requires_grad_()
    g = rand((8,), F32, 2)
    y = (w * g).sum()
    policy.clip_grads_([g], 0.1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
