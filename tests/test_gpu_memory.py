"""The operators of policies with a longer memory on a GPU against their definitions in float64, at the sizes, strides and
masks where they can go wrong. Tolerances follow from the operators' roundings: U[type] is half a unit in the last place
relative to the value (2^-24, 2^-8, 2^-11), and an output is rounded once; SUM = 64 2^-24 stands for float32 sums as in the
other policy operators' tests; what else an operator rounds is derived beside its check."""
import math

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
    got, want, bound = got.double().cpu(), want.double().cpu(), bound.double().cpu()
    assert got.shape == want.shape, name
    assert torch.isfinite(got).all(), f"{name}: not finite"
    over = (got - want).abs() - bound
    assert (over <= 0).all(), f"{name}: {int((over > 0).sum())} values off, the worst {over.max().item():.3g} over its bound"


def starts(lengths):
    return torch.tensor([0] + list(lengths), dtype=torch.int64).cumsum(0).to(torch.int32).cuda()


# ---- recurrence -----------------------------------------------------------------------------------------------------

# What a gate's sigmoid is off by, relative to it: the exponential's argument is rounded, |gate| 2^-24 of the result (|gate| < 16
# here: 2^-20), the exponential, the sum, the reciprocal and the product by 2^-23, 2^-24, 2^-23 and 2^-24; twice that leaves room for
# the rounding of each step's product and sum.
GATE = 2.0 ** -19


def recur64(x, f, lengths, initial, dh=None, dlast=None):
    """The definition step by step in float64 on the CPU, with each output's bound: magnitudes (m: the same sums of absolute
    values) and errors (e) run along, each step's product off by GATE of its magnitude."""
    dtype, (n, c) = x.dtype, x.shape
    x, f = x.detach().double().cpu(), f.detach().double().cpu()
    keep, take = torch.sigmoid(f), torch.sigmoid(-f)
    r = {"h": torch.zeros(n, c), "last": torch.zeros(len(lengths), c)}
    if dh is not None:
        r.update(dx=torch.zeros(n, c), dgate=torch.zeros(n, c), dinitial=torch.zeros(len(lengths), c))
        dh, dlast = dh.double().cpu(), dlast.double().cpu()
    r = {k: [v.double(), v.double()] for k, v in r.items()}
    u, tiny = U[dtype], TINY[dtype]

    def put(name, at, value, error, rounding=u, least=tiny):
        r[name][0][at], r[name][1][at] = value, error + rounding * value.abs() + least
    t = 0
    for s, length in enumerate(lengths):
        h = torch.zeros(c, dtype=torch.float64) if initial is None else initial[s].detach().double().cpu()
        m, e, before = h.abs(), torch.zeros(c, dtype=torch.float64), []
        for i in range(t, t + length):
            before.append((h, m, e))
            h = keep[i] * h + take[i] * x[i]
            e = keep[i] * (e + GATE * m) + GATE * take[i] * x[i].abs()
            m = keep[i] * m + take[i] * x[i].abs()
            put("h", i, h, e)
        put("last", s, h, e, U[F32], TINY[F32])
        if dh is not None:
            g = dlast[s].clone()
            m, e = g.abs(), torch.zeros(c, dtype=torch.float64)
            for i in range(t + length - 1, t - 1, -1):
                g, m = g + dh[i], m + dh[i].abs()
                e = e + U[F32] * m
                h0, m0, e0 = before[i - t]
                put("dx", i, take[i] * g, take[i] * (e + GATE * m))
                d = keep[i] * take[i]
                put("dgate", i, g * (h0 - x[i]) * d, d * ((e + 3 * GATE * m) * (m0 + x[i].abs()) + m * e0))
                g, m, e = keep[i] * g, keep[i] * m, keep[i] * (e + GATE * m)
            put("dinitial", s, g, e, U[F32], TINY[F32])
        t += length
    return {k: tuple(v) for k, v in r.items()}


def check_recurrence(x, f, lengths, initial=None, a=None):
    a = starts(lengths) if a is None else a
    leaves = [t.detach().requires_grad_() for t in (x, f)] + ([initial.detach().requires_grad_()] if initial is not None else [])
    h, last = policy.recurrence(leaves[0], leaves[1], a, leaves[2] if initial is not None else None)
    dh, dlast = rand(x.shape, x.dtype, 91), rand((len(lengths), x.shape[1]), F32, 92)
    grads = torch.autograd.grad((h, last), leaves, (dh, dlast))
    with torch.no_grad():
        again = policy.recurrence(x, f, a, initial)
    assert torch.equal(h, again[0]) and torch.equal(last, again[1])
    want = recur64(x, f, lengths, initial, dh, dlast)
    got = dict(zip(("h", "last", "dx", "dgate", "dinitial"), (h, last, *grads)))
    for name, t in got.items():
        within(name, t.detach(), *want[name])
    return got


def gated(n, c, dtype, seed=1, mean=1.5):
    return rand((n, c), dtype, seed), (rand((n, c), F32, seed + 1, 2.0) + mean).to(dtype)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("channels", [1, 2, 3, 7, 63, 64, 65, 127, 128, 129, 130, 257])
def test_recurrence_channels(dtype, channels):
    print("recurrence", dtype, channels, flush=True)
    lengths = [1, 33, 0, 70, 200, 5]
    x, f = gated(sum(lengths), channels, dtype, channels)
    check_recurrence(x, f, lengths, rand((len(lengths), channels), F32, 3))
    check_recurrence(x, f, lengths)


@pytest.mark.parametrize("lengths", [[1], [0], [], [15], [16], [17], [127], [128], [129], [1, 127], [127, 1, 128], [128, 128], [16] * 20,
                                     [300], [1] * 300, [0, 5, 0, 0, 7, 0], [0] * 40, [1000], [200, 0, 1, 900, 31, 32, 33], [5000]])
def test_recurrence_lengths(lengths):
    """One token to many chunks, sequences that end and start on the edges of stretches and chunks, several in one stretch,
    and those without tokens."""
    print("recurrence lengths", lengths[:6], len(lengths), flush=True)
    for dtype, c, mean in ((F32, 70, 1.5), (BF16, 130, 4.0)):
        x, f = gated(sum(lengths), c, dtype, len(lengths), mean)
        check_recurrence(x, f, lengths, rand((len(lengths), c), F32, 3))


def test_recurrence_long_memory_over_many_chunks():
    """More chunks than runs of the kernel that carries states over them, and gates whose states last for thousands of
    steps."""
    print("recurrence many chunks", flush=True)
    for lengths in ([20000], [9000, 3, 12000]):
        x, f = gated(sum(lengths), 5, F32, 1, 9.0)
        check_recurrence(x, f, lengths, rand((len(lengths), 5), F32, 3))


@pytest.mark.parametrize("seqs", [511, 512, 513, 3000, 300000])
def test_recurrence_many_sequences(seqs):
    """More sequences than a workgroup reads offsets of at once, and than two such reads find; half of them without tokens.
    Sequences of one token: h = a initial + (1 - a) x."""
    print("recurrence many sequences", seqs, flush=True)
    g = torch.Generator().manual_seed(seqs)
    lengths = torch.randint(0, 2, (seqs,), generator=g)
    lengths[:200] = 0  # many that start at one token
    n, c = int(lengths.sum()), 3
    x, f = gated(n, c, F32, 1)
    initial = rand((seqs, c), F32, 3)
    leaves = [t.detach().requires_grad_() for t in (x, f, initial)]
    h, last = policy.recurrence(*leaves[:2], starts(lengths.tolist()), leaves[2])
    dh, dlast = rand((n, c), F32, 5), rand((seqs, c), F32, 6)
    dx, df, di = torch.autograd.grad((h, last), leaves, (dh, dlast))
    some = (lengths == 1).cuda()
    xd, fd, s0 = x.double(), f.double(), initial.double()[some]
    keep, take = torch.sigmoid(fd), torch.sigmoid(-fd)
    want = keep * s0 + take * xd
    size = keep * s0.abs() + take * xd.abs()
    within("h", h.detach(), want, 2 * GATE * size)
    assert torch.equal(last[some], h) and torch.equal(last[~some], initial[~some]) and torch.equal(di[~some], dlast[~some])
    g0 = dh.double() + dlast.double()[some]
    gs = dh.double().abs() + dlast.double()[some].abs()
    within("dx", dx, take * g0, 2 * GATE * take * gs)
    within("dinitial", di[some], keep * g0, 2 * GATE * keep * gs)
    within("dgate", df, g0 * (s0 - xd) * keep * take, 6 * GATE * keep * take * gs * (s0.abs() + xd.abs()))


def test_recurrence_strides():
    """Slices of one projection at odd offsets, rows of a wider buffer, one gate row for all tokens, cotangents in other
    strides, an initial state that needs no gradient."""
    lengths = [40, 0, 150]
    for dtype in (F32, BF16, F16):
        wide = rand((190, 131), dtype, 6)
        for off in (0, 1, 3, 8):
            check_recurrence(wide[:, off:off + 50], wide[:, off + 51:off + 101] + 0, lengths, rand((3, 50), F32, 4))
            check_recurrence(wide[:, off:off + 50], wide[:, off + 51:off + 101], lengths)
    x, row = rand((190, 33), BF16, 1), rand((33,), BF16, 2).requires_grad_()
    h, _ = policy.recurrence(x, row.expand(190, 33), starts(lengths))
    dh = rand((190, 33), BF16, 3)
    each = rand((33,), BF16, 2).expand(190, 33).contiguous().requires_grad_()
    h2, _ = policy.recurrence(x, each, starts(lengths))
    assert torch.equal(h, h2)
    one, = torch.autograd.grad(h, row, dh)
    many, = torch.autograd.grad(h2, each, dh)
    assert torch.equal(one, many.sum(0))
    xs = rand((190, 33), F32, 1).requires_grad_()
    turned = rand((33, 190), F32, 4).t()
    a, = torch.autograd.grad(policy.recurrence(xs, xs, starts(lengths))[0], xs, turned)
    b, = torch.autograd.grad(policy.recurrence(xs, xs, starts(lengths))[0], xs, turned.contiguous())
    assert torch.equal(a, b)


def test_recurrence_partial_gradients():
    """Any of the inputs with a gradient and any of the outputs with a cotangent alone."""
    lengths, c = [70, 0, 200], 20
    x, f = gated(270, c, F32, 1)
    initial = rand((3, c), F32, 3)
    dh, dlast = rand((270, c), F32, 4), rand((3, c), F32, 5)
    leaves = [t.detach().requires_grad_() for t in (x, f, initial)]
    h, last = policy.recurrence(leaves[0], leaves[1], starts(lengths), leaves[2])
    for outs, cots, d, l in (((h,), (dh,), dh, 0 * dlast), ((last,), (dlast,), 0 * dh, dlast)):
        got = torch.autograd.grad(outs, leaves, cots, retain_graph=True)
        want = recur64(x, f, lengths, initial, d, l)
        for name, t in zip(("dx", "dgate", "dinitial"), got):
            within(name, t, *want[name])
    full = torch.autograd.grad((h, last), leaves, (dh, dlast))
    for i in range(3):
        some = [t.detach().requires_grad_(i == j) for j, t in enumerate((x, f, initial))]
        out = policy.recurrence(some[0], some[1], starts(lengths), some[2])
        assert torch.equal(torch.autograd.grad(out, some[i], (dh, dlast))[0], full[i])


def test_recurrence_padding():
    """Tokens behind the last sequence give zeros and take none, whatever they hold; the last sequence's state is whole."""
    for lengths, more in (([40, 100], 1), ([40, 100], 300), ([], 20), ([0, 0], 150), ([128], 128), ([120], 8)):
        n, c = sum(lengths), 33
        x, f = gated(n + more, c, BF16, 1)
        x[n:], f[n:] = math.nan, math.inf
        initial = rand((len(lengths), c), F32, 3)
        leaves = [t.detach().requires_grad_() for t in (x, f, initial)]
        h, last = policy.recurrence(leaves[0], leaves[1], starts(lengths), leaves[2])
        dh, dlast = rand(x.shape, BF16, 4), rand(initial.shape, F32, 5)
        dh[n:] = math.nan
        dx, df, di = torch.autograd.grad((h, last), leaves, (dh, dlast))
        assert not h[n:].any() and not dx[n:].any() and not df[n:].any()
        want = recur64(x[:n], f[:n], lengths, initial, dh[:n], dlast)
        for name, t in (("h", h[:n]), ("last", last), ("dx", dx[:n]), ("dgate", df[:n]), ("dinitial", di)):
            within(name, t.detach(), *want[name])


def test_recurrence_keeps_sequences_and_channels_apart():
    """What is not finite stays in its channel, and in its sequence from its token on (gradients: up to it)."""
    lengths, c = [40, 300, 5, 150], 66
    x, f = gated(495, c, F32, 1)
    initial, dh = rand((4, c), F32, 3), rand((495, c), F32, 4)

    def run(x, f, initial, dh):
        leaves = [t.detach().clone().requires_grad_() for t in (x, f, initial)]
        h, last = policy.recurrence(leaves[0], leaves[1], starts(lengths), leaves[2])
        return [h.detach(), last.detach(), *torch.autograd.grad(h, leaves, dh)]
    clean = run(x, f, initial, dh)
    for bad in (math.nan, math.inf):
        x2, i2, d2 = x.clone(), initial.clone(), dh.clone()
        x2[200, 3], i2[1, 4], d2[200, 5] = bad, bad, bad
        got = run(x2, f, i2, d2)
        others = [i for i in range(c) if i not in (3, 4, 5)]
        for a, b in zip(clean, got):
            assert torch.equal(a[:, others], b[:, others])
        for i in (0, 2, 3):  # by token
            for t in (slice(0, 40), slice(340, 495)):
                assert torch.equal(clean[i][t], got[i][t]), i
        assert torch.equal(clean[0][:200], got[0][:200][:, :]) or not torch.isfinite(got[0][40:200, 4]).any()
        assert torch.equal(clean[0][40:200, 3], got[0][40:200, 3]) and not torch.isfinite(got[0][200:340, 3]).any()
        assert not torch.isfinite(got[1][1, [3, 4]]).any() and torch.equal(clean[1][[0, 2, 3]], got[1][[0, 2, 3]])
        assert torch.equal(clean[2][201:340, 5], got[2][201:340, 5]) and not torch.isfinite(got[2][40:201, 5]).any()
        assert torch.equal(clean[4][[0, 2, 3]], got[4][[0, 2, 3]])


def test_recurrence_gates_at_their_ends():
    """Gates that keep all or take all: exactly 1 and 0; and far ones, whose small side keeps its own places."""
    x = rand((300, 8), F32, 1)
    f = torch.full((300, 8), math.inf, device="cuda")
    h, last = policy.recurrence(x, f, starts([300]), rand((1, 8), F32, 2))
    assert torch.equal(last, rand((1, 8), F32, 2)) and torch.equal(h, last.expand(300, 8))
    h, last = policy.recurrence(x, -f, starts([300]), rand((1, 8), F32, 2))
    assert torch.equal(h, x) and torch.equal(last, x[-1:])
    for dtype in (F32, BF16, F16):
        for far in (30.0, 60.0, 85.0):
            one, zero = torch.ones((1, 8), dtype=dtype, device="cuda"), torch.zeros((1, 8), dtype=dtype, device="cuda")
            g = torch.full((1, 8), far, dtype=dtype, device="cuda")
            small = torch.sigmoid(-g.double())
            off = (1 if dtype == F32 else far / 4) * GATE  # 16 bits: the argument's rounding, |gate| 2^-24
            within("take", policy.recurrence(one, g, starts([1]))[1], small, off * small)
            within("keep", policy.recurrence(zero, -g, starts([1]), torch.ones((1, 8), device="cuda"))[1], small, off * small)


def test_recurrence_offsets_that_are_wrong_stay_in_bounds():
    x, f = gated(500, 40, BF16, 1)
    for bad in ([0, 2 ** 31 - 1, 3], [0, -5, -(2 ** 31)], [7, 300, 100, 500], [0, 600, 400, 200], [500, 500]):
        a = torch.tensor(bad, dtype=torch.int32, device="cuda")
        leaves = [t.detach().requires_grad_() for t in (x, f, rand((len(bad) - 1, 40), F32, 2))]
        out = policy.recurrence(leaves[0], leaves[1], a, leaves[2])
        torch.autograd.grad(out, leaves, (x, leaves[2].detach()))
    torch.cuda.synchronize()


def test_recurrence_gradient_is_the_slope():
    """The gradients against central differences of the definition in float64, along random directions."""
    lengths, c = [20, 150], 30
    x, f = gated(170, c, F32, 1)
    initial, dh, dlast = rand((2, c), F32, 3), rand((170, c), F32, 4), rand((2, c), F32, 5)
    leaves = [t.clone().requires_grad_() for t in (x, f, initial)]
    grads = torch.autograd.grad(policy.recurrence(leaves[0], leaves[1], starts(lengths), leaves[2]), leaves, (dh, dlast))
    dirs = [rand(t.shape, torch.float64, 6 + i) for i, t in enumerate((x, f, initial))]
    step = 1e-6

    def value(s):
        xs, fs, h0 = (t.double() + s * step * d for t, d in zip((x, f, initial), dirs))
        keep, total, t = torch.sigmoid(fs), 0.0, 0
        for i, n in enumerate(lengths):
            h = h0[i]
            for j in range(t, t + n):
                h = keep[j] * h + (1 - keep[j]) * xs[j]
                total = total + (h * dh[j].double()).sum()
            total, t = total + (h * dlast[i].double()).sum(), t + n
        return total
    slope = (value(1) - value(-1)) / (2 * step)
    got = sum((g.double() * d).sum() for g, d in zip(grads, dirs))
    size = sum((g.double() * d).abs().sum() for g, d in zip(grads, dirs))
    assert abs(slope - got) <= 1e-6 * size, (slope.item(), got.item())


def test_recurrence_past_32_bits():
    """Tokens 2^20 elements apart: offsets past 2^31 elements."""
    big = torch.zeros((2200, 2 ** 20), dtype=BF16, device="cuda")
    x, f = gated(2200, 130, BF16, 1)
    big[:, 1:131], big[:, 140:270] = x, f

    def run(x, f):
        leaves = [t.detach().requires_grad_() for t in (x, f)]
        h, last = policy.recurrence(*leaves, starts([1000, 1200]))
        return [h, last, *torch.autograd.grad((h, last), leaves, (gated(2200, 130, BF16, 5)[0], last.detach()))]
    assert all(torch.equal(a, b) for a, b in zip(run(x, f), run(big[:, 1:131], big[:, 140:270])))


def test_recurrence_of_more_than_32_bits():
    """Outputs of more than 2^31 elements: one token for all, sequences as long as a chunk, so that each repeats the first bit
    for bit."""
    n, c, seqs = 64, 1030, 33000
    x, f = gated(1, c, BF16, 1)
    leaves = [t.expand(n * seqs, c).detach().requires_grad_() for t in (x, f)]
    h, last = policy.recurrence(*leaves, starts([n] * seqs))
    dh = rand((1, c), BF16, 3).expand(n * seqs, c)
    dx, df = torch.autograd.grad(h, leaves, dh)
    want = recur64(x.expand(n, c), f.expand(n, c), [n], None, dh[:n], torch.zeros((1, c)))
    for name, t in (("h", h.detach()), ("dx", dx), ("dgate", df)):
        within(name, t[:n], *want[name])
        t = t.view(seqs, n, c)
        for i in range(0, seqs, 3000):
            assert (t[i:i + 3000] == t[:1]).all(), (name, i)
    assert (last == last[:1]).all()


def test_recurrence_refusals():
    x, f, a, s = rand((10, 6), BF16, 1), rand((10, 6), BF16, 2), starts([4, 6]), rand((2, 6), F32, 3)
    for args in ((x.double(), f.double(), a), (x, f.float(), a), (x, f[:9], a), (x.t(), f.t(), a), (x, f, a.long()), (x, f, a[None]),
                 (x, f, a[:0]), (x, f, a[::2]), (x, f, a.cpu()), (x.cpu(), f.cpu(), a.cpu()), (x, f, a, s.to(BF16)), (x, f, a, s[:1]),
                 (x, f, a, rand((6, 2), F32).t()), (x[0], f[0], a), (x[:, :0], f[:, :0], a), (x, f, a, s.cpu()), (x, None, a)):
        with pytest.raises(TypeError):
            policy.recurrence(*args)
    with pytest.raises(ValueError):
        policy.recurrence(x[:1, :1].expand(2 ** 28, 1000), x[:1, :1].expand(2 ** 28, 1000), a)


# ---- one token a world ----------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("worlds,channels", [(0, 5), (1, 1), (3, 3), (1, 256), (7, 4), (5, 9), (300, 99), (1000, 130), (20000, 64),
                                             (3, 100001)])
def test_recurrence_step(dtype, worlds, channels):
    print("recurrence step", dtype, worlds, channels, flush=True)
    x, f = gated(worlds, channels, dtype, 1)
    s = rand((worlds, channels), F32, 3)
    h, new = policy.recurrence_step(x, f, s)
    keep, take = torch.sigmoid(f.double()), torch.sigmoid(-f.double())
    want, size = keep * s.double() + take * x.double(), keep * s.double().abs() + take * x.double().abs()
    within("state", new, want, 2 * GATE * size)
    assert h.dtype == dtype and torch.equal(h, new.to(dtype))


def test_recurrence_step_is_the_recurrence():
    """Strided rows, and one token a sequence of the packed form, bit for bit."""
    for dtype in (F32, BF16, F16):
        wide, s = rand((50, 210), dtype, 1), rand((50, 104), F32, 2)[:, 3:102]
        x, f = wide[:, 1:100], wide[:, 105:204]
        h, new = policy.recurrence_step(x, f, s)
        h2, last = policy.recurrence(x, f, starts([1] * 50), s.contiguous())
        assert torch.equal(h, h2) and torch.equal(new, last)


def test_recurrence_step_refusals():
    x, f, s = rand((10, 6), BF16, 1), rand((10, 6), BF16, 2), rand((10, 6), F32, 3)
    for args in ((x, f, s.to(BF16)), (x, f.float(), s), (x, f, s[:9]), (x.cpu(), f.cpu(), s.cpu()), (x, f, s.cpu()), (x.t(), f.t(), s.t()),
                 (x.double(), f.double(), s), (x[0], f[0], s[0])):
        with pytest.raises(TypeError):
            policy.recurrence_step(*args)
    with pytest.raises(RuntimeError):
        policy.recurrence_step(x, f, s.requires_grad_())
    with torch.no_grad():
        policy.recurrence_step(x, f, s)


# ---- gated residual -------------------------------------------------------------------------------------------------

def residual64(x, u, w, w2, gate, scale, eps, dy, dz):
    """The definition and its gradients in float64, and each output's bound. Written out a step at a time: a value's error is
    its inputs' errors through the formula's derivatives, and SUM of its terms' magnitudes for each float32 sum or product; the
    norms' factors are off by SUM of themselves, since all their squares are positive; a gate by GATE."""
    type_, n = x.dtype, x.shape[-1]
    one = torch.ones(n, dtype=torch.float64, device=x.device)
    wt, w2t, st = (p.dtype if p is not None else F32 for p in (w, w2, scale))
    w, w2, s = (p.double() if p is not None else one for p in (w, w2, scale))
    x, u, dy, dz = (t.double() for t in (x, u, dy, dz))
    sg = torch.sigmoid(gate.double()) if gate is not None else torch.ones_like(x)
    shut = torch.sigmoid(-gate.double()) if gate is not None else torch.zeros_like(x)
    mean = lambda v: v.mean(-1, keepdim=True)  # noqa: E731
    r = 1 / (mean(u * u) + eps).sqrt()
    uh = u * r
    f = s * sg * uh * w
    y = x + f
    ey = 2 * SUM * f.abs() + SUM * y.abs()  # the branch's factors, SUM each, and the sum
    r2 = 1 / (mean(y * y) + eps).sqrt()
    er2 = r2 * (SUM + r2 * r2 * mean(y.abs() * ey))
    yh = y * r2
    eyh = ey * r2 + y.abs() * er2 + SUM * yh.abs()
    out = {"y": (y, ey), "z": (yh * w2, (eyh + SUM * yh.abs()) * w2.abs())}
    gz = dz * w2
    q = mean(gz * yh)
    eq = mean(gz.abs() * eyh) + SUM * mean(gz.abs() * yh.abs())
    e = dy + r2 * (gz - yh * q)
    ee = er2 * (gz - yh * q).abs() + r2 * (eyh * q.abs() + yh.abs() * eq) + SUM * (dy.abs() + r2 * (gz.abs() + yh.abs() * q.abs()))
    out["dx"] = (e, ee)
    es, ees = e * s, ee * s.abs()
    out["dgate"] = (es * uh * w * sg * shut, (ees + 2 * SUM * es.abs()) * (uh * w).abs() * sg * shut)
    c, ec = es * sg * w, (ees + 2 * SUM * es.abs()) * sg * w.abs()
    p = mean(c * uh)
    ep = mean(ec * uh.abs()) + 2 * SUM * mean((c * uh).abs())
    out["du"] = (r * (c - uh * p), r * (ec + uh.abs() * ep + 2 * SUM * (uh * p).abs() + 2 * SUM * (c - uh * p).abs()))
    rows = lambda v: v.reshape(-1, n).sum(0)  # noqa: E731
    m, em = rows(e * sg * uh), rows((ee + 3 * SUM * e.abs()) * sg * uh.abs())
    out["dweight"], out["dscale"] = (s * m, s.abs() * em), (w * m, w.abs() * em)
    out["dnext_weight"] = (rows(dz * yh), rows(dz.abs() * eyh + SUM * (dz * yh).abs()))
    types = {"dweight": wt, "dnext_weight": w2t, "dscale": st}
    return {k: (v, b + U[types.get(k, type_)] * v.abs() + TINY[types.get(k, type_)]) for k, (v, b) in out.items()}


def check_residual(x, u, w=None, w2=None, gate=None, scale=None, eps=1e-5, dy=None, dz=None):
    given = {"x": x, "u": u, "weight": w, "next_weight": w2, "gate": gate, "scale": scale}
    leaves = {k: t.detach().requires_grad_() for k, t in given.items() if t is not None}
    opt = lambda k: leaves.get(k)  # noqa: E731
    y, z = policy.gated_residual(leaves["x"], leaves["u"], opt("weight"), opt("next_weight"), gate=opt("gate"), scale=opt("scale"), eps=eps)
    dy = rand(x.shape, x.dtype, 71) if dy is None else dy
    dz = rand(x.shape, x.dtype, 72) if dz is None else dz
    grads = torch.autograd.grad((y, z), list(leaves.values()), (dy, dz))
    with torch.no_grad():
        again = policy.gated_residual(x, u, w, w2, gate=gate, scale=scale, eps=eps)
    assert torch.equal(y, again[0]) and torch.equal(z, again[1])
    want = residual64(x, u, w, w2, gate, scale, eps, dy, dz)
    got = {"y": y.detach(), "z": z.detach(), **{f"d{k}": g for k, g in zip(leaves, grads)}}
    for name, t in got.items():
        within(name, t, *want[name])
    return got


def residual_inputs(rows, width, dtype, ptype=F32):
    x, u, g = (rand((rows, width), dtype, i, 1.5) for i in (1, 2, 3))
    return x, u, *((rand((width,), F32, 4 + i, 0.3) + 1).to(ptype) for i in range(2)), g, (rand((width,), F32, 6, 0.2) + 0.4).to(ptype)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("width", [1, 2, 7, 8, 9, 31, 32, 33, 63, 64, 65, 99, 127, 129, 255, 257, 511, 512, 513, 1023, 1025, 2047,
                                   2049, 4095, 4097, 8191, 8193, 16385])
def test_residual_widths(dtype, width):
    """Every group size and both sides of each change between them, the wide rows' kernels among them."""
    print("residual", dtype, width, flush=True)
    check_residual(*residual_inputs(37 if width < 4096 else 5, width, dtype))


@pytest.mark.parametrize("rows,width", [(1, 99), (2, 512), (5000, 99), (9000, 16), (20000, 64), (2100, 256), (1100, 1000), (600, 2050)])
def test_residual_rows(rows, width):
    """From one row to more than the backward's workgroups take at once."""
    print("residual rows", rows, width, flush=True)
    for dtype in (F32, BF16):
        check_residual(*residual_inputs(rows, width, dtype))


@pytest.mark.parametrize("which", range(16))
def test_residual_without(which):
    """Any of the weights, the gate and the scale missing; parameters in half precision."""
    x, u, *rest = residual_inputs(65, 77, BF16, BF16 if which % 2 else F32)
    check_residual(x, u, *[t if which >> i & 1 else None for i, t in enumerate(rest)])


def test_residual_strides_and_alignments():
    for dtype in (F32, BF16, F16):
        x, u, w, w2, g, s = residual_inputs(50, 131, dtype)
        for off in (0, 1, 3, 8):
            check_residual(x[:, off:off + 99], u[:, 5:104], w[:99], w2[1:100], g[:, off + 2:off + 101], s[3:102],
                           dy=rand((50, 104), dtype, 7)[:, 5:], dz=rand((99, 50), dtype, 8).t())
    x, u, w, w2, g, s = residual_inputs(24, 40, F32)
    check_residual(*(t.view(2, 3, 4, 40) if t.dim() == 2 else t for t in (x, u, w, w2, g, s)))
    check_residual(x, u[:1].expand(24, 40), w, w2, g[:1].expand(24, 40), s)
    with pytest.raises(TypeError):
        policy.gated_residual(x.t(), u.t())


def test_residual_partial_gradients():
    """Either output's cotangent alone, and any one input's gradient alone."""
    x, u, w, w2, g, s = residual_inputs(300, 90, F32)
    dy, dz = rand(x.shape, F32, 8), rand(x.shape, F32, 9)
    names = ("x", "u", "weight", "next_weight", "gate", "scale")

    def run(which):
        t = [v.detach().requires_grad_(which in (None, i)) for i, v in enumerate((x, u, w, w2, g, s))]
        return t, policy.gated_residual(*t[:4], gate=t[4], scale=t[5])
    t, out = run(None)
    for i, cots in ((0, (dy, 0 * dz)), (1, (0 * dy, dz))):
        # next_weight has no part in y
        some = [v for j, v in enumerate(t) if i == 1 or j != 3]
        grads = torch.autograd.grad(out[i], some, cots[i], retain_graph=True)
        want = residual64(x, u, w, w2, g, s, 1e-5, *cots)
        for name, v in zip([n for j, n in enumerate(names) if i == 1 or j != 3], grads):
            within(f"d{name}", v, *want[f"d{name}"])
    full = torch.autograd.grad(out, t, (dy, dz))
    for i in range(6):
        t, out = run(i)
        assert torch.equal(torch.autograd.grad(out, t[i], (dy, dz))[0], full[i]), names[i]


def test_residual_empty_rows():
    t = [v.requires_grad_() for v in residual_inputs(0, 9, F32)]
    y, z = policy.gated_residual(*t[:4], gate=t[4], scale=t[5])
    grads = torch.autograd.grad((y, z), t, (torch.empty_like(y), torch.empty_like(z)))
    assert y.shape == z.shape == (0, 9) and not any(g.any() for g in grads) and [g.shape for g in grads] == [v.shape for v in t]


def test_residual_extremes():
    """Rows of zeros, large and small values, closed and open gates, and what is not finite in a row of its own."""
    x, u, w, w2, g, s = residual_inputs(16, 333, F32)
    y, z = policy.gated_residual(torch.zeros_like(x), torch.zeros_like(u), w, w2, gate=g, scale=s)
    assert not y.any() and not z.any()
    for scale in (1e-12, 1e12):
        check_residual(scale * x, u, w, w2, g, scale * s, eps=0.0)
        check_residual(x, scale * u, w, w2, g, s, eps=0.0)
    full, none = torch.full_like(g, math.inf), torch.full_like(g, -math.inf)
    assert all(torch.equal(a, b) for a, b in zip(policy.gated_residual(x, u, w, w2, gate=full, scale=s),
                                                 policy.gated_residual(x, u, w, w2, scale=s)))
    y, z = policy.gated_residual(x, u, w, w2, gate=none, scale=s)
    assert torch.equal(y, x)
    check_residual(x, u, w, w2, 40 * g, s)
    leaves = [t.detach().clone().requires_grad_() for t in (x, u, g)]
    clean = policy.gated_residual(leaves[0], leaves[1], w, w2, gate=leaves[2], scale=s)
    cg = torch.autograd.grad(clean, leaves, (x, u))
    with torch.no_grad():
        leaves[0][1, 3], leaves[1][3, 332], leaves[2][5, 0] = math.inf, math.nan, math.nan
    bad = policy.gated_residual(leaves[0], leaves[1], w, w2, gate=leaves[2], scale=s)
    bg = torch.autograd.grad(bad, leaves, (x, u))
    good = [i for i in range(16) if i not in (1, 3, 5)]
    assert all(torch.equal(a[good], b[good]) for a, b in zip((*clean, *cg), (*bad, *bg)))
    assert torch.isnan(bad[1][[3, 5]]).all() and not torch.isfinite(bad[0][1, 3])


def test_residual_gradient_is_the_slope():
    x, u, w, w2, g, s = residual_inputs(33, 50, F32)
    dy, dz = rand(x.shape, F32, 8), rand(x.shape, F32, 9)
    at = (x, u, w, w2, g, s)
    t = [v.clone().requires_grad_() for v in at]
    grads = torch.autograd.grad(policy.gated_residual(*t[:4], gate=t[4], scale=t[5]), t, (dy, dz))
    dirs = [rand(v.shape, torch.float64, 10 + i) for i, v in enumerate(at)]
    h = 1e-6

    def value(sign):
        x, u, w, w2, g, s = (v.double() + sign * h * d for v, d in zip(at, dirs))
        rms = lambda v: v / (v.square().mean(-1, keepdim=True) + 1e-5).sqrt()  # noqa: E731
        y = x + s * torch.sigmoid(g) * rms(u) * w
        return (y * dy.double()).sum() + (rms(y) * w2 * dz.double()).sum()
    slope = (value(1) - value(-1)) / (2 * h)
    got = sum((a.double() * d).sum() for a, d in zip(grads, dirs))
    size = sum((a.double() * d).abs().sum() for a, d in zip(grads, dirs))
    assert abs(slope - got) <= 1e-6 * size, (slope.item(), got.item())


def test_residual_refusals():
    x, u, w, w2, g, s = residual_inputs(10, 6, BF16)
    for args, kw in (((x, u.float()), {}), ((x, u[:9]), {}), ((x, u, w[:5]), {}), ((x, u, w, w2.to(BF16)), {}), ((x, u, w.half()), {}),
                     ((x, u), dict(gate=g.float())), ((x, u), dict(gate=g[:, :5])), ((x, u), dict(scale=s[None])),
                     ((x.cpu(), u.cpu()), {}), ((x, u.cpu()), {}), ((x, u, w.cpu()), {}), ((x.double(), u.double()), {}), ((x, None), {}),
                     ((x[0, 0], u[0, 0]), {}), ((x[:, :0], u[:, :0]), {}), ((x, u), dict(gate=g.t().contiguous().t()))):
        with pytest.raises(TypeError):
            policy.gated_residual(*args, **kw)
    for eps in (-1.0, math.nan, math.inf):
        with pytest.raises(ValueError):
            policy.gated_residual(x, u, eps=eps)


# ---- paged histories ------------------------------------------------------------------------------------------------

EXP = 2.0 ** -12  # what float32 scores (|s| < 20 here, sums of at most 128 products) put on a probability


def visible(n, window, sinks):
    keys = torch.arange(n, device="cuda")
    return keys if window is None else keys[(keys >= n - window) | (keys < sinks)]


def paged_tables(lengths, page, most, spare=3, seed=0):
    """Each world's pages, drawn from a pool that holds a few more; entries past a world's last page name no page."""
    need = [-(-n // page) for n in lengths]
    order = torch.randperm(sum(need) + spare, generator=torch.Generator().manual_seed(seed)).tolist()
    table = torch.full((len(lengths), most), -1, dtype=torch.int32)
    for w, k in enumerate(need):
        table[w, :k] = torch.tensor(order[:k], dtype=torch.int32)
        order = order[k:]
    return table.cuda(), sum(need) + spare


def paged64(q, k, v, table, lengths, page, window, sinks, scale):
    out, bound = torch.zeros(q.shape, dtype=torch.float64, device="cuda"), torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    G, u = q.shape[1] // k.shape[2], U[q.dtype]
    for w, n in enumerate(lengths):
        keys = visible(n, window, sinks)
        if not len(keys):
            continue
        at, off = table[w].long()[keys // page], keys % page
        for h in range(q.shape[1]):
            K, V = k[at, off, h // G].double(), v[at, off, h // G].double()
            p = torch.softmax(K @ q[w, h].double() * scale, 0)
            out[w, h] = p @ V
            bound[w, h] = u * out[w, h].abs() + (2 * EXP + SUM) * (p @ V.abs()) + TINY[q.dtype]
    return out, bound


def check_paged(lengths, page, heads, kv, dim, dtype, window=None, sinks=0, scale=None, most=None):
    most = max([-(-n // page) for n in lengths] + [1]) if most is None else most
    table, count = paged_tables(lengths, page, most)
    q, k, v = rand((len(lengths), heads, dim), dtype, 1), rand((count, page, kv, dim), dtype, 2), rand((count, page, kv, dim), dtype, 3)
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    got = policy.attention_paged(q, k, v, table, n, scale=scale, window=window, sinks=sinks)
    within("out", got, *paged64(q, k, v, table, lengths, page, window, sinks, 1 / math.sqrt(dim) if scale is None else scale))
    return q, k, v, table, n, got


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("heads,kv,dim", [(1, 1, 64), (8, 2, 64), (6, 2, 128), (5, 5, 40), (8, 1, 8), (3, 1, 72), (7, 1, 120), (24, 2, 64),
                                          (70, 1, 128)])
def test_paged_heads(dtype, heads, kv, dim):
    print("paged", dtype, heads, kv, dim, flush=True)
    for window, sinks in ((None, 0), (20, 3)):
        check_paged([1, 0, 33, 16, 200, 17], 16, heads, kv, dim, dtype, window, sinks)


@pytest.mark.parametrize("page", [1, 2, 8, 16, 64, 256])
@pytest.mark.parametrize("window,sinks", [(None, 0), (None, 5), (1, 0), (1, 1), (16, 0), (16, 16), (17, 4), (100, 200), (1000, 0)])
def test_paged_windows(page, window, sinks):
    """Windows and sinks that begin and end inside pages, meet, and reach past the history."""
    print("paged window", page, window, sinks, flush=True)
    check_paged([0, 1, 2, 15, 16, 17, 18, 31, 33, 47, 64, 100, 116, 117, 300], page, 4, 2, 64, BF16, window, sinks)


@pytest.mark.parametrize("worlds,length,window,sinks", [(1, 5000, None, 0), (1, 70000, None, 0), (3, 9000, 4000, 100), (1, 600, 300, 4),
                                                        (40, 700, None, 0), (2100, 40, None, 0), (2100, 90, 30, 2), (1100, 64, None, 0)])
def test_paged_many_and_long(worlds, length, window, sinks):
    """Few worlds with long histories, whose stretches are joined, and many worlds, a wave each."""
    print("paged many", worlds, length, flush=True)
    g = torch.Generator().manual_seed(worlds)
    lengths = torch.randint(0, length + 1, (worlds,), generator=g).tolist()
    lengths[0] = length
    check_paged(lengths, 16, 4, 2, 64, BF16, window, sinks)


def test_paged_is_the_dense_form():
    """Pages in order are a cache: the same tokens give the dense form's results, bit for bit where no window hides any."""
    lengths, page, most = [0, 1, 100, 512, 333], 32, 16
    q, cache = rand((5, 8, 64), BF16, 1), rand((2, 5, 512, 2, 64), BF16, 2)
    table = torch.arange(5 * most, dtype=torch.int32, device="cuda").view(5, most)
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    got = policy.attention_paged(q, cache[0].view(-1, page, 2, 64), cache[1].view(-1, page, 2, 64), table, n)
    assert torch.equal(got, policy.attention_step(q, cache[0], cache[1], n))


def test_paged_reads_only_what_is_in_sight():
    """Tokens past the length and outside the window hold NaN, their pages' entries any number; lengths outside the table are
    moved inside it."""
    page, lengths, window, sinks = 8, [100, 37, 64, 9, 0], 20, 5
    q, k, v, table, n, want = check_paged(lengths, page, 4, 2, 64, BF16, window, sinks, most=13)
    k2, v2, t2 = torch.full_like(k, math.nan), torch.full_like(v, math.nan), torch.full_like(table, -7)
    for w, length in enumerate(lengths):
        keys = visible(length, window, sinks)
        at, off = table[w].long()[keys // page], keys % page
        k2[at, off], v2[at, off] = k[at, off], v[at, off]
        t2[w, keys // page] = table[w, keys // page]
    t2[4] = 2 ** 31 - 1
    assert torch.equal(policy.attention_paged(q, k2, v2, t2, n, window=window, sinks=sinks), want)
    full = torch.arange(13, dtype=torch.int32, device="cuda").expand(5, 13)
    far = torch.tensor([2 ** 31 - 1, 104, -1, -(2 ** 31), 0], dtype=torch.int32, device="cuda")
    near = torch.tensor([104, 104, 0, 0, 0], dtype=torch.int32, device="cuda")
    a, b = (policy.attention_paged(q, k, v, full, x, window=window, sinks=sinks) for x in (far, near))
    assert torch.equal(a, b) and not a[2:].any()


def test_paged_pages_that_are_not_there():
    """A world that needs one gives NaN in all its heads, its neighbours are as they were."""
    for lengths in ([100, 37, 64], [3000, 2900, 2000]):  # whole, and in stretches
        q, k, v, table, n, want = check_paged(lengths, 16, 4, 2, 64, BF16)
        for bad in (-1, k.shape[0], 2 ** 31 - 1, -(2 ** 31)):
            t2 = table.clone()
            t2[1, 1] = bad
            got = policy.attention_paged(q, k, v, t2, n)
            assert torch.isnan(got[1]).all() and torch.equal(got[[0, 2]], want[[0, 2]])
    none = policy.attention_paged(q, k[:0], v[:0], table, n)
    assert torch.isnan(none).all()
    assert not policy.attention_paged(q, k, v, table[:, :0], n).any()  # no entries: no tokens


def test_paged_strides():
    """Pools that are halves of one, heads before tokens, tables and queries that are slices; worlds that share pages."""
    lengths = [40, 0, 77]
    q, k, v, table, n, want = check_paged(lengths, 16, 4, 2, 64, F16)
    both = torch.stack([k, v], 1)
    wide = torch.full((3, 40), -1, dtype=torch.int32, device="cuda")
    wide[:, 7:7 + table.shape[1]] = table
    qs = rand((3, 9, 70), F16, 9)
    qs[:, 3:7, 5:69] = q
    assert torch.equal(policy.attention_paged(qs[:, 3:7, 5:69], both[:, 0], both[:, 1], wide[:, 7:7 + table.shape[1]], n), want)
    kt, vt = (x.transpose(1, 2).contiguous().transpose(1, 2) for x in (k, v))
    assert torch.equal(policy.attention_paged(q, kt, vt, table, n), want)
    shared = policy.attention_paged(q, k, v, table[2:].expand(3, -1), n[2:].expand(3).contiguous())
    assert torch.equal(shared[2], want[2])


def test_paged_scores_that_are_not_finite():
    """Every score -inf: NaN, as the dense form; an infinite value reaches its own column."""
    q = torch.ones((1, 1, 8), dtype=BF16, device="cuda")
    k, v = torch.full((2, 16, 1, 8), -math.inf, dtype=BF16, device="cuda"), rand((2, 16, 1, 8), BF16, 2)
    table, n = torch.tensor([[1, 0]], dtype=torch.int32, device="cuda"), torch.tensor([20], dtype=torch.int32, device="cuda")
    assert torch.isnan(policy.attention_paged(q, k, v, table, n)).all()
    k[0, 3] = 1
    assert torch.equal(policy.attention_paged(q, k, v, table, n)[0, 0], v[0, 3, 0])
    v[0, 3, 0, 5] = math.inf
    assert torch.isinf(policy.attention_paged(q, k, v, table, n)[0, 0, 5])


def test_paged_past_32_bits():
    """Pages 2^20 elements apart: offsets past 2^31 elements."""
    big = torch.zeros((2200, 2 ** 20), dtype=BF16, device="cuda")
    q, k, v = rand((2, 4, 64), BF16, 1), rand((2200, 4, 2, 64), BF16, 2), rand((2200, 4, 2, 64), BF16, 3)
    kb, vb = (big[:, 512 * i:512 * i + 512].view(2200, 4, 2, 64) for i in (1, 2))
    table = torch.randperm(2200, generator=torch.Generator().manual_seed(1)).to(torch.int32).cuda().view(2, 1100)
    n, zero = torch.tensor([4400, 4001], dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    packed = [x[table.long()].flatten(1, 2) for x in (k, v)]
    new = [torch.cat([x[0, :4400], x[1, :4001]]) for x in packed]
    policy.cache_append_(kb, vb, *new, table, zero, starts([4400, 4001]))
    k2, v2 = torch.zeros_like(k), torch.zeros_like(v)
    policy.cache_append_(k2, v2, *new, table, zero, starts([4400, 4001]))
    assert torch.equal(kb, k2) and torch.equal(vb, v2) and k2.any()
    assert torch.equal(policy.attention_paged(q, kb, vb, table, n), policy.attention_paged(q, k, v, table, n))


def append_by_hand(kp, vp, k, v, table, lengths, counts):
    t, page = 0, kp.shape[1]
    for w, (n, c) in enumerate(zip(lengths, counts)):
        for i in range(c):
            at = n + i
            if 0 <= at < table.shape[1] * page and 0 <= int(table[w, at // page]) < len(kp):
                kp[int(table[w, at // page]), at % page], vp[int(table[w, at // page]), at % page] = k[t], v[t]
            t += 1


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("kv,dim,page", [(1, 8, 1), (2, 64, 16), (3, 40, 8), (5, 128, 32)])
def test_append(dtype, kv, dim, page):
    """One token a world, and packed ones: none, one and many a world, over pages' edges, without a place or a page."""
    print("append", dtype, kv, dim, page, flush=True)
    lengths, most = [0, 1, 15, 16, 31, 64, -3, 100, 2 ** 31 - 1], -(-110 // page)
    table = torch.randperm(most * 9 + 4, generator=torch.Generator().manual_seed(1))[:most * 9].view(9, most).to(torch.int32).cuda()
    table[3, 0:2], table[4, -1] = -1, most * 9 + 4
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    for counts in ([1] * 9, [0, 3, 40, 2, 0, 50, 7, 30, 4]):
        t = sum(counts)
        kp, vp = rand((most * 9 + 4, page, kv, dim), dtype, 2), rand((most * 9 + 4, page, kv, dim), dtype, 3)
        both = rand((t + 2, 2 * kv + 1, dim + 3), dtype, 4)
        k, v = both[:t, :kv, 1:dim + 1], both[:t, kv:2 * kv, 2:dim + 2]  # slices at odd offsets
        want = kp.clone(), vp.clone()
        append_by_hand(*want, k, v, table.cpu(), lengths, counts)
        policy.cache_append_(kp, vp, k, v, table, n, None if counts == [1] * 9 else starts(counts))
        assert torch.equal(kp, want[0]) and torch.equal(vp, want[1])


def test_append_of_nothing_and_of_much():
    kp, vp = rand((700, 16, 2, 64), BF16, 1), rand((700, 16, 2, 64), BF16, 2)
    keep = kp.clone()
    none = torch.zeros((0, 2, 64), dtype=BF16, device="cuda")
    table, zero = torch.arange(700, dtype=torch.int32, device="cuda")[None], torch.zeros(1, dtype=torch.int32, device="cuda")
    policy.cache_append_(kp, vp, none, none, table[:0], zero[:0])
    policy.cache_append_(kp, vp, none, none, table, zero, starts([0]))
    assert torch.equal(kp, keep)
    k, v = rand((11000, 2, 64), BF16, 3), rand((11000, 2, 64), BF16, 4)
    policy.cache_append_(kp, vp, k, v, table, zero + 9, starts([11000]))
    assert torch.equal(kp.flatten(0, 1)[9:11009], k) and torch.equal(vp.flatten(0, 1)[9:11009], v)
    assert torch.equal(kp.flatten(0, 1)[:9], keep.flatten(0, 1)[:9])
    bad = torch.tensor([5, -9, 2 ** 31 - 1], dtype=torch.int32, device="cuda")  # offsets that are wrong stay in bounds
    policy.cache_append_(kp, vp, k[:40], v[:40], table.expand(2, 700), zero.expand(2).contiguous(), bad)
    torch.cuda.synchronize()


def test_append_and_attend_step_by_step():
    """A control loop's calls: each step's token appended, lengths counted on, and what the query sees, with pages that leave
    the window given to the next tokens; against the packed form over the whole history with the same window."""
    worlds, steps, page, window, sinks = 3, 70, 4, 13, 2
    kv, heads, dim = 2, 4, 64
    k, v, q = (rand((steps, worlds, n, dim), BF16, n + i) for i, n in enumerate((kv, kv, heads)))
    # pages of the sinks, and five in turn: the window's 13 tokens touch at most five pages
    kp, vp = torch.full((worlds * 6, page, kv, dim), math.nan, dtype=BF16, device="cuda"), rand((worlds * 6, page, kv, dim), BF16, 9)
    vp[:] = math.nan
    table = torch.full((worlds, -(-steps // page)), -1, dtype=torch.int32, device="cuda")
    lengths = torch.zeros(worlds, dtype=torch.int32, device="cuda")
    kd, vd, qd = (x.double() for x in (k, v, q))
    for t in range(steps):
        if t % page == 0:
            for w in range(worlds):
                table[w, t // page] = w * 6 + (0 if t == 0 else 1 + t // page % 5)
        policy.cache_append_(kp, vp, k[t], v[t], table, lengths)
        lengths += 1
        got = policy.attention_paged(q[t], kp, vp, table, lengths, window=window, sinks=sinks)
        keys = visible(t + 1, window, sinks)
        for w in range(worlds):
            for h in range(heads):
                p = torch.softmax(kd[keys, w, h // 2] @ qd[t, w, h] / 8, 0)
                V = vd[keys, w, h // 2]
                within(f"step {t}", got[w, h], p @ V, U[BF16] * (p @ V).abs() + (2 * EXP + SUM) * (p @ V.abs()))


def test_paged_refusals():
    q, kp, vp = rand((3, 4, 64), BF16, 1), rand((9, 16, 2, 64), BF16, 2), rand((9, 16, 2, 64), BF16, 3)
    t, n = torch.zeros((3, 5), dtype=torch.int32, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")
    k, v = rand((3, 2, 64), BF16, 4), rand((3, 2, 64), BF16, 5)
    for args in ((q.float(), kp.float(), vp.float(), t, n), (q, kp.half(), vp.half(), t, n), (q, kp, vp[:8], t, n), (q, kp, vp, t.long(), n),
                 (q, kp, vp, t[:2], n), (q, kp, vp, t, n[:2]), (q, kp, vp, t, n.long()), (q[:2], kp, vp, t, n), (q[:, :3], kp, vp, t, n),
                 (q, kp[..., :32], vp[..., :32], t, n), (q, kp[0], vp[0], t, n), (q.cpu(), kp.cpu(), vp.cpu(), t.cpu(), n.cpu()),
                 (q, kp, vp, t.cpu(), n), (q, kp, vp, t.t().contiguous().t(), n), (q, kp, None, t, n), (q, kp, vp, t[0], n)):
        with pytest.raises(TypeError):
            policy.attention_paged(*args)
    for kw in (dict(window=0), dict(window=-1), dict(sinks=-1), dict(scale=0.0), dict(scale=math.nan)):
        with pytest.raises(ValueError):
            policy.attention_paged(q, kp, vp, t, n, **kw)
    with pytest.raises(TypeError):
        policy.attention_paged(q, kp, vp, t, n, window=1.5)
    with pytest.raises(ValueError):
        policy.attention_paged(q, kp[:, :12], vp[:, :12], t, n)
    with pytest.raises(ValueError):
        policy.attention_paged(q, kp, vp, torch.zeros((3, 2 ** 26), dtype=torch.int32, device="cuda"), n)
    with pytest.raises(RuntimeError):
        policy.attention_paged(q.clone().requires_grad_(), kp, vp, t, n)
    for args in ((kp, vp, k.half(), v.half(), t, n), (kp, vp, k[:, :1], v[:, :1], t, n), (kp, vp, k, v[:2], t, n), (kp, vp, k, v, t[:2], n),
                 (kp, vp, k[:2], v[:2], t, n), (kp, vp, k, v, t, n.long()), (kp, vp, k, v, t, n, n), (kp, vp, k, v, t, n, starts([1, 1, 1]).long()),
                 (kp[:1].expand(9, 16, 2, 64), vp, k, v, t, n), (kp, vp, k, v, t, n[0]), (kp, vp, k.cpu(), v.cpu(), t, n),
                 (kp, vp, k, rand((3, 64, 2), BF16).transpose(1, 2), t, n), (kp, None, k, v, t, n)):
        with pytest.raises(TypeError):
            policy.cache_append_(*args)
    with pytest.raises(ValueError):
        policy.cache_append_(kp[:, :12], vp[:, :12], k, v, t, n)
    with pytest.raises(RuntimeError):
        policy.cache_append_(kp, vp, k.clone().requires_grad_(), v, t, n)


def test_append_refuses_what_lies_over_the_pages():
    kp, vp = rand((9, 16, 2, 64), BF16, 2), rand((9, 16, 2, 64), BF16, 3)
    t, n = torch.zeros((3, 5), dtype=torch.int32, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")
    k, v = rand((3, 2, 64), BF16, 4), rand((3, 2, 64), BF16, 5)
    was = kp.clone(), vp.clone()
    for args in ((kp, kp, k, v), (kp, vp, kp[0, :3], v), (kp, vp, vp[0, :3], v), (kp, vp, k, kp[0, 5:8]), (kp, vp, k, vp[8, 13:])):
        with pytest.raises(ValueError):
            policy.cache_append_(*args, t, n)
    assert torch.equal(kp, was[0]) and torch.equal(vp, was[1])
    t = torch.arange(15, dtype=torch.int32, device="cuda").view(3, 5) % 9  # each world's first page is its own
    for both in (rand((9, 2, 16, 2, 64), BF16, 6).unbind(1), rand((2, 9, 16, 2, 64), BF16, 7).unbind(0)):
        policy.cache_append_(*both, k, v, t, n)
        assert torch.equal(both[0][t[:, 0].long(), 0], k) and torch.equal(both[1][t[:, 0].long(), 0], v)


def test_appending_marks_what_it_writes():
    """A graph that saved a pool which appending then overwrites notices."""
    w = rand((4, 16, 1, 8), BF16, 1).requires_grad_()
    kp, vp = rand((4, 16, 1, 8), BF16, 2), rand((4, 16, 1, 8), BF16, 3)
    y = (w * kp).float().sum()
    one = torch.ones((1, 1, 8), dtype=BF16, device="cuda")
    policy.cache_append_(kp, vp, one, one, torch.zeros((1, 1), dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda"))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


# ---- attention with a window ----------------------------------------------------------------------------------------

def window64(q, k, v, lq, lk, scale, window, sinks, dout):
    """The definition in float64, and the bounds of each output's error: {name: (value, bound)}. Probabilities and score
    gradients are rounded to the inputs' type (U) and come of float32 scores (EXP), as attention's without a window. Narrow windows
    (64 keys with the sinks) take delta = dout . out from the output and what its rounding took off, others from the rounded
    output, but for rows whose keys all lie in a sequence's first 64."""
    u, tiny = U[q.dtype], TINY[q.dtype]
    q, k, v, dout = (x.double() for x in (q, k, v, dout))
    G = q.shape[1] // k.shape[1]
    r = {n: (torch.zeros_like(x), torch.zeros_like(x)) for n, x in (("out", q), ("dq", q), ("dk", k), ("dv", v))}
    aq = ak = 0
    for nq, nk in zip(lq, lk):
        sq, sk = slice(aq, aq + nq), slice(ak, ak + nk)
        aq, ak = aq + nq, ak + nk
        place, key = torch.arange(nq, device=q.device)[:, None] + nk - nq, torch.arange(nk, device=q.device)
        mask = (key <= place) & ((key > place - window) | (key < sinks))
        for h in range(q.shape[1]):
            Q, K, V, d = q[sq, h], k[sk, h // G], v[sk, h // G], dout[sq, h]
            some = mask.any(1, keepdim=True)
            s = (Q @ K.t() * scale).masked_fill(~mask, -math.inf)
            p = torch.where(some, torch.softmax(torch.where(some, s, 0.0), 1), 0.0) * mask
            o = p @ V
            ob = (u + 2 * EXP) * (p @ V.abs())
            r["out"][0][sq, h], r["out"][1][sq, h] = o, u * o.abs() + ob + tiny
            r["dv"][0][sk, h // G] += p.t() @ d
            r["dv"][1][sk, h // G] += (u + 2 * EXP) * (p.t() @ d.abs())
            ds = p * (d @ V.t() - (d * o).sum(1, keepdim=True))
            left = u * u if window + sinks <= 64 else u  # of the output, after what was kept of its rounding
            doff = (d.abs() * (left * o.abs() + ob)).sum(1, keepdim=True) + 2 * SUM * (d.abs() @ V.abs().t())
            dsb = (u + 2 * EXP) * ds.abs() + p * doff
            r["dq"][0][sq, h], r["dq"][1][sq, h] = ds @ K * scale, dsb @ K.abs() * scale
            r["dk"][0][sk, h // G] += ds.t() @ Q * scale
            r["dk"][1][sk, h // G] += dsb.t() @ Q.abs() * scale
    return {n: (x, b + u * x.abs() + tiny if n != "out" else b) for n, (x, b) in r.items()}


def run_window(q, k, v, lq, lk, window, sinks, dout, scale=None):
    leaves = [x.detach().requires_grad_() for x in (q, k, v)]
    out = policy.attention(*leaves, starts(lq), starts(lk), scale=scale, window=window, sinks=sinks)
    return dict(zip(("out", "dq", "dk", "dv"), (out.detach(), *torch.autograd.grad(out, leaves, dout))))


def check_window(q, k, v, lq, lk, window, sinks=0, scale=None):
    dout = rand(q.shape, q.dtype, 99)
    got = run_window(q, k, v, lq, lk, window, sinks, dout, scale)
    with torch.no_grad():
        assert torch.equal(got["out"], policy.attention(q, k, v, starts(lq), starts(lk), scale=scale, window=window, sinks=sinks))
    want = window64(q, k, v, lq, lk, 1 / math.sqrt(q.shape[2]) if scale is None else scale, window, sinks, dout)
    for name, t in got.items():
        within(name, t, *want[name])
    return got


def heads_of(lq, lk, heads, kv, dim, dtype=BF16):
    return rand((sum(lq), heads, dim), dtype, 1), rand((sum(lk), kv, dim), dtype, 2), rand((sum(lk), kv, dim), dtype, 3)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("heads,kv,dim", [(1, 1, 64), (4, 2, 64), (6, 2, 128), (5, 5, 40), (8, 1, 8), (3, 1, 72), (70, 1, 64), (130, 1, 128)])
def test_window_heads(dtype, heads, kv, dim):
    print("window", dtype, heads, kv, dim, flush=True)
    lq = [1, 33, 70, 0, 300, 5]
    for window, sinks in ((20, 3), (100, 0)):
        check_window(*heads_of(lq, lq, heads, kv, dim, dtype), lq, lq, window, sinks)


@pytest.mark.parametrize("window", [1, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129, 200, 500, 699, 700, 5000])
@pytest.mark.parametrize("sinks", [0, 1, 4, 32, 64, 65, 130, 1000])
def test_windows(window, sinks):
    """Windows and sinks that end inside tiles and on their edges, meet, leave hidden tiles between them or none, and reach
    past a sequence; long sequences, one with earlier keys, and many short ones (a wave alone takes their keys' gradients)."""
    print("window", window, sinks, flush=True)
    lq, lk = [700, 3, 260], [700, 3, 500]
    check_window(*heads_of(lq, lk, 4, 2, 64), lq, lk, window, sinks)
    short, past = [40, 0, 17, 90, 1] * 8, [60, 3, 17, 90, 100] * 8
    check_window(*heads_of(short, past, 4, 2, 64, F16), short, past, window, sinks)


@pytest.mark.parametrize("lq,lk", [([1], [1]), ([1], [300]), ([0], [5]), ([5], [0]), ([300], [1]), ([70, 3], [20, 200]), ([64], [65]),
                                   ([129, 1], [127, 640]), ([1] * 90, [7] * 90), ([2, 0, 0, 4], [0, 9, 0, 4]), ([513], [520])])
def test_window_lengths(lq, lk):
    print("window lengths", lq[:4], lk[:4], flush=True)
    for dim, heads in ((64, 2), (128, 6)):
        for window, sinks in ((5, 2), (40, 0), (1, 0)):
            check_window(*heads_of(lq, lk, heads, 2, dim), lq, lk, window, sinks)


@pytest.mark.parametrize("dtype,dim,heads", [(BF16, 64, 2), (F16, 128, 6), (BF16, 40, 8)])
@pytest.mark.parametrize("lq,lk", [([1], [4000]), ([5, 60], [1800, 2100]), ([1500], [1500]), ([1300, 700], [257, 1900]), ([129], [5000]),
                                   ([4000], [4000])])
def test_window_few_sequences(dtype, dim, heads, lq, lk):
    """Few tiles, long sequences: a tile's keys (rows) are split among workgroups."""
    print("window few", dtype, dim, heads, lq, lk, flush=True)
    for window, sinks in ((1200, 70), (100, 4)):
        check_window(*heads_of(lq, lk, heads, 2, dim, dtype), lq, lk, window, sinks)


@pytest.mark.parametrize("dim", [64, 128])
def test_window_long_sequences(dim):
    """Sequences long enough that their tiles are listed one by one, and enough of them that none is split."""
    print("window long", dim, flush=True)
    lq, lk = [2500, 1900], [2500, 2100]
    check_window(*heads_of(lq, lk, 16, 8, dim), lq, lk, 300, 20)


def test_window_as_long_as_the_keys_hides_nothing():
    lq, lk = [300, 7, 512], [310, 7, 600]
    q, k, v = heads_of(lq, lk, 4, 2, 64)
    dout = rand(q.shape, BF16, 9)
    leaves = [x.detach().requires_grad_() for x in (q, k, v)]
    out = policy.attention(*leaves, starts(lq), starts(lk))
    want = (out, *torch.autograd.grad(out, leaves, dout))
    for window, sinks in ((sum(lk), 0), (2 ** 40, 2 ** 40), (None, 5)):
        got = run_window(q, k, v, lq, lk, window, sinks, dout)
        assert all(torch.equal(a, b) for a, b in zip(want, got.values()))


def test_windows_and_sinks_past_64_bits():
    lq = [300, 7, 512]
    q, k, v = heads_of(lq, lq, 4, 2, 64)
    dout = rand(q.shape, BF16, 9)
    for big, plain in (((2 ** 63 - 1, 4), (None, 0)), ((2 ** 70, 2 ** 70), (None, 0)), ((100, 2 ** 70), (100, sum(lq)))):
        want, got = (run_window(q, k, v, lq, lq, *s, dout) for s in (plain, big))
        assert all(torch.equal(want[name], got[name]) for name in want)


def test_window_rounds_as_finely_as_few_keys_need():
    """A window of one key: the output is the value and the scores have no part, so their gradients are exactly 0."""
    lq = [300, 40]
    for dtype in (BF16, F16):
        q, k, v = heads_of(lq, lq, 4, 2, 64, dtype)
        dout = rand(q.shape, dtype, 9)
        got = run_window(q, k, v, lq, lq, 1, 0, dout)
        assert torch.equal(got["out"], v.repeat_interleave(2, 1))
        # P = 1, dP and delta the same sum in two orders
        bound = (dout.double().abs() * got["out"].double().abs()).sum(2, keepdim=True) * (2 * SUM + U[dtype] ** 2)
        within("dq", got["dq"], torch.zeros_like(got["dq"]), bound * k.repeat_interleave(2, 1).double().abs())


def test_window_padding():
    lq, lk, more = [40, 0, 130], [60, 10, 130], 70
    q, k, v = heads_of(lq + [more], lk + [more], 4, 2, 64)
    q[sum(lq):], k[sum(lk):], v[sum(lk):] = math.nan, math.inf, math.nan
    dout = rand(q.shape, BF16, 99)
    dout[sum(lq):] = math.nan
    leaves = [x.detach().requires_grad_() for x in (q, k, v)]
    out = policy.attention(*leaves, starts(lq), starts(lk), window=30, sinks=2)
    grads = torch.autograd.grad(out, leaves, dout)
    nq, nk = sum(lq), sum(lk)
    want = window64(q[:nq], k[:nk], v[:nk], lq, lk, 0.125, 30, 2, dout[:nq])
    for name, t, n in (("out", out.detach(), nq), ("dq", grads[0], nq), ("dk", grads[1], nk), ("dv", grads[2], nk)):
        within(name, t[:n], *want[name])
        assert not t[n:].any(), name


@pytest.mark.parametrize("dtype,dim,heads,n", [(BF16, 64, 2, 400), (F16, 64, 6, 400), (BF16, 128, 4, 400), (F16, 40, 2, 90), (BF16, 64, 2, 2500)])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_window_what_it_hides(dtype, dim, heads, n, bad):
    """A key, value, query or cotangent that is not finite reaches the rows and keys that see it, and no others: not those
    behind the window, nor, for a row, the keys before it; a bad sink reaches every later row."""
    print("window hidden", dtype, dim, heads, n, bad, flush=True)
    lq, lk, window, sinks, at = [n, 30], [n, 30], 40, 3, 41
    q, k, v = heads_of(lq, lk, heads, 2, dim, dtype)
    dout = rand(q.shape, dtype, 99)
    want = window64(q, k, v, lq, lk, 1 / math.sqrt(dim), window, sinks, dout)

    def same(got, name, rows, cols=slice(None)):
        w, b = want[name]
        within(f"{name} {rows}", got[name][rows, :, cols], w[rows, :, cols], b[rows, :, cols])
    unseen = [i for i in range(n + 30) if not at <= i < at + window]
    v2 = v.clone()
    v2[at, :, 7] = bad
    got = run_window(q, k, v2, lq, lk, window, sinks, dout)
    for name in ("out", "dq"):
        same(got, name, unseen)
    seen7 = got["out"][at:at + window, :, 7]
    assert torch.isnan(seen7).all() if math.isnan(bad) else (seen7 == bad).all()
    same(got, "dv", slice(None))
    same(got, "dk", [i for i in range(n + 30) if i >= at + window + window or i >= n])
    k2 = k.clone()
    k2[at] = bad
    got = run_window(q, k2, v, lq, lk, window, sinks, dout)
    for name in ("out", "dq"):
        same(got, name, unseen)
    for name in ("dk", "dv"):
        same(got, name, [i for i in range(n + 30) if i >= at + window or i >= n])
    row = 60  # sees keys 21 .. 60 and the sinks
    others = [i for i in range(n + 30) if not (row - window < i <= row or i < sinks)]
    for which in ("q", "dout"):
        q2, d2 = q.clone(), dout.clone()
        (q2 if which == "q" else d2)[row] = bad
        got = run_window(q2, k, v, lq, lk, window, sinks, d2)
        for name in ("out", "dq"):
            same(got, name, [i for i in range(n + 30) if i != row])
        for name in ("dk", "dv"):
            same(got, name, others)
    v3 = v.clone()
    v3[1, :, 5] = bad
    got = run_window(q, k, v3, lq, lk, window, sinks, dout)
    same(got, "out", [0]), same(got, "out", slice(n, None)), same(got, "out", slice(1, n), slice(0, 5))
    assert not torch.isfinite(got["out"][1:n, :, 5]).any()


def test_window_scores_that_are_all_minus_infinity():
    """Rows whose every key in sight has a score of -inf give NaN, rows that see another one its value."""
    q = torch.ones((300, 1, 64), dtype=BF16, device="cuda")
    k, v = torch.full((300, 1, 64), -math.inf, dtype=BF16, device="cuda"), rand((300, 1, 64), BF16, 2)
    k[100] = 1
    out = policy.attention(q, k, v, starts([300]), window=20, sinks=2)
    assert torch.isnan(out[:100]).all() and torch.isnan(out[120:]).all()
    assert torch.equal(out[100:120], v[100:101].expand(20, 1, 64))
    k[1] = 1  # a sink
    out = policy.attention(q, k, v, starts([300]), window=20, sinks=2)
    assert torch.isnan(out[0]).all() and torch.equal(out[120:], v[1:2].expand(180, 1, 64))


def test_window_offsets_that_are_wrong_stay_in_bounds():
    q, k, v = heads_of([500], [500], 4, 2, 64)
    for bad in ([0, 2 ** 31 - 1, 3], [0, -5, -(2 ** 31)], [7, 300, 100, 500], [0, 600, 400, 200]):
        a = torch.tensor(bad, dtype=torch.int32, device="cuda")
        leaves = [x.detach().requires_grad_() for x in (q, k, v)]
        torch.autograd.grad(policy.attention(*leaves, a, window=50, sinks=5), leaves, q)
    torch.cuda.synchronize()


def test_window_gradient_is_the_slope():
    lq, lk, window, sinks = [20, 95], [33, 95], 30, 3
    q, k, v = heads_of(lq, lk, 4, 2, 64, F16)
    dout = rand(q.shape, F16, 4)
    got = run_window(q, k, v, lq, lk, window, sinks, dout)
    want = window64(q, k, v, lq, lk, 0.125, window, sinks, dout)
    for i, name in enumerate(("dq", "dk", "dv")):
        xs = [x.double() for x in (q, k, v)]
        d = rand(xs[i].shape, torch.float64, 7)

        def value(s):
            ys = list(xs)
            ys[i] = ys[i] + s * d
            total, aq, ak = 0.0, 0, 0
            for nq, nk in zip(lq, lk):
                place, key = torch.arange(nq, device="cuda")[:, None] + nk - nq, torch.arange(nk, device="cuda")
                mask = (key <= place) & ((key > place - window) | (key < sinks))
                for h in range(4):
                    p = torch.softmax((ys[0][aq:aq + nq, h] @ ys[1][ak:ak + nk, h // 2].t() * 0.125).masked_fill(~mask, -math.inf), 1)
                    total = total + ((p @ ys[2][ak:ak + nk, h // 2]) * dout[aq:aq + nq, h].double()).sum()
                aq, ak = aq + nq, ak + nk
            return total
        slope = (value(1e-5) - value(-1e-5)) / 2e-5
        along = (got[name].double() * d).sum()
        assert abs(slope - along) <= (want[name][1] * d.abs()).sum() + 1e-6 * abs(slope), name


def test_window_past_32_bits():
    """Tokens 2^20 elements apart: offsets past 2^31 elements."""
    big = torch.zeros((2200, 2 ** 20), dtype=BF16, device="cuda")
    q, k, v = (rand((2200, 1, 64), BF16, n) for n in (1, 2, 3))
    views = []
    for i, x in enumerate((q, k, v)):
        view = big[:, 64 * i:64 * i + 64].unflatten(1, (1, 64))
        view.copy_(x)
        views.append(view)
    run = lambda *xs: run_window(*xs, [1000, 1200], [1000, 1200], 200, 4, q).values()  # noqa: E731
    assert all(torch.equal(a, b) for a, b in zip(run(q, k, v), run(*views)))


def test_window_is_what_the_paged_form_sees():
    """The last query of each sequence against the control loop's form over the same history in pages."""
    lengths, window, sinks = [1, 17, 40, 300], 16, 3
    q, k, v = heads_of([1] * 4, lengths, 4, 2, 64)
    a = policy.attention(q, k, v, starts([1] * 4), starts(lengths), window=window, sinks=sinks)
    table, count = paged_tables(lengths, 8, 40)
    kp, vp = (torch.zeros((count, 8, 2, 64), dtype=BF16, device="cuda") for _ in range(2))
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    policy.cache_append_(kp, vp, k, v, table, torch.zeros_like(n), starts(lengths))
    b = policy.attention_paged(q, kp, vp, table, n, window=window, sinks=sinks)
    within("paged", b, a, 2 * U[BF16] * a.double().abs() + (U[BF16] + 4 * EXP + 2 * SUM) * v.double().abs().amax())


def test_window_refusals():
    q, k, v = heads_of([10], [10], 4, 2, 64)
    for kw in (dict(window=0), dict(window=-3), dict(window=5, sinks=-1), dict(sinks=-1)):
        with pytest.raises(ValueError):
            policy.attention(q, k, v, starts([10]), **kw)
    for kw in (dict(window=2.5), dict(window="3"), dict(window=3, sinks=1.0)):
        with pytest.raises(TypeError):
            policy.attention(q, k, v, starts([10]), **kw)
    with pytest.raises(TypeError):
        policy.attention(q.float(), k.float(), v.float(), starts([10]), window=3)


# ---- streams, graphs, compilation, runs together --------------------------------------------------------------------

def all_operators():
    lq = [70, 3, 190]
    x, f = gated(263, 40, F32, 1)
    s0, dh, dl = rand((3, 40), F32, 3), rand((263, 40), F32, 4), rand((3, 40), F32, 5)
    r = residual_inputs(300, 99, F32)
    dy, dz = rand((300, 99), F32, 8), rand((300, 99), F32, 9)
    q, k, v = heads_of(lq, lq, 4, 2, 64)
    dout, a = rand(q.shape, BF16, 6), starts(lq)
    table, count = paged_tables([0, 1, 600, 33, 599, 2], 16, 40)
    n = torch.tensor([0, 1, 600, 33, 599, 2], dtype=torch.int32, device="cuda")
    kp, vp, qs = rand((count, 16, 2, 64), BF16, 11), rand((count, 16, 2, 64), BF16, 12), rand((6, 4, 64), BF16, 13)
    new = rand((6, 4, 64), BF16, 14)

    def run():
        leaves = [t.detach().requires_grad_() for t in (x, f, s0)]
        out = policy.recurrence(leaves[0], leaves[1], a, leaves[2])
        res = [*out, *torch.autograd.grad(out, leaves, (dh, dl)), *policy.recurrence_step(x, f, dh)]
        leaves = [t.detach().requires_grad_() for t in r]
        out = policy.gated_residual(*leaves[:4], gate=leaves[4], scale=leaves[5])
        res += [*out, *torch.autograd.grad(out, leaves, (dy, dz))]
        for window, sinks in ((20, 3), (100, 0)):
            leaves = [t.detach().requires_grad_() for t in (q, k, v)]
            o = policy.attention(*leaves, a, window=window, sinks=sinks)
            res += [o, *torch.autograd.grad(o, leaves, dout)]
        policy.cache_append_(kp, vp, new[:, :2], new[:, 2:], table, n - 1)
        res += [kp.clone(), vp.clone()] + [policy.attention_paged(qs, kp, vp, table, n, window=w, sinks=3) for w in (None, 50)]
        return [t.detach() for t in res]
    return run, (x, f, s0, dh, dl, *r, dy, dz, q, k, v, dout, kp, vp, qs, new)


def test_operators_are_the_same_every_time():
    run, _ = all_operators()
    assert all(torch.equal(a, b) for a, b in zip(run(), run()))


def test_operators_on_another_stream():
    run, _ = all_operators()
    want = run()
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = run()
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_operators_on_two_streams_at_once():
    run, _ = all_operators()
    want = run()
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for _ in range(3):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(run())
    torch.cuda.synchronize()
    for one in got:  # (the appended tokens are the same ones)
        assert all(torch.equal(a, b) for a, b in zip(want, one))


def test_operators_in_graphs():
    """Two captured graphs of the same calls, replayed in turn over new inputs with eager work between."""
    run, inputs = all_operators()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        run()
    torch.cuda.current_stream().wait_stream(s)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            held = run()
        graphs.append((g, held))
    for turn in range(4):
        for i, t in enumerate(inputs):
            t.copy_(rand(t.shape, t.dtype, 100 * turn + i))
        want = [t.clone() for t in run()]
        torch.cuda.synchronize()
        for g, held in graphs:
            g.replay()
            torch.cuda.synchronize()
            for i, (a, b) in enumerate(zip(want, held)):
                assert torch.equal(a, b), (turn, i)


def test_operators_compiled_over_sizes():
    """torch.compile keeps each operator as one node of a full graph, forward and backward, over several batches: eager's
    results for each."""
    w = rand((64,), F32, 2)

    def loss(x, f, heads, a, s0):
        h, last = policy.recurrence(torch.sin(x), f, a, s0)
        y, z = policy.gated_residual(x, h, w, None, gate=f, scale=w)
        o = policy.attention(heads[:, :2], heads[:, 2:4], heads[:, 4:], a, window=20, sinks=2)
        return (y * z).sum() + last.sum() + (o.float() * 3).sum()

    def run(fn, lq):
        n = sum(lq)
        leaves = [t.detach().requires_grad_() for t in (*gated(n, 64, F32, 1), rand((n, 6, 64), BF16, 4))]
        s0 = rand((len(lq), 64), F32, 5).requires_grad_()
        value = fn(*leaves, starts(lq), s0)
        return [value.detach(), *torch.autograd.grad(value, [*leaves, s0])]
    torch._dynamo.reset()
    compiled = torch.compile(loss, fullgraph=True, backend="aot_eager")
    for lq in ([20, 0, 44, 11], [7, 300], [1], [500, 900, 2, 2, 2], [33] * 40):
        for i, (e, c) in enumerate(zip(run(loss, lq), run(compiled, lq))):
            assert torch.equal(e, c), (lq[:4], i)


def test_appending_compiled():
    """The pages are written under torch.compile as they are without, and read after."""
    def step(kp, vp, k, q, table, n):
        policy.cache_append_(kp, vp, k, k * 2, table, n)
        return policy.attention_paged(q, kp, vp, table, n + 1, window=9) * 2
    table, count = paged_tables([20, 5, 40], 8, 6)
    n = torch.tensor([19, 4, 39], dtype=torch.int32, device="cuda")
    k, q = rand((3, 2, 64), BF16, 1), rand((3, 4, 64), BF16, 2)
    pools = [[rand((count, 8, 2, 64), BF16, i) for i in (3, 4)] for _ in range(2)]
    compiled = torch.compile(step, fullgraph=True, backend="aot_eager")
    assert torch.equal(step(*pools[0], k, q, table, n), compiled(*pools[1], k, q, table, n))
    assert all(torch.equal(a, b) for a, b in zip(*pools))


def test_gradients_in_a_graph_of_gradients():
    """Under create_graph the gradients are those without it, and differentiating them again raises."""
    lq = [20, 70]
    a, r = starts(lq), residual_inputs(40, 99, F32)
    q, k, v = heads_of(lq, lq, 4, 2, 64)
    x, f = gated(90, 30, F32, 1)
    for call, at in ((lambda x, f: policy.recurrence(x, f, a)[0], (x, f)),
                     (lambda x, u, w, w2, g, s: policy.gated_residual(x, u, w, w2, gate=g, scale=s)[1], r),
                     (lambda *t: policy.attention(*t, a, window=9, sinks=2), (q, k, v))):
        leaves = [t.detach().requires_grad_() for t in at]
        cot = rand(at[0].shape, at[0].dtype, 9)
        want = torch.autograd.grad(call(*leaves), leaves, cot)
        got = torch.autograd.grad(call(*leaves), leaves, cot, create_graph=True)
        assert all(torch.equal(p, r) and r.requires_grad and not p.requires_grad for p, r in zip(want, got))
        with pytest.raises(RuntimeError, match="differentiated again"):
            sum(g.float().square().sum() for g in got).backward()
