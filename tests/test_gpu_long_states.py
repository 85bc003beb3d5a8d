"""The recurrence where its states last long: what each step's roundings are off by must not add up over the tokens. Float32 on a
GPU against closed forms in float64.

U = 2^-24 is half a unit in the last place. A state reaches a token through at most MAPS stretches' maps, each applied with two
roundings (U each, relative to a state that does not cancel): of n tokens' chunks of 64, the runs of the chain over them that are
joined by doubling (7) and the chunks of its own run, its chunk's stretches (8 at most) and its stretch's tokens (16 at most). A
map's own sums over its tokens (64 at most) are off by U a token relative to what they add, and so are their contributions in sum.
A gate's small side is off by SMALL: the exponential by 2^-23, the reciprocal by 2^-23, the sum before it, the product behind and the
correction of the exponential's argument by 2^-24 each, rounded up to a power of two."""
import math

import pytest
import torch

from nablaengine_amd import policy

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
SMALL = 8 * U


@pytest.fixture(autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.fail("no GPU visible")


def roundings(n):
    chunks = -(-n // 64)
    return 2 * (7 + -(-chunks // 128) + 8 + 16) + 2 * 64


def one_sequence(n):
    return torch.tensor([0, n], dtype=torch.int32, device="cuda")


def full(n, c, value):
    return torch.full((n, c), value, dtype=torch.float32, device="cuda")


@pytest.mark.parametrize("n", [100, 5000, 65536])
@pytest.mark.parametrize("gate", [8.0, 9.3, 12.0, 15.0, 17.0, 20.0])
def test_a_state_that_its_input_repeats_stays(n, gate):
    """x = initial = c: every state is c. Two channels, of which one is negative."""
    print("constant", n, gate, flush=True)
    value = torch.tensor([1.0, -0.7], device="cuda")
    h, last = policy.recurrence(value.expand(n, 2), full(n, 2, gate), one_sequence(n), value[None].clone())
    for name, got in (("h", h), ("last", last)):
        off = ((got.double() - value.double()) / value.double()).abs().max().item()
        assert off <= roundings(n) * U, (name, off)


@pytest.mark.parametrize("gate", [12.0, 15.0, 17.0])
def test_a_state_that_its_input_repeats_stays_over_many_chunks(gate):
    """2^25 tokens, 4096 chunks a run of the chain: the maps of many chunks, too, are no products of roundings."""
    n = 2 ** 25
    print("many chunks", gate, flush=True)
    value = torch.tensor([1.0, -0.7], device="cuda")
    h, last = policy.recurrence(value.expand(n, 2), torch.tensor([[gate]], device="cuda").expand(n, 2).contiguous(), one_sequence(n),
                                value[None].clone())
    off = (h / value - 1).abs().max().item()
    assert off <= (roundings(n) + 1) * U, off


def test_a_state_that_its_input_repeats_stays_at_any_gate():
    """Gates 0.01 apart from 0 to 20, a channel each."""
    n, gates = 65536, torch.linspace(0, 20, 2001, device="cuda")
    print("gates", flush=True)
    x = torch.full((n, 2001), -0.7, device="cuda")
    h, _ = policy.recurrence(x, gates.expand(n, 2001), one_sequence(n), x[:1].clone())
    off = (h.double() / x.double() - 1).abs().amax(0)
    assert (off <= roundings(n) * U).all(), (off.max().item(), gates[off.argmax()].item())


@pytest.mark.parametrize("n", [100, 5000, 65536])
@pytest.mark.parametrize("gate", [2.0, 5.5, 8.0, 9.3, 12.0, 15.0, 17.0, 20.0])
def test_decay_and_its_gradients(n, gate):
    """x = 0, initial = 1: h_t = a^t; a cotangent of the last state alone: dx_t = (1 - a) a^(n - t), dinitial = a^n, dgate_t = a (1 - a)
    a^(t - 1) a^(n - t). Each by its own size: an error of the gate's small side of SMALL counts (1 - a) t times."""
    print("decay", n, gate, flush=True)
    x, f, initial = full(n, 1, 0.0).requires_grad_(), full(n, 1, gate).requires_grad_(), full(1, 1, 1.0).requires_grad_()
    h, last = policy.recurrence(x, f, one_sequence(n), initial)
    dx, df, di = torch.autograd.grad(last, (x, f, initial))
    take = 1 / (1 + math.exp(gate))
    log_keep = math.log1p(-take)
    t = torch.arange(1, n + 1, dtype=torch.float64)
    off = (2 * roundings(n) + 1) * U  # of a state and of a cotangent (dgate), and each output's own rounding

    def check(name, got, want, steps):
        got, bound = got.detach().double().cpu().flatten(), (off + SMALL * (1 + take * steps) + U * steps * (take > 0.005)) * want.abs() + 1e-37
        assert torch.isfinite(got).all()
        over = ((got - want).abs() / bound).max().item()
        assert over <= 1, (name, over)
    check("h", h, torch.exp(t * log_keep), t)
    check("last", last, torch.exp(t[-1:] * log_keep), t[-1:])
    check("dinitial", di, torch.exp(t[-1:] * log_keep), t[-1:])
    check("dx", dx, take * torch.exp((n - t) * log_keep), n - t)
    check("dgate", df, take * math.exp(n * log_keep) + 0 * t, n + 0 * t)


@pytest.mark.parametrize("gate", [8.0, 12.0, 17.0])
def test_segments_carried_on_are_the_sequence(gate):
    """A long sequence in segments of 37 tokens, each from the state of the one before: a constant stays. Each segment adds the
    roundings of its own maps at most."""
    print("segments", gate, flush=True)
    n, most = 37, 100
    value = torch.tensor([1.0, -0.7, 3.3], device="cuda")
    state, f = value[None].clone(), full(n, 3, gate)
    for _ in range(most):
        _, state = policy.recurrence(value.expand(n, 3), f, one_sequence(n), state)
    off = ((state.double() - value.double()) / value.double()).abs().max().item()
    assert off <= most * 2 * 4 * U, off  # four maps of 16 tokens a segment, two roundings each


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_steps_of_a_constant_stay(dtype):
    """The control loop's form: a state that its input repeats is the same after any number of steps, bit for bit."""
    gates = torch.tensor([-3.0, 0.0, 1.5, 8.0, 9.5, 12.0, 15.0, 17.0], device="cuda").to(dtype)[None]
    x = torch.tensor([1.0, -0.71875, 3.25, 1.0, 0.40625, -1.0, 1.0, 7.0], device="cuda").to(dtype)[None]
    state = x.float()
    for _ in range(2000):
        _, state = policy.recurrence_step(x, gates, state)
    assert torch.equal(state, x.float())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_states_at_the_ends_of_float32(dtype):
    """States and inputs near the largest value, of opposite signs, do not overflow between them; an infinite input or state
    stays infinite within a stretch and a step, as step by step."""
    big = torch.tensor(3e38, dtype=dtype, device="cuda").float().item()
    gates = torch.tensor([[-20.0, -2.0, 0.0, 2.0, 20.0]], device="cuda").to(dtype)
    f, want = gates, lambda x, s: torch.sigmoid(gates.double()) * s + torch.sigmoid(-gates.double()) * x
    for a, b in ((big, -big), (-big, big)):
        x, s = torch.full((1, 5), a, device="cuda").to(dtype), torch.full((1, 5), b, device="cuda")
        for got in (policy.recurrence_step(x, f, s)[1], policy.recurrence(x, f, one_sequence(1), s)[1]):
            assert ((got.double() - want(a, b)).abs() <= 2.0 ** -19 * big).all()
        n = 12  # a stretch
        h, last = policy.recurrence(x.expand(n, 5), f.expand(n, 5), one_sequence(n), s)
        assert torch.isfinite(last).all()
        leaves = [t.detach().clone().requires_grad_() for t in (x.expand(n, 5), f.expand(n, 5), s)]
        out = policy.recurrence(leaves[0], leaves[1], one_sequence(n), leaves[2])
        dx, _, di = torch.autograd.grad(out[1], leaves, torch.full((1, 5), 1e-10, device="cuda"))
        assert torch.isfinite(dx).all() and torch.isfinite(di).all()
    inf = torch.full((1, 5), math.inf, device="cuda")
    zero = torch.zeros((1, 5), device="cuda")
    for x, s in ((inf.to(dtype), zero), (zero.to(dtype), inf), (-inf.to(dtype), zero), (inf.to(dtype), inf)):
        sign = torch.sign((x.float() + s)[0, 0]).item() * math.inf
        assert (policy.recurrence_step(x, f, s)[1] == sign).all()
        h, last = policy.recurrence(x, f, one_sequence(1), s)
        assert (last == sign).all() and (h.float() == sign).all()
