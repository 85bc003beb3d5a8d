"""The example policy with a longer memory (examples/train_memory_policy.py): training through the control step and the control
loop run, the three forms of the policy (whole episodes, a step at a time with gradients, the control loop over states and pages)
give the same controls, and the gradients of whole episodes are those of its definition in float64."""
import importlib.util
import math
import os

import pytest
import torch

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def example():
    if not torch.cuda.is_available():
        pytest.fail("no GPU visible")
    spec = importlib.util.spec_from_file_location("train_memory_policy", os.path.join(ROOT, "examples", "train_memory_policy.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def test_training_and_control_loop(example):
    steps = 12  # twice the window: pages are used again
    net, losses, (state, friction, com, height) = example.train(worlds=64, steps=steps, updates=3, report=lambda s: print(s, flush=True))
    assert all(math.isfinite(x) for x in losses), losses
    with torch.no_grad():
        _, seen, trained = example.rollout(net, state, friction, com, steps)
        starts = torch.arange(65, dtype=torch.int32, device="cuda") * steps
        whole, _ = net(torch.stack(seen, 1).flatten(0, 1), starts)
    _, looped = example.control_loop(net, state, friction, com, steps)
    # controls are 0.3 tanh of a product with weights of about 0.01 x sqrt(128); what differs is the attention's roundings
    # (bfloat16: 2^-8 of values that a norm follows), and in the control loop also the states that came of them
    for t in range(steps):
        assert (trained[t] - whole.view(64, steps, -1)[:, t]).abs().max() < 2e-3, t
    assert (trained[0] - looped[0]).abs().max() < 2e-3
    assert (trained[3] - looped[3]).abs().max() < 2e-2


def test_control_loop_is_the_policy_on_what_it_saw(example):
    """The control loop's controls at every step, past many turns of the pages, against whole episodes of the same observations."""
    net, _, (state, friction, com, _) = example.train(worlds=33, steps=2, updates=1, report=lambda s: None)
    steps = 40
    states, looped = example.control_loop(net, state, friction, com, steps)
    seen = [example.observe(q, v) for q, v in [state[:2]] + states[:-1]]
    with torch.no_grad():
        whole, _ = net(torch.stack(seen, 1).flatten(0, 1), torch.arange(34, dtype=torch.int32, device="cuda") * steps)
    assert (torch.stack(looped, 1).flatten(0, 1) - whole).abs().max() < 2e-3


def test_training_is_the_same_every_time(example):
    a, b = (example.train(worlds=33, steps=3, updates=2, report=lambda s: None) for _ in range(2))
    assert a[1] == b[1]


def plain64(example, net, observations, lengths, initial):
    """The policy's definition in float64, by torch's own operations and derivatives."""
    p = {k: v.detach().double().requires_grad_() for k, v in net.named_parameters()}
    vec = [p[f"vectors.{i}"] for i in range(8)]
    linear = lambda name, x: x @ p[name + ".weight"].t() + p[name + ".bias"]  # noqa: E731
    rms = lambda v: v / (v.square().mean(-1, keepdim=True) + 1e-5).sqrt()  # noqa: E731
    y = linear("embed", observations.double())
    z = torch.nn.functional.layer_norm(y, (example.WIDTH,), vec[0], vec[1], 1e-5)
    x, gate, open_ = linear("recur", z).chunk(3, 1)
    hs, t = [], 0
    for s, n in enumerate(lengths):
        h = initial[s].double()
        for i in range(t, t + n):
            a = torch.sigmoid(gate[i])
            h = a * h + (1 - a) * x[i]
            hs.append(h)
        t += n
    y = y + vec[4] * torch.sigmoid(open_) * rms(linear("mix", torch.stack(hs))) * vec[2]
    out = linear("project", rms(y) * vec[3])
    heads, open_ = out[:, :-example.WIDTH].view(len(out), -1, example.DIM), out[:, -example.WIDTH:]
    seen, t, H, K = [], 0, example.HEADS, example.KV_HEADS
    for n in lengths:
        i, j = torch.arange(n, device="cuda")[:, None], torch.arange(n, device="cuda")
        mask = (j <= i) & ((j > i - example.WINDOW) | (j < example.SINKS))
        one = []
        for h in range(H):
            k = H + h // (H // K)
            q, key, value = heads[t:t + n, h], heads[t:t + n, k], heads[t:t + n, k + K]
            one.append(torch.softmax((q @ key.t() / math.sqrt(example.DIM)).masked_fill(~mask, -math.inf), 1) @ value)
        seen.append(torch.stack(one, 1))
        t += n
    y = y + vec[7] * torch.sigmoid(open_) * rms(linear("join", torch.cat(seen).flatten(1))) * vec[5]
    return net.nominal.double() + 0.3 * torch.tanh(linear("head", rms(y) * vec[6])), p


def test_gradients_of_whole_episodes(example):
    """All parameters' gradients of a packed batch against the definition in float64. The policy rounds to bfloat16 the queries, keys
    and values, the probabilities and the outputs, and on the way back the outputs' gradients, the probabilities, the score gradients
    and the three gradients: eight roundings of at most 2^-8 of what they round, and each of those is a part of what the gradients
    are made of; their norm is off by less than the eight together."""
    torch.manual_seed(3)
    lengths = [30, 1, 7, 64]
    net = example.MemoryPolicy(torch.zeros(example.torch_ffi.NU)).cuda()
    with torch.no_grad():
        net.head.weight.mul_(30)  # as much for the controls as training makes it
    observations = torch.randn(sum(lengths), example.OBSERVATIONS, device="cuda")
    initial = torch.randn(len(lengths), example.WIDTH, device="cuda")
    cot = torch.randn(sum(lengths), example.torch_ffi.NU, device="cuda")
    starts = torch.tensor([0] + lengths).cumsum(0).to(torch.int32).cuda()
    names, leaves = zip(*net.named_parameters())
    u, _ = net(observations, starts, initial)
    got = torch.autograd.grad(u, leaves, cot)
    want_u, p = plain64(example, net, observations, lengths, initial)
    want = torch.autograd.grad(want_u, [p[n] for n in names], cot.double())
    assert (u - want_u).norm() <= 2.0 ** -8 * want_u.norm()
    for name, g, w in zip(names, got, want):
        assert (g.double() - w).norm() <= 8 * 2.0 ** -8 * w.norm(), (name, ((g.double() - w).norm() / w.norm()).item())
