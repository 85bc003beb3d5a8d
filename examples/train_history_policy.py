"""A policy with memory, trained through the control step: backpropagation through a rollout of the G1 with the operators
of nablaengine_amd.policy, then the same policy in the control loop over cached histories.

    python examples/train_history_policy.py [--worlds 256] [--steps 8] [--updates 5]

Each world's policy sees its states so far. A state is normed and embedded (layer_norm), its query attends over the
world's states from the rollout's start (attention: one query a sequence, with gradients; attention_step over a cache in
the control loop, without), and the result is normed once more and mapped to controls about the nominal ones. The loss asks the
base to stay at its height and the body to be still; its gradient runs back through every step's contact dynamics, which
makes it large now and then: clip_grad_norm_ bounds what the optimizer sees.
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from nablaengine_amd import policy, synthetic, torch_ffi  # noqa: E402

HEADS, KV_HEADS, DIM, WIDTH = 4, 2, 32, 128
KEYS = ("qpos", "qvel", "warm", "ctrl", "friction", "com")


class HistoryPolicy(torch.nn.Module):
    def __init__(self, nominal):
        super().__init__()
        self.register_buffer("nominal", nominal)
        observations = torch_ffi.NQ - 2 + torch_ffi.NV  # where the base is on the plane is not observed
        self.embed = torch.nn.Linear(observations, WIDTH)
        self.project = torch.nn.Linear(WIDTH, (HEADS + 2 * KV_HEADS) * DIM)
        self.head = torch.nn.Linear(WIDTH, torch_ffi.NU)
        self.scales = torch.nn.ParameterList([torch.ones(WIDTH) for _ in range(2)])
        self.shifts = torch.nn.ParameterList([torch.zeros(WIDTH) for _ in range(2)])
        torch.nn.init.normal_(self.head.weight, std=0.01)
        torch.nn.init.zeros_(self.head.bias)

    def tokens(self, qpos, qvel):
        """The state's embedding (worlds, WIDTH), its query (worlds, HEADS, DIM), key and value (worlds, KV_HEADS, DIM)."""
        x = policy.layer_norm(self.embed(torch.cat([qpos[:, 2:], qvel], 1)), self.scales[0], self.shifts[0])
        heads = self.project(x).bfloat16().view(len(x), HEADS + 2 * KV_HEADS, DIM)
        return x, heads[:, :HEADS], heads[:, HEADS:HEADS + KV_HEADS], heads[:, HEADS + KV_HEADS:]

    def controls(self, x, seen):
        x = policy.layer_norm(x + seen.float().flatten(1), self.scales[1], self.shifts[1])
        return self.nominal + 0.3 * torch.tanh(self.head(x))


def rollout(net, state, friction, com, steps):
    """`steps` differentiable steps: [(qpos, qvel)] and the controls."""
    q, v, warm = state
    worlds, keys, values, states, controls = len(q), [], [], [], []
    one = torch.arange(worlds + 1, dtype=torch.int32, device=q.device)
    for t in range(steps):
        x, query, key, value = net.tokens(q, v)
        keys.append(key)
        values.append(value)
        past = [torch.stack(s, 1).flatten(0, 1) for s in (keys, values)]  # each world's tokens, one after another
        u = net.controls(x, policy.attention(query, *past, one, one * (t + 1)))
        q, v, warm = torch_ffi.step(q, v, warm, u, friction, com, normal=0)
        states.append((q, v))
        controls.append(u)
    return states, controls


@torch.no_grad()
def control_loop(net, state, friction, com, steps):
    """The same policy without gradients, its histories in caches of `steps` tokens."""
    q, v, warm = state
    cache = torch.empty((2, len(q), steps, KV_HEADS, DIM), dtype=torch.bfloat16, device=q.device)
    lengths = torch.zeros(len(q), dtype=torch.int32, device=q.device)
    states, controls = [], []
    for t in range(steps):
        x, query, cache[0, :, t], cache[1, :, t] = net.tokens(q, v)
        lengths += 1
        u = net.controls(x, policy.attention_step(query, cache[0], cache[1], lengths))
        q, v, warm = torch_ffi.step(q, v, warm, u, friction, com)
        states.append((q, v))
        controls.append(u)
    return states, controls


def loss_of(states, height):
    return sum(10 * ((q[:, 2] - height) ** 2).mean() + 0.1 * (v ** 2).sum(1).mean() for q, v in states) / len(states)


def train(worlds=256, steps=8, updates=5, seed=0, report=print):
    """Returns the trained policy, its loss before each update, and the arrays of its worlds."""
    torch_ffi.init()
    torch.manual_seed(seed)
    st = {k: torch.from_numpy(x).cuda() for k, x in synthetic.states(worlds, config=1).items() if k in KEYS}
    state = (st["qpos"], st["qvel"], st["warm"])
    net = HistoryPolicy(st["ctrl"].mean(0)).cuda()
    optimizer = torch.optim.Adam(net.parameters(), lr=1e-3)
    height, losses = st["qpos"][:, 2].clone(), []
    for i in range(updates):
        states, _ = rollout(net, state, st["friction"], st["com"], steps)
        loss = loss_of(states, height)
        optimizer.zero_grad()
        loss.backward()
        norm = policy.clip_grad_norm_(net.parameters(), 1.0)
        optimizer.step()
        losses.append(loss.item())
        report(f"update {i}: loss {losses[-1]:.5f}, gradient norm before clipping {norm.item():.3g}")
    return net, losses, (state, st["friction"], st["com"], height)


def main():
    p = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    for name, default in (("worlds", 256), ("steps", 8), ("updates", 5)):
        p.add_argument(f"--{name}", type=int, default=default)
    a = p.parse_args()
    net, _, (state, friction, com, height) = train(a.worlds, a.steps, a.updates)
    states, _ = control_loop(net, state, friction, com, a.steps)
    print(f"control loop over cached histories: loss {loss_of(states, height).item():.5f}")


if __name__ == "__main__":
    main()
