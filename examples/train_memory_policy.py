"""A policy with a longer memory, trained through the control step: a recurrent block and a block of windowed attention, between
them the gated residual, all from nablaengine_amd.policy; then the same policy in the control loop, with a state and a few pages of
keys and values a world, however long it runs.

    python examples/train_memory_policy.py [--worlds 256] [--steps 12] [--updates 5]

Each world's policy reads its state so far. The recurrent block's state remembers all steps (recurrence: one token a sequence with
gradients through the carried state; recurrence_step in the control loop), the attention block sees the last WINDOW steps and the
first SINKS (attention with a window; attention_paged over pages in the control loop, which cache_append_ fills: pages that left the
window take the next steps' keys). Each block's output is normed, gated and scaled onto the residual stream (gated_residual).
The loss asks the base to stay at its height and the body to be still; clip_grad_norm_ bounds what the optimizer sees of the
contacts' gradients.
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from nablaengine_amd import policy, synthetic, torch_ffi  # noqa: E402

HEADS, KV_HEADS, DIM, WIDTH = 4, 2, 32, 128
WINDOW, SINKS, PAGE = 6, 1, 4
OBSERVATIONS = torch_ffi.NQ - 2 + torch_ffi.NV  # where the base is on the plane is not observed
KEYS = ("qpos", "qvel", "warm", "ctrl", "friction", "com")


class MemoryPolicy(torch.nn.Module):
    def __init__(self, nominal):
        super().__init__()
        self.register_buffer("nominal", nominal)
        self.embed = torch.nn.Linear(OBSERVATIONS, WIDTH)
        self.recur = torch.nn.Linear(WIDTH, 3 * WIDTH)  # the recurrence's input and gate, and the residual's gate
        self.mix = torch.nn.Linear(WIDTH, WIDTH)
        self.project = torch.nn.Linear(WIDTH, (HEADS + 2 * KV_HEADS) * DIM + WIDTH)  # queries, keys, values, the residual's gate
        self.join = torch.nn.Linear(HEADS * DIM, WIDTH)
        self.head = torch.nn.Linear(WIDTH, torch_ffi.NU)
        # of the input's norm and its bias, then each block's: its norm, the next norm, its residual's scale
        self.vectors = torch.nn.ParameterList([torch.full((WIDTH,), v) for v in (1.0, 0.0, 1.0, 1.0, 0.5, 1.0, 1.0, 0.5)])
        with torch.no_grad():
            self.recur.bias[WIDTH:2 * WIDTH] = 3.0  # states that last some 20 steps to begin with
        torch.nn.init.normal_(self.head.weight, std=0.01)
        torch.nn.init.zeros_(self.head.bias)

    def begin(self, observations):
        """The residual stream and its norm."""
        y = self.embed(observations)
        return y, policy.layer_norm(y, *self.vectors[:2])

    def recurrent(self, y, z, recurrence):
        """The recurrent block; recurrence(x, gate) -> (h, states)."""
        x, gate, open_ = self.recur(z).chunk(3, 1)
        h, state = recurrence(x, gate)
        w, after, scale = self.vectors[2:5]
        return *policy.gated_residual(y, self.mix(h), w, after, gate=open_, scale=scale), state

    def attending(self, y, z, attention):
        """The attention block and the controls; attention(q, k, v) -> out."""
        out = self.project(z)
        heads, open_ = out[:, :-WIDTH].bfloat16().view(len(z), HEADS + 2 * KV_HEADS, DIM), out[:, -WIDTH:]
        seen = attention(heads[:, :HEADS], heads[:, HEADS:HEADS + KV_HEADS], heads[:, HEADS + KV_HEADS:])
        w, after, scale = self.vectors[5:8]
        _, z = policy.gated_residual(y, self.join(seen.float().flatten(1)), w, after, gate=open_, scale=scale)
        return self.nominal + 0.3 * torch.tanh(self.head(z))

    def forward(self, observations, starts, initial=None):
        """The controls of whole episodes, packed one after another, and each one's last state."""
        y, z = self.begin(observations)
        y, z, state = self.recurrent(y, z, lambda x, gate: policy.recurrence(x, gate, starts, initial))
        return self.attending(y, z, lambda q, k, v: policy.attention(q, k, v, starts, window=WINDOW, sinks=SINKS)), state


def observe(qpos, qvel):
    return torch.cat([qpos[:, 2:], qvel], 1)


def rollout(net, state, friction, com, steps):
    """`steps` differentiable steps: [(qpos, qvel)], the observations and the controls."""
    q, v, warm = state
    worlds, keys, values, states, seen, controls = len(q), [], [], [], [], []
    one = torch.arange(worlds + 1, dtype=torch.int32, device=q.device)
    memory = torch.zeros((worlds, WIDTH), device=q.device)

    def attend(query, key, value):
        keys.append(key)
        values.append(value)
        past = [torch.stack(s, 1).flatten(0, 1) for s in (keys, values)]  # each world's tokens, one after another
        return policy.attention(query, *past, one, one * len(keys), window=WINDOW, sinks=SINKS)
    for _ in range(steps):
        seen.append(observe(q, v))
        y, z = net.begin(seen[-1])
        y, z, memory = net.recurrent(y, z, lambda x, gate: policy.recurrence(x, gate, one, memory))
        u = net.attending(y, z, attend)
        q, v, warm = torch_ffi.step(q, v, warm, u, friction, com, normal=0)
        states.append((q, v))
        controls.append(u)
    return states, seen, controls


def page_tables(worlds, steps):
    """Which page of the pool holds each world's tokens, and the pool's pages: the sinks' own, and a ring that the window turns
    over."""
    first, ring = -(-SINKS // PAGE), -(-WINDOW // PAGE) + 1
    page = torch.arange(-(-steps // PAGE))
    turn = torch.where(page < first, page, first + (page - first) % ring)
    return (torch.arange(worlds)[:, None] * (first + ring) + turn).to(torch.int32).cuda(), worlds * (first + ring)


@torch.no_grad()
def control_loop(net, state, friction, com, steps):
    """The same policy without gradients: a state and a few pages a world."""
    q, v, warm = state
    pages, count = page_tables(len(q), steps)
    pools = torch.empty((2, count, PAGE, KV_HEADS, DIM), dtype=torch.bfloat16, device=q.device)
    lengths = torch.zeros(len(q), dtype=torch.int32, device=q.device)
    memory = torch.zeros((len(q), WIDTH), device=q.device)
    states, controls = [], []

    def attend(query, key, value):
        policy.cache_append_(pools[0], pools[1], key, value, pages, lengths)
        lengths.add_(1)
        return policy.attention_paged(query, pools[0], pools[1], pages, lengths, window=WINDOW, sinks=SINKS)
    for _ in range(steps):
        y, z = net.begin(observe(q, v))
        y, z, memory = net.recurrent(y, z, lambda x, gate: policy.recurrence_step(x, gate, memory))
        u = net.attending(y, z, attend)
        q, v, warm = torch_ffi.step(q, v, warm, u, friction, com)
        states.append((q, v))
        controls.append(u)
    return states, controls


def loss_of(states, height):
    return sum(10 * ((q[:, 2] - height) ** 2).mean() + 0.1 * (v ** 2).sum(1).mean() for q, v in states) / len(states)


def train(worlds=256, steps=12, updates=5, seed=0, report=print):
    """Returns the trained policy, its loss before each update, and the arrays of its worlds."""
    torch_ffi.init()
    torch.manual_seed(seed)
    st = {k: torch.from_numpy(x).cuda() for k, x in synthetic.states(worlds, config=1).items() if k in KEYS}
    state = (st["qpos"], st["qvel"], st["warm"])
    net = MemoryPolicy(st["ctrl"].mean(0)).cuda()
    optimizer = torch.optim.Adam(net.parameters(), lr=1e-3)
    height, losses = st["qpos"][:, 2].clone(), []
    for i in range(updates):
        states, _, _ = rollout(net, state, st["friction"], st["com"], steps)
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
    for name, default in (("worlds", 256), ("steps", 12), ("updates", 5)):
        p.add_argument(f"--{name}", type=int, default=default)
    a = p.parse_args()
    net, _, (state, friction, com, height) = train(a.worlds, a.steps, a.updates)
    states, _ = control_loop(net, state, friction, com, a.steps)
    print(f"control loop over states and pages: loss {loss_of(states, height).item():.5f}")


if __name__ == "__main__":
    main()
