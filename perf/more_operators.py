"""Performance cases of the operators that policies with a longer memory are built from (the package's `policy` module), in
plain torch and as the package's calls.

A case is one operator (`op`) over a batch of the framework's shapes: thousands of worlds, rollouts of tens of steps,
episodes and recordings of up to some minutes of 20 ms steps.

  scan       policy.recurrence: a gated linear recurrence over packed episodes, from each one's carried state; train: with
             the gradients of x, gate and the carried states
  tick       policy.recurrence_step: the same recurrence one token a world, from the worlds' states to their next ones
  residual   policy.gated_residual: a block's output normed, gated and scaled onto the residual stream, and the stream
             normed for the next block; train: with the gradients of all that enter
  window     policy.attention over packed episodes with a sliding window and first tokens that stay visible (sinks);
             train: with the gradients of q, k and v
  paged      policy.cache_append_ and policy.attention_paged: each world's new key and value into its pages, then its one
             new query over the history that its pages hold, with or without a window
"""
import math
import random

import torch

own = False

_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_BYTES = {"f32": 4, "bf16": 2, "f16": 2}
EPS = 1e-5


def _scan(episodes, longest, channels, dtype, train, carried=True, **kw):
    return dict(op="scan", episodes=episodes, longest=longest, channels=channels, dtype=dtype, train=train, carried=carried, **kw)


def _tick(worlds, channels, dtype, **kw):
    return dict(op="tick", worlds=worlds, channels=channels, dtype=dtype, **kw)


def _residual(rows, width, dtype, train, gated=True, scaled=True, pad=0, **kw):
    return dict(op="residual", rows=rows, width=width, dtype=dtype, train=train, gated=gated, scaled=scaled, pad=pad, **kw)


def _window(episodes, longest, heads, kv_heads, dim, dtype, train, window, sinks, past=0, **kw):
    return dict(op="window", episodes=episodes, longest=longest, heads=heads, kv_heads=kv_heads, dim=dim, dtype=dtype, train=train,
                window=window, sinks=sinks, past=past, **kw)


def _paged(worlds, capacity, page, heads, kv_heads, dim, dtype, window=0, sinks=0, **kw):
    return dict(op="paged", worlds=worlds, capacity=capacity, page=page, heads=heads, kv_heads=kv_heads, dim=dim, dtype=dtype,
                window=window, sinks=sinks, **kw)


def listed():
    return [
        # rollout segments of at most 32 steps, cut short where a robot fell, each from the state that its world carried
        _scan(4096, 32, 512, "bf16", True, name="scan_segments"),
        # two long recordings, hundreds of seconds
        _scan(2, 32768, 1024, "bf16", True, carried=False, name="scan_long"),
        # one robot in the control loop, where latency is all there is
        _tick(1, 512, "f32", name="tick_control"),
        # all worlds of a large batch, one step
        _tick(16384, 1024, "bf16", name="tick_worlds"),
        # one robot in the control loop
        _residual(1, 256, "f32", False, name="residual_control"),
        # an odd batch of rows of a wider buffer, a block without a gate
        _residual(1331, 99, "f16", True, gated=False, pad=29, name="residual_odd"),
        # a policy's block over a whole rollout: 4096 worlds x 32 steps
        _residual(131072, 512, "bf16", True, name="residual_rollout"),
        # whole episodes of at most 20 s, each step seeing the last 2.5 s and the episode's start
        _window(256, 1000, 8, 2, 64, "bf16", True, 128, 4, name="window_episodes"),
        # two long recordings, the largest heads
        _window(2, 8192, 16, 4, 128, "bf16", True, 1000, 16, name="window_long"),
        # one robot in the control loop, attending to its last seconds and its start; the pages between are free again
        _paged(1, 4096, 16, 8, 8, 64, "bf16", 256, 4, name="paged_control"),
        # the headline batch of worlds, each with its own history in one pool of pages
        _paged(4096, 512, 16, 8, 2, 64, "bf16", name="paged_worlds"),
        # few worlds with long histories
        _paged(4, 131072, 64, 16, 4, 128, "f16", name="paged_long"),
    ]


def _spread(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49)))))))


def draw(rng):
    op = rng.choice(["scan", "scan", "tick", "residual", "window", "window", "paged", "paged"])
    if op == "scan":
        channels = _spread(rng, 16, 2048)
        longest = _spread(rng, 1, 32768)
        most = max(1, (1 << 25) // channels)
        longest = min(longest, most)
        return _scan(_spread(rng, 1, max(1, min(8192, most // longest))), longest, channels, rng.choice(["bf16", "bf16", "f16", "f32"]),
                     rng.choice([True, True, False]), carried=rng.choice([True, False]))
    if op == "tick":
        channels = _spread(rng, 16, 2048)
        return _tick(_spread(rng, 1, min(16384, (1 << 24) // channels)), channels, rng.choice(["bf16", "f16", "f32"]))
    if op == "residual":
        width = _spread(rng, 8, 8192)
        rows = _spread(rng, 1, min(131072, (1 << 26) // width // 2))
        return _residual(rows, width, rng.choice(["f32", "bf16", "f16"]), rng.choice([True, True, False]),
                         gated=rng.choice([True, True, False]), scaled=rng.choice([True, False]),
                         pad=rng.choice([0, 0, rng.randint(1, 64)]))
    dim, dtype = rng.choice([64, 64, 128, 40]), rng.choice(["bf16", "bf16", "f16"])
    kv_heads = rng.choice([1, 2, 4])
    heads = kv_heads * rng.choice([1, 2, 3, 4])
    if op == "window":
        longest = _spread(rng, 1, 4096)
        episodes = _spread(rng, 1, max(1, min(4096, 131072 // longest, (1 << 26) // longest ** 2)))
        return _window(episodes, longest, heads, kv_heads, dim, dtype, rng.choice([True, True, False]), _spread(rng, 1, 1500),
                       rng.choice([0, 1, 4, _spread(rng, 1, 200)]), past=rng.choice([0, 0, _spread(rng, 1, longest)]))
    page = rng.choice([1, 8, 16, 16, 32, 64, 128])
    capacity = -(-_spread(rng, 1, 65536) // page) * page
    window = rng.choice([0, 0, _spread(rng, 1, 4096)])
    return _paged(_spread(rng, 1, max(1, min(4096, (1 << 20) // capacity))), capacity, page, heads, kv_heads, dim, dtype, window,
                  rng.choice([0, 4, _spread(rng, 1, 64)]) if window else 0)


# ---- shapes and values ----------------------------------------------------------------------------------------------

def _lengths(case):
    """(queries, keys) of each episode: most run to the end, the others fall at any time; some have earlier keys
    (`past` at most) before their first query."""
    rng = random.Random(case["episodes"] * 100003 + case["longest"])
    most, past = case["longest"], case.get("past", 0)
    q = [most if rng.random() < 0.3 else rng.randint(1, most) for _ in range(case["episodes"])]
    q[0] = most
    return q, [n + (rng.randint(0, past) if past else 0) for n in q]


def _histories(case):
    """The length of each world's history with its new token: anything from that token alone (a world just reset) to the
    whole capacity."""
    rng = random.Random(case["worlds"] * 100003 + case["capacity"])
    n = [rng.randint(1, case["capacity"]) if rng.random() < 0.5 else case["capacity"] for _ in range(case["worlds"])]
    n[0] = case["capacity"]
    return n


def _seen(length, window, sinks):
    """How many of a history's `length` tokens its newest one sees."""
    return min(length, window + min(sinks, max(0, length - window))) if window else length


def _pairs(case):
    """The (query, key) pairs that the mask leaves, over all episodes."""
    w, s, total = case["window"], case["sinks"], 0
    upto = {}  # n -> the pairs of the queries at places 0 .. n - 1

    def prefix(n):
        if n not in upto:
            a = min(n, w + s)  # places that see everything before them
            upto[n] = a * (a + 1) // 2 + (n - a) * (w + s)
        return upto[n]
    for nq, nk in zip(*_lengths(case)):
        total += prefix(nk) - prefix(nk - nq)
    return total


def work(case):
    op, b = case["op"], _BYTES[case["dtype"]]
    if op == "scan":
        n, s = sum(_lengths(case)[0]) * case["channels"], case["episodes"] * case["channels"] * 4
        c = s if case["carried"] else 0
        if not case["train"]:
            return {"bytes": 3 * n * b + s + c, "flops": 8 * n}
        # x, gate, the two cotangents in; h, the last states and the gradients out
        return {"bytes": 6 * n * b + 2 * s + 2 * c, "flops": 24 * n}
    if op == "tick":
        n = case["worlds"] * case["channels"]
        return {"bytes": n * (3 * b + 8), "flops": 8 * n}
    if op == "residual":
        n, g, w = case["rows"] * case["width"], int(case["gated"]), case["width"] * 4 * (2 + case["scaled"])
        if not case["train"]:
            return {"bytes": (4 + g) * n * b + w, "flops": 16 * n}
        # x, u, gate, the two cotangents in; y, z and the gradients out
        return {"bytes": (8 + 2 * g) * n * b + 2 * w, "flops": 48 * n}
    h, kv, d = case["heads"], case["kv_heads"], case["dim"]
    if op == "window":
        nq, nk = (sum(x) for x in _lengths(case))
        flops = 4 * d * h * _pairs(case)  # two products, a multiplication and an addition each
        if not case["train"]:
            return {"bytes": b * d * (2 * nq * h + 2 * nk * kv), "flops": flops}
        # the gradients take five products more; q, k, v, the output's gradient in, the output and three gradients out
        return {"bytes": b * d * (4 * nq * h + 4 * nk * kv), "flops": flops * 7 // 2}
    n = sum(_seen(x, case["window"], case["sinks"]) for x in _histories(case))
    # what each query sees (its own new token among it), the queries and outputs, the new tokens in and into their pages
    return {"bytes": b * d * (2 * n * kv + 2 * case["worlds"] * h + 4 * case["worlds"] * kv), "flops": 4 * d * h * n}


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(g, shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def _starts(lengths):
    return torch.tensor([0] + lengths, dtype=torch.int64).cumsum(0).to(torch.int32).cuda()


def prepare(case, seed):
    g, op, dtype = _generator(seed), case["op"], _TYPES[case["dtype"]]
    s = {"case": dict(case)}
    if op == "scan":
        lengths, c, train = _lengths(case)[0], case["channels"], case["train"]
        # as they come: halves of one projection's output. Gates around 3: states that last some 20 steps
        both = _normal(g, (sum(lengths), 2 * c), dtype)
        both[:, c:] += 3.0
        s["x"], s["gate"] = (t.detach().requires_grad_(train) for t in (both[:, :c], both[:, c:]))
        s["starts"], s["longest"] = _starts(lengths), max(lengths)
        s["initial"] = _normal(g, (len(lengths), c)).requires_grad_(train) if case["carried"] else None
        if train:
            s["dh"], s["dlast"] = _normal(g, (sum(lengths), c), dtype), _normal(g, (len(lengths), c))
        return s
    if op == "tick":
        shape = (case["worlds"], case["channels"])
        s["x"], s["gate"], s["state"] = _normal(g, shape, dtype), (_normal(g, shape) + 3.0).to(dtype), _normal(g, shape)
        return s
    if op == "residual":
        rows, width, train = case["rows"], case["width"], case["train"]
        wide = lambda scale=1.0: _normal(g, (rows, width + case["pad"]), dtype, scale)[:, :width].detach().requires_grad_(train)  # noqa: E731
        s["x"], s["u"] = wide(1.5), wide(0.7)
        s["gate"] = wide() if case["gated"] else None
        s["weight"] = (1.0 + _normal(g, (width,), scale=0.2)).requires_grad_(train)
        s["next_weight"] = (1.0 + _normal(g, (width,), scale=0.2)).requires_grad_(train)
        s["scale"] = (0.3 + _normal(g, (width,), scale=0.1)).requires_grad_(train) if case["scaled"] else None
        if train:
            s["dy"], s["dz"] = _normal(g, (rows, width), dtype), _normal(g, (rows, width), dtype)
        return s
    h, kv, d = case["heads"], case["kv_heads"], case["dim"]
    s["scale"] = 1.0 / math.sqrt(d)
    if op == "window":
        lq, lk = _lengths(case)
        s["starts_q"], s["starts_k"], s["longest"] = _starts(lq), _starts(lk), (max(lq), max(lk))
        # as they come: slices of a projection's output
        if case["past"]:
            s["q"] = _normal(g, (sum(lq), h, d), dtype)
            both = _normal(g, (sum(lk), 2 * kv, d), dtype)
            s["k"], s["v"] = both[:, :kv], both[:, kv:]
        else:
            both = _normal(g, (sum(lq), h + 2 * kv, d), dtype)
            s["q"], s["k"], s["v"] = both[:, :h], both[:, h:h + kv], both[:, h + kv:]
        for name in ("q", "k", "v"):
            s[name] = s[name].detach().requires_grad_(case["train"])
        if case["train"]:
            s["dout"] = _normal(g, (sum(lq), h, d), dtype)
        return s
    worlds, page = case["worlds"], case["page"]
    n = _histories(case)
    # a pool of pages of which the worlds hold some, in no order; a page that no token in sight needs is free again (-1)
    lengths = torch.tensor(n, device="cuda")[:, None]
    begin = torch.arange(case["capacity"] // page, device="cuda") * page
    held = begin < lengths
    if case["window"]:
        held &= (begin + page > lengths - case["window"]) | (begin < case["sinks"])
    count = int(held.sum())
    s["pages"] = torch.full(held.shape, -1, dtype=torch.int32, device="cuda")
    s["pages"][held] = torch.randperm(count + 3, generator=g, device="cuda")[:count].to(torch.int32)
    s["k_pages"], s["v_pages"] = (_normal(g, (count + 3, page, kv, d), dtype) for _ in range(2))
    s["q"] = _normal(g, (worlds, h, d), dtype)
    both = _normal(g, (worlds, 2 * kv, d), dtype)
    s["k"], s["v"] = both[:, :kv], both[:, kv:]
    # the histories before the new token, and with it: a control loop adds one in place between the two calls
    s["before"] = torch.tensor([x - 1 for x in n], dtype=torch.int32, device="cuda")
    s["lengths"] = s["before"] + 1
    return s


# ---- the plain forms ------------------------------------------------------------------------------------------------

def _rolled(a, b):
    """h[t] = a[t] h[t - 1] + b[t] from nothing, over the first dimension, by doubling: after the pass of distance d each
    entry stands for its last 2 d steps."""
    n, d = len(a), 1
    while d < n:
        b = torch.cat([b[:d], b[d:] + a[d:] * b[:-d]])
        a = torch.cat([a[:d], a[d:] * a[:-d]])
        d *= 2
    return b


def _plain_scan(s):
    x, f, starts = s["x"].detach().float(), s["gate"].detach().float(), s["starts"].long()
    first, end = starts[:-1], starts[1:] - 1
    keep, take = 1.0 / (1.0 + torch.exp(-f)), 1.0 / (1.0 + torch.exp(f))
    initial = s["initial"].detach() if s["initial"] is not None else x.new_zeros((len(first), x.shape[1]))
    a, b = keep.clone(), take * x
    b[first] += keep[first] * initial
    a[first] = 0.0
    h = _rolled(a, b)
    out = {"h": h.to(s["x"].dtype), "last": h[end]}
    if "dh" in s:
        d = s["dh"].float().clone()
        d[end] += s["dlast"]
        after = torch.cat([a[1:], a.new_zeros((1, a.shape[1]))])  # what a step's state is kept by in the next one
        g = _rolled(after.flip(0), d.flip(0)).flip(0)
        before = torch.cat([h[:1], h[:-1]])
        before[first] = initial
        out["dx"] = (take * g).to(s["x"].dtype)
        out["dgate"] = (g * (before - x) * keep * take).to(s["x"].dtype)
        if s["initial"] is not None:
            out["dinitial"] = keep[first] * g[first]
    return out


def _plain_tick(s):
    f = s["gate"].float()
    new = s["state"] / (1.0 + torch.exp(-f)) + s["x"].float() / (1.0 + torch.exp(f))
    return {"h": new.to(s["x"].dtype), "state": new}


def _plain_residual(s):
    dtype = s["x"].dtype
    x, u, w, w2 = (s[n].detach().float() for n in ("x", "u", "weight", "next_weight"))
    r1 = 1.0 / torch.sqrt((u * u).mean(1, keepdim=True) + EPS)
    uh = u * r1
    sg = 1.0 / (1.0 + torch.exp(-s["gate"].detach().float())) if s["gate"] is not None else torch.ones_like(u)
    scale = s["scale"].detach() if s["scale"] is not None else torch.ones_like(w)
    y = x + scale * sg * (uh * w)
    r2 = 1.0 / torch.sqrt((y * y).mean(1, keepdim=True) + EPS)
    yh = y * r2
    out = {"y": y.to(dtype), "z": (yh * w2).to(dtype)}
    if "dy" in s:
        dz = s["dz"].float()
        gz = dz * w2
        dy = s["dy"].float() + r2 * (gz - yh * (gz * yh).mean(1, keepdim=True))
        out["dx"] = dy.to(dtype)
        gn = dy * scale * sg * w
        out["du"] = (r1 * (gn - uh * (gn * uh).mean(1, keepdim=True))).to(dtype)
        if s["gate"] is not None:
            out["dgate"] = (dy * scale * uh * w * sg * (1.0 - sg)).to(dtype)
        m = (dy * sg * uh).sum(0)
        out["dweight"], out["dnext_weight"] = scale * m, (dz * yh).sum(0)
        if s["scale"] is not None:
            out["dscale"] = w * m
    return out


def _places(starts, longest):
    """For each episode and each place up to the longest's: the token's index (0 where there is none), and whether there is one."""
    place = torch.arange(longest, device=starts.device)
    lengths = (starts[1:] - starts[:-1]).long()
    there = place < lengths[:, None]
    return torch.where(there, starts[:-1].long()[:, None] + place, 0), there, lengths


def _plain_window(s):
    q, k, v = (s[n].detach() for n in ("q", "k", "v"))
    heads, kv, window, sinks = q.shape[1], k.shape[1], s["case"]["window"], s["case"]["sinks"]
    iq, there_q, nq = _places(s["starts_q"], s["longest"][0])
    ik, there_k, nk = _places(s["starts_k"], s["longest"][1])
    # the mask of each episode: query i, of nq, is at place i + nk - nq, and sees the `window` keys up to there and the first ones
    place = (torch.arange(s["longest"][0], device=q.device) + (nk - nq)[:, None])[:, :, None]
    key = torch.arange(s["longest"][1], device=q.device)
    mask = (key <= place) & ((key > place - window) | (key < sinks)) & there_q[:, :, None] & there_k[:, None]
    G = heads // kv
    spread = lambda x, i: x[i].float().transpose(1, 2)  # noqa: E731   (episode, head, place, d)
    share = lambda x: x.repeat_interleave(G, 1)  # noqa: E731
    join = lambda x: x.view(len(nq), kv, G, *x.shape[2:]).sum(2)  # noqa: E731
    qs, ks, vs = spread(q, iq), share(spread(k, ik)), share(spread(v, ik))
    scores = torch.matmul(qs, ks.transpose(2, 3).contiguous()) * s["scale"]
    scores = scores.masked_fill(~mask[:, None], float("-inf"))
    p = torch.exp(scores - scores.amax(3, keepdim=True).clamp(min=-1e30))
    del scores
    p = p / p.sum(3, keepdim=True).clamp(min=1e-30)
    pack = lambda x, there: x.transpose(1, 2)[there].to(q.dtype)  # noqa: E731
    o = torch.matmul(p, vs)
    out = {"out": pack(o, there_q)}
    if "dout" in s:
        do = spread(s["dout"], iq).masked_fill(~there_q[:, None, :, None], 0.0)
        out["dv"] = pack(join(torch.matmul(p.transpose(2, 3).contiguous(), do)), there_k)
        ds = p * (torch.matmul(do, vs.transpose(2, 3).contiguous()) - (do * o).sum(3, keepdim=True)) * s["scale"]
        out["dq"] = pack(torch.matmul(ds, ks), there_q)
        out["dk"] = pack(join(torch.matmul(ds.transpose(2, 3).contiguous(), qs)), there_k)
    return out


def _plain_paged(s):
    case, q, kp, vp, table = s["case"], s["q"], s["k_pages"], s["v_pages"], s["pages"].long()
    worlds, kv, d, page = q.shape[0], kp.shape[2], q.shape[2], case["page"]
    at = s["before"].long()
    slot = table[torch.arange(worlds, device=q.device), at // page]
    kp[slot, at % page], vp[slot, at % page] = s["k"], s["v"]
    place, n = torch.arange(case["capacity"], device=q.device), s["lengths"].long()[:, None]
    there = place < n
    if case["window"]:
        there &= (place >= n - case["window"]) | (place < case["sinks"])
    held = table.clamp(min=0)
    qs = q.float().view(worlds, kv, -1, d)
    ks = kp[held].flatten(1, 2).permute(0, 2, 3, 1).float().contiguous()
    scores = (torch.matmul(qs, ks) * s["scale"]).masked_fill(~there[:, None, None], float("-inf"))
    p = torch.exp(scores - scores.amax(3, keepdim=True))
    p = p / p.sum(3, keepdim=True)
    vs = vp[held].flatten(1, 2).transpose(1, 2).float().contiguous()
    return {"out": torch.matmul(p, vs).view_as(q).to(q.dtype), "k_pages": kp, "v_pages": vp}


# ---- the package's calls --------------------------------------------------------------------------------------------

def _grads(outs, cotangents, leaves):
    """The gradients of those leaves that there are, by name."""
    leaves = {n: t for n, t in leaves.items() if t is not None}
    return dict(zip(leaves, torch.autograd.grad(outs, list(leaves.values()), cotangents)))


def _own(s):
    from nablaengine_amd import policy
    op = s["case"]["op"]
    if op == "scan":
        h, last = policy.recurrence(s["x"], s["gate"], s["starts"], s["initial"])
        if "dh" not in s:
            return {"h": h, "last": last}
        return {"h": h.detach(), "last": last.detach(),
                **_grads((h, last), (s["dh"], s["dlast"]), {"dx": s["x"], "dgate": s["gate"], "dinitial": s["initial"]})}
    if op == "tick":
        h, state = policy.recurrence_step(s["x"], s["gate"], s["state"])
        return {"h": h, "state": state}
    if op == "residual":
        y, z = policy.gated_residual(s["x"], s["u"], s["weight"], s["next_weight"], gate=s["gate"], scale=s["scale"], eps=EPS)
        if "dy" not in s:
            return {"y": y, "z": z}
        return {"y": y.detach(), "z": z.detach(),
                **_grads((y, z), (s["dy"], s["dz"]), {"dx": s["x"], "du": s["u"], "dgate": s["gate"], "dweight": s["weight"],
                                                      "dnext_weight": s["next_weight"], "dscale": s["scale"]})}
    window, sinks = s["case"]["window"] or None, s["case"]["sinks"]
    if op == "window":
        o = policy.attention(s["q"], s["k"], s["v"], s["starts_q"], s["starts_k"], scale=s["scale"], window=window, sinks=sinks)
        if "dout" not in s:
            return {"out": o}
        return {"out": o.detach(), **_grads(o, s["dout"], {"dq": s["q"], "dk": s["k"], "dv": s["v"]})}
    policy.cache_append_(s["k_pages"], s["v_pages"], s["k"], s["v"], s["pages"], s["before"])
    out = policy.attention_paged(s["q"], s["k_pages"], s["v_pages"], s["pages"], s["lengths"], scale=s["scale"], window=window, sinks=sinks)
    return {"out": out, "k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def run(state):
    if own:
        return _own(state)
    return {"scan": _plain_scan, "tick": _plain_tick, "residual": _plain_residual, "window": _plain_window, "paged": _plain_paged}[
        state["case"]["op"]](state)


# ---- the definitions in 64 bits -------------------------------------------------------------------------------------

def _softmax64(scores):
    """exp(s) / sum exp(s) over the last axis; zeros where every score is -inf."""
    top = scores.max(-1, keepdim=True).values
    e = torch.where(torch.isinf(scores), 0.0, (scores - torch.where(torch.isinf(top), 0.0, top)).exp())
    total = e.sum(-1, keepdim=True)
    return e / torch.where(total == 0, 1.0, total)


def _exact_scan(case, s):
    """Step by step, all episodes beside one another, the longer ones first: those that still run are a leading part."""
    lengths, c = _lengths(case)[0], case["channels"]
    order = sorted(range(len(lengths)), key=lambda i: -lengths[i])
    first = s["starts"].long()[:-1][torch.tensor(order, device="cuda")]
    running, alive = [], len(order)
    for t in range(max(lengths)):
        while lengths[order[alive - 1]] <= t:
            alive -= 1
        running.append(alive)
    x, keep = s["x"].detach().double(), torch.sigmoid(s["gate"].detach().double())
    h = torch.zeros((len(order), c), dtype=torch.float64, device="cuda")
    if case["carried"]:
        h = s["initial"].detach().double()[torch.tensor(order, device="cuda")]
    before, states = torch.empty_like(x), torch.empty_like(x)
    for t, n in enumerate(running):
        i = first[:n] + t
        before[i] = h[:n]
        h[:n] = x[i] + keep[i] * (h[:n] - x[i])
        states[i] = h[:n]
    back = torch.tensor(order, device="cuda").argsort()
    out = {"h": states, "last": h[back]}
    if case["train"]:
        dh, g = s["dh"].double(), s["dlast"].double()[torch.tensor(order, device="cuda")]
        gs = torch.empty_like(x)
        for t in range(len(running) - 1, -1, -1):
            n = running[t]
            i = first[:n] + t
            total = g[:n] + dh[i]
            gs[i] = total
            g[:n] = total * keep[i]
        out["dx"] = gs - gs * keep
        out["dgate"] = gs * (before - x) * (keep - keep * keep)
        if case["carried"]:
            out["dinitial"] = g[back]
    return out


def _exact_residual(case, s):
    """By torch's derivatives of the definition in float64."""
    names = [n for n in ("x", "u", "gate", "weight", "next_weight", "scale") if s[n] is not None]
    t = {n: s[n].detach().double().requires_grad_(case["train"]) for n in names}
    rms = lambda v: v / (v.square().mean(-1, keepdim=True) + EPS).sqrt()  # noqa: E731
    branch = rms(t["u"]) * t["weight"]
    if "gate" in t:
        branch = branch * torch.sigmoid(t["gate"])
    if "scale" in t:
        branch = branch * t["scale"]
    y = t["x"] + branch
    z = rms(y) * t["next_weight"]
    out = {"y": y.detach(), "z": z.detach()}
    if case["train"]:
        grads = torch.autograd.grad((y, z), list(t.values()), (s["dy"].double(), s["dz"].double()))
        out.update({f"d{n}": g for n, g in zip(t, grads)})
    return out


def exact(case, seed):
    s, op = prepare(case, seed), case["op"]
    if op == "scan":
        return _exact_scan(case, s)
    if op == "tick":
        keep = torch.sigmoid(s["gate"].double())
        new = keep * s["state"].double() + (1 - keep) * s["x"].double()
        return {"h": new, "state": new}
    if op == "residual":
        return _exact_residual(case, s)
    h, kv, d = case["heads"], case["kv_heads"], case["dim"]
    group, scale, window, sinks = h // kv, s["scale"], case["window"], case["sinks"]
    if op == "paged":
        kp, vp, page = s["k_pages"].clone(), s["v_pages"].clone(), case["page"]
        table = s["pages"].tolist()
        lengths = _histories(case)
        for w, n in enumerate(lengths):
            kp[table[w][(n - 1) // page], (n - 1) % page], vp[table[w][(n - 1) // page], (n - 1) % page] = s["k"][w], s["v"][w]
        out = torch.zeros(case["worlds"], h, d, dtype=torch.float64, device="cuda")
        for w, n in enumerate(lengths):
            keys = torch.arange(n, device="cuda")
            if window:
                keys = keys[(keys >= n - window) | (keys < sinks)]
            at, off = s["pages"][w].long()[keys // page], keys % page
            q = s["q"][w].double().view(kv, group, d)
            k, v = (x[at, off].double().transpose(0, 1).contiguous() for x in (kp, vp))
            out[w] = torch.bmm(_softmax64(torch.bmm(q, k.transpose(1, 2).contiguous()) * scale), v).view(h, d)
        return {"out": out, "k_pages": kp.double(), "v_pages": vp.double()}
    result = {name: torch.zeros(s[of].shape, dtype=torch.float64, device="cuda") for name, of in
              (("out", "q"), ("dq", "q"), ("dk", "k"), ("dv", "v"))}
    at_q = at_k = 0
    for nq, nk in zip(*_lengths(case)):
        tq, tk = slice(at_q, at_q + nq), slice(at_k, at_k + nk)
        at_q, at_k = at_q + nq, at_k + nk
        near = torch.ones(nq, nk, dtype=torch.bool, device="cuda").tril(nk - nq)
        mask = near & ~near.tril(nk - nq - window)
        mask[:, :sinks] = near[:, :sinks]
        for j in range(kv):
            hs = slice(j * group, (j + 1) * group)
            q = s["q"].detach()[tq, hs].double().transpose(0, 1).contiguous()
            k, v = (s[x].detach()[tk, j].double() for x in ("k", "v"))
            p = _softmax64((torch.matmul(q, k.t().contiguous()) * scale).masked_fill(~mask, float("-inf")))
            o = torch.matmul(p, v)
            result["out"][tq, hs] = o.transpose(0, 1)
            if case["train"]:
                do = s["dout"][tq, hs].double().transpose(0, 1).contiguous()
                result["dv"][tk, j] = torch.einsum("gqk,gqd->kd", p, do)
                ds = p * (torch.matmul(do, v.t().contiguous()) - (do * o).sum(2, keepdim=True))
                result["dq"][tq, hs] = torch.matmul(ds, k).transpose(0, 1) * scale
                result["dk"][tk, j] = torch.einsum("gqk,gqd->kd", ds, q) * scale
    return result if case["train"] else {"out": result["out"]}
