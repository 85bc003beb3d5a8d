"""Performance cases of the operators that a policy trained through the control step is built from (the package's
`policy` module), in plain torch and as the package's calls.

A case is one operator (`op`) over a batch of the framework's shapes: thousands of worlds, rollouts of tens of steps,
episodes of up to some minutes of 20 ms steps.

  norm       policy.layer_norm of (rows, width) activations; train: with the gradients of x, weight and bias
  clip       policy.clip_grads_ of a list of gradients into the optimizer's buffers (clip: with the copies; else the
             norm alone, policy.grad_norm)
  attend     policy.attention over packed episodes of different lengths, causal, query heads sharing key/value heads;
             train: with the gradients of q, k and v
  step       policy.attention_step: each world's one new query over its own cached history
"""
import math
import random

import torch

own = False

_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_BYTES = {"f32": 4, "bf16": 2, "f16": 2}
EPS = 1e-5


def _norm(rows, width, dtype, train, pad=0, affine=True, **kw):
    return dict(op="norm", rows=rows, width=width, dtype=dtype, train=train, pad=pad, affine=affine, **kw)


def _clip(layers, hidden, dtype, clip=True, limit=1.0, **kw):
    return dict(op="clip", layers=layers, hidden=hidden, dtype=dtype, clip=clip, limit=limit, **kw)


def _attend(episodes, longest, heads, kv_heads, dim, dtype, train, past=0, **kw):
    return dict(op="attend", episodes=episodes, longest=longest, heads=heads, kv_heads=kv_heads, dim=dim, dtype=dtype,
                train=train, past=past, **kw)


def _step(worlds, capacity, heads, kv_heads, dim, dtype, **kw):
    return dict(op="step", worlds=worlds, capacity=capacity, heads=heads, kv_heads=kv_heads, dim=dim, dtype=dtype, **kw)


def listed():
    return [
        # one robot in the control loop: a hidden layer's norm, where latency is all there is
        _norm(1, 256, "f32", False, name="norm_control"),
        # one update of a policy's hidden layer over the headline batch of worlds
        _norm(4096, 512, "f32", True, name="norm_worlds"),
        # the 99 observations of an odd batch, rows of a wider buffer, in half precision
        _norm(1331, 99, "f16", True, pad=29, name="norm_observations"),
        # a value network's layer over a whole rollout: 16384 worlds x 32 steps
        _norm(524288, 256, "bf16", True, name="norm_rollout"),
        # the gradients of a three-layer policy, which backpropagation through time makes large now and then
        _clip(3, 256, "f32", name="clip_mlp"),
        # the gradients of a history policy of 24 blocks, 302 million weights, matrices in bfloat16 and vectors in float32
        _clip(24, 1024, "mixed", limit=0.5, name="clip_transformer"),
        # rollout segments of at most 32 steps, cut short where a robot fell
        _attend(4096, 32, 8, 2, 64, "bf16", True, name="attend_segments"),
        # whole episodes of at most 20 s
        _attend(256, 1000, 8, 2, 64, "bf16", True, name="attend_episodes"),
        # two long recordings, the largest heads
        _attend(2, 8192, 16, 4, 128, "bf16", True, name="attend_long"),
        # one robot in the control loop, attending to its last seconds
        _step(1, 257, 8, 8, 64, "bf16", name="step_control"),
        # the headline batch of worlds, each with its own history
        _step(4096, 256, 8, 2, 64, "bf16", name="step_worlds"),
        # few worlds with long histories
        _step(4, 131072, 16, 4, 128, "f16", name="step_long"),
    ]


def _spread(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49)))))))


def draw(rng):
    op = rng.choice(["norm", "clip", "attend", "attend", "step"])
    if op == "norm":
        width = _spread(rng, 8, 8192)
        rows = _spread(rng, 1, min(524288, 524288 * 256 // width))
        return _norm(rows, width, rng.choice(["f32", "bf16", "f16"]), rng.choice([True, True, False]),
                     pad=rng.choice([0, 0, rng.randint(1, 64)]) if rows * width <= 1 << 25 else 0,
                     affine=rng.choice([True, True, False]))
    if op == "clip":
        hidden = _spread(rng, 16, 1024)
        return _clip(_spread(rng, 1, 24), hidden, rng.choice(["f32", "bf16", "mixed"] if hidden <= 512 else
                                                             ["bf16", "mixed"]),
                     clip=rng.choice([True, True, False]), limit=rng.choice([0.5, 1.0, 1e9]))
    dim, dtype = rng.choice([64, 64, 128, 40]), rng.choice(["bf16", "bf16", "f16"])
    kv_heads = rng.choice([1, 2, 4])
    heads = kv_heads * rng.choice([1, 2, 3, 4])
    if op == "attend":
        longest = _spread(rng, 1, 4096)
        episodes = _spread(rng, 1, max(1, min(4096, 131072 // longest, (1 << 26) // longest ** 2)))
        return _attend(episodes, longest, heads, kv_heads, dim, dtype, rng.choice([True, True, False]),
                       past=rng.choice([0, 0, _spread(rng, 1, longest)]))
    capacity = _spread(rng, 1, 131072)
    return _step(_spread(rng, 1, max(1, min(4096, (1 << 20) // capacity))), capacity, heads, kv_heads, dim, dtype)


# ---- shapes and values ----------------------------------------------------------------------------------------------

def _gradient_shapes(case):
    """(shape, type) of each gradient: a multilayer perceptron from 99 observations to 29 controls with a norm after
    each hidden layer, or the blocks of a history policy (queries, keys and values in one matrix, two matrices of the
    feed-forward part, two norms)."""
    h, mixed = case["hidden"], case["dtype"] == "mixed"
    mat = "bf16" if mixed else case["dtype"]
    vec = "f32" if mixed else case["dtype"]
    shapes = [((h, 99), mat), ((h,), vec)]
    for _ in range(case["layers"]):
        if mixed:
            shapes += [((3 * h, h), mat), ((h, h), mat), ((4 * h, h), mat), ((h, 4 * h), mat), ((4 * h,), vec)]
        else:
            shapes += [((h, h), mat)]
        shapes += [((h,), vec), ((h,), vec), ((h,), vec)]
    return shapes + [((29, h), mat), ((29,), vec)]


def _lengths(case):
    """(queries, keys) of each episode: most run to the end, the others fall at any time; some have earlier keys
    (`past` at most) before their first query."""
    rng = random.Random(case["episodes"] * 100003 + case["longest"])
    most = case["longest"]
    q = [most if rng.random() < 0.3 else rng.randint(1, most) for _ in range(case["episodes"])]
    q[0] = most
    return q, [n + (rng.randint(0, case["past"]) if case["past"] else 0) for n in q]


def _histories(case):
    """The length of each world's history: anything from none (a world just reset) to the whole cache."""
    rng = random.Random(case["worlds"] * 100003 + case["capacity"])
    n = [rng.randint(0, case["capacity"]) if rng.random() < 0.5 else case["capacity"] for _ in range(case["worlds"])]
    n[0] = case["capacity"]
    return n


def _pairs(case):
    """The (query, key) pairs that the causal mask leaves, over all episodes."""
    return sum(nq * nk - nq * (nq - 1) // 2 for nq, nk in zip(*_lengths(case)))


def work(case):
    if case["op"] == "norm":
        n, b, w = case["rows"] * case["width"], _BYTES[case["dtype"]], 4 * case["width"] if case["affine"] else 0
        if not case["train"]:
            return {"bytes": 2 * n * b + 2 * w, "flops": 8 * n}
        return {"bytes": 4 * n * b + 4 * w, "flops": 20 * n}
    if case["op"] == "clip":
        sizes = [(math.prod(s), _BYTES[t]) for s, t in _gradient_shapes(case)]
        moved = sum(n * b for n, b in sizes)
        n = sum(n for n, _ in sizes)
        return {"bytes": moved + (sum(4 * n for n, _ in sizes) if case["clip"] else 0) + 4,
                "flops": 3 * n if case["clip"] else 2 * n}
    h, kv, d, b = case["heads"], case["kv_heads"], case["dim"], _BYTES[case["dtype"]]
    if case["op"] == "attend":
        nq, nk = (sum(x) for x in _lengths(case))
        flops = 4 * d * h * _pairs(case)  # two products, a multiplication and an addition each
        if not case["train"]:
            return {"bytes": b * d * (2 * nq * h + 2 * nk * kv), "flops": flops}
        # the gradients take five products more; q, k, v, the output's gradient in, the output and three gradients out
        return {"bytes": b * d * (4 * nq * h + 4 * nk * kv), "flops": flops * 7 // 2}
    n = sum(_histories(case))
    return {"bytes": b * d * (2 * n * kv + 2 * case["worlds"] * h), "flops": 4 * d * h * n}


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(g, shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def _starts(lengths):
    return torch.tensor([0] + lengths, dtype=torch.int64).cumsum(0).to(torch.int32).cuda()


def prepare(case, seed):
    g = _generator(seed)
    s = {"case": dict(case)}
    if case["op"] == "norm":
        rows, width, dtype = case["rows"], case["width"], _TYPES[case["dtype"]]
        wide = _normal(g, (rows, width + case["pad"]), dtype, 1.5)
        wide += 0.5
        s["x"] = wide[:, :width].detach().requires_grad_(case["train"])
        if case["affine"]:
            s["weight"] = (1.0 + _normal(g, (width,), scale=0.2)).requires_grad_(case["train"])
            s["bias"] = _normal(g, (width,), scale=0.2).requires_grad_(case["train"])
        if case["train"]:
            s["dy"] = _normal(g, (rows, width), dtype)
        return s
    if case["op"] == "clip":
        shapes = _gradient_shapes(case)
        s["grads"] = [_normal(g, shape, _TYPES[t], 0.05) for shape, t in shapes]
        # the optimizer's float32 gradients, one after another in one flat buffer
        if case["clip"]:
            s["flat"] = torch.empty(sum(math.prod(shape) for shape, _ in shapes), device="cuda")
            s["out"], at = [], 0
            for shape, _ in shapes:
                s["out"].append(s["flat"][at:at + math.prod(shape)].view(shape))
                at += math.prod(shape)
        return s
    h, kv, d, dtype = case["heads"], case["kv_heads"], case["dim"], _TYPES[case["dtype"]]
    s["scale"] = 1.0 / math.sqrt(d)
    if case["op"] == "attend":
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
    s["q"] = _normal(g, (case["worlds"], h, d), dtype)
    s["k"] = _normal(g, (case["worlds"], case["capacity"], kv, d), dtype)
    s["v"] = _normal(g, (case["worlds"], case["capacity"], kv, d), dtype)
    s["lengths"] = torch.tensor(_histories(case), dtype=torch.int32, device="cuda")
    return s


# ---- the plain forms ------------------------------------------------------------------------------------------------

def _plain_norm(s):
    x = s["x"].detach().float()
    mean = x.mean(1, keepdim=True)
    centred = x - mean
    rstd = 1.0 / torch.sqrt((centred * centred).mean(1, keepdim=True) + EPS)
    xhat = centred * rstd
    affine = "weight" in s
    y = xhat * s["weight"].detach() + s["bias"].detach() if affine else xhat
    out = {"y": y.to(s["x"].dtype)}
    if "dy" in s:
        dy = s["dy"].float()
        g = dy * s["weight"].detach() if affine else dy
        dx = rstd * (g - g.mean(1, keepdim=True) - xhat * (g * xhat).mean(1, keepdim=True))
        out["dx"] = dx.to(s["x"].dtype)
        if affine:
            out["dweight"], out["dbias"] = (dy * xhat).sum(0), dy.sum(0)
    return out


def _plain_clip(s):
    squares = torch.stack([g.float().square().sum() for g in s["grads"]])
    norm = torch.sqrt(squares.sum())
    if "flat" not in s:
        return {"norm": norm}
    factor = torch.clamp(s["case"]["limit"] / (norm + 1e-6), max=1.0)
    [o.copy_(g.float() * factor) for o, g in zip(s["out"], s["grads"])]
    return {"norm": norm, "grads": s["flat"]}


def _places(starts, longest):
    """For each episode and each place up to the longest's: the token's index (0 where there is none), and whether there is one."""
    place = torch.arange(longest, device=starts.device)
    lengths = (starts[1:] - starts[:-1]).long()
    there = place < lengths[:, None]
    return torch.where(there, starts[:-1].long()[:, None] + place, 0), there, lengths


def _plain_attend(s):
    q, k, v = (s[n].detach() for n in ("q", "k", "v"))
    heads, kv, d = q.shape[1], k.shape[1], q.shape[2]
    iq, there_q, nq = _places(s["starts_q"], s["longest"][0])
    ik, there_k, nk = _places(s["starts_k"], s["longest"][1])
    # the mask of each episode: query i, of nq, has the keys up to nk - nq + i
    last = torch.arange(s["longest"][0], device=q.device) + (nk - nq)[:, None]
    mask = (torch.arange(s["longest"][1], device=q.device) <= last[:, :, None]) & there_q[:, :, None] & there_k[:, None]
    S, G = len(nq), heads // kv
    spread = lambda x, i: x[i].float().transpose(1, 2)  # noqa: E731   (episode, head, place, d)
    share = lambda x: x.repeat_interleave(G, 1)  # noqa: E731
    join = lambda x: x.view(S, kv, G, -1, d).sum(2)  # noqa: E731
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


def _plain_step(s):
    q, worlds, kv, d = s["q"], s["q"].shape[0], s["k"].shape[2], s["q"].shape[2]
    there = torch.arange(s["k"].shape[1], device=q.device) < s["lengths"][:, None]
    qs = q.float().view(worlds, kv, -1, d)
    ks = s["k"].float().permute(0, 2, 3, 1).contiguous()
    scores = (torch.matmul(qs, ks) * s["scale"]).masked_fill(~there[:, None, None], float("-inf"))
    p = torch.exp(scores - scores.amax(3, keepdim=True).clamp(min=-1e30))
    p = p / p.sum(3, keepdim=True).clamp(min=1e-30)
    vs = s["v"].float().masked_fill(~there[:, :, None, None], 0.0).transpose(1, 2).contiguous()
    return {"out": torch.matmul(p, vs).view_as(q).to(q.dtype)}


# ---- the package's calls --------------------------------------------------------------------------------------------

def _own(s):
    from nablaengine_amd import policy
    op = s["case"]["op"]
    if op == "norm":
        y = policy.layer_norm(s["x"], s.get("weight"), s.get("bias"), eps=EPS)
        if "dy" not in s:
            return {"y": y}
        if "weight" not in s:
            return {"y": y.detach(), "dx": torch.autograd.grad(y, s["x"], s["dy"])[0]}
        dx, dw, db = torch.autograd.grad(y, (s["x"], s["weight"], s["bias"]), s["dy"])
        return {"y": y.detach(), "dx": dx, "dweight": dw, "dbias": db}
    if op == "clip":
        if "flat" not in s:
            return {"norm": policy.grad_norm(s["grads"])}
        return {"norm": policy.clip_grads_(s["grads"], s["case"]["limit"], out=s["out"]), "grads": s["flat"]}
    if op == "attend":
        o = policy.attention(s["q"], s["k"], s["v"], s["starts_q"], s["starts_k"], scale=s["scale"])
        if "dout" not in s:
            return {"out": o}
        dq, dk, dv = torch.autograd.grad(o, (s["q"], s["k"], s["v"]), s["dout"])
        return {"out": o.detach(), "dq": dq, "dk": dk, "dv": dv}
    return {"out": policy.attention_step(s["q"], s["k"], s["v"], s["lengths"], scale=s["scale"])}


def run(state):
    if own:
        return _own(state)
    return {"norm": _plain_norm, "clip": _plain_clip, "attend": _plain_attend, "step": _plain_step}[
        state["case"]["op"]](state)


# ---- the definitions in 64 bits -------------------------------------------------------------------------------------

def _softmax64(scores):
    """exp(s) / sum exp(s) over the last axis; zeros where every score is -inf."""
    top = scores.max(-1, keepdim=True).values
    e = torch.where(torch.isinf(scores), 0.0, (scores - torch.where(torch.isinf(top), 0.0, top)).exp())
    total = e.sum(-1, keepdim=True)
    return e / torch.where(total == 0, 1.0, total)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        x = s["x"].detach().double()
        var, mean = torch.var_mean(x, 1, correction=0, keepdim=True)
        sd = (var + EPS).sqrt()
        xhat = (x - mean) / sd
        w = s["weight"].detach().double() if "weight" in s else torch.ones(x.shape[1], dtype=x.dtype, device=x.device)
        out = {"y": xhat * w + (s["bias"].detach().double() if "bias" in s else 0.0)}
        if case["train"]:
            dy = s["dy"].double()
            n = x.shape[1]
            a = (dy @ w) / n
            c = ((dy * xhat) @ w) / n
            out["dx"] = (dy * w - a[:, None] - xhat * c[:, None]) / sd
            if "weight" in s:
                out["dweight"] = torch.einsum("ij,ij->j", dy, xhat)
                out["dbias"] = torch.ones(len(dy), dtype=dy.dtype, device=dy.device) @ dy
        return out
    if case["op"] == "clip":
        flat = torch.cat([x.double().reshape(-1) for x in s["grads"]])
        norm = torch.linalg.vector_norm(flat)
        if not case["clip"]:
            return {"norm": norm}
        return {"norm": norm, "grads": flat * min(1.0, case["limit"] / (norm.item() + 1e-6))}
    h, kv, d = case["heads"], case["kv_heads"], case["dim"]
    group, scale = h // kv, s["scale"]
    if case["op"] == "step":
        out = torch.zeros(case["worlds"], h, d, dtype=torch.float64, device="cuda")
        if case["worlds"] * kv > 8192:
            return None
        for b, n in enumerate(_histories(case)):
            q = s["q"][b].double().view(kv, group, d)
            k, v = (s[x][b, :n].double().transpose(0, 1).contiguous() for x in ("k", "v"))
            if n:
                out[b] = torch.bmm(_softmax64(torch.bmm(q, k.transpose(1, 2).contiguous()) * scale), v).view(h, d)
        return {"out": out}
    result = {name: torch.zeros(s[of].shape, dtype=torch.float64, device="cuda") for name, of in
              (("out", "q"), ("dq", "q"), ("dk", "k"), ("dv", "v"))}
    at_q = at_k = 0
    for nq, nk in zip(*_lengths(case)):
        tq, tk = slice(at_q, at_q + nq), slice(at_k, at_k + nk)
        at_q, at_k = at_q + nq, at_k + nk
        mask = torch.ones(nq, nk, dtype=torch.bool, device="cuda").tril(nk - nq)
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
