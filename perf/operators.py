"""What is measured of the mixture-of-experts operators: cases over the range that serving and encoding meet,
the operators' plain forms in 32 bits, and their definition in 64.

  linear   y = act(x w^T + bias) + residual           x [tokens, inputs], w [outputs, inputs]
  route    scores, balance bias, groups, top-k, weights  logits [tokens, experts]
  experts  y = residual + sum_j weight_j * w_out[e_j] (act(gate_j) * up_j),  (gate_j; up_j) = w_in[e_j] x

`own` selects what run() calls: the plain forms, or the framework's operators.
"""
import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_ACTS = {"none": 0, "relu": 1, "gelu": 2, "silu": 3}
_SIZE = {"bf16": 2, "f16": 2, "f32": 4}


# ---------------------------------------------------------------------------- cases

def _linear(tokens, inputs, outputs, type, act="none", bias=False, residual=False):
    return {"op": "linear", "tokens": tokens, "inputs": inputs, "outputs": outputs, "type": type, "act": act,
            "bias": bias, "residual": residual}


def _route(tokens, experts, top_k, type, score="softmax", bias=False, groups=1, kept=1, group_top=1, scale=1.0,
           masked=False):
    return {"op": "route", "tokens": tokens, "experts": experts, "top_k": top_k, "type": type, "score": score,
            "bias": bias, "groups": groups, "kept": kept, "group_top": group_top, "scale": scale, "masked": masked}


def _experts(tokens, experts, top_k, width, hidden, type, act="silu", gated=True, residual=False, padded=False):
    return {"op": "experts", "tokens": tokens, "experts": experts, "top_k": top_k, "width": width, "hidden": hidden,
            "type": type, "act": act, "gated": gated, "residual": residual, "padded": padded}


def listed():
    return [
        # one decoded token through an output projection that adds its residual: latency and the weights' stream
        {"name": "linear 1 token", **_linear(1, 4096, 4096, "bf16", residual=True)},
        # a decode batch into a wide feed-forward layer
        {"name": "linear 64 tokens", **_linear(64, 4096, 11008, "f16", act="silu", bias=True)},
        # the attention output projection of a 12 x 64 encoder at batch 64, sequence 128
        {"name": "linear encoder", **_linear(8192, 768, 768, "bf16", bias=True, residual=True)},
        # rows whose length is not a multiple of anything: a layer of pruned width, a ragged batch
        {"name": "linear odd", **_linear(1537, 1003, 2051, "f16", act="relu", bias=True, residual=True)},
        # a prefill chunk through a wide feed-forward layer
        {"name": "linear prefill", **_linear(8192, 4096, 11008, "bf16", act="gelu", bias=True)},
        # routing of one decoded token
        {"name": "route 1 token", **_route(1, 128, 8, "bf16")},
        # routing with padding tokens and experts that are switched off, an odd number of experts
        {"name": "route masked", **_route(3001, 60, 4, "f16", masked=True)},
        # a prefill batch with sigmoid scores, the balance bias and node-limited groups
        {"name": "route grouped", **_route(16384, 256, 8, "f32", score="sigmoid", bias=True, groups=8, kept=4,
                                           group_top=2, scale=2.5)},
        # one decoded token through its 8 of 128 experts: the chosen experts' weights' stream
        {"name": "experts 1 token", **_experts(1, 128, 8, 2048, 768, "bf16")},
        # a decode batch that touches nearly every expert with a few tokens each
        {"name": "experts 64 tokens", **_experts(64, 128, 8, 2048, 768, "bf16", residual=True, padded=True)},
        # a prefill batch of many small experts
        {"name": "experts prefill", **_experts(8192, 128, 8, 2048, 768, "bf16", residual=True)},
        # few wide experts
        {"name": "experts wide", **_experts(2048, 8, 2, 4096, 11008, "f16", act="gelu")},
    ]


_MOST_FLOPS = 7.3e11   # the largest listed linear's
_MOST_EXPERT_FLOPS = 6.1e11
_MOST_WEIGHTS = 6.0e8  # the listed experts' weights, in values


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi):
    """A width: three of four a multiple of 64 or 8, the others any number."""
    n = _log(rng, lo, hi)
    kind = rng.random()
    return max(1, n if kind < 0.25 else (n + 7) // 8 * 8 if kind < 0.5 else (n + 63) // 64 * 64)


def draw(rng):
    op = rng.choice(["linear", "linear", "route", "experts", "experts"])
    if op == "linear":
        k, n = _size(rng, 128, 8192), _size(rng, 64, 11008)
        t = min(_log(rng, 1, 8192), max(1, int(_MOST_FLOPS / (2 * k * n))))
        return _linear(t, k, n, rng.choice(["bf16", "f16"]), act=rng.choice(list(_ACTS)),
                       bias=rng.random() < 0.5, residual=rng.random() < 0.5)
    if op == "route":
        groups = rng.choice([1, 1, 2, 4, 8])
        experts = groups * rng.randint(max(2, 8 // groups), max(3, 256 // groups))
        kept = rng.randint((groups + 1) // 2, groups)
        top_k = rng.randint(1, min(8, kept * (experts // groups)))
        score = rng.choice(["softmax", "sigmoid"])
        return _route(_log(rng, 1, 16384), experts, top_k, rng.choice(["bf16", "f16", "f32"]), score=score,
                      bias=score == "sigmoid", groups=groups, kept=kept, group_top=rng.choice([1, 2]),
                      scale=rng.choice([1.0, 2.5]), masked=rng.random() < 0.3)
    experts = rng.randint(2, 160)
    top_k = rng.randint(1, min(8, experts))
    width = _size(rng, 256, 4096)
    most = max(64, int(_MOST_WEIGHTS / (3 * experts * width)))
    hidden = min(_size(rng, 64, 4096), most)
    t = min(_log(rng, 1, 8192), max(1, int(_MOST_EXPERT_FLOPS / (6 * top_k * width * hidden))))
    gated = rng.random() < 0.7
    return _experts(t, experts, top_k, width, hidden, rng.choice(["bf16", "f16"]),
                    act=rng.choice(["silu", "gelu"] if gated else ["relu", "gelu", "silu"]), gated=gated,
                    residual=rng.random() < 0.5, padded=rng.random() < 0.3)


def work(c):
    t, size = c["tokens"], _SIZE[c["type"]]
    if c["op"] == "linear":
        k, n = c["inputs"], c["outputs"]
        values = t * k + n * k + t * n * (2 if c["residual"] else 1) + (n if c["bias"] else 0)
        return {"bytes": values * size, "flops": 2.0 * t * n * k}
    if c["op"] == "route":
        e = c["experts"]
        return {"bytes": t * e * size + t * c["top_k"] * 8 + (e * 4 if c["bias"] else 0) + (t if c["masked"] else 0),
                "flops": 8.0 * t * e}
    e, k, d, f = c["experts"], c["top_k"], c["width"], c["hidden"]
    up = 2 if c["gated"] else 1
    active = e * (1.0 - (1.0 - k / e) ** t)  # the experts that t tokens reach when each is as likely
    return {"bytes": active * (up + 1) * f * d * size + t * d * size * (3 if c["residual"] else 2) + t * k * 8,
            "flops": 2.0 * t * k * (up + 1) * f * d}


# ---------------------------------------------------------------------------- inputs

def _normal(gen, shape, dtype, std=1.0):
    return torch.empty(shape, dtype=dtype, device="cuda").normal_(0.0, std, generator=gen)


def _popular(gen, tokens, experts):
    """Router logits: each token's own preferences on top of the experts' popularity."""
    return _normal(gen, (tokens, experts), torch.float32, 1.5) + _normal(gen, (1, experts), torch.float32, 0.5)


def _gaps_clear(c, logits, bias, mask):
    """For each token, whether no two values that its choice orders are closer than rounding in 32 bits can tell
    apart (equal logits without a bias are a true tie, which goes to the lowest index)."""
    s = logits.double()
    dead = s == -math.inf
    s = torch.softmax(s, 1).nan_to_num(0.0) if c["score"] == "softmax" else torch.sigmoid(s)
    s = (s if bias is None else s + bias.double()).masked_fill(dead, -math.inf)
    tie = bias is None and c["groups"] == 1

    def clear(v, n):
        v = torch.sort(v, 1, descending=True).values[:, : n + 1]
        a, b = v[:, :-1], v[:, 1:]
        near = ((a - b) < 1e-5 * a.abs().clamp_min(1e-30)) & (b > -math.inf)
        return ~(near & ~((a == b) & tie)).any(1)

    ok = torch.ones(s.shape[0], dtype=torch.bool, device=s.device)
    if c["groups"] > 1:
        per = s.view(s.shape[0], c["groups"], -1)
        best = torch.topk(per, min(c["group_top"], per.shape[2]), 2).values
        g = best.masked_fill(best == -math.inf, 0.0).sum(2).masked_fill(best[:, :, 0] == -math.inf, -math.inf)
        ok &= clear(g, c["kept"])
        keep = torch.zeros_like(g, dtype=torch.bool).scatter_(1, torch.topk(g, c["kept"], 1).indices, True)
        s = per.masked_fill(~keep[:, :, None], -math.inf).view_as(s)
    ok &= clear(s, c["top_k"])
    return ok if mask is None else ok | (mask == 0)


def prepare(c, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dt, t = _TYPES[c["type"]], c["tokens"]
    st = {"case": c}
    if c["op"] == "linear":
        k, n = c["inputs"], c["outputs"]
        st["x"] = _normal(gen, (t, k), dt)
        st["w"] = _normal(gen, (n, k), dt, k ** -0.5)
        st["bias"] = _normal(gen, (n,), dt, 0.1) if c["bias"] else None
        st["residual"] = _normal(gen, (t, n), dt) if c["residual"] else None
        st["y"] = torch.empty((t, n), dtype=dt, device="cuda")
    elif c["op"] == "route":
        e = c["experts"]
        st["bias"] = _normal(gen, (e,), torch.float32, 0.05) if c["bias"] else None
        st["mask"] = None
        off = torch.zeros(e, dtype=torch.bool, device="cuda")
        if c["masked"]:  # padding tokens at the batch's end and between, and experts that are switched off
            st["mask"] = (torch.rand(t, generator=gen, device="cuda") < 0.9).to(torch.uint8)
            off = torch.rand(e, generator=gen, device="cuda") < 0.1
        logits = _popular(gen, t, e).to(dt).masked_fill(off, -math.inf)
        for _ in range(16):  # values that rounding would order either way have no right order: drawn again
            ok = _gaps_clear(c, logits, st["bias"], st["mask"])
            if bool(ok.all()):
                break
            again = _popular(gen, t, e).to(dt).masked_fill(off, -math.inf)
            logits = torch.where(ok[:, None], logits, again)
        st["logits"] = logits
        st["ids"] = torch.empty((t, c["top_k"]), dtype=torch.int32, device="cuda")
        st["weights"] = torch.empty((t, c["top_k"]), dtype=torch.float32, device="cuda")
    else:
        e, k, d, f = c["experts"], c["top_k"], c["width"], c["hidden"]
        st["x"] = _normal(gen, (t, d), dt)
        st["w_in"] = _normal(gen, (e, (2 if c["gated"] else 1) * f, d), dt, d ** -0.5)
        st["w_out"] = _normal(gen, (e, d, f), dt, f ** -0.5)
        top = torch.topk(_popular(gen, t, e), k, 1)
        st["ids"], st["weights"] = top.indices.to(torch.int32), torch.softmax(top.values, 1)
        if c["padded"]:  # padding tokens reach no expert
            pad = torch.rand(t, generator=gen, device="cuda") < 0.1
            st["ids"] = st["ids"].masked_fill(pad[:, None], -1)
            st["weights"] = st["weights"].masked_fill(pad[:, None], 0.0)
        st["residual"] = _normal(gen, (t, d), dt) if c["residual"] else None
        st["y"] = torch.empty((t, d), dtype=dt, device="cuda")
    torch.cuda.synchronize()  # a serving program's inputs are there before its own stream reads them
    return st


# ---------------------------------------------------------------------------- plain forms, 32 bits

def _act(v, act):
    if act == "relu":
        return torch.maximum(v, torch.zeros_like(v))
    if act == "gelu":
        return 0.5 * v * (1.0 + torch.tanh(0.7978845608028654 * (v + 0.044715 * v * v * v)))
    if act == "silu":
        return v / (1.0 + torch.exp(-v))
    return v


def _plain_linear(st):
    c = st["case"]
    y = st["x"].float() @ st["w"].float().t()
    if st["bias"] is not None:
        y = y + st["bias"].float()
    y = _act(y, c["act"])
    if st["residual"] is not None:
        y = y + st["residual"].float()
    return {"y": y.to(st["x"].dtype)}


def _plain_route(st):
    c = st["case"]
    l = st["logits"].float()
    live = l > -math.inf
    if c["score"] == "softmax":
        top = l.max(1, keepdim=True).values
        p = torch.where(live, torch.where(l == top, 1.0, torch.exp(l - top)), 0.0)
        total = p.sum(1, keepdim=True)
        s = torch.where(total > 0, p / total, 0.0)
    else:
        s = 1.0 / (1.0 + torch.exp(-l))
    choice = s if st["bias"] is None else s + st["bias"]
    choice = torch.where(live, choice, -math.inf)
    t, e = choice.shape
    if c["groups"] > 1:
        per = choice.view(t, c["groups"], -1)
        best = torch.sort(per, 2, descending=True).values[:, :, : c["group_top"]]
        g = torch.where(best > -math.inf, best, 0.0).sum(2)
        g = torch.where(best[:, :, 0] > -math.inf, g, -math.inf)
        order = torch.sort(g, dim=1, descending=True, stable=True).indices[:, : c["kept"]]
        keep = torch.zeros_like(g, dtype=torch.bool).scatter_(1, order, True)
        choice = torch.where(keep[:, :, None], per, -math.inf).view(t, e)
    top = torch.sort(choice, dim=1, descending=True, stable=True)
    ids, found = top.indices[:, : c["top_k"]], top.values[:, : c["top_k"]] > -math.inf
    if st["mask"] is not None:
        found = found & (st["mask"] != 0)[:, None]
    w = torch.where(found, s.gather(1, ids), 0.0)
    total = w.sum(1, keepdim=True)
    w = torch.where(total > 0, w / total, 0.0) * c["scale"]
    return {"ids": torch.where(found, ids, -1).to(torch.int32), "weights": w}


def _plain_experts(st):
    c = st["case"]
    x, ids, wts = st["x"].float(), st["ids"].long(), st["weights"]
    t, k = ids.shape
    e, f = c["experts"], c["hidden"]
    flat = ids.reshape(-1)
    tok = torch.arange(t * k, device=x.device) // k

    def hidden(a):
        return _act(a[..., :f], c["act"]) * a[..., f:] if c["gated"] else _act(a, c["act"])

    if t * k <= e:  # the chosen experts' weights, gathered
        at = flat.clamp(min=0)
        a = torch.bmm(st["w_in"][at].float(), x[tok][:, :, None])[:, :, 0]
        o = torch.bmm(st["w_out"][at].float(), hidden(a)[:, :, None])[:, :, 0]
    else:  # each expert's tokens, padded to the largest expert's
        bucket = torch.where(flat >= 0, flat, e)
        order = torch.sort(bucket, stable=True).indices
        count = torch.bincount(bucket, minlength=e + 1)[:e]
        first = torch.cumsum(count, 0) - count
        place = torch.arange(max(1, int(count.max())), device=x.device)
        used = place < count[:, None]
        slot = order[(first[:, None] + place).clamp(max=t * k - 1)]
        a = torch.bmm(x[tok[slot]], st["w_in"].float().transpose(1, 2))
        p = torch.bmm(hidden(a), st["w_out"].float().transpose(1, 2))
        o = torch.zeros((t * k, x.shape[1]), device=x.device)
        o[slot[used]] = p[used]
    o = torch.where((flat >= 0)[:, None], o, 0.0).view(t, k, -1)
    y = (wts[:, :, None] * o).sum(1)
    if st["residual"] is not None:
        y = y + st["residual"].float()
    return {"y": y.to(st["x"].dtype)}


# ---------------------------------------------------------------------------- the framework's operators

_backend = None


def _be():
    """The process's backend, on a stream of its own, as a serving program keeps one."""
    global _backend
    if _backend is None:
        from tpt_infer_b200 import CudaBackend

        _backend = CudaBackend.new(0)
    return _backend


def run(st):
    c = st["case"]
    if not own:
        return {"linear": _plain_linear, "route": _plain_route, "experts": _plain_experts}[c["op"]](st)
    be = _be()
    if c["op"] == "linear":
        be.linear_dev(st["x"], st["w"], st["bias"], _ACTS[c["act"]], st["residual"], st["y"])
        return {"y": st["y"]}
    if c["op"] == "route":
        be.route_experts_dev(st["logits"], c["top_k"], st["ids"], st["weights"], score=c["score"], bias=st["bias"],
                             groups=c["groups"], groups_kept=c["kept"], group_top=c["group_top"], renormalise=True,
                             scale=c["scale"], mask=st["mask"])
        return {"ids": st["ids"], "weights": st["weights"]}
    be.experts_mlp_dev(st["x"], st["ids"], st["weights"], st["w_in"], st["w_out"], _ACTS[c["act"]], c["gated"],
                       st["residual"], st["y"])
    return {"y": st["y"]}


# ---------------------------------------------------------------------------- the definition, 64 bits

def _exact_act(v, act):
    if act == "relu":
        return v.clamp(min=0.0)
    if act == "gelu":
        return v * torch.sigmoid(2.0 * math.sqrt(2.0 / math.pi) * (v + 0.044715 * v.pow(3)))
    if act == "silu":
        return v * torch.sigmoid(v)
    return v


def _exact_linear(st, c):
    y = torch.nn.functional.linear(st["x"].double(), st["w"].double(),
                                   None if st["bias"] is None else st["bias"].double())
    y = _exact_act(y, c["act"])
    return {"y": y if st["residual"] is None else y + st["residual"].double()}


def _exact_route(st, c):
    """Expert by expert from the largest down, each token's best remaining one."""
    l = st["logits"].double()
    s = torch.softmax(l, 1).nan_to_num(0.0) if c["score"] == "softmax" else torch.sigmoid(l)
    v = (s if st["bias"] is None else s + st["bias"].double()).masked_fill(l == -math.inf, -math.inf)
    t, e = v.shape
    if c["groups"] > 1:
        per = v.view(t, c["groups"], e // c["groups"]).clone()
        total = torch.zeros((t, c["groups"]), dtype=torch.float64, device=v.device)
        dead = per.amax(2) == -math.inf
        for _ in range(min(c["group_top"], e // c["groups"])):
            m, at = per.max(2)
            total += m.masked_fill(m == -math.inf, 0.0)
            per.scatter_(2, at[:, :, None], -math.inf)
        total.masked_fill_(dead, -math.inf)
        drop = torch.ones_like(dead)
        for _ in range(c["kept"]):
            at = total.argmax(1, keepdim=True)
            drop.scatter_(1, at, False)
            total.scatter_(1, at, -math.inf)
        v = v.masked_fill(drop.repeat_interleave(e // c["groups"], 1), -math.inf)
    v = v.clone()
    w = torch.zeros((t, c["top_k"]), dtype=torch.float64, device=v.device)
    for j in range(c["top_k"]):
        m, at = v.max(1, keepdim=True)
        w[:, j : j + 1] = s.gather(1, at).masked_fill(m == -math.inf, 0.0)
        v.scatter_(1, at, -math.inf)
    if st["mask"] is not None:
        w *= (st["mask"] != 0).double()[:, None]
    total = w.sum(1, keepdim=True)
    return {"ids": None, "weights": c["scale"] * w / total.masked_fill(total == 0.0, 1.0)}


def _exact_experts(st, c):
    x, f = st["x"].double(), c["hidden"]
    y = torch.zeros_like(x) if st["residual"] is None else st["residual"].double().clone()
    for e in range(c["experts"]):
        tok, j = (st["ids"] == e).nonzero(as_tuple=True)
        if tok.numel():
            a = x[tok] @ st["w_in"][e].double().t()
            h = _exact_act(a[:, :f], c["act"]) * a[:, f:] if c["gated"] else _exact_act(a, c["act"])
            y.index_add_(0, tok, st["weights"][tok, j].double()[:, None] * (h @ st["w_out"][e].double().t()))
    return {"y": y}


def exact(c, seed):
    return {"linear": _exact_linear, "route": _exact_route, "experts": _exact_experts}[c["op"]](prepare(c, seed), c)
