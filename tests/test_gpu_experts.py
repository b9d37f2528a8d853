"""Routing and the experts' products, against their definitions in 64 bits."""
import numpy as np
import pytest

from tests.test_gpu_linear16 import ACTS, ROUND, STEP, _types, act64, check

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------------------- routing

def route64(l, k, score, bias, groups, kept, group_top, renorm, scale, mask):
    """Token by token, by Python's sorting (stable, so ties keep the lowest index first)."""
    t, e = l.shape
    ids, wts = np.full((t, k), -1, np.int64), np.zeros((t, k))
    per = e // groups
    for r in range(t):
        if mask is not None and not mask[r]:
            continue
        x = l[r]
        live = x > -np.inf  # False for NaN
        if not live.any():
            continue
        if score == "softmax":
            top = x[live].max()
            s = np.array([0.0 if not ok else 1.0 if v == top else np.exp(v - top) for v, ok in zip(x, live)])
            s /= s.sum()
        else:
            s = np.where(live, 1.0 / (1.0 + np.exp(-np.where(live, x, 0.0))), 0.0)
        c = s if bias is None else s + bias
        can = [i for i in range(e) if live[i] and c[i] > -np.inf]
        if groups > 1:
            def rank(q):
                v = sorted((c[i] for i in can if i // per == q), reverse=True)[:group_top]
                return sum(v) if v else -np.inf
            stay = sorted(range(groups), key=lambda q: -rank(q))[:kept]
            can = [i for i in can if i // per in stay]
        chosen = sorted(can, key=lambda i: -c[i])[:k]
        total = sum(s[i] for i in chosen)
        for j, i in enumerate(chosen):
            ids[r, j] = i
            wts[r, j] = scale * ((s[i] / total if total > 0 else 0.0) if renorm else s[i])
    return ids, wts


def run_route(cuda, logits, k, score="softmax", bias=None, groups=1, kept=1, group_top=1, renorm=True, scale=1.0,
              mask=None):
    import torch

    t = logits.shape[0]
    ids = torch.full((t, k), 77, dtype=torch.int32, device="cuda")
    wts = torch.full((t, k), 7.0, dtype=torch.float32, device="cuda")
    b = None if bias is None else torch.tensor(bias, dtype=torch.float32, device="cuda")
    m = None if mask is None else torch.tensor(mask, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    cuda.route_experts_dev(logits, k, ids, wts, score=score, bias=b, groups=groups, groups_kept=kept,
                           group_top=group_top, renormalise=renorm, scale=scale, mask=m)
    cuda.sync()
    ref_ids, ref_w = route64(logits.double().cpu().numpy(), k, score, bias, groups, kept, group_top, renorm, scale,
                             mask)
    assert np.array_equal(ids.cpu().numpy(), ref_ids)
    # f32: exp (2 ulp), the sum of up to 1024 terms in a tree, two divisions, the scale: under 32 roundings
    np.testing.assert_allclose(wts.cpu().numpy(), ref_w, rtol=32 * 2.0**-24, atol=1e-37)


def grid_logits(t, e, seed, ty="f32"):
    """Multiples of 1/8 in [-4, 4]: exact in every type, with many true ties and no near ones."""
    import torch

    g = torch.Generator().manual_seed(seed)
    return (torch.randint(-32, 33, (t, e), generator=g).float() / 8).to(_types()[ty]).cuda()


@pytest.mark.parametrize("ty", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("t,e,k", [(1, 1, 1), (1, 128, 8), (5, 7, 7), (33, 31, 4), (33, 32, 32), (9, 33, 3), (64, 60, 4),
                                   (17, 127, 8), (50, 256, 8), (7, 300, 6), (6, 513, 10), (5, 1024, 32)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_route_sizes_and_ties(cuda, t, e, k, score, ty):
    run_route(cuda, grid_logits(t, e, t + e + k, ty), k, score, renorm=e % 2 == 0, scale=1.0 if e % 3 else 2.5)


@pytest.mark.parametrize("e,groups,kept,top,k", [(16, 4, 2, 1, 4), (16, 4, 2, 2, 8), (256, 8, 4, 2, 8), (60, 5, 1, 2, 6),
                                                 (64, 32, 7, 2, 10), (32, 32, 5, 2, 5), (96, 2, 2, 1, 9), (9, 3, 2, 1, 6)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_route_groups(cuda, e, groups, kept, top, k, score):
    rng = np.random.default_rng(e)
    bias = (rng.integers(-8, 9, e) / 4).astype(np.float32) if score == "sigmoid" else None
    run_route(cuda, grid_logits(40, e, e + groups), k, score, bias, groups, kept, top, True, 2.5)


@pytest.mark.parametrize("ty", ["f32", "bf16"])
@pytest.mark.parametrize("e,k,groups,kept,top", [(1, 1, 1, 1, 1), (7, 4, 1, 1, 1), (31, 8, 1, 1, 1), (32, 5, 1, 1, 1),
                                                 (60, 4, 1, 1, 1), (128, 8, 1, 1, 1), (300, 6, 1, 1, 1),
                                                 (1024, 8, 1, 1, 1), (256, 8, 8, 4, 2), (64, 3, 32, 7, 2),
                                                 (60, 8, 5, 2, 1), (765, 8, 17, 3, 2), (1020, 7, 17, 5, 2),
                                                 (200, 8, 2, 1, 1), (12, 4, 4, 1, 2)])
def test_route_many_tokens(cuda, e, k, groups, kept, top, ty):
    """Enough tokens for the kernel whose warps take several: every lane layout, with ties, masks and empty rows."""
    k = min(k, kept * (e // groups))
    l = grid_logits(601, e, e + groups, ty)
    l[5] = -np.inf
    l[6, e // 2:] = float("nan")
    l[600, : e // 3] = -np.inf
    mask = np.ones(601, np.uint8)
    mask[[3, 77, 599]] = 0
    rng = np.random.default_rng(e)
    for score, bias in (("softmax", None), ("sigmoid", (rng.integers(-8, 9, e) / 4).astype(np.float32))):
        run_route(cuda, l, k, score, bias, groups, kept, top, e % 2 == 0, 2.5, mask)


@pytest.mark.parametrize("t", [1, 591, 592, 700])
def test_route_strided_many_tokens(cuda, t):
    run_route(cuda, grid_logits(t, 80, 9, "bf16")[:, 5:75], 6)
    run_route(cuda, grid_logits(t, 80, 9, "f32")[:, 4:76], 3, groups=2, kept=1)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups,kept", [(1, 1), (4, 2)])
def test_route_masked_experts_and_tokens(cuda, score, groups, kept):
    """-inf and NaN logits, rows with fewer experts left than choices, none at all, masked tokens, lowest values."""
    import torch

    l = grid_logits(12, 24, 3)
    l[0, 3:] = -np.inf           # three experts left
    l[1] = -np.inf               # none
    l[2, ::2] = float("nan")
    l[3] = float("nan")
    l[4] = torch.finfo(torch.float32).min  # the type's lowest value is a logit like others
    l[5, 5] = float("inf")
    l[6, 1:] = torch.finfo(torch.float32).min
    l[7, :23] = -np.inf
    mask = [1] * 9 + [0, 1, 0]
    bias = None
    if score == "sigmoid":
        bias = np.zeros(24, np.float32)
        bias[2], bias[7], bias[11] = -np.inf, np.nan, 2.0
    run_route(cuda, l, 5, score, bias, groups, kept, 2 if groups > 1 else 1, True, 1.0, mask)


@pytest.mark.parametrize("e,k,groups,kept", [(64, 8, 1, 1), (256, 8, 1, 1), (256, 8, 8, 4), (1000, 32, 1, 1),
                                             (1024, 32, 4, 2), (96, 20, 2, 1)])
def test_route_best_experts_side_by_side(cuda, e, k, groups, kept):
    """The chosen experts lie next to one another, falling, rising, all equal, or tied in runs, anywhere in the row; and
    several biases of +inf."""
    import torch

    l = torch.full((40, e), -3.0)
    for t in range(40):
        at = (t * 37) % (e - k + 1)
        run = [torch.arange(k).flip(0), torch.arange(k), torch.zeros(k), torch.arange(k) // 4][t % 4].float()
        l[t, at:at + k] = run / 8
    l = l.cuda()
    run_route(cuda, l, k, groups=groups, kept=kept)
    bias = np.zeros(e, np.float32)
    bias[5:5 + 6] = np.inf
    bias[e - 2:] = np.inf
    run_route(cuda, l, k, "sigmoid", bias, groups, kept, 2)


def test_route_strided_rows_and_no_tokens(cuda):
    import torch

    wide = grid_logits(20, 50, 9, "bf16")
    run_route(cuda, wide[:, 3:43], 6)
    e = torch.empty(0, 4, dtype=torch.float32, device="cuda")
    cuda.route_experts_dev(e, 2, torch.empty(0, 2, dtype=torch.int32, device="cuda"),
                           torch.empty(0, 2, device="cuda"))
    cuda.sync()


def test_route_refusals(cuda):
    import torch

    from tpt_infer_b200 import OpError

    l = torch.zeros(3, 8, device="cuda")
    ids, w = torch.zeros(3, 2, dtype=torch.int32, device="cuda"), torch.zeros(3, 2, device="cuda")

    def refused(kind, *a, **kw):
        with pytest.raises(OpError) as e:
            cuda.route_experts_dev(*a, **kw)
        assert e.value.kind == kind

    refused("ShapeMismatch", l, 3, ids, w)
    refused("Unsupported", l, 2, ids.long(), w)
    refused("Unsupported", l.double(), 2, ids, w)
    refused("Unsupported", l, 2, ids, w, bias=torch.zeros(8, device="cuda", dtype=torch.float64))
    refused("ShapeMismatch", l, 2, ids, w, bias=torch.zeros(7, device="cuda"))
    refused("ShapeMismatch", l, 2, ids, w, mask=torch.zeros(2, device="cuda", dtype=torch.uint8))
    refused("Invalid", l, 2, ids, w, score="tanh")
    refused("Invalid", l, 2, ids, w, groups=3)
    refused("Invalid", l, 2, ids, w, groups=2, groups_kept=3)
    refused("Invalid", l, 2, ids, w, groups=8, groups_kept=1)
    refused("Invalid", l, 2, ids, w, groups=2, group_top=3)
    refused("Invalid", l[:, :1].contiguous(), 2, ids, w)
    refused("Unsupported", torch.zeros(3, 1025, device="cuda"), 2, ids, w)
    refused("Unsupported", torch.zeros(3, 64, device="cuda"), 33, torch.zeros(3, 33, dtype=torch.int32, device="cuda"),
            torch.zeros(3, 33, device="cuda"))
    cuda.sync()


# ---------------------------------------------------------------------------- the experts' products

def want_experts(x, ids, wts, w_in, w_out, act, gated, residual, t):
    """(y, bound) in 64 bits. h's error: the sums' ((k + 2) 2^-23 of the terms' magnitudes) through the activation
    (slope at most 1.13, own error 4e-6 (1 + |a|)) and the product, and its rounding to the type; it reaches y through
    |w_out|. Then the second sums, the sum over the choices, the residual and the last rounding."""
    import torch

    xd = x.double()
    d, f = w_out.shape[1], w_out.shape[2]
    y, err, mag = torch.zeros_like(xd), torch.zeros_like(xd), torch.zeros_like(xd)
    for e in range(w_out.shape[0]):
        tok, j = (ids == e).nonzero(as_tuple=True)
        if not tok.numel():
            continue
        wi, wo, xe = w_in[e].double(), w_out[e].double(), xd[tok]
        a = xe @ wi.t()
        ea = (d + 2) * 2.0**-23 * (xe.abs() @ wi.abs().t())
        h = act64(a[:, :f], act)
        eh = 1.13 * ea[:, :f] + (4e-6 * (1 + h.abs()) if act in ("gelu", "silu") else 0)
        if gated:
            u, eu = a[:, f:], ea[:, f:]
            eh = eh * (u.abs() + eu) + h.abs() * eu
            h = h * u
        eh = eh + 1.01 * ROUND[t] * (h.abs() + eh) + STEP[t]
        g = wts[tok, j].double()[:, None]
        o = h @ wo.t()
        big = (h.abs() + eh) @ wo.abs().t()
        y.index_add_(0, tok, g * o)
        err.index_add_(0, tok, g.abs() * (eh @ wo.abs().t() + (f + 2) * 2.0**-23 * big))
        mag.index_add_(0, tok, g.abs() * (o.abs() + big * 2.0**-9))
    err = err + (ids.shape[1] + 1) * 2.0**-23 * mag
    if residual is not None:
        r = residual.double()
        err = err + 2.0**-23 * (y.abs() + r.abs())
        y = y + r
    return y, err + 1.01 * ROUND[t] * (y.abs() + err) + STEP[t]


def expert_inputs(t, e, k, d, f, ty, gated, seed=0, skew=0.5):
    import torch

    dt = _types()[ty]
    g = torch.Generator(device="cuda").manual_seed(seed * 104729 + t * 13 + e * 7 + d + f)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    top = torch.topk(1.5 * r(t, e) + skew * r(1, e), k, 1)
    return (r(t, d).to(dt), top.indices.int().contiguous(), torch.softmax(top.values, 1).contiguous(),
            (r(e, (2 if gated else 1) * f, d) * d**-0.5).to(dt), (r(e, d, f) * f**-0.5).to(dt))


def run_experts(cuda, x, ids, wts, w_in, w_out, act, gated, residual, ty):
    import torch

    y = torch.full_like(x, float("nan"))
    torch.cuda.synchronize()
    cuda.experts_mlp_dev(x, ids, wts, w_in, w_out, ACTS[act], gated, residual, y)
    cuda.sync()
    check(y, *want_experts(x, ids, wts, w_in, w_out, act, gated, residual, ty))
    return y


EXPERT_SIZES = [(1, 1, 1, 8, 8), (1, 128, 8, 256, 96), (3, 4, 2, 64, 40), (2, 3, 1, 17, 5), (7, 5, 3, 72, 33),
                (33, 16, 4, 264, 136), (40, 8, 8, 100, 64), (64, 128, 8, 512, 96), (150, 12, 2, 1000, 104),
                (300, 3, 2, 520, 260), (400, 8, 1, 129, 77), (1000, 4, 2, 384, 256), (2000, 64, 6, 128, 72),
                (1, 8, 2, 4096, 512), (600, 2, 2, 776, 1032)]


@pytest.mark.parametrize("ty", ["bf16", "f16"])
@pytest.mark.parametrize("gated", [True, False])
@pytest.mark.parametrize("t,e,k,d,f", EXPERT_SIZES)
def test_experts_sizes(cuda, t, e, k, d, f, gated, ty):
    import torch

    i = EXPERT_SIZES.index((t, e, k, d, f))
    x, ids, wts, w_in, w_out = expert_inputs(t, e, k, d, f, ty, gated)
    if i % 3 == 2:
        ids[torch.rand(t, device="cuda") < 0.2] = -1
    act = ["silu", "gelu", "relu", "none"][i % 4]
    run_experts(cuda, x, ids, wts, w_in, w_out, act, gated, torch.randn_like(x) if i % 2 else None, ty)


@pytest.mark.parametrize("t,d,f", [(9, 136, 72), (700, 264, 136)])
def test_experts_one_expert_takes_all_and_repeated_choices(cuda, t, d, f):
    x, ids, wts, w_in, w_out = expert_inputs(t, 6, 3, d, f, "bf16", True)
    ids[:] = 4
    ids[1, 1] = 2
    ids[2, 0], ids[2, 2] = -1, -5
    run_experts(cuda, x, ids, wts, w_in, w_out, "silu", True, None, "bf16")


def test_experts_no_token_chooses(cuda):
    import torch

    x, ids, wts, w_in, w_out = expert_inputs(20, 4, 2, 64, 32, "bf16", True)
    ids[:] = -1
    y = run_experts(cuda, x, ids, wts, w_in, w_out, "silu", True, None, "bf16")
    assert (y == 0).all()
    r = torch.randn_like(x)
    assert torch.equal(run_experts(cuda, x, ids, wts, w_in, w_out, "silu", True, r, "bf16"), r)
    cuda.experts_mlp_dev(x[:0], ids[:0], wts[:0], w_in, w_out, 3, True, None, x[:0])
    cuda.sync()


@pytest.mark.parametrize("t,d,f,pad", [(30, 72, 40, 8), (30, 72, 40, 3), (300, 136, 64, 24)])
def test_experts_strided_rows_and_residual_in_place(cuda, t, d, f, pad):
    import torch

    x, ids, wts, w_in, w_out = expert_inputs(t, 5, 2, d, f, "f16", True)
    buf = torch.full((t, d + pad), 3.0, dtype=torch.float16, device="cuda")
    xs = buf[:, :d]
    xs.copy_(x)
    out = torch.full((t, d + pad), 5.0, dtype=torch.float16, device="cuda")
    r = torch.randn_like(x)
    out[:, :d] = r
    torch.cuda.synchronize()
    cuda.experts_mlp_dev(xs, ids, wts, w_in, w_out, 3, True, out[:, :d], out[:, :d])
    cuda.sync()
    check(out[:, :d], *want_experts(x, ids, wts, w_in, w_out, "silu", True, r, "f16"))
    assert (out[:, d:] == 5).all() and (buf[:, d:] == 3).all()


@pytest.mark.parametrize("t", [20, 600])
def test_experts_bad_tokens_stay_apart(cuda, t):
    """Infinities and NaN in one token, in an unused expert, and in a token that no expert takes."""
    import torch

    x, ids, wts, w_in, w_out = expert_inputs(t, 6, 2, 264, 136, "bf16", True)
    ids[ids == 5] = 4
    w_in[5] = float("nan")
    w_out[5] = float("inf")
    x[3] = float("nan")
    x[7, 5] = float("inf")
    ids[7] = -1
    wts[7] = float("nan")
    y = torch.empty_like(x)
    torch.cuda.synchronize()
    cuda.experts_mlp_dev(x, ids, wts, w_in, w_out, 3, True, None, y)
    cuda.sync()
    assert torch.isnan(y[3]).all() and (y[7] == 0).all()
    keep = torch.ones(t, dtype=torch.bool, device="cuda")
    keep[3] = keep[7] = False
    check(y[keep], *want_experts(x[keep], ids[keep], wts[keep], w_in, w_out, "silu", True, None, "bf16"))


@pytest.mark.parametrize("t", [3, 60, 700])
@pytest.mark.parametrize("bad", [float("inf"), float("nan"), 3e38])
def test_experts_bad_weights_stay_in_their_features(cuda, bad, t):
    """An infinity, a NaN or a product at the end of f32's range in one output feature of one expert, with products of
    very different size beside it: every other feature is right, for all tokens."""
    import torch

    x, ids, wts, w_in, w_out = expert_inputs(t, 4, 2, 200, 72, "bf16", True)
    w_out[1, 70, 3] = bad
    w_out[2, 40:60] *= 1e-20
    w_out[3] = 0
    y = torch.empty_like(x)
    torch.cuda.synchronize()
    cuda.experts_mlp_dev(x, ids, wts, w_in, w_out, 3, True, None, y)
    cuda.sync()
    clean = w_out.clone()
    clean[1, 70] = 0
    ref, bound = want_experts(x, ids, wts, w_in, clean, "silu", True, None, "bf16")
    hit = (ids == 1).any(1)
    keep = torch.ones(200, dtype=torch.bool, device="cuda")
    keep[70] = False
    check(y[:, keep], ref[:, keep], bound[:, keep])
    check(y[~hit], ref[~hit], bound[~hit])
    if bad != 3e38:
        assert not torch.isfinite(y[hit, 70]).any()


@pytest.mark.parametrize("ty", ["bf16", "f16"])
@pytest.mark.parametrize("t", [1, 4, 12, 60])
def test_experts_infinite_weight_gives_infinity(cuda, t, ty):
    """An infinite weight of one output makes it +inf or -inf, as the hidden value's sign says, not NaN: also where
    the hidden values are kept in two parts, whose signs differ."""
    import torch

    x, ids, wts, w_in, w_out = expert_inputs(t, 3, 2, 200, 72, ty, True)
    ids[:, 1] = -1  # one expert a token
    y = torch.empty_like(x)
    torch.cuda.synchronize()
    for k in range(72):  # every hidden value in turn, so that both signs of both parts come up
        w_out[:, 70, :] = 0
        w_out[:, 70, k] = float("inf")
        torch.cuda.synchronize()
        cuda.experts_mlp_dev(x, ids, wts, w_in, w_out, 3, True, None, y)
        cuda.sync()
        wi = w_in.double()[ids[:, 0].long()]
        gate, up = (wi[:, k] * x.double()).sum(1), (wi[:, 72 + k] * x.double()).sum(1)
        h = act64(gate, "silu") * up
        sure = h.abs() > 1e-3  # the products' errors are under 1e-4, and f16 holds it
        assert torch.equal(y[sure, 70].double(), h[sure].sign() * float("inf"))


def test_experts_many_tokens_in_chunks(cuda):
    """More intermediate results than the workspace takes at once."""
    x, ids, wts, w_in, w_out = expert_inputs(17000, 8, 8, 4096, 64, "bf16", True)
    run_experts(cuda, x, ids, wts, w_in, w_out, "silu", True, None, "bf16")


@pytest.mark.parametrize("t,e,k,d,f", [(1, 64, 8, 512, 136), (50, 16, 4, 264, 136), (900, 8, 2, 264, 136)])
def test_experts_repeat_bit_for_bit_and_in_a_graph(cuda, t, e, k, d, f):
    import torch

    x, ids, wts, w_in, w_out = expert_inputs(t, e, k, d, f, "bf16", True)
    first = run_experts(cuda, x, ids, wts, w_in, w_out, "silu", True, None, "bf16")
    y = torch.empty_like(x)
    torch.cuda.synchronize()
    g = cuda.capture(lambda: cuda.experts_mlp_dev(x, ids, wts, w_in, w_out, 3, True, None, y))
    for _ in range(3):
        y.fill_(float("nan"))
        torch.cuda.synchronize()
        g.launch()
        cuda.sync()
        assert torch.equal(y, first)
    g.close()


def test_experts_follow_new_choices_on_the_same_buffers(cuda):
    """Nothing of a call is kept for the next: other tokens and other choices in the same memory."""
    a = expert_inputs(70, 16, 4, 264, 136, "bf16", True, seed=1)
    b = expert_inputs(70, 16, 4, 264, 136, "bf16", True, seed=2)
    run_experts(cuda, *a, "silu", True, None, "bf16")
    for dst, src in zip(a, b):
        dst.copy_(src)
    run_experts(cuda, *a, "silu", True, None, "bf16")


def test_experts_refusals(cuda):
    import torch

    from tpt_infer_b200 import OpError

    x, ids, wts, w_in, w_out = expert_inputs(6, 4, 2, 32, 16, "bf16", True)
    y = torch.empty_like(x)

    def refused(kind, *a):
        with pytest.raises(OpError) as e:
            cuda.experts_mlp_dev(*a)
        assert e.value.kind == kind

    refused("ShapeMismatch", x, ids, wts, w_in, w_out, 3, False, None, y)
    refused("ShapeMismatch", x[:, :30], ids, wts, w_in, w_out, 3, True, None, y)
    refused("ShapeMismatch", x, ids[:5], wts, w_in, w_out, 3, True, None, y)
    refused("ShapeMismatch", x, ids, wts, w_in[:3], w_out, 3, True, None, y)
    refused("ShapeMismatch", x, ids, wts, w_in, w_out, 3, True, x[:5], y)
    refused("ShapeMismatch", x, ids, wts, w_in.transpose(1, 2).contiguous().transpose(1, 2), w_out, 3, True, None, y)
    refused("Unsupported", x, ids.long(), wts, w_in, w_out, 3, True, None, y)
    refused("Unsupported", x, ids, wts.bfloat16(), w_in, w_out, 3, True, None, y)
    refused("Unsupported", x.half(), ids, wts, w_in, w_out, 3, True, None, y)
    refused("Unsupported", *(v.float() if v.dtype == torch.bfloat16 else v for v in (x, ids, wts, w_in, w_out)), 3,
            True, None, y.float())
    refused("Invalid", x, ids, wts, w_in, w_out, 4, True, None, y)
    refused("Invalid", x.cpu(), ids, wts, w_in, w_out, 3, True, None, y)
    cuda.sync()


def test_experts_id_past_the_last_expert_is_reported(cuda):
    import torch

    from tpt_infer_b200 import OpError

    x, ids, wts, w_in, w_out = expert_inputs(6, 4, 2, 32, 16, "bf16", True)
    ids[2, 1] = 4
    y = torch.empty_like(x)
    torch.cuda.synchronize()
    cuda.experts_mlp_dev(x, ids, wts, w_in, w_out, 3, True, None, y)
    with pytest.raises(OpError) as e:
        cuda.sync()
    assert e.value.code == 9  # TPT_DEVICE_CHECK
    ids[2, 1] = -1
    check(y, *want_experts(x, ids, wts, w_in, w_out, "silu", True, None, "bf16"))
    run_experts(cuda, x, ids, wts, w_in, w_out, "silu", True, None, "bf16")


@pytest.mark.parametrize("t", [1, 3, 4, 40])
@pytest.mark.parametrize("d,f", [(1, 5), (1, 203), (1003, 1)])
def test_experts_what_lies_behind_a_single_row_stays_out(cuda, t, d, f):
    """One expert of one output or one hidden value: the weight is a single row, with NaN right behind it."""
    import torch

    x, ids, wts, w_in, w_out = expert_inputs(t, 1, 1, d, f, "bf16", False)

    def alone(w):
        buf = torch.full((w.numel() + 64,), float("nan"), dtype=w.dtype, device="cuda")
        v = buf[: w.numel()].view(w.shape)
        v.copy_(w)
        return v

    run_experts(cuda, x, ids, wts, alone(w_in), alone(w_out), "relu", False, None, "bf16")


@pytest.mark.parametrize("t,e,k,d,f", [(600, 2, 2, 776, 1032), (60, 4, 4, 2048, 264), (40, 16, 2, 1024, 520)])
def test_experts_wait_limit_reports_a_timeout_and_the_context_recovers(cuda, t, e, k, d, f):
    """Tiles of 256, 32 and 16 tokens under a wait limit of 100 cycles: a timeout, then right again."""
    import torch

    from tpt_infer_b200 import OpError
    from tpt_infer_b200._capi import lib

    x, ids, wts, w_in, w_out = expert_inputs(t, e, k, d, f, "bf16", True)
    y = torch.empty_like(x)
    flush = torch.empty(64 << 20, device="cuda")  # the operands' loads come from memory
    flush.zero_()
    torch.cuda.synchronize()
    try:
        assert lib.tpt_cuda_ctx_set_wait_limit(cuda.ctx, 100) == 0
        cuda.experts_mlp_dev(x, ids, wts, w_in, w_out, 3, True, None, y)
        with pytest.raises(OpError) as err:
            cuda.sync()
        assert err.value.code == 7  # TPT_TIMEOUT
    finally:
        assert lib.tpt_cuda_ctx_set_wait_limit(cuda.ctx, 0) == 0
    for _ in range(2):
        run_experts(cuda, x, ids, wts, w_in, w_out, "silu", True, None, "bf16")


@pytest.mark.parametrize("gated", [True, False])
@pytest.mark.parametrize("t,k,d,f", [(1, 3, 136, 72), (2, 8, 264, 40), (3, 3, 51, 33), (4, 8, 136, 72)])
def test_experts_few_tokens_repeated_choices(cuda, t, k, d, f, gated):
    """A token that names an expert two or more times takes it with each of its weights, beside tokens that name it
    once, that share all their experts, or that name none."""
    import torch

    for seed in range(6):
        x, ids, wts, w_in, w_out = expert_inputs(t, 12, k, d, f, "bf16", gated, seed=seed)
        g = torch.Generator(device="cuda").manual_seed(seed)
        ids.copy_(torch.randint(-1, [1, 2, 3, 12, 12, 12][seed], ids.shape, generator=g, device="cuda"))
        if seed == 4:
            ids[:] = 7
        if seed == 5:
            ids[t - 1] = -1
        wts.copy_(torch.randn(wts.shape, generator=g, device="cuda"))  # of either sign
        run_experts(cuda, x, ids, wts, w_in, w_out, "silu", gated, torch.randn_like(x) if seed % 2 else None, "bf16")


@pytest.mark.parametrize("t", [1, 4])
@pytest.mark.parametrize("bad", [6, 4096, 2**31 - 1])
def test_experts_few_tokens_id_past_the_last_expert_is_reported(cuda, t, bad):
    import torch

    from tpt_infer_b200 import OpError

    for d, f in ((32, 16), (33, 17)):  # read in place, and copied first
        x, ids, wts, w_in, w_out = expert_inputs(t, 6, 3, d, f, "bf16", True)
        ids[t - 1, 1] = bad
        y = torch.empty_like(x)
        torch.cuda.synchronize()
        cuda.experts_mlp_dev(x, ids, wts, w_in, w_out, 3, True, None, y)
        with pytest.raises(OpError) as e:
            cuda.sync()
        assert e.value.code == 9  # TPT_DEVICE_CHECK
        ids[t - 1, 1] = -1
        check(y, *want_experts(x, ids, wts, w_in, w_out, "silu", True, None, "bf16"))
        run_experts(cuda, x, ids, wts, w_in, w_out, "silu", True, None, "bf16")


@pytest.mark.parametrize("t", [1, 2, 4, 5])
@pytest.mark.parametrize("d,f,pad", [(72, 40, 8), (72, 40, 3), (136, 64, 24), (75, 33, 5)])
def test_experts_few_tokens_strided_rows(cuda, t, d, f, pad):
    """Strided x and out with the residual in place; NaN between x's rows stays out, what lies between out's stays."""
    import torch

    x, ids, wts, w_in, w_out = expert_inputs(t, 5, 2, d, f, "f16", True)
    xs = torch.full((t, d + pad), float("nan"), dtype=torch.float16, device="cuda")[:, :d]
    xs.copy_(x)
    out = torch.full((t, d + pad), 5.0, dtype=torch.float16, device="cuda")
    r = torch.randn_like(x)
    out[:, :d] = r
    torch.cuda.synchronize()
    cuda.experts_mlp_dev(xs, ids, wts, w_in, w_out, 3, True, out[:, :d], out[:, :d])
    cuda.sync()
    check(out[:, :d], *want_experts(x, ids, wts, w_in, w_out, "silu", True, r, "f16"))
    assert (out[:, d:] == 5).all()


@pytest.mark.parametrize("t", [1, 7, 8, 9, 600])
def test_route_around_a_blocks_tokens(cuda, t):
    """One warp a token and eight tokens a block: one token, a block less one, a full one and one more, many blocks;
    aligned rows, and strided ones off every word."""
    run_route(cuda, grid_logits(t, 256, t, "bf16"), 8, groups=8, kept=4, group_top=2)
    run_route(cuda, grid_logits(t, 80, 9, "bf16")[:, 5:75], 6)
    run_route(cuda, grid_logits(t, 80, 9, "f32")[:, 4:76], 3, groups=2, kept=1)


@pytest.mark.parametrize("ty", ["bf16", "f16"])
@pytest.mark.parametrize("t,e,k,d,f", [(3, 64, 4, 512, 200), (16, 64, 4, 512, 200), (12, 8, 8, 512, 200), (16, 2, 1, 520, 264),
                                       (11, 1, 1, 1000, 77), (16, 8, 8, 136, 72), (5, 4, 4, 12000, 40)])
def test_experts_up_to_16_tokens_keep_the_hidden_values_bits(cuda, t, e, k, d, f, ty):
    """However few experts share them: the error is the last rounding's. The hidden values' second plane leaves 2^-16 of
    each at most (bf16; f16 2^-22, and 2^-24 absolutely), the f32 sums some 2^-20: under 3 % of the rounding's own
    error, which is taken from the rounded 64-bit result. With hidden values of one plane it is 1.2 to 1.4 times that."""
    import torch

    x, ids, wts, w_in, w_out = expert_inputs(t, e, k, d, f, ty, True)
    y = run_experts(cuda, x, ids, wts, w_in, w_out, "silu", True, None, ty)
    ref, _ = want_experts(x, ids, wts, w_in, w_out, "silu", True, None, ty)
    off, least = (y.double() - ref).norm(), (ref.to(y.dtype).double() - ref).norm()
    assert off <= 1.03 * least, float(off / least)


@pytest.mark.parametrize("ty", ["bf16", "f16"])
@pytest.mark.parametrize("t,e,k,d,f", [(17, 2, 1, 256, 64), (17, 8, 3, 256, 65), (40, 16, 8, 1000, 200), (100, 3, 2, 264, 72),
                                       (128, 2, 1, 256, 64), (256, 2, 1, 136, 32)])
def test_experts_of_few_hidden_values_keep_their_bits(cuda, t, e, k, d, f, ty):
    """More than 16 tokens with narrow experts: as for up to 16 tokens, the error is the last rounding's. With hidden
    values of one plane it is 1.41 times that on average, and up to 1.6 times where few of them carry the result."""
    import torch

    x, ids, wts, w_in, w_out = expert_inputs(t, e, k, d, f, ty, True)
    y = run_experts(cuda, x, ids, wts, w_in, w_out, "silu", True, None, ty)
    ref, _ = want_experts(x, ids, wts, w_in, w_out, "silu", True, None, ty)
    off, least = (y.double() - ref).norm(), (ref.to(y.dtype).double() - ref).norm()
    assert off <= 1.03 * least, float(off / least)


@pytest.mark.parametrize("d,f", [(1001, 255), (1000, 255), (1001, 256)])
def test_experts_one_token_reserves_room_for_its_experts_alone(cuda, d, f):
    """Rows off 16 bytes (of both weights, of w_out, of w_in): 8 of 512 experts are copied, 13 MB of 786."""
    import torch

    from tpt_infer_b200 import CudaBackend

    x, ids, wts, w_in, w_out = expert_inputs(1, 512, 8, d, f, "bf16", True)
    run_experts(cuda, x, ids, wts, w_in, w_out, "silu", True, None, "bf16")  # the kernels are loaded
    y = torch.empty_like(x)
    torch.cuda.synchronize()
    free = torch.cuda.mem_get_info()[0]
    be = CudaBackend.new(0)
    try:
        be.experts_mlp_dev(x, ids, wts, w_in, w_out, 3, True, None, y)
        be.sync()
        assert free - torch.cuda.mem_get_info()[0] < 64 << 20
        check(y, *want_experts(x, ids, wts, w_in, w_out, "silu", True, None, "bf16"))
    finally:
        be.close()
