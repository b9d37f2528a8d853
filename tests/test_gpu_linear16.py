"""The 16-bit matrix product with its epilogue, against the formula in 64 bits.

Bounds. The operands are exact in 64 bits, products of two 16-bit values are
exact in f32, so a kernel's error is: the f32 sum's, at most (k + 2) 2^-23 S
with S = sum |x w| + |bias| (also for truncating adders); the activation's,
whose slope is at most 1.13 and whose own error is at most 4e-6 (1 + |value|);
the residual's addition, 2^-23 of the terms; and the rounding to the output's
type, 2^-8 (bf16) or 2^-11 (f16) of the result, plus f16's smallest step.
"""
import ctypes as C

import pytest

pytestmark = pytest.mark.gpu

ACTS = {"none": 0, "relu": 1, "gelu": 2, "silu": 3}
ROUND = {"bf16": 2.0**-8, "f16": 2.0**-11, "f32": 2.0**-24}
STEP = {"bf16": 1e-40, "f16": 2.0**-24, "f32": 1e-40}


def _types():
    import torch

    return {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def act64(v, act):
    import torch

    if act == "relu":
        return v.clamp(min=0)
    if act == "gelu":
        return 0.5 * v * (1 + torch.tanh(0.7978845608028654 * (v + 0.044715 * v**3)))
    if act == "silu":
        return v * torch.sigmoid(v)
    return v


def want(x, w, bias, act, residual, out_type):
    """(y, bound) in 64 bits."""
    xd, wd = x.double(), w.double()
    k = x.shape[1]
    v, s = xd @ wd.t(), xd.abs() @ wd.abs().t()
    if bias is not None:
        v, s = v + bias.double(), s + bias.double().abs()
    y = act64(v, act)
    err = 1.13 * (k + 2) * 2.0**-23 * s
    if act in ("gelu", "silu"):
        err = err + 4e-6 * (1 + y.abs())
    if residual is not None:
        r = residual.double()
        err = err + 2.0**-23 * (y.abs() + r.abs())
        y = y + r
    return y, err + 1.01 * ROUND[out_type] * y.abs() + STEP[out_type]


def inputs(m, n, k, t, bias, residual, out_type, seed=0):
    import torch

    ty = _types()
    g = torch.Generator(device="cuda").manual_seed(seed * 7919 + m * 31 + n * 17 + k)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    x, w = r(m, k).to(ty[t]), (r(n, k) * max(k, 1) ** -0.5).to(ty[t])
    return (x, w, r(n).to(ty[t]) if bias else None, r(m, n).to(ty[out_type]) if residual else None,
            torch.full((m, n), float("nan"), dtype=ty[out_type], device="cuda"))


def check(got, y, bound):
    d = (got.double() - y).abs()
    over = ~(d <= bound)  # a NaN is over, too
    assert not over.any(), (int(over.sum()), float(d[over].max()), over.nonzero()[:4].tolist())


SIZES = [(1, 1, 1), (1, 8, 8), (3, 5, 7), (2, 7, 0), (1, 128, 64), (1, 513, 2048), (4, 64, 4096), (8, 96, 1000),
         (16, 128, 256), (17, 129, 65), (31, 2, 130), (33, 1024, 512), (64, 200, 72), (65, 136, 776), (100, 77, 1003),
         (128, 256, 128), (130, 300, 1000), (250, 512, 64), (257, 513, 129), (300, 640, 2056), (513, 1024, 776),
         (1000, 2048, 96), (1, 4096, 4096), (129, 11008, 256), (2047, 385, 1024), (600, 4100, 520)]


@pytest.mark.parametrize("t", ["bf16", "f16"])
@pytest.mark.parametrize("m,n,k", SIZES)
def test_sizes(cuda, m, n, k, t):
    import torch

    i = SIZES.index((m, n, k))
    act, bias, residual = list(ACTS)[i % 4], i % 3 != 0, i % 2 == 1
    x, w, b, r, y = inputs(m, n, k, t, bias, residual, t)
    ref, bound = want(x, w, b, act, r, t)
    torch.cuda.synchronize()
    cuda.linear_dev(x, w, b, ACTS[act], r, y)
    cuda.sync()
    check(y, ref, bound)


@pytest.mark.parametrize("m,n,k", [(1, 40, 4096), (20, 130, 264), (256, 256, 512), (700, 520, 1032), (65, 33, 45)])
@pytest.mark.parametrize("act", list(ACTS))
def test_f32_output_and_every_activation(cuda, m, n, k, act):
    import torch

    x, w, b, r, y = inputs(m, n, k, "bf16", True, True, "f32")
    ref, bound = want(x, w, b, act, r, "f32")
    torch.cuda.synchronize()
    cuda.linear_dev(x, w, b, ACTS[act], r, y)
    cuda.sync()
    check(y, ref, bound)


@pytest.mark.parametrize("m,n,k,pad", [(5, 30, 64, 8), (70, 130, 72, 8), (70, 130, 72, 1), (300, 264, 520, 24),
                                       (300, 264, 520, 3), (1, 264, 512, 5)])
def test_strided_rows_and_offset_bases(cuda, m, n, k, pad):
    """Row strides that are and are not multiples of 16 bytes, bases one element into their buffers; what lies
    between the rows stays."""
    import torch

    x, w, b, r, _ = inputs(m, n, k, "f16", True, True, "f16")

    def strided(t, fill):
        buf = torch.full((t.shape[0] * (t.shape[1] + pad) + pad,), fill, dtype=t.dtype, device="cuda")
        v = buf[pad % 8:].as_strided((t.shape[0], t.shape[1]), (t.shape[1] + pad, 1))
        v.copy_(t)
        return buf, v

    (_, xs), (_, ws), (_, rs) = strided(x, 3.0), strided(w, -5.0), strided(r, 9.0)
    buf, ys = strided(torch.zeros(m, n, dtype=torch.float16, device="cuda"), 7.0)
    ref, bound = want(x, w, b, "relu", r, "f16")
    before = buf.clone()
    torch.cuda.synchronize()
    cuda.linear_dev(xs, ws, b, 1, rs, ys)
    cuda.sync()
    check(ys, ref, bound)
    ys.zero_()
    before_v = before[pad % 8:].as_strided((m, n), (n + pad, 1))
    before_v.zero_()
    assert torch.equal(buf, before)


@pytest.mark.parametrize("m,n,k", [(1, 300, 520), (48, 520, 256), (513, 264, 392), (40, 51, 77)])
def test_residual_in_place(cuda, m, n, k):
    import torch

    x, w, b, r, _ = inputs(m, n, k, "bf16", True, True, "bf16")
    ref, bound = want(x, w, b, "none", r, "bf16")
    torch.cuda.synchronize()
    cuda.linear_dev(x, w, b, 0, r, r)
    cuda.sync()
    check(r, ref, bound)


@pytest.mark.parametrize("m,n,k", [(6, 140, 264), (70, 300, 520), (600, 520, 392), (9, 33, 51)])
def test_infinities_and_nans_stay_in_their_rows(cuda, m, n, k):
    import torch

    x, w, b, r, y = inputs(m, n, k, "bf16", True, False, "bf16")
    x[m // 2, k // 3] = float("nan")
    x[m - 1, k - 1] = float("inf")
    w[n - 1, 0] = float("nan")
    ref, bound = want(x, w, b, "none", None, "bf16")
    torch.cuda.synchronize()
    cuda.linear_dev(x, w, b, 0, None, y)
    cuda.sync()
    bad = torch.zeros(m, n, dtype=torch.bool, device="cuda")
    bad[m // 2] = True
    bad[m - 1] = True
    bad[:, n - 1] = True
    assert torch.isnan(y[m // 2]).all() and torch.isnan(y[:, n - 1]).all()
    assert not torch.isfinite(y[m - 1]).any()
    check(y[~bad], ref[~bad], bound[~bad])


def test_large_activations_saturate_like_the_formula(cuda):
    """gelu and silu far from zero: 0 (or -0) on the left, the value itself on the right, no NaN from e^x."""
    import torch

    v = torch.tensor([-3e38, -1e4, -100.0, -90.0, -20.0, 0.0, 20.0, 90.0, 1e4, 3e38], device="cuda").bfloat16()
    x, w = v[:, None].contiguous(), torch.ones(1, 1, dtype=torch.bfloat16, device="cuda")
    for act in ("gelu", "silu"):
        y = torch.empty(10, 1, dtype=torch.float32, device="cuda")
        torch.cuda.synchronize()
        cuda.linear_dev(x, w, None, ACTS[act], None, y)
        cuda.sync()
        got = y[:, 0].double()
        left, right = v.double() < -80, v.double() > 15
        assert (got[left].abs() < 1e-30).all()
        assert ((got - v.double())[right].abs() <= 1e-6 * v.double()[right]).all()


def test_zero_sizes_do_nothing(cuda):
    import torch

    e = lambda *s: torch.empty(*s, dtype=torch.bfloat16, device="cuda")  # noqa: E731
    cuda.linear_dev(e(0, 8), e(4, 8), None, 0, None, e(0, 4))
    cuda.linear_dev(e(3, 8), e(0, 8), None, 0, None, e(3, 0))
    cuda.sync()


@pytest.mark.parametrize("m,n,k", [(3, 260, 1000), (90, 520, 264), (400, 384, 520), (50, 70, 99)])
def test_repeats_bit_for_bit_and_in_a_graph(cuda, m, n, k):
    import torch

    x, w, b, r, y = inputs(m, n, k, "f16", True, True, "f16")
    torch.cuda.synchronize()
    call = lambda: cuda.linear_dev(x, w, b, 2, r, y)  # noqa: E731
    call()
    cuda.sync()
    first = y.clone()
    g = cuda.capture(call)
    for _ in range(3):
        y.fill_(float("nan"))
        torch.cuda.synchronize()
        g.launch()
        cuda.sync()
        assert torch.equal(y, first)
    g.close()


def test_follows_the_backends_stream(cuda):
    """Calls that feed one another on the backend's stream need no wait between them."""
    import torch

    g = torch.Generator(device="cuda").manual_seed(5)
    x = torch.randn(64, 512, generator=g, device="cuda").bfloat16()
    ws = [(torch.randn(512, 512, generator=g, device="cuda") * 512**-0.5).bfloat16() for _ in range(6)]
    outs = [torch.empty_like(x) for _ in ws]
    torch.cuda.synchronize()
    cur = x
    for w, o in zip(ws, outs):
        cuda.linear_dev(cur, w, None, 0, None, o)
        cur = o
    cuda.sync()
    cur = x
    for w, o in zip(ws, outs):
        ref, bound = want(cur, w, None, "none", None, "bf16")
        check(o, ref, bound)
        cur = o


def test_refusals(cuda):
    import torch

    from tpt_infer_b200 import OpError
    from tpt_infer_b200._capi import lib

    z = lambda *s, dt=torch.bfloat16: torch.zeros(*s, dtype=dt, device="cuda")  # noqa: E731

    def refused(kind, *a):
        with pytest.raises(OpError) as e:
            cuda.linear_dev(*a)
        assert e.value.kind == kind

    refused("ShapeMismatch", z(2, 8), z(4, 9), None, 0, None, z(2, 4))
    refused("ShapeMismatch", z(2, 8), z(4, 8), z(5), 0, None, z(2, 4))
    refused("ShapeMismatch", z(2, 8), z(4, 8), None, 0, z(2, 5), z(2, 4))
    refused("ShapeMismatch", z(2, 8), z(4, 8), None, 0, None, z(4, 2))
    refused("ShapeMismatch", z(8, 2).t(), z(4, 8), None, 0, None, z(2, 4))
    refused("ShapeMismatch", z(1, 8).expand(2, 8), z(4, 8), None, 0, None, z(2, 4))
    refused("Unsupported", z(2, 8), z(4, 8, dt=torch.float16), None, 0, None, z(2, 4))
    refused("Unsupported", z(2, 8, dt=torch.float32), z(4, 8, dt=torch.float32), None, 0, None,
            z(2, 4, dt=torch.float32))
    refused("Unsupported", z(2, 8), z(4, 8), None, 0, None, z(2, 4, dt=torch.float16))
    refused("Invalid", z(2, 8), z(4, 8), None, 4, None, z(2, 4))
    refused("Invalid", z(2, 8).cpu(), z(4, 8), None, 0, None, z(2, 4))
    x, w, y = z(2, 8), z(4, 8), z(2, 4)
    p = lambda t, off=0: C.c_void_p(t.data_ptr() + off)  # noqa: E731
    bf = 2
    assert lib.tpt_cuda_linear_dev(None, bf, p(x), 8, 2, 8, p(w), 8, 4, None, 0, None, 0, p(y), 4, bf) == 4
    assert lib.tpt_cuda_linear_dev(cuda.ctx, bf, None, 8, 2, 8, p(w), 8, 4, None, 0, None, 0, p(y), 4, bf) == 4
    assert lib.tpt_cuda_linear_dev(cuda.ctx, bf, p(x, 1), 8, 2, 8, p(w), 8, 4, None, 0, None, 0, p(y), 4, bf) == 4
    assert lib.tpt_cuda_linear_dev(cuda.ctx, bf, p(x), 7, 2, 8, p(w), 8, 4, None, 0, None, 0, p(y), 4, bf) == 2
    assert lib.tpt_cuda_linear_dev(cuda.ctx, 7, p(x), 8, 2, 8, p(w), 8, 4, None, 0, None, 0, p(y), 4, 7) == 3
    assert lib.tpt_cuda_linear_dev(cuda.ctx, bf, p(x), 8, 1 << 31, 8, p(w), 8, 4, None, 0, None, 0, p(y), 4, bf) == 3
    cuda.sync()


@pytest.mark.parametrize("m,k,n", [(16, 4096, 32768), (48, 4096, 2048)])  # whole k in a CTA; k split over a cluster
def test_linear_wait_limit_reports_a_timeout_and_the_context_recovers(cuda, m, k, n):
    """With the wait limit cut to 100 cycles the waits of a normal launch run out over its loads from memory: the
    kernel leaves, the host reads a timeout, and with the default limit the next call is right."""
    import torch

    from tpt_infer_b200 import OpError
    from tpt_infer_b200._capi import lib

    g = torch.Generator(device="cuda").manual_seed(m)
    x = torch.randn(m, k, generator=g, device="cuda").bfloat16()
    w = torch.randn(n, k, generator=g, device="cuda").bfloat16()
    y = torch.empty(m, n, device="cuda")
    torch.cuda.synchronize()
    try:
        assert lib.tpt_cuda_ctx_set_wait_limit(cuda.ctx, 100) == 0
        cuda.linear_dev(x, w, None, 0, None, y)
        with pytest.raises(OpError) as e:
            cuda.sync()
        assert e.value.code == 7  # TPT_TIMEOUT
    finally:
        assert lib.tpt_cuda_ctx_set_wait_limit(cuda.ctx, 0) == 0
    ref = x.double() @ w.double().t()
    bound = (k + 2) * 2.0**-23 * (x.double().abs() @ w.double().abs().t())
    for _ in range(2):
        cuda.linear_dev(x, w, None, 0, None, y)
        cuda.sync()
        check(y, ref, bound)


def behind(rows, cols, ld, dtype, fill):
    """A [rows, cols] view, rows ld apart, into a buffer of `fill` that goes on behind its last value; the base is on
    16 bytes."""
    import torch

    buf = torch.full((rows * ld + 64,), fill, dtype=dtype, device="cuda")
    return buf, buf.as_strided((rows, cols), (ld, 1))


@pytest.mark.parametrize("t", ["bf16", "f16"])
@pytest.mark.parametrize("fill", [float("nan"), float("inf")])
@pytest.mark.parametrize("m,n,k,ld", [(1, 70, 1003, 1008), (4, 70, 1003, 1008), (5, 70, 1003, 1008),
                                      (3, 33, 70, 72), (2, 17, 1, 8), (4, 40, 63, 128), (1, 600, 4093, 4096),
                                      (1, 1, 1003, 1003), (4, 1, 1003, 1003), (4, 1, 1, 1), (1, 1, 9, 9), (2, 1, 65, 65),
                                      (200, 1, 1003, 1003), (300, 40, 1003, 1008)])
def test_what_lies_behind_a_row_stays_out(cuda, m, n, k, ld, fill, t):
    """Rows on 16 bytes whose length is not a multiple of 8, with NaN or infinities between and behind them, in both
    operands: few tokens give what many give."""
    x, w, b, r, y = inputs(m, n, k, t, True, True, t)
    ref, bound = want(x, w, b, "none", r, t)
    (_, xs), (_, ws) = behind(m, k, ld, x.dtype, fill), behind(n, k, ld, w.dtype, fill)
    xs.copy_(x)
    ws.copy_(w)
    import torch

    torch.cuda.synchronize()
    cuda.linear_dev(xs, ws, b, 0, r, y)
    cuda.sync()
    check(y, ref, bound)


@pytest.mark.parametrize("m", [1, 2, 3, 4])
@pytest.mark.parametrize("n,k", [(30, 64), (264, 512), (130, 1000)])
def test_few_tokens_with_strided_rows_on_16_bytes(cuda, m, n, k):
    """Strided operands that are read in place: x, w, residual and y; what lies between y's rows stays."""
    import torch

    x, w, b, r, _ = inputs(m, n, k, "bf16", True, True, "f32")
    (_, xs), (_, ws), (_, rs), (buf, ys) = (behind(m, k, k + 24, x.dtype, 3.0), behind(n, k, k + 8, w.dtype, -5.0),
                                            behind(m, n, n + 3, r.dtype, 9.0), behind(m, n, n + 5, r.dtype, 7.0))
    for v, src in ((xs, x), (ws, w), (rs, r)):
        v.copy_(src)
    ref, bound = want(x, w, b, "relu", r, "f32")
    torch.cuda.synchronize()
    cuda.linear_dev(xs, ws, b, 1, rs, ys)
    cuda.sync()
    check(ys, ref, bound)
    if m > 1:
        assert (buf[: m * (n + 5)].view(m, n + 5)[:, n:] == 7).all()
    assert (buf[m * (n + 5):] == 7).all()


@pytest.mark.parametrize("m,n", [(1, 3), (4, 4), (5, 130), (100, 40), (300, 257)])
@pytest.mark.parametrize("ld", [0, 1, 64, 4096])
def test_no_products_with_null_operands_and_any_stride(cuda, m, n, ld):
    """k = 0 through the C ABI: x and w may be null, whatever their strides say: act(bias) + residual."""
    import torch

    from tpt_infer_b200._capi import lib

    g = torch.Generator(device="cuda").manual_seed(m + n)
    b = torch.randn(n, generator=g, device="cuda").bfloat16()
    r = torch.randn(m, n, generator=g, device="cuda")
    y = torch.full((m, n), float("nan"), device="cuda")
    p = lambda t: C.c_void_p(t.data_ptr())  # noqa: E731
    torch.cuda.synchronize()
    assert lib.tpt_cuda_linear_dev(cuda.ctx, 2, None, ld, m, 0, None, ld, n, p(b), 1, p(r), n, p(y), n, 0) == 0
    cuda.sync()
    assert torch.equal(y, b.float().clamp(min=0) + r)


def runs_out_and_recovers(cuda, m, k, n, act=0):
    """A launch under a wait limit of 100 cycles is reported as a timeout; with the default limit the next are right."""
    import torch

    from tpt_infer_b200 import OpError
    from tpt_infer_b200._capi import lib

    x, w, b, r, y = inputs(m, n, k, "bf16", True, True, "bf16")
    flush = torch.empty(64 << 20, device="cuda")  # the operands' loads come from memory
    flush.zero_()
    torch.cuda.synchronize()
    try:
        assert lib.tpt_cuda_ctx_set_wait_limit(cuda.ctx, 100) == 0
        cuda.linear_dev(x, w, b, act, r, y)
        with pytest.raises(OpError) as e:
            cuda.sync()
        assert e.value.code == 7  # TPT_TIMEOUT
    finally:
        assert lib.tpt_cuda_ctx_set_wait_limit(cuda.ctx, 0) == 0
    ref, bound = want(x, w, b, "none", r, "bf16")
    for _ in range(2):
        y.fill_(float("nan"))
        torch.cuda.synchronize()
        cuda.linear_dev(x, w, b, act, r, y)
        cuda.sync()
        check(y, ref, bound)


@pytest.mark.parametrize("m,k,n", [(16, 64, 16384), (16, 128, 4096), (32, 192, 8192), (64, 256, 4096), (40, 512, 600)])
def test_linear_wait_limit_with_every_stage_issued(cuda, m, k, n):
    """k so short that all its copies are on their way when the products' wait runs out: they arrive before the CTAs
    leave."""
    runs_out_and_recovers(cuda, m, k, n)


@pytest.mark.parametrize("m,k,n", [(300, 4096, 2048), (1000, 128, 600), (200, 64, 16384), (2000, 776, 5000)])
def test_linear_wait_limit_in_the_pair_kernel(cuda, m, k, n):
    """More than 128 tokens: the SM pairs leave with their two producers at any stages, and the next call is right."""
    runs_out_and_recovers(cuda, m, k, n)


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("out", ["f32", "bf16"])
@pytest.mark.parametrize("m", [1, 4, 40, 300])
def test_smooth_activations_left_of_zero(cuda, m, out, act):
    """The left tails, relatively. y = x / (1 + e^-z), z = x (silu) or 2 sqrt(2/pi) (x + 0.044715 x^3) (gelu, within
    2 |z| 2^-23 relatively for its roundings and its constants'). f32: expf's 2 ulp, the sum's, the reciprocal's and the
    product's roundings, under 5 * 2^-23. bf16: the hardware exponential's documented 2 + 1.173 |z| ulp, 4 for the rest,
    and the last rounding."""
    import torch

    z = -torch.linspace(0.01, 85, 1000, dtype=torch.float64)
    v = z if act == "silu" else -torch.linspace(0.01, 10, 1000, dtype=torch.float64)
    v = v.bfloat16().cuda()
    x = torch.zeros(m, 8, dtype=torch.bfloat16, device="cuda")
    w = torch.zeros(1000, 8, dtype=torch.bfloat16, device="cuda")
    x[:, 0], w[:, 0] = 1, v
    y = torch.empty(m, 1000, dtype=_types()[out], device="cuda")
    torch.cuda.synchronize()
    cuda.linear_dev(x, w, None, ACTS[act], None, y)
    cuda.sync()
    v = v.double()
    z = v if act == "silu" else 2 * (2 / torch.pi) ** 0.5 * (v + 0.044715 * v**3)
    ref = v * torch.sigmoid(z)
    own = 0 if act == "silu" else 2 * z.abs()
    rel = (5 + own) * 2.0**-23 if out == "f32" else (6 + own + 1.173 * z.abs()) * 2.0**-23 + 1.01 * 2.0**-8
    d = (y.double() - ref).abs() / ref.abs()
    assert (d <= rel).all(), (float(d.max() * 2**23), float((d / rel).max()))
