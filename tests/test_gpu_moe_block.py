"""The mixture-of-experts block of examples/moe_block.py: its operators in the order a model runs them."""
import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _example():
    spec = importlib.util.spec_from_file_location("moe_block", os.path.join(ROOT, "examples", "moe_block.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


@pytest.mark.parametrize("tokens", [1, 7, 130, 1100])
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
def test_block_against_64_bits(cuda, tokens, dtype):
    """In 64 bits from the device's own choice of experts. Four roundings to the type lie between x and y (the shared
    layer's hidden values, the residual stream, an expert's hidden values, y), each at most 2^-8 (bf16) or 2^-11 (f16)
    of its values, whose norms are at most y's own and the hidden layers' images': under 8 roundings of |y| in all."""
    import torch

    dt = getattr(torch, dtype)
    block = _example().MoeBlock(width=512, hidden=136, experts=24, top_k=3, shared_hidden=520, dtype=dt, seed=tokens)
    x = torch.randn(tokens, 512, device="cuda").to(dt)
    y = torch.empty_like(x)
    torch.cuda.synchronize()
    ids, weights = block(cuda, x, y)
    cuda.sync()
    xd = x.double()
    logits = xd @ block.router.double().t()
    # f32 logits (error under 512 * 2^-23 * |x||w|, about 1e-4) choose the experts that 64 bits do, up to near ties
    top = torch.topk(logits, 4, 1).values
    clear = (top[:, :3] - top[:, 1:]).amin(1) > 1e-3
    assert torch.equal(ids.long()[clear], torch.topk(logits, 3, 1).indices[clear])
    torch.testing.assert_close(weights.double(), torch.softmax(torch.gather(logits, 1, ids.long()), 1), atol=2e-3, rtol=0)
    h = torch.nn.functional.gelu(xd @ block.w1.double().t() + block.b1.double(), approximate="tanh")
    ref = xd + h @ block.w2.double().t() + block.b2.double()
    for e in range(24):
        tok, j = (ids == e).nonzero(as_tuple=True)
        a = xd[tok] @ block.w_in[e].double().t()
        o = (torch.nn.functional.silu(a[:, :136]) * a[:, 136:]) @ block.w_out[e].double().t()
        ref.index_add_(0, tok, weights[tok, j].double()[:, None] * o)
    err = float((y.double() - ref).norm() / ref.norm())
    assert err < 8 * (2.0**-8 if dtype == "bfloat16" else 2.0**-11), err


def test_block_in_a_graph_with_new_tokens(cuda):
    """Recorded once, replayed on new contents of the same buffers: the same bits as the direct calls."""
    import torch

    block = _example().MoeBlock(width=256, hidden=72, experts=16, top_k=2, shared_hidden=264)
    x, y = torch.randn(40, 256, device="cuda").bfloat16(), torch.empty(40, 256, dtype=torch.bfloat16, device="cuda")
    torch.cuda.synchronize()
    block(cuda, x, y)
    cuda.sync()
    graph = cuda.capture(lambda: block(cuda, x, y))
    for seed in range(3):
        x.copy_(torch.randn(40, 256, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").bfloat16())
        torch.cuda.synchronize()
        graph.launch()
        cuda.sync()
        got = y.clone()
        torch.cuda.synchronize()
        block(cuda, x, y)
        cuda.sync()
        assert torch.equal(got, y)
    graph.close()
