"""A mixture-of-experts feed-forward block on the CUDA backend.

    y = x + W2 gelu(W1 x + b1) + b2 + sum_j w_j expert_{e_j}(x)

with e, w the router's choice of experts for each token: the router's logits
(a linear layer with an f32 output), the choice, the shared feed-forward layer
(two linear layers, the second adding the residual) and the experts' layers,
which add theirs on top. All of it runs on the backend's stream; nothing waits
in between, so a block of fixed shape can be recorded as a CUDA graph.

    python examples/moe_block.py [--tokens N] [--steps K]
"""
import argparse
import os
import sys

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import torch  # noqa: E402

from tpt_infer_b200 import ACT_GELU, ACT_NONE, ACT_SILU, CudaBackend  # noqa: E402


class MoeBlock:
    """The block's weights and, for one number of tokens, its intermediate buffers."""

    def __init__(self, width, hidden, experts, top_k, shared_hidden, dtype=torch.bfloat16, seed=0, device=0):
        g = torch.Generator(device=f"cuda:{device}").manual_seed(seed)

        def normal(*shape, std):
            return (torch.randn(*shape, generator=g, device=f"cuda:{device}") * std).to(dtype)

        self.top_k, self.experts = top_k, experts
        self.router = normal(experts, width, std=width**-0.5)
        self.w1, self.b1 = normal(shared_hidden, width, std=width**-0.5), normal(shared_hidden, std=0.02)
        self.w2, self.b2 = normal(width, shared_hidden, std=shared_hidden**-0.5), normal(width, std=0.02)
        self.w_in = normal(experts, 2 * hidden, width, std=width**-0.5)
        self.w_out = normal(experts, width, hidden, std=hidden**-0.5)
        self.buffers = {}

    def _buffers(self, x):
        t = x.shape[0]
        if t not in self.buffers:
            e = lambda *s, dt=x.dtype: torch.empty(*s, dtype=dt, device=x.device)  # noqa: E731
            self.buffers[t] = (e(t, self.experts, dt=torch.float32), e(t, self.top_k, dt=torch.int32),
                               e(t, self.top_k, dt=torch.float32), e(t, self.w1.shape[0]))
        return self.buffers[t]

    def __call__(self, be, x, out):
        """out = the block of x, enqueued on the backend's stream."""
        logits, ids, weights, h = self._buffers(x)
        be.linear_dev(x, self.router, None, ACT_NONE, None, logits)
        be.route_experts_dev(logits, self.top_k, ids, weights)
        be.linear_dev(x, self.w1, self.b1, ACT_GELU, None, h)
        be.linear_dev(h, self.w2, self.b2, ACT_NONE, x, out)
        be.experts_mlp_dev(x, ids, weights, self.w_in, self.w_out, ACT_SILU, True, out, out)
        return ids, weights


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--tokens", type=int, default=64)
    ap.add_argument("--steps", type=int, default=20)
    a = ap.parse_args()
    be = CudaBackend.new(0)
    if be is None:
        sys.exit("no sm_100 device")
    block = MoeBlock(width=2048, hidden=768, experts=64, top_k=4, shared_hidden=2048)
    x = torch.randn(a.tokens, 2048, device="cuda").bfloat16()
    y = torch.empty_like(x)
    torch.cuda.synchronize()
    block(be, x, y)  # sizes the workspace
    graph = be.capture(lambda: block(be, x, y))
    be.sync()
    s, e = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    with torch.cuda.stream(torch.cuda.ExternalStream(be.stream_handle)):
        s.record()
        for _ in range(a.steps):
            graph.launch()
        e.record()
    be.sync()
    print(f"{a.tokens} tokens: {s.elapsed_time(e) / a.steps * 1e3:.1f} us a block, {graph.kernels} kernels")
    graph.close()
    be.close()


if __name__ == "__main__":
    main()
