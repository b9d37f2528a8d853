"""A plan's ops refuse activations that their epilogues do not have (silu belongs to the 16-bit products)."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("act", [-1, 3, 4, 100])
def test_plan_refuses_unknown_activations(cuda, act):
    from tpt_infer_b200 import OpError
    from tpt_infer_b200 import graphs as G

    p = G.Plan(cuda)
    try:
        x, q, y, z = p.tensor(G.F32, 4 * 32), p.tensor(G.I8, 4 * 32), p.tensor(G.F32, 4 * 32), p.tensor(G.F32, 4 * 16)
        w, b = p.const(np.zeros((32, 16), np.float32)), p.const(np.zeros(32, np.float32))
        wq = cuda.upload_i8(np.zeros((16, 32), np.int8), np.ones(16, np.float32), 16, 32)
        p.op(G.OP_QUANTIZE, x, q, dims=(4 * 32,))
        for kind, args in ((G.OP_LINEAR, dict(in0=q, out=z, w=wq, dims=(4,))),
                           (G.OP_MATMUL, dict(in0=x, out=z, in1=w, dims=(4, 32, 16))),
                           (G.OP_BIAS_ACT, dict(in0=x, out=y, in1=b, dims=(4, 32))),
                           (G.OP_ADD_ACT, dict(in0=x, out=y, in1=x, dims=(4 * 32,)))):
            with pytest.raises(OpError) as e:
                p.op(kind, act=act, **args)
            assert e.value.kind == "Invalid"
            p.op(kind, act=2, **args)
    finally:
        p.close()
