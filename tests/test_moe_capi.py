"""The 16-bit and mixture-of-experts entry points without a device: declared, bound, and refusing a missing context;
and the cases in perf/operators.py, whose sizes stay in the range that their draws promise."""
import importlib.util
import os
import random

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_no_context_is_invalid():
    from tpt_infer_b200._capi import lib

    assert lib.tpt_cuda_linear_dev(None, 2, None, 8, 1, 8, None, 8, 8, None, 0, None, 0, None, 8, 2) == 4
    assert lib.tpt_cuda_route_experts_dev(None, None, 0, 8, 1, 8, 0, None, 1, 1, 1, 2, 1, 1.0, None, None, None) == 4
    assert lib.tpt_cuda_experts_mlp_dev(None, 2, None, 8, 1, 8, None, None, 2, None, None, 4, 8, 3, 1, None, 0, None, 8) == 4


def test_type_and_activation_codes_match_the_header():
    import re

    from tpt_infer_b200 import ACT_GELU, ACT_NONE, ACT_RELU, ACT_SILU
    from tpt_infer_b200 import backend as B

    h = open(os.path.join(ROOT, "include", "tpt_cuda.h")).read()
    code = lambda name: int(re.search(rf"\b{name} = (\d+)", h).group(1))  # noqa: E731
    assert (ACT_NONE, ACT_RELU, ACT_GELU, ACT_SILU) == tuple(
        code(f"TPT_ACT_{n}") for n in ("NONE", "RELU", "GELU", "SILU"))
    assert (B.DT_F32, B.DT_BF16, B.DT_F16) == tuple(code(f"TPT_DT_{n}") for n in ("F32", "BF16", "F16"))
    assert B._SCORES == {"softmax": code("TPT_SCORE_SOFTMAX"), "sigmoid": code("TPT_SCORE_SIGMOID")}


def test_codes_of_torch_types():
    import torch

    from tpt_infer_b200 import backend as B

    assert [B._CODE[t] for t in (torch.float32, torch.bfloat16, torch.float16)] == [B.DT_F32, B.DT_BF16, B.DT_F16]
    assert B._CODE[torch.float64] == -1 and B._CODE[torch.int32] not in (B.DT_F32, B.DT_BF16, B.DT_F16, -1)


def test_drawn_cases_stay_in_range():
    spec = importlib.util.spec_from_file_location("operators_cases", os.path.join(ROOT, "perf", "operators.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    most = max(mod.work(c)["flops"] for c in mod.listed())
    for seed in range(300):
        c = mod.draw(random.Random(seed))
        w = mod.work(c)
        assert w["bytes"] > 0 and 0 < w["flops"] <= most
        if c["op"] == "route":
            assert c["experts"] % c["groups"] == 0 and c["top_k"] <= c["kept"] * (c["experts"] // c["groups"])
        if c["op"] == "experts":
            assert c["top_k"] <= c["experts"]
