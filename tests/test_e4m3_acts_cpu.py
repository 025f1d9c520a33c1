"""Every activation that the products of rows in e4m3 accept has its function on a CPU, under each of its names."""
import pytest
import torch

from e4m3_rows import gen, rows, weight
from xfastertransformer_b200 import ops

SAME = {"none": None, "swiglu": "silu", "gelu_tanh": "gelu", "gelu_new": "gelu", "gelu_pytorch_tanh": "gelu"}


@pytest.mark.parametrize("act", ops._ROW_ACTS)
def test_activations_that_pass_the_check(act):
    g = gen(5)
    q, W = rows(torch.randn(3, 128, generator=g)), weight(g, 256, 128)
    for fn in (lambda a: ops.linear_e4m3(q, W, act=a), lambda a: ops.linear_gated_e4m3(q, W, a).values(),
               lambda a: ops.moe_experts_e4m3(q, torch.zeros(3, 1, dtype=torch.int32), torch.ones(3, 1), [(W, weight(gen(6), 128, 128))], a)):
        got = fn(act)
        assert torch.isfinite(got).all() and torch.equal(got, fn(SAME.get(act, act)))
