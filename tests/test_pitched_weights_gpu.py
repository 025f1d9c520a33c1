"""Weights whose rows do not start on 16 bytes: the copy that a captured product makes is the graph's, the one that an eager product makes is kept."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from e4m3_rows import gen
from xfastertransformer_b200 import ops
from xfastertransformer_b200.runtime.loader import LinearWeight, make_linear


def wide(W):
    """The same weight with rows on 16 bytes, which no product has to copy."""
    n = W.w.shape[1]
    room = torch.zeros(W.w.shape[0], (n + 15) // 16 * 16, dtype=torch.uint8, device="cuda")
    room[:, :n] = W.w.view(torch.uint8)
    return LinearWeight(W.kind, room.view(W.w.dtype)[:, :n], W.scale, W.zero, W.wsum, W.block, W.in_features, W.out_features)


@pytest.mark.parametrize("kind", ["fp8", "int8", "int4", "nf4"])
@pytest.mark.parametrize("T", [1, 40])
def test_capture_before_the_first_eager_call(kind, T):
    """The bits of a weight that lies on 16 bytes, from the eager product behind a capture and from the graph."""
    g = gen(T, 3)
    W = make_linear(torch.randn(256, 200, generator=g) * 0.05, kind).to("cuda")
    assert W.w.stride(0) % 16
    x = torch.randn(T, 200, generator=g).bfloat16().cuda()
    want = ops.linear(x, wide(W), out_dtype=torch.float32)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = ops.linear(x, W, out_dtype=torch.float32)
    assert "w_pitch16" not in W.cache
    eager = ops.linear(x, W, out_dtype=torch.float32)                  # before the graph's copy has been made once
    assert torch.equal(eager, want) and "w_pitch16" in W.cache
    for _ in range(2):
        y.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want)
