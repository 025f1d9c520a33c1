"""Products with e4m3 weights and activations of shares without columns and of batches without rows, on a CPU."""
import torch

from e4m3_rows import gen, weight
from xfastertransformer_b200 import ops
from xfastertransformer_b200.runtime.loader import LinearWeight


def test_products_of_no_columns_and_of_no_rows():
    """Activations that are not rows in e4m3 yet."""
    W = LinearWeight("fp8a", torch.zeros(64, 0).to(torch.float8_e4m3fn), torch.zeros(1, 0), in_features=0, out_features=64)
    r = torch.randn(3, 64, generator=gen(2))
    assert torch.equal(ops.linear(torch.zeros(3, 0), W, residual=r), r)
    q = ops.quantize_e4m3(torch.zeros(0, 200))
    assert q.shape == (0, 200) and q.scale.shape == (2, 0)
    V = weight(gen(3), 256, 200)
    assert ops.linear(torch.zeros(0, 200), V).shape == (0, 256) and ops.linear_gated(torch.zeros(0, 200), V).shape == (0, 128)
