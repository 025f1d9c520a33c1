"""Shares of a layer's e4m3 products that are empty on a rank, on a GPU: what they give is written, whatever lay in memory."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from e4m3_rows import gen, on, rows, rows_on, weight
from xfastertransformer_b200 import ops
from xfastertransformer_b200.runtime.loader import LinearWeight


def no_weight(n, k, kind="fp8a"):
    return LinearWeight(kind, torch.zeros(n, k).to(torch.float8_e4m3fn), torch.zeros(-(-n // 128), -(-k // 128)), in_features=k, out_features=n).to("cuda")


def soil():
    """What the next allocations find in memory."""
    for n in (1 << 12, 1 << 16, 1 << 20, 1 << 24):
        torch.full((n,), float("nan"), device="cuda")


@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T", [1, 5, 300])
def test_experts_without_features(T, out_dtype):
    """Experts whose features all lie on other ranks add nothing to what is added."""
    g = gen(T)
    H, E = 256, 3
    q = rows_on(rows(torch.randn(T, H, generator=g)))
    experts = [(no_weight(0, H), no_weight(H, 0)) for _ in range(E)]
    idx, w = torch.randint(0, E, (T, 2), generator=g).int().cuda(), torch.rand(T, 2, generator=g).cuda()
    for add in (None, torch.randn(T, H, generator=g).cuda(), torch.randn(T, H, generator=g).cuda().bfloat16()):
        for packed in (None, ops.pack_experts_e4m3(experts)):
            soil()
            got = ops.moe_experts_e4m3(q, idx, w, experts, packed=packed, add=add, out_dtype=out_dtype)
            want = torch.zeros(T, H, device="cuda") if add is None else add
            assert got.dtype == out_dtype and torch.equal(got, want.to(out_dtype))
            assert add is None or got.data_ptr() != add.data_ptr()


def test_gated_product_of_no_columns():
    """act(bias) * bias: the codes and scales of a CPU."""
    g = gen(2)
    none = ops.linear_gated_e4m3(rows_on(rows(torch.randn(4, 128, generator=g))), no_weight(0, 128))
    W, b = no_weight(512, 0), torch.randn(512, generator=g)
    for bias in (None, b.cuda()):
        soil()
        got = ops.linear_gated_e4m3(none, W, "relu", bias)
        y = torch.zeros(4, 512) if bias is None else b.expand(4, 512)
        want = ops.quantize_e4m3(y[:, :256].clamp_min(0) * y[:, 256:])
        assert torch.equal(got.codes.cpu().view(torch.uint8), want.codes.view(torch.uint8)) and torch.equal(got.scale.cpu(), want.scale)


def test_a_product_without_columns_is_refused_by_the_kernel():
    """Nothing would be written: an error, and not a result that stays as it was."""
    from xfastertransformer_b200.ops import native as N, native_e4m3 as E
    q, W = rows_on(rows(torch.randn(4, 128, generator=gen(3)))), on(weight(gen(4), 128, 128))
    with pytest.raises(N.KernelError):
        E._gemm(q, W.w, W.scale, torch.empty(4, 128, device="cuda"), 4, 128, 0)


def test_products_of_no_columns_and_of_no_rows():
    """Activations that are not rows in e4m3 yet."""
    W, r = no_weight(64, 0), torch.randn(3, 64, generator=gen(2)).bfloat16().cuda()
    soil()
    assert torch.equal(ops.linear(torch.zeros(3, 0, dtype=torch.bfloat16, device="cuda"), W, residual=r), r)
    V, none = on(weight(gen(3), 256, 200)), torch.zeros(0, 200, dtype=torch.bfloat16, device="cuda")
    assert ops.linear(none, V).shape == (0, 256) and ops.linear_gated(none, V).shape == (0, 128)


@pytest.mark.parametrize("T", [1, 5, 300])
def test_weights_alone_in_e4m3(T):
    """The type that keeps activations in bf16 has empty shares too."""
    g = gen(T, 2)
    H, E = 256, 3
    x, r, b = torch.randn(T, H, generator=g).bfloat16().cuda(), torch.randn(T, H, generator=g).bfloat16().cuda(), torch.randn(H, generator=g).cuda()
    experts = [(no_weight(0, H, "fp8"), no_weight(H, 0, "fp8")) for _ in range(E)]
    idx, w = torch.randint(0, E, (T, 2), generator=g).int().cuda(), torch.rand(T, 2, generator=g).cuda()
    for add in (None, torch.randn(T, H, generator=g).cuda(), torch.randn(T, H, generator=g).cuda().bfloat16()):
        soil()
        got = ops.moe_experts(x, idx, w, experts, add=add)
        assert got.dtype == torch.float32 and torch.equal(got, torch.zeros(T, H, device="cuda") if add is None else add.float())
        assert add is None or got.data_ptr() != add.data_ptr()
    mid = ops.linear_gated(x, experts[0][0])
    assert mid.shape == (T, 0)
    soil()
    assert torch.equal(ops.linear(mid, experts[0][1], out_dtype=torch.float32), torch.zeros(T, H, device="cuda"))
    assert torch.equal(ops.linear(mid, experts[0][1], residual=r), r)
    assert torch.equal(ops.linear(mid, experts[0][1], b, "relu", r, 0.5, torch.float32), b.clamp_min(0) + 0.5 * r.float())
