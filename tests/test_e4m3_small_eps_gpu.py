"""Norms in e4m3 whose factor 1 / rms, or a block's maximum in front of it, is at the ends of 32 bits (csrc/kernels/rows_e4m3.cu)."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from e4m3_rows import coded_error, gen, scale_error, values64
from xfastertransformer_b200 import ops


def norm64(x, gain, eps):
    d = x.double()
    return d * torch.rsqrt(d.pow(2).mean(-1, keepdim=True) + eps) * gain.double()


@pytest.mark.parametrize("residual", [None, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("eps", [1e-12, 1e-14, 1e-20])
@pytest.mark.parametrize("K", [8, 264, 1032, 4096])
def test_rows_of_zeros_and_of_small_numbers(K, eps, residual):
    """Zeros stay zeros, and what lies below the floor keeps its sign: 448 / 2^-100 times 1 / sqrt(eps) is beyond 32 bits.  The sum of squares of the
    small rows is below eps by more than 2^24, so the factor is known to the eight roundings that the norms of larger rows have as well."""
    g = gen(K, 3)
    x = torch.zeros(6, K)
    x[1] = torch.randn(K, generator=g) * 1e-36                        # 448 over its maximum is beyond 32 bits
    x[1, ::3] = 0
    x[2, :K // 2] = torch.randn(K // 2, generator=g) * 2e-7           # empty blocks beside blocks that are not
    x[3] = torch.randn(K, generator=g) * 1e-33
    x[4] = torch.randn(K, generator=g)
    x[5, 0] = 1e-30                                                   # one number in a row of zeros
    x, gain = x.bfloat16(), 1 + 0.2 * torch.randn(K, generator=g)
    r = None if residual is None else torch.zeros(6, K, dtype=residual, device="cuda")
    q, y, _ = ops.rmsnorm_e4m3(x.cuda(), gain.cuda(), eps, r, want_rows=True)
    want = norm64(x, gain, eps)
    err = (K / 256 + 21) * 2.0 ** -24 * want.abs()
    assert torch.isfinite(q.codes.cpu().float()).all() and torch.isfinite(q.scale.cpu()).all()
    assert bool((values64(q)[0] == 0).all())
    assert coded_error(q, want, err) <= 0 and scale_error(q, want, err) <= 0
    assert bool(((y.cpu().double() - want).abs() <= 2.0 ** -8 * want.abs() + err + 2.0 ** -126).all())


def test_a_factor_that_is_no_number():
    """eps 0: a row of zeros is 0 times infinity; one whose squares leave 32 bits is zero; a NaN or an infinity in a row makes its norm's codes NaN where
    the formula has NaN.  Codes and scales are those of the formula, and no other row's."""
    x = torch.zeros(6, 264)
    x[1], x[2, 7], x[3, 200], x[4], x[5] = 1.0, float("nan"), float("inf"), 1e30, torch.linspace(-2, 2, 264)
    x[2, 8:], x[3, :100] = 1.0, -2.0
    x, gain = x.bfloat16(), torch.ones(264)
    got, want = ops.rmsnorm_e4m3(x.cuda(), gain.cuda(), 0.0)[0], ops.rmsnorm_e4m3(x, gain, 0.0)[0]
    c, w = got.codes.cpu().float(), want.codes.float()
    assert torch.equal(torch.isnan(c), torch.isnan(w)) and torch.isnan(c[0]).all() and torch.isnan(c[2]).all() and torch.isnan(c[3]).sum() == 1
    assert torch.equal(c[:5].nan_to_num(), w[:5].nan_to_num())
    assert torch.equal(got.scale.cpu()[:, [0, 2, 3, 4]], want.scale[:, [0, 2, 3, 4]])
    assert bool((c[5] - w[5]).abs().le(0.125 * w[5].abs() + 2.0 ** -9).all())      # a rounding of the norm may cross the border of two codes
