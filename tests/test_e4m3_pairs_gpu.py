"""The sum of routed experts in e4m3: parts in fp32 wherever the result is fp32, at every number of rows per expert; many experts, and a rank's share of
them."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from e4m3_rows import dense64, gen, on, rows_on, sum_tol, values64
from test_e4m3_rows_gpu import check_status, experts64, routing, whole, whole_rows
from xfastertransformer_b200 import ops
from xfastertransformer_b200.ops import native_e4m3 as E4
from xfastertransformer_b200.ops import reference as R


def parts64(q, idx, w, experts, offset=0):
    """Sum of the magnitudes of what is added up: each of the k products and additions in fp32 is off by at most 2^-24 of it."""
    out = torch.zeros(q.shape[0], experts[0][1].out_features, dtype=torch.float64)
    for e, (gu, dn) in enumerate(experts):
        tok, slot = (idx == e + offset).nonzero(as_tuple=True)
        if tok.numel():
            y = values64(q)[tok] @ dense64(gu).t()
            i = y.shape[1] // 2
            s = sum_tol(R.quantize_e4m3((y[:, :i].clamp_min(0) * y[:, i:]).float()), dn)[0]
            out.index_add_(0, tok, s.abs() * w[tok, slot].double()[:, None])
    return out


# rows per expert: a few, 17 to 32, then both tiles of prompts and one step of them past a tile
@pytest.mark.parametrize("T,E,k,H,I", [(3, 4, 2, 256, 128), (40, 8, 3, 384, 256), (33, 1, 1, 128, 128), (300, 4, 3, 640, 384), (700, 3, 2, 256, 640),
                                       (3300, 2, 1, 256, 128)])
def test_fp32_results_add_fp32_parts(T, E, k, H, I):
    g = gen(T, E, k, H, I)
    q, experts = whole_rows(g, T, H), [(whole(g, 2 * I, H), whole(g, H, I)) for _ in range(E)]
    idx, w = routing(g, T, E, k, idle=False)
    (want, tol), mag = experts64(q, idx, w, experts), parts64(q, idx, w, experts)
    dev = [(on(a), on(b)) for a, b in experts]
    bound = tol + (2 * k + 1) * 2.0 ** -24 * mag
    add = torch.randn(T, H, generator=g)
    # also where the caller says that there are many rows, or few (the choice of a tile is the only thing that may follow)
    for expected in (None, 1, T * k, E * 2000):
        got = ops.moe_experts_e4m3(rows_on(q), idx.cuda(), w.cuda(), dev, "relu", expected_pairs=expected).cpu().double()
        assert bool(((got - want).abs() <= bound).all()), ((got - want).abs() / bound).max().item()
        got = ops.moe_experts_e4m3(rows_on(q), idx.cuda(), w.cuda(), dev, "relu", expected_pairs=expected, add=add.cuda()).cpu().double()
        assert bool(((got - want - add.double()).abs() <= bound + 2.0 ** -24 * (mag + add.double().abs())).all())
        # a bf16 result: half a step of it, and of each part where tiles are those of prompts
        avg = -(-(T * k if expected is None else min(expected, T * k)) // E)
        half = 2.0 ** -8 * mag if E4._tile_rows(max(1, avg)) >= 128 else 0.0
        got = ops.moe_experts_e4m3(rows_on(q), idx.cuda(), w.cuda(), dev, "relu", expected_pairs=expected, out_dtype=torch.bfloat16).cpu().double()
        assert bool(((got - want).abs() <= (bound + half) * (1 + 2.0 ** -8) + 2.0 ** -8 * want.abs()).all())
    check_status()


@pytest.mark.parametrize("share", [(0, 256), (64, 32), (248, 8)])
@pytest.mark.parametrize("T", [1, 30, 600])
def test_256_experts_and_a_share_of_them(T, share):
    """Eight of 256 experts per token, all of them here or a rank's part from `expert_offset` on."""
    first, count = share
    g = gen(T, first, count)
    H, I, k = 256, 128, 8
    q, experts = whole_rows(g, T, H), [(whole(g, 2 * I, H), whole(g, H, I)) for _ in range(count)]
    idx, w = routing(g, T, 256, k, idle=False)
    if T > 1:
        idx[0, :] = -1
        idx[1, :4] = first                                             # one expert four times
    want, tol = experts64(q, idx, w, experts, first)
    mag = parts64(q, idx, w, experts, first)
    add = torch.randn(T, H, generator=g)
    got = ops.moe_experts_e4m3(rows_on(q), idx.cuda(), w.cuda(), [(on(a), on(b)) for a, b in experts], "relu", first, add=add.cuda())
    check_status()
    full = want + add.double()
    assert bool(((got.cpu().double() - full).abs() <= tol + (2 * k + 2) * 2.0 ** -24 * (mag + add.double().abs())).all())
    if T > 1:
        assert torch.equal(got[0].cpu(), add[0])
