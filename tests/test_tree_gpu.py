"""Trees of drafted tokens on a GPU against 64 bits: masks, attention over the cache, sampling, accepted paths, and a step of all of them."""
import math
import random

import pytest
import torch

pytestmark = pytest.mark.gpu

from tree_cases import ancestors, batch, caches, parents_of
from xfastertransformer_b200 import ops
from xfastertransformer_b200.models.decoder import Batch
from xfastertransformer_b200.ops import reference as R

BF16 = torch.finfo(torch.bfloat16).eps / 2


def _ok():
    from xfastertransformer_b200.ops import native as N
    N.Workspace.get(torch.device("cuda", 0)).check_status()


def _meta(cu, kv, table):
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    return Batch(ids=None, positions=None, slots=None, cu_q=cu, kv_lens=kv, block_table=table, cu_q_dev=i32(cu), kv_lens_dev=i32(kv),
                 max_q=max(b - a for a, b in zip(cu, cu[1:])), max_kv=max(kv))


# -- masks ----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("lens", [[(1, 0)], [(5, 3), (1, 9), (17, 64)], [(130, 2), (64, 1), (65, 0)], [(0, 5), (256, 5), (193, 100000)],
                                  [(7, 3)] * 300])
def test_masks(lens):
    _, flat, cu, kv, _, _ = batch(lens, 7, roots=2 if lens[0][0] > 1 else 1)
    want = R.tree_mask(flat, cu, kv)
    for parents in (flat.cuda(), flat.long().cuda()):
        for got in (ops.tree_mask(parents, cu, kv), ops.tree_mask(parents, cu, kv, meta=_meta(cu, kv, None))):
            assert torch.equal(got[0].cpu(), want[0]) and torch.equal(got[1].cpu(), want[1])
    _ok()


def test_batches_that_understate_their_trees_are_reported():
    from xfastertransformer_b200.ops import native as N
    cu, kv = [0, 40], [50]
    meta = _meta(cu, kv, None)
    meta.max_q = 5
    up = torch.arange(-1, 39, dtype=torch.int32, device="cuda")
    c = torch.zeros(1, 1, 64, 128, dtype=torch.bfloat16, device="cuda")
    bits, table = torch.zeros(40, 1, dtype=torch.int64, device="cuda"), torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    for f in (lambda: ops.tree_mask(up, cu, kv, meta), lambda: ops.tree_accept(up, up, up, cu, kv, meta=meta),
              lambda: ops.tree_attention(torch.zeros(40, 2, 128, device="cuda").bfloat16(), c, c, table, cu, kv, bits, 0.1, meta=meta)):
        f()
        with pytest.raises(N.KernelError):
            N.Workspace.get(torch.device("cuda", 0)).check_status()


def test_a_parent_behind_its_child_is_reported():
    from xfastertransformer_b200.ops import native as N
    mask, pos = ops.tree_mask(torch.tensor([-1, 2, 0], dtype=torch.int32, device="cuda"), [0, 3], [5])
    assert mask[:, 0].tolist() == [1, 2, 5] and pos.tolist() == [2, 2, 3]
    with pytest.raises(N.KernelError):
        N.Workspace.get(torch.device("cuda", 0)).check_status()


# -- attention ------------------------------------------------------------------------------------------------------
def _attend(lens, hq, hkv, D, seed=0, bs=64, int8=False, mask=None, group=None, q_off=0, spoil=None, roots=1, scale=None, meta=True, gain=1.0,
            **kw):
    g = torch.Generator().manual_seed(seed)
    trees, flat, cu, kv, table, blocks = batch(lens, seed, bs, roots)
    kc, vc, ks, vs = caches(g, blocks, hkv, D, bs, int8)
    if spoil is not None:                                 # what lies behind the last key, and in blocks of no sequence
        for t in (kc, vc) if not int8 else (ks, vs):
            keep = torch.zeros(blocks, bs, dtype=torch.bool)
            for b, n in enumerate(kv):
                for p in range(n):
                    keep[table[b, p // bs], p % bs] = True
            t.permute(0, 2, 1, *range(3, t.dim()))[~keep] = spoil
    q = (gain * torch.randn(cu[-1], hq, D, generator=g)).bfloat16()
    bits, pos = R.tree_mask(flat, cu, kv)
    if mask is not None:
        bits = mask(bits)
    if kw.get("sinks") is True:
        kw["sinks"] = torch.randn(hq, generator=g)
    scale = D ** -0.5 if scale is None else scale
    f64 = torch.float64
    grp = group or max(hq // hkv, 1)
    # slots behind the last key are no part of the plain sums; 64-bit ones look at the sequence's positions alone
    want = R.tree_attention(q, kc, vc, table, cu, kv, bits, scale, ks, vs, grp, q_off, positions=pos, dtype=f64, **kw)
    size = R.tree_attention(q, kc, vc.abs(), table, cu, kv, bits, scale, ks, vs, grp, q_off, positions=pos, dtype=f64, **kw)
    c = lambda t: t.cuda() if isinstance(t, torch.Tensor) else t
    got = ops.tree_attention(c(q), c(kc), c(vc), c(table), cu, kv, c(bits), scale, c(ks), c(vs), group, q_off,
                             _meta(cu, kv, table) if meta else None, positions=c(pos), **{n: c(v) for n, v in kw.items()})
    _ok()
    # A weight is rounded to bf16 once, 2^-8 of it; the sum that divides either has the rounded weights (the same again at most) or the
    # whole ones; the result is rounded to bf16.  Scores in 32 bits: D + 8 roundings of 2^-24 of sums of |q k|, which move a weight and
    # the denominator by as much.
    qk = float(q.float().abs().max()) * (127 * float(ks.abs().nan_to_num().max()) if int8 else float(kc.float().nan_to_num().abs().max()))
    score = 2 * (D + 8) * 2.0 ** -24 * min(qk * D, 40 * gain * D ** 0.5 * qk ** 0.5) * scale
    bound = (2 * BF16 + score + 2.0 ** -12) * size + BF16 * 1.02 * want.abs() + 1e-30
    err = (got.double().cpu() - want).abs()
    assert bool((err <= bound).all()), (float((err / bound.clamp_min(1e-20)).max()), float(err.max()))
    return got


LENS = [[(1, 0)], [(1, 1), (3, 0)], [(2, 62), (5, 59), (4, 64)], [(16, 700)], [(33, 128), (7, 1000), (0, 40), (64, 31)], [(64, 4100)]]


@pytest.mark.parametrize("lens", LENS)
@pytest.mark.parametrize("hq,hkv", [(1, 1), (8, 2), (7, 1), (12, 4), (16, 1), (5, 5)])
def test_attention(lens, hq, hkv):
    _attend(lens, hq, hkv, 128, seed=hq)


@pytest.mark.parametrize("D", [64, 256])
@pytest.mark.parametrize("lens", LENS[2:5])
def test_other_heads(lens, D):
    _attend(lens, 6, 2, D)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("lens", LENS[1:5])
def test_int8_cache(lens, D):
    _attend(lens, 8, 2, D, int8=True)


@pytest.mark.parametrize("bs", [16, 128, 192])
@pytest.mark.parametrize("int8", [False, True])
def test_other_blocks(bs, int8):
    _attend([(9, 300), (31, 77)], 8, 2, 128, bs=bs, int8=int8)


@pytest.mark.parametrize("nodes", [65, 130, 256])
@pytest.mark.parametrize("roots", [1, 3])
def test_wide_trees(nodes, roots):
    _attend([(nodes, 300), (nodes - 64, 5)], 8, 1, 128, roots=roots)


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("spoil", [math.nan, math.inf, -math.inf])
def test_slots_behind_the_last_key(spoil, int8):
    _attend([(9, 300), (31, 0), (1, 64), (3, 2000)], 8, 2, 128, spoil=spoil, int8=int8)


@pytest.mark.parametrize("D,int8", [(64, False), (128, False), (128, True), (256, False)])
@pytest.mark.parametrize("kw", [{"softcap": 5.0}, {"window": 7}, {"window": 200, "keep_first": 5}, {"window": 1, "keep_first": 70},
                                {"sinks": True}, {"sinks": True, "softcap": 30.0, "window": 100, "keep_first": 4}])
def test_caps_windows_and_sinks(D, int8, kw):
    _attend([(20, 1500), (6, 40), (5, 0)], 8, 2, D, int8=int8, **kw)


@pytest.mark.parametrize("ctx", [0, 100, 3000])
@pytest.mark.parametrize("sinks", [None, True])
def test_masks_of_any_kind(ctx, sinks):
    def some(bits):
        bits = bits.clone()
        bits[::4] = 0                                      # sees no node, and with no context nothing at all
        bits[1::4] = -1                                    # every bit, those of no node among them
        bits[2::4] = -(1 << 63)                            # the last bit alone
        return bits
    got = _attend([(64, ctx), (21, ctx)], 8, 2, 128, mask=some, sinks=sinks)
    if ctx == 0:
        assert not bool(got[0].any())


def test_nodes_that_no_one_sees_may_hold_anything():
    g = torch.Generator().manual_seed(5)
    _, flat, cu, kv, table, blocks = batch([(10, 90)], 1)
    kc, vc, _, _ = caches(g, blocks, 2, 128)
    bits = torch.zeros(10, 1, dtype=torch.int64)
    for i in range(8):
        bits[i] = 1 << i | 1
    q = torch.randn(10, 4, 128, generator=g).bfloat16()
    want = R.tree_attention(q, kc, vc, table, cu, kv, bits, 0.1, group=2, dtype=torch.float64)
    for p in (98, 99):
        for t in (kc, vc):
            t[table[0, p // 64], :, p % 64] = math.nan
    got = ops.tree_attention(q.cuda(), kc.cuda(), vc.cuda(), table.cuda(), cu, kv, bits.cuda(), 0.1)
    assert bool(torch.isfinite(got).all())
    # a few values below 4 in size: two roundings of a weight, one of the result
    assert float((got.double().cpu() - want).abs().max()) <= 3 * BF16 * 5


def test_large_and_small_scores():
    _attend([(12, 500)], 8, 2, 128, gain=60.0)             # one key takes all of the weight
    _attend([(12, 500)], 8, 2, 128, scale=0.0)             # all keys the same
    _attend([(12, 500)], 8, 2, 128, scale=-0.05)


@pytest.mark.parametrize("hq,group,q_off", [(5, 4, 0), (5, 4, 3), (6, 8, 5), (4, 4, 2), (1, 4, 7)])
def test_uneven_shares_of_the_heads(hq, group, q_off):
    hkv = (hq - 1 + q_off) // group + 1
    _attend([(9, 300), (31, 77)], hq, hkv, 128, group=group, q_off=q_off)


def test_strided_inputs_and_lists():
    g = torch.Generator().manual_seed(9)
    _, flat, cu, kv, table, blocks = batch([(9, 200), (4, 70)], 3)
    kc, vc, _, _ = (t.cuda() if t is not None else None for t in caches(g, blocks, 2, 128))
    q = torch.randn(13, 8, 128, generator=g).bfloat16().cuda()
    bits = ops.tree_mask(flat.cuda(), cu, kv)[0]
    want = ops.tree_attention(q, kc, vc, table.cuda(), cu, kv, bits, 0.1)
    wide = torch.zeros(13, 8, 160, dtype=torch.bfloat16, device="cuda")
    wide[..., 3:131] = q
    tab = torch.zeros(2, 2 * table.shape[1], dtype=torch.int32, device="cuda")
    tab[:, ::2] = table.cuda()
    both = torch.zeros(13, 3, dtype=torch.int64, device="cuda")
    both[:, 1:2] = bits
    got = ops.tree_attention(wide[..., 3:131], kc, vc, tab[:, ::2], cu, kv, both[:, 1:2], 0.1, meta=_meta(cu, kv, table))
    assert torch.equal(got, want)
    more = ops.tree_attention(torch.cat([q, q[:3]]), kc, vc, table.cuda(), cu, kv, torch.cat([bits, bits[:3]]), 0.1)
    assert torch.equal(more[:13], want) and not bool(more[13:].any())
    padded = torch.cat([flat, flat[:3]]).cuda()
    for meta in (None, _meta(cu, kv, table)):             # rows behind the last sequence
        m, p = ops.tree_mask(padded, cu, kv, meta)
        assert torch.equal(m[:13], bits) and not bool(m[13:].any()) and not bool(p[13:].any())
        more = ops.tree_attention(torch.cat([q, q[:3]]), kc, vc, table.cuda(), cu, kv, m, 0.1, meta=meta)
        assert torch.equal(more[:13], want) and not bool(more[13:].any())
    emitted, path, count = ops.tree_accept(padded, padded, padded, cu, kv)
    assert emitted.shape == (2, 9) and count.shape == (2,)
    _ok()


def test_lengths_and_blocks_that_cannot_be_are_reported():
    from xfastertransformer_b200.ops import native as N
    q = torch.randn(4, 4, 128, device="cuda").bfloat16()
    c = torch.randn(2, 2, 64, 128, device="cuda").bfloat16()
    bits = torch.full((4, 1), 15, device="cuda")
    for table, kv in ((torch.tensor([[0, 7]]), 100), (torch.tensor([[0, -1]]), 100), (torch.tensor([[0, 1]]), 500)):
        ops.tree_attention(q, c, c, table.int().cuda(), [0, 4], [kv], bits, 0.1)
        with pytest.raises(N.KernelError):
            N.Workspace.get(torch.device("cuda", 0)).check_status()
    with pytest.raises(N.KernelError):
        ops.tree_attention(q.float(), c.float(), c.float(), table.int().cuda(), [0, 4], [100], bits, 0.1)
    with pytest.raises(N.KernelError):
        ops.tree_attention(q[..., :32].contiguous(), c[..., :32].contiguous(), c[..., :32].contiguous(), table.int().cuda(), [0, 4], [100], bits, 0.1)


# -- sampling -------------------------------------------------------------------------------------------------------
def _limits(rnd, rows, V):
    f = lambda *v: torch.tensor([rnd.choice(v) for _ in range(rows)], dtype=torch.float32)
    return (f(0.0, 0.3, 0.7, 1.0, 1.8, -1.0), torch.tensor([rnd.choice([0, -1, 1, 2, 40, 1000, V // 2, V, V + 5]) for _ in range(rows)], dtype=torch.int32),
            f(0.0, 0.1, 0.5, 0.9, 0.99, 1.0, 2.0), f(0.0, 0.0, 0.0, 0.01, 0.2, 1.0, 3.0))


@pytest.mark.parametrize("V", [1, 2, 31, 1000, 1025, 32000, 50257, 151936, 262147])
@pytest.mark.parametrize("kind", ["normal", "peaked", "ties", "bf16"])
def test_sampling(V, kind):
    g = torch.Generator().manual_seed(V)
    rnd = random.Random(V)
    rows = 24 if V < 100000 else 12
    x = 2.5 * torch.randn(rows, V, generator=g)
    if kind == "peaked":
        x = 4 * x + 30 * (torch.rand(rows, V, generator=g) < 20 / V)
    if kind == "ties":
        x = x.round()
    if kind == "bf16":
        x = x.bfloat16()
    u = torch.rand(rows, generator=g)
    u[0], u[-1] = 0.0, 1.0 - 2.0 ** -24
    args = _limits(rnd, rows, V) if rows > 1 else _limits(rnd, 1, V)
    want = R.sample(x, *args, u)
    got = ops.sample(x.cuda(), *(a.cuda() for a in args), u.cuda())
    assert got.dtype is torch.int64 and torch.equal(got.cpu(), want)


def test_one_number_for_all_rows_and_other_shapes():
    g = torch.Generator().manual_seed(0)
    x, u = torch.randn(3, 4, 500, generator=g), torch.rand(12, generator=g)
    want = R.sample(x, 0.8, 30, 0.9, 0.01, u)
    assert want.shape == (3, 4)
    assert torch.equal(ops.sample(x.cuda(), 0.8, 30, 0.9, 0.01, u.cuda()).cpu(), want)
    wide = torch.zeros(12, 600, device="cuda")
    wide[:, 3:503] = x.view(12, 500).cuda()
    assert torch.equal(ops.sample(wide[:, 3:503], torch.full((12,), 0.8), 30, torch.tensor([0.9]), 0.01, u).cpu(), want.view(-1))
    for n in (1, 2, 3):                                    # bf16 rows that start anywhere in 8 bytes
        wide = torch.zeros(12, 507, device="cuda", dtype=torch.bfloat16)
        wide[:, n:n + 500] = x.view(12, 500).bfloat16().cuda()
        assert torch.equal(ops.sample(wide[:, n:n + 500], 0.8, 30, 0.9, 0.01, u.cuda()).cpu(), R.sample(x.view(12, 500).bfloat16(), 0.8, 30, 0.9, 0.01, u))
    turned = x.view(12, 500).cuda().t().contiguous().t()
    assert torch.equal(ops.sample(turned, 0.8, 30, 0.9, 0.01, u.cuda()).cpu(), want.view(-1))
    assert ops.sample(x[:0].cuda(), 0.8, 30, 0.9, 0.01, u[:0].cuda()).shape == (0, 4)


def test_odd_logits():
    inf, nan = math.inf, math.nan
    x = torch.tensor([[-inf, -inf, -inf], [nan, -inf, 1.0], [inf, 0.0, inf], [nan, nan, nan], [-0.0, 0.0, -1.0], [3.0, 3.0, 3.0],
                      [1e-45, 0.0, 2e-45], [3e38, -3e38, 3.4e38], [-inf, -7.0, -inf]])
    for T in (1.0, 0.0, 1e-30, 1e30, inf, nan, 1e-45):
        for k, p, m in ((0, 1.0, 0.0), (2, 1.0, 0.0), (0, 0.5, 0.0), (0, 1.0, 1.0), (0, nan, nan)):
            for u in (0.0, 0.3, 0.5, 0.9, 1.0, nan, -1.0):
                want = R.sample(x, T, k, p, m, torch.full((9,), u))
                got = ops.sample(x.cuda(), T, k, p, m, torch.full((9,), u, device="cuda"))
                assert torch.equal(got.cpu(), want), (T, k, p, m, u)


@pytest.mark.parametrize("V", [4096, 32000, 151936])
def test_all_logits_equal(V):
    u = torch.rand(16, generator=torch.Generator().manual_seed(V))
    x = torch.full((16, V), 1.25)
    for k, p in ((0, 1.0), (0, 0.5), (V - 7, 0.25), (1500, 1.0)):
        assert torch.equal(ops.sample(x.cuda(), 1.0, k, p, 0.0, u.cuda()).cpu(), R.sample(x, 1.0, k, p, 0.0, u))


@pytest.mark.parametrize("V,width", [(20000, 0.02), (151936, 0.05), (200003, 0.3), (100000, 1e-6), (1 << 21, 0.01)])
def test_crowded_logits(V, width):
    g = torch.Generator().manual_seed(V)
    rows = 14 if V < 1 << 20 else 3
    x = 5 + width * torch.randn(rows, V, generator=g)
    u = torch.rand(rows, generator=g)
    for T, k, p, m in ((1.0, 0, 1.0, 0.0), (2.5, 0, 0.6, 0.0), (0.8, 5000, 0.9, 0.0), (1.3, V // 2, 1.0, 0.0), (0.02, 0, 0.7, 0.3), (1.0, 700, 0.5, 0.0)):
        assert torch.equal(ops.sample(x.cuda(), T, k, p, m, u.cuda()).cpu(), R.sample(x, T, k, p, m, u)), (T, k, p, m)


@pytest.mark.parametrize("masked", [-math.inf, torch.finfo(torch.float32).min, -1e4])
@pytest.mark.parametrize("V", [1000, 128256])
def test_rows_that_are_masked_but_for_a_few(V, masked):
    g = torch.Generator().manual_seed(V)
    x = torch.full((16, V), masked)
    for r in range(16):
        x[r, torch.randperm(V, generator=g)[:r + 1]] = 3 * torch.randn(r + 1, generator=g)
    u = torch.rand(16, generator=g)
    for T in (0.5, 1.0, 1.9, 2.5):
        for k, p, m in ((50, 1.0, 0.0), (50, 0.9, 0.0), (900, 0.7, 0.05), (5000, 0.9, 0.0), (5000, 1.0, 0.2), (0, 0.9, 0.0), (0, 1.0, 0.1), (3, 1.0, 0.0)):
            assert torch.equal(ops.sample(x.cuda(), T, k, p, m, u.cuda()).cpu(), R.sample(x, T, k, p, m, u)), (T, k, p, m)


def test_many_rows_of_a_wide_vocabulary():
    g = torch.Generator(device="cuda").manual_seed(4)
    x = 0.01 * torch.randn(160, 300001, generator=g, device="cuda")         # one bin: a slice's sums stay whole
    u = torch.rand(160, generator=g, device="cuda")
    got = ops.sample(x, 1.0, 0, 1.0, 0.0, u).cpu()
    few = [0, 1, 77, 159]
    assert torch.equal(got[few], R.sample(x[few].cpu(), 1.0, 0, 1.0, 0.0, u[few].cpu()))
    assert torch.equal(ops.sample(x[:1], 1e39, 0, 1.0, 0.0, u[:1]).cpu(), R.sample(x[:1].cpu(), 1e39, 0, 1.0, 0.0, u[:1].cpu()))


@pytest.mark.parametrize("T", [1e-6, 1e-4, 2e-3, 0.02])
def test_low_temperatures(T):
    g = torch.Generator().manual_seed(8)
    x = 3 * torch.randn(20, 50257, generator=g)
    x[::2] = (200 * x[::2]).round() / 200                  # largest logits that come more than once, or nearly
    x[3, :9000] = x[3].max()
    u = torch.rand(20, generator=g)
    for k, p, m in ((0, 1.0, 0.0), (0, 0.9, 0.1), (3, 0.5, 0.0), (0, 1.0, 0.5)):
        assert torch.equal(ops.sample(x.cuda(), T, k, p, m, u.cuda()).cpu(), R.sample(x, T, k, p, m, u)), (k, p, m)


def test_frequencies():
    w = torch.tensor([0.5, 0.25, 0.125, 0.125])
    n = 4096
    u = (torch.arange(n) + 0.5) / n                        # every place of the distribution once
    got = ops.sample(w.log().expand(n, 4).cuda(), 1.0, 0, 1.0, 0.0, u.cuda())
    assert torch.bincount(got.cpu(), minlength=4).tolist() == [2048, 1024, 512, 512]


# -- accepted paths -------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("bs,D,dtype", [(64, 128, torch.bfloat16), (64, 64, torch.int8), (16, 6, torch.bfloat16), (128, 256, torch.float32)])
@pytest.mark.parametrize("seed", range(3))
def test_accepted_paths(seed, bs, D, dtype):
    rnd = random.Random(seed)
    lens = [(rnd.randrange(1, 40), rnd.randrange(0, 200)) for _ in range(9)] + [(0, 3), (256, 1)]
    trees, flat, cu, kv, table, blocks = batch(lens, seed, bs)
    tokens = torch.tensor([rnd.randrange(3) for _ in range(cu[-1])])
    sampled = torch.tensor([rnd.randrange(3) for _ in range(cu[-1])])
    g = torch.Generator().manual_seed(seed)
    make = lambda *s: torch.randint(-100, 100, s, generator=g).to(dtype)
    k, v = ([make(blocks, h, bs, D) for h in (2, 3, 1)] for _ in range(2))
    ks = [torch.randn(blocks, h, bs, generator=g) for h in (2, 3, 1)]
    v[1] = None                                            # a layer of latents has no values
    host = [p for p in k + v + ks if p is not None]
    dev = [[None if p is None else p.cuda() for p in x] for x in (k, v, ks)]
    pools = ops.cache_pools(dev[0], dev[1], dev[2], None)
    got = ops.tree_accept(tokens.cuda(), flat.cuda(), sampled.int().cuda(), cu, kv, table.cuda(), pools, meta=_meta(cu, kv, table))
    want = R.tree_accept(tokens, flat, sampled, cu, kv, table, host)
    for a, b in zip(got, want):
        assert torch.equal(a.cpu(), b)
    for a, b in zip([p for x in dev for p in x if p is not None], host):
        assert torch.equal(a.cpu(), b)
    again = ops.tree_accept(tokens.cuda(), flat.cuda(), sampled.cuda(), cu, kv)
    assert torch.equal(again[1].cpu(), want[1])
    _ok()


def test_a_long_chain_moves_over_itself():
    n = 200                                                # node 1 is no part of the path: every row behind it moves by one
    parents = torch.tensor([-1, 0, 0] + list(range(2, n - 1)), dtype=torch.int32)
    tokens = torch.arange(n)
    sampled = torch.tensor([2, 0] + list(range(3, n + 1)))
    pool = torch.arange(8 * 64, dtype=torch.float32).view(8, 1, 64, 1).repeat(1, 2, 1, 4)
    table = torch.tensor([[5, 1, 6, 2]], dtype=torch.int32)
    dev = pool.cuda()
    got = ops.tree_accept(tokens.cuda(), parents.cuda(), sampled.cuda(), [0, n], [n + 30], table.cuda(), ops.cache_pools([dev]))
    want = R.tree_accept(tokens, parents, sampled, [0, n], [n + 30], table, [pool])
    assert int(got[2][0]) == n - 1 and torch.equal(got[0].cpu(), want[0]) and torch.equal(dev.cpu(), pool)


# -- all of them ----------------------------------------------------------------------------------------------------
def test_a_step_of_all_of_them():
    """Two sequences' trees over a cache: every node's output is that of a plain sequence of its ancestors, and after the step the caches
    hold what a program without trees would have in them."""
    from xfastertransformer_b200.runtime.kv_cache import PagedKVCache
    dev = torch.device("cuda", 0)
    hq, hkv, D, layers, V = 8, 2, 128, 3, 700
    rnd = random.Random(11)
    g = torch.Generator(device="cuda").manual_seed(11)
    ctx, nodes = [130, 61], [14, 9]
    trees = [parents_of(rnd, n) for n in nodes]
    cu, kv = [0, nodes[0], sum(nodes)], [c + n for c, n in zip(ctx, nodes)]
    table = R.rope_table(512, D).cuda()

    def cache():
        c = PagedKVCache(layers, hkv, D, D, "bf16", dev)
        c.ensure_blocks(16)
        for b in range(2):
            c.add_sequence(b)
        return c
    tree, plain = cache(), cache()
    past = [[(hq + 2 * hkv) * D, c] for c in ctx]
    for b, (w, n) in enumerate(past):                      # the same context in both
        for c in (tree, plain):
            c.append_slots(b, n)
        for l in range(layers):
            rows = torch.randn(n, w, generator=g, device="cuda").bfloat16()
            for c in (tree, plain):
                slots = torch.tensor([c.tables[b][p // 64] * 64 + p % 64 for p in range(n)], dtype=torch.int32, device=dev)
                ops.qkv_rope_cache(rows, hq, hkv, D, torch.arange(n, dtype=torch.int32, device=dev), table, D, "half", c.k[l], c.v[l], None, None,
                                   slots)
    flat = torch.tensor(trees[0] + trees[1], dtype=torch.int32, device=dev)
    mask, pos = ops.tree_mask(flat, cu, kv)
    slots = torch.tensor([s for b in range(2) for s in tree.append_slots(b, nodes[b])], dtype=torch.int32, device=dev)
    bt = tree.block_table([0, 1]).to(dev)
    qkv = [torch.randn(cu[-1], (hq + 2 * hkv) * D, generator=g, device="cuda").bfloat16() for _ in range(layers)]
    outs = []
    for l in range(layers):
        q = ops.qkv_rope_cache(qkv[l], hq, hkv, D, pos, table, D, "half", tree.k[l], tree.v[l], None, None, slots)
        outs.append(ops.tree_attention(q, tree.k[l], tree.v[l], bt, cu, kv, mask, D ** -0.5))
    head = 0.3 * torch.randn(hq * D, V, generator=g, device="cuda")
    logits = outs[-1].float().view(cu[-1], -1) @ head
    u = torch.rand(cu[-1], generator=g, device="cuda")
    sampled = ops.sample(logits, 0.7, 20, 0.95, 0.02, u)
    tokens = torch.randint(0, V, (cu[-1],), generator=g, device="cuda")
    for b in range(2):                                     # drafts that agree for a while
        at = 0
        for _ in range(3):
            kids = [i for i in range(nodes[b]) if trees[b][i] == at]
            if not kids:
                break
            at = kids[-1]
            tokens[cu[b] + at] = sampled[cu[b] + trees[b][at]]
    emitted, path, count = ops.tree_accept(tokens, flat, sampled, cu, kv, bt, tree.pools())
    assert torch.equal(sampled.cpu(), R.sample(logits.cpu(), 0.7, 20, 0.95, 0.02, u.cpu()))
    for b in range(2):
        line = [i for i in path[b].tolist() if i >= 0]
        assert len(line) == int(count[b]) >= 2 and line == list(reversed(ancestors(trees[b], line[-1])))
        tree.truncate(b, ctx[b] + len(line))
        rows = torch.tensor([cu[b] + i for i in line], device=dev)
        s2 = torch.tensor(plain.append_slots(b, len(line)), dtype=torch.int32, device=dev)
        p2 = torch.arange(ctx[b], ctx[b] + len(line), dtype=torch.int32, device=dev)
        n = ctx[b] + len(line)
        a, z = (torch.tensor([c.tables[b][p // 64] * 64 + p % 64 for p in range(n)], device=dev) for c in (tree, plain))
        for l in range(layers):
            q = ops.qkv_rope_cache(qkv[l][rows], hq, hkv, D, p2, table, D, "half", plain.k[l], plain.v[l], None, None, s2)
            out = ops.paged_attention(q, plain.k[l], plain.v[l], plain.block_table([b]).to(dev), [0, len(line)], [n], D ** -0.5)
            # both round weights (twice: the sum too) and the result once, of values up to 6 in size
            assert float((out.float() - outs[l][rows].float()).abs().max()) <= 2 * 3 * BF16 * 6
            for x, y in ((tree.k[l], plain.k[l]), (tree.v[l], plain.v[l])):
                assert torch.equal(x.transpose(1, 2).reshape(-1, hkv, D)[a], y.transpose(1, 2).reshape(-1, hkv, D)[z])
    _ok()


def test_captured_and_on_another_stream():
    g = torch.Generator(device="cuda").manual_seed(3)
    lens = [(12, 1500), (7, 300)]
    _, flat, cu, kv, table, blocks = batch(lens, 2)
    dev = lambda t: t.cuda()
    kc, vc = (torch.randn(blocks, 2, 64, 128, generator=g, device="cuda").bfloat16() for _ in range(2))
    q = torch.randn(19, 8, 128, generator=g, device="cuda").bfloat16()
    x, u = 3 * torch.randn(19, 32000, generator=g, device="cuda"), torch.rand(19, generator=g, device="cuda")
    tokens = torch.randint(0, 3, (19,), generator=g, device="cuda")
    up, bt, meta = dev(flat), dev(table), _meta(cu, kv, table)
    pools = ops.cache_pools([kc], [vc])

    def step():
        mask, pos = ops.tree_mask(up, cu, kv, meta)
        o = ops.tree_attention(q, kc, vc, bt, cu, kv, mask, 0.09, meta=meta)
        s = ops.sample(x, 0.9, 0, 0.9, 0.0, u)
        return mask, pos, o, s, *ops.tree_accept(tokens, up, s % 3, cu, kv, meta=meta)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = step()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):                                     # two graphs of the same step, replayed side by side
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step()
        graphs.append((graph, outs))
    for t, n in ((q, None), (x, None), (u, None)):
        t.copy_(torch.rand(t.shape, generator=g, device="cuda") if t is u else torch.randn(t.shape, generator=g, device="cuda"))
    want = step()
    assert not torch.equal(want[2], first[2])
    streams = [torch.cuda.Stream() for _ in graphs]
    torch.cuda.synchronize()
    for _ in range(3):
        for (graph, _), st in zip(graphs, streams):
            with torch.cuda.stream(st):
                graph.replay()
    torch.cuda.synchronize()
    for _, outs in graphs:
        for a, b in zip(outs, want):
            assert torch.equal(a, b)
    del pools
    _ok()
