"""Operators of a step with trees of drafted tokens on a GPU, at the edges of what they take."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from tree_cases import batch, caches
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


@pytest.mark.parametrize("rows", [3, 50, 100])                # 8, 4 and 2 CTAs a row
@pytest.mark.parametrize("T", [0.0, 0.8])
def test_clusters_of_short_rows_beside_other_work(rows, T):
    g = torch.Generator().manual_seed(rows)
    x, u = 3 * torch.randn(rows, 5000, generator=g), torch.rand(rows, generator=g)
    want = R.sample(x, T, 30, 0.9, 0.02, u)
    x, u, a = x.cuda(), u.cuda(), torch.randn(1024, 1024, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    outs = []
    for _ in range(30):
        with torch.cuda.stream(side):
            a = torch.tanh(a @ a)
        outs.append(ops.sample(x, T, 30, 0.9, 0.02, u))
    torch.cuda.synchronize()
    for got in outs:
        assert torch.equal(got.cpu(), want)


def test_a_pool_that_several_layers_read_moves_once():
    from test_tree_edges_cpu import chain_with_gaps
    pools = [torch.arange(64.0, device="cuda").view(1, 1, 64, 1).repeat(1, 2, 1, 128).bfloat16() for _ in range(3)]
    handle = ops.cache_pools([pools[i % 3] for i in range(80)])
    *_, count = ops.tree_accept(*chain_with_gaps("cuda"), handle)
    assert int(count[0]) == 4
    for p in pools:
        assert p[0, 1, 10:14, 5].tolist() == [10, 12, 14, 15]
    _ok()


def test_a_graph_captured_before_its_cache_grew_moves_nothing():
    from test_tree_edges_cpu import chain_with_gaps
    from xfastertransformer_b200.runtime.kv_cache import PagedKVCache
    c = PagedKVCache(3, 2, 128, 128, "bf16", torch.device("cuda", 0))
    c.ensure_blocks(2)
    pools, args = c.pools(), chain_with_gaps("cuda")
    meta = _meta(args[3], args[4], args[5])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        assert c.pools() is pools                         # (made already: nothing waits here)
        count = ops.tree_accept(*args, pools, meta=meta)[2]
    fill = torch.arange(64.0, device="cuda").bfloat16()[:, None]
    for l in range(3):
        c.k[l][0, :] = fill
    graph.replay()
    assert int(count[0]) == 4 and all(k[0, 1, 10:14, 7].tolist() == [10, 12, 14, 15] for k in c.k)
    old = c.k[2]                                          # (held, so that what a late move would write can be seen)
    c.ensure_blocks(64)
    for k in (old, *c.k):
        k[0, :] = fill
    graph.replay()
    torch.cuda.synchronize()
    assert int(count[0]) == 4 and all(k[0, 1, 10:14, 7].tolist() == [10, 11, 12, 13] for k in (old, *c.k))
    _ok()


def test_parents_beyond_32_bits():
    from xfastertransformer_b200.ops import native as N
    up = torch.tensor([-2 ** 40, 0, -2 ** 32, 1, -2 ** 32 + 1])
    cu, kv = [0, 5], [9]
    mask, pos = ops.tree_mask(up.cuda(), cu, kv)
    want = R.tree_mask(up, cu, kv)
    assert torch.equal(mask.cpu(), want[0]) and torch.equal(pos.cpu(), want[1])
    tokens, sampled = torch.zeros(5, dtype=torch.long), torch.zeros(5, dtype=torch.long)
    for a, b in zip(ops.tree_accept(tokens.cuda(), up.cuda(), sampled.cuda(), cu, kv), R.tree_accept(tokens, up, sampled, cu, kv)):
        assert torch.equal(a.cpu(), b)
    _ok()
    mask, _ = ops.tree_mask(torch.tensor([-1, 2 ** 32, 1], device="cuda"), [0, 3], [3])
    assert mask[:, 0].tolist() == [1, 2, 6]               # reported, and taken as a root
    with pytest.raises(N.KernelError):
        N.Workspace.get(torch.device("cuda", 0)).check_status()


# -- attention --------------------------------------------------------------------------------------------------------
def _close(got, q, kc, vc, table, cu, kv, bits, scale, ks=None, vs=None, **kw):
    """`got` against 64 bits.  A weight is rounded to bf16 once, 2^-8 of it; the sum that divides has the rounded weights (the same again) or
    the whole ones; the result is rounded to bf16.  Scores in 32 bits: D + 8 roundings of 2^-24 of sums of |q k| <= |q| |k|, which move a weight
    and the denominator by as much; 2^-12: exponentials and divisions, far below."""
    f64 = torch.float64
    args = (table, cu, kv, bits, scale, ks, vs)
    want = R.tree_attention(q, kc, vc, *args, dtype=f64, **kw)
    size = R.tree_attention(q, kc, vc.abs(), *args, dtype=f64, **kw)
    k = kc.double() * (1.0 if ks is None else ks.double()[..., None])
    norms = float(q.double().norm(dim=-1).max()) * float(k.nan_to_num(0, 0, 0).norm(dim=-1).max())
    score = 2 * (q.shape[2] + 8) * 2.0 ** -24 * norms * abs(scale)
    bound = (2 * BF16 + score + 2.0 ** -12) * size + BF16 * 1.02 * want.abs() + 1e-30
    err = (got.double().cpu() - want).abs()
    assert bool((err <= bound).all()), (float((err / bound.clamp_min(1e-20)).max()), float(err.max()))


def _where(table, p, bs):
    return int(table[p // bs]), p % bs


HEADS = [(64, 64, False), (128, 64, False), (256, 64, False), (128, 16, False), (128, 64, True), (64, 64, True), (256, 192, True)]


@pytest.mark.parametrize("D,bs,int8", HEADS)
@pytest.mark.parametrize("window,keep", [(7, 0), (100, 5), (64, 64), (130, 70), (1, 0), (1000, 3)])
@pytest.mark.parametrize("spoil", [math.nan, math.inf])
def test_values_that_a_window_leaves_to_no_node(D, bs, int8, window, keep, spoil):
    lens = [(9, 300), (4, 0), (17, 64), (1, 700), (70, 130)]
    g = torch.Generator().manual_seed(D + window)
    _, flat, cu, kv, table, blocks = batch(lens, D + window, bs)
    kc, vc, ks, vs = caches(g, blocks, 2, D, bs, int8)
    q = torch.randn(cu[-1], 6, D, generator=g).bfloat16()
    bits, pos = R.tree_mask(flat, cu, kv)
    hidden = 0
    for b, (n, c) in enumerate(lens):
        first = int(pos[cu[b]:cu[b + 1]].min()) - window + 1
        for p in range(c):
            if p < first and p >= keep:
                blk, off = _where(table[b], p, bs)
                for t in (ks, vs) if int8 else (kc, vc):
                    t[blk, :, off] = spoil
                hidden += 1
    assert hidden > 0 or window == 1000
    c = lambda t: None if t is None else t.cuda()
    got = ops.tree_attention(c(q), c(kc), c(vc), c(table), cu, kv, c(bits), D ** -0.5, c(ks), c(vs), window=window, keep_first=keep,
                             positions=c(pos), meta=_meta(cu, kv, table))
    _ok()
    assert bool(torch.isfinite(got).all())
    _close(got, q, kc, vc, table, cu, kv, bits, D ** -0.5, ks, vs, group=3, window=window, keep_first=keep, positions=pos)


@pytest.mark.parametrize("D,bs,int8", HEADS)
@pytest.mark.parametrize("ctx", [0, 3, 61, 200])
def test_nodes_that_only_the_window_hides(D, bs, int8, ctx):
    n, window = 70, 3
    g = torch.Generator().manual_seed(D + ctx)
    _, _, cu, kv, table, blocks = batch([(n, ctx)], 4, bs)
    kc, vc, ks, vs = caches(g, blocks, 2, D, bs, int8)
    q = torch.randn(n, 6, D, generator=g).bfloat16()
    bits = torch.full((n, 2), -1, dtype=torch.int64)       # every node sees every one, but for the window
    bits[[5, 66]] = 0                                      # these two see none, themselves neither
    for j in (5, 66):
        blk, off = _where(table[0], ctx + j, bs)
        for t in (ks, vs) if int8 else (kc, vc):
            t[blk, :, off] = math.nan
    c = lambda t: None if t is None else t.cuda()
    for keep in (0, 2):
        pos = ctx + 10 + torch.arange(n, dtype=torch.int32) // 2
        pos[[5, 66]] = keep                                # far behind all others, and not among the kept ones
        got = ops.tree_attention(c(q), c(kc), c(vc), c(table), cu, kv, c(bits), D ** -0.5, c(ks), c(vs), window=window, keep_first=keep,
                                 positions=c(pos), meta=_meta(cu, kv, table))
        _ok()
        assert bool(torch.isfinite(got).all())
        _close(got, q, kc, vc, table, cu, kv, bits, D ** -0.5, ks, vs, group=3, window=window, keep_first=keep, positions=pos)


@pytest.mark.parametrize("D,bs,int8", HEADS)
@pytest.mark.parametrize("gain", [0.01, 30.0])                 # scores far below the cap, and far above it
@pytest.mark.parametrize("kw", [{}, {"softcap": 5.0}, {"softcap": 5.0, "sinks": True}])
def test_a_key_that_is_not_a_number_makes_its_rows_so(D, bs, int8, gain, kw):
    g = torch.Generator().manual_seed(D)
    _, flat, cu, kv, table, blocks = batch([(9, 300), (12, 40)], 6, bs)
    kc, vc, ks, vs = caches(g, blocks, 2, D, bs, int8)
    q = (gain * torch.randn(cu[-1], 6, D, generator=g)).bfloat16()
    bits, _ = R.tree_mask(flat, cu, kv)
    seen = [torch.ones(9, dtype=torch.bool), (bits[9:, 0] >> 4 & 1).bool()]
    for b, p in ((0, 77), (1, 40 + 4)):                    # a key of the context, and one that a branch sees
        blk, off = _where(table[b], p, bs)
        (ks if int8 else kc)[blk, 1, off] = math.nan       # of one head
    kw = dict(kw, sinks=torch.randn(6, generator=g)) if "sinks" in kw else kw
    c = lambda t: t.cuda() if isinstance(t, torch.Tensor) else t
    got = ops.tree_attention(c(q), c(kc), c(vc), c(table), cu, kv, c(bits), 0.3, c(ks), c(vs), meta=_meta(cu, kv, table),
                             **{n: c(v) for n, v in kw.items()}).cpu()
    _ok()
    assert 0 < int(seen[1].sum()) < 12
    assert bool(torch.isfinite(got[:, :3]).all())
    assert torch.equal(torch.isnan(got[:, 3:]).all(-1).all(-1), torch.cat(seen)) and bool(torch.isfinite(got[:, 3:][~torch.cat(seen)]).all())


@pytest.mark.parametrize("lens", [[(9, 40), (4, 70)], [(9, 9000), (4, 70)], [(1, 3)]])         # (the second: several slices, joined)
@pytest.mark.parametrize("bs", [16, 64])
@pytest.mark.parametrize("with_meta", [False, True])
def test_rows_in_front_of_the_first_sequence(lens, bs, with_meta):
    g = torch.Generator().manual_seed(bs)
    _, flat, cu, kv, table, blocks = batch(lens, 3, bs)
    kc, vc, _, _ = caches(g, blocks, 2, 128, bs)
    q = torch.randn(cu[-1] + 8, 8, 128, generator=g).bfloat16().cuda()
    kc, vc, table = kc.cuda(), vc.cuda(), table.cuda()
    n, up = cu[-1], torch.cat([torch.full((5,), 7, dtype=torch.int32), flat, torch.full((3,), 7, dtype=torch.int32)]).cuda()
    later = [x + 5 for x in cu]
    meta = _meta(later, kv, table) if with_meta else None
    want, want_pos = ops.tree_mask(flat.cuda(), cu, kv)
    for _ in range(4):
        torch.full((1 << 22,), math.nan, device="cuda")    # what a fresh output may find in its memory
        mask, pos = ops.tree_mask(up, later, kv, meta)
        assert torch.equal(mask[5:n + 5], want) and torch.equal(pos[5:n + 5], want_pos)
        assert not any(bool(t[rows].any()) for t in (mask, pos) for rows in (slice(0, 5), slice(n + 5, None)))
        got = ops.tree_attention(q, kc, vc, table, later, kv, mask, 0.1, meta=meta)
        assert torch.equal(got[5:n + 5], ops.tree_attention(q[5:n + 5].contiguous(), kc, vc, table, cu, kv, want, 0.1))
        assert not bool(got[:5].any()) and not bool(got[n + 5:].any())
    tokens = torch.zeros(n + 8, dtype=torch.long, device="cuda")
    _, path, count = ops.tree_accept(tokens, up, tokens, later, kv, meta=meta)
    assert torch.equal(path.cpu(), R.tree_accept(tokens.cpu(), up.cpu(), tokens.cpu(), later, kv)[1])
    _ok()


@pytest.mark.parametrize("hkv", [0, 2])
@pytest.mark.parametrize("ctx", [10, 9000])
def test_a_share_without_heads(hkv, ctx):
    _, _, cu, kv, table, blocks = batch([(9, ctx)], 3)
    q, c = torch.zeros(9, 0, 128, device="cuda").bfloat16(), torch.zeros(blocks, hkv, 64, 128, device="cuda").bfloat16()
    bits = torch.ones(9, 1, dtype=torch.int64, device="cuda")
    assert ops.tree_attention(q, c, c, table.cuda(), cu, kv, bits, 0.1).shape == (9, 0, 128)
    assert torch.ones(3, device="cuda").sum().item() == 3   # no error is left behind
    _ok()


def test_more_sequences_than_a_grid_has_rows():
    from xfastertransformer_b200.ops import native as N
    B = 65536
    cu, kv = list(range(B + 1)), [1] * B
    up, tokens = torch.full((B,), -1, dtype=torch.int32, device="cuda"), torch.zeros(B, dtype=torch.long, device="cuda")
    mask, pos = ops.tree_mask(up, cu, kv)
    assert bool((mask == 1).all()) and not bool(pos.any())
    c, table = torch.ones(1, 1, 64, 64, device="cuda").bfloat16(), torch.zeros(B, 1, dtype=torch.int32, device="cuda")
    q = torch.zeros(B, 1, 64, device="cuda").bfloat16()
    for f in (lambda: ops.tree_accept(tokens, up, tokens, cu, kv), lambda: ops.tree_attention(q, c, c, table, cu, kv, mask, 0.1)):
        with pytest.raises(N.KernelError):
            f()
        assert torch.ones(3, device="cuda").sum().item() == 3           # no error is left behind
    count = ops.tree_accept(tokens[1:], up[1:], tokens[1:], cu[:-1], kv[1:])[2]
    assert bool((count == 1).all())
    assert bool((ops.tree_attention(q[1:], c, c, table[1:], cu[:-1], kv[1:], mask[1:], 0.1) == 1).all())
    _ok()


# -- sampling ---------------------------------------------------------------------------------------------------------
def test_limits_beyond_32_bits():
    g = torch.Generator().manual_seed(6)
    x, u = torch.randn(8, 500, generator=g), torch.rand(8, generator=g)
    k = torch.tensor([2 ** 32 + 5, 2 ** 31, 2 ** 31 - 1, -2 ** 31 - 1, -2 ** 32 + 3, 5, 2 ** 62, -2 ** 63])
    want = R.sample(x, 1.0, k, 1.0, 0.0, u)
    assert torch.equal(ops.sample(x.cuda(), 1.0, k.cuda(), 1.0, 0.0, u.cuda()).cpu(), want)
    for n in k.tolist():
        for one in (n, torch.tensor(n), torch.tensor([n], device="cuda")):
            assert torch.equal(ops.sample(x.cuda(), 1.0, one, 1.0, 0.0, u.cuda()).cpu(), R.sample(x, 1.0, n, 1.0, 0.0, u))


def _equal_rows(n, k, p, u):
    """Place of the token in a row of n equal logits, in whole numbers: the first ceil(p min(k, n)), of them the one behind a share u."""
    from fractions import Fraction
    n = min(k, n) if k > 0 else n
    if p < 1:
        n = max(1, math.ceil(Fraction(p) * n))
    return int(Fraction(u) * n)


@pytest.mark.parametrize("n", [1, 2, 3, 8, 100, 128, 1000, 1024, 1536, 2048, 2049, 5000, 8192, 32000, 1 << 18])
@pytest.mark.parametrize("fill", [None, -math.inf, -1e4])      # nothing else in the row, or what weighs nothing
def test_equal_logits_at_the_borders_of_equal_shares(n, fill):
    u = torch.arange(0, 64) / 64.0
    u[-1] = 1 - 2.0 ** -24
    V = n if fill is None else 2 * n + 5
    for top in (1.25, -3.7, 0.0, 41.3):
        x = torch.full((64, V), top)
        at = torch.arange(n)
        if fill is not None:
            at = torch.randperm(V, generator=torch.Generator().manual_seed(n))[:n].sort().values
            x = torch.full((64, V), fill)
            x[:, at] = top
        x = x.cuda()
        for T, k, p, m in ((1.0, 0, 1.0, 0.0), (0.7, 0, 0.5, 0.0), (1.0, 0, 0.375, 0.2), (3.0, 0, 0.75, 0.0), (0.9, 0, 1.0, 0.5), (1.1, n // 2, 1.0, 0.0),
                           (0.6, n // 2, 0.5, 0.0), (1.3, 40, 0.25, 0.1), (0.01, 0, 0.5, 0.0), (1.0, 1600, 0.625, 0.0), (2.1, 1, 0.5, 0.0)):
            if T > 2 and fill == -1e4:
                continue
            got = ops.sample(x, T, k, p, m, u.cuda()).tolist()
            assert got == [int(at[_equal_rows(n, k, p, v)]) for v in u.tolist()], (top, T, k, p, m)
