"""Trees of drafted tokens on a CPU: masks, attention, accepted paths and sampling with limits of each row, and what they refuse."""
import math
import random

import pytest
import torch

from tree_cases import ancestors, batch, caches
from xfastertransformer_b200 import ops
from xfastertransformer_b200.ops import reference as R


@pytest.mark.parametrize("lens", [[(1, 0)], [(5, 3), (1, 9), (17, 64)], [(130, 2), (64, 1), (65, 0)], [(0, 5), (3, 5)]])
def test_mask_and_positions(lens):
    trees, flat, cu, kv, _, _ = batch(lens, 3, roots=2)
    mask, pos = ops.tree_mask(flat, cu, kv)
    assert mask.shape[1] == -(-max(n for n, _ in lens) // 64)
    for b, t in enumerate(trees):
        for i in range(len(t)):
            line = ancestors(t, i)
            got = {64 * w + j for w in range(mask.shape[1]) for j in range(64) if int(mask[cu[b] + i, w]) >> j & 1}
            assert got == set(line)
            assert int(pos[cu[b] + i]) == lens[b][1] + len(line) - 1


def test_chain_is_causal_attention():
    g = torch.Generator().manual_seed(1)
    lens = [(4, 70), (1, 3), (9, 0)]
    _, _, cu, kv, table, blocks = batch(lens, 4)
    flat = torch.tensor([i - 1 for n, _ in lens for i in range(n)], dtype=torch.int32)
    kc, vc, _, _ = caches(g, blocks, 2, 64)
    q = torch.randn(cu[-1], 6, 64, generator=g)
    mask, pos = ops.tree_mask(flat, cu, kv)
    for kw in ({}, {"softcap": 20.0}, {"window": 5, "keep_first": 2}, {"sinks": torch.randn(6, generator=g)}):
        want = R.paged_attention(q, kc, vc, table, cu, kv, 0.125, **kw)
        got = ops.tree_attention(q, kc, vc, table, cu, kv, mask, 0.125, positions=pos, **kw)
        torch.testing.assert_close(got, want, rtol=1e-5, atol=1e-5)


def test_every_node_is_the_end_of_its_own_sequence():
    g = torch.Generator().manual_seed(2)
    trees, flat, cu, kv, table, blocks = batch([(12, 67)], 5)
    kc, vc, ks, vs = caches(g, blocks, 2, 64, int8=True)
    q = torch.randn(12, 4, 64, generator=g)
    mask, _ = ops.tree_mask(flat, cu, kv)
    got = ops.tree_attention(q, kc, vc, table, cu, kv, mask, 0.125, ks, vs)
    for i in range(12):
        at = list(range(67)) + [67 + j for j in reversed(ancestors(trees[0], i))]
        blk, off = table[0, [p // 64 for p in at]].long(), torch.tensor([p % 64 for p in at])
        k1, v1 = (c[blk, :, off].transpose(0, 1)[None] for c in (kc, vc))
        s1, s2 = (c[blk, :, off].transpose(0, 1)[None] for c in (ks, vs))
        want = R.paged_attention(q[i:i + 1], k1, v1, torch.zeros(1, 1, dtype=torch.int32), [0, 1], [len(at)], 0.125, s1, s2)
        torch.testing.assert_close(got[i:i + 1], want, rtol=1e-5, atol=1e-5)


def test_nodes_that_see_nothing_and_values_that_no_one_sees():
    g = torch.Generator().manual_seed(3)
    kc, vc, _, _ = caches(g, 1, 1, 64)
    kc[0, 0, 1] = vc[0, 0, 1] = math.nan                  # seen by no node; so are the slots behind
    vc[0, 0, 3:] = math.inf
    q = torch.randn(3, 2, 64, generator=g)
    out = ops.tree_attention(q, kc, vc, torch.zeros(1, 1, dtype=torch.int32), [0, 3], [3], torch.tensor([[1], [0], [5]]), 0.1)
    assert torch.equal(out[1], torch.zeros(2, 64))
    torch.testing.assert_close(out[0], vc[0, 0, 0].float().expand(2, 64))
    assert bool(torch.isfinite(out).all())
    with_sinks = ops.tree_attention(q, kc, vc, torch.zeros(1, 1, dtype=torch.int32), [0, 3], [3], torch.tensor([[1], [0], [5]]), 0.1,
                                    sinks=torch.tensor([0.5, -1.0]))
    assert torch.equal(with_sinks[1], torch.zeros(2, 64))


@pytest.mark.parametrize("seed", range(6))
def test_accepted_path_and_its_rows(seed):
    rnd = random.Random(seed)
    lens = [(rnd.randrange(1, 20), rnd.randrange(0, 130)) for _ in range(5)] + [(0, 7)]
    trees, flat, cu, kv, table, blocks = batch(lens, seed)
    tokens = torch.tensor([rnd.randrange(3) for _ in range(cu[-1])])
    sampled = torch.tensor([rnd.randrange(3) for _ in range(cu[-1])])
    g = torch.Generator().manual_seed(seed)
    pools = [torch.randn(blocks, 2, 64, 4, generator=g), torch.randn(blocks, 2, 64, generator=g)]
    was = [p.clone() for p in pools]
    emitted, path, count = ops.tree_accept(tokens, flat, sampled, cu, kv, table, ops.cache_pools(pools[:1], ks=pools[1:]))
    for b, (t, (n, c)) in enumerate(zip(trees, lens)):
        line = [0] if n else []
        while line:
            fits = [i for i in range(n) if t[i] == line[-1] and tokens[cu[b] + i] == sampled[cu[b] + line[-1]]]
            if not fits:
                break
            line.append(min(fits))
        assert int(count[b]) == len(line)
        assert path[b].tolist() == line + [-1] * (path.shape[1] - len(line))
        assert emitted[b].tolist() == [int(sampled[cu[b] + i]) for i in line] + [-1] * (path.shape[1] - len(line))
        rows = lambda p, at: p[table[b, [x // 64 for x in at]].long(), :, torch.tensor([x % 64 for x in at], dtype=torch.long)]
        for p, w in zip(pools, was):
            at = list(range(c)) + [c + i for i in line]
            assert torch.equal(rows(p, range(c + len(line))), rows(w, at))


def _token(row, T, k, p, m, u):
    """The definition, one element after the other."""
    order = sorted(range(len(row)), key=lambda i: (-row[i], i))
    if not T > 0:
        return order[0]
    order = order[:k] if k > 0 else order
    w = [math.exp((row[i] - row[order[0]]) / T) for i in order]
    kept, before = [], 0.0
    for j, x in enumerate(w):
        if j and (p < 1 and not before < p * math.fsum(w) or x < m):
            break
        kept.append(x)
        before += x
    upto, total = 0.0, math.fsum(kept)
    for j, x in enumerate(kept):
        upto += x
        if upto > u * total:
            return order[j]
    return order[len(kept) - 1]


@pytest.mark.parametrize("V", [1, 2, 7, 200])
def test_sampling_is_its_definition(V):
    g = torch.Generator().manual_seed(V)
    rnd = random.Random(V)
    rows = 60
    x = 2 * torch.randn(rows, V, generator=g)
    x[::3] = x[::3].round()                               # equal logits
    f = lambda v: float(torch.tensor(v, dtype=torch.float32))
    T = [f(rnd.choice([0.0, 0.3, 1.0, 2.5])) for _ in range(rows)]
    k = [rnd.choice([0, 1, 3, 50, V + 1]) for _ in range(rows)]
    p = [f(rnd.choice([0.0, 0.4, 0.9, 1.0])) for _ in range(rows)]
    m = [f(rnd.choice([0.0, 0.05, 0.5, 1.0])) for _ in range(rows)]
    u = torch.rand(rows, generator=g)
    got = ops.sample(x, torch.tensor(T), torch.tensor(k), torch.tensor(p), torch.tensor(m), u).tolist()
    assert got == [_token(x[r].tolist(), T[r], k[r], p[r], m[r], float(u[r])) for r in range(rows)]


def test_sampling_of_odd_logits():
    inf, nan = math.inf, math.nan
    x = torch.tensor([[-inf, -inf, -inf], [nan, -inf, 1.0], [inf, 0.0, inf], [nan, nan, nan], [-0.0, 0.0, -1.0], [3.0, 3.0, 3.0]])
    pick = lambda u, **kw: ops.sample(x, kw.get("T", 1.0), 0, 1.0, 0.0, torch.tensor([u])).tolist()
    assert pick(0.0) == [-1, 2, 0, -1, 0, 0]
    assert pick(1.0) == [-1, 2, 2, -1, 2, 2]              # a number that is not below one counts as the last one that is
    assert pick(0.5) == [-1, 2, 2, -1, 1, 1]
    assert pick(0.9, T=0.0) == [-1, 2, 0, -1, 0, 0]
    assert pick(0.4, T=inf) == [-1, 2, 0, -1, 1, 1]


def test_the_server_samples_with_min_p():
    from types import SimpleNamespace
    from serving.openai_server import Request, Scheduler
    row = 3 * torch.randn(50, generator=torch.Generator().manual_seed(1))
    pick = lambda seed, **kw: Scheduler._pick(SimpleNamespace(torch=torch), Request([1], 4, 0.8, kw.pop("top_p", 0.9), 20, [], seed, **kw), row)
    assert {pick(s, min_p=1.0) for s in range(20)} == {int(row.argmax())}
    for s in range(20):
        u = torch.rand(1, generator=torch.Generator().manual_seed(s))
        assert pick(s, min_p=0.05) == int(ops.sample(row[None], 0.8, 20, 0.9, 0.05, u))
    assert len({pick(s, top_p=1.0) for s in range(40)}) > 1 and pick(3) == pick(3)


def test_refusals():
    z = torch.zeros
    up = z(4, dtype=torch.int32) - 1
    bad = [
        lambda: ops.tree_mask(up.float(), [0, 4], [9]),
        lambda: ops.tree_mask(up, [0, 5], [9]),
        lambda: ops.tree_mask(up, [0, 4], [3]),
        lambda: ops.tree_mask(up, [0, 4], [9, 9]),
        lambda: ops.tree_mask(torch.arange(4, dtype=torch.int32), [0, 4], [9]),
        lambda: ops.tree_mask(z(300, dtype=torch.int32), [0, 300], [400]),
        lambda: ops.sample(z(2, 0), 1.0, 0, 1.0, 0.0, z(2)),
        lambda: ops.sample(z(1).expand(1, (1 << 21) + 1), 1.0, 0, 1.0, 0.0, z(1)),
        lambda: ops.sample(z(2, 5, dtype=torch.int32), 1.0, 0, 1.0, 0.0, z(2)),
        lambda: ops.sample(z(2, 5), z(3), 0, 1.0, 0.0, z(2)),
        lambda: ops.sample(z(2, 5), 1.0, 0, 1.0, 0.0, 0.5),
        lambda: ops.tree_accept(up.long(), up, up[:3], [0, 4], [9]),
        lambda: ops.tree_accept(up.long(), up, up.float(), [0, 4], [9]),
        lambda: ops.tree_accept(up.long(), up, up, [0, 4], [9], None, ops.cache_pools([z(1, 1, 64, 4)])),
        lambda: ops.cache_pools([]),
        lambda: ops.cache_pools([z(1, 1, 64, 4)], [z(2, 1, 64, 4)]),
        lambda: ops.cache_pools([z(1, 2, 64, 4).transpose(1, 2)]),
        lambda: ops.cache_pools([z(1, 1, 64, 3, dtype=torch.int8)]),
    ]
    for f in bad:
        with pytest.raises(ValueError):
            f()


def test_attention_refuses():
    q, c = torch.zeros(4, 4, 64), torch.zeros(2, 2, 64, 64)
    m, t = torch.zeros(4, 1, dtype=torch.int64), torch.zeros(1, 2, dtype=torch.int32)
    ok = dict(q=q, kc=c, vc=c, block_table=t, cu_q=[0, 4], kv_lens=[70], mask=m, scale=0.1)
    ops.tree_attention(**ok)
    s = torch.zeros(2, 2, 64)
    for bad in ({"q": q[0]}, {"vc": c[:1]}, {"q": torch.zeros(4, 4, 32)}, {"kc": c.transpose(0, 1), "vc": c.transpose(0, 1)}, {"ks": s},
                {"ks": s, "vs": s}, {"mask": m[:3]}, {"mask": m.int()}, {"mask": torch.zeros(4, 5, dtype=torch.int64)}, {"cu_q": [0, 3, 4]},
                {"kv_lens": [3]}, {"block_table": t.long()}, {"block_table": t[:0]}, {"window": 4}, {"window": -1}, {"softcap": -1.0},
                {"window": 4, "positions": torch.zeros(4)}, {"sinks": torch.zeros(2)}, {"group": 1}, {"q_off": 1}, {"group": -1}):
        with pytest.raises(ValueError):
            ops.tree_attention(**{**ok, **bad})
    with pytest.raises(ValueError):
        ops.tree_attention(torch.zeros(70, 4, 64), c, c, t, [0, 70], [100], torch.zeros(70, 1, dtype=torch.int64), 0.1)
