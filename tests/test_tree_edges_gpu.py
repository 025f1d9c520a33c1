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
