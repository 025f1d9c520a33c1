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
