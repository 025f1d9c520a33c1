"""Stacks of experts in e4m3 go with their experts."""
import gc

import pytest
import torch

pytestmark = pytest.mark.gpu

from e4m3_rows import gen, on
from test_e4m3_rows_gpu import experts64, whole, whole_rows
from xfastertransformer_b200 import ops


def test_stacks_of_lists_that_are_gone_are_dropped():
    g = gen(8)
    pair = lambda: (whole(g, 256, 128), whole(g, 128, 128))
    host = pair()
    first = (on(host[0]), on(host[1]))
    q = whole_rows(g, 9, 128)
    idx, w = torch.arange(9, dtype=torch.int32).view(9, 1) % 3, torch.ones(9, 1)

    def of(others):
        """A list with the same first expert that lives for one call."""
        experts = [first] + [(on(a), on(b)) for a, b in others]
        got = ops.moe_experts_e4m3(rows(q), idx.cuda(), w.cuda(), experts, "relu").cpu().double()
        want, tol = experts64(q, idx, w, [host] + others)
        assert bool(((got - want).abs() <= tol + 3 * 2.0 ** -24 * want.abs().amax(1, keepdim=True)).all())

    rows = lambda q: ops.RowsE4M3(q.codes.cuda(), q.scale.cuda())
    held = []
    for _ in range(6):
        of([pair(), pair()])
        gc.collect()
        torch.cuda.synchronize()
        held.append((len(first[0].cache["e4m3_packs"]), torch.cuda.memory_allocated()))
    assert [n for n, _ in held] == [1] * 6 and held[-1][1] <= held[1][1]


def test_stacks_of_lists_that_live_stay():
    """Also where another list was stacked meanwhile, and one that is held by its result alone."""
    g = gen(9)
    a, b, c, d = [(on(whole(g, 256, 128)), on(whole(g, 128, 128))) for _ in range(4)]
    one, two = [a, b], [a, c]
    p1, p2 = ops.pack_experts_e4m3(one), ops.pack_experts_e4m3(two)
    assert p1 is not p2 and ops.pack_experts_e4m3(one) is p1 and ops.pack_experts_e4m3(two) is p2
    q = whole_rows(g, 8, 128)
    dq = ops.RowsE4M3(q.codes.cuda(), q.scale.cuda())
    idx, w = (torch.arange(8, dtype=torch.int32).view(8, 1) % 2).cuda(), torch.ones(8, 1, device="cuda")
    static = torch.cuda.CUDAGraph()
    want = ops.moe_experts_e4m3(dq, idx, w, one, "relu")
    with torch.cuda.graph(static):
        y = ops.moe_experts_e4m3(dq, idx, w, one, "relu")
    del c, two
    gc.collect()
    p3 = ops.pack_experts_e4m3([a, d])
    assert len(a[0].cache["e4m3_packs"]) == 2 and ops.pack_experts_e4m3(one) is p1 and ops.pack_experts_e4m3([a, d]) is p3
    static.replay()
    assert torch.equal(y, want) and torch.equal(ops.moe_experts_e4m3(dq, idx, w, one, "relu"), want)
    assert p2["E"] == 2                                                # its holder's
