"""Operators of a step with trees of drafted tokens, at the edges of what they take: on a CPU, and in their sources."""
import os
import re

import pytest
import torch

from xfastertransformer_b200 import ops
from xfastertransformer_b200.ops import reference as R

KERNELS = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "csrc", "kernels")


def test_no_store_to_another_cta_before_all_have_started():
    """Shared memory of a cluster's other CTAs exists once those run: the sampler waits for them in front of its first store, on each way there."""
    text = re.sub(r"//[^\n]*", "", open(os.path.join(KERNELS, "sample_rows.cu")).read())
    body = text[text.index("sample_rows_kernel(const SampleArgs a)"):]
    assert 0 < body.index("cluster_arrive()") < body.index("all_here = ") < body.index("cluster_wait()")
    waits = [m.start() for m in re.finditer(r"\ball_here\(\)", body)]
    peers = [m.start() for m in re.finditer(r"\b(?:st|ld|add)_peer\(|cluster_barrier<C>\(\)", body)]
    end_of_greedy = body.index("return;", body.index("if (greedy) {"))
    for start, end in ((0, end_of_greedy), (end_of_greedy, len(body))):       # rows at temperature 0 leave early
        assert [w for w in waits if start < w < end][0] < [p for p in peers if start < p < end][0]


def test_attention_refuses_a_cache_without_blocks():
    q, m, t = torch.zeros(4, 4, 64), torch.ones(4, 1, dtype=torch.int64), torch.zeros(1, 2, dtype=torch.int32)
    for c in (torch.zeros(0, 2, 64, 64), torch.zeros(2, 2, 0, 64)):
        with pytest.raises(ValueError):                   # there is no block that an index outside the pool could be read as
            ops.tree_attention(q, c, c, t, [0, 4], [70], m, 0.1)
        assert ops.tree_attention(q[:0], c, c, t, [0, 0], [0], m[:0], 0.1).shape == (0, 4, 64)


def test_pools_start_on_an_even_byte():
    odd = torch.zeros(2 * 64 * 4 + 1, dtype=torch.int8)[1:].view(2, 1, 64, 4)          # rows move in pieces of two bytes at least
    assert odd.data_ptr() % 2 == 1 and odd.is_contiguous()
    with pytest.raises(ValueError):
        ops.cache_pools([odd])


def chain_with_gaps(dev="cpu"):
    """A tree whose accepted path is 0, 2, 4, 5: (tokens, parents, sampled, cu_q, kv_lens, table)."""
    t = lambda *x: torch.tensor(x, device=dev)
    return t(0, 9, 2, 9, 4, 5), t(-1, 0, 0, 2, 2, 4).int(), t(2, 0, 4, 0, 5, 7), [0, 6], [16], t(0).int()[None]


def test_a_pool_that_several_layers_read_moves_once():
    for dtype in (torch.float32, torch.int8):
        pools = [torch.arange(64).view(1, 1, 64, 1).repeat(1, 2, 1, 4).to(dtype) for _ in range(2)]
        scales = torch.arange(64.0).view(1, 1, 64)
        k = [pools[0], pools[1], pools[0], pools[0].view(1, 2, 64, 4)]
        *_, count = ops.tree_accept(*chain_with_gaps(), ops.cache_pools(k, ks=[scales, None, scales, scales]))
        assert int(count[0]) == 4
        for p in (*pools, scales[..., None]):
            assert p[0, 0, 10:14, 0].tolist() == [10, 12, 14, 15]


def test_pools_that_overlap_are_refused():
    flat = torch.zeros(3 * 64 * 4)
    a, b, c = flat[:512].view(2, 1, 64, 4), flat[256:].view(2, 1, 64, 4), torch.zeros(2, 1, 64, 4)
    for pools in ([a, b], [a, c, a.view(torch.int32)], [a, flat[:256].view(2, 1, 64, 2)]):
        with pytest.raises(ValueError):
            ops.cache_pools(pools)
    ops.cache_pools([flat[:256].view(2, 1, 64, 2), flat[256:512].view(2, 1, 64, 2)], [c], None)          # neighbours do not


@pytest.mark.parametrize("dtype", ["bf16", "int8"])
def test_the_handle_of_a_cache_is_made_once_and_refused_when_its_pools_have_moved(dtype):
    import gc
    import weakref
    from xfastertransformer_b200.runtime.kv_cache import PagedKVCache
    c = PagedKVCache(2, 2, 8, 8, dtype, torch.device("cpu"))
    c.ensure_blocks(2)
    handle = c.pools()
    assert c.pools() is handle and len(handle.pools) == (8 if dtype == "int8" else 4)
    c.k[1][0, :, 10:16] = torch.arange(10, 16)[:, None]
    ops.tree_accept(*chain_with_gaps(), handle)
    assert c.k[1][0, 1, 10:14, 3].tolist() == [10, 12, 14, 15]
    was = weakref.ref(c.k[0])
    c.ensure_blocks(9)                                    # grows: the rows are elsewhere now
    gc.collect()
    assert was() is None                                  # and the memory that they were in is free
    for pools in (handle, handle):
        with pytest.raises(ValueError):
            ops.tree_accept(*chain_with_gaps(), pools)
    new = c.pools()
    assert new is not handle and c.pools() is new and not bool(handle.table[:, 1:].any())
    c.k[1][0, :, 10:16] = torch.arange(10, 16)[:, None]
    ops.tree_accept(*chain_with_gaps(), new)
    assert c.k[1][0, 1, 10:14, 3].tolist() == [10, 12, 14, 15]


def test_attention_of_a_share_without_heads():
    m, t = torch.ones(4, 1, dtype=torch.int64), torch.zeros(1, 2, dtype=torch.int32)
    for hkv in (0, 2):
        c = torch.zeros(2, hkv, 64, 64)
        assert ops.tree_attention(torch.zeros(4, 0, 64), c, c, t, [0, 4], [70], m, 0.1).shape == (4, 0, 64)
    with pytest.raises(ValueError):                       # queries that have no keys
        ops.tree_attention(torch.zeros(4, 2, 64), torch.zeros(2, 0, 64, 64), torch.zeros(2, 0, 64, 64), t, [0, 4], [70], m, 0.1)


def test_the_server_takes_a_min_p_of_null(tmp_path, monkeypatch):
    import json
    import urllib.request
    import xfastertransformer_b200 as xft
    from serving import openai_server
    from xfastertransformer_b200.tools.synthetic import preset, write_synthetic_checkpoint
    monkeypatch.setenv("XFT_ENGINE", "CPU")
    write_synthetic_checkpoint(str(tmp_path), preset("tiny-llama", vocab_size=500), seed=3, dtype="fp32", std=0.1)
    httpd, sched, port = openai_server.serve(xft.AutoModel.from_pretrained(str(tmp_path), dtype="bf16"), 0, max_batch=4, model_name="tiny")

    def post(**body):
        body = json.dumps({"prompt": [5, 9, 100], "max_tokens": 4, **body}).encode()
        req = urllib.request.Request(f"http://127.0.0.1:{port}/v1/completions", data=body, headers={"Content-Type": "application/json"})
        return json.loads(urllib.request.urlopen(req, timeout=120).read())["choices"][0]["text"]
    try:
        assert post(min_p=None) == post()                 # as without it, which is what it was before the field had a meaning
        assert post(min_p=1.0, temperature=0.9, seed=1, top_k=-1) == post()
    finally:
        sched.shutdown()
        httpd.shutdown()


def test_a_limit_of_any_size():
    x, u = torch.randn(3, 50, generator=torch.Generator().manual_seed(1)), torch.tensor([0.1, 0.5, 0.9])
    want = ops.sample(x, 1.0, 0, 0.9, 0.01, u)
    for k in (50, 2 ** 31, 2 ** 63, 10 ** 30, -2 ** 63 - 1, -10 ** 30):          # a request's number may be any
        assert torch.equal(ops.sample(x, 1.0, k, 0.9, 0.01, u), want)


def test_tables_of_replaced_pools_stay_for_the_graphs_that_read_them():
    import gc
    import weakref
    from xfastertransformer_b200.runtime.kv_cache import PagedKVCache
    c = PagedKVCache(2, 2, 8, 8, "bf16", torch.device("cpu"))
    tables = []
    for blocks in (2, 9, 30):
        c.ensure_blocks(blocks)
        tables.append(weakref.ref(c.pools().table))       # the program keeps none of the handles
    gc.collect()
    assert all(t() is not None for t in tables)
    assert [bool(t()[:, 1:].any()) for t in tables] == [False, False, True]
