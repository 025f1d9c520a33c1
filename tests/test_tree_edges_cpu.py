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
