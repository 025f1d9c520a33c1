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
