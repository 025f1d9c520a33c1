"""A weight whose rows do not start on 16 bytes is copied inside a capture; the product behind that copy waits for all of it."""
import ctypes as C

import pytest
import torch

pytestmark = pytest.mark.gpu

from e4m3_rows import activations, gen, on, weight
from xfastertransformer_b200 import ops
from xfastertransformer_b200.ops import native_e4m3 as E

PROGRAMMATIC = 1               # CU_GRAPH_DEPENDENCY_TYPE_PROGRAMMATIC


class Edge(C.Structure):
    _fields_ = [("from_port", C.c_ubyte), ("to_port", C.c_ubyte), ("type", C.c_ubyte), ("reserved", C.c_ubyte * 5)]


def edges(graph):
    """Types of the dependencies of a captured graph."""
    get = C.CDLL("libcuda.so.1").cuGraphGetEdges_v2
    get.argtypes = [C.c_void_p] * 4 + [C.POINTER(C.c_size_t)]
    n, h = C.c_size_t(0), graph.raw_cuda_graph()
    assert get(h, None, None, None, C.byref(n)) == 0
    a, b, e = (C.c_void_p * n.value)(), (C.c_void_p * n.value)(), (Edge * n.value)()
    assert get(h, C.cast(a, C.c_void_p), C.cast(b, C.c_void_p), C.cast(e, C.c_void_p), C.byref(n)) == 0
    return [x.type for x in e[:n.value]]


def captured(call):
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        y = call()
    return graph, y


@pytest.mark.parametrize("T", [1, 20, 60])
def test_the_product_waits_for_the_copy(T):
    g = gen(T)
    even, odd = on(weight(g, 512, 208)), on(weight(g, 512, 200))
    assert odd.w.stride(0) % 16 and even.w.stride(0) % 16 == 0
    x = activations(g, T, 200).cuda()
    q = ops.quantize_e4m3(x)
    torch.cuda.synchronize()
    # rows, then a product whose weights were there before: it may start beside the rows' launch
    xe = activations(g, T, 208).cuda()
    graph, _ = captured(lambda: ops.linear_e4m3(ops.quantize_e4m3(xe), even))
    assert PROGRAMMATIC in edges(graph)
    for call in (lambda: ops.linear_e4m3(q, odd, out_dtype=torch.float32), lambda: ops.linear_gated_e4m3(q, odd).codes.float(),
                 lambda: E.gated_rows(q, odd, "silu")):
        graph, y = captured(call)
        kinds = edges(graph)
        assert kinds and PROGRAMMATIC not in kinds and "w_pitch16" not in odd.cache
        graph.instantiate()
        graph.replay()
        torch.cuda.synchronize()
        first = y.clone()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(first.view(torch.uint8), y.view(torch.uint8))      # (rows of 1e20 leave 32 bits in the gated products)
    graph, y = captured(lambda: ops.linear_e4m3(q, odd, out_dtype=torch.float32))
    graph.instantiate()
    graph.replay()
    want = ops.linear_e4m3(q, odd, out_dtype=torch.float32)            # eager: keeps the copy
    assert torch.equal(y.view(torch.uint8), want.view(torch.uint8)) and "w_pitch16" in odd.cache
    graph, _ = captured(lambda: ops.linear_e4m3(ops.quantize_e4m3(x), odd))
    assert PROGRAMMATIC in edges(graph)                                # made before the capture: as any other weight
