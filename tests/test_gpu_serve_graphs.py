"""What the operators of include/bpdq_serve.h record into a captured graph."""
import ctypes

import pytest
import torch

import paged_oracle as O
from bpd_substrate_amd import gpu, serve

pytestmark = pytest.mark.gpu

KERNEL = 0  # hipGraphNodeTypeKernel


def nodes(graph):
    """(type of each node of a captured graph, pairs of places that follow each other)"""
    gpu.lib()
    with open("/proc/self/maps") as f:
        hip = ctypes.CDLL(next(l.split()[-1] for l in f if "libamdhip64" in l))
    h, n, m = ctypes.c_void_p(graph.raw_cuda_graph()), ctypes.c_size_t(), ctypes.c_size_t()
    assert hip.hipGraphGetNodes(h, None, ctypes.byref(n)) == 0
    all_ = (ctypes.c_void_p * n.value)()
    assert hip.hipGraphGetNodes(h, all_, ctypes.byref(n)) == 0
    kinds = []
    for x in all_:
        t = ctypes.c_int(-1)
        assert hip.hipGraphNodeGetType(ctypes.c_void_p(x), ctypes.byref(t)) == 0
        kinds.append(t.value)
    assert hip.hipGraphGetEdges(h, None, None, ctypes.byref(m)) == 0
    a, b = (ctypes.c_void_p * m.value)(), (ctypes.c_void_p * m.value)()
    assert hip.hipGraphGetEdges(h, a, b, ctypes.byref(m)) == 0
    place = {x: i for i, x in enumerate(all_)}
    return kinds, sorted((place[x], place[y]) for x, y in zip(a, b))


@pytest.mark.parametrize("form,V,kernels", [("one token", 1000, 1 + 2 + 1), ("behind a prefix", 32769, 1 + 2 + 5),
                                            ("chunks", 40000, 1 + 3 + 5)])
def test_a_captured_step_is_kernels_one_after_the_other(dev, form, V, kernels):
    """No memset or copy among them: on replays after the first, memset nodes have not done their work."""
    new, P = [1, 20] if form == "chunks" else [1, 1], 70 if form == "behind a prefix" else 0
    b = O.Batch(5, new, [90, 40], P, 4, 2, 64, "f16", "f16", 16, decode=form != "chunks")
    cache, batch, q = b.device(dev)
    rope, T = serve.Rope(64, device=dev), b.T
    k = torch.randn(T, 2, 64, device=dev).half()
    logits, u = torch.randn(T, V, device=dev), torch.rand(T, device=dev)

    def step():
        r = serve.rope_append(cache, batch, q, k, k, rope=rope)
        return serve.attention(cache, batch, r), serve.sample(logits, u)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        step()
    kinds, edges = nodes(graph)
    assert kinds == [KERNEL] * kernels
    assert edges == [(i, i + 1) for i in range(kernels - 1)]
