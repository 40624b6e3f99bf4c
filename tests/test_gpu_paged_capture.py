"""PagedKVCache: attention first called in a capture, by graphs that run at once, and on streams of their own."""
import math

import pytest
import torch

import paged_plain as plain
from test_gpu_paged_cache import Cache, dev  # noqa: F401  (the fixture)

pytestmark = pytest.mark.gpu

R, LAYERS, HQ, HKV, D = 4, 3, 8, 2, 128
LENGTHS = [3000, 0, 1, 9000]                               # columns of many parts: counters that are not zero leave them unjoined


@pytest.fixture
def filled(Cache):  # noqa: F811
    cache = Cache(R, 800, LAYERS, HKV, D, page_size=16, max_tokens=9600)
    gen = torch.Generator(device="cuda").manual_seed(1)
    cache.begin(dev(LENGTHS), sum(LENGTHS))
    for layer in range(LAYERS):
        cache.append(None, *(torch.randn(sum(LENGTHS), HKV, D, generator=gen, device="cuda").half() for _ in range(2)), layer)
    q = torch.randn(R, HQ, D, generator=gen, device="cuda").half()
    wants = []
    for layer in range(LAYERS):
        want, _, bound, _ = plain.attend(q, cache.keys[layer], cache.values[layer], cache.table, LENGTHS, 1 / math.sqrt(D))
        wants.append((want, bound))
    return cache, q, wants


def right(outs, wants):
    return all(bool(((out.cpu().double() - want).abs() <= bound).all()) for out, (want, bound) in zip(outs, wants))


def capture(cache, q):
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = [cache.attend(q, layer) for layer in range(LAYERS)]
    return graph, outs


def test_first_call_in_a_capture(filled):
    """Memory that the graph's pool hands out is not zero: an eager call, and a second graph, before the first replay."""
    cache, q, wants = filled
    junk = torch.full((64 << 20,), 7, dtype=torch.int32, device="cuda")
    del junk
    graph, outs = capture(cache, q)
    assert right([cache.attend(q, layer) for layer in range(LAYERS)], wants)
    graph2, outs2 = capture(cache, q)
    graph2.replay()
    assert right(outs2, wants)
    for _ in range(3):
        graph.replay()
        assert right(outs, wants)
        graph2.replay()
        assert right(outs2, wants)
    assert right([cache.attend(q, layer) for layer in range(LAYERS)], wants)


def test_graphs_at_once(filled):
    """Two graphs and an eager loop on three streams, over one cache."""
    cache, q, wants = filled
    graphs, streams = [capture(cache, q) for _ in range(2)], [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    eager = []
    for _ in range(30):
        for (graph, _), stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        with torch.cuda.stream(streams[2]):
            eager = [cache.attend(q, layer) for layer in range(LAYERS)]
    torch.cuda.synchronize()
    assert right(graphs[0][1], wants) and right(graphs[1][1], wants) and right(eager, wants)


def test_layers_on_streams_of_their_own(filled):
    """Eager, and forked within one capture."""
    cache, q, wants = filled
    streams = [torch.cuda.Stream() for _ in range(LAYERS)]

    def forked():
        main, outs = torch.cuda.current_stream(), []
        for layer, stream in enumerate(streams):
            stream.wait_stream(main)
            with torch.cuda.stream(stream):
                outs.append(cache.attend(q, layer))
        for stream in streams:
            main.wait_stream(stream)
        return outs

    for _ in range(10):
        outs = forked()
    torch.cuda.synchronize()
    assert right(outs, wants)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = forked()
    for _ in range(5):
        graph.replay()
    torch.cuda.synchronize()
    assert right(outs, wants)
