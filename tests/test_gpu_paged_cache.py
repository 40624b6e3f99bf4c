"""PagedKVCache: requests come, grow and go over many steps, against a dense cache in 64 bits; a step captured and replayed."""
import copy
import math

import numpy as np
import pytest
import torch

import paged_plain as plain
from kvcomp_b200.utils.rotary import frequencies

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def Cache():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    from kvcomp_b200.cache import PagedKVCache
    return PagedKVCache


def dev(a, dtype=torch.int32):
    return torch.as_tensor(np.asarray(a)).to(dtype).cuda()


class Dense:
    """What the cache should hold: rotated keys (as it stores them, read back) and values of each request and layer, in the order of their tokens."""

    def __init__(self, requests, layers):
        self.k = [[[] for _ in range(layers)] for _ in range(requests)]
        self.v = [[[] for _ in range(layers)] for _ in range(requests)]

    def length(self, b):
        return len(self.k[b][0])


def attend_plain(dense, q, layer, scaling, window, dtype):
    """out and its bound for one token per request, from pages made of the dense rows."""
    lengths = [dense.length(b) for b in range(len(dense.k))]
    Hkv, D = next((dense.k[b][0][0].shape for b in range(len(lengths)) if lengths[b]), (1, q.shape[-1]))
    pages, table, rows = 1, np.full((len(lengths), max(max(lengths), 1)), -1, dtype=np.int32), []
    kp = torch.zeros(sum(lengths) + 1, 1, Hkv, D, dtype=dtype)
    vp = torch.zeros_like(kp)
    at = 0
    for b, n in enumerate(lengths):
        for t in range(n):
            kp[at, 0], vp[at, 0] = dense.k[b][layer][t], dense.v[b][layer][t]
            table[b, t] = at
            at += 1
    out, _, bound, _ = plain.attend(q, kp, vp, torch.as_tensor(table), lengths, scaling, window)
    return out, bound


@pytest.mark.parametrize("dtype,Hq,Hkv,D,page,layout,window,pages", [(torch.float16, 4, 4, 64, 8, "half", 0, 40), (torch.bfloat16, 8, 2, 128, 16, "interleaved", 0, 40),
                                                                     (torch.float16, 6, 2, 96, 5, "half", 20, 40), (torch.float16, 4, 1, 64, 8, "half", 0, 12)])
def test_requests_come_and_go(Cache, dtype, Hq, Hkv, D, page, layout, window, pages):
    """Prompts, single tokens and releases, pages used again; in a pool of 12 pages some are refused."""
    from kvcomp_b200 import _lib
    R, layers, steps = 6, 2, 24
    rng, gen = np.random.RandomState(page), torch.Generator(device="cuda").manual_seed(page)
    f, factor = frequencies(D // 2, scaling={"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 64})
    cache = Cache(R, pages, layers, Hkv, D, page_size=page, max_tokens=120, dtype=dtype, frequencies=f, layout=layout, factor=factor, window=window)
    dense, refused = Dense(R, layers), 0
    for step in range(steps):
        prompts = step % 4 == 0
        new = [int(rng.randint(1, 40)) if dense.length(b) == 0 and prompts else (1 if dense.length(b) else 0) for b in range(R)]
        tokens = sum(new)
        plan = cache.begin(dev(new), tokens)
        taken, starts, positions = plan.taken.tolist(), plan.starts.tolist(), plan.positions.cpu()
        refused += sum(t < 0 for t in taken)
        assert starts == [int(x) for x in np.concatenate([[0], np.cumsum(new)])]
        for layer in range(layers):
            qkv = torch.randn(tokens, Hq + 2 * Hkv, D, generator=gen, device="cuda").to(dtype)
            q, k, v = qkv[:, :Hq], qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:]
            rotated = cache.append(q, k, v, layer)
            want = plain.rotate(q.cpu(), positions, f, layout, factor)
            assert bool(((rotated.cpu().double() - want).abs() <= plain.rotate_bound(q.cpu(), want, f, layout, factor)).all())
            slots = plan.slots.tolist()
            for b in range(R):
                for row in range(starts[b], starts[b + 1]):
                    if taken[b] >= 0:
                        dense.k[b][layer].append(cache.keys[layer, slots[row] // page, slots[row] % page].cpu())
                        dense.v[b][layer].append(v[row].cpu())
                        wk = plain.rotate(k[row:row + 1].cpu(), positions[row:row + 1], f, layout, factor)
                        assert bool(((dense.k[b][layer][-1].double() - wk[0]).abs() <= plain.rotate_bound(k[row:row + 1].cpu(), wk, f, layout, factor)[0]).all())
                    else:
                        assert slots[row] == -1
            query = torch.randn(R, Hq, D, generator=gen, device="cuda").to(dtype)
            out = cache.attend(query, layer)
            want, bound = attend_plain(dense, query, layer, 1 / math.sqrt(D), window, dtype)
            assert bool(((out.cpu().double() - want).abs() <= bound).all()), (step, layer)
        assert cache.lengths.tolist() == [dense.length(b) for b in range(R)]
        held = sum(-(-dense.length(b) // page) for b in range(R))
        assert cache.head.item() == held
        table, owned = cache.table.cpu().numpy(), []
        for b in range(R):
            owned += table[b, :-(-dense.length(b) // page)].tolist()
        assert sorted(owned + cache.free[held:].tolist()) == list(range(pages))      # every page is somebody's or free, none twice
        flags = cache.check()
        assert flags == (_lib.FLAG_NO_PAGES if min(taken) < 0 else 0)
        if step % 5 == 4:
            done = [bool(dense.length(b) and rng.rand() < 0.6) for b in range(R)]
            cache.release(dev(done, torch.bool))
            for b in range(R):
                if done[b]:
                    dense.k[b], dense.v[b] = [[] for _ in range(layers)], [[] for _ in range(layers)]
    assert (refused > 0 or pages == 40) and cache.get_seq_length(0) == dense.length(0)


def test_a_step_in_a_graph(Cache):
    """A decode step captured once and replayed: lengths, tables and pages go on as they do step by step; a release between replays; two graphs that share a cache."""
    R, layers, Hq, Hkv, D, page = 5, 2, 8, 2, 128, 4
    f, _ = frequencies(D)
    gen = torch.Generator(device="cuda").manual_seed(1)
    a = Cache(R, 64, layers, Hkv, D, page_size=page, max_tokens=80, frequencies=f)
    prompt = [9, 0, 17, 4, 1]
    a.begin(dev(prompt), sum(prompt))
    for layer in range(layers):
        a.append(None, *(torch.randn(sum(prompt), Hkv, D, generator=gen, device="cuda").half() for _ in range(2)), layer)
    b = copy.deepcopy(a)
    rows = torch.randn(R, Hq + 2 * Hkv, D, device="cuda").half()
    ones = dev([1] * R)

    def step(cache):
        cache.begin(ones, R)
        outs = []
        for layer in range(layers):
            q = cache.append(rows[:, :Hq], rows[:, Hq:Hq + Hkv], rows[:, Hq + Hkv:], layer)
            outs.append(cache.attend(q, layer))
        return outs

    step(a), step(b)                                       # (workspaces are made here)
    torch.cuda.synchronize()
    graphs = []
    state = [t.clone() for t in (a.lengths, a.head, a.table)]
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs = step(a)
        graphs.append((g, outs))
    assert all(torch.equal(x, y) for x, y in zip(state, (a.lengths, a.head, a.table)))       # captured, not run
    for n in range(12):
        rows.copy_(torch.randn(rows.shape, generator=gen, device="cuda"))
        if n == 7:
            done = dev([False, True, False, False, True], torch.bool)
            a.release(done), b.release(done)
        g, outs = graphs[n % 2]
        g.replay()
        want = step(b)
        assert all(torch.equal(x, y) for x, y in zip(outs, want)), n
        assert torch.equal(a.lengths, b.lengths) and torch.equal(a.head, b.head) and torch.equal(a.table, b.table) and torch.equal(a.keys, b.keys)
    assert a.lengths.tolist() == [9 + 13, 5, 17 + 13, 4 + 13, 5] and a.check() == 0


def test_a_step_captured_behind_two_streams(Cache):
    """The step's first kernels follow a copy, a memset and another stream's kernels in one graph."""
    from kvcomp_b200 import ops
    R, D = 3, 64
    cache = Cache(R, 30, 1, 2, D, page_size=8, frequencies=frequencies(D)[0])
    rows, new = torch.randn(R, 6, D, device="cuda").half(), dev([0] * R)
    counts, scratch = dev([2, 1, 3]).cpu().pin_memory(), torch.ones(100000, device="cuda")
    x = torch.randn(6, 6, D, device="cuda").half()
    cache.attend(rows[:, :2], 0)                           # (the workspace)
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph):
        main = torch.cuda.current_stream()
        side.wait_stream(main)
        with torch.cuda.stream(side):
            for _ in range(20):
                scratch.mul_(1.0)
            turned = ops.rotary(x, cache_positions := torch.zeros(6, dtype=torch.int32, device="cuda"), cache.frequencies)
        new.copy_(counts, non_blocking=True)
        main.wait_stream(side)
        plan = cache.begin(new, 6)
        cache_positions.zero_()
        q = cache.append(turned[:, :2], x[:, 2:4], x[:, 4:], 0)
        out = cache.attend(rows[:, :2], 0)
    want, lengths = None, [0] * R
    for _ in range(4):
        graph.replay()
        lengths = [n + k for n, k in zip(lengths, [2, 1, 3])]
        assert cache.lengths.tolist() == lengths and plan.positions.tolist() == [n - k + j for n, k in zip(lengths, [2, 1, 3]) for j in range(k)]
        want, _, bound, _ = plain.attend(rows[:, :2], cache.keys[0], cache.values[0], cache.table, lengths, 1 / math.sqrt(D))
        assert bool(((out.cpu().double() - want).abs() <= bound).all())
        rot = plain.rotate(x[:, :2].cpu(), plan.positions.cpu(), cache.frequencies.cpu(), "half")
        assert bool(((q.cpu().double() - rot).abs() <= plain.rotate_bound(x[:, :2].cpu(), rot, cache.frequencies, "half", 1.0)).all())
    assert cache.check() == 0


def test_refusals(Cache):
    from kvcomp_b200._lib import KvcError
    for kw in (dict(dtype=torch.float32), dict(device="cpu"), dict(page_size=0)):
        with pytest.raises(KvcError):
            Cache(2, 4, 1, 2, 64, **kw)
    cache = Cache(2, 4, 1, 2, 64)
    x = torch.zeros(2, 2, 64, dtype=torch.float16, device="cuda")
    with pytest.raises(KvcError):
        cache.append(x, x, x, 0)
    with pytest.raises(KvcError):
        cache.begin(dev([1, 1, 1]), 3)
    cache.begin(dev([1, 1]), 2)
    with pytest.raises(KvcError):
        cache.append(x, x.bfloat16(), x, 0)
    with pytest.raises(KvcError):
        cache.attend(x[:, :1], 0)
