"""PagedKVCache in 8 bits and with requests that follow others: whole steps, eager and captured, against the plain attention over what the cache should hold."""
import copy
import io
import math
import pickle

import numpy as np
import pytest
import torch

import codes_plain
import paged_plain as plain
from test_gpu_paged_cache import Cache, dev  # noqa: F401  (the fixture)
from kvcomp_b200.utils.rotary import frequencies

pytestmark = pytest.mark.gpu


def randn(gen, dtype, *shape):
    return torch.randn(shape, generator=gen, device="cuda").to(dtype)


def near(got, want, bound):
    assert bool(((got.cpu().double() - want).abs() <= bound).all()), float(((got.cpu().double() - want).abs() / bound).max())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("codes", ["int8", "e4m3"])
@pytest.mark.parametrize("D,page", [(64, 5), (96, 16), (128, 16), (256, 8)])
def test_steps(Cache, codes, dtype, D, page):  # noqa: F811
    """Prompts, single tokens, releases: attention over the pages is the plain one over the rows that the cache reads back; these are within half a step of what was appended."""
    R, Hq, Hkv, layers = 4, 4, 2, 2
    gen = torch.Generator(device="cuda").manual_seed(D)
    f = frequencies(D)[0]
    cache = Cache(R, 200 // page + 8, layers, Hkv, D, page_size=page, max_tokens=100, dtype=dtype, frequencies=f, codes=codes)
    held = [[] for _ in range(R)]                                   # of layer 0: (rotated key, value) in 64 bits
    for step, new in enumerate([[7, 0, 30, 1], [1, 1, 1, 1], [1, 0, 1, 0], [0, 20, 0, 3], [1, 1, 1, 1]]):
        n = sum(new)
        q, k, v = (randn(gen, dtype, n, h, D) for h in (Hq, Hkv, Hkv))
        plan = cache.begin(dev(new), n)
        turned = plain.rotate(k.cpu(), plan.positions.cpu(), f, "half")
        for layer in range(layers):
            rotated = cache.append(q, k, v, layer)
        at = 0
        for b, m in enumerate(new):
            held[b] += [(turned[at + i], v[at + i].cpu().double()) for i in range(m)]
            at += m
        total = sum(len(h) for h in held)
        slots, starts = cache.slots(total)
        rows = [cache.rows(layer, slots) for layer in range(layers)]
        assert starts.tolist() == np.cumsum([0] + [len(h) for h in held]).tolist()
        assert all(torch.equal(a, b) for a, b in zip(rows[0], rows[1]))
        eps = torch.finfo(dtype).eps / 2
        for got, i in zip(rows[0], (0, 1)):
            x = torch.stack([row[i] for h in held for row in h])
            s = codes_plain.scale(x, codes)
            near(got, x, codes_plain.half_step(x, s, codes) * (1 + 2.0 ** -10) + eps * x.abs() + s * 2.0 ** -10)
        if max(new) == 1:
            owners = [b for b in range(R) if new[b]]
            out, lse = cache.attend(rotated, 1, return_lse=True)
            kp, vp = (codes_plain.values(p, s) for p, s in ((cache.keys[1], cache.key_scales[1]), (cache.values[1], cache.value_scales[1])))
            w, w_lse, off, lse_off = plain.attend(rotated, kp, vp, cache.table[owners], [len(held[b]) for b in owners], 1 / math.sqrt(D))
            near(out, w, off + eps * (w.abs() + off) + (2.0 ** -25 if dtype == torch.float16 else 0) + 100 * 2.0 ** -39 * float(vp.abs().max()))
            near(lse, w_lse, lse_off)
        if step == 2:
            cache.release(dev([False, False, True, False], torch.bool))
            held[2] = []
    assert cache.check() == 0


def test_prompt_in_chunks(Cache):  # noqa: F811
    """The rows of a chunked prompt in 16 bits are the rotated keys and the values, in order; a copy of the cache and one that was saved read the same."""
    D, cache = 128, Cache(2, 40, 1, 2, 128, page_size=8, dtype=torch.bfloat16, frequencies=frequencies(128)[0])
    gen = torch.Generator(device="cuda").manual_seed(1)
    keys, values = [], []
    for n in (33, 40, 1):
        k, v = randn(gen, torch.bfloat16, n, 2, D), randn(gen, torch.bfloat16, n, 2, D)
        plan = cache.begin(dev([0, n]), n)
        cache.append(None, k, v, 0)
        from kvcomp_b200 import ops
        keys.append(ops.rotary(k, plan.positions, cache.frequencies))
        values.append(v)
        slots, starts = cache.slots(sum(len(x) for x in keys) + 3)
        k, v = cache.rows(0, slots)
        assert torch.equal(k[:-3], torch.cat(keys)) and torch.equal(v[:-3], torch.cat(values)) and not bool(k[-3:].any())
    for other in (copy.deepcopy(cache), pickle.load(io.BytesIO(pickle.dumps(cache)))):
        assert all(torch.equal(a, b) for a, b in zip(cache.rows(0, slots), other.rows(0, slots)))


def test_captured_steps_in_8_bits(Cache):  # noqa: F811
    R, Hq, Hkv, D = 3, 4, 2, 128
    caches = [Cache(R, 60, 1, Hkv, D, page_size=8, max_tokens=100, frequencies=frequencies(D)[0], codes="int8") for _ in range(2)]
    gen = torch.Generator(device="cuda").manual_seed(3)
    k, v = randn(gen, torch.float16, 40, Hkv, D), randn(gen, torch.float16, 40, Hkv, D)
    for cache in caches:
        cache.begin(dev([30, 0, 10]), 40)
        cache.append(None, k, v, 0)
    new, qkv = dev([1, 1, 1]), randn(gen, torch.float16, R, Hq + 2 * Hkv, D)

    def step(cache):
        cache.begin(new, R)
        return cache.attend(cache.append(qkv[:, :Hq], qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:], 0), 0)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        got = step(caches[0])
    for counts in ([1, 1, 1], [0, 1, 0], [1, 0, 1], [1, 1, 1]):
        new.copy_(dev(counts))
        qkv.copy_(randn(gen, torch.float16, *qkv.shape))
        graph.replay()
        assert torch.equal(got, step(caches[1]))
    assert torch.equal(caches[0].key_scales, caches[1].key_scales) and torch.equal(caches[0].values, caches[1].values)


# ---- requests that follow others -------------------------------------------------------------------

class Pair:
    """A cache whose requests follow others, and one where each has the prefix as tokens of its own."""

    def __init__(self, Cache, dtype, D, Hkv, layers=1, R=7):  # noqa: F811
        make = lambda pages, R: Cache(R, pages, layers, Hkv, D, page_size=16, max_tokens=400, dtype=dtype, frequencies=frequencies(D)[0])  # noqa: E731
        self.a, self.b, self.R, self.gen = make(120, R), make(220, R), R, torch.Generator(device="cuda").manual_seed(D)

    def near(self, x, y, v):
        """Two results of the same definition: both within the bounds of weights in 16 bits and the result's rounding."""
        eps = torch.finfo(x.dtype).eps / 2
        assert bool(((x.double() - y.double()).abs() <= (4 * eps + 2.0 ** -10) * v).all())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D,Hq,Hkv", [(128, 8, 2), (64, 4, 4), (96, 6, 2)])
def test_followers(Cache, dtype, D, Hq, Hkv):  # noqa: F811
    """Positions go on behind the prefix, results are those of requests that have all tokens themselves; followers end and come, another prefix is followed."""
    p = Pair(Cache, dtype, D, Hkv)
    n = [0] * p.R                                                   # tokens that the plain requests have
    prompts = {0: 200, 3: 37}
    follows = {1: 0, 2: 0, 4: 3, 5: 0}
    stuff = {b: [randn(p.gen, dtype, m, Hkv, D) for _ in range(2)] for b, m in prompts.items()}
    p.a.begin(dev([prompts.get(b, 0) for b in range(p.R)]), sum(prompts.values()))
    p.a.append(None, *(torch.cat([stuff[b][i] for b in sorted(stuff)]) for i in (0, 1)), 0)
    p.a.follow(dev([follows.get(b, -1) for b in range(p.R)]))
    has = [prompts.get(follows.get(b, b), 0) for b in range(p.R)]
    p.b.begin(dev(has), sum(has))
    p.b.append(None, *(torch.cat([stuff[follows.get(b, b)][i] for b in range(p.R) if has[b]]) for i in (0, 1)), 0)
    assert [p.a.get_seq_length(b) for b in range(p.R)] == [p.b.get_seq_length(b) for b in range(p.R)]
    for counts in ([0, 9, 0, 0, 20, 1, 5], [0, 1, 1, 0, 1, 1, 1], [0, 1, 0, 0, 1, 1, 0], [0, 1, 1, 0, 0, 1, 1]):
        total = sum(counts)
        q, k, v = (randn(p.gen, dtype, total, h, D) for h in (Hq, Hkv, Hkv))
        plans = [c.begin(dev(counts), total) for c in (p.a, p.b)]
        assert torch.equal(plans[0].positions, plans[1].positions)
        rotated = [c.append(q, k, v, 0) for c in (p.a, p.b)]
        assert torch.equal(*rotated)
        if max(counts) == 1:
            (x, lx), (y, ly) = (c.attend(r, 0, return_lse=True) for c, r in zip((p.a, p.b), rotated))
            p.near(x, y, 4.0)
            assert bool(((lx - ly).abs() <= 1e-4).all())
    done = dev([False, True, False, False, False, False, False], torch.bool)
    for c in (p.a, p.b):
        c.release(done)
        assert c.check() == 0
    assert p.a.parents.tolist() == [-1, -1, 0, -1, 3, 0, -1] and p.a.get_seq_length(1) == 0
    q, k, v = (randn(p.gen, dtype, 2, h, D) for h in (Hq, Hkv, Hkv))
    rotated = [(c.begin(dev([0, 1, 1, 0, 0, 0, 0]), 2), c.append(q, k, v, 0))[1] for c in (p.a, p.b)]
    p.near(*(c.attend(r, 0) for c, r in zip((p.a, p.b), rotated)), 4.0)      # the one in its place follows no one
    for c in (copy.deepcopy(p.a), pickle.load(io.BytesIO(pickle.dumps(p.a)))):
        assert torch.equal(c.attend(rotated[0], 0), p.a.attend(rotated[0], 0))


def test_a_prefix_that_goes_too_early(Cache):  # noqa: F811
    """Its followers follow no one then, and check raises."""
    from kvcomp_b200._lib import KvcError
    cache = Cache(3, 20, 1, 1, 64, page_size=8, max_tokens=50)
    k = torch.randn(10, 1, 64, device="cuda").half()
    cache.begin(dev([10, 0, 0]), 10)
    cache.append(None, k, k, 0)
    cache.follow(dev([-1, 0, -1]))
    cache.release(dev([True, False, False], torch.bool))
    assert cache.parents.tolist() == [-1, -1, -1]
    with pytest.raises(KvcError):
        cache.check()


@pytest.mark.parametrize("parents,shared", [([-1, 0, 7, 0], None), ([-1, 0, 4, 0], [0, 9, 9, 9]), ([-1, 0, 2, 0], [0, 5, 5, 5]), ([-1, 0, 0, 0], [0, 9, -3, 9]), ([-1, 0, 1 << 30, 0], None)], ids=str)
def test_parents_that_are_none(Cache, parents, shared):  # noqa: F811
    """A request that says it follows no request, itself, or tokens below none is one that follows no one: positions, lengths, results and releases; check raises."""
    from kvcomp_b200._lib import KvcError
    R, Hq, Hkv, D = 4, 4, 2, 64
    gen = torch.Generator(device="cuda").manual_seed(2)
    caches = [Cache(R, 40, 1, Hkv, D, page_size=8, max_tokens=80, frequencies=frequencies(D)[0]) for _ in range(2)]
    k, v = randn(gen, torch.float16, 20, Hkv, D), randn(gen, torch.float16, 20, Hkv, D)
    qkv = randn(gen, torch.float16, R, Hq + 2 * Hkv, D)
    results = []
    for cache, of in zip(caches, (parents, [p if b != 2 else -1 for b, p in enumerate(parents)])):
        cache.begin(dev([20, 0, 0, 0]), 20)
        cache.append(None, k, v, 0)
        cache.follow(dev(of), None if shared is None else dev(shared))
        plan = cache.begin(dev([0, 1, 1, 1]), 3)
        q = cache.append(qkv[:3, :Hq], qkv[:3, Hq:Hq + Hkv], qkv[:3, Hq + Hkv:], 0)
        results.append((plan.positions, q, cache.attend(q, 0), cache.parents.clone(), cache.shared.clone(), torch.tensor([cache.get_seq_length(b) for b in range(R)])))
    assert all(torch.equal(a, b) for a, b in zip(*results)) and results[0][0][1] == 0 and results[0][5][2] == 1
    with pytest.raises(KvcError):
        caches[0].check()
    assert caches[1].check() == 0
    for cache in caches:                                            # the last request ends: nobody's prefix does
        cache.release(dev([False, False, False, True], torch.bool))
        assert cache.check() == 0 and cache.parents.tolist() == [-1, 0, -1, -1]


def test_captured_steps_of_followers(Cache):  # noqa: F811
    """One graph: followers that change between replays are those that it goes by, also where the release is part of it."""
    R, Hq, Hkv, D = 4, 4, 2, 128
    caches = [Cache(R, 60, 1, Hkv, D, page_size=8, max_tokens=200, frequencies=frequencies(D)[0]) for _ in range(2)]
    gen = torch.Generator(device="cuda").manual_seed(3)
    k, v = randn(gen, torch.float16, 150, Hkv, D), randn(gen, torch.float16, 150, Hkv, D)
    for cache in caches:
        cache.begin(dev([150, 0, 0, 0]), 150)
        cache.append(None, k, v, 0)
        cache.follow(dev([-1, 0, 0, -1]))
    new, done, qkv = dev([0, 1, 1, 1]), dev([False] * R, torch.bool), randn(gen, torch.float16, R, Hq + 2 * Hkv, D)

    def step(cache):
        cache.begin(new, R)
        out = cache.attend(cache.append(qkv[:, :Hq], qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:], 0), 0)
        cache.release(done)
        return out
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        got = step(caches[0])
    for counts, ends in (([0, 1, 1, 1], []), ([0, 0, 1, 1], []), ([0, 1, 1, 1], [2]), ([0, 1, 1, 0], []), ([0, 1, 1, 1], [])):
        new.copy_(dev(counts))
        done.copy_(dev([b in ends for b in range(R)], torch.bool))
        qkv.copy_(randn(gen, torch.float16, *qkv.shape))
        graph.replay()
        want = step(caches[1])
        assert torch.equal(got, want) and torch.equal(caches[0].prefixes.words[:1], caches[1].prefixes.words[:1])
    for cache in caches:
        cache.follow(dev([-1, 0, -1, -1]))
    graph.replay()
    assert torch.equal(got, step(caches[1]))
    assert [c.check() for c in caches] == [0, 0]


def test_followers_on_two_streams(Cache):  # noqa: F811
    """Two layers attended at once, each with a workspace of its own."""
    R, Hq, Hkv, D = 9, 8, 2, 64
    cache = Cache(R, 300, 2, Hkv, D, page_size=8, max_tokens=1200, frequencies=frequencies(D)[0])
    gen = torch.Generator(device="cuda").manual_seed(5)
    k, v = randn(gen, torch.float16, 1100, Hkv, D), randn(gen, torch.float16, 1100, Hkv, D)
    cache.begin(dev([1100] + [0] * (R - 1)), 1100)
    for layer in range(2):
        cache.append(None, k, v * (layer + 1), layer)
    cache.follow(dev([-1] + [0] * (R - 1)))
    cache.begin(dev([0] + [1] * (R - 1)), R - 1)
    q = [cache.append(randn(gen, torch.float16, R - 1, Hq, D), k[:R - 1], v[:R - 1], layer) for layer in range(2)]
    want = [cache.attend(q[layer], layer) for layer in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(20):
        for layer, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[layer].append(cache.attend(q[layer], layer))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want[layer]) for layer in range(2) for x in got[layer])


def test_refused(Cache):  # noqa: F811
    from kvcomp_b200._lib import KvcError
    i = dev([-1, 0])
    for cache in (Cache(2, 8, 1, 1, 64, window=5), Cache(2, 8, 1, 1, 256), Cache(2, 8, 1, 1, 64, codes="int8")):
        with pytest.raises(KvcError):
            cache.follow(i)
    cache = Cache(2, 8, 1, 1, 64)
    for parents, shared in ((i[:1], None), (i.long(), None), (i.cpu(), None), (i, i[:1]), ([-1, 0], None)):
        with pytest.raises(KvcError):
            cache.follow(parents, shared)


def test_more_requests_than_a_plan_takes(Cache):  # noqa: F811
    """A refused follow leaves a cache as it was: lengths, steps, copies; the largest number is taken."""
    from kvcomp_b200._lib import KvcError
    for R, taken in ((16385, False), (16384, True)):
        cache = Cache(R, 8, 1, 1, 64, page_size=8, max_tokens=16)
        k = torch.randn(9, 1, 64, device="cuda").half()
        new = torch.zeros(R, dtype=torch.int32, device="cuda")
        new[5] = 9
        cache.begin(new, 9)
        cache.append(None, k, k, 0)
        parents = torch.full((R,), -1, dtype=torch.int32, device="cuda")
        parents[7] = 5
        if taken:
            cache.follow(parents)
        else:
            with pytest.raises(KvcError):
                cache.follow(parents)
        assert cache.get_seq_length(7) == (9 if taken else 0) and (cache.prefixes is None) == (cache.parents is None) == (cache.shared is None) == (not taken)
        new.zero_()
        new[7] = 1
        plan = cache.begin(new, 1)
        q = cache.append(torch.randn(1, 2, 64, device="cuda").half(), k[:1], k[:1], 0)
        assert plan.positions.tolist() == [9 if taken else 0]
        near(cache.attend(q, 0), *plain_of(q, k if taken else k[:0], k[:1]))
        cache.release(new.bool())
        assert cache.check() == 0


def plain_of(q, *tokens):
    """(result, bound) of one request with these tokens as keys and values."""
    x = torch.cat(tokens)[:, 0].double().cpu()
    w = torch.softmax(q[0].double().cpu() @ x.T / math.sqrt(x.shape[1]), -1)
    return (w @ x)[None], 2.0 ** -9 * x.abs().max()
