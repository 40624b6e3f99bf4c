"""PagedKVCache.attend of rows as append returns them: packed request by request, some requests without one."""
import math

import pytest
import torch

import paged_plain as plain
from test_gpu_paged_cache import Cache, dev  # noqa: F401  (the fixture)
from kvcomp_b200.utils.rotary import frequencies

pytestmark = pytest.mark.gpu

R, HQ, HKV, D = 6, 8, 2, 128


def filled(Cache, prompt, dtype=torch.float16, **kw):
    cache = Cache(R, 64, 1, HKV, D, page_size=8, max_tokens=100, dtype=dtype, frequencies=frequencies(D)[0], **kw)
    gen = torch.Generator(device="cuda").manual_seed(sum(prompt))
    if sum(prompt):
        cache.begin(dev(prompt), sum(prompt))
        cache.append(None, *(torch.randn(sum(prompt), HKV, D, generator=gen, device="cuda").to(dtype) for _ in range(2)), 0)
    return cache


def want_rows(cache, q, owners):
    """The plain attention of each row: over all tokens of the request that it belongs to; none: 0."""
    lengths = cache.lengths.tolist()
    want, lse, bound, lse_bound = plain.attend(q, cache.keys[0], cache.values[0], cache.table[[max(b, 0) for b in owners]], [lengths[b] if b >= 0 else 0 for b in owners],
                                               1 / math.sqrt(D), cache.window)
    return want, lse, bound, lse_bound


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("new", [[1, 0, 1, 1, 0, 1], [0, 0, 0, 0, 0, 1], [1, 1, 1, 1, 1, 1], [0, 1, 0, 0, 0, 0]])
@pytest.mark.parametrize("spare", [True, False])
def test_idle_requests(Cache, new, spare, dtype):  # noqa: F811
    """A step of as many rows as there are requests (what a captured one has), or of no more than it needs: rows go on in order, those behind the last are 0."""
    cache = filled(Cache, [9, 20, 0, 70, 33, 1], dtype, window=40)
    tokens = R if spare else sum(new)
    qkv = torch.randn(tokens, HQ + 2 * HKV, D, device="cuda").to(dtype)
    cache.begin(dev(new), tokens)
    q = cache.append(qkv[:, :HQ], qkv[:, HQ:HQ + HKV], qkv[:, HQ + HKV:], 0)
    out, lse = cache.attend(q, 0, return_lse=True)
    owners = [b for b in range(R) if new[b]]
    want, want_lse, bound, lse_bound = want_rows(cache, q, owners + [-1] * (tokens - len(owners)))
    assert bool(((out.cpu().double() - want).abs() <= bound).all())
    n = len(owners)
    assert bool(((lse.cpu().double() - want_lse).abs() <= lse_bound)[:n].all()) and bool(torch.isneginf(lse[n:]).all()) and not bool(out[n:].any())
    assert cache.check() == 0


def test_rows_of_a_captured_step(Cache):  # noqa: F811
    """One graph, counts that change from replay to replay: idle requests take neither tokens nor pages."""
    cache = filled(Cache, [9, 20, 0, 70, 33, 1])
    new, qkv = dev([0] * R), torch.randn(R, HQ + 2 * HKV, D, device="cuda").half()

    def step():
        cache.begin(new, R)
        q = cache.append(qkv[:, :HQ], qkv[:, HQ:HQ + HKV], qkv[:, HQ + HKV:], 0)
        return q, cache.attend(q, 0)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q, out = step()
    lengths = [9, 20, 0, 70, 33, 1]
    for n in range(8):
        counts = [(n >> b) & 1 for b in range(3)] + [1, n % 2, 0]
        new.copy_(dev(counts))
        qkv.copy_(torch.randn_like(qkv))
        graph.replay()
        lengths = [held + add for held, add in zip(lengths, counts)]
        assert cache.lengths.tolist() == lengths and cache.head.item() == sum(-(-held // 8) for held in lengths)
        owners = [b for b in range(R) if counts[b]]
        want, _, bound, _ = want_rows(cache, q, owners + [-1] * (R - len(owners)))
        assert bool(((out.cpu().double() - want).abs() <= bound).all()), n
    assert cache.check() == 0


def test_rows_by_request(Cache):  # noqa: F811
    """Rows of one's own, one for each request whatever it brings: told so, or known by their number."""
    cache = filled(Cache, [9, 20, 0, 70, 33, 1])
    query = torch.randn(R, HQ, D, device="cuda").half()
    want, _, bound, _ = want_rows(cache, query, list(range(R)))
    assert bool(((cache.attend(query, 0).cpu().double() - want).abs() <= bound).all())       # (the prompts had 133 rows)
    cache.begin(dev([0] * R), R)
    assert torch.equal(cache.attend(query, 0, by_request=True), cache.attend(query, 0, by_request=True))
    assert bool(((cache.attend(query, 0, by_request=True).cpu().double() - want).abs() <= bound).all())
    assert not bool(cache.attend(query, 0).any())           # rows of a step in which no request has one


def test_more_than_one_row(Cache):  # noqa: F811
    """Two rows of a request are reported and 0, the others are right; a prompt's rows are refused."""
    from kvcomp_b200 import _lib
    cache = filled(Cache, [9, 20, 0, 70, 33, 1])
    cache.begin(dev([1, 2, 0, 1, 0, 0]), 5)
    q = torch.randn(5, HQ, D, device="cuda").half()
    out = cache.attend(q, 0)
    want, _, bound, _ = want_rows(cache, q, [0, -1, -1, 3, -1])
    assert bool(((out.cpu().double() - want).abs() <= bound).all())
    with pytest.raises(_lib.KvcError):
        cache.check()
    cache.begin(dev([4, 4, 0, 0, 0, 0]), 8)
    for q in (torch.randn(8, HQ, D, device="cuda").half(), torch.randn(3, HQ, D, device="cuda").half()):
        with pytest.raises(_lib.KvcError):
            cache.attend(q, 0)


def test_refused_requests(Cache):  # noqa: F811
    """A request that found no pages has a row without a slot: it attends over what it has, which may be nothing."""
    cache = Cache(R, 3, 1, HKV, D, page_size=8, max_tokens=100)
    x = torch.randn(R, HQ + 2 * HKV, D, device="cuda").half()
    cache.begin(dev([1, 1, 0, 1, 1, 0]), R)
    q = cache.append(x[:, :HQ], x[:, HQ:HQ + HKV], x[:, HQ + HKV:], 0)
    assert cache.lengths.tolist() == [1, 1, 0, 1, 0, 0]
    out = cache.attend(q, 0)
    group = HQ // HKV
    for row in range(3):
        assert torch.equal(out[row], x[row, HQ + HKV:].repeat_interleave(group, 0))        # one token: its value
    assert not bool(out[3:].any())


@pytest.mark.parametrize("heads,D,dtype", [((8, 2), 64, torch.float16), ((4, 4), 96, torch.bfloat16), ((16, 1), 128, torch.float16), ((6, 2), 128, torch.bfloat16), ((11, 1), 256, torch.float16),
                                           ((34, 2), 128, torch.float16)])
@pytest.mark.parametrize("lengths", ["edges", "many", "long"])
def test_operator(heads, D, dtype, lengths):
    """Every third request without a row, one with two; q and out are parts of larger tensors, whose other rows stay."""
    import numpy as np
    from kvcomp_b200 import _lib, ops
    from test_gpu_paged import LENGTHS
    lengths, page = LENGTHS[lengths], 16
    B, rng = len(lengths), np.random.RandomState(D)
    new = [b % 3 != 1 for b in range(B)]
    if B > 2:
        new[3] = 2
    starts, rows = np.concatenate([[0], np.cumsum(new)]).astype(np.int32), sum(new) + 5
    gen = torch.Generator(device="cuda").manual_seed(D)
    pages = int(sum(-(-n // page) for n in lengths)) + 3
    table, _, _ = plain.tables(rng, lengths, page, pages)
    kp, vp = (plain.pool(gen, pages, page, heads[1], D, dtype, "cuda") for _ in range(2))
    q = torch.randn(rows, heads[0] + 1, D, generator=gen, device="cuda").to(dtype)[:, 1:]
    whole = torch.full((rows + 2, heads[0], D), 7.0, device="cuda", dtype=dtype)
    status = ops.new_status("cuda")
    out, lse = ops.paged_attn(q, kp, vp, dev(table), dev(lengths), 0.2, out=whole[1:-1], return_lse=True, status=status, starts=dev(starts))
    assert status.item() == (_lib.FLAG_BAD_LENGTH if B > 2 else 0)
    owners = [b if new[b] == 1 else -1 for b in range(B) for _ in range(new[b])] + [-1] * 5
    want, want_lse, bound, lse_bound = plain.attend(q, kp, vp, dev(table[[max(b, 0) for b in owners]]), [lengths[b] if b >= 0 else 0 for b in owners], 0.2)
    assert bool(((out.cpu().double() - want).abs() <= bound).all())
    none = torch.isinf(want_lse)
    assert torch.equal(torch.isneginf(lse.cpu()), none) and bool(((lse.cpu().double() - want_lse).abs() <= lse_bound)[~none].all())
    assert bool((whole[0] == 7).all()) and bool((whole[-1] == 7).all())


def test_operator_keeps_inside_its_rows():
    """Numbers that are no plan's: nothing outside the tensors is read or written."""
    from kvcomp_b200 import ops
    gen = torch.Generator(device="cuda").manual_seed(2)
    kp, vp = (plain.pool(gen, 8, 16, 2, 64, torch.float16, "cuda") for _ in range(2))
    table, lengths = dev([[0, 1], [2, 3], [4, 5]]), dev([30, 20, 10])
    q = torch.randn(3, 4, 64, device="cuda").half()
    whole = torch.full((5, 4, 64), 7.0, device="cuda", dtype=torch.float16)
    for starts in ([-5, 1 << 30, -(1 << 31), (1 << 31) - 1], [3, 2, 1, 0], [7, 8, 9, 10], [-3, -2, -1, 0], [2, 3, 4, 5]):
        ops.paged_attn(q, kp, vp, table, lengths, 0.1, out=whole[1:-1], starts=dev(starts))
        assert bool((whole[0] == 7).all()) and bool((whole[-1] == 7).all())
    from kvcomp_b200._lib import KvcError
    for bad in (dev([0, 1, 2]), dev([0, 1, 2, 3], torch.int64), torch.zeros(4, dtype=torch.int32), [0, 1, 2, 3]):
        with pytest.raises(KvcError):
            ops.paged_attn(q, kp, vp, table, lengths, 0.1, starts=bad)
    assert ops.paged_attn(q[:0], kp, vp, table, lengths, 0.1, starts=dev([0, 0, 0, 0])).shape == (0, 4, 64)
