"""Attention over values (and keys) that are infinite or no numbers in rows that count: what the definition says, channel by channel."""
import math

import numpy as np
import pytest
import torch

import paged_plain as plain
from test_gpu_paged import dev, ops  # noqa: F401  (the fixture)

pytestmark = pytest.mark.gpu

INF, NAN = math.inf, math.nan


def check(ops, lengths, Hq, Hkv, D, dtype, plant, page=16, window=0, sharp=1.0, seed=0):
    """plant(put): put(request, token, KV head, channel, value, keys=False) changes single elements of the pools."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    pages = int(sum(-(-n // page) for n in lengths)) + 3
    table, _, _ = plain.tables(np.random.RandomState(seed), lengths, page, pages)
    kp, vp = (plain.pool(gen, pages, page, Hkv, D, dtype, "cuda") for _ in range(2))
    q = sharp * torch.randn(len(lengths), Hq, D, generator=gen, device="cuda").to(dtype)

    def put(b, t, h, d, value, keys=False):
        (kp if keys else vp)[int(table[b, t // page]), t % page, h, d] = value
    plant(put)
    args = (q, kp, vp, dev(table), dev(lengths), 1 / math.sqrt(D))
    out, lse = ops.paged_attn(*args, window=window, return_lse=True)
    want, want_lse, bound, lse_bound = plain.attend(*args[:4], lengths, args[5], window)
    got, odd = out.cpu().double(), ~torch.isfinite(want)
    assert bool(odd.any())
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(torch.isposinf(got), torch.isposinf(want)) and torch.equal(torch.isneginf(got), torch.isneginf(want))
    assert bool(((got - want).abs() <= bound)[~odd].all())
    fine = torch.isfinite(want_lse)
    assert bool(((lse.cpu().double() - want_lse).abs() <= lse_bound)[fine].all())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("Hq,Hkv,D", [(4, 4, 64), (8, 2, 96), (4, 2, 128), (2, 1, 256), (16, 1, 128), (20, 1, 64)])
def test_values(ops, Hq, Hkv, D, dtype):  # noqa: F811
    """One infinity of each sign, both in one channel, no number, in requests of one token, of one tile, of many parts; rows beside them are as ever."""
    lengths = [1, 17, 64, 5000, 0, 300, 12000]

    def plant(put):
        for b, n in enumerate(lengths):
            if not n or b == 5:                             # (request 5 stays finite)
                continue
            for h in range(Hkv):
                put(b, 0, h, 3, INF)
                put(b, n - 1, h, 17 + h, -INF)
                put(b, n // 2, h, D - 1, NAN)
                if n > 1:
                    put(b, n // 3, h, 40, INF), put(b, n - 1, h, 40, -INF)
                    put(b, n // 2, h, 8, INF), put(b, n - 1, h, 8, INF)
    check(ops, lengths, Hq, Hkv, D, dtype, plant)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_small_weights(ops, dtype):  # noqa: F811
    """Weights that are nothing in 32 bits are none by the definition: their infinities count."""
    check(ops, [40, 700, 2000], 4, 2, 128, dtype, lambda put: [put(b, t, h, 5 + t % 7, (-1) ** t * INF) for b in range(3) for h in range(2) for t in (0, 13, 39)], sharp=12.0)


@pytest.mark.parametrize("window", [16, 100])
def test_windows(ops, window):  # noqa: F811
    """Infinities before a window are not there, those inside are."""
    lengths = [90, 500, 3000]

    def plant(put):
        for b, n in enumerate(lengths):
            for h in range(2):
                put(b, n - window - 1 if n > window else 0, h, 1, INF)
                put(b, max(0, n - window), h, 2, -INF)
    check(ops, lengths, 4, 2, 64, torch.float16, plant, window=window)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_keys(ops, dtype):  # noqa: F811
    """A key of infinite size: scores of +inf leave no number; of -inf no weight, and 0 times an infinite value is none either."""
    def plant(put):
        for t in (3, 900):
            put(1, t, 0, 9, INF, keys=True)                 # (heads whose query is above 0 there: +inf; the others: -inf)
        put(1, 3, 0, 11, INF)
        put(2, 5, 0, 2, NAN, keys=True)
    check(ops, [50, 1000, 30], 4, 1, 64, dtype, plant, seed=5)


@pytest.mark.parametrize("Hq,Hkv,D", [(8, 4, 64), (4, 4, 96), (16, 2, 128), (4, 2, 256)])
def test_signs_side_by_side(ops, Hq, Hkv, D):  # noqa: F811
    """Infinities of two signs in neighbouring channels, everywhere; whole rows that are infinite, or no numbers."""
    lengths = [3, 700, 64, 2500]

    def plant(put):
        for h in range(Hkv):
            for d in range(0, 16, 2):
                put(0, 1, h, d, INF), put(0, 1, h, d + 1, -INF), put(1, 650, h, d, -INF), put(1, 2, h, d + 1, INF)
            for d in range(D):
                put(2, 63, h, d, INF if d % 3 else NAN), put(3, 2000, h, d, -INF)
    for dtype in (torch.float16, torch.bfloat16):
        check(ops, lengths, Hq, Hkv, D, dtype, plant)


@pytest.mark.parametrize("Hq,Hkv,D", [(8, 2, 64), (6, 3, 96), (16, 1, 128), (9, 1, 256)])
def test_packed_rows_and_in_place(ops, Hq, Hkv, D):  # noqa: F811
    """Infinities of requests whose rows are packed, some requests without one; where the result takes the queries' place."""
    gen = torch.Generator(device="cuda").manual_seed(D)
    lengths, page = [5000, 40, 1, 0, 9000, 300], 16
    pages = sum(-(-n // page) for n in lengths) + 1
    table, _, _ = plain.tables(np.random.RandomState(D), lengths, page, pages)
    kp, vp = (plain.pool(gen, pages, page, Hkv, D, torch.float16, "cuda") for _ in range(2))
    for b, n in enumerate(lengths):
        for t in {0, n // 2, n - 1} if n else ():
            vp[int(table[b, t // page]), t % page, :, 3 + b] = -INF if t and b > 3 else INF
    q = torch.randn(6, Hq, D, generator=gen, device="cuda").half()
    args = (kp, vp, dev(table), dev(lengths), 0.2)
    want = ops.paged_attn(q, *args)
    assert torch.isposinf(want).nonzero()[:, ::2].unique(dim=0).tolist() == [[0, 3], [1, 4], [2, 5]]
    assert torch.isnan(want).nonzero()[:, ::2].unique(dim=0).tolist() == [[4, 7], [5, 8]]
    rows = [0, 1, 2, 4, 5]
    got = ops.paged_attn(q[rows], *args, starts=dev([0, 1, 2, 3, 3, 4, 5]))
    torch.testing.assert_close(got, want[rows], rtol=0, atol=0, equal_nan=True)
    assert ops.paged_attn(q, *args, out=q) is q
    torch.testing.assert_close(q, want, rtol=0, atol=0, equal_nan=True)
