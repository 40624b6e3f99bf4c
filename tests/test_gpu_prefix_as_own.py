"""Requests that follow a prefix have the results of requests that hold the same tokens themselves: as exact, and the same where values are infinite."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.float16, torch.bfloat16]


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    from kvcomp_b200 import ops
    return ops


def ints(a):
    return torch.tensor(a, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 96, 128])
@pytest.mark.parametrize("members,Hq,tokens", [(1, 1, 512), (3, 4, 700), (40, 8, 900), (2, 1, 30000)])
def test_weights_that_round_alike(ops, dtype, D, members, Hq, tokens):
    """All but every 64th token have a weight next to the middle of two numbers of 16 bits: one rounding of weights is off by half a step, in one direction, beside the result's."""
    eps = torch.finfo(dtype).eps / 2
    weight = (1 + 0.97 * eps) / 8
    scaling = -math.log(weight)
    page = 64
    pages = -(-tokens // page) + members
    kp, vp = (torch.zeros(pages, page, 1, D, dtype=dtype, device="cuda") for _ in range(2))
    kp[:, 1:, 0, 0] = -1.0
    v = (1 + torch.arange(D, device="cuda") / D).to(dtype)
    vp[:, 1:, 0] = v
    q = torch.zeros(members + 1, Hq, D, dtype=dtype, device="cuda")
    q[:, :, 0] = 1.0
    table = torch.full((members + 1, pages), -1, dtype=torch.int32, device="cuda")
    own = 33
    table[0, :pages - members] = torch.arange(pages - members)
    table[1:, 0] = torch.arange(pages - members, pages)
    plan = ops.prefix_plan(ints([-1] + [0] * members), ints([0] + [tokens] * members))
    out = ops.paged_attn_shared(q, kp, vp, table, ints([tokens] + [own] * members), plan, scaling)
    large = -(-tokens // 64) + 1
    small = tokens + own - large
    want = v.double() * small * weight / (large + small * weight)
    # A score is one product (the others are 0), scaled: with the sum's steps its weight is off by (D + 4) 2^-23 of 2.1 and 27 2^-22 (as in the tests of prefixes), two pieces of 16 bits by
    # 2^-20 (fp16) and 2^-16 (bf16); the sums by 2^-23 a step, of up to 128 tokens' partial sums and the parts that are joined; then the result is rounded.
    d = 2.1 * (D + 4) * 2.0 ** -23 + 27 * 2.0 ** -22
    off = want * (2 * d + (2.0 ** -20 if dtype == torch.float16 else 2.0 ** -16) + (tokens / 8 + 512) * 2.0 ** -23)
    bound = off + eps * (want + off)
    error = (out[1:].double() - want).abs()
    assert bool((error <= bound).all()), float((error / bound).max())


def both(ops, kp, vp, q, prefix, owns, page, Hq):
    """(with a prefix, by a table that names its pages) of requests 1.. behind request 0."""
    R = len(owns) + 1
    n = prefix // page
    table = torch.full((R, 12), -1, dtype=torch.int32, device="cuda")
    table[0, :n] = torch.arange(n)
    whole, at = table.clone(), n
    for b, own in enumerate(owns):
        more = -(-own // page)
        table[b + 1, :more] = torch.arange(at, at + more)
        whole[b + 1, :n], whole[b + 1, n:n + more] = torch.arange(n), torch.arange(at, at + more)
        at += more
    plan = ops.prefix_plan(ints([-1] + [0] * (R - 1)), ints([0] + [prefix] * (R - 1)))
    shared = ops.paged_attn_shared(q.clone(), kp, vp, table, ints([prefix] + owns), plan, 0.1)
    place = q.clone()
    assert torch.equal(ops.paged_attn_shared(place, kp, vp, table, ints([prefix] + owns), plan, 0.1, out=place).nan_to_num(7.0, 8.0, 9.0), shared.nan_to_num(7.0, 8.0, 9.0))
    alone = ops.paged_attn(q, kp, vp, whole, ints([prefix] + [prefix + own for own in owns]), 0.1)
    return shared, alone


VALUES = {"inf": [(17, 3, math.inf)], "-inf": [(300, 0, -math.inf)], "both": [(17, 3, math.inf), (120, 3, -math.inf)], "nan": [(5, 60, math.nan)], "own": [(401, 9, math.inf)], "own and prefix": [(402, 9, math.inf), (3, 9, -math.inf)],
          "two": [(17, 3, math.inf), (399, 3, math.inf), (50, 63, -math.inf)], "many": [(t, t % 64, math.inf if t % 2 else -math.inf) for t in range(0, 64)]}


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D,Hq,Hkv,members", [(64, 2, 2, 3), (128, 8, 2, 3), (96, 6, 1, 30), (128, 16, 1, 20)])
@pytest.mark.parametrize("case", sorted(VALUES))
@pytest.mark.parametrize("far", [False, True])
def test_infinite_values(ops, case, dtype, D, Hq, Hkv, members, far):
    """An infinity that counts is the result, however small its weight; two of different signs, or what is no number, none: as in calls without prefixes."""
    gen = torch.Generator(device="cuda").manual_seed(D + Hq)
    page, prefix = 16, 160
    owns = [1 + 7 * i % 30 for i in range(members)]
    pages = prefix // page + sum(-(-o // page) for o in owns)
    kp, vp = (torch.randn(pages, page, Hkv, D, generator=gen, device="cuda").to(dtype) for _ in range(2))
    q = torch.randn(members + 1, Hq, D, generator=gen, device="cuda").to(dtype)
    for t, c, x in VALUES[case]:
        at = prefix + t - 401 if t > 400 else t % prefix
        vp[at // page, at % page, 0, c % D] = x
        if far:                                                     # a weight of nothing in 16 bits, and in 32
            kp[at // page, at % page, 0] = -40.0 * q[1, 0]
    shared, alone = both(ops, kp, vp, q, prefix, owns, page, Hq)
    for f in (torch.isnan, torch.isposinf, torch.isneginf):
        assert torch.equal(f(shared), f(alone))
    fine = torch.isfinite(alone)
    assert bool((~fine).any()) and bool(((shared.double() - alone.double()).abs()[fine] <= 4 * torch.finfo(dtype).eps).all())


@pytest.mark.parametrize("dtype", DTYPES)
def test_infinities_without_any_weight(ops, dtype):
    """An infinite value whose score is -infinity (an infinite key) is 0 times an infinity: no number; keys that are infinite beside finite values leave no trace."""
    gen = torch.Generator(device="cuda").manual_seed(1)
    D, page, prefix, owns = 128, 16, 96, [5, 20]
    kp, vp = (torch.randn(12, page, 1, D, generator=gen, device="cuda").to(dtype) for _ in range(2))
    q = torch.randn(3, 2, D, generator=gen, device="cuda").abs().to(dtype)
    for at, value in ((7, None), (50, math.inf), (prefix + 2, None)):
        kp[at // page, at % page, 0, 5] = -math.inf
        if value is not None:
            vp[at // page, at % page, 0, 9] = value
    shared, alone = both(ops, kp, vp, q, prefix, owns, page, 2)
    assert torch.equal(torch.isnan(shared), torch.isnan(alone)) and bool(torch.isnan(shared[1:, :, 9]).all()) and bool(torch.isfinite(shared[..., :9]).all())
    fine = torch.isfinite(alone)
    assert bool(((shared.double() - alone.double()).abs()[fine] <= 4 * torch.finfo(dtype).eps).all())


def test_few_rows_behind_a_long_prefix(ops):
    """Columns of many parts, joined by several warps, with one infinity far from the others."""
    gen = torch.Generator(device="cuda").manual_seed(3)
    D, page, tokens = 128, 64, 20032
    kp, vp = (torch.randn(tokens // page + 2, page, 2, D, generator=gen, device="cuda").half() for _ in range(2))
    q = torch.randn(3, 8, D, generator=gen, device="cuda").half()
    vp[200, 7, 1, 100] = -math.inf
    n = tokens // page
    table = torch.full((3, n + 1), -1, dtype=torch.int32, device="cuda")
    table[0, :n], table[1, 0], table[2, 0] = torch.arange(n), n, n + 1
    plan = ops.prefix_plan(ints([-1, 0, 0]), ints([0, tokens, tokens]))
    out = ops.paged_attn_shared(q, kp, vp, table, ints([tokens, 30, 1]), plan, 0.1)
    want = torch.zeros_like(out, dtype=torch.bool)
    want[:, 4:, 100] = True
    assert torch.equal(torch.isneginf(out), want) and bool(torch.isfinite(out[~want]).all())
