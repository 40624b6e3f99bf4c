"""Attention of requests that continue common prefixes, and the plan of who follows whom."""
import math

import numpy as np
import pytest
import torch

import paged_plain as plain

pytestmark = pytest.mark.gpu

DTYPES = [torch.float16, torch.bfloat16]


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    from kvcomp_b200 import ops
    return ops


def dev(a, dtype=torch.int32):
    return torch.as_tensor(np.asarray(a), dtype=dtype).cuda()


def groups_of(plan):
    """{(parent, shared): members in order} and each request's (group, rank) of a plan."""
    w, B = plan.words.tolist(), plan.requests
    groups = [w[4 + 4 * i:8 + 4 * i] for i in range(B)]             # first member, members, parent, shared
    assert all(g == [0] * 4 for g in groups[w[0]:])
    owners, order = w[4 + 4 * B:4 + 6 * B], w[4 + 6 * B:4 + 7 * B]
    return {(parent, shared): order[first:first + n] for first, n, parent, shared in groups[:w[0]]}, list(zip(owners[::2], owners[1::2]))


@pytest.mark.parametrize("B,holders", [(1, 1), (2, 1), (40, 3), (257, 5), (1025, 1), (2100, 700)])
def test_plan(ops, B, holders):
    rng = np.random.RandomState(B)
    parents = np.where(np.arange(B) < holders, -1, rng.randint(-1, holders, B))
    shared = rng.randint(0, 3, B) * 10
    order = rng.permutation(B)                                      # (who is followed lies anywhere)
    at = np.argsort(order)
    parents, shared = np.where(parents >= 0, at[parents], -1)[order], shared[order]
    status = ops.new_status(torch.device("cuda"))
    plan = ops.prefix_plan(dev(parents), dev(shared), status=status)
    want = {}
    for b in range(B):
        if parents[b] >= 0:
            want.setdefault((int(parents[b]), int(shared[b])), []).append(b)
    got, of = groups_of(plan)
    assert got == want and list(got) == list(want) and int(status.item()) == 0
    for b in range(B):
        key = (int(parents[b]), int(shared[b]))
        assert (of[b][0] == -1) if parents[b] < 0 else (list(want)[of[b][0]] == key and want[key][of[b][1]] == b)
    again = ops.prefix_plan(dev(parents), dev(shared), out=ops.PrefixPlan(torch.full_like(plan.words, 7), B))
    assert groups_of(again) == (got, of)


def test_plan_of_bad_parents(ops):
    from kvcomp_b200 import _lib
    for parents, shared, want in (([-1, 0, 9, 2], [5, 5, 5, 5], {(0, 5): [1], (2, 5): [3]}), ([0, 0], [1, 1], {(0, 1): [1]}), ([-1, 0], [1, -1], {}), ([-1, 0, 1], [0, 4, 4], {(0, 4): [1], (1, 4): [2]})):
        status = ops.new_status(torch.device("cuda"))
        got, _ = groups_of(ops.prefix_plan(dev(parents), dev(shared), status=status))
        assert got == want and int(status.item()) == _lib.FLAG_BAD_LENGTH


def test_a_plan_of_no_requests(ops):
    """It says so, and touches nothing around it, whatever the kernels ahead of it left in shared memory."""
    all_words = torch.full((1 << 16,), 7, dtype=torch.int32, device="cuda")
    plan = ops.PrefixPlan(all_words[1 << 15:(1 << 15) + 4], 0)
    want = all_words.clone()
    want[1 << 15] = 0
    for i in range(50):
        torch.sort(torch.full((1 << 14,), -1 - i, dtype=torch.int32, device="cuda"))
        plan.words[0] = 7
        assert ops.prefix_plan(dev([]), dev([]), out=plan) is plan and torch.equal(all_words, want)


def attend(ops, prefixes, members, own, Hq, Hkv, D, dtype, page=16, seed=0, sharp=1.0, scaling=None, order="token", rows="followers", shares=None, alone=0):
    """prefixes[i] tokens that members[i] requests follow, own tokens of each request from `own` in turn; `alone` requests follow no one."""
    rng = np.random.RandomState(seed + sum(prefixes) + page)
    gen = torch.Generator(device="cuda").manual_seed(seed + D)
    n = len(prefixes) + sum(members) + alone
    lengths = list(prefixes) + [own[i % len(own)] for i in range(sum(members) + alone)]
    parents = [-1] * len(prefixes) + [g for g, m in enumerate(members) for _ in range(m)] + [-1] * alone
    shared = [0] * len(prefixes) + [prefixes[g] if shares is None else shares[i % len(shares)] for i, g in enumerate(parents[len(prefixes):len(prefixes) + sum(members)])] + [0] * alone
    at = rng.permutation(n)                                         # the places of the requests in the cache
    place = lambda a, zero: np.array([a[i] for i in np.argsort(at)]) if zero is None else None  # noqa: E731
    lengths, shared = place(lengths, None), place(shared, None)
    parents = np.array([at[x] if x >= 0 else -1 for x in np.array(parents)[np.argsort(at)]])
    pages = sum(-(-int(x) // page) for x in lengths) + 3
    table, _, used = plain.tables(rng, [int(x) for x in lengths], page, pages, extra=1)
    kp, vp = (plain.pool(gen, pages, page, Hkv, D, dtype, "cuda", order) for _ in range(2))
    free = torch.ones(pages, page, dtype=torch.bool)
    for b, x in enumerate(lengths):
        for i in range(-(-int(x) // page)):
            free[table[b, i], :max(0, min(page, int(x) - i * page))] = False
    for pool in (kp, vp):                                           # what no request holds is never read
        pool[free.cuda()] = math.nan
    has = [rows == "all" or parents[b] >= 0 or (alone and b in set(at[n - alone:])) for b in range(n)]
    starts = None if rows == "all" else np.concatenate([[0], np.cumsum(has)])
    count = n if rows == "all" else int(starts[-1])
    spare = 0 if rows == "all" else 2
    q = (torch.randn(count + spare, Hq, D, generator=gen, device="cuda") * sharp).to(dtype)
    scaling = 1 / math.sqrt(D) if scaling is None else scaling
    status = ops.new_status(torch.device("cuda"))
    plan = ops.prefix_plan(dev(parents), dev(shared), status=status)
    workspace = ops.paged_attn_shared_workspace(n, Hq, Hkv, D, "cuda")
    from kvcomp_b200 import _lib
    workspace[_lib.load().kvc_paged_attn_cleared():].view(torch.int32).fill_(0x7fc00000)            # (nothing relies on what was there: NaN)
    call = lambda: ops.paged_attn_shared(q, kp, vp, dev(table), dev(lengths), plan, scaling, return_lse=True, workspace=workspace, status=status, starts=None if starts is None else dev(starts))  # noqa: E731
    out, lse = call()
    assert int(status.item()) == 0
    again, lse2 = call()
    assert torch.equal(out, again) and torch.equal(lse, lse2)
    assert not bool(out[count:].any()) and bool(torch.isneginf(lse[count:]).all())
    out, lse, x = out.cpu().double(), lse.cpu().double(), q.cpu().double()
    kc, vc = kp.cpu().double(), vp.cpu().double()
    g, eps, worst = Hq // Hkv, torch.finfo(dtype).eps / 2, 0.0
    for b in range(n):
        if not has[b]:
            continue
        row = b if starts is None else int(starts[b])
        t = [(table[b, i // page], i % page) for i in range(int(lengths[b]))]
        if parents[b] >= 0:
            t = [(table[parents[b], i // page], i % page) for i in range(int(shared[b]))] + t
        if not t:
            assert not bool(out[row].any()) and bool(torch.isneginf(lse[row]).all())
            continue
        t = torch.as_tensor(np.array(t)).long()
        k, v = kc[t[:, 0], t[:, 1]], vc[t[:, 0], t[:, 1]]           # [tokens, kv heads, D]
        y = x[row].view(Hkv, g, D)
        s = torch.einsum("hgd,thd->hgt", y, k) * scaling
        size = abs(scaling) * torch.einsum("hgd,thd->hgt", y.abs(), k.abs())
        w = torch.softmax(s, -1)
        want, want_lse = torch.einsum("hgt,thd->hgd", w, v), torch.logsumexp(s, -1)
        # An fp32 score is off by D products and sums of magnitude sum |q k| (2^-23 each: tensor cores may cut off) and by roundings on the way to the exponent; with d that sum over the
        # largest token, a weight and the sum of weights are off by a factor 1 + d each.  A weight is rounded to 16 bits: half a step, and below 2^-21 of the largest in fp16 half of 2^-31 of that
        # (2^7 times it, in steps of 2^-24).  The sums over L tokens: 2^-23 a step.
        d = size.amax(-1, keepdim=True) * (D + 4) * 2.0 ** -23 + (s.abs().amax(-1, keepdim=True) + 24) * 2.0 ** -22
        far = w.amax(-1, keepdim=True) * v.abs().sum(0)[:, None] * 2.0 ** -24 if dtype == torch.float16 else 0.0
        off = torch.einsum("hgt,thd->hgd", w, v.abs()) * (2 * d + eps + (len(t) + 64) * 2.0 ** -23) + far
        bound = off + eps * (want.abs() + off) + (2.0 ** -25 if dtype == torch.float16 else 0.0)
        near = (out[row].view(Hkv, g, D) - want).abs()
        worst = max(worst, float((near / bound).max()))
        assert bool((near <= bound).all()), (b, row, (near > bound).nonzero()[:4].tolist(), float((near / bound).max()))
        assert bool(((lse[row].view(Hkv, g) - want_lse).abs() <= 2 * d[..., 0] + (len(t) + 64) * 2.0 ** -23 + want_lse.abs() * 2.0 ** -23).all())
    return worst


@pytest.mark.parametrize("D", [128, 64, 96])
@pytest.mark.parametrize("dtype", DTYPES)
def test_one_tile(ops, dtype, D):
    attend(ops, [100], [2], [5], 1, 1, D, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 96, 128])
@pytest.mark.parametrize("Hq,Hkv", [(2, 2), (8, 2), (7, 1), (16, 1), (34, 2), (40, 10)])
def test_heads(ops, dtype, D, Hq, Hkv):
    attend(ops, [300], [3], [40, 1, 200], Hq, Hkv, D, dtype)


@pytest.mark.parametrize("members", [1, 15, 16, 17, 32, 33, 64, 65, 100])
@pytest.mark.parametrize("prefix", [1, 127, 128, 129, 1000])
def test_rows_of_a_group(ops, members, prefix):
    """8 query heads on a KV head: half a set of rows, one, two, and columns of 256 rows with a rest."""
    attend(ops, [prefix], [members], [3, 0, 130], 16, 2, 128, torch.bfloat16, seed=members)


@pytest.mark.parametrize("page", [1, 5, 16, 24, 64, 128, 256])
@pytest.mark.parametrize("dtype", DTYPES)
def test_pages(ops, page, dtype):
    attend(ops, [777, 130, 1], [3, 17, 2], [0, 1, 15, 16, 127, 128, 129, 300], 8, 2, 128, dtype, page=page)


@pytest.mark.parametrize("order", ["head", "padded"])
@pytest.mark.parametrize("D", [64, 96, 128])
def test_strides(ops, order, D):
    attend(ops, [400, 20], [5, 3], [33, 1], 8, 4, D, torch.float16, order=order, page=24)


def test_different_shares_of_one_parent(ops):
    """Followers of one request with prefixes of different length: groups of their own."""
    attend(ops, [500], [20], [7], 8, 2, 128, torch.float16, shares=[500, 100, 0, 127, 128])


@pytest.mark.parametrize("rows", ["all", "followers"])
def test_requests_that_follow_no_one(ops, rows):
    attend(ops, [300, 0], [4, 2], [50, 0, 260], 8, 2, 128, torch.float16, rows=rows, alone=3)


@pytest.mark.parametrize("dtype", DTYPES)
def test_weights_of_every_size(ops, dtype):
    """Sharp weights, whose maximum grows late and often; scores of both signs and none."""
    attend(ops, [2000], [20], [300], 8, 2, 128, dtype, sharp=20.0)
    attend(ops, [2000], [20], [300], 8, 2, 64, dtype, scaling=-0.3)
    attend(ops, [700], [3], [30], 8, 2, 128, dtype, scaling=0.0)
    attend(ops, [700], [3], [30], 8, 2, 96, dtype, scaling=3.0)


@pytest.mark.parametrize("dtype", DTYPES)
def test_long_prefixes(ops, dtype):
    """Columns that several CTAs share, narrow and wide ones in one share."""
    attend(ops, [6000, 3001], [9, 3], [100, 700], 32, 2, 128, dtype, page=64)
    attend(ops, [9000], [40], [100, 300, 0], 8, 1, 64, dtype, page=64)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("prefix", [128, 500, 640, 5000, 20001])
def test_few_rows_behind_long_prefixes(ops, prefix, dtype):
    """Few rows, whose columns are cut into one to more than a hundred parts: these are joined by four warps a head, from some number of rows on by one."""
    attend(ops, [prefix, prefix // 2], [3, 1], [25, 0, 7], 14, 2, 128, dtype, page=24)
    attend(ops, [prefix], [2], [0], 36, 1, 64, dtype, page=24)
    attend(ops, [prefix], [2], [3], 38, 1, 96, dtype, page=24, sharp=20.0)


def test_many_requests(ops):
    """More items than a CTA looks at at once."""
    attend(ops, [200] * 5, [90] * 5, [1, 0, 3], 2, 1, 64, torch.float16, page=8)


def test_bad_pages_and_lengths(ops):
    from kvcomp_b200 import _lib
    kp, vp = (torch.randn(4, 16, 1, 64, device="cuda").half() for _ in range(2))
    q, status = torch.randn(3, 2, 64, device="cuda").half(), ops.new_status(torch.device("cuda"))
    plan = ops.prefix_plan(dev([-1, 0, 0]), dev([0, 20, 20]))
    table = dev([[0, 1], [2, 9], [3, -1]])
    out = ops.paged_attn_shared(q, kp, vp, table, dev([20, 20, 3]), plan, 0.1, status=status)
    assert int(status.item()) == _lib.FLAG_BAD_PAGE
    for b, t in ((0, [(0, 16), (1, 4)]), (1, [(0, 16), (1, 4), (2, 16)]), (2, [(0, 16), (1, 4), (3, 3)])):
        k, v = (torch.cat([pool[p, :n, 0] for p, n in t]).double() for pool in (kp, vp))
        want = torch.softmax(0.1 * (q[b].double() @ k.T), -1) @ v
        assert bool(((out[b].double() - want).abs() <= 2e-3 * v.abs().max()).all())
    for lengths in ([10, 20, 3], [99, 1, 1], [20, -1, 3]):          # a parent that has fewer tokens than are shared, lengths that are none
        status.zero_()
        out = ops.paged_attn_shared(q, kp, vp, dev([[0, 1], [2, 2], [3, 3]]), dev(lengths), plan, 0.1, status=status)
        assert int(status.item()) == _lib.FLAG_BAD_LENGTH and bool(torch.isfinite(out).all())
    status.zero_()
    out = ops.paged_attn_shared(q, kp, vp, dev([[0, 1], [2, 2], [3, 3]]), dev([20, 20, 3]), plan, 0.1, status=status, starts=dev([0, 0, 2, 3]))       # two rows of one request
    assert int(status.item()) == _lib.FLAG_BAD_LENGTH and not bool(out[:2].any()) and bool(out[2].any())


def test_many_groups(ops):
    """More groups than a CTA has threads, of one request each."""
    attend(ops, [17] * 600, [1] * 600, [2, 0], 2, 1, 64, torch.bfloat16, page=8)


def test_many_heads_of_one_request(ops):
    """One follower with more query heads on a KV head than both sets have rows."""
    attend(ops, [500], [1], [30], 300, 1, 64, torch.float16)
    attend(ops, [500], [2], [30], 260, 2, 128, torch.bfloat16)


def test_the_result_in_the_queries_place(ops):
    kp, vp = (torch.randn(8, 16, 2, 128, device="cuda").half() for _ in range(2))
    q, plan = torch.randn(3, 8, 128, device="cuda").half(), ops.prefix_plan(dev([-1, 0, 0]), dev([0, 40, 40]))
    args = kp, vp, dev([[0, 1, 2], [3, 4, 5], [6, 7, 7]]), dev([40, 33, 1]), plan, 0.1
    want = ops.paged_attn_shared(q, *args)
    wide = torch.randn(3, 10, 128, device="cuda").half()
    into = ops.paged_attn_shared(q, *args, out=wide[:, 1:9])
    assert into.data_ptr() == wide[:, 1:9].data_ptr() and torch.equal(into, want)
    assert torch.equal(ops.paged_attn_shared(q, *args, out=q), want) and torch.equal(q, want)


def test_long_offsets(ops):
    """Pages that lie behind 2^32 elements of the pool."""
    pages, page, Hkv, D = 36000, 64, 16, 128
    pool = torch.zeros(pages, page, Hkv, D, dtype=torch.float16, device="cuda")
    table = np.array([[35999, 35000, 1, 35998], [35997, 2, 35996, 0], [3, 35995, 0, 0]])
    for p in np.unique(table):
        pool[int(p)] = torch.randn(page, Hkv, D, device="cuda").half()
    q = torch.randn(3, 2 * Hkv, D, device="cuda").half()
    plan = ops.prefix_plan(dev([-1, 0, 0]), dev([0, 250, 250]))
    out = ops.paged_attn_shared(q, pool, pool, dev(table), dev([250, 200, 70]), plan, 0.1)
    for b, own in ((1, 200), (2, 70)):
        for h in (0, 31):
            rows = torch.cat([torch.cat([pool[int(p), :, h // 2] for p in table[i]])[:n] for i, n in ((0, 250), (b, own))]).double()
            want = torch.softmax(0.1 * (q[b, h].double() @ rows.T), -1) @ rows
            assert bool(((out[b, h].double() - want).abs() <= 2.0 ** -9 * rows.abs().max()).all())


def test_refusals(ops):
    from kvcomp_b200._lib import KvcError
    kp, vp = (torch.randn(4, 16, 2, 128, device="cuda").half() for _ in range(2))
    q, table, lengths, plan = torch.randn(2, 4, 128, device="cuda").half(), dev([[0], [1]]), dev([3, 4]), ops.prefix_plan(dev([-1, 0]), dev([0, 3]))
    good = dict(q=q, kpages=kp, vpages=vp, table=table, lengths=lengths, plan=plan, scaling=0.1)
    workspace = ops.paged_attn_shared_workspace(2, 4, 2, 128, "cuda")
    ops.paged_attn_shared(**good, workspace=workspace)
    odd = torch.empty(workspace.numel() + 16, dtype=torch.uint8, device="cuda")[16:]
    bad_pool = torch.randn(4, 16, 2, 256, device="cuda").half()
    for change in (dict(plan=ops.prefix_plan(dev([-1]), dev([0]))), dict(plan=None), dict(plan=ops.PrefixPlan(plan.words.cpu(), 2)), dict(lengths=lengths[:1]), dict(table=table.long()), dict(kpages=kp.float()),
                   dict(q=q.bfloat16()), dict(workspace=workspace[:-32]), dict(workspace=odd), dict(q=torch.randn(2, 4, 256, device="cuda").half(), kpages=bad_pool, vpages=bad_pool), dict(starts=dev([0, 1])),
                   dict(out=torch.empty(2, 4, 64, device="cuda").half()), dict(out=q.expand(2, 4, 128).as_strided((2, 4, 128), (128, 128, 1)))):
        with pytest.raises(KvcError):
            ops.paged_attn_shared(**{**good, **change})
    for parents, shared in ((dev([0]), dev([0, 1])), (dev([0]).long(), dev([0])), (dev([0]), dev([0]).cpu())):
        with pytest.raises(KvcError):
            ops.prefix_plan(parents, shared)
    assert ops.paged_attn_shared(q[:0], kp, vp, table[:0], lengths[:0], ops.prefix_plan(dev([]), dev([])), 0.1).shape == (0, 4, 128)
