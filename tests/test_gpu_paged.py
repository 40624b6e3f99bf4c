"""The paged cache's operators against plain forms in 64 bits, at the sizes and masks where they can go wrong."""
import math

import numpy as np
import pytest
import torch

import paged_plain as plain

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    from kvcomp_b200 import ops
    return ops


def dev(a, dtype=torch.int32):
    return torch.as_tensor(np.asarray(a)).to(dtype).cuda()


# ---- pages ------------------------------------------------------------------------------------------------------

def check_plan(ops, lengths, new, table, free, head, page, tokens, in_place=False):
    want = plain.plan(list(lengths), list(new), table, free, head, page, tokens)
    d = dict(lengths=dev(lengths), new=dev(new), table=dev(table), free=dev(free), head=dev([head]))
    status = ops.new_status("cuda")
    out = None
    if in_place:
        B = len(lengths)
        spare = torch.full((2 * B + 1 + 2 * tokens,), -7, dtype=torch.int32, device="cuda").split((B + 1, B, tokens, tokens))
        out = ops.PagePlan(d["lengths"], d["head"], *spare)
    got = ops.page_plan(d["lengths"], d["new"], d["table"], d["free"], d["head"], page, tokens, out=out, status=status)
    for name in ("lengths", "starts", "taken", "slots", "positions"):
        assert getattr(got, name).tolist() == want[name], name
    assert got.head.item() == want["head"]
    assert np.array_equal(d["table"].cpu().numpy(), want["table"])
    assert d["free"].tolist() == list(free)
    if not in_place:
        assert d["lengths"].tolist() == list(lengths) and d["head"].item() == head
    from kvcomp_b200 import _lib
    flags = (_lib.FLAG_NO_PAGES if want["refused"] else 0) | (_lib.FLAG_BAD_LENGTH if min(list(lengths) + list(new) + [0]) < 0 else 0)
    assert status.item() == flags


@pytest.mark.parametrize("page", [1, 7, 16, 64])
@pytest.mark.parametrize("requests,most", [(1, 1), (1, 300), (3, 0), (33, 5), (257, 40), (1024, 1), (1025, 3), (4099, 2), (40, 3000)])
@pytest.mark.parametrize("in_place", [False, True])
def test_plan(ops, page, requests, most, in_place):
    rng = np.random.RandomState(page * 1000 + requests)
    lengths = rng.randint(0, 4 * page + 2, requests)
    new = rng.randint(0, most + 1, requests)
    need = int((-(-(lengths + new) // page) - -(-lengths // page)).sum())
    held = int((-(-lengths // page)).sum())
    table, free, head = plain.tables(rng, lengths, page, held + need + 3, extra=-(-most // page) + 1)
    check_plan(ops, lengths, new, table, free, head, page, int(new.sum()) + 5, in_place)


@pytest.mark.parametrize("requests,tokens", [(20, 64), (1500, 9000)])
def test_plan_refuses_whole_requests(ops, requests, tokens):
    """Pages run out in the middle, table rows are too short for some, negative numbers, rows for some tokens only."""
    rng = np.random.RandomState(requests)
    page = 8
    lengths, new = rng.randint(0, 40, requests), rng.randint(0, 30, requests)
    held = int((-(-lengths // page)).sum())
    need = int((-(-(lengths + new) // page) - -(-lengths // page)).sum())
    table, free, head = plain.tables(rng, lengths, page, held + need // 2, extra=1)
    check_plan(ops, lengths, new, table, free, head, page, tokens)
    check_plan(ops, lengths, new, table, free, head, page, int(new.sum()))
    lengths[3], new[5] = -4, -2
    check_plan(ops, lengths, new, table, free, head, page, int(np.maximum(new, 0).sum()))


def test_plan_of_nothing(ops):
    """No requests; no tokens; a pool without pages."""
    check_plan(ops, [], [], np.zeros((0, 4), np.int32), [3, 1, 2, 0], 1, 16, 0)
    check_plan(ops, [], [], np.zeros((0, 4), np.int32), [3, 1, 2, 0], 1, 16, 70)
    check_plan(ops, [5], [0], np.array([[2, -1]], np.int32), [2, 1], 1, 16, 0)
    check_plan(ops, [0, 0], [1, 0], np.zeros((2, 2), np.int32), [], 0, 16, 1)


def test_plan_of_one_long_prompt(ops):
    """Token rows of many pages, one request; behind it one that has room in its last page only."""
    rng = np.random.RandomState(4)
    table, free, head = plain.tables(rng, [100, 3], 16, 12000, extra=11000)
    check_plan(ops, [100, 3], [150001, 13], table, free, head, 16, 150014)


def test_plan_keeps_out_of_a_bad_free_list(ops):
    """Entries outside the pool (free list, table): their tokens have no slot, nothing is written elsewhere."""
    from kvcomp_b200 import _lib
    status = ops.new_status("cuda")
    table = dev([[9, -1, -1], [1, -1, -1]])
    p = ops.page_plan(dev([3, 4]), dev([1, 5]), table, dev([1, 0, -5, 70000000, 2, 3]), dev([2]), 4, 6, status=status)
    assert p.slots.tolist() == [-1] * 6 and p.positions.tolist() == [3, 4, 5, 6, 7, 8]
    assert status.item() == _lib.FLAG_BAD_PAGE
    status.zero_()
    p = ops.page_plan(dev([0]), dev([4]), dev([[-1]]), dev([1, 0]), dev([-9]), 4, 4, status=status)
    assert p.slots.tolist() == [4, 5, 6, 7] and status.item() == _lib.FLAG_BAD_LENGTH


@pytest.mark.parametrize("page,requests,longest", [(1, 5, 30), (16, 1, 1000), (16, 70, 100), (64, 1300, 300), (8, 3, 40000), (24, 2500, 500)])
@pytest.mark.parametrize("in_place", [False, True])
def test_release(ops, page, requests, longest, in_place):
    rng = np.random.RandomState(page + requests)
    lengths, done = rng.randint(0, longest + 1, requests), rng.rand(requests) < 0.5
    held = int((-(-lengths // page)).sum())
    table, free, head = plain.tables(rng, lengths, page, held + 9)
    want = plain.release(list(lengths), done, table, free, head, page)
    dl, dh, df = dev(lengths), dev([head]), dev(free)
    status = ops.new_status("cuda")
    out_lengths, out_head = ops.page_release(dl, dev(done, torch.bool), dev(table), df, dh, page, out=(dl, dh) if in_place else None, status=status)
    assert out_lengths.tolist() == want["lengths"] and out_head.item() == want["head"] and status.item() == 0
    assert np.array_equal(df.cpu().numpy(), want["free"])
    assert in_place or (dl.tolist() == list(lengths) and dh.item() == head)


def test_release_of_more_than_was_taken(ops):
    """A head below the requests' pages: the requests behind the last that fits keep theirs."""
    from kvcomp_b200 import _lib
    rng = np.random.RandomState(1)
    lengths, done = [30, 9, 64, 10], [True, True, True, True]
    table, free, _ = plain.tables(rng, lengths, 8, 20)
    want = plain.release(lengths, done, table, free, 7, 8)
    df, status = dev(free), ops.new_status("cuda")
    got, head = ops.page_release(dev(lengths), dev(done, torch.bool), dev(table), df, dev([7]), 8, status=status)
    assert got.tolist() == want["lengths"] == [0, 0, 64, 10] and head.item() == want["head"] == 1
    assert np.array_equal(df.cpu().numpy(), want["free"]) and status.item() == _lib.FLAG_NO_PAGES


def test_plan_and_release_in_a_graph(ops):
    """Prompts admitted and given back by replays, in place, with rows and pages enough for the second kernels."""
    rng = np.random.RandomState(5)
    page, B, pages = 4, 70, 9000
    new = rng.randint(0, 300, B)
    tokens = int(new.sum())
    table, free, _ = plain.tables(rng, [0] * B, page, pages, extra=200)
    state = [dev([0] * B), dev(table), dev(free), dev([0])]
    done = dev(rng.rand(B) < 0.5, torch.bool)
    out = ops.PagePlan(state[0], state[3], *torch.zeros(2 * B + 1 + 2 * tokens, dtype=torch.int32, device="cuda").split((B + 1, B, tokens, tokens)))
    status = ops.new_status("cuda")
    dnew = dev(new)

    def step():
        ops.page_plan(state[0], dnew, state[1], state[2], state[3], page, tokens, out=out, status=status)
        ops.page_release(state[0], done, state[1], state[2], state[3], page, out=(state[0], state[3]), status=status)

    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    from kvcomp_b200 import _lib
    lengths, head, refused = [0] * B, 0, False
    for _ in range(3):
        want = plain.plan(lengths, list(new), table, list(free), head, page, tokens)
        refused |= want["refused"]                          # (the third time some table rows are full)
        table = want["table"]
        graph.replay()
        assert out.slots.tolist() == want["slots"] and out.positions.tolist() == want["positions"] and out.starts.tolist() == want["starts"]
        back = plain.release(want["lengths"], done.tolist(), table, free, want["head"], page)
        lengths, head, free = back["lengths"], back["head"], back["free"]
        assert state[0].tolist() == lengths and state[3].item() == head
        assert np.array_equal(state[1].cpu().numpy(), table) and np.array_equal(state[2].cpu().numpy(), free)
    assert status.item() == (_lib.FLAG_NO_PAGES if refused else 0)


# ---- rotation ---------------------------------------------------------------------------------------------------

def freqs(n, base=10000.0):
    return base ** (-torch.arange(n, dtype=torch.float64) / max(n, 1))


def near(got, want, bound):
    d = (got.cpu().double() - want.cpu()).abs()
    assert bool((d <= bound.cpu()).all()), float((d - bound.cpu()).max())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("N,H,D,r", [(1, 1, 128, 128), (7, 32, 128, 128), (33, 5, 96, 96), (19, 3, 96, 72), (65, 4, 256, 64), (5, 2, 80, 20), (1031, 8, 128, 32), (3, 1, 6, 2),
                                     (130, 3, 64, 64), (2, 130, 64, 0), (300, 1, 40, 6)])
def test_rotary(ops, dtype, layout, N, H, D, r):
    gen = torch.Generator(device="cuda").manual_seed(N + D)
    x = torch.randn(N, H, D, generator=gen, device="cuda").to(dtype)
    pos = torch.randint(0, 1 << 20, (N,), generator=gen, device="cuda", dtype=torch.int32)
    pos[0] = 0
    f = freqs(r // 2).cuda()
    for inverse, factor in ((False, 1.0), (True, 1.25)):
        got = ops.rotary(x, pos, f, layout=layout, factor=factor, inverse=inverse)
        want = plain.rotate(x.cpu(), pos.cpu(), f.cpu(), layout, factor, inverse)
        near(got, want, plain.rotate_bound(x.cpu(), want, f, layout, factor))
        assert torch.equal(got[..., r:], x[..., r:])
    if r:
        assert torch.equal(ops.rotary(x, torch.zeros_like(pos), f, layout=layout), x)
    assert torch.equal(ops.rotary(x, pos, None), x)


def test_rotary_in_place_far_and_negative(ops):
    """Positions up to the largest, below 0, on strided rows, written where they were read."""
    x = torch.randn(6, 3, 3, 64, device="cuda").half()
    part = x[:, :, 1]
    pos = dev([2 ** 31 - 1, -(2 ** 31), -1, 123456789, 1, 0])
    f = freqs(32).cuda()
    want = plain.rotate(part.cpu(), pos.cpu(), f.cpu(), "half")
    bound = plain.rotate_bound(part.cpu(), want, f, "half", 1.0) + 4 * 2.0 ** 31 * 2.0 ** -53 * part.cpu().double().abs().max()      # the fp64 angle's own rounding, twice
    rest = x[:, :, 0].clone(), x[:, :, 2].clone()
    ops.rotary(part, pos, f, out=part)
    near(part, want, bound)
    assert torch.equal(x[:, :, 0], rest[0]) and torch.equal(x[:, :, 2], rest[1])


def test_rotary_gradient(ops):
    """The inverse rotation is the rotation's gradient: against differences of the plain form, and <R x, g> = <x, R^-1 g>."""
    gen = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(4, 2, 32, generator=gen, device="cuda").half()
    g = torch.randn(4, 2, 32, generator=gen, device="cuda").half()
    pos, f = dev([0, 5, 1000, 70000]), freqs(12).cuda()
    for layout in ("half", "interleaved"):
        back = ops.rotary(g, pos, f, layout=layout, factor=1.5, inverse=True)
        xd, gd = x.cpu().double(), g.cpu().double()
        want = torch.zeros_like(xd)
        for d in range(32):
            e = torch.zeros(32, dtype=torch.float64)
            e[d] = 2.0 ** -10
            up, down = (plain.rotate(xd + s * e, pos.cpu(), f.cpu(), layout, 1.5) for s in (1, -1))
            want[..., d] = ((up - down) * gd).sum(-1) / 2.0 ** -9
        bound = plain.rotate_bound(g.cpu(), want, f, layout, 1.5) + 2.0 ** -40 * 100
        near(back, want, bound)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("N,Hq,Hkv,D,r,page,order,layout", [
    (1, 32, 32, 128, 128, 64, "token", "half"), (13, 8, 2, 128, 96, 16, "head", "half"), (50, 6, 3, 96, 96, 24, "padded", "interleaved"),
    (700, 5, 5, 64, 32, 7, "token", "interleaved"), (9, 0, 4, 256, 256, 1, "token", "half"), (21, 7, 1, 72, 18, 5, "head", "half"), (257, 40, 10, 128, 0, 128, "token", "half")])
def test_store(ops, dtype, N, Hq, Hkv, D, r, page, order, layout):
    """A projection's slices go rotated to q's output and to their slots; rows without a slot, and every other row of the pools, stay."""
    from kvcomp_b200 import _lib
    gen = torch.Generator(device="cuda").manual_seed(N)
    rng = np.random.RandomState(N)
    qkv = torch.randn(N, Hq + 2 * Hkv, D, generator=gen, device="cuda").to(dtype)
    q, k, v = qkv[:, :Hq], qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:]
    pages = -(-N // page) + 3
    kp, vp = (plain.pool(gen, pages, page, Hkv, D, dtype, "cuda", order) for _ in range(2))
    k0, v0 = kp.clone(), vp.clone()
    slots = rng.permutation(pages * page)[:N].astype(np.int32)
    kept = np.ones(N, bool)
    if N > 4:
        slots[2], slots[4] = -1, pages * page
        kept[2] = kept[4] = False
    pos = dev(rng.randint(0, 100000, N))
    f = freqs(r // 2).cuda() if r else None
    status = ops.new_status("cuda")
    out = ops.rotary_paged_store(q if Hq else None, k, v, pos, dev(slots), f, kp, vp, layout=layout, factor=1.1, status=status)
    fc = f.cpu() if r else torch.zeros(0, dtype=torch.float64)
    if Hq:
        want = plain.rotate(q.cpu(), pos.cpu(), fc, layout, 1.1)
        near(out, want, plain.rotate_bound(q.cpu(), want, fc, layout, 1.1))
    else:
        assert out is None
    rows, cols = torch.as_tensor(slots[kept] // page).long().cuda(), torch.as_tensor(slots[kept] % page).long().cuda()
    at = torch.as_tensor(kept)
    want = plain.rotate(k.cpu(), pos.cpu(), fc, layout, 1.1)[at]
    near(kp[rows, cols], want, plain.rotate_bound(k.cpu()[at], want, fc, layout, 1.1))
    assert torch.equal(vp[rows, cols], v[at.cuda()])
    kp[rows, cols], vp[rows, cols] = k0[rows, cols], v0[rows, cols]
    assert torch.equal(kp, k0) and torch.equal(vp, v0)
    assert status.item() == (_lib.FLAG_BAD_PAGE if N > 4 else 0)


# ---- attention --------------------------------------------------------------------------------------------------

LENGTHS = {"edges": [0, 1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 128, 129, 255, 257, 500, 0],
           "one": [1], "none": [0, 0, 0], "long": [5000, 3], "even": [640] * 9, "many": [(7 * i) % 90 for i in range(300)]}


def attend(ops, lengths, Hq, Hkv, D, dtype, page=16, window=0, order="token", seed=0, poison=True, sharp=1.0, workspace=None):
    """Runs the operator and the plain form on a pool whose unread rows hold NaN and infinities."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rng = np.random.RandomState(seed)
    pages = int(sum(-(-n // page) for n in lengths)) + 3
    table, _, _ = plain.tables(rng, lengths, page, pages, extra=1)
    kp, vp = (plain.pool(gen, pages, page, Hkv, D, dtype, "cuda", order) for _ in range(2))
    q = sharp * torch.randn(len(lengths), Hq + 2, D, generator=gen, device="cuda").to(dtype)[:, 1:Hq + 1]
    if poison:
        used = torch.zeros(pages, page, dtype=torch.bool)
        for b, n in enumerate(lengths):
            t = np.arange(max(0, n - window) if window else 0, n)
            used[torch.as_tensor(table[b, t // page]).long(), torch.as_tensor(t % page).long()] = True
        bad = torch.where(torch.rand(pages, page) < 0.5, math.nan, math.inf)
        for x in (kp, vp):
            x[~used.cuda()] = bad[~used].to(dtype).cuda()[:, None, None]
    scaling = 1.0 / math.sqrt(D)
    status = ops.new_status("cuda")
    args = (q, kp, vp, dev(table), dev(lengths), scaling)
    out, lse = ops.paged_attn(*args, window=window, return_lse=True, workspace=workspace, status=status)
    assert status.item() == 0
    want, want_lse, bound, lse_bound = plain.attend(*args[:4], lengths, scaling, window)
    near(out, want, bound)
    none = torch.isinf(want_lse)
    assert torch.equal(torch.isinf(lse.cpu()), none) and bool((lse.cpu()[none] < 0).all())
    near(lse.cpu()[~none], want_lse[~none], lse_bound[~none])
    return args, out, lse


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D", [64, 96, 128, 256])
@pytest.mark.parametrize("Hq,Hkv", [(2, 2), (8, 2), (7, 1), (9, 1), (16, 1), (34, 2), (40, 1)])
def test_attend_heads(ops, dtype, D, Hq, Hkv):
    attend(ops, LENGTHS["edges"], Hq, Hkv, D, dtype, page=16)


@pytest.mark.parametrize("lengths", sorted(LENGTHS))
@pytest.mark.parametrize("page", [1, 5, 16, 24, 64, 256])
@pytest.mark.parametrize("Hq,Hkv", [(3, 3), (8, 2)])
def test_attend_pages(ops, lengths, page, Hq, Hkv):
    attend(ops, LENGTHS[lengths], Hq, Hkv, 128, torch.float16, page=page, seed=page)


@pytest.mark.parametrize("window", [1, 2, 15, 16, 17, 64, 100, 4000])
@pytest.mark.parametrize("lengths", ["edges", "long"])
def test_attend_window(ops, window, lengths):
    attend(ops, LENGTHS[lengths], 8, 2, 64, torch.bfloat16, page=16, window=window)


@pytest.mark.parametrize("order", ["head", "padded"])
@pytest.mark.parametrize("D", [96, 128])
def test_attend_strides(ops, order, D):
    attend(ops, LENGTHS["edges"], 6, 3, D, torch.float16, page=24, order=order)


@pytest.mark.parametrize("D", [64, 96, 128, 256])
@pytest.mark.parametrize("heads", [(4, 2), (20, 2)])
def test_attend_pools_of_different_strides(ops, D, heads):
    """Keys with each head's rows together, values token by token with room between the rows."""
    gen = torch.Generator(device="cuda").manual_seed(D)
    lengths = LENGTHS["edges"]
    table, _, _ = plain.tables(np.random.RandomState(D), lengths, 16, 200)
    kp, vp = plain.pool(gen, 200, 16, 2, D, torch.bfloat16, "cuda", "head"), plain.pool(gen, 200, 16, 2, D, torch.bfloat16, "cuda", "padded")
    q = torch.randn(len(lengths), heads[0], D, generator=gen, device="cuda").bfloat16()
    args = (q, kp, vp, dev(table), dev(lengths), 0.1)
    want, _, bound, _ = plain.attend(*args[:4], lengths, 0.1)
    near(ops.paged_attn(*args), want, bound)
    want, _, bound, _ = plain.attend(q, vp, kp, *args[3:4], lengths, 0.1)
    near(ops.paged_attn(q, vp, kp, *args[3:]), want, bound)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_attend_sharp(ops, dtype):
    """Scores in the hundreds: weights from 1 to nothing, the maximum anywhere; with half of one sign only."""
    attend(ops, LENGTHS["edges"] + [3000], 8, 2, 128, dtype, sharp=100.0)


@pytest.mark.parametrize("scaling", [-0.3, 0.0, 1e-30, 4.0])
def test_attend_scalings(ops, scaling):
    """A negative scaling, none at all (the mean of the values), a large one."""
    gen = torch.Generator(device="cuda").manual_seed(2)
    lengths = [0, 1, 5, 77, 300]
    table, _, _ = plain.tables(np.random.RandomState(2), lengths, 16, 40)
    kp, vp = (plain.pool(gen, 40, 16, 2, 64, torch.float16, "cuda") for _ in range(2))
    q = torch.randn(5, 6, 64, generator=gen, device="cuda").half()
    args = (q, kp, vp, dev(table), dev(lengths), scaling)
    out, lse = ops.paged_attn(*args, return_lse=True)
    want, want_lse, bound, lse_bound = plain.attend(*args[:4], lengths, scaling)
    near(out, want, bound)
    near(lse[1:], want_lse[1:], lse_bound[1:])


def test_attend_small_weights_count(ops):
    """One token of weight 1 before 40 000 of weight 2^-26: together they are 0.0006 of the result, and none may be lost to a 16-bit weight."""
    n, D, page = 40001, 64, 64
    pages = -(-n // page)
    kp = torch.zeros(pages, page, 1, D, device="cuda", dtype=torch.float16)
    vp = torch.zeros_like(kp)
    kp.view(-1, D)[0, 0] = 1.0
    vp.view(-1, D)[1:n, 0] = 1000.0
    q = torch.zeros(1, 1, D, device="cuda", dtype=torch.float16)
    q[0, 0, 0] = 1.0
    scaling = 26 * math.log(2)
    table, lengths = dev(np.arange(pages)[None]), dev([n])
    out, lse = ops.paged_attn(q, kp, vp, table, lengths, scaling, return_lse=True)
    want, want_lse, bound, lse_bound = plain.attend(q, kp, vp, table, [n], scaling)
    assert 0.5 < want[0, 0, 0] < 0.7
    near(out, want, bound)
    near(lse, want_lse, lse_bound)
    assert abs(out[0, 0, 0].item() / want[0, 0, 0].item() - 1) < 2.0 ** -9


def test_attend_leaves_out_bad_pages(ops):
    """Pages outside the pool, a length below 0, one beyond the table row: reported, and their tokens left out."""
    from kvcomp_b200 import _lib
    lengths = [100, 64, -3, 1000, 70, 20]
    gen = torch.Generator(device="cuda").manual_seed(1)
    table = np.arange(6 * 8, dtype=np.int32).reshape(6, 8)
    table[0, 2], table[0, 6], table[1] = -1, 1 << 30, 48
    table[4, 4] = 2 ** 31 - 1
    kp, vp = (plain.pool(gen, 48, 16, 2, 128, torch.float16, "cuda") for _ in range(2))
    q = torch.randn(6, 4, 128, generator=gen, device="cuda").half()
    status = ops.new_status("cuda")
    args = (q, kp, vp, dev(table), dev(lengths), 0.1)
    out, lse = ops.paged_attn(*args, return_lse=True, status=status)
    assert status.item() == _lib.FLAG_BAD_PAGE | _lib.FLAG_BAD_LENGTH
    want, want_lse, bound, _ = plain.attend(*args[:4], lengths, 0.1)
    near(out, want, bound)
    assert lse[1].tolist() == [-math.inf] * 4 and lse[2].tolist() == [-math.inf] * 4
    out2 = ops.paged_attn(*args)                       # without a status word: the same, unreported
    assert torch.equal(out, out2)


def test_attend_again_and_workspaces(ops):
    """The same bits again and again, from a workspace that other shapes have used, on another stream, without a workspace."""
    ws = ops.paged_attn_workspace(300, 40, 10, 256, "cuda")
    args, out, lse = attend(ops, LENGTHS["edges"] + [9000], 8, 2, 128, torch.float16, workspace=ws)
    for lengths, heads, D in (("many", (10, 10), 64), ("long", (16, 1), 256), ("none", (4, 4), 96)):
        attend(ops, LENGTHS[lengths], *heads, D, torch.bfloat16, workspace=ws)
    for _ in range(20):
        again, lse2 = ops.paged_attn(*args, return_lse=True, workspace=ws)
        assert torch.equal(again, out) and torch.equal(lse, lse2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = ops.paged_attn(*args, workspace=ws)
    side.synchronize()
    assert torch.equal(again, out)
    assert torch.equal(ops.paged_attn(*args), out)
    mine = torch.full_like(out, 7.0)
    assert ops.paged_attn(*args, out=mine, workspace=ws) is mine and torch.equal(mine, out)


@pytest.mark.parametrize("D,tokens", [(64, 60000), (96, 46000), (128, 46000)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_attend_long_shares(ops, D, tokens, dtype):
    """So many tokens that CTAs draw the last of them (96 tiles of 64 for each CTA, up to four of which are on an SM).  The requests share their pages, one reads
    another's backwards; some are short or empty.  The same bits again."""
    Hq, Hkv, page = 16, 8, 64
    lengths = [tokens, tokens - 1, 0, tokens + 777, tokens, 64, tokens, tokens - 4000, tokens, tokens + 1, 1]
    assert sum(lengths) * Hkv > 96 * 64 * (4 if D == 64 else 3) * torch.cuda.get_device_properties(0).multi_processor_count
    gen = torch.Generator(device="cuda").manual_seed(D)
    pages = -(-max(lengths) // page)
    rows = np.random.RandomState(D).permutation(pages).astype(np.int32)
    table = np.stack([rows if b % 3 else rows[::-1] for b in range(len(lengths))])
    kp, vp = (plain.pool(gen, pages, page, Hkv, D, dtype, "cuda") for _ in range(2))
    q = torch.randn(len(lengths), Hq, D, generator=gen, device="cuda").to(dtype)
    ws = ops.paged_attn_workspace(len(lengths), Hq, Hkv, D, "cuda")
    args = (q, kp, vp, dev(table), dev(lengths), 0.3)
    status = ops.new_status("cuda")
    out, lse = ops.paged_attn(*args, return_lse=True, workspace=ws, status=status)
    assert status.item() == 0
    for _ in range(3):
        again, lse2 = ops.paged_attn(*args, return_lse=True, workspace=ws)
        assert torch.equal(out, again) and torch.equal(lse, lse2)
    some = [0, 2, 3, 5, 9, 10]
    want, want_lse, bound, lse_bound = plain.attend(q[some], kp, vp, dev(table[some]), [lengths[b] for b in some], 0.3)
    near(out[some], want, bound)
    there = [i for i, b in enumerate(some) if lengths[b]]
    near(lse[some][there], want_lse[there], lse_bound[there])


def test_attend_on_two_streams(ops):
    """Two calls at once with workspaces of their own; out may be q."""
    args, out, _ = attend(ops, [5000, 70, 9000, 0], 8, 2, 128, torch.float16)
    args2, out2, _ = attend(ops, [3000] * 6, 16, 1, 64, torch.bfloat16, seed=3)
    streams, ws = [torch.cuda.Stream() for _ in range(2)], [ops.paged_attn_workspace(4, 8, 2, 128, "cuda"), ops.paged_attn_workspace(6, 16, 1, 64, "cuda")]
    got = [[], []]
    torch.cuda.synchronize()
    for _ in range(10):
        for i, a in enumerate((args, args2)):
            with torch.cuda.stream(streams[i]):
                got[i].append(ops.paged_attn(*a, workspace=ws[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(x, out) for x in got[0]) and all(torch.equal(x, out2) for x in got[1])
    q = args[0].clone()
    ops.paged_attn(q, *args[1:], out=q, workspace=ws[0])
    assert torch.equal(q, out)


def test_attend_long_offsets(ops):
    """Pages whose offsets pass 32 bits: a pool of 5 GB of keys, the request's pages at both ends."""
    page, D = 64, 128
    pages = 5 * (1 << 30) // (page * D * 2) + 1
    kp = torch.empty(pages, page, 1, D, dtype=torch.float16, device="cuda")
    rows = [0, pages - 1, pages - 2, 1, pages // 2 + 7]
    kp[rows] = torch.randn(5, page, 1, D, device="cuda").half()
    q = torch.randn(1, 4, D, device="cuda").half()
    table, n = dev([rows]), 5 * page - 3
    out = ops.paged_attn(q, kp, kp, table, dev([n]), 0.2)
    small = kp[rows]
    want, _, bound, _ = plain.attend(q, small, small, dev([[0, 1, 2, 3, 4]]), [n], 0.2)
    near(out, want, bound)
    slots = dev([(pages - 1) * page + 3, 5])
    k = torch.randn(2, 1, D, device="cuda").half()
    ops.rotary_paged_store(None, k, k, None, slots, None, kp, kp)
    assert torch.equal(kp[pages - 1, 3], k[0]) and torch.equal(kp[0, 5], k[1])


def test_refusals(ops):
    """Arguments that do not fit are errors before anything is launched."""
    from kvcomp_b200._lib import KvcError
    q = torch.zeros(2, 4, 128, device="cuda", dtype=torch.float16)
    kp = torch.zeros(3, 16, 2, 128, device="cuda", dtype=torch.float16)
    table, lengths = dev([[0, 1], [2, 0]]), dev([20, 3])
    ws = ops.paged_attn_workspace(2, 4, 2, 128, "cuda")
    ops.paged_attn(q, kp, kp, table, lengths, 0.1, workspace=ws)
    odd = torch.zeros(3, 16, 2, 136, device="cuda", dtype=torch.float16)[..., 4:132]
    for bad in (dict(q=q.cpu()), dict(q=q.float()), dict(q=q[0]), dict(kp=kp.bfloat16()), dict(kp=odd), dict(table=table.long()), dict(table=table[:1]),
                dict(lengths=lengths.long()), dict(lengths=lengths[:1]), dict(ws=ws[:16]), dict(window=-1), dict(kp=kp[..., :64]), dict(q=q[:, :3]),
                dict(kp=kp.cpu()), dict(kp=kp.permute(0, 1, 3, 2)), dict(q=torch.zeros(2, 4, 112, device="cuda", dtype=torch.float16), kp=kp[..., :112]),
                dict(out=torch.zeros(2, 4, 128, device="cuda")), dict(status=torch.zeros(1, device="cuda"))):
        a = dict(q=q, kp=kp, table=table, lengths=lengths, ws=ws, window=0, out=None, status=None)
        a.update(bad)
        with pytest.raises(KvcError):
            ops.paged_attn(a["q"], a["kp"], a["kp"], a["table"], a["lengths"], 0.1, window=a["window"], out=a["out"], workspace=a["ws"], status=a["status"])
    k = torch.zeros(2, 2, 128, device="cuda", dtype=torch.float16)
    f, pos, slots = freqs(64).cuda(), dev([0, 1]), dev([1, 2])
    for bad in (dict(k=k.float()), dict(v=k[:, :1]), dict(pos=pos[:1]), dict(slots=slots.long()), dict(f=freqs(65).cuda()), dict(f=freqs(8).float().cuda()),
                dict(f=freqs(8)), dict(layout="both"), dict(kp=kp[:, :, :1]), dict(q=k.bfloat16()), dict(pos=None)):
        a = dict(q=q, k=k, v=k, pos=pos, slots=slots, f=f, kp=kp, layout="half")
        a.update(bad)
        with pytest.raises(KvcError):
            ops.rotary_paged_store(a["q"], a["k"], a["v"], a["pos"], a["slots"], a["f"], a["kp"], a["kp"], layout=a["layout"])
    with pytest.raises(KvcError):
        ops.rotary(k.cpu(), pos, f)
    with pytest.raises(KvcError):
        ops.rotary(k, pos, f, out=k[:1])
    free, head = dev([0, 1, 2]), dev([3])
    for bad in (dict(page=0), dict(tokens=-1), dict(free=free.long()), dict(head=head.cpu()), dict(new=lengths[:1]), dict(table=table.T)):
        a = dict(lengths=lengths, new=lengths, table=table, free=free, head=head, page=16, tokens=64)
        a.update(bad)
        with pytest.raises((KvcError, RuntimeError)):
            ops.page_plan(a["lengths"], a["new"], a["table"], a["free"], a["head"], a["page"], a["tokens"])
    with pytest.raises(KvcError):
        ops.page_release(lengths, lengths, table, free, head, 16)
