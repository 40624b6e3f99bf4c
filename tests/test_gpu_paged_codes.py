"""Paged caches in 8 bits: rows coded as they are written, read back, and attended."""
import math

import numpy as np
import pytest
import torch

import codes_plain
import paged_plain as plain

pytestmark = pytest.mark.gpu

DTYPES = [torch.float16, torch.bfloat16]
CODES = ["int8", "e4m3"]


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    from kvcomp_b200 import ops
    return ops


def dev(a, dtype=torch.int32):
    return torch.as_tensor(np.asarray(a), dtype=dtype).cuda()


def freqs(n):
    return torch.tensor(10000.0 ** (-np.arange(n) / max(n, 1)), dtype=torch.float64).cuda()


def pools(pages, page, heads, dim, codes, seed=0):
    """Pools full of something: codes and scales that nothing may change but what is asked for."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    made = [torch.randint(-100, 100, (pages, page, heads, dim), generator=gen, device="cuda", dtype=torch.int8).view(codes_plain.TYPES[codes]) for _ in range(2)]
    return made + [torch.rand(pages, heads, page, generator=gen, device="cuda") for _ in range(2)]


def same(a, b):
    """The same bits, where they are numbers (e4m3 has two codes that are none)."""
    return torch.allclose(a, b, rtol=0, atol=0, equal_nan=True)


def store(ops, dtype, codes, N, Hq, Hkv, D, r, page, layout, views="slices", inverse_scale=1.0):
    gen = torch.Generator(device="cuda").manual_seed(N + D + r)
    heads = Hq + 2 * Hkv
    wide = torch.randn(N, heads, D + (8 if views == "odd" else 0), generator=gen, device="cuda") * torch.exp(torch.randn(N, heads, 1, generator=gen, device="cuda")) * inverse_scale
    qkv = wide.to(dtype)[:, :, 4:4 + D] if views == "odd" else wide.to(dtype)       # (odd: rows that start on 8 bytes)
    q, k, v = qkv[:, :Hq], qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:]
    pages = -(-N // page) + 2
    rng = np.random.RandomState(N + page)
    slots = rng.permutation(pages * page)[:N].astype(np.int32)
    if N > 3:
        slots[2] = -1                                               # a refused token
    positions = rng.randint(0, 50000, N)
    f = freqs(r // 2) if r else None
    kp, vp, ks, vs = pools(pages, page, Hkv, D, codes)
    before = [t.clone() for t in (kp, vp, ks, vs)]
    status = ops.new_status(torch.device("cuda"))
    got = ops.rotary_paged_store(q if Hq else None, k, v, dev(positions), dev(slots), f, kp, vp, layout=layout, status=status, kscales=ks, vscales=vs)
    return q, k, v, positions, slots, f, got, (kp, vp, ks, vs), before, status


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("N,Hq,Hkv,D,r,page,layout,views", [
    (1, 2, 2, 128, 128, 16, "half", "slices"), (7, 32, 32, 128, 128, 64, "interleaved", "slices"), (33, 8, 2, 96, 96, 5, "half", "slices"), (65, 5, 5, 64, 32, 16, "interleaved", "slices"),
    (19, 16, 1, 256, 64, 24, "half", "slices"), (40, 6, 2, 96, 24, 16, "half", "slices"), (40, 6, 2, 128, 12, 1, "interleaved", "slices"), (21, 0, 3, 80, 80, 16, "half", "slices"),
    (21, 4, 4, 128, 0, 16, "half", "slices"), (33, 4, 2, 128, 128, 16, "half", "odd"), (17, 4, 2, 512, 512, 16, "half", "slices"), (9, 2, 1, 1024, 64, 16, "half", "slices"),
    (1500, 40, 10, 128, 96, 128, "half", "slices"), (700, 8, 8, 96, 96, 16, "interleaved", "slices")])
def test_store(ops, dtype, codes, N, Hq, Hkv, D, r, page, layout, views):
    """Values' codes and scales are the definition's; keys' too, up to what a rotation in 32 bits is off: a key is within half a step of its code, and that."""
    q, k, v, positions, slots, f, got, (kp, vp, ks, vs), before, status = store(ops, dtype, codes, N, Hq, Hkv, D, r, page, layout, views)
    assert int(status.item()) == 0
    f = f.cpu() if f is not None else torch.zeros(0, dtype=torch.float64)
    at = torch.as_tensor(positions)
    if Hq:
        want = plain.rotate(q.cpu(), at, f, layout)
        assert bool(((got.cpu().double() - want).abs() <= plain.rotate_bound(q.cpu(), want, f, layout, 1.0)).all())
    on = torch.as_tensor(slots) >= 0
    where = dev(slots)[on.cuda()]
    x = v.cpu().double()[on]
    s = codes_plain.scale(x, codes)
    assert torch.equal(codes_plain.at_slots(vs, where).cpu().double(), s[..., 0])
    assert torch.equal(codes_plain.bits(codes_plain.at_slots(vp, where)).cpu(), codes_plain.bits(codes_plain.code(x, s, codes)))
    x = plain.rotate(k.cpu(), at, f, layout)[on]
    eps = torch.finfo(dtype).eps / 2
    off = plain.rotate_bound(k.cpu()[on], x, f, layout, 1.0) - eps * x.abs()        # (without the rounding to 16 bits, which there is none of)
    got_s = codes_plain.at_slots(ks, where).cpu().double()[..., None]
    assert bool(((got_s - codes_plain.scale(x, codes)).abs() <= off.amax(-1, keepdim=True) / 127 + got_s * 2.0 ** -23).all())
    held = codes_plain.at_slots(kp, where).cpu().float().double() * got_s
    assert bool(((held - x).abs() <= codes_plain.half_step(x, got_s, codes) * (1 + 2.0 ** -20) + off).all())
    # everything else is as it was
    mask = torch.ones(kp.shape[0] * page, dtype=torch.bool, device="cuda")
    mask[where.long()] = False
    rest = mask.nonzero()[:, 0]
    for now, then in zip((kp, vp, ks, vs), before):
        a, b = codes_plain.at_slots(now, rest), codes_plain.at_slots(then, rest)
        assert torch.equal(a if a.dtype == torch.float32 else codes_plain.bits(a), b if b.dtype == torch.float32 else codes_plain.bits(b))


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("D", [64, 96, 128, 256])
def test_borders_of_codes(ops, codes, D):
    """Values on the border of two codes and next to it, rows of zeros, of one value, of the smallest and the largest, infinite ones and no numbers."""
    rows = []
    base = torch.arange(D, dtype=torch.float64) - D // 2
    for top, step in ((127.0, 0.5), (254.0, 1.0), (381.0, 1.5), (63.5, 0.25), (448.0, 3.5), (449.0, 1.0), (224.0, 0.875), (447.9, 1.75)):
        x = base * step
        x[0] = top
        rows.append(x.clamp(-top, top))
    for x in (0.0, 1.0, -3.0, 6e-8, 65504.0, 2.0 ** -14, math.inf, -math.inf, math.nan):
        row = torch.zeros(D, dtype=torch.float64)
        row[D // 3] = x
        rows.append(row)
    for dtype in DTYPES:
        x = torch.stack(rows + ([torch.full((D,), 1e-36, dtype=torch.float64), torch.full((D,), 3e38, dtype=torch.float64)] if dtype == torch.bfloat16 else [])).to(dtype)
        n = len(x)
        kp, vp, ks, vs = pools(4, 16, 1, D, codes)
        slots = dev(np.arange(n)[::-1].copy())
        ops.rotary_paged_store(None, x.cuda()[:, None], x.cuda()[:, None], None, slots, None, kp, vp, kscales=ks, vscales=vs)
        s = codes_plain.scale(x.double(), codes)
        for pool, scales in ((kp, ks), (vp, vs)):
            got = codes_plain.at_slots(scales, slots).cpu()[:, 0, None].double()
            assert torch.equal(torch.isnan(got), torch.isnan(s)) and torch.equal(got.nan_to_num(), s.nan_to_num())
            fine = ~torch.isnan(s[:, 0])
            assert torch.equal(codes_plain.bits(codes_plain.at_slots(pool, slots))[:, 0].cpu()[fine], codes_plain.bits(codes_plain.code(x.double()[fine], s[fine], codes)))
        k, v = ops.paged_rows(kp, vp, slots, ks, vs, dtype=dtype)
        assert torch.equal(torch.isnan(k[:, 0]).all(-1).cpu(), ~fine) and torch.equal(torch.isnan(v[:, 0]).any(-1).cpu(), ~fine)


def test_slots_outside_the_pool(ops):
    x = torch.randn(3, 2, 128, device="cuda").half()
    kp, vp, ks, vs = pools(2, 16, 2, 128, "int8")
    before = [t.clone() for t in (kp, vp, ks, vs)]
    status = ops.new_status(torch.device("cuda"))
    ops.rotary_paged_store(None, x, x, None, dev([32, -1, 1 << 30]), None, kp, vp, kscales=ks, vscales=vs, status=status)
    from kvcomp_b200 import _lib
    assert int(status.item()) == _lib.FLAG_BAD_PAGE and all(torch.equal(a, b) for a, b in zip(before, (kp, vp, ks, vs)))
    k, v = ops.paged_rows(kp, vp, dev([32, -1, 5]), ks, vs, dtype=torch.float16, status=status)
    assert int(status.item()) == _lib.FLAG_BAD_PAGE and not bool(k[:2].any()) and not bool(v[:2].any()) and bool(k[2].any())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("codes", CODES + [None])
@pytest.mark.parametrize("N,H,D,page", [(1, 1, 64, 16), (5, 32, 128, 1), (333, 3, 96, 24), (70, 8, 256, 64), (4000, 10, 128, 128), (9, 7, 16, 8), (20, 2, 1040, 16)])
def test_rows(ops, dtype, codes, N, H, D, page):
    """Rows are codes times scales in 32 bits, rounded once; rows of 16 bits are copied.  Into tensors of any strides, too."""
    pages = -(-N // page) + 2
    if codes:
        kp, vp, ks, vs = pools(pages, page, H, D, codes, seed=N)
    else:
        kp, vp = (torch.randn(pages, page, H, D, device="cuda").to(dtype) for _ in range(2))
        ks = vs = None
    slots = dev(np.random.RandomState(N).randint(-1, pages * page, N))
    out = torch.full((2, N, H + 1, D + 8), 7.0, dtype=dtype, device="cuda")
    got = ops.paged_rows(kp, vp, slots, ks, vs, dtype=dtype)
    into = ops.paged_rows(kp, vp, slots, ks, vs, dtype=dtype, out=(out[0, :, :H, :D], out[1, :, :H, :D]))
    for pool, scales, k, k2 in zip((kp, vp), (ks, vs), got, into):
        want = codes_plain.at_slots(pool, slots.clamp(min=0))
        if codes:
            want = (want.float() * codes_plain.at_slots(scales, slots.clamp(min=0))[..., None]).to(dtype)
        want[slots < 0] = 0
        assert same(k, want) and same(k2, want)
    assert bool((out[:, :, H] == 7).all()) and bool((out[..., D:] == 7).all())


@pytest.mark.parametrize("page", [1, 7, 16, 64])
@pytest.mark.parametrize("requests,longest,spare", [(1, 1, 0), (1, 5000, 3), (3, 0, 2), (33, 40, 0), (200, 10, 1), (1500, 9, 0), (70, 300, 5)])
def test_page_slots(ops, page, requests, longest, spare):
    rng = np.random.RandomState(requests + longest + page)
    lengths = rng.randint(0, longest + 1, requests)
    table, _, used = plain.tables(rng, lengths, page, int((-(-lengths // page)).sum()) + 1, extra=2)
    tokens = int(lengths.sum()) + spare
    status = ops.new_status(torch.device("cuda"))
    slots, starts = ops.page_slots(dev(table), dev(lengths), page, tokens, status=status)
    want = [int(table[b, t // page]) * page + t % page for b, n in enumerate(lengths) for t in range(n)] + [-1] * spare
    assert slots.tolist() == want and starts.tolist() == [0] + np.cumsum(lengths).tolist() and int(status.item()) == 0
    first, positions = dev(rng.randint(0, 1000, requests)), torch.arange(tokens, dtype=torch.int32, device="cuda")
    ops.page_shift(starts, first, positions)
    assert positions.tolist() == (np.arange(tokens) + np.concatenate([np.repeat(first.cpu().numpy(), lengths), np.zeros(spare, dtype=np.int64)])).tolist()


def test_page_slots_of_bad_requests(ops):
    from kvcomp_b200 import _lib
    status = ops.new_status(torch.device("cuda"))
    slots, starts = ops.page_slots(dev([[3, -1], [4, 5]]), dev([3, 4]), 2, 7, status=status)
    assert int(status.item()) == _lib.FLAG_BAD_PAGE and slots.tolist() == [6, 7, -1, 8, 9, 10, 11]
    status.zero_()
    slots, starts = ops.page_slots(dev([[3, 6], [4, 5], [1, 2]]), dev([-2, 99, 3]), 2, 6, status=status)           # no length, one that the table does not hold, one too many rows
    assert int(status.item()) == _lib.FLAG_BAD_LENGTH and slots.tolist() == [8, 9, 10, 11, 2, 3] and starts.tolist() == [0, 0, 4, 6]


# ---- attention -------------------------------------------------------------------------------------

LENGTHS = {"edges": [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 0], "long": [5000, 3, 0, 1301], "one": [777], "many": [64] * 70 + [0, 1] * 40}


def want(q, kp, vp, ks, vs, table, lengths, scaling, window=0):
    """(out, lse, bound of out, bound of lse).  Beside the plain form's bound (its pieces of weights are coarser than these): the result's rounding, and what is lost of weights far below the
    largest: 2^-25 of 2^14 for each token, times the largest value."""
    k, v = codes_plain.values(kp, ks), codes_plain.values(vp, vs)
    k, v = k.nan_to_num(nan=0.0), v.nan_to_num(nan=0.0)             # (only places that are not read hold any)
    out, lse, off, lse_off = plain.attend(q, k, v, table, lengths, scaling, window)
    off = off + len(k) * k.shape[1] * 2.0 ** -39 * v.abs().max().item()
    tiny = 2.0 ** -25 if q.dtype == torch.float16 else 0.0
    return out, lse, off + torch.finfo(q.dtype).eps / 2 * (out.abs() + off) + tiny, lse_off


def attend(ops, lengths, Hq, Hkv, D, dtype, codes, page=16, window=0, seed=0, sharp=1.0, scaling=None, order="token", starts=None, spread=0.0):
    rng = np.random.RandomState(seed + len(lengths) + page)
    gen = torch.Generator(device="cuda").manual_seed(seed + D)
    pages = sum(-(-n // page) for n in lengths) + 3
    table, order_of, used = plain.tables(rng, lengths, page, pages, extra=1)
    x = torch.randn(2, pages, page, Hkv, D, generator=gen, device="cuda") * torch.exp(spread * torch.randn(2, pages, page, Hkv, 1, generator=gen, device="cuda"))
    (kp, ks), (vp, vs) = (codes_plain.coded(t, codes) for t in x)
    # what no request holds is never read: scales that are no numbers, and rows behind lengths too
    free = torch.ones(pages, page, dtype=torch.bool)
    for b, n in enumerate(lengths):
        for i in range(-(-n // page)):
            free[table[b, i], :max(0, min(page, n - i * page))] = False
    for s in (ks, vs):
        s.transpose(1, 2)[free.cuda()] = math.nan
    if order == "head":                                             # each head's rows of a page lie together
        kp, vp = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (kp, vp))
    elif order == "padded":
        wide = [torch.zeros(pages, page, Hkv + 1, D + 16, dtype=torch.int8, device="cuda") for _ in range(2)]
        for w, t in zip(wide, (kp, vp)):
            w[:, :, :Hkv, :D] = codes_plain.bits(t)
        kp, vp = (w.view(t.dtype)[:, :, :Hkv, :D] for w, t in zip(wide, (kp, vp)))
        ks, vs = (torch.nn.functional.pad(s, (0, 3, 0, 2))[:, :Hkv, :page] for s in (ks, vs))
    rows = len(lengths) if starts is None else int(starts[-1])
    q = (torch.randn(max(rows, 1), Hq, D, generator=gen, device="cuda") * sharp).to(dtype)[:rows]
    scaling = 1 / math.sqrt(D) if scaling is None else scaling
    status = ops.new_status(torch.device("cuda"))
    out, lse = ops.paged_attn(q, kp, vp, dev(table), dev(lengths), scaling, window=window, return_lse=True, status=status, starts=None if starts is None else dev(starts), kscales=ks, vscales=vs)
    assert int(status.item()) == 0
    of = range(len(lengths)) if starts is None else [b for b in range(len(lengths)) if starts[b + 1] > starts[b]]
    w, w_lse, bound, lse_bound = want(q, kp, vp, ks, vs, torch.as_tensor(table[list(of)]), [lengths[b] for b in of], scaling, window)
    near = (out.cpu().double() - w).abs() <= bound
    assert bool(near.all()), (~near).nonzero()[:5]
    empty = torch.isneginf(w_lse)
    assert torch.equal(torch.isneginf(lse.cpu()), empty) and bool(((lse.cpu().double() - w_lse).abs() <= lse_bound)[~empty].all())
    assert not bool(out.cpu()[empty].any())
    return out


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 96, 128, 256])
@pytest.mark.parametrize("Hq,Hkv", [(2, 2), (8, 2), (7, 1), (9, 1), (16, 1), (34, 2), (3, 3)])
def test_attend_heads(ops, dtype, codes, D, Hq, Hkv):
    attend(ops, [40, 0, 333, 1], Hq, Hkv, D, dtype, codes)


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("lengths", sorted(LENGTHS))
@pytest.mark.parametrize("page", [1, 5, 16, 24, 64, 256])
def test_attend_pages(ops, lengths, page, codes):
    attend(ops, LENGTHS[lengths], 8, 2, 128, torch.float16, codes, page=page)


@pytest.mark.parametrize("window", [1, 15, 16, 17, 33, 100, 4000])
@pytest.mark.parametrize("D", [64, 128])
def test_attend_window(ops, window, D):
    attend(ops, LENGTHS["edges"], 4, 2, D, torch.bfloat16, "int8", page=5, window=window)
    attend(ops, LENGTHS["long"], 4, 2, D, torch.float16, "e4m3", window=window)


@pytest.mark.parametrize("order", ["head", "padded"])
@pytest.mark.parametrize("D", [64, 96, 128, 256])
@pytest.mark.parametrize("codes", CODES)
def test_attend_strides(ops, order, D, codes):
    attend(ops, [100, 31, 0, 600], 8, 4, D, torch.float16, codes, order=order, page=24)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("codes", CODES)
def test_attend_scales_of_every_size(ops, dtype, codes):
    """Rows whose sizes lie orders of magnitude apart, and weights that are all but one nothing."""
    attend(ops, [300, 1000, 65], 4, 2, 128, dtype, codes, spread=2.0)
    attend(ops, [300, 1000, 65], 4, 2, 128, dtype, codes, sharp=30.0)
    attend(ops, [300, 1000, 65], 4, 2, 64, dtype, codes, spread=1.0, scaling=-0.3)
    attend(ops, [300, 1000, 65], 4, 2, 96, dtype, codes, scaling=0.0)


@pytest.mark.parametrize("codes", CODES)
def test_attend_rows(ops, codes):
    attend(ops, [40, 0, 333, 1, 77], 8, 2, 128, torch.float16, codes, starts=[0, 1, 1, 2, 2, 3])


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_first_token_without_a_value(ops, dtype):
    """The first token takes nearly all the weight and has a value of all but nothing, as models' first tokens do: what the others bring is kept."""
    D, n = 128, 2000
    gen = torch.Generator(device="cuda").manual_seed(4)
    k, v = (torch.randn(1, n, 1, D, generator=gen, device="cuda") for _ in range(2))
    q = torch.randn(1, 1, D, generator=gen, device="cuda")
    k[0, 0, 0] = q[0, 0] * 2
    v[0, 0] *= 1e-6
    (kp, ks), (vp, vs) = codes_plain.coded(k, "int8"), codes_plain.coded(v, "int8")
    table, q = dev([[0]]), q.to(dtype)
    out, lse = ops.paged_attn(q, kp, vp, table, dev([n]), 0.1, return_lse=True, kscales=ks, vscales=vs)
    w, _, bound, _ = want(q, kp, vp, ks, vs, table, [n], 0.1)
    assert bool(((out.cpu().double() - w).abs() <= bound).all()) and float(w.abs().max()) < 0.05


@pytest.mark.parametrize("codes", CODES)
def test_rows_without_a_number_that_count(ops, codes):
    """A key or a value whose scale is no number makes its KV head's results none, and no other's."""
    (kp, ks), (vp, vs) = (codes_plain.coded(torch.randn(4, 16, 2, 128, device="cuda"), codes) for _ in range(2))
    q, table, lengths = torch.randn(2, 4, 128, device="cuda").half(), dev([[0, 1], [2, 3]]), dev([30, 20])
    for s in (ks, vs):
        was = s[1, 1, 3].clone()
        s[1, 1, 3] = math.nan                                       # token 19 of request 0, head 1
        out = ops.paged_attn(q, kp, vp, table, lengths, 0.1, kscales=ks, vscales=vs)
        assert bool(torch.isnan(out[0, 2:]).all()) and not bool(torch.isnan(out[0, :2]).any()) and not bool(torch.isnan(out[1]).any())
        s[1, 1, 3] = was


def test_attend_leaves_out_bad_pages(ops):
    from kvcomp_b200 import _lib
    (kp, ks), (vp, vs) = (codes_plain.coded(torch.randn(4, 16, 2, 128, device="cuda"), "int8") for _ in range(2))
    q = torch.randn(2, 4, 128, device="cuda").half()
    table, status = torch.tensor([[0, 9, 1], [2, -1, 3]]), ops.new_status(torch.device("cuda"))
    out = ops.paged_attn(q, kp, vp, dev(table), dev([48, 40]), 0.1, kscales=ks, vscales=vs, status=status)
    w, _, bound, _ = want(q, kp, vp, ks, vs, table, [48, 40], 0.1)
    assert int(status.item()) == _lib.FLAG_BAD_PAGE and bool(((out.cpu().double() - w).abs() <= bound).all())


@pytest.mark.parametrize("D,dtype,codes", [(64, torch.float16, "e4m3"), (96, torch.bfloat16, "int8"), (128, torch.float16, "int8"), (128, torch.bfloat16, "e4m3")])
def test_attend_long_shares(ops, D, dtype, codes):
    """Shares long enough to be drawn in part, and columns that many CTAs join; twice the same bits."""
    gen = torch.Generator(device="cuda").manual_seed(D)
    lengths, page, Hkv = [60000, 30011, 1, 0, 45000], 64, 8
    pages = sum(-(-n // page) for n in lengths)
    rng = np.random.RandomState(D)
    table, _, _ = plain.tables(rng, lengths, page, pages)
    (kp, ks), (vp, vs) = (codes_plain.coded(torch.randn(pages, page, Hkv, D, generator=gen, device="cuda"), codes) for _ in range(2))
    q = torch.randn(len(lengths), 2 * Hkv, D, generator=gen, device="cuda").to(dtype)
    workspace = ops.paged_attn_workspace(len(lengths), 2 * Hkv, Hkv, D, "cuda")
    runs = [ops.paged_attn(q, kp, vp, dev(table), dev(lengths), 0.1, kscales=ks, vscales=vs, workspace=workspace) for _ in range(3)]
    assert torch.equal(runs[0], runs[1]) and torch.equal(runs[0], runs[2])
    one = slice(4, 5)                                               # one KV head's queries in 64 bits
    w, _, bound, _ = want(q[:, one], kp[:, :, 2:3], vp[:, :, 2:3], ks[:, 2:3], vs[:, 2:3], torch.as_tensor(table), lengths, 0.1)
    assert bool(((runs[0][:, one].cpu().double() - w).abs() <= bound).all())


def test_store_rows_and_attention_in_a_graph(ops):
    """A step's calls captured and replayed with other inputs give what the calls give."""
    D, Hq, Hkv, page, n = 128, 8, 2, 16, 5
    kp, vp, ks, vs = pools(20, page, Hkv, D, "int8")
    ks.fill_(0.01), vs.fill_(0.01)
    table, lengths = dev(np.arange(20).reshape(5, 4)), dev([3, 17, 33, 50, 1])
    qkv = torch.randn(n, Hq + 2 * Hkv, D, device="cuda").half()
    slots = table[:, 3] * page + 2
    positions, f = dev(np.arange(n)), freqs(D // 2)
    workspace = ops.paged_attn_workspace(n, Hq, Hkv, D, "cuda")

    def step():
        q = ops.rotary_paged_store(qkv[:, :Hq], qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:], positions, slots, f, kp, vp, kscales=ks, vscales=vs)
        out = ops.paged_attn(q, kp, vp, table, lengths, 0.1, kscales=ks, vscales=vs, workspace=workspace)
        return (q, out, *ops.paged_rows(kp, vp, ops.page_slots(table, lengths, page, 110)[0], ks, vs, dtype=torch.float16))

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for seed in range(3):
        qkv.copy_(torch.randn(qkv.shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").half())
        graph.replay()
        torch.cuda.synchronize()
        kept = [t.clone() for t in got]
        assert all(torch.equal(a, b) for a, b in zip(kept, step()))


@pytest.mark.parametrize("codes", CODES)
def test_long_offsets(ops, codes):
    """Pages that lie behind 2^32 codes of the pool: stored, read back and attended."""
    pages, page, Hkv, D = 36000, 64, 16, 128
    kp, vp = (torch.zeros(pages, page, Hkv, D, dtype=torch.int8, device="cuda").view(codes_plain.TYPES[codes]) for _ in range(2))
    ks, vs = (torch.zeros(pages, Hkv, page, device="cuda") for _ in range(2))
    slots = dev(np.concatenate([35999 * page + np.arange(64), 7 * page + np.arange(40)]))
    x = torch.randn(104, Hkv, D, device="cuda").half()
    ops.rotary_paged_store(None, x, x, None, slots, None, kp, vp, kscales=ks, vscales=vs)
    s = codes_plain.scale(x.double(), codes)
    held = (codes_plain.code(x.double(), s, codes).float() * s.float()).half()
    k, v = ops.paged_rows(kp, vp, slots, ks, vs, dtype=torch.float16)
    assert torch.equal(k, held) and torch.equal(v, held)
    q = torch.randn(1, Hkv, D, device="cuda").half()
    out = ops.paged_attn(q, kp, vp, dev([[35999, 7]]), dev([104]), 0.1, kscales=ks, vscales=vs)
    rows = codes_plain.code(x.double(), s, codes).float().double() * s
    want = torch.einsum("ht,thd->hd", torch.softmax(0.1 * torch.einsum("hd,thd->ht", q[0].double(), rows), -1), rows)
    assert bool(((out[0].double() - want).abs() <= 2.0 ** -10 * rows.abs().max()).all())


def test_refusals(ops):
    from kvcomp_b200._lib import KvcError
    kp, vp, ks, vs = pools(4, 16, 2, 128, "int8")
    x, i, q, table, lengths = torch.randn(3, 2, 128, device="cuda").half(), dev([0, 1, 2]), torch.randn(2, 4, 128, device="cuda").half(), dev([[0], [1]]), dev([3, 4])
    store = dict(q=None, k=x, v=x, positions=None, slots=i, frequencies=None, kpages=kp, vpages=vp, kscales=ks, vscales=vs)
    rows = dict(kpages=kp, vpages=vp, slots=i, kscales=ks, vscales=vs, dtype=torch.float16)
    attn = dict(q=q, kpages=kp, vpages=vp, table=table, lengths=lengths, scaling=0.1, kscales=ks, vscales=vs)
    ops.rotary_paged_store(**store), ops.paged_rows(**rows), ops.paged_attn(**attn)
    both = [dict(kscales=None), dict(kscales=None, vscales=None), dict(kscales=ks.double()), dict(kscales=ks[:3]), dict(vscales=vs.transpose(1, 2)), dict(kscales=ks.cpu()), dict(vpages=vp.view(torch.float8_e4m3fn)),
            dict(kpages=kp.half(), vpages=vp.half()), dict(kpages=kp[..., :120], vpages=vp[..., :120]), dict(vpages=vp[:2])]
    for call, good, more in ((ops.rotary_paged_store, store, [dict(vscales=ks), dict(vpages=kp), dict(k=x.float()), dict(slots=i.long())]),
                             (ops.paged_rows, rows, [dict(dtype=None), dict(dtype=torch.float32), dict(out=(x, x)), dict(out=(x, x[:1])), dict(slots=i[None])]),
                             (ops.paged_attn, attn, [dict(kscales=torch.cat([ks, ks], 1)[:, :2]), dict(vpages=torch.cat([vp, vp], 2)[:, :, :2])])):
        for change in both + more:
            with pytest.raises(KvcError):
                call(**{**good, **change})
    with pytest.raises(KvcError):
        ops.paged_rows(x[None].contiguous(), x[None].contiguous(), i, dtype=torch.bfloat16)          # (rows of 16 bits come as they are)
    assert ops.paged_rows(kp, vp, i[:0], ks, vs, dtype=torch.float16)[0].shape == (0, 2, 128)
    slots, starts = ops.page_slots(table[:0], lengths[:0], 16, 3)
    assert slots.tolist() == [-1, -1, -1] and starts.tolist() == [0]
    ops.page_shift(starts, lengths[:0], slots)
    assert slots.tolist() == [-1, -1, -1]
