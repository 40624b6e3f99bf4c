"""Attention over codes whose rows' sizes lie far apart: a value's size counts with its weight, not by itself."""
import math

import pytest
import torch

import codes_plain

pytestmark = pytest.mark.gpu

DTYPES = [torch.float16, torch.bfloat16]
CODES = ["int8", "e4m3"]


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    from kvcomp_b200 import ops
    return ops


def check(ops, q, k, v, codes, scaling, page=16, lengths=None):
    """q [B, Hq, D] over the tokens k, v [B, tokens, Hkv, D], of request b the first lengths[b]."""
    B, n, Hkv, D = k.shape
    Hq, g = q.shape[1], q.shape[1] // Hkv
    lengths = [n] * B if lengths is None else lengths
    pages = -(-n // page)
    pad = lambda x: torch.nn.functional.pad(x, (0, 0, 0, 0, 0, pages * page - n)).reshape(B * pages, page, Hkv, D)  # noqa: E731
    (kp, ks), (vp, vs) = codes_plain.coded(pad(k), codes), codes_plain.coded(pad(v), codes)
    table = torch.arange(B * pages, dtype=torch.int32, device="cuda").view(B, pages)
    out, lse = ops.paged_attn(q, kp, vp, table, torch.tensor(lengths, dtype=torch.int32, device="cuda"), scaling, return_lse=True, kscales=ks, vscales=vs)
    kd, vd = (codes_plain.values(p, s).view(B, -1, Hkv, D) for p, s in ((kp, ks), (vp, vs)))
    eps = torch.finfo(q.dtype).eps / 2
    for b, m in enumerate(lengths):
        if m == 0:
            assert not bool(out[b].any()) and bool(torch.isneginf(lse[b]).all())
            continue
        x, kb, vb = q[b].double().view(Hkv, g, D), kd[b, :m], vd[b, :m]
        s = scaling * torch.einsum("hgd,thd->hgt", x, kb)
        size = abs(scaling) * torch.einsum("hgd,thd->hgt", x.abs(), kb.abs())
        w = torch.softmax(s, -1)
        want, want_lse = torch.einsum("hgt,thd->hgd", w, vb), torch.logsumexp(s, -1)
        # A token's score is off by D products and sums (2^-23 of the sum of their sizes) and by roundings on the way to the exponent, of the score and of the largest one; its weight by a factor 1
        # + d, the sum of weights by their mean.  A weight times its value's scale has two pieces of 16 bits (2^-21) and is off by 2^-39 of the largest such product besides; a code is 448 at most
        # where the scale is more than a 448th of the row's largest, or 127 where it is a 127th: 2^-38 of the largest product of a weight and a row's largest value.  Sums of m tokens: 2^-23 a step.
        d = size * (D + 4) * 2.0 ** -23 + (s.abs() + s.abs().amax(-1, keepdim=True) + 24) * 2.0 ** -22
        mean = (w * d).sum(-1, keepdim=True)
        of = torch.einsum("hgt,thd->hgd", w * (d + mean + 2.0 ** -21 + (m + 64) * 2.0 ** -23), vb.abs())
        of = of + m * 2.0 ** -38 * (w * vb.abs().amax(-1).T[:, None]).amax(-1, keepdim=True)
        # A weight is a number of 32 bits, 1 the largest of a head: below 2^-126 it is no normal one and may be taken for nothing (2^-125: its own error; e^-87 is 2^-125.5).
        of = of + torch.einsum("hgt,thd->hgd", w * (w < 2.0 ** -125 * w.amax(-1, keepdim=True)), vb.abs())
        bound = of + eps * (want.abs() + of) + (2.0 ** -25 if q.dtype == torch.float16 else 2.0 ** -134)
        off = (out[b].double().view(Hkv, g, D) - want).abs()
        assert bool((off <= bound).all()), (b, float((off / bound).max()), out[b].view(Hkv, g, D)[..., :2].tolist(), want[..., :2].tolist())
        lse_bound = 2 * mean[..., 0] + (m + 64) * 2.0 ** -23 + want_lse.abs() * 2.0 ** -22
        assert bool(((lse[b].double().view(Hkv, g) - want_lse).abs() <= lse_bound).all())
    return out


def rows(gen, *shape):
    return torch.randn(shape, generator=gen, device="cuda")


def with_scores(q, scores, scaling):
    """A key whose scores with the queries [g, D] are these."""
    return torch.linalg.pinv(q.double()) @ (torch.as_tensor(scores, dtype=torch.float64, device="cuda") / scaling)


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("dtype,small,large", [(torch.float16, 1e-4, 6e4), (torch.bfloat16, 1.0, 1e13), (torch.bfloat16, 1e-10, 1e28), (torch.float16, 1.0, 6e4)])
@pytest.mark.parametrize("D,g", [(64, 1), (96, 4), (128, 3), (128, 12), (256, 8)])
@pytest.mark.parametrize("at", [0, 350, 699])
def test_a_large_value_with_next_to_no_weight(ops, dtype, small, large, codes, D, g, at):
    """One token's value is many orders of magnitude larger; heads that give it no weight have the others' result, heads that give it some have its part, and one may lie beside the other."""
    gen = torch.Generator(device="cuda").manual_seed(D + g + at)
    n, scaling = 700, 1 / math.sqrt(D)
    q = rows(gen, 1, g, D).to(dtype)
    k, v = rows(gen, 1, n, 1, D) * 0.5, rows(gen, 1, n, 1, D) * small
    v[0, at] *= large / small
    ratio = math.log(large / small)
    k[0, at, 0] = with_scores(q[0], [(-200.0, -ratio, 0.0, -1.5 * ratio, -0.5 * ratio)[h % 5] for h in range(g)], scaling).float()
    check(ops, q, k, v, codes, scaling)


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128, 256])
def test_sizes_that_rise_and_fall(ops, dtype, codes, D):
    """Scores rise from token to token while values shrink, and the other way round; in between they do as they like."""
    gen = torch.Generator(device="cuda").manual_seed(D)
    n, scaling = 400, 1 / math.sqrt(D)
    q = rows(gen, 3, 2, D).to(dtype)
    k, v = rows(gen, 3, n, 1, D) * 0.1, rows(gen, 3, n, 1, D)
    way = torch.linspace(-1, 1, n, device="cuda")
    sizes = 4.0 if dtype == torch.float16 else 15.0                 # (powers of ten, up and down)
    for b, (up, grow) in enumerate(((60.0, -sizes), (-60.0, sizes), (30.0, sizes))):
        k[b] += way[:, None, None] * up * with_scores(q[b].float(), [1.0, 1.0], scaling).float()
        v[b] *= 10.0 ** (grow * way)[:, None, None]
    v[2] *= 10.0 ** (rows(gen, n, 1, 1).clamp(-2, 2) * 0.2 * sizes)
    check(ops, q, k, v, codes, scaling, page=8, lengths=[n, n - 7, 33])


@pytest.mark.parametrize("codes", CODES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_of_zeros(ops, dtype, codes):
    """Rows of zeros, whose scale is the least, with all the weight and with some, beside the largest values; and nothing but zeros."""
    D, n, scaling = 128, 300, 0.1
    gen = torch.Generator(device="cuda").manual_seed(2)
    q = rows(gen, 3, 2, D).to(dtype)
    k, v = rows(gen, 3, n, 1, D), rows(gen, 3, n, 1, D) * (3e4 if dtype == torch.float16 else 1e37)
    v[0, 1:] = 0.0
    v[1, ::2] = 0.0
    v[2] = 0.0
    k[0, 0, 0] = with_scores(q[0], [-5.0, -40.0], scaling).float()
    k[1, 0, 0] = with_scores(q[1], [30.0, 90.0], scaling).float()
    out = check(ops, q, k, v, codes, scaling)
    assert not bool(out[2].any())


@pytest.mark.parametrize("codes", CODES)
def test_long_requests(ops, codes):
    """A large value without weight in a column that many CTAs have parts of."""
    D, n, scaling = 128, 40000, 1 / math.sqrt(128)
    gen = torch.Generator(device="cuda").manual_seed(5)
    q = rows(gen, 1, 4, D).to(torch.bfloat16)
    k, v = rows(gen, 1, n, 2, D) * 0.5, rows(gen, 1, n, 2, D)
    for at, head in ((20000, 0), (17, 1)):
        v[0, at, head] *= 1e13
        k[0, at, head] = with_scores(q[0, 2 * head:2 * head + 2], [-200.0, -30.0], scaling).float()
    check(ops, q, k, v, codes, scaling, page=64)


@pytest.mark.parametrize("codes", CODES)
def test_keys_whose_products_leave_32_bits(ops, codes):
    """Keys of 1e37 and queries of 1e-37 have scores like any other's."""
    D, n = 64, 50
    gen = torch.Generator(device="cuda").manual_seed(7)
    q = (rows(gen, 1, 2, D) * 1e-37).to(torch.bfloat16)
    k, v = rows(gen, 1, n, 1, D) * 1e37, rows(gen, 1, n, 1, D)
    check(ops, q, k, v, codes, 0.1)
