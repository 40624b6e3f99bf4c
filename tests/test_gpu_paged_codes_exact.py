"""e4m3 keys: codes and scales of rows as they are rotated in 64 bits, whatever a rotation in 32 is off by."""
import math

import pytest
import torch

import codes_plain

pytestmark = pytest.mark.gpu

DTYPES = [torch.float16, torch.bfloat16]


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    from kvcomp_b200 import ops
    return ops


def rotate(x, positions, f, layout, factor=1.0):
    """x [N, H, D] in 64 bits, on the device."""
    y, r = x.double().clone(), 2 * len(f)
    angle = positions.double()[:, None, None] * f
    c, s = factor * torch.cos(angle), factor * torch.sin(angle)
    i0, i1 = (slice(0, r // 2), slice(r // 2, r)) if layout == "half" else (slice(0, r, 2), slice(1, r, 2))
    a, b = x[..., i0].double(), x[..., i1].double()
    y[..., i0], y[..., i1] = a * c - b * s, b * c + a * s
    return y


def check(ops, k, positions, f, layout, factor=1.0, views="slices"):
    """Codes and scales are the definition's to the bit, but where the 64-bit rotation itself is next to a border (its angles are off by 2^-52 of themselves: 1e-10 of a row's largest value here)."""
    N, H, D = k.shape
    page = 16
    pages = -(-N // page)
    kp, vp = (torch.zeros(pages, page, H, D, dtype=torch.int8, device="cuda").view(torch.float8_e4m3fn) for _ in range(2))
    ks, vs = (torch.zeros(pages, H, page, device="cuda") for _ in range(2))
    if views == "odd":
        wide = torch.zeros(N, H, D + 8, dtype=k.dtype, device="cuda")
        wide[..., 4:4 + D] = k
        k = wide[..., 4:4 + D]
    slots = torch.arange(N, dtype=torch.int32, device="cuda")
    ops.rotary_paged_store(None, k, k, positions, slots, f, kp, vp, layout=layout, factor=factor, kscales=ks, vscales=vs)
    x = rotate(k, positions, f, layout, factor)
    top = x.abs().amax(-1, keepdim=True)
    got_s = codes_plain.at_slots(ks, slots)[..., None].double()
    sure = (codes_plain.scale(x * (1 + 1e-10), "e4m3") == codes_plain.scale(x * (1 - 1e-10), "e4m3"))
    s = codes_plain.scale(x, "e4m3")
    wrong = (got_s != s) & sure
    assert not bool(wrong.any()), int(wrong.sum())
    got = codes_plain.bits(codes_plain.at_slots(kp, slots))
    want = codes_plain.bits(codes_plain.code(x, s, "e4m3"))
    wrong = (got != want) & sure
    wrong &= codes_plain.bits(codes_plain.code(x + 1e-10 * top, s, "e4m3")) == codes_plain.bits(codes_plain.code(x - 1e-10 * top, s, "e4m3"))
    wrong &= ~((x.abs() < s * 2.0 ** -10 * 1.01) & ((got & 0x7f) == (want & 0x7f)))                 # (zeros of either sign)
    assert not bool(wrong.any()), int(wrong.sum())


def freqs(n):
    return 10000.0 ** (-torch.arange(n, dtype=torch.float64, device="cuda") / max(n, 1))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("D,r,views", [(128, 128, "slices"), (128, 64, "slices"), (96, 24, "slices"), (64, 64, "odd")])
def test_random_keys(ops, dtype, layout, D, r, views):
    gen = torch.Generator(device="cuda").manual_seed(D + r)
    N, H = 12000, 8
    k = (torch.randn(N, H, D, generator=gen, device="cuda") * torch.exp(torch.randn(N, H, 1, generator=gen, device="cuda"))).to(dtype)
    check(ops, k, torch.randint(0, 50000, (N,), generator=gen, device="cuda", dtype=torch.int32), freqs(r // 2), layout, views=views)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("factor", [1.0, 1.2079441541679836])
@pytest.mark.parametrize("r,views", [(128, "slices"), (40, "slices"), (128, "odd")])
def test_pairs_that_cancel(ops, dtype, layout, factor, r, views):
    """Pairs of which one value is what the other's rounding leaves: products that are off by the last bits of theirs, and by many of their difference's."""
    gen = torch.Generator(device="cuda").manual_seed(r)
    N, H, D = 4000, 2, 128
    f, positions = freqs(r // 2), torch.randint(1, 50000, (N,), generator=gen, device="cuda", dtype=torch.int32)
    k = torch.randn(N, H, D, generator=gen, device="cuda").to(dtype)
    angle = positions.double()[:, None, None] * f
    size = torch.exp(torch.randn(N, H, r // 2, generator=gen, device="cuda"))
    a, b = (size * torch.sin(angle)).to(dtype), (size * torch.cos(angle)).to(dtype)           # a cos - b sin is next to nothing
    if layout == "half":
        k[..., :r // 2], k[..., r // 2:r] = a, b
    else:
        k[..., 0:r:2], k[..., 1:r:2] = a, b
    check(ops, k, positions, f, layout, factor, views)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("views", ["slices", "odd"])
def test_rows_at_the_border_of_two_scales(ops, dtype, views):
    """Rows whose largest value lies next to 448 times a power of two, on either side; the smallest of the others show which scale was taken."""
    gen = torch.Generator(device="cuda").manual_seed(3)
    D, f, found = 64, freqs(32), []
    for _ in range(8):
        n = 1 << 23
        position, i = torch.randint(1, 50000, (n,), generator=gen, device="cuda"), torch.randint(0, 32, (n,), generator=gen, device="cuda")
        a, b = (torch.randn(n, generator=gen, device="cuda").to(dtype) for _ in range(2))
        angle = position.double() * f[i]
        m, _ = torch.frexp((a.double() * torch.cos(angle) - b.double() * torch.sin(angle)).abs())
        at = ((m / 0.875 - 1).abs() < 2.5e-7).nonzero()[:, 0]
        found += list(zip(position[at].tolist(), i[at].tolist(), a[at].tolist(), b[at].tolist()))
    assert len(found) >= 10
    positions = torch.tensor([p for p, *_ in found], dtype=torch.int32, device="cuda")
    k = torch.zeros(len(found), 1, D, dtype=dtype, device="cuda")
    for n, (p, i, a, b) in enumerate(found):
        y = math.hypot(a, b)
        k[n, 0] = torch.randn(D, generator=gen, device="cuda").clamp(-3, 3).to(dtype) * (y * 1e-5)
        c, s = math.cos(p * float(f[i])), math.sin(p * float(f[i]))
        k[n, 0, i], k[n, 0, i + 32] = (a, b) if abs(a * c - b * s) >= abs(b * c + a * s) else (0.0, 0.0)
    check(ops, k, positions, f, "half", views=views)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("views", ["slices", "odd"])
def test_first_positions(ops, dtype, views):
    """Position 0 turns nothing: with a factor of 1 keys are coded as they are, ties and all; with another they are products."""
    gen = torch.Generator(device="cuda").manual_seed(4)
    k = torch.randn(30000, 4, 64, generator=gen, device="cuda").to(dtype)
    positions = torch.zeros(30000, dtype=torch.int32, device="cuda")
    check(ops, k, positions, freqs(32), "half", views=views)
    for factor in (1.2079441541679836, 0.1, 1.0 + 2.0 ** -20):
        check(ops, k, positions, freqs(32), "interleaved", factor=float(torch.tensor(factor, dtype=torch.float32)), views=views)
