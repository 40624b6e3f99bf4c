"""Plain forms of rows in 8 bits for the tests, in 64 bits."""
import torch

LEAST = 2.0 ** -100
TYPES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}


def scale(x, codes):
    """The scale of each row of x (64 bits): [..., 1], a number of 32 bits."""
    top = x.abs().amax(-1, keepdim=True)
    if codes == "int8":
        s = (top / 127).float().double()
    else:
        m, e = torch.frexp(top)                                     # top = m 2^e, m in [1/2, 1); 448 = 7/8 2^9
        s = torch.where(top > 0, torch.ldexp(torch.ones_like(top), e - 9 + (m > 0.875).int()), 0.0)
    s = torch.clamp(s, min=LEAST)
    return torch.where(torch.isfinite(x).all(-1, keepdim=True), s, torch.nan)


def code(x, s, codes):
    """Codes of rows of x (64 bits) with scales s: to the nearest, ties to even."""
    if codes == "int8":
        return torch.round(x / s).clamp(-127, 127).to(torch.int8)
    t = x / s
    step = torch.ldexp(torch.ones_like(t), torch.clamp(torch.frexp(t)[1] - 4, min=-9))
    return (torch.round(t / step) * step).float().to(torch.float8_e4m3fn)


def half_step(x, s, codes):
    """How far a value is from its code's, at most: half a step, of e4m3 where it lies (2^-4 of it, 2^-10 of the scale below the normal codes)."""
    return s / 2 if codes == "int8" else torch.maximum(x.abs() * 2.0 ** -4, s * 2.0 ** -10)


def bits(t):
    return t.view(torch.int8)


def at_slots(pool, slots):
    """Rows of a pool of codes or of scales [pages, heads, page_size]."""
    page = pool.shape[1] if pool.dim() == 4 else pool.shape[2]
    slots = slots.long()
    if pool.dim() == 3:
        return pool.transpose(1, 2)[slots // page, slots % page]
    rows = (bits(pool) if pool.element_size() == 1 else pool)[slots // page, slots % page]
    return rows.view(pool.dtype)


def values(pool, scales):
    """A pool of codes and its scales as 64-bit values."""
    return pool.float().double() * scales.double().transpose(1, 2)[..., None]


def coded(x, codes):
    """(codes, scales) of a pool of values [pages, page_size, heads, channels]."""
    s = scale(x.double(), codes)
    return code(x.double(), s, codes), s[..., 0].transpose(1, 2).float().contiguous()
