"""Plain forms of the paged cache's operators for the tests: numpy and torch in 64 bits, one request after the other."""
import math

import numpy as np
import torch


def plan(lengths, new, table, free, head, page, tokens):
    """What ops.page_plan answers, from lists and a numpy table (a copy of which comes back with the new pages)."""
    table, pool = table.copy(), len(free)
    out_lengths, starts, taken, slots, positions = [], [], [], [-1] * tokens, [0] * tokens
    start, asked, used = 0, 0, 0
    refused = False
    for b, (held, add) in enumerate(zip(lengths, new)):
        held, add = max(held, 0), max(add, 0)
        owned, wanted = -(-held // page), -(-(held + add) // page)
        starts.append(min(start, tokens))
        fits = wanted <= table.shape[1] and start + add <= tokens
        need = wanted - owned if fits else 0
        served = fits and (need == 0 or head + asked + need <= pool)
        taken.append(min(head + asked, pool) if served else -1)
        if served and need:
            table[b, owned:wanted] = free[head + asked:head + asked + need]
            used = asked + need
        for j in range(add):
            if start + j < tokens:
                positions[start + j] = held + j
                if served:
                    slots[start + j] = int(table[b, (held + j) // page]) * page + (held + j) % page
        out_lengths.append(held + add if served else held)
        refused |= not served
        start += add
        asked += need
    starts.append(min(start, tokens))
    return dict(lengths=out_lengths, head=head + used, starts=starts, taken=taken, slots=slots, positions=positions, table=table, refused=refused)


def release(lengths, done, table, free, head, page):
    pages, out = [], []
    full = False
    for b, held in enumerate(lengths):
        n = -(-held // page) if done[b] else 0
        full |= n > 0 and len(pages) + n > head
        if done[b] and not full:
            pages += [int(p) for p in table[b, :n]]
        out.append(0 if done[b] and not full else held)
    free = np.array(free)
    free[head - len(pages):head] = pages
    return dict(lengths=out, head=head - len(pages), free=free, refused=full)


def rotate(x, positions, frequencies, layout, factor=1.0, inverse=False):
    """x [N, H, D] in 64 bits, angles by positions [N] x frequencies [r / 2]."""
    y = x.double().clone()
    r = 2 * len(frequencies)
    angle = positions.double()[:, None, None] * frequencies.double()
    c, s = factor * torch.cos(angle), factor * torch.sin(angle) * (-1 if inverse else 1)
    i0, i1 = (slice(0, r // 2), slice(r // 2, r)) if layout == "half" else (slice(0, r, 2), slice(1, r, 2))
    a, b = x[..., i0].double(), x[..., i1].double()
    y[..., i0], y[..., i1] = a * c - b * s, b * c + a * s
    return y


def rotate_bound(x, want, frequencies, layout, factor):
    """How far a rotation in fp32, rounded once, may be off.  cos and sin: their fp32 values are off by 2^-24 of 1, the argument (half turns up to 1, rounded to
    fp32) moves them by pi 2^-24, the factor by a rounding more: 6 2^-24 of the factor; two products, their sum: 3 2^-24 of the pair's sum of magnitudes."""
    eps = torch.finfo(x.dtype).eps / 2
    tiny = 2.0 ** -25 if x.dtype == torch.float16 else 0.0            # half a step of the smallest numbers
    size = x.double().abs().clone()
    r = 2 * len(frequencies)
    i0, i1 = (slice(0, r // 2), slice(r // 2, r)) if layout == "half" else (slice(0, r, 2), slice(1, r, 2))
    both = size[..., i0] + size[..., i1]
    size[..., i0], size[..., i1] = both, both
    off = size * abs(factor) * 10 * 2.0 ** -24
    off[..., r:] = 0
    return off + eps * (want.abs() + off) + tiny


def attend(q, kpages, vpages, table, lengths, scaling, window=0):
    """(out, lse, bound of out, bound of lse) in 64 bits.  Tokens whose page is outside the pool are left out.

    The bound: an fp32 score is off by D products and sums of magnitude sum |q k| (2^-23 each: tensor cores may cut off) and by three roundings on the way to the
    exponent; with d that sum over the largest token, a weight and the sum of weights are off by a factor 1 + d each, the weights besides by
    what their two 16-bit pieces leave (2^-20 fp16, 2^-16 bf16) and the sums over L tokens by 2^-23 a step."""
    B, Hq, D = q.shape
    pool, page, Hkv, _ = kpages.shape
    group = Hq // Hkv
    out = torch.zeros(B, Hq, D, dtype=torch.float64)
    off = torch.zeros(B, Hq, D, dtype=torch.float64)
    lse = torch.full((B, Hq), -math.inf, dtype=torch.float64)
    lse_off = torch.zeros(B, Hq, dtype=torch.float64)
    q, table = q.cpu().double(), table.cpu()
    piece = 2.0 ** -20 if kpages.dtype == torch.float16 else 2.0 ** -16
    eps = torch.finfo(kpages.dtype).eps / 2
    for b, n in enumerate(int(v) for v in lengths):
        n = min(max(n, 0), table.shape[1] * page)
        t = torch.arange(max(0, n - window) if window else 0, n)
        p = table[b, t // page].long() if len(t) else t
        t, p = t[(p >= 0) & (p < pool)], p[(p >= 0) & (p < pool)]
        if len(t) == 0:
            continue
        k = kpages[p.to(kpages.device), (t % page).to(kpages.device)].cpu().double()
        v = vpages[p.to(kpages.device), (t % page).to(kpages.device)].cpu().double()
        for h in range(Hq):
            kh, vh = k[:, h // group], v[:, h // group]
            s = scaling * (kh @ q[b, h])
            size = abs(scaling) * (kh.abs() @ q[b, h].abs())
            w = torch.softmax(s, -1)
            out[b, h], lse[b, h] = w @ vh, torch.logsumexp(s, -1)
            d = float(size.max()) * (D + 4) * 2.0 ** -23 + (float(s.abs().max()) + 24) * 2.0 ** -22
            off[b, h] = (w @ vh.abs()) * (2 * d + piece + (len(t) + 64) * 2.0 ** -23)
            lse_off[b, h] = 2 * d + (len(t) + 64) * 2.0 ** -23 + float(lse[b, h].abs()) * 2.0 ** -23
    tiny = 2.0 ** -25 if kpages.dtype == torch.float16 else 0.0
    return out, lse, off + eps * (out.abs() + off) + tiny, lse_off


def pool(gen, pages, page, kv_heads, dim, dtype, device, order="token"):
    """A pool [pages, page, kv heads, dim] of normal values; order "head": each head's rows of a page lie together; "padded": rows lie apart."""
    if order == "head":
        return torch.randn(pages, kv_heads, page, dim, generator=gen, device=device).to(dtype).transpose(1, 2)
    if order == "padded":
        return torch.randn(pages, page, kv_heads + 1, dim + 8, generator=gen, device=device).to(dtype)[:, :, :kv_heads, :dim]
    return torch.randn(pages, page, kv_heads, dim, generator=gen, device=device).to(dtype)


def tables(rng, lengths, page, pages, extra=0):
    """Block table of requests over pages in random order, -1 behind a request's pages."""
    need = [-(-max(n, 0) // page) for n in lengths]
    assert sum(need) <= pages
    order = rng.permutation(pages).astype(np.int32)
    table = np.full((len(lengths), max(need + [1]) + extra), -1, dtype=np.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return table, order, at
