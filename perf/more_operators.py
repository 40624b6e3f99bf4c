"""Operators of a paged key-value cache whose tokens are held in 8 bits, and of a batch whose requests continue common prefixes: what is measured of them, their
plain forms, and their values in 64 bits.

    write     queries and keys rotated, keys and values coded in 8 bits as they go to their slots, and the step's rows as the cache then holds them
                                                                                  (ops.rotary_paged_store with scales, ops.paged_rows)
    read      the tokens that requests have, out of their pages into packed rows  (ops.page_slots, ops.paged_rows)
    attend    one new token per request over pages of 8-bit codes                 (ops.paged_attn with scales)
    shared    one new token per request over a prefix that several requests share and its own tokens behind it
                                                                                  (ops.prefix_plan, ops.paged_attn_shared)

A row (a token's channels of a head) has one scale.  int8: amax / 127 in 32 bits, codes round(x / scale), ties to even; e4m3: the least power of two with amax / scale <= 448,
codes x / scale rounded to e4m3; no scale is below 2^-100.
"""
import math

import numpy as np
import torch

own = False

TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
CODES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
LEAST = 2.0 ** -100                                                 # of a scale


# ---- the cases -------------------------------------------------------------------------------------

def listed():
    return [
        # a decode step of one layer, Llama-2-7B's heads, batch 8
        dict(name="write step", op="write", tokens=8, heads=32, kv_heads=32, dim=128, rotary=128, layout="half", type="fp16", codes="int8", held=4096, page=64),
        # prompts of one layer, Phi-3-medium's heads in bf16, part of the head rotated, slices of one projection
        dict(name="write prompts", op="write", tokens=16384, heads=40, kv_heads=10, dim=128, rotary=96, layout="half", type="bf16", codes="int8", held=16384, page=128),
        # an odd number of tokens, interleaved pairs, floating codes
        dict(name="write odd e4m3", op="write", tokens=4099, heads=32, kv_heads=8, dim=128, rotary=128, layout="interleaved", type="fp16", codes="e4m3", held=131072, page=16),
        # the prefix of one short prompt whose next chunk attends with rows in hand
        dict(name="read short", op="read", requests=1, kv_heads=32, dim=128, type="fp16", codes="int8", longest=777, page=16),
        # prefixes of a batch of prompts in chunks, of every length, Mistral-7B's heads
        dict(name="read chunks", op="read", requests=16, kv_heads=8, dim=128, type="bf16", codes="e4m3", longest=16384, page=64),
        # the first answer to one short request, Llama-2-7B's heads
        dict(name="attend one short", op="attend", requests=1, heads=32, kv_heads=32, dim=128, type="fp16", codes="int8", longest=777, ragged=False, page=16, window=0),
        # Llama-2-7B's heads, batch 8, 4096 tokens
        dict(name="attend 8 x 4096", op="attend", requests=8, heads=32, kv_heads=32, dim=128, type="fp16", codes="int8", longest=4096, ragged=False, page=64, window=0),
        # Mistral-7B's grouped heads in bf16, batch 16, 32768 tokens, floating codes
        dict(name="attend 16 x 32768 e4m3", op="attend", requests=16, heads=32, kv_heads=8, dim=128, type="bf16", codes="e4m3", longest=32768, ragged=False, page=64, window=0),
        # a serving batch: lengths of every size, some requests idle, Phi-3-medium's heads, a sliding window
        dict(name="attend ragged window", op="attend", requests=64, heads=40, kv_heads=10, dim=128, type="bf16", codes="int8", longest=16384, ragged=True, page=128, window=4096),
        # a few answers to one question about a short common text
        dict(name="shared 4 x 777", op="shared", groups=1, members=4, prefix=777, longest=50, heads=32, kv_heads=32, dim=128, type="fp16", page=16),
        # a serving batch behind one long system prompt, Mistral-7B's grouped heads
        dict(name="shared 64 x 16384", op="shared", groups=1, members=64, prefix=16384, longest=500, heads=32, kv_heads=8, dim=128, type="bf16", page=64),
        # eight documents with sixteen requests each, Phi-3-medium's heads
        dict(name="shared 8 x 16 x 8000", op="shared", groups=8, members=16, prefix=8000, longest=1000, heads=40, kv_heads=10, dim=128, type="fp16", page=128),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["write", "read", "attend", "attend", "shared", "shared"])
    page = rng.choice([8, 16, 24, 32, 64, 128, 256])
    kind, codes = rng.choice(["fp16", "bf16"]), rng.choice(["int8", "e4m3"])
    dim = rng.choice([64, 96, 128, 128, 256])
    kv_heads, group = rng.choice([(32, 1), (8, 4), (10, 4), (4, 8), (1, 16), (2, 7), (5, 3), (12, 1)])
    if op == "write":
        tokens = _log(rng, 1, max(16, 16384 * 60 * 128 // (kv_heads * (group + 2) * dim)))
        return dict(op=op, tokens=tokens, heads=kv_heads * group, kv_heads=kv_heads, dim=dim, rotary=rng.choice([dim, dim, dim // 2, dim // 4]),
                    layout=rng.choice(["half", "interleaved"]), type=kind, codes=codes, held=_log(rng, 1, 1000000), page=page)
    if op == "read":
        requests = _log(rng, 1, 64)
        return dict(op=op, requests=requests, kv_heads=kv_heads, dim=dim, type=kind, codes=codes, longest=_log(rng, 1, max(1, 100000000 // (requests * kv_heads * dim))), page=page)
    if op == "attend":
        requests = _log(rng, 1, 256)
        longest = _log(rng, 1, max(1, min(131072, 500000000 // (requests * kv_heads * dim))))
        return dict(op=op, requests=requests, heads=kv_heads * group, kv_heads=kv_heads, dim=dim, type=kind, codes=codes, longest=longest, ragged=rng.random() < 0.6,
                    page=page, window=rng.choice([0, 0, _log(rng, 1, 8192)]))
    dim = min(dim, 128)
    groups = rng.choice([1, 1, 2, 3, 8])
    members = _log(rng, 2, 256 // groups)
    prefix = _log(rng, 16, min(32768, 60000000 // (groups * kv_heads * dim), 4000000000 // (groups * members * kv_heads * group * dim)))
    return dict(op=op, groups=groups, members=members, prefix=prefix, longest=_log(rng, 1, min(1000, 120000000 // (groups * members * kv_heads * dim))),
                heads=kv_heads * group, kv_heads=kv_heads, dim=dim, type=kind, page=page)


# ---- what a user's program has in hand -------------------------------------------------------------

def _lengths(case):
    """The requests' lengths, in no order: the same numbers whatever the seed."""
    if case["op"] == "shared":                                      # the groups' prefixes, then the members' own tokens
        r = np.random.RandomState(5 + case["members"] + 7919 * case["prefix"])
        prefixes = np.maximum(1, np.floor(case["prefix"] * (1 - 0.3 * r.random_sample(case["groups"])))).astype(np.int64)
        prefixes[0] = case["prefix"]
        return prefixes, r.randint(1, case["longest"] + 1, case["groups"] * case["members"]).astype(np.int64)
    n, top = case["requests"], case["longest"]
    if case["op"] == "attend" and not case["ragged"]:
        return np.full(n, top, dtype=np.int64)
    r = np.random.RandomState(1 + n + 7919 * top)
    got = np.floor(top * r.random_sample(n) ** 2).astype(np.int64) + (r.random_sample(n) < 0.9)      # many short ones, a few idle, one of full length
    got[0] = top
    return np.minimum(got, top)


def _pages_of(lengths, page):
    return (lengths + page - 1) // page


def _table(order, lengths, page, width):
    """Block table rows of requests whose pages come one after the other from `order`; behind a row's pages -1."""
    need = _pages_of(lengths, page)
    first = np.cumsum(need) - need
    at = np.arange(width)[None, :]
    table = np.where(at < need[:, None], order[np.minimum(first[:, None] + at, len(order) - 1)], -1)
    return table.astype(np.int32)


def _gpu(a, dtype=None):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda() if dtype is None else torch.from_numpy(np.ascontiguousarray(a)).to(dtype).cuda()


def _coded_pool(pool, codes):
    """A pool's rows in 8 bits: codes [pages, page_size, heads, channels] and scales [pages, heads, page_size]."""
    c, s = _coded(pool, codes)
    return c, s[..., 0].transpose(1, 2).contiguous()


def prepare(case, seed):
    rng = np.random.RandomState(seed % (1 << 31))
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    op, page, dim, hkv = case["op"], case["page"], case["dim"], case["kv_heads"]
    dtype = TYPES[case["type"]]
    state = dict(case=case)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda", dtype=dtype)

    def channels(*shape):                                           # channels of different size, as keys have them
        x = normal(*shape)
        return x.mul_(torch.exp(0.5 * torch.randn(shape[-2:], generator=gen, device="cuda")).to(dtype))

    if op == "write":
        tokens, hq = case["tokens"], case["heads"]
        qkv = channels(tokens, hq + 2 * hkv, dim)                   # one projection's output: its slices have rows that lie apart
        pages = -(-tokens // page) + 2
        state.update(q=qkv[:, :hq], k=qkv[:, hq:hq + hkv], v=qkv[:, hq + hkv:], slots=_gpu(rng.permutation(pages * page)[:tokens], torch.int32),
                     positions=_gpu(rng.randint(0, case["held"], tokens), torch.int32),
                     frequencies=_gpu(10000.0 ** (-np.arange(0, case["rotary"], 2, dtype=np.float64) / case["rotary"])),
                     kpages=torch.zeros(pages, page, hkv, dim, dtype=CODES[case["codes"]], device="cuda"),
                     vpages=torch.zeros(pages, page, hkv, dim, dtype=CODES[case["codes"]], device="cuda"),
                     kscales=torch.zeros(pages, hkv, page, device="cuda"), vscales=torch.zeros(pages, hkv, page, device="cuda"))
        return state
    if op == "shared":
        groups, members = case["groups"], case["members"]
        prefixes, mine = _lengths(case)
        n = groups + groups * members
        at = rng.permutation(n)                                     # which request of the cache each is
        lengths, parents, shared = np.zeros(n, dtype=np.int64), np.full(n, -1, dtype=np.int64), np.zeros(n, dtype=np.int64)
        lengths[at] = np.concatenate([prefixes, mine])
        of = np.repeat(np.arange(groups), members)
        parents[at[groups:]], shared[at[groups:]] = at[of], prefixes[of]
        follows = parents >= 0                                      # the followers bring a token each; those that hold a prefix bring none
        starts = np.concatenate([[0], np.cumsum(follows)])
        pool = int(_pages_of(lengths, page).sum()) + 2
        state.update(q=normal(groups * members, case["heads"], dim), kpages=channels(pool, page, hkv, dim), vpages=normal(pool, page, hkv, dim),
                     table=_gpu(_table(rng.permutation(pool), lengths, page, int(_pages_of(lengths, page).max()))), lengths=_gpu(lengths, torch.int32),
                     parents=_gpu(parents, torch.int32), shared=_gpu(shared, torch.int32), starts=_gpu(starts, torch.int32), scaling=1.0 / math.sqrt(dim),
                     holders=_gpu(at[:groups]), followers=_gpu(at[groups:].reshape(groups, members)))
        if own:                                                     # what the program keeps as long as the same requests follow the same prefixes, and for all its steps
            from kvcomp_b200 import ops
            state["plan"] = ops.prefix_plan(state["parents"], state["shared"])
            state["workspace"] = ops.paged_attn_shared_workspace(n, case["heads"], hkv, dim, "cuda")
        return state
    lengths = rng.permutation(_lengths(case))
    pool = int(_pages_of(lengths, page).sum()) + 2
    width = max(1, int(_pages_of(lengths, page).max()))
    kpages, kscales = _coded_pool(channels(pool, page, hkv, dim), case["codes"])
    vpages, vscales = _coded_pool(normal(pool, page, hkv, dim), case["codes"])
    state.update(kpages=kpages, kscales=kscales, vpages=vpages, vscales=vscales, table=_gpu(_table(rng.permutation(pool), lengths, page, width)),
                 lengths=_gpu(lengths, torch.int32), tokens=int(lengths.sum()))
    if op == "attend":
        state.update(q=normal(case["requests"], case["heads"], dim), scaling=1.0 / math.sqrt(dim))
        if own:                                                     # what the program's cache keeps for all its steps
            from kvcomp_b200 import ops
            state["workspace"] = ops.paged_attn_workspace(case["requests"], case["heads"], hkv, dim, "cuda")
    return state


# ---- one pass --------------------------------------------------------------------------------------

def run(state):
    if own:
        return _run_own(state)
    return PLAIN[state["case"]["op"]](state)


def _run_own(state):
    from kvcomp_b200 import ops
    case = state["case"]
    pools = [state[name] for name in ("kpages", "vpages")]
    if case["op"] == "shared":
        out, lse = ops.paged_attn_shared(state["q"], *pools, state["table"], state["lengths"], state["plan"], state["scaling"], return_lse=True,
                                         workspace=state["workspace"], starts=state["starts"])
        return dict(out=out, lse=lse)
    scales = dict(kscales=state["kscales"], vscales=state["vscales"])
    if case["op"] == "write":
        q = ops.rotary_paged_store(state["q"], state["k"], state["v"], state["positions"], state["slots"], state["frequencies"], *pools, layout=case["layout"], **scales)
        k, v = ops.paged_rows(*pools, state["slots"], dtype=TYPES[case["type"]], **scales)
        return dict(q=q, k=k, v=v)
    if case["op"] == "read":
        slots, starts = ops.page_slots(state["table"], state["lengths"], case["page"], state["tokens"])
        k, v = ops.paged_rows(*pools, slots, dtype=TYPES[case["type"]], **scales)
        return dict(k=k, v=v, starts=starts)
    out, lse = ops.paged_attn(state["q"], *pools, state["table"], state["lengths"], state["scaling"], window=case["window"], return_lse=True,
                              workspace=state["workspace"], **scales)
    return dict(out=out, lse=lse)


def _power(e):
    """2^e in 64 bits."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _coded(x, codes):
    """Rows of x in 8 bits, and their scales [..., 1].  In 64 bits where a value lies next to the border of two codes."""
    x = x.float()
    top = x.abs().amax(-1, keepdim=True)
    if codes == "int8":
        s = (top.double() / 127).float().clamp(min=LEAST)
        return torch.round(x.double() / s.double()).clamp(-127, 127).to(torch.int8), s
    m, e = torch.frexp(top.double() / 448)                           # m 2^e with m in [1/2, 1)
    s = _power(torch.where(m == 0.5, e - 1, e).clamp(min=-100)).float()
    s = torch.where(top > 0, s, LEAST)
    return (x / s).to(torch.float8_e4m3fn), s


def _at(state):
    slots = state["slots"].long()
    return slots // state["case"]["page"], slots % state["case"]["page"]


def _rows_of(state, pool, scales, page, row):
    dtype = TYPES[state["case"]["type"]]
    bits = pool.view(torch.int8)[page, row].view(pool.dtype)
    return (bits.float() * scales.transpose(1, 2)[page, row][..., None]).to(dtype)


def _rotated(state, x):
    case = state["case"]
    angle = state["positions"].double()[:, None, None] * state["frequencies"]                   # in 64 bits: far positions turn often
    c, s = torch.cos(angle).float(), torch.sin(angle).float()
    r, x = case["rotary"], x.float()
    if case["layout"] == "half":
        a, b = x[..., :r // 2], x[..., r // 2:r]
        return torch.cat([a * c - b * s, b * c + a * s, x[..., r:]], -1)
    a, b = x[..., 0:r:2], x[..., 1:r:2]
    return torch.cat([torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2), x[..., r:]], -1)


def _write(state):
    page, row = _at(state)
    codes = state["case"]["codes"]
    out = dict(q=_rotated(state, state["q"]).to(state["q"].dtype))
    for name, x in (("k", _rotated(state, state["k"])), ("v", state["v"])):
        c, s = _coded(x, codes)
        state[name + "pages"].view(torch.int8)[page, row] = c.view(torch.int8)
        state[name + "scales"].transpose(1, 2)[page, row] = s[..., 0]
        out[name] = _rows_of(state, state[name + "pages"], state[name + "scales"], page, row)
    return out


def _read(state):
    size, lengths = state["case"]["page"], state["lengths"].long()
    ends = torch.cumsum(lengths, 0)
    rows = torch.arange(state["tokens"], device=ends.device)
    b = torch.searchsorted(ends, rows, right=True)
    t = rows - (ends - lengths)[b]
    page, row = state["table"].long()[b, t // size], t % size
    out = {name: _rows_of(state, state[name + "pages"], state[name + "scales"], page, row) for name in ("k", "v")}
    return dict(out, starts=torch.cat([torch.zeros_like(ends[:1]), ends]).int())


def _attention(s, seen, v):
    """Scores [b, h, g, t] of tokens that are `seen` [b, t], values [b, t, h, d]: outputs [b, h, g, d] and the log of the weights' sums."""
    s = s.masked_fill(~seen[:, None, None], -math.inf)
    m = s.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)                      # (a row without tokens: exp(-inf) everywhere)
    w = torch.exp(s - m)
    total = w.sum(-1, keepdim=True)
    out = torch.einsum("bhgt,bthd->bhgd", w, v) / total.clamp(min=torch.finfo(torch.float32).tiny)
    return out, torch.where(total > 0, m + torch.log(total), -math.inf)[..., 0]


def _attend(state):
    case, q, lengths = state["case"], state["q"], state["lengths"]
    n, hq, dim = q.shape
    hkv, table = case["kv_heads"], state["table"].long().clamp(min=0)

    def tokens(name):
        codes = state[name + "pages"].view(torch.int8)[table].view(state[name + "pages"].dtype)  # [requests, pages, tokens, kv heads, dim]
        return (codes.float() * state[name + "scales"][table].transpose(2, 3)[..., None]).flatten(1, 2)

    s = torch.einsum("bhgd,bthd->bhgt", q.view(n, hkv, hq // hkv, dim).float(), tokens("k")) * state["scaling"]
    at = torch.arange(s.shape[-1], device=q.device)
    seen = at < lengths[:, None]
    if case["window"]:
        seen &= at >= lengths[:, None] - case["window"]
    out, lse = _attention(s, seen, tokens("v"))
    return dict(out=out.view(n, hq, dim).to(q.dtype), lse=lse.view(n, hq))


def _shared(state):
    """Each group's prefix once for all its members (they are the rows of one product), the members' own tokens one by one, and both joined."""
    case, q, table, lengths = state["case"], state["q"], state["table"].long().clamp(min=0), state["lengths"]
    n, hq, dim = q.shape
    hkv, g, members = case["kv_heads"], hq // case["kv_heads"], state["followers"]
    rows = state["starts"].long()[members].flatten()                                            # rows of q, group by group
    x = q[rows].view(*members.shape, hkv, g, dim).float()

    def part(x, requests, count):                                                               # x [b, h, rows, d] over the first count[b] tokens of requests[b]
        k, v = (state[name][table[requests]].flatten(1, 2).float() for name in ("kpages", "vpages"))
        s = torch.einsum("bhgd,bthd->bhgt", x, k) * state["scaling"]
        return _attention(s, torch.arange(s.shape[-1], device=q.device) < count[:, None], v)

    a, la = part(x.transpose(1, 2).flatten(2, 3), state["holders"], lengths[state["holders"]])
    a, la = (y.unflatten(2, (members.shape[1], g)).transpose(1, 2).flatten(0, 1) for y in (a, la))
    b, lb = part(x.flatten(0, 1), members.flatten(), lengths[members.flatten()])
    lse = torch.logaddexp(la, lb)
    y = a * torch.exp(la - lse)[..., None] + b * torch.exp(lb - lse)[..., None]
    out, all_lse = torch.empty_like(q), torch.empty(n, hq, device=q.device)
    out[rows] = y.reshape(n, hq, dim).to(q.dtype)
    all_lse[rows] = lse.reshape(n, hq)
    return dict(out=out, lse=all_lse)


PLAIN = dict(write=_write, read=_read, attend=_attend, shared=_shared)


# ---- what a pass cannot do without -----------------------------------------------------------------

def work(case):
    op, dim, hkv = case["op"], case["dim"], case["kv_heads"]
    row = 2 * hkv * (dim + 4)                                       # a token's codes and scales, keys and values
    if op == "write":
        heads = case["heads"] + hkv
        return dict(bytes=case["tokens"] * (2 * 2 * case["heads"] * dim + 2 * 2 * hkv * dim + row + 2 * 2 * hkv * dim + 8) + 4 * case["rotary"],
                    flops=case["tokens"] * (3 * heads * case["rotary"] + 6 * hkv * dim))
    if op == "shared":
        prefixes, mine = _lengths(case)
        rows, token = len(mine), 2 * hkv * dim * 2
        pages = int(_pages_of(prefixes, case["page"]).sum() + _pages_of(mine, case["page"]).sum())
        return dict(bytes=int(prefixes.sum() + mine.sum()) * token + 4 * pages + rows * (20 + case["heads"] * (4 * dim + 4)),
                    flops=4 * case["heads"] * dim * (case["members"] * int(prefixes.sum()) + int(mine.sum())))
    lengths = _lengths(case)
    if op == "read":
        total = int(lengths.sum())
        return dict(bytes=total * (row + 2 * 2 * hkv * dim) + 4 * int(_pages_of(lengths, case["page"]).sum()) + 8 * case["requests"], flops=2 * total * hkv * dim)
    counted = np.minimum(lengths, case["window"]) if case["window"] else lengths
    return dict(bytes=int(counted.sum()) * row + 4 * int(_pages_of(counted, case["page"]).sum()) + case["requests"] * (4 + case["heads"] * (4 * dim + 4)),
                flops=4 * int(counted.sum()) * case["heads"] * dim)


# ---- the values in 64 bits -------------------------------------------------------------------------

def _turned(case, x, positions, f):
    """The rotation as a product of complex numbers."""
    r = case["rotary"]
    z = torch.exp(1j * positions.double()[:, None, None] * f)
    y = x.double().clone()
    if case["layout"] == "half":
        w = torch.complex(y[..., :r // 2], y[..., r // 2:r]) * z
        y[..., :r // 2], y[..., r // 2:r] = w.real, w.imag
    else:
        w = torch.view_as_complex(y[..., :r].unflatten(-1, (r // 2, 2)).contiguous()) * z
        y[..., :r] = torch.view_as_real(w).flatten(-2)
    return y


def _held(x, codes):
    """What codes and scale of a row stand for.  (The scale is a number of 32 bits by definition.)"""
    top = x.abs().amax(-1, keepdim=True)
    if codes == "int8":
        s = torch.maximum((top / 127).float().double(), torch.full_like(top, LEAST))
        return s * torch.clamp(torch.round(x / s), -127, 127)
    m, e = torch.frexp(top)                                          # top = m 2^e with m in [1/2, 1): 448 = 7/8 2^9
    s = torch.where(top > 0, _power(torch.clamp(e - 9 + (m > 0.875).int(), min=-100)), LEAST)
    t = x / s
    step = _power(torch.clamp(torch.frexp(t)[1] - 4, min=-9))                                    # four significant bits, the least step 2^-9
    return s * step * torch.round(t / step)


def exact(case, seed):
    op = case["op"]
    state = prepare(case, seed)
    if op == "write":
        q, k = (_turned(case, state[name], state["positions"], state["frequencies"]) for name in ("q", "k"))
        return dict(q=q, k=_held(k, case["codes"]), v=_held(state["v"].double(), case["codes"]))
    lengths, size = state["lengths"].tolist(), case["page"]

    def token_rows(name, b, t, h=slice(None)):                       # tokens t of request b: [tokens, heads, dim] or of one head [tokens, dim]
        page, row = state["table"][b].long()[t // size], t % size
        x = state[name + "pages"]
        if x.dtype in (torch.float16, torch.bfloat16):
            return x[page, row][:, h].double()
        values = x.view(torch.int8)[page, row].view(x.dtype)[:, h].double()
        return values * state[name + "scales"][page, :, row][:, h].double()[..., None]

    if op == "read":
        out = {name: torch.cat([token_rows(name, b, torch.arange(n, device="cuda")) for b, n in enumerate(lengths)]) for name in ("k", "v")}
        return dict(out, starts=None)
    hkv, group = case["kv_heads"], case["heads"] // case["kv_heads"]
    out = torch.zeros(state["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.full(state["q"].shape[:2], -math.inf, dtype=torch.float64, device="cuda")
    if op == "shared":
        starts, parents = state["starts"].tolist(), state["parents"].tolist()
        for holder in state["holders"].tolist():
            before = torch.arange(lengths[holder], device="cuda")
            for h in range(hkv):
                kp, vp = (token_rows(name, holder, before, h) for name in ("k", "v"))
                for b in (b for b, parent in enumerate(parents) if parent == holder):
                    mine, at, of = torch.arange(lengths[b], device="cuda"), starts[b], slice(h * group, (h + 1) * group)
                    x = state["q"][at, of].double()
                    s = state["scaling"] * torch.cat([x @ kp.T, x @ token_rows("k", b, mine, h).T], -1)
                    w = torch.softmax(s, -1)
                    lse[at, of] = torch.logsumexp(s, -1)
                    out[at, of] = w[:, :len(before)] @ vp + w[:, len(before):] @ token_rows("v", b, mine, h)
        return dict(out=out, lse=lse)
    for b, n in enumerate(lengths):
        first = max(0, n - case["window"]) if case["window"] else 0
        if n <= first:
            continue
        t = torch.arange(first, n, device="cuda")
        for h in range(hkv):
            of = slice(h * group, (h + 1) * group)
            s = state["scaling"] * (state["q"][b, of].double() @ token_rows("k", b, t, h).T)
            lse[b, of] = torch.logsumexp(s, -1)
            out[b, of] = torch.softmax(s, -1) @ token_rows("v", b, t, h)
    return dict(out=out, lse=lse)
