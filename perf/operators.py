"""Operators of a paged key-value cache: what is measured of them, their plain forms, and their values in 64 bits.

    plan      pages for the tokens that a step brings, and where each token goes      (ops.page_plan)
    release   the pages of finished requests go back to the free list                (ops.page_release)
    store     queries and keys rotated, keys and values written to their slots       (ops.rotary_paged_store)
    rotate    keys moved to other positions, or back to none                         (ops.rotary)
    attend    one new token per request over the pages                               (ops.paged_attn)
"""
import math

import numpy as np
import torch

own = False

TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


# ---- the cases -------------------------------------------------------------------------------------

def listed():
    return [
        # a decode step of a small batch: every request gets one token, latency is all that counts
        dict(name="plan step", op="plan", requests=16, new=1, held=4096, page=64, short=False),
        # prompts of many requests are admitted at once behind short prefixes
        dict(name="plan prompts", op="plan", requests=256, new=512, held=300, page=16, short=False),
        # some requests of a batch have ended
        dict(name="release few", op="release", requests=32, held=2048, page=64, done=0.25),
        # a large batch of long requests is dropped
        dict(name="release many", op="release", requests=1024, held=16384, page=32, done=0.5),
        # a decode step of one layer, Llama-2-7B's heads, batch 8
        dict(name="store step", op="store", tokens=8, heads=32, kv_heads=32, dim=128, rotary=128, layout="half", type="fp16", held=4096, page=64, scaled=False),
        # prompts of one layer, Phi-3-medium's heads in bf16, part of the head rotated, frequencies stretched for long contexts, slices of one projection
        dict(name="store prompts", op="store", tokens=16384, heads=40, kv_heads=10, dim=128, rotary=96, layout="half", type="bf16", held=16384, page=128, scaled=True),
        # cached keys are turned back before they move to other positions; interleaved pairs, an odd number of tokens
        dict(name="rotate back", op="rotate", tokens=32749, heads=8, dim=128, rotary=128, layout="interleaved", type="fp16", held=131072, scaled=False, inverse=True),
        # the first answer to one short request, Llama-2-7B's heads
        dict(name="attend one short", op="attend", requests=1, heads=32, kv_heads=32, dim=128, type="fp16", longest=777, ragged=False, page=16, window=0),
        # Llama-2-7B's heads, batch 8, 4096 tokens
        dict(name="attend 8 x 4096", op="attend", requests=8, heads=32, kv_heads=32, dim=128, type="fp16", longest=4096, ragged=False, page=64, window=0),
        # Mistral-7B's grouped heads, batch 16, 32768 tokens
        dict(name="attend 16 x 32768", op="attend", requests=16, heads=32, kv_heads=8, dim=128, type="fp16", longest=32768, ragged=False, page=64, window=0),
        # a serving batch: lengths of every size, some requests idle, Phi-3-medium's heads in bf16, a sliding window
        dict(name="attend ragged window", op="attend", requests=64, heads=40, kv_heads=10, dim=128, type="bf16", longest=16384, ragged=True, page=128, window=4096),
        # one long document, few key-value heads: the length has to be split
        dict(name="attend one long", op="attend", requests=1, heads=32, kv_heads=8, dim=128, type="bf16", longest=131072, ragged=False, page=256, window=0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["plan", "release", "store", "store", "rotate", "attend", "attend", "attend"])
    page = rng.choice([8, 16, 24, 32, 64, 128, 256])
    kind = rng.choice(["fp16", "bf16"])
    if op == "plan":
        requests = _log(rng, 1, 4096)
        new = 1 if rng.random() < 0.4 else _log(rng, 1, max(1, 131072 // requests))
        return dict(op=op, requests=requests, new=new, held=_log(rng, 1, min(32768, 4000000 // requests)), page=page, short=rng.random() < 0.3)
    if op == "release":
        requests = _log(rng, 1, 4096)
        return dict(op=op, requests=requests, held=_log(rng, 1, min(32768, 16000000 // requests)), page=page, done=rng.choice([0.1, 0.5, 1.0]))
    dim = rng.choice([64, 96, 128, 128, 256])
    kv_heads, group = rng.choice([(32, 1), (8, 4), (10, 4), (4, 8), (1, 16), (2, 7), (5, 3), (12, 1)])
    layout, rotary = rng.choice(["half", "interleaved"]), rng.choice([dim, dim, dim // 2, dim // 4])
    if op == "store":
        tokens = _log(rng, 1, max(16, 16384 * 60 * 128 // (kv_heads * (group + 2) * dim)))
        return dict(op=op, tokens=tokens, heads=kv_heads * group, kv_heads=kv_heads, dim=dim, rotary=rotary, layout=layout, type=kind,
                    held=_log(rng, 1, 1000000), page=page, scaled=rng.random() < 0.5)
    if op == "rotate":
        return dict(op=op, tokens=_log(rng, 1, 33000000 // (kv_heads * dim)), heads=kv_heads, dim=dim, rotary=rotary, layout=layout, type=kind,
                    held=_log(rng, 1, 1000000), scaled=rng.random() < 0.5, inverse=rng.random() < 0.5)
    requests = _log(rng, 1, 256)
    longest = _log(rng, 1, max(1, min(131072, 500000000 // (requests * kv_heads * dim))))
    return dict(op=op, requests=requests, heads=kv_heads * group, kv_heads=kv_heads, dim=dim, type=kind, longest=longest, ragged=rng.random() < 0.6,
                page=page, window=rng.choice([0, 0, _log(rng, 1, 8192)]))


# ---- what a user's program has in hand -------------------------------------------------------------

def _lengths(case):
    """The requests' lengths, in no order: the same numbers whatever the seed."""
    n, top = case["requests"], case.get("longest") or case["held"]
    if "longest" in case and not case["ragged"]:
        return np.full(n, top, dtype=np.int64)
    r = np.random.RandomState(1 + n + 7919 * top)
    got = np.floor(top * r.random_sample(n) ** 2).astype(np.int64) + (r.random_sample(n) < 0.9)      # many short ones, a few idle, one of full length
    got[0] = top
    return np.minimum(got, top)


def _new(case):
    """How many tokens each request brings."""
    n, most = case["requests"], case["new"]
    if most == 1:
        return np.ones(n, dtype=np.int64)
    return np.random.RandomState(3 + n + 104729 * most).randint(0, 2 * most, n).astype(np.int64)


def _pages_of(lengths, page):
    return (lengths + page - 1) // page


def _need(case):
    held, new = _lengths(case), _new(case)
    return _pages_of(held + new, case["page"]) - _pages_of(held, case["page"])


def _frequencies(case):
    """fp64 angles per position and the factor on cos and sin: base 10000, and with `scaled` the long-context form that stretches slow pairs eightfold,
    leaves fast ones and goes over linearly between 32 turns and one turn in 4096 positions."""
    r = case["rotary"]
    f = 10000.0 ** (-np.arange(0, r, 2, dtype=np.float64) / r)
    if not case["scaled"]:
        return f, 1.0
    turns = 4096 * f / (2 * math.pi)
    keep = np.clip((turns - 1.0) / (32.0 - 1.0), 0.0, 1.0)
    return f * keep + f / 8.0 * (1.0 - keep), 0.1 * math.log(8.0) + 1.0


def _table(order, lengths, page, width):
    """Block table rows of requests whose pages come one after the other from `order`; behind a row's pages -1."""
    need = _pages_of(lengths, page)
    first = np.cumsum(need) - need
    at = np.arange(width)[None, :]
    table = np.where(at < need[:, None], order[np.minimum(first[:, None] + at, len(order) - 1)], -1)
    return table.astype(np.int32)


def _gpu(a, dtype=None):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda() if dtype is None else torch.from_numpy(np.ascontiguousarray(a)).to(dtype).cuda()


def prepare(case, seed):
    rng = np.random.RandomState(seed % (1 << 31))
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    op = case["op"]
    state = dict(case=case)
    if op in ("plan", "release"):
        order, page = rng.permutation(case["requests"]), case["page"]
        lengths = _lengths(case)[order]
        held = int(_pages_of(lengths, page).sum())
        if op == "plan":
            new, need = _new(case)[order], int(_need(case).sum())
            pool = held + (need // 2 if case["short"] else need + 5)
            width = int(_pages_of(lengths + new, page).max()) + 3
            state.update(new=_gpu(new, torch.int32), tokens=int(new.sum()))
        else:
            pool, width = held + 100, int(_pages_of(lengths, page).max()) + 1
            done = np.zeros(len(lengths), dtype=bool)
            done[rng.permutation(len(lengths))[:max(1, int(case["done"] * len(lengths)))]] = True
            state.update(done=_gpu(done))
        order = rng.permutation(pool)
        state.update(lengths=_gpu(lengths, torch.int32), table=_gpu(_table(order, lengths, page, width)), free=_gpu(order, torch.int32),
                     head=_gpu(np.array([held]), torch.int32))
        return state
    dtype, dim = TYPES[case["type"]], case["dim"]

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda", dtype=dtype)

    if op in ("store", "rotate"):
        tokens = case["tokens"]
        f, factor = _frequencies(case)
        top = max(case["held"], 1)
        state.update(frequencies=_gpu(f), factor=factor, positions=_gpu(rng.randint(0, top, tokens), torch.int32))
        if op == "rotate":
            state.update(x=normal(tokens, case["heads"], dim))
            return state
        hq, hkv, page = case["heads"], case["kv_heads"], case["page"]
        qkv = normal(tokens, hq + 2 * hkv, dim)                     # one projection's output: its slices have rows that lie apart
        pages = -(-tokens // page) + 2
        state.update(q=qkv[:, :hq], k=qkv[:, hq:hq + hkv], v=qkv[:, hq + hkv:], slots=_gpu(rng.permutation(pages * page)[:tokens], torch.int32),
                     kpages=normal(pages, page, hkv, dim), vpages=normal(pages, page, hkv, dim))
        return state
    lengths, page, hkv = rng.permutation(_lengths(case)), case["page"], case["kv_heads"]
    pool = int(_pages_of(lengths, page).sum()) + 2
    width = max(1, int(_pages_of(lengths, page).max()))
    kpages = normal(pool, page, hkv, dim)
    kpages.mul_(torch.exp(0.5 * torch.randn(hkv, dim, generator=gen, device="cuda")).to(dtype))      # channels of different size
    state.update(q=normal(case["requests"], case["heads"], dim), kpages=kpages, vpages=normal(pool, page, hkv, dim),
                 table=_gpu(_table(rng.permutation(pool), lengths, page, width)), lengths=_gpu(lengths, torch.int32), scaling=1.0 / math.sqrt(dim))
    if own:                                                         # what the program's cache keeps for all its steps
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
    if case["op"] == "plan":
        p = ops.page_plan(state["lengths"], state["new"], state["table"], state["free"], state["head"], case["page"], state["tokens"])
        return dict(lengths=p.lengths, head=p.head, starts=p.starts, slots=p.slots, positions=p.positions, table=state["table"])
    if case["op"] == "release":
        lengths, head = ops.page_release(state["lengths"], state["done"], state["table"], state["free"], state["head"], case["page"])
        return dict(lengths=lengths, head=head, free=state["free"])
    if case["op"] == "store":
        q = ops.rotary_paged_store(state["q"], state["k"], state["v"], state["positions"], state["slots"], state["frequencies"], state["kpages"],
                                   state["vpages"], layout=case["layout"], factor=state["factor"])
        return dict(q=q, kpages=state["kpages"], vpages=state["vpages"])
    if case["op"] == "rotate":
        return ops.rotary(state["x"], state["positions"], state["frequencies"], layout=case["layout"], factor=state["factor"], inverse=case["inverse"])
    out, lse = ops.paged_attn(state["q"], state["kpages"], state["vpages"], state["table"], state["lengths"], state["scaling"], window=case["window"],
                              return_lse=True, workspace=state["workspace"])
    return dict(out=out, lse=lse)


def _plan(state):
    page, table, free, tokens = state["case"]["page"], state["table"], state["free"], state["tokens"]
    held, new, head = state["lengths"].long(), state["new"].long(), state["head"].long()
    owned, total = (held + page - 1) // page, (held + new + page - 1) // page
    fits = total <= table.shape[1]
    need = (total - owned) * fits
    upto = torch.cumsum(need, 0)
    served = fits & ((need == 0) | (head + upto <= free.numel()))
    ends = torch.cumsum(new, 0)
    rows = torch.arange(tokens, device=held.device)
    r = torch.searchsorted(ends, rows, right=True)
    position = held[r] + rows - (ends - new)[r]
    p = position // page
    taken = head + (upto - need)[r] + p - owned[r]
    fresh = (p >= owned[r]) & served[r]
    number = torch.where(fresh, free[taken.clamp(0, free.numel() - 1)], table[r, p.clamp(0, table.shape[1] - 1)])
    table[r[fresh], p[fresh]] = number[fresh]
    slots = torch.where(served[r], number.long() * page + position % page, -1)
    starts = torch.cat([torch.zeros_like(ends[:1]), ends])
    return dict(lengths=(held + new * served).int(), head=(head + (need * served).sum()).int(), starts=starts.int(), slots=slots.int(),
                positions=position.int(), table=table)


def _release(state):
    page, table, free, done = state["case"]["page"], state["table"], state["free"], state["done"]
    held, head = state["lengths"].long(), state["head"].long()
    back = (held + page - 1) // page * done
    ends = torch.cumsum(back, 0)
    at = torch.arange(table.shape[1], device=held.device)
    freed = at < back[:, None]
    to = (head - ends[-1]) + (ends - back)[:, None] + at
    free[to[freed]] = table[freed]
    return dict(lengths=(held * ~done).int(), head=(head - ends[-1]).int(), free=free)


def _rotated(state, x, inverse=False):
    case = state["case"]
    angle = state["positions"].double()[:, None, None] * state["frequencies"]                   # in 64 bits: far positions turn often
    c, s = (state["factor"] * torch.cos(angle)).float(), (state["factor"] * torch.sin(angle)).float()
    s = -s if inverse else s
    r, x = case["rotary"], x.float()
    if case["layout"] == "half":
        a, b = x[..., :r // 2], x[..., r // 2:r]
        y = torch.cat([a * c - b * s, b * c + a * s, x[..., r:]], -1)
    else:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        y = torch.cat([torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2), x[..., r:]], -1)
    return y.to(TYPES[case["type"]])


def _store(state):
    kpages, vpages, slots = state["kpages"], state["vpages"], state["slots"].long()
    kpages.view(-1, *kpages.shape[2:])[slots] = _rotated(state, state["k"])
    vpages.view(-1, *vpages.shape[2:])[slots] = state["v"]
    return dict(q=_rotated(state, state["q"]), kpages=kpages, vpages=vpages)


def _rotate(state):
    return _rotated(state, state["x"], state["case"]["inverse"])


def _attend(state):
    case, q, lengths = state["case"], state["q"], state["lengths"]
    n, hq, dim = q.shape
    hkv, table = case["kv_heads"], state["table"].long().clamp(min=0)
    k = state["kpages"][table].flatten(1, 2).float()                                            # [requests, tokens, kv heads, dim]
    s = torch.einsum("bhgd,bthd->bhgt", q.view(n, hkv, hq // hkv, dim).float(), k) * state["scaling"]
    del k
    at = torch.arange(s.shape[-1], device=q.device)
    seen = at < lengths[:, None]
    if case["window"]:
        seen &= at >= lengths[:, None] - case["window"]
    s = s.masked_fill(~seen[:, None, None], -math.inf)
    m = s.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)                      # (a row without tokens: exp(-inf) everywhere)
    w = torch.exp(s - m)
    total = w.sum(-1, keepdim=True)
    v = state["vpages"][table].flatten(1, 2).float()
    out = torch.einsum("bhgt,bthd->bhgd", w, v) / total.clamp(min=torch.finfo(torch.float32).tiny)
    lse = torch.where(total > 0, m + torch.log(total), -math.inf)
    return dict(out=out.view(n, hq, dim).to(q.dtype), lse=lse.view(n, hq))


PLAIN = dict(plan=_plan, release=_release, store=_store, rotate=_rotate, attend=_attend)


# ---- what a pass cannot do without -----------------------------------------------------------------

def work(case):
    op = case["op"]
    if op == "plan":
        need, tokens = int(_need(case).sum()), int(_new(case).sum())
        return dict(bytes=16 * case["requests"] + 8 * tokens + 8 * need + 8, flops=0)
    if op == "release":
        back = int(case["done"] * _pages_of(_lengths(case), case["page"]).sum())
        return dict(bytes=9 * case["requests"] + 8 * back + 8, flops=0)
    size = 2 * case["dim"]
    if op == "store":
        heads = case["heads"] + 2 * case["kv_heads"]
        return dict(bytes=case["tokens"] * (2 * heads * size + 8) + 4 * case["rotary"],
                    flops=3 * case["tokens"] * (case["heads"] + case["kv_heads"]) * case["rotary"])
    if op == "rotate":
        return dict(bytes=case["tokens"] * (2 * case["heads"] * size + 4) + 4 * case["rotary"], flops=3 * case["tokens"] * case["heads"] * case["rotary"])
    lengths = _lengths(case)
    seen = int((np.minimum(lengths, case["window"]) if case["window"] else lengths).sum())
    pages = int(_pages_of(np.minimum(lengths, case["window"]) if case["window"] else lengths, case["page"]).sum())
    return dict(bytes=2 * seen * case["kv_heads"] * size + 4 * pages + case["requests"] * (4 + case["heads"] * (2 * size + 4)),
                flops=4 * seen * case["heads"] * case["dim"])


# ---- the values in 64 bits -------------------------------------------------------------------------

def _turned(case, x, positions, f, factor, inverse):
    """The rotation as a product of complex numbers."""
    r = case["rotary"]
    z = torch.polar(torch.full_like(f, factor)[None].expand(len(positions), -1).contiguous(), positions.double()[:, None] * f[None])[:, None]
    z = z.conj() if inverse else z
    y = x.double().clone()
    if case["layout"] == "half":
        w = torch.complex(y[..., :r // 2], y[..., r // 2:r]) * z
        y[..., :r // 2], y[..., r // 2:r] = w.real, w.imag
    else:
        w = torch.view_as_complex(y[..., :r].unflatten(-1, (r // 2, 2)).contiguous()) * z
        y[..., :r] = torch.view_as_real(w).flatten(-2)
    return y


def exact(case, seed):
    op = case["op"]
    if op in ("plan", "release"):                                    # whole numbers
        return None
    state = prepare(case, seed)
    if op == "rotate":
        return _turned(case, state["x"], state["positions"], state["frequencies"], state["factor"], case["inverse"])
    if op == "store":
        pages = {}
        for name, rows in (("k", _turned(case, state["k"], state["positions"], state["frequencies"], state["factor"], False)), ("v", state["v"].double())):
            old = state[name + "pages"]
            pages[name] = old.double()
            at = state["slots"].long()
            pages[name][at // case["page"], at % case["page"]] = rows
        return dict(q=_turned(case, state["q"], state["positions"], state["frequencies"], state["factor"], False), kpages=pages["k"], vpages=pages["v"])
    lengths, group = state["lengths"].tolist(), case["heads"] // case["kv_heads"]
    out = torch.zeros(state["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.full(state["q"].shape[:2], -math.inf, dtype=torch.float64, device="cuda")
    for b, n in enumerate(lengths):
        first = max(0, n - case["window"]) if case["window"] else 0
        if n <= first:
            continue
        t = torch.arange(first, n, device="cuda")
        page, row = state["table"][b].long()[t // case["page"]], t % case["page"]
        for h in range(case["kv_heads"]):
            of = slice(h * group, (h + 1) * group)
            s = state["scaling"] * (state["q"][b, of].double() @ state["kpages"][page, row, h].double().T)
            lse[b, of] = torch.logsumexp(s, -1)
            out[b, of] = torch.softmax(s, -1) @ state["vpages"][page, row, h].double()
    return dict(out=out, lse=lse)
