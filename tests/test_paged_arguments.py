"""The paged cache's calls: the packed arguments have the header's layout, and what cannot be done is an error code before anything is launched (CPU)."""
import ctypes as C

import pytest
import torch

from kvcomp_b200 import _lib, ops
from test_packed_arguments import _header_fields

STRUCTS = {"kvc_page_plan": ("kvc_page_plan_args", "PAGE_PLAN_ARGS"), "kvc_page_release": ("kvc_page_release_args", "PAGE_RELEASE_ARGS"),
           "kvc_rotary_store": ("kvc_rotary_args", "ROTARY_ARGS"), "kvc_paged_attn": ("kvc_paged_attn_args", "PAGED_ATTN_ARGS")}


def letters(packer):
    import re
    return re.sub(r"(\d+)(\w)", lambda m: int(m.group(1)) * m.group(2), packer.format.lstrip("<"))


@pytest.mark.parametrize("call", sorted(STRUCTS))
def test_layouts(call):
    struct, packer = STRUCTS[call]
    fields, packer = _header_fields(struct), getattr(_lib, packer)
    assert "".join(letter for _, letter in fields) == letters(packer)

    class Args(C.Structure):
        _fields_ = [(name, {"q": C.c_int64, "i": C.c_int32, "f": C.c_float}[letter]) for name, letter in fields]
    assert C.sizeof(Args) == packer.size


def good(call):
    """Arguments that the checks accept: pointers are never followed by them."""
    at = 1 << 20
    if call == "kvc_page_plan":
        return dict(lengths=at, new_tokens=at, free_pages=at, head=at, table=at, table_stride=8, table_width=8, B=4, n_pages=100, page_size=16, tokens=10,
                    lengths_out=at, head_out=at, starts=at, taken=at, slots=at, positions=at, status=0)
    if call == "kvc_page_release":
        return dict(lengths=at, done=at, table=at, table_stride=8, table_width=8, free_pages=at, head=at, B=4, n_pages=100, page_size=16, lengths_out=at, head_out=at,
                    first=at, status=0)
    if call == "kvc_rotary_store":
        d = dict(q=at, k=at, v=at, q_out=at, kpages=at, vpages=at, positions=at, slots=at, frequencies=at, N=4, Hq=8, Hkv=2, D=128, rotary=64, n_pages=10, page_size=16,
                 status=0, layout=0, inverse=0, type=0, factor=1.0)
    else:
        d = dict(q=at, kpages=at, vpages=at, table=at, lengths=at, out=at, lse=0, workspace=at, workspace_bytes=1 << 40, B=4, Hq=8, Hkv=2, D=128, n_pages=10,
                 page_size=16, table_stride=8, table_width=8, window=0, status=0, scaling=0.1, type=0)
    for name, _ in _header_fields(STRUCTS[call][0]):
        d.setdefault(name, 128)
    return d


BAD = {
    "kvc_page_plan": [dict(lengths=0), dict(head=0), dict(slots=0), dict(table=0), dict(free_pages=0), dict(page_size=0), dict(page_size=-1), dict(B=-1), dict(tokens=-1),
                      dict(tokens=1 << 31), dict(n_pages=1 << 28), dict(n_pages=-1), dict(table_stride=7), dict(page_size=1 << 21), dict(starts=0), dict(taken=0)],
    "kvc_page_release": [dict(lengths=0), dict(done=0), dict(first=0), dict(head_out=0), dict(table=0), dict(page_size=0), dict(n_pages=1 << 28), dict(table_stride=1), dict(B=-1)],
    "kvc_rotary_store": [dict(q=0), dict(k=0), dict(v=0), dict(q_out=0), dict(kpages=0), dict(slots=0), dict(positions=0), dict(frequencies=0), dict(rotary=63), dict(rotary=130),
                         dict(rotary=-2), dict(D=0), dict(N=-1), dict(Hq=-1), dict(Hkv=-1), dict(type=2), dict(layout=2), dict(page_size=0), dict(n_pages=1 << 28), dict(N=1 << 31)],
    "kvc_paged_attn": [dict(q=0), dict(kpages=0), dict(vpages=0), dict(table=0), dict(lengths=0), dict(out=0), dict(workspace=0), dict(D=112), dict(Hq=7), dict(Hkv=0), dict(B=-1),
                       dict(window=-1), dict(type=2), dict(q=(1 << 20) + 8), dict(kpages=(1 << 20) + 2), dict(kp_row=132), dict(out_head=4), dict(page_size=0),
                       dict(table_width=1 << 28), dict(workspace=(1 << 20) + 8), dict(n_pages=-1)],
}


@pytest.mark.parametrize("call,change", [(c, d) for c in sorted(BAD) for d in BAD[c]], ids=str)
def test_refusals(call, change):
    lib = _lib.load()
    struct, packer = STRUCTS[call]
    values = dict(good(call), **change)
    assert getattr(lib, call)(getattr(_lib, packer).pack(*(values[name] for name, _ in _header_fields(struct))), None) == 1
    assert call.encode() in lib.kvc_last_error()


def test_workspace_too_small_and_null():
    lib = _lib.load()
    need = lib.kvc_paged_attn_workspace(4, 8, 2, 128)
    values = dict(good("kvc_paged_attn"), workspace_bytes=need - 1)
    assert lib.kvc_paged_attn(_lib.PAGED_ATTN_ARGS.pack(*(values[n] for n, _ in _header_fields("kvc_paged_attn_args"))), None) == 3
    for call in STRUCTS:
        assert getattr(lib, call)(None, None) == 1


def test_nothing_to_do():
    """Calls without requests or tokens return without a launch (there is no device here)."""
    lib = _lib.load()
    for call, change in (("kvc_paged_attn", dict(B=0)), ("kvc_rotary_store", dict(N=0)), ("kvc_rotary_store", dict(Hq=0, Hkv=0))):
        values = dict(good(call), **change)
        assert getattr(lib, call)(getattr(_lib, STRUCTS[call][1]).pack(*(values[n] for n, _ in _header_fields(STRUCTS[call][0]))), None) == 0


def test_no_cpu_path():
    i, x = torch.zeros(2, dtype=torch.int32), torch.zeros(2, 2, 64, dtype=torch.float16)
    pool = torch.zeros(4, 16, 2, 64, dtype=torch.float16)
    for call in (lambda: ops.page_plan(i, i, i[None], i, i[:1], 16, 2), lambda: ops.page_release(i, i > 0, i[None], i, i[:1], 16),
                 lambda: ops.rotary(x, i, None), lambda: ops.rotary_paged_store(None, x, x, i, i, None, pool, pool),
                 lambda: ops.paged_attn(x, pool, pool, i[None], i, 1.0)):
        with pytest.raises(_lib.KvcError):
            call()
