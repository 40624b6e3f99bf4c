"""Calls with prefixes: the packed arguments have the header's layout, and what cannot be done is refused before anything is launched (CPU)."""
import pytest
import torch

from kvcomp_b200 import _lib, ops
from test_packed_arguments import _header_fields
from test_paged_arguments import good, letters

AT = 1 << 20


def test_layout():
    assert "".join(letter for _, letter in _header_fields("kvc_prefix_plan_args")) == letters(_lib.PREFIX_PLAN_ARGS)


def plan(**change):
    values = dict(parents=AT, shared=AT, B=4, plan=AT, status=0, **{})
    values.update(change)
    return _lib.load().kvc_prefix_plan(_lib.PREFIX_PLAN_ARGS.pack(*(values[n] for n, _ in _header_fields("kvc_prefix_plan_args"))), None)


@pytest.mark.parametrize("change", [dict(parents=0), dict(shared=0), dict(plan=0), dict(plan=AT + 4), dict(B=-1), dict(B=16385)], ids=str)
def test_plan_refusals(change):
    assert plan(**change) == 1 and b"kvc_prefix_plan" in _lib.load().kvc_last_error()


def attn(plan=AT, starts=None, rows=0, **change):
    values = dict(good("kvc_paged_attn"), out=2 * AT, **{})
    values.update(change)
    return _lib.load().kvc_paged_attn_shared(_lib.PAGED_ATTN_ARGS.pack(*(values[n] for n, _ in _header_fields("kvc_paged_attn_args"))), plan, starts, rows, None)


@pytest.mark.parametrize("change", [dict(plan=None), dict(plan=AT + 4), dict(q=0), dict(kpages=0), dict(vpages=0), dict(table=0), dict(lengths=0), dict(out=0), dict(workspace=0), dict(D=256), dict(D=112),
                                    dict(Hq=7), dict(Hkv=0), dict(B=-1), dict(B=16385), dict(window=5), dict(window=-1), dict(type=2), dict(q=AT + 8), dict(kpages=AT + 2), dict(kp_row=132), dict(out_head=4),
                                    dict(page_size=0), dict(table_width=1 << 28), dict(workspace=AT + 16), dict(n_pages=-1), dict(out_token=64, out_head=64), dict(starts=AT, rows=-1),
                                    dict(B=16384, Hkv=64, Hq=64, table_width=1 << 16, page_size=1 << 10)], ids=str)
def test_refusals(change):
    assert attn(**change) == 1 and b"kvc_paged_attn_shared" in _lib.load().kvc_last_error()


@pytest.mark.parametrize("change", [dict(kp_head=1 << 31), dict(vp_head=1 << 31), dict(kp_head=1 << 32), dict(kp_row=1 << 28), dict(vp_row=1 << 28), dict(page_size=1 << 20, kp_row=1 << 12, kp_head=128),
                                    dict(page_size=1 << 20, vp_row=1 << 12, vp_head=128), dict(kp_row=1 << 62), dict(vp_head=1 << 62), dict(kp_row=-256), dict(vp_row=-256), dict(kp_head=-128), dict(vp_head=-128),
                                    dict(kp_page=-4096), dict(vp_page=-4096)], ids=str)
@pytest.mark.parametrize("call", ["kvc_paged_attn_shared", "kvc_paged_attn", "kvc_paged_attn_rows"])
def test_pages_that_reach_too_far(call, change):
    """A row's place in its page is a number of 32 bits, for the requests' own tokens as in calls without prefixes."""
    values = dict(good("kvc_paged_attn"), out=2 * AT, **change)
    packed, lib = _lib.PAGED_ATTN_ARGS.pack(*(values[n] for n, _ in _header_fields("kvc_paged_attn_args"))), _lib.load()
    rc = lib.kvc_paged_attn_shared(packed, AT, None, 0, None) if call.endswith("shared") else lib.kvc_paged_attn(packed, None) if call == "kvc_paged_attn" else lib.kvc_paged_attn_rows(packed, AT, 4, None)
    why = lib.kvc_last_error().decode()
    assert rc == 1 and why.startswith(call.replace("_rows", "") + ":") and ("more than 2^31 elements" in why or "negative stride" in why), why      # (where there is no device a launch is refused, too)


def test_workspaces_and_nothing_to_do():
    lib = _lib.load()
    need = lib.kvc_paged_attn_shared_workspace(4, 8, 2, 128)
    assert attn(workspace_bytes=need - 1) == 3
    assert attn(B=0) == 0 and attn(starts=AT, rows=0) == 0
    assert lib.kvc_prefix_plan(None, None) == 1 and lib.kvc_paged_attn_shared(None, AT, None, 0, None) == 1
    assert lib.kvc_paged_attn_shared_workspace(-1, 8, 2, 128) == 0 and lib.kvc_prefix_plan_words(-1) == 0
    assert need > lib.kvc_paged_attn_cleared() and lib.kvc_prefix_plan_words(0) > 0
    for B in (1, 3, 100):                                           # more requests or heads never need less
        assert lib.kvc_paged_attn_shared_workspace(B, 8, 2, 128) <= lib.kvc_paged_attn_shared_workspace(B + 1, 8, 2, 128) <= lib.kvc_paged_attn_shared_workspace(B + 1, 16, 2, 128)


def test_no_cpu_path():
    i, x, pool = torch.zeros(2, dtype=torch.int32), torch.zeros(2, 2, 64, dtype=torch.float16), torch.zeros(4, 16, 2, 64, dtype=torch.float16)
    some = ops.PrefixPlan(torch.zeros(22, dtype=torch.int32), 2)
    for call in (lambda: ops.prefix_plan(i, i), lambda: ops.paged_attn_shared(x, pool, pool, i[None], i, some, 1.0), lambda: ops.paged_attn_shared(x, pool, pool, i[None], i, i, 1.0),
                 lambda: ops.paged_attn_shared_workspace(1, 1, 1, 64, "cpu")):
        with pytest.raises(_lib.KvcError):
            call()
