"""Results and pools whose rows overlap are refused before anything is launched (CPU: only calls that are refused)."""
import pytest

from kvcomp_b200 import _lib
from test_packed_arguments import _header_fields
from test_paged_arguments import STRUCTS, good

N, HQ, HKV, D, PAGES, PAGE = 4, 8, 2, 128, 10, 16
MB = 1 << 20


def rotary(**change):
    """Everything apart: each tensor contiguous, in a megabyte of its own."""
    values = dict(good("kvc_rotary_store"), q=1 * MB, q_out=2 * MB, k=3 * MB, v=4 * MB, kpages=5 * MB, vpages=6 * MB, N=N, Hq=HQ, Hkv=HKV, D=D, n_pages=PAGES, page_size=PAGE,
                  q_token=HQ * D, q_head=D, out_token=HQ * D, out_head=D, k_token=HKV * D, k_head=D, v_token=HKV * D, v_head=D,
                  kp_page=PAGE * HKV * D, kp_row=HKV * D, kp_head=D, vp_page=PAGE * HKV * D, vp_row=HKV * D, vp_head=D)
    return dict(values, **change)


def attn(**change):
    values = dict(good("kvc_paged_attn"), q=1 * MB, out=2 * MB, kpages=5 * MB, vpages=6 * MB, workspace=16 * MB, B=N, Hq=HQ, Hkv=HKV, D=D, n_pages=PAGES, page_size=PAGE,
                  q_token=HQ * D, q_head=D, out_token=HQ * D, out_head=D,
                  kp_page=PAGE * HKV * D, kp_row=HKV * D, kp_head=D, vp_page=PAGE * HKV * D, vp_row=HKV * D, vp_head=D)
    return dict(values, **change)


def refused(call, values):
    struct, packer = STRUCTS[call]
    assert getattr(_lib.load(), call)(getattr(_lib, packer).pack(*(values[name] for name, _ in _header_fields(struct))), None) == 1
    assert b"overlap" in _lib.load().kvc_last_error()


TOKENS = HQ * D * 2 * N                                     # bytes of the queries
OUTPUTS = [dict(out_token=0), dict(out_head=0), dict(out_head=D - 8), dict(out_token=HQ * D - 8), dict(out_token=D, out_head=D),       # rows of the output among one another
           dict(at=2 * D), dict(at=-2 * D), dict(at=TOKENS - 2 * D), dict(at=16), dict(at=-TOKENS + 2 * D),                            # beside the queries by a head, by a piece
           dict(at=0, out_token=D, out_head=N * D), dict(at=0, q_token=0)]                                                            # in another order; a query for all tokens


@pytest.mark.parametrize("change", OUTPUTS, ids=str)
def test_outputs(change):
    change = dict(change)
    at = change.pop("at", None)
    refused("kvc_rotary_store", rotary(**change, **({} if at is None else dict(q_out=1 * MB + at))))
    refused("kvc_paged_attn", attn(**change, **({} if at is None else dict(out=1 * MB + at))))


@pytest.mark.parametrize("change", [dict(kp_page=0), dict(vp_page=0), dict(kp_row=0), dict(vp_head=0), dict(kp_row=D), dict(vp_page=PAGE * HKV * D - 8), dict(vpages=5 * MB),
                                    dict(vpages=5 * MB + 2 * D), dict(vpages=5 * MB + 2 * PAGE * HKV * D * (PAGES - 1)), dict(q_out=3 * MB, Hq=HKV, out_token=HKV * D),
                                    dict(q_out=4 * MB + 2 * D), dict(q_out=4 * MB - TOKENS + 16)], ids=str)
def test_pools_and_keys(change):
    refused("kvc_rotary_store", rotary(**change))


def test_one_pool_for_both():
    """Keys and values to one pool: only where they are the same and nothing is rotated."""
    refused("kvc_rotary_store", rotary(vpages=5 * MB, v=3 * MB))
    refused("kvc_rotary_store", rotary(vpages=5 * MB, rotary=0))
