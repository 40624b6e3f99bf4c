"""kvc_paged_attn_rows: what cannot be done is an error code before anything is launched (CPU)."""
import pytest

from kvcomp_b200 import _lib
from test_packed_arguments import _header_fields
from test_paged_arguments import BAD, good


def call(starts, rows, **change):
    values = dict(good("kvc_paged_attn"), **change)
    return _lib.load().kvc_paged_attn_rows(_lib.PAGED_ATTN_ARGS.pack(*(values[n] for n, _ in _header_fields("kvc_paged_attn_args"))), starts, rows, None)


@pytest.mark.parametrize("change", BAD["kvc_paged_attn"], ids=str)
def test_refusals(change):
    assert call(1 << 20, 3, **change) == 1
    assert b"kvc_paged_attn" in _lib.load().kvc_last_error()


def test_rows():
    assert call(None, 3) == 1 and call(1 << 20, -1) == 1 and call(1 << 20, 1 << 24) == 1 and call(1 << 20, 3, B=0) == 1
    assert call(1 << 20, 0) == 0 and call(1 << 20, 0, B=0) == 0
    assert _lib.load().kvc_paged_attn_rows(None, 1 << 20, 1, None) == 1
