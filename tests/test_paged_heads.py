"""PagedKVCache of heads that its attention does not take is refused where it is made (CPU)."""
import pytest

from kvcomp_b200 import _lib, ops
from kvcomp_b200.cache import PagedKVCache
from test_packed_arguments import _header_fields
from test_paged_arguments import good


@pytest.mark.parametrize("head_dim", [32, 80, 112, 192, 512])
def test_refused(head_dim):
    with pytest.raises(_lib.KvcError, match="channels"):
        PagedKVCache(2, 4, 1, 2, head_dim)


def test_the_library_says_the_same():
    """Rows: 0: what is checked, and nothing to launch."""
    lib, fields = _lib.load(), _header_fields("kvc_paged_attn_args")
    for D in range(1, 600):
        values = dict(good("kvc_paged_attn"), D=D)
        assert (lib.kvc_paged_attn_rows(_lib.PAGED_ATTN_ARGS.pack(*(values[n] for n, _ in fields)), 1 << 20, 0, None) == 0) == (D in ops.PAGED_HEADS)
