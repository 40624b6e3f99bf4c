"""PagedKVCache in codes that there are not (CPU)."""
import pytest

from kvcomp_b200 import _lib
from kvcomp_b200.cache import PagedKVCache


@pytest.mark.parametrize("codes", ["int4", "fp8", 8, True])
def test_refused(codes):
    with pytest.raises(_lib.KvcError, match="codes"):
        PagedKVCache(2, 4, 1, 2, 64, codes=codes)
