"""Where the attention's partial results lie: every place starts on 16 bytes, whatever the heads (CPU)."""
import pytest

from kvcomp_b200 import _lib


@pytest.mark.parametrize("D", [64, 96, 128, 256])
def test_places_lie_on_16_bytes(D):
    lib = _lib.load()

    def results(group):
        return lib.kvc_paged_attn_workspace(4, group, 1, D) - lib.kvc_paged_attn_cleared()
    most = 8 if D == 256 else 16                                # query heads that a column serves
    values, rest = divmod(results(most), 4 * most * (D + 2))   # of `most` heads a place has no room to spare
    assert rest == 0 and values > 0 and lib.kvc_paged_attn_cleared() % 16 == 0
    for group in range(1, most + 1):
        place, rest = divmod(results(group), values)
        assert rest == 0 and place % 16 == 0 and place >= 4 * group * (D + 2), group
