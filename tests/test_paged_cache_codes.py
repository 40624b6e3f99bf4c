"""PagedKVCache in codes that there are not (CPU)."""
import types

import pytest
import torch

from kvcomp_b200 import _lib
from kvcomp_b200.cache import PagedKVCache


@pytest.mark.parametrize("codes", ["int4", "fp8", 8, True])
def test_refused(codes):
    with pytest.raises(_lib.KvcError, match="codes"):
        PagedKVCache(2, 4, 1, 2, 64, codes=codes)


def test_the_first_follow_is_not_captured(monkeypatch):
    """What says whether it would be is the stream of the cache's device, not of the current one."""
    asked = []
    monkeypatch.setattr(_lib, "torch_calls", lambda: types.SimpleNamespace(stream_of=lambda device: asked.append(device) or (0, 7)))
    cache = PagedKVCache.__new__(PagedKVCache)
    cache.__setstate__(dict(requests=2, window=0, codes=None, head_dim=64, device=torch.device("cpu"), lengths=torch.zeros(2, dtype=torch.int32)))
    with pytest.raises(_lib.KvcError, match="must not be captured"):
        cache.follow(torch.tensor([-1, 0], dtype=torch.int32))
    assert asked == [None] and cache.prefixes is None and cache.parents is None
