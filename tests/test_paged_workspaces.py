"""Which workspace PagedKVCache.attend takes: one for each stream and for each capture (CPU, nothing is launched)."""
import copy

import pytest
import torch

from kvcomp_b200 import _lib, ops
from kvcomp_b200.cache import PagedKVCache


class Calls:
    """The calls for torch, on a stream and in a capture that the test says."""
    at = (0, 0)
    used = None

    def stream_of(self, device):
        return self.at

    def paged_attn(self, *args):
        self.used = next(a for a in args if isinstance(a, str) and a.startswith("workspace"))


@pytest.fixture
def attend(monkeypatch):
    calls, made = Calls(), []
    monkeypatch.setattr(_lib, "torch_calls", lambda: calls)
    monkeypatch.setattr(ops, "paged_attn_workspace", lambda *a: made.append(a) or "workspace %d" % len(made))
    cache = object.__new__(PagedKVCache)
    vars(cache).update(requests=3, kv_heads=2, head_dim=64, device=torch.device("cuda", 0), keys=[None], values=[None], table=None, lengths=None, plan=None, window=0,
                       status=None, _workspaces={})

    def attend(stream=0, capture=0, heads=4, cache=cache):
        calls.at = (stream, capture)
        cache.attend(torch.zeros(3, heads, 64), 0)
        return calls.used
    attend.cache = cache
    return attend


def test_a_capture_keeps_its_own(attend):
    """The zeros of a workspace that is made in a capture are only recorded: nothing outside that graph may use it."""
    inside = attend(7, 1)
    assert attend(7, 1) == inside
    assert attend(0) != inside and attend(7) != inside
    assert attend(7, 2) not in (inside, attend(0), attend(7))


def test_streams_keep_their_own(attend):
    first, second = attend(0), attend(5)
    assert first != second and (attend(0), attend(5)) == (first, second)
    assert attend(0, heads=8) not in (first, second)


def test_captures_that_are_over_are_dropped(attend):
    eager = attend(7)
    for capture in range(1, 20):
        attend(7, capture), attend(7, capture, heads=8)
    assert len(attend.cache._workspaces) == 3 and attend(7) == eager
    attend(8, 19)
    assert attend(7, 19) == attend(7, 19) and len(attend.cache._workspaces) == 4


def test_copies_make_their_own(attend):
    mine = attend(0)
    other = copy.copy(attend.cache)
    assert attend(0, cache=other) != mine and attend(0) == mine


def test_states_of_older_caches(attend):
    """One that was pickled with its workspaces, under the name that they had."""
    state = dict(vars(attend.cache), _workspace={4: "workspace of another process"})
    del state["_workspaces"]
    other = object.__new__(PagedKVCache)
    other.__setstate__(state)
    assert attend(0, cache=other) == "workspace 1"
