"""utils.rotary.frequencies of configurations as models hold them: YaRN pair by pair, lengths beside the dict, fields that are not known (CPU)."""
import math

import pytest
import torch

from kvcomp_b200.utils.rotary import frequencies


def yarn(r, base, s, L, beta_fast=32.0, beta_slow=1.0, truncate=True):
    """The formula, written out for each pair."""
    def pair(turns):
        return r / 2 * math.log(L / (2 * math.pi * turns)) / math.log(base)
    low, high = pair(beta_fast), pair(beta_slow)
    if truncate:
        low, high = float(math.floor(low)), float(math.ceil(high))
    low, high = max(low, 0.0), min(high, r - 1.0)
    got = []
    for i in range(r // 2):
        x = base ** (-2 * i / r)
        stretched = min(max((i - low) / (high - low), 0.0), 1.0)
        got.append(x * (1 - stretched) + x / s * stretched)
    return got


@pytest.mark.parametrize("truncate", [True, False, None])
@pytest.mark.parametrize("r,base,s,L", [(64, 150000.0, 32.0, 4096), (128, 10000.0, 16.0, 4096), (64, 1e6, 4.0, 32768)])
def test_yarn_pair_by_pair(r, base, s, L, truncate):
    scaling = {"rope_type": "yarn", "factor": s, "original_max_position_embeddings": L, "beta_fast": 32.0, "beta_slow": 1.0}
    if truncate is not None:
        scaling["truncate"] = truncate
    f, factor = frequencies(r, base, scaling)
    torch.testing.assert_close(f, torch.tensor(yarn(r, base, s, L, truncate=truncate is not False), dtype=torch.float64), rtol=1e-13, atol=0)
    assert abs(factor - (0.1 * math.log(s) + 1)) < 1e-15


@pytest.mark.parametrize("mscale,all_dim,want", [(1.0, 1.0, 1.0), (0.707, 0.707, 1.0), (1.0, 0.5, (0.1 * math.log(40) + 1) / (0.05 * math.log(40) + 1)), (1.0, None, 0.1 * math.log(40) + 1),
                                                 (None, None, 0.1 * math.log(40) + 1), (1.0, 0.0, 0.1 * math.log(40) + 1)])
def test_yarn_factor_of_two_terms(mscale, all_dim, want):
    scaling = {"type": "yarn", "factor": 40, "original_max_position_embeddings": 4096, "beta_fast": 32, "beta_slow": 1, "mscale": mscale, "mscale_all_dim": all_dim}
    assert abs(frequencies(64, 10000.0, scaling)[1] - want) < 1e-15
    assert frequencies(64, 10000.0, dict(scaling, attention_factor=1.5))[1] == 1.5
    assert frequencies(64, 10000.0, dict(scaling, factor=1.0))[1] == 1.0


@pytest.mark.parametrize("mscale,all_dim", [(0.707, None), (None, 1.0), (0.5, 0.0)])
def test_yarn_terms_go_together(mscale, all_dim):
    with pytest.raises(ValueError):
        frequencies(64, 10000.0, {"rope_type": "yarn", "factor": 40, "original_max_position_embeddings": 4096, "mscale": mscale, "mscale_all_dim": all_dim})


def test_fields_that_are_not_known():
    for scaling in ({"rope_type": "linear", "factor": 2.0, "mrope_section": [16, 24, 24]}, {"rope_type": "dynamic", "factor": 2.0, "alpha": 1000.0, "original_max_position_embeddings": 4096}):
        with pytest.raises(ValueError, match="mrope_section|alpha"):
            frequencies(64, 10000.0, scaling)
    assert torch.equal(frequencies(64, 10000.0, {"rope_type": "linear", "factor": 2.0, "alpha": None, "finetuned": True, "partial_rotary_factor": 0.5})[0],
                       frequencies(64, 10000.0, {"rope_type": "linear", "factor": 2.0})[0])


def test_base_of_the_configuration():
    plain = frequencies(64, 500000.0)[0]
    assert torch.equal(frequencies(64, scaling={"rope_type": "default", "rope_theta": 500000.0})[0], plain)
    assert torch.equal(frequencies(64, 500000, {"rope_type": "default", "rope_theta": 500000.0})[0], plain)
    assert torch.equal(frequencies(64)[0], frequencies(64, 10000.0)[0])
    with pytest.raises(ValueError):
        frequencies(64, 10000.0, {"rope_type": "default", "rope_theta": 500000.0})


def test_lengths_beside_the_dict():
    """A configuration that holds them itself: the same as in the dict."""
    short, long = [1.0 + 0.01 * i for i in range(32)], [1.0 + 0.5 * i for i in range(32)]
    inside = {"type": "longrope", "short_factor": short, "long_factor": long, "original_max_position_embeddings": 4096, "max_position_embeddings": 131072}
    beside = {"type": "longrope", "short_factor": short, "long_factor": long}
    for length in (4096, 4097):
        f, factor = frequencies(64, 10000.0, beside, length, original_max_position_embeddings=4096, max_position_embeddings=131072)
        want, want_factor = frequencies(64, 10000.0, inside, length)
        assert torch.equal(f, want) and factor == want_factor == math.sqrt(1 + math.log(32) / math.log(4096))
    with pytest.raises(ValueError):                                # (how far the context was stretched is not said)
        frequencies(64, 10000.0, beside, original_max_position_embeddings=4096)
    assert frequencies(64, 10000.0, dict(beside, factor=32.0), original_max_position_embeddings=4096)[1] == math.sqrt(1 + math.log(32) / math.log(4096))
    for length in (100, 9000):
        f = frequencies(64, 10000.0, {"rope_type": "dynamic", "factor": 2.0}, length, max_position_embeddings=2048)[0]
        assert torch.equal(f, frequencies(64, 10000.0, {"rope_type": "dynamic", "factor": 2.0, "original_max_position_embeddings": 2048}, length)[0])
    with pytest.raises(ValueError):
        frequencies(64, 10000.0, {"rope_type": "dynamic", "factor": 2.0})
