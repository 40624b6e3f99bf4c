"""utils.rotary.frequencies against the formulas, pair by pair (CPU)."""
import math

import pytest
import torch

from kvcomp_b200.utils.rotary import frequencies

R, BASE, L = 64, 500000.0, 8192


def plain():
    return [BASE ** (-2 * i / R) for i in range(R // 2)]


def close(got, want):
    assert got.dtype == torch.float64
    torch.testing.assert_close(got, torch.tensor(want, dtype=torch.float64), rtol=1e-14, atol=0)


def test_plain_and_linear():
    f, factor = frequencies(R, BASE)
    close(f, plain())
    assert factor == 1.0
    close(frequencies(R, BASE, {"rope_type": "linear", "factor": 4.0})[0], [x / 4 for x in plain()])
    close(frequencies(R, BASE, {"type": "default"})[0], plain())
    assert frequencies(0)[0].numel() == 0


def test_ntk_stretches_the_slowest_pair_by_the_factor():
    f, _ = frequencies(R, BASE, {"rope_type": "ntk", "factor": 8.0})
    assert f[0] == 1.0
    assert abs(f[-1].item() / (plain()[-1] / 8.0) - 1) < 1e-12


def test_dynamic_depends_on_the_length():
    scaling = {"rope_type": "dynamic", "factor": 2.0, "original_max_position_embeddings": L}
    for length in (None, 100, L):
        close(frequencies(R, BASE, scaling, length=length)[0], plain())
    grow = 2.0 * 3 - 1.0
    close(frequencies(R, BASE, scaling, length=3 * L)[0], [(BASE * grow ** (R / (R - 2))) ** (-2 * i / R) for i in range(R // 2)])


def test_yarn():
    f, factor = frequencies(R, BASE, {"rope_type": "yarn", "factor": 16.0, "original_max_position_embeddings": L})
    assert abs(factor - (0.1 * math.log(16.0) + 1)) < 1e-15
    for i, (got, x) in enumerate(zip(f.tolist(), plain())):
        turns = L * x / (2 * math.pi)
        if turns > 40:
            assert got == x
        if turns < 0.8:
            assert abs(got - x / 16) <= 1e-15 * x
        assert x / 16 * (1 - 1e-12) <= got <= x
    assert all(a > b for a, b in zip(f.tolist(), f.tolist()[1:]))
    assert frequencies(R, BASE, {"rope_type": "yarn", "factor": 16.0, "original_max_position_embeddings": L, "attention_factor": 1.25})[1] == 1.25


def test_llama3():
    scaling = {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0, "original_max_position_embeddings": L}
    want = []
    for x in plain():
        wave = 2 * math.pi / x
        if wave < L / 4.0:
            want.append(x)
        elif wave > L / 1.0:
            want.append(x / 8.0)
        else:
            smooth = (L / wave - 1.0) / (4.0 - 1.0)
            want.append((1 - smooth) * x / 8.0 + smooth * x)
    close(frequencies(R, BASE, scaling)[0], want)


def test_longrope():
    short, long = [1.0 + 0.01 * i for i in range(R // 2)], [1.0 + 0.5 * i for i in range(R // 2)]
    scaling = {"rope_type": "longrope", "short_factor": short, "long_factor": long, "original_max_position_embeddings": 4096, "max_position_embeddings": 131072}
    f, factor = frequencies(R, 10000.0, scaling, length=4096)
    close(f, [10000.0 ** (-2 * i / R) / s for i, s in enumerate(short)])
    assert abs(factor - math.sqrt(1 + math.log(32) / math.log(4096))) < 1e-15
    close(frequencies(R, 10000.0, scaling, length=4097)[0], [10000.0 ** (-2 * i / R) / s for i, s in enumerate(long)])


def test_refusals():
    for args in ((63,), (-2,), (R, BASE, {"rope_type": "spiral"}), (R, BASE, {"rope_type": "yarn", "factor": 2.0}),
                 (R, BASE, {"rope_type": "longrope", "short_factor": [1.0], "long_factor": [1.0], "original_max_position_embeddings": L})):
        with pytest.raises(ValueError):
            frequencies(*args)
