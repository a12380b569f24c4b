"""The frequencies of a rotary table's pairs, on the host."""
import math

import pytest

from torchpairwise_b200 import attention_ops


@pytest.fixture
def frequencies(monkeypatch):
    monkeypatch.setattr(attention_ops, "_table", lambda f, length, magnitude: f.tolist())
    return lambda features, **how: attention_ops.rotary_table(1, features, device="cpu", **how)


@pytest.mark.parametrize("features", [2, 8, 64, 128])
@pytest.mark.parametrize("original", [1, 4, 6, 7, 100, 4096, 1 << 20])
@pytest.mark.parametrize("fast,slow", [(32.0, 1.0), (2.0, 1.5)])
def test_bands(frequencies, features, original, fast, slow):
    """Pairs of more than `fast` turns over the original length keep their frequency, those of fewer than `slow` turns are divided, the others lie
    between, and no faster pair is divided more than a slower one."""
    factor = 16.0
    plain = frequencies(features)
    got = frequencies(features, scaling="bands", factor=factor, original_length=original, fast_turns=fast, slow_turns=slow)
    ratios = [a / b for a, b in zip(plain, got)]
    # the band's ends are whole indexes, so the pairs beside it may share in it
    step = 10000.0 ** (2 / features)
    for f, r in zip(plain, ratios):
        turns = original * f / (2 * math.pi)
        assert 1 - 1e-12 <= r <= factor * (1 + 1e-12)
        if turns > fast * step:
            assert r == pytest.approx(1.0)
        if turns < slow / step or turns <= slow and f == plain[0]:
            assert r == pytest.approx(factor), (turns, r)
    assert all(a <= b * (1 + 1e-12) for a, b in zip(ratios, ratios[1:]))
