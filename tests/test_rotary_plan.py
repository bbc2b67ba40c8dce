"""What a RotaryPlan makes of its arguments; nothing here reaches a GPU."""
import math

import pytest
import torch


@pytest.fixture(scope="module")
def A():
    import __graft_entry__
    __graft_entry__.build()
    import aethelstream_b200
    return aethelstream_b200


def by_index(dim, base, factor, length, fast, slow):
    """Pairs mixed linearly in their index between those that turn `fast` and `slow`
    times in `length` positions."""
    def pair(turns):
        return dim * math.log(length / (turns * math.tau)) / (2 * math.log(base))

    low, high = max(math.floor(pair(fast)), 0), min(math.ceil(pair(slow)), dim // 2 - 1)
    out = []
    for p in range(dim // 2):
        f = base ** (-2 * p / dim)
        keep = 1 - min(max((p - low) / (high - low), 0.0), 1.0)
        out.append(f * keep + f / factor * (1 - keep))
    return out


def test_the_two_mixtures_of_yarn(A):
    """The plan's is linear in the turns; the other one is taken as numbers."""
    d, base, factor, length = 128, 10000.0, 16.0, 4096
    plan = A.RotaryPlan(d, base=base, scaling="yarn", factor=factor, original_length=length)
    other = by_index(d, base, factor, length, 32.0, 1.0)
    between = 0
    for p, (f, g) in enumerate(zip(plan.inv_freq, other)):
        own = base ** (-2 * p / d)
        turns = length * own / math.tau
        keep = min(max((turns - 1.0) / 31.0, 0.0), 1.0)
        assert f == pytest.approx(own * keep + own / factor * (1 - keep), rel=1e-14)
        if turns >= 32.0 or turns <= 0.9:
            assert f == pytest.approx(g, rel=0.1)
        between += abs(f - g) > 0.2 * f
    assert between > 5  # not small where they differ
    given = A.RotaryPlan(d, inv_freq=other, amplitude=plan.amplitude)
    assert given.inv_freq == tuple(other) and given.amplitude == plan.amplitude == pytest.approx(0.1 * math.log(factor) + 1)
    for f, t in zip(other, given.freq.tolist()):
        assert (t % 2 ** 64) / 2.0 ** 64 == pytest.approx(f / math.tau, rel=1e-15, abs=2.0 ** -64)
    assert given.freq.dtype == torch.int64
