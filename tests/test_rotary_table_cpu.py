"""The ladder of frequencies of stretched contexts, from its definition in turns."""
import math

import pytest

import dtb200


def _ladder(rotary, **kw):
    t = dtb200.make_rotary_table(rotary, device="cpu", **kw)
    return [x * 2 * math.pi for x in t.turns.tolist()]


def _slowed(n, base, factor, original, fast=32.0, slow=1.0):
    """By how much each pair is slowed: its place on the ramp between the pairs of `fast` and of `slow` turns, rounded outwards."""
    place = {t: n * math.log(original / (t * 2 * math.pi)) / math.log(base) for t in (fast, slow)}
    low, high = max(math.floor(place[fast]), 0), math.ceil(place[slow])
    return [1 / (1 + (1 / factor - 1) * min(max((j - low) / (high - low), 0.0), 1.0)) for j in range(n)]


@pytest.mark.parametrize("n, base, original, factor", [(32, 1e4, 4096, 4.0), (64, 1e4, 65536, 4.0), (64, 1e4, 131072, 4.0), (32, 1e4, 1 << 20, 8.0),
                                                       (64, 5e5, 8192, 8.0), (16, 100.0, 2048, 2.0), (64, 1e4, 100, 4.0), (1, 1e4, 8192, 2.0)])
def test_yarn(n, base, original, factor):
    got = _ladder(2 * n, base=base, scaling="yarn", factor=factor, original_length=original)
    want = _slowed(n, base, factor, original)
    for j in range(n):
        assert abs(base ** (-j / n) / got[j] - want[j]) <= 1e-12 * want[j], (j, base ** (-j / n) / got[j], want[j])


def test_yarn_slows_a_pair_by_its_turns():
    """Figures worked out by hand for the slowest of 64 pairs: 1.20 turns over 65536 positions, 2.41 over 131072."""
    for original, turns, slowed in ((65536, 1.20, 3.23), (131072, 2.41, 2.17)):
        slowest = 1e4 ** (-63 / 64)
        assert abs(original * slowest / (2 * math.pi) - turns) < 0.01
        assert abs(slowest / _ladder(128, scaling="yarn", factor=4.0, original_length=original)[-1] - slowed) < 0.01


def test_yarn_slows_all_pairs_where_none_makes_a_turn():
    got = _ladder(16, scaling="yarn", factor=4.0, original_length=5)
    assert all(abs(1e4 ** (-j / 8) / x - 4.0) < 1e-12 for j, x in enumerate(got))
