"""Frequencies scaled by the trained length: which pairs keep theirs and which are
divided, whatever the length is, against the statement itself (CPU only)."""
import math

import pytest

from aethelstream_amd import rotary

FACTOR = 4.0


def _parts(rot, base, trained, fast=32.0, slow=1.0):
    """Plain and scaled frequencies, and each pair's turns within the trained length."""
    f, _ = rotary.frequencies(rot, base=base)
    g, _ = rotary.frequencies(rot, base=base, factor=FACTOR, trained=trained, fast=fast, slow=slow)
    return f, g, [trained * v / (2 * math.pi) for v in f]


@pytest.mark.parametrize("rot,base", [(128, 1e4), (64, 1e4), (128, 5e5), (40, 100.0), (2, 1e4)])
@pytest.mark.parametrize("trained", [1, 5, 6, 64, 200, 202, 4096, 8192, 65536, 131072, 1 << 20,
                                     1 << 24])
@pytest.mark.parametrize("fast,slow", [(32.0, 1.0), (8.0, 0.25)])
def test_fast_pairs_keep_theirs_and_slow_ones_are_divided(rot, base, trained, fast, slow):
    f, g, turns = _parts(rot, base, trained, fast, slow)
    # (Turns within 1e-9 of a limit may count on either side of it.)
    for a, b, n in zip(f, g, turns):
        if n >= fast * (1 + 1e-9):
            assert b == a
        elif n <= slow * (1 - 1e-9):
            assert b == pytest.approx(a / FACTOR, rel=1e-12)
        else:
            assert a / FACTOR * (1 - 1e-12) <= b <= a * (1 + 1e-12)


@pytest.mark.parametrize("trained", [5, 64, 8192, 65536, 131072, 1 << 20])
def test_the_ramp_is_linear_in_the_index(trained):
    """The share of the division grows by the same amount from pair to pair, also where
    the ramp begins before the first pair or ends behind the last."""
    rot, base = 128, 1e4
    f, g, turns = _parts(rot, base, trained)
    share = [(1 - b / a) / (1 - 1 / FACTOR) for a, b in zip(f, g)]

    def index(n):
        return rot * math.log(trained / (n * 2 * math.pi)) / (2 * math.log(base))

    first, last = math.floor(index(32.0)), math.ceil(index(1.0))
    for i, s in enumerate(share):
        assert s == pytest.approx(min(max((i - first) / (last - first), 0.0), 1.0), abs=1e-12)


def test_a_last_pair_that_turns_more_than_once():
    """The head's slowest pair turns 1.2 and 2.4 times in these lengths: it is slowed by
    less than the factor."""
    for trained, turns in ((65536, 1.204), (131072, 2.409)):
        f, g, n = _parts(128, 1e4, trained)
        assert n[-1] == pytest.approx(turns, abs=1e-3)
        assert g[-1] > f[-1] / FACTOR * 1.1


def test_a_first_pair_that_turns_less_than_once():
    f, g, n = _parts(128, 1e4, 5)
    assert n[0] < 1 and g == [v / FACTOR for v in f]


def test_limits_next_to_each_other():
    slow = 8192 / (2 * math.pi)  # what the first pair turns
    f, g, _ = _parts(128, 1e4, 8192, fast=slow * (1 + 2.0 ** -52), slow=slow)
    assert g[2:] == [v / FACTOR for v in f[2:]]
