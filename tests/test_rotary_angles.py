"""The table of rotary positions' frequencies against whole numbers of any length."""
import pytest

import rotary_exactly as exact


@pytest.mark.parametrize("sign", [1, -1])
def test_table_is_rounded(hip, sign):
    """Half of 2^-64 turns for the rounding, and 2^-64 of up to 0.16 turns for the division in 64 bits."""
    f = [sign * 10 ** (-9 * i / 96) for i in range(97)]
    got = [v % 2 ** 64 for v in hip.Rotary(194, frequencies=f, device="cpu").turns.tolist()]
    for v, frequency in zip(got, f):
        off = abs(v - exact.turns(1, frequency) * 2 ** 64) % 2 ** 64
        assert min(off, 2 ** 64 - off) <= 0.67


def test_entries_at_the_ends_of_a_turn(hip):
    """Next below a whole number of turns: rounded up, that is none."""
    got = hip.Rotary(4, frequencies=[-2.0 ** -70, 2.0 ** -70], device="cpu").turns.tolist()
    assert got == [0, 0]
