"""Calls of the operators on a paged cache that are refused before anything is launched."""
import pytest

from test_attention import attend


@pytest.mark.parametrize("strides", [dict(ot=64, oh=128), dict(ot=512), dict(qt=512), dict(qh=128, qt=512)], ids=str)
def test_out_in_the_memory_of_q_in_another_order(hip, strides):
    assert attend(hip, **strides) == hip.E_INVALID_ARG
    assert b"other strides" in hip.lib.sarek_hip_last_error()


def test_strides_that_are_not_used_may_differ(hip):
    """No token: nothing is launched, and nothing is wrong with one token of one head either way."""
    assert attend(hip, tokens=0, starts=1 << 20, qt=512) == 0
    assert attend(hip, tokens=1, batch=1, q_heads=2, qt=512, held=-1) == hip.E_WORKSPACE
