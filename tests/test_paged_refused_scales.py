"""Scales and caps with which a score of 0 would be NaN are refused, without a GPU (as tests/test_paged_refusals.py)."""
import pytest

from test_paged_refusals import ARG, accepted, attn, bits, prefix


@pytest.mark.parametrize("change", [dict(scale=bits(float("inf"))), dict(scale=bits(float("-inf"))), dict(scale=bits(3e38)), dict(softcap=bits(float("inf"))),
                                    dict(softcap=bits(3e38)), dict(softcap=bits(1e-45)), dict(scale=bits(1e30), softcap=bits(1e-20))])
def test_refused(change):
    assert attn(**change) == ARG and prefix(**change) == ARG


@pytest.mark.parametrize("change", [dict(scale=0), dict(scale=bits(1e30)), dict(scale=bits(-1e-30)), dict(softcap=bits(1e-30)), dict(softcap=bits(1e30))])
def test_accepted(change):
    assert accepted(attn(**change)) and accepted(prefix(**change))
