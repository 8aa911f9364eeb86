"""The error bounds that burn_dragon_amd.activations states, held to the definition
of the 8-bit values (tests/trainref.py)."""
import re

import numpy as np
import pytest

from burn_dragon_amd import activations
from tests import trainref as R


def _stated():
    """The docstring's (share of a value, share of its block's largest, least step's half)."""
    text = " ".join(activations.__doc__.split())
    share = re.search(r"off by at most 2\^(-\d+) of its magnitude", text).group(1)
    top = re.search(r"by 2\^(-\d+) of its block's largest", text).group(1)
    least = re.search(r"by 2\^(-\d+) in a block", text)
    return 2.0 ** int(share), 2.0 ** int(top), 2.0 ** int(least.group(1)) if least else 0.0


def _blocks(top):
    """Blocks with the largest magnitude `top`: values of all sizes below it, and those
    half a step from their neighbours."""
    g = np.random.default_rng(5)
    x = top * np.exp2(-24 * g.random((64, 32))) * np.where(g.random((64, 32)) < 0.5, -1, 1)
    e = np.frexp(top)[1] + np.arange(-24, 1)[:, None] - 1
    ties = np.ldexp((2 * (np.arange(31) % 16) + 17) / 16.0, e)       # between two of e4m3's
    ties = np.where(ties < top, ties, 0.0)
    x = np.concatenate([x[:, 1:], ties, -ties]).astype(np.float32).astype(float)
    return np.concatenate([np.full((len(x), 1), top), x], 1)


@pytest.mark.parametrize("top", [448.0, 224.0 * (1 + 2.0 ** -20), 3.5 * 2.0 ** 90, 3.5001, 0.01, 2.0 ** -100])
def test_values_are_as_close_as_stated(top):
    top = float(np.float32(top))
    x = _blocks(top)
    share, of_top, least = _stated()
    off = np.abs(R.in8(x)[0] - x)
    assert (off <= np.maximum(share * np.abs(x), max(of_top * top, least))).all()


def test_blocks_of_the_least_power():
    share, of_top, least = _stated()
    for top in (2.0 ** -109, 2.0 ** -118, 2.0 ** -126, 2.0 ** -140):
        x = _blocks(top)
        off = np.abs(R.in8(x)[0] - x)
        assert (off <= np.maximum(share * np.abs(x), max(of_top * top, least))).all()
