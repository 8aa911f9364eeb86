"""bdh_sample_tokens' refusals and the sampling oracle, on the CPU: argument
checks run before any device call."""
import ctypes
import math

import numpy as np
import pytest

from burn_dragon_amd import _lib
from tests import sampleref

GOOD = 0x10000


def call(logits=GOOD, dtype=_lib.BDH_F32, rows=2, vocab=8, stride=8, uniform=GOOD, tokens=GOOD, logprob=None,
         options=None):
    return _lib.load().bdh_sample_tokens(logits, dtype, rows, vocab, stride, uniform,
                                         ctypes.byref(options) if options else None, tokens, logprob, None)


def opts(**kw):
    o = _lib.BdhSampleOptions(1.0, 1.0, 0.0, 0, None, None, None, None)
    for k, v in kw.items():
        setattr(o, k, v)
    return o


@pytest.mark.parametrize("kw,status,why", [
    (dict(rows=0), _lib.BDH_UNSUPPORTED, "zero"), (dict(vocab=0), _lib.BDH_UNSUPPORTED, "zero"),
    (dict(vocab=(1 << 20) + 1, stride=1 << 21), _lib.BDH_UNSUPPORTED, "vocab"),
    (dict(rows=1 << 22), _lib.BDH_UNSUPPORTED, "rows"),
    (dict(logits=None), _lib.BDH_EINVAL, "null"), (dict(uniform=None), _lib.BDH_EINVAL, "null"),
    (dict(tokens=None), _lib.BDH_EINVAL, "null"), (dict(dtype=7), _lib.BDH_EINVAL, "dtype"),
    (dict(stride=-1), _lib.BDH_EINVAL, "row_stride"), (dict(stride=1 << 62), _lib.BDH_EINVAL, "row_stride"),
    (dict(logits=GOOD + 2), _lib.BDH_EINVAL, "aligned"),
    (dict(logits=GOOD + 1, dtype=_lib.BDH_BF16), _lib.BDH_EINVAL, "aligned"),
    (dict(uniform=GOOD + 2), _lib.BDH_EINVAL, "aligned"), (dict(tokens=GOOD + 1), _lib.BDH_EINVAL, "aligned"),
    (dict(logprob=GOOD + 2), _lib.BDH_EINVAL, "aligned"),
    (dict(options=opts(temperature_rows=GOOD + 2)), _lib.BDH_EINVAL, "aligned"),
    (dict(options=opts(temperature=-0.5)), _lib.BDH_EINVAL, "temperature"),
    (dict(options=opts(temperature=math.nan)), _lib.BDH_EINVAL, "temperature"),
    (dict(options=opts(temperature=math.inf)), _lib.BDH_EINVAL, "temperature"),
    (dict(options=opts(top_p=1.25)), _lib.BDH_EINVAL, "top_p"),
    (dict(options=opts(top_p=math.nan)), _lib.BDH_EINVAL, "top_p"),
    (dict(options=opts(min_p=-0.25)), _lib.BDH_EINVAL, "min_p"),
    (dict(options=opts(top_k=-1)), _lib.BDH_EINVAL, "top_k"),
])
def test_refusals(kw, status, why):
    assert call(**kw) == status
    assert why in _lib.last_error()


def test_python_surface_without_a_device():
    torch = pytest.importorskip("torch")
    if torch.cuda.is_available():
        pytest.skip("a GPU is present: covered by the gpu tests")
    import burn_dragon_amd as bd
    assert bd.sample_tokens(torch.zeros(2, 8), torch.zeros(2)) is None


def test_oracle_by_hand():
    x = np.log(np.array([0.1, 0.4, 0.2, 0.3]))
    assert [sampleref.sample_row(x, u)[0] for u in (0.05, 0.2, 0.55, 0.75)] == [0, 1, 2, 3]
    # the first two in order: 1 (0.4) and 3 (0.3), drawn in index order
    assert [sampleref.sample_row(x, u, top_k=2)[0] for u in (0.5, 0.6)] == [1, 3]
    # before 3 there is 0.4 of weight, before 2 there is 0.7
    assert [sampleref.sample_row(x, u, top_p=0.65)[0] for u in (0.5, 0.6)] == [1, 3]
    assert sampleref.sample_row(x, 0.99, top_p=0.39)[0] == 1
    assert sampleref.sample_row(x, 0.0, min_p=0.5)[0] == 1
    assert sampleref.sample_row(x, 0.0, min_p=0.49)[0] == 1
    assert sampleref.sample_row([1.0, 2.0, 2.0], 0.9, temperature=0.0) == (1, 0.0)
    assert sampleref.sample_row([-np.inf, np.nan], 0.5) == (-1, -math.inf)
    # ties by index
    assert sampleref.sample_row([1.0, 1.0, 1.0, 1.0], 0.99, top_k=2)[0] == 1
    token, lp = sampleref.sample_row(x, 0.55, top_k=3)
    assert token == 2 and abs(lp - math.log(0.2 / 0.9)) < 1e-12
