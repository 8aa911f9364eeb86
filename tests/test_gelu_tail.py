"""The polynomial of the normal distribution's tail (normal(), burn_dragon_amd/csrc/gated.hip):
its constants, as the kernel holds them in f32, are as close as the comment
beside them says, and a fit made here by the same method does no better than
their rounding."""
import os
import re

import numpy as np

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
FAR = 14.5  # past it exp(-q^2 / 2) is 0 in f32


def _source():
    """(text of the comment, slope, coefficients from the highest power down)."""
    text = open(os.path.join(ROOT, "burn_dragon_amd", "csrc", "gated.hip")).read()
    comment = text[text.index("// The normal distribution at q"):text.index("struct Normal {")]
    body = text[text.index("Normal normal(float q)"):text.index("const float tail = f * t * bell;")]
    slope = float(re.search(r"fmaf\(([\d.]+)f, fabsf\(q\), 1\.0f\)", body).group(1))
    terms = [float(re.search(r"float f = (-?[\d.]+)f;", body).group(1))]
    terms += [float(x) for x in re.findall(r"f = fmaf\(f, t, (-?[\d.]+)f\);", body)]
    return " ".join(comment.replace("//", " ").split()), slope, terms


def _stated(comment, pattern):
    return float(re.search(pattern, comment).group(1))


def _scaled_tail(q):
    """exp(q^2 / 2) (1 - Phi(q))."""
    from scipy.special import erfcx
    return 0.5 * erfcx(q / np.sqrt(2.0))


def _poly(terms, t):
    f = np.zeros_like(t)
    for c in terms:
        f = f * t + c
    return f * t


def test_constants_are_as_close_as_stated():
    comment, slope, terms = _source()
    assert len(terms) == 9
    q = np.linspace(0.0, FAR, 200001)
    held = [float(np.float32(c)) for c in terms]
    off = np.abs(_poly(held, 1.0 / (1.0 + float(np.float32(slope)) * q)) / _scaled_tail(q) - 1.0).max()
    assert off <= _stated(comment, r"([\d.e-]+) of a tail to")


def test_f32_steps_are_as_close_as_stated():
    # Every step rounded to f32; exp and the reciprocal to nearest, the kernel's are off
    # by a step or so each: 1.2e-7 of a tail, and of 1/2 at most.
    from scipy.special import ndtr
    comment, slope, terms = _source()
    f32 = np.float32
    q = np.linspace(-FAR, FAR, 400001).astype(f32)
    fma = lambda x, y, z: (x.astype(float) * np.asarray(y, float) + np.asarray(z, float)).astype(f32)  # noqa: E731
    bell = np.exp((f32(-0.5) * q * q).astype(float)).astype(f32)
    t = f32(1) / fma(np.abs(q), f32(slope), f32(1))
    f = np.full_like(q, f32(terms[0]))
    for c in terms[1:]:
        f = fma(f, t, f32(c))
    tail = f * t * bell
    cdf = np.where(q > 0, f32(1) - tail, tail).astype(float)
    want = ndtr(q.astype(float))
    other = 2 * 1.2e-7
    assert np.abs(cdf - want).max() <= _stated(comment, r"within ([\d.e-]+) of Phi") + other * 0.5
    near = (q < 0) & (q >= -6)
    assert np.abs(cdf[near] / want[near] - 1).max() <= _stated(comment, r"is ([\d.e-]+) of a tail at \|q\| = 6") + other


def test_a_fit_made_here_gives_such_constants():
    # Least squares of the relative error, the weights moved towards the largest.
    _, slope, terms = _source()
    slope = float(np.float32(slope))
    q = 0.5 * FAR * (1.0 - np.cos(np.pi * (np.arange(2000) + 0.5) / 2000))
    t, want = 1.0 / (1.0 + slope * q), _scaled_tail(q)
    basis = np.stack([t ** k for k in range(9, 0, -1)], 1) / want[:, None]
    weight, best = np.ones_like(q), 1.0
    for _ in range(200):
        root = np.sqrt(weight)
        fit = np.linalg.lstsq(basis * root[:, None], root, rcond=None)[0]
        off = np.abs(basis @ fit - 1.0)
        best = min(best, off.max())
        weight *= off
        weight /= weight.sum()
    assert best <= 1e-7
    mine = np.abs(basis @ np.array([float(np.float32(c)) for c in terms]) - 1.0).max()
    assert mine <= best + 2.0 ** -23  # two roundings' share
