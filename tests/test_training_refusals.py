"""The training operators' refusals, on the CPU: the argument checks run
before any device call."""
import ctypes
import math

import pytest

from burn_dragon_amd import _lib

MB = 1 << 20
OK_SIZES = dict(n=3, vocab=10, embd=16)


def embed(dtype=_lib.BDH_F32, tokens=MB, table=2 * MB, out=3 * MB, scale=1.0, **sizes):
    s = {**OK_SIZES, **sizes}
    return _lib.load().bdh_embed_tokens(tokens, s["n"], table, dtype, s["vocab"], s["embd"], scale, 0, out, None)


def embed_vjp(dtype=_lib.BDH_F32, tokens=MB, table=2 * MB, grad=3 * MB, out=4 * MB, scale=1.0, norm=1, **sizes):
    s = {**OK_SIZES, **sizes}
    return _lib.load().bdh_embed_tokens_vjp(tokens, s["n"], table, dtype, s["vocab"], s["embd"], scale, norm, grad,
                                            out, 0, None)


SIZES = [
    *[({k: v}, _lib.BDH_UNSUPPORTED, "zero") for k in OK_SIZES for v in (0, -1)],
    (dict(dtype=5), _lib.BDH_EINVAL, "dtype"),
    (dict(scale=math.nan), _lib.BDH_EINVAL, "finite"),
    (dict(scale=math.inf), _lib.BDH_EINVAL, "finite"),
    (dict(embd=2049), _lib.BDH_UNSUPPORTED, "2048"),
    (dict(vocab=(1 << 24) + 1), _lib.BDH_UNSUPPORTED, "2^24"),
    (dict(n=(1 << 24) + 1), _lib.BDH_UNSUPPORTED, "2^24"),
    (dict(tokens=MB + 2), _lib.BDH_EINVAL, "aligned"),
    (dict(out=9 * MB + 2), _lib.BDH_EINVAL, "aligned"),
    (dict(dtype=_lib.BDH_BF16, out=9 * MB + 1), _lib.BDH_EINVAL, "aligned"),
    (dict(tokens=None), _lib.BDH_EINVAL, "null"),
    (dict(out=None), _lib.BDH_EINVAL, "null"),
    (dict(out=2 * MB + 4), _lib.BDH_EINVAL, "shares"),
    (dict(out=MB + 8), _lib.BDH_EINVAL, "shares"),
]


@pytest.mark.parametrize("kw,status,why", SIZES + [(dict(table=None), _lib.BDH_EINVAL, "null"),
                                                   (dict(table=9 * MB + 2), _lib.BDH_EINVAL, "aligned")])
def test_embed_tokens(kw, status, why):
    assert embed(**kw) == status
    assert why in _lib.last_error()


@pytest.mark.parametrize("kw,status,why", SIZES + [
    (dict(table=None), _lib.BDH_EINVAL, "null"), (dict(grad=None), _lib.BDH_EINVAL, "null"),
    (dict(grad=9 * MB + 2), _lib.BDH_EINVAL, "aligned"), (dict(out=3 * MB + 100), _lib.BDH_EINVAL, "shares")])
def test_embed_tokens_vjp(kw, status, why):
    assert embed_vjp(**kw) == status
    assert why in _lib.last_error()


def save(x=MB, dtype=_lib.BDH_BF16, rows=4, cols=64, codes=2 * MB, scales=3 * MB):
    return _lib.load().bdh_activations_save(x, dtype, rows, cols, codes, scales, None)


def restore(x=MB, dtype=_lib.BDH_BF16, rows=4, cols=64, codes=2 * MB, scales=3 * MB):
    return _lib.load().bdh_activations_restore(codes, scales, rows, cols, dtype, x, None)


@pytest.mark.parametrize("call", [save, restore])
@pytest.mark.parametrize("kw,status,why", [
    *[({k: v}, _lib.BDH_UNSUPPORTED, "zero") for k in ("rows", "cols") for v in (0, -3)],
    *[({k: None}, _lib.BDH_EINVAL, "null") for k in ("x", "codes", "scales")],
    (dict(dtype=2), _lib.BDH_EINVAL, "dtype"),
    (dict(cols=(1 << 30) + 1), _lib.BDH_UNSUPPORTED, "large"),
    (dict(rows=1 << 40, cols=33), _lib.BDH_UNSUPPORTED, "large"),
    (dict(x=9 * MB + 1), _lib.BDH_EINVAL, "aligned"),
    (dict(dtype=_lib.BDH_F32, x=9 * MB + 2), _lib.BDH_EINVAL, "aligned"),
    (dict(codes=MB + 100), _lib.BDH_EINVAL, "share"),
    (dict(scales=MB + 10), _lib.BDH_EINVAL, "share"),
    (dict(scales=2 * MB + 255), _lib.BDH_EINVAL, "share"),
])
def test_activations(call, kw, status, why):
    assert call(**kw) == status
    assert why in _lib.last_error()


PLAN = dict(batch=2, heads=3, time=5, latent=64, embd=32)
TENSORS = ("current", "context", "up", "gate")


def _gated(kw, names, call):
    p = _lib.BdhLayerPlan(*[kw.pop(k, v) for k, v in PLAN.items()])
    o = _lib.BdhGatedOptions(kw.pop("activation", _lib.BDH_RELU), kw.pop("threshold", 0.0), kw.pop("mask", None))
    plan = ctypes.byref(p) if kw.pop("plan", True) else None
    at = {n: (i + 1) * MB for i, n in enumerate(TENSORS + names)}
    at.update(kw)
    return call(plan, *[at[n] for n in TENSORS], ctypes.byref(o), *[at[n] for n in names], None)


FWD = ("out", "up_codes", "up_scales", "gate_codes", "gate_scales")
BWD = ("grad_out", *FWD[1:], "grad_current", "grad_context", "grad_up", "grad_gate")
BOTH = [
    (dict(plan=False), _lib.BDH_EINVAL, "null"),
    *[({k: v}, _lib.BDH_UNSUPPORTED, "zero") for k in PLAN for v in (0, -1)],
    *[({k: None}, _lib.BDH_EINVAL, "null") for k in ("current", "up", "gate")],
    (dict(latent=60), _lib.BDH_UNSUPPORTED, "multiples"),
    (dict(embd=36), _lib.BDH_UNSUPPORTED, "multiples"),
    (dict(time=1 << 22), _lib.BDH_UNSUPPORTED, "large"),
    (dict(batch=1 << 62, time=1 << 62), _lib.BDH_UNSUPPORTED, "large"),
    (dict(heads=513), _lib.BDH_UNSUPPORTED, "large"),
    (dict(latent=(1 << 20) + 8), _lib.BDH_UNSUPPORTED, "large"),
    (dict(embd=(1 << 16) + 8), _lib.BDH_UNSUPPORTED, "large"),
    (dict(heads=256, latent=(1 << 16) + 8), _lib.BDH_UNSUPPORTED, "large"),
    (dict(batch=1 << 10, time=1 << 10, heads=1, latent=1 << 15), _lib.BDH_UNSUPPORTED, "large"),
    (dict(activation=3), _lib.BDH_EINVAL, "activation"),
    (dict(threshold=math.inf), _lib.BDH_EINVAL, "finite"),
    (dict(activation=_lib.BDH_SILU, threshold=0.5), _lib.BDH_EINVAL, "BDH_RELU"),
    (dict(activation=_lib.BDH_GELU, mask=60 * MB), _lib.BDH_EINVAL, "BDH_RELU"),
    (dict(mask=60 * MB + 4), _lib.BDH_EINVAL, "aligned"),
    *[({k: 60 * MB + 8}, _lib.BDH_EINVAL, "aligned") for k in TENSORS],
    *[({k: None}, _lib.BDH_EINVAL, "together") for k in FWD[1:]],
]


@pytest.mark.parametrize("kw,status,why", BOTH + [
    (dict(out=None), _lib.BDH_EINVAL, "null"), (dict(out=60 * MB + 2), _lib.BDH_EINVAL, "aligned"),
    (dict(up_codes=60 * MB + 8), _lib.BDH_EINVAL, "aligned"),
    (dict(out=MB + 16), _lib.BDH_EINVAL, "shares"), (dict(out=3 * MB), _lib.BDH_EINVAL, "shares"),
    (dict(gate_codes=6 * MB + 16), _lib.BDH_EINVAL, "shares"), (dict(up_scales=5 * MB), _lib.BDH_EINVAL, "shares"),
    (dict(mask=5 * MB), _lib.BDH_EINVAL, "shares")])
def test_gated_block(kw, status, why):
    assert _gated(dict(kw), FWD, _lib.load().bdh_gated_block_fwd) == status
    assert why in _lib.last_error()


@pytest.mark.parametrize("kw,status,why", BOTH + [
    *[({k: None}, _lib.BDH_EINVAL, "null") for k in ("grad_out", "grad_current", "grad_up", "grad_gate")],
    (dict(grad_context=None), _lib.BDH_EINVAL, "together"), (dict(context=None), _lib.BDH_EINVAL, "together"),
    *[({k: 60 * MB + 8}, _lib.BDH_EINVAL, "aligned") for k in ("grad_out", "gate_codes", *BWD[5:])],
    (dict(grad_current=MB), _lib.BDH_EINVAL, "shares"), (dict(grad_up=13 * MB), _lib.BDH_EINVAL, "shares"),
    (dict(grad_gate=5 * MB + 16), _lib.BDH_EINVAL, "shares")])
def test_gated_block_vjp(kw, status, why):
    assert _gated(dict(kw), BWD, _lib.load().bdh_gated_block_vjp) == status
    assert why in _lib.last_error()


def test_more_tiles_than_a_launch_has():
    kw = dict(batch=1 << 11, time=1 << 11, heads=512, latent=8)
    for names, call in ((FWD, _lib.load().bdh_gated_block_fwd), (BWD, _lib.load().bdh_gated_block_vjp)):
        assert _gated(dict(kw), names, call) == _lib.BDH_UNSUPPORTED
        assert "large" in _lib.last_error()


def test_python_surface_without_a_device():
    torch = pytest.importorskip("torch")
    if torch.cuda.is_available():
        pytest.skip("a GPU is present: covered by the gpu tests")
    import burn_dragon_amd as bd
    t = torch.zeros(4, dtype=torch.int32)
    assert bd.embed_tokens(t, torch.zeros(5, 8)) is None
    assert bd.embed_tokens_vjp(torch.zeros(4, 8), t, torch.zeros(5, 8)) is None
    assert bd.checkpoint_activations(torch.zeros(4, 8)) is None
    u8 = torch.zeros(4, 8, dtype=torch.uint8)
    assert bd.restore_activations(bd.ActivationCheckpoint(u8, u8[:, :1])) is None
    b = torch.zeros(1, 8, 8, dtype=torch.bfloat16)
    w = bd.GatedWeights(b, b)
    assert bd.gated_block(b, w) is None and bd.gated_block_vjp(b, b, w) is None
