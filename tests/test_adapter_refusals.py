"""bdh_apply_adapters' refusals, on the CPU: the argument checks run before
any device call."""
import ctypes

import pytest

from burn_dragon_amd import _lib

MB = 1 << 20
SIZES = dict(batch=2, time=3, in_dim=8, out_dim=16, rank=4, adapters=5)


def call(dtype=_lib.BDH_F32, base=MB, hidden=2 * MB, a=3 * MB, b=4 * MB, scale=5 * MB, ids=6 * MB, out=7 * MB,
         plan=True, **sizes):
    p = _lib.BdhAdapterPlan(*{**SIZES, **sizes}.values())
    return _lib.load().bdh_apply_adapters(ctypes.byref(p) if plan else None, dtype, base, hidden, a, b, scale, ids,
                                          out, None)


@pytest.mark.parametrize("kw,status,why", [
    (dict(plan=False), _lib.BDH_EINVAL, "null"),
    *[({k: 0}, _lib.BDH_UNSUPPORTED, "zero") for k in SIZES],
    *[({k: -1}, _lib.BDH_UNSUPPORTED, "zero") for k in SIZES],
    *[({k: None}, _lib.BDH_EINVAL, "null") for k in ("base", "hidden", "a", "b", "scale", "ids", "out")],
    (dict(dtype=3), _lib.BDH_EINVAL, "dtype"),
    (dict(rank=129), _lib.BDH_UNSUPPORTED, "rank"),
    (dict(batch=70000), _lib.BDH_UNSUPPORTED, "batch"),
    (dict(out_dim=(1 << 22) + 1), _lib.BDH_UNSUPPORTED, "large"),
    (dict(batch=60000, time=1000), _lib.BDH_UNSUPPORTED, "large"),
    *[({k: MB * 9 + 2}, _lib.BDH_EINVAL, "aligned") for k in ("base", "hidden", "out", "scale", "ids")],
    *[({k: MB * 9 + 1}, _lib.BDH_EINVAL, "aligned") for k in ("a", "b")],
    (dict(dtype=_lib.BDH_BF16, out=MB * 9 + 1), _lib.BDH_EINVAL, "aligned"),
    (dict(out=MB + 4), _lib.BDH_EINVAL, "shares"),            # a shifted base
    (dict(out=MB - 4), _lib.BDH_EINVAL, "shares"),
    (dict(out=2 * MB), _lib.BDH_EINVAL, "shares"),
    (dict(out=4 * MB + 64), _lib.BDH_EINVAL, "shares"),
    (dict(out=6 * MB + 4), _lib.BDH_EINVAL, "shares"),
])
def test_refusals(kw, status, why):
    assert call(**kw) == status
    assert why in _lib.last_error()


def test_python_surface_without_a_device():
    torch = pytest.importorskip("torch")
    if torch.cuda.is_available():
        pytest.skip("a GPU is present: covered by the gpu tests")
    import burn_dragon_amd as bd
    s = bd.AdapterSet(torch.zeros(1, 2, 4, dtype=torch.bfloat16), torch.zeros(1, 8, 2, dtype=torch.bfloat16),
                      torch.ones(1))
    assert bd.apply_adapters(torch.zeros(2, 8), torch.zeros(2, 4), s, torch.zeros(2, dtype=torch.int32)) is None


def test_time_past_the_grid_is_refused():
    assert call(batch=1, time=65535 * 64 + 1) == _lib.BDH_UNSUPPORTED
    assert "large" in _lib.last_error()


def test_the_plan_s_limits_are_the_library_s():
    # The largest of each size that the plan takes passes the library's check of
    # sizes too (and ends at the misaligned base); one more is refused by both.
    torch = pytest.importorskip("torch")
    from burn_dragon_amd import AdapterSet
    from burn_dragon_amd import adapters as ad

    def plan(batch, time, in_dim, out_dim, rank, adapters):
        one = torch.zeros(1, dtype=torch.bfloat16)
        s = AdapterSet(one.expand(adapters, rank, in_dim), one.expand(adapters, out_dim, rank),
                       torch.ones(1).expand(adapters))
        return ad.adapter_plan((batch, time, out_dim), (batch, time, in_dim), torch.device("cpu"), s,
                               torch.zeros(1, dtype=torch.int32).expand(batch))
    for size, most in (("batch", 65535), ("time", 65535 * 64), ("in_dim", 1 << 20), ("out_dim", 1 << 22),
                       ("rank", 128), ("adapters", 1 << 20)):
        small = dict(batch=1, time=1, in_dim=1, out_dim=1, rank=1, adapters=1)
        p = plan(**{**small, size: most})
        assert [getattr(p, k) for k in SIZES] == [{**small, size: most}[k] for k in SIZES]
        assert call(base=MB + 2, **{**small, size: most}) == _lib.BDH_EINVAL and "aligned" in _lib.last_error()
        assert plan(**{**small, size: most + 1}) is None
        assert call(base=MB + 2, **{**small, size: most + 1}) == _lib.BDH_UNSUPPORTED
    rows = dict(batch=4, in_dim=1, out_dim=1, rank=1, adapters=1)
    assert plan(time=1 << 21, **rows) is not None and plan(time=(1 << 21) + 1, **rows) is None
    assert call(base=MB + 2, **rows, time=1 << 21) == _lib.BDH_EINVAL
    assert call(base=MB + 2, **rows, time=(1 << 21) + 1) == _lib.BDH_UNSUPPORTED
