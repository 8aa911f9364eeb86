"""bdh_state_copy_streams' and its Python surface's refusals, on the CPU: the
argument checks run before any device call, so no address is read."""
import ctypes

import pytest

from burn_dragon_amd import _lib

MB = 1 << 20


def call(layers, rho, dst, src, src_layers=None, src_rho=None, n=None):
    def arrays(shapes, ptrs):
        d = (_lib.BdhLayerStateDesc * max(1, len(shapes)))()
        for i, s in enumerate(shapes):
            d[i].batch, d[i].heads, d[i].latent, d[i].embd = s
        return d, (ctypes.c_void_p * max(1, len(ptrs)))(*ptrs)
    d, p = arrays(layers, rho)
    sd, sp = arrays(src_layers, src_rho) if src_layers is not None else (None, None)
    k = len(dst) if n is None else n
    return _lib.load().bdh_state_copy_streams(
        len(layers), d, p, sd, sp, k, (ctypes.c_int32 * max(1, len(dst)))(*dst),
        (ctypes.c_int32 * max(1, len(src)))(*src), None)


SHAPE = (4, 2, 16, 8)


@pytest.mark.parametrize("dst,src,why", [
    ([4], [0], "outside"), ([-1], [0], "outside"), ([0], [4], "outside"), ([0], [-2], "outside"),
    ([1, 1], [0, 2], "twice"),
])
def test_slots_outside_the_batch_or_written_twice(dst, src, why):
    assert call([SHAPE], [MB], dst, src) == _lib.BDH_EINVAL
    assert why in _lib.last_error()


@pytest.mark.parametrize("layers,rho,why", [
    ([SHAPE], [MB + 2], "aligned"), ([SHAPE], [None], "null"),
    ([SHAPE, (3, 2, 16, 8)], [MB, 2 * MB], "batches"),
    ([SHAPE, SHAPE], [MB, MB], "share"), ([SHAPE, SHAPE], [MB, MB + 64], "share"),
    ([(4, 0, 16, 8)], [MB], "dimension"), ([(-1, 2, 16, 8)], [MB], "dimension"),
])
def test_layers_that_do_not_fit(layers, rho, why):
    assert call(layers, rho, [0], [1]) == _lib.BDH_EINVAL
    assert why in _lib.last_error()


def test_sources_that_do_not_fit():
    one = [(1, 2, 16, 8)]
    assert call([SHAPE], [MB], [0], [1], one, [2 * MB]) == _lib.BDH_EINVAL  # the source has one stream
    assert call([SHAPE], [MB], [0], [0], [(1, 2, 16, 4)], [2 * MB]) == _lib.BDH_EINVAL
    assert "shapes" in _lib.last_error()
    assert call([SHAPE], [MB], [0], [0], one, [MB + 1024]) == _lib.BDH_EINVAL
    assert "share" in _lib.last_error()
    assert call([SHAPE], [MB], [0], [0], [(0, 0, 0, 0)], [None]) == _lib.BDH_EINVAL


def test_sizes_beyond_a_launch():
    assert call([(32768, 1, 1, 1)], [MB], [0], [1]) == _lib.BDH_UNSUPPORTED
    assert call([(2, 1 << 20, 1 << 20, 1)], [MB], [0], [1]) == _lib.BDH_UNSUPPORTED
    assert call([(2, 1 << 40, 1 << 40, 1 << 40)], [MB], [0], [1]) == _lib.BDH_UNSUPPORTED


def test_nothing_to_move_is_no_error():
    assert call([SHAPE], [MB], [], []) == _lib.BDH_OK
    assert call([], [], [], []) == _lib.BDH_OK
    assert call([(0, 0, 0, 0)], [None], [], []) == _lib.BDH_OK
    assert call([SHAPE], [MB], [0], [0], n=-1) == _lib.BDH_EINVAL


def test_python_surface_without_a_device():
    torch = pytest.importorskip("torch")
    if torch.cuda.is_available():
        pytest.skip("a GPU is present: covered by the gpu tests")
    import burn_dragon_amd as bd
    rho = [torch.zeros(4, 2, 16, 8)]
    assert bd.copy_streams(rho, [0], [1]) is None
    assert bd.free_streams(rho, [0]) is None
