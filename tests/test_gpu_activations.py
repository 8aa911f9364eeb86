"""checkpoint_activations and restore_activations: bit for bit what the
definition gives in 64 bits (tests/trainref.py)."""
import numpy as np
import pytest

from tests import trainref as R
from tests.gpu_util import announce, need_gpu

pytestmark = pytest.mark.gpu


def run(torch, x):
    """Saves and restores x and holds every code, power and value to the definition."""
    import burn_dragon_amd as bd
    announce("activations", tuple(x.shape), x.dtype, tuple(x.stride()))
    c = bd.checkpoint_activations(x)
    back = [bd.restore_activations(c, dtype=t) for t in (torch.float32, torch.bfloat16)]
    torch.cuda.synchronize()
    C = x.shape[-1]
    want, e = R.in8(x.reshape(-1, C).double().cpu().numpy())
    assert tuple(c.codes.shape) == tuple(x.shape) and tuple(c.scales.shape) == (*x.shape[:-1], -(-C // 32))
    assert np.array_equal(c.scales.cpu().numpy().reshape(e.shape), e + 127)
    p = np.ldexp(1.0, np.repeat(e, 32, 1)[:, :C])
    codes = c.codes.cpu().numpy().reshape(want.shape).astype(int)
    held = np.append(R.E4M3, np.nan)[codes & 127] * np.where(codes >> 7, -1.0, 1.0) * p
    for got in [held] + [b.double().cpu().numpy().reshape(want.shape) for b in back]:
        assert np.array_equal(got, want, equal_nan=True)
    assert back[0].dtype == torch.float32 and back[1].dtype == torch.bfloat16


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("rows", [1, 3, 130])
@pytest.mark.parametrize("C", [1, 7, 8, 9, 31, 32, 33, 63, 64, 100, 256, 1001, 8192])
def test_sizes(rows, C, dtype):
    torch = need_gpu()
    g = torch.Generator(device="cuda").manual_seed(rows * 10007 + C)
    x = torch.randn(rows, C, generator=g, device="cuda") * torch.exp(3 * torch.randn(rows, 1, generator=g, device="cuda"))
    run(torch, x.to(getattr(torch, dtype)))


def test_more_work_than_a_launch_has_threads():
    torch = need_gpu()
    x = torch.randn(3, 1 << 23, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).bfloat16()
    run(torch, x[:, :8000064])


def test_borders_and_ties():
    # Every code's value, the middles between neighbours and the values beside them, at
    # powers from the least to the largest.
    torch = need_gpu()
    middles = (R.E4M3[1:] + R.E4M3[:-1]) / 2
    v = np.concatenate([R.E4M3, middles, np.nextafter(middles.astype(np.float32), np.float32(0)),
                        np.nextafter(middles.astype(np.float32), np.float32(1e9))])
    v = np.concatenate([v, -v]).astype(np.float32)
    blocks = np.full((len(v), 32), 448.0, np.float32)   # (448 sets the block's power to 1)
    blocks[:, 1:31] = v[:, None]
    for k in (0, -30, 40, 119, -117):
        run(torch, torch.from_numpy(np.ldexp(blocks, k)).cuda())
    # A block's largest value on either side of 448 times a power of two.
    tops = [np.ldexp(np.float32(m), k) for k in (-140, -126, -110, -20, 0, 100, 120)
            for m in (447.0, 448.0, np.nextafter(np.float32(448), np.float32(1e9)), 449.0, 256.0, 255.9)]
    x = np.zeros((len(tops), 64), np.float32)
    x[:, 5] = tops
    x[:, 6] = np.array(tops) / 3
    x[:, 40] = -np.array(tops)
    run(torch, torch.from_numpy(x[np.isfinite(x).all(1)]).cuda())


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_infinities_nan_zeros_and_subnormals(dtype):
    torch = need_gpu()
    x = torch.randn(6, 96, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2))
    x[0] = 0.0
    x[1, :40] = -0.0
    x[2, 3], x[2, 50], x[2, 51] = float("inf"), -float("inf"), float("nan")
    x[3] = float("nan")
    x[4] *= 1e-39
    x[5, :64] *= 3e38 / x[5, :64].abs().max()
    run(torch, x.to(getattr(torch, dtype)))


def test_strides_streams_and_out():
    torch = need_gpu()
    import burn_dragon_amd as bd
    x = torch.randn(5, 7, 66, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3))
    run(torch, x.transpose(0, 1))
    run(torch, x[:, :, 1:])
    run(torch, x.flatten()[1:2300])
    a = bd.checkpoint_activations(x)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    announce("activations on a stream and in a graph")
    b = bd.ActivationCheckpoint(torch.zeros_like(a.codes), torch.zeros_like(a.scales))
    y = torch.zeros_like(x)
    with torch.cuda.stream(s):
        assert bd.checkpoint_activations(x, out=b) is b
        assert bd.restore_activations(b, out=y) is y
    s.synchronize()
    assert torch.equal(a.codes, b.codes) and torch.equal(a.scales, b.scales)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        bd.restore_activations(bd.checkpoint_activations(x, out=b), out=y)
    for k in range(3):
        x.copy_(torch.randn_like(x))
        graph.replay()
        want = bd.restore_activations(bd.checkpoint_activations(x), dtype=torch.float32)
        torch.cuda.synchronize()
        assert torch.equal(y, want)


def test_refusals():
    torch = need_gpu()
    import burn_dragon_amd as bd
    x = torch.randn(4, 64, device="cuda")
    c = bd.checkpoint_activations(x)
    assert bd.checkpoint_activations(x.half()) is None
    assert bd.checkpoint_activations(x[:0]) is None
    assert bd.restore_activations(c, dtype=torch.float16) is None
    for call in (lambda: bd.checkpoint_activations(x[:3], out=c),
                 lambda: bd.restore_activations(bd.ActivationCheckpoint(c.codes, c.scales[:3])),
                 lambda: bd.restore_activations(bd.ActivationCheckpoint(c.codes, c.scales.cpu())),
                 lambda: bd.restore_activations(c, out=torch.empty(4, 63, device="cuda"))):
        with pytest.raises(ValueError):
            call()
