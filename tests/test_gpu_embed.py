"""embed_tokens and embed_tokens_vjp against the formula in 64 bits (bounds:
tests/trainref.py)."""
import numpy as np
import pytest

from tests import trainref as R
from tests.gpu_util import announce, need_gpu

pytestmark = pytest.mark.gpu

DIMS = [1, 3, 4, 63, 64, 65, 200, 256, 257, 511, 512, 1000, 1024, 1027, 2047, 2048]


def make(torch, n, V, D, dtype, seed, tokens=None, shift=0.5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    table = (shift + torch.randn(V, D, generator=g, device="cuda")).to(dtype)
    grad = torch.randn(n, D, generator=g, device="cuda").to(dtype)
    if tokens is None:
        tokens = torch.randint(-2, V + 2, (n,), generator=g, device="cuda", dtype=torch.int32)
    return tokens, table, grad


def f64(t):
    return t.cpu().double().numpy()


def check(got, want, bound):
    off = np.abs(f64(got).reshape(want.shape) - want)
    assert np.all(off <= bound), (float(off.max()), float((off / bound).max()))


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("D", DIMS)
def test_rows(D, norm, dtype):
    torch = need_gpu()
    import burn_dragon_amd as bd
    dtype = getattr(torch, dtype)
    tokens, table, _ = make(torch, 37, 11, D, dtype, D)
    announce("embed", D, norm, dtype)
    out = bd.embed_tokens(tokens, table, scale=1.7, norm=norm)
    torch.cuda.synchronize()
    assert out.dtype == dtype and tuple(out.shape) == (37, D)
    check(out, *R.embed(tokens.cpu().numpy(), f64(table), float(np.float32(1.7)), norm, torch.finfo(dtype).eps))


@pytest.mark.parametrize("n,V", [(1, 1), (1, 256), (5, 100003), (4097, 300)])
def test_shapes_and_out(n, V):
    torch = need_gpu()
    import burn_dragon_amd as bd
    tokens, table, _ = make(torch, n, V, 96, torch.float32, n + V)
    announce("embed", n, V)
    out = torch.full((n, 1, 96), float("nan"), device="cuda")
    assert bd.embed_tokens(tokens[:, None], table, out=out) is out
    want = R.embed(tokens.cpu().numpy(), f64(table), 1.0, False, torch.finfo(torch.float32).eps)
    check(out, *want)
    # A table whose rows lie apart, tokens that are a slice of a batch, both at odd offsets.
    wide = torch.zeros(V, 97, device="cuda")
    wide[:, 1:] = table
    pairs = torch.stack([tokens, tokens], 1)
    check(bd.embed_tokens(pairs[:, 1], wide[:, 1:]), *want)


def test_norm_is_the_models_input():
    # The lookup that model_forward_logits begins with, within both kernels' bounds.
    torch = need_gpu()
    import ctypes

    import burn_dragon_amd as bd
    from burn_dragon_amd import _lib
    tokens, table, _ = make(torch, 100, 256, 256, torch.float32, 3)
    announce("embed against embed_norm")
    out = bd.embed_tokens(tokens, table, norm=True)
    ref = torch.empty_like(out)
    p = lambda t: ctypes.c_void_p(t.data_ptr())  # noqa: E731
    assert _lib.load().bdh_embed_norm(p(tokens), 100, p(table), 256, 256, p(ref), None) == _lib.BDH_OK
    torch.cuda.synchronize()
    want, bound = R.embed(tokens.cpu().numpy(), f64(table), 1.0, True, torch.finfo(torch.float32).eps)
    check(out, want, bound)
    # (embed_norm's one mean: its 17 U of the values stays.)
    check(ref, want, bound + 40 * R.U * (1 + np.abs(f64(table)).max()))


# The ids' patterns of the gradient.
def ids(kind, n, V, rng):
    if kind == "uniform":
        return rng.integers(-2, V + 2, n)
    if kind == "one":
        return np.full(n, V // 2)
    if kind == "none":
        return np.where(rng.random(n) < 0.5, -1, V)
    if kind == "extremes":
        return rng.choice([0, V - 1, -2147483648, 2147483647], n)
    if kind == "ordered":
        return np.arange(n) % V
    return np.minimum(rng.zipf(1.3, n) - 1, V - 1)   # "zipf"


def run_vjp(n, V, D, dtype, norm, kind, accumulate=False, seed=0):
    torch = need_gpu()
    import burn_dragon_amd as bd
    dtype = getattr(torch, dtype)
    rng = np.random.default_rng(n * 31 + V * 7 + D + seed)
    tokens = torch.from_numpy(ids(kind, n, V, rng).astype(np.int32)).cuda()
    tokens, table, grad = make(torch, n, V, D, dtype, n + D, tokens)
    old = torch.randn(V, D, device="cuda").to(dtype) if accumulate else None
    announce("embed vjp", n, V, D, dtype, norm, kind, accumulate)
    out = old.clone() if accumulate else torch.full((V, D), float("nan"), device="cuda", dtype=dtype)
    assert bd.embed_tokens_vjp(grad, tokens, table, scale=1.7, norm=norm, out=out, accumulate=accumulate) is out
    torch.cuda.synchronize()
    want, bound = R.embed_vjp(f64(grad), tokens.cpu().numpy(), f64(table), float(np.float32(1.7)), norm,
                              torch.finfo(dtype).eps, f64(old) if accumulate else None)
    check(out, want, bound)
    again = old.clone() if accumulate else torch.empty_like(out)
    bd.embed_tokens_vjp(grad, tokens, table, scale=1.7, norm=norm, out=again, accumulate=accumulate)
    assert torch.equal(out, again)   # bit for bit


@pytest.mark.parametrize("kind", ["uniform", "one", "none", "extremes", "ordered", "zipf"])
@pytest.mark.parametrize("n,V", [(1, 1), (1, 300), (15, 2), (16, 7), (17, 256), (100, 511), (2048, 512),
                                 (2049, 5000), (5000, 100)])
def test_vjp_ids(n, V, kind):
    run_vjp(n, V, 20, "float32", False, kind)
    run_vjp(n, V, 20, "bfloat16", True, kind, accumulate=True)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("D", DIMS)
def test_vjp_columns(D, norm, dtype):
    run_vjp(333, 50, D, dtype, norm, "zipf")


@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("n,V,D,dtype,norm,kind", [
    (20000, 300, 64, "float32", True, "zipf"), (70000, 50000, 8, "bfloat16", False, "uniform"),
    (140000, 262144, 4, "float32", False, "zipf"), (3000, 300000, 12, "float32", True, "uniform"),
    (140000, 3, 16, "float32", True, "uniform"), (17000, 256, 256, "float32", True, "one")])
def test_vjp_large(n, V, D, dtype, norm, kind, accumulate):
    run_vjp(n, V, D, dtype, norm, kind, accumulate)


def test_vjp_is_the_difference_of_the_rows():
    # d/ds of sum(g * embed(E + s dE)) at s = 0, by a central difference in 64 bits of the
    # formula, against <grad, dE>.
    torch = need_gpu()
    import burn_dragon_amd as bd
    tokens, table, grad = make(torch, 64, 9, 33, torch.float32, 5)
    announce("embed vjp by differences")
    out = f64(bd.embed_tokens_vjp(grad, tokens, table, scale=0.5, norm=True))
    t, e, g = tokens.cpu().numpy(), f64(table), f64(grad)
    d = np.random.default_rng(1).standard_normal(e.shape)
    h = 1e-4
    f = lambda x: float((g * R.embed(t, x, 0.5, True, 0)[0]).sum())  # noqa: E731
    slope = (f(e + h * d) - f(e - h * d)) / (2 * h)
    # h^2 / 6 of a third derivative of a few hundred; f32's share of the sums beside it
    assert abs(float((out * d).sum()) - slope) <= 1e-5 * float(np.abs(out * d).sum() + 1)


def test_vjp_in_a_graph_and_on_streams():
    torch = need_gpu()
    import burn_dragon_amd as bd
    cases = [make(torch, n, 300, 64, torch.float32, n) for n in (3000, 2999)]
    want = [bd.embed_tokens_vjp(g, t, e, norm=True) for t, e, g in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    announce("embed vjp on two streams")
    got = []
    for s, (t, e, g) in zip(streams, cases):
        with torch.cuda.stream(s):
            got.append([bd.embed_tokens_vjp(g, t, e, norm=True) for _ in range(3)])
    torch.cuda.synchronize()
    for w, o in zip(want, got):
        assert all(torch.equal(w, x) for x in o)
    s, (t, e, g) = streams[0], cases[0]
    out = torch.empty_like(want[0])
    announce("embed vjp captured")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        assert bd.embed_tokens_vjp(g, t, e, norm=True, out=out) is not None
    for k in range(3):
        new = make(torch, 3000, 300, 64, torch.float32, 50 + k)
        for to, from_ in zip((t, e, g), new):
            to.copy_(from_)
        out.fill_(float("nan"))
        graph.replay()
        eager = bd.embed_tokens_vjp(g, t, e, norm=True)
        torch.cuda.synchronize()
        assert torch.equal(out, eager)
    del graph
    for s in streams:
        with torch.cuda.stream(s):
            bd.release_stream_scratch(s)


def test_refusals():
    torch = need_gpu()
    import burn_dragon_amd as bd
    tokens, table, grad = make(torch, 10, 7, 16, torch.float32, 1)
    assert bd.embed_tokens(tokens, table.half()) is None
    assert bd.embed_tokens(tokens[:0], table) is None
    assert bd.embed_tokens(tokens, torch.zeros(3, 2049, device="cuda")) is None
    assert bd.embed_tokens_vjp(grad[:0], tokens[:0], table) is None
    for call in (lambda: bd.embed_tokens(tokens.long(), table), lambda: bd.embed_tokens(tokens.cpu(), table),
                 lambda: bd.embed_tokens(tokens, table, out=torch.empty(10, 17, device="cuda")),
                 lambda: bd.embed_tokens_vjp(grad[:5], tokens, table),
                 lambda: bd.embed_tokens_vjp(grad.bfloat16(), tokens, table),
                 lambda: bd.embed_tokens_vjp(grad, tokens, table, accumulate=True)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(Exception, match="finite"):
        bd.embed_tokens(tokens, table, scale=float("inf"))


# Tokens at the borders of a workgroup's share of the sort, in two passes.
@pytest.mark.parametrize("n", [4096, 4097, 5119, 5120, 5121, 131072, 131073])
def test_vjp_borders_of_the_sort(n):
    run_vjp(n, 1000, 4, "float32", False, "uniform")


# Few tokens, in one launch.
@pytest.mark.parametrize("kind", ["uniform", "one", "none", "zipf"])
@pytest.mark.parametrize("D,dtype,norm", [(2048, "float32", True), (2047, "bfloat16", True), (1001, "float32", False),
                                          (513, "bfloat16", False), (3, "float32", True)])
@pytest.mark.parametrize("n", [1, 31, 32, 33, 63, 64, 65])
def test_vjp_few(n, D, dtype, norm, kind):
    run_vjp(n, 90, D, dtype, norm, kind)
    run_vjp(n, 40000 if D == 3 else 700, D, dtype, norm, kind, accumulate=n % 2 == 0)


def test_places_past_32_bits():
    # Rows and table of more than 2^31 elements; the gradient is of the last 500 tokens alone.
    torch = need_gpu()
    import burn_dragon_amd as bd
    n, D, last = (1 << 20) + 77, 2048, 500
    V = n + 5
    gen = torch.Generator(device="cuda").manual_seed(4)
    tokens = torch.randint(0, V, (n,), generator=gen, device="cuda", dtype=torch.int32)
    tokens[-last::2] = torch.randint(V - 40, V, (last // 2,), generator=gen, device="cuda", dtype=torch.int32)
    table = torch.empty(V, D, device="cuda", dtype=torch.bfloat16).normal_(generator=gen)
    announce("embed past 2^31 elements")
    out = bd.embed_tokens(tokens, table)
    assert torch.equal(out[-last:], table[tokens[-last:].long()])
    grad = out.zero_()
    grad[-last:].normal_(generator=gen)
    del table
    announce("embed vjp past 2^31 elements")
    got = bd.embed_tokens_vjp(grad, tokens, torch.empty(V, D, device="cuda", dtype=torch.bfloat16))
    want = torch.zeros(V, D, device="cuda", dtype=torch.float32).index_add_(0, tokens[-last:].long(), grad[-last:].float())
    # A rounding to bf16; f32 sums of up to 500 rows in another order.
    rows = tokens[-last:].long().unique()
    assert float((got[rows].float() - want[rows]).abs().max()) <= (2.0 ** -8 + 1e-4) * float(want[rows].abs().max())
    got[rows] = 0
    assert not got.any()
