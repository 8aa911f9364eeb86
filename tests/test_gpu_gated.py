"""gated_block and gated_block_vjp against the formula in 64 bits (bounds:
tests/trainref.py)."""
import numpy as np
import pytest

from tests import trainref as R
from tests.gpu_util import announce, need_gpu

pytestmark = pytest.mark.gpu

BF16 = 2.0 ** -8   # half a step of bf16, relative


def make(torch, B, T, H, D, N, context, masked=False, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + B * 3 + T * 5 + H * 7 + D * 11 + N)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    b = torch.bfloat16
    return dict(x=rnd(B, T, D).to(b), up=(rnd(H, D, N) / D ** 0.5).to(b), gate=(rnd(H, D, N) / D ** 0.5).to(b),
                c=rnd(B, H, T, D).to(b) if context else None, g=rnd(B, T, H * N).to(b),
                mask=torch.where(rnd(N) > 0, rnd(N).abs(), 0.0) if masked else None)


def f64(t):
    return t.cpu().double().numpy()


def plain(t):
    """x [M, D], c [H, M, D], up, gate, g [H, M, N], mask."""
    B, T, D = t["x"].shape
    H, _, N = t["up"].shape
    x = f64(t["x"]).reshape(B * T, D)
    c = np.stack([x] * H) if t["c"] is None else f64(t["c"]).transpose(1, 0, 2, 3).reshape(H, B * T, D)
    g = f64(t["g"]).reshape(B * T, H, N).transpose(1, 0, 2)
    m = np.ones(N) if t["mask"] is None else f64(t["mask"])
    return x, c, f64(t["up"]), f64(t["gate"]), g, m


def heads(t, H):
    """[B, T, H * N] or [B, T, H, N] -> [H, M, N]."""
    B, T = t.shape[:2]
    return f64(t).reshape(B * T, H, -1).transpose(1, 0, 2)


def check(got, want, off, name):
    bound = off + BF16 * (np.abs(want) + off) + 1e-38
    got = got.reshape(want.shape)
    d = np.abs(got - want)
    assert np.all(d <= bound), (name, float(d.max()), float((d / bound).max()), np.argwhere(~(d <= bound))[:4].tolist())


def check_grads(d, want, t):
    B, T, D = t["x"].shape
    H = t["up"].shape[0]
    if t["c"] is None:
        v, o = want["current"]
        v, o = v + want["context"][0].sum(0), o + want["context"][1].sum(0) + 2 * H * R.U * np.abs(want["context"][0]).sum(0)
        check(f64(d.current), v, o, "current")
        assert d.context is None
    else:
        check(f64(d.current), *want["current"], "current")
        check(f64(d.context).transpose(1, 0, 2, 3), *want["context"], "context")
    check(f64(d.up), *want["up"], "up")
    check(f64(d.gate), *want["gate"], "gate")


def run(B, T, H, D, N, act="relu", context=True, th=0.0, masked=False, seed=0, t=None):
    torch = need_gpu()
    import burn_dragon_amd as bd
    t = t or make(torch, B, T, H, D, N, context, masked, seed)
    how = dict(activation=act, relu_threshold=th, latent_mask=t["mask"])
    w = bd.GatedWeights(t["up"], t["gate"])
    announce("gated", B, T, H, D, N, act, context, th, masked)
    out = bd.gated_block(t["x"], w, t["c"], **how)
    both = bd.gated_block(t["x"], w, t["c"], save=True, **how)
    announce("gated vjp", B, T, H, D, N, act, context, th, masked)
    d = bd.gated_block_vjp(t["g"], t["x"], w, t["c"], **how)
    d8 = bd.gated_block_vjp(t["g"], t["x"], w, t["c"], saved=both.saved, **how)
    kept = [bd.restore_activations(c, dtype=torch.float32) for c in both.saved]
    torch.cuda.synchronize()
    assert out.saved is None and torch.equal(out.out, both.out)
    x, c, wu, wg, g, m = plain(t)
    p, q, op, oq = R.project(x, c, wu, wg, np.float32(th).astype(float))
    check(heads(out.out, H), *R.forward(act, p, q, op, oq, m), "out")
    check_grads(d, R.backward(act, g, x, c, wu, wg, p, q, op, oq, m), t)
    # What was kept: the projections to half a step of e4m3, and of its least step far below the
    # block's largest (a power of two up to 2 * largest / 448, steps of 2^-10 of it).
    kept = [heads(k, H) for k in kept]
    for k, v, o in zip(kept, (p, q), (op, oq)):
        v = R.act("relu", v)[0] if act == "relu" else v
        top = np.pad(np.abs(v) + o, ((0, 0), (0, 0), (0, -N % 32))).reshape(*v.shape[:2], -1, 32).max(3)
        top = np.repeat(top, 32, 2)[:, :, :N]
        d_ = np.abs(k - v)
        assert np.all(d_ <= 2.0 ** -4 * (np.abs(v) + o) + o + top * 2 / 448 * 2.0 ** -10 + 1e-36), float(d_.max())
    # The backward at exactly those values.
    z = np.zeros_like(p)
    check_grads(d8, R.backward(act, g, x, c, wu, wg, *kept, z, z, m), t)


@pytest.mark.parametrize("act", ["relu", "silu", "gelu"])
@pytest.mark.parametrize("context", [True, False])
@pytest.mark.parametrize("B,T,H,D,N", [(1, 1, 1, 8, 8), (2, 3, 2, 40, 72), (1, 130, 1, 64, 256), (3, 77, 3, 200, 200),
                                       (2, 128, 1, 256, 128), (5, 1, 4, 264, 1000), (1, 300, 2, 32, 512)])
def test_shapes(B, T, H, D, N, context, act):
    run(B, T, H, D, N, act, context)


@pytest.mark.parametrize("T", [1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 129, 255, 257])
def test_lengths(T):
    run(2, T, 2, 64, 136, "silu", True)
    run(1, T, 1, 72, 64, "gelu", False)


@pytest.mark.parametrize("D", [8, 24, 32, 56, 248, 256, 264, 520])
@pytest.mark.parametrize("N", [8, 24, 32, 120, 128, 264])
def test_dims(D, N):
    run(2, 9, 2, D, N, "relu", True)


@pytest.mark.parametrize("th", [0.0, 1.5, -0.5])
@pytest.mark.parametrize("masked", [False, True])
def test_threshold_and_mask(th, masked):
    run(2, 40, 2, 64, 200, "relu", True, th, masked)
    run(1, 70, 1, 64, 64, "relu", False, th, masked)


@pytest.mark.parametrize("B,T", [(64, 1), (33, 3), (1, 2000), (700, 3)])
def test_many_tokens(B, T):
    run(B, T, 1, 32, 64, "silu", True)
    run(B, T, 2, 16, 40, "relu", True)


def test_deep_and_wide():
    run(1, 20, 1, 2048, 64, "silu", False)
    run(1, 5, 1, 40, 8200, "gelu", False)


# Without a context these calls go in tiles of 192 or 256 tokens (some kinds in 128).
@pytest.mark.parametrize("T,D,N,act", [(1499, 520, 4088, "relu"), (1499, 1032, 4088, "gelu"), (1537, 2056, 4096, "silu"),
                                       (1001, 1048, 8184, "relu"), (1023, 1040, 8192, "silu"), (1023, 1040, 8192, "gelu")])
def test_larger_tiles(T, D, N, act):
    run(1, T, 1, D, N, act, False, 0.25 if act == "relu" else 0.0, act == "relu")


# More tiles of 128 by 128 than a chip has CUs, of few steps.
@pytest.mark.parametrize("act", ["relu", "silu", "gelu"])
@pytest.mark.parametrize("context", [False, True])
def test_many_tiles(act, context):
    run(1, 2055, 1, 72, 4104, act, context)


# The backward of saved values without the projections' gradients in memory begins at 2^23 of them.
@pytest.mark.parametrize("B,T,H,D,N,act,context,masked", [
    (3, 375, 1, 200, 7504, "relu", True, True), (1, 4097, 2, 72, 1032, "relu", True, False),
    (5, 411, 2, 256, 2056, "silu", False, False), (1, 1025, 1, 256, 8192, "gelu", True, False),
    (70, 61, 4, 8, 496, "relu", False, True), (2, 999, 3, 136, 1408, "silu", True, False)])
def test_many_latents(B, T, H, D, N, act, context, masked):
    assert B * T * H * N >= 1 << 23
    run(B, T, H, D, N, act, context, 0.5 if masked else 0.0, masked)


def test_differences():
    # <gradient, direction> against central differences of sum(g * out) in 64 bits.  The
    # gradients' bf16 (2^-7 of a term, twice) adds at random over thousands of terms, but is
    # counted in full.
    torch = need_gpu()
    import burn_dragon_amd as bd
    t = make(torch, 2, 9, 2, 24, 40, True)
    w = bd.GatedWeights(t["up"], t["gate"])
    announce("gated by differences")
    d = bd.gated_block_vjp(t["g"], t["x"], w, t["c"], activation="gelu")
    x, c, wu, wg, g, m = plain(t)
    got = (f64(d.current).reshape(x.shape), f64(d.context).transpose(1, 0, 2, 3).reshape(c.shape), f64(d.up), f64(d.gate))
    rng = np.random.default_rng(4)
    at = [x, c, wu, wg]
    for k in range(4):
        v = rng.standard_normal(at[k].shape)

        def f(s):
            a = list(at)
            a[k] = at[k] + s * v
            p, q, op, oq = R.project(*a, 0.0)
            return float((g * R.forward("gelu", p, q, op, oq, m)[0]).sum())
        slope = (f(1e-4) - f(-1e-4)) / 2e-4
        assert abs(float((got[k] * v).sum()) - slope) <= 2 * 2.0 ** -7 * float(np.abs(got[k] * v).sum()) + 1e-4


def test_infinities_and_nan_reach_their_own():
    # A NaN of one token: its row of out and gradients, and the weights' gradients; no other row.
    torch = need_gpu()
    import burn_dragon_amd as bd
    t = make(torch, 2, 70, 2, 64, 96, True)
    w = bd.GatedWeights(t["up"], t["gate"])
    for act in ("relu", "silu"):
        want = bd.gated_block(t["x"], w, t["c"], activation=act, save=True)
        dw = bd.gated_block_vjp(t["g"], t["x"], w, t["c"], saved=want.saved, activation=act)
        x = t["x"].clone()
        x[1, 3, 5] = float("nan")
        announce("gated with a NaN", act)
        out = bd.gated_block(x, w, t["c"], activation=act, save=True)
        d = bd.gated_block_vjp(t["g"], x, w, t["c"], saved=out.saved, activation=act)
        d2 = bd.gated_block_vjp(t["g"], x, w, t["c"], activation=act)
        torch.cuda.synchronize()
        rows = torch.ones(2, 70, dtype=torch.bool, device="cuda")
        rows[1, 3] = False
        if act == "silu":
            assert out.out[1, 3].isnan().all()
        else:
            assert out.out[1, 3].isnan().any()
        assert torch.equal(out.out[rows], want.out[rows])
        assert torch.equal(d.current[rows], dw.current[rows]) and not d2.current[rows].isnan().any()
        assert d.up.isnan().any() and d2.up.isnan().any()


def test_rows_do_not_depend_on_the_batch_around_them():
    torch = need_gpu()
    import burn_dragon_amd as bd
    t = make(torch, 3, 100, 2, 64, 96, True)
    w = bd.GatedWeights(t["up"], t["gate"])
    announce("gated, sequences alone")
    out = bd.gated_block(t["x"], w, t["c"], save=True)
    for b in range(3):
        one = bd.gated_block(t["x"][b:b + 1], w, t["c"][b:b + 1], save=True)
        assert torch.equal(one.out, out.out[b:b + 1])
        assert torch.equal(one.saved.up.codes, out.saved.up.codes[b:b + 1])


def test_strides_streams_and_graph():
    torch = need_gpu()
    import burn_dragon_amd as bd
    t = make(torch, 3, 90, 2, 64, 96, True)
    w = bd.GatedWeights(t["up"], t["gate"])

    def step(t, w):
        o = bd.gated_block(t["x"], w, t["c"], save=True)
        d = bd.gated_block_vjp(t["g"], t["x"], w, t["c"], saved=o.saved)
        return (o.out, *d, *bd.gated_block_vjp(t["g"], t["x"], w, t["c"]))
    want = step(t, w)
    # Views that lie apart or at odd offsets.
    apart = dict(t)
    apart["x"] = torch.cat([t["x"], t["x"]], 2)[:, :, :64]
    apart["c"] = t["c"].transpose(1, 2).contiguous().transpose(1, 2)
    odd = torch.empty(t["g"].numel() + 1, device="cuda", dtype=torch.bfloat16)[1:].view_as(t["g"])
    apart["g"] = odd.copy_(t["g"])
    announce("gated with strides")
    for a, b in zip(want, step(apart, bd.GatedWeights(t["up"].transpose(1, 2).contiguous().transpose(1, 2), w.gate))):
        assert torch.equal(a, b)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    announce("gated on two streams")
    for s in streams:
        with torch.cuda.stream(s):
            got.append([step(t, w) for _ in range(2)])
    torch.cuda.synchronize()
    for o in got[0] + got[1]:
        assert all(torch.equal(a, b) for a, b in zip(want, o))
    announce("gated captured")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=streams[0]):
        held = step(t, w)
    for k in range(3):
        for name, v in make(torch, 3, 90, 2, 64, 96, True, seed=100 + k).items():
            if v is not None:
                t[name].copy_(v)
        graph.replay()
        eager = step(t, w)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, eager))
    del graph
    for s in streams:
        bd.release_stream_scratch(s)


def test_refusals():
    torch = need_gpu()
    import burn_dragon_amd as bd
    t = make(torch, 2, 5, 2, 32, 40, True)
    w = bd.GatedWeights(t["up"], t["gate"])
    o = bd.gated_block(t["x"], w, t["c"], save=True)
    assert bd.gated_block(t["x"].float(), w, t["c"]) is None
    assert bd.gated_block(t["x"][:, :0], w, t["c"][:, :, :0]) is None
    assert bd.gated_block(t["x"][:, :, :28], bd.GatedWeights(t["up"][:, :28], t["gate"][:, :28])) is None
    assert bd.gated_block(t["x"], bd.GatedWeights(t["up"][:, :, :36], t["gate"][:, :, :36])) is None
    assert bd.gated_block_vjp(t["g"].float(), t["x"], w, t["c"]) is None
    ones = torch.ones(40, device="cuda")
    for call in (lambda: bd.gated_block(t["x"], w, t["c"], activation="tanh"),
                 lambda: bd.gated_block(t["x"], w, t["c"], activation="silu", relu_threshold=1.0),
                 lambda: bd.gated_block(t["x"], w, t["c"], activation="gelu", latent_mask=ones),
                 lambda: bd.gated_block(t["x"], w, t["c"], latent_mask=ones[:39]),
                 lambda: bd.gated_block(t["x"], w, t["c"], latent_mask=ones.cpu()),
                 lambda: bd.gated_block(t["x"], w, t["c"][:1]),
                 lambda: bd.gated_block(t["x"][:, :, :24], w),
                 lambda: bd.gated_block_vjp(t["g"][:1], t["x"], w, t["c"]),
                 lambda: bd.gated_block_vjp(t["g"], t["x"], w, t["c"], saved=bd.GatedSaved(o.saved.up, bd.ActivationCheckpoint(
                     o.saved.gate.codes[:1], o.saved.gate.scales)))):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(Exception, match="finite"):
        bd.gated_block(t["x"], w, t["c"], relu_threshold=float("nan"))


def test_places_past_32_bits():
    # 2.15e9 latents; the gradient is of the last 300 tokens alone, so the calls on these
    # alone give the same.  (Other tiles and parts: two roundings to bf16 of sums in another order.)
    torch = need_gpu()
    import burn_dragon_amd as bd
    T, D, N, last = 131104, 8, 16400, 300
    assert T * N > 1 << 31
    gen = torch.Generator(device="cuda").manual_seed(3)
    rnd = lambda *s: torch.randn(*s, generator=gen, device="cuda").to(torch.bfloat16)  # noqa: E731
    x, c = rnd(1, T, D), rnd(1, 1, T, D)
    w = bd.GatedWeights(rnd(1, D, N), rnd(1, D, N))
    g = torch.zeros(1, T, N, device="cuda", dtype=torch.bfloat16)
    g[:, -last:] = rnd(1, last, N)
    announce("gated past 2^31 latents")
    o = bd.gated_block(x, w, c, save=True)
    few = bd.gated_block(x[:, -last:], w, c[:, :, -last:], save=True)
    assert torch.equal(o.out[:, -last:], few.out)
    for a, b in zip(o.saved, few.saved):
        assert torch.equal(a.codes[:, -last:], b.codes) and torch.equal(a.scales[:, -last:], b.scales)
    for saved, few_saved in ((o.saved, few.saved), (None, None)):
        announce("gated vjp past 2^31 latents", saved is not None)
        d = bd.gated_block_vjp(g, x, w, c, saved=saved)
        e = bd.gated_block_vjp(g[:, -last:], x[:, -last:], w, c[:, :, -last:], saved=few_saved)
        assert not d.current[:, :-last].any() and not d.context[:, :, :-last].any()
        for a, b in ((d.current[:, -last:], e.current), (d.context[:, :, -last:], e.context), (d.up, e.up), (d.gate, e.gate)):
            a, b = a.double(), b.double()
            assert float((a - b).norm()) <= 2.0 ** -7 * float(b.norm())
