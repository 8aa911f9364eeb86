"""sample_tokens against the definition in 64 bits (tests/sampleref.py).

Tokens are whole numbers and have to be equal: the kernel's sums are exact in
units of 2^-42 of the largest weight, so one differs from the oracle's only
where a border falls within V units of a sum, a chance of less than
V^2 * 2^-42 a row (2^-8 at V = 131072 if every weight were as large as the
largest, and then the borders are whole units apart: the cases' inputs are
fixed).  The log-probability is computed in 64 bits and rounded once: half a
step of f32, and the sum's V * 2^-43 of its units, 2^-24 + V * 2^-43 relative
to max(1, |logprob|)."""
import math

import numpy as np
import pytest

from tests import sampleref
from tests.gpu_util import announce, need_gpu

pytestmark = pytest.mark.gpu


def logits_of(rng, rows, V, kind):
    if kind == "normal":
        return rng.standard_normal((rows, V)) * 3
    if kind == "peaked":
        x = rng.standard_normal((rows, V)) * 2
        for r in range(rows):
            x[r, rng.integers(0, V, 8)] += 6 + 3 * rng.random(8)
        return x
    if kind == "ties":  # a few values, many times each
        return np.round(rng.standard_normal((rows, V)) * 1.5) / 2
    if kind == "equal":
        return np.full((rows, V), -3.25)
    if kind == "masked":
        x = rng.standard_normal((rows, V)) * 3
        x[rng.random((rows, V)) < 0.9] = -np.inf
        x[:, V // 2] = 0.5
        return x
    if kind == "lowest":  # masked by the type's lowest value
        x = rng.standard_normal((rows, V)) * 3
        x[rng.random((rows, V)) < 0.9] = -sampleref.F32_MAX
        return x
    if kind == "steep":  # weights past 2^-42, far apart
        return rng.standard_normal((rows, V)) * 40
    raise ValueError(kind)


CUTS = {
    "none": {},
    "k": dict(top_k=20),
    "k_large": dict(top_k=700),
    "p": dict(top_p=0.9),
    "p_small": dict(top_p=0.05),
    "p_near_1": dict(top_p=0.999),
    "m": dict(min_p=0.1),
    "kp": dict(top_k=50, top_p=0.8),
    "all": dict(top_k=100, top_p=0.95, min_p=0.02, temperature=0.7),
    "hot": dict(temperature=3.0, top_p=0.7),
    "cold": dict(temperature=0.05, top_k=5),
}


def run(torch, bd, x, u, dtype=None, **kw):
    t = torch.from_numpy(np.ascontiguousarray(x, dtype=np.float32)).cuda()
    if dtype is not None:
        t = t.to(dtype)
    out = bd.sample_tokens(t, torch.from_numpy(np.asarray(u, np.float32)).cuda(), want_logprob=True, **kw)
    torch.cuda.synchronize()
    return t.float().cpu().numpy(), out.tokens.cpu().numpy(), out.logprob.cpu().numpy()


def check(torch, bd, x, u, dtype=None, settings=None, **kw):
    seen, tokens, logprob = run(torch, bd, x, u, dtype, **(settings or kw))
    want, want_lp = sampleref.sample(seen, np.asarray(u, np.float32), **kw)
    assert np.array_equal(tokens, want), (tokens, want)
    tol = (2.0 ** -24 + seen.shape[1] * 2.0 ** -43) * np.maximum(1.0, np.abs(want_lp))
    fine = np.isfinite(want_lp)
    assert np.array_equal(fine, np.isfinite(logprob))
    assert np.all(np.abs(logprob[fine] - want_lp[fine]) <= tol[fine])


SIZES = [1, 2, 5, 64, 255, 256, 257, 1000, 1024, 1025, 4096, 4099, 8192, 8195, 16384, 16390, 32768,
         32769, 50001, 131072]


@pytest.mark.parametrize("cut", sorted(CUTS))
@pytest.mark.parametrize("V", SIZES)
def test_cuts_at_every_size(V, cut):
    torch = need_gpu()
    import burn_dragon_amd as bd
    rng = np.random.default_rng(V * 31 + len(cut))
    rows = 5 if V < 10000 else 3
    announce("sample", V, cut)
    for kind in ("normal", "peaked"):
        u = rng.random(rows).astype(np.float32)
        check(torch, bd, logits_of(rng, rows, V, kind).astype(np.float32), u, **CUTS[cut])


@pytest.mark.parametrize("kind", ["ties", "equal", "masked", "lowest", "steep"])
@pytest.mark.parametrize("V", [7, 256, 1000, 9000, 20000, 70001])
def test_ties_masks_and_steep_rows(V, kind):
    # Cuts fall among equal logits: those of the lowest indices stay.
    torch = need_gpu()
    import burn_dragon_amd as bd
    rng = np.random.default_rng(V)
    for cut in ("none", "k", "k_large", "p", "kp", "m", "cold", "hot"):
        announce("sample", kind, V, cut)
        u = rng.random(3).astype(np.float32)
        check(torch, bd, logits_of(rng, 3, V, kind).astype(np.float32), u, **CUTS[cut])


@pytest.mark.parametrize("V", [6, 300, 5000, 40000])
def test_bf16_logits_and_every_token_of_a_small_kept_set(V):
    torch = need_gpu()
    import burn_dragon_amd as bd
    rng = np.random.default_rng(V + 1)
    x = logits_of(rng, 1, V, "normal").astype(np.float32)
    u = np.linspace(0, 1, 33, endpoint=False).astype(np.float32)
    announce("sample bf16", V)
    check(torch, bd, np.repeat(x, 33, 0), u, torch.bfloat16, top_k=5, temperature=2.0)


@pytest.mark.parametrize("V", [10, 3000, 40000])
def test_nan_infinities_zeros_and_empty_rows(V):
    torch = need_gpu()
    import burn_dragon_amd as bd
    rng = np.random.default_rng(V + 2)
    x = logits_of(rng, 10, V, "normal").astype(np.float32)
    x[0] = -np.inf                       # nothing to draw
    x[1] = np.nan
    x[2, ::2] = np.nan                   # NaN in masked places
    x[3, [1, V - 1]] = np.inf            # two infinite ones share the draw
    x[4] = -np.inf
    x[4, V - 1] = -7.0                   # one left
    x[5] = -sampleref.F32_MAX            # all at the lowest value
    x[6] = np.where(np.arange(V) % 2, 0.0, -0.0)  # equal zeros of both signs
    x[7, 3] = sampleref.F32_MAX
    x[8] = np.nan
    x[8, V // 2] = np.inf
    u = np.array([0.5, 0.5, 0.3, 0.6, 0.99, 0.7, 0.45, 0.2, 0.1, 0.0], np.float32)
    for kw in ({}, dict(top_k=4), dict(top_p=0.6), dict(top_k=3, top_p=0.5, min_p=0.3), dict(temperature=0.0),
               dict(top_k=1)):
        announce("sample special", V, kw)
        check(torch, bd, x, u, **kw)


@pytest.mark.parametrize("low", [-sampleref.F32_MAX, -3e37])
def test_only_lowest_values_beside_masked_stretches(low):
    # A stretch of 8192 without a logit beside others at the lowest value: it
    # weighs nothing and is not read.
    torch = need_gpu()
    import burn_dragon_amd as bd
    x = np.full((6, 40000), -np.inf, np.float32)
    x[:, 9000:9010] = low
    x[:, 33000] = low
    u = np.array([0.0, 0.2, 0.4, 0.6, 0.8, 0.99], np.float32)
    for kw in ({}, dict(top_k=3), dict(top_k=700), dict(top_p=0.5), dict(min_p=0.5), dict(top_k=8, top_p=0.6)):
        announce("sample lowest", low, kw)
        for _ in range(2):  # the second call finds the first's scratch
            check(torch, bd, x, u, **kw)
        check(torch, bd, np.where(x == -np.inf, np.float32(1.0), x), u, **kw)


@pytest.mark.parametrize("V", [40, 2000, 60000])
def test_settings_one_a_row(V):
    # Greedy, uncut, cut and out-of-range rows side by side.
    torch = need_gpu()
    import burn_dragon_amd as bd
    rng = np.random.default_rng(V + 3)
    n = 12
    x = logits_of(rng, n, V, "peaked").astype(np.float32)
    u = rng.random(n).astype(np.float32)
    inf, nan = np.inf, np.nan
    host = dict(
        temperature=np.array([1, 0, -1, nan, 0.5, 2, 1, 1, 1, 1e-30, inf, 1], np.float32),
        top_k=np.array([0, 5, 5, 5, 1, V, V + 9, -3, 7, 0, 30, 0], np.int32),
        top_p=np.array([1, 0.5, 1, 1, 1, 0.9, 1.5, nan, -1, 1, 0.5, 0], np.float32),
        min_p=np.array([0, 0, 0, 0, 0, 0.2, nan, -1, 0, 0, 0, 2], np.float32))
    dev = {k: torch.from_numpy(v).cuda() for k, v in host.items()}
    seen = dict(host)
    seen["top_p"] = np.where(np.isnan(host["top_p"]), 1.0, host["top_p"]).astype(np.float32)
    seen["min_p"] = np.where(np.isnan(host["min_p"]), 0.0, host["min_p"]).astype(np.float32)
    announce("sample rows", V)
    check(torch, bd, x, u, settings=dev, **seen)


@pytest.mark.parametrize("V", [20000, 131072, 300000])
def test_top_k_around_what_the_chunks_list(V):
    # Up to 256 a chunk go to its list: k about that, ties that overflow it,
    # rows with fewer logits than k.
    torch = need_gpu()
    import burn_dragon_amd as bd
    rng = np.random.default_rng(V)
    for k in (2, 63, 64, 65, 200, 255, 256, 257, 600):
        x = logits_of(rng, 4, V, "peaked").astype(np.float32)
        x[1] = np.round(x[1])                                   # hundreds of equal logits at the k-th
        x[2, rng.random(V) < 1 - 300 / V] = -np.inf             # about 300 logits
        x[3] = -np.inf
        x[3, rng.integers(0, V, 40)] = rng.standard_normal(40)  # fewer than k
        u = rng.random(4).astype(np.float32)
        for kw in (dict(top_k=k), dict(top_k=k, top_p=0.7), dict(top_k=k, min_p=0.05, top_p=0.99, temperature=1.5)):
            announce("sample lists", V, kw)
            check(torch, bd, x, u, **kw)


def test_random_numbers_at_the_ends():
    torch = need_gpu()
    import burn_dragon_amd as bd
    rng = np.random.default_rng(11)
    for V in (50, 20000, 40000):
        x = logits_of(rng, 6, V, "normal").astype(np.float32)
        u = np.array([0.0, 1 - 2.0 ** -24, 1.0, -0.5, np.nan, 7.0], np.float32)
        announce("sample ends", V)
        check(torch, bd, x, u, top_k=10)
        check(torch, bd, x, u)


def test_strided_rows_shared_rows_and_a_given_output():
    torch = need_gpu()
    import burn_dragon_amd as bd
    g = torch.Generator(device="cuda").manual_seed(3)
    full = torch.randn(4, 3, 1001, generator=g, device="cuda") * 3
    u = torch.rand(4, generator=g, device="cuda")
    announce("sample strided")
    out = torch.full((4,), -9, device="cuda", dtype=torch.int32)
    got = bd.sample_tokens(full[:, -1], u, top_k=9, out=out)
    assert got.tokens is out and got.logprob is None
    want, _ = sampleref.sample(full[:, -1].cpu().numpy(), u.cpu().numpy(), top_k=9)
    assert np.array_equal(out.cpu().numpy(), want)
    # the same logits for every row
    got = bd.sample_tokens(full[1, 1:2].expand(4, 1001), u, top_p=0.9)
    want, _ = sampleref.sample(np.repeat(full[1, 1:2].cpu().numpy(), 4, 0), u.cpu().numpy(), top_p=0.9)
    assert np.array_equal(got.tokens.cpu().numpy(), want)
    # vocabulary not contiguous, rows at odd addresses
    got = bd.sample_tokens(full.transpose(1, 2)[0].t(), u[:3])
    want, _ = sampleref.sample(full[0].cpu().numpy(), u[:3].cpu().numpy())
    assert np.array_equal(got.tokens.cpu().numpy(), want)
    half = full.to(torch.bfloat16).view(-1)[1:1 + 3 * 999].view(3, 999)
    got = bd.sample_tokens(half, u[:3], min_p=0.05)
    want, _ = sampleref.sample(half.float().cpu().numpy(), u[:3].cpu().numpy(), min_p=0.05)
    assert np.array_equal(got.tokens.cpu().numpy(), want)


def test_offsets_past_32_bits():
    # Rows 2^28 elements apart, the last 2^31 elements (8 GiB) from the first.
    torch = need_gpu()
    import burn_dragon_amd as bd
    V, stride, rows = 40000, 1 << 28, 9
    store = torch.empty((rows - 1) * stride + V, device="cuda")
    x = store.as_strided((rows, V), (stride, 1))
    x.normal_()
    u = torch.rand(rows, device="cuda")
    announce("sample far rows")
    for view in (x, x[:, :1000]):
        got = bd.sample_tokens(view, u, top_k=40, top_p=0.9)
        want, _ = sampleref.sample(view.cpu().numpy(), u.cpu().numpy(), top_k=40, top_p=0.9)
        assert np.array_equal(got.tokens.cpu().numpy(), want)


def test_the_largest_vocabulary_and_many_rows():
    torch = need_gpu()
    import burn_dragon_amd as bd
    rng = np.random.default_rng(5)
    for rows, V in ((2, 1 << 20), (1100, 33000), (5000, 300)):
        x = (rng.standard_normal((rows, V), dtype=np.float32) * 2)
        u = rng.random(rows).astype(np.float32)
        announce("sample many", rows, V)
        t = torch.from_numpy(x).cuda()
        got = bd.sample_tokens(t, torch.from_numpy(u).cuda(), top_k=60, top_p=0.9)
        check_rows = np.r_[0:3, rows // 2, rows - 2:rows] if rows > 6 else np.arange(rows)
        want, _ = sampleref.sample(x[check_rows], u[check_rows], top_k=60, top_p=0.9)
        assert np.array_equal(got.tokens.cpu().numpy()[check_rows], want)


def test_rows_do_not_depend_on_their_batch():
    torch = need_gpu()
    import burn_dragon_amd as bd
    g = torch.Generator(device="cuda").manual_seed(9)
    for V in (700, 12000, 45000):
        x = torch.randn(20, V, generator=g, device="cuda") * 2
        u = torch.rand(20, generator=g, device="cuda")
        announce("sample batch", V)
        whole = bd.sample_tokens(x, u, top_p=0.95, want_logprob=True)
        for i in (0, 7, 19):
            one = bd.sample_tokens(x[i:i + 1], u[i:i + 1], top_p=0.95, want_logprob=True)
            assert torch.equal(one.tokens[0], whole.tokens[i]) and torch.equal(one.logprob[0], whole.logprob[i])


def test_draws_follow_the_distribution():
    # 200000 draws of 8 tokens: a count's deviation is below 5 standard deviations
    # (a chance of 6e-7 each; the random numbers are fixed).
    torch = need_gpu()
    import burn_dragon_amd as bd
    n = 200000
    x = torch.tensor([0.0, 1.0, 2.0, -1.0, 0.5, -math.inf, 1.5, 3.0], device="cuda")
    u = torch.rand(n, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
    announce("sample distribution")
    got = bd.sample_tokens(x.expand(n, 8), u, temperature=1.3).tokens.cpu().numpy()
    p = np.exp(x.cpu().numpy().astype(np.float64) / 1.3)
    p /= p.sum()
    counts = np.bincount(got, minlength=8)
    assert counts[5] == 0
    assert np.all(np.abs(counts - n * p) <= 5 * np.sqrt(n * p * (1 - p)))


@pytest.mark.parametrize("V", [500, 50000])
def test_captured_into_a_graph(V):
    torch = need_gpu()
    import burn_dragon_amd as bd
    g = torch.Generator(device="cuda").manual_seed(4)
    x = torch.randn(6, V, generator=g, device="cuda") * 3
    u = torch.rand(6, generator=g, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        bd.sample_tokens(x, u, top_k=50, top_p=0.9)  # the stream's scratch
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    announce("sample graph", V)
    with torch.cuda.graph(graph, stream=side):
        out = bd.sample_tokens(x, u, top_k=50, top_p=0.9, want_logprob=True)
    for i in range(4):
        x.normal_(generator=g).mul_(3)
        u.uniform_(generator=g)
        want = bd.sample_tokens(x, u, top_k=50, top_p=0.9, want_logprob=True)
        torch.cuda.synchronize()
        graph.replay()
        with torch.cuda.stream(side):
            bd.sample_tokens(x * 2, u, top_p=0.5)  # eager work on the capturing stream
        torch.cuda.synchronize()
        assert torch.equal(out.tokens, want.tokens) and torch.equal(out.logprob, want.logprob), i


def test_two_streams_at_once():
    torch = need_gpu()
    import burn_dragon_amd as bd
    g = torch.Generator(device="cuda").manual_seed(6)
    xs = [torch.randn(40, 60000 + i, generator=g, device="cuda") * 2 for i in range(2)]
    u = torch.rand(40, generator=g, device="cuda")
    want = [bd.sample_tokens(x, u, top_p=0.9).tokens.clone() for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    got = [[], []]
    announce("sample two streams")
    for _ in range(5):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(bd.sample_tokens(xs[i], u, top_p=0.9).tokens)
    torch.cuda.synchronize()
    assert all(torch.equal(t, w) for w, ts in zip(want, got) for t in ts)


def test_unsupported_and_refused():
    torch = need_gpu()
    import burn_dragon_amd as bd
    from burn_dragon_amd import _lib
    x = torch.zeros(2, 8, device="cuda")
    u = torch.zeros(2, device="cuda")
    assert bd.sample_tokens(x.double(), u) is None
    assert bd.sample_tokens(x.half(), u) is None
    assert bd.sample_tokens(x[0], u) is None
    assert bd.sample_tokens(x[:, :0], u) is None
    assert bd.sample_tokens(x.cpu(), u) is None
    assert bd.sample_tokens(torch.zeros(1, (1 << 20) + 1, device="cuda"), u[:1]) is None
    for bad in (dict(uniform=u[:1]), dict(uniform=u.double()), dict(temperature=u[:1]),
                dict(top_k=u), dict(top_p=u.double()), dict(min_p=u.cpu()),
                dict(out=torch.zeros(2, device="cuda"))):
        with pytest.raises(ValueError):
            bd.sample_tokens(x, bad.pop("uniform", u), **bad)
    for bad in (dict(temperature=-1.0), dict(temperature=math.nan), dict(top_p=1.5), dict(top_p=-0.1),
                dict(min_p=2.0), dict(top_k=-1), dict(temperature=math.inf)):
        with pytest.raises(_lib.BdhError):
            bd.sample_tokens(x, u, **bad)


@pytest.mark.parametrize("V,rows", [(1 << 20, 300), (400000, 700), (20000, 2100)])
def test_rows_in_groups(V, rows):
    # Long rows go through the scratch some at a time: one row of logits, shared.
    torch = need_gpu()
    import burn_dragon_amd as bd
    rng = np.random.default_rng(V)
    x = (rng.standard_normal((1, V)) * 3).astype(np.float32)
    u = rng.random(rows).astype(np.float32)
    announce("sampling in groups", V, rows)
    t = torch.from_numpy(x).cuda().expand(rows, V)
    got = bd.sample_tokens(t, torch.from_numpy(u).cuda(), top_p=0.9).tokens.cpu().numpy()
    some = np.r_[0:3, 127:130, 255:258, rows - 2:rows]
    want, _ = sampleref.sample(np.repeat(x, len(some), 0), u[some], top_p=0.9)
    assert np.array_equal(got[some], want)
    one = bd.sample_tokens(t[:1].expand(100, V), torch.from_numpy(u[-100:]).cuda(), top_p=0.9).tokens
    assert np.array_equal(got[-100:], one.cpu().numpy())


@pytest.mark.parametrize("V,spread", [(60000, 0.02), (131072, 0.2), (131072, 0.02), (200000, 0.7)])
def test_flat_rows_with_many_candidates(V, spread):
    # A cut's bin holds more than a workgroup's list, or than the scratch's.
    torch = need_gpu()
    import burn_dragon_amd as bd
    rng = np.random.default_rng(V)
    for kw in (dict(top_p=0.9), dict(min_p=0.05 if spread > 0.5 else 0.98), dict(top_k=2000),
               dict(top_k=20000, top_p=0.5), dict(top_k=V - 5, top_p=0.3, min_p=0.5)):
        announce("flat rows", V, spread, kw)
        check(torch, bd, rng.standard_normal((3, V)) * spread, rng.random(3), **kw)


@pytest.mark.parametrize("V", [40, 3000, 40000])
@pytest.mark.parametrize("temperature,scale", [(1e31, 1e31), (1e33, 2e33), (1e37, 2e37), (3e38, 6e37),
                                               (math.inf, 6e37), (1e-28, 2e-28), (1e-33, 3e-33), (1e-37, 3e-37),
                                               (1e-42, 2e-42), (1e-45, 6e-45)])
def test_temperatures_from_the_least_to_the_largest(V, temperature, scale):
    # Logits as large as the temperature: their weights are those of ordinary rows.
    torch = need_gpu()
    import burn_dragon_amd as bd
    rng = np.random.default_rng(V + 17)
    x = np.clip(rng.standard_normal((4, V)) * scale, -sampleref.F32_MAX, sampleref.F32_MAX).astype(np.float32)
    u = rng.random(4).astype(np.float32)
    rows = np.full(4, temperature, np.float32)
    for cut in ({}, dict(top_k=20), dict(top_k=V // 2), dict(top_p=0.7), dict(top_k=V // 3, top_p=0.8, min_p=0.05)):
        announce("sample hot", V, temperature, cut)
        check(torch, bd, x, u, settings=dict(temperature=torch.from_numpy(rows).cuda(), **cut), temperature=rows, **cut)


@pytest.mark.parametrize("V", [40, 3000, 40000])
@pytest.mark.parametrize("offset,temperature", [(1e5, 0.1), (-1e5, 1.0), (3e7, 1.0), (-3e7, 0.3), (2e8, 1.0), (1e9, 9.0)])
def test_logits_far_from_zero(V, offset, temperature):
    # Neighbouring values of f32 are up to 42 octaves of weight apart: bins are off
    # by more than their width there, and have to hold what is drawn all the same.
    torch = need_gpu()
    import burn_dragon_amd as bd
    rng = np.random.default_rng(V + 23)
    x = (offset + rng.standard_normal((4, V)) * temperature * 6).astype(np.float32)
    u = rng.random(4).astype(np.float32)
    for cut in ({}, dict(top_k=20), dict(top_k=V // 2), dict(top_p=0.7), dict(top_k=V // 3, top_p=0.8, min_p=1e-4)):
        announce("sample far from zero", V, offset, cut)
        check(torch, bd, x, u, temperature=temperature, **cut)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("rows,V", [(20000, 260), (4000, 1500), (1500, 16384), (600, 40001)])
def test_every_draw_finds_its_token(rows, V, dtype):
    # A weight is computed at several places, which have to agree to the unit: a
    # draw at the far end of the sum still ends in a token that is kept.
    torch = need_gpu()
    import burn_dragon_amd as bd
    g = torch.Generator(device="cuda").manual_seed(V)
    x = (torch.randn(rows, V, generator=g, device="cuda") * 5).to(getattr(torch, dtype))
    u = torch.rand(rows, generator=g, device="cuda")
    u[::2] = 1 - 2.0 ** -24
    temperature = 0.3 + torch.rand(rows, generator=g, device="cuda")
    out = torch.full((rows,), -9, dtype=torch.int32, device="cuda")
    for cut in ({}, dict(top_k=37), dict(top_k=700), dict(top_p=0.8), dict(min_p=0.01), dict(top_k=90, top_p=0.9)):
        announce("sample every draw", rows, V, dtype, cut)
        out.fill_(-9)
        got = bd.sample_tokens(x, u, temperature=temperature, out=out, want_logprob=True, **cut)
        torch.cuda.synchronize()
        assert int(out.min()) >= 0 and int(out.max()) < V
        t = (x.gather(1, out[:, None].long())[:, 0].double() - x.amax(1).double()) / temperature.double()
        # kept: by min-p from its threshold up (half a step of f32 off at most), else from 2^-42 up
        least = math.log(0.01) if "min_p" in cut else -42 * math.log(2)
        assert bool((t >= least - 1e-6).all()) and bool((got.logprob >= t - 20).all()) and bool((got.logprob <= 0).all())
