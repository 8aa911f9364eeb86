"""apply_adapters against the formula in 64 bits.

Bound of an element, with P = scale |hidden| |A|^T |B|^T, the same products
of absolute values: an f32 operand of a product is held to 2^-24 of it (three
bf16 parts of 2^-8 each), bf16 calls hold the values between the two products
to 2^-16 (two parts); each of the up to 3 (D + R) terms of a sum, and a dozen
steps beside them, rounds by a step (2^-23) of what is summed; the result rounds
once to its type, by half a step, eps / 2:
    |error| <= P (2^-16 [bf16] + (3 D + 3 R + 16) 2^-23) + |out| eps / 2."""
import numpy as np
import pytest

from tests.gpu_util import announce, need_gpu

pytestmark = pytest.mark.gpu


def make(torch, B, T, D, V, R, n, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + B * 7 + T * 5 + D * 3 + V + R)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    return (rnd(B, T, V).to(dtype), rnd(B, T, D).to(dtype),
            (rnd(n, R, D) / D ** 0.5).to(torch.bfloat16), (rnd(n, V, R) / R ** 0.5).to(torch.bfloat16),
            rnd(n).abs() + 0.5)


def check(torch, out, base, hidden, a, b, scale, ids):
    base, hidden, a, b, scale = (t.cpu().double().numpy() for t in (base, hidden, a, b, scale))
    B, T, D = hidden.shape
    R = a.shape[1]
    eps = torch.finfo(out.dtype).eps
    got = out.cpu().double().numpy()
    for i, id_ in enumerate(ids.tolist()):
        if not 0 <= id_ < a.shape[0]:
            assert np.array_equal(got[i], base[i]), i
            continue
        want = base[i] + scale[id_] * (hidden[i] @ a[id_].T) @ b[id_].T
        P = scale[id_] * (np.abs(hidden[i]) @ np.abs(a[id_]).T) @ np.abs(b[id_]).T
        parts = 2.0 ** -16 if eps > 1e-3 else 0.0
        bound = P * (parts + (3 * D + 3 * R + 16) * 2.0 ** -23) + np.abs(want) * eps / 2 + 1e-38
        off = np.abs(got[i] - want)
        assert np.all(off <= bound), (i, float(off.max()), float((off / bound).max()))


def run(B, T, D, V, R, n, dtype, ids, in_place=False):
    torch = need_gpu()
    import burn_dragon_amd as bd
    dtype = getattr(torch, dtype)
    base, hidden, a, b, scale = make(torch, B, T, D, V, R, n, dtype)
    ids = torch.tensor(ids, dtype=torch.int32, device="cuda")
    announce("adapters", B, T, D, V, R, n, dtype, in_place)
    kept = base.clone()
    out = bd.apply_adapters(base, hidden, bd.AdapterSet(a, b, scale), ids, out=base if in_place else None)
    torch.cuda.synchronize()
    assert (out is base) if in_place else torch.equal(base, kept)
    check(torch, out, kept, hidden, a, b, scale, ids)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("T", [1, 2, 15, 16, 17, 63, 65, 130])
@pytest.mark.parametrize("D,V,R", [(256, 256, 16), (64, 1000, 8), (33, 257, 3), (1000, 65, 100), (1, 1, 1),
                                   (128, 515, 32), (7, 2050, 17), (520, 300, 64), (96, 4100, 128)])
def test_sizes(T, D, V, R, dtype):
    run(3, T, D, V, R, 4, dtype, [2, 0, 3])


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("T", [1, 3, 40])
@pytest.mark.parametrize("name,ids", [
    ("none", [-1] * 5), ("out_of_range", [7, -5, 1, 2147483647, -2147483648]), ("all_one", [1] * 29),
    ("mixed", [0, 1, -1, 0, 1, 1, 0, 2, 0, 0, 0, 0, 0, 0, -1, 0, 0, 0, 2, 1]),
])
def test_which_sequences_have_which_adapter(name, ids, T, dtype):
    run(len(ids), T, 48, 700, 12, 3, dtype, ids)
    run(len(ids), T, 48, 700, 12, 3, dtype, ids, in_place=True)


@pytest.mark.parametrize("B,n", [(300, 5), (513, 513)])
def test_many_sequences(B, n):
    ids = np.random.default_rng(B).integers(-1, n, B).tolist()
    run(B, 1, 64, 130, 16, n, "float32", ids)


def test_a_large_call():
    run(4, 300, 512, 9001, 64, 2, "bfloat16", [1, 0, -1, 1])


def test_tokens_one_a_sequence_in_two_dimensions_and_views():
    torch = need_gpu()
    import burn_dragon_amd as bd
    base, hidden, a, b, scale = make(torch, 6, 4, 40, 90, 8, 3, torch.float32)
    ids = torch.tensor([0, 2, 1, -1, 0, 2], dtype=torch.int32, device="cuda")
    s = bd.AdapterSet(a, b, scale)
    announce("adapters views")
    # rows that are not contiguous, weights given as views
    got = bd.apply_adapters(base[:, -1], hidden[:, -1], s, ids)
    check(torch, got[:, None], base[:, -1:], hidden[:, -1:], a, b, scale, ids)
    at = a.transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(bd.apply_adapters(base, hidden, bd.AdapterSet(at, b, scale), ids),
                       bd.apply_adapters(base, hidden, s, ids))


def test_unaligned_memory_and_borders():
    # Tensors one element into their memory; the elements around out stay.
    torch = need_gpu()
    import burn_dragon_amd as bd
    for dtype in (torch.float32, torch.bfloat16):
        for T in (1, 20):
            B, D, V, R, n = 3, 24, 71, 8, 2
            base, hidden, a, b, scale = make(torch, B, T, D, V, R, n, dtype)

            def shifted(t):
                flat = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")
                view = flat[1:].view(t.shape)
                view.copy_(t)
                return view
            ids = torch.tensor([1, 0, 1], dtype=torch.int32, device="cuda")
            room = torch.full((base.numel() + 9,), 5.0, dtype=dtype, device="cuda")
            out = room[1:1 + base.numel()].view(base.shape)
            announce("adapters unaligned", dtype, T)
            args = [shifted(t) for t in (base, hidden, a, b, scale)]
            assert bd.apply_adapters(args[0], args[1], bd.AdapterSet(*args[2:]), ids, out=out) is out
            torch.cuda.synchronize()
            check(torch, out, base, hidden, a, b, scale, ids)
            assert float(room[0]) == 5.0 and bool((room[1 + base.numel():] == 5.0).all())


def test_what_is_masked_does_not_spread():
    # NaN and infinities in a padded token's hidden values, in a sequence
    # without an adapter and in an adapter that nobody has stay where they are.
    torch = need_gpu()
    import burn_dragon_amd as bd
    for T in (2, 40):
        base, hidden, a, b, scale = make(torch, 4, T, 32, 100, 5, 3, torch.float32)
        ids = torch.tensor([0, 2, -1, 0], dtype=torch.int32, device="cuda")
        announce("adapters masked", T)
        want = bd.apply_adapters(base, hidden, bd.AdapterSet(a, b, scale), ids)
        h = hidden.clone()
        h[0, -1] = float("nan")
        h[3, 0, 3] = float("inf")
        h[2] = float("nan")
        a2, b2, s2 = a.clone(), b.clone(), scale.clone()
        a2[1], b2[1], s2[1] = float("nan"), float("inf"), float("nan")
        got = bd.apply_adapters(base, h, bd.AdapterSet(a2, b2, s2), ids)
        torch.cuda.synchronize()
        assert torch.equal(got[1], want[1]) and torch.equal(got[2], base[2])
        assert torch.equal(got[0, :-1], want[0, :-1]) and torch.equal(got[3, 1:], want[3, 1:])
        assert bool(got[0, -1].isnan().all()) and not bool(got[3, 0].isfinite().any())


def test_results_repeat_and_do_not_depend_on_the_batch():
    torch = need_gpu()
    import burn_dragon_amd as bd
    for T in (1, 50):
        base, hidden, a, b, scale = make(torch, 12, T, 128, 600, 16, 2, torch.float32)
        ids = torch.tensor([0, 1] * 6, dtype=torch.int32, device="cuda")
        s = bd.AdapterSet(a, b, scale)
        announce("adapters batch", T)
        whole = bd.apply_adapters(base, hidden, s, ids)
        assert torch.equal(whole, bd.apply_adapters(base, hidden, s, ids))
        for i in (0, 5, 11):
            one = bd.apply_adapters(base[i:i + 1], hidden[i:i + 1], s, ids[i:i + 1])
            assert torch.equal(one[0], whole[i])


@pytest.mark.parametrize("T", [1, 33])
def test_captured_into_a_graph(T):
    torch = need_gpu()
    import burn_dragon_amd as bd
    base, hidden, a, b, scale = make(torch, 5, T, 64, 300, 16, 3, torch.float32)
    ids = torch.tensor([0, 1, 2, -1, 1], dtype=torch.int32, device="cuda")
    s = bd.AdapterSet(a, b, scale)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        bd.apply_adapters(base, hidden, s, ids)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    announce("adapters graph", T)
    with torch.cuda.graph(graph, stream=side):
        out = bd.apply_adapters(base, hidden, s, ids)
    for i in range(4):
        hidden.normal_()
        ids.copy_(torch.roll(ids, 1))  # the ids are read on the device: a replay sees new ones
        want = bd.apply_adapters(base, hidden, s, ids)
        torch.cuda.synchronize()
        graph.replay()
        with torch.cuda.stream(side):
            bd.apply_adapters(base, hidden * 2, s, ids)  # eager work on the capturing stream
        torch.cuda.synchronize()
        assert torch.equal(out, want), i


def test_model_logits_with_adapters():
    # model_forward_logits(adapters=) is its logits and hidden through
    # apply_adapters; a prompt and a generated token, state carried.
    torch = need_gpu()
    import burn_dragon_amd as bd
    V, D, H, N, L, B = 257, 64, 2, 256, 2, 3
    g = torch.Generator(device="cuda").manual_seed(2)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    w = bd.pack_model(rnd(V, D), rnd(1, H, D, N) / D ** 0.5, rnd(1, H, D, N) / D ** 0.5,
                      rnd(H * N, D) / (H * N) ** 0.5, rnd(D, V) / D ** 0.5, L)
    s = bd.AdapterSet((rnd(2, 4, D) / 8).to(torch.bfloat16), rnd(2, V, 4).to(torch.bfloat16),
                      torch.tensor([1.0, 2.0], device="cuda"))
    ids = torch.tensor([1, -1, 0], dtype=torch.int32, device="cuda")
    tokens = torch.randint(0, V, (B, 21), generator=g, device="cuda", dtype=torch.int32)
    nxt = torch.randint(0, V, (B, 1), generator=g, device="cuda", dtype=torch.int32)
    announce("adapters model")
    plain, with_ = (bd.new_model_state(w, B, torch.device("cuda")) for _ in range(2))
    for tok in (tokens, nxt):
        want = bd.model_forward_logits(tok, w, state=plain)
        got = bd.model_forward_logits(tok, w, state=with_, adapters=s, adapter_ids=ids)
        assert torch.equal(got[1], want[1])
        assert not torch.equal(got[0], want[0]) and not torch.equal(got[2], want[2])
        # the added part has the adapter's rank
        for i, id_ in ((0, 1), (2, 0)):
            d = (got[i] - want[i]).double().cpu().numpy()
            bw = s.b[id_].double().cpu().numpy()
            fit = bw @ np.linalg.lstsq(bw, d.T, rcond=None)[0]
            # (the sum with the logits rounds to f32: 2^-24 of logits up to ~10, beside the product's own bound)
            assert np.abs(fit.T - d).max() <= 1e-4 * max(1.0, np.abs(d).max())
    assert plain.position == with_.position == 22
    with pytest.raises(ValueError):
        bd.model_forward_logits(nxt, w, adapters=s)
    # adapters that do not fit are refused before a layer moves the state on
    kept = [r.clone() for r in with_.rho]
    for bad, bad_ids in ((bd.AdapterSet(s.a, s.b[:, :-1], s.scale), ids), (s, ids[:2])):
        with pytest.raises(ValueError):
            bd.model_forward_logits(nxt, w, state=with_, adapters=bad, adapter_ids=bad_ids)
    wide = bd.AdapterSet(s.a.repeat(1, 40, 1), s.b.repeat(1, 1, 40), s.scale)  # rank 160
    assert bd.model_forward_logits(nxt, w, state=with_, adapters=wide, adapter_ids=ids) is None
    assert with_.position == 22 and all(torch.equal(r, k) for r, k in zip(with_.rho, kept))


def test_unsupported_and_refused():
    torch = need_gpu()
    import burn_dragon_amd as bd
    base, hidden, a, b, scale = make(torch, 2, 3, 8, 16, 4, 3, torch.float32)
    ids = torch.zeros(2, dtype=torch.int32, device="cuda")
    s = bd.AdapterSet(a, b, scale)
    assert bd.apply_adapters(base.double(), hidden.double(), s, ids) is None
    assert bd.apply_adapters(base, hidden.bfloat16(), s, ids) is None
    assert bd.apply_adapters(base, hidden, bd.AdapterSet(a.float(), b, scale), ids) is None
    assert bd.apply_adapters(base[:, :0], hidden[:, :0], s, ids) is None
    assert bd.apply_adapters(base.cpu(), hidden.cpu(), s, ids) is None
    wide = bd.AdapterSet(torch.zeros(1, 129, 8, device="cuda").bfloat16(),
                         torch.zeros(1, 16, 129, device="cuda").bfloat16(), scale[:1])
    assert bd.apply_adapters(base, hidden, wide, ids) is None
    for args in ((base, hidden[:1], s, ids), (base, hidden, s, ids[:1]), (base, hidden, s, ids.long()),
                 (base, hidden, bd.AdapterSet(a, b[:, :-1], scale), ids),
                 (base, hidden, bd.AdapterSet(a, b, scale.double()), ids), (base, hidden, s, ids.cpu())):
        with pytest.raises(ValueError):
            bd.apply_adapters(*args)
    with pytest.raises(ValueError):
        bd.apply_adapters(base, hidden, s, ids, out=base.transpose(0, 1))


@pytest.mark.parametrize("T,D,R", [(1, 64, 16), (2, 64, 8), (3, 64, 16), (16, 20, 5)])
def test_more_sequences_than_are_gathered_together(T, D, R):
    # The batch is gathered 512 sequences at a time.
    B = 1100
    run(B, T, D, 70, R, 3, "float32", np.random.default_rng(T).integers(-1, 3, B).tolist())
    run(B, T, D, 70, R, 3, "float32", [1] * B, in_place=True)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("T,D,R,n", [(1, 24, 8, 16), (2, 24, 8, 20), (1, 512, 16, 10), (2, 512, 16, 30), (2, 64, 16, 2)])
def test_few_rows_of_an_adapter_in_a_large_call(T, D, R, n, dtype):
    # 40 x 30001: with and without tiles by the number of adapters.
    run(40, T, D, 30001, R, n, dtype, np.random.default_rng(n).integers(-1, n, 40).tolist())


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("T,D,R", [(1, 64, 16), (1, 64, 32), (40, 64, 16), (40, 64, 64), (20, 33, 5), (1, 33, 5),
                                   (40, 2048, 8)])
def test_values_up_to_f32_s_largest(T, D, R, dtype):
    # hidden, and scale hidden A^T, between bf16's largest finite value and f32's.
    torch = need_gpu()
    import burn_dragon_amd as bd
    dtype = getattr(torch, dtype)
    V = 300
    base, hidden, a, b, scale = make(torch, 2, T, D, V, R, 2, dtype)
    top = float(torch.finfo(dtype).max)
    hidden.zero_()
    hidden[0, :, 0] = top                      # f32: 2^128 (1 - 2^-24)
    hidden[1, :, 1] = -top
    a.zero_()
    a[0, :, 0] = 0.5
    a[1, :, 1] = 1.0
    b.mul_(2.0 ** -100)
    # f32: 0.5 top * 1.99 and -top; bf16, whose largest is 2^128 (1 - 2^-8): beyond that again
    scale = torch.tensor([1.99, 1.0 if dtype == torch.float32 else 1.003], device="cuda")
    ids = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    base.mul_(2.0 ** 28)
    announce("adapters near the largest", T, D, R, dtype)
    out = bd.apply_adapters(base, hidden, bd.AdapterSet(a, b, scale), ids)
    torch.cuda.synchronize()
    assert bool(out.isfinite().all())
    check(torch, out, base, hidden, a, b, scale, ids)


@pytest.mark.parametrize("T,D,R", [(1, 64, 32), (40, 64, 16), (20, 33, 5)])
def test_small_values_hold_to_2_134(T, D, R):
    # Parts below 2^-126 are subnormal: an operand is held to half the least of
    # them, 2^-134, where that is more than 2^-24 of it.  Of a row each operand
    # meets one value of the other here, so that what it lost is seen alone.
    torch = need_gpu()
    import burn_dragon_amd as bd
    V = 300
    base, hidden, a, b, scale = make(torch, 1, T, D, V, R, 1, torch.float32)
    g = torch.Generator(device="cuda").manual_seed(T + D)
    a.zero_()
    b.zero_()
    for k in range(R):
        a[0, k, k] = 1.0
        b[0, k, k] = 2.0 ** 90
    ids = torch.zeros(1, dtype=torch.int32, device="cuda")
    m = 1 + torch.rand(1, T, D, generator=g, device="cuda")
    announce("adapters small", T, D, R)
    for e in (-100, -110, -114, -120, -126):
        for h, s in ((m * 2.0 ** e, 2.0 ** 20), (m, 2.0 ** e)):
            out = bd.apply_adapters(torch.zeros_like(base), h, bd.AdapterSet(a, b, torch.tensor([s], device="cuda")), ids)
            u = h[..., :R].double() * s
            off = (out[..., :R].double() / 2.0 ** 90 - u).abs()
            lost = 2.0 ** -134 * (s if s > 1 else 1.0)
            # three roundings to f32 beside the parts' (u, its product, the sum with base)
            assert bool((off <= u * (2.0 ** -24 + 3 * 2.0 ** -24) + lost).all()), (e, s)
            assert not out[..., R:].any()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("T,D,V,R", [(1, 64, 300, 16), (1, 64, 300, 8), (1, 64, 300, 32), (1, 64, 300000, 16), (1, 64, 70000, 8),
                                     (1, 2048, 9000, 64),
                                     (2, 64, 300000, 16), (3, 64, 300, 16), (40, 64, 300, 16), (40, 64, 300, 24),
                                     (300, 512, 2000, 64), (70, 64, 300, 128)])
def test_what_is_masked_does_not_spread_from_aligned_rows(T, D, V, R, dtype):
    # Ranks and widths that are multiples of 8: without tiles, gathered tiles and
    # tiles of one sequence, u in the workgroup and from its own launch.  The first
    # and the last sequence share their adapter, and so their tile where gathered.
    torch = need_gpu()
    import burn_dragon_amd as bd
    base, hidden, a, b, scale = make(torch, 4, T, D, V, R, 3, getattr(torch, dtype))
    ids = torch.tensor([0, 2, -1, 0], dtype=torch.int32, device="cuda")
    announce("adapters masked, aligned", T, D, V, R, dtype)
    want = bd.apply_adapters(base, hidden, bd.AdapterSet(a, b, scale), ids)
    h = hidden.clone()
    h[0, -1] = float("nan")
    h[2] = float("nan")
    a2, b2, s2 = a.clone(), b.clone(), scale.clone()
    a2[1], b2[1], s2[1] = float("nan"), float("inf"), float("nan")
    s = bd.AdapterSet(a2, b2, s2)
    got = bd.apply_adapters(base, h, s, ids)
    torch.cuda.synchronize()
    assert torch.equal(got[1], want[1]) and torch.equal(got[2], base[2]) and torch.equal(got[3], want[3])
    assert torch.equal(got[0, :-1], want[0, :-1]) and bool(got[0, -1].isnan().all())
    h[0, -1] = hidden[0, -1]
    h[3, 0, 3] = float("inf")
    got = bd.apply_adapters(base, h, s, ids)
    torch.cuda.synchronize()
    assert torch.equal(got[:2], want[:2]) and torch.equal(got[3, 1:], want[3, 1:])
    assert not bool(got[3, 0].isfinite().any())


@pytest.mark.parametrize("T,D,V,R,n,B", [(1, 128, 600, 16, 2, 40), (1, 64, 4000, 16, 2, 300), (50, 128, 600, 16, 2, 400),
                                         (2, 64, 30000, 8, 20, 64), (40, 1024, 300, 64, 2, 30), (1, 64, 70000, 8, 40, 64)])
def test_a_sequence_in_small_and_large_batches(T, D, V, R, n, B):
    # A call's kernels go by its batch (without tiles or with, u computed in place or
    # by its own launch), which sum in different orders: a sequence's results in
    # different batches are the same within the bound of each, not bit for bit.
    torch = need_gpu()
    import burn_dragon_amd as bd
    for dtype in (torch.float32, torch.bfloat16):
        base, hidden, a, b, scale = make(torch, B, T, D, V, R, n, dtype)
        ids = (torch.arange(B, device="cuda") % n).to(torch.int32)
        s = bd.AdapterSet(a, b, scale)
        announce("adapters small and large", T, D, V, R, n, B, dtype)
        whole = bd.apply_adapters(base, hidden, s, ids)
        assert torch.equal(whole, bd.apply_adapters(base, hidden, s, ids))  # the same call: bit for bit
        for i in (0, B // 2, B - 1):
            at = slice(i, i + 1)
            one = bd.apply_adapters(base[at], hidden[at], s, ids[at])
            torch.cuda.synchronize()
            check(torch, one, base[at], hidden[at], a, b, scale, ids[at])
            check(torch, whole[at], base[at], hidden[at], a, b, scale, ids[at])


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("B,T,D,V,R,n", [(40, 1, 24, 30001, 8, 20), (40, 2, 512, 30001, 16, 40), (9, 1, 64, 130000, 16, 5),
                                         (5, 1, 256, 70000, 16, 2), (5, 2, 256, 53000, 8, 2), (64, 1, 64, 4096, 16, 32),
                                         (64, 1, 64, 4097, 16, 32), (64, 1, 64, 17000, 16, 8), (64, 1, 64, 16000, 16, 8)])
def test_few_rows_of_an_adapter_around_the_choice(B, T, D, V, R, n, dtype):
    # With and without tiles by rows an adapter, columns and type.
    run(B, T, D, V, R, n, dtype, np.random.default_rng(V).integers(-1, n, B).tolist())


def test_a_set_given_as_a_tuple():
    torch = need_gpu()
    import burn_dragon_amd as bd
    base, hidden, a, b, scale = make(torch, 3, 2, 64, 100, 8, 2, torch.float32)
    ids = torch.tensor([1, 0, -1], dtype=torch.int32, device="cuda")
    announce("adapters tuple")
    assert torch.equal(bd.apply_adapters(base, hidden, (a, b, scale), ids),
                       bd.apply_adapters(base, hidden, bd.AdapterSet(a, b, scale), ids))
