"""copy_streams, free_streams and compact_streams against the same assignment
done one slot at a time from a copy.  Values are moved, so results are equal
bit for bit."""
import numpy as np
import pytest

from tests.gpu_util import announce, need_gpu

pytestmark = pytest.mark.gpu


def state(torch, L, B, H, N, D, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [torch.randn(B, H, N, D, generator=g, device="cuda") for _ in range(L)]


def expected(rho, source, dst, src):
    out = [r.clone() for r in rho]
    for o, s in zip(out, source):
        for d, f in zip(dst, src):
            o[d] = s[f] if f >= 0 else 0.0
    return out


def check(torch, bd, rho, dst, src, source=None):
    want = expected(rho, [s.clone() for s in (source or rho)], dst, src)
    kept = [s.clone() for s in source] if source else None
    assert bd.copy_streams(rho, dst, src, source=source) is rho
    torch.cuda.synchronize()
    for r, w in zip(rho, want):
        assert torch.equal(r, w)
    if source:
        for s, k in zip(source, kept):
            assert torch.equal(s, k)


PATTERNS = {
    "one": ([2], [0]),
    "itself": ([1], [1]),
    "fork": ([1, 2, 3, 4, 5, 6, 7], [0] * 7),
    "swap": ([3, 5], [5, 3]),
    "cycle_of_3": ([0, 4, 6], [4, 6, 0]),
    "chain": ([0, 1, 2, 3, 4, 5, 6, 7, 8, 9], [1, 2, 3, 4, 5, 6, 7, 8, 9, 10]),
    "chain_back": ([1, 2, 3, 4, 5, 6, 7, 8, 9, 10], [0, 1, 2, 3, 4, 5, 6, 7, 8, 9]),
    "reverse": (list(range(11)), list(range(10, -1, -1))),
    "turn_all": (list(range(11)), [(i + 1) % 11 for i in range(11)]),
    "swap_and_fork": ([0, 1, 2, 3, 4], [1, 0, 0, 1, 2]),
    "clear_what_is_read": ([0, 1, 2], [-1, 0, 0]),
    "clear_all": (list(range(11)), [-1] * 11),
    "none": ([], []),
}


@pytest.mark.parametrize("name", sorted(PATTERNS))
@pytest.mark.parametrize("shape", [(2, 11, 4, 64, 16), (1, 11, 3, 7, 5), (3, 11, 1, 1, 1)])
def test_patterns_in_place(name, shape):
    torch = need_gpu()
    import burn_dragon_amd as bd
    announce("streams", name, shape)
    check(torch, bd, state(torch, *shape, seed=5), *PATTERNS[name])


@pytest.mark.parametrize("B", [2, 9, 40, 700])
def test_random_assignments_in_place(B):
    # Every kind of component at once, over several launches at B = 700.
    torch = need_gpu()
    import burn_dragon_amd as bd
    rng = np.random.default_rng(B)
    for seed in range(6):
        n = int(rng.integers(1, B + 1))
        dst = rng.permutation(B)[:n]
        if seed % 2:
            src = dst[rng.permutation(n)]  # cycles only
        else:
            src = rng.integers(-1, B, n)
        announce("streams random", B, seed, n)
        check(torch, bd, state(torch, 2, B, 2, 9, 7, seed), dst.tolist(), src.tolist())


def test_one_cycle_longer_than_a_launch():
    torch = need_gpu()
    import burn_dragon_amd as bd
    B = 1500
    order = np.random.default_rng(3).permutation(B)
    announce("streams one cycle", B)
    check(torch, bd, state(torch, 1, B, 1, 5, 4, 1), order.tolist(), np.roll(order, 1).tolist())


@pytest.mark.parametrize("B,S,n", [(8, 1, 8), (5, 3, 4), (300, 2, 300), (1, 1, 1)])
def test_from_another_state(B, S, n):
    torch = need_gpu()
    import burn_dragon_amd as bd
    rng = np.random.default_rng(B + S)
    announce("streams from another", B, S, n)
    check(torch, bd, state(torch, 2, B, 2, 10, 6, 1), rng.permutation(B)[:n].tolist(),
          rng.integers(-1, S, n).tolist(), state(torch, 2, S, 2, 10, 6, 2))


def test_more_layers_than_a_launch_and_layers_without_rho():
    torch = need_gpu()
    import burn_dragon_amd as bd
    rho = state(torch, 60, 4, 1, 6, 3, 9)
    want = expected(rho, rho, [0, 3], [3, 1])
    announce("streams 60 layers")
    mixed = [None] + rho[:30] + [None] + rho[30:]
    assert bd.copy_streams(mixed, [0, 3], [3, 1]) is mixed
    torch.cuda.synchronize()
    assert all(torch.equal(r, w) for r, w in zip(rho, want))


def test_layers_of_different_sizes_and_unaligned_memory():
    # Slots at addresses that are a multiple of 4 bytes only.
    torch = need_gpu()
    import burn_dragon_amd as bd
    g = torch.Generator(device="cuda").manual_seed(8)
    rho = []
    for i, (h, n, d) in enumerate([(2, 8, 8), (1, 7, 3), (3, 129, 5)]):
        flat = torch.randn(4 * h * n * d + 4, generator=g, device="cuda")
        rho.append(flat[1 + i % 3:1 + i % 3 + 4 * h * n * d].view(4, h, n, d))
    announce("streams unaligned")
    check(torch, bd, rho, [0, 1, 2], [2, 0, 3])


def test_rows_around_the_state_stay():
    torch = need_gpu()
    import burn_dragon_amd as bd
    flat = torch.full((3 * 37 + 16,), 7.0, device="cuda")
    rho = [flat[8:8 + 3 * 37].view(3, 1, 37, 1)]
    announce("streams borders")
    bd.free_streams(rho, [0, 2])
    torch.cuda.synchronize()
    want = torch.full_like(flat, 7.0)
    want[8:8 + 37] = 0.0
    want[8 + 74:8 + 111] = 0.0
    assert torch.equal(flat, want)


def test_nan_and_infinity_move_unchanged():
    torch = need_gpu()
    import burn_dragon_amd as bd
    bits = torch.tensor([0x7fc00001, 0x7f800000, -0x800000, 1, -0x80000000, 0x7f800001, 5, 6],
                        dtype=torch.int32, device="cuda")
    rho = [torch.zeros(2, 1, 8, 1, device="cuda")]
    rho[0].view(torch.int32)[1, 0, :, 0] = bits
    announce("streams bits")
    bd.copy_streams(rho, [0], [1])
    torch.cuda.synchronize()
    assert torch.equal(rho[0].view(torch.int32)[0, 0, :, 0], bits)


def test_offsets_past_32_bits():
    # 5 slots of 2^29 f32 (2 GiB each): element offsets pass 2^31, byte offsets 2^33.
    torch = need_gpu()
    import burn_dragon_amd as bd
    n = 1 << 29
    rho = [torch.zeros(5, 1, n, 1, device="cuda")]
    for i in range(5):
        rho[0][i, 0, :4, 0] = torch.arange(4, device="cuda") + 10.0 * i
        rho[0][i, 0, -4:, 0] = torch.arange(4, device="cuda") + 10.0 * i + 5
    announce("streams 10 GiB")
    bd.copy_streams(rho, [0, 4], [4, 0])
    torch.cuda.synchronize()
    for slot, was in ((0, 4), (1, 1), (4, 0)):
        assert rho[0][slot, 0, :4, 0].tolist() == [10.0 * was + j for j in range(4)]
        assert rho[0][slot, 0, -4:, 0].tolist() == [10.0 * was + 5 + j for j in range(4)]
        assert float(rho[0][slot].sum()) == 80.0 * was + 32


def test_states_positions_and_refusals():
    torch = need_gpu()
    import burn_dragon_amd as bd
    dev = torch.device("cuda:0")
    a = bd.BdhModelState(2, 4, 1, 8, 4, dev, position=5)
    b = bd.BdhModelState(2, 1, 1, 8, 4, dev, position=6)
    for s in (a, b):
        for r in s.rho:
            r.normal_()
    with pytest.raises(ValueError, match="position"):
        bd.copy_streams(a, [1], [0], source=b)
    b.position = 5
    assert bd.copy_streams(a, [1, 3], [0, -1], source=b) is a
    torch.cuda.synchronize()
    for ra, rb in zip(a.rho, b.rho):
        assert torch.equal(ra[1], rb[0]) and not ra[3].any()
    for bad in (dict(dst=[4], src=[0]), dict(dst=[0], src=[-2]), dict(dst=[0, 0], src=[1, 2]),
                dict(dst=[0], src=[1, 2])):
        with pytest.raises(ValueError):
            bd.copy_streams(a, bad["dst"], bad["src"])
    with pytest.raises(ValueError):
        bd.copy_streams([a.rho[0].transpose(2, 3)], [0], [1])
    with pytest.raises(ValueError):
        bd.copy_streams([a.rho[0].double()], [0], [1])
    with pytest.raises(ValueError):
        bd.copy_streams(a, [0], [0], source=b.rho[:1])
    with pytest.raises(ValueError):
        bd.compact_streams(a, [])
    with pytest.raises(ValueError):
        bd.compact_streams(a, [0, 1, 2, 3, 0])


def test_compact_gives_the_first_slots_of_the_same_memory():
    torch = need_gpu()
    import burn_dragon_amd as bd
    a = bd.BdhModelState(3, 6, 2, 8, 4, torch.device("cuda:0"), position=11)
    for r in a.rho:
        r.normal_()
    old = [r.clone() for r in a.rho]
    announce("streams compact")
    c = bd.compact_streams(a, [5, 0, 3, 3])
    torch.cuda.synchronize()
    assert c.position == 11 and len(c.rho) == 3
    for r, o, full in zip(c.rho, old, a.rho):
        assert r.shape[0] == 4 and r.data_ptr() == full.data_ptr()
        assert torch.equal(r, o[[5, 0, 3, 3]]) and torch.equal(full[4:], o[4:])


def test_captured_into_a_graph_and_on_another_stream():
    # The slots travel with the launch, so a replay repeats the captured
    # assignment on whatever the memory then holds; no scratch is shared.
    torch = need_gpu()
    import burn_dragon_amd as bd
    rho = state(torch, 2, 6, 2, 32, 16, 3)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    announce("streams graph")
    with torch.cuda.graph(graph, stream=side):
        bd.copy_streams(rho, [0, 1, 2, 5], [1, 2, 0, -1])
    torch.cuda.synchronize()
    for i in range(3):
        want = expected(rho, rho, [0, 1, 2, 5], [1, 2, 0, -1])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(r, w) for r, w in zip(rho, want)), i
        want = expected(rho, rho, [4], [0])
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            bd.copy_streams(rho, [4], [0])  # eager work between the replays
        torch.cuda.synchronize()
        assert all(torch.equal(r, w) for r, w in zip(rho, want)), i


@pytest.mark.parametrize("name", ["fork", "close_up", "cycle", "cycle_and_forks", "from_another"])
def test_calls_larger_than_the_caches(name):
    # 16.8 MB a slot: each of these moves more than the last-level cache holds.
    torch = need_gpu()
    import burn_dragon_amd as bd
    B, shape = 48, (4, 4096, 256)
    dst, src = {
        "fork": (list(range(1, 41)), [0] * 40),
        "close_up": (list(range(40)), list(range(8, 48))),
        "cycle": (list(range(40)), list(range(1, 40)) + [0]),
        "cycle_and_forks": (list(range(40)), list(range(1, 12)) + [0] + [i % 12 for i in range(28)]),
        "from_another": (list(range(8, 48)), list(range(40))),
    }[name]
    announce("streams past the caches", name)
    g = torch.Generator(device="cuda").manual_seed(12)
    rho = [torch.randn(B, *shape, generator=g, device="cuda")]
    source = [torch.randn(B, *shape, generator=g, device="cuda")] if name == "from_another" else None
    for _ in range(2):
        check(torch, bd, rho, dst, src, source)


@pytest.mark.parametrize("name", ["swaps", "cycles_of_3", "cycles_of_8", "last_step_of_1", "last_step_of_2",
                                  "last_step_of_3", "clears_and_moves", "clears_alone", "from_another_and_clears"])
def test_calls_larger_than_the_caches_at_odd_sizes(name):
    # 16.7 MB a slot, not a multiple of 16 bytes, at addresses that are not one
    # either.  All but clears_alone pass the caches by: 33 slots or more are read and
    # written, at most three written for one read, none in a cycle past eight.
    torch = need_gpu()
    import burn_dragon_amd as bd
    B, shape = 40, (3, 1367, 1021)
    turn = lambda n, k: (list(range(n * k)), [i // k * k + (i + 1) % k for i in range(n * k)])  # noqa: E731
    chain = lambda n: (list(range(n)), list(range(1, n + 1)))  # noqa: E731
    dst, src = {
        "swaps": turn(10, 2), "cycles_of_3": turn(7, 3), "cycles_of_8": turn(4, 8),
        "last_step_of_1": chain(17), "last_step_of_2": chain(18), "last_step_of_3": chain(35),
        "clears_and_moves": (list(range(30)), [-1 if i % 3 == 0 else i + 10 for i in range(30)]),
        "clears_alone": (list(range(0, 40, 2)), [-1] * 20),
        "from_another_and_clears": (list(range(40)), [-1 if i % 4 == 0 else i for i in range(40)]),
    }[name]
    announce("streams past the caches, odd", name)
    g = torch.Generator(device="cuda").manual_seed(15)
    slot = shape[0] * shape[1] * shape[2]

    def odd(first):
        flat = torch.empty(B * slot + 8, device="cuda")
        flat.normal_(generator=g)
        return flat, [flat[first:first + B * slot].view(B, *shape)]
    flat, rho = odd(1)
    source = odd(3)[1] if name == "from_another_and_clears" else None
    around = flat[:1].clone(), flat[1 + B * slot:].clone()
    for _ in range(2):
        check(torch, bd, rho, dst, src, source)
    assert torch.equal(flat[:1], around[0]) and torch.equal(flat[1 + B * slot:], around[1])
