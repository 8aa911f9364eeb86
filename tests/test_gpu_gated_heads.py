"""gated_block_vjp with so many heads that a workgroup sums several of them for
current's gradient, against the formula in 64 bits, and the scratch that such
calls take."""
import numpy as np
import pytest

from tests import trainref as R
from tests.gpu_util import announce, need_gpu
from tests.test_gpu_gated import check, check_grads, f64, heads, make, plain

pytestmark = pytest.mark.gpu

SUMS = 1 << 28  # bytes of d_x's partial sums in f32, past which they are grouped


def sums_of(B, T, H, D, context):
    return (1 if context else 2) * H * B * T * D * 4


def reference(act, t, p, q, op, oq):
    """R.backward's, where current's gradient may be one f32 sum over all heads' latents."""
    x, c, wu, wg, g, m = plain(t)
    H, _, N = wu.shape
    want = R.backward(act, g, x, c, wu, wg, p, q, op, oq, m)
    u, du = R.up(act, p)
    a, da = R.act(act, q)
    products = [(g * m * m * a * du, wu)] + ([] if t["c"] is not None else [(g * m * m * u * da, wg)])
    size = sum(np.abs(d[h]) @ np.abs(w[h]).T for d, w in products for h in range(H))
    v, o = want["current"]
    want["current"] = v, o + len(products) * H * N * R.U * 1.01 * size
    return want


def run(B, T, H, D, N, act, context, saved):
    torch = need_gpu()
    import burn_dragon_amd as bd
    t = make(torch, B, T, H, D, N, context)
    w = bd.GatedWeights(t["up"], t["gate"])
    announce("gated vjp, many heads", B, T, H, D, N, act, context, saved)
    kept = bd.gated_block(t["x"], w, t["c"], activation=act, save=True).saved if saved else None
    d = bd.gated_block_vjp(t["g"], t["x"], w, t["c"], saved=kept, activation=act)
    again = bd.gated_block_vjp(t["g"], t["x"], w, t["c"], saved=kept, activation=act)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(d, again) if a is not None)
    x, c, wu, wg, _, _ = plain(t)
    if saved:
        p, q = (heads(bd.restore_activations(k, dtype=torch.float32), H) for k in kept)
        op = oq = np.zeros_like(p)
    else:
        p, q, op, oq = R.project(x, c, wu, wg, 0.0)
    check_grads(d, reference(act, t, p, q, op, oq), t)


# Latents that end inside a step of 32, an odd number of heads (a group has the last of up's
# products and the first of gate's), last groups that are shorter, small and large tiles.
@pytest.mark.parametrize("B,T,H,D,N,act,context,saved", [
    (2, 300, 64, 1024, 40, "silu", False, False), (1, 600, 128, 1024, 24, "relu", True, False),
    (3, 200, 128, 1024, 8, "gelu", True, True), (2, 300, 128, 1024, 72, "silu", True, False),
    (2, 260, 33, 2048, 72, "gelu", False, True),
    (1, 1100, 25, 2048, 136, "silu", False, False), (1, 2100, 10, 4096, 264, "relu", True, False),
    (5, 420, 5, 4096, 64, "silu", False, False)])
def test_heads_in_groups(B, T, H, D, N, act, context, saved):
    assert sums_of(B, T, H, D, context) > max(SUMS, 4 * B * T * H * N)
    run(B, T, H, D, N, act, context, saved)


# Saved values of D up to 256, which are read without dp and dq in memory where the sums are few.
@pytest.mark.parametrize("context", [True, False])
def test_heads_in_groups_from_saved_values(context):
    B, T, H, D, N = 2, 1024, 136, 256, 32
    assert B * T * H * N >= 1 << 23 and sums_of(B, T, H, D, context) > max(SUMS, 4 * B * T * H * N)
    run(B, T, H, D, N, "relu", context, True)


@pytest.mark.parametrize("context", [True, False])
def test_scratch_of_many_heads(context):
    # dp and dq take 4 bytes a latent, the sums of d_x no more than SUMS; both grow by a quarter.
    torch = need_gpu()
    import burn_dragon_amd as bd
    B, T, H, D, N = 1, 2048, 64, 4096, 16
    assert sums_of(B, T, H, D, context) >= 8 * SUMS
    t = make(torch, B, T, H, D, N, context)
    w = bd.GatedWeights(t["up"], t["gate"])
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    announce("gated vjp, scratch of many heads", context)
    with torch.cuda.stream(st):
        bd.gated_block_vjp(t["g"][:, :128], t["x"][:, :128], w, None if t["c"] is None else t["c"][:, :, :128])
        torch.cuda.synchronize()
        out = [torch.empty_like(v) for v in (t["x"], t["up"], t["gate"]) + ((t["c"],) if context else ())]
        torch.cuda.synchronize()
        del out  # the caching allocator has room for the outputs
        free = torch.cuda.mem_get_info()[0]
        d = bd.gated_block_vjp(t["g"], t["x"], w, t["c"])
        torch.cuda.synchronize()
        took = free - torch.cuda.mem_get_info()[0]
    assert d is not None
    bd.release_stream_scratch(st)
    assert took <= 1.25 * (SUMS + 4 * B * T * H * N) + (64 << 20)


def with_little_memory(torch, left, call):
    """call() with about `left` bytes of the device's memory free, its outputs' room kept."""
    import burn_dragon_amd as bd
    torch.cuda.synchronize()
    bd.release_stream_scratch()
    torch.cuda.empty_cache()
    hold = []
    try:
        free = torch.cuda.mem_get_info()[0]
        while free > left + (16 << 20):
            hold.append(torch.empty(min(free - left, 32 << 30), dtype=torch.uint8, device="cuda"))
            free = torch.cuda.mem_get_info()[0]
        assert free > left - (16 << 20)
        out = call()
        torch.cuda.synchronize()
    finally:
        del hold
        bd.release_stream_scratch()
        torch.cuda.empty_cache()
    return out


# What is planned does not fit in `left` MiB: 8 of dp and dq with 64 of partial sums; 66 with 139;
# 128 to 131 of dp and dq alone, which go in groups of tokens, of whole sequences (three, or
# one) or pieces of one; from saved values 128 of partial sums, of which 8 are left without
# parts; 98, then 64, where dp and dq take 33.
@pytest.mark.parametrize("B,T,H,D,N,act,context,saved,left", [
    (1, 4096, 1, 1024, 512, "silu", False, False, 40), (2, 1000, 33, 1024, 264, "relu", True, True, 88),
    (1, 8192, 1, 64, 4096, "silu", False, False, 64), (3, 1400, 2, 64, 4096, "gelu", True, False, 64),
    (3, 1400, 2, 64, 4096, "relu", True, False, 36), (7, 600, 2, 320, 4096, "silu", False, True, 108),
    (7, 600, 2, 64, 4096, "silu", True, False, 108), (1, 4096, 1, 256, 8192, "relu", False, True, 64),
    (2, 8192, 2, 256, 264, "relu", False, True, 56)])
def test_little_memory(B, T, H, D, N, act, context, saved, left):
    torch = need_gpu()
    import burn_dragon_amd as bd
    t = make(torch, B, T, H, D, N, context)
    w = bd.GatedWeights(t["up"], t["gate"])
    kept = bd.gated_block(t["x"], w, t["c"], activation=act, save=True).saved if saved else None
    call = lambda: bd.gated_block_vjp(t["g"], t["x"], w, t["c"], saved=kept, activation=act)  # noqa: E731
    announce("gated vjp, memory short", B, T, H, D, N, act, context, saved, left)
    room = [torch.empty_like(v) for v in (t["x"], t["up"], t["gate"], t["c"]) if v is not None]

    def short():
        room.clear()  # (to the caching allocator)
        return call()
    usual = call()
    d = with_little_memory(torch, left << 20, short)
    x, c, wu, wg, _, _ = plain(t)
    if saved:
        p, q = (heads(bd.restore_activations(k, dtype=torch.float32), H) for k in kept)
        op = oq = np.zeros_like(p)
    else:
        p, q, op, oq = R.project(x, c, wu, wg, 0.0)
    want = reference(act, t, p, q, op, oq)
    check_grads(d, want, t)
    # With the memory there again the call goes as planned.
    check_grads(usual, want, t)
    assert all(torch.equal(a, b) for a, b in zip(usual, call()) if a is not None)
