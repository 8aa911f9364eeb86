"""A training step with the operators as they are used together: tokens through
the embedding's norm, the recurrent attention, the gated block (its
projections kept in 8 bits), a decoder, a loss; back through all of them to
the embedding table and the block's weights."""
import math

import pytest

from tests.gpu_util import announce, need_gpu, rel_l2

pytestmark = pytest.mark.gpu

EPS = 1e-5


def norm(torch, x):
    c = x - x.mean(-1, keepdim=True)
    return c / torch.sqrt((c * c).mean(-1, keepdim=True) + EPS)


def norm_vjp(x, g):
    """The gradient of norm(x), by its formula."""
    c = x - x.mean(-1, keepdim=True)
    r = 1 / (c.pow(2).mean(-1, keepdim=True) + EPS).sqrt()
    xh = c * r
    return r * (g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True))


def reference(torch, p, tokens, targets, H, saved=None):
    """The loss and its gradients by autograd in 64 bits, on the host; saved: the block's
    projections as kept, which the backward then takes the slopes and factors from."""
    q = {k: v.double().cpu().requires_grad_() for k, v in p.items()}
    B, T = tokens.shape
    D = q["embed"].shape[1]
    cur = norm(torch, q["embed"][tokens.cpu().long()])                       # [B, T, D]
    x = torch.relu(torch.einsum("btd,hdn->bhtn", cur, q["up"]))             # queries = keys
    s = torch.tril(x @ x.transpose(-1, -2), -1)
    a = norm(torch, s @ cur[:, None])                                        # [B, H, T, D]
    pu, pg = torch.einsum("btd,hdn->bthn", cur, q["up"]), torch.einsum("bhtd,hdn->bthn", a, q["gate"])
    if saved is None:
        y = torch.relu(pu) * torch.relu(pg)
    else:  # straight through the 8 bits: the value as it is, the derivative at what was kept
        u, g = (v.double().cpu() for v in saved)
        y = (torch.relu(pu) * torch.relu(pg)).detach()
        y = y + (pu - pu.detach()) * (u > 0) * g + (pg - pg.detach()) * (g > 0) * u
    z = y.reshape(B, T, -1) @ q["decoder"]
    logits = norm(torch, cur + z) @ q["embed"].t()
    loss = torch.nn.functional.cross_entropy(logits.reshape(B * T, -1), targets.cpu().long().reshape(-1))
    loss.backward()
    return float(loss.detach()), {k: v.grad for k, v in q.items()}


def step(torch, bd, p, tokens, targets, H, save):
    """The same by the operators; torch for what they are not (norms, the decoder, the loss)."""
    b = torch.bfloat16
    B, T = tokens.shape
    V, D = p["embed"].shape
    N = p["up"].shape[2]
    w = bd.GatedWeights(p["up"].to(b), p["gate"].to(b))
    cur = bd.embed_tokens(tokens, p["embed"], norm=True)
    x = torch.relu(torch.matmul(cur[:, None], w.up.float()))
    att = bd.try_fused_recurrent_attention(x, cur[:, None].contiguous()).context
    a = norm(torch, att)
    out = bd.gated_block(cur.to(b), w, a.to(b), save=save)
    z = out.out.float() @ p["decoder"]
    hidden = norm(torch, cur + z)
    logits = (hidden @ p["embed"].t()).reshape(B * T, V)
    logp = torch.log_softmax(logits, 1)
    index = targets.long().reshape(-1, 1)
    loss = -logp.gather(1, index).mean()
    # Back.
    dlogits = (logp.exp() - torch.zeros_like(logp).scatter_(1, index, 1.0)) / (B * T)
    grads = {"embed": dlogits.t() @ hidden.reshape(B * T, D)}
    dsum = norm_vjp(cur + z, (dlogits @ p["embed"]).reshape(B, T, D))
    grads["decoder"] = out.out.float().reshape(B * T, -1).t() @ dsum.reshape(B * T, D)
    dy = (dsum @ p["decoder"].t()).to(b)
    d = bd.gated_block_vjp(dy, cur.to(b), w, a.to(b), saved=out.saved)
    datt = norm_vjp(att, d.context.float())
    v = bd.recurrent_attention_vjp(datt, x, cur[:, None].contiguous())
    dx = torch.where(x > 0, v.grad_query, 0.0)
    grads["up"] = d.up.float() + torch.matmul(cur.reshape(B * T, D).t(), dx.transpose(0, 1).reshape(H, B * T, N))
    grads["gate"] = d.gate.float()
    dcur = dsum + d.current.float() + v.grad_value[:, 0] + torch.matmul(dx, w.up.float().transpose(1, 2)).sum(1)
    assert bd.embed_tokens_vjp(dcur, tokens, p["embed"], norm=True, out=grads["embed"], accumulate=True) is not None
    return float(loss), grads, out.saved


def make(torch, V, D, H, N, B, T):
    g = torch.Generator(device="cuda").manual_seed(11)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    b = torch.bfloat16
    p = {"embed": rnd(V, D), "up": (rnd(H, D, N) / math.sqrt(D)).to(b).float(),
         "gate": (rnd(H, D, N) / math.sqrt(D)).to(b).float(), "decoder": rnd(H * N, D) / math.sqrt(H * N)}
    tokens = torch.randint(0, V, (B, T + 1), generator=g, device="cuda", dtype=torch.int32)
    return p, tokens[:, :-1].contiguous(), tokens[:, 1:].contiguous()


@pytest.mark.parametrize("save", [False, True])
def test_a_step_of_training(save):
    torch = need_gpu()
    import burn_dragon_amd as bd
    H = 2
    p, tokens, targets = make(torch, 61, 64, H, 256, 3, 40)
    announce("training step", save)
    loss, grads, saved = step(torch, bd, p, tokens, targets, H, save)
    kept = None
    if save:
        kept = [bd.restore_activations(c, dtype=torch.float32) for c in saved]
    torch.cuda.synchronize()
    want, exact = reference(torch, p, tokens, targets, H, kept)
    # Each value passes at most a dozen roundings to bf16 between the parameters and a
    # gradient (activations, the block's output, gradients, weights' gradients), each of
    # 2^-8 at most and independent of the others: sqrt(12) 2^-8 = 1.4 % of a gradient's
    # norm; signs of ReLUs near zero that they turn add less.
    assert abs(loss - want) <= 1e-2 * abs(want)
    for k in p:
        assert rel_l2(grads[k].cpu().numpy(), exact[k].numpy()) <= 3e-2, k


def test_a_captured_step_follows_its_inputs():
    torch = need_gpu()
    import burn_dragon_amd as bd
    V, D, H, N, B, T = 61, 64, 2, 256, 3, 40
    p, tokens, _ = make(torch, V, D, H, N, B, T)
    b = torch.bfloat16
    w = bd.GatedWeights(p["up"].to(b), p["gate"].to(b))
    context = torch.randn(B, H, T, D, device="cuda").to(b)
    dy = torch.randn(B, T, H * N, device="cuda").to(b)
    table = torch.zeros(V, D, device="cuda")

    def part():
        cur = bd.embed_tokens(tokens, p["embed"], norm=True).to(b)
        kept = bd.checkpoint_activations(cur)
        o = bd.gated_block(cur, w, context, save=True)
        d = bd.gated_block_vjp(dy, bd.restore_activations(kept), w, context, saved=o.saved)
        g = bd.embed_tokens_vjp(d.current.float(), tokens, p["embed"], norm=True, out=table, accumulate=True)
        return [o.out, *d, g]
    s = torch.cuda.Stream()
    announce("captured training step")
    with torch.cuda.stream(s):
        part()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        held = part()
    for k in range(3):
        tokens.copy_(torch.randint(-1, V + 1, (B, T), device="cuda", dtype=torch.int32))
        dy.copy_(torch.randn(B, T, H * N, device="cuda"))
        table.zero_()
        graph.replay()
        got = [t.clone() for t in held]
        table.zero_()
        want = part()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want)), k
    del graph
    with torch.cuda.stream(s):
        bd.release_stream_scratch(s)
