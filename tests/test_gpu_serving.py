"""The operators of a serving step together, as a server uses them: prompts
forked into slots, forwards with an adapter a request, draws with each
request's settings, streams closed up and slots refilled."""
import numpy as np
import pytest

from tests import sampleref
from tests.gpu_util import announce, need_gpu

pytestmark = pytest.mark.gpu

V, D, H, N, L = 500, 64, 2, 512, 2


def build(torch, bd):
    g = torch.Generator(device="cuda").manual_seed(12)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    w = bd.pack_model(rnd(V, D), rnd(1, H, D, N) / D ** 0.5, rnd(1, H, D, N) / D ** 0.5,
                      rnd(H * N, D) / (H * N) ** 0.5, 3 * rnd(D, V) / D ** 0.5, L)
    s = bd.AdapterSet((rnd(3, 8, D) / 8).to(torch.bfloat16), rnd(3, V, 8).to(torch.bfloat16),
                      torch.tensor([0.5, 1.0, 2.0], device="cuda"))
    return g, w, s


def test_a_server_s_steps():
    torch = need_gpu()
    import burn_dragon_amd as bd
    g, w, adapters = build(torch, bd)
    dev = torch.device("cuda:0")
    B = 6
    # one prompt into slots 1, 3 and 4, another into 0; 2 and 5 begin empty
    prompt = torch.randint(0, V, (2, 13), generator=g, device="cuda", dtype=torch.int32)
    batch = bd.new_model_state(w, B, dev, position=13)
    announce("serving prompts")
    for p, slots in ((0, [1, 3, 4]), (1, [0])):
        one = bd.new_model_state(w, 1, dev)
        bd.model_forward_logits(prompt[p:p + 1], w, state=one)
        assert bd.copy_streams(batch, slots, [0] * len(slots), source=one) is batch
        for r, o in zip(batch.rho, one.rho):
            assert all(torch.equal(r[s], o[0]) for s in slots)
    tokens = torch.randint(0, V, (B, 1), generator=g, device="cuda", dtype=torch.int32)
    tokens[[3, 4]] = tokens[1].clone()
    ids = torch.tensor([2, 0, -1, 0, 1, 2], dtype=torch.int32, device="cuda")
    settings = dict(temperature=torch.tensor([1, 1, 0, 1, 0.7, 2], device="cuda"),
                    top_k=torch.tensor([0, 40, 5, 40, 3, 0], dtype=torch.int32, device="cuda"),
                    top_p=torch.tensor([0.9, 1, 1, 1, 0.8, 1], device="cuda"),
                    min_p=torch.tensor([0, 0.01, 0, 0.01, 0, 0.2], device="cuda"))
    for step in range(8):
        announce("serving step", step)
        logits = bd.model_forward_logits(tokens, w, state=batch, adapters=adapters, adapter_ids=ids)
        u = torch.rand(B, generator=g, device="cuda")
        if step == 0:
            # forks of one prompt with one adapter see the same logits, another adapter's others
            assert torch.equal(logits[1], logits[3]) and not torch.equal(logits[1], logits[4])
        drawn = bd.sample_tokens(logits[:, -1], u, want_logprob=True, **settings)
        want, _ = sampleref.sample(logits[:, -1].cpu().numpy(), u.cpu().numpy(),
                                   **{k: v.cpu().numpy() for k, v in settings.items()})
        assert np.array_equal(drawn.tokens.cpu().numpy(), want)
        tokens = drawn.tokens.unsqueeze(1)
        if step == 3:
            # requests 1 and 2 have ended: the others close up, every setting with them
            old = [r.clone() for r in batch.rho]
            keep = [0, 3, 4, 5]
            batch = bd.compact_streams(batch, keep)
            assert all(torch.equal(r, o[keep]) for r, o in zip(batch.rho, old))
            tokens, ids = tokens[keep].contiguous(), ids[keep].contiguous()
            settings = {k: v[keep].contiguous() for k, v in settings.items()}
            B = 4
        if step == 5:
            # a new request begins in slot 2, slot 3 goes on as a copy of slot 0
            bd.free_streams(batch, [2])
            bd.copy_streams(batch, [3], [0])
            assert all(not r[2].any() and torch.equal(r[3], r[0]) for r in batch.rho)
    assert batch.position == 13 + 8


def test_generate_tokens_is_its_steps():
    torch = need_gpu()
    import burn_dragon_amd as bd
    g, w, adapters = build(torch, bd)
    B, steps = 3, 6
    prompt = torch.randint(0, V, (B, 9), generator=g, device="cuda", dtype=torch.int32)
    u = torch.rand(steps, B, generator=g, device="cuda")
    ids = torch.tensor([1, -1, 2], dtype=torch.int32, device="cuda")
    kw = dict(top_k=50, top_p=0.95, temperature=0.9)
    announce("generate")
    got = bd.generate_tokens(prompt, w, u, adapters=adapters, adapter_ids=ids, want_logprob=True, **kw)
    assert got.tokens.shape == got.logprob.shape == (B, steps) and got.state.position == 9 + steps - 1
    state = bd.new_model_state(w, B, prompt.device)
    cur = prompt
    for i in range(steps):
        logits = bd.model_forward_logits(cur, w, state=state, adapters=adapters, adapter_ids=ids)
        one = bd.sample_tokens(logits[:, -1], u[i], want_logprob=True, **kw)
        assert torch.equal(one.tokens, got.tokens[:, i]) and torch.equal(one.logprob, got.logprob[:, i])
        cur = one.tokens.unsqueeze(1)
    assert all(torch.equal(a, b) for a, b in zip(state.rho, got.state.rho))
    # in two calls: the second begins with the token that the first drew last
    first = bd.generate_tokens(prompt, w, u[:2], adapters=adapters, adapter_ids=ids, **kw)
    second = bd.generate_tokens(first.tokens[:, -1:].contiguous(), w, u[2:], state=first.state, adapters=adapters,
                                adapter_ids=ids, **kw)
    assert torch.equal(torch.cat([first.tokens, second.tokens], 1), got.tokens)
    with pytest.raises(ValueError):
        bd.generate_tokens(prompt, w, u[:, :2])


def test_a_step_of_generation_replays_from_a_graph():
    # forward with adapters, draw and the token's way into the next step, captured
    # once; the state moves on in place, so replays are compared step by step.
    torch = need_gpu()
    import burn_dragon_amd as bd
    g, w, adapters = build(torch, bd)
    B = 4
    ids = torch.tensor([0, 1, 2, -1], dtype=torch.int32, device="cuda")
    tokens = torch.randint(0, V, (B, 1), generator=g, device="cuda", dtype=torch.int32)
    u = torch.rand(B, generator=g, device="cuda")

    def step(tok, state):
        state.position = 20  # (a captured step keeps its position)
        logits = bd.model_forward_logits(tok, w, state=state, adapters=adapters, adapter_ids=ids)
        drawn = bd.sample_tokens(logits[:, -1], u, top_k=30, top_p=0.9)
        tok.copy_(drawn.tokens.unsqueeze(1))

    a = bd.new_model_state(w, B, torch.device("cuda:0"), position=20)
    for r in a.rho:
        r.normal_(generator=g).mul_(0.1)
    b = bd.new_model_state(w, B, torch.device("cuda:0"), position=20)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(tokens.clone(), b)  # warms the stream's scratch
    torch.cuda.synchronize()
    for r, s in zip(a.rho, b.rho):
        s.copy_(r)
    ta, tb = tokens.clone(), tokens.clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    announce("serving graph")
    with torch.cuda.graph(graph, stream=side):
        step(tb, b)
    for i in range(4):
        u.uniform_(generator=g)
        step(ta, a)  # eager, on the current stream
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(ta, tb), i
        assert all(torch.equal(r, s) for r, s in zip(a.rho, b.rho)), i
