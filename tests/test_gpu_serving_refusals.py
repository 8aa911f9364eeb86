"""A call that is refused has not touched the state that it was given: the
same call with the argument put right continues the sequence as if the
refused one had not been made."""
import pytest

from tests.gpu_util import announce, need_gpu

pytestmark = pytest.mark.gpu

V, D, H, N, L, B = 257, 64, 2, 256, 2, 3


def build(torch, bd):
    g = torch.Generator(device="cuda").manual_seed(21)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    w = bd.pack_model(rnd(V, D), rnd(1, H, D, N) / D ** 0.5, rnd(1, H, D, N) / D ** 0.5,
                      rnd(H * N, D) / (H * N) ** 0.5, rnd(D, V) / D ** 0.5, L)
    s = bd.AdapterSet((rnd(2, 4, D) / 8).to(torch.bfloat16), rnd(2, V, 4).to(torch.bfloat16),
                      torch.tensor([1.0, 2.0], device="cuda"))
    state = bd.new_model_state(w, B, torch.device("cuda:0"), position=7)
    for r in state.rho:
        r.normal_(generator=g).mul_(0.1)
    tokens = torch.randint(0, V, (B, 5), generator=g, device="cuda", dtype=torch.int32)
    ids = torch.tensor([1, -1, 0], dtype=torch.int32, device="cuda")
    return g, w, s, state, tokens, ids


def refused(torch, state, kept, call, error):
    """The call raises `error`, or returns None where that is None."""
    if error is None:
        assert call() is None
    else:
        with pytest.raises(error):
            call()
    torch.cuda.synchronize()
    assert state.position == 7
    assert all(torch.equal(r, k) for r, k in zip(state.rho, kept))


# How each changes (adapters, ids), and what the call does.
BAD = {
    "ids_int64": (lambda s, i: (s, i.long()), ValueError),
    "ids_on_the_host": (lambda s, i: (s, i.cpu()), ValueError),
    "ids_of_another_batch": (lambda s, i: (s, i[:2]), ValueError),
    "scale_f64": (lambda s, i: (s._replace(scale=s.scale.double()), i), ValueError),
    "scale_of_another_set": (lambda s, i: (s._replace(scale=s.scale[:1]), i), ValueError),
    "scale_on_the_host": (lambda s, i: (s._replace(scale=s.scale.cpu()), i), ValueError),
    "a_on_the_host": (lambda s, i: (s._replace(a=s.a.cpu()), i), ValueError),
    "b_on_the_host": (lambda s, i: (s._replace(b=s.b.cpu()), i), ValueError),
    "b_of_another_vocabulary": (lambda s, i: (s._replace(b=s.b[:, :-1]), i), ValueError),
    "a_of_another_width": (lambda s, i: (s._replace(a=s.a[:, :, :-1]), i), ValueError),
    "no_adapters": (lambda s, i: (type(s)(s.a[:0], s.b[:0], s.scale[:0]), i), None),
    "rank_0": (lambda s, i: (s._replace(a=s.a[:, :0], b=s.b[:, :, :0]), i), None),
    "rank_132": (lambda s, i: (s._replace(a=s.a.repeat(1, 33, 1), b=s.b.repeat(1, 1, 33)), i), None),
    "a_f32": (lambda s, i: (s._replace(a=s.a.float()), i), None),
    "b_of_two_dimensions": (lambda s, i: (s._replace(b=s.b[0]), i), None),
}


@pytest.mark.parametrize("name", sorted(BAD))
def test_adapters_that_a_forward_refuses(name):
    torch = need_gpu()
    import burn_dragon_amd as bd
    _, w, s, state, tokens, ids = build(torch, bd)
    change, error = BAD[name]
    bad, bad_ids = change(s, ids)
    kept = [r.clone() for r in state.rho]
    announce("forward refuses", name)
    refused(torch, state, kept,
            lambda: bd.model_forward_logits(tokens, w, state=state, adapters=bad, adapter_ids=bad_ids), error)
    # then the call put right is the first one
    again = bd.new_model_state(w, B, torch.device("cuda:0"), position=7)
    for r, k in zip(again.rho, kept):
        r.copy_(k)
    got = bd.model_forward_logits(tokens, w, state=state, adapters=s, adapter_ids=ids)
    want = bd.model_forward_logits(tokens, w, state=again, adapters=s, adapter_ids=ids)
    torch.cuda.synchronize()
    assert torch.equal(got, want) and state.position == again.position == 12


def per_row(torch, v, dtype, n=B):
    return torch.full((n,), v, dtype=getattr(torch, dtype), device="cuda")


# How each changes generate_tokens' arguments, given torch and uniform, and the error.
BAD_DRAWS = {
    "uniform_f64": (lambda t, u: dict(uniform=u.double()), ValueError),
    "uniform_on_the_host": (lambda t, u: dict(uniform=u.cpu()), ValueError),
    "uniform_of_another_batch": (lambda t, u: dict(uniform=u[:, :2]), ValueError),
    "top_k_int64": (lambda t, u: dict(top_k=per_row(t, 5, "int64")), ValueError),
    "top_k_of_another_batch": (lambda t, u: dict(top_k=per_row(t, 5, "int32", 2)), ValueError),
    "temperature_f64": (lambda t, u: dict(temperature=per_row(t, 1, "float64")), ValueError),
    "top_p_on_the_host": (lambda t, u: dict(top_p=per_row(t, 1, "float32").cpu()), ValueError),
    "min_p_int": (lambda t, u: dict(min_p=per_row(t, 0, "int32")), ValueError),
    "temperature_negative": (lambda t, u: dict(temperature=-1.0), "BdhError"),
    "temperature_nan": (lambda t, u: dict(temperature=float("nan")), "BdhError"),
    "temperature_past_f32": (lambda t, u: dict(temperature=1e39), "BdhError"),
    "top_p_above_1": (lambda t, u: dict(top_p=1.5), "BdhError"),
    "min_p_negative": (lambda t, u: dict(min_p=-0.1), "BdhError"),
    "top_k_negative": (lambda t, u: dict(top_k=-1), "BdhError"),
    "top_k_0_mod_2_32": (lambda t, u: dict(top_k=-2 ** 32), "BdhError"),
}


@pytest.mark.parametrize("name", sorted(BAD_DRAWS))
def test_draws_that_generation_refuses(name):
    torch = need_gpu()
    import burn_dragon_amd as bd
    from burn_dragon_amd import _lib
    g, w, _, state, tokens, _ = build(torch, bd)
    u = torch.rand(3, B, generator=g, device="cuda")
    change, error = BAD_DRAWS[name]
    error = _lib.BdhError if error == "BdhError" else error
    bad = {**dict(uniform=u), **change(torch, u)}
    kept = [r.clone() for r in state.rho]
    announce("generation refuses", name)
    refused(torch, state, kept,
            lambda: bd.generate_tokens(tokens, w, bad["uniform"], state=state,
                                       **{k: v for k, v in bad.items() if k != "uniform"}), error)
    # sample_tokens says the same of these arguments
    logits = torch.zeros(B, V, device="cuda")
    with pytest.raises(error):
        bd.sample_tokens(logits, bad["uniform"][0], **{k: v for k, v in bad.items() if k != "uniform"})


def test_adapters_and_prompts_that_generation_refuses():
    torch = need_gpu()
    import burn_dragon_amd as bd
    g, w, s, state, tokens, ids = build(torch, bd)
    u = torch.rand(2, B, generator=g, device="cuda")
    kept = [r.clone() for r in state.rho]
    announce("generation refuses adapters, prompts")
    for kw, error in ((dict(adapters=s, adapter_ids=ids.long()), ValueError), (dict(adapters=s), ValueError),
                      (dict(adapters=s._replace(scale=s.scale.double()), adapter_ids=ids), ValueError)):
        refused(torch, state, kept, lambda: bd.generate_tokens(tokens, w, u, state=state, **kw), error)
    refused(torch, state, kept, lambda: bd.generate_tokens(tokens.long(), w, u, state=state), None)
    refused(torch, state, kept, lambda: bd.generate_tokens(tokens[:, :0], w, u, state=state), None)
    refused(torch, state, kept, lambda: bd.generate_tokens(tokens, w, u[:0], state=state), ValueError)
