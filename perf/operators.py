"""What a server of many requests does around the model's forward, as timed
cases: the operators of a serving step beside model_forward_logits.

  sample    the next token of every row from its logits and a given random
            number, with temperature, top-k, top-p and min-p (sample_tokens)
  adapters  low-rank adapters of many requests beside the shared logits
            projection (apply_adapters): out = base + s (hidden A^T) B^T with
            the adapter of each sequence
  streams   the recurrent states of the batch's streams moved between slots
            (copy_streams, compact_streams, free_streams): a prompt's state forked into
            samples, a batch closed up after requests ended, slots exchanged
            and cleared

With own = False the plain forms run: elementary torch operations, sampling in
64 bits (a token goes by which side of a border a sum falls).
"""
import math

import numpy as np
import torch

own = False

LOG2E = 1.4426950408889634
LEAST = -42.0  # log2 of the smallest weight, relative to the largest, that is drawn
HEADS = 4


def listed():
    return [
        # One user's next byte: the model's 256-token vocabulary, launches and latency.
        dict(name="sample_1", op="sample", rows=1, V=256, dtype="f32", temperature=0.8, top_k=40, top_p=0.95,
             min_p=0.0, masked=0.0),
        # A serving batch's next tokens with the usual settings, an ordinary vocabulary.
        dict(name="sample_64", op="sample", rows=64, V=32000, dtype="f32", temperature=0.8, top_k=50, top_p=0.95,
             min_p=0.0, masked=0.0),
        # Nucleus sampling of a large batch over a large vocabulary: no top-k bounds the candidates.
        dict(name="sample_256", op="sample", rows=256, V=131072, dtype="f32", temperature=1.0, top_k=0, top_p=0.9,
             min_p=0.0, masked=0.0),
        # An odd vocabulary in bf16, most of it masked by a grammar, cut by min-p.
        dict(name="sample_bf16", op="sample", rows=17, V=100003, dtype="bf16", temperature=1.2, top_k=0, top_p=1.0,
             min_p=0.05, masked=0.75),
        # One user's next byte with an adapter: latency.
        dict(name="adapters_1", op="adapters", B=1, T=1, D=256, V=256, R=8, n=4, dtype="f32"),
        # A serving batch's next tokens, 32 adapters.
        dict(name="adapters_64", op="adapters", B=64, T=1, D=256, V=32000, R=16, n=32, dtype="f32"),
        # Prompts through the byte model (the model configuration of the benchmark).
        dict(name="adapters_1024", op="adapters", B=16, T=1024, D=256, V=256, R=16, n=8, dtype="f32"),
        # Ragged prompts of a wide model in bf16, an odd vocabulary, large ranks.
        dict(name="adapters_bf16", op="adapters", B=3, T=1001, D=1024, V=50001, R=64, n=3, dtype="bf16"),
        # One small state copied to three streams: latency.
        dict(name="streams_1", op="streams", kind="fork", L=1, B=4, N=256, D=64, n=3),
        # A prompt's state (one stream, six layers of the benchmark's size) into 8 of 16 slots.
        dict(name="streams_fork", op="streams", kind="fork", L=6, B=16, N=8192, D=256, n=8),
        # 5 of 16 requests have ended: the others close up, in order.
        dict(name="streams_compact", op="streams", kind="compact", L=6, B=16, N=8192, D=256, n=11),
        # Odd sizes: slots exchanged in cycles, others cleared.
        dict(name="streams_odd", op="streams", kind="exchange", L=3, B=13, N=1001, D=63, n=9),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["sample", "adapters", "streams"])
    if op == "sample":
        V = rng.choice([_log(rng, 2, 262144), _log(rng, 256, 262144)])
        rows = max(1, min(_log(rng, 1, 1024), 256 * 131072 // V))
        form = rng.choice(["k", "p", "m", "kp", "all", "none"])
        return dict(op=op, rows=rows, V=V, dtype=rng.choice(["f32", "f32", "bf16"]),
                    temperature=rng.choice([0.3, 0.7, 1.0, 1.5]),
                    top_k=rng.choice([1, 20, 64, 300, 2000]) if form in ("k", "kp", "all") else 0,
                    top_p=rng.choice([0.1, 0.5, 0.9, 0.99]) if form in ("p", "kp", "all") else 1.0,
                    min_p=rng.choice([0.01, 0.1]) if form in ("m", "all") else 0.0,
                    masked=rng.choice([0.0, 0.0, 0.5]))
    if op == "adapters":
        V = _log(rng, 64, 131072)
        D = rng.choice([64, 128, 256, 512, 1024, 2048, _log(rng, 64, 2048)])
        R = rng.choice([4, 8, 16, 32, 64, 128, rng.randrange(1, 128)])
        # the plain form lays out one B of rank R a sequence
        B = max(1, min(_log(rng, 1, 64), 2 ** 27 // (V * R)))
        T = rng.choice([1, 1, _log(rng, 2, 1024)])
        T = max(1, min(T, 2 ** 27 // (V * B)))
        n = max(1, min(rng.randrange(1, 64), 2 ** 27 // (V * R)))
        return dict(op=op, B=B, T=T, D=D, V=V, R=R, n=n, dtype=rng.choice(["f32", "f32", "bf16"]))
    kind = rng.choice(["fork", "compact", "exchange"])
    L, N, D = rng.randrange(1, 7), _log(rng, 128, 8192), rng.choice([16, 64, 128, 256, rng.randrange(3, 256)])
    B = max(3, min(_log(rng, 3, 64), 6 * 16 * 8192 * 256 // (L * N * D)))
    return dict(op=op, kind=kind, L=L, B=B, N=N, D=D, n=rng.randrange(1, B))


def _rng(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _types(dtype):
    return torch.bfloat16 if dtype == "bf16" else torch.float32


def _moves(c, seed):
    """The slots (dst, src) that a streams case moves; src -1: cleared."""
    r = np.random.default_rng(seed)
    if c["kind"] == "fork":  # a prompt's one stream into n slots
        return sorted(r.permutation(c["B"])[:c["n"]].tolist()), [0] * c["n"]
    if c["kind"] == "compact":  # n of B streams go on
        keep = sorted(r.permutation(c["B"])[:c["n"]].tolist())
        return list(range(c["n"])), keep
    dst = r.permutation(c["B"])[:c["n"]]  # n slots take one another's streams, one of four is cleared
    src = np.where(r.random(c["n"]) < 0.25, -1, dst[r.permutation(c["n"])])
    return dst.tolist(), src.tolist()


def prepare(case, seed):
    c, g = case, _rng(seed)
    if c["op"] == "sample":
        R, V = c["rows"], c["V"]
        # A language model's logits: a broad bulk, and a few candidates well above it.
        x = torch.randn(R, V, generator=g, device="cuda") * 2.0
        few = torch.randint(0, V, (R, 12), generator=g, device="cuda")
        x.scatter_reduce_(1, few, 6.0 + 2.5 * torch.randn(R, 12, generator=g, device="cuda"), "amax")
        if c["masked"]:
            away = torch.rand(R, V, generator=g, device="cuda") < c["masked"]
            away[:, :1] = False
            x.masked_fill_(away, -math.inf)
        rows = lambda v, t: torch.full((R,), v, device="cuda", dtype=t)  # noqa: E731
        # each request has its own settings; one in eight is greedy
        temperature = c["temperature"] * (0.9 + 0.2 * torch.rand(R, generator=g, device="cuda"))
        temperature = torch.where(torch.rand(R, generator=g, device="cuda") < 0.125,
                                  torch.zeros_like(temperature), temperature)
        return dict(op="sample", logits=x.to(_types(c["dtype"])),
                    u=torch.rand(R, generator=g, device="cuda"), temperature=temperature,
                    top_k=rows(c["top_k"], torch.int32), top_p=rows(c["top_p"], torch.float32),
                    min_p=rows(c["min_p"], torch.float32))
    if c["op"] == "adapters":
        t = _types(c["dtype"])
        n, D, R, V = c["n"], c["D"], c["R"], c["V"]
        a = (torch.randn(n, R, D, generator=g, device="cuda") / math.sqrt(D)).to(torch.bfloat16)
        b = (torch.randn(n, V, R, generator=g, device="cuda") / math.sqrt(R)).to(torch.bfloat16)
        scale = 0.5 + torch.rand(n, generator=g, device="cuda")
        # one request in eight has no adapter
        ids = torch.randint(0, n, (c["B"],), generator=g, device="cuda", dtype=torch.int32)
        ids = torch.where(torch.rand(c["B"], generator=g, device="cuda") < 0.125, torch.full_like(ids, -1), ids)
        hidden = torch.randn(c["B"], c["T"], D, generator=g, device="cuda").to(t)
        base = torch.randn(c["B"], c["T"], V, generator=g, device="cuda").to(t)
        return dict(op="adapters", a=a, b=b, scale=scale, ids=ids, hidden=hidden, base=base)
    dst, src = _moves(c, seed)
    shape = (c["B"], HEADS, c["N"], c["D"])
    rho = [torch.randn(shape, generator=g, device="cuda") for _ in range(c["L"])]
    from_ = rho
    if c["kind"] == "fork":
        from_ = [torch.randn((1,) + shape[1:], generator=g, device="cuda") for _ in range(c["L"])]
    return dict(op="streams", kind=c["kind"], rho=rho, source=from_, dst=dst, src=src)


def _sample(s):
    """In 64 bits, by a sort of every row."""
    x = s["logits"].double()
    x = torch.where(torch.isnan(x), -math.inf, x)
    R, V = x.shape
    greedy = s["temperature"] <= 0
    tau = torch.where(greedy, 1.0, s["temperature"].double())[:, None]
    k = torch.where(greedy, 1, torch.where(s["top_k"] > 0, s["top_k"], V))[:, None]
    p = s["top_p"].double()[:, None]
    ordered, index = torch.sort(x, dim=1, descending=True, stable=True)
    t = (ordered - ordered[:, :1]) / tau * LOG2E
    w = torch.where(t < LEAST, 0.0, torch.exp2(t))
    rank = torch.arange(V, device=x.device)[None]
    w = torch.where(rank < k, w, 0.0)
    before = torch.cumsum(w, 1) - w
    kept = (rank == 0) | (p >= 1) | (before < p * w.sum(1, keepdim=True))
    kept &= w >= s["min_p"].double()[:, None]
    w = torch.zeros_like(w).scatter_(1, index, torch.where(kept, w, 0.0))
    sums = torch.cumsum(w, 1)
    total = sums[:, -1:]
    token = (sums <= s["u"].double()[:, None] * total).sum(1, keepdim=True)
    logprob = torch.log(torch.gather(w, 1, token) / total)
    return token[:, 0].to(torch.int32), logprob[:, 0].float()


def _adapters(s):
    a, b = s["a"].float(), s["b"].float()
    at = s["ids"].long().clamp(min=0)
    scale = torch.where(s["ids"] < 0, 0.0, s["scale"][at])
    u = torch.bmm(s["hidden"].float(), a.transpose(1, 2)[at]) * scale[:, None, None]
    return (s["base"].float() + torch.bmm(u, b.transpose(1, 2)[at])).to(s["base"].dtype)


def _streams(s):
    dst = torch.tensor(s["dst"], device="cuda")
    src = torch.tensor(s["src"], device="cuda")
    for rho, source in zip(s["rho"], s["source"]):
        taken = source[src.clamp(min=0)]
        taken[src < 0] = 0.0
        rho[dst] = taken
    return s["rho"]


def run(state):
    s = state
    if not own:
        return {"sample": _sample, "adapters": _adapters, "streams": _streams}[s["op"]](s)
    import burn_dragon_amd as bd
    if s["op"] == "sample":
        out = bd.sample_tokens(s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"],
                               top_p=s["top_p"], min_p=s["min_p"], want_logprob=True)
        return out.tokens, out.logprob
    if s["op"] == "adapters":
        return bd.apply_adapters(s["base"], s["hidden"], bd.AdapterSet(s["a"], s["b"], s["scale"]), s["ids"])
    if s["kind"] == "compact":
        bd.compact_streams(s["rho"], s["src"])
    else:
        bd.copy_streams(s["rho"], s["dst"], s["src"], source=None if s["source"] is s["rho"] else s["source"])
    return s["rho"]


def work(case):
    c = case
    size = 2 if c.get("dtype") == "bf16" else 4
    if c["op"] == "sample":
        # every logit read once; the random number and four settings of a row; token and log-probability
        return {"bytes": c["rows"] * (c["V"] * size + 20 + 8), "flops": 0}
    if c["op"] == "adapters":
        M, n = c["B"] * c["T"], min(c["n"], c["B"])
        return {"bytes": M * (2 * c["V"] + c["D"]) * size + n * c["R"] * (c["D"] + c["V"]) * 2 + c["B"] * 4,
                "flops": 2 * M * c["R"] * (c["D"] + c["V"])}
    # distinct sources read, destinations written, without the streams that stay where they are (their mean number)
    slab, B, n = c["L"] * HEADS * c["N"] * c["D"] * 4, c["B"], c["n"]
    if c["kind"] == "fork":
        moved = 1 + n
    elif c["kind"] == "compact":
        moved = 2 * (n - sum(math.comb(B - i - 1, n - i - 1) for i in range(n)) / math.comb(B, n))
    else:
        moved = 1.75 * n - 1.5
    return {"bytes": slab * moved, "flops": 0}


def _exact_row(x, u, tau, k, p, least):
    """(token, log-probability) of one row, written as a walk down the order."""
    x = np.where(np.isnan(x), -np.inf, x)
    if tau <= 0:
        return int(np.argmax(x)), 0.0
    order = np.lexsort((np.arange(x.size), -x))[:k if k > 0 else x.size]
    t = (x[order] - x[order[0]]) / tau
    share = np.where(t < LEAST * math.log(2), 0.0, np.exp(t))
    if p < 1:
        run_ = np.cumsum(share / share.sum())
        order = order[:1 + int(np.searchsorted(run_, p))]
        share = share[:order.size]
    share = np.where(share >= least, share, 0.0)
    by_index = np.argsort(order)
    sums = np.cumsum(share[by_index])
    at = by_index[int(np.searchsorted(sums, u * sums[-1], side="right"))]
    return int(order[at]), math.log(share[at] / share.sum())


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "sample":
        host = {k: s[k].double().cpu().numpy() for k in ("logits", "u", "temperature", "top_k", "top_p", "min_p")}
        rows = [_exact_row(host["logits"][r], host["u"][r], host["temperature"][r], int(host["top_k"][r]),
                           host["top_p"][r], host["min_p"][r]) for r in range(case["rows"])]
        return np.array([r[0] for r in rows], np.int32), np.array([r[1] for r in rows])
    if case["op"] == "adapters":
        out = s["base"].double()
        for i, a in enumerate(s["ids"].tolist()):
            if a >= 0:
                low = torch.matmul(s["hidden"][i].double(), s["a"][a].double().t().contiguous())
                out[i] += float(s["scale"][a].double()) * torch.matmul(low, s["b"][a].double().t().contiguous())
        return out
    old = [x.clone() for x in s["source"]]
    for layer, rho in enumerate(s["rho"]):
        for d, f in zip(s["dst"], s["src"]):
            rho[d].copy_(old[layer][f]) if f >= 0 else rho[d].zero_()
    return [x.double() for x in s["rho"]]
