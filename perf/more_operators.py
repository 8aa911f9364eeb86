"""What a training step runs around the recurrent attention, as timed cases.

  embed   the token embedding with its scale or the model's input norm
          (embed_tokens), and the table's gradient (embed_tokens_vjp)
  save    activations kept between forward and backward in 8 bits
          (checkpoint_activations, restore_activations): e4m3 values with one
          power of two for 32 neighbours of a row
  gated   the gated block out = up(x U - th) m * act(c G - th) m, a head of latents
          at a time (gated_block): BDH's y = ReLU(a Ev) * ReLU(cur E), or an
          ordinary gated feed-forward block; its backward pass, recomputing or
          from what the forward saved in 8 bits (gated_block_vjp)

With own = False the plain forms run: elementary torch operations in 32 bits.
"""
import math

import torch

own = False

BLOCK = 32      # neighbours that share a power of two
LEAST = -117    # its least exponent
EPS = 1e-5      # of the input norm


def listed():
    return [
        # The model's input for one generated token: latency.
        dict(name="embed_1", op="embed", grad=False, M=1, V=256, D=256, dtype="f32", norm=True, zipf=False),
        # A batch of long sequences over an ordinary vocabulary, rows scaled by sqrt(D).
        dict(name="embed_65536", op="embed", grad=False, M=65536, V=32000, D=1024, dtype="bf16", norm=False, zipf=True),
        # The byte model's training batch (the model configuration of the benchmark): every row meets many tokens.
        dict(name="embed_grad_bytes", op="embed", grad=True, M=16384, V=256, D=256, dtype="f32", norm=True, zipf=True),
        # A large vocabulary, most rows of which a batch does not meet.
        dict(name="embed_grad_vocab", op="embed", grad=True, M=32768, V=131072, D=1024, dtype="bf16", norm=False,
             zipf=True),
        # One layer's activations of a training batch.
        dict(name="save_large", op="save", rows=16384, C=8192, dtype="bf16", hole=0.0),
        # Odd rows in f32, some of them zeros.
        dict(name="save_odd", op="save", rows=777, C=1001, dtype="f32", hole=0.3),
        # One generated token through the benchmark model's projections: bound by the weights.
        dict(name="gated_1", op="gated", kind="fwd", B=1, T=1, H=4, D=256, N=8192, act="relu", context=True, th=0.0,
             masked=0.0),
        # A serving batch through an ordinary gated block.
        dict(name="gated_64", op="gated", kind="fwd", B=64, T=1, H=1, D=2048, N=8192, act="silu", context=False, th=0.0,
             masked=0.0),
        # Prompts through an ordinary gated block.
        dict(name="gated_4096", op="gated", kind="fwd", B=4, T=1024, H=1, D=2048, N=8192, act="silu", context=False,
             th=0.0, masked=0.0),
        # A training pass of the benchmark model's block: forward with what it saves, then backward.
        dict(name="gated_train", op="gated", kind="train", B=16, T=1024, H=4, D=256, N=8192, act="relu", context=True,
             th=0.0, masked=0.0),
        # Backward with recomputation, ragged sequences.
        dict(name="gated_back", op="gated", kind="back", B=3, T=1001, H=1, D=1024, N=4096, act="gelu", context=False,
             th=0.0, masked=0.0),
        # Odd sizes, a threshold that leaves few neurons active, half of the latents masked.
        dict(name="gated_odd", op="gated", kind="train", B=5, T=77, H=3, D=200, N=1000, act="relu", context=True, th=1.5,
             masked=0.5),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["embed", "save", "gated", "gated"])
    dtype = rng.choice(["f32", "bf16"])
    if op == "embed":
        D = rng.choice([64, 256, 512, 1024, 2048, _log(rng, 3, 2048)])
        V = min(_log(rng, 2, 262144), 2 ** 27 // D)
        M = min(_log(rng, 1, 131072), 2 ** 26 // D)
        return dict(op=op, grad=rng.random() < 0.6, M=M, V=V, D=D, dtype=dtype, norm=rng.random() < 0.5,
                    zipf=rng.random() < 0.7)
    if op == "save":
        C = _log(rng, 1, 32768)
        return dict(op=op, rows=max(1, min(_log(rng, 1, 65536), 2 ** 27 // C)), C=C, dtype=dtype,
                    hole=rng.choice([0.0, 0.0, 0.5]))
    D = rng.choice([64, 256, 1024, 2048, 8 * _log(rng, 2, 256)])
    N = rng.choice([256, 1024, 8192, 8 * _log(rng, 2, 1024)])
    H = rng.choice([1, 1, 2, 4])
    B, T = _log(rng, 1, 32), rng.choice([1, _log(rng, 2, 2048), _log(rng, 2, 2048)])
    kind = rng.choice(["fwd", "train", "back"])
    T = max(1, min(T, 2 ** 36 // (B * H * N * D), 2 ** 28 // (B * H * N)))
    act = rng.choice(["relu", "silu", "gelu"])
    return dict(op=op, kind=kind, B=B, T=T, H=H, D=D, N=N, act=act, context=rng.random() < 0.5,
                th=rng.choice([0.0, 1.0]) if act == "relu" else 0.0,
                masked=rng.choice([0.0, 0.5]) if act == "relu" else 0.0)


def _types(dtype):
    return torch.bfloat16 if dtype == "bf16" else torch.float32


def prepare(case, seed):
    c, dev = case, "cuda"
    g = torch.Generator(device=dev).manual_seed(int(seed))
    normal = lambda *shape: torch.randn(shape, generator=g, device=dev)  # noqa: E731
    if c["op"] == "embed":
        t, M, V, D = _types(c["dtype"]), c["M"], c["V"], c["D"]
        u = torch.rand(M, generator=g, device=dev)
        # a text's tokens: few make up most of it (rank r with a share of about 1 / r), spread over the ids
        ids = ((V + 1.0) ** u - 1.0).long().clamp(0, V - 1) if c["zipf"] else (u * V).long().clamp(0, V - 1)
        ids = torch.randperm(V, generator=g, device=dev)[ids].to(torch.int32)
        # one token in 64 is padding, the first never
        away = torch.rand(M, generator=g, device=dev) < 1 / 64
        away[0] = False
        ids = torch.where(away, torch.full_like(ids, -1), ids)
        return dict(c, tokens=ids, table=(0.5 + 0.02 * normal(V, D)).to(t) if c["norm"] else normal(V, D).to(t),
                    scale=1.0 if c["norm"] else math.sqrt(D), g=normal(M, D).to(t) if c["grad"] else None)
    if c["op"] == "save":
        x = normal(c["rows"], c["C"]) * torch.exp(2.0 * normal(c["rows"], 1))
        if c["hole"]:
            x *= torch.rand(c["rows"], 1, generator=g, device=dev) >= c["hole"]
        return dict(c, x=x.to(_types(c["dtype"])))
    B, T, H, D, N = (c[k] for k in "BTHDN")
    b = torch.bfloat16
    s = dict(c, x=normal(B, T, D).to(b), up=(normal(H, D, N) / math.sqrt(D)).to(b),
             gate=(normal(H, D, N) / math.sqrt(D)).to(b), c=normal(B, H, T, D).to(b) if c["context"] else None,
             mask=(torch.rand(N, generator=g, device=dev) >= c["masked"]).float() if c["masked"] else None)
    if c["kind"] != "fwd":
        s["g"] = (normal(B, T, H * N) / math.sqrt(N)).to(b)
    return s


def _rows_of(s):
    """The table's rows in f32, as the lookup gives them, and the norm's parts."""
    e = s["table"].float()
    if not s["norm"]:
        return e, None, None
    e = e - e.mean(1, keepdim=True)
    r = torch.rsqrt((e * e).mean(1, keepdim=True) + EPS)
    return e * r, e * r, r


def _embed(s):
    t = s["tokens"].long()
    at, there = t.clamp(min=0), (t >= 0)[:, None]
    if not s["grad"]:
        e = s["table"][at].float()
        if s["norm"]:
            e = e - e.mean(1, keepdim=True)
            e = e * torch.rsqrt((e * e).mean(1, keepdim=True) + EPS)
        return torch.where(there, e * s["scale"], 0.0).to(s["table"].dtype)
    g = torch.where(there, s["g"].float(), 0.0)
    d = torch.zeros(s["V"], s["D"], device=g.device).index_add_(0, at, g) * s["scale"]
    if s["norm"]:
        _, xh, r = _rows_of(s)
        d = r * (d - d.mean(1, keepdim=True) - xh * (d * xh).mean(1, keepdim=True))
    return d.to(s["table"].dtype)


def _in8(x):
    """The values that x (f32, rows of any length) has in 8 bits, in f32."""
    C = x.shape[-1]
    y = torch.nn.functional.pad(x, (0, -C % BLOCK)).unflatten(-1, (-1, BLOCK))
    m, e = torch.frexp(y.abs().amax(-1, keepdim=True))  # amax = m 2^e, m in [1/2, 1); 448 = 7/8 2^9
    e = (torch.where(m > 0.875, e + 1, e) - 9).clamp(min=LEAST)
    power = lambda k: ((k + 127).to(torch.int32) << 23).view(torch.float32)  # noqa: E731 (2^k)
    y = (y * power(-e)).to(torch.float8_e4m3fn).float() * power(e)
    return y.flatten(-2)[..., :C]


def _save(s):
    return _in8(s["x"].float()).to(torch.bfloat16)


def _project(s):
    """Both projections [H, B * T, N] in f32, less the threshold."""
    H, M = s["H"], s["B"] * s["T"]
    x = s["x"].float().reshape(1, M, -1).expand(H, -1, -1)
    c = s["c"].float().transpose(0, 1).reshape(H, M, -1) if s["c"] is not None else x
    return x, c, torch.bmm(x, s["up"].float()) - s["th"], torch.bmm(c, s["gate"].float()) - s["th"]


def _values(s, p, q):
    """(up(p), up'(p), act(q), act'(q)), with the mask's square in the second pair."""
    m = 1.0 if s["mask"] is None else s["mask"] * s["mask"]
    if s["act"] == "relu":
        return torch.relu(p), (p > 0).float(), torch.relu(q) * m, (q > 0).float() * m
    if s["act"] == "silu":
        z = torch.sigmoid(q)
        return p, torch.ones_like(p), q * z, z * (1 + q * (1 - z))
    z = 0.5 * (1 + torch.erf(q * math.sqrt(0.5)))
    return p, torch.ones_like(p), q * z, z + q * torch.exp(-0.5 * q * q) * math.sqrt(0.5 / math.pi)


def _gated(s):
    B, T, H, D, N = (s[k] for k in "BTHDN")
    b = torch.bfloat16
    x, c, p, q = _project(s)
    flat = lambda h: h.reshape(H, B, T, N).permute(1, 2, 0, 3).reshape(B, T, H * N)  # noqa: E731
    out = None
    if s["kind"] != "back":
        u, _, v, _ = _values(s, p, q)
        out = flat((u * v).to(b))
        if s["kind"] == "fwd":
            return out
        if s["act"] == "relu":
            p, q = torch.relu(p), torch.relu(q)
        p, q = _in8(p), _in8(q)
    u, du, v, dv = _values(s, p, q)
    g = s["g"].float().reshape(B * T, H, N).transpose(0, 1)
    dp, dq = g * v * du, g * u * dv
    dx = torch.bmm(dp, s["up"].float().transpose(1, 2)).sum(0)
    dc = torch.bmm(dq, s["gate"].float().transpose(1, 2))
    if s["c"] is None:
        dx, dc = dx + dc.sum(0), None
    else:
        dc = dc.reshape(H, B, T, D).transpose(0, 1).contiguous().to(b)
    grads = [dx.reshape(B, T, D).to(b), dc, torch.bmm(x.transpose(1, 2), dp).to(b),
             torch.bmm(c.transpose(1, 2), dq).to(b)]
    return [t for t in [out] + grads if t is not None]


def run(state):
    s = state
    if not own:
        return {"embed": _embed, "save": _save, "gated": _gated}[s["op"]](s)
    import burn_dragon_amd as bd
    if s["op"] == "embed":
        if s["grad"]:
            return bd.embed_tokens_vjp(s["g"], s["tokens"], s["table"], scale=s["scale"], norm=s["norm"])
        return bd.embed_tokens(s["tokens"], s["table"], scale=s["scale"], norm=s["norm"])
    if s["op"] == "save":
        return bd.restore_activations(bd.checkpoint_activations(s["x"]))
    w = bd.GatedWeights(s["up"], s["gate"])
    how = dict(activation=s["act"], relu_threshold=s["th"], latent_mask=s["mask"])
    if s["kind"] == "fwd":
        return bd.gated_block(s["x"], w, s["c"], **how).out
    out = saved = None
    if s["kind"] == "train":
        out, saved = bd.gated_block(s["x"], w, s["c"], save=True, **how)
    d = bd.gated_block_vjp(s["g"], s["x"], w, s["c"], saved=saved, **how)
    return [t for t in (out, d.current, d.context, d.up, d.gate) if t is not None]


def work(case):
    c = case
    size = 2 if c.get("dtype") == "bf16" else 4
    if c["op"] == "embed":
        M, V, D = c["M"], c["V"], c["D"]
        # the rows that a batch meets, about: of ids with a share of 1 / ((r + 1) ln(V + 1)) or 1 / V
        share = lambda r: 1 / ((r + 1) * math.log(V + 1)) if c["zipf"] else 1 / V  # noqa: E731
        step = max(1, V // 4096)
        met = min(M, sum(step * (1 - (1 - min(1.0, share(r + (step - 1) / 2))) ** M) for r in range(0, V, step)), V)
        if c["grad"]:
            return {"bytes": M * (D * size + 4) + V * D * size + (met * D * size if c["norm"] else 0), "flops": M * D}
        return {"bytes": M * (D * size + 4) + met * D * size, "flops": 0}
    if c["op"] == "save":
        n = c["rows"] * c["C"]
        return {"bytes": n * (size + 2) + 2 * c["rows"] * (c["C"] + -(-c["C"] // BLOCK)), "flops": 0}
    B, T, H, D, N = (c[k] for k in "BTHDN")
    M, weights = B * T, 2 * H * D * N
    inputs = M * D * (1 + (H if c["context"] else 0))
    products = {"fwd": 2, "back": 6, "train": 6}[c["kind"]]
    passed = {"fwd": M * H * N, "back": M * H * N, "train": 2 * M * H * N}[c["kind"]]
    both = 1 if c["kind"] == "fwd" else 2
    return {"bytes": 2 * (both * (inputs + weights) + passed), "flops": products * 2 * M * H * N * D}


def _exact_embed(s):
    table, t = s["table"].double(), s["tokens"].long()
    mean = table.mean(1, keepdim=True)
    sigma = torch.sqrt(((table - mean) ** 2).mean(1, keepdim=True) + EPS)
    if not s["grad"]:
        rows = (table - mean) / sigma if s["norm"] else table
        out = torch.zeros(s["M"], s["D"], dtype=torch.float64, device=table.device)
        out[t >= 0] = s["scale"] * rows[t[t >= 0]]
        return out
    # by a matrix of counts where it is small, else by sorted runs
    order = torch.argsort(t)
    t, g = t[order], s["g"].double()[order]
    g, t = g[t >= 0], t[t >= 0]
    ids, n = torch.unique_consecutive(t, return_counts=True)
    sums = torch.cat([torch.zeros_like(g[:1]), g.cumsum(0)])
    end = n.cumsum(0)
    total = s["scale"] * (sums[end] - sums[end - n])
    out = torch.zeros_like(table)
    if not s["norm"]:
        out[ids] = total
        return out
    # the transposed Jacobian of (e - mean) / sigma
    e, sig = (table - mean)[ids], sigma[ids]
    total = total - total.mean(1, keepdim=True)
    out[ids] = total / sig - e * (total * e).mean(1, keepdim=True) / sig ** 3
    return out


def _exact_in8(x):
    """Rounded to four significant bits, by hand: ties to even, subnormals below 2^-6 of the block's power of two."""
    two = lambda k: ((k.long() + 1023) << 52).view(torch.float64)  # noqa: E731 (2^k, to the bit)
    out = torch.empty_like(x)
    for i in range(0, x.shape[-1], BLOCK):
        v = x[..., i:i + BLOCK]
        top = v.abs().amax(-1, keepdim=True)
        e = torch.where(top > 0, torch.ceil(torch.log2(torch.clamp(top, min=1e-300) / 448.0)), LEAST).clamp(min=LEAST)
        e = torch.where(top > 448.0 * two(e), e + 1, torch.where((top <= 224.0 * two(e)) & (e > LEAST), e - 1, e))
        w = v / two(e)
        k = torch.floor(torch.log2(torch.clamp(w.abs(), min=2.0 ** -6)))
        k = torch.where(w.abs() < two(k), k - 1, torch.where(w.abs() >= two(k + 1), k + 1, k)).clamp(min=-6)
        out[..., i:i + BLOCK] = torch.round(w / two(k - 3)) * two(k - 3) * two(e)
    return out


def _exact_gated(s):
    B, T, H, D, N = (s[k] for k in "BTHDN")
    dev = s["x"].device
    f64 = lambda *shape: torch.zeros(shape, dtype=torch.float64, device=dev)  # noqa: E731
    train, back = s["kind"] == "train", s["kind"] != "fwd"
    m = torch.ones(N, dtype=torch.float64, device=dev) if s["mask"] is None else s["mask"].double() ** 2
    x = s["x"].double().reshape(B * T, D)
    out = f64(B * T, H * N) if s["kind"] != "back" else None
    dx, dc = f64(B * T, D), f64(B, H, T, D)
    du, dg = f64(H, D, N), f64(H, D, N)
    for h in range(H):
        c = x if s["c"] is None else s["c"][:, h].double().reshape(B * T, D)
        wu, wg = s["up"][h].double(), s["gate"][h].double()
        for n in range(0, N, 1024):  # (a multiple of a block)
            cols = slice(n, min(n + 1024, N))
            a, z = x @ wu[:, cols] - s["th"], c @ wg[:, cols] - s["th"]
            if s["act"] == "relu":
                a, z = a.clamp(min=0), z.clamp(min=0)
            phi = lambda v: 0.5 * torch.special.erfc(-v / math.sqrt(2.0))  # noqa: E731
            act = {"relu": lambda v: v, "silu": lambda v: v / (1 + torch.exp(-v)), "gelu": lambda v: v * phi(v)}[s["act"]]
            at = slice(h * N + n, h * N + cols.stop)
            if out is not None:
                out[:, at] = a * act(z) * m[cols]
            if not back:
                continue
            if train:
                a, z = _exact_in8(a), _exact_in8(z)
            if s["act"] == "relu":
                slope = (z > 0).double()
            elif s["act"] == "silu":
                sig = 1 / (1 + torch.exp(-z))
                slope = sig + z * sig * (1 - sig)
            else:
                slope = phi(z) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
            g = s["g"].reshape(B * T, H * N)[:, at].double() * m[cols]
            da, dz = g * act(z), g * a * slope
            if s["act"] == "relu":
                da = da * (a > 0)
            dx += da @ wu[:, cols].t()
            back_c = dz @ wg[:, cols].t()
            if s["c"] is None:
                dx += back_c
            else:
                dc[:, h] += back_c.reshape(B, T, D)
            du[h, :, cols], dg[h, :, cols] = x.t() @ da, c.t() @ dz
    out = None if out is None else out.reshape(B, T, H * N)
    if not back:
        return out
    return [t for t in (out, dx.reshape(B, T, D), dc if s["c"] is not None else None, du, dg) if t is not None]


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "embed":
        return _exact_embed(s)
    if case["op"] == "save":
        return _exact_in8(s["x"].double())
    return _exact_gated(s)
