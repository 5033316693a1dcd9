"""What is timed of the network operators: rotary positions, group norm with an activation
(channels last) and its backward pass, the gated projection and its backward pass, and the
RoFormer mask head, each over the sizes that the separators' networks have around the front and
back halves, from the smallest calls to the largest.

Where `own` is true, `run` calls the framework; where it is false, it computes the same in
elementary torch operations, in 32 bits (angles in 64), rounded once at the end.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZES = {"f32": 4, "bf16": 2, "f16": 2}

# The bands of the repository's two RoFormer configurations (n_fft 2048, 44.1 kHz): frequencies per band.
MEL = ((7,) + (6,) * 14 + (7,) * 3 + (9,) * 3 + (10,) * 2 + (11,) + (13,) * 3 + (15, 16, 17, 19, 20, 20, 22, 24, 26, 28, 29, 31, 33,
       36, 39, 41, 44, 47, 50, 54, 57, 61, 66, 71, 76, 80, 86, 93, 99, 105, 113, 122, 130))
BS = (2,) * 24 + (4,) * 12 + (12,) * 8 + (24,) * 8 + (48,) * 8 + (128, 129)
BANDS = {"mel": MEL, "bs": BS}
HOP = 441


def listed():
    return [
        # RoFormer's time attention over one chunk: 60 bands x 801 frames, queries and keys of 8 heads
        dict(name="rotary_time_attention", op="rotary", dtype="bf16", batch=60, tokens=801, heads=8, kv_heads=8, head_dim=64, rotary_dim=64,
             layout="interleaved", scaling="none", factor=1.0, far=0, inverse=False, strided=True),
        # one new frame of 4 streams far into a long session, half layout, part of the head, scaled positions
        dict(name="rotary_one_token", op="rotary", dtype="f16", batch=4, tokens=1, heads=16, kv_heads=4, head_dim=80, rotary_dim=32,
             layout="half", scaling="yarn", factor=8.0, far=1000003, inverse=False, strided=False),
        # HTDemucs' innermost residual branch: a short row of 48 channels
        dict(name="norm_short", op="norm", dtype="f32", batch=1, positions=336, channels=48, groups=1, activation="gelu", params="f32"),
        # an outer layer of a spectral U-Net: 512 bins x 336 frames x 96 channels, 4 segments
        dict(name="norm_outer_layer", op="norm", dtype="bf16", batch=4, positions=172032, channels=96, groups=8, activation="gelu", params="f32"),
        # training a middle layer: 128 x 336 positions
        dict(name="norm_back_middle_layer", op="norm_back", dtype="f32", batch=2, positions=43008, channels=192, groups=4, activation="silu", params="f32"),
        # odd sizes: nothing is a whole vector
        dict(name="norm_back_odd", op="norm_back", dtype="f16", batch=3, positions=1237, channels=75, groups=5, activation="gelu", params="f16"),
        # the feed-forward of RoFormer's layers over one chunk: 60 bands x 801 frames
        dict(name="gated_chunk", op="gated", dtype="bf16", rows=48060, features=384, width=1408, activation="silu", bias=True),
        # one frame at a time: the weights are all there is to read
        dict(name="gated_one_row", op="gated", dtype="bf16", rows=1, features=2048, width=5461, activation="gelu", bias=False),
        # training it, half a chunk
        dict(name="gated_back_chunk", op="gated_back", dtype="bf16", rows=24030, features=384, width=1408, activation="silu", bias=True),
        # odd sizes in 32 bits
        dict(name="gated_back_odd", op="gated_back", dtype="f32", rows=777, features=301, width=515, activation="gelu", bias=True),
        # the last layer of a Mel-Band RoFormer over one chunk, into the masks that the back half reads
        dict(name="mask_head_mel", op="head", dtype="bf16", bands="mel", chunks=1, stems=1, frames=801, hidden=1536, bias=True),
        # short chunks of a two-stem BS-RoFormer, two of them in a batch, a hidden width that is no whole vector
        dict(name="mask_head_bs_short", op="head", dtype="f16", bands="bs", chunks=2, stems=2, frames=87, hidden=250, bias=False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rotary", "norm", "norm_back", "gated", "gated_back", "head"])
    dtype = rng.choice(["bf16", "f16", "f32"])
    if op == "rotary":
        dim = 2 * rng.randint(8, 128)
        heads = rng.randint(1, 16)
        most = 24_600_000 // (dim * heads)
        batch = _log(rng, 1, 60)
        return dict(op=op, dtype=dtype, batch=batch, tokens=_log(rng, 1, max(1, most // batch)), heads=heads,
                    kv_heads=rng.choice([h for h in range(1, heads + 1) if heads % h == 0]), head_dim=dim,
                    rotary_dim=dim if rng.random() < 0.5 else 2 * rng.randint(2, dim // 2), layout=rng.choice(["interleaved", "half"]),
                    scaling=rng.choice(["none", "linear", "ntk", "yarn"]), factor=rng.choice([2.0, 4.0, 8.0]),
                    far=rng.choice([0, 0, rng.randint(1, 100_000_000)]), inverse=rng.random() < 0.3, strided=rng.random() < 0.3)
    if op in ("norm", "norm_back"):
        groups = rng.choice([1, 1, 2, 4, 8, 32])
        channels = groups * _log(rng, 1, 768 // groups)
        batch = rng.randint(1, 4)
        most = (66_000_000 if op == "norm" else 40_000_000) // (batch * channels)
        least = 1 if op == "norm" else -(-64 * groups // channels)   # a gradient over a few values is all cancellation
        return dict(op=op, dtype=dtype, batch=batch, positions=_log(rng, least, min(most, 172032)), channels=channels, groups=groups,
                    activation=rng.choice(["none", "silu", "gelu"] + ["relu"] * (op == "norm")), params=rng.choice(["f32", dtype]))
    if op in ("gated", "gated_back"):
        features, width = _log(rng, 16, 2048), _log(rng, 16, 5461)
        if rng.random() < 0.5:
            features, width = -(-features // 8) * 8, -(-width // 8) * 8
        most = (13_000_000_000 if op == "gated_back" else 26_000_000_000) // (features * width)
        if dtype == "f32":
            most //= 8
        return dict(op=op, dtype=dtype, rows=_log(rng, 1, max(1, min(48060, most))), features=features, width=width,
                    activation=rng.choice(["silu", "gelu", "sigmoid"]), bias=rng.random() < 0.5)
    bands, stems = rng.choice(["mel", "bs"]), rng.choice([1, 1, 2])
    hidden = _log(rng, 32, 1536)
    if rng.random() < 0.7:
        hidden = -(-hidden // 8) * 8
    chunks = rng.choice([1, 1, 2])
    most = 39_000_000_000 // (4 * 4 * sum(BANDS[bands]) * stems * hidden * chunks)
    if dtype == "f32":
        most //= 8
    return dict(op=op, dtype=dtype, bands=bands, chunks=chunks, stems=stems, frames=max(8, _log(rng, 8, max(8, min(801, most)))), hidden=hidden,
                bias=rng.random() < 0.5)


def work(case):
    c = case
    es = SIZES[c["dtype"]]
    if c["op"] == "rotary":
        n = c["batch"] * c["tokens"] * (c["heads"] + c["kv_heads"]) * c["head_dim"]
        return {"bytes": 2 * n * es + 4 * c["tokens"], "flops": 3 * n}
    if c["op"] in ("norm", "norm_back"):
        n, ps = c["batch"] * c["positions"] * c["channels"], SIZES[c["params"]]
        if c["op"] == "norm":
            return {"bytes": 2 * n * es + 2 * c["channels"] * ps, "flops": 10 * n}
        return {"bytes": 3 * n * es + 4 * c["channels"] * ps, "flops": 20 * n}
    if c["op"] in ("gated", "gated_back"):
        m, k, n = c["rows"], c["features"], c["width"]
        if c["op"] == "gated":
            return {"bytes": (m * k + 2 * n * k + m * n) * es, "flops": 4 * m * n * k}
        return {"bytes": (2 * m * k + 4 * n * k + m * n) * es, "flops": 12 * m * n * k}   # both projections again, dx, dw
    din = 4 * sum(BANDS[c["bands"]])
    rows = c["chunks"] * c["stems"] * c["frames"]
    return {"bytes": (rows * len(BANDS[c["bands"]]) + 2 * c["stems"] * din) * c["hidden"] * es + 4 * rows * din, "flops": 4 * rows * din * c["hidden"]}


def _inputs(case, seed):
    """The case's inputs, from the seed alone."""
    c, dt = case, DTYPES[case["dtype"]]
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, scale=1.0, shift=0.0, dtype=dt):
        return (torch.randn(*shape, generator=gen, device="cuda") * scale + shift).to(dtype)

    if c["op"] == "rotary":
        b, t, h, hk, d = c["batch"], c["tokens"], c["heads"], c["kv_heads"], c["head_dim"]
        if c["strided"]:   # queries, keys and values as one projection wrote them
            qkv = normal(b, t, h + 2 * hk, d)
            q, k = qkv[:, :, :h], qkv[:, :, h:h + hk]
        else:
            q, k = normal(b, t, h, d), normal(b, t, hk, d)
        return dict(q=q, k=k, pos=torch.arange(c["far"], c["far"] + t, dtype=torch.int32, device="cuda"))
    if c["op"] in ("norm", "norm_back"):
        b, p, n, pt = c["batch"], c["positions"], c["channels"], DTYPES[c["params"]]
        x = normal(b, p, n, scale=2.0, shift=0.5)
        s = dict(x=x, gamma=normal(n, scale=0.2, shift=1.0, dtype=pt), beta=normal(n, scale=0.2, dtype=pt))
        if c["op"] == "norm_back":   # the forward pass's statistics are in hand
            s["dy"] = normal(b, p, n)
            g = x.reshape(b, p, c["groups"], -1).double()
            mean = g.mean((1, 3))
            var = (g - mean[:, None, :, None]).square().mean((1, 3))
            s["mean"], s["rstd"] = mean.float(), (var + 1e-5).rsqrt().float()
        return s
    if c["op"] in ("gated", "gated_back"):
        m, k, n = c["rows"], c["features"], c["width"]
        s = dict(x=normal(m, k), wg=normal(n, k, scale=k ** -0.5), wu=normal(n, k, scale=k ** -0.5), bg=None, bu=None)
        if c["bias"]:
            s["bg"], s["bu"] = normal(n, scale=0.3), normal(n, scale=0.3)
        if c["op"] == "gated_back":
            s["dy"] = normal(m, n)
        return s
    nb, din, k = len(BANDS[c["bands"]]), 4 * sum(BANDS[c["bands"]]), c["hidden"]
    hidden = torch.tanh(torch.randn(c["chunks"], c["stems"], nb, c["frames"], k, generator=gen, device="cuda")).to(dt)
    return dict(hidden=hidden, w=normal(c["stems"], 2 * din, k, scale=1.5 * k ** -0.5), b=normal(c["stems"], 2 * din, scale=0.3) if c["bias"] else None)


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if own:   # the handles that a user's program keeps: an engine, and for the mask head the separation's plan
        import __graft_entry__
        pkg = __graft_entry__.load_package()
        s["engine"] = pkg.Engine(torch.cuda.current_device())
        if case["op"] == "head":
            sizes, freqs = pkg.bands.mel_bands() if case["bands"] == "mel" else pkg.bands.bs_bands()
            chunk = HOP * (case["frames"] - 1)
            s["plan"] = s["engine"].plan_roformer(chunk, sizes, freqs, n_stems=case["stems"], hop=HOP, chunk=chunk, num_overlap=1)
    elif case["op"] == "head":
        s.update(_bands(case))
    return s


def run(state):
    c, s = state["case"], state
    if own:
        e = s["engine"]
        if c["op"] == "rotary":
            return e.rotary(s["q"], s["k"], positions=s["pos"], rotary_dim=c["rotary_dim"], layout=c["layout"], scaling=c["scaling"],
                            factor=c["factor"], original_length=4096, inverse=c["inverse"])
        if c["op"] == "norm":
            return e.group_norm(s["x"], c["groups"], s["gamma"], s["beta"], activation=c["activation"])
        if c["op"] == "norm_back":
            return e.group_norm_backward(s["dy"], s["x"], c["groups"], s["gamma"], s["beta"], s["mean"], s["rstd"], activation=c["activation"])
        if c["op"] == "gated":
            return e.gated(s["x"], s["wg"], s["wu"], s["bg"], s["bu"], activation=c["activation"])
        if c["op"] == "gated_back":
            return e.gated_backward(s["dy"], s["x"], s["wg"], s["wu"], s["bg"], s["bu"], activation=c["activation"])
        return s["plan"].mask_head(s["hidden"], s["w"], s["b"])
    return {"rotary": _rotary, "norm": _norm, "norm_back": _norm_back, "gated": _gated, "gated_back": _gated_back, "head": _head}[c["op"]](c, s)


# ---- the plain forms -------------------------------------------------------------------------

def _act(kind, z):
    if kind == "silu":
        return z * torch.sigmoid(z)
    if kind == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if kind == "sigmoid":
        return torch.sigmoid(z)
    return z.clamp_min(0) if kind == "relu" else z


def _act_grad(kind, z):
    if kind == "silu":
        s = torch.sigmoid(z)
        return s * (1 + z * (1 - s))
    if kind == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) * (0.5 / math.pi) ** 0.5
    if kind == "sigmoid":
        s = torch.sigmoid(z)
        return s * (1 - s)
    return (z > 0).to(z.dtype) if kind == "relu" else torch.ones_like(z)


def _frequencies(c, device):
    """(radians a position [rotary_dim / 2] in 64 bits, factor on the rotated values)."""
    half, base, f = c["rotary_dim"] // 2, 10000.0, c["factor"]
    i = torch.arange(half, dtype=torch.float64, device=device)
    if c["scaling"] == "ntk":
        base *= f ** (half / (half - 1))
    freq = base ** (-i / half)
    if c["scaling"] == "linear":
        freq = freq / f
    if c["scaling"] != "yarn":
        return freq, 1.0
    lo, hi = (c["rotary_dim"] * math.log(4096 / (turns * 2 * math.pi)) / (2 * math.log(base)) for turns in (32.0, 1.0))
    lo, hi = max(math.floor(lo), 0), min(math.ceil(hi), half - 1)
    ramp = ((i - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
    return freq * (1 - ramp) + freq / f * ramp, 0.1 * math.log(f) + 1


def _rotary(c, s):
    freq, mag = _frequencies(c, s["q"].device)
    angle = s["pos"].double()[:, None] * freq
    cos, sin = (mag * angle.cos()).float()[None, :, None], (mag * angle.sin()).float()[None, :, None]
    if c["inverse"]:
        sin = -sin
    r = c["rotary_dim"]

    def turn(x):
        y = x.float()
        if c["layout"] == "interleaved":
            a, b = y[..., 0:r:2], y[..., 1:r:2]
            z = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
        else:
            a, b = y[..., :r // 2], y[..., r // 2:r]
            z = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
        return torch.cat((z, y[..., r:]), -1).to(x.dtype)

    return turn(s["q"]), turn(s["k"])


def _norm(c, s):
    x = s["x"].float()
    b, p, n = x.shape
    g = x.view(b, p, c["groups"], -1)
    g = g - g.mean((1, 3), keepdim=True)
    g = g * (g.square().mean((1, 3), keepdim=True) + 1e-5).rsqrt()
    return _act(c["activation"], g.view(b, p, n) * s["gamma"].float() + s["beta"].float()).to(s["x"].dtype)


def _norm_back(c, s):
    x = s["x"].float()
    b, p, n = x.shape
    k = c["groups"]
    gamma, rstd = s["gamma"].float(), s["rstd"][:, None, :, None]
    xh = ((x.view(b, p, k, -1) - s["mean"][:, None, :, None]) * rstd).view(b, p, n)
    dz = s["dy"].float() * _act_grad(c["activation"], xh * gamma + s["beta"].float())
    dgamma, dbeta = (dz * xh).sum((0, 1)), dz.sum((0, 1))
    d, xh = (dz * gamma).view(b, p, k, -1), xh.view(b, p, k, -1)
    dx = rstd * (d - d.mean((1, 3), keepdim=True) - xh * (d * xh).mean((1, 3), keepdim=True))
    return dx.view(b, p, n).to(s["x"].dtype), dgamma.to(s["gamma"].dtype), dbeta.to(s["beta"].dtype)


def _projections(s):
    x = s["x"].float()
    g, u = x @ s["wg"].float().t(), x @ s["wu"].float().t()
    return (g, u) if s["bg"] is None else (g + s["bg"].float(), u + s["bu"].float())


def _gated(c, s):
    g, u = _projections(s)
    return (_act(c["activation"], g) * u).to(s["x"].dtype)


def _gated_back(c, s):
    g, u = _projections(s)
    dy, dt = s["dy"].float(), s["x"].dtype
    dg, du = dy * u * _act_grad(c["activation"], g), dy * _act(c["activation"], g)
    x = s["x"].float()
    out = [dg @ s["wg"].float() + du @ s["wu"].float(), dg.t() @ x, du.t() @ x]
    if s["bg"] is not None:
        out += [dg.sum(0), du.sum(0)]
    return [v.to(dt) for v in out]


def _bands(c):
    """What a program that pads the ragged bands to the widest one keeps: the weights' rows of each band's values and gates, and where
    the padded products have the masks' values."""
    d = 4 * torch.tensor(BANDS[c["bands"]], device="cuda")
    col = torch.arange(int(d.max()), device="cuda")
    values = (2 * (d.cumsum(0) - d))[:, None] + torch.minimum(col, d[:, None] - 1)
    held = (col < d[:, None])[:, None].expand(-1, c["frames"], -1)
    return dict(values=values, gates=values + d[:, None], held=held.flatten().nonzero().flatten())


def _head(c, s):
    x, w = s["hidden"].float(), s["w"].float()
    v, g = x @ w[:, s["values"]].transpose(-1, -2), x @ w[:, s["gates"]].transpose(-1, -2)
    if s["b"] is not None:
        b = s["b"].float()
        v, g = v + b[:, s["values"]][:, :, None], g + b[:, s["gates"]][:, :, None]
    return (v * torch.sigmoid(g)).flatten(2).index_select(2, s["held"]).flatten(1)


# ---- the definitions in 64 bits ---------------------------------------------------------------

def exact(case, seed):
    c, s = case, _inputs(case, seed)
    d = {k: v.double() if v is not None else None for k, v in s.items()}
    kind = c.get("activation")

    def act(z):
        if kind == "silu":
            return z / (1 + torch.exp(-z))
        if kind == "gelu":
            return z * torch.special.ndtr(z)
        if kind == "sigmoid":
            return 1 / (1 + torch.exp(-z))
        return torch.where(z > 0, z, torch.zeros_like(z)) if kind == "relu" else z

    def slope(z):
        z = z.detach().requires_grad_(True)
        with torch.enable_grad():
            return torch.autograd.grad(act(z).sum(), z)[0]

    if c["op"] == "rotary":
        half = c["rotary_dim"] // 2
        freq, mag = [], 1.0
        for i in range(half):
            f = 10000.0 ** (-i / half)
            if c["scaling"] == "linear":
                f /= c["factor"]
            elif c["scaling"] == "ntk":
                f = (10000.0 * c["factor"] ** (half / (half - 1))) ** (-i / half)
            elif c["scaling"] == "yarn":
                at = [half * math.log(4096 / (2 * math.pi * turns)) / math.log(10000.0) for turns in (32.0, 1.0)]
                lo, hi = max(math.floor(at[0]), 0), min(math.ceil(at[1]), half - 1)
                share = min(max((i - lo) / max(hi - lo, 1e-3), 0.0), 1.0)
                f = f * (1 - share) + f / c["factor"] * share
                mag = 1 + 0.1 * math.log(c["factor"])
            freq.append(f)
        angle = d["pos"][:, None] * torch.tensor(freq, dtype=torch.float64, device="cuda") * (-1 if c["inverse"] else 1)
        turn = torch.polar(torch.full_like(angle, mag), angle)[None, :, None]

        def rotated(x):
            head = x[..., :c["rotary_dim"]]
            pairs = head.unflatten(-1, (half, 2)) if c["layout"] == "interleaved" else head.unflatten(-1, (2, half)).transpose(-1, -2)
            z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
            z = z if c["layout"] == "interleaved" else z.transpose(-1, -2)
            return torch.cat((z.reshape(head.shape), x[..., c["rotary_dim"]:]), -1)

        return rotated(d["q"]), rotated(d["k"])
    if c["op"] in ("norm", "norm_back"):
        b, p, n = d["x"].shape
        x = d["x"].reshape(b, p, c["groups"], n // c["groups"])
        gamma, beta = d["gamma"].view(c["groups"], -1), d["beta"].view(c["groups"], -1)
        if c["op"] == "norm":
            var, mean = torch.var_mean(x, (1, 3), correction=0, keepdim=True)
            return act((x - mean) / torch.sqrt(var + 1e-5) * gamma + beta).reshape(b, p, n)
        rstd = d["rstd"][:, None, :, None]
        xh = (x - d["mean"][:, None, :, None]) * rstd
        dz = d["dy"].view_as(x) * slope(xh * gamma + beta)
        dxh, m = dz * gamma, p * (n // c["groups"])
        first, second = dxh.sum((1, 3), keepdim=True) / m, (dxh * xh).sum((1, 3), keepdim=True) / m
        return (rstd * (dxh - first - xh * second)).reshape(b, p, n), torch.einsum("bpgc,bpgc->gc", dz, xh).reshape(-1), dz.sum((0, 1)).reshape(-1)
    if c["op"] in ("gated", "gated_back"):
        zero = torch.zeros((), dtype=torch.float64, device="cuda")
        g = torch.nn.functional.linear(d["x"], d["wg"]) + (zero if d["bg"] is None else d["bg"])
        u = torch.nn.functional.linear(d["x"], d["wu"]) + (zero if d["bu"] is None else d["bu"])
        if c["op"] == "gated":
            return act(g) * u
        dg, du = d["dy"] * u * slope(g), d["dy"] * act(g)
        out = [torch.mm(dg, d["wg"]) + torch.mm(du, d["wu"]), torch.einsum("mn,mk->nk", dg, d["x"]), torch.einsum("mn,mk->nk", du, d["x"])]
        return out + ([dg.sum(0), du.sum(0)] if c["bias"] else [])
    sizes = BANDS[c["bands"]]
    rows = []
    for chunk in range(c["chunks"]):
        for stem in range(c["stems"]):
            at = 0
            for band, size in enumerate(sizes):
                value, gate = d["w"][stem, at:at + 4 * size], d["w"][stem, at + 4 * size:at + 8 * size]
                x = d["hidden"][chunk, stem, band]
                v, g = torch.einsum("tk,nk->tn", x, value), torch.einsum("tk,nk->tn", x, gate)
                if d["b"] is not None:
                    v, g = v + d["b"][stem, at:at + 4 * size], g + d["b"][stem, at + 4 * size:at + 8 * size]
                rows.append((v / (1 + torch.exp(-g))).reshape(-1))
                at += 8 * size
    return torch.cat(rows).view(c["chunks"], -1)
