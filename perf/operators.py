"""Cases of the operators of an encoder layer beside the attention: the embedding of species, the norms of queries and keys with
the rotation by positions, and the gated feed-forward block, forward and backward, over the sizes they are run at.

  embed   ``embedding.embed_species``: scaled rows of a table by id; the gradient of the table by sorted ids
  heads   ``qk_norm.normalize_rotate``: root-mean-square norm of every query and key head, then the rotation by positions
  gated   ``feedforward.gated_feed_forward``: both projections, the activation, the product and the projection back

``train`` cases return the gradients of everything that has one beside the output; the others are a served forward pass.
Sizes are those of the framework's model (128 features, 8 heads of 16, 512 hidden features, 98 species, batches of one crystal up to
4096 crystals of 1-64 atoms) and of wider models of the same build."""
import math

import torch

own = False

TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
SPECIES, MODEL_DIM, FF_DIM, HEADS, HEAD_DIM = 98, 128, 512, 8, 16
EPS = 1e-6


def _embed(rows, ids, dim, dtype="float32", layout="table", padding=False, train=True, scale=0.25):
    return dict(op="embed", rows=rows, ids=ids, dim=dim, dtype=dtype, layout=layout, padding=padding, train=train, scale=scale)


def _heads(rows, q_heads, k_heads, dim, pairs, axes, dtype="float32", interleaved=False, wave_heads=1, weights="shared", reach=1.0,
           joint=True, train=True):
    return dict(op="heads", rows=rows, q_heads=q_heads, k_heads=k_heads, dim=dim, pairs=pairs, axes=axes, dtype=dtype,
                interleaved=interleaved, wave_heads=wave_heads, weights=weights, reach=reach, joint=joint, train=train)


def _gated(rows, dim, hidden, dtype="float32", act="silu", bias=True, train=True):
    return dict(op="gated", rows=rows, dim=dim, hidden=hidden, dtype=dtype, act=act, bias=bias, train=train)


def listed():
    cases = {
        # one structure of eight atoms, as an interactive prediction asks for: launches and host time
        "embed-single": _embed(8, SPECIES, MODEL_DIM, train=False),
        # a training step on 4096 crystals: few ids, each of them some thousand times; the table is the model's Linear weight
        "embed-species-train": _embed(133120, SPECIES, MODEL_DIM, layout="linear"),
        # a large vocabulary of site labels (species, charge, environment) of uneven frequency, some rows padded
        "embed-labels-train": _embed(32768, 50021, 1024, "bfloat16", padding=True),
        # one small crystal in a model of grouped heads with part of the head rotated: odd sizes, latency
        "heads-ragged-serve": _heads(17, 12, 4, 80, 20, 3, "float16", interleaved=True, train=False),
        # a training step on 4096 crystals: eight heads of sixteen, a set of waves for each head, fractional coordinates
        "heads-crystals-train": _heads(133120, HEADS, HEADS, HEAD_DIM, HEAD_DIM // 2, 3, wave_heads=HEADS, weights="each"),
        # long sequences of a wider model: shared key heads, one position axis, positions far from the origin
        "heads-long-train": _heads(16384, 32, 8, 128, 64, 1, "bfloat16", reach=1e6),
        # one atom through the model's own sizes: latency
        "gated-single": _gated(1, MODEL_DIM, FF_DIM, train=False),
        # four rows through a wide block: the weights are all there is to read
        "gated-few-rows": _gated(4, 2048, 5632, "bfloat16", bias=False, train=False),
        # a training step on the benchmark's batch of 128 crystals
        "gated-batch-train": _gated(1984, MODEL_DIM, FF_DIM),
        # a training step on 4096 crystals
        "gated-crystals-train": _gated(133120, MODEL_DIM, FF_DIM),
        # odd sizes everywhere: rows that are no multiple of 16 bytes
        "gated-ragged-train": _gated(4999, 201, 517, "float16", act="gelu"),
        # a training step of a wide model
        "gated-wide-train": _gated(8192, 1024, 2816, "bfloat16", bias=False),
    }
    return [dict(c, name=n) for n, c in cases.items()]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("embed", "heads", "gated"))
    dtype = rng.choice(tuple(TYPES))
    train = rng.random() < 0.7
    if op == "embed":
        dim = _log(rng, 16, 2048)
        return _embed(_log(rng, 1, 30_000_000 // dim if dim > 150 else 200_000), _log(rng, 2, 50_000_000 // dim if dim > 500 else 100_000), dim, dtype,
                      rng.choice(("table", "linear")), rng.random() < 0.5, train, rng.choice((1.0, 0.25, 3.7)))
    if op == "heads":
        k_heads, dim = rng.randint(1, 8), rng.choice((16, 16, 32, 64, 128)) if rng.random() < 0.6 else rng.randint(8, 200)
        q_heads = k_heads * rng.choice((1, 1, 2, 3, 4))
        pairs = rng.choice((dim // 2, dim // 2, dim // 4, 0))
        axes = rng.randint(1, 3)
        return _heads(_log(rng, 1, min(150_000, 60_000_000 // (dim * (q_heads + k_heads)))), q_heads, k_heads, dim, pairs, axes, dtype,
                      rng.random() < 0.5, rng.choice((1, k_heads)), rng.choice(("shared", "each", "none")),
                      1.0 if axes == 3 else 10.0 ** rng.uniform(0, 6), rng.random() < 0.5, train)
    dim, hidden = _log(rng, 16, 2048), _log(rng, 16, 6000)
    rows = _log(rng, 1, min(133_120, 23_000_000_000 // (dim * hidden), 60_000_000 // max(dim, hidden)) if dtype != "float32"
                else min(133_120, 8_000_000_000 // (dim * hidden), 60_000_000 // max(dim, hidden)))
    return _gated(rows, dim, hidden, dtype, rng.choice(("silu", "gelu", "relu")), rng.random() < 0.5, train)


def prepare(case, seed):
    c, dtype = dict(case), TYPES[case["dtype"]]
    gen = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *shape, std=1.0: torch.randn(shape, generator=gen, device="cuda").mul_(std).to(dtype)  # noqa: E731
    uniform = lambda *shape: torch.rand(shape, generator=gen, device="cuda")  # noqa: E731
    s = dict(case=c)
    if c["op"] == "embed":
        # ids of uneven frequency, as species and labels have
        ids = uniform(c["rows"]).mul_(math.log(c["ids"] + 1)).exp_().to(torch.int64).sub_(1).clamp_(0, c["ids"] - 1)
        ids = torch.randperm(c["ids"], generator=gen, device="cuda")[ids]
        if c["padding"]:
            ids = torch.where(uniform(c["rows"]) < 0.05, -1, ids)
        shape = (c["ids"], c["dim"]) if c["layout"] == "table" else (c["dim"], c["ids"])
        s.update(ids=ids, weight=normal(*shape, std=0.1).requires_grad_(c["train"]))
        s["gout"] = normal(c["rows"], c["dim"])
    elif c["op"] == "heads":
        N, D = c["rows"], c["dim"]
        width = (c["q_heads"] + c["k_heads"]) * D
        if c["joint"]:  # queries and keys as views into one projection, with the values behind them
            both = normal(N, width + c["k_heads"] * D, std=1.5)
            q, k = both[:, :c["q_heads"] * D], both[:, c["q_heads"] * D:width]
        else:
            q, k = normal(N, c["q_heads"] * D, std=1.5), normal(N, c["k_heads"] * D, std=1.5)
        weight = lambda heads: None if c["weights"] == "none" else (  # noqa: E731
            1 + 0.2 * torch.randn((heads, D) if c["weights"] == "each" else (D,), generator=gen, device="cuda")).to(dtype)
        s.update(q=q.view(N, c["q_heads"], D), k=k.view(N, c["k_heads"], D), wq=weight(c["q_heads"]), wk=weight(c["k_heads"]))
        if c["axes"] == 3:  # fractional coordinates and whole waves
            s["pos"] = uniform(N, 3)
            s["waves"] = torch.randint(-4, 5, (c["wave_heads"], c["pairs"], 3), generator=gen, device="cuda").float()
        else:  # whole positions up to the reach, wave lengths from six to some ten thousand positions
            s["pos"] = uniform(N, c["axes"]).mul_(c["reach"]).floor_()
            s["waves"] = (-uniform(c["wave_heads"], c["pairs"], c["axes"]).mul_(math.log(10000.0))).exp_().div_(2 * math.pi)
        for n in ("q", "k", "wq", "wk"):
            if c["train"] and s[n] is not None:
                s[n] = s[n].detach().requires_grad_()
        s["gq"], s["gk"] = normal(N, c["q_heads"], D), normal(N, c["k_heads"], D)
    else:
        N, D, F = c["rows"], c["dim"], c["hidden"]
        s.update(x=normal(N, D), w_gate=normal(F, D, std=D ** -0.5), w_up=normal(F, D, std=D ** -0.5), w_down=normal(D, F, std=F ** -0.5))
        s.update(b_gate=normal(F, std=0.1) if c["bias"] else None, b_up=normal(F, std=0.1) if c["bias"] else None,
                 b_down=normal(D, std=0.1) if c["bias"] else None)
        for n in ("x", "w_gate", "w_up", "w_down", "b_gate", "b_up", "b_down"):
            if c["train"] and s[n] is not None:
                s[n].requires_grad_()
        s["gy"] = normal(N, D)
    return s


# ---- the framework's operators, as a user calls them ------------------------------------------------------------------------
def _gradients(outputs, leaves, gradients):
    leaves = [t for t in leaves if t is not None]
    return torch.autograd.grad(outputs, leaves, gradients)


def _own_embed(s):
    from crystalformer_b200.embedding import embed_species
    c, w = s["case"], s["weight"]
    out = embed_species(s["ids"], w if c["layout"] == "table" else w.t(), c["scale"])
    return (out, *_gradients(out, (w,), (s["gout"],))) if c["train"] else out


def _own_heads(s):
    from crystalformer_b200.qk_norm import normalize_rotate
    c = s["case"]
    q, k = normalize_rotate(s["q"], s["k"], s["wq"], s["wk"], s["pos"], s["waves"], eps=EPS, interleaved=c["interleaved"])
    return (q, k, *_gradients((q, k), (s["q"], s["k"], s["wq"], s["wk"]), (s["gq"], s["gk"]))) if c["train"] else (q, k)


def _own_gated(s):
    from crystalformer_b200.feedforward import gated_feed_forward
    c, names = s["case"], ("x", "w_gate", "w_up", "w_down", "b_gate", "b_up", "b_down")
    y = gated_feed_forward(*(s[n] for n in names), activation=c["act"])
    return (y, *_gradients(y, [s[n] for n in names], (s["gy"],))) if c["train"] else y


# ---- plain forms ------------------------------------------------------------------------------------------------------------
def _plain_embed(s):
    c, dtype = s["case"], TYPES[s["case"]["dtype"]]
    ids, w = s["ids"], s["weight"].detach()
    valid = (ids >= 0) & (ids < c["ids"])
    at = torch.where(valid, ids, 0)
    rows = w[at] if c["layout"] == "table" else w.t()[at]
    out = torch.where(valid[:, None], rows.float() * c["scale"], 0.0).to(dtype)
    if not c["train"]:
        return out
    g = torch.where(valid[:, None], s["gout"].float() * c["scale"], 0.0)
    gw = torch.zeros((c["ids"], c["dim"]), device=g.device).index_add_(0, at, g)
    return out, (gw if c["layout"] == "table" else gw.t().contiguous()).to(dtype)


def _angles(s, heads):
    """Cosine and sine (rows, heads, pairs): the angles of far positions need 64 bits until they are reduced."""
    turns = (s["pos"].double()[:, None, None, :] * s["waves"].double()).sum(-1)
    theta = ((turns - turns.round()) * (2 * math.pi)).float()
    cos, sin = theta.cos(), theta.sin()
    if cos.shape[1] > 1 and heads != cos.shape[1]:
        cos, sin = (t.repeat_interleave(heads // t.shape[1], dim=1) for t in (cos, sin))
    return cos, sin


def _turn(x, cos, sin, pairs, interleaved, back=False):
    """x with its pairs turned by the angles (``back``: by their negatives)."""
    sin = -sin if back else sin
    if interleaved:
        a, b = x[..., 0:2 * pairs:2], x[..., 1:2 * pairs:2]
    else:
        a, b = x[..., :pairs], x[..., pairs:2 * pairs]
    y = x.clone()
    u, v = a * cos - b * sin, a * sin + b * cos
    if interleaved:
        y[..., 0:2 * pairs:2], y[..., 1:2 * pairs:2] = u, v
    else:
        y[..., :pairs], y[..., pairs:2 * pairs] = u, v
    return y


def _plain_heads(s):
    c, dtype = s["case"], TYPES[s["case"]["dtype"]]
    outs, grads, wgrads = [], [], []
    for x, w, g in ((s["q"], s["wq"], s["gq"]), (s["k"], s["wk"], s["gk"])):
        x = x.detach().float()
        cos, sin = _angles(s, x.shape[1])
        r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
        n = x * r
        y = n if w is None else n * w.detach().float()
        outs.append(_turn(y, cos, sin, c["pairs"], c["interleaved"]).to(dtype))
        if c["train"]:
            g = _turn(g.float(), cos, sin, c["pairs"], c["interleaved"], back=True)
            if w is not None:
                wgrads.append(((g * n).sum(0) if w.dim() == 2 else (g * n).sum((0, 1))).to(dtype))
                g = g * w.detach().float()
            grads.append((r * (g - n * (g * n).mean(-1, keepdim=True))).to(dtype))
    return (*outs, *grads, *wgrads)


def _plain_gated(s):
    c, dtype = s["case"], TYPES[s["case"]["dtype"]]
    f = {n: None if s[n] is None else s[n].detach().float() for n in ("x", "w_gate", "w_up", "w_down", "b_gate", "b_up", "b_down")}
    plus = lambda t, b: t if b is None else t + b  # noqa: E731
    g = plus(f["x"] @ f["w_gate"].t(), f["b_gate"])
    u = plus(f["x"] @ f["w_up"].t(), f["b_up"])
    if c["act"] == "silu":
        p = 1 / (1 + torch.exp(-g))
        a, da = g * p, p * (1 + g * (1 - p)) if c["train"] else None
    elif c["act"] == "gelu":
        p = 0.5 * (1 + torch.erf(g * 0.5 ** 0.5))
        a, da = g * p, p + g * torch.exp(-0.5 * g * g) * (2 * math.pi) ** -0.5 if c["train"] else None
    else:
        a, da = torch.where(g > 0, g, 0.0), (g > 0).float()
    h = a * u
    y = plus(h @ f["w_down"].t(), f["b_down"]).to(dtype)
    if not c["train"]:
        return y
    gy = s["gy"].float()
    dh = gy @ f["w_down"]
    dg, du = dh * u * da, dh * a
    grads = [dg @ f["w_gate"] + du @ f["w_up"], dg.t() @ f["x"], du.t() @ f["x"], gy.t() @ h]
    if c["bias"]:
        grads += [dg.sum(0), du.sum(0), gy.sum(0)]
    return (y, *(t.to(dtype) for t in grads))


def run(state):
    op = state["case"]["op"]
    if own:
        return {"embed": _own_embed, "heads": _own_heads, "gated": _own_gated}[op](state)
    with torch.no_grad():
        return {"embed": _plain_embed, "heads": _plain_heads, "gated": _plain_gated}[op](state)


# ---- what a pass cannot do without ---------------------------------------------------------------------------------------------
def work(case):
    c, size = case, TYPES[case["dtype"]].itemsize
    if c["op"] == "embed":
        rows = c["rows"] * c["dim"]
        n = 8 * c["rows"] + size * (rows + min(c["rows"], c["ids"]) * c["dim"])
        return dict(bytes=n + (size * (rows + c["ids"] * c["dim"]) if c["train"] else 0), flops=rows * (2 if c["train"] else 1))
    if c["op"] == "heads":
        n = c["rows"] * (c["q_heads"] + c["k_heads"]) * c["dim"]
        angles = 4 * c["axes"] * (c["rows"] + c["wave_heads"] * c["pairs"])
        # forward: read and written; backward: inputs and gradients read, gradients written
        return dict(bytes=size * n * (4 if c["train"] else 2) + angles, flops=n * (22 if c["train"] else 8))
    N, D, F = c["rows"], c["dim"], c["hidden"]
    weights = 3 * D * F + ((2 * F + D) if c["bias"] else 0)
    return dict(bytes=size * ((4 * N * D + 2 * weights) if c["train"] else (2 * N * D + weights)), flops=6 * N * D * F * (3 if c["train"] else 1))


# ---- from the definitions, in 64 bits ------------------------------------------------------------------------------------------
def exact(case, seed):
    c, s = case, prepare(case, seed)
    leaf = lambda t: None if t is None else t.detach().double().requires_grad_(c["train"])  # noqa: E731
    with torch.enable_grad():
        if c["op"] == "embed":
            w = leaf(s["weight"])
            table = torch.cat(((w if c["layout"] == "table" else w.transpose(0, 1)) * c["scale"], torch.zeros((1, c["dim"]), dtype=torch.float64, device="cuda")))
            ids = s["ids"]
            out = table.index_select(0, ids.masked_fill((ids < 0) | (ids >= c["ids"]), c["ids"]))
            outs, leaves, gs = (out,), (w,), (s["gout"],)
        elif c["op"] == "heads":
            leaves, outs = [leaf(s[n]) for n in ("q", "k", "wq", "wk")], []
            for x, w in zip(leaves[:2], leaves[2:]):
                N, H, D, P = *x.shape, c["pairs"]
                y = x / x.square().mean(2, keepdim=True).add(EPS).sqrt()
                y = y if w is None else y * w
                phase = torch.einsum("nc,hpc->nhp", s["pos"].double(), s["waves"].double())
                phase = phase.unsqueeze(2).expand(N, c["wave_heads"], H // c["wave_heads"], P).reshape(N, H, P)
                turn = torch.polar(torch.ones_like(phase), 2 * math.pi * torch.frac(phase))
                head = y[..., :2 * P]
                pair = head.unflatten(-1, (P, 2)) if c["interleaved"] else head.unflatten(-1, (2, P)).transpose(-1, -2)
                z = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * turn)
                z = z.flatten(-2) if c["interleaved"] else z.transpose(-1, -2).flatten(-2)
                outs.append(torch.cat((z, y[..., 2 * P:]), -1))
            gs = (s["gq"], s["gk"])
        else:
            leaves = [leaf(s[n]) for n in ("x", "w_gate", "w_up", "w_down", "b_gate", "b_up", "b_down")]
            x, wg, wu, wd, bg, bu, bd = leaves
            act = dict(silu=torch.nn.functional.silu, gelu=torch.nn.functional.gelu, relu=torch.relu)[c["act"]]
            linear = torch.nn.functional.linear
            outs, gs = (linear(act(linear(x, wg, bg)) * linear(x, wu, bu), wd, bd),), (s["gy"],)
        if not c["train"]:
            return outs if c["op"] == "heads" else outs[0]
        grads = torch.autograd.grad(outs, [t for t in leaves if t is not None], [g.double() for g in gs])
    return (*(t.detach() for t in outs), *grads)
