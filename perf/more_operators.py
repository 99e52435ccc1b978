"""Performance cases of the operators inside a training step's transformer block.

Three operators, each in its plain form (``own`` false: elementary torch operations in 32 bits, 64
where 32 lose what matters, rounded once) and through the package's public entry points (``own``
true): the gated feed-forward block with its backward pass, rotary positions with several axes,
and dropout from a counter-based generator alone, with the residual sum, and with the next norm.
A case is a plain dict; ``op`` selects one of the handlers at the end of the file. ``draw`` spreads
over the ranges between the listed cases.
"""
from __future__ import annotations

import math

import torch

own = False

DEVICE = "cuda:0"
EPS = 1e-6
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # one token through a 768-wide model's feed-forward block: launch and host time
        dict(name="ffn_token_768", op="ffn", tokens=1, hidden=768, inter=2048, dtype="fp16",
             act="gelu_tanh", down=True, train=False),
        # one decoding step of 16 sequences of an 8B model: the weights are read once
        dict(name="ffn_decode_8b", op="ffn", tokens=16, hidden=4096, inter=14336, dtype="bf16",
             act="silu", down=True, train=False),
        # a ragged batch of a 768-wide model in training, GELU
        dict(name="ffn_train_768", op="ffn", tokens=2045, hidden=768, inter=2048, dtype="fp16",
             act="gelu_tanh", down=True, train=True),
        # an 8B model in training, 4 sequences of 2048 tokens
        dict(name="ffn_train_8b", op="ffn", tokens=8192, hidden=4096, inter=14336, dtype="bf16",
             act="silu", down=True, train=True),
        # one decoding step of 16 sequences behind images, positions along time, height and width
        dict(name="rope_decode", op="rope", batch=16, seq=1, heads=32, kv_heads=8, dim=128,
             rotary=128, axes=3, layout="blocks", dtype="bf16", start=30000, packed=False,
             train=False),
        # a vision encoder's patches, 37 x 37 of them, a progression for each of the two axes
        dict(name="rope_vision", op="rope", batch=8, seq=1369, heads=16, kv_heads=16, dim=80,
             rotary=80, axes=2, layout="separate", dtype="fp16", start=0, packed=True, train=True),
        # a packed row of text and video in training, the axes interleaved
        dict(name="rope_video", op="rope", batch=1, seq=32768, heads=64, kv_heads=8, dim=128,
             rotary=128, axes=3, layout="interleaved", dtype="bf16", start=0, packed=False,
             train=True),
        # a small batch of a 768-wide model in fp32: the residual sum of one block
        dict(name="dropout_add_768", op="dropout", kind="add", rows=258, cols=768, dtype="fp32",
             p=0.1, train=True),
        # the same model's block boundary, a ragged batch
        dict(name="dropout_norm_768", op="dropout", kind="norm", rows=8191, cols=768,
             dtype="fp32", p=0.1, train=True),
        # the boundary of an 8B-class model in training
        dict(name="dropout_norm_8b", op="dropout", kind="norm", rows=16384, cols=4096,
             dtype="bf16", p=0.1, train=True),
        # an 8B-class feed-forward block's activations
        dict(name="dropout_plain_8b", op="dropout", kind="plain", rows=8192, cols=14336,
             dtype="bf16", p=0.05, train=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["ffn", "ffn", "rope", "dropout"])
    if op == "ffn":
        hidden, inter = _log_int(rng, 64, 4096), _log_int(rng, 64, 14336)
        if rng.random() < 0.8:
            hidden, inter = hidden // 64 * 64, inter // 64 * 64
        return dict(op=op, tokens=_log_int(rng, 1, 8192), hidden=hidden, inter=inter,
                    dtype=rng.choice(["bf16", "bf16", "fp16"]),
                    act=rng.choice(["silu", "silu", "gelu_tanh", "gelu", "relu"]),
                    down=rng.random() < 0.75, train=rng.random() < 0.6)
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op == "rope":
        dim = rng.choice([32, 64, 72, 80, 96, 128, 128, 256])
        kv = rng.choice([1, 2, 4, 8, 16])
        heads = kv * rng.choice([1, 2, 4])
        most = (32768 * 72 * 128 // 2) // (dim * (heads + kv))
        batch = rng.choice([1, 2, 3, 8, 16])
        return dict(op=op, batch=batch, seq=_log_int(rng, 1, min(32768, most // batch)),
                    heads=heads, kv_heads=kv, dim=dim,
                    rotary=rng.choice([dim, dim, dim, dim // 4 * 2]),
                    axes=rng.choice([2, 3, 3, 4]),
                    layout=rng.choice(["blocks", "interleaved", "separate"]), dtype=dtype,
                    start=rng.choice([0, 0, 5000, 1000000]), packed=rng.random() < 0.5,
                    train=rng.random() < 0.7)
    cols = _log_int(rng, 16, 8192)
    if rng.random() < 0.7:
        cols = max(16, cols // 64 * 64)
    return dict(op=op, kind=rng.choice(["plain", "add", "norm", "norm"]),
                rows=_log_int(rng, 1, max(2, (1 << 26) // cols)), cols=cols, dtype=dtype,
                p=rng.choice([0.05, 0.1, 0.1, 0.5]), train=rng.random() < 0.8)


# ---------------------------------------------------------------------------
# Inputs: seeded on the device
# ---------------------------------------------------------------------------

class _Inputs:
    def __init__(self, seed, dtype="bf16"):
        self.g = torch.Generator(device=DEVICE)
        self.g.manual_seed(int(seed))
        self.dtype = DTYPES.get(dtype)

    def randn(self, *shape, std=1.0, mean=0.0):
        t = torch.randn(shape, generator=self.g, device=DEVICE, dtype=torch.float32)
        return t.mul_(std).add_(mean).to(self.dtype)


def _elt(c):
    return 4 if c["dtype"] == "fp32" else 2


def prepare(case, seed):
    return _HANDLERS[case["op"]][0](case, seed)


def run(state):
    return _HANDLERS[state["c"]["op"]][1](state)


def work(case):
    return _HANDLERS[case["op"]][2](case)


def exact(case, seed):
    return _HANDLERS[case["op"]][3](case, seed)


# ---------------------------------------------------------------------------
# Gated feed-forward block: a = act(x Wg^T) * (x Wu^T), y = a Wd^T (down false: y = a)
# ---------------------------------------------------------------------------

def _ffn_prepare(c, seed):
    i = _Inputs(seed, c["dtype"])
    n, h, f = c["tokens"], c["hidden"], c["inter"]
    s = dict(c=c, x=i.randn(n, h), wg=i.randn(f, h, std=1.5 / math.sqrt(h)),
             wu=i.randn(f, h, std=1 / math.sqrt(h)))
    if c["down"]:
        s["wd"] = i.randn(h, f, std=1 / math.sqrt(f))
    if c["train"]:
        for k in ("x", "wg", "wu", "wd"):
            if k in s:
                s[k].requires_grad_()
        s["dy"] = i.randn(n, h if c["down"] else f)
    return s


def _ffn_act(act, g):
    """act(g) and its derivative."""
    if act == "relu":
        pos = (g > 0).to(g.dtype)
        return g * pos, pos
    if act == "silu":
        sg = 1 / (1 + torch.exp(-g))
        return g * sg, sg * (1 + g * (1 - sg))
    if act == "gelu_tanh":
        k = math.sqrt(2 / math.pi)
        th = torch.tanh(k * (g + 0.044715 * g * g * g))
        return (0.5 * g * (1 + th),
                0.5 * (1 + th) + 0.5 * g * (1 - th * th) * k * (1 + 3 * 0.044715 * g * g))
    cdf = 0.5 * torch.erfc(g * -math.sqrt(0.5))
    return g * cdf, cdf + g * torch.exp(-0.5 * g * g) / math.sqrt(2 * math.pi)


def _ffn_run(s):
    c = s["c"]
    names = [k for k in ("x", "wg", "wu", "wd") if k in s]
    if own:
        from trainscale_amd.kernels import fused_gated_linear, fused_gated_mlp
        if c["down"]:
            y = fused_gated_mlp(s["x"], s["wg"], s["wu"], s["wd"], activation=c["act"])
        else:
            y = fused_gated_linear(s["x"], s["wg"], s["wu"], activation=c["act"])
        if not c["train"]:
            return y
        grads = torch.autograd.grad(y, [s[k] for k in names], s["dy"])
        return dict(y=y, **{"d" + k: g for k, g in zip(names, grads)})
    dtype = s["x"].dtype
    x, wg, wu = (s[k].detach().float() for k in ("x", "wg", "wu"))
    g, u = x @ wg.t(), x @ wu.t()
    t, dt = _ffn_act(c["act"], g)
    a = t * u
    wd = s["wd"].detach().float() if c["down"] else None
    y = a if wd is None else a @ wd.t()
    if not c["train"]:
        return y.to(dtype)
    out = dict(y=y.to(dtype))
    dy = s["dy"].float()
    da = dy if wd is None else dy @ wd
    dg, du = da * u * dt, da * t
    out["dx"] = (dg @ wg + du @ wu).to(dtype)
    out["dwg"] = (dg.t() @ x).to(dtype)
    out["dwu"] = (du.t() @ x).to(dtype)
    if wd is not None:
        out["dwd"] = (dy.t() @ a).to(dtype)
    return out


def _ffn_work(c):
    n, h, f, m = c["tokens"], c["hidden"], c["inter"], 3 if c["down"] else 2
    out = h if c["down"] else f
    moved = n * h + m * h * f + n * out
    if c["train"]:
        moved += n * out + n * h + m * h * f
    return dict(bytes=2 * moved, flops=2 * m * n * h * f * (3 if c["train"] else 1))


def _ffn_exact(c, seed):
    s = _ffn_prepare(c, seed)
    leaf = {k: s[k].detach().double().requires_grad_(c["train"])
            for k in ("x", "wg", "wu", "wd") if k in s}
    g = torch.mm(leaf["x"], leaf["wg"].t())
    u = torch.mm(leaf["x"], leaf["wu"].t())
    if c["act"] == "relu":
        t = torch.where(g > 0, g, torch.zeros_like(g))
    elif c["act"] == "silu":
        t = g * torch.sigmoid(g)
    elif c["act"] == "gelu_tanh":  # (1 + tanh z) / 2 = sigmoid(2 z)
        t = g * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (g + 0.044715 * g.pow(3)))
    else:
        t = g * torch.special.ndtr(g)
    y = t * u
    if c["down"]:
        y = torch.mm(y, leaf["wd"].t())
    if not c["train"]:
        return y
    grads = torch.autograd.grad(y, list(leaf.values()), s["dy"].double())
    return dict(y=y.detach(), **{"d" + k: v for k, v in zip(leaf, grads)})


# ---------------------------------------------------------------------------
# Rotary positions with several axes: pair (i, i + R/2) of a head's first R elements turned by
# pos[axis(i)] f(i); the elements behind them stay
# ---------------------------------------------------------------------------

def _rope_sections(c):
    half, a = c["rotary"] // 2, c["axes"]
    rest = half // a if c["layout"] == "separate" else half * 3 // (4 * a) if a > 2 else half // a
    return [half - rest * (a - 1)] + [rest] * (a - 1)


def _rope_freq(c):
    """The fp32 frequency and the axis of each pair."""
    sec, base, half = _rope_sections(c), 500000.0, c["rotary"] // 2
    one = lambda n: 1.0 / (base ** (torch.arange(0, 2 * n, 2, dtype=torch.float32) / (2 * n)))
    if c["layout"] == "separate":
        return torch.cat([one(n) for n in sec]), [a for a, n in enumerate(sec) for _ in range(n)]
    if c["layout"] == "blocks":
        return one(half), [a for a, n in enumerate(sec) for _ in range(n)]
    axis = [i % len(sec) if i < len(sec) * sec[i % len(sec)] else 0 for i in range(half)]
    return one(half), axis


def _rope_prepare(c, seed):
    i = _Inputs(seed, c["dtype"])
    b, n, d = c["batch"], c["seq"], c["dim"]
    hq, hk = c["heads"], c["kv_heads"]
    if c["packed"]:  # views into one projection's output
        qkv = i.randn(b, n, hq + 2 * hk, d)
        q, k = qkv[:, :, :hq], qkv[:, :, hq:hq + hk]
    else:
        q, k = i.randn(b, n, hq, d), i.randn(b, n, hk, d)
    s = dict(c=c, q=q.detach().requires_grad_(c["train"]), k=k.detach().requires_grad_(c["train"]))
    # rows of text with grids of patches between them: in a grid the axes count frames, rows and
    # columns, in text all axes count tokens
    t = torch.arange(n, device=DEVICE)
    side = max(1, int(math.sqrt(min(n, 4096)) * 0.7))
    at = t % (side * side + 64) - 64
    grid = [t // (side * side + 64), at // side, at % side, at % 7]
    pos = torch.stack([torch.where(at < 0, t, t // 2 + grid[a]) for a in range(c["axes"])])
    lag = torch.randint(0, 50, (c["axes"], b, 1), generator=i.g, device=DEVICE)
    s["pos"] = pos[:, None, :] + lag + c["start"]
    freq, axis = _rope_freq(c)
    s["freq"], s["axis"] = freq.to(DEVICE), torch.tensor(axis, device=DEVICE)
    if own:
        from trainscale_amd.kernels import RopeAxes
        s["plan"] = RopeAxes(_rope_sections(c), layout=c["layout"], inv_freq=freq)
    if c["train"]:
        s.update(dq=i.randn(b, n, hq, d), dk=i.randn(b, n, hk, d))
    return s


def _rope_run(s):
    c = s["c"]
    if own:
        from trainscale_amd.kernels import apply_rope_axes
        q, k = apply_rope_axes(s["q"], s["k"], s["pos"], s["plan"])
        if not c["train"]:
            return dict(q=q, k=k)
        dq, dk = torch.autograd.grad((q, k), (s["q"], s["k"]), (s["dq"], s["dk"]))
        return dict(q=q, k=k, dq=dq, dk=dk)
    # the angles of far positions in 64 bits
    angle = s["pos"].double()[s["axis"]].permute(1, 2, 0) * s["freq"].double()
    cos, sin = angle.cos().float()[:, :, None], angle.sin().float()[:, :, None]
    half = c["rotary"] // 2

    def turn(x, sin):
        x1, x2 = x[..., :half].float(), x[..., half:2 * half].float()
        return torch.cat([(x1 * cos - x2 * sin).to(x.dtype), (x2 * cos + x1 * sin).to(x.dtype),
                          x[..., 2 * half:]], -1)

    out = dict(q=turn(s["q"].detach(), sin), k=turn(s["k"].detach(), sin))
    if c["train"]:
        out.update(dq=turn(s["dq"], -sin), dk=turn(s["dk"], -sin))
    return out


def _rope_work(c):
    tokens, passes = c["batch"] * c["seq"], 2 if c["train"] else 1
    n = tokens * (c["heads"] + c["kv_heads"]) * c["dim"]
    return dict(bytes=passes * (2 * n * _elt(c) + 8 * c["axes"] * tokens), flops=passes * 3 * n)


def _rope_exact(c, seed):
    s = _rope_prepare(c, seed)
    freq, axis = _rope_freq(c)
    half = c["rotary"] // 2
    cols = [s["pos"][axis[i]].double() * float(freq[i]) for i in range(half)]
    z = torch.polar(torch.ones((), dtype=torch.float64, device=DEVICE),
                    torch.stack(cols, -1))[:, :, None]

    def turn(x, z):
        w = torch.view_as_real(torch.complex(x[..., :half].double(),
                                             x[..., half:2 * half].double()) * z)
        return torch.cat([w[..., 0], w[..., 1], x[..., 2 * half:].double()], -1)

    out = dict(q=turn(s["q"].detach(), z), k=turn(s["k"].detach(), z))
    if c["train"]:
        out.update(dq=turn(s["dq"], z.conj()), dk=turn(s["dk"], z.conj()))
    return out


# ---------------------------------------------------------------------------
# Dropout from a counter-based generator: element (r, c) is kept where its 16 random bits are at
# least round(65536 p), and kept elements are divided by the probability of being kept. The bits
# are those of Philox 4x32 with 10 rounds (Salmon, Moraes, Dror and Shaw, 2011) under key `seed`
# for the counter (r ceil(cols / 8) + c / 8, offset): 8 elements a counter, low halves first.
# "plain": y = D(x). "add": h = residual + D(x). "norm": also y = h rstd(h) w
# ---------------------------------------------------------------------------

def _dropout_prepare(c, seed):
    i = _Inputs(seed, c["dtype"])
    n, m = c["rows"], c["cols"]
    s = dict(c=c, x=i.randn(n, m, std=0.7),
             rng=(((seed * 7919 + 1) << 20 | 12345) % (1 << 63), seed + 3))
    if c["kind"] != "plain":
        s["res"] = i.randn(n, m, std=2.0)
    if c["kind"] == "norm":
        s["w"] = i.randn(m, std=0.1, mean=1.0)
    if c["train"]:
        for k in ("x", "res", "w"):
            if k in s:
                s[k].requires_grad_()
        s["dy"] = i.randn(n, m)
        if c["kind"] == "norm":
            s["dh"] = i.randn(n, m)
    return s


def _dropout_keep(c, rng):
    """The kept elements, [rows, cols]."""
    groups, low = (c["cols"] + 7) // 8, 0xFFFFFFFF
    n = torch.arange(c["rows"] * groups, device=DEVICE)
    a, b = n & low, n >> 32
    x, y = torch.full_like(n, rng[1] & low), torch.full_like(n, rng[1] >> 32)
    k0, k1 = rng[0] & low, rng[0] >> 32 & low
    for _ in range(10):
        p, q = a * 0xD2511F53, x * 0xCD9E8D57  # modulo 2^64, in two's complement
        a, b, x, y = (q >> 32 & low) ^ b ^ k0, q & low, (p >> 32 & low) ^ y ^ k1, p & low
        k0, k1 = k0 + 0x9E3779B9 & low, k1 + 0xBB67AE85 & low
    bits = torch.stack([t >> h & 0xFFFF for t in (a, b, x, y) for h in (0, 16)], -1)
    bits = bits.view(c["rows"], groups * 8)[:, :c["cols"]]
    return bits >= round(c["p"] * 65536)


def _dropout_run(s):
    c = s["c"]
    names = [k for k in ("x", "res", "w") if k in s]
    if own:
        from trainscale_amd.kernels import (fused_dropout, fused_dropout_add,
                                            fused_dropout_add_rms_layernorm)
        if c["kind"] == "plain":
            out = dict(y=fused_dropout(s["x"], c["p"], rng=s["rng"]))
        elif c["kind"] == "add":
            out = dict(y=fused_dropout_add(s["x"], s["res"], c["p"], rng=s["rng"]))
        else:
            y, h = fused_dropout_add_rms_layernorm(s["x"], s["res"], s["w"], c["p"], eps=EPS,
                                                   rng=s["rng"])
            out = dict(y=y, h=h)
        if not c["train"]:
            return out
        grads = torch.autograd.grad(list(out.values()), [s[k] for k in names],
                                    [s["d" + k] for k in out])
        return dict(**out, **{"d" + k: g for k, g in zip(names, grads)})
    dtype, scale = s["x"].dtype, 65536 / (65536 - round(c["p"] * 65536))
    keep = _dropout_keep(c, s["rng"])
    kept = lambda t: torch.where(keep, t * scale, 0.0)
    h = kept(s["x"].detach().float())
    if c["kind"] == "plain":
        out = dict(y=h.to(dtype))
        if c["train"]:
            out["dx"] = kept(s["dy"].float()).to(dtype)
        return out
    h = h + s["res"].detach().float()
    if c["kind"] == "add":
        out = dict(y=h.to(dtype))
        if c["train"]:
            out.update(dx=kept(s["dy"].float()).to(dtype), dres=s["dy"])
        return out
    w = s["w"].detach().float()
    r = 1 / (h.square().mean(-1, keepdim=True) + EPS).sqrt()
    hat = h * r
    out = dict(y=(hat * w).to(dtype), h=h.to(dtype))
    if c["train"]:
        dy = s["dy"].float()
        e = dy * w
        dh = s["dh"].float() + r * (e - hat * (e * hat).mean(-1, keepdim=True))
        out.update(dx=kept(dh).to(dtype), dres=dh.to(dtype), dw=(dy * hat).sum(0).to(dtype))
    return out


def _dropout_work(c):
    n = c["rows"] * c["cols"]
    # plain: x in, y out, and dy in, dx out; with the residual it too; norm: x, res, dy and dh in,
    # y, h, dx and dres out
    tensors = {"plain": (2, 4), "add": (3, 5), "norm": (4, 8)}[c["kind"]][c["train"]]
    params = c["cols"] * (2 if c["train"] else 1) if c["kind"] == "norm" else 0
    flops = {"plain": (1, 2), "add": (2, 3), "norm": (6, 20)}[c["kind"]][c["train"]]
    return dict(bytes=(tensors * n + params) * _elt(c), flops=flops * n)


def _dropout_exact(c, seed):
    s = _dropout_prepare(c, seed)
    key, offset = s["rng"]

    def mul(m, v):  # high and low words of a 32-bit constant and a word, by halves of the word
        lo, hi = m * (v & 0xFFFF), m * (v >> 16)
        mid = (lo >> 16) + hi
        return mid >> 16, ((mid & 0xFFFF) << 16) | (lo & 0xFFFF)

    groups = -(-c["cols"] // 8)
    index = (torch.arange(c["rows"], device=DEVICE)[:, None] * groups
             + torch.arange(groups, device=DEVICE)[None])
    ctr = [index % (1 << 32), index // (1 << 32), torch.full_like(index, offset % (1 << 32)),
           torch.full_like(index, offset // (1 << 32))]
    for r in range(10):
        k = [(key % (1 << 32) + r * 0x9E3779B9) % (1 << 32),
             (key // (1 << 32) + r * 0xBB67AE85) % (1 << 32)]
        (h0, l0), (h1, l1) = mul(0xD2511F53, ctr[0]), mul(0xCD9E8D57, ctr[2])
        ctr = [h1 ^ ctr[1] ^ k[0], l1, h0 ^ ctr[3] ^ k[1], l0]
    drop = torch.empty(c["rows"], groups, 8, dtype=torch.bool, device=DEVICE)
    limit = int(c["p"] * 65536 + 0.5)
    for j in range(8):
        drop[:, :, j] = (ctr[j // 2] >> (16 * (j % 2))) % 65536 < limit
    drop = drop.view(c["rows"], groups * 8)[:, :c["cols"]]
    leaf = {k: s[k].detach().double().requires_grad_(c["train"])
            for k in ("x", "res", "w") if k in s}
    h = (leaf["x"] / (1 - limit / 65536)).masked_fill(drop, 0.0)
    if "res" in leaf:
        h = leaf["res"] + h
    out = dict(y=h)
    if c["kind"] == "norm":
        out = dict(y=h / torch.sqrt((h * h).mean(-1, keepdim=True) + EPS) * leaf["w"], h=h)
    if not c["train"]:
        return out
    grads = torch.autograd.grad(list(out.values()), list(leaf.values()),
                                [s["d" + k].double() for k in out])
    return dict(**{k: v.detach() for k, v in out.items()},
                **{"d" + k: g for k, g in zip(leaf, grads)})


_HANDLERS = {
    "ffn": (_ffn_prepare, _ffn_run, _ffn_work, _ffn_exact),
    "rope": (_rope_prepare, _rope_run, _rope_work, _rope_exact),
    "dropout": (_dropout_prepare, _dropout_run, _dropout_work, _dropout_exact),
}
