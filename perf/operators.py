"""Performance cases of the operators around a policy-gradient training step's model.

Four operators, each in its plain form (``own`` false: elementary torch operations in 32 bits, 64
where 32 lose what matters, rounded once) and through the package's public entry points (``own``
true): the scaled embedding with its gradient, the norms before and after a block fused with the
block's gate and residual, the clipped policy loss with its KL term, and the global gradient norm
with clipping. A case is a plain dict; ``op`` selects one of the handlers at the end of the file.
``draw`` spreads over the ranges between the listed cases.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DEVICE = "cuda:0"
EPS = 1e-6
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # one decoding step of 16 sequences: the lookup alone, launch and host time
        dict(name="embed_decode", op="embed", tokens=16, vocab=128256, hidden=4096, dtype="bf16",
             scale=64.0, padded=0.0, train=False),
        # the embedding of an 8B model in training, 8 sequences of 2048 tokens: the dense gradient
        dict(name="embed_train_8b", op="embed", tokens=16384, vocab=128256, hidden=4096,
             dtype="bf16", scale=64.0, padded=0.0, train=True),
        # a 768-wide model over GPT-2's vocabulary in fp32, a ragged batch half of padding
        dict(name="embed_train_padded", op="embed", tokens=8191, vocab=50257, hidden=768,
             dtype="fp32", scale=1.0, padded=0.5, train=True),
        # the boundary between two blocks for one decoding step of 16 sequences
        dict(name="sandwich_decode", op="sandwich", batch=16, seq=1, hidden=4096, dtype="bf16",
             gate="none", residual_scale=1.0, offset=1.0, train=False),
        # the same boundary in training, an 8B-class width
        dict(name="sandwich_train_8b", op="sandwich", batch=4, seq=2048, hidden=4096,
             dtype="bf16", gate="none", residual_scale=1.0, offset=1.0, train=True),
        # a gate for each sequence (conditioned blocks), a 70B-class width and a ragged length
        dict(name="sandwich_gated_70b", op="sandwich", batch=3, seq=1365, hidden=8192,
             dtype="bf16", gate="batch", residual_scale=0.5, offset=0.0, train=True),
        # group-relative policy update of 4 completions of 500 tokens
        dict(name="policy_group_small", op="policy", batch=4, seq=500, dtype="fp32",
             advantages="sequence", ref=True, kl_coef=0.04, reduction="token"),
        # an actor update with an advantage for each token, 16-bit log-probs, an odd length
        dict(name="policy_actor_bf16", op="policy", batch=64, seq=2047, dtype="bf16",
             advantages="token", ref=False, kl_coef=0.0, reduction="sequence"),
        # a large rollout batch of long completions
        dict(name="policy_group_large", op="policy", batch=512, seq=8192, dtype="fp32",
             advantages="sequence", ref=True, kl_coef=0.04, reduction="sequence"),
        # adapters of 32 projections, below the limit: nothing is scaled; host and launch time
        dict(name="clip_adapters", op="clip", tensors="adapters", dtype="bf16", inplace=True,
             max_norm=1e4),
        # a 768-wide model's fp32 gradients clipped into the optimizer's buffers
        dict(name="clip_768_fp32", op="clip", tensors="gpt", dtype="fp32", inplace=False,
             max_norm=1.0),
        # one pipeline stage of an 8B model: bf16 gradients clipped into fp32 main gradients
        dict(name="clip_stage_8b", op="clip", tensors="stage", dtype="bf16", inplace=False,
             max_norm=1.0),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["embed", "sandwich", "policy", "clip"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op == "embed":
        hidden = _log_int(rng, 64, 4096)
        if rng.random() < 0.7:
            hidden = max(64, hidden // 64 * 64)
        most = (1 << 30) // (hidden * (4 if dtype == "fp32" else 2))
        return dict(op=op, tokens=_log_int(rng, 1, 16384), hidden=hidden, dtype=dtype,
                    vocab=_log_int(rng, 1000, min(128256, most)),
                    scale=rng.choice([1.0, round(math.sqrt(hidden), 3)]),
                    padded=rng.choice([0.0, 0.0, 0.3, 0.9]), train=rng.random() < 0.8)
    if op == "sandwich":
        hidden = _log_int(rng, 256, 8192)
        if rng.random() < 0.7:
            hidden = hidden // 64 * 64
        batch, most = rng.choice([1, 2, 3, 8, 16]), (1 << 24) // hidden * 2
        return dict(op=op, batch=batch, seq=_log_int(rng, 1, max(2, most // batch // 2)),
                    hidden=hidden, dtype=dtype, gate=rng.choice(["none", "channel", "batch"]),
                    residual_scale=rng.choice([1.0, 1.0, 0.5]), offset=rng.choice([0.0, 1.0]),
                    train=rng.random() < 0.8)
    if op == "policy":
        ref = rng.random() < 0.6
        return dict(op=op, batch=_log_int(rng, 1, 512), seq=_log_int(rng, 1, 8192), dtype=dtype,
                    advantages=rng.choice(["sequence", "token"]), ref=ref,
                    kl_coef=rng.choice([0.0, 0.04]) if ref else 0.0,
                    reduction=rng.choice(["token", "sequence", "sum"]))
    inplace = rng.random() < 0.4  # below the limit, so that a pass leaves the gradients as they are
    return dict(op=op, tensors="drawn", count=_log_int(rng, 1, 200),
                largest=_log_int(rng, 64, 4 << 20), sizes=rng.randrange(1 << 30),
                dtype=rng.choice([dtype, dtype, "mixed"]), inplace=inplace,
                max_norm=1e4 if inplace else rng.choice([1.0, 1e4]))


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

    def rand(self, *shape):
        return torch.rand(shape, generator=self.g, device=DEVICE, dtype=torch.float64)


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
# Embedding: out[n] = scale weight[id[n]]; grad[v] = scale sum over id[n] = v of dout[n], the
# padding token's row zero
# ---------------------------------------------------------------------------

def _embed_prepare(c, seed):
    i = _Inputs(seed, c["dtype"])
    n, v = c["tokens"], c["vocab"]
    # token frequencies fall off as 1 / rank; ranks are spread over the vocabulary
    rank = (float(v) ** i.rand(n)).long().clamp_(1, v) - 1
    ids = (rank * 48271 + 11) % v
    pad = None
    if c["padded"] > 0:
        pad = v - 1
        ids[i.rand(n) < c["padded"]] = pad
    weight = i.randn(v, c["hidden"], std=0.02)
    s = dict(c=c, ids=ids, weight=weight, pad=pad)
    if c["train"]:
        s.update(weight=weight.requires_grad_(), dout=i.randn(n, c["hidden"]))
    return s


def _embed_run(s):
    c, ids, w = s["c"], s["ids"], s["weight"]
    if own:
        from trainscale_amd.kernels import scaled_embedding
        out = scaled_embedding(ids, w, scale=c["scale"], padding_idx=s["pad"])
        if not c["train"]:
            return out
        (grad,) = torch.autograd.grad(out, w, s["dout"])
        return dict(out=out, grad=grad)
    w = w.detach()
    out = (w[ids].float() * c["scale"]).to(w.dtype)
    if not c["train"]:
        return out
    grad = torch.zeros(w.shape, dtype=torch.float32, device=w.device)
    grad.index_add_(0, ids, s["dout"].float())
    if s["pad"] is not None:
        grad[s["pad"]] = 0
    return dict(out=out, grad=grad.mul_(c["scale"]).to(w.dtype))


def _embed_work(c):
    n, v, row = c["tokens"], c["vocab"], c["hidden"] * _elt(c)
    moved = 8 * n + min(n, v) * row + n * row
    if c["train"]:
        moved += n * row + v * row
    return dict(bytes=moved, flops=(2 if c["train"] else 1) * n * c["hidden"])


def _embed_exact(c, seed):
    s = _embed_prepare(c, seed)
    w, ids = s["weight"].detach(), s["ids"]
    out = w.index_select(0, ids).double() * c["scale"]
    if not c["train"]:
        return out
    # tokens in the vocabulary's order: each row's sum from running sums over column blocks
    order = torch.argsort(ids, stable=True)
    last = torch.searchsorted(ids[order], torch.arange(c["vocab"], device=DEVICE), right=True)
    grad = torch.empty(w.shape, dtype=torch.float64, device=DEVICE)
    for a in range(0, c["hidden"], 512):
        run_sum = s["dout"][order, a:a + 512].double().cumsum(0)
        run_sum = torch.cat([torch.zeros_like(run_sum[:1]), run_sum])
        upto = run_sum[last]
        grad[:, a:a + 512] = upto
        grad[1:, a:a + 512] -= upto[:-1]
    # rows without a token: exactly zero
    none = torch.ones(c["vocab"], dtype=torch.bool, device=DEVICE)
    none[ids] = False
    if s["pad"] is not None:
        none[s["pad"]] = True
    grad[none] = 0
    return dict(out=out, grad=grad.mul_(c["scale"]))


# ---------------------------------------------------------------------------
# Norms before and after a block: h = residual_scale x + gate * norm(y) (offset + post),
# n = norm(h) (offset + pre), y the block's output and x the residual stream
# ---------------------------------------------------------------------------

def _sandwich_prepare(c, seed):
    i = _Inputs(seed, c["dtype"])
    b, t, h = c["batch"], c["seq"], c["hidden"]
    mean = 1.0 - c["offset"]
    s = dict(c=c, y=i.randn(b, t, h, std=0.7), x=i.randn(b, t, h, std=2.0),
             post=i.randn(h, std=0.1, mean=mean), pre=i.randn(h, std=0.1, mean=mean), gate=None)
    if c["gate"] == "channel":
        s["gate"] = i.randn(h, std=0.2, mean=0.3)
    elif c["gate"] == "batch":
        s["gate"] = i.randn(b, 1, h, std=0.2, mean=0.3)
    if c["train"]:
        for k in ("y", "x", "post", "pre", "gate"):
            if s[k] is not None:
                s[k].requires_grad_()
        s.update(dn=i.randn(b, t, h), dh=i.randn(b, t, h))
    return s


def _sandwich_run(s):
    c = s["c"]
    if own:
        from trainscale_amd.kernels import fused_sandwich_rms_layernorm
        n, h = fused_sandwich_rms_layernorm(s["y"], s["x"], s["post"], s["pre"], gate=s["gate"],
                                            eps=EPS, residual_scale=c["residual_scale"],
                                            weight_offset=c["offset"])
        if not c["train"]:
            return dict(n=n, h=h)
        names = [k for k in ("y", "x", "post", "pre", "gate") if s[k] is not None]
        grads = torch.autograd.grad((n, h), [s[k] for k in names], (s["dn"], s["dh"]))
        return dict(n=n, h=h, **{"d" + k: g for k, g in zip(names, grads)})
    dtype = s["y"].dtype
    y, x = s["y"].detach().float(), s["x"].detach().float()
    post, pre = s["post"].detach().float() + c["offset"], s["pre"].detach().float() + c["offset"]
    ry = 1 / (y.square().mean(-1, keepdim=True) + EPS).sqrt()
    yhat = y * ry
    branch = yhat * post
    gate = None
    if s["gate"] is not None:
        gate = s["gate"].detach().float()
        branch = branch * gate
    h = x * c["residual_scale"] + branch
    rh = 1 / (h.square().mean(-1, keepdim=True) + EPS).sqrt()
    hhat = h * rh
    out = dict(n=(hhat * pre).to(dtype), h=h.to(dtype))
    if not c["train"]:
        return out
    dn, dh = s["dn"].float(), s["dh"].float()
    e = dn * pre
    dt = dh + rh * (e - hhat * (e * hhat).mean(-1, keepdim=True))
    p = dt * yhat
    dg = dt * gate if gate is not None else dt
    q = dg * post
    out["dy"] = (ry * (q - yhat * (q * yhat).mean(-1, keepdim=True))).to(dtype)
    out["dx"] = (dt * c["residual_scale"]).to(dtype)
    out["dpost"] = (p * gate if gate is not None else p).sum((0, 1)).to(dtype)
    out["dpre"] = (dn * hhat).sum((0, 1)).to(dtype)
    if gate is not None:
        dgate = p.sum(1, keepdim=True) * post
        out["dgate"] = (dgate if c["gate"] == "batch" else dgate.sum((0, 1))).to(dtype)
    return out


def _sandwich_work(c):
    n = c["batch"] * c["seq"] * c["hidden"]
    gates = {"none": 0, "channel": 1, "batch": c["batch"]}[c["gate"]]
    params = (2 + gates) * c["hidden"] * (2 if c["train"] else 1)
    # x and y in, n and h out; in training dn and dh in, dx and dy out as well
    return dict(bytes=((8 if c["train"] else 4) * n + params) * _elt(c),
                flops=(45 if c["train"] else 12) * n)


def _sandwich_exact(c, seed):
    s = _sandwich_prepare(c, seed)
    leaf = {k: s[k].detach().double().requires_grad_(c["train"])
            for k in ("y", "x", "post", "pre", "gate") if s[k] is not None}

    def norm(t, w):
        return t / torch.sqrt((t * t).mean(-1, keepdim=True) + EPS) * (w + c["offset"])

    branch = norm(leaf["y"], leaf["post"])
    if "gate" in leaf:
        branch = leaf["gate"] * branch
    h = c["residual_scale"] * leaf["x"] + branch
    n = norm(h, leaf["pre"])
    if not c["train"]:
        return dict(n=n, h=h)
    grads = torch.autograd.grad((n, h), list(leaf.values()), (s["dn"].double(), s["dh"].double()))
    return dict(n=n.detach(), h=h.detach(), **{"d" + k: g for k, g in zip(leaf, grads)})


# ---------------------------------------------------------------------------
# Clipped policy loss: per token -min(r A, clip(r, 1 - low, 1 + high) A) + kl_coef k,
# r = exp(logp - old), k = exp(ref - logp) - (ref - logp) - 1, averaged over the valid tokens
# ("token"), over each sequence's and then the sequences ("sequence"), or summed ("sum")
# ---------------------------------------------------------------------------

CLIP_LOW, CLIP_HIGH = 0.2, 0.28


def _policy_prepare(c, seed):
    i = _Inputs(seed, c["dtype"])
    b, t = c["batch"], c["seq"]
    wide = _Inputs(seed + 1, "fp32")
    logp = -wide.randn(b, t).abs() - 0.02
    s = dict(c=c, logps=logp.to(i.dtype).requires_grad_(),
             old=(logp + 0.15 * wide.randn(b, t)).to(i.dtype),
             ref=(logp + 0.3 * wide.randn(b, t)).to(i.dtype) if c["ref"] else None,
             adv=wide.randn(b) if c["advantages"] == "sequence" else wide.randn(b, t))
    # completions end early; of many sequences one has no token at all
    length = (t * (0.25 + 0.75 * wide.rand(b))).ceil().long()
    if b >= 8:
        length[b // 2] = 0
    s["mask"] = torch.arange(t, device=DEVICE)[None, :] < length[:, None]
    return s


def _policy_run(s):
    c = s["c"]
    if own:
        from trainscale_amd.loss import clipped_policy_loss
        r = clipped_policy_loss(s["logps"], s["old"], s["adv"], mask=s["mask"], ref_logps=s["ref"],
                                clip_low=CLIP_LOW, clip_high=CLIP_HIGH, kl_coef=c["kl_coef"],
                                reduction=c["reduction"])
        (grad,) = torch.autograd.grad(r.loss, s["logps"])
        return dict(loss=r.loss, policy=r.policy_loss, kl=r.kl, clipped=r.clip_fraction, grad=grad)
    lp, mask = s["logps"].detach(), s["mask"]
    adv = s["adv"].float()
    adv = adv[:, None] if adv.dim() == 1 else adv
    # the log ratio in 64 bits: whether a token is clipped is decided next to the border
    d = lp.double() - s["old"].double()
    over = ((adv > 0) & (d > math.log1p(CLIP_HIGH))) | ((adv < 0) & (d < math.log1p(-CLIP_LOW)))
    ratio = d.float().exp()
    bound = torch.where(adv > 0, 1 + CLIP_HIGH, 1 - CLIP_LOW)
    pol = -torch.where(over, bound, ratio) * adv
    grad = torch.where(over, 0.0, -ratio * adv)
    kl = torch.zeros_like(ratio)
    if s["ref"] is not None:
        x = s["ref"].double() - lp.double()
        rise = x.expm1()
        kl = (rise - x).float()
        grad = grad - c["kl_coef"] * rise.float()
    count = mask.sum(1)
    if c["reduction"] == "token":
        weight = (1.0 / count.sum().clamp(min=1).double()).expand(lp.shape[0])
    elif c["reduction"] == "sequence":
        weight = 1.0 / (count.clamp(min=1) * (count > 0).sum().clamp(min=1)).double()
    else:
        weight = torch.ones(lp.shape[0], dtype=torch.float64, device=lp.device)
    total = [(torch.where(mask, v, 0.0).sum(1, dtype=torch.float64) * weight).sum()
             for v in (pol, kl, over.float())]
    grad = torch.where(mask, grad, 0.0) * weight.float()[:, None]
    return dict(loss=(total[0] + c["kl_coef"] * total[1]).float(), policy=total[0].float(),
                kl=total[1].float(), clipped=total[2].float(), grad=grad.to(lp.dtype))


def _policy_work(c):
    n = c["batch"] * c["seq"]
    read = (3 if c["ref"] else 2) * n * _elt(c) + n
    read += 4 * (n if c["advantages"] == "token" else c["batch"])
    return dict(bytes=read + n * _elt(c), flops=30 * n)


def _policy_exact(c, seed):
    s = _policy_prepare(c, seed)
    keep = s["mask"]
    lp = s["logps"].detach().double().requires_grad_()
    adv = s["adv"].double()
    adv = adv[:, None].expand_as(lp) if adv.dim() == 1 else adv
    r = torch.exp(lp - s["old"].double())
    free, held = r * adv, r.clamp(1 - CLIP_LOW, 1 + CLIP_HIGH) * adv
    pol = -torch.minimum(free, held)
    k = torch.zeros_like(lp)
    if s["ref"] is not None:
        x = s["ref"].double() - lp
        k = torch.special.expm1(x) - x

    def reduced(v):
        rows = torch.where(keep, v, torch.zeros_like(v)).sum(1)
        lens = keep.sum(1).double()
        if c["reduction"] == "sum":
            return rows.sum()
        if c["reduction"] == "token":
            return rows.sum() / max(1.0, float(lens.sum()))
        some = lens > 0
        return (rows[some] / lens[some]).sum() / max(1, int(some.sum()))

    policy, kl = reduced(pol), reduced(k)
    loss = policy + c["kl_coef"] * kl
    (grad,) = torch.autograd.grad(loss, lp)
    return dict(loss=loss.detach(), policy=policy.detach(), kl=kl.detach(),
                clipped=reduced((held < free).double()), grad=grad)


# ---------------------------------------------------------------------------
# Gradient norm over many tensors and clipping: g min(1, max_norm / (norm + 1e-6)), in place or
# into fp32 buffers. The gradients are views into one flat buffer for each type, as gradient
# buckets are; the buffers are what a pass returns
# ---------------------------------------------------------------------------

def _clip_sizes(c):
    if c["tensors"] == "adapters":  # rank 16 on 32 projections of a 4096-wide model
        return [16 * 4096] * 64
    if c["tensors"] == "gpt":  # 12 layers of a 768-wide model without biases, and its embedding
        sq = 768 * 768
        return [50257 * 768] + [768, 3 * sq, sq, 768, 4 * sq, 4 * sq] * 12 + [768]
    if c["tensors"] == "stage":  # embedding and 4 layers of an 8B model
        h, kv, f = 4096, 1024, 14336
        return [128256 * h] + [h, h * h, h * kv, h * kv, h * h, h, h * f, h * f, h * f] * 4
    r = np.random.RandomState(c["sizes"] % (1 << 31))
    return [int(math.exp(u * math.log(c["largest"]))) for u in r.rand(c["count"])]


def _clip_types(c, sizes):
    if c["dtype"] == "mixed":
        return [("bf16", "fp32")[k % 2] for k in range(len(sizes))]
    return [c["dtype"]] * len(sizes)


def _clip_prepare(c, seed):
    i = _Inputs(seed, c["dtype"])
    sizes = _clip_sizes(c)
    types = _clip_types(c, sizes)
    flat, views, at = {}, [], {}
    for t in sorted(set(types)):
        n = sum(z for z, u in zip(sizes, types) if u == t)
        flat[t], at[t] = torch.empty(n, dtype=DTYPES[t], device=DEVICE), 0
    for k, (z, t) in enumerate(zip(sizes, types)):
        g = flat[t][at[t]:at[t] + z]
        at[t] += z
        for a in range(0, z, 1 << 27):
            part = g[a:a + (1 << 27)]
            part.copy_(torch.randn(part.shape, generator=i.g, device=DEVICE))
        g.mul_((1e-2, 1e-3, 3e-4, 1e-4)[k % 4])
        if k == 0 and z > 1 << 20:  # an embedding's gradient: most rows have no token
            g.view(-1, z // 1024)[:900].zero_() if z % 1024 == 0 else g[:z // 8 * 7].zero_()
        views.append(g)
    s = dict(c=c, flat=flat, grads=views, max_norm=c["max_norm"])
    if c["inplace"]:
        s["params"] = [torch.nn.Parameter(torch.empty_like(g)) for g in views]
        for p, g in zip(s["params"], views):
            p.grad = g
    else:
        s["flat_out"] = torch.empty(sum(sizes), dtype=torch.float32, device=DEVICE)
        s["out"] = list(s["flat_out"].split(sizes))
    return s


def _clip_run(s):
    if own:
        from trainscale_amd.kernels import clip_grad_norm_, clipped_grads
        if s["c"]["inplace"]:
            return dict(norm=clip_grad_norm_(s["params"], s["max_norm"]), grads=s["flat"])
        norm = clipped_grads(s["grads"], s["max_norm"], out=s["out"])
        return dict(norm=norm, grads=s["flat_out"])
    total = torch.stack([g.float().square().sum() for g in s["grads"]]).sum().sqrt()
    coef = (s["max_norm"] / (total + 1e-6)).clamp(max=1.0)
    if s["c"]["inplace"]:
        _ = [g.mul_(coef) for g in s["grads"]]
        return dict(norm=total, grads=s["flat"])
    _ = [torch.mul(g, coef, out=o) if g.dtype == o.dtype else o.copy_(g).mul_(coef)
         for g, o in zip(s["grads"], s["out"])]
    return dict(norm=total, grads=s["flat_out"])


def _clip_work(c):
    sizes = _clip_sizes(c)
    types = _clip_types(c, sizes)
    read = sum(z * (4 if t == "fp32" else 2) for z, t in zip(sizes, types))
    # in place the gradients, below the limit, stay as they are
    write = 0 if c["inplace"] else 4 * sum(sizes)
    return dict(bytes=read + write, flops=3 * sum(sizes))


def _clip_exact(c, seed):
    s = _clip_prepare(c, seed)
    sq = sum(float(torch.linalg.vector_norm(g, dtype=torch.float64)) ** 2 for g in s["grads"])
    norm = math.sqrt(sq)
    coef = min(1.0, c["max_norm"] / (norm + 1e-6))
    if c["inplace"]:
        return dict(norm=norm, grads={t: f.double().mul_(coef) for t, f in s["flat"].items()})
    return dict(norm=norm, grads=torch.cat([g.double() for g in s["grads"]]).mul_(coef))


_HANDLERS = {
    "embed": (_embed_prepare, _embed_run, _embed_work, _embed_exact),
    "sandwich": (_sandwich_prepare, _sandwich_run, _sandwich_work, _sandwich_exact),
    "policy": (_policy_prepare, _policy_run, _policy_work, _policy_exact),
    "clip": (_clip_prepare, _clip_run, _clip_work, _clip_exact),
}
