"""Performance cases of the transformer operators: layer norm, layer norm behind a residual sum, and softmax attention.

Every case is one pass of one operator, forward alone (forecasts) or forward and backward (training), in the types that the
token networks run it in: bf16 activations (fp32 for the residual stream under autocast), fp32 parameters.  Sizes are those of
the recipes in `config/`: 90 x 180 tokens of 384 or 768 channels, 103 x 180 tokens of 1024 channels, 8 or 12 heads, the tiny
recipe of 8 x 16 tokens of 32 channels, and packed sequences of different lengths as regional crops have them.

`own` chooses between the plain form (elementary torch operations in 32 bits, rounded once at the end) and the framework's
operators.  `exact` is the definition in 64 bits.
"""

import math
import random

import torch

own = False

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
EPS = 1e-5


# ---------------------------------------------------------------------------------------------------- cases

def listed():
    return [
        # norm of a block of the tiny recipe, two samples of 8 x 16 tokens, forward: latency
        dict(name="norm_tiny_infer", op="norm", rows=256, C=32, x="bf16", y="bf16", train=False),
        # norm of the queries of one sample per head (q_norm / k_norm): many short rows
        dict(name="norm_heads_train", op="norm", rows=16200 * 8, C=48, x="bf16", y="bf16", train=True),
        # the fp32 residual stream of a ViT under autocast, handed on in bf16 to the projection; a ragged number of rows and columns
        dict(name="norm_fp32_train", op="norm", rows=16471, C=387, x="fp32", y="bf16", train=True),
        # norm of the widest recipe, four samples of 103 x 180 tokens: memory rate
        dict(name="norm_wide_train", op="norm", rows=4 * 18540, C=1024, x="bf16", y="bf16", train=True),
        # sum and norm in a forecast step of one sample of 90 x 180 tokens
        dict(name="add_norm_infer", op="add_norm", rows=16200, C=768, x="bf16", y="bf16", train=False),
        # sum and norm in a training step of four samples
        dict(name="add_norm_train", op="add_norm", rows=4 * 16200, C=768, x="bf16", y="bf16", train=True),
        # attention of the tiny recipe: latency
        dict(name="attn_tiny_train", op="attn", B=2, N=128, H=4, Hk=4, D=8, S=0, causal=False, fused=True, train=True),
        # forecast step of the 384-channel recipe: 90 x 180 tokens, 8 heads of 48
        dict(name="attn_vit_infer", op="attn", B=1, N=16200, H=8, Hk=8, D=48, S=0, causal=False, fused=True, train=False),
        # training step of the 768-channel recipe: 12 heads of 64
        dict(name="attn_vit_train", op="attn", B=1, N=16200, H=12, Hk=12, D=64, S=0, causal=False, fused=True, train=True),
        # training step of the 1024-channel recipe: 103 x 180 tokens, 8 heads of 128
        dict(name="attn_big_train", op="attn", B=1, N=18540, H=8, Hk=8, D=128, S=0, causal=False, fused=True, train=True),
        # packed sequences of different lengths (regional crops, histories), causal, four query heads to a key head
        dict(name="attn_packed_causal_train", op="attn", B=1, N=9113, H=16, Hk=4, D=64, S=7, causal=True, fused=False, train=True),
        # many short packed sequences, some of one token or none
        dict(name="attn_packed_infer", op="attn", B=1, N=7001, H=8, Hk=8, D=96, S=41, causal=False, fused=False, train=False),
    ]


def _log(rng, lo, hi, step=1):
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(lo, min(hi, int(round(v / step)) * step))


def draw(rng):
    """One more case of the same ranges: one row to four samples of the widest recipe, odd widths; one token to a whole grid,
    every head width that is a multiple of eight, grouped heads, packed and batched sequences."""
    op = rng.choice(["norm", "norm", "add_norm", "attn", "attn", "attn", "attn"])
    train = rng.random() < 0.6
    if op != "attn":
        x = rng.choice(["bf16", "bf16", "fp32"])
        C = _log(rng, 8, 1024) if rng.random() < 0.3 else _log(rng, 8, 1024, 8)
        rows = _log(rng, 1, min(4 * 18540, 4 * 18540 * 1024 // (C * (2 if x == "fp32" else 1))))
        return dict(op=op, rows=rows, C=C, x=x, y="bf16" if rng.random() < 0.7 else x, train=train)
    D = rng.choice([8, 16, 24, 32, 40, 48, 48, 64, 64, 64, 72, 80, 96, 112, 128, 128])
    Hk = rng.choice([1, 2, 3, 4, 6, 8])
    H = Hk * rng.choice([g for g in (1, 1, 1, 2, 3, 4) if g * Hk <= 12])
    packed = rng.random() < 0.4
    most = int(18540 * math.sqrt(8 * 128 / (H * D)))        # no more products than the largest listed case
    N = _log(rng, 1, min(most, 9113 if packed else 16200))
    B = 1 if packed or N > 4000 else rng.choice([1, 2, 3])
    S = _log(rng, 1, max(1, min(64, N))) if packed else 0
    return dict(op=op, B=B, N=N, H=H, Hk=Hk, D=D, S=S, causal=rng.random() < 0.5, fused=rng.random() < 0.5, train=train)


def _lengths(case):
    """Lengths of the packed sequences: very different ones, some of one token, some of none; they add up to the tokens less a few
    rows behind the last sequence."""
    N, S = case["N"], case["S"]
    rng = random.Random(N * 1000003 + S)
    left = N - N // 100
    if S == 1:
        return [left]
    weight = [rng.random() ** 3 + 0.02 for _ in range(S)]
    lens = [int(left * w / sum(weight)) for w in weight]
    if S > 8:
        for i in rng.sample(range(S), S // 8):
            lens[i] = rng.randint(0, 1)
    big = max(range(S), key=lambda i: lens[i])
    lens[big] += left - sum(lens)
    return lens


def _pairs(case):
    """Products of one query with one key, a head."""
    lens = _lengths(case) if case["S"] else [case["N"]] * case["B"]
    return sum(n * (n + 1) // 2 if case["causal"] else n * n for n in lens)


# ---------------------------------------------------------------------------------------------------- inputs

def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def prepare(case, seed):
    g = _gen(seed)
    train = case["train"]
    if case["op"] != "attn":
        R, C, xt, yt = case["rows"], case["C"], TYPES[case["x"]], TYPES[case["y"]]
        # a residual stream: every channel has a mean and a spread of its own
        loc, spread = torch.randn(C, device=DEV, generator=g), 0.5 + torch.rand(C, device=DEV, generator=g)
        x = (torch.randn(R, C, device=DEV, generator=g) * spread + loc).to(xt)
        st = dict(x=x, weight=1 + 0.2 * torch.randn(C, device=DEV, generator=g), bias=0.2 * torch.randn(C, device=DEV, generator=g), y=yt)
        if case["op"] == "add_norm":
            st["r"] = torch.randn(R, C, device=DEV, generator=g).to(xt)
        if train:
            st["dy"] = torch.randn(R, C, device=DEV, generator=g).to(yt)
            if case["op"] == "add_norm":
                st["ds"] = torch.randn(R, C, device=DEV, generator=g).to(xt)
        leaves = ("x", "weight", "bias") + (("r",) if "r" in st else ())
    else:
        B, N, H, Hk, D = (case[n] for n in ("B", "N", "H", "Hk", "D"))
        st = dict(offsets=None, H=H, Hk=Hk)
        if case["S"]:
            off = [0]
            for n in _lengths(case):
                off.append(off[-1] + n)
            st["offsets"] = torch.tensor(off, dtype=torch.int32, device=DEV)
        lead = (N,) if case["S"] else (B, N)
        if case["fused"]:
            st["qkv"] = torch.randn(*lead, (H + 2 * Hk) * D, device=DEV, generator=g).to(torch.bfloat16)
            leaves = ("qkv",)
        else:
            for n, h in (("q", H), ("k", Hk), ("v", Hk)):
                st[n] = torch.randn(*lead, h, D, device=DEV, generator=g).to(torch.bfloat16)
            leaves = ("q", "k", "v")
        if train:
            st["do"] = torch.randn(*lead, H, D, device=DEV, generator=g).to(torch.bfloat16)
    if train:
        for n in leaves:
            st[n].requires_grad_()
    st["case"] = case
    return st


# ---------------------------------------------------------------------------------------------------- the operators, plain and own

def _plain_norm(st):
    """The formulas; outputs as they are before the rounding at the end."""
    case = st["case"]
    x, w, b = (st[n].detach().float() for n in ("x", "weight", "bias"))
    out = {}
    if "r" in st:
        out["s"] = (x + st["r"].detach().float()).to(st["x"].dtype)
        x = out["s"].float()                     # the sum that the network holds is the one that is normalised
    mean = x.mean(-1, keepdim=True)
    xc = x - mean
    rstd = 1.0 / torch.sqrt((xc * xc).mean(-1, keepdim=True) + EPS)
    xh = xc * rstd
    out["y"] = xh * w + b
    if case["train"]:
        dy = st["dy"].float()
        g = dy * w
        dx = rstd * (g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True))
        if "r" in st:
            dx = dx + st["ds"].float()
            out["dr"] = dx
        out["dx"], out["dweight"], out["dbias"] = dx, (dy * xh).sum(0), dy.sum(0)
    return out


def _norm(st):
    case = st["case"]
    if not own:
        out = _plain_norm(st)
        xt = st["x"].dtype
        types = dict(s=xt, y=st["y"], dx=xt, dr=xt, dweight=torch.float32, dbias=torch.float32)
        return {n: v.to(types[n]) for n, v in out.items()}
    from makani_b200.ops import norm as norm_ops
    if case["op"] == "norm":
        y = norm_ops.layer_norm(st["x"], st["weight"], st["bias"], EPS, out_dtype=st["y"])
        out = dict(y=y)
        if case["train"]:
            out["dx"], out["dweight"], out["dbias"] = torch.autograd.grad(y, (st["x"], st["weight"], st["bias"]), st["dy"])
    else:
        s, y = norm_ops.add_layer_norm(st["x"], st["r"], st["weight"], st["bias"], EPS, out_dtype=st["y"])
        out = dict(s=s, y=y)
        if case["train"]:
            out["dx"], out["dr"], out["dweight"], out["dbias"] = torch.autograd.grad(
                (s, y), (st["x"], st["r"], st["weight"], st["bias"]), (st["ds"], st["dy"]))
    return {n: v.detach() for n, v in out.items()}


def _split(st):
    """q, k, v as [B, N, heads, D]."""
    if "qkv" in st:
        D = st["case"]["D"]
        qkv = st["qkv"].detach().unflatten(-1, (-1, D))
        q, k, v = qkv.split([st["H"], st["Hk"], st["Hk"]], dim=-2)
    else:
        q, k, v = (st[n].detach() for n in ("q", "k", "v"))
    return (t[None] if st["offsets"] is not None else t for t in (q, k, v))


def _seen(st, N):
    """[N, N]: whether a query sees a key; None: all of them.  Second: the queries that belong to a sequence."""
    case = st["case"]
    at = torch.arange(N, device=DEV)
    mask, rows = None, None
    if st["offsets"] is not None:
        seq = torch.searchsorted(st["offsets"][1:].contiguous(), at.int(), right=True)
        rows = seq < case["S"]
        mask = (seq[:, None] == seq[None, :]) & rows[:, None]
    if case["causal"]:
        below = at[:, None] >= at[None, :]
        mask = below if mask is None else mask & below
    return mask, rows


def _attend(q, k, v, do, mask, rows, scale):
    """One or several heads [.., N, D] in the type of q: o and, with `do`, the gradients."""
    p = torch.matmul(q, k.transpose(-1, -2)).mul_(scale)
    if mask is not None:
        p.masked_fill_(~mask, -math.inf)
    if rows is not None:
        p.masked_fill_(~rows[:, None], 0.0)                 # (rows of no sequence: any finite value, they are cleared below)
    p = p.sub_(p.amax(-1, keepdim=True)).exp_()
    p.div_(p.sum(-1, keepdim=True))
    if rows is not None:
        p.masked_fill_(~rows[:, None], 0.0)
    o = torch.matmul(p, v)
    if do is None:
        return o, None, None, None
    dv = torch.matmul(p.transpose(-1, -2), do)
    ds = torch.matmul(do, v.transpose(-1, -2))
    ds = ds.sub_((do * o).sum(-1, keepdim=True)).mul_(p)
    del p
    dq = torch.matmul(ds, k).mul_(scale)
    dk = torch.matmul(ds.transpose(-1, -2), q).mul_(scale)
    return o, dq, dk, dv


def _gathered(st, o, dq, dk, dv):
    """Outputs in the layout of the inputs from [B, heads, N, D] (dk and dv of every query head)."""
    H, Hk = st["H"], st["Hk"]
    lay = (lambda t: t.transpose(1, 2)[0]) if st["offsets"] is not None else (lambda t: t.transpose(1, 2))
    out = dict(o=lay(o))
    if dq is not None:
        dk, dv = (t.unflatten(1, (Hk, H // Hk)).sum(2) for t in (dk, dv))
        dq, dk, dv = lay(dq), lay(dk), lay(dv)
        if "qkv" in st:
            out["dqkv"] = torch.cat([dq, dk, dv], dim=-2).flatten(-2)
        else:
            out.update(dq=dq, dk=dk, dv=dv)
    return out


def _heads(st, t):
    """q, k, v, do as [B, heads, N, D] in the type `t`, keys and values repeated for the heads that share them."""
    G = st["H"] // st["Hk"]
    q, k, v = (x.to(t).transpose(1, 2) for x in _split(st))
    k, v = (x.repeat_interleave(G, 1) if G > 1 else x for x in (k, v))
    do = None
    if st["case"]["train"]:
        do = st["do"].to(t)
        do = (do[None] if st["offsets"] is not None else do).transpose(1, 2)
    return q, k, v, do


def _attention(st):
    case = st["case"]
    if not own:
        q, k, v, do = _heads(st, torch.float32)
        mask, rows = _seen(st, case["N"])
        got = _attend(q, k, v, do, mask, rows, case["D"] ** -0.5)
        return {n: t.to(torch.bfloat16).contiguous() for n, t in _gathered(st, *got).items()}
    from makani_b200.ops import attention as attn_ops
    if "qkv" in st:
        o = attn_ops.attention_qkv(st["qkv"], st["H"], st["Hk"], causal=case["causal"], offsets=st["offsets"])
        out = dict(o=o)
        if case["train"]:
            out["dqkv"] = torch.autograd.grad(o, st["qkv"], st["do"])[0]
    else:
        o = attn_ops.attention(st["q"], st["k"], st["v"], causal=case["causal"], offsets=st["offsets"])
        out = dict(o=o)
        if case["train"]:
            out["dq"], out["dk"], out["dv"] = torch.autograd.grad(o, (st["q"], st["k"], st["v"]), st["do"])
    return {n: t.detach() for n, t in out.items()}


def run(state):
    return _attention(state) if state["case"]["op"] == "attn" else _norm(state)


# ---------------------------------------------------------------------------------------------------- what a pass cannot do without

def work(case):
    """Bytes: every input read once, every output written once.  Flops: the products of attention (two forward; backward the four of its
    formulas, the probabilities taken as known), a few operations per element of the norms."""
    train = case["train"]
    if case["op"] != "attn":
        n, C = case["rows"] * case["C"], case["C"]
        bx, by = (4 if case[t] == "fp32" else 2 for t in ("x", "y"))
        add = case["op"] == "add_norm"
        size = n * (bx + by) + 8 * C + (n * 2 * bx if add else 0)
        if train:       # x (s) is read again, behind the gradient of y that the program between makes
            size += n * (bx + by + bx) + 8 * C + (n * bx if add else 0)
        return {"bytes": size, "flops": n * ((8 if not train else 24) + (1 if add else 0))}
    B, N, H, Hk, D = (case[n] for n in ("B", "N", "H", "Hk", "D"))
    rows, keys = 2 * B * N * H * D, 2 * B * N * Hk * D
    size = 2 * rows + 2 * keys
    if train:
        size += 3 * rows + 4 * keys + rows      # q, o, do, dq; k, v, dk, dv
    return {"bytes": size, "flops": _pairs(case) * H * D * 2 * (6 if train else 2)}


# ---------------------------------------------------------------------------------------------------- definition in 64 bits

def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] != "attn":
        return _exact_norm(st)
    return _exact_attention(st)


def _exact_norm(st):
    case = st["case"]
    x, w, b = (st[n].detach().double() for n in ("x", "weight", "bias"))
    out = {}
    if "r" in st:
        s = x + st["r"].detach().double()
        out["s"] = s
        x = (st["x"].detach().float() + st["r"].detach().float()).to(st["x"].dtype).double()     # the rounded sum is what the norm is given
    x.requires_grad_()
    w.requires_grad_()
    b.requires_grad_()
    var, mean = torch.var_mean(x, dim=-1, correction=0, keepdim=True)
    y = (x - mean) / torch.sqrt(var + EPS) * w + b
    out["y"] = y.detach()
    if case["train"]:
        out["dx"], out["dweight"], out["dbias"] = torch.autograd.grad(y, (x, w, b), st["dy"].double())
        if "r" in st:
            out["dx"] = out["dx"] + st["ds"].double()
            out["dr"] = out["dx"]
    return out


def _exact_attention(st):
    """Sequence by sequence and head by head, gradients by the chain rule of the definition."""
    case = st["case"]
    B, N, H, Hk, D, G = *(case[n] for n in ("B", "N", "H", "Hk", "D")), case["H"] // case["Hk"]
    packed = st["offsets"] is not None
    if "qkv" in st:
        x = st["qkv"].detach().double()
        x = x if not packed else x[None]
        q, k, v = (x[..., a * D:e * D].reshape(B, N, -1, D) for a, e in ((0, H), (H, H + Hk), (H + Hk, H + 2 * Hk)))
    else:
        q, k, v = (st[n].detach().double().reshape(B, N, -1, D) for n in ("q", "k", "v"))
    do = st["do"].double().reshape(B, N, H, D) if case["train"] else None
    o, dq, dk, dv = torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    bounds = []
    if packed:
        at = 0
        for n in _lengths(case):
            bounds.append((at, at + n))
            at += n
    else:
        bounds.append((0, N))
    for bi in range(B):
        for lo, hi in bounds:
            n = hi - lo
            if n == 0:
                continue
            for h in range(H):
                qs, ks, vs = q[bi, lo:hi, h], k[bi, lo:hi, h // G], v[bi, lo:hi, h // G]
                logits = (qs @ ks.mT) / math.sqrt(D)
                if case["causal"]:
                    logits = logits + torch.full((n, n), -math.inf, dtype=torch.float64, device=DEV).triu(1)
                prob = torch.exp(logits - torch.logsumexp(logits, -1, keepdim=True))
                del logits
                o[bi, lo:hi, h] = prob @ vs
                if do is None:
                    continue
                gs = do[bi, lo:hi, h]
                dv[bi, lo:hi, h // G] += prob.mT @ gs
                dprob = gs @ vs.mT
                dlogit = prob * (dprob - (prob * dprob).sum(-1, keepdim=True))
                del dprob, prob
                dq[bi, lo:hi, h] = dlogit @ ks / math.sqrt(D)
                dk[bi, lo:hi, h // G] += dlogit.mT @ qs / math.sqrt(D)
    lay = (lambda t: t[0]) if packed else (lambda t: t)
    out = dict(o=lay(o))
    if do is not None:
        if "qkv" in st:
            out["dqkv"] = lay(torch.cat([dq.flatten(2), dk.flatten(2), dv.flatten(2)], -1))
        else:
            out.update(dq=lay(dq), dk=lay(dk), dv=lay(dv))
    return out
