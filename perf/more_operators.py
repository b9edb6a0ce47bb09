"""Performance cases of what a transformer block on a grid of tokens does around its products: rotary positions with several axes, norms of
queries and keys with the rotation in the same pass, attention with a sliding window and first tokens that stay visible, and dropout whose mask
is made from a counter and never stored.

Every case is one pass, forward alone (forecasts) or forward and backward (training), in the types that the token networks run in: bf16
activations (fp32 for a residual stream under autocast), fp32 parameters.  Sizes are those of the recipes in `config/`: 90 x 180 tokens of
384 or 768 channels, 103 x 180 tokens of 1024 channels, 8 or 12 heads, the tiny recipe of 8 x 16 tokens of 32 channels, and packed sequences of
different lengths as regional crops and histories have them.  A window is some rows of latitude to either side.

`own` chooses between the plain form (elementary torch operations in 32 bits, angles in 64, rounded once at the end) and the framework's
operators.  `exact` is the definition in 64 bits.
"""

import math
import random

import numpy as np
import torch

own = False

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
EPS = 1e-5


# ---------------------------------------------------------------------------------------------------- cases

def listed():
    return [
        # queries and keys of the tiny recipe turned by latitude and longitude, in a forecast: latency
        _rotary("rot_tiny_infer", B=2, N=128, H=4, Hk=4, D=8, bands=(4, 4)),
        # the 768-channel recipe in training: 90 x 180 tokens, 12 heads of 64, halves of a band turned against one another
        _rotary("rot_vit_train", N=16200, H=12, Hk=12, D=64, bands=(32, 32), train=True),
        # time (hours, fractions of them, far from the origin), height and width; grouped heads, a part of the channels left as it is
        _rotary("rot_time_train", N=9113, H=16, Hk=4, D=96, bands=(16, 40, 32), inter=True, pos="float", train=True),
        # one new token of each of some series in a forecast, root-mean-square norms: latency
        _normed("qkn_single_infer", B=37, N=1, H=16, Hk=4, D=128, bands=(128,), norm="rms", pos="float"),
        # the 384-channel recipe with layer norms of queries and keys, in training: 8 heads of 48
        _normed("qkn_vit_train", N=16200, H=8, Hk=8, D=48, bands=(24, 24), norm="layer", train=True),
        # the widest recipe: two samples of 103 x 180 tokens, 8 heads of 128
        _normed("qkn_big_train", B=2, N=18540, H=8, Hk=8, D=128, bands=(32, 48, 48), norm="rms", train=True),
        # windowed attention of the tiny recipe: two rows to either side, one register token
        _window("win_tiny_train", B=2, N=129, H=4, Hk=4, D=8, left=32, right=32, sinks=1, train=True),
        # forecast step of the 384-channel recipe: four rows of latitude to either side, four register tokens
        _window("win_vit_infer", N=16204, H=8, Hk=8, D=48, left=720, right=720, sinks=4),
        # packed histories, causal, the last 512 tokens and the first of each, four query heads to a key head
        _window("win_packed_train", N=9113, H=16, Hk=4, D=64, S=7, causal=True, left=512, right=0, sinks=4, train=True),
        # a training step of the 768-channel recipe from its fused projection: rotation and windowed attention in one call
        _window("win_path_train", N=16204, H=12, Hk=12, D=64, left=720, right=720, sinks=4, path=True, bands=(32, 32), train=True),
        # dropout behind a projection of 16200 x 768, a ragged number of elements
        _drop("drop_ragged_train", n=16200 * 768 - 3, p=0.1, train=True),
        # dropout and residual sum of a training step of four samples, the residual stream in fp32
        _drop("drop_add_train", n=4 * 16200 * 768, p=0.1, residual="fp32", train=True),
    ]


def _case(name, op, train, **kw):
    case = dict(op=op, train=train, **kw)
    return case if name is None else dict(name=name, **case)


def _rotary(name, B=1, N=1, H=1, Hk=1, D=8, bands=(8,), inter=False, pos="int", train=False):
    return _case(name, "rotary", train, B=B, N=N, H=H, Hk=Hk, D=D, bands=",".join(map(str, bands)), inter=inter, pos=pos, S=0)


def _normed(name, norm="layer", **kw):
    return dict(_rotary(name, **kw), op="normed", norm=norm)


def _window(name, B=1, N=1, H=1, Hk=1, D=8, S=0, causal=False, left=0, right=0, sinks=0, path=False, bands=(), train=False):
    return _case(name, "window", train, B=B, N=N, H=H, Hk=Hk, D=D, S=S, causal=causal, left=left, right=right, sinks=sinks, path=path,
                 bands=",".join(map(str, bands)), inter=False, pos="int")


def _drop(name, n, p, x="bf16", residual="", train=False):
    return _case(name, "dropout", train, n=n, p=p, x=x, residual=residual)


def _log(rng, lo, hi, step=1):
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(lo, min(hi, int(round(v / step)) * step))


def _bands(rng, D):
    """One to three bands of even widths; sometimes they leave channels out."""
    axes = rng.choice([1, 2, 2, 3]) if D >= 16 else rng.choice([1, 2])
    unit = rng.choice([u for u in (2, 8, 16, 16) if u * axes <= D])
    left, bands = D // unit, []
    for a in range(axes):
        most = left - (axes - 1 - a)
        take = most if a == axes - 1 and rng.random() < 0.7 else rng.randint(1, max(1, min(most, D // unit // axes + 1)))
        bands.append(take * unit)
        left -= take
    return tuple(bands)


def draw(rng):
    """One more case of the same ranges: one token to a whole grid, every head width that is a multiple of eight, one to three axes, grouped heads,
    packed and batched sequences, windows of one token to most of a grid, a handful of elements to four samples."""
    op = rng.choice(["rotary", "normed", "normed", "window", "window", "window", "dropout"])
    train = rng.random() < 0.6
    if op == "dropout":
        residual = rng.choice(["", "bf16", "fp32"])
        x = "fp32" if residual == "fp32" and rng.random() < 0.3 else rng.choice(["bf16", "bf16", "fp32"]) if not residual else "bf16"
        return _drop(None, _log(rng, 1, 4 * 16200 * 768 // (2 if x == "fp32" else 1)), rng.choice([0.1, 0.1, 0.05, 0.25, 0.5, 0.9]), x, residual, train)
    D = rng.choice([8, 16, 24, 32, 40, 48, 48, 64, 64, 64, 72, 80, 96, 112, 128, 128])
    Hk = rng.choice([1, 2, 3, 4, 6, 8])
    H = Hk * rng.choice([g for g in (1, 1, 1, 2, 3, 4) if g * Hk <= 12])
    bands = _bands(rng, D)
    if op != "window":
        N = _log(rng, 1, min(18540, 2 * 18540 * 16 * 128 // ((H + Hk) * D)))
        B = rng.choice([1, 1, 2]) if N < 9000 else 1
        kw = dict(B=B, N=N, H=H, Hk=Hk, D=D, bands=bands, inter=rng.random() < 0.4, pos=rng.choice(["int", "int", "float"]), train=train)
        if op == "rotary":
            return _rotary(None, **kw)
        return _normed(None, norm=rng.choice(["layer", "rms"]), **kw)
    packed = rng.random() < 0.4
    most = int(16204 * math.sqrt(12 * 64 / (H * D)))         # no more products than the largest listed case
    # (gradients of queries and keys of a token by itself are zero but for rounding: in training there are several to a sequence)
    N = _log(rng, 2 if train else 1, min(most, 9113 if packed else 16204))
    B = 1 if packed or N > 4000 else rng.choice([1, 2, 3])
    S = _log(rng, 1, max(1, min(64, N // 8 if train else N))) if packed else 0
    causal = rng.random() < 0.5
    # (a window's work is its width: wide ones go with fewer tokens)
    wide = max(1, min(N, 12 * 64 * 16204 * 1440 // (2 * N * H * D)))
    left = _log(rng, 1, wide)
    right = 0 if causal else rng.choice([left, left, 0, _log(rng, 1, wide)])
    path = not packed and rng.random() < 0.3
    return _window(None, B, N, H, Hk, D, S, causal, left, right, rng.choice([0, 1, 4, 4, 16, 130]), path, bands if path else (),
                   train)


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


def _visible(case, n):
    """Pairs of a query and a key that it sees, of a sequence of n tokens."""
    i = np.arange(n, dtype=np.int64)
    first = np.maximum(i - case["left"], 0)
    last = i if case["causal"] else np.minimum(i + case["right"], n - 1)
    seen = last - first + 1
    sinks = np.minimum(case["sinks"], i + 1 if case["causal"] else n)
    return int((seen + sinks - np.maximum(0, np.minimum(last + 1, sinks) - first)).sum())      # (less the sinks that the window holds)


def _sizes(case):
    return [int(b) for b in case["bands"].split(",")] if case["bands"] else []


# ---------------------------------------------------------------------------------------------------- inputs

def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _positions(case, g):
    """[N, axes]: time, row and column of every token; whole numbers, or times in hours and coordinates in degrees, far from the origin."""
    N, axes = case["N"], len(_sizes(case))
    at = torch.arange(N, device=DEV)
    cols = torch.stack([at // 8100, (at // 180) % 103, at % 180][3 - axes:] if axes > 1 else [at + 100000], -1)
    if case["pos"] == "int":
        return cols.int()
    far = torch.tensor([70000.0, 17.5, -33.25][:axes], device=DEV)
    return (cols * 0.25 + far + 0.1 * torch.rand(N, axes, device=DEV, generator=g)).float()


def prepare(case, seed):
    g = _gen(seed)
    r = lambda *s: torch.randn(*s, device=DEV, generator=g)  # noqa: E731
    train, op = case["train"], case["op"]
    st = dict(case=case)
    if op == "dropout":
        n, xt = case["n"], TYPES[case["x"]]
        st["x"] = r(n).to(xt)
        leaves = ["x"]
        if case["residual"]:
            st["residual"] = r(n).to(TYPES[case["residual"]])
            leaves.append("residual")
        # the seed, and the number of the call
        st["seed"] = torch.tensor([(int(seed) * 7919 + 12345) % 2**63, int(seed) % 2**31 + 3], dtype=torch.int64, device=DEV)
        if train:
            st["dy"] = r(n).to(_sum_type(case))
    else:
        B, N, H, Hk, D = (case[n] for n in ("B", "N", "H", "Hk", "D"))
        lead = (N,) if case["S"] else (B, N)
        fused = op != "window" or case["path"]
        if fused:           # the output of a projection: a mean and a spread of its own for every channel
            loc, spread = 0.3 * r((H + 2 * Hk) * D), 0.5 + torch.rand((H + 2 * Hk) * D, device=DEV, generator=g)
            st["qkv"] = (r(*lead, (H + 2 * Hk) * D) * spread + loc).to(torch.bfloat16)
            leaves = ["qkv"]
            if op != "window":          # queries and keys as they lie in it
                st["q"], st["k"], _ = _split(st)
                leaves = ["q", "k"]
        else:
            for n, h in (("q", H), ("k", Hk), ("v", Hk)):
                st[n] = r(*lead, h, D).to(torch.bfloat16)
            leaves = ["q", "k", "v"]
        if case["bands"]:
            st["positions"] = _positions(case, g)
        if case.get("norm"):
            for n in ("q_weight", "k_weight"):
                st[n] = 1 + 0.2 * r(D)
                leaves.append(n)
            if case["norm"] == "layer":
                for n in ("q_bias", "k_bias"):
                    st[n] = 0.2 * r(D)
                    leaves.append(n)
        st["offsets"] = None
        if case["S"]:
            off = [0]
            for n in _lengths(case):
                off.append(off[-1] + n)
            st["offsets"] = torch.tensor(off, dtype=torch.int32, device=DEV)
        if train:
            for n, h in (("do", H),) if op == "window" else (("dq", H), ("dk", Hk)):
                st[n] = r(*lead, h, D).to(torch.bfloat16)
    st["leaves"] = leaves
    if train:
        for n in leaves:
            st[n].requires_grad_()
    if own and case.get("bands"):
        # what a program keeps beside its weights
        from makani_b200.ops.rotary import RotaryAxes
        st["axes"] = RotaryAxes(_sizes(case), base=10000.0, interleaved=case["inter"])
    return st


def _sum_type(case):
    return torch.float32 if "fp32" in (case["x"], case["residual"]) else TYPES[case["x"]]


# ---------------------------------------------------------------------------------------------------- the operators, plain and own

def _angles(case, positions):
    """cos and signed sin of every channel [N, D] in 32 bits from angles in 64, and the channel that it is turned with.  Pair i of a band of b
    channels turns by position * 10000^(-2 i / b)."""
    D, N = case["D"], case["N"]
    cos, sin = torch.ones(N, D, device=DEV), torch.zeros(N, D, device=DEV)
    partner = torch.arange(D, device=DEV)
    at = 0
    for a, b in enumerate(_sizes(case)):
        i = torch.arange(b // 2, device=DEV)
        turn = positions[:, a, None].double() * 10000.0 ** (-2.0 * i.double() / b)
        lo, hi = (at + 2 * i, at + 2 * i + 1) if case["inter"] else (at + i, at + b // 2 + i)
        c, s = torch.cos(turn).float(), torch.sin(turn).float()
        cos[:, lo], cos[:, hi], sin[:, lo], sin[:, hi] = c, c, -s, s
        partner[lo], partner[hi] = hi, lo
        at += b
    return cos[:, None, :], sin[:, None, :], partner


def _plain_norm(case, x, w, b):
    """(normalised x, its factor, xh) in 32 bits."""
    if case["norm"] == "layer":
        x = x - x.mean(-1, keepdim=True)
    rstd = 1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)
    xh = x * rstd
    y = xh * w
    return (y if b is None else y + b), rstd, xh


def _plain_qk(st, x, which, grad):
    """Queries or keys [.., heads, D] normed and turned, in 32 bits (None: only their gradient, without a norm), and with `grad` the gradients of x,
    weight and bias."""
    case = st["case"]
    norm = case.get("norm")
    w, b = (st[which + n].detach() if which + n in st else None for n in ("_weight", "_bias"))
    cos, sin, partner = st.get("angles") or _angles(case, st["positions"])
    y, rstd, xh = _plain_norm(case, x, w, b) if norm else (x, None, None)
    if x is not None:
        y = y * cos + y[..., partner] * sin
    if grad is None:
        return y, None, None, None
    g = grad.float()
    g = g * cos - g[..., partner] * sin
    if not norm:
        return y, g, None, None
    dw, db = (g * xh).flatten(0, -2).sum(0), (None if b is None else g.flatten(0, -2).sum(0))
    g = g * w
    dx = g - xh * (g * xh).mean(-1, keepdim=True)
    if norm == "layer":
        dx = dx - g.mean(-1, keepdim=True)
    return y, dx * rstd, dw, db


def _split(st):
    case = st["case"]
    return st["qkv"].detach().unflatten(-1, (-1, case["D"])).split([case["H"], case["Hk"], case["Hk"]], dim=-2)


def _rotated(st):
    """Rotary positions, with or without norms in front: queries and keys out of a fused projection."""
    case = st["case"]
    if not own:
        out = {}
        for n in ("q", "k"):
            y, dx, dw, db = _plain_qk(st, st[n].detach().float(), n, st.get("d" + n))
            out[n] = y.to(torch.bfloat16)
            if dx is not None:
                out["d" + n] = dx.to(torch.bfloat16)
            if dw is not None:
                out["d" + n + "_weight"] = dw
            if db is not None:
                out["d" + n + "_bias"] = db
        return out
    from makani_b200.ops import rotary as rot
    if case.get("norm"):
        q, k = rot.norm_rotary_qk(st["q"], st["k"], st["q_weight"], st["k_weight"], st["positions"], st["axes"], q_bias=st.get("q_bias"), k_bias=st.get("k_bias"),
                                  eps=EPS, norm=case["norm"])
    else:
        q, k = rot.rotary_qk(st["q"], st["k"], st["positions"], st["axes"])
    out = dict(q=q.detach(), k=k.detach())
    if case["train"]:
        grads = torch.autograd.grad((q, k), [st[n] for n in st["leaves"]], (st["dq"], st["dk"]))
        out.update({"d" + n: g for n, g in zip(st["leaves"], grads)})
    return out


def _seen(st, N):
    """[N, N]: whether a query sees a key, and the queries that belong to a sequence (None: all)."""
    case = st["case"]
    at = torch.arange(N, device=DEV)
    first, rows = torch.zeros_like(at), None
    mask = torch.ones(N, N, dtype=torch.bool, device=DEV)
    if st["offsets"] is not None:
        seq = torch.searchsorted(st["offsets"][1:].contiguous(), at.int(), right=True)
        rows = seq < case["S"]
        first = st["offsets"][seq.clamp(max=case["S"] - 1)].long()
        mask = (seq[:, None] == seq[None, :]) & rows[:, None]
    i, j = at[:, None], at[None, :]
    mask &= ((j >= i - case["left"]) & (j <= i + case["right"])) | (j - first[None, :] < case["sinks"])
    if case["causal"]:
        mask &= j <= i
    return mask, rows


def _attend(q, k, v, do, mask, rows, scale):
    """Heads [.., N, D] in the type of q: o and, with `do`, the gradients."""
    p = torch.matmul(q, k.transpose(-1, -2)).mul_(scale)
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


def _windowed(st):
    case = st["case"]
    B, N, H, Hk, D, G = *(case[n] for n in ("B", "N", "H", "Hk", "D")), case["H"] // case["Hk"]
    if own:
        return _windowed_own(st)
    packed, train = st["offsets"] is not None, case["train"]
    lead = (lambda t: t[None]) if packed else (lambda t: t)
    if case["path"]:
        q, k, v = (t.float() for t in _split(st))
        st = dict(st, angles=_angles(case, st["positions"]))
        # (attention takes queries and keys in the type of the projection)
        q, k = (_plain_qk(st, t, n, None)[0].to(torch.bfloat16).float() for n, t in (("q", q), ("k", k)))
    else:
        q, k, v = (lead(st[n].detach().float()) for n in ("q", "k", "v"))
    q, k, v = (t.transpose(1, 2) for t in (q, k, v))        # [B, heads, N, D]
    k, v = (t.repeat_interleave(G, 1) if G > 1 else t for t in (k, v))
    do = lead(st["do"].float()).transpose(1, 2) if train else None
    mask, rows = _seen(st, N)
    o, dq, dk, dv = _attend(q, k, v, do, mask, rows, D ** -0.5)
    back = (lambda t: t.transpose(1, 2)[0]) if packed else (lambda t: t.transpose(1, 2))
    out = dict(o=back(o))
    if train:
        dk, dv = (t.unflatten(1, (Hk, G)).sum(2) for t in (dk, dv))
        dq, dk, dv = back(dq), back(dk), back(dv)
        if case["path"]:
            (_, dq, _, _), (_, dk, _, _) = (_plain_qk(st, None, n, d) for n, d in (("q", dq), ("k", dk)))
            out["dqkv"] = torch.cat([dq, dk, dv], dim=-2).flatten(-2)
        else:
            out.update(dq=dq, dk=dk, dv=dv)
    return {n: t.to(torch.bfloat16).contiguous() for n, t in out.items()}


def _windowed_own(st):
    case = st["case"]
    more = dict(causal=case["causal"], window=(case["left"], case["right"]), sinks=case["sinks"])
    if case["path"]:
        from makani_b200.ops import rotary as rot
        o = rot.rotary_attention_qkv(st["qkv"], case["H"], case["Hk"], st["positions"], st["axes"], **more)
    else:
        from makani_b200.ops import attention as attn_ops
        o = attn_ops.attention(st["q"], st["k"], st["v"], offsets=st["offsets"], **more)
    out = dict(o=o.detach())
    if case["train"]:
        out.update({"d" + n: g for n, g in zip(st["leaves"], torch.autograd.grad(o, [st[n] for n in st["leaves"]], st["do"]))})
    return out


def _words(seed, n):
    """32 random bits of every element, as int64: Philox4x32 of ten rounds (Salmon et al. 2011); element i has word i % 4 of the block whose counter is
    (number of the call, i // 4), 64 bits each, and whose key is the seed."""
    m = 0xFFFFFFFF
    block = torch.arange((n + 3) // 4, dtype=torch.int64, device=DEV)
    number = seed[1].expand_as(block)
    c = [number & m, (number >> 32) & m, block & m, block >> 32]
    k0, k1 = seed[0] & m, (seed[0] >> 32) & m
    for _ in range(10):
        p0, p1 = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [((p1 >> 32) & m) ^ c[1] ^ k0, p1 & m, ((p0 >> 32) & m) ^ c[3] ^ k1, p0 & m]
        k0, k1 = (k0 + 0x9E3779B9) & m, (k1 + 0xBB67AE85) & m
    return torch.stack(c, -1).flatten()[:n]


def _dropped(st):
    """x / (1 - p) where the element's word is at least p 2^32, else 0; plus the residual."""
    case = st["case"]
    if not own:
        keep = _words(st["seed"], case["n"]) >= round(case["p"] * 2 ** 32)
        f = keep.float() / (1 - case["p"])
        y = st["x"].detach().float() * f
        if "residual" in st:
            y = y + st["residual"].detach().float()
        out = dict(y=y.to(_sum_type(case)))
        if case["train"]:
            out["dx"] = (st["dy"].float() * f).to(st["x"].dtype)
            if "residual" in st:
                out["dresidual"] = st["dy"].to(st["residual"].dtype)
        return out
    from makani_b200.ops import dropout as drop_ops
    if "residual" in st:
        y = drop_ops.dropout_add(st["x"], st["residual"], case["p"], seed=st["seed"])
    else:
        y = drop_ops.dropout(st["x"], case["p"], seed=st["seed"])
    out = dict(y=y.detach())
    if case["train"]:
        out.update({"d" + n: g for n, g in zip(st["leaves"], torch.autograd.grad(y, [st[n] for n in st["leaves"]], st["dy"]))})
    return out


def run(state):
    return {"rotary": _rotated, "normed": _rotated, "window": _windowed, "dropout": _dropped}[state["case"]["op"]](state)


# ---------------------------------------------------------------------------------------------------- what a pass cannot do without

def work(case):
    """Bytes: every input read once, every output written once.  Flops: the products of attention (two forward; backward the four of its
    formulas, the probabilities taken as known), a few operations per element of the rest."""
    train, op = case["train"], case["op"]
    if op == "dropout":
        n, bx, br = case["n"], 4 if case["x"] == "fp32" else 2, {"": 0, "bf16": 2, "fp32": 4}[case["residual"]]
        by = max(bx, br)
        size = n * (bx + br + by) + 16
        if train:
            size += n * (by + bx) + (n * br if br and br < by else 0)       # (the residual's gradient is dy itself, or its rounding)
        return {"bytes": size, "flops": n * (12 if train else 6)}
    B, N, H, Hk, D = (case[n] for n in ("B", "N", "H", "Hk", "D"))
    q, k = 2 * B * N * H * D, 2 * B * N * Hk * D
    place = N * len(_sizes(case)) * 4
    norm = bool(case.get("norm"))
    if op != "window":
        size = 2 * (q + k) + place
        if train:           # gradients in and out; with norms x is read again
            size += 2 * (q + k) + place + ((q + k) if norm else 0)
        return {"bytes": size, "flops": B * N * (H + Hk) * D * ((3 if not norm else 8) + (0 if not train else 3 if not norm else 18))}
    size = 2 * q + 2 * k + (place if case["path"] else 0)
    if train:
        size += 3 * q + 4 * k + q       # q, o, do, dq; k, v, dk, dv
    pairs = sum(_visible(case, n) for n in (_lengths(case) if case["S"] else [N] * B))
    return {"bytes": size, "flops": pairs * H * D * 2 * (6 if train else 2)}


# ---------------------------------------------------------------------------------------------------- definition in 64 bits

def exact(case, seed):
    st = prepare(case, seed)
    return {"rotary": _exact_rotated, "normed": _exact_rotated, "window": _exact_windowed, "dropout": _exact_dropped}[case["op"]](st)


def _exact_turned(st, x, which):
    """Norm and rotation of one tensor in 64 bits as a function that autograd can follow; complex numbers turn."""
    case = st["case"]
    if case.get("norm"):
        w, b = st[which + "_weight64"], st.get(which + "_bias64")
        if case["norm"] == "layer":
            var, mean = torch.var_mean(x, dim=-1, correction=0, keepdim=True)
            x = (x - mean) / torch.sqrt(var + EPS) * w
        else:
            x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + EPS) * w
        x = x if b is None else x + b
    parts, at = [], 0
    for a, n in enumerate(_sizes(case)):
        band = x[..., at:at + n]
        pairs = band.unflatten(-1, (n // 2, 2)) if case["inter"] else band.unflatten(-1, (2, n // 2)).transpose(-1, -2)
        angle = st["positions"].double()[:, None, a, None] / 10000.0 ** (torch.arange(0, n, 2, device=DEV, dtype=torch.float64) / n)
        turned = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * torch.polar(torch.ones_like(angle), angle))
        parts.append(turned.flatten(-2) if case["inter"] else turned.transpose(-1, -2).flatten(-2))
        at += n
    return torch.cat(parts + [x[..., at:]], -1)


def _leaves64(st):
    for n in ("q_weight", "k_weight", "q_bias", "k_bias"):
        if n in st:
            st[n + "64"] = st[n].detach().double().requires_grad_(st["case"]["train"])


def _exact_rotated(st):
    case = st["case"]
    _leaves64(st)
    x = [st[n].detach().double().requires_grad_(case["train"]) for n in ("q", "k")]
    q, k = (_exact_turned(st, t, n) for t, n in zip(x, ("q", "k")))
    out = dict(q=q.detach(), k=k.detach())
    if case["train"]:
        grads = torch.autograd.grad((q, k), x + [st[n + "64"] for n in st["leaves"][2:]], (st["dq"].double(), st["dk"].double()))
        out.update({"d" + n: g for n, g in zip(st["leaves"], grads)})
    return out


def _exact_windowed(st):
    """Sequence by sequence and head by head, gradients by the chain rule of the definition."""
    case = st["case"]
    B, N, H, Hk, D, G = *(case[n] for n in ("B", "N", "H", "Hk", "D")), case["H"] // case["Hk"]
    if case["path"]:
        x = st["qkv"].detach().double().requires_grad_(case["train"])
        q0, k0, v = x.unflatten(-1, (-1, D)).split([H, Hk, Hk], dim=-2)
        q0, k0 = _exact_turned(st, q0, "q"), _exact_turned(st, k0, "k")
        q, k, v = q0.detach().to(torch.bfloat16).double(), k0.detach().to(torch.bfloat16).double(), v.detach()
    else:
        q, k, v = (st[n].detach().double().reshape(B, N, -1, D) for n in ("q", "k", "v"))
    do = st["do"].double().reshape(B, N, H, D) if case["train"] else None
    o, dq, dk, dv = torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    lens, at, bounds = _lengths(case) if case["S"] else [N], 0, []
    for n in lens:
        bounds.append((at, at + n))
        at += n
    for lo, hi in bounds:
        n = hi - lo
        if n == 0:
            continue
        away = torch.arange(n, device=DEV)[:, None] - torch.arange(n, device=DEV)[None, :]         # query less key
        hidden = (away > case["left"]) | (away < -case["right"])
        hidden[:, :case["sinks"]] = False
        if case["causal"]:
            hidden |= away < 0
        for b in range(B):
            for h in range(H):
                qs, ks, vs = q[b, lo:hi, h], k[b, lo:hi, h // G], v[b, lo:hi, h // G]
                logits = ((qs @ ks.mT) / math.sqrt(D)).masked_fill_(hidden, -math.inf)
                prob = torch.exp(logits - torch.logsumexp(logits, -1, keepdim=True))
                del logits
                o[b, lo:hi, h] = prob @ vs
                if do is None:
                    continue
                gs = do[b, lo:hi, h]
                dv[b, lo:hi, h // G] += prob.mT @ gs
                dprob = gs @ vs.mT
                dlogit = prob * (dprob - (prob * dprob).sum(-1, keepdim=True))
                del dprob, prob
                dq[b, lo:hi, h] = dlogit @ ks / math.sqrt(D)
                dk[b, lo:hi, h // G] += dlogit.mT @ qs / math.sqrt(D)
    lay = (lambda t: t[0]) if case["S"] else (lambda t: t)
    out = dict(o=lay(o))
    if do is not None:
        if case["path"]:
            grad, = torch.autograd.grad((q0, k0), x, (dq, dk))
            grad[..., (H + Hk) * D:] = dv.flatten(-2)
            out["dqkv"] = grad
        else:
            out.update(dq=lay(dq), dk=lay(dk), dv=lay(dv))
    return out


def _exact_dropped(st):
    """The generator in unsigned arithmetic on the host."""
    case = st["case"]
    n, key, number = case["n"], *(int(v) for v in st["seed"].tolist())
    low, half = np.uint64(0xFFFFFFFF), np.uint64(32)
    block = np.arange((n + 3) // 4, dtype=np.uint64)
    state = np.stack([np.full_like(block, number & 0xFFFFFFFF), np.full_like(block, (number >> 32) & 0xFFFFFFFF), block & low, block >> half])
    keys = [key & 0xFFFFFFFF, (key >> 32) & 0xFFFFFFFF]
    for _ in range(10):
        a, b = state[0] * np.uint64(0xD2511F53), state[2] * np.uint64(0xCD9E8D57)
        state = np.stack([(b >> half) ^ state[1] ^ np.uint64(keys[0]), b & low, (a >> half) ^ state[3] ^ np.uint64(keys[1]), a & low])
        keys = [(keys[0] + 0x9E3779B9) & 0xFFFFFFFF, (keys[1] + 0xBB67AE85) & 0xFFFFFFFF]
    words = torch.from_numpy(state.T.reshape(-1)[:n].astype(np.int64)).to(DEV)
    keep = words >= round(case["p"] * 2 ** 32)
    zero = torch.zeros((), dtype=torch.float64, device=DEV)
    y = torch.where(keep, st["x"].detach().double() / (1 - case["p"]), zero)
    out = dict(y=y + st["residual"].detach().double() if "residual" in st else y)
    if case["train"]:
        out["dx"] = torch.where(keep, st["dy"].double() / (1 - case["p"]), zero)
        if "residual" in st:
            out["dresidual"] = st["dy"].double()
    return out
