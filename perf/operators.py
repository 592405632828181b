"""The operators of packed training batches, as timed cases: attention under document, prefix and distance rules, rotary positions with
several axes, and the global gradient norm with clipping.

A packed batch holds several documents per sequence.  Its attention may not cross them, may look both ways inside a document's prefix, and
may cap its scores or lower them with distance; images inside it are positioned by time, height and width; and the step ends with the norm of
all gradients.  ``own`` false: elementary torch operations in 32 bits.  ``own`` true: the calls that a user makes of ``lightron_b200``.
"""
from __future__ import annotations

import math
import random

import torch

own = False

BF16 = torch.bfloat16
THETA = 10000.0


def listed():
    return [
        # a micro-batch of the small decoder's sample run, scores lowered with distance: launches and latency
        dict(name="attn_alibi_small", kind="attn", B=4, S=128, heads=12, kv=12, d=64, causal=True, docs=0, prefix=0.0, cap=0.0, alibi=True, grad=True),
        # the 1.1 B decoder at its training batch, documents of 300 tokens on average packed into 2048, a padded end
        dict(name="attn_docs_1b", kind="attn", B=8, S=2048, heads=32, kv=4, d=64, causal=True, docs=300, prefix=0.0, cap=0.0, alibi=False, grad=True),
        # the 8 B decoder at its training sequence with capped scores: the largest
        dict(name="attn_softcap_8b", kind="attn", B=1, S=8192, heads=32, kv=8, d=128, causal=True, docs=0, prefix=0.0, cap=50.0, alibi=False, grad=True),
        # documents of prompt and answer, the prompt seen both ways, in sequences of a ragged length
        dict(name="attn_prefix_docs_ragged", kind="attn", B=3, S=1531, heads=32, kv=8, d=128, causal=True, docs=500, prefix=0.4, cap=0.0, alibi=False, grad=True),
        # evaluation of packed texts that are seen both ways, capped: forward only, an odd length
        dict(name="attn_twoway_cap_eval", kind="attn", B=2, S=4099, heads=16, kv=16, d=64, causal=False, docs=900, prefix=0.0, cap=30.0, alibi=False, grad=False),
        # everything at once, at a head size between the usual ones
        dict(name="attn_alibi_cap_prefix_d96", kind="attn", B=2, S=1000, heads=16, kv=4, d=96, causal=True, docs=0, prefix=0.3, cap=30.0, alibi=True, grad=True),
        # queries and keys of the 1.1 B decoder at its training batch, positioned by time, height and width, and back
        dict(name="rope_axes_1b", kind="rope", B=8, S=2048, heads=36, d=64),
        # one short sequence with an image
        dict(name="rope_axes_small", kind="rope", B=1, S=300, heads=40, d=128),
        # gradients of the four-layer configuration in fp32, clipped
        dict(name="clip_tiny_fp32", kind="clip", dim=256, layers=4, hidden=688, kvdim=256, vocab=8192, type="fp32", clip=True),
        # gradients of the small decoder, clipped
        dict(name="clip_small", kind="clip", dim=768, layers=12, hidden=2048, kvdim=768, vocab=32000, type="bf16", clip=True),
        # gradients of the 1.1 B decoder, clipped
        dict(name="clip_1b", kind="clip", dim=2048, layers=22, hidden=5632, kvdim=256, vocab=32000, type="bf16", clip=True),
        # the norm alone, over matrices in bf16 and vectors in fp32 whose sizes are odd
        dict(name="norm_mixed_odd", kind="clip", dim=1021, layers=16, hidden=2731, kvdim=255, vocab=8191, type="mixed", clip=False),
    ]


def _log_int(rng, lo, hi, step=1):
    v = math.exp(rng.uniform(math.log(lo), math.log(hi + step)))
    return max(lo, min(hi, int(v) // step * step))


def draw(rng):
    kind = rng.choice(["attn", "attn", "attn", "rope", "clip"])
    if kind == "attn":
        d = rng.choice([64, 128, 64, 128, 80, 96, 32])
        kv = rng.choice([1, 2, 4, 8])
        heads = kv * rng.choice([1, 2, 4, 8] if kv < 8 else [1, 4])
        causal = rng.random() < 0.75
        # (one token alone has no gradient by its scores: there is nothing to compare)
        S = _log_int(rng, 2, 8192 if causal else 5700)
        return dict(kind=kind, B=rng.randint(1, max(1, min(8, 8192 // S))), S=S, heads=heads, kv=kv, d=d, causal=causal,
                    docs=rng.choice([0, _log_int(rng, 20, 2000)]) if S >= 16 else 0, prefix=rng.choice([0.0, 0.0, 0.4]) if causal else 0.0,
                    cap=rng.choice([0.0, 0.0, 30.0, 50.0]), alibi=rng.random() < 0.3, grad=rng.random() < 0.75)
    if kind == "rope":
        S = _log_int(rng, 1, 8192)
        return dict(kind=kind, B=rng.randint(1, max(1, min(8, 16384 // S))), S=S, heads=_log_int(rng, 1, 48), d=rng.choice([32, 64, 80, 96, 128]))
    dim = _log_int(rng, 64, 1280)
    return dict(kind=kind, dim=dim, layers=rng.randint(1, 16), hidden=_log_int(rng, dim, 4 * dim), kvdim=max(1, dim // rng.choice([1, 4, 8])),
                vocab=rng.choice([1000, 8191, 32000]), type=rng.choice(["bf16", "fp32", "mixed"]), clip=rng.random() < 0.7)


# ---- inputs ------------------------------------------------------------------------------------


class _Draws:
    """Normal tensors on the GPU from one seeded generator."""

    def __init__(self, seed):
        self.g = torch.Generator(device="cuda").manual_seed(int(seed))

    def __call__(self, *shape, std=1.0, dtype=BF16):
        return (torch.randn(*shape, generator=self.g, device="cuda", dtype=torch.float32) * std).to(dtype)


def _documents(c):
    """Lengths of the documents of every sequence, spread over a factor of 16 around the mean, and of the padding behind them: the same for
    every seed but for their order."""
    rng = random.Random("%d %d %d" % (c["B"], c["S"], c["docs"]))
    rows = []
    for _ in range(c["B"]):
        left, lens = c["S"], []
        while left > 0 and c["docs"]:
            n = min(left, max(1, int(c["docs"] * 4 ** rng.uniform(-1, 1))))
            if n == left and lens and rng.random() < 0.5:
                break                                   # what does not fit is padding
            lens.append(n)
            left -= n
        rows.append((lens or [c["S"]], left if lens else 0))
    return rows


def _prefix(c, n):
    return int(n * c["prefix"])


def _slopes(heads):
    return 2.0 ** (-8.0 * (torch.arange(heads, device="cuda", dtype=torch.float32) + 1) / heads)


def _grad_shapes(c):
    """Parameters of a decoder in the order of its modules."""
    shapes = [(c["vocab"], c["dim"])]
    for _ in range(c["layers"]):
        shapes += [(c["dim"], c["dim"]), (c["kvdim"], c["dim"]), (c["kvdim"], c["dim"]), (c["dim"], c["dim"]), (c["hidden"], c["dim"]),
                   (c["hidden"], c["dim"]), (c["dim"], c["hidden"]), (c["dim"],), (c["dim"],)]
    return shapes + [(c["dim"],), (c["vocab"], c["dim"])]


def _views(flat, shapes):
    out, off = [], 0
    for s in shapes:
        n = math.prod(s)
        out.append(flat[off:off + n].view(s))
        off += n
    return out


def _axes(d):
    """Axis of each pair: an eighth of the head for time, the rest of the pairs for height and width."""
    t = d // 8
    h = (d // 2 - t) // 2
    return [0] * t + [1] * h + [2] * (d // 2 - t - h)


def prepare(c, seed):
    r = _Draws(seed)
    c = dict(c)
    if c["kind"] == "attn":
        return _prepare_attention(c, seed, r)
    if c["kind"] == "rope":
        return _prepare_rope(c, seed, r)
    shapes = _grad_shapes(c)
    types = {"bf16": [BF16], "fp32": [torch.float32], "mixed": [BF16, torch.float32]}[c["type"]]
    grads = [r(*s, std=1e-3, dtype=types[-1] if len(s) == 1 else types[0]) for s in shapes]
    st = dict(c=c, grads=grads, max_norm=1.0)
    if c["clip"]:
        # clipped gradients go to buffers of their own, one for each type, as they would for a flat optimizer
        st["flat"] = [torch.empty(sum(g.numel() for g in grads if g.dtype == t), dtype=t, device="cuda") for t in types]
        views = {t: iter(_views(f, [g.shape for g in grads if g.dtype == t])) for t, f in zip(types, st["flat"])}
        st["out"] = [next(views[g.dtype]) for g in grads]
    return st


def _prepare_attention(c, seed, r):
    B, S, hq, hkv, d = c["B"], c["S"], c["heads"], c["kv"], c["d"]
    # the fused projection's output: heads of q, k and v side by side in a token's row; scores have a standard deviation of 4 where they are capped
    std = 2.0 if c["cap"] else 1.0
    qkv = r(B, S, (hq + 2 * hkv) * d, std=std)
    q, k, v = (t.unflatten(2, (-1, d)) for t in qkv.split([hq * d, hkv * d, hkv * d], dim=2))
    st = dict(c=c, q=q, k=k, v=v, do=r(B, S, hq, d) if c["grad"] else None, scale=d ** -0.5, causal=c["causal"], cap=c["cap"],
              slopes=_slopes(hq) if c["alibi"] else None, documents=None, prefix=None)
    ids, marks = torch.full((B, S), -1, dtype=torch.int32), torch.zeros(B, S, dtype=torch.bool)
    for b, (lens, _) in enumerate(_documents(c)):
        lens = list(lens)
        random.Random(seed * 1000 + b).shuffle(lens)
        at = 0
        for i, n in enumerate(lens):
            ids[b, at:at + n] = i
            marks[b, at:at + _prefix(c, n)] = True
            at += n
    if c["docs"]:
        st["documents"] = ids.cuda()
    if c["prefix"]:
        st["prefix"] = marks.cuda()
    if c["grad"]:
        st.update({n: st[n].detach().requires_grad_() for n in ("q", "k", "v")})
    return st


def _prepare_rope(c, seed, r):
    B, S, h, d = c["B"], c["S"], c["heads"], c["d"]
    inv = THETA ** (-torch.arange(0, d, 2, device="cuda", dtype=torch.float64) / d)
    ang = torch.outer(torch.arange(S + 64, device="cuda", dtype=torch.float64), inv)
    # text counts on all three axes together; an image of w columns stays at one time
    rng = random.Random(seed)
    pos = torch.empty(3, B, S, dtype=torch.int32)
    for b in range(B):
        at, now = 0, 0
        while at < S:
            n = min(S - at, rng.randint(5, 200))
            i = torch.arange(n, dtype=torch.int32)
            if rng.random() < 0.5:
                w = rng.randint(3, 16)
                pos[0, b, at:at + n], pos[1, b, at:at + n], pos[2, b, at:at + n] = now, now + i // w, now + i % w
                now += max((n - 1) // w, min(w, n) - 1) + 1
            else:
                pos[:, b, at:at + n] = now + i
                now += n
            at += n
    rows = r(B, S, (h + 2) * d)                          # heads of a wider row, as of a fused projection
    x = rows.unflatten(2, (-1, d))[:, :, :h]
    return dict(c=c, x=x.detach().requires_grad_(), dy=r(B, S, h, d), cos=ang.cos().float(), sin=ang.sin().float(), positions=pos.cuda(), axes=_axes(d))


# ---- one pass ----------------------------------------------------------------------------------


def run(st):
    kind = st["c"]["kind"]
    if own:
        return {"attn": _attention_own, "rope": _rope_own, "clip": _clip_own}[kind](st)
    with torch.no_grad():
        return {"attn": _attention_plain, "rope": _rope_plain, "clip": _clip_plain}[kind](st)


def _attention_own(st):
    from lightron_b200.ops import functional as OF
    q, k, v = st["q"], st["k"], st["v"]
    mask = None
    if st["documents"] is not None or st["prefix"] is not None:
        # (a model makes it once per batch, for all of its layers)
        mask = OF.attention_mask(documents=st["documents"], prefix=st["prefix"], causal=st["causal"])
    o = OF.masked_attention(q, k, v, mask=mask, causal=st["causal"], scale=st["scale"], softcap=st["cap"], slopes=st["slopes"])
    if st["do"] is None:
        return o
    return (o, *torch.autograd.grad(o, (q, k, v), st["do"]))


def _visible(st):
    """[B, 1, 1, S, S]: whether query i sees key j."""
    c = st["c"]
    i = torch.arange(c["S"], device="cuda")
    see = (i[None, :] <= i[:, None])[None] if c["causal"] else torch.ones(1, c["S"], c["S"], dtype=torch.bool, device="cuda")
    if st["prefix"] is not None:
        see = see | st["prefix"][:, None, :]
    if st["documents"] is not None:
        ids = st["documents"]
        see = see & (ids[:, :, None] == ids[:, None, :]) & (ids[:, :, None] >= 0)
    return see[:, None, None]


def _attention_plain(st):
    c = st["c"]
    rep = c["heads"] // c["kv"]
    q = st["q"].float().unflatten(2, (-1, rep)).permute(0, 2, 3, 1, 4)      # [B, kv, rep, S, d]
    k, v = (st[n].float().permute(0, 2, 1, 3)[:, :, None] for n in ("k", "v"))      # [B, kv, 1, S, d]
    s = (q @ k.transpose(-1, -2)).mul_(st["scale"])
    if c["cap"]:
        t = torch.tanh(s / c["cap"])
        s = c["cap"] * t
    if st["slopes"] is not None:
        i = torch.arange(c["S"], device="cuda", dtype=torch.float32)
        s -= st["slopes"].view(c["kv"], rep, 1, 1) * (i[:, None] - i[None, :]).abs()
    s.masked_fill_(~_visible(st), float("-inf"))
    p = torch.exp(s.sub_(s.amax(dim=-1, keepdim=True).clamp_min(-3e38)))
    del s
    p /= p.sum(dim=-1, keepdim=True).clamp_min(1e-38)
    o = p @ v

    def tokens_first(x):
        return x.flatten(1, 2).transpose(1, 2).to(BF16)

    if st["do"] is None:
        return tokens_first(o)
    do = st["do"].float().unflatten(2, (-1, rep)).permute(0, 2, 3, 1, 4)
    dv = (p.transpose(-1, -2) @ do).sum(2, keepdim=True)
    ds = (do @ v.transpose(-1, -2)).sub_((o * do).sum(dim=-1, keepdim=True)).mul_(p).mul_(st["scale"])
    del p
    if c["cap"]:
        ds *= 1 - t * t
    dq, dk = ds @ k, (ds.transpose(-1, -2) @ q).sum(2, keepdim=True)
    return tuple(tokens_first(x) for x in (o, dq, dk, dv))


def _rope_own(st):
    from lightron_b200.ops import functional as OF
    y = OF.rope_axes(st["x"], st["cos"], st["sin"], st["positions"], st["axes"])
    return y, torch.autograd.grad(y, st["x"], st["dy"])[0]


def _rope_plain(st):
    axis = torch.tensor(st["axes"], device="cuda")
    pair = torch.arange(axis.numel(), device="cuda")
    at = st["positions"].long()[axis].permute(1, 2, 0)                 # [B, S, d/2]
    cos, sin = st["cos"][at, pair][:, :, None], st["sin"][at, pair][:, :, None]

    def turn(x, sin):
        x = x.float()
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack((a * cos - b * sin, a * sin + b * cos), dim=-1).flatten(-2).to(BF16)

    return turn(st["x"], sin), turn(st["dy"], -sin)


def _clip_own(st):
    from lightron_b200.ops import functional as OF
    if not st["c"]["clip"]:
        return OF.grad_norm(st["grads"])
    norm = OF.clip_grad_norm(st["grads"], st["max_norm"], out=st["out"])
    return [norm, *st["flat"]]


def _clip_plain(st):
    norm = torch.stack([g.float().square().sum() for g in st["grads"]]).sum().sqrt()
    if not st["c"]["clip"]:
        return norm
    scale = (st["max_norm"] / (norm + 1e-6)).clamp_max(1.0)
    torch._foreach_copy_(st["out"], [(g.float() * scale).to(g.dtype) for g in st["grads"]])
    return [norm, *st["flat"]]


# ---- what a pass cannot do without -------------------------------------------------------------


def _pairs(c):
    """Pairs of query and key that see each other, over all sequences."""
    n = 0
    for lens, _ in _documents(c):
        for s in lens:
            p = _prefix(c, s)
            n += s * s if not c["causal"] else s * (s + 1) // 2 + p * (p - 1) // 2
    return n


def work(c):
    if c["kind"] == "attn":
        tokens = c["B"] * c["S"]
        once = tokens * (2 * c["heads"] + 2 * c["kv"]) * c["d"] * 2                         # q, k, v, o
        if c["grad"]:
            once += tokens * (2 * c["heads"] + 2 * c["kv"]) * c["d"] * 2                    # do, dq, dk, dv
        return {"bytes": once, "flops": _pairs(c) * c["heads"] * c["d"] * (14 if c["grad"] else 4)}
    if c["kind"] == "rope":
        n = c["B"] * c["S"] * c["heads"] * c["d"]
        return {"bytes": 4 * n * 2 + 3 * c["B"] * c["S"] * 4, "flops": 2 * n * 3}
    size = {"bf16": (2, 2), "fp32": (4, 4), "mixed": (2, 4)}[c["type"]]
    shapes = _grad_shapes(c)
    read = sum(math.prod(s) * size[len(s) == 1] for s in shapes)
    n = sum(math.prod(s) for s in shapes)
    return {"bytes": read * (2 if c["clip"] else 1), "flops": n * (3 if c["clip"] else 2)}


# ---- 64 bits -----------------------------------------------------------------------------------


def exact(c, seed):
    st = prepare(c, seed)
    if c["kind"] == "attn":
        return _attention_exact(c, st)
    if c["kind"] == "rope":
        return _rope_exact(c, st)
    total = sum(float((g.double() ** 2).sum()) for g in st["grads"])
    norm = torch.tensor(math.sqrt(total), dtype=torch.float64, device="cuda")
    if not c["clip"]:
        return norm
    by = min(1.0, st["max_norm"] / (math.sqrt(total) + 1e-6))
    types = list(dict.fromkeys(f.dtype for f in st["flat"]))
    return [norm, *[torch.cat([g.double().flatten() * by for g in st["grads"] if g.dtype == t]) for t in types]]


def _attention_exact(c, st):
    B, S, hq, hkv, d = c["B"], c["S"], c["heads"], c["kv"], c["d"]
    f64 = dict(dtype=torch.float64, device="cuda")
    q, k, v = (st[n].detach().double() for n in ("q", "k", "v"))
    o = torch.zeros(B, S, hq, d, **f64)
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    for b in range(B):
        # documents one by one: a query's keys are those of its own document
        ids = st["documents"][b].tolist() if st["documents"] is not None else [0] * S
        edges = [i for i in range(S) if i == 0 or ids[i] != ids[i - 1]] + [S]
        for lo, hi in zip(edges[:-1], edges[1:]):
            if ids[lo] < 0:
                continue
            n = hi - lo
            first = int(st["prefix"][b, lo:hi].sum()) if st["prefix"] is not None else 0
            row = torch.arange(n, device="cuda")
            last = torch.full_like(row, n - 1) if not c["causal"] else row.clamp_min(first - 1)      # last key of each query
            hide = row[None, :] > last[:, None]
            away = (row[:, None] - row[None, :]).abs().double()
            for h in range(hq):
                g = h // (hq // hkv)
                x, y, z = (t[b, lo:hi, n_].clone().requires_grad_(c["grad"]) for t, n_ in ((q, h), (k, g), (v, g)))
                s = x @ y.t() * st["scale"]
                if c["cap"]:
                    s = c["cap"] * torch.tanh(s / c["cap"])
                if st["slopes"] is not None:
                    s = s - float(st["slopes"][h]) * away
                r = torch.softmax(s.masked_fill(hide, float("-inf")), dim=-1) @ z
                o[b, lo:hi, h] = r.detach()
                if c["grad"]:
                    gx, gy, gz = torch.autograd.grad(r, (x, y, z), st["do"][b, lo:hi, h].double())
                    dq[b, lo:hi, h] = gx
                    dk[b, lo:hi, g] += gy
                    dv[b, lo:hi, g] += gz
    return (o, dq, dk, dv) if c["grad"] else o


def _rope_exact(c, st):
    axis = st["axes"]
    cos, sin = st["cos"].double(), st["sin"].double()
    y, dx = [], []
    for src, sign, to in ((st["x"], 1.0, y), (st["dy"], -1.0, dx)):
        z = torch.view_as_complex(src.detach().double().unflatten(-1, (-1, 2)).contiguous())
        for i, a in enumerate(axis):
            at = st["positions"][a].long()
            w = torch.complex(cos[at, i], sign * sin[at, i])
            to.append(torch.view_as_real(z[..., i] * w[..., None]))
    return torch.stack(y, dim=-2).flatten(-2), torch.stack(dx, dim=-2).flatten(-2)
