"""The operators of decoders with local attention, as timed cases: attention under a window with sinks, norms of queries and keys for each head
with the position rotation, and the scaled embedding with its gradient by sorted tokens.

Such a decoder scales its embeddings, norms and turns the heads of queries and keys in one pass, and lets a position see a window of the keys before it
and the first few of its document.  ``own`` false: elementary torch operations in 32 bits.  ``own`` true: the calls that a user makes of ``lightron_b200``.
"""
from __future__ import annotations

import math
import random

import torch

own = False

BF16 = torch.bfloat16
THETA = 10000.0
EPS = 1e-6


def listed():
    return [
        # a micro-batch of the small decoder's sample run under a short window: launches and latency
        dict(name="window_small", kind="attn", B=4, Sq=512, S=512, heads=12, kv=12, d=64, window=128, sinks=0, causal=True, docs=0, cap=0.0, alibi=False, grad=True),
        # the 1.1 B decoder at its training batch: documents of 900 tokens packed into 2048, each with four sinks of its own, a padded end
        dict(name="window_docs_1b", kind="attn", B=8, Sq=2048, S=2048, heads=32, kv=4, d=64, window=512, sinks=4, causal=True, docs=900, cap=0.0, alibi=False, grad=True),
        # the 8 B decoder at its training sequence, a window of 1024 and four sinks: the largest
        dict(name="window_8b", kind="attn", B=1, Sq=8192, S=8192, heads=32, kv=8, d=128, window=1024, sinks=4, causal=True, docs=0, cap=0.0, alibi=False, grad=True),
        # capped scores, a ragged length, an odd window, more sinks than a tile holds
        dict(name="window_cap_ragged", kind="attn", B=3, Sq=1531, S=1531, heads=16, kv=4, d=96, window=333, sinks=130, causal=True, docs=0, cap=30.0, alibi=False, grad=True),
        # one new token of eight sequences over a long cache of the 8 B decoder
        dict(name="window_decode_8b", kind="attn", B=8, Sq=1, S=32768, heads=32, kv=8, d=128, window=4096, sinks=4, causal=True, docs=0, cap=0.0, alibi=False, grad=False),
        # queries and keys of the 1.1 B decoder at its training batch, and back
        dict(name="qk_norm_1b", kind="norm", B=8, S=2048, heads=32, kv=4, d=64, far=0, grad=True),
        # of the 8 B decoder, packed documents that count from places of their own
        dict(name="qk_norm_8b", kind="norm", B=1, S=8192, heads=32, kv=8, d=128, far=4000, grad=True),
        # the step of one token in each of 16 sequences
        dict(name="qk_norm_decode", kind="norm", B=16, S=1, heads=32, kv=8, d=128, far=30000, grad=False),
        # one sequence of the small decoder: launches and latency
        dict(name="embed_small", kind="embed", T=512, vocab=32000, dim=768, pad=0.0),
        # the 1.1 B decoder's training batch
        dict(name="embed_1b", kind="embed", T=16384, vocab=32000, dim=2048, pad=0.0),
        # the 8 B decoder's vocabulary: a gradient of a gigabyte
        dict(name="embed_8b", kind="embed", T=8192, vocab=128256, dim=4096, pad=0.0),
        # batches that are padded for the most part, odd sizes: one id has two thirds of all places
        dict(name="embed_padded_odd", kind="embed", T=15001, vocab=8191, dim=1021, pad=0.65),
    ]


def _log_int(rng, lo, hi, step=1):
    v = math.exp(rng.uniform(math.log(lo), math.log(hi + step)))
    return max(lo, min(hi, int(v) // step * step))


def draw(rng):
    kind = rng.choice(["attn", "attn", "attn", "norm", "embed"])
    if kind == "attn":
        d = rng.choice([64, 128, 64, 128, 80, 96, 32])
        kv = rng.choice([1, 2, 4, 8])
        heads = kv * rng.choice([1, 2, 4, 8] if kv < 8 else [1, 4])
        few = rng.random() < 0.25
        c = dict(kind=kind, heads=heads, kv=kv, d=d, sinks=rng.choice([0, 0, 1, 4, 16, 150]), cap=rng.choice([0.0, 0.0, 0.0, 30.0, 50.0]), alibi=rng.random() < 0.15)
        if few:                                          # a few new tokens over a cache
            S = _log_int(rng, 64, 32768)
            return dict(c, B=_log_int(rng, 1, 8), Sq=rng.choice([1, 1, 2, 5, 16]), S=S, window=_log_int(rng, 1, S), causal=True, docs=0, grad=False)
        causal = rng.random() < 0.85
        # (a position that sees itself alone has no gradient by its scores: there would be nothing to compare)
        S = _log_int(rng, 4, 8192 if causal else 5700)
        return dict(c, B=rng.randint(1, max(1, min(8, 8192 // S))), Sq=S, S=S, window=_log_int(rng, 2, S), causal=causal,
                    docs=rng.choice([0, _log_int(rng, 20, 2000)]) if S >= 16 else 0, grad=rng.random() < 0.75)
    if kind == "norm":
        kv = rng.choice([1, 2, 4, 8])
        S = _log_int(rng, 1, 8192)
        return dict(kind=kind, B=rng.randint(1, max(1, min(16, 16384 // S))), S=S, heads=kv * rng.choice([1, 2, 4]), kv=kv, d=rng.choice([32, 64, 80, 96, 128, 256]),
                    far=rng.choice([0, 0, _log_int(rng, 1, 30000)]), grad=rng.random() < 0.75)
    vocab = rng.choice([1000, 8191, 32000, 50257])
    dim = _log_int(rng, 64, 2500)
    return dict(kind=kind, T=_log_int(rng, 1, 32768), vocab=vocab, dim=dim if rng.random() < 0.3 else max(8, dim // 8 * 8), pad=rng.choice([0.0, 0.0, 0.3, 0.9]))


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


def prepare(c, seed):
    return {"attn": _prepare_attention, "norm": _prepare_norm, "embed": _prepare_embedding}[c["kind"]](dict(c), seed, _Draws(seed))


def _prepare_attention(c, seed, r):
    B, Sq, S, hq, hkv, d = c["B"], c["Sq"], c["S"], c["heads"], c["kv"], c["d"]
    std = 2.0 if c["cap"] else 1.0                       # scores have a standard deviation of 4 where they are capped
    if Sq == S:
        # the fused projection's output: heads of q, k and v side by side in a token's row
        q, k, v = (t.unflatten(2, (-1, d)) for t in r(B, S, (hq + 2 * hkv) * d, std=std).split([hq * d, hkv * d, hkv * d], dim=2))
    else:
        q, k, v = r(B, Sq, hq, d, std=std), r(B, S, hkv, d, std=std), r(B, S, hkv, d, std=std)
    slopes = 2.0 ** (-8.0 * (torch.arange(hq, device="cuda", dtype=torch.float32) + 1) / hq) if c["alibi"] else None
    st = dict(c=c, q=q, k=k, v=v, do=r(B, Sq, hq, d) if c["grad"] else None, scale=d ** -0.5, slopes=slopes, documents=None)
    if c["docs"]:
        ids = torch.full((B, S), -1, dtype=torch.int32)
        for b, (lens, _) in enumerate(_documents(c)):
            lens = list(lens)
            random.Random(seed * 1000 + b).shuffle(lens)
            ids[b, :sum(lens)] = torch.repeat_interleave(torch.arange(len(lens), dtype=torch.int32), torch.tensor(lens))
        st["documents"] = ids.cuda()
    if c["grad"]:
        st.update({n: st[n].detach().requires_grad_() for n in ("q", "k", "v")})
    return st


def _prepare_norm(c, seed, r):
    B, S, hq, hkv, d = c["B"], c["S"], c["heads"], c["kv"], c["d"]
    inv = THETA ** (-torch.arange(0, d, 2, device="cuda", dtype=torch.float64) / d)
    ang = torch.outer(torch.arange(S + c["far"], device="cuda", dtype=torch.float64), inv)
    # projections have other sizes in other heads and tokens; weights lie around one
    qkv = r(B, S, (hq + 2 * hkv) * d) * torch.exp(r(B, S, 1, std=0.5))
    q, k = (t.unflatten(2, (-1, d)).detach() for t in qkv.split([hq * d, hkv * d, hkv * d], dim=2)[:2])
    wq, wk = ((1 + r(d, std=0.2, dtype=torch.float32)).to(BF16) for _ in range(2))
    st = dict(c=c, q=q, k=k, wq=wq, wk=wk, cos=ang.cos().float(), sin=ang.sin().float(), positions=None)
    if c["far"]:                                         # every sequence begins at a place of its own
        rng = random.Random(seed)
        first = torch.tensor([rng.randint(0, c["far"]) for _ in range(B)], dtype=torch.int32)
        st["positions"] = (first[:, None] + torch.arange(S, dtype=torch.int32)).cuda()
    if c["grad"]:
        st.update({n: st[n].requires_grad_() for n in ("q", "k", "wq", "wk")}, dq=r(B, S, hq, d), dk=r(B, S, hkv, d))
    return st


def _prepare_embedding(c, seed, r):
    T, V, H = c["T"], c["vocab"], c["dim"]
    # words by the logarithm of their rank, at places of their own in the vocabulary; padding, id 0, behind them
    g = torch.Generator(device="cuda").manual_seed(int(seed) + 1)
    rank = (torch.exp(torch.rand(T, generator=g, device="cuda", dtype=torch.float64) * math.log(V)).long() - 1).clamp(0, V - 1)
    tokens = torch.randperm(V, generator=g, device="cuda")[rank]
    tokens[T - int(T * c["pad"]):] = 0
    return dict(c=c, tokens=tokens, w=r(V, H, std=0.02).requires_grad_(), dy=r(T, H), scale=math.sqrt(H))


# ---- one pass ----------------------------------------------------------------------------------


def run(st):
    kind = st["c"]["kind"]
    if own:
        return {"attn": _attention_own, "norm": _norm_own, "embed": _embedding_own}[kind](st)
    with torch.no_grad():
        return {"attn": _attention_plain, "norm": _norm_plain, "embed": _embedding_plain}[kind](st)


def _attention_own(st):
    from lightron_b200.ops import functional as OF
    c, q, k, v = st["c"], st["q"], st["k"], st["v"]
    # (a model makes the mask once per batch, for all of its layers)
    mask = None if st["documents"] is None else OF.attention_mask(documents=st["documents"], causal=c["causal"])
    o = OF.masked_attention(q, k, v, mask=mask, causal=c["causal"], scale=st["scale"], softcap=c["cap"], slopes=st["slopes"], window=c["window"], sinks=c["sinks"])
    if st["do"] is None:
        return o
    return (o, *torch.autograd.grad(o, (q, k, v), st["do"]))


def _visible(st):
    """[B, 1, 1, Sq, S]: whether query i sees key j."""
    c = st["c"]
    j = torch.arange(c["S"], device="cuda")
    i = j[c["S"] - c["Sq"]:]
    away = i[:, None] - j[None, :]
    near = (away.abs() < c["window"])[None]
    if st["documents"] is None:
        see = near | (j < c["sinks"])
    else:
        ids = st["documents"]
        # place of every key in its document: how far behind the last change of ids
        fresh = torch.ones_like(ids, dtype=torch.bool)
        fresh[:, 1:] = ids[:, 1:] != ids[:, :-1]
        place = j - (j * fresh).cummax(dim=1).values
        see = (near | (place < c["sinks"])[:, None, :]) & (ids[:, c["S"] - c["Sq"]:, None] == ids[:, None, :]) & (ids[:, None, :] >= 0)
    if c["causal"]:
        see = see & (away >= 0)
    return see[:, None, None]


def _attention_plain(st):
    c = st["c"]
    rep = c["heads"] // c["kv"]
    q = st["q"].float().unflatten(2, (-1, rep)).permute(0, 2, 3, 1, 4)      # [B, kv, rep, Sq, d]
    k, v = (st[n].float().permute(0, 2, 1, 3)[:, :, None] for n in ("k", "v"))      # [B, kv, 1, S, d]
    s = (q @ k.transpose(-1, -2)).mul_(st["scale"])
    if c["cap"]:
        t = torch.tanh(s / c["cap"])
        s = c["cap"] * t
    if st["slopes"] is not None:
        j = torch.arange(c["S"], device="cuda", dtype=torch.float32)
        s -= st["slopes"].view(c["kv"], rep, 1, 1) * (j[c["S"] - c["Sq"]:, None] - j[None, :]).abs()
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


def _norm_own(st):
    from lightron_b200.ops import functional as OF
    if not st["c"]["grad"]:
        return OF.qk_norm_rope(st["q"], st["k"], st["wq"], st["wk"], st["cos"], st["sin"], positions=st["positions"], eps=EPS)
    leaves = tuple(st[n] for n in ("q", "k", "wq", "wk"))
    y = OF.qk_norm_rope(*leaves, st["cos"], st["sin"], positions=st["positions"], eps=EPS)
    return (*y, *torch.autograd.grad(y, leaves, (st["dq"], st["dk"])))


def _turned(x, cos, sin):
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack((a * cos - b * sin, a * sin + b * cos), dim=-1).flatten(-2)


def _norm_plain(st):
    S = st["c"]["S"]
    cos, sin = (t[:S][None] if st["positions"] is None else t[st["positions"].long()] for t in (st["cos"], st["sin"]))
    cos, sin = cos[:, :, None], sin[:, :, None]
    y, dx, dw = [], [], []
    for x, w, dy in ((st["q"], st["wq"], st.get("dq")), (st["k"], st["wk"], st.get("dk"))):
        x, w = x.float(), w.float()
        rstd = torch.rsqrt((x * x).mean(dim=-1, keepdim=True) + EPS)
        hat = x * rstd
        y.append(_turned(hat * w, cos, sin).to(BF16))
        if dy is not None:
            g = _turned(dy.float(), cos, -sin)
            dw.append((g * hat).sum(dim=(0, 1, 2)).to(BF16))
            g = g * w
            dx.append((rstd * (g - hat * (g * hat).mean(dim=-1, keepdim=True))).to(BF16))
    return (*y, *dx, *dw)


def _embedding_own(st):
    from lightron_b200.ops import functional as OF
    y = OF.scaled_embedding(st["tokens"], st["w"], st["scale"])
    return y, torch.autograd.grad(y, st["w"], st["dy"])[0]


def _embedding_plain(st):
    w = st["w"]
    y = (w[st["tokens"]].float() * st["scale"]).to(BF16)
    dw = torch.zeros(w.shape, device="cuda").index_add_(0, st["tokens"], st["dy"].float())
    return y, dw.mul_(st["scale"]).to(BF16)


# ---- what a pass cannot do without -------------------------------------------------------------


def _pairs(c):
    """Pairs of query and key that see each other, over all sequences."""
    n = 0
    for lens, _ in _documents(c):
        for s in lens:
            i = torch.arange(s - min(s, c["Sq"]), s)
            first = (i - c["window"] + 1).clamp_min(0)                       # of the window, and its last key
            last = i if not c["causal"] else i.clone()
            if not c["causal"]:
                last = (i + c["window"] - 1).clamp_max(s - 1)
            n += int((last - first + 1).sum()) + int(first.clamp_max(c["sinks"]).sum())
            if not c["causal"]:                                              # sinks behind the window
                n += int((min(c["sinks"], s) - last - 1).clamp_min(0).sum())
    return n


def work(c):
    if c["kind"] == "attn":
        queries, keys = c["B"] * c["Sq"], c["B"] * min(c["S"], c["Sq"] + c["window"] - 1 + c["sinks"] if c["causal"] else c["S"])
        once = (queries * 2 * c["heads"] + keys * 2 * c["kv"]) * c["d"] * 2                 # q, o, and the k, v that any query sees
        if c["grad"]:
            once *= 2                                                                       # do, dq, dk, dv
        return {"bytes": once, "flops": _pairs(c) * c["heads"] * c["d"] * (14 if c["grad"] else 4)}
    if c["kind"] == "norm":
        n = c["B"] * c["S"] * (c["heads"] + c["kv"]) * c["d"]
        return {"bytes": n * 2 * (5 if c["grad"] else 2) + c["S"] * c["d"] * 4, "flops": n * (20 if c["grad"] else 7)}
    T, V, H = c["T"], c["vocab"], c["dim"]
    return {"bytes": 2 * T * 8 + 3 * T * H * 2 + V * H * 2, "flops": 3 * T * H}


# ---- 64 bits -----------------------------------------------------------------------------------


def exact(c, seed):
    st = prepare(c, seed)
    return {"attn": _attention_exact, "norm": _norm_exact, "embed": _embedding_exact}[c["kind"]](c, st)


def _attention_exact(c, st):
    B, Sq, S, hq, hkv, d = c["B"], c["Sq"], c["S"], c["heads"], c["kv"], c["d"]
    f64 = dict(dtype=torch.float64, device="cuda")
    q, k, v = (st[n].detach().double() for n in ("q", "k", "v"))
    o = torch.zeros(B, Sq, hq, d, **f64)
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    for b in range(B):
        # documents one by one: a query's keys are those of its own document
        ids = st["documents"][b].tolist() if st["documents"] is not None else [0] * S
        edges = [i for i in range(S) if i == 0 or ids[i] != ids[i - 1]] + [S]
        for lo, hi in zip(edges[:-1], edges[1:]):
            if ids[lo] < 0:
                continue
            n, m = hi - lo, min(hi - lo, Sq)             # (with fewer queries than keys there is one document)
            col = torch.arange(n, device="cuda")
            row = col[n - m:]
            hide = torch.ones(m, n, dtype=torch.bool, device="cuda").tril(n - m - c["window"]) | torch.ones(m, n, dtype=torch.bool, device="cuda").triu(n - m + c["window"])
            hide[:, :c["sinks"]] = False
            if c["causal"]:
                hide |= col[None, :] > row[:, None]
            away = (row[:, None] - col[None, :]).abs().double()
            at = slice(lo, hi) if Sq == S else slice(0, Sq)
            for h in range(hq):
                g = h // (hq // hkv)
                x, y, z = (t[b, s, n_].clone().requires_grad_(c["grad"]) for t, s, n_ in ((q, at, h), (k, slice(lo, hi), g), (v, slice(lo, hi), g)))
                s = x @ y.t() * st["scale"]
                if c["cap"]:
                    s = c["cap"] * torch.tanh(s / c["cap"])
                if st["slopes"] is not None:
                    s = s - float(st["slopes"][h]) * away
                r = torch.softmax(s.masked_fill(hide, float("-inf")), dim=-1) @ z
                o[b, at, h] = r.detach()
                if c["grad"]:
                    gx, gy, gz = torch.autograd.grad(r, (x, y, z), st["do"][b, at, h].double())
                    dq[b, at, h] = gx
                    dk[b, lo:hi, g] += gy
                    dv[b, lo:hi, g] += gz
    return (o, dq, dk, dv) if c["grad"] else o


def _norm_exact(c, st):
    at = torch.arange(c["S"], device="cuda").expand(c["B"], -1) if st["positions"] is None else st["positions"].long()
    turn = torch.complex(st["cos"].double(), st["sin"].double())[at][:, :, None]
    leaves = [st[n].detach().double().requires_grad_(c["grad"]) for n in ("q", "k", "wq", "wk")]
    y = []
    for x, w in ((leaves[0], leaves[2]), (leaves[1], leaves[3])):
        z = x / (x.square().sum(dim=-1, keepdim=True) / c["d"] + EPS).sqrt() * w
        y.append(torch.view_as_real(torch.view_as_complex(z.unflatten(-1, (-1, 2))) * turn).flatten(-2))
    if not c["grad"]:
        return tuple(y)
    grads = torch.autograd.grad(y, leaves, (st["dq"].double(), st["dk"].double()))
    return (*(t.detach() for t in y), *grads)


def _embedding_exact(c, st):
    order = torch.argsort(st["tokens"], stable=True)
    ids, counts = torch.unique_consecutive(st["tokens"][order], return_counts=True)
    sums = torch.segment_reduce(st["dy"][order].double(), "sum", lengths=counts, axis=0)
    dw = torch.zeros(c["vocab"], c["dim"], dtype=torch.float64, device="cuda")
    dw[ids] = sums * st["scale"]
    return torch.nn.functional.embedding(st["tokens"], st["w"].detach().double()) * st["scale"], dw
