"""Packed batches for the tests, and attention, rotation and clipping restated in 64 bits from their definitions, position by position."""
import random

import torch


def visible(B, Sq, Sk, causal, ids=None, marks=None):
    """[B, Sq, Sk] bool from the definition: same run of equal ids, no padding, up to the own position or in the document's marked start."""
    see = torch.zeros(B, Sq, Sk, dtype=torch.bool)
    for b in range(B):
        row = [0] * Sk if ids is None else ids[b].tolist()
        run, n = [], 0
        for j in range(Sk):
            n += j > 0 and row[j] != row[j - 1]
            run.append(n)
        lead, open_ = [False] * Sk, False
        for j in range(Sk):
            if j == 0 or run[j] != run[j - 1]:
                open_ = True
            open_ = open_ and marks is not None and bool(marks[b][j])
            lead[j] = open_
        for i in range(Sq):
            at = i + Sk - Sq
            if row[at] < 0:
                continue
            for j in range(Sk):
                see[b, i, j] = run[j] == run[at] and (not causal or j <= at or lead[j])
    return see


def documents(B, S, mean, seed, pad=True):
    """[B, S] int32 ids: documents of random lengths, padding between some of them and at the end."""
    rng = random.Random(seed)
    ids = torch.full((B, S), -1, dtype=torch.int32)
    for b in range(B):
        at, n = 0, 0
        while at < S:
            m = min(S - at, rng.randint(1, 2 * mean))
            if not (pad and rng.random() < 0.2):
                ids[b, at:at + m] = n
            n += 1
            at += m
    return ids


def attention64(q, k, v, see, scale, cap=0.0, slopes=None, do=None):
    """o, and with ``do`` (o, dq, dk, dv), in 64 bits."""
    q, k, v = (t.detach().double().requires_grad_(do is not None) for t in (q, k, v))
    Sq, Sk, rep = q.shape[1], k.shape[1], q.shape[2] // k.shape[2]
    kk, vv = (t.repeat_interleave(rep, 2).transpose(1, 2) for t in (k, v))
    s = q.transpose(1, 2) @ kk.transpose(-1, -2) * scale
    if cap:
        s = cap * torch.tanh(s / cap)
    if slopes is not None:
        i, j = torch.arange(Sq, device=q.device) + Sk - Sq, torch.arange(Sk, device=q.device)
        s = s - slopes.double().view(-1, 1, 1) * (i[:, None] - j[None, :]).abs()
    see = see.to(q.device)[:, None]
    s = s.masked_fill(~see, -1e300)
    p = s.softmax(-1) * see                    # (rows that see nothing: zero)
    o = (p @ vv).transpose(1, 2)
    if do is None:
        return o
    return (o.detach(), *torch.autograd.grad(o, (q, k, v), do.double()))


def rel(got, want):
    return ((got.double() - want.double()).norm() / want.double().norm().clamp_min(1e-30)).item()
