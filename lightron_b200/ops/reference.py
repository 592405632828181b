"""Plain PyTorch restatement of every hot op.  It is (a) the numeric oracle that the CUDA
kernels are tested against, (b) the CPU / gloo execution path and (c) the "library" baseline.

Math follows the reference model: RMSNorm computed in fp32 then cast then scaled
(``layers/layers.py:11-16``), RoPE on interleaved pairs (``layers/layers.py:18-24,44-70``),
SwiGLU ``silu(w1 x) * w3 x`` (``model/model.py:69``), causal softmax attention with scale
1/sqrt(d) (``model/model.py:193-198``) and token-mean cross-entropy (``trainer.py:52``).
GQA is handled by indexing, not by materialising repeated KV (``model/model.py:11-34``).
"""
from __future__ import annotations

import math
from typing import Optional, Tuple

import torch
import torch.nn.functional as F


def rmsnorm(x: torch.Tensor, weight: torch.Tensor, eps: float) -> torch.Tensor:
    xf = x.float()
    y = xf * torch.rsqrt(xf.pow(2).mean(-1, keepdim=True) + eps)
    return y.type_as(x) * weight


def rope_tables(head_dim: int, end: int, theta: float = 10000.0,
                device=None) -> Tuple[torch.Tensor, torch.Tensor]:
    """cos/sin tables [end, head_dim/2] in fp32 (kept real so a dtype cast of the model cannot
    drop the imaginary part, which happens to the reference's complex buffer under bf16)."""
    freqs = 1.0 / (theta ** (torch.arange(0, head_dim, 2, device=device)[: head_dim // 2].float() / head_dim))
    t = torch.arange(end, device=device).float()
    ang = torch.outer(t, freqs)
    return torch.cos(ang), torch.sin(ang)


def rope(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
         positions: Optional[torch.Tensor] = None, inverse: bool = False) -> torch.Tensor:
    """x: [B, S, h, d]; rotates pairs (x[2i], x[2i+1]) by angle pos * theta^(-2i/d).
    ``positions`` [S] selects table rows (context parallel shards); default arange(S).
    ``inverse`` applies the transpose rotation (the backward of RoPE)."""
    B, S, h, d = x.shape
    if positions is None:
        c, s = cos[:S], sin[:S]
    else:
        c, s = cos[positions], sin[positions]
    c = c.view(1, S, 1, d // 2).float()
    s = s.view(1, S, 1, d // 2).float()
    if inverse:
        s = -s
    xf = x.float().reshape(B, S, h, d // 2, 2)
    x0, x1 = xf[..., 0], xf[..., 1]
    out = torch.stack((x0 * c - x1 * s, x0 * s + x1 * c), dim=-1)
    return out.reshape(B, S, h, d).type_as(x)


def swiglu(gate: torch.Tensor, up: torch.Tensor) -> torch.Tensor:
    return (F.silu(gate.float()) * up.float()).type_as(gate)


def swiglu_bwd(gate, up, dy):
    g, u, d = gate.float(), up.float(), dy.float()
    sig = torch.sigmoid(g)
    dgate = d * u * sig * (1 + g * (1 - sig))
    dup = d * g * sig
    return dgate.type_as(gate), dup.type_as(up)


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, causal: bool = True,
              scale: Optional[float] = None, q_pos: Optional[torch.Tensor] = None,
              k_pos: Optional[torch.Tensor] = None, return_lse: bool = False):
    """q: [B, Sq, hq, d]; k, v: [B, Sk, hkv, d] -> [B, Sq, hq, d].  fp32 math.
    With ``q_pos``/``k_pos`` (global positions) the causal mask is q_pos >= k_pos, which is what
    context-parallel shards need."""
    B, Sq, hq, d = q.shape
    Sk, hkv = k.shape[1], k.shape[2]
    rep = hq // hkv
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    qf = q.float().permute(0, 2, 1, 3).reshape(B, hkv, rep, Sq, d)
    kf = k.float().permute(0, 2, 1, 3)                      # [B, hkv, Sk, d]
    vf = v.float().permute(0, 2, 1, 3)
    s = torch.einsum("bgrqd,bgkd->bgrqk", qf, kf) * scale
    if causal:
        qp = torch.arange(Sq, device=q.device) + (Sk - Sq) if q_pos is None else q_pos
        kp = torch.arange(Sk, device=q.device) if k_pos is None else k_pos
        mask = qp[:, None] >= kp[None, :]
        s = s.masked_fill(~mask, float("-inf"))
    lse = torch.logsumexp(s, dim=-1)                         # [B, hkv, rep, Sq]
    p = torch.exp(s - lse.unsqueeze(-1))
    p = torch.nan_to_num(p, nan=0.0)                        # fully masked rows
    o = torch.einsum("bgrqk,bgkd->bgrqd", p, vf)
    o = o.reshape(B, hq, Sq, d).permute(0, 2, 1, 3).type_as(q)
    if return_lse:
        return o, lse.reshape(B, hq, Sq)
    return o


def mask_bounds(S: int, documents: Optional[torch.Tensor], prefix: Optional[torch.Tensor], causal: bool) -> Tuple[torch.Tensor, torch.Tensor]:
    """Intervals of ``functional.attention_mask``: keys [lo, hi) that a position sees, positions [lo, hi) that see a key, both [B, S, 2] int32.
    ``documents`` [B, S] ids or None, ``prefix`` [B, S] marks, [B] lengths or None."""
    B, dev = (documents if documents is not None else prefix).shape[0], (documents if documents is not None else prefix).device
    i = torch.arange(S, device=dev).expand(B, S)
    ids = documents if documents is not None else torch.zeros(B, S, dtype=torch.int32, device=dev)
    first = torch.ones(B, S, dtype=torch.bool, device=dev)
    first[:, 1:] = ids[:, 1:] != ids[:, :-1]
    start = torch.where(first, i, -1).cummax(dim=1).values
    after = torch.cat((torch.where(first, i, S)[:, 1:], torch.full((B, 1), S, device=dev)), dim=1)
    end = after.flip(1).cummin(dim=1).values.flip(1)
    if prefix is None:
        part = start
    else:
        marks = prefix.bool() if prefix.dim() == 2 else i < prefix[:, None]
        plain = torch.where(marks, S, i).flip(1).cummin(dim=1).values.flip(1)          # first position from here on that is not marked
        part = torch.minimum(plain.gather(1, start), end)
    hi = torch.maximum(i + 1, part) if causal else end
    q = torch.stack((start, hi), dim=-1)
    k = torch.stack((torch.where(i < part, start, i) if causal else start, end), dim=-1)
    pad = torch.stack((i, i), dim=-1)
    hide = (ids < 0)[..., None]
    return torch.where(hide, pad, q).int(), torch.where(hide, pad, k).int()


def masked_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, bounds: Optional[torch.Tensor] = None, causal: bool = True,
                     scale: Optional[float] = None, softcap: float = 0.0, slopes: Optional[torch.Tensor] = None, window: Optional[int] = None, sinks: int = 0) -> torch.Tensor:
    """q [B, Sq, hq, d], k / v [B, Sk, hkv, d]; query i sits at position i + Sk - Sq and sees the keys of ``bounds`` [B, Sk, 2] there (None:
    all keys, with ``causal`` those up to its own); with ``window`` of those the ones less than ``window`` positions away, and the first ``sinks``.  Scores are ``softcap * tanh(x / softcap) - slopes[h] * distance``; fp32 math."""
    B, Sq, hq, d = q.shape
    Sk, hkv = k.shape[1], k.shape[2]
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    dt = torch.float64 if q.dtype == torch.float64 else torch.float32
    qf = q.to(dt).permute(0, 2, 1, 3).reshape(B, hkv, hq // hkv, Sq, d)
    kf, vf = k.to(dt).permute(0, 2, 1, 3), v.to(dt).permute(0, 2, 1, 3)
    s = torch.einsum("bgrqd,bgkd->bgrqk", qf, kf) * scale
    if softcap:
        s = softcap * torch.tanh(s / softcap)
    at, key = torch.arange(Sk - Sq, Sk, device=q.device), torch.arange(Sk, device=q.device)
    if slopes is not None:
        s = s - slopes.to(dt).view(hkv, hq // hkv, 1, 1) * (at[:, None] - key[None, :]).abs()
    if bounds is not None:
        row = bounds[:, Sk - Sq:].to(q.device)
        see = ((key >= row[..., :1]) & (key < row[..., 1:]))[:, None, None]
    else:
        see = (key[None, :] <= at[:, None]) if causal else torch.ones(Sq, Sk, dtype=torch.bool, device=q.device)
        see = see[None, None, None]
    if window is not None:
        near = (at[:, None] - key[None, :]).abs() < window
        first = bounds[:, Sk - Sq:].to(q.device)[..., :1][:, None, None] if bounds is not None else 0
        see = see & (near | (key < first + sinks))
    s = s.masked_fill(~see, float("-inf"))
    top = s.amax(dim=-1, keepdim=True).detach() if Sk else s.new_zeros(*s.shape[:-1], 1)
    e = torch.exp(s - torch.where(top == float("-inf"), torch.zeros_like(top), top))
    total = e.sum(dim=-1, keepdim=True)
    p = e / torch.where(total == 0, torch.ones_like(total), total)                       # rows that see nothing: zero
    o = torch.einsum("bgrqk,bgkd->bgrqd", p, vf)
    return o.reshape(B, hq, Sq, d).permute(0, 2, 1, 3).to(q.dtype)


def rope_axes(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, positions: torch.Tensor, axes, inverse: bool = False) -> torch.Tensor:
    """x [B, S, h, d]; pair i turns by the table row ``positions[axes[i]]`` ([A, B, S] or [A, S]) of its token, and is NaN where there is none."""
    axis, pair = torch.as_tensor(axes, device=x.device), torch.arange(x.shape[-1] // 2, device=x.device)
    at = positions.long()[axis]                                                          # [d/2, (B,) S]
    at = (at if at.dim() == 3 else at[:, None]).permute(1, 2, 0)
    away, at = (at < 0) | (at >= cos.shape[0]), at.clamp(0, max(cos.shape[0] - 1, 0))    # (an index outside of the table would be refused, or on a GPU end the process)
    c, s = (t[at, pair].masked_fill(away, float("nan"))[:, :, None] for t in (cos, sin))
    s = -s if inverse else s
    a, b = x.to(c.dtype)[..., 0::2], x.to(c.dtype)[..., 1::2]
    return torch.stack((a * c - b * s, a * s + b * c), dim=-1).flatten(-2).type_as(x)


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, q_weight: torch.Tensor, k_weight: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, positions: torch.Tensor, axes,
                 eps: float) -> Tuple[torch.Tensor, torch.Tensor]:
    """Heads of q [B, S, hq, d] and k [B, S, hkv, d] normed, times their weights, and turned as by :func:`rope_axes`; rounded once."""
    dt = torch.float64 if q.dtype == torch.float64 else torch.float32
    out = []
    for x, w in ((q, q_weight), (k, k_weight)):
        xf = x.to(dt)
        out.append(rope_axes(xf * torch.rsqrt(xf.pow(2).mean(-1, keepdim=True) + eps) * w.to(dt), cos.to(dt), sin.to(dt), positions, axes).type_as(x))
    return out[0], out[1]


def scaled_embedding(tokens: torch.Tensor, w: torch.Tensor, scale: float, vocab_start: int = 0) -> torch.Tensor:
    """``scale`` times rows of ``w``, rounded once; ids outside of [vocab_start, vocab_start + w.shape[0]) give zero rows.  The gradient is summed up in 32 bits at least."""
    dt = torch.float64 if w.dtype == torch.float64 else torch.float32
    local = tokens.long() - vocab_start
    away = (local < 0) | (local >= w.shape[0])
    if w.shape[0] == 0:
        return w.new_zeros(*tokens.shape, w.shape[1])
    local = local.masked_fill(away, 0)
    # (the gradient is summed up in the type that rows are gathered in; without one only the rows are cast)
    rows = F.embedding(local, w.to(dt)) if w.requires_grad and torch.is_grad_enabled() else F.embedding(local, w).to(dt)
    return (rows * scale).masked_fill(away.unsqueeze(-1), 0.0).type_as(w)


def grad_sumsq(tensors) -> torch.Tensor:
    """Sum of the squares of all elements of all tensors, fp32."""
    parts = [t.detach().float().square().sum() for t in tensors]
    return torch.stack(parts).sum() if parts else torch.zeros(())


def cross_entropy(logits: torch.Tensor, targets: torch.Tensor, ignore_index: int = -100) -> torch.Tensor:
    """Token-mean NLL over [T, V] logits (fp32 math)."""
    return F.cross_entropy(logits.float(), targets, reduction="mean", ignore_index=ignore_index)


def adamw_step(p, g, m, v, lr, beta1, beta2, eps, wd, step):
    """One decoupled-weight-decay Adam update in fp32 (torch.optim.AdamW semantics)."""
    g = g.float()
    p.mul_(1 - lr * wd)
    m.mul_(beta1).add_(g, alpha=1 - beta1)
    v.mul_(beta2).addcmul_(g, g, value=1 - beta2)
    bc1 = 1 - beta1 ** step
    bc2 = 1 - beta2 ** step
    denom = (v.sqrt() / math.sqrt(bc2)).add_(eps)
    p.addcdiv_(m, denom, value=-lr / bc1)
