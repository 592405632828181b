"""Local attention, per-head norms and scaled embeddings for the tests, restated in 64 bits from their definitions."""
import torch


def local(B, Sq, Sk, causal, window, sinks, ids=None, marks=None):
    """[B, Sq, Sk] bool from the definition: same run of equal ids, no padding, up to the own position or in the document's marked start; and less than ``window`` positions away or among
    the first ``sinks`` places of the run."""
    ids = torch.zeros(B, Sk, dtype=torch.int32) if ids is None else ids.cpu()
    j = torch.arange(Sk)
    fresh = torch.ones(B, Sk, dtype=torch.bool)
    fresh[:, 1:] = ids[:, 1:] != ids[:, :-1]
    run = fresh.cumsum(1)
    place = j - (j * fresh).cummax(1).values
    at = j[Sk - Sq:]
    see = (run[:, Sk - Sq:, None] == run[:, None, :]) & (ids[:, None, :] >= 0)
    if causal:
        ahead = j[None, :] <= at[:, None]
        if marks is not None:
            open_ = (~marks.bool()).long().cumsum(1)               # places outside of the marks, up to each
            before = torch.where(place == 0, open_ - (~marks.bool()).long(), 0).cummax(1).values       # up to the document's start
            ahead = ahead[None] | (open_ == before)[:, None, :]
        see = see & ahead
    near = (at[:, None] - j[None, :]).abs() < window
    return see & (near[None] | (place < sinks)[:, None, :])


def norm_rope64(x, w, cos, sin, positions, axes, eps):
    """One tensor of heads [B, S, h, d], differentiable: complex numbers for the pairs; ``positions`` [A, B, S]."""
    z = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * w
    z = torch.view_as_complex(z.unflatten(-1, (-1, 2)).contiguous())
    turn = torch.stack([torch.complex(cos.double()[positions[a].long(), i], sin.double()[positions[a].long(), i]) for i, a in enumerate(axes)], dim=-1)
    return torch.view_as_real(z * turn[:, :, None]).flatten(-2)


def embedding64(tokens, w, scale, start, dy):
    """(y, dw), token by token."""
    V, H = w.shape
    flat, g = tokens.reshape(-1).tolist(), dy.reshape(-1, H).double()
    y, dw = torch.zeros(len(flat), H, dtype=torch.float64, device=w.device), torch.zeros(V, H, dtype=torch.float64, device=w.device)
    for t, i in enumerate(flat):
        if 0 <= i - start < V:
            y[t] = w[i - start].double() * scale
            dw[i - start] += g[t] * scale
    return y.view(*tokens.shape, H), dw
