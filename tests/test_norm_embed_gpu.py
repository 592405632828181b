"""Norms of queries and keys with the rotation, and the scaled embedding with its gradient by sorted tokens, against 64 bits.

Bounds.  A result is rounded once to bf16: at most 2^-8 of its value, so 2^-8 of the 2-norm.  What 32 bits leave before that: a head's sum of squares, two products and the rotation's sums are some
16 roundings of 2^-24 of values no larger than the head's norm, below 1e-5 of the 2-norm; sums over n terms add at most n 2^-24 of the terms' absolute sum.
"""
import math

import pytest
import torch

from local_oracle import embedding64, norm_rope64
from packed_oracle import rel

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16
HALF = 2.0 ** -8


def _rand(*shape, scale=1.0, seed=0, dtype=BF16):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32) * scale).to(dtype)


def _norm_case(B, S, hq, hkv, d, layout="apart", rows=None, seed=0):
    from lightron_b200.ops import reference as ref
    size = torch.exp(_rand(B, S, 1, 1, seed=seed + 9, dtype=torch.float32))
    if layout == "fused":                              # columns of a projection's output
        both = (_rand(B, S, hq + 2 * hkv, d, seed=seed) * size).to(BF16)
        q, k = both[:, :, :hq], both[:, :, hq:hq + hkv]
    elif layout == "heads first":
        q, k = ((_rand(B, h, S, d, seed=seed + i) * size.transpose(1, 2)).to(BF16).transpose(1, 2) for i, h in enumerate((hq, hkv)))
    elif layout == "askew":                            # not on 16 bytes: copied first
        q, k = ((_rand(B, S, h, d + 1, seed=seed + i) * size).to(BF16)[..., 1:] for i, h in enumerate((hq, hkv)))
    else:
        q, k = ((_rand(B, S, h, d, seed=seed + i) * size).to(BF16) for i, h in enumerate((hq, hkv)))
    wq, wk = ((1 + _rand(d, scale=0.3, seed=seed + 2 + i, dtype=torch.float32)).to(BF16) for i in range(2))
    cos, sin = ref.rope_tables(d, rows or S, device="cuda")
    return q, k, wq, wk, cos, sin


def _check_norm(q, k, wq, wk, cos, sin, positions=None, axes=None, eps=1e-6):
    from lightron_b200.ops import functional as OF
    B, S, hq, d = q.shape
    ins = [t.detach().requires_grad_() for t in (q, k, wq, wk)]
    before = [t.detach().clone() for t in ins]
    yq, yk = OF.qk_norm_rope(*ins, cos, sin, positions=positions, axes=axes, eps=eps)
    dq, dk = _rand(*yq.shape, seed=20), _rand(*yk.shape, seed=21)
    grads = torch.autograd.grad((yq, yk), ins, (dq, dk))
    with torch.no_grad():
        plain = OF.qk_norm_rope(*ins, cos, sin, positions=positions, axes=axes, eps=eps)
    assert torch.equal(plain[0], yq) and torch.equal(plain[1], yk)
    assert all(torch.equal(a, b) for a, b in zip(before, ins))
    at = torch.arange(S, device="cuda") if positions is None else positions
    if axes is None:
        at, axes = at.expand(B, S)[None], [0] * (d // 2)
    elif at.dim() == 1:
        at = at.expand(max(axes) + 1, B, S)
    elif at.dim() == 2:
        at = at[:, None].expand(-1, B, -1)
    exact = [t.detach().double().requires_grad_() for t in ins]
    e32 = torch.tensor(eps, dtype=torch.float32).item()
    zq, zk = norm_rope64(exact[0], exact[2], cos, sin, at, axes, e32), norm_rope64(exact[1], exact[3], cos, sin, at, axes, e32)
    want = torch.autograd.grad((zq, zk), exact, (dq.double(), dk.double()))
    for got, w, name in ((yq, zq, "yq"), (yk, zk, "yk"), (grads[0], want[0], "dq"), (grads[1], want[1], "dk")):
        assert got.dtype == BF16 and got.shape == w.shape
        assert rel(got.detach(), w.detach()) < HALF + 1e-4, (name, rel(got.detach(), w.detach()))
    for x, dy, got, w, name in ((exact[0], dq, grads[2], want[2], "dwq"), (exact[1], dk, grads[3], want[3], "dwk")):
        # terms of a sum: |g xhat| <= |dy of the pair| |xhat|
        n = x.shape[0] * x.shape[1] * x.shape[2]
        hat = (x / (x.square().mean(-1, keepdim=True) + e32).sqrt()).detach().abs()
        pair = dy.double().unflatten(-1, (-1, 2)).norm(dim=-1).repeat_interleave(2, -1)
        bound = HALF * w.abs() + (n + 32) * 2.0 ** -24 * (hat * pair).sum((0, 1, 2))
        assert ((got.double() - w).abs() <= bound).all(), name


@pytest.mark.parametrize("B,S,hq,hkv,d", [
    (1, 1, 1, 1, 64),
    (2, 5, 4, 2, 8),              # a head is one lane's
    (1, 3, 3, 1, 16),
    (2, 33, 6, 2, 32),
    (3, 70, 12, 12, 64),
    (2, 65, 32, 8, 128),
    (2, 17, 5, 1, 80),            # lanes without columns
    (1, 300, 16, 4, 96),
    (1, 9, 7, 3, 200),
    (2, 40, 3, 2, 256),           # a head is a warp's
    (8, 1, 64, 1, 128),           # one token in each sequence
    (1, 2500, 4, 1, 64),
])
def test_norm_rope(B, S, hq, hkv, d):
    _check_norm(*_norm_case(B, S, hq, hkv, d))


@pytest.mark.parametrize("layout", ["fused", "heads first", "askew"])
@pytest.mark.parametrize("d", [64, 96])
def test_norm_rope_layouts(layout, d):
    _check_norm(*_norm_case(2, 37, 6, 2, d, layout))


def test_norm_rope_positions():
    case = _norm_case(3, 21, 4, 2, 64, rows=400)
    g = torch.Generator().manual_seed(5)
    one, each = torch.randint(0, 400, (21,), generator=g).cuda(), torch.randint(0, 400, (3, 21), generator=g).cuda()
    axes = [0] * 10 + [1] * 11 + [2] * 11
    _check_norm(*case, positions=one)
    _check_norm(*case, positions=each.int())
    _check_norm(*case, positions=torch.randint(0, 400, (3, 3, 21), generator=g).cuda().int(), axes=axes)
    _check_norm(*case, positions=torch.randint(0, 400, (3, 21), generator=g).cuda().int(), axes=axes)
    _check_norm(*case, positions=one.int(), axes=axes)
    _check_norm(*case, axes=axes)
    _check_norm(*case, positions=torch.randint(0, 400, (21, 3), generator=g).cuda().int().t())           # tokens apart


def test_norm_rope_outside_the_tables():
    from lightron_b200.ops import functional as OF
    q, k, wq, wk, cos, sin = _norm_case(1, 4, 2, 1, 64, rows=10)
    pos = torch.tensor([0, 9, 10, -1], device="cuda", dtype=torch.int32)
    y = OF.qk_norm_rope(q, k, wq, wk, cos, sin, positions=pos)
    far = OF.qk_norm_rope(q, k, wq, wk, cos, sin, positions=torch.tensor([0, 9, 2 ** 32, -2 ** 32 + 1], device="cuda"))
    for a, b in zip(y, far):
        assert torch.isfinite(a[:, :2]).all() and torch.isnan(a[:, 2:]).all()
        assert torch.equal(a[:, :2], b[:, :2]) and torch.isnan(b[:, 2:]).all()
    # no positions: tokens past the table
    y = OF.qk_norm_rope(q, k, wq, wk, cos[:3], sin[:3])
    assert torch.isfinite(y[0][:, :3]).all() and torch.isnan(y[0][:, 3:]).all()


def test_norm_rope_of_zeros_and_large_heads():
    """A head of zeros stays zero with a gradient of dy w / sqrt(eps); with eps far below the heads' squares it has no part."""
    from lightron_b200.ops import functional as OF
    q, k, wq, wk, cos, sin = _norm_case(1, 6, 2, 1, 64)
    q = q.clone()
    q[0, 2] = 0
    leaf = q.detach().requires_grad_()
    yq, _ = OF.qk_norm_rope(leaf, k, wq, wk, cos, sin, eps=1e-2)
    assert (yq[0, 2] == 0).all()
    dy = _rand(*yq.shape, seed=3)
    dq, = torch.autograd.grad(yq, leaf, dy)
    from lightron_b200.ops import reference as ref
    back = ref.rope(dy.double(), cos.double(), sin.double(), inverse=True)[0, 2] * wq.double() / math.sqrt(1e-2)
    assert rel(dq[0, 2], back) < HALF + 1e-4
    _check_norm((q * 1e15).to(BF16) + 1, k, wq, wk, cos, sin)
    _check_norm(q, k, wq, wk, cos, sin, eps=1.0)


def test_norm_rope_same_bits_each_time():
    from lightron_b200.ops import functional as OF
    q, k, wq, wk, cos, sin = _norm_case(4, 700, 8, 2, 64)
    ins = [t.detach().requires_grad_() for t in (q, k, wq, wk)]
    runs = []
    for _ in range(3):
        y = OF.qk_norm_rope(*ins, cos, sin)
        runs.append((*y, *torch.autograd.grad(y, ins, [_rand(*t.shape, seed=4) for t in y])))
    assert all(torch.equal(a, b) for r in runs[1:] for a, b in zip(runs[0], r))


def test_python_nodes_are_the_same(monkeypatch):
    from lightron_b200.ops import functional as OF, native
    q, k, wq, wk, cos, sin = _norm_case(2, 30, 4, 2, 64)
    w, tokens = _rand(50, 64, seed=7), torch.randint(0, 60, (5, 20), generator=torch.Generator().manual_seed(1)).cuda()
    ins = [t.detach().requires_grad_() for t in (q, k, wq, wk, w)]

    def step(**kw):
        y = OF.qk_norm_rope(*ins[:4], cos, sin, **kw)
        e = OF.scaled_embedding(tokens, ins[4], 1.5, 3)
        return (*y, e, *torch.autograd.grad((*y, e), ins, (y[0].detach(), y[1].detach(), _rand(5, 20, 64, seed=9))))
    each = torch.randint(0, 30, (3, 2, 30), generator=torch.Generator().manual_seed(2)).cuda().int()
    axes = [0] * 10 + [1] * 11 + [2] * 11
    cases = [{}, dict(positions=each[0, 0]), dict(positions=each[0]), dict(positions=each, axes=axes), dict(positions=each[:, 0].contiguous(), axes=axes), dict(axes=axes),
             dict(positions=each[0, 0], axes=axes)]
    want = [step(**kw) for kw in cases]
    monkeypatch.setattr(native, "host_ops", lambda: None)
    for kw, e in zip(cases, want):
        assert all(torch.equal(a, b) for a, b in zip(step(**kw), e)), kw


def test_nodes_refuse_a_second_derivative():
    from lightron_b200.ops import functional as OF
    q, k, wq, wk, cos, sin = _norm_case(1, 3, 2, 1, 64)
    leaf, w = q.detach().requires_grad_(), _rand(5, 8).requires_grad_()
    for y, x in ((OF.qk_norm_rope(leaf, k, wq, wk, cos, sin)[0], leaf), (OF.scaled_embedding(torch.zeros(2, dtype=torch.long, device="cuda"), w), w)):
        g, = torch.autograd.grad(y.float().square().sum(), x, create_graph=True)
        with pytest.raises(RuntimeError):
            g.sum().backward()


def test_norm_rope_parts_of_the_gradients():
    """One output used, or weights without gradients."""
    from lightron_b200.ops import functional as OF
    q, k, wq, wk, cos, sin = _norm_case(2, 9, 4, 2, 64)
    ins = [t.detach().requires_grad_() for t in (q, k, wq, wk)]
    y = OF.qk_norm_rope(*ins, cos, sin)
    g = _rand(*y[0].shape, seed=4)
    full = torch.autograd.grad(y, ins, (g, torch.zeros_like(y[1])), retain_graph=True)
    part = torch.autograd.grad(y[0], ins, g, allow_unused=True)
    assert all(torch.equal(a, b) for a, b in zip(full[:1] + full[2:3], part[:1] + part[2:3])) and (part[1] == 0).all() and (part[3] == 0).all()
    y = OF.qk_norm_rope(ins[0], k, wq, wk, cos, sin)
    assert torch.equal(torch.autograd.grad(y[0], ins[0], g)[0], full[0])


# ---- embedding -----------------------------------------------------------------------------------


def _check_embedding(tokens, V, H, scale=1.0, start=0, w=None, dy=None):
    from lightron_b200.ops import functional as OF
    w = (_rand(V, H, seed=1) if w is None else w).detach().requires_grad_()
    y = OF.scaled_embedding(tokens, w, scale, start)
    dy = _rand(*tokens.shape, H, seed=2) if dy is None else dy
    dw, = torch.autograd.grad(y, w, dy)
    assert y.shape == (*tokens.shape, H) and dw.shape == w.shape
    with torch.no_grad():
        assert torch.equal(OF.scaled_embedding(tokens, w, scale, start), y)
    yw, dww = embedding64(tokens, w.detach(), scale, start, dy)
    assert ((y.double() - yw).abs() <= (HALF + 2.0 ** -23) * yw.abs()).all()
    _, size = embedding64(tokens, w.detach(), abs(scale), start, dy.abs())
    most = int(tokens.reshape(-1).unique(return_counts=True)[1].max())
    assert ((dw.double() - dww).abs() <= (HALF + 2.0 ** -23) * dww.abs() + (most + 4) * 2.0 ** -24 * size).all()
    return dw


@pytest.mark.parametrize("T,V,H", [
    (1, 1, 8), (1, 10, 64), (3, 5, 1), (7, 4, 2), (8, 100, 1021), (65, 30, 6), (300, 7, 264), (511, 2000, 2048), (700, 50, 4104), (2100, 900, 72), (5000, 64, 33),
    (4096, 3000, 16), (4097, 1023, 24), (4097, 1024, 7), (9000, 140000, 8), (8191, 2, 16), (20000, 1100000, 1), (16384, 32000, 8), (16385, 1000, 5), (16383, 70000, 3), (12000, 1, 9), (33000, 300, 2),
])
@pytest.mark.parametrize("wide", [True, False])
def test_embedding(T, V, H, wide):
    tokens = torch.randint(0, V, (T,), generator=torch.Generator().manual_seed(T)).cuda()
    _check_embedding(tokens if wide else tokens.int(), V, H, scale=math.sqrt(H))


def test_embedding_shapes_and_strides():
    tokens = torch.randint(0, 40, (6, 50), generator=torch.Generator().manual_seed(1)).cuda()
    _check_embedding(tokens, 40, 64)
    _check_embedding(tokens.t(), 40, 64, scale=-0.3)
    _check_embedding(tokens[:, ::2], 40, 64, scale=0.0)
    _check_embedding(tokens[0, 0], 40, 64)
    wide = _rand(40, 72, seed=8)
    _check_embedding(tokens, 40, 64, w=wide[:, :64])                    # rows apart
    _check_embedding(tokens, 40, 63, w=wide[:, 1:64])
    _check_embedding(tokens, 40, 64, dy=_rand(6, 50, 1, seed=3).expand(6, 50, 64))
    _check_embedding(tokens, 40, 64, w=_rand(64, 40, seed=8).t())
    flat = _rand(40 * 64 + 1, seed=5)
    _check_embedding(tokens, 40, 64, w=flat[1:].view(40, 64))          # rows of eight columns, not on 16 bytes


@pytest.mark.parametrize("T,top", [(1000, 1.0), (3000, 0.6), (9000, 0.95), (20000, 1.0)])
def test_embedding_of_one_id_often(T, top):
    """A row whose tokens fill many chunks, alone or between others."""
    g = torch.Generator().manual_seed(2)
    tokens = torch.randint(0, 300, (T,), generator=g)
    tokens[torch.rand(T, generator=g) < top] = 150
    _check_embedding(tokens.cuda(), 300, 40, scale=2.0)


def test_embedding_ids_outside():
    """A part of the vocabulary, ids of other ranks, below zero and beyond 32 bits: zero rows, no gradient; rows without tokens get zeros."""
    tokens = torch.tensor([[5, 99, 100, 131, 132, -1], [2 ** 40 + 110, -2 ** 35, 110, 110, 2 ** 32 + 110, 0]]).cuda()
    dw = _check_embedding(tokens, 32, 24, scale=3.0, start=100)
    assert (dw[1:10] == 0).all() and (dw[11:31] == 0).all() and (dw[31] != 0).any()
    away = torch.full((2000,), 500).cuda()
    assert (_check_embedding(away, 32, 24) == 0).all()
    away[1000:] = 3
    _check_embedding(away, 32, 24)


def test_embedding_many_rows_and_bits():
    """Rows beyond what ten bits, and three passes of ten, hold; most of them without a token."""
    from lightron_b200.ops import functional as OF
    g = torch.Generator().manual_seed(3)
    V, T = 40_000_000, 6000
    tokens = torch.randint(0, V, (T,), generator=g)
    tokens[::7] = V - 1
    tokens[3::7] = 0
    w = torch.zeros(V, 2, dtype=BF16, device="cuda").requires_grad_()
    dy = _rand(T, 2, seed=2)
    dw, = torch.autograd.grad(OF.scaled_embedding(tokens.cuda(), w, 3.0), w, dy)
    ids, back = tokens.unique(return_inverse=True)
    want = torch.zeros(ids.numel(), 2, dtype=torch.float64).index_add_(0, back, dy.double().cpu()) * 3.0
    size = torch.zeros(ids.numel(), 2, dtype=torch.float64).index_add_(0, back, dy.double().abs().cpu()) * 3.0
    assert ((dw[ids.cuda()].double().cpu() - want).abs() <= (HALF + 2.0 ** -23) * want.abs() + 1000 * 2.0 ** -24 * size).all()
    dw[ids.cuda()] = 0
    assert not dw.any()


def test_embedding_same_bits_each_time():
    from lightron_b200.ops import functional as OF
    tokens = (torch.rand(6000, generator=torch.Generator().manual_seed(1)) ** 3 * 500).long().cuda()
    w = _rand(500, 128, seed=1).requires_grad_()
    runs = [torch.autograd.grad(OF.scaled_embedding(tokens, w, 2.0), w, _rand(6000, 128, seed=2))[0] for _ in range(4)]
    assert all(torch.equal(runs[0], r) for r in runs)


def test_embedding_sums_in_32_bits():
    """A thousand small gradients on one row beside a large one: in the weight's type they would be lost."""
    tokens = torch.zeros(1025, dtype=torch.long, device="cuda")
    dy = torch.full((1025, 8), 2.0 ** -9, device="cuda", dtype=BF16)
    dy[0] = 1.0
    dw = _check_embedding(tokens, 1, 8, dy=dy)
    assert (dw == 3.0).all()


def test_embedding_without_tokens_or_rows():
    from lightron_b200.ops import functional as OF
    w = _rand(10, 8, seed=1).requires_grad_()
    y = OF.scaled_embedding(torch.zeros(0, 4, dtype=torch.long, device="cuda"), w, 2.0)
    assert y.shape == (0, 4, 8) and (torch.autograd.grad(y.sum(), w)[0] == 0).all()
    assert (OF.scaled_embedding(torch.zeros(3, dtype=torch.long, device="cuda"), w[:0]) == 0).all()


def test_non_finite_rows_stay_their_own():
    """Infinities and NaN in one row of weights or one gradient reach no other."""
    from lightron_b200.ops import functional as OF
    w = _rand(20, 16, seed=1)
    w[3], w[4] = float("inf"), float("nan")
    w.requires_grad_()
    tokens = torch.tensor([1, 3, 4, 2, 2], device="cuda")
    y = OF.scaled_embedding(tokens, w, 2.0)
    assert (y[1] == float("inf")).all() and torch.isnan(y[2]).all() and torch.isfinite(y[[0, 3, 4]]).all()
    dy = _rand(5, 16, seed=2)
    dy[0] = float("nan")
    dw, = torch.autograd.grad(y, w, dy)
    assert torch.isnan(dw[1]).all() and torch.isfinite(dw[2:]).all() and torch.isfinite(dw[0]).all()


# ---- graphs, streams ------------------------------------------------------------------------------


def test_captured_and_replayed():
    """Both operators with their backward in one graph, replayed on new inputs: what eager calls give."""
    from lightron_b200.ops import functional as OF
    q, k, wq, wk, cos, sin = _norm_case(2, 50, 4, 2, 64)
    w = _rand(300, 64, seed=7)
    tokens = torch.randint(0, 300, (600,), generator=torch.Generator().manual_seed(1)).cuda()
    ins = [t.detach().clone().requires_grad_() for t in (q, k, wq, wk, w)]
    dy = _rand(600, 64, seed=8)

    def step():
        y = OF.qk_norm_rope(*ins[:4], cos, sin)
        e = OF.scaled_embedding(tokens, ins[4], 1.5)
        return (*y, e, *torch.autograd.grad((*y, e), ins, (y[0].detach(), y[1].detach(), dy)))
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in (30, 31):
        with torch.no_grad():
            ins[0].copy_(_rand(*ins[0].shape, seed=seed))
            ins[4].copy_(_rand(300, 64, seed=seed))
            tokens.copy_(torch.randint(0, 300, (600,), generator=torch.Generator().manual_seed(seed)))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        assert all(torch.equal(a, b) for a, b in zip(got, step()))


def test_on_two_streams():
    from lightron_b200.ops import functional as OF
    q, k, wq, wk, cos, sin = _norm_case(4, 300, 8, 2, 64)
    w, dy = _rand(1000, 256, seed=7).requires_grad_(), _rand(4000, 256, seed=8)
    tokens = [torch.randint(0, 1000, (4000,), generator=torch.Generator().manual_seed(i)).cuda() for i in range(2)]
    want = [torch.autograd.grad(OF.scaled_embedding(t, w, 2.0), w, dy)[0] for t in tokens]
    y = OF.qk_norm_rope(q, k, wq, wk, cos, sin)
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], [[], []]
    for _ in range(5):
        for s, t, g in zip(streams, tokens, got):
            with torch.cuda.stream(s):
                g.append(torch.autograd.grad(OF.scaled_embedding(t, w, 2.0), w, dy)[0])
                g.append(OF.qk_norm_rope(q, k, wq, wk, cos, sin)[0])
    torch.cuda.synchronize()
    for g, e in zip(got, want):
        assert all(torch.equal(x, e) for x in g[::2]) and all(torch.equal(x, y[0]) for x in g[1::2])


# ---- refusals, hooks ------------------------------------------------------------------------------


def test_refusals_on_the_gpu():
    from lightron_b200.ops import functional as OF
    q, k, wq, wk, cos, sin = _norm_case(1, 4, 2, 1, 64)
    w, tokens = _rand(5, 8), torch.zeros(3, dtype=torch.long, device="cuda")
    for call in (lambda: OF.qk_norm_rope(q, k, wq.float(), wk, cos, sin), lambda: OF.qk_norm_rope(q, k, wq, wk.cpu(), cos, sin), lambda: OF.qk_norm_rope(q, k, wq, wk, cos.cpu(), sin.cpu()),
                 lambda: OF.qk_norm_rope(q, k.cpu(), wq, wk, cos, sin), lambda: OF.qk_norm_rope(q, k, wq, wk, cos, sin, eps=float("nan")),
                 lambda: OF.qk_norm_rope(q, k, wq, wk, cos, sin, positions=torch.zeros(4, dtype=torch.int32)), lambda: OF.qk_norm_rope(q, k[:, :3], wq, wk, cos, sin),
                 lambda: OF.scaled_embedding(tokens.cpu(), w), lambda: OF.scaled_embedding(tokens.to(torch.int16), w), lambda: OF.scaled_embedding(tokens, w, float("inf")),
                 lambda: OF.scaled_embedding(tokens, w, 1.0, -1), lambda: OF.scaled_embedding(tokens, w[0]),
                 lambda: OF.masked_attention(q, k, k, window=0), lambda: OF.masked_attention(q, k, k, window=2, sinks=-1), lambda: OF.masked_attention(q, k, k, sinks=2),
                 lambda: OF.masked_attention(q, k, k, window=True), lambda: OF.masked_attention(_rand(1, 4, 2, 136), _rand(1, 4, 2, 136), _rand(1, 4, 2, 136), window=2)):
        with pytest.raises(ValueError):
            call()


def test_sizes_past_31_bits_are_refused():
    """Views of one row, so that nothing of such a size is there."""
    from lightron_b200.ops import functional as OF
    q, k, wq, wk, cos, sin = _norm_case(1, 1, 1, 1, 8)
    w, tokens, most = _rand(1, 8), torch.zeros(3, dtype=torch.long, device="cuda"), 1 << 31
    for call in (lambda: OF.qk_norm_rope(q.expand(1, most, 1, 8), k.expand(1, most, 1, 8), wq, wk, cos, sin), lambda: OF.qk_norm_rope(q, k.expand(1, 1, most + 1, 8), wq, wk, cos, sin),
                 lambda: OF.scaled_embedding(tokens, w.expand(most, 8)), lambda: OF.scaled_embedding(tokens, w[:, :1].expand(1, most + 8)),
                 lambda: OF.scaled_embedding(tokens[:1].expand(most), w), lambda: OF.scaled_embedding(tokens, w, 1.0, (1 << 64) + 1)):
        with pytest.raises(ValueError):
            call()


def test_other_types_and_sizes_run_without_the_kernels():
    """fp32, fp16 and head sizes that the kernels do not take, by PyTorch operations."""
    from lightron_b200.ops import functional as OF
    from lightron_b200.ops import reference as ref
    for d, dtype, bound in ((64, torch.float32, 1e-5), (64, torch.float16, 2.0 ** -11 + 1e-5), (6, BF16, HALF + 1e-4), (264, BF16, HALF + 1e-4)):
        q, k, wq, wk = _rand(2, 5, 4, d, seed=1, dtype=dtype), _rand(2, 5, 2, d, seed=2, dtype=dtype), _rand(d, seed=3, dtype=dtype), _rand(d, seed=4, dtype=dtype)
        cos, sin = ref.rope_tables(d, 9, device="cuda")
        y = OF.qk_norm_rope(q, k, wq, wk, cos, sin)
        at = torch.arange(5, device="cuda").expand(1, 2, 5)
        for got, x, w in ((y[0], q, wq), (y[1], k, wk)):
            assert got.dtype == dtype and rel(got, norm_rope64(x.double(), w.double(), cos, sin, at, [0] * (d // 2), 1e-6)) < bound
    w = _rand(5, 8, dtype=torch.float32).requires_grad_()
    tokens = torch.tensor([1, 1, 4, 9], device="cuda")
    y = OF.scaled_embedding(tokens, w, 3.0)
    dw, = torch.autograd.grad(y.sum(), w)
    assert torch.equal(y, torch.cat((w.detach()[tokens[:3]] * 3, torch.zeros(1, 8, device="cuda")))) and dw[1].eq(6).all() and dw[4].eq(3).all() and dw[[0, 2, 3]].eq(0).all()


def test_saved_tensors_may_wait_on_the_cpu():
    from lightron_b200.ops import functional as OF
    q, k, wq, wk, cos, sin = _norm_case(2, 30, 4, 2, 64)
    v = _rand(2, 30, 2, 64, seed=6)
    w, tokens = _rand(50, 64, seed=7), torch.randint(0, 60, (300,), generator=torch.Generator().manual_seed(1)).cuda()
    ins = [t.detach().requires_grad_() for t in (q, k, wq, wk, v, w)]

    def step():
        tq, tk = OF.qk_norm_rope(*ins[:4], cos, sin)
        o = OF.masked_attention(tq, tk, ins[4], window=7, sinks=2)
        e = OF.scaled_embedding(tokens, ins[5], 1.5)
        return (o, e), lambda: torch.autograd.grad((o, e), ins, (_rand(*o.shape, seed=8), _rand(*e.shape, seed=9)))
    out, back = step()
    want = back()
    with torch.autograd.graph.save_on_cpu():
        other, back = step()
    got = back()
    assert all(torch.equal(a, b) for a, b in zip(out, other)) and all(torch.equal(a, b) for a, b in zip(got, want))


def test_arguments_written_to_are_noticed():
    """What backward needs is not what it was: an error, no other gradient."""
    from lightron_b200.ops import functional as OF
    q, k, wq, wk, cos, sin = _norm_case(1, 3, 2, 1, 64)
    leaf = q.detach().requires_grad_()
    x = leaf * 1
    y, _ = OF.qk_norm_rope(x, k, wq, wk, cos, sin)
    with torch.no_grad():
        x.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    tokens = torch.zeros(3, dtype=torch.long, device="cuda")
    w = _rand(5, 8).requires_grad_()
    e = OF.scaled_embedding(tokens, w)
    tokens.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        e.sum().backward()
