"""Kernels of packed batches against 64 bits: attention under interval masks with caps and biases, rotary positions with axes, norm and clipping.

Bounds, derived as in the edge tests of the other kernels: a bf16 result is one rounding (2^-9 / sqrt(3) = 1.1e-3 in the 2-norm) of fp32 sums; P and
dS enter a product in bf16, which adds as much again: 5e-3 covers both with room.  Sums of squares in fp32: 1e-6; scaled fp32 values: two roundings, 2^-23.
"""
import ctypes

import pytest
import torch

from packed_oracle import attention64, documents, rel, visible

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def _rand(*shape, scale=1.0, seed=0, dtype=BF16):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32) * scale).to(dtype)


def _status_ok():
    from lightron_b200.ops import native
    assert native.device_status() == {}


def _mask(B, Sk, causal, docs, prefix, seed=0):
    """(mask, ids, marks)"""
    from lightron_b200.ops import functional as OF
    ids = documents(B, Sk, docs, seed) if docs else None
    marks = torch.rand(B, Sk, generator=torch.Generator().manual_seed(seed)) < 0.9 if prefix else None
    if ids is None and marks is None:
        return None, None, None
    return OF.attention_mask(documents=None if ids is None else ids.cuda(), prefix=None if marks is None else marks.cuda(), causal=causal), ids, marks


def _run(q, k, v, do, **kw):
    from lightron_b200.ops import functional as OF
    q, k, v = (t.detach().requires_grad_() for t in (q, k, v))
    o = OF.masked_attention(q, k, v, **kw)
    return (o.detach(), *torch.autograd.grad(o, (q, k, v), do))


@pytest.mark.parametrize("S", [1, 2, 31, 1000, 1024, 1025, 5000, 40001, 327680])
@pytest.mark.parametrize("docs,prefix,causal", [(3, "none", True), (700, "marks", True), (0, "marks", True), (0, "lengths", True), (40, "none", False), (40, "lengths", True)])
def test_intervals(S, docs, prefix, causal):
    from lightron_b200.ops import functional as OF
    from lightron_b200.ops import reference as ref
    B = 3
    ids = documents(B, S, docs, seed=S) if docs else None
    mark = {"none": None, "marks": torch.rand(B, S, generator=torch.Generator().manual_seed(S)) < 0.95, "lengths": torch.tensor([0, S // 3, S])}[prefix]
    for wide in (torch.int32, torch.int64):
        mask = OF.attention_mask(documents=None if ids is None else ids.cuda().to(wide), prefix=None if mark is None else mark.cuda(), causal=causal, length=S)
        want = ref.mask_bounds(S, ids, mark, causal)
        assert torch.equal(mask.q_bounds.cpu(), want[0]) and torch.equal(mask.k_bounds.cpu(), want[1])


@pytest.mark.parametrize("d", [64, 128, 96, 8])
@pytest.mark.parametrize("B,Sq,Sk,hq,hkv,causal,docs,prefix,cap,alibi,scale", [
    (2, 1, 1, 2, 1, True, 0, False, 0.0, False, 1.0),            # one token
    (1, 2, 2, 1, 1, True, 0, False, 20.0, True, 1.0),
    (2, 128, 128, 4, 2, True, 0, False, 0.0, True, 1.0),         # one tile
    (2, 129, 129, 4, 4, True, 30, False, 0.0, False, 1.0),       # one row over, documents that end inside tiles, padding
    (1, 300, 300, 2, 1, False, 70, False, 30.0, False, 2.0),     # both ways
    (1, 257, 257, 8, 1, True, 0, True, 0.0, False, 1.0),         # one long prefix
    (2, 384, 384, 2, 2, True, 90, True, 50.0, True, 2.0),        # everything
    (1, 100, 400, 4, 2, True, 0, False, 30.0, True, 1.0),        # the last queries of a longer sequence
    (2, 1, 333, 4, 1, True, 50, True, 0.0, True, 1.0),           # a single query
    (1, 130, 260, 2, 1, False, 100, False, 0.0, True, 1.0),
    (1, 700, 700, 4, 1, True, 0, False, 0.0, False, 8.0),        # large scores: the running maximum moves
    (1, 640, 640, 2, 1, True, 0, False, 5.0, False, 8.0),        # most scores at the cap
    (1, 640, 640, 2, 1, False, 0, False, 200.0, True, 8.0),      # a cap that lets exponentials overflow without a maximum
    (17, 200, 200, 8, 4, True, 64, False, 0.0, False, 1.0),      # many short sequences
])
def test_attention(B, Sq, Sk, hq, hkv, causal, docs, prefix, cap, alibi, scale, d):
    q, k, v, do = _rand(B, Sq, hq, d, scale=scale, seed=1), _rand(B, Sk, hkv, d, seed=2), _rand(B, Sk, hkv, d, seed=3), _rand(B, Sq, hq, d, seed=4)
    mask, ids, marks = _mask(B, Sk, causal, docs, prefix, seed=5)
    slopes = 2.0 ** -torch.arange(1, hq + 1, device="cuda", dtype=torch.float32) if alibi else None
    got = _run(q, k, v, do, mask=mask, causal=causal, softcap=cap, slopes=slopes)
    _status_ok()
    see = visible(B, Sq, Sk, causal, ids, marks)
    want = attention64(q, k, v, see, d ** -0.5, cap, slopes, do)
    for name, g, w in zip(("o", "dq", "dk", "dv"), got, want):
        assert torch.isfinite(g).all(), name
        if w.norm() > 1e-6 * do.double().norm():                 # (where every row sees one key, dq and dk vanish)
            assert rel(g, w) < 5e-3, name
        else:
            assert g.double().norm() < 1e-4 * do.double().norm(), name
    empty = ~see.any(-1).cuda()
    assert (got[0][empty] == 0).all() and (got[1][empty] == 0).all()
    unseen = ~see.any(1).cuda()
    assert (got[2][unseen] == 0).all() and (got[3][unseen] == 0).all()


@pytest.mark.parametrize("cap,alibi", [(0.0, False), (25.0, True)])
def test_gradients_against_differences(cap, alibi):
    B, S, hq, hkv, d = 1, 200, 4, 2, 64
    q, k, v, do = _rand(B, S, hq, d, seed=1), _rand(B, S, hkv, d, seed=2), _rand(B, S, hkv, d, seed=3), _rand(B, S, hq, d, seed=4)
    mask, ids, marks = _mask(B, S, True, 60, True, seed=6)
    slopes = 2.0 ** -torch.arange(1, hq + 1, device="cuda", dtype=torch.float32) if alibi else None
    got = _run(q, k, v, do, mask=mask, softcap=cap, slopes=slopes)[1:]
    see, eps = visible(B, S, S, True, ids, marks), 1e-4
    for i, name in enumerate("qkv"):
        x = [q.double(), k.double(), v.double()]
        # along the gradient itself: the difference quotient is its squared norm
        u = got[i].double()
        f = []
        for sign in (1, -1):
            y = list(x)
            y[i] = x[i] + sign * eps * u
            f.append((attention64(*y, see, d ** -0.5, cap, slopes) * do.double()).sum())
        assert abs(((f[0] - f[1]) / (2 * eps) / u.square().sum()).item() - 1) < 5e-3, name


@pytest.mark.parametrize("d", [64, 128, 40])
@pytest.mark.parametrize("B,Sq,Sk,hq,hkv,causal,docs,prefix,cap,alibi,scale", [
    (1, 1, 2300, 2, 1, True, 0, False, 0.0, False, 4.0),         # one query over many keys
    (3, 1, 1030, 4, 2, True, 200, False, 30.0, True, 2.0),
    (1, 70, 2300, 2, 2, True, 0, False, 0.0, True, 4.0),
    (1, 1300, 1300, 2, 1, True, 0, False, 0.0, False, 8.0),      # tiles of which some shares hold nothing
    (1, 1300, 1300, 1, 1, True, 150, True, 50.0, False, 4.0),
    (1, 1100, 1100, 2, 1, False, 400, False, 200.0, True, 4.0),
    (2, 1025, 1025, 2, 2, True, 300, False, 0.0, False, 2.0),    # padding: rows that no share sees
])
def test_attention_split_over_keys(B, Sq, Sk, hq, hkv, causal, docs, prefix, cap, alibi, scale, d):
    """Few tiles: their key blocks are shared between CTAs and the parts joined."""
    from lightron_b200.ops import native
    assert native.require().lb_masked_attn_fwd_ws_bytes(B, Sq, Sk, hq, hkv, d) > 0
    test_attention(B, Sq, Sk, hq, hkv, causal, docs, prefix, cap, alibi, scale, d)


@pytest.mark.parametrize("cap", [0.0, 20.0, 200.0])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("S,d", [(300, 64), (500, 128)])
def test_attention_slopes(S, d, causal, cap):
    """From no slope to slopes that leave a row its own key alone, with scores that are large enough for far keys to count."""
    slopes = torch.tensor([0.0, 0.01, 1.3, 1.4, 5.0, 100.0], device="cuda")
    q, k, v, do = _rand(1, S, 6, d, scale=6.0, seed=1), _rand(1, S, 2, d, seed=2), _rand(1, S, 2, d, seed=3), _rand(1, S, 6, d, seed=4)
    got = _run(q, k, v, do, causal=causal, softcap=cap, slopes=slopes)
    _status_ok()
    for name, g, w in zip(("o", "dq", "dk", "dv"), got, attention64(q, k, v, visible(1, S, S, causal), d ** -0.5, cap, slopes, do)):
        assert torch.isfinite(g).all() and rel(g, w) < 5e-3, name


@pytest.mark.parametrize("B,S,hq,hkv,d", [(1, 500, 8, 1, 64), (6, 300, 8, 4, 128)])
def test_attention_repeats_its_bits(B, S, hq, hkv, d):
    """o, dk and dv are summed in a fixed order, also where a key block's walk is cut into parts (the first); so is dq up to 128 keys."""
    q, k, v, do = _rand(B, S, hq, d, seed=1), _rand(B, S, hkv, d, seed=2), _rand(B, S, hkv, d, seed=3), _rand(B, S, hq, d, seed=4)
    mask, _, _ = _mask(B, S, True, 90, False, seed=1)
    first = _run(q, k, v, do, mask=mask, softcap=30.0)
    for _ in range(3):
        again = _run(q, k, v, do, mask=mask, softcap=30.0)
        assert torch.equal(first[0], again[0]) and torch.equal(first[2], again[2]) and torch.equal(first[3], again[3])
    short = [t[:, :120] for t in (q, k, v, do)]
    assert torch.equal(_run(*short)[1], _run(*short)[1])


def test_attention_strides():
    """Heads ahead of tokens, a fused projection's columns, every other token, an expanded gradient: the same bits as contiguous copies."""
    B, S, hq, hkv, d = 2, 150, 4, 2, 64
    qkv = _rand(B, S, (hq + 2 * hkv) * d, seed=1)
    q, k, v = (t.unflatten(2, (-1, d)) for t in qkv.split([hq * d, hkv * d, hkv * d], dim=2))
    do = _rand(B, S, hq, d, seed=2)
    want = _run(q.contiguous(), k.contiguous(), v.contiguous(), do)
    kt = k.transpose(1, 2).contiguous().transpose(1, 2)
    vt = torch.empty(B, 2 * S, hkv, d, dtype=BF16, device="cuda")[:, ::2].copy_(v)
    odd = torch.empty(q.numel() + 1, dtype=BF16, device="cuda")[1:].view(q.shape).copy_(q)      # not aligned to 16 bytes
    for args in ((q, k, v, do), (odd, kt, vt, do), (q, kt, v, do.transpose(1, 2).contiguous().transpose(1, 2))):
        got = _run(*args)
        assert torch.equal(got[0], want[0]) and torch.equal(got[2], want[2]) and torch.equal(got[3], want[3])
        assert rel(got[1], want[1]) < 2e-3                       # (dq is added up as key tiles come)
    ones = torch.ones(1, device="cuda", dtype=BF16).expand(B, S, hq, d)
    assert rel(_run(q, k, v, ones)[3], _run(q, k, v, ones.contiguous())[3]) == 0.0
    _status_ok()


def test_hidden_scores_of_any_value():
    """Queries and keys whose masked scores are infinite or NaN: the visible ones are untouched."""
    B, S, h, d = 1, 256, 2, 64
    q, k, v, do = (_rand(B, S, h, d, seed=i) for i in range(4))
    ids = torch.zeros(B, S, dtype=torch.int32)
    ids[:, 100:] = 1
    from lightron_b200.ops import functional as OF
    mask = OF.attention_mask(documents=ids.cuda())
    big = k.clone()
    big[:, 100:] *= 1e18                                         # products up to 1e19: as a score of the first document's rows out of any range
    want = _run(q[:, :100], k[:, :100], v[:, :100], do[:, :100])
    got = _run(q, big, v, do, mask=mask)
    assert torch.isfinite(got[0]).all()
    assert rel(got[0][:, :100], want[0]) < 1e-6 and rel(got[3][:, :100], want[3]) < 2e-3


def test_one_sequence_against_the_causal_kernel():
    """No documents, cap or bias: what flash_attention computes."""
    from lightron_b200.ops import functional as OF
    q, k, v = _rand(2, 700, 8, 128, seed=1), _rand(2, 700, 2, 128, seed=2), _rand(2, 700, 2, 128, seed=3)
    assert rel(OF.masked_attention(q, k, v), OF.flash_attention(q, k, v, causal=True)) < 3e-3
    assert rel(OF.masked_attention(q, k, v, causal=False), OF.flash_attention(q, k, v, causal=False)) < 3e-3


def test_attention_on_another_stream_and_in_a_graph():
    from lightron_b200.ops import functional as OF
    q, k, v, do = (_rand(2, 333, 4, 64, seed=i) for i in range(4))
    ids = documents(2, 333, 80, seed=1).cuda()

    def step():
        mask = OF.attention_mask(documents=ids)
        return _run(q, k, v, do, mask=mask)
    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
        graph = torch.cuda.CUDAGraph()
    side.synchronize()
    with torch.cuda.graph(graph, stream=side):
        captured = step()
    graph.replay()
    torch.cuda.synchronize()
    for a, b, w in zip(other, captured, want):
        assert rel(a, w) < 2e-3 and rel(b, w) < 2e-3


def test_nodes_in_python_and_in_cpp(monkeypatch):
    """The autograd functions in Python and the C++ nodes: the same bits (dq beyond 128 keys: the same up to the order of its sums), the same version counts."""
    from lightron_b200.ops import functional as OF
    from lightron_b200.ops import native
    from lightron_b200.ops import reference as ref
    assert native.host_ops() is not None
    q, k, v, do = _rand(2, 100, 4, 64, seed=1), _rand(2, 120, 2, 64, seed=2), _rand(2, 120, 2, 64, seed=3), _rand(2, 100, 4, 64, seed=4)
    ids, slopes = documents(2, 120, 30, seed=1).cuda(), torch.rand(4, device="cuda")
    cos, sin = ref.rope_tables(64, 200, device="cuda")
    pos = torch.arange(100, device="cuda", dtype=torch.int32).expand(3, 100).contiguous()
    grads = [_rand(100, 33, seed=5), _rand(7, seed=6, dtype=torch.float32)]

    def everything():
        mask = OF.attention_mask(documents=ids)
        x = q.detach().requires_grad_()
        y = OF.rope_axes(x, cos, sin, pos, [0, 1, 2, 0] * 8)
        mine = [g.clone() for g in grads]
        before = [g._version for g in mine]
        norm = OF.clip_grad_norm(mine, 1.0)
        assert [g._version - n for g, n in zip(mine, before)] == [1, 1]
        with torch.no_grad():
            alone = OF.masked_attention(q, k, v, mask=mask, softcap=20.0)
        return [mask.q_bounds, mask.k_bounds, *_run(q, k, v, do, mask=mask, softcap=20.0, slopes=slopes), alone, y, *torch.autograd.grad(y, x, do), OF.grad_norm(grads), norm, *mine]
    fast = everything()
    monkeypatch.setattr(native, "_HOST", None)
    for a, b in zip(fast, everything()):
        assert torch.equal(a, b)


def test_saved_tensors_that_come_back_otherwise():
    from lightron_b200.ops import functional as OF
    q = _rand(1, 50, 2, 64).requires_grad_()
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.clone(), lambda t: t):            # copies are fine
        o = OF.masked_attention(q, q, q)
    o.sum().backward()
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t[:, :10], lambda t: t):
        o = OF.masked_attention(q, q, q)
    with pytest.raises(RuntimeError):
        o.sum().backward()


def test_attention_refusals_on_the_gpu():
    from lightron_b200.ops import functional as OF
    q = _rand(1, 8, 2, 136)
    with pytest.raises(ValueError):
        OF.masked_attention(q, q, q)                             # heads wider than 128
    q = _rand(1, 8, 2, 20)
    with pytest.raises(ValueError):
        OF.masked_attention(q, q, q)                             # not a multiple of 8
    with pytest.raises(ValueError):
        OF.attention_mask(documents=torch.zeros(1, 327681, dtype=torch.int32, device="cuda"))
    q = _rand(1, 8, 2, 64)
    cpu = OF.attention_mask(documents=torch.zeros(1, 8, dtype=torch.int32))
    with pytest.raises(ValueError):
        OF.masked_attention(q, q, q, mask=cpu)
    with pytest.raises(ValueError):
        OF.masked_attention(q, q.cpu(), q)


@pytest.mark.parametrize("kw", [{}, dict(attn_softcap=5.0, attn_alibi=True), dict(rope_sections=(8, 12, 12))])
def test_packed_model(kw):
    """Documents packed into one sequence against each alone, and the fused projection's node against its parts: logits, loss, gradients."""
    from lightron_b200 import mesh
    from lightron_b200.config import ModelArgs
    from lightron_b200.models import LightronTransformer, init_weights
    from lightron_b200.ops import functional as OF
    mesh.set_context(None)
    args = ModelArgs(dim=256, n_layers=2, n_heads=4, n_kv_heads=2, vocab_size=512, intermediate_size=384, max_seq_len=512, **kw)
    model = LightronTransformer(args, dtype=BF16, device="cuda")
    init_weights(model, 0, std=0.05)
    lens = [130, 70, 256, 44]
    tokens = torch.randint(0, 512, (1, sum(lens)), device="cuda", generator=torch.Generator(device="cuda").manual_seed(0))
    ids = torch.cat([torch.full((n,), i) for i, n in enumerate(lens)])[None].cuda()
    pos = torch.cat([torch.arange(n) for n in lens])[None].cuda()
    if "rope_sections" in kw:
        pos = torch.stack([pos, pos // 16, pos % 16])
    mask = OF.attention_mask(documents=ids)
    packed = model(tokens, positions=pos, mask=mask)
    with torch.no_grad():
        assert torch.equal(packed, model(tokens, positions=pos, mask=mask))
        at = 0
        for n in lens:
            assert rel(packed[:, at:at + n], model(tokens[:, at:at + n], positions=pos[..., at:at + n])) < 1e-2      # (GEMMs of other sizes round otherwise)
            at += n
    model.loss(tokens, tokens.roll(-1, 1), positions=pos, mask=mask).backward()
    norm = OF.clip_grad_norm([p.grad for p in model.parameters()], 1e-3)
    assert 0 < norm.item() < 1e4
    assert abs(OF.grad_norm([p.grad for p in model.parameters()]).item() / 1e-3 - 1) < 1e-2
    _status_ok()


def test_fused_projection_node_against_its_parts():
    from lightron_b200.ops import functional as OF
    from lightron_b200.ops import reference as ref
    B, S, hq, hkv, d = 2, 150, 4, 2, 64
    qkv, do = _rand(B * S, (hq + 2 * hkv) * d, seed=1), _rand(B * S, hq * d, seed=2)
    cos, sin = ref.rope_tables(d, 200, device="cuda")
    pos = torch.randint(0, 200, (3, B, S), device="cuda", dtype=torch.int32)
    axes = [0] * 10 + [1] * 11 + [2] * 11
    mask, slopes = OF.attention_mask(documents=documents(B, S, 40, 3).cuda()), torch.rand(hq, device="cuda")
    x = qkv.clone().requires_grad_()
    o = OF.packed_attention_qkv(x * 1, cos, sin, pos, B, S, hq, hkv, d, axes=axes, mask=mask, softcap=20.0, slopes=slopes)
    dx, = torch.autograd.grad(o, x, do)
    y = qkv.clone().requires_grad_()
    q, k, v = (t.unflatten(1, (-1, d)).unflatten(0, (B, S)) for t in y.split([hq * d, hkv * d, hkv * d], dim=1))
    w = OF.masked_attention(OF.rope_axes(q, cos, sin, pos, axes), OF.rope_axes(k, cos, sin, pos, axes), v, mask=mask, softcap=20.0, slopes=slopes)
    dy, = torch.autograd.grad(w, y, do.view_as(w))
    assert torch.equal(o.view_as(w), w)
    assert rel(dx, dy) < 4e-3                                    # (dq is rounded before it is turned back, in both; it is added up as key tiles come)


# ---- rotary positions -------------------------------------------------------------------------------


@pytest.mark.parametrize("B,S,h,d", [(1, 1, 1, 8), (2, 7, 3, 64), (3, 130, 5, 128), (1, 300, 40, 96), (2, 33, 2, 80), (1, 20, 9, 256), (1, 4099, 2, 32)])
@pytest.mark.parametrize("per_batch", [True, False])
def test_rope_axes(B, S, h, d, per_batch):
    from lightron_b200.ops import functional as OF
    from lightron_b200.ops import reference as ref
    cos, sin = ref.rope_tables(d, 512, device="cuda")
    g = torch.Generator().manual_seed(S)
    pos = torch.randint(0, 512, (3, B, S) if per_batch else (3, S), generator=g).cuda()
    axes = torch.randint(0, 3, (d // 2,), generator=g).tolist()
    x = _rand(B, S, h + 1, d, seed=1)[:, :, 1:].detach().requires_grad_()      # heads of a wider row
    dy = _rand(B, S, h, d, seed=2)
    y = OF.rope_axes(x, cos, sin, pos, axes)
    dx, = torch.autograd.grad(y, x, dy)
    want = ref.rope_axes(x.detach().double(), cos.double(), sin.double(), pos, axes)
    back = ref.rope_axes(dy.double(), cos.double(), sin.double(), pos, axes, inverse=True)
    for got, w in ((y, want), (dx, back)):
        assert ((got.double() - w).abs() <= 2.0 ** -8 * w.abs() + 1e-5).all()  # one rounding, and that of the fp32 sum


def test_rope_axes_positions_outside_the_tables():
    from lightron_b200.ops import functional as OF
    from lightron_b200.ops import reference as ref
    cos, sin = ref.rope_tables(16, 10, device="cuda")
    pos = torch.tensor([[0, 9, 10, -1]] * 2, device="cuda")
    y = OF.rope_axes(_rand(1, 4, 2, 16), cos, sin, pos, [0, 1] * 4)
    assert torch.isfinite(y[:, :2]).all() and torch.isnan(y[:, 2:]).all()


# ---- norm and clipping ------------------------------------------------------------------------------


def _tensors(sizes, dtypes, seed=0):
    return [_rand(*s, seed=seed + i, dtype=dtypes[i % len(dtypes)]) for i, s in enumerate(sizes)]


SIZES = [[(1,)], [(7,), (0,), (3, 5)], [(16384,), (16385,), (1,), (40000,)], [(1000, 333), (5,)] * 3, [(3,)] * 900, [(2048, 1500)]]


@pytest.mark.parametrize("sizes", SIZES, ids=range(len(SIZES)))
@pytest.mark.parametrize("dtypes", [(BF16,), (torch.float32,), (torch.float16,), (BF16, torch.float32, torch.float16)], ids=["bf16", "fp32", "fp16", "mixed"])
def test_norm_and_clip(sizes, dtypes):
    from lightron_b200.ops import functional as OF
    ts = _tensors(sizes, dtypes)
    want = sum(t.double().square().sum() for t in ts).sqrt().item()
    norm = OF.grad_norm(ts)
    assert norm.dtype == torch.float32 and norm.dim() == 0 and abs(norm.item() / want - 1) < 1e-6
    assert torch.equal(norm, OF.grad_norm(ts))                                 # the same bits
    flat = {t: torch.empty(sum(x.numel() for x in ts if x.dtype == t) + 1, dtype=t, device="cuda") for t in dtypes}
    at, out = {t: 1 for t in dtypes}, []
    for x in ts:                                                               # outputs of no alignment
        out.append(flat[x.dtype][at[x.dtype]:at[x.dtype] + x.numel()].view(x.shape))
        at[x.dtype] += x.numel()
    by = min(1.0, 0.5 / (want + 1e-6))
    assert torch.equal(OF.clip_grad_norm(ts, 0.5, out=out), norm)
    eps = {BF16: 2.0 ** -8, torch.float16: 2.0 ** -10, torch.float32: 2.0 ** -22}
    for t, o in zip(ts, out):
        assert ((o.double() - t.double() * by).abs() <= eps[t.dtype] * (t.double() * by).abs() + 1e-7).all()
    inplace = [t.clone() for t in ts]
    OF.clip_grad_norm(inplace, 0.5)
    assert all(torch.equal(a, b) for a, b in zip(inplace, out))
    OF.clip_grad_norm(inplace, 1.0)                                            # below the limit
    assert all(torch.equal(a, b) for a, b in zip(inplace, out))


def test_clip_views_and_orders():
    from lightron_b200.ops import functional as OF
    base = _rand(300, 200, seed=1, dtype=torch.float32)
    ts = [base.clone()[:, 3:77], base.clone().t(), base.clone()[::2], base.clone()]
    want = sum(t.double().square().sum() for t in ts).sqrt().item()
    expect = [t.double() / (want + 1e-6) for t in ts]
    outs = [torch.empty_like(t) for t in ts[:3]] + [torch.empty(200, 300, device="cuda").t()]
    OF.clip_grad_norm(ts, 1.0, out=outs)
    norm = OF.clip_grad_norm(ts, 1.0)
    assert abs(norm.item() / want - 1) < 1e-6
    for t, o, e in zip(ts, outs, expect):
        assert torch.equal(t, o) and ((t.double() - e).abs() <= 2.0 ** -22 * e.abs() + 1e-9).all()


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_norms_that_are_not_finite(bad):
    from lightron_b200.ops import functional as OF
    ts = [torch.ones(100, device="cuda"), torch.ones(50, device="cuda", dtype=BF16)]
    ts[0][3] = bad
    norm = OF.clip_grad_norm(ts, 1.0)
    if bad != bad:
        assert torch.isnan(norm) and torch.isnan(ts[0]).all() and torch.isnan(ts[1]).all()
    else:
        assert torch.isinf(norm) and torch.isnan(ts[0][3]) and (ts[1] == 0).all()


def test_clip_refusals_of_the_library():
    """What the entry points themselves refuse, with nothing launched."""
    from lightron_b200.ops import native
    lib = native.require()
    t = torch.ones(4, device="cuda")
    one = (ctypes.c_void_p * 1)(t.data_ptr())
    filled = ctypes.c_int(0)
    for n, count, kind, room in ((-1, 4, 2, 9999), (1, -4, 2, 9999), (1, 4, 3, 9999), (1, 4, 2, 0)):
        rc = lib.lb_grad_squares(n, one, (ctypes.c_longlong * 1)(count), (ctypes.c_int * 1)(kind), t.data_ptr(), room, ctypes.byref(filled), native.stream_ptr())
        assert rc < 0
