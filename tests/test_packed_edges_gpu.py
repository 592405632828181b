"""Operators of packed batches where they can go wrong: biases that rise with distance, caps near zero, heads in several groups, scores out of range,
two streams, arguments that are written to, lists that change meanwhile.

Bounds as in the tests of the same kernels beside this file: 5e-3 in the 2-norm for attention (one rounding to bf16 of the result, of P and of dS: 1.7e-3 each, with
room); 1e-6 for norms.  A bias of up to 4000 in units of log2 rounds exponents by 2^-13 at most, which leaves the bound as it is.
"""
import threading

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


def _run(q, k, v, do, **kw):
    from lightron_b200.ops import functional as OF
    q, k, v = (t.detach().requires_grad_() for t in (q, k, v))
    o = OF.masked_attention(q, k, v, **kw)
    return (o.detach(), *torch.autograd.grad(o, (q, k, v), do))


def _see(Sq, Sk, causal):
    at, key = torch.arange(Sk - Sq, Sk, device="cuda"), torch.arange(Sk, device="cuda")
    return (key[None, :] <= at[:, None] if causal else torch.ones(Sq, Sk, dtype=torch.bool, device="cuda"))[None]


def _close(got, want, bound=5e-3):
    for name, g, w in zip(("o", "dq", "dk", "dv"), got, want):
        assert torch.isfinite(g).all(), name
        assert rel(g, w) < bound, (name, rel(g, w))


def _norm64(ts):
    return sum(t.double().square().sum() for t in ts).sqrt().item()


def test_norm_of_views_that_are_not_dense():
    """Their copies live until the sums are made: beside lists that take many rounds of the CTAs, and more than one launch."""
    from lightron_b200.ops import functional as OF
    base = _rand(120, 90, seed=1, dtype=torch.float32)
    views = [base[:, 3:77], base[::2], base.t()[5:50, ::3]]
    large = _rand(60_000_000, seed=2)
    many = [_rand(40, seed=i) for i in range(800)]
    for ts in (views, [large] + views, many + views, views + many + [large] + views):
        want = _norm64(ts)
        first = OF.grad_norm(ts)
        assert abs(first.item() / want - 1) < 1e-6
        assert all(torch.equal(OF.grad_norm(ts), first) for _ in range(3))


def test_rope_axes_outside_the_tables_in_the_form_for_other_types():
    """fp32, odd head sizes and more than eight axes are rotated by PyTorch operations: NaN there, too, and no access."""
    from lightron_b200.ops import functional as OF
    from lightron_b200.ops import reference as ref
    for d, axes, dtype in ((16, 2, torch.float32), (12, 2, BF16), (32, 9, BF16)):
        cos, sin = ref.rope_tables(d, 10, device="cuda")
        pos = torch.tensor([[0, 9, 10, -1]] * axes, device="cuda", dtype=torch.int32)
        y = OF.rope_axes(_rand(1, 4, 2, d, dtype=dtype), cos, sin, pos, [i % axes for i in range(d // 2)])
        assert torch.isfinite(y[:, :2]).all() and torch.isnan(y[:, 2:]).all()


def test_list_that_changes_meanwhile():
    """Another thread empties and refills the list while it is clipped: each call sees one whole list."""
    from lightron_b200.ops import functional as OF
    grads = [torch.ones(100 + i, device="cuda") for i in range(60)]
    total = sum(t.numel() for t in grads) ** 0.5
    box, stop = list(grads), threading.Event()

    def turn():
        while not stop.is_set():
            box[:] = [t.clone() for t in grads]
    side = threading.Thread(target=turn)
    side.start()
    try:
        for _ in range(300):
            assert abs(OF.grad_norm(box).item() / total - 1) < 1e-6
            assert abs(OF.clip_grad_norm(box, 1e9).item() / total - 1) < 1e-6
    finally:
        stop.set()
        side.join()
    torch.cuda.synchronize()


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two GPUs in one process")
def test_second_device_of_a_process():
    from lightron_b200.ops import functional as OF
    outs = []
    for dev in ("cuda:0", "cuda:1"):
        q, k, v, do = (_rand(2, 700, 4, 64, seed=i).to(dev) for i in range(4))
        ids = documents(2, 700, 150, seed=1).to(dev)
        outs.append([t.cpu() for t in _run(q, k, v, do, mask=OF.attention_mask(documents=ids), softcap=20.0)])
    assert all(torch.equal(outs[0][i], outs[1][i]) for i in (0, 2, 3))


RISING = [-0.01, -0.3, -1.3, -1.4, -5.0, 0.25]


@pytest.mark.parametrize("cap", [0.0, 20.0, 200.0])
@pytest.mark.parametrize("Sq,Sk,d,causal,docs,prefix", [
    (300, 300, 64, True, 0, False),
    (500, 500, 128, False, 0, False),
    (700, 700, 96, True, 0, False),
    (640, 640, 64, True, 200, True),          # documents with prefixes, padding
    (100, 400, 128, True, 0, False),          # the last queries of a longer sequence
    (1, 2300, 64, True, 0, False),            # split over keys
    (70, 1100, 128, False, 400, False),
])
def test_slopes_below_zero(Sq, Sk, d, causal, docs, prefix, cap):
    """Scores that rise with distance: the formula holds for every sign."""
    from lightron_b200.ops import functional as OF
    hq, hkv = 6, 2
    q, k, v, do = _rand(1, Sq, hq, d, scale=4.0, seed=1), _rand(1, Sk, hkv, d, seed=2), _rand(1, Sk, hkv, d, seed=3), _rand(1, Sq, hq, d, seed=4)
    mask, see = None, _see(Sq, Sk, causal)
    if docs:
        ids = documents(1, Sk, docs, seed=7)
        marks = torch.rand(1, Sk, generator=torch.Generator().manual_seed(7)) < 0.95 if prefix else None
        mask = OF.attention_mask(documents=ids.cuda(), prefix=None if marks is None else marks.cuda(), causal=causal)
        see = visible(1, Sq, Sk, causal, ids, marks)
    slopes = torch.tensor(RISING, device="cuda")
    got = _run(q, k, v, do, mask=mask, causal=causal, softcap=cap, slopes=slopes)
    with torch.no_grad():
        alone = OF.masked_attention(q, k, v, mask=mask, causal=causal, softcap=cap, slopes=slopes)
    _status_ok()
    want = attention64(q, k, v, see, d ** -0.5, cap, slopes, do)
    _close(got, want)
    assert rel(alone, want[0]) < 5e-3


def test_text_counts_on_all_axes():
    """Positions of one dimension, or none, on several axes: the bits of the same positions written out for each."""
    from lightron_b200.ops import functional as OF
    from lightron_b200.ops import reference as ref
    B, S, hq, hkv, d = 2, 150, 4, 2, 64
    qkv, do = _rand(B * S, (hq + 2 * hkv) * d, seed=1), _rand(B * S, hq * d, seed=2)
    cos, sin = ref.rope_tables(d, 200, device="cuda")
    axes = [0] * 10 + [1] * 11 + [2] * 11

    def both(pos, **kw):
        x = qkv.clone().requires_grad_()
        o = OF.packed_attention_qkv(x * 1, cos, sin, pos, B, S, hq, hkv, d, **kw)
        return o.detach(), torch.autograd.grad(o, x, do)[0]
    text = torch.arange(S, device="cuda", dtype=torch.int32)
    want = both(text.expand(3, B, S).contiguous(), axes=axes)
    for got in (both(None, axes=axes), both(text, axes=axes), both(text.long(), axes=axes), both(text.expand(3, S), axes=axes), both(None)):
        assert torch.equal(got[0], want[0]) and rel(got[1], want[1]) < 2e-3         # (dq is added up as key tiles come)


def _packed(B=1, S=40, hq=2, hkv=1, d=64):
    from lightron_b200.ops import functional as OF
    from lightron_b200.ops import reference as ref
    cos, sin = ref.rope_tables(d, 64, device="cuda")
    return _rand(B * S, (hq + 2 * hkv) * d, seed=1), lambda t: OF.packed_attention_qkv(t, cos, sin, None, B, S, hq, hkv, d)


def test_packed_attention_counts_its_writing():
    """The rotation of q and k inside the argument is seen by whoever has saved it; a leaf that asks for a gradient is not written to."""
    qkv, call = _packed()
    x = qkv.clone()
    before = x._version
    call(x)
    assert x._version > before
    w = qkv.clone().requires_grad_()
    y = w * 1
    z = y * y                                                     # saves y
    call(y)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        z.sum().backward()
    leaf = qkv.clone().requires_grad_()
    first = call(leaf)
    assert torch.equal(leaf, qkv) and torch.equal(call(leaf), first)
    grad, = torch.autograd.grad(first.float().sum(), leaf)
    other = qkv.clone().requires_grad_()
    assert torch.equal(grad[:, 3 * 64:], torch.autograd.grad(call(other * 1).float().sum(), other)[0][:, 3 * 64:])      # dv: the same bits


def test_packed_attention_without_gradients():
    qkv, call = _packed()
    want = call(qkv.clone())
    with torch.no_grad():
        assert torch.equal(call(qkv.clone()), want)
    with torch.inference_mode():
        assert torch.equal(call(qkv.clone()), want)


def test_clip_by_the_norm_of_others():
    """``counted``: pieces of the tensors, none, and pieces that are not dense."""
    from lightron_b200.ops import functional as OF
    ts = [_rand(3000, seed=1, dtype=torch.float32), _rand(40, 70, seed=2)]
    for counted in ([ts[0][5:1000], ts[0][2000:]], [ts[1][:, 3:50]], []):
        own = [t.clone() for t in ts]
        norm = OF.clip_grad_norm(own, 0.5, counted=counted)
        assert torch.equal(norm, OF.grad_norm(counted).to(norm.device))
        by = min(1.0, 0.5 / (norm.item() + 1e-6))
        for t, o, e in zip(ts, own, (2.0 ** -22, 2.0 ** -8)):
            assert ((o.double() - t.double() * by).abs() <= e * (t.double() * by).abs()).all()


def test_clip_refuses_memory_that_overlaps():
    """Two entries that share memory would be scaled once or twice, as it comes: refused, with nothing written."""
    from lightron_b200.ops import functional as OF
    a = torch.ones(100, device="cuda")
    b = torch.ones(50, device="cuda")
    buf = torch.zeros(200, device="cuda")
    for ts, out in (([a, b, a], None), ([a[:60], a[40:]], None), ([a, b], [buf[:100], buf[60:110]]), ([a[:50], a[50:]], [a[50:], a[:50]]), ([a[:99], b], [a[1:], buf[:50]])):
        with pytest.raises(ValueError):
            OF.clip_grad_norm(ts, 1e-3, out=out)
    assert (a == 1).all() and (b == 1).all() and (buf == 0).all()
    # neighbours, and the same list as its own result, are not that
    OF.clip_grad_norm([a[:50], a[50:], b, a[:0], a[:0]], 1.0)
    OF.clip_grad_norm([a, b], 1.0, out=[a, b])
    assert abs(_norm64([a, b]) - 1) < 1e-5


def test_gradients_that_are_missing_are_refused():
    from lightron_b200.ops import functional as OF
    for ts in ([torch.ones(3, device="cuda"), None], [None]):
        with pytest.raises(ValueError):
            OF.grad_norm(ts)
        with pytest.raises(ValueError):
            OF.clip_grad_norm(ts, 1.0)


def test_a_rank_that_holds_nothing_takes_part(monkeypatch):
    """An empty list has no device: its zero is added where the group's backend works."""
    import torch.distributed as dist
    from lightron_b200.ops import functional as OF
    seen = []
    monkeypatch.setattr(dist, "get_world_size", lambda g=None: 2)
    monkeypatch.setattr(dist, "get_backend", lambda g=None: "nccl")
    monkeypatch.setattr(dist, "all_reduce", lambda t, group=None: seen.append(t.device.type) or t.add_(9.0))
    for call in (OF.grad_norm, lambda ts, group: OF.clip_grad_norm(ts, 1.0, group=group)):
        assert call([], group="others").item() == 3.0
    assert seen == ["cuda", "cuda"]


def test_whole_numbers_beyond_32_bits():
    """Positions past the tables, prefix lengths past the sequence: as such, not what their low 32 bits say."""
    from lightron_b200.ops import functional as OF
    from lightron_b200.ops import reference as ref
    cos, sin = ref.rope_tables(16, 10, device="cuda")
    pos = torch.tensor([[0, 9, 2 ** 32 + 1, -2 ** 32]] * 2, device="cuda")
    y = OF.rope_axes(_rand(1, 4, 2, 16), cos, sin, pos, [0, 1] * 4)
    assert torch.isfinite(y[:, :2]).all() and torch.isnan(y[:, 2:]).all()
    lens = torch.tensor([2 ** 32, -2 ** 32 + 3, 2], device="cuda")
    mask = OF.attention_mask(prefix=lens, length=5)
    want = ref.mask_bounds(5, None, lens.cpu(), True)
    assert torch.equal(mask.q_bounds.cpu(), want[0]) and torch.equal(mask.k_bounds.cpu(), want[1])


@pytest.mark.parametrize("cap", [1e-6, 1e-9, 1e-20])
@pytest.mark.parametrize("d", [64, 128])
def test_caps_near_zero(d, cap):
    """Scores of exactly zero beside others that are all at the cap."""
    S = 256
    q, k, v, do = _rand(1, S, 2, d, seed=1), _rand(1, S, 1, d, seed=2), _rand(1, S, 1, d, seed=3), _rand(1, S, 2, d, seed=4)
    q[:, :128] = 0
    got = _run(q, k, v, do, softcap=cap)
    _status_ok()
    _close(got, attention64(q, k, v, _see(S, S, True), d ** -0.5, cap, None, do))


def test_rope_axes_tables_of_any_alignment():
    from lightron_b200.ops import functional as OF
    from lightron_b200.ops import reference as ref
    cos, sin = ref.rope_tables(64, 50, device="cuda")
    flat = torch.empty(2 * cos.numel() + 1, device="cuda")
    c, s = flat[1:1 + cos.numel()].view(cos.shape).copy_(cos), flat[1 + cos.numel():].view(cos.shape).copy_(sin)
    assert c.data_ptr() % 16 and c.is_contiguous()
    pos = torch.arange(20, device="cuda", dtype=torch.int32).expand(2, 20).contiguous()
    x = _rand(1, 20, 3, 64)
    assert torch.equal(OF.rope_axes(x, c, s, pos, [0, 1] * 16), OF.rope_axes(x, cos, sin, pos, [0, 1] * 16))


@pytest.mark.parametrize("cap,alibi", [(0.0, False), (0.0, True), (30.0, False), (200.0, True)])
def test_hidden_scores_out_of_range(cap, alibi):
    """Finite queries and keys of two documents whose scores across them pass fp32: infinite, and NaN where infinities meet.  Both documents as if alone."""
    from lightron_b200.ops import functional as OF
    S, cut, h, d = 256, 100, 2, 64
    q, k, v, do = (_rand(1, S, h, d, seed=i) for i in range(1, 5))
    up = torch.ones(S, 1, 1, device="cuda")
    up[:cut], up[cut:] = 2.0 ** 60, 2.0 ** -100
    q, k = (q.float() * up).to(BF16), (k.float() / up).to(BF16)
    ids = torch.zeros(1, S, dtype=torch.int32, device="cuda")
    ids[:, cut:] = 1
    slopes = torch.tensor([0.1, 0.02], device="cuda") if alibi else None
    got = _run(q, k, v, do, mask=OF.attention_mask(documents=ids), softcap=cap, slopes=slopes)
    _status_ok()
    for part in (slice(0, cut), slice(cut, S)):
        n = part.stop - part.start
        want = attention64(q[:, part], k[:, part], v[:, part], _see(n, n, True), d ** -0.5, cap, slopes, do[:, part])
        _close([g[:, part] for g in got], want)


def test_heads_in_several_groups_forward():
    """K and V of more heads than are kept in L2 together: groups of 4, 4 and 2 of ten heads."""
    from lightron_b200.ops import functional as OF
    from lightron_b200.ops import native
    Sq, Sk, h, d = 2000, 40960, 10, 64
    assert native.require().lb_masked_attn_fwd_ws_bytes(1, Sq, Sk, h, h, d) == 0          # (not split)
    q, k, v = _rand(1, Sq, h, d, seed=1), _rand(1, Sk, h, d, seed=2), _rand(1, Sk, h, d, seed=3)
    with torch.no_grad():
        o = OF.masked_attention(q, k, v)
    _status_ok()
    see = _see(Sq, Sk, True)
    for i in range(h):
        w = attention64(*(t[:, :, i:i + 1] for t in (q, k, v)), see, d ** -0.5)
        assert rel(o[:, :, i:i + 1], w) < 5e-3, i


def test_heads_in_several_groups_backward():
    """236 pairs of batch and key head in groups of 32, the last one smaller."""
    B, S, h, d = 59, 400, 4, 64
    q, k, v, do = (_rand(B, S, h, d, seed=i) for i in range(1, 5))
    got = _run(q, k, v, do)
    _status_ok()
    _close(got, attention64(q, k, v, _see(S, S, True), d ** -0.5, 0.0, None, do))


def test_two_streams_at_a_time():
    from lightron_b200.ops import functional as OF

    def work(i):
        q, k, v, do = (_rand(2, 700, 4, 64, seed=10 * i + j) for j in range(4))
        grads = [_rand(300 + i, 77, seed=i), _rand(5000, seed=i, dtype=torch.float32)]
        ids = documents(2, 700, 150, seed=i).cuda()
        torch.cuda.synchronize()

        def step():
            mask = OF.attention_mask(documents=ids)
            out = _run(q, k, v, do, mask=mask, softcap=20.0)
            outs = [torch.empty_like(g) for g in grads]
            return [out[0], out[2], out[3], OF.clip_grad_norm(grads, 1.0, out=outs), *outs]
        return step
    steps = [work(1), work(2)]
    want = [s() for s in steps]
    streams = [torch.cuda.Stream() for _ in steps]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, (s, st) in enumerate(zip(steps, streams)):
            with torch.cuda.stream(st):
                got[i].append(s())
    torch.cuda.synchronize()
    _status_ok()
    for w, runs in zip(want, got):
        for g in runs:
            assert all(torch.equal(a, b) for a, b in zip(g, w))


@pytest.mark.parametrize("d", [64, 128])
def test_wide_caps(d):
    """Scores near 9000 of 20000 whose differences decide: tanh has to be as exact in every block, also where hidden scores beside the visible ones are larger.  (32 bits
    leave 2^-11 of such scores, and tanh by its definition 1.5e-7 caps, 3e-3 of a weight, at random over the keys: the bound stays.)"""
    from lightron_b200.ops import functional as OF
    S, cut, h = 256, 200, 2
    q, k, v, do = (_rand(1, S, h, d, seed=i) for i in range(1, 5))
    q[..., 0], k[:, :cut, :, 0], k[:, cut:, :, 0] = 256.0, 9000.0 * d ** 0.5 / 256.0, 80000.0
    ids = torch.zeros(1, S, dtype=torch.int32, device="cuda")
    ids[:, cut:] = 1
    got = _run(q, k, v, do, mask=OF.attention_mask(documents=ids), softcap=20000.0)
    _status_ok()
    want = attention64(q[:, :cut], k[:, :cut], v[:, :cut], _see(cut, cut, True), d ** -0.5, 20000.0, None, do[:, :cut])
    for name, g, w in zip(("o", "dq", "dk", "dv"), got, want):
        g, w = (t[:, :cut, :, 1:] if name in ("dq", "dk") else t[:, :cut] for t in (g, w[:, :cut] if w.shape[1] > cut else w))      # (the first column of dq and dk is a sum that all but cancels)
        assert rel(g, w) < 5e-3, (name, rel(g, w))


@pytest.mark.parametrize("cap", [30.0, 200.0])
@pytest.mark.parametrize("scale", [1e-12, 1e-6, 1e-3, 1e3, 1e6])
@pytest.mark.parametrize("d", [64, 128])
def test_scales_of_any_size(d, scale, cap):
    """Queries and keys that are as large or small as the scale asks for: scores with a standard deviation of 8."""
    S, h = 200, 2
    size = (8.0 / scale / d ** 0.5) ** 0.5
    q, k, v, do = _rand(1, S, h, d, scale=size, seed=1), _rand(1, S, h, d, scale=size, seed=2), _rand(1, S, h, d, seed=3), _rand(1, S, h, d, seed=4)
    got = _run(q, k, v, do, softcap=cap, scale=scale)
    _status_ok()
    _close(got, attention64(q, k, v, _see(S, S, True), scale, cap, None, do))


@pytest.mark.parametrize("d", [8, 24, 32, 40, 64, 72, 80, 96, 104, 128])
@pytest.mark.parametrize("B,S,hq,hkv,docs", [(2, 1300, 8, 2, 0), (3, 400, 4, 4, 60)])
def test_query_gradients_of_every_head_size(B, S, hq, hkv, docs, d):
    """dQ leaves in pieces of 32 columns, an odd or even number of them, through two places in turn."""
    from lightron_b200.ops import functional as OF
    q, k, v, do = _rand(B, S, hq, d, seed=1), _rand(B, S, hkv, d, seed=2), _rand(B, S, hkv, d, seed=3), _rand(B, S, hq, d, seed=4)
    mask, see = None, _see(S, S, True)
    if docs:
        ids = documents(B, S, docs, seed=7)
        mask = OF.attention_mask(documents=ids.cuda())
        at = torch.arange(S, device="cuda")
        see = (at >= mask.q_bounds[..., :1]) & (at < mask.q_bounds[..., 1:])
    want = attention64(q, k, v, see, d ** -0.5, 0.0, None, do)
    for _ in range(8):
        _close(_run(q, k, v, do, mask=mask), want)
    _status_ok()


def test_gradients_of_gradients_are_refused(monkeypatch):
    """With ``create_graph`` the gradients say that they cannot be differentiated again; as constants they would be left out of a sum's gradient."""
    from lightron_b200.ops import functional as OF
    from lightron_b200.ops import native
    from lightron_b200.ops import reference as ref
    cos, sin = ref.rope_tables(64, 64, device="cuda")
    pos = torch.arange(40, device="cuda", dtype=torch.int32)[None]
    q = _rand(1, 40, 2, 64, seed=1).requires_grad_()
    for host in (True, False):
        if not host:
            monkeypatch.setattr(native, "_HOST", None)
        for call in (lambda: OF.masked_attention(q, q, q), lambda: OF.rope_axes(q, cos, sin, pos, [0] * 32)):
            g, = torch.autograd.grad(call().float().square().sum(), q, create_graph=True)
            with pytest.raises(RuntimeError, match="differentiate twice"):
                (g.float().square().sum() + q.float().sum()).backward()
