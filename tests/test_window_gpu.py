"""Attention under a window with sinks on the GPU, against 64 bits.

Bounds as in the tests of the same kernels without a window: 5e-3 in the 2-norm (one rounding to bf16 of the result, of P and of dS: 1.7e-3 each, with room).
"""
import pytest
import torch

from local_oracle import local
from packed_oracle import attention64, documents, rel

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


def _close(got, want, bound=5e-3):
    for name, g, w in zip(("o", "dq", "dk", "dv"), got, want):
        assert torch.isfinite(g).all(), name
        assert rel(g, w) < bound, (name, rel(g, w))


def _inputs(B, Sq, Sk, hq, hkv, d, scale=1.0, seed=0):
    return (_rand(B, Sq, hq, d, scale=scale, seed=seed + 1), _rand(B, Sk, hkv, d, scale=scale, seed=seed + 2), _rand(B, Sk, hkv, d, seed=seed + 3), _rand(B, Sq, hq, d, seed=seed + 4))


def _check(B, Sq, Sk, hq, hkv, d, window, sinks, causal=True, docs=0, prefix=False, cap=0.0, slopes=None, scale=1.0, seed=0):
    from lightron_b200.ops import functional as OF
    q, k, v, do = _inputs(B, Sq, Sk, hq, hkv, d, scale, seed)
    ids = documents(B, Sk, docs, seed=seed + 7) if docs else None
    marks = torch.rand(B, Sk, generator=torch.Generator().manual_seed(seed)) < 0.97 if prefix else None
    mask = None
    if docs or prefix:
        mask = OF.attention_mask(documents=None if ids is None else ids.cuda(), prefix=None if marks is None else marks.cuda(), causal=causal)
    kw = dict(mask=mask, causal=causal, softcap=cap, slopes=None if slopes is None else torch.tensor(slopes, device="cuda"), window=window, sinks=sinks)
    got = _run(q, k, v, do, **kw)
    with torch.no_grad():
        alone = OF.masked_attention(q, k, v, **kw)
    _status_ok()
    see = local(B, Sq, Sk, causal, window, sinks, ids, marks)
    want = attention64(q, k, v, see, d ** -0.5, cap, kw["slopes"], do)
    _close(got, want)
    assert rel(alone, want[0]) < 5e-3
    empty = ~see.any(-1).cuda()
    assert (got[0][empty] == 0).all() and (got[1][empty] == 0).all()
    return got


@pytest.mark.parametrize("S", [2, 3, 17, 127, 128, 129, 255, 300, 513, 1000])
@pytest.mark.parametrize("window,sinks", [(2, 0), (2, 1), (64, 0), (127, 3), (128, 0), (129, 128), (130, 129), (200, 4), (500, 300)])
@pytest.mark.parametrize("d", [64, 128])
def test_lengths(S, window, sinks, d):
    if window > S + 1 and S > 3:
        pytest.skip("no window")
    _check(1, S, S, 4, 2, d, window, sinks)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("window,sinks", [(5, 0), (40, 7), (150, 0), (150, 140), (300, 1), (8, 400)])
@pytest.mark.parametrize("hq,hkv,d", [(6, 2, 96), (8, 1, 64), (3, 3, 128), (2, 1, 8)])
def test_both_ways_and_heads(causal, window, sinks, hq, hkv, d):
    """Sinks ahead of a row are seen where the mask is not causal, however far."""
    _check(2, 700, 700, hq, hkv, d, window, sinks, causal=causal)


@pytest.mark.parametrize("docs,window,sinks,prefix,causal", [
    (30, 16, 0, False, True), (30, 16, 4, False, True), (200, 50, 3, False, True), (400, 100, 130, False, True), (900, 128, 4, False, True), (300, 64, 5, True, True),
    (300, 64, 5, False, False), (700, 200, 150, False, False), (500, 33, 0, True, True),
])
@pytest.mark.parametrize("d", [64, 128])
def test_documents(docs, window, sinks, prefix, causal, d):
    """Every document has its own sinks; padding sees nothing."""
    _check(3, 1100, 1100, 4, 2, d, window, sinks, causal=causal, docs=docs, prefix=prefix)


@pytest.mark.parametrize("Sq,Sk,window,sinks", [
    (1, 1, 1, 0), (1, 700, 64, 4), (1, 5000, 300, 0), (1, 5000, 2500, 4), (1, 5000, 4000, 0), (5, 3000, 1500, 200), (100, 900, 130, 4), (128, 2000, 1, 1), (129, 2000, 700, 4),
    (300, 2500, 2000, 3), (1, 4097, 4096, 1),
])
@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 128), (4, 4, 64), (12, 2, 96), (5, 1, 64)])
def test_last_queries_of_a_longer_sequence(Sq, Sk, window, sinks, hq, hkv, d):
    """Single tokens and chunks over a cache; walks split over keys, with and without blocks of sinks."""
    from lightron_b200.ops import functional as OF
    q, k, v, do = _inputs(2, Sq, Sk, hq, hkv, d)
    with torch.no_grad():
        o = OF.masked_attention(q, k, v, window=window, sinks=sinks)
    see = local(1, Sq, Sk, True, window, sinks).expand(2, -1, -1)
    got = _run(q, k, v, do, window=window, sinks=sinks)
    _status_ok()
    want = attention64(q, k, v, see, d ** -0.5, do=do)
    assert rel(o, want[0]) < 5e-3 and rel(got[0], want[0]) < 5e-3
    assert rel(got[3], want[3]) < 5e-3
    if window > 1 and Sk > 1:
        _close(got, want)
    hidden = ~see[0].any(0).cuda()
    assert (got[2][:, hidden] == 0).all() and (got[3][:, hidden] == 0).all()


@pytest.mark.parametrize("Sq,Sk,window,sinks,causal,docs", [(70, 1100, 90, 5, False, 0), (5, 900, 200, 140, False, 0), (3, 700, 60, 4, True, 250), (100, 700, 150, 3, True, 300), (40, 640, 33, 200, False, 200),
                                                            (1, 300, 40, 2, True, 90)])
@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 64), (32, 1, 128), (64, 1, 64), (6, 2, 96)])
def test_few_queries_with_documents_and_both_ways(Sq, Sk, window, sinks, causal, docs, hq, hkv, d):
    """The heads of a group as a tile's rows, two to 32 of them, and groups that are not taken so."""
    _check(2, Sq, Sk, hq, hkv, d, window, sinks, causal=causal, docs=docs, seed=3)


def test_many_key_heads_and_pieces():
    """Walks of sinks in many pieces, more key blocks than are listed at once, and fewer pieces than there is room for."""
    _check(1, 2000, 2000, 16, 1, 64, 40, 300)
    _check(5, 900, 900, 2, 2, 64, 20, 3, docs=40)
    q, k, v, do = _inputs(3, 130000, 130000, 1, 1, 8)
    got = _run(q, k, v, do, window=5, sinks=2)
    _status_ok()
    at = torch.arange(130000, device="cuda")
    keys = torch.stack([torch.zeros_like(at), torch.ones_like(at)] + [at - 4 + i for i in range(5)], dim=1)      # sinks, and the window where it does not hold them
    see = (keys >= 0) & (keys <= at[:, None])
    see[:, 2:] &= keys[:, 2:] >= 2
    pick = keys.clamp_min(0)
    qd, kd, vd = (t[:, :, 0].double().requires_grad_() for t in (q, k, v))
    s = (qd[:, :, None] * kd[:, pick]).sum(-1) * 8 ** -0.5
    p = s.masked_fill(~see, -1e300).softmax(-1)
    o = (p[..., None] * vd[:, pick]).sum(2)
    want = (o.detach(), *torch.autograd.grad(o, (qd, kd, vd), do[:, :, 0].double()))
    _close([g[:, :, 0] for g in got], want)


def test_on_two_streams():
    cases = [(_inputs(1, 1500, 1500, 8, 2, 64, seed=i), dict(window=200, sinks=140 * i)) for i in range(2)]
    want = [_run(*t, **kw) for t, kw in cases]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in cases], [[], []]
    for _ in range(4):
        for st, (t, kw), g in zip(streams, cases, got):
            with torch.cuda.stream(st):
                g.append(_run(*t, **kw))
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        for r in g:
            assert all(torch.equal(r[i], w[i]) for i in (0, 2, 3)) and rel(r[1], w[1]) < 2e-3


@pytest.mark.parametrize("cap", [0.0, 20.0, 200.0])
@pytest.mark.parametrize("slopes", [None, [0.5, 0.01, 0.0, 0.25], [-0.01, -0.3, -1.3, 0.25]])
@pytest.mark.parametrize("Sq,Sk,d,window,sinks,causal,docs", [
    (600, 600, 64, 100, 5, True, 0), (600, 600, 128, 300, 140, True, 0), (500, 500, 96, 90, 3, False, 0), (800, 800, 64, 70, 4, True, 250), (1, 2600, 64, 2200, 4, True, 0), (70, 1500, 128, 200, 2, True, 0),
    (700, 700, 128, 60, 3, False, 300),
])
def test_caps_and_biases(Sq, Sk, d, window, sinks, causal, docs, slopes, cap):
    if cap == 0.0 and slopes is None:
        pytest.skip("elsewhere")
    _check(1, Sq, Sk, 4, 2, d, window, sinks, causal=causal, docs=docs, cap=cap, slopes=slopes, scale=2.0)


@pytest.mark.parametrize("d", [64, 128])
def test_a_window_of_one_is_the_value(d):
    q, k, v, do = _inputs(2, 300, 300, 4, 2, d)
    o, dq, dk, dv = _run(q, k, v, do, window=1)
    _status_ok()
    assert torch.equal(o, v.repeat_interleave(2, 2))
    assert rel(dv, do.double().unflatten(2, (2, 2)).sum(3)) < 2.0 ** -8
    assert dq.abs().max() < 1e-2 and dk.abs().max() < 1e-2          # zero, but for D's rounding


def test_windows_over_everything_are_none():
    """The same bits as without one (o, dk and dv; dq is added up as key tiles come)."""
    from lightron_b200.ops import functional as OF
    q, k, v, do = _inputs(2, 700, 700, 4, 2, 64)
    for causal in (True, False):
        want = _run(q, k, v, do, causal=causal)
        for window, sinks in ((700, 0), (701, 5), (10 ** 12, 10 ** 12), (2 ** 31, 2 ** 40)):
            got = _run(q, k, v, do, causal=causal, window=window, sinks=sinks)
            assert all(torch.equal(got[i], want[i]) for i in (0, 2, 3))
    # sinks over everything
    want = attention64(q, k, v, torch.ones(2, 700, 700, dtype=torch.bool).tril(), 64 ** -0.5, do=do)
    _close(_run(q, k, v, do, window=3, sinks=10 ** 12), want)
    assert OF.masked_attention(q, k, v, window=5, sinks=2).shape == q.shape


def test_hidden_scores_may_be_anything():
    """Keys outside of every window with the largest scores, and weights that would overflow: as if they were not there."""
    q, k, v, do = _inputs(1, 600, 600, 2, 1, 64)
    k = k.clone()
    k[:, 100:140] = 3e18
    see = local(1, 600, 600, True, 50, 4)
    o, dq, dk, dv = _run(q, k, v, do, window=50, sinks=4)
    rows = torch.arange(600, device="cuda") >= 140 + 50
    want = attention64(q, torch.where((k.abs() > 1e10), 0, k), v, see, 64 ** -0.5, do=do)
    assert rel(o[:, rows], want[0][:, rows]) < 5e-3 and rel(dq[:, rows], want[1][:, rows]) < 5e-3
    assert torch.isfinite(o[:, :100]).all() and rel(o[:, :100], want[0][:, :100]) < 5e-3


@pytest.mark.parametrize("order", ["heads first", "batch inside", "fused", "askew"])
def test_strides(order):
    B, S, hq, hkv, d = 2, 400, 4, 2, 64
    q, k, v, do = _inputs(B, S, S, hq, hkv, d)
    want = _run(q, k, v, do, window=70, sinks=3)
    if order == "fused":
        both = torch.cat((q, k, v), dim=2)
        q, k, v = both[:, :, :hq], both[:, :, hq:hq + hkv], both[:, :, hq + hkv:]
    else:
        move = {"heads first": lambda t: t.transpose(1, 2).contiguous().transpose(1, 2), "batch inside": lambda t: t.permute(1, 2, 0, 3).contiguous().permute(2, 0, 1, 3),
                "askew": lambda t: torch.nn.functional.pad(t, (1, 0))[..., 1:]}[order]
        q, k, v, do = map(move, (q, k, v, do))
    got = _run(q, k, v, do, window=70, sinks=3)
    assert all(torch.equal(got[i], want[i]) for i in (0, 2, 3)) and rel(got[1], want[1]) < 2e-3


def test_same_bits_each_time():
    q, k, v, do = _inputs(2, 1500, 1500, 8, 2, 64)
    runs = [_run(q, k, v, do, window=200, sinks=140) for _ in range(3)]
    for r in runs[1:]:
        assert all(torch.equal(r[i], runs[0][i]) for i in (0, 2, 3)) and rel(r[1], runs[0][1]) < 2e-3


def test_python_node_is_the_same(monkeypatch):
    from lightron_b200.ops import functional as OF, native
    q, k, v, do = _inputs(2, 500, 500, 4, 2, 64)
    ids = documents(2, 500, 200, seed=3).cuda()
    mask = OF.attention_mask(documents=ids)
    want = _run(q, k, v, do, mask=mask, window=60, sinks=3, softcap=20.0)
    monkeypatch.setattr(native, "host_ops", lambda: None)
    got = _run(q, k, v, do, mask=mask, window=60, sinks=3, softcap=20.0)
    assert all(torch.equal(got[i], want[i]) for i in (0, 2, 3)) and rel(got[1], want[1]) < 2e-3


def test_captured_and_replayed():
    from lightron_b200.ops import functional as OF
    q, k, v, do = _inputs(1, 900, 900, 4, 2, 64)
    ids = documents(1, 900, 300, seed=3).cuda()
    ins = [t.clone().requires_grad_() for t in (q, k, v)]

    def step():
        o = OF.masked_attention(*ins, mask=OF.attention_mask(documents=ids), window=100, sinks=4)
        return (o, *torch.autograd.grad(o, ins, do))
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    outs = []
    for g in graphs:
        with torch.cuda.graph(g):
            outs.append(step())
    for seed in (5, 6):
        with torch.no_grad():
            ins[0].copy_(_rand(1, 900, 4, 64, seed=seed))
            ids.copy_(documents(1, 900, 300, seed=seed))
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        want = step()
        for out in outs:
            assert all(torch.equal(out[i], want[i]) for i in (0, 2, 3)) and rel(out[1], want[1]) < 2e-3


def test_long_cache():
    """Keys past 2^31 elements: the last token of a cache of 2.2 billion."""
    from lightron_b200.ops import functional as OF
    Sk, hkv, d = 1100000, 16, 128
    k = torch.empty(1, Sk, hkv, d, dtype=BF16, device="cuda")
    v = torch.empty_like(k)
    k.zero_()
    v.zero_()
    near = 600
    k[:, -near:], v[:, -near:] = _rand(1, near, hkv, d, seed=1), _rand(1, near, hkv, d, seed=2)
    k[:, :4], v[:, :4] = _rand(1, 4, hkv, d, seed=3), _rand(1, 4, hkv, d, seed=4)
    q = _rand(1, 2, 2 * hkv, d, seed=5)
    with torch.no_grad():
        o = OF.masked_attention(q, k, v, window=500, sinks=4)
    _status_ok()
    small_k, small_v = (torch.cat((t[:, :4], t[:, -near:]), dim=1) for t in (k, v))
    see = torch.zeros(1, 2, 4 + near, dtype=torch.bool)
    see[:, :, :4] = True
    see[0, 0, 4 + near - 1 - 500:4 + near - 1] = True
    see[0, 1, 4 + near - 500:] = True
    assert rel(o, attention64(q, small_k, small_v, see, d ** -0.5)) < 5e-3
