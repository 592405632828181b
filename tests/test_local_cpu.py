"""Windows with sinks, per-head norms with the rotation and scaled embeddings on the CPU: against their definitions, gradients against differences, refusals."""
import pytest
import torch

from lightron_b200.ops import functional as OF
from lightron_b200.ops import reference as ref
from local_oracle import embedding64, local, norm_rope64
from packed_oracle import attention64, documents, rel


def _rand(*shape, seed=0, grad=True):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed), dtype=torch.float64, requires_grad=grad)


@pytest.mark.parametrize("Sq,Sk", [(1, 1), (1, 9), (5, 9), (9, 9)])
@pytest.mark.parametrize("window,sinks", [(1, 0), (2, 1), (3, 5), (9, 0), (100, 2), (2, 100)])
@pytest.mark.parametrize("causal,docs,prefix", [(True, 0, False), (False, 0, False), (True, 3, False), (False, 3, False), (True, 4, True)])
def test_window_is_its_definition(Sq, Sk, window, sinks, causal, docs, prefix):
    B, d = 2, 6
    q, k, v = _rand(B, Sq, 4, d, seed=1), _rand(B, Sk, 2, d, seed=2), _rand(B, Sk, 2, d, seed=3)
    ids = documents(B, Sk, docs, seed=4) if docs else None
    marks = torch.rand(B, Sk, generator=torch.Generator().manual_seed(5)) < 0.7 if prefix else None
    mask = OF.attention_mask(documents=ids, prefix=marks, causal=causal) if docs or prefix else None
    o = OF.masked_attention(q, k, v, mask=mask, causal=causal, scale=1.3, window=window, sinks=sinks)
    see = local(B, Sq, Sk, causal, window, sinks, ids, marks)
    do = _rand(B, Sq, 4, d, seed=6, grad=False)
    want = attention64(q, k, v, see, 1.3, do=do)
    assert rel(o, want[0]) < 1e-12
    for g, w in zip(torch.autograd.grad(o, (q, k, v), do), want[1:]):
        assert (g - w).abs().max() < 1e-12


def test_window_gradients_against_differences():
    q, k, v = _rand(1, 6, 2, 4, seed=1), _rand(1, 8, 1, 4, seed=2), _rand(1, 8, 1, 4, seed=3)
    fn = lambda q, k, v: OF.masked_attention(q, k, v, window=3, sinks=2, softcap=4.0)  # noqa: E731
    assert torch.autograd.gradcheck(fn, (q, k, v), eps=1e-6, atol=1e-7)


@pytest.mark.parametrize("axes", [None, [0, 2, 1, 0]])
def test_norm_rope(axes):
    B, S, d = 2, 5, 8
    q, k, wq, wk = _rand(B, S, 4, d, seed=1), _rand(B, S, 2, d, seed=2), _rand(d, seed=3), _rand(d, seed=4)
    cos, sin = ref.rope_tables(d, 50)
    A = 1 if axes is None else 3
    pos = torch.randint(0, 50, (A, B, S), generator=torch.Generator().manual_seed(7))
    fn = lambda *t: OF.qk_norm_rope(*t, cos, sin, positions=pos[0] if axes is None else pos, axes=axes, eps=0.01)  # noqa: E731
    y = fn(q, k, wq, wk)
    for got, x, w in ((y[0], q, wq), (y[1], k, wk)):
        assert rel(got, norm_rope64(x, w, cos, sin, pos, axes or [0] * (d // 2), 0.01)) < 1e-12
    assert torch.autograd.gradcheck(fn, (q, k, wq, wk))
    # none, [S] and [B, S] positions of text are the same
    text = torch.arange(S)
    plain = [OF.qk_norm_rope(q, k, wq, wk, cos, sin, positions=p, axes=a) for p, a in ((None, None), (text, None), (text.expand(B, S), None), (None, axes), (text, axes)) if a is None or axes]
    assert all(torch.equal(x, z) for p in plain for x, z in zip(p, plain[0]))
    assert rel(plain[0][0], OF.rope(OF.rmsnorm(q, wq, 1e-6), cos, sin)) < 1e-6


def test_norm_rope_outside_the_tables():
    cos, sin = ref.rope_tables(8, 3)
    q = torch.ones(1, 5, 1, 8)
    y, _ = OF.qk_norm_rope(q, q, torch.ones(8), torch.ones(8), cos, sin)
    assert torch.isfinite(y[:, :3]).all() and torch.isnan(y[:, 3:]).all()


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("start", [0, 7])
def test_scaled_embedding(dtype, start):
    tokens = torch.tensor([[7, 8, 7, 12], [3, 11, 40, -1]], dtype=dtype)
    w, dy = _rand(5, 6, seed=1), _rand(2, 4, 6, seed=2, grad=False)
    y = OF.scaled_embedding(tokens, w, -1.5, start)
    want = embedding64(tokens, w.detach(), -1.5, start, dy)
    assert rel(y, want[0]) < 1e-14 and rel(torch.autograd.grad(y, w, dy)[0], want[1]) < 1e-14
    assert OF.scaled_embedding(tokens[:0], w).shape == (0, 4, 6)


def test_scaled_embedding_sums_in_32_bits():
    """A thousand small gradients beside a large one, in bf16."""
    w = torch.zeros(1, 2, dtype=torch.bfloat16, requires_grad=True)
    dy = torch.full((1025, 2), 2.0 ** -9, dtype=torch.bfloat16)
    dy[0] = 1.0
    dw, = torch.autograd.grad(OF.scaled_embedding(torch.zeros(1025, dtype=torch.long), w), w, dy)
    assert (dw == 3.0).all()


def _attn(**kw):
    a = dict(q=torch.zeros(2, 4, 4, 8), k=torch.zeros(2, 4, 2, 8), v=torch.zeros(2, 4, 2, 8))
    a.update(kw)
    return lambda: OF.masked_attention(**a)


def _norm(**kw):
    cos, sin = ref.rope_tables(8, 16)
    a = dict(q=torch.zeros(2, 3, 4, 8), k=torch.zeros(2, 3, 2, 8), q_weight=torch.ones(8), k_weight=torch.ones(8), cos=cos, sin=sin)
    a.update(kw)
    return lambda: OF.qk_norm_rope(**a)


def _embed(**kw):
    a = dict(tokens=torch.zeros(3, dtype=torch.long), w=torch.zeros(5, 4))
    a.update(kw)
    return lambda: OF.scaled_embedding(**a)


@pytest.mark.parametrize("call", [
    _attn(window=0), _attn(window=-1), _attn(window=2.0), _attn(window=True), _attn(sinks=1), _attn(window=2, sinks=-1), _attn(window=2, sinks=None), _attn(window=2, sinks=1.0),
    _norm(k=torch.zeros(2, 4, 2, 8)), _norm(k=torch.zeros(2, 3, 2, 16)), _norm(q=torch.zeros(2, 3, 8)), _norm(q_weight=torch.ones(4)), _norm(k_weight=torch.ones(8).double()),
    _norm(k=torch.zeros(2, 3, 2, 8).double()), _norm(eps=-1.0), _norm(eps=float("nan")), _norm(eps=float("inf")), _norm(cos=torch.zeros(16, 3)), _norm(cos=torch.zeros(16, 4).double()),
    _norm(positions=torch.zeros(2, 4, dtype=torch.int32)), _norm(positions=torch.zeros(3)), _norm(axes=[0, 1]), _norm(axes=[0, 1, -1, 0]),
    _norm(axes=[0, 0, 1, 1], positions=torch.zeros(1, 2, 3, dtype=torch.int32)), _norm(cos=torch.zeros(0, 4), sin=torch.zeros(0, 4)),
    _embed(w=torch.zeros(5)), _embed(w=torch.zeros(5, 4, dtype=torch.int32)), _embed(tokens=torch.zeros(3)), _embed(tokens=torch.zeros(3, dtype=torch.int16)), _embed(scale=float("inf")),
    _embed(scale=float("nan")), _embed(scale=1e39), _embed(vocab_start=-1),
])
def test_refusals(call):
    with pytest.raises(ValueError):
        call()
