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


@pytest.mark.parametrize("start", [1 << 63, (1 << 64) + 2, 1.5, True, None])
def test_a_vocab_start_that_is_no_id_is_refused(start):
    with pytest.raises(ValueError):
        _embed(vocab_start=start)()


# ---- in the model -----------------------------------------------------------------------------------

LOCAL = dict(attn_window=4, attn_sinks=2, qk_norm=True, embed_scale=3.0)


def _model(ctx=None, **kw):
    from lightron_b200 import mesh
    from lightron_b200.config import ModelArgs
    from lightron_b200.models import LightronTransformer, init_weights
    if ctx is None:
        mesh.set_context(None)
    args = ModelArgs(**{**dict(dim=32, n_layers=3, n_heads=4, n_kv_heads=2, vocab_size=64, intermediate_size=48, max_seq_len=64), **kw})
    model = LightronTransformer(args, ctx=ctx, dtype=torch.float32, device="cpu")
    init_weights(model, 0, std=0.2)
    with torch.no_grad():
        for n, p in model.named_parameters():
            if p.dim() == 1:                                       # the same on every rank
                p.add_(0.3 * torch.randn(p.shape, generator=torch.Generator().manual_seed(len(n))))
    return model


@pytest.mark.parametrize("kw", [dict(attn_window=4), LOCAL, dict(LOCAL, attn_global_freq=2, attn_softcap=5.0), dict(qk_norm=True, rope_sections=(2, 1, 1)), dict(embed_scale=0.5)])
def test_model_of_documents_is_each_alone(kw):
    model = _model(**kw)
    lens = [5, 14, 9]
    tokens = torch.randint(0, 64, (1, sum(lens)), generator=torch.Generator().manual_seed(0))
    ids = torch.cat([torch.full((n,), i) for i, n in enumerate(lens)])[None]
    pos = torch.cat([torch.arange(n) for n in lens])[None]
    packed = model(tokens, positions=pos, mask=OF.attention_mask(documents=ids))
    at = 0
    for n in lens:
        assert torch.allclose(packed[:, at:at + n], model(tokens[:, at:at + n]), atol=1e-5)
        at += n
    model.loss(tokens, tokens, positions=pos, mask=OF.attention_mask(documents=ids)).backward()
    assert all(torch.isfinite(p.grad).all() and p.grad.abs().sum() > 0 for p in model.parameters())


def test_model_layers_see_their_windows():
    """A change of one token reaches as far as the windows of the layers and the layers without one let it."""
    tokens = torch.randint(0, 64, (1, 40), generator=torch.Generator().manual_seed(1))
    other = tokens.clone()
    other[0, 10] = (other[0, 10] + 1) % 64
    for kw, last in ((dict(attn_window=4), 10 + 3 * 3), (dict(attn_window=4, attn_global_freq=3), 39), (dict(attn_window=64), 39), (dict(attn_window=1), 10)):
        model = _model(**kw)
        changed = (model(tokens) - model(other)).abs().amax(-1)[0] > 1e-6
        assert changed.nonzero().max() == last and not changed[:10].any()
    sinks = _model(attn_window=2, attn_sinks=11)                   # position 10 is a sink
    assert ((sinks(tokens) - sinks(other)).abs().amax(-1)[0, 10:] > 1e-7).all()


def test_scaled_embedding_in_the_model():
    """Embeddings that are multiplied by c are those of weights c times as large."""
    tokens = torch.randint(0, 64, (2, 9), generator=torch.Generator().manual_seed(1))
    a, b = _model(embed_scale=3.0), _model()
    with torch.no_grad():
        b.tok_embeddings.weight.mul_(3.0)
    assert torch.allclose(a(tokens), b(tokens), atol=1e-5)
    assert torch.allclose(a.tok_embeddings(tokens), b.tok_embeddings(tokens), atol=1e-6)


def test_model_arguments_are_checked():
    from lightron_b200.config import ModelArgs
    for bad in (dict(attn_window=0), dict(attn_window=1.5), dict(attn_sinks=2), dict(attn_window=4, attn_sinks=-1), dict(attn_global_freq=2), dict(attn_window=4, attn_global_freq=-1),
                dict(embed_scale=float("inf")), dict(attn_window=4, cp_size=2), dict(qk_norm=True, cp_size=2)):
        with pytest.raises(ValueError):
            ModelArgs(dim=32, n_heads=4, **bad)
    args = ModelArgs(dim=32, n_heads=4, n_layers=2, attn_window=4, attn_global_freq=2, qk_norm=True)
    assert [args.window_of(i) for i in range(4)] == [4, None, 4, None] and args.packed_attention
    assert args.num_params() == ModelArgs(dim=32, n_heads=4, n_layers=2).num_params() + 2 * 2 * 8


def test_norm_weights_of_other_layouts():
    """Weights of heads whose pairs lie half a head apart, there and back, and what they compute."""
    from lightron_b200.utils.hf import convert_hf_llama_state_dict, export_hf_llama_state_dict
    model = _model(qk_norm=True)
    sd = model.state_dict()
    out = export_hf_llama_state_dict(sd, 4, 2)
    assert "model.layers.0.self_attn.q_norm.weight" in out
    assert torch.equal(out["model.layers.0.self_attn.q_norm.weight"], torch.cat((sd["layers.0.attention.q_norm.weight"][0::2], sd["layers.0.attention.q_norm.weight"][1::2])))
    back = convert_hf_llama_state_dict(out, 4, 2)
    assert back.keys() == sd.keys() and all(torch.equal(back[k], sd[k]) for k in sd)


def _local_worker(rank, world, sp):
    import torch.distributed as dist
    from lightron_b200 import mesh
    ctx = mesh.setup_distributed(tp_size=world, backend="gloo")
    model = _model(ctx=ctx, tp_size=world, sequence_parallel=sp, **LOCAL)
    tokens = torch.randint(0, 64, (2, 12), generator=torch.Generator().manual_seed(1))
    loss = model.loss(tokens, tokens.roll(-1, 1))
    loss.backward()
    grads = {}
    for n, p in model.named_parameters():
        if p.dim() == 1:
            g = p.grad.clone()
            if sp:                                                 # parts, which the optimizers add up
                dist.all_reduce(g, group=ctx.tp_group)
            grads[n] = g.numpy()
    grads["tok_embeddings.weight"] = model.tok_embeddings.weight.grad.numpy()
    return float(loss.detach()), grads


@pytest.mark.parametrize("sp", [False, True])
def test_tensor_parallel_gradients(sp):
    """Norm weights of heads that are spread over ranks, and embeddings of parts of the vocabulary: the gradients of one process."""
    from dist_utils import run_distributed
    got = run_distributed(_local_worker, 2, sp)
    model = _model(**LOCAL)
    tokens = torch.randint(0, 64, (2, 12), generator=torch.Generator().manual_seed(1))
    loss = model.loss(tokens, tokens.roll(-1, 1))
    loss.backward()
    for rank, (value, grads) in enumerate(got):
        assert abs(value - float(loss.detach())) < 1e-5
        for n, g in grads.items():
            want = dict(model.named_parameters())[n].grad
            want = want if n != "tok_embeddings.weight" else want[rank * 32:(rank + 1) * 32]
            assert torch.allclose(torch.from_numpy(g), want, atol=1e-5, rtol=1e-4), n


def test_trainer_takes_the_keys():
    """The run configuration's section, with clipping and two pipeline-free steps."""
    from lightron_b200 import mesh
    from lightron_b200.config import parse_config
    from lightron_b200.trainer import Trainer
    mesh.set_context(None)
    raw = {"distributed": {}, "model": {"name": "tiny", "attn_window": 16, "attn_sinks": 2, "attn_global_freq": 4, "qk_norm": True, "embed_scale": 16.0}, "dataset": {"name": "synthetic"},
           "training": {"micro_batch_size": 2, "gradient_accumulation_steps": 1, "seq_length": 64, "learning_rate": 3e-4, "total_steps": 2, "seed": 0, "dtype": "fp32", "grad_clip": 1.0,
                        "log_interval": 1000}}
    tr = Trainer(parse_config(raw, env={}))
    losses = [float(tr.train_step()) for _ in range(2)]
    mesh.set_context(None)
    assert all(0 < x < 20 for x in losses)
