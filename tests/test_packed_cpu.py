"""Masks, attention, rotation and clipping of packed batches on the CPU: the intervals against the definition, gradients against differences, refusals."""
import pytest
import torch

from lightron_b200.ops import functional as OF
from lightron_b200.ops import reference as ref
from packed_oracle import attention64, documents, rel, visible


def _see(mask, Sq):
    """[B, Sq, Sk] from the mask's intervals, once by the queries' and once by the keys'."""
    S = mask.length
    at = torch.arange(S)
    row = mask.q_bounds[:, S - Sq:].cpu()
    by_q = (at >= row[..., :1]) & (at < row[..., 1:])
    col = mask.k_bounds.cpu()
    by_k = (at >= col[..., :1]) & (at < col[..., 1:])              # [B, key, position]
    return by_q, by_k.transpose(1, 2)[:, S - Sq:]


@pytest.mark.parametrize("S", [1, 2, 7, 64, 129])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("docs", [0, 1, 9])
@pytest.mark.parametrize("prefix", ["none", "marks", "lengths"])
def test_intervals_are_the_mask(S, causal, docs, prefix):
    if (prefix == "none" and not docs) or (prefix != "none" and not causal):
        pytest.skip("no such mask")
    B = 3
    ids = documents(B, S, docs, seed=S + docs) if docs else None
    marks = lens = None
    if prefix == "marks":
        marks = torch.rand(B, S, generator=torch.Generator().manual_seed(S)) < 0.6
        marks[0] = True
    if prefix == "lengths":
        lens = torch.tensor([0, S // 2, S])
        marks = torch.arange(S)[None] < lens[:, None]
    mask = OF.attention_mask(documents=ids, prefix=lens if prefix == "lengths" else marks, causal=causal, length=S)
    want = visible(B, S, S, causal, ids, marks)
    by_q, by_k = _see(mask, S)
    assert torch.equal(by_q, want) and torch.equal(by_k, want)
    for bounds in (mask.q_bounds, mask.k_bounds):                  # what the kernels rely on: ends never fall
        assert (bounds[:, 1:] >= bounds[:, :-1]).all()


def test_equal_ids_apart_are_two_documents():
    mask = OF.attention_mask(documents=torch.tensor([[5, 5, 2, 5]], dtype=torch.int64))
    assert mask.q_bounds[0].tolist() == [[0, 1], [0, 2], [2, 3], [3, 4]]


@pytest.mark.parametrize("cap,alibi,prefix", [(0.0, False, False), (5.0, False, True), (0.0, True, True), (5.0, True, False)])
def test_attention_gradients_against_differences(cap, alibi, prefix):
    g = torch.Generator().manual_seed(0)
    B, Sq, Sk, hq, hkv, d = 2, 5, 7, 4, 2, 6
    q, k, v = (torch.randn(B, s, h, d, generator=g, dtype=torch.float64, requires_grad=True) for s, h in ((Sq, hq), (Sk, hkv), (Sk, hkv)))
    ids = documents(B, Sk, 3, seed=4)
    mask = OF.attention_mask(documents=ids, prefix=torch.ones(B, Sk, dtype=torch.bool) if prefix else None)
    slopes = torch.tensor([0.5, 0.25, 0.1, 0.0]) if alibi else None
    fn = lambda q, k, v: OF.masked_attention(q, k, v, mask=mask, scale=1.3, softcap=cap, slopes=slopes)  # noqa: E731
    assert torch.autograd.gradcheck(fn, (q, k, v), eps=1e-6, atol=1e-7)
    see = visible(B, Sq, Sk, True, ids, torch.ones(B, Sk) if prefix else None)
    assert rel(fn(q, k, v), attention64(q, k, v, see, 1.3, cap, slopes)) < 1e-12


def test_rows_that_see_nothing():
    q, k, v = (torch.randn(1, 5, 2, 8, generator=torch.Generator().manual_seed(3), requires_grad=True) for _ in range(3))
    mask = OF.attention_mask(documents=torch.tensor([[-1, 0, 0, -7, -7]], dtype=torch.int32))
    o = OF.masked_attention(q, k, v, mask=mask)
    empty = torch.tensor([True, False, False, True, True])
    assert (o[0, empty] == 0).all() and (o[0, ~empty] != 0).all()
    for t, grad in zip("qkv", torch.autograd.grad(o.sum(), (q, k, v))):
        assert (grad[0, empty] == 0).all(), t


def test_attention_without_keys_or_queries():
    q = torch.zeros(2, 0, 4, 8)
    assert OF.masked_attention(q, torch.zeros(2, 3, 2, 8), torch.zeros(2, 3, 2, 8)).shape == (2, 0, 4, 8)
    assert OF.masked_attention(torch.zeros(0, 3, 4, 8), torch.zeros(0, 3, 2, 8), torch.zeros(0, 3, 2, 8)).shape == (0, 3, 4, 8)


def test_rotation_by_axes():
    g = torch.Generator().manual_seed(1)
    x = torch.randn(2, 5, 3, 8, generator=g, dtype=torch.float64, requires_grad=True)
    cos, sin = ref.rope_tables(8, 50)
    pos = torch.randint(0, 50, (3, 2, 5), generator=g)
    axes = [0, 2, 1, 2]
    y = ref.rope_axes(x, cos.double(), sin.double(), pos, axes)
    for i, a in enumerate(axes):                                   # a complex number per pair
        z = torch.complex(x[..., 2 * i], x[..., 2 * i + 1]) * torch.complex(cos[pos[a], i].double(), sin[pos[a], i].double())[..., None]
        assert torch.allclose(y[..., 2 * i], z.real) and torch.allclose(y[..., 2 * i + 1], z.imag)
    # all axes equal: the rotation of rope(); forth and back: the input
    one = torch.arange(5).expand(3, 5)
    assert torch.allclose(OF.rope_axes(x.float(), cos, sin, one, axes), OF.rope(x.float(), cos, sin), atol=1e-6)
    assert torch.allclose(ref.rope_axes(y, cos.double(), sin.double(), pos, axes, inverse=True), x, atol=1e-6)
    assert torch.autograd.gradcheck(lambda t: ref.rope_axes(t, cos.double(), sin.double(), pos, axes), (x,))


def test_norm_and_clip():
    g = torch.Generator().manual_seed(2)
    ts = [torch.randn(3, 5, generator=g), torch.randn(7, generator=g).bfloat16(), torch.zeros(0), torch.randn(4, 6, generator=g).t()]
    want = sum(t.double().square().sum() for t in ts).sqrt()
    assert abs(float(OF.grad_norm(ts)) / float(want) - 1) < 1e-6
    out = [torch.empty_like(t) for t in ts]
    assert float(OF.clip_grad_norm(ts, 1.0, out=out)) == float(OF.grad_norm(ts))
    for t, o in zip(ts, out):
        assert torch.allclose(o.float(), t.float() / float(want), rtol=1e-2 if t.dtype == torch.bfloat16 else 1e-5)
    small = [t.clone() for t in ts]
    OF.clip_grad_norm(small, 100.0)                                # below the limit: as they were
    assert all(torch.equal(a, b) for a, b in zip(small, ts))
    assert float(OF.grad_norm([])) == 0.0 and float(OF.clip_grad_norm([], 1.0)) == 0.0


def _packed_model(**kw):
    from lightron_b200 import mesh
    from lightron_b200.config import ModelArgs
    from lightron_b200.models import LightronTransformer, init_weights
    mesh.set_context(None)
    args = ModelArgs(dim=32, n_layers=2, n_heads=4, n_kv_heads=2, vocab_size=64, intermediate_size=48, max_seq_len=64, **kw)
    model = LightronTransformer(args, dtype=torch.float32, device="cpu")
    init_weights(model, 0, std=0.2)
    return model


@pytest.mark.parametrize("kw", [{}, dict(attn_softcap=5.0), dict(attn_alibi=True), dict(rope_sections=(2, 1, 1), attn_softcap=3.0)])
def test_packed_model_is_its_documents(kw):
    """Logits of documents packed into one sequence, with positions of their own: those of each document alone."""
    model = _packed_model(**kw)
    lens = [5, 9, 3]
    tokens = torch.randint(0, 64, (1, sum(lens)), generator=torch.Generator().manual_seed(0))
    ids = torch.cat([torch.full((n,), i) for i, n in enumerate(lens)])[None]
    pos = torch.cat([torch.arange(n) for n in lens])[None]
    if "rope_sections" in kw:
        pos = torch.stack([pos, pos // 2, pos % 3])
    packed = model(tokens, positions=pos, mask=OF.attention_mask(documents=ids))
    at = 0
    for n in lens:
        alone = model(tokens[:, at:at + n], positions=pos[..., at:at + n])
        assert torch.allclose(packed[:, at:at + n], alone, atol=1e-5)
        at += n
    loss = model.loss(tokens, tokens, positions=pos, mask=OF.attention_mask(documents=ids))
    loss.backward()
    assert all(torch.isfinite(p.grad).all() for p in model.parameters())


def _example():
    import importlib.util
    import os
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "packed_documents.py")
    spec = importlib.util.spec_from_file_location("packed_documents", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_example_runs():
    losses = _example().main(["--steps", "4", "--batch", "2", "--seq-length", "96", "--dim", "64", "--layers", "1", "--device", "cpu"])
    assert len(losses) == 4 and all(0 < x < 20 for x in losses)


@pytest.mark.gpu
def test_example_learns_on_the_gpu():
    losses = _example().main(["--steps", "30", "--device", "cuda"])
    assert losses[-1] < losses[0] - 0.3


def test_model_arguments_are_checked():
    from lightron_b200.config import ModelArgs
    for bad in (dict(rope_sections=(2, 1)), dict(attn_softcap=-1.0), dict(attn_alibi=True, cp_size=2)):
        with pytest.raises(ValueError):
            ModelArgs(dim=32, n_heads=4, **bad)


def _clipped_worker(rank, world, clip):
    from lightron_b200 import mesh
    from lightron_b200.parallel import apply_fsdp2
    from lightron_b200.parallel.fsdp import FSDPOptimizer
    ctx = mesh.setup_distributed(dp_size=world, backend="gloo")
    model = _packed_model()
    apply_fsdp2(model, ctx=ctx, param_dtype=torch.float32)
    opt = FSDPOptimizer(model, lr=1e-2, weight_decay=0.0, grad_clip=clip, groups=(ctx.dpcp_group, ctx.tp_group))
    tokens = torch.randint(0, 64, (2, 8), generator=torch.Generator().manual_seed(1))
    norms = []
    for _ in range(2):
        opt.zero_grad()
        model.loss(tokens[rank % 2:rank % 2 + 1], tokens[rank % 2:rank % 2 + 1].roll(-1, 1)).backward()
        opt.step()
        norms.append(float(opt.last_grad_norm))
    return {k: v.numpy().copy() for k, v in model._fsdp.full_state_dict().items()}, norms


def test_sharded_optimizer_clips_by_the_global_norm():
    from dist_utils import run_distributed
    (got, norms), (_, other) = run_distributed(_clipped_worker, 2, 0.05)
    assert norms == other
    model = _packed_model()
    opt = torch.optim.AdamW(model.parameters(), lr=1e-2, weight_decay=0.0)
    tokens = torch.randint(0, 64, (2, 8), generator=torch.Generator().manual_seed(1))
    for n in norms:
        opt.zero_grad()
        model.loss(tokens, tokens.roll(-1, 1)).backward()
        want = torch.nn.utils.clip_grad_norm_(model.parameters(), 0.05)
        assert abs(n / float(want) - 1) < 1e-4
        opt.step()
    for k, v in model.state_dict().items():
        assert torch.allclose(torch.from_numpy(got[k]), v, atol=1e-4), k


def _attn(**kw):
    a = dict(q=torch.zeros(2, 4, 4, 8), k=torch.zeros(2, 4, 2, 8), v=torch.zeros(2, 4, 2, 8))
    a.update(kw)
    return lambda: OF.masked_attention(**a)


def _mask(**kw):
    return lambda: OF.attention_mask(**kw)


def _rope(**kw):
    cos, sin = ref.rope_tables(8, 16)
    a = dict(x=torch.zeros(2, 3, 1, 8), cos=cos, sin=sin, positions=torch.zeros(3, 3, dtype=torch.int32), axes=[0, 1, 2, 2])
    a.update(kw)
    return lambda: OF.rope_axes(**a)


IDS = torch.zeros(2, 4, dtype=torch.int32)


@pytest.mark.parametrize("call", [
    _attn(k=torch.zeros(2, 4, 3, 8), v=torch.zeros(2, 4, 3, 8)),                           # 4 query heads of 3
    _attn(v=torch.zeros(2, 5, 2, 8)), _attn(k=torch.zeros(2, 4, 2, 16), v=torch.zeros(2, 4, 2, 16)), _attn(q=torch.zeros(2, 4, 8)),
    _attn(q=torch.zeros(2, 5, 4, 8)),                                                      # more queries than positions
    _attn(v=torch.zeros(2, 4, 2, 8, dtype=torch.bfloat16)),
    _attn(softcap=-1.0), _attn(softcap=float("inf")), _attn(softcap=float("nan")),
    _attn(slopes=torch.zeros(2)), _attn(slopes=torch.zeros(4, dtype=torch.float64)), _attn(slopes=torch.zeros(4, requires_grad=True)),
    _attn(mask=IDS), _attn(mask=OF.attention_mask(documents=IDS[:, :3])), _attn(mask=OF.attention_mask(documents=IDS[:1])),
    _attn(mask=OF.attention_mask(documents=IDS), causal=False),
    _mask(), _mask(documents=IDS.float()), _mask(documents=IDS[0]), _mask(documents=IDS, prefix=IDS.bool(), causal=False),
    _mask(documents=IDS, prefix=IDS.float()), _mask(documents=IDS, prefix=IDS[:, :3].bool()), _mask(prefix=torch.tensor([1, 2])), _mask(documents=IDS, length=5),
    _rope(axes=[0, 1, 2]), _rope(axes=[0, 1, 2, 3]), _rope(axes=[0, 1, 2, -1]), _rope(positions=torch.zeros(3, 2, dtype=torch.int32)),
    _rope(positions=torch.zeros(3, 3)), _rope(cos=torch.zeros(16, 3)), _rope(x=torch.zeros(2, 3, 8)),
    lambda: OF.grad_norm([torch.zeros(2, dtype=torch.int32)]), lambda: OF.grad_norm([torch.zeros(2, dtype=torch.float64)]),
    lambda: OF.clip_grad_norm([torch.zeros(2)], -1.0), lambda: OF.clip_grad_norm([torch.zeros(2)], float("nan")),
    lambda: OF.clip_grad_norm([torch.zeros(2)], 1.0, out=[torch.zeros(3)]), lambda: OF.clip_grad_norm([torch.zeros(2)], 1.0, out=[]),
])
def test_refusals(call):
    with pytest.raises(ValueError):
        call()
