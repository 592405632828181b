"""Operators of packed batches where they can go wrong, on the CPU: what a launch is given, positions outside of tables, text for a model with several axes,
norms of sharded gradients."""
import gc
import weakref

import pytest
import torch

from lightron_b200.ops import functional as OF
from lightron_b200.ops import native
from lightron_b200.ops import reference as ref


class _Library:
    """Stands in for the kernels' library."""

    def lb_grad_norm_parts(self, n):
        return 8

    def lb_masked_attn_fwd_ws_bytes(self, *sizes):
        return 0


def _fake_launches(monkeypatch, call):
    monkeypatch.setattr(native, "require", lambda: _Library())
    monkeypatch.setattr(native, "use_native", lambda t: True)
    monkeypatch.setattr(native, "host_ops", lambda: None)
    monkeypatch.setattr(native, "on_device", lambda t: native._HERE)
    monkeypatch.setattr(native, "stream_ptr", lambda: 0)
    monkeypatch.setattr(native, "call", call)


def test_copies_live_until_their_launch(monkeypatch):
    """A tensor that is not dense is copied for the sum of squares: the copy's address is not handed over without the copy."""
    copies, alive, contiguous = [], [], torch.Tensor.contiguous

    def copying(t, *a, **kw):
        c = contiguous(t, *a, **kw)
        if c is not t:
            copies.append(weakref.ref(c))
        return c

    def call(name, *args):
        gc.collect()
        alive.append((name, [c() is not None for c in copies]))
    _fake_launches(monkeypatch, call)
    monkeypatch.setattr(torch.Tensor, "contiguous", copying)
    OF._grad_parts([torch.randn(8, 8)[:, 1:5], torch.randn(6), torch.randn(9, 4)[::2]], torch.device("cpu"))
    assert alive == [("lb_grad_squares", [True, True])]


def test_tables_of_another_device_are_refused(monkeypatch):
    """Tables and positions that do not lie where ``qkv`` does never reach a kernel."""
    def call(name, *args):
        raise AssertionError(f"{name} was launched")
    _fake_launches(monkeypatch, call)
    qkv, cos, sin = torch.zeros(8, 4 * 8), *ref.rope_tables(8, 16)
    pos = torch.zeros(1, 8, dtype=torch.int32)
    for tables in ((cos.to("meta"), sin.to("meta"), pos.to("meta")), (cos, sin, pos.to("meta")), (cos, sin.to("meta"), pos), (cos.to("meta"), sin.to("meta"), pos)):
        with pytest.raises(ValueError):
            OF.packed_attention_qkv(qkv, *tables, 1, 8, 2, 1, 8, axes=[0] * 4)
        with pytest.raises(ValueError):
            OF.rope_axes(qkv.view(1, 8, 4, 8), *tables, [0] * 4)


@pytest.mark.parametrize("outside", [16, -1, -16, 1000])
def test_positions_outside_the_tables(outside):
    """NaN in the pairs of that axis, values elsewhere, on every path; no access, which on a GPU would end the process."""
    cos, sin = ref.rope_tables(8, 16)
    x = torch.randn(1, 3, 2, 8, generator=torch.Generator().manual_seed(0), requires_grad=True)
    pos = torch.tensor([[0, 15, 3], [0, 15, outside]], dtype=torch.int32)
    y = OF.rope_axes(x, cos, sin, pos, [0, 1, 0, 1])
    away = torch.zeros(1, 3, 2, 8, dtype=torch.bool)
    away[:, 2, :, [2, 3, 6, 7]] = True
    assert torch.equal(torch.isnan(y), away)
    dx, = torch.autograd.grad(y, x, torch.ones_like(y))
    assert torch.equal(torch.isnan(dx), away)


def _model(**kw):
    from lightron_b200 import mesh
    from lightron_b200.config import ModelArgs
    from lightron_b200.models import LightronTransformer, init_weights
    mesh.set_context(None)
    model = LightronTransformer(ModelArgs(dim=32, n_layers=2, n_heads=4, n_kv_heads=2, vocab_size=64, intermediate_size=48, max_seq_len=64, **kw),
                                dtype=torch.float32, device="cpu")
    init_weights(model, 0, std=0.2)
    return model


@pytest.mark.parametrize("B", [1, 2, 3, 4])
def test_text_counts_on_all_axes(B):
    """Without positions, with [S] and with [B, S] (three sequences as well as three axes): the ordinary rotation."""
    plain, axes = _model(), _model(rope_sections=(2, 1, 1))
    tokens = torch.randint(0, 64, (B, 9), generator=torch.Generator().manual_seed(0))
    own = torch.stack([torch.arange(9) + 3 * b for b in range(B)])
    for pos in (None, torch.arange(9), torch.arange(5, 14), own):
        want = plain(tokens, positions=pos)
        assert torch.allclose(axes(tokens, positions=pos), want, atol=1e-5)
    three = own.expand(3, B, 9)
    assert torch.allclose(axes(tokens, positions=three), plain(tokens, positions=own), atol=1e-5)
    loss = axes.loss(tokens, tokens)
    loss.backward()
    assert torch.isfinite(loss)


def test_packed_attention_without_positions():
    B, S, hq, hkv, d = 2, 5, 2, 1, 8
    cos, sin = ref.rope_tables(d, 16)
    qkv = torch.randn(B * S, (hq + 2 * hkv) * d, generator=torch.Generator().manual_seed(0))
    want = OF.packed_attention_qkv(qkv, cos, sin, None, B, S, hq, hkv, d)
    for pos in (None, torch.arange(S), torch.arange(S).expand(3, S), torch.arange(S).expand(3, B, S)):
        assert torch.equal(OF.packed_attention_qkv(qkv, cos, sin, pos, B, S, hq, hkv, d, axes=[0, 1, 2, 2]), want)


def test_trainer_takes_rope_sections():
    """The key of the configuration, through the trainer's own data: the losses of one axis."""
    from lightron_b200 import mesh
    from lightron_b200.config import parse_config
    from lightron_b200.trainer import Trainer
    losses = []
    for model in ({}, {"rope_sections": [2, 4, 2]}):
        mesh.set_context(None)
        trainer = Trainer(parse_config({"distributed": {}, "model": {"name": "tiny", "dim": 64, "n_heads": 4, "n_kv_heads": 2, **model}, "dataset": {"name": "synthetic"},
                                        "training": {"micro_batch_size": 4, "gradient_accumulation_steps": 1, "seq_length": 64, "learning_rate": 3e-4, "total_steps": 2, "seed": 0,
                                                     "dtype": "fp32", "log_interval": 1000}}, env={}))
        losses.append([float(trainer.train_step()) for _ in range(2)])
    assert losses[1] == pytest.approx(losses[0], rel=1e-5)


def _engine(dist_kw, clip):
    return {"distributed": dist_kw, "model": {"name": "tiny"}, "dataset": {"name": "synthetic"},
            "training": {"micro_batch_size": 4, "gradient_accumulation_steps": 1, "seq_length": 64, "learning_rate": 3e-4, "total_steps": 4, "seed": 0, "dtype": "fp32",
                         "log_interval": 1000, "grad_clip": clip}}


def _engine_steps(raw, steps=3):
    """(losses, norms before clipping, replicated parameters after the steps)"""
    from lightron_b200.config import parse_config
    from lightron_b200.trainer import Trainer
    trainer = Trainer(parse_config(raw, env={}))
    losses, norms = [], []
    for _ in range(steps):
        losses.append(float(trainer.train_step()))
        norms.append(float(trainer.optimizer.last_grad_norm) if raw["training"]["grad_clip"] else 0.0)
    state = trainer.net._fsdp.full_state_dict() if hasattr(trainer.net, "_fsdp") else trainer.net.state_dict()
    return losses, norms, {k: v.float().numpy().copy() for k, v in state.items() if v.dim() == 1}


def _engine_worker(rank, world, raw):
    return _engine_steps(raw)


def _against_one_process(dist_kw, world, clip, norm_bound=2e-5):
    from dist_utils import run_distributed
    from lightron_b200 import mesh
    mesh.set_context(None)
    one = _engine({}, clip)
    one["training"]["gradient_accumulation_steps"] = dist_kw.get("dp_size", 1)      # one process sees the whole batch
    losses, norms, params = _engine_steps(one)
    mesh.set_context(None)
    ranks = run_distributed(_engine_worker, world, _engine({"fsdp": True, **dist_kw}, clip))
    for i in range(3):
        mean = sum(r[0][i] for r in ranks) / world
        assert abs(mean - losses[i]) < 2e-4 * losses[i]
        for r in ranks:
            assert abs(r[1][i] - norms[i]) <= norm_bound * norms[i], (r[1], norms)
    for r in ranks:
        for k, v in params.items():
            assert abs(r[2][k] - ranks[0][2][k]).max() == 0, k                     # every rank holds the same
            assert abs(r[2][k] - v).max() < 1e-4, k                                # (a step of AdamW is 3e-4)


def test_sharded_engine_with_context_parallelism():
    """Ranks of a sequence's parts hold the same parameters: gradients are averaged over them, and count once in the norm."""
    _against_one_process({"cp_size": 2}, 2, 0.5)


def test_sharded_engine_sums_partial_gradients():
    """Norm weights under sequence parallelism: every rank of the TP group has seen its own rows only."""
    _against_one_process({"dp_size": 2, "tp_size": 2, "sequence_parallel": True}, 4, 0.0)


@pytest.mark.parametrize("sp", [False, True])
def test_sharded_engine_counts_replicated_parameters_once(sp):
    """Parameters that all ranks of a TP group hold, in the global norm."""
    _against_one_process({"dp_size": 2, "tp_size": 2, "sequence_parallel": sp}, 4, 0.5)


def test_clip_by_the_norm_of_others():
    g = torch.Generator().manual_seed(0)
    ts = [torch.randn(30, generator=g), torch.randn(4, 5, generator=g)]
    own = [t.clone() for t in ts]
    norm = OF.clip_grad_norm(own, 0.5, counted=ts[:1])
    assert torch.equal(norm, OF.grad_norm(ts[:1]))
    for t, o in zip(ts, own):
        assert torch.allclose(o, t * 0.5 / (norm + 1e-6), rtol=1e-6)
    assert float(OF.clip_grad_norm(own, 0.5, counted=[])) == 0.0
    with pytest.raises(ValueError):
        OF.clip_grad_norm(own, 0.5, counted=[torch.zeros(2, dtype=torch.int32)])
    with pytest.raises(ValueError):
        OF.clip_grad_norm(own, 0.5, counted=[torch.zeros(2, device="meta")])


def test_clip_refuses_memory_that_overlaps():
    """As on the GPU, where two entries that share memory would be scaled once or twice, as it comes."""
    a, b, buf = torch.ones(100), torch.ones(50), torch.zeros(200)
    for ts, out in (([a, b, a], None), ([a[:60], a[40:]], None), ([a, b], [buf[:100], buf[60:110]]), ([a[:50], a[50:]], [a[50:], a[:50]]), ([a[:99], b], [a[1:], buf[:50]])):
        with pytest.raises(ValueError):
            OF.clip_grad_norm(ts, 1e-3, out=out)
    assert (a == 1).all() and (b == 1).all() and (buf == 0).all()
    OF.clip_grad_norm([a[:50], a[50:], b, a[:0], a[:0]], 1.0)
    OF.clip_grad_norm([a, b], 1.0, out=[a, b])
    # columns of one matrix lie between each other, and share nothing
    m = torch.ones(10, 4)
    norm = OF.clip_grad_norm([m[:, :2], m[:, 2:]], 1.0)
    assert abs(float(norm) - 40 ** 0.5) < 1e-5 and torch.allclose(m, torch.full((10, 4), 40 ** -0.5))


@pytest.mark.parametrize("bad", [[torch.ones(3), None], [None], [1.0]])
def test_gradients_that_are_missing_are_refused(bad):
    with pytest.raises(ValueError):
        OF.grad_norm(bad)
    with pytest.raises(ValueError):
        OF.clip_grad_norm(bad, 1.0)


def test_positions_beyond_32_bits():
    cos, sin = ref.rope_tables(8, 16)
    x = torch.randn(1, 3, 1, 8, generator=torch.Generator().manual_seed(0))
    y = OF.rope_axes(x, cos, sin, torch.tensor([[1, 2 ** 32 + 1, -2 ** 32]]), [0] * 4)
    assert torch.isfinite(y[:, 0]).all() and torch.isnan(y[:, 1:]).all()


@pytest.mark.parametrize("kw", [dict(softcap=1e-45), dict(softcap=1e-50), dict(softcap=1e39), dict(scale=1e-46), dict(scale=1e39)])
def test_numbers_that_32_bits_do_not_hold_are_refused(kw):
    """A cap that became zero would be no cap at all."""
    q = torch.zeros(1, 4, 2, 8)
    with pytest.raises(ValueError):
        OF.masked_attention(q, q, q, **kw)
