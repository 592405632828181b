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
