"""Operators of local attention at the borders of what they take, on the CPU: sizes that kernels count in 32 bits, workspaces, figures of a run."""
import pytest
import torch

from lightron_b200.ops import functional as OF
from lightron_b200.ops import native

SHAPE = -3


def _library():
    lib = native._load()
    if lib is None:
        pytest.skip("native library not built")
    return lib


@pytest.mark.parametrize("H", [(1 << 30) + 1, (1 << 31) - 256, (1 << 31) - 3, (1 << 31) - 1])
def test_rows_past_30_bits_are_refused_by_the_library(H):
    """Columns are counted in 32 bits and in steps: a count that passes them would begin again below zero.  (Null pointers: nothing could be launched.)"""
    lib = _library()
    assert lib.lb_embed_scaled(0, 8, 0, 0, 1, H, 0, 1, 1.0, 0) == SHAPE
    assert lib.lb_embed_sorted_ws_bytes(1, H) == 0
    assert lib.lb_embed_sorted_bwd(0, 8, 0, 0, 0, 1 << 62, 1, H, 0, 1, 1.0, 0) == SHAPE
    assert lib.lb_embed_scaled(0, 8, 0, 0, 1, 1 << 30, 0, 1, 1.0, 0) == -1 and lib.lb_embed_sorted_ws_bytes(1, 1 << 30) > 1 << 33


@pytest.mark.parametrize("H", [(1 << 30) + 1, (1 << 31) - 3])
def test_rows_past_30_bits_are_refused(H, monkeypatch):
    def call(name, *args):
        raise AssertionError(f"{name} was launched")
    monkeypatch.setattr(native, "use_native", lambda t: True)
    monkeypatch.setattr(native, "host_ops", lambda: None)
    monkeypatch.setattr(native, "call", call)
    monkeypatch.setattr(torch.Tensor, "contiguous", lambda t, *a, **kw: t)      # (one number stands for all of them)
    with pytest.raises(ValueError, match="columns"):
        OF.scaled_embedding(torch.zeros(1, dtype=torch.long), torch.zeros(1, 1).expand(1, H))


# ---- the windowed backward's workspace -------------------------------------------------------------


def _window_bytes(B, S, hq, hkv, d, window, sinks, masked, Sq=None, causal=True):
    """(bytes of the workspace, of the row statistics and dQ's sums in it)."""
    Sq = S if Sq is None else Sq
    rows = B * hq * -(-Sq // 128) * 128
    return _library().lb_window_attn_bwd_ws_bytes(B, Sq, S, hq, hkv, d, int(causal), window, sinks, int(masked)), 4 * rows * (2 + (-(-d // 32) * 32 if S > 128 else 0))


def test_workspace_of_a_mask_is_its_own():
    """Packed documents do not pay for the pieces of a call without a mask, whose sinks are seen by all queries."""
    size, fixed = _window_bytes(4, 8192, 32, 32, 128, 256, 4096, masked=True)
    assert size - fixed < 1 << 29
    size, fixed = _window_bytes(4, 8192, 32, 8, 128, 128, 4096, masked=True)
    assert size - fixed < 1 << 28
