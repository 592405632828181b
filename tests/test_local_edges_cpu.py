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


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_rows_alone_are_cast_without_gradients(dtype, monkeypatch):
    """The same values with and without a gradient, and no copy of the table in another type where none is asked for."""
    from lightron_b200.ops import reference as ref
    w = torch.randn(11, 6, generator=torch.Generator().manual_seed(1)).to(dtype).requires_grad_()
    tokens = torch.tensor([[3, 4, 13], [2, 9, 3]])
    want = OF.scaled_embedding(tokens, w, 1.7, 3)
    gather, tables = ref.F.embedding, []
    monkeypatch.setattr(ref.F, "embedding", lambda i, t: tables.append(t) or gather(i, t))
    with torch.no_grad():
        assert torch.equal(OF.scaled_embedding(tokens, w, 1.7, 3), want)
    assert torch.equal(OF.scaled_embedding(tokens, w.detach(), 1.7, 3), want)
    assert len(tables) == 2 and all(t.dtype == dtype and t.data_ptr() == w.data_ptr() for t in tables)


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


@pytest.mark.parametrize("B,S,hq,hkv,d,window,sinks", [
    (4, 8192, 32, 32, 128, 256, 4096), (1, 32768, 32, 8, 128, 512, 4096), (1, 65536, 32, 8, 128, 128, 4096), (1, 131072, 32, 8, 128, 128, 8192), (4, 8192, 32, 8, 128, 128, 4096),
    (8, 8192, 32, 8, 128, 1024, 1024), (1, 8192, 32, 8, 128, 128, 1024), (32, 2048, 32, 32, 128, 512, 4), (1024, 256, 32, 32, 128, 64, 4), (1, 131072, 32, 8, 128, 4096, 4096),
    (3, 130000, 1, 1, 8, 5, 2), (1, 2000, 16, 1, 64, 40, 300), (1, 500, 4, 2, 64, 130, 130), (2, 129, 1, 1, 8, 1, 1), (7, 128, 4, 4, 64, 5, 1), (5, 1, 4, 4, 64, 1, 0),
])
@pytest.mark.parametrize("masked,causal", [(False, True), (True, True), (False, False), (True, False)])
def test_workspace_of_pieces_has_a_bound(B, S, hq, hkv, d, window, sinks, masked, causal):
    """What pieces of walks leave, for dK and dV together, takes no more than dQ's sums or 64 MB, however many sinks there are; the list itself 28 bytes a key block and 16 a piece."""
    size, fixed = _window_bytes(B, S, hq, hkv, d, window, sinks, masked, causal=causal)
    blocks = B * -(-S // 128)
    most = max(fixed, 1 << 26)
    assert 0 <= size - fixed <= most + 28 * blocks + 16 * (most // (2 * 4 * 128 * 64 * hkv) + 1) + 16


def test_workspace_without_a_mask_is_what_is_used():
    """1 x 8192 with a window of 1024 and four sinks: the sinks' walk of 256 blocks in eight pieces at most of each of 8 heads, nothing else."""
    size, fixed = _window_bytes(1, 8192, 32, 8, 128, 1024, 4, masked=False)
    assert size - fixed in [2 * n * 8 * 128 * 128 * 4 + 16 * (64 + n - 1) + 12 * 64 + 16 for n in range(2, 9)]


def test_walks_are_no_longer_than_the_plan_of_the_pieces_takes_them_for():
    """Query blocks that see a key block, counted, against the bound that sizes lists without a mask: blocks of sinks may be seen by all, others by the window's span."""
    for Sq, Sk, window, sinks, causal in [(700, 700, 1, 0, True), (700, 700, 130, 4, True), (700, 700, 129, 200, True), (600, 700, 64, 3, True), (601, 900, 257, 0, True), (700, 700, 130, 4, False),
                                          (640, 640, 1, 0, False), (500, 900, 300, 129, False), (129, 1000, 128, 1, True)]:
        off = Sk - Sq
        at, key = torch.arange(Sq)[:, None] + off, torch.arange(Sk)[None]
        see = ((at - key).abs() < window) | (key < sinks)
        if causal:
            see &= key <= at
        span = 128 + (1 if causal else 2) * (window - 1)
        near = min(-(-span // 128) + (1 if off % 128 or not causal else 0), -(-Sq // 128))
        for n0 in range(0, Sk, 128):
            rows = see[:, n0:n0 + 128].any(1).nonzero()
            walk = 0 if not len(rows) else int(rows[-1]) // 128 - int(rows[0]) // 128 + 1
            assert walk <= (-(-Sq // 128) if n0 < sinks else near)


# ---- figures of a run ------------------------------------------------------------------------------


@pytest.mark.parametrize("S,window,sinks,freq", [(64, 16, 0, 0), (64, 16, 3, 2), (64, 16, 60, 0), (64, 1, 5, 3), (64, 64, 2, 0), (64, 200, 0, 0), (50, 49, 1, 0), (64, None, 0, 0)])
def test_operations_of_a_step_count_visible_keys(S, window, sinks, freq):
    from lightron_b200.config import ModelArgs
    args = ModelArgs(dim=32, n_heads=4, n_layers=4, vocab_size=64, attn_window=window, attn_sinks=sinks, attn_global_freq=freq)
    keys = 0.0
    for layer in range(4):
        w = args.window_of(layer)
        if w is None or w >= S:
            keys += S / 2
        else:
            keys += sum(1 for i in range(S) for j in range(i + 1) if i - j < w or j < sinks) / S
    assert args.flops_per_token(S) == pytest.approx(6.0 * args.num_active_params() + 12.0 * 32 * keys, rel=1e-12)
    if window is None:
        assert args.flops_per_token(S) == 6.0 * args.num_active_params() + 6.0 * 4 * 32 * S


def test_logged_mfu_counts_the_window(tmp_path):
    import json
    from lightron_b200 import mesh
    from lightron_b200.config import parse_config
    from lightron_b200.trainer import Trainer
    mesh.set_context(None)
    log = tmp_path / "run.jsonl"
    raw = {"distributed": {}, "model": {"name": "tiny", "attn_window": 16, "attn_sinks": 2, "attn_global_freq": 4}, "dataset": {"name": "synthetic"},
           "training": {"micro_batch_size": 1, "gradient_accumulation_steps": 1, "seq_length": 128, "learning_rate": 3e-4, "total_steps": 1, "seed": 0, "dtype": "fp32", "log_interval": 1,
                        "jsonl_log": str(log), "save_interval": 0, "save_final": False}}
    tr = Trainer(parse_config(raw, env={}))
    tr.fit()
    mesh.set_context(None)
    row = json.loads(log.read_text().splitlines()[-1])
    keys = 64 + 3 * sum(1 for i in range(128) for j in range(i + 1) if i - j < 16 or j < 2) / 128
    want = (6.0 * tr.args.num_active_params() + 12.0 * tr.args.dim * keys) * row["tokens_per_s_device"] / (row["mfu_peak_tflops"] * 1e12)
    assert row["mfu"] == pytest.approx(want, rel=1e-9)


@pytest.mark.parametrize("B,hq,hkv,d", [(8, 32, 8, 128), (8, 32, 8, 64), (1, 32, 4, 128)])
@pytest.mark.parametrize("S", [2048, 4095, 4096, 20000])
def test_single_tokens_are_split_alike_where_the_cache_fills_the_window(B, hq, hkv, d, S):
    """The heads of a group as a tile's rows, and walks split over keys, for a window of all keys as for one that is a key short of them."""
    lib = _library()
    size = [lib.lb_window_attn_fwd_ws_bytes(B, 1, S, hq, hkv, d, 1, window, 0) for window in (S - 1, S, S + 1, 1 << 30)]
    assert size[0] > 0 and size == size[:1] * 4


def test_many_queries_take_a_window_over_all_keys_as_none():
    lib = _library()
    for S, Sq in ((700, 700), (9000, 300), (20000, 128), (40000, 100)):
        assert lib.lb_window_attn_fwd_ws_bytes(1, Sq, S, 8, 2, 64, 1, S, 3) == lib.lb_masked_attn_fwd_ws_bytes(1, Sq, S, 8, 2, 64)
        assert lib.lb_window_attn_bwd_ws_bytes(1, Sq, S, 8, 2, 64, 1, S, 3, 0) == lib.lb_masked_attn_bwd_ws_bytes(1, Sq, S, 8, 2, 64, 1)
