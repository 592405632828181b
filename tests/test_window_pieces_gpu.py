"""The windowed backward where walks of sinks are cut into pieces, where they are not, and where pieces go head by head: several heads of keys, against 64 bits, the same bits in every run."""
import pytest
import torch

from packed_oracle import rel
from test_window_gpu import _check, _inputs, _run, _status_ok

pytestmark = pytest.mark.gpu


def _again(B, S, hq, hkv, d, window, sinks, causal=True):
    t = _inputs(B, S, S, hq, hkv, d)
    runs = [_run(*t, causal=causal, window=window, sinks=sinks) for _ in range(2)]
    assert all(torch.equal(runs[0][i], runs[1][i]) for i in (0, 2, 3)) and rel(runs[0][1], runs[1][1]) < 2e-3
    return runs[0]


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("S,hq,hkv,window,sinks", [
    (4700, 16, 8, 1000, 4), (4700, 16, 8, 1000, 200), (4800, 8, 8, 1500, 4), (4700, 16, 8, 300, 4), (4700, 16, 8, 300, 200), (4700, 8, 8, 128, 900), (3800, 10, 10, 2000, 130),
])
def test_pieces_of_several_key_heads(S, hq, hkv, window, sinks, d):
    """More key blocks over heads than two for each SM.  With long windows and few sinks pieces go head by head, all of one head of keys before the next one's."""
    got = _check(1, S, S, hq, hkv, d, window, sinks)
    again = _again(1, S, hq, hkv, d, window, sinks)
    assert all(torch.equal(got[i], again[i]) for i in (0, 2, 3))


@pytest.mark.parametrize("B,S,hq,hkv,d,window,sinks,causal,docs", [
    (2, 2500, 8, 8, 64, 600, 4, True, 0), (3, 1700, 16, 8, 128, 400, 3, True, 0), (2, 2500, 8, 8, 64, 600, 4, True, 900), (1, 4700, 16, 8, 64, 500, 4, True, 2500), (1, 4700, 8, 8, 64, 700, 130, False, 0),
    (12, 600, 8, 8, 64, 130, 5, True, 200), (12, 600, 8, 8, 64, 130, 5, True, 600),
])
def test_pieces_of_several_sequences(B, S, hq, hkv, d, window, sinks, causal, docs):
    _check(B, S, S, hq, hkv, d, window, sinks, causal=causal, docs=docs)
    _again(B, S, hq, hkv, d, window, sinks, causal)


def test_memory_of_many_sinks():
    """The backward's memory at a short window and many sinks: gradients, dQ's sums and no more than as much again."""
    q, k, v, do = _inputs(2, 8192, 8192, 8, 8, 64)
    _run(q, k, v, do, window=128, sinks=2048)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    _run(q, k, v, do, window=128, sinks=2048)
    _status_ok()
    n = q.numel()
    # o, what its rounding left, dq, dk, dv in bf16; lse and two row statistics in fp32; dQ's sums, and what pieces leave
    assert torch.cuda.max_memory_allocated() - before < 10 * n + 12 * n // 64 + 4 * n + max(4 * n, 1 << 26) + (8 << 20)


@pytest.mark.parametrize("B,S,hq,hkv,d,window,sinks,causal", [
    (6, 700, 16, 16, 64, 600, 4, True), (8, 600, 16, 8, 64, 100, 3, True), (4, 900, 16, 16, 64, 300, 700, True), (8, 513, 12, 12, 128, 500, 0, True), (3, 2000, 8, 8, 64, 64, 1500, True),
    (4, 1000, 12, 12, 64, 100, 900, False),
])
def test_whole_walks_in_their_order(B, S, hq, hkv, d, window, sinks, causal):
    """Nothing cut: key blocks sorted by their walks, head by head or those of the sinks ahead of all heads."""
    _check(B, S, S, hq, hkv, d, window, sinks, causal=causal)
    _again(B, S, hq, hkv, d, window, sinks, causal)
