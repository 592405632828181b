"""Operators of local attention at the borders of what they take, on the GPU."""
import pytest
import torch

from lightron_b200.ops import reference as ref

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def _rand(*shape, scale=1.0, seed=0, dtype=BF16):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32) * scale).to(dtype)


@pytest.mark.parametrize("axes", [None, [0] * 16 + [1] * 16])
@pytest.mark.parametrize("shape", [(), (5,), (2, 2, 2, 4)])
def test_positions_of_no_shape_that_is_taken_are_refused(axes, shape):
    from lightron_b200.ops import functional as OF
    q, k, w = _rand(2, 4, 2, 64), _rand(2, 4, 1, 64), _rand(64)
    cos, sin = ref.rope_tables(64, 8, device="cuda")
    with pytest.raises(ValueError):
        OF.qk_norm_rope(q, k, w, w, cos, sin, positions=torch.zeros(shape, dtype=torch.int32, device="cuda"), axes=axes)


# ---- few queries, and windows that hold all keys ---------------------------------------------------


@pytest.mark.parametrize("B,Sq,Sk,hq,hkv,d", [
    (2, 1, 3000, 8, 2, 64), (1, 1, 2048, 32, 1, 128), (20, 1, 130, 8, 2, 128), (40, 1, 1, 4, 1, 64), (5, 40, 40, 32, 8, 64), (10, 64, 300, 16, 8, 128), (3, 31, 2500, 12, 3, 96), (50, 3, 77, 6, 3, 8),
    (3, 1, 2600, 12, 2, 64), (40, 65, 200, 8, 2, 64),
])
@pytest.mark.parametrize("cap,slopes", [(0.0, False), (20.0, False), (0.0, True), (90.0, True)])
@pytest.mark.parametrize("how", ["causal", "both", "documents"])
def test_few_queries_under_a_window_over_all_keys(B, Sq, Sk, hq, hkv, d, cap, slopes, how):
    """One key short of all, all, and more: against 64 bits, with and without gradients (5e-3 in the 2-norm, as in the tests of the window), the two that hold all keys with the same bits."""
    from lightron_b200.ops import functional as OF, native
    from local_oracle import local
    from packed_oracle import attention64, documents, rel
    q, k, v, do = _rand(B, Sq, hq, d, scale=2.0 if cap else 1.0, seed=1), _rand(B, Sk, hkv, d, seed=2), _rand(B, Sk, hkv, d, seed=3), _rand(B, Sq, hq, d, seed=4)
    ids = documents(B, Sk, max(Sk // 2, 2), seed=5) if how == "documents" else None
    causal = how != "both"
    kw = dict(softcap=cap, slopes=torch.linspace(0.0, 0.3, hq, device="cuda") if slopes else None)
    if ids is None:
        kw["causal"] = causal
    else:
        kw["mask"] = OF.attention_mask(documents=ids.cuda())
    runs, wants = [], []
    for window, sinks in ((max(Sk - 1, 1), 1), (Sk, 0), (Sk + 1, 7)):
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        o = OF.masked_attention(*leaves, window=window, sinks=sinks, **kw)
        with torch.no_grad():
            alone = OF.masked_attention(q, k, v, window=window, sinks=sinks, **kw)
        runs.append((o.detach(), alone, *torch.autograd.grad(o, leaves, do)))
        wants.append(attention64(q, k, v, local(B, Sq, Sk, causal, window, sinks, ids), d ** -0.5, cap, kw["slopes"], do))
    assert native.device_status() == {}
    for run, want in zip(runs, wants):
        for name, g, w in zip(("o", "alone", "dq", "dk", "dv"), run, (want[0], *want)):
            assert torch.isfinite(g).all(), name
            if name not in ("dq", "dk") or Sk > 1:           # (one key: no gradient by its score)
                assert rel(g, w) < 5e-3, (name, rel(g, w))
    assert all(torch.equal(runs[1][i], runs[2][i]) for i in (0, 1, 3, 4)) and (Sk == 1 or rel(runs[1][2], runs[2][2]) < 2e-3)
