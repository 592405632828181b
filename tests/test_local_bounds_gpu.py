"""Gradients of a whole model with local attention, and of the norms' weights through the fused projection, by their distance to 64 bits.

Bounds.  A rounding to bf16 is 1.7e-3 in the 2-norm.  Weights of the norms in the fused projection: their terms have what dq or dk has (up to 2.7e-3), its rounding between the two operators, that of the
turned queries and keys ahead, and the sum is rounded once: in quadrature 4e-3, within 6e-3.

A step of three layers rounds some dozen times a layer between its loss and its first weights: an activation or its gradient is off by e = sqrt(36) * 1.7e-3 = 1e-2.  A weight's gradient is a sum of
products of the two: sqrt(2) e = 1.4e-2, within 2e-2.  Queries and keys have more: dq is a sum over keys of P (do.v - D) k, in which do, v and k are off by e each, and P by what its score is off, which is
the product of a query and a key that are off by e each, sqrt(2) e of a score, and scores of normed heads have a standard deviation of 1: sqrt(1 + 1 + 1 + 2) e = 2.2e-2, within 3e-2, for the
projections of queries and keys and the weights of their norms.  A gradient without a scale, or counted twice, is off by 0.5 or more.
"""
import pytest
import torch

from local_oracle import local, norm_rope64
from packed_oracle import attention64, documents, rel
from test_local_model_gpu import _models, _rand

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


@pytest.mark.parametrize("kw", [dict(attn_window=100, attn_sinks=3, qk_norm=True, embed_scale=16.0, attn_global_freq=3), dict(attn_window=64, attn_softcap=20.0), dict(qk_norm=True, embed_scale=4.0)])
def test_gradients_of_a_training_step(kw):
    from lightron_b200.ops import functional as OF, native
    gpu, exact = _models(**kw)
    tokens = torch.randint(0, 512, (2, 400), generator=torch.Generator().manual_seed(1))
    ids = documents(2, 400, 150, seed=5)
    targets = torch.where(ids >= 0, tokens.roll(-1, 1), -100)
    n = int((targets >= 0).sum())
    exact.loss(tokens, targets, mask=OF.attention_mask(documents=ids), n_tokens=n).backward()
    gpu.loss(tokens.cuda(), targets.cuda(), mask=OF.attention_mask(documents=ids.cuda()), n_tokens=n).backward()
    assert native.device_status() == {}
    want = dict(exact.named_parameters())
    off = {name: rel(p.grad.cpu(), want[name].grad) for name, p in gpu.named_parameters()}
    for name, x in off.items():
        assert x < (3e-2 if any(part in name for part in (".wq.", ".wk.", ".q_norm.", ".k_norm.")) else 2e-2), (name, x)


@pytest.mark.parametrize("B,S,hq,hkv,d,window,sinks,docs,cap", [
    (2, 300, 4, 2, 64, 50, 3, 0, 0.0), (2, 500, 8, 2, 128, 130, 4, 200, 0.0), (1, 257, 6, 3, 96, None, 0, 0, 20.0), (1, 700, 4, 4, 64, 64, 130, 0, 30.0),
])
def test_weights_of_norms_in_the_fused_projection(B, S, hq, hkv, d, window, sinks, docs, cap):
    from lightron_b200.ops import functional as OF, native, reference as ref
    qkv = _rand(B * S, (hq + 2 * hkv) * d, seed=1)
    ins = [qkv.detach().requires_grad_(), *((1 + _rand(d, scale=0.3, seed=2 + i, dtype=torch.float32)).to(BF16).requires_grad_() for i in range(2))]
    cos, sin = ref.rope_tables(d, S, device="cuda")
    ids = documents(B, S, docs, seed=3) if docs else None
    mask = None if ids is None else OF.attention_mask(documents=ids.cuda())
    do = _rand(B * S, hq * d, seed=4)
    o = OF.packed_attention_qkv(ins[0], cos, sin, None, B, S, hq, hkv, d, q_norm=ins[1], k_norm=ins[2], mask=mask, softcap=cap, window=window, sinks=sinks)
    got = torch.autograd.grad(o, ins, do)
    assert native.device_status() == {}
    heads = qkv.view(B, S, -1, d).double()
    wq, wk = (t.detach().double().requires_grad_() for t in ins[1:])
    at, axes = torch.arange(S, device="cuda").expand(1, B, S), [0] * (d // 2)
    zq, zk = norm_rope64(heads[:, :, :hq], wq, cos, sin, at, axes, 1e-6), norm_rope64(heads[:, :, hq:hq + hkv], wk, cos, sin, at, axes, 1e-6)
    _, dq, dk, _ = attention64(zq, zk, heads[:, :, hq + hkv:], local(B, S, S, True, window or S, sinks, ids), d ** -0.5, cap, None, do.view(B, S, hq, d))
    for g, w in zip(got[1:], torch.autograd.grad((zq, zk), (wq, wk), (dq, dk))):
        assert rel(g, w) < 6e-3, rel(g, w)
