"""Local attention in the model on the GPU: the fused projection with norms and windows, and a training step through everything, against 64 bits.

Bounds.  Attention: 5e-3 in the 2-norm as in its own tests (one rounding each of P, dS and the result); with norms queries and keys are rounded once more before it and their gradients once
between the two (1.7e-3 each), in quadrature within 6e-3.
"""
import pytest
import torch

from local_oracle import local, norm_rope64
from packed_oracle import attention64, documents, rel

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def _rand(*shape, scale=1.0, seed=0, dtype=BF16):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32) * scale).to(dtype)


@pytest.mark.parametrize("B,S,hq,hkv,d,window,sinks,docs,cap", [
    (2, 300, 4, 2, 64, 50, 3, 0, 0.0), (2, 500, 8, 2, 128, 130, 4, 200, 0.0), (1, 257, 6, 3, 96, None, 0, 0, 20.0), (3, 1, 4, 1, 64, 5, 1, 0, 0.0), (1, 700, 4, 4, 64, 64, 130, 0, 30.0),
])
def test_fused_projection_with_norms(B, S, hq, hkv, d, window, sinks, docs, cap):
    from lightron_b200.ops import functional as OF
    from lightron_b200.ops import native, reference as ref
    qkv = _rand(B * S, (hq + 2 * hkv) * d, seed=1)
    wq, wk = ((1 + _rand(d, scale=0.3, seed=2 + i, dtype=torch.float32)).to(BF16) for i in range(2))
    cos, sin = ref.rope_tables(d, S + 7, device="cuda")
    ids = documents(B, S, docs, seed=3) if docs else None
    mask = None if ids is None else OF.attention_mask(documents=ids.cuda())
    pos = torch.arange(S, device="cuda", dtype=torch.int32).expand(B, S) + torch.arange(B, device="cuda", dtype=torch.int32)[:, None]
    do = _rand(B * S, hq * d, seed=4)
    ins = [t.detach().requires_grad_() for t in (qkv, wq, wk)]
    kw = dict(mask=mask, softcap=cap, window=window, sinks=sinks, norm_eps=1e-6)
    o = OF.packed_attention_qkv(ins[0], cos, sin, pos, B, S, hq, hkv, d, q_norm=ins[1], k_norm=ins[2], **kw)
    grads = torch.autograd.grad(o, ins, do)
    assert torch.equal(ins[0], qkv)                                # with norms the projection's output stays
    # the two operators one after the other: the same bits, but for dq's order of sums
    heads = qkv.view(B, S, -1, d)
    parts = [heads[:, :, :hq].detach().requires_grad_(), heads[:, :, hq:hq + hkv].detach().requires_grad_(), heads[:, :, hq + hkv:].detach().requires_grad_(), ins[1], ins[2]]
    tq, tk = OF.qk_norm_rope(parts[0], parts[1], ins[1], ins[2], cos, sin, positions=pos, eps=1e-6)
    apart = OF.masked_attention(tq, tk, parts[2], mask=mask, softcap=cap, window=window, sinks=sinks)
    assert torch.equal(apart.reshape(o.shape), o)
    two = torch.autograd.grad(apart, parts, do.view(B, S, hq, d))
    assert torch.equal(grads[0].view(B, S, -1, d)[:, :, hq:], torch.cat((two[1], two[2]), dim=2)) and torch.equal(grads[2], two[4])
    assert native.device_status() == {}
    # 64 bits
    e = [t.detach().double().requires_grad_() for t in parts]
    at = pos[None]
    axes = [0] * (d // 2)
    zq, zk = norm_rope64(e[0], e[3], cos, sin, at, axes, 1e-6), norm_rope64(e[1], e[4], cos, sin, at, axes, 1e-6)
    see = local(B, S, S, True, window or S, sinks, ids)
    o64, dq64, dk64, dv64 = attention64(zq, zk, e[2], see, d ** -0.5, cap, None, do.view(B, S, hq, d))
    want = torch.autograd.grad((zq, zk), (e[0], e[1], e[3], e[4]), (dq64, dk64))
    assert rel(o, o64.reshape(o.shape)) < 6e-3
    if S > 1:
        got = grads[0].view(B, S, -1, d)
        for g, w in ((got[:, :, :hq], want[0]), (got[:, :, hq:hq + hkv], want[1]), (got[:, :, hq + hkv:], dv64)):
            assert rel(g, w) < 6e-3


def _models(**kw):
    from lightron_b200 import mesh
    from lightron_b200.config import ModelArgs
    from lightron_b200.models import LightronTransformer, init_weights
    mesh.set_context(None)
    args = ModelArgs(dim=256, n_layers=3, n_heads=4, n_kv_heads=2, vocab_size=512, intermediate_size=512, max_seq_len=512, **kw)
    gpu = LightronTransformer(args, dtype=BF16, device="cuda")
    init_weights(gpu, 0, std=0.05)
    exact = LightronTransformer(args, dtype=torch.float64, device="cpu")
    exact.load_state_dict({k: v.double().cpu() for k, v in gpu.state_dict().items()})
    return gpu, exact


@pytest.mark.parametrize("kw", [dict(attn_window=100, attn_sinks=3, qk_norm=True, embed_scale=16.0, attn_global_freq=3), dict(attn_window=64, attn_softcap=20.0), dict(qk_norm=True, embed_scale=4.0)])
def test_training_step(kw):
    """Loss and gradients of a packed batch.  A model of three layers in bf16 rounds some dozen times (2^-9 of a value each in the mean) between its loss and its first weights, in quadrature
    below 2e-2 of a gradient's 2-norm."""
    from lightron_b200.ops import functional as OF, native
    gpu, exact = _models(**kw)
    tokens = torch.randint(0, 512, (2, 400), generator=torch.Generator().manual_seed(1))
    ids = documents(2, 400, 150, seed=5)
    targets = torch.where(ids >= 0, tokens.roll(-1, 1), -100)
    n = int((targets >= 0).sum())
    want = exact.loss(tokens, targets, mask=OF.attention_mask(documents=ids), n_tokens=n)
    want.backward()
    loss = gpu.loss(tokens.cuda(), targets.cuda(), mask=OF.attention_mask(documents=ids.cuda()), n_tokens=n)
    loss.backward()
    assert native.device_status() == {}
    assert abs(float(loss.detach()) - float(want.detach())) < 1e-2 * float(want.detach())
    exact_grads = dict(exact.named_parameters())
    for name, p in gpu.named_parameters():
        g, w = p.grad.double().cpu(), exact_grads[name].grad
        cos = float((g * w).sum() / (g.norm() * w.norm()))
        assert cos > 0.99, (name, cos)


def test_single_tokens_continue_a_sequence():
    """A cache that grows token by token, norms and rotation at each token's place: the rows of the whole sequence."""
    from lightron_b200.ops import functional as OF
    from lightron_b200.ops import reference as ref
    B, S, hq, hkv, d, window, sinks = 2, 40, 8, 2, 64, 9, 2
    q, k, v = _rand(B, S, hq, d, seed=1), _rand(B, S, hkv, d, seed=2), _rand(B, S, hkv, d, seed=3)
    wq, wk = _rand(d, seed=4), _rand(d, seed=5)
    cos, sin = ref.rope_tables(d, S, device="cuda")
    with torch.no_grad():
        tq, tk = OF.qk_norm_rope(q, k, wq, wk, cos, sin)
        whole = OF.masked_attention(tq, tk, v, window=window, sinks=sinks)
        cache = torch.zeros(B, S, hkv, d, dtype=BF16, device="cuda")
        for i in range(S):
            at = torch.full((B, 1), i, dtype=torch.int32, device="cuda")
            one_q, one_k = OF.qk_norm_rope(q[:, i:i + 1], k[:, i:i + 1], wq, wk, cos, sin, positions=at)
            assert torch.equal(one_q, tq[:, i:i + 1]) and torch.equal(one_k, tk[:, i:i + 1])
            cache[:, i:i + 1] = one_k
            o = OF.masked_attention(one_q, cache[:, :i + 1], v[:, :i + 1], window=window, sinks=sinks)
            assert rel(o, whole[:, i:i + 1]) < 5e-3
