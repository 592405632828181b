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
