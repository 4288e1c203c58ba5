"""Sequence operators at the limits of what their documentation allows."""
import pytest
import torch
from torch.autograd import forward_ad

import _seq_reference as ref

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


def randn(seed, *shape, dtype=F32):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def test_calls_without_tangents_inside_a_forward_mode_level():
    from scenario_wise_rec import ops
    q, cu, x = randn(1, 20, 2, 16), torch.tensor([0, 20], dtype=torch.int32, device="cuda"), randn(2, 5, 8)
    base, norm = ops.seq_attention(q, q, q, cu), ops.norm_gate_residual(x, x)
    with forward_ad.dual_level():
        assert torch.equal(base, ops.seq_attention(q, q, q, cu)) and torch.equal(norm, ops.norm_gate_residual(x, x))
        dual = forward_ad.make_dual(q, torch.ones_like(q))
        with pytest.raises(NotImplementedError):
            ops.seq_attention(dual, q, q, cu)
