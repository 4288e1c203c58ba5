"""Host side of the sequence operators at their limits: forward-mode tangents, launch geometry, workspaces (nothing is launched)."""
import pytest
import torch
from torch.autograd import forward_ad


def test_forward_mode_tangents_are_refused(monkeypatch):
    """A dual tensor does not require grad: without a check its tangent would be dropped in silence."""
    from scenario_wise_rec import _hip as H, ops
    monkeypatch.setattr(H, "require_device", lambda *t: None)
    q, cu = torch.zeros(4, 2, 8, device="meta"), torch.zeros(2, dtype=torch.int32, device="meta")
    bias, table = torch.zeros(2, 4, device="meta"), torch.zeros(9, dtype=torch.int32, device="meta")
    x, w = torch.zeros(4, 8, device="meta"), torch.ones(8, device="meta")
    with forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))
        for args, kw in [((dual(q), q, q), {}), ((q, dual(q), q), {}), ((q, q, dual(q)), {}), ((q, q, q), {"bias": dual(bias), "buckets": table})]:
            with pytest.raises(NotImplementedError, match="forward-mode"):
                ops.seq_attention(*args, cu, **kw)
        for kw in ({"x": dual(x), "y": x}, {"x": x, "y": dual(x)}, {"x": x, "y": x, "gate": dual(x)}, {"x": x, "y": x, "w_post": dual(w)},
                   {"x": x, "w_pre": dual(w)}):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                ops.norm_gate_residual(**kw)
