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


def test_many_sequences_and_one_long():
    """More workgroups than a grid takes if each sequence got the long one's: 65 536 of up to two rows, one of 2 048."""
    from scenario_wise_rec import _hip as H
    from scenario_wise_rec import ops
    B, Hq, Hk, D = 65536, 16, 4, 8
    lens = torch.ones(B, dtype=torch.int64)
    lens[::7] = 2
    lens[::11] = 0
    lens[40001] = 2048
    cu = torch.cat([torch.zeros(1, dtype=torch.int64), lens.cumsum(0)])
    T = int(cu[-1])
    q, k, v, dout = randn(3, T, Hq, D), randn(4, T, Hk, D), randn(5, T, Hk, D), randn(6, T, Hq, D)
    bias, table = randn(7, Hq, 4), torch.arange(4, dtype=torch.int32, device="cuda")
    leaves = [t.requires_grad_(True) for t in (q, k, v, bias)]
    out = ops.seq_attention(*leaves[:3], cu.to(torch.int32).cuda(), max_q=2048, bias=bias, buckets=table)
    got = dict(zip(("out", "dq", "dk", "dv", "dbias"), (out.detach(),) + torch.autograd.grad(out, leaves, dout)))
    H.check_errors()
    leaves = [t.detach() for t in leaves]
    a, n = int(cu[40001]), 2048
    some = [(a, n)] + [(int(cu[b]), int(lens[b])) for b in (0, 1, 2, 3, 7, 11, 40000, 40002, B - 2, B - 1)]
    qs, q0 = [s[1] for s in some], [s[0] for s in some]
    want = ref.attention(*leaves[:3], dout, qs, qs, q0, q0, True, None, leaves[3], table)
    for name in ("out", "dq", "dk", "dv"):
        rows = torch.cat([torch.arange(s, s + n) for s, n in some]).cuda()
        ref.check(got[name][rows], tuple(t[rows] for t in want[name]), name)
    # the short ones by hand: one row attends to itself, out = v
    one = cu[:-1][lens == 1].cuda()
    assert torch.equal(out.detach()[one], v.detach()[one].repeat_interleave(Hq // Hk, 1))
    assert torch.isfinite(got["dbias"]).all()


@pytest.mark.parametrize("hash_seed", [0, 7])
def test_attention_pooling_of_minus_one_padding(hash_seed):
    """Without a padding_idx the padding is -1, as for the other poolings: not an id, not looked up, no gradient."""
    from scenario_wise_rec import _hip as H
    from scenario_wise_rec.basic.features import SequenceFeature
    from scenario_wise_rec.basic.layers import EmbeddingLayer
    H.check_errors()

    def layer(pad):
        torch.manual_seed(1)
        f = [SequenceFeature("h", 40, 16, pooling="attention", padding_idx=pad, hash_seed=hash_seed, attention={"n_heads": 2, "max_distance": 16})]
        m = EmbeddingLayer(f)
        with torch.no_grad():
            m.embed_dict["h"].weight.normal_(0, 0.5)
        return f, m.to("cuda").train()
    g = torch.Generator(device="cuda")
    g.manual_seed(2)
    ids = torch.randint(1, 40, (30, 7), generator=g, device="cuda")
    hidden = torch.rand(30, 7, generator=g, device="cuda") < 0.4
    hidden[3] = True
    d = torch.randn(30, 16, generator=g, device="cuda")
    res = []
    for pad, value in ((0, 0), (None, -1)):                       # (id 0 is nobody's in this batch: the two mean the same)
        f, m = layer(pad)
        out = m({"h": ids.masked_fill(hidden, value)}, f, squeeze_dim=True)
        out.backward(d)
        H.check_errors()
        res.append([out.detach()] + [p.grad for p in m.parameters()])
    for a, b in zip(*res):
        assert torch.equal(a, b)
    assert not res[1][0][3].any() and torch.isfinite(res[1][0]).all()
