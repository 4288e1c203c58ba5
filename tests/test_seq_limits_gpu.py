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


@pytest.mark.parametrize("family", ["SharedBottom", "MMOE", "PLE", "Star", "HamurSmall", "HamurLarge", "M3oE"])
def test_every_model_that_looks_up_through_the_embedding_layer(family):
    """An attention-pooled history in each of them: a step runs and every parameter of the block gets a gradient."""
    from scenario_wise_rec import _hip as H
    from scenario_wise_rec.basic.features import SequenceFeature, SparseFeature
    from scenario_wise_rec.models import multi_domain as md
    from scenario_wise_rec.trainers import CTRTrainer
    D, B = 3, 300
    feats = [SparseFeature("s0", 17, 16), SequenceFeature("h", 60, 16, pooling="attention", padding_idx=0, attention={"n_heads": 2, "max_distance": 16}),
             SparseFeature("s1", 900, 16), SequenceFeature("m", 30, 16, pooling="mean", padding_idx=0)]
    deep = {"expert_params": {"dims": [16]}, "tower_params": {"dims": [8]}}
    torch.manual_seed(3)
    model = {"SharedBottom": lambda: md.SharedBottom(feats, domain_num=D, bottom_params={"dims": [32]}, tower_params={"dims": [8]}),
             "MMOE": lambda: md.MMOE(feats, domain_num=D, n_expert=2, **deep),
             "PLE": lambda: md.PLE(feats, domain_num=D, n_level=1, n_expert_specific=2, n_expert_shared=1, **deep),
             "Star": lambda: md.Star(feats, D, [32, 16], [16]),
             "HamurSmall": lambda: md.HamurSmall(feats, D, [32, 16], [16], 8),
             "HamurLarge": lambda: md.HamurLarge(feats, D, [32, 16, 16, 16, 16, 16, 16], [16], 8),
             "M3oE": lambda: md.M3oE(feats, domain_num=D, fcn_dims=[32, 16, 16, 8], expert_num=2, exp_d=1, exp_t=1, bal_d=1, bal_t=1, device="cuda")}[family]()
    with torch.no_grad():
        for n, w in model.named_parameters():
            if "embed_dict" in n or "position" in n:
                w.normal_(0, 0.3)
    trainer = CTRTrainer(model, "attention", optimizer_params={"lr": 1e-3, "weight_decay": 1e-5}, device="cuda")
    model.train()
    g = torch.Generator(device="cuda")
    g.manual_seed(4)
    ids = lambda hi, *s: torch.randint(0, hi, s, generator=g, device="cuda")
    x = {"s0": ids(17, B), "s1": ids(900, B), "h": ids(60, B, 9), "m": ids(30, B, 4), "domain_indicator": ids(D, B)}
    y = (torch.rand(B, generator=g, device="cuda") < 0.3).float()
    model.zero_grad()
    trainer.criterion(model(x), y).backward()
    for n, w in model.named_parameters():
        if "seq_blocks" in n:
            assert w.grad is not None and torch.isfinite(w.grad).all() and w.grad.any(), n
    trainer.train_step(x, y)
    H.check_errors()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("aligned", [True, False])
@pytest.mark.parametrize("D", [4, 16, 20, 33, 64, 128])
def test_hidden_keys_and_rows_in_use_at_every_width(D, aligned, causal, dtype):
    """A padded batch with hidden keys, unused rows behind q_len and NaN in all of them, walked in one and in several rounds, in every width's
    kernels and for rows off every alignment."""
    from scenario_wise_rec import _hip as H
    from scenario_wise_rec import ops
    B, L, Hq, Hk = 3, 150, 4, 2
    used = [150, 97, 0]
    lens, at = torch.tensor(used, dtype=torch.int32, device="cuda"), [0, 150, 300]
    mask = torch.rand(B * L, generator=torch.Generator("cuda").manual_seed(8), device="cuda") < 0.6
    mask[:40] = False                                  # (causal: the first rows see nothing)
    unused = torch.cat([torch.arange(L, device="cuda") >= n for n in used])
    def rows(seed, heads):
        t = randn(seed, B * L, heads, D, dtype=dtype)
        if not aligned:
            wide = torch.empty(B * L * heads * (D + 1) + 1, dtype=dtype, device="cuda")[1:].view(B * L, heads, D + 1)[..., :D]
            t = wide.copy_(t)
        return t
    q, k, v, dout = rows(1, Hq), rows(2, Hk), rows(3, Hk), rows(4, Hq)
    for t in (q, dout):
        t[unused] = float("nan")
    for t in (k, v):
        t[unused | ~mask] = float("nan")
    bias, table = randn(5, Hq, 8), ops.seq_buckets(8, 30, causal)
    want = ref.attention(q, k, v, dout, used, used, at, at, causal, None, bias, table, mask)
    for hint in (150, 1):
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v, bias)]
        out = ops.seq_attention(*leaves[:3], torch.tensor([0, 150, 300, 450], dtype=torch.int32, device="cuda"), max_q=hint, causal=causal,
                                bias=leaves[3], buckets=table, key_mask=mask, q_len=lens)
        got = dict(zip(("out", "dq", "dk", "dv", "dbias"), (out.detach(),) + torch.autograd.grad(out, leaves, dout)))
        for n, t in got.items():
            ref.check(t, want[n], f"{n} hint {hint}")
    H.check_errors()


@pytest.mark.parametrize("D", [16, 64, 128])
def test_bias_gradient_of_fp32_has_no_drift_over_many_rows(D):
    """The score gradients of a causal row cancel, so the bias gradient's sum over all buckets is zero, and what is left of it is the sum of
    the rows' rounding errors.  Each is the error of do . v, weighted by p, and of do . o: both at most 6 D / 16 accumulator steps of 2^-24 of
    sum |do||v|, uniform in that half step (2^-24 / sqrt 3).  Without a common sign T rows add up to sqrt(T) of it; 4 of these standard
    deviations are allowed.  A rounding of one sign adds up to T of it."""
    from scenario_wise_rec import ops
    n, L, H = (16384, 50, 2) if D < 128 else (4096, 100, 2)
    T = n * L
    q, k, v, dout = (randn(10 + i, T, H, D) for i in range(4))
    bias, table = randn(15, H, 8).mul_(0.5), ops.seq_buckets(8, 40)
    leaves = [t.requires_grad_(True) for t in (q, k, v, bias)]
    out = ops.seq_attention(*leaves[:3], torch.arange(0, T + 1, L, dtype=torch.int32, device="cuda"), max_q=L, bias=bias, buckets=table)
    drift = torch.autograd.grad(out, leaves, dout)[3].double().sum(1)
    size = D * float(dout.abs().mean()) * float(v.detach().abs().mean())
    row = 2 * (6 * D / 16) ** 0.5 * 2.0 ** -24 / 3 ** 0.5 * size
    assert (drift.abs() <= 4 * T ** 0.5 * row).all(), (drift.tolist(), 4 * T ** 0.5 * row)
