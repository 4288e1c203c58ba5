"""Attention-pooled histories: SequenceBlock and SequenceFeature(pooling="attention") as models use them -- the norms, projections,
attention, bias gradient and pooling together, against the same block written in 64-bit torch."""
import math

import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu


def plain_block(p, x, seen, H, Hk, causal, buckets, eps=1e-6):
    """The block on one history, [L, dim] in 64 bits; p: its parameters by name."""
    L, dim = x.shape
    D = dim // H
    rms = lambda t: (t.square().mean(1, keepdim=True) + eps).rsqrt()
    u = x * rms(x) * p["norm_in"]
    qkv = (u @ p["qkv.weight"].t()).view(L, H + 2 * Hk, D)
    q, k, v = qkv[:, :H], qkv[:, H:H + Hk].repeat_interleave(H // Hk, 1), qkv[:, H + Hk:].repeat_interleave(H // Hk, 1)
    dist = torch.arange(L, device=x.device)[:, None] - torch.arange(L, device=x.device)[None]
    R = buckets.numel() - 1 if causal else buckets.numel() // 2
    slot = buckets[dist.clamp(0, R) if causal else dist.clamp(-R, R) + R].long()
    s = torch.matmul(q.transpose(0, 1), k.permute(1, 2, 0)) / math.sqrt(D) + p["position"][:, slot]
    ok = seen[None, :] & (dist >= 0 if causal else torch.ones_like(dist, dtype=torch.bool))
    some = ok.any(1)
    a = torch.softmax(s.masked_fill(~ok, -1e300), -1) * some[:, None]
    o = torch.matmul(a, v.transpose(0, 1)).transpose(0, 1).reshape(L, dim) @ p["out.weight"].t()
    h = F.relu(u @ p["gate.network.0.weight"].t() + p["gate.network.0.bias"])
    g = torch.sigmoid(h @ p["gate.network.2.weight"].t() + p["gate.network.2.bias"])
    return x + 2 * g * (o * rms(o) * p["norm_out"])


def make_block(dim, H, Hk, causal, seed=0):
    from scenario_wise_rec.basic.layers import SequenceBlock
    torch.manual_seed(seed)
    block = SequenceBlock(dim, H, Hk, n_buckets=8, max_distance=12, causal=causal)
    with torch.no_grad():
        for n, w in block.named_parameters():
            w.add_(0.2 * torch.randn_like(w))
    return block.to("cuda")


# Five products of at most 64 terms follow one another, each within 48 2^-24 of its magnitudes (six bf16 products per fp32 one), and the
# softmax multiplies an error of its scores by at most |s| <= 8: 5 * 48 * 8 * 2^-24 < 2^-13 of a tensor's norm.
BOUND = 2.0 ** -13


def close(a, b, what):
    b = b.double()
    assert float((a.double() - b).norm()) <= BOUND * float(b.norm()) + 1e-12, (what, float((a.double() - b).norm() / b.norm()))


@pytest.mark.parametrize("dim,H,Hk,causal", [(16, 4, 4, True), (64, 4, 2, True), (40, 2, 1, False)])
def test_block_and_its_gradients(dim, H, Hk, causal):
    from scenario_wise_rec import _hip as Hip
    block, B, L = make_block(dim, H, Hk, causal), 6, 21
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    x = torch.randn(B, L, dim, generator=g, device="cuda", requires_grad=True)
    d = torch.randn(B, dim, generator=g, device="cuda")
    seen = torch.rand(B, L, generator=g, device="cuda") < 0.7
    seen[0] = True
    seen[1, 5:] = False
    seen[2, :9] = False
    y = block.train().pool(x.reshape(B, L * dim), seen)
    y.backward(d)
    p = {n: w.detach().double().requires_grad_(True) for n, w in block.named_parameters()}
    x64, want = x.detach().double().requires_grad_(True), []
    for b in range(B):
        z = plain_block(p, x64[b], seen[b], H, Hk, causal, block.buckets)
        want.append(z[seen[b]].mean(0))
    want = torch.stack(want)
    want.backward(d.double())
    close(y.detach(), want.detach(), "pooled")
    close(x.grad, x64.grad, "x")
    for n, w in block.named_parameters():
        close(w.grad, p[n].grad, n)
    Hip.check_errors()
    with torch.no_grad():                                  # serving: the same values without the tape
        close(block.eval().pool(x.reshape(B, L * dim), seen), want.detach(), "serving")


def test_empty_history_pools_to_zero():
    block = make_block(16, 4, 4, True)
    x = torch.randn(3, 5 * 16, device="cuda", requires_grad=True)
    seen = torch.zeros(3, 5, dtype=torch.bool, device="cuda")
    seen[1, 2] = True
    y = block.pool(x, seen)
    assert not y[0].any() and not y[2].any() and y[1].any()
    y.sum().backward()
    assert not x.grad[0].any() and not x.grad[2].any() and torch.isfinite(x.grad).all()
    assert block.pool(x[:, :0], seen[:, :0]).shape == (3, 16)


def features(pad=0):
    from scenario_wise_rec.basic.features import DenseFeature, SequenceFeature, SparseFeature
    return [SparseFeature("s0", 17, 16), DenseFeature("d0"),
            SequenceFeature("h", 60, 16, pooling="attention", padding_idx=pad, attention={"n_heads": 2, "max_distance": 16}),
            SparseFeature("s1", 9, 8), SequenceFeature("m", 30, 16, pooling="mean", padding_idx=pad)]


def batch(B, L, g, pad=0):
    ri = lambda hi, *s: torch.randint(0, hi, s, generator=g, device="cuda")
    x = {"s0": ri(17, B), "s1": ri(9, B), "d0": torch.rand(B, generator=g, device="cuda"), "h": ri(60, B, L), "m": ri(30, B, 4),
         "domain_indicator": ri(3, B)}
    x["h"][torch.rand(B, L, generator=g, device="cuda") < 0.3] = pad
    return x, (torch.rand(B, generator=g, device="cuda") < 0.3).float()


def test_embedding_layer_columns():
    """The history's block sits at its place in the concatenation; the other columns are the plain lookup's bits; the table's gradient
    comes through the attention."""
    from scenario_wise_rec.basic.layers import EmbeddingLayer
    feats = features()
    torch.manual_seed(3)
    layer = EmbeddingLayer(feats)
    with torch.no_grad():
        for t in layer.embed_dict.values():
            t.weight.normal_(0, 0.5)
    layer.to("cuda").train()
    g = torch.Generator(device="cuda")
    g.manual_seed(4)
    x, _ = batch(50, 11, g)
    out = layer(x, feats, squeeze_dim=True)
    assert out.shape == (50, 16 + 16 + 8 + 16 + 1)
    others = [f for f in feats if f.name != "h"]
    rest = layer(x, others, squeeze_dim=True).detach()
    assert torch.equal(torch.cat([out[:, :16], out[:, 32:]], 1).detach(), rest)
    table = layer.embed_dict["h"].weight.detach().double().requires_grad_(True)
    p = {n: w.detach().double() for n, w in layer.seq_blocks["h"].named_parameters()}
    block, want = layer.seq_blocks["h"], []
    for b in range(50):
        seen = x["h"][b] != 0
        e = table[x["h"][b]] * seen[:, None]
        z = plain_block(p, e, seen, 2, 2, True, block.buckets)
        want.append(z[seen].mean(0) if seen.any() else torch.zeros(16, dtype=torch.float64, device="cuda"))
    want = torch.stack(want)
    close(out[:, 16:32].detach(), want.detach(), "pooled")
    d = torch.randn(50, 16, generator=g, device="cuda")
    (out[:, 16:32] * d).sum().backward()
    want.backward(d.double())
    close(layer.embed_dict["h"].weight.grad, table.grad, "table")


def test_models_train_and_replay():
    """A model with an attention-pooled history under CTRTrainer: the captured step replays to the eager steps' bits."""
    from scenario_wise_rec.models.multi_domain import MMOE
    from scenario_wise_rec.trainers import CTRTrainer
    from scenario_wise_rec.trainers.graph import GraphedStep

    def train(graphed):
        torch.manual_seed(5)
        model = MMOE(features(), domain_num=3, n_expert=2, expert_params={"dims": [16]}, tower_params={"dims": [8]})
        with torch.no_grad():
            for n, w in model.named_parameters():
                if "embed_dict" in n:
                    w.normal_(0, 0.3)
        tr = CTRTrainer(model, "attention", optimizer_params={"lr": 1e-2, "weight_decay": 1e-5}, device="cuda")
        model.train()
        g = torch.Generator(device="cuda")
        g.manual_seed(6)
        x, y = batch(500, 9, g)
        before = {k: v.detach().clone() for k, v in model.state_dict().items()}
        if graphed:
            step = GraphedStep(tr, x, y, warmup=2)
            for _ in range(4):
                step.replay()
        else:
            for _ in range(6):
                tr.train_step(x, y)
        torch.cuda.synchronize()
        return before, {k: v.detach().clone() for k, v in model.state_dict().items()}
    before, a = train(False)
    _, b = train(True)
    for k in a:
        assert torch.equal(a[k], b[k]), k
        if "seq_blocks" in k:
            assert not torch.equal(a[k], before[k]), k         # every parameter of the block learns


def test_refusals():
    from scenario_wise_rec.basic.layers import EmbeddingLayer, SequenceBlock, fused_lookup
    feats = features()
    layer = EmbeddingLayer(feats).to("cuda")
    g = torch.Generator(device="cuda")
    g.manual_seed(7)
    x, _ = batch(8, 3, g)
    with pytest.raises(ValueError):
        layer(x, feats, squeeze_dim=False)
    with pytest.raises(NotImplementedError):
        fused_lookup(x, [(EmbeddingLayer(feats[:2]).to("cuda"), feats)])
    with pytest.raises(NotImplementedError):
        fused_lookup(x, [(layer, feats)])
    for args in ((10, 4), (16, 4, 3)):
        with pytest.raises(ValueError):
            SequenceBlock(*args)
