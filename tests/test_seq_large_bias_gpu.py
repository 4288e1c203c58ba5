"""Sequence attention where a row's visible keys all carry a bias of large magnitude (masks of the type's lowest value, -1e9, ...).

Scores are held in fp32, s = scale q . k + bias: a bias whose step is wider than the products absorbs them and the row's keys count
alike, p = 1 / (number of visible keys), in the output and in every gradient.  The allowed errors below are of that p: they do not grow
with the bias that all scores of a row share."""
import pytest
import torch

import _seq_reference as ref

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16
LOWEST = torch.finfo(F32).min


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def randn(g, *shape, dtype=F32, scale=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def prefix(*lens):
    return torch.tensor([0] + list(lens), dtype=torch.int32, device="cuda").cumsum(0, dtype=torch.int32)


def one_each(n):
    """A table with a bucket for every distance below n - 1, the last one for all further ones."""
    return torch.arange(n, dtype=torch.int32, device="cuda")


def alike(v, lq, causal, train):
    """out of one head whose visible keys count alike, with its allowed error (v [lk, D], the last query at the last key)."""
    lk = v.shape[0]
    u = 2.0 ** -8 if v.dtype == BF16 else 2.0 ** -24
    rf = (2.0 ** -16 if train else u) if v.dtype == BF16 else ref.f(16)
    dist = (torch.arange(lq, device="cuda") + lk - lq)[:, None] - torch.arange(lk, device="cuda")[None]
    ok = (dist >= 0 if causal else torch.ones_like(dist, dtype=torch.bool)).double()
    p = ok / ok.sum(1, keepdim=True).clamp(min=1)
    out = p @ v.double()
    return out, (2.0 ** -20 + rf + ref.f(lk)) * (p @ v.double().abs()) + u * out.abs()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("bias,spread", [(LOWEST, 1.0), (LOWEST, 30.0), (-1e9, 1.0), (1e9, 1.0), (-1e6, 0.0), (-3000.0, 0.0)])
def test_keys_count_alike_on_both_sides_of_the_reach(bias, spread, causal, dtype):
    """Sequences longer than the table's reach: blocks that touch the table and blocks that lie wholly beyond it give the same row the
    same weights, also where the products (spread 30: scores up to some thousand) would overflow an exponent."""
    from scenario_wise_rec import ops
    g, lens, H, D = gen(1), [230, 70], 2, 32
    q, k, v = (randn(g, 300, H, D, dtype=dtype, scale=spread) for _ in range(3))
    v = randn(g, 300, H, D, dtype=dtype)
    n = 21
    table = one_each(n) if causal else torch.cat([one_each(n).flip(0), one_each(n)[1:]])
    b = torch.full((H, n), bias, device="cuda")
    out = ops.seq_attention(q, k, v, prefix(*lens), max_q=230, causal=causal, bias=b, buckets=table)
    few = ops.seq_attention(q[225:230], k[:230], v[:230], prefix(5), prefix(230), max_q=5, max_k=230, causal=causal, bias=b, buckets=table)
    for h in range(H):
        for rows in (slice(0, 230), slice(230, 300)):
            ref.check(out[rows, h], alike(v[rows, h], rows.stop - rows.start, causal, False), "out")
        ref.check(few[:, h], alike(v[:230, h], 5, causal, False), "few")


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_far_keys_of_lowest_bias_beside_ordinary_ones(dtype):
    """A bucket of the lowest value, or of -1e9, beyond a window hides those keys from rows that see ordinary ones, as -inf does."""
    from scenario_wise_rec import ops
    g, L, H, D, n = gen(2), 200, 2, 32, 41
    q, k, v = (randn(g, L, H, D, dtype=dtype) for _ in range(3))
    hidden = randn(g, H, n)
    hidden[:, -1] = float("-inf")
    want = ref.attention(q, k, v, v, [L], [L], [0], [0], True, None, hidden, one_each(n), train=False)["out"]
    for far in (LOWEST, -1e9, float("-inf")):
        b = hidden.clone()
        b[:, -1] = far
        ref.check(ops.seq_attention(q, k, v, prefix(L), max_q=L, bias=b, buckets=one_each(n)), want, f"out {far}")
