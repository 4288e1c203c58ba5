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


# ---------------------------------------------------------------------------------------------------------------- gradients
def one_head(q, k, v, dout, add, slot, n_buckets, causal, scale):
    """-> {name: (value, allowed error)} of one head in 64 bits.  add [lq, lk]: the bias of every score; where it is 1e9 or more in
    magnitude it absorbs the product, and where the row's products are zeros (q = 0) and its biases equal the scores are exact: neither
    adds an error of the scores.  The other errors are counted as in _seq_reference."""
    lq, lk, D = q.shape[0], k.shape[0], q.shape[1]
    bf16, f = q.dtype == BF16, ref.f
    u = 2.0 ** -8 if bf16 else 2.0 ** -24
    r, rf = (u, 2.0 ** -16) if bf16 else (f(16), f(16))
    Q, K, V, dO, add = (t.double() for t in (q, k, v, dout, add))
    dist = (torch.arange(lq, device="cuda") + lk - lq)[:, None] - torch.arange(lk, device="cuda")[None]
    ok = dist >= 0 if causal else torch.ones_like(dist, dtype=torch.bool)
    mag = Q.abs() @ K.abs().t() * scale
    s = torch.where(add.abs() >= 1e9, add, Q @ K.t() * scale + add)
    exact = (add.abs() >= 1e9) | ((mag == 0) & (add == add[:, :1]))
    es = torch.where(exact, 0., (f(D) + 4 * 2.0 ** -24) * (mag + add.abs()) + 2.0 ** -23 * s.abs())
    p = torch.softmax(s.masked_fill(~ok, float("-inf")), 1)
    es = torch.where(p > 0, es, 0.)                       # (keys that weigh nothing beside the row's others)
    ep = (es + es.max(1, keepdim=True).values + 2.0 ** -20) * p
    o = p @ V
    eo = ep @ V.abs() + (rf + f(lk)) * (p @ V.abs())
    dp, delta = dO @ V.t(), (dO * o).sum(1, keepdim=True)
    size = dO.abs() @ V.abs().t() + (dO.abs() * o.abs()).sum(1, keepdim=True)
    ed = (dO.abs() * (2.0 ** -24 * o.abs() + eo)).sum(1, keepdim=True) + f(D) * size
    ds = p * (dp - delta)
    eds = ep * (dp - delta).abs() + p * ed + 4 * 2.0 ** -24 * p * size
    edsr, acc = eds + r * ds.abs(), f(lk) + f(lq)
    gq, gk, gv = ds @ K * scale, ds.t() @ Q * scale, p.t() @ dO
    res = {"out": (o, eo + u * o.abs()),
           "dq": (gq, (edsr @ K.abs() + acc * (ds.abs() @ K.abs())) * scale + u * gq.abs()),
           "dk": (gk, (edsr.t() @ Q.abs() + acc * (ds.abs().t() @ Q.abs())) * scale + u * gk.abs()),
           "dv": (gv, (ep + r * p).t() @ dO.abs() + acc * (p.t() @ dO.abs()) + u * gv.abs())}
    db, eb = (torch.zeros(n_buckets, dtype=torch.float64, device="cuda") for _ in range(2))
    db.index_add_(0, slot.reshape(-1), ds.reshape(-1))
    eb.index_add_(0, slot.reshape(-1), (eds + f(lk) * ds.abs()).reshape(-1))
    res["dbias"] = (db, eb)
    return res


def check_gradients(q, k, v, dout, bias, table, qs, ks, causal, what, **hints):
    """Every head of packed sequences (as many key heads as query heads) against one_head."""
    from scenario_wise_rec import _hip as Hip
    from scenario_wise_rec import ops
    leaves = [t.detach().clone().requires_grad_(True) for t in (q, k, v, bias)]
    out = ops.seq_attention(*leaves[:3], prefix(*qs), prefix(*ks), causal=causal, bias=leaves[3], buckets=table, **hints)
    got = dict(zip(("out", "dq", "dk", "dv", "dbias"), (out.detach(),) + torch.autograd.grad(out, leaves, dout)))
    R = table.numel() - 1 if causal else table.numel() // 2
    for h in range(q.shape[1]):
        dbias, aq, ak = 0, 0, 0
        for lq, lk in zip(qs, ks):
            sq, sk = slice(aq, aq + lq), slice(ak, ak + lk)
            dist = (torch.arange(lq, device="cuda") + lk - lq)[:, None] - torch.arange(lk, device="cuda")[None]
            slot = table[dist.clamp(0, R) if causal else dist.clamp(-R, R) + R].long()
            want = one_head(q[sq, h], k[sk, h], v[sk, h], dout[sq, h], bias[h][slot], slot, bias.shape[1], causal, q.shape[2] ** -0.5)
            for n in ("out", "dq", "dk", "dv"):
                ref.check(got[n][sk if n in ("dk", "dv") else sq, h], want[n], f"{what} head {h} {n}")
            dbias = [a + b for a, b in zip(dbias, want["dbias"])] if dbias else list(want["dbias"])
            aq, ak = aq + lq, ak + lk
        ref.check(got["dbias"][h], dbias, f"{what} head {h} dbias")
    Hip.check_errors()


def both_sides(n, causal):
    return one_each(n) if causal else torch.cat([one_each(n).flip(0), one_each(n)[1:]])


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("D", [16, 64, 128])
@pytest.mark.parametrize("value", [LOWEST, -1e9, 1e9, -1e6, -3000.0, 100.0])
def test_gradients_of_rows_under_one_large_bias(value, D, causal, dtype):
    """Head 0: every bucket holds the value (products of zero where it does not absorb them); head 1: ordinary biases."""
    g, lens, H, n = gen(3), [150, 40], 2, 21
    q, k, v, dout = (randn(g, 190, H, D, dtype=dtype) for _ in range(4))
    if abs(value) < 1e9:
        q[:, 0] = 0
    bias = randn(g, H, n)
    bias[0] = value
    check_gradients(q, k, v, dout, bias, both_sides(n, causal), lens, lens, causal, str(value), max_q=150)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("value", [LOWEST, -1e9])
def test_gradients_where_some_rows_see_only_masked_buckets(value, dtype):
    """Near distances under a large bias: the first rows of a causal sequence see nothing else and count alike, the rows behind them see
    ordinary keys, and for them those keys are hidden.  Far distances the same way: there no row is left with them alone."""
    g, L, H, D, n = gen(4), 140, 2, 32, 31
    for near in (True, False):
        q, k, v, dout = (randn(g, L, H, D, dtype=dtype) for _ in range(4))
        bias = randn(g, H, n)
        bias[:, :11 if near else 0] = value
        if not near:
            bias[:, 25:] = value
        check_gradients(q, k, v, dout, bias, one_each(n), [L], [L], True, f"near {near}", max_q=L)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("value", [LOWEST, -1e9, 1e9])
def test_gradients_through_joined_key_ranges(value, dtype):
    """A few queries over many keys, whose ranges are joined: the row's two parts come from the join."""
    from scenario_wise_rec import _hip as Hip
    g, qs, ks, H, D, n = gen(5), [3, 1], [2000, 700], 2, 64, 21
    q, dout = randn(g, 4, H, D, dtype=dtype), randn(g, 4, H, D, dtype=dtype)
    k, v = randn(g, 2700, H, D, dtype=dtype), randn(g, 2700, H, D, dtype=dtype)
    bias = randn(g, H, n)
    bias[0] = value
    for causal in (True, False):
        check_gradients(q, k, v, dout, bias, both_sides(n, causal), qs, ks, causal, "joined", max_q=3, max_k=2000)
    a = Hip.SeqAttentionArgs()
    a.Tq, a.Tk, a.B, a.Hq, a.Hk, a.D, a.dtype, a.causal, a.max_q, a.max_k = 4, 2700, 2, H, H, D, Hip.dtype_code(q), 1, 3, 2000
    for name in ("q", "k", "v", "out", "cu_q", "cu_k"):
        setattr(a, name, 4096)
    assert Hip.lib.swr_seq_attention_fwd_workspace_bytes(Hip.C.byref(a)) > 0         # (ranges to join)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("causal", [True, False])
def test_gradients_of_large_scores(causal, dtype):
    """Scores of 800, 804 and 808 without a bias: exact products, their weights are known.  800 log2 e = 1154: a rounding of 2^-14 in x and
    in the row's exponent each, for a key and for the row's sum."""
    g, L, H, D = gen(6), 90, 1, 16
    q, k = torch.zeros(L, H, D, dtype=dtype, device="cuda"), torch.zeros(L, H, D, dtype=dtype, device="cuda")
    q[..., 0] = 32.0
    k[..., 0] = torch.randint(0, 3, (L, H), generator=g, device="cuda").to(dtype) / 2 + 100
    v, dout = randn(g, L, H, D, dtype=dtype), randn(g, L, H, D, dtype=dtype)
    from scenario_wise_rec import ops
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    out = ops.seq_attention(*leaves, prefix(L), max_q=L, causal=causal)
    dv = torch.autograd.grad(out, leaves, dout)[2].double()[:, 0]
    s = (q[:, 0].double() @ k[:, 0].double().t()) * 0.25
    hidden = torch.arange(L, device="cuda")[:, None] < torch.arange(L, device="cuda")
    p = torch.softmax(s.masked_fill(hidden & causal, float("-inf")), 1)
    ep = (4 * 2.0 ** -14 + 2.0 ** -20) * p
    r, u = (2.0 ** -8, 2.0 ** -8) if dtype == BF16 else (ref.f(16), 2.0 ** -24)
    want, dO = p.t() @ dout[:, 0].double(), dout[:, 0].double().abs()
    ref.check(dv, (want, (ep + r * p).t() @ dO + 2 * ref.f(L) * (p.t() @ dO) + u * want.abs()), "dv")
