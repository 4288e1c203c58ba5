"""Sequence attention (csrc/seq_attention_*.hip) against its 64-bit definition: values and gradients within counted roundings."""
import pytest
import torch

import _seq_reference as ref

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


def prefix(lens, device="cuda"):
    return torch.tensor([0] + list(torch.tensor(list(lens) or [0]).cumsum(0))[:len(lens)], dtype=torch.int32, device=device)


def starts(lens):
    out, at = [], 0
    for n in lens:
        out.append(at)
        at += n
    return out


def randn(g, *shape, dtype=F32, scale=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def run(q, k, v, dout, bias=None, grads=True, **kw):
    """-> {name: tensor}; q, k, v may be views: gradients are taken of detached leaves of the same strides."""
    from scenario_wise_rec import ops
    leaf = lambda t: None if t is None else t.detach().requires_grad_(grads)
    q, k, v, bias = leaf(q), leaf(k), leaf(v), leaf(bias)
    out = ops.seq_attention(q, k, v, bias=bias, **kw)
    got = {"out": out.detach()}
    if grads:
        names = ["dq", "dk", "dv"] + (["dbias"] if bias is not None else [])
        got.update(zip(names, torch.autograd.grad(out, [t for t in (q, k, v, bias) if t is not None], dout)))
    return got


def compare(got, want):
    from scenario_wise_rec import _hip as H
    torch.cuda.synchronize()
    for name, t in got.items():
        ref.check(t, want[name], name)
    H.check_errors()


def table(n, far, causal):
    from scenario_wise_rec import ops
    return ops.seq_buckets(n, far, causal)


PACKED = [
    # lens, heads, key heads, D
    ([1], 1, 1, 8),
    ([0, 3, 0, 65, 0], 2, 2, 16),
    ([32, 33, 31], 4, 4, 16),
    ([50, 7, 64, 1, 20], 4, 2, 32),
    ([129, 200, 63], 6, 2, 20),
    ([300, 1], 5, 1, 33),
    ([257, 64], 4, 4, 64),
    ([190], 3, 3, 96),
    ([140, 33], 4, 2, 128),
    ([70, 2], 2, 1, 1),
]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("with_bias", [True, False])
@pytest.mark.parametrize("case", range(len(PACKED)))
def test_packed_sequences_and_gradients(case, with_bias, causal, dtype):
    lens, H, Hk, D = PACKED[case]
    g, T = gen(case), sum(lens)
    q, k, v, dout = randn(g, T, H, D, dtype=dtype), randn(g, T, Hk, D, dtype=dtype), randn(g, T, Hk, D, dtype=dtype), randn(g, T, H, D, dtype=dtype)
    bias, tab = (randn(g, H, 12), table(12, 40, causal)) if with_bias else (None, None)
    got = run(q, k, v, dout, bias, cu_q=prefix(lens), max_q=max(lens), causal=causal, buckets=tab)
    compare(got, ref.attention(q, k, v, dout, lens, lens, starts(lens), starts(lens), causal, None, bias, tab))


CACHED = [
    # new tokens, key lengths, room behind each, heads, key heads, D
    ([1], [500], [12], 4, 4, 16),
    ([1, 1, 1], [1, 700, 64], [0, 5, 64], 8, 2, 64),
    ([5, 0, 3], [5, 90, 2000], [1, 0, 48], 6, 3, 40),
    ([13] * 4, [13, 400, 77, 1025], [3, 0, 51, 7], 8, 2, 128),
    ([33, 20], [600, 33], [0, 31], 8, 1, 80),
    ([9, 4], [3, 0], [2, 6], 2, 1, 32),            # fewer keys than queries: rows without a key
    ([150, 64], [400, 333], [10, 3], 4, 2, 64),    # a chunk of a prompt
]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("case", range(len(CACHED)))
def test_new_tokens_over_cached_keys(case, causal, dtype):
    qs, ks, room, H, Hk, D = CACHED[case]
    cap = [a + b for a, b in zip(ks, room)]
    g = gen(100 + case)
    q, dout = randn(g, sum(qs), H, D, dtype=dtype), randn(g, sum(qs), H, D, dtype=dtype)
    k, v = randn(g, sum(cap), Hk, D, dtype=dtype), randn(g, sum(cap), Hk, D, dtype=dtype)
    for b, n in enumerate(ks):                     # what lies behind the used keys does not count
        k[starts(cap)[b] + n:starts(cap)[b] + cap[b]] = float("nan")
        v[starts(cap)[b] + n:starts(cap)[b] + cap[b]] = float("inf")
    bias, tab = randn(g, H, 16), table(16, 64, causal)
    kw = dict(cu_q=prefix(qs), cu_k=prefix(cap), max_q=max(qs), max_k=max(cap), causal=causal, buckets=tab,
              k_len=torch.tensor(ks, dtype=torch.int32, device="cuda"))
    want = ref.attention(q, k, v, dout, qs, ks, starts(qs), starts(cap), causal, None, bias, tab)
    compare(run(q, k, v, dout, bias, **kw), want)
    compare(run(q, k, v, dout, bias, grads=False, **kw), ref.attention(q, k, v, dout, qs, ks, starts(qs), starts(cap), causal, None, bias, tab, train=False))


def test_bias_gradient_of_bf16_tensors_has_fp32_accuracy():
    """Every row's score gradients cancel, so the bias gradient shows a delta that does not belong to them (off by 2.8e-3 of its norm
    with rows kept in bf16).  Its terms are fp32 sums: 2^-16 of what remains of p in two bf16 terms, averaged over >= 2^4 keys of
    random sign, bounds it by 2^-14 of the norm."""
    g, lens = gen(12), [900, 300]
    q, k, v, dout = (randn(g, 1200, 4, 64, dtype=BF16) for _ in range(4))
    bias, tab = randn(g, 4, 16, scale=0.5), table(16, 100, True)
    got = run(q, k, v, dout, bias, cu_q=prefix(lens), max_q=900, buckets=tab)["dbias"].double()
    want = ref.attention(q, k, v, dout, lens, lens, [0, 900], [0, 900], True, None, bias, tab)["dbias"][0]
    assert float((got - want).norm() / want.norm()) <= 2.0 ** -14


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_long_reach_table_and_far_distances(dtype):
    """Sequences much longer than the table's reach, both ways, and a table longer than the sequences."""
    g = gen(7)
    lens = [700, 90]
    for far, causal in ((20, False), (20, True), (1000, True), (600, False)):
        q, k, v, dout = (randn(g, 790, 2, 64, dtype=dtype) for _ in range(4))
        bias, tab = randn(g, 2, 8), table(8, far, causal)
        got = run(q, k, v, dout, bias, cu_q=prefix(lens), causal=causal, buckets=tab)
        compare(got, ref.attention(q, k, v, dout, lens, lens, [0, 700], [0, 700], causal, None, bias, tab))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_padded_batch_with_hidden_keys(dtype):
    """A padded [B, L] batch: left- and right-padded and scattered masks, one row all hidden; hidden keys hold NaN and infinities."""
    B, L, H, Hk, D = 5, 70, 4, 2, 32
    g = gen(3)
    q, dout = randn(g, B * L, H, D, dtype=dtype), randn(g, B * L, H, D, dtype=dtype)
    k, v = randn(g, B * L, Hk, D, dtype=dtype), randn(g, B * L, Hk, D, dtype=dtype)
    mask = torch.zeros(B, L, dtype=torch.bool, device="cuda")
    mask[0, 40:] = True
    mask[1, :13] = True
    mask[2] = torch.rand(L, generator=g, device="cuda") < 0.4
    mask[4] = True
    k[~mask.reshape(-1)] = float("nan")
    v[~mask.reshape(-1)] = float("-inf")
    bias, tab = randn(g, H, 16), table(16, 30, True)
    lens = [L] * B
    got = run(q, k, v, dout, bias, cu_q=prefix(lens), max_q=L, buckets=tab, key_mask=mask.reshape(-1))
    want = ref.attention(q, k, v, dout, lens, lens, starts(lens), starts(lens), True, None, bias, tab, mask.reshape(-1))
    compare(got, want)
    assert not got["out"][3 * L:4 * L].any() and not got["out"][:40].any()
    assert not got["dk"][~mask.reshape(-1)].any() and not got["dv"][~mask.reshape(-1)].any()
    got8 = run(q, k, v, dout, bias, cu_q=prefix(lens), buckets=tab, key_mask=mask.reshape(-1).to(torch.uint8))
    compare(got8, want)            # (no max_q: another tiling, so not the same bits)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_rows_in_use_and_rows_of_no_sequence(dtype):
    """q_len / k_len of a padded batch, rows before the first and behind the last sequence: zeros, whatever lies there."""
    g, H, D = gen(4), 2, 16
    cu = torch.tensor([5, 45, 85], dtype=torch.int32, device="cuda")
    used = torch.tensor([33, 0], dtype=torch.int32, device="cuda")
    q, k, v, dout = (randn(g, 100, H, D, dtype=dtype) for _ in range(4))
    for t in (q, k, v, dout):
        t[:5] = float("nan")
        t[38:] = float("nan")
    for extra in ({}, {"max_q": 40}):
        got = run(q, k, v, dout, cu_q=cu, q_len=used, **extra)
        compare(got, ref.attention(q, k, v, dout, [33], [33], [5], [5], True))
    # the same rows with few queries a sequence: the split form
    got = run(q, k, v, dout, grads=False, cu_q=torch.tensor([5, 6, 6], dtype=torch.int32, device="cuda"),
              cu_k=cu, k_len=used, max_q=1, max_k=40, causal=False)
    compare(got, ref.attention(q, k, v, dout, [1], [33], [5], [5], False, train=False))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_lowest_and_infinite_bias(dtype):
    """A bias of fp32's lowest value does not empty a row (all scores equal: uniform), -inf does."""
    g, H, D, L = gen(5), 2, 16, 40
    q, k, v, dout = (randn(g, L, H, D, dtype=dtype) for _ in range(4))
    tab = torch.arange(L, dtype=torch.int32, device="cuda").clamp(max=20)
    bias = torch.zeros(H, 21, device="cuda")
    bias[0] = torch.finfo(F32).min
    bias[1, 3:] = float("-inf")
    out = run(q, k, v, dout, bias, cu_q=prefix([L]), buckets=tab)["out"].double()
    mean = v[:, 0].double().cumsum(0) / torch.arange(1, L + 1, device="cuda")[:, None]
    assert (out[:, 0] - mean).abs().max() <= 2.0 ** -7 * v.double().abs().max()
    want = ref.attention(q[:, 1:], k[:, 1:], v[:, 1:], dout[:, 1:], [L], [L], [0], [0], True, None, bias[1:], tab)["out"]
    ref.check(out[:, 1:], want, "out")
    bias[1] = float("-inf")
    got = run(q, k, v, dout, bias, cu_q=prefix([L]), buckets=tab)
    assert not got["out"][:, 1].any() and not got["dq"][:, 1].any() and not got["dk"][:, 1].any() and not got["dbias"][1].any()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_strides_and_alignments(dtype):
    """Heads of one fused projection, a transposed head order, an expanded key: the bits of the contiguous call.  Rows off every
    alignment take another tiling, whose sums are grouped otherwise: within the same counted roundings of the definition."""
    g, T, H, D = gen(6), 100, 4, 24
    fused = randn(g, T, 3, H, D, dtype=dtype)
    lens, kw = [37, 63], dict(cu_q=prefix([37, 63]))
    dout = randn(g, T, H, D, dtype=dtype)
    base = run(*(fused[:, i].contiguous() for i in range(3)), dout, **kw)
    want = ref.attention(fused[:, 0], fused[:, 1], fused[:, 2], dout, lens, lens, [0, 37], [0, 37], True)
    compare(base, want)
    heads_first = [fused[:, i].transpose(0, 1).contiguous().transpose(0, 1) for i in range(3)]
    odd = [torch.empty(T * H * (D + 1) + 1, dtype=dtype, device="cuda")[1:].view(T, H, D + 1)[..., :D] for _ in range(3)]
    for t, i in zip(odd, range(3)):
        t.copy_(fused[:, i])
    every_other = [torch.empty(T, H, 2 * D, dtype=dtype, device="cuda")[..., ::2] for _ in range(3)]
    for t, i in zip(every_other, range(3)):
        t.copy_(fused[:, i])
    for form in ([fused[:, i] for i in range(3)], heads_first, odd, every_other):
        got = run(*form, dout.transpose(0, 1).contiguous().transpose(0, 1), **kw)
        compare(got, want)
        for n in base:
            assert form is odd or torch.equal(base[n], got[n]), n
    one = randn(g, T, 1, D, dtype=dtype)
    got = run(fused[:, 0], one.expand(T, H, D), one.expand(T, H, D), dout, grads=False, **kw)
    same = run(fused[:, 0], one, one, dout, grads=False, **kw)
    want = ref.attention(fused[:, 0], one, one, dout, lens, lens, [0, 37], [0, 37], True, train=False)       # (one key head: another tiling, too)
    compare(got, want)
    compare(same, want)


def test_hints_and_repeats_do_not_change_results():
    """max_q / max_k choose the launch and its tiling, right for any hint; two calls of the same hints give the same bits, side by
    side on two streams too."""
    g, H, Hk, D, lens = gen(8), 4, 2, 64, [200, 130, 77]
    T = sum(lens)
    q, k, v, dout = randn(g, T, H, D), randn(g, T, Hk, D), randn(g, T, Hk, D), randn(g, T, H, D)
    bias, tab = randn(g, H, 16), table(16, 50, True)
    kw = dict(cu_q=prefix(lens), buckets=tab)
    base = run(q, k, v, dout, bias, max_q=200, **kw)
    compare(base, ref.attention(q, k, v, dout, lens, lens, starts(lens), starts(lens), True, None, bias, tab))
    again = run(q, k, v, dout, bias, max_q=200, **kw)
    assert all(torch.equal(base[n], again[n]) for n in base)
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(other):
        beside = run(q, k, v, dout, bias, max_q=200, **kw)
    again = run(q, k, v, dout, bias, max_q=200, **kw)
    torch.cuda.current_stream().wait_stream(other)
    assert all(torch.equal(base[n], again[n]) and torch.equal(base[n], beside[n]) for n in base)
    want = ref.attention(q, k, v, dout, lens, lens, starts(lens), starts(lens), True, None, bias, tab)
    for hint in (1, 40, 0, None):
        compare(run(q, k, v, dout, bias, max_q=hint, **kw), want)


def test_bad_prefix_sums_lengths_and_buckets_are_clamped_and_reported():
    from scenario_wise_rec import _hip as H
    g = gen(9)
    q, k, v, dout = (randn(g, 64, 2, 16) for _ in range(4))
    H.check_errors()
    bad = [dict(cu_q=torch.tensor([0, 90, 40], dtype=torch.int32, device="cuda")),
           dict(cu_q=torch.tensor([-3, 20, 64], dtype=torch.int32, device="cuda")),
           dict(cu_q=prefix([64]), q_len=torch.tensor([65], dtype=torch.int32, device="cuda")),
           dict(cu_q=prefix([64]), k_len=torch.tensor([-1], dtype=torch.int32, device="cuda")),
           dict(cu_q=prefix([64]), bias=randn(g, 2, 4), buckets=torch.tensor([0, 4, -1], dtype=torch.int32, device="cuda"))]
    for kw in bad:
        run(q, k, v, dout, kw.pop("bias", None), **kw)
        with pytest.raises(IndexError):
            H.check_errors()
    H.check_errors()


def test_captured_step_replays_with_new_inputs():
    """Forward and backward captured into one graph and replayed with other inputs and lengths, eager work in between."""
    from scenario_wise_rec import ops
    g, H, D, T = gen(10), 4, 32, 256
    q, k, v, dout = (randn(g, T, H, D) for _ in range(4))
    bias, tab, cu = randn(g, H, 16), table(16, 60, True), prefix([100, 156])
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v, bias)]
    d = dout.clone()

    def step():
        out = ops.seq_attention(*leaves[:3], cu, max_q=256, bias=leaves[3], buckets=tab)
        return [out.detach()] + list(torch.autograd.grad(out, leaves, d))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for lens in ([100, 156], [3, 200], [256, 0]):
        with torch.no_grad():
            for t in leaves:
                t.copy_(randn(g, *t.shape))
            d.copy_(randn(g, T, H, D))
            cu.copy_(prefix(lens))
        graph.replay()
        torch.cuda.synchronize()
        eager = run(*[t.detach().clone() for t in leaves[:3]], d, leaves[3].detach().clone(), cu_q=prefix(lens), max_q=256, buckets=tab)
        for a, n in zip(outs, ("out", "dq", "dk", "dv", "dbias")):
            assert torch.equal(a, eager[n]), (lens, n)


def test_gradients_against_differences():
    """Directional central differences of the fp32 forward.  h = 2^-5: the cubic term of a smooth function of O(1) slopes is below
    h^2 of the derivative's scale; the outputs' fp32 roundings (2^-20 of their magnitude, 2 / (2 h) of them) add 2^-15 of it."""
    from scenario_wise_rec import ops
    g, H, Hk, D, lens = gen(11), 4, 2, 16, [40, 25]
    T = sum(lens)
    args = [randn(g, T, H, D), randn(g, T, Hk, D), randn(g, T, Hk, D), randn(g, H, 8)]
    dout, tab, h = randn(g, T, H, D), table(8, 20, True), 2.0 ** -5
    grads = list(run(*args[:3], dout, args[3], cu_q=prefix(lens), buckets=tab).values())[1:]
    for i in range(4):
        way = randn(g, *args[i].shape)
        way /= way.norm()
        side = []
        for s in (1, -1):
            a = list(args)
            a[i] = a[i] + s * h * way
            side.append((ops.seq_attention(*a[:3], prefix(lens), bias=a[3], buckets=tab).double() * dout.double()).sum())
        got, want = float((grads[i].double() * way.double()).sum()), float((side[0] - side[1]) / (2 * h))
        scale = float(grads[i].double().norm())
        assert abs(got - want) <= (4 * h * h + 2.0 ** -12) * scale, (i, got, want, scale)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("scale", [0.0, -0.3, 2.0])
def test_given_scales(scale, dtype):
    g, lens = gen(13), [150, 40]
    q, k, v, dout = (randn(g, 190, 2, 32, dtype=dtype) for _ in range(4))
    bias, tab = randn(g, 2, 8), table(8, 20, True)
    got = run(q, k, v, dout, bias, cu_q=prefix(lens), max_q=150, buckets=tab, scale=scale)
    compare(got, ref.attention(q, k, v, dout, lens, lens, [0, 150], [0, 150], True, scale, bias, tab))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_one_long_sequence_among_many_without_hints(dtype):
    """The default launch is sized for four times the mean length: the long sequence is walked in rounds."""
    g, lens = gen(14), [3] * 60 + [900] + [1] * 60
    T = sum(lens)
    q, k, v, dout = randn(g, T, 2, 32, dtype=dtype), randn(g, T, 1, 32, dtype=dtype), randn(g, T, 1, 32, dtype=dtype), randn(g, T, 2, 32, dtype=dtype)
    bias, tab = randn(g, 2, 8), table(8, 20, True)
    got = run(q, k, v, dout, bias, cu_q=prefix(lens), buckets=tab)
    compare(got, ref.attention(q, k, v, dout, lens, lens, starts(lens), starts(lens), True, None, bias, tab))


def test_largest_table_and_widest_group():
    """The largest distance table the backward has room for, and many query heads on one key head; one more is refused."""
    from scenario_wise_rec import _hip as H
    from scenario_wise_rec import ops
    g = gen(15)
    for dtype in (F32, BF16):
        q, k, v, dout = (randn(g, 70, 2, 128, dtype=dtype) for _ in range(4))
        for causal in (True, False):
            bias, tab = randn(g, 2, 256), table(256, 2048 if causal else 1024, causal)
            got = run(q, k, v, dout, bias, cu_q=prefix([70]), causal=causal, buckets=tab)
            compare(got, ref.attention(q, k, v, dout, [70], [70], [0], [0], causal, None, bias, tab))
        q, dout = randn(g, 40, 93, 128, dtype=dtype), randn(g, 40, 93, 128, dtype=dtype)
        k, v = randn(g, 40, 1, 128, dtype=dtype), randn(g, 40, 1, 128, dtype=dtype)
        compare(run(q, k, v, dout, cu_q=prefix([40])), ref.attention(q, k, v, dout, [40], [40], [0], [0], True))
    with pytest.raises(H.SwrError):
        ops.seq_attention(q[:, :1].expand(40, 94, 128), k, v, prefix([40]))


def test_rows_behind_the_last_sequence_are_zeros_in_a_large_buffer():
    """A buffer of fixed size whose last rows no sequence uses, odd row sizes: every output row of them is zero."""
    g = gen(16)
    for H, D in ((3, 5), (2, 64)):
        T = 60001
        q, k, v, dout = (randn(g, T, H, D, dtype=BF16) for _ in range(4))
        got = run(q, k, v, dout, cu_q=torch.tensor([7, 50, 107], dtype=torch.int32, device="cuda"), max_q=57)
        for n, t in got.items():
            assert not t[:7].any() and not t[107:].any() and t[7:107].any(), n


def test_offsets_beyond_32_bits():
    """A cache of more than 2^31 elements: its last sequence starts past 2^31."""
    rows, H, D = (1 << 24) + 600, 1, 128
    k, v = (torch.empty(rows, H, D, dtype=BF16, device="cuda") for _ in range(2))
    g = gen(17)
    first = (1 << 24) + 100
    k[first:], v[first:] = randn(g, 500, H, D, dtype=BF16), randn(g, 500, H, D, dtype=BF16)
    q, dout = randn(g, 40, 2, D, dtype=BF16), randn(g, 40, 2, D, dtype=BF16)
    cu_k = torch.tensor([first, first + 500], dtype=torch.int32, device="cuda")
    for new in (1, 40):
        got = run(q[:new], k, v, dout[:new], grads=False, cu_q=prefix([new]), cu_k=cu_k, max_q=new, max_k=500)
        compare(got, ref.attention(q[:new], k[first:], v[first:], dout[:new], [new], [500], [0], [0], True, train=False))


def test_saved_tensors_may_move_and_the_graph_may_be_walked_twice():
    """Saved tensors kept on the host between the passes; a second backward over the same graph; an expanded output gradient."""
    from scenario_wise_rec import ops
    g = gen(18)
    for dtype in (F32, BF16):
        leaves = [randn(g, 50, 2, 32, dtype=dtype).requires_grad_(True) for _ in range(3)]
        out = ops.seq_attention(*leaves, prefix([50]))
        base = torch.autograd.grad(out.sum(), leaves, retain_graph=True)
        again = torch.autograd.grad(out.sum(), leaves)
        with torch.autograd.graph.save_on_cpu():
            out = ops.seq_attention(*leaves, prefix([50]))
        moved = torch.autograd.grad(out.sum(), leaves)
        for a, b, c in zip(base, again, moved):
            assert torch.equal(a, b) and torch.equal(a, c)


def test_empty_inputs():
    from scenario_wise_rec import ops
    for tq, tk in ((0, 0), (0, 8), (8, 0)):
        q = torch.randn(tq, 2, 16, device="cuda", requires_grad=True)
        k, v = (torch.randn(tk, 2, 16, device="cuda", requires_grad=True) for _ in range(2))
        out = ops.seq_attention(q, k, v, prefix([tq]), prefix([tk]))
        assert out.shape == q.shape and not out.any()
        for gr in torch.autograd.grad(out.sum(), (q, k, v)):
            assert not gr.any()
    q = torch.randn(8, 2, 16, device="cuda")
    assert not ops.seq_attention(q, q, q, torch.zeros(1, dtype=torch.int32, device="cuda")).any()      # no sequence at all


def test_refusals():
    from scenario_wise_rec import _hip as H
    from scenario_wise_rec import ops
    q, cu = torch.randn(8, 4, 16, device="cuda"), prefix([8])
    kv = torch.randn(8, 2, 16, device="cuda")
    ops.seq_attention(q, kv, kv, cu)
    bias, tab = torch.zeros(4, 8, device="cuda"), table(8, 20, True)
    E, V = H.SwrError, ValueError
    for err, args, kw in [
            (V, (q[0], kv, kv, cu), {}), (V, (q, kv, kv[:4], cu), {}), (V, (q, kv[..., :8], kv[..., :8], cu), {}),
            (E, (q, kv.bfloat16(), kv, cu), {}), (E, (q.half(), kv.half(), kv.half(), cu), {}), (E, (q.cpu(), kv, kv, cu), {}),
            (V, (q, kv[:, :1].expand(8, 3, 16), kv[:, :1].expand(8, 3, 16), cu), {}),
            (V, (torch.randn(8, 1, 129, device="cuda"),) * 3 + (cu,), {}),
            (V, (q, kv, kv, cu.long()), {}), (V, (q, kv, kv, cu[:0]), {}), (E, (q, kv, kv, cu, cu.cpu()), {}),
            (V, (q, kv[:4], kv[:4], cu), {}), (V, (q, kv, kv, cu, prefix([4, 4])), {}),
            (V, (q, kv, kv, cu), {"k_len": prefix([8])}), (V, (q, kv, kv, cu), {"key_mask": torch.ones(7, device="cuda", dtype=torch.bool)}),
            (V, (q, kv, kv, cu), {"key_mask": torch.ones(8, device="cuda")}),
            (V, (q, kv, kv, cu), {"bias": bias}), (V, (q, kv, kv, cu), {"buckets": tab}),
            (V, (q, kv, kv, cu), {"bias": bias[:3], "buckets": tab}), (V, (q, kv, kv, cu), {"bias": bias.bfloat16(), "buckets": tab}),
            (V, (q, kv, kv, cu), {"bias": bias, "buckets": tab[:20], "causal": False}),
            (V, (q, kv, kv, cu), {"bias": bias, "buckets": tab.long()})]:
        with pytest.raises(err):
            ops.seq_attention(*args, **kw)
    H.check_errors()
