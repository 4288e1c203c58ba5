"""Norms around a block (csrc/norm_gate.hip) against their 64-bit definition, within counted roundings."""
import itertools

import pytest
import torch

import _seq_reference as ref

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16
PARTS = ("y", "gate", "w_post", "w_pre")


def make(M, N, dtype, parts, seed=0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")
    t = {"x": r(M, N).to(dtype), "y": (2 * r(M, N)).to(dtype), "gate": r(M, N).to(dtype), "w_post": 1 + 0.2 * r(N), "w_pre": 1 + 0.2 * r(N)}
    t = {k: v for k, v in t.items() if k == "x" or k in parts}
    return t, r(M, N).to(dtype), r(M, N).to(dtype)


def run(t, dz, du, scale=0.7, eps=1e-6):
    from scenario_wise_rec import ops
    t = {k: v.detach().requires_grad_(True) for k, v in t.items()}
    res = ops.norm_gate_residual(scale=scale, eps=eps, **t)
    outs = list(res) if isinstance(res, tuple) else [res]
    names = (["z"] if "y" in t else []) + (["u"] if "w_pre" in t else [])
    got = dict(zip(names, (o.detach() for o in outs)))
    grads = torch.autograd.grad(outs, list(t.values()), [{"z": dz, "u": du}[n] for n in names])
    got.update(("d" + k, g) for k, g in zip(t, grads))
    return got


def compare(got, t, dz, du, scale=0.7, eps=1e-6):
    a = [t.get(k) for k in ("x",) + PARTS]
    want = ref.norm_gate(*a, scale, eps, dz if "y" in t else None, du if "w_pre" in t else None)
    torch.cuda.synchronize()
    for n, v in got.items():
        ref.check(v, want[n], n)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("M,N", [(1, 1), (37, 64), (5, 7), (300, 65), (1000, 130), (64, 452), (33, 513), (700, 1024), (9, 1030),
                                 (20, 2500), (6, 8192)])
def test_shapes(M, N, dtype):
    t, dz, du = make(M, N, dtype, PARTS, N)
    compare(run(t, dz, du), t, dz, du)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("parts", [p for n in range(5) for p in itertools.combinations(PARTS, n)
                                   if ("y" in p or p == ("w_pre",))])
def test_every_combination_of_parts(parts, dtype):
    for M, N in ((50, 96), (11, 1500)):
        t, dz, du = make(M, N, dtype, parts, len(parts))
        compare(run(t, dz, du), t, dz, du)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_many_rows_and_one_sided_gradients(dtype):
    """More rows than workgroups take at once; gradients of z alone and of u alone."""
    from scenario_wise_rec import ops
    t, dz, du = make(9000, 40, dtype, PARTS, 5)
    compare(run(t, dz, du), t, dz, du)
    leaves = {k: v.clone().requires_grad_(True) for k, v in t.items()}
    z, u = ops.norm_gate_residual(scale=0.7, **leaves)
    zero = torch.zeros_like(dz)
    for out, d, pair in ((z, dz, (dz, zero)), (u, du, (zero, du))):
        got = dict(zip(("d" + k for k in leaves), torch.autograd.grad(out, list(leaves.values()), d, retain_graph=True, allow_unused=True)))
        want = ref.norm_gate(*[t[k] for k in ("x",) + PARTS], 0.7, 1e-6, *pair)
        for n, v in got.items():
            if v is None:
                assert n == "dw_pre" and out is z
            else:
                ref.check(v, want[n], n)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_strided_rows_are_bitwise_the_same(dtype):
    t, dz, du = make(60, 52, dtype, PARTS, 1)
    base = run(t, dz, du)
    for pad in (4, 1, 12):
        view = lambda v: torch.empty(60, 52 + pad, dtype=dtype, device="cuda")[:, pad:].copy_(v) if v.dim() == 2 else v
        got = run({k: view(v) for k, v in t.items()}, view(dz), view(du))
        assert all(torch.equal(base[n], got[n]) for n in base)
    got = run({k: v.t().contiguous().t() if v.dim() == 2 else v for k, v in t.items()}, dz.t().contiguous().t(), du)
    assert all(torch.equal(base[n], got[n]) for n in base)


def test_extreme_rows():
    """A row of zeros (only eps under the root), gates far out on both sides, one large entry; NaN stays in its row."""
    t, dz, du = make(6, 64, F32, PARTS, 2)
    t["y"][0] = 0
    t["gate"][1] = 100
    t["gate"][2] = -100
    t["x"][3, 5] = 1e8
    compare(run(t, dz, du), t, dz, du)
    t["x"][4, 1] = float("nan")
    got = run(t, dz, du)
    for n in ("z", "u", "dx", "dy"):
        assert torch.isfinite(got[n][[0, 1, 2, 3, 5]]).all(), n
    assert got["u"][4].isnan().all() and got["z"][4].isnan().sum() == 1


def test_one_weight_in_both_places():
    """The same parameter behind the block and before the next: its gradient is the sum of both."""
    from scenario_wise_rec import ops
    t, dz, du = make(70, 96, F32, ("y", "w_post"), 6)
    w = t["w_post"].clone().requires_grad_(True)
    z, u = ops.norm_gate_residual(t["x"], t["y"], w_post=w, w_pre=w, scale=0.7)
    got = torch.autograd.grad((z, u), w, (dz, du))[0]
    want = ref.norm_gate(t["x"], t["y"], None, t["w_post"], t["w_post"], 0.7, 1e-6, dz, du)
    ref.check(got, tuple(a + b for a, b in zip(want["dw_post"], want["dw_pre"])), "dw")
    w2 = t["w_post"].clone().requires_grad_(True)
    w2.grad, w2._swr_hooked = torch.ones_like(w2), True            # (as a parameter of a gradient arena)
    z, u = ops.norm_gate_residual(t["x"], t["y"], w_post=w2, w_pre=w2, scale=0.7)
    torch.autograd.backward((z, u), (dz, du))
    ref.check(w2.grad - 1, tuple(a + b + (2.0 ** -22 if i else 0) for i, (a, b) in enumerate(zip(want["dw_post"], want["dw_pre"]))), "arena")


def test_captured_and_replayed():
    from scenario_wise_rec import ops
    t, dz, du = make(500, 200, BF16, PARTS, 3)
    leaves = {k: v.clone().requires_grad_(True) for k, v in t.items()}

    def step():
        z, u = ops.norm_gate_residual(scale=0.7, **leaves)
        return [z.detach(), u.detach()] + list(torch.autograd.grad((z, u), list(leaves.values()), (dz, du)))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for seed in (10, 11, 12):
        new, dz2, du2 = make(500, 200, BF16, PARTS, seed)
        with torch.no_grad():
            for k in leaves:
                leaves[k].copy_(new[k])
            dz.copy_(dz2)
            du.copy_(du2)
        graph.replay()
        torch.cuda.synchronize()
        eager = run(new, dz2, du2)
        assert all(torch.equal(a, b) for a, b in zip(outs, eager.values()))


def test_gradients_against_differences():
    """h = 2^-4 over unit directions in fp32: cubic terms h^2, output roundings 2^-20 / h of the derivative's scale."""
    from scenario_wise_rec import ops
    t, dz, du = make(20, 48, F32, PARTS, 4)
    got, h = run(t, dz, du), 2.0 ** -4
    for k in t:
        way = torch.randn_like(t[k])
        way /= way.norm()
        side = []
        for s in (1, -1):
            z, u = ops.norm_gate_residual(scale=0.7, **{**t, k: t[k] + s * h * way})
            side.append((z.double() * dz.double()).sum() + (u.double() * du.double()).sum())
        have, want, size = float((got["d" + k].double() * way.double()).sum()), float((side[0] - side[1]) / (2 * h)), float(got["d" + k].norm())
        assert abs(have - want) <= (4 * h * h + 2.0 ** -12) * size, k


def test_empty_and_refusals():
    from scenario_wise_rec import _hip as H
    from scenario_wise_rec import ops
    x, w = torch.randn(4, 16, device="cuda"), torch.ones(16, device="cuda")
    e, we = torch.empty(0, 16, device="cuda", requires_grad=True), w.clone().requires_grad_(True)
    z, u = ops.norm_gate_residual(e, e, w_pre=we)
    assert z.shape == u.shape == (0, 16)
    assert all(not g.any() for g in torch.autograd.grad(z.sum() + u.sum(), (e, we)))
    for err, args in [(ValueError, dict(x=x[0], w_pre=w)), (ValueError, dict(x=x)), (ValueError, dict(x=x, gate=x, w_pre=w)),
                      (ValueError, dict(x=x, y=x[:2])), (ValueError, dict(x=x, y=x.bfloat16())), (ValueError, dict(x=x, y=x, gate=x[:, :4])),
                      (ValueError, dict(x=x, y=x, w_post=w[:4])), (ValueError, dict(x=x, y=x, w_pre=w.bfloat16())),
                      (H.SwrError, dict(x=x.half(), y=x.half())), (H.SwrError, dict(x=x.cpu(), y=x)),
                      (ValueError, dict(x=torch.zeros(2, 8193, device="cuda"), y=torch.zeros(2, 8193, device="cuda")))]:
        with pytest.raises(err):
            ops.norm_gate_residual(**args)
