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


GEOMETRY = r"""
#include <cstdio>
#include <vector>
#include "seq_geometry.h"
// sa_unit of the kernels
static int unit_of(int id, const SaGrid& g, int& within) {
    const int slot = id >> 3, round = slot / (g.per_unit * g.together), r = slot % (g.per_unit * g.together);
    within = r / g.together;
    return (round * g.together + r % g.together) * 8 + (id & 7);
}
int main() {
    int bad = 0;
    // every piece of work has one workgroup, so have the rows of no sequence
    for (int64_t units : {0, 1, 7, 8, 300}) for (int64_t tiles : {1, 3, 40}) for (int64_t inner : {1, 5}) for (int64_t together : {0, 1, 3}) {
        const SaGrid g = sa_grid(units, tiles, inner, together, 64);
        std::vector<int> hit((units + g.rest) * g.per_unit, 0);
        for (unsigned id = 0; id < g.blocks; ++id) {
            int within;
            const int u = unit_of(id, g, within);
            if (u < units + g.rest) ++hit[u * g.per_unit + within];
        }
        for (int h : hit) bad += h != 1;
        bad += g.tiles != tiles || g.per_unit != tiles * inner || g.rest * g.per_unit < 256;
    }
    printf("small %d\n", bad);
    // at the cap: tiles cut down, consistent in themselves, and the same when asked with what came out
    const int64_t big[][3] = {{8000007, 500, 1}, {131072, 32, 4}, {524288, 16, 4}, {1 << 27, 1, 1}, {1 << 20, 1 << 26, 93}, {1, 1 << 26, 4096}, {(1 << 30) - 1, 1, 1}};
    for (auto& c : big) for (int64_t together : {0, 1}) for (int threads : {64, 128, 256}) {
        const SaGrid g = sa_grid(c[0], c[1], c[2], together, threads);
        if (!g.blocks) { printf("none\n"); continue; }
        const SaGrid again = sa_grid(c[0], g.tiles, c[2], together, threads);
        printf("%d %d %d %d %u\n", g.tiles, g.per_unit == g.tiles * (int)c[2] && g.tiles >= 1, again.tiles == g.tiles && again.blocks >= g.blocks / 2,
               (long long)g.blocks * threads < (1ll << 32), g.blocks);
    }
}
"""


def geometry(tmp_path):
    import os
    import subprocess
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    (tmp_path / "g.cpp").write_text(GEOMETRY)
    subprocess.run(["g++", "-std=c++17", "-I", os.path.join(root, "scenario-wise-rec_amd", "csrc"), str(tmp_path / "g.cpp"), "-o", str(tmp_path / "g")], check=True)
    return subprocess.run([str(tmp_path / "g")], check=True, capture_output=True, text=True).stdout.split("\n")


def test_launch_geometry_is_whole_and_computed_once(tmp_path):
    """Every piece of work belongs to one workgroup; a launch cut down at the grid's cap is consistent with the tiles that partial sums
    are laid out by, also when it is asked for again with them."""
    lines = geometry(tmp_path)
    assert lines[0] == "small 0"
    cut = [line.split() for line in lines[1:] if line and line != "none"]
    assert cut and all(c[1:3] == ["1", "1"] for c in cut), lines
    assert all(c[3] == "1" for c in cut), lines                      # (fewer than 2^32 threads)


def test_backward_workspace_follows_the_launched_tiles():
    """Partial sums of the bias gradient: one per bucket, sequence and launched tile, for a launch at the cap of the grid, too."""
    from test_seq_ops_cpu import attention_args
    import ctypes as C
    from scenario_wise_rec import _hip as H
    a = attention_args(B=8000007, Hq=1, Hk=1, Tq=64000, Tk=64000, max_q=64000, max_k=64, n_dist=9, n_buckets=4, bias=4096, buckets=4096,
                       lse=4096, dout=4096, dq=4096, dk=4096, dv=4096, dbias=4096)
    nbytes = H.lib.swr_seq_attention_bwd_workspace_bytes(C.byref(a))
    tiles, left = divmod(nbytes - 256 - 64000 * 4, 8000007 * 4 * 4)
    assert left == 0 and 1 <= tiles <= 500


def test_launches_of_many_sequences_stay_below_the_grid_limit():
    """Many sequences with one long one among them: fewer tiles are launched (and walked in more rounds), not more threads than a grid takes.
    More sequences than workgroups fit are refused."""
    from test_seq_ops_cpu import attention_args
    import ctypes as C
    from scenario_wise_rec import _hip as H
    back = dict(lse=4096, dout=4096, dq=4096, dk=4096, dv=4096)
    tab = dict(n_dist=9, n_buckets=4, bias=4096, buckets=4096, dbias=4096)
    for B, Hk, G, longest in ((16384, 8, 4, 4096), (65536, 4, 4, 2048)):
        a = attention_args(B=B, Hq=Hk * G, Hk=Hk, Tq=1 << 20, Tk=1 << 20, max_q=longest, max_k=longest, D=64, **back, **tab)
        nbytes = H.lib.swr_seq_attention_bwd_workspace_bytes(C.byref(a))
        tiles, left = divmod(nbytes - 256 - (1 << 22) * Hk * G, B * 4 * Hk * G * 4)
        assert left == 0 and 1 <= tiles and B * Hk * G * tiles * 256 < 1 << 32
    a = attention_args(B=1 << 26, Hq=1, Hk=1, **back)
    assert H.lib.swr_seq_attention_fwd(C.byref(a), None, 0, None) == -5 and H.lib.swr_seq_attention_bwd(C.byref(a), None, 0, None) == -5
    # (two million rows of 93 heads: the launch that joins key ranges would not fit, so none are made)
    a = attention_args(Tq=1 << 21, B=1, Hq=93, Hk=1, max_q=1, Tk=20000, max_k=20000)
    assert H.lib.swr_seq_attention_fwd_workspace_bytes(C.byref(a)) == 0


def test_a_max_q_below_the_mean_does_not_blow_up_the_workspace():
    """The hint is right for any value: one sequence of a million queries called with max_q = 1 asked for 64 key ranges of every row."""
    from test_seq_ops_cpu import attention_args
    import ctypes as C
    from scenario_wise_rec import _hip as H
    need = lambda **kw: H.lib.swr_seq_attention_fwd_workspace_bytes(C.byref(attention_args(**kw)))
    for dtype in (H.F32, H.BF16):
        for rows in (1, 100, 5000, 1 << 17, 1 << 20):
            assert need(dtype=dtype, B=1, Tq=rows, max_q=1, Tk=1 << 20, max_k=1 << 20) <= 1 << 27, rows
    assert need(B=1, Tq=1, max_q=1, Tk=20000, max_k=20000) > 0                   # (an honest hint still splits the keys)


def test_norm_backward_refuses_a_missing_row_statistic():
    """The kernel reads rz wherever w_pre is given, with or without du; a NULL there was a read through it."""
    import ctypes as C
    from scenario_wise_rec import _hip as H
    a = H.NormGateArgs()
    for name, value in dict(M=8, N=64, dtype=H.F32, x=4096, y=4096, w_pre=4096, dz=4096, dx=4096, dy=4096, dw_post=4096).items():
        setattr(a, name, value)
    assert H.lib.swr_norm_gate_bwd(C.byref(a), None, 0, None) == -1
    a.rz = 4096                                            # (the next check is the workspace's)
    assert H.lib.swr_norm_gate_bwd(C.byref(a), None, 0, None) == -6


def test_as_many_sequences_as_documented_fit():
    """B * Hq = 2^24 - 4096 in any split over heads: a workspace (of the backward) is given, nothing is refused."""
    from test_seq_ops_cpu import attention_args
    import ctypes as C
    from scenario_wise_rec import _hip as H
    for Hq, Hk in ((1, 1), (4, 1), (4, 4), (64, 8), (32, 1)):
        for D in (16, 33, 128):
            a = attention_args(B=((1 << 24) - 4096) // Hq, Hq=Hq, Hk=Hk, D=D, max_q=5000, max_k=5000, lse=4096, dout=4096, dq=4096, dk=4096, dv=4096)
            assert H.lib.swr_seq_attention_bwd(C.byref(a), None, 0, None) == -6, (Hq, Hk, D)         # (only the workspace is missing)
