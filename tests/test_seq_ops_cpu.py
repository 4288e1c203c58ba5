"""Host side of the sequence operators: struct layouts, the bucket table, and the refusals of the C entries (nothing is launched)."""
import ctypes as C
import os
import subprocess
import tempfile

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_struct_layouts_and_limits_match_the_header():
    from scenario_wise_rec import _hip as H
    structs = {"swr_seq_attention_args": H.SeqAttentionArgs, "swr_norm_gate_args": H.NormGateArgs}
    limits = {"SWR_SEQ_MAX_DIM": H.SEQ_MAX_DIM, "SWR_SEQ_MAX_DIST": H.SEQ_MAX_DIST, "SWR_SEQ_MAX_BUCKETS": H.SEQ_MAX_BUCKETS,
              "SWR_SEQ_MAX_TABLE": H.SEQ_MAX_TABLE, "SWR_NORM_GATE_MAX_WIDTH": H.NORM_GATE_MAX_WIDTH}
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "swr.h"', "int main(void){"]
    for cname, ct in structs.items():
        lines.append(f'printf("{cname} %zu\\n", sizeof({cname}));')
        lines += [f'printf("{cname}.{f} %zu\\n", offsetof({cname}, {f}));' for f, _ in ct._fields_]
    lines += [f'printf("{n} %d\\n", {n});' for n in limits] + ["return 0;}"]
    with tempfile.TemporaryDirectory() as d:
        src, exe = os.path.join(d, "t.c"), os.path.join(d, "t")
        open(src, "w").write("\n".join(lines))
        subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), src, "-o", exe], check=True)
        out = subprocess.run([exe], check=True, capture_output=True, text=True).stdout
    got = {k: int(v) for k, v in (line.split() for line in out.strip().splitlines())}
    for cname, ct in structs.items():
        assert got[cname] == C.sizeof(ct)
        assert all(got[f"{cname}.{f}"] == getattr(ct, f).offset for f, _ in ct._fields_)
    assert all(got[n] == v for n, v in limits.items())


@pytest.mark.parametrize("n,far,causal", [(2, 2, True), (3, 9, True), (16, 64, True), (32, 128, True), (32, 128, False), (4, 3, False),
                                          (33, 1000, True), (256, 2000, True), (8, 1000, False)])
def test_bucket_table(n, far, causal):
    from scenario_wise_rec import ops
    t = ops.seq_buckets(n, far, causal, device="cpu")
    assert t.dtype == torch.int32
    side = n if causal else n // 2
    half, one = side // 2, (t if causal else t[far:]).tolist()
    assert len(one) == far + 1 and one[:half] == list(range(half)) and one[-1] == side - 1
    assert all(a <= b <= a + 1 or b >= half for a, b in zip(one, one[1:])) and one == sorted(one)
    for r in range(half, far + 1):                 # bucket half + t: ratio >= t / (side - half) of the way, in logarithms
        step = (one[r] - half) / (side - half)
        assert (r / half) >= (far / half) ** step * (1 - 1e-12)
        assert one[r] == side - 1 or (r / half) < (far / half) ** (step + 1 / (side - half)) * (1 + 1e-12)
    if not causal:
        back = t[:far].flip(0).tolist()            # distances -1, -2, ...: the other half of the buckets
        assert back == [b + side for b in one[1:]]


def test_bucket_table_refusals():
    from scenario_wise_rec import ops
    for args in ((1, 10, True), (0, 10, True), (7, 10, False), (2, 10, False), (300, 1000, True), (32, 16, True), (32, 5000, True), (32, 1100, False)):
        with pytest.raises(ValueError):
            ops.seq_buckets(*args, device="cpu")


def attention_args(**kw):
    from scenario_wise_rec import _hip as H
    a = H.SeqAttentionArgs()
    # (addresses that are never read: every call below is refused before a launch)
    a.Tq = a.Tk = 64
    a.B, a.Hq, a.Hk, a.D, a.dtype, a.causal, a.max_q, a.max_k, a.scale = 2, 4, 2, 16, H.F32, 1, 64, 64, 1.0
    for n in ("q", "k", "v", "out", "cu_q", "cu_k"):
        setattr(a, n, 4096)
    for n, v in kw.items():
        setattr(a, n, v)
    return a


def test_attention_entry_refuses():
    from scenario_wise_rec import _hip as H
    lib = H.lib
    call = lambda a, ws=None, n=0: lib.swr_seq_attention_fwd(C.byref(a), ws, n, None)
    assert lib.swr_seq_attention_fwd(None, None, 0, None) == -1
    for want, kw in [(-1, dict(B=-1)), (-1, dict(q=None)), (-1, dict(v=None)), (-1, dict(cu_q=None)), (-1, dict(out=None)), (-1, dict(D=0)),
                     (-1, dict(Hk=0)), (-1, dict(Hq=1)), (-1, dict(max_q=-1)), (-1, dict(n_dist=-1)), (-1, dict(n_dist=9)),
                     (-2, dict(dtype=H.F16)), (-2, dict(dtype=0)), (-3, dict(out=4104)), (-5, dict(D=129)), (-5, dict(Hk=3)),
                     (-5, dict(Tq=1 << 31)), (-5, dict(n_dist=8, n_buckets=4, bias=4096, buckets=4096, causal=0)),
                     (-5, dict(n_dist=5000, n_buckets=4, bias=4096, buckets=4096)),
                     (-5, dict(n_dist=2049, n_buckets=4, bias=4096, buckets=4096, Hq=12)), (-5, dict(Hq=200)), (-5, dict(B=1 << 30)),
                     (-5, dict(n_dist=9, n_buckets=257, bias=4096, buckets=4096))]:
        a = attention_args(**kw)
        assert call(a) == want, kw
        assert lib.swr_seq_attention_fwd_workspace_bytes(C.byref(a)) == 0
    # few queries over many keys: split, and refused without its workspace
    a = attention_args(Tq=2, max_q=1, Tk=20000, max_k=10000)
    need = lib.swr_seq_attention_fwd_workspace_bytes(C.byref(a))
    assert need > 0
    assert call(a) == -6 and call(a, 4096, need - 1) == -6 and call(a, 4104, need) == -3
    back = dict(lse=4096, dout=4096, dq=4096, dk=4096, dv=4096)
    bwd = lambda a, ws=None, n=0: lib.swr_seq_attention_bwd(C.byref(a), ws, n, None)
    for want, kw in [(-1, dict(back, lse=None)), (-1, dict(back, dk=None)), (-1, dict(back, dtype=H.BF16)), (-3, dict(back, dq=4100)), (-6, back)]:
        assert bwd(attention_args(**kw)) == want, kw
    a = attention_args(**back)
    assert bwd(a, 4096, lib.swr_seq_attention_bwd_workspace_bytes(C.byref(a)) - 1) == -6


def test_attention_refuses_a_bias_elsewhere(monkeypatch):
    """A bias (or its buckets) on another device than the queries is refused before any pointer is taken."""
    from scenario_wise_rec import _hip as H, ops
    monkeypatch.setattr(H, "require_device", lambda *t: None)
    q = torch.zeros(4, 2, 8, device="meta")
    cu = torch.zeros(2, dtype=torch.int32, device="meta")
    table = ops.seq_buckets(4, 8, device="cpu")
    with pytest.raises(H.SwrError, match="bias is on cpu"):
        ops.seq_attention(q, q, q, cu, bias=torch.zeros(2, 4), buckets=table.to("meta"))
    with pytest.raises(H.SwrError, match="buckets is on cpu"):
        ops.seq_attention(q, q, q, cu, bias=torch.zeros(2, 4, device="meta"), buckets=table)


def test_norm_entry_refuses():
    from scenario_wise_rec import _hip as H
    lib = H.lib
    base = dict(M=8, N=64, dtype=H.BF16, x=4096, y=4096, z=4096)

    def args(**kw):
        a = H.NormGateArgs()
        for n, v in dict(base, **kw).items():
            setattr(a, n, v)
        return a
    for want, kw in [(-1, dict(M=-1)), (-1, dict(N=0)), (-1, dict(x=None)), (-1, dict(y=None)), (-1, dict(z=None)), (-1, dict(w_pre=4096)),
                     (-1, dict(y=None, w_pre=4096, u=4096, gate=4096)), (-2, dict(dtype=H.F64)), (-5, dict(N=8193))]:
        assert lib.swr_norm_gate_fwd(C.byref(args(**kw)), None) == want, kw
    back = dict(dz=4096, dx=4096, dy=4096)
    for want, kw in [(-1, dict(back, dx=None)), (-1, dict(back, dy=None)), (-1, dict(back, dz=None)), (-1, dict(back, du=4096)),
                     (-1, dict(back, gate=4096)), (-1, dict(back, w_post=4096)), (-6, dict(back, w_post=4096, ry=4096, dw_post=4096))]:
        assert lib.swr_norm_gate_bwd(C.byref(args(**kw)), None, 0, None) == want, kw
    assert lib.swr_norm_gate_bwd_workspace_bytes(8, 8193) == 0 and lib.swr_norm_gate_bwd_workspace_bytes(100, 64) > 0


def test_only_attention_pooling_adds_parameters():
    from scenario_wise_rec.basic.features import SequenceFeature, SparseFeature
    from scenario_wise_rec.basic.layers import EmbeddingLayer
    plain = EmbeddingLayer([SparseFeature("a", 5, 4), SequenceFeature("h", 7, 4, pooling="mean")])
    assert sorted(plain.state_dict()) == ["embed_dict.a.weight", "embed_dict.h.weight"]
    att = EmbeddingLayer([SequenceFeature("h", 7, 8, pooling="attention", attention={"n_heads": 2, "n_buckets": 4, "max_distance": 9})])
    keys = sorted(k for k in att.state_dict() if k.startswith("seq_blocks.h."))
    assert [k[len("seq_blocks.h."):] for k in keys] == [
        "gate.network.0.bias", "gate.network.0.weight", "gate.network.2.bias", "gate.network.2.weight", "norm_in", "norm_out",
        "out.weight", "position", "qkv.weight"]
    assert tuple(att.state_dict()["seq_blocks.h.position"].shape) == (2, 4)
