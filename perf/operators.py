"""Measured cases of the sequence operators: packed attention with a bucketed relative position bias (training, whole prompts,
a few new tokens over cached histories) and the norms around a block fused with its gate and residual scale.

`run` computes a case in plain torch operations where `own` is false, through `scenario_wise_rec.ops` where it is true; `exact` is
the definition in 64 bits, one sequence and head at a time.
"""
import math
import os
import random
import sys

import torch

own = False

_DT = {"fp32": torch.float32, "bf16": torch.bfloat16}


def _ops():
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "scenario-wise-rec_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from scenario_wise_rec import ops
    return ops


# ---------------------------------------------------------------------------------------------------------------- cases
def _attn(name, **kw):
    case = {"op": "attention", "train": False, "dtype": "bf16", "n": 1, "lo": 1, "hi": 1, "mix": 1, "new": 0, "heads": 4,
            "kv_heads": 4, "dim": 16, "causal": True, "buckets": 32, "max_distance": 128}
    case.update(kw)
    if name:
        case["name"] = name
    return case


def _norm(name, **kw):
    case = {"op": "norm", "train": False, "dtype": "fp32", "rows": 1, "width": 64, "gate": True, "post": True, "pre": True}
    case.update(kw)
    if name:
        case["name"] = name
    return case


def listed():
    return [
        # one user's next event against a cached history: the smallest call, latency counts
        _attn("step_one_fp32", dtype="fp32", n=1, lo=500, hi=500, new=1, heads=4, kv_heads=4, dim=16, buckets=16, max_distance=64),
        # a training step over short behaviour histories at this framework's embedding width (E = 64 as 4 heads of 16)
        _attn("train_short_fp32", train=True, dtype="fp32", n=1024, lo=1, hi=50, heads=4, kv_heads=4, dim=16, buckets=16,
              max_distance=64),
        # longer histories, shared key / value heads
        _attn("train_history_fp32", train=True, dtype="fp32", n=512, lo=20, hi=200, heads=8, kv_heads=4, dim=32),
        # packed sequences of very different lengths
        _attn("train_packed_bf16", train=True, n=24, lo=1, hi=2048, heads=16, kv_heads=4, dim=64),
        # long sequences, wide heads
        _attn("train_long_bf16", train=True, n=4, lo=2000, hi=4096, heads=16, kv_heads=8, dim=128),
        # whole prompts before the first answer: the largest product
        _attn("prompt_bf16", n=8, lo=300, hi=8192, heads=32, kv_heads=8, dim=128),
        # histories scored in both directions (no causal border), a head width between two tile sizes
        _attn("prompt_both_ways_fp32", dtype="fp32", n=64, lo=100, hi=600, heads=8, kv_heads=8, dim=48, causal=False, buckets=32,
              max_distance=100),
        # one new token for each of many users over long caches: the keys and values are read once
        _attn("step_many_bf16", n=128, lo=1, hi=8192, new=1, heads=32, kv_heads=8, dim=128),
        # a few new events (or candidates) at a time over fp32 caches
        _attn("chunk_fp32", dtype="fp32", n=32, lo=100, hi=4000, new=13, heads=8, kv_heads=2, dim=64),
        # norms of one small serving request
        _norm("norm_serve_fp32", rows=37, width=64),
        # norms of a training step, wide rows
        _norm("norm_train_bf16", train=True, dtype="bf16", rows=32768, width=1024),
        # ... and at this framework's widest concat (452 columns, batch 32 768), no post-norm
        _norm("norm_train_fp32", train=True, dtype="fp32", rows=32768, width=452, post=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw_once(rng):
    kind = rng.choice(["train", "train", "prompt", "step", "chunk", "norm", "norm"])
    dtype = rng.choice(["fp32", "bf16"])
    if kind == "norm":
        return _norm(None, train=rng.random() < 0.6, dtype=dtype, rows=_log(rng, 1, 40000), width=_log(rng, 16, 2048),
                     gate=rng.random() < 0.7, post=rng.random() < 0.7, pre=rng.random() < 0.8)
    kv = rng.choice([1, 2, 3, 4, 8])
    group = rng.choice([1, 2, 4, 5])
    dim = rng.choice([8, 12, 16, 20, 24, 32, 40, 48, 64, 64, 80, 96, 112, 128, 128])
    hi = _log(rng, 16, 8192)
    lo = rng.choice([1, max(1, hi // 3), hi])
    rel = rng.choice([0, 8, 16, 32])
    kw = dict(dtype=dtype, n=_log(rng, 1, 512), lo=lo, hi=hi, mix=rng.randrange(1 << 16), heads=kv * group, kv_heads=kv, dim=dim,
              buckets=rel, max_distance=rng.choice([33, 64, 128, 200]))
    if kind == "train":
        return _attn(None, train=True, causal=rng.random() < 0.75, **kw)
    if kind == "prompt":
        return _attn(None, causal=rng.random() < 0.75, **kw)
    return _attn(None, new=1 if kind == "step" else rng.randrange(2, 33), **kw)


def draw(rng):
    """One more case: as the listed ones, sizes spread over their ranges, no dearer than the dearest listed one of its kind."""
    flops, nbytes = {}, {}
    for c in listed():
        w, key = work(c), (c["op"], c["dtype"])
        flops[key] = max(flops.get(key, 0), w["flops"])
        nbytes[key] = max(nbytes.get(key, 0), w["bytes"])
    while True:
        c = _draw_once(rng)
        w, key = work(c), (c["op"], c["dtype"])
        if w["flops"] > flops[key] or w["bytes"] > nbytes[key]:
            continue
        if c["op"] == "attention":
            # the plain form's padded score blocks: those of the largest listed cases at most
            scores = c["heads"] * c["n"] * c["hi"] * (c["new"] or c["hi"])
            if scores > (1 << 31 if c["train"] else 1 << 34):
                continue
        return c


def _lengths(case):
    """(new tokens, history length) of every sequence; new == history for prompts and training."""
    rng = random.Random(case["mix"] * 7919 + case["n"])
    ks = [rng.randint(case["lo"], case["hi"]) for _ in range(case["n"])]
    if case["n"] > 1:
        ks[rng.randrange(case["n"])] = case["hi"]
    if case["new"]:
        qs = [case["new"]] * case["n"]
        ks = [max(k, case["new"]) for k in ks]
    else:
        qs = list(ks)
    return qs, ks


def _pairs(case):
    total = 0
    for lq, lk in zip(*_lengths(case)):
        total += (lq * (lk - lq) + lq * (lq + 1) // 2) if case["causal"] else lq * lk
    return total


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "norm":
        mats = 2 + int(case["gate"]) + 1 + int(case["pre"])                    # x, y, gate -> z, u
        flops = 14 * case["rows"] * case["width"]
        if case["train"]:
            mats += 1 + int(case["pre"]) + 2 + int(case["gate"])                # dz, du -> dx, dy, dgate
            flops *= 3
        return {"bytes": mats * case["rows"] * case["width"] * size + 16 * case["width"], "flops": flops}
    qs, ks = _lengths(case)
    tq, tk, d = sum(qs), sum(ks), case["dim"]
    q, kv = tq * case["heads"] * d * size, 2 * tk * case["kv_heads"] * d * size
    per_pair = 4 * d * case["heads"]
    if not case["train"]:
        return {"bytes": 2 * q + kv, "flops": per_pair * _pairs(case)}
    # forward 2 products, backward 5; q, k, v, out, dout in, out, dq, dk, dv out
    return {"bytes": 4 * q + 2 * kv, "flops": per_pair * 7 // 2 * _pairs(case)}


# --------------------------------------------------------------------------------------------------------------- inputs
def _bucket_table(n_buckets, max_distance, causal):
    """Bucket of every relative distance: exact up to half of the (one-sided) buckets, then logarithmic up to max_distance.
    Causal: entry r = distance r = 0 .. max_distance.  Both ways: entry r = distance r - max_distance, halves by sign."""
    side = n_buckets if causal else n_buckets // 2
    half = side // 2

    def one(r):
        if r < half:
            return r
        b = half
        # the largest b with half * (max_distance / half)^((b - half) / (side - half)) <= r, in whole numbers
        while b + 1 < side and max_distance ** (b + 1 - half) * half ** (side - half) <= r ** (side - half) * half ** (b + 1 - half):
            b += 1
        return b
    if causal:
        return [one(r) for r in range(max_distance + 1)]
    return [one(abs(r)) + (side if r < 0 else 0) for r in range(-max_distance, max_distance + 1)]


def prepare(case, seed):
    dev, dt = torch.device("cuda"), _DT[case["dtype"]]
    g = torch.Generator(device=dev)
    g.manual_seed(seed)

    def rand(*shape, dtype=dt, scale=1.0):
        t = torch.randn(*shape, generator=g, device=dev, dtype=dtype)
        return t.mul_(scale) if scale != 1.0 else t
    st = {"case": case}
    if case["op"] == "norm":
        M, N = case["rows"], case["width"]
        st["x"], st["y"] = rand(M, N), rand(M, N, scale=1.5)
        st["gate"] = rand(M, N) if case["gate"] else None
        st["w_post"] = 1 + rand(N, dtype=torch.float32, scale=0.1) if case["post"] else None
        st["w_pre"] = 1 + rand(N, dtype=torch.float32, scale=0.1) if case["pre"] else None
        st["scale"] = 0.5
        if case["train"]:
            st["dz"], st["du"] = rand(M, N, scale=0.1), (rand(M, N, scale=0.1) if case["pre"] else None)
            for k in ("x", "y", "gate", "w_post", "w_pre"):
                if st[k] is not None:
                    st[k].requires_grad_(True)
        return st
    qs, ks = _lengths(case)
    H, Hk, D = case["heads"], case["kv_heads"], case["dim"]
    cap = list(ks)
    if case["new"]:                            # a cache: every history has room to grow behind it
        cap = [(k + 63) // 64 * 64 for k in ks]
    st["q"] = rand(sum(qs), H, D)
    st["k"], st["v"] = rand(sum(cap), Hk, D), rand(sum(cap), Hk, D)
    prefix = lambda v: torch.tensor([0] + list(torch.tensor(v).cumsum(0)), dtype=torch.int32, device=dev)
    st["cu_q"] = prefix(qs)
    st["cu_k"] = prefix(cap) if case["new"] else st["cu_q"]
    st["k_len"] = torch.tensor(ks, dtype=torch.int32, device=dev) if case["new"] else None
    st["q_lens"], st["k_lens"], st["max_q"], st["max_k"] = qs, ks, max(qs), max(ks)
    st["bias"], st["table"] = None, None
    if case["buckets"]:
        st["bias"] = rand(H, case["buckets"], dtype=torch.float32, scale=0.5)
        st["table"] = torch.tensor(_bucket_table(case["buckets"], case["max_distance"], case["causal"]), dtype=torch.int32, device=dev)
    if case["train"]:
        st["dout"] = rand(sum(qs), H, D, scale=0.1)
        for k in ("q", "k", "v", "bias"):
            if st[k] is not None:
                st[k].requires_grad_(True)
    return st


# ----------------------------------------------------------------------------------------------------------- plain forms
def _plain_attention(q, k, v, bias, st, added):
    """Sequences padded to a rectangle (as many at a time as keep the score block below 2^30 elements), masked softmax.  `added`
    collects (bias of every score, bucket of every score) for the bias gradient."""
    case = st["case"]
    H, Hk, D = case["heads"], case["kv_heads"], case["dim"]
    n, dev = case["n"], q.device
    cu_q, cu_k = st["cu_q"].long(), st["cu_k"].long()
    lq_all, lk_all = torch.tensor(st["q_lens"], device=dev), torch.tensor(st["k_lens"], device=dev)
    out = torch.zeros_like(q)
    parts, rows = [], []
    step = max(1, (1 << 30) // (H * st["max_q"] * st["max_k"]))
    for b0 in range(0, n, step):
        b1 = min(b0 + step, n)
        LQ, LK = max(st["q_lens"][b0:b1]), max(st["k_lens"][b0:b1])
        iq, ik = torch.arange(LQ, device=dev), torch.arange(LK, device=dev)
        lq, lk = lq_all[b0:b1, None], lk_all[b0:b1, None]
        has_q, has_k = iq < lq, ik < lk
        at_q = torch.where(has_q, cu_q[b0:b1, None] + iq, 0)
        at_k = torch.where(has_k, cu_k[b0:b1, None] + ik, 0)
        qq = q[at_q].transpose(1, 2)                                            # [b, H, LQ, D]
        kk = k[at_k].transpose(1, 2).repeat_interleave(H // Hk, 1)
        vv = v[at_k].transpose(1, 2).repeat_interleave(H // Hk, 1)
        s = torch.matmul(qq, kk.transpose(2, 3)) * (1.0 / math.sqrt(D))
        dist = (iq + (lk - lq))[:, :, None] - ik                               # [b, LQ, LK]
        keep = has_q[:, :, None] & has_k[:, None, :]
        if case["causal"]:
            keep = keep & (dist >= 0)
        if bias is not None:
            if case["causal"]:
                entry = dist.clamp(0, case["max_distance"])
            else:
                entry = dist.clamp(-case["max_distance"], case["max_distance"]) + case["max_distance"]
            slot = st["table"][entry].long()
            add = bias.detach()[:, slot].transpose(0, 1).requires_grad_(case["train"])
            added.append((add, slot))
            s = s + add
        s = s.masked_fill(~keep[:, None], float("-inf"))
        top = s.amax(3, keepdim=True).detach()
        p = torch.exp(s - torch.where(top == float("-inf"), 0.0, top))
        total = p.sum(3, keepdim=True)
        o = torch.matmul(p / torch.where(total == 0, 1.0, total), vv)
        parts.append(o.transpose(1, 2)[has_q])
        rows.append(at_q[has_q])
    return out.index_copy(0, torch.cat(rows), torch.cat(parts))


def _plain_bias_grad(dscores, slots, n_buckets):
    """Sum of the score gradients of every (head, bucket): a product with the buckets' 0 / 1 columns."""
    total = 0
    for ds, slot in zip(dscores, slots):
        n, H, scores = ds.shape[0], ds.shape[1], ds.shape[2] * ds.shape[3]
        step = max(1, (1 << 30) // (scores * n_buckets))
        for b in range(0, n, step):
            columns = (slot[b:b + step].reshape(-1, scores, 1) == torch.arange(n_buckets, device=ds.device)).float()
            total = total + torch.matmul(ds[b:b + step].reshape(-1, H, scores), columns).sum(0)
    return total


def _plain_norm(x, y, gate, w_post, w_pre, scale, eps=1e-6):
    t = y
    if w_post is not None:
        t = y * torch.rsqrt((y * y).mean(1, keepdim=True) + eps) * w_post
    if gate is not None:
        t = t / (1 + torch.exp(-gate))
    z = x + scale * t
    if w_pre is None:
        return z, None
    return z, z * torch.rsqrt((z * z).mean(1, keepdim=True) + eps) * w_pre


def _leaves(st, names):
    return [None if st[k] is None else st[k].detach().float().requires_grad_(st["case"]["train"]) for k in names]


def _grads(outs, douts, leaves, st, names):
    have = [i for i, t in enumerate(leaves) if t is not None]
    got = torch.autograd.grad(outs, [leaves[i] for i in have], douts)
    return [g.to(st[names[i]].dtype) for i, g in zip(have, got)]


def run(state):
    st, case = state, state["case"]
    if case["op"] == "norm":
        names = ("x", "y", "gate", "w_post", "w_pre")
        if own:
            got = _ops().norm_gate_residual(st["x"], st["y"], gate=st["gate"], w_post=st["w_post"], w_pre=st["w_pre"], scale=st["scale"])
            outs = list(got) if case["pre"] else [got]
            if not case["train"]:
                return outs
            grads = torch.autograd.grad(outs, [st[k] for k in names if st[k] is not None], [st["dz"], st["du"]][:len(outs)])
            return [o.detach() for o in outs] + list(grads)
        leaves = _leaves(st, names)
        outs = [o for o in _plain_norm(*leaves, st["scale"]) if o is not None]
        res = [o.detach().to(st["x"].dtype) for o in outs]
        if case["train"]:
            res += _grads(outs, [d.float() for d in (st["dz"], st["du"]) if d is not None], leaves, st, names)
        return res
    names = ("q", "k", "v", "bias")
    if own:
        out = _ops().seq_attention(st["q"], st["k"], st["v"], st["cu_q"], st["cu_k"], max_q=st["max_q"], max_k=st["max_k"],
                                   k_len=st["k_len"], causal=case["causal"], bias=st["bias"], buckets=st["table"])
        if not case["train"]:
            return out
        return [out.detach()] + list(torch.autograd.grad(out, [st[k] for k in names if st[k] is not None], st["dout"]))
    leaves, added = _leaves(st, names), []
    out = _plain_attention(*leaves, st, added)
    if not case["train"]:
        return out.to(st["q"].dtype)
    got = torch.autograd.grad(out, leaves[:3] + [a for a, _slot in added], st["dout"].float())
    res = [out.detach().to(st["q"].dtype)] + [g.to(st["q"].dtype) for g in got[:3]]
    if case["buckets"]:
        res.append(_plain_bias_grad(got[3:], [slot for _a, slot in added], case["buckets"]))
    return res


# ------------------------------------------------------------------------------------------------------- 64-bit definition
def exact(case, seed):
    st = prepare(case, seed)
    d64 = lambda t: None if t is None else t.detach().double()
    if case["op"] == "norm":
        x, y, gate, wp, wn = (d64(st[k]) for k in ("x", "y", "gate", "w_post", "w_pre"))
        N, s, eps = case["width"], st["scale"], 1e-6
        ry = (y.square().sum(1, keepdim=True) / N + eps).sqrt().reciprocal() if wp is not None else None
        yhat = y * ry if wp is not None else y
        sig = torch.sigmoid(gate) if gate is not None else torch.ones_like(x)
        z = x + s * sig * (yhat * wp if wp is not None else yhat)
        res = [z]
        if wn is not None:
            rz = (z.square().sum(1, keepdim=True) / N + eps).sqrt().reciprocal()
            res.append(z * rz * wn)
        if not case["train"]:
            return res
        dz, g_wn = d64(st["dz"]), None
        if wn is not None:
            du, zhat = d64(st["du"]), z * rz
            g_wn = (du * zhat).sum(0)
            dzh = du * wn
            dz = dz + rz * (dzh - zhat * (dzh * zhat).mean(1, keepdim=True))
        t = dz * (s * sig)
        g_gate = dz * s * (yhat * wp if wp is not None else yhat) * sig * (1 - sig) if gate is not None else None
        if wp is not None:
            g_wp, th = (t * yhat).sum(0), t * wp
            dy = ry * (th - yhat * (th * yhat).mean(1, keepdim=True))
        else:
            g_wp, dy = None, t
        return res + [g for g in (dz, dy, g_gate, g_wp, g_wn) if g is not None]
    H, Hk, D, G = case["heads"], case["kv_heads"], case["dim"], case["heads"] // case["kv_heads"]
    # whole tensors stay in their own type, 64-bit copies are made of one head at a time
    q, k, v, bias = (st[n] if st[n] is None else st[n].detach() for n in ("q", "k", "v", "bias"))
    dev, train = q.device, case["train"]
    out = torch.zeros(q.shape, dtype=torch.float64, device=dev)
    if train:
        dq, dk, dv = (torch.zeros(t.shape, dtype=torch.float64, device=dev) for t in (q, k, v))
        dbias = torch.zeros(bias.shape, dtype=torch.float64, device=dev) if bias is not None else None
    cq, ck = st["cu_q"].tolist(), st["cu_k"].tolist()
    R = case["max_distance"]
    for b in range(case["n"]):
        lq, lk = st["q_lens"][b], st["k_lens"][b]
        sq, sk = slice(cq[b], cq[b] + lq), slice(ck[b], ck[b] + lk)
        far = torch.arange(lk - lq, lk, device=dev)[:, None] - torch.arange(lk, device=dev)[None, :]
        hidden = far < 0 if case["causal"] else torch.zeros_like(far, dtype=torch.bool)
        if bias is not None:
            slot = st["table"][far.clamp(min=0, max=R) if case["causal"] else far.clamp(min=-R, max=R) + R].long()
        wide = max(1, (1 << 27) // (lq * lk))                       # heads at a time
        for h0 in range(0, H, wide):
            hs = slice(h0, min(h0 + wide, H))
            of = torch.arange(h0, min(h0 + wide, H), device=dev) // G
            Q = q[sq, hs].double().permute(1, 0, 2).contiguous()
            K, V = (t[sk][:, of].double().permute(1, 0, 2).contiguous() for t in (k, v))
            S = torch.bmm(Q, K.permute(0, 2, 1).contiguous()).div_(D ** 0.5)
            if bias is not None:
                S += bias[hs].double()[:, slot]
            S.masked_fill_(hidden, -math.inf)
            P = torch.softmax(S, -1)
            del S
            O = torch.bmm(P, V)
            out[sq, hs] = O.permute(1, 0, 2)
            if not train:
                continue
            dO = st["dout"][sq, hs].double().permute(1, 0, 2).contiguous()
            dS = torch.bmm(dO, V.permute(0, 2, 1).contiguous())
            dS = P * (dS - (dO * O).sum(-1, keepdim=True))
            dq[sq, hs] = (torch.bmm(dS, K) / D ** 0.5).permute(1, 0, 2)
            gk = torch.bmm(dS.permute(0, 2, 1).contiguous(), Q) / D ** 0.5
            gv = torch.bmm(P.permute(0, 2, 1).contiguous(), dO)
            dk[sk] = dk[sk].index_add(1, of, gk.permute(1, 0, 2))
            dv[sk] = dv[sk].index_add(1, of, gv.permute(1, 0, 2))
            if dbias is not None:
                for i in range(dS.shape[0]):
                    dbias[h0 + i] += torch.zeros_like(dbias[0]).index_add(0, slot.reshape(-1), dS[i].reshape(-1))
    if not train:
        return out
    return [out, dq, dk, dv] + ([dbias] if dbias is not None else [])
