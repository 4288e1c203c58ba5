"""64-bit definitions of the sequence operators with the rounding errors their kernels may make, for the tests.

Errors are counted, not fitted.  u = half a step of the tensors' type (bf16 2^-8, fp32 2^-24).  fp32 products run as six products of
three bf16 terms: what is dropped is below 3 * 2^-24 of |a||b|, and the fp32 accumulator takes at most 6 D / 16 steps, so a product of
length D is within f(D) = (6 D / 16 + 24) 2^-24 of its sum of magnitudes (bf16 tensors: D / 16 steps, covered by the same f)."""
import math

import torch


def f(n):
    return (6 * n / 16 + 24) * 2.0 ** -24


def attention(q, k, v, dout, qs, ks, q0, k0, causal, scale=None, bias=None, buckets=None, key_mask=None, train=True):
    """Lists of lengths and first rows per sequence.  -> {name: (value, allowed error)} for out, dq, dk, dv, dbias, in 64 bits.
    bf16: p enters its product rounded to bf16, in a training forward in two bf16 terms (2^-16 of p at most remains); the backward's
    delta starts from the unrounded rows of that forward, and the bias gradient sums fp32 values that were never rounded further."""
    dt, dev = q.dtype, q.device
    bf16 = dt == torch.bfloat16
    u = 2.0 ** -8 if bf16 else 2.0 ** -24
    r = u if bf16 else f(16)                                      # rounding of p and ds before they are multiplied, backward
    rf = (2.0 ** -16 if train else u) if bf16 else r              # ... of p, forward
    H, Hk, D = q.shape[1], k.shape[1], q.shape[2]
    G = H // Hk
    scale = D ** -0.5 if scale is None else scale
    z = lambda t: torch.zeros(t.shape, dtype=torch.float64, device=dev)
    res = {n: [z(t), z(t)] for n, t in (("out", q), ("dq", q), ("dk", k), ("dv", v))}
    if bias is not None:
        res["dbias"] = [z(bias), z(bias)]
        R = buckets.numel() - 1 if causal else buckets.numel() // 2
    for b, (lq, lk) in enumerate(zip(qs, ks)):
        sq, sk = slice(q0[b], q0[b] + lq), slice(k0[b], k0[b] + lk)
        dist = (torch.arange(lq, device=dev) + lk - lq)[:, None] - torch.arange(lk, device=dev)[None]
        ok = dist >= 0 if causal else torch.ones_like(dist, dtype=torch.bool)
        if key_mask is not None:
            ok = ok & key_mask[sk].bool()[None]
        for h in range(H):
            Q, K, V, dO = (t.double() for t in (q[sq, h], k[sk, h // G], v[sk, h // G], dout[sq, h]))
            seen = ok.any(0)[:, None]                             # values nobody sees may be anything
            K, V = torch.where(seen, K, 0.), torch.where(seen, V, 0.)
            s = Q @ K.t() * scale
            mag = Q.abs() @ K.abs().t() * abs(scale)
            if bias is not None:
                slot = buckets[dist.clamp(0, R) if causal else dist.clamp(-R, R) + R].long()
                add = bias.double()[h][slot]
                s = s + add
                mag = mag + torch.where(add.abs() < 1e30, add.abs(), 0.)
            s = s.masked_fill(~ok, -math.inf)
            top = s.max(1, keepdim=True).values if lk else torch.zeros(lq, 1, dtype=torch.float64, device=dev)
            p = torch.exp(s - torch.where(top == -math.inf, 0., top))
            l = p.sum(1, keepdim=True)
            p = torch.where(ok & (l > 0), p / torch.where(l > 0, l, 1.), 0.)
            # a score's error: the product, the scaling and the bias in fp32, the subtraction of the row's maximum
            es = (f(D) + 4 * 2.0 ** -24) * mag + 2.0 ** -23 * torch.where(ok & torch.isfinite(s), s.abs(), 0.)
            row = es.max(1, keepdim=True).values if lk else top
            ep = (es + row + 2.0 ** -20) * p                      # ... of p: numerator, sum of the row, exp2 and division
            o = p @ V
            eo = ep @ V.abs() + (rf + f(lk)) * (p @ V.abs())
            res["out"][0][sq, h] += o
            res["out"][1][sq, h] += eo + u * o.abs()
            dp = dO @ V.t()
            delta = (dO * o).sum(1, keepdim=True)
            size = dO.abs() @ V.abs().t() + (dO.abs() * o.abs()).sum(1, keepdim=True)
            ed = (dO.abs() * (2.0 ** -24 * o.abs() + eo)).sum(1, keepdim=True) + f(D) * size
            ds = p * (dp - delta)
            eds = ep * (dp - delta).abs() + p * ed + 4 * 2.0 ** -24 * p * size
            edsr = eds + r * ds.abs()
            acc = f(lk) + f(lq) * G
            gq, gk, gv = ds @ K * scale, ds.t() @ Q * scale, p.t() @ dO
            res["dq"][0][sq, h] += gq
            res["dq"][1][sq, h] += (edsr @ K.abs() + acc * (ds.abs() @ K.abs())) * abs(scale) + u * gq.abs()
            res["dk"][0][sk, h // G] += gk
            res["dk"][1][sk, h // G] += (edsr.t() @ Q.abs() + acc * (ds.abs().t() @ Q.abs())) * abs(scale) + u * gk.abs()
            res["dv"][0][sk, h // G] += gv
            res["dv"][1][sk, h // G] += (ep + r * p).t() @ dO.abs() + acc * (p.t() @ dO.abs()) + u * gv.abs()
            if bias is not None:
                flat = slot.reshape(-1)
                res["dbias"][0][h].index_add_(0, flat, ds.reshape(-1))
                res["dbias"][1][h].index_add_(0, flat, (eds + f(lk) * ds.abs()).reshape(-1))
    return {n: (t, e) for n, (t, e) in res.items()}


def norm_gate(x, y, gate, w_post, w_pre, scale, eps, dz=None, du=None):
    """-> {name: (value, allowed error)}: z, u and the gradients.  fp32 arithmetic: a value that n roundings lead to is off by at
    most n 2^-24 of its terms' magnitudes; the row sums of N products add log-depth trees of at most 8 * 4 + 8 steps."""
    dt = x.dtype
    u_ = 2.0 ** -8 if dt == torch.bfloat16 else 2.0 ** -24
    e32 = 2.0 ** -24
    d = lambda t: None if t is None else t.double()
    x, y, gate, wp, wn, dz, du = (d(t) for t in (x, y, gate, w_post, w_pre, dz, du))
    rms = lambda t: (t.square().mean(1, keepdim=True) + eps).rsqrt()
    res, rel = {}, 64 * e32
    if y is not None:
        ry = rms(y) if wp is not None else 1.
        yh = y * ry
        n = yh * wp if wp is not None else yh
        sg = torch.sigmoid(gate) if gate is not None else torch.ones_like(x)
        t = scale * sg * n
        z = x + t
        ez = rel * t.abs() + 2 * e32 * (x.abs() + t.abs())
        res["z"] = (z, ez + u_ * z.abs())
    else:
        z, ez = x, torch.zeros_like(x)
    if wn is not None:
        rz = rms(z)
        zh = z * rz
        ezh = ez * rz + zh.abs() * (rel + (ez * z.abs()).mean(1, keepdim=True) * rz * rz)
        res["u"] = (zh * wn, ezh * wn.abs() + (rel + u_) * (zh * wn).abs())
    if dz is None and du is None:
        return res
    g = dz if dz is not None else torch.zeros_like(x)
    eg = torch.zeros_like(x)
    if du is not None:
        a = du * wn
        c = (a * zh).mean(1, keepdim=True)
        ec = (a.abs() * ezh).mean(1, keepdim=True) + rel * (a * zh).abs().mean(1, keepdim=True)
        step = rz * (a - zh * c)
        erz = rel + (ez * z.abs()).mean(1, keepdim=True) * rz * rz
        eg = erz * rz * (a.abs() + (zh * c).abs()) + rz * (ezh * c.abs() + zh.abs() * ec) + rel * rz * (a.abs() + (zh * c).abs())
        g = g + step
        M = x.shape[0]
        res["dw_pre"] = ((du * zh).sum(0), (du.abs() * ezh).sum(0) + (M * e32 + rel) * (du * zh).abs().sum(0))
    eg = eg + 2 * e32 * (g.abs() + (dz.abs() if dz is not None else 0))
    res["dx"] = (g, eg + u_ * g.abs())
    if y is not None:
        dn = g * scale * sg
        edn = eg * abs(scale) * sg + rel * dn.abs()
        if gate is not None:
            # (1 - sigmoid in fp32: off by 4 * 2^-24 absolutely where sigmoid is near 1)
            dgate = g * scale * n * sg * (1 - sg)
            res["dgate"] = (dgate, (eg * abs(scale) * n.abs() + rel * (g * scale * n).abs()) * sg * (1 - sg)
                            + 4 * e32 * (g * scale * n).abs() * sg + (rel + u_) * dgate.abs())
        if wp is not None:
            M = x.shape[0]
            res["dw_post"] = ((dn * yh).sum(0), (edn * yh.abs()).sum(0) + (M * e32 + rel) * (dn * yh).abs().sum(0))
            e = dn * wp
            ee = edn * wp.abs()
            q = (e * yh).mean(1, keepdim=True)
            eq = (ee * yh.abs()).mean(1, keepdim=True) + rel * (e * yh).abs().mean(1, keepdim=True)
            dy = ry * (e - yh * q)
            edy = ry * (ee + yh.abs() * eq + rel * (e.abs() + (yh * q).abs()))
        else:
            dy, edy = dn, edn
        res["dy"] = (dy, edy + (rel + u_) * dy.abs())
    return res


def check(got, want, what, tiny=1e-30):
    value, allowed = want
    err = (got.double() - value).abs()
    bad = ~(err <= allowed + tiny)
    if bad.any():
        i = int((err - allowed).nan_to_num(nan=math.inf).argmax())
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} off; worst {float(got.reshape(-1)[i])} against "
                             f"{float(value.reshape(-1)[i])}, allowed error {float(allowed.reshape(-1)[i]):.3g}, off by {float(err.reshape(-1)[i]):.3g}")
