"""The label and attention operators in 64 bits, from their formulas, with a bound on how far the kernels' results may be.

Bounds: a sum of n products in fp32, whatever its order, is off by at most n 2^-24 of the sum of its magnitudes if every addition
is rounded to nearest; the matrix instructions round at most once a product and once a block, not always to nearest, so
2^-23 is taken. `half`: half a step of the inputs' type (0 for float32 itself: the fp32 terms cover it), by which the
weights are rounded before a product with 16-bit rows, and every result when it is written.
"""
import math

import torch

HALF = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
U = 2.0 ** -23
# binary16 below 2^-14 has a fixed step of 2^-24: rounding is off by up to half of it, whatever the value (bfloat16 and float32
# have such steps below 2^-126, far below the other terms)
TINY = {torch.float32: 0.0, torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}


def labels(x, w, t, b=None, g=None, ignore=-100):
    """x (N,D), w (V,D), t (N), b (V), g (N): per-ray upstream gradient. Returns {name: (value, bound)} for loss, dx, dw, db."""
    half, tiny, N, D, V = HALF[x.dtype], TINY[x.dtype], x.size(0), x.size(1), w.size(0)
    x, w = x.double(), w.double()
    off_label = torch.zeros(V, dtype=torch.bool, device=x.device) if b is None else torch.isinf(b)
    bias = torch.zeros(V, dtype=torch.float64, device=x.device) if b is None else b.double()
    use = t != ignore
    x = torch.where(use[:, None], x, torch.zeros_like(x))
    at = torch.where(use, t, torch.zeros_like(t))
    s = x @ w.T + bias
    lse = torch.logsumexp(s, 1)
    loss = torch.where(use, lse - s.gather(1, at[:, None])[:, 0], 0.0)
    finite = torch.where(off_label, 0.0, s.abs())
    size = (x.abs() @ w.abs().T + torch.where(off_label, 0.0, bias.abs())).amax(1)
    wrong = (D + 4) * U * size                                                  # of a logit
    rel = 2 * wrong + 2 * U * (finite.amax(1) + lse.abs() + 1) + (V / 32 + 16) * U   # of a weight, and of lse
    out = {"loss": (loss, torch.where(use, 2 * rel, 0.0) + U * loss.abs())}
    if g is None:
        return out
    g = torch.where(use, g.double(), 0.0)[:, None]
    p = (s - lse[:, None]).exp()
    hot = torch.zeros_like(p).scatter_(1, at[:, None], 1.0)
    ds = g * (p - hot)
    e32 = g.abs() * (p * rel[:, None] + U)
    e = e32 + half * ds.abs()
    dx, dw, db = ds @ w, ds.T @ x, ds.sum(0)
    return dict(out,
                dx=(dx, e @ w.abs() + (V / 16 + 8) * U * (ds.abs() @ w.abs()) + (half + 2 * U) * dx.abs() + tiny),
                dw=(dw, e.T @ x.abs() + (N / 16 + 8) * U * (ds.abs().T @ x.abs()) + (half + 2 * U) * dw.abs() + tiny),
                db=(db, e32.sum(0) + (N + 8) * U * ds.abs().sum(0)))


def attend(q, k, v, lengths=None, scale=None, up=None):
    """{name: (value, bound)} for out, dq, dk, dv; q (B,Lq,H,D), k, v (B,Lk,Hkv,.)."""
    half, tiny = HALF[q.dtype], TINY[q.dtype]
    B, Lq, H, D = q.shape
    Lk, Hkv, Dv = k.size(1), k.size(2), v.size(3)
    scale = D ** -0.5 if scale is None else scale
    z = lambda *n: torch.zeros(*n, dtype=torch.float64, device=q.device)  # noqa: E731
    res = {"out": (z(B, Lq, H, Dv), z(B, Lq, H, Dv)), "dq": (z(B, Lq, H, D), z(B, Lq, H, D)),
           "dk": (z(B, Lk, Hkv, D), z(B, Lk, Hkv, D)), "dv": (z(B, Lk, Hkv, Dv), z(B, Lk, Hkv, Dv))}
    for i in range(B):
        n = Lk if lengths is None else max(0, min(Lk, int(lengths[i])))
        if n == 0:
            continue
        for h in range(H):
            kv = h // (H // Hkv)
            Q, K, V = q[i, :, h].double(), k[i, :n, kv].double(), v[i, :n, kv].double()
            s = scale * (Q @ K.T)
            lse = torch.logsumexp(s, 1)
            wrong = (D + 4) * U * abs(scale) * (Q.abs() @ K.abs().T).amax(1)
            rel = (2 * wrong + 2 * U * (s.abs().amax(1) + lse.abs() + 1) + (n / 32 + 16) * U)[:, None]
            p = (s - lse[:, None]).exp()
            o = p @ V
            ep = p * (rel + half)
            eo = (ep + tiny) @ V.abs() + (n / 16 + 8) * U * (p @ V.abs()) + (half + 2 * U + rel) * o.abs() + tiny   # (weights and results)
            res["out"][0][i, :, h], res["out"][1][i, :, h] = o, eo
            if up is None:
                continue
            dO = up[i, :, h].double()
            dp, delta = dO @ V.T, (dO * o).sum(1, keepdim=True)
            edp = (Dv + 4) * U * (dO.abs() @ V.abs().T) + (Dv + 4) * U * (dO * o).abs().sum(1, keepdim=True) \
                + (dO.abs() * eo).sum(1, keepdim=True)
            ds = scale * p * (dp - delta)
            eds = abs(scale) * p * (rel * (dp - delta).abs() + edp) + (half + 4 * U) * ds.abs()
            dq, dk, dv = ds @ K, ds.T @ Q, p.T @ dO
            res["dq"][0][i, :, h] = dq
            res["dq"][1][i, :, h] = eds @ K.abs() + (n / 16 + 8) * U * (ds.abs() @ K.abs()) + (half + 2 * U) * dq.abs() + tiny
            rows = Lq * (H // Hkv) / 16 + 8
            res["dk"][0][i, :n, kv] += dk
            res["dk"][1][i, :n, kv] += eds.T @ Q.abs() + rows * U * (ds.abs().T @ Q.abs())
            res["dv"][0][i, :n, kv] += dv
            res["dv"][1][i, :n, kv] += ep.T @ dO.abs() + rows * U * (p.T @ dO.abs())
    for name in ("dk", "dv"):   # (what is written is the sum over the heads)
        res[name][1].add_((half + 2 * U) * res[name][0].abs() + tiny)
    return res


def check(got, ref, name):
    value, bound = ref
    assert got.shape == value.shape, (name, got.shape, value.shape)
    got = got.double()
    assert torch.isfinite(got).all(), name
    over = (got - value).abs() - bound
    worst = float(over.max()) if over.numel() else -math.inf
    assert worst <= 1e-30, "%s: %.3g beyond a bound of %.3g" % (name, worst, float(bound.reshape(-1)[over.argmax()]))
