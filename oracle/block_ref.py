"""Group norm and differential attention restated in float64 numpy (TEST INFRASTRUCTURE ONLY).

Values come with ``*_bound``s where a caller passes ``u``, half a step of the
type (``finfo.eps / 2``): how far a result may be off elementwise when the
softmax weights, the score gradients and the outputs are each rounded once to that type (relative error ``u``), plus ``SLOP``
relative to the absolute terms of every sum for the f32 arithmetic (products
of 64 or 128 terms: 128 * 2^-24 = 8e-6; exponentials 2^-21 and the f32 error of
their arguments, below 3e-5 for scores up to a few hundred).
"""
from __future__ import annotations

import numpy as np

SLOP = 1e-4


def _sigmoid(z):
    return 1.0 / (1.0 + np.exp(-z))


def group_norm(x, groups, weight, bias, eps, cu, silu):
    """Per sequence and group over rows x channels; ``x`` (N, C)."""
    x = np.asarray(x, np.float64)
    c = x.shape[1]
    y = np.zeros_like(x)
    for lo, hi in zip(cu[:-1], cu[1:]):
        if hi == lo:
            continue
        part = x[lo:hi].reshape(hi - lo, groups, c // groups)
        mean = part.mean((0, 2), keepdims=True)
        var = part.var((0, 2), keepdims=True)
        z = ((part - mean) / np.sqrt(var + eps)).reshape(hi - lo, c)
        z = z * (1.0 if weight is None else weight) + (0.0 if bias is None else bias)
        y[lo:hi] = z * _sigmoid(z) if silu else z
    return y


def group_norm_backward(x, dy, groups, weight, bias, eps, cu, silu):
    """(dx, dweight, dbias) of ``sum(dy * group_norm(x))``."""
    x, dy = np.asarray(x, np.float64), np.asarray(dy, np.float64)
    c = x.shape[1]
    w = np.ones(c) if weight is None else np.asarray(weight, np.float64)
    b = np.zeros(c) if bias is None else np.asarray(bias, np.float64)
    dx, dw, db = np.zeros_like(x), np.zeros(c), np.zeros(c)
    for lo, hi in zip(cu[:-1], cu[1:]):
        if hi == lo:
            continue
        n = hi - lo
        part = x[lo:hi].reshape(n, groups, c // groups)
        rstd = 1.0 / np.sqrt(part.var((0, 2), keepdims=True) + eps)
        xhat = (part - part.mean((0, 2), keepdims=True)) * rstd
        xf = xhat.reshape(n, c)
        dz = dy[lo:hi]
        if silu:
            z = xf * w + b
            s = _sigmoid(z)
            dz = dz * s * (1 + z * (1 - s))
        dw += (dz * xf).sum(0)
        db += dz.sum(0)
        t = (dz * w).reshape(part.shape)
        d = t - t.mean((0, 2), keepdims=True) - xhat * (t * xhat).mean((0, 2), keepdims=True)
        dx[lo:hi] = (d * rstd).reshape(n, c)
    return dx, dw, db


def diff_attention(q, k, v, lam, cu_q, cu_kv=None, scale=0.125, causal=False, dout=None, u=0.0):
    """Dict with ``out`` and, given ``dout``, ``dq``, ``dk``, ``dv``, ``dlam`` (one
    per head), each with its ``*_bound``.  ``q`` (N, 2H, 64), ``k`` (M, 2Hk,
    64), ``v`` (M, Hk, 128), ``lam`` (H,)."""
    q, k, v, lam = (np.asarray(t, np.float64) for t in (q, k, v, lam))
    cu_kv = cu_q if cu_kv is None else cu_kv
    heads, rep = q.shape[1] // 2, q.shape[1] // 2 // v.shape[1]
    out = np.zeros((q.shape[0], heads, v.shape[2]))
    res = {"out": out, "out_bound": np.zeros_like(out)}
    if dout is not None:
        dout = np.asarray(dout, np.float64)
        for n, t in (("dq", q), ("dk", k), ("dv", v), ("dlam", np.zeros(heads))):
            res[n], res[n + "_bound"] = np.zeros_like(t), np.zeros_like(t)
    for q0, q1, k0, k1 in zip(cu_q[:-1], cu_q[1:], cu_kv[:-1], cu_kv[1:]):
        lq, lk = q1 - q0, k1 - k0
        if lq == 0 or lk == 0:
            continue
        see = np.ones((lq, lk), bool)
        if causal:
            see = np.arange(lk)[None] <= np.arange(lq)[:, None] + lk - lq
        for h in range(heads):
            g = h // rep
            vv, p, o, ob = v[k0:k1, g], [], [], []
            for m in (0, 1):
                s = np.where(see, q[q0:q1, 2 * h + m] @ k[k0:k1, 2 * g + m].T * scale, -np.inf)
                top = s.max(1, keepdims=True)
                e = np.exp(s - np.where(np.isfinite(top), top, 0.0))
                total = e.sum(1, keepdims=True)
                p.append(e / np.where(total > 0, total, 1.0))
                o.append(p[m] @ vv)
                ob.append((u + SLOP) * (p[m] @ np.abs(vv)))
            lh, al = lam[h], abs(lam[h])
            oh = o[0] - lh * o[1]
            out[q0:q1, h] = oh
            ob_out = ob[0] + al * ob[1] + u * np.abs(oh)
            res["out_bound"][q0:q1, h] = ob_out
            if dout is None:
                continue
            do = dout[q0:q1, h]
            ado = np.abs(do)
            delta = [(do * t).sum(1, keepdims=True) for t in o]
            off = [(ado * t).sum(1, keepdims=True) for t in ob]  # the products are kept in f32
            dp, adp = do @ vv.T, ado @ np.abs(vv).T
            sign = (1.0, -lh)
            pd = p[0] - lh * p[1]
            dv, apd = pd.T @ do, np.abs(pd) * u + SLOP * (p[0] + al * p[1])
            res["dv"][k0:k1, g] += dv
            res["dv_bound"][k0:k1, g] += apd.T @ ado
            for m in (0, 1):
                ds = sign[m] * p[m] * (dp - delta[m]) * scale
                eds = u * np.abs(ds) + abs(sign[m]) * scale * p[m] * (
                    off[m] + SLOP * (adp + (ado * (p[m] @ np.abs(vv))).sum(1, keepdims=True)))
                qq, kk = q[q0:q1, 2 * h + m], k[k0:k1, 2 * g + m]
                res["dq"][q0:q1, 2 * h + m] = ds @ kk
                res["dq_bound"][q0:q1, 2 * h + m] = eds @ np.abs(kk)
                res["dk"][k0:k1, 2 * g + m] += ds.T @ qq
                res["dk_bound"][k0:k1, 2 * g + m] += eds.T @ np.abs(qq)
            res["dlam"][h] -= delta[1].sum()
            res["dlam_bound"][h] += off[1].sum()
    if dout is not None:
        for n in ("dq", "dk", "dv", "dlam"):
            res[n + "_bound"] += u * np.abs(res[n])
    return res
