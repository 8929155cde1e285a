"""CPU restatement of the layer operators in float64, and how far a kernel's result may be from it.

``u`` below is half a step of the tensors' type, ``U`` half a step of float32: a rounding is off by at most that much
relative to the value.  Bounds follow the kernels' roundings one by one and take no account of their signs."""
from __future__ import annotations

import numpy as np

U = 2.0 ** -24
HALF_STEP = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11, "f32": 2.0 ** -24}
TINY = {"bf16": 2.0 ** -126, "f16": 2.0 ** -24, "f32": 2.0 ** -126}     # a step of the subnormals, or what is flushed


def default_positions(q_lens, k_lens):
    return np.concatenate([np.arange(a) + b - a for a, b in zip(q_lens, k_lens)] or [np.zeros(0)]).astype(np.int64)


def attention(q, k, v, q_lens, k_lens, window=(-1, -1), sinks=0, positions=None, scale=None, table=None, buckets=None,
              dout=None, kernel_out=None, dtype="f32"):
    """Every output with its bound: ``{"out": (value, bound), "lse": ..., "dq": ...}``.  Hidden pairs are left out of every
    sum, whatever they hold.  ``kernel_out``: the rounded output the backward kernels were given (for their bound)."""
    q, k, v = (np.asarray(x, np.float64) for x in (q, k, v))
    h, hk, d = q.shape[1], k.shape[1], q.shape[2]
    g = h // hk
    scale = d ** -0.5 if scale is None else scale
    pos = default_positions(q_lens, k_lens) if positions is None else np.asarray(positions, np.int64)
    u, tiny = HALF_STEP[dtype], TINY[dtype]
    uw = 0.0 if dtype == "f32" else u                 # rounding of P and dS for the second products
    nq, nk = int(sum(q_lens)), int(sum(k_lens))
    r = {"out": np.zeros((nq, h, d)), "lse": np.full((h, nq), -np.inf)}
    e = {"out": np.zeros((nq, h, d)), "lse": np.zeros((h, nq))}
    if dout is not None:
        dout = np.asarray(dout, np.float64)
        for n, like in (("dq", q[:nq]), ("dk", k[:nk]), ("dv", v[:nk])):
            r[n], e[n] = np.zeros_like(like), np.zeros_like(like)
        if table is not None:
            r["dtable"], e["dtable"] = np.zeros(table.shape), np.zeros(table.shape)
    q0 = k0 = 0
    for a, b in zip(q_lens, k_lens):
        if a and b:
            p_i = pos[q0:q0 + a][:, None]
            j = np.arange(b)[None]
            see = np.ones((a, b), bool)
            if window[1] >= 0:
                see &= j <= p_i + window[1]
            if window[0] >= 0:
                see &= (j >= p_i - window[0]) | (j < sinks)
            if table is not None:
                reach = len(buckets) // 2
                of = np.asarray(buckets)[np.clip(j - p_i, -reach, reach) + reach]
            for n in range(h):
                Q, K, V = q[q0:q0 + a, n], k[k0:k0 + b, n // g], v[k0:k0 + b, n // g]
                bias = np.asarray(table, np.float64)[of, n] if table is not None else np.zeros((a, b))
                ok = see & (bias > -2.0 ** 100)
                Kc, Vc = np.where(ok.any(0)[:, None], K, 0), np.where(ok.any(0)[:, None], V, 0)
                with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
                    s = np.where(ok, scale * (Q @ Kc.T) + np.where(ok, bias, 0), -np.inf)
                    top = s.max(1, keepdims=True)
                    top = np.where(np.isfinite(top), top, 0)
                    w = np.where(ok, np.exp(s - top), 0)
                    z = w.sum(1, keepdims=True)
                    P = w / np.where(z > 0, z, 1)
                    lse = np.log(z) + top
                    out = P @ Vc
                    # scores: D products summed in any order, the scale, the bias, their sums and the change to log2
                    es = (d + 8) * U * (scale * np.abs(Q) @ np.abs(Kc).T + np.abs(np.where(ok, bias, 0))) + 4 * U * np.abs(top)
                    es = np.where(ok, es, 0).max(1, keepdims=True)
                    ep = 2 * es + (b + 16) * U            # of a weight: its own score and the row's sum, exp2, divide
                    eo = u * np.abs(out) + (uw + ep) * (P @ np.abs(Vc)) * (1 + u) + tiny * (1 + np.abs(Vc).sum(0) * 2.0 ** -10)
                    some = (z[:, 0] > 0)
                    r["out"][q0:q0 + a, n], e["out"][q0:q0 + a, n] = out, eo
                    r["lse"][n, q0:q0 + a] = np.where(some, lse[:, 0], -np.inf)
                    e["lse"][n, q0:q0 + a] = np.where(some, es[:, 0] + (b + 8) * U + 4 * U * np.abs(lse[:, 0]), 0)
                    if dout is None:
                        continue
                    G = dout[q0:q0 + a, n]
                    dP = np.where(ok, G @ Vc.T, 0)
                    delta = (G * out).sum(1, keepdims=True)
                    dS = P * (dP - delta)
                    eout = np.abs(np.asarray(kernel_out, np.float64)[q0:q0 + a, n] - out) if kernel_out is not None else eo
                    # the weight from the stored lse: its error joins the score's, and the score's sum starts from it
                    epb = ep + 2 * e["lse"][n, q0:q0 + a][:, None] + 2 * (d + 8) * U * np.where(some, np.abs(lse[:, 0]), 0)[:, None]
                    eds = P * (epb * np.abs(dP - delta) + (d + 4) * U * (np.abs(G) @ np.abs(Vc).T) +
                               (np.abs(G) * eout).sum(1, keepdims=True) + (d + 4) * U * (np.abs(G) * np.abs(out)).sum(1, keepdims=True))
                    eds = np.where(ok, eds, 0)
                    eds2 = eds + uw * (np.abs(dS) + eds) + np.where(ok, tiny, 0)
                    Qc = np.where(ok.any(1)[:, None], Q, 0)
                    Gc = np.where(ok.any(1)[:, None], G, 0)
                    r["dq"][q0:q0 + a, n] = scale * dS @ Kc
                    e["dq"][q0:q0 + a, n] = scale * (eds2 + (b + 4) * U * np.abs(dS)) @ np.abs(Kc)
                    r["dk"][k0:k0 + b, n // g] += scale * dS.T @ Qc
                    e["dk"][k0:k0 + b, n // g] += scale * (eds2 + (a * g + 4) * U * np.abs(dS)).T @ np.abs(Qc)
                    r["dv"][k0:k0 + b, n // g] += P.T @ Gc
                    e["dv"][k0:k0 + b, n // g] += (P * (uw + epb + (a * g + 4) * U) + np.where(ok, tiny, 0)).T @ np.abs(Gc)
                    if table is not None:
                        np.add.at(r["dtable"][:, n], of, dS)
                        np.add.at(e["dtable"][:, n], of, eds + (a + b + 64) * U * np.abs(dS))
        q0, k0 = q0 + a, k0 + b
    for n in ("dq", "dk", "dv", "dtable"):
        if n in r:
            e[n] += u * np.abs(r[n]) * (1 + u) + tiny
    return {n: (r[n], e[n]) for n in r}


def _turn(x, cos, sin, interleaved, direction):
    if interleaved:
        a, b = x[..., 0::2], x[..., 1::2]
    else:
        a, b = np.split(x, 2, -1)
    y = np.stack([a * cos - direction * b * sin, b * cos + direction * a * sin], -1)
    return y.reshape(x.shape) if interleaved else np.concatenate([y[..., 0], y[..., 1]], -1)


def qk_norm_rope(x, gain, cos, sin, positions, eps=1e-6, interleaved=False, dy=None, dtype="f32"):
    """One of the two tensors: ``y``, and with ``dy`` also ``dx`` and ``dgain``, each with its bound."""
    x = np.asarray(x, np.float64)
    d = x.shape[-1]
    u, tiny = HALF_STEP[dtype], TINY[dtype]
    c, s = (np.asarray(t, np.float64)[positions][:, None] for t in (cos, sin))
    g = np.ones(d) if gain is None else np.asarray(gain, np.float64)
    r = np.ones(x.shape[:-1] + (1,)) if gain is None else 1 / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    y = _turn(x * r * g, c, s, interleaved, 1)
    # both members of a pair enter an output element: d products of the norm, root, divide, two products, the rotation
    size = _turn(np.abs(x * r * g), np.abs(c), -np.abs(s), interleaved, 1)
    size = np.maximum(size, _turn(np.abs(x * r * g), np.abs(c), np.abs(s), interleaved, 1))
    found = {"y": (y, u * np.abs(y) * (1 + u) + (d + 12) * U * size + tiny)}
    if dy is None:
        return found
    dz = _turn(np.asarray(dy, np.float64), c, s, interleaved, -1)
    az = np.maximum(_turn(np.abs(np.asarray(dy, np.float64)), np.abs(c), -np.abs(s), interleaved, 1),
                    _turn(np.abs(np.asarray(dy, np.float64)), np.abs(c), np.abs(s), interleaved, 1))
    if gain is None:
        found["dx"] = (dz, u * np.abs(dz) * (1 + u) + 4 * U * az + tiny)
        return found
    m = (dz * g * x).mean(-1, keepdims=True)
    dx = r * (dz * g - x * r * r * m)
    adx = r * (az * np.abs(g) + np.abs(x) * r * r * (az * np.abs(g * x)).mean(-1, keepdims=True))
    found["dx"] = (dx, u * np.abs(dx) * (1 + u) + (3 * d + 24) * U * adx + tiny)
    n = x.shape[0] * x.shape[1]
    found["dgain"] = ((dz * x * r).sum((0, 1)), ((d + n / 64 + 300) * U * (az * np.abs(x) * r).sum((0, 1))))
    return found
