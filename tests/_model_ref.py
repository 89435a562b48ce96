"""
The operators of whole language models in 64 bits, from their definitions: plain numpy, no code of the package.
"""

from __future__ import annotations

import numpy


def _lens(lens, T, B):
    return numpy.full((B,), T) if lens is None else numpy.clip(numpy.asarray(lens), 0, T)


def delta(q, k, v, g, b, s0=None, lens=None, direction=1, scale=None):
    """
    :param q, k: [T,B,key_heads,dk]
    :param v: [T,B,heads,dv]
    :param g, b: [T,B,heads]
    :return: y [T,B,heads,dv], s [B,heads,dk,dv], and of every frame what the gradient needs
    """
    q, k, v, g, b = (numpy.asarray(x, numpy.float64) for x in (q, k, v, g, b))
    T, B, H, dv = v.shape
    Hk, dk = q.shape[2:]
    share = numpy.arange(H) // (H // Hk)
    scale = 1.0 / numpy.sqrt(dk) if scale is None else scale
    s = numpy.zeros((B, H, dk, dv)) if s0 is None else numpy.array(s0, numpy.float64)
    lens = _lens(lens, T, B)
    y, trace = numpy.zeros((T, B, H, dv)), []
    for t in range(T) if direction > 0 else range(T - 1, -1, -1):
        inside = (t < lens)[:, None]
        qt, kt, vt = (numpy.where(inside[..., None], x, 0.0) for x in (q[t][:, share], k[t][:, share], v[t]))  # (whatever lies past a sequence's end)
        a, bt = numpy.where(inside, numpy.exp(g[t]), 1.0), numpy.where(inside, b[t], 0.0)
        kept = a[..., None, None] * s
        missing = vt - numpy.einsum("bhij,bhi->bhj", kept, kt)
        after = kept + kt[..., :, None] * (bt[..., None] * missing)[..., None, :]
        y[t] = numpy.where(inside[..., None], scale * numpy.einsum("bhij,bhi->bhj", after, qt), 0.0)
        trace.append((t, inside, qt, kt, a, bt, s, kept, missing, after))
        s = after
    return y, s, trace


def delta_grad(q, k, v, g, b, dy, ds, s0=None, lens=None, direction=1, scale=None):
    """:return: dq, dk, dv, dg, db, ds0"""
    Hk, dk = numpy.shape(q)[2:]
    T, B, H, dv = numpy.shape(v)
    scale = 1.0 / numpy.sqrt(dk) if scale is None else scale
    trace = delta(q, k, v, g, b, s0, lens, direction, scale)[2]
    dq, dkey, dval, dg, db = numpy.zeros((T, B, Hk, dk)), numpy.zeros((T, B, Hk, dk)), numpy.zeros((T, B, H, dv)), numpy.zeros((T, B, H)), numpy.zeros((T, B, H))
    d = numpy.array(ds, numpy.float64)
    for t, inside, qt, kt, a, bt, s, kept, missing, after in reversed(trace):
        e = scale * numpy.where(inside[..., None], numpy.asarray(dy[t], numpy.float64), 0.0)
        into = d + qt[..., :, None] * e[..., None, :]
        du = numpy.einsum("bhij,bhi->bhj", into, kt)
        dm = bt[..., None] * du
        of_kept = into - kt[..., :, None] * dm[..., None, :]
        of_k = numpy.einsum("bhij,bhj->bhi", into, bt[..., None] * missing) - numpy.einsum("bhij,bhj->bhi", kept, dm)
        of_q = numpy.einsum("bhij,bhj->bhi", after, e)
        dq[t] = numpy.where(inside[..., None], of_q, 0.0).reshape(B, Hk, H // Hk, dk).sum(axis=2)
        dkey[t] = numpy.where(inside[..., None], of_k, 0.0).reshape(B, Hk, H // Hk, dk).sum(axis=2)
        dval[t] = numpy.where(inside[..., None], dm, 0.0)
        db[t] = numpy.where(inside, (du * missing).sum(axis=-1), 0.0)
        dg[t] = numpy.where(inside, (of_kept * kept).sum(axis=(-1, -2)), 0.0)
        d = a[..., None, None] * of_kept
    return dq, dkey, dval, dg, db, d


def embed(tokens, weight, scale=1.0):
    tokens, weight = numpy.asarray(tokens), numpy.asarray(weight, numpy.float64)
    V = weight.shape[0]
    y = scale * weight[numpy.clip(tokens, 0, V - 1)]
    return numpy.where((tokens < 0)[..., None], 0.0, numpy.where((tokens >= V)[..., None], numpy.nan, y))


def embed_grad(tokens, dy, V, scale=1.0):
    """:return: dW [V,D], sums of absolute values [V,D], how many there are of each token"""
    flat, dy = numpy.asarray(tokens).reshape(-1), numpy.asarray(dy, numpy.float64)
    dy = dy.reshape(flat.size, dy.shape[-1])
    inside = (flat >= 0) & (flat < V)
    out, most = numpy.zeros((2, V, dy.shape[1]))
    numpy.add.at(out, flat[inside], scale * dy[inside])
    numpy.add.at(most, flat[inside], abs(scale * dy[inside]))
    return out, most, numpy.bincount(flat[inside], minlength=V)


def beam(scores, totals, beam, ended=None, end_token=None):
    """
    :param scores: [B,K,V] float32 values
    :return: totals [B,beam] float32, sources, tokens: by their definition, one addition in float32
    """
    scores, totals = numpy.array(scores, numpy.float32), numpy.asarray(totals, numpy.float32)
    B, K, V = scores.shape
    if ended is not None:
        scores[numpy.asarray(ended)] = -numpy.inf
        scores[numpy.asarray(ended), end_token] = 0.0
    with numpy.errstate(invalid="ignore"):
        joint = (totals[..., None] + scores).reshape(B, K * V)
    # a NaN before everything, then in descending order; what is equal in the order of its index
    at = numpy.stack([numpy.lexsort((numpy.arange(K * V), -numpy.where(numpy.isnan(j), 0.0, j), ~numpy.isnan(j)))[:beam] for j in joint])
    return numpy.take_along_axis(joint, at, 1), at // V, at % V
