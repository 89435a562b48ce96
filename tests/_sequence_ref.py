"""
The sequence operators in 64 bits, from their definitions: plain numpy, no code of the package.
"""

from __future__ import annotations

import numpy


def sigmoid(x):
    with numpy.errstate(over="ignore"):
        return 1.0 / (1.0 + numpy.exp(-x))


def recurrence(x, c0=None, lens=None, direction=1):
    """
    :param x: [T,B,4n]
    :return: y [T,B,n], c [B,n], and what the gradient and the error bounds need
    """
    x = numpy.asarray(x, numpy.float64)
    T, B, n4 = x.shape
    n = n4 // 4
    c = numpy.zeros((B, n)) if c0 is None else numpy.array(c0, numpy.float64)
    lens = numpy.full((B,), T) if lens is None else numpy.clip(numpy.asarray(lens), 0, T)
    frames = list(range(T)) if direction > 0 else list(range(T - 1, -1, -1))
    y = numpy.zeros((T, B, n))
    trace = []
    summed, most = numpy.zeros((B, n)), numpy.ones((B, n))
    for t in frames:
        inside = (t < lens)[:, None]
        gates = numpy.where(inside, x[t], 0.0)  # (whatever lies past a sequence's end)
        z, i, f, o = gates.reshape(B, 4, n).transpose(1, 0, 2)
        z, i, f, o = numpy.tanh(z), sigmoid(i), sigmoid(f), sigmoid(o)
        before = c
        c = numpy.where(inside, f * c + i * z, c)
        y[t] = numpy.where(inside, o * c, 0.0)
        summed = numpy.where(inside, f * summed + 1.0, summed)
        most = numpy.maximum(most, summed)
        trace.append((t, inside, z, i, f, o, before, c))
    return y, c, dict(trace=trace, most=most.max(initial=1.0), largest=max([1.0] + [numpy.abs(v[7]).max(initial=0.0) for v in trace] + [numpy.abs(c).max(initial=0.0)]))


def recurrence_grad(x, dy, dc, c0=None, lens=None, direction=1):
    """:return: dx [T,B,4n], dc0 [B,n], the largest error of a state, the longest sum of errors"""
    T, B, n4 = numpy.shape(x)
    _, _, info = recurrence(x, c0, lens, direction)
    dx = numpy.zeros((T, B, 4, n4 // 4))
    g = numpy.array(dc, numpy.float64)
    largest, summed, most = numpy.abs(g).max(initial=0.0), numpy.ones_like(g), 1.0
    for t, inside, z, i, f, o, before, after in reversed(info["trace"]):
        e = numpy.where(inside, numpy.asarray(dy[t], numpy.float64), 0.0)
        total = g + e * o
        parts = (total * i * (1 - z * z), total * z * i * (1 - i), total * before * f * (1 - f), e * after * o * (1 - o))
        dx[t] = numpy.where(inside[:, None, :], numpy.stack(parts, axis=1), 0.0)
        g = numpy.where(inside, total * f, g)
        largest = max(largest, numpy.abs(total).max(initial=0.0))
        summed = numpy.where(inside, f * summed + 1.0, summed)
        most = max(most, summed.max(initial=1.0))
    return dx.reshape(T, B, n4), g, largest, most


def philox(counter, key):
    """Philox4x32-10: four words from four words of counter and two of key."""
    c, k = [int(v) for v in counter], [int(v) for v in key]
    for _ in range(10):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [(b >> 32) ^ c[1] ^ k[0], b & 0xFFFFFFFF, (a >> 32) ^ c[3] ^ k[1], a & 0xFFFFFFFF]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return c


def draws(first, count, seed, offset):
    """The 16-bit draws of the elements first .. first+count-1."""
    out = []
    for g in range(first // 8, (first + count + 7) // 8):
        words = philox((g & 0xFFFFFFFF, g >> 32, offset & 0xFFFFFFFF, offset >> 32), (seed & 0xFFFFFFFF, seed >> 32))
        out += [w >> s & 0xFFFF for w in words for s in (0, 16)]
    skip = first % 8
    return numpy.array(out[skip : skip + count], numpy.int64)


def keep_factors(shape, drop_prob, seed, offset, same_over_time=False):
    """What dropout multiplies the elements of an array of this shape with."""
    of = shape[1:] if same_over_time else shape
    count = int(numpy.prod(of, dtype=numpy.int64))
    threshold = int(round(drop_prob * 65536))
    factor = 65536.0 / (65536 - threshold) if threshold < 65536 else 0.0
    keep = (draws(0, count, seed, offset) >= threshold) * factor
    return numpy.broadcast_to(keep.reshape(of), shape)


def scores(logits, targets=None, top_k=0):
    """
    :param logits: [R,V]
    :return: log_prob [R] or None, entropy [R], top_log_prob [R,k], top_ids [R,k], log p [R,V]
    """
    x = numpy.asarray(logits, numpy.float64)
    R, V = x.shape
    log_prob, entropy = numpy.zeros(R), numpy.zeros(R)
    top, ids, log_p = numpy.full((R, top_k), -numpy.inf), numpy.full((R, top_k), -1, numpy.int64), numpy.zeros((R, V))
    for r in range(R):
        if targets is not None and targets[r] < 0:
            continue
        m = x[r].max()
        if m == -numpy.inf:
            log_p[r] = -numpy.inf
        else:
            with numpy.errstate(invalid="ignore"):  # (the difference first: next to 1e38 a logarithm is nothing)
                d = x[r] - m
                log_p[r] = d - numpy.log(numpy.exp(d).sum())
        with numpy.errstate(invalid="ignore"):
            p = numpy.exp(log_p[r])
            entropy[r] = -numpy.where(p == 0, 0.0, p * log_p[r]).sum()
        if targets is not None:
            log_prob[r] = log_p[r, targets[r]] if targets[r] < V else numpy.nan
        # descending, a NaN first, among equal ones the lower index first
        order = numpy.lexsort((numpy.arange(V), -numpy.nan_to_num(x[r], nan=0.0, posinf=numpy.inf, neginf=-numpy.inf), ~numpy.isnan(x[r])))
        ids[r] = order[:top_k]
        top[r] = log_p[r, order[:top_k]]
    return (None if targets is None else log_prob), entropy, top, ids, log_p


def scores_grad(logits, targets, d_log_prob, d_entropy):
    """:return: [R,V]"""
    _, entropy, _, _, log_p = scores(logits, targets)
    R, V = log_p.shape
    out = numpy.zeros((R, V))
    for r in range(R):
        if (targets is not None and targets[r] < 0) or log_p[r].max() == -numpy.inf:
            continue
        if targets is not None and targets[r] >= V:
            out[r] = numpy.nan
            continue
        p = numpy.exp(log_p[r])
        out[r] = -p * d_entropy[r] * (numpy.where(p == 0, 0.0, log_p[r]) + entropy[r])
        if targets is not None:
            out[r] -= p * d_log_prob[r]
            out[r, targets[r]] += d_log_prob[r]
    return out
