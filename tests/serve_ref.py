"""Plain 64-bit forms of llapis_step.h's operators before and after a step's attention
(pages and slots, query and key norms with positions, sampling), and bounds on how far
the library's results may be from them."""
import math

import torch

from step_ref import DT, EPS


def extend(table, lens, n_new, free, n_free, n_tokens, page_size, n_pages):
    """(table, lens, n_free, new_start, pos, seq, slots), in the order of the rules"""
    table, lens = [list(r) for r in table], [max(n, 0) for n in lens]
    n_free = min(max(n_free, 0), n_pages)
    width = len(table[0]) if table else 0
    asked = need = taken = 0
    start, pos, seq, slots = [0], [], [], []
    for s, n in enumerate(lens):
        want = max(n_new[s], 0)
        if n + want > width * page_size:
            want = 0
        asked += want
        if asked > n_tokens:
            want = 0
        pages = -(-(n + want) // page_size) - -(-n // page_size)
        need += pages
        if pages and need > n_free:
            want = pages = 0
        for i in range(pages):
            table[s][-(-n // page_size) + i] = free[n_free - 1 - taken]
            taken += 1
        lens[s] = n + want
        start.append(start[-1] + want)
        for t in range(n, n + want):
            pg = table[s][t // page_size]
            pos.append(t)
            seq.append(s)
            slots.append(pg * page_size + t % page_size if 0 <= pg < n_pages else -1)
    rest = [-1] * (n_tokens - len(pos))
    return table, lens, n_free - taken, start, pos + rest, seq + rest, slots + rest


def rope(x, pos, freq, weight, norm, eps, magnitude, layout_half, tag):
    """(y, tol) for heads x [T, n, D] (host): fp64 results and the bound on their error.

    The norm's sum of D squares in fp32, at most 16 of them in a lane in order and 6 more sums
    over lanes, is off by 24 2^-24 of itself, its root by half of that; with the quotient, the
    root's and the products' roundings a normed value is off by 18 2^-24 of itself.  Cosine and
    sine: the angle is exact but for 2^-51 of itself and for what its fp32 remainder of a quarter turn is
    rounded by, 2^-25; the function adds 2 2^-24, the factor and its product 2^-23.  A turned value is the sum of two
    products: three roundings more.  All of it on |a| + |b|, then its own rounding."""
    T, n, D = x.shape
    y = x.double()
    if norm:
        y = y / (y.square().mean(-1, keepdim=True) + eps).sqrt() * (1 if weight is None else weight.double())
    mag = y.abs()
    err = (18 * 2 ** -24 if norm else 0) * mag
    if freq is not None and len(freq):
        rot = 2 * len(freq)
        angle = pos.double()[:, None] * freq
        cos, sin = (magnitude * angle.cos())[:, None], (magnitude * angle.sin())[:, None]
        a, b = (slice(0, rot // 2), slice(rot // 2, rot)) if layout_half else (slice(0, rot, 2), slice(1, rot, 2))
        u, v = y[..., a].clone(), y[..., b].clone()
        both = (mag[..., a] + mag[..., b]) * abs(magnitude)
        off = both * ((18 + 9) * 2 ** -24 + angle.abs()[:, None] * 2 ** -51)
        y[..., a], y[..., b] = u * cos - v * sin, v * cos + u * sin
        err = err.clone()
        err[..., a], err[..., b] = off, off
    return y, err + EPS[tag] * (y.abs() + err)


def kept(x, t, k, p, m):
    """The probabilities of one row of logits after the filters, in Python's floats' precision:
    weights of a float64 tensor [V], 0 where a value is not kept; None where there is no value"""
    x = torch.where(torch.isnan(x.double()), -math.inf, x.double()) + 0.0
    V = len(x)
    top = float(x.max())
    if top == -math.inf:
        return None
    z, order = torch.sort(x, descending=True, stable=True)
    if not t > 0 or k == 1 or p <= 0 or m > 1:
        w = torch.zeros(V, dtype=torch.float64)
        w[order[0]] = 1
        return w
    w = torch.where(z == top, 1.0, torch.zeros((), dtype=torch.float64) if top == math.inf else ((z - top) / t).exp())
    w = torch.where(z == -math.inf, 0.0, w)
    if k > 0:
        w[k:] = 0
    if p < 1:
        upto = w.cumsum(0)
        w = torch.where(upto - w < p * upto[-1], w, 0.0)
    if m > 0:
        w = torch.where(w >= m, w, 0.0)
    return torch.zeros(V, dtype=torch.float64).scatter_(0, order, w)


def sample(logits, u, temperature, top_k, top_p, min_p):
    """(tokens, probabilities [S, V] in fp64)"""
    S, V = logits.shape
    tokens, probs = [], torch.zeros(S, V, dtype=torch.float64)
    get = lambda v, i, off: off if v is None else float(v[i])
    for i in range(S):
        w = kept(logits[i], get(temperature, i, 1.0), int(get(top_k, i, 0)), get(top_p, i, 1.0), get(min_p, i, 0.0))
        if w is None:
            tokens.append(-1)
            continue
        cum = w.cumsum(0)
        over = ((w > 0) & (cum > float(u[i]) * cum[-1])).nonzero()
        tokens.append(int(over[0]) if len(over) else int(w.nonzero()[-1]))
        probs[i] = w / cum[-1]
    return tokens, probs
