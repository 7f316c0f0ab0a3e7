"""Plain 64-bit forms of the operators of llapis_step.h, sequence by sequence,
and bounds on how far the library's results may be from them."""
import math

import torch

import llapis_amd as la

DT = {la.F32: torch.float32, la.F16: torch.float16, la.BF16: torch.bfloat16}
EPS = {t: torch.finfo(d).eps / 2 for t, d in DT.items()}     # a rounding: half a step


def pack_cache(tag, kv):
    """What a cache of `tag` holds for values kv [..., head_dim]: the values
    after the rounding, in fp64, and for Q8_0 (int8, fp16 scales)."""
    if tag != la.Q8_0:
        return kv.to(DT[tag])
    x = kv.float().reshape(*kv.shape[:-1], -1, 32)
    amax = x.abs().amax(-1, keepdim=True)
    d = amax / 127
    inv = torch.where(d > 0, 1 / d, torch.zeros_like(d))
    return (x * inv).round().to(torch.int8).reshape(kv.shape), d.squeeze(-1).half()


def unpack(cache, page, is_v):
    """One page's values [n_kv, page_size, head_dim] in fp64 (host)."""
    H, P, D = cache.n_kv, cache.page_size, cache.head_dim
    raw = (cache.v if is_v else cache.k)[page].cpu()
    if cache.type != la.Q8_0:
        return raw.double().transpose(1, 2) if is_v else raw.double()
    raw = raw.view(torch.uint8).reshape(H, -1)
    q = raw[:, :P * D].contiguous().view(torch.int8).double()
    d = raw[:, P * D:].contiguous().view(torch.float16).double().reshape(H, D // 32, P)
    q = q.reshape(H, D, P).transpose(1, 2) if is_v else q.reshape(H, P, D)
    return q * d.transpose(1, 2).repeat_interleave(32, 2)


def sequence(cache, row, n):
    """(k, v [n_kv, n, head_dim], there [n]) of a sequence's keys, fp64; keys without a page are zeros."""
    P = cache.page_size
    ks, vs, there = [], [], []
    for i in range(-(-n // P)):
        pg = int(row[i])
        ok = 0 <= pg < cache.n_pages
        one = (unpack(cache, pg, False), unpack(cache, pg, True)) if ok else (torch.zeros(cache.n_kv, P, cache.head_dim, dtype=torch.float64),) * 2
        ks.append(one[0])
        vs.append(one[1])
        there += [ok] * P
    if not ks:
        z = torch.zeros(cache.n_kv, 0, cache.head_dim, dtype=torch.float64)
        return z, z, torch.zeros(0, dtype=torch.bool)
    return torch.cat(ks, 1)[:, :n], torch.cat(vs, 1)[:, :n], torch.tensor(there)[:n]


def attention(cache, table, lens, start, q, scale, window=0):
    """(out, lse, tol): fp64 results for q [T, n_head, D] (host) and the bound on out's error.

    The bound, for a row over n keys with scores s and results of type t: a
    score is an fp32 sum of D products of 16-bit parts, the query's parts equal
    to it up to 2^-22 (fp16, bf16 caches with fp32 queries: 2^-24): |ds| <=
    (D + 8) 2^-24 scale sum |q k| + 2^-22 scale sum |q k|, and its scaling to
    base 2 and the subtraction of the maximum add 2^-22 (|s| + |m|) at most.  A
    weight's relative error is |ds| of its key and of the maximum's key's row
    alike, plus 2^-21 of exp2, plus 2^-17 where 16-bit results let P be two bf16
    parts (fp16: 2^-22); the weighted sum of n weights in fp32, 32 keys a
    product and the products in order, adds (n / 32 + 40) 2^-24.  Both the
    numerator and the sum carry them, so the result is off by twice that times
    the largest |v|, and by its own rounding."""
    T, n_head, D = q.shape
    tag = {v: k for k, v in DT.items()}[q.dtype]
    out = torch.full((T, n_head, D), float("nan"), dtype=torch.float64)
    lse = torch.full((T, n_head), float("nan"), dtype=torch.float64)
    tol = torch.zeros(T, n_head, D, dtype=torch.float64)
    G = n_head // cache.n_kv
    for s, n in enumerate(lens):
        rows = range(start[s], start[s + 1])
        if not len(rows):
            continue
        k, v, there = sequence(cache, table[s], max(min(n, len(table[s]) * cache.page_size), 0))
        at = torch.arange(k.shape[1])
        for j, r in enumerate(rows):
            t = n - len(rows) + j
            see = there & (at <= t)
            if window:
                see &= at > t - window
            for a in range(n_head):
                kk, vv = k[a // G][see], v[a // G][see]
                if not len(kk):
                    out[r, a], lse[r, a] = 0, -math.inf
                    continue
                x = q[r, a].double()
                z = scale * (kk @ x)
                m = z.max()
                w = (z - m).exp()
                out[r, a], lse[r, a] = (w @ vv) / w.sum(), m + w.sum().log()
                mag = abs(scale) * (kk.abs() @ x.abs()).max()
                ds = ((D + 8) * 2 ** -24 + 2 ** -22) * mag + 2 ** -22 * 2 * z.abs().max()
                p_err = 2 ** -17 if tag != la.F32 and cache.type != la.F16 else 2 ** -21
                rel = 2 * ds + 2 ** -21 + p_err + (len(kk) / 32 + 40) * 2 ** -24
                tol[r, a] = 2 * rel * vv.abs().max() + EPS[tag] * (out[r, a].abs() + 2 * rel * vv.abs().max())
    return out, lse, tol


def fork(table, lens, forks, page_size, n_pages):
    """(table, lens, copies) after the forks; copies: (from, to) pages."""
    table, lens, copies = [list(r) for r in table], list(lens), []
    was, was_len = [list(r) for r in table], list(lens)
    for src, dst, fresh in forks:
        if not (0 <= src < len(was) and 0 <= dst < len(was)) or src == dst:
            continue
        n = was_len[src]
        if n < 0 or n > len(was[src]) * page_size:
            continue
        full, part = divmod(n, page_size)
        last = was[src][full] if part else -1
        if part and (not 0 <= last < n_pages or not 0 <= fresh < n_pages or last == fresh):
            continue
        table[dst] = was[src][:full] + ([fresh] if part else [])
        table[dst] += [-1] * (len(was[src]) - len(table[dst]))
        lens[dst] = n
        if part:
            copies.append((last, fresh))
    return table, lens, copies


def page_refs(table, lens, page_size, n_pages):
    refs = [0] * n_pages
    for row, n in zip(table, lens):
        for pg in row[:-(-max(n, 0) // page_size)]:
            if 0 <= pg < n_pages:
                refs[pg] += 1
    return refs


def compact(table, lens, page_size, n_pages):
    """(table, refs, n_live, moves)"""
    refs = page_refs(table, lens, page_size, n_pages)
    live = [p for p in range(n_pages) if refs[p]]
    n = len(live)
    moves = list(zip([p for p in live if p >= n], [p for p in range(n) if not refs[p]]))
    place = {p: p for p in live if p < n} | dict(moves)
    out = [[place[pg] if i * page_size < k and 0 <= pg < n_pages else -1 for i, pg in enumerate(row)]
           for row, k in zip(table, lens)]
    after = [0] * n_pages
    for p in live:
        after[place[p]] = refs[p]
    return out, after, n, moves


def block_norm(h, y, post_weight, post_norm, gate, alpha, beta, weights, eps):
    """(h', [x_j]) in fp64"""
    rms = lambda z: z / (z.square().mean(-1, keepdim=True) + eps).sqrt()
    h = alpha * h.double()
    if y is not None:
        u = y.double()
        if post_norm:
            u = rms(u) * (1 if post_weight is None else post_weight.double())
        h = h + beta * (u if gate is None else gate.double() * u)
    return h, [rms(h) * (1 if w is None else w.double()) for w in weights]


def verify(target, draft, drafts, u, u_next, n_draft):
    """(tokens, accepted) as lists, in Python's floats"""
    S, n1, V = target.shape
    clean = lambda t: torch.where((t > 0) & (t < math.inf), t.double(), torch.zeros((), dtype=torch.float64))
    tokens, accepted = [], []
    for s in range(S):
        n = min(max(int(n_draft[s]), 0), n1 - 1) if n_draft is not None else n1 - 1
        a = 0
        while a < n:
            x = int(drafts[s, a])
            if not 0 <= x < V:
                break
            p = float(clean(target[s, a, x]))
            q = 1.0 if draft is None else float(clean(draft[s, a, x]))
            if not float(u[s, a]) * q < p:
                break
            a += 1
        p = clean(target[s, a])
        r = p
        if a < n:
            off = torch.zeros_like(p)
            if draft is not None:
                off = clean(draft[s, a])
            elif 0 <= int(drafts[s, a]) < V:
                off[int(drafts[s, a])] = 1
            r = (p - off).clamp(min=0)
            if r.sum() == 0:
                r = p
        cum = r.cumsum(0)
        over = (cum > float(u_next[s]) * cum[-1]).nonzero()
        nxt = int(over[0]) if len(over) else int(r.nonzero()[-1]) if (r > 0).any() else -1
        tokens.append([int(drafts[s, i]) for i in range(a)] + [nxt] + [-1] * (n1 - 1 - a))
        accepted.append(a)
    return tokens, accepted
