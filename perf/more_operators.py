"""Measured cases of the operators that a serving step has before and after attention, and of
attention over a shared prefix: pages and slots for a step's new tokens, the norms of queries and
keys with their rotary positions, attention of sequences that begin with the same tokens, and
sampling.

`run` computes them in elementary torch operations (`own` false) or through the library (`own`
true); `exact` is each operator's definition in 64 bits.

The cache: a K page holds [n_kv][page][head_dim], a V page [n_kv][head_dim][page].  A q8_0 page holds,
for each head, int8 values in that order and then their fp16 scales, one for 32 values of a head's
vector, [head_dim / 32][page].
"""
import math

import torch

own = False

DEV = "cuda"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2, "q8_0": 34 / 32}


# ----------------------------------------------------------------- cases

def listed():
    return [
        # one decode step of a serving batch, a token each
        dict(name="extend 48 decode", op="extend", n_seq=48, new=1, max_len=5000, page=16, short=False),
        # chunks of prompts for a whole batch, and a free list too short for the last of them
        dict(name="extend 24 prompt chunks", op="extend", n_seq=24, new=2048, max_len=9000, page=32, short=True),
        # a speculative verify of one user: four tokens behind a long prompt
        dict(name="rope 4 x 24 x 256", op="rope", T=4, n_head=16, n_kv=8, hd=256, rot=256, layout="half", io="f32",
             scaling="plain", norm=True, top=11203),
        # a prompt chunk in bf16, a quarter of each head rotated, positions past the trained length
        dict(name="rope 8192 x 40 x 128 bf16", op="rope", T=8192, n_head=32, n_kv=8, hd=128, rot=32, layout="pairs",
             io="bf16", scaling="yarn", norm=True, top=131072),
        # ... without norms, whole heads
        dict(name="rope 2048 x 24 x 192 f16", op="rope", T=2048, n_head=20, n_kv=4, hd=192, rot=192, layout="half",
             io="f16", scaling="bands", norm=False, top=32000),
        # parallel samples of one prompt, where latency counts
        dict(name="prefix 8 on 1500", op="prefix", groups=1, n_seq=8, new=1, prefix=1500, lo=20, hi=300, n_head=16,
             n_kv=8, hd=256, page=64, kv="f16", io="f32", even=True),
        # a serving batch behind one long system prompt
        dict(name="prefix 64 on 32768 bf16", op="prefix", groups=1, n_seq=64, new=1, prefix=32768, lo=100, hi=1500,
             n_head=32, n_kv=8, hd=128, page=16, kv="bf16", io="bf16", even=True),
        # three documents with questions to each, drafts to verify, in an 8-bit cache
        dict(name="prefix 3 x 16 on 20011 q8_0", op="prefix", groups=3, n_seq=48, new=3, prefix=20011, lo=10, hi=700,
             n_head=32, n_kv=8, hd=128, page=128, kv="q8_0", io="bf16", even=False),
        # the next token of one user, all filters on
        dict(name="sample 1 of 32003", op="sample", n_seq=1, vocab=32003, io="f32", temp=0.8, top_k=40, top_p=0.95,
             min_p=0.05, mixed=False, probs=False),
        # a batch over a large vocabulary, every user with settings of their own
        dict(name="sample 32 of 262144", op="sample", n_seq=32, vocab=262144, io="f32", temp=1.0, top_k=64, top_p=0.9,
             min_p=0.02, mixed=True, probs=False),
        # nucleus sampling of drafts, whose probabilities the verification needs
        dict(name="sample 64 of 128001 bf16", op="sample", n_seq=64, vocab=128001, io="bf16", temp=0.7, top_k=0,
             top_p=0.95, min_p=0.0, mixed=False, probs=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["extend", "rope", "rope", "prefix", "prefix", "prefix", "sample", "sample"])
    io = rng.choice(["f32", "f16", "bf16"])
    page = rng.choice([16, 32, 64, 128])
    if op == "extend":
        n_seq = _log(rng, 1, 500)
        return dict(op=op, n_seq=n_seq, new=_log(rng, 1, max(2, 40000 // n_seq)), max_len=_log(rng, 10, 9000), page=page,
                    short=rng.random() < 0.3)
    if op == "rope":
        hd = rng.choice([64, 96, 128, 192, 256, 512])
        n_kv = rng.choice([1, 2, 3, 4, 8])
        n_head = n_kv * rng.choice([1, 2, 4, 5])
        return dict(op=op, T=_log(rng, 1, max(2, min(8192, int(4e7 / ((n_head + n_kv) * hd))))), n_head=n_head, n_kv=n_kv, hd=hd,
                    rot=rng.choice([hd, hd, hd // 2, hd // 4]), layout=rng.choice(["half", "pairs"]), io=io,
                    scaling=rng.choice(["plain", "linear", "ntk", "yarn", "bands"]), norm=rng.random() < 0.7,
                    top=_log(rng, 100, 1000000))
    if op == "prefix":
        hd, n_kv = rng.choice([64, 96, 128, 192, 256]), rng.choice([1, 2, 4, 8])
        n_seq = _log(rng, 2, 64)
        groups = rng.choice([1, 1, 2, 3])
        hi = _log(rng, 10, 1200)
        return dict(op=op, groups=min(groups, n_seq), n_seq=n_seq, new=rng.choice([1, 1, 2, 4]),
                    prefix=_log(rng, 100, min(32000, int(3e7 / (groups * n_kv * hd)))), lo=min(8, hi), hi=hi,
                    n_head=n_kv * rng.choice([1, 2, 4]), n_kv=n_kv, hd=hd, page=page,
                    kv=rng.choice(["f16", "bf16", "q8_0"]), io=io, even=rng.random() < 0.5)
    return dict(op=op, n_seq=_log(rng, 1, 64), vocab=_log(rng, 500, 130000), io=io, temp=rng.choice([0.3, 0.7, 1.0, 1.5]),
                top_k=rng.choice([0, 0, 1, 20, 50, 1000]), top_p=rng.choice([1.0, 0.5, 0.9, 0.95, 0.99]),
                min_p=rng.choice([0.0, 0.0, 0.02, 0.1]), mixed=rng.random() < 0.4, probs=rng.random() < 0.4)


# ---------------------------------------------------------------- inputs

def _ints(g, lo, hi, n):
    """n whole numbers of lo .. hi, as a list"""
    return torch.randint(lo, hi + 1, (n,), generator=g).tolist()


def _pool(c, n_pages, gd):
    """K and V pools with random contents: typed tensors, or bytes for q8_0."""
    H, P, D = c["n_kv"], c["page"], c["hd"]
    if c["kv"] != "q8_0":
        make = lambda *s: torch.randn(n_pages, H, *s, generator=gd, device=DEV, dtype=torch.float32).to(TYPES[c["kv"]])
        return make(P, D), make(D, P)
    made = []
    for _ in range(2):
        q = torch.randint(-127, 128, (n_pages, H, P * D), generator=gd, device=DEV, dtype=torch.int8)
        d = (0.005 + 0.02 * torch.rand(n_pages, H, P * D // 32, generator=gd, device=DEV)).half()
        made.append(torch.cat([q.view(torch.uint8), d.view(torch.uint8)], -1).reshape(n_pages, -1))
    return tuple(made)


def frequencies(scaling, rot):
    """(frequency of each rotated pair in 64 bits, the factor on cosine and sine) by the published rules."""
    base, factor, trained = 500000.0, 8.0, 8192.0
    i = torch.arange(rot // 2, dtype=torch.float64)
    if scaling == "ntk" and rot > 2:
        base *= factor ** (rot / (rot - 2))
    f = base ** (-2 * i / rot)
    if scaling == "linear":
        f = f / factor
    if scaling == "yarn":
        at = lambda turns: rot * math.log(trained / (turns * 2 * math.pi)) / (2 * math.log(base))
        lo, hi = max(math.floor(at(32.0)), 0), min(math.ceil(at(1.0)), rot - 1)
        ramp = ((i - lo) / max(hi - lo, 0.001)).clamp(0, 1)
        f = f / factor * ramp + f * (1 - ramp)
    if scaling == "bands":
        turns = trained * f / (2 * math.pi)
        s = ((turns - 1.0) / (4.0 - 1.0)).clamp(0, 1)
        f = (1 - s) * f / factor + s * f
    return f, 0.1 * math.log(factor) + 1.0 if scaling == "yarn" else 1.0


def prepare(case, seed):
    c, g = case, torch.Generator().manual_seed(seed)
    gd = torch.Generator(DEV).manual_seed(seed)
    s = {"c": c}
    # the sizes are the case's, their order among the sequences is the seed's
    sizes = torch.Generator().manual_seed(7)
    up = lambda v, t=torch.int32: torch.as_tensor(v, dtype=t).to(DEV)
    randn = lambda *n: torch.randn(*n, generator=gd, device=DEV)
    if c["op"] == "extend":
        P, S = c["page"], c["n_seq"]
        order = torch.randperm(S, generator=g).tolist()
        lens, new = _ints(sizes, 0, c["max_len"], S), _ints(sizes, 0 if c["new"] > 1 else 1, c["new"], S)
        lens, new = [lens[o] for o in order], [new[o] for o in order]
        width = -(-(c["max_len"] + c["new"]) // P)
        held = sum(-(-n // P) for n in lens)
        need = sum(-(-(n + k) // P) - -(-n // P) for n, k in zip(lens, new))
        n_free = max(need * 2 // 3, 1) if c["short"] else need + 5
        ids = torch.randperm(held + n_free, generator=g).to(torch.int32)
        table, at = torch.full((S, width), -1, dtype=torch.int32), 0
        for i, n in enumerate(lens):
            k = -(-n // P)
            table[i, :k] = ids[at:at + k]
            at += k
        free = torch.full((held + n_free,), -1, dtype=torch.int32)
        free[:n_free] = ids[held:]
        # some rows more than tokens, as a step of fixed size has them
        T = sum(new) + 3
        s.update(table=table.to(DEV), lens=up(lens), new=up(new), free=free.to(DEV), n_free=up([n_free]), T=T,
                 n_pages=held + n_free, lens_out=up([0] * S), n_free_out=up([0]), start=up([0] * (S + 1)), pos=up([0] * T),
                 seq=up([0] * T), slots=up([0] * T, torch.int64))
    elif c["op"] == "rope":
        io, T, D = TYPES[c["io"]], c["T"], c["hd"]
        # rows of a fused projection: queries, keys, values
        s["qkv"] = randn(T, c["n_head"] + 2 * c["n_kv"], D).mul_(2).to(io)
        s["q"], s["k"] = s["qkv"][:, :c["n_head"]], s["qkv"][:, c["n_head"]:c["n_head"] + c["n_kv"]]
        s["wq"], s["wk"] = (1 + 0.2 * randn(D) if c["norm"] else None for _ in range(2))
        first = _ints(g, 0, max(c["top"] - T, 0), 1)[0]
        s["pos"] = up(list(range(first, first + T)))
        freq, s["magnitude"] = frequencies(c["scaling"], c["rot"])
        s["freq"] = freq.to(DEV)
        s["q_out"], s["k_out"] = (torch.empty(t.shape, dtype=io, device=DEV) for t in (s["q"], s["k"]))
    elif c["op"] == "prefix":
        S, N, P = c["n_seq"], c["groups"], c["page"]
        order = torch.randperm(S, generator=g).tolist()
        lo, hi = math.log(c["lo"]), math.log(c["hi"])
        tails = [max(round(math.exp(lo + (hi - lo) * r)), c["new"]) for r in torch.rand(S, generator=sizes).tolist()]
        new = [c["new"] if c["even"] else min(k, c["new"]) for k in _ints(sizes, 1, c["new"], S)]
        tails, new = [tails[o] for o in order], [new[o] for o in order]
        # a group's sequences share the prefix's full pages; its last tokens are each one's own
        share = [c["prefix"] // (1 + i) // P * P for i in range(N)]
        members = [S * (i + 1) // N - S * i // N for i in range(N)]
        lens, width = [], 0
        for n, k in zip(share, members):
            lens += [n + t for t in tails[len(lens):len(lens) + k]]
        width = max(-(-n // P) for n in lens)
        own_pages = [-(-t // P) for t in tails]
        n_pages = sum(n // P for n in share) + sum(own_pages) + 3
        ids = torch.randperm(n_pages, generator=g).to(torch.int32)
        table, at, q = torch.full((S, width), -1, dtype=torch.int32), 0, 0
        for n, k in zip(share, members):
            row = ids[at:at + n // P]
            at += n // P
            for _ in range(k):
                table[q, :n // P] = row
                table[q, n // P:n // P + own_pages[q]] = ids[at:at + own_pages[q]]
                at += own_pages[q]
                q += 1
        start, first = [0], [0]
        for n in new:
            start.append(start[-1] + n)
        for k in members:
            first.append(first[-1] + k)
        io = TYPES[c["io"]]
        s["k"], s["v"] = _pool(c, n_pages, gd)
        s["q"] = (1.5 * randn(start[-1], c["n_head"], c["hd"])).to(io)
        s.update(table=table.to(DEV), lens=up(lens), start=up(start), groups=up(first), prefix=up(share), T=start[-1],
                 max_new=max(new), share=share, first=first, tails=tails, rows=start, out=torch.empty_like(s["q"]),
                 lse=torch.empty(start[-1], c["n_head"], device=DEV))
    else:
        S, V = c["n_seq"], c["vocab"]
        logits = 2.2 * randn(S, V)
        # what the text allows stands out
        likely = torch.randint(0, V, (S, 24), generator=gd, device=DEV)
        logits.scatter_add_(1, likely, 4 + 4 * torch.rand(S, 24, generator=gd, device=DEV))
        s["logits"] = logits.to(TYPES[c["io"]])
        s["u"] = torch.rand(S, generator=gd, device=DEV)
        pick = _ints(sizes, 0, 5, S) if c["mixed"] else [5] * S
        s["temp"] = up([0.0 if p == 0 else c["temp"] for p in pick], torch.float32)
        s["top_k"] = up([0 if p in (1, 2) else c["top_k"] for p in pick])
        s["top_p"] = up([1.0 if p in (1, 3) else c["top_p"] for p in pick], torch.float32)
        s["min_p"] = up([0.0 if p in (1, 4) else c["min_p"] for p in pick], torch.float32)
        s["tokens"] = up([0] * S)
        s["probs"] = torch.empty_like(s["logits"]) if c["probs"] else None
    if own:
        _handles(c, s)
    return s


def _handles(c, s):
    """What a program keeps of the library between calls: descriptors and workspaces."""
    import llapis_amd as la
    s["la"] = la
    if c["op"] == "extend":
        pool = torch.empty(s["n_pages"], 1, c["page"], 64, dtype=torch.float16, device=DEV)
        s["pages"] = la.KvPages([la.KvCache(pool, pool.view(s["n_pages"], 1, 64, c["page"]))])
        s["ws"] = s["pages"].extend_workspace(c["n_seq"])
    elif c["op"] == "prefix":
        geo = dict(type=la.Q8_0, n_kv=c["n_kv"], head_dim=c["hd"], page_size=c["page"]) if c["kv"] == "q8_0" else {}
        s["cache"] = la.KvCache(s["k"], s["v"], **geo)
        s["batch"] = la.KvBatch(s["table"], s["lens"], s["start"], n_tokens=s["T"], max_new=s["max_new"])
        s["ws"] = s["cache"].prefix_workspace(s["batch"], c["n_head"], c["groups"])
    elif c["op"] == "sample":
        s["ws"] = la.sample_workspace(c["n_seq"], c["vocab"], DEV)
    else:
        s["layout"] = la.ROPE_HALF if c["layout"] == "half" else la.ROPE_PAIRS


# ------------------------------------------------------------- operators

def run(state):
    return (_own if own else _plain)[state["c"]["op"]](state)


def _extend_out(s):
    return s["table"], s["lens_out"], s["n_free_out"], s["start"], s["pos"], s["seq"], s["slots"]


def _own_extend(s):
    s["pages"].extend(s["table"], s["lens"], s["new"], s["free"], s["n_free"], s["T"], lens_out=s["lens_out"],
                      n_free_out=s["n_free_out"], new_start=s["start"], pos=s["pos"], seq=s["seq"], slots=s["slots"],
                      workspace=s["ws"])
    return _extend_out(s)


def _own_rope(s):
    s["la"].qk_rope(s["q"], s["k"], s["pos"], s["freq"], q_weight=s["wq"], k_weight=s["wk"], norm=s["c"]["norm"], eps=1e-6,
                    magnitude=s["magnitude"], layout=s["layout"], q_out=s["q_out"], k_out=s["k_out"])
    return s["q_out"], s["k_out"]


def _own_prefix(s):
    s["cache"].prefix_attention(s["batch"], s["q"], s["groups"], s["prefix"], scale=s["c"]["hd"] ** -0.5, out=s["out"],
                                lse=s["lse"], workspace=s["ws"])
    return s["out"], s["lse"]


def _own_sample(s):
    s["la"].sample(s["logits"], s["u"], temperature=s["temp"], top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"],
                   tokens=s["tokens"], probs=s["probs"], workspace=s["ws"])
    return s["tokens"], s["probs"]


_own = dict(extend=_own_extend, rope=_own_rope, prefix=_own_prefix, sample=_own_sample)


def _plain_extend(s):
    P, T, table = s["c"]["page"], s["T"], s["table"]
    S, width = table.shape
    n, want = s["lens"].long(), s["new"].long()
    # the sequences whose rows and pages fit, in order
    want = torch.where(n + want <= width * P, want, 0)
    want = torch.where(want.cumsum(0) <= T, want, 0)
    pages = lambda k: (k + P - 1) // P
    need = pages(n + want) - pages(n)
    want = torch.where((need == 0) | (need.cumsum(0) <= s["n_free"]), want, 0)
    need = pages(n + want) - pages(n)
    upto, ends = need.cumsum(0), want.cumsum(0)
    s["lens_out"].copy_(n + want)
    s["start"][0] = 0
    s["start"][1:] = ends
    s["n_free_out"].copy_(s["n_free"] - upto[-1])
    # new table entries, from the free list's end
    i = torch.arange(width, device=DEV) - pages(n)[:, None]
    take = (upto - need)[:, None] + i
    fresh = s["free"][(s["n_free"].long() - 1 - take).clamp(0, s["free"].shape[0] - 1)]
    table.copy_(torch.where((i >= 0) & (i < need[:, None]), fresh, table))
    r = torch.arange(T, device=DEV)
    seq = torch.searchsorted(ends, r, right=True)
    there, q = seq < S, seq.clamp(max=S - 1)
    pos = (n + want)[q] - ends[q] + r
    page = table[q, (pos // P).clamp(0, width - 1)].long()
    ok = there & (page >= 0) & (page < s["n_pages"])
    s["pos"].copy_(torch.where(there, pos, -1))
    s["seq"].copy_(torch.where(there, seq, -1))
    s["slots"].copy_(torch.where(ok, page * P + pos % P, -1))
    return _extend_out(s)


def _plain_rope(s):
    c, rot = s["c"], s["c"]["rot"]
    # far positions: angles in 64 bits
    angle = s["pos"].double()[:, None] * s["freq"]
    cos, sin = ((f(angle) * s["magnitude"]).float()[:, None] for f in (torch.cos, torch.sin))
    for x, w, out in ((s["q"], s["wq"], s["q_out"]), (s["k"], s["wk"], s["k_out"])):
        x = x.float()
        if c["norm"]:
            x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w
        if c["layout"] == "half":
            a, b = x[..., :rot // 2], x[..., rot // 2:rot]
            y = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
        else:
            a, b = x[..., 0:rot:2], x[..., 1:rot:2]
            y = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
        out.copy_(torch.cat([y, x[..., rot:]], -1))
    return s["q_out"], s["k_out"]


def _values(pages, c, is_v):
    """Gathered pages' values in 32 bits: [..., n_kv, page, hd], for V [..., n_kv, hd, page]."""
    if c["kv"] != "q8_0":
        return pages.float()
    H, P, D = c["n_kv"], c["page"], c["hd"]
    by_head = pages.reshape(*pages.shape[:-1], H, -1)
    q = by_head[..., :P * D].contiguous().view(torch.int8).float()
    d = by_head[..., P * D:].contiguous().view(torch.float16).float()
    if is_v:
        return (q.reshape(*q.shape[:-1], D // 32, 32, P) * d.reshape(*d.shape[:-1], D // 32, 1, P)).flatten(-3, -2)
    d = d.reshape(*d.shape[:-1], D // 32, P).transpose(-1, -2)
    return (q.reshape(*q.shape[:-1], P, D // 32, 32) * d[..., None]).flatten(-2)


def _keys(s, page_ids):
    """K and V [..., n_kv, keys, hd] of pages [..., n]"""
    c, n = s["c"], page_ids.dim()
    k, v = _values(s["k"][page_ids], c, False), _values(s["v"][page_ids], c, True)
    return (t.transpose(n - 1, n).flatten(n, n + 1) for t in (k, v.transpose(-1, -2)))


def _part(q, k, v, seen=None):
    """Unnormalised result, maximum and sum of softmax attention over these keys; q [..., n_kv, rows, hd]."""
    z = torch.matmul(q, k.transpose(-1, -2).contiguous()).mul_(q.shape[-1] ** -0.5)
    if seen is not None:
        z.masked_fill_(~seen, -math.inf)
    m = z.amax(-1, keepdim=True)
    p = torch.exp(z.sub_(m.clamp(min=-3e38)))
    return torch.matmul(p, v.contiguous()), m, p.sum(-1, keepdim=True)


def _plain_prefix(s):
    c = s["c"]
    H, D, P, G, N = c["n_kv"], c["hd"], c["page"], c["n_head"] // c["n_kv"], s["max_new"]
    table, start, lens = s["table"].long().clamp(min=0), s["start"].long(), s["lens"].long()
    j = torch.arange(N, device=DEV)
    for share, f, e in zip(s["share"], s["first"], s["first"][1:]):
        # queries of the group, rows that a sequence lacks filled up: [sequences, n_kv, new x heads, hd]
        new = start[f + 1:e + 1] - start[f:e]
        there = j < new[:, None]
        rows = (start[f:e, None] + j).clamp(max=s["T"] - 1)
        q = s["q"][rows].float().reshape(e - f, N, H, G, D).permute(0, 2, 1, 3, 4).reshape(e - f, H, N * G, D)
        # the sequences' own keys, then the prefix once for all rows of the group
        tail = max(-(-n // P) for n in s["tails"][f:e])
        k, v = _keys(s, torch.nn.functional.pad(table[f:e], (0, tail))[:, share // P:share // P + tail])
        last = (lens[f:e] - share - new)[:, None] + j
        seen = torch.arange(tail * P, device=DEV) <= torch.where(there, last, 0)[..., None]
        o, m, l = _part(q, k, v, seen.repeat_interleave(G, 1)[:, None])
        if share:
            k, v = _keys(s, table[f, :share // P])
            o2, m2, l2 = (t.unflatten(1, (e - f, N * G)).transpose(0, 1) for t in _part(q.transpose(0, 1).flatten(1, 2), k, v))
            top = torch.maximum(m, m2)
            a, a2 = torch.exp(m - top), torch.exp(m2 - top)
            o, m, l = o * a + o2 * a2, top, l * a + l2 * a2
        by_row = lambda t: t.unflatten(2, (N, G)).transpose(1, 2).flatten(2, 3)[there]
        s["out"][rows[there]] = by_row(o / l).to(s["out"].dtype)
        s["lse"][rows[there]] = by_row(m + torch.log(l)).squeeze(-1)
    return s["out"], s["lse"]


def _plain_sample(s):
    # weights and their sums in 64 bits: draws lie next to borders
    x = s["logits"].double()
    S, V = x.shape
    temp, top_p, min_p = (s[k].double()[:, None] for k in ("temp", "top_p", "min_p"))
    x, order = torch.sort(x, dim=-1, descending=True, stable=True)
    w = torch.exp((x - x[:, :1]) / temp.clamp(min=1e-30))
    rank = torch.arange(V, device=DEV)
    k = torch.where(s["top_k"] > 0, s["top_k"], V)[:, None]
    k = torch.where(temp > 0, k, 1)
    w = w.masked_fill_(rank >= k, 0.0)
    upto = w.cumsum(1)
    keep = (top_p >= 1) | (upto - w < top_p * upto[:, -1:])
    keep &= w >= min_p
    keep[:, 0] = True
    w = torch.zeros_like(w).scatter_(1, order, torch.where(keep, w, 0.0))
    cum = w.cumsum(1)
    s["tokens"].copy_((cum <= s["u"].double()[:, None] * cum[:, -1:]).sum(1).clamp(max=V - 1))
    if s["probs"] is not None:
        s["probs"].copy_(w / cum[:, -1:])
    return s["tokens"], s["probs"]


_plain = dict(extend=_plain_extend, rope=_plain_rope, prefix=_plain_prefix, sample=_plain_sample)


# ------------------------------------------------------------------ work

def work(case):
    c, op = case, case["op"]
    if op == "extend":
        # rows are 16 bytes of positions, sequences and slots
        new = c["n_seq"] * (1 if c["new"] == 1 else c["new"] / 2)
        return {"bytes": 16 * new + 8 * new / c["page"] + 16 * c["n_seq"], "flops": 0}
    if op == "rope":
        values = c["T"] * (c["n_head"] + c["n_kv"]) * c["hd"]
        return {"bytes": 2 * values * SIZE[c["io"]] + 4 * c["T"], "flops": values * (4 * c["norm"] + 3 * c["rot"] / c["hd"])}
    if op == "prefix":
        shared = [c["prefix"] // (1 + i) // c["page"] * c["page"] for i in range(c["groups"])]
        tail = (c["hi"] - c["lo"]) / math.log(c["hi"] / c["lo"]) if c["hi"] > c["lo"] else c["hi"]
        new = c["new"] if c["even"] else (1 + c["new"]) / 2
        keys = sum(shared) + c["n_seq"] * tail
        seen = sum(shared) / c["groups"] + tail
        return {"bytes": 2 * keys * c["n_kv"] * c["hd"] * SIZE[c["kv"]]
                + 2 * c["n_seq"] * new * c["n_head"] * c["hd"] * SIZE[c["io"]],
                "flops": 4 * seen * c["n_seq"] * new * c["n_head"] * c["hd"]}
    return {"bytes": c["n_seq"] * c["vocab"] * SIZE[c["io"]] * (2 if c["probs"] else 1), "flops": 4 * c["n_seq"] * c["vocab"]}


# ----------------------------------------------------------------- exact

def exact(case, seed):
    c = case
    if c["op"] == "extend":
        return None  # whole numbers
    global own
    was, own = own, False
    try:
        s = prepare(c, seed)
    finally:
        own = was
    if c["op"] == "rope":
        return _exact_rope(c, s)
    if c["op"] == "prefix":
        return _exact_prefix(c, s)
    if s["probs"] is None:
        return None
    p = torch.zeros(c["n_seq"], c["vocab"], dtype=torch.float64, device=DEV)
    for i in range(c["n_seq"]):
        x, (t, k) = s["logits"][i].double(), (float(s["temp"][i]), int(s["top_k"][i]))
        if t <= 0:
            p[i, int((x == x.max()).nonzero()[0])] = 1
            continue
        p[i] = torch.softmax(x / t, 0)
        z, at = torch.sort(x, descending=True, stable=True)
        if k > 0:
            p[i, at[k:]] = 0
        if float(s["top_p"][i]) < 1:
            mass = p[i, at].cumsum(0)
            n = int((mass < float(s["top_p"][i]) * mass[-1]).sum()) + 1
            p[i, at[n:]] = 0
        p[i] *= p[i] >= float(s["min_p"][i]) * p[i].max()
        p[i] /= p[i].sum()
    return None, p


def _exact_rope(c, s):
    rot, made = c["rot"], []
    freq, magnitude = frequencies(c["scaling"], rot)
    turn = torch.polar(torch.full((c["T"], rot // 2), magnitude, dtype=torch.float64, device=DEV),
                       s["pos"].double()[:, None] * freq.to(DEV))[:, None]
    for x, w in ((s["q"], s["wq"]), (s["k"], s["wk"])):
        x = x.double()
        if c["norm"]:
            x = x / ((x * x).sum(-1, keepdim=True) / c["hd"] + 1e-6).sqrt() * w.double()
        else:
            x = x.clone()
        a, b = ((slice(0, rot // 2), slice(rot // 2, rot)) if c["layout"] == "half" else (slice(0, rot, 2), slice(1, rot, 2)))
        z = torch.complex(x[..., a], x[..., b]) * turn
        x[..., a], x[..., b] = z.real, z.imag
        made.append(x)
    return tuple(made)


def _exact_prefix(c, s):
    P, D, G = c["page"], c["hd"], c["n_head"] // c["n_kv"]
    out = torch.zeros(s["T"], c["n_head"], D, dtype=torch.float64, device=DEV)
    lse = torch.zeros(s["T"], c["n_head"], dtype=torch.float64, device=DEV)
    for i, n in enumerate(s["lens"].tolist()):
        pages = s["table"][i, :-(-n // P)].long()
        new = s["rows"][i + 1] - s["rows"][i]
        for h in range(c["n_kv"]):
            if c["kv"] == "q8_0":
                part = [t.view(t.shape[0], c["n_kv"], -1)[pages, h] for t in (s["k"], s["v"])]
                q8 = [t[:, :P * D].contiguous().view(torch.int8).double() for t in part]
                sc = [t[:, P * D:].contiguous().view(torch.float16).double() for t in part]
                k = q8[0].view(-1, D) * sc[0].view(-1, D // 32, P).transpose(1, 2).reshape(-1, D // 32).repeat_interleave(32, 1)
                v = q8[1].view(-1, D, P) * sc[1].view(-1, D // 32, P).repeat_interleave(32, 1)
            else:
                k, v = s["k"][pages, h].double().view(-1, D), s["v"][pages, h].double()
            v = v.transpose(1, 2).reshape(-1, D)
            for j in range(new):
                end, r = n - new + j + 1, s["rows"][i] + j
                z = (s["q"][r, h * G:(h + 1) * G].double() @ k[:end].T) / math.sqrt(D)
                top = z.max(1, keepdim=True).values
                e = (z - top).exp()
                out[r, h * G:(h + 1) * G] = (e @ v[:end]) / e.sum(1, keepdim=True)
                lse[r, h * G:(h + 1) * G] = top[:, 0] + e.sum(1).log()
    return out, lse
