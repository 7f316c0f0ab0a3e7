"""Measured cases of the operators of a decode step around the MoE layer: attention over a paged
key-value cache and its append, forks and compaction of the cache's pages, the norms before and
after a block, and the verification of drafted tokens.

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
        # one user's chat, one token: a short cache, where latency counts
        dict(name="attn 1 token of 700", op="attn", n_seq=1, new=1, min_len=700, max_len=700, n_head=16, n_kv=8,
             hd=256, page=64, window=0, kv="f16", io="f32", even=True),
        # a speculative verify of the token and three drafts behind a long prompt
        dict(name="attn 4 tokens of 11203", op="attn", n_seq=1, new=4, min_len=11203, max_len=11203, n_head=16, n_kv=2,
             hd=512, page=64, window=0, kv="f16", io="f32", even=True),
        # a serving batch in bf16, lengths and draft counts ragged, small pages
        dict(name="attn 48 ragged bf16", op="attn", n_seq=48, new=4, min_len=17, max_len=5000, n_head=32, n_kv=8,
             hd=128, page=16, window=0, kv="bf16", io="bf16", even=False),
        # two long documents in an 8-bit cache
        dict(name="attn 2 of 131072 q8_0", op="attn", n_seq=2, new=1, min_len=131071, max_len=131072, n_head=32, n_kv=8,
             hd=128, page=128, window=0, kv="q8_0", io="bf16", even=True),
        # the cache write of a decode batch, and of a prompt chunk
        dict(name="append 48 decode", op="append", n_seq=48, new=4, max_len=600, n_kv=8, hd=128, page=16, kv="bf16",
             io="bf16", even=False),
        dict(name="append 2048 prompt", op="append", n_seq=2, new=1024, max_len=1500, n_kv=8, hd=256, page=64,
             kv="f16", io="f32", even=True),
        # parallel samples of one prompt: its full pages shared, the last one copied in every layer
        dict(name="fork 3 in 30 layers", op="fork", layers=30, n_seq=6, forks=3, max_len=300, n_kv=8, hd=128, page=16,
             kv="f16"),
        # the pool's tail emptied after many sequences ended
        dict(name="compact 1024 pages", op="compact", layers=4, n_seq=64, n_pages=1024, max_len=1500, n_kv=8, hd=128,
             page=64, kv="bf16"),
        # the glue of one decode step of 4 tokens: the experts' and the router's inputs from one residual stream
        dict(name="norm 4 x 2816", op="norm", T=4, d=2816, outs=2, post=True, gate="none", io="f32"),
        # ... and of a long prompt, gated, in bf16
        dict(name="norm 11200 x 2816 bf16", op="norm", T=11200, d=2816, outs=2, post=True, gate="channel", io="bf16"),
        # a batch of depth-3 drafts over a large vocabulary
        dict(name="verify 32 x 3 of 262144", op="verify", n_seq=32, drafts=3, vocab=262144, io="f32", onehot=False,
             even=False),
        # one user's greedy drafts, whose drafting model kept no probabilities
        dict(name="verify 1 x 3 of 32003", op="verify", n_seq=1, drafts=3, vocab=32003, io="f32", onehot=True,
             even=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attn", "attn", "attn", "append", "fork", "compact", "norm", "verify"])
    kv, io = rng.choice(["f16", "bf16", "q8_0"]), rng.choice(["f32", "f16", "bf16"])
    page, hd = rng.choice([16, 32, 64, 128]), rng.choice([64, 96, 128, 192, 256])
    n_kv = rng.choice([1, 2, 3, 4, 8])
    if op == "attn":
        n_seq = _log(rng, 1, 64)
        top = max(64, int(min(131072, 1.2e8 / (n_seq * n_kv * hd))))
        max_len = _log(rng, 32, top)
        return dict(op=op, n_seq=n_seq, new=rng.choice([1, 1, 2, 3, 4, 6]), min_len=rng.randint(8, max_len), max_len=max_len,
                    n_head=n_kv * rng.choice([1, 2, 4, 5, 8]), n_kv=n_kv, hd=hd, page=page,
                    window=rng.choice([0, 0, rng.randint(1, 2000)]), kv=kv, io=io, even=rng.random() < 0.5)
    if op == "append":
        n_seq = _log(rng, 1, 64)
        new = _log(rng, 1, max(2, 2048 // n_seq))
        return dict(op=op, n_seq=n_seq, new=new, max_len=new + rng.randint(1, 500), n_kv=n_kv, hd=hd, page=page,
                    kv=rng.choice(["f16", "bf16"]), io=io, even=rng.random() < 0.5)
    if op == "fork":
        n_seq = rng.randint(2, 24)
        return dict(op=op, layers=rng.randint(1, 32), n_seq=n_seq, forks=rng.randint(1, n_seq // 2),
                    max_len=rng.randint(20, 300), n_kv=min(n_kv, 4), hd=min(hd, 128), page=page,
                    kv=rng.choice(["f16", "bf16"]))
    if op == "compact":
        return dict(op=op, layers=rng.randint(1, 4), n_seq=rng.randint(3, 64), n_pages=_log(rng, 40, 1024),
                    max_len=rng.randint(100, 2000), n_kv=min(n_kv, 4), hd=min(hd, 128), page=page,
                    kv=rng.choice(["f16", "bf16"]))
    if op == "norm":
        return dict(op=op, T=_log(rng, 1, 11200), d=rng.choice([_log(rng, 64, 2900), 512, 1024, 2048, 2816]),
                    outs=rng.randint(1, 3), post=rng.random() < 0.7,
                    gate=rng.choice(["none", "token", "channel", "full"]), io=io)
    return dict(op=op, n_seq=_log(rng, 1, 32), drafts=rng.randint(1, 6), vocab=_log(rng, 500, 130000), io=io,
                onehot=rng.random() < 0.3, even=rng.random() < 0.5)


# ---------------------------------------------------------------- inputs

def _ints(g, lo, hi, n):
    """n whole numbers of lo .. hi, as a list"""
    return torch.randint(lo, hi + 1, (n,), generator=g).tolist()


def _pool(c, n_pages, gd, layers=None):
    """K and V pools with random contents: typed tensors, or bytes for q8_0."""
    lead = (n_pages,) if layers is None else (layers, n_pages)
    H, P, D = c["n_kv"], c["page"], c["hd"]
    if c["kv"] != "q8_0":
        make = lambda *s: torch.randn(*lead, H, *s, generator=gd, device=DEV, dtype=torch.float32).to(TYPES[c["kv"]])
        return make(P, D), make(D, P)
    made = []
    for _ in range(2):
        q = torch.randint(-127, 128, (*lead, H, P * D), generator=gd, device=DEV, dtype=torch.int8)
        d = (0.005 + 0.02 * torch.rand(*lead, H, P * D // 32, generator=gd, device=DEV)).half()
        made.append(torch.cat([q.view(torch.uint8), d.view(torch.uint8)], -1).reshape(*lead, -1))
    return tuple(made)


def _pages(c, lens, g, spare=3, width=None):
    """A page table with the pages in random order, and the pool's size."""
    need = [-(-n // c["page"]) for n in lens]
    n_pages = sum(need) + spare
    order = torch.randperm(n_pages, generator=g).tolist()
    table = torch.full((len(lens), width or max(1, max(need))), -1, dtype=torch.int32)
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
        at += n
    return table, n_pages


def _rows(c, lens, sizes, order):
    """New tokens of each sequence and the first row of each."""
    most = _ints(sizes, 1, c["new"], len(lens))
    new = [min(n, c["new"] if c["even"] else most[o]) for n, o in zip(lens, order)]
    start = [0]
    for n in new:
        start.append(start[-1] + n)
    return new, start


def prepare(case, seed):
    c, g = case, torch.Generator().manual_seed(seed)
    gd = torch.Generator(DEV).manual_seed(seed)
    s = {"c": c}
    # the sizes are the case's, their order among the sequences is the seed's
    sizes, order = torch.Generator().manual_seed(7), None
    if "n_seq" in c:
        order = torch.randperm(c["n_seq"] - c.get("forks", 0), generator=g).tolist()
    mixed = lambda v: [v[o] for o in order]
    up = lambda v: torch.as_tensor(v, dtype=torch.int32).to(DEV)
    randn = lambda *n: torch.randn(*n, generator=gd, device=DEV)
    if c["op"] in ("attn", "append"):
        if c["op"] == "attn":
            lo, hi = math.log(c["min_len"]), math.log(c["max_len"])
            lens = [round(math.exp(lo + (hi - lo) * r)) for r in torch.rand(c["n_seq"], generator=sizes).tolist()]
            lens[0] = c["max_len"]
        else:
            lens = _ints(sizes, c["new"], c["max_len"], c["n_seq"])
        lens = mixed(lens)
        table, n_pages = _pages(c, lens, g)
        new, start = _rows(c, lens, sizes, order)
        s.update(k=None, table=table.to(DEV), lens=up(lens), start=up(start), max_new=max(new), T=start[-1])
        s["k"], s["v"] = _pool(c, n_pages, gd)
        io = TYPES[c["io"]]
        if c["op"] == "attn":
            s["q"] = (1.5 * randn(s["T"], c["n_head"], c["hd"])).to(io)
            s["out"] = torch.empty_like(s["q"])
            s["lse"] = torch.empty(s["T"], c["n_head"], device=DEV)
        else:
            s["kn"], s["vn"] = (randn(s["T"], c["n_kv"], c["hd"]).to(io) for _ in range(2))
    elif c["op"] in ("fork", "compact"):
        if c["op"] == "fork":
            lens = mixed(_ints(sizes, 1, c["max_len"], c["n_seq"])) + [0] * c["forks"]
            table, n_pages = _pages(c, lens, g, spare=c["forks"], width=-(-c["max_len"] // c["page"]) + 1)
            taken = set(table[table >= 0].tolist())
            fresh = [p for p in range(n_pages) if p not in taken][:c["forks"]]
            src = _ints(g, 0, c["n_seq"] - c["forks"] - 1, c["forks"])
            dst = range(c["n_seq"] - c["forks"], c["n_seq"])
            s["forks"] = up(list(zip(src, dst, fresh)))
        else:
            # sequences until the pool is full, then about half of them ended
            n_pages, left, lens = c["n_pages"], c["n_pages"], []
            for n in mixed(_ints(sizes, 1, c["max_len"], c["n_seq"])):
                n = min(n, left * c["page"])
                left -= -(-n // c["page"])
                lens.append(n)
            table, _ = _pages(c, lens, g, spare=left)
            ended = torch.rand(c["n_seq"], generator=g).tolist()
            lens = [0 if e < 0.5 else n for n, e in zip(lens, ended)]
            s["table_out"] = torch.empty_like(table, device=DEV)
            s["refs"] = torch.empty(n_pages, dtype=torch.int32, device=DEV)
            s["n_live"] = torch.empty(1, dtype=torch.int32, device=DEV)
        s.update(table=table.to(DEV), lens=up(lens), n_pages=n_pages)
        s["k"], s["v"] = _pool(c, n_pages, gd, c["layers"])
    elif c["op"] == "norm":
        T, d, io = c["T"], c["d"], TYPES[c["io"]]
        s["y"], s["h"] = (0.3 * randn(T, d)).to(io), (2 * randn(T, d)).to(io)
        s["post"] = 1 + 0.2 * randn(d) if c["post"] else None
        s["pre"] = [1 + 0.2 * randn(d) for _ in range(c["outs"])]
        shape = {"none": None, "token": (T, 1), "channel": (1, d), "full": (T, d)}[c["gate"]]
        s["gate"] = None if shape is None else torch.sigmoid(randn(*shape)).to(io)
        s["h_out"], s["x"] = torch.empty_like(s["h"]), [torch.empty_like(s["h"]) for _ in range(c["outs"])]
    else:
        S, n, V = c["n_seq"], c["drafts"], c["vocab"]
        logits = 2.5 * randn(S, n + 1, V)
        s["p"] = torch.softmax(logits, -1).to(TYPES[c["io"]])
        q = torch.softmax(logits[:, :n] + 0.7 * randn(S, n, V), -1)
        noise = torch.rand(S, n, V, generator=gd, device=DEV).clamp_(min=1e-20).log_().neg_()
        s["drafts"] = (q / noise).argmax(-1).to(torch.int32)
        s["q"] = None if c["onehot"] else q.to(TYPES[c["io"]])
        s["n_draft"] = up([n] * S if c["even"] else _ints(g, 0, n, S))
        s["u"] = torch.rand(S, n, generator=gd, device=DEV)
        s["u_next"] = torch.rand(S, generator=gd, device=DEV)
        s["tokens"] = torch.empty(S, n + 1, dtype=torch.int32, device=DEV)
        s["accepted"] = torch.empty(S, dtype=torch.int32, device=DEV)
    if own:
        _handles(c, s)
    return s


def _handles(c, s):
    """What a program keeps of the library between calls: descriptors and workspaces."""
    import llapis_amd as la
    s["la"] = la
    if c["op"] in ("attn", "append", "fork", "compact"):
        geo = dict(type=la.Q8_0, n_kv=c["n_kv"], head_dim=c["hd"], page_size=c["page"]) if c["kv"] == "q8_0" else {}
        if c["op"] in ("attn", "append"):
            s["cache"] = la.KvCache(s["k"], s["v"], **geo)
            s["batch"] = la.KvBatch(s["table"], s["lens"], s["start"], n_tokens=s["T"], max_new=s["max_new"])
            if c["op"] == "attn":
                s["ws"] = s["cache"].attention_workspace(s["batch"], c["n_head"])
        else:
            s["pages"] = la.KvPages([la.KvCache(k, v, **geo) for k, v in zip(s["k"], s["v"])])
            if c["op"] == "compact":
                s["ws"] = s["pages"].workspace()
    elif c["op"] == "verify":
        s["ws"] = la.verify_workspace(c["n_seq"], c["vocab"], DEV)


# ------------------------------------------------------------- operators

def run(state):
    return (_own if own else _plain)[state["c"]["op"]](state)


def _own_attn(s):
    c = s["c"]
    s["cache"].attention(s["batch"], s["q"], scale=c["hd"] ** -0.5, window=c["window"], out=s["out"], lse=s["lse"],
                         workspace=s["ws"])
    return s["out"], s["lse"]


def _own_append(s):
    s["cache"].append(s["batch"], s["kn"], s["vn"])
    return s["k"], s["v"]


def _own_fork(s):
    s["pages"].fork(s["table"], s["lens"], s["forks"])
    return s["k"].view(torch.uint8), s["v"].view(torch.uint8), s["table"], s["lens"]


def _own_compact(s):
    s["pages"].compact(s["table"], s["lens"], table_out=s["table_out"], refs=s["refs"], n_live=s["n_live"],
                       workspace=s["ws"])
    return s["k"].view(torch.uint8), s["v"].view(torch.uint8), s["table_out"], s["refs"], s["n_live"]


def _own_norm(s):
    s["la"].block_norm(s["h"], s["y"], post_weight=s["post"], post_norm=s["c"]["post"], gate=s["gate"], alpha=0.9, beta=0.8,
                       weights=s["pre"], eps=1e-6, h_out=s["h_out"], out=s["x"])
    return s["h_out"], s["x"]


def _own_verify(s):
    s["la"].verify_drafts(s["p"], s["q"], s["drafts"], s["u"], s["u_next"], n_draft=s["n_draft"], tokens=s["tokens"],
                          accepted=s["accepted"], workspace=s["ws"])
    return s["tokens"], s["accepted"]


_own = dict(attn=_own_attn, append=_own_append, fork=_own_fork, compact=_own_compact, norm=_own_norm, verify=_own_verify)


def _values(pool, c, is_v):
    """A pool's (or gathered pages') values in 32 bits: [..., n_kv, page, hd], for V [..., n_kv, hd, page]."""
    if c["kv"] != "q8_0":
        return pool.float()
    H, P, D = c["n_kv"], c["page"], c["hd"]
    by_head = pool.reshape(*pool.shape[:-1], H, -1)
    q = by_head[..., :P * D].contiguous().view(torch.int8).float()
    d = by_head[..., P * D:].contiguous().view(torch.float16).float()
    if is_v:
        return (q.reshape(*q.shape[:-1], D // 32, 32, P) * d.reshape(*d.shape[:-1], D // 32, 1, P)).flatten(-3, -2)
    d = d.reshape(*d.shape[:-1], D // 32, P).transpose(-1, -2)
    return (q.reshape(*q.shape[:-1], P, D // 32, 32) * d[..., None]).flatten(-2)


def _where(s):
    """Per sequence and new-token slot j: the token's row, its position, and whether there is one."""
    new = (s["start"][1:] - s["start"][:-1]).long()
    j = torch.arange(s["max_new"], device=DEV)
    there = j < new[:, None]
    rows = (s["start"][:-1, None].long() + j).clamp(max=s["T"] - 1)
    pos = s["lens"][:, None].long() - new[:, None] + j
    return rows, pos, there


def _plain_attn(s):
    c = s["c"]
    S, H, D, P, N = c["n_seq"], c["n_kv"], c["hd"], c["page"], s["max_new"]
    G = c["n_head"] // H
    rows, pos, there = _where(s)
    tab = s["table"].long().clamp(min=0)
    L = tab.shape[1] * P
    k = _values(s["k"][tab], c, False).permute(0, 2, 1, 3, 4).reshape(S, H, L, D)
    v = _values(s["v"][tab], c, True).permute(0, 2, 1, 4, 3).reshape(S, H, L, D)
    q = s["q"][rows].float().reshape(S, N, H, G, D).permute(0, 2, 1, 3, 4).reshape(S, H, N * G, D)
    score = torch.matmul(q, k.transpose(-1, -2).contiguous()).mul_(D ** -0.5).reshape(S, H, N, G, L)
    key = torch.arange(L, device=DEV)
    seen = (key <= pos[..., None]) & there[..., None]
    if c["window"]:
        seen &= key > pos[..., None] - c["window"]
    score.masked_fill_(~seen[:, None, :, None, :], -math.inf)
    m = score.amax(-1, keepdim=True)
    p = torch.exp(score - m.clamp(min=-3e38))
    l = p.sum(-1, keepdim=True)
    o = torch.matmul(p.reshape(S, H, N * G, L), v).reshape(S, H, N, G, D) / l
    lse = (m + torch.log(l)).squeeze(-1)
    o, lse = o.permute(0, 2, 1, 3, 4).reshape(S, N, H * G, D), lse.permute(0, 2, 1, 3).reshape(S, N, H * G)
    s["out"][rows[there]] = o[there].to(s["out"].dtype)
    s["lse"][rows[there]] = lse[there]
    return s["out"], s["lse"]


def _plain_append(s):
    rows, pos, there = _where(s)
    rows, at = rows[there], pos[there]
    seq = torch.arange(s["c"]["n_seq"], device=DEV)[:, None].expand_as(there)[there]
    page, slot = s["table"][seq, at // s["c"]["page"]].long(), at % s["c"]["page"]
    s["k"][page, :, slot] = s["kn"][rows].to(s["k"].dtype)
    s["v"][page, :, :, slot] = s["vn"][rows].to(s["v"].dtype)
    return s["k"], s["v"]


def _plain_fork(s):
    P, table, lens = s["c"]["page"], s["table"], s["lens"]
    src, dst, fresh = s["forks"].long().unbind(1)
    n = lens[src].long()
    i = torch.arange(table.shape[1], device=DEV)
    full, part = n // P, n % P > 0
    last = table[src, full].long()
    row = torch.where(i < full[:, None], table[src], -1)
    row = torch.where((i == full[:, None]) & part[:, None], fresh[:, None].to(torch.int32), row)
    table[dst], lens[dst] = row, lens[src]
    frm, to = last[part], fresh[part]
    s["k"][:, to], s["v"][:, to] = s["k"][:, frm], s["v"][:, frm]
    return s["k"].view(torch.uint8), s["v"].view(torch.uint8), table, lens


def _plain_compact(s):
    P, table, n = s["c"]["page"], s["table"], s["n_pages"]
    i = torch.arange(table.shape[1], device=DEV)
    held = (i * P < s["lens"][:, None]) & (table >= 0)
    refs = torch.bincount(table[held], minlength=n)
    page, live = torch.arange(n, device=DEV), refs > 0
    n_live = live.sum()
    frm, to = page[live & (page >= n_live)], page[~live & (page < n_live)]
    moved = page.clone()
    moved[frm] = to
    s["k"][:, to], s["v"][:, to] = s["k"][:, frm], s["v"][:, frm]
    s["table_out"].copy_(torch.where(held, moved[table.long().clamp(min=0)], -1))
    after = torch.zeros_like(refs)
    after[moved[live]] = refs[live]
    s["refs"].copy_(after)
    s["n_live"].copy_(n_live)
    return s["k"].view(torch.uint8), s["v"].view(torch.uint8), s["table_out"], s["refs"], s["n_live"]


def _rms(x):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6)


def _plain_norm(s):
    u = s["y"].float()
    if s["c"]["post"]:
        u = _rms(u) * s["post"]
    if s["gate"] is not None:
        u = u * s["gate"].float()
    h = 0.9 * s["h"].float() + 0.8 * u
    x = _rms(h)
    return h.to(s["h"].dtype), [(x * w).to(s["h"].dtype) for w in s["pre"]]


def _plain_verify(s):
    p, d, n = s["p"], s["drafts"].long(), s["n_draft"].long()
    S, N, V = s["c"]["n_seq"], s["c"]["drafts"], s["c"]["vocab"]
    px = p[:, :N].gather(2, d[..., None]).squeeze(2).double()
    qx = torch.ones_like(px) if s["q"] is None else s["q"].gather(2, d[..., None]).squeeze(2).double()
    i = torch.arange(N, device=DEV)
    ok = (s["u"].double() * qx < px) & (i < n[:, None])
    a = ok.long().cumprod(1).sum(1)
    seq, at = torch.arange(S, device=DEV), a.clamp(max=N - 1)
    target = p[seq, a].double()
    if s["q"] is None:
        draft = torch.zeros_like(target).scatter_(1, d[seq, at][:, None], 1.0)
    else:
        draft = s["q"][seq, at].double()
    rest = (target - draft).clamp(min=0)
    whole = ((a == n) | (rest.sum(1) == 0))[:, None]
    cum = torch.where(whole, target, rest).cumsum(1)
    nxt = (cum <= s["u_next"].double()[:, None] * cum[:, -1:]).sum(1).clamp(max=V - 1)
    slot = torch.arange(N + 1, device=DEV)
    padded = torch.cat([d, d[:, :1]], 1)
    tokens = torch.where(slot < a[:, None], padded, torch.where(slot == a[:, None], nxt[:, None], -1))
    return tokens.to(torch.int32), a.to(torch.int32)


_plain = dict(attn=_plain_attn, append=_plain_append, fork=_plain_fork, compact=_plain_compact, norm=_plain_norm,
              verify=_plain_verify)


# ------------------------------------------------------------------ work

def work(case):
    c, op = case, case["op"]
    if op == "attn":
        # lengths are spread evenly over their logarithm
        lo, hi = c["min_len"], c["max_len"]
        mean = hi if lo >= hi else (hi - lo) / math.log(hi / lo)
        keys = hi + (c["n_seq"] - 1) * mean
        if c["window"]:
            keys = min(keys, c["n_seq"] * (c["window"] + c["new"] - 1))
        new = c["new"] if c["even"] else (1 + c["new"]) / 2
        return {"bytes": 2 * keys * c["n_kv"] * c["hd"] * SIZE[c["kv"]]
                + 2 * c["n_seq"] * new * c["n_head"] * c["hd"] * SIZE[c["io"]],
                "flops": 4 * keys * new * c["n_head"] * c["hd"]}
    if op == "append":
        new = c["new"] if c["even"] else (1 + c["new"]) / 2
        return {"bytes": 2 * c["n_seq"] * new * c["n_kv"] * c["hd"] * (SIZE[c["io"]] + SIZE[c["kv"]]), "flops": 0}
    if op in ("fork", "compact"):
        page = 2 * c["layers"] * c["n_kv"] * c["page"] * c["hd"] * SIZE[c["kv"]]
        if op == "fork":
            return {"bytes": 2 * page * c["forks"], "flops": 0}
        # a half of the pages in use stay, and about a half of those lie behind the new end
        used = min(c["n_pages"], c["n_seq"] * (c["max_len"] / 2 / c["page"] + 0.5))
        live = used / 2
        return {"bytes": 2 * page * live * (1 - live / c["n_pages"]) + 8 * used, "flops": 0}
    if op == "norm":
        full = 2 + 1 + c["outs"] + (c["gate"] == "full")
        return {"bytes": full * c["T"] * c["d"] * SIZE[c["io"]] + 4 * c["d"] * (c["outs"] + c["post"]),
                "flops": c["T"] * c["d"] * (8 + c["outs"])}
    # a target row for every sequence, and a draft row where a draft was refused
    rows = 1 if c["onehot"] else 1.5
    return {"bytes": c["n_seq"] * rows * c["vocab"] * SIZE[c["io"]], "flops": 2 * c["n_seq"] * c["vocab"]}


# ----------------------------------------------------------------- exact

def exact(case, seed):
    c = case
    global own
    was, own = own, False
    try:
        s = prepare(c, seed)
    finally:
        own = was
    if c["op"] == "attn":
        return _exact_attn(c, s)
    if c["op"] == "append":
        k, v = s["k"].double(), s["v"].double()
        table, lens, start = s["table"].tolist(), s["lens"].tolist(), s["start"].tolist()
        for i, n in enumerate(lens):
            for r in range(start[i], start[i + 1]):
                at = n - (start[i + 1] - r)
                k[table[i][at // c["page"]], :, at % c["page"]] = s["kn"][r].double()
                v[table[i][at // c["page"]], :, :, at % c["page"]] = s["vn"][r].double()
        return k, v
    if c["op"] == "norm":
        y, h = s["y"].double(), s["h"].double()
        norm = lambda z: z / ((z * z).sum(1, keepdim=True) / c["d"] + 1e-6).sqrt()
        u = norm(y) * s["post"].double() if c["post"] else y
        h = 0.9 * h + 0.8 * (u if s["gate"] is None else s["gate"].double() * u)
        return h, [norm(h) * w.double() for w in s["pre"]]
    return None  # bytes, tables and tokens: whole numbers


def _exact_attn(c, s):
    P, D, G = c["page"], c["hd"], c["n_head"] // c["n_kv"]
    out = torch.zeros(s["T"], c["n_head"], D, dtype=torch.float64, device=DEV)
    lse = torch.zeros(s["T"], c["n_head"], dtype=torch.float64, device=DEV)
    start = s["start"].tolist()
    for i, n in enumerate(s["lens"].tolist()):
        pages = s["table"][i, :-(-n // P)].long()
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
            for r in range(start[i], start[i + 1]):
                end = n - (start[i + 1] - r) + 1
                begin = max(0, end - c["window"]) if c["window"] else 0
                q = s["q"][r, h * G:(h + 1) * G].double()
                z = (q @ k[begin:end].T) / math.sqrt(D)
                top = z.max(1, keepdim=True).values
                e = (z - top).exp()
                out[r, h * G:(h + 1) * G] = (e @ v[begin:end]) / e.sum(1, keepdim=True)
                lse[r, h * G:(h + 1) * G] = top[:, 0] + e.sum(1).log()
    return out, lse
