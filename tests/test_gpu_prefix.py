"""Attention of sequences that share a prefix (llapis_kv_prefix_attention) on the GPU against
the plain 64-bit form of attention (step_ref.py), which reads every sequence's own row of the page table.

The bound is step_ref.attention's.  What the prefix adds to its error: parts are joined by their
maxima in base 2, whose difference is rounded once, 2^-24 (|s| + |m|), and 2^x of it, 2^-23: within the bound's
2^-22 (|s| + |m|) and its 2^-21."""
import math

import pytest
import torch

import llapis_amd as la
import step_ref as ref
from test_gpu_step import i32, poisoned

pytestmark = pytest.mark.gpu

DT = ref.DT


class Shared:
    """Groups of sequences on the same first pages, every other place NaN.  groups: (shared
    tokens, [(own tokens, new ones among them)]) each; a lone sequence is a group of nothing shared."""

    def __init__(self, gpu, seed, tag, D, H, P, groups, io, before=0, spare=3):
        g = torch.Generator().manual_seed(seed)
        self.P, self.io = P, io
        self.lens, self.new, first, rows = [], [], [before], []
        need = sum(-(-n // P) + sum(-(-t // P) for t, _ in m) for n, m in groups) + before
        n_pages = need + spare
        order = torch.randperm(n_pages, generator=g).tolist()
        for _ in range(before):
            self.lens.append(P // 2)
            self.new.append(1)
            rows.append([order.pop()])
        for n, members in groups:
            assert n % P == 0
            head = [order.pop() for _ in range(n // P)]
            for t, k in members:
                rows.append(head + [order.pop() for _ in range(-(-t // P))])
                self.lens.append(n + t)
                self.new.append(k)
            first.append(first[-1] + len(members))
        width = max(len(r) for r in rows) + 1
        self.table = [r + [-1] * (width - len(r)) for r in rows]
        self.cache = poisoned(la.KvCache.empty(n_pages, P, H, D, tag, gpu))
        self.tb = i32(self.table, gpu)
        kv = lambda n: [torch.randn(max(n, 1), H, D, generator=g).to(gpu) for _ in range(2)]
        # whole sequences as prompts, one of each group first: the others' prefix is the same
        lead = {}
        for s, (n, i) in enumerate(zip(self.lens, range(len(self.lens)))):
            g_i = next((j for j in range(len(groups)) if first[j] <= s < first[j + 1]), None)
            skip = 0
            if g_i is not None:
                skip = groups[g_i][0] if g_i in lead else 0
                if n >= groups[g_i][0]:
                    lead.setdefault(g_i, s)
            new = n - skip
            if new > 0:
                b = la.KvBatch(self.tb[s:s + 1], i32([n], gpu), i32([0, new], gpu), n_tokens=new, max_new=new)
                self.cache.append(b, *kv(new))
        self.start = [0]
        for k in self.new:
            self.start.append(self.start[-1] + k)
        self.T = self.start[-1]
        self.groups, self.prefix = i32(first, gpu), i32([n for n, _ in groups], gpu)
        self.first, self.shared = first, [n for n, _ in groups]
        self.batch = la.KvBatch(self.tb, i32(self.lens, gpu), i32(self.start, gpu), n_tokens=self.T, max_new=max(max(self.new), 1))

    def queries(self, seed, n_head, factor=1.5):
        g = torch.Generator().manual_seed(seed)
        return (factor * torch.randn(max(self.T, 1), n_head, self.cache.head_dim, generator=g)).to(DT[self.io])

    def check(self, q, scale=None, groups=None, prefix=None, table=None):
        dev = self.cache.device
        scale = self.cache.head_dim ** -0.5 if scale is None else scale
        lse = torch.full(q.shape[:2], 7.0, device=dev)
        out = torch.full((q.shape[0], q.shape[1] + 1, q.shape[2]), 5.0, dtype=q.dtype, device=dev)[:, :q.shape[1]]
        self.cache.prefix_attention(self.batch, q.to(dev), self.groups if groups is None else groups,
                                    self.prefix if prefix is None else prefix, scale=scale, out=out, lse=lse)
        want, want_lse, tol = ref.attention(self.cache, self.table if table is None else table, self.lens, self.start, q, scale)
        out, lse = out.cpu(), lse.cpu()
        off = (out.double() - want).abs()
        assert not torch.isnan(out[:self.T]).any()
        assert (off <= tol)[:self.T].all(), f"off by {float((off / (tol + 1e-30))[:self.T].max()):.3g} of the bound"
        empty = want_lse == -math.inf
        assert (lse[empty] == -math.inf).all() and (out[empty] == 0).all()
        near = (lse.double() - want_lse).abs()[~empty]
        assert (near <= 2e-5 + 2 ** -22 * want_lse[~empty].abs()).all(), float(near.max())
        return out


SHAPES = [(64, 16), (96, 32), (128, 64), (192, 128), (256, 256), (512, 64)]


@pytest.mark.parametrize("D,P", SHAPES)
@pytest.mark.parametrize("io", [la.F32, la.F16, la.BF16])
@pytest.mark.parametrize("tag", [la.F16, la.BF16, la.Q8_0])
def test_types(gpu, tag, io, D, P):
    """Every cache type, query type and head size: two groups, a sequence before them, several tokens."""
    n = max(P, 64)
    s = Shared(gpu, D, tag, D, 2, P, [(5 * n, [(3, 1), (70, 3), (1, 1), (P, 2)]), (2 * n, [(40, 1), (9, 4)])], io, before=1)
    s.check(s.queries(D + 1, 6))


@pytest.mark.parametrize("n_seq,group,H", [(1, 1, 1), (2, 1, 3), (5, 3, 2), (17, 4, 1), (40, 8, 2), (70, 5, 1)])
@pytest.mark.parametrize("io,tag,D", [(la.F32, la.F16, 64), (la.BF16, la.BF16, 128), (la.F32, la.BF16, 128), (la.F16, la.Q8_0, 256)])
def test_rows(gpu, n_seq, group, H, io, tag, D):
    """Query rows from one to several tiles of a group, tiles of all, some and one of a workgroup's waves."""
    s = Shared(gpu, n_seq, tag, D, H, 16, [(320, [(1 + (7 * i) % 50, 1 + (i % 2 if (7 * i) % 50 else 0)) for i in range(n_seq)])], io)
    s.check(s.queries(4, group * H))


@pytest.mark.parametrize("n", [64, 128, 192, 1024, 2048, 6400])
def test_lengths(gpu, n):
    """Prefixes of one unit and of many, in runs that end inside them."""
    s = Shared(gpu, n, la.F16, 64, 1, 64, [(n, [(5, 1), (300, 2)]), (64, [(1, 1)])], la.F32)
    s.check(s.queries(n, 3))


@pytest.mark.parametrize("given", [-5, 0, 1, 63, 64, 100, 319, 320, 330, 10 ** 9])
def test_cut(gpu, given):
    """A prefix that is no multiple of a unit, none, or longer than what the sequences share or hold: it
    is cut to what each had before its new tokens."""
    s = Shared(gpu, 3, la.F16, 64, 2, 16, [(320, [(1, 1), (4, 4), (90, 1)])], la.F32)
    q = s.queries(5, 4)
    if given > 320:
        # longer than the shared pages' tokens, but not than the shortest sequence's own before its new ones
        assert min(n - k for n, k in zip(s.lens, s.new)) == 320
    s.check(q, prefix=i32([given], gpu))


def test_members(gpu):
    """A group's first sequence ended, members without new tokens, a member shorter than the
    prefix, groups of one and of none, sequences in no group."""
    s = Shared(gpu, 6, la.BF16, 128, 2, 32, [(256, [(0, 0), (40, 0), (3, 1), (65, 2)]), (128, [(20, 1)]), (64, [])], la.BF16, before=2)
    s.lens[2] = 0
    s.batch.lens[2] = 0
    s.tb[2] = 12345
    s.table[2] = [12345] * len(s.table[2])
    q = s.queries(7, 8)
    s.check(q)
    # a member with new tokens that has less than the others share: the prefix is cut for all
    s.lens[4] = s.lens[4] - 200
    s.batch.lens[4] = s.lens[4]
    s.check(q)
    s.lens[4] = 1
    s.batch.lens[4] = 1
    s.check(q)
    s.lens[4] = 0                      # more new tokens than tokens
    s.batch.lens[4] = 0
    s.check(q)
    # groups that leave all sequences out, and no groups at all
    for groups, prefix in (([6, 6], [128]), ([0, 0], [128]), ([2], [])):
        s.check(q, groups=i32(groups, gpu), prefix=i32(prefix, gpu))


def test_holes(gpu):
    """Entries without a page, in the prefix and behind it: their keys are masked."""
    s = Shared(gpu, 8, la.F16, 64, 1, 16, [(256, [(30, 1), (50, 2)])], la.F32)
    for i, pg in ((3, -1), (7, 10 ** 6), (8, -7)):
        for r in range(2):
            s.tb[r, i] = pg
            s.table[r][i] = pg
    s.tb[1, 17] = -1
    s.table[1][17] = -1
    q = s.queries(9, 2)
    s.check(q)
    s.check(q, scale=0.0)
    s.check(q, scale=-1e-38)
    for r in range(2):
        s.tb[r, :16] = -1
        s.table[r][:16] = [-1] * 16
    s.check(q)
    # nothing left to see
    s.tb[:] = -1
    s.table = [[-1] * len(r) for r in s.table]
    assert (s.check(q) == 0).all()


@pytest.mark.parametrize("tag,D", [(la.F16, 128), (la.BF16, 128), (la.Q8_0, 64), (la.F16, 512), (la.Q8_0, 512)])
def test_hidden_non_finite(gpu, tag, D):
    """A later draft's NaN key and value stay out of the rows that do not see it; one in the prefix is in every row."""
    P, N = 16, 4
    s = Shared(gpu, 10, tag, D, 1, P, [(128, [(20, N), (7, 1)])], la.F32)
    q = s.queries(11, 2)
    clean = s.check(q)

    def poison(row, at):
        pg, slot = s.table[row][at // P], at % P
        for t in (s.cache.k, s.cache.v):
            if tag == la.Q8_0:
                t[pg].view(torch.float16)[P * D // 2:].view(D // 32, P)[:, slot] = float("nan")
            elif t is s.cache.k:
                t[pg, 0, slot] = float("nan")
            else:
                t[pg, 0, :, slot] = float("nan")

    run = lambda: s.cache.prefix_attention(s.batch, q.to(gpu), s.groups, s.prefix).cpu()
    poison(0, s.lens[0] - 2)
    got = run()
    assert torch.equal(got[[0, 1, 4]], clean[[0, 1, 4]]) and torch.isnan(got[2:4]).all()
    poison(0, 70)
    assert torch.isnan(run()).all()


def test_scores(gpu):
    """Scores all equal, far apart, of either sign of scale; the prefix far above the rest and far below it."""
    s = Shared(gpu, 12, la.F16, 128, 1, 64, [(640, [(30, 1), (200, 2)])], la.F32)
    q = s.queries(13, 4)
    s.check(torch.zeros_like(q))
    s.check(q * 300)
    s.check(q, scale=-0.3)
    s.check(q * 1e-6)
    for size, where in ((40.0, slice(0, 10)), (0.0, slice(0, 10))):
        held = s.cache.k.clone()
        s.cache.k[torch.tensor(s.table[0][where])] *= size
        s.check(q)
        s.cache.k.copy_(held)


@pytest.mark.parametrize("size", [1e-9, 3e4])
def test_query_range(gpu, size):
    s = Shared(gpu, 14, la.F16, 64, 1, 16, [(128, [(30, 1)])], la.F32)
    s.check(s.queries(15, 2) * size, scale=0.125 / size)


def test_many(gpu):
    """As many groups as a call takes, and one more; hundreds of sequences of one group."""
    s = Shared(gpu, 16, la.F16, 64, 1, 16, [(64, [(1 + i % 5, 1)]) for i in range(256)], la.F16)
    s.check(s.queries(17, 1))
    with pytest.raises(ValueError, match="prefix_attention"):
        s.cache.prefix_attention(s.batch, s.queries(17, 1).to(gpu), torch.zeros(258, dtype=torch.int32, device=gpu),
                                 torch.zeros(257, dtype=torch.int32, device=gpu))
    s = Shared(gpu, 18, la.BF16, 64, 1, 16, [(192, [(1 + i % 7, 1) for i in range(600)])], la.BF16)
    s.check(s.queries(19, 2))


def test_one_row_each(gpu):
    """A batch without row starts."""
    s = Shared(gpu, 20, la.F16, 64, 2, 16, [(128, [(5, 1), (33, 1), (2, 1)])], la.F32)
    q = s.queries(21, 4).to(gpu)
    b = la.KvBatch(s.tb, s.batch.lens)
    assert torch.equal(s.cache.prefix_attention(b, q, s.groups, s.prefix), s.cache.prefix_attention(s.batch, q, s.groups, s.prefix))


def test_out_of_order(gpu):
    """Groups and row starts that are in no order, or past the batch: results are not defined, memory is safe."""
    s = Shared(gpu, 22, la.F16, 64, 1, 16, [(128, [(5, 1), (33, 2)]), (64, [(2, 1)])], la.F32)
    q = s.queries(23, 4).to(gpu)
    out = torch.full((s.T + 2, 4, 64), 5.0, device=gpu)
    for groups in ([3, 0, 2], [0, 99, 3], [-7, 2, 1], [2 ** 31 - 1, -2 ** 31, 5]):
        s.cache.prefix_attention(s.batch, q, i32(groups, gpu), s.prefix, out=out)
    for start in ([4, 0, 2, 1], [0, 2 ** 31 - 1, -5, 3], [9, 9, 9, 9]):
        b = la.KvBatch(s.tb, s.batch.lens, i32(start, gpu), n_tokens=s.T, max_new=2)
        s.cache.prefix_attention(b, q, s.groups, s.prefix, out=out)
    assert (out[s.T:] == 5).all()
    s.check(q.cpu())


def test_beyond_32_bits(gpu):
    """Pages past 4 GiB of a pool (strides apart, so that little memory is written)."""
    D, H, P = 64, 1, 16
    s = Shared(gpu, 27, la.F16, D, H, P, [(64, [(5, 1), (20, 2)])], la.F32, spare=0)
    n_pages, gap = s.cache.n_pages, 1 << 28                       # values between pages: 512 MiB
    pool = [torch.empty((n_pages - 1) * gap + H * P * D, dtype=torch.float16, device=gpu) for _ in range(2)]
    k = pool[0].as_strided((n_pages, H, P, D), (gap, P * D, D, 1))
    v = pool[1].as_strided((n_pages, H, D, P), (gap, P * D, P, 1))
    for t, src in ((k, s.cache.k), (v, s.cache.v)):
        for i in range(n_pages):
            t[i] = src[i]
    q = s.queries(28, 2).to(gpu)
    assert torch.equal(la.KvCache(k, v).prefix_attention(s.batch, q, s.groups, s.prefix), s.cache.prefix_attention(s.batch, q, s.groups, s.prefix))
    del pool, k, v
    torch.cuda.empty_cache()


def test_repeats_and_graphs(gpu):
    """Two captured graphs with one workspace, replayed in turn as the lengths and the prefix
    change, equal to eager calls bit for bit; a call on another stream."""
    s = [Shared(gpu, 24 + i, la.BF16, 128, 2, 16, [(640 * (1 + i), [(90, 1), (200, 2), (5, 1)])], la.BF16) for i in range(2)]
    qs = [x.queries(26, 8).to(gpu) for x in s]
    ws = max((x.cache.prefix_workspace(x.batch, 8, 1) for x in s), key=lambda t: t.numel())
    outs, graphs = [], []
    for x, q in zip(s, qs):
        out = x.cache.prefix_attention(x.batch, q, x.groups, x.prefix, workspace=ws)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            x.cache.prefix_attention(x.batch, q, x.groups, x.prefix, out=out, workspace=ws)
        outs.append(out)
        graphs.append(g)
    for step in range(4):
        for x, q, out, g in zip(s, qs, outs, graphs):
            ws.random_(0, 255)
            out.fill_(float("nan"))
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, x.cache.prefix_attention(x.batch, q, x.groups, x.prefix))
            x.prefix.sub_(100)
            x.batch.lens.sub_(torch.tensor([20, 3, 0], dtype=torch.int32, device=gpu))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = s[0].cache.prefix_attention(s[0].batch, qs[0], s[0].groups, s[0].prefix)
    side.synchronize()
    assert torch.equal(got, s[0].cache.prefix_attention(s[0].batch, qs[0], s[0].groups, s[0].prefix))


def test_refusals(gpu):
    s = Shared(gpu, 30, la.F16, 64, 2, 16, [(64, [(5, 1)])], la.F32)
    q = s.queries(31, 4).to(gpu)
    call = lambda **kw: s.cache.prefix_attention(**{**dict(batch=s.batch, q=q, groups=s.groups, prefix=s.prefix), **kw})
    for bad, what in ((dict(groups=s.groups[:1]), "groups"), (dict(groups=s.groups.long()), "groups"), (dict(prefix=s.prefix.float()), "prefix"),
                      (dict(prefix=s.prefix[0]), "prefix"), (dict(q=q[:, :3]), "unsupported"), (dict(q=q.double()), "float32"),
                      (dict(lse=torch.zeros(1, 3, device=gpu)), "lse"), (dict(out=q.half()), "out"), (dict(groups=s.groups.cpu()), "groups")):
        with pytest.raises(ValueError, match=what):
            call(**bad)
    with pytest.raises(la.LlapisError, match="workspace"):
        call(workspace=torch.empty(64, dtype=torch.uint8, device=gpu))
    with pytest.raises(la.LlapisError, match="out may not be q"):
        call(out=q)


def past_the_table(gpu, tag, io, D, P, max_new=None, huge=False):
    """A batch whose table ends nine pages behind the prefix, among and before its sequences' ends"""
    n, own = max(P, 64) * 3, 9 * P
    members = [(own + over, k) for over, k in ((-5, 1), (0, 2), (1, 3), (P, 1), (129, 4), (2500, 2))]
    s = Shared(gpu, 40 + D, tag, D, 2, P, [(n, members), (n + max(P, 64), [(own - max(P, 64) + 1, 1), (own + 700, 3)])], io, before=1)
    width = (n + own) // P
    s.table = [r[:width] for r in s.table]
    if huge:
        for i in (3, 6):
            s.lens[i] = s.batch.lens[i] = 2 ** 31 - 1
    s.batch = la.KvBatch(s.tb[:, :width], s.batch.lens, s.batch.new_start, n_tokens=s.T, max_new=max_new or 4)
    # what an earlier call may have left: ids of pages that there are
    room = s.cache.prefix_workspace
    s.cache.prefix_workspace = lambda *a: room(*a).view(torch.int32).random_(0, s.cache.n_pages).view(torch.uint8)
    return s


@pytest.mark.parametrize("huge", [False, True])
@pytest.mark.parametrize("tag,io,D,P", [(la.F16, la.F32, 64, 16), (la.BF16, la.BF16, 128, 16), (la.Q8_0, la.F16, 256, 64), (la.F16, la.F32, 512, 128)])
def test_lengths_past_the_table(gpu, tag, io, D, P, huge):
    """Keys past max_pages * page_size are not attended, whatever the workspace held: lengths of a token, a
    page, a unit and thousands of tokens past it, and the largest that there is."""
    s = past_the_table(gpu, tag, io, D, P, huge=huge)
    q = s.queries(41, 4)
    first = s.check(q)
    assert torch.equal(s.check(q)[:s.T], first[:s.T])


def test_cut_rows_past_the_table(gpu):
    """... with new tokens past max_new, which are left out, the last ones of each sequence."""
    s = past_the_table(gpu, la.F16, la.F32, 64, 16, max_new=2)
    q = s.queries(42, 4)
    out = torch.full(q.shape, 5.0, device=gpu)
    s.cache.prefix_attention(s.batch, q.to(gpu), s.groups, s.prefix, out=out)
    want, _, tol = ref.attention(s.cache, s.table, s.lens, s.start, q, 64 ** -0.5)
    for i, k in enumerate(s.new):
        rows = range(s.start[i], s.start[i + 1])
        for r in rows[:2]:
            assert ((out[r].cpu().double() - want[r]).abs() <= tol[r]).all(), (i, r)
        for r in rows[2:]:
            assert (out[r] == 5).all(), (i, r)


def made(gpu, tag, heads, keys, values, own):
    """Two sequences of one kv head of 64 values behind `heads` tokens of keys[:heads]; behind these each has the `own`
    tokens that follow.  keys [heads + own]: a key's first two values; values: its V's first."""
    P, n = 16, heads + own
    held, rest = -(-heads // P), -(-own // P)
    table = [list(range(held)) + [held + rest * i + j for j in range(rest)] for i in range(2)]
    cache = poisoned(la.KvCache.empty(held + 2 * rest, P, 1, 64, tag, gpu))
    k, v = torch.zeros(n, 1, 64), torch.zeros(n, 1, 64)
    k[:, 0, :2], v[:, 0, 0] = keys, values
    for row in table:
        cache.append(la.KvBatch(i32([row], gpu), i32([n], gpu), i32([0, n], gpu), n_tokens=n, max_new=n), k.to(gpu), v.to(gpu))
    batch = la.KvBatch(i32(table, gpu), i32([n, n], gpu))
    return cache, batch, i32([0, 2], gpu), i32([heads], gpu)


@pytest.mark.parametrize("tag", [la.F16, la.BF16])
@pytest.mark.parametrize("far", [0, 416, 2912, 3616])
def test_parts_join_exactly_far_from_zero(gpu, tag, far):
    """Scores that are whole numbers in base 2, about `far`, in the prefix and behind it: every weight is a power of 2, so
    that the result is off by what fp32 sums are, whatever the scores' size.

    The scale is fp32's ln 2, which times fp32's log2 e is 1: scores, maxima and their differences are exact.
    2^x of a whole number is off by 2^-23, a sum of n weights in fp32 by (n / 32 + 40) 2^-24 (the numerator and
    the sum, of values up to 1), the quotient by 2^-23."""
    g = torch.Generator().manual_seed(far)
    heads, own = 128, 100
    n = heads + own
    near = torch.randint(0, 6, (n,), generator=g)
    keys = torch.stack([torch.full((n,), far / 64.0), near.float()], 1)
    values = torch.randint(0, 65, (n,), generator=g) / 64.0
    values[:heads] *= -1                                  # either part's weight shows
    cache, batch, groups, prefix = made(gpu, tag, heads, keys, values, own)
    q = torch.zeros(2, 1, 64, device=gpu)
    q[:, 0, 0], q[:, 0, 1] = 64, 1
    lse = torch.empty(2, 1, device=gpu)
    ln2 = float(torch.tensor(math.log(2), dtype=torch.float32))
    out = cache.prefix_attention(batch, q, groups, prefix, scale=ln2, lse=lse)
    w = 2.0 ** near.double()
    want = float((w * values).sum() / w.sum())
    tol = 2 * (n / 32 + 40) * 2 ** -24 + 2 * 2 ** -23 + 2 ** -23
    off = (out[:, 0, 0].cpu().double() - want).abs()
    assert (off <= tol).all(), float((off / tol).max())
    assert (out[:, 0, 1:] == 0).all()
    # the logarithm: the sum's error, log2's and its product's roundings
    want = math.log(2) * (far + math.log2(float(w.sum())))
    assert (lse.cpu().double() - want).abs().max() <= tol + 3 * 2 ** -24 * max(want, 16)


def test_probabilities_keep_17_bits_over_bf16_pages(gpu):
    """Two kinds of keys, of weight 1 and x = e^-0.6809, whose two BF16 parts are off by 2^-20.4 of it if both are rounded and by
    2^-16.05 if the first is cut off.  Their values are 1 and -1 and their sums nearly the same, so that the result is off by half of
    what x is: by 2^-18 and by what scores (2^-22) and 2^x (2^-22) add, with fp16's half step."""
    heads, own, scale = 192, 1, 2789 / 4096
    # (both kinds in every unit: its largest weight is 1)
    kind = torch.tensor([0, 1, 1]).repeat(heads // 3 + 1)[:heads + own]
    kind[190:] = 2
    keys = torch.stack([torch.zeros(heads + own), torch.tensor([0.0, -1.0, -60.0])[kind]], 1)
    values = torch.tensor([1.0, -1.0, 0.0])[kind]
    cache, batch, groups, prefix = made(gpu, la.BF16, heads, keys, values, own)
    q = torch.zeros(2, 1, 64, dtype=torch.float16, device=gpu)
    q[:, 0, 1] = 1
    out = cache.prefix_attention(batch, q, groups, prefix, scale=scale)
    x = math.exp(-scale)
    n = [int((kind == i).sum()) for i in range(2)]
    want = (n[0] - n[1] * x) / (n[0] + n[1] * x)
    off = (out[:, 0, 0].cpu().double() - want).abs().max()
    assert off <= 2 ** -18 + 2 * 2 ** -22 + 2 ** -11 * abs(want), float(off) * 2 ** 18
