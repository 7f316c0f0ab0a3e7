"""The operators of llapis_step.h on the GPU against their plain 64-bit forms
(step_ref.py): the paged cache's append, attention and page operations, the
block norms, the verification of drafts, and a run of them together."""
import math

import pytest
import torch

import llapis_amd as la
import step_ref as ref

pytestmark = pytest.mark.gpu

DT = ref.DT


def i32(v, dev):
    return torch.tensor(v, dtype=torch.int32).to(dev)


def poisoned(cache):
    """Fill the pools with NaN (0xFF bytes are NaN in every 16-bit type, scales among them)."""
    for t in (cache.k, cache.v):
        t.view(torch.uint8).fill_(0xFF) if t.dtype == torch.uint8 else t.fill_(float("nan"))
    return cache


class Filled:
    """A cache whose sequences' tokens were appended, every other place NaN."""

    def __init__(self, gpu, seed, tag, D, H, P, lens, new, io, holes=(), spare=3, width=None, x_io=la.F32):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.new = lens, new
        need = [-(-max(n, 0) // P) for n in lens]
        n_pages = max(sum(need), 1) + spare
        order = torch.randperm(n_pages, generator=g).tolist()
        width = width or max(1, max(need, default=1))
        self.table = [[order.pop() if i < k else -1 for i in range(width)] for k in need]
        for s, i, pg in holes:
            self.table[s][i] = pg
        self.cache = poisoned(la.KvCache.empty(n_pages, P, H, D, tag, gpu))
        self.tb = i32(self.table, gpu).reshape(len(lens), width)
        # every token in one call, as a prompt
        tot = [0]
        for n in lens:
            tot.append(tot[-1] + max(n, 0))
        self.kv = [torch.randn(max(tot[-1], 1), H, D, generator=g).to(DT[x_io]) for _ in range(2)]
        self.tot = tot
        b = la.KvBatch(self.tb, i32(lens, gpu), i32(tot, gpu), n_tokens=tot[-1], max_new=max(max(lens), 1))
        self.cache.append(b, *(t.to(gpu) for t in self.kv))
        self.start = [0]
        for n in new:
            self.start.append(self.start[-1] + n)
        self.T = self.start[-1]
        self.batch = la.KvBatch(self.tb, i32(lens, gpu), i32(self.start, gpu), n_tokens=self.T, max_new=max(max(new), 1))
        self.io = io

    def queries(self, seed, n_head, factor=1.5):
        g = torch.Generator().manual_seed(seed)
        return (factor * torch.randn(max(self.T, 1), n_head, self.cache.head_dim, generator=g)).to(DT[self.io])

    def check(self, q, window=0, scale=None):
        dev = self.cache.device
        scale = self.cache.head_dim ** -0.5 if scale is None else scale
        lse = torch.full(q.shape[:2], 7.0, device=dev)
        out = torch.full(q.shape, 5.0, dtype=q.dtype, device=dev)
        self.cache.attention(self.batch, q.to(dev), scale=scale, window=window, out=out, lse=lse)
        want, want_lse, tol = ref.attention(self.cache, self.table, self.lens, self.start, q, scale, window)
        out, lse = out.cpu(), lse.cpu()
        off = (out.double() - want).abs()
        assert not torch.isnan(out[:self.T]).any()
        assert (off <= tol)[:self.T].all(), f"off by {float((off / (tol + 1e-30))[:self.T].max()):.3g} of the bound"
        empty = want_lse == -math.inf
        assert (lse[empty] == -math.inf).all() and (out[empty] == 0).all()
        # the sum's relative error is the weights'; the logarithm's own rounding and its scaling add 2^-22 of itself
        near = (lse.double() - want_lse).abs()[~empty]
        assert (near <= 2e-5 + 2 ** -22 * want_lse[~empty].abs()).all(), float(near.max())
        return out


# -------------------------------------------------------------- append

@pytest.mark.parametrize("P,D", [(16, 64), (32, 96), (64, 128), (128, 192), (256, 256), (64, 512)])
@pytest.mark.parametrize("x_io", [la.F32, la.F16, la.BF16])
@pytest.mark.parametrize("tag", [la.F16, la.BF16, la.Q8_0])
def test_append(gpu, tag, x_io, P, D):
    """Every appended value bit for bit, and nothing else written."""
    H, lens = 2, [1, 37, 0, P, 2 * P + 9]
    f = Filled(gpu, 11 + D, tag, D, H, P, lens, [0] * 5, la.F32, x_io=x_io)
    kv = [t.to(torch.float32) for t in f.kv]
    want = [torch.full((f.cache.n_pages, H, P, D), float("nan")) for _ in range(2)]
    if tag == la.Q8_0:
        raw = [torch.full((f.cache.n_pages, H, f.cache.page_bytes // H), 0xFF, dtype=torch.uint8) for _ in range(2)]
    for s, n in enumerate(lens):
        for t in range(n):
            pg, slot = f.table[s][t // P], t % P
            for w in range(2):
                x = kv[w][f.tot[s] + t]
                if tag == la.Q8_0:
                    q, d = ref.pack_cache(tag, x)
                    vals = raw[w][pg, :, :P * D].view(torch.int8).reshape(H, *((P, D), (D, P))[w])
                    sc = raw[w][pg, :, P * D:].view(torch.float16).reshape(H, D // 32, P)
                    if w:
                        vals[:, :, slot] = q
                    else:
                        vals[:, slot] = q
                    sc[:, :, slot] = d
                    raw[w][pg, :, :P * D] = vals.reshape(H, -1).view(torch.uint8)
                    raw[w][pg, :, P * D:] = sc.reshape(H, -1).view(torch.uint8)
                else:
                    want[w][pg, :, slot] = ref.pack_cache(tag, x).float()
    for w, t in enumerate((f.cache.k, f.cache.v)):
        got = t.cpu()
        if tag == la.Q8_0:
            assert torch.equal(got.reshape(raw[w].shape), raw[w])
        else:
            exp = want[w].transpose(2, 3) if w else want[w]
            assert torch.equal(torch.isnan(got), torch.isnan(exp))
            assert torch.equal(torch.nan_to_num(got.float()), torch.nan_to_num(exp))


def test_append_places(gpu):
    """Rows of a fused projection, holes in the table, a table that ends before
    the sequence, rows past n_tokens: what has no place is dropped."""
    D, H, P = 64, 2, 16
    c = la.KvCache.empty(6, P, H, D, la.F16, gpu)
    c.k.zero_(), c.v.zero_()
    qkv = torch.randn(40, 4 * H, D, device=gpu).half()
    k, v = qkv[:, H:2 * H], qkv[:, 2 * H:3 * H]
    table = i32([[2, 99], [0, 4], [-1, 1]], gpu)
    lens, start = i32([20, 40, 18], gpu), i32([0, 8, 16, 24], gpu)
    c.append(la.KvBatch(table, lens, start, n_tokens=22, max_new=8), k, v)
    want_k, want_v = torch.zeros(6, H, P, D).half(), torch.zeros(6, H, P, D).half()
    kc, vc = k.cpu(), v.cpu()
    for s, (n, row) in enumerate(zip((20, 40, 18), ((2, 99), (0, 4), (-1, 1)))):
        for j in range(8):
            r, t = 8 * s + j, n - 8 + j
            if r >= 22 or t >= 2 * P or not 0 <= row[t // P] < 6:
                continue
            want_k[row[t // P], :, t % P], want_v[row[t // P], :, t % P] = kc[r], vc[r]
    assert torch.equal(c.k.cpu(), want_k) and torch.equal(c.v.cpu().transpose(2, 3), want_v)
    assert want_k[2].abs().sum() > 0 and want_k[4].abs().sum() == 0


def test_append_one_each(gpu):
    """new_start None: row s is sequence s's last token; a sequence of no tokens takes none."""
    D, H, P = 128, 1, 32
    c = la.KvCache.empty(4, P, H, D, la.BF16, gpu)
    c.k.zero_(), c.v.zero_()
    table, lens = i32([[3, 1], [2, 0], [0, 0]], gpu), i32([33, 32, 0], gpu)
    k, v = torch.randn(3, H, D, device=gpu), torch.randn(3, H, D, device=gpu)
    c.append(la.KvBatch(table, lens), k, v)
    want = torch.zeros(4, H, P, D, device=gpu).bfloat16()
    wv = want.clone()
    for row, pg, slot in ((0, 1, 0), (1, 2, 31)):
        want[pg, :, slot], wv[pg, :, slot] = k[row].bfloat16(), v[row].bfloat16()
    assert torch.equal(c.k, want) and torch.equal(c.v.transpose(2, 3), wv)


def test_append_q8_non_finite(gpu):
    """A NaN or an infinity among a block's 32 values makes that block NaN, and no other."""
    D, H, P = 96, 1, 16
    c = la.KvCache.empty(2, P, H, D, la.Q8_0, gpu)
    k, v = torch.randn(12, H, D), torch.randn(12, H, D)
    k[3, 0, 40], k[5, 0, 95], v[2, 0, 0], v[9, 0, 33] = float("nan"), float("inf"), -float("inf"), float("nan")
    c.append(la.KvBatch(i32([[1]], gpu), i32([12], gpu), i32([0, 12], gpu), n_tokens=12, max_new=12), k.to(gpu), v.to(gpu))
    for x, is_v in ((k, False), (v, True)):
        got = ref.unpack(c, 1, is_v)[0, :12]
        bad = ~torch.isfinite(x[:, 0].reshape(12, 3, 32)).all(-1)
        assert torch.equal(torch.isnan(got.reshape(12, 3, 32)).all(-1), bad)
        assert torch.isfinite(got.reshape(12, 3, 32)[~bad]).all()


# ----------------------------------------------------------- attention

SHAPES = [(64, 16), (96, 32), (128, 64), (192, 128), (256, 256), (512, 64)]


@pytest.mark.parametrize("D,P", SHAPES)
@pytest.mark.parametrize("io", [la.F32, la.F16, la.BF16])
@pytest.mark.parametrize("tag", [la.F16, la.BF16, la.Q8_0])
def test_attention_types(gpu, tag, io, D, P):
    """Every cache type, query type and head size: one and several tokens, ragged lengths that end inside tiles and pages."""
    f = Filled(gpu, D, tag, D, 2, P, [1, 200, 45, 129], [1, 3, 2, 1], io)
    f.check(f.queries(D + 1, 6))


@pytest.mark.parametrize("new", [1, 2, 5, 16])
@pytest.mark.parametrize("group,H", [(1, 3), (4, 2), (7, 1), (16, 1)])
def test_attention_rows(gpu, group, H, new):
    """Query rows from one to 256 a kv head: padded tiles, two tiles, several passes."""
    f = Filled(gpu, 3, la.F16, 64, H, 32, [300, 16, 33], [new, new, 1], la.F32)
    f.check(f.queries(4, group * H))


@pytest.mark.parametrize("n", [1, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 1000])
@pytest.mark.parametrize("D,tag", [(128, la.BF16), (256, la.F16), (128, la.Q8_0)])
def test_attention_lengths(gpu, D, tag, n):
    f = Filled(gpu, n, tag, D, 1, 16, [n], [1], la.F32)
    f.check(f.queries(n, 4))


@pytest.mark.parametrize("window", [1, 2, 31, 32, 33, 100, 128, 299, 5000, 2 ** 31 - 1])
@pytest.mark.parametrize("tag,D", [(la.F16, 64), (la.Q8_0, 256)])
def test_attention_window(gpu, tag, D, window):
    f = Filled(gpu, 5, tag, D, 2, 16, [300, 40, 3, 129], [4, 1, 3, 2], la.F32)
    f.check(f.queries(6, 4), window=window)


@pytest.mark.parametrize("group,new", [(8, [4, 3, 1, 2]), (3, [16, 1, 11, 2])])
@pytest.mark.parametrize("D,P", SHAPES)
@pytest.mark.parametrize("io", [la.F32, la.F16, la.BF16])
@pytest.mark.parametrize("tag", [la.F16, la.BF16, la.Q8_0])
def test_attention_types_two_tiles(gpu, tag, io, D, P, group, new):
    """The same with 32 query rows a kv head, and with 48: two tiles of 16 rows in
    a workgroup, a second workgroup that is half empty, items that several runs
    share, and a window of fewer keys than new tokens."""
    f = Filled(gpu, D + group, tag, D, 2, P, [4, 700, 45, 129], new, io)
    q = f.queries(D + 1, 2 * group)
    f.check(q)
    f.check(q, window=3)


@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
@pytest.mark.parametrize("tag,D", [(la.F16, 512), (la.BF16, 512), (la.Q8_0, 512), (la.F16, 96), (la.BF16, 192), (la.Q8_0, 192),
                                   (la.Q8_0, 64)])
def test_attention_hidden_non_finite_two_tiles(gpu, tag, D, bad):
    """What the step's earlier tokens and the window's later ones do not see, with 40 query rows a kv head."""
    P, N, n, window = 16, 4, 140, 20
    f = Filled(gpu, 23, tag, D, 1, P, [n], [N], la.F32)
    q = f.queries(24, 10)
    clean = f.check(q, window=window)
    for at, seen in ((n - 2, (2, 3)), (n - N + 1 - window + 1, (0, 1))):
        pg, slot = f.table[0][at // P], at % P
        pools = [(t[pg].view(torch.float16)[P * D // 2:].view(D // 32, P)[:, slot] if tag == la.Q8_0 else
                  t[pg, 0, slot] if t is f.cache.k else t[pg, 0, :, slot]) for t in (f.cache.k, f.cache.v)]
        held = [t.clone() for t in pools]
        for t in pools:
            t.fill_(bad)
        got = f.cache.attention(f.batch, q.to(gpu), window=window).cpu()
        for t, was in zip(pools, held):
            t.copy_(was)
        for j in range(N):
            if j in seen:
                assert not torch.isfinite(got[j]).any(-1).all()
            else:
                assert torch.equal(got[j], clean[j])


@pytest.mark.parametrize("io", [la.F32, la.F16, la.BF16])
@pytest.mark.parametrize("D", [64, 256])
def test_attention_q8_range(gpu, io, D):
    """Values up to 65504 are read as they are, larger ones as NaN: a key of them in the
    rows that see it, a value in its column of them.

    Filled.check's bound on lse is for scores near 1.  Here they reach 6e4, with sums of
    products several times as large: as a function of the scores lse moves by no more
    than the score that moves most, and a score by (D + 8) 2^-24 + 2^-22 of its sum of
    |q k| (ref.attention)."""
    P, n, at = 16, 40, 38
    f = Filled(gpu, 25, la.Q8_0, D, 1, P, [n], [3], io)
    q = f.queries(26, 4)
    clean = f.check(q)
    pg, slot = f.table[0][at // P], at % P
    half = lambda t: t[pg].view(torch.float16)[P * D // 2:].view(D // 32, P)
    k_was = half(f.cache.k)[0, slot].clone()
    for t in (f.cache.k, f.cache.v):
        half(t)[0, slot] = 515.0                              # 127 * 515 = 65405
        lse = torch.empty(q.shape[:2], device=gpu)
        out = f.cache.attention(f.batch, q.to(gpu), lse=lse).cpu()
        want, want_lse, tol = ref.attention(f.cache, f.table, f.lens, f.start, q, D ** -0.5)
        assert ((out.double() - want).abs() <= tol).all()
        keys = ref.sequence(f.cache, f.table[0], n)[0][0].abs()
        ds = ((D + 8) * 2 ** -24 + 2 ** -22) * D ** -0.5 * (q.double().abs() @ keys.T).amax(-1)
        assert ((lse.cpu().double() - want_lse).abs() <= 2e-5 + 2 ** -22 * want_lse.abs() + ds).all()
    half(f.cache.k)[0, slot] = 600.0
    got = f.cache.attention(f.batch, q.to(gpu)).cpu()
    assert torch.equal(got[0], clean[0]) and torch.isnan(got[1:]).all()
    half(f.cache.k)[0, slot] = k_was
    half(f.cache.v)[0, slot] = 600.0
    got = f.cache.attention(f.batch, q.to(gpu)).cpu()
    past = ref.unpack(f.cache, pg, True)[0, slot].abs() >= 65520      # halfway to fp16's next
    assert past.any() and not past.all()
    assert torch.equal(got[0], clean[0])
    assert torch.equal(torch.isnan(got[1:]), past.expand(2, 4, D))


@pytest.mark.parametrize("n_head", [1, 20])
@pytest.mark.parametrize("D,P", SHAPES)
@pytest.mark.parametrize("io", [la.F32, la.F16, la.BF16])
def test_attention_q8_values(gpu, io, D, P, n_head):
    """8-bit values enter results with all their bits.  With queries of zeros every
    weight is the same power of two, so that a row that sees one key is its value
    rounded once, bit for bit; means of up to four keys are off by their rounding
    and by what fp32 sums of four products, their number's reciprocal and the product
    with it leave: six roundings, 6 * 4 * 2^-24 < 2^-19 of the largest value."""
    f = Filled(gpu, D + n_head, la.Q8_0, D, 1, P, [1, 4], [1, 4], io)
    q = torch.zeros(f.T, n_head, D, dtype=DT[io])
    out = f.cache.attention(f.batch, q.to(gpu)).cpu()
    for s, n in enumerate(f.lens):
        _, v, _ = ref.sequence(f.cache, f.table[s], n)
        assert torch.equal(out[f.start[s]], v[:, 0].to(DT[io]).expand(n_head, D))
        for t in range(1, n):
            want = v[:, :t + 1].mean(1)
            off = (out[f.start[s] + t].double() - want).abs()
            assert (off <= ref.EPS[io] * want.abs() + 2 ** -19 * v[:, :t + 1].abs().max()).all()


def test_attention_empty_rows(gpu):
    """Sequences without tokens, without new ones, more new rows than tokens,
    and keys without a page: rows that see nothing get 0 and -inf."""
    f = Filled(gpu, 8, la.F16, 64, 1, 16, [0, 20, 2, 16, 70], [1, 0, 4, 1, 2], la.F32,
               holes=[(3, 0, -1), (4, 0, 77), (4, 2, -5)])
    out = f.check(f.queries(9, 2))
    assert (out[0] == 0).all() and (out[1:3] == 0).all() and (out[5] == 0).all()


def test_attention_hole_hides_whole_window(gpu):
    f = Filled(gpu, 8, la.BF16, 128, 1, 16, [64], [2], la.BF16, holes=[(0, 3, 1000)])
    out = f.check(f.queries(9, 2), window=8)
    assert (out == 0).all()


@pytest.mark.parametrize("bad", [float("inf"), -float("inf"), float("nan")])
@pytest.mark.parametrize("tag,D,n", [(la.F16, 64, 70), (la.BF16, 128, 129), (la.F16, 256, 257), (la.Q8_0, 128, 40), (la.BF16, 512, 66)])
def test_attention_hidden_non_finite(gpu, tag, D, n, bad):
    """A later token's infinite or NaN key and value stay out of the rows that
    do not see it (the earlier tokens of the step; later ones by the window)."""
    H, P, N = 1, 16, 4
    f = Filled(gpu, 21, tag, D, H, P, [n], [N], la.F32)
    q = f.queries(22, 3)
    clean = f.check(q, window=20)

    def poison(at):
        pg, slot = f.table[0][at // P], at % P
        if tag == la.Q8_0:
            for t in (f.cache.k, f.cache.v):
                t[pg].view(torch.float16)[P * D // 2:].view(D // 32, P)[:, slot] = bad
        else:
            f.cache.k[pg, :, slot] = bad
            f.cache.v[pg, :, :, slot] = bad

    def run():
        return f.cache.attention(f.batch, q.to(gpu), window=20).cpu()

    poison(n - 2)                                             # tokens 2 and 3 of the step see it
    got = run()
    assert torch.equal(got[:2], clean[:2]) and not torch.isfinite(got[2:]).any(-1).all(-1).any()
    f = Filled(gpu, 21, tag, D, H, P, [n], [N], la.F32)
    poison(n - N + 1 - 20 + 1)                                # tokens 0 and 1 see it, 2 is past it
    got = run()
    assert torch.equal(got[2:], clean[2:]) and not torch.isfinite(got[:2]).any(-1).all(-1).any()


def test_attention_flat_and_steep(gpu):
    """Scores all equal, and scores hundreds apart whose order changes along the keys."""
    f = Filled(gpu, 31, la.F16, 128, 1, 64, [2000, 700], [1, 2], la.F32)
    q = f.queries(32, 2)
    f.check(torch.zeros_like(q))
    f.check(q * 300)
    f.check(q * 1e-6)
    f.check(q, scale=-0.3)


@pytest.mark.parametrize("size", [1e-9, 3e4])
def test_attention_query_range(gpu, size):
    """fp32 queries far from 1: the parts keep their precision."""
    f = Filled(gpu, 33, la.F16, 64, 1, 16, [100], [1], la.F32)
    q = f.queries(34, 2)
    f.check(q * size, scale=0.125 / size)


def test_attention_many_sequences(gpu):
    """More sequences than threads that count them, most of them short."""
    n = 700
    g = torch.Generator().manual_seed(1)
    lens = torch.randint(0, 40, (n,), generator=g).tolist()
    lens[5], lens[650] = 900, 333
    new = [min(k, 1 + i % 2) for i, k in enumerate(lens)]
    f = Filled(gpu, 41, la.BF16, 64, 1, 16, lens, new, la.BF16)
    f.check(f.queries(42, 2))


def test_attention_layouts(gpu):
    """Rows of a fused projection, pages apart, a table and results wider than
    needed; rows behind the last sequence stay."""
    D, H, P, n_head = 64, 2, 16, 4
    g = torch.Generator().manual_seed(2)
    f = Filled(gpu, 51, la.F16, D, H, P, [50, 33], [2, 1], la.F32)
    big_k = torch.full((f.cache.n_pages, 3, H, P, D), float("nan"), dtype=torch.float16, device=gpu)
    big_v = torch.full((f.cache.n_pages, 2, H, D, P), float("nan"), dtype=torch.float16, device=gpu)
    big_k[:, 1], big_v[:, 1] = f.cache.k, f.cache.v
    cache = la.KvCache(big_k[:, 1], big_v[:, 1])
    table = torch.full((2, 9), 12345, dtype=torch.int32, device=gpu)
    table[:, 1:1 + f.tb.shape[1]] = f.tb
    b = la.KvBatch(table[:, 1:1 + f.tb.shape[1]], i32(f.lens, gpu), i32(f.start, gpu), n_tokens=3, max_new=2)
    qkv = torch.randn(6, n_head + 2 * H, D, generator=g).to(gpu)
    out = torch.full((6, n_head + 1, D), 5.0, device=gpu)[:, :n_head]
    cache.attention(b, qkv[:, :n_head], out=out)
    want = f.cache.attention(f.batch, qkv[:3, :n_head].contiguous())
    assert torch.equal(out[:3], want) and (out[3:] == 5).all()
    f.check(qkv[:3, :n_head].cpu())


def test_attention_long_split(gpu):
    """One sequence over every workgroup: the join of hundreds of parts."""
    D, P = 64, 256
    f = Filled(gpu, 61, la.F16, D, 1, P, [150000], [1], la.F32, spare=1)
    f.check(f.queries(62, 2))


def test_attention_beyond_32_bits(gpu):
    """Pages past 4 GiB of a pool (strides apart, so that little memory is written)."""
    D, H, P = 64, 1, 16
    n_pages, gap = 9, 1 << 28                       # values between pages: 512 MiB
    pool = [torch.empty(8 * gap + H * P * D, dtype=torch.float16, device=gpu) for _ in range(2)]
    k = pool[0].as_strided((n_pages, H, P, D), (gap, P * D, D, 1))
    v = pool[1].as_strided((n_pages, H, D, P), (gap, P * D, P, 1))
    cache = la.KvCache(k, v)
    f = Filled(gpu, 71, la.F16, D, H, P, [9 * P - 3], [2], la.F32, spare=0)
    for t, src in ((k, f.cache.k), (v, f.cache.v)):
        for i in range(n_pages):
            t[i] = src[i]
    q = f.queries(72, 2).to(gpu)
    assert torch.equal(cache.attention(f.batch, q), f.cache.attention(f.batch, q))
    # and an append there
    b = la.KvBatch(i32([[8]], gpu), i32([5], gpu))
    x = torch.randn(1, H, D, device=gpu)
    cache.append(b, x, 2 * x)
    assert torch.equal(k[8, :, 4], x[0].half()) and torch.equal(v[8, :, :, 4], (2 * x[0]).half())
    del pool, k, v, cache
    torch.cuda.empty_cache()


def test_attention_repeats(gpu):
    f = Filled(gpu, 81, la.BF16, 128, 2, 16, [3000, 77, 1, 512], [4, 1, 1, 2], la.BF16)
    q = f.queries(82, 8).to(gpu)
    first = f.cache.attention(f.batch, q)
    for _ in range(5):
        assert torch.equal(f.cache.attention(f.batch, q), first)


def test_attention_graphs_share_a_workspace(gpu):
    """Two captured graphs with one workspace, replayed in turn as the lengths
    grow, equal to eager calls every time; a call on another stream."""
    f = Filled(gpu, 91, la.F16, 128, 2, 16, [700, 45], [1, 1], la.F32, width=50)
    f2 = Filled(gpu, 92, la.F16, 128, 2, 16, [260], [2], la.F32, width=40)
    ws = max((x.cache.attention_workspace(x.batch, 4) for x in (f, f2)), key=lambda t: t.numel())
    qs, outs, graphs = [x.queries(93, 4).to(gpu) for x in (f, f2)], [], []
    for x, q in zip((f, f2), qs):
        out = torch.empty_like(q)
        x.cache.attention(x.batch, q, out=out, workspace=ws)          # loaded before the capture
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            x.cache.attention(x.batch, q, out=out, workspace=ws)
        outs.append(out)
        graphs.append(g)
    for step in range(4):
        for x, q, out, g in zip((f, f2), qs, outs, graphs):
            out.fill_(float("nan"))
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, x.cache.attention(x.batch, q))
        f.batch.lens.sub_(torch.tensor([130, 7], dtype=torch.int32, device=gpu))
        f2.batch.lens.sub_(60)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = f.cache.attention(f.batch, qs[0])
    side.synchronize()
    assert torch.equal(got, f.cache.attention(f.batch, qs[0]))


def test_cache_refusals(gpu):
    c = la.KvCache.empty(4, 16, 2, 64, la.F16, gpu)
    b = la.KvBatch(i32([[0, 1]], gpu), i32([5], gpu))
    with pytest.raises(ValueError, match="new_start needs"):
        la.KvBatch(i32([[0, 1]], gpu), i32([5], gpu), i32([0, 1], gpu))
    with pytest.raises(ValueError, match="lens"):
        la.KvBatch(i32([[0, 1]], gpu), i32([5, 6], gpu))
    with pytest.raises(ValueError, match="page must be"):
        la.KvCache(c.k.transpose(2, 3), c.v.transpose(2, 3))
    with pytest.raises(ValueError, match="q must"):
        c.attention(b, torch.zeros(1, 4, 128, device=gpu))
    with pytest.raises(ValueError, match="unsupported|n_head"):
        c.attention(b, torch.zeros(1, 3, 64, device=gpu))
    with pytest.raises(ValueError, match="float32, float16"):
        c.attention(b, torch.zeros(1, 4, 64, device=gpu, dtype=torch.float64))
    with pytest.raises(ValueError, match="k must"):
        c.append(b, torch.zeros(1, 3, 64, device=gpu), torch.zeros(1, 3, 64, device=gpu))
    with pytest.raises(la.LlapisError, match="workspace"):
        c.attention(b, torch.zeros(1, 4, 64, device=gpu), workspace=torch.empty(16, dtype=torch.uint8, device=gpu))


# --------------------------------------------------------------- pages

def pools(gpu, seed, n_pages, layers, tag=la.F16, H=2, P=16, D=64):
    g = torch.Generator(gpu).manual_seed(seed)
    caches = []
    for _ in range(layers):
        c = la.KvCache.empty(n_pages, P, H, D, tag, gpu)
        for t in (c.k, c.v):
            t.view(torch.uint8).copy_(torch.randint(0, 256, t.view(torch.uint8).shape, generator=g, device=gpu, dtype=torch.uint8))
        caches.append(c)
    return la.KvPages(caches)


def planes_of(pages):
    return [t.view(torch.uint8).cpu().reshape(pages.n_pages, -1) for c in pages.caches for t in (c.k, c.v)]


def check_moved(before, after, moves):
    for a, b in zip(before, after):
        want = a.clone()
        for frm, to in moves:
            want[to] = a[frm]
        assert torch.equal(b, want)


@pytest.mark.parametrize("tag,layers,P,D", [(la.F16, 1, 16, 64), (la.Q8_0, 3, 32, 96), (la.BF16, 70, 16, 64), (la.F16, 2, 256, 256)])
def test_copy_pages(gpu, tag, layers, P, D):
    """Pairs in every plane of 1 to 140 planes; ids outside the pool are skipped."""
    p = pools(gpu, 1, 9, layers, tag, P=P, D=D)
    before = planes_of(p)
    p.copy(i32([[0, 5], [0, 6], [3, 8], [-1, 4], [2, 9], [9, 4]], gpu))
    check_moved(before, planes_of(p), [(0, 5), (0, 6), (3, 8)])
    p.copy(torch.empty(0, 2, dtype=torch.int32, device=gpu))


def test_fork(gpu):
    """Partly filled and full last pages, an empty source, two forks of one
    source, and forks that are skipped: rows outside, onto itself, no fresh page,
    a source without its page, a length past the table."""
    for layers in (2, 66):
        p = pools(gpu, 2, 24, layers)
        table = [[0, 1, 2, -1], [3, 4, -1, -1], [-1] * 4, [5, -1, 9, -1], [6, 7, 8, 10]] + [[20 + i, 21, 22, 23] for i in range(8)]
        lens = [40, 32, 0, 30, 65] + [1] * 8
        forks = [[0, 5, 11], [0, 6, 12], [1, 7, 13], [2, 8, 14], [0, 0, 15], [0, 99, 15], [-1, 9, 15], [0, 9, 24],
                 [3, 10, 16], [4, 11, 17], [0, 12, 2]]
        tb, ln, before = i32(table, gpu), i32(lens, gpu), planes_of(p)
        p.fork(tb, ln, i32(forks, gpu))
        want_t, want_l, copies = ref.fork(table, lens, forks, 16, 24)
        assert tb.tolist() == want_t and ln.tolist() == want_l and copies == [(2, 11), (2, 12)]
        check_moved(before, planes_of(p), copies)


def random_tables(seed, n_seq, width, n_pages, P, shared=0.2, bad=0.05):
    g = torch.Generator().manual_seed(seed)
    r = lambda: float(torch.rand((), generator=g))
    order = torch.randperm(n_pages, generator=g).tolist()[:max(1, int(0.6 * n_pages))]
    used, table, lens = [], [], []
    for _ in range(n_seq):
        row = []
        for _ in range(width):
            x = r()
            if x < bad:
                row.append([-1, n_pages, 10 ** 9, -7][int(r() * 4)])
            elif x < bad + shared and used:
                row.append(used[int(r() * len(used))])
            elif order:
                row.append(order.pop())
                used.append(row[-1])
            else:
                row.append(-1)
        table.append(row)
        lens.append([0, int(r() * width * P), width * P, width * P + 50, -3, 1][int(r() * 6)])
    return table, lens


@pytest.mark.parametrize("n_seq,width,n_pages", [(1, 1, 1), (3, 4, 16), (40, 30, 1000), (300, 3, 2500), (2, 600, 1025)])
def test_page_refs(gpu, n_seq, width, n_pages):
    P = 16
    table, lens = random_tables(n_pages, n_seq, width, n_pages, P)
    p = pools(gpu, 3, n_pages, 1, H=1)
    refs, free, n_free = p.refs(i32(table, gpu), i32(lens, gpu))
    want = ref.page_refs(table, lens, P, n_pages)
    want_free = [i for i, r in enumerate(want) if r == 0]
    assert refs.tolist() == want and int(n_free) == len(want_free)
    assert free.tolist() == want_free + [-1] * (n_pages - len(want_free))


@pytest.mark.parametrize("n_seq,width,n_pages,layers", [(1, 1, 1, 1), (3, 4, 16, 2), (40, 30, 1000, 2), (300, 3, 2500, 1),
                                                        (2, 600, 1025, 1), (6, 5, 40, 67)])
def test_compact(gpu, n_seq, width, n_pages, layers):
    P = 16
    table, lens = random_tables(n_pages + 1, n_seq, width, n_pages, P)
    p = pools(gpu, 4, n_pages, layers, H=1)
    tb, ln, before = i32(table, gpu), i32(lens, gpu), planes_of(p)
    out, refs, n_live = p.compact(tb, ln)
    want, after, n, moves = ref.compact(table, lens, P, n_pages)
    assert out.tolist() == want and refs.tolist() == after and int(n_live) == n and tb.tolist() == table
    check_moved(before, planes_of(p), moves)
    # again, in place, on what is compact already: nothing moves
    before = planes_of(p)
    p.compact(out, ln, table_out=out)
    assert out.tolist() == want
    check_moved(before, planes_of(p), [])


@pytest.mark.parametrize("n_seq,width,n_pages,layers", [(30, 40, 8193, 1), (300, 230, 1000, 2), (220, 300, 20000, 1), (5, 13200, 8500, 66)])
@pytest.mark.parametrize("in_place", [False, True])
def test_compact_large(gpu, n_seq, width, n_pages, layers, in_place):
    """Pools of more than 8192 pages and tables of more than 65536 entries, moved
    in place too, and by two calls a compaction in the last case."""
    P = 16
    table, lens = random_tables(n_pages + 1, n_seq, width, n_pages, P)
    p = pools(gpu, 6, n_pages, layers, H=1)
    tb, ln = i32(table, gpu), i32(lens, gpu)
    before = [c.k.clone() for c in p.caches] + [c.v.clone() for c in p.caches]
    out, refs, n_live = p.compact(tb, ln, table_out=tb if in_place else None)
    want, after, n, moves = ref.compact(table, lens, P, n_pages)
    assert out.tolist() == want and refs.tolist() == after and int(n_live) == n
    assert in_place or tb.tolist() == table
    assert len(moves) > 0
    frm, to = torch.tensor(moves).to(gpu).T
    for was, now in zip(before, [c.k for c in p.caches] + [c.v for c in p.caches]):
        was.view(torch.int16)[to] = was.view(torch.int16)[frm]
        assert torch.equal(was.view(torch.int16), now.view(torch.int16))


@pytest.mark.parametrize("in_place", [False, True])
def test_compact_many_planes(gpu, in_place):
    """More planes than a call takes, pages that do move: every plane's move and the table's are the same."""
    P, n_pages = 16, 40
    table, lens = [[39, 3, 38, 20], [20, 1, 37, -1], [30, 31, 32, 33]], [64, 40, 17]
    p = pools(gpu, 7, n_pages, 67, H=1)
    tb, ln, before = i32(table, gpu), i32(lens, gpu), planes_of(p)
    out, refs, n_live = p.compact(tb, ln, table_out=tb if in_place else None)
    want, after, n, moves = ref.compact(table, lens, P, n_pages)
    assert len(moves) == 6 and n == 8
    assert out.tolist() == want and refs.tolist() == after and int(n_live) == n
    check_moved(before, planes_of(p), moves)


def test_compact_full_and_empty(gpu):
    p = pools(gpu, 5, 8, 1)
    full = [[7, 6, 5, 4], [3, 2, 1, 0]]
    out, refs, n_live = p.compact(i32(full, gpu), i32([64, 64], gpu))
    assert out.tolist() == full and int(n_live) == 8 and refs.tolist() == [1] * 8
    out, refs, n_live = p.compact(i32(full, gpu), i32([0, 0], gpu))
    assert out.tolist() == [[-1] * 4] * 2 and int(n_live) == 0 and refs.tolist() == [0] * 8
    with pytest.raises(la.LlapisError, match="workspace"):
        p.compact(i32(full, gpu), i32([0, 0], gpu), workspace=torch.empty(8, dtype=torch.uint8, device=gpu))


# --------------------------------------------------------------- norms

def norm_bound(h64, x64, u_mag, w, tag, alpha, beta, d):
    """Bounds of (h', x).  fp32 steps on the way to h': the mean of squares of d
    values summed in 64 lanes and waves has a relative error of (d / 64 + 32)
    2^-24 at most (all terms positive), its square root and quotient two
    roundings more, the products and the sum five: (d / 128 + 24) 2^-24 of each
    term's magnitude.  x: the same again relative to itself, and h's error over
    rms(h).  Each output is rounded once into its type."""
    e = (d / 128 + 24) * 2 ** -24
    h_abs = e * u_mag
    rms = h64.square().mean(-1, keepdim=True).sqrt()
    x_abs = e * x64.abs() + 2 * (h_abs + h_abs.square().mean(-1, keepdim=True).sqrt()) / rms * (1 if w is None else w.double().abs())
    tiny = torch.finfo(DT[tag]).smallest_normal * ref.EPS[tag] * 2
    return h_abs + ref.EPS[tag] * (h64.abs() + h_abs) + tiny, x_abs + ref.EPS[tag] * (x64.abs() + x_abs) + tiny


@pytest.mark.parametrize("gate", ["none", "token", "channel", "full", "one"])
@pytest.mark.parametrize("T,d", [(1, 1), (3, 7), (2, 64), (5, 153), (4, 2816), (600, 515), (530, 2816), (2, 4099), (1, 16384), (700, 5000)])
@pytest.mark.parametrize("tag", [la.F32, la.F16, la.BF16])
def test_block_norm(gpu, tag, T, d, gate):
    g = torch.Generator().manual_seed(d)
    r = lambda *s: torch.randn(*s, generator=g)
    h, y = (2 * r(T, d)).to(DT[tag]), (0.3 * r(T, d)).to(DT[tag])
    shape = {"none": None, "token": (T, 1), "channel": (1, d), "full": (T, d), "one": (1, 1)}[gate]
    gt = None if shape is None else torch.sigmoid(r(*shape)).to(DT[tag])
    post, weights = 1 + 0.2 * r(d), [1 + 0.2 * r(d), None, r(d)]
    up = lambda t: None if t is None else t.to(gpu)
    got_h, got_x = la.block_norm(up(h), up(y), post_weight=up(post), gate=up(gt), alpha=0.9, beta=0.7, weights=[up(w) for w in weights])
    want_h, want_x = ref.block_norm(h, y, post, True, gt, 0.9, 0.7, weights, 1e-6)
    u = ref.block_norm(0 * h, y, post, True, gt, 0.9, 0.7, (), 1e-6)[0]
    mag = 0.9 * h.double().abs() + u.abs()
    for got, want, w in zip(got_x, want_x, weights):
        bh, bx = norm_bound(want_h, want, mag, w, tag, 0.9, 0.7, d)
        assert ((got.cpu().double() - want).abs() <= bx).all()
    assert ((got_h.cpu().double() - want_h).abs() <= bh).all()


def test_block_norm_parts(gpu):
    """Without y, without the post-norm, without outputs, in place, rows apart and off 16 bytes."""
    T, d = 9, 130
    h, y = torch.randn(T, d, device=gpu), torch.randn(T, d, device=gpu)
    full, (x,) = la.block_norm(h, y, post_norm=False, weights=[None], alpha=1.0, beta=1.0)
    assert torch.equal(full, h + y)
    h2 = h.clone()
    x2 = la.residual_rmsnorm(h2, y)
    assert torch.equal(h2, full)
    assert ((x - x2).abs() <= 2 ** -20 * x2.abs()).all()              # the same sums in another order
    only, (n,) = la.block_norm(h, weights=[None])
    assert torch.equal(only, h)
    wide = torch.zeros(T, 2 * d + 3, device=gpu)
    a, b = wide[:, 1:1 + d], wide[:, d + 2:2 * d + 2]
    a.copy_(h), b.copy_(y)
    out = torch.full((T, d + 5), 3.0, device=gpu)
    got, (z,) = la.block_norm(a, b, post_norm=False, weights=[None], h_out=a, out=[out[:, 2:2 + d]])
    assert torch.equal(a, full) and torch.equal(z, x) and (out[:, :2] == 3).all() and (out[:, 2 + d:] == 3).all()
    assert torch.equal(wide[:, d + 2:2 * d + 2], y) and (wide[:, 0] == 0).all() and (wide[:, -1] == 0).all()
    got, none = la.block_norm(h, y, beta=0.5)
    assert none == [] and got.shape == h.shape
    zero, (z,) = la.block_norm(0 * h, 0 * y, weights=[None])
    assert (zero == 0).all() and (z == 0).all()
    assert la.block_norm(h[:0], weights=[None])[1][0].shape == (0, d)


def test_block_norm_refusals(gpu):
    h = torch.zeros(3, 64, device=gpu)
    for bad, words in ((dict(y=h.half()), "y must"), (dict(gate=h[:, :3]), "gate must"), (dict(weights=[h[0].half()]), "weights"),
                       (dict(weights=[None] * 5), "at most 4"), (dict(weights=[None], out=[]), "out needs"),
                       (dict(post_weight=h[0, :5]), "post_weight"), (dict(h_out=h.t()), "h_out")):
        with pytest.raises(ValueError, match=words):
            la.block_norm(h, **bad)
    with pytest.raises(la.LlapisError, match="16384"):
        la.block_norm(torch.zeros(1, 16385, device=gpu))


# --------------------------------------------------------- verification

def drafted(seed, S, n, V, tag, noise=0.7):
    g = torch.Generator().manual_seed(seed)
    logits = 2.0 * torch.randn(S, n + 1, V, generator=g)
    p = torch.softmax(logits, -1).to(DT[tag])
    q = torch.softmax(logits[:, :n] + noise * torch.randn(S, n, V, generator=g), -1)
    drafts = (q / -torch.rand(S, n, V, generator=g).clamp(min=1e-20).log()).argmax(-1).to(torch.int32)
    return p, q.to(DT[tag]), drafts, torch.rand(S, n, generator=g), torch.rand(S, generator=g)


def check_verify(gpu, p, q, d, u, un, n_draft=None):
    up = lambda t: None if t is None else t.to(gpu)
    nd = None if n_draft is None else i32(n_draft, gpu)
    tokens, accepted = la.verify_drafts(up(p), up(q), up(d), up(u), up(un), n_draft=nd)
    want_t, want_a = ref.verify(p, q, d, u, un, n_draft)
    assert accepted.tolist() == want_a and tokens.tolist() == want_t
    return want_t, want_a


@pytest.mark.parametrize("S,n,V", [(1, 1, 1), (1, 3, 2), (5, 3, 37), (20, 4, 1000), (3, 3, 8192), (3, 2, 8193), (2, 3, 70001), (1, 0, 50),
                                   (2, 63, 11), (1, 1, 3000000)])
@pytest.mark.parametrize("tag", [la.F32, la.F16, la.BF16])
def test_verify(gpu, tag, S, n, V):
    for onehot in (False, True):
        p, q, d, u, un = drafted(V + n, S, n, V, tag)
        check_verify(gpu, p, None if onehot else q, d, u, un)
        check_verify(gpu, p, None if onehot else q, d, u, un, [(3 * s) % (n + 2) - 1 for s in range(S)])


def test_verify_corners(gpu):
    """All taken, none taken, drafts outside the vocabulary, equal rows (nothing
    left to draw from), u_next at 0 and at 1, non-finite and negative values, a
    row of nothing."""
    S, n, V = 6, 3, 500
    p, q, d, u, un = drafted(5, S, n, V, la.F32)
    _, a = check_verify(gpu, p, p[:, :n].clone(), d, u * 0, un)
    assert a == [n] * S
    _, a = check_verify(gpu, p, q, d, u * 0 + 1e30, un)
    assert a == [0] * S
    check_verify(gpu, p, p[:, :n].clone(), d, u * 0 + 1.0, un)          # u q = p: refused, and nothing left of p - q
    for edge in (0.0, 1.0, 1.0 - 2 ** -24):
        check_verify(gpu, p, q, d, u, un * 0 + edge)
    bad = d.clone()
    bad[0, 0], bad[1, 1], bad[2, 2] = -1, V, 2 ** 31 - 1
    check_verify(gpu, p, q, bad, u, un)
    check_verify(gpu, p, None, bad, u, un)
    odd = p.clone()
    odd[0, 0, ::3], odd[1, :, 5], odd[2, 1, :] = float("nan"), float("inf"), -1.0
    odd[3] = 0
    t, a = check_verify(gpu, odd, q, d, u, un)
    assert a[3] == 0 and t[3][0] == -1
    oq = q.clone()
    oq[:, :, ::7], oq[:, :, 3] = float("nan"), -2.0
    check_verify(gpu, p, oq, d, u, un)
    # the last and the first token of the vocabulary
    one = torch.zeros(2, 2, V)
    one[0, :, V - 1], one[1, :, 0] = 1, 1
    t, a = check_verify(gpu, one, None, torch.tensor([[3], [3]], dtype=torch.int32), torch.rand(2, 1), torch.rand(2))
    assert t == [[V - 1, -1], [0, -1]]


def test_verify_layouts(gpu):
    """Rows apart and off 16 bytes; a graph replayed with new numbers in place."""
    S, n, V = 4, 3, 777
    p, q, d, u, un = drafted(6, S, n, V, la.F32)
    wide_p, wide_q = torch.full((S, n + 1, V + 10), float("nan"), device=gpu), torch.full((S, n, V + 5), float("nan"), device=gpu)
    pp, qq = wide_p[:, :, 3:3 + V], wide_q[:, :, 1:1 + V]
    pp.copy_(p), qq.copy_(q)
    args = [pp, qq, d.to(gpu), u.to(gpu), un.to(gpu)]
    ws = la.verify_workspace(S, V, gpu)
    tokens, accepted = la.verify_drafts(*args, workspace=ws)
    assert tokens.tolist() == ref.verify(p, q, d, u, un, None)[0]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        la.verify_drafts(*args, tokens=tokens, accepted=accepted, workspace=ws)
    for seed in range(4):
        u, un = torch.rand(S, n), torch.rand(S)
        args[3].copy_(u), args[4].copy_(un)
        g.replay()
        assert tokens.tolist() == ref.verify(p, q, d, u, un, None)[0]
        assert torch.equal(la.verify_drafts(*args)[0], tokens)


def test_verify_draws_the_target(gpu):
    """The drawn tokens' frequencies are the target's, whatever drafted them: a
    chi-square over 16 tokens and 20000 steps (15 degrees of freedom: above 50
    once in 10^5)."""
    V, S = 16, 20000
    g = torch.Generator().manual_seed(9)
    p1, q1 = torch.softmax(torch.randn(V, generator=g), 0), torch.softmax(torch.randn(V, generator=g), 0)
    p, q = p1.expand(S, 2, V).contiguous(), q1.expand(S, 1, V).contiguous()
    d = torch.multinomial(q1, S, replacement=True, generator=g)[:, None].to(torch.int32)
    tokens, _ = la.verify_drafts(p.to(gpu), q.to(gpu), d.to(gpu), torch.rand(S, 1, generator=g).to(gpu), torch.rand(S, generator=g).to(gpu))
    seen = torch.bincount(tokens[:, 0].cpu().long(), minlength=V).double()
    want = S * p1.double()
    assert float(((seen - want) ** 2 / want).sum()) < 50


# ------------------------------------------------------------ together

class Step:
    """A decode / verify step of a two-layer sandwich-normed model as a user
    runs it: the norms and the residual stream between attention and the MoE
    layer, the cache of every layer behind one page table, and the verification of
    the step's drafts against the model's own probabilities."""
    EPS = 1e-6

    def __init__(self, gpu, spec, n_seq, width, page):
        from helpers import layer
        D, self.H, self.G, self.hd = spec.d_model, 2, 4, 64
        g = torch.Generator().manual_seed(77)
        mat = lambda *s: (torch.randn(*s, generator=g) / math.sqrt(s[0])).to(gpu)
        w = lambda: (1 + 0.1 * torch.randn(D, generator=g)).to(gpu)
        nh = self.H * self.G
        self.layers = [dict(qkv=mat(D, (nh + 2 * self.H) * self.hd), o=mat(nh * self.hd, D), attn_in=w(), attn_out=w(), moe_in=w(),
                            router_in=w(), moe_out=w(), scale=0.9 + 0.1 * i,
                            moe=la.DeviceLayer(layer(spec, 40 + i, [1, 4, 6, 9, 12], scales=True), gpu),
                            cache=la.KvCache.empty(n_seq * width + 4, page, self.H, self.hd, la.F16, gpu)) for i in range(2)]
        self.final, self.head = w(), mat(D, 300)
        self.pages = la.KvPages([l["cache"] for l in self.layers])

    def run(self, h, batch, record=None):
        """Probabilities [T, vocab] of the new tokens' embeddings h [T, D]."""
        T, nh = h.shape[0], self.H * self.G
        note = record if record is not None else lambda *a: None
        h, (x,) = la.block_norm(h, weights=[self.layers[0]["attn_in"]], eps=self.EPS)
        for i, l in enumerate(self.layers):
            qkv = (x @ l["qkv"]).view(T, nh + 2 * self.H, self.hd)
            q, k, v = qkv[:, :nh], qkv[:, nh:nh + self.H], qkv[:, nh + self.H:]
            l["cache"].append(batch, k, v)
            a = l["cache"].attention(batch, q, window=40 if i else 0)
            note("attention", i, q, k, v, a)
            y = a.reshape(T, -1) @ l["o"]
            h2, xs = la.block_norm(h, y, post_weight=l["attn_out"], weights=[l["moe_in"], l["router_in"]], eps=self.EPS)
            note("norm", h, y, l["attn_out"], 1.0, [l["moe_in"], l["router_in"]], h2, xs)
            m, _, _ = l["moe"].forward(xs[0], x_router=xs[1])
            then = self.layers[1]["attn_in"] if i == 0 else self.final
            h3, (x,) = la.block_norm(h2, m, post_weight=l["moe_out"], alpha=l["scale"], beta=l["scale"], weights=[then], eps=self.EPS)
            note("norm", h2, m, l["moe_out"], l["scale"], [then], h3, [x])
            h = h3
        return torch.softmax(x @ self.head, -1)


def test_decode_steps_together(gpu):
    """Prompts appended, a verify step of four tokens a sequence, one sequence
    forked and another freed, the pool compacted, and single-token steps: every
    stage of every step against its 64-bit form on the stage's own inputs, and a
    captured step's replays bit for bit against eager ones."""
    from helpers import SMALL
    n_seq, width, page = 4, 8, 16
    m = Step(gpu, SMALL, n_seq, width, page)
    g = torch.Generator().manual_seed(78)
    emb = torch.randn(300, SMALL.d_model, generator=g).to(gpu)
    history = [[(torch.zeros(0, m.H, m.hd),) * 2 for _ in range(n_seq)] for _ in m.layers]      # of each layer and sequence, fp16

    def check(starts, lens):
        def record(kind, *a):
            if kind == "norm":
                h, y, post, scale, weights, h2, xs = a
                up = lambda t: t.cpu()
                want_h, want_x = ref.block_norm(up(h), up(y), up(post), True, None, scale, scale, [up(w) for w in weights], m.EPS)
                u = ref.block_norm(0 * up(h), up(y), up(post), True, None, scale, scale, (), m.EPS)[0]
                mag = scale * up(h).double().abs() + u.abs()
                for x, want, w in zip(xs, want_x, weights):
                    bh, bx = norm_bound(want_h, want, mag, up(w), la.F32, scale, scale, h.shape[1])
                    assert ((up(x).double() - want).abs() <= bx).all()
                assert ((up(h2).double() - want_h).abs() <= bh).all()
                return
            i, q, k, v, out = a
            q, k, v, out = (t.cpu() for t in (q, k, v, out))
            for s in range(n_seq):
                rows = slice(starts[s], starts[s + 1])
                hk, hv = history[i][s]
                history[i][s] = (torch.cat([hk, k[rows].half().float()]), torch.cat([hv, v[rows].half().float()]))
            cache = m.layers[i]["cache"]
            want, _, tol = ref.attention(cache, table.tolist(), lens, starts, q, m.hd ** -0.5, 40 if i else 0)
            assert ((out.double() - want).abs() <= tol).all()
            for s in range(n_seq):                   # and the cache holds what was appended, where the table says
                ck, cv, there = ref.sequence(cache, table.tolist()[s], lens[s])
                assert there.all() and torch.equal(ck.transpose(0, 1).float(), history[i][s][0])
                assert torch.equal(cv.transpose(0, 1).float(), history[i][s][1])
        return record

    order = torch.randperm(n_seq * width + 4, generator=g).tolist()
    table = i32([[order.pop() for _ in range(width)] for _ in range(n_seq)], gpu)
    spare = order.pop()

    def step(new, tokens, lens):
        starts = [0]
        for n in new:
            starts.append(starts[-1] + n)
        b = la.KvBatch(table, i32(lens, gpu), i32(starts, gpu), n_tokens=starts[-1], max_new=max(new))
        return m.run(emb[tokens], b, check(starts, lens)), starts

    # prompts of ragged lengths, 16 tokens a call
    lens, prompt = [0] * n_seq, [50, 17, 0, 33]
    while any(a < b for a, b in zip(lens, prompt)):
        new = [min(16, b - a) for a, b in zip(lens, prompt)]
        lens = [a + n for a, n in zip(lens, new)]
        step(new, torch.randint(0, 300, (sum(new),), generator=g), lens)
    # a verify step: the last token and three drafts of each living sequence
    new = [4, 4, 0, 4]
    lens = [a + n for a, n in zip(lens, new)]
    tok = torch.randint(0, 300, (12,), generator=g).to(torch.int32)
    p, _ = step(new, tok.long(), lens)
    u, un = torch.rand(3, 3, generator=g), torch.rand(3, generator=g)
    drafts = tok.reshape(3, 4)[:, 1:].contiguous()
    target = p.reshape(3, 4, 300)
    got, taken = la.verify_drafts(target, None, drafts.to(gpu), u.to(gpu), un.to(gpu))
    want, want_taken = ref.verify(target.cpu(), None, drafts, u, un, None)
    assert got.tolist() == want and taken.tolist() == want_taken
    # refused drafts leave the cache by their length alone
    for s, a in zip((0, 1, 3), want_taken):
        lens[s] -= 3 - a
        for i in range(2):
            history[i][s] = tuple(t[:lens[s]] for t in history[i][s])
    # sequence 0 is forked into row 2, sequence 1 ends, and the pool is compacted
    ln = i32(lens, gpu)
    m.pages.fork(table, ln, i32([[0, 2, spare]], gpu))
    lens[2] = lens[0]
    lens[1] = 0
    ln[1] = 0
    for i in range(2):
        history[i][2], history[i][1] = history[i][0], history[i][1]
        history[i][1] = (torch.zeros(0, m.H, m.hd),) * 2
    refs, _, n_free = m.pages.refs(table, ln)
    _, after, n_live = m.pages.compact(table, ln, table_out=table)
    used = int(n_live)
    assert used + int(n_free) == m.pages.n_pages and int(refs.sum()) == int(after.sum()) == sum(-(-n // page) for n in lens)
    assert ln.tolist() == lens
    # room to grow: the free pages lie behind the live ones
    free = iter(range(used, m.pages.n_pages))
    rows = table.tolist()
    for s in range(n_seq):
        for i in range(-(-lens[s] // page), width):
            rows[s][i] = next(free, -1)
    # the fork's partly filled last page is its own
    if lens[0] % page:
        assert rows[0][lens[0] // page] != rows[2][lens[0] // page]
    table.copy_(i32(rows, gpu))
    # single-token steps; lengths that the table holds
    for _ in range(3):
        new = [1, 0, 1, 1]
        lens = [a + n for a, n in zip(lens, new)]
        step(new, torch.randint(0, 300, (3,), generator=g), lens)
    # the step as a graph: every replay against the eager step
    ln, st = i32(lens, gpu), i32([0, 1, 1, 2, 3], gpu)
    b = la.KvBatch(table, ln, st, n_tokens=3, max_new=1)
    x = emb[:3].clone()
    eager = m.run(x, b)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = m.run(x, b)
    for k in range(3):
        x.copy_(emb[10 * k:10 * k + 3])
        ln.add_(torch.tensor([1, 0, 1, 1], dtype=torch.int32, device=gpu))
        out.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, m.run(x, b))
    assert torch.isfinite(eager).all()


# ------------------------------------------------------------ the largest
def test_sizes_past_32_bits_are_refused(gpu):
    """The library's sizes have 32 bits: what is larger would wrap around to a size that fits."""
    c = la.KvCache.empty(4, 16, 2, 64, la.F16, gpu)
    table, lens = i32([[0, 1]], gpu), i32([5], gpu)
    with pytest.raises(ValueError, match="2\\^31"):
        c.attention(la.KvBatch(table, lens), torch.zeros(1, 4, 64, device=gpu), window=(1 << 32) + 1)
    for n_tokens, max_new in (((1 << 32) + 1, 1), (1, (1 << 32) + 1), (-1, 1), (1, -1)):
        with pytest.raises(ValueError, match="2\\^31"):
            la.KvBatch(table, lens, i32([0, 1], gpu), n_tokens, max_new)
    with pytest.raises(ValueError, match="2\\^31"):
        la.block_norm(torch.zeros(1, 1, device=gpu).expand((1 << 32) + 1, 1))
    with pytest.raises(ValueError, match="2\\^31"):
        la.verify_drafts(torch.zeros(1, 1, 1, device=gpu).expand(1, 1, (1 << 32) + 1), None, torch.zeros(1, 0, dtype=torch.int32, device=gpu),
                         torch.zeros(1, 0, device=gpu), torch.zeros(1, device=gpu))


def test_block_norm_most_tokens(gpu):
    """2^31 - 1 tokens: no count wraps around on the way to the launch, and each token is written."""
    T = (1 << 31) - 1
    h = torch.tensor([[3.0]], device=gpu, dtype=torch.float16).expand(T, 1)
    out = torch.zeros(T, 1, dtype=torch.float16, device=gpu)
    w = torch.tensor([4.0], device=gpu)
    h_out, _ = la.block_norm(h, weights=[w], eps=7.0, out=[out])         # 3, 3 / sqrt(9 + 7) * 4 = 3
    for x in (h_out, out):
        for at in range(0, T, 1 << 29):
            assert bool((x[at:at + (1 << 29)] == 3.0).all())


# ------------------------------------------------------------- two at once
def test_two_threads_and_streams_at_once(gpu):
    """Host threads with a stream and workspaces of their own run every operator at
    once: as each does alone, bit for bit, and a refusal is its own thread's."""
    import threading
    f = Filled(gpu, 301, la.BF16, 128, 2, 16, [2500, 77, 0, 512], [4, 1, 0, 2], la.BF16)
    g = torch.Generator().manual_seed(302)
    q = [f.queries(303 + i, 8).to(gpu) for i in range(2)]
    h, y = (torch.randn(2, 300, 777, generator=g).to(gpu) for _ in range(2))
    target = torch.softmax(3 * torch.randn(2, 3, 4, 9001, generator=g), -1).to(gpu)
    draft = torch.softmax(3 * torch.randn(2, 3, 3, 9001, generator=g), -1).to(gpu)
    drafts = torch.randint(0, 9001, (3, 3), generator=g, dtype=torch.int32).to(gpu)
    u, u_next = torch.rand(3, 3, generator=g).to(gpu), torch.rand(3, generator=g).to(gpu)

    def work(i):
        out = f.cache.attention(f.batch, q[i])
        h2, (x,) = la.block_norm(h[i], y[i], weights=[None])
        tokens, accepted = la.verify_drafts(target[i], draft[i], drafts, u, u_next)
        return [out, h2, x, tokens, accepted]

    alone = [work(i) for i in range(2)]
    torch.cuda.synchronize()
    failed = []

    def thread(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    got = work(i)
                    with pytest.raises(la.LlapisError, match="16384" if i else "16-byte aligned"):
                        if i:
                            la.block_norm(torch.zeros(1, 16385, device=gpu))
                        else:
                            f.cache.attention(f.batch, torch.zeros(8 * 8 * 128 + 1, device=gpu)[1:].view(8, 8, 128))
                    torch.cuda.current_stream().synchronize()
                    assert all(torch.equal(a, b) for a, b in zip(got, alone[i]))
        except BaseException as e:
            failed.append(e)

    threads = [threading.Thread(target=thread, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed
