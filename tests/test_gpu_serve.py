"""Pages and slots, query and key norms with positions, and sampling (llapis_step.h) on
the GPU against their plain 64-bit forms (serve_ref.py)."""
import math

import pytest
import torch

import llapis_amd as la
import serve_ref as ref
import step_ref
from step_ref import DT, EPS

pytestmark = pytest.mark.gpu


def i32(v, dev):
    return torch.tensor(v, dtype=torch.int32).to(dev)


def f32(v, dev):
    return torch.tensor(v, dtype=torch.float32).to(dev)


# -------------------------------------------------------------- extend

def pages(gpu, n_pages, P):
    return la.KvPages([la.KvCache.empty(n_pages, P, 1, 64, la.F16, gpu)]) if P in (16, 32, 64, 128, 256) else None


def run_extend(gpu, P, table, lens, n_new, free, n_free, n_tokens, in_place=False):
    n_pages = len(free)
    pg = pages(gpu, n_pages, P)
    S, width = len(table), len(table[0])
    tb = torch.full((S, width + 3), 12345, dtype=torch.int32, device=gpu)      # rows apart
    tb[:, 1:1 + width] = i32(table, gpu).reshape(S, width)
    view = tb[:, 1:1 + width]
    ln, nf = i32(lens, gpu), i32([n_free], gpu)
    out = (None, None) if in_place else (torch.full_like(ln, 777), torch.full_like(nf, 777))
    got = pg.extend(view, ln, i32(n_new, gpu), i32(free, gpu), nf, n_tokens, lens_out=out[0], n_free_out=out[1])
    want = ref.extend(table, lens, n_new, free, n_free, n_tokens, P, n_pages)
    assert view.tolist() == want[0]
    assert (tb[:, 0] == 12345).all() and (tb[:, 1 + width:] == 12345).all()
    assert (ln if in_place else out[0]).tolist() == want[1]
    assert int(nf if in_place else out[1]) == want[2]
    if not in_place:
        assert ln.tolist() == lens and int(nf) == n_free
    for g, w in zip(got, want[3:]):
        assert g.tolist() == w
    return want


def batch_of(seed, S, width, P, most_new, spare, holes=False):
    g = torch.Generator().manual_seed(seed)
    r = lambda lo, hi: torch.randint(lo, hi + 1, (S,), generator=g).tolist()
    lens = [min(n, width * P) for n in r(0, width * P)]
    n_new = r(0, most_new)
    held = [-(-n // P) for n in lens]
    n_pages = sum(held) + spare
    order = torch.randperm(n_pages, generator=g).tolist()
    table = [[order.pop() if i < k else -1 for i in range(width)] for k in held]
    if holes:
        for s in range(0, S, 3):
            if held[s]:
                table[s][held[s] - 1] = (-1, n_pages, 2 ** 31 - 1)[s % 2 + s % 3 // 2]
    free = order + [-1] * (n_pages - spare)
    return table, lens, n_new, free, spare


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("S,width,P,new,spare", [(1, 1, 16, 1, 1), (1, 4, 16, 20, 5), (7, 6, 32, 40, 9), (48, 12, 16, 1, 60),
                                                 (1023, 3, 16, 4, 900), (1025, 3, 16, 4, 700), (2047, 2, 16, 3, 2000),
                                                 (2049, 2, 16, 1, 2500), (5000, 2, 16, 2, 3000)])
def test_extend(gpu, S, width, P, new, spare, in_place):
    """Every combination of sums cut short: rows, pages, the table's width."""
    table, lens, n_new, free, n_free = batch_of(S + width, S, width, P, new, spare, holes=S > 5)
    total = sum(n_new)
    for n_tokens, n in ((total + 3, n_free), (total // 2, n_free), (total + 3, n_free // 2), (total, 0), (0, n_free)):
        run_extend(gpu, P, table, lens, n_new, free, n, n_tokens, in_place)


@pytest.mark.parametrize("n_tokens", [1023, 1024, 1025, 4095, 4096, 4097, 30000])
def test_extend_prompts(gpu, n_tokens):
    """Prompt chunks: many rows and pages a sequence, on either side of the rows that one workgroup fills."""
    want = run_extend(gpu, 16, [[-1] * 700 for _ in range(9)], [0, 5, 16, 17, 0, 300, 0, 1, 33][:9],
                      [5000, 1, 0, 4000, 300, 700, 11200, 11200, 9000], list(range(5000)), 3000, n_tokens, n_tokens % 2 == 0)
    assert want[3][-1] <= n_tokens


def test_extend_corners(gpu):
    """Negative lengths and numbers, lengths past the table, a count of free pages outside the
    list, free pages that are none, page sizes that are no power of two are the library's alone."""
    run_extend(gpu, 16, [[3, -1], [4, 5], [-1, -1], [6, 7]], [-5, 40, 0, 32], [4, 1, -3, 1], [0, 1, 2, -1, 9, 99, -7, 8], 8, 10)
    run_extend(gpu, 16, [[3, -1], [4, -1]], [16, 16], [1, 1], [0, 1, 2, 5, 6], 99, 4)
    run_extend(gpu, 16, [[3, -1], [4, -1]], [16, 15], [1, 1], [0, 1, 2, 5, 6], -4, 4)
    run_extend(gpu, 16, [[0, -1]], [2 ** 31 - 1], [2 ** 31 - 1], [1], 1, 4)
    # no sequences
    pg = pages(gpu, 4, 16)
    nf = i32([3], gpu)
    got = pg.extend(torch.zeros(0, 2, dtype=torch.int32, device=gpu), i32([], gpu), i32([], gpu), i32([0, 1, 2, -1], gpu), nf, 5)
    assert got[0].tolist() == [0] and int(nf) == 3 and all(t.tolist() == [-1] * 5 for t in got[1:])


def test_extend_graph(gpu):
    """A captured step grows its sequences in place at every replay, as eager calls do."""
    P, S = 16, 5
    pg = pages(gpu, 64, P)
    new, free = i32([1, 3, 0, 16, 1], gpu), i32(list(range(64)), gpu)

    def state():
        return torch.full((S, 12), -1, dtype=torch.int32, device=gpu), i32([0] * S, gpu), i32([64], gpu)

    a, b = state(), state()
    ws = pg.extend_workspace(S)
    outs = pg.extend(*a[:2], new, free, a[2], 30, workspace=ws)
    pg.extend(*b[:2], new, free, b[2], 30)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        pg.extend(*a[:2], new, free, a[2], 30, new_start=outs[0], pos=outs[1], seq=outs[2], slots=outs[3], workspace=ws)
    for _ in range(13):
        graph.replay()
        torch.cuda.synchronize()
        want = pg.extend(*b[:2], new, free, b[2], 30)
        assert all(torch.equal(x, y) for x, y in zip((*a, *outs), (*b, *want)))
    assert b[1].tolist()[3] == 192          # its row is full


# ---------------------------------------------------------------- rope

def run_rope(gpu, seed, T, n_head, n_kv, D, rot, half, tag, norm, weights=True, magnitude=1.0, pos=None, eps=1e-6, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    qkv = (scale * torch.randn(T, n_head + 2 * n_kv + 1, D, generator=g)).to(DT[tag])
    q, k = qkv[:, :n_head], qkv[:, n_head:n_head + n_kv]
    wq, wk = ((1 + 0.3 * torch.randn(D, generator=g)) if weights else None for _ in range(2))
    pos = torch.randint(0, 40000, (T,), generator=g, dtype=torch.int32) if pos is None else pos
    freq, _ = la.rope_frequencies(rot, device="cpu") if rot else (None, 1)
    to = lambda t: None if t is None else t.to(gpu)
    dq = qkv.to(gpu)
    out_q = torch.full((T, n_head + 1, D), 5.0, dtype=DT[tag], device=gpu)[:, :n_head]
    got = la.qk_rope(dq[:, :n_head], dq[:, n_head:n_head + n_kv] if n_kv else None, pos.to(gpu), to(freq), q_weight=to(wq),
                     k_weight=to(wk), norm=norm, eps=eps, magnitude=magnitude, layout=la.ROPE_HALF if half else la.ROPE_PAIRS,
                     q_out=out_q)
    for x, w, y in ((q, wq, got[0]), (k, wk, got[1])):
        if y is None:
            continue
        want, tol = ref.rope(x, pos, freq, w, norm, eps, magnitude, half, tag)
        live = pos >= 0
        off = (y.cpu().double() - want).abs()[live]
        assert (off <= tol[live] + (2 ** -25 if tag == la.F16 else 0)).all(), f"off by {float((off / (tol[live] + 1e-30)).max()):.3g} of the bound"
    assert torch.equal(dq.cpu(), qkv)
    return got


@pytest.mark.parametrize("norm", [True, False])
@pytest.mark.parametrize("half", [True, False])
@pytest.mark.parametrize("D,rot", [(64, 64), (96, 96), (96, 24), (128, 32), (192, 192), (256, 64), (512, 512), (512, 0), (80, 20),
                                   (10, 6), (7, 2), (1, 0), (333, 130)])
@pytest.mark.parametrize("tag", [la.F32, la.F16, la.BF16])
def test_rope(gpu, tag, D, rot, half, norm):
    """Every type, both layouts, heads of vectors and odd ones, whole, part and none of a head turned."""
    run_rope(gpu, D + rot, 5, 3, 2, D, rot, half, tag, norm, magnitude=1.25)


@pytest.mark.parametrize("T,n_head,n_kv", [(1, 1, 0), (1, 16, 8), (2047, 3, 1), (2048, 3, 1), (2049, 5, 3), (3, 300, 7)])
def test_rope_shapes(gpu, T, n_head, n_kv):
    """One token and many, both sides of the change to several tokens a workgroup, many heads."""
    run_rope(gpu, T, T, n_head, n_kv, 128, 128, True, la.BF16, True)
    run_rope(gpu, T, T, n_head, n_kv, 64, 32, False, la.F32, True)


def test_rope_far_positions(gpu):
    """Positions up to 2^31 - 1, and the first."""
    pos = torch.tensor([0, 1, 131071, 1000003, 16777217, 2 ** 31 - 1], dtype=torch.int32)
    run_rope(gpu, 1, 6, 2, 1, 64, 64, True, la.F32, False, pos=pos)


def test_rope_rows_left(gpu):
    """Rows of a negative position are neither read nor written, in place or not; a turned pair of the others only."""
    D, pos = 64, torch.tensor([3, -1, 7, -2 ** 31, 0], dtype=torch.int32)
    g = torch.Generator().manual_seed(3)
    x = torch.randn(5, 2, D, generator=g)
    x[1], x[3] = float("nan"), float("inf")
    freq, _ = la.rope_frequencies(D, device=gpu)
    dx, out = x.to(gpu), torch.full((5, 2, D), 9.0, device=gpu)
    la.qk_rope(dx, None, pos.to(gpu), freq, q_out=out)
    assert (out[[1, 3]] == 9).all() and torch.isfinite(out).all()
    la.qk_rope(dx, None, pos.to(gpu), freq, q_out=dx)
    assert torch.equal(dx[[0, 2, 4]], out[[0, 2, 4]]) and torch.isnan(dx[1]).all() and torch.isinf(dx[3]).all()


@pytest.mark.parametrize("T", [3, 4097])
@pytest.mark.parametrize("tag,D,rot,half", [(la.F32, 128, 128, True), (la.BF16, 128, 64, False), (la.F16, 80, 20, True), (la.BF16, 96, 24, False)])
def test_rope_in_place(gpu, tag, D, rot, half, T):
    """Queries and keys of a fused projection where they lie: as elsewhere bit for bit, values as they were."""
    qkv = torch.randn(T, 3 + 2 + 2, D, generator=torch.Generator().manual_seed(D + T)).to(DT[tag]).to(gpu)
    freq, _ = la.rope_frequencies(rot, device=gpu)
    pos, layout = torch.arange(7, T + 7, dtype=torch.int32, device=gpu), la.ROPE_HALF if half else la.ROPE_PAIRS
    q, k, v = qkv[:, :3], qkv[:, 3:5], qkv[:, 5:].clone()
    want = la.qk_rope(q, k, pos, freq, layout=layout)
    la.qk_rope(q, k, pos, freq, layout=layout, q_out=q, k_out=k)
    assert torch.equal(q, want[0]) and torch.equal(k, want[1]) and torch.equal(qkv[:, 5:], v)


def test_rope_norms(gpu):
    """Without weights, rows of zeros, a large eps, values whose squares are small; norms alone without positions."""
    run_rope(gpu, 4, 4, 2, 1, 128, 128, True, la.F32, True, weights=False)
    run_rope(gpu, 5, 4, 2, 1, 128, 64, False, la.F32, True, eps=3.0)
    run_rope(gpu, 6, 4, 2, 1, 128, 64, False, la.F32, True, scale=1e-6, eps=1e-12)
    z = torch.zeros(3, 2, 64, device=gpu)
    freq, _ = la.rope_frequencies(64, device=gpu)
    assert (la.qk_rope(z, None, i32([1, 2, 3], gpu), freq)[0] == 0).all()
    x = torch.randn(3, 2, 64, device=gpu)
    want, tol = ref.rope(x.cpu(), None, None, None, True, 1e-6, 1.0, True, la.F32)
    assert ((la.qk_rope(x)[0].cpu().double() - want).abs() <= tol).all()


def test_rope_unaligned(gpu):
    """Rows that start at any value."""
    base = torch.randn(1 + 4 * 301, device=gpu).half()
    x = base[1:].as_strided((4, 2, 128), (301, 128, 1), 1)
    freq, _ = la.rope_frequencies(128, device=gpu)
    pos = i32([5, 6, 7, 8], gpu)
    got, _ = la.qk_rope(x, None, pos, freq)
    assert torch.equal(got, la.qk_rope(x.contiguous(), None, pos, freq)[0])


def test_rope_graph_and_stream(gpu):
    freq, _ = la.rope_frequencies(64, device=gpu)
    q, k, pos = torch.randn(4, 3, 64, device=gpu), torch.randn(4, 1, 64, device=gpu), i32([1, 2, 3, 4], gpu)
    qo, ko = la.qk_rope(q, k, pos, freq)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        la.qk_rope(q, k, pos, freq, q_out=qo, k_out=ko)
    for _ in range(3):
        pos.add_(1000)
        qo.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        want = la.qk_rope(q, k, pos, freq)
        assert torch.equal(qo, want[0]) and torch.equal(ko, want[1])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = la.qk_rope(q, k, pos, freq)
    side.synchronize()
    assert torch.equal(got[0], want[0])


# -------------------------------------------------------------- sample

def run_sample(gpu, logits, u, temperature=None, top_k=None, top_p=None, min_p=None):
    dev = lambda v, t: None if v is None else torch.tensor(v, dtype=t).to(gpu)
    S, V = logits.shape
    wide = torch.full((S, V + 5), 50.0, dtype=logits.dtype)
    wide[:, 2:2 + V] = logits
    wide = wide.to(gpu)
    probs = torch.full((S, V + 3), 7.0, dtype=logits.dtype, device=gpu)
    args = (dev(temperature, torch.float32), dev(top_k, torch.int32), dev(top_p, torch.float32), dev(min_p, torch.float32))
    got = la.sample(wide[:, 2:2 + V], f32(u, gpu), *args, probs=probs[:, 1:1 + V])
    up = lambda v: None if v is None else torch.tensor(v, dtype=torch.float32).tolist()
    tokens, want = ref.sample(logits, f32(u, "cpu"), up(temperature), top_k, up(top_p), up(min_p))
    assert got.tolist() == tokens
    # rounded once; fp16's least step
    tag = {v: k for k, v in DT.items()}[logits.dtype]
    p = probs[:, 1:1 + V].cpu().double()
    off = (p - want).abs()
    assert (off <= want * (EPS[tag] + 1e-12) + (2 ** -25 if tag == la.F16 else 2 ** -63)).all(), float(off.max())
    assert (probs[:, 0] == 7).all() and (probs[:, 1 + V:] == 7).all()
    # without probabilities, and again
    for _ in range(2):
        assert la.sample(wide[:, 2:2 + V], f32(u, gpu), *args).tolist() == tokens
    return tokens, want


def logits_of(seed, S, V, tag, width=2.5):
    g = torch.Generator().manual_seed(seed)
    x = width * torch.randn(S, V, generator=g)
    x[:, ::max(V // 7, 1)] += 5
    return x.to(DT[tag]), torch.rand(S, generator=g).tolist()


@pytest.mark.parametrize("V", [1, 2, 37, 1000, 2048, 2049, 32003, 32768, 32769, 128001])
@pytest.mark.parametrize("tag", [la.F32, la.F16, la.BF16])
def test_sample(gpu, tag, V):
    """Each filter alone, pairs, all and none, sizes around segments and chunks, types whose values tie."""
    settings = [(1.0, 0, 1.0, 0.0), (0.7, 40, 1.0, 0.0), (1.0, 0, 0.9, 0.0), (1.3, 0, 1.0, 0.05), (0.8, 40, 0.95, 0.05), (1.0, 1000, 0.999, 0.0),
                (0.0, 5, 0.5, 0.5), (2.0, 1, 0.9, 0.0), (0.3, 3, 0.3, 0.0), (5.0, 500, 0.5, 0.001), (1.0, 10 ** 9, 0.01, 1.0), (0.1, 2000, 0.9999, 0.0)]
    x, u = logits_of(V, len(settings), V, tag)
    run_sample(gpu, x, u, *zip(*settings))


@pytest.mark.parametrize("S", [1, 3, 64])
def test_sample_large(gpu, S):
    x, u = logits_of(S, S, 262144, la.F32, 2.2)
    run_sample(gpu, x, u, [1.0] * S, [64 * (i % 3) for i in range(S)], [(0.9, 0.99, 1.0)[i % 3 - 1] for i in range(S)], None)


@pytest.mark.parametrize("S,V", [(32, 65536), (33, 65536), (32, 65537), (1, 2097152), (2, 2100001)])
def test_sample_borders(gpu, S, V):
    """Either side of the rows that go to more workgroups, and of the segments that a thread has one of."""
    x, u = logits_of(V + S, S, V, la.BF16, 2.2)
    run_sample(gpu, x, u, None, [(50, 0, 1000)[i % 3] for i in range(S)], [(0.9, 0.99)[i % 2] for i in range(S)], [(0.0, 0.01)[i % 2] for i in range(S)])


@pytest.mark.parametrize("V", [700, 3001, 6000, 8192, 8193, 30000])
def test_sample_flat(gpu, V):
    """Values so near each other that all may be the last kept: candidates up to what is held at once, and more."""
    x = 0.03 * torch.rand(4, V, generator=torch.Generator().manual_seed(V))
    run_sample(gpu, x, [0.3, 0.999, 0.5, 0.0], None, [0, V // 3, V // 3, 1], [0.5, 1.0, 0.7, 0.5], [0.0, 0.0, 0.985, 0.0])


@pytest.mark.parametrize("V", [300, 5000, 60000, 100000])
def test_sample_many_ties(gpu, V):
    """Hundreds and thousands of equal values where a filter ends: the first indices are kept, whichever filter it is."""
    g = torch.Generator().manual_seed(V)
    x = torch.randint(-40, 1, (6, V), generator=g) / 8.0
    x[3] = torch.where(torch.arange(V) % 3 > 0, 1.0, -3.0)
    x[4, V // 2:] = 0.25
    k = [V // 3, 0, V // 2, V // 2, V // 5, 0]
    p = [1.0, 0.6, 0.8, 0.7, 0.9, 0.35]
    for tag in (la.F32, la.BF16):
        run_sample(gpu, x.to(DT[tag]), [0.1, 0.999, 0.5, 0.7, 0.999, 0.3], [1.0, 1.0, 2.0, 1.0, 0.5, 3.0], k, p)


@pytest.mark.parametrize("V,k,p", [(20000, 7000, 1.0), (20000, 0, 0.4), (20000, 9000, 0.5), (5000, 4999, 0.999), (70000, 69999, 0.7),
                                   (4096, 100, 0.5), (4097, 4000, 0.9)])
def test_sample_ties(gpu, V, k, p):
    """Equal logits: the first indices are kept, by candidates that are sorted and by more than that."""
    x = torch.full((3, V), 1.5)
    x[1, V // 3::5] = 2.0
    x[2] = torch.randint(0, 3, (V,), generator=torch.Generator().manual_seed(V)) / 64.0
    _, want = run_sample(gpu, x, [0.1, 0.9, 0.5], None, [k] * 3, [p] * 3)
    if p == 1.0:
        assert (want[0, :k] > 0).all() and (want[0, k:] == 0).all()


def test_sample_values(gpu):
    """NaN and infinities, rows without a value, zeros of both signs, far temperatures and settings off the scale."""
    inf, nan, V = math.inf, math.nan, 300
    x = torch.randn(12, V, generator=torch.Generator().manual_seed(5))
    x[0] = -inf
    x[1] = nan
    x[2, ::2] = nan
    x[3, 1::3] = -inf
    x[4, [7, 90]] = inf
    x[5, 10:] = -inf
    x[6] = 0.0
    x[6, ::2] = -0.0
    x[7] *= 1e30
    x[8] *= 1e-30
    x[9, 5] = 3e38
    x[10, 5] = -3e38
    u = [0.5, 0.5, 0.7, 0.2, 0.6, 0.99, 0.4, 0.5, 0.3, 0.9, 0.1, 0.0]
    for k, p, m in ((0, 1.0, 0.0), (5, 1.0, 0.0), (0, 0.8, 0.0), (20, 0.9, 0.1), (1, 1.0, 0.0), (-3, 1.5, -1.0), (10, 0.0, 0.0), (10, -1.0, 0.0), (0, 1.0, 1.0),
                    (0, 1.0, 1.5), (2 ** 31 - 1, 0.5, 0.0)):
        for t in (1.0, 0.0, -1.0, 1e-40, 1e30, inf, nan):
            run_sample(gpu, x, u, [t] * 12, [k] * 12, [p] * 12, [m] * 12)
    # settings that are no numbers are off
    a = run_sample(gpu, x, u, None, [5] * 12, [nan] * 12, [nan] * 12)
    assert a[0] == run_sample(gpu, x, u, None, [5] * 12)[0]


def test_sample_draws(gpu):
    """u of 0, next to 1, and outside [0, 1): the first and the last kept value."""
    x, _ = logits_of(8, 6, 5000, la.F32)
    run_sample(gpu, x, [0.0, 1 - 2 ** -24, 1.0, 7.0, -0.5, 0.5], None, [50] * 6)
    run_sample(gpu, x, [0.0, 1 - 2 ** -24, 1.0, 7.0, -0.5, 0.5])
    # every value is drawn where its share of u is
    y = torch.tensor([[1.0, 2.0, 0.5, 3.0]]).log().expand(13, 4).contiguous()
    got, _ = run_sample(gpu, y, [(i + 0.5) / 13 for i in range(13)])
    assert got == [0] * 2 + [1] * 4 + [2] + [3] * 6


def test_sample_feeds_verification(gpu):
    """Drafts sampled with their probabilities, then verified against the same model's: all are taken."""
    S, V = 4, 3001
    x, u = logits_of(9, S, V, la.F32)
    x = x.to(gpu)
    probs = torch.empty(S, V, device=gpu)
    k = i32([50] * S, gpu)
    d = la.sample(x, f32(u, gpu), top_k=k, probs=probs)
    target = torch.stack([probs, probs], 1)
    tokens, accepted = la.verify_drafts(target, probs[:, None], d[:, None].contiguous(), f32([[0.99]] * S, gpu), f32(u, gpu))
    assert accepted.tolist() == [1] * S and torch.equal(tokens[:, 0], d)
    assert torch.equal(tokens[:, 1], d)                 # the same u, the same probabilities


def test_sample_graphs_share_a_workspace(gpu):
    x = [logits_of(i, 3, 40000 + i, la.BF16)[0].to(gpu) for i in range(2)]
    u, p = f32([0.2, 0.6, 0.9], gpu), f32([0.9, 0.95, 1.0], gpu)
    ws = la.sample_workspace(3, 40001, gpu)
    toks, graphs = [], []
    for y in x:
        tok = la.sample(y, u, top_p=p, workspace=ws)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            la.sample(y, u, top_p=p, tokens=tok, workspace=ws)
        toks.append(tok)
        graphs.append(g)
    for step in range(4):
        for y, tok, g in zip(x, toks, graphs):
            tok.fill_(-5)
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(tok, la.sample(y, u, top_p=p))
        u.mul_(0.7)


# ------------------------------------------------------------ together

class Serve:
    """A serving step of a two-layer model, from its tokens to the next ones: pages and
    slots, norms and rotary positions, the cache, attention behind a shared prefix, sampling.  `check`
    compares every stage with its 64-bit form on the stage's own inputs."""
    V, H, N, D, P, WIDTH = 700, 2, 6, 64, 16, 12

    def __init__(self, gpu, n_seq):
        g = torch.Generator().manual_seed(901)
        mat = lambda *s: (torch.randn(*s, generator=g) / math.sqrt(s[0])).to(gpu)
        d = 96
        self.gpu, self.n_seq, self.n_pages = gpu, n_seq, n_seq * self.WIDTH
        self.emb, self.head = mat(self.V, d) * math.sqrt(self.V), 5 * mat(d, self.V)
        self.layers = [dict(qkv=mat(d, (self.N + 2 * self.H) * self.D), o=mat(self.N * self.D, d),
                            wq=(1 + 0.2 * torch.randn(self.D, generator=g)).to(gpu), wk=(1 + 0.2 * torch.randn(self.D, generator=g)).to(gpu),
                            cache=la.KvCache.empty(self.n_pages, self.P, self.H, self.D, la.F16, gpu)) for _ in range(2)]
        self.pages = la.KvPages([l["cache"] for l in self.layers])
        self.freq, self.magnitude = la.rope_frequencies(self.D, 500000.0, la.ROPE_YARN, 8.0, 64.0, device=gpu)

    def state(self):
        S, dev = self.n_seq, self.gpu
        return dict(table=torch.full((S, self.WIDTH), -1, dtype=torch.int32, device=dev), lens=i32([0] * S, dev),
                    free=i32(list(range(self.n_pages)), dev), n_free=i32([self.n_pages], dev), tokens=i32([3 + 5 * i for i in range(S)], dev),
                    probs=torch.zeros(S, self.V, device=dev), groups=i32([0, 0], dev), prefix=i32([0], dev), u=f32([0.0] * S, dev))

    def step(self, s, tokens, n_new, T, max_new, check=False):
        """tokens [T] of the new rows; their logits [T, V]"""
        before = check and [s[k].tolist() for k in ("table", "lens")] + [n_new.tolist(), s["free"].tolist(), int(s["n_free"])]
        start, pos, seq, slots = self.pages.extend(s["table"], s["lens"], n_new, s["free"], s["n_free"], T)
        if check:
            want = ref.extend(*before, T, self.P, self.n_pages)
            assert [s["table"].tolist(), s["lens"].tolist(), int(s["n_free"]), start.tolist(), pos.tolist(), seq.tolist(), slots.tolist()] == list(want)
        batch = la.KvBatch(s["table"], s["lens"], start, n_tokens=T, max_new=max_new)
        x = self.emb[tokens.long()]
        for l in self.layers:
            qkv = (x @ l["qkv"]).view(T, self.N + 2 * self.H, self.D)
            q, k, v = qkv[:, :self.N], qkv[:, self.N:self.N + self.H], qkv[:, self.N + self.H:]
            q2, k2 = la.qk_rope(q, k, pos, self.freq, l["wq"], l["wk"], magnitude=self.magnitude)
            l["cache"].append(batch, k2, v)
            a = l["cache"].prefix_attention(batch, q2, s["groups"], s["prefix"], out=torch.zeros_like(q2))
            if check:
                rows = int(start[-1])
                for raw, w, y in ((q, l["wq"], q2), (k, l["wk"], k2)):
                    want, tol = ref.rope(raw.cpu(), pos.cpu(), self.freq.cpu(), w.cpu(), True, 1e-6, self.magnitude, True, la.F32)
                    assert ((y.cpu().double() - want).abs() <= tol)[:rows].all()
                flat = lambda t: t.transpose(1, 2).reshape(-1, self.H, self.D)
                at = slots[:rows].long()
                assert torch.equal(flat(l["cache"].k)[at], k2[:rows].half())
                assert torch.equal(flat(l["cache"].v.transpose(2, 3))[at], v[:rows].half())
                want, _, tol = step_ref.attention(l["cache"], s["table"].tolist(), s["lens"].tolist(), start.tolist(), q2.cpu(), self.D ** -0.5)
                # (the prefix's sums are joined by their logarithms, which stays within twice the bound)
                assert ((a.cpu().double() - want).abs() <= 2 * tol)[:rows].all()
            x = x + a.reshape(T, -1) @ l["o"]
        return start, x @ self.head

    def sample(self, s, logits, check=False):
        la.sample(logits, s["u"], s.get("temperature"), s.get("top_k"), s.get("top_p"), s.get("min_p"), tokens=s["tokens"], probs=s["probs"])
        if check:
            cpu = lambda k: s[k].tolist() if k in s else None
            tokens, want = ref.sample(logits.cpu(), s["u"].cpu(), cpu("temperature"), cpu("top_k"), cpu("top_p"), cpu("min_p"))
            assert s["tokens"].tolist() == tokens
            assert ((s["probs"].cpu().double() - want).abs() <= want * (EPS[la.F32] + 1e-12) + 2 ** -63).all()


def test_serving_steps_together(gpu):
    """One user's prompt in chunks, forked for parallel samples and another user's beside it; decode
    steps behind the shared prefix; a verify step whose refused draft leaves; and decode steps as a
    graph, replay by replay against eager steps of a twin."""
    S = 5
    m = Serve(gpu, S)
    s = m.state()
    g = torch.Generator().manual_seed(902)
    draw = lambda n: torch.randint(0, m.V, (n,), generator=g, dtype=torch.int32).to(gpu)
    # 45 tokens of sequence 0 and 19 of sequence 4, 16 at most a call, a row of each call unused
    for a, b in ((16, 16), (16, 3), (13, 0)):
        m.step(s, draw(a + b + 1), i32([a, 0, 0, 0, b], gpu), a + b + 1, 16, True)
    # rows 1 to 3 go on from sequence 0: its two full pages are theirs too
    _, free, n_free = m.pages.refs(s["table"], s["lens"])
    spare = free[:3].tolist()
    m.pages.fork(s["table"], s["lens"], i32([[0, i + 1, spare[i]] for i in range(3)], gpu))
    refs, s["free"], s["n_free"] = m.pages.refs(s["table"], s["lens"])
    assert s["lens"].tolist() == [45] * 4 + [19] and refs.max() == 4 and int(s["n_free"]) == m.n_pages - (2 + 4 + 2)
    s["groups"], s["prefix"] = i32([0, 4], gpu), i32([32], gpu)
    s.update(temperature=f32([0.8, 1.0, 0.0, 1.5, 0.7], gpu), top_k=i32([0, 40, 0, 7, 0], gpu), top_p=f32([0.9, 1.0, 1.0, 0.8, 1.0], gpu),
             min_p=f32([0.0, 0.05, 0.0, 0.0, 0.02], gpu))
    one = i32([1] * S, gpu)
    for _ in range(4):
        s["u"] = torch.rand(S, generator=g).to(gpu)
        _, logits = m.step(s, s["tokens"], one, S, 1, True)
        m.sample(s, logits, True)
    # two tokens a sequence, the second a draft, verified against the model's probabilities after the filters
    last, lens = s["tokens"].clone(), s["lens"].clone()
    drafts, u, u_next = s["tokens"][:, None].roll(1, 0).contiguous(), torch.rand(S, 1, generator=g).to(gpu), torch.rand(S, generator=g).to(gpu)
    start, logits = m.step(s, torch.stack([last, drafts[:, 0]], 1).flatten(), i32([2] * S, gpu), 2 * S, 2, True)
    probs = torch.empty(2 * S, m.V, device=gpu)
    two = {k: s[k].repeat_interleave(2) for k in ("temperature", "top_k", "top_p", "min_p", "u")}
    la.sample(logits, two["u"], two["temperature"], two["top_k"], two["top_p"], two["min_p"], probs=probs)
    s["tokens"], accepted = la.verify_drafts(probs.view(S, 2, m.V), None, drafts, u, u_next)
    want, taken = step_ref.verify(probs.view(S, 2, m.V).cpu(), None, drafts.cpu(), u.cpu(), u_next.cpu(), None)
    assert s["tokens"].tolist() == want and accepted.tolist() == taken
    s["tokens"] = s["tokens"].gather(1, accepted[:, None].long())[:, 0].contiguous()
    s["lens"].copy_(lens + 1 + accepted)
    _, s["free"], s["n_free"] = m.pages.refs(s["table"], s["lens"])
    # the step as a graph, across page ends, and a twin of everything in eager steps
    twin = Serve(gpu, S)
    for x, y in zip(m.layers, twin.layers):
        y["cache"].k.copy_(x["cache"].k)
        y["cache"].v.copy_(x["cache"].v)
    t = {k: v.clone() for k, v in s.items()}

    def run(m, s):
        _, logits = m.step(s, s["tokens"], one, S, 1)
        m.sample(s, logits)

    warm = {k: v.clone() for k, v in s.items()}
    run(twin, warm)                     # (its pages' rows are written again by the first step, alike)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run(m, s)
    for i in range(20):
        for x in (s, t):
            x["u"].copy_(torch.rand(S, generator=torch.Generator().manual_seed(i)))
        graph.replay()
        torch.cuda.synchronize()
        run(twin, t)
        for k in ("table", "lens", "n_free", "tokens", "probs"):
            assert torch.equal(s[k], t[k]), (i, k)
    assert s["lens"].tolist() == (lens + 1 + accepted + 20).tolist()
    assert all(torch.equal(x["cache"].k, y["cache"].k) and torch.equal(x["cache"].v, y["cache"].v) for x, y in zip(m.layers, twin.layers))


def test_threads_and_streams_at_once(gpu):
    """Host threads with a stream and workspaces of their own run every operator at once: as
    each does alone, bit for bit, and a refusal is its own thread's."""
    import threading
    S = 6
    models = [Serve(gpu, S) for _ in range(2)]
    logits = torch.randn(2, 3, 50001, generator=torch.Generator().manual_seed(903)).to(gpu)
    u, k = f32([0.1, 0.5, 0.9], gpu), i32([50, 0, 3], gpu)

    def work(i):
        m = models[i]
        s = m.state()
        s["u"].fill_(0.3 + 0.2 * i)
        one = i32([1] * S, gpu)
        for _ in range(4):
            _, x = m.step(s, s["tokens"], one, S, 1)
            m.sample(s, x)
        return [s["table"], s["lens"], s["tokens"], s["probs"], la.sample(logits[i], u, top_k=k)]

    alone = [work(i) for i in range(2)]
    torch.cuda.synchronize()
    failed = []

    def thread(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(10):
                    got = work(i)
                    with pytest.raises((ValueError, la.LlapisError), match="layout" if i else "workspace"):
                        if i:
                            la.qk_rope(torch.zeros(1, 2, 64, device=gpu), pos=i32([0], gpu), freq=models[0].freq, layout=7)
                        else:
                            la.sample(logits[i], u, workspace=torch.zeros(8, dtype=torch.uint8, device=gpu))
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


# ------------------------------------------------- borders far below the largest value

def exact_kept(x, k, p):
    """The indices that top_k and top_p keep of a row (float64, no NaN), their weights as whole numbers of 2^-200, and how
    far the border is from another one, in weights of its value"""
    z, order = torch.sort(x, descending=True, stable=True)
    z, order = z[:k] if k else z, order[:k] if k else order
    w = [int(math.ldexp(v, 200)) for v in (z - z[0]).exp().tolist()]
    num, den = p.as_integer_ratio()
    goal, n, upto = num * sum(w), 0, 0
    while upto * den < goal:
        upto += w[n]
        n += 1
    near = min(upto * den - goal, goal - (upto - w[n - 1]) * den) / (w[n - 1] * den)
    return order[:n], w[:n], near


def deep(kind, V, depth, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.full((V,), -float(depth))
    if kind == "band":
        x -= 0.02 * torch.rand(V, generator=g)
    if kind == "few":
        x[torch.randperm(V, generator=g)[8000:]] = -math.inf
    if kind == "tail":
        x = 2.5 * torch.randn(V, generator=g) - depth
    x[V // 3] = 0.0
    return x


@pytest.mark.parametrize("kind,V,depth,k,p", [
    ("equal", 1 << 18, 20.5, 0, 0.9999), ("equal", 1 << 20, 23.25, 0, 0.99995), ("equal", 1 << 18, 16, 0, 0.98), ("equal", 1 << 20, 24, 0, 0.99999),
    ("equal", 1 << 18, 20.25, 200000, 0.9999), ("equal", 60000, 19, 0, 0.9999), ("equal", 2100001, 22, 0, 0.9999),
    ("band", 1 << 18, 20.8, 0, 0.9999), ("band", 10 ** 6, 21, 0, 0.9997), ("band", 1 << 18, 18, 0, 0.999), ("band", 30000, 18, 0, 0.9999),
    ("band", 10 ** 6, 22, 900001, 0.9999), ("band", 2100001, 24, 0, 0.99999), ("tail", 1 << 18, 12, 0, 0.9999999), ("tail", 10 ** 6, 20, 0, 0.999999),
    ("tail", 2100001, 16, 0, 0.99999), ("few", 70000, 24.59375, 0, 1 - 2 ** -24), ("few", 70000, 24.90625, 0, 1 - 2 ** -24),
    ("few", 70000, 24.21875, 0, 1 - 2 ** -22), ("few", 70000, 20.0, 0, 1 - 2 ** -17)])
def test_sample_border_below_a_dominant_value(gpu, kind, V, depth, k, p):
    """One value has nearly all of the weight and top_p ends among thousands to millions 16 to 25 below it, as many as
    are held at once and more.  Their weights' sum decides to a small part of one of them (checked here), so the kept sets are equal."""
    p = float(torch.tensor(p, dtype=torch.float32))
    for tag in (la.F32, la.BF16) if kind == "equal" else (la.F32,):
        x = deep(kind, V, depth, V).to(DT[tag])
        want, w, near = exact_kept(x.double(), k, p)
        assert 1 < len(want) < V and near > 1e-3
        probs = torch.empty(1, V, dtype=DT[tag], device=gpu)
        u = 1.0 - 2.0 ** -22
        tok = la.sample(x[None].to(gpu), f32([u], gpu), top_k=i32([k], gpu), top_p=f32([p], gpu), probs=probs)
        got = (probs[0] > 0).nonzero()[:, 0].cpu()
        assert len(got) == len(want), (len(got), len(want))
        assert torch.equal(got, want.sort().values)
        # the first at which the sum passes u of the whole
        num, den = u.as_integer_ratio()
        goal, upto = num * sum(w), 0
        for v, i in sorted(zip(want.tolist(), w)):
            upto += i
            if upto * den > goal:
                break
        assert int(tok) == v


@pytest.mark.parametrize("tag", [la.F16, la.BF16])
def test_sample_probabilities_are_rounded_once(gpu, tag):
    """Probabilities next to the middle of two 16-bit numbers, nearer than fp32 tells: temperatures at which the first of
    two values has one 2^-34 to 2^-26 above or below it."""
    step, half = EPS[tag], 0.5
    temps, want = [], []
    for i in range(1, 60):
        middle = half + (i + 0.5) * step                  # (numbers from 1/2 to 1 are EPS apart)
        t0 = torch.tensor(half / math.log(middle / (1 - middle)), dtype=torch.float32)
        for j in range(-40, 41):
            t = float((t0.view(torch.int32) + j).view(torch.float32))
            p = 1 / (1 + math.exp(-half / t))
            if 2 ** -34 < abs(p - middle) < 2 ** -26:
                temps.append(t)
                want.append(half + (i + (p > middle)) * step)
    assert len(temps) > 300
    x = torch.tensor([[half, 0.0]], dtype=DT[tag]).expand(len(temps), 2).contiguous().to(gpu)
    probs = torch.empty_like(x)
    la.sample(x, f32([0.5] * len(temps), gpu), f32(temps, gpu), probs=probs)
    assert probs[:, 0].double().tolist() == want


def test_serving_steps_behind_a_prefix_that_is_read_once(gpu):
    """Parallel samples of one prompt of 140 tokens and another user beside them: the samples' first 128 are read once (two
    units, where what is not a multiple of 64 is each one's own).  Every stage is held to its own bound, attention to that of
    attention without a prefix; then the step as a graph against a twin's eager steps."""
    S = 5
    m = Serve(gpu, S)
    s = m.state()
    g = torch.Generator().manual_seed(904)
    draw = lambda n: torch.randint(0, m.V, (n,), generator=g, dtype=torch.int32).to(gpu)
    for n in [16] * 8 + [12]:
        m.step(s, draw(n + 2), i32([n, 0, 0, 0, 2], gpu), n + 2, 16, True)
    _, free, n_free = m.pages.refs(s["table"], s["lens"])
    spare = free[:3].tolist()
    m.pages.fork(s["table"], s["lens"], i32([[0, i + 1, spare[i]] for i in range(3)], gpu))
    _, s["free"], s["n_free"] = m.pages.refs(s["table"], s["lens"])
    s["groups"], s["prefix"] = i32([0, 4], gpu), i32([128], gpu)
    s.update(temperature=f32([0.8, 1.0, 0.0, 1.5, 0.7], gpu), top_k=i32([0, 40, 0, 7, 0], gpu), top_p=f32([0.9, 1.0, 1.0, 0.8, 1.0], gpu))
    one, seen = i32([1] * S, gpu), []

    def within_the_bound(cache):
        plain = cache.prefix_attention

        def call(batch, q, groups, prefix, out):
            a = plain(batch, q, groups, prefix, out=out)
            rows = int(batch.new_start[-1])
            want, _, tol = step_ref.attention(cache, s["table"].tolist(), s["lens"].tolist(), batch.new_start.tolist(), q.cpu(), m.D ** -0.5)
            assert ((a.cpu().double() - want).abs() <= tol)[:rows].all()
            # what the samples' rows of the table hold within the prefix is not looked at but in the first of them
            other = s["table"].clone()
            other[1:4, :8] = s["table"][4, 0]
            held = la.KvBatch(other, s["lens"], batch.new_start, n_tokens=batch.n_tokens, max_new=batch.max_new)
            assert torch.equal(plain(held, q, groups, prefix, out=torch.zeros_like(q)), a)
            seen.append(rows)
            return a

        return call

    for l in m.layers:
        l["cache"].prefix_attention = within_the_bound(l["cache"])
    for n_new, T in (([1] * S, S), ([1] * S, S), ([2, 1, 3, 0, 1], 8), ([1] * S, S)):
        s["u"] = torch.rand(S, generator=g).to(gpu)
        _, logits = m.step(s, s["tokens"] if T == S else draw(T), i32(n_new, gpu), T, max(n_new), True)
        if T == S:
            m.sample(s, logits, True)
    assert seen == [5, 5, 5, 5, 7, 7, 5, 5]
    twin = Serve(gpu, S)
    for x, y in zip(m.layers, twin.layers):
        del x["cache"].prefix_attention
        y["cache"].k.copy_(x["cache"].k)
        y["cache"].v.copy_(x["cache"].v)
    t = {k: v.clone() for k, v in s.items()}

    def run(m, s):
        _, logits = m.step(s, s["tokens"], one, S, 1)
        m.sample(s, logits)

    run(twin, {k: v.clone() for k, v in s.items()})
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run(m, s)
    for i in range(12):
        for x in (s, t):
            x["u"].copy_(torch.rand(S, generator=torch.Generator().manual_seed(i)))
        graph.replay()
        torch.cuda.synchronize()
        run(twin, t)
        for k in ("table", "lens", "n_free", "tokens", "probs"):
            assert torch.equal(s[k], t[k]), (i, k)


@pytest.mark.parametrize("T", [8191, 8192, 8195])
@pytest.mark.parametrize("tag,D,rot,half", [(la.BF16, 128, 64, True), (la.F16, 80, 20, False), (la.F32, 128, 128, False)])
def test_rope_many_tokens(gpu, tag, D, rot, half, T):
    """Either side of the number of tokens from which a workgroup takes four, of more heads than it has places for."""
    pos = torch.arange(T, dtype=torch.int32) * 3
    run_rope(gpu, T + D, T, 7, 2, D, rot, half, tag, True, pos=pos)
