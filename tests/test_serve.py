"""The operators before and after a step's attention (llapis_step.h) without a GPU: struct
layouts, sizes, rotary frequencies, and the calls that are refused before anything is launched."""
import ctypes as C
import math

import pytest

import llapis_amd as la
from llapis_amd import _lib
from test_abi import INCLUDE, compile_layouts
from test_step import P, refused

STRUCTS = {
    "llapis_kv_extend_args": _lib.LlapisKvExtendArgs, "llapis_rope_rule": _lib.LlapisRopeRule,
    "llapis_qk_rope_args": _lib.LlapisQkRopeArgs, "llapis_sample_args": _lib.LlapisSampleArgs,
    "llapis_kv_prefix": _lib.LlapisKvPrefix,
}


def test_ctypes_mirror_matches_header(tmp_path):
    structs = {k: [f[0] for f in v._fields_] for k, v in STRUCTS.items()}
    got = compile_layouts(tmp_path, str(INCLUDE / "llapis_step.h"), structs)
    for s, cls in STRUCTS.items():
        assert got[(s, "sizeof")] == C.sizeof(cls), s
        for f in structs[s]:
            assert got[(s, f)] == getattr(cls, f).offset, (s, f)


# -------------------------------------------------------------- extend

def extend_args(**kw):
    a = dict(page_size=16, n_pages=8, n_seq=2, n_tokens=4, max_pages=4, table_stride=4, page_table=P, lens=P, n_new=P, free_pages=P,
             n_free=P, lens_out=P, n_free_out=P, new_start=P, pos=P, seq=P, slots=P)
    a.update(kw)
    return _lib.LlapisKvExtendArgs(**a)


@pytest.mark.parametrize("bad", [dict(page_size=0), dict(n_pages=0), dict(n_pages=(1 << 30) + 1), dict(n_seq=-1), dict(n_seq=1 << 24),
                                 dict(n_tokens=-1), dict(n_tokens=(1 << 30) + 1), dict(max_pages=0), dict(table_stride=3),
                                 dict(max_pages=1 << 27, table_stride=1 << 27), dict(page_table=None), dict(lens=None), dict(n_new=None),
                                 dict(free_pages=None), dict(n_free=None), dict(lens_out=None), dict(n_free_out=None),
                                 dict(new_start=None)], ids=str)
def test_extend_refusals(bad):
    a = extend_args(**bad)
    refused(la.lib().llapis_kv_extend(C.byref(a), P, 1 << 40, None), "llapis_kv_extend")


def test_extend_workspace():
    a, lib = extend_args(), la.lib()
    need = lib.llapis_kv_extend_workspace_size(2)
    assert need > 0 and lib.llapis_kv_extend_workspace_size(1 << 24) == 0 == lib.llapis_kv_extend_workspace_size(-1)
    for n in (0, 1, 1000):
        assert 0 < lib.llapis_kv_extend_workspace_size(n) < lib.llapis_kv_extend_workspace_size(n + 1)
    refused(lib.llapis_kv_extend(C.byref(a), P, need - 1, None), "workspace")
    refused(lib.llapis_kv_extend(C.byref(a), P + 2, need, None), "workspace")
    refused(lib.llapis_kv_extend(C.byref(a), None, need, None), "workspace")
    refused(lib.llapis_kv_extend(None, P, need, None), "null")


# ---------------------------------------------------------------- rope

def test_frequencies():
    freq = lambda *a, **kw: (lambda f, m: (f.tolist(), m))(*la.rope_frequencies(*a, device="cpu", **kw))
    f, m = freq(64, 10000.0)
    assert m == 1.0 and f == pytest.approx([10000.0 ** (-i / 32) for i in range(32)], rel=1e-14)
    f2, _ = freq(64, 10000.0, divisors=[1.0 + i for i in range(32)])
    assert f2 == pytest.approx([x / (1 + i) for i, x in enumerate(f)], rel=1e-14)
    assert freq(64, 10000.0, la.ROPE_LINEAR, 4.0)[0] == pytest.approx([x / 4 for x in f], rel=1e-14)
    # the base grows such that the slowest frequency is divided by the factor, the fastest kept
    f3, _ = freq(64, 10000.0, la.ROPE_NTK, 4.0)
    assert f3[0] == 1.0 and f3[-1] == pytest.approx(f[-1] / 4, rel=1e-13)
    # by turns over the trained length: above `high` kept, below `low` divided
    for kind, low, high in ((la.ROPE_YARN, 1.0, 32.0), (la.ROPE_BANDS, 1.0, 4.0)):
        g, m = freq(128, 500000.0, kind, 8.0, 8192.0)
        h, _ = freq(128, 500000.0)
        assert m == pytest.approx(0.1 * math.log(8) + 1 if kind == la.ROPE_YARN else 1.0, rel=1e-7)
        between = 0
        for i, (x, y) in enumerate(zip(g, h)):
            turns = 8192 * y / (2 * math.pi)
            if kind == la.ROPE_BANDS:
                s = min(max((turns - low) / (high - low), 0), 1)
            else:
                at = lambda t: 128 * math.log(8192 / (t * 2 * math.pi)) / (2 * math.log(500000.0))
                lo, hi = math.floor(at(high)), math.ceil(at(low))
                s = 1 - min(max((i - lo) / (hi - lo), 0), 1)
            between += 0 < s < 1
            assert x == pytest.approx(y * s + y / 8 * (1 - s), rel=1e-12), i
        assert between > 2 and g[0] == h[0] and g[-1] == pytest.approx(h[-1] / 8, rel=1e-13)
    # ramps of no width, one pair, no stretching
    assert freq(2, 10000.0, la.ROPE_NTK, 4.0)[0] == [1.0]
    assert freq(2, 10000.0, la.ROPE_YARN, 1.0, 10.0)[1] == 1.0
    assert all(math.isfinite(x) for x in freq(4, 1e6, la.ROPE_YARN, 16.0, 5.0, low=1.0, high=1.5)[0])


@pytest.mark.parametrize("bad", [dict(rot_dim=0), dict(rot_dim=7), dict(rot_dim=514), dict(kind=5), dict(kind=-1), dict(base=1.0),
                                 dict(base=math.nan), dict(base=math.inf), dict(kind=1, factor=0.0), dict(kind=2, factor=math.inf),
                                 dict(kind=3, factor=math.nan), dict(kind=3, factor=2.0), dict(kind=4, factor=2.0, trained=100.0, low=4.0, high=4.0),
                                 dict(kind=4, factor=2.0, trained=100.0, low=0.0, high=4.0)], ids=str)
def test_frequency_refusals(bad):
    a = dict(kind=0, rot_dim=64, base=10000.0, factor=1.0, trained=0.0, low=1.0, high=32.0)
    a.update(bad)
    rule, out, m = _lib.LlapisRopeRule(**a), (C.c_double * 256)(), C.c_float()
    refused(la.lib().llapis_rope_frequencies(C.byref(rule), out, C.byref(m)), "llapis_rope_frequencies")
    assert not any(out) and m.value == 0
    refused(la.lib().llapis_rope_frequencies(None, out, C.byref(m)), "null")
    zero = (C.c_double * 32)()
    rule = _lib.LlapisRopeRule(kind=0, rot_dim=64, base=10000.0, divisors=C.addressof(zero))
    refused(la.lib().llapis_rope_frequencies(C.byref(rule), out, C.byref(m)), "divisors")


def rope_args(**kw):
    a = dict(type=la.F32, n_tokens=2, n_head=4, n_kv=2, head_dim=64, rot_dim=64, layout=0, norm=1, eps=1e-6, magnitude=1.0, pos=P, freq=P,
             q=P, q_stride=256, q_out=P, q_out_stride=256, k=P, k_stride=128, k_out=P, k_out_stride=128)
    a.update(kw)
    return _lib.LlapisQkRopeArgs(**a)


@pytest.mark.parametrize("bad", [dict(type=la.Q8_0), dict(n_tokens=-1), dict(n_tokens=1 << 24), dict(n_head=-1), dict(n_kv=-1), dict(n_head=65537),
                                 dict(n_kv=65537), dict(head_dim=0), dict(head_dim=513), dict(rot_dim=65), dict(rot_dim=66), dict(rot_dim=-2),
                                 dict(layout=2), dict(layout=-1), dict(pos=None), dict(freq=None), dict(q=None), dict(q_out=None), dict(k=None),
                                 dict(k_out=None), dict(q_out_stride=255), dict(k_out_stride=127)], ids=str)
def test_rope_refusals(bad):
    a = rope_args(**bad)
    refused(la.lib().llapis_qk_rope(C.byref(a), None), "llapis_qk_rope")


def test_rope_of_nothing():
    for nothing in (dict(n_tokens=0), dict(n_head=0, n_kv=0)):
        a = rope_args(**nothing)
        assert la.lib().llapis_qk_rope(C.byref(a), None) == 0
    refused(la.lib().llapis_qk_rope(None, None), "null")


# -------------------------------------------------------------- sample

def sample_args(**kw):
    a = dict(type=la.F32, n_seq=2, vocab=100, logits=P, logits_stride=100, u=P, tokens=P, probs=2 * P, probs_stride=100)
    a.update(kw)
    return _lib.LlapisSampleArgs(**a)


@pytest.mark.parametrize("bad", [dict(type=la.Q8_0), dict(n_seq=-1), dict(n_seq=65536), dict(vocab=0), dict(vocab=(1 << 30) + 1), dict(logits=None),
                                 dict(u=None), dict(tokens=None), dict(logits_stride=99), dict(probs_stride=99), dict(probs=P)], ids=str)
def test_sample_refusals(bad):
    a = sample_args(**bad)
    refused(la.lib().llapis_sample(C.byref(a), P, 1 << 50, None), "llapis_sample")


def test_sample_workspace():
    a, lib = sample_args(), la.lib()
    need = lib.llapis_sample_workspace_size(2, 100)
    assert need > 0
    refused(lib.llapis_sample(C.byref(a), P, need - 1, None), "workspace")
    refused(lib.llapis_sample(C.byref(a), P + 8, need, None), "workspace")
    refused(lib.llapis_sample(C.byref(a), None, need, None), "workspace")
    refused(lib.llapis_sample(None, P, need, None), "null")
    a = sample_args(n_seq=0)
    assert lib.llapis_sample(C.byref(a), None, 0, None) == 0
    for s, v in ((0, 10), (65536, 10), (1, 0), (1, (1 << 30) + 1), (-1, 5)):
        assert lib.llapis_sample_workspace_size(s, v) == 0
    # a workspace for more serves less
    for s, v in ((1, 1), (3, 32768), (64, 128001)):
        n = lib.llapis_sample_workspace_size(s, v)
        assert 0 < n <= lib.llapis_sample_workspace_size(s + 1, v) and n <= lib.llapis_sample_workspace_size(s, v + 1)
    assert lib.llapis_sample_workspace_size(65535, 1 << 30) > 1 << 48


# -------------------------------------------------------------- python

def test_python_refuses_host_tensors():
    import torch
    with pytest.raises(ValueError, match="GPU"):
        la.qk_rope(torch.zeros(2, 2, 64))
    with pytest.raises(ValueError, match="GPU"):
        la.sample(torch.zeros(2, 10), torch.zeros(2))


def test_python_checks(monkeypatch):
    """Host tensors stand in for the GPU's, and nothing is called."""
    import torch
    from llapis_amd import step
    called = []
    monkeypatch.setattr(step, "_on_gpu", lambda t, what: t.device)
    monkeypatch.setattr(step, "_call", lambda *a: called.append(a[0]))
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32)
    pages = step.KvPages([step.KvCache.empty(4, 16, 1, 64, la.F16, "cpu")])
    table, lens, new, free, one = i32([0, -1], [1, -1]), i32(3, 4), i32(1, 1), i32(2, 3, -1, -1), i32(2)
    extend = lambda **kw: pages.extend(*(kw.get(k, v) for k, v in (("table", table), ("lens", lens), ("new", new), ("free", free), ("one", one), ("n", 4))),
                                       **{k: v for k, v in kw.items() if k not in ("table", "lens", "new", "free", "one", "n")})
    extend()
    for bad, what in ((dict(table=table.long()), "page_table"), (dict(table=table[:1].expand(2, 2)), "overlap"), (dict(lens=i32(3)), "lens"),
                      (dict(new=i32(1)), "n_new"), (dict(free=i32(2, 3)), "free"), (dict(one=i32(2, 2)), "n_free"), (dict(n=1 << 32), "2\\^31"),
                      (dict(lens_out=i32(3)), "lens_out"), (dict(n_free_out=lens), "n_free_out"), (dict(new_start=lens), "new_start"),
                      (dict(pos=lens), "pos"), (dict(seq=lens), "seq"), (dict(slots=torch.zeros(4, dtype=torch.int32)), "slots"),
                      (dict(workspace=torch.zeros(1, dtype=torch.uint8).expand(1 << 20)), "workspace")):
        with pytest.raises(ValueError, match=what):
            extend(**bad)
    q, k, pos, freq = torch.zeros(3, 4, 64), torch.zeros(3, 2, 64), i32(1, 2, 3), torch.ones(32, dtype=torch.float64)
    step.qk_rope(q, k, pos, freq)
    for bad, what in ((dict(q=q[0]), "q must"), (dict(k=k[:2]), "k must"), (dict(k=k.half()), "k must"), (dict(k=k[0]), "k must"), (dict(pos=None), "pos"),
                      (dict(pos=pos.long()), "pos"), (dict(freq=freq.float()), "freq"), (dict(q=q.transpose(0, 1), k=None, pos=None, freq=None), "q must"),
                      (dict(q=q.to(torch.int32), k=None, pos=None, freq=None), "float32"), (dict(q_weight=freq), "weights"), (dict(k_weight=torch.ones(63)), "weights"),
                      (dict(q_out=k), "q_out"), (dict(k_out=q), "k_out"), (dict(q=torch.zeros(3, 4, 128)[..., ::2], k=None, pos=None, freq=None), "q must"),
                      (dict(q=torch.zeros(1, 1, 1).expand((1 << 32) + 1, 1, 1)), "2\\^31")):
        with pytest.raises(ValueError, match=what):
            step.qk_rope(**{**dict(q=q, k=k, pos=pos, freq=freq), **bad})
    x, u = torch.zeros(2, 10), torch.zeros(2)
    step.sample(x, u, workspace=torch.empty(1 << 20, dtype=torch.uint8))
    for bad, what in ((dict(logits=x[0]), "logits"), (dict(logits=torch.zeros(10, 2).t()), "logits"), (dict(logits=x.to(torch.int32)), "float32"), (dict(u=u.double()), "u must"),
                      (dict(temperature=u.half()), "temperature"), (dict(top_k=u), "top_k"), (dict(top_p=u[:1]), "top_p"), (dict(min_p=1.0 * pos), "min_p"),
                      (dict(tokens=u), "tokens"), (dict(probs=x.half()), "probs"), (dict(probs=x[:, :5]), "probs"),
                      (dict(workspace=torch.zeros(1, dtype=torch.uint8).expand(1 << 20)), "workspace")):
        with pytest.raises(ValueError, match=what):
            step.sample(**{**dict(logits=x, u=u), **bad})
    assert called == ["llapis_kv_extend", "llapis_qk_rope", "llapis_sample"]


# -------------------------------------------------- attention with a prefix

def test_prefix_refusals():
    from test_step import BAD_BATCH, BAD_CACHE, batch, cache, query
    lib = la.lib()
    prefix = lambda **kw: _lib.LlapisKvPrefix(**{**dict(n_group=1, groups=P, prefix=P), **kw})

    def call(c=cache(), b=batch(), q=query(), x=prefix(), ws=P, n=1 << 40):
        ref = lambda s: None if s is None else C.byref(s)
        return lib.llapis_kv_prefix_attention(ref(c), ref(b), ref(q), ref(x), ws, n, None)

    who = "llapis_kv_prefix_attention"
    for bad in BAD_CACHE:
        refused(call(c=cache(**bad)), who)
    for bad in BAD_BATCH:
        refused(call(b=batch(**bad)), who)
    two = batch(n_seq=2, n_tokens=2)
    for bad in (dict(type=la.Q8_0), dict(n_head=3), dict(n_head=0), dict(n_head=2048), dict(window=-1), dict(window=5), dict(scale=float("nan")),
                dict(q=None), dict(out=None), dict(q=P + 4), dict(q_stride=258), dict(out_stride=250), dict(out=P)):
        refused(call(b=two, q=query(**bad)), who)
    for bad in (dict(n_group=-1), dict(n_group=257), dict(groups=None), dict(prefix=None)):
        refused(call(x=prefix(**bad)), who)
    for bad in (dict(c=None), dict(b=None), dict(q=None), dict(x=None)):
        refused(call(**bad), "null")
    refused(call(b=batch(new_start=P, max_new=17, n_tokens=17)), "16 new tokens")
    need = lib.llapis_kv_prefix_attention_workspace_size(C.byref(cache()), C.byref(batch()), 4, 1)
    assert need > lib.llapis_kv_attention_workspace_size(C.byref(cache()), C.byref(batch()), 4)
    refused(call(n=64), "workspace")
    refused(call(ws=P + 8), "workspace")
    refused(call(ws=None), "workspace")
    # nothing to do is no error
    for nothing in (dict(n_seq=0, page_table=None, lens=None), dict(n_tokens=0)):
        assert call(b=batch(**nothing), ws=None, n=0) == 0
    size = lambda c=cache(), b=batch(), h=4, g=1: lib.llapis_kv_prefix_attention_workspace_size(C.byref(c), C.byref(b), h, g)
    assert size(h=3) == size(g=257) == size(g=-1) == size(b=batch(new_start=P, max_new=17)) == 0
    # more units than 32 bits count: 1024 heads, 2^22 pages of 256 keys
    big = cache(n_kv=1024, head_dim=512, page_size=256, k_stride=1 << 28, v_stride=1 << 28)
    b = batch(max_pages=1 << 22, table_stride=1 << 22)
    assert size(big, b, 1024) == 0
    refused(call(c=big, b=b, q=query(n_head=1024, q_stride=1 << 19, out_stride=1 << 19)), who)


@pytest.mark.parametrize("kind", [la.F16, la.BF16])
@pytest.mark.parametrize("head_dim", [64, 128, 512])
def test_prefix_workspace_serves_less(head_dim, kind):
    from test_step import batch, cache
    lib, c = la.lib(), cache(type=kind, n_kv=2, head_dim=head_dim, page_size=64, k_stride=1 << 20, v_stride=1 << 20)

    def size(n_seq, new, pages, groups, tokens=None):
        b = batch(n_seq=n_seq, n_tokens=n_seq * new if tokens is None else tokens, max_new=new, max_pages=pages, table_stride=pages, new_start=P)
        return lib.llapis_kv_prefix_attention_workspace_size(C.byref(c), C.byref(b), 16, groups)

    for n_seq, new, pages, groups in ((1, 16, 3, 1), (64, 16, 512, 7), (300, 9, 100, 256)):
        most = size(n_seq, new, pages, groups)
        for less in ((n_seq, new - 1, pages, groups), (max(n_seq - 1, 1), new, pages, groups), (n_seq, new, pages - 1, groups), (n_seq, new, pages, groups - 1),
                     (n_seq, new, pages, groups, 1), (1, 1, 1, 0)):
            assert 0 < size(*less) <= most, less


def test_prefix_limits_and_their_names():
    """Groups have limits of their own, each refused by its name; without groups the call is attention's."""
    from test_step import batch, cache, query
    lib, c, q = la.lib(), cache(n_kv=1, k_stride=1 << 20, v_stride=1 << 20), query(n_head=1)
    new = lambda **kw: batch(**{**dict(n_seq=1 << 12, max_new=16, new_start=P, max_pages=4, table_stride=4), **kw})

    def size(b, groups, heads=1):
        return lib.llapis_kv_prefix_attention_workspace_size(C.byref(c), C.byref(b), heads, groups)

    def call(b, groups, n, q=q):
        x = _lib.LlapisKvPrefix(groups, P if groups else None, P if groups else None)
        return lib.llapis_kv_prefix_attention(C.byref(c), C.byref(b), C.byref(q), C.byref(x), P, n, None)

    many = new(n_tokens=(1 << 24) + 1)
    assert size(many, 1) == 0 < size(many, 0) == lib.llapis_kv_attention_workspace_size(C.byref(c), C.byref(many), 1)
    refused(call(many, 1, 1 << 40), "llapis_kv_prefix_attention", "2^24 rows")
    refused(call(many, 0, 64), "llapis_kv_prefix_attention", "workspace")
    assert size(new(n_tokens=1 << 24), 1) > 0
    # query rows of a kv head past 31 bits
    heads = query(n_head=256, q_stride=1 << 14, out_stride=1 << 14)
    assert size(new(n_tokens=1 << 23), 1, 256) == 0
    refused(call(new(n_tokens=1 << 23), 1, 1 << 40, heads), "2^31 query rows")
    # a table of one unit needs no join of its own, one with a prefix does
    short = batch(n_seq=1 << 24, n_tokens=1, max_pages=1, table_stride=1)
    assert size(short, 1) == 0 < size(short, 0)
    refused(call(short, 1, 1 << 40), "32 query rows")
    refused(call(short, 0, 64), "workspace")
    # prefixes of more units than 31 bits count
    wide = batch(n_seq=64, n_tokens=1 << 22, max_new=16, new_start=P, max_pages=1 << 14, table_stride=1 << 14)
    assert size(wide, 1, 16) == 0 < size(wide, 0, 16)
    refused(call(wide, 1, 1 << 40, query(n_head=16, q_stride=1 << 10, out_stride=1 << 10)), "2^30 units")
