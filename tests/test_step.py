"""The operators of llapis_step.h without a GPU: struct layouts, sizes and the
calls that are refused before anything is launched."""
import ctypes as C

import pytest

import llapis_amd as la
from llapis_amd import _lib
from test_abi import INCLUDE, compile_layouts

STRUCTS = {
    "llapis_kv_cache": _lib.LlapisKvCache, "llapis_kv_batch": _lib.LlapisKvBatch, "llapis_kv_query": _lib.LlapisKvQuery,
    "llapis_kv_planes": _lib.LlapisKvPlanes, "llapis_block_norm_args": _lib.LlapisBlockNormArgs,
    "llapis_verify_args": _lib.LlapisVerifyArgs,
}


def test_ctypes_mirror_matches_header(tmp_path):
    structs = {k: [f[0] for f in v._fields_] for k, v in STRUCTS.items()}
    got = compile_layouts(tmp_path, str(INCLUDE / "llapis_step.h"), structs)
    for s, cls in STRUCTS.items():
        assert got[(s, "sizeof")] == C.sizeof(cls), s
        for f in structs[s]:
            assert got[(s, f)] == getattr(cls, f).offset, (s, f)


def test_page_bytes():
    f = la.lib().llapis_kv_page_bytes
    assert f(la.F16, 8, 128, 16) == 8 * 128 * 16 * 2 == f(la.BF16, 8, 128, 16)
    assert f(la.Q8_0, 2, 64, 32) == 2 * 64 * 32 * 34 // 32
    for bad in ((la.F32, 8, 128, 16), (la.Q4_K, 8, 128, 16), (la.F16, 0, 128, 16), (la.F16, 8, 80, 16),
                (la.F16, 8, 128, 8), (la.F16, 8, 128, 48), (la.F16, 8, 128, 512), (la.F16, 1025, 64, 16)):
        assert f(*bad) == 0, bad


P = 0x10000          # an address that a refused call must not touch


def cache(**kw):
    a = dict(type=la.F16, n_kv=2, head_dim=64, page_size=16, n_pages=4, k=P, v=P, k_stride=4096, v_stride=4096)
    a.update(kw)
    return _lib.LlapisKvCache(**a)


def batch(**kw):
    a = dict(n_seq=1, n_tokens=1, max_new=1, max_pages=4, table_stride=4, page_table=P, lens=P, new_start=None)
    a.update(kw)
    return _lib.LlapisKvBatch(**a)


def query(**kw):
    a = dict(type=la.F32, n_head=4, window=0, scale=0.125, q=P, q_stride=256, out=2 * P, out_stride=256, lse=None)
    a.update(kw)
    return _lib.LlapisKvQuery(**a)


def refused(rc, *words):
    assert rc == -1
    said = la.lib().llapis_last_error().decode()
    assert all(w in said for w in words), said


BAD_CACHE = [dict(type=la.F32), dict(head_dim=72), dict(page_size=24), dict(n_pages=0), dict(k=None), dict(v=P + 8),
             dict(k_stride=4088), dict(v_stride=2048), dict(n_kv=0)]
BAD_BATCH = [dict(n_seq=-1), dict(max_pages=0), dict(table_stride=3), dict(page_table=None), dict(lens=None),
             dict(max_pages=1 << 27, table_stride=1 << 27), dict(n_tokens=-1)]


@pytest.mark.parametrize("bad", BAD_CACHE, ids=str)
def test_cache_refusals(bad):
    c, b, q = cache(**bad), batch(), query()
    refused(la.lib().llapis_kv_append(C.byref(c), C.byref(b), la.F32, P, 128, P, 128, None), "llapis_kv_append")
    refused(la.lib().llapis_kv_attention(C.byref(c), C.byref(b), C.byref(q), P, 1 << 40, None), "llapis_kv_attention")


@pytest.mark.parametrize("bad", BAD_BATCH, ids=str)
def test_batch_refusals(bad):
    c, b, q = cache(), batch(**bad), query()
    refused(la.lib().llapis_kv_append(C.byref(c), C.byref(b), la.F32, P, 128, P, 128, None), "llapis_kv_append")
    refused(la.lib().llapis_kv_attention(C.byref(c), C.byref(b), C.byref(q), P, 1 << 40, None), "llapis_kv_attention")


@pytest.mark.parametrize("bad", [dict(type=la.Q8_0), dict(n_head=3), dict(n_head=0), dict(n_head=2048), dict(window=-1),
                                 dict(scale=float("nan")), dict(q=None), dict(out=None), dict(q=P + 4),
                                 dict(q_stride=258), dict(out_stride=250), dict(out=P)], ids=str)
def test_query_refusals(bad):
    c, b, q = cache(), batch(n_seq=2, n_tokens=2), query(**bad)
    refused(la.lib().llapis_kv_attention(C.byref(c), C.byref(b), C.byref(q), P, 1 << 40, None), "llapis_kv_attention")


def test_attention_limits():
    c, q = cache(), query()
    b = batch(new_start=P, max_new=17, n_tokens=17)
    refused(la.lib().llapis_kv_attention(C.byref(c), C.byref(b), C.byref(q), P, 1 << 40, None), "16 new tokens")
    assert la.lib().llapis_kv_attention_workspace_size(C.byref(c), C.byref(b), 4) == 0
    b = batch()
    need = la.lib().llapis_kv_attention_workspace_size(C.byref(c), C.byref(b), 4)
    assert need > 0
    refused(la.lib().llapis_kv_attention(C.byref(c), C.byref(b), C.byref(q), P, need - 1, None), "workspace")
    refused(la.lib().llapis_kv_attention(C.byref(c), C.byref(b), C.byref(q), None, need, None), "workspace")
    refused(la.lib().llapis_kv_attention(None, C.byref(b), C.byref(q), P, need, None), "null cache")
    refused(la.lib().llapis_kv_attention(C.byref(c), C.byref(b), None, P, need, None), "null query")
    # a workspace for more serves less
    more = batch(n_seq=5, n_tokens=80, max_new=16, new_start=P)
    assert la.lib().llapis_kv_attention_workspace_size(C.byref(c), C.byref(more), 4) >= need
    # nothing to do is no error
    for nothing in (dict(n_seq=0, page_table=None, lens=None), dict(n_tokens=0)):
        b = batch(**nothing)
        assert la.lib().llapis_kv_attention(C.byref(c), C.byref(b), C.byref(q), None, 0, None) == 0
        assert la.lib().llapis_kv_append(C.byref(c), C.byref(b), la.F32, P, 128, P, 128, None) == 0


@pytest.mark.parametrize("head_dim", [64, 96, 128, 256, 512])
@pytest.mark.parametrize("n_kv,group", [(8, 1), (8, 8), (2, 9), (1, 64), (1, 1024)])
def test_attention_workspace_serves_less(head_dim, n_kv, group):
    """A workspace for the most sequences, new tokens and pages of a program serves each of its smaller steps."""
    lib, n_head = la.lib(), n_kv * group
    c = cache(n_kv=n_kv, head_dim=head_dim, page_size=64, k_stride=1 << 20, v_stride=1 << 20)

    def size(n_seq, new, pages):
        b = batch(n_seq=n_seq, n_tokens=n_seq * new, max_new=new, max_pages=pages, table_stride=pages, new_start=P)
        return lib.llapis_kv_attention_workspace_size(C.byref(c), C.byref(b), n_head)

    for n_seq, new, pages in ((1, 16, 3), (7, 16, 40), (64, 16, 512), (300, 9, 100)):
        most = size(n_seq, new, pages)
        for less in [(n_seq, i, pages) for i in range(1, new)] + [(max(n_seq - 1, 1), new, pages), (n_seq, new, pages - 1), (1, 1, 1)]:
            assert 0 < size(*less) <= most, less


def test_append_refusals():
    c, b = cache(), batch(n_seq=2, n_tokens=2)
    call = lambda t=la.F32, k=P, ks=128, v=P, vs=128: la.lib().llapis_kv_append(C.byref(c), C.byref(b), t, k, ks, v, vs, None)
    refused(call(t=la.Q8_0), "F32, F16 or BF16")
    refused(call(k=None), "null")
    refused(call(v=P + 8), "aligned")
    refused(call(ks=130), "aligned")
    refused(call(vs=64), "shorter")


def planes(n=2, **kw):
    s = _lib.LlapisKvPlanes(n, kw.get("n_pages", 4), kw.get("page_size", 16))
    for i in range(min(n, 128)):
        s.base[i], s.stride[i], s.bytes[i] = kw.get("base", P), kw.get("stride", 4096), kw.get("bytes", 4096)
    return s


@pytest.mark.parametrize("bad", [dict(n=0), dict(n=129), dict(n_pages=0), dict(page_size=0), dict(base=None),
                                 dict(base=P + 8), dict(stride=4090), dict(bytes=4097), dict(bytes=0), dict(stride=2048)], ids=str)
def test_plane_refusals(bad):
    p, lib = planes(**bad), la.lib()
    refused(lib.llapis_kv_copy_pages(C.byref(p), P, 1, None), "llapis_kv_copy_pages")
    refused(lib.llapis_kv_fork(C.byref(p), P, 4, 4, P, 2, P, 1, None), "llapis_kv_fork")
    refused(lib.llapis_kv_compact(C.byref(p), P, 4, 4, P, 2, P, None, P, P, 1 << 20, None), "llapis_kv_compact")


def test_page_refusals():
    p, lib = planes(), la.lib()
    refused(lib.llapis_kv_copy_pages(C.byref(p), None, 1, None), "null pairs")
    refused(lib.llapis_kv_copy_pages(C.byref(p), P, -1, None), "negative")
    assert lib.llapis_kv_copy_pages(C.byref(p), None, 0, None) == 0
    refused(lib.llapis_kv_fork(C.byref(p), P, 3, 4, P, 2, P, 1, None), "table_stride")
    refused(lib.llapis_kv_fork(C.byref(p), None, 4, 4, P, 2, P, 1, None), "null")
    refused(lib.llapis_kv_fork(C.byref(p), P, 4, 4, P, 2, None, 1, None), "null forks")
    refused(lib.llapis_kv_fork(C.byref(p), P, 4, 4, P, 2, P, 65536, None), "n_forks")
    assert lib.llapis_kv_fork(C.byref(p), P, 4, 4, P, 2, None, 0, None) == 0
    refused(lib.llapis_kv_page_refs(0, 16, P, 4, 4, P, 2, P, P, P, None), "n_pages")
    refused(lib.llapis_kv_page_refs(4, 16, P, 4, 4, P, 2, None, P, P, None), "null refs")
    need = lib.llapis_kv_compact_workspace_size(4)
    assert need > 0 and lib.llapis_kv_compact_workspace_size(0) == 0
    refused(lib.llapis_kv_compact(C.byref(p), P, 4, 4, P, 2, P, None, P, P, need - 1, None), "workspace")
    refused(lib.llapis_kv_compact(C.byref(p), P, 4, 4, P, 2, None, None, P, P, need, None), "table_out")
    refused(lib.llapis_kv_compact(C.byref(p), P, 4, 4, P, 2, P, None, None, P, need, None), "n_live")


def norm_args(**kw):
    a = dict(type=la.F32, n_tokens=2, d=64, n_out=1, post_norm=1, eps=1e-6, alpha=1.0, beta=1.0, h=P, h_stride=64,
             h_out=P, h_out_stride=64)
    a.update({k: v for k, v in kw.items() if k != "x"})
    s = _lib.LlapisBlockNormArgs(**a)
    for i in range(4):
        s.x[i], s.x_stride[i] = kw.get("x", P), 64
    return s


@pytest.mark.parametrize("bad", [dict(type=la.Q8_0), dict(d=0), dict(d=16385), dict(n_tokens=-1), dict(n_out=5), dict(n_out=-1),
                                 dict(h=None), dict(x=None), dict(h_out=None, n_out=0), dict(h_out_stride=63),
                                 dict(gate=P, gate_value_stride=2)], ids=str)
def test_norm_refusals(bad):
    a = norm_args(**bad)
    refused(la.lib().llapis_block_norm(C.byref(a), None), "llapis_block_norm")


def test_norm_of_nothing():
    a = norm_args(n_tokens=0)
    assert la.lib().llapis_block_norm(C.byref(a), None) == 0
    refused(la.lib().llapis_block_norm(None, None), "null")


def verify_args(**kw):
    a = dict(type=la.F32, n_seq=2, max_draft=3, vocab=100, target=P, target_stride=100, draft=P, draft_stride=100, drafts=P,
             n_draft=None, u=P, u_next=P, tokens=P, accepted=P)
    a.update(kw)
    return _lib.LlapisVerifyArgs(**a)


@pytest.mark.parametrize("bad", [dict(type=la.Q4_K), dict(n_seq=-1), dict(n_seq=65536), dict(max_draft=-1), dict(max_draft=64),
                                 dict(vocab=0), dict(target=None), dict(u_next=None), dict(tokens=None), dict(accepted=None),
                                 dict(drafts=None), dict(u=None), dict(target_stride=99), dict(draft_stride=99)], ids=str)
def test_verify_refusals(bad):
    a = verify_args(**bad)
    refused(la.lib().llapis_verify_drafts(C.byref(a), P, 1 << 20, None), "llapis_verify_drafts")


def test_verify_workspace():
    a, lib = verify_args(), la.lib()
    need = lib.llapis_verify_drafts_workspace_size(2, 100)
    assert need > 0
    refused(lib.llapis_verify_drafts(C.byref(a), P, need - 1, None), "workspace")
    refused(lib.llapis_verify_drafts(C.byref(a), P + 4, need, None), "workspace")
    a = verify_args(n_seq=0)
    assert lib.llapis_verify_drafts(C.byref(a), None, 0, None) == 0


def test_python_refuses_host_tensors():
    import torch
    with pytest.raises(ValueError, match="GPU"):
        la.KvBatch(torch.zeros(1, 4, dtype=torch.int32), torch.ones(1, dtype=torch.int32))
    with pytest.raises(ValueError, match="GPU"):
        la.KvCache(torch.zeros(2, 1, 16, 64).half(), torch.zeros(2, 1, 64, 16).half())
    with pytest.raises(ValueError, match="GPU"):
        la.block_norm(torch.zeros(2, 64))
    with pytest.raises(ValueError, match="GPU"):
        la.verify_drafts(torch.zeros(1, 2, 10), None, torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, 1), torch.zeros(1))


def test_launch_limits():
    """A launch has fewer than 2^32 threads in x.  Calls with a kernel past that, or whose
    units of work pass 64 bits, are refused as calls, before a first kernel of theirs runs."""
    lib, many = la.lib(), 1 << 24
    b = batch(n_seq=many, n_tokens=many, max_new=1)
    refused(lib.llapis_kv_append(C.byref(cache()), C.byref(b), la.F32, P, 128, P, 128, None), "llapis_kv_append", "2^24")
    for n in (many, (1 << 31) - 1):
        refused(lib.llapis_kv_page_refs(4, 16, P, 4, 4, P, n, P, P, P, None), "llapis_kv_page_refs", "2^24")
        refused(lib.llapis_kv_compact(C.byref(planes()), P, 4, 4, P, n, P, None, P, P, 1 << 20, None), "llapis_kv_compact", "2^24")
    # attention: (sequence, kv head, tile of query rows), which the second kernel has a workgroup for
    many_heads = cache(n_kv=8, head_dim=64, page_size=256, k_stride=1 << 19, v_stride=1 << 19)
    for c, b, n_head in ((many_heads, batch(n_seq=1 << 21, n_tokens=1 << 21), 8),
                         (many_heads, batch(n_seq=1 << 17, n_tokens=1 << 21, max_new=16, new_start=P), 256)):
        q = query(n_head=n_head, q_stride=64 * n_head, out_stride=64 * n_head)
        assert lib.llapis_kv_attention_workspace_size(C.byref(c), C.byref(b), n_head) == 0
        refused(lib.llapis_kv_attention(C.byref(c), C.byref(b), C.byref(q), P, 1 << 40, None), "llapis_kv_attention", "2^24")
        b.n_seq -= 1
        assert lib.llapis_kv_attention_workspace_size(C.byref(c), C.byref(b), n_head) > 0
    # one kernel does where every item is a unit, whatever their number (a page of 16 keys)
    c, b = cache(n_kv=8, k_stride=1 << 14, v_stride=1 << 14), batch(n_seq=1 << 21, n_tokens=1 << 21, max_pages=1, table_stride=1)
    assert lib.llapis_kv_attention_workspace_size(C.byref(c), C.byref(b), 8) > 0
    # 2^24 units of a sequence, 1024 heads and 2^30 sequences: 2^64
    c = cache(n_kv=1024, head_dim=512, page_size=256, k_stride=1 << 28, v_stride=1 << 28)
    b = batch(n_seq=1 << 30, n_tokens=1, max_pages=1 << 22, table_stride=1 << 22)
    q = query(n_head=1024, q_stride=1 << 19, out_stride=1 << 19)
    assert lib.llapis_kv_attention_workspace_size(C.byref(c), C.byref(b), 1024) == 0
    refused(lib.llapis_kv_attention(C.byref(c), C.byref(b), C.byref(q), P, 1 << 62, None), "units")


def test_python_refuses_overlapping_table_rows(monkeypatch):
    """Rows of a page table that share entries (one row for all sequences, expanded; rows
    a few entries apart): the library would take them for rows of their whole width,
    past the table's memory.  Host tensors stand in for the GPU's, and nothing is called."""
    import torch
    from llapis_amd import step
    called = []
    monkeypatch.setattr(step, "_on_gpu", lambda t, what: t.device)
    monkeypatch.setattr(step, "_call", lambda *a: called.append(a))
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32)
    caches = [step.KvCache.empty(8, 16, 1, 64, la.F16, "cpu") for _ in range(2)]
    pages, lens = step.KvPages(caches), i32(5, 5, 5)
    one = i32([0, 1, 2, 3])
    for table in (one.expand(3, 4), torch.arange(10, dtype=torch.int32).as_strided((3, 4), (3, 1))):
        for call in (lambda: step.KvBatch(table, lens), lambda: step.KvBatch(table, lens, i32(0, 1, 2, 3), 3),
                     lambda: pages.fork(table, lens, i32([0, 1, 6])), lambda: pages.refs(table, lens),
                     lambda: pages.compact(table, lens), lambda: pages.compact(table, lens, table_out=table)):
            with pytest.raises(ValueError, match="overlap"):
                call()
    assert not called
    # one row's stride says nothing, and rows may lie apart
    assert step.KvBatch(one, lens[:1]).struct.table_stride == 4 == step.KvBatch(one.expand(1, 4), lens[:1]).struct.table_stride
    assert step.KvBatch(one.as_strided((1, 4), (0, 1)), lens[:1]).struct.table_stride == 4
    assert step.KvBatch(torch.zeros(3, 9, dtype=torch.int32)[:, 1:5], lens).struct.table_stride == 9
    pages.refs(one.as_strided((1, 4), (0, 1)), lens[:1])
    assert [a[5] for a in called] == [4]


@pytest.mark.parametrize("bad", ["expanded", "elsewhere"])
def test_python_checks_workspaces(monkeypatch, bad):
    """A workspace has to be memory of the call's device, all of it: one value expanded to the
    size, or memory of another device, is no workspace.  Host tensors stand in for the GPU's."""
    import torch
    from llapis_amd import step
    called = []
    monkeypatch.setattr(step, "_on_gpu", lambda t, what: t.device)
    monkeypatch.setattr(step, "_call", lambda *a: called.append(a))
    ws = torch.zeros(1, dtype=torch.uint8).expand(1 << 24) if bad == "expanded" else torch.empty(1 << 24, dtype=torch.uint8, device="meta")
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32)
    cache = step.KvCache.empty(8, 16, 1, 64, la.F16, "cpu")
    table, lens = i32([0, 1], [2, 3]), i32(5, 7)
    calls = (lambda w: cache.attention(step.KvBatch(table, lens), torch.zeros(2, 4, 64), workspace=w),
             lambda w: step.KvPages([cache]).compact(table, lens, workspace=w),
             lambda w: step.verify_drafts(torch.rand(2, 2, 9), None, torch.zeros(2, 1, dtype=torch.int32), torch.rand(2, 1), torch.rand(2), workspace=w))
    for call in calls:
        with pytest.raises(ValueError, match="workspace"):
            call(ws)
    assert not called
    for call in calls:
        call(torch.empty(1 << 24, dtype=torch.uint8))
    assert [a[0] for a in called] == ["llapis_kv_attention", "llapis_kv_compact", "llapis_verify_drafts"]


def test_largest_counts():
    """Counts that loops would run past 32 bits with are refused, and have no workspace."""
    lib, big = la.lib(), (1 << 30) + 1
    refused(lib.llapis_kv_page_refs(big, 16, P, 4, 4, P, 2, P, P, P, None), "n_pages")
    refused(lib.llapis_kv_page_refs(4, 16, P, big, big, P, 2, P, P, P, None), "max_pages")
    refused(lib.llapis_kv_fork(C.byref(planes()), P, big, big, P, 2, P, 1, None), "max_pages")
    refused(lib.llapis_kv_copy_pages(C.byref(planes(n_pages=big)), P, 1, None), "n_pages")
    assert lib.llapis_kv_compact_workspace_size(big) == 0
    assert lib.llapis_kv_compact_workspace_size(1 << 30) == ((4 << 30) + 1) * 4
    assert lib.llapis_verify_drafts_workspace_size(1, big) == 0 == lib.llapis_verify_drafts_workspace_size(1 << 16, 10)
    assert lib.llapis_verify_drafts_workspace_size(1, (1 << 31) - 1) == 0
    assert lib.llapis_verify_drafts_workspace_size(1, 1 << 30) > 0
