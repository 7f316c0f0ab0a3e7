"""The operators of a decode step around the MoE layer (include/llapis_step.h):

* ``KvCache`` -- one layer's paged key-value cache: ``append`` writes a step's
  new keys and values, ``attention`` attends the new tokens over it.
* ``KvBatch`` -- a step's sequences: page table, lengths, new tokens.
* ``KvPages`` -- page operations over every layer's pools at once: copy, fork,
  references and free pages, compaction, room for a step's new tokens.
* ``qk_rope`` -- the norms of queries and keys and their rotary positions, whose
  frequencies ``rope_frequencies`` computes.
* ``block_norm`` -- post-norm, gate, residual and the next block's norms.
* ``sample`` -- the next tokens from logits, with the probabilities they were drawn with.
* ``verify_drafts`` -- accept or refuse drafted tokens, draw the next one.

torch is used for device memory and the current stream alone.  A call runs on
the current stream of its tensors' device, allocates only what it is not handed
(outputs, workspaces) and can be captured in a graph.  Arguments that do not fit
raise ValueError, what the library refuses LlapisError.
"""
import ctypes as C

from . import _lib as L
from ._lib import BF16, F16, F32, Q8_0, check, lib

_module = None
_tags = {}


def _torch():
    """torch, imported at the first call (an import statement costs every call 0.3 us)."""
    global _module
    if _module is None:
        import torch
        _tags.update({torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16})
        _module = torch
    return _module


def _tag(dtype):
    tag = _tags.get(dtype)
    if tag is None:
        raise ValueError(f"need float32, float16 or bfloat16 values, got {dtype}")
    return tag


def _need(ok, what):
    if not ok:
        raise ValueError(what)


def _is(t, dtype, shape, dev, what):
    if t.dtype != dtype or t.shape != shape or t.device != dev or not t.is_contiguous():
        raise ValueError(f"{what} must be a contiguous {dtype} tensor of shape {tuple(shape)} on {dev}")


def _count(*values):
    """Sizes as the library takes them: a larger one would wrap around in 32 bits.  (Calls
    of a step ask with a shift first: the loop here costs them 0.3 us.)"""
    for x in values:
        if not 0 <= x < 1 << 31:
            raise ValueError(f"a size of {x} is negative or 2^31 and more")


def _ptr(t):
    return None if t is None else t.data_ptr()


def _call(name, dev, *args):
    """The entry point on the current stream of `dev`, which becomes the current device for it."""
    fn, index, gpu = getattr(lib(), name), dev.index, _module._C
    # (the raw handle: torch.cuda.current_stream builds an object around it, 2 us a call)
    stream = gpu._cuda_getCurrentRawStream(index)
    if index == gpu._cuda_getDevice():
        check(fn(*args, stream), name)
    else:
        with _module.cuda.device(dev):
            check(fn(*args, stream), name)


def _table_stride(table):
    """Entries from a page table's row to the next.  A single row's stride says
    nothing; the rows of several must not overlap (an expanded row has a stride of 0)."""
    stride, (n, width) = table.stride(0), table.shape
    if stride < width:
        if n > 1:
            raise ValueError("page_table's rows overlap: each sequence needs a row of its own")
        return width
    return stride


def _bytes(sizer, dev, *args):
    """A workspace of the size that the library names"""
    return _torch().empty(int(getattr(lib(), sizer)(*args)), dtype=_torch().uint8, device=dev)


def _scratch(workspace, dev):
    """(address, bytes) of a caller's workspace"""
    if workspace.device != dev or not workspace.is_contiguous():
        raise ValueError(f"the workspace must be contiguous and on {dev}")
    return workspace.data_ptr(), workspace.numel() * workspace.element_size()


def _on_gpu(t, what):
    _need(t.device.type == "cuda", f"{what} must be on the GPU")
    return t.device


class KvBatch:
    """The sequences of a step.  page_table int32 [n_seq, max_pages] (-1: no
    page), lens int32 [n_seq] with the new tokens, new_start int32 [n_seq + 1]
    the first activation row of each sequence's new tokens (None: one each, row
    s), all on the GPU and read when a call runs.  n_tokens: activation rows in
    use, max_new: the most new tokens of a sequence (both needed with
    new_start)."""

    def __init__(self, page_table, lens, new_start=None, n_tokens=None, max_new=1):
        torch = _torch()
        self.device = _on_gpu(page_table, "page_table")
        _need(page_table.dtype == torch.int32 and page_table.dim() == 2 and page_table.stride(1) == 1
              and page_table.shape[1] > 0, "page_table must be int32 [n_seq, max_pages], rows of consecutive entries")
        n = page_table.shape[0]
        _is(lens, torch.int32, (n,), self.device, "lens")
        if new_start is not None:
            _is(new_start, torch.int32, (n + 1,), self.device, "new_start")
            _need(n_tokens is not None, "new_start needs n_tokens")
        else:
            _need(max_new == 1 and n_tokens in (None, n), "without new_start every sequence has one new token")
            n_tokens = n
        _count(n, n_tokens, max_new, page_table.shape[1])
        self.page_table, self.lens, self.new_start = page_table, lens, new_start
        self.n_seq, self.n_tokens, self.max_new, self.max_pages = n, n_tokens, max_new, page_table.shape[1]
        self.struct = L.LlapisKvBatch(n, n_tokens, max_new, self.max_pages, _table_stride(page_table),
                                      page_table.data_ptr(), lens.data_ptr(), _ptr(new_start))
        self._ref = C.byref(self.struct)


class KvCache:
    """One layer's cache.  k [n_pages, n_kv, page_size, head_dim] and v [n_pages,
    n_kv, head_dim, page_size] in float16 or bfloat16 (pages may lie further
    apart), or bytes [n_pages, page bytes] with type Q8_0 and the geometry."""

    def __init__(self, k, v, type=None, n_kv=None, head_dim=None, page_size=None):
        torch = _torch()
        self.device = _on_gpu(k, "k")
        _need(v.device == self.device and v.dtype == k.dtype and v.shape[0] == k.shape[0],
              "k and v must agree in device, type and pages")
        if type in (None, F16, BF16) and k.dim() == 4:
            tag = _tag(k.dtype)
            _need(tag != F32 and type in (None, tag), "the pools must be float16 or bfloat16, or bytes of Q8_0")
            n_pages, H, P, D = k.shape
            _need(tuple(v.shape) == (n_pages, H, D, P), "v must be [n_pages, n_kv, head_dim, page_size]")
            _need(k.stride()[1:] == (P * D, D, 1) and v.stride()[1:] == (P * D, P, 1), "a page must be contiguous")
            _need((n_kv, head_dim, page_size) in ((None,) * 3, (H, D, P)), "geometry and pools differ")
        else:
            _need(type == Q8_0 and k.dim() == 2 and k.dtype in (torch.uint8, torch.int8) and None not in
                  (n_kv, head_dim, page_size), "bytes need type Q8_0, n_kv, head_dim and page_size")
            tag, n_pages, H, P, D = type, k.shape[0], n_kv, page_size, head_dim
            need = int(lib().llapis_kv_page_bytes(tag, H, D, P))
            _need(k.shape[1] == need and v.shape == k.shape and k.stride(1) == 1 and v.stride(1) == 1,
                  f"a page must be {need} contiguous bytes")
        _count(n_pages, H, P, D)
        es = k.element_size()
        self.k, self.v, self.type = k, v, tag
        self.n_pages, self.n_kv, self.page_size, self.head_dim = n_pages, H, P, D
        self.page_bytes = int(lib().llapis_kv_page_bytes(tag, H, D, P))
        # the stride of a single page says nothing
        step = lambda t: t.stride(0) * es if n_pages > 1 else self.page_bytes
        self.struct = L.LlapisKvCache(tag, H, D, P, n_pages, k.data_ptr(), v.data_ptr(), step(k), step(v))
        self._ref = C.byref(self.struct)

    @classmethod
    def empty(cls, n_pages, page_size, n_kv, head_dim, type=F16, device="cuda"):
        """A cache of its own, its pages not initialised (masked places are never read into results)."""
        torch = _torch()
        if type == Q8_0:
            n = int(lib().llapis_kv_page_bytes(type, n_kv, head_dim, page_size))
            _need(n > 0, "unsupported geometry")
            make = lambda: torch.empty(n_pages, n, dtype=torch.uint8, device=device)
            return cls(make(), make(), type, n_kv, head_dim, page_size)
        dt = {F16: torch.float16, BF16: torch.bfloat16}.get(type)
        _need(dt is not None, "type must be F16, BF16 or Q8_0")
        return cls(torch.empty(n_pages, n_kv, page_size, head_dim, dtype=dt, device=device),
                   torch.empty(n_pages, n_kv, head_dim, page_size, dtype=dt, device=device))

    def _rows(self, t, batch, n_heads, what):
        D, shape, stride = self.head_dim, t.shape, t.stride()
        if (len(shape) != 3 or shape[0] < batch.n_tokens or shape[1] != n_heads or shape[2] != D or stride[2] != 1
                or (n_heads > 1 and stride[1] != D) or t.device != self.device):
            raise ValueError(f"{what} must be [{batch.n_tokens} or more, {n_heads}, {D}] on {self.device}, rows of consecutive values")
        return stride[0]

    def append(self, batch, k, v):
        """Write the new tokens' keys and values (k, v [n_tokens, n_kv, head_dim],
        float32, float16 or bfloat16) into their pages."""
        ks, vs = self._rows(k, batch, self.n_kv, "k"), self._rows(v, batch, self.n_kv, "v")
        _need(k.dtype == v.dtype and batch.device == self.device, "k and v must be of one type, the batch on their device")
        _call("llapis_kv_append", self.device, self._ref, batch._ref, _tag(k.dtype), k.data_ptr(), ks, v.data_ptr(), vs)

    def attention_workspace(self, batch, n_head):
        """Scratch for attention calls of this geometry and of batches within this one's
        bounds, for a caller that keeps it: calls that share it must not overlap."""
        n = int(lib().llapis_kv_attention_workspace_size(self._ref, batch._ref, n_head))
        if n == 0:
            raise ValueError("attention: unsupported geometry (n_head, max_new or lengths)")
        return _torch().empty(n, dtype=_torch().uint8, device=self.device)

    def attention(self, batch, q, scale=None, window=0, out=None, lse=None, workspace=None):
        """Attend the new tokens' queries q [n_tokens, n_head, head_dim] over the
        cache they have been appended to -> out, shaped and typed as q.  scale:
        head_dim ** -0.5 by default; window > 0: each token sees that many keys at
        most, itself the last; lse [rows, n_head] float32 receives the logarithm
        of the softmax sums.  Rows of no sequence are left as they are (in an
        out made here: as the allocation holds them)."""
        a = self._query(batch, q, scale, window, out, lse)
        if workspace is None:
            workspace = self.attention_workspace(batch, a.n_head)
        _call("llapis_kv_attention", self.device, self._ref, batch._ref, C.byref(a), *_scratch(workspace, self.device))
        return a.result

    def _query(self, batch, q, scale, window, out, lse):
        """Attention's arguments, the output among them as `result`"""
        torch = _torch()
        _need(q.dim() == 3 and batch.device == self.device, "q must be [n_tokens, n_head, head_dim], the batch on its device")
        n_head = q.shape[1]
        qs = self._rows(q, batch, n_head, "q")
        if out is None:
            out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        os_ = self._rows(out, batch, n_head, "out")
        _need(out.dtype == q.dtype, "out must be of q's type")
        if lse is not None:
            shape = lse.shape
            _need(lse.dtype == torch.float32 and lse.device == self.device and lse.is_contiguous() and len(shape) == 2
                  and shape[0] >= batch.n_tokens and shape[1] == n_head,
                  "lse must be a contiguous float32 [n_tokens, n_head]")
        if window >> 31:
            _count(window)
        a = L.LlapisKvQuery(_tag(q.dtype), n_head, window, self.head_dim ** -0.5 if scale is None else scale,
                            q.data_ptr(), qs, out.data_ptr(), os_, _ptr(lse))
        a.result = out
        return a

    def prefix_workspace(self, batch, n_head, n_group):
        """Scratch for prefix_attention calls of this geometry and of batches and groups within these bounds."""
        n = int(lib().llapis_kv_prefix_attention_workspace_size(self._ref, batch._ref, n_head, n_group))
        if n == 0:
            raise ValueError("prefix_attention: unsupported geometry (n_head, max_new, groups or lengths)")
        return _torch().empty(n, dtype=_torch().uint8, device=self.device)

    def prefix_attention(self, batch, q, groups, prefix, scale=None, out=None, lse=None, workspace=None):
        """attention without a window where sequences begin on the same pages (as
        fork leaves them): sequences groups[g] .. groups[g + 1] - 1 share their first
        prefix[g] tokens, which are read once for all of them.  groups int32
        [n_group + 1] in order, prefix int32 [n_group], on the GPU; sequences in no group share nothing."""
        torch = _torch()
        n = prefix.shape[0] if prefix.dim() == 1 else -1
        _is(prefix, torch.int32, (n,), self.device, "prefix")
        _is(groups, torch.int32, (n + 1,), self.device, "groups")
        a = self._query(batch, q, scale, 0, out, lse)
        if workspace is None:
            workspace = self.prefix_workspace(batch, a.n_head, n)
        x = L.LlapisKvPrefix(n, groups.data_ptr(), prefix.data_ptr())
        _call("llapis_kv_prefix_attention", self.device, self._ref, batch._ref, C.byref(a), C.byref(x),
              *_scratch(workspace, self.device))
        return a.result


class KvPages:
    """Page operations over the pools of all layers' caches (of one geometry in
    pages: the same n_pages and page_size), which share a page table."""

    def __init__(self, caches):
        _need(len(caches) > 0, "need a cache")
        c0 = caches[0]
        _need(all((c.n_pages, c.page_size, c.device) == (c0.n_pages, c0.page_size, c0.device) for c in caches),
              "the caches must agree in n_pages, page_size and device")
        self.caches, self.device = list(caches), c0.device
        self.n_pages, self.page_size = c0.n_pages, c0.page_size
        planes = [p for c in caches for p in ((c.struct.k, c.struct.k_stride, c.page_bytes),
                                              (c.struct.v, c.struct.v_stride, c.page_bytes))]
        self.structs = []
        for i in range(0, len(planes), L.KV_MAX_PLANES):
            group = planes[i:i + L.KV_MAX_PLANES]
            s = L.LlapisKvPlanes(len(group), self.n_pages, self.page_size)
            for j, (base, stride, nbytes) in enumerate(group):
                s.base[j], s.stride[j], s.bytes[j] = base, stride, nbytes
            self.structs.append(s)

    def _table(self, page_table, lens):
        torch = _torch()
        shape, stride = page_table.shape, page_table.stride()
        if (page_table.dtype != torch.int32 or len(shape) != 2 or stride[1] != 1 or shape[1] == 0
                or page_table.device != self.device):
            raise ValueError(f"page_table must be int32 [n_seq, max_pages] on {self.device}, rows of consecutive entries")
        _is(lens, torch.int32, (shape[0],), self.device, "lens")
        if (shape[0] | shape[1]) >> 31:
            _count(*shape)
        return page_table.data_ptr(), _table_stride(page_table), shape[1]

    def copy(self, pairs):
        """Copy page pairs[i, 0] to page pairs[i, 1] (int32 [n, 2] on the GPU) in every layer."""
        _is(pairs, _torch().int32, (pairs.shape[0], 2), self.device, "pairs")
        _count(pairs.shape[0])
        for s in self.structs:
            _call("llapis_kv_copy_pages", self.device, C.byref(s), pairs.data_ptr(), pairs.shape[0])

    def fork(self, page_table, lens, forks):
        """Fork sequences, forks int32 [n, 3] of (source row, target row, fresh
        page): the target shares the source's full pages and gets a copy of its
        partly filled last one.  Updates page_table and lens."""
        table, stride, width = self._table(page_table, lens)
        _is(forks, _torch().int32, (forks.shape[0], 3), self.device, "forks")
        _count(forks.shape[0])
        for s in self.structs:
            _call("llapis_kv_fork", self.device, C.byref(s), table, stride, width, lens.data_ptr(), page_table.shape[0],
                  forks.data_ptr(), forks.shape[0])

    def refs(self, page_table, lens):
        """(refs [n_pages], free [n_pages], n_free [1]), int32: how many entries
        within the lengths name each page, the pages without any in ascending
        order (then -1), and their number.  A sequence of length 0 holds none."""
        torch = _torch()
        table, stride, width = self._table(page_table, lens)
        out = [torch.empty(n, dtype=torch.int32, device=self.device) for n in (self.n_pages, self.n_pages, 1)]
        _call("llapis_kv_page_refs", self.device, self.n_pages, self.page_size, table, stride, width, lens.data_ptr(),
              page_table.shape[0], *(t.data_ptr() for t in out))
        return tuple(out)

    def workspace(self):
        """Scratch for compact, for a caller that keeps it: calls that share it must not overlap."""
        n = int(lib().llapis_kv_compact_workspace_size(self.n_pages))
        return _torch().empty(n, dtype=_torch().uint8, device=self.device)

    def compact(self, page_table, lens, table_out=None, refs=None, n_live=None, workspace=None):
        """Move the pages in use to the front of the pools -> (table_out, refs,
        n_live [1]): pages n_live and up are free.  page_table is left as it is
        unless it is table_out too."""
        torch = _torch()
        table, stride, width = self._table(page_table, lens)
        if table_out is None:
            table_out = torch.empty_strided(page_table.shape, page_table.stride(), dtype=torch.int32, device=self.device)
        _need(table_out.dtype == torch.int32 and table_out.shape == page_table.shape and table_out.device == self.device
              and table_out.stride() == page_table.stride(), "table_out must be laid out as page_table")
        if refs is None:
            refs = torch.empty(self.n_pages, dtype=torch.int32, device=self.device)
        _is(refs, torch.int32, (self.n_pages,), self.device, "refs")
        if n_live is None:
            n_live = torch.empty(1, dtype=torch.int32, device=self.device)
        _is(n_live, torch.int32, (1,), self.device, "n_live")
        if workspace is None:
            workspace = self.workspace()
        scratch = _scratch(workspace, self.device)
        if len(self.structs) > 1 and table_out.data_ptr() == page_table.data_ptr():
            # every group of planes has to see the table as it was
            page_table = page_table.clone()
            table = page_table.data_ptr()
            _need(_table_stride(page_table) == stride, "in place, more than 64 layers need a contiguous page_table")
        for s in self.structs:
            _call("llapis_kv_compact", self.device, C.byref(s), table, stride, width, lens.data_ptr(), table_out.shape[0],
                  table_out.data_ptr(), refs.data_ptr(), n_live.data_ptr(), *scratch)
        return table_out, refs, n_live

    def extend_workspace(self, n_seq):
        """Scratch for extend with up to n_seq sequences, for a caller that keeps it: calls that share it must not overlap."""
        return _bytes("llapis_kv_extend_workspace_size", self.device, n_seq)

    def extend(self, page_table, lens, n_new, free, n_free, n_tokens, lens_out=None, n_free_out=None, new_start=None, pos=None,
               seq=None, slots=None, workspace=None):
        """Make room for n_new [n_seq] more tokens of each sequence -> (new_start
        [n_seq + 1], pos, seq [n_tokens] int32, slots [n_tokens] int64).  free
        [n_pages], of which the first n_free [1] are free pages (as refs returns
        them): the last of them are taken first, entered into page_table and off
        n_free.  A sequence gets room for all of its new tokens or, where its row,
        the n_tokens rows or the free pages do not suffice for it and those before it,
        for none.  lens and n_free are updated in place unless lens_out and n_free_out
        are given.  pos, seq, slots: each row's position, sequence and page * page_size
        + place, -1 past the last row (or without a page)."""
        torch = _torch()
        table, stride, width = self._table(page_table, lens)
        n, dev, int32 = page_table.shape[0], self.device, torch.int32
        _is(n_new, int32, (n,), dev, "n_new")
        _is(free, int32, (self.n_pages,), dev, "free")
        _is(n_free, int32, (1,), dev, "n_free")
        _count(n_tokens)
        if lens_out is None:
            lens_out = lens
        if n_free_out is None:
            n_free_out = n_free

        def made(t, shape, dtype, what):
            if t is None:
                return torch.empty(shape, dtype=dtype, device=dev)
            _is(t, dtype, shape, dev, what)
            return t

        _is(lens_out, int32, (n,), dev, "lens_out")
        _is(n_free_out, int32, (1,), dev, "n_free_out")
        new_start = made(new_start, (n + 1,), int32, "new_start")
        pos, seq = made(pos, (n_tokens,), int32, "pos"), made(seq, (n_tokens,), int32, "seq")
        slots = made(slots, (n_tokens,), torch.int64, "slots")
        if workspace is None:
            workspace = self.extend_workspace(n)
        a = L.LlapisKvExtendArgs(self.page_size, self.n_pages, n, n_tokens, width, 0, stride, table, lens.data_ptr(),
                                 n_new.data_ptr(), free.data_ptr(), n_free.data_ptr(), lens_out.data_ptr(),
                                 n_free_out.data_ptr(), new_start.data_ptr(), pos.data_ptr(), seq.data_ptr(), slots.data_ptr())
        _call("llapis_kv_extend", dev, C.byref(a), *_scratch(workspace, dev))
        return new_start, pos, seq, slots


def rope_frequencies(rot_dim, base=10000.0, kind=L.ROPE_PLAIN, factor=1.0, trained=0.0, low=1.0, high=None, divisors=None,
                     device="cuda"):
    """(freq float64 [rot_dim / 2] on `device`, magnitude): the frequencies of a
    rotation of rot_dim values, computed on the host.  kind: ROPE_PLAIN,
    ROPE_LINEAR, ROPE_NTK, ROPE_YARN or ROPE_BANDS, stretched by `factor` over the
    `trained` length; low and high (32, for ROPE_BANDS 4): the turns over that length
    from which a frequency starts to be kept and is kept whole; divisors [rot_dim /
    2]: numbers that the frequencies are divided by."""
    torch = _torch()
    n = max(rot_dim // 2, 0)
    if divisors is not None:
        divisors = torch.as_tensor(divisors, dtype=torch.float64, device="cpu").contiguous()
        _need(divisors.shape == (n,), f"divisors must be {n} numbers")
    freq, magnitude = torch.empty(n, dtype=torch.float64), C.c_float()
    rule = L.LlapisRopeRule(kind, rot_dim, base, factor, trained, low, (4.0 if kind == L.ROPE_BANDS else 32.0) if high is None else high,
                            _ptr(divisors))
    check(lib().llapis_rope_frequencies(C.byref(rule), freq.data_ptr(), C.byref(magnitude)), "llapis_rope_frequencies")
    return freq.to(device), magnitude.value


def qk_rope(q, k=None, pos=None, freq=None, q_weight=None, k_weight=None, norm=True, eps=1e-6, magnitude=1.0, layout=L.ROPE_HALF,
            q_out=None, k_out=None):
    """Norm each head of q [T, n_head, head_dim] and k [T, n_kv, head_dim] (None:
    no k; float32, float16 or bfloat16) and turn its first 2 len(freq) values by
    pos [T] (int32) times freq (float64; None: not turned) -> (q_out, k_out), which may be q and k.
    norm: x / rms(x) * weight, weights float32 [head_dim] or None; layout:
    ROPE_HALF pairs value i with i + len(freq), ROPE_PAIRS 2 i with 2 i + 1;
    magnitude: factor on cosine and sine.  Rows with a negative position are
    left as they are (in outputs made here: as the allocation holds them)."""
    torch = _torch()
    shape, dtype, dev = q.shape, q.dtype, _on_gpu(q, "q")
    _need(len(shape) == 3, "q must be [T, n_head, head_dim]")
    T, n_head, D = shape
    if (T | n_head | D) >> 31:
        _count(T, n_head, D)

    def heads(t, n, what):
        stride = t.stride()
        if (t.shape != (T, n, D) or t.dtype != dtype or t.device != dev or (stride[2] != 1 and D > 1)
                or (stride[1] != D and n > 1)):
            raise ValueError(f"{what} must be [{T}, {n}, {D}] of q's type and device, rows of consecutive values")
        return t.data_ptr(), stride[0]

    rot = 0
    if freq is not None:
        rot = 2 * freq.shape[0]
        _is(freq, torch.float64, (rot // 2,), dev, "freq")
        _need(pos is not None, "freq needs pos")
    if pos is not None:
        _is(pos, torch.int32, (T,), dev, "pos")
    if q_out is None:
        q_out = torch.empty(shape, dtype=dtype, device=dev)
    n_kv, k_in, k_to = 0, (None, 0), (None, 0)
    if k is not None:
        _need(k.dim() == 3, "k must be [T, n_kv, head_dim]")
        n_kv = k.shape[1]
        if n_kv >> 31:
            _count(n_kv)
        if k_out is None:
            k_out = torch.empty(k.shape, dtype=dtype, device=dev)
        k_in, k_to = heads(k, n_kv, "k"), heads(k_out, n_kv, "k_out")
    for w in (q_weight, k_weight):
        if w is not None:
            _is(w, torch.float32, (D,), dev, "weights")
    a = L.LlapisQkRopeArgs(_tag(dtype), T, n_head, n_kv, D, rot, layout, int(norm), eps, magnitude, _ptr(pos), _ptr(freq),
                           *heads(q, n_head, "q"), *heads(q_out, n_head, "q_out"), _ptr(q_weight), *k_in, *k_to, _ptr(k_weight))
    _call("llapis_qk_rope", dev, C.byref(a))
    return q_out, k_out


def block_norm(h, y=None, post_weight=None, post_norm=True, gate=None, alpha=1.0, beta=1.0, weights=(), eps=1e-6,
               h_out=None, out=None):
    """h' = alpha h + beta gate u, u = rms_norm(y) * post_weight (post_norm) or
    y; x_j = rms_norm(h') * weights[j] -> (h', [x_0, ...]).  h, y [T, d] of
    float32, float16 or bfloat16; gate of that type, [T, d], [1, d], [T, 1] or
    [1, 1]; weights float32 [d] or None each (at most 4), post_weight too.  h_out
    may be h; out: the x_j's tensors."""
    torch = _torch()
    shape, dtype, dev = h.shape, h.dtype, _on_gpu(h, "h")
    _need(len(shape) == 2 and h.stride(1) == 1, "h must be [T, d], rows of consecutive values")
    T, d = shape
    if (T | d) >> 31:
        _count(T, d)

    def row(t, what):
        stride = t.stride()
        if t.shape != shape or t.dtype != dtype or t.device != dev or stride[1] != 1:
            raise ValueError(f"{what} must be shaped and typed as h, rows of consecutive values")
        return t.data_ptr(), stride[0]

    n_out = len(weights)
    _need(n_out <= L.NORM_MAX_OUT, "at most 4 outputs")
    y_row = (None, 0) if y is None else row(y, "y")
    if post_weight is not None:
        _is(post_weight, torch.float32, (d,), dev, "post_weight")
    gate_at = (None, 0, 0)
    if gate is not None:
        gs, stride = gate.shape, gate.stride()
        _need(len(gs) == 2 and gs[0] in (1, T) and gs[1] in (1, d) and gate.dtype == dtype and gate.device == dev
              and (gs[1] == 1 or stride[1] == 1), "gate must be [T or 1, d or 1] of h's type, rows of consecutive values")
        gate_at = gate.data_ptr(), stride[0] if gs[0] > 1 else 0, 1 if gs[1] > 1 else 0
    if h_out is None:
        h_out = torch.empty(T, d, dtype=dtype, device=dev)
    if out is None:
        out = [torch.empty(T, d, dtype=dtype, device=dev) for _ in weights]
    _need(len(out) == n_out, "out needs a tensor for each of weights")
    a = L.LlapisBlockNormArgs(_tag(dtype), T, d, n_out, int(post_norm), eps, alpha, beta, h.data_ptr(), h.stride(0), *y_row,
                              _ptr(post_weight), *gate_at, *row(h_out, "h_out"))
    w_at, x_at, x_stride = a.weight, a.x, a.x_stride
    for i, x in enumerate(out):
        w = weights[i]
        if w is not None:
            _is(w, torch.float32, (d,), dev, "weights")
            w_at[i] = w.data_ptr()
        x_at[i], x_stride[i] = row(x, "out")
    _call("llapis_block_norm", dev, C.byref(a))
    return h_out, out


def sample_workspace(n_seq, vocab, device="cuda"):
    """Scratch for sample, for a caller that keeps it: calls that share it must not overlap."""
    return _bytes("llapis_sample_workspace_size", device, n_seq, vocab)


def sample(logits, u, temperature=None, top_k=None, top_p=None, min_p=None, tokens=None, probs=None, workspace=None):
    """The next token of each sequence -> tokens [n_seq] int32, from logits [n_seq,
    vocab] (float32, float16 or bfloat16) and u [n_seq] float32 in [0, 1): softmax at
    the temperature, the top_k most probable (0: all), of those the fewest whose
    probability is top_p of theirs (1: all), of those the ones of at least min_p
    times the largest probability; the first token in the vocabulary's order at which the sum of what is left
    passes u of the whole.  Settings are tensors [n_seq] (float32, top_k int32) or None:
    temperature 1, the others off; a temperature of 0 takes the most probable.  Ties go
    to the lowest index.  probs [n_seq, vocab] of the logits' type receives the
    probabilities drawn with, as verify_drafts takes them."""
    torch = _torch()
    shape, dtype, dev = logits.shape, logits.dtype, _on_gpu(logits, "logits")
    _need(len(shape) == 2, "logits must be [n_seq, vocab]")
    S, V = shape
    if (S | V) >> 31:
        _count(S, V)
    f32 = torch.float32

    def rows(t, what):
        stride = t.stride()
        if t.shape != shape or t.dtype != dtype or t.device != dev or (V > 1 and stride[1] != 1):
            raise ValueError(f"{what} must be [{S}, {V}] of the logits' type and device, rows of consecutive values")
        return t.data_ptr(), stride[0] if S > 1 else V

    _is(u, f32, (S,), dev, "u")
    for t, dt, what in ((temperature, f32, "temperature"), (top_k, torch.int32, "top_k"), (top_p, f32, "top_p"), (min_p, f32, "min_p")):
        if t is not None:
            _is(t, dt, (S,), dev, what)
    if tokens is None:
        tokens = torch.empty(S, dtype=torch.int32, device=dev)
    _is(tokens, torch.int32, (S,), dev, "tokens")
    if workspace is None:
        workspace = sample_workspace(S, V, dev)
    a = L.LlapisSampleArgs(_tag(dtype), S, V, *rows(logits, "logits"), u.data_ptr(), _ptr(temperature), _ptr(top_k), _ptr(top_p),
                           _ptr(min_p), tokens.data_ptr(), *((None, 0) if probs is None else rows(probs, "probs")))
    _call("llapis_sample", dev, C.byref(a), *_scratch(workspace, dev))
    return tokens


def verify_workspace(n_seq, vocab, device="cuda"):
    """Scratch for verify_drafts, for a caller that keeps it: calls that share it must not overlap."""
    n = int(lib().llapis_verify_drafts_workspace_size(n_seq, vocab))
    return _torch().empty(n, dtype=_torch().uint8, device=device)


def verify_drafts(target, draft, drafts, u, u_next, n_draft=None, tokens=None, accepted=None, workspace=None):
    """Take drafted tokens from the front while u q(x) < p(x) and draw the next
    one from what is left -> (tokens [n_seq, n + 1] int32, the taken drafts, the
    next token, -1 behind; accepted [n_seq] int32).  target [n_seq, n + 1,
    vocab] and draft [n_seq, n, vocab] (None: the drafts were certain)
    probabilities, drafts [n_seq, n] int32, u [n_seq, n] and u_next [n_seq]
    float32 in [0, 1), n_draft [n_seq] int32 where sequences have fewer drafts."""
    torch = _torch()
    shape, dtype, dev = target.shape, target.dtype, _on_gpu(target, "target")
    _need(len(shape) == 3 and shape[1] > 0, "target must be [n_seq, drafts + 1, vocab]")
    S, n, V = shape[0], shape[1] - 1, shape[2]
    if (S | n | V) >> 31:
        _count(S, n, V)

    def rows(t, k, what):
        stride = t.stride()
        if (t.shape != (S, k, V) or t.dtype != dtype or t.device != dev or stride[2] != 1
                or (S > 1 and k > 1 and stride[0] != k * stride[1])):
            raise ValueError(f"{what} must be [{S}, {k}, {V}] of target's type, rows evenly spaced")
        # a sequence's rows follow each other; with one row each, the sequences' do
        return t.data_ptr(), (stride[1] if k > 1 else stride[0]) if S * k > 1 else V

    target_rows = rows(target, n + 1, "target")
    draft_rows = rows(draft, n, "draft") if draft is not None and n > 0 else (None, 0)
    _is(drafts, torch.int32, (S, n), dev, "drafts")
    _is(u, torch.float32, (S, n), dev, "u")
    _is(u_next, torch.float32, (S,), dev, "u_next")
    if n_draft is not None:
        _is(n_draft, torch.int32, (S,), dev, "n_draft")
    if tokens is None:
        tokens = torch.empty(S, n + 1, dtype=torch.int32, device=dev)
    if accepted is None:
        accepted = torch.empty(S, dtype=torch.int32, device=dev)
    _is(tokens, torch.int32, (S, n + 1), dev, "tokens")
    _is(accepted, torch.int32, (S,), dev, "accepted")
    if workspace is None:
        workspace = verify_workspace(S, V, dev)
    a = L.LlapisVerifyArgs(_tag(dtype), S, n, V, *target_rows, *draft_rows, drafts.data_ptr(), _ptr(n_draft), u.data_ptr(),
                           u_next.data_ptr(), tokens.data_ptr(), accepted.data_ptr())
    _call("llapis_verify_drafts", dev, C.byref(a), *_scratch(workspace, dev))
    return tokens, accepted
