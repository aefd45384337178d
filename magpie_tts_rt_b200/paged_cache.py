"""Paged key/value cache shared by many token sequences, and the attention
that reads it (C ABI section 7 of include/magpie_tts_rt_b200.h).

``PagedCache`` holds a pool of pages ``[pages, layers, 2, kv_heads, page_size,
head_dim]`` (keys at index 0, values at 1), a page table and a length per
slot, and a reference count per page, all on the device:

* ``extend`` / ``store``: room for new tokens, and their keys and values;
* ``fork``: slots take over other slots' tokens, full pages shared (sessions
  started from one prefilled voice; reordering of slots);
* ``free`` / ``compact``: slots closed, pages in use moved to the pool's start;
* ``attend``: attention of each slot's newest token, or of runs of new tokens
  (a prompt), with an optional sliding window and a few first tokens
  (``sinks``) that stay visible;
* ``attend_shared``: the newest tokens' attention where groups of slots share a
  prefix (``PrefixGroups``), computed once for each group.

Every call is enqueued on the current (or given) CUDA stream of the pool's
device and returns without waiting; no gradient is recorded (this is a decoder's
cache).  What an upkeep call cannot do on the device (no free page, rows that do
not fit) it reports in ``status``; what can be seen on the host (types, shapes,
strides, streams of another device) raises ValueError before anything is
launched.

Calls that change a cache, and the calls that read it, must be ordered with
each other by the caller when they use different streams; a tensor given to a
call on another stream than its own is the caller's to keep until the call is
done.  Every call can be captured into a CUDA graph after one such call on the
capturing stream (which makes that stream's workspace).  A graph goes on using
that workspace: its replays must be ordered with that stream's other calls, and
with the replays of other graphs captured on it.
"""
from __future__ import annotations

import bisect
import contextlib
import ctypes
import itertools
from typing import Optional

import torch

from magpie_tts_rt_b200 import _lib as L

PAGE_SIZES = (16, 32, 64, 128)
HEAD_DIMS = (64, 128)
MAX_SLOTS = 16384
MAX_GROUP = 64
MAX_ROWS = 1 << 22
MAX_TOKENS = 1 << 30  # more than a slot can have
_DTYPES = {torch.bfloat16: L.DTYPE_BF16, torch.float16: L.DTYPE_F16}


def _check(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(what)


# the current device's index (torch.cuda.current_device takes several times as long)
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


def _raw_stream(device: torch.device):
    """A function that returns the handle of the device's current stream
    (torch.cuda.current_stream builds a Stream object for it, which costs as
    much as the rest of a small call)."""
    raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)
    if raw is None:
        return lambda index: torch.cuda.current_stream(index).cuda_stream
    return raw


class PagedCache:
    def __init__(self, pool: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor, refs: torch.Tensor):
        """Adopts the tensors of a cache: pool [pages, layers, 2, kv_heads,
        page_size, head_dim] bf16 or f16, page_table [slots, table_pages] int32
        (-1: no page), lengths [slots] int32, refs [pages] int32; contiguous
        and on one CUDA device."""
        _check(pool.is_cuda, "the pool must be a CUDA tensor")
        _check(pool.dim() == 6 and pool.shape[2] == 2, "pool must be [pages, layers, 2, kv_heads, page_size, head_dim]")
        _check(pool.dtype in _DTYPES, "pool must be bfloat16 or float16")
        pages, layers, _, kv_heads, page_size, head_dim = pool.shape
        _check(min(pages, layers, kv_heads) >= 1, "a pool needs a page, a layer and a key head")
        _check(page_size in PAGE_SIZES, f"page_size must be one of {PAGE_SIZES}")
        _check(head_dim in HEAD_DIMS, f"head_dim must be one of {HEAD_DIMS}")
        _check(page_table.dim() == 2 and min(page_table.shape) >= 1, "page_table must be [slots, table_pages]")
        slots, table_pages = page_table.shape
        _check(slots <= MAX_SLOTS, f"at most {MAX_SLOTS} slots")
        _check(tuple(lengths.shape) == (slots,), "lengths must be [slots]")
        _check(tuple(refs.shape) == (pages,), "refs must be [pages]")
        for name, t in (("page_table", page_table), ("lengths", lengths), ("refs", refs)):
            _check(t.dtype == torch.int32, f"{name} must be int32")
        for name, t in (("pool", pool), ("page_table", page_table), ("lengths", lengths), ("refs", refs)):
            _check(t.is_contiguous(), f"{name} must be contiguous")
            _check(t.device == pool.device, f"{name} is on another device than the pool")
        _check(pool.data_ptr() % 128 == 0 and refs.data_ptr() % 16 == 0,
               "the pool must be 128-byte aligned, refs 16-byte aligned")
        self.pool, self.page_table, self.lengths, self.refs = pool, page_table, lengths, refs
        self.device = pool.device
        self._index = pool.device.index
        self._raw = _raw_stream(pool.device)
        self.dtype = pool.dtype
        self.pages, self.layers, self.kv_heads, self.page_size, self.head_dim = (
            pages, layers, kv_heads, page_size, head_dim)
        self.slots, self.table_pages = slots, table_pages
        self.status = torch.zeros(slots, dtype=torch.int32, device=self.device)
        self.live = torch.zeros(1, dtype=torch.int32, device=self.device)
        self.refused = torch.zeros(slots, dtype=torch.int32, device=self.device)
        c = L.PagedCache()
        c.pages, c.layers, c.kv_heads, c.page_size, c.head_dim = pages, layers, kv_heads, page_size, head_dim
        c.dtype, c.slots, c.table_pages = _DTYPES[pool.dtype], slots, table_pages
        c.pool, c.page_table, c.lengths, c.refs = (t.data_ptr() for t in (pool, page_table, lengths, refs))
        c.status, c.live, c.refused = (t.data_ptr() for t in (self.status, self.live, self.refused))
        self._c = c
        self._ref = ctypes.byref(c)
        self._scale = head_dim ** -0.5
        self._streams = set()  # that calls were made on
        self._spaces = {}  # (stream, query heads) -> workspace
        self._outgrown = []
        _check(L.lib.mtt_b200_paged_cache_workspace_size(self._ref, kv_heads, 0) > 0, "this cache is too large")

    @staticmethod
    def allocate(pages: int, slots: int, max_tokens: int, layers: int, kv_heads: int, head_dim: int,
                 page_size: int = 16, dtype: torch.dtype = torch.bfloat16, device="cuda") -> "PagedCache":
        """An empty cache: no slot has tokens, every page is free (the pool is not cleared)."""
        _check(page_size in PAGE_SIZES, f"page_size must be one of {PAGE_SIZES}")
        _check(max_tokens >= 1, "max_tokens must be at least 1")
        table_pages = (max_tokens + page_size - 1) // page_size
        i32 = dict(dtype=torch.int32, device=device)
        return PagedCache(
            pool=torch.empty(pages, layers, 2, kv_heads, page_size, head_dim, dtype=dtype, device=device),
            page_table=torch.full((slots, table_pages), -1, **i32), lengths=torch.zeros(slots, **i32),
            refs=torch.zeros(pages, **i32))

    # -- plumbing -----------------------------------------------------------

    def _handle(self, stream) -> int:
        if stream is None:
            handle = self._raw(self._index)
        elif stream.device.index == self._index:
            handle = stream.cuda_stream
        else:
            raise ValueError("the stream belongs to another device than the pool")
        if handle not in self._streams:
            self._keep(stream, self.pool, self.page_table, self.lengths, self.refs, self.status, self.live, self.refused)
            self._streams.add(handle)
        return handle

    def _keep(self, stream, *tensors) -> None:
        """Tensors that calls on this stream use, whichever stream they were made
        on: when they are dropped, their memory is not reused before those calls
        are done."""
        if stream is None:
            stream = torch.cuda.current_stream(self.device)
        for t in tensors:
            t.record_stream(stream)

    def _workspace(self, handle: int, stream, q_heads: int, rows: int = 0):
        """(address, bytes) of the workspace of calls on one stream: kept, and
        one for each stream, as the streams' calls may overlap."""
        space = self._spaces.get((handle, q_heads))
        if space is None or rows > space[2]:
            most = max(1024, 1 << (rows - 1).bit_length()) if rows else 0
            size = L.lib.mtt_b200_paged_cache_workspace_size(self._ref, q_heads, most)
            _check(size > 0, "this cache and number of heads or rows are not supported")
            with self._on(stream):
                data = torch.empty(size, dtype=torch.uint8, device=self.device)
            if space is not None:
                self._outgrown.append(space)  # a CUDA graph captured with it may still replay
            space = self._spaces[handle, q_heads] = (data.data_ptr(), size, most, data)
        return space

    @staticmethod
    def _on(stream):
        """Where a call's own tensors are allocated: the stream that the caller gave, if any."""
        return contextlib.nullcontext() if stream is None else torch.cuda.stream(stream)

    def _vector(self, t: torch.Tensor, n: int, dtype: torch.dtype, name: str) -> int:
        if t.dtype is not dtype or t.shape != (n,) or t.get_device() != self._index or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous {dtype} vector of {n} on the pool's device")
        return t.data_ptr()

    def _call(self, name: str, *args) -> None:
        """One launch, on the pool's device whichever is current."""
        call = getattr(L.lib, name)
        if _current_device() == self._index:
            rc = call(*args)
        else:
            with torch.cuda.device(self._index):
                rc = call(*args)
        if rc != L.STATUS_OK:
            raise RuntimeError(f"{name} failed with status {rc}")

    # -- upkeep -------------------------------------------------------------

    def extend(self, counts: torch.Tensor, stream=None) -> None:
        """lengths += counts ([slots] int32), with the pages that takes.  A slot
        that does not get them stays as it is, and ``store`` leaves it alone until
        the next ``extend`` (``refused`` [slots])."""
        at = self._vector(counts, self.slots, torch.int32, "counts")
        handle = self._handle(stream)
        ws = self._workspace(handle, stream, self.kv_heads)
        self._call("mtt_b200_launch_paged_cache_extend", self._ref, at, ws[0], ws[1], handle)

    def fork(self, source: torch.Tensor, deep: bool = False, stream=None) -> None:
        """Slot d takes over the tokens that slot source[d] had before the call
        (source [slots] int32; -1 or d: slot d stays).  Full pages are shared
        unless ``deep``, a partial last page is always copied."""
        at = self._vector(source, self.slots, torch.int32, "source")
        handle = self._handle(stream)
        ws = self._workspace(handle, stream, self.kv_heads)
        self._call("mtt_b200_launch_paged_cache_fork", self._ref, at, 1 if deep else 0, ws[0], ws[1], handle)

    def free(self, mask: torch.Tensor, stream=None) -> None:
        """Closes every slot with mask ([slots] bool): its pages are released."""
        at = self._vector(mask, self.slots, torch.bool, "mask")
        self._call("mtt_b200_launch_paged_cache_free", self._ref, at, self._handle(stream))

    def compact(self, stream=None) -> None:
        """Moves the pages in use to [0, live); ``live`` [1] holds their number."""
        handle = self._handle(stream)
        ws = self._workspace(handle, stream, self.kv_heads)
        self._call("mtt_b200_launch_paged_cache_compact", self._ref, ws[0], ws[1], handle)

    def store(self, k: torch.Tensor, v: torch.Tensor, layer: Optional[int] = None,
              offsets: Optional[torch.Tensor] = None, stream=None) -> None:
        """Writes the keys and values of each slot's last tokens: rows
        [offsets[i], offsets[i + 1]) are slot i's (offsets [slots + 1] int32), or,
        without offsets, row i is slot i's last token.  With ``layer`` k and v are
        [rows, kv_heads, head_dim]; without it [layers, rows, kv_heads, head_dim],
        every layer at once.  The last two dimensions must be contiguous.  Rows of
        slots whose tokens ``extend`` has refused are not written."""
        shape, ks, vs = k.shape, k.stride(), v.stride()
        if (len(shape) != (4 if layer is None else 3) or v.shape != shape or shape[-1] != self.head_dim or
                shape[-2] != self.kv_heads):
            raise ValueError("k and v must be [rows, kv_heads, head_dim], or [layers, rows, kv_heads, head_dim] without a "
                             "layer, with the cache's heads")
        args = L.CacheRows()
        if layer is None:
            _check(shape[0] == self.layers, "k and v have other layers than the cache")
            args.n_layers = self.layers
        else:
            _check(0 <= layer < self.layers, "no such layer")
            args.layer, args.n_layers = layer, 1
        args.rows = shape[-3]
        args.k, args.v = k.data_ptr(), v.data_ptr()
        args.k_row_stride = self._rows_of(k, shape[-3:], ks[-3:], "k")
        args.v_row_stride = self._rows_of(v, shape[-3:], vs[-3:], "v")
        if layer is None and shape[0] > 1:  # the stride of a dimension of one has no meaning
            args.k_layer_stride, args.v_layer_stride = ks[0], vs[0]
            if ks[0] % 8 or vs[0] % 8:
                raise ValueError("layers of k and v must be 16-byte aligned")
        if offsets is not None:
            args.offsets = self._vector(offsets, self.slots + 1, torch.int32, "offsets")
        else:
            _check(args.rows <= self.slots, "more rows than slots: offsets are needed")
        self._call("mtt_b200_launch_paged_cache_store", self._ref, ctypes.byref(args), self._handle(stream))

    # -- attention ----------------------------------------------------------

    def _attention(self, layer, q, out, window, sinks, scale, return_lse, stream):
        """The fields that the attention calls share; (args, out, lse)."""
        shape, st, d = q.shape, q.stride(), self.head_dim
        if len(shape) != 3 or shape[2] != d:
            raise ValueError("q must be [rows, q_heads, head_dim]")
        rows, q_heads, _ = shape
        if q_heads < 1 or q_heads % self.kv_heads or q_heads // self.kv_heads > MAX_GROUP:
            raise ValueError(f"q_heads must be a multiple of kv_heads, at most {MAX_GROUP} query heads per key head")
        if rows > MAX_ROWS:
            raise ValueError(f"at most {MAX_ROWS} rows")
        if not 0 <= layer < self.layers:
            raise ValueError("no such layer")
        if window < 0 or sinks < 0:
            raise ValueError("window and sinks must not be negative")
        window, sinks = min(window, MAX_TOKENS), min(sinks, MAX_TOKENS)  # the struct's fields would wrap
        if scale is None:
            scale = self._scale
        elif not 0 < scale < float("inf"):
            raise ValueError("scale must be positive")
        if out is None:
            with self._on(stream):
                out = torch.empty(shape, dtype=self.dtype, device=self.device)
            out_row = q_heads * d
        else:
            if out.shape != shape:
                raise ValueError("out must have q's shape")
            out_row = self._rows_of(out, shape, out.stride(), "out")
        q_row = self._rows_of(q, shape, st, "q")
        lse = None
        args = L.CacheAttention(layer, q_heads, rows, window, sinks, scale, q.data_ptr(), q_row, out.data_ptr(), out_row)
        if return_lse:
            with self._on(stream):
                lse = torch.empty((rows, q_heads), dtype=torch.float32, device=self.device)
            args.lse = lse.data_ptr()
        return args, out, lse

    def _rows_of(self, t, shape, st, name) -> int:
        """The stride of t's rows [rows, heads, head_dim]; that of a dimension of
        one has no meaning and is not looked at."""
        if t.dtype is not self.dtype or t.get_device() != self._index:
            raise ValueError(f"{name} must have the pool's type and device")
        if st[2] != 1 or (st[1] != self.head_dim and shape[1] > 1):
            raise ValueError(f"{name} must be contiguous in its heads")
        row = st[0] if shape[0] > 1 else shape[1] * self.head_dim
        if t.data_ptr() % 16 or row % 8:
            raise ValueError(f"rows of {name} must be 16-byte aligned")
        return row

    def attend(self, layer: int, q: torch.Tensor, out: Optional[torch.Tensor] = None, *,
               offsets: Optional[torch.Tensor] = None, window: int = 0, sinks: int = 0,
               scale: Optional[float] = None, key_mask: Optional[torch.Tensor] = None, return_lse: bool = False,
               stream=None):
        """Attention of q [rows, q_heads, head_dim] over one layer of the cache.

        Without offsets row i is the last token of slot i (a decode step); with
        offsets ([slots + 1] int32) rows [offsets[i], offsets[i + 1]) are slot i's
        last tokens, whose keys and values are already stored (a prompt).  A
        query sees the keys up to its own position, those less than ``window``
        back (0: all) or among the first ``sinks``, and of these the ones with
        key_mask ([slots, >= table_pages * page_size] bool).  A row that sees
        none gets 0, and so does one that no slot has (offsets may end before the
        last row, or begin after the first).  Returns out, or (out, lse) with the natural log of the sum
        of exponentials ([rows, q_heads] f32, -inf for a row that sees none)."""
        args, out, lse = self._attention(layer, q, out, window, sinks, scale, return_lse, stream)
        if offsets is not None:
            args.offsets = self._vector(offsets, self.slots + 1, torch.int32, "offsets")
        elif args.rows > self.slots:
            raise ValueError("more rows than slots: offsets are needed")
        if key_mask is not None:
            _check(key_mask.dtype is torch.bool and key_mask.dim() == 2 and key_mask.shape[0] == self.slots and
                   key_mask.shape[1] >= self.table_pages * self.page_size and key_mask.stride(1) == 1 and
                   key_mask.get_device() == self._index and
                   (self.slots == 1 or key_mask.stride(0) >= key_mask.shape[1]),
                   "key_mask must be a [slots, >= table_pages * page_size] bool tensor with contiguous rows")
            args.key_mask, args.mask_stride = key_mask.data_ptr(), max(key_mask.stride(0), key_mask.shape[1])
        handle = self._handle(stream)
        ws = self._workspace(handle, stream, args.q_heads, args.rows)
        self._call("mtt_b200_launch_paged_attention", self._ref, ctypes.byref(args), ws[0], ws[1], handle)
        return (out, lse) if return_lse else out

    def attend_shared(self, layer: int, q: torch.Tensor, groups: "PrefixGroups", out: Optional[torch.Tensor] = None, *,
                      window: int = 0, sinks: int = 0, scale: Optional[float] = None, return_lse: bool = False,
                      stream=None):
        """``attend`` without offsets for slots that share prefixes: the keys and
        values of a group's prefix are read and multiplied once for all its
        members.  Slots in no group, slots that no longer hold their group's
        pages, and groups whose prefix is longer than ``sinks`` under a window
        are attended one by one; the result is the same."""
        _check(groups.cache is self, "these groups belong to another cache")
        args, out, lse = self._attention(layer, q, out, window, sinks, scale, return_lse, stream)
        _check(args.q_heads == groups.q_heads, "these groups were made for another number of heads")
        _check(args.rows <= self.slots, "more rows than slots")
        handle = self._handle(stream)
        ws = groups._workspace(handle, stream)
        self._call("mtt_b200_launch_paged_attention_shared", self._ref, ctypes.byref(args), groups._seen(window, sinks),
                   ws[0], ws[1], handle)
        return (out, lse) if return_lse else out


class PrefixGroups:
    """Which slots of a cache share which prefix, for ``attend_shared``: made
    when sessions open or close, used for every layer of every step between.

    groups: (voice, tokens, members) for each: the members' first ``tokens``
    tokens are those of slot ``voice``, on the same pages (the members were
    forked from it; the voice itself may be one of them).  ``tokens`` is
    rounded down to full pages.  The voice must stay open while the groups are
    used; a member whose slot has been closed or reopened since is attended on
    its own.  Groups may be dropped while calls that use them are still queued, but
    must outlive CUDA graphs captured with them."""

    def __init__(self, cache: PagedCache, groups, q_heads: int):
        _check(q_heads >= 1 and q_heads % cache.kv_heads == 0 and q_heads // cache.kv_heads <= MAX_GROUP,
               f"q_heads must be a multiple of kv_heads, at most {MAX_GROUP} query heads per key head")
        voices, tokens, offsets, members = [], [], [0], []
        for voice, count, slots in groups:
            _check(0 <= voice < cache.slots, "no such voice slot")
            _check(0 <= count <= cache.table_pages * cache.page_size, "a prefix longer than a slot")
            _check(all(0 <= s < cache.slots for s in slots), "no such member slot")
            count = count // cache.page_size * cache.page_size
            if count == 0 or len(slots) == 0:
                continue
            voices.append(voice)
            tokens.append(count)
            members.extend(slots)
            offsets.append(len(members))
        _check(len(set(members)) == len(members), "a slot can be in one group only")
        self.cache, self.q_heads = cache, q_heads
        self.n_members = len(members)
        n = len(voices)
        self._data = torch.tensor(voices + tokens + offsets + members, dtype=torch.int32).to(cache.device)
        at = self._data.data_ptr()
        c = L.PrefixGroups()
        c.n_groups, c.n_members = n, len(members)
        c.voice, c.tokens, c.offsets, c.members = at, at + 4 * n, at + 8 * n, at + 4 * (3 * n + 1)
        c.shared_tokens = sum(t * (b - a) for t, a, b in zip(tokens, offsets, offsets[1:]))
        self._c = c
        self._ref = ctypes.byref(c)
        self._spaces = {}
        # prefix lengths in order, and the members' tokens of the groups up to each
        sizes = sorted((t, t * (b - a)) for t, a, b in zip(tokens, offsets, offsets[1:]))
        self._lengths = [t for t, _ in sizes]
        self._shared_up_to = [0] + list(itertools.accumulate(n for _, n in sizes))

    def _seen(self, window: int, sinks: int):
        """The groups for a call: under a window only prefixes among the sinks are
        shared, so only these speak for the prefix pass, and without one there is
        none."""
        n = len(self._lengths) if window == 0 else bisect.bisect_right(self._lengths, sinks)
        if n == len(self._lengths):
            return self._ref
        c = L.PrefixGroups.from_buffer_copy(self._c)
        if n == 0:
            c.n_groups = c.n_members = 0
        elif c.shared_tokens > 0:
            c.shared_tokens = self._shared_up_to[n]
        return ctypes.byref(c)

    def _workspace(self, handle: int, stream):
        space = self._spaces.get(handle)
        if space is None:
            size = L.lib.mtt_b200_paged_shared_workspace_size(self.cache._ref, self.q_heads, self.n_members)
            with PagedCache._on(stream):
                data = torch.empty(size, dtype=torch.uint8, device=self.cache.device)
            self.cache._keep(stream, self._data)
            space = self._spaces[handle] = (data.data_ptr(), size, data)
        return space
