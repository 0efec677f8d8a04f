"""A paged fp16 K/V cache of many sequences on one MI355X: the operators of
include/hq.h's paged cache and `PagedCache`, which holds its tensors.

Sequence b's pages stand in order in row b of `table` (int32 [sequences,
max_pages], -1: none), its positions in `lengths` (int32 [sequences]), and
`refs` (int32 [pages]) counts the table entries that hold each page, so that
sequences may share pages.  A layer's keys and values are float16 [pages,
kv_heads, page_size, head_dim].  All of it lives on the device and every
operator reads it there: a captured graph of a step is valid at every length,
past page borders too.

A batch brings new tokens for some or all of the sequences: rows starts[b] ..
starts[b+1] - 1 of its tensors belong to sequence b (starts: int32 [sequences
+ 1] on the device; None: one row for every sequence).  One step of a model:

    cache.resize(new_lengths)                  # pages for the new tokens
    for layer in range(layers):
        q = cache.append(layer, qkv, ...)      # norms, rotation, K/V rows
        x = cache.attend(layer, q, ...)        # each token sees its sequence

No reference counterpart (the reference keeps one contiguous cache per
session, cpu_lightspark.py:275-309).  There is no host fallback.
"""
from __future__ import annotations

import functools
import struct

import torch

from . import _native
from ._native import check

MAX_SEQUENCES = 0xFFFFFF
PAGE_SIZES = (16, 32, 64, 128, 256)
HEAD_DIMS = (16, 32, 64, 128)
MAX_GROUPS = 8


# --------------------------------------------------------------------------- checks
# (the host's time is most of a small call's: checks written out, one attribute
# at a time, the C struct packed as bytes; of an attention call's 8.0 to 8.6 us
# they are 3.8, the launch is 3.6)
_I32, _F32, _F16 = torch.int32, torch.float32, torch.float16
_pack = struct.Struct("8i6P").pack
_current_device = torch._C._cuda_getDevice
_raw_stream = torch._C._cuda_getCurrentRawStream
_alloc = torch._C._cuda_cudaCachingAllocator_raw_alloc
_free = torch._C._cuda_cudaCachingAllocator_raw_delete


def _refuse(name: str, t, dtype, index: int, what: str):
    if isinstance(t, torch.Tensor) and t.is_cuda and t.dtype is dtype and t.get_device() != index:
        raise ValueError(f"{name} is on another device")
    raise ValueError(f"{name} must be a contiguous {str(dtype)[6:]} device tensor {what}")


def _index(table) -> int:
    if not isinstance(table, torch.Tensor) or not table.is_cuda:
        raise ValueError("table must be a contiguous int32 device tensor [sequences, max_pages]")
    return table.get_device()


def _cache(index: int, keys, values, table, lengths, refs, status, dims: int, pools: bool = True):
    """The tables' C struct (hq_pages) as bytes, after its checks, and the
    sizes the callers need; keys/values [layers, pages, kv_heads, page_size,
    head_dim] (dims 5) or one layer of them (dims 4)."""
    layers, kv_heads, page_size, head_dim = 1, 1, 16, 16
    key_ptr = value_ptr = 0
    if pools:
        if keys.dtype is not _F16 or keys.get_device() != index or not keys.is_contiguous():
            _refuse("keys", keys, _F16, index, "of pages")
        if values.dtype is not _F16 or values.get_device() != index or not values.is_contiguous():
            _refuse("values", values, _F16, index, "of pages")
        shape = keys.shape
        if len(shape) != dims:
            raise ValueError("keys must be [pages, kv_heads, page_size, head_dim]" if dims == 4 else
                             "keys must be [layers, pages, kv_heads, page_size, head_dim]")
        if values.shape != shape:
            raise ValueError("keys and values must have the same shape")
        if dims == 5:
            layers = shape[0]
        pages, kv_heads, page_size, head_dim = shape[-4:]
        if page_size not in PAGE_SIZES:
            raise ValueError(f"page_size must be one of {PAGE_SIZES}")
        if head_dim not in HEAD_DIMS:
            raise ValueError(f"head_dim must be one of {HEAD_DIMS}")
        if layers == 0 or pages == 0 or kv_heads == 0:
            raise ValueError("keys/values hold no pages")
        key_ptr, value_ptr = keys.data_ptr(), values.data_ptr()
    else:
        pages = refs.shape[0] if isinstance(refs, torch.Tensor) and refs.dim() == 1 else 0
    shape = table.shape
    if len(shape) != 2 or table.dtype is not _I32 or table.get_device() != index or not table.is_contiguous():
        _refuse("table", table, _I32, index, "[sequences, max_pages]")
    sequences, max_pages = shape
    if (sequences == 0 or max_pages == 0 or max_pages * page_size > 0x7FFFFF00 or sequences * max_pages > 0x7FFFFFFF or
            sequences > MAX_SEQUENCES):
        raise ValueError("table must be [sequences, max_pages] with fewer than 2^24 sequences, fewer than 2^31 entries "
                         "and 2^31 - 256 positions a row")
    length_ptr = ref_ptr = status_ptr = 0
    if lengths is not None:
        if (lengths.shape != (sequences,) or lengths.dtype is not _I32 or lengths.get_device() != index or
                not lengths.is_contiguous()):
            _refuse("lengths", lengths, _I32, index, "[sequences]")
        length_ptr = lengths.data_ptr()
    if refs is not None:
        if (refs.shape != (pages,) or pages == 0 or refs.dtype is not _I32 or refs.get_device() != index or
                not refs.is_contiguous()):
            _refuse("refs", refs, _I32, index, "[pages]")
        ref_ptr = refs.data_ptr()
    if status is not None:
        if status.numel() != 1 or status.dtype is not _I32 or status.get_device() != index:
            _refuse("status", status, _I32, index, "[1]")
        status_ptr = status.data_ptr()
    return (_pack(layers, pages, page_size, kv_heads, head_dim, sequences, max_pages, 0, key_ptr, value_ptr,
                  table.data_ptr(), length_ptr, ref_ptr, status_ptr), sequences, kv_heads, head_dim)


def _per_sequence(t, name: str, sequences: int, index: int) -> None:
    if t.shape != (sequences,) or t.dtype is not _I32 or t.get_device() != index or not t.is_contiguous():
        _refuse(name, t, _I32, index, "[sequences]")


def _starts(starts, sequences: int, tokens: int, index: int) -> int | None:
    if starts is None:
        if tokens != sequences:
            raise ValueError("without starts a batch has one row for every sequence")
        return None
    if (starts.shape != (sequences + 1,) or starts.dtype is not _I32 or starts.get_device() != index or
            not starts.is_contiguous()):
        _refuse("starts", starts, _I32, index, "[sequences + 1]")
    return starts.data_ptr()


def _launch(entry, args: tuple, nbytes: int | None, index: int, stream, tensors, what: str) -> None:
    """entry(*args[, workspace], stream handle) on `stream` (None: the current
    one of the tensors' GPU) with a workspace of this call alone (nbytes None:
    an entry without one): memory of any contents from torch's allocator, which
    hands it out in the stream's order and inside a capture from the graph's
    own pool (straight from it: a tensor's making takes 0.9 us more)."""
    if nbytes == 0:                            # (what the size functions return for sizes that the entries refuse)
        raise ValueError(f"{what}: sizes outside the entry's range")
    if index != _current_device():
        with torch.cuda.device(index):
            return _launch(entry, args, nbytes, index, stream, tensors, what)
    if stream is None:
        handle = _raw_stream(index)
    else:
        if stream.device.index != index:
            raise ValueError("the stream belongs to another device than the tensors")
        # the stream waits for what the caller's has enqueued, and the tensors'
        # memory is not reused before the stream is done with them
        stream.wait_stream(torch.cuda.current_stream(index))
        for t in tensors:
            if t is not None:
                t.record_stream(stream)
        handle = stream.cuda_stream
    if nbytes is None:
        status = entry(*args, handle)
    else:
        workspace = _alloc(nbytes, handle)
        try:
            status = entry(*args, workspace, handle)
        finally:
            _free(workspace)                   # (to the stream's pool: what follows on it may have it)
    if status:
        check(status, what)


def _span(t) -> tuple[int, int]:
    return t.data_ptr(), t.numel() * t.element_size()


def _apart(outputs, inputs) -> None:
    """Refuse outputs that overlap each other or an input: (address, bytes) each."""
    for i, (at, size) in enumerate(outputs):
        for other, length in inputs:
            if -length < other - at < size:
                break
        else:
            for other, length in outputs[:i]:
                if -length < other - at < size:
                    break
            else:
                continue
        raise ValueError("outputs must not overlap each other or an input")


# --------------------------------------------------------------------------- append, attention
def paged_append(qkv: torch.Tensor, q_norm: torch.Tensor, k_norm: torch.Tensor, rope_cos: torch.Tensor,
                 rope_sin: torch.Tensor, eps: float, keys: torch.Tensor, values: torch.Tensor, table: torch.Tensor,
                 lengths: torch.Tensor, status: torch.Tensor, starts: torch.Tensor | None = None,
                 out: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """One layer's new tokens into its pages (hq_paged_append): q/k head norm,
    rotation, fp16 K/V rows with the decode step's bits; returns the queries,
    float32 [tokens, heads, head_dim].  qkv: raw projection rows float32
    [tokens, (heads + 2 kv_heads) * head_dim]; `lengths` count the new tokens
    already (pages_resize)."""
    if status is None or lengths is None:
        raise ValueError("paged_append needs the cache's lengths and status")
    index = _index(table)
    cache, sequences, kv, d = _cache(index, keys, values, table, lengths, None, status, 4)
    shape = qkv.shape
    if len(shape) != 2 or qkv.dtype is not _F32 or qkv.get_device() != index or not qkv.is_contiguous():
        _refuse("qkv", qkv, _F32, index, "[tokens, (heads + 2 kv_heads) * head_dim]")
    tokens, width = shape
    heads = width // d - 2 * kv
    if width % d or heads < 1 or heads % kv or heads // kv > MAX_GROUPS:
        raise ValueError("qkv must be [tokens, (heads + 2 kv_heads) * head_dim] with 1 to 8 heads a kv head")
    if (q_norm.shape != (d,) or q_norm.dtype is not _F32 or q_norm.get_device() != index or
            not q_norm.is_contiguous()):
        _refuse("q_norm", q_norm, _F32, index, "[head_dim]")
    if (k_norm.shape != (d,) or k_norm.dtype is not _F32 or k_norm.get_device() != index or
            not k_norm.is_contiguous()):
        _refuse("k_norm", k_norm, _F32, index, "[head_dim]")
    shape = rope_cos.shape
    if (len(shape) != 2 or rope_cos.dtype is not _F32 or rope_cos.get_device() != index or
            not rope_cos.is_contiguous() or rope_sin.dtype is not _F32 or rope_sin.get_device() != index or
            not rope_sin.is_contiguous()):
        raise ValueError("rope_cos and rope_sin must be contiguous float32 device tensors of the cache's GPU")
    positions, half = shape
    if rope_sin.shape != shape or 2 * half != d or positions < 1:
        raise ValueError("rope_cos and rope_sin must be [positions, head_dim / 2]")
    first = _starts(starts, sequences, tokens, index)
    if out is None:
        out = torch.empty((tokens, heads, d), dtype=_F32, device=qkv.device)
    elif (out.shape != (tokens, heads, d) or out.dtype is not _F32 or out.get_device() != index or
          not out.is_contiguous()):
        _refuse("out", out, _F32, index, "[tokens, heads, head_dim]")
    elif -4 * out.numel() < out.data_ptr() - qkv.data_ptr() < 4 * qkv.numel():
        raise ValueError("out must not overlap qkv")
    if tokens:
        _launch(_native.lib().hq_paged_append,
                (cache, qkv.data_ptr(), first, tokens, heads, q_norm.data_ptr(), k_norm.data_ptr(), eps,
                 rope_cos.data_ptr(), rope_sin.data_ptr(), positions, out.data_ptr()), None, index, stream,
                (qkv, q_norm, k_norm, rope_cos, rope_sin, keys, values, table, lengths, status, starts, out),
                "hq_paged_append")
    return out


@functools.lru_cache(maxsize=1024)
def _attention_workspace_bytes(tokens: int, heads: int, kv_heads: int, head_dim: int, single: bool) -> int:
    return _native.lib().hq_paged_attention_workspace_bytes(tokens, heads, kv_heads, head_dim, single)


def paged_attention(query: torch.Tensor, keys: torch.Tensor, values: torch.Tensor, table: torch.Tensor,
                    lengths: torch.Tensor, starts: torch.Tensor | None = None, window: int = 0, sinks: int = 0,
                    out: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """Grouped-query attention of a batch's new tokens, float32 [tokens, heads,
    head_dim], over one layer's pages (hq_paged_attention).  The token at
    position p sees the positions up to its own that have a page; with
    `window` > 0 the last `window` of them and the first `sinks` positions.  A
    token that sees nothing gets zeros; rows past the last sequence's are not
    touched."""
    if lengths is None:
        raise ValueError("paged_attention needs the cache's lengths")
    index = _index(table)
    cache, sequences, kv, d = _cache(index, keys, values, table, lengths, None, None, 4)
    shape = query.shape
    if len(shape) != 3 or query.dtype is not _F32 or query.get_device() != index or not query.is_contiguous():
        _refuse("query", query, _F32, index, "[tokens, heads, head_dim]")
    tokens, heads, width = shape
    if width != d or heads < 1 or heads % kv or heads // kv > MAX_GROUPS:
        raise ValueError("query must be [tokens, heads, head_dim] with 1 to 8 heads a kv head")
    if not 0 <= window <= 0x7FFFFFFF or not 0 <= sinks <= 0x7FFFFFFF:
        raise ValueError("window and sinks must not be negative")
    first = _starts(starts, sequences, tokens, index)
    if out is None:
        out = torch.empty_like(query)
    elif out.shape != shape or out.dtype is not _F32 or out.get_device() != index or not out.is_contiguous():
        _refuse("out", out, _F32, index, "like query")
    elif abs(out.data_ptr() - query.data_ptr()) < 4 * tokens * heads * d:
        raise ValueError("out must not overlap query")
    if tokens:
        _launch(_native.lib().hq_paged_attention,
                (cache, query.data_ptr(), first, tokens, heads, window, sinks, out.data_ptr()),
                _attention_workspace_bytes(tokens, heads, kv, d, first is None), index, stream,
                (query, keys, values, table, lengths, starts, out), "hq_paged_attention")
    return out


# --------------------------------------------------------------------------- page management
@functools.lru_cache(maxsize=1024)
def _pages_workspace_bytes(pages: int, sequences: int, max_pages: int) -> int:
    cache = _pack(1, pages, 16, 1, 16, sequences, max_pages, 0, 0, 0, 0, 0, 0, 0)
    return _native.lib().hq_pages_workspace_bytes(cache)


def pages_resize(keys: torch.Tensor, values: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor,
                 refs: torch.Tensor, status: torch.Tensor, new_lengths: torch.Tensor, window: int = 0, sinks: int = 0,
                 stream=None) -> None:
    """Set the sequences' lengths (hq_pages_resize): int32 [sequences] on the
    device, a negative one leaves its sequence as it is.  Growth takes the
    lowest free pages, and copies the partly filled page it goes on in where
    others hold it too; shrinking releases pages, and `window` > 0 those that
    no later query sees.  Too few free pages, or a length past the table, set
    HQ_PAGES_FULL in `status` and change nothing; so does, with HQ_PAGES_BAD
    and HQ_PAGES_REFUSED, growth from the middle of a page that was
    released."""
    if lengths is None or refs is None or status is None:
        raise ValueError("pages_resize needs lengths, refs and status")
    index = _index(table)
    cache, sequences, _, _ = _cache(index, keys, values, table, lengths, refs, status, 5)
    _per_sequence(new_lengths, "new_lengths", sequences, index)
    if not 0 <= window <= 0x7FFFFFFF or not 0 <= sinks <= 0x7FFFFFFF:
        raise ValueError("window and sinks must not be negative")
    _launch(_native.lib().hq_pages_resize, (cache, new_lengths.data_ptr(), window, sinks),
            _pages_workspace_bytes(refs.shape[0], sequences, table.shape[1]), index, stream,
            (keys, values, table, lengths, refs, status, new_lengths), "hq_pages_resize")


def pages_fork(table: torch.Tensor, lengths: torch.Tensor, refs: torch.Tensor, status: torch.Tensor,
               parents: torch.Tensor, stream=None) -> None:
    """Every sequence b becomes a fork of sequence parents[b] (int32
    [sequences] on the device; negative or b: unchanged) as it was before the
    call, sharing all its pages (hq_pages_fork); what it held is released."""
    if lengths is None or refs is None or status is None:
        raise ValueError("pages_fork needs lengths, refs and status")
    index = _index(table)
    cache, sequences, _, _ = _cache(index, None, None, table, lengths, refs, status, 5, pools=False)
    _per_sequence(parents, "parents", sequences, index)
    _launch(_native.lib().hq_pages_fork, (cache, parents.data_ptr()),
            _pages_workspace_bytes(refs.shape[0], sequences, table.shape[1]), index, stream,
            (table, lengths, refs, status, parents), "hq_pages_fork")


def pages_compact(keys: torch.Tensor, values: torch.Tensor, table: torch.Tensor, refs: torch.Tensor,
                  live: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """Move the pages in use to the lowest places (hq_pages_compact), tables
    and refs with them; returns their number, int32 [1] on the device."""
    if refs is None:
        raise ValueError("pages_compact needs refs")
    index = _index(table)
    cache, sequences, _, _ = _cache(index, keys, values, table, None, refs, None, 5)
    if live is None:
        live = torch.empty(1, dtype=_I32, device=table.device)
    elif live.numel() != 1 or live.dtype is not _I32 or live.get_device() != index:
        _refuse("live", live, _I32, index, "[1]")
    _launch(_native.lib().hq_pages_compact, (cache, live.data_ptr()),
            _pages_workspace_bytes(refs.shape[0], sequences, table.shape[1]), index, stream,
            (keys, values, table, refs, live), "hq_pages_compact")
    return live


# --------------------------------------------------------------------------- the cache
class PagedCache:
    """The tensors of a paged cache (see the module) and the calls over them.

    `keys`/`values` float16 [layers, pages, kv_heads, page_size, head_dim],
    `table`, `lengths`, `refs`, and `status`, whose HQ_PAGES_* bits stay set
    until the caller clears them."""

    def __init__(self, layers: int, pages: int, kv_heads: int, head_dim: int, sequences: int, max_pages: int,
                 page_size: int = 64, device=None):
        if min(layers, pages, kv_heads, sequences, max_pages) < 1:
            raise ValueError("layers, pages, kv_heads, sequences and max_pages must be positive")
        if page_size not in PAGE_SIZES:
            raise ValueError(f"page_size must be one of {PAGE_SIZES}")
        if head_dim not in HEAD_DIMS:
            raise ValueError(f"head_dim must be one of {HEAD_DIMS}")
        if device is None:
            from .lightspark import _device
            device = _device()
        self.page_size = page_size
        ints = dict(dtype=torch.int32, device=device)
        self.keys = torch.empty((layers, pages, kv_heads, page_size, head_dim), dtype=torch.float16, device=device)
        self.values = torch.empty_like(self.keys)
        self.table = torch.full((sequences, max_pages), -1, **ints)
        self.lengths = torch.zeros(sequences, **ints)
        self.refs = torch.zeros(pages, **ints)
        self.status = torch.zeros(1, **ints)

    def _ints(self, values) -> torch.Tensor:
        if isinstance(values, torch.Tensor):
            return values
        return torch.tensor(list(values), dtype=torch.int32).to(self.table.device)

    def resize(self, new_lengths, window: int = 0, sinks: int = 0, stream=None) -> None:
        """pages_resize; a list or a device tensor of one length a sequence."""
        pages_resize(self.keys, self.values, self.table, self.lengths, self.refs, self.status,
                     self._ints(new_lengths), window, sinks, stream)

    def fork(self, parents, stream=None) -> None:
        """pages_fork; a list or a device tensor of one parent a sequence."""
        pages_fork(self.table, self.lengths, self.refs, self.status, self._ints(parents), stream)

    def compact(self, stream=None) -> torch.Tensor:
        return pages_compact(self.keys, self.values, self.table, self.refs, stream=stream)

    def append(self, layer: int, qkv, q_norm, k_norm, rope_cos, rope_sin, eps: float, starts=None, out=None,
               stream=None) -> torch.Tensor:
        """paged_append of one layer."""
        return paged_append(qkv, q_norm, k_norm, rope_cos, rope_sin, eps, self.keys[layer], self.values[layer],
                            self.table, self.lengths, self.status, starts, out, stream)

    def attend(self, layer: int, query, starts=None, window: int = 0, sinks: int = 0, out=None,
               stream=None) -> torch.Tensor:
        """paged_attention over one layer."""
        return paged_attention(query, self.keys[layer], self.values[layer], self.table, self.lengths, starts, window,
                               sinks, out, stream)

    def plan_tree(self, parents, starts, stream=None):
        """tree_plan; lists or device tensors."""
        from .tree import tree_plan
        return tree_plan(self._ints(parents), self._ints(starts), self.status, stream=stream)

    def append_tree(self, layer: int, qkv, q_norm, k_norm, rope_cos, rope_sin, eps: float, tree, out=None,
                    stream=None) -> torch.Tensor:
        """paged_append_tree of one layer."""
        from .tree import paged_append_tree
        return paged_append_tree(qkv, q_norm, k_norm, rope_cos, rope_sin, eps, self.keys[layer], self.values[layer],
                                 self.table, self.lengths, self.status, tree, out, stream)

    def attend_tree(self, layer: int, query, tree, window: int = 0, sinks: int = 0, out=None,
                    stream=None) -> torch.Tensor:
        """paged_attention_tree over one layer."""
        from .tree import paged_attention_tree
        return paged_attention_tree(query, self.keys[layer], self.values[layer], self.table, self.lengths, tree, window,
                                    sinks, out, stream)

    def accept(self, tree, drafted, choices=None, logits=None, levels: int = 256, stream=None):
        """pages_accept over all layers; drafted and choices: lists or device tensors."""
        from .tree import pages_accept
        return pages_accept(self.keys, self.values, self.table, self.lengths, self.status, tree, self._ints(drafted),
                            None if choices is None else self._ints(choices), logits, levels, stream=stream)

    def check_status(self) -> None:
        """Wait for the calls so far, on whatever stream, and raise where one was refused."""
        torch.cuda.synchronize(self.status.device)
        code = int(self.status.item())
        if code & _native.HQ_PAGES_FULL:
            raise ValueError("the cache's free pages, or a sequence's table entries, did not suffice")
        if code & _native.HQ_PAGES_BAD:
            raise ValueError("a table entry, length, start or parent outside its range reached the device")
