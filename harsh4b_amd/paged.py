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

import ctypes
import functools

import torch

from . import _native
from ._native import HqPages, check

PAGE_SIZES = (16, 32, 64, 128, 256)
HEAD_DIMS = (16, 32, 64, 128)
MAX_GROUPS = 8


# --------------------------------------------------------------------------- checks
def _tensor(t, name: str, dtype, dims: int, device=None) -> None:
    if not isinstance(t, torch.Tensor) or t.dtype != dtype or t.dim() != dims or not t.is_cuda or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {str(dtype)[6:]} device tensor of {dims} dimensions")
    if device is not None and t.device != device:
        raise ValueError(f"{name} is on another device")


def _cache(keys, values, table, lengths, refs, status, dims: int, pools: bool = True) -> HqPages:
    """The tables' C struct, checked; keys/values [layers, pages, kv_heads,
    page_size, head_dim] (dims 5) or one layer of them (dims 4)."""
    _tensor(table, "table", torch.int32, 2)
    device = table.device
    layers, kv_heads, page_size, head_dim = 1, 1, PAGE_SIZES[0], HEAD_DIMS[0]
    if pools:
        _tensor(keys, "keys", torch.float16, dims, device)
        _tensor(values, "values", torch.float16, dims, device)
        shape = keys.shape
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
    else:
        pages = refs.shape[0] if isinstance(refs, torch.Tensor) and refs.dim() == 1 else 0
    sequences, max_pages = table.shape
    if sequences == 0 or max_pages == 0 or max_pages * page_size > 0x7FFFFFFF or sequences * max_pages > 0x7FFFFFFF:
        raise ValueError("table must be [sequences, max_pages] with fewer than 2^31 entries and positions a row")
    if lengths is not None:
        _tensor(lengths, "lengths", torch.int32, 1, device)
        if lengths.shape[0] != sequences:
            raise ValueError("lengths must be [sequences]")
    if refs is not None:
        _tensor(refs, "refs", torch.int32, 1, device)
        if refs.shape[0] != pages or pages == 0:
            raise ValueError("refs must be [pages]")
    if status is not None:
        _tensor(status, "status", torch.int32, 1, device)
        if status.shape[0] != 1:
            raise ValueError("status must hold one int32")
    return HqPages(layers, pages, page_size, kv_heads, head_dim, sequences, max_pages, 0,
                   keys.data_ptr() if pools else None, values.data_ptr() if pools else None, table.data_ptr(),
                   None if lengths is None else lengths.data_ptr(), None if refs is None else refs.data_ptr(),
                   None if status is None else status.data_ptr())


def _per_sequence(t, name: str, table) -> None:
    _tensor(t, name, torch.int32, 1, table.device)
    if t.shape[0] != table.shape[0]:
        raise ValueError(f"{name} must be [sequences]")


def _starts(starts, table, tokens: int) -> int | None:
    if starts is None:
        if tokens != table.shape[0]:
            raise ValueError("without starts a batch has one row for every sequence")
        return None
    _tensor(starts, "starts", torch.int32, 1, table.device)
    if starts.shape[0] != table.shape[0] + 1:
        raise ValueError("starts must be [sequences + 1]")
    return starts.data_ptr()


def _launch(call, nbytes: int, device, stream, tensors, what: str) -> None:
    """call(workspace pointer, stream handle) on `stream` (None: the current
    one of `device`) with a workspace of this call alone: memory of any
    contents from torch's allocator, which hands it out in the stream's order
    and inside a capture from the graph's own pool."""
    if device.index != torch.cuda.current_device():
        with torch.cuda.device(device):
            return _launch(call, nbytes, device, stream, tensors, what)
    if stream is None:
        ws = torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None
        check(call(None if ws is None else ws.data_ptr(), torch._C._cuda_getCurrentRawStream(device.index)), what)
        return
    if stream.device != device:
        raise ValueError("the stream belongs to another device than the tensors")
    # the stream waits for what the caller's has enqueued, and the tensors'
    # memory is not reused before the stream is done with them
    stream.wait_stream(torch.cuda.current_stream(device))
    with torch.cuda.stream(stream):
        ws = torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None
    for t in tensors:
        if t is not None:
            t.record_stream(stream)
    check(call(None if ws is None else ws.data_ptr(), stream.cuda_stream), what)


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
    cache = _cache(keys, values, table, lengths, None, status, 4)
    device, d, kv = table.device, cache.head_dim, cache.kv_heads
    if status is None:
        raise ValueError("paged_append needs the cache's status")
    _tensor(qkv, "qkv", torch.float32, 2, device)
    tokens, width = qkv.shape
    heads = width // d - 2 * kv
    if width % d or heads < 1 or heads % kv or heads // kv > MAX_GROUPS:
        raise ValueError("qkv must be [tokens, (heads + 2 kv_heads) * head_dim] with 1 to 8 heads a kv head")
    for t, name in ((q_norm, "q_norm"), (k_norm, "k_norm")):
        _tensor(t, name, torch.float32, 1, device)
        if t.shape[0] != d:
            raise ValueError(f"{name} must be [head_dim]")
    for t, name in ((rope_cos, "rope_cos"), (rope_sin, "rope_sin")):
        _tensor(t, name, torch.float32, 2, device)
    if rope_cos.shape != rope_sin.shape or rope_cos.shape[1] != d // 2 or rope_cos.shape[0] < 1:
        raise ValueError("rope_cos and rope_sin must be [positions, head_dim / 2]")
    first = _starts(starts, table, tokens)
    if out is None:
        out = torch.empty((tokens, heads, d), dtype=torch.float32, device=device)
    else:
        _tensor(out, "out", torch.float32, 3, device)
        if out.shape != (tokens, heads, d):
            raise ValueError("out must be [tokens, heads, head_dim]")
    if tokens == 0:
        return out
    lib = _native.lib()
    _launch(lambda ws, s: lib.hq_paged_append(
        ctypes.byref(cache), qkv.data_ptr(), first, tokens, heads, q_norm.data_ptr(), k_norm.data_ptr(), float(eps),
        rope_cos.data_ptr(), rope_sin.data_ptr(), rope_cos.shape[0], out.data_ptr(), s), 0, device, stream,
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
    cache = _cache(keys, values, table, lengths, None, None, 4)
    device, d, kv = table.device, cache.head_dim, cache.kv_heads
    _tensor(query, "query", torch.float32, 3, device)
    tokens, heads, width = query.shape
    if width != d or heads < 1 or heads % kv or heads // kv > MAX_GROUPS:
        raise ValueError("query must be [tokens, heads, head_dim] with 1 to 8 heads a kv head")
    if not 0 <= window <= 0x7FFFFFFF or not 0 <= sinks <= 0x7FFFFFFF:
        raise ValueError("window and sinks must not be negative")
    first = _starts(starts, table, tokens)
    if out is None:
        out = torch.empty_like(query)
    else:
        _tensor(out, "out", torch.float32, 3, device)
        if out.shape != query.shape:
            raise ValueError("out must be like query")
    if tokens == 0:
        return out
    lib = _native.lib()
    _launch(lambda ws, s: lib.hq_paged_attention(
        ctypes.byref(cache), query.data_ptr(), first, tokens, heads, window, sinks, out.data_ptr(), ws, s),
        _attention_workspace_bytes(tokens, heads, kv, d, starts is None), device, stream,
        (query, keys, values, table, lengths, starts, out), "hq_paged_attention")
    return out


# --------------------------------------------------------------------------- page management
def _pages_workspace(cache: HqPages) -> int:
    return _native.lib().hq_pages_workspace_bytes(ctypes.byref(cache))


def pages_resize(keys: torch.Tensor, values: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor,
                 refs: torch.Tensor, status: torch.Tensor, new_lengths: torch.Tensor, window: int = 0, sinks: int = 0,
                 stream=None) -> None:
    """Set the sequences' lengths (hq_pages_resize): int32 [sequences] on the
    device, a negative one leaves its sequence as it is.  Growth takes the
    lowest free pages, and copies the partly filled page it goes on in where
    others hold it too; shrinking releases pages, and `window` > 0 those that
    no later query sees.  Too few free pages, or a length past the table, set
    HQ_PAGES_FULL in `status` and change nothing."""
    cache = _cache(keys, values, table, lengths, refs, status, 5)
    if lengths is None or refs is None or status is None:
        raise ValueError("pages_resize needs lengths, refs and status")
    _per_sequence(new_lengths, "new_lengths", table)
    if not 0 <= window <= 0x7FFFFFFF or not 0 <= sinks <= 0x7FFFFFFF:
        raise ValueError("window and sinks must not be negative")
    lib = _native.lib()
    _launch(lambda ws, s: lib.hq_pages_resize(ctypes.byref(cache), new_lengths.data_ptr(), window, sinks, ws, s),
            _pages_workspace(cache), table.device, stream,
            (keys, values, table, lengths, refs, status, new_lengths), "hq_pages_resize")


def pages_fork(table: torch.Tensor, lengths: torch.Tensor, refs: torch.Tensor, status: torch.Tensor,
               parents: torch.Tensor, stream=None) -> None:
    """Every sequence b becomes a fork of sequence parents[b] (int32
    [sequences] on the device; negative or b: unchanged) as it was before the
    call, sharing all its pages (hq_pages_fork); what it held is released."""
    if lengths is None or refs is None or status is None:
        raise ValueError("pages_fork needs lengths, refs and status")
    cache = _cache(None, None, table, lengths, refs, status, 5, pools=False)
    _per_sequence(parents, "parents", table)
    lib = _native.lib()
    _launch(lambda ws, s: lib.hq_pages_fork(ctypes.byref(cache), parents.data_ptr(), ws, s), _pages_workspace(cache),
            table.device, stream, (table, lengths, refs, status, parents), "hq_pages_fork")


def pages_compact(keys: torch.Tensor, values: torch.Tensor, table: torch.Tensor, refs: torch.Tensor,
                  live: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """Move the pages in use to the lowest places (hq_pages_compact), tables
    and refs with them; returns their number, int32 [1] on the device."""
    if refs is None:
        raise ValueError("pages_compact needs refs")
    cache = _cache(keys, values, table, None, refs, None, 5)
    if live is None:
        live = torch.empty(1, dtype=torch.int32, device=table.device)
    else:
        _tensor(live, "live", torch.int32, 1, table.device)
        if live.shape[0] != 1:
            raise ValueError("live must hold one int32")
    lib = _native.lib()
    _launch(lambda ws, s: lib.hq_pages_compact(ctypes.byref(cache), live.data_ptr(), ws, s), _pages_workspace(cache),
            table.device, stream, (keys, values, table, refs, live), "hq_pages_compact")
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

    def check_status(self) -> None:
        """Wait for the calls so far and raise where one was refused."""
        code = int(self.status.item())
        if code & _native.HQ_PAGES_FULL:
            raise ValueError("the cache's free pages, or a sequence's table entries, did not suffice")
        if code & _native.HQ_PAGES_BAD:
            raise ValueError("a table entry, length, start or parent outside its range reached the device")
