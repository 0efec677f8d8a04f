"""The paged K/V cache (harsh4b_amd/paged.py, csrc/hq_paged.hip, hq_pages.hip)
against plain implementations: attention and append in float64, the page
management against lists.  No reference counterpart (the reference keeps one
contiguous cache per session, cpu_lightspark.py:275-309)."""
import ctypes
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

gpu = pytest.mark.gpu


def native():
    from harsh4b_amd import _native
    return _native


@pytest.fixture(autouse=True)
def _announce(request):
    if request.node.get_closest_marker("gpu"):
        print(f"\n[gpu] {request.node.nodeid}", flush=True)
        yield
        torch.cuda.synchronize()
    else:
        yield


# ------------------------------------------------------------------ refusals (no launch)
def _struct(**change):
    n = native()
    buf = ctypes.create_string_buffer(4096)
    p = (ctypes.addressof(buf) + 255) & ~255
    f = dict(layers=2, pages=8, page_size=16, kv_heads=2, head_dim=32, sequences=3, max_pages=4, reserved=0, keys=p,
             values=p, table=p, lengths=p, refs=p, status=p)
    f.update(change)
    return n.HqPages(*[f[name] for name, _ in n.HqPages._fields_]), p, buf


BAD_SHAPES = [dict(pages=0), dict(page_size=8), dict(page_size=48), dict(page_size=512), dict(head_dim=24),
              dict(head_dim=256), dict(kv_heads=0), dict(sequences=0), dict(max_pages=0), dict(max_pages=1 << 28), dict(max_pages=(1 << 27) - 15)]


@pytest.mark.parametrize("change", BAD_SHAPES + [dict(keys=None), dict(table=None), dict(lengths=None)])
def test_c_entries_refuse_bad_caches(change):
    lib = native().lib()
    c, p, _ = _struct(**change)
    c = ctypes.byref(c)
    assert lib.hq_paged_attention(c, p, None, 3, 4, 0, 0, p, p, None) == 1
    assert lib.hq_paged_append(c, p, None, 3, 4, p, p, 1e-6, p, p, 10, p, None) == 1
    assert lib.hq_pages_resize(c, p, 0, 0, p, None) == 1
    if "keys" not in change:
        assert lib.hq_pages_fork(c, p, p, None) == 1
    if "lengths" not in change:
        assert lib.hq_pages_compact(c, None, p, None) == 1
    if not {"keys", "table", "lengths"} & set(change):
        assert lib.hq_pages_workspace_bytes(c) == 0


def test_c_entries_refuse_bad_arguments():
    lib = native().lib()
    s, p, _ = _struct()
    c = ctypes.byref(s)
    at = lib.hq_paged_attention
    assert at(c, None, None, 3, 4, 0, 0, p, p, None) == 1 and at(c, p, None, 3, 4, 0, 0, None, p, None) == 1
    assert at(c, p, None, 3, 4, 0, 0, p, None, None) == 1            # workspace
    assert at(c, p, None, 2, 4, 0, 0, p, p, None) == 1               # a row for every sequence
    assert at(c, p, None, 3, 5, 0, 0, p, p, None) == 1               # heads % kv_heads
    assert at(c, p, None, 3, 18, 0, 0, p, p, None) == 1              # 9 heads a kv head
    assert at(c, p, None, 3, 4, -1, 0, p, p, None) == 1 and at(c, p, None, 3, 4, 8, -1, p, p, None) == 1
    assert at(c, p, p, -1, 4, 0, 0, p, p, None) == 1
    assert at(c, p + 4, None, 3, 4, 0, 0, p, p, None) == 2 and at(c, p, None, 3, 4, 0, 0, p + 8, p, None) == 2
    assert at(c, p, None, 3, 4, 0, 0, p, p + 16, None) == 2          # workspace: 256 bytes
    assert at(c, p, p, 0, 4, 0, 0, p, p, None) == 0                  # no rows: nothing to do
    assert at(c, p, p, 2**24, 4, 0, 0, p, p, None) == 1              # more blocks than a launch has
    ap = lib.hq_paged_append
    assert ap(c, p, None, 3, 4, None, p, 1e-6, p, p, 10, p, None) == 1
    assert ap(c, p, None, 3, 4, p, p, 1e-6, p, p, 0, p, None) == 1   # rope positions
    assert ap(c, p, p, 0, 4, p, p, 1e-6, p, p, 10, p, None) == 0
    n, _, _ = _struct(status=None)
    assert ap(ctypes.byref(n), p, None, 3, 4, p, p, 1e-6, p, p, 10, p, None) == 1
    assert lib.hq_pages_resize(ctypes.byref(n), p, 0, 0, p, None) == 1
    assert lib.hq_pages_fork(ctypes.byref(n), p, p, None) == 1
    many, _, _ = _struct(sequences=2**24, max_pages=1)
    assert at(ctypes.byref(many), p, p, 5, 4, 0, 0, p, p, None) == 1
    assert lib.hq_pages_workspace_bytes(ctypes.byref(many)) == 0
    assert lib.hq_pages_fork(ctypes.byref(many), p, p, None) == 1
    for bad in (dict(keys=p + 8), dict(values=p + 2)):
        u, _, _ = _struct(**bad)
        assert at(ctypes.byref(u), p, None, 3, 4, 0, 0, p, p, None) == 2
        assert lib.hq_pages_resize(ctypes.byref(u), p, 0, 0, p, None) == 2
        assert lib.hq_pages_compact(ctypes.byref(u), None, p, None) == 2
    assert lib.hq_pages_resize(c, None, 0, 0, p, None) == 1 and lib.hq_pages_resize(c, p, -1, 0, p, None) == 1
    assert lib.hq_pages_resize(c, p, 0, 0, p + 64, None) == 2 and lib.hq_pages_fork(c, p, p + 4, None) == 2
    assert lib.hq_paged_attention_workspace_bytes(3, 5, 2, 32, 0) == 0
    assert lib.hq_paged_attention_workspace_bytes(3, 4, 2, 32, 1) > 0
    # the plan's lists: two of a page or sequence, three of a page, three ints a copy, the table and the lengths
    assert lib.hq_pages_workspace_bytes(c) >= 4 * (2 * 8 + 3 * 8 + 3 * 3 + 12 + 3)


def test_python_refuses_host_tensors_and_bad_caches():
    from harsh4b_amd import paged
    k = torch.zeros((4, 2, 16, 32), dtype=torch.float16)
    table, lengths = torch.zeros((2, 3), dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="device tensor"):
        paged.paged_attention(torch.zeros(2, 4, 32), k, k, table, lengths)
    with pytest.raises(ValueError, match="device tensor"):
        paged.pages_fork(table, lengths, lengths, lengths, lengths)
    with pytest.raises(ValueError, match="page_size"):
        paged.PagedCache(1, 4, 2, 32, 2, 3, page_size=24, device="cpu")
    with pytest.raises(ValueError, match="head_dim"):
        paged.PagedCache(1, 4, 2, 48, 2, 3, device="cpu")
    with pytest.raises(ValueError, match="positive"):
        paged.PagedCache(1, 0, 2, 32, 2, 3, device="cpu")


def test_sizes_that_the_entries_refuse():
    # the size functions return 0 for them: an error, and no call without the workspace
    from harsh4b_amd import paged
    with pytest.raises(ValueError, match="2\\^24 sequences"):
        paged._cache(-1, None, None, torch.empty((2**24, 1), dtype=torch.int32), None, None, None, 5, pools=False)
    paged._cache(-1, None, None, torch.empty((2**24 - 1, 1), dtype=torch.int32), None, None, None, 5, pools=False)
    calls = []
    with pytest.raises(ValueError, match="hq_some_entry: sizes"):
        paged._launch(lambda *args: calls.append(args) or 0, (1, 2), 0, 0, None, (), "hq_some_entry")
    assert calls == []


@gpu
def test_tables_of_too_many_sequences():
    from harsh4b_amd import paged
    ints = dict(dtype=torch.int32, device="cuda")
    table, each, refs = torch.full((2**24, 1), -1, **ints), torch.zeros(2**24, **ints), torch.zeros(4, **ints)
    status, pool = torch.zeros(1, **ints), torch.zeros((1, 4, 1, 16, 16), dtype=torch.float16, device="cuda")
    for call in (lambda: paged.pages_fork(table, each, refs, status, each),
                 lambda: paged.pages_resize(pool, pool.clone(), table, each, refs, status, each),
                 lambda: paged.pages_compact(pool, pool.clone(), table, refs)):
        with pytest.raises(ValueError, match="fewer than 2\\^24 sequences"):
            call()


@gpu
def test_python_refuses_bad_device_arguments():
    from harsh4b_amd import paged
    c = paged.PagedCache(1, 6, 2, 32, sequences=3, max_pages=2, page_size=16)
    k, v = c.keys[0], c.values[0]
    q = torch.zeros((3, 4, 32), device="cuda")

    def refuse(match, query=q, keys=k, values=v, table=c.table, lengths=c.lengths, **more):
        with pytest.raises(ValueError, match=match):
            paged.paged_attention(query, keys, values, table, lengths, **more)

    refuse("query", query=q.half())
    refuse("query", query=q.transpose(0, 1))
    refuse("query", query=torch.zeros((3, 5, 32), device="cuda"))
    refuse("query", query=torch.zeros((3, 18, 32), device="cuda"))
    refuse("one row", query=q[:2])
    refuse("keys", keys=k.float())
    refuse("same shape", values=v[:5])
    refuse("page_size", keys=k[:, :, :8].contiguous(), values=v[:, :, :8].contiguous())
    refuse("head_dim", keys=k[..., :24].contiguous(), values=v[..., :24].contiguous())
    refuse("table", table=c.table.long())
    refuse("table", table=c.table.t())
    refuse("lengths", lengths=c.lengths[:2])
    refuse("starts", starts=torch.zeros(3, dtype=torch.int32, device="cuda"))
    refuse("out", out=torch.empty((3, 4, 16), device="cuda"))
    refuse("negative", window=-1)
    refuse("negative", window=4, sinks=-1)
    norm, rope = torch.ones(32, device="cuda"), torch.ones((8, 16), device="cuda")
    qkv = torch.zeros((3, 8 * 32), device="cuda")

    def refuse_append(match, qkv=qkv, norm=norm, rope=rope, **more):
        with pytest.raises(ValueError, match=match):
            paged.paged_append(qkv, norm, norm, rope, rope, 1e-6, k, v, c.table, c.lengths, c.status, **more)

    refuse_append("qkv", qkv=torch.zeros((3, 7 * 32), device="cuda"))      # 3 heads of 2 kv heads
    refuse_append("qkv", qkv=torch.zeros((3, 4 * 32), device="cuda"))      # no query head
    refuse_append("qkv", qkv=torch.zeros((3, 8 * 32 + 16), device="cuda"))
    refuse_append("q_norm", norm=norm[:16])
    refuse_append("rope", rope=rope[:, :8].contiguous())
    with pytest.raises(ValueError, match="new_lengths"):
        c.resize([1, 2])
    with pytest.raises(ValueError, match="parents"):
        c.fork(torch.zeros(3, dtype=torch.int64, device="cuda"))
    with pytest.raises(ValueError, match="negative"):
        c.resize([1, 2, 3], window=-2)
    out = paged.paged_attention(q[:0], k, v, c.table, c.lengths,
                                starts=torch.zeros(4, dtype=torch.int32, device="cuda"))
    assert out.shape == (0, 4, 32)


# ------------------------------------------------------------------ attention
def _reference(query, keys, values, table, counts, lengths, window, sinks):
    """The definition in float64, a row at a time; a page outside the pool is
    none.  Returns the output and the bound of each row's error."""
    query, keys, values = (np.asarray(a, dtype=np.float64) for a in (query, keys, values))
    pages, kv, ps, d = keys.shape
    heads = query.shape[1]
    out = np.full(query.shape, np.nan)
    bound = np.zeros(query.shape[0])
    t = 0
    for b, n in enumerate(counts):
        for i in range(n):
            p = lengths[b] - n + i
            j = np.arange(0, min(p + 1, table.shape[1] * ps))
            page = table[b][j // ps]
            keep = (page >= 0) & (page < pages)
            if window:
                keep &= (j > p - window) | (j < sinks)
            j, page = j[keep], page[keep]
            if j.size == 0:
                out[t] = 0.0
                t += 1
                continue
            k, v = keys[page, :, j % ps], values[page, :, j % ps]             # [n, kv, d]
            for h in range(heads):
                kh, vh, q = k[:, h // (heads // kv)], v[:, h // (heads // kv)], query[t, h]
                with np.errstate(all="ignore"):
                    s = kh @ q / math.sqrt(d)
                    e = np.exp(s - s.max())
                    out[t, h] = (e[:, None] * vh).sum(axis=0) / e.sum()
                # a score's rounding: d products and sums of fp32, and 8 more
                # roundings (the query's parts, the scale, the exponent)
                fine = np.where(np.isfinite(kh), np.abs(kh), 0.0)
                size = (fine @ np.abs(q)).max() / math.sqrt(d)
                error = (d + 8) * 2.0 ** -24 * size
                # the weights move by 2 errors at most, the sums over n keys by n roundings
                top = np.where(np.isfinite(vh), np.abs(vh), 0.0).max()
                bound[t] = max(bound[t], top * (2 * error + (j.size + 64) * 2.0 ** -24))
            t += 1
    return out, bound


class Scene:
    """A batch over a pool whose pages are scattered, its unused places full of NaN."""

    def __init__(self, counts, lengths, kv=2, groups=4, d=128, page=16, seed=0, spare=2, layers=None):
        rng = np.random.default_rng(seed)
        self.rng, self.counts, self.lengths = rng, list(counts), list(lengths)
        need = [-(-max(0, n) // page) for n in lengths]
        pages = sum(need) + spare
        order = rng.permutation(pages)
        self.table = np.full((len(need), max(max(need), 1) + 1), -1, dtype=np.int32)
        self.keys = np.full((pages, kv, page, d), np.nan, dtype=np.float16)
        self.values = np.full((pages, kv, page, d), np.nan, dtype=np.float16)
        at = 0
        for r, n in enumerate(need):
            self.table[r, :n] = order[at:at + n]
            at += n
            for j in range(max(0, lengths[r])):
                p = self.table[r, j // page]
                self.keys[p, :, j % page] = rng.standard_normal((kv, d))
                self.values[p, :, j % page] = rng.standard_normal((kv, d))
        self.tokens = sum(self.counts)
        self.starts = np.concatenate([[0], np.cumsum(self.counts)]).astype(np.int32)
        self.query = rng.standard_normal((self.tokens, kv * groups, d)).astype(np.float32)

    def place(self, b, j):
        page = self.keys.shape[2]
        return self.table[b, j // page], slice(None), j % page

    def device(self):
        def up(a):
            return torch.from_numpy(np.ascontiguousarray(a)).cuda()
        self.dev = dict(query=up(self.query), keys=up(self.keys), values=up(self.values), table=up(self.table),
                        lengths=up(np.asarray(self.lengths, dtype=np.int32)))
        return self.dev

    def attend(self, window=0, sinks=0, starts=True, **more):
        from harsh4b_amd.paged import paged_attention
        d = self.device()
        s = torch.from_numpy(self.starts).cuda() if starts else None
        out = paged_attention(**d, starts=s, window=window, sinks=sinks, **more)
        torch.cuda.synchronize()
        return out.cpu().numpy()

    def check(self, window=0, sinks=0, starts=True, **more):
        """With the table as it is, and as a row of a longer cache's: tiles
        are cut in pieces and joined only where a table is long."""
        got = self._check(window, sinks, starts, **more)
        table, page = self.table, self.keys.shape[2]
        wide = -(-1100 // page)
        if table.shape[1] < wide:
            self.table = np.full((table.shape[0], wide), -1, dtype=np.int32)
            self.table[:, :table.shape[1]] = table
            self._check(window, sinks, starts, **more)
            self.table = table
        return got

    def _check(self, window=0, sinks=0, starts=True, **more):
        got = self.attend(window, sinks, starts, **more)
        expect, bound = _reference(self.query, self.keys, self.values, self.table, self.counts, self.lengths, window,
                                   sinks)
        np.testing.assert_array_equal(np.isnan(got), np.isnan(expect))
        with np.errstate(invalid="ignore"):
            off = np.abs(got - expect)
        off[np.isnan(expect) | (got == expect)] = 0.0
        worst = off.reshape(off.shape[0], -1).max(axis=1) if off.size else np.zeros(0)
        assert (worst <= bound).all(), (np.argmax(worst - bound), worst.max(), bound[np.argmax(worst - bound)])
        return got


SHAPES = [(2, 4, 128), (1, 8, 128), (3, 1, 128), (2, 3, 64), (1, 5, 64), (2, 7, 32), (2, 6, 16), (8, 4, 128)]


@gpu
@pytest.mark.parametrize("kv,groups,d", SHAPES)
@pytest.mark.parametrize("page", [16, 64, 256])
def test_single_tokens(kv, groups, d, page):
    s = Scene([1] * 6, [1, 15, 16, 17, 64, 301], kv, groups, d, page, seed=d + groups)
    a = s.check(starts=False)
    b = s.check(starts=True)
    np.testing.assert_allclose(a, b, rtol=0, atol=1e-4)


@gpu
@pytest.mark.parametrize("kv,groups,d", SHAPES)
def test_chunks(kv, groups, d):
    # whole prompts, chunks after a history, single tokens and sequences without new tokens in one batch
    s = Scene([5, 0, 1, 37, 130, 0, 2, 64], [5, 40, 77, 100, 130, 0, 300, 65], kv, groups, d, 32, seed=d)
    s.check()


@gpu
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (7, 0), (16, 4), (64, 70), (33, 17), (1000, 4), (2**31 - 1, 3),
                                          (100, 2**31 - 1)])
def test_window_and_sinks(window, sinks):
    s = Scene([1, 3, 90, 150], [300, 200, 90, 260], page=16, seed=window % 1000)
    s.check(window, sinks)
    Scene([1] * 4, [300, 2, 17, 511], page=64, seed=sinks % 1000).check(window, sinks, starts=False)


@gpu
@pytest.mark.parametrize("count,length", [(1, 1100), (4, 2050), (129, 1111), (257, 700)])
def test_longer(count, length):
    Scene([count, 1], [length, 900], page=64, seed=count).check()


@gpu
@pytest.mark.parametrize("counts,lengths", [([600], [600]), ([300], [1500]), ([352], [1500]), ([1, 900, 1], [700, 1300, 90]),
                                            ([1100], [1100]), ([64, 256, 1, 256], [400, 1000, 800, 256])])
def test_many_tiles(counts, lengths):
    # 16 tokens a tile and 8 kv heads: 152 to 552 tiles, whole and cut, more and fewer than there are places
    Scene(counts, lengths, 8, 8, 16, 64, seed=len(counts) + counts[-1])._check()


def _reference_of_heads(s, window=0, sinks=0):
    """_reference, a sequence's head at a time, where everything visible is finite."""
    kv, d, heads = s.keys.shape[1], s.keys.shape[3], s.query.shape[1]
    out, bound = np.zeros(s.query.shape), np.zeros(s.tokens)
    for b, (n, length) in enumerate(zip(s.counts, s.lengths)):
        if n == 0:
            continue
        j, p = np.arange(length), np.arange(length - n, length)[:, None]
        seen = j <= p
        if window:
            seen &= (j > p - window) | (j < sinks)
        keys, values = (pool[s.place(b, j)[0], :, j % pool.shape[2]].astype(np.float64) for pool in (s.keys, s.values))
        rows = slice(s.starts[b], s.starts[b + 1])
        for h in range(heads):
            k, v, q = keys[:, h // (heads // kv)], values[:, h // (heads // kv)], s.query[rows, h].astype(np.float64)
            score = np.where(seen, q @ k.T / math.sqrt(d), -np.inf)
            e = np.exp(score - score.max(axis=1, keepdims=True))
            out[rows, h] = e @ v / e.sum(axis=1, keepdims=True)
            size = np.where(seen, np.abs(q) @ np.abs(k).T, 0.0).max(axis=1) / math.sqrt(d)
            bound[rows] = np.maximum(bound[rows], np.abs(v).max() * (2 * (d + 8) * 2.0 ** -24 * size +
                                                                     (seen.sum(axis=1) + 64) * 2.0 ** -24))
    return out, bound


def _check_heads(s, window=0, sinks=0):
    got = s.attend(window, sinks)
    expect, bound = _reference_of_heads(s, window, sinks)
    off = np.abs(got - expect).reshape(s.tokens, -1).max(axis=1)
    assert (off <= bound).all(), (np.argmax(off - bound), off.max(), bound[np.argmax(off - bound)])


@gpu
@pytest.mark.parametrize("kv,groups", [(2, 5), (1, 6), (2, 7)])
def test_joins_with_threads_left_over(kv, groups):
    # 5 to 7 heads of 128: one set of the join's threads and some of a second, which have nothing to store
    for starts in False, True:
        Scene([1] * 6, [1, 15, 16, 17, 64, 301], kv, groups, 128, 16, seed=groups).check(starts=starts)
    Scene([5, 0, 1, 37, 130, 0, 2, 64], [5, 40, 77, 100, 130, 0, 300, 65], kv, groups, 128, 32, seed=groups).check()
    Scene([129, 1], [1111, 900], kv, groups, 128, 64, seed=groups).check()


@gpu
def test_more_rows_than_the_join_has_blocks():
    # every tile in two pieces, 4200 tokens of a kv head to join
    _check_heads(Scene([2100], [2100], 2, 7, 128, 64, seed=71))


@gpu
@pytest.mark.parametrize("count", [1, 2, 40])
@pytest.mark.parametrize("window,sinks", [(0, 0), (50, 3)])
def test_border_positions_count(count, window, sinks):
    # the borders of what is seen carry nearly all the weight: one position more or fewer changes the result
    s = Scene([count], [200 + count], page=16, seed=count)
    s.query[:] = 1.0
    last = 200 + count - 1
    for j in {last, last - 1, 200, 199, last - window, last - window + 1, 200 - window + 1, 200 - window, 0, 2, 3, 4}:
        if 0 <= j <= last:
            s.keys[s.place(0, j)] = 1.0 + (j % 7) / 8
    s.check(window, sinks)


@gpu
def test_rows_that_see_nothing_and_rows_of_nobody():
    from harsh4b_amd.paged import paged_attention
    # more new tokens than positions: the first rows lie before the sequence
    s = Scene([6, 1, 3], [4, 0, 20], page=16, seed=3)
    s.lengths = [4, 0, 20]
    got = s.check()
    assert (got[:2] == 0).all() and (got[6] == 0).all()
    # rows past the last start, and a hole where all of a sequence's pages were
    s.table[2] = -1
    d = s.device()
    out = torch.full((s.tokens + 3, 8, 128), 7.0, device="cuda")
    query = torch.cat((d.pop("query"), torch.ones((3, 8, 128), device="cuda")))
    paged_attention(query, **d, starts=torch.from_numpy(s.starts).cuda(), out=out)
    host = out.cpu().numpy()
    assert (host[s.tokens:] == 7.0).all() and (host[7:10] == 0).all()


@gpu
def test_holes_and_bad_entries():
    # released pages (-1) inside a sequence, and entries that name no page: neither is followed
    s = Scene([1, 20, 40], [300, 280, 100], page=16, seed=11)
    s.table[0, 2:9] = -1
    s.table[1, 0] = s.keys.shape[0]
    s.table[1, 3] = 2**31 - 1
    s.table[1, 5] = -(2**31)
    s.table[2, 0:3] = -1
    s.check()
    s.check(window=90, sinks=20)


@gpu
@pytest.mark.parametrize("lengths", [[2**31 - 1, 20], [-5, 20], [-(2**31), 20], [1000, 20]])
def test_lengths_outside_the_table(lengths):
    s = Scene([2, 3], [40, 20], page=16, seed=5)
    s.lengths = lengths
    s.check(window=0)


@gpu
@pytest.mark.parametrize("starts", [[0, 2, 1], [0, 9, 10], [-3, 2, 5], [4, 2, 5], [0, 0, 0]])
def test_starts_out_of_order(starts):
    # rows of a sequence whose range is not one are not touched
    from harsh4b_amd.paged import paged_attention
    s = Scene([2, 3], [40, 20], page=16, seed=6)
    d = s.device()
    out = torch.full((5, 8, 128), 7.0, device="cuda")
    paged_attention(**d, starts=torch.tensor(starts, dtype=torch.int32, device="cuda"), out=out)
    host = out.cpu().numpy()
    for b in range(2):
        a, z = starts[b], starts[b + 1]
        if 0 <= a < z <= 5 and starts == sorted(starts):
            s2 = host[a:z]
            assert np.isfinite(s2).all() and (s2 != 7.0).any()
    if starts == [0, 0, 0]:
        assert (host == 7.0).all()


@gpu
@pytest.mark.parametrize("starts", [[0, 2, 5], [1, 3, 4], [0, 0, 0], [5, 5, 5], [0, 2, 1], [0, 9, 10], [-3, 2, 5], [4, 2, 5],
                                    [0, 5, 6], [0, 2**31 - 1, 2**31 - 1], [-(2**31), 0, 5]])
@pytest.mark.parametrize("spare", [0, 300])
def test_rows_of_starts_outside_the_batch(starts, spare):
    # the rows of ranges in the batch have their values, the others stay; where starts fall all do (spare: sequences
    # without rows behind, for the plan's own launch)
    from harsh4b_amd.paged import paged_attention
    s = Scene([2, 3] + [0] * spare, [40, 20] + [0] * spare, page=16, seed=6)
    d = s.device()
    out = torch.full((5, 8, 128), 7.0, device="cuda")
    at = torch.tensor(starts + [starts[-1]] * spare, dtype=torch.int32, device="cuda")
    paged_attention(**d, starts=at, out=out)
    host = out.cpu().numpy()
    for b, (a, z) in enumerate(zip(starts, starts[1:])):
        if sorted(starts) == starts and 0 <= a < z <= 5:
            expect, bound = _reference(s.query[a:z], s.keys, s.values, s.table[b:b + 1], [z - a], s.lengths[b:b + 1], 0, 0)
            assert (np.abs(host[a:z] - expect).reshape(z - a, -1).max(axis=1) <= bound).all()
            host[a:z] = 7.0
    assert (host == 7.0).all()


@gpu
@pytest.mark.parametrize("kv,groups,counts,lengths,window,sinks", [
    (8, 8, [600], [600], 0, 0),                    # 304 tiles whole, the second half of the places the other way round
    (8, 4, [300], [1500], 0, 0),                   # 80 tiles, cut
    (8, 4, [1, 900, 1], [700, 1300, 90], 0, 0),    # 232 tiles and single tokens, cut
    (4, 4, [1100], [1300], 333, 5),                # a window: tiles of different chunks
    (8, 5, [500, 3], [1800, 40], 0, 0),            # tiles that are not full: 25 tokens of 5 heads
    (8, 8, [1100], [1100], 0, 0),                  # 552 tiles: more than places
])
def test_many_tiles_of_128_dims(kv, groups, counts, lengths, window, sinks):
    _check_heads(Scene(counts, lengths, kv, groups, 128, 64, seed=groups + counts[-1]), window, sinks)


@gpu
@pytest.mark.parametrize("sequences", [255, 256, 300, 1300])
def test_plans_of_many_sequences(sequences):
    # the plan in every wave, and in a launch of its own (more than one round of its block)
    from harsh4b_amd.paged import paged_attention
    rng = np.random.default_rng(sequences)
    counts = rng.integers(0, 4, sequences)
    counts[[0, 7, sequences - 1]] = 30, 0, 9
    lengths = counts + rng.integers(0, 60, sequences)
    lengths[[0, 9, 200, 254]] = 700, 900, 30, 301
    s = Scene(counts.tolist(), lengths.tolist(), 1, 2, 16, seed=sequences)
    s.check()
    s.check(window=40, sinks=5)
    one = Scene([1] * sequences, np.maximum(lengths, 1).tolist(), 2, 2, 16, seed=sequences)
    one.check(starts=False)
    s.starts[100] = s.starts[101] + 1              # starts that fall: no row is touched
    out = torch.full((s.tokens, 2, 16), 7.0, device="cuda")
    paged_attention(**s.device(), starts=torch.from_numpy(s.starts).cuda(), out=out)
    assert (out == 7.0).all()


@gpu
@pytest.mark.parametrize("sequences", [64, 65, 128, 129, 4096, 4097])
def test_rows_find_their_sequence(sequences):
    # one row each, at the borders of the search; every third sequence without a row
    from harsh4b_amd.paged import paged_attention
    counts = np.array([0 if b % 3 == 1 else 1 for b in range(sequences)])
    s = Scene(counts.tolist(), [3] * sequences, 1, 1, 16, seed=sequences)
    s.values[:] = 0.0
    for b in range(sequences):
        for j in range(3):
            s.values[s.place(b, j)] = b % 2048
    starts = torch.from_numpy(s.starts).cuda()
    out = paged_attention(**s.device(), starts=starts).cpu().numpy()
    np.testing.assert_allclose(out[:, 0, 0], np.flatnonzero(counts) % 2048, rtol=1e-5)
    dev = s.dev
    qkv = torch.zeros((s.tokens, 3 * 16), device="cuda")
    qkv[:, 32:] = torch.arange(s.tokens, device="cuda")[:, None] % 2048
    norm, rope = torch.ones(16, device="cuda"), torch.ones((3, 8), device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    from harsh4b_amd.paged import paged_append
    paged_append(qkv, norm, norm, rope, rope, 1e-6, dev["keys"], dev["values"], dev["table"], dev["lengths"], status,
                 starts=starts)
    assert int(status.item()) == 0
    rows = dev["values"].cpu().numpy()[s.table[np.flatnonzero(counts), 0], 0, 2, 0]
    np.testing.assert_array_equal(rows, np.arange(s.tokens) % 2048)


@gpu
@pytest.mark.parametrize("what", ["nan", "inf", "-inf"])
@pytest.mark.parametrize("count,window", [(1, 0), (1, 30), (3, 30), (60, 0), (60, 30)])
def test_masked_places_of_any_value(what, count, window):
    # positions that a row does not see may hold anything; the rows that see them take it
    s = Scene([count, 5], [150, 60], page=16, seed=count + window)
    x = float(what)
    for j in {149, 148, 120, 100, 40}:
        s.values[s.place(0, j)][0, 3::17] = x
    for j in {147, 110, 60}:
        s.keys[s.place(0, j)][1, 5] = x
    s.check(window)


@gpu
def test_infinite_scores():
    # a key that scores -inf has no weight; a row whose keys all do has no softmax (NaN), as 0/0
    s = Scene([1, 2, 30], [70, 3, 90], page=16, seed=8)
    s.query[:, :, 0] = 1.0
    s.keys[s.place(0, 11)][:, 0] = -np.inf
    s.keys[s.place(2, 65)][:, 0] = -np.inf
    for j in range(3):
        s.keys[s.place(1, j)][:, 0] = -np.inf
    s.check()


@gpu
@pytest.mark.parametrize("scale", [1e-30, 1e-3, 300.0, 1e6, 1e36])
def test_queries_of_any_size(scale):
    s = Scene([1, 40], [100, 90], page=16, seed=9)
    s.query *= np.float32(scale)
    s.check()


@gpu
def test_large_and_small_values():
    s = Scene([1, 40], [100, 90], page=16, seed=10)
    s.values[:] = np.where(np.isnan(s.values), s.values, s.values * np.float16(12000))
    s.keys[:, :, ::2] *= np.float16(2.0 ** -14)           # subnormal keys
    s.check()


@gpu
def test_other_streams():
    # a stream of the caller's, and two calls side by side on two streams: each has its own workspace
    from harsh4b_amd.paged import paged_attention
    scenes = [Scene([1, 40], [100, 1090], page=16, seed=12), Scene([33, 2], [2000, 700], page=16, seed=13)]
    expect = [s.check() for s in scenes]
    np.testing.assert_array_equal(scenes[0].attend(stream=torch.cuda.Stream()), expect[0])
    streams = [torch.cuda.Stream() for _ in scenes]
    inputs = [(s.device(), torch.from_numpy(s.starts).cuda()) for s in scenes]
    for _ in range(20):
        outs = [paged_attention(**d, starts=a, stream=x) for (d, a), x in zip(inputs, streams)]
    torch.cuda.synchronize()
    for out, e in zip(outs, expect):
        np.testing.assert_array_equal(out.cpu().numpy(), e)


@gpu
def test_outputs_over_inputs_are_refused():
    from harsh4b_amd import paged
    c = paged.PagedCache(1, 6, 2, 32, sequences=2, max_pages=2, page_size=16)
    q = torch.zeros((5, 4, 32), device="cuda")
    for out in (q[:2], q[1:3]):
        with pytest.raises(ValueError, match="overlap"):
            paged.paged_attention(q[:2], c.keys[0], c.values[0], c.table, c.lengths, out=out)
    flat = torch.zeros(2 * 8 * 32 + 64, device="cuda")
    rope = torch.ones((8, 16), device="cuda")
    with pytest.raises(ValueError, match="overlap"):
        paged.paged_append(flat[:512].view(2, 256), torch.ones(32, device="cuda"), torch.ones(32, device="cuda"), rope,
                           rope, 1e-6, c.keys[0], c.values[0], c.table, c.lengths, c.status,
                           out=flat[320:576].view(2, 4, 32))


@gpu
@pytest.mark.parametrize("what", ["nan", "inf", "-inf"])
def test_queries_that_are_not_finite(what):
    # a row's value makes its own result NaN and no other
    s = Scene([1, 3, 60], [90, 150, 100], page=16, seed=41)
    for t, h, i in ((0, 1, 7), (2, 5, 127), (30, 0, 0), (63, 7, 64)):
        s.query[t, h, i] = float(what)
    got = s.check()
    assert np.isnan(got).any(axis=-1).sum() == 4


@gpu
def test_many_sequences():
    rng = np.random.default_rng(4)
    lengths = rng.integers(0, 60, 300).tolist()
    counts = [min(n, int(c)) for n, c in zip(lengths, rng.integers(0, 4, 300))]
    Scene(counts, lengths, 1, 2, 32, 16, seed=13).check()
    Scene([1] * 300, [max(1, n) for n in lengths], 1, 4, 64, 16, seed=14).check(starts=False)


@gpu
def test_offsets_past_32_bits():
    # a pool of more than 2^32 bytes and 2^31 elements: the pages in use lie at its end
    from harsh4b_amd.paged import paged_attention
    s = Scene([1, 20], [50, 40], kv=8, groups=1, d=128, page=256, seed=15, spare=0)
    pages = (1 << 31) // (8 * 256 * 128) + 8
    keys = torch.zeros((pages, 8, 256, 128), dtype=torch.float16, device="cuda")
    values = torch.zeros_like(keys)
    n = s.keys.shape[0]
    keys[-n:] = torch.from_numpy(s.keys).cuda()
    values[-n:] = torch.from_numpy(s.values).cuda()
    d = s.device()
    table = torch.where(d["table"] >= 0, d["table"] + (pages - n), d["table"])
    got = paged_attention(d["query"], keys, values, table, d["lengths"], starts=torch.from_numpy(s.starts).cuda())
    np.testing.assert_array_equal(got.cpu().numpy(), s.check())


# ------------------------------------------------------------------ append
def _append_reference(qkv, qn, kn, cos, sin, eps, heads, kv, d, positions):
    x = qkv.astype(np.float64).reshape(len(positions), heads + 2 * kv, d)

    def turned(a, w):
        a = a / np.sqrt((a * a).mean(axis=-1, keepdims=True) + eps) * w
        c, s = cos[positions][:, None].astype(np.float64), sin[positions][:, None].astype(np.float64)
        lo, hi = a[..., :d // 2], a[..., d // 2:]
        return np.concatenate((lo * c - hi * s, hi * c + lo * s), axis=-1)

    return turned(x[:, :heads], qn), turned(x[:, heads:heads + kv], kn), x[:, heads + kv:]


def _append_inputs(s, kv, groups, d, positions=600):
    rng = s.rng
    qkv = (2 * rng.standard_normal((s.tokens, (kv * groups + 2 * kv) * d))).astype(np.float32)
    qn, kn = (rng.uniform(0.9, 1.1, d).astype(np.float32) for _ in range(2))
    angle = np.arange(positions)[:, None] * 10000.0 ** (-np.arange(0, d, 2) / d)
    return qkv, qn, kn, np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)


@gpu
@pytest.mark.parametrize("kv,groups,d", SHAPES)
@pytest.mark.parametrize("starts", [False, True])
def test_append(kv, groups, d, starts):
    from harsh4b_amd.paged import paged_append
    counts = [5, 0, 1, 33] if starts else [1] * 4
    s = Scene(counts, [5, 3, 260, 49], kv, groups, d, 16, seed=d)
    inputs = _append_inputs(s, kv, groups, d)
    dev = s.device()
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    q = paged_append(*[torch.from_numpy(a).cuda() for a in inputs], 1e-6, dev["keys"], dev["values"], dev["table"],
                     dev["lengths"], status, starts=torch.from_numpy(s.starts).cuda() if starts else None)
    assert int(status.item()) == 0
    rows = [(b, s.lengths[b] - n + i) for b, n in enumerate(counts) for i in range(n)]
    positions = np.array([p for _, p in rows])
    eq, ek, ev = _append_reference(*inputs, 1e-6, kv * groups, kv, d, positions)
    # the mean of d squares, a root, two divisions and products, two products and a sum: d/64 + 14 roundings of
    # the norm's size at most, of sums of two terms no larger than sqrt(2) times the largest value
    tol = (d + 14) * 2.0 ** -24 * np.abs(eq).max(axis=-1, keepdims=True) * 2
    assert (np.abs(q.cpu().numpy() - eq) <= tol).all()
    keys, values = dev["keys"].cpu().numpy(), dev["values"].cpu().numpy()
    expect_k, expect_v = s.keys.copy(), s.values.copy()
    for (b, p), k, v in zip(rows, ek, ev):
        at = s.place(b, p)
        tol = (d + 14) * 2.0 ** -24 * np.abs(k).max() * 2 + np.abs(k) * 2.0 ** -11 + 2.0 ** -25
        assert (np.abs(keys[at] - k) <= tol).all()
        np.testing.assert_array_equal(values[at], v.astype(np.float32).astype(np.float16))
        expect_k[at], expect_v[at] = keys[at], values[at]
    # nothing else was written
    np.testing.assert_array_equal(keys.view(np.uint16), expect_k.view(np.uint16))
    np.testing.assert_array_equal(values.view(np.uint16), expect_v.view(np.uint16))


@gpu
def test_append_of_rows_without_a_place():
    from harsh4b_amd.paged import paged_append
    s = Scene([3, 2, 4, 1], [2, 40, 50, 20], page=16, seed=2)     # row 0 lies before its sequence
    s.table[1, 2] = -1                                            # positions 38, 39 have no page
    inputs = _append_inputs(s, 2, 4, 128, positions=48)           # 48, 49 are past the rope tables
    dev = s.device()
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    extra = torch.cat((torch.from_numpy(inputs[0]).cuda(), torch.ones((2, 12 * 128), device="cuda")))
    out = torch.full((12, 8, 128), 7.0, device="cuda")
    paged_append(extra, *[torch.from_numpy(a).cuda() for a in inputs[1:]], 1e-6, dev["keys"], dev["values"],
                 dev["table"], dev["lengths"], status, starts=torch.from_numpy(s.starts).cuda(), out=out)
    host = out.cpu().numpy()
    assert int(status.item()) == native().HQ_PAGES_BAD
    zero = [0, 3, 4, 7, 8]
    assert (host[zero] == 0).all() and (host[10:] == 7.0).all()
    assert all((host[i] != 0).any() for i in range(10) if i not in zero)
    before, after = s.values.view(np.uint16), dev["values"].cpu().numpy().view(np.uint16)
    changed = {(int(p), int(j)) for p, _, j, _ in np.argwhere(before != after)}
    assert changed == {(int(s.table[b, j // 16]), j % 16) for b, j in [(0, 0), (0, 1), (2, 46), (2, 47), (3, 19)]}
    # a cache that could not grow takes no rows
    for code in native().HQ_PAGES_FULL, native().HQ_PAGES_REFUSED:
        status.fill_(code)
        dev = s.device()
        paged_append(torch.from_numpy(inputs[0]).cuda(), *[torch.from_numpy(a).cuda() for a in inputs[1:]], 1e-6,
                     dev["keys"], dev["values"], dev["table"], dev["lengths"], status,
                     starts=torch.from_numpy(s.starts).cuda())
        np.testing.assert_array_equal(dev["values"].cpu().numpy().view(np.uint16), before)


@gpu
@pytest.mark.parametrize("starts", [[0, 2, 5], [1, 3, 4], [0, 0, 0], [5, 5, 5], [0, 2, 1], [0, 9, 10], [-3, 2, 5], [4, 2, 5],
                                    [0, 5, 6], [0, 0, 6], [2, 2, 1], [0, 2**31 - 1, 2**31 - 1], [-(2**31), 0, 5]])
def test_append_reports_starts_outside_the_batch(starts):
    # a range that is none loses its sequence's rows: reported, and nothing else is written in their place
    from harsh4b_amd.paged import paged_append
    s = Scene([2, 3], [40, 20], page=16, seed=6)
    inputs, dev = _append_inputs(s, 2, 4, 128), s.device()
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = torch.full((5, 8, 128), 7.0, device="cuda")
    paged_append(*[torch.from_numpy(a).cuda() for a in inputs], 1e-6, dev["keys"], dev["values"], dev["table"],
                 dev["lengths"], status, starts=torch.tensor(starts, dtype=torch.int32, device="cuda"), out=out)
    good = [0 <= a <= z <= 5 for a, z in zip(starts, starts[1:])]
    assert int(status.item()) == (0 if all(good) else native().HQ_PAGES_BAD)
    rows, host = set(), out.cpu().numpy()
    values, written = s.values.copy(), dev["values"].cpu().numpy()
    for b, (a, z) in enumerate(zip(starts, starts[1:])):
        if good[b] and sorted(starts) == starts:
            rows |= set(range(a, z))
            for t in range(a, z):
                values[s.place(b, s.lengths[b] - (z - a) + t - a)] = inputs[0][t, 10 * 128:].reshape(2, 128)
    if sorted(starts) == starts:
        np.testing.assert_array_equal(written.view(np.uint16), values.view(np.uint16))
        assert all((host[t] != 7.0).any() == (t in rows) for t in range(5))


@gpu
def test_append_looks_at_all_starts():
    # more sequences than the launch has threads, the bad one among the last
    from harsh4b_amd.paged import paged_append
    n, d = 2000, 16
    ints = dict(dtype=torch.int32, device="cuda")
    starts = torch.ones(n + 1, **ints)
    starts[0] = 0
    pool, rope, norm = (torch.zeros((4, 1, 16, d), dtype=torch.float16, device="cuda"), torch.ones((16, d // 2), device="cuda"),
                        torch.ones(d, device="cuda"))
    table, lengths = torch.zeros((n, 1), **ints), torch.ones(n, **ints)
    for bad in None, n - 1, n, 1500, 1:
        status, at = torch.zeros(1, **ints), starts.clone()
        if bad is not None:
            at[bad:] = 2 if bad != 1500 else -1
        paged_append(torch.ones((1, 3 * d), device="cuda"), norm, norm, rope, rope, 1e-6, pool, pool.clone(), table, lengths,
                     status, starts=at)
        assert int(status.item()) == (0 if bad is None else native().HQ_PAGES_BAD), bad


@gpu
def test_append_of_the_most_tokens():
    # as many as a launch has blocks: those that look at the starts have a launch of their own
    from harsh4b_amd.paged import paged_append
    tokens, d = 2**24 - 1, 16
    pages = 2**24 // 256
    ints = dict(dtype=torch.int32, device="cuda")
    keys = torch.zeros((pages, 1, 256, d), dtype=torch.float16, device="cuda")
    values, rope, norm = torch.zeros_like(keys), torch.ones((tokens, d // 2), device="cuda"), torch.ones(d, device="cuda")
    qkv = torch.zeros((tokens, 3 * d), device="cuda")
    qkv[:, 2 * d:] = (torch.arange(tokens, device="cuda") % 2039)[:, None]
    table, lengths = torch.arange(pages, **ints)[None], torch.full((1,), tokens, **ints)
    for end in tokens, 2**24:
        status = torch.zeros(1, **ints)
        values.zero_()
        paged_append(qkv, norm, norm, rope, rope, 1e-6, keys, values, table, lengths, status,
                     starts=torch.tensor([0, end], **ints))
        good = end == tokens
        assert int(status.item()) == (0 if good else native().HQ_PAGES_BAD)
        expect = torch.arange(2**24, device="cuda").remainder_(2039).mul_(good).half()
        expect[-1] = 0.0
        assert torch.equal(values[:, 0].reshape(-1, d), expect[:, None].expand(-1, d))


# ------------------------------------------------------------------ page management
class Book:
    """The tables as lists, and what the calls do to them."""

    def __init__(self, sequences, max_pages, pages, page):
        self.table = [[-1] * max_pages for _ in range(sequences)]
        self.lengths, self.refs = [0] * sequences, [0] * pages
        self.page, self.copies, self.status = page, [], 0

    def resize(self, want, window=0, sinks=0):
        ps, self.copies = self.page, []
        new = [old if w < 0 else w for old, w in zip(self.lengths, want)]
        growing = [r for r, n in enumerate(new) if n > self.lengths[r]]
        writes = {r: self.table[r][self.lengths[r] // ps] for r in growing if self.lengths[r] % ps}
        refused = 0
        for r, n in enumerate(new):
            if writes.get(r, 0) < 0:              # growth from the middle of a page that is not there
                refused |= 6
            elif -(-n // ps) > len(self.table[0]):
                refused |= 1
        if refused:
            self.status |= refused
            return False
        copied = []
        for r, p in writes.items():
            same = [x for x in writes if writes[x] == p]
            if p >= 0 and self.refs[p] > 1 and not (min(same) == r and len(same) == self.refs[p]):
                copied.append(r)
        free = [p for p, n in enumerate(self.refs) if n == 0]
        taken = []
        for r, n in enumerate(new):
            old = self.lengths[r]
            for e in range(len(self.table[0])):
                if r in copied and e == old // ps or -(-old // ps) <= e < -(-n // ps):
                    taken.append((r, e))
        if len(taken) > len(free):
            self.status |= 1
            return False
        rows = [list(x) for x in self.table]
        for (r, e), p in zip(taken, free):
            rows[r][e] = p
            if r in copied and e == self.lengths[r] // ps:
                self.copies.append((writes[r], p, self.lengths[r] % ps))
        for r, n in enumerate(new):
            low = min(self.lengths[r], n) - window + 1 if window else 0
            for e in range(len(rows[r])):
                if e >= -(-n // ps) or ((e + 1) * ps <= low and e * ps >= sinks and (r, e) not in taken):
                    rows[r][e] = -1
        self.table, self.lengths = rows, new
        self._count()
        return True

    def fork(self, parents):
        rows = [(list(self.table[p]), self.lengths[p]) if p >= 0 else (self.table[r], self.lengths[r])
                for r, p in enumerate(parents)]
        self.table, self.lengths = [t for t, _ in rows], [n for _, n in rows]
        self._count()

    def compact(self):
        live = sum(n > 0 for n in self.refs)
        source = [p for p, n in enumerate(self.refs) if n and p >= live]
        target = [p for p, n in enumerate(self.refs) if not n and p < live]
        to = dict(zip(source, target))
        self.copies = [(a, b, self.page) for a, b in to.items()]
        self.table = [[to.get(p, p) for p in row] for row in self.table]
        self._count()
        return live

    def _count(self):
        self.refs = [0] * len(self.refs)
        for row in self.table:
            for p in row:
                if p >= 0:
                    self.refs[p] += 1


def _agree(cache, book, pools):
    np.testing.assert_array_equal(cache.table.cpu().numpy(), book.table)
    np.testing.assert_array_equal(cache.lengths.cpu().numpy(), book.lengths)
    np.testing.assert_array_equal(cache.refs.cpu().numpy(), book.refs)
    assert int(cache.status.item()) == book.status
    for pool, have in zip(pools, (cache.keys, cache.values)):
        for a, b, n in book.copies:
            pool[:, b, :, :n] = pool[:, a, :, :n]
        np.testing.assert_array_equal(have.cpu().numpy().view(np.uint16), pool.view(np.uint16))
    book.copies = []


def _cache_and_book(sequences, max_pages, pages, page, layers=3, kv=2, d=32, seed=0):
    from harsh4b_amd.paged import PagedCache
    rng = np.random.default_rng(seed)
    cache = PagedCache(layers, pages, kv, d, sequences, max_pages, page_size=page)
    pools = [rng.standard_normal(cache.keys.shape).astype(np.float16) for _ in range(2)]
    cache.keys.copy_(torch.from_numpy(pools[0]))
    cache.values.copy_(torch.from_numpy(pools[1]))
    return cache, Book(sequences, max_pages, pages, page), pools, rng


@gpu
@pytest.mark.parametrize("sequences,max_pages,pages,page,d", [(1, 1, 1, 16, 16), (5, 7, 20, 16, 32), (9, 12, 60, 32, 64),
                                                              (40, 5, 120, 64, 128), (3, 40, 70, 256, 16)])
def test_page_management_at_random(sequences, max_pages, pages, page, d):
    cache, book, pools, rng = _cache_and_book(sequences, max_pages, pages, page, d=d, seed=pages)
    for step in range(40):
        what = rng.integers(0, 10)
        if what < 6:
            kind = rng.integers(0, 4)
            grow = rng.integers(0, 5 if kind else 2 * page, sequences)
            new = [int(n + g) for n, g in zip(book.lengths, grow)]
            if kind == 1:
                new = [int(rng.integers(0, n + 1)) if rng.random() < 0.5 else n for n in new]
            if kind == 2:
                new = [-1 if rng.random() < 0.5 else n for n in new]
            window, sinks = (int(rng.integers(1, 3 * page)), int(rng.integers(0, 2 * page))) if kind == 3 else (0, 0)
            book.resize(new, window, sinks)
            cache.resize(new, window, sinks)
        elif what < 9:
            parents = rng.integers(-1, sequences, sequences).tolist()
            book.fork(parents)
            cache.fork(parents)
        else:
            live = book.compact()
            assert int(cache.compact().item()) == live
        _agree(cache, book, pools)
        if book.status:                       # refused calls left everything; go on
            book.status = 0
            cache.status.zero_()


@gpu
def test_growth_of_forks_copies_the_shared_page_once_less():
    cache, book, pools, _ = _cache_and_book(4, 4, 16, 16)
    for call in ("resize", [21, 0, 0, 0]), ("fork", [0, 0, 0, -1]), ("resize", [22, 23, 30, -1]):
        getattr(book, call[0])(call[1])
        getattr(cache, call[0])(call[1])
        _agree(cache, book, pools)
    # the first of the three keeps the page that they shared, and all share the full one
    assert book.table[0][:2] == [0, 1] and book.refs[:4] == [3, 1, 1, 1]


@gpu
def test_a_full_pool_changes_nothing():
    cache, book, pools, _ = _cache_and_book(3, 4, 5, 16)
    for want in [33, 17, 0], [33, 17, 1], [48, 32, -1], [49, 17, 0], [33, 17, 65], [33, 17, 2**31 - 1]:
        book.resize(want)
        cache.resize(want)
        _agree(cache, book, pools)
        if book.status:
            with pytest.raises(ValueError, match="free pages"):
                cache.check_status()
            book.status = 0
            cache.status.zero_()
    # forks need no page until they grow: two forks of a partly filled page, one free page short
    for call in ("resize", [17, 0, 0]), ("fork", [0, 0, 0]), ("resize", [18, 18, 18]), ("resize", [64, 18, 18]):
        getattr(book, call[0])(call[1])
        getattr(cache, call[0])(call[1])
        _agree(cache, book, pools)
    assert book.status == 1


@gpu
def test_bad_books_are_refused():
    cache, book, pools, _ = _cache_and_book(3, 4, 9, 16)
    book.resize([20, 40, 5])
    cache.resize([20, 40, 5])
    refused = native().HQ_PAGES_BAD | native().HQ_PAGES_REFUSED
    book.status = refused
    cache.fork([0, 3, 1])                          # no sequence 3: nothing changes
    _agree(cache, book, pools)
    with pytest.raises(ValueError, match="outside its range"):
        cache.check_status()
    good = cache.lengths.clone()
    for bad in (-1, 65, 2**31 - 1, -(2**31)):
        cache.lengths[1] = bad
        cache.status.zero_()
        cache.resize([21, -1, 6])
        assert int(cache.status.item()) == refused
        cache.lengths.copy_(good)
        _agree(cache, book, pools)
    # nothing grows from the middle of a page that is not there
    for bad in (100, 9, -1, -7):
        cache.table[0, 1] = bad
        cache.status.zero_()
        cache.resize([21, 41, -1])
        assert int(cache.status.item()) == refused
        cache.table[0, 1] = book.table[0][1]
        _agree(cache, book, pools)


@gpu
def test_a_window_s_sequence_cut_back_too_far_does_not_grow():
    cache, book, pools, _ = _cache_and_book(2, 20, 24, 16)
    calls = [([200, 30], 0), ([210, 31], 50), ([206, 31], 50), ([208, 31], 0), ([70, 31], 0)]
    for want, window in calls:                     # (position 70 is in a page that went with the window)
        book.resize(want, window)
        cache.resize(want, window)
        _agree(cache, book, pools)
    assert book.table[0][4] == -1 and book.status == 0
    book.resize([71, 32])
    cache.resize([71, 32])
    assert book.status == native().HQ_PAGES_BAD | native().HQ_PAGES_REFUSED
    _agree(cache, book, pools)
    with pytest.raises(ValueError, match="outside its range"):
        cache.check_status()
    cache.status.zero_()
    book.status = 0
    for want in [64, -1], [71, 32]:                # from a page's start it does
        book.resize(want)
        cache.resize(want)
        _agree(cache, book, pools)
    assert book.status == 0


@gpu
def test_status_of_calls_on_another_stream():
    from harsh4b_amd.paged import PagedCache
    cache = PagedCache(1, 4, 1, 16, sequences=2, max_pages=8, page_size=16)
    want = torch.tensor([200, 0], dtype=torch.int32, device="cuda")
    busy, stream = torch.zeros((8192, 8192), dtype=torch.float16, device="cuda"), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):                # the refused call waits behind some 100 ms of other work
        for _ in range(100):
            busy = busy @ busy
    cache.resize(want, stream=stream)
    with pytest.raises(ValueError, match="free pages"):
        cache.check_status()


@gpu
def test_large_pools():
    # more pages than one round of the free-page search looks at, the free ones at its end
    cache, book, pools, _ = _cache_and_book(4, 9000, 36000, 16, layers=1, kv=1, d=16)
    for want in [16 * 8999, 16 * 8000 + 5, 16 * 8990, 3], [-1, 16 * 8100, 0, 16 * 8000], [7, -1, 16 * 8000, -1]:
        book.resize(want)
        cache.resize(want)
        _agree(cache, book, pools)
    cache.fork([1, -1, 3, -1])
    book.fork([1, -1, 3, -1])
    assert int(cache.compact().item()) == book.compact()
    _agree(cache, book, pools)


@gpu
def test_many_rows_at_once():
    # more sequences than the planning block has threads
    cache, book, pools, rng = _cache_and_book(2500, 3, 9000, 16, layers=1, kv=1, d=16, seed=3)
    new = rng.integers(0, 30, 2500).tolist()
    parents = rng.integers(-1, 2500, 2500).tolist()
    for call in ("resize", new), ("fork", parents), ("resize", None):
        args = [n + 3 for n in book.lengths] if call[1] is None else call[1]
        getattr(book, call[0])(args)
        getattr(cache, call[0])(args)
        _agree(cache, book, pools)
    assert book.status == 0


# ------------------------------------------------------------------ together
@gpu
@pytest.mark.parametrize("window,sinks", [(0, 0), (40, 5)])
def test_a_server_s_life(window, sinks):
    """Prompts in chunks, forks, single tokens, an end, compaction: every
    step's attention against float64 over lists of the same rows."""
    from harsh4b_amd.paged import PagedCache
    layers, kv, groups, d, page = 2, 2, 4, 128, 16
    rng = np.random.default_rng(21)
    cache = PagedCache(layers, 60, kv, d, sequences=6, max_pages=16, page_size=page)
    cache.keys.fill_(float("nan"))
    cache.values.fill_(float("nan"))
    angle = np.arange(300)[:, None] * 10000.0 ** (-np.arange(0, d, 2) / d)
    cos, sin = np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)
    norm = np.ones(d, dtype=np.float32)
    dc, ds, dn = (torch.from_numpy(a).cuda() for a in (cos, sin, norm))
    history = [[] for _ in range(6)]          # per sequence the raw rows of every position, [layers][...]

    def step(counts):
        lengths = [len(h) for h in history]
        new = [n + c for n, c in zip(lengths, counts)]
        cache.resize(new, window, sinks)
        tokens = sum(counts)
        starts = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        raw = (2 * rng.standard_normal((layers, tokens, (groups + 2) * kv * d))).astype(np.float32)
        for b, c in enumerate(counts):
            for i in range(c):
                history[b].append(raw[:, starts[b] + i])
        for layer in range(layers):
            q = cache.append(layer, torch.from_numpy(raw[layer]).cuda(), dn, dn, dc, ds, 1e-6,
                             starts=torch.from_numpy(starts).cuda())
            got = cache.attend(layer, q, torch.from_numpy(starts).cuda(), window, sinks).cpu().numpy()
            q = q.cpu().numpy()
            for b, c in enumerate(counts):
                if c == 0:
                    continue
                rows = np.stack([r[layer] for r in history[b]])
                at = np.arange(len(rows))
                _, k, v = _append_reference(rows, norm, norm, cos, sin, 1e-6, kv * groups, kv, d, at)
                # the rows as the table finds them, against float64; then what attends to them
                entries = cache.table[b, :-(-len(rows) // page)].cpu().numpy()
                held = np.repeat(entries >= 0, page)[:len(rows)]
                pools = [x[layer].cpu().numpy()[entries] for x in (cache.keys, cache.values)]
                for x, y in zip(pools, (k, v)):
                    x = x.transpose(0, 2, 1, 3).reshape(-1, kv, d)[:len(rows)][held].astype(np.float64)
                    y = y[held]
                    # the append's bound, then fp16's half step
                    tol = (d + 14) * 2.0 ** -23 * np.abs(y).max() + np.abs(y) * 2.0 ** -11 + 2.0 ** -25
                    assert (np.abs(x - y) <= tol).all()
                expect, bound = _reference(q[starts[b]:starts[b] + c], *pools,
                                           np.where(entries >= 0, np.arange(len(entries)), -1)[None], [c], [len(rows)],
                                           window, sinks)
                off = np.abs(got[starts[b]:starts[b] + c] - expect).reshape(c, -1).max(axis=1)
                assert (off <= bound).all(), (layer, b, off.max(), bound.max())
                # every page that is seen is held
                p = len(rows) - c
                need = (at > p - window) | (at < sinks) if window else at >= 0
                assert held[need].all()
        cache.check_status()

    step([33, 0, 70, 1, 0, 0])
    step([20, 0, 1, 1, 0, 5])
    cache.fork([-1, 0, -1, -1, 2, -1])
    history[1], history[4] = list(history[0]), list(history[2])
    step([1, 1, 1, 1, 1, 1])
    step([1, 3, 1, 0, 40, 1])
    cache.resize([0, -1, -1, -1, -1, 0])
    history[0], history[5] = [], []
    live = int(cache.compact().item())
    assert live == int((cache.refs > 0).sum().item()) and (cache.refs[live:] == 0).all()
    step([9, 1, 1, 1, 1, 0])
    cache.fork([1, 2, -1, -1, -1, -1])        # two change places in a chain: both as they were before
    history[0], history[1] = list(history[1]), list(history[2])
    step([1, 1, 1, 1, 1, 17])


@gpu
def test_captured_steps():
    """Growth across page borders, append and attention as a graph, replayed
    with eager work between; a second graph of the same cache beside it."""
    from harsh4b_amd.paged import PagedCache, paged_attention
    kv, groups, d, page = 2, 4, 128, 16
    rng = np.random.default_rng(31)

    def fresh():
        c = PagedCache(1, 40, kv, d, sequences=3, max_pages=8, page_size=page)
        c.resize([14, 30, 1])
        c.keys.copy_(torch.from_numpy(np.random.default_rng(1).standard_normal(c.keys.shape).astype(np.float16)))
        c.values.copy_(torch.from_numpy(np.random.default_rng(2).standard_normal(c.values.shape).astype(np.float16)))
        return c

    cos = torch.rand((200, d // 2), device="cuda")
    norm = torch.ones(d, device="cuda")
    qkv = torch.zeros((3, (groups + 2) * kv * d), device="cuda")
    one = torch.ones(3, dtype=torch.int32, device="cuda")

    def step(c):
        want = c.lengths + one
        c.resize(want)
        q = c.append(0, qkv, norm, norm, cos, cos, 1e-6)
        return c.attend(0, q), c.attend(0, q, window=9, sinks=2)

    eager, replayed = fresh(), fresh()
    step(fresh())
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs = step(replayed)
        graphs.append((g, outs))
    for i in range(12):
        qkv.copy_(torch.from_numpy(rng.standard_normal(tuple(qkv.shape)).astype(np.float32)))
        expect = step(eager)
        g, outs = graphs[i % 2]
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, expect):
            assert torch.equal(a, b), i
        for name in ("table", "lengths", "refs", "status"):
            assert torch.equal(getattr(eager, name), getattr(replayed, name)), (i, name)
        assert torch.equal(eager.keys, replayed.keys)
    assert eager.lengths.tolist() == [26, 42, 13]


@gpu
@pytest.mark.parametrize("sequences", [2, 300])
def test_captured_batches_that_are_cut(sequences):
    """Tiles in pieces and their join, with the plan in every wave and in a
    launch of its own: two graphs, replayed in turn with eager work between."""
    from harsh4b_amd.paged import paged_attention
    scenes = []
    for seed, counts, lengths in ((61, [1, 129], [900, 1111]), (62, [200, 3], [1300, 700])):
        spare = sequences - 2
        s = Scene(counts + [1] * spare, lengths + [30] * spare, 2, 5, 128, 64, seed=seed)
        d, starts = s.device(), torch.from_numpy(s.starts).cuda()
        scenes.append((d, starts, paged_attention(**d, starts=starts).clone()))
    torch.cuda.synchronize()
    graphs = []
    for d, starts, _ in scenes:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = paged_attention(**d, starts=starts)
        graphs.append((g, out))
    for i in range(6):
        (g, out), (d, starts, expect) = graphs[i % 2], scenes[i % 2]
        out.fill_(7.0)
        g.replay()
        other = scenes[1 - i % 2]
        assert torch.equal(paged_attention(**other[0], starts=other[1]), other[2]), i
        torch.cuda.synchronize()
        assert torch.equal(out, expect), i


@gpu
def test_captured_bookkeeping_of_many_rows():
    # more rows than the planning block has threads, a table past one block's fork: replays against an eager twin
    from harsh4b_amd.paged import PagedCache
    rows, rng = 1100, np.random.default_rng(63)
    eager, replayed = (PagedCache(1, 9000, 1, 16, sequences=rows, max_pages=16, page_size=16) for _ in range(2))
    first = rng.integers(0, 30, rows).tolist()
    parents = torch.from_numpy(rng.integers(-1, rows, rows).astype(np.int32)).cuda()
    for c in eager, replayed:
        c.keys.zero_()
        c.values.copy_(torch.arange(9000, device="cuda")[None, :, None, None, None] % 2039)
        c.resize(first)
    want = torch.empty(rows, dtype=torch.int32, device="cuda")

    def step(c):
        c.fork(parents)
        torch.add(c.lengths, 3, out=want)
        c.resize(want)
        c.compact()

    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step(replayed)
    for i in range(5):
        step(eager)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        for name in ("table", "lengths", "refs", "status", "values"):
            assert torch.equal(getattr(eager, name), getattr(replayed, name)), (i, name)
    assert int(eager.status.item()) == 0


@gpu
def test_appended_rows_are_the_decode_step_s():
    """The rows that paged_append writes, and its queries, have the bits of the
    decode step's norm and rotation (the oracle's)."""
    import oracle
    from harsh4b_amd.paged import paged_append
    kv, groups, d = 2, 4, 128
    s = Scene([7], [27], kv, groups, d, 16, seed=40)
    inputs = _append_inputs(s, kv, groups, d)
    dev = s.device()
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    q = paged_append(*[torch.from_numpy(a).cuda() for a in inputs], 1e-6, dev["keys"], dev["values"], dev["table"],
                     dev["lengths"], status, starts=torch.from_numpy(s.starts).cuda()).cpu().numpy()
    keys = dev["keys"].cpu().numpy()
    qkv, qn, kn, cos, sin = inputs
    rows = qkv.reshape(7, -1, d)
    for i in range(7):
        p = 20 + i
        eq = oracle.rope(oracle.head_norm(rows[i, :8].copy(), qn, 1e-6), cos[p], sin[p])
        ek = oracle.rope(oracle.head_norm(rows[i, 8:10].copy(), kn, 1e-6), cos[p], sin[p])
        np.testing.assert_array_equal(q[i].view(np.uint32), eq.view(np.uint32))
        np.testing.assert_array_equal(keys[s.place(0, p)].view(np.uint16), ek.astype(np.float16).view(np.uint16))
