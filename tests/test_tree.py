"""Steps over trees of drafted tokens (harsh4b_amd/tree.py, csrc/hq_tree.hip,
hq_tree_attn.hip) and the rows between the int4 products (add_rmsnorm_quant,
csrc/hq_norm.hip) against plain implementations: attention and append in
float64, plan and paths against lists, the rows against the oracle's bits.  No
reference counterpart."""
import ctypes
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from tests.test_paged import SHAPES, Scene, _append_inputs, _append_reference, _struct, native

gpu = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _announce(request):
    if request.node.get_closest_marker("gpu"):
        print(f"\n[gpu] {request.node.nodeid}", flush=True)
        yield
        torch.cuda.synchronize()
    else:
        yield


def up(a, dtype=None):
    return torch.from_numpy(np.ascontiguousarray(a if dtype is None else np.asarray(a, dtype=dtype))).cuda()


def ints(a):
    return up(a, np.int32)


# ------------------------------------------------------------------ trees
def random_tree(rng, n, deep=1000, roots=False):
    """Parents of n nodes; with `roots` some others than the first have none."""
    parents, depth = [], []
    for i in range(n):
        p = -1
        if i and not (roots and rng.random() < 0.2):
            open_nodes = [j for j in range(i) if depth[j] < deep]
            p = int(open_nodes[int(rng.integers(0, len(open_nodes)))])
        parents.append(p)
        depth.append(0 if p < 0 else depth[p] + 1)
    return parents


def chain(n):
    return list(range(-1, n - 1))


def star(n):
    return [-1] + [0] * (n - 1)


def depths_of(parents):
    d = []
    for p in parents:
        d.append(0 if p < 0 else d[p] + 1)
    return d


def ancestors_of(parents):
    n = len(parents)
    sees = np.zeros((n, n), dtype=bool)
    for i, p in enumerate(parents):
        if p >= 0:
            sees[i] = sees[p]
        sees[i, i] = True
    return sees


def starts_of(trees):
    return np.concatenate([[0], np.cumsum([len(t) for t in trees])]).astype(np.int32)


def plan(trees, status=None, **more):
    from harsh4b_amd.tree import tree_plan
    status = ints([0]) if status is None else status
    parents = np.concatenate([np.asarray(t, dtype=np.int32) for t in trees]) if trees else np.zeros(0, np.int32)
    return tree_plan(ints(parents), ints(starts_of(trees)), status, **more)


def bits_of(words):
    return np.unpackbits(words.cpu().numpy().view(np.uint8), axis=1, bitorder="little").astype(bool)


# ------------------------------------------------------------------ refusals (no launch)
def _tree_struct(p, **change):
    f = dict(tokens=3, reserved=0, starts=p, parents=p, depths=p, ancestors=p)
    f.update(change)
    n = native()
    return n.HqTree(*[f[name] for name, _ in n.HqTree._fields_])


def test_c_entries_refuse_bad_trees():
    lib = native().lib()
    c, p, _ = _struct()
    c = ctypes.byref(c)
    for change, code in ((dict(tokens=-1), 1), (dict(starts=None), 1), (dict(parents=None), 1), (dict(depths=None), 1),
                         (dict(ancestors=None), 1), (dict(parents=p + 2), 2), (dict(ancestors=p + 4), 2),
                         (dict(starts=p + 1), 2)):
        t = ctypes.byref(_tree_struct(p, **change))
        assert lib.hq_tree_plan(t, 3, p, None) == code, change
        assert lib.hq_paged_append_tree(c, p, t, 4, p, p, 1e-6, p, p, 10, p, None) == code, change
        assert lib.hq_paged_attention_tree(c, p, t, 4, 0, 0, p, p, None) == code, change
        assert lib.hq_pages_accept(c, t, p, p, None, 0, 4, p, p, p, p, None) == code, change
    assert lib.hq_tree_plan(None, 3, p, None) == 1


@pytest.mark.parametrize("change", [dict(pages=0), dict(page_size=48), dict(head_dim=24), dict(kv_heads=0), dict(sequences=0),
                                    dict(max_pages=1 << 28), dict(keys=None), dict(table=None), dict(lengths=None),
                                    dict(status=None)])
def test_c_entries_refuse_bad_caches(change):
    lib = native().lib()
    c, p, _ = _struct(**change)
    c, t = ctypes.byref(c), ctypes.byref(_tree_struct(p))
    if "status" not in change:
        assert lib.hq_paged_attention_tree(c, p, t, 4, 0, 0, p, p, None) == 1
    assert lib.hq_paged_append_tree(c, p, t, 4, p, p, 1e-6, p, p, 10, p, None) == 1
    assert lib.hq_pages_accept(c, t, p, p, None, 0, 4, p, p, p, p, None) == 1


def test_c_entries_refuse_bad_arguments():
    lib = native().lib()
    s, p, _ = _struct()
    c, t, none = ctypes.byref(s), ctypes.byref(_tree_struct(p)), ctypes.byref(_tree_struct(p, tokens=0))
    assert lib.hq_tree_plan(t, 0, p, None) == 1 and lib.hq_tree_plan(t, 3, None, None) == 1
    assert lib.hq_tree_plan(t, 1 << 24, p, None) == 1
    at = lib.hq_paged_attention_tree
    assert at(None, p, t, 4, 0, 0, p, p, None) == 1 and at(c, None, t, 4, 0, 0, p, p, None) == 1
    assert at(c, p, t, 5, 0, 0, p, p, None) == 1 and at(c, p, t, 18, 0, 0, p, p, None) == 1
    assert at(c, p, t, 4, -1, 0, p, p, None) == 1 and at(c, p, t, 4, 1, -1, p, p, None) == 1
    assert at(c, p, t, 4, 0, 0, None, p, None) == 1 and at(c, p, t, 4, 0, 0, p, None, None) == 1
    assert at(c, p, t, 4, 0, 0, p, p + 16, None) == 2 and at(c, p + 4, t, 4, 0, 0, p, p, None) == 2
    assert at(c, p, none, 4, 0, 0, p, p, None) == 0
    ap = lib.hq_paged_append_tree
    assert ap(c, p, t, 4, None, p, 1e-6, p, p, 10, p, None) == 1 and ap(c, p, t, 4, p, p, 1e-6, p, p, 0, p, None) == 1
    assert ap(c, p, none, 4, p, p, 1e-6, p, p, 10, p, None) == 0
    assert lib.hq_paged_attention_tree_workspace_bytes(3, 5, 2, 32) == 0
    assert lib.hq_paged_attention_tree_workspace_bytes(3, 4, 2, 32) > 0
    ac = lib.hq_pages_accept
    assert ac(None, t, p, p, None, 0, 4, p, p, p, p, None) == 1
    assert ac(c, t, None, p, None, 0, 4, p, p, p, p, None) == 1       # drafted
    assert ac(c, t, p, None, None, 0, 4, p, p, p, p, None) == 1       # neither choices nor logits
    assert ac(c, t, p, p, p, 9, 4, p, p, p, p, None) == 1             # both
    assert ac(c, t, p, None, p, 0, 4, p, p, p, p, None) == 1 and ac(c, t, p, p, None, 9, 4, p, p, p, p, None) == 1
    assert ac(c, t, p, p, None, 0, 0, p, p, p, p, None) == 1 and ac(c, t, p, p, None, 0, 257, p, p, p, p, None) == 1
    assert ac(c, t, p, p, None, 0, 4, None, p, p, p, None) == 1 and ac(c, t, p, p, None, 0, 4, p, None, p, p, None) == 1
    assert ac(c, t, p, p, None, 0, 4, p, p, None, p, None) == 1 and ac(c, t, p, p, None, 0, 4, p, p, p, None, None) == 1
    assert ac(c, t, p, p, None, 0, 4, p, p, p, p + 64, None) == 2 and ac(c, t, p, p + 2, None, 0, 4, p, p, p, p, None) == 2
    few, _, _ = _struct(layers=0)
    assert ac(ctypes.byref(few), t, p, p, None, 0, 4, p, p, p, p, None) == 1
    size = lib.hq_pages_accept_workspace_bytes
    assert size(-1, 1, 0, 4) == 0 and size(3, 0, 0, 4) == 0 and size(3, 1, -1, 4) == 0 and size(3, 1, 9, 257) == 0
    assert size(3, 1, 0, 4) == 256 and size(600, 1, 151936, 256) >= 8 * 600
    norm = lib.hq_add_rmsnorm_quant
    for bad in ((None, p, p, p, p, p), (p, p, None, p, p, p), (p, p, p, None, p, p), (p, p, p, p, None, p),
                (p, p, p, p, p, None)):
        assert norm(*bad, 2, 8, 1e-6, None) == 1
    assert norm(p, None, p, None, p, p, 2, 0, 1e-6, None) == 1 and norm(p, None, p, None, p, p, -1, 8, 1e-6, None) == 1
    assert norm(p, None, p, None, p, p, 1 << 24, 8, 1e-6, None) == 1
    assert norm(p, None, p, None, p, p, 2, (1 << 30) + 1, 1e-6, None) == 1
    assert norm(p + 2, None, p, None, p, p, 2, 8, 1e-6, None) == 2
    assert norm(p, None, p, None, p, p, 0, 8, 1e-6, None) == 0


def test_python_refuses_host_tensors():
    from harsh4b_amd import lightspark, tree
    i = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(ValueError, match="device tensor"):
        tree.tree_plan(i, i, i[:1])
    k = torch.zeros((4, 2, 16, 32), dtype=torch.float16)
    t = tree.DraftTree(i, i, i, torch.zeros((3, 8), dtype=torch.int32))
    with pytest.raises(ValueError, match="device tensor"):
        tree.paged_attention_tree(torch.zeros(3, 4, 32), k, k, torch.zeros((2, 3), dtype=torch.int32), i[:2], t)
    with pytest.raises(ValueError, match="device tensor"):
        tree.pages_accept(k[None], k[None], torch.zeros((2, 3), dtype=torch.int32), i[:2], i[:1], t, i, choices=i)
    with pytest.raises(ValueError, match="device tensor"):
        lightspark.add_rmsnorm_quant(torch.zeros(2, 8), torch.zeros(8), 1e-6)


@gpu
def test_python_refuses_bad_device_arguments():
    from harsh4b_amd import lightspark, paged, tree
    c = paged.PagedCache(2, 6, 2, 32, sequences=3, max_pages=2, page_size=16)
    t = plan([[-1], [-1, 0], [-1]])
    q, qkv = torch.zeros((4, 4, 32), device="cuda"), torch.zeros((4, 8 * 32), device="cuda")
    norm, rope = torch.ones(32, device="cuda"), torch.ones((8, 16), device="cuda")

    def refuse(match, call, *args, **more):
        with pytest.raises(ValueError, match=match):
            call(*args, **more)

    attend = lambda query=q, tr=t, **more: tree.paged_attention_tree(query, c.keys[0], c.values[0], c.table, c.lengths, tr, **more)
    refuse("starts", attend, tr=t._replace(starts=t.starts[:3]))
    refuse("starts", attend, tr=t._replace(starts=None))
    refuse("parents", attend, tr=t._replace(parents=t.parents[:3]))
    refuse("depths", attend, tr=t._replace(depths=t.depths.long()))
    refuse("ancestors", attend, tr=t._replace(ancestors=t.ancestors[:, :4].contiguous()))
    refuse("query", attend, query=q.half())
    refuse("query", attend, query=torch.zeros((4, 5, 32), device="cuda"))
    refuse("negative", attend, window=-1)
    refuse("overlap", attend, out=q)
    refuse("out", attend, out=q[:3])
    append = lambda x=qkv, tr=t, **more: tree.paged_append_tree(x, norm, norm, rope, rope, 1e-6, c.keys[0], c.values[0], c.table,
                                                                c.lengths, c.status, tr, **more)
    refuse("qkv", append, x=qkv[:, :200].contiguous())
    refuse("parents", append, x=qkv, tr=t._replace(parents=t.parents.float()))
    refuse("overlap", append, out=qkv.view(-1)[:512].view(4, 4, 32))
    drafted = ints([1, 2, 3, 4])
    accept = lambda ids=drafted, tr=t, **more: tree.pages_accept(c.keys, c.values, c.table, c.lengths, c.status, tr, ids, **more)
    refuse("either", accept)
    refuse("either", accept, choices=drafted, logits=torch.zeros((4, 9), device="cuda"))
    refuse("drafted", accept, ids=drafted.long(), choices=drafted)
    refuse("choices", accept, choices=drafted[:3])
    refuse("logits", accept, logits=torch.zeros((3, 9), device="cuda"))
    refuse("logits", accept, logits=torch.zeros((9, 4), device="cuda").t())
    refuse("levels", accept, choices=drafted, levels=0)
    refuse("levels", accept, choices=drafted, levels=257)
    kept = torch.empty(3, dtype=torch.int32, device="cuda")
    refuse("overlap", accept, choices=drafted, out=(kept, drafted, kept.clone()))
    refuse("overlap", accept, choices=drafted, out=(kept, drafted.clone(), kept))
    refuse("status", tree.tree_plan, t.parents, t.starts, c.status.long())
    refuse("parents", tree.tree_plan, t.parents.long(), t.starts, c.status)
    refuse("overlap", tree.tree_plan, t.parents, t.starts, c.status, depths=t.parents)
    x, gamma = torch.zeros((4, 32), device="cuda"), torch.ones(32, device="cuda")
    rows = lightspark.add_rmsnorm_quant
    refuse("x must", rows, x.t(), gamma, 1e-6)
    refuse("x must", rows, x[0], gamma, 1e-6)
    refuse("gamma", rows, x, gamma[:16], 1e-6)
    refuse("gamma", rows, x, None, 1e-6)
    refuse("delta", rows, x, gamma, 1e-6, delta=x[:3])
    refuse("q must", rows, x, gamma, 1e-6, q=x)
    refuse("overlap", rows, x[:3], gamma, 1e-6, delta=torch.ones((3, 32), device="cuda"), out=x[1:])
    delta = torch.ones_like(x)
    refuse("overlap", rows, x, gamma, 1e-6, delta=delta, out=delta)
    assert int(c.status.item()) == 0


# ------------------------------------------------------------------ rows between the products
def _norm_expect(x, delta, gamma, eps):
    import oracle
    total = x if delta is None else (x + delta).astype(np.float32)
    rows = [oracle.quantize_activation(oracle.rmsnorm(r, gamma, eps)) for r in total]
    return total, np.stack([q for q, _ in rows]), np.array([s for _, s in rows], dtype=np.float32)


@gpu
@pytest.mark.parametrize("rows,n", [(1, 1), (3, 2), (2, 63), (5, 64), (3, 255), (4, 256), (5, 257), (2, 1000), (7, 2560),
                                    (33, 2560), (4, 4099), (3, 8192), (3, 9728), (2, 16384), (2, 20001), (1500, 320),
                                    (1, 100003)])
@pytest.mark.parametrize("with_delta", [False, True])
def test_rows_have_the_single_row_calls_bits(rows, n, with_delta):
    from harsh4b_amd.lightspark import add_rmsnorm_quant
    rng = np.random.default_rng(rows * 7 + n)
    x = (3 * rng.standard_normal((rows, n))).astype(np.float32)
    delta = rng.standard_normal((rows, n)).astype(np.float32) if with_delta else None
    gamma = rng.uniform(0.5, 1.5, n).astype(np.float32)
    total, eq, es = _norm_expect(x, delta, gamma, 1e-6)
    for place in ("in place", "out"):
        dx = up(x)
        out = torch.full((rows, n), 7.0, device="cuda") if place == "out" else None
        q, s = add_rmsnorm_quant(dx, up(gamma), 1e-6, delta=None if delta is None else up(delta), out=out)
        np.testing.assert_array_equal(q.cpu().numpy(), eq)
        np.testing.assert_array_equal(s.cpu().numpy().view(np.uint32), es.view(np.uint32))
        if with_delta or out is not None:
            np.testing.assert_array_equal((dx if out is None else out).cpu().numpy().view(np.uint32), total.view(np.uint32))
        if out is not None:
            np.testing.assert_array_equal(dx.cpu().numpy(), x)


@gpu
@pytest.mark.parametrize("n", [512, 513, 2560])
def test_rows_at_any_alignment(n):
    # every array at an odd element, its neighbours left as they were
    from harsh4b_amd.lightspark import add_rmsnorm_quant
    rng = np.random.default_rng(n)
    x, delta = (rng.standard_normal((5, n)).astype(np.float32) for _ in range(2))
    gamma = rng.uniform(0.5, 1.5, n).astype(np.float32)
    total, eq, es = _norm_expect(x, delta, gamma, 1e-5)
    for shift in (1, 2, 3):
        def at(a, dtype=torch.float32):
            flat = torch.full((a.size + 8,), 9, dtype=dtype, device="cuda")
            view = flat[shift:shift + a.size].view(a.shape)
            view.copy_(up(a))
            return flat, view
        (_, dx), (_, dd), (_, dg) = at(x), at(delta), at(gamma)
        (fo, out), (fq, q), (fs, s) = at(0 * x), at(0 * x, torch.int8), at(np.zeros(5, np.float32))
        add_rmsnorm_quant(dx, dg, 1e-5, delta=dd, out=out, q=q, act_scales=s)
        np.testing.assert_array_equal(q.cpu().numpy(), eq)
        np.testing.assert_array_equal(out.cpu().numpy(), total)
        np.testing.assert_array_equal(s.cpu().numpy(), es)
        for flat, size in ((fo, x.size), (fq, x.size), (fs, 5)):
            rest = flat.cpu().numpy()
            assert (rest[:shift] == 9).all() and (rest[shift + size:] == 9).all()


@gpu
@pytest.mark.parametrize("n", [300, 2560])
def test_rows_that_are_not_finite(n):
    # zeros, infinities, NaN, values whose squares overflow or vanish: the single row calls' bits, row by row
    from harsh4b_amd.lightspark import add_rmsnorm_quant, quantize_activation, rmsnorm
    rng = np.random.default_rng(n)
    x = rng.standard_normal((8, n)).astype(np.float32)
    x[1] = 0
    x[2, 5] = np.inf
    x[3, 7] = np.nan
    x[4] *= np.float32(1e30)
    x[5] *= np.float32(1e-30)
    x[6, 3] = -np.inf
    x[7] = np.finfo(np.float32).max
    gamma = rng.uniform(0.5, 1.5, n).astype(np.float32)
    dx, dg = up(x), up(gamma)
    q, s = add_rmsnorm_quant(dx, dg, 1e-6)
    for i in range(8):
        eq, es = quantize_activation(rmsnorm(dx[i].contiguous(), dg, 1e-6))
        assert torch.equal(q[i], eq), i
        assert s[i].cpu().numpy().tobytes() == es[0].cpu().numpy().tobytes() or (s[i].isnan() and es[0].isnan()), i


@gpu
def test_rows_feed_the_product():
    # what int4_i8_gemm makes of them is what the fused product makes of the normed rows
    from harsh4b_amd import lightspark as ls
    from tests.gpu_util import random_int4
    rng = np.random.default_rng(3)
    w = ls.LiteSparkProjection(up(ls.pack_int4(random_int4(rng, 384, 512))), up(rng.uniform(0.005, 0.02, 384).astype(np.float32)))
    x, gamma = up(rng.standard_normal((19, 512)).astype(np.float32)), up(rng.uniform(0.5, 1.5, 512).astype(np.float32))
    q, s = ls.add_rmsnorm_quant(x, gamma, 1e-6)
    normed = torch.stack([ls.rmsnorm(r.contiguous(), gamma, 1e-6) for r in x])
    assert torch.equal(ls.int4_i8_gemm(q, s, w), ls.quant_int4_gemm(normed, w))


@gpu
def test_rows_of_more_than_2_31_values():
    from harsh4b_amd.lightspark import add_rmsnorm_quant
    rows, n = (1 << 31) // 4096 + 3, 4096
    x = torch.empty((rows, n), device="cuda")
    x[:] = (torch.arange(n, device="cuda") % 17).float()
    x[-1] = (torch.arange(n, device="cuda") % 13).float()
    gamma = torch.ones(n, device="cuda")
    q, s = add_rmsnorm_quant(x, gamma, 1e-6)
    eq, es = add_rmsnorm_quant(x[-3:].clone(), gamma, 1e-6)
    assert torch.equal(q[-3:], eq) and torch.equal(s[-3:], es)


# ------------------------------------------------------------------ plan
def _check_plan(trees):
    status = ints([0])
    t = plan(trees, status)
    depths, bits = t.depths.cpu().numpy(), bits_of(t.ancestors)
    at = 0
    for parents in trees:
        n = len(parents)
        np.testing.assert_array_equal(depths[at:at + n], depths_of(parents))
        np.testing.assert_array_equal(bits[at:at + n, :n], ancestors_of(parents))
        assert not bits[at:at + n, n:].any()
        at += n
    assert int(status.item()) == 0


@gpu
@pytest.mark.parametrize("n", [1, 2, 5, 31, 32, 33, 63, 64, 65, 128, 200, 255, 256])
def test_plan(n):
    rng = np.random.default_rng(n)
    _check_plan([random_tree(rng, n), [], chain(n), star(n), random_tree(rng, n, 3), random_tree(rng, n, roots=True), [-1]])


@gpu
def test_plan_of_many_trees():
    rng = np.random.default_rng(9)
    _check_plan([random_tree(rng, int(rng.integers(0, 20))) for _ in range(900)])


@gpu
def test_plan_reports_trees_that_are_none():
    rng = np.random.default_rng(2)
    for bad in ([0], [-1, 1], [-1, 0, 5], [-1, -2], [-1] + [2**31 - 1] * 3, [-2**31], chain(257), [-1] * 300):
        trees = [random_tree(rng, 9), bad, random_tree(rng, 4)]
        status = ints([0])
        t = plan(trees, status)
        depths, bits = t.depths.cpu().numpy(), t.ancestors.cpu().numpy()
        n = len(bad)
        assert int(status.item()) == 2
        assert (depths[9:9 + n] == -1).all() and not bits[9:9 + n].any()
        np.testing.assert_array_equal(depths[:9], depths_of(trees[0]))
        np.testing.assert_array_equal(depths[9 + n:], depths_of(trees[2]))


@gpu
@pytest.mark.parametrize("starts,good", [([0, 2, 1, 4], [0, 2]), ([-3, 2, 5, 6], [1, 2]), ([0, 2, 9, 10], [0]), ([4, 2, 5, 6], [1, 2]),
                                         ([1, 3, 3, 4], [0, 1, 2])])
def test_plan_of_starts_outside_the_batch(starts, good):
    from harsh4b_amd.tree import tree_plan
    status, parents = ints([0]), ints([-1] * 6)
    depths, ancestors = ints([77] * 6), ints(np.full((6, 8), 77))
    tree_plan(parents, ints(starts), status, depths=depths, ancestors=ancestors)
    rows = [r for b in good for r in range(starts[b], starts[b + 1])]
    expect = np.full(6, 77)
    expect[rows] = 0
    np.testing.assert_array_equal(depths.cpu().numpy(), expect)
    assert (ancestors.cpu().numpy()[expect == 77] == 77).all()
    assert int(status.item()) == (2 if len(good) < 3 else 0)


# ------------------------------------------------------------------ attention
def _reference(s, trees, window, sinks):
    """The definition in float64, a sequence's head at a time, and the bound of
    each row's error (that of tests/test_paged.py: a score's products and sums,
    the weights' error, the sums over the positions)."""
    pages, kv, ps, d = s.keys.shape
    heads = s.query.shape[1]
    out, bound = np.zeros(s.query.shape), np.zeros(s.tokens)
    for b, parents in enumerate(trees):
        n, length = len(parents), s.lengths[b]
        if n == 0:
            continue
        rows = slice(s.starts[b], s.starts[b + 1])
        base = length - n
        j = np.arange(0, max(0, min(length, s.table.shape[1] * ps)))
        page = s.table[b][j // ps]
        there = (page >= 0) & (page < pages)
        depth = np.array(depths_of(parents))
        sees = np.zeros((n, len(j)), dtype=bool)
        sees[:, j < base] = True
        tree = ancestors_of(parents)
        position = j.copy()
        for i in range(n):
            if 0 <= base + i < len(j):
                sees[:, base + i] = tree[:, i]
                position[base + i] = base + depth[i]
        if base < 0:
            sees[:-base] = False                       # (nodes before the sequence)
        if window:
            sees &= ((position[None, :] > base + depth[:, None] - window) | (position < sinks)[None, :])
        sees &= there[None, :]
        some = sees.any(axis=1)
        if not some.any():
            continue
        use = sees.any(axis=0)
        keys, values = (np.where(use[:, None, None], pool[np.where(there, page, 0), :, j % ps], 0).astype(np.float64)
                        for pool in (s.keys, s.values))
        for h in range(heads):
            k, v, q = keys[:, h // (heads // kv)], values[:, h // (heads // kv)], s.query[rows, h].astype(np.float64)
            score = np.where(sees, q @ k.T / math.sqrt(d), -np.inf)
            with np.errstate(invalid="ignore"):
                e = np.where(sees, np.exp(score - score.max(axis=1, keepdims=True)), 0.0)
                out[rows, h] = np.where(some[:, None], e @ v / e.sum(axis=1, keepdims=True), 0.0)
            size = np.where(sees, np.abs(q) @ np.abs(k).T, 0.0).max(axis=1) / math.sqrt(d)
            bound[rows] = np.maximum(bound[rows], np.abs(v).max() * (2 * (d + 8) * 2.0 ** -24 * size +
                                                                     (sees.sum(axis=1) + 64) * 2.0 ** -24))
    return out, bound


class Trees(Scene):
    """A Scene whose new tokens are the nodes of trees."""

    def __init__(self, trees, bases, *shape, **more):
        super().__init__([len(t) for t in trees], [b + len(t) for b, t in zip(bases, trees)], *shape, **more)
        self.trees = trees

    def attend(self, window=0, sinks=0, plan_stream=None, **more):
        from harsh4b_amd.tree import paged_attention_tree
        d = self.device()
        t = plan(self.trees)
        out = paged_attention_tree(**d, tree=t, window=window, sinks=sinks, **more)
        torch.cuda.synchronize()
        return out.cpu().numpy()

    def _check(self, window=0, sinks=0, **more):
        got = self.attend(window, sinks, **more)
        expect, bound = _reference(self, self.trees, window, sinks)
        off = np.abs(got - expect).reshape(self.tokens, -1).max(axis=1)
        assert (off <= bound).all(), (np.argmax(off - bound), off.max(), bound[np.argmax(off - bound)])
        return got

    def check(self, window=0, sinks=0):
        """With the table as it is, and as a row of a longer cache's."""
        got = self._check(window, sinks)
        table, page = self.table, self.keys.shape[2]
        wide = -(-1100 // page)
        if table.shape[1] < wide:
            self.table = np.full((table.shape[0], wide), -1, dtype=np.int32)
            self.table[:, :table.shape[1]] = table
            self._check(window, sinks)
            self.table = table
        return got


def some_trees(seed, sizes, **more):
    rng = np.random.default_rng(seed)
    return [random_tree(rng, n, **more) if n else [] for n in sizes]


@gpu
@pytest.mark.parametrize("kv,groups,d", SHAPES)
@pytest.mark.parametrize("page", [16, 64, 256])
def test_small_trees(kv, groups, d, page):
    Trees(some_trees(d + groups, [1, 2, 4, 3, 0, 2]), [0, 15, 16, 61, 5, 301], kv, groups, d, page, seed=d).check()


@gpu
@pytest.mark.parametrize("kv,groups,d", SHAPES)
def test_trees_of_all_sizes(kv, groups, d):
    Trees(some_trees(d, [5, 0, 1, 37, 130, 0, 2, 64, 8, 16]), [0, 40, 77, 63, 1, 0, 300, 65, 129, 31], kv, groups, d, 32,
          seed=d).check()


@gpu
@pytest.mark.parametrize("n", [1, 7, 8, 9, 15, 16, 17, 31, 32, 33, 63, 64, 65, 100, 128, 129, 255, 256])
@pytest.mark.parametrize("kind", ["chain", "star", "random", "forest"])
def test_kinds_of_trees(n, kind):
    rng = np.random.default_rng(n)
    tree = dict(chain=chain(n), star=star(n), random=random_tree(rng, n), forest=random_tree(rng, n, roots=True))[kind]
    Trees([tree, [-1]], [n % 70, 3], 1, 4, 64, 16, seed=n).check()


@gpu
@pytest.mark.parametrize("base", [0, 1, 31, 32, 33, 63, 64, 65, 95, 96, 127, 128])
def test_bases_in_a_chunk(base):
    # where the tree begins in a chunk of 64 positions and its halves
    for seed, n in ((1, 3), (2, 20), (3, 90)):
        Trees(some_trees(seed + base, [n]), [base], 2, 4, 32, 16, seed=base).check()


@gpu
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (2, 0), (3, 40), (7, 0), (16, 4), (33, 17), (64, 70), (1000, 4),
                                          (2**31 - 1, 3), (100, 2**31 - 1), (5, 303)])
def test_window_and_sinks(window, sinks):
    # windows shorter than the trees' paths among them
    trees = some_trees(window % 1000, [3, 1, 40, 100]) + [chain(90), chain(30)]
    Trees(trees, [297, 0, 50, 160, 211, 2], 2, 4, 64, 16, seed=sinks % 1000).check(window, sinks)


@gpu
@pytest.mark.parametrize("sizes,bases", [([4], [1100]), ([16, 1], [2050, 3000]), ([64, 60], [1111, 200]), ([256], [700]),
                                         ([8] * 9, list(range(900, 1800, 100)))])
def test_longer(sizes, bases):
    Trees(some_trees(len(sizes), sizes), bases, 2, 4, 128, 64, seed=sizes[0]).check()
    Trees(some_trees(len(sizes), sizes), bases, 8, 2, 64, 32, seed=sizes[0]).check(window=500, sinks=2)


@gpu
@pytest.mark.parametrize("sequences", [64, 65, 255, 256, 300, 1300])
def test_many_sequences(sequences):
    rng = np.random.default_rng(sequences)
    sizes = [int(n) for n in rng.integers(0, 9, sequences)]
    Trees(some_trees(5, sizes), [int(b) for b in rng.integers(0, 50, sequences)], 1, 3, 32, 16, seed=5).check()


@gpu
def test_a_chain_sees_what_a_chunk_sees():
    from harsh4b_amd.paged import paged_attention
    for counts, window in (([3, 40, 1], 0), ([130, 2], 50)):
        s = Trees([chain(n) for n in counts], [200, 33, 90][:len(counts)], 2, 4, 128, 16, seed=2)
        d = s.device()
        expect = paged_attention(**d, starts=ints(s.starts), window=window, sinks=1)
        got = s.attend(window, 1)
        _, bound = _reference(s, s.trees, window, 1)
        assert (np.abs(got - expect.cpu().numpy()).reshape(s.tokens, -1).max(axis=1) <= 2 * bound).all()


@gpu
@pytest.mark.parametrize("what", ["nan", "inf", "-inf"])
@pytest.mark.parametrize("n", [4, 20, 60])
def test_hidden_nodes_of_any_value(what, n):
    # K and V of nodes that a row does not see, and of positions behind its window, never reach it
    trees = [star(n), random_tree(np.random.default_rng(n), n), [-1]]
    s = Trees(trees, [70, 130, 9], 2, 4, 128, 16, seed=n)
    for b, parents in enumerate(trees[:2]):
        base = s.lengths[b] - n
        sees = ancestors_of(parents)
        leaf = int(np.flatnonzero(sees.sum(axis=0) == 1)[-1])       # (seen by itself alone)
        for pool in (s.keys, s.values):
            pool[s.place(b, base + leaf)] = float(what)
            pool[s.place(b, 3)] = float(what)                       # (behind the window)
        s.leaf = leaf
    got = s.attend(window=60)
    clean = Trees(trees, [70, 130, 9], 2, 4, 128, 16, seed=n)
    expect, bound = _reference(clean, trees, 60, 0)
    own = []
    for b, parents in enumerate(trees[:2]):
        own.append(s.starts[b] + int(np.flatnonzero(ancestors_of(parents).sum(axis=0) == 1)[-1]))
    rest = np.setdiff1d(np.arange(s.tokens), own)
    off = np.abs(got - expect).reshape(s.tokens, -1).max(axis=1)
    assert (off[rest] <= bound[rest]).all(), what
    assert not np.isfinite(got[own]).all()


@gpu
def test_rows_that_see_nothing():
    from harsh4b_amd.tree import paged_attention_tree
    # nodes before the sequence; a window of one over a page that is gone; trees that are none; rows of nobody
    s = Trees(some_trees(3, [6, 40, 3]), [10, 50, 7], 2, 4, 64, 16, seed=3)
    s.lengths[0] = 4
    got = s._check()
    assert (got[:2] == 0).all()
    s.table[2] = -1
    assert (s._check()[46:] == 0).all()
    d = s.device()
    parents = np.concatenate(s.trees).astype(np.int32)
    for b, at in ((0, 5), (1, 30), (1, 6)):
        bad = parents.copy()
        bad[at] = 200
        starts = ints(np.concatenate([s.starts[:3], s.starts[2:3]]))
        from harsh4b_amd.tree import tree_plan
        t = tree_plan(ints(bad), starts, ints([0]), depths=ints(np.full(49, 5)), ancestors=ints(np.full((49, 8), -1)))
        out = torch.full_like(d["query"], 7.0)
        paged_attention_tree(**d, tree=t, out=out)
        out = out.cpu().numpy()
        assert (out[s.starts[b]:s.starts[b + 1]] == 0).all()
        other = slice(s.starts[1 - b], s.starts[2 - b])
        np.testing.assert_array_equal(out[other], got[other])
        assert (out[46:] == 7.0).all()


@gpu
def test_holes_and_bad_entries():
    s = Trees(some_trees(8, [3, 50, 9]), [300, 200, 1200], 2, 4, 64, 16, seed=8)
    s.table[0, 2:5] = -1
    s.table[1, 0] = 10**6
    s.table[1, 7] = -5
    s.table[2, 75] = -1                               # a page of the tree
    s.check()
    s.check(window=100, sinks=30)


@gpu
@pytest.mark.parametrize("lengths", [[2**31 - 1, 20], [-5, 20], [-(2**31), 20], [1000, 20], [2, 20]])
def test_lengths_outside_the_table(lengths):
    # no access out of range: sequence 1 has its result, sequence 0 any that the table gives
    s = Trees(some_trees(6, [30, 7]), [10, 13], 2, 4, 64, 16, seed=6)
    expect, bound = _reference(s, s.trees, 0, 0)
    s.lengths = lengths
    got = s.attend()
    off = np.abs(got - expect)[30:].reshape(7, -1).max(axis=1)
    assert (off <= bound[30:]).all()


@gpu
@pytest.mark.parametrize("starts", [[0, 2, 1], [0, 9, 10], [-3, 2, 5], [4, 2, 5], [0, 0, 0]])
def test_starts_out_of_order(starts):
    from harsh4b_amd.tree import paged_attention_tree
    s = Trees([[-1, 0], [-1, 0, 0]], [10, 20], page=16, seed=11)
    d, t = s.device(), plan(s.trees)
    out = torch.full_like(d["query"], 7.0)
    paged_attention_tree(**d, tree=t._replace(starts=ints(starts)), out=out)
    torch.cuda.synchronize()
    if any(a > z for a, z in zip(starts, starts[1:])) or starts == [0, 0, 0]:
        assert (out == 7.0).all()


@gpu
def test_other_streams():
    from harsh4b_amd.tree import paged_attention_tree
    scenes = [Trees(some_trees(12, [1, 40]), [100, 1090], page=16, seed=12), Trees(some_trees(13, [33, 2]), [2000, 700], page=16, seed=13)]
    expect = [s.check() for s in scenes]
    streams = [torch.cuda.Stream() for _ in scenes]
    inputs = [(s.device(), plan(s.trees)) for s in scenes]
    torch.cuda.synchronize()
    for _ in range(20):
        outs = [paged_attention_tree(**d, tree=t, stream=x) for (d, t), x in zip(inputs, streams)]
    torch.cuda.synchronize()
    for out, e in zip(outs, expect):
        np.testing.assert_array_equal(out.cpu().numpy(), e)


# ------------------------------------------------------------------ append
def _append(s, trees, inputs, **more):
    from harsh4b_amd.tree import paged_append_tree
    dev = s.device()
    status = ints([0])
    t = plan(trees, ints([0]))
    q = paged_append_tree(*[up(a) for a in inputs], 1e-6, dev["keys"], dev["values"], dev["table"], dev["lengths"], status,
                          t, **more)
    torch.cuda.synchronize()
    return q.cpu().numpy(), dev["keys"].cpu().numpy(), dev["values"].cpu().numpy(), int(status.item())


@gpu
@pytest.mark.parametrize("kv,groups,d", SHAPES)
def test_append(kv, groups, d):
    trees = some_trees(d, [1, 0, 5, 40, 17]) + [chain(9), star(12)]
    s = Trees(trees, [0, 9, 30, 100, 15, 64, 3], kv, groups, d, 16, seed=d)
    inputs = _append_inputs(s, kv, groups, d)
    q, keys, values, status = _append(s, trees, inputs)
    position = np.concatenate([np.array(depths_of(t), dtype=int) + n - len(t) for t, n in zip(trees, s.lengths)])
    eq, ek, ev = _append_reference(*inputs, 1e-6, kv * groups, kv, d, position)
    # the norm: d + 4 roundings of its sum, root and products; the rotation: 3; of values up to 2 |x|
    big = np.abs(eq).max()
    assert np.abs(q - eq).max() <= (d / 2 + 8) * 2.0 ** -24 * 2 * big
    before = Trees(trees, [0, 9, 30, 100, 15, 64, 3], kv, groups, d, 16, seed=d)
    t = 0
    for b, tree in enumerate(trees):
        for i in range(len(tree)):
            place = s.place(b, s.lengths[b] - len(tree) + i)
            # (an fp16 rounding: half a step, subnormal below 2^-14)
            np.testing.assert_allclose(keys[place], ek[t], rtol=2.0 ** -11 + 2.0 ** -16, atol=2.0 ** -24 + 2e-5)
            np.testing.assert_array_equal(values[place], ev[t].astype(np.float16))
            before.keys[place], before.values[place] = keys[place], values[place]
            t += 1
    np.testing.assert_array_equal(keys, before.keys)                  # nothing else is written
    np.testing.assert_array_equal(values, before.values)
    assert status == 0


@gpu
def test_append_of_a_chain_has_the_chunk_s_bits():
    from harsh4b_amd.paged import paged_append
    counts = [3, 1, 200]
    s = Trees([chain(n) for n in counts], [20, 0, 31], 2, 4, 128, 16, seed=4)
    inputs = _append_inputs(s, 2, 4, 128)
    q, keys, values, _ = _append(s, s.trees, inputs)
    dev, status = s.device(), ints([0])
    eq = paged_append(*[up(a) for a in inputs], 1e-6, dev["keys"], dev["values"], dev["table"], dev["lengths"], status,
                      starts=ints(s.starts))
    np.testing.assert_array_equal(q, eq.cpu().numpy())
    np.testing.assert_array_equal(keys, dev["keys"].cpu().numpy())
    np.testing.assert_array_equal(values, dev["values"].cpu().numpy())


@gpu
def test_append_of_nodes_without_a_place():
    # a tree that is none, one before its sequence, one whose deepest positions the tables do not hold, one without a page
    trees = [[-1, 7], [-1, 0, 1], chain(4) + [0], [-1, 0]]
    s = Trees(trees, [20, 5, 6, 40], 2, 2, 32, 16, seed=5)
    s.lengths[1] = 2
    s.table[3, 2] = -1
    inputs = _append_inputs(s, 2, 2, 32, positions=8)
    kept = s.keys.copy(), s.values.copy()
    q, keys, values, status = _append(s, trees, inputs)
    assert status == 2
    done = [5, 6, 9]                                   # of the third tree, at positions 6, 7 and (its last node) 7
    assert (q[[r for r in range(12) if r not in done]] == 0).all() and (q[done] != 0).any(axis=(1, 2)).all()
    for i in (0, 1, 4):
        place = s.place(2, 6 + i)
        kept[0][place], kept[1][place] = keys[place], values[place]
    np.testing.assert_array_equal(keys, kept[0])
    np.testing.assert_array_equal(values, kept[1])


# ------------------------------------------------------------------ accept
def walk(parents, drafted, choices, levels=256):
    path = [0]
    while True:
        choice = choices[path[-1]]
        fits = [i for i, p in enumerate(parents) if p == path[-1] and drafted[i] == choice]
        if not fits or len(path) >= levels:
            return path, choice
        path.append(fits[0])


def _cache_of(trees, bases, layers=3, kv=2, d=32, page=16, seed=0):
    rng = np.random.default_rng(seed)
    lengths = [b + len(t) for b, t in zip(bases, trees)]
    need = [-(-n // page) for n in lengths]
    table = np.full((len(trees), max(need) + 1), -1, dtype=np.int32)
    order = rng.permutation(sum(need) + 2)
    at = 0
    for r, n in enumerate(need):
        table[r, :n] = order[at:at + n]
        at += n
    shape = layers, sum(need) + 2, kv, page, d
    keys, values = (rng.standard_normal(shape).astype(np.float16) for _ in range(2))
    return table, lengths, keys, values


def _expect_accept(trees, bases, table, keys, values, drafted, choices, levels=256):
    keys, values = keys.copy(), values.copy()
    page = keys.shape[3]
    kept, path, after = [], [], []
    at = 0
    for b, tree in enumerate(trees):
        n = len(tree)
        if n == 0:
            kept.append(-1)
            after.append(-1)
            continue
        p, choice = walk(tree, drafted[at:at + n], choices[at:at + n], levels)
        kept.append(bases[b] + len(p))
        after.append(choice)
        path += p + [-1] * (n - len(p))
        for pool in (keys, values):
            rows = [pool[:, table[b, (bases[b] + v) // page], :, (bases[b] + v) % page].copy() for v in p]
            for i, row in enumerate(rows):
                pool[:, table[b, (bases[b] + i) // page], :, (bases[b] + i) % page] = row
        at += n
    return keys, values, kept, path, after


def _check_accept(trees, bases, drafted, choices, levels=256, vocab=0, **shape):
    """Once with the choices, and with `vocab` by logits whose argmax they are."""
    from harsh4b_amd.tree import pages_accept
    table, lengths, keys, values = _cache_of(trees, bases, **shape)
    ek, ev, kept, path, after = _expect_accept(trees, bases, table, keys, values, drafted, choices, levels)
    for by in ("choices", "logits") if vocab else ("choices",):
        status = ints([0])
        t, dk, dv, dl, dt = plan(trees, status), up(keys), up(values), ints(lengths), ints(table)
        how = dict(choices=ints(choices))
        if by == "logits":
            logits = torch.randn((len(choices), vocab), device="cuda")
            logits[torch.arange(len(choices), device="cuda"), ints(choices).long()] = 9.0
            how = dict(logits=logits)
        gk, gp, ga = pages_accept(dk, dv, dt, dl, status, t, ints(drafted), levels=levels, **how)
        assert gk.tolist() == kept and gp.tolist() == path and ga.tolist() == after, by
        np.testing.assert_array_equal(dk.cpu().numpy(), ek)
        np.testing.assert_array_equal(dv.cpu().numpy(), ev)
        assert dl.tolist() == lengths and dt.tolist() == table.tolist() and int(status.item()) == 0


def some_choices(seed, trees, few=3):
    """Drafted tokens and choices from few values, so that paths are long and siblings alike."""
    rng = np.random.default_rng(seed)
    n = sum(len(t) for t in trees)
    return rng.integers(0, few, n).tolist(), rng.integers(0, few, n).tolist()


@gpu
@pytest.mark.parametrize("d", [16, 32, 64, 128])
@pytest.mark.parametrize("few", [1, 2, 5])
def test_accept(d, few):
    trees = some_trees(few, [1, 0, 5, 40, 17, 64, 65, 200, 256], deep=30) + [chain(70), star(12)]
    drafted, choices = some_choices(d + few, trees, few)
    _check_accept(trees, [0, 9, 30, 100, 15, 64, 3, 1, 0, 17, 5], drafted, choices, vocab=300, d=d, seed=d)


@gpu
@pytest.mark.parametrize("levels", [1, 2, 3, 7, 256])
def test_accept_of_so_many_levels(levels):
    trees = [chain(9), chain(200), [-1], random_tree(np.random.default_rng(1), 60, 12)]
    drafted, choices = some_choices(levels, trees, 1)
    _check_accept(trees, [5, 7, 0, 30], drafted, choices, levels, vocab=77)


@gpu
def test_accept_moves_rows_over_each_other():
    # every second node of a chain of pairs: sources and targets overlap all along
    n = 255
    parents = [-1]
    for i in range(1, n):
        parents.append(0 if i <= 2 else (i - 1) // 2 * 2)
    drafted = [i % 2 for i in range(n)]               # the path takes the even ones: 2, 4, ..
    for d in (16, 32, 64, 128):
        _check_accept([parents, parents], [3, 64], drafted * 2, [0] * (2 * n), kv=1, d=d, layers=2)


@gpu
@pytest.mark.parametrize("vocab,tokens,levels", [(1, 30, 256), (2, 30, 256), (63, 30, 256), (1000, 30, 256), (1001, 1200, 256),
                                                 (151936, 30, 256), (20001, 1200, 5), (50002, 600, 3), (151936, 240, 4)])
def test_accept_by_logits(vocab, tokens, levels):
    # few levels of many rows are read level by level, the others all at once: ties, NaN and infinities as np.argmax
    from harsh4b_amd.tree import pages_accept
    rng = np.random.default_rng(vocab)
    trees = some_trees(vocab, [60] * (tokens // 60) or [8, 0, 21, 1], deep=9)
    n = sum(len(t) for t in trees)
    logits = np.round(rng.standard_normal((n, vocab))).astype(np.float32)
    for r in range(0, n, 5):
        logits[r, rng.integers(0, vocab, 2)] = np.nan
    logits[1::7] = -np.inf
    logits[2::7, -1] = np.inf
    logits[3::7] = 0.0
    choices = logits.argmax(axis=1)
    drafted = np.where(rng.random(n) < 0.8, 0, rng.integers(0, vocab, n))
    at = 0
    for t in trees:                                   # (children often hold what their parent chooses)
        for i, p in enumerate(t):
            if p >= 0 and rng.random() < 0.7:
                drafted[at + i] = choices[at + p]
        at += len(t)
    bases = [int(b) for b in rng.integers(0, 20, len(trees))]
    table, lengths, keys, values = _cache_of(trees, bases, layers=1, kv=1, d=16)
    ek, ev, kept, path, after = _expect_accept(trees, bases, table, keys, values, drafted.tolist(), choices.tolist(), levels)
    status, dk, dv = ints([0]), up(keys), up(values)
    got = pages_accept(dk, dv, ints(table), ints(lengths), status, plan(trees), ints(drafted), logits=up(logits), levels=levels)
    assert [g.tolist() for g in got] == [kept, path, after]
    np.testing.assert_array_equal(dk.cpu().numpy(), ek)


@gpu
def test_accept_refuses():
    from harsh4b_amd.tree import pages_accept
    trees = [[-1, 0, 0], [-1, 5, 0], [-1, 0, 1], [-1, 0, 0]]
    bases = [14, 4, 20, 2]
    table, lengths, keys, values = _cache_of(trees, bases, d=64)
    lengths[3] = 1                                     # a base before the sequence
    table[2, 1] = -1                                   # the path's page is gone
    drafted, choices = [9, 1, 2] * 4, [2, 0, 0] + [2, 0, 0] + [1, 2, 7] + [2, 0, 0]
    drafted[7], drafted[8] = 1, 2
    for held in (0, 1, 4):
        status, dk, dv = ints([held]), up(keys), up(values)
        t = plan(trees, ints([0]))
        out = ints([50] * 4), ints([50] * 12), ints([50] * 4)
        got = pages_accept(dk, dv, ints(table), ints(lengths), status, t, ints(drafted), choices=ints(choices), out=out)
        assert got[0] is out[0]
        if held:
            assert [g.tolist() for g in got] == [[-1] * 4, [-1] * 12, [-1] * 4]
            np.testing.assert_array_equal(dk.cpu().numpy(), keys)
            continue
        assert [g.tolist() for g in got] == [[16, -1, 23, -1], [0, 2, -1] + [-1] * 3 + [0, 1, 2] + [-1] * 3, [0, -1, 7, -1]]
        assert int(status.item()) == 2
        expect = keys.copy()
        expect[:, table[0, 0], :, 15] = keys[:, table[0, 1], :, 0]
        np.testing.assert_array_equal(dk.cpu().numpy(), expect)
    # a move from a page that is gone stays undone and is reported
    trees, bases = [[-1, 0, 0]], [15]
    table, lengths, keys, values = _cache_of(trees, bases)
    table[0, 1] = -1
    status, dk = ints([0]), up(keys)
    got = pages_accept(dk, up(values), ints(table), ints(lengths), status, plan(trees), ints([0, 1, 2]), choices=ints([2, 0, 0]))
    assert [g.tolist() for g in got] == [[17], [0, 2, -1], [0]] and int(status.item()) == 2
    np.testing.assert_array_equal(dk.cpu().numpy(), keys)


@gpu
def test_accept_of_starts_outside_the_batch_and_of_nothing():
    from harsh4b_amd.tree import DraftTree, pages_accept, tree_plan
    table, lengths, keys, values = _cache_of([[-1, 0], [-1, 0, 0]], [3, 4])
    for starts, expect in (([0, 2, 1], [[5, -1], [0, 1, 9, 9, 9]]), ([0, 9, 10], [[-1, -1], [9] * 5]),
                           ([-3, 2, 5], [[-1, 6], [9, 9, 0, 1, -1]]), ([1, 3, 3], [[5, -1], [9, 0, 1, 9, 9]])):
        status = ints([0])
        parents, drafted = ints([-1, 0, 0, 0, 0]), ints([4] * 5)
        parents = ints([-1, -1, -1, 0, 0]) if starts == [-3, 2, 5] else ints([-1, 0, 0, 0, 0])
        if starts == [1, 3, 3]:
            parents = ints([5, -1, 0, 5, 5])
        t = tree_plan(parents, ints(starts), ints([0]))
        out = ints([9, 9]), ints([9] * 5), ints([9, 9])
        pages_accept(up(keys), up(values), ints(table), ints(lengths), status, t, drafted, choices=drafted, out=out)
        assert [out[0].tolist(), out[1].tolist()] == expect, starts
    none = DraftTree(ints([]), ints([0, 0, 0]), ints([]), ints(np.zeros((0, 8))))
    status = ints([0])
    for how in (dict(choices=ints([])), dict(logits=torch.zeros((0, 50), device="cuda"))):
        got = pages_accept(up(keys), up(values), ints(table), ints(lengths), status, none, ints([]), **how)
        assert [g.tolist() for g in got] == [[-1, -1], [], [-1, -1]] and int(status.item()) == 0


@gpu
def test_accept_of_many_sequences():
    rng = np.random.default_rng(3)
    sizes = rng.integers(0, 6, 70000).tolist()
    trees = [chain(n) for n in sizes]
    drafted, choices = some_choices(3, trees, 2)
    _check_accept(trees, [int(b) for b in rng.integers(0, 3, 70000)], drafted, choices, layers=1, kv=1, d=16)


# ------------------------------------------------------------------ together
def _model():
    from harsh4b_amd.synthetic import random_model
    config = dict(hidden_size=512, intermediate_size=1024, num_attention_heads=8, num_key_value_heads=2, head_dim=128,
                  num_hidden_layers=3, vocab_size=2000, rms_norm_eps=1e-6, rope_theta=1000000, max_position_embeddings=512,
                  tie_word_embeddings=True)
    return random_model(config, seed=5)


class Server:
    """A model's step over drafted trees, made of the public operators."""

    def __init__(self, model, sequences):
        from harsh4b_amd.lightspark import LiteSparkProjection
        from harsh4b_amd.paged import PagedCache
        self.m, c = model, model.config
        self.kv, self.heads = int(c["num_key_value_heads"]), int(c["num_attention_heads"])
        self.cache = PagedCache(len(model.layers), 60, self.kv, 128, sequences=sequences, max_pages=12, page_size=16)
        self.lm = LiteSparkProjection(model.embedding, model.embedding_scales)
        packed = model.embedding.to(torch.int16)
        table = torch.stack((packed & 15, packed >> 4), dim=-1).view(packed.shape[0], -1)
        self.embedding = torch.where(table > 7, table - 16, table).float() * model.embedding_scales[:, None]
        self.cos, self.sin = up(model.rope_cos_host), up(model.rope_sin_host)
        self.eps = float(c["rms_norm_eps"])

    def forward(self, tree, tokens):
        from harsh4b_amd.lightspark import add_rmsnorm_quant, int4_i8_gemm, quant_int4_gemm
        x = self.embedding[tokens.long()].contiguous()
        delta = None
        for i, layer in enumerate(self.m.layers):
            q, s = add_rmsnorm_quant(x, layer.input_norm, self.eps, delta=delta)
            query = self.cache.append_tree(i, int4_i8_gemm(q, s, layer.qkv), layer.q_norm, layer.k_norm, self.cos, self.sin,
                                           self.eps, tree)
            a = self.cache.attend_tree(i, query, tree)
            delta = quant_int4_gemm(a.view(x.shape[0], -1), layer.o)
            q, s = add_rmsnorm_quant(x, layer.post_norm, self.eps, delta=delta)
            gate, upper = int4_i8_gemm(q, s, layer.gate_up).chunk(2, dim=-1)
            delta = quant_int4_gemm((torch.nn.functional.silu(gate) * upper).contiguous(), layer.down)
        q, s = add_rmsnorm_quant(x, self.m.final_norm, self.eps, delta=delta)
        return int4_i8_gemm(q, s, self.lm)


@gpu
def test_drafted_steps_give_the_greedy_tokens():
    """Prompts as chains, then steps over drafted trees that hold the model's own
    next tokens, wrong ones, or some: the tokens are the greedy decode's."""
    model = _model()
    rng = np.random.default_rng(8)
    prompts = [rng.integers(0, 2000, n).tolist() for n in (5, 30, 64)]
    steps = 24
    greedy, logits_of = [], []
    for prompt in prompts:
        state = model.new_state(256)
        rows, tokens = [], list(prompt)
        for i in range(len(prompt) + steps):
            logits = model.forward_token(tokens[i], state).cpu().numpy()
            rows.append(logits)
            if i + 1 >= len(prompt):
                tokens.append(int(logits.argmax()))
        greedy.append(tokens)
        logits_of.append(rows)
    server = Server(model, 3)
    # the prompts, but for their last tokens, as chains
    trees = [chain(len(p) - 1) for p in prompts]
    server.cache.resize([len(t) for t in trees])
    tree = server.cache.plan_tree(np.concatenate(trees).tolist(), starts_of(trees).tolist())
    server.forward(tree, ints(np.concatenate([p[:-1] for p in prompts])))
    done = [len(p) - 1 for p in prompts]              # positions in the cache
    # One activation that a rounding tips over to the next int8 step moves every value of the next rows, and some of
    # those tip too: in the end the two runs' steps fall independently of each other.  A step is 1/127 of a row's
    # largest value, which is 3.6 deviations off for rows of 512 to 1024: 0.028 deviations, its error's deviation
    # 0.028 / sqrt(12), of two runs' difference sqrt(2) times that, 0.0115, in each of 13 products (4 a layer and
    # the last) relative to its output: 0.0115 sqrt(13) = 0.041 of the logits' deviation, and five times that for the
    # largest of 2000 logits and 40 rows.  Choices whose lead is less than twice that are not compared with the greedy ones.
    slack = 5 * 0.041 * float(np.std(logits_of[0][0]))
    for step in range(9):
        trees, drafted = [], []
        for b, tokens in enumerate(greedy):
            right = tokens[done[b]:done[b] + 1 + int(rng.integers(0, 4))]
            parents, ids, at = [-1], [right[0]], 0
            for token in right[1:]:
                parents += [at, at]                    # a wrong child before the right one
                ids += [(token + 1) % 2000, token]
                at = len(ids) - 1
            trees.append(parents + [at])
            drafted.append(ids + [int(rng.integers(0, 2000))])
        server.cache.resize([n + len(t) for n, t in zip(done, trees)])
        tree = server.cache.plan_tree(np.concatenate(trees).tolist(), starts_of(trees).tolist())
        ids = np.concatenate(drafted)
        logits = server.forward(tree, ints(ids))
        kept, path, after = server.cache.accept(tree, ids.tolist(), logits=logits, levels=6)
        kept, path, after, rows = kept.tolist(), path.tolist(), after.tolist(), logits.cpu().numpy()
        at = 0
        for b, t in enumerate(trees):
            mine = [v for v in path[at:at + len(t)] if v >= 0]
            expect, choice = walk(t, drafted[b], rows[at:at + len(t)].argmax(axis=1).tolist(), 6)
            assert mine == expect and after[b] == choice
            assert kept[b] == done[b] + len(mine)
            for i, v in enumerate(mine):
                ref = logits_of[b][done[b] + i]
                assert np.abs(rows[at + v] - ref).max() <= slack, (step, b, i)
                lead = np.partition(ref, -2)
                nxt = drafted[b][mine[i + 1]] if i + 1 < len(mine) else after[b]
                if lead[-1] - lead[-2] > 2 * slack:
                    assert nxt == greedy[b][done[b] + i + 1], (step, b, i)
            at += len(t)
            if kept[b] + 5 > len(greedy[b]) - 1:
                kept[b] = done[b]                      # (near the end: the same step again)
        server.cache.resize(kept)
        done = kept
        server.cache.check_status()
    assert all(n > len(p) + 8 for n, p in zip(done, prompts)), done


@gpu
def test_captured_steps():
    """A step of all operators as two graphs of one cache, replayed in turn with
    other trees and eager work between, against an eager twin."""
    from harsh4b_amd.paged import PagedCache
    from harsh4b_amd.tree import pages_accept, paged_append_tree, paged_attention_tree, tree_plan
    from harsh4b_amd.lightspark import add_rmsnorm_quant
    kv, groups, d, rows, n = 2, 4, 128, 3, 12
    rng = np.random.default_rng(31)

    def fresh():
        c = PagedCache(2, 60, kv, d, sequences=rows, max_pages=20, page_size=16)
        c.resize([14, 700 // 16, 1])
        c.keys.copy_(up(np.random.default_rng(1).standard_normal(c.keys.shape).astype(np.float16)))
        c.values.copy_(up(np.random.default_rng(2).standard_normal(c.values.shape).astype(np.float16)))
        return c

    cos = torch.rand((400, d // 2), device="cuda")
    norm = torch.ones(d, device="cuda")
    width = (groups + 2) * kv * d
    qkv, delta = torch.zeros((n, width), device="cuda"), torch.zeros((n, width), device="cuda")
    gamma = torch.ones(width, device="cuda")
    parents, starts, drafted = ints([-1] * n), ints([0, 4, 8, 12]), ints([0] * n)
    logits = torch.zeros((n, 500), device="cuda")

    def step(c):
        c.resize(c.lengths + (starts[1:] - starts[:-1]))
        tree = tree_plan(parents, starts, c.status)
        summed = torch.empty_like(qkv)
        q, s = add_rmsnorm_quant(qkv, gamma, 1e-6, delta=delta, out=summed)
        outs = [q, s, summed]
        for layer in range(2):
            query = c.append_tree(layer, summed, norm, norm, cos, cos, 1e-6, tree)
            outs += [query, c.attend_tree(layer, query, tree), c.attend_tree(layer, query, tree, window=9, sinks=2)]
        outs += list(pages_accept(c.keys, c.values, c.table, c.lengths, c.status, tree, drafted, logits=logits, levels=4))
        c.resize(outs[-3])
        return outs

    eager, replayed = fresh(), fresh()
    step(fresh())
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs = step(replayed)
        graphs.append((g, outs))
    for i in range(10):
        qkv.copy_(up(rng.standard_normal((n, width)).astype(np.float32)))
        delta.copy_(up(rng.standard_normal((n, width)).astype(np.float32)))
        sizes = [[4, 4, 4], [1, 6, 5], [0, 11, 1]][i % 3]
        starts.copy_(ints(np.concatenate([[0], np.cumsum(sizes)])))
        parents.copy_(ints(np.concatenate([random_tree(rng, k) for k in sizes if k])))
        drafted.copy_(ints(rng.integers(0, 3, n)))
        logits.zero_()
        logits[torch.arange(n, device="cuda"), up(rng.integers(0, 3, n))] = 1.0
        expect = step(eager)
        g, outs = graphs[i % 2]
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, expect):
            assert torch.equal(a, b), i
        for name in ("table", "lengths", "refs", "status", "keys", "values"):
            assert torch.equal(getattr(eager, name), getattr(replayed, name)), (i, name)
    assert int(eager.status.item()) == 0


@gpu
def test_calls_on_other_streams():
    # each call on a stream of its own, which waits for the caller's
    from harsh4b_amd.lightspark import add_rmsnorm_quant
    from harsh4b_amd.tree import pages_accept, paged_append_tree
    trees = some_trees(4, [9, 30, 2])
    s = Trees(trees, [20, 33, 7], 2, 4, 64, 16, seed=4)
    inputs = _append_inputs(s, 2, 4, 64)
    expect = _append(s, trees, inputs)
    stream = torch.cuda.Stream()
    got = _append(s, trees, inputs, stream=stream)
    for a, b in zip(got, expect):
        np.testing.assert_array_equal(a, b)
    t = plan(trees, stream=stream)
    torch.cuda.synchronize()
    assert torch.equal(t.ancestors, plan(trees).ancestors)
    table, lengths, keys, values = _cache_of(trees, [20, 33, 7])
    drafted, choices = some_choices(5, trees)
    ek, _, kept, path, after = _expect_accept(trees, [20, 33, 7], table, keys, values, drafted, choices)
    dk = up(keys)
    out = pages_accept(dk, up(values), ints(table), ints(lengths), ints([0]), t, ints(drafted), choices=ints(choices), stream=stream)
    torch.cuda.synchronize()
    assert [o.tolist() for o in out] == [kept, path, after]
    np.testing.assert_array_equal(dk.cpu().numpy(), ek)
    x, gamma = up(np.ones((9, 300), np.float32)), up(np.ones(300, np.float32))
    q, scale = add_rmsnorm_quant(x, gamma, 1e-6, stream=stream)
    torch.cuda.synchronize()
    assert (q == 127).all() and torch.equal(scale, add_rmsnorm_quant(x, gamma, 1e-6)[1])


# ------------------------------------------------------------------ every kind of tile, join and path
def crowd(trees, bases, others=140):
    """With many sequences of one node beside them: no tiles of 16 rows for few."""
    return trees + [[-1]] * others, bases + [2] * others


@gpu
@pytest.mark.parametrize("groups,d", [(4, 128), (8, 64), (3, 128), (5, 32), (4, 16)])
@pytest.mark.parametrize("rows", [16, 17, 24, 31, 32, 33, 64, 65, 128, 129])
def test_tiles_of_so_many_rows(groups, d, rows):
    n = max(1, rows // groups)
    trees, bases = crowd(some_trees(rows, [n, n + 1]), [77, 600])
    Trees(trees, bases, 2, groups, d, 16, seed=rows).check()


@gpu
@pytest.mark.parametrize("groups,d", [(4, 128), (2, 128), (4, 64), (8, 64), (8, 32)])
def test_joins_of_many_rows(groups, d):
    # more than 2048 rows to join, of tiles in several pieces and of tiles in one
    rng = np.random.default_rng(d)
    sizes = [int(n) for n in rng.integers(9, 17, 24)]
    s = Trees(some_trees(d, sizes), [int(b) for b in rng.integers(300, 1500, 24)], 8, groups, d, 64, seed=d)
    assert s.tokens * 8 >= 2048
    s._check()
    s._check(window=700, sinks=3)


@gpu
@pytest.mark.parametrize("what", ["nan", "inf", "-inf"])
@pytest.mark.parametrize("n", [7, 40])
def test_queries_that_are_not_finite(what, n):
    # a row's value makes its own result NaN and no other
    trees, bases = crowd(some_trees(n, [n, n]), [90, 700])
    s = Trees(trees, bases, page=16, seed=41)
    expect, bound = _reference(s, trees, 0, 0)
    bad = ((0, 1, 7), (2, 5, 127), (n + 1, 0, 0), (2 * n - 1, 7, 64), (2 * n + 5, 3, 1))
    for t, h, i in bad:
        s.query[t, h, i] = float(what)
    got = s.attend()
    lost = np.isnan(got).any(axis=-1)
    assert sorted(map(tuple, np.argwhere(lost))) == sorted((t, h) for t, h, _ in bad)
    off = np.where(lost[..., None], 0.0, np.abs(got - expect)).reshape(s.tokens, -1).max(axis=1)
    assert (off <= bound).all()


@gpu
@pytest.mark.parametrize("scale", [1e-30, 1e-3, 300.0, 1e6, 1e36])
def test_queries_of_any_size(scale):
    for trees, bases in (crowd(some_trees(1, [7, 40]), [100, 90]), (some_trees(1, [7, 40]), [100, 90])):
        s = Trees(trees, bases, page=16, seed=9)
        s.query *= np.float32(scale)
        s.check()


@gpu
def test_large_and_small_values():
    trees, bases = crowd(some_trees(2, [8, 30, 100]), [100, 90, 300])
    s = Trees(trees, bases, page=16, seed=10)
    s.values[:] = np.where(np.isnan(s.values), s.values, s.values * np.float16(12000))
    s.keys[:, :, ::2] *= np.float16(2.0 ** -14)           # subnormal keys
    s.check()


@gpu
def test_offsets_past_32_bits():
    # pools of more than 2^32 bytes and 2^31 elements: the pages in use lie at their end
    from harsh4b_amd.tree import pages_accept, paged_append_tree, paged_attention_tree
    trees = [chain(1), random_tree(np.random.default_rng(1), 20)]
    s = Trees(trees, [49, 20], kv=8, groups=1, d=128, page=256, seed=15, spare=0)
    pages = (1 << 31) // (8 * 256 * 128) + 8
    keys = torch.zeros((1, pages, 8, 256, 128), dtype=torch.float16, device="cuda")
    values = torch.zeros_like(keys)
    n = s.keys.shape[0]
    keys[0, -n:], values[0, -n:] = up(s.keys), up(s.values)
    d, t = s.device(), plan(trees)
    table = torch.where(d["table"] >= 0, d["table"] + (pages - n), d["table"])
    got = paged_attention_tree(d["query"], keys[0], values[0], table, d["lengths"], t)
    np.testing.assert_array_equal(got.cpu().numpy(), s.check())
    inputs = [up(a) for a in _append_inputs(s, 8, 1, 128)]
    status = ints([0])
    paged_append_tree(*inputs, 1e-6, keys[0], values[0], table, d["lengths"], status, t)
    paged_append_tree(*inputs, 1e-6, d["keys"], d["values"], d["table"], d["lengths"], status, t)
    assert torch.equal(keys[0, -n:].nan_to_num(5.0), d["keys"].nan_to_num(5.0)) and int(status.item()) == 0
    choices = ints([1] * 21)
    drafted = ints([0] + [1] * 20)
    for pools, book in (((keys, values), table), ((d["keys"][None], d["values"][None]), d["table"])):
        pages_accept(*pools, book, d["lengths"], status, t, drafted, choices=choices)
    assert torch.equal(keys[0, -n:].nan_to_num(5.0), d["keys"].nan_to_num(5.0)) and int(status.item()) == 0
    assert not keys[0, :-n].any()


@gpu
@pytest.mark.parametrize("sequences", [2, 300])
def test_captured_batches_that_are_cut(sequences):
    """Tiles in pieces and their joins, with the plan in every wave and in a
    launch of its own: two graphs, replayed in turn with eager work between."""
    from harsh4b_amd.tree import paged_attention_tree
    scenes = []
    for seed, sizes, bases in ((61, [8, 60], [900, 1111]), (62, [100, 3], [1300, 700])):
        spare = sequences - 2
        s = Trees(some_trees(seed, sizes) + [[-1, 0]] * spare, bases + [30] * spare, 8, 4, 128, 64, seed=seed)
        d, t = s.device(), plan(s.trees)
        scenes.append((d, t, paged_attention_tree(**d, tree=t).clone()))
    torch.cuda.synchronize()
    graphs = []
    for d, t, _ in scenes:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = paged_attention_tree(**d, tree=t)
        graphs.append((g, out))
    for i in range(6):
        (g, out), (d, t, expect) = graphs[i % 2], scenes[i % 2]
        out.fill_(7.0)
        g.replay()
        other = scenes[1 - i % 2]
        assert torch.equal(paged_attention_tree(**other[0], tree=other[1]), other[2]), i
        torch.cuda.synchronize()
        assert torch.equal(out, expect), i


@gpu
def test_captured_greedy_paths():
    # chains of a large vocabulary, replayed on other logits and drafts with eager work between
    from harsh4b_amd.tree import pages_accept
    rng = np.random.default_rng(6)
    trees = some_trees(6, [9, 16, 1, 30], deep=6)
    table, lengths, keys, values = _cache_of(trees, [5, 30, 0, 17])
    n, vocab = sum(len(t) for t in trees), 60001
    eager, replayed = ([up(keys), up(values)] for _ in range(2))
    t, book, size, status = plan(trees), ints(table), ints(lengths), ints([0])
    logits, drafted = torch.zeros((n, vocab), device="cuda"), ints([0] * n)
    call = lambda pools: pages_accept(*pools, book, size, status, t, drafted, logits=logits, levels=7)
    call([up(keys), up(values)])
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        outs = call(replayed)
    for i in range(6):
        logits.copy_(torch.randn_like(logits))
        choices = rng.integers(0, vocab, n)
        logits[torch.arange(n, device="cuda"), up(choices)] = 30.0
        ids, at = rng.integers(0, vocab, n), 0
        for tree in trees:
            for k, p in enumerate(tree):
                if p >= 0 and rng.random() < 0.7:
                    ids[at + k] = choices[at + p]
            at += len(tree)
        drafted.copy_(ints(ids))
        expect = call(eager)
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, expect)), i
        assert torch.equal(eager[0], replayed[0]) and torch.equal(eager[1], replayed[1]), i
        at = 0
        for b, tree in enumerate(trees):
            path, choice = walk(tree, ids[at:at + len(tree)].tolist(), choices[at:at + len(tree)].tolist(), 7)
            assert expect[1][at:at + len(path)].tolist() == path and int(expect[2][b]) == choice
            at += len(tree)


@gpu
def test_drafted_tokens_outside_the_vocabulary():
    # they are nobody's choice; given choices are any numbers
    from harsh4b_amd.tree import pages_accept
    trees = [[-1, 0, 0, 0], [-1, 0]]
    table, lengths, keys, values = _cache_of(trees, [3, 4])
    drafted = ints([0, -1, 50, 2**31 - 1, 0, -2**31])
    logits = torch.zeros((6, 50), device="cuda")
    logits[:, 49] = 1.0
    got = pages_accept(up(keys), up(values), ints(table), ints(lengths), ints([0]), plan(trees), drafted, logits=logits)
    assert [g.tolist() for g in got] == [[4, 5], [0, -1, -1, -1, 0, -1], [49, 49]]
    got = pages_accept(up(keys), up(values), ints(table), ints(lengths), ints([0]), plan(trees), drafted,
                       choices=ints([2**31 - 1, 7, 7, -5, -2**31, 9]))
    assert [g.tolist() for g in got] == [[5, 6], [0, 3, -1, -1, 0, 1], [-5, 9]]


@gpu
def test_trees_that_were_not_planned():
    # depths and ancestors of any contents: no access out of range, and rows of other sequences have their results
    from harsh4b_amd.tree import paged_append_tree, paged_attention_tree
    trees = some_trees(9, [9, 70, 12])
    s = Trees(trees, [40, 300, 7], 2, 4, 64, 16, seed=9)
    d, t = s.device(), plan(trees)
    expect = s.check()
    rng = np.random.default_rng(2)
    inputs = [up(a) for a in _append_inputs(s, 2, 4, 64)]
    for _ in range(3):
        depths, ancestors = t.depths.clone(), t.ancestors.clone()
        depths[9:79] = ints(rng.integers(-2**31, 2**31, 70))
        ancestors[9:79] = ints(rng.integers(-2**31, 2**31, (70, 8)))
        for window in (0, 5):
            out = paged_attention_tree(**d, tree=t._replace(depths=depths, ancestors=ancestors), window=window)
        out = paged_attention_tree(**d, tree=t._replace(depths=depths, ancestors=ancestors))
        keep = [*range(9), *range(79, 91)]
        np.testing.assert_array_equal(out.cpu().numpy()[keep], expect[keep])
        status = ints([0])
        paged_append_tree(*inputs, 1e-6, d["keys"].clone(), d["values"].clone(), d["table"], d["lengths"], status,
                          t._replace(depths=depths))
        assert int(status.item()) == 2


@gpu
@pytest.mark.parametrize("kv,groups", [(2, 4), (1, 8)])
def test_few_trees_among_many_sequences(kv, groups):
    # the plan in a launch of its own, with tiles of 16 rows
    trees = [[] for _ in range(300)]
    for b, n in ((3, 5), (77, 20), (299, 9)):
        trees[b] = random_tree(np.random.default_rng(b), n)
    Trees(trees, [int(b) for b in np.random.default_rng(1).integers(0, 90, 300)], kv, groups, 32, 16, seed=2).check()


@gpu
@pytest.mark.parametrize("held", [1, 4])
def test_append_while_the_cache_refuses(held):
    # the queries as ever, no K and V
    from harsh4b_amd.tree import paged_append_tree
    trees = some_trees(3, [5, 9])
    s = Trees(trees, [20, 33], 2, 4, 64, 16, seed=3)
    inputs = _append_inputs(s, 2, 4, 64)
    expect, _, _, _ = _append(s, trees, inputs)
    d, status = s.device(), ints([held])
    q = paged_append_tree(*[up(a) for a in inputs], 1e-6, d["keys"], d["values"], d["table"], d["lengths"], status, plan(trees))
    np.testing.assert_array_equal(q.cpu().numpy(), expect)
    np.testing.assert_array_equal(d["keys"].cpu().numpy(), s.keys)
    np.testing.assert_array_equal(d["values"].cpu().numpy(), s.values)
    assert int(status.item()) == held


@gpu
@pytest.mark.parametrize("window,sinks", [(0, 0), (40, 5)])
def test_a_server_s_trees(window, sinks):
    """Steps of sequences that come, grow by accepted paths across page borders,
    pause and end, against a list of each one's rows; growth straight from one
    tree to the next, or under a window through the kept length."""
    from harsh4b_amd.paged import PagedCache
    kv, groups, d, rows = 2, 4, 32, 5
    rng = np.random.default_rng(window + 1)
    c = PagedCache(2, 90, kv, d, sequences=rows, max_pages=20, page_size=16)
    c.keys.fill_(float("nan"))
    c.values.fill_(float("nan"))
    angle = np.arange(320)[:, None] * 10000.0 ** (-np.arange(0, d, 2) / d)
    cos, sin = up(np.cos(angle).astype(np.float32)), up(np.sin(angle).astype(np.float32))
    norm = torch.ones(d, device="cuda")
    kept_rows = [[] for _ in range(rows)]             # of each sequence: [(keys, values) of both layers, ..] by position
    kept = [0] * rows
    for step in range(30):
        for b in range(rows):
            if kept[b] > 200 or (kept[b] and rng.random() < 0.05):
                kept[b], kept_rows[b] = 0, []
        sizes = [int(n) if rng.random() < 0.8 else 0 for n in rng.integers(1, 24, rows)]
        trees = [random_tree(rng, n, 6) if n else [] for n in sizes]
        bases = list(kept)
        if window:
            c.resize(kept, window, sinks)
        c.resize([k + n for k, n in zip(kept, sizes)], window, sinks)
        tree = c.plan_tree(np.concatenate([t for t in trees if t] or [[]]).astype(int).tolist(), starts_of(trees).tolist())
        tokens = sum(sizes)
        if tokens == 0:
            continue
        queries = []
        for layer in range(2):
            qkv = up((2 * rng.standard_normal((tokens, (kv * groups + 2 * kv) * d))).astype(np.float32))
            queries.append(c.append_tree(layer, qkv, norm, norm, cos, sin, 1e-6, tree))
        table, keys, values = c.table.cpu().numpy(), c.keys.cpu().numpy(), c.values.cpu().numpy()
        lengths = c.lengths.tolist()
        assert lengths == [k + n for k, n in zip(kept, sizes)]
        for b in range(rows):
            low = max(0, bases[b] - window + 1) if window else 0
            for j in range(lengths[b]):
                if sinks <= j < low:
                    continue
                page = table[b, j // 16]
                assert page >= 0, (step, b, j)
                here = keys[:, page, :, j % 16], values[:, page, :, j % 16]
                if j < bases[b]:
                    np.testing.assert_array_equal(here[0], kept_rows[b][j][0])
                    np.testing.assert_array_equal(here[1], kept_rows[b][j][1])
        for layer in range(2):
            out = c.attend_tree(layer, queries[layer], tree, window, sinks).cpu().numpy()
            s = Scene.__new__(Scene)
            s.keys, s.values, s.table, s.lengths = keys[layer], values[layer], table, lengths
            s.query, s.starts, s.tokens = queries[layer].cpu().numpy(), starts_of(trees), tokens
            expect, bound = _reference(s, trees, window, sinks)
            off = np.abs(out - expect).reshape(tokens, -1).max(axis=1)
            assert (off <= bound).all(), (step, layer, off.max())
        drafted, choices = some_choices(step, trees, 2)
        got, path, after = c.accept(tree, drafted, choices=choices, levels=7)
        got, path, after, at = got.tolist(), path.tolist(), after.tolist(), 0
        for b, t in enumerate(trees):
            if not t:
                assert got[b] == -1 and after[b] == -1
                continue
            p, choice = walk(t, drafted[at:at + len(t)], choices[at:at + len(t)], 7)
            assert path[at:at + len(t)] == p + [-1] * (len(t) - len(p)) and after[b] == choice
            for v in p:
                j = bases[b] + v
                page = table[b, j // 16]
                kept_rows[b].append((keys[:, page, :, j % 16].copy(), values[:, page, :, j % 16].copy()))
            kept[b] = bases[b] + len(p)
            assert got[b] == kept[b] == len(kept_rows[b])
            at += len(t)
        c.check_status()
    assert max(kept) > 30


@gpu
@pytest.mark.parametrize("base", [0, 5, 16, 27, 31])
def test_forks_between_trees(base):
    """A path kept, its sequence forked at its end, and other trees in both: they
    share what was kept, and neither's nodes or moves reach the other."""
    from harsh4b_amd.paged import PagedCache
    kv, groups, d = 2, 4, 16
    rng = np.random.default_rng(base)
    c = PagedCache(2, 16, kv, d, sequences=3, max_pages=6, page_size=16)
    cos, sin = torch.ones((96, d // 2), device="cuda"), torch.zeros((96, d // 2), device="cuda")
    norm = torch.ones(d, device="cuda")

    def rows_of(b, n):                                 # K and V of both layers at positions 0 .. n - 1
        table, keys, values = c.table.cpu().numpy(), c.keys.cpu().numpy(), c.values.cpu().numpy()
        return [np.stack([pool[:, table[b, j // 16], :, j % 16] for j in range(n)]) for pool in (keys, values)]

    def step(bases, trees):
        c.resize([b + len(t) if t else -1 for b, t in zip(bases, trees)])
        tree = c.plan_tree(np.concatenate(trees).astype(int).tolist(), starts_of(trees).tolist())
        tokens = sum(len(t) for t in trees)
        for layer in range(2):
            c.append_tree(layer, up(rng.standard_normal((tokens, (groups + 2) * kv * d)).astype(np.float32)), norm, norm,
                          cos, sin, 1e-6, tree)
        return tree

    if base:
        step([0] * 3, [chain(base), [], []])
    comb = [-1, 0, 0, 2, 2, 4, 4, 6, 6, 8, 8, 10, 10, 12, 12, 14, 14, 16, 16, 18]    # the even nodes are the path
    tree = step([base] * 3, [comb, [], []])
    before = rows_of(0, base + len(comb))
    kept, path, _ = c.accept(tree, [i % 2 for i in range(len(comb))], choices=[0] * len(comb))
    n = base + 10
    assert kept.tolist() == [n, -1, -1] and path.tolist()[:11] == list(range(0, 20, 2)) + [-1]
    c.resize(kept)
    c.fork([-1, 0, 0])
    assert c.lengths.tolist() == [n] * 3
    shared = [np.concatenate([pool[:base], pool[base:][::2]]) for pool in before]
    tree = step([n] * 3, [chain(7), comb, []])
    nodes = [rows_of(0, n + 7), rows_of(1, n + len(comb))]
    kept, _, _ = c.accept(tree, [0] * 7 + [i % 2 for i in range(len(comb))], choices=[0] * (7 + len(comb)))
    assert kept.tolist() == [n + 7, n + 10, -1]
    c.resize(kept)
    expect = [nodes[0], [np.concatenate([pool[:n], pool[n:][::2]]) for pool in nodes[1]], shared]
    for b, length in enumerate((n + 7, n + 10, n)):
        for got, want, start in zip(rows_of(b, length), expect[b], shared):
            np.testing.assert_array_equal(got, want)
            np.testing.assert_array_equal(got[:n], start)
    c.check_status()


# ------------------------------------------------------------------ accept: lengths, plans and vocabularies that do not fit
@gpu
@pytest.mark.parametrize("by", ["choices", "logits"])
@pytest.mark.parametrize("length", [-2**31, -2**31 + 5, -2**31 + 9, -5, -1, 0, 9])
def test_accept_of_lengths_below_the_tree(length, by):
    # a base before the sequence, at the lowest lengths too: it takes no part, and the others do
    from harsh4b_amd.tree import pages_accept
    trees, bases = [chain(6), star(10), chain(4)], [20, 30, 5]
    table, lengths, keys, values = _cache_of(trees, bases, d=64)
    n = sum(len(t) for t in trees)
    drafted, choices = [1] * n, [1] * n
    drafted[6 + 1:6 + 9] = [0] * 8                      # (the star's last child: a row that would move)
    ek, ev, kept, path, after = _expect_accept([trees[0], [], trees[2]], bases, table, keys, values,
                                               drafted[:6] + drafted[16:], choices[:6] + choices[16:])
    lengths[1] = length
    how = dict(choices=ints(choices))
    if by == "logits":
        how = dict(logits=torch.zeros((n, 40), device="cuda"))
        how["logits"][:, 1] = 1.0
    status, dk, dv, size = ints([0]), up(keys), up(values), ints(lengths)
    got = pages_accept(dk, dv, ints(table), size, status, plan(trees), ints(drafted), **how)
    assert [g.tolist() for g in got] == [kept, path[:6] + [-1] * 10 + path[6:], after]
    assert int(status.item()) == 2 and size.tolist() == lengths
    np.testing.assert_array_equal(dk.cpu().numpy(), ek)
    np.testing.assert_array_equal(dv.cpu().numpy(), ev)


@gpu
@pytest.mark.parametrize("what", ["zeros", "short", "largest", "random"])
def test_accept_of_depths_that_are_not_the_trees(what):
    # a plan of other trees: by logits the path ends at its deepest level and says so, choices do not look at depths;
    # two runs agree, and the other sequences have their paths
    from harsh4b_amd.tree import pages_accept
    trees, bases = [chain(9), chain(40), random_tree(np.random.default_rng(5), 30, 6)], [20, 3, 50]
    n, at = sum(len(t) for t in trees), slice(9, 49)
    drafted, choices = [7] * n, [7] * n
    table, lengths, keys, values = _cache_of(trees, bases)
    logits = torch.zeros((n, 5000), device="cuda")
    logits[:, 7] = 1.0
    t = plan(trees)
    rng = np.random.default_rng(8)
    for _ in range(3):
        depths = t.depths.clone()
        false = {"zeros": np.zeros(40), "short": np.minimum(np.arange(40), 11), "largest": np.full(40, 2**31 - 1),
                 "random": rng.integers(-2**31, 2**31, 40)}[what].astype(np.int64)
        false[0] = abs(false[0]) % 2**31
        depths[at] = ints(false)
        levels = min(40, int(max(0, false.max())) + 1)
        for how, expect in ((dict(logits=logits), levels), (dict(choices=ints(choices)), 40)):
            runs = []
            for _ in range(2):
                status, dk = ints([0]), up(keys)
                got = pages_accept(dk, up(values), ints(table), ints(lengths), status, t._replace(depths=depths),
                                   ints(drafted), **how)
                runs.append([g.tolist() for g in got] + [int(status.item())])
            assert runs[0] == runs[1]
            kept, path, after, code = runs[0]
            assert path[at] == list(range(expect)) + [-1] * (40 - expect) and code == (0 if expect == 40 else 2)
            assert kept[1] == 3 + expect and after == [7, 7, 7]
            for b, rows in ((0, slice(0, 9)), (2, slice(49, n))):
                p, _ = walk(trees[b], drafted[rows], choices[rows])
                assert path[rows] == p + [-1] * (len(trees[b]) - len(p)) and kept[b] == bases[b] + len(p)


# ------------------------------------------------------------------ joins and plans of mixed batches
@gpu
@pytest.mark.parametrize("kv,groups,d", [(8, 6, 128), (8, 8, 128), (8, 5, 128), (4, 6, 64)])
def test_joins_of_rows_of_other_widths(kv, groups, d):
    # 192 and 256 threads a row (a wave left over, none); rows that are no whole waves
    rng = np.random.default_rng(groups * d)
    sizes = [int(n) for n in rng.integers(17, 27, 26)]
    s = Trees(some_trees(d, sizes), [int(b) for b in rng.integers(300, 1500, 26)], kv, groups, d, 64, seed=d)
    assert s.tokens * kv >= 2048
    s._check()
    s._check(window=700, sinks=3)


# ------------------------------------------------------------------ vocabularies past what the kernels count
def test_accept_refuses_vocabularies_past_2_30():
    lib = native().lib()
    c, p, _ = _struct()
    t = ctypes.byref(_tree_struct(p))
    for vocab in ((1 << 30) + 1, (1 << 31) - 256, (1 << 31) - 1):
        assert lib.hq_pages_accept(ctypes.byref(c), t, p, None, p, vocab, 4, p, p, p, p, None) == 1
        assert lib.hq_pages_accept_workspace_bytes(3, 1, vocab, 4) == 0
    assert lib.hq_pages_accept_workspace_bytes(3, 1, 1 << 30, 4) > 0


@gpu
def test_python_refuses_vocabularies_past_2_30():
    from harsh4b_amd.tree import DraftTree, pages_accept
    table, lengths, keys, values = _cache_of([[-1]], [3])
    none = DraftTree(ints([]), ints([0, 0]), ints([]), ints(np.zeros((0, 8))))
    for vocab in ((1 << 30) + 1, (1 << 32) + 5):
        with pytest.raises(ValueError, match="vocabulary"):
            pages_accept(up(keys), up(values), ints(table), ints(lengths), ints([0]), none, ints([]),
                         logits=torch.zeros((0, vocab), device="cuda"))


# ------------------------------------------------------------------ rows longer than a block holds in registers
@gpu
@pytest.mark.parametrize("n", [10240, 10241, 12001, 20001])
def test_long_rows_that_are_not_finite(n):
    # as test_rows_that_are_not_finite, in place and beside the input: the single row calls' bits, row by row
    from harsh4b_amd.lightspark import add_rmsnorm_quant, quantize_activation, rmsnorm
    rng = np.random.default_rng(n)
    x = rng.standard_normal((9, n)).astype(np.float32)
    x[1] = 0
    x[2, n - 1] = np.inf
    x[3, 7] = np.nan
    x[4] *= np.float32(1e30)
    x[5] *= np.float32(1e-30)
    x[6, n - 257] = -np.inf
    x[7] = np.finfo(np.float32).max
    x[8, 300], x[8, n - 1] = np.inf, -np.inf
    gamma, delta = rng.uniform(0.5, 1.5, n).astype(np.float32), rng.standard_normal((9, n)).astype(np.float32)
    delta[1] = 0
    dg, total = up(gamma), up(x) + up(delta)
    for out in (None, torch.empty((9, n), device="cuda")):
        dx = up(x)
        q, s = add_rmsnorm_quant(dx, dg, 1e-6, delta=up(delta), out=out)
        assert (dx if out is None else out).cpu().numpy().tobytes() == total.cpu().numpy().tobytes()
        for i in range(9):
            eq, es = quantize_activation(rmsnorm(total[i].contiguous(), dg, 1e-6))
            assert torch.equal(q[i], eq), i
            assert s[i].cpu().numpy().tobytes() == es[0].cpu().numpy().tobytes() or (s[i].isnan() and es[0].isnan()), i


# ------------------------------------------------------------------ pieces of batches of long and short chats
def _pieces(s, groups):
    """Pieces of each sequence's first tile, as the attention leaves them in its workspace: behind the plan (256 bytes,
    tokens + 1 ints and tokens times four, each up to 256 bytes) a row's and kv head's 2 * pieces + small, first part."""
    from harsh4b_amd import paged, tree
    lib = native().lib()
    d, t = s.device(), plan(s.trees)
    kv, dim = s.keys.shape[1], s.keys.shape[3]
    size = lib.hq_paged_attention_tree_workspace_bytes(s.tokens, kv * groups, kv, dim)
    workspace = torch.zeros(size + 256, dtype=torch.uint8, device="cuda")
    at = -workspace.data_ptr() % 256
    index = d["keys"].get_device()
    cache, sequences, _, _ = paged._cache(index, d["keys"], d["values"], d["table"], d["lengths"], None, None, 4)
    out = torch.empty_like(d["query"])
    code = lib.hq_paged_attention_tree(cache, d["query"].data_ptr(), tree._tree(t, s.tokens, sequences, index), kv * groups,
                                       0, 0, out.data_ptr(), workspace.data_ptr() + at, torch.cuda.current_stream().cuda_stream)
    assert code == 0
    torch.cuda.synchronize()
    up256 = lambda n: (n + 255) // 256 * 256
    at += 256 + up256(4 * (s.tokens + 1)) + up256(16 * s.tokens)
    desc = workspace[at:at + 8 * s.tokens * kv].cpu().numpy().view(np.int32).reshape(s.tokens, kv, 2)
    return [int(desc[first, 0, 0]) >> 1 for first in s.starts[:-1]], out.cpu().numpy()


def _check_pieces(s, groups):
    """No piece has more than a small multiple of the chunks that the batch's work gives each of 512 places: sizes go up
    to 2.04 times those (at least 4; tiles of 16 rows, at most 256 of 8 chunks, add 4), and a sequence of less than 3/2
    sizes is one piece, as are large tiles of up to 16 chunks."""
    pieces, out = _pieces(s, groups)
    kv, dim = s.keys.shape[1], s.keys.shape[3]
    chunks = [-(-n // 64) for n in s.lengths]
    tiles = [1 if len(t) * groups <= 32 else -(-len(t) // (128 // groups)) for t in s.trees]
    target = -(-sum(c * t for c, t in zip(chunks, tiles)) * kv // 512)
    longest = max(-(-c // p) for c, p in zip(chunks, pieces))
    assert longest <= max(16, 3.1 * (target + 4) + 2), (longest, target)
    return out


@gpu
@pytest.mark.parametrize("bases,nodes,kv,groups", [([300] * 59 + [20000], 8, 8, 4), ([300] * 46 + [40960], 16, 8, 2),
                                                   ([40000] + [300] * 10, 16, 32, 1), ([3000] * 31 + [30000] + [3000] * 30, 5, 8, 3),
                                                   ([500] * 56 + [16384], 16, 8, 4)])
def test_one_long_chat_among_short_ones(bases, nodes, kv, groups):
    # the long one is cut, though the short ones take most places, and the results are the definition's
    rng = np.random.default_rng(nodes + kv)
    s = Trees([random_tree(rng, nodes) for _ in bases], bases, kv, groups, 16, 64, seed=kv)
    out = _check_pieces(s, groups)
    expect, bound = _reference(s, s.trees, 0, 0)
    off = np.abs(out - expect).reshape(s.tokens, -1).max(axis=1)
    assert (off <= bound).all(), (off.max(), bound[np.argmax(off - bound)])


@gpu
def test_pieces_of_drawn_batches():
    rng = np.random.default_rng(77)
    for i in range(40):
        kv, groups = [(8, 4), (8, 1), (16, 2), (32, 1), (4, 8), (2, 6)][i % 6]
        count = int(rng.integers(2, 65))
        bases = [int(np.exp(rng.uniform(np.log(20), np.log(rng.choice([400, 4000]))))) for _ in range(count)]
        for b in rng.integers(0, count, rng.integers(1, 4)):
            bases[b] = int(rng.integers(8000, 24000))
        trees = [random_tree(rng, int(n)) for n in rng.integers(1, rng.choice([8, 40]), count)]
        print(f"[gpu] drawn {i}: {count} sequences, {kv} kv heads of {groups}", flush=True)
        _check_pieces(Trees(trees, bases, kv, groups, 16, 64, seed=i), groups)
