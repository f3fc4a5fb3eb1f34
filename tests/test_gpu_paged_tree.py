"""PagedKV.attend_tree against its 64-bit statement, with the tolerances of the paged attention."""

import numpy as np
import pytest
import torch

from oracle import paged as op
from tests.test_gpu_paged import E4M3, check, make, queries

pytestmark = pytest.mark.gpu


def trees(seed, B, S, kind="random"):
    rng = np.random.default_rng(seed)
    if kind == "chain":
        return np.tile(np.arange(S, dtype=np.int32) - 1, (B, 1))
    if kind == "star":
        return np.tile(np.array([-1] + [0] * (S - 1), dtype=np.int32), (B, 1))
    p = np.array([[-1] + [int(rng.integers(0, i)) for i in range(1, S)] for _ in range(B)], dtype=np.int32).reshape(B, S)
    if kind == "forest":  # several roots, of every value that is no node
        p[rng.random((B, S)) < 0.3] = -1
        p[0, S // 2] = S
        p[-1, S - 1] = -2 ** 31
    return p


def run(gpu, cache, tab, lens, parent, q, scale, **more):
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=gpu)  # noqa: E731
    if more.get("count") is not None:
        more["count"] = i32(more["count"])
    return cache.attend_tree(q, tab, i32(lens), torch.from_numpy(parent).to(gpu), scale, **more)


MANY = 9000  # pages of a table that a call cannot take for a small one

LAYOUTS = [  # HK, g, D, shared
    (2, 4, 128, False), (8, 1, 128, False), (1, 16, 64, False), (2, 3, 64, False), (2, 5, 256, False),
    (1, 8, 128, True), (1, 5, 256, True), (1, 16, 512, True), (1, 20, 512, True),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, E4M3])
@pytest.mark.parametrize("HK,g,D,shared", LAYOUTS)
@pytest.mark.parametrize("S", [1, 7, 33])
@pytest.mark.parametrize("width", [None, MANY])
def test_layouts(gpu, width, S, HK, g, D, shared, dtype):
    """Head layouts and widths, ragged prefixes among them none, trees smaller and larger than a tile; tables as wide as
    the sequences, whose rows go 16 at a time, and much wider ones, whose rows go together."""
    lens = [S + n for n in (0, 1, 16, 31, 100, 300)]
    cache, vals, tab, table = make(gpu, D + HK + g, lens, HK=HK, D=D, page=16, dtype=dtype, shared=shared, width=width)
    q, qd = queries(gpu, g, len(lens), S, HK * g, D, strided=True)
    parent = trees(S, len(lens), S)
    o = run(gpu, cache, tab, lens, parent, q, D ** -0.5)
    check(o, op.attend_tree(vals, qd, table, lens, parent, D ** -0.5), D)


@pytest.mark.parametrize("kind", ["chain", "star", "random", "forest"])
@pytest.mark.parametrize("S,page", [(2, 16), (16, 64), (63, 32), (64, 1024)])
@pytest.mark.parametrize("width", [None, MANY])
def test_shapes_of_trees(gpu, width, S, page, kind):
    """Chains, stars, forests whose roots hang on the prefix; more rows than a unit; a sink; lengths at and off the
    tiles' borders; sequences that hold less than their tree."""
    lens = [S, 0, 1, S + 31, 128, 129, 257, 700]
    HK, g, D = 2, 8, 64
    cache, vals, tab, table = make(gpu, S + page, lens, HK=HK, D=D, page=page, width=width)
    q, qd = queries(gpu, S, len(lens), S, HK * g, D, scale=1.5)
    sink = torch.linspace(-3, 4, HK * g)
    parent = trees(S + page, len(lens), S, kind)
    o = run(gpu, cache, tab, lens, parent, q, D ** -0.5, attn_sink=sink.to(gpu))
    check(o, op.attend_tree(vals, qd, table, lens, parent, D ** -0.5, sink.double().numpy()), D)


def test_a_chain_is_attend(gpu):
    """The chain's rows are attend's up to the rounding of both."""
    S, lens, HK, g, D = 9, [300, 77, 9], 2, 4, 128
    cache, vals, tab, table = make(gpu, 3, lens, HK=HK, D=D, page=32)
    q, qd = queries(gpu, 3, 3, S, HK * g, D)
    ref = op.attend(vals, qd, table, lens, D ** -0.5)
    n = torch.tensor(lens, dtype=torch.int32, device=gpu)
    check(cache.attend(q, tab, n, D ** -0.5), ref, D)
    check(run(gpu, cache, tab, lens, trees(0, 3, S, "chain"), q, D ** -0.5), ref, D)


def test_parents_in_any_order_and_rings(gpu):
    """A parent may stand behind its child; parents that lead in a ring end (every node of it sees the others)."""
    S, lens, HK, g, D = 6, [90, 41], 1, 4, 64
    cache, vals, tab, table = make(gpu, 8, lens, HK=HK, D=D, page=16)
    q, qd = queries(gpu, 8, 2, S, HK * g, D)
    parent = np.array([[3, 0, 1, -1, 5, 0], [1, 2, 0, 4, 3, 3]], dtype=np.int32)
    o = run(gpu, cache, tab, lens, parent, q, D ** -0.5)
    check(o, op.attend_tree(vals, qd, table, lens, parent, D ** -0.5), D)


@pytest.mark.parametrize("HK,g,D,shared,n", [(1, 4, 128, False, 4000), (1, 40, 64, False, 1500), (1, 16, 512, True, 900)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, E4M3])
@pytest.mark.parametrize("width", [None, MANY])
def test_padded_batches_over_many_workgroups(gpu, width, HK, g, D, shared, n, dtype):
    """Sequences with fewer nodes than the batch's, none and more than it; a long one that many workgroups share."""
    S, count = 21, [21, 1, 0, 8, 99, -3]
    lens = [n, 40, 55, 8, 64, 33]
    cache, vals, tab, table = make(gpu, 11, lens, HK=HK, D=D, page=64, dtype=dtype, shared=shared, width=width)
    q, qd = queries(gpu, 12, len(lens), S, HK * g, D, scale=2.0)
    parent = trees(5, len(lens), S)
    out = torch.full((len(lens), S, HK * g, D), float("nan"), dtype=torch.bfloat16, device=gpu)
    o = run(gpu, cache, tab, lens, parent, q, D ** -0.5, count=count, out=out)
    check(o, op.attend_tree(vals, qd, table, lens, parent, D ** -0.5, count=count), D)
    assert (o[2] == 0).all() and (o[1, 1:] == 0).all() and (o[5] == 0).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, E4M3])
@pytest.mark.parametrize("HK,g,D,shared", [(2, 2, 64, False), (1, 16, 128, False), (1, 24, 128, False), (2, 8, 256, False),
                                           (1, 6, 128, True), (1, 16, 512, True), (1, 64, 512, True)])
@pytest.mark.parametrize("n", [6, 40, 600])
@pytest.mark.parametrize("width", [None, MANY])
def test_a_node_takes_nothing_from_branches_it_does_not_see(gpu, width, n, HK, g, D, shared, dtype):
    """NaN in the K of one node and the V of another: every node that has neither above it stays as it was."""
    S, lens = 6, [n, n + 27]
    cache, vals, tab, table = make(gpu, 13, lens, HK=HK, D=D, page=16, dtype=dtype, shared=shared, width=width)
    q, qd = queries(gpu, 4, 2, S, HK * g, D)
    parent = np.array([[-1, 0, 0, 1, 2, 2], [-1, 0, 0, 1, 2, 2]], dtype=np.int32)
    ref = op.attend_tree(vals, qd, table, lens, parent, D ** -0.5)
    for b, m in enumerate(lens):
        for node, pool in ((1, cache.k), (4, cache.k if shared else cache.v)):
            t = m - S + node
            row = pool[table[b, t // 16], :, t % 16]
            row.view(torch.uint8 if dtype == E4M3 else torch.int16).fill_(0x7F if dtype == E4M3 else 0x7FC0)
    o = run(gpu, cache, tab, lens, parent, q, D ** -0.5)
    clean = [0, 2, 5]
    check(o[:, clean], tuple(x[:, clean] if i < 2 else x for i, x in enumerate(ref)), D)
    assert torch.isnan(o[:, [1, 3, 4]]).all()


def test_missing_pages_long_lengths_and_none(gpu):
    page, HK, D, S = 16, 2, 128, 4
    lens = [64, 64, 61, 32]
    cache, vals, tab, table = make(gpu, 9, lens, HK=HK, D=D, page=page)
    table[0, 0], table[0, 2], table[1, 3], table[1, 1] = -1, cache.pages, 2 ** 31 - 1, -(2 ** 31)
    table[3, :] = -1
    q, qd = queries(gpu, 3, 4, S, HK * 2, D)
    parent = trees(2, 4, S)
    o = run(gpu, cache, torch.from_numpy(table).to(gpu), [144, 64, 61, 32], parent, q, D ** -0.5)
    check(o, op.attend_tree(vals, qd, table, [64, 64, 61, 32], parent, D ** -0.5), D)
    assert (o[3] == 0).all()
    assert (run(gpu, cache, tab, [-5, -1, 0, -2 ** 31], parent, q, D ** -0.5) == 0).all()
    empty = run(gpu, cache, tab[:0], [], trees(0, 0, S), q[:0], 1.0)
    assert empty.shape == (0, S, HK * 2, D)


def test_more_trees_than_workers(gpu):
    B, S, HK, g, D = 300, 5, 4, 3, 64
    lens = [5 + (7 * b) % 60 for b in range(B)]
    cache, vals, tab, table = make(gpu, 21, lens, HK=HK, D=D, page=16)
    q, qd = queries(gpu, 21, B, S, HK * g, D)
    parent = trees(21, B, S)
    o = run(gpu, cache, tab, lens, parent, q, D ** -0.5)
    check(o, op.attend_tree(vals, qd, table, lens, parent, D ** -0.5), D)


def test_pool_past_32_bits(gpu):
    """Pages behind the first 2^32 bytes of a pool."""
    pages, page, HK, D, S = 40, 1024, 1024, 64, 3  # 128 MiB a page and side: 5.4 GB
    from wanferenz_amd.paged import PagedKV

    k = torch.zeros(pages, HK, page, D, dtype=torch.bfloat16, device=gpu)
    cache = PagedKV(k, k)
    lens, H = [30], HK
    g = torch.Generator().manual_seed(0)
    rows = torch.randn(30, D, generator=g).to(torch.bfloat16)
    cache.k[39, :, :30] = rows.to(gpu)
    table = np.array([[39]], dtype=np.int32)
    q = torch.randn(1, S, 1, D, generator=g).to(torch.bfloat16).expand(1, S, H, D).contiguous()
    parent = trees(1, 1, S)
    o = run(gpu, cache, torch.from_numpy(table).to(gpu), lens, parent, q.to(gpu), D ** -0.5)
    small = {"k": np.zeros((1, 1, 32, D))}
    small["k"][0, 0, :30] = rows.double().numpy()
    ref = op.attend_tree(small, q[:, :, :1].double().numpy(), np.array([[0]]), lens, parent, D ** -0.5)
    for h in (0, 511, 1023):
        check(o[:, :, h:h + 1], ref, D)


def test_refusals_workspace_and_outputs(gpu):
    S, lens, HK, g, D = 4, [40, 33], 2, 2, 64
    cache, vals, tab, table = make(gpu, 17, lens, HK=HK, D=D, page=16)
    q, qd = queries(gpu, 17, 2, S, HK * g, D)
    parent = trees(3, 2, S)
    p, n = torch.from_numpy(parent).to(gpu), torch.tensor(lens, dtype=torch.int32, device=gpu)
    ref = op.attend_tree(vals, qd, table, lens, parent, D ** -0.5)
    ws = torch.empty(cache.attend_tree_workspace_bytes(2, S, HK * g, tab.shape[1]), dtype=torch.uint8, device=gpu)
    out = torch.empty(2, S, HK * g, D, dtype=torch.bfloat16, device=gpu)
    torch.cuda.synchronize()
    before = torch.cuda.memory_stats()["allocation.all.allocated"]
    assert cache.attend_tree(q, tab, n, p, D ** -0.5, out=out, workspace=ws) is out
    assert torch.cuda.memory_stats()["allocation.all.allocated"] == before
    check(out, ref, D)
    # parents as a view of a wider tensor are copied
    wide = torch.zeros(2, 9, dtype=torch.int32, device=gpu)
    wide[:, :S] = p
    check(cache.attend_tree(q, tab, n, wide[:, :S], D ** -0.5), ref, D)
    with pytest.raises(ValueError, match="parent must be int32"):
        cache.attend_tree(q, tab, n, p.long(), 1.0)
    with pytest.raises(ValueError, match="parent must be int32"):
        cache.attend_tree(q, tab, n, p[:, :3], 1.0)
    with pytest.raises(ValueError, match="parent is on cpu"):
        cache.attend_tree(q, tab, n, p.cpu(), 1.0)
    with pytest.raises(ValueError, match="count must be"):
        cache.attend_tree(q, tab, n, p, 1.0, count=n[:1])
    with pytest.raises(ValueError, match="out must be"):
        cache.attend_tree(q, tab, n, p, 1.0, out=out[:, :2])
    with pytest.raises(Exception, match="workspace of 64 bytes"):
        cache.attend_tree(q, tab, n, p, 1.0, workspace=ws[:64])
    with pytest.raises(Exception, match="S=65"):
        z = torch.zeros(2, 65, HK * g, D, dtype=torch.bfloat16, device=gpu)
        cache.attend_tree(z, tab, n, torch.zeros(2, 65, dtype=torch.int32, device=gpu), 1.0, workspace=ws)


WIDE = [  # HK, g, S, D, shared: 65 rows and more a KV head
    (1, 5, 13, 64, False), (2, 8, 24, 64, False), (1, 7, 40, 64, False), (1, 4, 32, 128, False), (2, 3, 43, 128, False),
    (1, 8, 64, 128, False), (1, 2, 40, 128, True), (1, 9, 30, 128, True)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, E4M3])
@pytest.mark.parametrize("HK,g,S,D,shared", WIDE)
def test_many_rows_of_padded_trees(gpu, HK, g, S, D, shared, dtype):
    """Trees of every size from none to S, so that waves and whole units have no node's row, over prefixes at the tiles'
    borders and one that many workgroups share; pages that end inside a tile; a sink."""
    count = [S, 0, 1, S // 3, S - 1, S, 2 * S, -1, S // 2]
    pre = [0, 70, 63, 64, 128, 3000, 17, 30, 700]
    lens = [min(max(c, 0), S) + p for c, p in zip(count, pre)]
    cache, vals, tab, table = make(gpu, S + g, lens, HK=HK, D=D, page=16 if S % 2 else 32, dtype=dtype, shared=shared, width=MANY)
    q, qd = queries(gpu, S, len(lens), S, HK * g, D, scale=1.5, strided=True)
    parent = trees(S, len(lens), S, "forest")
    sink = torch.linspace(-2, 3, HK * g)
    out = torch.full((len(lens), S, HK * g, D), float("nan"), dtype=torch.bfloat16, device=gpu)
    o = run(gpu, cache, tab, lens, parent, q, D ** -0.5, attn_sink=sink.to(gpu), count=count, out=out)
    check(o, op.attend_tree(vals, qd, table, lens, parent, D ** -0.5, sink.double().numpy(), count=count), D)
    for b, c in enumerate(count):
        assert (o[b, min(max(c, 0), S):] == 0).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, E4M3])
@pytest.mark.parametrize("HK,g,S,D,shared", WIDE)
@pytest.mark.parametrize("n", [0, 50, 900])
def test_many_rows_take_nothing_from_branches_they_do_not_see(gpu, n, HK, g, S, D, shared, dtype):
    """NaN in the K of one node and the V of others, over two tiles of the tree: rows without them above stay as they were."""
    lens = [S + n, S + n + 37]
    cache, vals, tab, table = make(gpu, 13, lens, HK=HK, D=D, page=16, dtype=dtype, shared=shared, width=MANY)
    q, qd = queries(gpu, 4, 2, S, HK * g, D)
    parent = trees(3, 2, S)
    ref = op.attend_tree(vals, qd, table, lens, parent, D ** -0.5)
    bad = {1: cache.k, S // 2: cache.k if shared else cache.v, S - 2: cache.k if shared else cache.v}
    for b, m in enumerate(lens):
        for node, pool in bad.items():
            t = m - S + node
            row = pool[table[b, t // 16], :, t % 16]
            row.view(torch.uint8 if dtype == E4M3 else torch.int16).fill_(0x7F if dtype == E4M3 else 0x7FC0)
    o = run(gpu, cache, tab, lens, parent, q, D ** -0.5)
    for b in range(2):
        dirty = [i for i, seen in enumerate(op.tree_sight(parent[b], S)) if seen & set(bad)]
        clean = [i for i in range(S) if i not in dirty]
        check(o[b:b + 1, clean], tuple(x[b:b + 1, clean] if i < 2 else x for i, x in enumerate(ref)), D)
        assert torch.isnan(o[b, dirty]).all()


@pytest.mark.parametrize("HK,g,S,D,shared", [(1, 5, 13, 64, False), (1, 4, 32, 128, False), (1, 8, 40, 128, False)])
def test_many_rows_of_more_units_than_workers(gpu, HK, g, S, D, shared):
    B = 560
    lens = [S + (7 * b) % 90 for b in range(B)]
    cache, vals, tab, table = make(gpu, 21, lens, HK=HK, D=D, page=16, width=400)
    q, qd = queries(gpu, 21, B, S, HK * g, D)
    parent = trees(21, B, S)
    o = run(gpu, cache, tab, lens, parent, q, D ** -0.5)
    some = [0, 1, 255, 256, 300, 511, 512, 559]
    pick = lambda x: np.ascontiguousarray(x[some])  # noqa: E731
    ref = op.attend_tree(vals, pick(qd), pick(table), [lens[b] for b in some], pick(parent), D ** -0.5)
    check(o[some], ref, D)
    assert torch.isfinite(o).all()


@pytest.mark.parametrize("scale", [-0.2, 0.0, 1e-30, 3.0])
@pytest.mark.parametrize("g,S,D", [(4, 3, 64), (8, 20, 64), (8, 30, 128)])
def test_scales_of_any_sign(gpu, g, S, D, scale):
    lens = [S + 5, S + 200]
    cache, vals, tab, table = make(gpu, 31, lens, HK=1, D=D, page=16, width=MANY)
    q, qd = queries(gpu, 31, 2, S, g, D)
    parent = trees(31, 2, S)
    o = run(gpu, cache, tab, lens, parent, q, scale)
    ref = op.attend_tree(vals, qd, table, lens, parent, scale)
    check(o, (*ref[:3], abs(ref[3]) if scale >= 0 else float(np.abs(op.attend_tree(vals, -qd, table, lens, parent, -scale)[3]))), D)


@pytest.mark.parametrize("g,S,D", [(8, 24, 64), (8, 12, 128), (8, 40, 128)])
def test_many_rows_whose_maximum_moves(gpu, g, S, D):
    """K that grows along the sequence, so that the maximum moves far at many tiles."""
    lens = [S + 900, S + 333]
    cache, vals, tab, table = make(gpu, 5, lens, HK=1, D=D, page=32, width=MANY)
    grow = torch.ones(cache.pages, 1, 32, 1)
    for b, n in enumerate(lens):
        for p in range(-(-n // 32)):
            grow[table[b, p]] = 2.0 ** (p // 4)
    k = (torch.from_numpy(vals["k"]) * grow).to(torch.bfloat16)
    cache.k.copy_(torch.where(torch.isnan(cache.k.cpu()), cache.k.cpu(), k).to(gpu))
    vals["k"] = k.double().numpy()
    q, qd = queries(gpu, 6, 2, S, g, D)
    parent = trees(6, 2, S)
    o = run(gpu, cache, tab, lens, parent, q, 0.3)
    check(o, op.attend_tree(vals, qd, table, lens, parent, 0.3), D)
