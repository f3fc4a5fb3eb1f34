"""The paged attention where a worker's part of a sequence has many tiles: the running maximum and the
rescaled sums inside a part, the ring's and the buffers' reuse, the reload of page ids, tokens that are
not finite in two neighbouring tiles, and joins of more partials than a workgroup has threads.

A call cuts all its tiles into one equal share for each worker of the chip, so small calls have parts of one
tile.  Sequences here point at shared read-only pages, which makes calls large and the 64-bit statements
small, and every test counts the tiles of its parts from the lengths (``parts``) before it relies on them.
Tolerances are test_gpu_paged's.
"""

import math

import numpy as np
import pytest
import torch

from tests.test_gpu_paged import E4M3, bounds
from wanferenz_amd.paged import PagedKV

pytestmark = pytest.mark.gpu


def workers(cache, S, H):
    """The number of shares a call is cut into, from the size of its partials (2 a share, m and l in whole 16
    bytes and O) and records (16 bytes)."""
    R = S * (H // cache.kv_heads)
    rows = min(R, 16 if R <= 16 else 32 if R <= 32 else 64)
    one = 2 * 4 * ((2 * rows + 3) // 4 * 4 + rows * cache.head_dim) + 16
    w, rest = divmod(cache.attend_workspace_bytes(1, S, H, 1), one)
    assert rest == 0 and w > 0
    return w


def parts(cache, lens, S, H):
    """Tiles of every part that the call is cut into: each sequence's units laid end to end, their tiles and a
    start of a few, in one equal share a worker."""
    R = S * (H // cache.kv_heads)
    latent = cache.v is None and cache.head_dim == 512
    tile, start = (64, 4) if latent else (32, 3)
    units = [-(-n // tile) + start for n in lens if n > 0
             for _ in range(cache.kv_heads * -(-R // (16 if R <= 16 else 32 if R <= 32 else 64)))]
    W, total = workers(cache, S, H), sum(units)
    count = total if total <= W // 2 else min((total + 1) // 2, W)
    each, rest = divmod(total, count)
    ends = np.cumsum([each + 1] * rest + [each] * (count - rest))
    out, at = [], 0
    for cost in units:
        edges = [at, *[int(e) for e in ends[np.searchsorted(ends, at, "right"):np.searchsorted(ends, at + cost)]], at + cost]
        cut = [max(b - at - start, 0) - max(a - at - start, 0) for a, b in zip(edges, edges[1:])]
        out.append([x for x in cut if x > 0])
        at += cost
    return out


def rows_of(cache, table_row, n):
    """K and V [HK, n, D] of a sequence in 64 bits."""
    out = []
    for pool, scale in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        if pool is None:
            out.append(out[0])
            continue
        x = pool[table_row].double()
        if scale is not None:
            x = x * scale[table_row].double()[..., None]
        out.append(x.transpose(0, 1).reshape(cache.kv_heads, -1, cache.head_dim)[:, :n].contiguous())
    return out


def plain(cache, q, table_row, n, scale, sink=None):
    """One sequence's attention from its definition, in 64 bits: (o, abs [S, H, D], the weight of each slot
    [HK, n], the largest sum |q k| scale); an element that a token which is not finite reaches is not finite."""
    S, H, D = q.shape
    g = H // cache.kv_heads
    k, v = rows_of(cache, table_row, n)
    o, mag = (torch.zeros(S, H, D, dtype=torch.float64, device=q.device) for _ in range(2))
    add = torch.zeros(cache.kv_heads, n, dtype=torch.float64, device=q.device)
    reach = 0.0
    for i in range(S):
        seen = n - (S - 1 - i)
        if seen <= 0:
            continue
        for hk in range(cache.kv_heads):
            kk, vv = k[hk, :seen], v[hk, :seen]
            x = q[i, hk * g:(hk + 1) * g].double()
            s = torch.matmul(x, kk.t().contiguous()) * scale
            reach = max(reach, float(torch.nan_to_num(torch.matmul(x.abs(), kk.abs().t().contiguous()), 0, 0, 0).max()) * scale)
            top = s.amax(1, keepdim=True)
            if sink is not None:
                top = torch.maximum(top, sink[hk * g:(hk + 1) * g, None].double())
            e = torch.exp(s - top)
            den = e.sum(1, keepdim=True)
            if sink is not None:
                den = den + torch.exp(sink[hk * g:(hk + 1) * g, None].double() - top)
            p = e / den
            o[i, hk * g:(hk + 1) * g] = torch.matmul(p, vv)
            mag[i, hk * g:(hk + 1) * g] = torch.matmul(p, vv.abs())
            add[hk, :seen] += p.sum(0)
    return o, mag, add, reach


def compare(got, ref, D):
    """Elements that are finite in 64 bits within the tolerance, the others not finite."""
    o, mag, _, reach = (x.cpu().numpy() if torch.is_tensor(x) else x for x in ref)
    got = got.double().cpu().numpy()
    fine = np.isfinite(o)
    assert (np.isfinite(got) == fine).all(), "not finite elsewhere"
    tol, _ = bounds(np.where(fine, o, 0), np.where(fine, mag, 0), reach, D)
    err = np.abs(np.where(fine, got - np.where(fine, o, 0), 0.0))
    assert (err <= tol).all(), (float((err / tol).max()), np.unravel_index((err / tol).argmax(), err.shape))


def pools(gpu, seed, P, HK, D, page, dtype, shared, shape=None, **tracked):
    """A cache of P random pages; ``shape`` scales or changes the rows of K [P, HK, page, D] first."""
    g = torch.Generator(device=gpu).manual_seed(seed)
    sides, scales = [], []
    for side in range(1 if shared else 2):
        x = torch.randn(P, HK, page, D, device=gpu, generator=g)
        if side == 0 and shape is not None:
            x = shape(x)
        x = x.to(torch.bfloat16)
        if dtype == E4M3:
            x = x.float()
            s = x.abs().amax(-1).clamp(min=1e-4) * (1.0 / 448.0)
            x = (x / s[..., None]).clamp(-448, 448).to(E4M3)
            scales.append(s)
        sides.append(x)
    scales += [None] * (2 - len(scales))
    return PagedKV(sides[0], None if shared else sides[1], k_scale=scales[0], v_scale=scales[1], **tracked)


def query(gpu, seed, B, S, H, D, scale=1.0):
    g = torch.Generator(device=gpu).manual_seed(seed)
    return (torch.randn(B, S, H, D, device=gpu, generator=g) * scale).to(torch.bfloat16)


def repeated(gpu, seed, distinct, copies, page, P):
    """Tables of ``distinct`` lengths, each ``copies`` times: random pages of P, the same in every copy."""
    rng = np.random.default_rng(seed)
    width = -(-max(distinct) // page)
    rows = rng.integers(0, P, (len(distinct), width)).astype(np.int32)
    return torch.from_numpy(np.repeat(rows, copies, 0)).to(gpu), [n for n in distinct for _ in range(copies)]


# R rows a KV head: one, two and four tiles of 16, the last by two waves; latents of the same
LAYOUTS = [  # HK, g, S, D, shared, copies
    (2, 4, 1, 128, False, 24), (2, 4, 3, 128, False, 24), (1, 24, 1, 128, False, 48), (2, 12, 4, 128, False, 12),
    (2, 8, 1, 64, False, 48), (2, 2, 16, 64, False, 48), (1, 40, 1, 64, False, 64), (2, 4, 1, 256, False, 24),
    (1, 9, 6, 256, False, 24), (1, 16, 1, 128, True, 48), (1, 64, 1, 256, True, 24),
    (1, 16, 1, 512, True, 24), (1, 32, 1, 512, True, 24), (1, 64, 1, 512, True, 24),
    (1, 16, 2, 512, True, 24), (1, 32, 2, 512, True, 24), (1, 8, 2, 512, True, 24), (1, 64, 2, 512, True, 12),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, E4M3])
@pytest.mark.parametrize("HK,g,S,D,shared,copies", LAYOUTS)
def test_parts_of_many_tiles(gpu, HK, g, S, D, shared, copies, dtype):
    """Four tiles and more in most parts: random rows, ragged ends, a sink."""
    page, distinct, H = 32, [4090, 2049, 4128], HK * g
    cache = pools(gpu, D + g, 150, HK, D, page, dtype, shared)
    table, lens = repeated(gpu, S + g, distinct, copies, page, cache.pages)
    tiles = [x for unit in parts(cache, lens, S, H) for x in unit]
    assert np.median(tiles) >= 4
    q = query(gpu, g, len(distinct), S, H, D, 1.5)
    sink = torch.linspace(-2, 3, H, device=gpu)
    o = cache.attend(q.repeat_interleave(copies, 0), table, torch.tensor(lens, dtype=torch.int32, device=gpu), D ** -0.5,
                     attn_sink=sink)
    for i, n in enumerate(distinct):
        ref = plain(cache, q[i], table[i * copies].long(), n, D ** -0.5, sink)
        for x in o[i * copies:(i + 1) * copies]:
            compare(x, ref, D)


def along(gpu, lens, page, height):
    """Tables of consecutive pages, and height(t / n) of every slot [pages, 1, page, 1]."""
    need = [-(-n // page) for n in lens]
    table = torch.zeros(len(lens), max(need), dtype=torch.int32)
    level, at = torch.zeros(sum(need), page), 0
    for b, (n, c) in enumerate(zip(lens, need)):
        table[b, :c] = torch.arange(at, at + c)
        level[at:at + c] = height(torch.arange(c * page) / n).view(c, page)
        at += c
    return table.to(gpu), level[:, None, :, None].to(gpu)


HEIGHTS = {  # the scores' course along a sequence, in powers of two (the maximum is moved past a rise of 8)
    "rise": lambda x: 300 * x,
    "slow": lambda x: 24 * x,
    "steps": lambda x: 7.0 * torch.floor(12 * x),
    "far steps": lambda x: 40.0 * torch.floor(5 * x) - 100,
    "fall": lambda x: 200 * (1 - x),
    "hill": lambda x: 120 * torch.sin(math.pi * x) - 60,
    "late peak": lambda x: torch.where((x > 0.62) & (x < 0.6205), 60.0, 0.0),
}


@pytest.mark.parametrize("dtype", [torch.bfloat16, E4M3])
@pytest.mark.parametrize("HK,g,S,D,shared", [(1, 4, 1, 128, False), (1, 24, 1, 64, False), (1, 48, 1, 128, False),
                                             (1, 16, 1, 512, True), (1, 32, 1, 512, True), (1, 64, 1, 512, True),
                                             (1, 32, 2, 512, True)])
@pytest.mark.parametrize("course", HEIGHTS)
def test_running_maximum_inside_a_part(gpu, course, HK, g, S, D, shared, dtype):
    """Scores that rise and fall along a part, by less and by more than the maximum is moved at."""
    page, distinct, H, copies = 64, [4000, 2700], HK * g, 80 if D == 64 else 64
    table, level = along(gpu, distinct, page, HEIGHTS[course])
    # one coordinate carries the course: q has 8 there, k the height over 8 (in bits of the exponent)
    scale = D ** -0.5

    def shape(x):
        x = x * 0.5
        x[..., 5:6] = (level * (math.log(2.0) / (8.0 * scale))).to(x.dtype)
        return x

    cache = pools(gpu, 7, level.shape[0], HK, D, page, dtype, shared, shape)
    tables, lens = table.repeat_interleave(copies, 0), [n for n in distinct for _ in range(copies)]
    tiles = [x for unit in parts(cache, lens, S, H) for x in unit]
    assert np.median(tiles) >= 4
    q = query(gpu, g, len(distinct), S, H, D, 0.5)
    q[..., 5] = 8.0
    o = cache.attend(q.repeat_interleave(copies, 0), tables, torch.tensor(lens, dtype=torch.int32, device=gpu), scale)
    for i, n in enumerate(distinct):
        ref = plain(cache, q[i], table[i].long(), n, scale)
        for x in o[i * copies:(i + 1) * copies]:
            compare(x, ref, D)


@pytest.mark.parametrize("dtype", [torch.bfloat16, E4M3])
@pytest.mark.parametrize("HK,g,D,shared,page,copies,least", [(4, 4, 128, False, 16, 48, 33), (4, 4, 128, False, 32, 96, 65),
                                                             (1, 40, 64, False, 16, 96, 33), (1, 40, 128, False, 64, 192, 65),
                                                             (1, 16, 512, True, 64, 80, 65), (1, 64, 512, True, 16, 80, 65)])
def test_page_ids_are_fetched_again_inside_a_part(gpu, HK, g, D, shared, page, copies, least, dtype):
    """More tiles in a part than a wave holds page ids for (64 ids, two a tile for pages of 16), in an order
    that does not repeat."""
    distinct, H = [9000, 7001] if D == 512 else [4090, 3333], HK * g
    if dtype == E4M3 and D == 64:
        copies *= 2
    cache = pools(gpu, page, 97, HK, D, page, dtype, shared)
    table, lens = repeated(gpu, page + g, distinct, copies, page, cache.pages)
    assert max(x for unit in parts(cache, lens, 1, H) for x in unit) >= least
    q = query(gpu, g, len(distinct), 1, H, D)
    o = cache.attend(q.repeat_interleave(copies, 0), table, torch.tensor(lens, dtype=torch.int32, device=gpu), D ** -0.5)
    for i, n in enumerate(distinct):
        ref = plain(cache, q[i], table[i * copies].long(), n, D ** -0.5)
        for x in o[i * copies:(i + 1) * copies]:
            compare(x, ref, D)


@pytest.mark.parametrize("dtype", [torch.bfloat16, E4M3])
@pytest.mark.parametrize("g,D,shared,n,least", [(3, 64, False, 12000, 257), (1, 64, False, 30001, 257), (24, 128, False, 12000, 257),
                                                (64, 512, True, 16000, 100)])
def test_joins_of_many_partials(gpu, g, D, shared, n, least, dtype):
    """A sequence cut into more parts than the join's workgroup has threads; odd numbers of rows."""
    cache = pools(gpu, n, 180, 1, D, 64, dtype, shared)
    table, lens = repeated(gpu, g, [n], 1, 64, cache.pages)
    assert max(len(unit) for unit in parts(cache, lens, 1, g)) >= least
    q = query(gpu, g, 1, 1, g, D, 2.0)
    o = cache.attend(q, table, torch.tensor(lens, dtype=torch.int32, device=gpu), D ** -0.5)
    compare(o[0], plain(cache, q[0], table[0].long(), n, D ** -0.5), D)


@pytest.mark.parametrize("dtype", [torch.bfloat16, E4M3])
@pytest.mark.parametrize("HK,g,D,shared,copies", [(1, 1, 128, False, 64), (1, 2, 128, False, 64), (1, 4, 64, False, 64),
                                                  (1, 1, 512, True, 24), (1, 2, 512, True, 24), (1, 4, 512, True, 24)])
def test_values_that_are_not_finite_in_two_tiles_of_a_part(gpu, HK, g, D, shared, copies, dtype):
    """The newest 16 tokens lie in two tiles, and each has one that is not finite: rows take them where they see
    them and nothing where they do not."""
    page, S, H = 16, 16, HK * g
    n = 64 * 64 + 9  # the newest tokens from 64 x 64 - 7 on
    cache = pools(gpu, g, -(-n // page), HK, D, page, dtype, shared)
    table = torch.arange(cache.pages, dtype=torch.int32, device=gpu)[None].repeat(copies, 1)
    lens = [n] * copies
    cut = parts(cache, lens, S, H)
    assert sum(unit[-1] >= 2 for unit in cut) >= copies // 4  # both tiles in one part of these
    pool = cache.k if shared else cache.v
    for t, c in ((n - 12, 3), (n - 5, 40)):
        if dtype == E4M3:
            pool[t // page, :, t % page, c].view(torch.uint8).fill_(0x7F)
        else:
            pool[t // page, :, t % page, c] = float("inf") if not shared else float("nan")
    q = query(gpu, g, 1, S, H, D)
    o = cache.attend(q.repeat(copies, 1, 1, 1), table, torch.tensor(lens, dtype=torch.int32, device=gpu), D ** -0.5)
    ref = plain(cache, q[0], table[0].long(), n, D ** -0.5)
    assert torch.isfinite(ref[0][:4]).all() and not torch.isfinite(ref[0][4:, :, 3]).any()
    assert torch.isfinite(ref[0][4:11, :, 40]).all() != shared
    for x in o:
        compare(x, ref, D)


@pytest.mark.parametrize("dtype", [torch.bfloat16, E4M3])
@pytest.mark.parametrize("HK,g,S,D,shared,n", [(2, 4, 1, 64, False, 40000), (2, 4, 3, 128, False, 40000), (1, 48, 1, 64, False, 40000),
                                               (1, 16, 1, 512, True, 20011), (1, 64, 1, 512, True, 20011),
                                               (1, 16, 4, 512, True, 20011)])
def test_weights_of_parts_of_many_tiles(gpu, HK, g, S, D, shared, n, dtype):
    """The weights that slots get where the scores come from parts of several tiles, of a cache with pages of
    its own for every sequence."""
    page, lens, H = 64, [n, n // 2, n, n - 33], HK * g
    need = [-(-x // page) for x in lens]
    P = sum(need)
    w, pos = torch.zeros(P, HK, page, device=gpu), torch.zeros(P, HK, page, dtype=torch.int32, device=gpu)
    cache = pools(gpu, n + g, P, HK, D, page, dtype, shared, weights=w, positions=pos)
    order = torch.randperm(P, generator=torch.Generator().manual_seed(n)).to(torch.int32)
    table = torch.full((4, max(need)), -1, dtype=torch.int32)
    for b, c in enumerate(need):
        table[b, :c] = order[sum(need[:b]):sum(need[:b]) + c]
    table = table.to(gpu)
    assert np.median([x for unit in parts(cache, lens, S, H) for x in unit]) >= 2
    q = query(gpu, g, 4, S, H, D, 1.5)
    o = cache.attend(q, table, torch.tensor(lens, dtype=torch.int32, device=gpu), D ** -0.5, accumulate=True)
    for b, x in enumerate(lens):
        row = table[b, :need[b]].long()
        ref = plain(cache, q[b], row, x, D ** -0.5)
        compare(o[b], ref, D)
        got = w[row].transpose(0, 1).reshape(HK, -1).double()
        _, e32 = bounds(ref[0].cpu().numpy(), ref[1].cpu().numpy(), ref[3], D)
        # a sum of S g float32 terms
        assert ((got[:, :x] - ref[2]).abs() <= (e32 + S * g * 2.0 ** -24) * ref[2] + 1e-30).all()
        assert (got[:, x:] == 0).all()
