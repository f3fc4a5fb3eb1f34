"""The paged cache (wanferenz_amd.paged.PagedKV) against 64-bit statements of its operators.

Tolerances of the attention, per element, from what is rounded: the output to bf16, half a step
2^-8 |o|; every p_j (times an e4m3 row's scale) to bf16 before the product with V, 2^-8 sum p_j |v_j|;
and 32-bit arithmetic: a score of D products is off by at most (D + 8) 2^-24 sum |q k| scale (plus its
maximum's own 2^-23), which moves a p_j by twice that relatively, with 2^-20 for the exponentials,
their sum and the joined parts.  A slot's accumulated weight has the last part only.
"""

import numpy as np
import pytest
import torch

from oracle import paged as op
from wanferenz_amd import _native as N
from wanferenz_amd.paged import PagedKV

pytestmark = pytest.mark.gpu
E4M3 = torch.float8_e4m3fn


def make(gpu, seed, lens, *, HK, D, page, dtype=torch.bfloat16, shared=False, track=False, spare=2, width=None,
         fill=None, kv_scale=1.0):
    """A cache whose sequences hold random rows; every other slot of the pools holds ``fill`` (NaN)."""
    rng = np.random.default_rng(seed)
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // page) for n in lens]
    width = max(need + [1]) if width is None else width
    P = sum(need) + spare
    order = rng.permutation(P)
    table = np.full((len(lens), width), -1, dtype=np.int32)
    at = 0
    for b, c in enumerate(need):
        table[b, :c] = order[at:at + c]
        at += c
    sides = ["k"] if shared else ["k", "v"]
    q = dtype == E4M3
    pools, vals = {}, {}
    live = np.zeros((P, page), dtype=bool)
    for b, n in enumerate(lens):
        for t in range(n):
            live[table[b, t // page], t % page] = True
    lv = torch.from_numpy(live)[:, None, :].expand(P, HK, page)
    for s in sides:
        x = (torch.randn(P, HK, page, D, generator=g) * kv_scale).to(torch.bfloat16)
        if q:
            sc = x.float().abs().amax(-1).clamp(min=1e-4) * (1.0 / 448.0)
            code = (x.float() / sc[..., None]).clamp(-448, 448).to(E4M3)
            vals[s] = code.double().numpy() * sc.double().numpy()[..., None]
            raw = code.view(torch.uint8).clone()
            raw[~lv] = 0x7F  # NaN
            pools[s] = raw.view(E4M3)
            pools[s + "_scale"] = torch.where(lv, sc, torch.tensor(float("nan")))
        else:
            vals[s] = x.double().numpy()
            pools[s] = torch.where(lv[..., None], x, torch.tensor(float("nan"), dtype=torch.bfloat16))
    if track:
        pools["weights"] = torch.rand(P, HK, page, generator=g)
        pools["positions"] = torch.from_numpy(rng.permutation(P * HK * page).astype(np.int32)).view(P, HK, page)
    dev = {n: t.to(gpu).contiguous() for n, t in pools.items()}
    cache = PagedKV(dev.pop("k"), dev.pop("v", None), **dev)
    return cache, vals, torch.from_numpy(table).to(gpu), table


def queries(gpu, seed, B, S, H, D, scale=1.0, strided=False):
    g = torch.Generator().manual_seed(seed + 1000)
    q = (torch.randn(B, S, H, D, generator=g) * scale).to(torch.bfloat16)
    if not strided:
        return q.to(gpu), q.double().numpy()
    rows = torch.full((B, S, (H + 2) * D), float("nan"), dtype=torch.bfloat16)
    rows[..., D:(H + 1) * D] = q.view(B, S, H * D)
    return rows.to(gpu)[..., D:(H + 1) * D].view(B, S, H, D), q.double().numpy()


def bounds(o, mag, reach, D):
    e32 = 2 * (D + 10) * 2.0 ** -24 * max(reach, 1.0) + 2.0 ** -20
    return 2.0 ** -8 * (np.abs(o) + mag) * 1.01 + e32 * mag + 1e-30, e32


def check(got, ref, D):
    o, mag, _, reach = ref
    tol, _ = bounds(o, mag, reach, D)
    err = np.abs(got.double().cpu().numpy() - o)
    assert np.isfinite(err).all(), "not finite"
    assert (err <= tol).all(), (float((err / tol).max()), np.unravel_index((err / tol).argmax(), err.shape))


LAYOUTS = [  # HK, g, D, shared
    (2, 4, 128, False), (8, 1, 128, False), (1, 16, 64, False), (2, 3, 64, False), (2, 5, 256, False),
    (1, 8, 128, True), (1, 20, 256, True), (1, 16, 512, True), (1, 64, 512, True),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, E4M3])
@pytest.mark.parametrize("HK,g,D,shared", LAYOUTS)
def test_attend_layouts(gpu, HK, g, D, shared, dtype):
    """Head layouts and widths, one token, ragged lengths among them 0 and 1, NaN in every slot
    that no sequence holds."""
    lens = [0, 1, 16, 17, 33, 64, 130, 700]
    cache, vals, tab, table = make(gpu, D + HK + g, lens, HK=HK, D=D, page=16, dtype=dtype, shared=shared)
    q, qd = queries(gpu, g, len(lens), 1, HK * g, D, strided=True)
    o = cache.attend(q, tab, torch.tensor(lens, dtype=torch.int32, device=gpu), D ** -0.5)
    check(o, op.attend(vals, qd, table, lens, D ** -0.5), D)
    assert (o[0] == 0).all()


@pytest.mark.parametrize("page", [16, 32, 64, 128, 1024])
@pytest.mark.parametrize("S", [1, 2, 4, 16])
def test_attend_pages_and_new_tokens(gpu, S, page):
    """Pages smaller and larger than a tile, several new tokens (rows of one, two and four tiles, and
    more than one group), lengths at and off the tiles' and granules' borders, a sink."""
    lens = [S, 0, 1, 31, 32, 128, 129, 257, 1000]
    HK, g, D = 2, 8, 64
    cache, vals, tab, table = make(gpu, S + page, lens, HK=HK, D=D, page=page)
    q, qd = queries(gpu, S, len(lens), S, HK * g, D, scale=1.5)
    sink = torch.linspace(-3, 4, HK * g)
    o = cache.attend(q, tab, torch.tensor(lens, dtype=torch.int32, device=gpu), D ** -0.5, attn_sink=sink.to(gpu))
    check(o, op.attend(vals, qd, table, lens, D ** -0.5, sink.double().numpy()), D)


@pytest.mark.parametrize("S,g,D,shared", [(1, 4, 128, False), (4, 8, 128, False), (3, 16, 256, False), (2, 64, 512, True)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, E4M3])
def test_attend_long(gpu, S, g, D, shared, dtype):
    """One long sequence over many workgroups, next to short ones."""
    lens = [4099, 5, 900] if D < 512 else [1500, 40]
    cache, vals, tab, table = make(gpu, S, lens, HK=1, D=D, page=64, dtype=dtype, shared=shared)
    q, qd = queries(gpu, S, len(lens), S, g, D, scale=2.0)
    o = cache.attend(q, tab, torch.tensor(lens, dtype=torch.int32, device=gpu), D ** -0.5)
    check(o, op.attend(vals, qd, table, lens, D ** -0.5), D)


def test_attend_running_maximum_moves(gpu):
    """Rows that grow along the sequence, so that the maximum moves far at many tiles."""
    lens, D = [900, 333], 128
    cache, vals, tab, table = make(gpu, 5, lens, HK=1, D=D, page=32)
    grow = torch.ones(cache.pages, 1, 32, 1)
    for b, n in enumerate(lens):
        for p in range(-(-n // 32)):
            grow[table[b, p]] = 2.0 ** (p // 4)
    k = (torch.from_numpy(vals["k"]) * grow).to(torch.bfloat16)
    cache.k.copy_(torch.where(torch.isnan(cache.k.cpu()), cache.k.cpu(), k).to(gpu))
    vals["k"] = k.double().numpy()
    q, qd = queries(gpu, 6, 2, 1, 4, D)
    o = cache.attend(q, tab, torch.tensor(lens, dtype=torch.int32, device=gpu), 0.3)
    check(o, op.attend(vals, qd, table, lens, 0.3), D)


@pytest.mark.parametrize("dtype", [torch.bfloat16, E4M3])
@pytest.mark.parametrize("page", [16, 64])
def test_attend_missing_pages_and_long_lengths(gpu, page, dtype):
    """Table entries below 0 and past the pool, at the start, inside and at the end; lengths beyond
    the table; negative ones."""
    lens = [page * 4, page * 4, page * 4 - 3, page * 2]
    HK, D = 2, 128
    cache, vals, tab, table = make(gpu, 9, lens, HK=HK, D=D, page=page, dtype=dtype)
    table[0, 0], table[0, 2], table[1, 3], table[1, 1] = -1, cache.pages, 2 ** 31 - 1, -(2 ** 31)
    table[3, :] = -1
    asked = [page * 9, page * 4, page * 4 - 3, page * 2]
    q, qd = queries(gpu, 3, 4, 2, HK * 2, D)
    o = cache.attend(q, torch.from_numpy(table).to(gpu), torch.tensor(asked, dtype=torch.int32, device=gpu), D ** -0.5)
    check(o, op.attend(vals, qd, table, asked, D ** -0.5), D)
    assert (o[3] == 0).all()
    o = cache.attend(q, tab, torch.tensor([-5, -1, 0, -2 ** 31], dtype=torch.int32, device=gpu), D ** -0.5)
    assert (o == 0).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, E4M3])
@pytest.mark.parametrize("HK,g,D,shared", [(2, 2, 64, False), (1, 16, 128, False), (2, 8, 256, False), (1, 6, 128, True),
                                           (1, 16, 512, True), (1, 64, 512, True)])
def test_attend_row_takes_nothing_from_tokens_it_does_not_see(gpu, HK, g, D, shared, dtype):
    """The newest tokens hold NaN (K of one, V of another): the rows before them stay finite, and the
    weights that every token gets are those of the formula."""
    lens, S = [200, 33, 3], 4
    cache, vals, tab, table = make(gpu, 13, lens, HK=HK, D=D, page=16, dtype=dtype, shared=shared, track=True)
    q, qd = queries(gpu, 4, len(lens), S, HK * g, D)
    ref = op.attend(vals, qd, table, lens, D ** -0.5)
    n = torch.tensor(lens, dtype=torch.int32, device=gpu)

    def poison(t, pool, b):
        row = pool[table[b, t // 16], :, t % 16]
        row.view(torch.uint8 if dtype == E4M3 else torch.int16).fill_(0x7F if dtype == E4M3 else 0x7FC0)

    if not shared:  # V alone: no score changes
        for b, m in enumerate(lens):
            poison(m - 2, cache.v, b)
        before = cache.weights.cpu().double().numpy()
        cache.attend(q, tab, n, D ** -0.5, accumulate=True)
        got = cache.weights.cpu().double().numpy()
        _, e32 = bounds(ref[0], ref[1], ref[3], D)
        assert (np.abs(got - before - ref[2]) <= e32 * ref[2] + 2.0 ** -23 * (np.abs(got) + 1e-30)).all()
    for b, m in enumerate(lens):
        poison(m - 1, cache.k, b)
        poison(m - 2, cache.k if shared else cache.v, b)
    o = cache.attend(q, tab, n, D ** -0.5)
    check(o[:, :2], tuple(x[:, :2] if i < 2 else x for i, x in enumerate(ref)), D)
    assert torch.isnan(o[:, 2:]).all()


def test_attend_infinite_values_and_scores(gpu):
    """An infinite value reaches its column only, as the formula has it; a row whose every score is
    -inf takes nothing; a NaN query row stays alone."""
    lens, HK, D = [77], 1, 128
    cache, vals, tab, table = make(gpu, 14, lens, HK=HK, D=D, page=32)
    q, qd = queries(gpu, 5, 1, 1, 4, D)
    cache.v[table[0, 2], 0, 76 % 32, 3] = float("inf")
    vals["v"][table[0, 2], 0, 76 % 32, 3] = np.inf
    n = torch.tensor(lens, dtype=torch.int32, device=gpu)
    o = cache.attend(q, tab, n, D ** -0.5)
    assert torch.isposinf(o[..., 3]).all()
    keep = [c for c in range(D) if c != 3]
    ref = op.attend(vals, qd, table, lens, D ** -0.5)
    check(o[..., keep], tuple(x[..., keep] if i < 2 else x for i, x in enumerate(ref)), D)
    q2 = q.clone()
    q2[0, 0, 1] = float("nan")
    o2 = cache.attend(q2, tab, n, D ** -0.5)
    assert torch.isnan(o2[0, 0, 1]).all()
    for h in (0, 2, 3):
        assert torch.equal(o2[0, 0, h], o[0, 0, h])
    # every visible key far along one axis, the query against it: all scores -inf
    cache.v.zero_()
    cache.k.zero_()
    cache.k[..., 0] = float("inf")
    q3 = torch.zeros_like(q)
    q3[..., 0] = -1.0
    cache.v[...] = 1.0
    assert (cache.attend(q3, tab, n, D ** -0.5) == 0).all()
    q3[...] = -1.0
    cache.k.fill_(float("inf"))
    assert (cache.attend(q3, tab, n, D ** -0.5) == 0).all()
    sink = torch.zeros(4, device=gpu)
    assert (cache.attend(q3, tab, n, D ** -0.5, attn_sink=sink) == 0).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, E4M3])
@pytest.mark.parametrize("S,HK,g,D,shared,page", [(1, 2, 4, 128, False, 16), (3, 2, 16, 64, False, 32), (1, 1, 64, 512, True, 64)])
def test_accumulated_weights(gpu, S, HK, g, D, shared, page, dtype):
    """Every slot's weight grows by what the rows of its head gave it, twice over; no other does."""
    lens = [1, 0, 100, 517, 2]
    cache, vals, tab, table = make(gpu, 21, lens, HK=HK, D=D, page=page, dtype=dtype, shared=shared, track=True)
    q, qd = queries(gpu, 22, len(lens), S, HK * g, D, scale=1.5)
    n = torch.tensor(lens, dtype=torch.int32, device=gpu)
    sink = torch.linspace(-1, 2, HK * g)
    for _ in range(2):
        before = cache.weights.cpu().double().numpy()
        o = cache.attend(q, tab, n, D ** -0.5, attn_sink=sink.to(gpu), accumulate=True)
        ref = op.attend(vals, qd, table, lens, D ** -0.5, sink.double().numpy())
        check(o, ref, D)
        _, e32 = bounds(ref[0], ref[1], ref[3], D)
        after = cache.weights.cpu().double().numpy()
        assert (np.abs(after - before - ref[2]) <= e32 * ref[2] + 2.0 ** -23 * (np.abs(after) + 1e-30)).all()
        assert (after[ref[2] == 0] == before[ref[2] == 0]).all()
    first = cache.weights.clone()
    cache.weights.zero_()
    cache.attend(q, tab, n, D ** -0.5, accumulate=True)
    again = cache.weights.clone()
    cache.weights.zero_()
    cache.attend(q, tab, n, D ** -0.5, accumulate=True)
    assert torch.equal(again, cache.weights) and not torch.equal(first, again)


def test_attend_pool_past_32_bits(gpu):
    """Pages whose rows lie past 4 GiB of each pool."""
    HK, D, page, P = 8, 128, 64, 36000
    k = torch.empty(P, HK, page, D, dtype=torch.bfloat16, device=gpu)
    v = torch.empty_like(k)
    ids = torch.tensor([P - 1, 3, P - 2, 17000, P - 7], device=gpu)
    g = torch.Generator(device=gpu).manual_seed(1)
    small_k = torch.randn(5, HK, page, D, device=gpu, generator=g).to(torch.bfloat16)
    small_v = torch.randn(5, HK, page, D, device=gpu, generator=g).to(torch.bfloat16)
    k[ids], v[ids] = small_k, small_v
    n = torch.tensor([5 * page - 9], dtype=torch.int32, device=gpu)
    q, _ = queries(gpu, 2, 1, 1, 32, D)
    o = PagedKV(k, v).attend(q, ids.to(torch.int32)[None], n, D ** -0.5)
    few = torch.arange(5, dtype=torch.int32, device=gpu)[None]
    assert torch.equal(o, PagedKV(small_k, small_v).attend(q, few, n, D ** -0.5))
    new = torch.randn(1, 2, HK, D, device=gpu, generator=g).to(torch.bfloat16)
    PagedKV(k, v).write(new, new, ids.to(torch.int32)[None], n)
    assert torch.equal(k[P - 7, :, 55:57], new[0].transpose(0, 1)) and torch.equal(v[P - 7, :, 55:57], new[0].transpose(0, 1))
    assert torch.equal(k[P - 7, :, :55], small_k[4, :, :55]) and torch.equal(k[P - 7, :, 57:], small_k[4, :, 57:])


# ---------------------------------------------------------------- write -------


def quantise(x):
    s = x.float().abs().amax(-1).clamp(min=1e-4) * (1.0 / 448.0)
    return (x.float() / s[..., None]).clamp(-448, 448).to(E4M3), s


@pytest.mark.parametrize("dtype", [torch.bfloat16, E4M3])
@pytest.mark.parametrize("HK,D,shared,page", [(2, 64, False, 16), (3, 128, False, 64), (1, 256, False, 32), (2, 128, True, 16),
                                             (1, 256, True, 128), (1, 512, True, 64)])
@pytest.mark.parametrize("S", [1, 37])
def test_write(gpu, S, HK, D, shared, page, dtype):
    """Rows land in their slots bit for bit (e4m3: codes and scales of the row), a padded batch's spare
    rows and slots without a page are dropped, and no other slot changes."""
    B, width = 6, 5
    cache = PagedKV.empty(B * width + 2, page, HK, D, dtype=dtype, shared=shared, track=True, device=gpu)
    rng = np.random.default_rng(S + D)
    table = rng.permutation(cache.pages)[:B * width].reshape(B, width).astype(np.int32)
    table[3, 1], table[4, 0] = -1, cache.pages
    start = np.array([0, 5, page - 1, page - 3, 2, width * page - 2], dtype=np.int32)
    count = np.array([S, max(0, S - 3), S, S, 0, S], dtype=np.int32)
    position = np.array([0, 100, 7, 2 ** 30, 1, 50], dtype=np.int32)
    g = torch.Generator().manual_seed(D)
    rows = torch.randn(B, S, 2 * HK * D + 8, generator=g).to(torch.bfloat16)
    rows[0, 0] = 0
    rows[1, :, :3] = 3e38
    dev = rows.to(gpu)
    k, v = dev[..., :HK * D].view(B, S, HK, D), dev[..., HK * D:2 * HK * D].view(B, S, HK, D)
    cache.weights.fill_(3.0)
    cache.positions.fill_(-7)
    to = lambda a: torch.from_numpy(a).to(gpu)  # noqa: E731
    for use_count, use_pos in ((True, True), (False, False)):
        want = {n: getattr(cache, n).cpu().clone() for n in ("k", "v", "k_scale", "v_scale", "weights", "positions")
                if getattr(cache, n) is not None}
        for b in range(B):
            for i in range(int(count[b]) if use_count else S):
                (pid, r), = op.slot_places(table[b], cache.pages, page, [int(start[b]) + i])
                if pid < 0:
                    continue
                for name, x in (("k", rows[b, i, :HK * D]),) + (() if shared else (("v", rows[b, i, HK * D:2 * HK * D]),)):
                    x = x.view(HK, D)
                    if dtype == E4M3:
                        code, s = quantise(x)
                        want[name].view(torch.uint8)[pid, :, r] = code.view(torch.uint8)
                        want[name + "_scale"][pid, :, r] = s
                    else:
                        want[name][pid, :, r] = x
                want["weights"][pid, :, r] = 0.0
                want["positions"][pid, :, r] = int(position[b] if use_pos else start[b]) + i
        cache.write(k, None if shared else v, to(table), to(start), count=to(count) if use_count else None,
                    position=to(position) if use_pos else None)
        for name, x in want.items():
            got = getattr(cache, name).cpu()
            if dtype == E4M3 and name in ("k", "v"):
                x, got = x.view(torch.uint8), got.view(torch.uint8)
            assert torch.equal(got, x), name
        start[:] = [9, 0, 1, 0, 3, 1]


def test_write_unaligned_rows(gpu):
    """Rows that do not begin on 16 bytes, and strides that are no multiple of eight."""
    cache = PagedKV.empty(4, 16, 2, 64, device=gpu)
    base = torch.randn(3 * (2 * 64 + 3) + 1, device=gpu).to(torch.bfloat16)[1:]
    k = base.view(1, 3, 2 * 64 + 3)[..., :128].unflatten(-1, (2, 64))
    table = torch.tensor([[2]], dtype=torch.int32, device=gpu)
    cache.write(k, k, table, torch.tensor([4], dtype=torch.int32, device=gpu))
    assert torch.equal(cache.k[2, :, 4:7], k[0].transpose(0, 1)) and torch.equal(cache.v[2, :, 4:7], k[0].transpose(0, 1))


# ---------------------------------------------------------------- evict -------


def arrays(cache):
    return {n: (t.view(torch.uint8) if t.dtype == E4M3 else t.view(torch.int16) if t.dtype == torch.bfloat16 else
                t.view(torch.int32) if n.endswith("_scale") else t).cpu().numpy().copy()
            for n in ("k", "v", "k_scale", "v_scale", "weights", "positions") if (t := getattr(cache, n)) is not None}


@pytest.mark.parametrize("dtype,HK,D,shared,page", [(torch.bfloat16, 2, 64, False, 16), (E4M3, 2, 128, False, 32),
                                                   (torch.bfloat16, 1, 512, True, 64), (E4M3, 1, 256, True, 16)])
@pytest.mark.parametrize("keep,first,recent", [(0, 0, 0), (1, 0, 1), (50, 4, 10), (64, 0, 0), (200, 200, 0), (1000, 3, 300),
                                              (1000, 0, 1000)])
@pytest.mark.parametrize("slots", [0, 9000])
def test_evict(gpu, dtype, HK, D, shared, page, keep, first, recent, slots):
    """The slots that stay, and where they lie, against the sorted order: ragged lengths around the budget,
    many equal weights, infinities and NaN among them, positions in any order.  A table of 9000 slots has
    several workgroups share a unit."""
    lens = [0, 1, keep, keep + 1, keep + 7, 2 * keep + 3, 1300]
    cache, _, tab, table = make(gpu, 3 + keep, lens, HK=HK, D=D, page=page, dtype=dtype, shared=shared, track=True,
                                width=max(-(-max(lens) // page), -(-slots // page)))
    g = torch.Generator().manual_seed(keep)
    w = torch.randint(0, 6, cache.weights.shape, generator=g).float() / 4
    w[torch.rand(w.shape, generator=g) < 0.05] = float("nan")
    w[torch.rand(w.shape, generator=g) < 0.02] = float("inf")
    w[torch.rand(w.shape, generator=g) < 0.02] = -0.0
    w[torch.rand(w.shape, generator=g) < 0.02] = -1.5
    cache.weights.copy_(w)
    for b, n in enumerate(lens):  # a sequence's positions are its own tokens, in any order
        for h in range(HK):
            p = torch.randperm(n + 5, generator=g)[:n].to(torch.int32)
            for t in range(n):
                cache.positions[table[b, t // page], h, t % page] = int(p[t]) if n < 400 else 3 * t
    want = arrays(cache)
    n = torch.tensor(lens, dtype=torch.int32, device=gpu)
    ref = op.evict(want, table, lens, keep, first, recent)
    got = cache.evict(tab, n, keep, first=first, recent=recent)
    assert np.array_equal(got.cpu().numpy(), ref) and n.tolist() == lens
    for name, x in arrays(cache).items():
        assert np.array_equal(x, want[name], equal_nan=name == "weights"), name


@pytest.mark.parametrize("slots", [0, 9000])
def test_evict_in_place_and_missing_pages(gpu, slots):
    """lens as its own output; pages that the table lacks lose first and are not moved."""
    lens, page, keep = [160, 90, 30], 16, 64
    cache, _, tab, table = make(gpu, 31, lens, HK=2, D=64, page=page, track=True, width=max(10, -(-slots // page)))
    table[0, 1], table[0, 9], table[1, 2] = -1, cache.pages + 5, -3
    want = arrays(cache)
    n = torch.tensor(lens, dtype=torch.int32, device=gpu)
    ref = op.evict(want, table, lens, keep, 2, 8)
    out = cache.evict(torch.from_numpy(table).to(gpu), n, keep, first=2, recent=8, out=n)
    assert out is n and np.array_equal(n.cpu().numpy(), ref)
    for name, x in arrays(cache).items():
        assert np.array_equal(x, want[name]), name


@pytest.mark.parametrize("n,keep", [(5000, 4096), (8200, 4000), (20000, 1500), (70001, 8192), (300000, 100000),
                                    (8192, 5000), (1025, 600)])
def test_evict_long(gpu, n, keep):
    """Lengths of many rounds of a workgroup, against torch's stable sort."""
    page, HK = 64, 2
    cache = PagedKV.empty(-(-n // page) + 1, page, HK, 64, track=True, device=gpu)
    g = torch.Generator().manual_seed(n)
    table = torch.randperm(cache.pages, generator=g)[:-(-n // page)].to(torch.int32)[None].to(gpu)
    cache.weights.copy_(torch.randn(cache.weights.shape, generator=g).mul(8).round().div(8).exp())
    slot = torch.arange(table.shape[1] * page, dtype=torch.int32, device=gpu).view(-1, page)
    cache.positions[table[0].long()] = slot[:, None, :].expand(-1, HK, page).contiguous()
    cache.k[..., 0] = cache.positions.to(torch.bfloat16)
    cache.k.view(torch.int16)[..., 1] = (cache.positions & 0x7FFF).to(torch.int16)
    flat = lambda x: x[table[0].long()].transpose(0, 1).reshape(HK, -1)  # noqa: E731
    w, p = flat(cache.weights), flat(cache.positions)
    first, recent = 4, 512
    safe = (p < first) | (p >= n - recent)
    key = torch.where(safe, torch.tensor(float("inf"), device=gpu), w)
    key[:, n:] = -1
    order = torch.sort(key, dim=1, descending=True, stable=True).indices
    kept = torch.zeros_like(safe).scatter_(1, order[:, :keep], True)
    out = cache.evict(table, torch.tensor([n], dtype=torch.int32, device=gpu), keep, first=first, recent=recent)
    assert out.tolist() == [keep]
    after = flat(cache.positions)
    for h in range(HK):
        want = torch.arange(table.shape[1] * page, dtype=torch.int32, device=gpu)
        holes, movers = torch.nonzero(~kept[h, :keep])[:, 0], torch.nonzero(kept[h, keep:])[:, 0] + keep
        want[holes] = movers.to(torch.int32)
        assert torch.equal(after[h], want)
    assert torch.equal(flat(cache.weights), torch.gather(w, 1, after.long()))
    low = cache.k.view(torch.int16)[..., 1]
    assert torch.equal(flat(low), (after & 0x7FFF).to(torch.int16))


@pytest.mark.parametrize("inplace", [False, True])
@pytest.mark.parametrize("slots", [0, 9000])
def test_evict_keeps_protected_slots_beside_missing_pages(gpu, slots, inplace):
    """What ``first`` and ``recent`` protect stays below the new length wherever pages are missing, as long as the
    pages below keep hold as many; no page below keep at all leaves everything where it is.  A page's slots of
    NaN weight count, and are the first to go."""
    lens, page, keep, first, recent = [300, 200, 120, 97], 16, 96, 6, 20
    cache, _, _, table = make(gpu, 33, lens, HK=2, D=64, page=page, track=True, width=max(19, -(-slots // page)))
    for b, n in enumerate(lens):
        for t in range(n):
            cache.positions[table[b, t // page], :, t % page] = (7 * t + 3) % n if b else t
    cache.weights[table[1, 3]] = float("nan")
    table[0, 1], table[0, 4] = -1, cache.pages
    table[1, 2], table[1, 9] = -1, -1
    table[2, :6] = -1
    want = arrays(cache)
    n = torch.tensor(lens, dtype=torch.int32, device=gpu)
    ref = op.evict(want, table, lens, keep, first, recent)
    got = cache.evict(torch.from_numpy(table).to(gpu), n, keep, first=first, recent=recent, out=n if inplace else None)
    assert np.array_equal(got.cpu().numpy(), ref)
    after = arrays(cache)
    for name, x in after.items():
        assert np.array_equal(x, want[name], equal_nan=name == "weights"), name
    pos = after["positions"]
    held = [[set(pos[table[b, t // page], h, t % page] for t in range(keep) if 0 <= table[b, t // page] < cache.pages)
             for h in range(2)] for b in range(4)]
    for h in range(2):
        assert set(range(first)) | set(range(300 - recent, 300)) <= held[0][h]
        gone = {(7 * t + 3) % 200 for t in [*range(32, 48), *range(144, 160)]}
        newest = max(p for p in range(200) if p not in gone)
        assert {p for p in [*range(first), *range(newest - recent + 1, newest + 1)] if p not in gone} <= held[1][h]
        assert not held[2][h]


# ---------------------------------------------------------------- together ----


@pytest.mark.parametrize("dtype,S", [(torch.bfloat16, 1), (E4M3, 3)])
def test_decode_under_a_budget(gpu, dtype, S):
    """A prompt's write, then steps of write, attend and evict as a serving loop makes them, against
    a cache that the plain statements keep (its choice of what stays is made from the same weights)."""
    B, HK, g, D, page, keep = 3, 2, 4, 64, 16, 48
    width = 6
    cache = PagedKV.empty(B * width, page, HK, D, dtype=dtype, track=True, device=gpu)
    rng = np.random.default_rng(1)
    table = rng.permutation(B * width).reshape(B, width).astype(np.int32)
    tab = torch.from_numpy(table).to(gpu)
    plain = {"k": np.zeros((B * width, HK, page, D)), "v": np.zeros((B * width, HK, page, D)),
             "weights": np.zeros((B * width, HK, page)), "positions": np.zeros((B * width, HK, page), dtype=np.int64)}
    gen = torch.Generator().manual_seed(2)
    lens, pos = np.zeros(B, dtype=np.int32), np.zeros(B, dtype=np.int32)
    n = torch.zeros(B, dtype=torch.int32, device=gpu)
    p = torch.zeros(B, dtype=torch.int32, device=gpu)
    for step in range(14):
        s = 30 if step == 0 else S
        count = np.array([30, 7, 0], dtype=np.int32) if step == 0 else np.full(B, s, dtype=np.int32)
        k = torch.randn(B, s, HK, D, generator=gen).to(torch.bfloat16)
        v = torch.randn(B, s, HK, D, generator=gen).to(torch.bfloat16)
        c = torch.from_numpy(count).to(gpu)
        cache.write(k.to(gpu), v.to(gpu), tab, n, count=c, position=p)
        for b in range(B):
            for i in range(count[b]):
                (pid, r), = op.slot_places(table[b], B * width, page, [int(lens[b]) + i])
                for name, x in (("k", k), ("v", v)):
                    x = x[b, i]
                    if dtype == E4M3:
                        code, sc = quantise(x)
                        x = code.double() * sc.double()[:, None]
                    plain[name][pid, :, r] = x.double().numpy()
                plain["weights"][pid, :, r], plain["positions"][pid, :, r] = 0.0, pos[b] + i
        lens, pos = lens + count, pos + count
        n, p = n + c, p + c
        if step == 0:
            continue
        q, qd = queries(gpu, step, B, S, HK * g, D, scale=2.0)
        o = cache.attend(q, tab, n, D ** -0.5, accumulate=True)
        ref = op.attend(plain, qd, table, lens, D ** -0.5)
        check(o, ref, D)
        plain["weights"] += ref[2]
        got = cache.weights.cpu().numpy()
        assert np.abs(got - plain["weights"]).max() < 1e-4
        plain["weights"] = got.astype(np.float64)  # what stays is chosen from the cache's own sums
        n = cache.evict(tab, n, keep, first=2, recent=8)
        lens = op.evict(plain, table, lens, keep, 2, 8)
        assert np.array_equal(n.cpu().numpy(), lens)
        assert np.array_equal(cache.positions.cpu().numpy(), plain["positions"])


def test_captured_loop_replays(gpu):
    """Write, attend and evict captured as one graph and replayed, with eager work on the same cache and
    other streams between the replays: every replay equals the eager result."""
    HK, g, D, page, keep = 2, 4, 128, 16, 96
    lens = [96, 50, 0]
    cache, _, tab, _ = make(gpu, 41, lens, HK=HK, D=D, page=page, track=True, width=8, spare=40)
    tab = torch.arange(24, dtype=torch.int32, device=gpu).view(3, 8)
    for t in (cache.k, cache.v):
        t.copy_(torch.randn(t.shape, device=gpu))
    q, _ = queries(gpu, 1, 3, 1, HK * g, D)
    k = torch.randn(3, 1, HK, D, device=gpu).to(torch.bfloat16)
    n = torch.tensor(lens, dtype=torch.int32, device=gpu)
    start = torch.empty_like(n)

    def step():
        cache.write(k, k, tab, n, position=p)
        m = n + 1
        o = cache.attend(q, tab, m, D ** -0.5, accumulate=True)
        n.copy_(cache.evict(tab, m, keep, first=2, recent=4))
        p.add_(1)
        return o

    held = (cache.k, cache.v, cache.weights, cache.positions, n)
    p = n.clone()
    held += (p,)
    saved = [t.clone() for t in held]
    want = []
    for i in range(5):
        k.fill_(0.1 * i)
        want.append((step().clone(), *[t.clone() for t in held]))
    for t, x in zip(held, saved):
        t.copy_(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = step()
    for t, x in zip(held, saved):
        t.copy_(x)
    other = torch.cuda.Stream()
    for i in range(5):
        k.fill_(0.1 * i)
        graph.replay()
        torch.cuda.synchronize()
        for a, x in zip((o, *held), want[i]):
            assert torch.equal(a, x)
        with torch.cuda.stream(other):  # eager work of the same kind between the replays
            e = cache.attend(q, tab, n, D ** -0.5)
        torch.cuda.synchronize()
        assert torch.equal(e, cache.attend(q, tab, n, D ** -0.5))


def test_two_streams_at_once(gpu):
    """Two calls in flight on two streams, each with its own workspace."""
    HK, D = 4, 128
    cache, vals, tab, table = make(gpu, 51, [3000, 2000, 900], HK=HK, D=D, page=64)
    n = torch.tensor([3000, 2000, 900], dtype=torch.int32, device=gpu)
    q1, _ = queries(gpu, 1, 3, 1, 16, D)
    q2, _ = queries(gpu, 2, 3, 1, 16, D)
    a, b = cache.attend(q1, tab, n, D ** -0.5), cache.attend(q2, tab, n, D ** -0.5)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(10):
        with torch.cuda.stream(s1):
            x = cache.attend(q1, tab, n, D ** -0.5)
        with torch.cuda.stream(s2):
            y = cache.attend(q2, tab, n, D ** -0.5)
        torch.cuda.synchronize()
        assert torch.equal(x, a) and torch.equal(y, b)


def test_workspace_and_outputs_of_the_caller(gpu):
    """A given workspace and out are used; two graphs that share a workspace replay one after the other."""
    HK, D = 2, 128
    cache, _, tab, _ = make(gpu, 61, [700, 45], HK=HK, D=D, page=32, track=True)
    n = torch.tensor([700, 45], dtype=torch.int32, device=gpu)
    q, _ = queries(gpu, 1, 2, 1, 8, D)
    want = cache.attend(q, tab, n, D ** -0.5)
    ws = torch.empty(cache.attend_workspace_bytes(2, 1, 8, tab.shape[1]), dtype=torch.uint8, device=gpu)
    out = torch.empty_like(want)
    assert cache.attend(q, tab, n, D ** -0.5, out=out, workspace=ws) is out and torch.equal(out, want)
    q2 = q.flip(2).contiguous()
    want2 = cache.attend(q2, tab, n, D ** -0.5)
    graphs, outs = [], []
    for x in (q, q2):
        graphs.append(torch.cuda.CUDAGraph())
        outs.append(torch.empty_like(out))
        with torch.cuda.graph(graphs[-1]):
            cache.attend(x, tab, n, D ** -0.5, out=outs[-1], workspace=ws)
    for _ in range(3):
        for t in outs:
            t.zero_()
        graphs[0].replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want) and torch.equal(outs[1], want2)


# ---------------------------------------------------------------- the calls at the edges ----


@pytest.mark.parametrize("dtype", [torch.bfloat16, E4M3])
@pytest.mark.parametrize("B,HK,g,D,shared", [(300, 8, 2, 64, False), (600, 2, 3, 128, False), (300, 1, 16, 512, True)])
def test_more_sequences_than_workers(gpu, B, HK, g, D, shared, dtype):
    """More (sequence, head) units than the chip has workers, most of them short and every seventh empty; the
    weights as well."""
    rng = np.random.default_rng(B)
    lens = [0 if b % 7 == 0 else int(n) for b, n in enumerate(rng.integers(1, 70, B))]
    cache, vals, tab, table = make(gpu, B, lens, HK=HK, D=D, page=16, dtype=dtype, shared=shared, track=True)
    q, qd = queries(gpu, g, B, 1, HK * g, D)
    n = torch.tensor(lens, dtype=torch.int32, device=gpu)
    ref = op.attend(vals, qd, table, lens, D ** -0.5)
    before = cache.weights.cpu().double().numpy()
    o = cache.attend(q, tab, n, D ** -0.5, accumulate=True)
    check(o, ref, D)
    _, e32 = bounds(ref[0], ref[1], ref[3], D)
    after = cache.weights.cpu().double().numpy()
    assert (np.abs(after - before - ref[2]) <= e32 * ref[2] + 2.0 ** -23 * (np.abs(after) + 1e-30)).all()
    assert torch.equal(cache.attend(q, tab, n, D ** -0.5), o)


@pytest.mark.parametrize("dtype", [torch.bfloat16, E4M3])
@pytest.mark.parametrize("S,g,D,shared", [(16, 24, 128, False), (16, 9, 64, False), (5, 30, 256, True), (16, 20, 512, True)])
def test_many_rows_of_a_head(gpu, S, g, D, shared, dtype):
    """More rows of a KV head than a group holds, lengths shorter than the new tokens, the weights and their
    fixed order."""
    lens = [S - 1, 700, 0, 64]
    cache, vals, tab, table = make(gpu, S + g, lens, HK=1, D=D, page=32, dtype=dtype, shared=shared, track=True)
    q, qd = queries(gpu, g, len(lens), S, g, D)
    n = torch.tensor(lens, dtype=torch.int32, device=gpu)
    ref = op.attend(vals, qd, table, lens, D ** -0.5)
    cache.weights.zero_()
    check(cache.attend(q, tab, n, D ** -0.5, accumulate=True), ref, D)
    _, e32 = bounds(ref[0], ref[1], ref[3], D)
    once = cache.weights.clone()
    w = once.cpu().double().numpy()
    # a sum of S g float32 terms of at most 1
    assert (np.abs(w - ref[2]) <= (e32 + S * g * 2.0 ** -24) * ref[2] + 1e-30).all()
    cache.weights.zero_()
    cache.attend(q, tab, n, D ** -0.5, accumulate=True)
    assert torch.equal(once, cache.weights)


def test_nothing_to_do(gpu):
    """No sequences, no new tokens, a table without pages, only empty sequences: zeros, and nothing changes."""
    cache, _, tab, _ = make(gpu, 71, [40, 20], HK=2, D=64, page=16, track=True)
    want = arrays(cache)
    n = torch.tensor([40, 20], dtype=torch.int32, device=gpu)
    none, no_table = n[:0], tab[:, :0]
    q = torch.randn(2, 1, 4, 64, device=gpu).to(torch.bfloat16)
    k = torch.randn(2, 3, 2, 64, device=gpu).to(torch.bfloat16)
    assert cache.attend(q[:0], tab[:0], none, 0.1).shape == (0, 1, 4, 64)
    assert cache.attend(q[:, :0], tab, n, 0.1).shape == (2, 0, 4, 64)
    assert (cache.attend(q, no_table, n, 0.1, accumulate=True) == 0).all()
    assert (cache.attend(q, tab, torch.zeros_like(n), 0.1, accumulate=True) == 0).all()
    assert (cache.attend(q, tab, -n, 0.1, accumulate=True) == 0).all()
    cache.write(k[:0], k[:0], tab[:0], none)
    cache.write(k[:, :0], k[:, :0], tab, n)
    cache.write(k, k, no_table, n)
    cache.write(k, k, tab, n, count=-n)
    cache.write(k, k, tab, torch.full_like(n, -7))
    cache.write(k, k, tab, torch.full_like(n, 2 ** 31 - 2))
    assert cache.evict(tab[:0], none, 5).shape == (0,)
    assert cache.evict(no_table, n, 7).tolist() == [7, 7]
    assert cache.evict(tab, n, 100).tolist() == [40, 20]
    assert cache.evict(tab, n, 2 ** 31 - 1, first=5, recent=2 ** 31 - 6).tolist() == [40, 20]
    for name, x in arrays(cache).items():
        assert np.array_equal(x, want[name], equal_nan=name == "weights"), name


def test_write_counts_past_the_rows(gpu):
    """A count above the rows given means all of them."""
    cache = PagedKV.empty(4, 16, 2, 64, device=gpu)
    k = torch.randn(1, 3, 2, 64, device=gpu).to(torch.bfloat16)
    one = lambda x: torch.tensor([x], dtype=torch.int32, device=gpu)  # noqa: E731
    cache.write(k, k, torch.tensor([[2]], dtype=torch.int32, device=gpu), one(-1), count=one(2 ** 31 - 1))
    assert torch.equal(cache.k[2, :, :2], k[0, 1:].transpose(0, 1)) and not cache.k[2, :, 2:].any() and not cache.k[:2].any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, E4M3])
def test_write_negative_counts_of_many_tokens(gpu, dtype):
    """A negative count means no rows, down to -2^31, also for the tokens behind a workgroup's first."""
    B, S, HK, D, page = 6, 70, 2, 64, 16  # 32 tokens a workgroup
    cache = PagedKV.empty(B * 8, page, HK, D, dtype=dtype, track=True, device=gpu)
    cache.weights.fill_(3.0)
    want = arrays(cache)
    k = torch.randn(B, S, HK, D, device=gpu).to(torch.bfloat16)
    table = torch.arange(B * 8, dtype=torch.int32, device=gpu).view(B, 8)
    start = torch.full((B,), 5, dtype=torch.int32, device=gpu)
    low = -2 ** 31
    cache.write(k, k, table, start, torch.tensor([low, low + 1, low + 31, low + 33, -1, -70], dtype=torch.int32, device=gpu))
    for name, x in arrays(cache).items():
        assert np.array_equal(x, want[name]), name


def test_captured_cut_of_long_sequences(gpu):
    """Units that several workgroups share, cut in a captured graph: every replay equals the eager call."""
    page, HK, n, keep = 64, 2, 12000, 1000
    cache = PagedKV.empty(200, page, HK, 64, track=True, device=gpu)
    table = torch.randperm(200, generator=torch.Generator().manual_seed(5))[:188].to(torch.int32)[None].to(gpu)
    lens = torch.tensor([n], dtype=torch.int32, device=gpu)
    graph, out = torch.cuda.CUDAGraph(), torch.empty_like(lens)

    def fill(seed):
        g = torch.Generator(device=gpu).manual_seed(seed)
        cache.weights.copy_(torch.rand(cache.weights.shape, generator=g, device=gpu))
        cache.k.copy_(torch.randn(cache.k.shape, generator=g, device=gpu))
        slot = torch.arange(188 * page, dtype=torch.int32, device=gpu).view(188, 1, page)
        cache.positions[table[0].long()] = slot.expand(-1, HK, -1).contiguous()

    fill(0)
    cache.evict(table, lens, keep, 4, 100)
    fill(0)
    with torch.cuda.graph(graph):
        cache.evict(table, lens, keep, 4, 100, out=out)
    for seed in range(4):
        fill(seed)
        cache.evict(table, lens, keep, 4, 100)
        want = arrays(cache)
        fill(seed)
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert out.tolist() == [keep]
        for name, x in arrays(cache).items():
            assert np.array_equal(x, want[name]), (seed, name)


def test_refusals_with_device_tensors(gpu):
    """What does not fit is refused before a kernel runs."""
    cache, _, tab, _ = make(gpu, 81, [40, 20], HK=2, D=64, page=16, track=True)
    want = arrays(cache)
    n = torch.tensor([40, 20], dtype=torch.int32, device=gpu)
    q = torch.randn(2, 1, 4, 64, device=gpu).to(torch.bfloat16)
    ws = torch.empty(16, dtype=torch.uint8, device=gpu)
    for kw, error, what in (
            (dict(q=q.float()), TypeError, "bf16 q"), (dict(q=q[..., :32]), ValueError, "q must be"),
            (dict(q=q[:, :, :3]), N.WzError, "3 heads on 2"), (dict(q=q.expand(2, 17, 4, 64)), N.WzError, "S=17"),
            (dict(q=q.cpu()), ValueError, "q is on cpu"), (dict(table=tab.long()), ValueError, "table must be int32"),
            (dict(table=tab[:1]), ValueError, "table must be int32"), (dict(table=tab.cpu()), ValueError, "table is on cpu"),
            (dict(lens=n.long()), ValueError, "lens must be int32"), (dict(lens=n.cpu()), ValueError, "lens is on cpu"),
            (dict(attn_sink=torch.zeros(3, device=gpu)), ValueError, "attn_sink"),
            (dict(out=torch.empty(2, 1, 4, 64, device=gpu)), ValueError, "out must be"),
            (dict(workspace=ws), N.WzError, "workspace of 16 bytes"), (dict(workspace=ws.float()), ValueError, "workspace must be")):
        args = {**dict(q=q, table=tab, lens=n, softmax_scale=0.1), **kw}
        with pytest.raises(error, match=what):
            cache.attend(**args)
    k = torch.randn(2, 3, 2, 64, device=gpu).to(torch.bfloat16)
    for kw, error, what in ((dict(v=None), ValueError, "v is given"), (dict(v=k[:, :2]), ValueError, "does not match"),
                            (dict(k=k[..., :32]), ValueError, "k must be"), (dict(k=k.half(), v=k.half()), TypeError, "bf16 k"),
                            (dict(start=n[:1]), ValueError, "start must be"), (dict(count=n.float()), ValueError, "count must be"),
                            (dict(position=n.cpu()), ValueError, "position is on cpu")):
        with pytest.raises(error, match=what):
            cache.write(**{**dict(k=k, v=k, table=tab, start=n), **kw})
    for kw, error, what in ((dict(keep=-1), N.WzError, "keep -1"), (dict(keep=5, first=3, recent=3), N.WzError, "first 3"),
                            (dict(keep=5, out=n[:1]), ValueError, "out must be"),
                            (dict(keep=5, lens=n.view(1, 2)), ValueError, "table must be"),
                            (dict(keep=5, workspace=ws[:0]), N.WzError, "workspace of")):
        with pytest.raises(error, match=what):
            cache.evict(**{**dict(table=tab, lens=n), **kw})
    with pytest.raises(ValueError, match="contiguous"):
        PagedKV(cache.k[:, :1], cache.v[:, :1])
    plain = PagedKV(cache.k, cache.v)
    with pytest.raises(ValueError, match="not tracked"):
        plain.evict(tab, n, 5)
    with pytest.raises(N.WzError, match="not tracked"):
        plain.attend(q, tab, n, 0.1, accumulate=True)
    for name, x in arrays(cache).items():
        assert np.array_equal(x, want[name], equal_nan=name == "weights"), name


@pytest.mark.parametrize("HK,D,shared", [(2, 64, False), (1, 128, False), (1, 512, True)])
def test_write_of_rows_that_are_not_finite(gpu, HK, D, shared):
    """An e4m3 row follows act_quant's arithmetic: with an infinity its scale is inf and the infinity's code NaN,
    with a NaN all of it is NaN, a row of tiny values has the floor's scale; other rows are not touched by it."""
    cache = PagedKV.empty(4, 16, HK, D, dtype=E4M3, shared=shared, track=True, device=gpu)
    x = torch.randn(1, 9, HK, D, generator=torch.Generator().manual_seed(D)).to(torch.bfloat16)
    inf, nan = float("inf"), float("nan")
    x[0, 1, 0, D - 1], x[0, 3, 0, 0], x[0, 4, HK - 1, 9] = inf, -inf, nan
    x[0, 5, 0, 3], x[0, 5, 0, 4] = inf, nan
    x[0, 6] = 3.3e38
    x[0, 7] *= 1e-38
    x[0, 8] = 0
    one = lambda n: torch.tensor([n], dtype=torch.int32, device=gpu)  # noqa: E731
    cache.write(x.to(gpu), None if shared else x.to(gpu), one(3)[None], one(2))
    code, s = quantise(x)
    for pool, scale in ((cache.k, cache.k_scale),) + (() if shared else ((cache.v, cache.v_scale),)):
        got, want = pool[3, :, 2:11].cpu().float(), code[0].transpose(0, 1).float()
        assert torch.equal(scale[3, :, 2:11].cpu().nan_to_num(-1), s[0].t().nan_to_num(-1))
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        assert torch.equal(got.nan_to_num(0), want.nan_to_num(0))
        assert torch.isnan(got).any(-1).sum(0).tolist() == [0, 1, 0, 1, 1, 1, 0, 0, 0]
        assert not pool[:3].view(torch.uint8).any() and not pool[3, :, :2].view(torch.uint8).any()


def test_calls_with_workspace_and_out_allocate_nothing(gpu):
    """Contiguous int32 tables and lengths, aligned rows, out and workspace given: no device memory is asked for."""
    B, HK, H, D, page = 3, 2, 8, 128, 16
    cache = PagedKV.empty(3 * 600, page, HK, D, track=True, device=gpu)
    for width in (20, 600):  # eviction by one workgroup a unit, and by several
        table = torch.arange(B * width, dtype=torch.int32, device=gpu).view(B, width)
        lens = torch.tensor([100, 250, 9], dtype=torch.int32, device=gpu)
        rows = torch.randn(B, 2, (H + 2 * HK) * D, device=gpu).to(torch.bfloat16)
        q, k, v = (t.unflatten(-1, (-1, D)) for t in rows.split([H * D, HK * D, HK * D], -1))
        o, new, sink = torch.empty(B, 2, H, D, dtype=torch.bfloat16, device=gpu), torch.empty_like(lens), torch.zeros(H, device=gpu)
        ws = torch.empty(max(cache.attend_workspace_bytes(B, 2, H, width, True), cache.evict_workspace_bytes(B, width, 64)),
                         dtype=torch.uint8, device=gpu)

        def calls():
            cache.write(k, v, table, lens, position=lens)
            cache.attend(q, table, lens, 0.1, sink, accumulate=True, out=o, workspace=ws)
            cache.attend(q, table, lens, 0.1, out=o, workspace=ws)
            cache.evict(table, lens, 64, 2, 8, out=new, workspace=ws)

        calls()
        torch.cuda.synchronize()
        before = torch.cuda.memory_stats(gpu)["allocation.all.allocated"]
        calls()
        torch.cuda.synchronize()
        assert torch.cuda.memory_stats(gpu)["allocation.all.allocated"] == before


@pytest.mark.parametrize("dtype", [torch.bfloat16, E4M3])
@pytest.mark.parametrize("HK,g,D,shared", [(2, 4, 64, False), (1, 16, 512, True)])
def test_a_wide_table_changes_nothing(gpu, HK, g, D, shared, dtype):
    """The loop of write, attend and evict with a table far wider than its sequences (the cut then goes by
    chunks, the workspaces grow): bit for bit that of a narrow table."""
    B, page, keep, steps = 3, 16, 80, 12
    narrow = PagedKV.empty(B * 8, page, HK, D, dtype=dtype, shared=shared, track=True, device=gpu)
    wide = PagedKV.empty(B * 8, page, HK, D, dtype=dtype, shared=shared, track=True, device=gpu)
    tables = [torch.arange(B * 8, dtype=torch.int32, device=gpu).view(B, 8).flip(1).contiguous()]
    tables.append(torch.cat([tables[0], torch.full((B, 700), -1, dtype=torch.int32, device=gpu)], 1))
    n = [torch.zeros(B, dtype=torch.int32, device=gpu) for _ in range(2)]
    pos = torch.zeros(B, dtype=torch.int32, device=gpu)
    gen = torch.Generator(device=gpu).manual_seed(D)
    for step in range(steps):
        s = 70 if step == 0 else 2
        k = torch.randn(B, s, HK, D, device=gpu, generator=gen).to(torch.bfloat16)
        q = torch.randn(B, min(s, 2), HK * g, D, device=gpu, generator=gen).to(torch.bfloat16)
        count = torch.tensor([s, s // 2, s], dtype=torch.int32, device=gpu)
        out = []
        for i, (c, t) in enumerate(zip((narrow, wide), tables)):
            c.write(k, None if shared else k.flip(3).contiguous(), t, n[i], count=count, position=pos)
            n[i] = n[i] + count
            out.append(c.attend(q, t, n[i], D ** -0.5, accumulate=True))
            n[i] = c.evict(t, n[i], keep, first=2, recent=10)
        pos = pos + count
        assert torch.equal(*out) and torch.equal(*n)
        for name, x in arrays(narrow).items():
            assert np.array_equal(x, arrays(wide)[name], equal_nan=name == "weights"), (step, name)
    assert n[0].tolist() == [keep, 46, keep] and pos.tolist() == [92, 46, 92]
