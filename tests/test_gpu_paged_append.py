"""PagedKV.append and accept against their 64-bit statements.

Tolerances of append, per element: one rounding to bf16, 2^-8 |x|, and the 32-bit arithmetic before it: the sum of D
squares and its root, 2^-24 (D / 16 + 16) relative, then products with the norm and the turn, 2^-22 of the pair's
larger element.  An e4m3 row's scale is amax / 448 with that arithmetic; a code is off by half a step of its
binade, 2^-4 relative or 2^-10 of the scale among the subnormals, and what the scale's error moves."""

import numpy as np
import pytest
import torch

from oracle import paged as op
from tests.test_gpu_paged import E4M3
from wanferenz_amd.paged import PagedKV

pytestmark = pytest.mark.gpu
F32 = 2.0 ** -18  # of the pair's larger element; 48 + 16 steps of 2^-24 for D = 512 and the turn


def i32(x, gpu):
    return torch.tensor(x, dtype=torch.int32, device=gpu)


def setup(gpu, seed, starts, S, H, HK, D, page, dtype, shared, track=False):
    need = [-(-(max(s, 0) + S) // page) for s in starts]
    P = sum(need) + 2
    cache = PagedKV.empty(P, page, HK, D, dtype=dtype, shared=shared, track=track, device=gpu)
    rng = np.random.default_rng(seed)
    order, at = rng.permutation(P), 0
    table = np.full((len(starts), max(need)), -1, dtype=np.int32)
    for b, c in enumerate(need):
        table[b, :c] = order[at:at + c]
        at += c
    g = torch.Generator().manual_seed(seed)
    width = H + (1 if shared else 2) * HK
    rows = torch.randn(len(starts), S, width * D, generator=g).mul_(1.7).to(torch.bfloat16)
    dev = rows.to(gpu)
    parts = [(dev[..., a * D:e * D].view(len(starts), S, e - a, D), rows[..., a * D:e * D].view(len(starts), S, e - a, D))
             for a, e in ((0, H), (H, H + HK), (H + HK, width))]
    return cache, table, parts, g


def close(got, want, big, rel=2.0 ** -8):
    err = np.abs(got - want)
    tol = rel * np.abs(want) + F32 * big + 1e-30
    assert (err <= tol).all(), float((err / tol).max())


def pair_max(x, R, halves, leading):
    """The larger magnitude of each element's pair (its own where it is not turned)."""
    y = np.abs(x).copy()
    lo = 0 if leading else x.shape[-1] - R
    pair = np.arange(R // 2)
    i = lo + (pair if halves else 2 * pair)
    j = i + (R // 2 if halves else 1)
    m = np.maximum(y[..., i], y[..., j]) * 1.5
    y[..., i], y[..., j] = m, m
    return y


@pytest.mark.parametrize("dtype", [torch.bfloat16, E4M3])
@pytest.mark.parametrize("H,HK,D,R,shared,page", [
    (8, 2, 128, 128, False, 16), (3, 3, 64, 32, False, 32), (4, 1, 256, 64, False, 16), (5, 1, 512, 64, True, 64),
    (2, 2, 128, 16, True, 16), (7, 1, 64, 64, False, 16), (6, 2, 256, 240, False, 16), (4, 1, 512, 512, True, 16)])
@pytest.mark.parametrize("halves,leading", [(False, False), (True, True), (False, True), (True, False)])
def test_append(gpu, halves, leading, H, HK, D, R, shared, page, dtype):
    starts, S = [0, 5, 29, 40], 7
    cache, table, parts, g = setup(gpu, D + R + H, starts, S, H, HK, D, page, dtype, shared, track=True)
    cache.weights.fill_(3.0)
    qn, kn = (1 + 0.3 * torch.randn(D, generator=g) for _ in range(2))
    ang = torch.randn(60, R // 2, generator=g, dtype=torch.float64) * 3
    freqs = torch.polar(torch.ones_like(ang), ang).to(torch.complex64)
    before = {n: getattr(cache, n).clone() for n in ("k", "v", "k_scale", "v_scale") if getattr(cache, n) is not None}
    count = [7, 7, 3, 0]
    (q, qc), (k, kc), (v, vc) = parts
    o = cache.append(q, k, None if shared else v, torch.from_numpy(table).to(gpu), i32(starts, gpu), freqs.to(gpu),
                     count=i32(count, gpu), position=i32([1, 50, 20, 9], gpu), q_norm=qn.to(gpu), k_norm=kn.to(gpu),
                     eps=1e-5, halves=halves, leading=leading)
    assert o.is_contiguous() and o.dtype == torch.bfloat16
    z = freqs.to(torch.complex128).numpy()
    pos = np.array([1, 50, 20, 9])[:, None] + np.arange(S)
    want = {}
    for name, x, w, heads in (("q", qc, qn, H), ("k", kc, kn, HK)):
        x = op.turned(x.double().numpy(), w.double().numpy(), 1e-5, np.ones((1, 1, 1, 8)), True, True)
        want[name] = (op.turned(x, None, 0, z[pos][:, :, None], halves, leading), pair_max(x, R, halves, leading))
    if not shared:
        want["v"] = (vc.double().numpy(), np.zeros(()))
    live = np.arange(S)[None] < np.array(count)[:, None]
    close(o.double().cpu().numpy() * live[..., None, None], want["q"][0] * live[..., None, None], want["q"][1])
    assert (o.cpu()[torch.from_numpy(~live)] == 0).all()
    touched = torch.zeros(cache.pages, HK, page, dtype=torch.bool)
    for name in [n for n in ("k", "v") if n in want]:
        pool = getattr(cache, name).cpu()
        sc = getattr(cache, name + "_scale")
        for b, s in enumerate(starts):
            for i in range(count[b]):
                pg, r = table[b, (s + i) // page], (s + i) % page
                touched[pg, :, r] = True
                x, big = want[name][0][b, i], np.broadcast_to(want[name][1], want[name][0].shape)[b, i]
                if sc is None:
                    close(pool[pg, :, r].double().numpy(), x, big)
                else:
                    scale = sc[pg, :, r].double().cpu().numpy()
                    ws = np.maximum(np.abs(x).max(-1), 1e-4) / 448
                    assert (np.abs(scale - ws) <= ws * 2.0 ** -22 + F32 / 448 * (big.max(-1) + 1e-30)).all()
                    got = pool[pg, :, r].double().numpy() * scale[:, None]
                    tol = 2.0 ** -4 * np.abs(x) + (2.0 ** -10 + 448 * F32) * scale[:, None] * 1.01 + F32 * big
                    assert (np.abs(got - x) <= tol).all()
                    # nearest codes: no element is off by more than its binade's half step (and the scale's error)
                    assert (np.abs(got - x) / np.maximum(np.abs(x), 2.0 ** -6 * scale[:, None])).max() <= 2.0 ** -4 * 1.02
                assert (cache.weights[pg, :, r] == 0).all()
                assert (cache.positions[pg, :, r] == int(pos[b, i])).all()
    for n, x in before.items():  # every other slot stays as it was
        now = getattr(cache, n).cpu().view(torch.uint8).view(*touched.shape, -1)
        assert torch.equal(now[~touched], x.cpu().view(torch.uint8).view(*touched.shape, -1)[~touched])
    assert (cache.weights.cpu()[~touched] == 3).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, E4M3])
def test_append_without_norm_or_turn_is_write(gpu, dtype):
    starts, S, H, HK, D = [3, 0], 5, 4, 2, 128
    cache, table, ((q, _), (k, _), (v, _)), _ = setup(gpu, 1, starts, S, H, HK, D, 16, dtype, False, track=True)
    other, *_ = setup(gpu, 1, starts, S, H, HK, D, 16, dtype, False, track=True)
    t, st = torch.from_numpy(table).to(gpu), i32(starts, gpu)
    o = cache.append(q, k, v, t, st)
    other.write(k, v, t, st)
    assert torch.equal(o, q)
    for n in ("k", "v", "k_scale", "v_scale", "weights", "positions"):
        a, b = getattr(cache, n), getattr(other, n)
        assert a is None and b is None or torch.equal(a.view(torch.uint8), b.view(torch.uint8)), n


def test_append_positions_of_each_token_and_outside_the_table(gpu):
    starts, S, H, HK, D, R = [4, 9], 4, 2, 1, 64, 32
    cache, table, ((q, qc), (k, kc), (v, _)), g = setup(gpu, 2, starts, S, H, HK, D, 16, torch.bfloat16, False)
    ang = torch.randn(10, R // 2, generator=g, dtype=torch.float64)
    freqs = torch.polar(torch.ones_like(ang), ang).to(torch.complex64)
    pos = np.array([[4, 5, 5, 6], [9, 10, -1, 9]])
    t, st = torch.from_numpy(table).to(gpu), i32(starts, gpu)
    o = cache.append(q, k, v, t, st, freqs.to(gpu), position=i32(pos.tolist(), gpu)).double().cpu().numpy()
    z = freqs.to(torch.complex128).numpy()
    for b in range(2):
        for i in range(S):
            pg, r = table[b, (starts[b] + i) // 16], (starts[b] + i) % 16
            row = cache.k[pg, :, r].double().cpu().numpy()
            if not 0 <= pos[b, i] < 10:  # turned dims are NaN, the others and v as they were
                assert np.isnan(o[b, i, :, D - R:]).all() and np.isnan(row[:, D - R:]).all()
                assert (o[b, i, :, :D - R] == qc[b, i, :, :D - R].double().numpy()).all()
                continue
            x = qc[b, i].double().numpy()
            close(o[b, i], op.turned(x, None, 0, z[pos[b, i]][None], False, False), pair_max(x, R, False, False))
            x = kc[b, i].double().numpy()
            close(row, op.turned(x, None, 0, z[pos[b, i]][None], False, False), pair_max(x, R, False, False))
    # slots are the positions without one; slots past the table and missing pages are dropped, q is turned all the same
    t2 = t.clone()
    t2[0, 0] = -1
    was = cache.k.clone()
    o = cache.append(q, k, v, t2, i32([4, t.shape[1] * 16 - 2], gpu), freqs.to(gpu), position=i32([0, 0], gpu))
    assert torch.isfinite(o).all()
    changed = (cache.k.view(torch.int16) != was.view(torch.int16)).any(-1).any(1)  # the bits: there is NaN
    assert int(changed.sum()) <= 2 and not changed[table[0, 0]].any()


def test_append_rows_that_are_not_finite_and_zero_rows(gpu):
    """A NaN or an infinity stays in its row; a row of zeros is zeros."""
    for dtype in (torch.bfloat16, E4M3):
        cache, table, ((q, _), (k, _), (v, _)), g = setup(gpu, 3, [0], 4, 2, 2, 128, 16, dtype, False)
        w = torch.ones(128, device=gpu)
        q, k, v = q.clone(), k.clone(), v.clone()
        q[0, 0, 0, 5], k[0, 1, 0, 7], v[0, 2, 1, 3] = float("nan"), float("inf"), float("nan")
        k[0, 3] = 0
        o = cache.append(q, k, v, torch.from_numpy(table).to(gpu), i32([0], gpu), q_norm=w, k_norm=w)
        assert torch.isnan(o[0, 0, 0]).all() and torch.isfinite(o[0, 0, 1]).all() and torch.isfinite(o[0, 1:]).all()
        kk = cache.k[table[0, 0]].float()
        assert not torch.isfinite(kk[0, 1]).all() and torch.isfinite(kk[1]).all() and (kk[:, 3] == 0).all()
        assert torch.isfinite(kk[0, [0, 2, 3]]).all()
        assert not torch.isfinite(cache.v[table[0, 0]].float()[1, 2]).all()


def test_append_in_place_unaligned_and_refusals(gpu):
    cache, table, ((q, _), (k, _), (v, _)), g = setup(gpu, 4, [2, 0], 3, 4, 2, 64, 16, torch.bfloat16, False)
    t, st = torch.from_numpy(table).to(gpu), i32([2, 0], gpu)
    w = 1 + 0.1 * torch.randn(64, generator=g).to(gpu)
    freqs = torch.polar(torch.ones(9, 16), torch.randn(9, 16, generator=g)).to(torch.complex64).to(gpu)
    args = dict(q_norm=w, k_norm=w, halves=True)
    want = cache.append(q, k, v, t, st, freqs, **args)
    pool = cache.k.clone()
    own = q.contiguous()
    assert cache.append(own, k, v, t, st, freqs, out=own, **args) is own and torch.equal(own, want)
    # rows that are not 16-byte aligned, or strided inside, are copied
    odd = torch.empty(2, 3, 4 * 64 + 1, dtype=torch.bfloat16, device=gpu)[..., 1:].view(2, 3, 4, 64)
    odd.copy_(q)
    cache.k.zero_()
    assert torch.equal(cache.append(odd, k.repeat_interleave(2, -1)[..., ::2], v, t, st, freqs, **args), want)
    assert torch.equal(cache.k, pool)
    fused = torch.cat([q.flatten(2), k.flatten(2)], -1)
    qf = fused[..., :256].view(2, 3, 4, 64)
    with pytest.raises(Exception, match="overlaps an input"):
        cache.append(qf, k, v, t, st, freqs, out=fused.view(-1)[:qf.numel()].view(2, 3, 4, 64))
    for bad, match in ((dict(q_norm=w[:32]), "q_norm must be"), (dict(k_norm=w.double()), "k_norm must be"),
                       (dict(position=t[:, :1].expand(2, 2)), "position must be"), (dict(count=st.long()), "count must be"),
                       (dict(out=want.float()), "out must be")):
        with pytest.raises(ValueError, match=match):
            cache.append(q, k, v, t, st, freqs, **bad)
    with pytest.raises(ValueError, match="complex64"):
        cache.append(q, k, v, t, st, torch.view_as_real(freqs))
    with pytest.raises(ValueError, match="conjugated"):
        cache.append(q, k, v, t, st, freqs.conj())
    with pytest.raises(Exception, match="rotary dims"):
        cache.append(q, k, v, t, st, freqs[:, :5].contiguous())
    with pytest.raises(TypeError, match="bf16 q"):
        cache.append(q.float(), k, v, t, st)
    with pytest.raises(ValueError, match="v is given"):
        cache.append(q, k, None, t, st)
    assert cache.append(q[:0], k[:0], v[:0], t[:0], st[:0], freqs).shape == (0, 3, 4, 64)


# ---- accept ----


@pytest.mark.parametrize("HK,D,dtype,shared,page,track", [
    (2, 64, torch.bfloat16, False, 16, True), (8, 128, torch.bfloat16, False, 64, False), (3, 128, E4M3, False, 16, True),
    (1, 512, torch.bfloat16, True, 16, False), (1, 512, E4M3, True, 32, True), (65, 256, E4M3, False, 16, False)])
@pytest.mark.parametrize("S", [1, 2, 17, 64])
def test_accept(gpu, S, HK, D, dtype, shared, page, track):
    """Random trees and paths from none to all of their depth, every array of the cache, other slots as they were."""
    rng = np.random.default_rng(S + HK)
    starts = [0, 3, 16, 31, 50, 7, 7]
    B = len(starts)
    need = [-(-(s + S) // page) for s in starts]
    P, width = sum(need) + 1, max(need)
    cache = PagedKV.empty(P, page, HK, D, dtype=dtype, shared=shared, track=track, device=gpu)
    names = [n for n in ("k", "v", "k_scale", "v_scale", "weights", "positions") if getattr(cache, n) is not None]
    for n in names:
        x = getattr(cache, n)
        x.view(torch.uint8).copy_(torch.from_numpy(rng.integers(0, 256, x.numel() * x.element_size(), dtype=np.uint8))
                                  .view(x.view(torch.uint8).shape))
    table, at, order = np.full((B, width), -1, dtype=np.int32), 0, rng.permutation(P)
    for b, c in enumerate(need):
        table[b, :c] = order[at:at + c]
        at += c
    parent = np.array([[-1] + [int(rng.integers(max(0, i - 5), i)) for i in range(1, S)] for _ in range(B)],
                      dtype=np.int32).reshape(B, S)
    sampled = rng.integers(0, 3, (B, S)).astype(np.int32)
    drafted = rng.integers(0, 3, (B, S)).astype(np.int32)
    if S > 1:
        chain = np.arange(S, dtype=np.int32) - 1
        parent[1], drafted[1, 1:], sampled[1] = chain, np.arange(S - 1) + 10, np.arange(S) + 10  # all of it: nothing moves
        parent[2], drafted[2] = chain, 77  # nothing
        drafted[3, 1:] = sampled[3][parent[3, 1:]]  # wherever the lowest child leads
    count = np.array([S, S, S, S, S // 2, 0, -4], dtype=np.int32)
    was = {n: getattr(cache, n).cpu().clone() for n in names}
    lens, tokens, path = cache.accept(*(torch.from_numpy(x).to(gpu) for x in (drafted, parent, sampled, table)),
                                      i32(starts, gpu), count=torch.from_numpy(count).to(gpu))
    want = {n: x.view(torch.uint8).view(P, HK, page, -1).clone() for n, x in was.items()}
    for b, s in enumerate(starts):
        p = op.accept(drafted[b], parent[b], sampled[b], max(int(count[b]), 0))
        assert path[b].tolist() == p + [-1] * (S - len(p)) and int(lens[b]) == s + len(p)
        assert tokens[b].tolist() == [int(sampled[b, i]) for i in p] + [-1] * (S - len(p))
        for x in want.values():
            for i, node in enumerate(p):
                x[table[b, (s + i) // page], :, (s + i) % page] = x[table[b, (s + node) // page], :, (s + node) % page]
    for n, x in want.items():
        assert torch.equal(getattr(cache, n).cpu().view(torch.uint8).view(P, HK, page, -1), x), n


def test_accept_missing_pages_and_odd_parents(gpu):
    """A row without a page at either end stays; a child before its parent and a parent that is no node are never reached;
    slots past the table are dropped."""
    page, HK, D, S = 16, 1, 64, 8
    cache = PagedKV.empty(8, page, HK, D, device=gpu)
    cache.k.copy_(torch.arange(8 * page, device=gpu).view(8, 1, page, 1).expand_as(cache.k))
    cache.v.copy_(cache.k + 500)
    parent = np.array([[-1, 0, 1, 1, 3, 0, 5, 2], [-1, 4, 0, -7, 2, 99, 1, 4], [-1, 0, 0, 2, 2, 4, 4, 6]], dtype=np.int32)
    drafted = np.array([[1, 9, 9, 7, 6, 1, 1, 1], [1, 1, 7, 7, 7, 7, 7, 5], [1, 9, 7, 7, 5, 1, 5, 5]], dtype=np.int32)
    sampled = np.array([[9, 7, 1, 6, 2, 2, 2, 2], [7, 7, 7, 7, 5, 7, 7, 2], [7, 1, 5, 1, 5, 1, 5, 8]], dtype=np.int32)
    table = np.array([[4, -1], [2, 3], [6, 7]], dtype=np.int32)
    starts = [12, 20, 28]
    was = {n: getattr(cache, n).clone() for n in ("k", "v")}
    lens, tokens, path = cache.accept(*(torch.from_numpy(x).to(gpu) for x in (drafted, parent, sampled, table)), i32(starts, gpu))
    assert path[0].tolist() == [0, 1, 3, 4] + [-1] * 4 and path[1].tolist() == [0, 2, 4, 7] + [-1] * 4
    assert path[2].tolist() == [0, 2, 4, 6, 7, -1, -1, -1] and lens.tolist() == [16, 24, 33]
    assert tokens[1].tolist() == [7, 7, 5, 2] + [-1] * 4
    for n, x in was.items():
        x = x.cpu().clone()
        x[4, 0, 14] = x[4, 0, 15]  # node 3 to place 2; node 4 has no page
        x[3, 0, 5], x[3, 0, 6], x[3, 0, 7] = x[3, 0, 6].clone(), x[3, 0, 8].clone(), x[3, 0, 11].clone()
        x[7, 0, 13] = x[7, 0, 14]  # slots 28 + 4, + 6, + 7 are past the table
        assert torch.equal(getattr(cache, n).cpu(), x), n


def test_accept_outputs_and_refusals(gpu):
    cache = PagedKV.empty(4, 16, 1, 64, device=gpu)
    z = torch.zeros(2, 3, dtype=torch.int32, device=gpu)
    t, st = torch.zeros(2, 1, dtype=torch.int32, device=gpu), i32([0, 1], gpu)
    out = i32([9, 9], gpu), torch.full((2, 3), 9, dtype=torch.int32, device=gpu), torch.full((2, 3), 9, dtype=torch.int32, device=gpu)
    assert cache.accept(z, z - 1, z, t, st, out=out) is out
    assert out[0].tolist() == [1, 2] and out[1].tolist() == [[0, -1, -1]] * 2 and out[2].tolist() == [[0, -1, -1]] * 2
    with pytest.raises(Exception, match="overlaps an input"):
        cache.accept(z, z - 1, z, t, st, out=(st, out[1], out[2]))
    with pytest.raises(ValueError, match="sampled must be"):
        cache.accept(z, z, z.long(), t, st)
    with pytest.raises(ValueError, match="parent must be"):
        cache.accept(z, z[:, :2], z, t, st)
    with pytest.raises(ValueError, match="drafted must be"):
        cache.accept(z[0], z, z, t, st)
    big = torch.zeros(2, 65, dtype=torch.int32, device=gpu)
    with pytest.raises(Exception, match="S=65"):
        cache.accept(big, big, big, t, st)
    e = torch.zeros(0, 3, dtype=torch.int32, device=gpu)
    assert cache.accept(e, e, e, t[:0], st[:0])[0].shape == (0,)
    none = torch.zeros(2, 0, dtype=torch.int32, device=gpu)
    assert cache.accept(none, none, none, t, st)[0].tolist() == [0, 1]
