"""CPU checks of the paged cache: the C ABI's refusals and sizes (no pointer below is ever
dereferenced), the Python side's, and the plain statements that the GPU tests compare with."""

import ctypes

import numpy as np
import pytest
import torch

from oracle import paged as op
from wanferenz_amd import _native as N
from wanferenz_amd.paged import PagedKV, WzPagedKV

I3 = ctypes.c_int64 * 3


def err():
    return N.lib().wz_last_error().decode()


def cache(k=16, v=32, ks=None, vs=None, w=None, p=None, pages=10, page=16, heads=2, dim=64, dtype=N.WZ_KV_BF16):
    return WzPagedKV(k, v, ks, vs, w, p, pages, page, heads, dim, dtype)


def write(c, k=16, ks=(0, 128, 64), v=32, vs=(0, 128, 64), table=4, width=3, start=4, B=1, S=1):
    return N.lib().wz_paged_kv_write(ctypes.byref(c), k, None if ks is None else I3(*ks), v,
                                     None if vs is None else I3(*vs), table, width, start, None, None, B, S, None)


def attn(c, q=16, qs=(0, 0, 64), table=4, width=3, lens=4, o=16, B=1, S=1, H=2, acc=0, ws=None, wsb=0):
    return N.lib().wz_paged_attn(ctypes.byref(c), q, None if qs is None else I3(*qs), None, table, width, lens, o, B, S, H,
                                 0.1, acc, ws, wsb, None)


def evict(c, table=4, width=3, lens=4, new=4, B=1, keep=8, first=0, recent=0, ws=None, wsb=0):
    return N.lib().wz_paged_evict(ctypes.byref(c), table, width, lens, new, B, keep, first, recent, ws, wsb, None)


TRACK = dict(w=4, p=4)


@pytest.mark.parametrize("bad,what", [
    (dict(dtype=7), "cache type"), (dict(dim=96), "head dim"), (dict(dim=512), "head dim"), (dict(v=None, dim=64), "head dim"),
    (dict(page=8), "page size"), (dict(page=48), "page size"), (dict(page=2048), "page size"), (dict(pages=0), "pages"),
    (dict(heads=0), "heads"), (dict(k=None), "null pointer"), (dict(k=8), "16-byte aligned"), (dict(v=40), "16-byte aligned"),
    (dict(dtype=N.WZ_KV_E4M3), "scales"), (dict(dtype=N.WZ_KV_E4M3, ks=4), "scales"), (dict(w=4), "weights and positions"),
    (dict(p=4), "weights and positions"),
])
def test_bad_caches_are_refused_by_every_entry(bad, what):
    c = cache(**bad)
    for call in (write, attn, evict):
        assert call(c) == -1 and what in err(), (call, err())


def test_write_refusals():
    c = cache()
    assert write(c, k=None) == -1 and "null" in err()
    assert write(c, v=None) == -1 and "null" in err()
    assert write(c, ks=None) == -1 and "null" in err()
    assert write(c, table=None) == -1 and "null" in err()
    assert write(c, start=None) == -1 and "null" in err()
    assert write(c, k=24) == -1 and "16-byte" in err()
    assert write(c, vs=(0, 12, 64)) == -1 and "multiples of 8" in err()
    assert write(c, B=-1) == -1 and "bad shape" in err()
    assert write(c, B=2 ** 31 - 1, S=2 ** 31 - 1) == -1 and "tokens" in err()
    assert write(c, width=2 ** 27) == -1 and "table width" in err()
    assert write(c, B=0, k=None) == 0 and write(c, S=0, k=None) == 0 and write(c, width=0, table=None) == 0


def test_attend_refusals_and_workspace():
    L = N.lib()
    c = cache()
    assert attn(c, H=3) == -1 and "3 heads on 2" in err()
    assert attn(c, H=0) == -1 and "heads" in err()
    assert attn(c, S=17) == -1 and "S=17" in err()
    assert attn(c, B=65536) == -1 and "B=65536" in err()
    assert attn(c, q=None) == -1 and "null" in err()
    assert attn(c, lens=None) == -1 and "null" in err()
    assert attn(c, o=None) == -1 and "null" in err()
    assert attn(c, table=None) == -1 and "null" in err()
    assert attn(c, q=24) == -1 and "16-byte" in err()
    assert attn(c, qs=(0, 4, 64)) == -1 and "16-byte" in err()
    assert attn(c, acc=1) == -1 and "not tracked" in err()
    assert attn(c) == -3 and "workspace of 0 bytes" in err()
    assert attn(c, ws=16, wsb=64) == -3 and "workspace of 64 bytes" in err()
    assert attn(c, B=0, q=None) == 0 and attn(c, S=0, q=None) == 0

    def need(B, S, H, width, acc=0, c=c):
        return L.wz_paged_attn_workspace_bytes(ctypes.byref(c), B, S, H, width, acc)

    # partials do not grow with the batch or the table; scores are 4 bytes a row and slot
    assert need(1, 1, 2, 3) == need(64, 1, 2, 4096) > 0
    c2 = cache(**TRACK)
    grown = need(8, 2, 4, 5, 1, c2) - need(8, 2, 4, 5, 0, c2)
    assert grown == 4 * 8 * 2 * 4 * 5 * 16 + 4 * (2 * 8 * 2 * 4)
    assert need(0, 1, 2, 3) == 0 and need(1, 17, 2, 3) == 0


def test_evict_refusals_and_workspace():
    c = cache()
    assert evict(c) == -1 and "not tracked" in err()
    c = cache(**TRACK)
    assert evict(c, keep=-1) == -1 and "keep -1" in err()
    assert evict(c, keep=8, first=5, recent=4) == -1 and "first + recent <= keep" in err()
    assert evict(c, first=-1) == -1 and "first -1" in err()
    assert evict(c, keep=2 ** 31) == -1 and "keep" in err()
    assert evict(c, B=40000) == -1 and "65535" in err()
    assert evict(c, lens=None) == -1 and "null" in err()
    assert evict(c, new=None) == -1 and "null" in err()
    assert evict(c, table=None) == -1 and "null" in err()
    assert evict(c) == -3 and "needed" in err()
    assert evict(c, ws=16, wsb=8) == -3 and "workspace of 8 bytes" in err()
    assert evict(c, B=0, lens=None) == 0


def test_python_side_refuses_what_does_not_fit():
    bf = torch.bfloat16
    k = torch.zeros(4, 2, 16, 64, dtype=bf)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        PagedKV(k, k)
    with pytest.raises(ValueError, match="page_size, head_dim"):
        PagedKV(k[0], k[0])
    with pytest.raises(TypeError, match="bf16 or float8"):
        PagedKV(k.float(), k.float())
    with pytest.raises(ValueError, match="does not match"):
        PagedKV(k, k[:2])
    with pytest.raises(ValueError, match="belong to e4m3"):
        PagedKV(k, k, k_scale=torch.zeros(4, 2, 16))
    with pytest.raises(ValueError, match="belong to e4m3"):
        PagedKV(k.to(torch.float8_e4m3fn), None)
    with pytest.raises(ValueError, match="both weights and positions"):
        PagedKV(k, k, weights=torch.zeros(4, 2, 16))
    with pytest.raises(ValueError, match="weights must be"):
        PagedKV(k, k, weights=torch.zeros(4, 16, 2), positions=torch.zeros(4, 2, 16, dtype=torch.int32))
    with pytest.raises(ValueError, match="positions must be"):
        PagedKV(k, k, weights=torch.zeros(4, 2, 16), positions=torch.zeros(4, 2, 16))


def test_plain_attend_is_softmax_attention():
    """Dense torch attention in float64 over the gathered rows, causal, with a sink as one more key
    whose value is zero."""
    rng = np.random.default_rng(0)
    P, HK, page, D, B, S, H = 7, 2, 16, 8, 2, 3, 6
    c = {n: rng.standard_normal((P, HK, page, D)) for n in ("k", "v")}
    table = np.array([[3, 1, 5], [6, 0, 2]], dtype=np.int32)
    lens, sink = [40, 19], rng.standard_normal(H)
    q = rng.standard_normal((B, S, H, D))
    o, mag, add, _ = op.attend(c, q, table, lens, 0.4, sink)
    total = 0.0
    for b in range(B):
        k = torch.from_numpy(c["k"][table[b]].transpose(1, 0, 2, 3).reshape(HK, -1, D)[:, :lens[b]])
        v = torch.from_numpy(c["v"][table[b]].transpose(1, 0, 2, 3).reshape(HK, -1, D)[:, :lens[b]])
        k, v = k.repeat_interleave(3, 0), v.repeat_interleave(3, 0)
        s = torch.einsum("shd,hnd->hsn", torch.from_numpy(q[b]), k) * 0.4
        seen = torch.arange(lens[b])[None] <= lens[b] - S + torch.arange(S)[:, None]
        s = s.masked_fill(~seen, -np.inf)
        s = torch.cat([s, torch.from_numpy(sink)[:, None, None].expand(H, S, 1)], 2)
        p = torch.softmax(s, 2)[..., :-1]
        assert np.allclose(o[b], torch.einsum("hsn,hnd->shd", p, v).numpy(), atol=1e-12)
        assert np.allclose(mag[b], torch.einsum("hsn,hnd->shd", p, v.abs()).numpy(), atol=1e-12)
        total += float(p.sum())
    assert abs(add.sum() - total) < 1e-9
    assert add[4].sum() == 0  # the page that nobody holds


def test_plain_evict_keeps_the_heaviest():
    w = [5, 1, 4, 1, 3, 1, 9, 2]
    pos = list(range(8))
    assert op.evict_pairs(w, pos, 8, 4, 0, 0) == ([1, 3], [4, 6])
    # the first two and the newest stay whatever they weigh; one place is left for the heaviest
    assert op.evict_pairs(w, pos, 8, 4, 2, 1) == ([2, 3], [6, 7])
    # equal weights: the lower slot stays
    assert op.evict_pairs([1] * 6, list(range(6)), 6, 3, 0, 0) == ([], [])
    assert op.evict_pairs([1] * 6, [9, 8, 7, 6, 5, 4], 6, 3, 0, 1) == ([], [])
    assert op.evict_pairs([float("nan"), 0, 0], [0, 1, 2], 3, 2, 0, 0) == ([0], [2])
    assert op.evict_pairs(w, pos, 4, 4, 0, 0) == ([], [])


def test_workspace_is_sized_on_the_cache_s_device(monkeypatch):
    """The partials' number goes by the device that is current in the library: the cache's own is made current."""
    seen = []

    class Guard:
        def __init__(self, device):
            self.device = device

        def __enter__(self):
            seen.append(("in", self.device))

        def __exit__(self, *_):
            seen.append(("out", self.device))

    class Lib:
        @staticmethod
        def wz_paged_attn_workspace_bytes(ref, b, s, h, width, acc):
            seen.append((b, s, h, width, acc))
            return 64

    monkeypatch.setattr(torch.cuda, "device", Guard)
    monkeypatch.setattr(N, "lib", Lib)
    cache = object.__new__(PagedKV)
    cache.device, cache._ref = torch.device("cuda", 5), None
    assert cache.attend_workspace_bytes(2, 1, 8, 3, True) == 64
    assert seen == [("in", cache.device), (2, 1, 8, 3, 1), ("out", cache.device)]


def test_write_refuses_more_tokens_than_a_grid_has():
    """Some 2^24 workgroups of 32 tokens each (2 heads of 64), of one each (64 heads)."""
    assert write(cache(), S=2 ** 29) == -1 and "1 x 536870912 tokens" in err()
    assert write(cache(), S=2 ** 31 - 1) == -1 and "tokens" in err()
    assert write(cache(heads=64), S=2 ** 24) == -1 and "1 x 16777216 tokens" in err()


def test_evict_sizes_that_do_not_fit_64_bits_are_refused():
    """B kv_heads and B kv_heads slots are not multiplied out before B is checked."""
    L = N.lib()
    c = cache(heads=4, **TRACK)
    for B in (16384, 2 ** 61, 2 ** 62, 2 ** 62 + 1, 2 ** 63 - 1):
        assert evict(c, B=B) == -1 and "65535" in err(), B
        assert L.wz_paged_evict_workspace_bytes(ctypes.byref(c), B, 3, 8) == 0
    assert evict(c, B=16383) == -3
    assert L.wz_paged_evict_workspace_bytes(ctypes.byref(c), 16383, 3, 8) == 4 * 65532 + 8 * 65532 * 8
    for B, width, keep in ((1, 2 ** 62, 8), (1, -1, 8), (1, 3, -1), (1, 3, 2 ** 40), (0, 3, 8), (-1, 3, 8)):
        assert L.wz_paged_evict_workspace_bytes(ctypes.byref(c), B, width, keep) == 0
    assert L.wz_paged_evict_workspace_bytes(None, 1, 3, 8) == 0


def test_evict_is_sized_before_its_pools_exist():
    """The workspace goes by the shape: pointers that are not there yet change nothing."""
    L = N.lib()
    for width in (3, 1000):
        full, bare = cache(**TRACK), cache(k=None, v=None)
        need = L.wz_paged_evict_workspace_bytes(ctypes.byref(full), 2, width, 8)
        assert need > 0 and L.wz_paged_evict_workspace_bytes(ctypes.byref(bare), 2, width, 8) == need


def test_partials_of_odd_rows_lie_on_16_bytes():
    """A worker has two partials of m and l (rounded up to 16 bytes together) and O [rows, 64], and one record
    of 16 bytes; the number of workers is the same for 1, 2 and 3 rows a KV head."""
    c = cache()
    need = [N.lib().wz_paged_attn_workspace_bytes(ctypes.byref(c), 1, 1, 2 * rows, 3, 0) for rows in (1, 2, 3)]
    slots = [16 + 4 * 64, 16 + 4 * 2 * 64, 32 + 4 * 3 * 64]
    workers = need[1] // (2 * slots[1] + 16)
    assert need == [workers * (2 * s + 16) for s in slots]


def test_evict_refuses_lengths_that_overlap_at_an_offset():
    """new_lens may be lens, or apart from it: shifted by less than the batch it would be read half written."""
    c = cache(**TRACK)
    for new in (4096 - 8, 4096 - 4, 4096 + 4, 4096 + 8):
        assert evict(c, lens=4096, new=new, B=3) == -1 and "overlaps lens" in err()
    for new in (4096 - 12, 4096, 4096 + 12):
        assert evict(c, lens=4096, new=new, B=3) == -3 and "needed" in err()


def test_plain_evict_leaves_missing_pages_out():
    """A missing slot below keep takes no kept slot with it: as many stay as have a place, protected ones first."""
    w = [1.0] * 8
    missing = [False, False, True, True, True, True, True, True]  # two of the four places have no page
    assert op.evict_pairs(w, list(range(8)), 8, 4, 0, 2, missing) == ([2, 3], [6, 7])
    missing = [True, True, False, True, True, True, True, False]
    assert op.evict_pairs([5, 1, 9, 2, 3, 4, 6, 9], list(range(8)), 8, 4, 1, 0, missing) == ([1, 3], [5, 6])
    assert op.evict_pairs(w, list(range(8)), 8, 4, 4, 0, [False] * 4 + [True] * 4) == ([], [])
