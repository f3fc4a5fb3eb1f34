"""CPU checks of the operators of a step that verifies drafted tokens (PagedKV.append, attend_tree and accept,
kernels.sample): the C ABI's refusals (no pointer below is ever dereferenced), the Python side's, and the plain
statements that the GPU tests compare with."""

import ctypes

import numpy as np
import pytest
import torch

from oracle import paged as op
from oracle import sampling as osm
from tests.launch_recorder import record
from tests.test_paged import I3, cache, err
from wanferenz_amd import _native as N
from wanferenz_amd import kernels


def append(c, q=16, qs=(0, 128, 64), k=16, ks=(0, 128, 64), v=32, vs=(0, 128, 64), out=1 << 20, H=2, qn=None, kn=None, fr=64,
           turns=8, R=64, halves=0, off=0, table=4, width=3, start=4, B=1, S=1):
    I = lambda x: None if x is None else I3(*x)  # noqa: E731
    return N.lib().wz_paged_append(ctypes.byref(c), q, I(qs), k, I(ks), v, I(vs), out, H, qn, kn, 1e-6, fr, turns, R, halves,
                                   off, table, width, start, None, None, 0, B, S, None)


def tree(c, q=16, qs=(0, 0, 64), table=4, width=3, lens=4, parent=4, o=16, B=1, S=1, H=2, ws=None, wsb=0):
    return N.lib().wz_paged_tree_attn(ctypes.byref(c), q, None if qs is None else I3(*qs), None, table, width, lens, parent,
                                      None, o, B, S, H, 0.1, ws, wsb, None)


def accept(c, d=4096, p=8192, s=12288, table=16384, width=3, start=20480, count=None, lens=24576, tokens=28672, path=32768,
           B=1, S=4):
    return N.lib().wz_paged_accept(ctypes.byref(c), d, p, s, table, width, start, count, lens, tokens, path, B, S, None)


def sample(logits=16, bf16=0, stride=100, u=4, tokens=4, probs=4, n=1, V=100, ws=None, wsb=0):
    return N.lib().wz_sample(logits, bf16, stride, u, None, 1.0, None, 0, None, 1.0, None, 0.0, tokens, probs, n, V, ws, wsb,
                             None)


@pytest.mark.parametrize("call", [append, tree, accept])
@pytest.mark.parametrize("bad,what", [(dict(dtype=7), "cache type"), (dict(dim=96), "head dim"), (dict(page=48), "page size"),
                                      (dict(k=None), "null pointer"), (dict(dtype=N.WZ_KV_E4M3), "scales")])
def test_bad_caches_are_refused(call, bad, what):
    assert call(cache(**bad)) == -1 and what in err()


def test_append_refusals():
    c = cache()
    for name in ("q", "k", "v", "qs", "ks", "vs", "out", "start", "table", "fr"):
        assert append(c, **{name: None}) == -1 and "null" in err(), name
    for name in ("q", "k", "v"):
        assert append(c, **{name: 24}) == -1 and "16-byte" in err(), name
    assert append(c, ks=(0, 12, 64)) == -1 and "multiples of 8" in err()
    assert append(c, qs=(0, -128, 64)) == -1 and "not negative" in err()
    assert append(c, out=(1 << 20) + 8) == -1 and append(c, qn=8) == -1 and append(c, fr=72) == -1 and "16-byte" in err()
    assert append(c, R=80) == -1 and append(c, R=8) == -1 and append(c, R=-16) == -1 and "rotary dims" in err()
    assert append(c, R=32, off=8) == -1 and append(c, R=32, off=48) == -1 and append(c, R=32, off=-16) == -1
    assert append(c, turns=-1) == -1 and append(c, turns=0) == -1 and "turns" in err()
    assert append(c, turns=0, R=0, fr=None, B=0) == 0
    assert append(c, H=0) == -1 and append(c, B=-1) == -1 and "bad shape" in err()
    assert append(c, B=2 ** 31 - 1, S=2 ** 31 - 1) == -1 and "tokens" in err()
    # 2^32 threads: 1024 heads and 2 x 2 rows of 4 threads
    assert append(c, H=1020, S=2 ** 20, qs=(0, 0, 0), ks=(0, 0, 0), vs=(0, 0, 0)) == -1 and "tokens" in err()
    assert append(c, B=0, q=None) == 0 and append(c, S=0, q=None) == 0
    # q may be turned in place, and in no other way over an input
    assert append(c, q=1 << 16, out=(1 << 16) + 16) == -1 and "overlaps" in err()
    assert append(c, q=1 << 16, qs=(0, 192, 64), S=2, out=1 << 16) == -1 and "overlaps" in err()
    assert append(c, k=1 << 16, out=(1 << 16) - 128) == -1 and "overlaps" in err()


def test_tree_refusals_and_workspace():
    c = cache()
    assert tree(c, S=65) == -1 and "S=65 (up to 64)" in err()
    assert tree(c, H=3) == -1 and "3 heads on 2" in err()
    for name in ("q", "lens", "o", "table", "parent"):
        assert tree(c, **{name: None}) == -1 and "null" in err(), name
    assert tree(c, q=24) == -1 and "16-byte" in err()
    assert tree(c, S=64, H=512, qs=(0, 0, 64)) == -1 and "query rows" in err()
    assert tree(c) == -3 and "workspace of 0 bytes" in err()
    assert tree(c, B=0, q=None) == 0 and tree(c, S=0, q=None) == 0
    need = N.lib().wz_paged_tree_attn_workspace_bytes
    assert need(ctypes.byref(c), 1, 64, 2, 3) > 0
    assert need(ctypes.byref(c), 1, 65, 2, 3) == 0 and need(ctypes.byref(c), 1, 0, 2, 3) == 0


def test_accept_refusals():
    c = cache()
    for name in ("d", "p", "s", "table", "start", "lens", "tokens", "path"):
        assert accept(c, **{name: None}) == -1 and "null" in err(), name
    assert accept(c, S=65) == -1 and "S=65" in err()
    assert accept(c, lens=20480) == -1 and "overlaps an input" in err()
    assert accept(c, tokens=12284) == -1 and "overlaps an input" in err()
    assert accept(c, count=24576) == -1 and "overlaps an input" in err()
    assert accept(c, path=28676) == -1 and "outputs overlap" in err()
    assert accept(c, B=0, d=None) == 0


def test_sample_refusals():
    assert sample(V=0) == -1 and sample(V=2 ** 21 + 1, stride=2 ** 22) == -1 and sample(n=-1) == -1 and "rows" in err()
    assert sample(stride=99) == -1 and "apart" in err()
    for name in ("logits", "u", "tokens", "probs"):
        assert sample(**{name: None}) == -1 and "null" in err(), name
    assert sample(logits=18) == -1 and sample(logits=17, bf16=1) == -1 and "aligned" in err()
    assert sample(n=0, u=None) == 0
    # few long rows are shared by workgroups, many are not; a larger batch's workspace need not serve a smaller one
    need = N.lib().wz_sample_workspace_bytes
    assert need(1, 131072) > need(1, 40000) > 0 and need(512, 131072) == 0 and need(1, 32767) == 0
    assert need(0, 100) == 0 and need(1, 0) == 0 and need(-1, 100) == 0 and need(1, 2 ** 21 + 1) == 0
    assert sample(V=131072, stride=131072) == -3 and "workspace of 0 bytes" in err()
    assert sample(V=131072, stride=131072, ws=16, wsb=100) == -3 and "workspace of 100 bytes" in err()
    assert sample(V=131072, stride=131072, ws=8, wsb=1 << 30) == -1 and "16-byte" in err()
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        kernels.sample(torch.zeros(1, 5), torch.zeros(1))


def test_sample_outputs_over_inputs_are_refused():
    places = dict(logits=1 << 20, u=16, t=32, k=48, p=64, m=80, tokens=96, probs=112)

    def call(**over):
        a = {**places, **over}
        return N.lib().wz_sample(a["logits"], 0, 100, a["u"], a["t"], 1.0, a["k"], 0, a["p"], 1.0, a["m"], 0.0, a["tokens"],
                                 a["probs"], 3, 100, None, 0, None)

    for out in ("tokens", "probs"):
        for name in ("u", "t", "k", "p", "m"):
            assert call(**{out: places[name] + 8}) == -1 and "an output overlaps an input" in err(), (out, name)
        assert call(**{out: (1 << 20) + 296 * 4}) == -1 and "an output overlaps an input" in err()
    assert call(tokens=104) == -1 and "outputs overlap" in err()


def test_plain_tree_of_a_chain_is_causal_attention():
    rng = np.random.default_rng(0)
    c = {"k": rng.standard_normal((5, 2, 16, 8)), "v": rng.standard_normal((5, 2, 16, 8))}
    table, lens, S = np.array([[3, 1, 0], [4, 2, -1]]), [40, 20], 5
    q = rng.standard_normal((2, S, 4, 8))
    parent = np.tile(np.arange(S) - 1, (2, 1))
    a, b = op.attend(c, q, table, lens, 0.3), op.attend_tree(c, q, table, lens, parent, 0.3)
    assert np.allclose(a[0], b[0], atol=1e-12) and np.allclose(a[1], b[1], atol=1e-12)
    # siblings: each sees the root and itself, so the second one's result is the first's with its own slot
    o = op.attend_tree(c, q, table, lens, np.tile([-1, 0, 0, 0, 0], (2, 1)), 0.3)[0]
    for i in range(1, S):
        t2 = table.copy()
        swapped = {n: x.copy() for n, x in c.items()}
        for n in swapped:  # node i's row into node 1's slot: the plain attention of two new tokens
            for b_, ln in enumerate(lens):
                s1, si = ln - S + 1, ln - S + i
                swapped[n][t2[b_, s1 // 16], :, s1 % 16] = c[n][t2[b_, si // 16], :, si % 16]
        two = op.attend(swapped, q[:, [0, i]], t2, [ln - S + 2 for ln in lens], 0.3)[0]
        assert np.allclose(o[:, i], two[:, 1], atol=1e-12)
    # padded: the tree ends with its count, the rows behind it are 0
    o = op.attend_tree(c, q, table, [ln - 2 for ln in lens], parent, 0.3, count=[3, 3])[0]
    assert np.allclose(o[:, :3], a[0][:, :3], atol=1e-12) and not o[:, 3:].any()


def test_plain_turn_is_the_rotation_of_pairs():
    rng = np.random.default_rng(1)
    x = rng.standard_normal((3, 48))
    z = np.exp(1j * rng.standard_normal((3, 16)))
    for halves in (False, True):
        for leading in (False, True):
            y = op.turned(x, None, 0.0, z, halves, leading)
            part = slice(0, 32) if leading else slice(16, 48)
            rest = slice(32, 48) if leading else slice(0, 16)
            assert (y[:, rest] == x[:, rest]).all()
            a, b = x[:, part], y[:, part]
            pairs = (lambda t: (t[:, :16], t[:, 16:])) if halves else (lambda t: (t[:, ::2], t[:, 1::2]))
            (ar, ai), (br, bi) = pairs(a), pairs(b)
            assert np.allclose(br + 1j * bi, (ar + 1j * ai) * z)
    w = rng.standard_normal(48)
    y = op.turned(x, w, 1e-6, np.ones((3, 8)), True, True)
    assert np.allclose(np.mean((y / w) ** 2, axis=-1), 1.0, atol=1e-5)


def test_plain_accept_walks_down_the_tree():
    parent = [-1, 0, 0, 1, 1, 3]
    assert op.accept([9, 5, 6, 7, 8, 1], parent, [6, 0, 4, 0, 0, 0], 6) == [0, 2]
    assert op.accept([9, 6, 6, 7, 8, 1], parent, [6, 8, 4, 0, 0, 0], 6) == [0, 1, 4]
    assert op.accept([9, 6, 6, 7, 8, 1], parent, [6, 8, 4, 0, 0, 0], 2) == [0, 1]
    assert op.accept([9, 6], parent, [6, 8], 0) == []


def test_plain_sample_filters():
    row = np.log(np.array([0.1, 0.4, 0.1, 0.4]))
    assert osm.sample(row, 0.0)[0] == 1 and osm.sample(row, 0.41)[0] == 3 and osm.sample(row, 0.85)[0] == 0
    assert osm.sample(row, 0.95)[0] == 2 and osm.sample(row, 0.999, top_k=1)[:3] == (1, 1.0, 1.0)
    assert osm.sample(row, 0.99, top_p=0.7)[:2] == (3, 0.5) and osm.sample(row, 0.99, top_k=3)[0] == 0
    assert osm.sample(row, 0.99, min_p=0.5)[0] == 3 and osm.sample(row, 0.99, temperature=0)[0] == 1
    assert osm.sample([np.nan, -np.inf], 0.5)[:2] == (-1, 0.0)
    assert osm.sample([np.inf, 3.0, np.inf], 0.6)[:2] == (2, 0.5)


# ---- which kernels a call takes, on a recording HIP runtime of 256 compute units ----

P, BIG = 1 << 20, 1 << 40


def launches(tmp_path, *call):
    _, events = record(tmp_path, [call])
    return [(e["name"].split("(")[0].split("wz::")[1], e["grid"], e["block"], e["bytes"]) for e in events if e["kind"] == "launch"]


def raw(c):
    return bytes(ctypes.string_at(ctypes.byref(c), ctypes.sizeof(c)))


@pytest.mark.parametrize("S,g,D,shared,kernel", [
    (4, 4, 128, False, "paged_attn_kernel<128, false, false, 1, 1, true>"),
    (16, 4, 128, False, "paged_attn_kernel<128, false, false, 2, 2, true>"),
    (13, 5, 128, False, "paged_wide_kernel<128, false, false, 4>"), (16, 8, 128, False, "paged_wide_kernel<128, false, false, 4>"),
    (43, 3, 128, False, "paged_wide_kernel<128, false, false, 8>"), (64, 16, 128, True, "paged_wide_kernel<128, false, true, 8>"),
    (64, 16, 64, False, "paged_wide_kernel<64, false, false, 4>"), (64, 1, 64, False, "paged_attn_kernel<64, false, false, 2, 2, true>"),
    (33, 4, 256, False, "paged_attn_kernel<256, false, false, 2, 2, true>"),
    (8, 64, 512, True, "paged_latent_kernel<false, 4, true, true>")])
def test_tree_routes(tmp_path, S, g, D, shared, kernel):
    c = cache(k=P, v=None if shared else P, heads=1, dim=D)
    got = launches(tmp_path, "wz_paged_tree_attn", raw(c), P, raw(I3(0, 0, D)), None, P, 5000, P, P, None, P, 4, S, g, 0.1, P, BIG, None)
    assert [x[0] for x in got][0] == kernel and "join" in got[1][0] and len(got) == 2
    assert got[0][3] * max(1, 512 // got[0][2] if "wide" in kernel else 1) <= 160 * 1024


@pytest.mark.parametrize("width,rows", [(4, 16), (378, 16), (380, 64), (5000, 64)])
def test_tables_of_few_slots_take_units_of_16_rows(tmp_path, width, rows):
    """64 rows on 2 KV heads of 4 sequences: 32 units of 16 rows, width / 2 + 3 tiles each, up to 24 a compute unit; the workspace
    holds the partials of the kernel that runs."""
    c = cache(k=P, v=P, heads=2, dim=128, page=16)
    assert (32 * (width // 2 + 3) <= 24 * 256) == (rows == 16)
    got = launches(tmp_path, "wz_paged_tree_attn", raw(c), P, raw(I3(0, 0, 128)), None, P, width, P, P, None, P, 4, 16, 8, 0.1, P,
                   BIG, None)
    assert got[0][0] == f"paged_attn_kernel<128, false, false, {'1, 1' if rows == 16 else '2, 2'}, true>"
    need = N.lib().wz_paged_tree_attn_workspace_bytes(ctypes.byref(c), 4, 16, 8, width)
    assert need == got[0][1] * (2 * 4 * (2 * rows + rows * 128) + 16)


@pytest.mark.parametrize("n,V,greedy,names", [
    (1, 32767, False, ["sample_kernel", "sample_dense_kernel"]), (1, 32768, False, ["sample_top_kernel", "sample_histogram_kernel", "sample_pick_kernel"]),
    (64, 131072, False, ["sample_top_kernel", "sample_histogram_kernel", "sample_pick_kernel"]),
    (64, 131072, True, ["sample_top_kernel", "sample_pick_kernel"]), (512, 100003, True, ["sample_kernel"]),
    (129, 100003, False, ["sample_kernel", "sample_dense_kernel"])])
def test_sample_routes(tmp_path, n, V, greedy, names):
    u, tokens, probs = (P + (1 << 40) + i * 4096 for i in range(3))
    got = launches(tmp_path, "wz_sample", P, 0, V, u, None, 0.0 if greedy else 1.0, None, 0, None, 1.0, None, 0.0, tokens, probs, n,
                   V, P, BIG, None)
    assert [x[0].split("<")[0] for x in got] == names
