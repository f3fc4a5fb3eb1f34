"""A step that verifies drafted tokens as a serving loop runs it: append, attend_tree, sample, accept, together, eagerly, in
a captured graph and on two streams."""

import numpy as np
import pytest
import torch

from oracle import paged as op
from oracle import sampling as osm
from tests.test_gpu_paged import E4M3, check
from wanferenz_amd import kernels
from wanferenz_amd.paged import PagedKV

pytestmark = pytest.mark.gpu


class Loop:
    """Sequences of a toy model whose q, k and v of a token are rows of a table, so that any order of the same tokens leaves
    the same rows in the cache."""

    def __init__(self, gpu, seed, B, S, H, HK, D, dtype, shared, V=300, slots=160, page=16):
        g = torch.Generator().manual_seed(seed)
        self.B, self.S, self.H, self.HK, self.D, self.V, self.page, self.dev = B, S, H, HK, D, V, page, gpu
        self.width = (H + (1 if shared else 2) * HK) * D
        self.rows = torch.randn(V, self.width, generator=g).to(torch.bfloat16).to(gpu)
        self.head = (torch.randn(H * D, V, generator=g) / 4).to(gpu)
        ang = torch.arange(slots + 70, dtype=torch.float64)[:, None] * 0.3 ** torch.arange(D // 4, dtype=torch.float64)
        self.freqs = torch.polar(torch.ones_like(ang), ang).to(torch.complex64).to(gpu)
        self.qn, self.kn = ((1 + 0.1 * torch.randn(D, generator=g)).to(gpu) for _ in range(2))
        n = -(-slots // page)
        self.table = torch.randperm(B * n, generator=g).to(torch.int32).view(B, n).to(gpu)
        self.cache = PagedKV.empty(B * n, page, HK, D, dtype=dtype, shared=shared, track=True, device=gpu)
        self.shared = shared

    def split(self, tokens):
        x = self.rows[tokens.long()]
        b, s = tokens.shape
        H, HK, D = self.H, self.HK, self.D
        return (x[..., :H * D].view(b, s, H, D), x[..., H * D:(H + HK) * D].view(b, s, HK, D),
                None if self.shared else x[..., (H + HK) * D:].view(b, s, HK, D))

    def append(self, cache, tokens, start, **more):
        q, k, v = self.split(tokens)
        return cache.append(q, k, v, self.table, start, self.freqs, q_norm=self.qn, k_norm=self.kn, **more)

    def step(self, tokens, parent, depth, lens, u, **sampling):
        """-> (attention, sampled tokens, what accept gives)."""
        S = tokens.shape[1]
        q = self.append(self.cache, tokens, lens, position=lens[:, None] + depth)
        o = self.cache.attend_tree(q, self.table, lens + S, parent, self.D ** -0.5)
        logits = o.float().flatten(2).flatten(0, 1) @ self.head
        new, prob = kernels.sample(logits, u.flatten(), **sampling)
        new = new.view(tokens.shape)
        return o, logits, new, self.cache.accept(tokens, parent, new, self.table, lens)


def trees(rng, B, S):
    parent = np.array([[-1] + [int(rng.integers(max(0, i - 4), i)) for i in range(1, S)] for _ in range(B)], dtype=np.int32)
    depth = np.zeros_like(parent)
    for b in range(B):
        for i in range(1, S):
            depth[b, i] = depth[b, parent[b, i]] + 1
    return parent, depth


@pytest.mark.parametrize("dtype,H,HK,D,shared", [(torch.bfloat16, 8, 2, 64, False), (E4M3, 12, 2, 128, False),
                                                 (torch.bfloat16, 20, 1, 512, True)])
def test_accepted_tokens_stand_as_if_they_had_come_one_by_one(gpu, dtype, H, HK, D, shared):
    """Several steps, each with its own trees; the drafted tokens are made from the samples of a first pass, so that paths of
    every length are accepted.  Afterwards the cache holds what appending the accepted tokens alone would."""
    B, S = 3, 17
    L = Loop(gpu, D, B, S, H, HK, D, dtype, shared)
    rng = np.random.default_rng(D)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=gpu)  # noqa: E731
    lens, root = i32([0, 0, 0]), i32(rng.integers(0, L.V, B))
    said = [[] for _ in range(B)]  # the tokens whose rows are cached, in order
    taken = 0
    for step in range(4):
        parent, depth = trees(rng, B, S)
        u = torch.rand(B, S, generator=torch.Generator().manual_seed(step)).to(gpu)
        tokens = i32(rng.integers(0, L.V, (B, S)))
        tokens[:, 0] = root
        P, Dp = i32(parent), i32(depth)
        for _ in range(int(rng.integers(0, 5))):  # a draft that agrees with the samples a level further down
            kept = {n: getattr(L.cache, n).clone() for n in ("k", "v", "k_scale", "v_scale", "weights", "positions")
                    if getattr(L.cache, n) is not None}
            *_, new, _ = L.step(tokens, P, Dp, lens, u, temperature=0.9, top_p=0.9)
            for n, x in kept.items():
                getattr(L.cache, n).copy_(x)
            better = torch.gather(new, 1, P.clamp(min=0).long())
            tokens = torch.where((torch.arange(S, device=gpu) > 0) & (i32(rng.integers(0, 4, (B, S))) > 0), better, tokens)
        o, logits, new, (after, out, path) = L.step(tokens, P, Dp, lens, u, temperature=0.9, top_p=0.9)
        for r in range(B * S):  # the sampler's tokens are the statement's
            want = osm.sample(logits[r].cpu().numpy(), float(u.flatten()[r]), float(np.float32(0.9)), 0, float(np.float32(0.9)))
            assert want[2] < 1e-9 or int(new.flatten()[r]) == want[0]
        for b in range(B):
            p = op.accept(tokens[b].tolist(), parent[b], new[b].tolist(), S)
            assert path[b, :len(p)].tolist() == p and int(after[b]) == len(said[b]) + len(p)
            said[b] += tokens[b, p].tolist()
            taken += len(p) - 1
            root[b] = out[b, len(p) - 1]
            assert int(root[b]) == int(new[b, p[-1]])
        lens = after
    assert taken > B
    # one by one
    other = PagedKV.empty(L.cache.pages, L.page, HK, D, dtype=dtype, shared=shared, track=True, device=gpu)
    for b in range(B):
        for t, tok in enumerate(said[b]):
            one = torch.zeros(B, 1, dtype=torch.int32, device=gpu)
            one[b] = tok
            count = [0] * B
            count[b] = 1
            L.append(other, one, i32([t] * B), count=i32(count))
    for n in ("k", "v", "k_scale", "v_scale", "weights", "positions"):
        x, y = getattr(L.cache, n), getattr(other, n)
        if x is None:
            continue
        for b in range(B):
            at = [(int(L.table[b, t // L.page]), t % L.page) for t in range(len(said[b]))]
            pg, r = [a for a, _ in at], [c for _, c in at]
            assert torch.equal(x[pg, :, r].view(torch.uint8), y[pg, :, r].view(torch.uint8)), n
    # and the plain attention of the next token over either cache is the same
    q = L.append(L.cache, root[:, None].contiguous(), lens)
    L.append(other, root[:, None].contiguous(), lens)
    a, c = (x.attend(q, L.table, lens + 1, D ** -0.5) for x in (L.cache, other))
    assert torch.equal(a, c)


@pytest.mark.parametrize("rows", [6, 600])
def test_captured_step_replays(gpu, rows):
    """The four calls captured once and replayed with other tokens, trees, lengths and numbers, with eager calls and
    synchronisations between, against the same calls made eagerly."""
    B, S, H, HK, D = (2, 3, 8, 2, 64) if rows == 6 else (30, 20, 8, 2, 64)
    V = 40000 if rows == 6 else 300  # few long rows are shared by workgroups
    L, E = (Loop(gpu, 7, B, S, H, HK, D, torch.bfloat16, False, V=V) for _ in range(2))
    rng = np.random.default_rng(7)

    def inputs():
        parent, depth = trees(rng, B, S)
        return [torch.tensor(x, dtype=torch.int32) for x in (rng.integers(0, V, (B, S)), parent, depth,
                                                             rng.integers(0, 100, B))] + [torch.rand(B, S)]

    held = [x.to(gpu) for x in inputs()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        L.step(*held, temperature=0.8, top_k=40)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = L.step(*held, temperature=0.8, top_k=40)
    L.cache.k.zero_(), L.cache.v.zero_(), E.cache.k.zero_(), E.cache.v.zero_()
    L.cache.weights.zero_(), L.cache.positions.zero_(), E.cache.weights.zero_(), E.cache.positions.zero_()
    for turn in range(5):
        fresh = inputs()
        if turn == 3:
            fresh[3] = torch.zeros(B, dtype=torch.int32)  # no prefix
        for x, y in zip(held, fresh):
            x.copy_(y)
        graph.replay()
        want = E.step(*[x.to(gpu) for x in fresh], temperature=0.8, top_k=40)
        torch.cuda.synchronize()
        for x, y in zip((*got[:1], got[2], *got[3]), (*want[:1], want[2], *want[3])):
            assert torch.equal(x, y), turn
        assert torch.equal(L.cache.k, E.cache.k) and torch.equal(L.cache.positions, E.cache.positions)


def test_two_streams_at_once(gpu):
    """Two loops on streams of their own, without a wait between them, each with its own workspaces, give what they give alone."""
    loops = [Loop(gpu, 20 + i, 4, 12, 16, 2, 128, torch.bfloat16, False, V=40000) for i in range(2)]
    alone = [Loop(gpu, 20 + i, 4, 12, 16, 2, 128, torch.bfloat16, False, V=40000) for i in range(2)]
    rng = np.random.default_rng(1)
    args = []
    for _ in range(2):
        parent, depth = trees(rng, 4, 12)
        args.append([torch.tensor(x, dtype=torch.int32, device=gpu) for x in
                     (rng.integers(0, 40000, (4, 12)), parent, depth, [0, 40, 99, 120])] + [torch.rand(4, 12, device=gpu)])
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for _ in range(4):
        for L, s, a in zip(loops, streams, args):
            with torch.cuda.stream(s):
                got.append(L.step(*a, top_p=0.9))
    torch.cuda.synchronize()
    for i in range(2):
        for t in range(4):
            want = alone[i].step(*args[i], top_p=0.9)
            x = got[2 * t + i]
            assert torch.equal(x[0], want[0]) and torch.equal(x[2], want[2])
            assert all(torch.equal(p, q) for p, q in zip(x[3], want[3]))


def test_calls_with_workspace_and_out_allocate_nothing(gpu):
    L = Loop(gpu, 3, 2, 9, 16, 2, 64, torch.bfloat16, False, V=40000)
    rng = np.random.default_rng(3)
    parent, depth = (torch.tensor(x, dtype=torch.int32, device=gpu) for x in trees(rng, 2, 9))
    tokens = torch.tensor(rng.integers(0, 40000, (2, 9)), dtype=torch.int32, device=gpu)
    lens = torch.tensor([5, 70], dtype=torch.int32, device=gpu)
    u = torch.rand(18, device=gpu)
    logits = torch.randn(18, 40000, device=gpu)
    q, k, v = L.split(tokens)
    pos, total = lens[:, None] + depth, lens + 9
    out = torch.empty(2, 9, 16, 64, dtype=torch.bfloat16, device=gpu)
    heard = torch.empty_like(out)
    ws = torch.empty(L.cache.attend_tree_workspace_bytes(2, 9, 16, L.table.shape[1]), dtype=torch.uint8, device=gpu)
    sw = torch.empty(kernels.sample_workspace_bytes(18, 40000), dtype=torch.uint8, device=gpu)
    so = torch.empty(18, dtype=torch.int32, device=gpu), torch.empty(18, device=gpu)
    ao = lens.clone(), tokens.clone(), tokens.clone()
    torch.cuda.synchronize()
    before = torch.cuda.memory_stats()["allocation.all.allocated"]
    o = L.cache.append(q, k, v, L.table, lens, L.freqs, position=pos, q_norm=L.qn, k_norm=L.kn, out=out)
    a = L.cache.attend_tree(o, L.table, total, parent, 0.1, out=heard, workspace=ws)
    t = kernels.sample(logits, u, top_p=0.9, out=so, workspace=sw)
    r = L.cache.accept(tokens, parent, so[0].view(2, 9), L.table, lens, out=ao)
    torch.cuda.synchronize()
    assert torch.cuda.memory_stats()["allocation.all.allocated"] == before
    assert o is out and t is so and r is ao and a is heard
    with pytest.raises(Exception, match="workspace of 64 bytes"):
        kernels.sample(logits, u, workspace=sw[:64])
    with pytest.raises(ValueError, match="contiguous uint8"):
        kernels.sample(logits, u, workspace=sw[::2])
    # what a smaller call left in the workspace does not count
    want = kernels.sample(logits[:3], u[:3], top_p=0.9)
    kernels.sample(logits, u, temperature=0.0, workspace=sw)
    ws3 = sw if sw.numel() >= kernels.sample_workspace_bytes(3, 40000) else None
    got = kernels.sample(logits[:3], u[:3], top_p=0.9, workspace=ws3)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
