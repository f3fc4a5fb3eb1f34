"""The operators of a step that verifies drafted tokens over a paged cache: the new tokens' norms,
rotation and write, the attention of a tree of drafted tokens, the sampling of the tokens that follow
each of them, and the acceptance of the path that the samples agree with, through
``wanferenz_amd.paged.PagedKV`` and ``wanferenz_amd.kernels.sample``.

Pools are [pages, kv heads, page, head dim], a sequence's slot t lies in row t % page of page
table[b, t // page]; pages are handed out in random order.  Widths are the V4-Flash latent (64 heads on
one shared row of 512, its last 64 dimensions rotated) and the generic grouped layouts (8 KV heads of 64
or 128 with 4 or 8 query heads each); vocabularies are generic.

Kinds of case:
  append  q, k and v, views of a fused projection's rows: q and k normed for each head and rotated, k and v
          written into their pages (bf16 or e4m3)
  tree    q [B, S, H, D], the S drafted tokens of a tree, against the cached prefix and their own ancestors
  sample  one token a row of logits by temperature, min-p, top-k and top-p from a given uniform number
  accept  the walk down the tree along the sampled tokens, and its rows moved to the prefix's end
"""

import math
import random

import numpy as np
import torch

own = False

EPS = 1e-6


def listed():
    cache = {"e4m3": False, "shared": False, "page": 64, "spread": 0.0, "pad": False}

    def append(name, B, S, H, HK, D, R, n, **more):
        return {"name": name, "kind": "append", **cache, "B": B, "S": S, "H": H, "HK": HK, "D": D, "R": R, "n": n,
                "halves": True, "leading": True, "tree": False, **more}

    def tree(name, B, S, H, HK, D, n, **more):
        return {"name": name, "kind": "tree", **cache, "B": B, "S": S, "H": H, "HK": HK, "D": D, "n": n, "sink": False,
                **more}

    def sample(name, rows, V, **more):
        return {"name": name, "kind": "sample", "rows": rows, "V": V, "bf16": False, "t": 1.0, "k": 0, "p": 1.0, "m": 0.0,
                "mixed": False, **more}

    def accept(name, B, S, HK, D, n, **more):
        return {"name": name, "kind": "accept", **cache, "B": B, "S": S, "HK": HK, "D": D, "n": n, **more}

    return [
        # one decode step of a serving batch, at mixed lengths
        append("append_step_b64", 64, 1, 32, 8, 128, 128, 8000, page=16, spread=6.0),
        # the drafted trees of a batch into an 8-bit cache of narrow heads, rotated in part, at their depths
        append("append_tree_e4m3", 16, 31, 64, 8, 64, 32, 9001, e4m3=True, page=32, spread=3.0, tree=True),
        # a long prompt of V4-Flash heads and latents
        append("append_prompt_latent", 1, 8191, 64, 1, 512, 64, 0, shared=True, halves=False, leading=False),
        # one user's chat, sixteen drafted tokens: the smallest call
        tree("tree_b1_s16", 1, 16, 32, 8, 128, 999, page=16),
        # wide trees over a batch of long sequences: the products count
        tree("tree_b8_s64", 8, 64, 64, 8, 128, 8191),
        # trees of different sizes on an 8-bit cache of narrow heads at mixed lengths, with sinks
        tree("tree_b24_e4m3", 24, 24, 64, 8, 64, 9001, e4m3=True, page=32, spread=3.0, sink=True, pad=True),
        # V4-Flash heads, eight drafted tokens over the whole latent cache
        tree("tree_latent_b4", 4, 8, 64, 1, 512, 16383, shared=True, sink=True),
        # one user's next token, the usual filters: latency
        sample("sample_b1", 1, 131072, t=0.7, k=50, p=0.9),
        # a serving batch, each row with its own temperature and filters, bf16 logits
        sample("sample_b64_mixed", 64, 131072, bf16=True, mixed=True),
        # every node of a batch of trees, filtered by the mass alone over an odd vocabulary
        sample("sample_b512_top_p", 512, 100003, p=0.95),
        # the accepted path of one chat
        accept("accept_b1_s16", 1, 16, 8, 128, 999, page=16),
        # the accepted paths of a batch of wide trees
        accept("accept_b64_s64", 64, 64, 8, 128, 501, spread=1.0),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("append", "tree", "tree", "sample", "accept"))
    if kind == "sample":
        V = _log_int(rng, 1000, 200_000)
        return {"kind": kind, "rows": _log_int(rng, 1, min(1024, 50_000_000 // V)), "V": V, "bf16": rng.random() < 0.5,
                "t": round(rng.uniform(0.3, 1.5), 2), "k": rng.choice((0, 0, 1, 20, 50, 400)),
                "p": rng.choice((1.0, 0.95, 0.9, 0.5)), "m": rng.choice((0.0, 0.0, 0.02, 0.1)),
                "mixed": rng.random() < 0.3}
    shared = rng.random() < 0.3
    D = 512 if shared else rng.choice((64, 128, 128))
    HK = 1 if shared else rng.choice((1, 2, 4, 8, 8))
    H = rng.choice((16, 32, 64)) if shared else HK * rng.choice((1, 3, 4, 8))
    case = {"kind": kind, "e4m3": rng.random() < 0.4, "shared": shared, "page": rng.choice((16, 16, 32, 64, 256)),
            "spread": rng.choice((0.0, 1.0, 4.0)), "pad": rng.random() < 0.3, "H": H, "HK": HK, "D": D}
    if kind == "append":
        case["tree"] = rng.random() < 0.3
        case["R"] = rng.choice((D, D // 2, 32))
        case["halves"], case["leading"] = rng.random() < 0.6, rng.random() < 0.5
        if not case["tree"] and rng.random() < 0.3:
            case["B"], case["n"] = 1 if shared else rng.randint(1, 3), rng.choice((0, 77))
            case["S"] = _log_int(rng, 100, 8191)
        else:
            case["B"], case["n"] = _log_int(rng, 1, 120), _log_int(rng, 1, 9001)
            case["S"] = rng.randint(2, 64) if case["tree"] else rng.choice((1, 1, 4))
        return case
    case["S"] = rng.randint(2, 64)
    if kind == "tree":
        case["sink"] = rng.random() < 0.4
        case["B"] = _log_int(rng, 1, 32)
        most = 120_000_000_000 // (4 * case["B"] * case["S"] * H * D)
        row = HK * D * (2 - shared) * 2 * case["B"]
        case["n"] = _log_int(rng, 64, max(65, min(32767, most, 500_000_000 // row)))
    else:
        del case["H"]
        case["B"] = _log_int(rng, 1, 64)
        case["n"] = _log_int(rng, 1, 1000)
    return case


def _spread_out(case):
    """A fixed spread-out sequence in [0, 1), so that the work is known without the inputs."""
    return [((b + 1) * 0.6180339887498949) % 1.0 for b in range(case["B"])]


def _lengths(case):
    """Tokens that each sequence holds before the new ones: n for the longest, down to n / 2^spread."""
    lens = [int(case["n"] * 2.0 ** (-case["spread"] * f)) for f in _spread_out(case)]
    lens[0] = case["n"]
    return lens


def _counts(case):
    """New tokens of each sequence: S, or with pad from 1 on."""
    return [1 + int(f * case["S"]) if case["pad"] else case["S"] for f in _spread_out(case)]


def _trees(case):
    """(parents, depths) of each sequence's S nodes: a parent precedes its children, near ones are likelier."""
    rng = random.Random(1000 * case["B"] + case["S"])
    parents, depths = [], []
    for _ in range(case["B"]):
        parent, depth = [-1], [0]
        for i in range(1, case["S"]):
            parent.append(max(0, i - 1 - int(rng.random() ** 2 * i)))
            depth.append(depth[parent[-1]] + 1)
        parents.append(parent)
        depths.append(depth)
    return parents, depths


def _targets(case):
    """The node of each sequence at which the samples leave its tree."""
    return [int(f * n) for f, n in zip(_spread_out({"B": case["B"]}), _counts(case))]


# ---------------------------------------------------------------- inputs ------


def _pools(st, case, g):
    dev, B, S, HK, D, page = "cuda", *(case[k] for k in ("B", "S", "HK", "D", "page"))
    lens = _lengths(case)
    width = -(-(max(lens) + S) // page)
    held = [-(-(n + S) // page) for n in lens]
    pages = sum(held) + 3
    order = torch.randperm(pages, device=dev, generator=g).to(torch.int32)
    at = (torch.arange(width)[None, :] < torch.tensor(held)[:, None]).to(dev)
    first = torch.cumsum(torch.tensor([0] + held[:-1]), 0).to(dev)
    place = (first[:, None] + torch.arange(width, device=dev)[None, :]).clamp(max=pages - 1)
    st["table"] = torch.where(at, order[place], -1).to(torch.int32).contiguous()

    def pool():
        x = torch.randn(pages, HK, page, D, device=dev, generator=g, dtype=torch.bfloat16)
        if not case["e4m3"]:
            return x, None
        x = x.float()
        s = x.abs().amax(-1).clamp(min=1e-4) * (1.0 / 448.0)
        return (x / s[..., None]).clamp(-448.0, 448.0).to(torch.float8_e4m3fn), s

    st["k"], st["ks"] = pool()
    st["v"], st["vs"] = (st["k"], st["ks"]) if case["shared"] else pool()
    st["start"] = torch.tensor(lens, dtype=torch.int32, device=dev)
    st["count"] = torch.tensor(_counts(case), dtype=torch.int32, device=dev) if case["pad"] else None


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed((int(seed) * 1013 + 41) & 0x7FFFFFFF)
    dev, st = "cuda", {"case": dict(case)}
    if case["kind"] == "sample":
        # what a language model's head gives: a broad bulk, and a few dozen tokens that stand out of it
        n, V = case["rows"], case["V"]
        x = torch.randn(n, V, device=dev, generator=g).mul_(2.0)
        likely = torch.randint(0, V, (n, 48), device=dev, generator=g)
        lift = torch.rand(n, 48, device=dev, generator=g).mul_(10.0).add_(6.0)
        x.scatter_(1, likely, x.gather(1, likely) + lift)
        st["logits"] = x.to(torch.bfloat16) if case["bf16"] else x
        st["u"] = torch.rand(n, device=dev, generator=g)
        if case["mixed"]:
            r = torch.rand(4, n, device=dev, generator=g)
            st["t"] = torch.where(r[0] < 0.15, 0.0, 0.4 + r[0])  # some rows are greedy
            st["k"] = torch.where(r[1] < 0.4, 0, (r[1] * 200).to(torch.int32)).to(torch.int32)
            st["p"] = torch.where(r[2] < 0.3, 1.0, 0.5 + 0.5 * r[2])
            st["m"] = torch.where(r[3] < 0.6, 0.0, 0.1 * r[3])
        else:
            st["t"], st["k"], st["p"], st["m"] = case["t"], case["k"], case["p"], case["m"]
        return st
    B, S, HK, D = (case[k] for k in ("B", "S", "HK", "D"))
    _pools(st, case, g)
    parents, depths = _trees(case)
    st["parent"] = torch.tensor(parents, dtype=torch.int32, device=dev)
    if case["kind"] == "append":
        H, R = case["H"], case["R"]
        rows = torch.randn(B, S, (H + (2 - case["shared"]) * HK) * D, device=dev, generator=g).to(torch.bfloat16)
        st["q"] = rows[..., :H * D].view(B, S, H, D)
        st["new_k"] = rows[..., H * D:(H + HK) * D].view(B, S, HK, D)
        st["new_v"] = None if case["shared"] else rows[..., (H + HK) * D:].view(B, S, HK, D)
        st["q_norm"] = 1.0 + 0.2 * torch.randn(D, device=dev, generator=g)
        st["k_norm"] = 1.0 + 0.2 * torch.randn(D, device=dev, generator=g)
        turn = torch.arange(case["n"] + S, dtype=torch.float64, device=dev)[:, None]
        freq = 10000.0 ** (-torch.arange(0, R, 2, dtype=torch.float64, device=dev) / R)
        st["freqs"] = torch.polar(torch.ones_like(turn * freq), turn * freq).to(torch.complex64)
        st["position"] = None
        if case["tree"]:
            st["position"] = st["start"][:, None] + torch.tensor(depths, dtype=torch.int32, device=dev)
    elif case["kind"] == "tree":
        # q is a view of the rows of a fused projection where K and V come from one too
        rest = 0 if case["shared"] else 2 * HK
        rows = torch.randn(B, S, (case["H"] + rest) * D, device=dev, generator=g).mul_(1.5).to(torch.bfloat16)
        st["q"] = rows[..., :case["H"] * D].view(B, S, case["H"], D)
        st["lens"] = st["start"] + (st["count"] if case["pad"] else S)
        st["sink"] = torch.randn(case["H"], device=dev, generator=g) + 0.5 if case["sink"] else None
        st["scale"] = D ** -0.5
    else:
        # the samples agree with the drafted tokens down to one node, and with no other branch
        st["sampled"] = torch.randint(0, 100_000, (B, S), device=dev, generator=g, dtype=torch.int32)
        before = torch.gather(st["sampled"], 1, st["parent"].clamp(min=0).long())
        on = np.zeros((B, S), dtype=bool)
        for b, node in enumerate(_targets(case)):
            while node >= 0:
                on[b, node] = True
                node = parents[b][node]
        st["drafted"] = torch.where(torch.from_numpy(on).to(dev), before, before + 1).to(torch.int32)
    return st


# ---------------------------------------------------------------- plain forms --


def _places(table, slots, page):
    """(page, row) of slots [B, ...] of the sequences; page -1 where there is none."""
    B = table.shape[0]
    p = (slots // page).view(B, -1).long()
    pg = torch.gather(table, 1, p.clamp(0, table.shape[1] - 1))
    return torch.where(p < table.shape[1], pg, -1).view(slots.shape).long(), (slots % page).long()


def _norm(x, w):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w


def _rotate(x, cos, sin, c):
    """x [B, S, heads, D]; cos, sin [B, S, 1, R / 2]."""
    R, lo = c["R"], 0 if c["leading"] else c["D"] - c["R"]
    y = x.clone()
    if c["halves"]:
        i, j = slice(lo, lo + R // 2), slice(lo + R // 2, lo + R)
    else:
        i, j = slice(lo, lo + R, 2), slice(lo + 1, lo + R, 2)
    y[..., i] = x[..., i] * cos - x[..., j] * sin
    y[..., j] = x[..., i] * sin + x[..., j] * cos
    return y


def _plain_append(st):
    c = st["case"]
    B, S = c["B"], c["S"]
    step = torch.arange(S, device="cuda", dtype=torch.int32)
    slots = st["start"][:, None] + step
    pos = slots if st["position"] is None else st["position"]
    turn = torch.view_as_real(st["freqs"])[pos.long()][:, :, None]
    cos, sin = turn[..., 0], turn[..., 1]
    q = _rotate(_norm(st["q"].float(), st["q_norm"]), cos, sin, c).to(torch.bfloat16)
    k = _rotate(_norm(st["new_k"].float(), st["k_norm"]), cos, sin, c)
    pg, r = _places(st["table"], slots, c["page"])
    if st["count"] is not None:
        live = step < st["count"][:, None]
        q = torch.where(live[:, :, None, None], q, 0.0)
        # a row that is not written is put back
    else:
        live = None
    heads = torch.arange(c["HK"], device="cuda")
    at = (pg[..., None], heads, r[..., None])
    sides = [("k", "ks", k)] + ([] if c["shared"] else [("v", "vs", st["new_v"].float())])
    for pool, scale, x in sides:
        if scale and st[scale] is not None:
            s = x.abs().amax(-1).clamp(min=1e-4) * (1.0 / 448.0)
            code = (x / s[..., None]).clamp(-448.0, 448.0).to(torch.float8_e4m3fn).view(torch.uint8)
            old = st[pool].view(torch.uint8)
            if live is not None:
                code = torch.where(live[:, :, None, None], code, old[at])
                s = torch.where(live[:, :, None], s, st[scale][at])
            old[at] = code
            st[scale][at] = s
        else:
            x = x.to(torch.bfloat16)
            st[pool][at] = x if live is None else torch.where(live[:, :, None, None], x, st[pool][at])
    return {"q": q, **_state_of(st)}


def _rows_of(pool, scale, table, n):
    """[B, HK, n, D] of the first n slots of every sequence, 32 bits."""
    page = pool.shape[2]
    pages = table[:, :-(-n // page)].clamp(min=0).long()
    x = pool[pages].permute(0, 2, 1, 3, 4).reshape(pages.shape[0], pool.shape[1], -1, pool.shape[3])[:, :, :n].float()
    if scale is not None:
        x = x * scale[pages].permute(0, 2, 1, 3).reshape(x.shape[0], x.shape[1], -1)[:, :, :n, None]
    return x


def _ancestors(parent):
    """[B, S, S]: whether node j is node i or above it."""
    node = torch.arange(parent.shape[1], device=parent.device)
    step = (node[:, None] == node)[None] | (parent[:, :, None] == node)
    return torch.linalg.matrix_power(step.float(), 64) > 0  # 64 steps up reach the root of 64 nodes


def _plain_tree(st):
    c = st["case"]
    B, S, H, HK = (c[k] for k in ("B", "S", "H", "HK"))
    n, g, dev = max(_lengths(c)) + S, c["H"] // c["HK"], "cuda"
    K = _rows_of(st["k"], st["ks"], st["table"], n)
    V = K if c["shared"] else _rows_of(st["v"], st["vs"], st["table"], n)
    node = torch.arange(S, device=dev)
    count = torch.full((B,), S, device=dev) if st["count"] is None else st["count"]
    first = (st["lens"] - count)[:, None, None]
    rel = torch.arange(n, device=dev)[None, None, :] - first  # [B, 1, n]
    seen = torch.gather(_ancestors(st["parent"]), 2, rel.clamp(0, S - 1).expand(B, S, n))
    seen = (rel < 0) | (seen & (rel < count[:, None, None]))
    live = (node < count[:, None])[:, :, None]
    seen = seen & live
    q = st["q"].float().view(B, S, HK, g, -1).permute(0, 2, 1, 3, 4).reshape(B, HK, S * g, -1)
    s = torch.matmul(q, K.transpose(-1, -2).contiguous()) * st["scale"]
    s = torch.where(seen[:, None, :, None, :].expand(B, 1, S, g, n).reshape(B, 1, S * g, n), s, -math.inf)
    m = s.amax(-1, keepdim=True)
    if c["sink"]:
        sink = st["sink"].view(1, HK, 1, g, 1).expand(B, HK, S, g, 1).reshape(B, HK, S * g, 1)
        m = torch.maximum(m, sink)
    m = torch.where(m == -math.inf, 0.0, m)
    e = torch.exp(s - m)
    den = e.sum(-1, keepdim=True)
    if c["sink"]:
        den = den + torch.exp(sink - m)
    p = e / torch.where(den == 0, 1.0, den)
    return torch.matmul(p, V).view(B, HK, S, g, -1).permute(0, 2, 1, 3, 4).reshape(B, S, H, -1).to(torch.bfloat16)


def _plain_sample(st):
    """The order is by logit, equal ones by index; every filter keeps a first part of it."""
    x = st["logits"].float()
    n, V = x.shape
    t, p, m = (torch.as_tensor(st[k], dtype=torch.float32, device=x.device).double().expand(n)[:, None]
               for k in ("t", "p", "m"))
    k = torch.as_tensor(st["k"], device=x.device).expand(n)[:, None]
    order = torch.sort(x, dim=1, descending=True, stable=True)
    z = order.values.double()
    w = torch.exp((z - z[:, :1]) / torch.where(t == 0, 1.0, t))
    place = torch.arange(V, device=x.device)
    w = torch.where((w >= m) & ((k <= 0) | (place < k)) & ((t != 0) | (place == 0)), w, 0.0)
    total = torch.cumsum(w, 1)
    w = torch.where((place == 0) | (p >= 1.0) | (total - w < p * total[:, -1:]), w, 0.0)
    total = torch.cumsum(w, 1)
    at = (total <= st["u"].double()[:, None] * total[:, -1:]).sum(1, keepdim=True)
    at = torch.minimum(at, (w > 0).sum(1, keepdim=True) - 1)
    prob = (w.gather(1, at) / total[:, -1:]).float()[:, 0]
    return {"token": order.indices.gather(1, at)[:, 0].to(torch.int32), "prob": prob}


def _plain_accept(st):
    c = st["case"]
    B, S = c["B"], c["S"]
    node = torch.arange(S, device="cuda")
    count = torch.full((B,), S, device="cuda") if st["count"] is None else st["count"]
    # a node is taken if it and all above it have the token that was sampled at their parent, up to the root
    astray = (st["drafted"] != torch.gather(st["sampled"], 1, st["parent"].clamp(min=0).long())) & (node > 0)
    up = _ancestors(st["parent"])
    taken = up[:, :, 0] & ~(up & astray[:, None, :]).any(-1) & (node < count[:, None])
    m = taken.sum(1)
    path = torch.sort(torch.where(taken, node, S), dim=1).values
    on = node < m[:, None]
    tokens = torch.where(on, torch.gather(st["sampled"], 1, path.clamp(max=S - 1)), -1)
    fro = torch.where(on, path, node)  # past the path a slot is put back onto itself
    heads = torch.arange(c["HK"], device="cuda")
    fpg, fr = _places(st["table"], st["start"][:, None] + fro, c["page"])
    tpg, tr = _places(st["table"], st["start"][:, None] + node, c["page"])
    for x in [st["k"], st["ks"]] + ([] if c["shared"] else [st["v"], st["vs"]]):
        if x is not None:
            x = x.view(torch.uint8) if x.dtype == torch.float8_e4m3fn else x
            x[tpg[..., None], heads, tr[..., None]] = x[fpg[..., None], heads, fr[..., None]]
    return {"lens": (st["start"] + m).to(torch.int32), "tokens": tokens.to(torch.int32),
            "path": torch.where(on, path, -1).to(torch.int32), **_state_of(st)}


# ---------------------------------------------------------------- passes ------


def _cache(st):
    """The handle on the pools that a program keeps."""
    if "cache" not in st:
        from wanferenz_amd.paged import PagedKV

        st["cache"] = PagedKV(st["k"], None if st["case"]["shared"] else st["v"], k_scale=st["ks"],
                              v_scale=None if st["case"]["shared"] else st["vs"])
    return st["cache"]


def _state_of(st):
    names = ["k", "ks"] + ([] if st["case"]["shared"] else ["v", "vs"])
    return {x: st[x] for x in names if st[x] is not None}


def run(st):
    c = st["case"]
    if not own:
        return {"append": _plain_append, "tree": _plain_tree, "sample": _plain_sample, "accept": _plain_accept}[c["kind"]](st)
    if c["kind"] == "sample":
        from wanferenz_amd import kernels

        token, prob = kernels.sample(st["logits"], st["u"], temperature=st["t"], top_k=st["k"], top_p=st["p"],
                                     min_p=st["m"])
        return {"token": token, "prob": prob}
    cache = _cache(st)
    if c["kind"] == "append":
        q = cache.append(st["q"], st["new_k"], st["new_v"], st["table"], st["start"], st["freqs"], count=st["count"],
                         position=st["position"], q_norm=st["q_norm"], k_norm=st["k_norm"], eps=EPS,
                         halves=c["halves"], leading=c["leading"])
        return {"q": q, **_state_of(st)}
    if c["kind"] == "tree":
        return cache.attend_tree(st["q"], st["table"], st["lens"], st["parent"], st["scale"], attn_sink=st["sink"],
                                 count=st["count"])
    lens, tokens, path = cache.accept(st["drafted"], st["parent"], st["sampled"], st["table"], st["start"],
                                      count=st["count"])
    return {"lens": lens, "tokens": tokens, "path": path, **_state_of(st)}


def work(case):
    if case["kind"] == "sample":
        n, V = case["rows"], case["V"]
        return {"bytes": n * (V * (2 if case["bf16"] else 4) + 28), "flops": 3 * n * V}
    B, S, HK, D = (case[k] for k in ("B", "S", "HK", "D"))
    sides = 1 if case["shared"] else 2
    row = sides * (D + 4 if case["e4m3"] else 2 * D)  # of one slot and head
    lens, counts = _lengths(case), _counts(case)
    _, depths = _trees(case)
    if case["kind"] == "append":
        new = sum(counts)
        turns = sum(len({n + d for d in dep[:c]}) for n, c, dep in zip(lens, counts, depths)) if case["tree"] else new
        nbytes = (2 * B * S + 2 * new) * case["H"] * D + new * HK * (sides * 2 * D + row) + turns * 4 * case["R"] + 8 * D
        return {"bytes": nbytes, "flops": new * (case["H"] + HK) * (4 * D + 3 * case["R"])}
    if case["kind"] == "tree":
        H = case["H"]
        flops = sum(4 * H * D * (n + dep[i] + 1) for n, c, dep in zip(lens, counts, depths) for i in range(c))
        pages = sum(-(-(n + c) // case["page"]) for n, c in zip(lens, counts))
        nbytes = (sum(lens) + sum(counts)) * HK * row + 2 * (sum(counts) + B * S) * H * D + 4 * (pages + 2 * B + B * S)
        return {"bytes": nbytes, "flops": flops}
    parents, _ = _trees(case)
    moved = 0
    for b, node in enumerate(_targets(case)):
        while node >= 0:
            moved += node != depths[b][node]
            node = parents[b][node]
    return {"bytes": moved * HK * 2 * row + B * S * 20 + 8 * B, "flops": B * S}


# ---------------------------------------------------------------- 64 bits -----


def _exact_append(st):
    c = st["case"]
    B, S, D, R, page = (c[k] for k in ("B", "S", "D", "R", "page"))
    lens, counts = _lengths(c), _counts(c)
    lo = 0 if c["leading"] else D - R
    pair = torch.arange(R // 2, device="cuda")
    i = lo + (pair if c["halves"] else 2 * pair)
    j = i + (R // 2 if c["halves"] else 1)

    def turned(x, w, z):
        x = x.double()
        x = x / torch.sqrt(torch.mean(x * x, dim=-1, keepdim=True) + EPS) * w.double()
        y = torch.complex(x[..., i], x[..., j]) * z
        x[..., i], x[..., j] = y.real, y.imag
        return x

    out = {"q": torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")}
    out |= {name: x.double() for name, x in _state_of(st).items()}
    for b in range(B):
        t, n = lens[b], counts[b]
        pos = torch.arange(t, t + n, device="cuda") if st["position"] is None else st["position"][b, :n].long()
        z = st["freqs"][pos].to(torch.complex128)[:, None]
        out["q"][b, :n] = turned(st["q"][b, :n], st["q_norm"], z)
        new = [("k", "ks", turned(st["new_k"][b, :n], st["k_norm"], z))]
        if not c["shared"]:
            new.append(("v", "vs", st["new_v"][b, :n].double()))
        for p in range(t // page, (t + n - 1) // page + 1):
            a, e = max(t, p * page), min(t + n, (p + 1) * page)
            pg = int(st["table"][b, p])
            for pool, scale, x in new:
                rows = x[a - t:e - t].transpose(0, 1)
                if c["e4m3"]:
                    s = rows.abs().amax(-1).clamp(min=1e-4) / 448.0
                    out[scale][pg, :, a - p * page:e - p * page] = s
                    rows = (rows / s[..., None]).float().to(torch.float8_e4m3fn).double()
                out[pool][pg, :, a - p * page:e - p * page] = rows
    return out


def _exact_tree(st):
    c = st["case"]
    B, S, H, HK, D, page = (c[k] for k in ("B", "S", "H", "HK", "D", "page"))
    g = H // HK
    parents, _ = _trees(c)
    o = torch.zeros(B, S, H, D, dtype=torch.float64, device="cuda")
    for b, (t, n) in enumerate(zip(_lengths(c), _counts(c))):
        pages = st["table"][b, :-(-(t + n) // page)].long()

        def rows(pool, scale):
            x = pool[pages].double()
            if scale is not None:
                x = x * scale[pages].double()[..., None]
            return x.transpose(0, 1).reshape(HK, -1, D)[:, :t + n].contiguous()

        K = rows(st["k"], st["ks"])
        V = K if c["shared"] else rows(st["v"], st["vs"])
        hidden = np.ones((n, n), dtype=bool)
        for i in range(n):
            a = i
            while a >= 0:
                hidden[i, a] = False
                a = parents[b][a]
        q = st["q"][b, :n].double().reshape(n, HK, g, D).permute(1, 0, 2, 3).reshape(HK, n * g, D)
        s = torch.bmm(K, q.transpose(1, 2).contiguous()).transpose(1, 2).reshape(HK, n, g, t + n) * st["scale"]
        s[..., t:] = s[..., t:].masked_fill(torch.from_numpy(hidden).cuda()[None, :, None, :], -math.inf)
        if c["sink"]:
            s = torch.cat([s, st["sink"].double().view(HK, 1, g, 1).expand(HK, n, g, 1)], dim=3)
        p = torch.softmax(s, dim=3)[..., :t + n].reshape(HK, n * g, t + n).contiguous()
        o[b, :n] = torch.bmm(p, V).view(HK, n, g, D).permute(1, 0, 2, 3).reshape(n, H, D)
    return o


def _exact_sample(st):
    x = st["logits"].float().cpu().numpy().astype(np.float64)
    n = x.shape[0]
    t, k, p, m, u = (np.broadcast_to(np.asarray(torch.as_tensor(v).cpu(), dtype=np.float32), (n,)).astype(np.float64)
                     for v in (st["t"], st["k"], st["p"], st["m"], st["u"]))
    token, prob = np.zeros(n, dtype=np.int32), np.zeros(n)
    for r in range(n):
        row = x[r]
        if t[r] == 0:
            token[r], prob[r] = int(np.argmax(row)), 1.0
            continue
        order = np.argsort(-row, kind="stable")
        w = np.exp((row[order] - row[order[0]]) / t[r])
        keep = len(w) if k[r] <= 0 else min(len(w), int(k[r]))
        w = w[:keep]
        w = w[w >= m[r]]
        if p[r] < 1.0:
            w = w[:max(1, int(np.searchsorted(np.cumsum(w), p[r] * np.cumsum(w)[-1], side="left")) + 1)]
        acc = np.cumsum(w)
        at = min(int(np.searchsorted(acc, u[r] * acc[-1], side="right")), len(w) - 1)
        token[r], prob[r] = order[at], w[at] / acc[-1]
    return {"token": torch.from_numpy(token).cuda(), "prob": torch.from_numpy(prob).cuda()}


def _exact_accept(st):
    c = st["case"]
    B, S, page = c["B"], c["S"], c["page"]
    drafted, sampled, table = (st[k].cpu().tolist() for k in ("drafted", "sampled", "table"))
    parents, _ = _trees(c)
    out = {name: x.double() for name, x in _state_of(st).items()}
    lens, tokens, paths = [], [], []
    for b, (t, n) in enumerate(zip(_lengths(c), _counts(c))):
        path = [0]
        while True:
            last = path[-1]
            more = [i for i in range(n) if parents[b][i] == last and drafted[b][i] == sampled[b][last]]
            if not more:
                break
            path.append(more[0])
        for i, node in enumerate(path):
            to, fro = t + i, t + node
            for x in out.values():
                x[table[b][to // page], :, to % page] = x[table[b][fro // page], :, fro % page]
        lens.append(t + len(path))
        tokens.append([sampled[b][i] for i in path] + [-1] * (S - len(path)))
        paths.append(path + [-1] * (S - len(path)))
    whole = [torch.tensor(v, dtype=torch.int32, device="cuda") for v in (lens, tokens, paths)]
    return {"lens": whole[0], "tokens": whole[1], "path": whole[2], **out}


def exact(case, seed):
    st = prepare(case, seed)
    return {"append": _exact_append, "tree": _exact_tree, "sample": _exact_sample, "accept": _exact_accept}[case["kind"]](st)
