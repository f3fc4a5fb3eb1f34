"""The paged key-value cache's operators as a serving loop runs them: the write of new tokens,
the attention of one or a few new tokens over the cache, and the eviction of the tokens that
attention has weighed least, through ``wanferenz_amd.paged.PagedKV``.

Pools are [pages, kv heads, page, head dim], a sequence's slot t lies in row t % page of page
table[b, t // page]; pages are handed out in random order.  Widths are the V4-Flash latent
(64 heads on one shared row of 512, as the sparse attention's cases) and the generic grouped
layouts (8 KV heads of 64 or 128 with 4 or 8 query heads each).

Kinds of case:
  attend  q [B, S, H, D] against every cached token, S new tokens causal among themselves,
          bf16 or e4m3 rows, with or without a sink, the weight that each cached token gets
          added to an accumulator where the cache is tracked
  write   the new tokens' K and V, views of a fused projection's rows, into their pages
  evict   a pass of a loop with a budget: new tokens written, then the cache cut to `keep`
"""

import math

import torch

own = False

SINK_SHARE = 0.5  # sinks are N(0, 1) + this


def listed():
    base = {"S": 1, "spread": 0.0, "e4m3": False, "shared": False, "sink": False, "track": False}

    def attend(name, B, H, HK, D, page, n, **more):
        return {"name": name, "kind": "attend", **base, "B": B, "H": H, "HK": HK, "D": D, "page": page, "n": n, **more}

    def write(name, B, S, HK, D, page, n, **more):
        return {"name": name, "kind": "write", **base, "B": B, "H": HK, "HK": HK, "D": D, "page": page, "n": n, **more,
                "S": S}

    def evict(name, B, HK, D, page, keep, new, **more):
        return {"name": name, "kind": "evict", **base, "B": B, "H": HK, "HK": HK, "D": D, "page": page, "keep": keep,
                "n": new, "track": True, **more}

    return [
        # one user's chat: the smallest call, where the launches and the join count
        attend("attend_b1_n999", 1, 32, 8, 128, 16, 999),
        # one user's long document: a single row of queries, so the length has to fill the chip
        attend("attend_b1_n131071", 1, 32, 8, 128, 64, 131071),
        # a serving batch at mixed lengths, from a few tokens to 16k
        attend("attend_b64_ragged", 64, 64, 8, 128, 64, 16384, spread=10.0),
        # the same kind of batch on an 8-bit cache, narrow heads, with sinks
        attend("attend_b48_e4m3", 48, 64, 8, 64, 32, 9001, spread=3.0, e4m3=True, sink=True),
        # V4-Flash heads over the whole latent cache of four sequences (K = V, sink)
        attend("attend_latent_b4", 4, 64, 1, 512, 64, 65535, shared=True, sink=True),
        # verification of four drafted tokens a sequence
        attend("attend_verify_s4", 16, 32, 8, 128, 64, 8191, S=4),
        # decode under a cache budget: the weights are added up for the eviction
        attend("attend_track_b16", 16, 32, 8, 128, 16, 4160, track=True, spread=1.0),
        # one decode step's write into an 8-bit cache, a batch of 64
        write("write_step_e4m3", 64, 1, 8, 128, 16, 5000, e4m3=True, spread=8.0),
        # a prompt's write, odd length, behind a cached prefix
        write("write_prompt", 2, 8191, 8, 128, 64, 100),
        # the cut of a full budget after 64 decoded tokens (some sequences are not full yet)
        evict("evict_step_b16", 16, 8, 128, 16, 4096, 64, spread=0.5),
        # a long prompt written and cut to a budget
        evict("evict_prompt", 2, 8, 128, 64, 4096, 32767),
        # the same of one sequence's latent rows
        evict("evict_prompt_latent", 1, 1, 512, 64, 8192, 65535, shared=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("attend", "attend", "attend", "write", "evict"))
    shared = rng.random() < 0.3
    D = 512 if shared else rng.choice((64, 128, 128))
    HK = 1 if shared else rng.choice((1, 2, 4, 8, 8))
    H = rng.choice((16, 32, 64)) if shared else HK * rng.choice((1, 3, 4, 8, 16))
    case = {"kind": kind, "S": 1, "spread": rng.choice((0.0, 1.0, 4.0, 10.0)), "e4m3": rng.random() < 0.4,
            "shared": shared, "sink": rng.random() < 0.4, "track": False, "H": H, "HK": HK, "D": D,
            "page": rng.choice((16, 16, 32, 64, 128, 256))}
    row = HK * D * (1 if case["e4m3"] else 2) * (1 if shared else 2)
    if kind == "attend":
        case["S"] = rng.choice((1, 1, 1, 2, 4, 7))
        case["track"] = rng.random() < 0.25
        case["B"] = _log_int(rng, 1, 64)
        case["n"] = _log_int(rng, 64, min(131071, 400_000_000 // (row * case["B"])))
    elif kind == "write":
        if rng.random() < 0.5:
            case["B"], case["S"], case["n"] = _log_int(rng, 1, 256), rng.choice((1, 1, 2, 5)), _log_int(rng, 1, 9001)
        else:
            case["B"], case["S"], case["n"] = rng.randint(1, 4), _log_int(rng, 100, 8191), rng.choice((0, 77))
    else:
        case["track"] = True
        case["keep"] = _log_int(rng, 256, 8192)
        if rng.random() < 0.5:
            case["B"], case["n"] = _log_int(rng, 1, 16), _log_int(rng, 1, min(256, case["keep"] // 4))
        else:
            case["B"] = rng.randint(1, 2)
            case["n"] = _log_int(rng, case["keep"] + 100, 32767)
    return case


def _lengths(case):
    """Tokens that each sequence holds before a pass (attend: in it): n for the longest, down to
    n / 2^spread, by a fixed spread-out sequence, so that the work is known without the inputs."""
    full = case["keep"] if case["kind"] == "evict" else case["n"]
    if case["kind"] == "evict" and case["n"] > case["keep"]:
        return [0] * case["B"]  # a prompt fills the cache from its start
    frac = [((b + 1) * 0.6180339887498949) % 1.0 for b in range(case["B"])]
    lens = [int(full * 2.0 ** (-case["spread"] * (f if case["kind"] != "evict" else max(0.0, f - 0.5)))) for f in frac]
    lens[0] = full
    return lens


def _first_recent(case):
    """The slots of a budget that are kept whatever they weigh."""
    return min(4, case["keep"] // 8), case["keep"] // 4


# ---------------------------------------------------------------- inputs ------


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed((int(seed) * 1009 + 77) & 0x7FFFFFFF)
    dev = "cuda"
    B, S, H, HK, D, page = (case[k] for k in ("B", "S", "H", "HK", "D", "page"))
    lens = _lengths(case)
    new = {"attend": 0, "write": S, "evict": case["n"]}[case["kind"]]
    top = max(lens) + new
    width = -(-top // page)
    every = case["track"] or case["kind"] != "attend"  # pages for the whole table, else for what is held
    held = [width if every else -(-n // page) for n in lens]
    pages = sum(held) + 3
    order = torch.randperm(pages, device=dev, generator=g).to(torch.int32)
    at = (torch.arange(width)[None, :] < torch.tensor(held)[:, None]).to(dev)
    first = (torch.cumsum(torch.tensor([0] + held[:-1]), 0)).to(dev)
    place = (first[:, None] + torch.arange(width, device=dev)[None, :]).clamp(max=pages - 1)
    table = torch.where(at, order[place], -1).to(torch.int32).contiguous()

    st = {"case": dict(case), "table": table, "scale": D ** -0.5, "width": top}

    def pool():
        x = torch.randn(pages, HK, page, D, device=dev, generator=g, dtype=torch.bfloat16)
        if not case["e4m3"]:
            return x, None
        x = x.float()
        s = x.abs().amax(-1).clamp(min=1e-4) * (1.0 / 448.0)
        return (x / s[..., None]).clamp(-448.0, 448.0).to(torch.float8_e4m3fn), s

    st["k"], st["ks"] = pool()
    st["v"], st["vs"] = (st["k"], st["ks"]) if case["shared"] else pool()
    held_t = torch.tensor(lens, dtype=torch.int32, device=dev)
    st["w"] = st["p"] = None
    if case["track"]:
        # what a heavy-tailed attention leaves: a few tokens with most of the weight (attend: after
        # the first few steps, so that one step's weights are of the sums' size)
        st["w"] = torch.randn(pages, HK, page, device=dev, generator=g).mul_(2.0).exp_()
        if case["kind"] == "attend":
            st["w"].mul_(1e-3)
        slot = torch.arange(width * page, dtype=torch.int32, device=dev).view(width, page)
        st["p"] = torch.zeros(pages, HK, page, dtype=torch.int32, device=dev)
        st["p"][table.long()] = (4 * slot)[None, :, None, :].expand(B, width, HK, page)
    if case["kind"] == "attend":
        # q is a view of the rows of a fused projection where K and V come from one too
        rest = 0 if case["shared"] else 2 * HK
        rows = torch.randn(B, S, (H + rest) * D, device=dev, generator=g).mul_(1.5).to(torch.bfloat16)
        st["q"] = rows[..., :H * D].view(B, S, H, D)
        st["lens"] = held_t
        st["sink"] = (torch.randn(H, device=dev, generator=g) + SINK_SHARE) if case["sink"] else None
        return st
    T = S if case["kind"] == "write" else case["n"]
    rows = torch.randn(B, T, (2 - case["shared"]) * HK * D, device=dev, generator=g).to(torch.bfloat16)
    st["new_k"] = rows[..., :HK * D].view(B, T, HK, D)
    st["new_v"] = None if case["shared"] else rows[..., HK * D:].view(B, T, HK, D)
    st["start"] = held_t
    if case["kind"] == "evict":
        st["after"] = held_t + case["n"]
        st["pos"] = 4 * held_t
    return st


# ---------------------------------------------------------------- plain forms --


def _rows_of(pool, scale, table, n):
    """[B, HK, n, D] of the first n slots of every sequence, 32 bits."""
    page = pool.shape[2]
    pages = table[:, :-(-n // page)].clamp(min=0).long()
    x = pool[pages].permute(0, 2, 1, 3, 4).reshape(pages.shape[0], pool.shape[1], -1, pool.shape[3])[:, :, :n].float()
    if scale is not None:
        x = x * scale[pages].permute(0, 2, 1, 3).reshape(x.shape[0], x.shape[1], -1)[:, :, :n, None]
    return x


def _places(table, slots, page):
    """(page, row) of slots [B, ...] of the sequences."""
    B = table.shape[0]
    pg = torch.gather(table, 1, (slots // page).view(B, -1).long()).view(slots.shape).long()
    return pg, (slots % page).long()


def _plain_attend(st):
    c = st["case"]
    B, S, H, HK, n = c["B"], c["S"], c["H"], c["HK"], st["width"]
    g = H // HK
    K = _rows_of(st["k"], st["ks"], st["table"], n)
    V = K if c["shared"] else _rows_of(st["v"], st["vs"], st["table"], n)
    q = st["q"].float().view(B, S, HK, g, -1).permute(0, 2, 1, 3, 4).reshape(B, HK, S * g, -1)
    s = torch.matmul(q, K.transpose(-1, -2).contiguous()) * st["scale"]
    limit = st["lens"][:, None] - (S - 1) + torch.arange(S, device=s.device)
    limit = limit[:, None, :, None, None].expand(B, 1, S, g, 1).reshape(B, 1, S * g, 1)
    s = torch.where(torch.arange(n, device=s.device) < limit, s, -math.inf)
    m = s.amax(-1, keepdim=True)
    if c["sink"]:
        sink = st["sink"].view(1, HK, 1, g, 1).expand(B, HK, S, g, 1).reshape(B, HK, S * g, 1)
        m = torch.maximum(m, sink)
    m = torch.where(m == -math.inf, 0.0, m)
    e = torch.exp(s - m)
    l = e.sum(-1, keepdim=True)
    if c["sink"]:
        l = l + torch.exp(sink - m)
    p = e / torch.where(l == 0, 1.0, l)
    o = torch.matmul(p, V).view(B, HK, S, g, -1).permute(0, 2, 1, 3, 4).reshape(B, S, H, -1).to(torch.bfloat16)
    if not c["track"]:
        return {"o": o}
    slots = torch.arange(n, device=s.device, dtype=torch.int32)[None, :].expand(B, n)
    pg, r = _places(st["table"], slots, c["page"])
    heads = torch.arange(HK, device=s.device)[None, :, None]
    at = (pg[:, None, :], heads, r[:, None, :])
    st["w"][at] = st["w"][at] + p.sum(2)
    return {"o": o, "weights": st["w"]}


def _plain_put(pool, scale, at, x):
    """Rows x [B, T, HK, D] at their places, in 8 bits with a scale for each row where the pool has one."""
    pg, r = at
    heads = torch.arange(x.shape[2], device=x.device)
    if scale is None:
        pool[pg[..., None], heads, r[..., None]] = x
        return
    x = x.float()
    s = x.abs().amax(-1).clamp(min=1e-4) * (1.0 / 448.0)
    code = (x / s[..., None]).clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
    pool.view(torch.uint8)[pg[..., None], heads, r[..., None]] = code.view(torch.uint8)
    scale[pg[..., None], heads, r[..., None]] = s


def _plain_write(st, position=None):
    c = st["case"]
    T = st["new_k"].shape[1]
    step = torch.arange(T, device="cuda", dtype=torch.int32)
    slots = st["start"][:, None] + step
    at = _places(st["table"], slots, c["page"])
    _plain_put(st["k"], st["ks"], at, st["new_k"])
    if not c["shared"]:
        _plain_put(st["v"], st["vs"], at, st["new_v"])
    if c["track"]:
        heads = torch.arange(c["HK"], device="cuda")
        st["w"][at[0][..., None], heads, at[1][..., None]] = 0.0
        first = st["start"] if position is None else position
        st["p"][at[0][..., None], heads, at[1][..., None]] = (first[:, None] + step)[..., None].expand(-1, -1, c["HK"])


def _plain_evict(st):
    c = st["case"]
    B, HK, page, keep, n = c["B"], c["HK"], c["page"], c["keep"], st["width"]
    first, recent = _first_recent(c)
    if n <= keep:
        return st["after"].clamp(max=keep)
    slots = torch.arange(n, device="cuda", dtype=torch.int32)
    pg, r = _places(st["table"], slots[None, :].expand(B, n), page)
    heads = torch.arange(HK, device="cuda")[None, :, None]
    w, p = st["w"][pg[:, None], heads, r[:, None]], st["p"][pg[:, None], heads, r[:, None]]
    held = (slots < st["after"][:, None])[:, None, :].expand(B, HK, n)
    last = torch.where(held, p, -1).amax(-1, keepdim=True)
    safe = (p < first) | (p >= last + 1 - recent)
    key = torch.where(held, torch.where(safe, math.inf, w), -math.inf)
    rank = torch.empty(B, HK, n, dtype=torch.int64, device="cuda")
    rank.scatter_(2, torch.sort(key, dim=-1, descending=True, stable=True).indices,
                  torch.arange(n, device="cuda").expand(B, HK, n))
    kept = (rank < keep) & held
    hole, mover = held & ~kept & (slots < keep), kept & (slots >= keep)
    moves = min(keep, n - keep)
    to = torch.sort((~hole).to(torch.int8), dim=-1, stable=True).indices[..., :moves]
    fro = torch.sort((~mover).to(torch.int8), dim=-1, stable=True).indices[..., :moves]
    # past a head's last pair a slot is put back onto itself
    fro = torch.where(torch.arange(moves, device="cuda") < hole.sum(-1, keepdim=True), fro, to)
    to_pg, to_r = _places(st["table"], to, page)
    fro_pg, fro_r = _places(st["table"], fro, page)
    pools = [st["k"], st["ks"], st["w"], st["p"]] + ([] if c["shared"] else [st["v"], st["vs"]])
    for x in pools:
        if x is not None:
            x = x.view(torch.uint8) if x.dtype == torch.float8_e4m3fn else x
            x[to_pg, heads, to_r] = x[fro_pg, heads, fro_r]
    return st["after"].clamp(max=keep)


# ---------------------------------------------------------------- passes ------


def _cache(st):
    """The handle on the pools that a program keeps."""
    if "cache" not in st:
        from wanferenz_amd.paged import PagedKV

        st["cache"] = PagedKV(st["k"], None if st["case"]["shared"] else st["v"], k_scale=st["ks"],
                              v_scale=None if st["case"]["shared"] else st["vs"], weights=st["w"], positions=st["p"])
    return st["cache"]


def _state_of(st):
    names = ["k", "ks", "w", "p"] + ([] if st["case"]["shared"] else ["v", "vs"])
    return {x: st[x] for x in names if st[x] is not None}


def run(st):
    c = st["case"]
    if c["kind"] == "attend":
        if not own:
            return _plain_attend(st)
        o = _cache(st).attend(st["q"], st["table"], st["lens"], st["scale"], attn_sink=st["sink"],
                              accumulate=c["track"])
        return {"o": o, "weights": st["w"]} if c["track"] else {"o": o}
    if c["kind"] == "write":
        if own:
            _cache(st).write(st["new_k"], st["new_v"], st["table"], st["start"])
        else:
            _plain_write(st)
        return _state_of(st)
    if own:
        _cache(st).write(st["new_k"], st["new_v"], st["table"], st["start"], position=st["pos"])
        first, recent = _first_recent(c)
        lens = _cache(st).evict(st["table"], st["after"], c["keep"], first=first, recent=recent)
    else:
        _plain_write(st, st["pos"])
        lens = _plain_evict(st)
    if c["n"] < c["keep"]:
        st["pos"] += c["n"]  # the loop goes on: a prompt begins again
    return {"lens": lens, **_state_of(st)}


def work(case):
    B, S, H, HK, D = (case[k] for k in ("B", "S", "H", "HK", "D"))
    lens = _lengths(case)
    sides = 1 if case["shared"] else 2
    row = sides * (D + 4 if case["e4m3"] else 2 * D)  # of one slot and head
    pages = sum(-(-n // case["page"]) for n in lens)
    if case["kind"] == "attend":
        flops = sum(4 * H * D * max(0, n - S + 1 + i) for n in lens for i in range(S))
        nbytes = sum(lens) * HK * (row + (8 if case["track"] else 0)) + 4 * B * S * H * D + 4 * (pages + B)
        return {"bytes": nbytes, "flops": flops}
    new = S if case["kind"] == "write" else case["n"]
    nbytes = B * new * HK * (sides * 2 * D + row + (8 if case["track"] else 0)) + 4 * B
    flops = B * new * HK * D * sides * (3 if case["e4m3"] else 0)
    if case["kind"] == "evict":
        keep = case["keep"]
        first, recent = _first_recent(case)
        for n in (n + new for n in lens):
            if n <= keep:
                continue
            late = min(recent, n - keep)  # kept slots past the budget: the newest, and their share of the rest
            moves = late + (keep - first - recent) * (n - keep - late) / max(1, n - first - recent)
            nbytes += HK * (8 * n + 2 * (row + 8) * min(moves, keep, n - keep))
            flops += HK * n
    return {"bytes": float(nbytes), "flops": float(flops)}


# ---------------------------------------------------------------- 64 bits -----


def _exact_rows(pool, scale, pages, n):
    x = pool[pages.long()].double()  # [np, HK, page, D]
    if scale is not None:
        x = x * scale[pages.long()].double().unsqueeze(-1)
    return x.transpose(0, 1).reshape(pool.shape[1], -1, pool.shape[3])[:, :n]


def _exact_attend(st):
    c = st["case"]
    B, S, H, HK, D, page = (c[k] for k in ("B", "S", "H", "HK", "D", "page"))
    o = torch.zeros(B, S, H, D, dtype=torch.float64, device="cuda")
    w = st["w"].double() if c["track"] else None
    for b, n in enumerate(_lengths(c)):
        if n == 0:
            continue
        pages = st["table"][b, :-(-n // page)]
        K = _exact_rows(st["k"], st["ks"], pages, n)
        V = _exact_rows(st["v"], st["vs"], pages, n)
        for i in range(S):
            seen = n - (S - 1 - i)
            if seen <= 0:
                continue
            q = st["q"][b, i].double().view(HK, H // HK, D)
            s = torch.bmm(K[:, :seen].contiguous(), q.transpose(1, 2).contiguous()).transpose(1, 2) * st["scale"]
            if c["sink"]:
                s = torch.cat([s, st["sink"].double().view(HK, H // HK, 1)], dim=2)
            p = torch.softmax(s, dim=2)[..., :seen].contiguous()
            o[b, i] = torch.bmm(p, V[:, :seen].contiguous()).reshape(H, D)
            if c["track"]:
                add = torch.zeros(HK, pages.numel() * page, dtype=torch.float64, device="cuda")
                add[:, :seen] = p.sum(1)
                w[pages.long()] += add.view(HK, pages.numel(), page).transpose(0, 1)
    return {"o": o, "weights": w} if c["track"] else {"o": o}


def _exact_write(st):
    c = st["case"]
    page, T = c["page"], st["new_k"].shape[1]
    sides = (("k", "ks", "new_k"),) + (() if c["shared"] else (("v", "vs", "new_v"),))
    out = {}
    for name, scale, rows in sides:
        out[name] = st[name].double()
        if c["e4m3"]:
            out[scale] = st[scale].double()
    if c["track"]:
        out["w"], out["p"] = st["w"].double(), st["p"].clone()
    for b, start in enumerate(_lengths(c)):
        pos = int(st["pos"][b]) if c["kind"] == "evict" else start
        for p in range(start // page, (start + T - 1) // page + 1):
            lo, hi = max(start, p * page), min(start + T, (p + 1) * page)
            pg, a = int(st["table"][b, p]), lo - p * page
            for name, scale, rows in sides:
                x = st[rows][b, lo - start:hi - start].double().transpose(0, 1)
                if c["e4m3"]:
                    s = x.abs().amax(-1).clamp(min=1e-4) / 448.0
                    out[scale][pg, :, a:a + hi - lo] = s
                    x = (x / s[..., None]).float().to(torch.float8_e4m3fn).double()
                out[name][pg, :, a:a + hi - lo] = x
            if c["track"]:
                out["w"][pg, :, a:a + hi - lo] = 0.0
                out["p"][pg, :, a:a + hi - lo] = torch.arange(pos + lo - start, pos + hi - start, device="cuda")
    return out


def _exact_evict(st):
    c = st["case"]
    keep, page = c["keep"], c["page"]
    first, recent = _first_recent(c)
    out = _exact_write(st)
    lens = []
    for b, start in enumerate(_lengths(c)):
        n = start + c["n"]
        lens.append(min(n, keep))
        if n <= keep:
            continue
        pages = st["table"][b, :-(-n // page)].long()
        for h in range(c["HK"]):
            pg, r = pages.repeat_interleave(page)[:n], torch.arange(page, device="cuda").repeat(pages.numel())[:n]
            w, p = out["w"][pg, h, r].cpu(), out["p"][pg, h, r].cpu().long()
            safe = (p < first) | (p > int(p.max()) - recent)
            order = torch.sort(torch.where(safe, torch.tensor(math.inf, dtype=torch.float64), w), descending=True,
                               stable=True).indices
            kept = torch.zeros(n, dtype=torch.bool)
            kept[order[:keep]] = True
            to = torch.nonzero(~kept[:keep])[:, 0].cuda()
            fro = torch.nonzero(kept[keep:])[:, 0].cuda() + keep
            for x in out.values():
                x[pg[to], h, r[to]] = x[pg[fro], h, r[fro]]
    return {"lens": torch.tensor(lens, dtype=torch.int32, device="cuda"), **out}


def exact(case, seed):
    if case["kind"] == "write" and case["S"] * case["B"] * case["HK"] * case["D"] > 1 << 28:
        return None
    st = prepare(case, seed)
    return {"attend": _exact_attend, "write": _exact_write, "evict": _exact_evict}[case["kind"]](st)
