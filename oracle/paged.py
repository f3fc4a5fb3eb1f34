"""Plain statements of the paged cache's operators, in 64 bits on the CPU (numpy).

A cache is a dict of arrays: k, v [P, HK, page, D] float64 values (v missing: K = V), and
weights, positions [P, HK, page] where it is tracked.  Nothing here follows the kernels'
order of work.
"""

from __future__ import annotations

import numpy as np


def slot_places(table_row, pages, page, slots):
    """(page id, row) of slots; page id -1 where the table has none."""
    out = []
    for t in slots:
        p = t // page
        pid = int(table_row[p]) if 0 <= t and p < len(table_row) else -1
        out.append((pid if 0 <= pid < pages else -1, t % page))
    return out


def attend(cache, q, table, lens, scale, sink=None):
    """-> (o [B, S, H, D], abs [B, S, H, D] = sum_j p_j |v_j|, add [P, HK, page] the weight each
    slot gets, reach = the largest sum_d |q_d k_d| scale of a visible slot)."""
    k, v = cache["k"], cache.get("v", cache["k"])
    P, HK, page, D = k.shape
    B, S, H, _ = q.shape
    g = H // HK
    o, mag = np.zeros((B, S, H, D)), np.zeros((B, S, H, D))
    add = np.zeros((P, HK, page))
    reach = 0.0
    for b in range(B):
        n = int(min(max(int(lens[b]), 0), table.shape[1] * page))
        at = slot_places(table[b], P, page, range(n))
        for i in range(S):
            seen = [x for x in at[:max(0, n - (S - 1 - i))] if x[0] >= 0]
            if not seen:
                continue
            pid, row = np.array([x[0] for x in seen]), np.array([x[1] for x in seen])
            for h in range(H):
                hk = h // g
                kk, vv = k[pid, hk, row], v[pid, hk, row]
                with np.errstate(all="ignore"):
                    s = (kk @ q[b, i, h]) * scale
                    reach = max(reach, float(np.nanmax(np.abs(kk) @ np.abs(q[b, i, h]) * scale)))
                    m = max(float(s.max()), -np.inf if sink is None else float(sink[h]))
                    if m == -np.inf:
                        continue
                    e = np.exp(s - m)
                    p = e / (e.sum() + (0.0 if sink is None else np.exp(float(sink[h]) - m)))
                    o[b, i, h] = p @ vv
                    mag[b, i, h] = p @ np.abs(vv)
                np.add.at(add, (pid, hk, row), p)
    return o, mag, add, reach


def evict_pairs(weights, positions, n, keep, first, recent, present=None):
    """One head's (holes, movers) among its n slots: lists of slots, paired in order.  Slots that are not
    present are neither kept nor filled, so as many stay as are present below keep."""
    if n <= keep:
        return [], []
    slots = [t for t in range(n) if present is None or present[t]]
    last = max((int(positions[t]) for t in slots), default=0)

    def key(t):
        if positions[t] < first or positions[t] > last - recent:
            return (2, 0.0)
        w = float(weights[t])
        return (0, 0.0) if np.isnan(w) else (1, w)

    order = sorted(slots, key=lambda t: (-key(t)[0], -key(t)[1], t))
    kept = set(order[:sum(t < keep for t in slots)])
    return [t for t in slots if t < keep and t not in kept], [t for t in slots if t >= keep and t in kept]


def evict(cache, table, lens, keep, first=0, recent=0):
    """In place over every array of the cache; -> new lengths."""
    P, HK, page = cache["weights"].shape
    out = []
    for b in range(table.shape[0]):
        n = int(min(max(int(lens[b]), 0), table.shape[1] * page))
        out.append(min(int(lens[b]), keep))
        at = slot_places(table[b], P, page, range(n))
        present = [x[0] >= 0 for x in at]
        for h in range(HK):
            w = [cache["weights"][p, h, r] if p >= 0 else 0.0 for p, r in at]
            pos = [cache["positions"][p, h, r] if p >= 0 else 0 for p, r in at]
            holes, movers = evict_pairs(w, pos, n, keep, first, recent, present)
            assert len(holes) == len(movers)
            moved = [(at[a], at[c]) for a, c in zip(holes, movers)]
            for x in cache.values():
                for (tp, tr), (fp, fr) in moved:
                    x[tp, h, tr] = x[fp, h, fr]
    return np.array(out, dtype=np.int32)


def tree_sight(parent, nodes):
    """Row i: the set of nodes that node i of a tree sees, itself and those above it."""
    out = []
    for i in range(nodes):
        seen, at = set(), i
        while 0 <= at < nodes and at not in seen:
            seen.add(at)
            at = int(parent[at])
        out.append(seen)
    return out


def attend_tree(cache, q, table, lens, parent, scale, sink=None, count=None):
    """attend for trees of drafted tokens -> (o, abs, None, reach), as attend's."""
    k, v = cache["k"], cache.get("v", cache["k"])
    P, HK, page, D = k.shape
    B, S, H, _ = q.shape
    o, mag, reach = np.zeros((B, S, H, D)), np.zeros((B, S, H, D)), 0.0
    for b in range(B):
        n = int(min(max(int(lens[b]), 0), table.shape[1] * page))
        nodes = S if count is None else min(max(int(count[b]), 0), S)
        at = slot_places(table[b], P, page, range(n))
        for i, sight in enumerate(tree_sight(parent[b], nodes)):
            seen = [x for t, x in enumerate(at) if x[0] >= 0 and (t < n - nodes or t - (n - nodes) in sight)]
            if not seen:
                continue
            pid, row = np.array([x[0] for x in seen]), np.array([x[1] for x in seen])
            for h in range(H):
                kk, vv = k[pid, h // (H // HK), row], v[pid, h // (H // HK), row]
                with np.errstate(all="ignore"):
                    s = (kk @ q[b, i, h]) * scale
                    reach = max(reach, float(np.nanmax(np.abs(kk) @ np.abs(q[b, i, h]) * scale)))
                    m = max(float(s.max()), -np.inf if sink is None else float(sink[h]))
                    if m == -np.inf:
                        continue
                    e = np.exp(s - m)
                    p = e / (e.sum() + (0.0 if sink is None else np.exp(float(sink[h]) - m)))
                    o[b, i, h], mag[b, i, h] = p @ vv, p @ np.abs(vv)
    return o, mag, None, reach


def turned(x, norm, eps, turns, halves, leading):
    """Rows x [.., D] float64, normed by `norm` (None: as they are) and rotated by `turns` [.., R / 2] complex."""
    x = np.array(x, dtype=np.float64)
    if norm is not None:
        x = x / np.sqrt(np.mean(x * x, axis=-1, keepdims=True) + eps) * norm
    R, D = 2 * turns.shape[-1], x.shape[-1]
    lo = 0 if leading else D - R
    pair = np.arange(R // 2)
    i = lo + (pair if halves else 2 * pair)
    j = i + (R // 2 if halves else 1)
    z = (x[..., i] + 1j * x[..., j]) * turns
    x[..., i], x[..., j] = z.real, z.imag
    return x


def accept(drafted, parent, sampled, nodes):
    """One tree's accepted nodes, in order."""
    path = [0] if nodes > 0 else []
    while path:
        on = [c for c in range(path[-1] + 1, nodes)
              if parent[c] == path[-1] and drafted[c] == sampled[path[-1]]]
        if not on:
            break
        path.append(on[0])
    return path
