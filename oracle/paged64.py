"""The paged cache's operators and beam search's selection, restated sequence by sequence in float64 / integers. TEST
INFRASTRUCTURE ONLY (see oracle/__init__.py). Nothing in wasiqnauman/cudallm corresponds to them: the definitions
are those of include/cudallm.h."""
from __future__ import annotations

import numpy as np


def attend64(q, k, v, table, lens, scale=None, window=0):
    """q [B][H][D], k and v [pages][KV][page][D] as float64, table [B][P] -> (out, lse, abs_scores): abs_scores[b][h] is the
    largest scale * sum_d |q_d k_td|, what the scores' rounding errors are proportional to."""
    B, H, D = q.shape
    pages, KV, page, _ = k.shape
    scale = D ** -0.5 if scale is None else scale
    out, lse, size = np.zeros((B, H, D)), np.full((B, H), -np.inf), np.zeros((B, H))
    for b in range(B):
        n = min(max(int(lens[b]), 0), table.shape[1] * page)
        slots = [(int(table[b][t // page]), t % page) for t in range(max(0, n - window) if window else 0, n)
                 if 0 <= table[b][t // page] < pages]
        if not slots:
            continue
        p, s = (np.array(x) for x in zip(*slots))
        for h in range(H):
            kk, vv = k[p, h // (H // KV), s], v[p, h // (H // KV), s]
            x = scale * (kk @ q[b, h])
            m = x.max()
            e = np.exp(x - m)
            out[b, h], lse[b, h] = e @ vv / e.sum(), m + np.log(e.sum())
            size[b, h] = np.max(abs(scale) * (np.abs(kk) @ np.abs(q[b, h])))
    return out, lse, size


def rotate64(x, positions, inv_freq, interleaved, factor):
    """x [tokens][heads][D] float64, rotated; the angle is formed in fp32 as the kernels do."""
    y, n = np.array(x), len(inv_freq)
    ang = (positions.astype(np.float32)[:, None] * inv_freq.astype(np.float32)).astype(np.float64)[:, None]
    c, s = factor * np.cos(ang), factor * np.sin(ang)
    i, j = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if interleaved else (slice(0, n), slice(n, 2 * n))
    y[..., i], y[..., j] = x[..., i] * c - x[..., j] * s, x[..., j] * c + x[..., i] * s
    return y


def fork_ref(tables, lens, refs, parents, page, room):
    """-> (tables, lens, refs, missing, copies [(source page, new page, tokens)])."""
    R, P = tables.shape
    N = len(refs)
    is_page = lambda e: 0 <= e < N  # noqa: E731
    out, new_refs, free = np.full((len(parents), P), -1, np.int64), refs.astype(np.int64).copy(), [i for i in range(N) if refs[i] == 0]
    new_lens, missing, copies, kept = np.zeros(len(parents), np.int64), 0, [], {}
    length = [min(max(int(n), 0), P * page) for n in lens]
    held = []
    for r in range(R):
        full = length[r] // page
        end = full
        while end < P and is_page(tables[r][end]):
            end += 1
        held.append(end)
        for e in tables[r][:end]:
            if is_page(e):
                new_refs[e] -= 1
    for i, p in enumerate(parents):
        if not 0 <= p < R:
            continue
        n = length[p]
        full, tail = divmod(n, page)
        first_alone = held[p] > full and refs[tables[p][full]] == 1 and p not in kept
        kept[p] = True
        have = held[p] if first_alone else full
        row = [int(e) if is_page(e) else -1 for e in tables[p][:have]]
        want = -(-(n + room) // page)
        missing += max(0, want - P)
        for j in range(have, min(want, P)):
            if free:
                e = free.pop(0)
                if j == full and tail and held[p] > full and not first_alone:
                    copies.append((int(tables[p][full]), e, tail))
                row.append(e)
            else:
                row.append(-1)
                missing += 1
        for e in row:
            if e >= 0:
                new_refs[e] += 1
        out[i, :len(row)] = row
        new_lens[i] = n
    return out, new_lens, new_refs, missing, copies


def compact_ref(tables, refs):
    """-> (tables, refs, live, moves [(from, to)])."""
    N = len(refs)
    used = [i for i in range(N) if refs[i] > 0]
    holes = [i for i in range(len(used)) if refs[i] <= 0]
    moves = list(zip([i for i in used if i >= len(used)], holes))
    to = dict(moves)
    new_refs = np.zeros(N, np.int64)
    for i in used:
        new_refs[to.get(i, i)] = refs[i]
    out = np.array([[to.get(int(e), int(e)) if 0 <= e < N else -1 for e in row] for row in tables], np.int64).reshape(tables.shape)
    return out, new_refs, len(used), moves


def beam_ref(logits, scores, keep, finished=None, eos=0):
    """logits [G * W][V], scores [G][W], float64 -> (scores, parents, tokens); candidates are kept in float64."""
    G, W = scores.shape
    V = logits.shape[1]
    out = []
    for g in range(G):
        found = []
        for w in range(W):
            x = logits[g * W + w].astype(np.float64)
            if finished is not None and finished[g][w]:
                x = np.where(np.arange(V) == eos, 0.0, -np.inf)
            key = np.where(np.isnan(x), -np.inf, x)
            with np.errstate(all="ignore"):
                m = np.nan if np.isnan(x).any() else x.max()
                cand = scores[g][w] + (x - (m + np.log(np.exp(x - m).sum())))
            for rank, t in enumerate(np.lexsort((np.arange(V), -key))[:keep]):
                found.append((-np.inf if np.isnan(cand[t]) else cand[t], w, rank, int(t)))
        found.sort(key=lambda f: (-f[0], f[1], f[2]))
        out.append(found[:keep])
    return (np.array([[f[0] for f in g] for g in out]), np.array([[i * W + f[1] for f in g] for i, g in enumerate(out)]),
            np.array([[f[3] for f in g] for g in out]))
