"""The operators of beam-search decoding over a paged key-value cache, as cases to measure.

  attention  one new token of each sequence attends to that sequence's pages
  rope       new tokens' queries are rotated, their keys rotated and stored with their values in pages
  fork       the sequences of the next step take over, share and copy the pages of their parents
  compact    the pages in use are moved to the front of the pool
  beam       the best continuations of each group of beams over beams and vocabulary

With `own` false, `run` computes an operator in elementary torch operations; with `own` true it calls
cudallm_b200.paged. `exact` states the same definitions once more in 64 bits, sequence by sequence.

Definitions.
  Pages: k, v [layers][pages][kv heads][page size][dim]; row r of a table lists the pages of sequence r's
  tokens 0, 1, ...; an entry outside [0, pages) holds no page and its tokens are masked.
  attention: softmax(scale q.k) v over positions max(0, len - window) <= t < len (window 0: all), fp32;
  lse is the natural logarithm of the sum; no position left: out 0, lse -inf.
  rope: angle of pair i = float32(position) * inv_freq[i] rounded to fp32; cos and sin times `factor`; pairs
  (i, i + n) or (2i, 2i + 1) of the first 2n dims.
  fork: see plain_fork. beam: see plain_beam.
"""
import math

import numpy as np
import torch

own = False

ENGINE = {"heads": 32, "kv_heads": 8, "dim": 64}  # the framework's model
TORCH = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}


def listed():
    return [
        # A single short conversation of the engine (fp32 activations, fp16 cache): latency alone.
        {"name": "attention one short", "op": "attention", "seqs": 1, **ENGINE, "page": 16, "shortest": 33, "longest": 33,
         "window": 0, "empty": 0, "q": "float32", "kv": "float16", "order": "heads"},
        # The batched engine's benchmark: 64 sequences of 512 to 767 cached tokens.
        {"name": "attention batch", "op": "attention", "seqs": 64, **ENGINE, "page": 16, "shortest": 512, "longest": 767,
         "window": 0, "empty": 0, "q": "float32", "kv": "bfloat16", "order": "heads"},
        # One sequence of the long-context configuration: the length has to be split.
        {"name": "attention one long", "op": "attention", "seqs": 1, **ENGINE, "page": 64, "shortest": 32768, "longest": 32768,
         "window": 0, "empty": 0, "q": "bfloat16", "kv": "bfloat16", "order": "heads"},
        # A ragged batch with empty rows, eight queries a key head, wider heads, token-major pages of an odd size.
        {"name": "attention ragged", "op": "attention", "seqs": 37, "heads": 32, "kv_heads": 4, "dim": 128, "page": 24, "shortest": 1,
         "longest": 8111, "window": 0, "empty": 3, "q": "bfloat16", "kv": "bfloat16", "order": "tokens"},
        # One decode step of four beams: latency alone.
        {"name": "rope four beams", "op": "rope", "seqs": 4, "each": 1, **ENGINE, "rotary": 64, "interleaved": False, "scaling": "llama3",
         "start": 700, "x": "float32", "kv": "float16", "page": 16, "order": "heads"},
        # A long prompt's chunk, interleaved pairs in part of the head, positions past the trained range.
        {"name": "rope prompt", "op": "rope", "seqs": 3, "each": 5461, "heads": 32, "kv_heads": 8, "dim": 128, "rotary": 64, "interleaved": True,
         "scaling": "yarn", "start": 30011, "x": "bfloat16", "kv": "bfloat16", "page": 64, "order": "heads"},
        # Four beams after one step: two tails to copy, over all the engine's layers.
        {"name": "fork four beams", "op": "fork", "groups": 1, "beams": 4, "layers": 16, "kv_heads": 8, "dim": 64, "page": 16, "shortest": 155,
         "longest": 155, "prompt": 0.5, "room": 1, "kv": "float16", "order": "heads"},
        # Sixteen groups of eight beams with long pages: bandwidth counts.
        {"name": "fork many beams", "op": "fork", "groups": 16, "beams": 8, "layers": 16, "kv_heads": 8, "dim": 64, "page": 64, "shortest": 301,
         "longest": 2045, "prompt": 0.7, "room": 1, "kv": "bfloat16", "order": "heads"},
        # A small pool, a third in use.
        {"name": "compact small", "op": "compact", "pages": 192, "live": 61, "seqs": 7, "layers": 2, "kv_heads": 8, "dim": 64, "page": 16,
         "kv": "float16", "order": "heads"},
        # A large pool, half in use, before its upper half is given back.
        {"name": "compact large", "op": "compact", "pages": 3001, "live": 1500, "seqs": 64, "layers": 16, "kv_heads": 8, "dim": 64, "page": 16,
         "kv": "bfloat16", "order": "heads"},
        # Four beams over the engine's vocabulary.
        {"name": "beam four", "op": "beam", "groups": 1, "beams": 4, "keep": 4, "vocab": 128256, "finished": 0, "x": "float32"},
        # The batch of 64 rows, two candidates a beam kept, a few beams finished.
        {"name": "beam batch", "op": "beam", "groups": 8, "beams": 8, "keep": 16, "vocab": 128256, "finished": 5, "x": "bfloat16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case: sizes by their logarithm over the listed ranges."""
    op = rng.choice(["attention", "attention", "rope", "fork", "compact", "beam"])
    kv = rng.choice(["float16", "bfloat16"])
    x = rng.choice(["float32", kv])
    order = rng.choice(["heads", "heads", "tokens"])
    if op == "attention":
        kv_heads, dim = rng.choice([(8, 64), (8, 64), (4, 128), (2, 128), (8, 80), (1, 256)])
        group = rng.choice([1, 3, 4, 4, 7, 8, 16])
        longest = _log(rng, 1, 32768)
        seqs = max(1, min(_log(rng, 1, 128), 134_000_000 // (longest * kv_heads * dim)))
        return {"op": op, "seqs": seqs, "heads": kv_heads * group, "kv_heads": kv_heads, "dim": dim, "page": rng.choice([1, 8, 16, 16, 24, 64, 100, 128]),
                "shortest": max(1, int(longest * rng.random())), "longest": longest, "window": rng.choice([0, 0, 0, _log(rng, 1, 4096)]),
                "empty": rng.choice([0, 0, min(3, seqs - 1)]), "q": x, "kv": kv, "order": order}
    if op == "rope":
        dim = rng.choice([64, 64, 128, 80, 256])
        rotary = rng.choice([dim, dim, dim // 2, 16])
        kv_heads = rng.choice([1, 2, 8])
        heads = kv_heads * rng.choice([1, 4, 7])
        each = rng.choice([1, 1, _log(rng, 2, 8192)])
        seqs = max(1, min(_log(rng, 1, 128), 60_000_000 // (each * (heads + 2 * kv_heads) * dim)))
        return {"op": op, "seqs": seqs, "each": each, "heads": heads, "kv_heads": kv_heads, "dim": dim, "rotary": rotary, "interleaved": rng.random() < 0.5,
                "scaling": rng.choice(["none", "linear", "llama3", "yarn"]), "start": _log(rng, 1, 100000) - 1, "x": x, "kv": kv,
                "page": rng.choice([1, 16, 24, 64]), "order": order}
    if op == "fork":
        beams, page = rng.choice([2, 3, 4, 8, 16]), rng.choice([8, 16, 24, 64])
        groups, longest = max(1, _log(rng, 1, 128) // beams), _log(rng, 2, 2048)
        return {"op": op, "groups": groups, "beams": beams, "layers": rng.choice([1, 5, 16]), "kv_heads": rng.choice([2, 8]), "dim": 64, "page": page,
                "shortest": max(1, int(longest * rng.random())), "longest": longest, "prompt": round(0.5 + 0.5 * rng.random(), 3), "room": rng.choice([0, 1, 5, 40]),
                "kv": kv, "order": order}
    if op == "compact":
        pages = _log(rng, 16, 3001)
        return {"op": op, "pages": pages, "live": max(1, int(pages * (0.1 + 0.8 * rng.random()))), "seqs": _log(rng, 1, 64), "layers": rng.choice([1, 5, 16]),
                "kv_heads": rng.choice([2, 8]), "dim": 64, "page": 16, "kv": kv, "order": order}
    groups, beams = _log(rng, 1, 16), rng.choice([1, 2, 4, 5, 8])
    return {"op": op, "groups": groups, "beams": beams, "keep": rng.choice([1, beams, 2 * beams]), "vocab": _log(rng, 1000, 128256),
            "finished": rng.randrange(0, beams), "x": rng.choice(["float32", "float16", "bfloat16"])}


# ---- inputs -----------------------------------------------------------------------------------

def _lens(c, rng):
    """The sequences' lengths: evenly from the shortest to the longest, the `empty` shortest of them 0; `rng` orders them."""
    n = np.linspace(c["longest"], c["shortest"], c["seqs"]).round().astype(np.int64)
    if c["empty"]:
        n[-c["empty"]:] = 0
    return rng.permutation(n) if rng is not None else n


def _pool(c, layers, pages, gen):
    """k and v [layers][pages][kv heads][page][dim], whose memory is head by head or token by token within a page."""
    shape = (layers, pages, c["kv_heads"], c["page"], c["dim"])
    if c["order"] == "tokens":
        shape = (layers, pages, c["page"], c["kv_heads"], c["dim"])
    pool = [torch.randn(shape, generator=gen, device="cuda", dtype=TORCH[c["kv"]]) for _ in range(2)]
    return [p.transpose(2, 3) for p in pool] if c["order"] == "tokens" else pool


def _tables(counts, width, pages, rng):
    """Rows of `counts` pages each, all different, anywhere in the pool; -1 after a row's last."""
    ids = rng.permutation(pages)
    t = np.full((len(counts), width), -1, np.int32)
    at = 0
    for r, n in enumerate(counts):
        t[r, :n] = ids[at:at + n]
        at += n
    return t


def _inv_freq(c):
    """Inverse frequencies (base 500000), as they come or scaled for contexts `s` times as long; and the factor of cos and sin."""
    d, base, s = c["rotary"], 500000.0, 32.0
    f = base ** (-np.arange(0, d, 2, dtype=np.float64) / d)
    if c["scaling"] == "linear":
        return f / s, 1.0
    if c["scaling"] == "llama3":
        turns = 8192.0 * f / (2 * math.pi)
        ramp = np.clip((turns - 1.0) / (4.0 - 1.0), 0.0, 1.0)
        return f * (ramp + (1 - ramp) / s), 1.0
    if c["scaling"] == "yarn":
        turns = 8192.0 * f / (2 * math.pi)
        ramp = np.clip((turns - 1.0) / (32.0 - 1.0), 0.0, 1.0)
        return f * (ramp + (1 - ramp) / s), 0.1 * math.log(s) + 1.0
    return f, 1.0


def _fork_rows(c):
    """Per row of the tables: its length, and how many of its first pages the group's beams share."""
    lens = np.linspace(c["longest"], c["shortest"], c["groups"]).round().astype(np.int64).repeat(c["beams"])
    return lens, (lens * c["prompt"]).astype(np.int64) // c["page"]


def prepare(case, seed):
    c, rng = case, np.random.default_rng(seed)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": c}
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    if c["op"] == "attention":
        lens = _lens(c, rng)
        counts = -(-lens // c["page"])
        pages = int(counts.sum()) + 3
        s["k"], s["v"] = _pool(c, 1, pages, gen)
        s["tables"] = dev(_tables(counts, int(counts.max()), pages, rng))
        s["lens"] = dev(lens.astype(np.int32))
        s["q"] = torch.randn((c["seqs"], c["heads"], c["dim"]), generator=gen, device="cuda").to(TORCH[c["q"]])
    elif c["op"] == "rope":
        n, each, dim = c["seqs"] * c["each"], c["each"], c["dim"]
        starts = c["start"] + rng.integers(0, 16, c["seqs"])
        ends = starts + each
        first = starts // c["page"]  # earlier pages are not written: they are left out of this pool
        counts = -(-ends // c["page"]) - first
        width = -(-(c["start"] + 15 + each) // c["page"])
        pages = c["seqs"] * (width - c["start"] // c["page"]) + 3
        s["k"], s["v"] = _pool(c, 1, pages, gen)
        t = np.full((c["seqs"], width), -1, np.int32)
        short = _tables(counts, int(counts.max()), pages, rng)
        for r in range(c["seqs"]):
            t[r, first[r]:first[r] + counts[r]] = short[r, :counts[r]]
        s["tables"] = dev(t)
        s["positions"] = dev((starts[:, None] + np.arange(each)).reshape(-1).astype(np.int32))
        s["rows"] = dev(np.arange(c["seqs"], dtype=np.int32).repeat(each))
        qkv = torch.randn((n, c["heads"] + 2 * c["kv_heads"], dim), generator=gen, device="cuda").to(TORCH[c["x"]])  # the packed projection's output
        s["q"], s["new_k"], s["new_v"] = qkv.split([c["heads"], c["kv_heads"], c["kv_heads"]], 1)
        f, s["factor"] = _inv_freq(c)
        s["inv_freq"] = dev(f.astype(np.float32))
    elif c["op"] == "fork":
        lens, shared = _fork_rows(c)
        rows, W = len(lens), c["beams"]
        counts = -(-lens // c["page"])
        mine = counts - shared
        used = int(mine.sum() + shared[::W].sum())
        pages = used + used // 4 + rows * (2 + c["room"] // c["page"]) + 1
        ids = rng.permutation(pages)
        t = np.full((rows, int(counts.max()) + 2 + c["room"] // c["page"]), -1, np.int32)
        at = 0
        for r in range(rows):
            lead = r - r % W
            if r == lead:
                t[r, :shared[r]] = ids[at:at + shared[r]]
                at += shared[r]
            t[r, :shared[r]] = t[lead, :shared[r]]
            t[r, shared[r]:counts[r]] = ids[at:at + mine[r]]
            at += mine[r]
        s["k"], s["v"] = _pool(c, c["layers"], pages, gen)
        s["tables"], s["lens"] = dev(t), dev(lens.astype(np.int32))
        s["refs"] = dev(np.bincount(t[t >= 0], minlength=pages).astype(np.int32))
        who = rng.permuted(np.tile(np.arange(W) // 2, (c["groups"], 1)), axis=1)  # half of the beams go on, twice each
        pick = rng.permuted(np.tile(np.arange(W), (c["groups"], 1)), axis=1)
        s["parents"] = dev((np.take_along_axis(pick, who, 1) + W * np.arange(c["groups"])[:, None]).reshape(-1).astype(np.int32))
    elif c["op"] == "compact":
        N, n = c["pages"], c["live"]
        move = n * (N - n) // N
        live = np.concatenate([rng.permutation(n)[:n - move], n + rng.permutation(N - n)[:move]])
        live = rng.permutation(live)
        share = live[: n // 4]  # a quarter of the pages, in every row's front
        rest = np.array_split(live[n // 4:], c["seqs"])
        t = np.full((c["seqs"], len(share) + max(len(r) for r in rest) + 1), -1, np.int32)
        for r, own_pages in enumerate(rest):
            t[r, :len(share)] = share
            t[r, len(share):len(share) + len(own_pages)] = own_pages
        s["k"], s["v"] = _pool(c, c["layers"], N, gen)
        s["tables"] = dev(t)
        s["refs"] = dev(np.bincount(t[t >= 0], minlength=N).astype(np.int32))
    else:
        rows = c["groups"] * c["beams"]
        logits = 2.5 * torch.randn((rows, c["vocab"]), generator=gen, device="cuda")
        logits[:, 5::97] = -math.inf  # tokens that the caller bans
        s["logits"] = logits.to(TORCH[c["x"]])
        s["scores"] = dev((-12.0 + 3.0 * rng.standard_normal((c["groups"], c["beams"]))).astype(np.float32))
        done = np.zeros((c["groups"], c["beams"]), np.int32)
        for g in range(c["groups"]):
            done[g, rng.permutation(c["beams"])[:c["finished"]]] = 1
        s["finished"], s["eos"] = dev(done), 128001 % c["vocab"]
    if own:  # the cache, the rotation and the next step's tables that a program keeps
        from cudallm_b200 import paged
        s["paged"] = paged
        if "k" in s:
            s["cache"] = paged.PagedCache(s["k"], s["v"])
        if c["op"] == "rope":
            s["rope"] = paged.Rope(s["inv_freq"], interleaved=c["interleaved"], factor=s["factor"])
    return s


# ---- one pass ---------------------------------------------------------------------------------

def run(s):
    c = s["case"]
    if own:
        if c["op"] == "attention":
            out, lse = s["cache"].attend(s["q"], s["tables"], s["lens"], window=c["window"], with_lse=True)
            return {"out": out, "lse": lse}
        if c["op"] == "rope":
            q = s["cache"].append(s["q"], s["new_k"], s["new_v"], s["positions"], s["tables"], s["rope"], rows=s["rows"])
            return {"q": q, "k": s["k"], "v": s["v"]}
        if c["op"] == "fork":
            t, n, r, missing = s["cache"].fork(s["tables"], s["lens"], s["refs"], s["parents"], room=c["room"])
            return {"tables": t, "lens": n, "refs": r, "missing": missing, "k": s["k"], "v": s["v"]}
        if c["op"] == "compact":
            t, r, live = s["cache"].compact(s["tables"], s["refs"])
            return {"tables": t, "refs": r, "live": live, "k": s["k"], "v": s["v"]}
        scores, parents, tokens = s["paged"].beam_select(s["logits"], s["scores"], keep=c["keep"], finished=s["finished"], eos=s["eos"])
        return {"scores": scores, "parents": parents, "tokens": tokens}
    return {"attention": plain_attention, "rope": plain_rope, "fork": plain_fork, "compact": plain_compact, "beam": plain_beam}[c["op"]](s)


def plain_attention(s):
    c, q, t, lens = s["case"], s["q"].float(), s["tables"].long(), s["lens"].long()
    B, P = t.shape
    kv, page, dim = c["kv_heads"], c["page"], c["dim"]
    T = P * page
    at = torch.arange(T, device="cuda")
    keep = (at < lens[:, None]) & ((t >= 0) & (t < s["k"].shape[1])).repeat_interleave(page, 1)
    if c["window"]:
        keep &= at >= lens[:, None] - c["window"]
    ids = t.clamp(0, s["k"].shape[1] - 1)
    k = s["k"][0][ids].float().transpose(1, 2).reshape(B, kv, T, dim)
    v = s["v"][0][ids].float().transpose(1, 2).reshape(B, kv, T, dim)
    v = torch.where(keep[:, None, :, None], v, 0.0)  # what lies in unused places may be anything
    x = torch.matmul(q.view(B, kv, -1, dim), k.transpose(2, 3)) * (1.0 / math.sqrt(dim))
    x = torch.where(keep[:, None, None], x, -math.inf)
    m = x.amax(3, keepdim=True)
    p = torch.exp(x - torch.where(m > -math.inf, m, 0.0))
    total = p.sum(3, keepdim=True)
    out = torch.matmul(p, v) / torch.where(total > 0, total, 1.0)
    return {"out": out.view(B, -1, dim).to(s["q"].dtype), "lse": (m + torch.log(total)).view(B, -1)}


def plain_rope(s):
    c, pos = s["case"], s["positions"].long()
    n = s["inv_freq"].numel()
    angle = pos.float()[:, None] * s["inv_freq"]
    cos, sin = (torch.cos(angle) * s["factor"])[:, None], (torch.sin(angle) * s["factor"])[:, None]

    def turned(x):
        x = x.float()
        rot, rest = x[..., :2 * n], x[..., 2 * n:]
        a, b = (rot[..., 0::2], rot[..., 1::2]) if c["interleaved"] else (rot[..., :n], rot[..., n:])
        y = [a * cos - b * sin, b * cos + a * sin]
        y = torch.stack(y, -1).flatten(-2) if c["interleaved"] else torch.cat(y, -1)
        return torch.cat([y, rest], -1)

    page = s["tables"].long()[s["rows"].long(), pos // c["page"]]
    s["k"][0][page, :, pos % c["page"]] = turned(s["new_k"]).to(s["k"].dtype)
    s["v"][0][page, :, pos % c["page"]] = s["new_v"].to(s["v"].dtype)
    return {"q": turned(s["q"]).to(s["q"].dtype), "k": s["k"], "v": s["v"]}


def plain_fork(s):
    """Row i of the new tables continues row parents[i] (outside the rows: an empty row). Its full pages are its parent's, shared. The
    first child of a parent also keeps the parent's pages from the first not full one on, if nobody else refers to that one; any
    other child gets a page of its own with a copy of the tokens of that page. Then each row gets the pages that `room` more
    tokens need. New pages are the lowest of those with no reference before, in the order of the rows; where there
    are too few the entry is -1. refs counts each page's references by rows; `missing` is how many pages there were too few."""
    c, t, refs, par = s["case"], s["tables"].long(), s["refs"].long(), s["parents"].long()
    lens, page, N = s["lens"].long(), c["page"], s["refs"].numel()
    R, P = t.shape
    rows, col = torch.arange(len(par), device="cuda"), torch.arange(P, device="cuda")
    alive = (par >= 0) & (par < R)
    p = par.clamp(0, R - 1)
    spot = torch.where(alive, par, R)
    children = torch.zeros(R + 1, dtype=torch.long, device="cuda").scatter_add(0, spot, torch.ones_like(par))
    first = torch.full((R + 1,), len(par), device="cuda").scatter_reduce(0, spot, rows, "amin")
    full, tail = lens // page, lens % page
    good = (t >= 0) & (t < N)
    held = ((col < full[:, None]) | good).long().cumprod(1).sum(1)
    at = t.clamp(0, N - 1).gather(1, full.clamp(max=P - 1)[:, None])[:, 0]
    alone = (held > full) & (refs[at] == 1)
    keeps = alive & (first[p] == rows) & alone[p]
    want = torch.where(alive, (lens[p] + c["room"] + page - 1) // page, 0)
    base = torch.where(keeps, held[p], full[p])
    fresh = torch.where(alive, (want.clamp(max=P) - base).clamp(min=0), 0)
    start = fresh.cumsum(0) - fresh
    free = torch.argsort((refs != 0).long(), stable=True)
    n_free = (refs == 0).sum()
    rank = start[:, None] + col - base[:, None]
    new = (col >= base[:, None]) & (col < (base + fresh)[:, None])
    got = new & (rank < n_free)
    out = torch.where(alive[:, None] & (col < base[:, None]) & good[p], t[p], -1)
    out = torch.where(got, free[rank.clamp(0, N - 1)], out)
    missing = (new & ~got).sum() + torch.where(alive, (want - P).clamp(min=0), 0).sum()
    gain = torch.where(col < full[:, None], children[:R, None] - 1, torch.where((alone & (children[:R] > 0))[:, None], 0, -1))
    gain = torch.where(good & (col < held[:, None]), gain, 0)
    refs = torch.cat([refs, refs.new_zeros(1)])
    refs = refs.scatter_add(0, torch.where(good, t, N).view(-1), gain.view(-1))
    refs = refs.scatter_add(0, torch.where(got, out, N).view(-1), got.long().view(-1))[:N]
    src, dst = at[p], out.gather(1, full[p].clamp(max=P - 1)[:, None])[:, 0]
    copies = alive & ~keeps & (tail[p] > 0) & (held > full)[p] & (full[p] < P) & (dst >= 0)
    lead = copies.long().argmax()  # a row without a copy repeats the first one; without any, page 0 is written over itself
    some = copies.any()
    src = torch.where(copies, src, torch.where(some, src[lead], 0))
    dst = torch.where(copies, dst, torch.where(some, dst[lead], 0))
    n = torch.where(copies, tail[p], tail[p][lead])
    fill = (torch.arange(page, device="cuda") < n[:, None])[None, :, None, :, None]
    for_k = torch.where(fill, s["k"][:, src], s["k"][:, dst])
    for_v = torch.where(fill, s["v"][:, src], s["v"][:, dst])
    s["k"][:, dst] = for_k
    s["v"][:, dst] = for_v
    return {"tables": out.int(), "lens": torch.where(alive, lens[p], 0).int(), "refs": refs.int(), "missing": missing.int().view(1), "k": s["k"], "v": s["v"]}


def plain_compact(s):
    """The n pages with references come to be the first n: the k-th lowest page without one among the first n takes the k-th lowest page in use
    that lies after them, with its content in every layer. Entries of the tables and references follow; entries without a page become -1."""
    t, refs = s["tables"].long(), s["refs"]
    N = refs.numel()
    idx = torch.arange(N, device="cuda")
    used = refs > 0
    n = used.sum()
    src = torch.nonzero(used & (idx >= n))[:, 0]
    dst = torch.nonzero(~used & (idx < n))[:, 0]
    to = idx.scatter(0, src, dst)
    s["k"][:, dst] = s["k"][:, src]
    s["v"][:, dst] = s["v"][:, src]
    good = (t >= 0) & (t < N)
    new_refs = torch.zeros_like(refs).scatter_add(0, torch.where(used, to, N - 1), torch.where(used, refs, 0))
    return {"tables": torch.where(good, to[t.clamp(0, N - 1)], -1).int(), "refs": new_refs, "live": n.int().view(1), "k": s["k"], "v": s["v"]}


def plain_beam(s):
    """Candidate (w, t) of a group: scores[w] + (logits[w, t] - lse(logits[w])); the row of a finished beam is read as 0 at `eos` and -inf elsewhere; a
    candidate that is not a number counts as -inf. The `keep` best of a group: by candidate, then the lower beam, then the larger
    logit (not a number: -inf), then the lower token. Parents are rows of the logits."""
    c, x = s["case"], s["logits"].float()
    W, K, V = c["beams"], c["keep"], c["vocab"]
    done = s["finished"].view(-1, 1) != 0
    x = torch.where(done, torch.where(torch.arange(V, device="cuda") == s["eos"], 0.0, -math.inf), x)
    m = x.amax(1, keepdim=True)
    lse = m + torch.log(torch.exp(x - m).sum(1, keepdim=True))
    key = torch.where(torch.isnan(x), -math.inf, x)
    order = torch.sort(key, dim=1, descending=True, stable=True).indices[:, :K]
    cand = s["scores"].view(-1, 1) + (x.gather(1, order) - lse)
    cand = torch.where(torch.isnan(cand), -math.inf, cand).reshape(c["groups"], -1)
    best = torch.sort(cand, dim=1, descending=True, stable=True).indices[:, :K]
    width = order.shape[1]
    parents = best // width + W * torch.arange(c["groups"], device="cuda")[:, None]
    return {"scores": cand.gather(1, best), "parents": parents.int(), "tokens": order.reshape(c["groups"], -1).gather(1, best).int()}


# ---- what a pass cannot do without -------------------------------------------------------------

def work(case):
    c = case
    es = 2  # of the cache
    if c["op"] == "attention":
        lens = _lens(c, None)
        seen = int(np.minimum(lens, c["window"] or lens).sum())
        xs = TORCH[c["q"]].itemsize
        rows = c["seqs"] * c["heads"]
        return {"bytes": 2 * seen * c["kv_heads"] * c["dim"] * es + rows * (2 * c["dim"] * xs + 4) + 4 * int((-(-lens // c["page"])).sum()) + 4 * c["seqs"],
                "flops": 4 * seen * c["heads"] * c["dim"]}
    if c["op"] == "rope":
        n, xs = c["seqs"] * c["each"], TORCH[c["x"]].itemsize
        return {"bytes": n * c["dim"] * ((2 * c["heads"] + 2 * c["kv_heads"]) * xs + 2 * c["kv_heads"] * es) + 12 * n,
                "flops": 3 * n * c["rotary"] * (c["heads"] + c["kv_heads"])}
    if c["op"] == "fork":
        lens, shared = _fork_rows(c)
        W = c["beams"]
        more = W - -(-W // 2)
        copied = int((lens % c["page"])[::W].sum()) * more * c["layers"] * c["kv_heads"] * c["dim"] * es * 2
        entries = int((-(-lens // c["page"])).sum())
        return {"bytes": 2 * copied + 8 * entries + 12 * len(lens), "flops": 0}
    if c["op"] == "compact":
        n = c["live"]
        move = n * (c["pages"] - n) // c["pages"]
        page = c["layers"] * c["kv_heads"] * c["page"] * c["dim"] * es * 2
        return {"bytes": 2 * move * page + 8 * c["pages"] + 8 * (n - n // 4 + c["seqs"] * (n // 4)), "flops": 0}
    rows = c["groups"] * c["beams"]
    read = (rows - c["groups"] * c["finished"]) * c["vocab"]
    return {"bytes": read * TORCH[c["x"]].itemsize + 8 * rows + 12 * c["groups"] * c["keep"], "flops": 4 * read}


# ---- the definitions again, in 64 bits -------------------------------------------------------------

def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    c = case
    host = {n: x.cpu().numpy() for n, x in s.items() if torch.is_tensor(x) and x.dtype == torch.int32}
    if c["op"] == "attention":
        outs, lses = [], []
        for b in range(c["seqs"]):
            n = int(host["lens"][b])
            q = s["q"][b].double().view(c["kv_heads"], -1, c["dim"])
            ids = torch.from_numpy(host["tables"][b][:-(-n // c["page"])].astype(np.int64)).cuda()
            k, v = (s[w][0][ids].permute(1, 0, 2, 3).reshape(c["kv_heads"], -1, c["dim"])[:, :n].double() for w in "kv")
            first = max(0, n - c["window"]) if c["window"] else 0
            x = torch.einsum("hgd,htd->hgt", q, k[:, first:]) / math.sqrt(c["dim"])
            lse = torch.logsumexp(x, 2) if n else torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device="cuda")
            outs.append(torch.einsum("hgt,htd->hgd", torch.exp(x - lse[..., None]), v[:, first:]).reshape(-1, c["dim"]) if n else torch.zeros_like(q).view(-1, c["dim"]))
            lses.append(lse.reshape(-1))
        return {"out": torch.stack(outs), "lse": torch.stack(lses)}
    if c["op"] == "rope":
        f32 = s["positions"].to(torch.float32)[:, None] * s["inv_freq"][None]
        turn = torch.polar(torch.full_like(f32, s["factor"], dtype=torch.float64), f32.double())[:, None]
        n = s["inv_freq"].numel()

        def turned(x):
            x = x.double()
            y = x.clone()
            pair = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if c["interleaved"] else (slice(0, n), slice(n, 2 * n))
            z = torch.complex(x[..., pair[0]].contiguous(), x[..., pair[1]].contiguous()) * turn
            y[..., pair[0]], y[..., pair[1]] = z.real, z.imag
            return y

        k, v = s["k"].double(), s["v"].double()
        new_k, new_v, each = turned(s["new_k"]), s["new_v"].double(), c["each"]
        for r in range(c["seqs"]):
            pos = host["positions"][r * each:(r + 1) * each].astype(np.int64)
            page = torch.from_numpy(host["tables"][r][pos // c["page"]].astype(np.int64)).cuda()
            slot = torch.from_numpy(pos % c["page"]).cuda()
            for h in range(c["kv_heads"]):
                k[0, :, h][page, slot] = new_k[r * each:(r + 1) * each, h]
                v[0, :, h][page, slot] = new_v[r * each:(r + 1) * each, h]
        return {"q": turned(s["q"]), "k": k, "v": v}
    if c["op"] == "fork":
        t, lens, refs, par, page = host["tables"], host["lens"], host["refs"].copy(), host["parents"], c["page"]
        free = list(np.nonzero(refs == 0)[0])
        k, v = s["k"].double(), s["v"].double()
        out, new_lens, missing, kept, gone = np.full((len(par), t.shape[1]), -1, np.int32), [], 0, set(), host["refs"].copy()
        for r in range(len(t)):
            for j in t[r][t[r] >= 0]:
                gone[j] -= 1
        for i, p in enumerate(par):
            n = int(lens[p])
            full, tail = divmod(n, page)
            row = list(t[p][:full])
            if p not in kept and t[p][full] >= 0 and refs[t[p][full]] == 1:
                kept.add(p)
                row += [j for j in t[p][full:] if j >= 0]
            elif tail:
                got = free.pop(0)
                k[:, got, :, :tail], v[:, got, :, :tail] = k[:, t[p][full], :, :tail], v[:, t[p][full], :, :tail]
                row.append(got)
            while len(row) * page < n + c["room"]:
                row.append(free.pop(0))
            out[i, :len(row)] = row
            for j in row:
                gone[j] += 1
            new_lens.append(n)
        return {"tables": out, "lens": np.array(new_lens, np.int32), "refs": gone, "missing": np.array([missing], np.int32), "k": k, "v": v}
    if c["op"] == "compact":
        t, refs = host["tables"].copy(), host["refs"]
        n = int((refs > 0).sum())
        k, v = s["k"].double(), s["v"].double()
        to, holes, new = {}, [i for i in range(n) if refs[i] == 0], np.zeros_like(refs)
        for i in np.nonzero(refs)[0]:
            to[i] = holes[len([j for j in to if j >= n])] if i >= n else i
            new[to[i]] = refs[i]
            if i >= n:
                k[:, to[i]], v[:, to[i]] = s["k"][:, int(i)].double(), s["v"][:, int(i)].double()
        for r in range(t.shape[0]):
            t[r] = [to[j] if j >= 0 else -1 for j in t[r]]
        return {"tables": t, "refs": new, "live": np.array([n], np.int32), "k": k, "v": v}
    scores, parents, tokens = [], [], []
    for g in range(c["groups"]):
        found = []
        for w in range(c["beams"]):
            row = s["logits"][g * c["beams"] + w].double().cpu().numpy()
            base = float(s["scores"][g, w])
            if host["finished"][g, w]:
                row = np.full_like(row, -math.inf)
                row[s["eos"]] = 0.0
            lse = row.max() + math.log(np.exp(row - row.max()).sum())
            order = np.lexsort((np.arange(row.size), -row))[:c["keep"]]
            found += [(-(base + row[t] - lse), w, i, t) for i, t in enumerate(order)]
        found = sorted(found)[:c["keep"]]
        scores.append([-f[0] for f in found])
        parents.append([g * c["beams"] + f[1] for f in found])
        tokens.append([f[3] for f in found])
    return {"scores": np.array(scores), "parents": np.array(parents, np.int32), "tokens": np.array(tokens, np.int32)}
