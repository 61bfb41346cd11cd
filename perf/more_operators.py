"""Performance cases of streams that generate row after row: attention under a window that keeps a clip's first rows in
sight, attention of new rows (single ones, drafted trees, chunks) over kept rows in pages, and what is done with the
pages: taking, writing, forking, copying, freeing and compacting them.

The shapes are those of the two workloads that this repository measures: 40 heads of the 768p block (129,536 rows a batch)
and 56 of the H3 block at 960 x 544 (19,305 rows: 37 frames of 510 and 435 text rows, which are what stays in sight), and
single images, short clips and packed batches of them. `draw` gives more of the same ranges.
"""
import math
import random
import sys
from pathlib import Path

import torch

own = False

DEV = "cuda"
BF16, F32, F64, I32 = torch.bfloat16, torch.float32, torch.float64, torch.int32


def _lib():
    if "mako_h3" in sys.modules:
        return sys.modules["mako_h3"]
    root = str(Path(__file__).resolve().parent.parent / "mako-video_amd")
    if root not in sys.path:
        sys.path.insert(0, root)
    import mako_h3

    return mako_h3


def listed():
    return [
        # A single 480 x 272 image (135 rows and 77 of text) generated row after row, a few first rows kept in sight: the
        # smallest call, all latency.
        {"name": "window_image", "op": "window", "heads": 40, "kv_heads": 8, "docs": 1, "rows": 212, "sinks": 4,
         "window": 64, "causal": True, "cap": 0.0, "layout": "rows"},
        # Five clips of uneven lengths packed into one batch, each row looking two 510-row frames either way and at its
        # clip's text, scores capped.
        {"name": "window_packed_clips", "op": "window", "heads": 40, "kv_heads": 40, "docs": 5, "rows": 14925,
         "sinks": 77, "window": 1020, "causal": False, "cap": 30.0, "layout": "rows"},
        # The whole 960 x 544 clip, causal over eight frames and the text: the largest call.
        {"name": "window_960x544", "op": "window", "heads": 56, "kv_heads": 56, "docs": 1, "rows": 19305, "sinks": 435,
         "window": 4080, "causal": True, "cap": 0.0, "layout": "heads"},
        # One new row of each of three streams, all their kept rows (those of the 768p batch) in sight.
        {"name": "pages_new_rows", "op": "pages", "heads": 40, "kv_heads": 8, "streams": 3, "kept": 129536, "new": 1,
         "tree": False, "page": 64, "sinks": 0, "window": 0, "cap": 0.0, "layout": "rows", "page_layout": "heads"},
        # One new row of each of 64 streams under a window; the pages behind it were freed.
        {"name": "pages_window_rows", "op": "pages", "heads": 40, "kv_heads": 8, "streams": 64, "kept": 129536, "new": 1,
         "tree": False, "page": 16, "sinks": 16, "window": 1020, "cap": 0.0, "layout": "rows", "page_layout": "rows"},
        # Eight drafts over a short clip's kept rows: all latency.
        {"name": "pages_tree_clip", "op": "pages", "heads": 56, "kv_heads": 56, "streams": 1, "kept": 2985, "new": 8,
         "tree": True, "page": 32, "sinks": 0, "window": 0, "cap": 0.0, "layout": "heads", "page_layout": "heads"},
        # 63 drafts of each of five streams over long histories.
        {"name": "pages_tree_long", "op": "pages", "heads": 40, "kv_heads": 8, "streams": 5, "kept": 129536, "new": 63,
         "tree": True, "page": 64, "sinks": 0, "window": 0, "cap": 0.0, "layout": "heads", "page_layout": "heads"},
        # The next frame of two streams (510 rows, row after row) over eight frames and the text.
        {"name": "pages_frame", "op": "pages", "heads": 56, "kv_heads": 56, "streams": 2, "kept": 19305, "new": 510,
         "tree": False, "page": 64, "sinks": 435, "window": 4080, "cap": 0.0, "layout": "heads",
         "page_layout": "heads"},
        # Places for 510 new rows of each of three streams, and the rows into them, two layers.
        {"name": "append_frame", "op": "append", "kv_heads": 8, "streams": 3, "kept": 14925, "new": 510, "page": 64,
         "layers": 2, "layout": "rows", "accepted": False},
        # Eight candidates that go on from two of them: full pages shared, the ones begun copied.
        {"name": "fork_candidates", "op": "fork", "kv_heads": 8, "streams": 8, "kept": 16384, "page": 64, "layers": 4},
        # 512 pages of one layer copied.
        {"name": "copy_pages", "op": "copy", "kv_heads": 8, "streams": 3, "kept": 65536, "page": 64, "layers": 1,
         "pairs": 512},
        # Two of five streams end: their pages are freed, and the others' moved together.
        {"name": "free_compact", "op": "compact", "kv_heads": 8, "streams": 5, "kept": 129536, "page": 64, "layers": 2},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["window"] * 4 + ["pages"] * 5 + ["append", "fork", "copy", "compact"])
    heads = rng.choice([7, 40, 56])
    kv_heads = rng.choice([heads, 8 if heads > 7 else 1])
    if op == "window":
        case = {"op": op, "heads": heads, "kv_heads": kv_heads, "docs": rng.randint(1, 5), "rows": _log(rng, 64, 16000),
                "sinks": rng.choice([0, 1, 4, 77, 435]), "window": _log(rng, 1, 8000), "causal": rng.random() < 0.7,
                "cap": rng.choice([0.0, 0.0, 30.0]), "layout": rng.choice(["heads", "rows"])}
        case["docs"] = min(case["docs"], case["rows"] // 16)
        return case
    streams, page = _log(rng, 1, 64), rng.choice([16, 32, 64, 128])
    if op == "pages":
        kind = rng.choice(["row", "row", "tree", "tree", "chunk"])
        new = 1 if kind == "row" else _log(rng, 2, 64) if kind == "tree" else _log(rng, 2, 510)
        if kind == "chunk":
            streams = min(streams, 4)
        kept = _log(rng, 64, min(129536, 1 << 24 if new == 1 else 40_000_000 // (new * min(streams, 8))))
        if kv_heads > 8:
            kept = min(kept, 40000)
        return {"op": op, "heads": heads, "kv_heads": kv_heads, "streams": streams, "kept": kept, "new": new,
                "tree": kind == "tree", "page": page, "sinks": rng.choice([0, 1, 4, 77, 435]),
                "window": rng.choice([0, _log(rng, 1, 8000)]), "cap": rng.choice([0.0, 0.0, 30.0]),
                "layout": rng.choice(["heads", "rows"]), "page_layout": rng.choice(["heads", "rows"])}
    case = {"op": op, "kv_heads": min(kv_heads, 8), "streams": min(streams, 24), "kept": _log(rng, 200, 65536), "page": page,
            "layers": rng.randint(1, 3)}
    if op == "append":
        case.update(new=_log(rng, 1, 510), layout=rng.choice(["heads", "rows"]), accepted=rng.random() < 0.5)
    elif op == "copy":
        case.update(pairs=_log(rng, 1, max(1, case["kept"] // page // 2)))
    return case


# ---- inputs ----------------------------------------------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _uneven(total, n):
    """n whole numbers, 1 : 2 : 3 ..., that add up to total."""
    cuts = [total * i * (i + 1) // (n * (n + 1)) for i in range(n + 1)]
    return [b - a for a, b in zip(cuts, cuts[1:])]


def _ints(x):
    return torch.tensor(x, dtype=I32, device=DEV)


def _offsets(lengths):
    return torch.tensor([0] + lengths, device=DEV).cumsum(0).int()


def _rows_of(x, layout):
    """[heads][rows][128] as the layout holds it."""
    return x if layout == "heads" else x.transpose(0, 1).contiguous().view(x.shape[1], -1)


def _heads_of(x, layout):
    """[heads][rows][128] of a tensor in the layout."""
    return x if layout == "heads" else x.view(x.shape[0], -1, 128).transpose(0, 1)


def _content(g, heads, rows, mix):
    """Head rows of unit variance: a few directions that all of a head's rows mix, and noise."""
    c = torch.randn((heads, rows, 8), generator=g, device=DEV)
    return (0.8 * torch.randn((heads, rows, 128), generator=g, device=DEV) + 0.6 / math.sqrt(8) * (c @ mix)).to(BF16)


def _live(case, kept):
    """The kept rows of a stream that a new row may see, as spans of whole pages [first, last): the first rows', and those
    that the window reaches."""
    page, count = case["page"], -(-kept // case["page"])
    if not case["window"]:
        return [(0, count)]
    reach = max(0, kept - case["window"] + 1) // page
    front = min(-(-min(case["sinks"], kept) // page), reach)
    return [(0, front), (reach, count)]


def _tables(case, seed, lengths, spare, live=None):
    """A table of shuffled pages for the lengths (of the spans live(length) only), the pages' reference counts, and how many
    pages there are."""
    page, rng = case["page"], random.Random(seed)
    spans = [live(n) if live else [(0, -(-n // page))] for n in lengths]
    used = sum(b - a for sp in spans for a, b in sp)
    pages = used + spare
    numbers = rng.sample(range(pages), used)
    cols = max(max((-(-n // page) for n in lengths), default=1), 1) + spare // max(len(lengths), 1) + 1
    table = torch.full((len(lengths), cols), -1, dtype=I32)
    at = 0
    for s, sp in enumerate(spans):
        for a, b in sp:
            table[s, a:b] = torch.tensor(numbers[at:at + b - a], dtype=I32)
            at += b - a
    refs = torch.zeros(pages, dtype=I32)
    refs[torch.tensor(numbers, dtype=torch.long)] = 1
    return table.to(DEV), refs.to(DEV), pages


def _trees(case, seed):
    """Each new row's parent among its stream's, -1 for a root: a row goes on from one of the eight before it."""
    rng = random.Random(seed + 1)
    return [[-1 if i == 0 else rng.randint(max(0, i - 8), i - 1) for i in range(case["new"])]
            for _ in range(case["streams"])]


def prepare(case, seed):
    g, op, s = _gen(seed), case["op"], {"case": case}
    if op == "window":
        heads, kv_heads, rows = case["heads"], case["kv_heads"], case["rows"]
        mix = torch.randn((heads, 8, 128), generator=g, device=DEV)
        q = _content(g, heads, rows, mix)
        k = _content(g, kv_heads, rows, mix[::heads // kv_heads])
        v = torch.randn((kv_heads, rows, 128), generator=g, device=DEV).to(BF16)
        s["q"], s["k"], s["v"] = (_rows_of(x, case["layout"]) for x in (q, k, v))
        s["off"] = _offsets(_uneven(rows, case["docs"]))
        s["sinks"] = torch.full((case["docs"],), case["sinks"], dtype=I32, device=DEV)
        return s
    lengths = _uneven(case["kept"], case["streams"])
    s["lengths"] = _ints(lengths)
    kv_heads, page = case["kv_heads"], case["page"]
    if op == "pages":
        heads, new = case["heads"], case["new"] * case["streams"]
        s["table"], _, pages = _tables(case, seed, lengths, 16, lambda n: _live(case, n))
        mix = torch.randn((heads, 8, 128), generator=g, device=DEV)
        share = mix[::heads // kv_heads]
        q, k = _content(g, heads, new, mix), _content(g, kv_heads, new, share)
        v = torch.randn((kv_heads, new, 128), generator=g, device=DEV).to(BF16)
        s["q"], s["k"], s["v"] = (_rows_of(x, case["layout"]) for x in (q, k, v))
        pools = (_content(g, kv_heads, pages * page, share),
                 torch.randn((kv_heads, pages * page, 128), generator=g, device=DEV).to(BF16))
        for name, pool in zip(("k_pages", "v_pages"), pools):
            pool = pool.view(kv_heads, pages, page, 128)
            s[name] = pool.transpose(0, 1).contiguous() if case["page_layout"] == "heads" else \
                pool.permute(1, 2, 0, 3).reshape(pages, page, -1)
        s["q_off"] = _offsets([case["new"]] * case["streams"])
        s["parents"] = _ints(sum(_trees(case, seed), [])) if case["tree"] else None
        s["sinks"] = torch.full((case["streams"],), case["sinks"], dtype=I32, device=DEV) if case["sinks"] else None
        return s
    extra = case["streams"] * (2 + (case.get("new", 0) + page - 1) // page) + case.get("pairs", 0)
    s["table"], s["refs"], pages = _tables(case, seed, lengths, extra)
    s["pool"] = torch.randn((pages, case["layers"], 2, kv_heads, page, 128), generator=g, device=DEV, dtype=F32).to(BF16)
    rng = random.Random(seed + 2)
    if op == "append":
        new = case["new"] * case["streams"]
        s["k"], s["v"] = ([_rows_of(torch.randn((kv_heads, new, 128), generator=g, device=DEV).to(BF16), case["layout"])
                           for _ in range(case["layers"])] for _ in range(2))
        counts, rows = [case["new"]] * case["streams"], None
        if case["accepted"]:    # of each stream's drafts the rows of one path
            paths = [sorted(rng.sample(range(case["new"]), rng.randint(1, case["new"]))) for _ in counts]
            counts = [len(p) for p in paths]
            rows = _ints([i * case["new"] + j for i, p in enumerate(paths) for j in p])
        s["off"], s["rows"] = _offsets(counts), rows
        s["first"] = _ints([-(-n // page) for n in lengths])
        s["last"] = _ints([-(-(n + c) // page) for n, c in zip(lengths, counts)])
    elif op == "fork":
        alive = rng.sample(range(case["streams"]), max(1, case["streams"] // 4))
        parents = [rng.choice(alive) for _ in lengths]
        for a in alive:
            parents[a] = a
        s["parents"], s["rows"] = _ints(parents), _ints([lengths[p] for p in parents])
    elif op == "copy":
        refs = s["refs"].cpu()
        s["src"] = _ints(rng.choices(torch.nonzero(refs > 0).flatten().tolist(), k=case["pairs"]))
        s["dst"] = _ints(rng.sample(torch.nonzero(refs == 0).flatten().tolist(), case["pairs"]))
    else:
        ended = rng.sample(range(case["streams"]), -(-2 * case["streams"] // 5))
        s["first"] = torch.zeros(case["streams"], dtype=I32, device=DEV)
        s["last"] = _ints([s["table"].shape[1] if i in ended else 0 for i in range(case["streams"])])
    return s


# ---- the plain forms -------------------------------------------------------------------------------------------------

def _plain_softmax_v(p, v):
    """Softmax of the scores p over the last dimension, times v; rows that are all -inf are zero."""
    m = p.amax(-1, keepdim=True)
    p.sub_(m.masked_fill(m == -math.inf, 0.0)).exp_()
    total = p.sum(-1, keepdim=True)
    return torch.bmm(p.view(v.shape[0], -1, v.shape[1]), v).view(*p.shape[:-1], 128) / total.masked_fill(total == 0, 1.0)


def _plain_cap(p, cap):
    return p.div_(cap).tanh_().mul_(cap) if cap else p


def _plain_window(s, case):
    q, k, v = (_heads_of(s[n], case["layout"]) for n in ("q", "k", "v"))
    rows, share = q.shape[1], case["heads"] // case["kv_heads"]
    at = torch.arange(rows, device=DEV, dtype=I32)
    doc = torch.searchsorted(s["off"][1:].contiguous(), at, right=True)
    start, w = s["off"][doc][:, None], case["window"]
    seen = (at > at[:, None] - w) | (at < start + s["sinks"][doc][:, None])
    seen &= (at <= at[:, None]) if case["causal"] else (at < at[:, None] + w) | (at < start + s["sinks"][doc][:, None])
    seen &= doc == doc[:, None]
    masked = ~seen
    del seen
    out = torch.empty(q.shape, dtype=BF16, device=DEV)
    step = max(1, (1 << 31) // (share * rows * rows))   # a few key heads at a time: the scores of all would not fit
    for i in range(0, case["kv_heads"], step):
        heads = slice(i * share, min(i + step, case["kv_heads"]) * share)
        kt = k[i:i + step].float().transpose(1, 2).contiguous()
        x = q[heads].float().reshape(kt.shape[0], share * rows, 128)
        p = _plain_cap(torch.bmm(x * (1 / math.sqrt(128)), kt).view(-1, rows, rows), case["cap"])
        out[heads] = _plain_softmax_v(p.masked_fill_(masked, -math.inf), v[i:i + step].float()).to(BF16)
    return _rows_of(out, case["layout"])


def _plain_ancestors(parents):
    """Whether row j is row i or one of its ancestors [new][new], and the rows' depths, from one stream's parents."""
    new = parents.shape[0]
    line = torch.eye(new, dtype=torch.bool, device=DEV)
    depth = torch.zeros(new, dtype=I32, device=DEV)
    at = parents.clone()
    for _ in range(new - 1):
        up = at >= 0
        line |= (at[:, None] == torch.arange(new, device=DEV)) & up[:, None]
        depth += up
        at = torch.where(up, parents[at.clamp(min=0)], at)
    return line, depth


def _plain_pages(s, case):
    q, k, v = (_heads_of(s[n], case["layout"]) for n in ("q", "k", "v"))
    page, new, share, w = case["page"], case["new"], case["heads"] // case["kv_heads"], case["window"]
    out = torch.empty(q.shape, dtype=BF16, device=DEV)
    for i, kept in enumerate(_uneven(case["kept"], case["streams"])):
        entries = torch.cat([torch.arange(a, b, device=DEV) for a, b in _live(case, kept)])
        numbers = s["table"][i, entries]
        at = (entries[:, None] * page + torch.arange(page, device=DEV)).view(-1)     # the gathered rows' places
        mine = slice(i * new, (i + 1) * new)

        def keys(pool, fresh):
            rows = pool[numbers].float()
            rows = rows.transpose(0, 1) if case["page_layout"] == "heads" else \
                rows.view(-1, page, case["kv_heads"], 128).permute(2, 0, 1, 3)
            return torch.cat([rows.reshape(case["kv_heads"], -1, 128), fresh[:, mine].float()], 1)

        if s["parents"] is None:
            line = torch.ones((new, new), dtype=torch.bool, device=DEV).tril()
            depth = torch.arange(new, device=DEV)
        else:
            line, depth = _plain_ancestors(s["parents"][mine])
        place = torch.cat([at, kept + depth])
        seen = torch.cat([(at < kept).expand(new, -1), line], 1)
        if w:
            first = s["sinks"][i] if s["sinks"] is not None else 0
            seen = seen & ((place > (kept + depth)[:, None] - w) | (place < first))
        x = q[:, mine].float().reshape(case["kv_heads"], share * new, 128) * (1 / math.sqrt(128))
        p = torch.bmm(x, keys(s["k_pages"], k).transpose(1, 2).contiguous()).view(case["heads"], new, -1)
        p = _plain_cap(p, case["cap"]).masked_fill_(~seen, -math.inf)
        out[:, mine] = _plain_softmax_v(p, keys(s["v_pages"], v)).to(BF16)
    return _rows_of(out, case["layout"])


def _plain_append(s, case):
    table, refs, pool, page = s["table"].clone(), s["refs"].clone(), s["pool"], case["page"]
    cols = torch.arange(table.shape[1], device=DEV)
    want = (cols >= s["first"][:, None]) & (cols < s["last"][:, None]) & (table < 0)
    free = torch.nonzero(refs == 0).flatten()[:int(want.sum())]
    table[want] = free.int()
    refs[free] = 1
    count = s["off"][1:] - s["off"][:-1]
    n = int(s["off"][-1])
    stream = torch.repeat_interleave(torch.arange(case["streams"], device=DEV), count.long())
    place = s["lengths"][stream] + torch.arange(n, device=DEV) - s["off"][stream]
    number, row = table[stream, place // page].long(), place % page
    for layer in range(case["layers"]):
        for j, fresh in enumerate((s["k"][layer], s["v"][layer])):
            x = _heads_of(fresh, case["layout"]).transpose(0, 1)
            pool[number, layer, j, :, row] = x[s["rows"]] if s["rows"] is not None else x
    return table, refs, pool


def _plain_fork(s, case):
    table, page, streams = s["table"], case["page"], case["streams"]
    stays = (s["parents"] == torch.arange(streams, device=DEV))[:, None]
    cols = torch.arange(table.shape[1], device=DEV)
    full = (s["rows"] // page)[:, None]
    theirs = table[s["parents"]]
    new = torch.where(stays | (cols < full), theirs, -1)
    begun = ~stays & (cols == full) & (s["rows"] % page > 0)[:, None]
    src = theirs[begun]
    dst = torch.nonzero(s["refs"] == 0).flatten()[:src.shape[0]].int()
    new[begun] = dst
    refs = s["refs"].clone()
    for t, sign in ((table, -1), (new, 1)):
        refs.scatter_add_(0, t.clamp(min=0).view(-1).long(), (t >= 0).view(-1).int() * sign)
    s["pool"][dst.long()] = s["pool"][src.long()]
    return new, refs, s["pool"]


def _plain_compact(s, case):
    table, refs, pool = s["table"].clone(), s["refs"].clone(), s["pool"]
    cols = torch.arange(table.shape[1], device=DEV)
    gone = (cols >= s["first"][:, None]) & (cols < s["last"][:, None]) & (table >= 0)
    refs.scatter_add_(0, table.clamp(min=0).view(-1).long(), gone.view(-1).int().neg())
    table[gone] = -1
    used = refs > 0
    at = torch.arange(refs.shape[0], device=DEV)
    below = at < used.sum()
    src, dst = torch.nonzero(used & ~below).flatten(), torch.nonzero(~used & below).flatten()
    moved = torch.where(used, at, -1).int()
    moved[src] = dst.int()
    pool[dst] = pool[src]
    table = torch.where(table >= 0, moved[table.clamp(min=0)], -1)
    refs[dst] = refs[src]
    refs[src] = 0
    return table, refs, moved, pool


# ---- the calls -------------------------------------------------------------------------------------------------------

def _own_run(s, case):
    mh, op = _lib(), case["op"]
    if op == "window":
        rows = s["q"].shape[1] if case["layout"] == "heads" else s["q"].shape[0]
        ranges, sinks = mh.attn_window_ranges(s["off"], s["off"], rows, rows, case["window"], sinks=s["sinks"],
                                              causal=case["causal"])
        return mh.flash_attn_128(s["q"], s["k"], s["v"], ranges=ranges, sinks=sinks, cap=case["cap"],
                                 layout=case["layout"])
    if op == "pages":
        return mh.flash_attn_pages_128(s["q"], s["k"], s["v"], s["k_pages"], s["v_pages"], s["table"], s["lengths"],
                                       s["q_off"], parents=s["parents"], window=case["window"], sinks=s["sinks"],
                                       cap=case["cap"], layout=case["layout"], page_layout=case["page_layout"])
    # The table and the counts of a pass are the next one's too: each pass changes its own.
    if op == "append":
        table, refs = s["table"].clone(), s["refs"].clone()
        mh.pages_take(table, refs, s["first"], s["last"])
        for layer in range(case["layers"]):
            mh.pages_write(s["k"][layer], s["v"][layer], s["pool"][:, layer, 0], s["pool"][:, layer, 1], table,
                           s["lengths"], s["off"], rows=s["rows"], layout=case["layout"])
        return table, refs, s["pool"]
    if op == "fork":
        refs = s["refs"].clone()
        table, _ = mh.pages_fork(s["pool"], s["table"], refs, s["parents"], s["rows"], case["page"])
        return table, refs, s["pool"]
    if op == "copy":
        mh.pages_copy(s["pool"], s["src"], s["dst"])
        return s["pool"]
    table, refs = s["table"].clone(), s["refs"].clone()
    mh.pages_free(table, refs, s["first"], s["last"])
    moved, _ = mh.pages_compact(s["pool"], table, refs)
    return table, refs, moved, s["pool"]


def run(s):
    case, op = s["case"], s["case"]["op"]
    if own:
        return _own_run(s, case)
    if op == "window":
        return _plain_window(s, case)
    if op == "pages":
        return _plain_pages(s, case)
    if op == "append":
        return _plain_append(s, case)
    if op == "fork":
        return _plain_fork(s, case)
    if op == "copy":
        s["pool"][s["dst"].long()] = s["pool"][s["src"].long()]
        return s["pool"]
    return _plain_compact(s, case)


# ---- what a pass needs -----------------------------------------------------------------------------------------------

def _window_pairs(n, w, sinks, causal):
    """Query and key pairs of a document of n rows."""
    pairs, sinks = 0, min(sinks, n)
    for i in range(n):
        lo, hi = max(0, i - w + 1), i + 1 if causal else min(n, i + w)
        pairs += hi - lo + min(sinks, lo)
        if not causal and hi < sinks:
            pairs += sinks - hi
    return pairs


def _page_bytes(case):
    return case["layers"] * 2 * case["kv_heads"] * case["page"] * 256


def work(case):
    op = case["op"]
    if op == "window":
        pairs = sum(_window_pairs(n, case["window"], case["sinks"], case["causal"])
                    for n in _uneven(case["rows"], case["docs"]))
        return {"bytes": 512 * (case["heads"] + case["kv_heads"]) * case["rows"], "flops": 512.0 * case["heads"] * pairs}
    lengths = _uneven(case["kept"], case["streams"])
    if op == "pages":
        new, w, keys, pairs = case["new"], case["window"], 0, 0
        line = (new + 1) / 2 if not case["tree"] else min(new, 2 + new / 5)   # an ancestor line's rows, about
        for n in lengths:
            seen = n if not w else min(n, w - 1) + min(case["sinks"], max(0, n - w + 1))
            keys += seen
            pairs += new * (seen + line)
        rows = new * case["streams"]
        return {"bytes": 512 * (case["heads"] + case["kv_heads"]) * rows + 512 * case["kv_heads"] * keys,
                "flops": 512.0 * case["heads"] * pairs}
    if op == "append":
        rows = case["new"] * case["streams"] * (0.5 if case["accepted"] else 1)
        return {"bytes": int(1024 * rows * case["kv_heads"] * case["layers"]) + 4 * sum(lengths) // case["page"], "flops": 0}
    entries = 4 * sum(-(-n // case["page"]) for n in lengths)
    if op == "fork":
        return {"bytes": 2 * _page_bytes(case) * (case["streams"] - max(1, case["streams"] // 4)) + 4 * entries, "flops": 0}
    if op == "copy":
        return {"bytes": 2 * _page_bytes(case) * case["pairs"], "flops": 0}
    # Of the used pages' three fifths, two fifths of the places lie past where they end.
    return {"bytes": int(2 * _page_bytes(case) * entries / 4 * 0.24) + 4 * entries, "flops": 0}


# ---- the same in 64 bits ---------------------------------------------------------------------------------------------

def _exact_scores(x, keys, cap):
    score = x.double() @ keys.double().T.contiguous() / math.sqrt(128)
    return cap * torch.tanh(score / cap) if cap else score


def _exact_window(s, case):
    q, k, v = (_heads_of(s[n], case["layout"]) for n in ("q", "k", "v"))
    out, w, at = torch.zeros(q.shape, dtype=F64, device=DEV), case["window"], 0
    for n in _uneven(case["rows"], case["docs"]):
        hidden = torch.ones((n, n), dtype=torch.bool, device=DEV)
        hidden = hidden.triu(w) | hidden.tril(-w)
        hidden[:, :case["sinks"]] = False
        if case["causal"]:
            hidden |= torch.ones_like(hidden).triu(1)
        for h in range(case["heads"]):
            kh = h * case["kv_heads"] // case["heads"]
            score = _exact_scores(q[h, at:at + n], k[kh, at:at + n], case["cap"])
            out[h, at:at + n] = torch.softmax(score.masked_fill_(hidden, -math.inf), -1) @ v[kh, at:at + n].double()
        at += n
    return _rows_of(out, case["layout"])


def _exact_pages(s, case, seed):
    q, k, v = (_heads_of(s[n], case["layout"]) for n in ("q", "k", "v"))
    page, new, w = case["page"], case["new"], case["window"]
    out = torch.zeros(q.shape, dtype=F64, device=DEV)
    trees = _trees(case, seed) if case["tree"] else [list(range(-1, new - 1))] * case["streams"]
    for i, kept in enumerate(_uneven(case["kept"], case["streams"])):
        near = range(max(0, kept - w + 1) if w else 0, kept)
        places = list(range(0, min(case["sinks"], near.start))) + list(near)
        seen = torch.zeros((new, len(places) + new), dtype=torch.bool)
        spots = torch.tensor(places, dtype=torch.long)
        depth = []
        for r, up in enumerate(trees[i]):
            depth.append(0 if up < 0 else depth[up] + 1)
            mine = kept + depth[r]
            seen[r, :len(places)] = (spots > mine - w) | (spots < case["sinks"]) if w else True
            at = r
            while at >= 0:
                place = kept + depth[at]
                if not w or place > mine - w or place < case["sinks"]:
                    seen[r, len(places) + at] = True
                at = trees[i][at]
        hidden, spots = ~seen.to(DEV), spots.to(DEV)
        number, row = s["table"][i, spots // page].long(), spots % page
        for h in range(case["heads"]):
            kh = h * case["kv_heads"] // case["heads"]

            def rows(pool, fresh):
                kept_rows = pool[number, kh, row] if case["page_layout"] == "heads" else \
                    pool[number, row, 128 * kh:128 * kh + 128]
                return torch.cat([kept_rows, fresh[kh, i * new:(i + 1) * new]])

            score = _exact_scores(q[h, i * new:(i + 1) * new], rows(s["k_pages"], k), case["cap"])
            p = torch.softmax(score.masked_fill_(hidden, -math.inf), -1)
            out[h, i * new:(i + 1) * new] = p @ rows(s["v_pages"], v).double()
    return _rows_of(out, case["layout"])


def exact(case, seed):
    op = case["op"]
    if op == "pages" and case["streams"] * case["heads"] > 3000:
        return None     # minutes of small products
    s = prepare(case, seed)
    if op == "window":
        return _exact_window(s, case)
    if op == "pages":
        return _exact_pages(s, case, seed)
    # The tables and counts entry by entry, on the host; the pages as they then lie.
    table, refs, pool, page = s["table"].tolist(), s["refs"].tolist(), s["pool"], case["page"]
    lengths = s["lengths"].tolist()
    if op == "copy":
        for a, b in zip(s["src"].tolist(), s["dst"].tolist()):
            pool[b] = pool[a]
        return pool
    if op == "append":
        first, last, off = s["first"].tolist(), s["last"].tolist(), s["off"].tolist()
        for i, line in enumerate(table):
            for e in range(first[i], last[i]):
                if line[e] < 0:
                    line[e] = refs.index(0)
                    refs[line[e]] = 1
        source = s["rows"].tolist() if s["rows"] is not None else list(range(off[-1]))
        for layer in range(case["layers"]):
            for j, fresh in enumerate((s["k"][layer], s["v"][layer])):
                x = _heads_of(fresh, case["layout"])
                for i, line in enumerate(table):
                    for n in range(off[i], off[i + 1]):
                        place = lengths[i] + n - off[i]
                        pool[line[place // page], layer, j, :, place % page] = x[:, source[n]]
        return _ints(table), _ints(refs), pool
    if op == "fork":
        parents, rows, free = s["parents"].tolist(), s["rows"].tolist(), [p for p, r in enumerate(refs) if r == 0]
        new = []
        for i, p in enumerate(parents):
            if p == i:
                new.append(list(table[i]))
                continue
            line = [e if at < rows[i] // page else -1 for at, e in enumerate(table[p])]
            if rows[i] % page:
                line[rows[i] // page] = free.pop(0)
                pool[line[rows[i] // page]] = pool[table[p][rows[i] // page]]
            new.append(line)
        counts = [0] * len(refs)
        for line in new:
            for e in line:
                if e >= 0:
                    counts[e] += 1
        return _ints(new), _ints(counts), pool
    last = s["last"].tolist()
    for i, line in enumerate(table):
        for e in range(last[i]):
            if line[e] >= 0:
                refs[line[e]] -= 1
            line[e] = -1
    used = [p for p, r in enumerate(refs) if r > 0]
    moved = [p if r > 0 else -1 for p, r in enumerate(refs)]
    holes = [p for p in range(len(used)) if refs[p] == 0]
    for p, hole in zip([p for p in used if p >= len(used)], holes):
        moved[p], refs[hole], refs[p] = hole, refs[p], 0
        pool[hole] = pool[p]
    return _ints([[moved[e] if e >= 0 else -1 for e in line] for line in table]), _ints(refs), _ints(moved), pool
