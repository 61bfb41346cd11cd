"""Performance cases of a block's dense path: rotary positions with several axes, attention over whole rows under a
document or prefix mask, a score cap or a distance bias, and products of 4-bit microscaled operands.

The shapes are those of the two workloads that this repository measures: the 768p block (dim 5120, 40 heads, FFN
13,824, a 32 x 48 x 84 token grid) and the H3 block at 960 x 544 (dim 5376, 56 heads, FFN 14,336, a 37 x 17 x 30 grid,
435 text rows), and single images, short clips, packed batches of them and single rows of the same models. `draw` gives
more of the same ranges.
"""
import math
import sys
from pathlib import Path

import torch

own = False

DEV = "cuda"
MODELS = {  # dim, heads, ffn
    "768p": (5120, 40, 13824),
    "h3": (5376, 56, 14336),
}
BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
PAIRS = (16, 16, 16)             # rotary pairs of time, height and width: 96 rotating values a head
THETA = (10000.0, 10000.0, 10000.0)
STEP = (0.25, 1.0, 1.0)          # four latent frames to a unit of time
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


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
        # The cos / sin tables of a single 480 x 272 image (1 x 9 x 15 tokens and 77 text rows): the smallest call of a
        # generation, all latency.
        {"name": "table_image", "op": "table", "t": 1, "h": 9, "w": 15, "text": 77},
        # Head norms, rotary from positions and the head tiles of a single 960 x 544 image.
        {"name": "heads_image", "op": "heads", "model": "h3", "t": 1, "h": 17, "w": 30, "text": 435, "layout": "rows"},
        # The same of the whole 960 x 544 clip: the streaming case.
        {"name": "heads_960x544", "op": "heads", "model": "h3", "t": 37, "h": 17, "w": 30, "text": 435,
         "layout": "heads"},
        # Attention of a single 960 x 544 image, every row over every row.
        {"name": "attn_image", "op": "attn", "heads": 56, "kv_heads": 56, "docs": 1, "rows": 945, "queries": 0,
         "text": 435, "mask": "all", "cap": 0.0, "bias": False, "layout": "rows"},
        # The whole 960 x 544 clip without the sparse selection: the largest call.
        {"name": "attn_960x544", "op": "attn", "heads": 56, "kv_heads": 56, "docs": 1, "rows": 19305, "queries": 0,
         "text": 435, "mask": "all", "cap": 0.0, "bias": False, "layout": "heads"},
        # Five clips of uneven lengths packed into one batch, each attending itself, scores capped.
        {"name": "attn_packed_clips", "op": "attn", "heads": 40, "kv_heads": 40, "docs": 5, "rows": 14925,
         "queries": 0, "text": 435, "mask": "docs", "cap": 30.0, "bias": False, "layout": "rows"},
        # Two packed streams that generate frame after frame: the text is a prefix that every row sees, the rest is
        # causal; eight key heads are shared by the 40.
        {"name": "attn_prefix_causal", "op": "attn", "heads": 40, "kv_heads": 8, "docs": 2, "rows": 8191,
         "queries": 0, "text": 512, "mask": "prefix", "cap": 0.0, "bias": True, "layout": "heads"},
        # One new row a stream against three streams' kept rows (129,536 in all, the rows of the 768p batch).
        {"name": "attn_new_rows", "op": "attn", "heads": 40, "kv_heads": 8, "docs": 3, "rows": 129536, "queries": 1,
         "text": 512, "mask": "docs", "cap": 0.0, "bias": False, "layout": "heads"},
        # fc2 on three rows (one a modulation level), into the residual: the weights' bytes.
        {"name": "mx4_fc2_rows", "op": "mx4", "model": "768p", "layer": "fc2", "rows": 3},
        # The out projection of a short clip (5 x 17 x 30 tokens and 435 text rows), into the residual.
        {"name": "mx4_out_clip", "op": "mx4", "model": "h3", "layer": "out", "rows": 2985},
        # The QKV projection of a single 960 x 544 image (odd rows).
        {"name": "mx4_qkv_image", "op": "mx4", "model": "h3", "layer": "qkv", "rows": 945},
        # fc1 with SwiGLU of the 960 x 544 clip, the largest product of that block.
        {"name": "mx4_fc1_960x544", "op": "mx4", "model": "h3", "layer": "fc1", "rows": 19305},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["table", "heads", "heads", "attn", "attn", "attn", "mx4", "mx4", "mx4"])
    model = rng.choice(list(MODELS))
    if op in ("table", "heads"):
        t, h, w = rng.randint(1, 37), rng.randint(9, 17), rng.randint(15, 30)
        case = {"op": op, "t": t, "h": h, "w": w, "text": rng.randint(16, 435)}
        if op == "heads":
            case.update(model=model, layout=rng.choice(["heads", "rows"]))
        return case
    if op == "mx4":
        return {"op": op, "model": model, "layer": rng.choice(["qkv", "out", "fc1", "fc2"]),
                "rows": _log(rng, 1, 19305)}
    heads = rng.choice([7, 40, 56])
    case = {"op": op, "heads": heads, "kv_heads": rng.choice([heads, heads, 8 if heads > 7 else 1]),
            "docs": rng.randint(1, 5), "rows": 0, "queries": 0, "text": rng.randint(16, 512),
            "mask": rng.choice(["all", "docs", "prefix"]), "cap": rng.choice([0.0, 0.0, 30.0, 50.0]),
            "bias": rng.random() < 0.3, "layout": rng.choice(["heads", "rows"])}
    if rng.random() < 0.35:
        case.update(rows=_log(rng, 3000, 129536), queries=_log(rng, 1, 64), mask=rng.choice(["docs", "prefix"]))
    else:
        case["rows"] = _log(rng, 700, 16000)
    case["text"] = min(case["text"], case["rows"] // (4 * case["docs"]))
    return case


# ---- inputs ----------------------------------------------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(g, *shape, scale=1.0, dtype=BF16):
    return (torch.randn(shape, generator=g, device=DEV) * scale).to(dtype)


def _positions(case):
    """int32 [rows][3]: the text rows count along time, the video rows that follow lie on the grid behind them."""
    t, h, w = case["t"], case["h"], case["w"]
    text = torch.zeros((case["text"], 3), dtype=torch.int32, device=DEV)
    text[:, 0] = torch.arange(case["text"], device=DEV)
    grid = torch.stack(torch.meshgrid(torch.arange(t, device=DEV) + case["text"], torch.arange(h, device=DEV),
                                      torch.arange(w, device=DEV), indexing="ij"), -1).view(-1, 3)
    return torch.cat([text, grid.int()]).contiguous()


def _lengths(case):
    """The documents' key rows, uneven (1 : 2 : 3 ...), and their query rows: all of them, or `queries` new ones each."""
    n, rows = case["docs"], case["rows"]
    cuts = [rows * i * (i + 1) // (n * (n + 1)) for i in range(n + 1)]
    keys = [b - a for a, b in zip(cuts, cuts[1:])]
    return keys, [case["queries"] or k for k in keys]


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


def _to_mx4(x):
    """Rows to 4-bit floats in blocks of 32 columns that share a power of two, as they are kept: two values a byte, the
    first in its low half, and the blocks' exponent bytes eight columns of blocks at a time, [cols / 256][rows][8]."""
    rows, cols = x.shape
    b = x.float().view(rows, cols // 32, 32)
    top = b.abs().amax(-1)
    e = (torch.frexp(top).exponent - 3).clamp(-127, 127)
    e = torch.where(top > 0, e, -127)
    y = torch.ldexp(b, -e[..., None])
    a = y.abs()
    lim = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    a = (torch.round(a / lim) * lim).clamp(max=6.0)
    code = torch.where(a < 2, 2 * a, torch.where(a < 4, a + 2, a / 2 + 4)).to(torch.uint8)
    code = (code | (torch.signbit(y).to(torch.uint8) << 3)).view(rows, cols)
    packed = code[:, 0::2] | (code[:, 1::2] << 4)
    s = (e + 127).to(torch.uint8).view(rows, cols // 256, 8).transpose(0, 1).contiguous()
    return packed.contiguous(), s


def _from_mx4(packed, s, dtype=F32):
    """The values that _to_mx4's bytes stand for."""
    rows = packed.shape[0]
    code = torch.stack([packed & 15, packed >> 4], -1).view(rows, -1).long()
    table = torch.tensor(E2M1 + tuple(-v for v in E2M1), dtype=dtype, device=packed.device)
    e = s.transpose(0, 1).reshape(rows, -1, 1).int() - 127
    return torch.ldexp(table[code].view(rows, -1, 32), e).view(rows, -1)


def _layer(case):
    """Columns in and out of a layer's weight, and its rows (twice the columns out under SwiGLU)."""
    dim, heads, ffn = MODELS[case["model"]]
    k, n = {"qkv": (dim, 3 * heads * 128), "out": (heads * 128, dim), "fc1": (dim, ffn), "fc2": (ffn, dim)}[case["layer"]]
    return k, n, 2 * n if case["layer"] == "fc1" else n


def prepare(case, seed):
    g, op, s = _gen(seed), case["op"], {"case": case}
    if op in ("table", "heads"):
        s["pos"] = _positions(case) + torch.randint(0, 4096, (1, 3), generator=g, device=DEV, dtype=torch.int32)
    if op == "heads":
        heads = MODELS[case["model"]][1]
        s["qkv"] = _randn(g, s["pos"].shape[0], 3 * heads * 128)
        s["qw"], s["kw"] = (1 + 0.05 * torch.randn(128, generator=g, device=DEV) for _ in range(2))
    elif op == "attn":
        keys, queries = _lengths(case)
        mix = torch.randn((case["heads"], 8, 128), generator=g, device=DEV)
        share = case["heads"] // case["kv_heads"]
        q = _content(g, case["heads"], sum(queries), mix)
        k = _content(g, case["kv_heads"], sum(keys), mix[::share])
        v = _randn(g, case["kv_heads"], sum(keys), 128)
        s["q"], s["k"], s["v"] = (_rows_of(x, case["layout"]) for x in (q, k, v))
        s["q_off"], s["k_off"] = _offsets(queries), _offsets(keys)
        s["prefix"] = torch.full((case["docs"],), case["text"], dtype=torch.int32, device=DEV)
        # Slopes of a geometric row, and rows' places in time: 510 rows to a frame.
        s["slopes"] = 0.5 ** torch.linspace(1.0, 8.0, case["heads"], device=DEV)
        at = torch.arange(sum(keys), device=DEV, dtype=torch.int32)
        s["k_pos"] = at // 510
        s["q_pos"] = (s["k_off"][1:, None] - case["queries"] + at[:case["queries"]]).view(-1) // 510 \
            if case["queries"] else s["k_pos"].clone()
    elif op == "mx4":
        k, n, w_rows = _layer(case)
        s["x"] = _randn(g, case["rows"], k)
        s["w"], s["ws"] = _to_mx4(_randn(g, w_rows, k, scale=0.02))
        s["residual"] = _randn(g, case["rows"], n)
        s["gate"] = 0.1 * torch.randn(n, generator=g, device=DEV)
    return s


# ---- the plain forms -------------------------------------------------------------------------------------------------

def _plain_tables(pos):
    """cos and sin [rows][48], the angles in 64 bits: 32 lose a far position's."""
    angles = []
    for a, (pairs, theta, step) in enumerate(zip(PAIRS, THETA, STEP)):
        freq = theta ** (-torch.arange(pairs, dtype=F64, device=DEV) / pairs)
        angles.append(pos[:, a:a + 1].double() * (step * freq))
    angle = torch.cat(angles, 1)
    return torch.cos(angle).float(), torch.sin(angle).float()


def _plain_heads(s, layout):
    rows = s["pos"].shape[0]
    x = s["qkv"].view(rows, 3, -1, 128).float()
    cos, sin = (t[:, None] for t in _plain_tables(s["pos"]))

    def head(t, w):
        t = t * torch.rsqrt((t * t).mean(-1, keepdim=True) + 1e-6) * w
        a, b = t[..., :48], t[..., 48:96]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, t[..., 96:]], -1).to(BF16)

    out = head(x[:, 0], s["qw"]), head(x[:, 1], s["kw"]), s["qkv"].view(rows, 3, -1, 128)[:, 2]
    return tuple(t.transpose(0, 1).contiguous() if layout == "heads" else t.reshape(rows, -1) for t in out)


def _plain_ranges(s, case):
    """Each query row's keys [lo, hi): its document's, or of that the prefix and what lies before the row."""
    rows = int(s["q"].shape[1] if case["layout"] == "heads" else s["q"].shape[0])
    n_keys = int(s["k"].shape[1] if case["layout"] == "heads" else s["k"].shape[0])
    at = torch.arange(rows, device=DEV, dtype=torch.int32)
    if case["mask"] == "all":
        return torch.zeros_like(at), torch.full_like(at, n_keys)
    doc = torch.searchsorted(s["q_off"][1:].contiguous(), at, right=True)
    lo, end = s["k_off"][doc], s["k_off"][doc + 1]
    if case["mask"] == "docs":
        return lo, end
    own_key = at - s["q_off"][doc + 1] + end    # the last query row sits on the last key row
    return lo, torch.minimum(end, torch.maximum(own_key + 1, lo + s["prefix"][doc]))


def _plain_attention(s, case):
    q, k, v = (_heads_of(s[n], case["layout"]) for n in ("q", "k", "v"))
    lo, hi = _plain_ranges(s, case)
    share, n_keys = case["heads"] // case["kv_heads"], k.shape[1]
    at = torch.arange(n_keys, device=DEV, dtype=torch.int32)
    out = torch.empty(q.shape, dtype=BF16, device=DEV)
    # A few key heads at a time: the scores of all would not fit.
    step = max(1, (1 << 31) // (share * q.shape[1] * n_keys))
    masked = (at < lo[:, None]) | (at >= hi[:, None]) if case["mask"] != "all" else None
    for i in range(0, case["kv_heads"], step):
        heads = slice(i * share, min(i + step, case["kv_heads"]) * share)
        kt = k[i:i + step].float().transpose(1, 2).contiguous()
        x = q[heads].float().reshape(kt.shape[0], share * q.shape[1], 128)
        p = torch.bmm(x * (1 / math.sqrt(128)), kt).view(-1, q.shape[1], n_keys)
        if case["cap"]:
            p.div_(case["cap"]).tanh_().mul_(case["cap"])
        if case["bias"]:
            p.sub_(s["slopes"][heads, None, None] * (s["q_pos"][:, None] - s["k_pos"]).abs().float())
        if masked is not None:
            p.masked_fill_(masked, -math.inf)
        m = p.amax(-1, keepdim=True)
        p.sub_(m.masked_fill(m == -math.inf, 0.0)).exp_()
        total = p.sum(-1, keepdim=True)
        o = torch.bmm(p.view(kt.shape[0], -1, n_keys), v[i:i + step].float()).view(-1, q.shape[1], 128)
        out[heads] = (o / total.masked_fill(total == 0, 1.0)).to(BF16)
    return _rows_of(out, case["layout"])


def _plain_product(s, case):
    y = _from_mx4(*_to_mx4(s["x"])) @ _from_mx4(s["w"], s["ws"]).T
    if case["layer"] == "qkv":
        return y.to(BF16)
    if case["layer"] == "fc1":
        gate, up = y.chunk(2, dim=1)
        return (gate / (1 + torch.exp(-gate)) * up).to(BF16)
    return (s["residual"].float() + s["gate"] * y).to(BF16)


# ---- the calls -------------------------------------------------------------------------------------------------------

def _own_run(s, case):
    mh, op = _lib(), case["op"]
    if op == "table":
        return mh.rotary_axes(s["pos"], PAIRS, theta=THETA, step=STEP)
    if op == "heads":
        return mh.heads_partial_axes(s["qkv"], MODELS[case["model"]][1], s["pos"], PAIRS, s["qw"], s["kw"], theta=THETA,
                                     step=STEP, layout=case["layout"])
    if op == "attn":
        ranges = None
        if case["mask"] != "all":
            rows = s["q"].shape[1] if case["layout"] == "heads" else s["q"].shape[0]
            n_keys = s["k"].shape[1] if case["layout"] == "heads" else s["k"].shape[0]
            ranges = mh.attn_ranges(s["q_off"], s["k_off"], rows, n_keys,
                                    prefix=s["prefix"] if case["mask"] == "prefix" else None,
                                    causal=case["mask"] == "prefix")
        bias = {"slopes": s["slopes"], "q_pos": s["q_pos"], "k_pos": s["k_pos"]} if case["bias"] else {}
        return mh.flash_attn_128(s["q"], s["k"], s["v"], ranges=ranges, cap=case["cap"], layout=case["layout"], **bias)
    x, xs = mh.quant_rows_mx4(s["x"])
    if case["layer"] == "qkv":
        return mh.gemm_mx4(x, xs, s["w"], s["ws"])
    if case["layer"] == "fc1":
        return mh.gemm_mx4_swiglu(x, xs, s["w"], s["ws"])
    # The residual's first value stays with the caller (a step that is cached or guided reads it again).
    return mh.gemm_mx4_gate_add(x, xs, s["w"], s["ws"], s["residual"].clone(), s["gate"])


def run(s):
    case, op = s["case"], s["case"]["op"]
    if own:
        return _own_run(s, case)
    if op == "table":
        return _plain_tables(s["pos"])
    if op == "heads":
        return _plain_heads(s, case["layout"])
    if op == "attn":
        return _plain_attention(s, case)
    return _plain_product(s, case)


# ---- what a pass needs -----------------------------------------------------------------------------------------------

def _pairs(case):
    """Query and key pairs that the mask keeps."""
    keys, queries = _lengths(case)
    if case["mask"] == "all":
        return float(sum(keys)) * sum(queries)
    if case["mask"] == "docs":
        return float(sum(k * q for k, q in zip(keys, queries)))
    total = 0.0
    for k, q in zip(keys, queries):
        first, p = k - q + 1, min(case["text"], k)       # the first query row's causal keys; the prefix
        short = max(0, min(q, p - first))                # rows whose causal keys end inside the prefix
        total += short * p + (q - short) * (first + short + k) / 2
    return total


def work(case):
    op = case["op"]
    if op in ("table", "heads"):
        rows = case["t"] * case["h"] * case["w"] + case["text"]
        if op == "table":
            return {"bytes": rows * (12 + 48 * 8), "flops": 48.0 * 20 * rows}
        n = rows * 3 * MODELS[case["model"]][1] * 128
        return {"bytes": 4 * n + 12 * rows + 1024, "flops": 10.0 * n}
    if op == "attn":
        keys, queries = _lengths(case)
        return {"bytes": 512 * case["heads"] * sum(queries) + 512 * case["kv_heads"] * sum(keys),
                "flops": 512.0 * case["heads"] * _pairs(case)}
    k, n, w_rows = _layer(case)
    m = case["rows"]
    return {"bytes": 2 * m * k + w_rows * k * 17 // 32 + m * n * (4 if case["layer"] in ("out", "fc2") else 2),
            "flops": 2.0 * m * w_rows * k}


# ---- the same in 64 bits ---------------------------------------------------------------------------------------------

def _exact_turn(pos):
    """exp(i angle), complex [rows][48]."""
    parts = []
    for a in range(3):
        exponent = torch.arange(PAIRS[a], dtype=F64, device=DEV) * (-math.log(THETA[a]) / PAIRS[a])
        parts.append(torch.outer(pos[:, a].double() * STEP[a], torch.exp(exponent)))
    angle = torch.cat(parts, 1)
    return torch.polar(torch.ones_like(angle), angle)


def _exact_heads(s, case):
    rows = s["pos"].shape[0]
    turn = _exact_turn(s["pos"])
    q, k, v = s["qkv"].view(rows, 3, -1, 128).permute(1, 2, 0, 3).double()
    for t, w in ((q, s["qw"]), (k, s["kw"])):
        t /= torch.sqrt(t.square().mean(-1, keepdim=True) + 1e-6)
        t *= w.double()
        z = torch.complex(t[..., :48].contiguous(), t[..., 48:96].contiguous()) * turn
        t[..., :48], t[..., 48:96] = z.real, z.imag
    return tuple(_rows_of(t.contiguous(), case["layout"]) for t in (q, k, v))


def _exact_attention(s, case):
    q, k, v = (_heads_of(s[n], case["layout"]).double() for n in ("q", "k", "v"))
    share, out = case["heads"] // case["kv_heads"], torch.zeros(q.shape, dtype=F64, device=DEV)
    keys, queries = _lengths(case)
    spans = [(0, sum(queries), 0, sum(keys))]
    if case["mask"] != "all":
        spans = [(sum(queries[:d]), sum(queries[:d + 1]), sum(keys[:d]), sum(keys[:d + 1])) for d in range(case["docs"])]
    for h in range(case["heads"]):
        for q0, q1, k0, k1 in spans:
            score = q[h, q0:q1] @ k[h // share, k0:k1].T.contiguous() / math.sqrt(128)
            if case["cap"]:
                score = case["cap"] * torch.tanh(score / case["cap"])
            if case["bias"]:
                gap = s["q_pos"][q0:q1, None].double() - s["k_pos"][k0:k1].double()
                score = score - s["slopes"][h].double() * gap.abs()
            if case["mask"] == "prefix":
                seen = torch.ones_like(score, dtype=torch.bool).tril((k1 - k0) - (q1 - q0))
                seen[:, :case["text"]] = True
                score = torch.where(seen, score, -math.inf)
            out[h, q0:q1] = torch.softmax(score, -1) @ v[h // share, k0:k1]
    return _rows_of(out, case["layout"])


def _exact_blocks(x):
    """x as its 4-bit blocks stand for it: the nearest of the eight magnitudes, ties to the even code."""
    rows, cols = x.shape
    b = x.double().view(rows, -1, 32)
    scale = torch.exp2(torch.floor(torch.log2(b.abs().amax(-1, keepdim=True))) - 2)
    mags = torch.tensor(E2M1, dtype=F64, device=DEV)
    mids = (mags[1:] + mags[:-1]) / 2
    a = (b / scale).abs()
    below, above = torch.searchsorted(mids, a), torch.searchsorted(mids, a, right=True)
    code = torch.where(below % 2 == 0, below, above)     # they differ at a midpoint: the even one of the two
    return (torch.sign(b) * mags[code] * scale).view(rows, cols)


def _exact_product(s, case):
    w = _from_mx4(s["w"], s["ws"], F64)
    y = _exact_blocks(s["x"]) @ w.T.contiguous()
    if case["layer"] == "qkv":
        return y
    if case["layer"] == "fc1":
        n = y.shape[1] // 2
        return torch.sigmoid(y[:, :n]) * y[:, :n] * y[:, n:]
    return s["residual"].double() + s["gate"].double() * y


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "table":
        turn = _exact_turn(s["pos"])
        return turn.real.contiguous(), turn.imag.contiguous()
    if case["op"] == "heads":
        return _exact_heads(s, case)
    if case["op"] == "attn":
        return _exact_attention(s, case)
    return _exact_product(s, case)
