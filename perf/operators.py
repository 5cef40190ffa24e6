"""Performance cases of the grouped-query operators around `flash_forward`: rotary positions with several axes, the 8-bit
paged cache with the attention that reads it, and cross attention to an encoder's states.

A case is a dict of plain values.  `listed()` gives the fixed ones, `draw(rng)` one more of the same ranges, `prepare` what
a program holds before the call, `run` one pass (with `own` the calls of `dscuda_b200.flash`, else the plain form in
elementary torch operations in 32 bits), `exact` the same results from the definitions in 64 bits, `work` the bytes and
operations the pass cannot do without.

Operations:

    rope          rotary positions with several axes (time, height, width) on queries and keys, or on their gradients
    append        new tokens' keys and values into the paged 8-bit cache, one scale for each page and head
    decode        attention of the newest tokens over that cache
    step          the three in a row, as one layer of a decode step makes them
    cross         attention to an encoder's states of another length, forward
    cross_train   the same with its gradients

Lengths of ragged cases belong to the case (`layout` seeds them); all values come from the seed given to `prepare`.
"""
import math
import random

import torch

own = False

WIDTH = 128                     # columns of a head
SCALE = WIDTH ** -0.5
TINY = 2.0 ** -100              # a page whose largest value is below this is stored as zeros
LARGEST = {"int8": 127.0, "e4m3": 448.0}
DTYPES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}


# ---- the cases ---------------------------------------------------------------------------------------------------------

def listed():
    return [
        # a decode step of sixteen conversations: launch latency
        {"name": "rope_step", "op": "rope", "rows": 16, "heads": 32, "kv_heads": 8, "width": 128, "sections": "16,24,24", "restart": False, "inverse": False, "fused": True},
        # prompts with video frames, straight from the fused projection
        {"name": "rope_video", "op": "rope", "rows": 16384, "heads": 32, "kv_heads": 8, "width": 128, "sections": "16,24,24", "restart": False, "inverse": False, "fused": True},
        # gradients in an image encoder with two axes of their own frequencies; five images of 37 x 37 patches
        {"name": "rope_image_gradient", "op": "rope", "rows": 6845, "heads": 16, "kv_heads": 16, "width": 64, "sections": "16,16", "restart": True, "inverse": True, "fused": False},
        # one new token for each of 64 conversations, most of them in the middle of a page
        {"name": "append_step", "op": "append", "batch": 64, "tokens": 1, "kv_heads": 8, "page": 64, "low": 0, "high": 4000, "ragged": False, "kind": "int8", "layout": 1},
        # four uneven prompts
        {"name": "append_prompts", "op": "append", "batch": 4, "tokens": 4096, "kv_heads": 8, "page": 64, "low": 0, "high": 0, "ragged": True, "kind": "e4m3", "layout": 2},
        # one user, a short conversation: latency of the whole call
        {"name": "decode_one_short", "op": "decode", "batch": 1, "tokens": 1, "heads": 32, "kv_heads": 8, "page": 64, "low": 700, "high": 700, "kind": "int8", "layout": 3},
        # a loaded server with conversations of very uneven lengths
        {"name": "decode_ragged", "op": "decode", "batch": 32, "tokens": 1, "heads": 32, "kv_heads": 8, "page": 64, "low": 1, "high": 8192, "kind": "int8", "layout": 4},
        # four drafted tokens checked at once over long documents
        {"name": "decode_draft_long", "op": "decode", "batch": 8, "tokens": 4, "heads": 64, "kv_heads": 8, "page": 128, "low": 20000, "high": 40000, "kind": "e4m3", "layout": 5},
        # one layer of a decode step: rotary positions, append, attention
        {"name": "step_layer", "op": "step", "batch": 16, "tokens": 1, "heads": 32, "kv_heads": 8, "page": 64, "low": 500, "high": 4000, "kind": "int8", "layout": 6},
        # a decoder's next token over an encoder's states, padded to the longest
        {"name": "cross_step", "op": "cross", "batch": 16, "tokens": 1, "keys": 1500, "low": 300, "heads": 32, "kv_heads": 8, "layout": 7},
        # a small training step with odd lengths, three query heads to a key head and an entry without any states
        {"name": "cross_train_small", "op": "cross_train", "batch": 3, "tokens": 77, "keys": 333, "low": 0, "heads": 6, "kv_heads": 2, "layout": 8},
        # a training step of a text decoder over long image or audio sequences
        {"name": "cross_train_long", "op": "cross_train", "batch": 4, "tokens": 2048, "keys": 4096, "low": 2048, "heads": 32, "kv_heads": 8, "layout": 9},
    ]


def _log_uniform(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _split(rng, total, parts):
    """`total` as `parts` positive numbers."""
    cuts = sorted(rng.sample(range(1, total), parts - 1))
    return [b - a for a, b in zip([0] + cuts, cuts + [total])]


def draw(rng):
    op = rng.choice(("rope", "rope", "append", "append", "decode", "decode", "decode", "step", "cross", "cross", "cross_train", "cross_train"))
    heads, kv_heads = rng.choice(((32, 8), (32, 8), (64, 8), (16, 16), (8, 1), (16, 2), (6, 2), (5, 5), (28, 4), (12, 12)))
    layout = rng.randint(1, 1 << 20)
    while True:
        if op == "rope":
            width = rng.choice((64, 128, 128))
            case = {"op": op, "rows": _log_uniform(rng, 1, 16384), "heads": heads, "kv_heads": kv_heads, "width": width,
                    "sections": ",".join(map(str, _split(rng, width // 2, rng.choice((1, 2, 3, 3, 4))))), "restart": rng.random() < 0.4,
                    "inverse": rng.random() < 0.4, "fused": rng.random() < 0.5}
        elif op == "append":
            high = rng.choice((0, 1, _log_uniform(rng, 1, 8192)))
            case = {"op": op, "batch": _log_uniform(rng, 1, 64), "tokens": _log_uniform(rng, 1, 4096), "kv_heads": kv_heads, "page": rng.choice((16, 32, 64, 128)),
                    "low": min(high, 3), "high": high, "ragged": rng.random() < 0.5, "kind": rng.choice(("int8", "e4m3")), "layout": layout}
        elif op in ("decode", "step"):
            tokens = rng.choice((1, 1, 1, 2, 4, rng.randint(1, 8)))
            high = max(tokens, _log_uniform(rng, 1, 40000))
            case = {"op": op, "batch": _log_uniform(rng, 1, 64), "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "page": rng.choice((16, 32, 64, 64, 128)),
                    "low": max(tokens, _log_uniform(rng, max(1, high // 64), high)), "high": high, "kind": rng.choice(("int8", "e4m3")), "layout": layout}
            case["low"] = min(case["low"], high)
        else:
            keys = _log_uniform(rng, 1, 8192)
            case = {"op": op, "batch": _log_uniform(rng, 1, 16), "tokens": rng.choice((1, _log_uniform(rng, 1, 64), _log_uniform(rng, 1, 4096))) if op == "cross" else _log_uniform(rng, 1, 4096),
                    "keys": keys, "low": rng.choice((0, keys // 2, keys)), "heads": heads, "kv_heads": kv_heads, "layout": layout}
        # nothing dearer than the dearest listed case of its kind
        w = work(case)
        most = {"rope": 3.4e8, "append": 1.05e8, "decode": 5.0e8, "step": 5.0e8}.get(op, 3e8)
        pairs = case["batch"] * case["heads"] * case["tokens"] * case["keys"] if op.startswith("cross") else 0
        if w["bytes"] <= most and w["flops"] <= 1.5e12 and pairs <= 1.1e9:
            return case


def _lengths(case):
    """Tokens each sequence has: before the append, or in all for an attention."""
    rng = random.Random(case["layout"])
    if case["op"].startswith("cross"):
        lengths = [rng.randint(case["low"], case["keys"]) for _ in range(case["batch"])]
        if case["low"] == 0 and case["batch"] > 1:
            lengths[rng.randrange(case["batch"])] = 0
        return lengths
    return [rng.randint(case["low"], case["high"]) for _ in range(case["batch"])]


def _counts(case):
    """New tokens of each sequence of an append."""
    rng = random.Random(case["layout"] + 1)
    return [rng.randint(max(1, case["tokens"] // 2), case["tokens"]) if case["ragged"] else case["tokens"] for _ in range(case["batch"])]


# ---- what a program has in hand --------------------------------------------------------------------------------------------

def _fused(rows, heads, kv_heads, width, values, normal):
    """Queries, keys and (with `values`) values as the views of one projection's output that they are."""
    total = (heads + (2 if values else 1) * kv_heads) * width
    out = normal(*rows, total)
    parts = torch.split(out, [heads * width, kv_heads * width] + ([kv_heads * width] if values else []), dim=-1)
    return [p.view(*rows, -1, width) for p in parts]


def _positions(case, rows, generator):
    """Axes of a prompt with frames: time, then places inside a frame; int32 [axes, rows]."""
    axes = len(case["sections"].split(","))
    high = torch.tensor([32768] + [64] * (axes - 1), device="cuda")[:, None]
    return (torch.rand(axes, rows, device="cuda", generator=generator, dtype=torch.float64) * high).int().contiguous()


def _pages(lengths, page, generator):
    """Block table cut from one random permutation of all pages and a few more, and the number of pages."""
    need = [-(-n // page) for n in lengths]
    order = torch.randperm(sum(need) + 3, generator=generator, device="cuda").to(torch.int32)
    table = torch.zeros(len(lengths), max(max(need), 1), dtype=torch.int32, device="cuda")
    start = 0
    for b, n in enumerate(need):
        table[b, :n] = order[start:start + n]
        start += n
    return table, sum(need) + 3


def _cache(case, blocks, generator):
    """A filled cache: codes that use the range of their type, scales of keys and values as a model has them."""
    shape = (blocks, case["kv_heads"], case["page"], WIDTH)
    kind = case["kind"]
    caches = []
    for _ in range(2):
        x = torch.randn(shape, device="cuda", generator=generator, dtype=torch.float32).mul_(LARGEST[kind] / 4.0).clamp_(-LARGEST[kind], LARGEST[kind])
        caches.append(x.round_().to(torch.int8) if kind == "int8" else x.to(torch.float8_e4m3fn))
    scales = [(torch.randn(blocks, case["kv_heads"], device="cuda", generator=generator).mul_(0.2).exp_() * (4.0 / LARGEST[kind])).contiguous() for _ in range(2)]
    return caches[0], caches[1], scales[0], scales[1]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))

    def normal(*shape, std=1.0):
        return torch.randn(*shape, device="cuda", generator=g, dtype=torch.float32).mul_(std).bfloat16()

    def ints(values):
        return torch.tensor(values, dtype=torch.int32, device="cuda")

    op, s = case["op"], {"case": case}
    if op == "rope":
        s["sections"] = [int(x) for x in case["sections"].split(",")]
        s["positions"] = _positions(case, case["rows"], g)
        if case["fused"]:
            s["query"], s["key"] = _fused((case["rows"],), case["heads"], case["kv_heads"], case["width"], True, normal)[:2]
        else:
            s["query"], s["key"] = normal(case["rows"], case["heads"], case["width"]), normal(case["rows"], case["kv_heads"], case["width"])
    elif op == "append":
        starts, counts = _lengths(case), _counts(case)
        s["table"], blocks = _pages([a + n for a, n in zip(starts, counts)], case["page"], g)
        s["cache"] = _cache(case, blocks, g)
        s["starts"], s["counts"] = ints(starts), ints(counts) if case["ragged"] else None
        s["key"], s["value"] = (normal(case["batch"], case["tokens"], case["kv_heads"], WIDTH, std=1.5) for _ in range(2))
    elif op in ("decode", "step"):
        lengths = _lengths(case)
        s["table"], blocks = _pages(lengths, case["page"], g)
        s["cache"] = _cache(case, blocks, g)
        s["lengths"] = ints(lengths)
        rows = (case["batch"], case["tokens"])
        if op == "decode":
            s["query"] = normal(*rows, case["heads"], WIDTH)
        else:
            s["query"], s["key"], s["value"] = _fused(rows, case["heads"], case["kv_heads"], WIDTH, True, normal)
            s["starts"] = ints([n - case["tokens"] for n in lengths])
            s["sections"] = [16, 24, 24]
            # plain text: the same position on every axis
            s["positions"] = (s["starts"][:, None] + torch.arange(case["tokens"], device="cuda", dtype=torch.int32)).reshape(1, -1).repeat(3, 1).contiguous()
    else:
        b = case["batch"]
        s["query"] = normal(b, case["tokens"], case["heads"], WIDTH)
        s["key"], s["value"] = (normal(b, case["keys"], case["kv_heads"], WIDTH) for _ in range(2))
        s["lengths"] = ints(_lengths(case))
        if op == "cross_train":
            s["dout"] = normal(b, case["tokens"], case["heads"], WIDTH, std=0.1)
    return s


# ---- one pass --------------------------------------------------------------------------------------------------------------

def run(s):
    case = s["case"]
    return {"rope": _run_rope, "append": _run_append, "decode": _run_decode, "step": _run_step, "cross": _run_cross, "cross_train": _run_cross_train}[case["op"]](s, case)


def _run_rope(s, case):
    if own:
        from dscuda_b200 import flash
        return flash.rope(s["query"], s["key"], s["positions"], s["sections"], restart=case["restart"], inverse=case["inverse"])
    cos, sin = _plain_angles(s["positions"], s["sections"], case["restart"], case["inverse"])
    return _plain_rotate(s["query"], cos, sin), _plain_rotate(s["key"], cos, sin)


def _run_append(s, case):
    if own:
        from dscuda_b200 import flash
        flash.cache_append(*s["cache"], s["key"], s["value"], s["table"], s["starts"], s["counts"])
    else:
        _plain_append(case, s["cache"][0], s["cache"][2], s["key"], s["table"], s["starts"], s["counts"])
        _plain_append(case, s["cache"][1], s["cache"][3], s["value"], s["table"], s["starts"], s["counts"])
    return s["cache"]


def _run_decode(s, case):
    if own:
        from dscuda_b200 import flash
        return flash.decode(s["query"], *s["cache"], s["table"], s["lengths"], SCALE)
    return _plain_decode(case, s["query"], s["cache"], s["table"], s["lengths"])


def _run_step(s, case):
    b, t = case["batch"], case["tokens"]
    if own:
        from dscuda_b200 import flash
        query, key = flash.rope(s["query"], s["key"], s["positions"], s["sections"])
        flash.cache_append(*s["cache"], key, s["value"], s["table"], s["starts"])
        output, lse = flash.decode(query, *s["cache"], s["table"], s["lengths"], SCALE)
        return output, lse, *s["cache"]
    cos, sin = _plain_angles(s["positions"], s["sections"], False, False)
    query, key = (_plain_rotate(x.reshape(b * t, -1, WIDTH), cos, sin).view(b, t, -1, WIDTH) for x in (s["query"], s["key"]))
    _plain_append(case, s["cache"][0], s["cache"][2], key, s["table"], s["starts"], None)
    _plain_append(case, s["cache"][1], s["cache"][3], s["value"], s["table"], s["starts"], None)
    output, lse = _plain_decode(case, query, s["cache"], s["table"], s["lengths"])
    return output, lse, *s["cache"]


def _run_cross(s, case):
    if own:
        from dscuda_b200 import flash
        return flash.cross_forward(s["query"], s["key"], s["value"], SCALE, s["lengths"])
    output, lse, _ = _plain_cross(s["query"], s["key"], s["value"], s["lengths"])
    return output.bfloat16(), lse


def _run_cross_train(s, case):
    if own:
        from dscuda_b200 import flash
        output, lse = flash.cross_forward(s["query"], s["key"], s["value"], SCALE, s["lengths"])
        return output, lse, *flash.cross_backward(s["dout"], output, lse, s["query"], s["key"], s["value"], SCALE, s["lengths"])
    output, lse, probs = _plain_cross(s["query"], s["key"], s["value"], s["lengths"])
    return output.bfloat16(), lse, *_plain_cross_gradients(s["dout"], output, probs, s["query"], s["key"], s["value"])


# ---- the plain forms -------------------------------------------------------------------------------------------------------

def _plain_angles(positions, sections, restart, inverse):
    """cos and sin [rows, 1, width / 2] of every pair; the angles in 64 bits, as positions reach far."""
    counts = torch.tensor(sections)
    axis = torch.repeat_interleave(torch.arange(len(sections)), counts)
    index = torch.arange(len(axis))
    exponent = (index - (torch.cumsum(counts, 0) - counts)[axis]).double() / counts[axis] if restart else index.double() / len(axis)
    angle = positions.double().t()[:, axis.to(positions.device)] * torch.pow(10000.0, -exponent).to(positions.device)
    angle = -angle if inverse else angle
    return angle.cos().float()[:, None], angle.sin().float()[:, None]


def _plain_rotate(x, cos, sin):
    a, b = x.float().chunk(2, -1)
    return torch.cat([a * cos - b * sin, a * sin + b * cos], -1).bfloat16()


def _plain_append(case, cache, scales, x, table, starts, counts):
    """Every page that gets new tokens takes the scale that its old and new values need together."""
    page, kind = case["page"], case["kind"]
    b, t = x.shape[:2]
    pages = min(table.shape[1], (t + page - 1) // page + 1)
    first = starts // page                                                          # first logical page that is written
    slot = (first[:, None] * page + torch.arange(pages * page, device=x.device) - starts[:, None]).view(b, pages, page)    # new token in each slot
    fresh = (slot >= 0) & (slot < (t if counts is None else counts[:, None, None]))
    touched = fresh.any(-1)
    logical = (first[:, None] + torch.arange(pages, device=x.device)).clamp(max=table.shape[1] - 1)
    physical = torch.gather(table, 1, logical.long()).long()                          # [b, pages]
    rows = torch.gather(x.float().flatten(2), 1, slot.clamp(0, t - 1).view(b, -1, 1).expand(-1, -1, x.shape[2] * WIDTH).long())
    rows = (rows.view(b, pages, page, -1, WIDTH) * fresh[..., None, None]).transpose(2, 3)            # [b, pages, heads, page, width]
    amax = rows.abs().amax((-1, -2))
    needed = torch.where(amax < TINY, torch.zeros_like(amax), amax / LARGEST[kind])
    old = torch.where((slot[..., 0] < 0)[..., None], scales[physical], torch.zeros_like(needed))      # a page that starts here has none
    new = torch.maximum(old, needed)
    inverse = torch.where(new > 0, 1.0 / new, torch.zeros_like(new))
    codes = (rows * inverse[..., None, None])
    kept = cache[physical].float()
    moved = kept * torch.where(new > old, old * inverse, torch.ones_like(new))[..., None, None]
    codes = torch.where(fresh[:, :, None, :, None], codes, torch.where((slot < 0)[:, :, None, :, None], moved, kept))
    codes = codes.round().clamp(-LARGEST[kind], LARGEST[kind]) if kind == "int8" else codes.clamp(-LARGEST[kind], LARGEST[kind])
    at = touched.nonzero(as_tuple=True)
    cache.view(torch.int8)[physical[at]] = codes[at].to(DTYPES[kind]).view(torch.int8)
    scales[physical[at]] = new[at]


def _plain_softmax(scores):
    """Softmax over the last axis, its sum's logarithm; a row without any key gives zeros and -inf."""
    top = scores.amax(-1, keepdim=True)
    weights = torch.exp(scores - torch.where(torch.isfinite(top), top, torch.zeros_like(top)))
    total = weights.sum(-1, keepdim=True)
    return torch.where(total > 0, weights / total, torch.zeros_like(weights)), (torch.log(total) + top).squeeze(-1)


def _plain_decode(case, query, cache, table, lengths):
    b, t, hq, _ = query.shape
    hkv, page = case["kv_heads"], case["page"]
    keys, values = ((c[table.long()].float() * s[table.long()][..., None, None]).transpose(1, 2).reshape(b, hkv, -1, WIDTH) for c, s in ((cache[0], cache[2]), (cache[1], cache[3])))
    rows = query.float().view(b, t, hkv, hq // hkv, WIDTH).permute(0, 2, 3, 1, 4).reshape(b, hkv, -1, WIDTH)
    scores = (rows @ keys.transpose(-1, -2) * SCALE).view(b, hkv, -1, t, keys.shape[2])
    limit = lengths[:, None] - t + 1 + torch.arange(t, device=query.device)             # keys that each new token sees
    scores = scores.masked_fill(torch.arange(keys.shape[2], device=query.device) >= limit[:, None, None, :, None], -math.inf)
    probs, lse = _plain_softmax(scores)
    out = probs.view(b, hkv, -1, keys.shape[2]) @ values
    return out.view(b, hkv, -1, t, WIDTH).permute(0, 3, 1, 2, 4).reshape(b, t, hq, WIDTH).bfloat16(), lse.reshape(b, hq, t)


def _by_kv_head(x, kv_heads):
    """[b, t, heads, width] -> [b, kv_heads, group * t, width] in 32 bits."""
    b, t, h, _ = x.shape
    return x.float().view(b, t, kv_heads, h // kv_heads, WIDTH).permute(0, 2, 3, 1, 4).reshape(b, kv_heads, -1, WIDTH)


def _by_token(x, tokens):
    b, kv_heads, rows, _ = x.shape
    return x.view(b, kv_heads, rows // tokens, tokens, WIDTH).permute(0, 3, 1, 2, 4).reshape(b, tokens, -1, WIDTH)


def _plain_cross(query, key, value, lengths):
    b, t, hq, _ = query.shape
    hkv = key.shape[2]
    scores = _by_kv_head(query, hkv) @ key.float().permute(0, 2, 3, 1) * SCALE
    scores = scores.masked_fill(torch.arange(key.shape[1], device=query.device) >= lengths[:, None, None, None], -math.inf)
    probs, lse = _plain_softmax(scores)
    return _by_token(probs @ value.float().transpose(1, 2), t), lse.reshape(b, hq, t), probs


def _plain_cross_gradients(dout, output, probs, query, key, value):
    hkv, t = key.shape[2], query.shape[1]
    grad = _by_kv_head(dout, hkv)
    dv = probs.transpose(-1, -2) @ grad
    delta = (grad * _by_kv_head(output, hkv)).sum(-1, keepdim=True)
    dscores = probs * (grad @ value.float().permute(0, 2, 3, 1) - delta) * SCALE
    dq = _by_token(dscores @ key.float().transpose(1, 2), t)
    dk = dscores.transpose(-1, -2) @ _by_kv_head(query, hkv)
    return dq.bfloat16(), dk.transpose(1, 2).bfloat16(), dv.transpose(1, 2).bfloat16()


# ---- the definitions in 64 bits --------------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {"rope": _exact_rope, "append": _exact_append, "decode": _exact_decode, "step": _exact_step, "cross": _exact_cross, "cross_train": _exact_cross}[case["op"]](s, case)


def _turn(x, positions, sections, restart, inverse):
    """Each pair (i, i + width / 2) as a complex number, turned by its angle."""
    half = x.shape[-1] // 2
    frequency, axis = [], []
    for a, n in enumerate(sections):
        for j in range(n):
            frequency.append(10000.0 ** -(j / n if restart else len(frequency) / half))
            axis.append(a)
    angle = positions[torch.tensor(axis, device=x.device)].double().t() * torch.tensor(frequency, dtype=torch.float64, device=x.device)
    pairs = torch.complex(x[..., :half].double(), x[..., half:].double())
    turned = pairs * torch.polar(torch.ones_like(angle), -angle if inverse else angle)[:, None, :]
    return torch.cat([turned.real, turned.imag], -1)


def _exact_rope(s, case):
    return tuple(_turn(s[x], s["positions"], s["sections"], case["restart"], case["inverse"]) for x in ("query", "key"))


def _exact_pages(case, cache, scales, x, s, counts):
    """The append page by page: (codes, scales) of the whole cache in 64 bits."""
    page, top = case["page"], LARGEST[case["kind"]]
    codes, scales, x = cache.double(), scales.double(), x.double()
    table, starts = s["table"].tolist(), s["starts"].tolist()
    for b, (start, count) in enumerate(zip(starts, counts)):
        for logical in range(start // page, -(-(start + count) // page)):
            begin, end = max(start, logical * page), min(start + count, (logical + 1) * page)
            at, slot = table[b][logical], begin - logical * page
            rows = x[b, begin - start:end - start].transpose(0, 1)                     # [heads, tokens, width]
            need = rows.abs().amax((1, 2)) / top
            old = scales[at] if slot > 0 else torch.zeros_like(need)
            new = torch.maximum(old, need)
            if slot > 0:
                codes[at, :, :slot] *= (old / new)[:, None, None]
            codes[at, :, slot:slot + end - begin] = rows / new[:, None, None]
            codes[at] = _held(codes[at], case["kind"])
            scales[at] = new
    return codes, scales


def _held(x, kind):
    return x.round() if kind == "int8" else x.to(torch.float8_e4m3fn).double()


def _exact_append(s, case):
    k, v = (_exact_pages(case, s["cache"][i], s["cache"][2 + i], s[n], s, _counts(case)) for i, n in enumerate(("key", "value")))
    floats = case["kind"] == "e4m3"
    return k[0] if floats else None, v[0] if floats else None, k[1], v[1]


def _attend(query, keys, values, limits):
    """One sequence: query [t, hq, width], keys and values [n, hkv, width] in 64 bits, limits [t] -> output, lse [hq, t]."""
    t, hq, _ = query.shape
    hkv = keys.shape[1]
    out, lse = torch.zeros(t, hq, WIDTH, dtype=torch.float64, device=query.device), torch.full((hq, t), -math.inf, dtype=torch.float64, device=query.device)
    seen = torch.arange(keys.shape[0], device=query.device)[None, :] < limits[:, None]
    for h in range(hq):
        if not keys.shape[0]:
            break
        scores = torch.where(seen, query[:, h].double() @ keys[:, h // (hq // hkv)].t() * SCALE, -math.inf)
        lse[h] = torch.logsumexp(scores, -1)
        out[:, h] = torch.where(torch.isfinite(lse[h])[:, None], torch.exp(scores - lse[h][:, None]), 0.0) @ values[:, h // (hq // hkv)]
    return out, lse


def _exact_over_cache(case, query, codes, s):
    outs, lses = [], []
    for b, n in enumerate(s["lengths"].tolist()):
        at = s["table"][b, :-(-n // case["page"])].long()
        keys, values = ((codes[i][at].double() * codes[2 + i][at].double()[:, :, None, None]).transpose(1, 2).reshape(-1, case["kv_heads"], WIDTH)[:n] for i in range(2))
        limits = n - case["tokens"] + 1 + torch.arange(case["tokens"], device=query.device)
        o, l = _attend(query[b], keys, values, limits)
        outs.append(o)
        lses.append(l)
    return torch.stack(outs), torch.stack(lses)


def _exact_decode(s, case):
    return _exact_over_cache(case, s["query"], s["cache"], s)


def _exact_step(s, case):
    b, t = case["batch"], case["tokens"]
    query, key = (_turn(s[x].reshape(b * t, -1, WIDTH), s["positions"], s["sections"], False, False).view(b, t, -1, WIDTH).bfloat16() for x in ("query", "key"))
    k, v = (_exact_pages(case, s["cache"][i], s["cache"][2 + i], x, s, [t] * b) for i, x in enumerate((key, s["value"])))
    out, lse = _exact_over_cache(case, query, (k[0], v[0], k[1], v[1]), s)
    return out, lse, None, None, k[1], v[1]


def _exact_cross(s, case):
    train = case["op"] == "cross_train"
    hq, hkv, t = case["heads"], case["kv_heads"], case["tokens"]
    outs = [torch.zeros_like(s["query"], dtype=torch.float64), torch.full((case["batch"], hq, t), -math.inf, dtype=torch.float64, device="cuda")]
    outs += [torch.zeros_like(s[n], dtype=torch.float64) for n in ("query", "key", "value")] if train else []
    for b, n in enumerate(s["lengths"].tolist()):
        for h in range(hq if n else 0):
            g = h // (hq // hkv)
            q, k, v = s["query"][b, :, h].double(), s["key"][b, :n, g].double(), s["value"][b, :n, g].double()
            scores = q @ k.t() * SCALE
            outs[1][b, h] = torch.logsumexp(scores, -1)
            p = torch.softmax(scores, -1)
            outs[0][b, :, h] = p @ v
            if train:
                do = s["dout"][b, :, h].double()
                dp = do @ v.t()
                ds = p * (dp - (p * dp).sum(-1, keepdim=True)) * SCALE
                outs[2][b, :, h] = ds @ k
                outs[3][b, :n, g] += ds.t() @ q
                outs[4][b, :n, g] += p.t() @ do
    return tuple(outs)


# ---- what a pass cannot do without -----------------------------------------------------------------------------------------

def _pages_touched(start, count, page):
    return -(-(start + count) // page) - start // page


def work(case):
    op = case["op"]
    row = WIDTH * 2                                                     # bytes of a head's row in bf16
    if op == "rope":
        values = case["rows"] * (case["heads"] + case["kv_heads"]) * case["width"]
        return {"bytes": 4 * values + 4 * case["rows"] * len(case["sections"].split(",")), "flops": 3 * values}
    if op == "append":
        new = list(zip(_lengths(case), _counts(case)))
        tokens, pages = sum(n for _, n in new), sum(_pages_touched(a, n, case["page"]) for a, n in new)
        return {"bytes": case["kv_heads"] * (tokens * 2 * (row + WIDTH) + pages * 2 * 8) + pages * 4 + case["batch"] * 8, "flops": tokens * case["kv_heads"] * WIDTH * 2 * 3}
    if op in ("decode", "step"):
        lengths = _lengths(case)
        seen = sum(max(0, n - j) for n in lengths for j in range(case["tokens"]))
        pages = sum(-(-n // case["page"]) for n in lengths)
        queries = case["batch"] * case["tokens"] * case["heads"]
        n_bytes = sum(lengths) * case["kv_heads"] * 2 * WIDTH + pages * (case["kv_heads"] * 8 + 4) + queries * (2 * row + 4)
        if op == "step":
            new = case["batch"] * case["tokens"]
            n_bytes += new * (case["heads"] * 2 * row + case["kv_heads"] * (3 * row + 2 * WIDTH) + 12)
        return {"bytes": n_bytes, "flops": 4 * WIDTH * case["heads"] * seen}
    keys = sum(_lengths(case))
    pairs = case["heads"] * case["tokens"] * keys
    rows, states = case["batch"] * case["tokens"] * case["heads"], keys * case["kv_heads"]
    if op == "cross":
        return {"bytes": rows * (2 * row + 4) + states * 2 * row, "flops": 4 * WIDTH * pairs}
    padded = case["batch"] * case["keys"] * case["kv_heads"]
    return {"bytes": rows * (4 * row + 4) + states * 2 * row + padded * 2 * row, "flops": (4 + 10) * WIDTH * pairs}
