"""Workloads of the frame-attention operators: rotary positions over (time, height, width) written
into a paged cache, attention of new tokens over that cache, and the choice of the cache slots that
give way to new tokens by accumulated attention weight.

A video network keeps one token per position of its feature map (7 x 7, 14 x 14, 17 x 30, 34 x 60 for
the maps of the networks in this repository at 224 x 224 and 544 x 960) and attends over the tokens
of the last frames of its stream.  With ``own`` false every operator is computed from elementary
torch operations in 32 bits (64 for the angles of the rotation), rounded once at the end; with ``own``
true by the calls a user of the package makes.
"""
import math

import torch

own = False

DEV = "cuda"
TYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32}


def listed():
    def append(name, **kw):
        return dict(dict(name=name, op="append", interleaved=False, ragged=False), **kw)

    def attend(name, **kw):
        return dict(dict(name=name, op="attend", causal_block=0, decay=-1.0, ragged=False), **kw)

    def slots(name, **kw):
        return dict(dict(name=name, op="slots", ragged=False), **kw)

    return [
        # one read-out token of one stream joins 64 cached frames of a 7 x 7 map: latency
        append("append token", dtype="bfloat16", streams=1, tokens=1, cached=3136, q_heads=20, kv_heads=4, dim=64,
               page=64, sections="16,24,24", interleaved=True),
        # the frame of 32 streams processed as one batch (14 x 14 maps) takes the slots that were given up
        append("append 32 frames 14x14", dtype="float16", streams=32, tokens=196, cached=1568, q_heads=8, kv_heads=8,
               dim=64, page=49, sections="16,24,24"),
        # a whole clip enters an empty cache: 64 frames of a 17 x 30 map
        append("append clip 17x30", dtype="bfloat16", streams=1, tokens=32640, cached=32640, q_heads=16, kv_heads=4,
               dim=128, page=64, sections="32,48,48"),
        # one token of one stream reads 64 cached frames of a 7 x 7 map, their weights are renewed: latency
        attend("token over 64 frames 7x7", dtype="float16", streams=1, tokens=1, cached=3136, q_heads=20, kv_heads=4,
               dim=64, page=64, decay=0.0),
        # one token each of 32 streams with clips of different lengths: bound by reading the cache
        attend("token, 32 ragged streams", dtype="bfloat16", streams=32, tokens=1, cached=32640, q_heads=16, kv_heads=2,
               dim=128, page=64, ragged=True),
        # a frame of a 7 x 7 map over the last 64 such frames, one stream
        attend("frame 7x7", dtype="float16", streams=1, tokens=49, cached=3136, q_heads=20, kv_heads=4, dim=64, page=49),
        # a frame of a 17 x 30 map over the last 64, the accumulated weights kept for the next eviction
        attend("frame 17x30, weights", dtype="bfloat16", streams=1, tokens=510, cached=32640, q_heads=16, kv_heads=4,
               dim=128, page=64, decay=0.9),
        # 24 frames of a 17 x 30 map at once, every frame sees itself and the frames before it
        attend("clip 17x30 by frames", dtype="bfloat16", streams=1, tokens=12240, cached=12240, q_heads=16, kv_heads=4,
               dim=128, page=64, causal_block=510),
        # full precision: 8 x 8 maps, 64 frames, four streams
        attend("frame 8x8 float32", dtype="float32", streams=4, tokens=64, cached=4096, q_heads=8, kv_heads=8, dim=64,
               page=64, decay=0.0),
        # which 49 of the tokens of 64 frames of a 7 x 7 map give way to the next frame: latency
        slots("slots 7x7", streams=1, tokens=49, cached=3136, kv_heads=4, page=64, protect=2),
        # the same for 32 streams of 14 x 14 maps, 8 heads each with a choice of its own
        slots("slots 32 streams 14x14", streams=32, tokens=196, cached=12544, kv_heads=8, page=49, protect=1),
        # one long cache: 64 frames of a 34 x 60 map
        slots("slots 34x60", streams=1, tokens=2040, cached=130560, kv_heads=4, page=64, protect=4),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "attend", "slots"])
    kv = rng.choice([1, 2, 3, 4, 5, 8])
    streams = rng.choice([1, 1, 2, 3, 5, 8, 16, 32])
    page = rng.choice([16, 30, 32, 49, 64, 77, 100, 128, 196, 256])
    if op == "slots":
        cached = _log(rng, 64, 16 * 8160 // streams)
        return dict(op=op, streams=streams, tokens=_log(rng, 1, max(2, min(2040, cached // 2))), cached=cached, kv_heads=kv,
                    page=page, protect=rng.randint(0, 3), ragged=rng.random() < 0.4)
    heads = kv * rng.choice([1, 1, 2, 3, 4, 5, 8])
    dtype = rng.choice(["float16", "bfloat16", "bfloat16", "float32"])
    dim = rng.choice([32, 40, 64, 64, 72, 80, 96, 128, 128])
    if op == "append":
        tokens = _log(rng, 1, max(2, min(8160, 65280 // (streams * heads))))
        cached = tokens + _log(rng, 1, 4080)
        third = dim // 3 // 2 * 2
        sections = rng.choice(["%d,%d,%d" % (dim - 2 * third, third, third), "%d,%d,%d" % (third, third, third - 2),
                               "%d,%d" % (dim // 4 * 2, dim - dim // 4 * 2), "%d" % dim])
        return dict(op=op, dtype=dtype, streams=streams, tokens=tokens, cached=cached, q_heads=heads, kv_heads=kv, dim=dim,
                    page=page, sections=sections, interleaved=rng.random() < 0.5, ragged=rng.random() < 0.4)
    tokens = rng.choice([1, 1, _log(rng, 2, 64), _log(rng, 64, 2040)])
    most = 12240 * 12240 * 16 * 128 // (4 * streams * tokens * heads * dim)  # far below the largest listed case's work
    cached = tokens + _log(rng, 8, max(16, min(32640 // max(1, streams // 2), most)))
    block = rng.choice([0, 0, 1, max(1, tokens // 4)]) if tokens > 1 else 0
    return dict(op=op, dtype=dtype, streams=streams, tokens=tokens, cached=cached, q_heads=heads, kv_heads=kv, dim=dim,
                page=page, causal_block=block, decay=rng.choice([-1.0, 0.0, 0.5]), ragged=rng.random() < 0.5)


def _counts(case):
    """New tokens of every stream."""
    n, b = case["tokens"], case["streams"]
    return [max(1, n - (7 * i) % (n // 2 + 1)) if case["ragged"] else n for i in range(b)]


def _lengths(case):
    """Cached tokens of every stream (append, attend: the new ones among them)."""
    n = case["cached"]
    most = [c if case["op"] != "slots" else 1 for c in _counts(case)]
    return [max(most[i], n - n * (5 * i % 8) // 16) if case["ragged"] else n for i in range(case["streams"])]


def _frequencies(sections, base=10000.0):
    """One ladder of frequencies for each axis, in 64 bits."""
    rows = [base ** (-torch.arange(0, n, 2, dtype=torch.float64, device=DEV) / n) for n in sections]
    return torch.cat(rows)


def _pool(case, gen):
    """Page table of every stream over one pool whose pages are handed out in no order."""
    per = -(-case["cached"] // case["page"])
    pages = case["streams"] * per
    table = torch.randperm(pages, generator=gen, device=DEV).to(torch.int32).view(case["streams"], per)
    return table, pages


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(1000003 * seed + 17)

    def normal(*shape, dtype=torch.float32):
        return torch.randn(shape, generator=gen, device=DEV, dtype=torch.float32).to(dtype)

    counts, lengths = _counts(case), _lengths(case)
    starts = [0]
    for c in counts:
        starts.append(starts[-1] + c)
    total, kv, page = starts[-1], case["kv_heads"], case["page"]
    table, pages = _pool(case, gen)
    s = dict(case=case, page_table=table, total=total, most=max(counts),
             lens=torch.tensor(lengths, dtype=torch.int32, device=DEV),
             starts=torch.tensor(starts, dtype=torch.int32, device=DEV))
    if case["op"] != "append":
        # accumulated weights: many small, a few large, new tokens at zero (ties)
        w = torch.rand((pages, kv, page), generator=gen, device=DEV)
        s["weights"] = torch.where(w < 0.05, torch.zeros_like(w), -torch.log(w.clamp_min(1e-6)) ** 3)
    if case["op"] == "slots":
        # the stamp of a token: the frame it came from, in no order after earlier evictions
        frames = max(2, case["cached"] // case["tokens"])
        s["stamps"] = torch.randint(0, frames, (pages, kv, page), generator=gen, device=DEV, dtype=torch.int32)
        s["keep_from"] = torch.full((case["streams"],), frames - case["protect"], dtype=torch.int32, device=DEV)
        s["budget"] = case["cached"]
        return s
    dtype, dim = TYPES[case["dtype"]], case["dim"]
    s["keys"], s["values"] = normal(pages, kv, page, dim, dtype=dtype), normal(pages, kv, page, dim, dtype=dtype)
    # one row of a projection's output a token, q, k and v side by side
    heads = case["q_heads"]
    if case["op"] == "attend":
        s["q"] = normal(total, heads, dim, dtype=torch.float32).mul_(1.5).to(dtype)
        s["weights_before"] = s["weights"].clone()
        return s
    fused = normal(total, (heads + 2 * kv) * dim, dtype=dtype)
    s["q"] = fused[:, :heads * dim].view(total, heads, dim)
    s["k"] = fused[:, heads * dim:(heads + kv) * dim].view(total, kv, dim)
    s["v"] = fused[:, (heads + kv) * dim:].view(total, kv, dim)
    sections = [int(n) for n in case["sections"].split(",")]
    s["sections"], s["frequencies"] = sections, _frequencies(sections)
    place = torch.arange(total, device=DEV)
    # far into a stream: the frame index of a camera that has run for hours
    axes = [place // 510 + 400000 + seed, place % 510 // 30, place % 30][:len(sections)]
    s["positions"] = torch.stack(axes, 1).to(torch.int32).contiguous()
    if case["tokens"] == case["cached"]:
        slots = torch.cat([torch.arange(c, device=DEV) for c in counts]).expand(kv, total)
    else:
        order = torch.rand((kv, case["streams"], case["cached"]), generator=gen, device=DEV)
        order += (torch.arange(case["cached"], device=DEV) >= s["lens"][:, None]).float() * 2
        order = order.argsort(dim=2)
        slots = torch.cat([order[:, i, :c].sort(dim=1).values for i, c in enumerate(counts)], dim=1)
    s["slots"] = slots.to(torch.int32).contiguous()
    s["weights"] = torch.ones((pages, kv, page), device=DEV)
    s["stamps"] = torch.zeros((pages, kv, page), dtype=torch.int32, device=DEV)
    s["cache_lens"] = torch.zeros_like(s["lens"])
    return s


def _rotated(x, cos, sin, interleaved):
    """Pairs of elements of the rotated part of every head turned by their angle."""
    x = x.to(cos.dtype)
    n = 2 * cos.shape[1]
    cos, sin = cos[:, None], sin[:, None]
    a, b = (x[..., 0:n:2], x[..., 1:n:2]) if interleaved else (x[..., :n // 2], x[..., n // 2:n])
    a, b = a * cos - b * sin, a * sin + b * cos
    turned = torch.stack((a, b), -1).flatten(-2) if interleaved else torch.cat((a, b), -1)
    return torch.cat((turned, x[..., n:]), -1)


def _stream_of(s):
    """The stream of every new token."""
    return torch.searchsorted(s["starts"][1:].contiguous(), torch.arange(s["total"], device=DEV, dtype=torch.int32), right=True)


def _plain_append(s):
    case, page = s["case"], s["case"]["page"]
    axis = torch.repeat_interleave(torch.arange(len(s["sections"]), device=DEV),
                                   torch.tensor([n // 2 for n in s["sections"]], device=DEV), output_size=sum(s["sections"]) // 2)
    angle = s["positions"].double()[:, axis] * s["frequencies"]
    cos, sin = angle.cos().float(), angle.sin().float()
    q = _rotated(s["q"], cos, sin, case["interleaved"]).to(s["q"].dtype)
    k = _rotated(s["k"], cos, sin, case["interleaved"]).to(s["k"].dtype)
    slots = s["slots"].long()
    where = s["page_table"].long()[_stream_of(s).expand_as(slots), slots // page], torch.arange(case["kv_heads"], device=DEV)[:, None], slots % page
    s["keys"][where] = k.transpose(0, 1)
    s["values"][where] = s["v"].transpose(0, 1)
    s["weights"][where] = 0.0
    s["stamps"][where] = s["positions"][:, 0].expand_as(s["slots"])
    s["cache_lens"].copy_(s["lens"])
    return q, s["keys"], s["values"], s["weights"], s["stamps"], s["cache_lens"]


def _gathered(s, pages):
    """[streams, heads, slots, ...] of a pool [pages, heads, page, ...]."""
    x = pages[s["page_table"].long()].transpose(1, 2)
    return x.flatten(2, 3)


def _plain_attend(s):
    case = s["case"]
    kv, group, dim, n = case["kv_heads"], case["q_heads"] // case["kv_heads"], case["dim"], s["most"]
    if case["decay"] > 0:
        s["weights"].copy_(s["weights_before"])
    k, v = _gathered(s, s["keys"]).float(), _gathered(s, s["values"]).float()
    slot = torch.arange(k.shape[2], device=DEV)
    valid = slot < s["lens"][:, None]
    v = torch.where(valid[:, None, :, None], v, 0.0)
    counts = s["starts"][1:] - s["starts"][:-1]
    token = torch.arange(n, device=DEV)
    there = token < counts[:, None]
    row = (s["starts"][:-1, None] + token).clamp(max=s["total"] - 1).long()
    q = s["q"][row].float().unflatten(2, (kv, group)).permute(0, 2, 3, 1, 4).reshape(case["streams"], kv, group * n, dim)
    score = torch.matmul(q, k.transpose(2, 3)).mul_(dim ** -0.5).unflatten(2, (group, n))
    see = (valid[:, None] & there[:, :, None])
    if case["causal_block"]:
        limit = (s["lens"] - counts)[:, None] + (token // case["causal_block"] + 1) * case["causal_block"]
        see = see & (slot < limit[..., None])
    see = see[:, None, None]
    score = score.masked_fill_(~see, -math.inf)
    most = score.amax(-1, keepdim=True)
    p = score.sub_(torch.where(most == -math.inf, 0.0, most)).exp_()
    p = p.div_(p.sum(-1, keepdim=True).clamp_min(1e-38))
    out = torch.matmul(p.flatten(2, 3), v).unflatten(2, (group, n)).permute(0, 3, 1, 2, 4).flatten(2, 3)
    out = out[there].to(s["q"].dtype)
    if case["decay"] < 0:
        return out
    received = p.sum((2, 3))
    page = case["page"]
    where = s["page_table"].long()[:, slot // page][:, None], torch.arange(kv, device=DEV)[:, None], slot % page
    old = s["weights"][where]
    new = received if case["decay"] == 0 else case["decay"] * old + received
    s["weights"][where] = torch.where(valid[:, None], new, old)
    return out, s["weights"]


def _plain_slots(s):
    case = s["case"]
    weight, stamp = _gathered(s, s["weights"]), _gathered(s, s["stamps"])
    slot = torch.arange(weight.shape[2], device=DEV)
    rank = (stamp >= s["keep_from"][:, None, None]).to(torch.int32)
    rank = torch.where(slot < s["lens"][:, None, None], rank, 2)
    order = weight.argsort(dim=2, stable=True)
    order = order.gather(2, rank.gather(2, order).argsort(dim=2, stable=True))
    counts = s["starts"][1:] - s["starts"][:-1]
    out = torch.minimum((s["lens"] + counts - s["budget"]).clamp_min(0), s["lens"])
    place = torch.arange(min(s["most"], order.shape[2]), device=DEV)
    given = torch.where(place < out[:, None, None], order[..., :place.numel()], slot.numel()).sort(dim=2).values
    token = torch.arange(s["total"], device=DEV, dtype=torch.int32)
    stream = _stream_of(s)
    token = (token - s["starts"][stream]).long()
    freed = given[stream, :, token.clamp(max=place.numel() - 1)].T
    behind = s["lens"][stream] + token - out[stream]
    slots = torch.where(token < out[stream], freed, torch.where(behind < s["budget"], behind, -1))
    return slots.to(torch.int32), torch.clamp(s["lens"] + counts, max=s["budget"])


def run(s):
    case = s["case"]
    if not own:
        return {"append": _plain_append, "attend": _plain_attend, "slots": _plain_slots}[case["op"]](s)
    from deltacnn_amd import hip_kernels as hk
    starts = s["starts"] if case["ragged"] else None
    if case["op"] == "append":
        q = hk.rotary_append(s["q"], s["k"], s["v"], s["positions"], s["frequencies"], s["sections"], s["keys"], s["values"],
                             s["page_table"], s["slots"], starts=starts, weights=s["weights"], stamps=s["stamps"],
                             lens=s["cache_lens"], new_lens=s["lens"], interleaved=case["interleaved"])
        return q, s["keys"], s["values"], s["weights"], s["stamps"], s["cache_lens"]
    if case["op"] == "attend":
        if case["decay"] < 0:
            return hk.paged_attention(s["q"], s["keys"], s["values"], s["page_table"], s["lens"], starts=starts,
                                      causal_block=case["causal_block"])
        if case["decay"] > 0:
            s["weights"].copy_(s["weights_before"])
        out = hk.paged_attention(s["q"], s["keys"], s["values"], s["page_table"], s["lens"], starts=starts,
                                 causal_block=case["causal_block"], weights=s["weights"], decay=case["decay"])
        return out, s["weights"]
    return hk.cache_slots(s["weights"], s["page_table"], s["lens"], s["total"], s["budget"], starts=starts,
                          stamps=s["stamps"], keep_from=s["keep_from"])


def _pairs(case):
    """Visible (token, slot) pairs of all streams."""
    n, block = 0, case["causal_block"]
    for count, length in zip(_counts(case), _lengths(case)):
        if not block:
            n += count * length
            continue
        for first in range(0, count, block):
            n += min(block, count - first) * min(length, length - count + first + block)
    return n


def work(case):
    total, cached, kv = sum(_counts(case)), sum(_lengths(case)), case["kv_heads"]
    if case["op"] == "slots":
        return {"bytes": 8 * cached * kv + 4 * total * kv + 12 * case["streams"], "flops": 0}
    size = 4 if case["dtype"] == "float32" else 2
    heads, dim = case["q_heads"], case["dim"]
    if case["op"] == "append":
        axes = len(case["sections"].split(","))
        return {"bytes": 2 * total * (heads + 2 * kv) * dim * size + total * (4 * axes + 12 * kv), "flops": 6 * total * (heads + kv) * dim // 2}
    weights = 0 if case["decay"] < 0 else 4 * cached * kv if case["decay"] == 0 else 8 * cached * kv
    return {"bytes": 2 * total * heads * dim * size + 2 * cached * kv * dim * size + weights, "flops": 4 * _pairs(case) * heads * dim}


def exact(case, seed):
    if case["op"] == "slots":
        return None  # whole numbers alone
    s = prepare(case, seed)
    counts, lengths = _counts(case), _lengths(case)
    page, kv, dim, group = case["page"], case["kv_heads"], case["dim"], case["q_heads"] // case["kv_heads"]
    table = s["page_table"].long()
    first = 0
    if case["op"] == "append":
        parts = []
        for axis, n in enumerate(s["sections"]):
            j = torch.arange(n // 2, dtype=torch.float64, device=DEV)
            parts.append(s["positions"][:, axis:axis + 1].double() * torch.pow(torch.tensor(10000.0, dtype=torch.float64, device=DEV), -2 * j / n))
        turn = torch.polar(torch.ones((), dtype=torch.float64, device=DEV), torch.cat(parts, 1))[:, None]
        half = turn.shape[2]

        def rotate(x):
            y = x.double().clone()
            re, im = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if case["interleaved"] else (slice(0, half), slice(half, 2 * half))
            z = torch.complex(y[..., re], y[..., im]) * turn
            y[..., re], y[..., im] = z.real, z.imag
            return y

        q, k = rotate(s["q"]), rotate(s["k"])
        keys, values = s["keys"].double(), s["values"].double()
        weights = s["weights"].double()
        for b, count in enumerate(counts):
            for h in range(kv):
                slot = s["slots"][h, first:first + count].long()
                at = table[b, slot // page]
                keys[at, h, slot % page] = k[first:first + count, h]
                values[at, h, slot % page] = s["v"][first:first + count, h].double()
                weights[at, h, slot % page] = 0
            first += count
        return q, keys, values, weights, None, None
    out = torch.zeros(s["total"], case["q_heads"], dim, dtype=torch.float64, device=DEV)
    weights = s["weights_before"].double()
    for b, (count, length) in enumerate(zip(counts, lengths)):
        slot = torch.arange(length, device=DEV)
        limit = torch.full((count,), length, device=DEV)
        if case["causal_block"]:
            limit = length - count + (torch.arange(count, device=DEV) // case["causal_block"] + 1) * case["causal_block"]
        at, off = table[b, slot // page], slot % page
        for h in range(kv):
            k, v = s["keys"][at, h, off].double(), s["values"][at, h, off].double()
            received = torch.zeros(length, dtype=torch.float64, device=DEV)
            for g in range(h * group, (h + 1) * group):
                score = s["q"][first:first + count, g].double() @ k.T / math.sqrt(dim)
                score[slot >= limit[:, None]] = -math.inf
                p = torch.softmax(score, 1)
                out[first:first + count, g] = p @ v
                received += p.sum(0)
            if case["decay"] >= 0:
                weights[at, h, off] = case["decay"] * weights[at, h, off] + received
        first += count
    return out if case["decay"] < 0 else (out, weights)
