"""Performance cases of the operators for long contexts on device memory: the 4-bit paged KV cache
(written, read back, attended over by one new token a row), and attention over the pages that a
cheap score selects for each row and KV head, of a 4-bit or an 8-bit cache.

A cache has ``pages`` pages of ``page`` positions. In 4 bits, 32 elements that follow one another share
a scale: E2M1 codes with a power of two (one byte, E8M0), or INT4 codes (-7 .. 7, held as code + 8) with the
upper half of an F32 number (BF16). Two codes lie in a byte, the lower one first: a key's in
order, a value's with byte ``G c + g`` holding elements ``32 g + 2 c`` and the next (``G``: groups of a head).

A page's bounds are, for each KV head and channel, the largest and the smallest key element of its positions, as whole
numbers up to 127 times one power of two. A page's score for a query is the sum over channels of the larger product with
the two bounds, the query taken as whole numbers up to 127 times a power of two as well: scores are
exact, and so is the selection.

* ``write``: k rotated, k and v quantised into the 4-bit cache at the rows' slots, q rotated; then the
  rows are read back, as the values that the cache now holds for them (in 16 bits).
* ``read``: every position of some sequences read back, in order.
* ``attend``: one new token's attention for ``rows`` sequences over their cached positions.
* ``index``: the bounds of all pages of some prompts, and each row's first selection.
* ``sparse``: a decode step's attention: the bounds of the pages that took a new position, the selection of ``keep`` pages
  a row and KV head, and the attention over them.
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
BYTES = {"f16": 2, "bf16": 2, "f32": 4}
FOUR = ("e2m1", "int4")
HELD = {"e2m1": 17 / 32, "int4": 18 / 32}  # bytes an element, with its share of the scale


def listed():
    return [
        # The 64-row decode batch of the serving benchmark: each row's new position is cached.
        dict(name="write_64", kind="write", rows=64, q_heads=32, kv_heads=8, head_dim=128, rotary=128, interleaved=False,
             scaling="none", theta=1e6, dtype="f16", format="e2m1", page=64, token_major=False, low=32, high=2048),
        # A long prompt in one pass, head dimension 256.
        dict(name="write_2011_d256", kind="write", rows=2011, q_heads=20, kv_heads=4, head_dim=256, rotary=256,
             interleaved=False, scaling="linear", theta=1000042.0, dtype="bf16", format="int4", page=64,
             token_major=True, low=0, high=2010),
        # A long sequence read back as 16 bits for its next chunk's attention.
        dict(name="read_30000", kind="read", rows=1, low=30000, high=30000, kv_heads=8, head_dim=128, dtype="f16",
             format="e2m1", page=64, token_major=False),
        # Several sequences moved out in F32, short pages, head dimension 64.
        dict(name="read_7_d64", kind="read", rows=7, low=70, high=1100, kv_heads=8, head_dim=64, dtype="f32",
             format="int4", page=16, token_major=True),
        # One interactive request on a small model: the smallest call, where latency counts.
        dict(name="attend_1", kind="attend", rows=1, low=100, high=100, q_heads=16, kv_heads=8, head_dim=128,
             dtype="f16", format="e2m1", page=64, token_major=False),
        # The serving benchmark's 64 rows at its mix of contexts (mean about 480).
        dict(name="attend_64", kind="attend", rows=64, low=32, high=2048, q_heads=32, kv_heads=8, head_dim=128,
             dtype="f16", format="int4", page=64, token_major=False),
        # A large batch to contexts of 8192, head dimension 256, short pages, an odd group of heads, in F32.
        dict(name="attend_128_d256", kind="attend", rows=128, low=1, high=8192, q_heads=20, kv_heads=4, head_dim=256,
             dtype="f32", format="int4", page=16, token_major=False),
        # Two dozen long documents at once: the cache is all the work.
        dict(name="attend_24_long", kind="attend", rows=24, low=12000, high=30000, q_heads=32, kv_heads=8, head_dim=128,
             dtype="bf16", format="e2m1", page=64, token_major=True),
        # Prompts of some thousand tokens have been written: their pages' bounds, and the first selection.
        dict(name="index_8", kind="index", rows=8, low=2048, high=30000, q_heads=32, kv_heads=8, head_dim=128, dtype="f16",
             format="e2m1", page=16, token_major=False, keep=128, first=1, last=2),
        # One short sequence of an 8-bit cache, head dimension 64.
        dict(name="index_1_8bit", kind="index", rows=1, low=1100, high=1100, q_heads=32, kv_heads=8, head_dim=64, dtype="bf16",
             format="e4m3", page=64, token_major=False, keep=8, first=1, last=1),
        # 32 long documents, each head reading 2048 positions of its row.
        dict(name="sparse_32", kind="sparse", rows=32, low=12000, high=30000, q_heads=32, kv_heads=8, head_dim=128,
             dtype="f16", format="e2m1", page=16, token_major=False, keep=128, first=1, last=2),
        # A few rows over an 8-bit cache, head dimension 256, an odd group of heads, idle rows behind them.
        dict(name="sparse_9_8bit", kind="sparse", rows=9, low=300, high=16000, idle=2, q_heads=20, kv_heads=4, head_dim=256,
             dtype="bf16", format="int8", page=64, token_major=True, keep=16, first=1, last=1),
    ]


def _log_int(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["write", "read", "attend", "attend", "index", "sparse", "sparse"])
    kv_heads = rng.choice([1, 2, 4, 8])
    head_dim = rng.choice([64, 128, 256])
    case = dict(kind=kind, kv_heads=kv_heads, head_dim=head_dim, dtype=rng.choice(["f16", "f16", "bf16", "f32"]),
                format=rng.choice(FOUR), page=rng.choice([8, 16, 32, 64, 128]), token_major=rng.random() < 0.4)
    if kind != "read":
        case["q_heads"] = kv_heads * rng.randint(1, 32 // kv_heads if head_dim < 256 else max(1, 16 // kv_heads))
    if kind == "write":
        case["rotary"] = rng.choice([head_dim, head_dim, head_dim // 2, head_dim // 4, 20])
        case["interleaved"] = rng.random() < 0.4
        case["scaling"] = rng.choice(["none", "linear"])
        case["theta"] = rng.choice([1e4, 5e5, 1e6])
        case["rows"] = _log_int(rng, 1, 2048)
        case["low"] = _log_int(rng, 1, 100000)
        case["high"] = case["low"] + case["rows"] - 1 + _log_int(rng, 1, 2000)
    else:
        case["rows"] = _log_int(rng, 1, {"read": 8, "attend": 128, "index": 16, "sparse": 64}[kind])
        case["low"] = _log_int(rng, 1, 300)
        case["high"] = _log_int(rng, case["low"], 30000)
        if kind != "read":  # a batch padded with requests that hold nothing
            case["idle"] = rng.randint(0, case["rows"] // 2) if rng.random() < 0.3 else 0
    if kind in ("index", "sparse"):
        case["format"] = rng.choice(FOUR + FOUR + ("e4m3", "int8"))
        case["first"], case["last"] = rng.randint(0, 2), rng.randint(1, 3)
        case["keep"] = case["first"] + case["last"] + _log_int(rng, 1, 150)
    # No more work than the largest listed case has, and padded lengths that a gather can hold.
    most = max(work(c)["bytes"] for c in listed())
    while work(case)["bytes"] > most or _padded(case) > 1 << 30:
        if kind == "write":
            case["rows"] //= 2
            case["high"] = case["low"] + case["rows"]
        else:
            case["high"] = max(case["low"], case["high"] // 2)
            case["rows"] = case["rows"] if case["high"] > case["low"] else case["rows"] // 2
            case["idle"] = min(case.get("idle", 0), case["rows"] // 2)
    return case


# ------------------------------------------------------------------ what a case means


def _padded(case):
    """Elements of the keys (or of their bounds) with every sequence as long as the longest."""
    return 0 if case["kind"] == "write" else case["rows"] * case["high"] * case["kv_heads"] * case["head_dim"]


def _lengths(case):
    """The sequences' lengths: log-uniform quantiles of [low, high], and 0 for idle rows at the end."""
    idle = case.get("idle", 0)
    n, low, high = case["rows"] - idle, case["low"], case["high"]
    return [max(1, int(round(low * (high / low) ** ((i + 0.5) / n)))) for i in range(n)] + [0] * idle


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _heads(g, rows, heads, dim, dtype):
    """Activations of a projection: some channels several times wider than the others."""
    x = torch.randn(rows, heads, dim, generator=g, device="cuda")
    wide = 1 + 4 * (torch.rand(heads, dim, generator=g, device="cuda") < 0.05)
    return (x * wide).to(dtype)


# ------------------------------------------------------------------ the caches' formats, plainly


def _e2m1(x):
    """(codes 0 .. 15, scale bytes) of groups of 32 in the last dimension, in 32 bits."""
    most = x.abs().amax(-1).clamp_min(2.0 ** -100)
    # The smallest exponent that leaves the largest magnitude at most 7, at most 125.
    byte = ((most.view(torch.int32) + 0x1FFFFF) >> 23).sub(2).clamp_max(252)
    y = x * ((254 - byte) << 23).view(torch.float32)[..., None]
    a = y.abs()
    code = (a > 0.25).int() + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5)
    return (code + 8 * (y < 0)).to(torch.uint8), byte.to(torch.uint8)


def _int4(x):
    most = x.abs().amax(-1).clamp_min(2.0 ** -100)
    bits = (most.double() / 7).float().view(torch.int32) & -65536
    scale = bits.view(torch.float32)
    inverse = (1 / scale.double()).float()
    code = (x * inverse[..., None]).round().clamp(-7, 7) + 8
    return code.to(torch.uint8), scale.to(torch.bfloat16)


def _quantise(x, kind, values):
    """What a cache holds of vectors x [..., head_dim]: (codes as stored, scales as stored)."""
    x = x.float()
    if kind not in FOUR:
        peak = 448.0 if kind == "e4m3" else 127.0
        most = x.abs().amax(-1, keepdim=True).clamp_min(2.0 ** -100)
        y = x * (peak / most)
        codes = y.to(torch.float8_e4m3fn).view(torch.int8) if kind == "e4m3" else y.round().clamp(-127, 127).to(torch.int8)
        return codes, (most / peak).squeeze(-1)
    codes, scale = (_e2m1 if kind == "e2m1" else _int4)(x.unflatten(-1, (-1, 32)))
    codes = codes.unflatten(-1, (16, 2))                       # [..., group, pair, 2]
    if values:
        codes = codes.transpose(-3, -2)
    return (codes[..., 0] | codes[..., 1] << 4).flatten(-2), scale


def _stored_as(kind):
    return {"e2m1": (torch.uint8, torch.uint8), "int4": (torch.uint8, torch.bfloat16), "e4m3": (torch.float8_e4m3fn, torch.float32),
            "int8": (torch.int8, torch.float32)}[kind]


_VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _held(codes, scale, kind, values):
    """The vectors [..., head_dim] that codes and scales as stored stand for, in 32 bits."""
    if kind not in FOUR:
        return codes.view(_stored_as(kind)[0]).float() * scale[..., None]
    groups = scale.shape[-1]
    c = torch.stack((codes & 15, codes >> 4), -1)
    c = c.unflatten(-2, (16, groups) if values else (groups, 16))
    c = (c.transpose(-3, -2) if values else c).flatten(-2)      # [..., group, 32]
    if kind == "int4":
        return ((c.float() - 8) * scale.float()[..., None]).flatten(-2)
    table = torch.tensor(_VALUES + tuple(-v for v in _VALUES), device=c.device)
    return (table[c.int()] * (scale.int() << 23).view(torch.float32)[..., None]).flatten(-2)


def _cache(case, count, g):
    """Pages for `count` positions and a third more, with what earlier requests left in them."""
    kind, page, heads, dim = case["format"], case["page"], case["kv_heads"], case["head_dim"]
    pages = count // page * 4 // 3 + 2
    width = dim // 2 if kind in FOUR else dim

    def stale():
        bits = torch.randint(0, 120, (pages, page, heads, width) if case["token_major"] else (pages, heads, page, width),
                             generator=g, device="cuda", dtype=torch.int8)
        return (bits.permute(0, 2, 1, 3) if case["token_major"] else bits).view(_stored_as(kind)[0])

    def scales():
        if kind == "e2m1":
            return torch.randint(110, 130, (pages, heads, page, dim // 32), generator=g, device="cuda", dtype=torch.uint8)
        shape = (pages, heads, page) + ((dim // 32,) if kind == "int4" else ())
        return (torch.rand(shape, generator=g, device="cuda") * 0.02).to(_stored_as(kind)[1])

    return {"keys": stale(), "values": stale(), "key_scales": scales(), "value_scales": scales()}


def _bytes(codes):
    return codes.view(torch.uint8)


def _filled(case, lengths, g):
    """A cache that holds sequences of these lengths, and their page table. A head's keys drift along a sequence, so that
    pages differ in what they hold, as text does."""
    page, heads, dim = case["page"], case["kv_heads"], case["head_dim"]
    need = [-(-n // page) for n in lengths]
    cache = _cache(case, sum(need) * page, g)
    ids = torch.randperm(cache["keys"].shape[0], generator=g, device="cuda")[: sum(need)]
    width = max(need)
    own_pages = torch.arange(width, device="cuda")[None, :] < torch.tensor(need, device="cuda")[:, None]
    table = torch.full((len(need), width), -1, device="cuda", dtype=torch.int32)
    table[own_pages] = ids.int()
    step = 1 + (1 << 25) // (heads * page * dim)
    for name in ("keys", "values"):
        for at in range(0, len(ids), step):
            part = ids[at: at + step]
            x = torch.randn(len(part), heads, page, dim, generator=g, device="cuda")
            x = x * (0.3 + torch.rand(len(part), heads, page, 1, generator=g, device="cuda"))
            if name == "keys":
                x += torch.randn(len(part), heads, 1, dim, generator=g, device="cuda")
            codes, scale = _quantise(x, case["format"], name == "values")
            _bytes(cache[name])[part] = _bytes(codes)
            cache[name[:-1] + "_scales"][part] = scale
    return cache, table


def _frequencies(case):
    """Angle a position of each rotated pair in 64 bits."""
    n = case["rotary"]
    f = case["theta"] ** (-torch.arange(0, n, 2, dtype=torch.float64) / n)
    return f / 4.0 if case["scaling"] == "linear" else f


def prepare(case, seed):
    g = _generator(seed)
    rows, dtype, kind = case["rows"], DTYPES[case["dtype"]], case["kind"]
    state = {"case": case, "dtype": dtype, "read": dtype}
    if kind == "write":
        state["q"] = _heads(g, rows, case["q_heads"], case["head_dim"], dtype)
        state["k"] = _heads(g, rows, case["kv_heads"], case["head_dim"], dtype)
        state["v"] = _heads(g, rows, case["kv_heads"], case["head_dim"], dtype)
        span = case["high"] - case["low"] + 1
        if span <= rows:
            at = torch.arange(rows, device="cuda")
        else:
            at = torch.randint(0, span, (rows,), generator=g, device="cuda")
        state["positions"] = (case["low"] + at).int()
        state["frequencies"] = _frequencies(case).cuda()
        state["cache"] = _cache(case, rows, g)
        capacity = state["cache"]["keys"].shape[0] * case["page"]
        state["read"] = torch.float16 if case["dtype"] == "f32" else dtype
        state["slots"] = torch.randperm(capacity, generator=g, device="cuda")[:rows].int()
    else:
        lengths = _lengths(case)
        state["cache"], state["table"] = _filled(case, lengths, g)
        state["lengths"] = torch.tensor(lengths, device="cuda", dtype=torch.int32)
        state["longest"] = max(lengths)
    if kind == "read":
        page, table = case["page"], state["table"].long()
        slots = table[:, :, None] * page + torch.arange(page, device="cuda")
        held = torch.arange(slots.shape[1] * page, device="cuda")[None, :] < state["lengths"][:, None]
        state["slots"] = slots.reshape(len(lengths), -1)[held].int()
    if kind in ("attend", "index", "sparse"):
        state["q"] = _heads(g, rows, case["q_heads"], case["head_dim"], dtype)
    if kind in ("index", "sparse"):
        pages, heads = state["cache"]["keys"].shape[:2]
        state["bounds"] = {"codes": torch.zeros(pages, heads, 2, case["head_dim"], dtype=torch.int8, device="cuda"),
                           "scales": torch.zeros(pages, heads, device="cuda")}
        # The positions whose pages' bounds are to be made: all of them, or the step's new one.
        state["starts"] = torch.zeros_like(state["lengths"]) if kind == "index" else (state["lengths"] - 1).clamp_min(0)
        state["new"] = state["longest"] if kind == "index" else 1
        if kind == "sparse":  # earlier steps have made the others
            _bound(state, torch.zeros_like(state["lengths"]), state["lengths"] - 1)
    if own:  # what a program that serves keeps: the rotation's plan, the descriptions of the cache and of its bounds
        from hllm_amd import operators

        if kind == "write":
            scaling = {"rope_type": "linear", "factor": 4.0} if case["scaling"] == "linear" else None
            state["plan"] = operators.Rope(case["rotary"], theta=case["theta"], interleaved=case["interleaved"], scaling=scaling)
        state["pages"] = (operators.Kv4Pages if case["format"] in FOUR else operators.KvPages)(**state["cache"])
        if "bounds" in state:
            state["index"] = operators.KvBounds(state["pages"], **state["bounds"])
    return state


# ------------------------------------------------------------------ the operators, plainly


def _rotate(x, s):
    """Rotated rows in 32 bits; the angles in 64."""
    case, n = s["case"], s["case"]["rotary"]
    angle = s["positions"].double()[:, None] * s["frequencies"]
    cos, sin = angle.cos().float()[:, None, :], angle.sin().float()[:, None, :]
    x = x.float()
    if case["interleaved"]:
        a, b = x[..., 0:n:2], x[..., 1:n:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = x[..., : n // 2], x[..., n // 2: n]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((turned, x[..., n:]), -1)


def _gather(s, name, pages, offsets, heads=None):
    """The values of positions (page, offset) [..., kv_heads, head_dim] in 32 bits, or of (page, head, offset)
    [..., head_dim]."""
    codes, scale = _bytes(s["cache"][name]), s["cache"][name[:-1] + "_scales"]
    if heads is None:
        codes, scale = codes.transpose(1, 2)[pages, offsets], scale.transpose(1, 2)[pages, offsets]
    else:
        codes, scale = codes[pages, heads, offsets], scale[pages, heads, offsets]
    return _held(codes, scale, s["case"]["format"], name == "values")


def _read(s):
    slots, page = s["slots"].long(), s["case"]["page"]
    return [_gather(s, name, slots // page, slots % page).to(s["read"]) for name in ("keys", "values")]


def _write(s):
    slots, page = s["slots"].long(), s["case"]["page"]
    for name, x in (("keys", _rotate(s["k"], s)), ("values", s["v"])):
        codes, scale = _quantise(x, s["case"]["format"], name == "values")
        _bytes(s["cache"][name]).transpose(1, 2)[slots // page, slots % page] = codes
        s["cache"][name[:-1] + "_scales"].transpose(1, 2)[slots // page, slots % page] = scale
    return _rotate(s["q"], s).to(s["dtype"])


def _softmax_over(s, k, v, held):
    """k and v [rows, heads, positions, dim], held [rows, positions]."""
    rows, heads, _, dim = k.shape
    q = s["q"].float().view(rows, heads, -1, dim)
    score = torch.matmul(q, k.transpose(2, 3).contiguous()) / math.sqrt(dim)
    score = score.masked_fill(~held[:, None, None, :], -math.inf)
    p = (score - score.amax(-1, keepdim=True).clamp_min(-1e30)).exp()
    p = p / p.sum(-1, keepdim=True).clamp_min(1e-30)  # 0 where a row holds nothing
    return torch.matmul(p, v.contiguous()).view(rows, -1, dim).to(s["dtype"])


def _attend(s):
    at = torch.arange(s["longest"], device="cuda")
    pages = s["table"].long()[:, at // s["case"]["page"]].clamp_min(0)
    offsets = (at % s["case"]["page"]).expand_as(pages)
    k, v = (_gather(s, name, pages, offsets).transpose(1, 2) for name in ("keys", "values"))
    return _softmax_over(s, k, v, at[None, :] < s["lengths"][:, None])


def _whole(x):
    """(whole numbers up to 127, power of two) of vectors along the last dimension."""
    most = x.abs().amax(-1, keepdim=True).clamp_min(2.0 ** -100)
    byte = ((most.view(torch.int32) + 0x1FFFF) >> 23) - 6      # 127 = 1.984375 * 2^6
    return (x * ((254 - byte) << 23).view(torch.float32)).round(), (byte << 23).view(torch.float32)


def _bound(s, starts, lengths):
    """The bounds of the pages that hold positions starts .. lengths - 1 of a row, from all of their positions."""
    page = s["case"]["page"]
    at = torch.arange(s["table"].shape[1], device="cuda")
    n = torch.minimum(lengths[:, None] - at * page, torch.tensor(page, device="cuda"))
    row, column = ((n > 0) & ((at + 1) * page > starts[:, None])).nonzero(as_tuple=True)
    step = 1 + (1 << 27) // (s["case"]["kv_heads"] * page * s["case"]["head_dim"])
    for part in range(0, len(row), step):
        r, c = row[part: part + step], column[part: part + step]
        ids = s["table"][r, c].long()
        keys = _held(_bytes(s["cache"]["keys"])[ids], s["cache"]["key_scales"][ids], s["case"]["format"], False)
        held = (torch.arange(page, device="cuda") < n[r, c][:, None])[:, None, :, None]
        high, low = keys.masked_fill(~held, -math.inf).amax(2), keys.masked_fill(~held, math.inf).amin(2)
        codes, scale = _whole(torch.cat((high, low), -1))
        s["bounds"]["codes"][ids] = codes.to(torch.int8).unflatten(-1, (2, -1))
        s["bounds"]["scales"][ids] = scale.squeeze(-1)


def _select(s):
    """(pages [rows, kv_heads, keep], lengths): the selected pages in their order, -1 behind them."""
    case, table, lengths = s["case"], s["table"].long(), s["lengths"].long()
    rows, width = table.shape
    heads, dim, page, keep = case["kv_heads"], case["head_dim"], case["page"], case["keep"]
    count = (lengths + page - 1) // page
    q, q_scale = _whole(s["q"].float())
    q = torch.cat((q.clamp_min(0), q.clamp_max(0)), -1).view(rows, heads, -1, 2 * dim)
    bounds = s["bounds"]["codes"][table.clamp_min(0)].flatten(-2).float()     # [rows, width, heads, 2 dim]
    dots = torch.matmul(q, bounds.permute(0, 2, 3, 1).contiguous())             # exact: below 2^24
    scale = s["bounds"]["scales"][table.clamp_min(0)].transpose(1, 2)[:, :, None, :]
    score = (dots * scale * q_scale.view(rows, heads, -1, 1)).amax(2)
    at = torch.arange(width, device="cuda")
    forced = (at < case["first"]) | (at >= count[:, None] - case["last"])
    score = score.masked_fill(forced[:, None, :], math.inf).masked_fill((at >= count[:, None])[:, None, :], -math.inf)
    order = torch.sort(score, dim=-1, descending=True, stable=True).indices[..., :keep]
    if order.shape[-1] < keep:
        order = torch.nn.functional.pad(order, (0, keep - order.shape[-1]), value=width)
    order = torch.where(order < count[:, None, None], order, width).sort(-1).values
    picked = torch.cat((table, torch.full((rows, 1), -1, device="cuda")), 1)[:, None, :].expand(rows, heads, -1).gather(2, order)
    return picked.int(), torch.where(count <= keep, lengths, lengths - (count - keep) * page).int()


def _sparse(s):
    case = s["case"]
    picked, lengths = _select(s)
    at = torch.arange(picked.shape[2] * case["page"], device="cuda")
    pages = picked.long()[:, :, at // case["page"]].clamp_min(0)
    heads = torch.arange(case["kv_heads"], device="cuda")[None, :, None].expand_as(pages)
    offsets = (at % case["page"]).expand_as(pages)
    k, v = (_gather(s, name, pages, offsets, heads) for name in ("keys", "values"))
    return _softmax_over(s, k, v, at[None, :] < lengths[:, None]), picked, lengths


def run(state):
    case, kind = state["case"], state["case"]["kind"]
    if own:
        from hllm_amd import operators

        if kind == "write":
            q = operators.kv_append(state["pages"], state["slots"], state["k"], state["v"], q=state["q"],
                                    rope=state["plan"], positions=state["positions"])
            return q, *operators.kv_read(state["pages"], state["slots"], state["read"])
        if kind == "read":
            return operators.kv_read(state["pages"], state["slots"], state["read"])
        if kind == "attend":
            return operators.kv_attention(state["q"], state["pages"], state["table"], state["lengths"], state["longest"])
        operators.kv_bounds(state["pages"], state["index"], state["table"], state["starts"], state["lengths"], state["new"])
        picked, lengths = operators.kv_select(state["q"], state["index"], state["table"], state["lengths"], state["longest"],
                                              case["keep"], first=case["first"], last=case["last"])
        if kind == "index":
            return picked, lengths
        out = operators.kv_attention(state["q"], state["pages"], picked, lengths, case["keep"] * case["page"])
        return out, picked, lengths
    if kind == "write":
        return _write(state), *_read(state)
    if kind == "read":
        return tuple(_read(state))
    if kind == "attend":
        return _attend(state)
    _bound(state, state["starts"], state["lengths"])
    return _select(state) if kind == "index" else _sparse(state)


def work(case):
    dim, kv, size, page = case["head_dim"], case["kv_heads"], BYTES[case["dtype"]], case["page"]
    rows, q = case["rows"], case.get("q_heads", 0)
    vector = dim * HELD[case["format"]] if case["format"] in FOUR else dim + 4  # a key or value with its scales
    held = int(2 * kv * vector)
    if case["kind"] == "write":
        # k, v and q in; the cache's rows, q and the rows as read back out.
        return {"bytes": rows * (2 * (q + kv) * dim * size + 2 * kv * dim * min(size, 2) + held + 8),
                "flops": rows * (3 * (q + kv) * case["rotary"] + 6 * kv * dim)}
    lengths = _lengths(case)
    positions, pages = sum(lengths), sum(-(-n // page) for n in lengths)
    if case["kind"] == "read":
        return {"bytes": positions * (held + 2 * kv * dim * size + 4), "flops": 2 * positions * kv * dim}
    if case["kind"] == "attend":
        return {"bytes": positions * held + 2 * rows * q * dim * size + 4 * rows + 4 * pages, "flops": 4 * positions * q * dim}
    bounds = kv * (2 * dim + 4)
    kept = sum(min(n, max(0, n - (-(-n // page) - case["keep"]) * page)) for n in lengths)
    select = {"bytes": pages * (bounds + 4) + rows * (q * dim * size + 4 * kv * case["keep"] + 8), "flops": 4 * pages * q * dim}
    if case["kind"] == "index":
        return {"bytes": select["bytes"] + positions * held // 2 + pages * bounds, "flops": select["flops"] + 2 * positions * kv * dim}
    fresh = sum((n - 1) % page + 1 for n in lengths if n > 0)
    return {"bytes": select["bytes"] + fresh * held // 2 + kept * held + rows * q * dim * size,
            "flops": select["flops"] + 2 * fresh * kv * dim + 4 * kept * q * dim}


# ------------------------------------------------------------------ in 64 bits


def _turned(case, x, position):
    """Complex products: each pair as one number, turned by its angle."""
    n, y = case["rotary"], x.double().clone()
    f = torch.tensor([case["theta"] ** (-2.0 * i / n) / (4 if case["scaling"] == "linear" else 1) for i in range(n // 2)],
                     dtype=torch.float64, device="cuda")
    angle = position.double()[:, None] * f
    turn = torch.polar(torch.ones_like(angle), angle)[:, None, :]
    if case["interleaved"]:
        z = torch.view_as_complex(y[..., :n].unflatten(-1, (n // 2, 2)).contiguous()) * turn
        y[..., :n] = torch.view_as_real(z).flatten(-2)
    else:
        z = torch.complex(y[..., : n // 2], y[..., n // 2: n]) * turn
        y[..., : n // 2], y[..., n // 2: n] = z.real, z.imag
    return y


def _nearest(x, case):
    """The cache's values for vectors x: the format's nearest code to each element, times the group's scale."""
    y = x.unflatten(-1, (-1, 32))
    most = y.abs().amax(-1, keepdim=True).clamp_min(2.0 ** -100)
    if case["format"] == "int4":
        mantissa, exponent = torch.frexp(most / torch.full_like(most, 7))  # a quotient: by a number it would be a product
        scale = torch.floor(mantissa * 256) * _two_to(exponent - 8)        # eight bits, cut off
        return (torch.round(y / scale) * scale).flatten(-2)
    z = y / (scale := _power(most, 7))
    # E2M1: one bit after the leading one, steps of a half below 2; ties to even, no more than 6.
    step = _two_to(torch.frexp(z.abs().clamp_min(1.0))[1] - 2)
    return ((torch.round(z / step) * step).clamp(-6, 6) * scale).flatten(-2)


def _vectors(case, cache, name, ids):
    """A cache's vectors in pages `ids`: [pages, heads, page, dim] in 64 bits, element by element from its code."""
    codes, scale, dim = cache[name].view(torch.uint8)[ids], cache[name[:-1] + "_scales"][ids], case["head_dim"]
    if case["format"] not in FOUR:
        # code * scale, rounded to 32 bits: what the cache is read as.
        values = codes.view(torch.float8_e4m3fn if case["format"] == "e4m3" else torch.int8).double() * scale.double()[..., None]
        return values.float().double()
    element = torch.arange(dim, device="cuda")
    group, pair = element // 32, element % 32 // 2
    byte = codes[..., pair * (dim // 32) + group if name == "values" else element // 2]
    code = torch.where(element % 2 == 1, byte // 16, byte % 16).double()
    if case["format"] == "int4":
        return (code - 8) * scale.double()[..., group]
    low = code % 8
    magnitude = torch.where(low < 2, low / 2, (1 + low % 2 / 2) * _two_to(low // 2 - 1))
    return torch.where(code >= 8, -magnitude, magnitude) * _two_to(scale.int() - 127)[..., group]


def _two_to(exponent):
    """Powers of two, from their bits."""
    return ((exponent.long() + 1023) << 52).view(torch.float64)


def _power(x, top=127):
    """The smallest power of two that leaves the largest magnitude of the last dimension at most `top`."""
    mantissa, exponent = torch.frexp(x.abs().amax(-1, keepdim=True).clamp_min(2.0 ** -100))   # in [1 / 2, 1)
    own_mantissa, own_exponent = math.frexp(top)
    return _two_to(exponent - own_exponent + (mantissa > own_mantissa))


def _chosen(case, keys, q):
    """The selected pages of one row for one KV head, by their places: `keys` [pages, page, dim] with what takes no part
    NaN, q [group, dim]. The pages' bounds are whole numbers times powers of two."""
    high = torch.nan_to_num(keys, nan=-math.inf).amax(1)
    low = torch.nan_to_num(keys, nan=math.inf).amin(1)
    power, own_power = _power(torch.cat((high, low), -1)), _power(q)
    high, low, q = torch.round(high / power) * power, torch.round(low / power) * power, torch.round(q / own_power) * own_power
    score = torch.maximum(q[:, None, :] * high, q[:, None, :] * low).sum(-1).amax(0).tolist()
    places = range(len(score))
    forced = [p for p in places if p < case["first"] or p >= len(score) - case["last"]]
    rest = sorted((p for p in places if p not in set(forced)), key=lambda p: (-score[p], p))
    return sorted(forced + rest[: max(0, case["keep"] - len(forced))])


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "write":
        return (_turned(case, s["q"], s["positions"]), _nearest(_turned(case, s["k"], s["positions"]), case),
                _nearest(s["v"].double(), case))
    page, dim, heads = case["page"], case["head_dim"], case["kv_heads"]
    if case["kind"] in ("index", "sparse") and sum(_lengths(case)) * heads > 1 << 23:
        return None  # the selection in Python takes long
    out, tables, kept = [], [], []
    for r, n in enumerate(_lengths(case)):
        ids = s["table"][r, : -(-n // page)].long()
        k, v = (_vectors(case, s["cache"], x, ids).transpose(0, 1) for x in ("keys", "values"))  # [heads, pages, page, dim]
        if case["kind"] == "read":
            out.append(tuple(x.flatten(1, 2)[:, :n].transpose(0, 1) for x in (k, v)))
            continue
        q = s["q"][r].double().view(heads, -1, dim)
        places = [list(range(len(ids)))] * heads
        if case["kind"] in ("index", "sparse"):
            if len(ids) > case["keep"]:
                masked = k.clone()
                masked[:, -1, (n - 1) % page + 1:] = math.nan
                places = [_chosen(case, masked[h], q[h]) for h in range(heads)]
            tables.append([[int(ids[p]) for p in at] + [-1] * (case["keep"] - len(at)) for at in places])
            n -= (len(ids) - len(places[0])) * page
            kept.append(n)
        if case["kind"] != "index":
            for h in range(heads):
                kh, vh = (x[h, places[h]].flatten(0, 1)[:n] for x in (k, v))
                out.append(torch.softmax(q[h] @ kh.t().contiguous() / math.sqrt(dim), -1) @ vh)
    if case["kind"] == "read":
        return tuple(torch.cat(x) for x in zip(*out))
    if case["kind"] in ("index", "sparse"):
        ints = tuple(torch.tensor(x, dtype=torch.int32, device="cuda") for x in (tables, kept))
    if case["kind"] == "index":
        return ints
    attended = torch.cat(out).view(case["rows"], -1, dim)
    return attended if case["kind"] == "attend" else (attended, *ints)
