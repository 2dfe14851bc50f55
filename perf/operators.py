"""Performance cases of the operators on device memory: rotary positions, the 8-bit paged KV
cache (written, read back) and one new token's attention over it.

A cache has ``pages`` pages of ``page`` positions: codes ``[pages, kv_heads, page, head_dim]``
(E4M3 or INT8) and a scale ``[pages, kv_heads, page]`` for each position and head, for keys and
values each. ``token_major`` keeps a page's codes as ``[page, kv_heads, head_dim]`` in memory.

* ``rope``: q and k of ``rows`` rows rotated at their positions.
* ``write``: k rotated, k and v quantised into the cache at the rows' slots, q rotated; then the
  rows are read back, as the values that the cache now holds for them (in 16 bits).
* ``read``: every position of some sequences read back, in order.
* ``attend``: one new token's attention for ``rows`` sequences over their cached positions.
"""
from __future__ import annotations

import math

import torch

own = False

PEAK = {"e4m3": 448.0, "int8": 127.0}
CODES = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
BYTES = {"f16": 2, "bf16": 2, "f32": 4}


def listed():
    return [
        # One request's next token on a small model: the smallest call, where launches count.
        dict(name="rope_1", kind="rope", rows=1, q_heads=16, kv_heads=8, head_dim=128, rotary=128, interleaved=False,
             scaling="none", theta=1e6, dtype="f16", low=100, high=100),
        # A long prompt's chunk at contexts stretched eightfold, head dimension 64.
        dict(name="rope_8192_llama3", kind="rope", rows=8192, q_heads=32, kv_heads=8, head_dim=64, rotary=64,
             interleaved=False, scaling="llama3", theta=5e5, dtype="bf16", low=90000, high=98191),
        # A quarter of a wide head rotated in neighbouring pairs, F32 rows at far positions.
        dict(name="rope_517_partial", kind="rope", rows=517, q_heads=20, kv_heads=4, head_dim=256, rotary=64,
             interleaved=True, scaling="yarn", theta=1e4, dtype="f32", low=0, high=1000000),
        # The 64-row decode batch of the serving benchmark: each row's new position is cached.
        dict(name="write_64", kind="write", rows=64, q_heads=32, kv_heads=8, head_dim=128, rotary=128, interleaved=False,
             scaling="none", theta=1e6, dtype="f16", format="e4m3", page=64, token_major=False, low=32, high=2048),
        # A long prompt in one pass, head dimension 256.
        dict(name="write_2011_d256", kind="write", rows=2011, q_heads=20, kv_heads=4, head_dim=256, rotary=256,
             interleaved=False, scaling="linear", theta=1000042.0, dtype="bf16", format="int8", page=64,
             token_major=True, low=0, high=2010),
        # A long sequence read back as 16 bits for its next chunk's attention.
        dict(name="read_30000", kind="read", rows=1, low=30000, high=30000, kv_heads=8, head_dim=128, dtype="f16",
             format="e4m3", page=64, token_major=False),
        # Several sequences moved out in F32, short pages, head dimension 64.
        dict(name="read_7_d64", kind="read", rows=7, low=70, high=1100, kv_heads=8, head_dim=64, dtype="f32",
             format="int8", page=16, token_major=True),
        # One interactive request on a small model.
        dict(name="attend_1", kind="attend", rows=1, low=100, high=100, q_heads=16, kv_heads=8, head_dim=128,
             dtype="f16", format="e4m3", page=64, token_major=False),
        # The serving benchmark's 64 rows at its mix of contexts (mean about 480).
        dict(name="attend_64", kind="attend", rows=64, low=32, high=2048, q_heads=32, kv_heads=8, head_dim=128,
             dtype="f16", format="e4m3", page=64, token_major=False),
        # A handful of F32 rows, head dimension 64.
        dict(name="attend_7_d64", kind="attend", rows=7, low=70, high=1100, q_heads=32, kv_heads=8, head_dim=64,
             dtype="f32", format="int8", page=32, token_major=False),
        # Few requests near the models' longest context: the cache is all the work.
        dict(name="attend_3_long", kind="attend", rows=3, low=12000, high=30000, q_heads=32, kv_heads=8, head_dim=128,
             dtype="bf16", format="e4m3", page=64, token_major=True),
        # A large batch to contexts of 8192, head dimension 256, short pages, an odd group of heads.
        dict(name="attend_128_d256", kind="attend", rows=128, low=1, high=8192, q_heads=20, kv_heads=4, head_dim=256,
             dtype="bf16", format="int8", page=16, token_major=False),
    ]


def _log_int(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["rope", "write", "read", "attend", "attend"])
    kv_heads = rng.choice([1, 2, 4, 8])
    head_dim = rng.choice([64, 128, 256])
    case = dict(kind=kind, kv_heads=kv_heads, head_dim=head_dim, dtype=rng.choice(["f16", "f16", "bf16", "f32"]))
    if kind != "read":
        case["q_heads"] = kv_heads * rng.randint(1, 32 // kv_heads if head_dim < 256 else max(1, 16 // kv_heads))
    if kind in ("rope", "write"):
        case["rotary"] = rng.choice([head_dim, head_dim, head_dim // 2, head_dim // 4, 20])
        case["interleaved"] = rng.random() < 0.4
        case["scaling"] = rng.choice(["none", "linear", "llama3", "yarn"])
        case["theta"] = rng.choice([1e4, 5e5, 1e6])
        case["rows"] = _log_int(rng, 1, 4096 if kind == "rope" else 2048)
        case["low"] = _log_int(rng, 1, 100000)
        case["high"] = case["low"] + case["rows"] - 1 + _log_int(rng, 1, 2000)
    if kind != "rope":
        case["format"] = rng.choice(["e4m3", "int8"])
        case["page"] = rng.choice([8, 16, 32, 64, 128])
        case["token_major"] = rng.random() < 0.4
    if kind in ("read", "attend"):
        case["rows"] = _log_int(rng, 1, 8 if kind == "read" else 128)
        case["low"] = _log_int(rng, 1, 300)
        case["high"] = _log_int(rng, case["low"], 30000)
    if kind == "attend":  # a batch padded with requests that hold nothing
        case["idle"] = rng.randint(0, case["rows"] // 2) if rng.random() < 0.3 else 0
    # No more work than the largest listed case has, and padded lengths that a gather can hold.
    most = max(work(c)["bytes"] for c in listed())
    while work(case)["bytes"] > most or _padded(case) > 1 << 30:
        if kind in ("rope", "write"):
            case["rows"] //= 2
            case["high"] = case["low"] + case["rows"]
        else:
            case["high"] = max(case["low"], case["high"] // 2)
            case["rows"] = case["rows"] if case["high"] > case["low"] else case["rows"] // 2
            case["idle"] = min(case.get("idle", 0), case["rows"] // 2)
    return case


# ------------------------------------------------------------------ what a case means


def _padded(case):
    """Elements of the keys with every sequence as long as the longest."""
    return 0 if case["kind"] in ("rope", "write") else case["rows"] * case["high"] * case["kv_heads"] * case["head_dim"]


def _lengths(case):
    """The sequences' lengths: log-uniform quantiles of [low, high], and 0 for idle rows at the end."""
    idle = case.get("idle", 0)
    n, low, high = case["rows"] - idle, case["low"], case["high"]
    return [max(1, int(round(low * (high / low) ** ((i + 0.5) / n)))) for i in range(n)] + [0] * idle


def _scaling(case):
    """The long-context scaling as a model's configuration states it (None: unscaled)."""
    return {
        "none": None,
        "linear": {"rope_type": "linear", "factor": 4.0},
        "llama3": {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
                   "original_max_position_embeddings": 8192},
        "yarn": {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 32768},
    }[case["scaling"]]


def _frequencies(case):
    """Angle a position of each rotated pair in 64 bits, and the factor on the rotated values."""
    n, theta, s = case["rotary"], case["theta"], _scaling(case)
    f = theta ** (-torch.arange(0, n, 2, dtype=torch.float64) / n)
    if s is None:
        return f, 1.0
    if s["rope_type"] == "linear":
        return f / s["factor"], 1.0
    length = s["original_max_position_embeddings"]
    if s["rope_type"] == "llama3":
        low, high = s["low_freq_factor"], s["high_freq_factor"]
        keep = ((length * f / (2 * math.pi) - low) / (high - low)).clamp(0, 1)
        return f * keep + f / s["factor"] * (1 - keep), 1.0

    def turns(count):  # the pair that turns `count` times over the original length
        return n * math.log(length / (count * 2 * math.pi)) / (2 * math.log(theta))

    first, last = max(0, math.floor(turns(32))), min(n - 1, math.ceil(turns(1)))
    ramp = ((torch.arange(n // 2, dtype=torch.float64) - first) / max(0.001, last - first)).clamp(0, 1)
    return f * (1 - ramp) + f / s["factor"] * ramp, 0.1 * math.log(s["factor"]) + 1


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _heads(g, rows, heads, dim, dtype):
    """Activations of a projection: some channels several times wider than the others."""
    x = torch.randn(rows, heads, dim, generator=g, device="cuda")
    wide = 1 + 4 * (torch.rand(heads, dim, generator=g, device="cuda") < 0.05)
    return (x * wide).to(dtype)


def _quantise(x, kind):
    """(codes, scale) of vectors along the last dimension, in 32 bits."""
    x = x.float()
    most = x.abs().amax(-1, keepdim=True).clamp_min(2.0 ** -100)
    y = x * (PEAK[kind] / most)
    codes = y.to(torch.float8_e4m3fn) if kind == "e4m3" else y.round().clamp(-127, 127).to(torch.int8)
    return codes, (most / PEAK[kind]).squeeze(-1)


def _cache(case, count, g):
    """Pages for `count` positions and a third more, with what earlier requests left in them."""
    page, heads, dim = case["page"], case["kv_heads"], case["head_dim"]
    pages = count // page * 4 // 3 + 2

    def stale():
        bits = torch.randint(0, 120, (pages, page, heads, dim) if case["token_major"] else (pages, heads, page, dim),
                             generator=g, device="cuda", dtype=torch.int8)
        return (bits.permute(0, 2, 1, 3) if case["token_major"] else bits).view(CODES[case["format"]])

    def scales():
        return torch.rand(pages, heads, page, generator=g, device="cuda") * 0.02

    return {"keys": stale(), "values": stale(), "key_scales": scales(), "value_scales": scales()}


def _filled(case, lengths, g):
    """A cache that holds sequences of these lengths, and their page table."""
    page, heads, dim = case["page"], case["kv_heads"], case["head_dim"]
    need = [-(-n // page) for n in lengths]
    cache = _cache(case, sum(need) * page, g)
    ids = torch.randperm(cache["keys"].shape[0], generator=g, device="cuda")[: sum(need)]
    width = max(need)
    own_pages = torch.arange(width, device="cuda")[None, :] < torch.tensor(need, device="cuda")[:, None]
    table = torch.full((len(need), width), -1, device="cuda", dtype=torch.int32)
    table[own_pages] = ids.int()
    for name in ("keys", "values"):
        for at in range(0, len(ids), 1 + (1 << 25) // (heads * page * dim)):
            part = ids[at: at + 1 + (1 << 25) // (heads * page * dim)]
            x = torch.randn(len(part), heads, page, dim, generator=g, device="cuda")
            x = x * (0.3 + torch.rand(len(part), heads, page, 1, generator=g, device="cuda"))
            codes, scale = _quantise(x, case["format"])
            cache[name].view(torch.int8)[part] = codes.view(torch.int8)
            cache[name[:-1] + "_scales"][part] = scale
    return cache, table


def prepare(case, seed):
    g = _generator(seed)
    rows, dtype = case["rows"], DTYPES[case["dtype"]]
    state = {"case": case, "dtype": dtype, "read": dtype}
    if case["kind"] in ("rope", "write"):
        state["q"] = _heads(g, rows, case["q_heads"], case["head_dim"], dtype)
        state["k"] = _heads(g, rows, case["kv_heads"], case["head_dim"], dtype)
        span = case["high"] - case["low"] + 1
        if span <= rows:
            at = torch.arange(rows, device="cuda")
        else:
            at = torch.randint(0, span, (rows,), generator=g, device="cuda")
        state["positions"] = (case["low"] + at).int()
        frequencies, state["magnitude"] = _frequencies(case)
        state["frequencies"] = frequencies.cuda()
    if case["kind"] == "write":
        state["v"] = _heads(g, rows, case["kv_heads"], case["head_dim"], dtype)
        state["cache"] = _cache(case, rows, g)
        capacity = state["cache"]["keys"].shape[0] * case["page"]
        state["read"] = torch.float16 if case["dtype"] == "f32" else dtype
        state["slots"] = torch.randperm(capacity, generator=g, device="cuda")[:rows].int()
    if case["kind"] in ("read", "attend"):
        lengths = _lengths(case)
        state["cache"], state["table"] = _filled(case, lengths, g)
        state["lengths"] = torch.tensor(lengths, device="cuda", dtype=torch.int32)
        state["longest"] = max(lengths)
    if case["kind"] == "read":
        page, table = case["page"], state["table"].long()
        slots = table[:, :, None] * page + torch.arange(page, device="cuda")
        held = torch.arange(slots.shape[1] * page, device="cuda")[None, :] < state["lengths"][:, None]
        state["slots"] = slots.reshape(len(lengths), -1)[held].int()
    if case["kind"] == "attend":
        state["q"] = _heads(g, rows, case["q_heads"], case["head_dim"], dtype)
    if own:  # what a program that serves keeps: the rotation's plan, the cache's description
        from hllm_amd import operators

        if case["kind"] in ("rope", "write"):
            state["plan"] = operators.Rope(case["rotary"], theta=case["theta"], interleaved=case["interleaved"],
                                           scaling=_scaling(case))
        if "cache" in state:
            state["pages"] = operators.KvPages(**state["cache"])
    return state


# ------------------------------------------------------------------ the operators, plainly


def _rotate(x, s):
    """Rotated rows in 32 bits; the angles in 64."""
    case, n = s["case"], s["case"]["rotary"]
    angle = s["positions"].double()[:, None] * s["frequencies"]
    cos = (angle.cos() * s["magnitude"]).float()[:, None, :]
    sin = (angle.sin() * s["magnitude"]).float()[:, None, :]
    x = x.float()
    if case["interleaved"]:
        a, b = x[..., 0:n:2], x[..., 1:n:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = x[..., : n // 2], x[..., n // 2: n]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((turned, x[..., n:]), -1)


def _gather(s, name, pages, offsets):
    """The values of positions (page, offset): [..., kv_heads, head_dim] in 32 bits."""
    codes = s["cache"][name].view(torch.int8).permute(0, 2, 1, 3)[pages, offsets]
    scale = s["cache"][name[:-1] + "_scales"].permute(0, 2, 1)[pages, offsets]
    return codes.view(CODES[s["case"]["format"]]).float() * scale[..., None]


def _read(s):
    slots, page = s["slots"].long(), s["case"]["page"]
    return [_gather(s, name, slots // page, slots % page).to(s["read"]) for name in ("keys", "values")]


def _write(s):
    slots, page = s["slots"].long(), s["case"]["page"]
    for name, x in (("keys", _rotate(s["k"], s)), ("values", s["v"])):
        codes, scale = _quantise(x, s["case"]["format"])
        s["cache"][name].view(torch.int8).permute(0, 2, 1, 3)[slots // page, slots % page] = codes.view(torch.int8)
        s["cache"][name[:-1] + "_scales"].permute(0, 2, 1)[slots // page, slots % page] = scale
    return _rotate(s["q"], s).to(s["dtype"])


def _attend(s):
    case = s["case"]
    rows, heads, dim = case["rows"], case["kv_heads"], case["head_dim"]
    at = torch.arange(s["longest"], device="cuda")
    pages = s["table"].long()[:, at // case["page"]].clamp_min(0)
    offsets = (at % case["page"]).expand_as(pages)
    held = at[None, :] < s["lengths"][:, None]
    k = _gather(s, "keys", pages, offsets).permute(0, 2, 3, 1).contiguous()      # [rows, heads, dim, positions]
    q = s["q"].float().view(rows, heads, -1, dim)
    score = torch.matmul(q, k) / math.sqrt(dim)
    score = score.masked_fill(~held[:, None, None, :], -math.inf)
    p = (score - score.amax(-1, keepdim=True).clamp_min(-1e30)).exp()
    p = p / p.sum(-1, keepdim=True).clamp_min(1e-30)  # 0 where a row holds nothing
    v = _gather(s, "values", pages, offsets).permute(0, 2, 1, 3).contiguous()    # [rows, heads, positions, dim]
    return torch.matmul(p, v).view(rows, -1, dim).to(s["dtype"])


def run(state):
    kind = state["case"]["kind"]
    if own:
        from hllm_amd import operators

        if kind == "rope":
            return operators.rope(state["plan"], state["positions"], state["q"], state["k"])
        if kind == "write":
            q = operators.kv_append(state["pages"], state["slots"], state["k"], state["v"], q=state["q"],
                                    rope=state["plan"], positions=state["positions"])
            return q, *operators.kv_read(state["pages"], state["slots"], state["read"])
        if kind == "read":
            return operators.kv_read(state["pages"], state["slots"], state["read"])
        return operators.kv_attention(state["q"], state["pages"], state["table"], state["lengths"], state["longest"])
    if kind == "rope":
        return _rotate(state["q"], state).to(state["dtype"]), _rotate(state["k"], state).to(state["dtype"])
    if kind == "write":
        return _write(state), *_read(state)
    if kind == "read":
        return tuple(_read(state))
    return _attend(state)


def work(case):
    dim, kv, size = case["head_dim"], case["kv_heads"], BYTES[case["dtype"]]
    rows, q = case["rows"], case.get("q_heads", 0)
    held = 2 * kv * (dim + 4)  # a position's codes and scales
    if case["kind"] == "rope":
        return {"bytes": rows * (2 * (q + kv) * dim * size + 4), "flops": 3 * rows * (q + kv) * case["rotary"]}
    if case["kind"] == "write":
        # k, v and q in; the cache's rows, q and the rows as read back out.
        return {"bytes": rows * (2 * (q + kv) * dim * size + 2 * kv * dim * min(size, 2) + held + 8),
                "flops": rows * (3 * (q + kv) * case["rotary"] + 6 * kv * dim)}
    positions = sum(_lengths(case))
    if case["kind"] == "read":
        return {"bytes": positions * (held + 2 * kv * dim * size + 4), "flops": 2 * positions * kv * dim}
    return {"bytes": positions * held + 2 * rows * q * dim * size + 4 * rows + 4 * positions // case["page"],
            "flops": 4 * positions * q * dim}


# ------------------------------------------------------------------ in 64 bits


def _angles(case, position):
    """The angle of each pair at `position` and the factor, pair by pair, from the scalings' definitions."""
    n, s, out = case["rotary"], _scaling(case), []
    for i in range(n // 2):
        f = case["theta"] ** (-2.0 * i / n)
        if s is not None and s["rope_type"] == "linear":
            f /= s["factor"]
        elif s is not None:
            length = s["original_max_position_embeddings"]
            wave = 2 * math.pi / f
            if s["rope_type"] == "llama3":
                if wave > length / s["low_freq_factor"]:
                    f /= s["factor"]
                elif wave > length / s["high_freq_factor"]:
                    mix = (length / wave - s["low_freq_factor"]) / (s["high_freq_factor"] - s["low_freq_factor"])
                    f = (1 - mix) * f / s["factor"] + mix * f
            else:
                edge = [n / 2 * math.log(length / (2 * math.pi * t)) / math.log(case["theta"]) for t in (32.0, 1.0)]
                first, last = max(0, math.floor(edge[0])), min(n - 1, math.ceil(edge[1]))
                mix = min(1.0, max(0.0, (i - first) / max(0.001, last - first)))
                f = f / s["factor"] * mix + f * (1 - mix)
        out.append(f)
    factor = 1 + 0.1 * math.log(s["factor"]) if s is not None and s["rope_type"] == "yarn" else 1.0
    return position.double()[:, None] * torch.tensor(out, dtype=torch.float64, device="cuda"), factor


def _turned(case, x, position):
    """Complex products: each pair as one number, turned by its angle."""
    n = case["rotary"]
    angle, factor = _angles(case, position)
    y = x.double().clone()
    turn = torch.polar(torch.full_like(angle, factor), angle)[:, None, :]
    if case["interleaved"]:
        z = torch.view_as_complex(y[..., :n].unflatten(-1, (n // 2, 2)).contiguous()) * turn
        y[..., :n] = torch.view_as_real(z).flatten(-2)
    else:
        z = torch.complex(y[..., : n // 2], y[..., n // 2: n]) * turn
        y[..., : n // 2], y[..., n // 2: n] = z.real, z.imag
    return y


def _nearest(x, case):
    """The cache's values for vectors x: the format's nearest code to each element, times the scale."""
    scale = x.abs().amax(-1, keepdim=True).clamp_min(2.0 ** -100) / PEAK[case["format"]]
    y = x / scale
    if case["format"] == "int8":
        return torch.round(y) * scale
    # E4M3: three bits after the leading one, steps of 2^-9 below 2^-6; ties to even.
    step = 2.0 ** (torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6))) - 3)
    return torch.round(y / step) * step * scale


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "rope":
        return tuple(_turned(case, s[x], s["positions"]) for x in ("q", "k"))
    if case["kind"] == "write":
        return (_turned(case, s["q"], s["positions"]), _nearest(_turned(case, s["k"], s["positions"]), case),
                _nearest(s["v"].double(), case))
    out, page, dim = [], case["page"], case["head_dim"]
    for r, n in enumerate(_lengths(case)):
        ids = s["table"][r, : -(-n // page)].long()
        k, v = (s["cache"][x].view(torch.int8)[ids].view(CODES[case["format"]]).double()
                * s["cache"][x[:-1] + "_scales"][ids].double()[..., None] for x in ("keys", "values"))
        k, v = (x.transpose(1, 2).flatten(0, 1)[:n] for x in (k, v))   # [positions, kv_heads, head_dim]
        if case["kind"] == "read":
            out.append((k, v))
            continue
        k, v = (x.repeat_interleave(case["q_heads"] // case["kv_heads"], 1) for x in (k, v))
        weight = torch.softmax((k * s["q"][r].double()).sum(-1) / math.sqrt(dim), 0)
        out.append((v * weight[..., None]).sum(0))
    return tuple(torch.cat(x) for x in zip(*out)) if case["kind"] == "read" else torch.stack(out)
