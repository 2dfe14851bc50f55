"""Plain forms, in 64 bits, of the 4-bit paged cache and of the selection of pages, and inputs for their tests."""
from __future__ import annotations

import math

import torch

from tests.operator_forms import CODES, HALF_STEP, quantised

FOUR = ("e2m1", "int4")
MAGNITUDES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def two_to(exponent):
    """Powers of two in 64 bits, from their bits."""
    return ((exponent.long() + 1023) << 52).view(torch.float64)


def least_power(most, top):
    """The exponents of the smallest powers of two that leave `most` at most `top`; in 64 bits, exactly."""
    mantissa, exponent = torch.frexp(most.double())
    m, e = math.frexp(top)
    return exponent - e + (mantissa > m)


# ------------------------------------------------------------------ the formats


def quantised4(x, kind):
    """(codes 0 .. 15 [..., dim], scales as held [..., dim / 32]) of vectors x, with the cache's arithmetic: powers of two are
    exact, the two quotients of INT4 are rounded to 32 bits once each."""
    x = x.float().unflatten(-1, (-1, 32))
    finite = torch.isfinite(x).all(-1)
    x = torch.where(finite[..., None], x, 0.0)
    most = x.abs().amax(-1).clamp_min(2.0 ** -100)
    if kind == "e2m1":
        exponent = least_power(most, 7.0).clamp_max(125)
        y = x.double() * two_to(-exponent)[..., None]
        a = y.abs()
        # Halfway cases go to the even code.
        code = sum(((a >= b) if even else (a > b)).int() for b, even in
                   ((0.25, 0), (0.75, 1), (1.25, 0), (1.75, 1), (2.5, 0), (3.5, 1), (5.0, 0)))
        code = torch.where(y < 0, code + 8, code)
        return code.flatten(-2).to(torch.uint8), torch.where(finite, exponent + 127, 255).to(torch.uint8)
    scale = ((most.double() / torch.full_like(most, 7).double()).float().view(torch.int32) & -65536).view(torch.float32)
    inverse = (torch.ones_like(scale).double() / scale.double()).float()
    code = (x * inverse[..., None]).round().clamp(-7, 7) + 8
    return code.flatten(-2).to(torch.uint8), torch.where(finite, scale, math.nan).to(torch.bfloat16)


def packed(codes, values):
    """Codes [..., dim] as a cache holds them [..., dim / 2]."""
    dim, out = codes.shape[-1], []
    for byte in range(dim // 2):
        first = 32 * (byte % (dim // 32)) + 2 * (byte // (dim // 32)) if values else 2 * byte
        out.append(codes[..., first] | codes[..., first + 1] << 4)
    return torch.stack(out, -1)


def unpacked(held, values):
    dim = 2 * held.shape[-1]
    out = [None] * dim
    for byte in range(dim // 2):
        first = 32 * (byte % (dim // 32)) + 2 * (byte // (dim // 32)) if values else 2 * byte
        out[first], out[first + 1] = held[..., byte] & 15, held[..., byte] >> 4
    return torch.stack(out, -1)


def numbers4(codes, kind):
    """What codes stand for before their scale, in 64 bits."""
    if kind == "int4":
        return codes.double() - 8
    table = torch.tensor(MAGNITUDES + tuple(-m for m in MAGNITUDES), dtype=torch.float64, device=codes.device)
    return table[codes.long()]


def scales4(scales, kind):
    """Scales as held, as numbers in 64 bits; NaN where they are not finite."""
    if kind == "int4":
        s = scales.double()
        return torch.where(torch.isfinite(s), s, math.nan)
    return torch.where(scales == 255, math.nan, two_to(scales.int() - 127))


def parts(cache, kind, name):
    """(numbers [pages, heads, page, dim], scales [pages, heads, page, dim]) of a cache's keys or values, 4 or 8 bits."""
    held = cache[name[:-1] + "_scales"]
    if kind in FOUR:
        return (numbers4(unpacked(cache[name], name == "values"), kind),
                scales4(held, kind).repeat_interleave(32, -1))
    codes = cache[name].view(torch.int8).contiguous().view(CODES[kind]).double()
    return codes, held.double()[..., None].expand_as(codes)


# ------------------------------------------------------------------ caches


def make_pages(kind, pages, heads, page, dim, token_major=False, stale=None, seed=0, device="cuda"):
    """Tensors of a cache of either kind: random codes and scales (`stale`: every scale NaN instead, as memory that nothing
    has written may hold)."""
    from tests import operator_forms

    if kind not in FOUR:
        return operator_forms.make_pages(kind, pages, heads, page, dim, token_major, stale, seed, device)
    g = torch.Generator(device=device)
    g.manual_seed(seed)
    shape = (pages, page, heads, dim // 2) if token_major else (pages, heads, page, dim // 2)

    def codes():
        bits = torch.randint(0, 256, shape, generator=g, dtype=torch.uint8, device=device)
        return bits.permute(0, 2, 1, 3) if token_major else bits

    def scales():
        size = (pages, heads, page, dim // 32)
        if kind == "e2m1":
            return torch.full(size, 255, dtype=torch.uint8, device=device) if stale else \
                torch.randint(120, 128, size, generator=g, dtype=torch.uint8, device=device)
        x = torch.full(size, math.nan, device=device) if stale else 0.1 + 0.4 * torch.rand(size, generator=g, device=device)
        return x.to(torch.bfloat16)

    return dict(keys=codes(), values=codes(), key_scales=scales(), value_scales=scales())


def hold(cache, kind, name, ids, at, x):
    """Writes vectors x [n, heads, dim] to positions `at` of pages `ids`."""
    if kind in FOUR:
        codes, scale = quantised4(x, kind)
        codes = packed(codes, name == "values")
    else:
        codes, scale = quantised(x, kind)
        codes = codes.view(torch.uint8)
    cache[name].view(torch.uint8).transpose(1, 2)[ids, at] = codes
    cache[name[:-1] + "_scales"].transpose(1, 2)[ids, at] = scale


def fill(cache, kind, table, lengths, seed=1, spread=0.0):
    """Writes random positions into the cache's pages at every row's first `lengths` positions; the
    rest is left. `spread`: values spread over e^-spread .. e^spread."""
    heads, page = cache["keys"].shape[1:3]
    dim = cache["keys"].shape[3] * (2 if kind in FOUR else 1)
    g = torch.Generator(device=cache["keys"].device)
    g.manual_seed(seed)
    for r, n in enumerate(lengths):
        n = min(max(n, 0), table.shape[1] * page)
        if n == 0:
            continue
        for name in ("keys", "values"):
            x = torch.randn(n, heads, dim, generator=g, device=table.device)
            if name == "values" and spread:
                x = x * ((2 * torch.rand(n, heads, 1, generator=g, device=table.device) - 1) * spread).exp()
            at = torch.arange(n, device=table.device)
            ids = table[r].long()[at // page]
            here = (ids >= 0) & (ids < cache["keys"].shape[0])
            hold(cache, kind, name, ids[here], at[here] % page, x[here])


# ------------------------------------------------------------------ attention


def attended(q, cache, kind, table, lengths, scale, max_length=1 << 31):
    """(outputs in 64 bits, the bound of the kernel's error, element by element); rows of negative
    lengths are NaN. `table` [rows, width] or [rows, heads, width].

    As operator_forms.attended derives it for one scale a vector: a weight enters the products with half a step of F16 (two
    F16 parts of F32 tensors: 2^-22) or, below F16's normal range, 2^-25 of the largest weight, which counts with the
    position's largest value scale; p is off by what its score is: q's elements below F16's normal range by 2^-25 of the
    largest (2^-22 of each for two parts), dim roundings of the products' sums, one for each group's scale (8 at most) and 4 more,
    2 ulp of exp2 and 4 roundings of the score (base 2) itself. The weight is multiplied twice more (the
    reciprocal of the scaling, the value's scale): 4 roundings. Sums over positions round at most once for each 32
    positions and 64 times in all joins.

    16-bit tensors: the F16 weight has a power of two of its position's scales and is multiplied by the group's ratio to
    it, in F16. E2M1: a power of two, at most 1, so there is no second rounding. INT4: the ratio has eight bits and is below 2, so
    the product is rounded once more, and what is lost below the normal range is 2 * 2^-25 + 2^-25."""
    rows, q_heads, dim = q.shape
    pages, heads, page = cache["keys"].shape[:3]
    out = torch.full(q.shape, math.nan, dtype=torch.float64, device=q.device)
    off = torch.zeros_like(out)
    two = q.dtype == torch.float32
    again = kind == "int4" and not two
    kn, ks = parts(cache, kind, "keys")
    vn, vs = parts(cache, kind, "values")
    group = q_heads // heads
    for r in range(rows):
        for h in range(heads):
            pages_of = (table[r, h] if table.dim() == 3 else table[r]).long()
            n = min(int(lengths[r]), max_length, pages_of.shape[0] * page)
            if n < 0:
                continue
            at = torch.arange(n, device=q.device)
            ids = pages_of[at // page]
            here = (ids >= 0) & (ids < pages)
            ids, at = ids[here], at[here] % page
            mine = slice(h * group, (h + 1) * group)
            if len(at) == 0:
                out[r, mine] = 0
                continue
            qd = q[r, mine].double()
            k = (kn[ids, h, at] * ks[ids, h, at]).t().contiguous()
            vc, w = vn[ids, h, at], vs[ids, h, at]
            v = vc * w
            score = qd @ k * scale
            p = torch.softmax(score, -1)
            o = p @ v
            size = (qd.abs() @ k.abs()) * abs(scale)
            lost = (qd.abs().amax(-1, keepdim=True) * k.abs().sum(0)) * abs(scale) * 2.0 ** -25
            rounding = 2.0 ** -22 if two else 2.0 ** -10 if again else 2.0 ** -11
            e = lost + size * ((dim + 12) * 2.0 ** -24 + (2.0 ** -22 if two else 0.0))
            e = e + 4 * 2.0 ** -24 * (score - score.amax(-1, keepdim=True)).abs() + 4 * 2.0 ** -24 * score.abs().amax(-1, keepdim=True)
            e = e.amax(-1, keepdim=True) + 2.0 ** -22
            total = 2 * e + rounding + (len(at) / 32 + 68) * 2.0 ** -24
            least = (p * w.abs().amax(-1)).amax(-1, keepdim=True) * (3 if again else 1) * 2.0 ** -25
            bound = total * (p @ v.abs()) + least * vc.abs().sum(0)
            out[r, mine] = o
            off[r, mine] = bound + HALF_STEP[q.dtype] * (o.abs() + bound)
            if q.dtype == torch.float16:
                off[r, mine] += 2.0 ** -25  # F16's subnormals
    return out, off


# ------------------------------------------------------------------ selection


def whole(x):
    """(whole numbers of at most 127, powers of two) of vectors x in 64 bits: exact but for the numbers' rounding."""
    power = two_to(least_power(x.abs().amax(-1, keepdim=True).clamp_min(2.0 ** -100), 127.0))
    return torch.round(x / power), power.squeeze(-1)


def bounds_of(cache, kind, page, head, count):
    """(codes [2, dim], scale) of one page and KV head with `count` positions."""
    numbers, scale = (cached[page, head, :count] for cached in parts(cache, kind, "keys"))
    keys = (numbers * scale).float().double()  # what reading back gives in F32
    if not torch.isfinite(keys).all():
        return torch.zeros(2, keys.shape[-1], dtype=torch.int8, device=keys.device), math.nan
    codes, power = whole(torch.cat((keys.amax(0), keys.amin(0))))
    return codes.view(2, -1).to(torch.int8), power.item()


def selected(q, bounds_codes, bounds_scales, table, lengths, page, keep, first, last, max_length=1 << 31):
    """(pages [rows, heads, keep], lengths): the selection in 64 bits, in Python. Rows of negative lengths are left -7."""
    rows, q_heads, dim = q.shape
    pages, heads = bounds_scales.shape
    out = torch.full((rows, heads, keep), -7, dtype=torch.int32)
    new = torch.zeros(rows, dtype=torch.int32)
    numbers, power = whole(torch.nan_to_num(q.double(), nan=0.0, posinf=0.0, neginf=0.0))
    power = torch.where(torch.isfinite(q.double()).all(-1), power, math.nan)
    for r in range(rows):
        n = min(int(lengths[r]), max_length, table.shape[1] * page)
        count = -(-n // page)
        new[r] = n if count <= keep else n - (count - keep) * page
        if n < 0:
            continue
        ids = table[r, :max(count, 0)].long()
        if count <= keep:
            out[r] = torch.cat((ids, torch.full((keep - count,), -1, device=ids.device))).int().cpu()
            continue
        there = (ids >= 0) & (ids < pages)
        ids = torch.where(there, ids, 0)
        for h in range(heads):
            group = slice(h * q_heads // heads, (h + 1) * q_heads // heads)
            both = numbers[r, group][:, None, None, :] * bounds_codes[ids, h].double()[None]       # [group, pages, 2, dim]
            score = both.amax(2).sum(-1) * bounds_scales[ids, h].double() * power[r, group][:, None]
            score = torch.where(torch.isnan(score).any(0), math.inf, score.amax(0))
            score = torch.where(there, score, -math.inf).tolist()
            forced = [p for p in range(count) if p < first or p >= count - last]
            rest = sorted((p for p in range(count) if first <= p < count - last), key=lambda p: (-score[p], p))
            places = sorted(forced + rest[:keep - len(forced)])
            out[r, h] = table[r, places].cpu()
    return out, new
