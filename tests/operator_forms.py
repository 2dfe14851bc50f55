"""Plain forms, in 64 bits, of the operators on device memory, and inputs for their tests."""
from __future__ import annotations

import math

import torch

PEAK = {"e4m3": 448.0, "int8": 127.0}
CODES = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
# Half a step of a rounding, relative to the value.
HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
LLAMA3 = {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
          "original_max_position_embeddings": 8192}
YARN = {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 32768}


def frequencies(rotary, theta, scaling=None):
    """(angle a position of each pair, factor on cos and sin), pair by pair in Python floats."""
    s, out = scaling or {"rope_type": "default"}, []
    kind, factor = s["rope_type"], s.get("factor", 1.0)
    for i in range(rotary // 2):
        f = theta ** (-2.0 * i / rotary)
        if kind == "linear":
            f /= factor
        elif kind == "llama3":
            turns = s["original_max_position_embeddings"] * f / (2 * math.pi)
            if turns < s["low_freq_factor"]:
                f /= factor
            elif turns < s["high_freq_factor"]:
                keep = (turns - s["low_freq_factor"]) / (s["high_freq_factor"] - s["low_freq_factor"])
                f = keep * f + (1 - keep) * f / factor
        elif kind == "yarn":
            def pair(turns):
                return rotary * math.log(s["original_max_position_embeddings"] / (turns * 2 * math.pi)) / (2 * math.log(theta))
            first = max(math.floor(pair(s.get("beta_fast", 32.0))), 0)
            last = min(math.ceil(pair(s.get("beta_slow", 1.0))), rotary - 1)
            ramp = min(1.0, max(0.0, (i - first) / max(0.001, last - first)))
            f = f * (1 - ramp) + f / factor * ramp
        out.append(f)
    magnitude = s.get("attention_factor", 0.1 * math.log(factor) + 1) if kind == "yarn" else 1.0
    return out, magnitude


def rotated(x, positions, rotary, theta, interleaved=False, scaling=None):
    """(rotated rows in 64 bits, the bound of a 32-bit rotation's error, element by element).

    The angle is rounded to 2^-32 turn (1.5e-9) and, as an F32 value below pi / 4 times an F32
    constant, three times by 2^-24: 1.5e-7; the series, its roundings and the magnitude add at
    most 4 roundings and 3e-8. So cos and sin are off by 5e-7 of the magnitude at most; the two
    products and their sum add 3 roundings."""
    f, magnitude = frequencies(rotary, theta, scaling)
    angle = positions.double()[:, None] * torch.tensor(f, dtype=torch.float64, device=x.device)
    cos, sin = (angle.cos() * magnitude)[:, None], (angle.sin() * magnitude)[:, None]
    y, off = x.double().clone(), torch.zeros_like(x, dtype=torch.float64)
    first, second = (slice(0, rotary, 2), slice(1, rotary, 2)) if interleaved else \
        (slice(0, rotary // 2), slice(rotary // 2, rotary))
    a, b = y[..., first].clone(), y[..., second].clone()
    y[..., first], y[..., second] = a * cos - b * sin, b * cos + a * sin
    bound = (a.abs() + b.abs()) * magnitude * (5e-7 + 3 * 2.0 ** -24)
    off[..., first], off[..., second] = bound, bound
    return y, off


def quantised(x, kind):
    """(codes, scales) of vectors along the last dimension, with the cache's 32-bit arithmetic: the
    two quotients are rounded once each (of 64 bits, which a division of F32 values survives;
    torch divides by a number with its reciprocal, which rounds twice)."""
    x = x.float()
    finite = torch.isfinite(x).all(-1, keepdim=True)
    most = torch.where(finite, x, 0.0).abs().amax(-1, keepdim=True).clamp_min(2.0 ** -100)
    most = most.double()
    y = torch.where(finite, x, 0.0) * (PEAK[kind] / most).float()
    codes = y.to(torch.float8_e4m3fn) if kind == "e4m3" else y.round().clamp(-127, 127).to(torch.int8)
    return codes, torch.where(finite, (most / PEAK[kind]).float(), math.nan).squeeze(-1)


def code_step(kind, x, scale):
    """How far a code's value may be from x: half a step of the format, and what the scale's and
    the product's F32 roundings move (three of the value)."""
    x = x.abs()
    half = torch.maximum(x * 2.0 ** -4, scale[..., None] * 2.0 ** -10) if kind == "e4m3" else scale[..., None].expand_as(x) / 2
    return half * (1 + 2.0 ** -20) + 3 * 2.0 ** -24 * x


def make_pages(kind, pages, heads, page, dim, token_major=False, stale=None, seed=0, device="cuda"):
    """Tensors of a cache: random codes and scales (`stale`: every scale and, for E4M3, every code
    NaN instead, as memory that nothing has written may hold)."""
    g = torch.Generator(device=device)
    g.manual_seed(seed)
    shape = (pages, page, heads, dim) if token_major else (pages, heads, page, dim)

    def codes():
        if stale:
            bits = torch.full(shape, 0x7f, dtype=torch.int8, device=device)
        else:
            bits = torch.randint(-126, 127, shape, generator=g, dtype=torch.int8, device=device)
            bits = torch.where(bits == -1, 3, bits).to(torch.int8)
        return (bits.permute(0, 2, 1, 3) if token_major else bits).view(CODES[kind])

    def scales():
        if stale:
            return torch.full((pages, heads, page), math.nan, device=device)
        return 0.02 * (0.1 + torch.rand(pages, heads, page, generator=g, device=device)) / (8 if kind == "e4m3" else 1)

    return dict(keys=codes(), values=codes(), key_scales=scales(), value_scales=scales())


def fill(cache, kind, table, lengths, seed=1, spread=0.0):
    """Writes random positions into the cache's pages at every row's first `lengths` positions; the
    rest is left. `spread`: value scales spread over e^-spread .. e^spread."""
    heads, page, dim = cache["keys"].shape[1:]
    g = torch.Generator(device=cache["keys"].device)
    g.manual_seed(seed)
    for r, n in enumerate(lengths):
        n = min(max(n, 0), table.shape[1] * page)
        for name in ("keys", "values"):
            x = torch.randn(n, heads, dim, generator=g, device=table.device)
            if name == "values" and spread:
                x = x * ((2 * torch.rand(n, heads, 1, generator=g, device=table.device) - 1) * spread).exp()
            codes, scale = quantised(x, kind)
            at = torch.arange(n, device=table.device)
            ids = table[r].long()[at // page]
            here = (ids >= 0) & (ids < cache["keys"].shape[0])
            ids, at = ids[here], at[here]
            cache[name].view(torch.int8).permute(0, 2, 1, 3)[ids, at % page] = codes[here].view(torch.int8)
            cache[name[:-1] + "_scales"].permute(0, 2, 1)[ids, at % page] = scale[here]


def attended(q, cache, table, lengths, scale, max_length=1 << 31, exact_dots=False):
    """(outputs in 64 bits, the bound of the kernel's error, element by element); rows of negative
    lengths are NaN. `exact_dots`: q . k has no rounding (small whole numbers).

    A weight w_i = p_i s_i enters the products with half a step of F16 (2^-11; two F16 parts of
    F32 tensors: 2^-22) or, below F16's normal range, 2^-25 of the largest weight; p is off by what its
    score is: q's elements below F16's normal range by 2^-25 of the largest (2^-22 of each for two
    parts), dim + 4 roundings of the sum of |q k|, 2 ulp of exp2 and 4 roundings of the score (base
    2) itself, in the numerator and in the sum alike. Sums over positions round at most once for
    each 32 positions and 64 times in all joins; a term counts with its magnitude."""
    rows, q_heads, dim = q.shape
    pages, heads, page = cache["key_scales"].shape
    out = torch.full(q.shape, math.nan, dtype=torch.float64, device=q.device)
    off = torch.zeros_like(out)
    two = q.dtype == torch.float32
    for r in range(rows):
        n = min(int(lengths[r]), max_length, table.shape[1] * page)
        if n < 0:
            continue
        at = torch.arange(n, device=q.device)
        ids = table[r].long()[at // page]
        here = (ids >= 0) & (ids < pages)
        ids, at = ids[here], at[here] % page
        if len(at) == 0:
            out[r] = 0
            continue

        def values(name):
            codes = cache[name].view(torch.int8).permute(0, 2, 1, 3)[ids, at].view(cache[name].dtype).double()
            return codes, cache[name[:-1] + "_scales"].permute(0, 2, 1)[ids, at].double()

        (kc, ks), (vc, vs) = values("keys"), values("values")
        group = q_heads // heads
        qd = q[r].double().view(heads, group, dim)
        k = (kc * ks[..., None]).permute(1, 2, 0)                        # [heads, dim, n]
        v, w = (vc * vs[..., None]).transpose(0, 1), vs.t()[:, None, :]  # [heads, n, dim]
        score = qd @ k * scale
        p = torch.softmax(score, -1)
        o = p @ v
        size = (qd.abs() @ k.abs()) * abs(scale)
        lost = (qd.abs().amax(-1, keepdim=True) * k.abs().sum(1)[:, None, :]) * abs(scale) * 2.0 ** -25
        rounding = 2.0 ** -22 if two else 2.0 ** -11
        e = lost + size * ((dim + 4) * 2.0 ** -24 + (2.0 ** -22 if two else 0.0))
        if exact_dots:
            e = torch.zeros_like(e)
        e = e + 4 * 2.0 ** -24 * (score - score.amax(-1, keepdim=True)).abs() + 4 * 2.0 ** -24 * score.abs().amax(-1, keepdim=True)
        e = e.amax(-1, keepdim=True) + 2.0 ** -22
        total = 2 * e + rounding + (len(at) / 32 + 64) * 2.0 ** -24
        least = (p * w).amax(-1, keepdim=True) * 2.0 ** -25               # of a weight, in the sum's units
        bound = total * (p @ v.abs()) + least * vc.abs().sum(0)[:, None, :]
        out[r] = o.reshape(q_heads, dim)
        off[r] = (bound + HALF_STEP[q.dtype] * (o.abs() + bound)).reshape(q_heads, dim)
        if q.dtype == torch.float16:
            off[r] += 2.0 ** -25  # F16's subnormals
    return out, off
