"""The 4-bit paged cache against plain 64-bit forms (tests/long_context_forms.py, which derives every bound), at the sizes,
layouts and masks where it can go wrong."""
import math

import pytest
import torch

from tests import long_context_forms as forms
from tests import operator_forms
from tests.operator_forms import HALF_STEP, YARN
from tests.test_gpu_operators import EDGES, draw, near, paged, where

pytestmark = pytest.mark.gpu

DTYPES = [torch.float16, torch.bfloat16, torch.float32]
KINDS = ["e2m1", "int4"]


@pytest.fixture(scope="module")
def ops():
    from hllm_amd import operators

    return operators


# ------------------------------------------------------------------ written


def held(cache, name, ids, at):
    """(codes, scales as held) at positions `at` of pages `ids`."""
    codes = forms.unpacked(cache[name].transpose(1, 2)[ids, at], name == "values")
    return codes, cache[name[:-1] + "_scales"].transpose(1, 2)[ids, at]


def check_keys(cache, kind, ids, at, x, off):
    """Codes and scales of vectors x that are known to `off`: any choice that is right for a vector within that distance."""
    codes, scale = held(cache, "keys", ids, at)
    scale = forms.scales4(scale, kind)
    groups, far = x.unflatten(-1, (-1, 32)), off.unflatten(-1, (-1, 32)).amax(-1)
    most = groups.abs().amax(-1)
    if kind == "e2m1":  # the smallest power of two that leaves the largest magnitude at most 7
        assert (most - far <= 7 * scale).all() and (most + far >= 3.5 * scale).all()
    else:               # a seventh, its eight upper bits kept; the division's rounding
        seventh = 2.0 ** -23 * most / 7
        assert (scale <= (most + far) / 7 + seventh).all() and (scale >= (most - far) / 7 * (1 - 2.0 ** -7) - seventh).all()
    got = forms.numbers4(codes, kind).unflatten(-1, (-1, 32)) * scale[..., None]
    y = groups.abs() / scale[..., None]
    if kind == "e2m1":  # half a step: of 1/2 below 2, of 1 below 4, of 2 from there on
        step = torch.where(y < 2.25, 0.25, torch.where(y < 4.5, 0.5, 1.0))
    else:               # half a scale; 7 stands for up to 7 + 2^-7 * 7 of it, and x / scale is rounded three times
        step = torch.where(y > 7, (y - 7).clamp_min(0.5), 0.5) + 3 * 2.0 ** -24 * y
    # A value within `off` of a border may lie on either side of it.
    assert ((got - groups).abs() <= step * scale[..., None] + 2 * far[..., None]).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,heads,dim,page,token_major,rotary,interleaved", [
    (1, 8, 128, 64, False, 128, False), (33, 4, 256, 16, True, 64, True), (130, 1, 64, 8, False, 20, False),
    (5, 3, 128, 32, True, 0, False), (700, 2, 64, 128, False, 64, False), (2, 5, 256, 4096, False, 256, False),
    (40, 6, 128, 16, False, 48, False), (9, 2, 256, 16, True, 80, False), (17, 9, 64, 8, True, 6, True)])
def test_kv_append(ops, kind, dtype, rows, heads, dim, page, token_major, rotary, interleaved):
    count = rows // page + 3
    cache = forms.make_pages(kind, count, heads, page, dim, token_major)
    before = {n: x.clone() for n, x in cache.items()}
    pages = ops.Kv4Pages(**cache)
    g = torch.Generator(device="cuda")
    g.manual_seed(5)
    slots = torch.randperm(count * page, generator=g, device="cuda")[:rows].int()
    padding = torch.arange(rows, device="cuda") % 3 == 1
    bad = torch.tensor([-1, count * page, -2 ** 31, 2 ** 31 - 1], device="cuda", dtype=torch.int32)
    slots[padding] = bad[torch.arange(int(padding.sum()), device="cuda") % 4]
    q, k, v = draw(rows, heads * 3, dim, dtype, 1), draw(rows, heads, dim, dtype, 2), draw(rows, heads, dim, dtype, 3, 0.1)
    k[0, 0] *= 100 if dtype != torch.float16 else 10
    v[0, heads - 1] = 0
    at = where(rows)
    if rotary:
        plan = ops.Rope(rotary, theta=1e4, interleaved=interleaved, scaling=YARN)
        q_out = torch.full_like(q, 9.0)
        assert ops.kv_append(pages, slots, k, v, q=q, rope=plan, positions=at, q_out=q_out) is q_out
        assert torch.equal(q_out[~padding], ops.rope(plan, at, q)[~padding]) and (q_out[padding] == 9).all()
        key, off = operator_forms.rotated(k, at, rotary, 1e4, interleaved, YARN)
    else:
        assert ops.kv_append(pages, slots, k, v) is None
        key, off = k.double(), torch.zeros_like(k, dtype=torch.float64)
    here = slots[~padding].long()
    ids, p = here // page, here % page
    codes, scale = held(cache, "values", ids, p)
    expect_codes, expect_scale = forms.quantised4(v[~padding], kind)
    assert torch.equal(codes, expect_codes) and torch.equal(scale, expect_scale)
    check_keys(cache, kind, ids, p, key[~padding], off[~padding])
    if not rotary:
        codes, scale = held(cache, "keys", ids, p)
        expect_codes, expect_scale = forms.quantised4(k[~padding], kind)
        assert torch.equal(codes, expect_codes) and torch.equal(scale, expect_scale)
    # Nothing else of the cache changed.
    left = torch.ones(count * page, dtype=torch.bool, device="cuda")
    left[here] = False
    left = left.view(count, page)
    for name in cache:
        assert torch.equal(cache[name].transpose(1, 2)[left], before[name].transpose(1, 2)[left])


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_kv_append_of_extreme_values(ops, kind, dtype):
    """Zero, tiny, huge, infinite and NaN elements: their groups of the last two read back as NaN, the rest by the rule."""
    top = torch.finfo(dtype).max
    x = draw(8, 2, 64, dtype, 1)
    x[0] = 0
    x[1] = torch.finfo(dtype).tiny
    x[2, :, 5] = top
    x[2, :, 6] = -top
    x[3, 0, 63] = math.inf
    x[4, 1, 0] = -math.inf
    x[5, 0, 17] = math.nan
    x[6] = top
    x[7, 1, 40] = math.inf
    pages = ops.Kv4Pages.empty(kind, 2, 2, 8, 64)
    slots = torch.arange(8, dtype=torch.int32, device="cuda") + 3
    ops.kv_append(pages, slots, x, x)
    codes, scale = forms.quantised4(x, kind)
    k, v = ops.kv_read(pages, slots, torch.float32)
    expect = (forms.numbers4(codes, kind) * forms.scales4(scale, kind).repeat_interleave(32, -1)).float()
    for got in (k, v):
        assert torch.equal(torch.isnan(got), torch.isnan(expect)) and not torch.isinf(got).any()
        assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(expect))
    for r, h, group in ((3, 0, 1), (4, 1, 0), (5, 0, 0), (7, 1, 1)):
        assert torch.isnan(k[r, h].view(2, 32)[group]).all() and not torch.isnan(k[r, h].view(2, 32)[1 - group]).any()
        assert not torch.isnan(k[r, 1 - h]).any()


@pytest.mark.parametrize("kind", KINDS)
def test_codes_at_every_border(ops, kind):
    """Halfway between codes, a step of F32 to either side, and largest magnitudes around the scales' borders."""
    x = torch.zeros(4096, 1, 64)
    borders = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0] if kind == "e2m1" else [i + 0.5 for i in range(7)]
    values = [0.0]
    for b in borders:
        for s in (1, -1):
            values += [s * b, s * (b + b * 2.0 ** -23), s * (b - b * 2.0 ** -23)]
    g = torch.Generator().manual_seed(3)
    picks = torch.tensor(values)[torch.randint(0, len(values), x.shape, generator=g)]
    top = 6.0 if kind == "e2m1" else 7.0
    exponents = torch.randint(-90, 90, (4096, 1, 1), generator=g).double()
    largest = torch.tensor([top, 3.75, 7.0, 7.0 - 2.0 ** -21, 7.0 + 2.0 ** -21, 3.5, 3.5 + 2.0 ** -22, 6.999])
    picks[:, 0, 3::32] = largest[torch.randint(0, 8, (4096, 2), generator=g)]
    x = (picks.double() * 2.0 ** exponents).float().cuda()
    pages = ops.Kv4Pages.empty(kind, 64, 1, 64, 64)
    ops.kv_append(pages, torch.arange(4096, dtype=torch.int32, device="cuda"), x, -x)
    for name, y in (("keys", x), ("values", -x)):
        codes, scale = forms.quantised4(y, kind)
        got, got_scale = forms.unpacked(getattr(pages, name), name == "values"), getattr(pages, name[:-1] + "_scales")
        assert torch.equal(got_scale.view(4096, 1, 2), scale)
        got = got.view(4096, 1, 64)
        assert torch.equal(forms.numbers4(got, kind), forms.numbers4(codes, kind))


# ------------------------------------------------------------------ read back


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,heads,dim,page,token_major", [
    (1, 8, 128, 64, False), (61, 3, 64, 8, True), (1000, 1, 256, 16, False), (17, 5, 128, 32, True)])
def test_kv_read(ops, kind, dtype, rows, heads, dim, page, token_major):
    cache = forms.make_pages(kind, 9, heads, page, dim, token_major)
    if kind == "e2m1":
        cache["key_scales"][2] = 0      # 2^-127
        cache["value_scales"][3, 0] = 255
    else:
        cache["value_scales"][3, 0] = math.inf
        cache["key_scales"][4] *= -1
    pages = ops.Kv4Pages(**cache)
    g = torch.Generator(device="cuda")
    g.manual_seed(7)
    slots = torch.randint(0, 9 * page, (rows,), generator=g, device="cuda", dtype=torch.int32)  # repeats too
    slots[0] = 9 * page - 1
    padding = torch.arange(rows, device="cuda") % 5 == 2
    slots[padding] = torch.tensor([-1, 9 * page], device="cuda", dtype=torch.int32)[torch.arange(int(padding.sum()), device="cuda") % 2]
    joint = torch.full((rows, 2 * heads, dim), 3.0, dtype=dtype, device="cuda")
    k, v = ops.kv_read(pages, slots, k_out=joint[:, :heads], v_out=joint[:, heads:])
    ids = slots.long().clamp(0, 9 * page - 1)
    for name, got in (("keys", k), ("values", v)):
        numbers, scale = forms.parts(cache, kind, name)
        expect = (numbers * scale).transpose(1, 2)[ids // page, ids % page].float().to(dtype)  # the product is exact
        assert torch.equal(torch.nan_to_num(got[~padding], nan=5.0), torch.nan_to_num(expect[~padding], nan=5.0))
        assert (got[padding] == 3).all()
    if not padding.any():
        new = ops.kv_read(pages, slots, dtype)
        assert torch.equal(torch.nan_to_num(new[0]), torch.nan_to_num(k)) and torch.equal(torch.nan_to_num(new[1]), torch.nan_to_num(v))


# ------------------------------------------------------------------ attention


def attend_case(ops, kind, dtype, lengths, q_heads, heads, dim, page, token_major=False, stale=True, seed=0, scale=None,
                max_length=None, spread=0.0, q_scale=1.0):
    table, count = paged(lengths, page, seed)
    cache = forms.make_pages(kind, count, heads, page, dim, token_major, stale=stale)
    forms.fill(cache, kind, table, lengths, seed + 1, spread)
    q = draw(len(lengths), q_heads, dim, dtype, seed + 2, q_scale)
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    most = max(max(lengths), 0) if max_length is None else max_length
    pages = ops.Kv4Pages(**cache)
    out = torch.full_like(q, 5.0)
    assert ops.kv_attention(q, pages, table, n, most, scale=scale, out=out) is out
    expect, off = forms.attended(q, cache, kind, table, lengths, dim ** -0.5 if scale is None else scale, most)
    left = n < 0
    assert (out[left] == 5).all()
    near(out[~left], expect[~left], off[~left])
    assert (out[n == 0] == 0).all()
    return q, pages, table, n, most, out


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("q_heads,heads,dim,page,token_major", [
    (16, 8, 128, 64, False), (32, 8, 64, 32, True), (15, 3, 256, 16, False), (32, 1, 128, 8, True), (8, 8, 64, 8, False),
    (40, 2, 256, 128, True)])
def test_kv_attention_at_tile_edges(ops, kind, dtype, q_heads, heads, dim, page, token_major):
    attend_case(ops, kind, dtype, EDGES + [255, 256, 257, 300], q_heads, heads, dim, page, token_major)


@pytest.mark.parametrize("kind,dtype,dim", [("e2m1", torch.float16, 128), ("int4", torch.bfloat16, 256), ("e2m1", torch.float32, 64),
                                            ("int4", torch.float16, 64), ("e2m1", torch.bfloat16, 256), ("int4", torch.float32, 128)])
@pytest.mark.parametrize("lengths", [[1], [100], [5000], [9000, 3, 0, 1025], [16411], [129] * 70, [2048, -1, 40] * 9,
                                     [600] * 3 + [0, -1] * 70 + [513, 1], [700, 20] * 280])
def test_kv_attention_split_and_joined(ops, kind, dtype, dim, lengths):
    attend_case(ops, kind, dtype, lengths, 8, 2, dim, 16)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("dtype", DTYPES)
def test_kv_attention_of_peaked_scores_and_uneven_values(ops, dim, dtype):
    """Scores tens apart, value scales over nine powers of ten."""
    for kind, scale in (("e2m1", 0.5), ("int4", -0.5)):
        attend_case(ops, kind, dtype, [300, 1, 2000], 4, 2, dim, 32, scale=scale, spread=10.0, seed=11)
        attend_case(ops, kind, dtype, [300, 1, 2000], 4, 2, dim, 32, scale=0.0, spread=10.0, seed=12)


@pytest.mark.parametrize("dtype,q_scale", [(torch.bfloat16, 1e30), (torch.float32, 1e-30), (torch.float16, 1000.0), (torch.float32, 0.0)])
@pytest.mark.parametrize("kind", KINDS)
def test_kv_attention_of_large_and_small_queries(ops, kind, dtype, q_scale):
    attend_case(ops, kind, dtype, [70, 400], 8, 2, 128, 64, q_scale=q_scale, scale=0.05 / max(q_scale, 1e-30))


# ------------------------------------------------------------------ numbers that are none, masks, sizes


def cut(ops, pages, lengths, q_heads, most):
    """Whether a call with these rows cuts pairs (a call that does not has no workspace)."""
    return ops.kv_attention_workspace(pages, len(lengths), q_heads, most) > 0


def not_finite(kind, x):
    """The scale that stands for NaN, in scales x as held."""
    return 255 if kind == "e2m1" else math.nan


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_nan_stays_nan_where_work_is_cut(ops, kind, dtype, dim):
    """A NaN in a query or in key scales makes that head's (or KV head's) output NaN; in value scales, their groups' elements; and
    nothing else, at bounds of the lengths that cut a row and that do not."""
    lengths, page = [5000, 40, 3000], 64
    table, count = paged(lengths, page)
    cache = forms.make_pages(kind, count, 2, page, dim)
    pages = ops.Kv4Pages(**cache)
    q = draw(3, 8, dim, dtype, 1)
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    assert cut(ops, pages, lengths, 8, 5000) and not cut(ops, pages, lengths, 8, 300)

    def check(q, bad):
        for most in (5000, 2048, 300):
            out = ops.kv_attention(q, pages, table, n, most)
            assert torch.equal(torch.isnan(out), bad.expand_as(out)), most

    bad = torch.zeros(3, 8, 1, dtype=torch.bool, device="cuda")
    check(q, bad)
    wrong = q.clone()
    wrong[0, 3, 9] = math.nan
    wrong[1, 7, 0] = math.nan
    wrong[2] = math.nan
    bad[0, 3] = bad[1, 7] = bad[2] = True
    check(wrong, bad)
    before = {x: cache[x].clone() for x in ("key_scales", "value_scales")}
    cache["key_scales"][table[0].long(), 1, :, 1] = not_finite(kind, None)
    cache["key_scales"][table[2, 2].long(), 0, 5:9, 0] = not_finite(kind, None)
    if kind == "int4":
        cache["key_scales"][table[1, 0].long(), 0, 7, 1] = -math.inf
    bad[:] = False
    bad[0, 4:] = bad[2, :4] = True
    bad[1, :4] = kind == "int4"
    check(q, bad)
    cache["key_scales"].copy_(before["key_scales"])
    bad = torch.zeros(3, 8, dim, dtype=torch.bool, device="cuda")
    cache["value_scales"][table[0, 1].long(), 1, 3, 1] = not_finite(kind, None)
    cache["value_scales"][table[2, 0].long(), 0] = not_finite(kind, None)
    bad[0, 4:, 32:64] = bad[2, :4] = True
    # The position's own value has no group left that is a number: NaN still, of the whole vector, and of no other position's.
    check(q, bad)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("infinity", [math.inf, -math.inf])
def test_infinite_queries_give_nan(ops, kind, dtype, infinity):
    """Scores that are all infinite, of either sign, have no softmax: NaN, whether a row is cut or not; rows
    without positions stay zeros."""
    lengths, page = [5000, 40, 0, 700], 32
    table, count = paged(lengths, page)
    table[3] = -1
    cache = forms.make_pages(kind, count, 2, page, 128)
    cache["keys"][..., 4] = 0x33 if kind == "e2m1" else 0xbb  # elements 8 and 9: positive numbers
    pages = ops.Kv4Pages(**cache)
    q = draw(4, 8, 128, dtype, 1)
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    assert cut(ops, pages, lengths, 8, 5000) and not cut(ops, pages, lengths, 8, 300)
    for most in (5000, 300):
        clean = ops.kv_attention(q, pages, table, n, most)
        assert not torch.isnan(clean).any()
        wrong = q.clone()
        wrong[:, 2, 9] = infinity
        out = ops.kv_attention(wrong, pages, table, n, most)
        assert torch.isnan(out[:2, 2]).all() and (out[2:] == 0).all()
        out[:, 2] = clean[:, 2] = 0
        assert torch.equal(out, clean)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_values_near_the_largest_number(ops, kind, dtype, dim):
    """Means of values up to 1.3e38 are finite, though sums of three of them are not."""
    lengths, page = [5000, 300, 2, 9000], 32
    table, count = paged(lengths, page)
    cache = forms.make_pages(kind, count, 2, page, dim)
    if kind == "e2m1":
        cache["values"].copy_(cache["values"] & 0x77 | 0x44)     # 2 .. 6
        cache["value_scales"].fill_(127 + 124)                     # times 2.1e37
    else:
        cache["values"].copy_(cache["values"] & 0x33 | 0xcc)     # 4 .. 7
        cache["value_scales"].copy_((0.5 + cache["value_scales"]) * 1.8e37)
    q = draw(4, 8, dim, dtype, 1)
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    pages = ops.Kv4Pages(**cache)
    assert cut(ops, pages, lengths, 8, 9000)
    for most in (9000, 300):
        expect, off = forms.attended(q, cache, kind, table, lengths, dim ** -0.5, most)
        assert expect.max() > 6e37
        near(ops.kv_attention(q, pages, table, n, most), expect, off)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("kind", KINDS)
def test_groups_of_very_different_scales(ops, kind, dim, dtype):
    """Groups of one vector, and vectors of one row, up to 2^20 and 2^40 apart, in keys and in values; INT4 scales of
    either sign; E2M1's smallest and largest."""
    lengths, page = [300, 1, 2000, 63], 16
    table, count = paged(lengths, page)
    cache = forms.make_pages(kind, count, 2, page, dim)
    g = torch.Generator(device="cuda")
    g.manual_seed(2)

    def exponents(least, most):
        vector = torch.randint(least, most, cache["keys"].shape[:3], generator=g, device="cuda")
        return vector[..., None] + torch.randint(-10, 11, cache["key_scales"].shape, generator=g, device="cuda")

    def held(e):
        if kind == "e2m1":
            return (e + 127).to(torch.uint8)
        sign = torch.randint(0, 2, e.shape, generator=g, device="cuda") * 2 - 1
        return (sign * (1 + torch.rand(e.shape, generator=g, device="cuda")) * 2.0 ** e).to(torch.bfloat16)

    cache["key_scales"].copy_(held(exponents(-14, -12)))
    cache["value_scales"].copy_(held(exponents(-20, 20) - (9 if dtype == torch.float16 else 0)))
    if kind == "e2m1":
        cache["value_scales"][table[0, 3].long(), 0, 2] = 0
        if dtype != torch.float16:
            cache["value_scales"][table[2, 5].long(), 1, 7, 1] = 127 + 125
    q = draw(4, 8, dim, dtype, 1)
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    for scale in (dim ** -0.5, 0.0):
        out = ops.kv_attention(q, ops.Kv4Pages(**cache), table, n, 2000, scale=scale)
        expect, off = forms.attended(q, cache, kind, table, lengths, scale)
        fits = expect.abs() + off < torch.finfo(dtype).max
        assert fits.float().mean() > 0.9
        near(torch.where(fits, out, 0), torch.where(fits, expect, 0.0), off)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_pairs_of_more_than_64_parts(ops, kind, dtype, dim):
    """A pair that most workgroups share, whose first two thirds hold nothing."""
    lengths, page = [300000], 64
    table, count = paged(lengths, page)
    cache = forms.make_pages(kind, count, 1, page, dim, stale=True)
    forms.fill(cache, kind, table, lengths)
    q = draw(1, 4, dim, dtype, 1)
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    pages = ops.Kv4Pages(**cache)
    near(ops.kv_attention(q, pages, table, n, 300000), *forms.attended(q, cache, kind, table, lengths, dim ** -0.5))
    table[0, :3200] = -1
    near(ops.kv_attention(q, pages, table, n, 300000), *forms.attended(q, cache, kind, table, lengths, dim ** -0.5))


@pytest.mark.parametrize("kind,dtype,dim", [("e2m1", torch.float16, 128), ("int4", torch.bfloat16, 256), ("e2m1", torch.float32, 64),
                                            ("int4", torch.float32, 256)])
@pytest.mark.parametrize("lengths", [
    [10000] + [0, -1, 5, 40] * 16, [3, 0] * 32 + [8191], [-1] * 129 + [6000], [130, 1] * 40 + [12000, -1, 7000] + [0] * 47,
    [9000] + [20, -1, 0, 129, 3] * 139 + [-1, 2500, 1, 0], [-1, 64] * 511 + [20000, 9], [0] * 500 + [26000] + [1] * 523,
    ([3, 0, 70, -1, 600] * 220)[:1090]])
def test_shares_of_many_rows(ops, kind, dtype, dim, lengths):
    attend_case(ops, kind, dtype, lengths, 2, 1, dim, 16)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype,dim", [(torch.float16, 64), (torch.bfloat16, 128), (torch.float32, 128), (torch.float16, 256)])
@pytest.mark.parametrize("q_heads,heads", [(20, 1), (40, 2), (17, 1), (64, 1)])
def test_groups_of_more_than_sixteen_heads(ops, kind, dtype, dim, q_heads, heads):
    for lengths in ([5000], [129, 20000, -1, 0, 6400]):
        attend_case(ops, kind, dtype, lengths, q_heads, heads, dim, 32)


@pytest.mark.parametrize("kind", KINDS)
def test_kv_attention_leaves_out_dropped_pages(ops, kind):
    """Positions of pages that are not in the cache count as masked: some of a row's, then all."""
    for page, dim in ((8, 64), (16, 128), (64, 256)):
        lengths = [300, 5, 1000, 640]
        table, count = paged(lengths, page)
        table[0, 1::3] = -1
        table[2, : 1000 // page // 2] = count  # past the cache
        table[2, -1] = 2 ** 31 - 1
        table[3] = -7
        cache = forms.make_pages(kind, count, 2, page, dim, stale=True)
        forms.fill(cache, kind, table, lengths)
        q = draw(4, 6, dim, torch.float16, 1)
        n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        out = ops.kv_attention(q, ops.Kv4Pages(**cache), table, n, 1000)
        near(out, *forms.attended(q, cache, kind, table, lengths, dim ** -0.5))
        assert (out[3] == 0).all()


@pytest.mark.parametrize("kind", KINDS)
def test_page_offsets_past_32_bits(ops, kind):
    """A cache of more than 4 GiB of codes: written, read, bounded and attended at its end."""
    page, heads, dim = 4096, 8, 128
    count = (1 << 32) // (page * heads * dim // 2) + 3
    pages = ops.Kv4Pages.empty(kind, count, heads, page, dim)
    small = ops.Kv4Pages.empty(kind, 3, heads, page, dim)
    rows = 300
    k, v, q = draw(rows, heads, dim, torch.float16, 1), draw(rows, heads, dim, torch.float16, 2), draw(1, 16, dim, torch.float16, 3)
    at = torch.arange(rows, dtype=torch.int32, device="cuda") + page - 100
    ops.kv_append(pages, at + (count - 3) * page, k, v)
    ops.kv_append(small, at, k, v)
    for x, y in zip(ops.kv_read(pages, at + (count - 3) * page), ops.kv_read(small, at)):
        assert torch.equal(x, y)
    n = torch.tensor([page + 200], dtype=torch.int32, device="cuda")
    table = torch.tensor([[0, 1]], dtype=torch.int32, device="cuda")
    assert torch.equal(ops.kv_attention(q, pages, table + count - 3, n, page + 200), ops.kv_attention(q, small, table, n, page + 200))
    a, b = ops.KvBounds.empty(pages), ops.KvBounds.empty(small)
    zero = torch.zeros(1, dtype=torch.int32, device="cuda")
    ops.kv_bounds(pages, a, table + count - 3, zero, n, page + 200)
    ops.kv_bounds(small, b, table, zero, n, page + 200)
    assert torch.equal(a.codes[-3:], b.codes) and torch.equal(a.scales[-3:], b.scales) and b.codes[:2].any(-1).all()


@pytest.mark.parametrize("kind", KINDS)
def test_views(ops, kind):
    """Heads of one projection's rows, strided outputs, rows that repeat memory, a table inside a wider one."""
    lengths, dim = [100, 0, 400, 33], 128
    q, pages, table, n, most, out = attend_case(ops, kind, torch.float16, lengths, 8, 2, dim, 16)
    joint = draw(4, 20, dim, torch.float16, 9)
    joint[:, 3:11] = q
    wide = torch.full((4, 12, dim), 7.0, dtype=torch.float16, device="cuda")
    big = torch.full((4, table.shape[1] + 9), -1, dtype=torch.int32, device="cuda")
    big[:, 2:2 + table.shape[1]] = table
    assert torch.equal(ops.kv_attention(joint[:, 3:11], pages, big[:, 2:2 + table.shape[1]], n, most, out=wide[:, 2:10]), out)
    assert (wide[:, :2] == 7).all() and (wide[:, 10:] == 7).all()
    k = joint[:, 12:14]
    slots = torch.arange(4, dtype=torch.int32, device="cuda") * 5
    fresh, plain = (ops.Kv4Pages.empty(kind, 2, 2, 16, dim) for _ in range(2))
    ops.kv_append(fresh, slots, k, k[:1].expand(4, 2, dim))
    ops.kv_append(plain, slots, k.contiguous(), k[:1].repeat(4, 1, 1))
    for name in ("keys", "values", "key_scales", "value_scales"):
        assert torch.equal(getattr(fresh, name), getattr(plain, name))
