"""Attention over selected pages: the bounds of pages' keys, the selection by their scores and the attention over tables of
each KV head's own, against plain 64-bit forms (tests/long_context_forms.py). Bounds and selections are exact."""
import math

import pytest
import torch

from tests import long_context_forms as forms
from tests.test_gpu_operators import draw, near, paged

pytestmark = pytest.mark.gpu

DTYPES = [torch.float16, torch.bfloat16, torch.float32]
KINDS = ["e4m3", "int8", "e2m1", "int4"]


@pytest.fixture(scope="module")
def ops():
    from hllm_amd import operators

    return operators


def described(ops, kind, cache):
    return (ops.Kv4Pages if kind in forms.FOUR else ops.KvPages)(**cache)


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


# ------------------------------------------------------------------ bounds


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,dim,page,token_major", [
    (8, 128, 16, False), (1, 64, 8, False), (3, 256, 64, True), (2, 64, 128, True), (2, 128, 256, False), (1, 256, 1024, False),
    (5, 64, 4096, True), (3, 128, 8, True)])
def test_bounds(ops, kind, heads, dim, page, token_major):
    lengths = [1, 0, page, page + 1, 3 * page - 1, -1, 5 * page, 2 * page + 5]
    starts = [0, 0, 0, page - 1, page, 0, 5 * page - 1, -3]
    table, count = paged(lengths, page)
    table[6, 4] = -1
    table[7, 1] = count
    cache = forms.make_pages(kind, count, heads, page, dim, token_major, stale=True)
    forms.fill(cache, kind, table, lengths)
    pages = described(ops, kind, cache)
    bounds = ops.KvBounds.empty(pages)
    bounds.codes.fill_(55)
    bounds.scales.fill_(-1.0)
    ops.kv_bounds(pages, bounds, table, ints(starts), ints(lengths), 2 * page + 5)
    made = torch.zeros(count, dtype=torch.bool)
    for r, (start, length) in enumerate(zip(starts, lengths)):
        for p in range(max(start, 0) // page, -(-length // page) if start < length else 0):
            id = int(table[r, p])
            if not 0 <= id < count:
                continue
            made[id] = True
            for h in range(heads):
                codes, scale = forms.bounds_of(cache, kind, id, h, min(page, length - p * page))
                assert torch.equal(bounds.codes[id, h], codes) and bounds.scales[id, h].item() == scale
    assert made.sum() == 8  # 1 + 0 + 1 + 2 + 2 + 0 + 0 + 2 of the rows
    assert (bounds.codes[~made] == 55).all() and (bounds.scales[~made] == -1).all()


@pytest.mark.parametrize("kind", KINDS)
def test_bounds_of_extreme_keys(ops, kind):
    """Zero, tiny, huge and not finite keys; whole pages of one value; what lies behind the length is not looked at."""
    for page in (8, 256):
        heads, dim = 2, 64
        cache = forms.make_pages(kind, 7, heads, page, dim, stale=True)
        x = draw(7 * page, heads, dim, torch.float32, 1).view(7, page, heads, dim)
        x[0] = 0
        x[1] *= 2.0 ** -105
        x[2] *= 1e37
        x[3, 5, 0, 9] = math.nan
        x[4, 7, 1, 60] = -math.inf
        x[5] = 1.5
        for id in range(6):
            forms.hold(cache, kind, "keys", torch.full((page,), id, device="cuda"), torch.arange(page, device="cuda"), x[id])
        n = page - 3
        forms.hold(cache, kind, "keys", torch.full((n,), 6, device="cuda"), torch.arange(n, device="cuda"), x[6, :n])
        pages = described(ops, kind, cache)
        bounds = ops.KvBounds.empty(pages)
        table = torch.arange(7, dtype=torch.int32, device="cuda")[None]
        ops.kv_bounds(pages, bounds, table, ints([0]), ints([7 * page - 3]), 7 * page)
        for id in range(7):
            for h in range(heads):
                codes, scale = forms.bounds_of(cache, kind, id, h, n if id == 6 else page)
                assert torch.equal(bounds.codes[id, h], codes), (id, h)
                assert bounds.scales[id, h].item() == scale or (math.isnan(scale) and torch.isnan(bounds.scales[id, h]))
        assert torch.isnan(bounds.scales[3, 0]) and not torch.isnan(bounds.scales[3, 1]) and torch.isnan(bounds.scales[4, 1])


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim,page,places", [(128, 16, 9), (64, 8, 1100), (128, 256, 5), (256, 64, 7)])
def test_bounds_of_the_largest_keys(ops, kind, dim, page, places):
    """Keys up to the largest numbers of BF16 and F32, as they are written, and scales that a caller's own cache may hold beside
    small codes: finite where reading back is. A wave, a slot, and a workgroup for a page and KV head."""
    heads, rows = 2, 4
    assert rows * places * heads >= 8192 or places < 10
    table = torch.randperm(rows * places, generator=torch.Generator("cuda").manual_seed(1), device="cuda").int().view(rows, places)
    cache = forms.make_pages(kind, rows * places, heads, page, dim)
    most = torch.finfo(torch.float32).max
    at = torch.arange(page, device="cuda")
    x = draw(6 * page, heads, dim, torch.float32, 2).clamp(-1, 1).view(6, page, heads, dim)
    x[0] *= most
    x[1] *= torch.finfo(torch.bfloat16).max
    x[2, 3, 1, 40] = 3.2e38
    x[3, :, :, 32:] *= -2.99e38
    x[4, 1] *= 2.95e38
    for r in range(3):
        for p in range(min(places, 12)):
            forms.hold(cache, kind, "keys", table[r, p].long().expand(page), at, x[(r + p) % 6])
    last = table[3].long()
    if kind in forms.FOUR:  # codes of -1, 0 and 1, or of 0 to 1
        cache["keys"][last] = torch.randint(0, 3, cache["keys"][last].shape, device="cuda", dtype=torch.uint8) * 0x11 + (0x77 if kind == "int4" else 0)
        cache["key_scales"][last] = 254 if kind == "e2m1" else 3.3e38
    else:
        cache["keys"][last] = torch.randint(0, 2, cache["keys"][last].shape, device="cuda").to(cache["keys"].dtype)
        cache["key_scales"][last] = 3.3e38
    pages = described(ops, kind, cache)
    bounds = ops.KvBounds.empty(pages)
    lengths = [page * places, page * places - 3, page * places, page * places]
    ops.kv_bounds(pages, bounds, table, ints([0] * rows), ints(lengths), page * places)
    for r in range(rows):
        for p in (*range(min(places, 6)), places - 1):
            id, count = int(table[r, p]), min(page, lengths[r] - p * page)
            k, _ = ops.kv_read(pages, ints(list(range(id * page, id * page + count))), torch.float32)
            for h in range(heads):
                codes, scale = forms.bounds_of(cache, kind, id, h, count)
                finite = bool(torch.isfinite(k[:, h]).all())
                # INT8: 127 times a 127th of the largest number, rounded, may be past it, in reading back too.
                assert math.isfinite(scale) == finite and (finite or kind == "int8")
                assert torch.equal(bounds.codes[id, h], codes), (r, p, h)
                assert bounds.scales[id, h].item() == scale or not finite and torch.isnan(bounds.scales[id, h])


# ------------------------------------------------------------------ selection


def random_bounds(ops, pages, seed=0, ties=False):
    """Bounds as a cache's keys leave them; `ties`: of a few different pages only."""
    bounds = ops.KvBounds.empty(pages)
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    n, heads, _, dim = bounds.codes.shape
    codes = torch.randint(-127, 128, (6 if ties else n, heads, 2, dim), generator=g, device="cuda").sort(2, descending=True).values
    scales = 2.0 ** torch.randint(-8, -5, codes.shape[:2], generator=g, device="cuda").float()
    pick = torch.randint(0, 6, (n,), generator=g, device="cuda") if ties else torch.arange(n, device="cuda")
    bounds.codes.copy_(codes[pick])
    bounds.scales.copy_(scales[pick])
    return bounds


def select_case(ops, dtype, lengths, q_heads, heads, dim, page, keep, first=1, last=1, ties=False, max_length=None, width=None, seed=0,
                change=None):
    table, count = paged(lengths, page, seed, width=width)
    pages = ops.KvPages(**forms.make_pages("int8", count, heads, page, dim))
    bounds = random_bounds(ops, pages, seed, ties)
    q = draw(len(lengths), q_heads, dim, dtype, seed + 2)
    if change:
        change(q, bounds, table)
    most = max(max(lengths), 0) if max_length is None else max_length
    into = torch.full((len(lengths), heads, keep), -7, dtype=torch.int32, device="cuda")
    got, n = ops.kv_select(q, bounds, table, ints(lengths), most, keep, first=first, last=last, selected=into)
    assert got is into
    expect, expect_n = forms.selected(q, bounds.codes, bounds.scales, table, lengths, page, keep, first, last, most)
    assert torch.equal(n.cpu(), expect_n)
    assert torch.equal(got.cpu(), expect)
    return q, bounds, table, most, got, n


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("q_heads,heads,dim,page", [(32, 8, 128, 16), (8, 2, 64, 8), (15, 3, 256, 64), (20, 1, 128, 8), (40, 1, 64, 16), (4, 4, 256, 8)])
@pytest.mark.parametrize("keep,first,last", [(1, 0, 1), (5, 1, 2), (16, 0, 1), (33, 2, 3), (200, 1, 1)])
@pytest.mark.parametrize("ties", [False, True])
def test_selection(ops, dtype, q_heads, heads, dim, page, keep, first, last, ties):
    lengths = [page * keep, page * keep + 1, page * 70 - 3, 1, 0, -1, page, 40 * page, page * 129 + 1]
    select_case(ops, dtype, lengths, q_heads, heads, dim, page, keep, first, last, ties)


@pytest.mark.parametrize("ties", [False, True])
@pytest.mark.parametrize("length,keep", [(8 * 4096, 300), (8 * 4096 + 1, 300), (8 * 9001, 1), (8 * 12288, 4500), (8 * 5000 - 3, 4999)])
def test_selection_of_many_pages(ops, ties, length, keep):
    """More pages than a workgroup holds, on either side of the border."""
    select_case(ops, torch.float16, [length, 77, 8 * 4500, -1, 0], 4, 2, 64, 8, keep, 0 if keep == 1 else 1, 1, ties)


@pytest.mark.parametrize("dtype", DTYPES)
def test_scores_that_are_no_numbers(ops, dtype):
    """NaN pages and queries are above all others, pages outside the cache below them; infinite and zero queries."""
    def change(q, bounds, table):
        bounds.scales[table[0, 5].long(), 0] = math.nan
        bounds.scales[table[0, 9:12].long(), 1] = math.nan
        q[1, 0, 3] = math.nan
        q[2, 5, 7] = math.inf
        q[3] = 0
        q[4] *= -2.0 ** -10
        table[4, 3:30] = -1
        table[5, ::2] = bounds.pages
        table[6, 1:] = -9

    for keep in (4, 17, 30):
        q, bounds, table, most, got, n = select_case(ops, dtype, [16 * 40 - 1] * 7, 8, 2, 64, 16, keep, 1, 1, change=change)
        assert (got[0, 0] == table[0, 5]).any() and all((got[0, 1] == table[0, p]).any() for p in (9, 10))


def test_selection_counts_the_bounds_that_it_states(ops):
    """Lengths past max_length and past the table."""
    for most in (0, 1, 16 * 20, 16 * 33 + 5, 1 << 40):
        table, count = paged([16 * 50] * 3, 16)
        pages = ops.KvPages(**forms.make_pages("int8", count, 2, 16, 64))
        bounds, q = random_bounds(ops, pages), draw(3, 4, 64, torch.float16, 1)
        lengths = [16 * 50, 16 * 45 + 1, 2 ** 31 - 1]
        got, n = ops.kv_select(q, bounds, table, ints(lengths), most, 12)
        expect, expect_n = forms.selected(q, bounds.codes, bounds.scales, table, lengths, 16, 12, 1, 1, most)
        assert torch.equal(got.cpu(), expect) and torch.equal(n.cpu(), expect_n)


def test_selection_does_not_depend_on_the_rows_beside_it(ops):
    q, bounds, table, most, got, n = select_case(ops, torch.bfloat16, [16 * 300, 16 * 200 + 1, 16 * 41] * 5, 32, 8, 128, 16, 40)
    for r in (0, 7, 14):
        alone, m = ops.kv_select(q[r:r + 1], bounds, table[r:r + 1], ints([[16 * 300, 16 * 200 + 1, 16 * 41][r % 3]]), most, 40)
        assert torch.equal(alone[0], got[r]) and torch.equal(m, n[r:r + 1])


# ------------------------------------------------------------------ attention over tables by head


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("q_heads,heads,dim,page,lengths", [
    (16, 8, 128, 16, [1, 40, 0, -1, 300]), (20, 1, 64, 8, [700, 129]), (6, 3, 256, 64, [5000, 20]), (8, 2, 128, 32, [6000] * 3)])
def test_attention_by_head(ops, kind, dtype, q_heads, heads, dim, page, lengths):
    width = max(-(-n // page) for n in lengths)
    count = len(lengths) * heads * width + 3
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    table = torch.randperm(count, generator=g, device="cuda")[:len(lengths) * heads * width].int().view(len(lengths), heads, width)
    table[-1, heads - 1, 0] = -1
    cache = forms.make_pages(kind, count, heads, page, dim)
    pages = described(ops, kind, cache)
    q = draw(len(lengths), q_heads, dim, dtype, 4)
    n = ints(lengths)
    wide = torch.full((len(lengths), heads + 1, width + 5), count, dtype=torch.int32, device="cuda")
    wide[:, :heads, :width] = table
    out = ops.kv_attention(q, pages, table, n, max(lengths))
    expect, off = forms.attended(q, cache, kind, table, lengths, dim ** -0.5)
    live = n >= 0
    near(out[live], expect[live], off[live])
    assert torch.equal(ops.kv_attention(q, pages, wide[:, :heads, :width], n, max(lengths))[live], out[live])
    same = table[:, :1].expand(len(lengths), heads, width)
    assert torch.equal(ops.kv_attention(q, pages, same, n, max(lengths))[live],
                       ops.kv_attention(q, pages, table[:, 0], n, max(lengths))[live])


# ------------------------------------------------------------------ together


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_requests_served_over_selected_pages(ops, kind, dtype):
    """Prompts are written, then steps of one token a row: each step's selection and attention equal the plain forms over
    the cache as it is; with room for all pages, attention over all of them."""
    heads, q_heads, dim, page, keep, width = 2, 8, 64, 8, 6, 20
    lengths, rows = [70, 8, 1, 41], 4
    table = torch.randperm(rows * width, generator=torch.Generator("cuda").manual_seed(1), device="cuda").int().view(rows, width)
    cls = ops.Kv4Pages if kind in forms.FOUR else ops.KvPages
    pages = cls.empty(kind, rows * width, heads, page, dim)
    bounds = ops.KvBounds.empty(pages)
    plan = ops.Rope(dim, theta=1e4)
    cache = {x: getattr(pages, x) for x in ("keys", "values", "key_scales", "value_scales")}

    def slots_of(r, p):
        return table[r].long()[p // page] * page + p % page

    prompts = [(r, p) for r in range(rows) for p in range(lengths[r])]
    slots = ints([int(slots_of(r, p)) for r, p in prompts])
    k, v = draw(len(prompts), heads, dim, dtype, 1), draw(len(prompts), heads, dim, dtype, 2)
    ops.kv_append(pages, slots, k, v, rope=plan, positions=ints([p for _, p in prompts]))
    ops.kv_bounds(pages, bounds, table, ints([0] * rows), ints(lengths), max(lengths))
    for step in range(20):
        at = ints(lengths)
        slots = ints([int(slots_of(r, p)) for r, p in enumerate(lengths)])
        q, k, v = (draw(rows, h, dim, dtype, 10 * step + i) for i, h in enumerate((q_heads, heads, heads)))
        q = ops.kv_append(pages, slots, k, v, q=q, rope=plan, positions=at)
        lengths = [n + 1 for n in lengths]
        n = ints(lengths)
        ops.kv_bounds(pages, bounds, table, at, n, 1)
        picked, m = ops.kv_select(q, bounds, table, n, width * page, keep, first=1, last=2)
        expect, expect_m = forms.selected(q, bounds.codes, bounds.scales, table, lengths, page, keep, 1, 2)
        assert torch.equal(picked.cpu(), expect) and torch.equal(m.cpu(), expect_m)
        out = ops.kv_attention(q, pages, picked, m, keep * page)
        near(out, *forms.attended(q, cache, kind, picked, m.tolist(), dim ** -0.5))
        everything, m = ops.kv_select(q, bounds, table, n, width * page, width)
        assert torch.equal(ops.kv_attention(q, pages, everything, m, width * page), ops.kv_attention(q, pages, table, n, width * page))
    for r, length in enumerate(lengths):
        for p in range(-(-length // page)):
            id = int(table[r, p])
            for h in range(heads):
                codes, scale = forms.bounds_of(cache, kind, id, h, min(page, length - p * page))
                assert torch.equal(bounds.codes[id, h], codes) and bounds.scales[id, h].item() == scale
