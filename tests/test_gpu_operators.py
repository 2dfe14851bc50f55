"""The operators on device memory against plain 64-bit forms (tests/operator_forms.py, which
derives every bound), at the sizes, layouts and masks where they can go wrong."""
import ctypes as C
import math

import pytest
import torch

from hllm_amd import capi
from tests import operator_forms as forms
from tests.operator_forms import HALF_STEP, LLAMA3, YARN

pytestmark = pytest.mark.gpu

DTYPES = [torch.float16, torch.bfloat16, torch.float32]
KINDS = ["e4m3", "int8"]


@pytest.fixture(scope="module")
def ops():
    from hllm_amd import operators

    return operators


def near(got, expect, bound):
    assert got.shape == expect.shape
    assert not torch.isnan(got).any()
    worst = ((got.double() - expect).abs() - bound).max().item() if got.numel() else 0.0
    assert worst <= 0, worst


def draw(rows, heads, dim, dtype, seed, scale=1.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (torch.randn(rows, heads, dim, generator=g, device="cuda") * scale).to(dtype)


def where(rows, seed=3, low=-5, high=1 << 20):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    p = torch.randint(low, high, (rows,), generator=g, device="cuda", dtype=torch.int32)
    p[0] = 0
    if rows > 1:
        p[-1] = 2 ** 31 - 1
    return p


# ------------------------------------------------------------------ rotary positions


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,q_heads,k_heads,dim,rotary", [
    (1, 16, 8, 128, 128), (7, 32, 8, 64, 64), (5, 3, 1, 256, 64), (3, 12, 4, 80, 20), (2, 5, 0, 96, 96), (300, 4, 2, 128, 32),
    (4, 70, 1, 16, 2), (1, 1, 0, 256, 256), (2, 9, 3, 112, 6)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rope(ops, dtype, rows, q_heads, k_heads, dim, rotary, interleaved):
    scaling = {64: YARN, 20: LLAMA3, 32: {"rope_type": "linear", "factor": 4.0}}.get(rotary)
    plan = ops.Rope(rotary, theta=5e5, interleaved=interleaved, scaling=scaling)
    at = where(rows)
    tensors = [draw(rows, h, dim, dtype, i) for i, h in enumerate((q_heads, k_heads)) if h]
    before = [x.clone() for x in tensors]
    got = ops.rope(plan, at, *tensors)
    got = (got,) if k_heads == 0 else got
    for x, was, y in zip(tensors, before, got):
        assert torch.equal(x, was)
        expect, off = forms.rotated(x, at, rotary, 5e5, interleaved, scaling)
        near(y, expect, off + HALF_STEP[dtype] * (expect.abs() + off) + (2.0 ** -25 if dtype == torch.float16 else 0))
        assert torch.equal(y[..., rotary:], x[..., rotary:])
    # In place, the same bits.
    again = [x.clone() for x in tensors]
    ops.rope(plan, at, *again, *([] if k_heads else [None]), q_out=again[0], **({"k_out": again[1]} if k_heads else {}))
    for x, y in zip(again, got):
        assert torch.equal(x, y)


@pytest.mark.parametrize("rotary,interleaved", [(128, False), (20, False), (64, True)])
def test_rope_takes_views(ops, rotary, interleaved):
    """q and k inside one projection's rows, heads outside rows, rows and heads repeated."""
    plan = ops.Rope(rotary, interleaved=interleaved)
    rows, dim, at = 37, 128, where(37)
    joint = draw(rows, 24, dim, torch.float16, 1)
    q, k = joint[:, :16], joint[:, 16:20]
    for x in (k, q.transpose(0, 1).contiguous().transpose(0, 1), q[:1].expand(rows, 16, dim), q[:, :1].expand(rows, 16, dim)):
        expect = ops.rope(plan, at, x.contiguous())
        assert torch.equal(ops.rope(plan, at, x), expect)
    wide = torch.full((rows, 40, dim), 7.0, dtype=torch.float16, device="cuda")
    a, b = ops.rope(plan, at, q, k, q_out=wide[:, 4:20], k_out=wide[:, 30:34])
    assert torch.equal(a, ops.rope(plan, at, q.contiguous())) and torch.equal(b, ops.rope(plan, at, k.contiguous()))
    assert (wide[:, :4] == 7).all() and (wide[:, 20:30] == 7).all() and (wide[:, 34:] == 7).all()


def test_rope_of_no_rows(ops):
    empty = torch.empty(0, 4, 64, dtype=torch.float16, device="cuda")
    assert ops.rope(ops.Rope(64), torch.empty(0, dtype=torch.int32, device="cuda"), empty).shape == empty.shape


# ------------------------------------------------------------------ the cache, written


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,heads,dim,page,token_major,rotary,interleaved", [
    (1, 8, 128, 64, False, 128, False), (33, 4, 256, 16, True, 64, True), (130, 1, 64, 8, False, 20, False),
    (5, 3, 128, 32, True, 0, False), (700, 2, 64, 128, False, 64, False), (2, 5, 256, 4096, False, 256, False)])
def test_kv_append(ops, kind, dtype, rows, heads, dim, page, token_major, rotary, interleaved):
    count = rows // page + 3
    cache = forms.make_pages(kind, count, heads, page, dim, token_major)
    before = {n: x.clone() for n, x in cache.items()}
    pages = ops.KvPages(**cache)
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
        key, off = forms.rotated(k, at, rotary, 1e4, interleaved, YARN)
    else:
        assert ops.kv_append(pages, slots, k, v) is None
        key, off = k.double(), torch.zeros_like(k, dtype=torch.float64)
    here = slots[~padding].long()
    ids, p = here // page, here % page

    def written(name):
        codes = cache[name].view(torch.int8).permute(0, 2, 1, 3)[ids, p].view(forms.CODES[kind])
        return codes, cache[name[:-1] + "_scales"].permute(0, 2, 1)[ids, p]

    codes, scale = written("values")
    expect_codes, expect_scale = forms.quantised(v[~padding], kind)
    assert torch.equal(codes.view(torch.int8), expect_codes.view(torch.int8)) and torch.equal(scale, expect_scale)
    codes, scale = written("keys")
    x = key[~padding]
    # A rotated value's own error moves its code by as much again at most, and the scale with it.
    near(codes.double() * scale.double()[..., None], x,
         forms.code_step(kind, x, scale.double()) + 2 * off[~padding].amax(-1, keepdim=True))
    # Nothing else of the cache changed.
    held = torch.ones(count * page, dtype=torch.bool, device="cuda")
    held[here] = False
    held = held.view(count, page)
    for name in ("keys", "values"):
        now, was = cache[name].view(torch.int8).permute(0, 2, 1, 3), before[name].view(torch.int8).permute(0, 2, 1, 3)
        assert torch.equal(now[held], was[held])
        now, was = cache[name[:-1] + "_scales"].permute(0, 2, 1), before[name[:-1] + "_scales"].permute(0, 2, 1)
        assert torch.equal(now[held], was[held])


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_kv_append_of_extreme_values(ops, kind, dtype):
    """Zero, tiny, huge, infinite and NaN vectors: the last two read back as NaN, the rest by the rule."""
    top = torch.finfo(dtype).max
    x = draw(7, 2, 64, dtype, 1)
    x[0] = 0
    x[1] = torch.finfo(dtype).tiny
    x[2, :, 5] = top
    x[2, :, 6] = -top
    x[3, 0, 63] = math.inf
    x[4, 1, 0] = -math.inf
    x[5, 0, 17] = math.nan
    pages = ops.KvPages.empty(kind, 2, 2, 8, 64)
    slots = torch.arange(7, dtype=torch.int32, device="cuda") + 3
    ops.kv_append(pages, slots, x, x)
    codes, scale = forms.quantised(x, kind)
    k, v = ops.kv_read(pages, slots, torch.float32)
    expect = codes.float() * scale[..., None]
    for got in (k, v):
        assert torch.equal(torch.isnan(got), torch.isnan(expect))
        assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(expect))
    for r, h in ((3, 0), (4, 1), (5, 0)):
        assert torch.isnan(k[r, h]).all() and not torch.isnan(k[r, 1 - h]).any()


# ------------------------------------------------------------------ the cache, read back


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,heads,dim,page,token_major", [
    (1, 8, 128, 64, False), (61, 3, 64, 8, True), (1000, 1, 256, 16, False), (17, 5, 128, 32, True)])
def test_kv_read(ops, kind, dtype, rows, heads, dim, page, token_major):
    cache = forms.make_pages(kind, 9, heads, page, dim, token_major)
    pages = ops.KvPages(**cache)
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
        codes = cache[name].view(torch.int8).permute(0, 2, 1, 3)[ids // page, ids % page].view(forms.CODES[kind]).float()
        scale = cache[name[:-1] + "_scales"].permute(0, 2, 1)[ids // page, ids % page]
        expect = (codes * scale[..., None]).to(dtype)  # one F32 product, one rounding
        assert torch.equal(got[~padding], expect[~padding])
        assert (got[padding] == 3).all()
    if not padding.any():
        new = ops.kv_read(pages, slots, dtype)
        assert torch.equal(new[0], k) and torch.equal(new[1], v)


# ------------------------------------------------------------------ attention


def paged(lengths, page, seed=0, extra=3, width=None):
    """A page table of shuffled pages for these lengths, -1 behind them."""
    need = [-(-max(n, 0) // page) for n in lengths]
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    ids = torch.randperm(sum(need) + extra, generator=g, device="cuda").int()
    table = torch.full((len(lengths), width or max(max(need), 1)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for r, n in enumerate(need):
        table[r, :n] = ids[at:at + n]
        at += n
    return table, sum(need) + extra


def attend_case(ops, kind, dtype, lengths, q_heads, heads, dim, page, token_major=False, stale=True, seed=0, scale=None,
                max_length=None, spread=0.0, q_scale=1.0):
    table, count = paged(lengths, page, seed)
    cache = forms.make_pages(kind, count, heads, page, dim, token_major, stale=stale)
    forms.fill(cache, kind, table, lengths, seed + 1, spread)
    q = draw(len(lengths), q_heads, dim, dtype, seed + 2, q_scale)
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    most = max(max(lengths), 0) if max_length is None else max_length
    pages = ops.KvPages(**cache)
    out = torch.full_like(q, 5.0)
    assert ops.kv_attention(q, pages, table, n, most, scale=scale, out=out) is out
    expect, off = forms.attended(q, cache, table, lengths, dim ** -0.5 if scale is None else scale, most)
    left = n < 0
    assert (out[left] == 5).all()
    near(out[~left], expect[~left], off[~left])
    assert (out[n == 0] == 0).all()
    return q, pages, table, n, most, out


EDGES = [1, 0, 7, 8, 9, 31, 32, 33, -1, 63, 64, 65, 127, 128, 129, 200]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("q_heads,heads,dim,page,token_major", [
    (16, 8, 128, 64, False), (32, 8, 64, 32, True), (15, 3, 256, 16, False), (32, 1, 128, 8, True), (8, 8, 64, 8, False),
    (40, 2, 256, 128, True)])
def test_kv_attention_at_tile_edges(ops, kind, dtype, q_heads, heads, dim, page, token_major):
    attend_case(ops, kind, dtype, EDGES, q_heads, heads, dim, page, token_major)


@pytest.mark.parametrize("kind,dtype,dim", [("e4m3", torch.float16, 128), ("int8", torch.bfloat16, 256), ("e4m3", torch.float32, 64),
                                            ("int8", torch.float16, 64), ("e4m3", torch.bfloat16, 256), ("int8", torch.float32, 128)])
@pytest.mark.parametrize("lengths", [[1], [100], [5000], [9000, 3, 0, 1025], [16411], [129] * 70, [2048, -1, 40] * 9,
                                     [600] * 3 + [0, -1] * 70 + [513, 1], [700, 20] * 280])
def test_kv_attention_split_and_joined(ops, kind, dtype, dim, lengths):
    attend_case(ops, kind, dtype, lengths, 8, 2, dim, 16)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("dtype", DTYPES)
def test_kv_attention_of_peaked_scores_and_uneven_values(ops, dim, dtype):
    """Scores tens apart, value scales over nine powers of ten, either sign of the scale."""
    for kind, scale in (("e4m3", 0.5), ("int8", -0.5)):
        attend_case(ops, kind, dtype, [300, 1, 2000], 4, 2, dim, 32, scale=scale, spread=10.0, seed=11)
        attend_case(ops, kind, dtype, [300, 1, 2000], 4, 2, dim, 32, scale=0.0, spread=10.0, seed=12)


@pytest.mark.parametrize("dtype,q_scale", [(torch.bfloat16, 1e30), (torch.float32, 1e-30), (torch.float16, 1000.0), (torch.float32, 0.0)])
def test_kv_attention_of_large_and_small_queries(ops, dtype, q_scale):
    attend_case(ops, "e4m3", dtype, [70, 400], 8, 2, 128, 64, q_scale=q_scale, scale=0.05 / max(q_scale, 1e-30))


def test_kv_attention_of_the_largest_queries(ops):
    q, pages, table, n, most, _ = attend_case(ops, "int8", torch.bfloat16, [70, 400], 8, 2, 64, 64)
    top = torch.finfo(torch.bfloat16).max
    cache = {x: getattr(pages, x) for x in ("keys", "values", "key_scales", "value_scales")}
    for dtype in (torch.bfloat16, torch.float32):
        large = (q.sign() * top).to(dtype)
        out = ops.kv_attention(large, pages, table, n, most, scale=1e-39)
        expect, off = forms.attended(large, cache, table, n.tolist(), 1e-39)
        # 1e-39 is below F32's normal range: held to 2^-149.
        near(out, expect, off + 2.0 ** -149 * top * 64 * 4 * expect.abs().max())


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("dtype", DTYPES)
def test_kv_attention_weights_to_their_last_bits(ops, dim, dtype):
    """Whole numbers whose products are exact, so that only the weights' roundings are left: in F32
    tensors a weight is right to 2^-22, in both of its parts."""
    g = torch.Generator(device="cuda")
    g.manual_seed(4)
    lengths, heads, page = [7, 40, 300, 1100], 2, 32
    table, count = paged(lengths, page)
    cache = forms.make_pages("int8", count, heads, page, dim)
    cache["keys"].copy_(torch.randint(-3, 4, cache["keys"].shape, generator=g, device="cuda"))
    cache["key_scales"].fill_(2.0 ** -4)
    q = torch.randint(-2, 3, (4, 16, dim), generator=g, device="cuda").to(dtype)
    out = ops.kv_attention(q, ops.KvPages(**cache), table, torch.tensor(lengths, dtype=torch.int32, device="cuda"), 1100)
    expect, off = forms.attended(q, cache, table, lengths, dim ** -0.5, exact_dots=True)
    near(out, expect, off)


def test_kv_attention_of_more_rows_than_share_work(ops):
    """Past 1024 rows each pair has a workgroup of its own."""
    lengths = ([3, 0, 70, -1, 600] * 220)[:1090]
    attend_case(ops, "e4m3", torch.float16, lengths, 4, 1, 64, 16)


def test_kv_attention_leaves_out_dropped_pages(ops):
    """Positions of pages that are not in the cache count as masked: some of a row's, then all."""
    for kind, page in (("e4m3", 8), ("int8", 16), ("e4m3", 64)):
        lengths = [300, 5, 1000, 640]
        table, count = paged(lengths, page)
        table[0, 1::3] = -1
        table[2, : 1000 // page // 2] = count  # past the cache
        table[2, -1] = 2 ** 31 - 1
        table[3] = -7
        cache = forms.make_pages(kind, count, 2, page, 128, stale=True)
        forms.fill(cache, kind, table, lengths)
        q = draw(4, 6, 128, torch.float16, 1)
        n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        out = ops.kv_attention(q, ops.KvPages(**cache), table, n, 1000)
        expect, off = forms.attended(q, cache, table, lengths, 128 ** -0.5)
        near(out, expect, off)
        assert (out[3] == 0).all()


def test_kv_attention_counts_the_bounds_that_it_states(ops):
    """max_length, the table's width and lengths past both."""
    for most, width in ((100, 10), (1000, 3), (2 ** 40, 10), (0, 10)):
        lengths = [640, 2 ** 31 - 1, 50]
        table, count = paged([640, 640, 640], 64)
        table = table[:, :width].contiguous()
        cache = forms.make_pages("int8", count, 2, 64, 64)
        q = draw(3, 4, 64, torch.float16, 1)
        n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        out = ops.kv_attention(q, ops.KvPages(**cache), table, n, most)
        expect, off = forms.attended(q, cache, table, lengths, 64 ** -0.5, most)
        near(out, expect, off)


def test_kv_attention_keeps_nan_to_its_head_and_row(ops):
    cache = forms.make_pages("e4m3", 8, 2, 16, 64)
    cache["value_scales"][2, 1, 3] = math.nan
    table = torch.tensor([[0, 1], [2, 3], [4, 5]], dtype=torch.int32, device="cuda")
    n = torch.tensor([32, 32, 32], dtype=torch.int32, device="cuda")
    q = draw(3, 4, 64, torch.float16, 1)
    q[2, 3, 9] = math.nan
    bad = torch.isnan(ops.kv_attention(q, ops.KvPages(**cache), table, n, 32))
    assert bad[1, 2:].all() and bad[2, 3].all()
    bad[1, 2:] = False
    bad[2, 3] = False
    assert not bad.any()


def test_kv_attention_takes_views(ops):
    q, pages, table, n, most, out = attend_case(ops, "e4m3", torch.bfloat16, [77, 400, 31], 8, 2, 128, 32)
    joint = torch.zeros(3, 14, 128, dtype=q.dtype, device="cuda")
    joint[:, 3:11] = q
    wide = torch.full((3, 30, 20), -9, dtype=torch.int32, device="cuda")[:, 1]
    wide[:, 2:2 + table.shape[1]] = table
    result = torch.zeros(8, 3, 128, dtype=q.dtype, device="cuda").transpose(0, 1)
    ops.kv_attention(joint[:, 3:11], pages, wide[:, 2:2 + table.shape[1]], n, most, out=result)
    assert torch.equal(result, out)
    one = ops.kv_attention(q[:1].expand(3, 8, 128), pages, table[:1].expand(3, -1), n[:1].expand(3).contiguous(), most)
    assert torch.equal(one[0], one[1]) and torch.equal(one[0], one[2])
    near(one[0].double(), out[0].double(), 2 * 2.0 ** -8 * out[0].double().abs() + 1e-3)


def test_page_offsets_past_32_bits(ops):
    """A cache of 5 GB: the last pages are written, read and attended over."""
    pages = ops.KvPages.empty("int8", 320000, 2, 64, 128)
    assert pages.keys.numel() > 2 ** 32
    rows = 200
    k, v = draw(rows, 2, 128, torch.float16, 1), draw(rows, 2, 128, torch.float16, 2)
    table = (319999 - torch.arange(4, device="cuda", dtype=torch.int32))[None]
    slots = (table[0, torch.arange(rows, device="cuda") // 64] * 64 + torch.arange(rows, device="cuda") % 64).int()
    ops.kv_append(pages, slots, k, v)
    codes, scale = forms.quantised(k, "int8")
    got = ops.kv_read(pages, slots, torch.float32)
    assert torch.equal(got[0], codes.float() * scale[..., None])
    assert not pages.keys[:319000].any()
    near_pages = {n: getattr(pages, n)[-4:].clone() for n in ("keys", "values", "key_scales", "value_scales")}
    q = draw(1, 8, 128, torch.float16, 3)
    out = ops.kv_attention(q, pages, table, torch.tensor([rows], dtype=torch.int32, device="cuda"), rows)
    expect, off = forms.attended(q, near_pages, table - 319996, [rows], 128 ** -0.5)
    near(out, expect, off)


# ------------------------------------------------------------------ together


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_requests_served_over_an_8_bit_cache(ops, kind, dtype):
    """Prompts written, then tokens one by one: each step's rows are cached and attended over, and
    agree with the 64-bit forms over what the cache holds and, to the format's rounding, over the
    unquantised keys and values."""
    heads, q_heads, dim, page, theta = 2, 6, 64, 16, 1e4
    lengths = [45, 1, 130]
    table, count = paged([n + 8 for n in lengths], page)
    pages = ops.KvPages(**forms.make_pages(kind, count, heads, page, dim, stale=True))
    cache = {n: getattr(pages, n) for n in ("keys", "values", "key_scales", "value_scales")}
    plan = ops.Rope(dim, theta=theta, scaling=LLAMA3)

    def slot(r, p):
        return int(table[r, p // page]) * page + p % page

    kept = [[], [], []]
    for r, n in enumerate(lengths):
        k, v = draw(n, heads, dim, dtype, 10 + r), draw(n, heads, dim, dtype, 20 + r)
        at = torch.arange(n, dtype=torch.int32, device="cuda")
        slots = torch.tensor([slot(r, p) for p in range(n)], dtype=torch.int32, device="cuda")
        ops.kv_append(pages, slots, k, v, rope=plan, positions=at)
        kept[r] = [forms.rotated(k, at, dim, theta, False, LLAMA3)[0], v.double()]
    for step in range(8):
        q, k, v = (draw(3, h, dim, dtype, 100 * step + h) for h in (q_heads, heads, heads + 0))
        at = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        slots = torch.tensor([slot(r, n) for r, n in enumerate(lengths)], dtype=torch.int32, device="cuda")
        turned = ops.kv_append(pages, slots, k, v, q=q, rope=plan, positions=at)
        lengths = [n + 1 for n in lengths]
        n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        out = ops.kv_attention(turned, pages, table, n, max(lengths))
        expect, off = forms.attended(turned, cache, table, lengths, dim ** -0.5)
        near(out, expect, off)
        key = forms.rotated(k, at, dim, theta, False, LLAMA3)[0]
        for r in range(3):
            kept[r] = [torch.cat((kept[r][0], key[r:r + 1])), torch.cat((kept[r][1], v[r:r + 1].double()))]
            slots = torch.tensor([slot(r, p) for p in range(lengths[r])], dtype=torch.int32, device="cuda")
            read = ops.kv_read(pages, slots, torch.float32)
            for got, x in zip(read, kept[r]):
                scale = x.abs().amax(-1) / forms.PEAK[kind]
                near(got, x, forms.code_step(kind, x, scale * 1.001) + 1e-5)


def test_calls_follow_the_current_stream(ops):
    """Inputs made on a side stream after long work there are used in order, without a synchronisation."""
    q, pages, table, n, most, out = attend_case(ops, "e4m3", torch.float16, [3000, 50], 8, 2, 128, 64)
    plan, at = ops.Rope(128), torch.arange(2, dtype=torch.int32, device="cuda")
    turned = ops.rope(plan, at, q)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        late = torch.zeros_like(q)
        a = torch.randn(4096, 4096, device="cuda")
        for _ in range(20):
            a = a @ a * 1e-3
        late.copy_(q)
        first = ops.kv_attention(late, pages, table, n, most)
        second = ops.rope(plan, at, late)
    side.synchronize()
    assert torch.equal(first, out) and torch.equal(second, turned)


def test_two_calls_at_once(ops):
    """Split calls on two streams, each with a workspace of its own, over one cache."""
    made = [attend_case(ops, "int8", torch.float16, [6000, 2500], 8, 2, 64, 16, seed=s) for s in (0, 50)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    results = [[], []]
    for _ in range(10):
        for i, (q, pages, table, n, most, _) in enumerate(made):
            with torch.cuda.stream(streams[i]):
                results[i].append(ops.kv_attention(q, pages, table, n, most))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, made[i][5]) for x in results[i])


def test_results_do_not_depend_on_the_run(ops):
    q, pages, table, n, most, out = attend_case(ops, "e4m3", torch.float32, [8000, 300], 8, 2, 128, 64)
    for _ in range(5):
        junk = torch.full((ops.kv_attention_workspace(pages, 2, 8, most) + 48,), 0x7f, dtype=torch.uint8, device="cuda")
        assert torch.equal(ops.kv_attention(q, pages, table, n, most, workspace=junk), out)


def test_a_captured_step_is_replayed(ops):
    """One decode step (append, attention, read back) captured once and replayed with new inputs, slots,
    positions and lengths in the same memory, eager steps of another cache between the replays;
    every replay equals the eager step."""
    heads, q_heads, dim, page = 2, 8, 128, 32
    table, count = paged([3000, 600, 64], page)
    shape = forms.make_pages("e4m3", count, heads, page, dim)
    graph_pages, eager_pages = (ops.KvPages(**{n: x.clone() for n, x in shape.items()}) for _ in range(2))
    plan = ops.Rope(dim, scaling=YARN)
    q, k, v = (draw(3, h, dim, torch.float16, h) for h in (q_heads, heads, heads))
    at, slots, n = (torch.zeros(3, dtype=torch.int32, device="cuda") for _ in range(3))
    work = torch.empty(ops.kv_attention_workspace(graph_pages, 3, q_heads, 3000), dtype=torch.uint8, device="cuda")

    def step(pages, workspace=None):
        turned = ops.kv_append(pages, slots, k, v, q=q, rope=plan, positions=at)
        out = ops.kv_attention(turned, pages, table, n, 3000, workspace=workspace)
        return (turned, out, *ops.kv_read(pages, slots, torch.float16))

    def inputs(i):
        position = [2900 + i, 500 + i, i]
        for x, s in ((q, 1), (k, 2), (v, 3)):
            x.copy_(draw(*x.shape, torch.float16, 31 * i + s))
        at.copy_(torch.tensor(position, dtype=torch.int32))
        slots.copy_(torch.tensor([int(table[r, p // page]) * page + p % page for r, p in enumerate(position)], dtype=torch.int32))
        n.copy_(torch.tensor([p + 1 for p in position], dtype=torch.int32))

    inputs(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(graph_pages, work)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(graph_pages, work)
    for i in range(6):
        inputs(i)
        graph.replay()
        expect = step(eager_pages)
        for x, y in zip(captured, expect):
            assert torch.equal(x, y)
        torch.cuda.synchronize()
    assert torch.equal(graph_pages.keys.view(torch.int8), eager_pages.keys.view(torch.int8))


# ------------------------------------------------------------------ refusals of tensors


def test_tensors_are_checked(ops):
    pages = ops.KvPages.empty("e4m3", 4, 2, 16, 64)
    q, k = draw(3, 4, 64, torch.float16, 1), draw(3, 2, 64, torch.float16, 2)
    i = torch.zeros(3, dtype=torch.int32, device="cuda")
    plan, table = ops.Rope(64), torch.zeros(3, 2, dtype=torch.int32, device="cuda")
    wrong = [
        lambda: ops.rope(plan, i, q.cpu()), lambda: ops.rope(plan, i.cpu(), q), lambda: ops.rope(plan, i.long(), q),
        lambda: ops.rope(plan, i[:2], q), lambda: ops.rope(plan, i, q.double()), lambda: ops.rope(plan, i, q[0]),
        lambda: ops.rope(plan, i, q.transpose(1, 2)), lambda: ops.rope(plan, i, q, k[:2]), lambda: ops.rope(plan, i, q, q_out=q[:2]),
        lambda: ops.rope(plan, i, q, q_out=q.float()), lambda: ops.rope(plan, i, q, k_out=k),
        lambda: ops.rope(plan, torch.zeros(6, dtype=torch.int32, device="cuda")[::2], q),
        lambda: ops.kv_append(pages, i, k, k[:2]), lambda: ops.kv_append(pages, i, q, q), lambda: ops.kv_append(pages, i, k, k, rope=plan),
        lambda: ops.kv_append(pages, i, k, k, q_out=q), lambda: ops.kv_append(pages, i.long(), k, k),
        lambda: ops.kv_read(pages, i.long()), lambda: ops.kv_read(pages, i, k_out=k), lambda: ops.kv_read(pages, i, k_out=q, v_out=q),
        lambda: ops.kv_read(pages, i, torch.float64), lambda: ops.kv_read(pages, table),
        lambda: ops.kv_attention(q, pages, table[:2], i, 32), lambda: ops.kv_attention(q, pages, table.long(), i, 32),
        lambda: ops.kv_attention(q, pages, table, i[:2], 32), lambda: ops.kv_attention(q, pages, table, i, -1),
        lambda: ops.kv_attention(q, pages, table, i, 32, out=q[:2]), lambda: ops.kv_attention(q.cpu(), pages, table, i, 32),
        lambda: ops.kv_attention(q, pages, torch.zeros(3, 4, dtype=torch.int32, device="cuda")[:, ::2], i, 32),
        lambda: ops.KvPages(pages.keys, pages.values[:2], pages.key_scales, pages.value_scales),
        lambda: ops.KvPages(pages.keys, pages.values, pages.key_scales.half(), pages.value_scales),
        lambda: ops.KvPages(pages.keys, pages.values, pages.key_scales, pages.value_scales.transpose(1, 2)),
        lambda: ops.KvPages(pages.keys.half(), pages.values.half(), pages.key_scales, pages.value_scales),
        lambda: ops.KvPages(pages.keys.cpu(), pages.values, pages.key_scales, pages.value_scales),
        lambda: ops.KvPages.empty("int4", 4, 2, 16, 64)]
    for n, call in enumerate(wrong):
        with pytest.raises(ValueError):
            call()
            print("accepted:", n)
    from hllm_amd import capi

    for call in (lambda: ops.KvPages.empty("int8", 4, 2, 16, 96), lambda: ops.KvPages.empty("int8", 4, 2, 17, 64),
                 lambda: ops.kv_attention(q, pages, table, i, 32, out=q),
                 lambda: ops.kv_attention(draw(3, 3, 64, torch.float16, 1), pages, table, i, 32),
                 lambda: ops.rope(plan, i, torch.zeros(3 * 256 + 1, dtype=torch.float16, device="cuda")[1:].view(3, 4, 64))):
        with pytest.raises(capi.StageError) as e:
            call()
        assert e.value.status == capi.INVALID_REQUEST


def test_a_device_that_is_not_there_is_refused(ops):
    """... and leaves no error behind for the next call."""
    plan, at = ops.Rope(64), torch.arange(3, dtype=torch.int32, device="cuda")
    q = draw(3, 4, 64, torch.float16, 1)
    t = capi.Tensor(q.data_ptr(), capi.F16, 4, 256, 64)
    turned = ops.rope(plan, at, q)
    status = capi.library().hllm_rocm_rope_apply(torch.cuda.device_count(), None, plan.address, at.data_ptr(), 3, 64, C.byref(t),
                                                 C.byref(t), None, None)
    assert status == capi.INVALID_REQUEST
    assert torch.equal(ops.rope(plan, at, q), turned)


@pytest.mark.parametrize("scale", [math.nan, math.inf, -math.inf, 1e39, -3e38])
def test_scales_that_f32_does_not_hold_are_refused(ops, scale):
    q, pages, table, n, most, _ = attend_case(ops, "e4m3", torch.float16, [20, 50], 4, 2, 64, 16)
    with pytest.raises(ValueError):
        ops.kv_attention(q, pages, table, n, most, scale=scale)


def test_the_most_rows_of_a_call(ops):
    """1048576 rows at once equal the same rows in a call of their own."""
    rows, dim, page = 1 << 20, 64, 8
    pages = ops.KvPages.empty("int8", rows // page, 1, page, dim)
    generator = torch.Generator("cuda").manual_seed(5)
    q, k, v = (torch.randn(rows, 1, dim, generator=generator, device="cuda").half() for _ in range(3))
    slots = torch.randperm(rows, generator=generator, device="cuda", dtype=torch.int32)
    at = torch.arange(rows, dtype=torch.int32, device="cuda") * 2047 - (1 << 30)
    plan = ops.Rope(dim)
    turned = ops.kv_append(pages, slots, k, v, q=q, rope=plan, positions=at)
    assert torch.equal(ops.rope(plan, at, q), turned)
    keys, values = ops.kv_read(pages, slots)
    table = torch.arange(rows, dtype=torch.int32, device="cuda")[:, None] % (rows // page)
    n = torch.arange(rows, dtype=torch.int32, device="cuda") % (page + 1)
    out = ops.kv_attention(turned, pages, table, n, page)
    other = ops.KvPages.empty("int8", rows // page, 1, page, dim)
    for part in (slice(0, 700), slice(rows // 2 - 5, rows // 2 + 300), slice(rows - 513, rows)):
        one = ops.kv_append(other, slots[part], k[part], v[part], q=q[part], rope=plan, positions=at[part])
        assert torch.equal(one, turned[part])
        for x, y in zip(ops.kv_read(other, slots[part]), (keys, values)):
            assert torch.equal(x, y[part])
        assert torch.equal(ops.kv_attention(turned[part], pages, table[part], n[part], page), out[part])


@pytest.mark.parametrize("kind", KINDS)
def test_rows_that_name_one_slot_read_alike(ops, kind):
    """Equal rows written to one slot leave that row there; a slot may be read any number of times."""
    pages = ops.KvPages.empty(kind, 4, 3, 16, 128)
    k, v = (draw(1, 3, 128, torch.float16, s).expand(40, 3, 128) for s in (1, 2))
    slots = torch.full((40,), 21, dtype=torch.int32, device="cuda")
    ops.kv_append(pages, slots, k, v)
    alone = ops.KvPages.empty(kind, 4, 3, 16, 128)
    ops.kv_append(alone, slots[:1], k[:1], v[:1])
    for x, y in zip(ops.kv_read(pages, slots), ops.kv_read(alone, slots[:1])):
        assert torch.equal(x, y.expand(40, 3, 128))
    assert torch.equal(pages.keys.view(torch.int8), alone.keys.view(torch.int8))


# ------------------------------------------------------------------ rows whose work is cut


def cut(ops, pages, lengths, q_heads, most):
    """Whether a call with these rows cuts pairs (a call that does not has no workspace)."""
    return ops.kv_attention_workspace(pages, len(lengths), q_heads, most) > 0


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_nan_stays_nan_where_work_is_cut(ops, kind, dtype, dim):
    """A NaN in a query, in every key scale of a row and head, or in those of some positions makes that
    head's (or group's) output NaN and no other, at bounds of the lengths that cut a row and that do not."""
    lengths, page = [5000, 40, 3000], 64
    table, count = paged(lengths, page)
    cache = forms.make_pages(kind, count, 2, page, dim)
    pages = ops.KvPages(**cache)
    q = draw(3, 8, dim, dtype, 1)
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    assert cut(ops, pages, lengths, 8, 5000) and not cut(ops, pages, lengths, 8, 300)

    def check(q, bad):
        for most in (5000, 2048, 300):
            out = ops.kv_attention(q, pages, table, n, most)
            assert torch.equal(torch.isnan(out).all(-1), bad) and torch.equal(torch.isnan(out).any(-1), bad), most

    bad = torch.zeros(3, 8, dtype=torch.bool, device="cuda")
    check(q, bad)
    wrong = q.clone()
    wrong[0, 3, 9] = math.nan
    wrong[1, 7, 0] = math.nan
    wrong[2] = math.nan
    bad[0, 3] = bad[1, 7] = bad[2] = True
    check(wrong, bad)
    cache["key_scales"][table[0].long(), 1] = math.nan
    cache["key_scales"][table[2, 2].long(), 0, 5:9] = math.nan
    bad[:] = False
    bad[0, 4:] = bad[2, :4] = True
    check(q, bad)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("infinity", [math.inf, -math.inf])
def test_infinite_queries_give_nan(ops, dtype, infinity):
    """Scores that are all infinite, of either sign, have no softmax: NaN, whether a row is cut or not; rows
    without positions stay zeros."""
    lengths, page = [5000, 40, 0, 700], 32
    table, count = paged(lengths, page)
    table[3] = -1
    cache = forms.make_pages("int8", count, 2, page, 128)
    cache["keys"][..., 9] = 5
    pages = ops.KvPages(**cache)
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


@pytest.mark.parametrize("dtype", DTYPES)
def test_scores_of_minus_infinity_weigh_nothing(ops, dtype):
    """... beside finite ones, in the same tile or in other parts of a cut row: as if their pages were dropped."""
    lengths, page = [5000, 40, 700], 32
    table, count = paged(lengths, page)
    cache = forms.make_pages("int8", count, 2, page, 128)
    q = draw(3, 8, 128, dtype, 1).abs() + 0.25
    gone = table.clone()
    gone[0, 20:90] = gone[0, 101] = gone[1, 0] = gone[2, ::2] = -1
    there = torch.unique(gone[gone >= 0]).long()
    lost = torch.ones(count, dtype=torch.bool, device="cuda")
    lost[there] = False
    cache["keys"][lost] = -3
    cache["key_scales"][lost] = math.inf
    pages = ops.KvPages(**cache)
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    assert cut(ops, pages, lengths, 8, 5000) and not cut(ops, pages, lengths, 8, 300)
    for most in (5000, 300):
        assert torch.equal(ops.kv_attention(q, pages, table, n, most), ops.kv_attention(q, pages, gone, n, most))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_value_scales_of_either_sign(ops, dtype, dim):
    """Negated value scales with negated codes are the same values: the same bits come out."""
    lengths, page = [5000, 40, 1, 700], 32
    table, count = paged(lengths, page)
    cache = forms.make_pages("int8", count, 2, page, dim)
    other = {name: x.clone() for name, x in cache.items()}
    g = torch.Generator(device="cuda")
    g.manual_seed(9)
    flip = torch.rand(cache["value_scales"].shape, generator=g, device="cuda") < 0.5
    flip[table[1].long()] = True  # a row of negative scales alone
    other["value_scales"][flip] *= -1
    other["values"] = torch.where(flip[..., None], -other["values"], other["values"])
    q = draw(4, 8, dim, dtype, 1)
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    for most in (5000, 300):
        expect = ops.kv_attention(q, ops.KvPages(**cache), table, n, most)
        assert torch.equal(ops.kv_attention(q, ops.KvPages(**other), table, n, most), expect)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_values_near_the_largest_number(ops, dtype, dim):
    """Means of values up to 2.5e38 are finite, though sums of two of them are not."""
    lengths, page = [5000, 300, 2, 9000], 32
    table, count = paged(lengths, page)
    cache = forms.make_pages("int8", count, 2, page, dim)
    cache["values"].copy_(cache["values"].abs().clamp_min(60))
    cache["value_scales"].copy_((0.5 + 20 * cache["value_scales"]).clamp_max(1.0) * 2e36)
    q = draw(4, 8, dim, dtype, 1)
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    pages = ops.KvPages(**cache)
    assert cut(ops, pages, lengths, 8, 9000)
    for most in (9000, 300):
        expect, off = forms.attended(q, cache, table, lengths, dim ** -0.5, most)
        assert expect.max() > 1e38
        near(ops.kv_attention(q, pages, table, n, most), expect, off)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_pairs_of_more_than_64_parts(ops, dtype, dim):
    """A pair that most workgroups share, whose first two thirds hold nothing, nothing finite or NaN."""
    lengths, page = [150000], 64
    table, count = paged(lengths, page)
    cache = forms.make_pages("int8", count, 1, page, dim, stale=True)
    forms.fill(cache, "int8", table, lengths)
    q = draw(1, 4, dim, dtype, 1).abs() + 0.25
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    gone = table.clone()
    gone[0, :1600] = -1
    pages = ops.KvPages(**cache)
    expect, off = forms.attended(q, cache, table, lengths, dim ** -0.5)
    near(ops.kv_attention(q, pages, table, n, 150000), expect, off)
    expect, off = forms.attended(q, cache, gone, lengths, dim ** -0.5)
    dropped = ops.kv_attention(q, pages, gone, n, 150000)
    near(dropped, expect, off)
    lost = table[0, :1600].long()
    cache["keys"][lost] = -3
    cache["key_scales"][lost] = math.inf
    assert torch.equal(ops.kv_attention(q, pages, table, n, 150000), dropped)
    cache["key_scales"][lost[7], 0, 5] = math.nan
    assert torch.isnan(ops.kv_attention(q, pages, table, n, 150000)).all()


@pytest.mark.parametrize("kind,dtype,dim", [("e4m3", torch.float16, 128), ("int8", torch.bfloat16, 256), ("e4m3", torch.float32, 64),
                                            ("int8", torch.float32, 256)])
@pytest.mark.parametrize("lengths", [
    [10000] + [0, -1, 5, 40] * 16, [3, 0] * 32 + [8191], [-1] * 129 + [6000], [130, 1] * 40 + [12000, -1, 7000] + [0] * 47,
    [9000] + [20, -1, 0, 129, 3] * 139 + [-1, 2500, 1, 0], [-1, 64] * 511 + [10000, 9], [0] * 500 + [16000] + [1] * 523])
def test_shares_of_many_rows(ops, kind, dtype, dim, lengths):
    """65 to 1024 rows, several to a lane of the scan that finds a share's first row, of which one or two are long."""
    q, pages, *_ = attend_case(ops, kind, dtype, lengths, 2, 1, dim, 16)
    assert cut(ops, pages, lengths, 2, max(lengths))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype,dim", [(torch.float16, 64), (torch.bfloat16, 128), (torch.float32, 128), (torch.float16, 256),
                                       (torch.float32, 256)])
@pytest.mark.parametrize("q_heads,heads", [(20, 1), (32, 1), (40, 2), (17, 1), (64, 1)])
def test_cut_groups_of_more_than_sixteen_heads(ops, kind, dtype, dim, q_heads, heads):
    for lengths in ([5000], [129, 20000, -1, 0, 6400]):
        q, pages, *_ = attend_case(ops, kind, dtype, lengths, q_heads, heads, dim, 32)
        assert cut(ops, pages, lengths, q_heads, max(lengths))


def test_workspaces_are_checked(ops):
    q, pages, table, n, most, out = attend_case(ops, "e4m3", torch.float16, [5000, 50], 8, 2, 128, 64)
    need = ops.kv_attention_workspace(pages, 2, 8, most)
    good = torch.empty(need + 64, dtype=torch.uint8, device="cuda")
    for wrong in (need, good.data_ptr(), b"", good.cpu(), good.view(torch.int8), good[::2]):
        with pytest.raises(ValueError):
            ops.kv_attention(q, pages, table, n, most, workspace=wrong)
    for wrong in (good[:need - 1], good[8:], good[:0]):
        with pytest.raises(capi.StageError):
            ops.kv_attention(q, pages, table, n, most, workspace=wrong)
    assert torch.equal(ops.kv_attention(q, pages, table, n, most, workspace=good[16:]), out)
