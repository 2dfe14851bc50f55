"""The operators for long contexts where calls meet: rules that choose another kernel, cache lines that heads share, streams,
graphs, workspaces, the most rows and what is refused, against the plain 64-bit forms of tests/long_context_forms.py."""
import math

import pytest
import torch

from hllm_amd import capi
from tests import long_context_forms as forms
from tests.operator_forms import YARN
from tests.test_gpu_four_bit import attend_case, cut
from tests.test_gpu_operators import draw, near, paged
from tests.test_gpu_selected_pages import described, ints, random_bounds, select_case

pytestmark = pytest.mark.gpu

DTYPES = [torch.float16, torch.bfloat16, torch.float32]
KINDS = ["e2m1", "int4"]
ALL = ["e4m3", "int8", "e2m1", "int4"]


@pytest.fixture(scope="module")
def ops():
    from hllm_amd import operators

    return operators


# ------------------------------------------------------------------ weights against a reference that seldom moves


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("large_first", [False, True])
def test_values_that_outweigh_their_positions(ops, kind, dtype, dim, large_first):
    """Positions whose weights are 2^-30 of the others' and whose values 2^65 times as large: they are the output. Scores
    rise too, by head, from none to 2^30, so that heads beside each other raise their references or do not."""
    page, length, border = 64, 2000, 1000
    table, count = paged([length, 150], page)
    cache = forms.make_pages(kind, count, 2, page, dim, stale=True)
    for r, n in enumerate((length, 150)):
        edge = border if r == 0 else 70
        x = torch.zeros(n, 2, dim, device="cuda")
        later = (torch.arange(n, device="cuda") >= edge) != large_first
        x[:, :, 0] = torch.where(later, -4.0, 4.0)[:, None]
        v = draw(n, 2, dim, torch.float32, r + 1) * torch.where(later, 2.0 ** 40, 2.0 ** -25)[:, None, None]
        at = torch.arange(n, device="cuda")
        for name, y in (("keys", x), ("values", v)):
            forms.hold(cache, kind, name, table[r].long()[at // page], at % page, y)
    q = torch.zeros(2, 16, dim, dtype=dtype, device="cuda")
    q[:, :, 0] = torch.arange(16, device="cuda").to(dtype) % 8 / 4 + 0.25
    scale = 30 * math.log(2) / (8 * 2)
    pages = ops.Kv4Pages(**cache)
    n = ints([length, 150])
    for most in (length, 150):
        out = ops.kv_attention(q, pages, table, n, most, scale=scale)
        expect, off = forms.attended(q, cache, kind, table, [length, 150], scale, most)
        # From 65520 on, half a step past F16's largest number, rounding gives an infinity.
        top = 65520.0 if dtype == torch.float16 else math.inf
        past = expect.abs() - off >= top
        assert torch.equal(out[past].double(), expect[past].sign() * math.inf)
        inside = expect.abs() + off < top
        near(out[inside], expect[inside], off[inside])
        # Where both kinds count, the bound is small beside the output: what is lost of a weight counts with its value.
        assert most == 150 or (off[0] < 2.0 ** -4 * expect[0].abs().amax(-1, keepdim=True)).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("apart", [32, 64, 1024])
def test_waves_and_parts_of_very_different_values(ops, kind, dtype, dim, apart):
    """One in four stretches of `apart` positions (a wave's tiles, or a share's steps) holds the output: weights of 2^-80 and values
    2^190 times the others', behind others of that stretch with weights of 2^-40."""
    page, length = 64, 8000
    table, count = paged([length, 1500], page)
    cache = forms.make_pages(kind, count, 1, page, dim, stale=True)
    for r, n in enumerate((length, 1500)):
        at = torch.arange(n, device="cuda")
        here = at // apart % 4 == 1
        late = here & (at >= n // 2)
        x = torch.zeros(n, 1, dim, device="cuda")
        x[:, :, 0] = torch.where(late, -4.0, torch.where(here, 0.0, 4.0))[:, None]
        v = draw(n, 1, dim, torch.float32, r + 1) * torch.where(late, 2.0 ** 90, 2.0 ** -100)[:, None, None]
        for name, y in (("keys", x), ("values", v)):
            forms.hold(cache, kind, name, table[r].long()[at // page], at % page, y)
    q = torch.zeros(2, 4, dim, dtype=dtype, device="cuda")
    q[:, :, 0] = 1.0
    scale = 40 * math.log(2) / 4
    pages = ops.Kv4Pages(**cache)
    out = ops.kv_attention(q, pages, table, ints([length, 1500]), length, scale=scale)
    expect, off = forms.attended(q, cache, kind, table, [length, 1500], scale)
    near(out, expect, off)
    assert (off < 2.0 ** -3 * expect.abs().amax(-1, keepdim=True)).all()


@pytest.mark.parametrize("kind", ALL)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("values,weights", [(100, 90), (115, 120), (118, 118), (160, 200), (180, 230)])
def test_values_far_apart(ops, kind, dtype, dim, values, weights):
    """Some positions' values are 2^`values` times the others' and their weights, in half of the heads, 2^-`weights` (by head up to an
    eighth less), in others as large or as much larger: larger values first, last, and every other one, in rows of many tiles and
    of one. Weights below F32's range are not the output."""
    page, lengths = 32, [2000, 150, 40, 5, 1300, 64]
    table, count = paged(lengths, page)
    cache = forms.make_pages(kind, count, 2, page, dim, stale=True)
    large = 2.0 ** min(values, 120)
    for r, n in enumerate(lengths):
        at = torch.arange(n, device="cuda")
        big = [at < n // 2, at >= n // 2, at % 2 == 1][r % 3]
        x = torch.zeros(n, 2, dim, device="cuda")
        x[:, :, 0] = torch.where(big, -4.0, 4.0)[:, None]
        v = draw(n, 2, dim, torch.float32, r + 1) * torch.where(big, large, large * 2.0 ** -values)[:, None, None]
        for name, y in (("keys", x), ("values", v)):
            forms.hold(cache, kind, name, table[r].long()[at // page], at % page, y)
    q = torch.zeros(len(lengths), 16, dim, dtype=dtype, device="cuda")
    q[:, :, 0] = 1.0 if weights > 126 else 1 - torch.arange(16, device="cuda").to(dtype) % 5 / 32
    q[:, 1::4, 0] = 0.0
    q[:, 2::4, 0] = -1.0
    scale = weights * math.log(2) / 8
    pages = described(ops, kind, cache)
    for most in (2000, 150):
        out = ops.kv_attention(q, pages, table, ints(lengths), most, scale=scale)
        expect, off = forms.attended(q, cache, kind, table, lengths, scale, most)
        top = 65520.0 if dtype == torch.float16 else math.inf
        past = expect.abs() - off >= top
        assert torch.equal(out[past].double(), expect[past].sign() * math.inf)
        inside = expect.abs() + off < top
        near(out[inside], expect[inside], off[inside])


@pytest.mark.parametrize("kind", ALL)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("apart", [32, 64, 1024])
def test_waves_and_parts_whose_values_move_their_references(ops, kind, dtype, dim, apart):
    """Of every four stretches of `apart` positions (a wave's tiles, or a share's steps) one has scores of 0 beside -92 (base 2) with
    values of 2^88, so that what its weights are divided by lies far below its scores; the others have scores of -12 and values
    that grow 2^57-fold, so that theirs lies far above. The first has the output."""
    page, lengths = 64, [8000, 1500, 300]
    table, count = paged(lengths, page)
    cache = forms.make_pages(kind, count, 1, page, dim, stale=True)
    for r, n in enumerate(lengths):
        at = torch.arange(n, device="cuda")
        here, late = at // apart % 4 == 1, at >= n // 2
        large = here & (at % 8 == 0)
        x = torch.zeros(n, 1, dim, device="cuda")
        x[:, :, 0] = torch.where(large, -4.0, 0.0)[:, None]             # 92 / 4 each
        x[:, :, 32] = torch.where(here, 0.0, -4.0)[:, None]             # 12 / 4 each
        size = torch.where(large, 2.0 ** 88, torch.where(here | late, 1.0, 2.0 ** -57))
        v = draw(n, 1, dim, torch.float32, r + 1) * size[:, None, None]
        for name, y in (("keys", x), ("values", v)):
            forms.hold(cache, kind, name, table[r].long()[at // page], at % page, y)
    q = torch.zeros(3, 4, dim, dtype=dtype, device="cuda")
    q[:, :, 0], q[:, :, 32] = 1.0, 12 / 92
    scale = 92 * math.log(2) / 4
    pages = described(ops, kind, cache)
    for most in (8000, 300):
        out = ops.kv_attention(q, pages, table, ints(lengths), most, scale=scale)
        near(out, *forms.attended(q, cache, kind, table, lengths, scale, most))


@pytest.mark.parametrize("kind", ALL)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("apart", [0, 60, 120])
def test_equal_scores_of_any_size(ops, kind, dtype, dim, apart):
    """Keys that are all the same weigh the same, however large their scores are: past 2^24 (base 2) F32 has no fractions and then no odd
    numbers left beside them. Values 2^`apart` times as large first, last and every other one."""
    page, lengths = 32, [2000, 150, 40, 5, 1300, 64]
    table, count = paged(lengths, page)
    cache = forms.make_pages(kind, count, 2, page, dim, stale=True)
    for r, n in enumerate(lengths):
        at = torch.arange(n, device="cuda")
        big = [at < n // 2, at >= n // 2, at % 2 == 1][r % 3]
        v = draw(n, 2, dim, torch.float32, r + 1) * torch.where(big, 2.0 ** apart, 1.0)[:, None, None]
        for name, y in (("keys", torch.ones(n, 2, dim, device="cuda")), ("values", v)):
            forms.hold(cache, kind, name, table[r].long()[at // page], at % page, y)
    q = torch.ones(len(lengths), 8, dim, dtype=dtype, device="cuda")
    pages = described(ops, kind, cache)
    for most in (2000, 150):
        expect, off = forms.attended(q, cache, kind, table, lengths, 0.0, most)
        top = 65520.0 if dtype == torch.float16 else math.inf
        for scale in (0.0, -3.0, 1e4, 1.7e5, 1e7, -1e9, 1e20):
            out = ops.kv_attention(q, pages, table, ints(lengths), most, scale=scale)
            past = expect.abs() - off >= top
            assert torch.equal(out[past].double(), expect[past].sign() * math.inf)
            inside = expect.abs() + off < top
            near(out[inside], expect[inside], off[inside])


# ------------------------------------------------------------------ heads that share cache lines


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("q_heads,heads,dim", [(16, 8, 64), (6, 6, 64), (8, 8, 128), (5, 5, 128), (4, 2, 256), (128, 4, 64), (320, 4, 64), (40, 2, 128)])
@pytest.mark.parametrize("lengths", [[5000, 3, 0, 1025], [700, 20, -1] * 40])
def test_heads_within_a_cache_line(ops, kind, dtype, q_heads, heads, dim, lengths):
    """Clusters of 1, 2, 3, 4 and 8 pairs (and of 20, which is none), cut and whole."""
    if len(lengths) > 100 and q_heads > 16:
        lengths = lengths[:30]
    attend_case(ops, kind, dtype, lengths, q_heads, heads, dim, 16, token_major=True)


@pytest.mark.parametrize("seed", range(24))
def test_any_sizes(ops, seed):
    """Sizes drawn over the operators' ranges, the attention over selected pages among them."""
    g = torch.Generator().manual_seed(seed)

    def one(*of):
        return of[int(torch.randint(0, len(of), (1,), generator=g))]

    kind, dtype, dim, page = one(*KINDS), one(*DTYPES), one(64, 128, 256), one(8, 16, 32, 64, 128)
    heads, group = one(1, 2, 3, 4, 8), one(1, 2, 3, 5, 8, 17)
    most = one(60, 600, 5000, 20000)
    rows = one(1, 3, 17) if most > 1000 else one(1, 5, 130)
    lengths = torch.randint(-1, most + 1, (rows,), generator=g).tolist()
    attend_case(ops, kind, dtype, lengths, heads * group, heads, dim, page, bool(one(0, 1)), seed=seed)
    keep = one(2, 7, 40)
    select_case(ops, dtype, [min(n, 600 * page) for n in lengths[:8]], heads * group, heads, dim, page, keep, one(0, 1), 1,
                bool(one(0, 1)), seed=seed)


# ------------------------------------------------------------------ where a rule chooses another kernel


@pytest.mark.parametrize("rows,places", [(63, 36), (65, 72), (1, 2100)])
@pytest.mark.parametrize("kind,heads,dim", [("e2m1", 8, 64), ("int4", 7, 64), ("int8", 7, 128), ("e4m3", 9, 64), ("e2m1", 3, 256)])
def test_bounds_of_many_pages(ops, kind, rows, places, heads, dim):
    """A page and head for each wave and for each slot of one, heads that are no multiple of the slots, rows that end early."""
    page = 8
    table = torch.randperm(rows * places, generator=torch.Generator("cuda").manual_seed(1), device="cuda").int().view(rows, places)
    cache = forms.make_pages(kind, rows * places, heads, page, dim)
    pages = described(ops, kind, cache)
    bounds = ops.KvBounds.empty(pages)
    bounds.codes.fill_(55)
    lengths = [page * places - 8 * (r % 5) for r in range(rows)]
    ops.kv_bounds(pages, bounds, table, ints([8 * (r % 3) for r in range(rows)]), ints(lengths), page * places)
    numbers, scale = forms.parts(cache, kind, "keys")
    keys = (numbers * scale).float().double()
    codes, power = forms.whole(torch.cat((keys.amax(2), keys.amin(2)), -1))
    codes = codes.view(rows * places, heads, 2, dim).to(torch.int8)
    made = torch.zeros(rows, places, dtype=torch.bool, device="cuda")
    for r in range(rows):
        made[r, r % 3:places - r % 5] = True
    at = table[made].long()
    assert torch.equal(bounds.codes[at], codes[at]) and torch.equal(bounds.scales[at].double(), power[at])
    assert (bounds.codes[table[~made].long()] == 55).all()


@pytest.mark.parametrize("kind", ALL)
@pytest.mark.parametrize("heads,dim,page", [(2, 64, 8), (3, 128, 16), (5, 64, 32)])
def test_bounds_of_extreme_keys_among_many_pages(ops, kind, heads, dim, page):
    """Zero, tiny, huge and not finite keys beside each other, last pages that are not whole, pages outside the cache."""
    rows, places = 70, 60
    assert rows * places * heads >= 8192
    table = torch.randperm(rows * places, generator=torch.Generator("cuda").manual_seed(1), device="cuda").int().view(rows, places)
    table[3, 5], table[4, 6] = -1, rows * places
    cache = forms.make_pages(kind, rows * places, heads, page, dim, stale=True)
    lengths = [page * places - r % page for r in range(rows)]
    x = draw(8 * page, heads, dim, torch.float32, 1).view(8, page, heads, dim)
    x[1] = 0
    x[2] *= 2.0 ** -105
    x[3] *= 1e37
    x[4, 5, 0, 9] = math.nan
    x[5, 7, 1, 60] = -math.inf
    x[6] = -1.5
    at = torch.arange(page, device="cuda")
    for r in range(rows):
        for p in (0, 7, places - 1):
            n = page if p < places - 1 else lengths[r] - p * page
            forms.hold(cache, kind, "keys", table[r, p].long().expand(n), at[:n], x[(r + p) % 8, :n])
    pages = described(ops, kind, cache)
    bounds = ops.KvBounds.empty(pages)
    ops.kv_bounds(pages, bounds, table, ints([0] * rows), ints(lengths), page * places)
    for r in range(0, rows, 3):
        for p in (0, 7, places - 1):
            id = int(table[r, p])
            for h in range(heads):
                codes, scale = forms.bounds_of(cache, kind, id, h, page if p < places - 1 else lengths[r] - p * page)
                assert torch.equal(bounds.codes[id, h], codes), (r, p, h)
                assert bounds.scales[id, h].item() == scale or (math.isnan(scale) and torch.isnan(bounds.scales[id, h]))


@pytest.mark.parametrize("rows,heads", [(2, 4), (15, 8), (16, 8)])
@pytest.mark.parametrize("pages", [512, 513, 640, 641, 2304, 2305])
def test_selection_at_the_plans_borders(ops, rows, heads, pages):
    """Workgroups of 256 and of 1024 threads that score their own pages, and pages that others score."""
    lengths = [8 * (pages - 3 * r if r % 2 else pages) - r % 8 for r in range(rows)]
    select_case(ops, torch.bfloat16, lengths, 2 * heads, heads, 64, 8, 20, 1, 2, ties=pages % 2 == 1)


def test_selection_by_workgroups_that_score_many_pages(ops):
    """More pages than the workgroups of 512 pairs score at once, and than a workgroup holds; other rows are short."""
    page, width, heads = 8, 20000, 8
    lengths = [page * width - 3, 500] + [40] * 61 + [page * width]
    pages = ops.Kv4Pages.empty("e2m1", 3000, heads, page, 128)
    bounds = random_bounds(ops, pages)
    table = torch.randint(0, 3000, (64, width), generator=torch.Generator("cuda").manual_seed(1), device="cuda", dtype=torch.int32)
    q = draw(64, heads, 128, torch.bfloat16, 1)
    got, n = ops.kv_select(q, bounds, table, ints(lengths), page * width, 9)
    expect, expect_n = forms.selected(q, bounds.codes, bounds.scales, table, lengths, page, 9, 1, 1)
    assert torch.equal(got.cpu(), expect) and torch.equal(n.cpu(), expect_n)


def test_selection_of_a_bound_far_above_the_rows(ops):
    """A bound of 2^30 positions (a captured step's, say) over a table that is wide enough for it."""
    page = 4096
    table = torch.zeros(2, (1 << 30) // page, dtype=torch.int32, device="cuda")
    table[:, :900] = torch.randperm(1800, generator=torch.Generator("cuda").manual_seed(1), device="cuda").int().view(2, 900)
    pages = ops.Kv4Pages.empty("e2m1", 1800, 1, page, 64)
    bounds = random_bounds(ops, pages)
    q, lengths = draw(2, 4, 64, torch.float16, 1), [900 * page - 5, 40 * page]
    got, n = ops.kv_select(q, bounds, table, ints(lengths), 1 << 30, 30)
    expect, expect_n = forms.selected(q, bounds.codes, bounds.scales, table, lengths, page, 30, 1, 1)
    assert torch.equal(got.cpu(), expect) and torch.equal(n.cpu(), expect_n)


# ------------------------------------------------------------------ streams, graphs, workspaces


def served(ops, kind, seed=0, dtype=torch.float16, lengths=(9000, 700, 64, -1), page=8, heads=2, q_heads=8, dim=64):
    """A cache with its bounds, and a step's inputs."""
    table, count = paged(list(lengths), page, seed)
    cache = forms.make_pages(kind, count, heads, page, dim)
    pages = described(ops, kind, cache)
    bounds = ops.KvBounds.empty(pages)
    n = ints(list(lengths))
    ops.kv_bounds(pages, bounds, table, torch.zeros_like(n), n, max(lengths))
    return draw(len(lengths), q_heads, dim, dtype, seed + 2), pages, bounds, table, n


def step_over(ops, q, pages, bounds, table, n, keep=40, most=9000):
    picked, m = ops.kv_select(q, bounds, table, n, most, keep, selected=torch.full((len(n), pages.kv_heads, keep), -3, dtype=torch.int32,
                                                                                 device="cuda"))
    out = ops.kv_attention(q, pages, picked, m, keep * pages.page_tokens, out=torch.zeros_like(q))
    return picked, m, out, ops.kv_attention(q, pages, table, n, most, out=torch.zeros_like(q))


@pytest.mark.parametrize("kind", ALL)
def test_calls_follow_the_current_stream(ops, kind):
    q, pages, bounds, table, n = served(ops, kind)
    expect = step_over(ops, q, pages, bounds, table, n)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        late, made = torch.zeros_like(q), ops.KvBounds.empty(pages)
        a = torch.randn(4096, 4096, device="cuda")
        for _ in range(20):
            a = a @ a * 1e-3
        late.copy_(q)
        ops.kv_bounds(pages, made, table, torch.zeros_like(n), n, 9000)
        got = step_over(ops, late, pages, made, table, n)
    side.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got, expect))


@pytest.mark.parametrize("kind", ["e2m1", "int8"])
def test_two_calls_at_once(ops, kind):
    """On two streams, with workspaces of their own."""
    made = [served(ops, kind, seed) for seed in (0, 50)]
    expect = [step_over(ops, *x) for x in made]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    results = [[], []]
    for _ in range(10):
        for i, x in enumerate(made):
            with torch.cuda.stream(streams[i]):
                results[i].append(step_over(ops, *x))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(a, b) for got in results[i] for a, b in zip(got, expect[i]))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_results_do_not_depend_on_the_run_or_the_workspace(ops, kind, dtype):
    """Whatever a workspace holds, and nothing behind its bytes is written."""
    q, pages, bounds, table, n = served(ops, kind, dtype=dtype)
    expect = step_over(ops, q, pages, bounds, table, n)
    need = ops.kv_attention_workspace(pages, 4, 8, 9000), ops.kv_select_workspace(bounds, 4, 9000, 40)
    assert min(need) > 0
    for fill in (0, 0x7f, 0xff):
        work = [torch.full((size + 4096,), fill, dtype=torch.uint8, device="cuda") for size in need]
        out = ops.kv_attention(q, pages, table, n, 9000, out=torch.zeros_like(q), workspace=work[0][:need[0]])
        picked, m = ops.kv_select(q, bounds, table, n, 9000, 40, selected=torch.full_like(expect[0], -3), workspace=work[1][:need[1]])
        assert torch.equal(picked, expect[0]) and torch.equal(m, expect[1]) and torch.equal(out, expect[3])
        assert all((w[size:] == fill).all() for w, size in zip(work, need))
    for call in (lambda w: ops.kv_attention(q, pages, table, n, 9000, workspace=w), lambda w: ops.kv_select(q, bounds, table, n, 9000, 40, workspace=w)):
        with pytest.raises(capi.StageError):
            call(torch.empty(16, dtype=torch.uint8, device="cuda"))
        for wrong in (torch.empty(1 << 24, dtype=torch.int8, device="cuda"), torch.empty(1 << 24, dtype=torch.uint8),
                      torch.empty(1 << 24, dtype=torch.uint8, device="cuda")[::2]):
            with pytest.raises(ValueError):
                call(wrong)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("q_heads,heads,dim", [(8, 4, 64), (6, 2, 128), (40, 2, 128), (128, 4, 64), (5, 1, 256)])
def test_clusters_keep_to_their_workspace(ops, kind, dtype, q_heads, heads, dim):
    """Calls with heads that share cache lines write nothing behind the bytes that they ask for; INT4 scales may be negative."""
    lengths = [7000, 30, 2500]
    table, count = paged(lengths, 16)
    cache = forms.make_pages(kind, count, heads, 16, dim, True)
    if kind == "int4":
        cache["value_scales"][::2] *= -1
        cache["key_scales"][1::3, :, :, 1] *= -1
    pages = ops.Kv4Pages(**cache)
    q = draw(3, q_heads, dim, dtype, 1)
    need = ops.kv_attention_workspace(pages, 3, q_heads, 7000)
    assert need > 0
    work = torch.full((need + 8192,), 0x7b, dtype=torch.uint8, device="cuda")
    out = ops.kv_attention(q, pages, table, ints(lengths), 7000, workspace=work[:need])
    near(out, *forms.attended(q, cache, kind, table, lengths, dim ** -0.5))
    assert (work[need:] == 0x7b).all()
    assert torch.equal(ops.kv_attention(q, pages, table, ints(lengths), 7000), out)


@pytest.mark.parametrize("kind", ALL)
def test_a_captured_step_is_replayed(ops, kind):
    """Write, bounds, selection, both attentions and read back, captured once and replayed with new inputs and
    lengths in the same memory, with eager steps over another cache between the replays."""
    heads, q_heads, dim, page, keep = 2, 8, 128, 8, 24
    table, count = paged([8000, 600, 64], page)
    shape = forms.make_pages(kind, count, heads, page, dim)
    held = [described(ops, kind, {x: y.clone() for x, y in shape.items()}) for _ in range(2)]
    bounds = [ops.KvBounds.empty(pages) for pages in held]
    for pages, b in zip(held, bounds):
        ops.kv_bounds(pages, b, table, ints([0, 0, 0]), ints([7990, 590, 1]), 8000)
    plan = ops.Rope(dim, scaling=YARN)
    q, k, v = (draw(3, h, dim, torch.bfloat16, h) for h in (q_heads, heads, heads))
    at, slots, n = (torch.zeros(3, dtype=torch.int32, device="cuda") for _ in range(3))
    needs = (ops.kv_attention_workspace(held[0], 3, q_heads, 8000), ops.kv_select_workspace(bounds[0], 3, 8000, keep),
             ops.kv_attention_workspace(held[0], 3, q_heads, keep * page))
    assert min(needs[:2]) > 0
    works = [torch.empty(size, dtype=torch.uint8, device="cuda") for size in needs]

    def step(i, works=(None,) * 3):
        turned = ops.kv_append(held[i], slots, k, v, q=q, rope=plan, positions=at)
        ops.kv_bounds(held[i], bounds[i], table, at, n, 1)
        picked, m = ops.kv_select(turned, bounds[i], table, n, 8000, keep, workspace=works[1])
        out = ops.kv_attention(turned, held[i], picked, m, keep * page, workspace=works[2])
        every = ops.kv_attention(turned, held[i], table, n, 8000, workspace=works[0])
        return (turned, picked, m, out, every, *ops.kv_read(held[i], slots, torch.float16))

    def inputs(i):
        position = [7990 + i, 590 + i, i]
        for x, s in ((q, 1), (k, 2), (v, 3)):
            x.copy_(draw(*x.shape, torch.bfloat16, 31 * i + s))
        at.copy_(torch.tensor(position, dtype=torch.int32))
        slots.copy_(torch.tensor([int(table[r, p // page]) * page + p % page for r, p in enumerate(position)], dtype=torch.int32))
        n.copy_(at + 1)

    inputs(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(0, works)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(0, works)
    for i in range(6):
        inputs(i)
        graph.replay()
        expect = step(1)
        assert all(torch.equal(x, y) for x, y in zip(captured, expect)), i
        torch.cuda.synchronize()
    assert torch.equal(held[0].keys.view(torch.uint8), held[1].keys.view(torch.uint8))
    assert torch.equal(bounds[0].codes, bounds[1].codes) and torch.equal(bounds[0].scales, bounds[1].scales)


# ------------------------------------------------------------------ the most rows, none, refusals


@pytest.mark.parametrize("kind", KINDS)
def test_the_most_rows(ops, kind):
    """2^20 rows, a few of them real."""
    rows, page, dim = 1 << 20, 8, 64
    pages = ops.Kv4Pages.empty(kind, 64, 1, page, dim)
    bounds = ops.KvBounds.empty(pages)
    real = torch.tensor([0, 5, 1 << 19, rows - 1], device="cuda")
    slots = torch.full((rows,), -1, dtype=torch.int32, device="cuda")
    slots[real] = ints([8 * r for r in range(4)])
    one = draw(4, 2, dim, torch.float16, 1)
    k = torch.zeros(rows, 1, dim, dtype=torch.float16, device="cuda")
    k[real] = one[:, :1]
    ops.kv_append(pages, slots, k, k)
    alone = ops.Kv4Pages.empty(kind, 64, 1, page, dim)
    ops.kv_append(alone, slots[real], k[real], k[real])
    assert torch.equal(pages.keys, alone.keys) and torch.equal(pages.values, alone.values)
    out = torch.full((2, rows, 1, dim), 3.0, dtype=torch.float16, device="cuda")
    ops.kv_read(pages, slots, k_out=out[0], v_out=out[1])
    assert torch.equal(out[:, real], torch.stack(ops.kv_read(alone, slots[real]))) and (out[:, 1:5] == 3).all() and (out[:, -5:-1] == 3).all()
    n = torch.where(slots < 0, -1, 1).int()
    table = (slots.clamp_min(0) // 8)[:, None].expand(rows, 3).contiguous()
    table[:, 1:] = 60
    n[real] = ints([17, 8, 0, 24])
    ops.kv_bounds(pages, bounds, table, torch.zeros_like(n), n, 24)
    for r, id in ((0, 0), (5, 1), (rows - 1, 3)):
        codes, scale = forms.bounds_of({x: getattr(pages, x) for x in ("keys", "values", "key_scales", "value_scales")}, kind, id, 0, 8)
        assert torch.equal(bounds.codes[id, 0], codes) and bounds.scales[id, 0].item() == scale
    q = torch.ones(rows, 1, dim, dtype=torch.float16, device="cuda")
    picked, m = ops.kv_select(q, bounds, table, n, 24, 2, selected=torch.full((rows, 1, 2), -7, dtype=torch.int32, device="cuda"))
    assert m[real].tolist() == [9, 8, 0, 16] and (m[1:5] == -1).all()
    assert picked[real, 0].tolist() == [[0, 60], [1, -1], [-1, -1], [3, 60]] and (picked[1:5] == -7).all()
    held = torch.full_like(q, 5.0)
    ops.kv_attention(q, pages, table, n, 24, out=held)
    expect = ops.kv_attention(q[real], pages, table[real], n[real], 24)
    assert torch.equal(held[real], expect) and (held[1:5] == 5).all() and (held[-5:-1] == 5).all()


@pytest.mark.parametrize("kind", ALL)
def test_no_rows_and_no_width(ops, kind):
    pages = described(ops, kind, forms.make_pages(kind, 4, 2, 16, 64))
    bounds = ops.KvBounds.empty(pages)
    bounds.codes.fill_(9)
    none, table = ints([]), torch.zeros(0, 3, dtype=torch.int32, device="cuda")
    q = draw(0, 4, 64, torch.float16, 1)
    ops.kv_append(pages, none, q[:, :2], q[:, :2])
    assert ops.kv_read(pages, none)[0].shape == (0, 2, 64)
    ops.kv_bounds(pages, bounds, table, none, none, 5)
    picked, m = ops.kv_select(q, bounds, table, none, 100, 3)
    assert picked.shape == (0, 2, 3) and m.shape == (0,)
    assert ops.kv_attention(q, pages, picked, m, 48).shape == q.shape
    q, narrow, n = draw(2, 4, 64, torch.float16, 1), torch.zeros(2, 0, dtype=torch.int32, device="cuda"), ints([5, -1])
    ops.kv_bounds(pages, bounds, narrow, ints([0, 0]), n, 5)
    ops.kv_bounds(pages, bounds, torch.zeros(2, 3, dtype=torch.int32, device="cuda"), n, n, 5)
    picked, m = ops.kv_select(q, bounds, narrow, n, 5, 2)
    assert m.tolist() == [0, -1] and (picked[0] == -1).all()
    out = ops.kv_attention(q, pages, picked, m, 5)
    assert (out[0] == 0).all()
    assert (bounds.codes == 9).all()


def test_tensors_are_checked(ops):
    pages = ops.Kv4Pages.empty("int4", 4, 2, 16, 64)
    bounds = ops.KvBounds.empty(pages)
    q, k = draw(3, 4, 64, torch.float16, 1), draw(3, 2, 64, torch.float16, 2)
    i = torch.zeros(3, dtype=torch.int32, device="cuda")
    table = torch.zeros(3, 4, dtype=torch.int32, device="cuda")
    picked = torch.zeros(3, 2, 2, dtype=torch.int32, device="cuda")
    held = pages.keys, pages.values, pages.key_scales, pages.value_scales
    wrong = [
        lambda: ops.kv_append(pages, i, k, k[:2]), lambda: ops.kv_append(pages, i, q, q), lambda: ops.kv_append(pages, i.long(), k, k),
        lambda: ops.kv_read(pages, i.long()), lambda: ops.kv_read(pages, i, torch.float64), lambda: ops.kv_read(pages, i, k_out=k),
        lambda: ops.kv_attention(q, pages, table[:2], i, 32), lambda: ops.kv_attention(q, pages, picked[:, :1], i, 32),
        lambda: ops.kv_attention(q, pages, picked[:2], i, 32), lambda: ops.kv_attention(q, pages, picked.long(), i, 32),
        lambda: ops.kv_attention(q, pages, picked.transpose(1, 2), i, 32), lambda: ops.kv_attention(q, pages, picked[None], i, 32),
        lambda: ops.kv_attention(q, pages, table, i, -1), lambda: ops.kv_attention(q.double(), pages, table, i, 32),
        lambda: ops.kv_attention(q, pages, table, i, 32, scale=math.nan), lambda: ops.kv_attention(q[..., :32], pages, table, i, 32),
        lambda: ops.kv_bounds(pages, bounds, picked, i, i, 1), lambda: ops.kv_bounds(pages, bounds, table, i[:2], i, 1),
        lambda: ops.kv_bounds(pages, bounds, table, i, i.long(), 1), lambda: ops.kv_bounds(pages, bounds, table, i, i, -1),
        lambda: ops.kv_bounds(pages, bounds, table.cpu(), i, i, 1),
        lambda: ops.kv_select(q, bounds, picked, i, 64, 2), lambda: ops.kv_select(q[:2], bounds, table, i, 64, 2),
        lambda: ops.kv_select(q, bounds, table, i[:2], 64, 2), lambda: ops.kv_select(q, bounds, table, i, -1, 2),
        lambda: ops.kv_select(q, bounds, table, i, 64, 1), lambda: ops.kv_select(q, bounds, table, i, 64, 2, last=0),
        lambda: ops.kv_select(q, bounds, table, i, 64, 2, first=-1), lambda: ops.kv_select(q, bounds, table, i, 64, 1 << 31),
        lambda: ops.kv_select(q.cpu(), bounds, table, i, 64, 2), lambda: ops.kv_select(q, bounds, table, i, 64, 2, selected=picked[:, :1]),
        lambda: ops.kv_select(q, bounds, table, i, 64, 2, selected=picked.long()),
        lambda: ops.kv_select(q, bounds, table, i, 64, 2, selected=picked.cpu()),
        lambda: ops.kv_select(q, bounds, table, i, 64, 2, selected_lengths=i[:2]),
        lambda: ops.kv_select(q, bounds, table, i, 64, 2, selected_lengths=i.long()),
        lambda: ops.kv_select_workspace(bounds, -1, 64, 2),
        lambda: ops.Kv4Pages(held[0], held[1][:2], *held[2:]), lambda: ops.Kv4Pages(*held[:2], held[2].float(), held[3]),
        lambda: ops.Kv4Pages(*held[:2], held[2], held[3].view(torch.uint8)), lambda: ops.Kv4Pages(*held[:3], held[3][..., :1]),
        lambda: ops.Kv4Pages(held[0].view(torch.int8), *held[1:]), lambda: ops.Kv4Pages(held[0].cpu(), *held[1:]),
        lambda: ops.Kv4Pages(held[0][..., ::2], held[1][..., ::2], *held[2:]), lambda: ops.Kv4Pages.empty("e4m3", 4, 2, 16, 64),
        lambda: ops.KvBounds(pages, bounds.codes[:2], bounds.scales), lambda: ops.KvBounds(pages, bounds.codes, bounds.scales.half()),
        lambda: ops.KvBounds(pages, bounds.codes.cpu(), bounds.scales), lambda: ops.KvBounds(pages, bounds.codes.float(), bounds.scales)]
    for n, call in enumerate(wrong):
        with pytest.raises(ValueError):
            print(n)
            call()
    for call in (lambda: ops.Kv4Pages.empty("int4", 4, 2, 16, 96), lambda: ops.Kv4Pages.empty("e2m1", 4, 2, 12, 64),
                 lambda: ops.kv_select(draw(3, 5, 64, torch.float16, 1), bounds, table, i, 64, 2),
                 lambda: ops.kv_attention(q, pages, table, i, 32, out=q),
                 lambda: ops.kv_select(q, bounds, table, i, 64, 2, selected_lengths=i)):
        with pytest.raises(capi.StageError):
            call()
    other = ops.KvBounds.empty(ops.Kv4Pages.empty("int4", 5, 2, 16, 64))
    with pytest.raises(capi.StageError):
        ops.kv_bounds(pages, other, table, i, i + 1, 1)


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="one device")
def test_another_device_than_the_current_one(ops):
    with torch.cuda.device(1):
        q, pages, bounds, table, n = served(ops, "e2m1")
        expect = [x.cpu() for x in step_over(ops, q, pages, bounds, table, n)]
    there = [x.to("cuda:1") for x in (q, table, n)]
    assert there[0].device.index == 1
    picked, m = ops.kv_select(there[0], bounds, there[1], there[2], 9000, 40)
    assert torch.equal(picked[:3].cpu(), expect[0][:3]) and torch.equal(m.cpu(), expect[1])
