"""CPU checks of the operators for long contexts: every refusal of the 4-bit cache's, the bounds' and the selection's C entry
points (made before a device is touched), their ctypes layouts and the numbers that Python takes."""
import ctypes as C
import math
import os
import subprocess
import tempfile
from types import SimpleNamespace

import pytest

from hllm_amd import capi
from tests.test_operators import (ADDRESS, BAD_OUTPUTS, BAD_TENSORS, ROOT, by, plan, refused, tensor)

FAR = 1 << 30


def four(**changes):
    c = capi.Kv4Pages(capi.KV4_E2M1, 10, 64, 8, 128, 8 * 64 * 64, 64, 64 * 64, ADDRESS, 2 * ADDRESS, 3 * ADDRESS, 4 * ADDRESS)
    for name, value in changes.items():
        setattr(c, name, value)
    return c


def eight(**changes):
    c = capi.KvPages(capi.KV_INT8, 10, 64, 8, 128, 8 * 64 * 128, 128, 64 * 128, ADDRESS, 2 * ADDRESS, 3 * ADDRESS, 4 * ADDRESS)
    for name, value in changes.items():
        setattr(c, name, value)
    return c


def bounds(**changes):
    b = capi.KvBounds(10, 64, 8, 128, 5 * ADDRESS, 6 * ADDRESS)
    for name, value in changes.items():
        setattr(b, name, value)
    return b


BAD_FOUR = [(None, "null"), (dict(format=2), "format"), (dict(head_dimension=96), "head dimension"), (dict(head_dimension=32), "head dimension"),
            (dict(kv_heads=0), "heads"), (dict(kv_heads=1025), "heads"), (dict(page_tokens=48), "power of two"),
            (dict(page_tokens=4), "power of two"), (dict(page_tokens=8192), "power of two"), (dict(pages=0), "slots"),
            (dict(pages=1 << 25), "slots"), (dict(keys=None), "null"), (dict(value_scales=None), "null"),
            (dict(values=ADDRESS + 4), "aligned"), (dict(key_scales=ADDRESS + 8), "aligned"), (dict(token_stride=72), "16 bytes"),
            (dict(page_stride=8 * 64 * 64 - 16), "overlap"), (dict(token_stride=48), "overlap"), (dict(head_stride=64), "overlap"),
            (dict(page_stride=1 << 32), "too large"), (dict(token_stride=(1 << 28) + 16), "too large")]
BAD_BOUNDS = [(None, "null"), (dict(head_dimension=96), "head dimension"), (dict(kv_heads=0), "heads"), (dict(kv_heads=1025), "heads"),
              (dict(page_tokens=48), "power of two"), (dict(page_tokens=4), "power of two"), (dict(pages=0), "slots"),
              (dict(pages=1 << 25), "slots"), (dict(codes=None), "null"), (dict(scales=None), "null"),
              (dict(codes=5 * ADDRESS + 8), "aligned"), (dict(scales=6 * ADDRESS + 4), "aligned"), (dict(scales=5 * ADDRESS), "one memory")]


def of(make, changes):
    return None if changes is None else make(**changes)


def test_four_bit_append_refuses():
    lib = capi.library()

    def call(device=0, pages=four(), slots=ADDRESS, rows=4, k=tensor(), v=tensor(), rope=None, positions=None, q=None, q_out=None):
        return lib.hllm_rocm_kv4_append(device, None, by(pages), slots, rows, by(k), by(v), by(rope), positions, by(q), by(q_out))

    assert call(rows=0) == capi.OK
    for changes, text in BAD_FOUR:
        refused(call(pages=of(four, changes)), text)
    for changes, text in BAD_TENSORS:
        refused(call(k=of(tensor, changes)), text)
        refused(call(v=of(tensor, changes)), text)
    refused(call(device=-2), "device")
    refused(call(slots=None), "slots")
    refused(call(rows=(1 << 20) + 1), "rows")
    refused(call(k=tensor(heads=4)), "heads")
    refused(call(v=tensor(dtype=capi.F32)), "one dtype")
    refused(call(rope=plan()), "positions")
    refused(call(q=tensor(), q_out=tensor()), "rope")
    refused(call(q=tensor(), rope=plan(), positions=ADDRESS), "together")
    for one, other in (("keys", "values"), ("keys", "key_scales"), ("values", "value_scales"), ("key_scales", "value_scales")):
        refused(call(pages=four(**{one: 7 * ADDRESS, other: 7 * ADDRESS})), "one memory")
    at = dict(rope=plan(), positions=ADDRESS, q=tensor(data=8 * ADDRESS))
    for buffer in (2, 3, 4):
        refused(call(**at, q_out=tensor(data=buffer * ADDRESS)), "one memory")


def test_four_bit_read_refuses():
    lib = capi.library()

    def call(device=0, pages=four(), slots=ADDRESS, rows=4, k=tensor(), v=tensor(data=2 * ADDRESS)):
        return lib.hllm_rocm_kv4_read(device, None, by(pages), slots, rows, by(k), by(v))

    assert call(rows=0) == capi.OK
    for changes, text in BAD_FOUR:
        refused(call(pages=of(four, changes)), text)
    for changes, text in BAD_OUTPUTS:
        refused(call(k=of(tensor, changes)), text)
        refused(call(v=of(tensor, changes)), text)
    refused(call(slots=None), "slots")
    refused(call(device=-1), "device")
    refused(call(rows=(1 << 20) + 1), "rows")
    refused(call(k=tensor(heads=4)), "heads")
    refused(call(v=tensor(dtype=capi.F32)), "one dtype")
    refused(call(v=tensor()), "one memory")


def attention_args(**changes):
    a = capi.KvAttentionArgs(4, ADDRESS, 100, 100, ADDRESS, 6000, 0.1, tensor(heads=32), tensor(heads=32, data=2 * ADDRESS),
                             9 * ADDRESS, 1 << 30)
    for name, value in changes.items():
        setattr(a, name, value)
    return a


@pytest.mark.parametrize("kind", ["four", "by head"])
def test_attention_refuses(kind):
    lib = capi.library()
    name, make = ("hllm_rocm_kv4_attention", four) if kind == "four" else ("hllm_rocm_kv_attention_by_head", eight)

    def call(device=0, pages=make(), head_stride=25, **changes):
        return getattr(lib, name)(device, None, by(pages), C.byref(attention_args(**changes)), head_stride)

    assert call(rows=0) == capi.OK
    if kind == "four":
        for changes, text in BAD_FOUR:
            refused(call(pages=of(four, changes)), text)
    for changes, text in BAD_TENSORS[1:]:
        refused(call(q=tensor(**{"heads": 32, **changes})), text)
    for changes, text in BAD_OUTPUTS[1:]:
        refused(call(out=tensor(**{"heads": 32, "data": 2 * ADDRESS, **changes})), text)
    refused(getattr(lib, name)(0, None, by(make()), None, 0), "null")
    refused(call(device=-1), "device")
    refused(call(head_stride=(1 << 40) + 1), "table_head_stride")
    refused(call(table_stride=(1 << 40) + 1), "table_stride")
    refused(call(rows=(1 << 20) + 1), "rows")
    refused(call(out=tensor(heads=32)), "must not be q")
    refused(call(out=tensor(heads=16, data=2 * ADDRESS)), "heads")
    refused(call(q=tensor(heads=12), out=tensor(heads=12, data=2 * ADDRESS)), "multiple")
    for scale in (math.nan, math.inf, 3.4e38):
        refused(call(scale=scale), "scale")
    refused(call(lengths=None), "lengths")
    refused(call(page_table=None), "page_table")
    refused(call(table_width=(1 << 24) + 1), "page table")
    refused(call(workspace=None), "workspace")
    refused(call(workspace=ADDRESS + 4), "workspace")
    refused(call(workspace_bytes=16), "workspace")
    refused(call(workspace=2 * ADDRESS), "one memory")


def test_a_four_bit_grid_of_whole_clusters_stays_below_the_most_workgroups():
    """A launch has below 2^24 workgroups, and a 4-bit cache's as many as a multiple of eight clusters: as many rows
    as fit before that rounding are too many."""
    lib, need = capi.library(), C.c_uint64()
    beside = four(head_dimension=64, kv_heads=1020, token_stride=1020 * 32, head_stride=32, page_stride=64 * 1020 * 32)
    most = ((1 << 24) - 1) // 1020
    assert lib.hllm_rocm_kv4_attention_workspace(by(beside), most - 1, 1020, 100, C.byref(need)) == capi.OK
    heads = four(head_dimension=64, kv_heads=768, token_stride=768 * 32, head_stride=32, page_stride=64 * 768 * 32)
    fit = ((1 << 24) - 1 - 31) // 768  # clusters of four: multiples of 32
    assert lib.hllm_rocm_kv4_attention_workspace(by(heads), fit, 768, 100, C.byref(need)) == capi.OK
    refused(lib.hllm_rocm_kv4_attention_workspace(by(heads), fit + 1, 768, 100, C.byref(need)), "too many rows")


def test_four_bit_workspace_needs_no_device():
    lib, need = capi.library(), C.c_uint64(1)

    def size(rows, heads, length, pages=four()):
        status = lib.hllm_rocm_kv4_attention_workspace(by(pages), rows, heads, length, C.byref(need))
        assert status in (capi.OK, capi.INVALID_REQUEST)
        return need.value if status == capi.OK else None

    assert size(0, 32, 4096) == 0 and size(4, 32, 0) == 0 and size(1, 8, 20) == 0
    assert size(1, 32, 1 << 17) > 0
    assert size(1, 32, 1 << 20) <= 2 * size(1, 32, 1 << 19)
    assert size(3, 12, 100) is None and size(3, 0, 100) is None
    refused(lib.hllm_rocm_kv4_attention_workspace(None, 1, 8, 100, C.byref(need)), "null")
    refused(lib.hllm_rocm_kv4_attention_workspace(by(four()), 1, 8, 100, None), "null")


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("rows,heads,kv_heads", [(1, 32, 8), (64, 32, 8), (300, 64, 64), (1024, 1024, 1024), (1025, 8, 8), (5, 48, 1)])
def test_a_larger_bound_is_given_no_less_four_bit_workspace(rows, heads, kv_heads, dim):
    lib, need, last = capi.library(), C.c_uint64(0), 0
    pages = four(pages=1, kv_heads=kv_heads, head_dimension=dim, token_stride=dim // 2, head_stride=64 * dim // 2)
    for length in sorted({0, 1, *(1 << i for i in range(31)), *((1 << i) * 3 // 2 for i in range(1, 30))}):
        capi.check(lib.hllm_rocm_kv4_attention_workspace(by(pages), rows, heads, length, C.byref(need)))
        assert need.value >= last, length
        last = need.value


@pytest.mark.parametrize("kind", ["kv", "kv4"])
def test_bounds_update_refuses(kind):
    lib = capi.library()
    make = eight if kind == "kv" else four

    def call(device=0, pages=make(), of=bounds(), **changes):
        a = capi.KvBoundsArgs(4, ADDRESS, 100, 100, ADDRESS, ADDRESS, 64)
        for name, value in changes.items():
            setattr(a, name, value)
        return getattr(lib, f"hllm_rocm_{kind}_bounds_update")(device, None, by(pages), by(of), C.byref(a))

    assert call(rows=0) == capi.OK and call(max_new=0) == capi.OK and call(table_width=0) == capi.OK
    refused(call(pages=None), "null")
    refused(call(pages=make(page_tokens=48)), "power of two")
    for changes, text in BAD_BOUNDS:
        refused(call(of=None if changes is None else bounds(**changes)), text)
    for changes in (dict(pages=11), dict(page_tokens=128), dict(kv_heads=4), dict(head_dimension=64)):
        refused(call(of=bounds(**changes)), "another cache")
    refused(getattr(lib, f"hllm_rocm_{kind}_bounds_update")(0, None, by(make()), by(bounds()), None), "null")
    refused(call(device=-1), "device")
    refused(call(rows=(1 << 20) + 1), "rows")
    refused(call(page_table=None), "page_table")
    refused(call(starts=None), "starts")
    refused(call(lengths=None), "lengths")
    refused(call(table_width=(1 << 24) + 1), "page table")
    refused(call(table_stride=(1 << 40) + 1), "table_stride")
    refused(call(rows=1 << 20, max_new=64 * 40), "too many rows")
    for memory in (1, 3):  # the cache's keys and their scales
        refused(call(of=bounds(codes=memory * ADDRESS)), "one memory")
        refused(call(of=bounds(scales=memory * ADDRESS)), "one memory")


def select_args(**changes):
    a = capi.KvSelectArgs(4, 7 * ADDRESS, 3000, 3000, 8 * ADDRESS, 180000, 64, 1, 1, tensor(heads=32), 9 * ADDRESS, 10 * ADDRESS,
                          11 * ADDRESS, 1 << 30)
    for name, value in changes.items():
        setattr(a, name, value)
    return a


def test_select_refuses():
    lib = capi.library()

    def call(device=0, of=bounds(), **changes):
        return lib.hllm_rocm_kv_select(device, None, by(of), C.byref(select_args(**changes)))

    assert call(rows=0) == capi.OK
    for changes, text in BAD_BOUNDS:
        refused(call(of=None if changes is None else bounds(**changes)), text)
    for changes, text in BAD_TENSORS[1:]:
        refused(call(q=tensor(**{"heads": 32, **changes})), text)
    refused(lib.hllm_rocm_kv_select(0, None, by(bounds()), None), "null")
    refused(call(device=-1), "device")
    refused(call(rows=(1 << 20) + 1), "rows")
    refused(call(q=tensor(heads=12)), "multiple")
    refused(call(last=0), "last")
    refused(call(keep=1), "keep")
    refused(call(first=64), "keep")
    refused(call(first=(1 << 32) - 1, last=2, keep=1), "keep")
    refused(call(keep=(1 << 24) + 1), "selected pages")
    refused(call(table_width=(1 << 24) + 1), "page table")
    refused(call(table_stride=(1 << 40) + 1), "table_stride")
    for name in ("lengths", "page_table", "selected", "selected_lengths"):
        refused(call(**{name: None}), name)
    refused(call(workspace=None), "workspace")
    refused(call(workspace=11 * ADDRESS + 4), "workspace")
    refused(call(workspace_bytes=16), "workspace")
    for output in ("selected", "selected_lengths", "workspace"):
        for memory in (1, 5, 6, 7, 8):  # q, the bounds' codes and scales, the table, the lengths
            refused(call(**{output: memory * ADDRESS}), "one memory")
    refused(call(selected=10 * ADDRESS), "one memory")
    refused(call(workspace=9 * ADDRESS), "one memory")
    # Workgroups of 1024 threads: fewer rows than elsewhere, where the rows may have many pages.
    many = bounds(kv_heads=8)
    refused(call(of=many, rows=1 << 19), "too many rows")
    refused(call(of=many, rows=1 << 20, q=tensor(heads=32)), "too many rows")
    refused(call(of=bounds(kv_heads=16), rows=1 << 20, max_length=64), "too many rows")


def test_select_workspace_needs_no_device():
    lib, need = capi.library(), C.c_uint64(1)

    def size(rows, length, keep, of=bounds()):
        capi.check(lib.hllm_rocm_kv_select_workspace(by(of), rows, length, keep, C.byref(need)))
        return need.value

    assert size(0, 1 << 20, 4) == 0 and size(4, 0, 4) == 0
    assert size(1, 64 * 512, 4) == 0 and size(64, 64 * 2304, 4) == 0
    assert size(1, 64 * 3000, 3000) == 0 and size(1, 64 * 3000, 2999) > 0
    for rows in (1, 15, 16, 40):
        last = 0
        for length in sorted({0, 1, *(1 << i for i in range(31)), *((1 << i) * 3 // 2 for i in range(1, 30))}):
            now = size(rows, length, 16)
            assert now >= last
            last = now
        assert all(size(rows, 1 << 20, keep) >= size(rows, 1 << 20, keep + 1) for keep in (2, 500, (1 << 14) - 1, 1 << 14))
    refused(lib.hllm_rocm_kv_select_workspace(None, 1, 8, 100, C.byref(need)), "null")
    refused(lib.hllm_rocm_kv_select_workspace(by(bounds()), 1, 8, 100, None), "null")
    refused(lib.hllm_rocm_kv_select_workspace(by(bounds()), (1 << 20) + 1, 8, 100, C.byref(need)), "rows")


@pytest.mark.parametrize("kind", ["kv", "kv4", "select"])
def test_a_workspace_is_for_its_number_of_rows(kind):
    """Fewer rows may need more: a workspace for several batch sizes has the largest of their sizes, and a smaller one is
    refused."""
    lib, need = capi.library(), C.c_uint64(1)
    length = 1600 if kind != "select" else 64 * 2000

    def size(rows):
        if kind == "select":
            capi.check(lib.hllm_rocm_kv_select_workspace(by(bounds()), rows, length, 64, C.byref(need)))
        else:
            make, name = (four, "hllm_rocm_kv4_attention_workspace") if kind == "kv4" else (eight, "hllm_rocm_kv_attention_workspace")
            capi.check(getattr(lib, name)(by(make()), rows, 32, length, C.byref(need)))
        return need.value

    def call(rows, held):
        if kind == "select":
            args = select_args(rows=rows, max_length=length, workspace_bytes=held)
            return lib.hllm_rocm_kv_select(0, None, by(bounds()), C.byref(args))
        args = attention_args(rows=rows, max_length=length, workspace_bytes=held)
        if kind == "kv4":
            return lib.hllm_rocm_kv4_attention(0, None, by(four()), C.byref(args), 0)
        return lib.hllm_rocm_kv_attention(0, None, by(eight()), C.byref(args))

    sizes = {rows: size(rows) for rows in range(1, 300)}
    most = max(sizes, key=sizes.get)
    assert 1 < most < 299 and sizes[299] == 0 < sizes[most]
    refused(call(most, sizes[299]), "workspace")
    refused(call(most, sizes[most] - 1), "workspace")


@pytest.mark.parametrize("struct,cname", [(capi.Kv4Pages, "hllm_rocm_kv4_pages"), (capi.KvBounds, "hllm_rocm_kv_bounds"),
                                          (capi.KvBoundsArgs, "hllm_rocm_kv_bounds_args"), (capi.KvSelectArgs, "hllm_rocm_kv_select_args")])
def test_layouts_match_the_header(struct, cname):
    fields = [f for f, _ in struct._fields_]
    body = "\n".join(f'  printf("%zu ", offsetof({cname}, {f}));' for f in fields)
    source = f'#include <stddef.h>\n#include <stdio.h>\n#include "hllm_rocm.h"\nint main(void) {{\n{body}\n' \
             f'  printf("%zu\\n", sizeof({cname}));\n  return 0;\n}}\n'
    with tempfile.TemporaryDirectory() as d:
        c_file, exe = os.path.join(d, "probe.c"), os.path.join(d, "probe")
        with open(c_file, "w") as f:
            f.write(source)
        subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), c_file, "-o", exe], check=True)
        got = [int(x) for x in subprocess.run([exe], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [getattr(struct, f).offset for f in fields] + [C.sizeof(struct)]


def test_packed_bytes_have_the_structures_layouts():
    from hllm_amd import operators

    t = capi.Tensor(ADDRESS, 2, 7, 1 << 33, 1 << 34)
    fields = (ADDRESS, 2, 7, 1 << 33, 1 << 34)
    a = capi.KvBoundsArgs(3, ADDRESS, 5, 1 << 35, 2 * ADDRESS, 3 * ADDRESS, 1 << 36)
    assert operators.BOUNDS_ARGS.pack(3, ADDRESS, 5, 1 << 35, 2 * ADDRESS, 3 * ADDRESS, 1 << 36) == bytes(a)
    s = capi.KvSelectArgs(3, ADDRESS, 5, 1 << 35, 2 * ADDRESS, 1 << 36, 7, 8, 9, t, 3 * ADDRESS, 4 * ADDRESS, 5 * ADDRESS, 1 << 37)
    assert operators.SELECT_ARGS.pack(3, ADDRESS, 5, 1 << 35, 2 * ADDRESS, 1 << 36, 7, 8, 9, *fields, 3 * ADDRESS, 4 * ADDRESS,
                                      5 * ADDRESS, 1 << 37) == bytes(s)


def test_numbers_are_not_taken_modulo_2_to_the_32():
    from hllm_amd import operators

    b = bounds()
    held = SimpleNamespace(address=C.addressof(b))
    assert operators.kv_select_workspace(held, 1, 1 << 40, 16) == operators.kv_select_workspace(held, 1, 1 << 30, 16) > 0
    assert operators.kv_select_workspace(held, 1, 64 * 3000, (1 << 32) + 16) == 0
    with pytest.raises(capi.StageError):
        operators.kv_select_workspace(held, 1 << 32, 100, 16)
    for wrong in ((-1, 8, 8), (8, -1, 8), (8, 8, -1)):
        with pytest.raises(ValueError):
            operators.kv_select_workspace(held, *wrong)
