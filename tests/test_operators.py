"""CPU checks of the operators on device memory: rotation plans against the scalings' formulas,
every refusal of the C entry points (made before a device is touched) and the ctypes layouts."""
import ctypes as C
import math
import os
import subprocess
import tempfile

import pytest

from hllm_amd import capi
from tests.operator_forms import LLAMA3, YARN, frequencies

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
ADDRESS = 1 << 20  # a 16-byte aligned address that no refused call reads


def refused(status, text=""):
    assert status == capi.INVALID_REQUEST, (status, capi.library().hllm_rocm_last_error())
    assert text.encode() in capi.library().hllm_rocm_last_error(), capi.library().hllm_rocm_last_error()


# ------------------------------------------------------------------ plans


@pytest.mark.parametrize("rotary,theta", [(128, 1e6), (64, 5e5), (20, 1e4), (2, 10.0), (256, 1000042.0)])
@pytest.mark.parametrize("scaling", [None, {"rope_type": "linear", "factor": 4.0}, LLAMA3, YARN,
                                     dict(YARN, beta_fast=16.0, beta_slow=2.0, attention_factor=1.25)])
def test_plan_holds_the_frequencies(rotary, theta, scaling):
    from hllm_amd import operators

    plan = operators.Rope(rotary, theta=theta, scaling=scaling).plan
    expect, magnitude = frequencies(rotary, theta, scaling)
    for i, f in enumerate(expect):
        # Frequencies are doubles here: a few roundings of 2^-53, and half a unit of 2^-64 turn.
        assert math.isclose(plan.turns[i] / 2.0 ** 64, f / (2 * math.pi), rel_tol=1e-14, abs_tol=2.0 ** -65)
    assert all(t == 0 for t in plan.turns[rotary // 2:])
    assert plan.magnitude == pytest.approx(magnitude, rel=2.0 ** -23)
    assert plan.rotary_dimension == rotary and plan.layout == capi.ROPE_HALF


def config(**changes):
    c = capi.RopeConfig(rotary_dimension=64, theta=1e4, factor=2.0, original_length=4096.0, low_frequency_factor=1.0,
                        high_frequency_factor=4.0)
    for name, value in changes.items():
        setattr(c, name, value)
    return c


@pytest.mark.parametrize("changes", [
    dict(rotary_dimension=0), dict(rotary_dimension=7), dict(rotary_dimension=258), dict(layout=2), dict(scaling=4),
    dict(theta=1.0), dict(theta=math.nan), dict(theta=math.inf), dict(scaling=capi.ROPE_LINEAR, factor=0.5),
    dict(scaling=capi.ROPE_LINEAR, factor=math.nan), dict(scaling=capi.ROPE_LLAMA3, original_length=0.0),
    dict(scaling=capi.ROPE_LLAMA3, low_frequency_factor=-1.0), dict(scaling=capi.ROPE_LLAMA3, high_frequency_factor=1.0),
    dict(scaling=capi.ROPE_YARN, original_length=-1.0), dict(scaling=capi.ROPE_YARN, beta_fast=1.0),
    dict(scaling=capi.ROPE_YARN, beta_slow=-2.0), dict(scaling=capi.ROPE_YARN, magnitude=-1.0),
    dict(scaling=capi.ROPE_YARN, magnitude=math.nan)])
def test_plan_refuses(changes):
    lib = capi.library()
    assert lib.hllm_rocm_rope_plan(C.byref(config()), C.byref(capi.RopePlan())) == capi.OK
    plan = capi.RopePlan(rotary_dimension=5)
    refused(lib.hllm_rocm_rope_plan(C.byref(config(**changes)), C.byref(plan)))
    assert plan.rotary_dimension == 5  # untouched
    refused(lib.hllm_rocm_rope_plan(None, C.byref(plan)), "null")
    refused(lib.hllm_rocm_rope_plan(C.byref(config()), None), "null")


@pytest.mark.parametrize("scaling", [
    {"rope_type": "dynamic", "factor": 2.0}, {"factor": 2.0}, {"rope_type": "linear"},
    {"rope_type": "linear", "factor": 2.0, "mscale": 1.0}, {"rope_type": "default", "factor": 2.0},
    {"rope_type": "llama3", "factor": 8.0}, {"rope_type": "yarn", "type": "linear", "factor": 2.0},
    dict(YARN, truncate=False)])
def test_rope_refuses_scalings_it_does_not_know(scaling):
    from hllm_amd import operators

    with pytest.raises(ValueError):
        operators.Rope(64, scaling=scaling)


def test_rope_takes_checkpoint_forms():
    from hllm_amd import operators

    plain = operators.Rope(64, theta=1e4)
    for scaling in ({}, {"rope_type": "default"}, {"type": "default"}):
        assert list(operators.Rope(64, theta=1e4, scaling=scaling).plan.turns) == list(plain.plan.turns)
    both = operators.Rope(64, scaling={"rope_type": "linear", "type": "linear", "factor": 2.0})
    assert both.plan.turns[0] == plain.plan.turns[0] // 2


# ------------------------------------------------------------------ refusals


def tensor(heads=8, dim=128, dtype=capi.F16, **changes):
    t = capi.Tensor(ADDRESS, dtype, heads, heads * dim, dim)
    for name, value in changes.items():
        setattr(t, name, value)
    return t


def cache(**changes):
    c = capi.KvPages(capi.KV_E4M3, 10, 64, 8, 128, 8 * 64 * 128, 128, 64 * 128, ADDRESS, ADDRESS, ADDRESS, ADDRESS)
    for name, value in changes.items():
        setattr(c, name, value)
    return c


def plan(**changes):
    p = capi.RopePlan()
    capi.check(capi.library().hllm_rocm_rope_plan(C.byref(config(**changes)), C.byref(p)))
    return p


def by(x):
    return None if x is None else C.byref(x)


BAD_TENSORS = [(None, "null"), (dict(data=None), "no memory"), (dict(data=ADDRESS + 8), "aligned"), (dict(dtype=3), "dtype"),
               (dict(heads=0), "heads"), (dict(row_stride=1028), "16 bytes"), (dict(head_stride=1 << 41), "too large")]
BAD_OUTPUTS = BAD_TENSORS + [(dict(row_stride=0), "overlap"), (dict(head_stride=64), "overlap"), (dict(row_stride=512), "overlap")]
BAD_PAGES = [(None, "null"), (dict(format=2), "format"), (dict(head_dimension=96), "head dimension"), (dict(kv_heads=0), "heads"),
             (dict(page_tokens=48), "power of two"), (dict(page_tokens=4), "power of two"), (dict(page_tokens=8192), "power of two"),
             (dict(pages=0), "slots"), (dict(pages=1 << 25), "slots"), (dict(keys=None), "null"), (dict(value_scales=None), "null"),
             (dict(values=ADDRESS + 4), "aligned"), (dict(key_scales=ADDRESS + 4), "aligned"), (dict(token_stride=136), "16 bytes"),
             (dict(page_stride=8 * 64 * 128 - 16), "overlap"), (dict(token_stride=64), "overlap"), (dict(head_stride=128), "overlap"),
             (dict(page_stride=1 << 32), "too large"), (dict(token_stride=(1 << 28) + 16), "too large")]


def pages_or_none(changes):
    return None if changes is None else cache(**changes)


def test_rope_apply_refuses():
    lib = capi.library()

    def call(device=0, rope=plan(), positions=ADDRESS, rows=4, dim=128, q=tensor(), q_out=tensor(), k=None, k_out=None):
        return lib.hllm_rocm_rope_apply(device, None, by(rope), positions, rows, dim, by(q), by(q_out), by(k), by(k_out))

    assert call(rows=0) == capi.OK
    for changes, text in BAD_TENSORS:
        bad = None if changes is None else tensor(**changes)
        refused(call(q=bad), text)
        if changes is not None:
            refused(call(k=bad, k_out=tensor()), text)
    for changes, text in BAD_OUTPUTS:
        bad = None if changes is None else tensor(**changes)
        refused(call(q_out=bad), text)
        if changes is not None:
            refused(call(k=tensor(data=2 * ADDRESS), k_out=bad), text)
    refused(call(device=-1), "device")
    refused(call(rope=None), "rope")
    refused(call(rope=capi.RopePlan()), "plan")
    refused(call(positions=None), "positions")
    refused(call(rows=(1 << 20) + 1), "rows")
    for dim in (0, 8, 72, 272):
        refused(call(dim=dim), "head dimension")
    refused(call(dim=48), "rotary")
    refused(call(k=tensor()), "together")
    refused(call(k_out=tensor()), "together")
    refused(call(q_out=tensor(dtype=capi.BF16)), "dtype")
    refused(call(q_out=tensor(heads=4)), "heads")
    refused(call(k=tensor(dtype=capi.F32), k_out=tensor(dtype=capi.F32)), "one dtype")
    refused(call(q_out=tensor(row_stride=2048)), "strides")  # q's memory at other strides


def test_kv_append_refuses():
    lib = capi.library()

    def call(device=0, pages=cache(), slots=ADDRESS, rows=4, k=tensor(), v=tensor(), rope=None, positions=None, q=None, q_out=None):
        return lib.hllm_rocm_kv_append(device, None, by(pages), slots, rows, by(k), by(v), by(rope), positions, by(q), by(q_out))

    assert call(rows=0) == capi.OK
    for changes, text in BAD_PAGES:
        refused(call(pages=pages_or_none(changes)), text)
    for changes, text in BAD_TENSORS:
        bad = None if changes is None else tensor(**changes)
        refused(call(k=bad), text)
        refused(call(v=bad), text)
    refused(call(device=-2), "device")
    refused(call(slots=None), "slots")
    refused(call(rows=(1 << 20) + 1), "rows")
    refused(call(k=tensor(heads=4)), "heads")
    refused(call(v=tensor(heads=16)), "heads")
    refused(call(v=tensor(dtype=capi.F32)), "one dtype")
    refused(call(rope=plan()), "positions")
    refused(call(rope=plan(rotary_dimension=256), positions=ADDRESS), "rotary")
    refused(call(q=tensor(), q_out=tensor()), "rope")
    refused(call(q=tensor(), rope=plan(), positions=ADDRESS), "together")
    refused(call(q=tensor(dtype=capi.BF16), q_out=tensor(dtype=capi.BF16), rope=plan(), positions=ADDRESS), "one dtype")
    refused(call(q=tensor(), q_out=tensor(row_stride=0), rope=plan(), positions=ADDRESS), "overlap")


def test_kv_read_refuses():
    lib = capi.library()

    def call(device=0, pages=cache(), slots=ADDRESS, rows=4, k=tensor(), v=tensor()):
        return lib.hllm_rocm_kv_read(device, None, by(pages), slots, rows, by(k), by(v))

    assert call(rows=0) == capi.OK
    for changes, text in BAD_PAGES:
        refused(call(pages=pages_or_none(changes)), text)
    for changes, text in BAD_OUTPUTS:
        bad = None if changes is None else tensor(**changes)
        refused(call(k=bad), text)
        refused(call(v=bad), text)
    refused(call(slots=None), "slots")
    refused(call(device=-1), "device")
    refused(call(rows=(1 << 20) + 1), "rows")
    refused(call(k=tensor(heads=4)), "heads")
    refused(call(v=tensor(dtype=capi.F32)), "one dtype")
    wide = cache(kv_heads=1024, head_dimension=256, head_stride=64 * 256, token_stride=256, page_stride=1024 * 64 * 256)
    big = tensor(heads=1024, dim=256)
    refused(call(pages=wide, rows=1 << 20, k=big, v=big), "too many rows")


def test_kv_attention_refuses():
    lib = capi.library()

    def call(device=0, pages=cache(), **changes):
        a = capi.KvAttentionArgs(4, ADDRESS, 100, 100, ADDRESS, 6000, 0.1, tensor(heads=32), tensor(heads=32, data=2 * ADDRESS),
                                 ADDRESS, 1 << 30)
        for name, value in changes.items():
            setattr(a, name, value)
        return lib.hllm_rocm_kv_attention(device, None, by(pages), C.byref(a))

    assert call(rows=0) == capi.OK
    for changes, text in BAD_PAGES:
        refused(call(pages=pages_or_none(changes)), text)
    for changes, text in BAD_TENSORS[1:]:
        refused(call(q=tensor(**{"heads": 32, **changes})), text)
    for changes, text in BAD_OUTPUTS[1:]:
        refused(call(out=tensor(**{"heads": 32, "data": 2 * ADDRESS, **changes})), text)
    refused(lib.hllm_rocm_kv_attention(0, None, C.byref(cache()), None), "null")
    refused(call(device=-1), "device")
    refused(call(rows=(1 << 20) + 1), "rows")
    refused(call(out=tensor(heads=32)), "must not be q")
    refused(call(out=tensor(heads=32, data=2 * ADDRESS, dtype=capi.BF16)), "dtype")
    refused(call(out=tensor(heads=16, data=2 * ADDRESS)), "heads")
    refused(call(q=tensor(heads=12), out=tensor(heads=12, data=2 * ADDRESS)), "multiple")
    for scale in (math.nan, math.inf):
        refused(call(scale=scale), "scale")
    refused(call(lengths=None), "lengths")
    refused(call(page_table=None), "page_table")
    for width in (1 << 26, (1 << 24) + 1):
        refused(call(table_width=width), "page table")
    refused(call(table_stride=1 << 41), "table_stride")
    refused(call(workspace=None), "workspace")
    refused(call(workspace=ADDRESS + 4), "workspace")
    refused(call(workspace_bytes=16), "workspace")


def test_kv_attention_workspace_needs_no_device():
    lib, need = capi.library(), C.c_uint64(1)

    def size(rows, heads, length, pages=cache()):
        status = lib.hllm_rocm_kv_attention_workspace(by(pages), rows, heads, length, C.byref(need))
        assert status in (capi.OK, capi.INVALID_REQUEST)
        return need.value if status == capi.OK else None

    assert size(0, 32, 4096) == 0
    assert size(4, 32, 0) == 0 and size(1, 8, 20) == 0
    assert size(1, 32, 1 << 17) > 0
    # No more than a bounded number of parts, whatever the length's bound.
    assert size(1, 32, 1 << 20) <= 2 * size(1, 32, 1 << 19)
    assert size(3, 12, 100) is None and size(3, 0, 100) is None
    refused(lib.hllm_rocm_kv_attention_workspace(None, 1, 8, 100, C.byref(need)), "null")
    refused(lib.hllm_rocm_kv_attention_workspace(C.byref(cache()), 1, 8, 100, None), "null")


@pytest.mark.parametrize("struct,cname", [(capi.Tensor, "hllm_rocm_tensor"), (capi.RopeConfig, "hllm_rocm_rope_config"),
                                          (capi.RopePlan, "hllm_rocm_rope"), (capi.KvPages, "hllm_rocm_kv_pages"),
                                          (capi.KvAttentionArgs, "hllm_rocm_kv_attention_args")])
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

    def values(struct):
        return [v for f, _ in struct._fields_ for v in (values(getattr(struct, f)) if isinstance(getattr(struct, f), C.Structure)
                                                        else [getattr(struct, f) or 0])]

    t = capi.Tensor(ADDRESS, 2, 7, 1 << 33, 1 << 34)
    assert operators.TENSOR.pack(*values(t)) == bytes(t)
    a = capi.KvAttentionArgs(3, ADDRESS, 5, 1 << 35, 2 * ADDRESS, 1 << 36, 0.5, t, capi.Tensor(ADDRESS + 16, 1, 9, 8, 4), 0, 1 << 37)
    assert operators.ATTENTION_ARGS.pack(*values(a)) == bytes(a)
    assert operators.ATTENTION_ARGS.size == C.sizeof(capi.KvAttentionArgs)


def test_outputs_in_other_tensors_memory_are_refused():
    lib, other = capi.library(), tensor(data=2 * ADDRESS)
    third, fourth = tensor(data=3 * ADDRESS), tensor(data=4 * ADDRESS)

    def rope(q, q_out, k, k_out):
        return lib.hllm_rocm_rope_apply(0, None, by(plan()), ADDRESS, 4, 128, by(q), by(q_out), by(k), by(k_out))

    refused(rope(tensor(), other, third, other), "one memory")
    refused(rope(tensor(), other, other, third), "one memory")
    refused(rope(tensor(), other, third, tensor()), "one memory")
    apart = cache(values=2 * ADDRESS)

    def append(pages, k, v, q, q_out):
        return lib.hllm_rocm_kv_append(0, None, by(pages), ADDRESS, 4, by(k), by(v), by(plan()), ADDRESS, by(q), by(q_out))

    refused(append(apart, other, third, fourth, other), "one memory")
    refused(append(apart, other, third, fourth, third), "one memory")
    refused(append(cache(), other, third, fourth, fourth), "one memory")
    refused(lib.hllm_rocm_kv_read(0, None, by(apart), ADDRESS, 4, by(other), by(other)), "one memory")


def test_a_scale_that_overflows_with_its_factor_is_refused():
    a = capi.KvAttentionArgs(4, ADDRESS, 100, 100, ADDRESS, 6000, 3.4e38, tensor(), tensor(data=2 * ADDRESS), ADDRESS, 1 << 30)
    refused(capi.library().hllm_rocm_kv_attention(0, None, C.byref(cache()), C.byref(a)), "scale")


@pytest.mark.parametrize("rows,heads,kv_heads", [(1, 32, 8), (64, 32, 8), (300, 64, 64), (1024, 1024, 1024), (1025, 8, 8)])
def test_a_larger_bound_is_given_no_less_workspace(rows, heads, kv_heads):
    """A call's bound is the smaller of max_length and its table's positions, so a workspace sized for any
    larger max_length has to do."""
    lib, need, last = capi.library(), C.c_uint64(0), 0
    pages = cache(kv_heads=kv_heads, page_stride=kv_heads * 64 * 128)
    for length in (0, 1, 100, 640, 641, 2000, 5000, 1 << 15, 1 << 18, 1 << 21, 1 << 26, 1 << 30, 1 << 40, (1 << 64) - 1):
        assert lib.hllm_rocm_kv_attention_workspace(by(pages), rows, heads, length, C.byref(need)) == capi.OK
        assert need.value >= last
        last = need.value
    assert rows > 1024 or last > 0


def test_cache_buffers_and_a_workspace_in_one_memory_are_refused():
    lib = capi.library()
    k, v, q, q_out = (tensor(data=i * ADDRESS) for i in (5, 6, 7, 8))
    buffers = ("keys", "values", "key_scales", "value_scales")
    apart = {name: (i + 1) * ADDRESS for i, name in enumerate(buffers)}

    def append(pages, out=None):
        return lib.hllm_rocm_kv_append(0, None, by(pages), ADDRESS, 4, by(k), by(v), by(plan()), ADDRESS, by(q if out else None), by(out))

    for i, name in enumerate(buffers):
        for other in buffers[:i]:
            one = cache(**{**apart, name: apart[other]})
            refused(append(one), f"{other} and {name} are one memory")
            refused(append(one, q_out), f"{other} and {name} are one memory")
        refused(append(cache(**apart), tensor(data=apart[name])), f"q_out and the cache's {name} are one memory")
    for place in (7, 8):
        a = capi.KvAttentionArgs(4, ADDRESS, 100, 100, ADDRESS, 6000, 0.1, tensor(heads=32, data=7 * ADDRESS),
                                 tensor(heads=32, data=8 * ADDRESS), place * ADDRESS, 1 << 30)
        refused(lib.hllm_rocm_kv_attention(0, None, C.byref(cache(**apart)), C.byref(a)), "one memory")


def test_launches_of_too_many_threads_are_refused():
    """2^32 threads of sixteen elements: reached by many heads below the most rows."""
    lib = capi.library()
    q, q_out = tensor(heads=1024, dim=256), tensor(heads=1024, dim=256, data=2 * ADDRESS)
    k, k_out = tensor(heads=1024, dim=256, data=3 * ADDRESS), tensor(heads=1024, dim=256, data=4 * ADDRESS)

    def rope(rows, *tensors):
        return lib.hllm_rocm_rope_apply(0, None, by(plan()), ADDRESS, rows, 256, *(by(x) for x in (tensors + (None, None))[:4]))

    refused(rope(1 << 20, q, q_out), "too many rows")
    refused(rope(1 << 18, q, q_out), "too many rows")  # 64 workgroups a row: 2^24
    refused(rope(1 << 17, q, q_out, k, k_out), "too many rows")
    wide = cache(kv_heads=1024, head_dimension=256, head_stride=64 * 256, token_stride=256, page_stride=1024 * 64 * 256,
                 keys=5 * ADDRESS, values=6 * ADDRESS, key_scales=7 * ADDRESS, value_scales=8 * ADDRESS)
    refused(lib.hllm_rocm_kv_append(0, None, by(wide), ADDRESS, 1 << 17, by(q), by(k), None, None, None, None), "too many rows")


@pytest.mark.parametrize("magnitude", [3.5e38, 1e300, 1e-46])
def test_a_magnitude_that_f32_does_not_hold_is_refused(magnitude):
    lib, plan = capi.library(), capi.RopePlan(rotary_dimension=5)
    refused(lib.hllm_rocm_rope_plan(C.byref(config(scaling=capi.ROPE_YARN, magnitude=magnitude)), C.byref(plan)), "magnitude")
    assert plan.rotary_dimension == 5


def test_numbers_past_the_c_types_do_not_wrap():
    from types import SimpleNamespace

    from hllm_amd import operators

    for rotary in (-2, (1 << 32) + 64, 1 << 64):
        with pytest.raises(ValueError):
            operators.Rope(rotary)
    c = cache()
    pages = SimpleNamespace(address=C.addressof(c))
    need = operators.kv_attention_workspace(pages, 4, 32, 1 << 30)
    assert need > 0
    for length in ((1 << 32) - 1, 1 << 32, 1 << 64, (1 << 64) + 5):
        assert operators.kv_attention_workspace(pages, 4, 32, length) == need
    for sizes in ((-1, 32, 100), (4, -32, 100), (4, 32, -1), ((1 << 64) - 4, -8, -8)):
        with pytest.raises(ValueError):
            operators.kv_attention_workspace(pages, *sizes)
    for sizes in (((1 << 64) + 4, 32, 100), (4, (1 << 32) + 32, 100)):
        with pytest.raises(capi.StageError):
            operators.kv_attention_workspace(pages, *sizes)
