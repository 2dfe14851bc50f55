"""Operators on device memory, for torch tensors: rotary positions (``Rope``, ``rope``) and a paged KV
cache of 8 bits (``KvPages``) or 4 (``Kv4Pages``) that is written (``kv_append``), read back
(``kv_read``) and attended over by one new token a row (``kv_attention``): over all of a row's pages, or
over those that ``kv_select`` takes by the bounds of their keys (``KvBounds``, ``kv_bounds``).

Thin calls of the C ABI (include/hllm_rocm.h, which states what each operator computes): they
check types, shapes and devices, make the outputs that are not given, and enqueue on the current
stream of the tensors' device. What a tensor's memory holds (slots, page tables, lengths) is not
looked at on the host, and no gradients are recorded. Wrong tensors raise ValueError, what the
library refuses raises ``capi.StageError``.

    plan = Rope(128, theta=1e6, scaling={"rope_type": "yarn", "factor": 4.0,
                                         "original_max_position_embeddings": 32768})
    pages = KvPages.empty("e4m3", 4096, kv_heads=8, page_tokens=64, head_dim=128)
    q = kv_append(pages, slots, k, v, q=q, rope=plan, positions=positions)
    out = kv_attention(q, pages, page_table, lengths, max_length)

    bounds = KvBounds.empty(pages)          # long rows: over 64 pages of each
    kv_bounds(pages, bounds, page_table, starts, lengths, max_new=1)  # after each kv_append
    some, held = kv_select(q, bounds, page_table, lengths, max_length, keep=64)
    out = kv_attention(q, pages, some, held, 64 * pages.page_tokens)
"""
from __future__ import annotations

import ctypes as C
import struct
from typing import Callable, NamedTuple

import torch

from . import capi

_DTYPES = {torch.float32: capi.F32, torch.float16: capi.F16, torch.bfloat16: capi.BF16}
_FORMATS = {torch.float8_e4m3fn: capi.KV_E4M3, torch.int8: capi.KV_INT8}
_MOST = (1 << 32) - 1  # past every size that the library takes, and past every length that counts
_CODES = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
_FORMATS4 = {torch.uint8: capi.KV4_E2M1, torch.bfloat16: capi.KV4_INT4}
_SCALES4 = {"e2m1": torch.uint8, "int4": torch.bfloat16}
# capi.Tensor and capi.KvAttentionArgs as bytes: a quarter of the time of filling a ctypes structure.
TENSOR = struct.Struct("@PIIQQ")
ATTENTION_ARGS = struct.Struct("@QPQQPQf4xPIIQQPIIQQPQ")
BOUNDS_ARGS = struct.Struct("@QPQQPPQ")
SELECT_ARGS = struct.Struct("@QPQQPQIII4xPIIQQPPPQ")
_SCALINGS = {
    "linear": (capi.ROPE_LINEAR, ("factor",), ()),
    "llama3": (capi.ROPE_LLAMA3, ("factor", "original_max_position_embeddings", "low_freq_factor",
                                  "high_freq_factor"), ()),
    "yarn": (capi.ROPE_YARN, ("factor", "original_max_position_embeddings"),
             ("beta_fast", "beta_slow", "attention_factor")),
}
_FIELDS = {"factor": "factor", "original_max_position_embeddings": "original_length",
           "low_freq_factor": "low_frequency_factor", "high_freq_factor": "high_frequency_factor",
           "beta_fast": "beta_fast", "beta_slow": "beta_slow", "attention_factor": "magnitude"}


class Rope:
    """A rotation's plan: ``rotary_dim`` leading elements of a head in pairs (i, i + rotary_dim / 2),
    or ``interleaved`` (2 i, 2 i + 1). ``scaling`` is a checkpoint's ``rope_scaling``: a dict
    with ``rope_type`` "linear", "llama3" or "yarn" and that type's parameters."""

    def __init__(self, rotary_dim: int, theta: float = 10000.0, interleaved: bool = False,
                 scaling: dict | None = None):
        if not 0 <= rotary_dim < 1 << 32:  # ctypes would take it modulo 2^32
            raise ValueError("the rotary dimension is even, 2 to 256")
        c = capi.RopeConfig(rotary_dimension=rotary_dim, theta=theta,
                            layout=capi.ROPE_INTERLEAVED if interleaved else capi.ROPE_HALF)
        given = dict(scaling or {})
        kinds = {given.pop(key) for key in ("rope_type", "type") if key in given}
        if len(kinds) > 1 or (given and not kinds):
            raise ValueError("a scaling has one rope_type")
        kind = kinds.pop() if kinds else "default"
        if kind != "default":
            if kind not in _SCALINGS:
                raise ValueError(f"unknown rope_type {kind!r}")
            c.scaling, needed, optional = _SCALINGS[kind]
            missing = [n for n in needed if given.get(n) is None]
            unknown = [n for n in given if n not in needed + optional]
            if missing or unknown:
                raise ValueError(f"rope_type {kind!r}: missing {missing}, unknown {unknown}")
            for name, value in given.items():
                if value is not None:
                    setattr(c, _FIELDS[name], float(value))
        elif given:
            raise ValueError(f"rope_type 'default' takes no parameters: {sorted(given)}")
        self.rotary_dim = rotary_dim
        self.plan = capi.RopePlan()
        self.address = C.addressof(self.plan)
        capi.check(capi.library().hllm_rocm_rope_plan(C.byref(c), self.address))


class _Calls(NamedTuple):
    """The library's functions for a kind of cache."""
    append: Callable
    read: Callable
    attention: Callable
    bounds: Callable


class _Pages:
    """What both kinds of cache have in common: tensors that are held, and their description for the library."""

    names: tuple[str, ...]

    def _describe(self, keys, values, key_scales, value_scales, kind, format, head_dim):
        for x in (values, key_scales, value_scales):
            if x.device != keys.device:
                raise ValueError("a cache lies on one device")
        if min(keys.shape) < 1 or min(keys.stride()) < 0:
            raise ValueError("a cache has pages")
        self.keys, self.values, self.key_scales, self.value_scales = keys, values, key_scales, value_scales
        self.device, self.kv_heads, self.head_dim = keys.device, keys.shape[1], head_dim
        self.pages, self.page_tokens = keys.shape[0], keys.shape[2]
        self.calls = _Calls(*(getattr(capi.library(), "hllm_rocm_" + name) for name in self.names))
        size = keys.element_size()
        self.c = kind(format, self.pages, self.page_tokens, self.kv_heads, head_dim, keys.stride(0) * size,
                      keys.stride(2) * size, keys.stride(1) * size, keys.data_ptr(), values.data_ptr(),
                      key_scales.data_ptr(), value_scales.data_ptr())
        self.address = C.addressof(self.c)
        kv_attention_workspace(self, 0, self.kv_heads, 0)  # the library refuses a wrong description here


class KvPages(_Pages):
    """An 8-bit paged cache in the caller's tensors: ``keys`` and ``values`` [pages, kv_heads,
    page_tokens, head_dim] (torch.float8_e4m3fn or torch.int8; any strides of whole sixteen bytes
    with a contiguous last dimension, so a permuted [pages, page_tokens, kv_heads, head_dim] too)
    and F32 scales [pages, kv_heads, page_tokens]. Position p of a page is slot page * page_tokens
    + p. The tensors are held, and must not be resized."""

    names = "kv_append", "kv_read", "kv_attention_by_head", "kv_bounds_update"

    def __init__(self, keys: torch.Tensor, values: torch.Tensor, key_scales: torch.Tensor,
                 value_scales: torch.Tensor):
        for name, x in (("keys", keys), ("values", values), ("key_scales", key_scales), ("value_scales", value_scales)):
            _on_device(x, name)
        if keys.dtype not in _FORMATS or keys.dim() != 4:
            raise ValueError("keys must be [pages, kv_heads, page_tokens, head_dim] of float8_e4m3fn or int8")
        if values.shape != keys.shape or values.dtype != keys.dtype or values.stride() != keys.stride():
            raise ValueError("values must have the keys' shape, strides and dtype")
        if keys.stride(3) != 1:
            raise ValueError("the cache's last dimension must be contiguous")
        for name, x in (("key_scales", key_scales), ("value_scales", value_scales)):
            if x.shape != keys.shape[:3] or x.dtype != torch.float32 or not x.is_contiguous():
                raise ValueError(f"{name} must be contiguous float32 [pages, kv_heads, page_tokens]")
        self._describe(keys, values, key_scales, value_scales, capi.KvPages, _FORMATS[keys.dtype], keys.shape[3])

    @classmethod
    def empty(cls, format: str, pages: int, kv_heads: int, page_tokens: int, head_dim: int, device="cuda"):
        """A new cache; format "e4m3" or "int8"."""
        if format not in _CODES:
            raise ValueError(f"unknown cache format {format!r}")

        def codes():
            return torch.zeros(pages, kv_heads, page_tokens, head_dim, dtype=torch.int8, device=device)

        def scales():
            return torch.zeros(pages, kv_heads, page_tokens, dtype=torch.float32, device=device)

        return cls(codes().view(_CODES[format]), codes().view(_CODES[format]), scales(), scales())


class Kv4Pages(_Pages):
    """A 4-bit paged cache in the caller's tensors: ``keys`` and ``values`` [pages, kv_heads, page_tokens,
    head_dim / 2] (torch.uint8, two codes a byte; strides as in ``KvPages``) and scales [pages, kv_heads,
    page_tokens, head_dim / 32], one for 32 elements: torch.uint8 for E2M1 codes (a power of two's exponent + 127) or
    torch.bfloat16 for INT4 codes. include/hllm_rocm.h states the formats and the order of the codes. The
    tensors are held, and must not be resized."""

    names = "kv4_append", "kv4_read", "kv4_attention", "kv4_bounds_update"

    def __init__(self, keys: torch.Tensor, values: torch.Tensor, key_scales: torch.Tensor,
                 value_scales: torch.Tensor):
        for name, x in (("keys", keys), ("values", values), ("key_scales", key_scales), ("value_scales", value_scales)):
            _on_device(x, name)
        if keys.dtype != torch.uint8 or keys.dim() != 4:
            raise ValueError("keys must be [pages, kv_heads, page_tokens, head_dim / 2] of uint8")
        if values.shape != keys.shape or values.dtype != keys.dtype or values.stride() != keys.stride():
            raise ValueError("values must have the keys' shape, strides and dtype")
        if keys.stride(3) != 1:
            raise ValueError("the cache's last dimension must be contiguous")
        shape = (*keys.shape[:3], keys.shape[3] // 16)
        for name, x in (("key_scales", key_scales), ("value_scales", value_scales)):
            if x.shape != shape or x.dtype not in _FORMATS4 or x.dtype != key_scales.dtype or not x.is_contiguous():
                raise ValueError(f"{name} must be contiguous [pages, kv_heads, page_tokens, head_dim / 32] of uint8 "
                                 "(E2M1) or bfloat16 (INT4)")
        self._describe(keys, values, key_scales, value_scales, capi.Kv4Pages, _FORMATS4[key_scales.dtype], 2 * keys.shape[3])

    @classmethod
    def empty(cls, format: str, pages: int, kv_heads: int, page_tokens: int, head_dim: int, device="cuda"):
        """A new cache; format "e2m1" or "int4"."""
        if format not in _SCALES4:
            raise ValueError(f"unknown cache format {format!r}")

        def codes():
            return torch.zeros(pages, kv_heads, page_tokens, head_dim // 2, dtype=torch.uint8, device=device)

        def scales():
            return torch.zeros(pages, kv_heads, page_tokens, head_dim // 32, dtype=_SCALES4[format], device=device)

        return cls(codes(), codes(), scales(), scales())


class KvBounds:
    """The bounds of a cache's pages, by which ``kv_select`` selects some of them: for each page and KV head the largest and the
    smallest key element of every channel, ``codes`` [pages, kv_heads, 2, head_dim] (int8) times ``scales`` [pages,
    kv_heads] (F32). ``kv_bounds`` makes them. The tensors are held, and must not be resized."""

    def __init__(self, pages: KvPages | Kv4Pages, codes: torch.Tensor, scales: torch.Tensor):
        shape = (pages.pages, pages.kv_heads, 2, pages.head_dim)
        for name, x, size, dtype in (("codes", codes, shape, torch.int8), ("scales", scales, shape[:2], torch.float32)):
            if not isinstance(x, torch.Tensor) or x.device != pages.device or x.dtype != dtype or x.shape != size \
                    or not x.is_contiguous():
                raise ValueError(f"{name} must be contiguous {dtype} {list(size)} on {pages.device}")
        self.codes, self.scales, self.device = codes, scales, pages.device
        self.pages, self.kv_heads, self.head_dim, self.page_tokens = pages.pages, pages.kv_heads, pages.head_dim, pages.page_tokens
        self.c = capi.KvBounds(self.pages, self.page_tokens, self.kv_heads, self.head_dim, codes.data_ptr(), scales.data_ptr())
        self.address = C.addressof(self.c)
        kv_select_workspace(self, 0, 0, 1)  # the library refuses a wrong description here

    @classmethod
    def empty(cls, pages: KvPages | Kv4Pages):
        """Bounds for this cache, with nothing made yet."""
        return cls(pages, torch.zeros(pages.pages, pages.kv_heads, 2, pages.head_dim, dtype=torch.int8, device=pages.device),
                   torch.zeros(pages.pages, pages.kv_heads, dtype=torch.float32, device=pages.device))


def _on_device(x: torch.Tensor, name: str) -> None:
    if not isinstance(x, torch.Tensor) or not x.is_cuda:
        raise ValueError(f"{name} must be a tensor in device memory")


def _fields(x: torch.Tensor, name: str, device: torch.device, rows: int, dim: int, heads: int | None = None):
    """A tensor [rows, heads, dim] as the fields of capi.Tensor."""
    if not isinstance(x, torch.Tensor) or x.device != device:
        raise ValueError(f"{name} must be a tensor on {device}")
    dtype = _DTYPES.get(x.dtype)
    if dtype is None or x.dim() != 3:
        raise ValueError(f"{name} must be [rows, heads, head_dim] of float32, float16 or bfloat16")
    n, own, width = x.shape
    if n != rows or width != dim or (heads is not None and own != heads):
        raise ValueError(f"{name} must be [{rows}, {'heads' if heads is None else heads}, {dim}]: it is {list(x.shape)}")
    row, head, last = x.stride()
    if last != 1:
        raise ValueError(f"the last dimension of {name} must be contiguous")
    return x.data_ptr(), dtype, own, row, head


def _rows(x: torch.Tensor, name: str, device: torch.device, rows: int, dim: int, heads: int | None = None) -> bytes:
    return TENSOR.pack(*_fields(x, name, device, rows, dim, heads))


def _numbers(x: torch.Tensor, name: str, device: torch.device, rows: int) -> int:
    """The address of `rows` contiguous int32 numbers."""
    if not isinstance(x, torch.Tensor) or x.device != device or x.dtype != torch.int32:
        raise ValueError(f"{name} must be int32 on {device}")
    if x.dim() != 1 or x.shape[0] != rows or not x.is_contiguous():
        raise ValueError(f"{name} must be contiguous [{rows}]")
    return x.data_ptr()


def _table(page_table: torch.Tensor, device: torch.device, rows: int, kv_heads: int | None = None):
    """(address, width, row stride, head stride) of a page table [rows, width], or [rows, kv_heads, width] where it may be."""
    if not isinstance(page_table, torch.Tensor) or page_table.device != device or page_table.dtype != torch.int32:
        raise ValueError(f"page_table must be int32 on {device}")
    shape, stride = page_table.shape, page_table.stride()
    by_head = len(shape) == 3 and kv_heads is not None
    if shape[:-1] != ((rows, kv_heads) if by_head else (rows,)):
        raise ValueError("page_table must be [rows, width]" + ("" if kv_heads is None else " or [rows, kv_heads, width]"))
    if shape[-1] > 1 and stride[-1] != 1:
        raise ValueError("a row of page_table must be contiguous")
    return page_table.data_ptr(), shape[-1], stride[0], stride[1] if by_head else 0


def _stream(device: torch.device) -> int:
    # torch.cuda.current_stream(device).cuda_stream without the object around it: 0.1 us, not 1.9.
    return torch._C._cuda_getCurrentRawStream(device.index)


def _output(out, like: torch.Tensor, fields: tuple, name: str):
    """The output of an input with these fields, made unless given, and its fields."""
    if out is None:
        out = torch.empty_like(like)  # 1.2 us; torch.empty with a shape, dtype and device 3.6
        row, head, _ = out.stride()
        return out, (out.data_ptr(), fields[1], fields[2], row, head)
    if not isinstance(out, torch.Tensor) or out.dtype != like.dtype:
        raise ValueError(f"{name} must have the input's dtype")
    return out, _fields(out, name, like.device, like.shape[0], like.shape[2], fields[2])


def rope(plan: Rope, positions: torch.Tensor, q: torch.Tensor, k: torch.Tensor | None = None,
         q_out: torch.Tensor | None = None, k_out: torch.Tensor | None = None):
    """q and k [rows, heads, head_dim] rotated at ``positions`` [rows] (int32): (q_out, k_out), or
    q_out alone without k. An output may be its input."""
    _on_device(q, "q")
    if q.dim() != 3:
        raise ValueError("q must be [rows, heads, head_dim]")
    device = q.device
    rows, _, dim = q.shape
    a = _fields(q, "q", device, rows, dim)
    q_out, b = _output(q_out, q, a, "q_out")
    at = _numbers(positions, "positions", device, rows)
    k_to = k_from = None
    if k is not None:
        c = _fields(k, "k", device, rows, dim)
        k_out, d = _output(k_out, k, c, "k_out")
        k_from, k_to = TENSOR.pack(*c), TENSOR.pack(*d)
    elif k_out is not None:
        raise ValueError("k_out without k")
    capi.check(capi.library().hllm_rocm_rope_apply(device.index, _stream(device), plan.address, at, rows, dim, TENSOR.pack(*a),
                                                   TENSOR.pack(*b), k_from, k_to))
    return q_out if k is None else (q_out, k_out)


def kv_append(pages: KvPages | Kv4Pages, slots: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
              q: torch.Tensor | None = None, rope: Rope | None = None, positions: torch.Tensor | None = None,
              q_out: torch.Tensor | None = None):
    """Quantises k and v [rows, kv_heads, head_dim] into the cache at ``slots`` [rows] (int32, -1: a
    padding row). With ``rope``, k is rotated at ``positions`` [rows] first, and q as by
    ``rope``: returns q_out then, else None. Rows of a call name different slots."""
    if not isinstance(k, torch.Tensor) or k.dim() != 3:
        raise ValueError("k must be [rows, kv_heads, head_dim]")
    device, rows, dim = pages.device, k.shape[0], pages.head_dim
    a = _rows(k, "k", device, rows, dim, pages.kv_heads)
    b = _rows(v, "v", device, rows, dim, pages.kv_heads)
    to = _numbers(slots, "slots", device, rows)
    plan = at = q_from = q_to = None
    if rope is not None:
        plan, at = rope.address, _numbers(positions, "positions", device, rows)
    if q is not None:
        c = _fields(q, "q", device, rows, dim)
        q_out, d = _output(q_out, q, c, "q_out")
        q_from, q_to = TENSOR.pack(*c), TENSOR.pack(*d)
    elif q_out is not None:
        raise ValueError("q_out without q")
    capi.check(pages.calls.append(device.index, _stream(device), pages.address, to, rows, a, b, plan, at, q_from, q_to))
    return q_out


def kv_read(pages: KvPages | Kv4Pages, slots: torch.Tensor, dtype: torch.dtype = torch.float16,
            k_out: torch.Tensor | None = None, v_out: torch.Tensor | None = None):
    """The cached keys and values at ``slots`` [rows] (int32): (k, v) [rows, kv_heads, head_dim] of
    ``dtype``, or in k_out and v_out. Rows of slots outside the cache are left as they were (in
    new outputs: undefined)."""
    device = pages.device
    if not isinstance(slots, torch.Tensor) or slots.dim() != 1:
        raise ValueError("slots must be int32 [rows]")
    rows, heads, dim = slots.shape[0], pages.kv_heads, pages.head_dim
    at = _numbers(slots, "slots", device, rows)
    if (k_out is None) != (v_out is None):
        raise ValueError("k_out and v_out come together")
    if k_out is None:
        k_out, v_out = pages.key_scales.new_empty((2, rows, heads, dim), dtype=dtype)
    a, b = _rows(k_out, "k_out", device, rows, dim, heads), _rows(v_out, "v_out", device, rows, dim, heads)
    capi.check(pages.calls.read(device.index, _stream(device), pages.address, at, rows, a, b))
    return k_out, v_out


def kv_attention(q: torch.Tensor, pages: KvPages | Kv4Pages, page_table: torch.Tensor, lengths: torch.Tensor,
                 max_length: int, scale: float | None = None, out: torch.Tensor | None = None,
                 workspace: torch.Tensor | None = None) -> torch.Tensor:
    """softmax(scale q K^T) V of one new token a row, q [rows, q_heads, head_dim], over the first
    ``lengths`` [rows] (int32) positions of the row's pages in ``page_table`` [rows, width]
    (int32), or of each KV head's own in [rows, kv_heads, width], as ``kv_select`` leaves them.
    ``max_length`` bounds the lengths on the host; ``scale`` is 1 / sqrt(head_dim) unless given. A
    length of 0 gives zeros, a negative one leaves the row as it was (in a new output: undefined).
    ``workspace``: a contiguous uint8 tensor of at least ``kv_attention_workspace`` bytes that no
    concurrent call uses; made for the call unless given."""
    device = pages.device
    if not isinstance(q, torch.Tensor) or q.dim() != 3:
        raise ValueError("q must be [rows, heads, head_dim]")
    rows, heads, _ = q.shape
    a = _fields(q, "q", device, rows, pages.head_dim)
    out, b = _output(out, q, a, "out")
    n = _numbers(lengths, "lengths", device, rows)
    table, width, stride, head_stride = _table(page_table, device, rows, pages.kv_heads)
    if max_length < 0:
        raise ValueError("max_length is negative")
    if scale is not None and not abs(scale) < 2e38:
        raise ValueError("scale is not finite")  # in F32, with log2 e
    max_length = min(max_length, width * pages.page_tokens)
    if workspace is None:
        need = _workspace_bytes(pages, rows, heads, max_length)
        if need:
            workspace = pages.key_scales.new_empty(need, dtype=torch.uint8)
    elif not isinstance(workspace, torch.Tensor) or workspace.device != device or workspace.dtype != torch.uint8 \
            or not workspace.is_contiguous():
        raise ValueError(f"workspace must be contiguous uint8 on {device}")
    at, size = (0, 0) if workspace is None else (workspace.data_ptr(), workspace.numel())
    args = ATTENTION_ARGS.pack(rows, table, width, stride, n, max_length,
                               pages.head_dim ** -0.5 if scale is None else scale, *a, *b, at, size)
    capi.check(pages.calls.attention(device.index, _stream(device), pages.address, args, head_stride))
    return out


def kv_attention_workspace(pages: KvPages | Kv4Pages, rows: int, q_heads: int, max_length: int) -> int:
    """Bytes of workspace that ``kv_attention`` needs for these sizes, and for smaller lengths (0: none). Fewer rows may need
    more: one workspace for batches of several sizes has the largest of their sizes."""
    if min(rows, q_heads, max_length) < 0:
        raise ValueError("rows, q_heads and max_length are not negative")
    return _workspace_bytes(pages, min(rows, _MOST), min(q_heads, _MOST), min(max_length, _MOST))


def _workspace_bytes(pages: KvPages | Kv4Pages, rows: int, q_heads: int, max_length: int) -> int:
    need = C.c_uint64()
    lib = capi.library()
    call = lib.hllm_rocm_kv4_attention_workspace if isinstance(pages, Kv4Pages) else lib.hllm_rocm_kv_attention_workspace
    capi.check(call(pages.address, rows, q_heads, max_length, C.byref(need)))
    return need.value


def kv_bounds(pages: KvPages | Kv4Pages, bounds: KvBounds, page_table: torch.Tensor, starts: torch.Tensor,
              lengths: torch.Tensor, max_new: int) -> None:
    """Makes the bounds of the pages that hold positions ``starts`` .. ``lengths`` - 1 (int32 [rows]) of each row of
    ``page_table`` [rows, width] (int32), from all of their positions below the length: after these positions were
    written. ``max_new`` bounds lengths - starts on the host. Rows whose start is not below their length have nothing made."""
    device = pages.device
    if bounds.device != device:
        raise ValueError("the bounds lie on another device than the cache")
    if not isinstance(lengths, torch.Tensor) or lengths.dim() != 1:
        raise ValueError("lengths must be int32 [rows]")
    rows = lengths.shape[0]
    table, width, stride, _ = _table(page_table, device, rows)
    begin, n = _numbers(starts, "starts", device, rows), _numbers(lengths, "lengths", device, rows)
    if max_new < 0:
        raise ValueError("max_new is negative")
    args = BOUNDS_ARGS.pack(rows, table, width, stride, begin, n, min(max_new, width * pages.page_tokens))
    capi.check(pages.calls.bounds(device.index, _stream(device), pages.address, bounds.address, args))


def kv_select(q: torch.Tensor, bounds: KvBounds, page_table: torch.Tensor, lengths: torch.Tensor, max_length: int, keep: int,
              first: int = 1, last: int = 1, selected: torch.Tensor | None = None,
              selected_lengths: torch.Tensor | None = None, workspace: torch.Tensor | None = None):
    """The ``keep`` pages of each row, for each KV head, that q [rows, q_heads, head_dim] is taken to attend to most: the row's
    ``first`` first and ``last`` last pages, and those whose bounds allow the largest score of one of the KV head's
    queries. Returns (pages [rows, kv_heads, keep], lengths [rows], both int32) as ``kv_attention`` takes them, with the bound
    keep * page_tokens of the lengths: the selected entries of ``page_table`` [rows, width] (int32) in their order, -1
    behind them. A negative length is passed on, and the row's pages left as they were (in a new output:
    undefined). ``workspace`` as in ``kv_attention``, of ``kv_select_workspace`` bytes."""
    device = bounds.device
    if not isinstance(q, torch.Tensor) or q.dim() != 3:
        raise ValueError("q must be [rows, heads, head_dim]")
    rows = q.shape[0]
    a = _fields(q, "q", device, rows, bounds.head_dim)
    n = _numbers(lengths, "lengths", device, rows)
    table, width, stride, _ = _table(page_table, device, rows)
    if max_length < 0:
        raise ValueError("max_length is negative")
    if not (0 <= first and 1 <= last and first + last <= keep < 1 << 31):
        raise ValueError("first is at least 0, last at least 1 and keep at least their sum")
    max_length = min(max_length, width * bounds.page_tokens)
    if selected is None:
        selected = lengths.new_empty((rows, bounds.kv_heads, keep))
    elif not isinstance(selected, torch.Tensor) or selected.device != device or selected.dtype != torch.int32 \
            or selected.shape != (rows, bounds.kv_heads, keep) or not selected.is_contiguous():
        raise ValueError(f"selected must be contiguous int32 [{rows}, {bounds.kv_heads}, {keep}] on {device}")
    if selected_lengths is None:
        selected_lengths = torch.empty_like(lengths)
        to = selected_lengths.data_ptr()
    else:
        to = _numbers(selected_lengths, "selected_lengths", device, rows)
    if workspace is None:
        need = kv_select_workspace(bounds, rows, max_length, keep)
        if need:
            workspace = lengths.new_empty(need, dtype=torch.uint8)
    elif not isinstance(workspace, torch.Tensor) or workspace.device != device or workspace.dtype != torch.uint8 \
            or not workspace.is_contiguous():
        raise ValueError(f"workspace must be contiguous uint8 on {device}")
    at, size = (0, 0) if workspace is None else (workspace.data_ptr(), workspace.numel())
    args = SELECT_ARGS.pack(rows, table, width, stride, n, max_length, keep, first, last, *a, selected.data_ptr(), to, at, size)
    capi.check(capi.library().hllm_rocm_kv_select(device.index, _stream(device), bounds.address, args))
    return selected, selected_lengths


def kv_select_workspace(bounds: KvBounds, rows: int, max_length: int, keep: int) -> int:
    """Bytes of workspace that ``kv_select`` needs for these sizes, and for smaller lengths and larger ``keep`` (0: none). Fewer rows
    may need more, as for ``kv_attention_workspace``."""
    if min(rows, max_length, keep) < 0:
        raise ValueError("rows, max_length and keep are not negative")
    need = C.c_uint64()
    capi.check(capi.library().hllm_rocm_kv_select_workspace(bounds.address, min(rows, _MOST), min(max_length, _MOST), min(keep, _MOST),
                                                            C.byref(need)))
    return need.value
