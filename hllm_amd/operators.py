"""Operators on device memory, for torch tensors: rotary positions (``Rope``, ``rope``) and an
8-bit paged KV cache (``KvPages``) that is written (``kv_append``), read back (``kv_read``) and
attended over by one new token a row (``kv_attention``).

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
"""
from __future__ import annotations

import ctypes as C
import struct

import torch

from . import capi

_DTYPES = {torch.float32: capi.F32, torch.float16: capi.F16, torch.bfloat16: capi.BF16}
_FORMATS = {torch.float8_e4m3fn: capi.KV_E4M3, torch.int8: capi.KV_INT8}
_MOST = (1 << 32) - 1  # past every size that the library takes, and past every length that counts
_CODES = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
# capi.Tensor and capi.KvAttentionArgs as bytes: a quarter of the time of filling a ctypes structure.
TENSOR = struct.Struct("@PIIQQ")
ATTENTION_ARGS = struct.Struct("@QPQQPQf4xPIIQQPIIQQPQ")
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


class KvPages:
    """An 8-bit paged cache in the caller's tensors: ``keys`` and ``values`` [pages, kv_heads,
    page_tokens, head_dim] (torch.float8_e4m3fn or torch.int8; any strides of whole sixteen bytes
    with a contiguous last dimension, so a permuted [pages, page_tokens, kv_heads, head_dim] too)
    and F32 scales [pages, kv_heads, page_tokens]. Position p of a page is slot page * page_tokens
    + p. The tensors are held, and must not be resized."""

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
        for x in (values, key_scales, value_scales):
            if x.device != keys.device:
                raise ValueError("a cache lies on one device")
        if min(keys.shape) < 1 or min(keys.stride()) < 0:
            raise ValueError("a cache has pages")
        self.keys, self.values, self.key_scales, self.value_scales = keys, values, key_scales, value_scales
        self.device, self.kv_heads, self.head_dim = keys.device, keys.shape[1], keys.shape[3]
        self.pages, self.page_tokens = keys.shape[0], keys.shape[2]
        self.c = capi.KvPages(_FORMATS[keys.dtype], self.pages, self.page_tokens, self.kv_heads, self.head_dim,
                              keys.stride(0), keys.stride(2), keys.stride(1), keys.data_ptr(), values.data_ptr(),
                              key_scales.data_ptr(), value_scales.data_ptr())
        self.address = C.addressof(self.c)
        kv_attention_workspace(self, 0, self.kv_heads, 0)  # the library refuses a wrong description here

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


def kv_append(pages: KvPages, slots: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
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
    capi.check(capi.library().hllm_rocm_kv_append(device.index, _stream(device), pages.address, to, rows, a, b, plan, at,
                                                  q_from, q_to))
    return q_out


def kv_read(pages: KvPages, slots: torch.Tensor, dtype: torch.dtype = torch.float16,
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
    capi.check(capi.library().hllm_rocm_kv_read(device.index, _stream(device), pages.address, at, rows, a, b))
    return k_out, v_out


def kv_attention(q: torch.Tensor, pages: KvPages, page_table: torch.Tensor, lengths: torch.Tensor,
                 max_length: int, scale: float | None = None, out: torch.Tensor | None = None,
                 workspace: torch.Tensor | None = None) -> torch.Tensor:
    """softmax(scale q K^T) V of one new token a row, q [rows, q_heads, head_dim], over the first
    ``lengths`` [rows] (int32) positions of the row's pages in ``page_table`` [rows, width]
    (int32). ``max_length`` bounds the lengths on the host; ``scale`` is 1 / sqrt(head_dim) unless
    given. A length of 0 gives zeros, a negative one leaves the row as it was (in a new output:
    undefined). ``workspace``: a contiguous uint8 tensor of at least ``kv_attention_workspace``
    bytes that no concurrent call uses; made for the call unless given."""
    device = pages.device
    if not isinstance(q, torch.Tensor) or q.dim() != 3:
        raise ValueError("q must be [rows, heads, head_dim]")
    rows, heads, _ = q.shape
    a = _fields(q, "q", device, rows, pages.head_dim)
    out, b = _output(out, q, a, "out")
    n = _numbers(lengths, "lengths", device, rows)
    if not isinstance(page_table, torch.Tensor) or page_table.device != device or page_table.dtype != torch.int32 \
            or page_table.dim() != 2 or page_table.shape[0] != rows:
        raise ValueError(f"page_table must be int32 [rows, width] on {device}")
    width = page_table.shape[1]
    stride, last = page_table.stride()
    if width > 1 and last != 1:
        raise ValueError("a row of page_table must be contiguous")
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
    args = ATTENTION_ARGS.pack(rows, page_table.data_ptr(), width, stride, n, max_length,
                               pages.head_dim ** -0.5 if scale is None else scale, *a, *b, at, size)
    capi.check(capi.library().hllm_rocm_kv_attention(device.index, _stream(device), pages.address, args))
    return out


def kv_attention_workspace(pages: KvPages, rows: int, q_heads: int, max_length: int) -> int:
    """Bytes of workspace that ``kv_attention`` needs for these sizes (0: none)."""
    if min(rows, q_heads, max_length) < 0:
        raise ValueError("rows, q_heads and max_length are not negative")
    return _workspace_bytes(pages, min(rows, _MOST), min(q_heads, _MOST), min(max_length, _MOST))


def _workspace_bytes(pages: KvPages, rows: int, q_heads: int, max_length: int) -> int:
    need = C.c_uint64()
    capi.check(capi.library().hllm_rocm_kv_attention_workspace(pages.address, rows, q_heads, max_length, C.byref(need)))
    return need.value
