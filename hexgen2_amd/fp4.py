"""Caches and weights in four bits: the OCP microscaling format MXFP4, blocks of
32 consecutive elements that share a power of two (4.25 bits an element).

The reference holds both in the data type, 3.76 times the bytes.  How much of
the time that saves depends on the call (MI355X, us, four bits against 16): attention of
a Llama-3-8B layer, 64 sequences of 128 to 8192, 81 against 156; of one sequence
of 577, 6.8 against 6.0; a product of one token, 22528 x 4096, 11 against 30.  A 4-bit
cache is one layer's uint8 ``[batch, capacity, row_bytes(kv_heads, head_dim)]``,
a row one position's K and V of every KV head like the 16-bit cache's, so
``ops.pack_live`` and ``ops.unpack_live`` hand it over unchanged.  A 4-bit matrix
is an ``Fp4Tensor``: ``codes [n, k / 2]`` (two elements a byte, the earlier one in
the lower half) and ``powers [n, k / 32]`` (byte b: 2^(b - 127), 255: NaN), both
uint8, which is also how MXFP4 checkpoints hold their matrices.

What the functions here write has the smallest power that leaves no element of
its block above 6 times it, every element rounded to the nearest of 0, 0.5, 1,
1.5, 2, 3, 4 and 6 times the power (halfway: to the even code); a block that
holds an infinity or a NaN becomes NaN.  All work is enqueued on the
current stream of the tensors' device, as in ``ops``.
"""
from __future__ import annotations

import ctypes
import functools
from collections import OrderedDict
from typing import NamedTuple, Optional

import torch

from . import _lib
from .ops import _DTYPES, _raw_stream, _require_device, _stream

BLOCK = 32

# (torch's own accessor, as ``_raw_stream``: 0.1 us a call less)
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


class Fp4Tensor(NamedTuple):
    """A matrix ``[n, k]`` in four bits."""
    codes: torch.Tensor
    powers: torch.Tensor


@functools.lru_cache(maxsize=None)
def row_bytes(kv_heads: int, head_dim: int) -> int:
    """Bytes of one position's row in a 4-bit cache: its elements, their
    powers, and what fills them up to a multiple of 16."""
    if kv_heads < 1 or head_dim < BLOCK or head_dim % BLOCK:
        raise ValueError(f"head_dim {head_dim} must be a positive multiple of {BLOCK}")
    return -(-2 * kv_heads * (head_dim // 2 + head_dim // BLOCK) // 16) * 16


def kv_cache(batch: int, capacity: int, kv_heads: int, head_dim: int, device) -> torch.Tensor:
    """One layer's 4-bit cache, uninitialised as ``mha.inference_cache``'s is."""
    return torch.empty((batch, capacity, row_bytes(kv_heads, head_dim)), dtype=torch.uint8, device=device)


@functools.lru_cache(maxsize=256)
def _cache_geometry(shape, stride, kv_heads: int, head_dim: int):
    """(batch stride, row stride) in bytes of a 4-bit cache."""
    if len(shape) != 3 or shape[2] != row_bytes(kv_heads, head_dim):
        raise ValueError(f"a 4-bit cache of {kv_heads} heads of {head_dim} is [batch, capacity, "
                         f"{row_bytes(kv_heads, head_dim)}], got {tuple(shape)}")
    if stride[2] != 1 or (shape[1] > 1 and stride[1] < shape[2]) or (shape[0] > 1 and stride[0] < shape[1] * stride[1]):
        raise ValueError("cache rows must be contiguous and must not overlap")
    row = stride[1] if shape[1] > 1 else shape[2]
    return (stride[0] if shape[0] > 1 else shape[1] * row), row


def _check_cache(cache: torch.Tensor, kv_heads: int, head_dim: int):
    if cache.dtype != torch.uint8:
        raise ValueError(f"a 4-bit cache is uint8, got {cache.dtype}")
    return _cache_geometry(cache.shape, cache.stride(), kv_heads, head_dim)


def _counts(t: Optional[torch.Tensor], batch: int, device, name: str) -> Optional[int]:
    """Address of a device int32 tensor with one entry per sequence."""
    if t is None:
        return None
    if t.dtype != torch.int32 or t.device != device or t.numel() < batch or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 tensor with one entry per sequence on {device}")
    return t.data_ptr()


def _int32(value: int, name: str) -> int:
    """``value`` as the library's 32-bit argument (ctypes would wrap it)."""
    value = int(value)
    if not -(1 << 31) <= value < 1 << 31:
        raise ValueError(f"{name} {value} does not fit 32 bits")
    return value


def _call(name: str, tensor: torch.Tensor, *args) -> None:
    """One library call on the current stream of ``tensor``'s device."""
    fn = getattr(_lib.load(), name)
    index = tensor.get_device()
    if index == _current_device():
        rc = fn(*args, _raw_stream(index) if _raw_stream is not None else _stream(tensor))
    else:
        with torch.cuda.device(tensor.device):
            rc = fn(*args, _stream(tensor))
    if rc:
        _lib.check(rc, name)


@functools.lru_cache(maxsize=256)
def _rows_form(shape, stride, dtype):
    """``shape, stride`` and type code of checked rows (by what they depend on:
    most of a small call's time is the host's)."""
    if len(shape) != 5 or shape[2] != 2:
        raise ValueError(f"kv must be [batch, positions, 2, kv_heads, head_dim], got {tuple(shape)}")
    if dtype not in _DTYPES:
        raise ValueError("kv must be one of float16, bfloat16, float32")
    if stride[4] != 1 or (shape[3] > 1 and stride[3] != shape[4]):
        raise ValueError("kv heads must be contiguous [.., heads, head_dim]")
    for n in shape:
        _int32(n, "kv's size")
    return (*shape, *stride[:3], _DTYPES[dtype])


def store_kv(cache: torch.Tensor, kv: torch.Tensor, positions: Optional[torch.Tensor] = None,
             position_bias: int = 0) -> None:
    """Write the rows ``kv [b, s, 2, kv_heads, head_dim]`` into sequences
    ``[0, b)`` of a 4-bit cache at positions ``positions[b] + position_bias +
    [0, s)`` (``positions`` a device int32 tensor, or None for one offset).
    A row whose position, read from device memory, lies outside the cache is
    not written and flagged (``ops.check_device_status``)."""
    _require_device(cache, kv)
    b, s, _, heads, d, *strides, dtype = _rows_form(kv.shape, kv.stride(), kv.dtype)
    batch_bytes, row = _check_cache(cache, heads, d)
    if cache.device != kv.device or cache.shape[0] < b:
        raise ValueError(f"cache of {cache.shape[0]} sequences on {cache.device} for kv of {b} on {kv.device}")
    at = _counts(positions, b, kv.device, "positions")
    _call("hexkv_mx_store", kv, kv.data_ptr(), *strides, cache.data_ptr(), batch_bytes, row, cache.shape[1], b, s, heads, d,
          dtype, at, _int32(position_bias, "position_bias"))


def load_kv(cache: torch.Tensor, length: int, kv_heads: int, head_dim: int, dtype: torch.dtype,
            positions: Optional[torch.Tensor] = None, position_bias: int = 0, *,
            out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The mirror of ``store_kv``: positions ``positions[b] + position_bias +
    [0, length)`` of every sequence as ``[batch, length, 2, kv_heads, head_dim]``
    of ``dtype`` (``out``, if given, with heads contiguous).  Rows outside the
    cache come back as zeros and are flagged."""
    _require_device(cache)
    batch_bytes, row = _check_cache(cache, kv_heads, head_dim)
    b, length = cache.shape[0], _int32(length, "length")
    if dtype not in _DTYPES or length < 0:
        raise ValueError("load_kv gives float16, bfloat16 or float32 rows, none or more of them")
    if out is None:
        out = cache.new_empty((b, length, 2, kv_heads, head_dim), dtype=dtype)
    elif out.shape != (b, length, 2, kv_heads, head_dim) or out.dtype != dtype or out.device != cache.device:
        raise ValueError(f"out must be {dtype} [{b}, {length}, 2, {kv_heads}, {head_dim}] on {cache.device}")
    *_, s0, s1, s2, code = _rows_form(out.shape, out.stride(), dtype)
    if 0 in (s0, s1, s2) and any(s == 0 and n > 1 for s, n in zip((s0, s1, s2), out.shape)):
        raise ValueError("out's rows must not overlap")
    at = _counts(positions, b, cache.device, "positions")
    _call("hexkv_mx_load", cache, cache.data_ptr(), batch_bytes, row, cache.shape[1], out.data_ptr(), s0, s1, s2,
          b, length, kv_heads, head_dim, code, at, _int32(position_bias, "position_bias"))
    return out


def _attend_form(q, cache, kv_heads, out, kv_new, causal, softmax_scale, partition) -> _lib.MxAttendParams:
    """The checked parameter block of a call, without addresses and lengths."""
    if q.dim() != 4 or q.dtype not in _DTYPES:
        raise ValueError("q must be [batch, q_len, q_heads, head_dim] in float16, bfloat16 or float32")
    batch, q_len, q_heads, d = (_int32(n, "q's size") for n in q.shape)
    if kv_heads < 1 or q_heads % kv_heads:
        raise ValueError("q_heads must be a multiple of kv_heads")
    batch_bytes, row = _check_cache(cache, kv_heads, d)
    if cache.shape[0] < batch or cache.device != q.device:
        raise ValueError(f"cache of {cache.shape[0]} sequences on {cache.device} for q of {batch} on {q.device}")
    if out is not None and (out.shape != q.shape or out.dtype != q.dtype or out.device != q.device):
        raise ValueError("out must share q's shape, dtype and device")
    for name, t in (("q", q), ("out", out)):
        if t is not None and (t.stride(3) != 1 or (t.shape[2] > 1 and t.stride(2) != d)):
            raise ValueError(f"{name} heads must be contiguous [.., heads, head_dim]")
    if kv_new is not None and (kv_new.dtype != q.dtype or kv_new.device != q.device
                               or kv_new.numel() != batch * 2 * kv_heads * d or not kv_new.is_contiguous()):
        raise ValueError("kv_new must be contiguous [batch, 2, kv_heads, head_dim] like q")
    p = _lib.MxAttendParams()
    p.dtype, p.batch, p.q_len, p.q_heads, p.kv_heads, p.head_dim = _DTYPES[q.dtype], batch, q_len, q_heads, kv_heads, d
    p.causal = 1 if causal else 0
    p.softmax_scale = d ** -0.5 if softmax_scale is None else softmax_scale
    p.q_batch_stride, p.q_row_stride = q.stride()[:2]
    p.cache_batch_bytes, p.cache_row_bytes = batch_bytes, row
    # (a fresh output is contiguous)
    p.out_batch_stride, p.out_row_stride = (q_len * q_heads * d, q_heads * d) if out is None else out.stride()[:2]
    p.partition = _int32(partition, "partition")
    return p


# decode_attention's checked blocks by what they depend on (shapes, strides, types,
# devices and options, never an address), each with the workspace bytes per
# max_seqlen: a decode loop's calls differ in their lengths alone.
_FORMS: "OrderedDict[tuple, tuple]" = OrderedDict()


def _layout(t: Optional[torch.Tensor]):
    return None if t is None else (t.shape, t.stride(), t.dtype, t.get_device())


def decode_attention(q: torch.Tensor, cache: torch.Tensor, kv_heads: int, *, max_seqlen: int,
                     seqlens: Optional[torch.Tensor] = None, seqlen_bias: int = 0,
                     kv_new: Optional[torch.Tensor] = None, causal: bool = False,
                     softmax_scale: Optional[float] = None, out: Optional[torch.Tensor] = None,
                     workspace: Optional[torch.Tensor] = None, partition: int = 0) -> torch.Tensor:
    """``ops.decode_attention`` over a 4-bit cache: ``q [B, q_len, Hq, D]``, row b
    over its first ``seqlens[b] + seqlen_bias`` keys, with ``kv_new [B, 2, Hkv, D]``
    appended first (and attended as stored), with ``causal`` and ``q_len > 1``
    query t over ``q_len - 1 - t`` keys fewer than the last.  ``max_seqlen``
    bounds the attended length (the new row included).  ``partition``:
    positions per partition of a split row, a multiple of 32 (0: the
    library's choice); ``workspace``: scratch that is not shared with
    an overlapping call (default: one of this call's own)."""
    _require_device(q, cache)
    kv_heads = int(kv_heads)
    softmax_scale = None if softmax_scale is None else float(softmax_scale)
    shape = cache.shape
    key = (_layout(q), shape[0], shape[1] == 1, shape[2:], cache.stride(), cache.dtype, cache.get_device(), kv_heads, _layout(out),
           _layout(kv_new), bool(causal), softmax_scale, int(partition))
    form = _FORMS.get(key)
    if form is None:
        form = _attend_form(q, cache, kv_heads, out, kv_new, causal, softmax_scale, partition), {}
        _FORMS[key] = form
        while len(_FORMS) > 64:
            try:
                _FORMS.popitem(last=False)
            except KeyError:  # another thread emptied it
                break
    p, needs = _lib.MxAttendParams.from_buffer_copy(form[0]), form[1]
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    p.q, p.cache, p.out, p.capacity = q.data_ptr(), cache.data_ptr(), out.data_ptr(), shape[1]
    if kv_new is not None:
        p.kv_new = kv_new.data_ptr()
    p.seqlens_dev = _counts(seqlens, p.batch, q.device, "seqlens")
    p.seqlen_bias, p.max_seqlen = _int32(seqlen_bias, "seqlen_bias"), _int32(max_seqlen, "max_seqlen")
    if not 0 <= p.max_seqlen <= p.capacity:
        raise ValueError(f"max_seqlen {max_seqlen} outside [0, capacity {p.capacity}]")
    need = needs.get((p.max_seqlen, p.q % 16))
    if need is None:
        need = int(_lib.load().hexkv_mx_attend_workspace_bytes(ctypes.byref(p)))
        if len(needs) >= 64:
            needs.clear()
        needs[p.max_seqlen, p.q % 16] = need
    at, size = None, 0
    if need:
        if workspace is None:
            workspace = cache.new_empty(need)
        elif workspace.device != q.device or not workspace.is_contiguous():
            raise ValueError(f"workspace must be contiguous on {q.device}")
        at, size = workspace.data_ptr(), workspace.numel() * workspace.element_size()
    _call("hexkv_mx_attend", q, ctypes.byref(p), at, size)
    return out


def attend_workspace_bytes(q: torch.Tensor, cache: torch.Tensor, kv_heads: int, max_seqlen: int,
                           partition: int = 0, causal: bool = False) -> int:
    """Workspace bytes ``decode_attention`` needs for this geometry and bound."""
    p = _attend_form(q, cache, int(kv_heads), None, None, causal, None, partition)
    p.q, p.capacity, p.max_seqlen = q.data_ptr(), cache.shape[1], _int32(max_seqlen, "max_seqlen")
    return int(_lib.load().hexkv_mx_attend_workspace_bytes(ctypes.byref(p)))


def _row_stride(shape, stride, name: str) -> int:
    """Elements between consecutive rows (last dim) of a tensor whose outer dims
    fold into one."""
    if len(shape) == 2 and stride[1] == 1 and shape[0] > 1:
        return stride[0]
    step = 1
    for n, at in zip(reversed(shape), reversed(stride)):
        if n != 1 and at != step and 0 not in shape:
            raise ValueError(f"{name} rows must be contiguous and lie at one stride")
        step *= n
    return shape[-1]


def _matrix_rows(t: torch.Tensor, name: str) -> int:
    return _row_stride(t.shape, t.stride(), name)


def _matrix_size(shape) -> int:
    """Elements of a matrix's row."""
    return _int32(shape[-1], "a row of elements")


def quantize(x: torch.Tensor) -> Fp4Tensor:
    """``x [..., k]`` (k a multiple of 32) in four bits: ``codes [..., k / 2]``
    and ``powers [..., k / 32]``."""
    _require_device(x)
    if x.dtype not in _DTYPES or x.dim() < 1 or x.shape[-1] % BLOCK:
        raise ValueError(f"x must be float16, bfloat16 or float32 with rows of whole blocks of {BLOCK}, "
                         f"got {x.dtype} {tuple(x.shape)}")
    k = _matrix_size(x.shape)
    stride = _matrix_rows(x, "x")
    codes = torch.empty((*x.shape[:-1], k // 2), dtype=torch.uint8, device=x.device)
    powers = torch.empty((*x.shape[:-1], k // BLOCK), dtype=torch.uint8, device=x.device)
    _call("hexkv_mx_quantize", x, x.data_ptr(), stride, codes.data_ptr(), powers.data_ptr(), x.numel() // max(k, 1), k,
          _DTYPES[x.dtype])
    return Fp4Tensor(codes, powers)


@functools.lru_cache(maxsize=1024)
def _is_matrix(codes_shape, powers_shape) -> bool:
    return (len(codes_shape) >= 1 and codes_shape[:-1] == powers_shape[:-1]
            and codes_shape[-1] == powers_shape[-1] * (BLOCK // 2))


def _check_matrix(weight: Fp4Tensor):
    codes, powers = weight
    if codes.dtype != torch.uint8 or powers.dtype != torch.uint8 or codes.get_device() != powers.get_device() \
            or not _is_matrix(codes.shape, powers.shape) or not codes.is_contiguous() or not powers.is_contiguous():
        raise ValueError(f"a 4-bit tensor is contiguous uint8 codes [..., k / 2] and powers [..., k / {BLOCK}] on one "
                         f"device, got {tuple(codes.shape)} and {tuple(powers.shape)}")
    return codes, powers


def dequantize(weight: Fp4Tensor, dtype: torch.dtype) -> torch.Tensor:
    """The values of a 4-bit tensor, rounded to ``dtype``."""
    codes, powers = _check_matrix(weight)
    _require_device(codes)
    if dtype not in _DTYPES:
        raise ValueError("dequantize gives float16, bfloat16 or float32")
    k = _matrix_size((*powers.shape[:-1], powers.shape[-1] * BLOCK))
    out = torch.empty((*codes.shape[:-1], k), dtype=dtype, device=codes.device)
    _call("hexkv_mx_dequantize", codes, codes.data_ptr(), powers.data_ptr(), out.data_ptr(), k,
          out.numel() // max(k, 1), k, _DTYPES[dtype])
    return out


@functools.lru_cache(maxsize=1024)
def _linear_form(shape, stride, dtype, codes_shape, powers_shape):
    """A product's tokens, rows, inner dimension, token stride, type code,
    output shape and workspace bytes."""
    if len(codes_shape) != 2 or dtype not in _DTYPES or not shape or shape[-1] != codes_shape[1] * 2:
        raise ValueError(f"x {dtype} {tuple(shape)} does not fit a matrix [{codes_shape[0]}, {codes_shape[-1] * 2}]")
    n, k = codes_shape[0], shape[-1]
    if not k:
        raise ValueError("a product needs a block of elements")
    k, rows, n, code = _int32(k, "k"), _int32(shape.numel() // k, "tokens"), _int32(n, "rows"), _DTYPES[dtype]
    return (rows, n, k, _row_stride(shape, stride, "x"), code, torch.Size((*shape[:-1], n)),
            int(_lib.load().hexkv_mx_linear_workspace_bytes(rows, n, k, code)))


def linear(x: torch.Tensor, weight: Fp4Tensor) -> torch.Tensor:
    """``x @ weight.T`` for ``x [..., k]`` and a 4-bit matrix ``[n, k]``: sums in
    fp32 over the weights' exact values, rounded once to ``x``'s type."""
    codes, powers = _check_matrix(weight)
    _require_device(x, codes)
    if x.device != codes.device:
        raise ValueError(f"x on {x.device} for a matrix on {codes.device}")
    rows, n, k, stride, dtype, shape, need = _linear_form(x.shape, x.stride(), x.dtype, codes.shape, powers.shape)
    out = x.new_empty(shape)
    workspace = codes.new_empty(need) if need else None
    _call("hexkv_mx_linear", x, x.data_ptr(), stride, codes.data_ptr(), powers.data_ptr(), out.data_ptr(), rows, n, k, dtype,
          workspace.data_ptr() if need else None, need)
    return out
