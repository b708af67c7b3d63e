"""Caches by pages: a pool that sequences share, each with a table of its pages.

The reference gives every request a cache of its full length (mha.py:260-265); a
pool gives it a page of some positions when it gets there.  One layer's pool is
``[n_pages, page_size, 2, kv_heads, head_dim]``, a position's row as in the other
caches; position p of sequence b is row ``p % page_size`` of page ``tables[b, p //
page_size]`` (``tables`` int32 ``[batch, width]``, on the device; entries past a
sequence's last page are not looked at).  Strides are free but for the last dim:
``kv_pages`` lays a page's heads one after another, each with its keys and then
its values, which is what attention reads best.

The calls of one step take the same ``tables``, ``starts`` (int32 ``[batch]``: rows
cached before the step, negative for a sequence not in use) and ``cu_tokens``
(int32 ``[batch + 1]``: sequence b's new tokens are ``[cu_tokens[b], cu_tokens[b +
1])`` of the token tensors; None: an equal share each), so that single tokens and
chunks of prompts go through one call::

    q = paged.append(qkv, pages, tables, starts, q_heads=32, inv_freq=inv_freq, cu_tokens=cu)
    out = paged.attention(q, pages, tables, starts, max_seqlen=longest, cu_tokens=cu, max_tokens=most)

What these tensors hold is read on the device: a page outside the pool, a position past the
table or a length past ``max_seqlen`` is left out and flagged
(``ops.check_device_status``).  All work is enqueued on the current stream of the
tensors' device, as in ``ops``.
"""
from __future__ import annotations

import ctypes
import functools
from collections import OrderedDict
from typing import Optional, Sequence

import torch

from . import _lib
from .fp4 import _call, _int32, _layout
from .ops import (_DTYPES, TensorList, _as_layers, _check_lens, _layer_ptrs, _packed_ptrs, _ptr_array,
                  _require_device)


def kv_pages(n_pages: int, page_size: int, kv_heads: int, head_dim: int, dtype: torch.dtype, device,
             layers: Optional[int] = None) -> torch.Tensor:
    """One layer's pool, uninitialised as ``mha.inference_cache``'s caches are (``layers``: that many, stacked)."""
    shape = (n_pages, kv_heads, 2, page_size, head_dim)
    return torch.empty(shape if layers is None else (layers, *shape), dtype=dtype, device=device).transpose(-2, -4)


def pages_for(length: int, page_size: int) -> int:
    """Pages that hold ``length`` positions."""
    return -(-length // page_size)


@functools.lru_cache(maxsize=256)
def _pool_of(shape, stride, dtype, written: bool):
    """The checked ``hexkv_pool`` of a layer's pool."""
    if len(shape) != 5 or shape[2] != 2 or 0 in shape:
        raise ValueError(f"pages must be [n_pages, page_size, 2, kv_heads, head_dim], got {tuple(shape)}")
    if dtype not in _DTYPES:
        raise ValueError("pages must be one of float16, bfloat16, float32")
    if stride[4] != 1:
        raise ValueError("a head's elements must be contiguous")
    if written:
        span = 0
        for n, s in sorted(((n, s) for n, s in zip(shape, stride) if n > 1), key=lambda x: x[1]):
            if s <= span:
                raise ValueError("pages that are written must not share elements")
            span += (n - 1) * s
    p = _lib.Pool()
    p.dtype, p.kv_heads, p.head_dim = _DTYPES[dtype], _int32(shape[3], "kv_heads"), _int32(shape[4], "head_dim")
    p.n_pages, p.page_size = _int32(shape[0], "n_pages"), _int32(shape[1], "page_size")
    # (a stride of a dim of size 1 means nothing)
    p.page_stride, p.pos_stride, p.kv_stride, p.head_stride = (s if n > 1 else 0 for n, s in zip(shape[:4], stride))
    return p


def _check_pages(pages: torch.Tensor, written: bool) -> _lib.Pool:
    return _pool_of(pages.shape, pages.stride(), pages.dtype, written)


def _check_tables(tables: torch.Tensor, device) -> None:
    if tables.dtype != torch.int32 or tables.dim() != 2 or tables.device != device \
            or (tables.shape[1] > 1 and tables.stride(1) != 1):
        raise ValueError(f"tables must be int32 [batch, width] on {device} with contiguous rows, got {tables.dtype} "
                         f"{tuple(tables.shape)} on {tables.device}")


def _sequences(seqs: _lib.PagedBatch, tables, starts, cu_tokens, tokens: int, device) -> None:
    """Checks the tensors of a call's sequences and sets their sizes."""
    _check_tables(tables, device)
    batch, width = (_int32(n, "tables' size") for n in tables.shape)
    for t, n, name in ((starts, batch, "starts"), (cu_tokens, batch + 1, "cu_tokens")):
        if t is None and name == "cu_tokens":
            continue
        if t.dtype != torch.int32 or t.shape != (n,) or t.device != device or not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous int32 [{n}] on {device}")
    seqs.table_width, seqs.batch = width, batch
    seqs.table_stride = tables.stride(0) if batch > 1 else width
    seqs.tokens = _int32(tokens, "tokens")


def _set_sequences(seqs: _lib.PagedBatch, tables, starts, cu_tokens) -> None:
    """Sets the addresses of a call's sequences."""
    seqs.tables, seqs.starts = tables.data_ptr(), starts.data_ptr()
    if cu_tokens is not None:
        seqs.cu_tokens = cu_tokens.data_ptr()


def _token_rows(shape, stride, dims: int, name: str):
    """``(tokens, elements from token to token)`` of a tensor whose last ``dims`` dims are a token's."""
    inner = 1
    for n, s in zip(reversed(shape[-dims:]), reversed(stride[-dims:])):
        if n != 1 and s != inner:
            raise ValueError(f"a token's elements of {name} must be contiguous")
        inner *= n
    tokens, step, span = 1, inner, None
    for n, s in zip(reversed(shape[:-dims]), reversed(stride[:-dims])):
        tokens *= n
        if n == 1:
            continue
        if span is None:
            step, span = s, s
        if s != span:
            raise ValueError(f"the tokens of {name} must lie at one stride")
        span *= n
    return tokens, step


# The checked parameter blocks of append and attention, and the pools of the handoff, by what they depend on
# (shapes, strides, types, devices and options, never an address), as
# fp4.decode_attention keeps its own.
_FORMS: "OrderedDict[tuple, tuple]" = OrderedDict()


def _keep(key: tuple, form: tuple) -> tuple:
    _FORMS[key] = form
    while len(_FORMS) > 64:
        try:
            _FORMS.popitem(last=False)
        except KeyError:  # another thread emptied it
            break
    return form


def _append_form(qkv, pages, tables, starts, cu_tokens, q_heads, inv_freq, interleaved, rotary_scale, out):
    pool = _check_pages(pages, True)
    device, d = qkv.device, pool.head_dim
    width = (q_heads + 2 * pool.kv_heads) * d
    if qkv.dtype != pages.dtype or device != pages.device or qkv.dim() < 1 or q_heads < 0 or qkv.shape[-1] != width:
        raise ValueError(f"qkv must be [..., {width}] ({q_heads} + 2 x {pool.kv_heads} heads of {d}) like the pages, got "
                         f"{tuple(qkv.shape)} {qkv.dtype} on {device}")
    p = _lib.PagedAppendParams()
    p.pool = pool
    p.q_heads = _int32(q_heads, "q_heads")
    tokens, p.qkv_stride = _token_rows(qkv.shape, qkv.stride(), 1, "qkv")
    _sequences(p.seqs, tables, starts, cu_tokens, tokens, device)
    shape = torch.Size((*qkv.shape[:-1], q_heads, d))
    p.q_stride = q_heads * d
    if out is not None:
        if out.shape != shape or out.dtype != qkv.dtype or out.device != device:
            raise ValueError(f"out must be {tuple(shape)} like qkv, got {tuple(out.shape)} {out.dtype} on {out.device}")
        p.q_stride = _token_rows(out.shape, out.stride(), 2, "out")[1]
    if inv_freq is not None:
        if inv_freq.dtype != torch.float32 or inv_freq.dim() != 1 or 2 * inv_freq.shape[0] > d \
                or not inv_freq.is_contiguous() or inv_freq.device != device:
            raise ValueError(f"inv_freq must be contiguous float32, up to [{d // 2}], on {device}")
        p.rotary_dim = 2 * inv_freq.shape[0]
    p.interleaved, p.rotary_scale = 1 if interleaved else 0, rotary_scale
    return p, shape


def append(qkv: torch.Tensor, pages: torch.Tensor, tables: torch.Tensor, starts: torch.Tensor, *, q_heads: int,
           cu_tokens: Optional[torch.Tensor] = None, inv_freq: Optional[torch.Tensor] = None, interleaved: bool = False,
           rotary_scale: float = 1.0, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Rotate the new tokens' q and k heads to their positions, write k and v into
    the pages and return q, ``[..., q_heads, head_dim]`` (one launch).

    ``qkv [..., (q_heads + 2 kv_heads) * head_dim]`` are the joined product's rows
    (``q_heads`` 0: k and v alone).
    The first ``2 * len(inv_freq)`` dims of a head turn (None: no rotation), pair j by
    ``position * inv_freq[j]``, in pairs (j, j + half) or with ``interleaved`` (2j, 2j + 1); sines
    and cosines are multiplied by ``rotary_scale``.  (``rotary.frequencies`` makes these
    of a model's settings.)  Angles are reduced in 64 bits, so far positions
    lose nothing.  ``out`` may be q's part of ``qkv`` itself.  No two tokens may share a
    position of a page.  Tokens of no sequence, or of one not in use, are
    left as they were in ``out`` (and are not defined in a fresh one)."""
    q_heads, rotary_scale = int(q_heads), float(rotary_scale)
    key = (_layout(qkv), _layout(pages), _layout(tables), _layout(starts), _layout(cu_tokens), _layout(inv_freq),
           _layout(out), q_heads, bool(interleaved), rotary_scale)
    form = _FORMS.get(key)
    if form is None:
        _require_device(qkv, pages, tables, starts)
        form = _keep(key, _append_form(qkv, pages, tables, starts, cu_tokens, q_heads, inv_freq, interleaved, rotary_scale, out))
    p = _lib.PagedAppendParams.from_buffer_copy(form[0])
    if out is None:
        out = qkv.new_empty(form[1])
    p.qkv, p.q, p.pages = qkv.data_ptr(), out.data_ptr() if q_heads else None, pages.data_ptr()
    _set_sequences(p.seqs, tables, starts, cu_tokens)
    if inv_freq is not None:
        p.inv_freq = inv_freq.data_ptr()
    _call("hexkv_paged_append", qkv, ctypes.byref(p))
    return out


def _attend_form(q, pages, tables, starts, cu_tokens, max_tokens, causal, softmax_scale, out, partition):
    pool = _check_pages(pages, False)
    device, d = q.device, pool.head_dim
    if q.dim() < 2 or q.dtype != pages.dtype or device != pages.device or q.shape[-1] != d or q.shape[-2] < 1 \
            or q.shape[-2] % pool.kv_heads:
        raise ValueError(f"q must be [..., q_heads, {d}] like the pages, with a multiple of {pool.kv_heads} heads, got "
                         f"{tuple(q.shape)} {q.dtype} on {device}")
    if out is not None and (out.shape != q.shape or out.dtype != q.dtype or out.device != device):
        raise ValueError("out must share q's shape, dtype and device")
    p = _lib.PagedAttendParams()
    p.pool = pool
    p.q_heads = _int32(q.shape[-2], "q_heads")
    tokens, p.q_stride = _token_rows(q.shape, q.stride(), 2, "q")
    p.out_stride = p.q_heads * d if out is None else _token_rows(out.shape, out.stride(), 2, "out")[1]
    _sequences(p.seqs, tables, starts, cu_tokens, tokens, device)
    p.causal, p.max_tokens = 1 if causal else 0, _int32(max_tokens, "max_tokens")
    p.softmax_scale = d ** -0.5 if softmax_scale is None else softmax_scale
    p.partition = _int32(partition, "partition")
    return p, {}


def attention(q: torch.Tensor, pages: torch.Tensor, tables: torch.Tensor, starts: torch.Tensor, *, max_seqlen: int,
              cu_tokens: Optional[torch.Tensor] = None, max_tokens: int = 1, causal: bool = True,
              softmax_scale: Optional[float] = None, out: Optional[torch.Tensor] = None,
              workspace: Optional[torch.Tensor] = None, partition: int = 0) -> torch.Tensor:
    """Attention of the new tokens ``q [..., q_heads, head_dim]`` over their
    sequences' rows in the pages, their own (appended before) included.

    Token i of a sequence sees its first ``starts + i + 1`` rows, without ``causal``
    all that the sequence has.  ``max_seqlen`` bounds a sequence's rows and, with ``cu_tokens``,
    ``max_tokens`` its new tokens: both are host values that size the launch.
    Softmax sums are fp32.  ``out`` may be ``q``; tokens of no sequence, and those past
    ``max_tokens`` of one (flagged, but for ``max_tokens`` 0, which launches nothing), are left as they
    were in it (and are not defined in a fresh one), those of a sequence not in use become zero.  ``partition``: rows
    per partition of a split row, a multiple of 64 (0: the library's choice); ``workspace``:
    scratch that no overlapping call shares (default: one of this call's own)."""
    softmax_scale = None if softmax_scale is None else float(softmax_scale)
    key = (_layout(q), _layout(pages), _layout(tables), _layout(starts), _layout(cu_tokens), _layout(out), int(max_tokens),
           bool(causal), softmax_scale, int(partition))
    form = _FORMS.get(key)
    if form is None:
        _require_device(q, pages, tables, starts)
        form = _keep(key, _attend_form(q, pages, tables, starts, cu_tokens, max_tokens, causal, softmax_scale, out, partition))
    p, needs = _lib.PagedAttendParams.from_buffer_copy(form[0]), form[1]
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    p.q, p.out, p.pages = q.data_ptr(), out.data_ptr(), pages.data_ptr()
    _set_sequences(p.seqs, tables, starts, cu_tokens)
    p.max_seqlen = _int32(max_seqlen, "max_seqlen")
    need = needs.get(p.max_seqlen)
    if need is None:
        need = int(_lib.load().hexkv_paged_attend_workspace_bytes(ctypes.byref(p)))
        if len(needs) >= 64:
            needs.clear()
        needs[p.max_seqlen] = need
    at, size = None, 0
    if need:
        if workspace is None:
            workspace = q.new_empty(need, dtype=torch.uint8)
        elif workspace.device != q.device or not workspace.is_contiguous():
            raise ValueError(f"workspace must be contiguous on {q.device}")
        at, size = workspace.data_ptr(), workspace.numel() * workspace.element_size()
    _call("hexkv_paged_attend", q, ctypes.byref(p), at, size)
    return out


def attend_workspace_bytes(q: torch.Tensor, pages: torch.Tensor, tables: torch.Tensor, starts: torch.Tensor, *,
                           max_seqlen: int, cu_tokens: Optional[torch.Tensor] = None, max_tokens: int = 1,
                           causal: bool = True, partition: int = 0) -> int:
    """Workspace bytes ``attention`` needs for this geometry and these bounds (0: none)."""
    p, _ = _attend_form(q, pages, tables, starts, cu_tokens, max_tokens, causal, None, None, partition)
    _set_sequences(p.seqs, tables, starts, cu_tokens)
    p.max_seqlen = _int32(max_seqlen, "max_seqlen")
    lib = _lib.load()
    need = int(lib.hexkv_paged_attend_workspace_bytes(ctypes.byref(p)))
    if not need and lib.hexkv_last_error():  # bounds that attention refuses, too
        raise ValueError(lib.hexkv_last_error().decode())
    return need


def _copy_layers(pages_layers: TensorList, tables, lens, written: bool):
    """First layer, addresses, pool and checked lengths of a handoff call."""
    if isinstance(pages_layers, torch.Tensor):
        key = (_layout(pages_layers), _layout(tables), written)
        form = _FORMS.get(key)
        if form is None:
            if pages_layers.dim() != 6 or not pages_layers.shape[0]:
                raise ValueError("stacked pages must be [n_layers, n_pages, page_size, 2, kv_heads, head_dim]")
            _require_device(pages_layers, tables)
            pool = _pool_of(pages_layers.shape[1:], pages_layers.stride()[1:], pages_layers.dtype, written)
            if written and pages_layers.shape[0] > 1 and pages_layers.stride(0) == 0:
                raise ValueError("layers that are written must not share pages")
            _check_tables(tables, pages_layers.device)
            form = _keep(key, (pool,))
        return pages_layers, _layer_ptrs(pages_layers), form[0], _check_lens(lens, tables.shape[0])
    layers = _as_layers(pages_layers)
    if not layers:
        raise ValueError("no layers")
    _require_device(tables, *layers)
    first = layers[0]
    pool = _check_pages(first, written)
    if any(t.shape != first.shape or t.stride() != first.stride() or t.dtype != first.dtype or t.device != first.device
           for t in layers):
        raise ValueError("all layers must share shape, strides, dtype and device")
    _check_tables(tables, first.device)
    return first, _ptr_array([t.data_ptr() for t in layers]), pool, _check_lens(lens, tables.shape[0])


def _packed(packed: TensorList, n_layers: int, total: int, pool: _lib.Pool, first: torch.Tensor):
    """Addresses of the packed layers, checked once a form where they are stacked."""
    if not isinstance(packed, torch.Tensor):
        return _packed_ptrs(packed, n_layers, total, 2 * pool.kv_heads * pool.head_dim, first.dtype, first.device)
    key = (_layout(packed), n_layers, total, pool.kv_heads, pool.head_dim, first.dtype, first.get_device())
    if key not in _FORMS:
        _packed_ptrs(packed, n_layers, total, 2 * pool.kv_heads * pool.head_dim, first.dtype, first.device)
        _keep(key, ())
    return _layer_ptrs(packed)


def _copy(name, pool, source, target, n_layers, tables, lens, first) -> None:
    _call(name, first, ctypes.byref(pool), source, target, n_layers, tables.data_ptr(),
          tables.stride(0) if tables.shape[0] > 1 else tables.shape[1], _int32(tables.shape[1], "tables' width"), len(lens),
          (ctypes.c_int64 * len(lens))(*lens))


def pack_live(pages_layers: TensorList, tables: torch.Tensor, lens: Sequence[int],
              out: Optional[TensorList] = None) -> TensorList:
    """``ops.pack_live`` of a paged cache: rows ``[0, lens[b])`` of every sequence
    of every layer into the handoff layout ``[n_layers, sum(lens), 2, kv_heads,
    head_dim]``, one launch.  ``pages_layers``: the layers' pools, a list or stacked,
    with one ``tables`` for all.  The rows of a page outside the pool come out as zeros.
    ``out`` must not overlap the pools."""
    first, ptrs, pool, lens = _copy_layers(pages_layers, tables, lens, False)
    if out is None:
        out = first.new_empty((len(ptrs), sum(lens), 2, pool.kv_heads, pool.head_dim))
        dst = _layer_ptrs(out)
    else:
        dst = _packed(out, len(ptrs), sum(lens), pool, first)
    _copy("hexkv_paged_pack", pool, ptrs, dst, len(ptrs), tables, lens, first)
    return out


def unpack_live(packed: TensorList, pages_layers: TensorList, tables: torch.Tensor, lens: Sequence[int]) -> None:
    """``ops.unpack_live`` into a paged cache: the packed handoff layout into the
    pages that ``tables`` names; all other rows are left untouched.  No two
    sequences may share a page here."""
    first, ptrs, pool, lens = _copy_layers(pages_layers, tables, lens, True)
    src = _packed(packed, len(ptrs), sum(lens), pool, first)
    _copy("hexkv_paged_unpack", pool, src, ptrs, len(ptrs), tables, lens, first)
