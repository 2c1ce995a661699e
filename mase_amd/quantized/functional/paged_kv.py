"""Functions on a paged key-value cache: writing new tokens (with MX quantization on the way), reading sequences back
dense, attention of one new token, and eviction by accumulated attention weight.

They hold what the reference's quantized attention modules keep through ``kv_cache_mxfp`` / ``kv_cache_mxint`` and
``past_key_value.update`` (``chop/nn/quantized/functional/kvcache.py:8-43``,
``chop/nn/quantized/modules/llama/attention.py:182-187``) as codes in pages instead of fake-quantized 16-bit values, and
compute the attention core of a decoding step (``chop/models/llama/modeling_llama.py:362-480``) from the pages directly.
``mase_amd.quantized.PagedKVCache`` is the cache object built on them.

Arguments that all of them share:

``k_pages``, ``v_pages``  ``[pages, kv_heads, page_size, head_dim]`` (``kv_format="mxfp4"``: ``head_dim / 2``, the even
    element in the low half of a byte); bfloat16 / float16 with ``kv_format=None``, int8 codes with ``"mxint8"``, uint8
    codes with ``"mxfp8_e4m3"``, ``"mxfp8_e5m2"`` and ``"mxfp4"``.  Rows contiguous, the other strides free (multiples of
    16 bytes).  ``head_dim`` 64, 128 or 256, ``page_size`` a power of two from 16 to 4096.
``k_scales``, ``v_scales``  uint8 ``[pages, kv_heads, page_size, head_dim / 32]`` and ``[pages, kv_heads, head_dim / 32,
    page_size]``, contiguous (codes only).  Values are ``code * 2^(scale - 134)`` (MXINT8) or ``element * 2^(scale - 127)``;
    scale 255 stands for a block of NaN.
``page_table``  int32 ``[batch, table_pages]``: slot t of sequence b is row ``t % page_size`` of page
    ``page_table[b, t // page_size]``.

Lengths, slots and page numbers live on the device and are not looked at on the host (no call synchronizes, all can be
captured into a graph): a length counts for at most ``max_length``, and a page number outside the pool is never followed,
its slots being absent.  Inference only: tensors that record gradients are refused while gradients are enabled.
"""
from __future__ import annotations

import struct
from functools import lru_cache
from typing import Optional, Tuple

import torch
from torch import Tensor

from ... import _lib
from ..._tables import log2_table

KV_FORMATS = tuple(_lib.KV_FORMATS)
_HEAD_DIMS = (64, 128, 256)
_STATE_CODES = {torch.bfloat16: _lib.DT_BF16, torch.float16: _lib.DT_F16}
_raw_stream = torch._C._cuda_getCurrentRawStream
_current_device = torch._C._cuda_getDevice


def _int32(t: Tensor, name: str, shape, device) -> int:
    if t.dtype != torch.int32 or t.shape != shape or t.device != device or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 tensor of shape {tuple(shape)} on {device}, got {t.dtype} "
                         f"{tuple(t.shape)} on {t.device}")
    return t.data_ptr()


# mase_paged_kv of the C ABI as one packed record (the layout of _lib.PagedKv, which a test compares)
_record = struct.Struct("@5P13N2i").pack


class _Pool:
    """a pool after the checks that the host can make: its record for the C ABI and the sizes that the callers look at"""

    __slots__ = ("record", "device", "batch", "kv_heads", "head_dim", "slots", "format")

    def __init__(self, what: str, k_pages: Tensor, v_pages: Tensor, page_table: Tensor, kv_format, k_scales, v_scales, dtype):
        code = _lib.KV_FORMATS.get(kv_format)
        if code is None:
            raise ValueError(f"{what}: kv_format must be one of {KV_FORMATS}, got {kv_format!r}")
        if not k_pages.is_cuda:
            _lib.require_device(k_pages, what)
        device = self.device = k_pages.device
        shape = k_pages.shape
        if len(shape) != 4 or v_pages.shape != shape:
            raise ValueError(f"{what}: k_pages and v_pages must be [pages, kv_heads, page_size, head_dim] alike, got "
                             f"{tuple(shape)} and {tuple(v_pages.shape)}")
        pages, heads, page_size, width = shape
        head_dim = 2 * width if code == 4 else width
        if head_dim not in _HEAD_DIMS:
            raise ValueError(f"{what}: head_dim must be one of {_HEAD_DIMS}, got {head_dim}")
        if page_size < 16 or page_size > 4096 or page_size & (page_size - 1):
            raise ValueError(f"{what}: page_size must be a power of two from 16 to 4096, got {page_size}")
        dtype_code = _STATE_CODES.get(dtype)
        if dtype_code is None:
            raise ValueError(f"{what}: states must be bfloat16 or float16, got {dtype}")
        want = dtype if code == 0 else (torch.int8 if code == 1 else torch.uint8)
        if k_pages.dtype != want or v_pages.dtype != want:
            raise ValueError(f"{what}: pages must be {want} for kv_format={kv_format!r} and {dtype} states, got {k_pages.dtype} "
                             f"and {v_pages.dtype}")
        kp, kh, ks, k1 = k_pages.stride()
        vp, vh, vs, v1 = v_pages.stride()
        if v_pages.device != device or k1 != 1 or v1 != 1:
            raise ValueError(f"{what}: k_pages and v_pages must be on one device with contiguous rows")
        # strides of dimensions of size one mean nothing; a stride of zero would have pages or heads share their memory
        if pages == 1:
            kp = vp = 16
        if heads == 1:
            kh = vh = 16
        if not (kp and kh and ks and vp and vh and vs):
            raise ValueError(f"{what}: k_pages and v_pages must not be expanded tensors")
        if page_table.dim() != 2 or page_table.dtype != torch.int32 or page_table.device != device:
            raise ValueError(f"{what}: page_table must be an int32 tensor [batch, table_pages] on {device}")
        batch, table_pages = page_table.shape
        tb, t1 = page_table.stride()
        if batch <= 1:
            tb = table_pages
        if tb < table_pages or (t1 != 1 and table_pages > 1):
            raise ValueError(f"{what}: page_table must have contiguous rows, each sequence its own")
        sk = sv = 0
        if code:
            if k_scales is None or v_scales is None:
                raise ValueError(f"{what}: kv_format={kv_format!r} needs k_scales and v_scales")
            for name, t, want_shape in (("k_scales", k_scales, (pages, heads, page_size, head_dim // 32)),
                                        ("v_scales", v_scales, (pages, heads, head_dim // 32, page_size))):
                if t.dtype != torch.uint8 or t.shape != want_shape or t.device != device or not t.is_contiguous():
                    raise ValueError(f"{what}: {name} must be a contiguous uint8 tensor {want_shape} on {device}, got {t.dtype} "
                                     f"{tuple(t.shape)} on {t.device}")
            sk, sv = k_scales.data_ptr(), v_scales.data_ptr()
        item = 2 if code == 0 else 1
        self.batch, self.kv_heads, self.head_dim, self.slots, self.format = batch, heads, head_dim, table_pages * page_size, code
        self.record = _record(k_pages.data_ptr(), v_pages.data_ptr(), sk, sv, page_table.data_ptr(), pages, page_size, heads, head_dim,
                              batch, table_pages, tb, kp * item, kh * item, ks * item, vp * item, vh * item, vs * item, code,
                              dtype_code)


_entry = {}  # entry points of the library by name


def _call(name: str, device: torch.device, *args) -> None:
    """one entry point on the device's current stream, with that device current"""
    fn = _entry.get(name)
    if fn is None:
        fn = _entry[name] = getattr(_lib.load(), name)
    index = device.index
    if _current_device() == index:
        rc = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(device):
            rc = fn(*args, _raw_stream(index))
    if rc:
        _lib.check(rc, name)


@lru_cache(maxsize=4096)
def _workspace_bytes(name: str, index: int, *sizes: int) -> int:
    """what an entry point needs for these sizes on this device (it depends on nothing else)"""
    with torch.cuda.device(index):
        return getattr(_lib.load(), name)(*sizes)


def _states(t: Tensor) -> Tensor:
    """a tensor whose rows are contiguous and 16-byte aligned; a copy where the given one's are not"""
    if t.is_contiguous() and t.data_ptr() % 16 == 0:  # rows are multiples of 64 elements
        return t
    if t.stride(-1) != 1 or t.data_ptr() % 16 or any(s % 8 for s in _strides(t)):
        t = t.clone(memory_format=torch.contiguous_format)
    return t


def _strides(t: Tensor) -> Tuple[int, ...]:
    """element strides of all but the last dimension, those of dimensions of size one (which mean nothing) as zero"""
    return tuple([s if n > 1 else 0 for s, n in zip(t.stride(), t.shape)])[:-1]


def _own_rows(t: Tensor, dtype: torch.dtype, batch: int, heads: int, least: int, device) -> bool:
    """whether t is ``[batch, heads, at least least]`` of dtype on device with contiguous rows that share no memory"""
    if t.dtype != dtype or t.dim() != 3 or t.device != device:
        return False
    b, h, n = t.shape
    if b != batch or h != heads or n < least:
        return False
    sb, sh, s1 = t.stride()
    return (n <= 1 or s1 == 1) and (heads == 1 or sh >= n) and (batch == 1 or sb >= (heads - 1) * (sh if heads > 1 else 0) + n)


def _no_grad(what: str, *tensors: Optional[Tensor]) -> None:
    if torch.is_grad_enabled() and any([t is not None and t.requires_grad for t in tensors]):
        raise _lib.MaseAmdError(f"{what} is for inference and records no gradient: call it under torch.no_grad() or on detached tensors")


def paged_kv_append(key: Tensor, value: Tensor, k_pages: Tensor, v_pages: Tensor, page_table: Tensor, starts: Tensor, *,
                    counts: Optional[Tensor] = None, positions: Optional[Tensor] = None,
                    first_positions: Optional[Tensor] = None, kv_format: Optional[str] = None,
                    k_scales: Optional[Tensor] = None, v_scales: Optional[Tensor] = None) -> None:
    """Writes ``key``, ``value`` ``[batch, kv_heads, tokens, head_dim]`` into the pages: token j of sequence b to slot
    ``starts[b] + j`` (int32 ``[batch]``), for ``j < counts[b]`` where ``counts`` is given (a padded batch).  MX formats
    quantize blocks of 32 along ``head_dim`` as ``mxint_quantizer(..., 32, 8)`` and the packed MXFP operands of
    ``LinearMXFP`` do.  ``positions`` (int32 ``[batch, kv_heads, capacity]``, rows contiguous): entry slot becomes
    ``first_positions[b] + j`` (default ``starts[b] + j``).  Tokens without a slot in the table are not written."""
    what = "paged_kv_append"
    _no_grad(what, key, value, k_pages, v_pages)
    c = _Pool(what, k_pages, v_pages, page_table, kv_format, k_scales, v_scales, key.dtype)
    device = k_pages.device
    if key.dim() != 4 or value.shape != key.shape or value.dtype != key.dtype or (key.shape[0], key.shape[1], key.shape[3]) != (c.batch, c.kv_heads, c.head_dim):
        raise ValueError(f"{what}: key and value must be [{c.batch}, {c.kv_heads}, tokens, {c.head_dim}] of one type, got "
                         f"{tuple(key.shape)} {key.dtype} and {tuple(value.shape)} {value.dtype}")
    if key.device != device or value.device != device:
        raise ValueError(f"{what}: key and value must be on {device}")
    if key.numel() == 0:
        return
    key, value = _states(key), _states(value)
    sp = _int32(starts, "starts", (c.batch,), device)
    cp = _int32(counts, "counts", (c.batch,), device) if counts is not None else None
    pp = fp = None
    pos_b = pos_h = 0
    if positions is not None:
        # an entry is written for every slot of the table that a token goes to
        least = c.slots
        if not _own_rows(positions, torch.int32, c.batch, c.kv_heads, least, device):
            raise ValueError(f"{what}: positions must be int32 [{c.batch}, {c.kv_heads}, at least {least}] on {device} with contiguous rows")
        pp, pos_b, pos_h = positions.data_ptr(), positions.stride(0), positions.stride(1)
        fp = _int32(first_positions, "first_positions", (c.batch,), device) if first_positions is not None else None
    elif first_positions is not None:
        raise ValueError(f"{what}: first_positions without positions")
    tab = None
    if kv_format is not None:
        tab = log2_table(key.dtype if kv_format == "mxint8" else torch.float32, device).data_ptr()
    _call("mase_paged_kv_append", device, c.record, key.data_ptr(), value.data_ptr(), key.shape[2],
          *_strides(key), *_strides(value), sp, cp, pp, pos_b, pos_h, fp, tab)


def paged_kv_gather(k_pages: Tensor, v_pages: Tensor, page_table: Tensor, lengths: Tensor, max_length: int, *,
                    dtype: Optional[torch.dtype] = None, kv_format: Optional[str] = None, k_scales: Optional[Tensor] = None,
                    v_scales: Optional[Tensor] = None) -> Tuple[Tensor, Tensor]:
    """``(key, value)`` ``[batch, kv_heads, max_length, head_dim]`` of ``dtype`` (of the pages' type with
    ``kv_format=None``): the sequences' slots, zeros from ``lengths[b]`` (int32 ``[batch]``) on."""
    what = "paged_kv_gather"
    _no_grad(what, k_pages, v_pages)
    if dtype is None:
        if kv_format is not None:
            raise ValueError(f"{what}: dtype is needed with kv_format={kv_format!r}")
        dtype = k_pages.dtype
    c = _Pool(what, k_pages, v_pages, page_table, kv_format, k_scales, v_scales, dtype)
    device = k_pages.device
    max_length = int(max_length)
    if max_length < 0:
        raise ValueError(f"{what}: max_length must not be negative, got {max_length}")
    out = torch.empty((2, c.batch, c.kv_heads, max_length, c.head_dim), dtype=dtype, device=device)
    key, value = out[0], out[1]
    if out.numel():
        _call("mase_paged_kv_gather", device, c.record, _int32(lengths, "lengths", (c.batch,), device), max_length,
              key.data_ptr(), value.data_ptr())
    return key, value


def paged_attention_decode(query: Tensor, k_pages: Tensor, v_pages: Tensor, page_table: Tensor, lengths: Tensor,
                           max_length: int, *, scaling: Optional[float] = None, mask: Optional[Tensor] = None,
                           weights: Optional[Tensor] = None, kv_format: Optional[str] = None,
                           k_scales: Optional[Tensor] = None, v_scales: Optional[Tensor] = None) -> Tensor:
    """``softmax(scaling * query key^T + mask) value`` for one token per sequence, ``query`` ``[batch, heads, head_dim]``
    over the ``lengths[b]`` (int32 ``[batch]``, none above ``max_length``) slots of its sequence; query head h reads cached
    head ``h // (heads // kv_heads)``.  Returns ``[batch, heads, head_dim]``.

    ``scaling`` defaults to ``head_dim ** -0.5``.  ``mask``: added to the scores of every head, ``[batch or 1, >= max_length]``
    of ``query``'s type or float32 (also with dimensions of size one in between, as the 4-D masks of the attention modules
    have); a slot masked with -inf is left out whatever it holds.  A row without slots gives zeros; an
    infinite value in a slot that counts gives NaN (sums are formed before the division: bf16 values beyond about 2^120 over
    the number of slots may overflow).  ``weights`` (float32
    ``[batch, kv_heads, >= max_length]``, rows contiguous): grows by the probabilities, summed over the query heads of each
    cached head.  ``max_length`` fixes how the work is split: one value for all calls of a captured step."""
    what = "paged_attention_decode"
    _no_grad(what, query, k_pages, v_pages, mask, weights)
    c = _Pool(what, k_pages, v_pages, page_table, kv_format, k_scales, v_scales, query.dtype)
    device, batch, kv_heads, head_dim = k_pages.device, c.batch, c.kv_heads, c.head_dim
    if query.dim() != 3 or query.shape[0] != batch or query.shape[2] != head_dim or query.shape[1] % kv_heads or query.shape[1] == 0:
        raise ValueError(f"{what}: query must be [{batch}, a multiple of {kv_heads}, {head_dim}], got {tuple(query.shape)}")
    if query.device != device:
        raise ValueError(f"{what}: query must be on {device}")
    heads = query.shape[1]
    if heads // kv_heads > 256:
        raise ValueError(f"{what}: at most 256 query heads for one cached head, got {heads // kv_heads}")
    max_length = int(max_length)
    if max_length < 0 or max_length > c.slots:
        raise ValueError(f"{what}: max_length must be between 0 and the table's {c.slots} slots, got {max_length}")
    if scaling is None:
        scaling = head_dim ** -0.5
    query = _states(query)
    lp = _int32(lengths, "lengths", (batch,), device)
    mp, mcode, m_b = None, 0, 0
    if mask is not None:
        if mask.dim() < 2 or any(n != 1 for n in mask.shape[1:-1]) or mask.shape[0] not in (1, batch) or mask.shape[-1] < max_length:
            raise ValueError(f"{what}: mask must be [batch or 1, (1, ...) at least {max_length}], got {tuple(mask.shape)}")
        if mask.dtype not in (query.dtype, torch.float32) or mask.device != device:
            raise ValueError(f"{what}: mask must be {query.dtype} or float32 on {device}, got {mask.dtype} on {mask.device}")
        if mask.stride(-1) != 1:
            mask = mask.contiguous()
        mp, mcode, m_b = mask.data_ptr(), _lib.DTYPE_CODE[mask.dtype], mask.stride(0) if mask.shape[0] > 1 else 0
    wp, w_b, w_h = None, 0, 0
    if weights is not None:
        if not _own_rows(weights, torch.float32, batch, kv_heads, max_length, device):
            raise ValueError(f"{what}: weights must be float32 [{batch}, {kv_heads}, at least {max_length}] on {device} with contiguous rows")
        wp, w_b, w_h = weights.data_ptr(), weights.stride(0), weights.stride(1)
    out = torch.empty((batch, heads, head_dim), dtype=query.dtype, device=device)
    if batch == 0:
        return out
    n = _workspace_bytes("mase_paged_attention_decode_workspace_bytes", device.index, batch, heads, kv_heads, head_dim, c.format,
                         max_length, int(wp is not None))
    ws = torch.empty(n, dtype=torch.uint8, device=device)
    _call("mase_paged_attention_decode", device, c.record, query.data_ptr(), *_strides(query), heads, lp, max_length,
          float(scaling), mp, mcode, m_b, wp, w_b, w_h, out.data_ptr(), ws.data_ptr(), n)
    return out


def paged_kv_evict(k_pages: Tensor, v_pages: Tensor, page_table: Tensor, lengths: Tensor, weights: Tensor, positions: Tensor,
                   max_length: int, keep: int, *, recent: int = 0, first: int = 0, kv_format: Optional[str] = None,
                   k_scales: Optional[Tensor] = None, v_scales: Optional[Tensor] = None) -> Tuple[Tensor, Tensor, Tensor]:
    """Cuts every sequence longer than ``keep`` slots down to ``keep``, each cached head for itself: kept are the tokens at
    positions below ``first`` or among the last ``recent`` positions, then those of the largest weight, ties going to the
    lowest slot.  Kept slots below ``keep`` stay; the free ones there take the kept tokens behind them, in order: pages
    (and scales) are changed in place, and what lies behind slot ``keep`` can be given back.

    ``weights`` float32 and ``positions`` int32 ``[batch, kv_heads, capacity]``, contiguous, from
    ``paged_attention_decode`` and ``paged_kv_append``.  Returns new ``(weights, positions, lengths)``: what belongs to the
    slots now, zero and -1 behind.  A page must belong to one sequence only."""
    what = "paged_kv_evict"
    _no_grad(what, k_pages, v_pages, weights)
    c = _Pool(what, k_pages, v_pages, page_table, kv_format, k_scales, v_scales,
              k_pages.dtype if kv_format is None else torch.bfloat16)
    device = k_pages.device
    keep, recent, first, max_length = int(keep), int(recent), int(first), int(max_length)
    if keep < 1 or recent < 0 or first < 0 or first + recent > keep:
        raise ValueError(f"{what}: keep must be at least 1 and hold first + recent tokens, got keep={keep}, recent={recent}, first={first}")
    if max_length < 0 or max_length > c.slots:
        raise ValueError(f"{what}: max_length must be between 0 and the table's {c.slots} slots, got {max_length}")
    if keep >= max_length:  # no sequence is longer: nothing moves, and no room for moves is needed
        keep, recent, first = max(max_length, 1), 0, 0
    capacity = weights.shape[-1] if weights.dim() == 3 else 0
    shape = (c.batch, c.kv_heads, capacity)
    if weights.dtype != torch.float32 or weights.shape != shape or capacity < max(max_length, 1) or weights.device != device or not weights.is_contiguous():
        raise ValueError(f"{what}: weights must be a contiguous float32 tensor [{c.batch}, {c.kv_heads}, at least {max_length}] on {device}")
    pp = _int32(positions, "positions", shape, device)
    lp = _int32(lengths, "lengths", (c.batch,), device)
    new_weights, new_positions, new_lengths = torch.empty_like(weights), torch.empty_like(positions), torch.empty_like(lengths)
    if c.batch:
        n = _workspace_bytes("mase_paged_kv_evict_workspace_bytes", device.index, c.batch, c.kv_heads, keep)
        ws = torch.empty(n, dtype=torch.uint8, device=device)
        _call("mase_paged_kv_evict", device, c.record, lp, max_length, weights.data_ptr(), pp, capacity, keep, recent,
              first, new_weights.data_ptr(), new_positions.data_ptr(), new_lengths.data_ptr(), ws.data_ptr(), n)
    return new_weights, new_positions, new_lengths
