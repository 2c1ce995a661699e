"""``PagedKVCache``: the keys and values of a batch of sequences in pages, as 16-bit states or as MX codes.

It takes the place of the cache object that the attention modules call ``past_key_value.update`` on
(``chop/nn/quantized/modules/llama/attention.py:182-187``): ``update`` appends and returns the dense states, ``append`` and
``attend`` do a decoding step on the pages alone, and ``evict`` cuts the sequences down to a budget by the attention
weights that the steps have added up.  The functions underneath are in ``mase_amd.quantized.functional``.

The host keeps how long each sequence is, so no call waits for the GPU; a replayed graph would not move that on, so no
call can be captured: a step that is captured uses the functions directly, with lengths that the graph itself moves on.
"""
from __future__ import annotations

from typing import List, Optional, Sequence, Tuple

import torch
from torch import Tensor

from .. import _lib
from .functional import paged_kv as F

_capturing = torch._C._cuda_isCurrentStreamCapturing

# (kind, element bits or exponent and fraction bits) of the kv_cache quantizer that each code format holds the values of
_FORMAT_OF = {("mxint", 8): "mxint8", ("mxfp", 4, 3): "mxfp8_e4m3", ("mxfp", 5, 2): "mxfp8_e5m2", ("mxfp", 2, 1): "mxfp4"}


class PagedKVCache:
    """``batch_size`` sequences of at most ``max_length`` tokens at a time, ``num_layers`` layers that share one page table.

    ``kv_format``: None (states of ``dtype``), ``"mxint8"``, ``"mxfp8_e4m3"``, ``"mxfp8_e5m2"`` or ``"mxfp4"`` (blocks of 32
    along the head dimension).  ``num_pages`` (default: enough for every sequence at ``max_length``) is the pool's size for
    each layer; a sequence takes pages as it grows.  ``track_weights``: positions and the sums of the attention weights are
    kept, which ``evict`` needs; ``attend`` adds to them, and so do the attention modules' dense steps (``add_weights``)."""

    _most_sequences = 65535  # of one call of paged_attention_decode

    def __init__(self, batch_size: int, num_kv_heads: int, head_dim: int, max_length: int, num_layers: int = 1, *,
                 page_size: int = 64, num_pages: Optional[int] = None, kv_format: Optional[str] = None,
                 dtype: torch.dtype = torch.bfloat16, device="cuda", track_weights: bool = False):
        if kv_format not in F.KV_FORMATS:
            raise ValueError(f"kv_format must be one of {F.KV_FORMATS}, got {kv_format!r}")
        if min(batch_size, num_kv_heads, max_length, num_layers) < 1:
            raise ValueError("batch_size, num_kv_heads, max_length and num_layers must be at least 1")
        if head_dim not in (64, 128, 256) or page_size not in (16 << n for n in range(9)):
            raise ValueError(f"head_dim must be 64, 128 or 256 and page_size a power of two from 16 to 4096, got {head_dim} and {page_size}")
        if dtype not in (torch.bfloat16, torch.float16):
            raise ValueError(f"dtype must be bfloat16 or float16, got {dtype}")
        self.batch_size, self.num_kv_heads, self.head_dim, self.max_length = batch_size, num_kv_heads, head_dim, max_length
        self.num_layers, self.page_size, self.kv_format, self.dtype = num_layers, page_size, kv_format, dtype
        self.device = torch.device(device)
        table_pages = -(-max_length // page_size)
        self.num_pages = batch_size * table_pages if num_pages is None else int(num_pages)
        if self.num_pages < 1:
            raise ValueError("num_pages must be at least 1")
        shape = (num_layers, self.num_pages, num_kv_heads, page_size)
        if kv_format is None:
            self._k, self._v = (torch.zeros((*shape, head_dim), dtype=dtype, device=self.device) for _ in range(2))
            self._ks = self._vs = None
        else:
            width = head_dim // 2 if kv_format == "mxfp4" else head_dim
            code = torch.int8 if kv_format == "mxint8" else torch.uint8
            self._k, self._v = (torch.zeros((*shape, width), dtype=code, device=self.device) for _ in range(2))
            self._ks = torch.zeros((*shape, head_dim // 32), dtype=torch.uint8, device=self.device)
            self._vs = torch.zeros((*shape[:3], head_dim // 32, page_size), dtype=torch.uint8, device=self.device)
        self._table = torch.full((batch_size, table_pages), -1, dtype=torch.int32, device=self.device)
        self.device = self._table.device  # with its index, whichever device is current later
        self._on_gpu = self._table.is_cuda
        self._free = list(range(self.num_pages - 1, -1, -1))
        self._pages: List[List[int]] = [[] for _ in range(batch_size)]
        # per layer: slots held and tokens seen, on the host and on the device
        self._held = [[0] * batch_size for _ in range(num_layers)]
        self._seen = [[0] * batch_size for _ in range(num_layers)]
        self._held_dev, self._seen_dev = (torch.zeros((num_layers, batch_size), dtype=torch.int32, device=self.device) for _ in range(2))
        self.track_weights = track_weights
        self._weights = self._positions = None
        if track_weights:
            rows = (num_layers, batch_size, num_kv_heads, table_pages * page_size)
            self._weights = torch.zeros(rows, dtype=torch.float32, device=self.device)
            self._positions = torch.full(rows, -1, dtype=torch.int32, device=self.device)

    # -- what it holds ------------------------------------------------------------------------------------------------
    def get_seq_length(self, layer_idx: int = 0) -> int:
        """tokens that the longest sequence has seen: the position of the next one"""
        return max(self._seen[layer_idx])

    def lengths(self, layer_idx: int = 0) -> List[int]:
        """slots that each sequence holds (fewer than it has seen after an eviction)"""
        return list(self._held[layer_idx])

    def positions(self, layer_idx: int = 0) -> Tensor:
        """int32 ``[batch, kv_heads, capacity]``: where the token of each slot stood, -1 for free slots"""
        self._require_tracking("positions")
        return self._positions[layer_idx]

    def weights(self, layer_idx: int = 0) -> Tensor:
        """float32 ``[batch, kv_heads, capacity]``: attention weights added up by ``attend``"""
        self._require_tracking("weights")
        return self._weights[layer_idx]

    def require_kind(self, kind: Optional[str], config: dict) -> None:
        """raises ValueError unless states quantized by the module's ``kv_cache`` configuration (``kind`` None: not
        quantized) are what this cache holds: codes hold the values of one quantizer only, 16-bit pages those of any"""
        if self.kv_format is None:
            return
        if kind is None:
            raise ValueError(f"a PagedKVCache of {self.kv_format} codes quantizes what it holds, but the module's kv_cache quantizer is bypassed: use kv_format=None")
        bits = (config["data_in_width"],) if kind == "mxint" else (config["data_in_exponent_width"], config["data_in_frac_width"])
        if config["data_in_block_size"] != 32 or _FORMAT_OF.get((kind, *bits)) != self.kv_format:
            raise ValueError(f"a PagedKVCache of {self.kv_format} codes does not hold the values of the module's kv_cache quantizer ({kind}, {config}): use kv_format=None")

    # -- masks --------------------------------------------------------------------------------------------------------
    # A mask of a step has one column for each position, as the callers of the attention modules make it.  Until a layer is
    # evicted from, slots are positions; afterwards every cached head has an order of slots of its own.
    def _evicted(self, layer: int) -> bool:
        return self._held[layer] != self._seen[layer]

    def require_mask(self, mask: Optional[Tensor], tokens: int, layer_idx: int = 0, heads: Optional[int] = None) -> None:
        """raises ValueError unless ``mask`` (``[batch or 1, heads or 1, tokens or 1, columns]``, added to the scores of the
        next ``tokens`` tokens, one column for each position) can be laid over the layer's slots once they are appended;
        ``heads``: of the queries"""
        evicted, seen = self._evicted(layer_idx), self._seen[layer_idx]
        if mask is not None and min(seen) != max(seen):
            raise ValueError("a mask with one column for each position needs sequences that stand at the same one: these have seen "
                             f"{min(seen)} to {max(seen)} tokens (steps without a mask and attend() with one take such sequences)")
        if mask is None or not (evicted or tokens == 1):  # the dense chain's own business
            return
        total = self.get_seq_length(layer_idx) + tokens
        fits = mask.dim() == 4 and mask.shape[0] in (1, self.batch_size) and mask.shape[3] >= total
        if fits and evicted:
            each = mask.shape[1] % self.num_kv_heads == 0 if heads is None else mask.shape[1] == heads
            fits = mask.is_floating_point() and mask.shape[2] in (1, tokens) and (mask.shape[1] == 1 or each)
        if not fits:
            raise ValueError(f"mask must be a floating-point tensor [{self.batch_size} or 1, heads or 1, {tokens} or 1, at least {total}] with "
                             f"one column for each position, got {mask.dtype} {tuple(mask.shape)}")

    def slot_mask(self, mask: Optional[Tensor], heads: int, layer_idx: int = 0) -> Optional[Tensor]:
        """the mask over the rows that ``gather`` returns, of one whose columns are positions: the same one until the layer
        is evicted from, then ``[batch, heads, rows, longest]``.  The zeros behind shorter sequences are hidden by the type's
        lowest value (without a mask: by one of the states' type, ``[batch, 1, 1, longest]``)"""
        held, seen = self._held[layer_idx], self._seen[layer_idx]
        if mask is not None and held != seen:
            # the position of every slot has to be a column
            if mask.dim() != 4 or not mask.is_floating_point() or mask.shape[0] not in (1, self.batch_size) or mask.shape[1] not in (1, heads) or mask.shape[3] < max(seen):
                raise ValueError(f"mask must be a floating-point tensor [{self.batch_size} or 1, {heads} or 1, rows, at least {max(seen)}], got {mask.dtype} {tuple(mask.shape)}")
            mask = self._gather_columns(mask, heads, layer_idx)
        if min(held) == max(held):
            return mask
        if mask is None:
            mask = torch.zeros((self.batch_size, 1, 1, max(held)), dtype=self.dtype, device=self.device)
        behind = torch.arange(max(held), device=self.device) >= self._held_dev[layer_idx][:, None]
        return mask[..., :max(held)].masked_fill(behind[:, None, None], torch.finfo(mask.dtype).min)

    def _gather_columns(self, mask: Tensor, heads: int, layer_idx: int) -> Tensor:
        batch, rows, columns = self.batch_size, mask.shape[2], mask.shape[3]
        # the query heads of a cached head see the same slots: one row of columns for all of them where the mask has one
        group = heads // self.num_kv_heads if mask.shape[1] > 1 else 1
        at = self._slot_positions(layer_idx)[:, :, None, None]
        by_head = mask.expand(batch, group * self.num_kv_heads, rows, columns).unflatten(1, (self.num_kv_heads, group))
        got = by_head.gather(-1, at.expand(-1, -1, group, rows, -1))
        return got.expand(-1, -1, heads // self.num_kv_heads, -1, -1).flatten(1, 2)

    def _slot_positions(self, layer: int) -> Tensor:
        """int64 ``[batch, kv_heads, longest]``; 0 for slots behind a sequence's last one, which no kernel looks at"""
        return self._positions[layer][:, :, :max(self._held[layer])].clamp(min=0).long()

    # -- a step -------------------------------------------------------------------------------------------------------
    def append(self, key_states: Tensor, value_states: Tensor, layer_idx: int = 0, counts: Optional[Sequence[int]] = None) -> None:
        """adds ``[batch, kv_heads, tokens, head_dim]`` states behind what the layer holds; ``counts[b]`` of the tokens for
        sequence b where given (a padded batch)"""
        if key_states.dim() != 4 or key_states.shape[0] != self.batch_size or key_states.dtype != self.dtype:
            raise ValueError(f"states must be {self.dtype} [{self.batch_size}, {self.num_kv_heads}, tokens, {self.head_dim}], got {key_states.dtype} {tuple(key_states.shape)}")
        self._refuse_capture("append")
        n = key_states.shape[2]
        new = [n] * self.batch_size if counts is None else [int(c) for c in counts]
        if len(new) != self.batch_size or any(c < 0 or c > n for c in new):
            raise ValueError(f"counts must be {self.batch_size} numbers from 0 to {n}, got {new}")
        held, seen = self._held[layer_idx], self._seen[layer_idx]
        taken = self._grow([h + c for h, c in zip(held, new)])
        try:
            self._write(key_states, value_states, layer_idx, n, None if counts is None else new)
        except Exception:
            self._give_back([len(p) - k for p, k in zip(self._pages, taken)])  # a call that is refused takes no pages
            raise
        for b, c in enumerate(new):
            held[b] += c
            seen[b] += c

    def _write(self, key_states: Tensor, value_states: Tensor, layer_idx: int, n: int, new: Optional[List[int]]) -> None:
        """the states into their pages, and the lengths on the device moved on"""
        counts_dev = None if new is None else self._staged(new).to(torch.int32)
        track = dict(positions=self._positions[layer_idx], first_positions=self._seen_dev[layer_idx]) if self.track_weights else {}
        F.paged_kv_append(key_states, value_states, *self._pool(layer_idx), self._held_dev[layer_idx], counts=counts_dev, **track,
                          **self._codes(layer_idx))
        step = n if counts_dev is None else counts_dev
        self._held_dev[layer_idx] += step
        self._seen_dev[layer_idx] += step

    def update(self, key_states: Tensor, value_states: Tensor, layer_idx: int = 0, cache_kwargs=None) -> Tuple[Tensor, Tensor]:
        """appends, and returns all that the layer holds as ``[batch, kv_heads, longest, head_dim]``, zeros behind shorter
        sequences"""
        self.append(key_states, value_states, layer_idx)
        return self.gather(layer_idx)

    def gather(self, layer_idx: int = 0) -> Tuple[Tensor, Tensor]:
        self._refuse_capture("gather")
        return F.paged_kv_gather(*self._pool(layer_idx), self._held_dev[layer_idx], max(self._held[layer_idx]), dtype=self.dtype,
                                 **self._codes(layer_idx))

    def attend(self, query: Tensor, layer_idx: int = 0, *, scaling: Optional[float] = None, mask: Optional[Tensor] = None) -> Tensor:
        """attention of one token per sequence, ``[batch, heads, head_dim]``, over what the layer holds.  ``mask``
        (``[batch or 1, (1, ...) columns]`` of the states' type or float32): column c is added to the scores of the token at
        position c of its sequence, wherever an eviction has put it"""
        self._refuse_capture("attend")
        if mask is not None and self._evicted(layer_idx):
            return self._attend_by_position(query, layer_idx, scaling, mask)
        return F.paged_attention_decode(query, *self._pool(layer_idx), self._held_dev[layer_idx], max(self._held[layer_idx]),
                                        scaling=scaling, mask=mask, weights=self._weights[layer_idx] if self.track_weights else None,
                                        **self._codes(layer_idx))

    def add_weights(self, probabilities: Tensor, layer_idx: int = 0, mask: Optional[Tensor] = None) -> None:
        """adds the attention probabilities ``[batch, heads, tokens, longest]`` of a step that was computed on what ``update``
        returned to the weights that ``evict`` ranks by, summed over tokens and the query heads of each cached head (``attend``
        does so itself).  ``mask``: the one of that step; tokens whose row of it hides every slot are padding and do not count"""
        self._require_tracking("add_weights")
        self._refuse_capture("add_weights")
        longest = max(self._held[layer_idx])
        shape = tuple(probabilities.shape)
        if len(shape) != 4 or shape[0] != self.batch_size or shape[1] % self.num_kv_heads or shape[1] == 0 or shape[3] != longest:
            raise ValueError(f"probabilities must be [{self.batch_size}, a multiple of {self.num_kv_heads}, tokens, {longest}], got {shape}")
        p = probabilities.detach()
        if mask is not None and mask.is_floating_point() and shape[2] > 1:
            # half the lowest value: masks are also made by adding two of them up
            padding = mask[..., :longest].amax(-1, keepdim=True) <= torch.finfo(mask.dtype).min / 2
            p = p.masked_fill(padding, 0.0)
        by_head = p.unflatten(1, (self.num_kv_heads, -1))
        self._weights[layer_idx][:, :, :longest] += by_head.sum((2, 3), dtype=torch.float32)

    def _attend_by_position(self, query: Tensor, layer: int, scaling: Optional[float], mask: Tensor) -> Tensor:
        """``attend`` with a mask after an eviction: each cached head of a sequence has its own order of slots, so it becomes
        a sequence of one head, with its own mask row, in a pool whose pages are the heads of the pages"""
        batch, heads, columns = self.batch_size, self.num_kv_heads, max(self._seen[layer])
        if (mask.dim() < 2 or mask.shape[0] not in (1, batch) or any(n != 1 for n in mask.shape[1:-1]) or mask.shape[-1] < columns
                or mask.dtype not in (self.dtype, torch.float32)):
            raise ValueError(f"mask must be {self.dtype} or float32 [{batch} or 1, (1, ...) at least {columns}] with one column for each "
                             f"position, got {mask.dtype} {tuple(mask.shape)}")
        if query.dim() != 3 or query.shape[0] != batch or query.shape[1] % heads or query.shape[1] == 0:
            raise ValueError(f"query must be [{batch}, a multiple of {heads}, {self.head_dim}], got {tuple(query.shape)}")
        flat = mask.reshape(mask.shape[0], 1, mask.shape[-1]).expand(batch, heads, -1)
        rows = flat.gather(-1, self._slot_positions(layer))
        single = lambda t: t.flatten(0, 1).unsqueeze(1)  # noqa: E731  [pages, heads, ...] as [pages * heads, 1, ...]
        head = torch.arange(heads, dtype=torch.int32, device=self.device)[:, None]
        table = torch.where(self._table[:, None] < 0, -1, self._table[:, None] * heads + head)
        lengths = self._held_dev[layer].repeat_interleave(heads).view(batch, heads)
        k, v, codes = single(self._k[layer]), single(self._v[layer]), self._codes(layer)
        if codes:
            codes.update(k_scales=single(codes["k_scales"]), v_scales=single(codes["v_scales"]))
        query = query.unflatten(1, (heads, -1))
        parts = []
        each = max(1, self._most_sequences // heads)
        for lo in range(0, batch, each):
            some = slice(lo, lo + each)
            got = F.paged_attention_decode(query[some].flatten(0, 1), k, v, table[some].flatten(0, 1), lengths[some].flatten(),
                                           max(self._held[layer]), scaling=scaling, mask=rows[some].flatten(0, 1),
                                           weights=single(self._weights[layer][some]), **codes)
            parts.append(got.view(-1, query.shape[1] * query.shape[2], self.head_dim))
        return parts[0] if len(parts) == 1 else torch.cat(parts)

    # -- room ---------------------------------------------------------------------------------------------------------
    def evict(self, keep: int, *, recent: int = 0, first: int = 0) -> None:
        """cuts every sequence down to ``keep`` tokens in every layer and cached head (see ``paged_kv_evict``) and gives the
        pages behind them back; between steps, when all layers hold the same tokens"""
        self._require_tracking("evict")
        self._refuse_capture("evict")
        if any(h != self._held[0] for h in self._held):
            raise ValueError("evict() comes between steps: the layers do not hold the same number of tokens")
        if keep < 1 or recent < 0 or first < 0 or first + recent > keep:
            raise ValueError(f"keep must be at least 1 and hold first + recent tokens, got keep={keep}, recent={recent}, first={first}")
        longest = max(self._held[0])
        if longest <= keep:
            return
        for layer in range(self.num_layers):
            w, pos, n = F.paged_kv_evict(*self._pool(layer), self._held_dev[layer], self._weights[layer], self._positions[layer],
                                         longest, keep, recent=recent, first=first, **self._codes(layer))
            self._weights[layer].copy_(w)
            self._positions[layer].copy_(pos)
            self._held_dev[layer].copy_(n)
            self._held[layer] = [min(h, keep) for h in self._held[layer]]
        self._give_back([-(-h // self.page_size) for h in self._held[0]])

    def reset(self) -> None:
        """forgets every sequence"""
        self._refuse_capture("reset")
        self._free = list(range(self.num_pages - 1, -1, -1))
        self._pages = [[] for _ in range(self.batch_size)]
        self._held, self._seen = ([[0] * self.batch_size for _ in range(self.num_layers)] for _ in range(2))
        for t in (self._held_dev, self._seen_dev) + ((self._weights,) if self.track_weights else ()):
            t.zero_()
        self._table.fill_(-1)
        if self.track_weights:
            self._positions.fill_(-1)

    # -- inside -------------------------------------------------------------------------------------------------------
    def _require_tracking(self, what: str) -> None:
        if not self.track_weights:
            raise ValueError(f"{what} needs a cache made with track_weights=True")

    def _refuse_capture(self, what: str) -> None:
        if self._on_gpu and _capturing():
            raise _lib.MaseAmdError(f"PagedKVCache.{what} cannot be captured into a graph, which would not move the lengths on the host: "
                                    "capture the functions of mase_amd.quantized.functional instead")

    def _pool(self, layer: int):
        return self._k[layer], self._v[layer], self._table

    def _codes(self, layer: int) -> dict:
        if self.kv_format is None:
            return {}
        return dict(kv_format=self.kv_format, k_scales=self._ks[layer], v_scales=self._vs[layer])

    def _grow(self, lengths: Sequence[int]) -> List[int]:
        """pages for sequences of these lengths; how many each of them took"""
        if max(lengths) > self.max_length:
            raise ValueError(f"a sequence of {max(lengths)} tokens does not fit a cache of max_length {self.max_length}")
        need = [max(0, -(-n // self.page_size) - len(p)) for n, p in zip(lengths, self._pages)]
        if sum(need) > len(self._free):
            raise ValueError(f"the pool has {len(self._free)} free pages, {sum(need)} are needed")
        at, got = [], []
        for b, k in enumerate(need):
            for _ in range(k):
                at.append((b, len(self._pages[b])))
                got.append(self._free.pop())
                self._pages[b].append(got[-1])
        self._set_table(at, got)
        return need

    def _give_back(self, left: Sequence[int]) -> None:
        """the pages of each sequence behind its first left[b]"""
        dropped = []
        for b in range(self.batch_size - 1, -1, -1):  # the last one taken first
            pages, n = self._pages[b], left[b]
            dropped += [(b, i) for i in range(n, len(pages))]
            self._free += reversed(pages[n:])
            del pages[n:]
        self._set_table(dropped, [-1] * len(dropped))

    def _set_table(self, at, pages) -> None:
        if at:
            rows, cols, numbers = self._staged([(b, i, page) for (b, i), page in zip(at, pages)]).unbind(1)
            self._table[rows, cols] = numbers.to(torch.int32)

    def _staged(self, values) -> Tensor:
        """int64 numbers of the host on the device, in the order of the stream: a copy from pageable memory would wait for the
        GPU.  torch's allocator of pinned memory does not hand a block out again before the copies from it are done"""
        host = torch.tensor(values, dtype=torch.int64, pin_memory=self._on_gpu)
        return host.to(self.device, non_blocking=True)
