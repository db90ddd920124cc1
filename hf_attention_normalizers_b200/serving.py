"""Paged serving: one step of a batch whose sequences bring different numbers
of new tokens, on a paged KV cache that is written and cut in place.

A step calls, for every layer,

* ``paged_append``           the new tokens' K/V rows go into their pages,
* ``paged_chunk_attention``  the new tokens attend over the whole context (a
  prompt piece, a single token, or a mix of them in one batch) and, on request,
  add every key's attention weight to the cache's accumulators,
* ``paged_evict``            when a sequence outgrew its budget: every KV head
  keeps the keys with the most accumulated weight.

Shapes (T new tokens of B sequences packed one after the other):

* new rows ``[T, heads, dim]`` with ``cu_seqlens`` ``[B + 1]``; sequences may
  bring no token;
* caches ``[num_blocks * block_size, kv_heads, dim]``, any strides with a unit
  innermost one (K and V may interleave in one allocation);
* ``block_table`` ``[B, max_blocks]`` and ``sequence_lengths`` ``[B]``: the keys
  of each sequence, its new tokens included, which are its last ones;
* ``key_weights`` float32 ``[kv_heads, num_blocks * block_size]``: one
  accumulator per KV head and cache slot.

Inference only: nothing here has a gradient (``paged.paged_attention`` has).
No call waits for the GPU; lengths, offsets and page ids are checked on the
device, where a bad one is clamped or skipped and recorded in the status word
that ``device_status`` reads.  ``max_seqlen_q`` / ``max_seqlen_k`` are what the host
knows of the longest; without them the packed length and the block table's
capacity are taken, which costs idle thread blocks.  More new tokens than
``max_seqlen_q`` only cost time; keys past ``max_seqlen_k`` are cut off, as a
bad length.
"""

from __future__ import annotations

from dataclasses import dataclass
from typing import Callable, Optional, Sequence, Union

import torch

from . import _native as N
from . import ops
from .paged import _normalizer_name

__all__ = ["PagedServingCache", "paged_append", "paged_chunk_attention", "paged_evict", "device_status"]


_INTS = (torch.int32, torch.int64)


def _check_cache(key_cache, value_cache, block_table, sequence_lengths, block_size, key_weights, name) -> None:
    shape, tables, lens = key_cache.shape, block_table.shape, sequence_lengths.shape
    if len(shape) != 3 or shape != value_cache.shape:
        raise ValueError("key_cache/value_cache must have matching [pages, heads, dim] shapes.")
    if key_cache.dtype is not value_cache.dtype:
        raise ValueError("key_cache and value_cache must have one dtype.")
    if key_cache.stride(2) != 1 or value_cache.stride(2) != 1:
        raise ValueError("key_cache/value_cache must have a unit innermost stride.")
    if not key_cache.is_cuda or not value_cache.is_cuda:
        raise ValueError(f"{name} requires CUDA tensors.")
    if len(tables) != 2:
        raise ValueError("block_table must have shape [batch, max_blocks].")
    if len(lens) != 1 or lens[0] != tables[0]:
        raise ValueError("sequence_lengths must have shape [batch].")
    if tables[0] < 1:
        raise ValueError("The batch must hold at least one sequence.")
    if block_table.dtype not in _INTS or sequence_lengths.dtype not in _INTS:
        raise ValueError("block_table and sequence_lengths must use int32 or int64.")
    if block_size <= 0:
        raise ValueError("block_size must be positive.")
    if key_weights is not None:
        if key_weights.dtype is not torch.float32 or key_weights.shape != (shape[1], shape[0]):
            raise ValueError("key_weights must be float32 [kv_heads, num_blocks * block_size].")
        if key_weights.stride(1) != 1 or key_weights.stride(0) < shape[0]:
            raise ValueError("key_weights must have contiguous rows.")


def _check_rows(rows, key_cache, cu_seqlens, block_table, name) -> None:
    if cu_seqlens.shape != (block_table.shape[0] + 1,):
        raise ValueError(f"{name} must have shape [batch + 1].")
    if cu_seqlens.dtype not in _INTS:
        raise ValueError(f"{name} must use int32 or int64.")
    if rows.dtype is not key_cache.dtype:
        raise ValueError("New tokens and cache must have one dtype.")
    if rows.shape[-1] != key_cache.shape[-1]:
        raise ValueError("New tokens and cache head dimensions must match.")


_compiling, _grad_enabled = torch.compiler.is_compiling, torch.is_grad_enabled
_modes, _functorch = torch._C._len_torch_dispatch_stack, torch._C._functorch.peek_interpreter_stack
_profiling = torch._C._autograd._profiler_enabled
_Tensor, _Parameter = torch.Tensor, torch.nn.Parameter


def _check_placement(*tensors) -> bool:
    """Returns whether somebody listens for the call: it is then dispatched as a custom op, else launched directly
    (the dispatch costs as much host time as the launch)."""
    where = tensors[0].get_device()
    observed = _compiling() or _modes() > 0 or _functorch() is not None or _profiling()
    grad = _grad_enabled()
    for t in tensors:
        if t is None:
            continue
        if t.get_device() != where:
            raise ValueError("All tensors must be on one device.")
        if grad and t.requires_grad:
            raise ValueError("Paged serving is inference only: call it under torch.no_grad() or detach its inputs.")
        kind = type(t)
        if kind is not _Tensor and kind is not _Parameter:
            observed = True
    return observed


def _bound(given: Optional[int], most: int, name: str) -> int:
    if given is None:
        return most
    if given < 0:
        raise ValueError(f"{name} must not be negative.")
    return min(int(given), most)


def paged_append(key: torch.Tensor, value: torch.Tensor, key_cache: torch.Tensor, value_cache: torch.Tensor,
                 block_table: torch.Tensor, cu_seqlens: torch.Tensor, sequence_lengths: torch.Tensor, block_size: int,
                 key_weights: Optional[torch.Tensor] = None) -> None:
    """Write the new tokens' ``[T, kv_heads, dim]`` K/V rows into the pages, in place.

    Row ``i`` of the ``n`` new tokens of a sequence goes to its position
    ``length - n + i``; the written slots of ``key_weights`` start at zero.
    """
    _check_cache(key_cache, value_cache, block_table, sequence_lengths, block_size, key_weights, "paged_append")
    if key.ndim != 3 or key.shape != value.shape:
        raise ValueError("key/value must have matching [total_tokens, kv_heads, dim] shapes.")
    if value.dtype != key.dtype:
        raise ValueError("key and value must have one dtype.")
    if key.shape[1] != key_cache.shape[1]:
        raise ValueError("New keys and cache must have the same KV heads.")
    _check_rows(key, key_cache, cu_seqlens, block_table, "cu_seqlens")
    observed = _check_placement(key_cache, value_cache, key, value, block_table, cu_seqlens, sequence_lengths, key_weights)
    call = ops.paged_append if observed else ops.launch_paged_append
    call(key, value, key_cache, value_cache, block_table, cu_seqlens, sequence_lengths, int(block_size), key.shape[0],
         key_weights)


def paged_chunk_attention(query: torch.Tensor, key_cache: torch.Tensor, value_cache: torch.Tensor,
                          block_table: torch.Tensor, cu_seqlens_q: torch.Tensor, sequence_lengths: torch.Tensor,
                          block_size: int, normalizer: Union[str, Callable[..., torch.Tensor]] = "softmax1",
                          scale: Optional[float] = None, is_causal: bool = True,
                          key_weights: Optional[torch.Tensor] = None, max_seqlen_q: Optional[int] = None,
                          max_seqlen_k: Optional[int] = None) -> torch.Tensor:
    """Attention of a ragged chunk of new tokens ``[T, q_heads, dim]`` over the cached context.

    The causal mask is aligned to each sequence's end (its new tokens are its
    last keys); rows that see no key give zeros, and so do the packed rows that
    no sequence owns (padding before the first offset or past the last).  Cache
    slots past a sequence's length are never used, whatever they hold; a value
    row inside it that is not finite may reach rows of the call that the mask
    hides it from (0 x inf).  With ``key_weights`` the probabilities of every
    key, summed over the new tokens and the query heads of its KV head, are
    added to its accumulator.
    """
    _check_cache(key_cache, value_cache, block_table, sequence_lengths, block_size, key_weights,
                 "paged_chunk_attention")
    if query.ndim != 3:
        raise ValueError("query must have shape [total_tokens, heads, dim].")
    if query.shape[1] % key_cache.shape[1] != 0:
        raise ValueError("query heads must be divisible by KV heads.")
    _check_rows(query, key_cache, cu_seqlens_q, block_table, "cu_seqlens_q")
    observed = _check_placement(key_cache, value_cache, query, block_table, cu_seqlens_q, sequence_lengths, key_weights)
    norm = N.NORMALIZER_IDS.get(normalizer) if isinstance(normalizer, str) else None
    if norm is None:
        norm = N.NORMALIZER_IDS[_normalizer_name(normalizer)]
    max_q = _bound(max_seqlen_q, query.shape[0], "max_seqlen_q")
    max_k = _bound(max_seqlen_k, block_table.shape[1] * block_size, "max_seqlen_k")
    actual_scale = query.shape[-1] ** -0.5 if scale is None else float(scale)
    call = ops.paged_chunk_fwd if observed else ops.launch_paged_chunk_fwd
    return call(query, key_cache, value_cache, block_table, cu_seqlens_q, sequence_lengths, int(block_size), max_q, max_k,
                norm, actual_scale, bool(is_causal), key_weights)[0]


def paged_evict(key_cache: torch.Tensor, value_cache: torch.Tensor, key_weights: torch.Tensor,
                block_table: torch.Tensor, sequence_lengths: torch.Tensor, block_size: int, budget: int,
                recent: int = 0, max_seqlen_k: Optional[int] = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Cut every sequence longer than ``budget`` to ``budget`` keys, per KV head and in place.

    The ``recent`` last positions stay, the other places go to the largest
    ``key_weights`` (ties to the lowest position).  What is kept moves, in
    order, to the sequence's positions ``0 .. budget - 1``, so its pages past
    ``ceil(budget / block_size)`` are free; slots past the budget keep what they
    held.  The pages of a longer sequence must not be shared with another one.

    Returns the new lengths ``int32 [B]`` and the former positions of what is
    kept, ``int32 [B, kv_heads, budget]`` (-1 past a shorter sequence).
    """
    if key_weights is None:
        raise ValueError("paged_evict requires key_weights.")
    _check_cache(key_cache, value_cache, block_table, sequence_lengths, block_size, key_weights, "paged_evict")
    if budget < 1:
        raise ValueError("budget must be positive.")
    if recent < 0:
        raise ValueError("recent must not be negative.")
    observed = _check_placement(key_cache, value_cache, block_table, sequence_lengths, key_weights)
    max_k = _bound(max_seqlen_k, block_table.shape[1] * block_size, "max_seqlen_k")
    call = ops.paged_evict if observed else ops.launch_paged_evict
    return call(key_cache, value_cache, key_weights, block_table, sequence_lengths, int(block_size), max_k, int(budget),
                int(recent))


def device_status(clear: bool = True) -> int:
    """Wait for the current stream and read the device status word: 0, or the first error the kernels
    recorded (1: page id outside the cache, 2: a bounded wait ran out, 3: length or offset out of range)."""
    return N.device_status(torch.cuda.current_stream().cuda_stream, clear)


@dataclass
class ServingStep:
    """One step of a batch, as ``PagedServingCache.step`` laid it out (device tensors and their host bounds)."""

    block_table: torch.Tensor
    cu_seqlens: torch.Tensor
    lengths: torch.Tensor
    max_seqlen_q: int
    max_seqlen_k: int


class PagedServingCache:
    """The pages of a batch over all layers, with their bookkeeping on the host.

    ``step`` gives every sequence room for its new tokens; ``append`` and
    ``attend`` are called once per layer of that step; ``evict`` cuts every
    sequence to a budget and returns the freed pages; ``release`` ends one.
    Lengths follow from what the host has asked for, so no call waits for the
    GPU.  ``lengths`` count cached keys: after an eviction a text's positions
    (of its rotary embedding, say) run ahead of them, and the caller keeps them.
    """

    def __init__(self, num_layers: int, num_sequences: int, num_blocks: int, block_size: int, kv_heads: int, head_dim: int,
                 dtype: torch.dtype = torch.bfloat16, device: Union[str, torch.device] = "cuda", track_weights: bool = False):
        slots = num_blocks * block_size
        # K and V of a slot side by side: one allocation a layer
        self.layers = [torch.zeros(slots, 2, kv_heads, head_dim, dtype=dtype, device=device) for _ in range(num_layers)]
        self.weights = [torch.zeros(kv_heads, slots, device=device) if track_weights else None for _ in range(num_layers)]
        self.block_size = block_size
        self.lengths = [0] * num_sequences
        self._pages: list[list[int]] = [[] for _ in range(num_sequences)]
        self._free = list(range(num_blocks - 1, -1, -1))
        self._device = self.layers[0].device if self.layers else torch.device(device)

    def step(self, new_tokens: Sequence[int]) -> ServingStep:
        """Allocate pages for ``new_tokens[b]`` more tokens of every sequence (0: the sequence rests)."""
        if len(new_tokens) != len(self.lengths):
            raise ValueError("new_tokens must have one count per sequence.")
        if any(n < 0 for n in new_tokens):
            raise ValueError("new_tokens must not be negative.")
        need = [-(-(c + n) // self.block_size) - len(p) for c, n, p in zip(self.lengths, new_tokens, self._pages)]
        if sum(max(n, 0) for n in need) > len(self._free):
            raise ValueError("The cache has no room for the new tokens.")
        for b, n in enumerate(need):
            self._pages[b].extend(self._free.pop() for _ in range(n))
            self.lengths[b] += new_tokens[b]
        return self._describe(new_tokens)

    def release(self, sequence: int) -> None:
        """End a sequence: its pages are free, and its place takes a new text with the next step."""
        if not 0 <= sequence < len(self.lengths):
            raise ValueError(f"The cache has no sequence {sequence}.")
        self._free.extend(reversed(self._pages[sequence]))
        self._pages[sequence] = []
        self.lengths[sequence] = 0

    def _describe(self, new_tokens: Sequence[int]) -> ServingStep:
        width = max(1, max(len(p) for p in self._pages))
        offsets = [0]
        for n in new_tokens:
            offsets.append(offsets[-1] + n)
        host = offsets + self.lengths
        for p in self._pages:
            host = host + p + [0] * (width - len(p))
        flat = torch.tensor(host, dtype=torch.int32)
        if self._device.type == "cuda":
            flat = flat.pin_memory().to(self._device, non_blocking=True)
        b = len(self.lengths)
        return ServingStep(flat[2 * b + 1:].view(b, width), flat[:b + 1], flat[b + 1:2 * b + 1], max(new_tokens),
                           max(self.lengths))

    def append(self, layer: int, step: ServingStep, key: torch.Tensor, value: torch.Tensor) -> None:
        kv = self.layers[layer]
        paged_append(key, value, kv[:, 0], kv[:, 1], step.block_table, step.cu_seqlens, step.lengths, self.block_size,
                     key_weights=self.weights[layer])

    def attend(self, layer: int, step: ServingStep, query: torch.Tensor,
               normalizer: Union[str, Callable[..., torch.Tensor]] = "softmax1", scale: Optional[float] = None) -> torch.Tensor:
        kv = self.layers[layer]
        return paged_chunk_attention(query, kv[:, 0], kv[:, 1], step.block_table, step.cu_seqlens, step.lengths,
                                     self.block_size, normalizer, scale, key_weights=self.weights[layer],
                                     max_seqlen_q=step.max_seqlen_q, max_seqlen_k=step.max_seqlen_k)

    def evict(self, budget: int, recent: int = 0) -> None:
        """Cut every sequence longer than ``budget`` in all layers and free the pages that this empties."""
        if any(w is None for w in self.weights):
            raise ValueError("evict needs a cache made with track_weights=True.")
        if max(self.lengths) <= budget:
            return
        step = self._describe([0] * len(self.lengths))
        for kv, w in zip(self.layers, self.weights):
            paged_evict(kv[:, 0], kv[:, 1], w, step.block_table, step.lengths, self.block_size, budget, recent=recent,
                        max_seqlen_k=step.max_seqlen_k)
        for b, c in enumerate(self.lengths):
            self.lengths[b] = min(c, budget)
            keep = -(-self.lengths[b] // self.block_size)
            self._free.extend(reversed(self._pages[b][keep:]))
            del self._pages[b][keep:]
