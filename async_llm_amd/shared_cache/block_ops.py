"""Block merge and append: ``left + right`` as one block whose keys all live in
the left block's position frame.

Mirror of the KV side of the reference session (``python/minisgl/shared_cache/
session.py:330-528``: ``merge_blocks``, ``append_block``, ``_finish_block_merge``,
``_copy_block``, ``_copy_slots``, ``_shift_keys_``) with the same names, argument
meaning and block bookkeeping.  The reference copies K and V layer by layer with
``index_select`` / ``index_copy_`` and then gathers, rotates and scatters the
copied keys once more; here each half of the merge is ONE launch of
``va_copy_shift_kv`` over all layers, which rotates the keys on their way from
the source slots to the destination slots (fp32 rotation, one rounding, as the
reference).

Recurrent (Gated-DeltaNet) block state is not part of the attention path: its
dictionaries are merged with the reference's rules, and composing two affine
summaries is left to the ``compose_affines`` callable of the model that owns
them.
"""

from __future__ import annotations

from typing import Callable, Dict, Optional, Sequence, Tuple

import numpy as np
import torch

from .. import native
from ..kvcache.mha_pool import layer_runs
from ..kvcache.quantized_pool import QuantizedKVCache
from .eviction import CacheEviction
from .shared_block import CacheBlock


def token_slots(block: CacheBlock) -> np.ndarray:
    """Pool slot of every token of ``block`` (host, int64)."""
    if not block.num_tokens:
        return np.empty(0, dtype=np.int64)
    starts = np.asarray(block.page_starts, dtype=np.int64)
    grid = starts[:, None] + np.arange(block.page_size, dtype=np.int64)[None, :]
    return grid.reshape(-1)[: block.num_tokens]


def slots_meet(a: np.ndarray, b: np.ndarray) -> bool:
    """Whether two non-empty slot lists share a slot.  Slots of one pool lie in a range not much larger than
    the pool, where marking ``a``'s and looking ``b``'s up takes 25 us for 7000 slots against 200 for a sort.
    The marks stay under 64 MB (of which only the touched pages cost); wider ranges are sorted."""
    low, high = int(min(a.min(), b.min())), int(max(a.max(), b.max()))
    if high - low >= 1 << 26:
        return bool(np.intersect1d(a, b).size)
    marked = np.zeros(high - low + 1, dtype=bool)
    marked[a - low] = True
    return bool(marked[b - low].any())


class BlockKVOps:
    """``merge_blocks`` / ``append_block`` over a paged pool.

    The right block's keys are turned to where they now are, which a table with a factor (``RotaryEmbedding.cos_sin_cache``
    of a rotation with an attention factor) cannot do without making them longer: refused before anything is taken.

    ``kv_cache`` offers ``num_layers``, ``k_cache(layer)`` and ``v_cache(layer)``
    (contiguous ``[num_pages, page_size, kv_heads, head_dim]`` tensors on the
    GPU), or is the ``QuantizedKVCache`` of a ``QuantizedCacheAttention``, whose
    shifted keys are quantised anew; ``sc_attn`` is the ``SharedCacheAttention`` whose rotation the keys were
    stored with; ``page_allocator`` offers ``alloc_pages(n)``, and ``free_pages(page_starts)`` where pages of an eviction that
    fails are to go back to it.
    """

    def __init__(self, kv_cache, sc_attn, page_allocator,
                 compose_affines: Optional[Callable[..., Tuple[torch.Tensor, torch.Tensor]]] = None) -> None:
        if isinstance(kv_cache, QuantizedKVCache) and getattr(sc_attn, "kv_cache", None) is not kv_cache:
            raise ValueError("blocks of a QuantizedKVCache are moved by the QuantizedCacheAttention over it")
        self.kv_cache = kv_cache
        self.sc_attn = sc_attn
        self.page_allocator = page_allocator
        self.page_size = sc_attn.page_size
        self.device = sc_attn.device
        self.compose_affines = compose_affines
        self._refs: tuple = ()
        self._eviction: Optional[CacheEviction] = None

    def create_block(self) -> CacheBlock:
        return CacheBlock(self.device, self.page_size)

    # ------------------------------------------------------------------
    def merge_blocks(self, left: CacheBlock, right: CacheBlock) -> CacheBlock:
        """Copy ``left + right`` into a new compact block; both inputs stay
        valid and unchanged (reference ``session.py:330-377``)."""
        self._validate_block(left)
        self._validate_block(right)
        left_tokens, right_tokens = left.num_tokens, right.num_tokens
        left_span, right_span = left.mrope_span, right.mrope_span
        total_tokens = left_tokens + right_tokens
        if right_tokens and left_span:
            self.sc_attn._check_turns()

        merged = self.create_block()
        num_pages = -(-total_tokens // self.page_size)
        if num_pages:
            merged.page_starts = self.page_allocator.alloc_pages(num_pages).tolist()
        merged.num_tokens = total_tokens

        if left_tokens:
            self._copy_block(left, merged, destination_start=0)
        if right_tokens:
            self._copy_slots(token_slots(right), merged, destination_start=left_tokens, position_shift=left_span)
        self._finish_block_merge(destination=merged, left=left, right=right, left_span=left_span,
                                 right_span=right_span, keep_left_state=False)
        return merged

    def append_block(self, left: CacheBlock, right: CacheBlock) -> CacheBlock:
        """Append a copy of ``right`` to ``left`` and return ``left``; the free
        slots of ``left``'s last page are filled first.  ``append_block(b, b)``
        doubles ``b`` in place (reference ``session.py:379-420``)."""
        self._validate_block(left)
        self._validate_block(right)
        left_tokens, right_tokens = left.num_tokens, right.num_tokens
        left_span, right_span = left.mrope_span, right.mrope_span
        if right_tokens:
            if left_span:
                self.sc_attn._check_turns()
            # the source layout is taken before ``left`` grows: they may be the same object
            source_slots = token_slots(right)
            new_pages = self.page_allocator.alloc_pages(left.pages_needed(right_tokens))
            left.grow_pages(new_pages, right_tokens)
            self._copy_slots(source_slots, left, destination_start=left_tokens, position_shift=left_span)
        self._finish_block_merge(destination=left, left=left, right=right, left_span=left_span,
                                 right_span=right_span, keep_left_state=True)
        return left

    def evict_tokens(self, block: CacheBlock, weights: torch.Tensor, keep: int, first: int = 0, last: int = 0,
                     close_gaps: bool = False, others: Sequence[torch.Tensor] = ()) -> CacheBlock:
        """Copy what stays of ``block`` into a new compact block: ``keep`` tokens, the first ``first`` and the last ``last`` among
        them and the others by ``weights`` (``CacheEviction``), which move along.  Tokens leave all layers together: who keeps
        weights for each layer chooses by one of them, or by their sum, and names the ``others``, which move along too.
        ``block`` stays valid and unchanged; its pages are the caller's to hand back.

        Keys keep their positions and the new block spans as many as the old one; with ``close_gaps`` they are turned to
        the positions that the tokens have in the new block, which needs a block whose positions count its tokens.  A
        recurrent state, which holds all tokens, goes along as it is."""
        self._validate_block(block)
        if getattr(self.sc_attn, "kv_cache", None) is not self.kv_cache:
            raise ValueError("tokens are evicted with the attention over this pool")
        if self.device.type != "cuda":
            raise native.ViewAttnError("blocks are evicted from on the GPU only (HIP kernels, no CPU path)")
        if keep < 0 or first < 0 or last < 0:
            raise ValueError(f"keep, first and last must not be negative, got {keep}, {first} and {last}")
        if close_gaps and block.mrope_span != block.num_tokens:
            raise ValueError("close_gaps needs a block whose positions count its tokens")
        if self._eviction is None:
            self._eviction = CacheEviction(self.sc_attn)
        eviction = self._eviction
        moving = (weights, *others)
        for w in moving:
            eviction._check_weights(w)
        if close_gaps:
            self.sc_attn._check_turns()
        n = min(keep, block.num_tokens)
        result = self.create_block()
        span = n if close_gaps else block.mrope_span
        result.mrope_span_override = None if span == n else span
        result._replace_linear_states({i: (a.clone(), b.clone()) for i, (a, b) in block.linear_affine.items()},
                                      {i: s.clone() for i, s in block.linear_conv_state.items()})
        if n:
            pages = self.page_allocator.alloc_pages(-(-n // self.page_size))
            try:
                result.page_starts = pages.tolist()
                self._fill_evicted(result, block, moving, n, first, last, close_gaps)
            except BaseException:
                # nobody else knows of these pages
                hand_back = getattr(self.page_allocator, "free_pages", None)
                if hand_back is not None:
                    hand_back(pages)
                raise
        return result

    def _fill_evicted(self, result: CacheBlock, block: CacheBlock, weights: Sequence[torch.Tensor], n: int, first: int, last: int,
                      close_gaps: bool) -> None:
        eviction, source = self._eviction, token_slots(block)
        result.num_tokens = result.num_pages * self.page_size
        room = token_slots(result)  # whole pages
        result.num_tokens = n
        host = torch.from_numpy(np.concatenate([source, room])).pin_memory()
        dev = host.to(self.device, non_blocking=True)
        self._refs = (host, dev)
        for w in weights:
            eviction.clear(w, dev[source.size:])
        kept = eviction.select(weights[0], dev[: source.size], [source.size], n, first, last)
        eviction.move(kept.slots, dev[source.size: source.size + n], kept.shifts if close_gaps else None, weights)
        if len(block.token_ids) == block.num_tokens:
            result.token_ids = [block.token_ids[i] for i in kept.positions.tolist()]

    # ------------------------------------------------------------------
    def _finish_block_merge(self, *, destination: CacheBlock, left: CacheBlock, right: CacheBlock, left_span: int,
                            right_span: int, keep_left_state: bool) -> None:
        """Token ids, span and recurrent state of the result (reference
        ``session.py:422-477``)."""
        destination.token_ids = [*list(left.token_ids), *right.token_ids]
        merged_span = left_span + right_span
        destination.mrope_span_override = None if merged_span == destination.num_tokens else merged_span

        merged_affine: Dict[int, Tuple[torch.Tensor, torch.Tensor]] = {}
        for layer_idx in set(left.linear_affine) | set(right.linear_affine):
            left_pair = left.linear_affine.get(layer_idx)
            right_pair = right.linear_affine.get(layer_idx)
            if left_pair is None:
                merged_affine[layer_idx] = (right_pair[0].clone(), right_pair[1].clone())
            elif right_pair is None:
                merged_affine[layer_idx] = left_pair if keep_left_state else (left_pair[0].clone(), left_pair[1].clone())
            else:
                if self.compose_affines is None:
                    raise NotImplementedError(
                        "both blocks carry recurrent state for layer %d: pass compose_affines "
                        "(the model's composition of two affine summaries)" % layer_idx)
                merged_affine[layer_idx] = self.compose_affines(A_first=left_pair[0], B_first=left_pair[1],
                                                                A_second=right_pair[0], B_second=right_pair[1])
        merged_conv: Dict[int, torch.Tensor] = {}
        for layer_idx in set(left.linear_conv_state) | set(right.linear_conv_state):
            right_state = right.linear_conv_state.get(layer_idx)
            state = right_state if right_state is not None else left.linear_conv_state.get(layer_idx)
            merged_conv[layer_idx] = state if keep_left_state and right_state is None else state.clone()
        destination._replace_linear_states(merged_affine, merged_conv)

    def _validate_block(self, block: CacheBlock) -> None:
        if block.device != self.device:
            raise ValueError("block must belong to this session's device")
        if block.page_size != self.page_size:
            raise ValueError("block must use this session's page size")

    def _copy_block(self, source: CacheBlock, destination: CacheBlock, destination_start: int) -> None:
        """Copy all KV of ``source`` into one range of ``destination``."""
        self._copy_slots(token_slots(source), destination, destination_start)

    def _copy_slots(self, source_slots, destination: CacheBlock, destination_start: int,
                    position_shift: int = 0) -> None:
        """Copy KV from the given pool slots into ``destination`` from token
        ``destination_start`` on, in every layer; with ``position_shift`` the
        copied keys are rotated by it on the way (the reference's
        ``_copy_slots`` followed by ``_shift_keys_``)."""
        source = np.asarray(torch.as_tensor(source_slots).cpu(), dtype=np.int64).reshape(-1)
        n = source.size
        if n == 0:
            return
        target = token_slots(destination)[destination_start: destination_start + n]
        assert target.size == n, "destination block is too short for the copied run"
        # the kernel scatters while it gathers: a slot read by one token and written by another would race
        if slots_meet(source, target):
            raise ValueError("source and destination slots of a block copy overlap")
        self._launch(source, target, int(position_shift))

    def _shift_keys_(self, *, block: CacheBlock, start: int, num_tokens: int, position_shift: int) -> None:
        """Rotate stored keys ``[start, start + num_tokens)`` of ``block`` by
        ``position_shift`` in place (reference ``session.py:509-528``).  Merge and
        append do not need it here (the copy rotates); kept for callers that
        re-frame a block without copying it."""
        slots = token_slots(block)[start: start + num_tokens]
        if slots.size and position_shift:
            # source == destination row by row: every thread rewrites the pieces it read (the value
            # rows are rewritten unchanged)
            self._launch(slots, slots, int(position_shift))

    # ------------------------------------------------------------------
    def _launch(self, source: np.ndarray, target: np.ndarray, position_shift: int) -> None:
        att = self.sc_attn
        n = source.size
        if position_shift:
            att._check_turns()
        host = torch.from_numpy(np.stack([source, target]))
        if self.device.type != "cuda":
            raise native.ViewAttnError("block copies run on the GPU only (HIP kernel, no CPU path)")
        host = host.pin_memory()
        dev = host.to(self.device, non_blocking=True)
        self._refs = (host, dev)  # alive until the next copy on this stream has been queued
        if isinstance(self.kv_cache, QuantizedKVCache):
            att.copy_shifted(dev[0], dev[1], position_shift)
            return
        k0, v0 = self.kv_cache.k_cache(0), self.kv_cache.v_cache(0)
        assert k0.is_contiguous() and v0.is_contiguous(), "pool layers must be contiguous"
        width = att.num_kv_heads * att.head_dim
        rope = att._rope_descriptor() if position_shift else None
        stream = native.current_stream_ptr(self.device)
        for first, count, stride in layer_runs(self.kv_cache):
            k_pool, v_pool = self.kv_cache.k_cache(first), self.kv_cache.v_cache(first)
            native.check(native.lib.va_copy_shift_kv(
                k_pool.data_ptr(), v_pool.data_ptr(), width, stride, count, dev[0].data_ptr(), dev[1].data_ptr(),
                n, position_shift, att._shape, rope, stream))
