"""Eviction from a paged cache by accumulated attention weight.

Blocks of a view live long and only ever grow.  ``CacheEviction`` keeps count of what
attention looks at, chooses what stays of a block and moves that together:

* ``accumulate`` adds, for every cached token and kv head, the softmax weight that a
  step's queries gave the token (from the step's plan, its unrotated queries and its
  log-sums) to ``weights [kv_heads, slots]``;
* ``select`` keeps of each block the first and the last few tokens and the heaviest of
  the others;
* ``move`` copies tokens to other slots in all layers, each key turned by a shift of its
  own, and their weights with them.

``BlockKVOps.evict_tokens`` does the last two for a block.  The reference has no eviction;
what this stands beside is its block merge and append
(``python/minisgl/shared_cache/session.py:330-528``).

Weights are by slot: whoever hands pages back and gets them again clears theirs (``clear``).
A key keeps its position where it is moved without a shift: the block then spans as many
positions as before.
"""

from __future__ import annotations

import ctypes
import numbers
from dataclasses import dataclass
from typing import Dict, List, Optional, Sequence, Union

import numpy as np
import torch

from .. import native
from ..kvcache.mha_pool import MHAKVCache, layer_runs
from ..kvcache.quantized_pool import QuantizedKVCache
from .attention import SharedCacheAttention, SharedCacheAttnMetadata


@dataclass
class WeightPlan:
    """Who sees which token in a step, by token; serves all layers of the step."""

    rows: int  # query rows of the step
    counts: native.VaWeighCounts
    tables: tuple  # what the library takes of it: addresses of the plan and its header, of the step's rows and positions
    refs: tuple  # the tensors and arrays behind those


@dataclass
class KeptTokens:
    """What stays of some blocks, one after the other: positions in each block in rising order, slots, new position minus
    position (int64 on the device), and how many of each block (host)."""

    positions: torch.Tensor
    slots: torch.Tensor
    shifts: torch.Tensor
    counts: List[int]


class CacheEviction:
    """Eviction over the pool of ``op``, a ``SharedCacheAttention`` or ``QuantizedCacheAttention``."""

    def __init__(self, op: SharedCacheAttention) -> None:
        self.op = op
        self.kv_cache = op.kv_cache
        self.device = op.device
        if self.device.type == "cuda" and self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        if op.num_qo_heads % op.num_kv_heads:
            raise ValueError(f"{op.num_qo_heads} q heads are no multiple of {op.num_kv_heads} kv heads")
        self._coded = isinstance(self.kv_cache, QuantizedKVCache)
        if self._coded:
            self.num_pages = self.kv_cache.num_pages
        else:
            op._check_pool_layout()
            self.num_pages = self.kv_cache.k_cache(0).shape[0]
        self.num_slots = self.num_pages * op.page_size
        if self.num_slots > 2**31 - 1:
            raise ValueError(f"{self.num_pages} pages of {op.page_size} tokens are more slots than 32 bits address")
        self._weights_shape = (op.num_kv_heads, self.num_slots)
        self._key_addresses: Dict[int, int] = {}
        self._moved: Optional[list] = None

    # ------------------------------------------------------------------
    # weights
    # ------------------------------------------------------------------
    def new_weights(self) -> torch.Tensor:
        """Weights of a pool that nobody has looked at: float32 zeros ``[kv_heads, slots]``."""
        return torch.zeros((self.op.num_kv_heads, self.num_slots), dtype=torch.float32, device=self.device)

    def _check_weights(self, weights: torch.Tensor, name: str = "weights") -> None:
        if weights.shape != self._weights_shape or weights.dtype is not torch.float32 or weights.device != self.device \
                or not weights.is_contiguous():
            native.require_device(weights, name)
            raise ValueError(f"{name} must be a contiguous float32 tensor {list(self._weights_shape)} on {self.device}, got "
                             f"{weights.dtype} {list(weights.shape)} on {weights.device}")

    def clear(self, weights: torch.Tensor, slots: torch.Tensor) -> None:
        """Forget what the tokens of ``slots`` (whole numbers; those outside the pool are skipped) were given."""
        self._check_weights(weights)
        if slots.dim() != 1 or slots.is_floating_point() or slots.is_complex() or slots.dtype is torch.bool:
            raise ValueError(f"slots must be one row of whole numbers, got {slots.dtype} {tuple(slots.shape)}")
        native.require_device(weights, "weights")
        slots = slots.to(device=self.device, dtype=torch.int64).contiguous()
        native.call_on(self.device, native.lib.va_clear_weights, weights.data_ptr(), *self._weights_shape, slots.data_ptr(),
                       slots.numel(), native.current_stream_ptr(self.device))

    def plan(self, meta: SharedCacheAttnMetadata, window: int = 0) -> WeightPlan:
        """Turn a step's plan (of ``prepare``, ``prepare_prefill_batch`` or ``prepare_mixed``) round.  ``window > 0``: of many new
        tokens of a request only the last ``window`` are counted."""
        tables = None if meta.launch is None else meta.launch.host_tables
        if meta.shared_cache_op is not self.op or tables is None:
            raise ValueError("plan needs the metadata of a step that this op planned without fixed buffers")
        if window < 0:
            raise ValueError(f"window must not be negative, got {window}")
        arrays, sub_worker, n_rows = tables
        n_sub = len(arrays[3])
        subs = native.VaSubRequests(n_sub, len(sub_worker), n_rows, arrays[0].ctypes.data, arrays[1].ctypes.data,
                                    arrays[2].ctypes.data if arrays[2].size else None, arrays[3].ctypes.data,
                                    arrays[4].ctypes.data, None, None)
        counts = native.VaWeighCounts()
        pinned = self.device.type == "cuda"
        capacity = (1 << 14) + 2 * arrays[2].size + 8 * len(sub_worker)  # (room for most plans)
        while True:
            host = torch.empty(capacity, dtype=torch.int32, pin_memory=pinned)
            words = host.numpy()
            rc = native.lib.va_weigh_plan(subs, self.op._shape, int(self._coded), self.num_pages, window, host.data_ptr(), capacity, counts)
            if rc != native.VA_ERR_CAPACITY or counts.plan_words <= capacity:
                break
            capacity = counts.plan_words
        native.check(rc)
        blob = host[: counts.plan_words].to(self.device, non_blocking=True)
        header, sub_loc = words[: native.WEIGH_HEADER_WORDS].copy(), meta.sub_loc
        tables = (blob.data_ptr(), header.ctypes.data, meta.sub_worker.data_ptr(), sub_loc.data_ptr(),
                  sub_loc.stride(0) if sub_loc.dim() == 2 else 0)
        return WeightPlan(meta.num_workers, counts, tables, (host, blob, header, meta.sub_worker, sub_loc))

    def accumulate(self, q: torch.Tensor, lse: torch.Tensor, layer_id: int, plan: WeightPlan, weights: torch.Tensor,
                   out: Optional[torch.Tensor] = None, lse_base2: bool = False) -> torch.Tensor:
        """Add what the step's queries ``q`` (unrotated rows, as ``forward`` takes them) gave the tokens of layer ``layer_id``
        to ``weights``, and return it.  ``lse [rows, q_heads]``: the log-sums that ``forward_with_lse`` returned for the same
        queries.  With ``out`` the sums of the tokens in sight go there instead, and ``weights`` and the other slots of
        ``out`` stay as they are."""
        if not q.is_cuda:
            native.require_device(q, "q")
        op, device, rows = self.op, self.device, plan.rows
        q2, q_stride = op._rows(q, op.num_qo_heads)
        if q2.dtype is not op.dtype or q2.device != device or q2.shape[0] < rows:
            raise ValueError(f"q must be {rows} rows of {op.dtype} on {device}, got {q2.dtype} {tuple(q2.shape)} on {q2.device}")
        shape = lse.shape
        if len(shape) != 2 or shape[0] < rows or shape[1] != op.num_qo_heads or lse.dtype is not torch.float32 \
                or lse.device != device or not lse.is_contiguous():
            raise ValueError(f"lse must be a contiguous float32 tensor [{rows}, {op.num_qo_heads}] on {device}, got {lse.dtype} "
                             f"{tuple(shape)} on {lse.device}")
        self._check_weights(weights)
        if out is None:
            out = weights
        else:
            self._check_weights(out, "out")
        # (from the allocator, call by call: streams and graphs that share a plan have scratch of their own)
        nbytes = plan.counts.workspace_bytes
        workspace = torch.empty(nbytes, dtype=torch.uint8, device=device)
        tables = (*plan.tables, lse.data_ptr(), int(lse_base2), weights.data_ptr(), out.data_ptr(), workspace.data_ptr(), nbytes,
                  op._shape, op._rope_descriptor(), native.current_stream_ptr(device))
        if self._coded:
            native.call_on(device, native.lib.va_weigh_q8, q2.data_ptr(), q_stride, self.kv_cache.layer(layer_id), *tables)
        else:
            native.call_on(device, native.lib.va_weigh, q2.data_ptr(), q_stride, self._keys_at(layer_id),
                           op.num_kv_heads * op.head_dim, self.num_pages, *tables)
        return out

    def _keys_at(self, layer_id: int) -> int:
        """Address of a layer's keys, asked for once where the pool is this package's own, whose arrays stay."""
        at = self._key_addresses.get(layer_id)
        if at is None:
            pool, op = self.kv_cache.k_cache(layer_id), self.op
            if tuple(pool.shape) != (self.num_pages, op.page_size, op.num_kv_heads, op.head_dim) or pool.dtype != op.dtype \
                    or pool.device != self.device or not pool.is_contiguous():
                raise ValueError(f"kv_cache.k_cache({layer_id}) must be a contiguous {op.dtype} tensor of {self.num_pages} pages on "
                                 f"{self.device}")
            at = pool.data_ptr()
            if type(self.kv_cache) is MHAKVCache:
                self._key_addresses[layer_id] = at
        return at

    # ------------------------------------------------------------------
    # choosing
    # ------------------------------------------------------------------
    @staticmethod
    def select(weights: torch.Tensor, slots: torch.Tensor, counts: Sequence[int], keep: Union[int, Sequence[int]],
               first: int = 0, last: int = 0) -> KeptTokens:
        """What stays of blocks whose token slots are ``counts[b]`` consecutive entries of ``slots`` (int64): ``keep[b]`` tokens (all of
        a block with fewer), the first ``first`` and the last ``last`` among them (the lower positions where those are more), the
        others by ``weights [heads, slots]``, heaviest first; ties go to the lower position."""
        native.require_device(weights, "weights")
        device = weights.device
        if weights.dim() != 2 or weights.dtype != torch.float32 or not weights.is_contiguous():
            raise ValueError(f"weights must be a contiguous float32 tensor [heads, slots], got {weights.dtype} {tuple(weights.shape)}")
        if slots.dim() != 1 or slots.dtype != torch.int64 or slots.device != device:
            raise ValueError(f"slots must be one row of int64 on {device}, got {slots.dtype} {tuple(slots.shape)} on {slots.device}")
        tokens = [int(n) for n in counts]
        wanted = [int(keep)] * len(tokens) if isinstance(keep, numbers.Integral) else [int(n) for n in keep]
        if len(wanted) != len(tokens):
            raise ValueError(f"{len(wanted)} numbers of tokens to keep of {len(tokens)} blocks")
        if tokens and (min(tokens) < 0 or min(wanted) < 0) or first < 0 or last < 0:
            raise ValueError("counts, keep, first and last must not be negative")
        if sum(tokens) != slots.numel():
            raise ValueError(f"counts add up to {sum(tokens)} tokens, slots has {slots.numel()}")
        wanted = [min(a, b) for a, b in zip(wanted, tokens)]
        results = torch.empty((3, sum(wanted)), dtype=torch.int64, device=device)
        positions, kept_slots, shifts = results.unbind(0)
        many = ctypes.c_int64 * len(tokens)
        tokens, stay = many(*tokens), many(*wanted)
        nbytes = native.lib.va_select_workspace_bytes(len(wanted), tokens)
        if nbytes < 0:
            raise ValueError("a block holds at most 2^31 - 1 tokens")
        workspace = torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None
        slots = slots.contiguous()
        native.call_on(device, native.lib.va_select_tokens, weights.data_ptr(), weights.shape[0], weights.shape[1], slots.data_ptr(),
                       len(wanted), tokens, stay, first, last, positions.data_ptr(), kept_slots.data_ptr(), shifts.data_ptr(),
                       None if workspace is None else workspace.data_ptr(), nbytes, native.current_stream_ptr(device))
        return KeptTokens(positions, kept_slots, shifts, wanted)

    # ------------------------------------------------------------------
    # moving
    # ------------------------------------------------------------------
    def move(self, source: torch.Tensor, target: torch.Tensor, shifts: Optional[torch.Tensor] = None,
             weights: Union[None, torch.Tensor, Sequence[torch.Tensor]] = None) -> None:
        """Copy the tokens of slots ``source`` to slots ``target`` (int64 on the device, each target once, none of them a source of
        another token) in every layer, keys rotated by ``shifts`` (int64; ``None``: as they are), and their ``weights`` (a tensor, or
        several, as one for each layer)."""
        op, device, n = self.op, self.device, source.numel()
        for name, t in (("source", source), ("target", target), ("shifts", shifts)):
            if t is None and name == "shifts":
                continue
            if t.dim() != 1 or t.dtype is not torch.int64 or t.device != device or t.numel() != n:
                native.require_device(t, name)
                raise ValueError(f"{name} must be one row of {n} int64 numbers on {device}, got {t.dtype} {tuple(t.shape)} on {t.device}")
        native.require_device(source, "source")
        weights = () if weights is None else (weights,) if isinstance(weights, torch.Tensor) else tuple(weights)
        for w in weights:
            self._check_weights(w)
        if shifts is not None:
            op._check_turns()
        source, target = source.contiguous(), target.contiguous()
        shifts = None if shifts is None else shifts.contiguous()
        rest = (source.data_ptr(), target.data_ptr(), None if shifts is None else shifts.data_ptr(), n)
        shape, rope, stream = op._shape, None if shifts is None else op._rope_descriptor(), native.current_stream_ptr(device)
        sums = [w.data_ptr() for w in weights]
        if self._coded:
            pool = self.kv_cache
            if pool.num_layers:
                native.call_on(device, native.lib.va_move_kv_q8, pool.layer(0), pool.code_layer_bytes, pool.scale_layer_bytes,
                               pool.num_layers, *rest, sums.pop(0) if sums else None, shape, rope, stream)
        else:
            for run in self._layers_at():
                native.call_on(device, native.lib.va_move_kv, *run, *rest, sums.pop(0) if sums else None, shape, rope, stream)
        for w in sums:
            native.call_on(device, native.lib.va_move_kv, None, None, 0, 0, 0, self.num_slots, *rest, w, shape, None, stream)

    def _layers_at(self) -> list:
        """Where the pool's layers lie, as the library takes them; found once where the pool is this package's own."""
        runs = self._moved
        if runs is None:
            pool, op = self.kv_cache, self.op
            for layer in range(pool.num_layers):
                op._check_pool_layout(layer)
                if pool.k_cache(layer).shape[0] != self.num_pages or pool.v_cache(layer).shape[0] != self.num_pages:
                    raise ValueError(f"layer {layer} of kv_cache must hold {self.num_pages} pages")
            width = op.num_kv_heads * op.head_dim
            runs = [(pool.k_cache(first).data_ptr(), pool.v_cache(first).data_ptr(), width, stride, count, self.num_slots)
                    for first, count, stride in layer_runs(pool)]
            if type(pool) is MHAKVCache:
                self._moved = runs
        return runs
