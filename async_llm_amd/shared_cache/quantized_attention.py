"""Cache-view attention over an 8-bit pool.

``QuantizedCacheAttention`` is ``SharedCacheAttention`` over a ``QuantizedKVCache``: the
same constructor, planners, metadata and calls.  New keys are rotated to their
block-relative position in fp32 and quantised with their values as they are written;
attention reads the codes and takes each row's scale into the score (K) or the weight
(V), so nothing is read back on the way:

    score(row, t) = (R(loc) q . code_k[t]) * 2^e_k[t] / sqrt(head_dim)
    out(row)      = sum_t softmax(score)(t) * 2^e_v[t] * code_v[t]

Queries and weights are not rounded to the activations' type in between: a step over an
8-bit cache differs from one over its read-back values by the rounding of the result.

The reference has no such cache; its path over 16-bit pools is
``python/minisgl/shared_cache/attention.py:624-752``.
"""

from __future__ import annotations

import numpy as np
import torch

from .. import native
from ..kvcache.quantized_pool import QuantizedKVCache, store_quantized
from .attention import SharedCacheAttention, SharedCacheAttnMetadata


class QuantizedCacheAttention(SharedCacheAttention):
    """View attention over a :class:`QuantizedKVCache` whose ``dtype`` is the op's."""

    def __init__(self, kv_cache: QuantizedKVCache, cos_sin_cache: torch.Tensor, num_qo_heads: int, num_kv_heads: int,
                 head_dim: int, page_size: int, dtype: torch.dtype, device: torch.device, rotary_dim: int | None = None,
                 mrope_section: tuple | None = None, rope_base: float | None = None, kernel: str | None = None) -> None:
        if not isinstance(kv_cache, QuantizedKVCache):
            raise TypeError(f"kv_cache must be a QuantizedKVCache, got {type(kv_cache).__name__}")
        want = (num_kv_heads, head_dim, page_size, dtype)
        have = (kv_cache.num_kv_heads, kv_cache.head_dim, kv_cache.page_size, kv_cache.dtype)
        if want != have:
            raise ValueError(f"kv_cache holds (kv_heads, head_dim, page_size, dtype) = {have}, the op wants {want}")
        if num_qo_heads % num_kv_heads:
            raise ValueError(f"{num_qo_heads} q heads are no multiple of {num_kv_heads} kv heads")
        super().__init__(kv_cache, cos_sin_cache, num_qo_heads, num_kv_heads, head_dim, page_size, dtype, kv_cache.device,
                         rotary_dim=rotary_dim, mrope_section=mrope_section, rope_base=rope_base, kernel=kernel,
                         fused_store=False)
        device = torch.device(device)
        if device.type != self.device.type or device.index not in (None, self.device.index):
            raise ValueError(f"kv_cache lives on {self.device}, the op is to run on {device}")
        if page_size < 16 or page_size & (page_size - 1):
            self.plan_params.wide_tile = -1  # wide tiles take their tokens in halves of sixteen that lie inside a page

    # ------------------------------------------------------------------
    # planning
    # ------------------------------------------------------------------
    def _build_launch(self, qo_indptr, kv_indptr, kv_indices_host, seq_lens, flags, chain, sub_worker_host, n_rows,
                      tables, refs):
        kv = np.asarray(kv_indices_host)
        if kv.size:
            # page numbers, and token slots of sub-requests that list those
            slots = np.repeat(np.asarray(flags) & native.VA_SUB_SLOTS, np.diff(np.asarray(kv_indptr))) != 0
            limit = np.where(slots, self.kv_cache.num_pages * self.page_size, self.kv_cache.num_pages)
            bad = np.nonzero((kv < 0) | (kv >= limit))[0]
            if bad.size:
                raise ValueError(f"{'slot' if slots[bad[0]] else 'page'} {int(kv[bad[0]])} lies outside the pool of "
                                 f"{self.kv_cache.num_pages} pages of {self.page_size} tokens")
        return super()._build_launch(qo_indptr, kv_indptr, kv_indices_host, seq_lens, flags, chain, sub_worker_host, n_rows,
                                     tables, refs)

    # ------------------------------------------------------------------
    # execution
    # ------------------------------------------------------------------
    def store_new_kv(self, k: torch.Tensor, v: torch.Tensor, layer_id: int, batch) -> None:
        """Rotate the new keys to their block-relative positions, quantise K and V rows and write them to
        ``batch.out_loc`` (negative slots are skipped)."""
        where = batch.positions if batch.mrope_positions is None else batch.mrope_positions
        store_quantized(self.kv_cache, k, v, batch.out_loc, layer_id, where, self._rope_descriptor())

    def attend(self, q: torch.Tensor, layer_id: int, meta: SharedCacheAttnMetadata, return_lse: bool = False,
               lse_base2: bool = False, out: torch.Tensor | None = None, lse: torch.Tensor | None = None,
               static_scratch: bool = False):
        """Run the planned attention over the pool as it is now; returns ``out [rows, Hq*D]`` (and ``lse [rows, Hq]``
        fp32 on request).  ``static_scratch`` is refused: partial states go to the op's workspace."""
        if static_scratch:
            raise ValueError("attention over a quantised pool has no static scratch: reserve a workspace with prepare_workspace")
        native.require_device(q, "q")
        launch = meta.launch
        assert launch is not None, "metadata carries no launch plan"
        W, Hq, D = meta.num_workers, self.num_qo_heads, self.head_dim
        q2, q_stride = self._rows(q, Hq)
        if q2.shape[0] < W or q2.dtype != self.dtype or q2.device != self.device:
            raise ValueError(f"q must be {W} rows of {Hq * D} {self.dtype} elements on {self.device}, got {q2.dtype} "
                             f"{tuple(q2.shape)} on {q2.device}")
        if out is None:
            out = torch.empty((W, Hq * D), dtype=self.dtype, device=self.device)
        elif out.shape != (W, Hq * D) or out.dtype != self.dtype or not out.is_contiguous() or out.device != self.device:
            raise ValueError(f"out must be a contiguous {self.dtype} tensor [{W}, {Hq * D}] on {self.device}")
        if lse is None:
            lse = torch.empty((W, Hq), dtype=torch.float32, device=self.device) if return_lse else None
        elif lse.shape != (W, Hq) or lse.dtype != torch.float32 or not lse.is_contiguous() or lse.device != self.device:
            raise ValueError(f"lse must be a contiguous float32 tensor [{W}, {Hq}] on {self.device}")
        ws = launch.workspace
        native.call_on(self.device, native.lib.va_attention_q8, q2.data_ptr(), q_stride, self.kv_cache.layer(layer_id),
                       launch.blob.data_ptr(), launch.header_ptr, launch.kv_indices.data_ptr(), meta.sub_worker.data_ptr(),
                       meta.sub_loc.data_ptr(), meta.sub_loc.stride(0) if meta.sub_loc.dim() == 2 else 0, out.data_ptr(),
                       None if lse is None else lse.data_ptr(), int(lse_base2), None if ws is None else ws.data_ptr(),
                       0 if ws is None else ws.numel(), self._shape, self._rope_descriptor(),
                       native.current_stream_ptr(self.device))
        return (out, lse) if return_lse else out

    # ------------------------------------------------------------------
    # moving tokens
    # ------------------------------------------------------------------
    def copy_shifted(self, source: torch.Tensor, target: torch.Tensor, position_shift: int = 0) -> None:
        """Copy the tokens of slots ``source`` to slots ``target`` (int64 on the device, each target once, none of
        them a source of another token) in every layer, keys rotated by ``position_shift`` and quantised anew; values,
        and keys where nothing rotates, move code for code."""
        for name, t in (("source", source), ("target", target)):
            native.require_device(t, name)
            if t.dim() != 1 or t.dtype != torch.int64 or t.device != self.device or t.numel() != source.numel():
                raise ValueError(f"{name} must be one row of {source.numel()} int64 slots on {self.device}, got {t.dtype} "
                                 f"{tuple(t.shape)} on {t.device}")
        pool, source, target = self.kv_cache, source.contiguous(), target.contiguous()
        if pool.num_layers:
            native.call_on(self.device, native.lib.va_copy_shift_kv_q8, pool.layer(0), pool.code_layer_bytes,
                           pool.scale_layer_bytes, pool.num_layers, source.data_ptr(), target.data_ptr(), source.numel(),
                           int(position_shift), self._shape, self._rope_descriptor() if position_shift else None,
                           native.current_stream_ptr(self.device))
