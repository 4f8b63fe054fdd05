"""Cache-view attention over an 8-bit pool.

``QuantizedCacheAttention`` is ``SharedCacheAttention`` over a ``QuantizedKVCache``: the
same constructor, planners, metadata and calls.  New keys are rotated to their
block-relative position in fp32 and quantised with their values as they are written;
attention reads the codes and takes each row's scale into the score (K) or the weight
(V):

    score(row, t) = (R(loc) q . code_k[t]) * 2^e_k[t] / sqrt(head_dim)
    out(row)      = sum_t softmax(score)(t) * 2^e_v[t] * code_v[t]

Queries and weights are not rounded to the activations' type in between: such a step
differs from one over the read-back values by the rounding of the result.  Values are summed
in 32 bits under weights of up to 2^8: results are finite for |v| up to 2^119 divided by the
tokens in sight.  A key or value row that is not finite makes NaN of the results that see it, and
of no other; the lse of such results has no meaning (it is NaN for keys, and for values where the
step was read back).

Chunks of many new tokens read a token so often that it is converted once: their pages
are read back as float16, within range by powers of two, and the 16-bit attention's
matrix-core kernels run over that: for bf16 activations, whose results are rounded by more than
float16's eleven bits cost the operands.  One pair of powers serves a whole step, so
one whose rows differ too much in size for float16 -- a key of 1e6 in any of its requests, a
value 2^16 times as large as another -- is answered over the codes after all: the launch over
them stands behind the others and runs where these found that.  Plans over a workspace reserved
by ``prepare_workspace`` never read back.

The reference has no such cache; its path over 16-bit pools is
``python/minisgl/shared_cache/attention.py:624-752``.
"""

from __future__ import annotations

from dataclasses import dataclass
from typing import Optional

import numpy as np
import torch

from .. import native
from ..kvcache.quantized_pool import QuantizedKVCache, store_quantized
from .attention import LaunchPlan, SharedCacheAttention, SharedCacheAttnMetadata


@dataclass
class ReadBack:
    """The part of a step that runs over rows read back as float16: its plan, which knows the pages by their place in the
    scratch, and the slots that fill it."""

    launch: LaunchPlan
    first_row: int  # rows in front of it are the codes' launch
    sub_worker: torch.Tensor
    first_subrow: int
    slots: torch.Tensor  # int64, of every token of every page that it reads, -1 behind the last token of a page
    scratch: torch.Tensor  # its first word: whether float16 did not hold the step
    codes: LaunchPlan  # the same rows over the codes, for that case


class QuantizedCacheAttention(SharedCacheAttention):
    """View attention over a :class:`QuantizedKVCache` whose ``dtype`` is the op's."""

    _over_codes = True

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
        p = self.plan_params
        self._read_back_params = native.VaPlanParams(p.kernel, p.q_tile, p.kv_chunk, p.target_items, p.wide_tile)
        p.wide_tile = native.VA_TILES_APART  # codes are read by tiles of up to 16 rows, a workgroup each
        # one work item a tile: nothing to merge, no workspace
        self._uncut_params = native.VaPlanParams(p.kernel, p.q_tile, p.kv_chunk, 1, p.wide_tile)
        self._read_back_shape = native.make_shape(num_qo_heads, num_kv_heads, head_dim, page_size, torch.float16)
        self._matrix_core = p.kernel != native.VA_KERNEL_GENERIC and dtype != torch.float32 and head_dim in (64, 128, 256) \
            and num_qo_heads // num_kv_heads in (1, 2, 4, 8, 16)
        self._scratch: Optional[torch.Tensor] = None

    # ------------------------------------------------------------------
    # planning
    # ------------------------------------------------------------------
    def _check_entries(self, kv_indices, kv_indptr, flags) -> None:
        if not kv_indices.size:
            return
        # page numbers, and token slots of sub-requests that list those
        pages = self.kv_cache.num_pages
        if kv_indices.min() >= 0 and kv_indices.max() < pages:
            return
        slots = np.repeat(flags & native.VA_SUB_SLOTS, np.diff(kv_indptr)) != 0
        bad = np.flatnonzero((kv_indices < 0) | (kv_indices >= np.where(slots, pages * self.page_size, pages)))
        if bad.size:
            raise ValueError(f"{'slot' if slots[bad[0]] else 'page'} {int(kv_indices[bad[0]])} lies outside the pool of "
                             f"{pages} pages of {self.page_size} tokens")

    def _build_launch(self, qo_indptr, kv_indptr, kv_indices_host, seq_lens, flags, chain, sub_worker_host, n_rows,
                      tables, refs):
        kv = np.asarray(kv_indices_host)
        self._check_entries(kv, np.asarray(kv_indptr), np.asarray(flags))
        qo, kvp = np.asarray(qo_indptr), np.asarray(kv_indptr)
        # chains stand behind the decodes; their pages count by their place among the distinct ones
        n_codes = int(np.argmax(np.asarray(chain) >= 0)) if len(chain) and chain[-1] >= 0 else len(chain)
        pages = np.empty(0, dtype=np.int64)
        if n_codes < len(chain) and self._matrix_core and not self._workspace_prepared \
                and not (np.asarray(flags[n_codes:]) & native.VA_SUB_SLOTS).any():
            held = np.zeros(self.kv_cache.num_pages, dtype=np.int64)  # tokens of every page that someone sees
            lengths = np.asarray(seq_lens[n_codes:], dtype=np.int64)
            for begin, end, length in zip(kvp[n_codes:].tolist(), kvp[n_codes + 1:].tolist(), lengths.tolist()):
                full, rest = divmod(length, self.page_size)
                held[kv[begin: min(begin + full, end)]] = self.page_size
                if rest and begin + full < end:
                    held[kv[begin + full]] = max(held[kv[begin + full]], rest)
            pages = np.flatnonzero(held)
        if not len(pages) or not self._reads_back(int((np.diff(qo[n_codes:]) * lengths).sum()), len(pages)):
            return super()._build_launch(qo_indptr, kv_indptr, kv_indices_host, seq_lens, flags, chain, sub_worker_host,
                                         n_rows, tables, refs)
        first_entry, first_subrow = int(kvp[n_codes]), int(qo[n_codes])
        places = np.maximum(np.cumsum(held > 0)[kv[first_entry:]] - 1, 0)  # (a listed page that nobody sees: any of them)
        within = np.arange(self.page_size, dtype=np.int64)
        slots = np.where(within < held[pages, None], pages[:, None] * self.page_size + within, -1).reshape(-1)
        rows = np.asarray(sub_worker_host)[first_subrow:]
        first_row = int(rows.min())
        relative = (qo[n_codes:] - first_subrow, kvp[n_codes:] - first_entry)
        described = (seq_lens[n_codes:], flags[n_codes:], chain[n_codes:], rows - first_row, n_rows - first_row)
        over_codes, _ = super()._build_launch(*relative, kv[first_entry:], *described, (), refs, self._uncut_params)
        assert not over_codes.counts.n_partials
        scratch = self._ensure_scratch(int(native.lib.va_read_back_bytes(len(slots), n_rows - first_row, self._shape)))
        more = () if n_codes else tuple(tables)
        wide, (dev_rows, dev_slots, *dev_tables) = super()._build_launch(
            *relative, places, *described, (rows - first_row, slots, *more), refs, self._read_back_params,
            self._read_back_shape)
        back = ReadBack(wide, first_row, dev_rows, first_subrow, dev_slots, scratch, over_codes)
        if n_codes:
            launch, dev_tables = super()._build_launch(qo[: n_codes + 1], kvp[: n_codes + 1], kv[:first_entry],
                                                       seq_lens[:n_codes], flags[:n_codes], chain[:n_codes],
                                                       np.asarray(sub_worker_host)[:first_subrow], first_row, tables, refs)
        else:
            launch = LaunchPlan(wide.header, wide.blob, wide.kv_indices, wide.counts, wide.workspace)
        launch.readback = back
        arrays = [np.ascontiguousarray(a, dtype=np.int32) for a in (qo, kvp, kv, seq_lens, flags, chain)]
        launch.host_tables = (arrays, np.ascontiguousarray(sub_worker_host, dtype=np.int64), n_rows)
        return launch, dev_tables

    def _reads_back(self, pairs: int, pages: int) -> bool:
        """Whether the chains of a step, ``pairs`` of a row and a token that it may see, run over rows read back.

        Not those of float16 activations: operands of float16 put errors on the result that are larger than its own
        rounding.  Relative to the result (2-norms), over codes / read back, 64 rows over 7800 tokens, 32 q and 8 kv heads of
        128: float16 0.00021 / 0.00036, with scores up to +-100 0.00014 / 0.00063; bf16 0.00166 / 0.00172, 0.00106 / 0.00128.

        Reading back costs five launches more and 2 ns a token of 1024 elements, and takes half to two thirds off the products.
        Us read back / over codes, one chunk, 32 q and 8 kv heads of 128: 256 rows over 3000 tokens 61 / 52, 48 (64) rows over
        20000 84 / 80 (89 / 106), 24 rows 80 / 48; 8 and 8 heads: 128 (256) rows over 20000 81 / 62 (92 / 108); 16 and 4
        heads of 256: 64 (96) rows over 20000 86 / 78 (98 / 107), 256 rows over 3000 59 / 58; 64 and 16 heads of 64: 24 (32) rows
        over 20000 83 / 68 (85 / 91), 256 rows over 3000 64 / 59. They change sides between 2.4e9 and 7e9 products, most near 4e9,
        and at 120 to 350 query rows a token and kv head where the tokens are many.  One line for all of them is off by up to a
        tenth beside it: 64 rows of 16 and 4 heads of 256 over 20000 tokens are read back, 32 rows of 64 and 16 heads of 64 are not.
        """
        products = pairs * self.num_qo_heads * self.head_dim
        return self.dtype == torch.bfloat16 and products >= 4 << 30 and products >= 160 * pages * self.page_size * self.num_kv_heads * self.head_dim

    def _ensure_scratch(self, nbytes: int) -> torch.Tensor:
        """Room for rows read back, shared by the op's steps like their workspace; a plan keeps the tensor it was given."""
        if self._scratch is None or self._scratch.numel() < nbytes:
            self._scratch = torch.empty(nbytes, dtype=torch.uint8, device=self.device)
        return self._scratch

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
        launch, device = meta.launch, self.device
        W, Hq = meta.num_workers, self.num_qo_heads
        width = Hq * self.head_dim
        q2, q_stride = self._rows(q, Hq)
        if q2.dtype != self.dtype or q2.device != device or q2.shape[0] < W:
            native.require_device(q, "q")
            raise ValueError(f"q must be {W} rows of {width} {self.dtype} elements on {device}, got {q2.dtype} "
                             f"{tuple(q2.shape)} on {q2.device}")
        native.require_device(q2, "q")
        assert launch is not None, "metadata carries no launch plan"
        if out is None:
            # (empty_strided: 0.4 us less than empty)
            out = torch.empty_strided((W, width), (width, 1), dtype=self.dtype, device=device)
        elif out.shape != (W, width) or out.dtype != self.dtype or not out.is_contiguous() or out.device != device:
            raise ValueError(f"out must be a contiguous {self.dtype} tensor [{W}, {width}] on {device}")
        if lse is None:
            lse = torch.empty_strided((W, Hq), (Hq, 1), dtype=torch.float32, device=device) if return_lse else None
        elif lse.shape != (W, Hq) or lse.dtype != torch.float32 or not lse.is_contiguous() or lse.device != device:
            raise ValueError(f"lse must be a contiguous float32 tensor [{W}, {Hq}] on {device}")
        stream, rope = native.current_stream_ptr(device), self._rope_descriptor()
        lse_ptr = None if lse is None else lse.data_ptr()
        sub_loc = meta.sub_loc
        axis_stride = sub_loc.stride(0) if sub_loc.dim() == 2 else 0
        pool, back = self.kv_cache.layer(layer_id), launch.readback
        if back is None or back.first_row:
            ws = launch.workspace
            native.call_on(device, native.lib.va_attention_q8, q2.data_ptr(), q_stride, pool, launch.blob.data_ptr(),
                           launch.header_ptr, launch.kv_indices.data_ptr(), meta.sub_worker.data_ptr(),
                           sub_loc.data_ptr(), axis_stride, out.data_ptr(), lse_ptr, int(lse_base2),
                           None if ws is None else ws.data_ptr(), 0 if ws is None else ws.numel(), self._shape, rope, stream)
        if back is not None:
            plan, item = back.launch, q2.element_size()
            ws, scratch = plan.workspace, back.scratch.data_ptr()
            q_ptr = q2.data_ptr() + back.first_row * q_stride * item
            rows = (back.sub_worker.data_ptr(), sub_loc.data_ptr() + 8 * back.first_subrow, axis_stride,
                    out.data_ptr() + back.first_row * width * item,
                    None if lse is None else lse_ptr + 4 * back.first_row * Hq, int(lse_base2))
            native.call_on(device, native.lib.va_attention_read_back_q8, q_ptr, q_stride, pool, back.slots.data_ptr(),
                           back.slots.numel(), plan.blob.data_ptr(), plan.header_ptr, plan.kv_indices.data_ptr(), *rows,
                           None if ws is None else ws.data_ptr(), 0 if ws is None else ws.numel(), scratch,
                           back.scratch.numel(), self._shape, rope, stream)
            plan = back.codes
            native.call_on(device, native.lib.va_attention_if_q8, scratch, q_ptr, q_stride, pool, plan.blob.data_ptr(),
                           plan.header_ptr, plan.kv_indices.data_ptr(), *rows, self._shape, rope, stream)
        return (out, lse) if return_lse else out

    # ------------------------------------------------------------------
    # moving tokens
    # ------------------------------------------------------------------
    def copy_shifted(self, source: torch.Tensor, target: torch.Tensor, position_shift: int = 0) -> None:
        """Copy the tokens of slots ``source`` to slots ``target`` (int64 on the device, each target once, none of
        them a source of another token) in every layer, keys rotated by ``position_shift`` and quantised anew; values,
        and keys where nothing rotates, move code for code.  A table with a factor turns no stored keys: refused."""
        for name, t in (("source", source), ("target", target)):
            native.require_device(t, name)
            if t.dim() != 1 or t.dtype != torch.int64 or t.device != self.device or t.numel() != source.numel():
                raise ValueError(f"{name} must be one row of {source.numel()} int64 slots on {self.device}, got {t.dtype} "
                                 f"{tuple(t.shape)} on {t.device}")
        if position_shift:
            self._check_turns()
        pool, source, target = self.kv_cache, source.contiguous(), target.contiguous()
        if pool.num_layers:
            native.call_on(self.device, native.lib.va_copy_shift_kv_q8, pool.layer(0), pool.code_layer_bytes,
                           pool.scale_layer_bytes, pool.num_layers, source.data_ptr(), target.data_ptr(), source.numel(),
                           int(position_shift), self._shape, self._rope_descriptor() if position_shift else None,
                           native.current_stream_ptr(self.device))
