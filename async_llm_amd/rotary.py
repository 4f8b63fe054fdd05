"""Rotary positions for queries and keys as a layer makes them, on the GPU.

The counterpart of the reference's ``RotaryEmbedding`` (``python/minisgl/layers/rotary.py:12-119``):
the layers of batches without a cache view rotate q and k before the attention backend
sees them, and models with a view need the ``cos|sin`` table that ``SharedCacheAttention``
takes.  Both come from one set of frequencies here: unscaled, or stretched for contexts
longer than a model was trained on.

    f_i = base ** (-2 i / rotary_dim)
    linear   f_i / factor
    llama3   f_i / factor where a wave is longer than original / low_freq_factor positions, f_i where it is
             shorter than original / high_freq_factor, a blend in between
    yarn     f_i where a pair makes beta_fast turns and more within the original length, f_i / factor where it
             makes beta_slow and fewer, a ramp over the pairs in between; cosines and sines times a factor

Frequencies, and products of position and frequency, are 64-bit numbers: positions up to about 2^27 are
as exact as near ones (farther angles lose 2^-52 of themselves), and none is past the end of a table.
(A table of 32-bit products is off by up to position * 2^-24 in each angle.)
"""

from __future__ import annotations

import math
from typing import Optional, Tuple

import torch

from . import native


def _frequencies(rotary_dim: int, base: float, scaling: Optional[dict]) -> Tuple[list, float]:
    """Frequencies of the pairs, and the factor on cosines and sines."""
    plain = [base ** (-2.0 * i / rotary_dim) for i in range(rotary_dim // 2)]
    if scaling is None:
        return plain, 1.0
    given = dict(scaling)
    kind = given.pop("rope_type", given.pop("type", None))

    def take(name, default=None):
        value = given.pop(name, default)
        if isinstance(value, bool) or not isinstance(value, (int, float)) or not math.isfinite(value) or value <= 0:
            raise ValueError(f"scaling {kind!r} needs {name} > 0, got {value!r}")
        return float(value)

    factor, attention = 1.0, 1.0
    if kind == "default":
        out = plain
    elif kind == "linear":
        factor = take("factor")
        out = [f / factor for f in plain]
    elif kind == "llama3":
        factor, low, high = take("factor"), take("low_freq_factor"), take("high_freq_factor")
        original = take("original_max_position_embeddings")
        if high <= low:
            raise ValueError(f"scaling 'llama3' needs low_freq_factor < high_freq_factor, got {low} and {high}")
        out = []
        for f in plain:
            turns = original * f / (2 * math.pi)
            share = min(1.0, max(0.0, (turns - low) / (high - low)))
            out.append(share * f + (1 - share) * f / factor)
    elif kind == "yarn":
        factor, original = take("factor"), take("original_max_position_embeddings")
        fast, slow = take("beta_fast", 32.0), take("beta_slow", 1.0)
        attention = take("attention_factor", 0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0)
        if base == 1.0 or fast < slow:
            raise ValueError(f"scaling 'yarn' needs base != 1 and beta_slow <= beta_fast, got {base}, {slow} and {fast}")

        def pair_of(turns):
            return rotary_dim * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base))

        first, last = max(math.floor(pair_of(fast)), 0), min(math.ceil(pair_of(slow)), rotary_dim - 1)
        width = max(last - first, 0.001)
        out = []
        for i, f in enumerate(plain):
            share = min(1.0, max(0.0, (i - first) / width))
            out.append((1 - share) * f + share * f / factor)
    else:
        raise ValueError(f"scaling must be of rope_type 'default', 'linear', 'llama3' or 'yarn', got {kind!r}")
    if given:
        raise ValueError(f"scaling {kind!r} does not know {sorted(given)}")
    return out, attention


def _apart(x: torch.Tensor, y: torch.Tensor, n: int) -> bool:
    """Whether ``n`` rows of ``x`` and of ``y``, contiguous each, share no element: one behind the other, or side by side."""
    if n == 0 or x.numel() == 0 or y.numel() == 0 or x.untyped_storage().data_ptr() != y.untyped_storage().data_ptr():
        return True
    step = x.element_size()
    (a, wide_a, row_a), (b, wide_b, row_b) = sorted(
        (t.data_ptr(), t[0].numel() * step, t.stride(0) * step) for t in (x, y))
    if a + (n - 1) * max(row_a, 0) + wide_a <= b:
        return True
    at = (b - a) % row_a if n > 1 and row_a == row_b and row_a > 0 else 0
    return wide_a <= at <= row_a - wide_b


class RotaryEmbedding:
    """Rotates heads of ``head_dim`` elements, the first ``rotary_dim`` of them (all by default), as pairs ``(i, i +
    rotary_dim / 2)`` or, ``interleaved``, ``(2 i, 2 i + 1)``.  ``scaling``: a dictionary as model configurations have it
    (``rope_type``, ``factor``, ...)."""

    def __init__(self, head_dim: int, rotary_dim: Optional[int] = None, base: float = 10000.0, interleaved: bool = False,
                 scaling: Optional[dict] = None, device="cuda") -> None:
        rotary_dim = head_dim if rotary_dim is None else rotary_dim
        if head_dim <= 0 or head_dim % 2 or rotary_dim <= 0 or rotary_dim % 2 or rotary_dim > min(head_dim, 2048):
            raise ValueError(f"rotary_dim {rotary_dim} must be even, positive and within head_dim {head_dim} (at most 2048)")
        if not base > 0:
            raise ValueError(f"base must be positive, got {base}")
        self.head_dim, self.rotary_dim, self.interleaved = head_dim, rotary_dim, bool(interleaved)
        frequencies, self.attention_factor = _frequencies(rotary_dim, float(base), scaling)
        device = torch.device(device)
        if device.type == "cuda" and device.index is None:
            device = torch.device("cuda", torch.cuda.current_device())
        self.device = device
        self.inv_freq = torch.tensor(frequencies, dtype=torch.float64, device=device)
        self._quarters = self.inv_freq / (0.5 * math.pi)
        self._turns = native.VaTurns(rotary_dim, int(self.interleaved), self.attention_factor, self._quarters.data_ptr())

    def _rows(self, x: torch.Tensor, n: int, name: str):
        """``x`` as ``n`` rows of whole heads, how far apart they are, and how many heads that is."""
        shape, dim = x.shape, self.head_dim
        if len(shape) == 2 and shape[1] % dim == 0:
            heads = shape[1] // dim
            row, element = x.stride()
            if element != 1:
                x, row = x.contiguous(), heads * dim
        elif len(shape) == 3 and shape[2] == dim:
            heads = shape[1]
            row, head, element = x.stride()
            if element != 1 or (heads > 1 and head != dim):
                x, row = x.contiguous(), heads * dim
        else:
            raise ValueError(f"{name} must be rows of heads of {dim} elements, got {tuple(shape)}")
        if shape[0] != n or x.device != self.device:
            native.require_device(x, name)
            raise ValueError(f"{name} must be {n} rows on {self.device}, got {tuple(shape)} on {x.device}")
        return x, row, heads

    def __call__(self, positions: torch.Tensor, q: torch.Tensor, k: Optional[torch.Tensor] = None,
                 out: Optional[tuple] = None):
        """``q`` and ``k`` (``[n, heads * head_dim]`` or ``[n, heads, head_dim]``, rows may lie apart) rotated by
        ``positions [n]`` (int64 or int32): new contiguous tensors, or ``out``, a pair that may be ``(q, k)`` themselves.
        ``k`` may be ``None``."""
        device, n, wide = self.device, q.shape[0], positions.dtype is torch.int64
        if not q.is_cuda:
            native.require_device(q, "q")
        if positions.dim() != 1 or not (wide or positions.dtype is torch.int32) or positions.device != device \
                or positions.shape[0] != n:
            raise ValueError(f"positions must be {n} int64 or int32 numbers on {device}, got {positions.dtype} "
                             f"{tuple(positions.shape)} on {positions.device}")
        dtype = q.dtype
        if k is not None and k.dtype is not dtype:
            raise ValueError(f"q and k must be of one type, got {dtype} and {k.dtype}")
        dtype_id = native.dtype_id(dtype)
        q2, q_row, q_heads = self._rows(q, n, "q")
        dim = self.head_dim
        if out is None:
            out_q, out_k = torch.empty_like(q, memory_format=torch.contiguous_format), None
            keys = (None, 0, 0, None, 0)
            if k is not None:
                k2, k_row, k_heads = self._rows(k, n, "k")
                out_k = torch.empty_like(k, memory_format=torch.contiguous_format)
                keys = (k2.data_ptr(), k_row, k_heads, out_k.data_ptr(), k_heads * dim)
            queries = (q2.data_ptr(), q_row, q_heads, out_q.data_ptr(), q_heads * dim)
        else:
            out_q, out_k = out
            queries = (q2.data_ptr(), q_row, q_heads, *self._out(out_q, q, q2, n, "out[0]"))
            keys = (None, 0, 0, None, 0)
            if k is not None:
                k2, k_row, k_heads = self._rows(k, n, "k")
                keys = (k2.data_ptr(), k_row, k_heads, *self._out(out_k, k, k2, n, "out[1]"))
                if not (_apart(out_q, k2, n) and _apart(out_k, q2, n) and _apart(out_q, out_k, n)):
                    raise ValueError("what becomes of q must lie apart from k, and from what becomes of k, and the other way round")
        positions = positions.contiguous()
        native.call_on(device, native.lib.va_rotate_qk, *queries, *keys, positions.data_ptr(), int(wide), n, dim, dtype_id,
                       self._turns, native.current_stream_ptr(device))
        return out_q, out_k

    def _out(self, y, x, rows, n: int, name: str):
        """Where the results of ``x`` go, ``y``, and how far apart its rows are; ``rows``: what is read of ``x``."""
        if not isinstance(y, torch.Tensor) or y.shape != x.shape or y.dtype != x.dtype or y.device != self.device:
            raise ValueError(f"{name} must be a {x.dtype} tensor {tuple(x.shape)} on {self.device}")
        width, stride = x[:1].numel(), y.stride()
        inner = stride[1:] == (1,) if len(stride) == 2 else stride[2] == 1 and (y.shape[1] <= 1 or stride[1] == self.head_dim)
        if not inner or (n > 1 and stride[0] < width):
            raise ValueError(f"{name} must have contiguous rows that do not overlap")
        # results over the input row by row, or apart from it
        same = y.data_ptr() == rows.data_ptr() and (n == 1 or stride[0] == rows.stride(0))
        if not same and not _apart(y, rows, n):
            raise ValueError(f"{name} must be the input itself or lie apart from it")
        return y.data_ptr(), stride[0] if n > 1 else width

    def cos_sin_cache(self, max_position: int, unit: bool = False) -> torch.Tensor:
        """The fp32 ``[max_position, rotary_dim]`` table of cosines and sines that ``SharedCacheAttention`` takes.  Its keys and
        queries are pairs ``(i, i + rotary_dim / 2)``: an interleaved rotation has no such table.  ``unit``: without
        ``attention_factor``, for caches whose keys are turned again when blocks are merged or tokens move, which would grow by it
        each time.  The factor belongs to what rotates, on both sides: the first ``rotary_dim`` elements of every query head are
        then to be multiplied by its square before attention, those that pass through are not."""
        if self.interleaved:
            raise ValueError("the table's pairs are halves of a head: an interleaved rotation is applied to q and k only")
        if max_position <= 0:
            raise ValueError(f"max_position must be positive, got {max_position}")
        table = torch.empty((max_position, self.rotary_dim), dtype=torch.float32, device=self.device)
        native.require_device(table, "the table")
        turns = native.VaTurns(self.rotary_dim, 0, 1.0, self._quarters.data_ptr()) if unit else self._turns
        native.call_on(self.device, native.lib.va_rotary_table, turns, 0, max_position, table.data_ptr(),
                       native.current_stream_ptr(self.device))
        return table
