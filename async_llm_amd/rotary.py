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

Frequencies, and products of position and frequency, are 64-bit numbers: far positions are as exact
as near ones, and none is past the end of a table.  (A table of 32-bit products is off by up to
position * 2^-24 in each angle.)
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
        """``x`` as ``n`` rows of whole heads, and how many heads that is."""
        if x.dim() == 3 and x.shape[2] == self.head_dim:
            heads = x.shape[1]
            if x.stride(2) != 1 or (heads > 1 and x.stride(1) != self.head_dim):
                x = x.contiguous()
        elif x.dim() == 2 and x.shape[1] % self.head_dim == 0:
            heads = x.shape[1] // self.head_dim
            if x.stride(1) != 1:
                x = x.contiguous()
        else:
            raise ValueError(f"{name} must be rows of heads of {self.head_dim} elements, got {tuple(x.shape)}")
        if x.shape[0] != n or x.device != self.device:
            raise ValueError(f"{name} must be {n} rows on {self.device}, got {tuple(x.shape)} on {x.device}")
        return x, heads

    def __call__(self, positions: torch.Tensor, q: torch.Tensor, k: Optional[torch.Tensor] = None,
                 out: Optional[tuple] = None):
        """``q`` and ``k`` (``[n, heads * head_dim]`` or ``[n, heads, head_dim]``, rows may lie apart) rotated by
        ``positions [n]`` (int64 or int32): new contiguous tensors, or ``out``, a pair that may be ``(q, k)`` themselves.
        ``k`` may be ``None``."""
        native.require_device(q, "q")
        device, n = self.device, q.shape[0]
        if positions.dim() != 1 or positions.dtype not in (torch.int64, torch.int32) or positions.device != device \
                or positions.shape[0] != n:
            raise ValueError(f"positions must be {n} int64 or int32 numbers on {device}, got {positions.dtype} "
                             f"{tuple(positions.shape)} on {positions.device}")
        if k is not None and k.dtype != q.dtype:
            raise ValueError(f"q and k must be of one type, got {q.dtype} and {k.dtype}")
        dtype = native.dtype_id(q.dtype)
        q2, q_heads = self._rows(q, n, "q")
        k2, k_heads = (None, 0) if k is None else self._rows(k, n, "k")
        if out is None:
            out_q = torch.empty(q.shape, dtype=q.dtype, device=device)
            out_k = None if k is None else torch.empty(k.shape, dtype=k.dtype, device=device)
            q_out, k_out = out_q, out_k
        else:
            out_q, out_k = out
            q_out = self._out(out_q, q, n, "out[0]")
            k_out = None if k is None else self._out(out_k, k, n, "out[1]")
        positions = positions.contiguous()
        none = (None, 0, 0, None, 0)
        native.call_on(
            device, native.lib.va_rotate_qk, q2.data_ptr(), q2.stride(0), q_heads, q_out.data_ptr(), q_out.stride(0),
            *(none if k is None else (k2.data_ptr(), k2.stride(0), k_heads, k_out.data_ptr(), k_out.stride(0))),
            positions.data_ptr(), int(positions.dtype is torch.int64), n, self.head_dim, dtype, self._turns,
            native.current_stream_ptr(device))
        return out_q, out_k

    def _out(self, y, x, n: int, name: str) -> torch.Tensor:
        if not isinstance(y, torch.Tensor) or y.shape != x.shape or y.dtype != x.dtype or y.device != self.device:
            raise ValueError(f"{name} must be a {x.dtype} tensor {tuple(x.shape)} on {self.device}")
        inner = y.stride()[1:]
        if inner != ((1,) if y.dim() == 2 else (self.head_dim, 1)) or (n > 1 and y.stride(0) < x[0].numel()):
            raise ValueError(f"{name} must have contiguous rows that do not overlap")
        return y

    def cos_sin_cache(self, max_position: int) -> torch.Tensor:
        """The fp32 ``[max_position, rotary_dim]`` table of cosines and sines that ``SharedCacheAttention`` takes.  Its keys and
        queries are pairs ``(i, i + rotary_dim / 2)``: an interleaved rotation has no such table."""
        if self.interleaved:
            raise ValueError("the table's pairs are halves of a head: an interleaved rotation is applied to q and k only")
        if max_position <= 0:
            raise ValueError(f"max_position must be positive, got {max_position}")
        table = torch.empty((max_position, self.rotary_dim), dtype=torch.float32, device=self.device)
        native.require_device(table, "the table")
        native.call_on(self.device, native.lib.va_rotary_table, self._turns, 0, max_position, table.data_ptr(),
                       native.current_stream_ptr(self.device))
        return table
