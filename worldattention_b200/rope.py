"""q/k RMSNorm and causal rotary embedding of the DiT self-attention on the GPU.

`causal_rope_apply` keeps the reference's signature (wan/modules/causal_model.py:34-62); `qk_norm_rope` fuses the
RMSNorm in front of it (wan/modules/model.py:70-86), which the reference applies to q and k just before.  One kernel
launch per tensor, no float64 copy of the tokens, no loop over samples.

`axial_rope` is the rotary embedding for tokens that have positions of their own (samples of different grids in one batch, text
between pictures, single tokens), for q and k in one launch, with its gradient.
"""
from __future__ import annotations

import torch

from . import _lib

__all__ = ["causal_rope_apply", "qk_norm_rope", "axial_rope"]


def _table(freqs: torch.Tensor, dev: torch.device) -> torch.Tensor:
    """The reference's complex table `[rows, D/2]` as float64 `[rows, D/2, 2]` on the device."""
    if torch.is_complex(freqs):
        freqs = torch.view_as_real(freqs.to(torch.complex128))
    return freqs.to(device=dev, dtype=torch.float64).contiguous()


def _grid(grid_sizes) -> tuple[int, int, int]:
    if type(grid_sizes) is tuple and len(grid_sizes) == 3 and all(type(v) is int for v in grid_sizes):
        return grid_sizes
    rows = grid_sizes.tolist() if hasattr(grid_sizes, "tolist") else list(grid_sizes)
    if rows and isinstance(rows[0], (list, tuple)):
        if any(tuple(r) != tuple(rows[0]) for r in rows):
            raise NotImplementedError("samples of one batch must share a (frames, height, width) grid")
        rows = rows[0]
    f, h, w = (int(v) for v in rows)
    return f, h, w


def qk_norm_rope(x: torch.Tensor, norm_weight: torch.Tensor | None, eps: float, grid_sizes, freqs: torch.Tensor | None,
                 start_frame=0, *, heads: int | None = None, table: torch.Tensor | None = None) -> torch.Tensor:
    """RMSNorm over the last axis of `[B, L, H*D]` (or `[B, L, H, D]`), then the causal rotary embedding -> `[B, L, H, D]`.

    `table` is `_table(freqs)` kept by the caller (saves the conversion per call).  `start_frame` may be an int32 device
    tensor of one element: the kernel then reads the position when it runs (for launches replayed from a CUDA graph)."""
    if x.dim() == 3:
        if heads is None:
            raise ValueError("heads is needed to split the last axis of a [B, L, H*D] tensor")
        x = x.view(x.shape[0], x.shape[1], heads, -1)
    h = w = 1
    if freqs is not None or table is not None:
        f, h, w = _grid(grid_sizes)
        if f * h * w != x.shape[1]:
            raise NotImplementedError(f"the grid {f}x{h}x{w} must cover all {x.shape[1]} tokens")
        if table is None:
            table = _table(freqs, _lib.require_cuda(x))
    return _lib.host().qk_norm_rope(x, norm_weight, eps, table, start_frame, h, w)


def causal_rope_apply(x: torch.Tensor, grid_sizes, freqs: torch.Tensor, start_frame: int = 0) -> torch.Tensor:
    """Rotary embedding of `[B, L, H, D]` tokens laid out as a (frames, height, width) grid that starts at `start_frame`."""
    return qk_norm_rope(x, None, 0.0, grid_sizes, freqs, start_frame)


def axial_rope(x, positions: torch.Tensor, table: torch.Tensor, *, axes=None, interleaved: bool = True):
    """Rotary embedding of `[B, L, H, D]` tokens at positions of their own on several axes; differentiable in `x`.

    `x` is a tensor, or a tuple of up to four that share B, L and D (q and k: one launch).  `positions` `[L, A]` or `[B, L, A]`
    holds each token's place on each of the A axes (int32; other integers are converted), `table` the angles: float32
    `[rows, pairs, 2]` cosines and sines, or a complex table `[rows, pairs]` as `causal_rope_apply` takes, which is converted
    in every call.  `axes` says how many consecutive pairs each axis turns (default: all of them for one axis, and for three
    the time, height and width bands of `causal_rope_apply`).  A pair is two neighbouring channels, or with `interleaved=False`
    channels i and i + pairs.  Channels behind `2 * pairs` are copied.  A token whose position on an axis lies outside the
    table gets NaN in the pairs of that axis (nothing is read back to the host to refuse it).  The table has no gradient; one that
    requires a gradient is refused.

    Float32 arithmetic, rounded once.  New tensors are returned, contiguous; a tuple for a tuple.
    """
    alone = isinstance(x, torch.Tensor)
    xs = (x,) if alone else tuple(x)
    if torch.is_complex(table):
        table = torch.view_as_real(table.resolve_conj())
    if table.dtype != torch.float32:
        table = table.float()
    if positions.dtype != torch.int32:
        if positions.dtype.is_floating_point or positions.dtype.is_complex or positions.dtype == torch.bool:
            raise ValueError(f"positions must be integers, got {positions.dtype}")
        # what lies outside the table stays outside; clamped in 64 bits, since the types of 8 and 16 bits cannot hold the bounds
        positions = positions.long().clamp(-1, min(table.shape[0], 2 ** 31 - 1)).int()
    if axes is None:
        pairs, n = table.shape[1], positions.shape[-1]
        if n not in (1, 3):
            raise ValueError(f"axes is needed for {n} axes: how many pairs does each of them turn?")
        axes = (pairs,) if n == 1 else (pairs - 2 * (pairs // 3), pairs // 3, pairs // 3)
    out = _lib.host().axial_rope(xs, positions, table, axes, bool(interleaved))
    return out[0] if alone else tuple(out)
