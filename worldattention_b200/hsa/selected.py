"""Attention over selected key blocks with its gradient, for training and for single tokens.

`selected_attention` is the differentiable form of the sparse branch: what `build_block_routing` (or any other choice of blocks)
selected is attended to, `[B, L, H, D]` tensors are read in place, heads may share keys, and the gradient reaches q, k and v as the
reference's Triton autograd function does (wan/modules/hsa/block_sparse_triton.py:142-382).
"""
from __future__ import annotations

import torch

from .. import _lib

__all__ = ["selected_attention"]


def selected_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, index: torch.Tensor, num: torch.Tensor, block_size: int, *,
                       block_sizes: torch.Tensor | None = None, return_lse: bool = False):
    """Softmax attention of each query block over the key blocks listed for it -> `[B, Lq, H, D]`; differentiable in q, k and v.

    `q` `[B, Lq, H, D]`, `k` and `v` `[B, Lkv, Hkv, D]`, one dtype (float32 or bfloat16); H is a multiple of Hkv, and query head h reads key
    head `h // (H // Hkv)`.  Any strides with a contiguous last axis are read in place.  `index` `[B, H, Nq, S]` and `num` `[B, H, Nq]` (int32,
    `Nq = ceil(Lq / block_size)`) are the lists, as `build_block_routing` gives them: the first `num` ids of a row.  Lists are taken
    as sets: an id named twice counts once, an id that is no key block counts nothing.  Rows whose list is empty give zeros (and
    -inf as log-sum-exp) and have no part in the gradients.  `block_sizes` (int32 `[Nkv]`): only the first so many
    tokens of a block are keys, as in `block_sparse_attention`; what lies behind them is not read, and its gradients are zero.

    A NaN, or an infinite score, in what a row attends to shows in the row's result and normaliser and in the gradients that depend on it.

    The tensor cores (tcgen05) take bf16 with head_dim 128 and blocks of 64 or 128 without `block_sizes`, 16-byte aligned rows and positive strides between
    tokens and heads; other calls, key heads expanded with a stride of 0 among them, run on float32 multiply-adds, which take many times as long.

    `return_lse`: also the natural-log normalisers, float32 `[B, H, Lq]` (not differentiable).  Sums and statistics are float32; in bf16 the
    probabilities and dS are rounded to bf16 where they are factors of a product.  Equal calls give equal bits, gradients included.  The
    gradient of the gradient is not offered, nor are forward-mode derivatives.  A step can be captured into a CUDA graph, its backward pass included, unless
    an eager graph of the same leaves from the default stream is still alive (refused).
    """
    out, lse = _lib.host().selected_attention(q, k, v, index, num, block_size, block_sizes, False)
    return (out, lse) if return_lse else out
