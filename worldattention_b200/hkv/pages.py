"""Moves of cache pages in place: copying, forking, moving together, clearing.

The reference rolls its window through a clone of what it keeps (wan/modules/causal_model.py:331-360); here all tensors of a
call are rearranged by one launch, without scratch memory.
"""
from __future__ import annotations

from .. import _lib

__all__ = ["move_pages"]


def move_pages(caches, destination, source, page_tokens) -> None:
    """Page `destination[i]` becomes what page `source[i]` was, or zeros where that is None, for all i at once, in every cache.

    `caches`: CUDA tensors `[B, tokens, ...]` of any type (keys and values of any number of layers), changed in place; what lies
    behind the token axis must be contiguous, and no two of them may share memory.  A page is `page_tokens` consecutive
    tokens (a sequence: a length for each cache), page i of a cache begins at token `i * page_tokens`; the last one may be shorter, and a
    move between a whole and a shorter page moves the tokens that both have.  `destination` and `source` are page numbers on the
    host.  A page may be the source of several moves (a fork) and also a destination (a roll, a ring): every move
    reads what was there before the call.  A page can be the destination of one move only.

    Pages that are no destination keep their contents.  Nothing is copied to the device and nothing waits: the call can be captured
    into a CUDA graph, which then repeats these page numbers.
    """
    _lib.host().move_pages(caches, destination, source, page_tokens)
