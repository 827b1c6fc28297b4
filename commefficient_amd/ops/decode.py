"""Generation from a paged key-value cache: the operators of one answering step.

A cache holds the keys and values of ``layers`` layers in pages of ``page_size``
tokens, ``kv`` [layers, 2, pages, kv heads, page size, head dim]; a block table
(int32 [sequences, width]) names every sequence's pages in order and ``lens``
(int32 [sequences]) counts its tokens.  Slot ``s`` is token ``s % page_size`` of
page ``s // page_size``.  One step of a batch runs, without the host looking at
a length:

    kv_extend        the step's pages, slots and positions from the lengths
    paged_attention  per layer: the new token's row stored and attended in one launch
                     (prompts: kv_write stores their rows)
    beam_select      the best continuations of every request's beams
    beam_reorder     tables and part-filled pages follow the surviving beams

HIP kernels in csrc/kvcache.hip, paged_attention.hip and beam.hip, plain loops
for CPU tensors in csrc/decode_ops.cpp; both check their arguments alike (but for
the alignment that a kernel needs) and raise RuntimeError.  The operators run on
the current stream of their tensors' device, allocate their outputs and workspaces
per call and read nothing back, so a step can be captured into a graph.  None of
them has a gradient.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Tuple

import torch

from .._ext import ops as _ops

__all__ = ["KVExtend", "PagedKV", "beam_reorder", "beam_select", "kv_extend", "kv_write",
           "paged_attention"]


class KVExtend(NamedTuple):
    """What ``kv_extend`` says of the new tokens' rows (packed, sequence by sequence)."""
    slots: torch.Tensor   # int64 [rows]: where the row's key and value go, -1: nowhere
    pos: torch.Tensor     # int32 [rows]: its position in its sequence
    seq: torch.Tensor     # int32 [rows]: its sequence, -1 behind the last one
    start: torch.Tensor   # int32 [sequences + 1]: every sequence's first row
    lens: torch.Tensor    # int32 [sequences]: the lengths with the new tokens
    used: torch.Tensor    # int32 [1]: pages taken from the pool
    missed: torch.Tensor  # int32 [1]: sequences that were not extended


def kv_extend(table: torch.Tensor, lens: torch.Tensor, new: torch.Tensor, pool: torch.Tensor,
              used: torch.Tensor, page_size: int, rows: int, *, in_place: bool = False) -> KVExtend:
    """Room for ``new`` [sequences] more tokens of every sequence (all int32).

    Pages come from ``pool[used:]``, in the order of the sequences, and are
    entered into ``table``.  ``rows`` (host) is the number of packed rows that
    the new tokens take, or a bound on it: rows behind the last sequence get
    slot -1, position 0, sequence -1.  A sequence is left as it was -- its rows
    slot -1 and position 0 -- and counted in ``missed`` where its count is
    negative, its table row or ``rows`` too short for it, or the pool too small
    for it and the sequences before it.  ``in_place`` updates ``lens`` and
    ``used`` themselves (they are returned), else they are left alone."""
    r = _ops().kv_extend(table, lens, new, pool, used, page_size, rows, in_place)
    if in_place:
        return KVExtend(r[0], r[1], r[2], r[3], lens, used, r[4])
    return KVExtend(r[0], r[1], r[2], r[3], r[5], r[6], r[4])


def kv_write(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
             slots: torch.Tensor) -> None:
    """Rows k, v [rows, kv heads, head dim] into their slots (int64 [rows]) of one
    layer's caches [pages, kv heads, page size, head dim]; any row, head, page and
    slot strides that leave the caches' elements addresses of their own.  Slots
    outside the cache (-1) are skipped.  The slots of one call are distinct: a slot
    named twice ends with a mixture of its rows."""
    _ops().kv_write(k, v, k_cache, v_cache, slots)


def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, table: torch.Tensor,
                    lens: torch.Tensor, *, k: Optional[torch.Tensor] = None,
                    v: Optional[torch.Tensor] = None, scale: Optional[float] = None,
                    max_len: Optional[int] = None) -> torch.Tensor:
    """Attention of one token a sequence, q [sequences, heads, head dim], over its
    ``lens`` cached tokens: softmax(scale q k^T) v, scale head_dim^-0.5 by default.

    bfloat16, float16 or float32; head dim 32, 64, 128 or 256; ``heads`` a multiple
    of the cache's (head h reads cache head h // group).  With ``k``, ``v``
    [sequences, kv heads, head dim], the last of the ``lens`` tokens is the new one:
    its rows are read from there and stored into its slot by the same launch (a
    slot that no other sequence of the call reads or stores).  Rows of sequences
    without tokens, or with no score above -inf, are 0.  A row is NaN where the table
    names a page outside the cache (nothing is read through it) or is too short for
    ``lens``.  Caches as for ``kv_write``; on a GPU their pages, heads and slots start
    at multiples of 16 bytes.  An infinite value makes its column of the row infinite,
    and NaN where its weight is 0 in fp32 or the sum holds both infinities; finite
    values below 2^120 / tokens leave the sums finite.  ``max_len`` (host) is a hint of
    the longest sequence, for the split of the work alone."""
    return _ops().paged_attention(q, k_cache, v_cache, table, lens, k, v, scale, max_len)


def beam_select(logits: torch.Tensor, scores: torch.Tensor, keep: Optional[int] = None, *,
                finished: Optional[torch.Tensor] = None,
                eos: int = -1) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """The ``keep`` (default: beams, at most 64) best continuations of every request:
    (scores float32, parent beam int64, token int64), [requests, keep], best first.

    A continuation's score is scores[r, j] + log_softmax(logits[r, j])[v] (logits
    [requests, beams, vocabulary], any strides; scores float32), compared in 64
    bits; equal ones by the lower beam, then the lower token.  A ``finished`` beam
    (bool [requests, beams]) goes on with ``eos`` alone, at its own score.  A beam
    whose score is not finite, or whose logits hold NaN or +inf or nothing
    above -inf, has no continuations, a token at -inf is none: places that none
    is left for hold (-inf, 0, 0)."""
    return _ops().beam_select(logits, scores, logits.shape[1] if keep is None else keep, finished, eos)


def beam_reorder(parent: torch.Tensor, table: torch.Tensor, lens: torch.Tensor, kv: torch.Tensor) -> None:
    """Beam j of request r takes the history of its beam ``parent[r, j]`` (int64
    [requests, beams], at most 32 beams), in place: the ids of the parent's full
    pages, which both share from then on, and the content of the parent's
    part-filled page in every layer, copied into the page that beam j itself holds
    there.  ``table`` and ``lens`` list the beams request by request; ``kv`` [layers,
    2, pages, kv heads, page size, head dim].  The beams of a request have equal
    lengths and part-filled pages of their own; a beam whose length differs
    from its parent's, whose parent is none of the request's beams or whose
    page is outside the cache stays as it is.  Any strides as for ``kv_write``."""
    _ops().beam_reorder(parent, table, lens, kv)


class PagedKV:
    """Caches of all layers with their block tables, lengths and page pool.

    ``seqs`` sequences of at most ``max_tokens`` tokens out of ``pages`` pages; the
    tables start empty (-1).  Everything lives on ``device`` and changes in
    place, so that a captured step goes on where the last one stopped."""

    def __init__(self, layers: int, kv_heads: int, head_dim: int, seqs: int, pages: int,
                 page_size: int = 16, max_tokens: int = 1024, dtype=torch.bfloat16, device="cuda"):
        self.page_size, self.max_tokens = page_size, max_tokens
        self.kv = torch.empty(layers, 2, pages, kv_heads, page_size, head_dim, dtype=dtype, device=device)
        self.table = torch.full((seqs, -(-max_tokens // page_size)), -1, dtype=torch.int32, device=device)
        self.pool = torch.arange(pages, dtype=torch.int32, device=device)
        self.lens = torch.zeros(seqs, dtype=torch.int32, device=device)
        self.used = torch.zeros(1, dtype=torch.int32, device=device)
        self.missed = torch.zeros(1, dtype=torch.int32, device=device)
        self._layer = [(self.kv[i, 0], self.kv[i, 1]) for i in range(layers)]

    def reset(self) -> None:
        """Every sequence empty, every page back in the pool."""
        self.table.fill_(-1)
        self.lens.zero_()
        self.used.zero_()
        self.missed.zero_()

    def extend(self, new: torch.Tensor, rows: int) -> KVExtend:
        """``kv_extend`` of all sequences in place; ``self.missed`` adds up the calls'."""
        r = kv_extend(self.table, self.lens, new, self.pool, self.used, self.page_size, rows, in_place=True)
        self.missed.add_(r.missed)
        return r

    def write(self, layer: int, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
        kv_write(k, v, *self._layer[layer], slots)

    def attend(self, layer: int, q: torch.Tensor, k: Optional[torch.Tensor] = None,
               v: Optional[torch.Tensor] = None, *, scale: Optional[float] = None,
               max_len: Optional[int] = None) -> torch.Tensor:
        return paged_attention(q, *self._layer[layer], self.table, self.lens, k=k, v=v, scale=scale,
                               max_len=max_len)

    def reorder(self, parent: torch.Tensor) -> None:
        beam_reorder(parent, self.table, self.lens, self.kv)

    def share(self, beams: int) -> None:
        """Every request's other beams take the history of its first (their own is dropped)."""
        lens = self.lens.view(-1, beams)
        first = lens[:, :1].clone()
        new = (first % self.page_size).expand(-1, beams).contiguous()
        new[:, 0] = 0
        lens[:, 1:] = first // self.page_size * self.page_size
        # a page of their own for the part-filled one; the rows' slots are not needed
        self.extend(new.view(-1), lens.numel() * (self.page_size - 1))
        self.reorder(torch.zeros(lens.shape, dtype=torch.int64, device=lens.device))
