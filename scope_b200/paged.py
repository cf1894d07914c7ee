"""Operators of a paged key-value cache: page tables and slot maps from request lengths, rotary positions with
several axes, the append of rotated keys and values into pages, and the decode attention that reads them.

The reference reserves one row of ``max_seq`` tokens for every request (``InplaceKVCache``,
system/qwenoffload.py:59-141); a paged pool bounds the requests' summed length instead.  A pool is a pair of tensors
``k_pages [n_pages, page_size, Hkv, Dk]`` and ``v_pages [n_pages, page_size, Hkv, Dv]`` (any strides of whole 16 bytes
with unit stride on the head dim, so a head-major ``[n_pages, Hkv, page_size, D]`` buffer is passed as its
``transpose(1, 2)``) in bf16, fp16, or int8 with one fp32 scale per row (``k_scales``, ``v_scales``
``[n_pages, page_size, Hkv]``).  ``scope_b200.kv_cache.PagedKVCache`` holds the pools of a model's layers and the
requests' tables.

The operators are outside autograd: inputs that require gradients are read as they are, and results require none
(``rope`` with ``inverse`` is the rotation's gradient, for a caller's own ``torch.autograd.Function``).

A step's calls, all asynchronous on the current stream and free of host synchronisation, so they can be captured in a
CUDA graph (graphs captured on one stream share its workspace: replay them one after the other, and not beside launches
on that stream):

    step = paged_slots(seq_lens, new_lens, page_table, free_pages, ring, page_size, n_tokens)
    q = rope_append(q, k, v, step.positions, cos_sin, step.slots, k_pages, v_pages)       # per layer
    out, lse = paged_decode(q_last, k_pages, v_pages, page_table, step.seq_lens, scale)    # per layer
    seq_lens, ring = paged_release(step.seq_lens, done, page_table, free_pages, step.ring, page_size)
"""
from __future__ import annotations

import functools
from typing import NamedTuple, Sequence

import torch

from . import _lib

_c = None   # the compiled binding, once loaded


def _load():
    global _c
    _c = _lib.binding()
    return _c


class PagedStep(NamedTuple):
    """What ``paged_slots`` gives: the step's tokens are packed, request b's at rows [cu_new[b], cu_new[b+1])."""
    slots: torch.Tensor       # int64 [n_tokens]: page * page_size + offset, -1 for a token without a place
    positions: torch.Tensor   # int32 [n_tokens]: the token's place in its request
    cu_new: torch.Tensor      # int32 [B+1]
    seq_lens: torch.Tensor    # int32 [B], the lengths after the step
    ring: torch.Tensor        # int32 [3]: head, free pages, requests refused


def paged_slots(seq_lens: torch.Tensor, new_lens: torch.Tensor, page_table: torch.Tensor, free_pages: torch.Tensor,
                ring: torch.Tensor, page_size: int, n_tokens: int, *, seq_lens_out: torch.Tensor | None = None,
                ring_out: torch.Tensor | None = None) -> PagedStep:
    """One step's pages and slots, in one launch.

    seq_lens, new_lens int32 [B]: the tokens each request holds and adds.  page_table int32 [B, pages]: request b's
    pages in order; the pages it lacks for its new tokens are taken, in request order, from the ring of free pages
    (free_pages int32 [n], ring int32 [3]: head, free count, refused) and written into its row.  ``n_tokens`` is the
    number of rows the packed step has room for (the host's sum of new_lens, or any bound of it: rows past the last
    token get slot -1).

    A request is refused whole -- its length, row and the ring unchanged, its tokens' slots -1 -- when its pages would
    pass the table's width, its tokens would pass n_tokens, or the pages it lacks, added to those that the requests before
    it lack, are more than are free.  Requests are served in order: those refused for want of pages count against all
    later ones, so behind one that does not fit no later request gets a page in this step, even while some are free.
    ``ring[2]`` counts the refused; which they are shows in the lengths that did not grow.  Refused tokens have no place:
    the caller repeats them, or admits only what fits.
    ``seq_lens_out`` / ``ring_out`` may be the inputs, which a captured step wants, and share no memory with the others.
    """
    return (_c or _load()).paged_slots(seq_lens, new_lens, page_table, free_pages, ring, page_size, n_tokens, seq_lens_out,
                                       ring_out)


def paged_release(seq_lens: torch.Tensor, done: torch.Tensor, page_table: torch.Tensor, free_pages: torch.Tensor,
                  ring: torch.Tensor, page_size: int, *, seq_lens_out: torch.Tensor | None = None,
                  ring_out: torch.Tensor | None = None):
    """Give finished requests' pages back to the ring: done bool [B].  Returns (seq_lens, ring), the finished
    requests' lengths 0; the outputs may be the inputs.  One launch."""
    return (_c or _load()).paged_release(seq_lens, done, page_table, free_pages, ring, page_size, seq_lens_out, ring_out)


# ------------------------------------------------------------------ rotary positions


@functools.lru_cache(maxsize=256)
def rope_axis_map(rope_dim: int, sections: tuple[int, ...] | None, cyclic: bool) -> bytes:
    """The axis of each of the rope_dim / 2 pairs, two bits each.

    ``sections`` gives each axis its number of pairs (None: one axis takes all), either in blocks -- the first
    sections[0] pairs turn by axis 0, and so on -- or ``cyclic``: pair i turns by axis i % A as long as that axis has
    pairs left, else by axis 0.
    """
    n = rope_dim // 2
    if sections is None:
        axes = [0] * n
    else:
        A = len(sections)
        if not 1 <= A <= 4 or any(s < 0 for s in sections) or sum(sections) != n:
            raise RuntimeError("rope: sections must give one to four axes rope_dim / 2 pairs in all")
        if cyclic:
            axes = [i % A if i // A < sections[i % A] else 0 for i in range(n)]
            if any(axes.count(a) != s for a, s in enumerate(sections)):
                raise RuntimeError("rope: with cyclic axes only axis 0 may take more pairs than the others can reach")
        else:
            axes = [a for a, s in enumerate(sections) for _ in range(s)]
    words = [0] * 8
    for i, a in enumerate(axes[:128]):
        words[i >> 4] |= a << (2 * (i & 15))
    return b"".join(w.to_bytes(4, "little") for w in words)


def _axes(cos_sin, sections, cyclic):
    """(axis map, number of axes) for the binding: (None, 1) where one axis takes all pairs."""
    if sections is None:
        return None, 1
    sections = tuple(sections)
    return rope_axis_map(cos_sin.shape[-1], sections, bool(cyclic)), len(sections)


def rope(x: torch.Tensor, positions: torch.Tensor, cos_sin: torch.Tensor, *, sections: Sequence[int] | None = None,
         cyclic: bool = False, pairs: str = "half", inverse: bool = False, out: torch.Tensor | None = None):
    """Rotate the first ``rope_dim`` dims of x [N, heads, D] (bf16 or fp16, any strides) by the tokens' positions.

    cos_sin fp32 [max_pos, rope_dim]: the cosines of a position's rope_dim / 2 pairs, then the sines.  ``pairs``:
    'half' pairs dims (i, rope_dim/2 + i), 'adjacent' dims (2i, 2i+1).  positions int32 / int64 [N], or [A, N] with
    ``sections`` (the pairs of each of A <= 4 axes, see ``rope_axis_map``): time, height and width of images and
    video.  ``inverse`` turns back, which is also the gradient.  ``out`` may be x, whole.  Products and sums are rounded to
    fp32 one by one and the result once more to x's type.
    """
    axis_map, axes = _axes(cos_sin, sections, cyclic)
    return (_c or _load()).rope(x, positions, cos_sin, axis_map, axes, pairs, inverse, out)


# ------------------------------------------------------------------ the pool


def rope_append(q: torch.Tensor | None, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor | None,
                cos_sin: torch.Tensor | None, slots: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, *,
                k_scales: torch.Tensor | None = None, v_scales: torch.Tensor | None = None,
                sections: Sequence[int] | None = None, cyclic: bool = False, pairs: str = "half",
                q_out: torch.Tensor | None = None):
    """Rotate a step's queries and keys and write its keys and values into the pool, in one launch.

    q [N, H, Dk] (or None), k [N, Hkv, Dk], v [N, Hkv, Dv]: bf16 or fp16, any strides with a unit head dim (views of a
    packed projection are read in place).  slots int64 [N] (``PagedStep.slots``): token t's key and value rows go to
    slot slots[t]; a negative slot drops them.  An int8 pool gets codes and one scale per row, taken from the rotated
    row in fp32 (the rule of ``kv_quantize_bf16_to_int8``); a NaN in a row makes the row's scale NaN, an infinity makes it
    infinite over codes of 0, so either row reads back as NaN.  ``cos_sin`` None: no rotation.  Rotary arguments as in
    ``rope``.  Returns the rotated queries (``q_out``, which may be q), or None without q.
    """
    axis_map, axes = (None, 1) if cos_sin is None else _axes(cos_sin, sections, cyclic)
    return (_c or _load()).rope_append(q, k, v, positions, cos_sin, slots, k_pages, v_pages, k_scales, v_scales, axis_map,
                                       axes, pairs, q_out)


def paged_decode(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
                 seq_lens: torch.Tensor, scale: float, *, window: int = 0, k_scales: torch.Tensor | None = None,
                 v_scales: torch.Tensor | None = None, out: torch.Tensor | None = None,
                 lse: torch.Tensor | None = None):
    """Attention of one new token per request over a paged cache.

    q [B, H, Dk] bf16 or fp16 with H = Hkv * G (head h = kvh * G + g; any strides of whole 16 bytes); the pool holds
    q's type or int8.  page_table int32 [B, pages]; seq_lens int32 [B]: request b attends its first seq_lens[b] tokens
    (the new one included), with ``window`` > 0 the last ``window`` of them.  Returns (out [B, H, Dv] in q's type,
    normalised; lse fp32 [B, H]).  A request without tokens gives out = 0, lse = -inf.  What pages hold past a
    request's length is never used.  A page id outside the pool leaves its tokens out and is reported by
    ``scope_b200.status_take``.  How rows are fetched follows the table's width, as the lengths stay on the device: for
    requests known to be of 512 tokens or less, their part ``page_table[:, :n]`` is the faster argument.
    """
    return (_c or _load()).paged_decode(q, k_pages, v_pages, page_table, seq_lens, scale, window, k_scales, v_scales, out,
                                        lse)
