"""Operators of a paged key-value cache: page tables and slot maps from request lengths, rotary positions with
several axes, the append of rotated keys and values into pages, and the decode attention that reads them.

The reference reserves one row of ``max_seq`` tokens for every request (``InplaceKVCache``,
system/qwenoffload.py:59-141); a paged pool bounds the requests' summed length instead.  A pool is a pair of tensors
``k_pages [n_pages, page_size, Hkv, Dk]`` and ``v_pages [n_pages, page_size, Hkv, Dv]`` (any strides of whole 16 bytes
with unit stride on the head dim, so a head-major ``[n_pages, Hkv, page_size, D]`` buffer is passed as its
``transpose(1, 2)``) in bf16, fp16, or int8 with one fp32 scale per row (``k_scales``, ``v_scales``
``[n_pages, page_size, Hkv]``).  ``scope_b200.kv_cache.PagedKVCache`` holds the pools of a model's layers and the
requests' tables.

A step's calls, all asynchronous on the current stream and free of host synchronisation (so they can be captured in a
CUDA graph):

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
from ._lib import check, lib, on_device, paged_kv_pack, ptr, rope_pack, stream_ptr, workspaces

_HALF = {torch.bfloat16: _lib.WS_DTYPE_BF16, torch.float16: _lib.WS_DTYPE_F16}
_POOL = {**_HALF, torch.int8: _lib.WS_DTYPE_I8}
_I32 = torch.int32


class PagedStep(NamedTuple):
    """What ``paged_slots`` gives: the step's tokens are packed, request b's at rows [cu_new[b], cu_new[b+1])."""
    slots: torch.Tensor       # int64 [n_tokens]: page * page_size + offset, -1 for a token without a place
    positions: torch.Tensor   # int32 [n_tokens]: the token's place in its request
    cu_new: torch.Tensor      # int32 [B+1]
    seq_lens: torch.Tensor    # int32 [B], the lengths after the step
    ring: torch.Tensor        # int32 [3]: head, free pages, requests refused


def _want(what: str, name: str, t: torch.Tensor, dtype, dim: int, dev) -> None:
    if t.dtype != dtype or t.dim() != dim or t.device != dev or not t.is_contiguous():
        raise RuntimeError(f"{what}: {name} must be a contiguous {dtype} tensor of {dim} dimension(s) on {dev}")


def _table(what: str, t: torch.Tensor, B: int, dev) -> None:
    if t.dtype != _I32 or t.dim() != 2 or t.shape[0] != B or (t.numel() > 1 and t.stride(1) != 1) or t.device != dev:
        raise RuntimeError(f"{what}: page_table must be int32 [{B}, pages] on {dev} with unit stride on the pages")


def _bookkeeping(what, seq_lens, other, other_name, other_dtype, page_table, free_pages, ring):
    if not seq_lens.is_cuda:
        raise RuntimeError(f"{what}: CUDA tensors required (there is no CPU path)")
    dev, B = seq_lens.device, seq_lens.numel()
    _want(what, "seq_lens", seq_lens, _I32, 1, dev)
    _want(what, other_name, other, other_dtype, 1, dev)
    _table(what, page_table, B, dev)
    _want(what, "free_pages", free_pages, _I32, 1, dev)
    _want(what, "ring", ring, _I32, 1, dev)
    if other.numel() != B or ring.numel() != 3:
        raise RuntimeError(f"{what}: {other_name} must hold one entry per request, and ring three")
    return dev, B


def _out(what, name, t, n, dtype, dev):
    if t is None:
        return torch.empty(n, dtype=dtype, device=dev)
    _want(what, name, t, dtype, 1, dev)
    if t.numel() != n:
        raise RuntimeError(f"{what}: {name} must hold {n} entries")
    return t


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
    pass the table's width, its tokens would pass n_tokens, or too few pages are free; ``ring[2]`` counts them.
    ``seq_lens_out`` / ``ring_out`` may be the inputs, which a captured step wants.
    """
    dev, B = _bookkeeping("paged_slots", seq_lens, new_lens, "new_lens", _I32, page_table, free_pages, ring)
    seq_lens_out = _out("paged_slots", "seq_lens_out", seq_lens_out, B, _I32, dev)
    ring_out = _out("paged_slots", "ring_out", ring_out, 3, _I32, dev)
    slots = torch.empty(n_tokens, dtype=torch.int64, device=dev)
    positions = torch.empty(n_tokens, dtype=_I32, device=dev)
    cu_new = torch.empty(B + 1, dtype=_I32, device=dev)
    L_ = lib()
    with on_device(dev):
        ws = workspaces.get(L_.ws_paged_slots_workspace_size(), dev)
        rc = L_.ws_paged_slots(ptr(seq_lens), ptr(new_lens), B, ptr(page_table), page_table.stride(0),
                               page_table.shape[1], ptr(free_pages), free_pages.numel(), ptr(ring), page_size, n_tokens,
                               ptr(slots), ptr(positions), ptr(cu_new), ptr(seq_lens_out), ptr(ring_out), ptr(ws),
                               ws.numel(), stream_ptr(dev))
    check(rc, "ws_paged_slots")
    return PagedStep(slots, positions, cu_new, seq_lens_out, ring_out)


def paged_release(seq_lens: torch.Tensor, done: torch.Tensor, page_table: torch.Tensor, free_pages: torch.Tensor,
                  ring: torch.Tensor, page_size: int, *, seq_lens_out: torch.Tensor | None = None,
                  ring_out: torch.Tensor | None = None):
    """Give finished requests' pages back to the ring: done bool [B].  Returns (seq_lens, ring), the finished
    requests' lengths 0; the outputs may be the inputs.  One launch."""
    dev, B = _bookkeeping("paged_release", seq_lens, done, "done", torch.bool, page_table, free_pages, ring)
    seq_lens_out = _out("paged_release", "seq_lens_out", seq_lens_out, B, _I32, dev)
    ring_out = _out("paged_release", "ring_out", ring_out, 3, _I32, dev)
    L_ = lib()
    with on_device(dev):
        ws = workspaces.get(L_.ws_paged_slots_workspace_size(), dev)
        rc = L_.ws_paged_release(ptr(seq_lens), ptr(done), B, ptr(page_table), page_table.stride(0),
                                 page_table.shape[1], ptr(free_pages), free_pages.numel(), ptr(ring), page_size,
                                 ptr(seq_lens_out), ptr(ring_out), ptr(ws), ws.numel(), stream_ptr(dev))
    check(rc, "ws_paged_release")
    return seq_lens_out, ring_out


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


def _rope(what, positions, cos_sin, N, dev, sections, cyclic, pairs, inverse) -> bytes:
    if cos_sin.dtype != torch.float32 or cos_sin.dim() != 2 or not cos_sin.is_contiguous() or cos_sin.device != dev:
        raise RuntimeError(f"{what}: cos_sin must be contiguous fp32 [max_pos, rope_dim] on {dev}")
    if pairs not in ("half", "adjacent"):
        raise RuntimeError(f"{what}: pairs must be 'half' or 'adjacent'")
    top, rot = cos_sin.shape
    sections = None if sections is None else tuple(sections)
    axes = 1 if sections is None else len(sections)
    shape = positions.shape
    if positions.dtype not in (torch.int32, torch.int64) or positions.device != dev or \
            (shape != (axes, N) and (axes > 1 or shape != (N,))) or (N > 1 and positions.stride(-1) != 1):
        raise RuntimeError(f"{what}: positions must be int32 or int64 [{N}], or [{axes}, {N}], on {dev}, unit stride")
    return rope_pack(ptr(positions), ptr(cos_sin), positions.stride(0) if len(shape) == 2 else 0, top,
                     positions.dtype == torch.int64, axes, rot, pairs == "adjacent", inverse, 0,
                     rope_axis_map(rot, sections, bool(cyclic)))


def _rows(what, name, t, dtype, N, dev):
    if t.dtype != dtype or t.dim() != 3 or t.device != dev or t.shape[0] != N or (t.shape[2] > 1 and t.stride(2) != 1):
        raise RuntimeError(f"{what}: {name} must be {dtype} [{N}, heads, D] on {dev} with unit stride on the head dim")


def rope(x: torch.Tensor, positions: torch.Tensor, cos_sin: torch.Tensor, *, sections: Sequence[int] | None = None,
         cyclic: bool = False, pairs: str = "half", inverse: bool = False, out: torch.Tensor | None = None):
    """Rotate the first ``rope_dim`` dims of x [N, heads, D] (bf16 or fp16, any strides) by the tokens' positions.

    cos_sin fp32 [max_pos, rope_dim]: the cosines of a position's rope_dim / 2 pairs, then the sines.  ``pairs``:
    'half' pairs dims (i, rope_dim/2 + i), 'adjacent' dims (2i, 2i+1).  positions int32 / int64 [N], or [A, N] with
    ``sections`` (the pairs of each of A <= 4 axes, see ``rope_axis_map``): time, height and width of images and
    video.  ``inverse`` turns back, which is also the gradient.  ``out`` may be x.  Products and sums are rounded to
    fp32 one by one and the result once more to x's type.
    """
    if not x.is_cuda:
        raise RuntimeError("rope: CUDA tensors required (there is no CPU path)")
    dev, dt = x.device, x.dtype
    if dt not in _HALF:
        raise RuntimeError("rope: x must be bf16 or fp16")
    N = x.shape[0]
    _rows("rope", "x", x, dt, N, dev)
    r = _rope("rope", positions, cos_sin, N, dev, sections, cyclic, pairs, inverse)
    if out is None:
        out = torch.empty(x.shape, dtype=dt, device=dev)
    else:
        _rows("rope", "out", out, dt, N, dev)
        if out.shape != x.shape:
            raise RuntimeError("rope: out must have x's shape")
    with on_device(dev):
        rc = lib().ws_rope_append(r, ptr(x), x.stride(0), x.stride(1), x.shape[1], x.shape[2], ptr(out), out.stride(0),
                                  out.stride(1), None, 0, 0, None, 0, 0, _HALF[dt], N, None, None, stream_ptr(dev))
    check(rc, "ws_rope_append")
    return out


# ------------------------------------------------------------------ the pool


def _pool(what, k_pages, v_pages, k_scales, v_scales, dev):
    """(packed ws_paged_kv, Hkv, Dk, Dv, dtype) of a pool."""
    dt = k_pages.dtype
    if dt not in _POOL:
        raise RuntimeError(f"{what}: the pool must be bf16, fp16 or int8")
    ks, vs = k_pages.shape, v_pages.shape
    if len(ks) != 4 or len(vs) != 4 or ks[:3] != vs[:3] or v_pages.dtype != dt or k_pages.device != dev or \
            v_pages.device != dev:
        raise RuntimeError(f"{what}: k_pages, v_pages must be [n_pages, page_size, Hkv, D] of one type on {dev}")
    kst, vst = k_pages.stride(), v_pages.stride()
    if kst[3] != 1 or vst[3] != 1:
        raise RuntimeError(f"{what}: unit stride on the head dim required")
    sst = zst = (0, 0, 0)
    if dt == torch.int8:
        if k_scales is None or v_scales is None:
            raise RuntimeError(f"{what}: an int8 pool needs k_scales and v_scales")
        for s in (k_scales, v_scales):
            if s.dtype != torch.float32 or s.shape != ks[:3] or s.device != dev:
                raise RuntimeError(f"{what}: scales must be fp32 [n_pages, page_size, Hkv] on {dev}")
        sst, zst = k_scales.stride(), v_scales.stride()
    elif k_scales is not None or v_scales is not None:
        raise RuntimeError(f"{what}: scales belong to an int8 pool")
    packed = paged_kv_pack(ptr(k_pages), ptr(v_pages), ptr(k_scales) or 0, ptr(v_scales) or 0, ks[0], kst[0], kst[1],
                           kst[2], vst[0], vst[1], vst[2], *sst, *zst, ks[1], ks[2], ks[3], vs[3], _POOL[dt], 0)
    return packed, ks[2], ks[3], vs[3], dt


def rope_append(q: torch.Tensor | None, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor | None,
                cos_sin: torch.Tensor | None, slots: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, *,
                k_scales: torch.Tensor | None = None, v_scales: torch.Tensor | None = None,
                sections: Sequence[int] | None = None, cyclic: bool = False, pairs: str = "half",
                q_out: torch.Tensor | None = None):
    """Rotate a step's queries and keys and write its keys and values into the pool, in one launch.

    q [N, H, Dk] (or None), k [N, Hkv, Dk], v [N, Hkv, Dv]: bf16 or fp16, any strides with a unit head dim (views of a
    packed projection are read in place).  slots int64 [N] (``PagedStep.slots``): token t's key and value rows go to
    slot slots[t]; a negative slot drops them.  An int8 pool gets codes and one scale per row, taken from the rotated
    row in fp32 (the rule of ``kv_quantize_bf16_to_int8``).  ``cos_sin`` None: no rotation.  Rotary arguments as in
    ``rope``.  Returns the rotated queries (``q_out``, which may be q), or None without q.
    """
    if not k.is_cuda:
        raise RuntimeError("rope_append: CUDA tensors required (there is no CPU path)")
    dev, dt = k.device, k.dtype
    if dt not in _HALF:
        raise RuntimeError("rope_append: q, k, v must be bf16 or fp16")
    N = k.shape[0]
    _rows("rope_append", "k", k, dt, N, dev)
    _rows("rope_append", "v", v, dt, N, dev)
    pool, Hkv, Dk, Dv, pdt = _pool("rope_append", k_pages, v_pages, k_scales, v_scales, dev)
    if k.shape[1] != Hkv or v.shape[1] != Hkv or k.shape[2] != Dk or v.shape[2] != Dv:
        raise RuntimeError(f"rope_append: k, v must be [N, {Hkv}, {Dk}] and [N, {Hkv}, {Dv}] as the pool is")
    _want("rope_append", "slots", slots, torch.int64, 1, dev)
    if slots.numel() != N:
        raise RuntimeError("rope_append: slots must hold one entry per token")
    if (positions is None) != (cos_sin is None):
        raise RuntimeError("rope_append: positions and cos_sin: both or neither")
    r = None if cos_sin is None else _rope("rope_append", positions, cos_sin, N, dev, sections, cyclic, pairs, False)
    H, qs, os_ = 0, (0, 0), (0, 0)
    if q is not None:
        _rows("rope_append", "q", q, dt, N, dev)
        H, qs = q.shape[1], q.stride()
        if q.shape[2] != Dk:
            raise RuntimeError(f"rope_append: q must be [N, H, {Dk}]")
        if q_out is None:
            q_out = torch.empty(q.shape, dtype=dt, device=dev)
        else:
            _rows("rope_append", "q_out", q_out, dt, N, dev)
            if q_out.shape != q.shape:
                raise RuntimeError("rope_append: q_out must have q's shape")
        os_ = q_out.stride()
    elif q_out is not None:
        raise RuntimeError("rope_append: q_out without q")
    with on_device(dev):
        rc = lib().ws_rope_append(r, ptr(q), qs[0], qs[1], H, Dk, ptr(q_out), os_[0], os_[1], ptr(k), k.stride(0),
                                  k.stride(1), ptr(v), v.stride(0), v.stride(1), _HALF[dt], N, ptr(slots), pool,
                                  stream_ptr(dev))
    check(rc, "ws_rope_append")
    return q_out


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
    ``scope_b200.status_take``.
    """
    if not q.is_cuda:
        raise RuntimeError("paged_decode: CUDA tensors required (there is no CPU path)")
    dev, dt = q.device, q.dtype
    if dt not in _HALF or q.dim() != 3 or q.stride(2) != 1:
        raise RuntimeError("paged_decode: q must be bf16 or fp16 [B, H, Dk] with unit stride on the head dim")
    B, H, D = q.shape
    pool, Hkv, Dk, Dv, pdt = _pool("paged_decode", k_pages, v_pages, k_scales, v_scales, dev)
    if pdt != dt and pdt != torch.int8:
        raise RuntimeError("paged_decode: the pool must hold q's type or int8")
    if D != Dk or Hkv < 1 or H % Hkv:
        raise RuntimeError("paged_decode: q must be [B, Hkv * G, Dk]")
    _table("paged_decode", page_table, B, dev)
    _want("paged_decode", "seq_lens", seq_lens, _I32, 1, dev)
    if seq_lens.numel() != B:
        raise RuntimeError("paged_decode: seq_lens must hold one entry per request")
    if out is None:
        out = torch.empty(B, H, Dv, dtype=dt, device=dev)
    elif out.dtype != dt or out.shape != (B, H, Dv) or not out.is_contiguous() or out.device != dev:
        raise RuntimeError("paged_decode: out must be contiguous [B, H, Dv] in q's type")
    if lse is None:
        lse = torch.empty(B, H, dtype=torch.float32, device=dev)
    elif lse.dtype != torch.float32 or lse.shape != (B, H) or not lse.is_contiguous() or lse.device != dev:
        raise RuntimeError("paged_decode: lse must be contiguous fp32 [B, H]")
    L_ = lib()
    G = H // Hkv
    with on_device(dev):
        ws = workspaces.get(L_.ws_paged_decode_workspace_size(B, Hkv, G, Dv), dev)
        rc = L_.ws_paged_decode(ptr(q), q.stride(0), q.stride(1), _HALF[dt], B, G, pool, ptr(page_table),
                                page_table.stride(0), page_table.shape[1], ptr(seq_lens), window, scale, ptr(out),
                                ptr(lse), ptr(ws), ws.numel(), stream_ptr(dev))
    check(rc, "ws_paged_decode")
    return out, lse
