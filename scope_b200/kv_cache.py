"""Device-resident, sequence-sharded KV caches: the physically partitioned
format the decode kernels read, with append.

Mirrors the reference's caches -- ``InplaceKVCache`` (system/qwenoffload.py:59-141,
GQA: per layer k/v ``[B*Hkv, max_seq, D]``, ``append_4d``, ``get``, ``seq_len``,
``reset``) and ``InplaceKVCacheCompressed`` (system/deepseek.py:144-209,
absorbed MLA: per layer latent ``[B, max_seq, 512]`` and rope ``[B, max_seq, 64]``,
``append``) -- with the buffers in HBM instead of pinned host memory and the
host/GPU share replaced by contiguous token shards across GPUs: rank r of
`world` holds positions [r*cap, (r+1)*cap) with cap = ceil(max_seq / world),
so a decode step's new token lands on one rank only.  Appends run the
``ws_kv_append`` kernel; decodes run ``ws_gqa_decode`` / ``ws_mla_decode`` on
the local shard and (world > 1) merge the shards' partials with one exchange
(scope_b200.shard.PartialExchange).
"""
from __future__ import annotations

import torch

from . import _lib
from ._lib import check, lib, ptr, on_device, stream_ptr


def shard_capacity(max_seq: int, world: int) -> int:
    return -(-max_seq // world)


def local_slice(t: int, n_new: int, cap: int, rank: int) -> tuple[int, int, int]:
    """Of the new tokens at global positions [t, t + n_new), the ones rank
    `rank` stores: returns (first new-token index, count, local position)."""
    lo, hi = rank * cap, (rank + 1) * cap
    a, b = max(t, lo), min(t + n_new, hi)
    if b <= a:
        return 0, 0, 0
    return a - t, b - a, a - lo


def _append(dst: torch.Tensor, src: torch.Tensor, t0: int) -> None:
    """dst [rows, cap, D] <- src [rows, n, D] at local positions [t0, t0 + n)."""
    code = {torch.bfloat16: _lib.WS_DTYPE_BF16, torch.float32: _lib.WS_DTYPE_F32, torch.int8: _lib.WS_DTYPE_I8}[dst.dtype]
    if src.dtype != dst.dtype or src.device != dst.device:
        raise RuntimeError("append: source must match the cache's dtype and device")
    if src.stride(2) != 1:
        src = src.contiguous()
    rows, n, D = src.shape
    with on_device(dst.device):
        rc = lib().ws_kv_append(ptr(dst), dst.stride(0), dst.stride(1), dst.shape[1], ptr(src), src.stride(0),
                                src.stride(1), rows, n, D, code, t0, stream_ptr(dst.device))
    check(rc, "ws_kv_append")


class ShardedKVCache:
    """GQA cache (InplaceKVCache): per layer k, v [B*Hkv, cap, D] on this rank's GPU."""

    def __init__(self, num_layers, batch_size, num_kv_heads, max_seq, head_dim, dtype=torch.bfloat16,
                 world: int = 1, rank: int = 0, device=None):
        self._nl, self._bs, self._kv_h, self._max_seq, self._hd = num_layers, batch_size, num_kv_heads, max_seq, head_dim
        self._bkv = batch_size * num_kv_heads
        self._dtype = dtype
        self.world, self.rank = world, rank
        self.cap = shard_capacity(max_seq, world)
        self.device = torch.device(device) if device is not None else torch.device("cuda", torch.cuda.current_device())
        self.key_cache = [None] * num_layers
        self.value_cache = [None] * num_layers
        self._filled = [0] * num_layers

    def _ensure_buffer(self, li):
        if self.key_cache[li] is None:
            shape = (self._bkv, self.cap, self._hd)
            self.key_cache[li] = torch.empty(shape, dtype=self._dtype, device=self.device)
            self.value_cache[li] = torch.empty(shape, dtype=self._dtype, device=self.device)

    def append_4d(self, li, k_4d, v_4d):
        """k_4d, v_4d [B, Hkv, new_seq, D] on this rank's device (every rank is given
        the step's tokens; each stores the positions it owns)."""
        new_seq = k_4d.shape[2]
        if self._filled[li] + new_seq > self._max_seq:
            raise RuntimeError("KV cache full")
        self._ensure_buffer(li)
        t = self._filled[li]
        first, cnt, t0 = local_slice(t, new_seq, self.cap, self.rank)
        if cnt:
            k = k_4d.reshape(self._bkv, new_seq, self._hd)[:, first:first + cnt]
            v = v_4d.reshape(self._bkv, new_seq, self._hd)[:, first:first + cnt]
            _append(self.key_cache[li], k, t0)
            _append(self.value_cache[li], v, t0)
        self._filled[li] = t + new_seq

    def local_len(self, li) -> int:
        return min(max(self._filled[li] - self.rank * self.cap, 0), self.cap)

    def get(self, li):
        """This rank's filled part: k, v [B*Hkv, local_len, D] (views)."""
        self._ensure_buffer(li)
        n = self.local_len(li)
        return self.key_cache[li][:, :n], self.value_cache[li][:, :n]

    def seq_len(self, li) -> int:
        return self._filled[li]

    def reset(self):
        for i in range(self._nl):
            self.key_cache[i] = None
            self.value_cache[i] = None
            self._filled[i] = 0

    def decode(self, li, q, scale, exchange=None):
        """q [B, H, D] -> (out [B, H, D] bf16, lse [B, H] fp32) over all tokens of the
        layer.  With world > 1 pass the rank's PartialExchange(B*H, D, world)."""
        from .cpu_attn import gqa_decode
        k, v = self.get(li)
        B, H, D = q.shape
        qv = q.reshape(self._bkv, H // self._kv_h, D)
        if self.world == 1:
            out, lse = gqa_decode(qv, k, v, scale)
            return out.reshape(B, H, D), lse.reshape(B, H)
        if exchange is None:
            raise RuntimeError("decode: a PartialExchange is required when world > 1")
        # the kernel writes this rank's partial straight into the exchange block
        gqa_decode(qv, k, v, scale, out_dtype=torch.float32, out=exchange.part_o.view(self._bkv, H // self._kv_h, D),
                   lse=exchange.part_l.view(self._bkv, H // self._kv_h))
        out, lse = exchange.step(torch.bfloat16)
        return out.reshape(B, H, D), lse.reshape(B, H)


class ShardedKVCacheCompressed:
    """Absorbed-MLA cache (InplaceKVCacheCompressed): per layer c [B, cap, kv_lora_rank]
    and pe [B, cap, qk_rope_head_dim] on this rank's GPU."""

    def __init__(self, num_layers, batch_size, max_seq, kv_lora_rank, qk_rope_head_dim, dtype=torch.bfloat16,
                 world: int = 1, rank: int = 0, device=None):
        self._nl, self._B, self._ms, self._clr, self._qrd = num_layers, batch_size, max_seq, kv_lora_rank, qk_rope_head_dim
        self._dtype = dtype
        self.world, self.rank = world, rank
        self.cap = shard_capacity(max_seq, world)
        self.device = torch.device(device) if device is not None else torch.device("cuda", torch.cuda.current_device())
        self.cache_c = [None] * num_layers
        self.cache_pe = [None] * num_layers
        self._filled = [0] * num_layers

    def _ensure(self, li):
        if self.cache_c[li] is None:
            self.cache_c[li] = torch.empty(self._B, self.cap, self._clr, dtype=self._dtype, device=self.device)
            self.cache_pe[li] = torch.empty(self._B, self.cap, self._qrd, dtype=self._dtype, device=self.device)

    def append(self, li, c_kv, k_pe, non_blocking=False):
        """c_kv [B, new_seq, kv_lora_rank], k_pe [B, new_seq, rope] on this rank's device."""
        new_seq = c_kv.shape[1]
        if self._filled[li] + new_seq > self._ms:
            raise RuntimeError("KV cache full")
        self._ensure(li)
        t = self._filled[li]
        first, cnt, t0 = local_slice(t, new_seq, self.cap, self.rank)
        if cnt:
            _append(self.cache_c[li], c_kv[:, first:first + cnt], t0)
            _append(self.cache_pe[li], k_pe[:, first:first + cnt], t0)
        self._filled[li] = t + new_seq

    def local_len(self, li) -> int:
        return min(max(self._filled[li] - self.rank * self.cap, 0), self.cap)

    def get(self, li):
        self._ensure(li)
        n = self.local_len(li)
        return self.cache_c[li][:, :n], self.cache_pe[li][:, :n]

    def seq_len(self, li) -> int:
        return self._filled[li]

    def reset(self):
        for i in range(self._nl):
            self._filled[i] = 0

    def decode(self, li, q_proj, q_pe, scale, exchange=None):
        """Absorbed-MLA decode over all tokens of the layer: q_proj [B*nH, 512],
        q_pe [B*nH, 64] -> (out [B*nH, 512] bf16 normalised, lse [B*nH] fp32).
        With world > 1 pass the rank's PartialExchange(B*nH, 512, world): the
        kernel writes this rank's fp32 partial into its block, then one
        exchange merges the shards (a rank holding no token of the layer
        contributes lse = -inf)."""
        from .cpu_attn import mla_decode
        c, pe = self.get(li)   # views of the [B, cap, *] buffers: the kernel reads them in place by batch stride
        if self.world == 1:
            return mla_decode(q_proj, q_pe, c, pe, scale)
        if exchange is None:
            raise RuntimeError("decode: a PartialExchange is required when world > 1")
        mla_decode(q_proj, q_pe, c, pe, scale, out_dtype=torch.float32, out=exchange.part_o, lse=exchange.part_l)
        return exchange.step(torch.bfloat16)


class PagedKVCache:
    """Paged GQA cache of a model's layers on one GPU: a pool of pages per layer, and one page table, length array and
    ring of free pages that the layers share.

    Where ``ShardedKVCache`` reserves max_seq tokens for every row, a request here holds only the pages its tokens
    fill, so ``num_pages * page_size`` bounds the requests' summed length.  ``dtype`` bf16, fp16, int8 or
    float8_e4m3fn (codes with one fp32 scale for each head and ``scale_block`` tokens of a page, which it divides; 1: one
    per row).  In 8 bits decode is fastest over pages and blocks of 32, 64, ... tokens, at head dims of 64, 128, ... (8 requests
    of 16384 to 65536 tokens, 4 heads of 128, with blocks of 32 and of 16: int8 71 us and 78, e4m3 68 and 72).  Per step:

        step = cache.begin_step(new_lens, n_tokens)       # pages, slots, positions; lengths advance
        q = cache.append(li, q, k, v, step, cos_sin)      # each layer: rotate, write keys and values
        out, lse = cache.decode(li, q_last, scale)        # each layer: one query per request
        cache.release(done)                               # finished requests' pages go back

    ``read`` gives rows back, and ``diff_decode`` is differential attention, with the cache's heads in pairs.

    Nothing here waits for the device; ``free_pages()`` and ``refused()`` do.  The table, lengths and ring are updated
    in place, so the calls can be captured in a CUDA graph.  ``begin_step`` serves requests in order and refuses whole what
    does not fit; a request that lacks pages also keeps those behind it from new ones (``paged.paged_slots``), so admit
    only what the pool can hold to its end.
    """

    def __init__(self, num_layers, num_pages, page_size, num_kv_heads, head_dim, max_requests, max_seq,
                 v_head_dim=None, dtype=torch.bfloat16, device=None, scale_block=1):
        quantised = dtype in (torch.int8, torch.float8_e4m3fn)
        if scale_block < 1 or page_size % scale_block or (scale_block > 1 and not quantised):
            raise RuntimeError("PagedKVCache: scale_block must divide page_size, and belongs to an 8-bit cache")
        dev = torch.device(device) if device is not None else torch.device("cuda", torch.cuda.current_device())
        self.device, self.page_size, self.num_pages, self.max_requests = dev, page_size, num_pages, max_requests
        vd = head_dim if v_head_dim is None else v_head_dim
        # A head's rows of a page lie together where there is a scale a block: rows of 8 bits are short pieces otherwise
        # (32 requests of 65536 tokens, 8 heads of 128 in e4m3: 650 us, with a token's heads together 731).
        heads_major = quantised and (scale_block > 1 or dtype != torch.int8)

        def pages(D):
            if heads_major:
                return torch.empty(num_pages, num_kv_heads, page_size, D, dtype=dtype, device=dev).transpose(1, 2)
            return torch.empty(num_pages, page_size, num_kv_heads, D, dtype=dtype, device=dev)

        self.k_pages = [pages(head_dim) for _ in range(num_layers)]
        self.v_pages = [pages(vd) for _ in range(num_layers)]
        blocks = (num_pages, page_size // scale_block, num_kv_heads)
        self.k_scales = [torch.empty(blocks, device=dev) if quantised else None for _ in range(num_layers)]
        self.v_scales = [torch.empty(blocks, device=dev) if quantised else None for _ in range(num_layers)]
        self.page_table = torch.empty(max_requests, -(-max_seq // page_size), dtype=torch.int32, device=dev)
        self.seq_lens = torch.empty(max_requests, dtype=torch.int32, device=dev)
        self._free = torch.empty(num_pages, dtype=torch.int32, device=dev)
        self._ring = torch.empty(3, dtype=torch.int32, device=dev)
        self.reset()

    def reset(self):
        """Every request empty, every page free."""
        self.page_table.fill_(-1)
        self.seq_lens.zero_()
        torch.arange(self.num_pages, out=self._free)
        self._ring.zero_()
        self._ring[1].fill_(self.num_pages)

    def begin_step(self, new_lens, n_tokens):
        """new_lens int32 [max_requests] on the device: the tokens each request adds (0: none); n_tokens: the rows of
        the packed step.  Returns a ``paged.PagedStep``."""
        from .paged import paged_slots
        return paged_slots(self.seq_lens, new_lens, self.page_table, self._free, self._ring, self.page_size, n_tokens,
                           seq_lens_out=self.seq_lens, ring_out=self._ring)

    def append(self, li, q, k, v, step, cos_sin=None, positions=None, **rope):
        """Write the step's keys and values into layer li's pool and return its rotated queries.  ``positions``
        (default: ``step.positions``) is given for tokens with several axes; ``rope``: sections, cyclic, pairs,
        q_out of ``paged.rope_append``."""
        from .paged import rope_append
        if cos_sin is not None and positions is None:
            positions = step.positions
        return rope_append(q, k, v, positions, cos_sin, step.slots, self.k_pages[li], self.v_pages[li],
                           k_scales=self.k_scales[li], v_scales=self.v_scales[li], **rope)

    def decode(self, li, q, scale, window=0, out=None, lse=None):
        """q [max_requests, H, D], one query per request -> (out, lse) over the request's tokens."""
        from .paged import paged_decode
        return paged_decode(q, self.k_pages[li], self.v_pages[li], self.page_table, self.seq_lens, scale,
                            window=window, k_scales=self.k_scales[li], v_scales=self.v_scales[li], out=out, lse=lse)

    def diff_decode(self, li, q, scale, lam, norm_weight=None, norm_eps=1e-5, window=0, out=None, lse=None):
        """Differential attention, pool heads 2g and 2g + 1 a pair: q [max_requests, 2 * H, D] -> (out [max_requests, H,
        2 * v_head_dim], lse of each map); ``paged.paged_diff_decode``."""
        from .paged import paged_diff_decode
        return paged_diff_decode(q, self.k_pages[li], self.v_pages[li], self.page_table, self.seq_lens, scale, lam,
                                 norm_weight=norm_weight, norm_eps=norm_eps, window=window, k_scales=self.k_scales[li],
                                 v_scales=self.v_scales[li], out=out, lse=lse)

    def read(self, li, cu_seqlens, n_tokens, starts=None, dtype=None, k_out=None, v_out=None):
        """Rows of layer li, request b's at [cu_seqlens[b], cu_seqlens[b + 1]) from its token starts[b] on (default: the
        first) -> (k [n_tokens, kv heads, D], v); ``paged.paged_read``."""
        from .paged import paged_read
        return paged_read(self.k_pages[li], self.v_pages[li], self.page_table, cu_seqlens, n_tokens, starts=starts,
                          k_scales=self.k_scales[li], v_scales=self.v_scales[li], dtype=dtype, k_out=k_out, v_out=v_out)

    def release(self, done):
        """done bool [max_requests] on the device: these requests' pages go back and their lengths become 0."""
        from .paged import paged_release
        paged_release(self.seq_lens, done, self.page_table, self._free, self._ring, self.page_size,
                      seq_lens_out=self.seq_lens, ring_out=self._ring)

    def free_pages(self) -> int:
        """Pages free now (waits for the device)."""
        return int(self._ring[1])

    def refused(self) -> int:
        """How many requests the last begin_step refused (waits for the device).  Their lengths did not grow; their
        tokens were not written."""
        return int(self._ring[2])
