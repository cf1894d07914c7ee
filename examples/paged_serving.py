"""Serve prompts of any length from one paged cache, with requests joining and leaving while others run.

    python examples/paged_serving.py [--requests 40] [--batch 16] [--cache bf16|int8|e4m3]

A model of one attention layer with random weights, so that a prompt needs the attention of its last token only.  Every
step packs the tokens that the running requests add -- a whole prompt for a request that joins, one token for the others
-- and runs
    begin_step   pages, slots and positions from the lengths       (one launch)
    append       rotate q and k, write k and v into the pages      (one launch; long prompts into 8-bit blocks: two)
    decode       each request's last token over its pages          (one launch)
    release      the pages of requests that are done go back       (one launch)
A step without prompts has one shape, so its launches are captured in a CUDA graph once and replayed.
"""
from __future__ import annotations

import argparse
import os
import sys
import time

import torch

if __name__ == "__main__":
    sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from scope_b200 import PagedKVCache


class OneLayer:
    """Embedding, one attention layer with rotary positions, and the embedding again as the output projection."""

    def __init__(self, vocab=512, width=512, heads=16, kv_heads=4, head_dim=64, top=4096, device="cuda", seed=0):
        g = torch.Generator(device=device).manual_seed(seed)

        def weight(*shape):
            return (torch.randn(*shape, generator=g, device=device) * shape[0] ** -0.5).bfloat16()

        self.H, self.Hkv, self.D, self.scale = heads, kv_heads, head_dim, head_dim ** -0.5
        self.embed = torch.randn(vocab, width, generator=g, device=device).bfloat16()
        self.wqkv = weight(width, (heads + 2 * kv_heads) * head_dim)
        self.wo = weight(heads * head_dim, width)
        angle = torch.arange(top, dtype=torch.float64, device=device)[:, None] * 1e4 ** (
            -torch.arange(0, head_dim, 2, dtype=torch.float64, device=device) / head_dim)
        self.turns = torch.cat([angle.cos(), angle.sin()], 1).float()

    def step(self, cache: PagedKVCache, tokens, new_lens, last):
        """tokens int64 [N], packed; new_lens int32 [B]; last int64 [B], the row of each request's last token.  Returns
        the logits of every request's next token [B, vocab]."""
        N, H, Hkv, D = tokens.numel(), self.H, self.Hkv, self.D
        x = self.embed[tokens]
        q, k, v = (x @ self.wqkv).split([H * D, Hkv * D, Hkv * D], 1)
        step = cache.begin_step(new_lens, N)
        q = cache.append(0, q.view(N, H, D), k.view(N, Hkv, D), v.view(N, Hkv, D), step, self.turns)
        out, _ = cache.decode(0, q[last], self.scale)
        return (x[last] + out.flatten(1) @ self.wo) @ self.embed.t()


def serve(model: OneLayer, prompts, n_new: int, batch: int, num_pages: int, page_size: int = 16, graph: bool = True,
          on_step=None, dtype=None, scale_block=1):
    """Greedy continuations of ``n_new`` tokens for every prompt (lists of token ids), ``batch`` requests at a time.  A
    prompt is admitted when the pool holds every page that it and the running requests can still come to need.  ``dtype``
    and ``scale_block``: the cache's, for one in 8 bits."""
    def pages_of(tokens):
        return -(-tokens // page_size)

    def need_of(prompt):                        # the last token is emitted and never cached
        return pages_of(len(prompt) + n_new - 1)

    if n_new < 1 or not all(prompts):
        raise ValueError("serve: at least one new token, and one in every prompt")
    if any(need_of(p) > num_pages for p in prompts):
        raise ValueError("serve: a prompt and its continuation take more pages than the pool has")
    dev = model.embed.device
    longest = max((len(p) for p in prompts), default=0) + n_new
    held_as = {} if dtype is None else dict(dtype=dtype, scale_block=scale_block)
    cache = PagedKVCache(1, num_pages, page_size, model.Hkv, model.D, batch, longest, device=dev, **held_as)
    waiting, done = list(range(len(prompts))), {}
    slot_of, text = [None] * batch, {}          # which prompt each row of the batch serves; its tokens so far
    # the decode step's fixed buffers, and its graph
    tokens, ones = torch.zeros(batch, dtype=torch.int64, device=dev), torch.zeros(batch, dtype=torch.int32, device=dev)
    rows = torch.arange(batch, device=dev)
    captured, logits = None, None
    while waiting or any(s is not None for s in slot_of):
        new, joining = [0] * batch, []
        free = cache.free_pages()
        # the cache holds a running text without its last token, which the next step appends
        owed = sum(need_of(prompts[s]) - pages_of(len(text[s]) - 1) for s in slot_of if s is not None)
        for b in range(batch):
            if slot_of[b] is None and waiting:
                need = need_of(prompts[waiting[0]])
                if owed + need > free:          # it waits until pages come back
                    break
                owed += need
                slot_of[b] = waiting.pop(0)
                text[slot_of[b]] = list(prompts[slot_of[b]])
                joining.append(b)
        packed, last = [], []
        for b in range(batch):
            if slot_of[b] is not None:
                add = text[slot_of[b]] if b in joining else text[slot_of[b]][-1:]
                packed += add
                new[b] = len(add)
            last.append(max(len(packed) - 1, 0))
        if graph and not joining:
            tokens.copy_(torch.tensor([text[s][-1] if s is not None else 0 for s in slot_of]))
            ones.copy_(torch.tensor([int(s is not None) for s in slot_of], dtype=torch.int32))
            # rows of the packed step are the running requests in order; the fixed step keeps one row a request
            order = torch.cumsum(ones, 0) - 1
            packed_tokens = torch.zeros_like(tokens)
            packed_tokens[order[ones > 0].long()] = tokens[ones > 0]
            rows.copy_(order.clamp(min=0).long())
            tokens.copy_(packed_tokens)
            if captured is None:
                before = cache.seq_lens.clone(), cache._ring.clone()
                side = torch.cuda.Stream(dev)
                side.wait_stream(torch.cuda.current_stream(dev))
                with torch.cuda.stream(side):
                    model.step(cache, tokens, ones, rows)      # allocates the workspace and cuBLAS's
                    cache.seq_lens.copy_(before[0]), cache._ring.copy_(before[1])
                    captured = torch.cuda.CUDAGraph()
                    with torch.cuda.graph(captured, stream=side):
                        logits = model.step(cache, tokens, ones, rows)
                torch.cuda.current_stream(dev).wait_stream(side)
            captured.replay()
            got = logits
        else:
            got = model.step(cache, torch.tensor(packed, device=dev), torch.tensor(new, dtype=torch.int32, device=dev),
                             torch.tensor(last, device=dev))
        if cache.refused():
            raise RuntimeError("serve: a request found no page")
        if on_step is not None:
            on_step([text[s] if s is not None else None for s in slot_of], got)
        choice, leaving = got.argmax(1).tolist(), [False] * batch
        for b in range(batch):
            if slot_of[b] is not None:
                text[slot_of[b]].append(choice[b])
                if len(text[slot_of[b]]) == len(prompts[slot_of[b]]) + n_new:
                    done[slot_of[b]] = text[slot_of[b]]
                    slot_of[b], leaving[b] = None, True
        if any(leaving):
            cache.release(torch.tensor(leaving, device=dev))
    assert cache.free_pages() == num_pages
    return [done[i] for i in range(len(prompts))]


def main():
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--requests", type=int, default=40)
    ap.add_argument("--batch", type=int, default=16)
    ap.add_argument("--new", type=int, default=64)
    ap.add_argument("--cache", choices=["bf16", "int8", "e4m3"], default="bf16", help="8 bits: a scale a page and head")
    a = ap.parse_args()
    model = OneLayer()
    g = torch.Generator().manual_seed(1)
    prompts = [torch.randint(0, 512, (int(n),), generator=g).tolist() for n in torch.randint(1, 1500, (a.requests,), generator=g)]
    pages = 16 * a.batch + 200
    t = time.perf_counter()
    held_as = {"bf16": {}, "int8": dict(dtype=torch.int8, scale_block=16), "e4m3": dict(dtype=torch.float8_e4m3fn, scale_block=16)}
    texts = serve(model, prompts, a.new, a.batch, pages, **held_as[a.cache])
    torch.cuda.synchronize()
    t = time.perf_counter() - t
    held = sum(len(x) for x in texts)
    print(f"{a.requests} requests, {held} tokens through {pages} pages of 16 "
          f"({a.batch} rows reserved whole would take {a.batch * (1500 + a.new) // 16}): {a.requests * a.new / t:.0f} new tokens/s")


if __name__ == "__main__":
    main()
