"""The paged serving example's admission: no request it admits is ever refused a page, and what can never fit is turned
down.  On the CPU a counting cache stands in for the paged one; on the GPU the emitted tokens are compared with the plain
model's."""
import os
import sys

import numpy as np
import pytest
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))

import paged_serving  # noqa: E402


class CountingCache:
    """The pages of a PagedKVCache, counted on the host."""

    def __init__(self, layers, num_pages, page_size, kv_heads, head_dim, max_requests, max_seq, device=None):
        self.P, self.free, self.lens, self.most, self.last = page_size, num_pages, [0] * max_requests, max_seq, 0
        self.seq_lens = self._ring = torch.zeros(1)

    def pages(self, n):
        return -(-n // self.P)

    def begin_step(self, new_lens, n):
        self.last = 0
        for b, m in enumerate(new_lens.tolist()):
            need = self.pages(self.lens[b] + m) - self.pages(self.lens[b])
            if need > self.free or self.lens[b] + m > self.most:
                self.last += 1
            else:
                self.free -= need
                self.lens[b] += m

    def release(self, done):
        for b, d in enumerate(done.tolist()):
            if d:
                self.free += self.pages(self.lens[b])
                self.lens[b] = 0

    def free_pages(self):
        return self.free

    def refused(self):
        return self.last


class CountingModel:
    embed, Hkv, D = torch.zeros(8, 4), 1, 16

    def __init__(self):
        self.refused, self.steps = 0, 0

    def step(self, cache, tokens, new_lens, last):
        self.steps += 1
        assert self.steps < 5000, "the loop does not end"
        assert tokens.numel() == int(new_lens.sum())
        cache.begin_step(new_lens, tokens.numel())
        self.refused += cache.refused()
        return torch.zeros(last.numel(), 8)


def count(monkeypatch, lens, n_new, batch, pages, P):
    monkeypatch.setattr(paged_serving, "PagedKVCache", CountingCache)
    m = CountingModel()
    texts = paged_serving.serve(m, [[1] * n for n in lens], n_new, batch, pages, P, graph=False)
    assert [len(t) for t in texts] == [n + n_new for n in lens]
    return m


def test_whole_page_prompts_in_a_tight_pool(monkeypatch):
    assert count(monkeypatch, [16, 16], 24, 2, 5, 16).refused == 0


def test_no_admitted_request_is_refused(monkeypatch):
    r = np.random.RandomState(0)
    for _ in range(300):
        P = int(r.choice([1, 4, 16]))
        lens = [int(r.randint(1, 5)) * P if r.rand() < 0.7 else int(r.randint(1, 5 * P + 1)) for _ in range(r.randint(1, 9))]
        n_new = int(r.randint(1, 3 * P + 2))
        least = max(-(-(n + n_new - 1) // P) for n in lens)   # the pool that the largest just fits
        assert count(monkeypatch, lens, n_new, int(r.randint(1, 6)), least + int(r.randint(0, 2 * least)), P).refused == 0


@pytest.mark.parametrize("lens,n_new,pages", [([16, 90], 24, 7), ([5, 0], 3, 9), ([5], 0, 9)])
def test_what_cannot_be_served_is_turned_down(monkeypatch, lens, n_new, pages):
    with pytest.raises(ValueError, match="serve"):
        count(monkeypatch, lens, n_new, 2, pages, 16)


@pytest.mark.gpu
@pytest.mark.parametrize("graph", [False, True])
def test_tokens_in_a_tight_pool_are_the_plain_models(graph):
    from test_paged_example_gpu import plain_logits
    m = paged_serving.OneLayer(vocab=128, width=128, heads=8, kv_heads=2, head_dim=32, top=512)
    g = torch.Generator().manual_seed(8)
    prompts = [torch.randint(0, 128, (n,), generator=g).tolist() for n in (16, 16, 32, 48, 16, 64, 1, 32)]
    held, sure = [], 0

    def check(texts, logits):
        for t, row in zip(texts, logits):
            if t is not None:
                held.append((list(t), row.float().cpu()))

    texts = paged_serving.serve(m, prompts, n_new=24, batch=3, num_pages=9, graph=graph, on_step=check)
    for t, row in held:
        want = plain_logits(m, t).cpu()
        room = 0.03 * want.abs().max()   # bf16 logits of a few units over a width of 128, twice rounded on the way
        assert (row - want).abs().max() <= room
        next_tokens = {x[len(t)] for x in texts if len(x) > len(t) and x[:len(t)] == t}
        top = want.topk(2).values
        if top[0] - top[1] > 2 * room:   # the two cannot have changed places
            assert int(want.argmax()) in next_tokens
            sure += 1
    assert len(held) == 24 * len(prompts) and sure > 0
