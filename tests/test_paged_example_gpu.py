"""The paged serving example: every token it emits is the greedy one of a plain recomputation of the whole text in fp32
from the same bf16 queries, keys and values, with and without the captured step."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))

pytestmark = pytest.mark.gpu


def plain_logits(m, text):
    """The next token's logits from the whole text, no cache."""
    x = m.embed[torch.tensor(text, device=m.embed.device)]
    n = len(text)
    q, k, v = (x @ m.wqkv).split([m.H * m.D, m.Hkv * m.D, m.Hkv * m.D], 1)

    def turned(t, heads):
        t = t.reshape(n, heads, m.D).float()
        c, s = m.turns[:n, None, :m.D // 2], m.turns[:n, None, m.D // 2:]
        a, b = t[..., :m.D // 2], t[..., m.D // 2:]
        return torch.cat([a * c - b * s, b * c + a * s], -1).bfloat16().float()

    q, k = turned(q, m.H)[-1], turned(k, m.Hkv).repeat_interleave(m.H // m.Hkv, 1)
    v = v.reshape(n, m.Hkv, m.D).float().repeat_interleave(m.H // m.Hkv, 1)
    p = torch.softmax(torch.einsum("hd,nhd->hn", q, k) * m.scale, 1)
    out = torch.einsum("hn,nhd->hd", p, v).reshape(1, -1)
    return ((x[-1:].float() + out @ m.wo.float()) @ m.embed.float().t())[0]


@pytest.mark.parametrize("graph", [False, True])
def test_every_token_is_the_plain_models(graph):
    from paged_serving import OneLayer, serve
    m = OneLayer(vocab=128, width=128, heads=8, kv_heads=2, head_dim=32, top=512)
    g = torch.Generator().manual_seed(4)
    prompts = [torch.randint(0, 128, (n,), generator=g).tolist() for n in (1, 40, 17, 16, 100, 3, 64, 15, 33)]
    seen = []

    def check(texts, logits):
        for t, row in zip(texts, logits):
            if t is not None:
                want = plain_logits(m, t)
                # bf16 logits of a few units over a width of 128, twice rounded on the way
                assert (row.float() - want).abs().max() <= 0.03 * want.abs().max()
                seen.append(len(t))

    texts = serve(m, prompts, n_new=9, batch=4, num_pages=30, graph=graph, on_step=check)
    assert [t[:len(p)] for t, p in zip(texts, prompts)] == prompts
    assert [len(t) for t in texts] == [len(p) + 9 for p in prompts] and len(seen) == 9 * len(prompts)
