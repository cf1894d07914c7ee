"""The paged serving example with its cache in 8 bits, a scale a page and head: it runs to the end, with and without the
captured step."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.int8, torch.float8_e4m3fn])
def test_the_example_runs_in_8_bits(dtype):
    from paged_serving import OneLayer, serve
    m = OneLayer(vocab=128, width=128, heads=8, kv_heads=2, head_dim=32, top=512)
    g = torch.Generator().manual_seed(4)
    prompts = [torch.randint(0, 128, (n,), generator=g).tolist() for n in (1, 40, 17, 16, 100, 3, 64, 15, 33)]
    for graph in (False, True):
        texts = serve(m, prompts, n_new=9, batch=4, num_pages=30, graph=graph, dtype=dtype, scale_block=16)
        assert [t[:len(p)] for t, p in zip(texts, prompts)] == prompts
        assert [len(t) for t in texts] == [len(p) + 9 for p in prompts]
