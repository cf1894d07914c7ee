"""GPU checks of what the paged operators' binding turns down."""
import pytest
import torch

from scope_b200 import paged
from test_paged_gpu import BF, DEV, table_of

pytestmark = pytest.mark.gpu


def test_an_argument_whose_truth_raises_is_an_error():
    x = torch.ones(4, 2, 32, dtype=BF, device=DEV)
    pos, table = torch.zeros(4, dtype=torch.int32, device=DEV), table_of(8, 32)
    with pytest.raises(RuntimeError, match="ambiguous"):
        paged.rope(x, pos, table, inverse=torch.tensor([0, 1]))
    assert torch.equal(paged.rope(x, pos, table, inverse=torch.tensor(1)), paged.rope(x, pos, table, inverse=True))


def test_outputs_that_share_memory_with_what_is_read():
    """Each of these would be written while it is read; in place, whole, is allowed."""
    buf = torch.zeros(9, dtype=torch.int32, device=DEV)
    lens, new = buf[:8], torch.ones(8, dtype=torch.int32, device=DEV)
    table, free = torch.zeros(8, 4, dtype=torch.int32, device=DEV), torch.arange(32, dtype=torch.int32, device=DEV)
    ring = torch.tensor([0, 32, 0], dtype=torch.int32, device=DEV)
    done = torch.zeros(8, dtype=torch.bool, device=DEV)
    for kw in (dict(seq_lens_out=new), dict(seq_lens_out=buf[1:]), dict(ring_out=new[:3]), dict(ring_out=free[4:7]),
               dict(seq_lens_out=free[:8]), dict(seq_lens_out=table.view(-1)[:8])):
        with pytest.raises(RuntimeError, match="overlap|memory location"):
            paged.paged_slots(lens, new, table, free, ring, 16, 8, **kw)
    for kw in (dict(seq_lens_out=buf[1:]), dict(ring_out=lens[:3]), dict(ring_out=free[4:7])):
        with pytest.raises(RuntimeError, match="overlap|memory location"):
            paged.paged_release(lens, done, table, free, ring, 16, **kw)
    assert paged.paged_slots(lens, new, table, free, ring, 16, 8, seq_lens_out=lens, ring_out=ring).seq_lens is lens

    wide = torch.randn(5, 2, 32, device=DEV).to(BF)
    x, pos, turns = wide[:4], torch.zeros(4, dtype=torch.int32, device=DEV), table_of(8, 32)
    one = torch.zeros(1, 2, 32, dtype=BF, device=DEV)
    for out in (wide[1:], one.expand(4, 2, 32)):
        with pytest.raises(RuntimeError, match="overlap|memory location"):
            paged.rope(x, pos, turns, out=out)
    assert paged.rope(x, pos, turns, out=x) is x
    pool = torch.zeros(2, 2, 16, 2, 32, dtype=BF, device=DEV)
    slots = torch.arange(4, device=DEV)
    k = torch.zeros(4, 2, 32, dtype=BF, device=DEV)
    for q_out in (wide[1:], k, one.expand(4, 2, 32)):
        with pytest.raises(RuntimeError, match="overlap|memory location"):
            paged.rope_append(x, k, k, pos, turns, slots, pool[0], pool[1], q_out=q_out)
    with pytest.raises(RuntimeError, match="overlap|memory location"):   # every page the same memory
        paged.rope_append(x, k, k, pos, turns, slots, pool[0, :1].expand(2, 16, 2, 32), pool[1])
    qkv = torch.randn(4, 6, 32, device=DEV).to(BF)   # views of a packed projection lie between one another
    q = qkv[:, :2]
    assert paged.rope_append(q, qkv[:, 2:4], qkv[:, 4:], pos, turns, slots, pool[0], pool[1], q_out=q) is q
    q = torch.zeros(8, 4, 32, dtype=BF, device=DEV)
    with pytest.raises(RuntimeError, match="overlap|memory location"):
        paged.paged_decode(q, pool[0], pool[1], table, lens, 1.0, out=q)
    with pytest.raises(RuntimeError, match="overlap|memory location"):
        paged.paged_decode(q, pool[0], pool[1], table, lens, 1.0, lse=q.view(torch.float32).view(-1)[:32].view(8, 4))
