"""GPU checks of captured steps: a graph stays right whatever happens to the stream's workspace between its capture and
its replays.  Results of replays are compared with eager calls on the same inputs bit for bit (the operators repeat
themselves), bookkeeping with the definition."""
import numpy as np
import pytest
import torch

import scope_b200
from scope_b200 import _lib, paged

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF = torch.bfloat16


def decode_inputs(seed, lens=(9000, 40, 3000), H=8, Hkv=2, D=128, P=16):
    """Rows that cross several blocks, so that they are joined through the workspace."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    held = [-(-n // P) for n in lens]
    n_pages = sum(held) + 1
    ids = torch.randperm(n_pages, generator=g, device=DEV).int()
    table = torch.zeros(len(lens), max(held), dtype=torch.int32, device=DEV)
    at = 0
    for b, n in enumerate(held):
        table[b, :n] = ids[at:at + n]
        at += n
    k, v = (torch.randn(n_pages, P, Hkv, D, generator=g, device=DEV).to(BF) for _ in range(2))
    q = torch.randn(len(lens), H, D, generator=g, device=DEV).to(BF)
    return q, k, v, table, torch.tensor(lens, dtype=torch.int32, device=DEV), D ** -0.5


def occupy():
    """Tensors in whatever memory the allocator has to give, every byte set."""
    return [torch.full((n,), 0xff, dtype=torch.uint8, device=DEV) for n in (64 << 20, 4 << 20, 4 << 20, 1 << 20, 1 << 20)]


def untouched(tensors):
    return all(bool((t == 0xff).all()) for t in tensors)


def capture(side, body):
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = body()
    return graph, out


def cold_stream():
    """A stream whose workspace the pool has not made yet."""
    side = torch.cuda.Stream()
    key = (torch.cuda.current_device(), side.cuda_stream)
    if key in _lib.workspaces._bufs:
        _lib.workspaces._outgrown.append((key[0], _lib.workspaces._bufs.pop(key)))
    return side


def test_replays_after_a_reported_page_are_right():
    inputs = decode_inputs(1)
    want = [x.clone() for x in paged.paged_decode(*inputs)]
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        paged.paged_decode(*inputs)
        side.synchronize()
        graph, got = capture(side, lambda: paged.paged_decode(*inputs))
        good = int(inputs[3][0, 3])
        inputs[3][0, 3] = -1
        paged.paged_decode(*inputs)
        assert scope_b200.status_take() == _lib.WS_ERR_DEVICE
        inputs[3][0, 3] = good
        others = occupy()
        for _ in range(3):
            got[0].fill_(float("nan"))
            graph.replay()
            side.synchronize()
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert untouched(others) and scope_b200.status_take() == 0


def slots_state(seed, B=300, P=16, width=40, n=12000):
    r = np.random.RandomState(seed)
    n_pages = B * width // 2
    lens = torch.zeros(B, dtype=torch.int32, device=DEV)
    table = torch.full((B, width), -1, dtype=torch.int32, device=DEV)
    free = torch.from_numpy(r.permutation(n_pages).astype(np.int32)).to(DEV)
    ring = torch.tensor([n_pages - 7, n_pages, 0], dtype=torch.int32, device=DEV)
    return lens, table, free, ring, P, n, r


def plain_slots(lens, new, table, free, ring, P, n):
    """The definition, for steps that refuse nothing: (slots, positions, lengths, ring, table)."""
    table, at, slots, pos = table.copy(), int(ring[0]), [], []
    for b in range(len(lens)):
        for p in range(int(lens[b]), int(lens[b]) + int(new[b])):
            if p % P == 0:
                table[b, p // P] = free[at % len(free)]
                at += 1
            slots.append(int(table[b, p // P]) * P + p % P)
            pos.append(p)
    took = at - int(ring[0])
    fill = n - len(slots)
    return (np.array(slots + [-1] * fill, np.int64), np.array(pos + [0] * fill, np.int32), lens + new,
            np.array([at % len(free), int(ring[1]) - took, 0], np.int32), table)


@pytest.mark.parametrize("grow", [False, True])
def test_replays_of_an_in_place_step_of_several_blocks(grow):
    """Lengths and ring updated in place by the block that finishes last, step after step, also when a larger workspace
    has taken the place of the one that the graph was captured with."""
    lens, table, free, ring, P, n, r = slots_state(2)
    new = torch.zeros_like(lens)
    side = cold_stream()
    with torch.cuda.stream(side):
        def body():
            return paged.paged_slots(lens, new, table, free, ring, P, n, seq_lens_out=lens, ring_out=ring)
        body()   # adds nothing
        side.synchronize()
        graph, step = capture(side, body)
        others = []
        if grow:
            _lib.workspaces.get(64 << 20, torch.device(DEV))
            others = occupy()
        for _ in range(5):
            add = r.randint(0, 40, len(lens)).astype(np.int32)
            before = [x.cpu().numpy() for x in (lens, table, free, ring)]
            new.copy_(torch.from_numpy(add))
            graph.replay()
            side.synchronize()
            want = plain_slots(before[0], add, before[1], before[2], before[3], P, n)
            for x, y in zip((step.slots, step.positions, lens, ring, table), want):
                assert np.array_equal(x.cpu().numpy(), y)
    assert untouched(others) and scope_b200.status_take() == 0


def test_graphs_captured_on_a_fresh_stream_replay_in_any_order():
    one, two = decode_inputs(3), decode_inputs(4, lens=(20000,))
    want1, want2 = ([x.clone() for x in paged.paged_decode(*i)] for i in (one, two))
    side = cold_stream()
    dirty = torch.full((64 << 20,), 0xff, dtype=torch.uint8, device=DEV)   # what a buffer that nothing zeroed would hold
    del dirty
    with torch.cuda.stream(side):
        g1, got1 = capture(side, lambda: paged.paged_decode(*one))
        g2, got2 = capture(side, lambda: paged.paged_decode(*two))
        for g, got, want in ((g2, got2, want2), (g1, got1, want1), (g2, got2, want2)):
            got[0].fill_(float("nan"))
            g.replay()
            side.synchronize()
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        del g1
        out, lse = paged.paged_decode(*one)   # and the stream goes on without the graph
        side.synchronize()
        assert torch.equal(out, want1[0]) and torch.equal(lse, want1[1])


def test_workspaces_are_zeroed_where_they_lie():
    buf = _lib.workspaces.get(1 << 20, torch.device(DEV))
    buf[:64] = 1
    _lib.workspaces.rezero(torch.cuda.current_device())
    assert _lib.workspaces.get(1 << 20, torch.device(DEV)) is buf and not buf.any()


def test_a_cache_is_reset_without_waiting():
    """Nothing of it touches the host's memory, so it can be captured."""
    cache = scope_b200.PagedKVCache(1, 9, 16, 1, 32, 3, 64, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graph, _ = capture(side, cache.reset)
        cache.begin_step(torch.tensor([40, 20, 70], dtype=torch.int32, device=DEV), 130)
        assert cache.free_pages() == 4 and cache.refused() == 1 and cache.seq_lens.tolist() == [40, 20, 0]
        graph.replay()
        side.synchronize()
    assert cache.free_pages() == 9 and cache.refused() == 0 and cache.seq_lens.tolist() == [0, 0, 0]
    assert cache._free.tolist() == list(range(9)) and (cache.page_table == -1).all()
