"""Prep with positions on several axes, captured and replayed: the q rows and the pools' rows, bit for
bit, at the positions, starts and pages of the replay."""
import pytest
import torch

from test_gpu_paged import gen, i32
from test_gpu_tree_cache import bits, prep_inputs

pytestmark = pytest.mark.gpu

F16, I32 = torch.float16, torch.int32


@pytest.mark.parametrize("kv8", [False, True])
@pytest.mark.parametrize("spans", [[(20, 100), (9, 0)], [(300, 5), (1, 40), (260, 0)]], ids=str)
def test_a_replay_stores_the_rows_of_its_own_positions(fl, spans, kv8):
    x, pools, (pages, starts, pos0) = prep_inputs(fl, 9, spans, 16, kv8)
    blank, N = [p.clone() for p in pools], x[0].shape[0]
    g = gen(N)
    positions = torch.zeros(3, N, dtype=I32, device="cuda")
    q_out = torch.empty(N, 24, 256, dtype=F16, device="cuda")
    call = lambda q, p: fl.ops.attn_prep_axes(*x, *p, pages, starts, pos0, positions, page_size=16,
                                              sections=(11, 11, 10), interleaved=True, q_out=q)
    call(q_out, pools)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(q_out, pools)
    seen = []
    for step in range(4):
        positions.copy_(torch.randint(0, 50000, (3, N), generator=g, dtype=I32))
        x[1].mul_(-1.0)
        x[2].add_(1.0)
        if step == 1:                       # a sequence earlier in its pages, another with an absent page
            pos0.sub_(i32(*[min(3, p) for _, p in spans]))
            pages[1, 0] = -1
        if step == 2:                       # a token more for the first one
            starts[1:-1] += 1
        q_out.fill_(7.0)
        for p, b in zip(pools, blank):
            p.copy_(b)
        graph.replay()
        want, wp = torch.full_like(q_out, 7.0), [b.clone() for b in blank]
        call(want, wp)
        torch.cuda.synchronize()
        assert torch.equal(q_out, want)
        for p, w, b in zip(pools, wp, blank):
            assert torch.equal(bits(p), bits(w)), f"step {step}"
            assert not torch.equal(bits(p), bits(b))
        seen.append(bits(pools[0]).clone())
    assert all(not torch.equal(a, b) for a, b in zip(seen, seen[1:]))
