"""Trees of drafted tokens where the kernels' own borders are: plans of more than 64 tiles, several
heads a workgroup in graphs and on streams, contexts and states that sequences share."""
import pytest
import torch

import paged_tight as tight
import tree_ref
from test_gpu_paged import SCALE, filled, gen, i32, randn
from test_gpu_tree_attention import check as check_z, run as run_attention, seen_by
from test_gpu_tree_cache import (test_axes_that_hold_the_sequences_positions_give_the_plain_prep as plain_prep,
                                 test_every_pair_turns_by_its_own_axis as every_pair)
from test_gpu_tree_gdn import check, commit, run as run_gdn, tree

pytestmark = pytest.mark.gpu

F16, I32 = torch.float16, torch.int32


@pytest.mark.parametrize("kv8", [False, True])
@pytest.mark.parametrize("ctxs,window,sinks", [([50000], 0, 0), ([50000], 44999, 100), ([25000, 70, 31000], 0, 0)],
                         ids=["one", "window", "three"])
def test_runs_of_more_tiles_than_a_plan(fl, dev, ctxs, window, sinks, kv8):
    """1024 columns a kv head leave ten runs, so that one has up to 160 tiles; rows whose tile shows."""
    g = gen(len(ctxs))
    run_attention(fl, 3, ctxs, [tree(g, 64 - b, 64) for b in range(len(ctxs))], 64, kv8, n_q=64, window=window,
                  sinks=sinks, marked=True, q_scale=0.3)


@pytest.mark.parametrize("kv8", [False, True])
def test_other_trees_over_one_context(fl, dev, kv8):
    """Two sequences whose table rows name the same pages (the tree's rows are alike, the trees are not)."""
    g, T, ctx, P = gen(5), 21, 300, 16
    kp, vp, pages, _ = filled(fl, g, [ctx + T], P, kv8)
    n_rows = kp.numel() // (4 * 272) if kv8 else kp.shape[0] * P
    trees = [tree(g, T, T), tree(g, 9, T, "chain"), tree(g, T, T, "star")]
    q = randn(g, 3, T, 24, 512)
    z = fl.ops.attn_tree_paged(q, kp, vp, pages.expand(3, -1).contiguous(), i32(ctx, ctx, ctx - 40),
                               torch.tensor(trees, dtype=I32).cuda(), page_size=P)
    K, V = tight.kernel_values(kp, n_rows, 4, True), tight.kernel_values(vp, n_rows, 4, False)
    row = pages[0].long()
    rows = (row[:, None] * P + torch.arange(P, device="cuda")).flatten()
    for b, c in enumerate((ctx, ctx, ctx - 40)):
        here = torch.tensor([line is not None for line in tree_ref.lines(trees[b])]).cuda()
        idx = rows[:c + T]
        want, bound = tight.attention(q[b][here][..., :256], K[idx], V[idx], seen_by(trees[b], c)[here], SCALE,
                                      tight.TWO_TERMS if kv8 else tight.ONE_TERM, q[b][here][..., 256:])
        check_z(z[b][here], want, bound, f"tree {b}")


@pytest.mark.parametrize("N", [511, 512, 1001])
def test_many_tokens_turn_by_several_axes(fl, N):
    every_pair(fl, N, (11, 11, 10), True)


@pytest.mark.parametrize("kv8", [False, True])
def test_axes_prep_of_many_tokens_is_the_plain_one(fl, kv8):
    plain_prep(fl, [(300, 0), (255, 17), (400, 1000)], 3, (12, 10, 10), False, kv8)


def gdn_batch(seed, B, T):
    g = gen(seed)
    return g, tree_ref.gdn_layer(g, B, T), [tree(g, T - b, T) for b in range(B)]


@pytest.mark.parametrize("B,T", [(2, 64), (6, 40), (7, 16)])
def test_gdn_trees_at_once_on_two_streams(fl, B, T):
    _, d, parents = gdn_batch(B, B, T)
    e = dict(d, x=-d["x"])
    want = [run_gdn(fl, s, parents, [9] * B) for s in (d, e)]
    streams = [torch.cuda.Stream() for _ in want]
    torch.cuda.synchronize()
    got = []
    for _ in range(5):
        for stream, s in zip(streams, (d, e)):
            with torch.cuda.stream(stream):
                got.append(run_gdn(fl, s, parents, [9] * B))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[i % 2]) for i, y in enumerate(got))


def test_gdn_batches_in_a_graph(fl):
    B, T = 6, 45
    g, d, parents = gdn_batch(3, B, T)
    at, y = torch.tensor(parents, dtype=I32).cuda(), torch.empty(B, T, 48 * 128, dtype=F16, device="cuda")
    call = lambda y: fl.ops.gdn_tree_normed(d["x"], d["S"], d["a"], d["b"], d["A_log"], d["dt_bias"], d["z"],
                                            d["norm_w"], at, y, pos0s=[1] * B, conv_w=d["conv_w"], cst_in=d["cst"])
    call(y)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(y)
    for n in (45, 17, 1, 33):
        at.copy_(torch.tensor([tree(g, max(0, n - 4 * b), T, "binary" if b % 2 else "any") for b in range(B)], dtype=I32))
        d["x"].mul_(-1)
        graph.replay()
        eager = call(torch.empty_like(y))
        torch.cuda.synchronize()
        assert torch.equal(y, eager)


@pytest.mark.parametrize("B", [2, 6])
def test_sequences_that_share_a_state(fl, B):
    """Forks of one sequence: one state and one set of frames, other tokens."""
    T = 20
    g, d, parents = gdn_batch(B, B, T)
    d["S"], d["cst"] = [d["S"][0]] * B, [d["cst"][0]] * B
    want, bound = tree_ref.gdn_tree(d, parents, [False] * B)
    check(run_gdn(fl, d, parents, [12] * B), want, bound, f"{B} forks")
    S, frames = commit(fl, d, [[0, 3, 5]] * B, [12] * B, False)
    for b, (want, bound, f) in enumerate(tree_ref.gdn_commit(d, [[0, 3, 5]] * B, [False] * B)):
        check(S[b], want, bound, f"fork {b}")
        assert torch.equal(frames[b], f)


@pytest.mark.parametrize("kv8", [False, True])
@pytest.mark.parametrize("ctxs,T", [([1000], 16), ([40, 0, 900, 5], 33), ([20000, 300], 64), ([64] * 70, 2)])
def test_nothing_behind_the_buffers_is_written(fl, dev, ctxs, T, kv8):
    """The work buffer exactly as large as asked for, z with a wider pitch, both in the middle of others."""
    g, B = gen(T), len(ctxs)
    kp, vp, pages, _ = filled(fl, g, [c + T for c in ctxs], 16, kv8)
    q, parents = randn(g, B, T, 24, 512), torch.tensor([tree(g, T, T)] * B, dtype=I32).cuda()
    need = fl.ops.attn_tree_paged_work_bytes(B, T)
    work = torch.full((need + 8192,), 0x5A, dtype=torch.uint8, device="cuda")
    z = torch.full((B + 2, T, 24, 264), 7.0, dtype=F16, device="cuda")
    call = lambda **kw: fl.ops.attn_tree_paged(q, kp, vp, pages, i32(*ctxs), parents, page_size=16, **kw)
    call(work=work[4096:4096 + need], z=z[1:-1])
    assert torch.equal(z[1:-1, ..., :256], call())
    assert (z[1:-1, ..., 256:] == 7).all() and (z[0] == 7).all() and (z[-1] == 7).all()
    assert (work[:4096] == 0x5A).all() and (work[4096 + need:] == 0x5A).all()


@pytest.mark.parametrize("B,T", [(1, 3), (2, 64), (6, 40), (16, 17)])
def test_gdn_trees_write_their_outputs_alone(fl, B, T):
    _, d, parents = gdn_batch(B, B, T)
    wide = 48 * 128
    y = torch.full((B * T + 2, wide), 7.0, dtype=F16, device="cuda")
    out = y[1:-1].view(B, T, wide)
    S = torch.full((B + 2, 48, 128, 128), 7.0, device="cuda")
    frames = torch.full((B + 2, 10240, 3), 7.0, dtype=F16, device="cuda")
    at = torch.tensor(parents, dtype=I32).cuda()
    fl.ops.gdn_tree_normed(d["x"], d["S"], d["a"], d["b"], d["A_log"], d["dt_bias"], d["z"], d["norm_w"], at, out,
                           pos0s=[4] * B, conv_w=d["conv_w"], cst_in=d["cst"])
    assert torch.equal(out, run_gdn(fl, d, parents, [4] * B))
    path = torch.tensor([[0, 1, 2, -1]] * B, dtype=I32).cuda()
    fl.ops.gdn_tree_commit(d["x"], d["S"], d["a"], d["b"], d["A_log"], d["dt_bias"], path, list(S[1:-1]),
                           pos0s=[4] * B, conv_w=d["conv_w"], cst_in=d["cst"], cst_out=list(frames[1:-1]))
    torch.cuda.synchronize()
    for t in (y, S, frames):
        assert (t[0] == 7).all() and (t[-1] == 7).all()
    assert (S[1:-1] != 7).any(-1).all() and (frames[1:-1] != 7).any(-1).all()
