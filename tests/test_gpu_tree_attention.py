"""Attention of trees of drafted tokens over the paged cache against the formulas in float64
(paged_tight.py derives the bounds): contexts, trees, windows, absent places, long runs."""
import pytest
import torch

import paged_ref as ref
import paged_tight as tight
import tree_ref
from test_gpu_paged import SCALE, blank, filled, gen, i32, randn, starts_of, values
from test_gpu_tree_gdn import tree

pytestmark = pytest.mark.gpu

F16, F32, I32 = torch.float16, torch.float32, torch.int32


def seen_by(parents, ctx, window=0, sinks=0, present=None):
    """[T, ctx + T] truth values: what each token sees of the context's and the tree's rows."""
    T = len(parents)
    see = torch.zeros(T, ctx + T, dtype=torch.bool)
    r = torch.arange(ctx)
    for i, line in enumerate(tree_ref.lines(parents)):
        if line is None:
            continue
        p = ctx + len(line) - 1
        see[i, :ctx] = True if not window else (r > p - window) | (r < sinks)
        for depth, j in enumerate(line):
            see[i, ctx + j] = not window or ctx + depth > p - window or ctx + depth < sinks
    if present is not None:
        see &= present[None]
    return see.cuda()


def check(z, want, bound, what):
    err = (z.double() - want).abs()
    assert torch.isfinite(z).all(), f"{what}: not finite"
    worst = (err / bound).max().item()
    print(f"{what}: max|err| {err.max().item():.2e}, {worst:.2f} of the bound")
    assert worst <= 1.0, f"{what}: {worst} of the bound"


def spoil(pool, rows, n_rows, n_kv):
    """NaN in pool rows (int8: their scales)."""
    if pool.dtype == torch.int8:
        pool[n_rows * n_kv * 256:].view(F16).view(n_rows, -1)[rows] = float("nan")
    else:
        pool.view(n_rows, -1)[rows] = float("nan")


def run(fl, seed, ctxs, trees, page_size, kv8, n_q=24, n_kv=4, window=0, sinks=0, gate=True, marked=False,
        q_scale=1.0, pitch=512):
    """One call against the reference; trees: parents of every sequence, alike in length."""
    g, T = gen(seed), len(trees[0])
    lens = [c + T for c in ctxs]
    if marked:
        pages, n_pages = ref.make_pages(g, lens, page_size)
        kp, vp = (blank(fl, n_pages, page_size, kv8, n_kv) for _ in range(2))
        k, v = (torch.cat(x).cuda() for x in zip(*(tight.marked_rows(g, n, n_kv) for n in lens)))
        fl.ops.paged_kv_store(k, v, kp, vp, pages, starts_of(lens), torch.zeros(len(lens), dtype=I32, device="cuda"),
                              page_size=page_size, n_kv_heads=n_kv)
    else:
        kp, vp, pages, _ = filled(fl, g, lens, page_size, kv8, n_kv)
        n_pages = (kp.numel() // (page_size * n_kv * 272)) if kv8 else kp.shape[0]
    n_rows, host = n_pages * page_size, pages.cpu()
    rows = [ref.rows_of(host, b, page_size, torch.arange(n)).cuda() for b, n in enumerate(lens)]
    # places without a token hold NaN, and so does their q
    q = randn(g, len(ctxs), T, n_q, pitch, scale=q_scale)
    for b, parents in enumerate(trees):
        gone = [i for i, line in enumerate(tree_ref.lines(parents)) if line is None]
        if gone:
            for pool in (kp, vp):
                spoil(pool, rows[b][[ctxs[b] + i for i in gone]], n_rows, n_kv)
            q[b, gone] = float("nan")
    z = fl.ops.attn_tree_paged(q, kp, vp, pages, i32(*ctxs), torch.tensor(trees, dtype=I32).cuda(),
                               page_size=page_size, window=window, sinks=sinks, gate=gate, n_kv_heads=n_kv)
    K, V = tight.kernel_values(kp, n_rows, n_kv, True), tight.kernel_values(vp, n_rows, n_kv, False)
    for b, parents in enumerate(trees):
        see = seen_by(parents, ctxs[b], window, sinks)
        here = torch.tensor([line is not None for line in tree_ref.lines(parents)]).cuda()
        assert not z[b][~here].any()
        if not here.any():
            continue
        want, bound = tight.attention(q[b][here][..., :256], K[rows[b]], V[rows[b]], see[here], SCALE,
                                      tight.TWO_TERMS if kv8 else tight.ONE_TERM,
                                      q[b][here][..., 256:512] if gate else None)
        check(z[b][here], want, bound, f"sequence {b}, {ctxs[b]} rows")
    return z


@pytest.mark.parametrize("kv8", [False, True])
@pytest.mark.parametrize("T", [1, 2, 5, 6, 11, 16, 22, 33, 43, 64])
@pytest.mark.parametrize("ctxs", [[0], [1, 31], [33, 500, 15]], ids=str)
def test_trees_over_short_contexts(fl, dev, ctxs, T, kv8):
    g = gen(T)
    run(fl, T, ctxs, [tree(g, max(1, T - 3 * b), T) for b in range(len(ctxs))], 16, kv8)


@pytest.mark.parametrize("kv8", [False, True])
@pytest.mark.parametrize("n_q,n_kv,T", [(1, 1, 64), (8, 8, 20), (16, 2, 40), (3, 3, 7), (40, 4, 64), (64, 1, 9)])
def test_other_head_counts(fl, dev, n_q, n_kv, T, kv8):
    g = gen(n_q)
    run(fl, n_q, [70, 200], [tree(g, T, T), tree(g, T // 2, T)], 32, kv8, n_q, n_kv, pitch=520)


@pytest.mark.parametrize("kv8", [False, True])
@pytest.mark.parametrize("kind", ["chain", "star", "binary"])
@pytest.mark.parametrize("page_size", [16, 128])
def test_shapes_of_trees(fl, dev, kind, page_size, kv8):
    g = gen(1)
    run(fl, 1, [100, 41, 0], [tree(g, n, 50, kind) for n in (50, 17, 1)], page_size, kv8, gate=False)


@pytest.mark.parametrize("kv8", [False, True])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (3, 0), (3, 2), (10, 200), (40, 4), (100, 37), (2000, 5)])
def test_windows(fl, dev, window, sinks, kv8):
    g = gen(window)
    run(fl, window, [0, 5, 300, 91], [tree(g, n, 30, k) for n, k in ((30, "chain"), (30, "any"), (21, "binary"), (30, "chain"))],
        16, kv8, window=window, sinks=sinks)


@pytest.mark.parametrize("kv8", [False, True])
def test_places_without_a_token_and_padded_sequences(fl, dev, kv8):
    g, T = gen(5), 26
    trees = [tree(g, T, T) for _ in range(5)]
    for i, p in ((3, 3), (7, 12), (9, -2), (14, 9), (20, 2**31 - 1), (25, -2**31)):
        trees[0][i] = p
    trees[1] = [-2] * T
    trees[2] = [5] + trees[2][1:]
    run(fl, 5, [60, 33, 128, 0, 17], trees, 16, kv8)


@pytest.mark.parametrize("kv8", [False, True])
def test_positions_outside_the_cache(fl, dev, kv8):
    """Negative ones see nothing; rows past the table and on absent pages are not attended to."""
    g, T, P = gen(6), 20, 16
    kp, vp, pages, _ = filled(fl, g, [200, 200, 200, 200], P, kv8)
    pages = pages[:, :10].contiguous()      # 160 rows
    pages[3, 2:4] = -1
    pages[3, 9] = 10**6
    pos0 = [-1, 150, 2**31 - 5, 130]
    q = randn(g, 4, T, 24, 512)
    q[0] = float("nan")
    parents = [tree(g, T, T) for _ in pos0]
    z = fl.ops.attn_tree_paged(q, kp, vp, pages, i32(*pos0), torch.tensor(parents, dtype=I32).cuda(), page_size=P)
    assert not z[0].any()
    n_rows = kp.numel() // (4 * 272) if kv8 else kp.shape[0] * P
    K, V = tight.kernel_values(kp, n_rows, 4, True), tight.kernel_values(vp, n_rows, 4, False)
    host = pages.cpu()
    for b in (1, 2, 3):
        ctx = min(pos0[b], 160)
        at = ref.rows_of(host, b, P, torch.arange(ctx + T))
        at = torch.where((at >= 0) & (at < n_rows), at, -1)
        if pos0[b] > 160:
            at[160:] = -1
        see = seen_by(parents[b], ctx, present=at >= 0) if pos0[b] <= 160 else \
            torch.cat([(at[:160] >= 0).cuda().expand(T, 160), torch.zeros(T, T, dtype=torch.bool, device="cuda")], 1)
        idx = at.clamp_min(0).cuda()
        want, bound = tight.attention(q[b, ..., :256], K[idx], V[idx], see, SCALE,
                                      tight.TWO_TERMS if kv8 else tight.ONE_TERM, q[b, ..., 256:])
        check(z[b], want, bound, f"pos0 {pos0[b]}")
    # a window past the table: no rows at all
    z = fl.ops.attn_tree_paged(q, kp, vp, pages, i32(*[10**6] * 4), torch.tensor(parents, dtype=I32).cuda(), page_size=P,
                               window=100)
    assert not z.any()


@pytest.mark.parametrize("kv8", [False, True])
@pytest.mark.parametrize("ctxs,T", [([5000], 16), ([9000, 40, 2500], 33), ([20000], 64), ([3000] * 20, 3),
                                    ([100 + 37 * i for i in range(70)], 7), ([1] * 300, 4)],
                         ids=["5000", "3 ragged", "20000", "20 x 3000", "70 ragged", "300 x 1"])
def test_runs_of_many_tiles(fl, dev, ctxs, T, kv8):
    """Rows whose tile shows in z: one lost or counted twice is a good part of it."""
    g = gen(T)
    run(fl, T, ctxs, [tree(g, max(1, T - b % 5), T) for b in range(len(ctxs))], 64, kv8, marked=True, q_scale=0.3)


@pytest.mark.parametrize("kv8", [False, True])
def test_many_small_weights_beside_one_large(fl, dev, kv8):
    """As the decode's: a first row that holds nearly all the weight, its v 0."""
    g, P, L, T = gen(3), 64, 700, 10
    pages, n_pages = ref.make_pages(g, [L + T], P)
    K, V = torch.zeros(L + T, 4, 256), 1500 + 100 * torch.randn((L + T, 4, 256), generator=g)
    K[0, :, 0], V[0] = 15.734, 0
    kp, vp = (fl.ops.paged_pool(n_pages, P, kv8=kv8) for _ in range(2))
    fl.ops.paged_kv_store(K.to(F16).cuda(), V.to(F16).cuda(), kp, vp, pages, i32(0, L + T), i32(0), page_size=P)
    q = randn(g, 1, T, 24, 512)
    q[..., 0] = 16
    parents = tree(g, T, T)
    z = fl.ops.attn_tree_paged(q, kp, vp, pages, i32(L), torch.tensor([parents], dtype=I32).cuda(), page_size=P,
                               gate=False)
    rows = ref.rows_of(pages.cpu(), 0, P, torch.arange(L + T)).cuda()
    Kx, Vx = tight.kernel_values(kp, n_pages * P, 4, True)[rows], tight.kernel_values(vp, n_pages * P, 4, False)[rows]
    want, bound = tight.attention(q[0, ..., :256], Kx, Vx, seen_by(parents, L), SCALE,
                                  tight.TWO_TERMS if kv8 else tight.ONE_TERM)
    check(z[0], want, bound, "small weights")


@pytest.mark.parametrize("kv8", [False, True])
def test_a_chain_is_the_decode(fl, dev, kv8):
    """Both off by their own bound at most."""
    g, T = gen(7), 4
    ctxs = [900, 33]
    kp, vp, pages, _ = filled(fl, g, [c + T for c in ctxs], 16, kv8)
    q = randn(g, 2, T, 24, 512)
    a = fl.ops.attn_decode_paged(q, kp, vp, pages, i32(*ctxs), page_size=16)
    z = fl.ops.attn_tree_paged(q, kp, vp, pages, i32(*ctxs), i32(-1, 0, 1, 2).expand(2, 4).contiguous(), page_size=16)
    assert ((a.double() - z.double()).abs() <= 2.0 ** -9 * a.abs().amax(-1, keepdim=True) + 2.0 ** -24).all()


@pytest.mark.parametrize("kv8", [False, True])
def test_a_nan_in_a_row_that_nobody_sees_does_not_matter(fl, dev, kv8):
    """Behind the tree, ahead of the window, and of a page that is shared with other sequences."""
    g, T = gen(8), 12
    kp, vp, pages, _ = filled(fl, g, [400], 16, kv8)
    n_rows = kp.numel() // (4 * 272) if kv8 else kp.shape[0] * 16
    rows = ref.rows_of(pages.cpu(), 0, 16, torch.arange(400)).cuda()
    q, parents = randn(g, 1, T, 24, 512), i32(*tree(g, T, T)).view(1, T)
    call = lambda: fl.ops.attn_tree_paged(q, kp, vp, pages, i32(300), parents, page_size=16, window=50, sinks=3)
    want = call()
    depth = max(len(x) for x in tree_ref.lines(parents[0].tolist()))
    for pool in (kp, vp):
        spoil(pool, rows[list(range(3, 250)) + list(range(300 + T, 400))], n_rows, 4)
    assert depth < 50 and torch.equal(call(), want)


def test_strides_of_the_table_outputs_given_and_work(fl, dev):
    g, T = gen(9), 9
    kp, vp, pages, _ = filled(fl, g, [100, 64], 16, False)
    wide = torch.full((2, 40), 77, dtype=I32, device="cuda")
    wide[:, 5:5 + pages.shape[1]] = pages
    q, parents = randn(g, 2, T, 24, 512), torch.tensor([tree(g, T, T)] * 2, dtype=I32).cuda()
    want = fl.ops.attn_tree_paged(q, kp, vp, pages, i32(80, 50), parents, page_size=16)
    z = torch.full((2, T, 24, 264), 5.0, dtype=F16, device="cuda")
    work = torch.empty(fl.ops.attn_tree_paged_work_bytes(2, T), dtype=torch.uint8, device="cuda")
    r = fl.ops.attn_tree_paged(q, kp, vp, wide[:, 5:5 + pages.shape[1]], i32(80, 50), parents, page_size=16, z=z, work=work)
    assert r is z and torch.equal(z[..., :256], want) and (z[..., 256:] == 5).all()
    with pytest.raises(fl._lib.FlError, match="work"):
        fl.ops.attn_tree_paged(q, kp, vp, pages, i32(80, 50), parents, page_size=16, work=work[:64])


@pytest.mark.parametrize("kv8", [False, True])
def test_in_a_graph_at_other_positions_and_trees(fl, dev, kv8):
    g, T, B = gen(10), 24, 3
    kp, vp, pages, _ = filled(fl, g, [1500] * B, 32, kv8)
    q = randn(g, B, T, 24, 512)
    pos0, parents = i32(3, 4, 5), torch.tensor([tree(g, T, T)] * B, dtype=I32).cuda()
    z, work = torch.empty(B, T, 24, 256, dtype=F16, device="cuda"), torch.empty(
        fl.ops.attn_tree_paged_work_bytes(B, T), dtype=torch.uint8, device="cuda")
    call = lambda: fl.ops.attn_tree_paged(q, kp, vp, pages, pos0, parents, page_size=32, z=z, work=work)
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    other = torch.cuda.Stream()
    for step in range(4):
        pos0.copy_(torch.tensor([1400 - 400 * step, -1 if step == 2 else 7 * step, 100 * step], dtype=I32))
        parents.copy_(torch.tensor([tree(g, T - 5 * step - b, T) for b in range(B)], dtype=I32))
        q.mul_(-1.0)
        other.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(other):
            graph.replay()
        torch.cuda.current_stream().wait_stream(other)
        got = z.clone()
        assert torch.equal(got, fl.ops.attn_tree_paged(q, kp, vp, pages, pos0, parents, page_size=32))


def test_two_calls_at_once_on_two_streams(fl, dev):
    g, T = gen(11), 30
    kp, vp, pages, _ = filled(fl, g, [3000, 2000], 32, False)
    q, parents = randn(g, 2, T, 24, 512), torch.tensor([tree(g, T, T)] * 2, dtype=I32).cuda()
    pos = [i32(2900, 1500), i32(100, 1900)]
    call = lambda p: fl.ops.attn_tree_paged(q, kp, vp, pages, p, parents, page_size=32)
    want = [call(p) for p in pos]
    streams = [torch.cuda.Stream() for _ in pos]
    torch.cuda.synchronize()
    got = []
    for _ in range(5):
        for s, p in zip(streams, pos):
            with torch.cuda.stream(s):
                got.append(call(p))
    torch.cuda.synchronize()
    assert all(torch.equal(z, want[i % 2]) for i, z in enumerate(got))


@pytest.mark.parametrize("kv8", [False, True])
def test_a_round(fl, dev, kv8):
    """A tree prepared at its depths, attended to, its path kept: the same rows and outputs as the
    accepted tokens give when they are the sequence's, one behind the other."""
    g, T, P, ctx = gen(12), 13, 16, 75
    pages, n_pages = ref.make_pages(g, [ctx + T], P)
    pools = [fl.ops.paged_pool(n_pages, P, kv8=kv8) for _ in range(2)]
    wq, wk = (randn(g, 256, dtype=F32, scale=0.1) for _ in range(2))
    k, v = randn(g, ctx, 4, 256), randn(g, ctx, 4, 256)
    fl.ops.attn_prep_paged(randn(g, ctx, 24, 512), k, v, wq, wk, *pools, pages, i32(0, ctx), i32(0), page_size=P)
    again = [p.clone() for p in pools]
    parents = tree(g, T, T, "binary")
    depth = [len(x) - 1 for x in tree_ref.lines(parents)]
    qg, k, v = randn(g, T, 24, 512), randn(g, T, 4, 256), randn(g, T, 4, 256)
    q_out = qg.clone()
    fl.ops.attn_prep_axes(q_out, k, v, wq, wk, *pools, pages, i32(0, T), i32(ctx),
                          i32(*[ctx + d for d in depth]).view(1, T), page_size=P)
    z = fl.ops.attn_tree_paged(q_out[None], *pools, pages, i32(ctx), i32(*parents).view(1, T), page_size=P)
    path = [0, 2, 5, 11]
    fl.ops.paged_kv_keep(*pools, pages, i32(ctx), i32(*path, -1).view(1, 5), page_size=P)
    x = [t[path].contiguous() for t in (qg, k, v)]
    fl.ops.attn_prep_paged(*x, wq, wk, *again, pages, i32(0, 4), i32(ctx), page_size=P)
    kept = [fl.ops.paged_kv_load(*p, pages, i32(0, ctx + 4), i32(0), T=ctx + 4, page_size=P) for p in (pools, again)]
    for a, b in zip(*kept):
        assert torch.equal(a.view(torch.int16), b.view(torch.int16))
    want = fl.ops.attn_decode_paged(x[0][None], *again, pages, i32(ctx), page_size=P)[0]
    diff = (z[0, path].double() - want.double()).abs()
    assert (diff <= 2.0 ** -9 * want.abs().amax(-1, keepdim=True) + 2.0 ** -24).all()
