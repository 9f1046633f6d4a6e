"""The paged cache's part of a tree round on the GPU: prep with positions on several axes,
pages copied and accepted rows moved in the pools of several layers. Bit for bit against
this library's own prep and against indexing on the host; the rotation against float64."""
import math

import pytest
import torch

import paged_ref as ref
from test_gpu_paged import blank, gen, i32, randn, starts_of

pytestmark = pytest.mark.gpu

F16, F32, I32 = torch.float16, torch.float32, torch.int32


def bits(t):
    return t.view(torch.int8 if t.dtype == torch.int8 else torch.int16)


# ---------------------------------------------------------------------------
# prep
# ---------------------------------------------------------------------------

def prep_inputs(fl, seed, spans, page_size, kv8, pitch=512):
    g = gen(seed)
    N = sum(n for n, _ in spans)
    pages, n_pages = ref.make_pages(g, [p + n for n, p in spans], page_size)
    pools = [blank(fl, n_pages, page_size, kv8) for _ in range(2)]
    qg, k, v = randn(g, N, 24, pitch), randn(g, N, 4, 256), randn(g, N, 4, 256)
    wq, wk = (randn(g, 256, dtype=F32, scale=0.1) for _ in range(2))
    table = pages, starts_of([n for n, _ in spans]), i32(*[p for _, p in spans])
    return (qg, k, v, wq, wk), pools, table


SPANS = [[(1, 0)], [(5, 13), (0, 7), (40, 300)], [(300, 70)]]


@pytest.mark.parametrize("kv8", [False, True])
@pytest.mark.parametrize("axes,sections,interleaved", [
    (1, None, False), (3, (12, 10, 10), False), (3, (11, 11, 10), True), (2, (0, 32), False), (4, (8, 8, 8, 8), True)])
@pytest.mark.parametrize("spans", SPANS, ids=str)
def test_axes_that_hold_the_sequences_positions_give_the_plain_prep(fl, spans, axes, sections, interleaved, kv8):
    x, pools, table = prep_inputs(fl, 3, spans, 16, kv8)
    want = [p.clone() for p in pools]
    q_want = torch.empty(x[0].shape[0], 24, 256, dtype=F16, device="cuda")
    fl.ops.attn_prep_paged(x[0], *x[1:], *want, *table, page_size=16, q_out=q_want)
    pos = torch.cat([torch.arange(p, p + n, dtype=I32) for n, p in spans])
    q_out = torch.empty_like(q_want)
    qg = x[0].clone()
    r = fl.ops.attn_prep_axes(qg, *x[1:], *pools, *table, pos.expand(axes, -1).contiguous().cuda(),
                              page_size=16, sections=sections, interleaved=interleaved, q_out=q_out)
    assert r is q_out and torch.equal(qg, x[0])
    assert torch.equal(bits(q_out), bits(q_want))
    for a, b in zip(pools, want):
        assert torch.equal(bits(a), bits(b))
    # in place
    assert fl.ops.attn_prep_axes(qg, *x[1:], *pools, *table, pos.expand(axes, -1).contiguous().cuda(),
                                 page_size=16, sections=sections, interleaved=interleaved) is qg
    assert torch.equal(bits(qg[..., :256].contiguous()), bits(q_want))
    assert torch.equal(bits(qg[..., 256:].contiguous()), bits(x[0][..., 256:].contiguous()))


@pytest.mark.parametrize("N", [1, 3, 64, 257])
@pytest.mark.parametrize("sections,interleaved", [((16, 8, 8), False), ((11, 11, 10), True), ((32,), False),
                                                  ((1, 31), False), ((30, 1, 1), True)])
def test_every_pair_turns_by_its_own_axis(fl, N, sections, interleaved):
    """Against float64. One rounding a norm (half a step: 2^-11 of a value), one a rotation of two
    normed values (2^-11 of the result, and the operands' own 2^-11); cos and sin rounded to
    fp32 and the fp32 arithmetic are under 2^-20 of the operands: with |x| <= m in a row all in
    all 2^-11 (|y| + |cos a| + |sin b|) + 2^-20 m, doubled nowhere."""
    axes = len(sections)
    x, pools, (pages, starts, pos0) = prep_inputs(fl, 5, [(N, 40)], 32, False, pitch=256)
    g = gen(N)
    positions = torch.randint(-50, 100000, (axes, N), generator=g, dtype=I32)
    q_out = torch.empty(N, 24, 260, dtype=F16, device="cuda")
    fl.ops.attn_prep_axes(x[0], *x[1:], *pools, pages, starts, pos0, positions.cuda(), page_size=32,
                          sections=sections, interleaved=interleaved, q_out=q_out)
    owner = []
    for j in range(32):
        if interleaved:
            a = j % axes
            owner.append(a if j // axes < sections[a] else 0)
        else:
            owner.append(next(a for a in range(axes) if j < sum(sections[:a + 1])))
    host = pages.cpu()
    rows = ref.rows_of(host, 0, 32, torch.arange(40, 40 + N)).cuda()
    for got, src, w in ((q_out[..., :256], x[0], x[3]), (pools[0].view(-1, 4, 256)[rows], x[1], x[4])):
        t = src[..., :256].double()
        t = t / (t.square().mean(-1, keepdim=True) + 1e-6).sqrt() * (1 + w.double())
        want, slack = t.clone(), t.abs()
        for j, a in enumerate(owner):
            ang = positions[a].double() * 1e7 ** (-2 * j / 64)
            c, s = ang.cos().cuda()[:, None], ang.sin().cuda()[:, None]
            u, v = t[..., j], t[..., j + 32]
            want[..., j], want[..., j + 32] = u * c - v * s, v * c + u * s
            slack[..., j] = want[..., j].abs() + (u * c).abs() + (v * s).abs()
            slack[..., j + 32] = want[..., j + 32].abs() + (v * c).abs() + (u * s).abs()
        bound = slack * 2.0 ** -11 + 2.0 ** -20 * t.abs().amax(-1, keepdim=True)
        assert ((got.double() - want).abs() <= bound).all()
    assert torch.equal(bits(pools[1].view(-1, 4, 256)[rows]), bits(x[2]))


def test_axes_prep_in_a_graph_follows_positions(fl):
    x, pools, table = prep_inputs(fl, 9, [(20, 100), (9, 0)], 16, False)
    positions = torch.zeros(1, 29, dtype=I32, device="cuda")
    q_out = torch.empty(29, 24, 256, dtype=F16, device="cuda")
    call = lambda q, p: fl.ops.attn_prep_axes(*x, *p, *table, positions, page_size=16, q_out=q)
    call(q_out, pools)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(q_out, pools)
    for step in range(3):
        positions += 7 * step + 1
        graph.replay()
        want, wp = torch.empty_like(q_out), [p.clone() for p in pools]
        call(want, wp)
        torch.cuda.synchronize()
        assert torch.equal(q_out, want)


# ---------------------------------------------------------------------------
# pages, rows
# ---------------------------------------------------------------------------

def any_pools(g, n_pages, page_size, n_kv, kv8, layers):
    def one():
        if kv8:
            n = n_pages * page_size * n_kv * 272
            return torch.randint(-128, 128, (n,), generator=g, dtype=torch.int8).cuda()
        return torch.randint(-2**15, 2**15, (n_pages, page_size, n_kv, 256), generator=g,
                             dtype=torch.int16).cuda().view(F16)
    return [one() for _ in range(layers)], [one() for _ in range(layers)]


def rows_view(pool, n_rows, n_kv):
    """Two views of a pool's rows as bytes: values, scales (none over fp16)."""
    if pool.dtype == torch.int8:
        cut = n_rows * n_kv * 256
        return pool[:cut].view(n_rows, -1), pool[cut:].view(n_rows, -1)
    return (bits(pool).view(n_rows, -1),)


@pytest.mark.parametrize("kv8", [False, True])
@pytest.mark.parametrize("n_pages,page_size,n_kv,layers,n", [
    (5, 16, 4, 1, 1), (40, 16, 4, 16, 19), (9, 64, 1, 2, 4), (12, 32, 3, 3, 6), (7, 256, 4, 2, 3), (70, 16, 8, 64, 33)])
def test_pages_are_copied_in_every_layer(fl, n_pages, page_size, n_kv, layers, n, kv8):
    g = gen(n)
    ks, vs = any_pools(g, n_pages, page_size, n_kv, kv8, layers)
    order = torch.randperm(n_pages, generator=g)
    src, dst = order[:n].clone(), order[n_pages - n:].clone()
    left_out = n > 2
    if left_out:    # ids outside the pool
        src[0], dst[1] = -1, n_pages
    want = []
    for p in ks + vs:
        w = p.clone()
        for part in rows_view(w, n_pages * page_size, n_kv):
            part = part.view(n_pages, -1)
            for i in range(2 if left_out else 0, n):
                part[dst[i]] = part[src[i]]
        want.append(w)
    fl.ops.paged_kv_copy(ks, vs, src.to(I32).cuda(), dst.to(I32).cuda(), page_size=page_size, n_kv_heads=n_kv)
    for p, w in zip(ks + vs, want):
        assert torch.equal(bits(p), bits(w))


def test_a_single_pool_and_no_pages(fl):
    g = gen(1)
    (k,), (v,) = any_pools(g, 6, 16, 4, False, 1)
    before = k.clone()
    none = torch.empty(0, dtype=I32, device="cuda")
    fl.ops.paged_kv_copy(k, v, none, none, page_size=16)
    assert torch.equal(bits(k), bits(before))
    fl.ops.paged_kv_copy(k, v, i32(2, 4), i32(5, 4), page_size=16)   # (a page onto itself stays)
    assert torch.equal(bits(k[5]), bits(before[2])) and torch.equal(bits(k[:5]), bits(before[:5]))


def keep_want(pools, pages, pos0, path, page_size, n_pages, n_kv):
    want = [p.clone() for p in pools]
    table = pages.cpu()

    def at(b, p):
        if p < 0 or p // page_size >= table.shape[1]:
            return -1
        i = int(table[b, p // page_size])
        return i * page_size + p % page_size if 0 <= i < n_pages else -1
    for b, p0 in enumerate(pos0):
        last = -1
        for d, i in enumerate(path[b]):
            if i <= last or p0 < 0:
                break
            last = i
            src, dst = at(b, p0 + i), at(b, p0 + d)
            if src >= 0 and dst >= 0:
                for p, w in zip(pools, want):
                    for a, c in zip(rows_view(p, n_pages * page_size, n_kv), rows_view(w, n_pages * page_size, n_kv)):
                        c[dst] = a[src]
    return want


@pytest.mark.parametrize("kv8", [False, True])
@pytest.mark.parametrize("page_size,n_kv,layers,pos0,path", [
    (16, 4, 1, [13], [[0, 2, 3, 9]]),
    (16, 4, 16, [0, 30, 5, 47], [[1, 5, -1, -1], [0, 1, 2, 3], [-1, 3, 4, 5], [2, 2, 7, 9]]),
    (32, 3, 2, [31, -4], [[4, 9, 13], [1, 2, 3]]),
    (64, 8, 3, [60], [list(range(3, 33))]),
    (16, 1, 2, [0], [[0] + list(range(2, 32))]),
    (16, 4, 2, [100000], [[1, 3]]),            # (past the table)
    (16, 4, 2, [2**31 - 2], [[1, 3]]),
])
def test_accepted_rows_move_up(fl, page_size, n_kv, layers, pos0, path, kv8):
    g = gen(len(path[0]))
    lens = [(max(0, p) if p < 1000 else 40) + 64 for p in pos0]
    pages, n_pages = ref.make_pages(g, lens, page_size)
    if len(pos0) > 3:
        pages[3, (47 + 2) // 16] = -1          # an absent page
    ks, vs = any_pools(g, n_pages, page_size, n_kv, kv8, layers)
    want = keep_want(ks + vs, pages, pos0, path, page_size, n_pages, n_kv)
    fl.ops.paged_kv_keep(ks, vs, pages, i32(*pos0), torch.tensor(path, dtype=I32).cuda(), page_size=page_size,
                         n_kv_heads=n_kv)
    for p, w in zip(ks + vs, want):
        assert torch.equal(bits(p), bits(w))


def test_keep_and_copy_on_another_stream_and_in_a_graph(fl):
    g = gen(11)
    pages, n_pages = ref.make_pages(g, [100, 100], 16, spare=6)
    ks, vs = any_pools(g, n_pages, 16, 4, False, 3)
    pos0, path = i32(50, 20), torch.zeros(2, 4, dtype=I32, device="cuda")
    spare = [i for i in range(n_pages) if i not in pages.flatten().tolist()][:2]
    src, dst = pages[:, 0].contiguous(), i32(*spare)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        fl.ops.paged_kv_keep(ks, vs, pages, pos0, path, page_size=16)
        fl.ops.paged_kv_copy(ks, vs, src, dst, page_size=16)
    other = torch.cuda.Stream()
    for chosen in ([[0, 3, 5, -1], [2, 4, 6, 8]], [[1, -1, 0, 0], [0, 1, 2, 9]], [[-1] * 4, [5, 6, 7, 8]]):
        path.copy_(torch.tensor(chosen, dtype=I32))
        want = keep_want(ks + vs, pages, [50, 20], chosen, 16, n_pages, 4)
        for w in want:
            w.view(n_pages, -1)[spare] = w.view(n_pages, -1)[pages[:, 0].long().cpu()]
        other.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(other):
            graph.replay()
        torch.cuda.current_stream().wait_stream(other)
        for p, w in zip(ks + vs, want):
            assert torch.equal(bits(p), bits(w))
