"""The paged KV cache's operators on the GPU against the formulas in float64
(paged_ref.py, which derives the bounds), and the store, the read-back and the
prep bit for bit against this library's own contiguous operators."""
import pytest
import torch

import paged_ref as ref

pytestmark = pytest.mark.gpu

F16, F32, I32 = torch.float16, torch.float32, torch.int32
SCALE = 256 ** -0.5


def gen(seed):
    return torch.Generator().manual_seed(seed)


def randn(g, *shape, dtype=F16, scale=1.0):
    return (torch.randn(shape, generator=g) * scale).to(dtype).cuda()


def i32(*v):
    return torch.tensor(v, dtype=I32, device="cuda")


def starts_of(Ts):
    s = [0]
    for t in Ts:
        s.append(s[-1] + t)
    return i32(*s)


def blank(fl, n_pages, page_size, kv8, n_kv=4):
    """A pool whose unwritten rows are NaN (int8: scales of NaN)."""
    if not kv8:
        return torch.full((n_pages, page_size, n_kv, 256), float("nan"), dtype=F16, device="cuda")
    p = fl.ops.paged_pool(n_pages, page_size, kv8=True, n_kv_heads=n_kv)
    p[n_pages * page_size * n_kv * 256:].view(F16).fill_(float("nan"))
    return p


def values(pool, n_rows, n_kv):
    if pool.dtype == torch.int8:
        return ref.dequant(pool, n_rows, n_kv)
    return pool.view(n_rows, n_kv, 256)


def filled(fl, g, lens, page_size, kv8, n_kv=4):
    """Pools holding random rows of sequences of `lens` positions (NaN elsewhere):
    (kpool, vpool, pages, per-sequence K, V as the pool holds them)."""
    pages, n_pages = ref.make_pages(g, lens, page_size)
    kp, vp = (blank(fl, n_pages, page_size, kv8, n_kv) for _ in range(2))
    n = sum(lens)
    k, v = randn(g, n, n_kv, 256), randn(g, n, n_kv, 256)
    fl.ops.paged_kv_store(k, v, kp, vp, pages, starts_of(lens), torch.zeros(len(lens), dtype=I32, device="cuda"),
                          page_size=page_size, n_kv_heads=n_kv)
    host = pages.cpu()
    rows = [ref.rows_of(host, b, page_size, torch.arange(L)).cuda() for b, L in enumerate(lens)]
    kv, vv = (values(p, n_pages * page_size, n_kv) for p in (kp, vp))
    return kp, vp, pages, [(kv[r], vv[r]) for r in rows]


def seen_mask(n, p0, L, window, sinks, present=None):
    p = torch.arange(p0, p0 + n, device="cuda")[:, None]
    r = torch.arange(L, device="cuda")[None]
    s = r <= p
    if window:
        s &= (r > p - window) | (r < sinks)
    if present is not None:
        s &= present[None]
    return s


def check(z, want, bound, what):
    err = (z.double() - want).abs()
    assert torch.isfinite(z).all(), f"{what}: not finite"
    worst = (err / bound).max().item()
    print(f"{what}: max|err| {err.max().item():.2e}, {worst:.2f} of the bound")
    assert worst <= 1.0, f"{what}: {worst} of the bound, max|err| {err.max().item()}"


# ---------------------------------------------------------------------------
# store, load
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("kv8", [False, True])
@pytest.mark.parametrize("page_size,spans,n_kv", [
    (16, [(1, 0)], 4), (16, [(5, 13), (0, 7), (1, 16), (40, 0)], 4), (64, [(130, 60), (3, 1000)], 4),
    (256, [(1, 255)] * 70, 4), (32, [(37, 5), (64, 32)], 1), (16, [(9, 30)], 3), (128, [(700, 90)], 8),
])
def test_store_and_load(fl, dev, kv8, page_size, spans, n_kv):
    """Every stored row has the contiguous store's bits (kv_store / kv_store_q8), no
    other byte of the pools changes, and the read-back gives the rows' values."""
    g = gen(page_size + len(spans))
    ops = fl.ops
    Ts, p0s = [t for t, _ in spans], [p for _, p in spans]
    lens = [t + p for t, p in spans]
    N = sum(Ts)
    pages, n_pages = ref.make_pages(g, lens, page_size)
    k, v = randn(g, N + 2, n_kv, 256), randn(g, N + 2, n_kv, 256)
    k[0, 0, :32] = 0                                        # an all-zero block
    k[N - 1, n_kv - 1, 40] = 60000
    kp, vp = (blank(fl, n_pages, page_size, kv8, n_kv) for _ in range(2))
    before = kp.clone()
    table = (pages, starts_of(Ts), i32(*p0s))
    ops.paged_kv_store(k, v, kp, vp, *table, page_size=page_size, n_kv_heads=n_kv)
    rows = torch.cat([ref.rows_of(pages.cpu(), b, page_size, torch.arange(p, p + t))
                      for b, (t, p) in enumerate(spans)]).cuda()
    R = n_pages * page_size
    for x, pool in ((k[:N], kp), (v[:N], vp)):
        if kv8:
            dense = ops.kv8_cache(N, n_kv)
            other = ops.kv8_cache(N, n_kv)
            ops.kv_store_q8(x.contiguous(), x.contiguous(), dense, other, pos0=0, max_pos=N, n_kv_heads=n_kv)
            cut, dcut = R * n_kv * 256, N * n_kv * 256
            assert torch.equal(pool[:cut].view(R, -1)[rows], dense[:dcut].view(N, -1))
            assert torch.equal(pool[cut:].view(R, -1)[rows], dense[dcut:].view(N, -1))
        else:
            assert torch.equal(pool.view(R, n_kv, 256)[rows], x)
    mask = torch.ones(R, dtype=torch.bool, device="cuda")
    mask[rows] = False
    if kv8:
        cut = R * n_kv * 256
        for lo, hi in ((0, cut), (cut, None)):
            assert torch.equal(kp[lo:hi].view(R, -1)[mask], before[lo:hi].view(R, -1)[mask])
    else:
        assert torch.equal(kp.view(torch.int16).view(R, -1)[mask], before.view(torch.int16).view(R, -1)[mask])
    # back: new tensors have zeros behind the last sequence, given ones keep what they had
    k2, v2 = ops.paged_kv_load(kp, vp, *table, T=N + 2, page_size=page_size, n_kv_heads=n_kv)
    for x2, pool in ((k2, kp), (v2, vp)):
        assert torch.equal(x2[:N], values(pool, R, n_kv)[rows].to(F16)) and not x2[N:].any()
    ko, vo = torch.full_like(k2, 7.0), torch.full_like(v2, 7.0)
    ops.paged_kv_load(kp, vp, *table, T=N + 2, page_size=page_size, k=ko, v=vo, n_kv_heads=n_kv)
    assert torch.equal(ko[:N], k2[:N]) and bool((ko[N:] == 7).all()) and bool((vo[N:] == 7).all())


def test_int8_store_at_ties_and_non_finite_values(fl, dev):
    """The bytes and scales of kv_store_q8 where x / scale is a half integer, next to one,
    or not a number: blocks whose scale is a power of two (ties exact), every fp16 scale
    magnitude, subnormal blocks, infinities and NaN."""
    g, ops = gen(7), fl.ops
    N = 64
    x = torch.randn((N, 4, 8, 32), generator=g)
    for n in range(N):                                       # scale 2^(n % 24 - 20), ties below
        s = 2.0 ** (n % 24 - 20)
        if 127 * s <= 65504:
            x[n, 0] = (torch.randint(-127, 127, (8, 32), generator=g) + 0.5) * s
            x[n, 0, :, 0] = 127 * s
    x[:, 1] *= 10.0 ** (torch.rand((N, 8, 1), generator=g) * 9 - 6)
    x[0, 2, 0, 3], x[1, 2, 1, 4], x[2, 2, 2, 5] = float("inf"), float("nan"), -float("inf")
    x[3, 2, 3] = float("nan")
    x[4, 2, 4], x[5, 2, 5] = 0.0, 2.0 ** -24
    x = x.view(N, 4, 256).to(F16).cuda()
    kp, vp = (ops.paged_pool(4, 16, kv8=True) for _ in range(2))
    ops.paged_kv_store(x, x, kp, vp, i32(0, 1, 2, 3).view(1, 4), i32(0, N), i32(0), page_size=16)
    kc, vc = ops.kv8_cache(N), ops.kv8_cache(N)
    ops.kv_store_q8(x, x, kc, vc, pos0=0, max_pos=N)
    assert torch.equal(kp, kc) and torch.equal(vp, vc)


@pytest.mark.parametrize("kv8", [False, True])
def test_store_and_load_strided_absent_and_negative(fl, dev, kv8):
    """Token strides of a wider row, pages that are absent (negative, past the pool,
    past the table), and positions below zero."""
    g, ops, P = gen(3), fl.ops, 16
    wide = randn(g, 60, 3, 4, 256)
    k, v = wide[:, 0], wide[:, 2]
    pages = i32(2, -1, 0, 5, 4, 1000, 1, 3).view(2, 4)
    starts, pos0 = i32(0, 50, 60), i32(-3, 60)
    kp, vp = (ops.paged_pool(6, P, kv8=kv8) for _ in range(2))
    ops.paged_kv_store(k, v, kp, vp, pages, starts, pos0, page_size=P)
    k2 = torch.full((60, 4, 256), 9.0, dtype=F16, device="cuda")
    v2 = k2.clone()
    ops.paged_kv_load(kp, vp, pages, starts, pos0, T=60, page_size=P, k=k2, v=v2)
    # sequence 0: tokens 0-2 at negative positions; 3-18 page 2; 19-34 absent; 35-49 page 0
    # sequence 1 from position 60: 4 rows in page 3, the rest past the table
    want_rows = torch.zeros(60, dtype=torch.bool)
    want_rows[3:19] = want_rows[35:50] = want_rows[50:54] = True
    got = (k2 != 0).flatten(1).any(1).cpu()
    assert bool((k2[:3] == 9).all())                        # left as they were
    assert torch.equal(got[3:], want_rows[3:])
    for x, x2 in ((k, k2), (v, v2)):
        a, b = x[want_rows.cuda()].float(), x2[want_rows.cuda()].float()
        # int8: half a quantum of the block's scale, absmax / 127, and its roundings
        # (the scale's to fp16 moves the grid by 2^-11 of a value, the product's 2^-11)
        tol = a.abs().view(*a.shape[:-1], 8, 32).amax(-1, keepdim=True).expand(-1, -1, 8, 32).reshape(a.shape)
        assert bool(((a - b).abs() <= (tol * (0.5 / 127 + 2.0 ** -10) if kv8 else 0 * tol)).all())
    # the other pages stay empty
    left = values(kp, 6 * P, 4).view(6, P, -1)
    assert not left[1].any() and not left[4].any() and not left[5].any()


# ---------------------------------------------------------------------------
# prep
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("kv8", [False, True])
@pytest.mark.parametrize("spans", [[(1, 0)], [(1, 99999), (1, 5), (1, 70000)], [(40, 3), (0, 9), (230, 1000)]])
def test_prep_equals_the_contiguous_prep(fl, dev, kv8, spans):
    """q, k and v rows bit for bit those of attn_prep / attn_prep_q8 a sequence at a
    time; k is not rewritten; q_out and in place give the same rows."""
    g, ops, P = gen(len(spans)), fl.ops, 32
    Ts = [t for t, _ in spans]
    N = sum(Ts)
    # positions far out: only the pages that are written exist
    pages = torch.full((len(spans), max(t + p for t, p in spans) // P + 1), -1, dtype=I32)
    n = 0
    for b, (t, p) in enumerate(spans):
        for c in range(p // P, (t + p - 1) // P + 1 if t else p // P):
            pages[b, c] = n
            n += 1
    host, pages = pages, pages.cuda()
    kp, vp = (ops.paged_pool(n, P, kv8=kv8) for _ in range(2))
    qg, k, v = randn(g, N + 1, 24, 512), randn(g, N + 1, 4, 256), randn(g, N + 1, 4, 256)
    wq, wk = randn(g, 256, dtype=F32, scale=0.1), randn(g, 256, dtype=F32, scale=0.1)
    q_out = torch.full((N + 1, 24, 264), 5.0, dtype=F16, device="cuda")
    args = (wq, wk, kp, vp, pages, starts_of(Ts), i32(*[p for _, p in spans]))
    keep = qg.clone(), k.clone()
    ops.attn_prep_paged(qg, k, v, *args, page_size=P, q_out=q_out)
    assert torch.equal(qg, keep[0]) and torch.equal(k, keep[1])
    assert bool((q_out[N:] == 5).all()) and bool((q_out[..., 256:] == 5).all())
    ops.attn_prep_paged(qg, k, v, *args, page_size=P)
    assert torch.equal(qg[..., 256:], keep[0][..., 256:]) and torch.equal(k, keep[1])
    assert torch.equal(qg[:N, :, :256], q_out[:N, :, :256]) and torch.equal(qg[N], keep[0][N])
    at = 0
    for b, (t, p) in enumerate(spans):
        if t == 0:
            continue
        q1, k1, v1 = keep[0][at:at + t].clone(), k[at:at + t].clone(), v[at:at + t].clone()
        cap = p + t
        rows = ref.rows_of(host, b, P, torch.arange(p, p + t)).cuda()
        if kv8:
            kc, vc = ops.kv8_cache(cap), ops.kv8_cache(cap)
            ops.attn_prep_q8(q1, k1, v1, wq, wk, kc, vc, pos0=p, max_pos=cap)
        else:
            kc, vc = (torch.zeros((cap, 4, 256), dtype=F16, device="cuda") for _ in range(2))
            ops.attn_prep(q1, k1, v1, wq, wk, kc, vc, pos0=p)
        assert torch.equal(qg[at:at + t], q1)
        for pool, c in ((kp, kc), (vp, vc)):
            assert torch.equal(values(pool, n * P, 4)[rows].double(), values(c, cap, 4)[p:].double())
        at += t


@pytest.mark.parametrize("heads,rope_dim,N", [((6, 2), 32, 5), ((1, 1), 256, 3), ((24, 4), 128, 300),
                                              ((9, 3), 64, 270), ((40, 8), 2, 2)])
def test_prep_heads_and_rotations(fl, dev, heads, rope_dim, N):
    """Other head counts and rotary widths, one sequence: attn_prep's bits."""
    g, ops, P = gen(rope_dim), fl.ops, 16
    nq, nkv = heads
    p = 37
    pages, n_pages = ref.make_pages(g, [p + N], P)
    kp, vp = (ops.paged_pool(n_pages, P, n_kv_heads=nkv) for _ in range(2))
    qg, k, v = randn(g, N, nq, 264), randn(g, N, nkv, 256), randn(g, N, nkv, 256)
    wq, wk = randn(g, 256, dtype=F32, scale=0.1), randn(g, 256, dtype=F32, scale=0.1)
    q1, k1 = qg.clone(), k.clone()
    kc, vc = (torch.zeros((p + N, nkv, 256), dtype=F16, device="cuda") for _ in range(2))
    ops.attn_prep(q1, k1, v, wq, wk, kc, vc, pos0=p, n_q_heads=nq, n_kv_heads=nkv, q_pitch=264,
                  rope_dim=rope_dim)
    ops.attn_prep_paged(qg, k, v, wq, wk, kp, vp, pages, i32(0, N), i32(p), page_size=P, n_q_heads=nq,
                        n_kv_heads=nkv, rope_dim=rope_dim)
    rows = ref.rows_of(pages.cpu(), 0, P, torch.arange(p, p + N)).cuda()
    assert torch.equal(qg, q1)
    for pool, c in ((kp, kc), (vp, vc)):
        assert torch.equal(values(pool, n_pages * P, nkv)[rows], c[p:])


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------

def run_prefill(fl, seed, spans, page_size, kv8, window=0, sinks=0, heads=(24, 4), gated=True, extra=0,
                q_scale=1.0, absent=()):
    g = gen(seed)
    Hq, n_kv = heads
    lens = [t + p for t, p in spans]
    kp, vp, pages, caches = filled(fl, g, lens, page_size, kv8, n_kv)
    present = [torch.ones(L, dtype=torch.bool, device="cuda") for L in lens]
    for b, c, value in absent:
        pages[b, c] = value
        present[b][c * page_size:(c + 1) * page_size] = False
    Ts, p0s = [t for t, _ in spans], [p for _, p in spans]
    N = sum(Ts)
    qg = randn(g, N + extra, Hq, 512, scale=q_scale)
    z = torch.full((N + extra, Hq, 256), 3.0, dtype=F16, device="cuda")
    fl.ops.attention_prefill_paged(qg, kp, vp, pages, Ts, p0s, page_size=page_size, window=window,
                                   sinks=sinks, gated=gated, z=z, n_kv_heads=n_kv)
    assert bool((z[N:] == 3).all()), "rows behind the last chunk"
    at = 0
    for b, (t, p) in enumerate(spans):
        if t == 0:
            continue
        seen = seen_mask(t, p, lens[b], window, sinks, present[b])
        q = qg[at:at + t]
        want, bound = ref.attention(q[..., :256], *caches[b], p, seen, SCALE, kv8,
                                    q[..., 256:] if gated else None)
        blind = ~seen.any(-1)
        assert not z[at:at + t][blind].any(), "a query that sees no row gives 0"
        check(z[at:at + t], want, bound, f"sequence {b} ({t}@{p})")
        at += t


PREFILLS = [
    ([(1, 0)], 16), ([(2, 0), (1, 1)], 16), ([(33, 0)], 32), ([(31, 17), (0, 5), (1, 32), (65, 63)], 16),
    ([(300, 0)], 64), ([(257, 1000), (3, 511)], 128), ([(42, 2000), (43, 1999)], 256), ([(700, 345)], 16),
    ([(5, 4090)] * 9, 64), ([(1, 700)] * 64, 32), ([(1100, 900)], 64),
]


@pytest.mark.parametrize("kv8", [False, True])
@pytest.mark.parametrize("spans,page_size", PREFILLS, ids=str)
def test_prefill(fl, dev, spans, page_size, kv8):
    run_prefill(fl, 11, spans, page_size, kv8, extra=2)


@pytest.mark.parametrize("kv8", [False, True])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 4), (100, 0), (33, 40), (1000, 3), (5000, 7),
                                          (64, 64), (250, 1000)])
def test_prefill_window_and_sinks(fl, dev, window, sinks, kv8):
    run_prefill(fl, window, [(260, 0), (70, 777), (1, 900), (130, 100)], 32, kv8, window, sinks)


@pytest.mark.parametrize("heads", [(1, 1), (4, 4), (8, 1), (32, 8), (6, 2), (64, 2), (3, 3), (40, 1), (16, 16),
                                   (300, 1)])
def test_prefill_heads(fl, dev, heads):
    run_prefill(fl, 5, [(70, 130), (9, 0)], 16, False, heads=heads)
    run_prefill(fl, 6, [(33, 300)], 64, True, 50, 2, heads=heads, gated=False)


@pytest.mark.parametrize("kv8", [False, True])
def test_prefill_peaked_scores(fl, dev, kv8):
    """Scores of standard deviation 4: the running maximum moves often."""
    run_prefill(fl, 8, [(200, 300)], 32, kv8, q_scale=4.0)


@pytest.mark.parametrize("kv8", [False, True])
@pytest.mark.parametrize("page_size", [16, 32, 64])
def test_prefill_absent_pages(fl, dev, kv8, page_size):
    """Absent pages (negative, past the pool) inside, before and after the visible
    rows; all of a query's rows absent."""
    spans = [(100, 200), (20, 3), (4, 130)]
    absent = [(0, 0, -1), (0, 3, 1 << 20), (0, 5, -7)] + [(1, 0, -1), (1, 1, 999999)] + \
        [(2, c, -1) for c in range((134 + page_size - 1) // page_size)]
    absent = [a for a in absent if a[1] * page_size < [300, 23, 134][a[0]]]
    run_prefill(fl, 21, spans, page_size, kv8, absent=absent)
    run_prefill(fl, 22, spans, page_size, kv8, 40, 5, absent=absent)


def test_prefill_int8_copies_in_groups(fl, dev):
    """int8 contexts whose fp16 copies pass 1 GiB together: the call runs them in groups
    over one work buffer of that size."""
    lens, P = [100000, 99000, 98500, 70], 256
    g, ops = gen(23), fl.ops
    pages, n_pages = ref.make_pages(g, lens, P)
    kp, vp = (ops.paged_pool(n_pages, P, kv8=True) for _ in range(2))
    cut = n_pages * P * 1024
    for pool in (kp, vp):
        pool[:cut].random_(-127, 128)
        pool[cut:].view(F16).fill_(0.01).mul_(1 + torch.rand(1, device="cuda").half())
    Ts = [3, 1, 20, 70]
    p0s = [L - t for L, t in zip(lens, Ts)]
    need = ops.attention_prefill_paged_work_bytes(Ts, p0s, kv8=True)
    assert (1 << 29) < need < (1 << 30) + (200 << 20)
    qg = randn(g, sum(Ts), 24, 512)
    z = ops.attention_prefill_paged(qg, kp, vp, pages, Ts, p0s, page_size=P, gated=True)
    K, V = (ref.dequant(pool, n_pages * P, 4) for pool in (kp, vp))
    at = 0
    for b, (t, L) in enumerate(zip(Ts, lens)):
        rows = ref.rows_of(pages.cpu(), b, P, torch.arange(L)).cuda()
        want, bound = ref.attention(qg[at:at + t, :, :256], K[rows], V[rows], L - t,
                                    seen_mask(t, L - t, L, 0, 0), SCALE, True, qg[at:at + t, :, 256:])
        check(z[at:at + t], want, bound, f"sequence {b}")
        at += t


def test_table_of_a_wider_one(fl, dev):
    """A column slice of a wider table: its row stride is taken."""
    g = gen(24)
    kp, vp, pages, caches = filled(fl, g, [100, 40], 16, False)
    wide = torch.full((2, pages.shape[1] + 5), 10 ** 6, dtype=I32, device="cuda")
    wide[:, 2:2 + pages.shape[1]] = pages
    part = wide[:, 2:2 + pages.shape[1]]
    qg = randn(g, 2, 1, 24, 512)
    pos = i32(99, 39)
    assert torch.equal(fl.ops.attn_decode_paged(qg, kp, vp, part, pos, page_size=16),
                       fl.ops.attn_decode_paged(qg, kp, vp, pages, pos, page_size=16))
    args = dict(page_size=16, gated=True)
    assert torch.equal(fl.ops.attention_prefill_paged(qg[:, 0], kp, vp, part, [1, 1], [99, 39], **args),
                       fl.ops.attention_prefill_paged(qg[:, 0], kp, vp, pages, [1, 1], [99, 39], **args))
    for a, b in zip(fl.ops.paged_kv_load(kp, vp, part, i32(0, 9, 12), i32(5, 30), T=12, page_size=16),
                    fl.ops.paged_kv_load(kp, vp, pages, i32(0, 9, 12), i32(5, 30), T=12, page_size=16)):
        assert torch.equal(a, b)


def run_decode(fl, seed, lens, page_size, kv8, T=1, window=0, sinks=0, heads=(24, 4), gate=True, q_scale=1.0,
               absent=(), pad=0):
    """lens: each sequence's rows, its T tokens' own included (below T: the first
    tokens are at negative positions)."""
    g = gen(seed)
    Hq, n_kv = heads
    kp, vp, pages, caches = filled(fl, g, lens, page_size, kv8, n_kv)
    present = [torch.ones(L, dtype=torch.bool, device="cuda") for L in lens]
    for b, c, value in absent:
        pages[b, c] = value
        present[b][c * page_size:(c + 1) * page_size] = False
    pos0 = [L - T for L in lens]
    qg = randn(g, len(lens), T, Hq, 512 + pad, scale=q_scale)
    z = fl.ops.attn_decode_paged(qg, kp, vp, pages, i32(*pos0), page_size=page_size, window=window,
                                 sinks=sinks, gate=gate, n_kv_heads=n_kv)
    for b, L in enumerate(lens):
        seen = seen_mask(T, pos0[b], L, window, sinks, present[b])
        want, bound = ref.attention(qg[b][..., :256], *caches[b], pos0[b], seen, SCALE, kv8,
                                    qg[b][..., 256:512] if gate else None)
        assert not z[b][~seen.any(-1)].any(), "a query that sees no row gives 0"
        check(z[b], want, bound, f"sequence {b} (length {L}, T {T})")


@pytest.mark.parametrize("kv8", [False, True])
@pytest.mark.parametrize("lens,page_size,T", [
    ([1], 16, 1), ([2, 1, 3], 16, 2), ([17, 16, 15, 31, 32, 33], 16, 1), ([500], 16, 1),
    ([4096, 1, 777], 64, 1), ([1000, 64, 65], 32, 4), ([3001, 2999], 128, 3), ([257] * 70, 256, 1),
    ([9000, 50], 64, 1), ([3], 16, 4),
], ids=str)
def test_decode(fl, dev, lens, page_size, T, kv8):
    run_decode(fl, 31, lens, page_size, kv8, T)


@pytest.mark.parametrize("kv8", [False, True])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 2), (16, 4), (100, 0), (33, 40), (2000, 3), (64, 64),
                                          (250, 1000)])
@pytest.mark.parametrize("T", [1, 3])
def test_decode_window_and_sinks(fl, dev, window, sinks, kv8, T):
    run_decode(fl, 41, [1500, 40, 3, 290], 32, kv8, T, window, sinks)


@pytest.mark.parametrize("heads,T", [((1, 1), 1), ((1, 1), 32), ((8, 1), 4), ((32, 8), 3), ((6, 2), 2),
                                     ((64, 2), 1), ((3, 3), 1), ((16, 16), 2)])
def test_decode_heads(fl, dev, heads, T):
    run_decode(fl, 51, [100, 333, 32], 16, False, T, heads=heads, pad=8)
    run_decode(fl, 52, [444, 60], 64, True, T, 50, 2, heads=heads, gate=False)


@pytest.mark.parametrize("kv8", [False, True])
@pytest.mark.parametrize("heads,T,B,window", [((24, 4), 1, 64, 0), ((8, 8), 2, 40, 0), ((4, 2), 1, 150, 0),
                                              ((3, 3), 1, 90, 0), ((24, 4), 3, 64, 0), ((8, 4), 1, 130, 1500)])
def test_decode_many_long_contexts(fl, dev, heads, T, B, window, kv8):
    """Batches that give every run many tiles: sequences of unlike lengths over shared
    pages (one prefix of all, as long as the longest)."""
    g = gen(65 + B)
    L, page_size, (n_q, n_kv) = 2200, 32, heads
    kp, vp, pages, [(K, V)] = filled(fl, g, [L], page_size, kv8, n_kv)
    lens = [int(x) for x in torch.randint(1900, L + 1, (B,), generator=g)]
    qg = randn(g, B, T, n_q, 512)
    z = fl.ops.attn_decode_paged(qg, kp, vp, pages.repeat(B, 1), i32(*[n - T for n in lens]),
                                 page_size=page_size, n_kv_heads=n_kv, window=window)
    for b in range(0, B, 7):
        n = lens[b]
        want, bound = ref.attention(qg[b, :, :, :256], K[:n], V[:n], None,
                                    seen_mask(T, n - T, n, window, 0), SCALE, kv8, qg[b, :, :, 256:])
        check(z[b], want, bound, f"sequence {b}")


@pytest.mark.parametrize("kv8", [False, True])
def test_decode_peaked_scores(fl, dev, kv8):
    run_decode(fl, 61, [2000, 300], 32, kv8, 2, q_scale=4.0)


@pytest.mark.parametrize("kv8", [False, True])
@pytest.mark.parametrize("page_size", [16, 32, 64])
def test_decode_absent_pages(fl, dev, kv8, page_size):
    lens = [300, 23, 134, 1200]
    absent = [(0, 0, -1), (0, 3, 1 << 20), (0, 4, -7), (1, 0, -1), (1, 1, 99999)] + \
        [(2, c, -1) for c in range((134 + page_size - 1) // page_size)] + [(3, 7, -1)]
    absent = [a for a in absent if a[1] * page_size < lens[a[0]]]
    for T in (1, 3):
        run_decode(fl, 71, lens, page_size, kv8, T, absent=absent)
        run_decode(fl, 72, lens, page_size, kv8, T, 90, 5, absent=absent)


def test_decode_padded_batch(fl, dev):
    """A padded row: position -1 (T = 1), an all -1 table; its output is 0, and a
    sequence's result is the same bits as with another padded neighbour."""
    g = gen(81)
    kp, vp, pages, caches = filled(fl, g, [200, 16], 16, False)
    pages[1] = -1
    qg = randn(g, 2, 1, 24, 512)
    z = fl.ops.attn_decode_paged(qg, kp, vp, pages, i32(199, -1), page_size=16)
    assert not z[1].any() and torch.isfinite(z).all()
    z2 = fl.ops.attn_decode_paged(qg, kp, vp, pages, i32(199, -2147483648), page_size=16)
    assert torch.equal(z, z2)
    # past the table: the rows that the table has are seen, nothing else is read
    z3 = fl.ops.attn_decode_paged(qg, kp, vp, pages, i32(207, 2147483647), page_size=16)
    assert torch.isfinite(z3[1]).all() and not z3[1].any()


# ---------------------------------------------------------------------------
# together, graphs, streams, far rows
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("kv8", [False, True])
def test_a_prompt_and_its_decode_steps(fl, dev, kv8):
    """Prep, chunks and decode steps of three sequences over one pool against the
    contiguous operators on a cache each, and the read-back of what was cached."""
    g, ops, P = gen(91), fl.ops, 64
    prompts, steps = [300, 45, 130], 3
    total = [n + steps for n in prompts]
    pages, n_pages = ref.make_pages(g, total, P)
    kp, vp = (ops.paged_pool(n_pages, P, kv8=kv8) for _ in range(2))
    wq, wk = randn(g, 256, dtype=F32, scale=0.1), randn(g, 256, dtype=F32, scale=0.1)
    feeds = [(randn(g, L, 24, 512), randn(g, L, 4, 256), randn(g, L, 4, 256)) for L in total]
    dense = []
    for (qg, k, v), L in zip(feeds, total):
        q1, k1, v1 = qg.clone(), k.clone(), v.clone()
        if kv8:
            kc, vc = ops.kv8_cache(L), ops.kv8_cache(L)
            ops.attn_prep_q8(q1, k1, v1, wq, wk, kc, vc, pos0=0, max_pos=L)
            z = ops.attention_prefill_q8(q1, kc, vc, pos0=0, max_pos=L, gated=True)
        else:
            kc, vc = (torch.zeros((L, 4, 256), dtype=F16, device="cuda") for _ in range(2))
            ops.attn_prep(q1, k1, v1, wq, wk, kc, vc, pos0=0)
            z = ops.attention_prefill(q1, kc, vc, pos0=0, gated=True)
        dense.append((z, kc, vc))
    got = [[] for _ in prompts]
    done = [0, 0, 0]
    for chunk in (128, 128, 128):                           # the prompts in sub-chunks
        Ts = [min(chunk, n - d) for n, d in zip(prompts, done)]
        qg, k, v = (torch.cat([f[i][d:d + t] for f, d, t in zip(feeds, done, Ts)]) for i in range(3))
        ops.attn_prep_paged(qg, k, v, wq, wk, kp, vp, pages, starts_of(Ts), i32(*done), page_size=P)
        z = ops.attention_prefill_paged(qg, kp, vp, pages, Ts, done, page_size=P, gated=True)
        for b, part in enumerate(z.split(Ts)):
            got[b].append(part)
        done = [d + t for d, t in zip(done, Ts)]
    for _ in range(steps):
        qg, k, v = (torch.stack([f[i][d] for f, d in zip(feeds, done)]) for i in range(3))
        ops.attn_prep_paged(qg, k, v, wq, wk, kp, vp, pages, starts_of([1, 1, 1]), i32(*done), page_size=P)
        z = ops.attn_decode_paged(qg.unsqueeze(1), kp, vp, pages, i32(*done), page_size=P)
        for b in range(3):
            got[b].append(z[b])
        done = [d + 1 for d in done]
    for b, (want, kc, vc) in enumerate(dense):
        # both sides are within the attention bar of the formula (2e-3, 1e-2)
        torch.testing.assert_close(torch.cat(got[b]), want, atol=4e-3, rtol=2e-2)
        L = total[b]
        k2, v2 = ops.paged_kv_load(kp, vp, pages[b:b + 1], i32(0, L), i32(0), T=L, page_size=P)
        assert torch.equal(k2, values(kc, L, 4).to(F16)) and torch.equal(v2, values(vc, L, 4).to(F16))


@pytest.mark.parametrize("kv8", [False, True])
def test_a_captured_step_replays_at_new_positions(fl, dev, kv8):
    """Prep, decode and read-back captured once; replays after the positions, the
    inputs and the table changed equal the eager calls, with eager work of the same
    kind between them. Two graphs with work buffers of their own."""
    g, ops, P, B = gen(101), fl.ops, 32, 5
    lens = [700, 33, 64, 1, 2000]
    kp, vp, pages, _ = filled(fl, g, [L + 8 for L in lens], P, kv8)
    wq, wk = randn(g, 256, dtype=F32, scale=0.1), randn(g, 256, dtype=F32, scale=0.1)
    qg, k, v = randn(g, B, 24, 512), randn(g, B, 4, 256), randn(g, B, 4, 256)
    q = torch.zeros((B, 24, 512), dtype=F16, device="cuda")
    pos, starts = i32(*lens), starts_of([1] * B)

    def step():
        q.copy_(qg)
        ops.attn_prep_paged(q, k, v, wq, wk, kp, vp, pages, starts, pos, page_size=P)
        z = ops.attn_decode_paged(q.unsqueeze(1), kp, vp, pages, pos, page_size=P, window=600, sinks=4)
        return z, *ops.paged_kv_load(kp, vp, pages, starts, pos, T=B, page_size=P)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = step()
        graphs.append((gr, out))
    for i in range(6):
        qg.copy_(randn(g, B, 24, 512)), k.copy_(randn(g, B, 4, 256))
        pos.copy_(i32(*[L + i for L in lens]) if i != 4 else i32(-1, 3, 10, 5, 1999))
        gr, out = graphs[i % 2]
        gr.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        want = step()
        torch.cuda.synchronize()
        if i == 4:   # the row at position -1 is not read back
            got[1][0], got[2][0], want[1][0], want[2][0] = 0, 0, 0, 0
        for a, b in zip(got, want):
            assert torch.equal(a, b), i


@pytest.mark.parametrize("kv8", [False, True])
def test_captured_chunks_replay_over_new_rows(fl, dev, kv8):
    """Chunks of three sequences, some cut between workgroups, captured once; replays
    after the queries, the cached rows and the table changed equal the eager calls."""
    g, ops, P = gen(105), fl.ops, 32
    Ts, p0s = [200, 3, 70], [1500, 700, 0]
    lens = [t + p for t, p in zip(Ts, p0s)]
    kp, vp, pages, _ = filled(fl, g, lens, P, kv8)
    qg = randn(g, sum(Ts), 24, 512)
    tables = [pages.clone(), pages.clone()]
    tables[1][0, 3] = -1
    tables[1][0, 5:9] = pages[0, 5:9].flip(0)
    call = lambda: ops.attention_prefill_paged(qg, kp, vp, pages, Ts, p0s, page_size=P, gated=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        out = call()
    for i in range(4):
        qg.copy_(randn(g, sum(Ts), 24, 512))
        pages.copy_(tables[i % 2])
        rows = randn(g, lens[1], 4, 256)
        ops.paged_kv_store(rows, rows, kp, vp, pages[1:2], i32(0, lens[1]), i32(0), page_size=P)
        gr.replay()
        torch.cuda.synchronize()
        got, want = out.clone(), call()
        torch.cuda.synchronize()
        assert torch.isfinite(got).all() and torch.equal(got, want), i


@pytest.mark.parametrize("kv8", [False, True])
def test_decode_of_as_many_sequences_as_a_call_takes(fl, dev, kv8):
    """1024 sequences, a few rows each and some without any; then none with a row."""
    g, P, B = gen(106), 16, 1024
    lens = [int(x) for x in torch.randint(0, 60, (B,), generator=g)]
    kp, vp, pages, caches = filled(fl, g, lens, P, kv8)
    qg = randn(g, B, 1, 24, 512)
    z = fl.ops.attn_decode_paged(qg, kp, vp, pages, i32(*[n - 1 for n in lens]), page_size=P)
    for b in range(0, B, 31):
        if lens[b] == 0:
            assert not z[b].any()
            continue
        want, bound = ref.attention(qg[b, :, :, :256], *caches[b], None, seen_mask(1, lens[b] - 1, lens[b], 0, 0),
                                    SCALE, kv8, qg[b, :, :, 256:])
        check(z[b], want, bound, f"sequence {b} of {lens[b]} rows")
    empty = torch.tensor([n == 0 for n in lens], device="cuda")
    assert empty.any() and not z[empty].any()
    z = fl.ops.attn_decode_paged(qg, kp, vp, pages, i32(*([-1] * B)), page_size=P)
    assert not z.any()
    with pytest.raises((ValueError, fl._lib.FlError)):
        fl.ops.attn_decode_paged(torch.cat([qg, qg[:1]]), kp, vp, torch.cat([pages, pages[:1]]),
                                 i32(*([0] * (B + 1))), page_size=P)


def test_calls_on_two_streams(fl, dev):
    """Two decode and two prefill calls at once on streams of their own."""
    g = gen(111)
    sets = [filled(fl, g, [900, 120], 32, False) for _ in range(2)]
    qg = [randn(g, 2, 1, 24, 512) for _ in range(2)]
    qc = [randn(g, 120, 24, 512) for _ in range(2)]
    def both(i):
        kp, vp, pages, _ = sets[i]
        return (fl.ops.attn_decode_paged(qg[i], kp, vp, pages, i32(899, 119), page_size=32),
                fl.ops.attention_prefill_paged(qc[i], kp, vp, pages, [100, 20], [800, 100], page_size=32))
    want = [both(i) for i in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(3):
        got = [None, None]
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = both(i)
        torch.cuda.synchronize()
        for w, x in zip(want, got):
            assert torch.equal(w[0], x[0]) and torch.equal(w[1], x[1])


def test_calls_from_two_threads(fl, dev):
    """Two threads, each on a stream of its own, with chunks whose plans replace each
    other's in the library's cache."""
    import threading
    g = gen(113)
    sets = [filled(fl, g, [900, 120], 32, bool(i)) for i in range(2)]
    qg = [randn(g, 2, 1, 24, 512) for _ in range(2)]
    qc = [randn(g, 120, 24, 512) for _ in range(2)]
    pos = i32(899, 119)

    def once(i, n):
        kp, vp, pages, _ = sets[i]
        t = 60 + n % 11
        return (fl.ops.attn_decode_paged(qg[i], kp, vp, pages, pos, page_size=32),
                fl.ops.attention_prefill_paged(qc[i][:t + 20], kp, vp, pages, [t, 20], [800, 100], page_size=32))

    want = [[once(i, n) for n in range(11)] for i in range(2)]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for n in range(44):
                    got = once(i, n)
                    torch.cuda.current_stream().synchronize()
                    if not all(torch.equal(a, b) for a, b in zip(got, want[i][n % 11])):
                        wrong.append((i, n))
        except Exception as e:
            wrong.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not wrong, wrong


@pytest.mark.parametrize("kv8", [False, True])
def test_rows_past_4_gib(fl, dev, kv8):
    """Pages whose rows lie past 2^32 bytes of the pool."""
    P, ops = 256, fl.ops
    n_pages = (1 << 32) // (P * 4 * (256 if kv8 else 512)) + 40
    kp, vp = (ops.paged_pool(n_pages, P, kv8=kv8) for _ in range(2))
    g = gen(121)
    L = 900
    pages = i32(n_pages - 1, 3, n_pages - 7, n_pages - 2).view(1, 4)
    k, v = randn(g, L, 4, 256), randn(g, L, 4, 256)
    ops.paged_kv_store(k, v, kp, vp, pages, i32(0, L), i32(0), page_size=P)
    k2, v2 = ops.paged_kv_load(kp, vp, pages, i32(0, L), i32(0), T=L, page_size=P)
    if not kv8:
        assert torch.equal(k2, k) and torch.equal(v2, v)
    seen = seen_mask(60, L - 60, L, 0, 0)
    qg = randn(g, 60, 24, 512)
    # (int8: the read-back rounds byte * scale to fp16, as the kernels do)
    z = ops.attention_prefill_paged(qg, kp, vp, pages, [60], [L - 60], page_size=P)
    want, bound = ref.attention(qg[..., :256], k2, v2, L - 60, seen, SCALE)
    check(z, want, bound, "prefill")
    z = ops.attn_decode_paged(qg[-1:].unsqueeze(0), kp, vp, pages, i32(L - 1), page_size=P, gate=False)
    check(z[0], want[-1:], bound[-1:], "decode")


def test_refusals_on_the_gpu(fl, dev):
    """What the op layer refuses of GPU tensors: nothing is launched."""
    ops = fl.ops
    kp = ops.paged_pool(4, 16)
    pages, starts, pos0 = i32(0, 1, 2, 3).view(1, 4), i32(0, 3), i32(0)
    k = torch.zeros((3, 4, 256), dtype=F16, device="cuda")
    qg = torch.zeros((1, 1, 24, 512), dtype=F16, device="cuda")
    with pytest.raises(TypeError):
        ops.paged_kv_store(k.float(), k, kp, kp, pages, starts, pos0, page_size=16)
    with pytest.raises(TypeError):
        ops.paged_kv_store(k, k, kp, kp, pages.long(), starts, pos0, page_size=16)
    with pytest.raises(TypeError):
        ops.attn_decode_paged(qg, kp, kp, pages, pos0.long(), page_size=16)
    with pytest.raises(ValueError):
        ops.paged_kv_store(k.transpose(1, 2), k, kp, kp, pages, starts, pos0, page_size=16)
    with pytest.raises(ValueError):
        ops.paged_kv_store(k, k[:2], kp, kp, pages, starts, pos0, page_size=16)
    with pytest.raises(ValueError):
        ops.attn_decode_paged(qg, kp[:, ::2], kp, pages, pos0, page_size=16)
    with pytest.raises(ValueError):
        ops.attention_prefill_paged(qg[0], kp, kp, pages, [1], [64], page_size=16)
    with pytest.raises(ValueError):
        ops.attn_decode_paged(qg, kp, kp, pages, pos0, page_size=16, window=-1)


@pytest.mark.parametrize("kv8", [False, True])
def test_binding_and_ctypes_make_the_same_calls(fl, dev, kv8, monkeypatch):
    """Every operator through the compiled binding and, with it out of the way, through
    the Python checks and ctypes: the same bits, given and new outputs, and the same
    refusals."""
    ops, P = fl.ops, 32
    fl._lib.lib()
    assert fl._lib.lane is not None, "fl355_paged.so is not built"
    g = gen(141)
    lens = [100, 1, 333]
    Ts = [3, 1, 5]
    p0 = [n - t for n, t in zip(lens, Ts)]
    pages, n_pages = ref.make_pages(g, lens, P)
    x = {n: randn(g, 9, h, w) for n, h, w in (("k", 4, 256), ("v", 4, 256), ("qg", 24, 512))}
    wq, wk = randn(g, 256, dtype=F32, scale=0.1), randn(g, 256, dtype=F32, scale=0.1)
    rows = randn(g, sum(lens), 4, 256)
    starts, pos0 = starts_of(Ts), i32(*p0)

    def calls():
        kp, vp = (ops.paged_pool(n_pages, P, kv8=kv8) for _ in range(2))
        ops.paged_kv_store(rows, rows, kp, vp, pages, starts_of(lens), i32(0, 0, 0), page_size=P)
        q = x["qg"].clone()
        out = torch.zeros(9, 24, 512, dtype=F16, device="cuda")
        same = ops.attn_prep_paged(q, x["k"], x["v"], wq, wk, kp, vp, pages, starts, pos0, page_size=P)
        other = ops.attn_prep_paged(x["qg"], x["k"], x["v"], wq, wk, kp, vp, pages, starts, pos0, page_size=P,
                                    q_out=out)
        assert same is q and other is out
        got = list(ops.paged_kv_load(kp, vp, pages, starts_of(lens), i32(0, 0, 0), T=sum(lens) + 1, page_size=P))
        z = torch.full((9, 24, 300), 5.0, dtype=F16, device="cuda")
        work = torch.empty(ops.attention_prefill_paged_work_bytes(Ts, p0, kv8=kv8), dtype=torch.uint8,
                           device="cuda")
        assert ops.attention_prefill_paged(q, kp, vp, pages, Ts, p0, page_size=P, gated=True, z=z,
                                           work=work) is z
        got += [q, out, z, ops.attention_prefill_paged(q, kp, vp, pages, tuple(Ts), p0, page_size=P, window=20,
                                                       sinks=2),
                ops.attention_prefill_paged(q, kp, vp, pages, [3, 0, 5], p0, page_size=P)]
        qd = x["qg"][:6].view(3, 2, 24, 512)
        zd = torch.full((3, 2, 24, 256), 5.0, dtype=F16, device="cuda")
        work = torch.empty(ops.attn_decode_paged_work_bytes(3, 2), dtype=torch.uint8, device="cuda")
        assert ops.attn_decode_paged(qd, kp, vp, pages, pos0, page_size=P, z=zd, work=work) is zd
        return got + [zd, ops.attn_decode_paged(qd, kp, vp, pages, pos0, page_size=P, window=9, gate=False), kp, vp]

    def refused():
        """What each call says of arguments that it does not take."""
        kp, vp = (ops.paged_pool(n_pages, P, kv8=kv8) for _ in range(2))
        said = []
        bad = [
            lambda: ops.paged_kv_store(x["k"], x["v"], kp, vp, pages[:2], starts, pos0, page_size=P),
            lambda: ops.paged_kv_store(x["k"].float(), x["v"], kp, vp, pages, starts, pos0, page_size=P),
            lambda: ops.paged_kv_store(x["k"].cpu(), x["v"], kp, vp, pages, starts, pos0, page_size=P),
            lambda: ops.paged_kv_store(x["k"], x["v"][:8], kp, vp, pages, starts, pos0, page_size=P),
            lambda: ops.paged_kv_load(kp, vp, pages.long(), starts, pos0, T=9, page_size=P),
            lambda: ops.paged_kv_load(kp, vp, pages, starts, pos0, T=-1, page_size=P),
            lambda: ops.paged_kv_load(kp, vp, pages, starts[:3], pos0, T=9, page_size=P),
            lambda: ops.attn_prep_paged(x["qg"], x["k"], x["v"], wq[:100].clone(), wk, kp, vp, pages, starts, pos0, page_size=P),
            lambda: ops.attn_prep_paged(x["qg"], x["k"], x["v"], wq, wk, kp, vp, pages, starts, pos0, page_size=P,
                                        rope_dim=33),
            lambda: ops.attention_prefill_paged(x["qg"], kp, vp, pages, Ts, [1, 2], page_size=P),
            lambda: ops.attention_prefill_paged(x["qg"], kp, vp, pages, [3, -1, 5], p0, page_size=P),
            lambda: ops.attention_prefill_paged(x["qg"], kp, vp, pages, [30, 1, 5], p0, page_size=P),
            lambda: ops.attention_prefill_paged(x["qg"], kp, vp, pages, Ts, [10000, 1, 5], page_size=P),
            lambda: ops.attention_prefill_paged(x["qg"], kp, vp, pages, Ts, p0, page_size=P, window=-1),
            lambda: ops.attn_decode_paged(x["qg"][:3, None], kp, vp, pages, i32(1, 2), page_size=P),
            lambda: ops.attn_decode_paged(x["qg"].view(3, 3, 24, 512), kp, vp, pages, pos0, page_size=17),
            lambda: ops.attn_decode_paged(x["qg"][:3, None], kp, vp, pages, pos0, page_size=P, scale=0.0),
            lambda: ops.attn_decode_paged(torch.zeros(3, 6, 24, 512, dtype=F16, device="cuda"), kp, vp, pages, pos0,
                                          page_size=P),
            lambda: ops.attn_decode_paged(x["qg"][:3, None], kp, vp, pages, pos0, page_size=P,
                                          work=torch.empty(64, dtype=torch.uint8, device="cuda")),
        ]
        for i, call in enumerate(bad):
            try:
                call()
            except (TypeError, ValueError, fl._lib.FlError) as e:
                said.append((type(e), str(e)))
            else:
                pytest.fail(f"call {i} was taken")
        return said

    got, said = calls(), refused()
    monkeypatch.setattr(fl._lib, "lane", None)
    want, says = calls(), refused()
    torch.cuda.synchronize()
    for i, (a, b) in enumerate(zip(got, want)):
        assert a.dtype == b.dtype and a.shape == b.shape, i
        assert torch.equal(a.view(torch.int8) if a.dtype != torch.int8 else a,
                           b.view(torch.int8) if b.dtype != torch.int8 else b), i
    assert said == says
