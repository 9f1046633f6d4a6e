"""The paged attention on the GPU against bounds that start from the values the kernels form
(paged_tight.py; what those bounds reject is tested on the CPU): cached rows whose every tile
shows in z, runs long enough that a wave loads its page ids again, K exact and weights in two
terms in the int8 decode, the same bits from the same call."""
import pytest
import torch

import paged_ref as ref
import paged_tight as tight

pytestmark = pytest.mark.gpu

F16, I32 = torch.float16, torch.int32
SCALE = 256 ** -0.5


def gen(seed):
    return torch.Generator().manual_seed(seed)


def randn(g, *shape, scale=1.0):
    return (torch.randn(shape, generator=g) * scale).to(F16).cuda()


def i32(*v):
    return torch.tensor(v, dtype=I32, device="cuda")


def starts_of(Ts):
    return i32(*[sum(Ts[:i]) for i in range(len(Ts) + 1)])


def filled(fl, g, lens, page_size, kv8, n_kv):
    """Pools with marked rows of sequences of `lens` positions over shuffled pages: (kpool,
    vpool, pages, [a sequence's pool rows])."""
    ops = fl.ops
    pages, n_pages = ref.make_pages(g, lens, page_size)
    kp, vp = (ops.paged_pool(n_pages, page_size, kv8=kv8, n_kv_heads=n_kv) for _ in range(2))
    rows = [tight.marked_rows(g, n, n_kv) for n in lens]
    k, v = (torch.cat([r[i] for r in rows]).cuda() for i in range(2))
    ops.paged_kv_store(k, v, kp, vp, pages, starts_of(lens), i32(*[0] * len(lens)), page_size=page_size,
                       n_kv_heads=n_kv)
    host = pages.cpu()
    return kp, vp, pages, [ref.rows_of(host, b, page_size, torch.arange(n)).cuda() for b, n in enumerate(lens)]


def seen_mask(T, p0, L, window=0, sinks=0):
    p = torch.arange(p0, p0 + T, device="cuda")[:, None]
    r = torch.arange(L, device="cuda")[None]
    return (r <= p) & ((r > p - window) | (r < sinks)) if window else r <= p


def check(z, want, bound, what):
    assert torch.isfinite(z).all(), f"{what}: not finite"
    worst = ((z.double() - want).abs() / bound).max().item()
    print(f"{what}: {worst:.2f} of the bound")
    assert worst <= 1, f"{what}: {worst} of the bound"


def of_kernel(pools, page_size, n_kv):
    n = pools[0].numel() // (n_kv * (272 if pools[0].dtype == torch.int8 else 256))
    return (tight.kernel_values(pools[0], n, n_kv, True), tight.kernel_values(pools[1], n, n_kv, False))


def run_decode(fl, seed, lens, page_size, kv8, T=1, window=0, sinks=0, heads=(24, 4), q_scale=1.0):
    g = gen(seed)
    n_q, n_kv = heads
    kp, vp, pages, rows = filled(fl, g, lens, page_size, kv8, n_kv)
    K, V = of_kernel((kp, vp), page_size, n_kv)
    qg = randn(g, len(lens), T, n_q, 512, scale=q_scale)
    z = fl.ops.attn_decode_paged(qg, kp, vp, pages, i32(*[n - T for n in lens]), page_size=page_size,
                                 window=window, sinks=sinks, n_kv_heads=n_kv)
    for b, n in enumerate(lens):
        want, bound = tight.attention(qg[b, ..., :256], K[rows[b]], V[rows[b]],
                                      seen_mask(T, n - T, n, window, sinks), SCALE,
                                      tight.TWO_TERMS if kv8 else tight.ONE_TERM, qg[b, ..., 256:])
        check(z[b], want, bound, f"sequence {b} (length {n}, T {T})")


@pytest.mark.parametrize("kv8", [False, True])
@pytest.mark.parametrize("lens,page_size,T", [
    ([1], 16, 1), ([3], 16, 4), ([17, 16, 15, 31, 32, 33], 16, 1), ([500], 16, 1), ([4096, 1, 777], 64, 1),
    ([1000, 64, 65], 32, 4), ([3001, 2999], 128, 3), ([9000, 50], 64, 1), ([9000, 50], 16, 5),
], ids=str)
def test_decode(fl, dev, lens, page_size, T, kv8):
    run_decode(fl, 31, lens, page_size, kv8, T)


@pytest.mark.parametrize("kv8", [False, True])
@pytest.mark.parametrize("window,sinks,T", [(16, 4, 1), (100, 0, 3), (33, 40, 1), (2000, 3, 3), (250, 1000, 1)])
def test_decode_window_and_sinks(fl, dev, window, sinks, T, kv8):
    run_decode(fl, 41, [2500, 40, 3, 290], 32, kv8, T, window, sinks)


@pytest.mark.parametrize("kv8", [False, True])
@pytest.mark.parametrize("heads,T", [((1, 1), 32), ((8, 1), 4), ((32, 8), 3), ((6, 2), 2), ((64, 2), 1), ((3, 3), 1)])
def test_decode_heads_and_peaked_scores(fl, dev, heads, T, kv8):
    run_decode(fl, 51, [100, 1333, 32], 16, kv8, T, heads=heads)
    run_decode(fl, 52, [100, 1333, 32], 16, kv8, T, heads=heads, q_scale=4.0)


def longest_walk(tiles, B, n_kv, kv8, rows):
    """The page ids that a wave takes on one sequence's part of a run, at the most, by the
    decode's division of the stream (B sequences of `tiles` tiles)."""
    runs = max(1, torch.cuda.get_device_properties(0).multi_processor_count // n_kv)
    cost = 6 if kv8 else 2
    total, step = B * (tiles + cost), 1
    if kv8:
        step, heads_lg = (4, 0) if rows > 16 else (8, min(2, (n_kv & -n_kv).bit_length() - 1))
        if rows <= 16 and total // 64 >= runs:
            runs, step = runs << heads_lg, step >> heads_lg
    return min(tiles, int(total / runs)) // step


@pytest.mark.parametrize("kv8", [False, True])
@pytest.mark.parametrize("heads,T,B,L,page_size", [
    ((24, 4), 1, 64, 9700, 16), ((24, 4), 3, 64, 9700, 32), ((6, 3), 1, 90, 10000, 64), ((4, 1), 8, 300, 9000, 16),
])
def test_decode_runs_that_load_their_page_ids_again(fl, dev, heads, T, B, L, page_size, kv8):
    """Many sequences over one shared prefix in shuffled pages, of unlike lengths: a wave takes
    more than the 64 page ids that its first two loads hold (32 in the last case but one over int8,
    whose waves take every eighth tile)."""
    n_q, n_kv = heads
    walk = longest_walk(L // 32 - 20, B, n_kv, kv8, T * n_q // n_kv)
    assert walk > (32 if walk < 64 else 64)
    g = gen(65 + B)
    kp, vp, pages, [rows] = filled(fl, g, [L], page_size, kv8, n_kv)
    K, V = of_kernel((kp, vp), page_size, n_kv)
    K, V = K[rows], V[rows]
    lens = [int(x) for x in torch.randint(L - 600, L + 1, (B,), generator=g)]
    qg = randn(g, B, T, n_q, 512)
    z = fl.ops.attn_decode_paged(qg, kp, vp, pages.repeat(B, 1), i32(*[n - T for n in lens]),
                                 page_size=page_size, n_kv_heads=n_kv)
    for b in range(0, B, 3):
        n = lens[b]
        want, bound = tight.attention(qg[b, ..., :256], K[:n], V[:n], seen_mask(T, n - T, n), SCALE,
                                      tight.TWO_TERMS if kv8 else tight.ONE_TERM, qg[b, ..., 256:])
        check(z[b], want, bound, f"sequence {b} (length {n})")


def run_chunks(fl, seed, spans, page_size, kv8, window=0, sinks=0, heads=(24, 4)):
    g = gen(seed)
    n_q, n_kv = heads
    kp, vp, pages, rows = filled(fl, g, [t + p for t, p in spans], page_size, kv8, n_kv)
    K, V = of_kernel((kp, vp), page_size, n_kv)
    Ts, p0s = [t for t, _ in spans], [p for _, p in spans]
    qg = randn(g, sum(Ts), n_q, 512)
    z = fl.ops.attention_prefill_paged(qg, kp, vp, pages, Ts, p0s, page_size=page_size, window=window,
                                       sinks=sinks, gated=True, n_kv_heads=n_kv)
    at = 0
    for b, (t, p) in enumerate(spans):
        want, bound = tight.attention(qg[at:at + t, :, :256], K[rows[b]], V[rows[b]],
                                      seen_mask(t, p, t + p, window, sinks), SCALE,
                                      tight.TWO_TERMS if kv8 else tight.ONE_TERM, qg[at:at + t, :, 256:])
        check(z[at:at + t], want, bound, f"sequence {b} ({t}@{p})")
        at += t


@pytest.mark.parametrize("kv8", [False, True])
@pytest.mark.parametrize("spans,page_size", [
    ([(1, 0)], 16), ([(31, 17), (1, 32), (65, 63)], 16), ([(300, 0)], 64), ([(257, 1000), (3, 511)], 128),
    ([(20, 9000), (42, 2000)], 256), ([(700, 345)], 16), ([(5, 4090)] * 9, 64), ([(1, 700)] * 64, 32),
    ([(12, 30000)], 32),
], ids=str)
def test_chunks(fl, dev, spans, page_size, kv8):
    run_chunks(fl, 11, spans, page_size, kv8)


@pytest.mark.parametrize("kv8", [False, True])
@pytest.mark.parametrize("window,sinks", [(16, 4), (100, 0), (33, 40), (1000, 3), (250, 1000)])
def test_chunks_window_and_sinks(fl, dev, window, sinks, kv8):
    run_chunks(fl, window, [(260, 0), (70, 1777), (1, 900), (130, 100)], 32, kv8, window, sinks)


@pytest.mark.parametrize("heads", [(1, 1), (8, 1), (32, 8), (3, 3)])
@pytest.mark.parametrize("kv8", [False, True])
def test_chunks_heads(fl, dev, heads, kv8):
    run_chunks(fl, 5, [(70, 130), (33, 1300)], 16, kv8, heads=heads)


def test_int8_chunks_in_groups(fl, dev):
    """int8 contexts of 100k whose fp16 copies pass 1 GiB together: every tile is in z."""
    run_chunks(fl, 23, [(3, 99997), (1, 98999), (20, 98480), (70, 0)], 256, True)


@pytest.mark.parametrize("form,T,heads,B", [("decode", 1, (4, 1), 1), ("decode", 20, (1, 1), 1),
                                            ("decode", 3, (6, 1), 70), ("chunks", 1, (4, 1), 1),
                                            ("chunks", 50, (6, 1), 1), ("chunks", 40, (6, 1), 64)])
def test_int8_takes_k_exactly(fl, dev, form, T, heads, B):
    """Scores of 100 whose differences K's rounding to fp16 would move by 5 %: decode of up to 16
    rows and of 17 to 32, chunks (a page of 64 rows, shared by B sequences)."""
    L = 64
    kp, vp, q = tight.near_ties(L)
    qg = q.cuda().expand(B, T, heads[0], 256).contiguous()
    table = i32(0).view(1, 1).repeat(B, 1)
    if form == "decode":
        z = fl.ops.attn_decode_paged(qg, kp.cuda(), vp.cuda(), table, i32(*[L - T] * B), page_size=L, gate=False,
                                     n_kv_heads=1)
    else:
        z = fl.ops.attention_prefill_paged(qg.view(B * T, heads[0], 256), kp.cuda(), vp.cuda(), table, [T] * B,
                                           [L - T] * B, page_size=L, n_kv_heads=1).view(B, T, heads[0], 256)
    K, V = (tight.kernel_values(p, L, 1, e).cuda() for p, e in ((kp, True), (vp, False)))
    want, bound = tight.attention(qg[0], K, V, seen_mask(T, L - T, L), SCALE, tight.TWO_TERMS)
    for b in range(B):
        check(z[b], want, bound, f"sequence {b}")


@pytest.mark.parametrize("form,T", [("decode", 1), ("decode", 20), ("chunks", 30)])
def test_int8_takes_weights_in_two_terms(fl, dev, form, T):
    """600 sequences (60 chunks) of a page, so that one wave or pair has all its rows: the mean
    over the dims of z's relative error, whose part from z's own rounding is 2^-11 / sqrt(3 * 256),
    allowed 6 times; in one term it is more than twice that (tested on the CPU)."""
    L, B = 32, 600 if form == "decode" else 60
    kp, vp, q, off = tight.one_term_shows(L)
    qg = q.cuda().expand(B, T, 1, 256).contiguous()
    table = i32(0).view(1, 1).repeat(B, 1)
    if form == "decode":
        z = fl.ops.attn_decode_paged(qg, kp.cuda(), vp.cuda(), table, i32(*[L - T] * B), page_size=L, gate=False,
                                     n_kv_heads=1)
    else:
        z = fl.ops.attention_prefill_paged(qg.view(B * T, 1, 256), kp.cuda(), vp.cuda(), table, [T] * B,
                                           [L - T] * B, page_size=L, n_kv_heads=1).view(B, T, 1, 256)
    K, V = (tight.kernel_values(p, L, 1, e)[:, 0].cuda() for p, e in ((kp, True), (vp, False)))
    for t in (T // 2, T - 1):
        n = L - T + 1 + t
        want = torch.softmax(q.cuda().double() @ K[:n].t() * SCALE, -1) @ V[:n]
        mean = ((z[:, t, 0].double() - want) / want).mean(-1).abs().max().item()
        assert mean < 6 * 2.0 ** -11 / (3 * 256) ** 0.5, mean


@pytest.mark.parametrize("kv8", [False, True])
def test_the_same_call_gives_the_same_bits(fl, dev, kv8):
    """Sums have one order: nothing is added by atomics."""
    g = gen(7)
    lens = [4000, 33, 900, 12000]
    kp, vp, pages, _ = filled(fl, g, lens, 32, kv8, 4)
    qd, qc = randn(g, 4, 3, 24, 512), randn(g, 400, 24, 512)
    calls = [lambda: fl.ops.attn_decode_paged(qd, kp, vp, pages, i32(*[n - 3 for n in lens]), page_size=32),
             lambda: fl.ops.attention_prefill_paged(qc, kp, vp, pages, [100, 33, 67, 200],
                                                    [3900, 0, 833, 11800], page_size=32, gated=True)]
    for call in calls:
        first = call()
        for _ in range(4):
            assert torch.equal(call(), first)
