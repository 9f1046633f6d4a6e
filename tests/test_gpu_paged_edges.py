"""The paged operators where inputs and callers are unlike the ordinary: host threads beside a
call, gates and rows that are not numbers, contexts whose weights lie far below the largest."""
import ctypes

import pytest
import torch

import paged_ref as ref
import paged_tight as tight

pytestmark = pytest.mark.gpu

F16, F32, I32 = torch.float16, torch.float32, torch.int32
SCALE = 256 ** -0.5


def gen(seed):
    return torch.Generator().manual_seed(seed)


def randn(g, *shape, scale=1.0):
    return (torch.randn(shape, generator=g) * scale).to(F16).cuda()


def i32(*v):
    return torch.tensor(v, dtype=I32, device="cuda")


def test_the_plan_of_chunks_is_made_with_other_threads_running(fl, dev):
    """The binding asks for the work bytes, which makes the plan, and launches with the
    interpreter released. In place of the library stand the interpreter's own "do I hold it"
    (1 or 0, here the work bytes) and a callback that notes the bytes it is given."""
    L, lane = fl._lib.lib(), fl._lib.lane
    assert lane is not None, "fl355_paged.so is not built"
    real = [ctypes.cast(getattr(L, name), ctypes.c_void_p).value for name in fl._lib.BOUND]
    seen = []
    name = "fl_attention_prefill_paged"
    res, args = fl._lib.SIGNATURES[name]
    noted = ctypes.CFUNCTYPE(res, *args)(lambda *a: seen.append(a[-2]) or 0)
    held = ctypes.cast(ctypes.pythonapi.PyGILState_Check, ctypes.c_void_p).value
    fake = dict(zip(fl._lib.BOUND, real))
    fake[name] = ctypes.cast(noted, ctypes.c_void_p).value
    fake["fl_attention_prefill_paged_work_bytes"] = held
    q = torch.zeros((3, 24, 512), dtype=F16, device="cuda")
    kp = fl.ops.paged_pool(2, 16)
    try:
        lane.bind(*fake.values())
        fl.ops.attention_prefill_paged(q, kp, kp, i32(0, 1).view(1, 2), [3], [0], page_size=16)
    finally:
        lane.bind(*real)
    assert seen == [0]


@pytest.mark.parametrize("kv8", [False, True])
@pytest.mark.parametrize("T", [1, 4])
def test_decode_of_queries_that_see_nothing_gives_0_whatever_they_hold(fl, dev, kv8, T):
    """A padded batch's rows may hold anything, their gates too: at negative positions, and
    with every page absent, z is 0; also where the sequence's later tokens see a NaN."""
    g, P = gen(T), 16
    kp, vp = (fl.ops.paged_pool(4, P, kv8=kv8) for _ in range(2))
    pages = i32(0, 1, -1, -1, 2, 3).view(3, 2)
    pos0 = i32(-T, 20, -T + 1)
    rows = randn(g, 64, 4, 256)
    bad = rows.clone()
    bad[32:] = float("nan")   # pages 2 and 3: the third sequence's
    fl.ops.paged_kv_store(rows, bad, kp, vp, i32(0, 1, 2, 3).view(1, 4), i32(0, 64), i32(0), page_size=P)
    qg = torch.full((3, T, 24, 512), float("nan"), dtype=F16, device="cuda")
    qg[1, ..., :256] = 1.0
    qg[2, :T - 1] = float("inf")
    for gate in (True, False):
        z = fl.ops.attn_decode_paged(qg, kp, vp, pages, pos0, page_size=P, gate=gate)
        assert not z[:2].any() and not z[2, :T - 1].any()


@pytest.mark.parametrize("kv8", [False, True])
@pytest.mark.parametrize("spans", [[(37, 3001)], [(100, 0)], [(300, 700), (5, 40)]], ids=str)
def test_chunks_of_queries_that_see_nothing_give_0_whatever_they_hold(fl, dev, kv8, spans):
    """Every page absent, cut row tiles and whole ones, some rows' gates and q NaN or infinite."""
    P = 32
    kp, vp = (fl.ops.paged_pool(2, P, kv8=kv8) for _ in range(2))
    Ts, p0s = [t for t, _ in spans], [p for _, p in spans]
    pages = torch.full((len(spans), max(map(sum, spans)) // P + 1), -1, dtype=I32, device="cuda")
    qg = randn(gen(9), sum(Ts), 24, 512)
    qg[::3] = float("nan")
    qg[1::3, :, 256:] = float("-inf")
    qg[2::3, 5] = float("inf")
    for gated in (True, False):
        z = fl.ops.attention_prefill_paged(qg, kp, vp, pages, Ts, p0s, page_size=P, gated=gated)
        assert not z.any()


@pytest.mark.parametrize("kv8", [False, True])
def test_chunk_with_some_queries_that_see_nothing(fl, dev, kv8):
    """A window that lies on an absent page: those queries give 0 beside others that see rows."""
    P, T, window = 32, 200, 8
    g = gen(12)
    kp, vp = (fl.ops.paged_pool(7, P, kv8=kv8) for _ in range(2))
    pages = i32(0, 1, -1, 3, 4, 5, 6).view(1, 7)
    rows = randn(g, T, 4, 256)
    fl.ops.paged_kv_store(rows, rows, kp, vp, pages, i32(0, T), i32(0), page_size=P)
    qg = randn(g, T, 24, 512)
    qg[64 + window - 1:96, ::2, 256:] = float("nan")   # (these see rows 64 .. 95 alone)
    z = fl.ops.attention_prefill_paged(qg, kp, vp, pages, [T], [0], page_size=P, window=window, gated=True)
    assert torch.isfinite(z).all()
    blind = torch.zeros(T, dtype=torch.bool, device="cuda")
    blind[64 + window - 1:96] = True
    assert not z[blind].any() and bool((z[~blind] != 0).flatten(1).any(1).all())


@pytest.mark.parametrize("kv8", [False, True])
@pytest.mark.parametrize("form", ["decode1", "decode4", "chunks"])
def test_many_small_weights_beside_one_large(fl, dev, form, kv8):
    """A first row that holds nearly all the weight and a v of 0, as first tokens do: z is what
    the others leave, each 2^-22.7 of the largest. Weights go into the product with v as fp16
    with a step of 2^-24 (subnormal) at the least, of the largest's reference: that is 7 octaves
    or more above the running maximum's own 1, so a weight is off by 2^-11 of itself or 2^-32 of
    the largest. Beside that: z to fp16 (2^-11); in 32 bits the score (22.7 in log2 units, three
    roundings), the exponential (2 ulp) and 700 additions, numerator and denominator."""
    g, P, L, ops = gen(3), 64, 700, fl.ops
    pages, n_pages = ref.make_pages(g, [L], P)
    K, V = torch.zeros(L, 4, 256), 1500 + 100 * torch.randn((L, 4, 256), generator=g)
    K[0, :, 0], V[0] = 15.734, 0
    kp, vp = (ops.paged_pool(n_pages, P, kv8=kv8) for _ in range(2))
    ops.paged_kv_store(K.to(F16).cuda(), V.to(F16).cuda(), kp, vp, pages, i32(0, L), i32(0), page_size=P)
    T = {"decode1": 1, "decode4": 4, "chunks": 40}[form]
    B = 64 if form == "chunks" else 160          # (so many that a sequence stays in a run or two)
    q = randn(g, B, T, 24, 512)
    q[..., 0] = 16
    table = pages.repeat(B, 1)
    if form == "chunks":
        z = ops.attention_prefill_paged(q.view(B * T, 24, 512), kp, vp, table, [T] * B, [L - T] * B, page_size=P)
        z = z.view(B, T, 24, 256)
    else:
        z = ops.attn_decode_paged(q, kp, vp, table, i32(*[L - T] * B), page_size=P, gate=False)
    rows = ref.rows_of(pages.cpu(), 0, P, torch.arange(L)).cuda()
    K = tight.kernel_values(kp, n_pages * P, 4, True)[rows]
    V = tight.kernel_values(vp, n_pages * P, 4, False)[rows]
    s = 16 * K[:, 0, 0] * SCALE                  # the same for every head
    gap = (s[0] - s[1]).item() / torch.log(torch.tensor(2.0)).item()
    assert 22.5 < gap < 22.9
    rel = 2 * 2.0 ** -11 + 2.0 ** (gap - 32) + 2 * gap * 3 * 2.0 ** -24 + 2.0 ** -21 + 2 * 700 * 2.0 ** -24
    for t in range(T):
        n = L - T + 1 + t
        want = (torch.softmax(s[:n], 0)[:, None, None] * V[:n]).sum(0).repeat_interleave(6, 0)
        off = ((z[:, t].double() - want) / want).abs().max().item()
        assert off <= rel, f"token {t}: off by {off}, {rel} allowed"


GATES = [float("inf"), float("-inf"), 65504.0, -65504.0, 0.0, -0.0, 17.0, -17.0, 88.0, -88.0, -104.0, 2.0 ** -24]


def small_cache(fl, g, kv8, L=300, P=32, B=1, spoil=None):
    """Pools with B sequences of L random rows, `spoil` applied to the rows [B L, 4, 256] of k and v
    first: (kpool, vpool, pages, a sequence's rows of the pools)."""
    pages, n_pages = ref.make_pages(g, [L] * B, P)
    kp, vp = (fl.ops.paged_pool(n_pages, P, kv8=kv8) for _ in range(2))
    k, v = randn(g, B * L, 4, 256), randn(g, B * L, 4, 256)
    if spoil:
        spoil(k, v)
    fl.ops.paged_kv_store(k, v, kp, vp, pages, i32(*[L * b for b in range(B + 1)]), i32(*[0] * B), page_size=P)
    rows = [ref.rows_of(pages.cpu(), b, P, torch.arange(L)).cuda() for b in range(B)]
    return kp, vp, pages, rows, n_pages * P


def both_forms(fl, qg, kp, vp, pages, p0s, P=32, **args):
    """qg [B, T, 24, 512] as decode and as chunks: [(form, z [B, T, 24, 256])]."""
    B, T = qg.shape[:2]
    zd = fl.ops.attn_decode_paged(qg, kp, vp, pages, i32(*p0s), page_size=P, **args)
    zc = fl.ops.attention_prefill_paged(qg.reshape(B * T, 24, 512), kp, vp, pages, [T] * B, p0s, page_size=P,
                                        gated=True, **args)
    return [("decode", zd), ("chunks", zc.view(B, T, 24, 256))]


@pytest.mark.parametrize("kv8", [False, True])
@pytest.mark.parametrize("T", [1, 5])
def test_gates_of_every_size(fl, dev, kv8, T):
    """Infinite gates, the type's largest, and those whose sigmoid leaves fp16 or fp32: closed
    ones give 0 and open ones z."""
    g, L = gen(21), 300
    kp, vp, pages, [rows], n = small_cache(fl, g, kv8, L)
    qg = randn(g, 1, T, 24, 512)
    qg[..., 256:] = torch.tensor(GATES * 22)[:256].to(F16).cuda()
    seen = torch.arange(L, device="cuda")[None] <= torch.arange(L - T, L, device="cuda")[:, None]
    for form, z in both_forms(fl, qg, kp, vp, pages, [L - T]):
        K, V = tight.kernel_values(kp, n, 4, True)[rows], tight.kernel_values(vp, n, 4, False)[rows]
        want, bound = tight.attention(qg[0, ..., :256], K, V, seen, SCALE,
                                      tight.TWO_TERMS if kv8 else tight.ONE_TERM, qg[0, ..., 256:])
        assert ((z[0].double() - want).abs() <= bound).all(), form
        assert not z[0][qg[0, ..., 256:] <= -88].any()


@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
def test_v_rows_that_are_not_finite(fl, dev, value):
    """One v of a row that is in sight: the dim is not finite, or saturated, for the queries that
    see the row; every other dim of theirs, and every other sequence, is as without it. Tokens of
    the sequence that do not see it may have a NaN in that dim, and no more."""
    L, T, row, dim = 300, 4, 297, 40

    def spoil(k, v):
        v[row, 2, dim] = value

    clean = small_cache(fl, gen(22), False, L, B=3)
    spoiled = small_cache(fl, gen(22), False, L, B=3, spoil=spoil)
    qg = randn(gen(23), 3, T, 24, 512)
    p0s = [L - T] * 3                              # token 1 of the first sequence is that row
    for (form, want), (_, z) in zip(both_forms(fl, qg, *clean[:3], p0s), both_forms(fl, qg, *spoiled[:3], p0s)):
        hit = z[0, 1:, 12:18, dim]
        assert (hit.isnan() | (hit.abs() == 65504) | (hit == 0)).all(), form
        assert hit.isnan().all() or value == value
        before = z[0, 0, 12:18, dim]
        assert (before.isnan() | (before == want[0, 0, 12:18, dim])).all(), form
        z[0, :, 12:18, dim] = want[0, :, 12:18, dim]
        assert torch.equal(z, want), form


@pytest.mark.parametrize("kv8", [False, True])
def test_scores_that_are_infinite(fl, dev, kv8):
    """A k of infinity in a row in sight: minus infinity as a score leaves the row out, plus
    infinity gives NaN (int8: the block is stored with an infinite scale, and what the row's score
    is then is left open); queries before the row and other sequences are as without it."""
    L, T, row = 300, 4, 298

    def spoil(k, v):
        k[row, 1, 7] = float("inf")

    clean = small_cache(fl, gen(24), kv8, L, B=2)
    spoiled = small_cache(fl, gen(24), kv8, L, B=2, spoil=spoil)
    qg = randn(gen(25), 2, T, 24, 512)
    qg[..., 7] = torch.where(torch.arange(24, device="cuda") % 2 == 0, 1.0, -1.0).half()
    p0s = [L - T] * 2
    for (form, want), (_, z) in zip(both_forms(fl, qg, *clean[:3], p0s), both_forms(fl, qg, *spoiled[:3], p0s)):
        see = z[0, 2:, 6:12]                       # tokens 2 and 3, kv head 1's heads
        if not kv8:
            assert see[:, ::2].isnan().all(), form
            K, V = (tight.kernel_values(p, spoiled[4], 4, True)[spoiled[3][0]] for p in spoiled[:2])
            for t in (2, 3):
                for h in (7, 9, 11):
                    q = qg[0, t, h, :256].double()
                    s = q @ K[:L - T + t + 1, 1].t() * SCALE
                    out = torch.softmax(s, -1) @ V[:L - T + t + 1, 1] * torch.sigmoid(qg[0, t, h, 256:].double())
                    # P to fp16: 2^-11 of sum w |v|, under 2 here; z: 2^-11, under 1; the rest: 2^-11
                    assert (z[0, t, h].double() - out).abs().max() <= 2.0 ** -9, (form, t, h)
        z[0, 2:, 6:12] = want[0, 2:, 6:12]
        if form == "decode":
            assert torch.equal(z, want)
            continue
        # In chunks the queries of a wave move their references together, each to its own maximum,
        # so the infinite score moves where the others' weights round: not the same bits, but each
        # within the bound of what the clean rows give.
        seen = torch.arange(L, device="cuda")[None] <= torch.arange(L - T, L, device="cuda")[:, None]
        K, V = (tight.kernel_values(p, clean[4], 4, e) for p, e in zip(clean[:2], (True, False)))
        for b in range(2):
            exact, bound = tight.attention(qg[b, ..., :256], K[clean[3][b]], V[clean[3][b]], seen, SCALE,
                                           tight.TWO_TERMS if kv8 else tight.ONE_TERM, qg[b, ..., 256:])
            assert ((z[b].double() - exact).abs() <= bound).all()


@pytest.mark.parametrize("T", [1, 5])
def test_int8_scales_of_every_size(fl, dev, T):
    """K's block scales from 0 (whose bytes count for nothing) over subnormal ones to 0.1 side by
    side in a row, V's likewise: the chunk kernel forms a score by the ratios of its row's scales."""
    g, L, P = gen(31), 400, 16
    pages, n_pages = ref.make_pages(g, [L], P)
    sizes = torch.tensor([0.0, 2.0 ** -24, 2.0 ** -16, 1e-4, 0.003, 0.02, 0.1])
    pools = []
    for _ in range(2):
        scales = sizes[torch.randint(0, 7, (n_pages * P, 4, 8), generator=g)]
        pools.append(tight.int8_pool(torch.randint(-127, 128, (n_pages * P, 4, 256), generator=g), scales).cuda())
    kp, vp = pools
    rows = ref.rows_of(pages.cpu(), 0, P, torch.arange(L)).cuda()
    K, V = tight.kernel_values(kp, n_pages * P, 4, True)[rows], tight.kernel_values(vp, n_pages * P, 4, False)[rows]
    qg = randn(g, 1, T, 24, 512)
    seen = torch.arange(L, device="cuda")[None] <= torch.arange(L - T, L, device="cuda")[:, None]
    want, bound = tight.attention(qg[0, ..., :256], K, V, seen, SCALE, tight.TWO_TERMS, qg[0, ..., 256:])
    for form, z in both_forms(fl, qg, kp, vp, pages, [L - T], P):
        assert ((z[0].double() - want).abs() <= bound).all(), form
