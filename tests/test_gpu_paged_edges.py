"""The paged operators where inputs and callers are unlike the ordinary: host threads beside a
call, gates and rows that are not numbers, contexts whose weights lie far below the largest."""
import ctypes

import pytest
import torch

import paged_ref as ref

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


def kernel_values(pool, n_rows, exact):
    """A pool's rows as the kernels take them: fp16 pools as they are, int8 ones byte * scale,
    exact or rounded to fp16."""
    if pool.dtype != torch.int8:
        return pool.view(n_rows, 4, 256).double()
    v = ref.dequant(pool, n_rows, 4)
    return v if exact else v.to(F16).double()


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
    K = kernel_values(kp, n_pages * P, form != "chunks")[rows]
    V = kernel_values(vp, n_pages * P, False)[rows]
    s = 16 * K[:, 0, 0] * SCALE                  # the same for every head
    gap = (s[0] - s[1]).item() / torch.log(torch.tensor(2.0)).item()
    assert 22.5 < gap < 22.9
    rel = 2 * 2.0 ** -11 + 2.0 ** (gap - 32) + 2 * gap * 3 * 2.0 ** -24 + 2.0 ** -21 + 2 * 700 * 2.0 ** -24
    for t in range(T):
        n = L - T + 1 + t
        want = (torch.softmax(s[:n], 0)[:, None, None] * V[:n]).sum(0).repeat_interleave(6, 0)
        off = ((z[:, t].double() - want) / want).abs().max().item()
        assert off <= rel, f"token {t}: off by {off}, {rel} allowed"
