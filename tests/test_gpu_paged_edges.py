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
