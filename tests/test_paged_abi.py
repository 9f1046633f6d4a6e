"""The paged cache's entry points on the CPU: what they refuse, before any launch."""
import ctypes

import pytest
import torch

FAKE = 1 << 20   # an aligned address that is never read


def ints(*v):
    return (ctypes.c_int * max(1, len(v)))(*v)


POOL = dict(kpool=FAKE, vpool=FAKE, q8=0, n_pages=8, page_size=16, pages=FAKE, max_pages=4, stride=4)


def pool(over):
    p = {**POOL, **{k: v for k, v in over.items() if k in POOL}}
    return p["kpool"], p["vpool"], p["q8"], p["n_pages"], p["page_size"], p["pages"], p["max_pages"], \
        p["stride"]


def call(fl, name, over):
    """One call with every argument valid but those in `over`; N, or the chunks'
    total, is 0 unless given, so nothing would be launched either way."""
    a = dict(k=FAKE, v=FAKE, ks=1024, vs=1024, starts=FAKE, pos0=FAKE, B=2, N=0, kv=4, hd=256, nq=24,
             qp=512, zp=256, q=FAKE, z=FAKE, T=1, window=0, sinks=0, gated=1, wq=FAKE, wk=FAKE,
             q_out=None, qop=0, rope=64, Ts=ints(0, 0), pos0s=ints(0, 0), work=None, wb=0)
    a.update(over)
    f = getattr(fl._lib.lib(), name)
    if name == "fl_paged_kv_store":
        return f(a["k"], a["v"], a["ks"], a["vs"], *pool(over), a["starts"], a["pos0"], a["B"], a["N"],
                 a["kv"], a["hd"], None)
    if name == "fl_paged_kv_load":
        return f(*pool(over), a["starts"], a["pos0"], a["k"], a["v"], a["ks"], a["vs"], 0, a["B"],
                 a["N"], a["kv"], a["hd"], None)
    if name == "fl_attn_prep_paged":
        return f(a["q"], a["qp"], a["k"], a["v"], a["wq"], a["wk"], a["q_out"], a["qop"], *pool(over),
                 a["starts"], a["pos0"], a["B"], a["N"], a["nq"], a["kv"], a["hd"], a["rope"], 1e7, 1e-6,
                 None)
    if name == "fl_attention_prefill_paged":
        return f(a["q"], a["qp"], *pool(over), a["Ts"], a["pos0s"], a["B"], a["nq"], a["kv"], a["hd"],
                 0.0625, a["window"], a["sinks"], a["gated"], a["z"], a["zp"], a["work"], a["wb"], None)
    return f(a["q"], a["qp"], *pool(over), a["pos0"], a["B"], a["T"], a["nq"], a["kv"], a["hd"], 0.0625,
             a["window"], a["sinks"], a["gated"], a["z"], a["zp"], a["work"], a["wb"], None)


ALL = ["fl_paged_kv_store", "fl_paged_kv_load", "fl_attn_prep_paged", "fl_attention_prefill_paged",
       "fl_attn_decode_paged"]
COMMON = [dict(kpool=None), dict(vpool=None), dict(pages=None), dict(q8=2), dict(hd=128),
          dict(kv=0), dict(page_size=8), dict(page_size=48), dict(page_size=0), dict(n_pages=0),
          dict(max_pages=0), dict(stride=3), dict(B=0), dict(B=1025), dict(kpool=FAKE + 8),
          dict(n_pages=1 << 30), dict(max_pages=1 << 27, stride=1 << 27)]


@pytest.mark.parametrize("name", ALL)
@pytest.mark.parametrize("over", COMMON, ids=str)
def test_pool_and_table_refusals(fl, name, over):
    assert call(fl, name, over) == 1
    assert fl._lib.lib().fl_last_error()


@pytest.mark.parametrize("name,over", [
    *[(n, o) for n in ALL[:2] for o in (dict(k=None), dict(v=None), dict(starts=None), dict(pos0=None),
                                        dict(N=-1), dict(ks=1023), dict(vs=1028), dict(k=FAKE + 8))],
    *[("fl_attn_prep_paged", o) for o in (dict(q=None), dict(starts=None), dict(pos0=None), dict(N=-1),
                                          dict(wq=None), dict(qp=255), dict(rope=63), dict(rope=258),
                                          dict(nq=23), dict(q_out=FAKE, qop=128),
                                          dict(q_out=FAKE + 4, qop=256))],
    *[(n, o) for n in ALL[3:] for o in (dict(q=None), dict(z=None), dict(nq=23), dict(nq=0),
                                        dict(qp=256), dict(qp=516), dict(zp=128), dict(q=FAKE + 8),
                                        dict(window=-1), dict(sinks=-1))],
    ("fl_attention_prefill_paged", dict(Ts=None)), ("fl_attention_prefill_paged", dict(pos0s=None)),
    ("fl_attention_prefill_paged", dict(Ts=ints(1, -1))),
    ("fl_attention_prefill_paged", dict(pos0s=ints(0, -1))),
    ("fl_attention_prefill_paged", dict(Ts=ints(0, 4), pos0s=ints(0, 61))),
    ("fl_attention_prefill_paged", dict(B=65, Ts=ints(*[0] * 65), pos0s=ints(*[0] * 65))),
    ("fl_attn_decode_paged", dict(T=0)), ("fl_attn_decode_paged", dict(T=6)),
    ("fl_attn_decode_paged", dict(pos0=None)), ("fl_attn_decode_paged", dict(nq=132)),
], ids=str)
def test_argument_refusals(fl, name, over):
    assert call(fl, name, over) == 1
    assert fl._lib.lib().fl_last_error()


def test_nothing_to_do_is_ok(fl):
    for name in ALL[:4]:
        assert call(fl, name, {}) == 0


def test_op_layer_refuses_what_is_not_a_pool(fl):
    """Types, shapes and CPU tensors are refused before the library is called."""
    ops = fl.ops
    f16, i32 = torch.float16, torch.int32
    kp = torch.zeros((4, 16, 4, 256), dtype=f16)
    pages, starts, pos0 = torch.zeros((1, 4), dtype=i32), torch.zeros(2, dtype=i32), torch.zeros(1, dtype=i32)
    k = torch.zeros((3, 4, 256), dtype=f16)
    qg = torch.zeros((1, 1, 24, 512), dtype=f16)
    with pytest.raises(ValueError, match="GPU"):
        ops.paged_kv_store(k, k, kp, kp, pages, starts, pos0, page_size=16)
    with pytest.raises((TypeError, ValueError)):
        ops.paged_kv_store(k, k, kp, kp, pages, [0, 3], pos0, page_size=16)
    with pytest.raises(ValueError, match="starts"):
        ops.paged_kv_load(kp, kp, pages, starts[:1], pos0, T=3, page_size=16)
    with pytest.raises(ValueError):
        ops.attn_decode_paged(qg, kp, kp, pages, torch.zeros(2, dtype=i32), page_size=16)
    with pytest.raises(ValueError):
        ops.attn_decode_paged(qg, kp, kp, pages, pos0, page_size=32)
    with pytest.raises(TypeError):
        ops.attn_decode_paged(qg, None, kp, pages, pos0, page_size=16)
    with pytest.raises(ValueError):
        ops.attention_prefill_paged(qg[0], kp, kp, pages, [2], [0], page_size=16)
    with pytest.raises(ValueError):
        ops.attention_prefill_paged(qg[0], kp, kp, pages, [1, 0], [0], page_size=16)
    with pytest.raises(ValueError):
        ops.attention_prefill_paged(qg[0], kp, kp, pages, [], [], page_size=16)
    odd = torch.zeros(fl.geometry.kv8_nbytes(16) + 272, dtype=torch.int8)
    with pytest.raises(ValueError, match="pages"):
        ops.attn_decode_paged(qg, odd, odd, pages, pos0, page_size=16)


def test_int8_work_is_bounded_by_groups(fl):
    """Many long int8 contexts: the fp16 copies are made in groups of 1 GiB; fp16 pools need
    none, and work that is too small is refused."""
    f = fl.ops.attention_prefill_paged_work_bytes
    many = f([1] * 40, [100000] * 40, kv8=True)
    assert f([1], [100000], kv8=True) < many < (1 << 30) + (200 << 20)
    assert f([1] * 40, [100000] * 40) < 200 << 20
    assert f([0], [5], kv8=True) == 0 and f([1], [0]) == 0
    # a window's copy holds the window, not the context: 32-row tiles 2997 (row 95905 - 1)
    # .. 3126 and the first tokens' one, 4 KiB a row, beside an fp16 call's partials
    args = dict(window=4096, sinks=4)
    assert f([64], [100000], kv8=True, **args) - f([64], [100000], **args) == 131 * 32 * 4096
    for T, pos in (([1024], [30000]), ([1] * 40, [3000] * 40)):
        rc = call(fl, "fl_attention_prefill_paged",
                  dict(B=len(T), Ts=ints(*T), pos0s=ints(*pos), q8=1, max_pages=1 << 16, stride=1 << 16,
                       work=FAKE, wb=1024))
        assert rc == 3 and b"work" in fl._lib.lib().fl_last_error()
    assert call(fl, "fl_attn_decode_paged", dict(work=FAKE, wb=64)) == 3
    assert call(fl, "fl_attn_decode_paged", dict(work=FAKE + 8, wb=1 << 30)) == 1


def test_binding_is_built_and_declines_what_is_not_plain(fl):
    """The compiled binding loads with the library and leaves everything that is not a dense
    tensor on the current GPU (here: nothing is) to the checks in Python."""
    fl._lib.lib()
    lane = fl._lib.lane
    assert lane is not None, "fl355_paged.so is not built"
    F16, I32 = torch.float16, torch.int32
    k = torch.zeros(2, 4, 256, dtype=F16)
    pool, pages = torch.zeros(3, 16, 4, 256, dtype=F16), torch.zeros(1, 2, dtype=I32)
    starts, pos0 = torch.tensor([0, 2], dtype=I32), torch.zeros(1, dtype=I32)
    q, w = torch.zeros(2, 24, 512, dtype=F16), torch.zeros(256)
    calls = {
        "kv_store": (0, 0, k, k, starts, pos0, pool, pool, pages, 16, 4, 256),
        "kv_load": (0, 0, starts, pos0, pool, pool, pages, 2, 16, 4, 256),
        "prep": (0, 0, q, k, k, w, w, None, starts, pos0, pool, pool, pages, 16, 24, 4, 256, 64, 1e7, 1e-6),
        "prefill": (0, 0, q, pool, pool, pages, [2], [0], 16, 0, 0, True, None, None, 4, 0.0625),
        "decode": (0, 0, q[:, None], pool, pool, pages.expand(2, 2), pos0.expand(2), 16, 0, 0, True, None, None,
                   4, 0.0625),
    }
    for name, args in calls.items():
        call = getattr(lane, name)
        assert call(*args) is None and call(*args[:-1]) is None and call() is None
        for i in range(len(args)):          # any argument of another kind
            for other in (None, "x", 1 << 70, 0.5, [1], object()):
                assert call(*args[:i], other, *args[i + 1:]) is None, (name, i, other)
    with pytest.raises(TypeError):
        lane.bind(1, 2)
