"""The entry points of trees of drafted tokens on the CPU: what they refuse, before any launch."""
import ctypes

import pytest
import torch

FAKE = 1 << 20   # an aligned address that is never read

F16, F32, I32 = torch.float16, torch.float32, torch.int32


def ints(*v):
    return (ctypes.c_int * max(1, len(v)))(*v)


def ptrs(*v):
    return (ctypes.c_void_p * max(1, len(v)))(*v)


POOL = dict(q8=0, n_pages=8, page_size=16)
TABLE = dict(pages=FAKE, max_pages=4, stride=4)


def prep_axes(fl, **over):
    a = dict(q=FAKE, qp=512, k=FAKE, v=FAKE, wq=FAKE, wk=FAKE, q_out=None, qop=0, kpool=FAKE, vpool=FAKE,
             **POOL, **TABLE, starts=FAKE, pos0=FAKE, positions=FAKE, axes=3, of=ints(*[0] * 16, *[2] * 16),
             B=2, N=0, nq=24, kv=4, hd=256, rope=64)
    a.update(over)
    return fl._lib.lib().fl_attn_prep_axes(*a.values(), 1e7, 1e-6, None)


def copy(fl, **over):
    a = dict(ks=ptrs(FAKE, FAKE), vs=ptrs(FAKE, FAKE), layers=2, **POOL, src=FAKE, dst=FAKE, n=0, kv=4, hd=256)
    a.update(over)
    return fl._lib.lib().fl_paged_kv_copy(*a.values(), None)


def keep(fl, **over):
    a = dict(ks=ptrs(FAKE, FAKE), vs=ptrs(FAKE, FAKE), layers=2, **POOL, **TABLE, pos0=FAKE, path=FAKE, B=2, D=0,
             kv=4, hd=256)
    a.update(over)
    return fl._lib.lib().fl_paged_kv_keep(*a.values(), None)


SIZES = [dict(q8=2), dict(hd=128), dict(kv=0), dict(page_size=8), dict(page_size=48), dict(n_pages=0),
         dict(n_pages=1 << 30)]
TABLES = [dict(pages=None), dict(max_pages=0), dict(stride=3), dict(B=0), dict(B=1025),
          dict(max_pages=1 << 27, stride=1 << 27)]
LAYERS = [dict(ks=None), dict(vs=None), dict(layers=0), dict(layers=65, ks=ptrs(*[FAKE] * 65), vs=ptrs(*[FAKE] * 65)),
          dict(ks=ptrs(FAKE, None)), dict(vs=ptrs(FAKE, FAKE + 8))]


@pytest.mark.parametrize("f,over", [
    *[(prep_axes, o) for o in SIZES + TABLES + [
        dict(kpool=None), dict(vpool=FAKE + 8), dict(positions=None), dict(of=None), dict(axes=0), dict(axes=2),
        dict(axes=129), dict(of=ints(*[-1] * 32)), dict(starts=None), dict(pos0=None), dict(N=-1), dict(rope=63),
        dict(qp=255), dict(nq=23), dict(q_out=FAKE, qop=128)]],
    *[(copy, o) for o in SIZES + LAYERS + [dict(n=-1), dict(n=1, src=None), dict(n=1, dst=None),
                                           dict(n=1 << 30, page_size=1 << 15)]],
    *[(keep, o) for o in SIZES + TABLES + LAYERS + [dict(D=-1), dict(pos0=None), dict(D=1, path=None)]],
], ids=lambda x: getattr(x, "__name__", None) or str({k: v for k, v in x.items() if not isinstance(v, ctypes.Array)}))
def test_refusals(fl, f, over):
    assert f(fl, **over) == 1
    assert fl._lib.lib().fl_last_error()


def test_nothing_to_do_is_ok(fl):
    assert prep_axes(fl) == copy(fl) == keep(fl) == 0


def test_op_layer_refuses(fl):
    """Types, shapes and CPU tensors, before the library is called."""
    ops = fl.ops
    pool = torch.zeros((4, 16, 4, 256), dtype=F16)
    pages, starts, pos0 = torch.zeros((1, 4), dtype=I32), torch.tensor([0, 3], dtype=I32), torch.zeros(1, dtype=I32)
    ids, path = torch.zeros(2, dtype=I32), torch.zeros((1, 2), dtype=I32)
    with pytest.raises(ValueError, match="GPU"):
        ops.paged_kv_copy(pool, pool, ids, ids, page_size=16)
    with pytest.raises(ValueError, match="GPU"):
        ops.paged_kv_keep([pool], [pool], pages, pos0, path, page_size=16)
    with pytest.raises(ValueError, match="src"):
        ops.paged_kv_copy(pool, pool, ids, ids[:1], page_size=16)
    with pytest.raises(TypeError):
        ops.paged_kv_copy(pool, pool, [1], [2], page_size=16)
    with pytest.raises(ValueError, match="layer"):
        ops.paged_kv_copy([pool], [pool, pool], ids, ids, page_size=16)
    with pytest.raises(ValueError, match="layer"):
        ops.paged_kv_copy([], [], ids, ids, page_size=16)
    with pytest.raises(ValueError, match="path"):
        ops.paged_kv_keep([pool], [pool], pages, pos0, path[0], page_size=16)
    x = (torch.zeros((3, 24, 512), dtype=F16), torch.zeros((3, 4, 256), dtype=F16), torch.zeros((3, 4, 256), dtype=F16),
         torch.zeros(256), torch.zeros(256), pool, pool, pages, starts, pos0)
    at = torch.zeros((3, 3), dtype=I32)
    with pytest.raises(ValueError, match="sections"):
        ops.attn_prep_axes(*x, at, page_size=16)
    with pytest.raises(ValueError, match="sections"):
        ops.attn_prep_axes(*x, at, page_size=16, sections=(16, 8, 9))
    with pytest.raises(ValueError, match="sections"):
        ops.attn_prep_axes(*x, at, page_size=16, sections=(40, -4, -4))
    with pytest.raises(ValueError, match="axis 2"):
        ops.attn_prep_axes(*x, at, page_size=16, sections=(10, 11, 11), interleaved=True)
    with pytest.raises(ValueError, match="positions"):
        ops.attn_prep_axes(*x, at[0], page_size=16)
    with pytest.raises(TypeError):
        ops.attn_prep_axes(*x, None, page_size=16)
    with pytest.raises(ValueError, match="GPU"):
        ops.attn_prep_axes(*x, at, page_size=16, sections=(16, 8, 8))


def test_the_pairs_of_every_axis(fl):
    of = fl.ops._pair_axes
    assert of(3, (2, 1, 1), False, 8) == (0, 0, 1, 2)
    assert of(3, (12, 10, 10), True, 64) == tuple([0, 1, 2] * 10 + [0, 0])
    assert of(3, (11, 11, 10), True, 64) == tuple([0, 1, 2] * 10 + [0, 1])
    assert of(1, None, True, 64) == (0,) * 32
    for sections in ((24, 4, 4), (30, 1, 1), (32, 0, 0), (11, 11, 10)):
        assert [of(3, sections, True, 64).count(a) for a in range(3)] == list(sections)


def test_binding_declines_what_is_not_plain(fl):
    fl._lib.lib()
    lane = fl._lib.lane
    assert lane is not None, "fl355_paged.so is not built"
    k = torch.zeros(2, 4, 256, dtype=F16)
    pool, pages = torch.zeros(3, 16, 4, 256, dtype=F16), torch.zeros(1, 2, dtype=I32)
    starts, pos0 = torch.tensor([0, 2], dtype=I32), torch.zeros(1, dtype=I32)
    q, w, ids, path = torch.zeros(2, 24, 512, dtype=F16), torch.zeros(256), torch.zeros(2, dtype=I32), pages
    calls = {
        "prep_axes": (0, 0, q, k, k, w, w, None, starts, pos0, pool, pool, pages, 16, 24, 4, 256, 64, 1e7, 1e-6,
                      pages, (0,) * 32),
        "kv_copy": (0, 0, [pool], [pool], ids, ids, 16, 4, 256),
        "kv_keep": (0, 0, [pool], (pool,), pages, pos0, path, 16, 4, 256),
    }
    for name, args in calls.items():
        call = getattr(lane, name)
        assert call(*args) is None and call(*args[:-1]) is None and call() is None
        for i in range(len(args)):          # any argument of another kind
            for other in (None, "x", 1 << 70, 0.5, [1], [], [None], (pool, None), object()):
                assert call(*args[:i], other, *args[i + 1:]) is None, (name, i, other)
