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


def attn(fl, **over):
    a = dict(q=FAKE, qp=512, kpool=FAKE, vpool=FAKE, **POOL, **TABLE, pos0=FAKE, parents=FAKE, B=2, T=8, nq=24, kv=4,
             hd=256, scale=0.0625, window=0, sinks=0, gated=1, z=FAKE, zp=256, work=FAKE, wb=0)
    a.update(over)
    return fl._lib.lib().fl_attn_tree_paged(*a.values(), None)


def layer(**over):
    a = dict(x=FAKE, xs=10240, w=FAKE, cin=ptrs(FAKE, FAKE), pos0=ints(5, 5), nodes=FAKE, a=FAKE, b=FAKE, abs=48,
             A=FAKE, dt=FAKE, S=ptrs(FAKE, FAKE))
    return {**a, **{k: v for k, v in over.items() if k in a}}


def gdn_tree(fl, **over):
    a = dict(z=FAKE, zp=6144, nw=FAKE, y=FAKE, yp=6144, B=2, T=8, nk=16, nv=48, K=128, V=128, s=0.1, l2=1e-6, eps=1e-6)
    a.update({k: v for k, v in over.items() if k in a})
    return fl._lib.lib().fl_gdn_tree_normed(*layer(**over).values(), *a.values(), None)


BIG = 1 << 28


def gdn_commit(fl, **over):
    c = layer(**{"S": ptrs(BIG, 2 * BIG), **over})
    a = dict(cout=ptrs(3 * BIG, 4 * BIG), So=ptrs(BIG, 2 * BIG), B=2, T=8, D=4, nk=16, nv=48, K=128, V=128, l2=1e-6)
    a.update({k: v for k, v in over.items() if k in a})
    return fl._lib.lib().fl_gdn_tree_commit(c["x"], c["xs"], c["w"], c["cin"], a["cout"], c["pos0"], c["nodes"], c["a"],
                                            c["b"], c["abs"], c["A"], c["dt"], c["S"], a["So"], a["B"], a["T"], a["D"],
                                            a["nk"], a["nv"], a["K"], a["V"], a["l2"], None)


GDN = [dict(x=None), dict(w=None), dict(cin=None), dict(pos0=None), dict(nodes=None), dict(a=None), dict(b=None),
       dict(A=None), dict(dt=None), dict(S=None), dict(S=ptrs(FAKE, None)), dict(S=ptrs(FAKE, FAKE + 4)),
       dict(cin=ptrs(FAKE, FAKE + 8)), dict(pos0=ints(5, -1)), dict(B=0), dict(B=17), dict(T=0), dict(T=65), dict(K=64),
       dict(V=64), dict(nk=0), dict(nk=5), dict(nv=0), dict(xs=10232), dict(xs=10244), dict(x=FAKE + 8), dict(w=FAKE + 2),
       dict(abs=47)]
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
    *[(attn, o) for o in SIZES + TABLES + [
        dict(kpool=None), dict(vpool=FAKE + 8), dict(q=None), dict(z=None), dict(pos0=None), dict(parents=None), dict(T=0),
        dict(T=65), dict(nq=0), dict(nq=23), dict(nq=4100), dict(qp=256), dict(qp=516), dict(zp=128), dict(q=FAKE + 8),
        dict(window=-1), dict(sinks=-1), dict(scale=0.0), dict(work=FAKE + 8, wb=1 << 40)]],
    *[(copy, o) for o in SIZES + LAYERS + [dict(n=-1), dict(n=1, src=None), dict(n=1, dst=None),
                                           dict(n=1 << 30, page_size=1 << 15)]],
    *[(f, o) for f in (gdn_tree, gdn_commit) for o in GDN],
    *[(gdn_tree, o) for o in (dict(z=None), dict(nw=None), dict(y=None), dict(zp=6136), dict(yp=6140), dict(y=FAKE + 8),
                              dict(nw=FAKE + 4))],
    *[(gdn_commit, o) for o in (
        dict(cout=None), dict(So=None), dict(D=0), dict(D=65), dict(cout=ptrs(3 * BIG, None)), dict(So=ptrs(BIG, None)),
        dict(cout=ptrs(FAKE, 4 * BIG)), dict(cout=ptrs(3 * BIG, FAKE + 61424)), dict(cout=ptrs(3 * BIG, 3 * BIG + 32)),
        dict(So=ptrs(3 * BIG, 3 * BIG)), dict(So=ptrs(2 * BIG, BIG)), dict(So=ptrs(BIG + 64, 2 * BIG)))],
    *[(keep, o) for o in SIZES + TABLES + LAYERS + [dict(D=-1), dict(pos0=None), dict(D=1, path=None)]],
], ids=lambda x: getattr(x, "__name__", None) or str({k: v for k, v in x.items() if not isinstance(v, ctypes.Array)}))
def test_refusals(fl, f, over):
    assert f(fl, **over) == 1
    assert fl._lib.lib().fl_last_error()


def test_nothing_to_do_is_ok(fl):
    assert prep_axes(fl) == copy(fl) == keep(fl) == 0


def test_work_of_a_tree(fl):
    """Too little is refused; it does not grow with the batch but for 8 bytes a sequence."""
    f = fl.ops.attn_tree_paged_work_bytes
    assert attn(fl) == 3 and attn(fl, work=None, wb=1 << 40) == 3 and b"work" in fl._lib.lib().fl_last_error()
    assert 0 < f(1000, 26) - f(1, 26) <= 8000
    assert f(1, 65) == f(0, 1) == f(1, 1, 23) == f(1025, 1) == 0


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
    qg, parents = torch.zeros((1, 3, 24, 512), dtype=F16), torch.zeros((1, 3), dtype=I32)
    with pytest.raises(ValueError, match="GPU"):
        ops.attn_tree_paged(qg, pool, pool, pages, pos0, parents, page_size=16)
    with pytest.raises(ValueError, match="parents"):
        ops.attn_tree_paged(qg, pool, pool, pages, pos0, parents[:, :2], page_size=16)
    with pytest.raises(TypeError, match="parents"):
        ops.attn_tree_paged(qg, pool, pool, pages, pos0, [[-1, 0, 0]], page_size=16)


def test_op_layer_refuses_gdn_trees(fl):
    ops = fl.ops
    x, a, A = torch.zeros((1, 3, 10240), dtype=F16), torch.zeros((1, 3, 48)), torch.zeros(48)
    S, z, w = [torch.zeros(48, 128, 128)], torch.zeros((1, 3, 6144), dtype=F16), torch.zeros(128)
    nodes, cw, cst = torch.zeros((1, 3), dtype=I32), torch.zeros((10240, 4), dtype=F16), [torch.zeros((10240, 3), dtype=F16)]
    kw = dict(pos0s=[1], conv_w=cw, cst_in=cst)
    with pytest.raises(ValueError, match="GPU"):
        ops.gdn_tree_normed(x, S, a, a, A, A, z, w, nodes, **kw)
    with pytest.raises(ValueError, match="parents"):
        ops.gdn_tree_normed(x, S, a, a, A, A, z, w, nodes[:, :2], **kw)
    with pytest.raises(ValueError, match="x: shape"):
        ops.gdn_tree_normed(x[..., :8192], S, a, a, A, A, z, w, nodes, **kw)
    with pytest.raises(ValueError, match="a, b"):
        ops.gdn_tree_normed(x, S, a, a[:, :2], A, A, z, w, nodes, **kw)
    with pytest.raises(ValueError, match="one a sequence"):
        ops.gdn_tree_normed(x, S, a, a, A, A, z, w, nodes, pos0s=[1, 2], conv_w=cw, cst_in=cst)
    with pytest.raises(TypeError):
        ops.gdn_tree_commit(x, S, a, a, A, A, [[0, 1]], cst_out=cst, **kw)
    with pytest.raises(ValueError, match="GPU"):
        ops.gdn_tree_commit(x, S, a, a, A, A, nodes, cst_out=cst, **kw)


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
    calls["tree"] = (0, 0, q[None], pool, pool, pages, pos0, pages, 16, 0, 0, True, None, None, 4, 0.0625)
    x, a, A = torch.zeros((1, 3, 10240), dtype=F16), torch.zeros((1, 3, 48)), torch.zeros(48)
    layer = (0, 0, x, [torch.zeros(48, 128, 128)], a, a, A, A)
    cw, cst = torch.zeros((10240, 4), dtype=F16), [torch.zeros((10240, 3), dtype=F16)]
    calls["gdn_tree"] = (*layer, torch.zeros((1, 3, 6144), dtype=F16), A, pages, None, [1], cw, cst, 16, 48, 128, 128, 0.1,
                         1e-6, 1e-6)
    calls["gdn_commit"] = (*layer, pages, [torch.zeros(48, 128, 128)], [1], cw, cst, cst, 16, 48, 128, 128, 1e-6)
    for name, args in calls.items():
        call = getattr(lane, name)
        assert call(*args) is None and call(*args[:-1]) is None and call() is None
        for i in range(len(args)):          # any argument of another kind
            for other in (None, "x", 1 << 70, 0.5, [1], [], [None], (pool, None), object()):
                assert call(*args[:i], other, *args[i + 1:]) is None, (name, i, other)
