"""Calls of the tree operators that are refused on the host for what a kernel would do with them."""
import pytest

from test_tree_abi import BIG, attn, gdn_commit, gdn_tree, keep, ptrs


@pytest.mark.parametrize("B,pages,page_size,rc", [
    (1024, 1 << 22, 16, 1), (1024, (1 << 22) - 400, 16, 1), (1024, (1 << 22) - 4800, 16, 3), (32, 127, 1 << 24, 3),
    (33, 127, 1 << 24, 1), (1024, 1 << 21, 16, 3)])
def test_a_batch_of_more_tiles_than_a_run_can_count(fl, B, pages, page_size, rc):
    """A run is up to 1.0001 times all tiles and starts long, in 32 bits: with nearly 2^31 of them (and one
    workgroup a kv head) it would come out negative, and the merge would read slots that nobody wrote.
    Status 3: only the work is too small."""
    assert attn(fl, B=B, max_pages=pages, stride=pages, page_size=page_size, n_pages=8) == rc
    if rc == 1:
        assert b"max_pages" in fl._lib.lib().fl_last_error()


WIDTH, DIM, STATE = 6144, 10240, 48 * 128 * 128


def gdn(fl, **over):
    """gdn_tree of 2 sequences of 8 tokens, every buffer BIG bytes behind the one before it."""
    at = {name: (i + 1) * BIG for i, name in enumerate(
        ("x", "w", "nodes", "a", "b", "A", "dt", "z", "nw", "y", "S0", "S1", "c0", "c1"))}
    at.update({k: v for k, v in over.items() if k in at})
    args = {k: v for k, v in at.items() if k not in ("S0", "S1", "c0", "c1")}
    args.update({k: v for k, v in over.items() if k not in at})
    rc = gdn_tree(fl, S=ptrs(at["S0"], at["S1"]), cin=ptrs(at["c0"], at["c1"]), **args)
    return rc, fl._lib.lib().fl_last_error()


@pytest.mark.parametrize("name,bytes_", [
    ("x", 16 * DIM * 2), ("w", DIM * 8), ("nodes", 16 * 4), ("a", 16 * 48 * 4), ("b", 16 * 48 * 4), ("A", 48 * 4),
    ("dt", 48 * 4), ("z", 16 * WIDTH * 2), ("nw", 128 * 4), ("S0", STATE * 4), ("S1", STATE * 4), ("c0", DIM * 6),
    ("c1", DIM * 6)])
def test_y_over_an_input_of_the_gdn_layer(fl, name, bytes_):
    """Its first and its last 16 bytes: a workgroup that is done writes what another has yet to read."""
    for y in (BIG * 20 - 16 * WIDTH * 2 + 16, BIG * 20 + (bytes_ - 16) // 16 * 16):
        rc, error = gdn(fl, y=y, **{name: BIG * 20})
        assert rc == 1 and b"overlap" in error, (name, rc, error)


@pytest.mark.parametrize("over", [
    dict(z=BIG * 20, zp=WIDTH * 2, y=BIG * 20 + WIDTH * 2 - 16, yp=WIDTH * 2),
    dict(z=BIG * 20, zp=WIDTH * 2, y=BIG * 20 + WIDTH * 2 + 16, yp=WIDTH * 2),
    dict(z=BIG * 20, zp=WIDTH * 2, y=BIG * 20 + WIDTH * 2, yp=WIDTH * 2 + 8),
    dict(x=BIG * 20, xs=20480, y=BIG * 20 - WIDTH * 2 + 16, yp=20480)])
def test_y_in_the_rows_of_an_input(fl, over):
    rc, error = gdn(fl, **over)
    assert rc == 1 and b"overlap" in error, (rc, error)


def commit(fl, **over):
    at = {name: (i + 1) * BIG for i, name in enumerate(
        ("x", "w", "nodes", "a", "b", "A", "dt", "S0", "S1", "So0", "So1", "c0", "c1", "co0", "co1"))}
    at.update(over)
    pairs = dict(S="S", So="So", cin="c", cout="co")
    args = {k: v for k, v in at.items() if k.rstrip("01") not in pairs.values()}
    rc = gdn_commit(fl, **args, **{k: ptrs(at[v + "0"], at[v + "1"]) for k, v in pairs.items()})
    return rc, fl._lib.lib().fl_last_error()


@pytest.mark.parametrize("out,size", [("So0", STATE * 4), ("So1", STATE * 4), ("co0", DIM * 6), ("co1", DIM * 6)])
@pytest.mark.parametrize("name,bytes_", [
    ("x", 16 * DIM * 2), ("w", DIM * 8), ("nodes", 8 * 4), ("a", 16 * 48 * 4), ("b", 16 * 48 * 4), ("A", 48 * 4),
    ("dt", 48 * 4), ("S0", STATE * 4), ("S1", STATE * 4), ("c0", DIM * 6), ("c1", DIM * 6), ("So0", STATE * 4),
    ("So1", STATE * 4), ("co0", DIM * 6), ("co1", DIM * 6)])
def test_outputs_of_a_commit_over_other_buffers(fl, out, size, name, bytes_):
    if name == out:
        return
    for p in (BIG * 20 - size + 16, BIG * 20 + (bytes_ - 16) // 16 * 16):
        rc, error = commit(fl, **{out: p, name: BIG * 20})
        assert rc == 1 and b"overlap" in error, (rc, error)


def attention(fl, **over):
    """attn_tree_paged of 2 sequences of 8 tokens, every buffer BIG bytes behind the one before it."""
    names = ("q", "kpool", "vpool", "pages", "pos0", "parents", "z", "work")
    at = {name: (i + 1) * BIG for i, name in enumerate(names)}
    at["wb"] = fl.ops.attn_tree_paged_work_bytes(2, 8)
    at.update(over)
    return attn(fl, **at), fl._lib.lib().fl_last_error()


@pytest.mark.parametrize("q8", [0, 1])
@pytest.mark.parametrize("out", ["z", "work"])
@pytest.mark.parametrize("name", ["q", "kpool", "vpool", "pages", "pos0", "parents", "z", "work"])
def test_outputs_of_the_attention_over_other_buffers(fl, out, name, q8):
    work = fl.ops.attn_tree_paged_work_bytes(2, 8)
    sizes = dict(q=16 * 24 * 1024, kpool=8 * 16 * 4 * (272 if q8 else 512), vpool=8 * 16 * 4 * (272 if q8 else 512),
                 pages=8 * 4, pos0=2 * 4, parents=16 * 4, z=16 * 24 * 512, work=work)
    if name == out:
        return
    first = BIG * 20 - sizes[out] + 16
    for p in (first - first % 16, BIG * 20 + (sizes[name] - 4) // 16 * 16):
        rc, error = attention(fl, **{out: p, name: BIG * 20}, q8=q8)
        assert rc == 1 and b"overlap" in error, (rc, error)


@pytest.mark.parametrize("over", [dict(z=BIG * 20 + 512, zp=512), dict(z=BIG * 20, zp=512, gated=0),
                                  dict(z=BIG * 20 + 1016, zp=512, gated=0), dict(z=BIG * 20 + 1024, zp=520)])
def test_z_in_the_rows_of_q(fl, over):
    rc, error = attention(fl, q=BIG * 20, **over)
    assert rc == 1 and b"overlap" in error, (rc, error)


@pytest.mark.parametrize("q8,bytes_", [(0, 8 * 16 * 4 * 512), (1, 8 * 16 * 4 * 272)])
@pytest.mark.parametrize("ks,vs", [((1, 1), (2, 3)), ((1, 2), (1, 3)), ((3, 2), (1, 2))])
def test_accepted_rows_of_a_pool_that_is_there_twice(fl, ks, vs, q8, bytes_):
    """Two workgroups would move its rows, one of them from where the other has written."""
    for shift in (0, bytes_ - 16):      # the second time it comes
        at, seen = [], set()
        for n in (*ks, *vs):
            at.append(BIG * n + (shift if n in seen else 0))
            seen.add(n)
        assert keep(fl, ks=ptrs(*at[:2]), vs=ptrs(*at[2:]), q8=q8, D=1) == 1
        assert b"overlap" in fl._lib.lib().fl_last_error()
