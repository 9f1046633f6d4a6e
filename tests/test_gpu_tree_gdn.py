"""The GDN layer over trees of drafted tokens, and the state behind an accepted path, against
the recurrence in float64 (tree_ref.py, which derives the bounds)."""
import pytest
import torch

import tree_ref as ref

pytestmark = pytest.mark.gpu

F16, F32, I32 = torch.float16, torch.float32, torch.int32


def gen(seed):
    return torch.Generator().manual_seed(seed)


def tree(g, n, T, kind="any"):
    """n tokens' parents, then places without a token."""
    if kind == "chain":
        p = list(range(-1, n - 1))
    elif kind == "star":
        p = [-1] * n
    elif kind == "binary":
        p = [(i - 1) // 2 if i else -1 for i in range(n)]
    else:
        p = [int(torch.randint(-1, i, (1,), generator=g)) if i else -1 for i in range(n)]
    return p + [-2] * (T - n)


def i32(rows):
    return torch.tensor(rows, dtype=I32).cuda()


def run(fl, d, parents, pos0, **kw):
    return fl.ops.gdn_tree_normed(d["x"], d["S"], d["a"], d["b"], d["A_log"], d["dt_bias"], d["z"], d["norm_w"],
                                  i32(parents), pos0s=pos0, conv_w=d["conv_w"], cst_in=d["cst"],
                                  n_kheads=d["n_k"], n_vheads=d["n_v"], **kw)


def check(got, want, bound, what):
    err = (got.double() - want).abs()
    assert torch.isfinite(got).all(), f"{what}: not finite"
    worst = (err / bound.clamp_min(1e-300))[err > 0].max().item() if (err > 0).any() else 0.0
    print(f"{what}: max|err| {err.max().item():.2e}, {worst:.2f} of the bound")
    assert worst <= 1.0, f"{what}: {worst} of the bound"


@pytest.mark.parametrize("B,sizes,T,kind", [
    (1, [1], 1, "any"), (1, [2], 2, "chain"), (1, [5], 5, "star"), (1, [16], 16, "any"), (2, [17, 3], 17, "binary"),
    (3, [33, 0, 20], 33, "any"), (1, [48], 48, "binary"), (1, [64], 64, "chain"), (2, [64, 49], 64, "any"),
    (1, [64], 64, "star"), (16, [7] * 16, 7, "any")])
def test_against_the_recurrence(fl, B, sizes, T, kind):
    g = gen(T + B)
    d = ref.gdn_layer(g, B, T)
    parents = [tree(g, n, T, kind) for n in sizes]
    pos0 = [0 if b == 1 else 100 + b for b in range(B)]
    keep = [s.clone() for s in d["S"]], [c.clone() for c in d["cst"]]
    y = run(fl, d, parents, pos0)
    want, bound = ref.gdn_tree(d, parents, [p == 0 for p in pos0])
    check(y, want, bound, f"B {B} T {T} {kind}")
    for b in range(B):
        assert (y[b, sizes[b]:] == 0).all()
        assert torch.equal(d["S"][b], keep[0][b]) and torch.equal(d["cst"][b], keep[1][b])


@pytest.mark.parametrize("n_k,n_v", [(1, 1), (4, 4), (2, 10), (8, 16)])
def test_other_head_counts_and_strides(fl, n_k, n_v):
    g = gen(n_v)
    d = ref.gdn_layer(g, 2, 21, n_k, n_v, extra=24, ab_extra=3)
    parents = [tree(g, 21, 21), tree(g, 13, 21)]
    want, bound = ref.gdn_tree(d, parents, [False, False])
    y = torch.full((2, 21, n_v * 128), 7.0, dtype=F16, device="cuda")
    assert run(fl, d, parents, [5, 6], y=y) is y
    check(y, want, bound, f"{n_k} / {n_v} heads")


@pytest.mark.parametrize("n_k,n_v,B,T", [(16, 48, 6, 16), (16, 48, 7, 19), (16, 48, 6, 41), (16, 48, 6, 64),
                                         (16, 32, 9, 9), (8, 32, 16, 32), (16, 32, 12, 48), (3, 18, 15, 33),
                                         (5, 25, 11, 20)])
def test_batches_of_several_heads_a_workgroup(fl, n_k, n_v, B, T):
    g = gen(100 * B + T)
    d = ref.gdn_layer(g, B, T, n_k, n_v)
    parents = [tree(g, int(torch.randint(0, T + 1, (1,), generator=g)), T) for _ in range(B)]
    parents[0] = tree(g, T, T, "binary")
    pos0 = [b % 3 for b in range(B)]
    want, bound = ref.gdn_tree(d, parents, [p == 0 for p in pos0])
    check(run(fl, d, parents, pos0), want, bound, f"{n_k} / {n_v} heads, B {B} T {T}")


@pytest.mark.parametrize("state,values", [(0.0, 0.0), (0.0, 1.0), (1e-30, 0.0), (1e-30, 1e-3), (1e-6, 1.0),
                                          (1e6, 1.0), (1e15, 0.0), (1e15, 1.0)])
@pytest.mark.parametrize("B,T", [(1, 37), (6, 18)])
def test_states_and_values_of_other_sizes(fl, B, T, state, values):
    """Also rows of the state whose values are all 0 beside others: the scales of the terms are a row's."""
    g = gen(B)
    d = ref.gdn_layer(g, B, T)
    for s in d["S"]:
        s *= state * 20
        s[:, ::5] = 0
    d["conv_w"][2 * 16 * 128:] *= values
    d["conv_w"][2 * 16 * 128::3] = 0
    parents = [tree(g, T - b, T) for b in range(B)]
    want, bound = ref.gdn_tree(d, parents, [False] * B)
    check(run(fl, d, parents, [7] * B), want, bound, f"states {state}, values {values}")


def test_places_without_a_token_do_not_matter(fl):
    """Whatever they hold: parents out of order or range, descendants of such places, NaN rows."""
    g = gen(8)
    T = 40
    d = ref.gdn_layer(g, 1, T)
    parents = [tree(g, T, T)]
    for i, p in ((3, 3), (9, 30), (17, -2), (20, 17), (25, 20), (38, 2**31 - 1), (39, -2**31)):
        parents[0][i] = p
    gone = [i for i, line in enumerate(ref.lines(parents[0])) if line is None]
    assert {3, 9, 17, 20, 25, 38, 39} <= set(gone)
    want, bound = ref.gdn_tree(d, parents, [False])
    for t in (d["x"], d["a"], d["b"], d["z"]):
        t[0, gone] = float("nan")
    y = run(fl, d, parents, [9])
    check(y, want, bound, "absent places")
    assert (y[0, gone] == 0).all()


def test_extreme_gates(fl):
    """Decays that vanish (and states that are forgotten with them) and gates at 0 and 1."""
    g = gen(4)
    d = ref.gdn_layer(g, 1, 30)
    d["a"][0, ::3] = 300.0
    d["a"][0, 1::3] = -90.0
    d["b"][0, ::4] = 200.0
    d["b"][0, 1::4] = -200.0
    d["A_log"][:8] = 4.0
    d["A_log"][8:12] = -20.0
    parents = [tree(g, 30, 30, "binary")]
    y = run(fl, d, parents, [3])
    want, bound = ref.gdn_tree(d, parents, [False])
    check(y, want, bound, "extreme gates")


def test_a_chain_is_the_decode_step_by_step(fl):
    """The same tokens through gdn_decode_normed, one after the other: its conv output, q, k and o are
    rounded to fp16 (half a step each: 2^-11 of u's terms and of y), so the two differ by more than
    either from the formulas; 2^-7 of a row's largest value is 16 such roundings."""
    g = gen(6)
    T = 9
    d = ref.gdn_layer(g, 1, T)
    y = run(fl, d, [tree(g, T, T, "chain")], [50])
    S, ring = d["S"][0].clone(), [d["cst"][0].clone(), torch.empty_like(d["cst"][0])]
    for t in range(T):
        step = fl.ops.gdn_decode_normed(d["x"][0, t:t + 1], [S], d["a"][0, t:t + 1], d["b"][0, t:t + 1], d["A_log"],
                                        d["dt_bias"], d["z"][0, t:t + 1], d["norm_w"], pos0s=[50 + t],
                                        conv_w=d["conv_w"], cst_in=[ring[t % 2]], cst_out=[ring[1 - t % 2]])
        heads = step.double().view(48, 128), y[0, t].double().view(48, 128)
        assert ((heads[0] - heads[1]).abs() <= 2.0 ** -7 * heads[0].abs().amax(-1, keepdim=True)).all()
    out = torch.empty_like(d["cst"][0])
    fl.ops.gdn_tree_commit(d["x"], d["S"], d["a"], d["b"], d["A_log"], d["dt_bias"], i32([list(range(T))]),
                           pos0s=[50], conv_w=d["conv_w"], cst_in=d["cst"], cst_out=[out])
    assert torch.equal(out, ring[T % 2])
    assert ((d["S"][0] - S).abs() <= 2.0 ** -7 * S.abs().amax((-1, -2), keepdim=True)).all()


def commit(fl, d, paths, pos0, in_place):
    outs = [torch.full_like(c, 9.0) for c in d["cst"]]
    S = [s.clone() for s in d["S"]]
    to = None if in_place else [torch.full_like(s, 9.0) for s in S]
    fl.ops.gdn_tree_commit(d["x"], S, d["a"], d["b"], d["A_log"], d["dt_bias"], i32(paths), to, pos0s=pos0,
                           conv_w=d["conv_w"], cst_in=d["cst"], cst_out=outs, n_kheads=d["n_k"],
                           n_vheads=d["n_v"])
    if not in_place:
        for a, b in zip(S, d["S"]):
            assert torch.equal(a, b)
    return (S if in_place else to), outs


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("T,paths", [
    (1, [[0]]), (16, [[0, 3, 4, 9]]), (9, [[-1, 2, 3]]), (20, [[5], [-1], [19]]), (20, [[0, 1, -1], [2, 2, 3], [3, 4, 20]]),
    (64, [list(range(64))]), (26, [[i, i + 9, -1] for i in range(16)]), (12, [[2**31 - 1, 1], [11, -2**31]])])
def test_the_state_behind_a_path(fl, T, paths, in_place):
    g = gen(T)
    B = len(paths)
    d = ref.gdn_layer(g, B, T)
    pos0 = [0 if b % 3 == 1 else 40 for b in range(B)]
    S, frames = commit(fl, d, paths, pos0, in_place)
    for b, (want, bound, f) in enumerate(ref.gdn_commit(d, paths, [p == 0 for p in pos0])):
        check(S[b], want, bound, f"T {T} sequence {b}")
        assert torch.equal(frames[b].view(torch.int16), f.view(torch.int16))
        if not ref.accepted(paths[b], T):
            assert torch.equal(S[b], d["S"][b])


@pytest.mark.parametrize("n_k,n_v", [(1, 1), (2, 10), (4, 4)])
def test_commit_of_other_head_counts(fl, n_k, n_v):
    d = ref.gdn_layer(gen(n_v), 2, 8, n_k, n_v, extra=8, ab_extra=1)
    paths = [[0, 2, 7], [1, 3, 4]]
    S, frames = commit(fl, d, paths, [3, 3], True)
    for b, (want, bound, f) in enumerate(ref.gdn_commit(d, paths, [False] * 2)):
        check(S[b], want, bound, f"{n_k} / {n_v} heads, sequence {b}")
        assert torch.equal(frames[b], f)


def test_a_branch_after_its_commit_is_the_branch_in_the_tree(fl):
    """Verified in the tree or after its ancestors were committed: the same outputs but for fp32."""
    g = gen(12)
    T = 24
    d = ref.gdn_layer(g, 1, T)
    parents = tree(g, T, T, "binary")
    y = run(fl, d, [parents], [10])
    S, frames = commit(fl, d, [[0, 2, -1]], [10], False)
    rest = [i for i in range(T) if (ref.lines(parents)[i] + [-1, -1])[:2] == [0, 2] and i > 2]
    e = dict(d, S=S, cst=frames, **{n: d[n][:, rest].contiguous() for n in ("x", "a", "b", "z")})
    local = [rest.index(parents[i]) if parents[i] in rest else -1 for i in rest]
    y2 = run(fl, e, [local], [12])
    want, bound = ref.gdn_tree(d, [parents], [False])
    assert ((y2.double() - y[:, rest].double()).abs() <= 2 * bound[:, rest]).all()


def test_in_a_graph_with_other_trees_and_paths(fl):
    g = gen(20)
    T, B = 30, 2
    d = ref.gdn_layer(g, B, T)
    parents, path = i32([tree(g, T, T)] * B), i32([[0, -1, -1]] * B)
    y, outs = torch.empty(B, T, 48 * 128, dtype=F16, device="cuda"), [torch.empty_like(c) for c in d["cst"]]
    S_out = [torch.empty_like(s) for s in d["S"]]

    def calls(y, S_out, outs):
        fl.ops.gdn_tree_normed(d["x"], d["S"], d["a"], d["b"], d["A_log"], d["dt_bias"], d["z"], d["norm_w"],
                               parents, y, pos0s=[4, 0], conv_w=d["conv_w"], cst_in=d["cst"])
        fl.ops.gdn_tree_commit(d["x"], d["S"], d["a"], d["b"], d["A_log"], d["dt_bias"], path, S_out, pos0s=[4, 0],
                               conv_w=d["conv_w"], cst_in=d["cst"], cst_out=outs)
    calls(y, S_out, outs)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        calls(y, S_out, outs)
    for step in range(3):
        parents.copy_(torch.tensor([tree(g, 10 * step + 9, T), tree(g, T - step, T, "chain")], dtype=I32))
        path.copy_(torch.tensor([[step, step + 1, step + 7], [0, 5 - 3 * step, 9]], dtype=I32))
        d["x"].mul_(-1)
        graph.replay()
        y2, S2, o2 = torch.empty_like(y), [torch.empty_like(s) for s in S_out], [torch.empty_like(c) for c in outs]
        calls(y2, S2, o2)
        torch.cuda.synchronize()
        assert torch.equal(y, y2)
        assert all(torch.equal(a, b) for a, b in zip(S_out + outs, S2 + o2))
