"""The GDN layer over trees whose tokens are of very unlike sizes: what a token gets is as good as its
own path's terms allow (tree_ref.py's bound has no others), whatever its siblings, descendants
and the tokens behind it hold, and an infinity or NaN of one never becomes another's wrong number."""
import pytest
import torch

import tree_ref as ref
from test_gpu_tree_gdn import check, gen, run, tree

pytestmark = pytest.mark.gpu

F16 = torch.float16


def layer(g, B, T):
    """Random inputs, and trees in which every token from 1 on that is a multiple of 5 is a leaf."""
    d = ref.gdn_layer(g, B, T)
    parents = [tree(g, T, T) for _ in range(B)]
    for p in parents:
        for i in range(T):
            while p[i] > 0 and p[i] % 5 == 0:
                p[i] -= 1
    return d, parents


@pytest.mark.parametrize("large", [1e3, 1e4, 6e4])
@pytest.mark.parametrize("B,T,at", [(1, 7, 5), (1, 16, 10), (1, 40, 20), (1, 64, 0), (6, 16, 5), (6, 40, 35), (7, 33, 0)])
def test_a_large_token_leaves_the_others_their_precision(fl, B, T, at, large):
    """v of one leaf, or of every path's first token (at 0), up to `large`; the states are small."""
    g = gen(T + at)
    d, parents = layer(g, B, T)
    if at == 0:
        parents = [[-1] + [max(0, q) for q in p[1:]] for p in parents]
    d["x"][:, at, 2 * 16 * 128:] = large
    want, bound = ref.gdn_tree(d, parents, [False] * B)
    check(run(fl, d, parents, [7] * B), want, bound, f"B {B} T {T}, token {at} of {large}")


@pytest.mark.parametrize("B,T", [(1, 16), (1, 37), (6, 40)])
def test_large_values_and_small_states(fl, B, T):
    """The other way round: rows of S0 far below the tokens' v, which the tokens without a v see alone."""
    g = gen(T)
    d, parents = layer(g, B, T)
    for s in d["S"]:
        s *= 2.0 ** -14
    d["x"][:, 1::2, 2 * 16 * 128:] *= 2.0 ** 10
    d["b"][:, ::2] = -60.0
    want, bound = ref.gdn_tree(d, parents, [False] * B)
    check(run(fl, d, parents, [7] * B), want, bound, f"B {B} T {T}")


@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("B,T,at", [(1, 9, 5), (1, 40, 20), (6, 40, 20), (6, 16, 15), (1, 64, 60)])
def test_what_is_not_finite_never_becomes_a_wrong_number(fl, B, T, at, bad):
    """Tokens that do not descend from it have what they should, or NaN, and those of the 16 ahead of its
    own 16 and of the other sequences have what they should."""
    g = gen(at)
    d, parents = layer(g, B, T)
    parents[0] = [p if p != at else at - 1 for p in parents[0]]
    d["x"][0, at, 2 * 16 * 128:] = bad
    want, bound = ref.gdn_tree(d, parents, [False] * B)
    y = run(fl, d, parents, [7] * B).double()
    assert not torch.isfinite(y[0, at]).any()
    right = (y - want).abs() <= bound
    right[0, at] = True
    assert (right | torch.isnan(y)).all()
    assert right[1:].all() and right[0, :at // 16 * 16].all()
