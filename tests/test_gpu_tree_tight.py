"""The GDN layer over trees on inputs whose outputs are far smaller than their terms (tree_tight.py): there
the bound of tree_ref.py holds every operand to its documented bits (tests/test_tree_tight.py)."""
import pytest
import torch

import tree_ref as ref
import tree_tight as tight
from test_gpu_tree_gdn import check, gen, run, tree

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("near", [False, True])
@pytest.mark.parametrize("B,T,n_k,n_v,kind", [(1, 1, 8, 8, "star"), (1, 16, 8, 24, "star"), (1, 30, 16, 48, "any"), (6, 16, 16, 48, "chain"),
                                              (9, 20, 16, 32, "binary"), (1, 60, 8, 8, "star")])
def test_states_that_the_tokens_do_not_see(fl, B, T, n_k, n_v, kind, near):
    g = gen(T)
    d = tight.unseen_states(g, B, T, n_k, n_v, near, "cuda")
    parents = [tree(g, T, T, kind) for _ in range(B)]
    want, bound = ref.gdn_tree(d, parents, [False] * B)
    check(run(fl, d, parents, [5] * B), want, bound, f"B {B} T {T} {kind}")


@pytest.mark.parametrize("B,T,n_k,n_v", [(1, 2, 8, 8), (1, 16, 8, 24), (1, 33, 16, 16), (6, 16, 16, 48), (9, 40, 16, 32),
                                         (1, 64, 16, 16)])
def test_paths_whose_terms_cancel(fl, B, T, n_k, n_v):
    d, parents = tight.cancelling_paths(gen(T), B, T, n_k, n_v, "cuda")
    want, bound = ref.gdn_tree(d, parents, [False] * B)
    check(run(fl, d, parents, [5] * B), want, bound, f"B {B} T {T}")


@pytest.mark.parametrize("B,T", [(1, 6), (1, 40), (6, 18)])
def test_beside_a_large_token(fl, B, T):
    g = gen(T)
    d = tight.unseen_states(g, B, T, 16, 48, False, "cuda")
    parents = [[p if p != T - 2 else T - 3 for p in tree(g, T, T)] for _ in range(B)]
    for s in d["S"]:
        s *= 2.0 ** -6
    d["x"][:, T - 2, 2 * 16 * 128:] = 6e4
    want, bound = ref.gdn_tree(d, parents, [False] * B)
    check(run(fl, d, parents, [5] * B), want, bound, f"B {B} T {T}")
