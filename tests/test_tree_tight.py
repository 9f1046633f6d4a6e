"""What the bound of the GDN layer over trees (tree_ref.py) rejects on the inputs of tree_tight.py, on the
CPU: any operand of the kernel in fewer bits than it is documented with, or in a scale that tokens share."""
import pytest
import torch

import tree_ref as ref
import tree_tight as tight


def gen(seed):
    return torch.Generator().manual_seed(seed)


def exceeds(d, parents, **form):
    want, bound = ref.gdn_tree(d, parents, [False] * len(parents))
    return ((tight.kernel_form(d, parents, **form) - want).abs() / bound.clamp_min(1e-300)).max().item()


@pytest.mark.parametrize("T,kind", [(1, "star"), (5, "chain"), (16, "star")])
def test_states_keys_and_queries_in_one_term_are_rejected(T, kind):
    parents = [list(range(-1, T - 1)) if kind == "chain" else [-1] * T]
    d = tight.unseen_states(gen(T), 1, T, 8, 8, False)
    assert exceeds(d, parents) < 0.9
    assert exceeds(d, parents, S=1) > 1.2 and exceeds(d, parents, q=1) > 1.2
    d = tight.unseen_states(gen(T), 1, T, 8, 8, True)
    assert exceeds(d, parents) < 0.9 and exceeds(d, parents, k=1) > 1.2


def test_a_system_in_half_precision_is_rejected():
    d, parents = tight.cancelling_paths(gen(16), 1, 16, 8, 8)
    assert exceeds(d, parents) < 0.9
    for name in "uAP":
        assert exceeds(d, parents, system=name) > 1.2, name


@pytest.mark.parametrize("large", [1e4, 6e4])
def test_a_scale_that_tokens_share_is_rejected(large):
    d = tight.unseen_states(gen(3), 1, 6, 4, 4, False)
    d["S"][0] *= 2.0 ** -6
    d["x"][0, 5, 2 * 4 * 128:] = large
    parents = [[-1, 0, 1, 0, -1, 1]]
    assert exceeds(d, parents) < 0.9 and exceeds(d, parents, shared=True) > 1.2
