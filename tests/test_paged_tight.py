"""What the tight bounds of the paged attention (paged_tight.py) reject, on the CPU: the reference
with one tile of rows lost, twice in it or taken from elsewhere, K rounded to fp16, weights in
one fp16 term."""
import pytest
import torch

import paged_tight as tight

SCALE = 256 ** -0.5


def softmax_z(q, K, V):
    return torch.softmax(q.double() @ K.double().t() * SCALE, -1) @ V.double()


def exceeds(z, want, bound):
    return ((z - want).abs() / bound).max().item()


@pytest.mark.parametrize("L", [700, 9000, 100000])
@pytest.mark.parametrize("p_rel", [tight.ONE_TERM, tight.TWO_TERMS])
def test_a_tile_lost_repeated_or_swapped_is_rejected(L, p_rel):
    g = torch.Generator().manual_seed(L)
    k, v = tight.marked_rows(g, L, 1)
    q = torch.randn((1, 2, 256), generator=g).half()
    seen = torch.ones(1, L, dtype=torch.bool)
    want, bound = tight.attention(q, k, v, seen, SCALE, p_rel)
    K, V = k[:, 0], v[:, 0]
    assert exceeds(softmax_z(q[0], K, V), want[0], bound[0]) < 0.01
    for tile in (0, 9, L // 64, L // 32 - 1):
        rows = torch.arange(32 * tile, 32 * tile + 32)
        rest = torch.ones(L, dtype=torch.bool)
        rest[rows] = False
        assert exceeds(softmax_z(q[0], K[rest], V[rest]), want[0], bound[0]) > 2
        twice = torch.cat([torch.arange(L), rows])
        assert exceeds(softmax_z(q[0], K[twice], V[twice]), want[0], bound[0]) > 2
        other = torch.arange(L)
        other[rows] = (rows + 32 * 7) % L
        assert exceeds(softmax_z(q[0], K[other], V), want[0], bound[0]) > 2
        assert exceeds(softmax_z(q[0], K, V[other]), want[0], bound[0]) > 2


def test_k_rounded_to_fp16_is_rejected():
    L = 64
    kp, vp, q = tight.near_ties(L)
    K = tight.kernel_values(kp, L, 1, True)
    V = tight.kernel_values(vp, L, 1, False)
    seen = torch.ones(1, L, dtype=torch.bool)
    want, bound = tight.attention(q.view(1, 1, 256), K, V, seen, SCALE, tight.TWO_TERMS)
    s = (q.double() @ K[:2, 0].t() * SCALE)
    assert 95 < s.min() and s.max() < 105
    rounded = tight.kernel_values(kp, L, 1, False)
    assert exceeds(softmax_z(q.view(1, 256), rounded[:, 0], V[:, 0]), want[0], bound[0]) > 2


def test_weights_in_one_term_are_rejected_by_their_mean():
    """(That test's measure: the mean over the dims of (z - want) / want, whose part from z's own
    rounding is 2^-11 / sqrt(3 * 256) for errors spread over half a step, here 6 times that.)"""
    L = 64
    kp, vp, q, off = tight.one_term_shows(L)
    assert off > 0.8 * 2.0 ** -11
    K, V = (tight.kernel_values(p, L, 1, True)[:, 0] for p in (kp, vp))
    s = q.double() @ K.t() * SCALE
    p = torch.exp(s - s.max())
    want = (p @ V) / p.sum()
    mean = lambda z: ((z - want) / want).mean().abs().item()
    allowed = 6 * 2.0 ** -11 / (3 * 256) ** 0.5
    assert mean(want.half().double()) < allowed
    assert mean(((p.half().double() @ V) / p.sum()).half().double()) > 2 * allowed
