"""Cache rows of the tree that are not finite: who is reached. An infinity or NaN in a K row reaches the
tokens that see it and no others; in a V row it may make others of its sequence NaN, never wrong; other
sequences keep their bits."""
import pytest
import torch

import paged_ref as ref
import paged_tight as tight
import tree_ref
from test_gpu_paged import SCALE, filled, gen, i32, randn
from test_gpu_tree_attention import seen_by
from test_gpu_tree_gdn import tree

pytestmark = pytest.mark.gpu

F16, I32 = torch.float16, torch.int32


@pytest.mark.parametrize("kv8", [False, True])
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("pool", ["k", "v"])
@pytest.mark.parametrize("ctxs,T,at", [([40, 70], 16, 7), ([5000, 900], 26, 3), ([20000, 64], 60, 31)], ids=str)
def test_who_a_row_that_is_not_finite_reaches(fl, dev, ctxs, T, at, pool, bad, kv8):
    g, P = gen(at), 16
    kp, vp, pages, _ = filled(fl, g, [c + T for c in ctxs], P, kv8)
    n_rows = kp.numel() // (4 * 272) if kv8 else kp.shape[0] * P
    parents = [tree(g, T, T) for _ in ctxs]
    q, nodes = randn(g, 2, T, 24, 512), torch.tensor(parents, dtype=I32).cuda()
    call = lambda: fl.ops.attn_tree_paged(q, kp, vp, pages, i32(*ctxs), nodes, page_size=P)
    want = call()
    rows = ref.rows_of(pages.cpu(), 0, P, torch.arange(ctxs[0] + T)).cuda()
    K, V = tight.kernel_values(kp, n_rows, 4, True)[rows], tight.kernel_values(vp, n_rows, 4, False)[rows]
    exact, bound = tight.attention(q[0, ..., :256], K, V, seen_by(parents[0], ctxs[0]), SCALE,
                                   tight.TWO_TERMS if kv8 else tight.ONE_TERM, q[0, ..., 256:])
    to, row = (kp if pool == "k" else vp), rows[ctxs[0] + at]
    if kv8:
        to[n_rows * 4 * 256:].view(F16).view(n_rows, 4, 8)[row, :, 3] = bad
    else:
        to.view(n_rows, 4, 256)[row, :, 100] = bad
    z = call()
    sees = torch.tensor([at in line for line in tree_ref.lines(parents[0])]).cuda()
    assert sees.any() and not sees.all()
    assert torch.equal(z[1], want[1])
    if pool == "k":
        assert torch.equal(z[0][~sees], want[0][~sees])
    else:
        right = (z[0].double() - exact).abs() <= bound
        assert (right | torch.isnan(z[0]))[~sees].all()
        dims = slice(96, 128) if kv8 else slice(100, 101)
        rest = [i for i in range(256) if not dims.start <= i < dims.stop]
        assert right[..., rest].all()       # (also of those that see it)
