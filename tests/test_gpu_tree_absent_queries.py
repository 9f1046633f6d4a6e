"""Attention of trees in which places without a token lie between the tokens, in the same waves: whatever
their queries and gates hold, they give 0 and change nothing."""
import pytest
import torch

import paged_ref as ref
import paged_tight as tight
import tree_ref
from test_gpu_paged import SCALE, filled, gen, i32, randn
from test_gpu_tree_attention import check, seen_by

pytestmark = pytest.mark.gpu

I32 = torch.int32
INF, NAN = float("inf"), float("nan")


@pytest.mark.parametrize("kv8", [False, True])
@pytest.mark.parametrize("ctxs,T", [([5000], 16), ([40, 9000, 700], 7), ([20000, 300], 33), ([60], 64), ([0, 3], 5)],
                         ids=str)
@pytest.mark.parametrize("held", [(INF,), (-INF,), (INF, -INF), (NAN,), (6e4,)], ids=str)
def test_queries_of_absent_places(fl, dev, ctxs, T, kv8, held):
    g, B = gen(T + len(held)), len(ctxs)
    kp, vp, pages, _ = filled(fl, g, [c + T for c in ctxs], 32, kv8)
    n_rows = kp.numel() // (4 * 272) if kv8 else kp.shape[0] * 32
    parents = []
    for b in range(B):      # every third token is none; the others go on from the one before
        here = [i for i in range(T) if (i + b) % 3 != 1]
        parents.append([-2] * T)
        for n, i in enumerate(here):
            parents[b][i] = here[n - 1] if n % 4 else -1
    at, pos0 = torch.tensor(parents, dtype=I32).cuda(), i32(*ctxs)
    q = randn(g, B, T, 24, 512)
    call = lambda: fl.ops.attn_tree_paged(q, kp, vp, pages, pos0, at, page_size=32)
    want = call()
    for b in range(B):
        for i in range(T):
            if parents[b][i] == -2:
                for n, x in enumerate(held):
                    q[b, i, :, (37 * i + 5 * n) % 256] = x
                    q[b, i, :, 256 + n] = x
    z = call()
    K, V = tight.kernel_values(kp, n_rows, 4, True), tight.kernel_values(vp, n_rows, 4, False)
    for b in range(B):
        here = torch.tensor([p != -2 for p in parents[b]]).cuda()
        assert not z[b][~here].any(), f"sequence {b}"
        assert torch.equal(z[b], want[b])
        rows = ref.rows_of(pages.cpu(), b, 32, torch.arange(ctxs[b] + T)).cuda()
        exact, bound = tight.attention(q[b][here][..., :256], K[rows], V[rows], seen_by(parents[b], ctxs[b])[here], SCALE,
                                       tight.TWO_TERMS if kv8 else tight.ONE_TERM, q[b][here][..., 256:])
        check(z[b][here], exact, bound, f"sequence {b}")
