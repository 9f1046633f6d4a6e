"""Outputs of the tree operators in rows between an input's: columns of one buffer."""
import pytest
import torch

import tree_ref
from test_gpu_paged import filled, gen as randn_gen, randn
from test_gpu_tree_gdn import gen, i32, run, tree

pytestmark = pytest.mark.gpu

F16 = torch.float16


@pytest.mark.parametrize("first", ["z", "y"])
@pytest.mark.parametrize("B,T", [(1, 5), (6, 20)])
def test_y_of_the_gdn_layer_beside_z(fl, B, T, first):
    g = gen(T)
    d = tree_ref.gdn_layer(g, B, T)
    parents = [tree(g, T, T) for _ in range(B)]
    want = run(fl, d, parents, [4] * B)
    both = torch.full((B, T, 2, 6144), 7.0, dtype=F16, device="cuda")
    z, y = (both[:, :, i] for i in ((0, 1) if first == "z" else (1, 0)))
    z.copy_(d["z"])
    nodes, lib = i32(parents), fl._lib
    rc = lib.lib().fl_gdn_tree_normed(
        d["x"].data_ptr(), 10240, d["conv_w"].data_ptr(), lib.ptr_array([c.data_ptr() for c in d["cst"]]),
        lib.int_array([4] * B), nodes.data_ptr(), d["a"].data_ptr(), d["b"].data_ptr(), 48, d["A_log"].data_ptr(),
        d["dt_bias"].data_ptr(), lib.ptr_array([s.data_ptr() for s in d["S"]]), z.data_ptr(), 12288,
        d["norm_w"].data_ptr(), y.data_ptr(), 12288, B, T, 16, 48, 128, 128, 128 ** -0.5, 1e-6, 1e-6,
        torch.cuda.current_stream().cuda_stream)
    assert rc == 0, lib.lib().fl_last_error()
    assert torch.equal(y, want) and torch.equal(z, d["z"])


@pytest.mark.parametrize("kv8", [False, True])
def test_z_of_the_attention_in_place_of_a_gate_that_is_not_used(fl, dev, kv8):
    g, T, ctxs = randn_gen(3), 9, [70, 900]
    kp, vp, pages, _ = filled(fl, g, [c + T for c in ctxs], 16, kv8)
    qg, at, pos0 = randn(g, 2, T, 24, 512), i32([tree(g, T, T)] * 2), i32(ctxs)
    want = fl.ops.attn_tree_paged(qg, kp, vp, pages, pos0, at, page_size=16, gate=False)
    before, work = qg.clone(), torch.empty(fl.ops.attn_tree_paged_work_bytes(2, T), dtype=torch.uint8, device="cuda")
    n_pages = kp.numel() // (16 * 4 * 272) if kv8 else kp.shape[0]
    rc = fl._lib.lib().fl_attn_tree_paged(
        qg.data_ptr(), 512, kp.data_ptr(), vp.data_ptr(), int(kv8), n_pages, 16, pages.data_ptr(), pages.shape[1],
        pages.shape[1], pos0.data_ptr(), at.data_ptr(), 2, T, 24, 4, 256, 256 ** -0.5, 0, 0, 0, qg.data_ptr() + 512, 512,
        work.data_ptr(), work.numel(), torch.cuda.current_stream().cuda_stream)
    assert rc == 0, fl._lib.lib().fl_last_error()
    assert torch.equal(qg[..., 256:], want) and torch.equal(qg[..., :256], before[..., :256])
