"""The paged operators where inputs and callers are unlike the ordinary: host threads beside a
call, gates and rows that are not numbers, contexts whose weights lie far below the largest."""
import ctypes

import pytest
import torch

import paged_ref as ref

pytestmark = pytest.mark.gpu

F16, F32, I32 = torch.float16, torch.float32, torch.int32
SCALE = 256 ** -0.5


def gen(seed):
    return torch.Generator().manual_seed(seed)


def randn(g, *shape, scale=1.0):
    return (torch.randn(shape, generator=g) * scale).to(F16).cuda()


def i32(*v):
    return torch.tensor(v, dtype=I32, device="cuda")


def test_the_plan_of_chunks_is_made_with_other_threads_running(fl, dev):
    """The binding asks for the work bytes, which makes the plan, and launches with the
    interpreter released. In place of the library stand the interpreter's own "do I hold it"
    (1 or 0, here the work bytes) and a callback that notes the bytes it is given."""
    L, lane = fl._lib.lib(), fl._lib.lane
    assert lane is not None, "fl355_paged.so is not built"
    real = [ctypes.cast(getattr(L, name), ctypes.c_void_p).value for name in fl._lib.BOUND]
    seen = []
    name = "fl_attention_prefill_paged"
    res, args = fl._lib.SIGNATURES[name]
    noted = ctypes.CFUNCTYPE(res, *args)(lambda *a: seen.append(a[-2]) or 0)
    held = ctypes.cast(ctypes.pythonapi.PyGILState_Check, ctypes.c_void_p).value
    fake = dict(zip(fl._lib.BOUND, real))
    fake[name] = ctypes.cast(noted, ctypes.c_void_p).value
    fake["fl_attention_prefill_paged_work_bytes"] = held
    q = torch.zeros((3, 24, 512), dtype=F16, device="cuda")
    kp = fl.ops.paged_pool(2, 16)
    try:
        lane.bind(*fake.values())
        fl.ops.attention_prefill_paged(q, kp, kp, i32(0, 1).view(1, 2), [3], [0], page_size=16)
    finally:
        lane.bind(*real)
    assert seen == [0]
