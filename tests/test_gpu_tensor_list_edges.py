"""Uses of a tensor list that depend on whose memory is whose: workspaces, streams, alignments, launches."""
import math

import pytest

pytestmark = pytest.mark.gpu

U32 = 2.0 ** -24


def test_the_workspace_is_the_lists_own(al):
    """It is not memory that the caching allocator would hand on in the order of the stream it came from."""
    import torch
    t = torch.ones(1000, device="cuda")
    before = torch.cuda.memory_allocated()
    lst = al.TensorList([t])
    assert torch.cuda.memory_allocated() == before
    lst.destroy()


def test_a_list_dropped_while_a_call_runs(al):
    """The object goes while a call on another stream is under way, and its own stream fills new memory at once."""
    import gc
    import torch
    side = torch.cuda.Stream()
    a = torch.randn(4096, 4096, device="cuda")
    t = torch.full((3_000_000,), 0.5, device="cuda")
    norm = torch.zeros(1, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(30):
            a = a @ a * 1e-3
    lst = al.TensorList([t])
    handle = lst._h
    lst.clip_global_norm(norm, 1.0, eps=0.0, stream=side)
    del lst
    gc.collect()
    junk = [torch.full((al.TensorList.WORKSPACE_BYTES // 8,), float("nan"), dtype=torch.float64, device="cuda") for _ in range(8)]
    torch.cuda.synchronize()
    want = 0.5 * math.sqrt(t.numel())
    assert abs(float(norm) - want) <= 1.5 * U32 * want
    # the factor: its quotient; the product
    assert bool(((t - 0.5 / want).abs() <= 4 * U32 * 0.5 / want).all()) and len(junk) == 8
    assert al.load().alamd_tensor_list_destroy(handle) == 0
