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


def test_a_norm_or_workspace_inside_the_list(al):
    """Refused, with nothing written; right beside it they are taken."""
    import torch
    room = al.TensorList.WORKSPACE_BYTES // 4
    flat = torch.ones(5000 + 2 * room, device="cuda")
    ins = [flat[room:room + 2000], flat[room + 2001:room + 3000]]
    outs = [torch.ones(2001, device="cuda")[1:], torch.ones(999, device="cuda")]
    norm = torch.zeros(1, device="cuda")
    part = lambda t, at, n=1: t[at:at + n]  # noqa: E731
    here, there = al.TensorList(ins), al.TensorList(ins, outs)
    for lst, tensors in ((here, ins), (there, ins + outs)):
        for t in tensors:
            for at in (0, 1, t.numel() - 1):
                for call in (lambda: lst.global_norm(part(t, at)), lambda: lst.clip_global_norm(part(t, at), 1.0)):
                    with pytest.raises(al.AlError) as e:
                        call()
                    assert e.value.code == 5
    for at in (2, room + 1998, room + 2000, room + 2998):  # a workspace that begins, ends or lies in a tensor
        with pytest.raises(al.AlError) as e:
            here.global_norm(norm, workspace=part(flat, at, room))
        assert e.value.code == 5
    for t in outs:
        with pytest.raises(al.AlError) as e:
            there.clip_to_norm(part(t, 5), 1.0)
        assert e.value.code == 5
    with pytest.raises(al.AlError) as e:
        here.clip_to_norm(part(ins[1], 5), 1.0)
    assert e.value.code == 5
    torch.cuda.synchronize()
    assert bool((flat == 1).all()) and float(norm) == 0
    want = math.sqrt(2999)
    for space, at in ((part(flat, 0, room), room + 2000), (part(flat, room + 3000, room), room - 1)):
        flat.fill_(1)
        here.global_norm(part(flat, at), workspace=space)
        assert abs(float(flat[at]) - want) <= 1.5 * U32 * want
    there.clip_to_norm(part(ins[0], 5), 2.0)  # read by the call as well, and by nothing written
    torch.cuda.synchronize()
    assert bool((outs[0] == 1).all())
    here.destroy()
    there.destroy()


def test_types_that_the_library_does_not_know(al):
    import torch
    for dtype in (torch.float8_e4m3fn, torch.bool, torch.complex64, torch.float64, torch.uint8):
        for ins in ([torch.zeros(8, dtype=dtype, device="cuda")], [torch.zeros(8, device="cuda"), torch.zeros(0, dtype=dtype, device="cuda")]):
            with pytest.raises(al.AlError) as e:
                al.TensorList(ins)
            assert e.value.code == 3


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("lead,out_lead", [(0, 1), (1, 0), (1, 2), (3, 5), (2, 33), (31, 16)])
@pytest.mark.parametrize("count", [1, 30, 40_000, 36_000_001])
def test_outputs_that_lie_otherwise_than_their_inputs(al, dtype, lead, out_lead, count):
    """16-bit outputs may be apart from their inputs by no whole number of dwords, and any by no whole 64 bytes; the largest
    list is long enough to be clipped by the KiB."""
    import torch
    dt = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}[dtype]
    flat = torch.randn(lead + count, device="cuda", generator=torch.Generator(device="cuda").manual_seed(count)).to(dt)
    room = torch.full((out_lead + count + 40,), 7.0, dtype=dt, device="cuda")
    lst = al.TensorList([flat[lead:]], [room[out_lead:out_lead + count]])
    norm = torch.empty(1, device="cuda")
    want = float(flat[lead:].double().square().sum().sqrt())
    for both in (True, False):
        room.fill_(7)
        if both:
            lst.clip_global_norm(norm, want / 3, eps=0.0)
        else:
            lst.global_norm(norm)
            lst.clip_to_norm(norm, want / 3, eps=0.0)
        torch.cuda.synchronize()
        assert abs(float(norm) - want) <= 1.5 * U32 * want
        y = flat[lead:].double() / 3
        # max_norm as fp32, the norm, their quotient and the product in fp32; half a step of the output, or of its least number
        info = torch.finfo(dt)
        off = (room[out_lead:out_lead + count].double() - y).abs()
        assert bool((off <= (info.eps / 2 + 6 * U32) * y.abs() + info.tiny * info.eps / 2).all())
        assert bool((room[:out_lead] == 7).all()) and bool((room[out_lead + count:] == 7).all())
    lst.destroy()
