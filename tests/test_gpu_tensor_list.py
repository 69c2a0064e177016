"""The norm over a list of buffers and the clipping by it on the GPU, against the formulas in 64 bits, and a training
step's operators in a row."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U32 = 2.0 ** -24
CHUNK = 65536  # bytes, where a long tensor is cut


def _tensors(spec, seed=0, scale=1.0, lead=0):
    """(count, dtype) pairs as neighbours in one allocation of each type, `lead` elements from its start."""
    import torch
    gen = torch.Generator(device="cuda").manual_seed(seed)
    types = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
    room = {d: lead for d in types}
    places = []
    for n, d in spec:
        places.append((d, room[d], n))
        room[d] += n
    flats = {d: (torch.randn(room[d] + 1, device="cuda", generator=gen) * scale).to(types[d]) for d in types}
    return [flats[d][at:at + n] for d, at, n in places], flats


def _norm(tensors):
    return math.sqrt(sum(float(np.square(t.double().cpu().numpy()).sum()) for t in tensors))


def _call(al, tensors, **kw):
    import torch
    norm = torch.full((3,), 77.0, device="cuda")
    lst = al.TensorList(tensors, **kw)
    lst.global_norm(norm[1:2])
    torch.cuda.synchronize()
    assert norm[0] == 77 and norm[2] == 77
    return lst, norm[1:2]


SPECS = [
    [],
    [(0, "f32")],
    [(1, "f32")],
    [(1, "bf16"), (0, "f16"), (3, "f16"), (1, "f32")],
    [(CHUNK // 4 + k, "f32") for k in (-1, 0, 1)],
    [(CHUNK // 2 + k, "bf16") for k in (-1, 0, 1)] + [(2 * CHUNK // 2 + 7, "f16")],
    [(k, "f32") for k in range(1, 40)] + [(k, "bf16") for k in range(1, 40)],
    [(5000 + 13 * k, ("f32", "bf16", "f16")[k % 3]) for k in range(300)],
    [(30_000_001, "f32"), (50_000_003, "bf16"), (17, "f16")],  # more chunks than workgroups
]


@pytest.mark.parametrize("lead", [0, 1, 3])
@pytest.mark.parametrize("spec", range(len(SPECS)))
def test_norm_and_clipping(al, spec, lead):
    import torch
    tensors, flats = _tensors(SPECS[spec], seed=spec, scale=0.1, lead=lead)
    want = _norm(tensors)
    outs, out_flats = _tensors(SPECS[spec], seed=50, lead=lead)
    before = {d: t.clone() for d, t in out_flats.items()}
    lst, norm = _call(al, tensors, outs=outs)
    # squares and sums are made in 64 bits: one rounding, and far less than half of another
    assert abs(float(norm) - want) <= 1.5 * U32 * want
    for max_norm in (want * 2 + 1, want / 3, 0.0):
        both = torch.empty(1, device="cuda")
        lst.clip_global_norm(both, max_norm, eps=1e-6)
        torch.cuda.synchronize()
        assert torch.equal(both, norm)
        n = float(norm) + 1e-6
        factor = 1.0 if n <= max_norm else max_norm / n
        for a, b in zip(tensors, outs):
            w = a.double().cpu().numpy() * factor
            half, least = torch.finfo(a.dtype).eps / 2, torch.finfo(a.dtype).tiny * torch.finfo(a.dtype).eps / 2
            # the factor: its sum, its quotient and max_norm in fp32; the product
            assert np.all(np.abs(b.double().cpu().numpy() - w) <= (half * (1 + 8 * U32) + 4 * U32) * np.abs(w) + least)
            if factor == 1.0:
                assert torch.equal(a, b)
    # nothing but the outputs was written
    for d, at in {d: lead for d in flats}.items():
        used = sum(n for n, dd in SPECS[spec] if dd == d)
        assert torch.equal(out_flats[d][:at], before[d][:at]) and torch.equal(out_flats[d][at + used:], before[d][at + used:])
    lst.destroy()


@pytest.mark.parametrize("value", [1e30, 1e-30, 3e38, 1e-42])
def test_squares_beyond_fp32(al, value):
    import torch
    for dtype in (torch.float32, torch.bfloat16):
        t = torch.full((70_001,), value, device="cuda").to(dtype)
        _, norm = _call(al, [t])
        want = float(t[0].double()) * math.sqrt(70_001)
        if want > 3.4e38:
            assert math.isinf(float(norm))
        else:
            # half a step of a small result is half of the smallest number
            assert abs(float(norm) - want) <= 1.5 * U32 * want + 2.0 ** -150
    t = torch.full((70_001,), 65504.0, device="cuda").half()
    _, norm = _call(al, [t])
    assert abs(float(norm) - 65504 * math.sqrt(70_001)) <= 1.5 * U32 * 65504 * math.sqrt(70_001)


def test_numbers_of_every_size_together(al):
    """Ones next to numbers whose squares an fp32 sum of them would lose."""
    import torch
    n = 1 << 24
    t = torch.full((n,), 1e-4, device="cuda")
    t[0] = 1.0
    _, norm = _call(al, [t])
    want = math.sqrt(1 + (n - 1) * float(t[1].double()) ** 2)
    assert abs(float(norm) - want) <= 1.5 * U32 * want


def test_not_a_number_and_infinity(al):
    import torch
    for bad in (float("nan"), float("inf"), float("-inf")):
        t = [torch.ones(100_000, device="cuda"), torch.ones(37, device="cuda").bfloat16()]
        t[0][77_777] = bad
        lst, norm = _call(al, t)
        assert math.isnan(float(norm)) if math.isnan(bad) else float(norm) == math.inf
        lst.clip_to_norm(norm, 1.0)
        torch.cuda.synchronize()
        if math.isnan(bad):
            assert all(bool(torch.isnan(v).all()) for v in t)
        else:
            assert bool(torch.isnan(t[0][77_777])) and bool((t[1] == 0).all()) and int((t[0] == 0).sum()) == 99_999


def test_in_place_and_left_alone(al):
    """In place the buffers change by the factor, or, where it is 1, not in a bit: a NaN with a payload of its own stays."""
    import torch
    tensors, _ = _tensors([(1000, "f32"), (40_000, "bf16"), (9, "f16")], seed=4)
    whole = [t.clone() for t in tensors]
    lst, norm = _call(al, tensors)
    lst.clip_to_norm(norm, float(norm) * 2)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(tensors, whole))
    apart = [torch.empty_like(t) for t in tensors]
    other, _ = _call(al, whole, outs=apart)
    other.clip_to_norm(norm, 0.5)
    lst.clip_to_norm(norm, 0.5)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(tensors, apart))
    odd = torch.zeros(20_000, dtype=torch.int32, device="cuda")
    odd[5] = 0x7f800001
    lst, norm = _call(al, [odd.view(torch.float32)])
    norm.fill_(0.25)
    lst.clip_to_norm(norm, 1.0)
    torch.cuda.synchronize()
    assert int(odd[5]) == 0x7f800001


def test_clipping_by_nothing_at_all(al):
    """0 / 0 does not come up: gradients of zero under a largest norm of zero stay zero."""
    import torch
    t = [torch.zeros(5000, device="cuda")]
    lst, norm = _call(al, t)
    lst.clip_global_norm(norm, 0.0, eps=0.0)
    torch.cuda.synchronize()
    assert float(norm) == 0 and bool((t[0] == 0).all())


def test_the_same_bits_every_time(al):
    import torch
    tensors, _ = _tensors([(3_000_001, "f32"), (5_000_000, "bf16")], seed=8)
    lst, norm = _call(al, tensors)
    again = torch.empty(20, device="cuda")
    for k in range(20):
        lst.global_norm(again[k:k + 1])
    torch.cuda.synchronize()
    assert bool((again == norm).all())


def test_a_tensor_beyond_4_gib(al):
    import torch
    n = (1 << 31) + 100_003  # 8 GB and a bit
    t = torch.empty(n, device="cuda")
    t.fill_(0.5)
    t[-1] = 70_000.0
    lst, norm = _call(al, [t])
    want = math.sqrt(0.25 * (n - 1) + 70_000.0 ** 2)
    assert abs(float(norm) - want) <= 1.5 * U32 * want
    lst.clip_to_norm(norm, float(norm) / 2, eps=0.0)
    torch.cuda.synchronize()
    assert float(t[-1]) == 35_000.0 and float(t[0]) == 0.25 and float(t[n // 2]) == 0.25
    assert bool((t[-100_000:-1] == 0.25).all())


def test_more_chunks_than_one_launch_takes(al):
    """17 GB in three tensors, of which the first and the last end inside a chunk."""
    import torch
    per = CHUNK // 4
    sizes = [per * 1000 + 5, per * ((1 << 18) + 2) - 7, 3 * per + 1]
    flat = torch.empty(sum(sizes), device="cuda").fill_(0.5)
    tensors = list(flat.split(sizes))
    lst, norm = _call(al, tensors)
    want = 0.5 * math.sqrt(flat.numel())
    assert abs(float(norm) - want) <= 1.5 * U32 * want
    norm.fill_(4.0)
    lst.clip_to_norm(norm, 1.0, eps=0.0)
    torch.cuda.synchronize()
    for t in tensors:
        assert bool((t == 0.125).all())
    lst.clip_global_norm(norm, float(norm) + 1e9)  # nothing to clip, and the norm is made anew
    torch.cuda.synchronize()
    assert abs(float(norm) - want / 4) <= 1.5 * U32 * want / 4 and bool((tensors[2] == 0.125).all())


def test_many_small_tensors(al):
    """100 MB in tensors of a few KiB: long enough for the clipping by KiB, but of small chunks."""
    import torch
    sizes = [2000 + k % 977 for k in range(10_500)]
    flat = torch.randn(sum(sizes), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    out = torch.empty_like(flat)
    lst = al.TensorList(list(flat.split(sizes)), list(out.split(sizes)))
    norm = torch.empty(1, device="cuda")
    lst.clip_global_norm(norm, 1.0, eps=0.0)
    torch.cuda.synchronize()
    want = float(flat.double().square().sum().sqrt())
    assert abs(float(norm) - want) <= 1.5 * U32 * want
    w = flat.double() / want
    assert bool(((out.double() - w).abs() <= 5 * U32 * w.abs() + 2.0 ** -150).all())


def test_captured_and_on_another_stream(al):
    """Two lists captured into graphs of their own with a workspace each, replayed with new values and eager work in
    between."""
    import torch
    sets = []
    for k in range(2):
        tensors, _ = _tensors([(70_000 + k, "f32"), (33, "bf16"), (200_000, "f16")], seed=k)
        outs = [torch.empty_like(t) for t in tensors]
        norm = torch.empty(1, device="cuda")
        lst = al.TensorList(tensors, outs)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            lst.clip_global_norm(norm, 3.0)
        sets.append((tensors, outs, norm, lst, graph))
    side = [torch.cuda.Stream() for _ in range(2)]
    for rep in range(3):
        want = []
        for tensors, outs, norm, lst, _ in sets:
            for t in tensors:
                t.normal_().mul_(rep + 0.01)
            lst.clip_global_norm(norm, 3.0)
            torch.cuda.synchronize()
            want.append([v.clone() for v in outs + [norm]])
            for v in outs + [norm]:
                v.zero_()
        torch.cuda.synchronize()
        for k, (_, _, _, _, graph) in enumerate(sets):
            with torch.cuda.stream(side[k]):
                graph.replay()
        torch.cuda.synchronize()
        for w, (_, outs, norm, lst, _) in zip(want, sets):
            assert all(torch.equal(a, b) for a, b in zip(w, outs + [norm]))
            for v in outs + [norm]:
                v.zero_()
        torch.cuda.synchronize()
        for k, (_, _, norm, lst, _) in enumerate(sets):
            lst.clip_global_norm(norm, 3.0, stream=side[k])
        torch.cuda.synchronize()
        for w, (_, outs, norm, lst, _) in zip(want, sets):
            assert all(torch.equal(a, b) for a, b in zip(w, outs + [norm]))


def test_refusals(al):
    import torch
    t = [torch.ones(100, device="cuda"), torch.ones(100, device="cuda").half()]
    lst = al.TensorList(t)
    norm = torch.zeros(1, device="cuda")
    space = torch.zeros(al.TensorList.WORKSPACE_BYTES + 64, dtype=torch.uint8, device="cuda")
    for code, call in [
            (1, lambda: lst.global_norm(torch.zeros(2, device="cuda"))), (1, lambda: lst.global_norm(norm.double())),
            (1, lambda: lst.global_norm(norm.cpu())), (1, lambda: lst.global_norm(norm, workspace=space[:100])),
            (1, lambda: lst.global_norm(norm, workspace=space[4:])),
            (5, lambda: lst.global_norm(space.view(torch.float32)[4:5], workspace=space)),
            (5, lambda: lst.clip_global_norm(space.view(torch.float32)[-17:-16], 1.0, workspace=space)),
            (1, lambda: lst.clip_to_norm(norm, -1.0)), (1, lambda: lst.clip_to_norm(norm, float("nan"))),
            (1, lambda: lst.clip_global_norm(norm, 1.0, eps=-1e-6)), (1, lambda: lst.clip_global_norm(norm, 1.0, eps=float("nan"))),
            (5, lambda: al.TensorList([t[0], t[0]])), (5, lambda: al.TensorList([t[0], t[0][50:]])),
            (5, lambda: al.TensorList([t[0][:50]], [t[0][20:70]])),
            (1, lambda: al.TensorList(t, t[:1])), (1, lambda: al.TensorList(t, [t[1], t[0]])),
            (1, lambda: al.TensorList([torch.ones(8, 8, device="cuda").t()[1:]])),
            (3, lambda: al.TensorList([torch.ones(8, device="cuda", dtype=torch.int32)])),
            (3, lambda: al.TensorList([torch.ones(8, device="cuda", dtype=torch.float64)]))]:
        with pytest.raises(al.AlError) as e:
            call()
        assert e.value.code == code, e.value
    lst.destroy()
    lst.destroy()
    with pytest.raises(al.AlError):
        lst.global_norm(norm)
    torch.cuda.synchronize()
    assert all(bool((v == 1).all()) for v in t)


def test_a_training_step(al):
    """Two data-parallel ranks, each with a layer split over three: the norm over the three partial sums, its backward
    pass, the average of the two ranks' gradients, their norm and the clipping; against differentiation of the same
    step in 64 bits."""
    import torch
    rows, cols, split, data, eps, max_norm = 40, 258, 3, 2, 1e-5, 0.7
    gen = torch.Generator().manual_seed(3)
    rnd = lambda *s: torch.randn(*s, generator=gen).double()  # noqa: E731
    weight = rnd(cols)
    parts = [[rnd(rows, cols) for _ in range(split)] for _ in range(data)]
    res = [rnd(rows, cols) for _ in range(data)]
    t = [rnd(rows, cols) for _ in range(data)]
    # 64 bits
    w64 = weight.clone().requires_grad_()
    bias = torch.zeros(cols, dtype=torch.float64, requires_grad=True)  # added to the residual stream
    loss = 0
    for r in range(data):
        s = sum(parts[r]) + res[r] + bias
        y = s * (s.square().mean(1, keepdim=True) + eps).rsqrt() * w64
        loss = loss + (y * t[r] + 0.1 * s.square()).sum() / data
    loss.backward()
    total = math.sqrt(float(w64.grad.square().sum() + bias.grad.square().sum()))
    factor = min(1.0, max_norm / (total + 1e-6))
    # the framework's calls
    g = lambda v: v.float().cuda()  # noqa: E731
    dws, dbs = [], []
    for r in range(data):
        ins, out, s, dx = [g(p) for p in parts[r]], *(torch.empty(rows, cols, device="cuda") for _ in range(3))
        rstd, dw, w = torch.empty(rows, device="cuda"), torch.empty(cols, device="cuda"), g(weight)
        al.rms_norm(out, ins, weight=w, residual=g(res[r]), sum_out=s, rstd=rstd, eps=eps)
        ws = torch.empty(al.rms_norm_grad_workspace(rows, cols), dtype=torch.uint8, device="cuda")
        al.rms_norm_grad(dx, [g(t[r])], s, rstd, weight=w, dsum=0.2 * s, dweight=dw, workspace=ws)
        dws.append(dw)
        dbs.append(dx.sum(0))
    al.combine([dws[0]], dws, "avg")
    al.combine([dbs[0]], dbs, "avg")
    norm = torch.empty(1, device="cuda")
    grads = al.TensorList([dws[0], dbs[0]])
    grads.clip_global_norm(norm, max_norm)
    torch.cuda.synchronize()
    # sums over a few hundred fp32 terms of order one: 1e-4 of the largest is far above their roundings
    assert abs(float(norm) / total - 1) < 1e-5
    for got, want in ((dws[0], w64.grad * factor), (dbs[0], bias.grad * factor)):
        assert float((got.double().cpu() - want).abs().max()) < 1e-4 * float(want.abs().max())
    grads.destroy()
