"""Values at which the root-mean-square norm and its backward pass round, overflow or share elements between lanes.

u = 2^-24 is half a step of fp32 relative to the value."""
import pytest

pytestmark = pytest.mark.gpu

U32 = 2.0 ** -24
TYPES = ("bf16", "f16", "f32")


def _type(name):
    import torch
    return {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}[name]


def _to_e4m3(q):
    """Numbers in 64 bits rounded to those of e4m3, ties to even, up to 448."""
    import torch
    step = torch.exp2(torch.floor(torch.log2(q.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(q / step) * step


@pytest.mark.parametrize("dtype,rows,cols", [("f16", 8191, 4099), ("bf16", 4000, 4096), ("bf16", 33, 515), ("f32", 4000, 4099), ("f16", 9000, 5),
                                             ("f32", 5000, 3)])
@pytest.mark.parametrize("group", [0, 32, 64, 128])
def test_8_bits_are_the_nearest(al, dtype, rows, cols, group):
    """One rank, 16-bit rows with a weight of their type or fp32 rows without: s * w is exact, and so is its largest
    magnitude in a group.  448 / max is rounded once and the product with s * w once, so what is rounded to 8 bits is off by
    two half steps and far less than a hundredth of another."""
    import torch
    gen = torch.Generator(device="cuda").manual_seed(cols)
    x = torch.randn(rows, cols, device="cuda", generator=gen).to(_type(dtype))
    w = None if dtype == "f32" else (1 + 0.2 * torch.randn(cols, device="cuda", generator=gen)).to(x.dtype)
    if rows > 8:
        x[7] = 0
    groups = -(-cols // group) if group else 1
    out = torch.empty(rows, cols, dtype=torch.float8_e4m3fn, device="cuda")
    scales = torch.empty(rows, groups, device="cuda")
    al.rms_norm(out, [x], weight=w, scales=scales, group=group)
    size = group or cols
    s = x.double() if w is None else x.double() * w.double()
    s = torch.nn.functional.pad(s, (0, groups * size - cols)).view(rows, groups, size)
    largest = s.abs().amax(2, keepdim=True)
    q = (448 * s / torch.where(largest > 0, largest, 1)).view(rows, -1)[:, :cols]
    low, high = _to_e4m3(q * (1 - 2.01 * U32)), _to_e4m3(q * (1 + 2.01 * U32))
    got = out.to(torch.float64)
    bad = (got < torch.minimum(low, high)) | (got > torch.maximum(low, high))
    assert int(bad.sum()) == 0, "%d of %d are not the nearest" % (int(bad.sum()), bad.numel())


@pytest.mark.parametrize("dtype,cols", [("f16", 5), ("f32", 3), ("f16", 520)])
def test_8_bits_of_a_row_depend_on_it_alone(al, dtype, cols):
    """Rows whose numbers are too small for the usual way to their quotients, among others."""
    import torch
    rows = 9_000_000 // cols
    gen = torch.Generator(device="cuda").manual_seed(cols)
    x = torch.randn(rows, cols, device="cuda", generator=gen).to(_type(dtype))
    w = (1 + 0.2 * torch.randn(cols, device="cuda", generator=gen)).to(x.dtype)
    got = []
    for small in (False, True):
        if small:
            x[::61] *= 1e-38
        out = torch.empty(rows, cols, dtype=torch.float8_e4m3fn, device="cuda")
        al.rms_norm(out, [x], weight=w, scales=torch.empty(rows, 1, device="cuda"))
        got.append(out.view(torch.uint8))
    got[0][::61] = got[1][::61]
    assert torch.equal(*got)


def _shared_columns(dtype, cols):
    """A column that the last vector, moved back to end with the row, has in common with the vector in front."""
    ve = 16 // _type(dtype).itemsize
    assert cols > ve and cols % ve
    return cols - ve, cols // ve * ve - 1


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols", [9, 77, 513, 1029, 2051, 9001, 20001])
@pytest.mark.parametrize("value", [float("inf"), float("-inf")])
def test_infinity_in_elements_that_two_lanes_hold(al, dtype, cols, value):
    """rstd is 0 next to an infinity wherever it is: zeros, and 0 * inf in its own place."""
    import torch
    dt = _type(dtype)
    for column in (0, *_shared_columns(dtype, cols), cols - 1):
        for rows in (3, 700):
            x = torch.ones(rows, cols, device="cuda").to(dt)
            x[1, column] = value
            out, rstd = torch.empty_like(x), torch.empty(rows, device="cuda")
            al.rms_norm(out, [x], rstd=rstd)
            torch.cuda.synchronize()
            assert float(rstd[1]) == 0 and float(rstd[0]) > 0.9 and float(rstd[2]) > 0.9
            assert bool(torch.isnan(out[1, column])) and int((out[1] == 0).sum()) == cols - 1
            # a row of ones: 1 / sqrt(1 + 1e-6); half of the roundings of 1 / n, the product with it and the sum with eps, two
            # of the root, one of the output
            for row in (0, 2):
                off = (out[row].double() - (1 + 1e-6) ** -0.5).abs()
                assert float(off.max()) <= 4 * U32 + torch.finfo(dt).eps / 2


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols", [9, 77, 513, 1029, 2051, 9001, 20001])
def test_backward_infinity_in_elements_that_two_lanes_hold(al, dtype, cols):
    """With an infinite gradient the row's product sum is infinite, and so is dx where x is not 0: -inf where n is positive,
    inf where it is negative, and inf - inf in its own place; where x is 0 the product of the two is no number."""
    import torch
    dt = _type(dtype)
    for column in (0, *_shared_columns(dtype, cols), cols - 1):
        for rows in (3, 700):
            x = torch.ones(rows, cols, device="cuda").to(dt)
            x[:, 1] = -1
            x[:, column] = 1
            dy = torch.full((rows, cols), 0.5, device="cuda").to(dt)
            dy[1, column] = float("inf")
            dx, rstd, dw = torch.empty_like(x), torch.ones(rows, device="cuda"), torch.empty(cols, device="cuda", dtype=dt)
            ws = torch.empty(al.rms_norm_grad_workspace(rows, cols), dtype=torch.uint8, device="cuda")
            al.rms_norm_grad(dx, [dy], x, rstd, dweight=dw, workspace=ws)
            torch.cuda.synchronize()
            want = torch.where(x[1] > 0, -float("inf"), float("inf"))
            want[column] = float("nan")
            assert torch.equal(torch.isnan(dx[1]), torch.isnan(want))
            there = ~torch.isnan(want)
            assert torch.equal(dx[1][there].float(), want[there])
            assert bool(torch.isfinite(dx[0]).all()) and bool(torch.isfinite(dx[2]).all())
            assert float(dw[column]) == float("inf") and int(torch.isfinite(dw).sum()) == cols - 1


@pytest.mark.parametrize("dtype,cols", [("bf16", 513), ("f16", 1031), ("bf16", 4101), ("f32", 259), ("f32", 1025), ("f32", 4099), ("bf16", 6149),
                                        ("f16", 8199), ("f32", 4613), ("bf16", 16389), ("f32", 16386)])
@pytest.mark.parametrize("ranks", [1, 5])
def test_backward_in_dsums_place_where_waves_share_elements(al, dtype, cols, ranks):
    """The shared elements are read and written by the wave that holds the vector moved back and by the wave in front."""
    import torch
    rows = 1300
    gen = torch.Generator(device="cuda").manual_seed(cols)
    x, dsum, *dys = (torch.randn(rows, cols, device="cuda", generator=gen).to(_type(dtype)) for _ in range(ranks + 2))
    w = torch.randn(cols, device="cuda", generator=gen)
    rstd = torch.rand(rows, device="cuda", generator=gen) + 0.5
    ws = torch.empty(al.rms_norm_grad_workspace(rows, cols), dtype=torch.uint8, device="cuda")
    want, dw, dw1 = torch.empty_like(x), torch.empty_like(w), torch.empty_like(w)
    al.rms_norm_grad(want, dys, x, rstd, weight=w, dsum=dsum, dweight=dw, workspace=ws)
    al.rms_norm_grad(dsum, dys, x, rstd, weight=w, dsum=dsum, dweight=dw1, workspace=ws)
    torch.cuda.synchronize()
    assert torch.equal(dsum, want) and torch.equal(dw, dw1)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cols", [3, 9, 77, 513, 1029, 4101])
@pytest.mark.parametrize("group", [0, 32, 128])
def test_8_bits_next_to_an_infinity(al, dtype, cols, group):
    """In a row, y is 0 beside an infinity and no number in its place, which makes its group that; in the weight, y is infinite in
    its place, the group's scale with it, and other elements of the group are 0."""
    import torch
    dt = _type(dtype)
    size = group or cols
    groups = -(-cols // size)
    columns = (0, cols - 1) if cols < 9 else (0, *_shared_columns(dtype, cols), cols - 1)
    for column in columns:
        mine = torch.zeros(groups, dtype=torch.bool, device="cuda")
        mine[column // size] = True
        elements = mine.repeat_interleave(size)[:cols]
        for rows in (3, 700):
            for where in ("row", "weight"):
                x, w = torch.ones(rows, cols, device="cuda").to(dt), torch.ones(cols, device="cuda").to(dt)
                if where == "row":
                    x[1, column] = float("inf")
                else:
                    w[column] = float("inf")
                q, scales = torch.empty(rows, cols, dtype=torch.float8_e4m3fn, device="cuda"), torch.empty(rows, groups, device="cuda")
                al.rms_norm(q, [x], weight=w, scales=scales, group=group)
                q = q.float()
                if where == "row":
                    assert bool(torch.isnan(scales[1][mine]).all()) and bool((scales[1][~mine] == 2.0 ** -126).all())
                    assert bool(torch.isnan(q[1][elements]).all()) and bool((q[1][~elements] == 0).all())
                    assert bool((q[0] == 448).all()) and bool((q[2] == 448).all())
                else:
                    assert bool((scales[:, mine] == float("inf")).all()) and bool(torch.isfinite(scales[:, ~mine]).all())
                    assert bool(torch.isnan(q[:, column]).all()) and bool((q[:, ~elements] == 448).all())
                    elements_beside = elements.clone()
                    elements_beside[column] = False
                    assert bool((q[:, elements_beside] == 0).all())
