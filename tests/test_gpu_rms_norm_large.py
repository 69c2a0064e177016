"""The root-mean-square norm and its backward pass where calls are large: launch shapes of many rows, the load and store
policies of calls that caches do not hold, several launches of one call, offsets beyond 4 GiB.  Against the formulas in
64 bits, in the bounds of test_gpu_rms_norm, on every row or on a sample of them."""
import numpy as np
import pytest

from test_gpu_rms_norm import (E4M3_HALF, E4M3_MAX, U32, _half, _least, _np, _torch_type, check_backward, check_forward, forward_reference,
                               grad_reference)

pytestmark = pytest.mark.gpu


# One wave a row in teams of four (up to 512 columns of 16 bits), and two and three vectors a lane: in one wave (up to 1024 and
# 1536 columns) and in several.  fp32: half as many columns.
@pytest.mark.parametrize("dtype,cols", [("bf16", 505), ("f16", 517), ("bf16", 640), ("f16", 1021), ("bf16", 1025), ("f16", 1531), ("bf16", 1537),
                                        ("bf16", 2815), ("f16", 4099), ("f32", 259), ("f32", 515), ("f32", 767), ("f32", 771), ("f32", 2049)])
@pytest.mark.parametrize("rows", [600, 603])
def test_launch_shapes_of_many_rows(al, dtype, cols, rows):
    check_forward(al, rows, cols, 1, dtype, "same", True, seed=cols)
    check_forward(al, rows, cols, 3, dtype, "f32", False, group=0, seed=cols + 1)
    check_forward(al, rows, cols, 1, dtype, "none", rows % 2 == 0, group=64, seed=cols + 2)


def _randn(al, shape, dtype, seed):
    import torch
    out = torch.empty(shape, dtype=dtype, device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(seed)
    for part in out.split(max(1, (1 << 26) // shape[1])):
        part.copy_(torch.randn(part.shape, device="cuda", generator=gen))
    return out


def _sample(rows, *more):
    """The first and last rows, some from the middle, and those around `more`."""
    at = list(range(5)) + list(range(rows - 9, rows)) + [rows // 2 + k for k in range(-3, 4)] + [rows * k // 17 for k in range(17)]
    at += [m + k for m in more for k in range(-4, 5)]
    return sorted({a for a in at if 0 <= a < rows})


def check_rows(al, rows, cols, ranks, dtype, residual, group=None, more=(), eps=1e-5):
    """A call on the whole, its results held against the formula in a sample of rows."""
    import torch
    dt = _torch_type(dtype)
    ins = [_randn(al, (rows, cols), dt, 10 + k) for k in range(ranks)]
    res = _randn(al, (rows, cols), dt, 1) if residual else None
    total = torch.empty_like(ins[0]) if residual else None
    w = (1 + torch.randn(cols, generator=torch.Generator().manual_seed(3))).to(dt).cuda()
    rstd = torch.empty(rows, device="cuda")
    groups = 0 if group is None else -(-cols // group) if group else 1
    scales = torch.empty(rows, groups, device="cuda") if groups else None
    out = torch.empty(rows, cols, dtype=torch.float8_e4m3fn if groups else dt, device="cuda")
    al.rms_norm(out, ins, weight=w, residual=res, sum_out=total, rstd=rstd, scales=scales, group=group or 0, eps=eps)
    torch.cuda.synchronize()
    at = torch.tensor(_sample(rows, *more), device="cuda")
    s, s_off, r, r_rel, y, y_off = forward_reference([t[at] for t in ins], res[at] if residual else None, w, eps)
    assert np.all(np.abs(_np(rstd[at])[:, None] - r) <= r * (r_rel + U32))
    if residual:
        assert np.all(np.abs(_np(total[at]) - s) <= _half(dt) * (np.abs(s) + s_off) + s_off + _least(dt))
    got = _np(out.view(torch.uint8)[at].view(torch.float8_e4m3fn).float()) if groups else _np(out[at])
    if not groups:
        assert np.all(np.abs(got - y) <= _half(dt) * (np.abs(y) + y_off) + y_off + _least(dt))
        return
    sc, size = _np(scales[at]), group or cols
    for g in range(groups):
        a, b = g * size, min(cols, (g + 1) * size)
        want = np.maximum(np.abs(y[:, a:b]).max(1) / E4M3_MAX, 2.0 ** -126)
        assert np.all(np.abs(sc[:, g] - want) <= y_off[:, a:b].max(1) / E4M3_MAX + 2 * U32 * want)
        q_off = y_off[:, a:b] + 3 * U32 * np.abs(y[:, a:b])
        bound = np.maximum(E4M3_HALF * (np.abs(y[:, a:b]) + q_off), 2.0 ** -10 * sc[:, g:g + 1]) + q_off
        assert np.all(np.abs(got[:, a:b] * sc[:, g:g + 1] - y[:, a:b]) <= bound), g


@pytest.mark.parametrize("rows,cols,ranks,dtype,residual,group", [
    (8200, 4096, 1, "bf16", True, None),    # whole 64-byte pieces: written through
    (9400, 4096, 1, "f16", True, 128),
    (6600, 8192, 2, "bf16", False, 0),
    (2100, 8192, 8, "bf16", True, None),
    (2100, 8192, 8, "f16", True, 32),
    (4100, 4096, 3, "f32", True, None),
    (5100, 4096, 3, "f32", False, 64),
    (7001, 5125, 1, "bf16", True, None),    # rows that start in the middle of a dword
    (7601, 5125, 1, "f16", True, 128),
    (4001, 9001, 3, "f16", True, 0),
    (3001, 5002, 4, "f32", True, None),
    (40, 32768, 64, "f32", True, None),
])
def test_calls_that_caches_do_not_hold(al, rows, cols, ranks, dtype, residual, group):
    import torch
    es = 4 if dtype == "f32" else 2
    assert rows * cols * (es * (ranks + 2 * residual) + (es if group is None else 1)) >= 256 << 20
    check_rows(al, rows, cols, ranks, dtype, residual, group)
    torch.cuda.empty_cache()


@pytest.mark.parametrize("rows,cols,ranks,dtype,dsum", [(2100, 8192, 1, "bf16", True), (8200, 1024, 3, "f32", False), (3001, 5125, 4, "f16", True),
                                                        (4000, 5002, 1, "f32", True), (300, 32768, 2, "bf16", True), (300, 32768, 1, "f32", True),
                                                        (16390, 1031, 2, "bf16", True)])
def test_backward_calls_that_caches_do_not_hold(al, rows, cols, ranks, dtype, dsum):
    import torch
    dt = _torch_type(dtype)
    assert rows * cols * dt.itemsize * (ranks + 2 + dsum) >= 64 << 20
    dys = [_randn(al, (rows, cols), dt, 10 + k) for k in range(ranks)]
    x = _randn(al, (rows, cols), dt, 1)
    ds = _randn(al, (rows, cols), dt, 2) if dsum else None
    w = torch.randn(cols, generator=torch.Generator().manual_seed(3)).cuda()
    rstd = (x.double().square().mean(1) + 1e-5).rsqrt().float()
    dx, dw = torch.empty_like(x), torch.empty(cols, device="cuda")
    ws = torch.empty(al.rms_norm_grad_workspace(rows, cols), dtype=torch.uint8, device="cuda")
    al.rms_norm_grad(dx, dys, x, rstd, weight=w, dsum=ds, dweight=dw, workspace=ws)
    torch.cuda.synchronize()
    at = torch.tensor(_sample(rows), device="cuda")
    want, off, _, _ = grad_reference([t[at] for t in dys], x[at], rstd[at], w, ds[at] if dsum else None, 1)
    assert np.all(np.abs(_np(dx[at]) - want) <= _half(dt) * (np.abs(want) + off) + off + _least(dt))
    want, mag = torch.zeros(cols, dtype=torch.float64, device="cuda"), torch.zeros(cols, dtype=torch.float64, device="cuda")
    for a in range(0, rows, 1024):
        n = x[a:a + 1024].double() * rstd[a:a + 1024, None].double()
        want += (sum(t[a:a + 1024].double() for t in dys) * n).sum(0)
        mag += (sum(t[a:a + 1024].double().abs() for t in dys) * n.abs()).sum(0)
    off = (ranks + 2 + min(rows, rows // 128 + 150)) * U32 * mag
    assert bool(((dw.double() - want).abs() <= U32 * (want.abs() + off) + off).all())
    del dys, x, ds, dx
    torch.cuda.empty_cache()


@pytest.mark.parametrize("cols,rows,group", [(8, (1 << 23) + 9, None), (9, (1 << 23) + 2, 0), (2, (1 << 29) + 259, None)])
def test_more_workgroups_than_one_launch_takes(al, cols, rows, group):
    """2^21 workgroups of four rows, or of 256 rows shorter than a vector: the rows behind them are another launch's."""
    import torch
    check_rows(al, rows, cols, 1, "bf16", group is not None, group, more=(1 << 23, 1 << 29))
    torch.cuda.empty_cache()


def test_rows_on_both_sides_of_4_gib(al):
    """16384 bytes a row: the 262144th begins 2^32 bytes from the first."""
    import torch
    check_rows(al, 262_400, 8192, 1, "bf16", True, more=(1 << 18,))
    torch.cuda.empty_cache()


@pytest.mark.parametrize("dtype,cols", [("bf16", 6170), ("f16", 8190), ("f32", 3100)])
def test_backward_of_rows_that_one_team_takes_in_turn(al, dtype, cols):
    """Two vectors a lane: a workgroup has one row at a time."""
    check_backward(al, 700, cols, 1, dtype, "same", True)
    check_backward(al, 513, cols, 5, dtype, "f32", False)
