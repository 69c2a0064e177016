"""The root-mean-square norm over rank contributions and its backward pass on the GPU, against the formulas in
64 bits.

Tolerances are counted in half steps, u = eps / 2 of a type relative to the value: one for the rounding of the
output, the others for the fp32 arithmetic in front of it.  u32 = 2^-24.  A sum over a row runs through at most
54 additions in a row of one lane's elements (32), the lanes (6) and the waves (16), so ROW = 64 half steps
of the sum of the magnitudes cover it with the products' roundings."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U32, ROW = 2.0 ** -24, 64
E4M3_HALF, E4M3_MAX = 2.0 ** -4, 448.0


def _torch_type(name):
    import torch
    return {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}[name]


def _half(dtype):
    import torch
    return torch.finfo(dtype).eps / 2


def _least(dtype):
    """Half the distance between the smallest numbers of a type."""
    import torch
    f = torch.finfo(dtype)
    return f.tiny * f.eps / 2


def _np(t):
    return t.detach().double().cpu().numpy()


def _matrix(shape, dtype, pad=0, seed=0, scale=1.0):
    """A matrix whose rows are `pad` elements apart from their end, with sentinels around the whole and between."""
    import torch
    gen = torch.Generator().manual_seed(seed)
    rows, cols = shape
    canvas = torch.full((rows * (cols + pad) + 2,), 77.0, dtype=dtype, device="cuda")
    view = canvas[1:1 + rows * (cols + pad)].view(rows, cols + pad)[:, :cols]
    view.copy_((torch.randn(rows, cols, generator=gen) * scale).to(dtype))
    return view, canvas


def _assert_untouched(view, canvas, pad):
    rows, cols = view.shape
    c = canvas.float()
    assert c[0] == 77 and c[-1] == 77, "elements around the matrix were written"
    if pad:
        between = c[1:-1].view(rows, cols + pad)[:, cols:]
        assert bool((between == 77).all()), "elements between the rows were written"


def forward_reference(ins, res, w, eps):
    """s, the bound of its fp32 error, rstd, y and the bounds of theirs, in 64 bits."""
    terms = [_np(t) for t in ins] + ([_np(res)] if res is not None else [])
    s = sum(terms)
    s_off = len(terms) * U32 * sum(np.abs(t) for t in terms) * (len(terms) > 1)
    w = np.ones(s.shape[1]) if w is None else _np(w)
    ms = (s * s).mean(1, keepdims=True)
    rstd = 1 / np.sqrt(ms + eps)
    # d(rstd) / rstd = -rstd^2 mean(s ds); half of the row sum's own error; two half steps of the root
    r_rel = rstd ** 2 * (np.abs(s) * s_off).mean(1, keepdims=True) + (ROW / 2 + 4) * U32
    y = s * rstd * w
    y_off = np.abs(w) * rstd * s_off + np.abs(y) * (r_rel + 4 * U32)
    return s, s_off, rstd, r_rel, y, y_off


def check_forward(al, rows, cols, ranks, dtype, weight, residual, group=None, pads=(0, 0, 0), eps=1e-5, seed=0, edit=None):
    import torch
    dt = _torch_type(dtype)
    shape = (rows, cols)
    ins = [_matrix(shape, dt, pads[0], seed + 10 + k) for k in range(ranks)]
    res = _matrix(shape, dt, pads[1], seed + 1, 3.0) if residual else None
    sum_out = _matrix(shape, dt, pads[1], seed + 2) if residual else None
    wdt = {"same": dt, "f32": torch.float32, "none": None}[weight]
    w = None if wdt is None else torch.randn(cols, generator=torch.Generator().manual_seed(seed + 3)).to(wdt).cuda()
    rstd = torch.full((rows + 2,), 77.0, device="cuda")
    if edit:
        edit([v for v, _ in ins], res and res[0], w)
    if group is None:
        out, out_canvas = _matrix(shape, dt, pads[2], seed + 4)
        scales = None
    else:
        groups = -(-cols // group) if group else 1
        scales = torch.full((rows * groups + 2,), 77.0, device="cuda")
        out_canvas = torch.full((rows * (cols + pads[2]) + 2,), 77, dtype=torch.uint8, device="cuda")
        out = out_canvas[1:1 + rows * (cols + pads[2])].view(rows, cols + pads[2])[:, :cols].view(torch.float8_e4m3fn)
    al.rms_norm(out, [v for v, _ in ins], weight=w, residual=res and res[0], sum_out=sum_out and sum_out[0], rstd=rstd[1:-1],
                scales=None if scales is None else scales[1:-1].view(rows, -1), group=group or 0, eps=eps)
    torch.cuda.synchronize()
    s, s_off, r, r_rel, y, y_off = forward_reference([v for v, _ in ins], res and res[0], w, eps)
    assert rstd[0] == 77 and rstd[-1] == 77
    got_r = _np(rstd[1:-1])[:, None]
    assert np.all(np.abs(got_r - r) <= r * (r_rel + U32)), np.max(np.abs(got_r / r - 1))
    if sum_out is not None:
        assert np.all(np.abs(_np(sum_out[0]) - s) <= _half(dt) * (np.abs(s) + s_off) + s_off + _least(dt))
        _assert_untouched(*sum_out, pads[1])
    if group is None:
        assert np.all(np.abs(_np(out) - y) <= _half(dt) * (np.abs(y) + y_off) + y_off + _least(dt))
        _assert_untouched(out, out_canvas, pads[2])
        return out
    assert scales[0] == 77 and scales[-1] == 77
    got = _np(out.view(torch.uint8).view(torch.float8_e4m3fn).float())
    sc = _np(scales[1:-1]).reshape(rows, -1)
    step = group or cols
    for g in range(sc.shape[1]):
        a, b = g * step, min(cols, (g + 1) * step)
        amax = np.abs(y[:, a:b]).max(1)
        want = np.maximum(amax / E4M3_MAX, 2.0 ** -126)
        off = y_off[:, a:b].max(1) / E4M3_MAX + 2 * U32 * want
        assert np.all(np.abs(sc[:, g] - want) <= off), (g, sc[:, g], want)
        scale = sc[:, g:g + 1]
        # half a step of e4m3 (of its smallest numbers: 2^-10), with the error of what is rounded and three
        # half steps of fp32 in the quotient
        q_off = y_off[:, a:b] + 3 * U32 * np.abs(y[:, a:b])
        bound = np.maximum(E4M3_HALF * (np.abs(y[:, a:b]) + q_off), 2.0 ** -10 * scale) + q_off
        assert np.all(np.abs(got[:, a:b] * scale - y[:, a:b]) <= bound), g
        largest = np.abs(got[:, a:b]).max(1)
        assert np.all((largest == E4M3_MAX) | (amax / E4M3_MAX < 2.0 ** -126)), g
    c = out_canvas
    assert c[0] == 77 and c[-1] == 77
    if pads[2]:
        assert bool((c[1:-1].view(rows, cols + pads[2])[:, cols:] == 77).all())
    return out


COLS = [1, 2, 3, 4, 5, 7, 8, 9, 31, 64, 65, 129, 500, 511, 512, 513, 1024, 1027, 2048, 2049, 4095, 4097, 8192, 8199, 16384, 16391,
        32767, 32768]


@pytest.mark.parametrize("cols", COLS)
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_every_width(al, dtype, cols):
    check_forward(al, 3, cols, 1, dtype, "same", True, seed=cols)
    check_forward(al, 5, cols, 2, dtype, "f32", False, seed=cols + 1)
    for group in (0, 32, 128):
        check_forward(al, 2, cols, 1, dtype, "same", group == 32, group=group, seed=cols + 2)


@pytest.mark.parametrize("rows", [1, 2, 7, 64, 257, 1111, 5000])
@pytest.mark.parametrize("cols", [40, 123, 640, 2055, 4104])
def test_numbers_of_rows(al, rows, cols):
    check_forward(al, rows, cols, 2, "bf16", "same", True, seed=rows)
    check_forward(al, rows, cols, 1, "f16", "none", False, group=64, seed=rows)


@pytest.mark.parametrize("ranks", [1, 2, 3, 4, 5, 7, 8, 9, 13, 64])
@pytest.mark.parametrize("dtype,cols", [("bf16", 2051), ("f32", 300), ("f16", 5)])
def test_numbers_of_ranks(al, ranks, dtype, cols):
    check_forward(al, 4, cols, ranks, dtype, "same", True, seed=ranks)
    check_forward(al, 4, cols, ranks, dtype, "none", False, group=0, seed=ranks)


@pytest.mark.parametrize("pads", [(1, 0, 0), (0, 3, 5), (8, 8, 8), (2, 7, 1)])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("cols", [6, 96, 515, 4100])
def test_rows_apart(al, pads, dtype, cols):
    check_forward(al, 9, cols, 3, dtype, "f32", True, pads=pads)
    check_forward(al, 9, cols, 1, dtype, "same", True, group=32, pads=pads)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("cols", [3, 77, 1029, 9001])
@pytest.mark.parametrize("group", [None, 0, 64])
def test_rows_that_are_not_numbers(al, dtype, cols, group):
    """A row of zeros, one with a NaN, one with an infinity, one of the smallest numbers: each keeps to itself."""
    import torch
    dt = _torch_type(dtype)
    x = torch.randn(6, cols, generator=torch.Generator().manual_seed(1)).to(dt)
    x[1] = 0
    x[2, cols // 2] = float("nan")
    x[3, cols - 1] = float("inf")
    x[4] = torch.finfo(dt).tiny
    clean = x.clone()
    clean[2:4] = 1
    outs = []
    for m in (x, clean):
        out = torch.empty(m.shape, dtype=dt if group is None else torch.float8_e4m3fn, device="cuda")
        groups = 0 if group is None else -(-cols // group) if group else 1
        scales = torch.empty(6, groups, device="cuda") if groups else None
        rstd = torch.empty(6, device="cuda")
        al.rms_norm(out, [m.cuda()], rstd=rstd, scales=scales, group=group or 0, eps=1e-5)
        outs.append((out.float().cpu(), rstd.cpu(), scales.cpu() if groups else None))
    got, want = outs
    for r in (0, 1, 4, 5):
        assert torch.equal(got[0][r], want[0][r]) and got[1][r] == want[1][r]
        if group is not None:
            assert torch.equal(got[2][r], want[2][r])
    assert bool((got[0][1] == 0).all()) and abs(float(got[1][1]) * 1e-5 ** 0.5 - 1) < 1e-6
    if group is not None:
        assert bool((got[2][1] == 2.0 ** -126).all())
    assert torch.isnan(got[1][2]) and bool(torch.isnan(got[0][2]).all())
    # rstd = 0 next to an infinity: zeros, and 0 * inf in its own place
    assert got[1][3] == 0 and torch.isnan(got[0][3, cols - 1])
    if group is None:
        assert bool((got[0][3, :cols - 1] == 0).all())


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("cols", [5, 203, 2049, 8205, 20001])
def test_in_place(al, dtype, cols):
    """The sum in the residual's place and the output in an input's, at widths whose last vector is moved back."""
    import torch
    dt = _torch_type(dtype)
    rows = 700
    gen = torch.Generator(device="cuda").manual_seed(cols)
    a, b, res = (torch.randn(rows, cols, device="cuda", generator=gen).to(dt) for _ in range(3))
    w = torch.randn(cols, device="cuda", generator=gen).to(dt)
    out, total = torch.empty_like(a), torch.empty_like(a)
    al.rms_norm(out, [a, b], weight=w, residual=res, sum_out=total)
    a1, b1, r1 = a.clone(), b.clone(), res.clone()
    al.rms_norm(a1, [a1, b1], weight=w, residual=r1, sum_out=r1)
    a2, b2, r2 = a.clone(), b.clone(), res.clone()
    al.rms_norm(r2, [a2, b2], weight=w, residual=r2, sum_out=b2)
    torch.cuda.synchronize()
    assert torch.equal(a1, out) and torch.equal(r1, total) and torch.equal(b1, b)
    assert torch.equal(r2, out) and torch.equal(b2, total) and torch.equal(a2, a)


def test_columns_of_a_wider_matrix(al):
    """Inputs and output as columns of one buffer, side by side."""
    import torch
    wide = torch.randn(50, 700, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2)).bfloat16()
    before = wide.clone()
    x, y, res = wide[:, 3:203], wide[:, 203:403], wide[:, 450:650]
    want = torch.empty(50, 200, dtype=torch.bfloat16, device="cuda")
    al.rms_norm(want, [x.contiguous(), x.contiguous()], residual=res.contiguous())
    al.rms_norm(y, [x, x], residual=res)
    torch.cuda.synchronize()
    assert torch.equal(y, want)
    before[:, 203:403] = want
    assert torch.equal(wide, before)


def test_empty_calls(al):
    import torch
    e = torch.empty(0, 8, device="cuda")
    al.rms_norm(e.clone(), [e], rstd=torch.empty(0, device="cuda"))
    rstd = torch.full((4,), 7.0, device="cuda")
    z = torch.empty(4, 0, device="cuda")
    al.rms_norm(z.clone(), [z], rstd=rstd)
    dw = torch.full((8,), 7.0, device="cuda")
    al.rms_norm_grad(e.clone(), [e], e, torch.empty(0, device="cuda"), dweight=dw)
    torch.cuda.synchronize()
    assert bool((rstd == 7).all()) and bool((dw == 0).all())


def grad_reference(dys, x, rstd, w, dsum, parts):
    dy = sum(_np(d) for d in dys)
    mag = sum(np.abs(_np(d)) for d in dys)
    x, r = _np(x), _np(rstd)[:, None]
    w = np.ones(x.shape[1]) if w is None else _np(w)
    P, (rows, cols) = len(dys), x.shape
    n, g, gm = x * r, dy * w, mag * np.abs(w)
    c = (g * n).mean(1, keepdims=True)
    dx = r * (g - n * c)
    # P half steps for dy, one each for n, g, the product; the row sum; two for the last two operations
    c_off = (P + ROW + 4) * U32 * (gm * np.abs(n)).mean(1, keepdims=True)
    dx_off = r * ((P + 3) * U32 * gm + np.abs(n) * (c_off + 4 * U32 * np.abs(c))) + 2 * U32 * np.abs(dx)
    if dsum is not None:
        dx = dx + _np(dsum)
        dx_off = dx_off + U32 * np.abs(dx)
    dw = (dy * n).sum(0)
    # a lane adds at most rows / 128 products, or all of them, before the lanes, slices and workgroups meet
    dw_off = (P + 2 + min(rows, rows // 128 + 150)) * U32 * (mag * np.abs(n)).sum(0)
    return dx, dx_off, dw, dw_off


def check_backward(al, rows, cols, ranks, dtype, weight, dsum, pads=(0, 0, 0, 0), seed=0):
    import torch
    dt = _torch_type(dtype)
    shape = (rows, cols)
    dys = [_matrix(shape, dt, pads[0], seed + 10 + k) for k in range(ranks)]
    x = _matrix(shape, dt, pads[1], seed + 1, 2.0)
    ds = _matrix(shape, dt, pads[2], seed + 2) if dsum else None
    dx = _matrix(shape, dt, pads[3], seed + 5)
    wdt = {"same": dt, "f32": torch.float32, "none": None}[weight]
    w = None if wdt is None else torch.randn(cols, generator=torch.Generator().manual_seed(seed + 3)).to(wdt).cuda()
    dw_canvas = torch.full((cols + 2,), 77.0, dtype=wdt or torch.float32, device="cuda")
    rstd = (1 / (x[0].float().square().mean(1) + 1e-5).sqrt()).contiguous()
    ws = torch.full((al.rms_norm_grad_workspace(rows, cols) + 8,), 77, dtype=torch.uint8, device="cuda")
    al.rms_norm_grad(dx[0], [v for v, _ in dys], x[0], rstd, weight=w, dsum=ds and ds[0], dweight=dw_canvas[1:-1], workspace=ws[4:-4])
    torch.cuda.synchronize()
    want_dx, dx_off, want_dw, dw_off = grad_reference([v for v, _ in dys], x[0], rstd, w, ds and ds[0], 1)
    assert np.all(np.abs(_np(dx[0]) - want_dx) <= _half(dt) * (np.abs(want_dx) + dx_off) + dx_off + _least(dt))
    _assert_untouched(*dx, pads[3])
    h = _half(dw_canvas.dtype)
    assert np.all(np.abs(_np(dw_canvas[1:-1]) - want_dw) <= h * (np.abs(want_dw) + dw_off) + dw_off + _least(dw_canvas.dtype))
    assert dw_canvas[0] == 77 and dw_canvas[-1] == 77
    assert bool((ws[:4] == 77).all()) and bool((ws[-4:] == 77).all())
    # each of the two alone gives the same bits
    alone = torch.empty(shape, dtype=dt, device="cuda")
    al.rms_norm_grad(alone, [v for v, _ in dys], x[0], rstd, weight=w, dsum=ds and ds[0])
    dw = torch.empty(cols, dtype=dw_canvas.dtype, device="cuda")
    al.rms_norm_grad(None, [v for v, _ in dys], x[0], rstd, weight=w, dweight=dw, workspace=ws[4:-4])
    torch.cuda.synchronize()
    assert torch.equal(alone, dx[0]) and torch.equal(dw, dw_canvas[1:-1])


@pytest.mark.parametrize("cols", COLS)
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_backward_every_width(al, dtype, cols):
    check_backward(al, 3, cols, 1, dtype, "same", True, seed=cols)
    check_backward(al, 1, cols, 3, dtype, "f32", False, seed=cols + 1)


@pytest.mark.parametrize("rows", [1, 2, 7, 65, 1024, 1025, 5000])
@pytest.mark.parametrize("dtype,cols", [("bf16", 5), ("bf16", 100), ("f32", 257), ("f16", 2060), ("f32", 4099)])
def test_backward_numbers_of_rows(al, rows, dtype, cols):
    check_backward(al, rows, cols, 2, dtype, "none" if rows % 2 else "same", rows > 64, seed=rows)


@pytest.mark.parametrize("pads", [(1, 0, 3, 2), (4, 4, 4, 4), (0, 5, 0, 1)])
@pytest.mark.parametrize("cols", [6, 96, 515, 4100])
def test_backward_rows_apart(al, pads, cols):
    check_backward(al, 11, cols, 4, "bf16", "f32", True, pads=pads)


@pytest.mark.parametrize("ranks", [8, 64])
def test_backward_many_ranks(al, ranks):
    check_backward(al, 6, 1030, ranks, "f32", "same", True)
    check_backward(al, 6, 1030, ranks, "f16", "same", False)


@pytest.mark.parametrize("cols", [5, 203, 2049, 8205, 20001])
@pytest.mark.parametrize("place", ["dy", "x", "dsum"])
def test_backward_in_place(al, cols, place):
    import torch
    rows = 1500
    gen = torch.Generator(device="cuda").manual_seed(cols)
    t = {k: torch.randn(rows, cols, device="cuda", generator=gen).bfloat16() for k in ("dy", "other", "x", "dsum")}
    w = torch.randn(cols, device="cuda", generator=gen)
    rstd = torch.rand(rows, device="cuda", generator=gen) + 0.5
    ws = torch.empty(al.rms_norm_grad_workspace(rows, cols), dtype=torch.uint8, device="cuda")
    dx, dw, dw1 = torch.empty_like(t["x"]), torch.empty_like(w), torch.empty_like(w)
    al.rms_norm_grad(dx, [t["dy"], t["other"]], t["x"], rstd, weight=w, dsum=t["dsum"], dweight=dw, workspace=ws)
    al.rms_norm_grad(t[place], [t["dy"], t["other"]], t["x"], rstd, weight=w, dsum=t["dsum"], dweight=dw1, workspace=ws)
    torch.cuda.synchronize()
    assert torch.equal(t[place], dx) and torch.equal(dw, dw1)


@pytest.mark.parametrize("dtype,cols", [("bf16", 513), ("bf16", 1025), ("f16", 4101), ("f32", 257), ("f32", 2051), ("bf16", 8193),
                                        ("bf16", 16391), ("f32", 8194), ("f32", 16387)])
def test_backward_in_place_where_waves_share_elements(al, dtype, cols):
    """The last vector, moved back, is the first of a wave and shares elements with the wave's before, which writes them."""
    import torch
    rows = 600
    x, dy, dsum = (_matrix((rows, cols), _torch_type(dtype), 0, 30 + k)[0] for k in range(3))
    rstd = torch.rand(rows, device="cuda") + 0.5
    want = torch.empty_like(x)
    al.rms_norm_grad(want, [dy], x, rstd, dsum=dsum)
    al.rms_norm_grad(dsum, [dy], x, rstd, dsum=dsum)
    assert torch.equal(dsum, want)


def test_gradients_against_differences(al):
    """sum(out * t) moved along the axes, in 64 bits, against dx and dweight of a call in fp32."""
    import torch
    rows, cols, eps, h = 3, 37, 1e-3, 1e-5
    gen = torch.Generator().manual_seed(9)
    a, b, res, t, ds = (torch.randn(rows, cols, generator=gen, dtype=torch.float64) for _ in range(5))
    w = torch.randn(cols, generator=gen, dtype=torch.float64)
    a, b, res, t, ds, w = (v.float().double() for v in (a, b, res, t, ds, w))

    def loss(a, w):
        s = a + b + res
        return ((s * (s.square().mean(1, keepdim=True) + eps).rsqrt() * w) * t + s * ds).sum()

    out, total = torch.empty(rows, cols, device="cuda"), torch.empty(rows, cols, device="cuda")
    rstd = torch.empty(rows, device="cuda")
    g = lambda v: v.float().cuda()  # noqa: E731
    al.rms_norm(out, [g(a), g(b)], weight=g(w), residual=g(res), sum_out=total, rstd=rstd, eps=eps)
    dx, dw = torch.empty_like(out), torch.empty(cols, device="cuda")
    ws = torch.empty(al.rms_norm_grad_workspace(rows, cols), dtype=torch.uint8, device="cuda")
    al.rms_norm_grad(dx, [g(t)], total, rstd, weight=g(w), dsum=g(ds), dweight=dw, workspace=ws)
    dx, dw = dx.double().cpu(), dw.double().cpu()
    for i in range(rows):
        for j in range(cols):
            up, down = a.clone(), a.clone()
            up[i, j] += h
            down[i, j] -= h
            # h^2 for the difference, fp32 for the call: both far below 1e-4 of gradients of order one
            assert abs(float(loss(up, w) - loss(down, w)) / (2 * h) - float(dx[i, j])) < 1e-4
    for j in range(cols):
        up, down = w.clone(), w.clone()
        up[j] += h
        down[j] -= h
        assert abs(float(loss(a, up) - loss(a, down)) / (2 * h) - float(dw[j])) < 1e-4


def test_offsets_beyond_4_gib(al):
    """A matrix of 5 GB: the last rows against the same rows in a call of their own."""
    import torch
    rows, cols, tail = 310_003, 8192, 5
    x = torch.empty(rows, cols, dtype=torch.bfloat16, device="cuda")
    for k in range(0, rows, 50_000):
        x[k:k + 50_000].normal_(generator=torch.Generator(device="cuda").manual_seed(k))
    out, dx = torch.empty_like(x), torch.empty_like(x)
    rstd = torch.empty(rows, device="cuda")
    w = torch.rand(cols, device="cuda") + 0.5
    al.rms_norm(out, [x], weight=w, rstd=rstd)
    al.rms_norm_grad(dx, [out], x, rstd, weight=w)
    small, small_dx = torch.empty_like(x[-tail:]), torch.empty_like(x[-tail:])
    small_rstd = torch.empty(tail, device="cuda")
    al.rms_norm(small, [x[-tail:]], weight=w, rstd=small_rstd)
    al.rms_norm_grad(small_dx, [small], x[-tail:], small_rstd, weight=w)
    torch.cuda.synchronize()
    # another number of rows may be dealt to other teams, whose sums run in another order: 2 ROW half steps
    assert torch.allclose(rstd[-tail:], small_rstd, rtol=2 * ROW * U32, atol=0)
    for got, want in ((out, small), (dx, small_dx)):
        a, b = got[-tail:].double(), want.double()
        assert float((a - b).abs().max()) <= 2 * 2.0 ** -8 * float(b.abs().max())
        assert float((a != b).double().mean()) < 0.01


def test_captured_and_on_another_stream(al):
    """Both passes captured together, replayed with new inputs and eager work in between; the same on a stream of
    their own."""
    import torch
    rows, cols = 67, 1031
    ins = [torch.zeros(rows, cols, device="cuda") for _ in range(3)]
    res, t = torch.zeros(rows, cols, device="cuda"), torch.zeros(rows, cols, device="cuda")
    w = torch.rand(cols, device="cuda")
    out, total, dx = (torch.empty(rows, cols, device="cuda") for _ in range(3))
    q = torch.empty(rows, cols, dtype=torch.float8_e4m3fn, device="cuda")
    rstd, scales, dw = torch.empty(rows, device="cuda"), torch.empty(rows, 17, device="cuda"), torch.empty(cols, device="cuda")
    ws = torch.empty(al.rms_norm_grad_workspace(rows, cols), dtype=torch.uint8, device="cuda")

    def step(stream=None):
        al.rms_norm(out, ins, weight=w, residual=res, sum_out=total, rstd=rstd, stream=stream)
        al.rms_norm(q, ins, weight=w, residual=res, scales=scales, group=64, stream=stream)
        al.rms_norm_grad(dx, [t], total, rstd, weight=w, dweight=dw, workspace=ws, stream=stream)

    results = lambda: [v.clone() for v in (out, total, rstd, dx, dw, scales, q.view(torch.uint8))]  # noqa: E731
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    side = torch.cuda.Stream()
    for rep in range(3):
        for k, m in enumerate(ins + [res, t]):
            m.copy_(torch.randn(rows, cols, generator=torch.Generator().manual_seed(10 * rep + k)))
        step()
        torch.cuda.synchronize()
        want = results()
        for m in (out, total, dx, dw, rstd, scales):
            m.fill_(float("nan"))
        q.view(torch.uint8).zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(results(), want):
            assert torch.equal(a, b)
        for m in (out, total, dx, dw, rstd, scales):
            m.fill_(float("nan"))
        q.view(torch.uint8).zero_()
        torch.cuda.synchronize()
        step(side)
        side.synchronize()
        for a, b in zip(results(), want):
            assert torch.equal(a, b)


def test_refusals(al):
    """What the binding and the library refuse, with nothing written."""
    import torch
    x, y = torch.ones(6, 64, device="cuda"), torch.full((6, 64), 7.0, device="cuda")
    wide = torch.ones(6, 128, device="cuda")
    rstd, w = torch.ones(6, device="cuda"), torch.ones(64, device="cuda")
    q, sc = torch.zeros(6, 64, dtype=torch.float8_e4m3fn, device="cuda"), torch.ones(6, 2, device="cuda")
    dw = torch.full((64,), 7.0, device="cuda")
    ws = torch.empty(al.rms_norm_grad_workspace(6, 64), dtype=torch.uint8, device="cuda")
    for code, call in [
            (1, lambda: al.rms_norm(y, [])), (1, lambda: al.rms_norm(y, [x[0]])), (1, lambda: al.rms_norm(y[:5], [x])),
            (1, lambda: al.rms_norm(y.bfloat16(), [x])), (1, lambda: al.rms_norm(y, [x, x.bfloat16()])),
            (1, lambda: al.rms_norm(y, [x, wide[:, :64]])), (1, lambda: al.rms_norm(y, [x, x[:, :63]])),
            (1, lambda: al.rms_norm(y, [x.cpu()])), (1, lambda: al.rms_norm(y, [x, x.cpu()])), (1, lambda: al.rms_norm(y, [wide[:, ::2]])),
            (1, lambda: al.rms_norm(y, [x[:1].expand(6, 64)])), (3, lambda: al.rms_norm(y.double(), [x.double()])),
            (1, lambda: al.rms_norm(y, [x], weight=w[:63])), (3, lambda: al.rms_norm(y, [x], weight=w.half())),
            (1, lambda: al.rms_norm(y, [x], residual=x, sum_out=wide[:, :64])), (1, lambda: al.rms_norm(y, [x], rstd=rstd[:5])),
            (1, lambda: al.rms_norm(y, [x], rstd=rstd.double())), (1, lambda: al.rms_norm(y, [x], scales=sc, group=32)),
            (1, lambda: al.rms_norm(q, [x], scales=sc, group=48)), (1, lambda: al.rms_norm(q, [x], scales=sc)),
            (1, lambda: al.rms_norm(q, [x])), (1, lambda: al.rms_norm(y, [x], group=32)), (1, lambda: al.rms_norm(y, [x], eps=-1.0)),
            (5, lambda: al.rms_norm(wide[:, 1:65], [wide[:, :64]])), (5, lambda: al.rms_norm(y, [x], residual=x, sum_out=y)),
            (1, lambda: al.rms_norm_grad(y, [], x, rstd)), (1, lambda: al.rms_norm_grad(None, [x], x, rstd)),
            (1, lambda: al.rms_norm_grad(y, [x], x.half(), rstd)), (1, lambda: al.rms_norm_grad(y, [x], x, rstd[:5])),
            (1, lambda: al.rms_norm_grad(y, [x], x, rstd, dweight=dw)), (1, lambda: al.rms_norm_grad(y, [x], x, rstd, dweight=dw, workspace=ws[:-1])),
            (1, lambda: al.rms_norm_grad(y, [x], x, rstd, weight=w, dweight=dw.half(), workspace=ws)),
            (1, lambda: al.rms_norm_grad(None, [x], x, rstd, dsum=x, dweight=dw, workspace=ws)),
            (5, lambda: al.rms_norm_grad(wide[:, 1:65], [x], wide[:, :64], rstd)),
            (5, lambda: al.rms_norm_grad(y, [x], x, rstd, weight=w, dweight=ws.view(torch.float32)[:64], workspace=ws))]:
        with pytest.raises(al.AlError) as e:
            call()
        assert e.value.code == code, e.value
    torch.cuda.synchronize()
    assert bool((y == 7).all()) and bool((dw == 7).all()) and bool((x == 1).all()) and bool((wide == 1).all())


def test_two_streams_at_once(al):
    """Calls on two streams at once, each with its own buffers."""
    import torch
    side = [torch.cuda.Stream() for _ in range(2)]
    sets = []
    for k in range(2):
        gen = torch.Generator(device="cuda").manual_seed(k)
        x, t = (torch.randn(3000, 1537, device="cuda", generator=gen).bfloat16() for _ in range(2))
        w = torch.rand(1537, device="cuda", generator=gen)
        ws = torch.empty(al.rms_norm_grad_workspace(3000, 1537), dtype=torch.uint8, device="cuda")
        sets.append((x, t, w, ws, torch.empty_like(x), torch.empty_like(x), torch.empty(3000, device="cuda"), torch.empty_like(w)))

    def both(s, stream):
        x, t, w, ws, out, dx, rstd, dw = s
        al.rms_norm(out, [x, t], weight=w, rstd=rstd, stream=stream)
        al.rms_norm_grad(dx, [t], x, rstd, weight=w, dweight=dw, workspace=ws, stream=stream)

    want = []
    for s in sets:
        both(s, None)
        torch.cuda.synchronize()
        want.append([v.clone() for v in s[4:]])
        for v in s[4:]:
            v.zero_()
    torch.cuda.synchronize()
    for _ in range(5):
        for s, stream in zip(sets, side):
            both(s, stream)
    torch.cuda.synchronize()
    for s, w in zip(sets, want):
        assert all(torch.equal(a, b) for a, b in zip(s[4:], w))
