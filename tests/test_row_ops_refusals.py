"""What the root-mean-square norm and the tensor lists refuse, and that they do so before any GPU work: through the C ABI
with addresses that are never touched."""
import ctypes as C

import pytest

F16, BF16, F32, F64, I32 = 8, 9, 10, 11, 4
MAX_COLS = 32768


@pytest.fixture(scope="module")
def lib():
    import aluminum_amd
    return aluminum_amd.load()


def table(*p):
    return (C.c_void_p * max(1, len(p)))(*p)


IN, RES, SUM, OUT, W, RSTD, SCALES, WS = (k << 24 for k in range(1, 9))


def norm(lib, **kw):
    a = dict(out=OUT, out_stride=64, sum=SUM, res=RES, res_stride=64, ins=table(IN, IN + (1 << 20)), P=2, in_stride=64, w=W,
             wdt=BF16, rstd=RSTD, scales=None, group=0, rows=8, cols=64, dtype=BF16, eps=1e-6)
    a.update(kw)
    return lib.alamd_rms_norm(a["out"], a["out_stride"], a["sum"], a["res"], a["res_stride"], a["ins"], a["P"], a["in_stride"], a["w"],
                              a["wdt"], a["rstd"], a["scales"], a["group"], a["rows"], a["cols"], a["dtype"], a["eps"], None)


@pytest.mark.parametrize("code,kw", [
    (1, dict(P=0)), (1, dict(P=65)), (1, dict(ins=None)), (1, dict(ins=table(IN, None))), (1, dict(out=None)),
    (3, dict(dtype=F64)), (3, dict(dtype=I32)), (3, dict(dtype=-1)), (3, dict(wdt=F16)), (3, dict(wdt=F64)),
    (1, dict(cols=MAX_COLS + 1, in_stride=1 << 20, out_stride=1 << 20, res_stride=1 << 20)),
    (1, dict(in_stride=63)), (1, dict(out_stride=63)), (1, dict(res_stride=0)),
    (1, dict(in_stride=1 << 62)), (1, dict(rows=1 << 62)),
    (1, dict(group=32)), (1, dict(group=48, scales=SCALES)), (1, dict(group=256, scales=SCALES)),
    (1, dict(eps=-1.0)), (1, dict(eps=float("nan"))),
    (1, dict(out=OUT + 1)), (1, dict(ins=table(IN, IN + 1))), (1, dict(res=RES + 1)), (1, dict(sum=SUM + 1)), (1, dict(w=W + 1)),
    (1, dict(rstd=RSTD + 2)), (1, dict(scales=SCALES + 1)),
    (5, dict(out=IN + 2)), (5, dict(out=IN + 64)), (5, dict(out=IN, out_stride=128)), (5, dict(sum=OUT)), (5, dict(sum=RES + 128)),
    (5, dict(out=IN, scales=SCALES)), (5, dict(out=W)), (5, dict(rstd=IN + 4)), (5, dict(scales=RSTD + 4)), (5, dict(rstd=OUT)),
    (5, dict(out=IN + 66, in_stride=128, out_stride=128)),  # two columns into the next matrix in the same buffer
])
def test_norm_refuses(lib, code, kw):
    assert norm(lib, **kw) == code
    assert lib.alamd_last_error()


@pytest.mark.parametrize("kw", [dict(rows=0), dict(cols=0), dict(rows=0, ins=None, out=None)])
def test_norm_of_nothing(lib, kw):
    assert norm(lib, **kw) == 0


def grad(lib, **kw):
    a = dict(dx=OUT, dx_stride=64, dys=table(IN, IN + (1 << 20)), P=2, dy_stride=64, x=RES, x_stride=64, dsum=SUM, dsum_stride=64,
             rstd=RSTD, w=W, wdt=F32, dw=SCALES, rows=8, cols=64, dtype=BF16, ws=WS)
    a.update(kw)
    return lib.alamd_rms_norm_grad(a["dx"], a["dx_stride"], a["dys"], a["P"], a["dy_stride"], a["x"], a["x_stride"], a["dsum"],
                                   a["dsum_stride"], a["rstd"], a["w"], a["wdt"], a["dw"], a["rows"], a["cols"], a["dtype"], a["ws"],
                                   None)


@pytest.mark.parametrize("code,kw", [
    (1, dict(P=0)), (1, dict(P=65)), (1, dict(dys=None)), (1, dict(dys=table(None, IN))), (1, dict(x=None)), (1, dict(rstd=None)),
    (1, dict(dx=None, dw=None)), (1, dict(dx=None)), (1, dict(ws=None)), (1, dict(ws=WS + 2)),
    (3, dict(dtype=F64)), (3, dict(wdt=F16)), (3, dict(w=None, wdt=I32)),
    (1, dict(cols=MAX_COLS + 1, dx_stride=1 << 20, dy_stride=1 << 20, x_stride=1 << 20, dsum_stride=1 << 20)),
    (1, dict(dx_stride=63)), (1, dict(dy_stride=63)), (1, dict(x_stride=63)), (1, dict(dsum_stride=63)),
    (1, dict(dx=OUT + 1)), (1, dict(x=RES + 1)), (1, dict(dsum=SUM + 1)), (1, dict(rstd=RSTD + 1)), (1, dict(dw=SCALES + 2)),
    (5, dict(dx=RES + 2)), (5, dict(dx=IN, dx_stride=65)), (5, dict(dx=RSTD)), (5, dict(dx=W)), (5, dict(dx=SCALES)), (5, dict(dx=WS)),
    (5, dict(ws=SCALES)), (5, dict(dw=IN)), (5, dict(ws=IN + (1 << 20))),
])
def test_grad_refuses(lib, code, kw):
    assert grad(lib, **kw) == code
    assert lib.alamd_last_error()


@pytest.mark.parametrize("kw", [
    dict(out=W), dict(sum=W), dict(rstd=IN, cols=2), dict(rstd=W, cols=2), dict(scales=IN, cols=2),
])
def test_norm_of_one_row_replaces_rows_alone(lib, kw):
    """A single row of a written matrix is as long as what it may not replace."""
    assert norm(lib, rows=1, **kw) == 5


@pytest.mark.parametrize("kw", [
    dict(dx=W, wdt=BF16), dict(dx=RSTD, cols=2), dict(dw=IN, wdt=BF16), dict(dw=RES, wdt=BF16), dict(dw=W), dict(dw=RSTD, cols=1),
])
def test_grad_of_one_row_replaces_rows_alone(lib, kw):
    assert grad(lib, rows=1, **kw) == 5


def test_list_refuses_more_than_a_device_holds(lib):
    assert make(lib, [IN], [(1 << 39) // 4 + 1], [F32]) == 1


def test_grad_of_nothing(lib):
    assert grad(lib, rows=0, dw=None) == 0
    assert grad(lib, cols=0) == 0


def test_grad_workspace(lib):
    size = lib.alamd_rms_norm_grad_workspace
    assert size(0, 64) == 0 and size(1, 64) >= 64 * 4
    assert size(1 << 20, MAX_COLS) <= 1024 * MAX_COLS * 4


def make(lib, ins, counts, dtypes, outs=None, n=None):
    h = C.c_void_p(None)
    n = len(ins) if n is None else n
    rc = lib.alamd_tensor_list_create(C.byref(h), None if outs is None else table(*outs), table(*ins),
                                      (C.c_size_t * max(1, len(counts)))(*counts), (C.c_int * max(1, len(dtypes)))(*dtypes), n)
    assert rc == 0 or not h
    return rc


@pytest.mark.parametrize("code,args", [
    (3, ([IN], [8], [F64])), (3, ([IN], [8], [I32])), (1, ([None], [8], [F32])), (1, ([IN], [8], [F32], [None])),
    (1, ([IN + 2], [8], [F32])), (1, ([IN], [8], [F32], [OUT + 1])), (1, ([IN], [1 << 60], [F32])),
    (5, ([IN, IN], [8, 8], [F32, F32])),                      # the same buffer twice, in place
    (5, ([IN, IN + 28], [8, 8], [F32, F32])),                 # one element in common
    (5, ([IN + 28, RES, IN], [8, 8, 8], [F32, F32, F32])),
    (5, ([IN, RES], [8, 8], [F32, F32], [OUT, OUT])),         # two outputs in one place
    (5, ([IN, RES], [8, 8], [F32, F32], [RES, OUT])),         # an output over another tensor's input
    (5, ([IN, RES], [8, 8], [F32, F32], [IN + 4, OUT])),      # an output that is moved against its input
    (5, ([IN, RES], [8, 8], [F32, F32], [RES, IN])),
    (5, ([IN, RES, SUM], [8, 900, 8], [F32, F32, F32], [OUT, W, RES + 800])),
])
def test_list_refuses(lib, code, args):
    assert make(lib, *args) == code
    assert lib.alamd_last_error()


def test_list_arguments(lib):
    h = C.c_void_p(None)
    assert lib.alamd_tensor_list_create(None, None, None, None, None, 0) == 1
    assert lib.alamd_tensor_list_create(C.byref(h), None, None, None, None, 1) == 1
    assert lib.alamd_tensor_list_destroy(None) == 0
    assert lib.alamd_global_norm(None, RSTD, WS, None) == 1
    assert lib.alamd_clip_to_norm(None, RSTD, 1.0, 0.0, None) == 1
    assert lib.alamd_clip_global_norm(None, RSTD, 1.0, 0.0, WS, None) == 1


def test_binding_checks():
    """The Python binding's own checks: tensors on the host, shapes, types, strides."""
    import torch
    import aluminum_amd as al
    x = torch.zeros(4, 8)
    for call in (lambda: al.rms_norm(x, [x]), lambda: al.rms_norm(x, [x[0]]), lambda: al.rms_norm(x[:2], [x]),
                 lambda: al.rms_norm_grad(x, [x], x, x[:, 0]), lambda: al.TensorList([x]), lambda: al.TensorList([x], [x, x])):
        with pytest.raises(al.AlError) as e:
            call()
        assert e.value.code in (1, 3)
