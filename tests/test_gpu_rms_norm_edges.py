"""Values at which the root-mean-square norm and its backward pass round, overflow or share elements between lanes.

u = 2^-24 is half a step of fp32 relative to the value."""
import pytest

pytestmark = pytest.mark.gpu

U32 = 2.0 ** -24


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
