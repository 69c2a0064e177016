"""Cases for measuring the operators that follow a training step's two kinds of Allreduce: the
root-mean-square norm behind the sum of a layer's partial results over ranks (with the residual stream, 8-bit
outputs and the backward pass), and the norm over all gradients with the clipping by it.

`run` computes an operator in elementary torch operations, or, where `own` is set, by the calls a program makes
of this package."""
import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
EPS = 1e-6         # inside the root of the norm
CLIP_EPS = 1e-6    # added to the norm of the gradients
E4M3_MAX = 448.0
TINY = 2.0 ** -126  # the least scale of an 8-bit group
LARGEST = 1.2e9    # bytes of a drawn case


def _norm(name, rows, cols, ranks, dtype, residual, weight="same", group=-1):
    return {"name": name, "op": "norm", "rows": rows, "cols": cols, "ranks": ranks, "dtype": dtype, "residual": residual,
            "weight": weight, "group": group}


def _grad(name, rows, cols, ranks, dtype, residual, weight="same"):
    return {"name": name, "op": "grad", "rows": rows, "cols": cols, "ranks": ranks, "dtype": dtype, "residual": residual,
            "weight": weight}


def _list(name, op, layers, width, dtype, vectors, over=10.0):
    return {"name": name, "op": op, "layers": layers, "width": width, "dtype": dtype, "vectors": vectors, "over": over}


def listed():
    return [
        # one token generated, a layer split over eight ranks: nothing but latency
        _norm("norm token, 8 ranks", 1, 4096, 8, "bf16", True),
        # a prompt or a training batch of 8192 tokens on one rank, with the residual stream written back
        _norm("norm batch bf16", 8192, 8192, 1, "bf16", True),
        # the partial sums of eight ranks for 2048 tokens, folded on the way
        _norm("norm 2048 tokens, 8 ranks", 2048, 8192, 8, "bf16", True, "f32"),
        # 48 sequences in generation, the input of an 8-bit product with one scale a token
        _norm("norm 8 bits, 48 tokens", 48, 8192, 2, "bf16", True, "same", 0),
        # a prompt's tokens for an 8-bit product with a scale for each 128 columns, nothing a multiple of anything
        _norm("norm 8 bits, odd prompt f16", 8191, 4099, 1, "f16", False, "same", 128),
        # a short sequence of a small model trained in 32 bits
        _grad("grad 64 tokens f32", 64, 1024, 1, "f32", False),
        # a training batch: gradient of the norm joined with that of the residual stream, and the weight's
        _grad("grad batch bf16", 16384, 8192, 1, "bf16", True),
        # the gradients that four ranks hold of the norm's output, odd sizes
        _grad("grad odd, 4 ranks f16", 2777, 5125, 4, "f16", True, "f32"),
        # the gradients of a small model, only watched
        _list("global norm, small f32", "norm_of", 2, 64, "f32", "f32"),
        # the gradients of a medium model, 99 tensors: the norm that is logged, or joined with other devices'
        _list("global norm, medium bf16", "norm_of", 16, 2048, "bf16", "f32"),
        # matrices in 16 bits, vectors in 32: clipped before the optimizer's step
        _list("clip, 16 bits", "clip", 6, 4096, "bf16", "f32"),
        # an odd width in 32 bits: gradients that start anywhere in their bucket
        _list("clip, small model f32", "clip", 4, 513, "f32", "f32", 3.0),
    ]


def _between(rng, lo, hi):
    """Spread over the logarithm; half of them odd."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return max(lo, min(hi, v | 1 if rng.random() < 0.5 else v - v % 8 if v >= 16 else v))


def draw(rng):
    op = rng.choice(["norm", "norm", "norm8", "norm8", "grad", "grad", "norm_of", "clip"])
    while True:
        if op in ("norm", "norm8", "grad"):
            c = {"op": "grad" if op == "grad" else "norm", "rows": _between(rng, 1, 16384), "cols": _between(rng, 48, 16384),
                 "ranks": rng.choice([1, 1, 2, 3, 4, 8]), "dtype": rng.choice(["bf16", "bf16", "f16", "f32"]),
                 "residual": rng.random() < 0.6, "weight": rng.choice(["same", "same", "f32", "none"])}
            if op != "grad":
                c["group"] = -1 if op == "norm" else rng.choice([0, 0, 32, 64, 128])
            elif c["weight"] == "none":
                c["weight"] = "same"
        else:
            c = {"op": op, "layers": rng.randint(1, 24), "width": _between(rng, 32, 4096), "dtype": rng.choice(["bf16", "f16", "f32"]),
                 "vectors": "f32", "over": rng.choice([0.9, 2.0, 10.0])}
        if work(c)["bytes"] <= LARGEST:
            return c


def _shapes(case):
    """Numbers of elements of the tensors of a stack of layers: (the matrices, the vectors)."""
    w, n = case["width"], case["layers"]
    return [w * w, w * w, 2 * w * w, 2 * w * w] * n + [5 * w * w], [w, w] * n + [w, 1]


def work(case):
    if case["op"] in ("norm_of", "clip"):
        mats, vecs = _shapes(case)
        size = lambda t: TYPES[t].itemsize  # noqa: E731
        count = sum(mats) + sum(vecs)
        read = sum(mats) * size(case["dtype"]) + sum(vecs) * size(case["vectors"])
        return {"bytes": 4 + read * (2 if case["op"] == "clip" else 1), "flops": count * (3 if case["op"] == "clip" else 2)}
    rows, cols, e = case["rows"], case["cols"], TYPES[case["dtype"]].itemsize
    n, wide = rows * cols, {"same": e, "f32": 4, "none": 0}[case["weight"]] * cols
    if case["op"] == "grad":
        return {"bytes": n * e * (case["ranks"] + 2 + case["residual"]) + rows * 4 + 2 * wide, "flops": n * (case["ranks"] + 9 + case["residual"])}
    eight = case["group"] >= 0
    scales = 0 if not eight else rows * (1 if case["group"] == 0 else -(-cols // case["group"]))
    out = n * (1 if eight else e) + scales * 4
    return {"bytes": n * e * (case["ranks"] + 2 * case["residual"]) + wide + out + rows * 4, "flops": n * (case["ranks"] + 4 + 2 * eight + case["residual"])}


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(shape, dtype, by=1.0):
        return (torch.randn(shape, device="cuda", generator=gen) * by).to(dtype)

    dtype = TYPES[case["dtype"]]
    s = dict(case)
    if case["op"] in ("norm_of", "clip"):
        # the gradients of a model lie one behind another in buckets, one for each type
        mats, vecs = _shapes(case)
        s["flat"] = [normal(sum(mats), dtype, 1e-2), normal(sum(vecs), TYPES[case["vectors"]], 1e-1)]
        s["grads"] = list(s["flat"][0].split(mats)) + list(s["flat"][1].split(vecs))
        s["norm"] = torch.empty(1, dtype=torch.float32, device="cuda")
        # `over`: how often the expected norm goes into the largest one allowed
        s["max_norm"] = math.sqrt(sum(mats) * 1e-4 + sum(vecs) * 1e-2) / case["over"]
        if case["op"] == "clip":
            s["clipped"] = [torch.empty_like(f) for f in s["flat"]]
            s["outs"] = list(s["clipped"][0].split(mats)) + list(s["clipped"][1].split(vecs))
        if own:  # the table of the gradients, which a training program makes once
            import aluminum_amd as al
            s["list"] = al.TensorList(s["grads"], s.get("outs"))
        return s
    shape = (case["rows"], case["cols"])
    ranks = case["ranks"]
    # a few columns of a residual stream are far larger than the others
    by = torch.where(torch.rand(case["cols"], device="cuda", generator=gen) < 0.005, 20.0, 1.0)
    wtype = {"same": dtype, "f32": torch.float32, "none": None}[case["weight"]]
    s["weight"] = None if wtype is None else (1 + 0.2 * torch.randn(case["cols"], device="cuda", generator=gen)).to(wtype)
    if case["op"] == "norm":
        s["ins"] = [normal(shape, dtype, ranks ** -0.5) for _ in range(ranks)]
        s["res"] = normal(shape, dtype, by) if case["residual"] else None
        s["sum"] = torch.empty(shape, dtype=dtype, device="cuda") if case["residual"] else None
        s["rstd"] = torch.empty(case["rows"], dtype=torch.float32, device="cuda")
        s["out"] = torch.empty(shape, dtype=dtype if case["group"] < 0 else torch.float8_e4m3fn, device="cuda")
        groups = 0 if case["group"] < 0 else 1 if case["group"] == 0 else -(-case["cols"] // case["group"])
        s["scales"] = torch.empty((case["rows"], groups), dtype=torch.float32, device="cuda") if groups else None
        return s
    s["x"] = normal(shape, dtype, by)
    s["rstd"] = torch.rsqrt(s["x"].float().square().mean(1) + EPS)
    s["dys"] = [normal(shape, dtype, 0.1) for _ in range(ranks)]
    s["dsum"] = normal(shape, dtype, 0.1) if case["residual"] else None
    s["dx"] = torch.empty(shape, dtype=dtype, device="cuda")
    s["dweight"] = torch.empty(case["cols"], dtype=wtype, device="cuda")
    if own:  # room for the partial sums of the weight's gradient
        import aluminum_amd as al
        s["workspace"] = torch.empty(al.rms_norm_grad_workspace(*shape), dtype=torch.uint8, device="cuda")
    return s


def _sum_of(tensors):
    return sum((t.float() for t in tensors[1:]), tensors[0].float())


def _plain_norm(s):
    x = _sum_of(s["ins"])
    if s["res"] is not None:
        x = x + s["res"].float()
    rstd = torch.rsqrt(x.square().mean(1) + EPS)
    y = x * rstd[:, None]
    if s["weight"] is not None:
        y = y * s["weight"].float()
    got = {"rstd": rstd}
    if s["res"] is not None:
        got["sum"] = x.to(s["sum"].dtype)
    if s["group"] < 0:
        got["out"] = y.to(s["out"].dtype)
        return got
    rows, cols = y.shape
    group = s["group"] or cols
    groups = -(-cols // group)
    y = torch.nn.functional.pad(y, (0, groups * group - cols)).view(rows, groups, group)
    got["scales"] = (y.abs().amax(2) / E4M3_MAX).clamp(min=TINY)
    got["out"] = (y / got["scales"][:, :, None]).view(rows, groups * group)[:, :cols].to(torch.float8_e4m3fn)
    return got


def _plain_grad(s):
    dy, x, rstd = _sum_of(s["dys"]), s["x"].float(), s["rstd"][:, None]
    n = x * rstd
    g = dy * s["weight"].float()
    dx = rstd * (g - n * (g * n).mean(1, keepdim=True))
    if s["dsum"] is not None:
        dx = dx + s["dsum"].float()
    return {"dx": dx.to(s["dx"].dtype), "dweight": (dy * n).sum(0).to(s["dweight"].dtype)}


def _plain_global_norm(s):
    return torch.stack([t.double().square().sum() for t in s["grads"]]).sum().sqrt().float().view(1)


def run(s):
    if own:
        import aluminum_amd as al
        if s["op"] == "norm":
            al.rms_norm(s["out"], s["ins"], weight=s["weight"], residual=s["res"], sum_out=s["sum"], rstd=s["rstd"],
                        scales=s["scales"], group=max(0, s["group"]), eps=EPS)
            got = {"rstd": s["rstd"], "out": s["out"]}
            if s["sum"] is not None:
                got["sum"] = s["sum"]
            if s["scales"] is not None:
                got["scales"] = s["scales"]
            return got
        if s["op"] == "grad":
            al.rms_norm_grad(s["dx"], s["dys"], s["x"], s["rstd"], weight=s["weight"], dsum=s["dsum"], dweight=s["dweight"],
                             workspace=s["workspace"])
            return {"dx": s["dx"], "dweight": s["dweight"]}
        if s["op"] == "norm_of":
            s["list"].global_norm(s["norm"])
            return {"norm": s["norm"]}
        s["list"].clip_global_norm(s["norm"], s["max_norm"], eps=CLIP_EPS)
        return {"norm": s["norm"], "clipped": s["clipped"]}
    if s["op"] == "norm":
        return _plain_norm(s)
    if s["op"] == "grad":
        return _plain_grad(s)
    norm = _plain_global_norm(s)
    if s["op"] == "norm_of":
        return {"norm": norm}
    by = (s["max_norm"] / (norm + CLIP_EPS)).clamp(max=1.0)
    torch._foreach_copy_(s["outs"], [(t.float() * by).to(t.dtype) for t in s["grads"]])
    return {"norm": norm, "clipped": s["clipped"]}


def exact(case, seed):
    s = prepare(case, seed)
    wide = torch.float64
    if case["op"] in ("norm_of", "clip"):
        norm = sum((torch.dot(f.to(wide), f.to(wide)) for f in s["flat"]), torch.zeros((), dtype=wide, device="cuda")) ** 0.5
        got = {"norm": norm.reshape(1)}
        if case["op"] == "clip":
            by = torch.clamp(s["max_norm"] / (norm + CLIP_EPS), max=1.0)
            got["clipped"] = [f.to(wide) * by for f in s["flat"]]
        return got
    cols = case["cols"]
    w = torch.ones(cols, dtype=wide, device="cuda") if s["weight"] is None else s["weight"].to(wide)
    if case["op"] == "grad":
        dy = torch.zeros(s["x"].shape, dtype=wide, device="cuda")
        for t in s["dys"]:
            dy += t
        x, r = s["x"].to(wide), s["rstd"].to(wide).reshape(-1, 1)
        dweight = torch.einsum("rc,rc->c", dy, x * r)
        dot = torch.einsum("rc,rc->r", dy * w, x).reshape(-1, 1)
        dy *= w * r
        dy -= x * (dot * r ** 3 / cols)
        if s["dsum"] is not None:
            dy += s["dsum"]
        return {"dx": dy, "dweight": dweight}
    x = torch.zeros(s["ins"][0].shape, dtype=wide, device="cuda")
    for t in s["ins"] + ([s["res"]] if s["res"] is not None else []):
        x += t
    rstd = (torch.einsum("rc,rc->r", x, x) / cols + EPS) ** -0.5
    got = {"rstd": rstd}
    y = x * rstd.reshape(-1, 1) * w
    if s["res"] is not None:
        got["sum"] = x
    if case["group"] >= 0:
        # the scales as the formula gives them, and in the 8-bit values' place what they are rounded from
        edges = list(range(0, cols, case["group"] or cols)) + [cols]
        parts = [y[:, a:b] for a, b in zip(edges, edges[1:])]
        scales = torch.stack([p.abs().max(1).values for p in parts], 1).div(E4M3_MAX).clamp_min(TINY)
        y = torch.cat([p / scales[:, k:k + 1] for k, p in enumerate(parts)], 1)
        got["scales"] = scales
    got["out"] = y
    return got
