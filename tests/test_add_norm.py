"""add_norm: refusals on the CPU, and on the MI355X against the formulas in 64 bits.

Tolerance, element by element, from u = 2^-24, by carrying each value v with how far it may be off, e. A sum of a
row in FP32 has chains of at most 64 additions in a lane, 6 over the lanes and 16 over the wavefronts: C = 96
roundings. The mean of v is off by mean(e) + C u mean|v|; v less it by that, e and u of the difference. The mean
square is off by mean(2 |v| e + e^2) + C u of itself, its root's inverse by half of that, relative, and 4 u (to first
order: 1.05 of it, as the offs are below 1% of what they add to); the products that follow add u each. The row
gate's sigmoid as in the dense products: its exponential's argument is rounded, 128 u. Last each output's rounding:
half a step of its type, finfo.eps / 2 of the value or half of the smallest subnormal.
"""

import ctypes

import pytest
import torch

from gpu_helpers import announce
from uniserve_moe import abi, ops

U = 2.0**-24
C = 96
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def rounding(y, dtype):
    info = torch.finfo(dtype)
    return torch.maximum(y.abs() * (info.eps / 2), torch.full_like(y, info.tiny * info.eps / 2))


def normed(v, e, norm, weight, bias, offset, eps):
    if norm == "layer":
        shift = e.mean(1, keepdim=True) + C * U * v.abs().mean(1, keepdim=True)
        v = v - v.mean(1, keepdim=True)
        e = e + shift + U * (v.abs() + e + shift)
    square = (v * v).mean(1, keepdim=True)
    off = (2 * v.abs() * e + e * e).mean(1, keepdim=True) + C * U * square
    factor = 1.0 / torch.sqrt(square + eps)
    relative = 1.05 * (0.5 * off / (square + eps) + 4 * U)
    w = offset + weight.double().cpu()
    y = v * factor * w
    e = (factor * w).abs() * e * (1 + relative) + y.abs() * (relative + 4 * U)
    if bias is not None:
        y = y + bias.double().cpu()
        e = e + U * (y.abs() + e)
    return y, e


def reference(x, weight, residual=None, post=None, gate=None, channels=None, scale=1.0, residual_scale=1.0, norm="rms",
              bias=None, post_bias=None, offset=0.0, eps=1e-6):
    """(out, tolerance), (total, tolerance) in 64 bits on the CPU."""
    v = x.double().cpu()
    e = torch.zeros_like(v)
    if post is not None:
        v, e = normed(v, e, norm, post, post_bias, offset, eps)
    factor, relative = torch.full_like(v, scale), U  # (the scales are FP32)
    if channels is not None:
        factor, relative = factor * channels.double().cpu(), relative + U
    if gate is not None:
        factor, relative = factor * torch.special.expit(gate.double().cpu()), relative + 128 * U
    v, e = v * factor, factor.abs() * e * (1 + relative) + (v * factor).abs() * (relative + 2 * U)
    if residual is not None:
        r = residual.double().cpu() * residual_scale
        v = v + r
        e = e + U * (v.abs() + e) + U * r.abs()
    stream = x.dtype if residual is None else residual.dtype
    total = v, e + rounding(v.abs() + e, stream)
    if weight is None:
        return None, total
    y, e = normed(v, e, norm, weight, bias, offset, eps)
    return (y, e + rounding(y.abs() + e, x.dtype)), total


def assert_near(got, want, what=""):
    y, tolerance = want
    off = (got.double().cpu() - y).abs()
    assert got.shape == y.shape and torch.isfinite(got).all(), what
    worst = (off / tolerance).max().item() if off.numel() else 0.0
    assert worst <= 1.0, f"{what}: {worst:.3f} of the tolerance"


def normal(shape, seed, std=1.0, dtype=BF16, mean=0.0, device="cuda"):
    g = torch.Generator(device=device).manual_seed(seed)
    return (torch.randn(shape, generator=g, device=device) * std + mean).to(dtype)


# ---- without a GPU ----------------------------------------------------------------------------------


def filled_call():
    call = abi.AddNormCall()
    call.input, call.residual, call.weight, call.total, call.out = 1 << 20, 2 << 20, 3 << 20, 4 << 20, 5 << 20
    call.rows, call.width = 4, 64
    call.input_row_stride = call.residual_row_stride = call.total_row_stride = call.out_row_stride = 64
    call.dtype = call.total_dtype = call.vector_dtype = abi.DTYPE["bf16"]
    call.eps, call.scale, call.residual_scale = 1e-6, 1.0, 1.0
    return call


REFUSED = [
    ({"rows": -1}, "positive"), ({"width": 0}, "positive"), ({"width": 32769}, "32768"),
    ({"dtype": abi.DTYPE["i32"]}, "bf16, f16 or f32"), ({"total_dtype": abi.DTYPE["f16"]}, "residual and total"),
    ({"vector_dtype": abi.DTYPE["f16"]}, "vectors"), ({"norm": 2}, "rms or layer"),
    ({"bias": 9 << 20}, "no bias"), ({"post_bias": 9 << 20, "norm": 1}, "comes with post"),
    ({"weight": None}, "together"), ({"out": None}, "together"), ({"weight": None, "out": None, "bias": 9 << 20, "norm": 1}, "together"),
    ({"eps": -1.0}, "eps"), ({"eps": float("nan")}, "eps"),
    ({"input": None}, "needs"), ({"weight": None, "out": None, "total": None}, "needs"),
    ({"input_row_stride": 63}, "strides"), ({"residual_row_stride": 63}, "strides"), ({"total_row_stride": 63}, "strides"),
    ({"out_row_stride": 0}, "strides"), ({"gate": 9 << 20, "gate_stride": -1}, "gate stride"),
    ({"out_row_stride": 1 << 60}, "too large"), ({"gate": 9 << 20, "gate_stride": 1 << 60}, "too large"),
    # Outputs over an input in part, over a vector, over the gate and over each other.
    ({"out": (1 << 20) + 2}, "in part"), ({"total": (2 << 20) + 128}, "in part"), ({"total": (1 << 20) - 8}, "in part"),
    ({"total": 2 << 20, "total_row_stride": 72}, "in part"), ({"out": 3 << 20}, "vectors"), ({"out": (3 << 20) + 126}, "vectors"),
    ({"channels": (4 << 20) + 2}, "vectors"), ({"gate": (5 << 20) + 4, "gate_stride": 1}, "gate"),
    ({"gate": (4 << 20), "gate_stride": 0}, "gate"),
    ({"out": 4 << 20}, "outputs overlap"), ({"out": (4 << 20) + 500}, "outputs overlap"),
    ({"out": 2 << 20, "total": 2 << 20}, "outputs overlap"),
    ({"out": 2 << 20, "total_dtype": abi.DTYPE["f32"]}, "in part"), ({"total": 1 << 20, "total_dtype": abi.DTYPE["f32"]}, "in part"),
]


@pytest.mark.parametrize("fields, says", REFUSED)
def test_refusals(fields, says):
    call = filled_call()
    for name, value in fields.items():
        setattr(call, name, value)
    assert abi.library().uniserve_add_norm(ctypes.byref(call), None) != 0
    assert says in call.error.decode()


@pytest.mark.parametrize("fields", [
    {"rows": 1, "input_row_stride": 1 << 60}, {"rows": 1, "total_row_stride": -1}, {"rows": 1, "gate": 9 << 20, "gate_stride": -1},
    {"residual": None, "residual_row_stride": -1}, {"gate_stride": -1}, {"gate_stride": 1 << 60},
])
def test_unused_strides_are_not_read(fields):
    """The call comes to the last check, which refuses it (the outputs share their rows)."""
    call = filled_call()
    for name, value in {**fields, "out": 4 << 20}.items():
        setattr(call, name, value)
    assert abi.library().uniserve_add_norm(ctypes.byref(call), None) != 0
    assert "outputs overlap" in call.error.decode()


def test_no_rows_launch_nothing():
    call = filled_call()
    call.rows, call.input, call.out, call.weight = 0, None, None, None
    assert abi.library().uniserve_add_norm(ctypes.byref(call), None) == 0
    assert abi.library().uniserve_add_norm(None, None) != 0


def test_python_refusals():
    with pytest.raises(ValueError, match="on a GPU"):
        ops.add_norm(torch.zeros(2, 8), torch.zeros(8))


# ---- on the MI355X ----------------------------------------------------------------------------------

#: One element to the longest row, with both ends of every shape's widths; rows beyond them by tens and thousands.
WIDTHS = [1, 7, 8, 9, 64, 100, 511, 512, 513, 1000, 1024, 1031, 2048, 2056, 4095, 4096, 4104, 8192, 8200, 16384, 16392, 32760, 32767]


def inputs(rows, width, dtype, stream=None, vector=None, seed=0):
    vector = vector or dtype
    return dict(x=normal((rows, width), seed + 1, dtype=dtype), weight=normal((width,), seed + 2, 0.3, vector, 1.0),
                residual=normal((rows, width), seed + 3, 2.0, stream or dtype), post=normal((width,), seed + 4, 0.3, vector, 1.0),
                gate=normal((rows, 1), seed + 5, 2.0, dtype), channels=normal((width,), seed + 6, 0.5, vector),
                bias=normal((width,), seed + 7, 0.5, vector), post_bias=normal((width,), seed + 8, 0.5, vector))


@pytest.mark.gpu
@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_join_and_norm(device, width, dtype):
    for rows in (1, 5):
        announce("add_norm", rows, width, dtype)
        made = inputs(rows, width, dtype)
        call = {k: made[k] for k in ("x", "weight", "residual")}
        out, total = ops.add_norm(**call)
        want, want_total = reference(**call)
        assert out.dtype == total.dtype == dtype
        assert_near(total, want_total, "total")
        assert_near(out, want, "out")


@pytest.mark.gpu
@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("norm", ["rms", "layer"])
@pytest.mark.parametrize("dtype, stream, vector", [(BF16, F32, BF16), (F16, F16, F32), (F32, F32, F32), (F16, F32, F16), (BF16, BF16, F32)])
def test_everything(device, width, norm, dtype, stream, vector):
    announce("add_norm with everything", width, norm, dtype, stream, vector)
    call = inputs(3, width, dtype, stream, vector, seed=width)
    call.update(norm=norm, scale=0.25, residual_scale=1.5, offset=1.0, eps=1e-5)
    if norm == "rms":
        call.pop("bias"), call.pop("post_bias")
    out, total = ops.add_norm(**call)
    want, want_total = reference(**call)
    assert out.dtype == dtype and total.dtype == stream
    assert_near(total, want_total, "total")
    assert_near(out, want, "out")


@pytest.mark.gpu
@pytest.mark.parametrize("rows, width", [(1024, 64), (1500, 257), (1100, 520), (1031, 1024), (1024, 1500), (1027, 2048), (1100, 3001),
                                         (1025, 4096), (2000, 4104), (5000, 100)])
@pytest.mark.parametrize("dtype, norm", [(BF16, "rms"), (F16, "layer")])
def test_many_rows(device, rows, width, dtype, norm):
    announce("add_norm rows", rows, width, dtype, norm)
    call = inputs(rows, width, dtype, seed=7)
    if norm == "rms":
        call.pop("bias"), call.pop("post_bias")
    out, total = ops.add_norm(**call, norm=norm)
    want, want_total = reference(**call, norm=norm)
    assert_near(total, want_total, "total")
    assert_near(out, want, "out")


@pytest.mark.gpu
@pytest.mark.parametrize("parts", [(), ("residual",), ("post",), ("gate",), ("channels",), ("residual", "post"), ("gate", "post"),
                                   ("residual", "channels")])
@pytest.mark.parametrize("rows, width", [(3, 520), (1100, 72)])
def test_each_part_alone(device, parts, rows, width):
    announce("add_norm parts", parts, rows, width)
    made = inputs(rows, width, BF16, seed=3)
    call = {k: made[k] for k in ("x", "weight") + parts}
    out, total = ops.add_norm(**call)
    want, want_total = reference(**call)
    assert_near(out, want, "out")
    if parts:
        assert_near(total, want_total, "total")
    else:
        assert total is call["x"]
        given = torch.empty_like(total)
        assert ops.add_norm(**call, total=given)[1] is given and torch.equal(given, total)
    call["weight"] = None  # the join alone
    out, joined = ops.add_norm(**call, total=torch.empty_like(total))
    assert out is None and torch.equal(joined, total)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [6, 1100])
@pytest.mark.parametrize("shift", [0, 1, 8])
@pytest.mark.parametrize("width", [8, 75, 512, 1003])
def test_strides_and_alignments(device, rows, width, shift):
    """Column slices of wider buffers; what lies beside the outputs stays as it was, what lies beside the inputs
    (NaN) is not read into a sum."""
    announce("add_norm strides", rows, width, shift)
    made = inputs(rows, width, F16, seed=5)

    def inside(source, fill=float("nan")):
        buffer = torch.full((source.shape[0] + 2, width + 24), fill, dtype=source.dtype, device=device)
        return buffer, buffer[1:-1, shift:shift + width].copy_(source)

    call = dict(x=inside(made["x"])[1], residual=inside(made["residual"])[1], weight=inside(made["weight"][None])[1][0],
                post=inside(made["post"][None])[1][0], gate=normal((rows, 5), 9, dtype=F16)[:, 2:3])
    (around_out, out), (around_total, total) = inside(made["x"], 7.0), inside(made["x"], 7.0)
    ops.add_norm(**call, out=out, total=total)
    want, want_total = reference(**call)
    assert_near(out, want, "out")
    assert_near(total, want_total, "total")
    for around, inner in ((around_out, out), (around_total, total)):
        inner.fill_(7.0)
        assert (around == 7.0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("rows, width", [(2, 2048), (1200, 1000), (1, 20000)])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_in_place(device, rows, width, dtype):
    announce("add_norm in place", rows, width, dtype)
    made = inputs(rows, width, dtype, seed=11)
    call = {k: made[k] for k in ("x", "weight", "residual", "post")}
    out, total = ops.add_norm(**call)
    for out_over, total_over in (("x", "residual"), ("residual", "x")):
        again = dict(call, x=call["x"].clone(), residual=call["residual"].clone())
        got, got_total = ops.add_norm(**again, out=again[out_over], total=again[total_over])
        assert torch.equal(got, out) and torch.equal(got_total, total)
        assert got is again[out_over] and got_total is again[total_over]


@pytest.mark.gpu
def test_gates_of_fp32_rows(device):
    """sigmoid(g) = 1 / (1 + e) with e = exp(-g) off by 2 u (an ulp), the sum, the quotient and the product by u each, and
    the scales' one: 6 u, to first order; 8 are granted."""
    announce("add_norm f32 gates")
    rows, width = 481, 72
    x, gate = normal((rows, width), 1, dtype=F32), torch.linspace(-80.0, 40.0, rows, device=device)[:, None]
    _, total = ops.add_norm(x, None, gate=gate)
    want = x.double().cpu() * torch.special.expit(gate.double().cpu())
    assert ((total.double().cpu() - want).abs() <= 8 * U * want.abs()).all()
    x, gate = x.to(BF16), gate.to(BF16)
    _, total = ops.add_norm(x, None, gate=gate, total=torch.empty((rows, width), dtype=F32, device=device))
    want = x.double().cpu() * torch.special.expit(gate.double().cpu())
    assert ((total.double().cpu() - want).abs() <= 8 * U * want.abs()).all(), "f32 total of bf16 rows"
    x = x.float()
    ends = torch.tensor([float("-inf"), -1000.0, float("inf"), 1000.0, float("nan")], device=device)[:, None]
    _, total = ops.add_norm(x[:5].contiguous(), None, gate=ends)
    assert (total[:2] == 0).all() and torch.equal(total[2:4], x[2:4]) and torch.isnan(total[4]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("norm", ["rms", "layer"])
@pytest.mark.parametrize("rows", [1, 33])
def test_in_place_with_nothing_to_join(device, rows, norm):
    """The total is the rows before their norm, also where the norm overwrites them."""
    announce("add_norm in place alone", rows, norm)
    made = inputs(rows, 264, BF16, seed=3)
    x, weight = made["x"], made["weight"]
    before = x.clone()
    want, unjoined = ops.add_norm(x, weight, norm=norm)
    assert unjoined is x and torch.equal(x, before)
    out, total = ops.add_norm(x, weight, norm=norm, out=x)
    assert out is x and torch.equal(out, want) and torch.equal(total, before)


@pytest.mark.gpu
def test_rows_past_4_gib(device):
    announce("add_norm far rows")
    rows, width = 5, 264
    stride = (5 << 30) // 2 // rows // 8 * 8 + 8

    def spread(source):
        far = torch.empty(rows * stride, dtype=BF16, device=device).as_strided((rows, width), (stride, 1))
        return far.copy_(source)

    made = inputs(rows, width, BF16)
    call = {k: made[k] for k in ("x", "weight", "residual")}
    want, want_total = reference(**call)
    out, total = ops.add_norm(spread(call["x"]), call["weight"], residual=call["residual"], out=spread(call["x"]))
    assert_near(out, want, "far input and output")
    residual = spread(call["residual"])
    out, total = ops.add_norm(call["x"], call["weight"], residual=residual, total=residual)
    assert_near(out, want, "far residual")
    assert_near(total, want_total, "far total")


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [4, 1030])
def test_more_rows_than_workgroups_and_wavefronts_share(device, rows):
    """A narrow row each: the last workgroup's rows and the first's are apart."""
    announce("add_norm narrow rows", rows)
    made = inputs(rows, 16, BF16)
    call = {k: made[k] for k in ("x", "weight", "residual", "gate")}
    out, total = ops.add_norm(**call)
    want, want_total = reference(**call)
    assert_near(out, want)
    assert_near(total, want_total)


@pytest.mark.gpu
@pytest.mark.parametrize("width, rows", [(16, (1 << 20) + 300), (8, (1 << 22) + 9)])
def test_rows_past_the_grid(device, width, rows):
    """More rows than the largest grid's workgroups take at once."""
    announce("add_norm grid", rows, width)
    x, weight = normal((rows, width), 1), normal((width,), 2, 0.3, mean=1.0)
    out, _ = ops.add_norm(x, weight)
    for first in (0, (1 << 20) - 100, rows - 250):
        part = x[first:first + 250]
        assert_near(out[first:first + 250], reference(part, weight)[0], f"from {first}")


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [7, 1100])
@pytest.mark.parametrize("norm", ["rms", "layer"])
def test_infinities_and_nans_stay_in_their_rows(device, rows, norm):
    announce("add_norm non-finite", rows, norm)
    made = inputs(rows, 200, BF16)
    call = {k: made[k] for k in ("x", "weight", "residual", "post")}
    out, total = (t.clone() for t in ops.add_norm(**call, norm=norm))
    call["x"][2, 7] = float("nan")
    call["residual"][4, 100] = float("inf")
    got, got_total = ops.add_norm(**call, norm=norm)
    kept = [r for r in range(rows) if r not in (2, 4)]
    assert torch.equal(got[kept], out[kept]) and torch.equal(got_total[kept], total[kept])
    assert torch.isnan(got[2]).all() and torch.isnan(got[4, 100]) and torch.isinf(got_total[4, 100])
    assert torch.equal(got_total[4, :100], total[4, :100])


@pytest.mark.gpu
@pytest.mark.parametrize("norm", ["rms", "layer"])
def test_constant_and_zero_rows(device, norm):
    """Rows without spread: eps keeps them finite (zeros; a layer norm of a constant row gives its bias)."""
    announce("add_norm constant rows", norm)
    x = torch.zeros((4, 512), dtype=F32, device=device)
    x[1:] = 3.0
    weight = normal((512,), 1, dtype=F32, mean=1.0)
    bias = normal((512,), 2, dtype=F32) if norm == "layer" else None
    out, _ = ops.add_norm(x, weight, norm=norm, bias=bias)
    if norm == "layer":
        assert torch.equal(out, bias.expand(4, 512))
    else:
        assert (out[0] == 0).all()
        assert_near(out, reference(x, weight)[0])


@pytest.mark.gpu
@pytest.mark.parametrize("norm", ["rms", "layer"])
def test_large_means(device, norm):
    """A row far from zero: its spread is not the difference of two large sums."""
    announce("add_norm large means", norm)
    x = normal((3, 1000), 1, dtype=F32, mean=1000.0)
    weight = normal((1000,), 2, 0.3, F32, 1.0)
    assert_near(ops.add_norm(x, weight, norm=norm)[0], reference(x, weight, norm=norm)[0])


@pytest.mark.gpu
def test_shared_gate_and_streams(device):
    announce("add_norm streams")
    made = [inputs(rows, 768, BF16, seed=rows) for rows in (3, 1200)]
    calls = [{k: m[k] for k in ("x", "weight", "residual", "post")} for m in made]
    calls[0]["gate"] = normal((1, 1), 4).expand(3, 1)
    want = [ops.add_norm(**c) for c in calls]
    assert_near(want[0][0], reference(**calls[0])[0])
    torch.cuda.synchronize()
    sides, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for _ in range(4):
        for i, side in enumerate(sides):
            with torch.cuda.stream(side):
                got[i].append(ops.add_norm(**calls[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(a, b) for pair in got[i] for a, b in zip(pair, want[i]))


@pytest.mark.gpu
def test_captured_replays(device):
    announce("add_norm graph")
    made = inputs(40, 1000, BF16)
    call = {k: made[k] for k in ("x", "weight", "residual", "post")}

    def step():
        out, total = ops.add_norm(**call)
        return ops.add_norm(out, call["weight"], residual=total, gate=made["gate"])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        step()
        side.synchronize()
        with torch.cuda.graph(graph, stream=side):
            captured = step()
    torch.cuda.current_stream().wait_stream(side)
    for seed in (10, 11, 12):
        call["x"].copy_(normal((40, 1000), seed))
        graph.replay()
        torch.cuda.synchronize()
        replayed = [t.clone() for t in captured]
        assert all(torch.equal(a, b) for a, b in zip(step(), replayed))
        torch.cuda.synchronize()


@pytest.mark.gpu
def test_no_rows(device):
    out, total = ops.add_norm(torch.empty((0, 64), dtype=BF16, device=device), normal((64,), 1),
                              residual=torch.empty((0, 64), dtype=F32, device=device))
    assert out.shape == total.shape == (0, 64) and total.dtype == F32


@pytest.mark.gpu
@pytest.mark.parametrize("arguments, says", [
    (dict(norm="batch"), "norm"), (dict(weight="short"), "weight"), (dict(weight="half"), "vectors"), (dict(post="wide"), "vectors"),
    (dict(residual="half"), "residual"), (dict(residual="short"), "residual"), (dict(gate="wide"), "gate"), (dict(gate="flat"), "gate"),
    (dict(total="wide"), "total"), (dict(out="wide"), "output"), (dict(out="columns"), "output"), (dict(bias="row"), "bias"),
    (dict(weight=None, out="row"), "no out"), (dict(eps=-1.0), "eps"), (dict(post_bias="row", norm="layer"), "post_bias"),
    (dict(residual="host"), "residual"), (dict(channels="strided"), "channels"),
])
def test_python_refusals_of_device_calls(device, arguments, says):
    made = {
        "weight.short": lambda: normal((15,), 1), "weight.half": lambda: normal((16,), 1, dtype=F16),
        "post.wide": lambda: normal((16,), 1, dtype=F32), "residual.half": lambda: normal((4, 16), 1, dtype=F16),
        "residual.short": lambda: normal((3, 16), 1), "gate.wide": lambda: normal((4, 1), 1, dtype=F32),
        "gate.flat": lambda: normal((4,), 1), "total.wide": lambda: normal((4, 16), 1, dtype=F32),
        "out.wide": lambda: normal((4, 16), 1, dtype=F32), "out.columns": lambda: normal((16, 4), 1).t(),
        "bias.row": lambda: normal((16,), 1), "post_bias.row": lambda: normal((16,), 1), "out.row": lambda: normal((4, 16), 1),
        "residual.host": lambda: torch.zeros((4, 16), dtype=BF16), "channels.strided": lambda: normal((32,), 1)[::2],
    }
    call = dict(x=normal((4, 16), 1), weight=normal((16,), 2), residual=normal((4, 16), 3))
    call.update({k: made[f"{k}.{v}"]() if f"{k}.{v}" in made else v for k, v in arguments.items()})
    with pytest.raises((ValueError, RuntimeError), match=says):
        ops.add_norm(**call)
