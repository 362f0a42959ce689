"""linear and gated_linear: refusals on the CPU, and on the MI355X against the formulas in 64 bits.

Tolerance, element by element. With u = 2^-24 and S = sum |x w| (+ |bias|) of an output, a sum of K
exact products in FP32, in any order and with chopped or rounded additions, is off by at most
2 (K + 1) u S. The activation (steepest slope 1.13) passes that on and adds its own error: its
exponential's argument is rounded, which moves the result by |z| u relative, z < 104 wherever the
result is not zero, plus a few u: 128 u of its value. The row gate's sigmoid likewise, and the
residual's addition u of the larger operand. Last the output's rounding: half a step of its type,
finfo.eps / 2 of the value or half of the smallest subnormal.
"""

import ctypes

import numpy as np
import pytest
import torch

from gpu_helpers import announce, kernels_of
from uniserve_moe import abi, ops

U = 2.0**-24
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def activated(y, activation):
    if activation == "silu":
        return y * torch.special.expit(y)
    if activation == "gelu_tanh":
        return 0.5 * y * (1.0 + torch.tanh((2.0 / torch.pi) ** 0.5 * (y + 0.044715 * y**3)))
    return y


def rounding(y, dtype):
    info = torch.finfo(dtype)
    return torch.maximum(y.abs() * (info.eps / 2), torch.full_like(y, info.tiny * info.eps / 2))


def reference(x, w, bias=None, activation=None, gate=None, residual=None, out_dtype=None, gated=False):
    """The output in 64 bits and how far the kernel may be from it, both on the CPU."""
    out_dtype = out_dtype or x.dtype
    x, w = x.double().cpu(), w.double().cpu()
    y, s = x @ w.t(), x.abs() @ w.abs().t()
    if bias is not None:
        y, s = y + bias.double().cpu(), s + bias.double().cpu().abs()
    off = 2 * (x.shape[1] + 1) * U * s
    slope = 1.13
    if gated:
        n = w.shape[0] // 2
        up, g = y[:, :n], y[:, n:]
        act = activated(g, activation)
        off = act.abs() * off[:, :n] + slope * off[:, n:] * (up.abs() + off[:, :n])
        y = up * act
        off = off + 128 * U * y.abs()
    else:
        y = activated(y, activation)
        off = (off * slope if activation else off) + (128 * U * y.abs() if activation else 0.0)
    if gate is not None:
        factor = torch.special.expit(gate.double().cpu())
        off, y = off * factor + 128 * U * (y * factor).abs(), y * factor
    if residual is not None:
        r = residual.double().cpu()
        off, y = off + U * (y.abs() + r.abs()), y + r
    return y, off + U * off + rounding(y.abs() + off, out_dtype)


def assert_near(got, want, what=""):
    y, tolerance = want
    off = (got.double().cpu() - y).abs()
    assert got.shape == y.shape and torch.isfinite(got).all(), what
    worst = (off / tolerance).max().item() if off.numel() else 0.0
    assert worst <= 1.0, f"{what}: {worst:.3f} of the tolerance"


def normal(shape, seed, std=1.0, dtype=BF16, device="cuda"):
    g = torch.Generator(device=device).manual_seed(seed)
    return (torch.randn(shape, generator=g, device=device) * std).to(dtype)


# ---- without a GPU ----------------------------------------------------------------------------------


def filled_call(gated=False):
    call = abi.LinearCall()
    call.input, call.weight, call.out = 1 << 20, 2 << 20, 3 << 20
    call.m, call.n, call.k = 4, 32, 64
    call.input_row_stride, call.weight_row_stride, call.out_row_stride = 64, 64, 32
    call.dtype = call.bias_dtype = call.out_dtype = abi.DTYPE["bf16"]
    call.activation = abi.ACTIVATION["silu"] if gated else -1
    return call


REFUSED = [
    ({"m": -1}, "positive"), ({"n": 0}, "positive"), ({"k": 0}, "positive"),
    ({"input": None}, "needs"), ({"weight": None}, "needs"), ({"out": None}, "needs"),
    ({"dtype": abi.DTYPE["f32"]}, "bf16 or f16"), ({"out_dtype": abi.DTYPE["f16"]}, "inputs' type"),
    ({"bias": 8 << 20, "bias_dtype": abi.DTYPE["f16"]}, "bias"), ({"activation": 2}, "gelu_tanh"),
    ({"input_row_stride": 63}, "strides"), ({"weight_row_stride": 63}, "strides"), ({"out_row_stride": 31}, "strides"),
    ({"k": 1 << 31, "input_row_stride": 1 << 31, "weight_row_stride": 1 << 31}, "int32"),
    ({"input_row_stride": 1 << 60}, "too large"), ({"weight_row_stride": 1 << 60}, "too large"),
    # Outputs over an input: whole, in part, from below, and rows that meet within a shared buffer.
    ({"out": 1 << 20}, "overlaps"), ({"out": (1 << 20) + 130}, "overlaps"), ({"out": (1 << 20) - 254}, "overlaps"),
    ({"out": 2 << 20}, "overlaps"), ({"out": (2 << 20) + 4094}, "overlaps"),
    ({"bias": (3 << 20) + 2}, "overlaps"),
    ({"out": (1 << 20) + 126, "out_row_stride": 96, "input_row_stride": 96}, "overlaps"),
    ({"out": (1 << 20) + 130, "out_row_stride": 96, "input_row_stride": 96}, "overlaps"),
]


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("fields, says", REFUSED)
def test_refusals(gated, fields, says):
    call = filled_call(gated)
    for name, value in fields.items():
        setattr(call, name, value)
    entry = abi.library().uniserve_gated_linear if gated else abi.library().uniserve_linear
    assert entry(ctypes.byref(call), None) != 0
    assert says in call.error.decode()


@pytest.mark.parametrize("fields, says", [
    ({"gate": 8 << 20, "gate_stride": -1}, "gate stride"),
    ({"gate": (3 << 20) + 2, "gate_stride": 1}, "overlaps"),
    ({"residual": 8 << 20, "residual_row_stride": 31}, "strides"),
    ({"residual": (3 << 20) + 2, "residual_row_stride": 32}, "residual"),
    ({"residual": 3 << 20, "residual_row_stride": 40}, "residual"),
])
def test_linear_refusals(fields, says):
    call = filled_call()
    for name, value in fields.items():
        setattr(call, name, value)
    assert abi.library().uniserve_linear(ctypes.byref(call), None) != 0
    assert says in call.error.decode()


@pytest.mark.parametrize("fields, says", [
    ({"activation": -1}, "silu or gelu_tanh"), ({"out_dtype": abi.DTYPE["f32"]}, "inputs' type"),
    ({"gate": 8 << 20}, "no row gate"), ({"residual": 8 << 20}, "no residual"),
])
def test_gated_linear_refusals(fields, says):
    call = filled_call(gated=True)
    for name, value in fields.items():
        setattr(call, name, value)
    assert abi.library().uniserve_gated_linear(ctypes.byref(call), None) != 0
    assert says in call.error.decode()


#: Strides of arrays that a call does not have, and of single rows.
UNUSED = [
    {"residual_row_stride": 1 << 60}, {"residual_row_stride": -5}, {"gate_stride": 1 << 60}, {"gate_stride": -5},
    {"m": 1, "input_row_stride": 1 << 60}, {"m": 1, "input_row_stride": 0}, {"m": 1, "out_row_stride": 1 << 60},
    {"m": 1, "out_row_stride": -1}, {"m": 1, "residual": 8 << 20, "residual_row_stride": 1 << 60},
    {"m": 1, "gate": 9 << 20, "gate_stride": 1 << 60}, {"n": 1, "weight_row_stride": 1 << 60},
]


@pytest.mark.parametrize("gated, fields", [(False, fields) for fields in UNUSED] +
                         [(True, fields) for fields in UNUSED if not {"n", "gate", "residual"} & set(fields)])
def test_unused_strides_are_not_read(gated, fields):
    """An absent array and a single row have no stride: the call comes to the check after the strides' (the output
    is the input here)."""
    call = filled_call(gated)
    for name, value in {**fields, "out": 1 << 20}.items():
        setattr(call, name, value)
    entry = abi.library().uniserve_gated_linear if gated else abi.library().uniserve_linear
    assert entry(ctypes.byref(call), None) != 0
    assert "overlaps one of its inputs" in call.error.decode()


@pytest.mark.parametrize("gated, m, n", [(False, 64, (1 << 30) - 1), (False, 1 << 16, 1 << 20), (True, 64, 1 << 29), (True, 1 << 16, 1 << 19)])
def test_refusals_of_more_tiles_than_a_launch_holds(gated, m, n):
    call = filled_call(gated)
    call.m, call.n, call.out_row_stride, call.out, call.weight = m, n, n, 1 << 40, 1 << 50
    entry = abi.library().uniserve_gated_linear if gated else abi.library().uniserve_linear
    assert entry(ctypes.byref(call), None) != 0
    assert "too many tiles" in call.error.decode()


def test_no_rows_launch_nothing():
    call = filled_call()
    call.m, call.input, call.out = 0, None, None
    assert abi.library().uniserve_linear(ctypes.byref(call), None) == 0
    assert abi.library().uniserve_linear(None, None) != 0


def test_python_refusals():
    with pytest.raises(ValueError, match="on a GPU"):
        ops.linear(torch.zeros(2, 8, dtype=BF16), torch.zeros(4, 8, dtype=BF16))
    with pytest.raises(ValueError, match="up rows"):
        ops.gated_linear(torch.zeros(2, 8, dtype=BF16), torch.zeros(5, 8, dtype=BF16))


# ---- on the MI355X ----------------------------------------------------------------------------------

#: m, n, k: one row to several tiles, odd extents, single columns and elements, whole tiles.
SHAPES = [(1, 1, 1), (1, 2048, 1408), (1, 5, 4096), (2, 16, 8), (3, 1000, 72), (5, 33, 1000), (7, 64, 8192), (16, 256, 128),
          (17, 130, 264), (31, 96, 96), (33, 512, 520), (48, 2048, 64), (64, 128, 2048), (65, 65, 65), (100, 1, 2048),
          (129, 257, 384), (200, 704, 1024), (256, 256, 256), (257, 384, 1984), (300, 1001, 1000), (512, 1408, 192),
          (1000, 300, 128), (1025, 640, 640), (2048, 264, 2048)]


@pytest.mark.gpu
@pytest.mark.parametrize("m, n, k", SHAPES)
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_linear_plain(device, m, n, k, dtype):
    announce("linear", m, n, k, dtype)
    x, w = normal((m, k), m + k, dtype=dtype), normal((n, k), n + k + 1, 0.05, dtype)
    assert_near(ops.linear(x, w), reference(x, w))
    assert_near(ops.linear(x, w, out_dtype=F32), reference(x, w, out_dtype=F32), "f32")


@pytest.mark.gpu
@pytest.mark.parametrize("m, n, k", SHAPES)
@pytest.mark.parametrize("dtype, activation", [(BF16, "silu"), (F16, "gelu_tanh")])
def test_linear_with_everything(device, m, n, k, dtype, activation):
    announce("linear epilogue", m, n, k, dtype)
    x, w = normal((m, k), m + k, dtype=dtype), normal((n, k), n + k + 1, 0.05, dtype)
    gate, residual = normal((m, 1), 3, 2.0, dtype), normal((m, n), 4, 1.0, dtype)
    bias = normal((n,), 5, 0.5, F32 if n % 2 else dtype)
    got = ops.linear(x, w, bias=bias, activation=activation, gate=gate, residual=residual)
    assert_near(got, reference(x, w, bias, activation, gate, residual))
    wide = residual.float()
    out = ops.linear(x, w, bias=bias, activation=activation, gate=gate, residual=wide, out=wide)  # in place, f32
    assert out is wide
    assert_near(out, reference(x, w, bias, activation, gate, residual.float(), out_dtype=F32), "f32 in place")


@pytest.mark.gpu
@pytest.mark.parametrize("m, n, k", SHAPES)
@pytest.mark.parametrize("dtype, activation", [(BF16, "gelu_tanh"), (F16, "silu")])
def test_gated_linear(device, m, n, k, dtype, activation):
    announce("gated_linear", m, n, k, dtype)
    x, w = normal((m, k), m + k, dtype=dtype), normal((2 * n, k), n + k + 1, 0.05, dtype)
    assert_near(ops.gated_linear(x, w, activation=activation), reference(x, w, None, activation, gated=True))
    bias = normal((2 * n,), 5, 0.5, dtype if n % 2 else F32)
    assert_near(ops.gated_linear(x, w, bias=bias, activation=activation), reference(x, w, bias, activation, gated=True), "bias")


#: Calls that the choice gives to each kernel: tokens and weight rows of a tile, wavefronts over them, stages
#: of the ring, teams. K ends inside a stage, short of the ring, and leaves teams without a stage.
KERNELS = [
    (False, "256,256,2,4,2,1", 4000, 4088, 136), (True, "256,256,2,4,2,1", 700, 8200, 136),
    (False, "192,256,2,4,2,1", 1025, 8200, 72), (True, "192,256,2,4,2,1", 400, 8200, 72),
    (False, "128,256,2,4,3,1", 700, 8200, 72), (True, "128,256,2,4,3,1", 257, 8200, 72),
    (False, "192,128,4,2,3,1", 400, 8200, 72), (True, "192,128,4,2,3,1", 130, 8200, 136),
    (False, "128,128,2,2,2,1", 1400, 8200, 72), (True, "128,128,2,2,2,1", 1025, 8200, 72),
    (False, "128,128,2,4,3,1", 513, 4104, 72), (True, "128,128,2,4,3,1", 200, 4104, 72),
    (False, "96,128,2,2,4,1", 200, 8200, 520), (True, "96,128,2,2,4,1", 1025, 1000, 520),
    (False, "128,64,4,2,4,1", 200, 4104, 72), (True, "128,64,4,2,4,1", 100, 4104, 72),
    (False, "64,64,2,2,4,1", 100, 4104, 72), (True, "64,64,2,2,4,1", 5, 8200, 200),
    (False, "48,64,1,2,4,2", 33, 8200, 520), (True, "48,64,1,2,4,2", 33, 4104, 520),
    (False, "32,64,1,1,3,4", 5, 8200, 200), (True, "32,64,1,1,3,4", 5, 4104, 136),
    (False, "32,32,1,1,4,4", 17, 4104, 72), (True, "32,32,1,1,4,4", 65, 1000, 72),
    (False, "16,32,1,1,4,4", 17, 2056, 72), (True, "16,32,1,1,4,4", 5, 40, 136), (True, "16,32,1,1,4,4", 40, 136, 2056),
    (False, "16,16,1,1,4,4", 40, 136, 8), (False, "16,16,1,1,4,4", 17, 130, 1032), (False, "16,16,1,1,4,4", 5, 17, 2056),
]


@pytest.mark.gpu
@pytest.mark.parametrize("gated, shape, m, n, k", KERNELS)
def test_each_tile_kernel(device, gated, shape, m, n, k):
    announce("linear kernel", shape, gated, m, n, k)
    x, w, out = normal((m, k), 1), normal((n * (2 if gated else 1), k), 2, 0.05), normal((m, n), 3)
    gate, residual = normal((m, 1), 4), normal((m, n), 5)

    def call():
        if gated:
            return ops.gated_linear(x, w, out=out)
        return ops.linear(x, w, gate=gate, residual=residual, out=out)

    mangled = "TileShapeI" + "".join(f"Li{d}E" for d in shape.split(","))
    names = kernels_of(call)
    assert len(names) == 1 and mangled in names[0], names
    call()
    assert_near(out, reference(x, w, None, "silu", gated=True) if gated else reference(x, w, gate=gate, residual=residual))


@pytest.mark.gpu
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("m", [1, 2])
@pytest.mark.parametrize("k", [1, 7, 8, 505, 511, 512, 513, 1023, 1024, 1032, 1536, 1541, 2047, 2048, 2049, 3584, 4096, 4600])
def test_one_and_two_tokens(device, gated, m, k):
    """Every number of whole and partial chunks behind the walk's full steps."""
    announce("linear few tokens", gated, m, k)
    x, w, bias = normal((m, k), 1), normal((2 * 19, k), 2, 0.05), normal((38,), 3)
    if gated:
        call, want = (lambda: ops.gated_linear(x, w, bias=bias)), reference(x, w, bias, "silu", gated=True)
    else:
        call, want = (lambda: ops.linear(x, w, bias=bias)), reference(x, w, bias)
    names = kernels_of(call)
    assert len(names) == 1 and "few_tokens_kernel" in names[0], names
    assert_near(call(), want)


@pytest.mark.gpu
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("shape, m, n, k", [
    ("128,128,2,4,2,1", 1100, 3001, 507), ("128,128,2,4,2,1", 700, 5001, 507),
    ("96,128,2,2,2,1", 1100, 5001, 123), ("96,128,2,2,2,1", 2000, 3001, 123),
    ("64,64,2,2,2,1", 65, 5001, 5), ("64,64,2,2,2,1", 130, 3001, 5),
    ("32,32,1,1,2,4", 17, 5001, 2047), ("32,32,1,1,2,4", 130, 1001, 2047),
    ("16,32,1,1,2,4", 40, 300, 1181), ("16,32,1,1,2,4", 8, 40, 2047),
])
def test_each_kernel_for_unaligned_rows(device, gated, shape, m, n, k):
    announce("linear unaligned kernel", shape, gated, m, n, k)
    x, w, out = normal((m, k), 1), normal((n * (2 if gated else 1), k), 2, 0.05), normal((m, n), 3)

    def call():
        return ops.gated_linear(x, w, out=out) if gated else ops.linear(x, w, out=out)

    mangled = "TileShapeI" + "".join(f"Li{d}E" for d in shape.split(","))
    names = kernels_of(call)
    assert len(names) == 1 and mangled in names[0], names
    call()
    assert_near(out, reference(x, w, None, "silu", gated=True) if gated else reference(x, w))


@pytest.mark.gpu
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("k", [1, 2, 3, 5, 7, 9, 15, 17, 31, 57, 63, 65, 127, 129, 191, 255, 257, 511, 515])
def test_every_remainder_of_unaligned_rows(device, gated, k):
    """The last elements of rows that end inside 16 bytes, in every kernel through registers; what lies past
    the rows (NaN here) is neither read into a sum nor needed."""
    announce("linear remainders", gated, k)
    for m, n in ((3, 40), (20, 48), (150, 200), (600, 1100)):
        x = torch.full((m, k + 3), float("nan"), dtype=BF16, device=device)
        w = torch.full((n * (2 if gated else 1), k + 1), float("nan"), dtype=BF16, device=device)
        x[:, :k], w[:, :k] = normal((m, k), k), normal((w.shape[0], k), k + 1, 0.05)
        x, w = x[:, :k], w[:, :k]
        got = ops.gated_linear(x, w) if gated else ops.linear(x, w)
        assert_near(got, reference(x, w, None, "silu", gated=True) if gated else reference(x, w), f"{m} x {n}")


@pytest.mark.gpu
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("k", [8, 56, 64, 72, 128, 192, 256, 264, 512, 576, 2048, 2056])
def test_short_and_ragged_walks(device, gated, k):
    """Every count of stages around the rings' and the teams', whole and ragged."""
    announce("linear walks", gated, k)
    for m, n in ((20, 48), (150, 200)):
        x, w = normal((m, k), k), normal((n * (2 if gated else 1), k), k + 1, 0.05)
        got = ops.gated_linear(x, w) if gated else ops.linear(x, w)
        assert_near(got, reference(x, w, None, "silu", gated=True) if gated else reference(x, w), f"{m} x {n}")


@pytest.mark.gpu
@pytest.mark.parametrize("m, n, k", [(1, 40, 128), (4, 72, 320), (40, 136, 256), (130, 200, 192), (700, 264, 512)])
@pytest.mark.parametrize("shift", [0, 1, 8])
def test_strides_and_alignments(device, m, n, k, shift):
    """Column slices of wider buffers, shifted by whole 16 bytes or by one element; what lies beside
    the output stays as it was."""
    announce("linear strides", m, n, k, shift)
    wide_x, wide_w = normal((m, k + 24), 1), normal((2 * n, k + 40), 2, 0.05)
    x, w = wide_x[:, shift:shift + k], wide_w[:, shift:shift + k]
    wide_out = normal((m, n + 16), 3)
    before = wide_out.clone()
    out = wide_out[:, shift:shift + n]
    residual = normal((m, n + 9), 4)[:, :n]
    gate = normal((m, 7), 5)[:, 3:4]
    assert ops.linear(x, w[:n], gate=gate, residual=residual, out=out).data_ptr() == out.data_ptr()
    assert_near(out, reference(x, w[:n], gate=gate, residual=residual))
    assert torch.equal(wide_out[:, :shift], before[:, :shift]) and torch.equal(wide_out[:, shift + n:], before[:, shift + n:])
    wide_out.copy_(before)
    ops.linear(x, w[:n], residual=out, out=out)  # in place
    assert_near(out, reference(x, w[:n], residual=before[:, shift:shift + n]), "in place")
    wide_out.copy_(before)
    ops.gated_linear(x, w, out=out)
    assert_near(out, reference(x, w, None, "silu", gated=True), "gated")
    assert torch.equal(wide_out[:, :shift], before[:, :shift]) and torch.equal(wide_out[:, shift + n:], before[:, shift + n:])


@pytest.mark.gpu
def test_output_beside_its_input_in_one_buffer(device):
    """Interleaved rows share no byte and are served; a shared gate (stride 0) too."""
    announce("linear interleaved")
    buffer = normal((50, 96 + 64), 6)
    x, out = buffer[:, :96], buffer[:, 96:]
    w, kept = normal((64, 96), 7, 0.05), buffer[:, :96].clone()
    gate = normal((1, 1), 8).expand(50, 1)
    ops.linear(x, w, gate=gate, out=out)
    assert_near(out, reference(kept, w, gate=gate))
    assert torch.equal(buffer[:, :96], kept)
    with pytest.raises(RuntimeError, match="overlaps"):
        ops.linear(x, w, out=buffer[:, 95:159])


@pytest.mark.gpu
@pytest.mark.parametrize("m", [3, 40, 200])
def test_arrays_past_4_gib(device, m):
    """Rows of the input, the weight, the residual and the output lie beyond 32-bit byte offsets."""
    announce("linear far rows", m)
    k, n = 256, 136
    stride = (5 << 30) // 2 // m // 8 * 8 + 8  # the last row starts past 4 GiB

    def spread(rows, columns, source):
        far = torch.empty(rows * stride, dtype=BF16, device=device).as_strided((rows, columns), (stride, 1))
        return far.copy_(source)

    x, w = normal((m, k), 1), normal((n, k), 2, 0.05)
    w_far = spread(m, k, w[:m] if m <= n else torch.cat([w, w])[:m])
    x_far, residual = spread(m, k, x), spread(m, n, normal((m, n), 3))
    got = ops.linear(x_far, w, residual=residual, out=residual.clone() if m < 3 else residual)
    assert_near(got, reference(x, w, residual=normal((m, n), 3)), "far input and output")
    assert_near(ops.linear(x, w_far), reference(x, w_far), "far weight")


#: The DMA kernels' largest row stride, in elements.
FAR = 1 << 22


def spread(source, stride):
    """The rows `stride` elements apart."""
    rows, columns = source.shape
    far = torch.empty((rows - 1) * stride + columns, dtype=source.dtype, device=source.device)
    return far.as_strided((rows, columns), (stride, 1)).copy_(source)


@pytest.mark.gpu
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("stride, by_dma", [(FAR, True), (FAR + 8, False)])
@pytest.mark.parametrize("far, m, n, k", [
    ("input", 700, 136, 264), ("input", 700, 8200, 136), ("input", 1025, 8200, 72), ("input", 1100, 40, 136),
    ("weight", 40, 700, 264), ("weight", 300, 700, 136), ("weight", 3000, 700, 136),
])
def test_tiles_past_4_gib(device, gated, stride, by_dma, far, m, n, k):
    """Tiles of the input and the weight (gated: the gate rows, too) that start past 4 GiB, of up to 256 rows 8 MiB
    apart, by the kernels of ordinary rows and, one step of the stride further, by those through registers."""
    announce("linear far tiles", gated, stride, far, m, n, k)
    x, w = normal((m, k), 1), normal((n * (2 if gated else 1), k), 2, 0.05)
    x_far, w_far = (spread(x, stride), w) if far == "input" else (x, spread(w, stride))
    out = torch.empty((m, n), dtype=BF16, device=device)

    def call():
        return ops.gated_linear(x_far, w_far, out=out) if gated else ops.linear(x_far, w_far, out=out)

    names = kernels_of(call)
    kernel = f"tile_kernelINS0_4Bf16ELb{int(gated)}ELb{int(by_dma)}E"
    assert len(names) == 1 and kernel in names[0], names
    call()
    assert_near(out, reference(x, w, None, "silu", gated=True) if gated else reference(x, w))


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 2])
def test_one_and_two_tokens_past_4_gib(device, m):
    """Weight rows, and their gate rows, past 4 GiB; a second token's input, residual and output, too."""
    announce("linear few tokens far", m)
    n, k = 700, 264
    x, w, residual = normal((m, k), 1), normal((2 * n, k), 2, 0.05), normal((m, n), 3)
    w_far, stride = spread(w, FAR), (1 << 31) + 16
    assert_near(ops.linear(x, w_far), reference(x, w), "far weight")
    assert_near(ops.gated_linear(x, w_far), reference(x, w, None, "silu", gated=True), "far up and gate rows")
    x_far, out = spread(x, stride), spread(residual, stride)
    assert_near(ops.linear(x_far, w[:n], residual=out, out=out), reference(x, w[:n], residual=residual), "far rows")


@pytest.mark.gpu
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("m", [1, 2, 4])
def test_more_columns_than_a_launch_has_wavefronts(device, gated, m):
    announce("linear columns", gated, m)
    n, k = (1 << 26) + 5, 8
    x = normal((m, k), 1)
    w = torch.empty(((2 if gated else 1) * n, k), dtype=BF16, device=device)
    for first in range(0, w.shape[0], 1 << 24):
        part = w[first:first + (1 << 24)]
        part.copy_(normal(part.shape, first))
    got = ops.gated_linear(x, w) if gated else ops.linear(x, w)
    for first in (0, (1 << 25) - 100, n - 200):
        rows = w[first:first + 200]
        if gated:
            rows = torch.cat([rows, w[n + first:n + first + 200]])
        want = reference(x, rows, None, "silu", gated=True) if gated else reference(x, rows)
        assert_near(got[:, first:first + 200], want, f"from {first}")


@pytest.mark.gpu
@pytest.mark.parametrize("m, n, k", [(1, 64, 128), (64, 256, 512), (300, 320, 256)])
def test_infinities_and_nans_stay_in_their_rows(device, m, n, k):
    """A row's NaN or infinity reaches that row's outputs and no other's; a weight row's its column."""
    announce("linear non-finite", m, n, k)
    x, w = normal((m, k), 1), normal((n, k), 2, 0.05)
    want, tolerance = reference(x, w)
    x[m // 2, k - 1] = float("nan")
    w[n - 1, 0] = float("inf")
    got = ops.linear(x, w).double().cpu()
    rows = [r for r in range(m) if r != m // 2]
    assert torch.isnan(got[m // 2]).all()
    if rows:
        assert not torch.isfinite(got[rows][:, n - 1]).any()
        assert ((got[rows][:, :n - 1] - want[rows][:, :n - 1]).abs() <= tolerance[rows][:, :n - 1]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("m, n, k", [(2, 40, 72), (20, 72, 200), (90, 136, 328), (600, 264, 136), (70, 40, 75)])
def test_what_lies_beside_the_rows_is_not_multiplied(device, m, n, k):
    """Inputs are slices of buffers of NaN: before and behind each row, and rows above and below."""
    announce("linear beside", m, n, k)
    x, w = normal((m, k), 1), normal((2 * n, k), 2, 0.05)

    def inside(source):
        rows, columns = source.shape
        buffer = torch.full((rows + 300, columns + 72), float("nan"), dtype=BF16, device=device)
        return buffer[20:20 + rows, 8:8 + columns].copy_(source)

    x_in, w_in = inside(x), inside(w)
    assert_near(ops.linear(x_in, w_in), reference(x, w))
    assert_near(ops.gated_linear(x_in, w_in), reference(x, w, None, "silu", gated=True), "gated")


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 64, 300])
@pytest.mark.parametrize("dtype, low, high", [(F16, 2.0**-24, 2.0**14), (BF16, 2.0**-133, 2.0**60)])
def test_subnormal_inputs_count(device, m, dtype, low, high):
    announce("linear subnormal", m, dtype)
    x = torch.randint(-100, 101, (m, 128), generator=torch.Generator().manual_seed(1)).double().mul(low).to(dtype).to(device)
    w = normal((48, 128), 2, high, dtype=dtype) if dtype == BF16 else normal((48, 128), 2, 1.0, dtype=dtype) * high
    w = w.clamp(-2 * high, 2 * high)
    assert (x != 0).any()
    assert_near(ops.linear(x, w, out_dtype=F32), reference(x, w, out_dtype=F32))
    assert_near(ops.linear(w, x, out_dtype=F32), reference(w, x, out_dtype=F32), "as the weight")


@pytest.mark.gpu
def test_calls_on_two_streams_at_once(device):
    announce("linear two streams")
    sides = [torch.cuda.Stream(), torch.cuda.Stream()]
    inputs = [(normal((m, 1024), m), normal((1536, 1024), m + 1, 0.05)) for m in (700, 40)]
    want = [(ops.linear(x, w), ops.gated_linear(x, w)) for x, w in inputs]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(4):
        for i, side in enumerate(sides):
            with torch.cuda.stream(side):
                x, w = inputs[i]
                got[i].append((ops.linear(x, w), ops.gated_linear(x, w)))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(a, b) for pair in got[i] for a, b in zip(pair, want[i]))


@pytest.mark.gpu
def test_f16_overflow_and_large_activations(device):
    announce("linear overflow")
    x = torch.full((9, 64), 200.0, dtype=F16, device=device)
    w = torch.full((16, 64), 10.0, dtype=F16, device=device)
    w[8:] = -10.0
    got = ops.linear(x, w)
    assert (got[:, :8] == float("inf")).all() and (got[:, 8:] == -float("inf")).all()
    for activation in ("silu", "gelu_tanh"):
        act = ops.linear(x, w, activation=activation, out_dtype=F32)
        assert (act[:, :8] == 128000.0).all() and (act[:, 8:] == 0.0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("m, n, k", [(1, 512, 1024), (60, 256, 1024), (640, 512, 512)])
def test_results_repeat_and_rows_do_not_depend_on_the_batch_s_other_rows(device, m, n, k):
    announce("linear repeats", m, n, k)
    x, w = normal((m, k), 1), normal((n, k), 2, 0.05)
    first = ops.linear(x, w)
    for _ in range(3):
        assert torch.equal(ops.linear(x, w), first)
    x[0] = 0
    assert torch.equal(ops.linear(x, w)[1:], first[1:])


@pytest.mark.gpu
@pytest.mark.parametrize("m, n, k", [(2, 704, 2048), (5, 40, 136), (33, 4104, 520), (100, 4104, 72), (200, 1408, 4096),
                                     (777, 1408, 2048), (1100, 264, 515)])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_gated_results_repeat(device, m, n, k, dtype):
    """Bit for bit, whatever ran before on the same compute units: teams that share K add their sums in one order."""
    announce("gated_linear repeats", m, n, k, dtype)
    x, w = normal((m, k), 1, dtype=dtype), normal((2 * n, k), 2, 0.05, dtype)
    other = normal((1024, 1024), 3)
    first = ops.gated_linear(x, w)
    assert_near(first, reference(x, w, None, "silu", gated=True))
    for _ in range(4):
        ops.linear(other, other)
        assert torch.equal(ops.gated_linear(x, w), first)
        assert torch.equal(ops.gated_linear(x.clone(), w.clone()), first)


@pytest.mark.gpu
def test_captured_replays_and_other_streams(device):
    announce("linear graph")
    x, up_gate, down = normal((48, 256), 1), normal((384, 256), 2, 0.05), normal((256, 192), 3, 0.05)
    gate, residual = normal((48, 1), 4), normal((48, 256), 5)
    one, one_out = x[:1].clone(), torch.empty((1, 256), dtype=BF16, device=device)

    def step():
        ops.linear(ops.gated_linear(one, up_gate), down, out=one_out)
        return ops.linear(ops.gated_linear(x, up_gate), down, gate=gate, residual=residual)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        step()
        side.synchronize()
        with torch.cuda.graph(graph, stream=side):
            got = step()
    torch.cuda.current_stream().wait_stream(side)
    for seed in (10, 11, 12):
        x.copy_(normal((48, 256), seed))
        one.copy_(x[:1])
        graph.replay()
        torch.cuda.synchronize()
        replayed, replayed_one = got.clone(), one_out.clone()
        assert torch.equal(step(), replayed) and torch.equal(one_out, replayed_one)
        torch.cuda.synchronize()


@pytest.mark.gpu
def test_no_rows(device):
    w = normal((32, 64), 1)
    assert ops.linear(torch.empty((0, 64), dtype=BF16, device=device), w).shape == (0, 32)
    assert ops.gated_linear(torch.empty((0, 64), dtype=BF16, device=device), w).shape == (0, 16)


@pytest.mark.gpu
def test_strides_that_a_call_does_not_use(device):
    """The C entry with anything in the strides of absent arrays and of single rows."""
    announce("linear unused strides")
    x, w = normal((1, 256), 1), normal((48, 256), 2, 0.05)
    gate, residual, out = normal((1, 1), 3), normal((1, 48), 4), torch.empty((1, 48), dtype=BF16, device=device)
    call = filled_call()
    call.input, call.weight, call.out = x.data_ptr(), w.data_ptr(), out.data_ptr()
    call.m, call.n, call.k, call.weight_row_stride = 1, 48, 256, 256
    call.input_row_stride = call.out_row_stride = call.residual_row_stride = call.gate_stride = 1 << 60
    assert abi.library().uniserve_linear(ctypes.byref(call), None) == 0, call.error
    torch.cuda.synchronize()
    assert_near(out, reference(x, w))
    call.gate, call.residual = gate.data_ptr(), residual.data_ptr()
    assert abi.library().uniserve_linear(ctypes.byref(call), None) == 0, call.error
    torch.cuda.synchronize()
    assert_near(out, reference(x, w, gate=gate, residual=residual), "one row's gate and residual")


@pytest.mark.gpu
@pytest.mark.parametrize("arguments, says", [
    (dict(weight=torch.zeros(8, 16, dtype=F16)), "input's type"), (dict(weight=torch.zeros(8, 16, dtype=BF16)), "device"),
    (dict(weight="narrow"), "weight"), (dict(activation="relu"), "activation"), (dict(bias="short"), "bias"),
    (dict(bias="half"), "bias"), (dict(gate="flat"), "gate"), (dict(gate="host"), "gate"), (dict(residual="short"), "residual"),
    (dict(residual="wide"), "residual"), (dict(out="wide", out_dtype=BF16), "output"), (dict(out="short"), "output"),
    (dict(out="columns"), "output"), (dict(out_dtype=torch.int32), "output"),
])
def test_python_refusals_of_device_calls(device, arguments, says):
    made = {
        "weight.narrow": lambda: normal((8, 15), 1), "bias.short": lambda: normal((7,), 1),
        "bias.half": lambda: normal((8,), 1, dtype=F16), "gate.flat": lambda: normal((4,), 1),
        "gate.host": lambda: torch.zeros((4, 1), dtype=BF16), "residual.short": lambda: normal((3, 8), 1),
        "residual.wide": lambda: normal((4, 8), 1, dtype=F32), "out.wide": lambda: normal((4, 8), 1, dtype=F32),
        "out.short": lambda: normal((4, 7), 1), "out.columns": lambda: normal((8, 4), 1).t(),
    }
    arguments = {k: made[f"{k}.{v}"]() if f"{k}.{v}" in made else v for k, v in arguments.items()}
    weight = arguments.pop("weight", None)
    if weight is not None and weight.dtype == F16:
        weight = weight.to(device)
    with pytest.raises((ValueError, RuntimeError), match=says):
        ops.linear(normal((4, 16), 1), normal((8, 16), 2) if weight is None else weight, **arguments)
