"""adapter_linear and adapter_gated_linear: refusals on the CPU, and on the MI355X against the formulas in 64 bits.

Tolerance, element by element, with u = 2^-24. The product's part is test_linear's: S = sum |x w| (+ |bias|) of an
output, 2 (K + 1) u S. A rank value v_j = scale * sum x a has L_j = |scale| sum |x a|: its FP32 sum is off by
2 (K + 1) u L_j and the scale adds u L_j; held as a pair of elements it is off by half a step of its error's
type, eps / 2 of at most eps / 2 of |v_j| (bf16: 2^-18; f16, whose pairs share a power of two: 2^-24 of the largest of the
group besides, the errors' subnormals), and, where v_j is so small that the pair's second element is subnormal, by that
subnormal's half step (bf16: 2^-134). The second product's terms v_j b_j add R of those, and its sum over values and
errors 2 (2 R + 2) u of sum (L_j |b_j|), the addition to the product's sum included.
Behind the sum follow the activation, the gate, the residual and the rounding of test_linear.
"""

import ctypes
import subprocess
from pathlib import Path

import pytest
import torch

from gpu_helpers import announce, assert_as_the_formula, kernels_of
from test_linear import BF16, F16, F32, KERNELS, U, activated, assert_near, normal, rounding
from uniserve_moe import abi, ops


def reference(x, w, down, up, adapter, scales=None, bias=None, activation=None, gate=None, residual=None, out_dtype=None,
              gated=False):
    """The output in 64 bits and how far the kernel may be from it, both on the CPU."""
    dtype, out_dtype = x.dtype, out_dtype or x.dtype
    x, w, down, up = (t.double().cpu() for t in (x, w, down, up))
    tokens, k = x.shape
    halves = 2 if gated else 1
    rank, rows = up.shape[2], up.shape[1] // halves
    y, s = x @ w.t(), x.abs() @ w.abs().t()
    off = 2 * (k + 1) * U * s
    for a in range(up.shape[0]):
        at = torch.nonzero(adapter.cpu() == a).flatten()
        if at.numel() == 0:
            continue
        scale = 1.0 if scales is None else scales[a].double().cpu()
        for h in range(halves):
            factor, back = down[a, h * rank:(h + 1) * rank], up[a, h * rows:(h + 1) * rows]
            v, size = scale * x[at] @ factor.t(), abs(scale) * x[at].abs() @ factor.abs().t()
            e = (2 * (k + 1) + 1) * U * size
            if dtype == BF16:
                e = e + 2.0**-18 * (v.abs() + e) + 2.0**-134
            else:
                most = torch.cat([(c.abs() + d).amax(1, keepdim=True).expand_as(c) for c, d in zip(v.split(32, 1), e.split(32, 1))], 1)
                e = e + 2.0**-24 * (v.abs() + e) + 2.0**-24 * most
            place = slice(h * rows, (h + 1) * rows)
            y[at, place] += v @ back.t()
            part = size @ back.abs().t()
            s[at, place] += part
            off[at, place] += e @ back.abs().t() + 2 * (2 * rank + 2) * U * part + 2 * U * s[at, place]
    if bias is not None:
        y, s = y + bias.double().cpu(), s + bias.double().cpu().abs()
        off = off + 2 * U * s
    slope = 1.13
    if gated:
        n = w.shape[0] // 2
        first, g = y[:, :n], y[:, n:]
        act = activated(g, activation)
        off = act.abs() * off[:, :n] + slope * off[:, n:] * (first.abs() + off[:, :n])
        y = first * act
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


# ---- without a GPU ----------------------------------------------------------------------------------


def filled_call(gated=False):
    call = abi.AdapterLinearCall()
    call.input, call.weight, call.out = 1 << 20, 2 << 20, 3 << 20
    call.m, call.n, call.k = 4, 32, 64
    call.input_row_stride, call.weight_row_stride, call.out_row_stride = 64, 64, 32
    call.dtype = call.bias_dtype = call.out_dtype = abi.DTYPE["bf16"]
    call.activation = abi.ACTIVATION["silu"] if gated else -1
    call.down, call.up, call.adapter, call.scales, call.workspace = 4 << 20, 5 << 20, 6 << 20, 7 << 20, 8 << 20
    call.workspace_bytes, call.adapters, call.rank = 1 << 20, 3, 16
    call.down_stride, call.down_row_stride = (2 if gated else 1) * 16 * 64, 64
    call.up_stride, call.up_row_stride = (2 if gated else 1) * 32 * 16, 16
    return call


def entry_of(gated):
    return abi.library().uniserve_adapter_gated_linear if gated else abi.library().uniserve_adapter_linear


REFUSED = [
    ({"m": -1}, "positive"), ({"k": 0}, "positive"), ({"input": None}, "needs"), ({"dtype": abi.DTYPE["f32"]}, "bf16 or f16"),
    ({"out": 1 << 20}, "overlaps"), ({"input_row_stride": 63}, "strides"), ({"activation": 2}, "gelu_tanh"),
    ({"rank": 0}, "positive rank"), ({"rank": -8}, "positive rank"), ({"adapters": 0}, "positive rank"), ({"rank": 513}, "512"),
    ({"adapters": 1 << 31}, "int32"), ({"m": 1 << 28, "out": 1 << 50}, "rows"),
    ({"down": None}, "needs"), ({"up": None}, "needs"), ({"adapter": None}, "needs"), ({"workspace": None}, "needs"),
    ({"down_row_stride": 63}, "adapter strides"), ({"up_row_stride": 15}, "adapter strides"), ({"down_stride": -1}, "adapter strides"),
    ({"up_stride": -64}, "adapter strides"), ({"down_stride": 1 << 60}, "too large"), ({"up_row_stride": 1 << 60}, "too large"),
    ({"workspace_bytes": 4 * 80 - 1}, "workspace of"), ({"workspace": (8 << 20) + 8}, "aligned"),
    ({"out": 4 << 20}, "its adapters"), ({"out": (4 << 20) - 16}, "its adapters"), ({"out": (5 << 20) + 64}, "its adapters"),
    ({"adapter": (3 << 20) + 16}, "its adapters"), ({"scales": (3 << 20) + 128}, "its adapters"), ({"workspace": (3 << 20) - 16}, "its adapters"),
    ({"workspace": 1 << 20}, "workspace overlaps"), ({"workspace": 2 << 20}, "workspace overlaps"), ({"workspace": (4 << 20) + 64}, "workspace overlaps"),
    ({"workspace": 5 << 20}, "workspace overlaps"), ({"workspace": 6 << 20}, "workspace overlaps"), ({"bias": (8 << 20) + 4}, "workspace overlaps"),
]


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("fields, says", REFUSED)
def test_refusals(gated, fields, says):
    call = filled_call(gated)
    for name, value in fields.items():
        setattr(call, name, value)
    assert entry_of(gated)(ctypes.byref(call), None) != 0
    assert says in call.error.decode()


@pytest.mark.parametrize("fields", [{"gate": 8 << 20, "gate_stride": 1}, {"residual": 8 << 20, "residual_row_stride": 32}])
def test_workspace_over_the_epilogue_s_inputs(fields):
    call = filled_call()
    for name, value in fields.items():
        setattr(call, name, value)
    assert entry_of(False)(ctypes.byref(call), None) != 0
    assert "workspace overlaps" in call.error.decode()


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("fields", [{"adapters": 1, "down_stride": -1, "up_stride": 1 << 60}, {"rank": 1, "up_stride": 64, "down_row_stride": -1}])
def test_unused_strides_are_not_read(gated, fields):
    """The call comes to the last check (the workspace is the input here)."""
    if gated and "rank" in fields:
        return
    call = filled_call(gated)
    for name, value in {**fields, "workspace": 1 << 20}.items():
        setattr(call, name, value)
    assert entry_of(gated)(ctypes.byref(call), None) != 0
    assert "workspace overlaps" in call.error.decode()


@pytest.mark.parametrize("gated", [False, True])
def test_no_rows_launch_nothing(gated):
    call = filled_call(gated)
    call.m, call.input, call.out, call.workspace, call.adapter = 0, None, None, None, None
    assert entry_of(gated)(ctypes.byref(call), None) == 0
    assert entry_of(gated)(None, None) != 0


def test_workspace_sizes():
    """A group's values, their errors and 16 bytes: 8, 16 or 32 ranks; whichever of one half and two takes more."""
    size = ops.adapter_workspace
    assert size(1, 1) == 2 * 48 and size(10, 8) == 10 * 2 * 48 and size(1, 16) == 2 * 48 and size(3, 64) == 3 * 2 * 144
    assert size(2, 96) == 2 * 2 * 2 * 144 and size(0, 8) == 0 and size(-1, 8) == 0 and size(4, 1025) == 0


def test_lanes_read_within_their_row(tmp_path):
    """Every address that the second product's lanes take from a row's rank values, for each rank and half: the bytes
    read end within the row, as the workspace ends with the last one."""
    (tmp_path / "reads.cpp").write_text("""
#include <cstdio>
#include "low_layout.hpp"
int main() {
  for (int rank = 1; rank <= 512; ++rank) {
    const uniserve::linear::LowLayout layout(rank);
    for (int halves = 1; halves <= 2; ++halves)
      for (int part = 0; part < halves * layout.groups; ++part) {
        const int64_t group = static_cast<int64_t>(part) * layout.group_bytes(), row = layout.row_bytes(halves);
        for (int g = 0; g < 4; ++g) {
          int64_t end = group + layout.piece_at(g) + 16;
          if (layout.width == 32 && group + layout.errors_at(g) + 16 > end) end = group + layout.errors_at(g) + 16;
          if (group + layout.factor_at() + 4 > end) end = group + layout.factor_at() + 4;
          if (end > row || layout.piece_at(g) < 0 || (layout.has_piece(g) && layout.piece_at(g) != 16 * g))
            return std::printf("rank %d, %d halves, group %d, lanes %d: %lld of %lld bytes", rank, halves, part, g,
                               static_cast<long long>(end), static_cast<long long>(row)), 1;
        }
      }
  }
}
""")
    csrc = Path(__file__).resolve().parent.parent / "uniserve-v1_amd" / "csrc"
    subprocess.run(["g++", "-std=c++17", "-I", csrc, tmp_path / "reads.cpp", "-o", tmp_path / "reads"], check=True)
    ran = subprocess.run([tmp_path / "reads"], capture_output=True, text=True)
    assert ran.returncode == 0, ran.stdout


def test_python_refusals():
    zeros = [torch.zeros(s, dtype=BF16) for s in ((2, 8), (4, 8), (1, 4, 8), (1, 4, 4))]
    with pytest.raises(ValueError, match="on a GPU"):
        ops.adapter_linear(*zeros, torch.zeros(2, dtype=torch.int32))
    with pytest.raises(ValueError, match="up rows"):
        ops.adapter_gated_linear(zeros[0], torch.zeros(5, 8, dtype=BF16), *zeros[2:], torch.zeros(2, dtype=torch.int32))


# ---- on the MI355X ----------------------------------------------------------------------------------

SHAPES = [(1, 1, 1), (1, 2048, 1408), (2, 33, 72), (3, 1000, 72), (5, 33, 1000), (16, 256, 128), (17, 130, 264), (33, 512, 520),
          (64, 128, 2048), (65, 65, 65), (129, 257, 384), (200, 704, 1024), (257, 384, 1984), (300, 1001, 1000), (1025, 640, 640)]
RANKS = [1, 5, 8, 12, 16, 24, 32, 40, 64]


def stacks(adapters, rank, n, k, dtype=BF16, seed=50, halves=1):
    down = normal((adapters, halves * rank, k), seed, 0.05, dtype)
    up = normal((adapters, halves * n, rank), seed + 1, 0.1, dtype)
    scales = torch.rand(adapters, generator=torch.Generator().manual_seed(seed)).add_(0.5).to(down.device)
    return dict(down=down, up=up, scales=scales)


def each_other(tokens, adapters, seed=9):
    """A request a row in any order, some of them without an adapter."""
    return torch.randint(-1, adapters, (tokens,), generator=torch.Generator().manual_seed(seed), dtype=torch.int32).cuda()


def runs(tokens, adapters, seed=9):
    """Runs of rows with one adapter or none."""
    g = torch.Generator().manual_seed(seed)
    ends = torch.randint(0, tokens + 1, (7,), generator=g).sort().values.tolist() + [tokens]
    index, first = torch.empty(tokens, dtype=torch.int32), 0
    for i, end in enumerate(ends):
        index[first:end] = (i * 3) % (adapters + 1) - 1
        first = end
    return index.cuda()


@pytest.mark.gpu
@pytest.mark.parametrize("m, n, k", SHAPES)
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("order", [each_other, runs])
def test_adapter_linear(device, m, n, k, dtype, order):
    for rank in (RANKS[(m + n + k) % 9], RANKS[(m + n + k + 4) % 9]):
        announce("adapter_linear", m, n, k, dtype, rank)
        x, w = normal((m, k), m + k, dtype=dtype), normal((n, k), n + k + 1, 0.05, dtype)
        call = dict(stacks(6, rank, n, k, dtype), adapter=order(m, 6))
        assert_near(ops.adapter_linear(x, w, **call), reference(x, w, **call))
        assert_near(ops.adapter_linear(x, w, **call, out_dtype=F32), reference(x, w, **call, out_dtype=F32), "f32")


@pytest.mark.gpu
@pytest.mark.parametrize("m, n, k", SHAPES)
@pytest.mark.parametrize("dtype, activation", [(BF16, "silu"), (F16, "gelu_tanh")])
@pytest.mark.parametrize("order", [each_other, runs])
def test_adapter_gated_linear(device, m, n, k, dtype, activation, order):
    rank = RANKS[(m + n + k + 2) % 9]
    announce("adapter_gated_linear", m, n, k, dtype, rank)
    x, w, bias = normal((m, k), m + k, dtype=dtype), normal((2 * n, k), n + k + 1, 0.05, dtype), normal((2 * n,), 5, 0.5, F32)
    call = dict(stacks(5, rank, n, k, dtype, halves=2), adapter=order(m, 5), bias=bias, activation=activation)
    assert_near(ops.adapter_gated_linear(x, w, **call), reference(x, w, **call, gated=True))


@pytest.mark.gpu
@pytest.mark.parametrize("rank", RANKS + [33, 96, 128, 200, 512])
@pytest.mark.parametrize("m", [1, 2, 16, 70, 300])
@pytest.mark.parametrize("gated", [False, True])
def test_every_rank(device, rank, m, gated):
    announce("adapter ranks", rank, m, gated)
    n, k = 72, 136
    for dtype in (BF16, F16):
        x, w = normal((m, k), 1, dtype=dtype), normal((n * (2 if gated else 1), k), 2, 0.05, dtype)
        call = dict(stacks(3, rank, n, k, dtype, halves=2 if gated else 1), adapter=each_other(m, 3))
        if gated:
            assert_near(ops.adapter_gated_linear(x, w, **call), reference(x, w, **call, activation="silu", gated=True))
        else:
            assert_near(ops.adapter_linear(x, w, **call), reference(x, w, **call))


@pytest.mark.gpu
@pytest.mark.parametrize("m, n, k", [(1, 40, 128), (2, 520, 264), (40, 136, 256), (130, 200, 192), (700, 264, 512)])
@pytest.mark.parametrize("dtype, activation", [(BF16, "gelu_tanh"), (F16, "silu")])
def test_with_everything(device, m, n, k, dtype, activation):
    announce("adapter epilogue", m, n, k, dtype)
    x, w = normal((m, k), m + k, dtype=dtype), normal((n, k), n + k + 1, 0.05, dtype)
    call = dict(stacks(4, 16, n, k, dtype), adapter=each_other(m, 4), bias=normal((n,), 5, 0.5, dtype), activation=activation,
                gate=normal((m, 1), 3, 2.0, dtype), residual=normal((m, n), 4, 1.0, dtype))
    want = reference(x, w, **call)
    assert_near(ops.adapter_linear(x, w, **call), want)
    over = call["residual"]
    assert ops.adapter_linear(x, w, **call, out=over) is over
    assert_near(over, want, "in place")


@pytest.mark.gpu
@pytest.mark.parametrize("gated, shape, m, n, k", KERNELS)
@pytest.mark.parametrize("rank", [8, 40])
def test_each_tile_kernel(device, gated, shape, m, n, k, rank):
    """The products' shapes, each with rows of many adapters and with runs of a few."""
    announce("adapter kernel", shape, gated, m, n, k, rank)
    x, w, out = normal((m, k), 1), normal((n * (2 if gated else 1), k), 2, 0.05), normal((m, n), 3)
    call = dict(stacks(5, rank, n, k, halves=2 if gated else 1), adapter=each_other(m, 5))
    workspace = torch.empty(ops.adapter_workspace(m, rank * (2 if gated else 1)), dtype=torch.uint8, device=device)

    def run():
        entry = ops.adapter_gated_linear if gated else ops.adapter_linear
        return entry(x, w, **call, out=out, workspace=workspace)

    mangled = "TileShapeI" + "".join(f"Li{d}E" for d in shape.split(","))
    names = kernels_of(run)
    assert len(names) == 2 and "RankParams" in names[0] and mangled in names[1], names
    for order in (each_other, runs):
        call["adapter"].copy_(order(m, 5))
        run()
        assert_near(out, reference(x, w, **call, activation="silu" if gated else None, gated=gated))


@pytest.mark.gpu
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("m, n, k", [(1100, 3001, 507), (2000, 3001, 123), (130, 3001, 5), (130, 1001, 2047), (8, 40, 2047)])
def test_unaligned_rows(device, gated, m, n, k):
    announce("adapter unaligned", gated, m, n, k)
    x, w = normal((m, k), 1), normal((n * (2 if gated else 1), k), 2, 0.05)
    call = dict(stacks(4, 7, n, k, halves=2 if gated else 1), adapter=runs(m, 4))
    got = ops.adapter_gated_linear(x, w, **call) if gated else ops.adapter_linear(x, w, **call)
    assert_near(got, reference(x, w, **call, activation="silu" if gated else None, gated=gated))


#: The shapes that f16 rows have, too (the largest tiles do not serve them).
F16_KERNELS = [case for case in KERNELS if not case[1].startswith(("256,256", "192,256"))]
#: Shapes through registers, for rows that are not whole 16-byte pieces.
UNALIGNED_KERNELS = [(False, "96,128,2,2,2,1", 2000, 3001, 123), (True, "96,128,2,2,2,1", 2000, 3001, 123),
                     (False, "128,128,2,4,2,1", 1100, 3001, 507), (True, "128,128,2,4,2,1", 1100, 3001, 507),
                     (False, "64,64,2,2,2,1", 130, 3001, 5), (True, "32,32,1,1,2,4", 130, 1001, 2047), (False, "16,32,1,1,2,4", 8, 40, 2047)]


@pytest.mark.gpu
@pytest.mark.parametrize("gated, shape, m, n, k", F16_KERNELS + UNALIGNED_KERNELS)
@pytest.mark.parametrize("rank", [5, 8, 16, 40])
def test_each_tile_kernel_of_f16(device, gated, shape, m, n, k, rank):
    """f16 rows have a factor for each group of ranks, in the large tiles through LDS behind the walk: the shapes by DMA and
    through registers, each with rows of many adapters and with runs of a few; a row's rank values of far apart sizes in
    its halves and groups."""
    announce("adapter f16 kernel", shape, gated, m, n, k, rank)
    halves = 2 if gated else 1
    x, w, out = normal((m, k), 1, dtype=F16), normal((n * halves, k), 2, 0.05, F16), normal((m, n), 3, dtype=F16)
    call = dict(stacks(5, rank, n, k, F16, halves=halves), adapter=each_other(m, 5))
    sizes = 2.0 ** torch.tensor([-9.0, 6.0, 0.0, -3.0], device=device)[(torch.arange(halves * rank, device=device) * 5 // rank) % 4]
    call["down"] = (call["down"].float() * sizes[:, None]).to(F16)
    up_sizes = 1.0 / sizes.view(halves, rank).repeat_interleave(n, 0)  # (halves' rows by halves' ranks)
    call["up"] = (call["up"].float() * up_sizes).to(F16)
    workspace = torch.empty(ops.adapter_workspace(m, rank * halves), dtype=torch.uint8, device=device)

    def run():
        entry = ops.adapter_gated_linear if gated else ops.adapter_linear
        return entry(x, w, **call, out=out, workspace=workspace)

    mangled = "TileShapeI" + "".join(f"Li{d}E" for d in shape.split(","))
    names = kernels_of(run)
    assert len(names) == 2 and "RankParams" in names[0] and mangled in names[1], names
    for order in (each_other, runs):
        call["adapter"].copy_(order(m, 5))
        run()
        assert_near(out, reference(x, w, **call, activation="silu" if gated else None, gated=gated))


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 20, 300])
@pytest.mark.parametrize("shift", [0, 1, 8])
@pytest.mark.parametrize("rank", [5, 16])
def test_strides_of_stacks(device, m, shift, rank):
    """Slices of a pool of adapters, of more ranks and columns than are used; what lies beside them is NaN."""
    announce("adapter strides", m, shift, rank)
    n, k = 48, 72
    made = stacks(3, rank, n, k)

    def inside(source):
        adapters, rows, columns = source.shape
        pool = torch.full((adapters, 2, rows + 3, columns + 24), float("nan"), dtype=BF16, device=device)
        return pool[:, 1, 2:2 + rows, shift:shift + columns].copy_(source)

    x, w, adapter = normal((m, k), 1), normal((n, k), 2, 0.05), each_other(m, 3)
    call = dict(made, adapter=adapter)
    got = ops.adapter_linear(x, w, inside(made["down"]), inside(made["up"]), adapter, scales=made["scales"])
    assert_near(got, reference(x, w, **call))
    shared = dict(down=made["down"][:1].expand(3, -1, -1), up=made["up"][:1].expand(3, -1, -1), scales=made["scales"], adapter=adapter)
    assert_near(ops.adapter_linear(x, w, **shared), reference(x, w, **shared), "one factor for all")


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 2, 33, 300])
@pytest.mark.parametrize("gated", [False, True])
def test_no_adapter_gives_the_product(device, m, gated):
    """Indices outside the stack name none: the product's bits, whatever the stacks and the workspace hold."""
    announce("adapter none", m, gated)
    n, k, halves = 72, 136, 2 if gated else 1
    x, w = normal((m, k), 1), normal((n * halves, k), 2, 0.05)
    nan = dict(down=torch.full((2, halves * 16, k), float("nan"), dtype=BF16, device=device),
               up=torch.full((2, halves * n, 16), float("nan"), dtype=BF16, device=device))
    workspace = torch.full((ops.adapter_workspace(m, halves * 16),), 255, dtype=torch.uint8, device=device)
    index = torch.tensor([-1, 2, -2**31, 2**31 - 1, 7] * m, dtype=torch.int32, device=device)[:m]
    if gated:
        assert torch.equal(ops.adapter_gated_linear(x, w, **nan, adapter=index, workspace=workspace), ops.gated_linear(x, w))
    else:
        assert torch.equal(ops.adapter_linear(x, w, **nan, adapter=index, workspace=workspace), ops.linear(x, w))


@pytest.mark.gpu
@pytest.mark.parametrize("m", [2, 16, 60, 300, 1100])
@pytest.mark.parametrize("rank", [8, 16, 32])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_infinities_and_nans_stay_with_their_adapter(device, m, rank, dtype):
    announce("adapter non-finite", m, rank, dtype)
    n, k = 72, 136
    x, w = normal((m, k), 1, dtype=dtype), normal((n, k), 2, 0.05, dtype)
    call = dict(stacks(4, rank, n, k, dtype), adapter=(torch.arange(m) % 4 - 1).int().cuda())
    want = ops.adapter_linear(x, w, **call)
    call["down"][1, 3, 5], call["up"][3] = float("nan"), float("inf")
    call["up"][2, 7] = float("nan")
    call["down"][3, :, 0] = float("-inf")
    got = ops.adapter_linear(x, w, **call)
    clean = (call["adapter"] == -1) | (call["adapter"] == 0)
    assert torch.equal(got[clean], want[clean])
    one, two = call["adapter"] == 1, call["adapter"] == 2
    assert torch.isnan(got[one]).all() and not torch.isfinite(got[two][:, 7]).any()
    kept = [c for c in range(n) if c != 7]
    assert torch.equal(got[two][:, kept], want[two][:, kept])


@pytest.mark.gpu
@pytest.mark.parametrize("gated, shape, m, n, k", [case for case in KERNELS if "2,4," in case[1] or "128,128" in case[1] or "96,128" in case[1]])
@pytest.mark.parametrize("rank", [8, 40])
def test_infinities_and_nans_in_large_tiles(device, gated, shape, m, n, k, rank):
    """Tiles of rows of several adapters, one with up rows that are not finite: the others' rows are as without it."""
    announce("adapter non-finite tiles", shape, gated, m, n, k, rank)
    halves = 2 if gated else 1
    entry = ops.adapter_gated_linear if gated else ops.adapter_linear
    x, w, adapter = normal((m, k), 1), normal((n * halves, k), 2, 0.05), runs(m, 4)
    call = dict(stacks(4, rank, n, k, halves=halves), adapter=adapter)
    want, tolerance = reference(x, w, **call, activation="silu" if gated else None, gated=gated)
    call["up"][2, 5], call["up"][2, n * halves - 1, rank - 1] = float("nan"), float("inf")
    got = entry(x, w, **call).double().cpu()
    clean = adapter.cpu() != 2
    assert clean.any() and ((got[clean] - want[clean]).abs() <= tolerance[clean]).all()
    touched = ~clean
    assert not torch.isfinite(got[touched][:, [5, n - 1]]).any()
    kept = [c for c in range(n) if c not in (5, n - 1)]
    assert ((got[touched][:, kept] - want[touched][:, kept]).abs() <= tolerance[touched][:, kept]).all()


#: Calls of one and two rows.
FEW = [(False, "", 1, 520, 136), (False, "", 2, 72, 264), (True, "", 1, 72, 136), (True, "", 2, 520, 72)]


def columns_of(call, w, columns, halves):
    """The call on some output columns alone."""
    n = w.shape[0] // halves
    rows = torch.tensor([c + h * n for h in range(halves) for c in columns], device=w.device)
    return {**call, "w": w[rows], "up": call["up"][:, rows]}


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, gated, shape, m, n, k", [(BF16, *case) for case in KERNELS + FEW] + [(F16, *case) for case in F16_KERNELS + FEW])
@pytest.mark.parametrize("rank", [8, 24])
def test_infinite_up_weights_give_the_formula_s_infinities(device, dtype, gated, shape, m, n, k, rank):
    """Infinities and NaN in a few up rows, with rank values that one element holds (of which nothing is left for the pair's
    other one) and with any, in tiles of one adapter and of several: NaN and either infinity where the formula has them, the
    columns' other rows within the tolerance (large tiles make them again) and the other columns as they were."""
    announce("adapter infinite up weights", dtype, shape, gated, m, n, k, rank)
    halves, inf = 2 if gated else 1, float("inf")
    entry = ops.adapter_gated_linear if gated else ops.adapter_linear
    x, w = normal((m, k), 1, dtype=dtype), normal((n * halves, k), 2, 0.05, dtype)
    for order, exact in ((lambda m, _: torch.zeros(m, dtype=torch.int32, device=device), True), (runs, False), (each_other, True)):
        call = dict(stacks(4, rank, n, k, dtype, halves=halves), adapter=order(m, 4))
        if exact:  # rank values 1, 2, .. 5 times the row's first element
            call["down"][:] = 0
            call["down"][:, :, 0] = (torch.arange(halves * rank, device=device) % 5 + 1).to(dtype)
            call["scales"] = None
        want = entry(x, w, **call)
        columns = [0, 3, n // 2, n - 3, n - 1]
        for i, c in enumerate(columns):
            place = c + (n if gated and i % 2 else 0)
            for a in (0, 2):
                call["up"][a, place, (i * 5 + a) % rank] = (inf, -inf, inf, float("nan"), -inf)[i]
        call["up"][0, n // 2, 0] = inf
        got = entry(x, w, **call)
        y, tolerance = reference(x, **columns_of(call, w, columns, halves), activation="silu" if gated else None, gated=gated)
        assert_as_the_formula(got[:, columns], y)
        finite = torch.isfinite(y)
        assert ((got[:, columns].double().cpu() - y).abs()[finite] <= tolerance[finite]).all()
        kept = torch.ones(n, dtype=torch.bool, device=device)
        kept[columns] = False
        assert torch.equal(got[:, kept], want[:, kept])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, shape, m, n, k", [(BF16, *case[1:]) for case in KERNELS + FEW if case[0]] + [(F16, *case[1:]) for case in F16_KERNELS + FEW if case[0]])
@pytest.mark.parametrize("rank", [8, 40])
def test_infinite_rank_values_stay_in_their_half(device, dtype, shape, m, n, k, rank):
    """An infinity in one half's first factor makes that half's sums infinite, and not the other's, in tiles of one adapter
    and of several."""
    announce("adapter infinite rank values", dtype, shape, m, n, k, rank)
    x, w = normal((m, k), 1, dtype=dtype), normal((2 * n, k), 2, 0.05, dtype)
    columns = sorted({0, 1, n // 3, n // 2, n - 2, n - 1})
    for order in (lambda m, _: torch.zeros(m, dtype=torch.int32, device=device), runs, each_other):
        call = dict(stacks(4, rank, n, k, dtype, halves=2), adapter=order(m, 4))
        want = ops.adapter_gated_linear(x, w, **call)
        call["down"][0, 1, 3], call["down"][2, rank + rank - 1, 5] = float("inf"), float("-inf")
        got = ops.adapter_gated_linear(x, w, **call)
        y = reference(x, **columns_of(call, w, columns, 2), activation="silu", gated=True)[0]
        assert_as_the_formula(got[:, columns], y)
        clean = (call["adapter"] != 0) & (call["adapter"] != 2)
        assert torch.equal(got[clean], want[clean])


@pytest.mark.gpu
@pytest.mark.parametrize("gated, shape, m, n, k", [case for case in KERNELS if case[2] >= 100 and case[1] != "64,64,2,2,4,1"])
def test_rows_that_are_not_finite(device, gated, shape, m, n, k):
    """Rows of NaN, with a NaN and with an infinity, beside others, in tiles of one adapter and of several, one of them with
    an infinite up weight: what the formula makes of each."""
    announce("adapter rows not finite", shape, gated, m, n, k)
    halves, rank = 2 if gated else 1, 16
    entry = ops.adapter_gated_linear if gated else ops.adapter_linear
    x, w = normal((m, k), 1), normal((n * halves, k), 2, 0.05)
    x[3], x[7::11, k - 1], x[5, 2], x[8::13, 4] = float("nan"), float("nan"), float("inf"), float("-inf")
    columns = sorted({0, 1, n // 3, n - 2, n - 1})
    for order in (lambda m, _: torch.zeros(m, dtype=torch.int32, device=device), runs, each_other):
        call = dict(stacks(4, rank, n, k, halves=halves), adapter=order(m, 4))
        for poisoned in (False, True):
            if poisoned:
                call["up"][0, n - 1, 3], call["up"][1, n // 3, 9] = float("inf"), float("nan")
            got = entry(x, w, **call)
            y = reference(x, **columns_of(call, w, columns, halves), activation="silu" if gated else None, gated=gated)[0]
            assert_as_the_formula(got[:, columns], y)


@pytest.mark.gpu
@pytest.mark.parametrize("m, n", [(1, 72), (2, 72), (40, 72), (513, 4104)])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_finite_rank_values_beside_an_infinite_one(device, m, n, dtype):
    """180000 is no f16 number; beside an infinity, from which it is subtracted, it is finite all the same."""
    announce("adapter beside an infinite rank value", m, n, dtype)
    k, rank = 72, 8
    x, w = torch.zeros((m, k), dtype=dtype, device=device), normal((n, k), 2, 0.05, dtype)
    x[:, 0], x[:, 1] = 1.0, 2.0
    call = dict(stacks(2, rank, n, k, dtype), adapter=(torch.arange(m) % 2).int().to(device), scales=None)
    call["down"][:, :, :2] = 0
    call["down"][0, 0, 0], call["down"][:, 1, :2] = float("inf"), 60000.0
    call["up"][:, :, :2] = torch.tensor([1.0, -1.0], dtype=dtype)
    got, (y, tolerance) = ops.adapter_linear(x, w, **call, out_dtype=F32), reference(x, w, **call, out_dtype=F32)
    assert (got[0::2] == float("inf")).all() and torch.isfinite(got[1::2]).all()
    assert ((got.double().cpu() - y).abs()[1::2] <= tolerance[1::2]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 40, 300])
@pytest.mark.parametrize("size", [2.0**-20, 2.0**-10, 2.0**9])
def test_f16_rank_values_of_any_size(device, m, size):
    """Rank values beyond f16's largest number, and below its normal ones, brought back by the other factor."""
    announce("adapter f16 range", m, size)
    n, k, rank = 40, 512, 12
    x, w = normal((m, k), 1, dtype=F16), normal((n, k), 2, 0.05, F16)
    made = stacks(2, rank, n, k, F16)
    made["down"] = (made["down"].float() * 16 * size).to(F16)
    made["up"] = (made["up"].float() / (16 * max(size, 2.0**-10))).clamp(-1000, 1000).to(F16)
    made["scales"] = made["scales"] * (64.0 if size > 1 else 1.0)
    call = dict(made, adapter=each_other(m, 2))
    assert_near(ops.adapter_linear(x, w, **call, out_dtype=F32), reference(x, w, **call, out_dtype=F32))


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 40, 777, 4096])
def test_rank_values_past_bf16_are_infinite(device, m):
    """255 * 2^57 times 2^63 + 2^55 is (1 - 2^-16) 2^128: finite in FP32 and above (1 - 2^-9) 2^128, from where bf16 rounds
    to an infinity. The row is infinite, not NaN; the others are as they were."""
    announce("adapter past bf16", m)
    k, n, rank = 64, 2048, 16
    x = torch.zeros((m, k), dtype=BF16, device=device)
    x[0, :2], x[1:, 2] = 255 * 2.0**57, 1.0
    w = torch.zeros((n, k), dtype=BF16, device=device)
    down = torch.zeros((2, rank, k), dtype=BF16, device=device)
    down[0, 0, 0], down[0, 0, 1], down[:, :, 2] = 2.0**63, 2.0**55, 1.0
    up = torch.full((2, n, rank), 0.5, dtype=BF16, device=device)
    adapter = (torch.arange(m, device=device) % 2).int()
    got = ops.adapter_linear(x, w, down, up, adapter)
    assert (got[0] == float("inf")).all()
    assert (got[1:] == rank / 2).all()


@pytest.mark.gpu
def test_stacks_past_4_gib(device):
    """An adapter whose factors lie past 4 GiB, and rows of one that are 8 MiB apart."""
    announce("adapter far stacks")
    n, k, rank = 72, 264, 16
    made = stacks(3, rank, n, k)

    def spread(source, stride, row_stride):
        adapters, rows, columns = source.shape
        far = torch.empty((adapters - 1) * stride + (rows - 1) * row_stride + columns, dtype=BF16, device=device)
        return far.as_strided(source.shape, (stride, row_stride, 1)).copy_(source)

    for m in (2, 40, 300):
        x, w, adapter = normal((m, k), 1), normal((n, k), 2, 0.05), each_other(m, 3)
        want = reference(x, w, **made, adapter=adapter)
        far = (1 << 31) + 64
        got = ops.adapter_linear(x, w, spread(made["down"], far, k), spread(made["up"], far, rank), adapter, scales=made["scales"])
        assert_near(got, want, "far adapters")
        wide = 1 << 22
        got = ops.adapter_linear(x, w, spread(made["down"], rank * wide, wide), spread(made["up"], n * wide, wide), adapter, scales=made["scales"])
        assert_near(got, want, "far rows")


@pytest.mark.gpu
@pytest.mark.parametrize("m, n, k", [(1, 512, 1024), (60, 256, 1024), (640, 512, 512)])
@pytest.mark.parametrize("gated", [False, True])
def test_results_repeat_and_rows_do_not_depend_on_the_others(device, m, n, k, gated):
    announce("adapter repeats", m, n, k, gated)
    halves = 2 if gated else 1
    entry = ops.adapter_gated_linear if gated else ops.adapter_linear
    x, w = normal((m, k), 1), normal((n * halves, k), 2, 0.05)
    call = dict(stacks(9, 16, n, k, halves=halves), adapter=each_other(m, 9))
    other = normal((1024, 1024), 3)
    first = entry(x, w, **call)
    for _ in range(3):
        ops.linear(other, other)
        assert torch.equal(entry(x, w, **call), first)
    x[0], call["adapter"][0] = 0, 3
    assert torch.equal(entry(x, w, **call)[1:], first[1:])


@pytest.mark.gpu
def test_streams_and_captured_replays(device):
    """Two streams at once, a workspace each; a graph of two products that share one, replayed with other rows and
    other adapters of theirs."""
    announce("adapter streams and graphs")
    k, i, n, m = 256, 192, 256, 48
    x, up_gate, weight = normal((m, k), 1), normal((2 * i, k), 2, 0.05), normal((n, i), 3, 0.05)
    first, second = stacks(7, 16, i, k, halves=2), stacks(7, 8, n, i, seed=60)
    adapter = each_other(m, 7)
    workspace = torch.empty(max(ops.adapter_workspace(m, 32), ops.adapter_workspace(m, 8)), dtype=torch.uint8, device=device)

    def step(workspace=None):
        hidden = ops.adapter_gated_linear(x, up_gate, **first, adapter=adapter, workspace=workspace)
        return ops.adapter_linear(hidden, weight, **second, adapter=adapter, residual=x, workspace=workspace)

    want = step()
    torch.cuda.synchronize()
    sides, got = [torch.cuda.Stream(), torch.cuda.Stream()], []
    for _ in range(4):
        for side in sides:
            with torch.cuda.stream(side):
                got.append(step())
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)
    side, graph = sides[0], torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        step(workspace)
        side.synchronize()
        with torch.cuda.graph(graph, stream=side):
            captured = step(workspace)
    torch.cuda.current_stream().wait_stream(side)
    for seed in (10, 11, 12):
        x.copy_(normal((m, k), seed))
        adapter.copy_(each_other(m, 7, seed))
        graph.replay()
        torch.cuda.synchronize()
        replayed = captured.clone()
        assert torch.equal(step(), replayed)
        torch.cuda.synchronize()


@pytest.mark.gpu
def test_no_rows(device):
    empty, index = torch.empty((0, 64), dtype=BF16, device=device), torch.empty(0, dtype=torch.int32, device=device)
    assert ops.adapter_linear(empty, normal((32, 64), 1), **stacks(2, 8, 32, 64), adapter=index).shape == (0, 32)
    assert ops.adapter_gated_linear(empty, normal((32, 64), 1), **stacks(2, 8, 16, 64, halves=2), adapter=index).shape == (0, 16)


@pytest.mark.gpu
@pytest.mark.parametrize("arguments, says", [
    (dict(down="half"), "down"), (dict(down="rank"), "down"), (dict(down="flat"), "down"), (dict(down="count"), "down"),
    (dict(up="rows"), "up"), (dict(up="columns"), "up"), (dict(adapter="long"), "adapter"), (dict(adapter="short"), "adapter"),
    (dict(adapter="host"), "adapter"), (dict(scales="half"), "scales"), (dict(scales="short"), "scales"),
    (dict(workspace="host"), "workspace"), (dict(workspace="small"), "workspace"), (dict(activation="relu"), "activation"),
    (dict(residual="short"), "residual"),
])
def test_python_refusals_of_device_calls(device, arguments, says):
    made = {
        "down.half": lambda: normal((2, 8, 16), 1, dtype=F16), "down.rank": lambda: normal((2, 7, 16), 1),
        "down.flat": lambda: normal((8, 16), 1), "down.count": lambda: normal((3, 8, 16), 1),
        "up.rows": lambda: normal((2, 11, 8), 1), "up.columns": lambda: normal((2, 8, 12), 1).transpose(1, 2),
        "adapter.long": lambda: torch.zeros(4, dtype=torch.int64, device=device),
        "adapter.short": lambda: torch.zeros(3, dtype=torch.int32, device=device), "adapter.host": lambda: torch.zeros(4, dtype=torch.int32),
        "scales.half": lambda: normal((2,), 1), "scales.short": lambda: normal((1,), 1, dtype=F32),
        "workspace.host": lambda: torch.zeros(1024, dtype=torch.uint8),
        "workspace.small": lambda: torch.zeros(16, dtype=torch.uint8, device=device), "residual.short": lambda: normal((3, 12), 1),
    }
    call = dict(x=normal((4, 16), 1), weight=normal((12, 16), 2), down=normal((2, 8, 16), 3), up=normal((2, 12, 8), 4),
                adapter=torch.zeros(4, dtype=torch.int32, device=device))
    call.update({k: made[f"{k}.{v}"]() if f"{k}.{v}" in made else v for k, v in arguments.items()})
    with pytest.raises((ValueError, RuntimeError), match=says):
        ops.adapter_linear(**call)
