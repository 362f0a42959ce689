"""token_experts: refusals on the CPU, and on the MI355X against the formula in 64 bits.

Tolerance, element by element, with u = 2^-24. The first product's halves are off by 2 (H + 1) u S, S = sum |x w| of the
half; the gate and the product of the halves as in test_linear's gated products (slope 1.13, 128 u). The gated
value h, off by d so far, is then held as a pair of elements: half a step of the second of at most half a step of h,
2^-18 of |h| + d (bf16; subnormal steps from 2^-134) or 2^-24 of it and 2^-19 (f16: pairs at 2^-6 of the value, whose second
element's steps end at 2^-24). The second product adds sum d |w| and, over the values and the errors, 2 (2 I + 2) u of
sum (|h| + d) |w|; a route's weight u, and the additions over routes, wavefronts and the residual
(top + 6) u of the sum of their sizes. Last the output's rounding.
"""

import ctypes

import pytest
import torch

import test_expert_topk
from gpu_helpers import announce, assert_as_the_formula, kernels_of
from test_linear import BF16, F16, F32, U, activated, assert_near, normal, rounding
from uniserve_moe import abi, ops


def reference(x, ids, weights, up_gate, down, activation="silu", residual=None, first=0):
    """The output in 64 bits and how far the kernels may be from it, both on the CPU."""
    dtype = x.dtype
    x, weights, ids = x.double().cpu(), weights.double().cpu(), ids.cpu().long() - first
    tokens, hidden = x.shape
    experts, width = up_gate.shape[0], up_gate.shape[1] // 2
    y, size, off = (torch.zeros(tokens, hidden, dtype=torch.float64) for _ in range(3))
    for e in range(experts):
        rows, places = torch.nonzero(ids == e, as_tuple=True)
        if rows.numel() == 0:
            continue
        w1, w2 = up_gate[e].double().cpu(), down[e].double().cpu()
        both, s = x[rows] @ w1.t(), x[rows].abs() @ w1.abs().t()
        d = 2 * (hidden + 1) * U * s
        up, gate = both[:, :width], both[:, width:]
        act = activated(gate, activation)
        h = up * act
        d = act.abs() * d[:, :width] + 1.13 * d[:, width:] * (up.abs() + d[:, :width]) + 128 * U * h.abs()
        if dtype == BF16:
            d = d + 2.0**-18 * (h.abs() + d) + 2.0**-134
        else:
            d = d + 2.0**-24 * (h.abs() + d) + 2.0**-19
        w = weights[rows, places][:, None]
        part, wide = (h.abs() + d) @ w2.abs().t(), h @ w2.t()
        y.index_add_(0, rows, w * wide)
        size.index_add_(0, rows, w.abs() * part)
        off.index_add_(0, rows, w.abs() * (d @ w2.abs().t() + (2 * (2 * width + 2) + 2) * U * part))
    if residual is not None:
        r = residual.double().cpu()
        y, size = y + r, size + r.abs()
    off = off + (ids.shape[1] + 6) * U * size
    return y, off + rounding(y.abs() + off, dtype)


# ---- without a GPU ----------------------------------------------------------------------------------


def filled_call():
    call = abi.TokenExpertsCall()
    call.input, call.ids, call.weights, call.up_gate, call.down = 1 << 20, 2 << 20, 3 << 20, 4 << 20, 5 << 20
    call.out, call.workspace, call.workspace_bytes = 6 << 20, 7 << 20, 1 << 19
    call.tokens, call.top, call.hidden, call.width, call.experts = 4, 2, 64, 32, 8
    call.input_row_stride = call.residual_row_stride = call.out_row_stride = 64
    call.dtype, call.activation = abi.DTYPE["bf16"], 0
    return call


REFUSED = [
    ({"tokens": -1}, "positive"), ({"top": 0}, "positive"), ({"hidden": 0}, "positive"), ({"width": -3}, "positive"), ({"experts": 0}, "positive"),
    ({"tokens": 65}, "up to 64"), ({"top": 33}, "up to 64"), ({"experts": 1025}, "up to 64"), ({"hidden": 1 << 24}, "2^24"), ({"width": 1 << 24}, "2^24"),
    ({"dtype": abi.DTYPE["f32"]}, "bf16 or f16"), ({"activation": -1}, "gelu_tanh"), ({"activation": 2}, "gelu_tanh"),
    ({"first_expert": -1}, "first expert"), ({"first_expert": 2**31 - 8}, "first expert"),
    ({"input": None}, "needs"), ({"ids": None}, "needs"), ({"weights": None}, "needs"), ({"up_gate": None}, "needs"), ({"down": None}, "needs"),
    ({"out": None}, "needs"), ({"workspace": None}, "needs"),
    ({"input_row_stride": 63}, "strides"), ({"out_row_stride": 63}, "strides"), ({"residual": 9 << 20, "residual_row_stride": 1}, "strides"),
    ({"out_row_stride": 1 << 60}, "too large"), ({"hidden": (1 << 24) - 1, "width": (1 << 24) - 1, "input_row_stride": 1 << 24, "out_row_stride": 1 << 24}, "too large"),
    ({"workspace_bytes": 16 + 8 * (16 + 256) - 1}, "workspace of"), ({"workspace": (7 << 20) + 8}, "aligned"),
    ({"out": 1 << 20}, "output overlaps"), ({"out": 2 << 20}, "output overlaps"), ({"out": (3 << 20) + 16}, "output overlaps"),
    ({"out": (4 << 20) + 64}, "output overlaps"), ({"out": (5 << 20) - 32}, "output overlaps"),
    ({"workspace": 1 << 20}, "workspace overlaps one"), ({"workspace": 2 << 20}, "workspace overlaps one"), ({"workspace": 5 << 20}, "workspace overlaps one"),
    ({"workspace": 6 << 20}, "its output"), ({"residual": (7 << 20) + 64}, "its output"), ({"residual": (6 << 20) + 2}, "in part"),
    ({"residual": 6 << 20, "residual_row_stride": 72}, "in part"),
]


@pytest.mark.parametrize("fields, says", REFUSED)
def test_refusals(fields, says):
    call = filled_call()
    for name, value in fields.items():
        setattr(call, name, value)
    assert abi.library().uniserve_token_experts(ctypes.byref(call), None) != 0
    assert says in call.error.decode()


@pytest.mark.parametrize("fields", [{"tokens": 1, "input_row_stride": -1, "out_row_stride": 1 << 60}, {"residual_row_stride": -1}])
def test_unused_strides_are_not_read(fields):
    call = filled_call()
    for name, value in {**fields, "workspace": 6 << 20}.items():
        setattr(call, name, value)
    assert abi.library().uniserve_token_experts(ctypes.byref(call), None) != 0
    assert "its output" in call.error.decode()


def test_no_rows_launch_nothing():
    call = filled_call()
    call.tokens, call.input, call.out, call.ids, call.workspace = 0, None, None, None, None
    assert abi.library().uniserve_token_experts(ctypes.byref(call), None) == 0
    assert abi.library().uniserve_token_experts(None, None) != 0


def test_workspace_sizes():
    size = ops.token_experts_workspace
    assert size(1, 1, 1) == 16 + 16 + 256 and size(4, 2, 64) == 16 + 8 * (16 + 256) and size(64, 8, 768) == 16 + 512 * (16 + 4 * 768)
    assert size(0, 8, 64) == 0 and size(65, 8, 64) == 0 and size(4, 33, 64) == 0


def test_python_refusals():
    with pytest.raises(ValueError, match="on a GPU"):
        ops.token_experts(torch.zeros(1, 8, dtype=BF16), torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, 1),
                          torch.zeros(1, 8, 8, dtype=BF16), torch.zeros(1, 8, 4, dtype=BF16))


# ---- on the MI355X ----------------------------------------------------------------------------------


def inputs(tokens, hidden, width, experts, top, dtype=BF16, seed=0):
    g = torch.Generator().manual_seed(seed)
    ids = torch.rand(tokens, experts, generator=g).argsort(1)[:, :top].int().cuda()
    weights = torch.rand(tokens, top, generator=g).add_(0.05).cuda()
    return dict(x=normal((tokens, hidden), seed + 1, dtype=dtype), ids=ids, weights=weights,
                up_gate=normal((experts, 2 * width, hidden), seed + 2, 0.05, dtype),
                down=normal((experts, hidden, width), seed + 3, 0.05, dtype))


#: tokens, hidden, width, experts, top: single ones, odd extents, whole lines and their remainders, few and many experts.
SHAPES = [(1, 1, 1, 1, 1), (1, 2048, 768, 16, 8), (1, 64, 64, 4, 2), (2, 72, 40, 5, 3), (3, 100, 33, 7, 7), (5, 256, 704, 8, 6),
          (7, 520, 136, 64, 8), (15, 1000, 72, 3, 2), (16, 128, 128, 16, 4), (17, 130, 65, 2, 1), (31, 264, 192, 128, 8),
          (33, 64, 256, 300, 5), (64, 512, 128, 128, 8), (64, 96, 320, 1, 1), (64, 200, 64, 2, 2), (48, 128, 96, 1024, 32), (64, 64, 63, 40, 32),
          (4, 2120, 72, 6, 2), (20, 2051, 64, 8, 2), (64, 2056, 40, 6, 2), (3, 4100, 193, 9, 4), (64, 2600, 72, 64, 4)]


@pytest.mark.gpu
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dtype, activation", [(BF16, "silu"), (F16, "gelu_tanh"), (BF16, "gelu_tanh"), (F16, "silu")])
def test_token_experts(device, shape, dtype, activation):
    announce("token_experts", shape, dtype, activation)
    call = inputs(*shape, dtype)
    assert_near(ops.token_experts(**call, activation=activation), reference(**call, activation=activation))
    call["residual"] = normal((shape[0], shape[1]), 9, dtype=dtype)
    want = reference(**call, activation=activation)
    assert_near(ops.token_experts(**call, activation=activation), want, "residual")
    over = call["residual"]
    assert ops.token_experts(**call, activation=activation, out=over) is over
    assert_near(over, want, "in place")


@pytest.mark.gpu
@pytest.mark.parametrize("tokens, experts", [(1, 9), (6, 16), (40, 12), (64, 8)])
def test_windows_absent_routes_and_repeated_ids(device, tokens, experts):
    """A rank's window of the experts; ids of -1, beyond the window and at int32's ends; an id several times in a row;
    rows that route nowhere, which are the residual or zeros."""
    announce("token_experts windows", tokens, experts)
    call = inputs(tokens, 136, 72, experts, 6)
    g = torch.Generator().manual_seed(5)
    call["ids"] = torch.randint(90, 110 + experts, (tokens, 6), generator=g).int().cuda()
    call["ids"][:, 2] = call["ids"][:, 4]
    call["ids"][0, 1], call["ids"][-1, 3] = -1, 100
    if tokens > 4:
        call["ids"][1] = torch.tensor([-1, -2**31, 2**31 - 1, 99, 100 + experts, -7], dtype=torch.int32)
        call["ids"][2] = 100 + experts - 1
    call["weights"][call["ids"] < 100] = float("nan")
    call["weights"][call["ids"] >= 100 + experts] = float("inf")
    want = reference(**{**call, "weights": call["weights"].nan_to_num(0.0, 0.0)}, first=100)
    got = ops.token_experts(**call, first=100)
    assert_near(got, want)
    if tokens > 4:
        assert (got[1] == 0).all()
    residual = normal((tokens, 136), 8)
    got = ops.token_experts(**call, first=100, residual=residual)
    if tokens > 4:
        assert torch.equal(got[1], residual[1])
    nowhere = dict(call, ids=torch.full_like(call["ids"], -1))
    assert torch.equal(ops.token_experts(**nowhere, residual=residual), residual)
    assert (ops.token_experts(**nowhere) == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [17, 33, 64])
def test_one_expert_of_many_tokens(device, tokens):
    """Every token names the same experts: runs of sixteen, and the last one's rest."""
    announce("token_experts runs", tokens)
    call = inputs(tokens, 256, 128, 6, 2)
    call["ids"][:] = torch.tensor([4, 1], dtype=torch.int32)
    assert_near(ops.token_experts(**call), reference(**call))


@pytest.mark.gpu
@pytest.mark.parametrize("shift", [0, 1, 8])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_strides_and_alignments(device, shift, dtype):
    announce("token_experts strides", shift, dtype)
    tokens, hidden, width = 6, 136, 72
    call = inputs(tokens, hidden, width, 8, 3, dtype)

    def inside(source, fill=float("nan")):
        buffer = torch.full((source.shape[0] + 2, hidden + 24), fill, dtype=dtype, device=device)
        return buffer, buffer[1:-1, shift:shift + hidden].copy_(source)

    def shifted(source):
        flat = torch.full((source.numel() + 16,), float("nan"), dtype=dtype, device=device)
        return flat[shift:shift + source.numel()].view(source.shape).copy_(source)

    residual = normal((tokens, hidden), 9, dtype=dtype)
    want = reference(**call, residual=residual)
    around, out = inside(residual, 7.0)
    ops.token_experts(inside(call["x"])[1], call["ids"], call["weights"], shifted(call["up_gate"]), shifted(call["down"]),
                      residual=inside(residual)[1], out=out)
    assert_near(out, want)
    out.fill_(7.0)
    assert (around == 7.0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [2, 20, 64])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_infinities_and_nans_stay_with_their_rows(device, tokens, dtype):
    """A row's, and an expert's: only rows routed to it. What the workspace held before does not matter."""
    announce("token_experts non-finite", tokens, dtype)
    call = inputs(tokens, 136, 70, 6, 2, dtype)
    call["ids"][0] = torch.tensor([0, 1], dtype=torch.int32)
    call["ids"][1:] = torch.randint(1, 5, (tokens - 1, 2), generator=torch.Generator().manual_seed(3)).int().cuda()
    workspace = torch.full((ops.token_experts_workspace(tokens, 2, 70),), 255, dtype=torch.uint8, device=device)
    want = ops.token_experts(**call, workspace=workspace)
    call["up_gate"][0], call["down"][5] = float("nan"), float("inf")
    call["down"][0, 3], call["x"][0] = float("inf"), float("inf")
    got = ops.token_experts(**call, workspace=workspace.fill_(255))
    assert torch.equal(got[1:], want[1:]) and torch.isnan(got[0]).all()
    call["up_gate"][4, 3, 5] = float("nan")
    got = ops.token_experts(**call)
    touched = (call["ids"] == 4).any(1)
    touched[0] = True
    assert torch.equal(got[~touched], want[~touched]) and torch.isnan(got[touched]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [1, 3, 7, 20, 64])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("exact", [False, True])
def test_infinite_weights_give_the_formula_s_infinities(device, tokens, dtype, exact):
    """One infinity in a row of `down` is an infinity of the gated value's sign, two that oppose are NaN; gated values that
    one element holds (of which nothing is left for the pair's other one), and any."""
    announce("token_experts infinite weights", tokens, dtype, exact)
    call = inputs(tokens, 136, 70, 6, 2, dtype)
    if exact:  # up 1, -1 or 2, gate 64: gelu_tanh(64) is 64
        call["x"].zero_()[:, 0] = torch.tensor([1.0, -1.0, 2.0], dtype=dtype, device=device).repeat(22)[:tokens]
        call["x"][:, 1] = 64.0
        call["up_gate"][:] = 0
        call["up_gate"][:, :70, 0] = 1.0
        call["up_gate"][:, 70:, 1] = 1.0
    call["activation"] = "gelu_tanh"
    want = ops.token_experts(**call)
    inf = float("inf")
    call["down"][:, 5, 7], call["down"][:, 9, 64], call["down"][3, 135, 69] = inf, -inf, inf
    call["down"][:, 11], call["down"][2, 20, 3] = inf, float("nan")
    call["down"][:, 12, :2] = torch.tensor([inf, -inf], dtype=dtype)
    got = ops.token_experts(**call)
    y = reference(**call)[0]
    assert_as_the_formula(got, y)
    assert not torch.isfinite(y[:, [5, 9, 11, 12]]).any() and torch.isinf(y[:, [5, 9]]).any()
    finite = torch.isfinite(y).to(device)
    assert torch.equal(got[finite], want[finite])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("tokens", [3, 7, 16])
def test_gated_values_past_their_pairs_are_infinite(device, tokens, dtype):
    """Finite in FP32, an infinity in the pair's element: up times gate is 2^24 (f16 pairs reach 2^22) or, in bf16,
    nearly 2^128. The row is infinite, not NaN; the others are as they were."""
    announce("token_experts past the pairs", tokens, dtype)
    hidden, width, experts = 64, 72, 2
    x = torch.zeros((tokens, hidden), dtype=dtype, device=device)
    # (silu(g) is g in FP32 for these gates. bf16: 255 * 2^57 times 2^63 + 2^55 is (1 - 2^-16) 2^128, finite, and above
    # (1 - 2^-9) 2^128, from where bf16 rounds to an infinity.)
    up, gates = ((4096.0, 0.0), (4096.0, 0.0)) if dtype == F16 else ((255 * 2.0**57, 0.0), (2.0**63, 2.0**55))
    x[0, :2], x[1:, 2] = 1.0, 1.0
    up_gate = torch.zeros((experts, 2 * width, hidden), dtype=dtype, device=device)
    up_gate[:, :width, 0], up_gate[:, :width, 1] = up
    up_gate[:, width:, 0], up_gate[:, width:, 1] = gates
    up_gate[:, :, 2] = 1.0
    down = torch.full((experts, hidden, width), 0.5, dtype=dtype, device=device)
    ids = (torch.arange(tokens, device=device) % 2).int()[:, None].contiguous()
    call = dict(ids=ids, weights=torch.ones((tokens, 1), device=device), up_gate=up_gate, down=down)
    got = ops.token_experts(x, **call)
    assert (got[0] == float("inf")).all()
    plain = x.clone()
    plain[0] = plain[1]
    assert torch.equal(got[1:], ops.token_experts(plain, **call)[1:]) and got[1:].isfinite().all()


@pytest.mark.gpu
def test_large_gated_values_of_f16(device):
    """Gated values beyond f16's largest number, which the down product brings back."""
    announce("token_experts f16 range")
    call = inputs(5, 64, 64, 4, 2, F16)
    call["up_gate"] *= 200.0
    call["down"] *= 2.0**-10
    assert_near(ops.token_experts(**call), reference(**call))


def reference_of_f16(x, ids, weights, up_gate, down, activation="silu"):
    """The output in 64 bits and how far the f16 kernels may be from it, by the tolerance above but for the gated values: a
    line's (64 of a route) are FP32 until they are split into two elements, by a power of two that brings the line's
    largest to [1, 2). The first element leaves at most 2^-11 of a value, the second is off by half a step of that, 2^-23
    of the value, or by half a subnormal step, 2^-25 of at most the line's largest. A line's products are scaled back,
    2 u, and added: the 2 (2 I + 2) u hold that many additions twice."""
    x, weights, ids = x.double().cpu(), weights.double().cpu(), ids.cpu().long()
    tokens, hidden = x.shape
    experts, width = up_gate.shape[0], up_gate.shape[1] // 2
    y, size, off = (torch.zeros(tokens, hidden, dtype=torch.float64) for _ in range(3))
    for e in range(experts):
        rows, places = torch.nonzero(ids == e, as_tuple=True)
        if rows.numel() == 0:
            continue
        w1, w2 = up_gate[e].double().cpu(), down[e].double().cpu()
        both, s = x[rows] @ w1.t(), x[rows].abs() @ w1.abs().t()
        d = 2 * (hidden + 1) * U * s
        up, gate = both[:, :width], both[:, width:]
        act = activated(gate, activation)
        h = up * act
        d = act.abs() * d[:, :width] + 1.13 * d[:, width:] * (up.abs() + d[:, :width]) + 128 * U * h.abs()
        most = torch.cat([line.amax(1, keepdim=True).expand_as(line) for line in (h.abs() + d).split(64, 1)], 1)
        d = d + 2.0**-23 * (h.abs() + d) + 2.0**-25 * most
        w = weights[rows, places][:, None]
        part = (h.abs() + d) @ w2.abs().t()
        y.index_add_(0, rows, w * (h @ w2.t()))
        size.index_add_(0, rows, w.abs() * part)
        off.index_add_(0, rows, w.abs() * (d @ w2.abs().t() + (2 * (2 * width + 2) + 4) * U * part))
    off = off + (ids.shape[1] + 6) * U * size
    return y, off + rounding(y.abs() + off, F16)


@pytest.mark.gpu
@pytest.mark.parametrize("tokens, experts", [(1, 8), (4, 8), (8, 8), (16, 8), (40, 8), (64, 128)])
@pytest.mark.parametrize("size", [2.0**-12, 2.0**-8, 2.0**-5, 2.0**-2, 2.0**2, 2.0**6])
def test_f16_gated_values_of_any_size(device, tokens, experts, size):
    """Gated values from some 2^-26 to some 2^20, lines of one size and of many, brought to ordinary outputs by `down`."""
    announce("token_experts f16 sizes", tokens, experts, size)
    call = inputs(tokens, 264, 200, experts, 4, F16)
    call["x"] = (call["x"].float() * size).to(F16)
    h = reference_of_f16(**{**call, "down": torch.eye(200, dtype=F16).repeat(2, 1)[None, :264].expand(experts, -1, -1)})[0]
    call["down"] = (call["down"].float() / (0.05 * h.abs().mean().item() * 8)).clamp(-60000, 60000).to(F16)
    got, want = ops.token_experts(**call), reference_of_f16(**call)
    assert 2.0**-8 < want[0].abs().mean() < 2.0**12
    assert_near(got, want, "one size")
    up_gate = call["up_gate"].float()
    up_gate[:, :200] *= 2.0 ** -(torch.arange(200, device=device) * 7 % 13).float()[:, None]
    call["up_gate"] = up_gate.to(F16)
    assert_near(ops.token_experts(**call), reference_of_f16(**call), "many sizes")


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [1, 12, 64])
def test_results_repeat_and_rows_do_not_depend_on_the_others(device, tokens):
    announce("token_experts repeats", tokens)
    call = inputs(tokens, 512, 192, 24, 4)
    first = ops.token_experts(**call)
    other = normal((1024, 1024), 3)
    for _ in range(3):
        ops.linear(other, other)
        assert torch.equal(ops.token_experts(**call), first)
    row = tokens // 2
    alone = {**call, **{k: call[k][row:row + 1].contiguous() for k in ("x", "ids", "weights")}}
    assert torch.equal(ops.token_experts(**alone)[0], first[row])


@pytest.mark.gpu
@pytest.mark.parametrize("tokens, experts", [(4, 24), (12, 24), (40, 8), (64, 24)])
def test_f16_rows_do_not_depend_on_the_others(device, tokens, experts):
    """Jobs of 4, 8 and 16 tokens, and the row alone: the same bits."""
    announce("token_experts f16 rows", tokens, experts)
    call = inputs(tokens, 512, 200, experts, 4, F16)
    call["x"] *= 2.0 ** -(torch.arange(tokens, device=device) % 9)[:, None]
    together = ops.token_experts(**call)
    assert torch.equal(ops.token_experts(**call), together)
    for row in range(0, tokens, 3):
        alone = {**call, **{k: call[k][row:row + 1].contiguous() for k in ("x", "ids", "weights")}}
        assert torch.equal(ops.token_experts(**alone)[0], together[row]), row


@pytest.mark.gpu
def test_two_kernels(device):
    announce("token_experts kernels")
    call = inputs(8, 256, 128, 16, 4)
    out, workspace = torch.empty_like(call["x"]), torch.empty(ops.token_experts_workspace(8, 4, 128), dtype=torch.uint8, device=device)
    names = kernels_of(lambda: ops.token_experts(**call, out=out, workspace=workspace))
    assert len(names) == 2 and "gate_up_kernel" in names[0] and "down_kernel" in names[1], names


@pytest.mark.gpu
def test_stacks_past_4_gib(device):
    announce("token_experts far stacks")
    hidden, width, experts = 2048, 768, 500
    call = dict(x=normal((3, hidden), 1), ids=torch.tensor([[499, 0], [498, 499], [250, -1]], dtype=torch.int32, device=device),
                weights=torch.rand(3, 2, generator=torch.Generator().manual_seed(1)).cuda(),
                up_gate=torch.empty((experts, 2 * width, hidden), dtype=BF16, device=device),
                down=torch.empty((experts, hidden, width), dtype=BF16, device=device))
    for e in (0, 250, 498, 499):
        call["up_gate"][e], call["down"][e] = normal((2 * width, hidden), e, 0.05), normal((hidden, width), e + 1, 0.05)
    got = ops.token_experts(**call)
    kept = [0, 250, 498, 499]
    few = dict(call, ids=torch.tensor([[3, 0], [2, 3], [1, -1]], dtype=torch.int32), up_gate=call["up_gate"][kept], down=call["down"][kept])
    assert_near(got, reference(**few))


@pytest.mark.gpu
def test_with_its_router_and_norms_captured(device):
    """A decode step around an MoE block as a serving program runs it: the norm before it, logits, choice, experts for
    few tokens onto a shared expert with adapters, and the join and norm behind it - against the block by the sorted
    operators, and replayed from a graph."""
    announce("token_experts in a step")
    tokens, hidden, width, experts, top, shared = 12, 512, 128, 32, 4, 192
    made = inputs(tokens, hidden, width, experts, top)
    router, bias = normal((experts, hidden), 11, 0.05), test_expert_topk.bias_of(experts, 8).to(device)
    shared_up, shared_down = normal((2 * shared, hidden), 12, 0.05), normal((hidden, shared), 13, 0.05)
    down_factor, up_factor = normal((3, 2 * 8, hidden), 14, 0.05), normal((3, 2 * shared, 8), 15, 0.05)
    adapter = (torch.arange(tokens) % 4 - 1).int().to(device)
    norms = [normal((hidden,), seed, 0.1) for seed in (16, 17)]
    stream = normal((tokens, hidden), 18, 1.0, F32)
    block = made["x"]

    def step(few):
        x, total = ops.add_norm(block, norms[0], residual=stream, offset=1.0)
        logits = ops.linear(x, router, out_dtype=F32)
        ids, weights = ops.expert_topk(logits, top, bias=bias, groups=4, top_groups=2, factor=2.5)
        mlp = ops.adapter_gated_linear(x, shared_up, down_factor, up_factor, adapter)
        joined = ops.linear(mlp, shared_down)
        if few:
            joined = ops.token_experts(x, ids, weights, made["up_gate"], made["down"], residual=joined, out=joined)
        else:
            maps = ops.moe_sort(ids, weights, experts)
            gated = ops.gather_gemm(x, made["up_gate"], top, maps, ops.permuted_rows(tokens, top, experts))
            routed = ops.moe_unpermute(ops.route_gemm(gated, made["down"], maps), maps[ops.EXPANDED_TO_PERMUTED], weights)
            joined = joined + routed
        return ops.add_norm(joined, norms[1], residual=total, post=norms[0], offset=1.0)

    (out, total), (sorted_out, sorted_total) = step(True), step(False)
    # bf16 roundings of the sorted path's gated rows, products, sum and join, each 2^-8 of what it rounds at most.
    for got, want in ((out, sorted_out), (total, sorted_total)):
        assert (got.double() - want.double()).abs().max() <= 2.0**-5 * want.double().abs().max()
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(True)
        side.synchronize()
        with torch.cuda.graph(graph, stream=side):
            captured = step(True)
    torch.cuda.current_stream().wait_stream(side)
    for seed in (20, 21, 22):
        block.copy_(normal((tokens, hidden), seed))
        graph.replay()
        torch.cuda.synchronize()
        replayed = [t.clone() for t in captured]
        assert all(torch.equal(a, b) for a, b in zip(step(True), replayed))
        torch.cuda.synchronize()


@pytest.mark.gpu
def test_two_streams(device):
    announce("token_experts streams")
    calls = [inputs(tokens, 512, 128, 32, 4, seed=tokens) for tokens in (1, 40)]
    want = [ops.token_experts(**c) for c in calls]
    torch.cuda.synchronize()
    sides, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for _ in range(4):
        for i, side in enumerate(sides):
            with torch.cuda.stream(side):
                got[i].append(ops.token_experts(**calls[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[i]) for i in range(2) for g in got[i])


@pytest.mark.gpu
def test_no_rows(device):
    call = inputs(1, 64, 32, 4, 2)
    for name in ("x", "ids", "weights"):
        call[name] = call[name][:0]
    assert ops.token_experts(**call).shape == (0, 64)


@pytest.mark.gpu
@pytest.mark.parametrize("arguments, says", [
    (dict(ids="long"), "ids"), (dict(ids="flat"), "ids"), (dict(ids="host"), "ids"), (dict(weights="half"), "weights"), (dict(weights="short"), "weights"),
    (dict(weights="columns"), "weights"), (dict(up_gate="odd"), "up_gate"), (dict(up_gate="half"), "up_gate"), (dict(up_gate="strided"), "up_gate"),
    (dict(down="short"), "down"), (dict(activation=None), "activation"), (dict(residual="wide"), "residual"), (dict(out="wide"), "output"),
    (dict(out="short"), "output"), (dict(workspace="host"), "workspace"), (dict(workspace="small"), "workspace"), (dict(first=-1), "first"), (dict(x="many"), "up to 64"),
])
def test_python_refusals_of_device_calls(device, arguments, says):
    made = {
        "ids.long": lambda: torch.zeros((4, 2), dtype=torch.int64, device=device), "ids.flat": lambda: torch.zeros(8, dtype=torch.int32, device=device),
        "ids.host": lambda: torch.zeros((4, 2), dtype=torch.int32), "weights.half": lambda: normal((4, 2), 1),
        "weights.short": lambda: normal((3, 2), 1, dtype=F32), "weights.columns": lambda: normal((2, 4), 1, dtype=F32).t(),
        "up_gate.odd": lambda: normal((4, 31, 16), 1), "up_gate.half": lambda: normal((4, 32, 16), 1, dtype=F16),
        "up_gate.strided": lambda: normal((4, 64, 16), 1)[:, ::2], "down.short": lambda: normal((4, 15, 16), 1),
        "residual.wide": lambda: normal((4, 16), 1, dtype=F32), "out.wide": lambda: normal((4, 16), 1, dtype=F32),
        "out.short": lambda: normal((4, 15), 1), "workspace.host": lambda: torch.zeros(4096, dtype=torch.uint8),
        "workspace.small": lambda: torch.zeros(64, dtype=torch.uint8, device=device), "x.many": lambda: normal((65, 16), 1),
    }
    call = inputs(4, 16, 16, 4, 2)
    call.update({k: made[f"{k}.{v}"]() if f"{k}.{v}" in made else v for k, v in arguments.items()})
    if arguments.get("x"):
        call["ids"], call["weights"] = torch.zeros((65, 2), dtype=torch.int32, device=device), torch.zeros((65, 2), device=device)
    with pytest.raises((ValueError, RuntimeError), match=says):
        ops.token_experts(**call)
