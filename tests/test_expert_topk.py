"""expert_topk: its refusals on the CPU, and on the MI355X against the definition in 64 bits.

Ids are compared exactly. Scores, choices and group ranks are doubles on both sides, so two choices
would have to lie within a few 2^-53 of each other without being equal for the sides to order them
differently; the logits are drawn, and where choices are meant to tie their logits and biases are the
same values. Weights are the doubles rounded once into FP32: half a step, 2^-24 of the value, and a
few 2^-53 (WEIGHT below), or half of the smallest subnormal.
"""

import ctypes
import shutil
import subprocess
from pathlib import Path

import numpy as np
import pytest
import torch

from gpu_helpers import announce
from uniserve_moe import abi, ops

WEIGHT = 2.0**-24 * (1 + 2.0**-20)
TINY = 2.0**-150
INCLUDE = Path(__file__).resolve().parent.parent / "include"
BIG = float(np.finfo(np.float32).max)


def reference(logits, top, scoring="sigmoid", bias=None, groups=1, top_groups=1, group_top=2, renormalize=True,
              factor=1.0):
    """ids and weights (64 bits) of ``logits`` [T, E], row by row from the definition."""
    logits = np.asarray(logits, np.float64)
    tokens, experts = logits.shape
    bias = np.zeros(experts) if bias is None else np.asarray(bias, np.float64)
    ids, weights = np.full((tokens, top), -1, np.int32), np.zeros((tokens, top))
    size = experts // groups
    for t in range(tokens):
        l = np.minimum(logits[t], BIG)
        open_ = np.array([e for e in range(experts) if l[e] > -np.inf and bias[e] > -np.inf], dtype=int)
        score = np.zeros(experts)
        if len(open_):
            if scoring == "sigmoid":
                with np.errstate(over="ignore"):
                    score[open_] = 1.0 / (1.0 + np.exp(-l[open_]))
            else:
                powers = np.exp(l[open_] - l[open_].max())
                score[open_] = powers / powers.sum()
        choice = score + bias
        if groups > 1:
            ranks = []
            for g in range(groups):
                best = sorted((choice[e] for e in open_ if e // size == g), reverse=True)[:group_top]
                ranks.append(sum(best[1:], best[0]) if best else -np.inf)
            kept = sorted(range(groups), key=lambda g: (-ranks[g], g))[:top_groups]
            open_ = np.array([e for e in open_ if e // size in kept], dtype=int)
        picked = sorted(open_, key=lambda e: (-choice[e], e))[:top]
        total = sum(score[e] for e in picked)
        for j, e in enumerate(picked):
            ids[t, j] = e
            weights[t, j] = (score[e] if not renormalize else (score[e] / total if total > 0 else 0.0)) * factor
    return ids, weights


def assert_choice(got, want, what=""):
    ids, weights = got[0].cpu().numpy(), got[1].cpu().numpy().astype(np.float64)
    np.testing.assert_array_equal(ids, want[0], err_msg=what)
    off = np.abs(weights - want[1])
    assert (off <= WEIGHT * np.abs(want[1]) + TINY).all(), (what, off.max())


def logits_of(tokens, experts, dtype, seed, std=1.5):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn((tokens, experts), generator=g) * std).to(dtype)


def bias_of(experts, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(-100, 101, (experts,), generator=g).float() * 0.001


# ---- without a GPU ----------------------------------------------------------------------------------


def filled_call():
    call = abi.ExpertTopkCall()
    call.scores = call.ids = call.weights = 16
    call.row_stride, call.rows, call.experts, call.top = 64, 4, 64, 8
    call.groups, call.top_groups, call.group_top = 8, 4, 2
    call.score_dtype, call.scoring, call.renormalize, call.factor = abi.DTYPE["f32"], abi.SCORING["sigmoid"], 1, 1.0
    return call


@pytest.mark.parametrize("fields, says", [
    ({"experts": 0}, "1 to 1024 experts"),
    ({"experts": 1025, "row_stride": 1025, "groups": 1, "top_groups": 1}, "1 to 1024 experts"),
    ({"groups": 0}, "groups"), ({"groups": 7}, "equal size"), ({"groups": 128, "experts": 256, "row_stride": 256}, "groups"),
    ({"top_groups": 0}, "groups"), ({"top_groups": 9}, "groups"),
    ({"group_top": 0}, "best"), ({"group_top": 3}, "best"),
    ({"top": 0}, "picks"), ({"top": 33}, "picks"), ({"top_groups": 1, "top": 9}, "kept groups"),
    ({"score_dtype": abi.DTYPE["f8e4m3"]}, "f32, bf16 or f16"), ({"scoring": 2}, "softmax or sigmoid"),
    ({"factor": float("nan")}, "finite"), ({"factor": float("inf")}, "finite"),
    ({"rows": 1 << 26}, "rows in a call"), ({"row_stride": 1 << 60}, "too large"),
    ({"rows": -1}, "int32"), ({"rows": 1 << 29}, "int32"), ({"row_stride": 63}, "row stride"),
    ({"scores": None}, "needs scores"), ({"ids": None}, "needs scores"), ({"weights": None}, "needs scores"),
])
def test_refusals(fields, says):
    call = filled_call()
    for name, value in fields.items():
        setattr(call, name, value)
    assert abi.library().uniserve_expert_topk(ctypes.byref(call), None) != 0
    assert says in call.error.decode()


def test_no_rows_launch_nothing():
    call = filled_call()
    call.rows, call.scores, call.ids, call.weights = 0, None, None, None
    assert abi.library().uniserve_expert_topk(ctypes.byref(call), None) == 0
    assert abi.library().uniserve_expert_topk(None, None) != 0


def test_python_refusals():
    with pytest.raises(ValueError, match="on a GPU"):
        ops.expert_topk(torch.zeros(2, 8), 2)


@pytest.mark.parametrize("struct, mirror", [("uniserve_expert_topk_call", abi.ExpertTopkCall),
                                            ("uniserve_linear_call", abi.LinearCall)])
def test_structures_match_the_compiler(tmp_path, struct, mirror):
    compiler = shutil.which("g++") or shutil.which("c++")
    if compiler is None:
        pytest.skip("no host C++ compiler")
    lines = ["#include <cstddef>", "#include <cstdio>", '#include "uniserve_expert_topk.h"', '#include "uniserve_linear.h"',
             "int main() {", f'  std::printf("%zu\\n", sizeof({struct}));']
    lines += [f'  std::printf("%zu\\n", offsetof({struct}, {f[0]}));' for f in mirror._fields_] + ["}"]
    source = tmp_path / "layout.cpp"
    source.write_text("\n".join(lines) + "\n")
    subprocess.run([compiler, "-std=c++17", "-I", str(INCLUDE), str(source), "-o", str(tmp_path / "layout")], check=True)
    said = subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True, text=True).stdout.split()
    assert [int(s) for s in said] == [ctypes.sizeof(mirror)] + [getattr(mirror, f[0]).offset for f in mirror._fields_]


# ---- on the MI355X ----------------------------------------------------------------------------------

DTYPES = [torch.float32, torch.bfloat16, torch.float16]

CHOICES = [
    # experts, top, options
    (256, 8, dict(groups=8, top_groups=4, factor=2.5, bias=True)),
    (128, 8, dict(bias=True)),
    (160, 6, dict(scoring="softmax", groups=8, top_groups=3, group_top=1, renormalize=False, factor=16.0)),
    (1, 1, dict()),
    (7, 7, dict(bias=True)),
    (64, 32, dict(scoring="softmax", bias=True)),
    (65, 5, dict()),
    (130, 4, dict(groups=13, top_groups=2, bias=True)),
    (64, 3, dict(groups=64, top_groups=5, bias=True)),
    (63, 4, dict(groups=3, top_groups=3, group_top=1)),
    (511, 16, dict(groups=7, top_groups=1, bias=True)),
    (512, 9, dict(scoring="softmax", bias=True)),
    (1000, 12, dict(groups=8, top_groups=7)),
    (1024, 32, dict(bias=True, renormalize=False)),
    (1024, 1, dict(groups=64, top_groups=1, bias=True)),
]


@pytest.mark.gpu
@pytest.mark.parametrize("experts, top, options", CHOICES)
@pytest.mark.parametrize("tokens, dtype", [(1, torch.float32), (5, torch.bfloat16), (67, torch.float16), (301, torch.float32)])
def test_against_the_definition(device, experts, top, options, tokens, dtype):
    announce("expert_topk", tokens, dtype, experts, top, options)
    options = dict(options)
    bias = bias_of(experts, 7) if options.pop("bias", False) else None
    logits = logits_of(tokens, experts, dtype, experts + tokens)
    got = ops.expert_topk(logits.to(device), top, bias=None if bias is None else bias.to(device), **options)
    want = reference(logits.double().numpy(), top, bias=None if bias is None else bias.double().numpy(), **options)
    assert_choice(got, want)


#: 32 experts a lane (the most that a kernel holds, with their own error bound and slots), and sigmoid groups ranked by
#: their best expert.
WIDE = [(1023, 16, dict(groups=3, top_groups=2)), (1017, 8, dict(groups=9, top_groups=4)),
        (1010, 32, dict(groups=5, top_groups=1, group_top=1)), (1020, 5, dict(groups=17, top_groups=16, factor=2.5))]
BEST = [(96, 6, dict(groups=8, top_groups=3, group_top=1)), (160, 8, dict(groups=5, top_groups=2, group_top=1)),
        (60, 4, dict(groups=20, top_groups=7, group_top=1)), (12, 2, dict(groups=12, top_groups=3, group_top=1))]


@pytest.mark.gpu
@pytest.mark.parametrize("scoring", ["sigmoid", "softmax"])
@pytest.mark.parametrize("experts, top, options", WIDE + BEST)
def test_wide_groups_and_groups_by_their_best(device, scoring, experts, top, options):
    announce("expert_topk wide", scoring, experts, top, options)
    for seed, (dtype, biased, renormalize) in enumerate(((torch.float32, True, True), (torch.float32, False, False),
                                                         (torch.bfloat16, True, False), (torch.float16, False, True))):
        bias = bias_of(experts, seed) if biased else None
        logits = logits_of(60, experts, dtype, experts + seed)
        got = ops.expert_topk(logits.to(device), top, scoring=scoring, bias=None if bias is None else bias.to(device),
                              renormalize=renormalize, **options)
        want = reference(logits.double().numpy(), top, scoring=scoring, bias=None if bias is None else bias.double().numpy(),
                         renormalize=renormalize, **options)
        assert_choice(got, want, f"{dtype}, bias {biased}")


@pytest.mark.gpu
@pytest.mark.parametrize("scoring", ["sigmoid", "softmax"])
@pytest.mark.parametrize("experts, options", [(64, {}), (256, {}), (512, {}), (1024, {}), (256, dict(groups=8, top_groups=3)),
                                              (1023, dict(groups=3, top_groups=2)), (1017, dict(groups=9, top_groups=4))])
def test_biases_that_bring_choices_together(device, scoring, experts, options):
    """Biases that lift experts of unlike scores to one choice, but for the FP32 rounding of the bias: what orders
    them lies far below an FP32 score's error, of the softmax's sum included. Few experts, and every one."""
    announce("expert_topk lifted", scoring, experts, options)
    g = torch.Generator().manual_seed(experts + 1)
    base = torch.randn(experts, generator=g) * 2.0
    exact = torch.softmax(base.double(), 0) if scoring == "softmax" else torch.sigmoid(base.double())
    lifted = (1.0 - exact).float()
    few = torch.rand(experts, generator=g) < 24 / experts
    logits = base + torch.randint(-3, 4, (40, experts), generator=g) * 2.0**-22
    for bias in (torch.where(few, lifted, -1.0), lifted):
        got = ops.expert_topk(logits.to(device), 8, scoring=scoring, bias=bias.to(device), **options)
        assert_choice(got, reference(logits.numpy(), 8, scoring=scoring, bias=bias.numpy(), **options))


@pytest.mark.gpu
@pytest.mark.parametrize("scoring", ["sigmoid", "softmax"])
@pytest.mark.parametrize("groups", [1, 4])
def test_ties_go_to_the_lower_id(device, scoring, groups):
    """Rows of few distinct logits: experts tie within and across lanes, groups tie by their ranks."""
    announce("expert_topk ties", scoring, groups)
    g = torch.Generator().manual_seed(3)
    logits = torch.randint(-2, 3, (64, 96), generator=g).float() * 0.5
    logits[0] = 0.25
    logits[1] = 60.0  # every sigmoid is 1
    logits[2, 48:] = 60.0
    bias = torch.randint(0, 2, (96,), generator=g).float() * 0.5
    for b in (None, bias):
        options = dict(scoring=scoring, groups=groups, top_groups=max(1, groups // 2), group_top=2)
        got = ops.expert_topk(logits.to(device), 8, bias=None if b is None else b.to(device), **options)
        assert_choice(got, reference(logits.numpy(), 8, bias=None if b is None else b.numpy(), **options))


@pytest.mark.gpu
@pytest.mark.parametrize("scoring", ["sigmoid", "softmax"])
@pytest.mark.parametrize("groups", [1, 5])
@pytest.mark.parametrize("dtype", DTYPES)
def test_masked_infinite_and_nan_logits(device, scoring, groups, dtype):
    announce("expert_topk masks", scoring, groups, dtype)
    inf, nan = float("inf"), float("nan")
    logits = logits_of(12, 80, torch.float32, 5)
    logits[0] = -inf                       # an empty row
    logits[1] = nan
    logits[2] = -inf
    logits[2, 37] = -3.0                   # fewer candidates than top
    logits[3, ::2] = -inf
    logits[4, 1::3] = nan
    logits[5, 11] = logits[5, 70] = inf    # count as the largest finite float
    logits[6, :] = torch.finfo(dtype).min  # the lowest value is a candidate
    logits[7, 16:] = torch.finfo(dtype).min
    logits[8, 32:48] = -inf                # a group without candidates (groups of 16)
    logits[8, :15] = -inf                  # and one with a single one
    logits[9, 3], logits[9, 4], logits[9, 5] = inf, nan, -inf
    logits = logits.to(dtype)
    bias = bias_of(80, 9)
    bias[21], bias[22], bias[23] = -inf, nan, inf
    for b in (None, bias):
        options = dict(scoring=scoring, groups=groups, top_groups=max(1, groups - 2), renormalize=True)
        got = ops.expert_topk(logits.to(device), 8, bias=None if b is None else b.to(device), **options)
        assert torch.isfinite(got[1]).all()
        want = reference(logits.double().numpy(), 8, bias=None if b is None else b.double().numpy(), **options)
        assert_choice(got, want, f"bias {b is not None}")
    assert (got[0][0] == -1).all() and (got[1][0] == 0).all()


@pytest.mark.gpu
def test_choices_closer_than_fp32(device):
    """Neighbours whose sigmoids (plus bias) round to one float, ordered by the doubles."""
    announce("expert_topk near ties")
    base = np.float32(4.0)
    logits = np.full((32, 64), -2.0, np.float32)
    rng = np.random.default_rng(2)
    for t in range(32):
        places = rng.permutation(64)[:12]
        step = base
        for p in places:  # neighbouring floats: their sigmoids are 8e-9 apart, a quarter of an FP32 step
            logits[t, p] = step
            step = np.nextafter(step, np.float32(5.0))
    got = ops.expert_topk(torch.from_numpy(logits).to(device), 12)
    assert_choice(got, reference(logits, 12))
    single = 1.0 / (1.0 + np.exp(-logits[:, :].astype(np.float64)))
    assert len(np.unique(single[0].astype(np.float32))) < len(np.unique(single[0]))


@pytest.mark.gpu
@pytest.mark.parametrize("experts", [40, 64, 65, 256, 1000])
@pytest.mark.parametrize("distinct", [1, 2, 5, 40])
@pytest.mark.parametrize("options", [dict(), dict(scoring="softmax", renormalize=False), dict(top_groups=2)])
def test_few_distinct_logits(device, experts, distinct, options):
    """Ties within the picks, across their end and of more experts than a wavefront has lanes."""
    if "top_groups" in options:
        options = dict(options, groups=5 if experts % 5 == 0 else 4)
    announce("expert_topk few distinct", experts, distinct, options)
    g = torch.Generator().manual_seed(experts + distinct)
    values = torch.randn(distinct, generator=g)
    # Neighbours a few FP32 steps apart, too: the sigmoid's or the softmax's rounding decides in FP32.
    values[distinct // 2:] = 0.5 + torch.arange(distinct - distinct // 2) * 2.0**-23
    logits = values[torch.randint(0, distinct, (60, experts), generator=g)]
    for bias in (None, torch.tensor([0.0, 0.25])[torch.randint(0, 2, (experts,), generator=g)]):
        for top in (1, 8, 16):
            got = ops.expert_topk(logits.to(device), top, bias=None if bias is None else bias.to(device), **options)
            want = reference(logits.numpy(), top, bias=None if bias is None else bias.numpy(), **options)
            assert_choice(got, want, f"top {top}")


@pytest.mark.gpu
def test_group_ranks_past_fp32(device):
    """Two finite choices may add up past FP32's range; a group's two may cancel to far less than their rounding."""
    announce("expert_topk group ranks")
    g = torch.Generator().manual_seed(5)
    logits = logits_of(64, 16, torch.float32, 7)
    for sign in (-1.0, 1.0):
        bias = sign * (1.8e38 + 1.5e38 * torch.rand(16, generator=g))
        for top_groups in (1, 2):
            options = dict(groups=4, top_groups=top_groups)
            got = ops.expert_topk(logits.to(device), 4, bias=bias.to(device), **options)
            assert_choice(got, reference(logits.numpy(), 4, bias=bias.numpy(), **options), f"{sign} {top_groups}")
    logits = logits_of(2000, 64, torch.float32, 8)
    bias = 100.0 + 900.0 * torch.rand(32, generator=g)
    bias = torch.stack([bias, -bias], 1).reshape(-1)
    options = dict(groups=32, top_groups=8)
    got = ops.expert_topk(logits.to(device), 8, bias=bias.to(device), **options)
    assert_choice(got, reference(logits.numpy(), 8, bias=bias.numpy(), **options), "cancelled")


@pytest.mark.gpu
def test_small_scores_renormalise(device):
    """Sums far below FP32's epsilon, and picks whose scores are all zero (chosen by bias alone)."""
    announce("expert_topk small scores")
    logits = torch.full((3, 40), -60.0)
    logits[1] -= torch.arange(40) * 0.5
    logits[2] = -3.0e38
    bias = torch.zeros(40)
    bias[17:25] = 1.0
    for scoring in ("sigmoid", "softmax"):
        got = ops.expert_topk(logits.to(device), 4, scoring=scoring, bias=bias.to(device))
        assert_choice(got, reference(logits.numpy(), 4, scoring=scoring, bias=bias.numpy()), scoring)
    logits[:, 0] = 100.0  # the softmax of the biased experts underflows to zero
    logits[:, 1:] = -1000.0
    got = ops.expert_topk(logits.to(device), 4, scoring="softmax", bias=(2 * bias).to(device))
    assert_choice(got, reference(logits.numpy(), 4, scoring="softmax", bias=2 * bias.numpy()), "zeros")


@pytest.mark.gpu
def test_strided_rows_map_live_and_load(device):
    announce("expert_topk strides, map, live, load")
    buffer = logits_of(50, 200, torch.bfloat16, 11).to(device)
    scores = buffer[:, 13:141]
    scores[49] = float("-inf")
    mapping = torch.randperm(128, generator=torch.Generator().manual_seed(1)).to(torch.int32)
    load = torch.arange(128, dtype=torch.int64)
    live = torch.tensor([31], dtype=torch.int32)
    want_ids, want_weights = reference(scores.double().cpu().numpy(), 6)
    load_d = load.to(device)
    got = ops.expert_topk(scores, 6, mapping=mapping.to(device), live=live.to(device), load=load_d)
    mapped = np.where(want_ids >= 0, mapping.numpy()[np.maximum(want_ids, 0)], -1)
    assert_choice(got, (mapped, want_weights))
    counted = load.numpy() + np.bincount(want_ids[:31].reshape(-1), minlength=128)
    np.testing.assert_array_equal(load_d.cpu().numpy(), counted)
    ops.expert_topk(scores, 6, load=load_d)  # no live count: every row, on top of what is there
    counted += np.bincount(want_ids[:49].reshape(-1), minlength=128)
    np.testing.assert_array_equal(load_d.cpu().numpy(), counted)


@pytest.mark.gpu
def test_rows_past_2_gib_and_many(device):
    announce("expert_topk far rows")
    stride = (1 << 29) + 3
    buffer = torch.empty(3 * stride, dtype=torch.float32, device=device)
    scores = buffer.as_strided((3, 100), (stride, 1))
    logits = logits_of(3, 100, torch.float32, 2)
    scores.copy_(logits.to(device))
    assert_choice(ops.expert_topk(scores, 5), reference(logits.numpy(), 5))
    del buffer, scores
    announce("expert_topk many rows")
    logits = logits_of(70001, 9, torch.bfloat16, 4)
    got = ops.expert_topk(logits.to(device), 2)
    at = np.r_[0:50, 69900:70001]
    want = reference(logits[at].double().numpy(), 2)
    assert_choice((got[0][at], got[1][at]), want)


@pytest.mark.gpu
def test_no_rows(device):
    ids, weights = ops.expert_topk(torch.empty((0, 16), device=device), 4)
    assert ids.shape == weights.shape == (0, 4)


@pytest.mark.gpu
def test_captured_replays_and_other_streams(device):
    announce("expert_topk graph")
    scores = logits_of(40, 96, torch.float32, 21).to(device)
    bias = bias_of(96, 2).to(device)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        ops.expert_topk(scores, 8, bias=bias, groups=6, top_groups=2)
        side.synchronize()
        with torch.cuda.graph(graph, stream=side):
            got = ops.expert_topk(scores, 8, bias=bias, groups=6, top_groups=2)
    torch.cuda.current_stream().wait_stream(side)
    for seed in (30, 31, 32):
        logits = logits_of(40, 96, torch.float32, seed)
        scores.copy_(logits.to(device))
        graph.replay()
        torch.cuda.synchronize()
        want = reference(logits.numpy(), 8, bias=bias.double().cpu().numpy(), groups=6, top_groups=2)
        assert_choice(got, want, f"replay {seed}")
        eager = ops.expert_topk(scores, 8, bias=bias, groups=6, top_groups=2)
        assert torch.equal(eager[0], got[0]) and torch.equal(eager[1], got[1])


@pytest.mark.gpu
@pytest.mark.parametrize("arguments, says", [
    (dict(scoring="tanh"), "scoring"),
    (dict(bias=torch.zeros(15)), "bias"), (dict(bias="half"), "bias"), (dict(bias="host"), "bias"),
    (dict(mapping="long"), "mapping"), (dict(load="int"), "load"), (dict(live="two"), "live"),
])
def test_python_refusals_of_device_calls(device, arguments, says):
    scores = torch.zeros((4, 16), device=device)
    made = {"half": lambda: torch.zeros(16, dtype=torch.float16, device=device), "host": lambda: torch.zeros(16),
            "long": lambda: torch.zeros(16, dtype=torch.int64, device=device),
            "int": lambda: torch.zeros(16, dtype=torch.int32, device=device),
            "two": lambda: torch.zeros(2, dtype=torch.int32, device=device)}
    arguments = {k: made[v]() if isinstance(v, str) and v in made else v for k, v in arguments.items()}
    arguments = {k: v.to(device) if isinstance(v, torch.Tensor) and v.numel() == 15 else v for k, v in arguments.items()}
    with pytest.raises(ValueError, match=says):
        ops.expert_topk(scores, 2, **arguments)


@pytest.mark.gpu
def test_entry_refusals_reach_python(device):
    scores = torch.zeros((4, 16), device=device)
    with pytest.raises(RuntimeError, match="picks between"):
        ops.expert_topk(scores, 17)
    with pytest.raises(RuntimeError, match="equal size"):
        ops.expert_topk(scores, 2, groups=3)
    with pytest.raises(ValueError, match="contiguous"):
        ops.expert_topk(torch.zeros((16, 4), device=device).t(), 2)
