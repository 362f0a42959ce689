"""A whole MoE block with grouped sigmoid routing and a shared expert, operator by operator: the
router's FP32 logits (linear), the choice (expert_topk), the sort, the routed products and their
combine, and the shared expert (gated_linear, then linear with its row gate onto the routed sum),
against the same block in 64 bits.

Ids must be the definition's on the device's own logits. The output: bf16 roundings of the gated rows
and products (2^-8 each, relative) over sums of terms that partly cancel, held to the layer's bar.
"""

import numpy as np
import pytest
import torch

import test_expert_topk
from gpu_helpers import announce, assert_bf16_bar, bf16_values, normal_bf16
from uniserve_moe import ops

pytestmark = pytest.mark.gpu


def block(x, p, top, options):
    experts = p["router"].shape[0]
    logits = ops.linear(x, p["router"], out_dtype=torch.float32)
    ids, weights = ops.expert_topk(logits, top, **options)
    maps = ops.moe_sort(ids, weights, experts)
    gated = ops.gather_gemm(x, p["up_gate"], top, maps, ops.permuted_rows(x.shape[0], top, experts))
    products = ops.route_gemm(gated, p["down"], maps)
    routed = ops.moe_unpermute(products, maps[ops.EXPANDED_TO_PERMUTED], weights)
    shared = ops.gated_linear(x, p["shared_up_gate"])
    gate = ops.linear(x, p["shared_gate"])
    out = ops.linear(shared, p["shared_down"], gate=gate, residual=routed, out=routed)
    return out, logits, ids, weights


def mlp(x, up_gate, down):
    up, gate = (x @ up_gate.t()).split(up_gate.shape[0] // 2, dim=1)
    return (up * gate * torch.special.expit(gate)) @ down.t()


@pytest.mark.parametrize("tokens", [1, 37, 300])
def test_block(device, tokens):
    announce("MoE block", tokens)
    hidden, experts, top, intermediate, shared = 512, 32, 4, 256, 384
    p = {
        "router": normal_bf16((experts, hidden), 1, 0.05), "up_gate": normal_bf16((experts, 2 * intermediate, hidden), 2, 0.02),
        "down": normal_bf16((experts, hidden, intermediate), 3, 0.02), "shared_up_gate": normal_bf16((2 * shared, hidden), 4, 0.02),
        "shared_down": normal_bf16((hidden, shared), 5, 0.02), "shared_gate": normal_bf16((1, hidden), 6, 0.02),
    }
    x = normal_bf16((tokens, hidden), 7)
    bias = test_expert_topk.bias_of(experts, 8)
    options = dict(groups=4, top_groups=2, factor=2.5)
    out, logits, ids, weights = block(x, p, top, dict(options, bias=bias.to(device)))
    want = test_expert_topk.reference(logits.double().cpu().numpy(), top, bias=bias.double().numpy(), **options)
    test_expert_topk.assert_choice((ids, weights), want)

    q = {k: v.double().cpu() for k, v in p.items()}
    rows = x.double().cpu()
    expected = torch.zeros((tokens, hidden), dtype=torch.float64)
    for t in range(tokens):
        for e, w in zip(want[0][t], want[1][t]):
            expected[t] += w * mlp(rows[t:t + 1], q["up_gate"][e], q["down"][e])[0]
    expected += torch.special.expit(rows @ q["shared_gate"].t()) * mlp(rows, q["shared_up_gate"], q["shared_down"])
    assert_bf16_bar(bf16_values(out), expected.numpy(), f"{tokens} tokens")


def test_block_captured(device):
    """The whole block in a graph, replayed with other tokens, against the eager block: the same bits."""
    announce("MoE block captured")
    hidden, experts, top, intermediate, shared, tokens = 256, 16, 4, 128, 192, 45
    p = {
        "router": normal_bf16((experts, hidden), 1, 0.05), "up_gate": normal_bf16((experts, 2 * intermediate, hidden), 2, 0.02),
        "down": normal_bf16((experts, hidden, intermediate), 3, 0.02), "shared_up_gate": normal_bf16((2 * shared, hidden), 4, 0.02),
        "shared_down": normal_bf16((hidden, shared), 5, 0.02), "shared_gate": normal_bf16((1, hidden), 6, 0.02),
    }
    options = dict(groups=4, top_groups=2, bias=test_expert_topk.bias_of(experts, 8).to(device))
    x = normal_bf16((tokens, hidden), 7)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        block(x, p, top, options)
        side.synchronize()
        with torch.cuda.graph(graph, stream=side):
            captured = block(x, p, top, options)
    torch.cuda.current_stream().wait_stream(side)
    for seed in (8, 9, 10):
        x.copy_(normal_bf16((tokens, hidden), seed))
        graph.replay()
        torch.cuda.synchronize()
        replayed = [t.clone() for t in captured]
        for got, want in zip(replayed, block(x, p, top, options)):
            assert torch.equal(got, want), seed
        torch.cuda.synchronize()


def test_masked_tokens_get_the_shared_expert_alone(device):
    """Padding rows whose logits are all -inf route nowhere: ids -1, weight 0, no routed sum."""
    announce("MoE block masked tokens")
    hidden, experts, top, intermediate, tokens = 256, 16, 2, 128, 24
    x = normal_bf16((tokens, hidden), 1)
    logits = torch.randn((tokens, experts), generator=torch.Generator().manual_seed(2)).to(device)
    logits[5:9] = float("-inf")
    ids, weights = ops.expert_topk(logits, top)
    maps = ops.moe_sort(ids, weights, experts)
    up_gate, down = normal_bf16((experts, 2 * intermediate, hidden), 3, 0.02), normal_bf16((experts, hidden, intermediate), 4, 0.02)
    gated = ops.gather_gemm(x, up_gate, top, maps, ops.permuted_rows(tokens, top, experts))
    routed = ops.moe_unpermute(ops.route_gemm(gated, down, maps), maps[ops.EXPANDED_TO_PERMUTED], weights)
    assert (ids[5:9] == -1).all() and (routed[5:9] == 0).all()
    alone = torch.cat([torch.arange(5), torch.arange(9, tokens)]).to(device)
    ids2, weights2 = ops.expert_topk(logits[alone].contiguous(), top)
    assert torch.equal(ids[alone], ids2) and torch.equal(weights[alone], weights2)
    assert torch.isfinite(routed).all() and (routed[alone] != 0).any(dim=1).all()
