"""GPU suite: routing limited to groups, where groups run out of experts and where their worths are hard to compare in fp32."""
import numpy as np
import pytest
import torch

import fastertnn_b200 as ft
from i8_reference import DT, route
from test_gpu_route import INF, NAN, check, gen

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("score", [0, 1])
@pytest.mark.parametrize("group_top", [1, 2])
@pytest.mark.parametrize("masked_by", ["logits", "bias", "both"])
@pytest.mark.parametrize("E,k,groups,top_groups", [
    (64, 8, 8, 1), (64, 8, 8, 4), (32, 4, 16, 4), (256, 8, 8, 4), (128, 8, 4, 2), (160, 6, 8, 3), (384, 8, 8, 2), (96, 8, 3, 1), (1024, 32, 32, 4), (1024, 16, 2, 1),
    (1020, 10, 17, 3), (320, 32, 5, 2)], ids=str)
def test_kept_groups_run_out_of_experts(E, k, groups, top_groups, masked_by, group_top, score, gpu_ctx):
    """The best groups hold fewer experts than slots, the others (the first group among them) hold many: none of theirs is chosen."""
    g, T, size = gen(E + k + groups), 60, E // groups
    logits = torch.randn(T, E, generator=g) * 0.5 - 3
    best = torch.arange(groups) >= groups - top_groups if masked_by == "bias" else None  # (a bias is the same for all tokens)
    bias = torch.randn(E, generator=g) * 0.01 if masked_by != "logits" else None
    for t in range(T):
        chosen = torch.arange(groups)[best] if best is not None else 1 + torch.randperm(groups - 1, generator=g)[:top_groups] if groups > top_groups else torch.arange(groups)
        for i in chosen.tolist():
            there = torch.randperm(size, generator=g)[:t % 4]
            if masked_by == "bias":
                logits[t, i * size:(i + 1) * size] += 6
            else:
                keep = logits[t, i * size + there] + 6
                logits[t, i * size:(i + 1) * size] = [-INF, NAN][t % 2]
                logits[t, i * size + there] = keep
    if masked_by == "bias":
        for i in torch.arange(groups)[best].tolist():
            bias[i * size:(i + 1) * size] = [-INF, NAN][i % 2]
            bias[i * size + torch.randperm(size, generator=g)[:i % 3]] = 0.25
    r = ft.Route(E, k, score, groups, top_groups, group_top, 1, 2.5)
    check(gpu_ctx, r, logits, bias)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("with_bias", [False, True])
def test_one_expert_left_in_every_kept_group(with_bias, dtype, gpu_ctx):
    """Four kept groups with an expert each, four whole ones that are not kept: four slots stay empty."""
    logits = torch.randn(1, 256, generator=gen(1)) * 0.1
    logits[0, 128:] = -INF
    for e, v in ((130, 5.0), (165, 6.0), (200, 7.0), (230, 8.0)):
        logits[0, e] = v
    r = ft.Route(256, 8, 0, 8, 4, 1, 1, 1.0)
    logits, bias = logits.to(DT[dtype]), torch.zeros(256) if with_bias else None
    assert route(logits, bias, r)[0].tolist() == [[230, 200, 165, 130, -1, -1, -1, -1]]
    check(gpu_ctx, r, logits, bias)


LOWEST, LARGEST = -float(np.finfo(np.float32).max), float(np.finfo(np.float32).max)


@pytest.mark.parametrize("score", [0, 1])
@pytest.mark.parametrize("group_top", [1, 2])
@pytest.mark.parametrize("values", [[LOWEST], [LOWEST, 0.1], [LOWEST, -2e38, -1.8e38, 0.0], [LARGEST, 2e38, LOWEST], [INF, LARGEST, 0.0, -2e38]], ids=str)
@pytest.mark.parametrize("E,k,groups,top_groups", [(12, 6, 3, 2), (64, 16, 8, 2), (128, 16, 4, 2), (256, 8, 8, 4), (1024, 32, 16, 3)], ids=str)
def test_biases_whose_sums_leave_fp32(E, k, groups, top_groups, values, group_top, score, gpu_ctx):
    """Two biases of a group that add up to more (or less) than the largest float: such a group still has experts, and its place."""
    g, T, size = gen(E + len(values)), 80, E // groups
    bias = torch.tensor(values)[torch.randint(0, len(values), (E,), generator=g)]
    for i in range(0, groups, 2):  # groups all alike
        bias[i * size:(i + 1) * size] = values[i // 2 % len(values)]
    logits = torch.randn(T, E, generator=g)
    for t in range(1, T):  # groups without experts, in front of those and between them
        for i in torch.randperm(groups, generator=g)[:t % groups].tolist():
            logits[t, i * size:(i + 1) * size] = -INF
    check(gpu_ctx, ft.Route(E, k, score, groups, top_groups, group_top, 1, 1.0), logits, bias)


def test_lowest_biases_beside_a_group_without_experts(gpu_ctx):
    """Group 0 has no expert, group 1 the type's lowest value as its mask, group 2 ordinary biases: 2 and 1 are kept."""
    logits, bias = torch.zeros(1, 12), torch.zeros(12)
    logits[0, :4], bias[4:8] = -INF, LOWEST
    r = ft.Route(12, 6, 1, 3, 2, 2, 1, 1.0)
    assert route(logits, bias, r)[0].tolist() == [[8, 9, 10, 11, 4, 5]]
    check(gpu_ctx, r, logits, bias)


@pytest.mark.parametrize("score", [0, 1])
@pytest.mark.parametrize("size_of_bias", [30.0, 1000.0, 1e6])
@pytest.mark.parametrize("E,k,groups,top_groups", [(32, 4, 8, 3), (64, 8, 8, 2), (256, 8, 8, 4), (96, 8, 3, 1), (512, 16, 2, 1), (1024, 8, 32, 16)], ids=str)
def test_worths_of_parts_that_cancel(E, k, groups, top_groups, size_of_bias, score, gpu_ctx):
    """A group's two best are far above and far below zero, and their sum is not: groups are ranked by that sum as 64 bits have it."""
    g, T, size = gen(E + groups), 100, E // groups
    bias = torch.full((E,), -3 * size_of_bias)
    for i in range(groups):
        up, down = torch.randperm(size, generator=g)[:2].tolist()
        bias[i * size + up], bias[i * size + down] = size_of_bias, -size_of_bias
    logits = torch.randn(T, E, generator=g)
    check(gpu_ctx, ft.Route(E, k, score, groups, top_groups, 2, 1, 1.0), logits, bias)
