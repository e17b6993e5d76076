"""GPU suite: the choice of experts, their weights and the order of the pairs, against the definition in 64 bits."""
import numpy as np
import pytest
import torch

import fastertnn_b200 as ft
from i8_reference import DT, f64, plan, route

pytestmark = pytest.mark.gpu
CODE = {"f32": ft.F32, "f16": ft.F16, "bf16": ft.BF16}
INF, NAN = float("inf"), float("nan")


def gen(seed):
    return torch.Generator().manual_seed(seed)


def run(ctx, r, logits, bias=None, with_plan=True, stride=None):
    T, E = logits.shape
    stride = stride or E
    buf = torch.full((T * stride + 8,), NAN, dtype=logits.dtype, device="cuda")
    view = buf[:T * stride].view(T, stride)[:, :E]
    view.copy_(logits)
    db = None if bias is None else bias.float().cuda()
    i32 = torch.int32
    experts, weights = torch.full((T * r.top_k + 3,), -9, dtype=i32, device="cuda"), torch.full((T * r.top_k + 3,), -9.0, device="cuda")
    offsets, rows, slots = (torch.full((n + 3,), -9, dtype=i32, device="cuda") for n in (E + 1, T * r.top_k, T * r.top_k))
    for _ in range(2):
        ctx.route(r, view.data_ptr(), CODE[[n for n in DT if DT[n] == logits.dtype][0]], 0 if db is None else db.data_ptr(), T, experts.data_ptr(), weights.data_ptr(),
                  *([offsets.data_ptr(), rows.data_ptr(), slots.data_ptr()] if with_plan else [0, 0, 0]), stride=stride,
                  stream=torch.cuda.current_stream().cuda_stream)
    ctx.sync()
    for t in (experts, weights, offsets, rows, slots):
        assert (t[-3:] == -9).all()
    got = [t[:-3].cpu().numpy() for t in (experts, weights, offsets, rows, slots)]
    return got[0].reshape(T, -1), got[1].reshape(T, -1), got[2], got[3], got[4].reshape(T, -1)


def check(ctx, r, logits, bias=None, stride=None):
    got = run(ctx, r, logits, bias, stride=stride)
    experts, weights = route(logits, bias, r)
    assert np.array_equal(got[0], experts)
    for a, b in zip(got[2:], plan(experts, r.experts)):
        assert np.array_equal(a, b)
    # A score in fp32: the argument of the exponential is rounded (half a step of its size, at most 104 where the result counts), the
    # exponential is off by 2 steps, one addition and one division round; sums of scores inherit the same bound, each of their
    # additions (at most 1024 / 32 + 5 in a row) rounds once more; renormalising and scaling add four roundings.
    x = f64(logits)
    span = np.where(np.isfinite(x), np.abs(x), 0).max(1, keepdims=True) * 2
    rel = 2 * (np.minimum(span, 104) + 2 * 2 + 2 + 37 + 4) * 2.0 ** -24
    least = 2.0 ** -126 * max(1.0, abs(r.scale))  # scores below the normal numbers
    assert (np.abs(got[1] - weights) <= rel * np.abs(weights) + least * 2e20 * r.renormalise + least).all()
    bare = run(ctx, r, logits, bias, with_plan=False, stride=stride)
    assert np.array_equal(bare[0], experts) and np.array_equal(bare[1], got[1]) and (bare[2] == -9).all() and (bare[3] == -9).all() and (bare[4] == -9).all()


SHAPES = [  # T, E, k, groups, top_groups
    (1, 1, 1, 1, 1), (1, 2, 2, 1, 1), (3, 8, 2, 1, 1), (8, 64, 8, 1, 1), (5, 33, 5, 1, 1), (17, 100, 7, 1, 1), (64, 128, 6, 4, 2), (40, 256, 8, 8, 4), (33, 160, 6, 8, 3),
    (9, 1024, 32, 32, 16), (4, 1000, 10, 1, 1), (6, 512, 32, 1, 1), (300, 96, 4, 3, 1), (1000, 16, 2, 4, 2), (20, 32, 4, 32, 8), (30, 30, 30, 1, 1), (2100, 256, 8, 8, 4),
    (5, 384, 32, 8, 2)]


@pytest.mark.parametrize("score", [0, 1])
@pytest.mark.parametrize("with_bias", [False, True])
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("T,E,k,groups,top_groups", SHAPES, ids=str)
def test_route(T, E, k, groups, top_groups, dtype, with_bias, score, gpu_ctx):
    g = gen(T + E + k)
    logits = (torch.randn(T, E, generator=g) * 2).to(DT[dtype])
    bias = torch.randn(E, generator=g) * 0.2 if with_bias else None
    r = ft.Route(E, k, score, groups, top_groups, 1 + (T + score) % 2, (T + E) % 2, [1.0, 2.5][k % 2])
    check(gpu_ctx, r, logits, bias, E + (3 if T % 2 else 0))


@pytest.mark.parametrize("score", [0, 1])
@pytest.mark.parametrize("bias_kind", ["none", "zeros", "steps", "small"])
@pytest.mark.parametrize("E,k,groups,top_groups,group_top", [(256, 8, 8, 4, 2), (64, 6, 1, 1, 1), (128, 16, 4, 2, 1), (1024, 32, 16, 4, 2)], ids=str)
def test_ties(E, k, groups, top_groups, group_top, bias_kind, score, gpu_ctx):
    """Few different logits, so that most choices are ties; with biases that keep, break and reverse them."""
    g = gen(E + k)
    T = 200
    logits = torch.randint(-3, 4, (T, E), generator=g).float() / 2
    logits[50:100] = (torch.randint(0, 2, (50, E), generator=g)).float()
    logits[100] = 0.25
    bias = {"none": None, "zeros": torch.zeros(E), "steps": torch.randint(0, 3, (E,), generator=g).float() / 4, "small": torch.randint(0, 3, (E,), generator=g).float() * 1e-8}[bias_kind]
    check(gpu_ctx, ft.Route(E, k, score, groups, top_groups, group_top, 1, 1.0), logits, bias)


@pytest.mark.parametrize("score", [0, 1])
@pytest.mark.parametrize("gap", [1e-6, 1e-7, 1e-8, 1e-10])
@pytest.mark.parametrize("groups,top_groups", [(1, 1), (8, 3)])
def test_near_ties(groups, top_groups, gap, score, gpu_ctx):
    """Scores + biases closer to each other than fp32 tells apart: the order is that of the 64-bit values."""
    g = gen(int(1 / gap))
    T, E, k = 100, 128, 8
    logits = torch.randn(T, E, generator=g)
    p = torch.softmax(logits[:1].double(), 1) if score == 0 else torch.sigmoid(logits[:1].double())
    bias = (0.7 - p[0] + gap * torch.randn(E, generator=g).double()).float()  # the first token's keys nearly all alike
    logits[1:60] = logits[0] + gap * torch.randn(59, E, generator=g)
    x, b = f64(logits), f64(bias)
    keys = (1 / (1 + np.exp(-x)) if score else np.exp(x) / np.exp(x).sum(1, keepdims=True)) + b
    # tokens whose 64-bit keys differ by less than 64-bit arithmetic itself may round have no defined order: none of them here
    s = np.sort(keys, 1)
    gaps = np.diff(s, axis=1)
    assert ((gaps > 1e-14) | (gaps == 0)).all(1).mean() > 0.9
    fine = ((gaps > 1e-14) | (gaps == 0)).all(1)
    check(gpu_ctx, ft.Route(E, k, score, groups, top_groups, 2, 1, 1.0), logits[torch.from_numpy(fine)], bias)


@pytest.mark.parametrize("score", [0, 1])
@pytest.mark.parametrize("group_top", [1, 2])
@pytest.mark.parametrize("middle", [0.0, 17.0, 40.0, -30.0, 1000.0])
@pytest.mark.parametrize("E,groups,top_groups", [(128, 8, 3), (256, 4, 1), (60, 5, 2), (32, 1, 1)])
def test_logits_next_to_each_other(E, groups, top_groups, middle, group_top, score, gpu_ctx):
    """Logits that differ in their last bits only, where scores are steep and where they are all alike."""
    logits = middle + torch.randint(-3, 4, (150, E), generator=gen(E)) * max(abs(middle), 1.0) * 2.0 ** -23
    logits[::3] += torch.randint(0, 2, (50, E), generator=gen(E + 1)) * 0.5
    if score == 0 and group_top == 2:  # sums of a softmax's scores that differ by less than 64-bit arithmetic rounds have no defined order
        x = f64(logits)
        p = np.exp(x - x.max(1, keepdims=True))
        p /= p.sum(1, keepdims=True)
        worth = np.sort(np.sort(p.reshape(150, groups, -1), 2)[:, :, -2:].sum(2), 1)
        gaps = np.diff(worth, axis=1)
        logits = logits[torch.from_numpy(((gaps > 1e-14) | (gaps == 0)).all(1))]
        if not len(logits):
            pytest.skip("no row with a defined order")
    check(gpu_ctx, ft.Route(E, 6, score, groups, top_groups, group_top, 1, 1.0), logits.float())


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("with_bias", [False, True])
@pytest.mark.parametrize("score", [0, 1])
@pytest.mark.parametrize("groups,top_groups,group_top", [(1, 1, 1), (8, 2, 1), (8, 2, 2), (16, 8, 2)])
def test_barred_and_extreme(groups, top_groups, group_top, score, with_bias, dtype, gpu_ctx):
    """Rows that leave nothing, some, or one; NaN; infinities; the type's lowest value as a mask; scores that saturate."""
    E, k = 64, 8
    g = gen(3)
    low, top = torch.finfo(DT[dtype]).min, torch.finfo(DT[dtype]).max
    x = torch.randn(20, E, generator=g)
    x[0] = -INF
    x[1] = NAN
    x[2] = -INF
    x[2, 40] = 1.5
    x[3, ::2] = -INF
    x[4, 5:] = -INF
    x[5] = low
    x[6, :60] = low
    x[7, 3], x[7, 60] = INF, INF
    x[8, 10] = NAN
    x[9] = INF
    x[10, 7] = top
    x[11] *= 100
    x[12] = -60
    x[13] = torch.arange(E) * -0.5
    x[14] = torch.arange(E) * 0.5
    x[15, 20:] = NAN
    x[16] = -1000
    x[16, 9] = 1000
    bias = None
    if with_bias:
        bias = torch.randn(E, generator=g) * 0.1
        bias[4], bias[33], bias[50], bias[8:16] = -INF, NAN, INF, -INF
    for renormalise in (0, 1):
        check(gpu_ctx, ft.Route(E, k, score, groups, top_groups, group_top, renormalise, 2.0), x.to(DT[dtype]), bias)


def test_no_tokens(gpu_ctx):
    r = ft.Route(64, 4)
    offsets = torch.full((66,), 7, dtype=torch.int32, device="cuda")
    gpu_ctx.route(r, 0, ft.F32, 0, 0, 0, 0, offsets.data_ptr(), 0, 0)
    gpu_ctx.sync()
    assert (offsets[:65] == 0).all() and offsets[65] == 7


@pytest.mark.parametrize("T,E,k", [(20000, 64, 8), (5000, 1024, 4), (40000, 8, 2), (3001, 250, 32)])
def test_many_pairs(T, E, k, gpu_ctx):
    """The order of many pairs, some experts without any, one with nearly all."""
    g = gen(T)
    logits = torch.randn(T, E, generator=g)
    logits[:, 0] += 3
    logits[:, E // 2:E // 2 + 3] -= 30
    logits[T // 2:T // 2 + 500] = -INF
    experts, weights, offsets, rows, slots = run(gpu_ctx, ft.Route(E, k), logits)
    flat = experts.reshape(-1).astype(np.int64)
    order = np.argsort(np.where(flat < 0, E, flat), kind="stable")
    pairs = int((flat >= 0).sum())
    assert np.array_equal(offsets, np.searchsorted(np.where(flat < 0, E, flat)[order], np.arange(E + 1)))
    assert np.array_equal(rows[:pairs], order[:pairs] // k) and (rows[pairs:] == -1).all()
    want = np.full(T * k, -1)
    want[order[:pairs]] = np.arange(pairs)
    assert np.array_equal(slots.reshape(-1), want)
    key = torch.sort(logits, dim=1, descending=True, stable=True).indices[:, :k].numpy()
    assert np.array_equal(np.where(np.isneginf(logits.numpy()).all(1)[:, None], -1, key), experts)
