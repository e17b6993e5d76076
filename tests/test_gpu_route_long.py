"""GPU suite: the order of so many pairs that a block goes over its tokens in several slabs, and of as many as a call takes."""
import pytest
import torch

import fastertnn_b200 as ft

pytestmark = pytest.mark.gpu


def run(ctx, r, logits):
    T, E = logits.shape
    code = {torch.float32: ft.F32, torch.bfloat16: ft.BF16}[logits.dtype]
    experts, rows, slots = (torch.empty(T * r.top_k, dtype=torch.int32, device="cuda") for _ in range(3))
    weights, offsets = torch.empty(T * r.top_k, device="cuda"), torch.full((E + 2,), -9, dtype=torch.int32, device="cuda")
    ctx.route(r, logits.data_ptr(), code, 0, T, experts.data_ptr(), weights.data_ptr(), offsets.data_ptr(), rows.data_ptr(), slots.data_ptr(),
              stream=torch.cuda.current_stream().cuda_stream)
    ctx.sync()
    assert int(offsets[E + 1]) == -9
    return experts, weights, offsets[:E + 1], rows, slots


@pytest.mark.parametrize("T,E,k", [(40_000, 1024, 4), (200_003, 256, 8), (12_289, 1000, 32), (1_500_001, 60, 2), (3_000_000, 8, 1)], ids=str)
def test_many_slabs(T, E, k, gpu_ctx):
    g = torch.Generator(device="cuda").manual_seed(T)
    logits = torch.randn(T, E, generator=g, device="cuda")
    logits[:, 1] += 2
    logits[:, E // 2] = -float("inf")
    logits[T // 3:T // 3 + 777] = -float("inf")
    experts, _, offsets, rows, slots = run(gpu_ctx, ft.Route(E, k), logits)
    value, best = torch.sort(logits, dim=1, descending=True, stable=True)
    assert torch.equal(experts.view(T, k), torch.where(value[:, :k] > -float("inf"), best[:, :k], -1).int())
    del value, best
    key, order = torch.sort(torch.where(experts < 0, E, experts), stable=True)
    assert torch.equal(offsets, torch.searchsorted(key, torch.arange(E + 1, dtype=torch.int32, device="cuda")).int())
    pairs = int(offsets[E])
    assert pairs < T * k and torch.equal(rows[:pairs], (order[:pairs] // k).int()) and bool((rows[pairs:] == -1).all())
    want = torch.full((T * k,), -1, dtype=torch.int32, device="cuda")
    want[order[:pairs]] = torch.arange(pairs, dtype=torch.int32, device="cuda")
    assert torch.equal(slots, want)


def test_as_many_pairs_as_a_call_takes(gpu_ctx):
    """One of two experts for each of 2^31 - 2^16 tokens."""
    T = 0x7FFF0000
    if gpu_ctx.mem_info()[0] < 80 << 30:
        pytest.skip("needs 80 GB of device memory")
    logits = torch.zeros(T, 2, dtype=torch.bfloat16, device="cuda")
    logits[:, 1].copy_((torch.arange(T, device="cuda", dtype=torch.int32) % 3 == 0).to(torch.bfloat16)).sub_(0.5)  # expert 1: every third token
    with pytest.raises(ft.TnnsError):
        gpu_ctx.route(ft.Route(2, 1), logits.data_ptr(), ft.BF16, 0, T + 1, 16, 16)
    experts, weights, offsets, rows, slots = run(gpu_ctx, ft.Route(2, 1), logits)
    ones = (T + 2) // 3
    assert offsets.tolist() == [0, T - ones, T]
    del logits, weights
    step = 3 << 26
    for a in range(0, T, step):
        b = min(a + step, T)
        t = torch.arange(a, b, device="cuda")
        one = t % 3 == 0
        assert torch.equal(experts[a:b], one.int())
        third = (t + 2) // 3  # tokens of expert 1 before this one
        assert torch.equal(slots[a:b].long(), torch.where(one, T - ones + third, t - third))
        assert torch.equal(rows[slots[a:b].long()].long(), t)
        del t, one, third
    del experts, rows, slots
    torch.cuda.empty_cache()
