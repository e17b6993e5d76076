"""GPU suite: the longest rows that the 8-bit operators take."""
import numpy as np
import pytest
import torch

import fastertnn_b200 as ft
from i8_reference import DT, f64

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,K", [("bf16", 2 ** 31 - 1), ("f32", 2 ** 31 - 1), ("f16", 2 ** 31 - 8)])
def test_quantise_one_row_of_2_31(dtype, K, gpu_ctx):
    """A row as long as an int counts: its integers and its scale, nothing behind it."""
    if gpu_ctx.mem_info()[0] < 24 << 30:
        pytest.skip("needs 24 GB of device memory")
    g, n = torch.Generator().manual_seed(K % 1000), 5000
    x = torch.zeros(K, dtype=DT[dtype], device="cuda")
    parts = [0, 2 ** 30 - 7, K - n]
    for at in parts:
        x[at:at + n] = torch.randn(n, generator=g).to(DT[dtype]).cuda()
    x[K - 1] = -9.0  # the largest magnitude is the last
    pitch = ft.i8_pitch(K)
    q, s = torch.full((pitch + 16,), 77, dtype=torch.int8, device="cuda"), torch.full((2,), -1.0, device="cuda")
    gpu_ctx.quantise_i8(x.data_ptr(), {"f32": ft.F32, "f16": ft.F16, "bf16": ft.BF16}[dtype], q.data_ptr(), s.data_ptr(), 1, K,
                        stream=torch.cuda.current_stream().cuda_stream)
    gpu_ctx.sync()
    assert s.tolist() == [float(np.float32(9.0 / 127.0)), -1.0]
    assert bool((q[K:] == 77).all())
    found = 0
    for at in parts:
        want = np.rint(f64(x[at:at + n]) * 127.0 / 9.0).astype(np.int8)
        assert np.array_equal(q[at:at + n].cpu().numpy(), want)
        found += int(np.count_nonzero(want))
    assert sum(int(torch.count_nonzero(q[a:min(a + (1 << 28), K)])) for a in range(0, K, 1 << 28)) == found
    del x, q
    torch.cuda.empty_cache()
