"""GPU suite: 8-bit weights made on the device out of floats, as the documents describe it."""
import numpy as np
import pytest
import torch

import fastertnn_b200 as ft
from i8_reference import DT, f64, product, product_error, quantise

pytestmark = pytest.mark.gpu
CODE = {"f32": ft.F32, "f16": ft.F16, "bf16": ft.BF16}


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("E,N,K", [(1, 40, 64), (1, 129, 100), (1, 7, 1), (3, 50, 1000), (2, 64, 17)], ids=str)
def test_weights_of_quantised_floats(E, N, K, dtype, gpu_ctx):
    """quantise_i8 leaves its rows 16 bytes or a multiple apart; without those gaps they are the weights of an upload."""
    g, M, pitch = torch.Generator().manual_seed(N + K), 21, ft.i8_pitch(K)
    st = torch.cuda.current_stream().cuda_stream
    w, x = torch.randn(E * N, K, generator=g).to(DT[dtype]), torch.randn(M, K, generator=g).to(DT[dtype])
    dw, dx = w.cuda(), x.cuda()
    qw, qx = (torch.full((n, pitch), 99, dtype=torch.int8, device="cuda") for n in (E * N, M))
    sw, sx, y = torch.empty(E * N, device="cuda"), torch.empty(M, device="cuda"), torch.empty(M, N, device="cuda")
    gpu_ctx.quantise_i8(dw.data_ptr(), CODE[dtype], qw.data_ptr(), sw.data_ptr(), E * N, K, stream=st)
    gpu_ctx.quantise_i8(dx.data_ptr(), CODE[dtype], qx.data_ptr(), sx.data_ptr(), M, K, stream=st)
    rows = qw[:, :K].contiguous()  # the gaps go
    h = gpu_ctx.upload_weights_i8(rows.data_ptr(), sw.data_ptr(), N, K, experts=E)
    offsets = torch.tensor([0] + [M * (e + 1) // E for e in range(E)], dtype=torch.int32, device="cuda")
    if E == 1:
        gpu_ctx.gemm_i8(h, qx.data_ptr(), sx.data_ptr(), y.data_ptr(), ft.F32, M, stream=st)
    else:
        gpu_ctx.gemm_i8_experts(h, qx.data_ptr(), sx.data_ptr(), 0, offsets.data_ptr(), y.data_ptr(), ft.F32, M, M, stream=st)
    gpu_ctx.sync()
    h.free()
    (q, s), (v, t), o = quantise(x), quantise(w), offsets.tolist()
    want = np.concatenate([product(q[a:b], s[a:b], v[e * N:(e + 1) * N], t[e * N:(e + 1) * N], 1.0) for e, (a, b) in enumerate(zip(o, o[1:]))])
    assert (np.abs(f64(y) - want) <= product_error(want, "f32")).all()
