"""GPU suite: rows to 8-bit integers, their products with 8-bit weights (dense and by expert), and the sum back to the tokens,
against the definitions in 64 bits."""
import subprocess
import sys
from pathlib import Path

import numpy as np
import pytest
import torch

import fastertnn_b200 as ft
from i8_reference import DT, F32_STEP, HALF_STEP, LEAST, f64, plan, prelu, product, product_error, quantise, route

pytestmark = pytest.mark.gpu
CODE = {"f32": ft.F32, "f16": ft.F16, "bf16": ft.BF16}
MARK = 77  # what lies behind rows before a call, and has to lie there after it


def gen(seed):
    return torch.Generator().manual_seed(seed)


def stream():
    return torch.cuda.current_stream().cuda_stream


def strided(rows, cols, stride, dtype, fill, shift=0):
    """A flat device buffer and its rows x cols view at `stride`, `shift` elements behind the buffer's start."""
    flat = torch.full((shift + max(rows, 1) * stride + 64,), fill, dtype=dtype, device="cuda")
    return flat, flat[shift:shift + max(rows, 1) * stride].view(max(rows, 1), stride)[:rows, :cols]


def untouched(flat, view, fill):
    keep = torch.ones_like(flat, dtype=torch.bool)
    torch.as_strided(keep, view.shape, view.stride(), view.storage_offset())[:] = False
    return bool((flat[keep] == fill).all())


# --------------------------------------------------------------------------------------------
# quantise
# --------------------------------------------------------------------------------------------

def run_quantise(ctx, x, x_stride=None, q_stride=None, shift=0):
    M, K = x.shape
    flat, view = strided(M, K, x_stride or K, x.dtype, MARK, shift)
    view.copy_(x)
    fq, q = strided(M, K, q_stride or ft.i8_pitch(K), torch.int8, MARK)
    s = torch.full((M + 1,), -1.0, device="cuda")
    ctx.quantise_i8(view.data_ptr(), CODE[[n for n in DT if DT[n] == x.dtype][0]], q.data_ptr(), s.data_ptr(), M, K, x_stride or K,
                    q_stride or ft.i8_pitch(K), stream=stream())
    torch.cuda.synchronize()
    assert untouched(fq, q, MARK) and float(s[M]) == -1
    return q.cpu().numpy(), s[:M].cpu().numpy()


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("M,K,x_stride,q_stride,shift", [
    (1, 1, None, None, 0), (1, 64, None, None, 0), (3, 65, 67, 80, 1), (5, 127, None, None, 0), (2, 1024, None, None, 0), (7, 1000, 1003, 1024, 3),
    (300, 129, None, None, 0), (33, 4096, None, None, 0), (2, 5000, None, None, 0), (1, 16384, None, None, 0), (9, 16385, 16400, 16416, 0), (2, 50001, None, None, 1),
    (5000, 72, None, None, 0), (1200, 2048, 2056, 2064, 8), (4000, 1, None, None, 0), (3601, 1000, 1003, 1024, 1), (3600, 4097, 4099, 4112, 3), (9000, 512, 520, None, 8),
    (3700, 8192, None, None, 0), (7200, 40, 41, None, 0)], ids=str)
def test_quantise(M, K, x_stride, q_stride, shift, dtype, gpu_ctx):
    x = (torch.randn(M, K, generator=gen(M * 131 + K)) * torch.exp(torch.randn(M, 1, generator=gen(K)) * 4)).to(DT[dtype])
    q, s = run_quantise(gpu_ctx, x, x_stride, q_stride, shift)
    want_q, want_s = quantise(x)
    assert np.array_equal(q, want_q) and np.array_equal(s, want_s, equal_nan=True)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("K", [256, 2049, 20000])
def test_quantise_halves(K, dtype, gpu_ctx):
    """Values on, just below and just above every half, for many row maxima."""
    rng = np.random.default_rng(5)
    rows = []
    for _ in range(64):
        a = np.float64(torch.tensor(float(rng.uniform(1, 2) * 2.0 ** rng.integers(-10, 10)), dtype=DT[dtype]).double().item())
        base = torch.from_numpy((rng.integers(-127, 127, K) + 0.5) * a / 127).to(DT[dtype])
        up = torch.nextafter(base, torch.full_like(base, float("inf"))) if dtype == "f32" else (base.double() * (1 + 2 * HALF_STEP[dtype])).to(DT[dtype])
        x = torch.where(torch.from_numpy(rng.random(K) < 0.5), base, up)
        x = torch.where(x.double().abs() > a, torch.zeros_like(x), x)
        x[rng.integers(K)] = a
        rows.append(x)
    x = torch.stack(rows)
    q, s = run_quantise(gpu_ctx, x)
    want_q, want_s = quantise(x)
    assert np.array_equal(q, want_q) and np.array_equal(s, want_s, equal_nan=True)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("times", [1, 400])
@pytest.mark.parametrize("K", [40, 1536, 2049, 20001])
def test_quantise_special_rows(K, times, dtype, gpu_ctx):
    """Zeros, negative zeros, one value, infinities, NaN, the type's largest and smallest numbers."""
    top, small = torch.finfo(DT[dtype]).max, {"f32": 2.0 ** -149, "f16": 2.0 ** -24, "bf16": 2.0 ** -133}[dtype]
    x = torch.randn(11, K, generator=gen(K)).to(DT[dtype])
    x[0] = 0
    x[1] = -0.0
    x[2] = 0
    x[2, K - 1] = -3.0
    x[3, K // 2] = float("inf")
    x[4, 0] = float("-inf")
    x[5, K - 1] = float("nan")
    x[6, 1] = top
    x[7, 2] = -top
    x[8] = small
    x[9] = 0
    x[9, 3], x[9, 4] = 5 * small, 2 * small
    x[10, 0], x[10, 1] = float("nan"), float("inf")
    x = x.repeat(times if K < 10000 else 1, 1)
    q, s = run_quantise(gpu_ctx, x)
    want_q, want_s = quantise(x)
    assert np.array_equal(q, want_q) and np.array_equal(s, want_s, equal_nan=True)


def test_quantise_nothing(gpu_ctx):
    gpu_ctx.quantise_i8(0, ft.F32, 0, 0, 0, 64)


# --------------------------------------------------------------------------------------------
# dense product
# --------------------------------------------------------------------------------------------

def int8(g, *shape):
    return torch.randint(-128, 128, shape, generator=g, dtype=torch.int8)


def run_gemm(ctx, q, scale, w, w_scale, dtype, alpha, q_stride=None, y_stride=None, shift=0):
    (M, K), N = q.shape, w.shape[0]
    fq, dq = strided(M, K, q_stride or ft.i8_pitch(K), torch.int8, MARK)
    dq.copy_(q)
    fy, y = strided(M, N, y_stride or N, DT[dtype], MARK, shift)
    h = ctx.upload_weights_i8(w.contiguous().data_ptr(), w_scale.data_ptr(), N, K)
    ds = scale.cuda()
    try:
        for _ in range(2):
            ctx.gemm_i8(h, dq.data_ptr(), ds.data_ptr(), y.data_ptr(), CODE[dtype], M, alpha, q_stride or ft.i8_pitch(K), y_stride or N, stream=stream())
        ctx.sync()
    finally:
        h.free()
    assert untouched(fy, y, MARK)
    return f64(y)


GEMM = [
    (1, 1, 1), (1, 64, 16), (1, 4096, 1000), (2, 130, 257), (3, 100, 8), (7, 255, 129), (8, 512, 512), (9, 1234, 1000), (16, 1024, 640), (17, 640, 96), (31, 2000, 333),
    (33, 128, 128), (37, 1234, 1000), (64, 4096, 256), (65, 96, 4100), (100, 777, 300), (127, 384, 192), (128, 1024, 1024), (129, 1025, 1025), (200, 2048, 64),
    (257, 4100, 511), (300, 50, 2000), (513, 129, 700), (1000, 1500, 1000), (1024, 4096, 1024), (2049, 256, 513), (4100, 640, 1100)]


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("M,K,N", GEMM, ids=str)
def test_gemm(M, K, N, dtype, gpu_ctx):
    g = gen(M + 7 * K + 13 * N)
    q, w = int8(g, M, K), int8(g, N, K)
    scale, w_scale = torch.rand(M, generator=g) * 0.01, torch.rand(N, generator=g) * 0.001
    alpha = [1.0, 0.5, -0.25][(M + K + N) % 3]
    y = run_gemm(gpu_ctx, q, scale, w, w_scale, dtype, alpha)
    want = product(q.numpy(), scale.numpy(), w.numpy(), w_scale.numpy(), alpha)
    assert (np.abs(y - want) <= product_error(want, dtype)).all()


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("M,K,N,q_stride,y_stride,shift", [
    (5, 100, 70, 160, 75, 1), (5, 100, 72, 112, 96, 8), (70, 300, 130, 320, 131, 3), (300, 520, 264, 528, 272, 0), (300, 520, 264, 4096, 265, 5),
    (1000, 300, 500, 304, 502, 2), (2500, 256, 300, 272, 301, 1), (2500, 256, 640, 256, 656, 16), (600, 256, 1024, 256, 1032, 8)], ids=str)
def test_gemm_strides(M, K, N, q_stride, y_stride, shift, dtype, gpu_ctx):
    g = gen(M + N)
    q, w = int8(g, M, K), int8(g, N, K)
    scale, w_scale = torch.rand(M, generator=g), torch.rand(N, generator=g) * 0.001
    y = run_gemm(gpu_ctx, q, scale, w, w_scale, dtype, 0.5, q_stride, y_stride, shift)
    want = product(q.numpy(), scale.numpy(), w.numpy(), w_scale.numpy(), 0.5)
    assert (np.abs(y - want) <= product_error(want, dtype)).all()


# Fewer tiles than the GPU has SMs and long sums: blocks that share a tile's sum.
FEW_TILES = [
    (128, 4096, 4096, 4096, 0), (33, 2048, 4096, 4104, 8), (65, 4096, 2500, 2501, 1), (100, 2500, 2333, 2333, 0), (1, 131071, 4224, 4224, 0), (100, 131071, 300, 301, 3),
    (256, 4096, 4096, 4096, 0), (282, 14050, 1529, 1529, 0), (1030, 5000, 901, 904, 0), (1500, 3333, 231, 231, 1), (2738, 8443, 130, 132, 2), (640, 2100, 700, 704, 0),
    (500, 1024, 1000, 1000, 0), (320, 6000, 1536, 1600, 16), (257, 513, 1111, 1111, 0), (4000, 1030, 40, 41, 0),
    (9, 8200, 8190, 8190, 1), (20, 4100, 8200, 8208, 0), (32, 2050, 9001, 9001, 1)]


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("M,K,N,y_stride,shift", FEW_TILES, ids=str)
def test_gemm_few_tiles(M, K, N, y_stride, shift, dtype, gpu_ctx):
    g = gen(M + 3 * K + 5 * N)
    q, w = int8(g, M, K), int8(g, N, K)
    scale, w_scale = torch.rand(M, generator=g) * 0.01, torch.rand(N, generator=g) * 0.001
    alpha = [1.0, 0.5, -0.25][(M + K + N) % 3]
    y = run_gemm(gpu_ctx, q, scale, w, w_scale, dtype, alpha, y_stride=y_stride, shift=shift)
    want = product(q.numpy(), scale.numpy(), w.numpy(), w_scale.numpy(), alpha)
    assert (np.abs(y - want) <= product_error(want, dtype)).all()


def test_gemm_few_tiles_in_a_row(gpu_ctx):
    """Products whose blocks share sums, each reading what the one in front wrote, in one captured graph replayed: no run differs."""
    g = gen(77)
    M, D, H = 128, 4096, 2048
    s1, s2 = torch.rand(D, generator=g) * 1e-4, torch.rand(H, generator=g) * 1e-4
    up, down = (gpu_ctx.upload_weights_i8(int8(g, n, k).data_ptr(), s.data_ptr(), n, k) for n, k, s in ((H, D, s2), (D, H, s1)))
    x0 = torch.randn(M, D, generator=g).cuda()
    x, y = x0.clone(), torch.empty(M, H, device="cuda")
    qx, qy = torch.empty(M, D, dtype=torch.int8, device="cuda"), torch.empty(M, H, dtype=torch.int8, device="cuda")
    sx, sy = torch.empty(M, device="cuda"), torch.empty(M, device="cuda")

    def run():
        for _ in range(6):
            gpu_ctx.quantise_i8(x.data_ptr(), ft.F32, qx.data_ptr(), sx.data_ptr(), M, D, stream=stream())
            gpu_ctx.gemm_i8(up, qx.data_ptr(), sx.data_ptr(), y.data_ptr(), ft.F32, M, 0.5, stream=stream())
            gpu_ctx.quantise_i8(y.data_ptr(), ft.F32, qy.data_ptr(), sy.data_ptr(), M, H, stream=stream())
            gpu_ctx.gemm_i8(down, qy.data_ptr(), sy.data_ptr(), x.data_ptr(), ft.F32, M, 1.0, stream=stream())

    run()
    gpu_ctx.sync()
    want = x.clone()
    assert bool(torch.isfinite(want).all()) and bool(want.any())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    for _ in range(20):
        x.copy_(x0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(x, want)
    up.free()
    down.free()


@pytest.mark.parametrize("M", [1, 20, 300])
def test_gemm_largest_sums(M, gpu_ctx):
    """The longest rows of the largest products: the sum is a few products short of 2^31."""
    K, N = 131071, 24
    q, w = torch.full((M, K), -128, dtype=torch.int8), torch.full((N, K), -128, dtype=torch.int8)
    w[1::2] = 127
    ones = torch.ones(M), torch.ones(N)
    y = run_gemm(gpu_ctx, q, ones[0], w, ones[1], "f32", 1.0)
    assert (y[:, 0::2] == np.float32(K * 16384)).all() and (y[:, 1::2] == np.float32(-K * 16256)).all()


@pytest.mark.parametrize("M", [2, 40, 700])
def test_gemm_special_scales(M, gpu_ctx):
    """A NaN or infinite row scale stays in its row; a zero scale gives zeros; results past a type's range are infinite."""
    g = gen(M)
    q, w = int8(g, M, 200), int8(g, 90, 200)
    scale = torch.rand(M, generator=g)
    scale[0] = float("nan")
    if M > 2:
        scale[3], scale[M - 1], scale[7] = 0, float("inf"), 1e30
    y = run_gemm(gpu_ctx, q, scale, w, torch.ones(90), "f16", 0.5)
    with np.errstate(invalid="ignore", over="ignore"):
        want = product(q.numpy(), scale.numpy(), w.numpy(), np.ones(90, np.float32), 0.5)
        want = np.where(np.abs(want) >= 65520, np.copysign(np.inf, want), want)
    fine = np.isfinite(want)
    assert np.array_equal(np.isnan(want), np.isnan(y)) and np.array_equal(want[~fine & ~np.isnan(want)], y[~fine & ~np.isnan(want)])
    assert (np.abs(y - want)[fine] <= product_error(want, "f16")[fine]).all()


def test_gemm_nothing(gpu_ctx):
    w, s = int8(gen(1), 8, 32), torch.ones(8)
    h = gpu_ctx.upload_weights_i8(w.data_ptr(), s.data_ptr(), 8, 32)
    gpu_ctx.gemm_i8(h, 0, 0, 0, ft.F32, 0)
    h.free()


def test_refused_with_weights(gpu_ctx):
    w, s = int8(gen(1), 2, 8, 32), torch.ones(2, 8)
    h = gpu_ctx.upload_weights_i8(w.data_ptr(), s.data_ptr(), 8, 32, experts=2)
    one = gpu_ctx.upload_weights_i8(w.data_ptr(), s.data_ptr(), 8, 32)
    d = torch.zeros(4096, device="cuda").data_ptr()
    ok = dict(w=one, d_q=d, d_scale=d, d_y=d, dtype=0, M=3, alpha=1.0, q_stride=32, y_stride=8)
    try:
        for change in (dict(w=h), dict(dtype=3), dict(M=-1), dict(q_stride=16), dict(q_stride=40), dict(y_stride=7), dict(d_q=0), dict(d_scale=0), dict(d_y=0),
                       dict(d_q=d + 8), dict(d_y=d + 2), dict(d_scale=d + 1)):
            with pytest.raises(ft.TnnsError) as e:
                gpu_ctx.gemm_i8(**{**ok, **change})
            assert e.value.status == 1
        ok = dict(w=h, d_q=d, d_scale=d, d_rows=d, d_offsets=d, d_y=d, dtype=0, q_rows=3, places=4)
        for change in (dict(dtype=3), dict(q_rows=-1), dict(places=-1), dict(d_offsets=0), dict(d_q=0), dict(d_scale=0), dict(d_y=0), dict(d_rows=d + 2),
                       dict(d_offsets=d + 2), dict(q_stride=24), dict(y_stride=4)):
            with pytest.raises(ft.TnnsError) as e:
                gpu_ctx.gemm_i8_experts(**{**ok, **change})
            assert e.value.status == 1
    finally:
        h.free()
        one.free()


def test_weights_from_device_memory(gpu_ctx):
    g = gen(3)
    q, w, s, ws = int8(g, 5, 300), int8(g, 77, 300), torch.rand(5, generator=g), torch.rand(77, generator=g)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        dw, dws = w.cuda(non_blocking=True), ws.cuda(non_blocking=True)
        h = gpu_ctx.upload_weights_i8(dw.data_ptr(), dws.data_ptr(), 77, 300)
        dw.zero_()
    torch.cuda.synchronize()
    dq = torch.zeros(5, 304, dtype=torch.int8, device="cuda")
    dq[:, :300] = q
    ds, y = s.cuda(), torch.empty(5, 77, device="cuda")
    gpu_ctx.gemm_i8(h, dq.data_ptr(), ds.data_ptr(), y.data_ptr(), ft.F32, 5, stream=stream())
    want = product(q.numpy(), s.numpy(), w.numpy(), ws.numpy(), 1.0)
    assert (np.abs(f64(y) - want) <= product_error(want, "f32")).all()
    h.free()


def test_gemm_more_than_2_31(gpu_ctx):
    """Rows and results behind 2^31 bytes and elements."""
    M, K, N = 2_200_000, 1008, 1000
    if gpu_ctx.mem_info()[0] < 20 << 30:
        pytest.skip("needs 20 GB of device memory")
    q = torch.randint(-128, 128, (M, K), dtype=torch.int8, device="cuda")
    g = gen(9)
    w, ws, s = int8(g, N, K), torch.rand(N, generator=g) * 0.01, torch.rand(M, generator=g)
    ds, y = s.cuda(), torch.zeros(M, N, dtype=torch.bfloat16, device="cuda")
    h = gpu_ctx.upload_weights_i8(w.data_ptr(), ws.data_ptr(), N, K)
    gpu_ctx.gemm_i8(h, q.data_ptr(), ds.data_ptr(), y.data_ptr(), ft.BF16, M, 0.5, q_stride=K, stream=stream())
    gpu_ctx.sync()
    h.free()
    for at in (0, 1_000_001, 2_130_400, 2_147_484, M - 70):
        want = product(q[at:at + 70].cpu().numpy(), s[at:at + 70].numpy(), w.numpy(), ws.numpy(), 0.5)
        assert (np.abs(f64(y[at:at + 70]) - want) <= product_error(want, "bf16")).all()
    del q, y
    torch.cuda.empty_cache()


# --------------------------------------------------------------------------------------------
# products by expert
# --------------------------------------------------------------------------------------------

def run_experts(ctx, q, scale, rows, offsets, w, w_scale, dtype, alpha, places, y_stride=None):
    E, N, K = w.shape
    T = q.shape[0]
    fq, dq = strided(T, K, ft.i8_pitch(K), torch.int8, MARK)
    dq.copy_(q)
    fy, y = strided(places, N, y_stride or N, DT[dtype], MARK)
    h = ctx.upload_weights_i8(w.data_ptr(), w_scale.data_ptr(), N, K, experts=E)
    ds, do = scale.cuda(), offsets.cuda()
    dr = None if rows is None else rows.cuda()
    try:
        for _ in range(2):
            ctx.gemm_i8_experts(h, dq.data_ptr(), ds.data_ptr(), 0 if dr is None else dr.data_ptr(), do.data_ptr(), y.data_ptr(), CODE[dtype], T, places,
                                alpha, y_stride=y_stride or N, stream=stream())
        ctx.sync()
    finally:
        h.free()
    assert untouched(fy, y, MARK)
    return f64(y)


def expected_experts(q, scale, rows, offsets, w, w_scale, alpha, places):
    E, N, K = w.shape
    T = q.shape[0]
    want = np.full((places, N), float(MARK))
    o = [min(max(int(v), 0), places) for v in offsets]
    for e in range(E):
        a, b = o[e], max(o[e], o[e + 1])
        if a == b:
            continue
        r = np.arange(a, b) if rows is None else rows[a:b].numpy().astype(np.int64)
        ok = (r >= 0) & (r < T)
        qq = np.where(ok[:, None], q.numpy()[np.clip(r, 0, T - 1)], 0)
        ss = np.where(ok, scale.numpy()[np.clip(r, 0, T - 1)], 0)
        want[a:b] = product(qq, ss, w[e].numpy(), w_scale[e].numpy(), alpha)
    return want


COUNTS = [
    ([1], 64, 32), ([0, 3, 0, 1], 100, 50), ([8] * 8, 256, 256), ([0] * 5 + [9], 130, 96), ([17, 0, 33, 5, 64], 512, 200), ([1, 2, 3, 0, 0, 7, 130], 300, 129),
    ([128, 129, 127, 1], 384, 256), ([300, 0, 12, 500], 640, 520), ([5] * 150, 96, 130), ([1000, 3, 1, 700], 1024, 264), ([2] * 300 + [0] * 20, 64, 70),
    ([2000], 256, 513), ([40] * 30, 1100, 257), ([16] * 20 + [1], 777, 1000), ([3000, 2500], 500, 1300),
    ([700, 1, 900, 0, 257, 256, 255, 1400], 640, 2100),
    ([130] * 60, 2048, 1024), ([60] * 40, 4000, 200), ([90] * 6, 6000, 300),
    ([3, 0, 9, 1] * 20, 2000, 700), ([12, 20] * 30, 1300, 384), ([1] * 200, 130, 65), ([7] * 40, 5003, 1024)]


@pytest.mark.parametrize("gather", [True, False])
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("counts,K,N", COUNTS, ids=lambda v: str(v)[:24])
def test_experts(counts, K, N, dtype, gather, gpu_ctx):
    g = gen(sum(counts) + K + N)
    E, total = len(counts), sum(counts)
    places = total + 5
    T = max(1, total // 3) if gather else places
    q, w = int8(g, T, K), int8(g, E, N, K)
    scale, w_scale = torch.rand(T, generator=g), torch.rand(E, N, generator=g) * 0.001
    offsets = torch.tensor([0] + list(np.cumsum(counts)), dtype=torch.int32)
    rows = torch.randint(0, T, (places,), generator=g, dtype=torch.int32) if gather else None
    y = run_experts(gpu_ctx, q, scale, rows, offsets, w, w_scale, dtype, 0.5, places, N + (3 if K == 300 else 0))
    want = expected_experts(q, scale, rows, offsets, w, w_scale, 0.5, places)
    assert (y[total:] == MARK).all()
    assert (np.abs(y[:total] - want[:total]) <= product_error(want[:total], dtype)).all()


@pytest.mark.parametrize("places", [40, 900])
def test_experts_indices_out_of_range(places, gpu_ctx):
    """Rows outside of q read as zeros; offsets that fall or leave the places are clamped."""
    g = gen(places)
    T, E, K, N = 30, 6, 200, 96
    q, w = int8(g, T, K), int8(g, E, N, K)
    scale, w_scale = torch.rand(T, generator=g) + 0.1, torch.rand(E, N, generator=g)
    rows = torch.randint(0, T, (places,), generator=g, dtype=torch.int32)
    rows[::7], rows[3::11], rows[5::13] = -1, T, 2 ** 31 - 1
    rows[6::17] = -(2 ** 31)
    for offsets in ([0, 9, 9, 20, 30, 31, places], [-5, 10, 12, 20, 30, 35, places + 100], [0, places // 2, places // 2, places // 2, places, 2 ** 31 - 1, 2 ** 31 - 1],
                    [places, 2 * places, -1, 0, 5, 5, 8]):
        o = torch.tensor(offsets, dtype=torch.int32)
        y = run_experts(gpu_ctx, q, scale, rows, o, w, w_scale, "f32", 0.5, places)
        want = expected_experts(q, scale, rows, offsets, w, w_scale, 0.5, places)
        # ranges that overlap are the caller's mistake: any of their experts may have written those rows
        c = [min(max(v, 0), places) for v in offsets]
        times = np.zeros(places, int)
        for a, b in zip(c, c[1:]):
            times[a:max(a, b)] += 1
        once = times <= 1
        assert (np.abs(y - want)[once] <= product_error(want, "f32")[once]).all()


def test_experts_of_one_kernel(gpu_ctx):
    """A layer of one kernel takes the call too; no rows at all; no places at all."""
    g = gen(4)
    q, w, s, ws = int8(g, 20, 100), int8(g, 1, 40, 100), torch.rand(20, generator=g), torch.rand(1, 40, generator=g)
    o = torch.tensor([2, 15], dtype=torch.int32)
    y = run_experts(gpu_ctx, q, s, None, o, w, ws, "f32", 1.0, 20)
    want = expected_experts(q, s, None, [2, 15], w, ws, 1.0, 20)
    assert (np.abs(y - want) <= product_error(want, "f32")).all()
    h = gpu_ctx.upload_weights_i8(w.data_ptr(), ws.data_ptr(), 40, 100)
    do, dy = torch.tensor([0, 3], dtype=torch.int32, device="cuda"), torch.full((3, 40), 5.0, device="cuda")
    gpu_ctx.gemm_i8_experts(h, 0, 0, 0, do.data_ptr(), dy.data_ptr(), ft.F32, 0, 3, stream=stream())
    gpu_ctx.sync()
    assert (dy == 0).all()  # every row reads as zeros
    gpu_ctx.gemm_i8_experts(h, 0, 0, 0, 0, 0, ft.F32, 0, 0)
    h.free()


# --------------------------------------------------------------------------------------------
# combine
# --------------------------------------------------------------------------------------------

@pytest.mark.parametrize("out_dtype", DT)
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("T,k,N,y_stride,out_stride", [
    (1, 1, 1, 1, 1), (1, 8, 2048, 2048, 2048), (5, 3, 70, 71, 73), (40, 8, 1000, 1000, 1000), (300, 2, 264, 272, 280), (700, 8, 33, 33, 33), (9, 32, 4096, 4096, 4104),
    (2500, 4, 128, 128, 128), (64, 6, 10000, 10000, 10000)], ids=str)
def test_combine(T, k, N, y_stride, out_stride, dtype, out_dtype, gpu_ctx):
    g = gen(T + N)
    places = T * k
    slots = torch.randperm(places, generator=g).to(torch.int32).view(T, k)
    slots[torch.rand(T, k, generator=g) < 0.1] = -1
    if T > 4:
        slots[2] = -1
        slots[3, 0], slots[4, k - 1] = places, -7
        slots[1] = slots[0, 0]  # the same place several times
    weights = torch.randn(T, k, generator=g)
    fy, y = strided(places, N, y_stride, DT[dtype], MARK)
    y.copy_(torch.randn(places, N, generator=g))
    fo, out = strided(T, N, out_stride, DT[out_dtype], MARK)
    ds, dw = slots.cuda(), weights.cuda()
    gpu_ctx.combine(y.data_ptr(), CODE[dtype], places, ds.data_ptr(), dw.data_ptr(), k, out.data_ptr(), CODE[out_dtype], T, N, y_stride, out_stride,
                    stream=stream())
    gpu_ctx.sync()
    assert untouched(fo, out, MARK)
    s = slots.numpy().astype(np.int64)
    ok = (s >= 0) & (s < places)
    terms = np.where(ok[:, :, None], f64(weights)[:, :, None] * f64(y)[np.clip(s, 0, places - 1)], 0)
    want = terms.sum(1)
    # every addition rounds a partial sum of at most sum |terms|, then the result is rounded to its type
    bound = 1.01 * k * F32_STEP * np.abs(terms).sum(1)
    bound += (0 if out_dtype == "f32" else 1.01 * HALF_STEP[out_dtype]) * (np.abs(want) + bound) + LEAST[out_dtype]
    assert (np.abs(f64(out) - want) <= bound).all()


def test_combine_nothing(gpu_ctx):
    gpu_ctx.combine(0, ft.F32, 0, 0, 0, 2, 0, ft.F32, 0, 64)
    out, slots, weights = torch.full((3, 50), 9.0, device="cuda"), torch.zeros(3, 2, dtype=torch.int32, device="cuda"), torch.ones(3, 2, device="cuda")
    gpu_ctx.combine(0, ft.F32, 0, slots.data_ptr(), weights.data_ptr(), 2, out.data_ptr(), ft.F32, 3, 50, stream=stream())
    gpu_ctx.sync()
    assert (out == 0).all()


# --------------------------------------------------------------------------------------------
# the whole layer, streams, graphs, devices
# --------------------------------------------------------------------------------------------

class Layer:
    """route -> quantise -> product + PReLU -> quantise -> product -> combine over buffers of its own."""

    def __init__(self, ctx, T, E, k, D, H, seed, groups=1, top_groups=1):
        g = gen(seed)
        self.ctx, self.T, self.E, self.k, self.D, self.H = ctx, T, E, k, D, H
        self.w1, self.w2 = int8(g, E, H, D), int8(g, E, D, H)
        self.s1, self.s2 = torch.rand(E, H, generator=g) * 1e-3, torch.rand(E, D, generator=g) * 1e-3
        self.h1 = ctx.upload_weights_i8(self.w1.data_ptr(), self.s1.data_ptr(), H, D, experts=E)
        self.h2 = ctx.upload_weights_i8(self.w2.data_ptr(), self.s2.data_ptr(), D, H, experts=E)
        self.bias = torch.randn(E, generator=g) * 0.1
        self.r = ft.Route(E, k, ft.ROUTE_SIGMOID, groups, top_groups, 2, 1, 2.5)
        self.x, self.logits = torch.randn(T, D, generator=g).to(torch.bfloat16), torch.randn(T, E, generator=g)
        self.logits[T - T // 10:] = float("-inf")  # padding

        def new(*shape, dtype=torch.float32):
            return torch.zeros(*shape, dtype=dtype, device="cuda")
        i32, P = torch.int32, T * k
        self.dx, self.dl, self.db = self.x.cuda(), self.logits.cuda(), self.bias.cuda()
        self.experts, self.weights, self.offsets = new(T, k, dtype=i32), new(T, k), new(E + 1, dtype=i32)
        self.rows, self.slots = new(P, dtype=i32), new(T, k, dtype=i32)
        self.q1, self.sc1 = new(T, ft.i8_pitch(D), dtype=torch.int8), new(T)
        self.y1, self.q2, self.sc2 = new(P, H, dtype=torch.bfloat16), new(P, ft.i8_pitch(H), dtype=torch.int8), new(P)
        self.y2, self.out = new(P, D, dtype=torch.float32), new(T, D)

    def run(self, st):
        c, P, p = self.ctx, self.T * self.k, lambda t: t.data_ptr()
        c.route(self.r, p(self.dl), ft.F32, p(self.db), self.T, p(self.experts), p(self.weights), p(self.offsets), p(self.rows), p(self.slots), stream=st)
        c.quantise_i8(p(self.dx), ft.BF16, p(self.q1), p(self.sc1), self.T, self.D, stream=st)
        c.gemm_i8_experts(self.h1, p(self.q1), p(self.sc1), p(self.rows), p(self.offsets), p(self.y1), ft.BF16, self.T, P, 0.5, stream=st)
        c.quantise_i8(p(self.y1), ft.BF16, p(self.q2), p(self.sc2), P, self.H, stream=st)
        c.gemm_i8_experts(self.h2, p(self.q2), p(self.sc2), 0, p(self.offsets), p(self.y2), ft.F32, P, P, 1.0, stream=st)
        c.combine(p(self.y2), ft.F32, P, p(self.slots), p(self.weights), self.k, p(self.out), ft.F32, self.T, self.D, stream=st)

    def check(self):
        """Each step from the device's own input of that step, so that the bounds stay those of one step."""
        P = self.T * self.k
        experts, weights = route(self.dl, self.bias, self.r)
        assert np.array_equal(self.experts.cpu().numpy(), experts)
        for got, want in zip((self.offsets, self.rows, self.slots), plan(experts, self.E)):
            assert np.array_equal(got.cpu().numpy(), want)
        pairs = int(self.offsets[-1])
        q, s = quantise(self.dx)
        assert np.array_equal(self.q1.cpu().numpy()[:, :self.D], q) and np.array_equal(self.sc1.cpu().numpy(), s)
        o = self.offsets.tolist()
        want = expected_experts(torch.from_numpy(q), torch.from_numpy(s), self.rows.cpu(), o, self.w1, self.s1, 0.5, P)[:pairs]
        y1 = f64(self.y1)[:pairs]
        assert (np.abs(y1 - want) <= product_error(want, "bf16")).all()
        q, s = quantise(self.y1)
        assert np.array_equal(self.q2.cpu().numpy()[:, :self.H], q) and np.array_equal(self.sc2.cpu().numpy(), s)
        want = expected_experts(torch.from_numpy(q), torch.from_numpy(s), None, o, self.w2, self.s2, 1.0, P)[:pairs]
        assert (np.abs(f64(self.y2)[:pairs] - want) <= product_error(want, "f32")).all()
        slots = self.slots.cpu().numpy().astype(np.int64)
        terms = np.where((slots >= 0)[:, :, None], f64(self.weights)[:, :, None] * f64(self.y2)[np.clip(slots, 0, P - 1)], 0)
        assert (np.abs(f64(self.out) - terms.sum(1)) <= 1.01 * self.k * F32_STEP * np.abs(terms).sum(1) + 2.0 ** -149).all()

    def free(self):
        self.h1.free()
        self.h2.free()


LAYERS = [(1, 8, 2, 256, 128), (7, 16, 4, 300, 200), (64, 32, 8, 512, 256), (700, 16, 4, 384, 640)]


@pytest.mark.parametrize("T,E,k,D,H", LAYERS, ids=str)
def test_layer_of_experts(T, E, k, D, H, gpu_ctx):
    layer = Layer(gpu_ctx, T, E, k, D, H, T)
    layer.run(stream())
    gpu_ctx.sync()
    layer.check()
    layer.free()


@pytest.mark.parametrize("T,E,k,D,H", LAYERS[1:], ids=str)
def test_layer_captured_and_replayed(T, E, k, D, H, gpu_ctx):
    """Two captured layers of one context, replayed on new inputs, on two streams at once."""
    layers = [Layer(gpu_ctx, T, E, k, D, H, seed, 4, 2) for seed in (1, 2)]
    graphs, streams = [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for layer, st in zip(layers, streams):
        layer.run(st.cuda_stream)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            layer.run(torch.cuda.current_stream().cuda_stream)
        graphs.append(graph)
    for seed in (11, 12):
        for i, layer in enumerate(layers):
            layer.dx.copy_(torch.randn(T, D, generator=gen(seed + 100 * i)))
            layer.dl.copy_(torch.randn(T, E, generator=gen(seed + 200 * i)))
        torch.cuda.synchronize()
        for _ in range(5):
            for graph, st in zip(graphs, streams):
                with torch.cuda.stream(st):
                    graph.replay()
        torch.cuda.synchronize()
        gpu_ctx.sync()
        for layer in layers:
            layer.check()
    for layer in layers:
        layer.free()


FIRST_CALLS = """
import sys
sys.path[:0] = [%r, %r]
import torch
import fastertnn_b200 as ft
from test_gpu_i8 import Layer, gen
ctx = ft.Context(0)
for T, E, k, D, H in ((5, 16, 4, 256, 128), (300, 16, 4, 2048, 1024), (5000, 16, 4, 384, 640)):
    layer = Layer(ctx, T, E, k, D, H, T)
    graph, st = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=st):
        layer.run(torch.cuda.current_stream().cuda_stream)
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    ctx.sync()
    layer.check()
print("all captured")
"""


def test_first_calls_inside_a_capture():
    """A process whose first call of every kernel is made while a stream is captured."""
    here = Path(__file__).resolve().parent
    r = subprocess.run([sys.executable, "-c", FIRST_CALLS % (str(here), str(here.parent))], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "all captured" in r.stdout, r.stderr[-2000:]


def test_results_do_not_change_from_run_to_run(gpu_ctx):
    layer = Layer(gpu_ctx, 513, 16, 4, 512, 256, 5)
    layer.run(stream())
    torch.cuda.synchronize()
    first = layer.out.clone()
    for _ in range(20):
        layer.out.zero_()
        layer.run(stream())
        torch.cuda.synchronize()
        assert torch.equal(first, layer.out)
    layer.free()


def test_behind_a_slow_producer(gpu_ctx):
    """Inputs that are still being written by earlier work on the stream when the calls are made."""
    layer = Layer(gpu_ctx, 64, 32, 8, 512, 256, 8)
    x, logits = layer.dx.clone(), layer.dl.clone()
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        for _ in range(20):
            layer.dx.zero_()
            layer.dl.zero_()
            torch.cuda._sleep(200_000)
            layer.dx.copy_(x)
            layer.dl.copy_(logits)
            layer.run(st.cuda_stream)
    st.synchronize()
    layer.check()
    layer.free()


def test_outputs_of_one_call_as_inputs_of_the_next_without_a_pause(gpu_ctx):
    """Products in a row on one stream, each reading what the one before wrote (launches may overlap up to their waits)."""
    g = gen(21)
    D, M = 512, 300
    w, s = int8(g, D, D), torch.rand(D, generator=g) * 1e-3
    h = gpu_ctx.upload_weights_i8(w.data_ptr(), s.data_ptr(), D, D)
    x = torch.randn(M, D, generator=g).cuda()
    for rows in (1, 40, M):
        q, sc = torch.empty(rows, D, dtype=torch.int8, device="cuda"), torch.empty(rows, device="cuda")
        a = [x[:rows].clone()] + [torch.empty(rows, D, device="cuda") for _ in range(12)]
        for i in range(12):
            gpu_ctx.quantise_i8(a[i].data_ptr(), ft.F32, q.data_ptr(), sc.data_ptr(), rows, D, stream=stream())
            gpu_ctx.gemm_i8(h, q.data_ptr(), sc.data_ptr(), a[i + 1].data_ptr(), ft.F32, rows, 0.5, stream=stream())
        gpu_ctx.sync()
        for i in range(12):
            qq, ss = quantise(a[i])
            want = product(qq, ss, w.numpy(), s.numpy(), 0.5)
            assert (np.abs(f64(a[i + 1]) - want) <= product_error(want, "f32")).all()
    h.free()


def test_on_a_second_device(gpu_ctx):
    if torch.cuda.device_count() < 2:
        pytest.skip("one device")
    ctx = ft.Context(1)
    with torch.cuda.device(1):
        layer = Layer(ctx, 64, 32, 8, 512, 256, 8)
        torch.cuda.set_device(0)
        layer.run(0)
        ctx.sync()
        layer.check()
        with pytest.raises(ft.TnnsError):
            gpu_ctx.gemm_i8_experts(layer.h1, layer.q1.data_ptr(), layer.sc1.data_ptr(), 0, layer.offsets.data_ptr(), layer.y1.data_ptr(), ft.BF16, 64, 512)
        layer.free()
    ctx.close()
    torch.cuda.set_device(0)
