"""GPU suite: one captured layer of experts replayed on inputs that change from replay to replay, without a pause between them."""
import pytest
import torch

import fastertnn_b200 as ft  # noqa: F401
from test_gpu_i8 import Layer, gen

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T,E,k,D,H", [(1, 8, 2, 256, 128), (16, 32, 8, 512, 256), (300, 16, 4, 384, 640), (4000, 16, 4, 256, 128)], ids=str)
def test_replays_with_other_routing(T, E, k, D, H, gpu_ctx):
    """Every replay chooses other experts into the same buffers; no kernel reads what the replay before left there."""
    layer, st = Layer(gpu_ctx, T, E, k, D, H, T, 4, 2), torch.cuda.Stream()
    results = ("experts", "weights", "offsets", "rows", "slots", "out")
    sets = [(torch.randn(T, D, generator=gen(50 + i)).to(torch.bfloat16).cuda(), torch.randn(T, E, generator=gen(90 + i)).cuda()) for i in range(12)]
    want = []
    for x, logits in sets:
        layer.dx.copy_(x)
        layer.dl.copy_(logits)
        torch.cuda.synchronize()
        layer.run(st.cuda_stream)
        torch.cuda.synchronize()
        gpu_ctx.sync()
        layer.check()
        want.append([getattr(layer, n).clone() for n in results])
    assert not torch.equal(want[0][0], want[1][0])
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=st):
        layer.run(torch.cuda.current_stream().cuda_stream)
    got = [[torch.empty_like(t) for t in w] for w in want]
    torch.cuda.synchronize()
    order = torch.randperm(120, generator=gen(T)).tolist()
    for i in order:
        with torch.cuda.stream(st):
            layer.dx.copy_(sets[i % 12][0])
            layer.dl.copy_(sets[i % 12][1])
            graph.replay()
            for a, n in zip(got[i % 12], results):
                a.copy_(getattr(layer, n))
    torch.cuda.synchronize()
    gpu_ctx.sync()
    for g, w in zip(got, want):
        for a, b in zip(g, w):
            assert torch.equal(a, b)
    layer.free()
