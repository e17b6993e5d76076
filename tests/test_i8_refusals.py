"""CPU suite: calls of the 8-bit operators and the routing that are refused before anything reaches a device."""
import ctypes as C

import pytest

import fastertnn_b200 as ft

CTX = C.create_string_buffer(4096)  # never looked into: every call here is refused on its arguments
P = 1 << 20  # an address that is aligned and never read


def status(name, *args):
    return getattr(ft.load_library(), name)(*args)


QUANTISE = dict(ctx=CTX, x=P, dtype=0, xs=100, q=P, qs=112, scale=P, M=3, K=100, stream=0)


@pytest.mark.parametrize("change", [
    dict(ctx=None), dict(dtype=3), dict(dtype=-1), dict(M=-1), dict(K=0), dict(xs=99), dict(qs=96), dict(qs=104), dict(x=0), dict(q=0), dict(scale=0),
    dict(x=P + 2), dict(dtype=1, x=P + 1), dict(q=P + 8), dict(scale=P + 2)], ids=str)
def test_quantise(change):
    a = {**QUANTISE, **change}
    assert status("tnns_cuda_quantise_i8", *a.values()) == 1
    assert ft.load_library().tnns_cuda_error_detail()


COMBINE = dict(ctx=CTX, y=P, dtype=0, ys=64, places=16, slots=P, weights=P, k=4, out=P, out_dtype=2, os=64, T=4, N=64, stream=0)


@pytest.mark.parametrize("change", [
    dict(ctx=None), dict(dtype=7), dict(out_dtype=7), dict(T=-1), dict(N=0), dict(places=-1), dict(k=0), dict(ys=63), dict(os=63), dict(y=0), dict(slots=0),
    dict(weights=0), dict(out=0), dict(y=P + 2), dict(out=P + 1), dict(slots=P + 2), dict(weights=P + 1)], ids=str)
def test_combine(change):
    assert status("tnns_cuda_combine", *{**COMBINE, **change}.values()) == 1


ROUTE = dict(ctx=CTX, r=None, logits=P, dtype=0, stride=64, bias=0, T=4, experts=P, weights=P, offsets=P, rows=P, slots=P, stream=0)
OK = dict(experts=64, top_k=8, score=0, groups=8, top_groups=4, group_top=2, renormalise=1, scale=1.0)


@pytest.mark.parametrize("change", [
    dict(ctx=None), dict(dtype=3), dict(T=-1), dict(T=1 << 28), dict(stride=63), dict(logits=0), dict(experts=0), dict(weights=0), dict(offsets=0), dict(rows=0),
    dict(slots=0), dict(logits=P + 2), dict(bias=P + 1), dict(experts=P + 2), dict(offsets=P + 2), dict(rows=P + 3), dict(slots=P + 1)], ids=str)
def test_route_arguments(change):
    a = {**ROUTE, "r": C.byref(ft.Route(**OK)), **change}
    assert status("tnns_cuda_route", *a.values()) == 1


@pytest.mark.parametrize("change", [
    dict(experts=0), dict(experts=1025), dict(experts=63), dict(groups=0), dict(groups=64), dict(top_groups=0), dict(top_groups=9), dict(top_k=0), dict(top_k=33),
    dict(top_groups=1, top_k=9), dict(score=2), dict(group_top=0), dict(group_top=3)], ids=str)
def test_route_descriptions(change):
    r = ft.Route(**{**OK, **change})
    assert status("tnns_cuda_route", *{**ROUTE, "r": C.byref(r), "stride": 2000}.values()) == 1


def test_route_without_description():
    assert status("tnns_cuda_route", *ROUTE.values()) == 1


@pytest.mark.parametrize("experts,N,K", [(0, 8, 8), (65536, 8, 8), (1, 0, 8), (1, 8, 0), (1, 8, 131072)])
def test_upload(experts, N, K):
    h = C.c_void_p(123)
    assert status("tnns_cuda_upload_weights_i8", CTX, P, P, experts, N, K, C.byref(h)) == 1
    assert not h.value
    assert status("tnns_cuda_upload_weights_i8", CTX, 0, P, 1, 8, 8, C.byref(h)) == 1
    assert status("tnns_cuda_upload_weights_i8", CTX, P, 0, 1, 8, 8, C.byref(h)) == 1


def test_products_without_weights():
    assert status("tnns_cuda_gemm_i8", CTX, None, P, 16, P, P, 0, 8, 1, 1.0, 0) == 1
    assert status("tnns_cuda_gemm_i8_experts", CTX, None, P, 16, P, 1, P, P, P, 0, 8, 1, 1.0, 0) == 1


def test_sizes():
    assert [ft.i8_pitch(k) for k in (1, 16, 17)] == [16, 16, 32]
    assert C.sizeof(ft.Route) == 8 * 4
